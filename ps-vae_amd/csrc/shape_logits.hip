// Between the vocabulary layer's logits and the next token: penalties for tokens of the past, a bias, a temperature and a
// grammar's mask (shape), the log-probability of a given token under the result and its gradient (log_prob), and one
// token drawn from it (draw).  For row r = (b, t), with c_i the number of times id i occurs in the first len_r ids of history[b]:
//     a_i = l_i;  c_i > 0:  a_i = (l_i > 0 ? l_i / rep_b : l_i * rep_b) - freq_b c_i - pres_b
//     y_i = (a_i + bias_i) / T_b   where bit i of allowed[state_r] is set (state < 0: every bit; state >= S: no bit), else -inf
//     log_prob = y_tok - m - log s,  m = max y, s = sum exp(y - m);  d log_prob / d l_i = ([i = tok] - exp(y_i - m) / s) dy_i/dl_i
//     draw:  min(#{i : cdf_i <= u cdf_last}, last i of positive probability),  cdf the running sum of exp(y - m) in index order
//
// Layout.  A row is cut into units of THREADS * VEC * K elements, a thread's VEC neighbours being one 16-byte load; inside a unit
// every wave owns a contiguous piece, so a wave's partial results are results of an index range.  The counts c_i of a unit live in
// LDS only: the unit's threads walk the row's history (8 bytes an entry, from L2 after the row's first unit) and add to 32-bit
// LDS counters, whose sums do not depend on the order.  No count table of [rows, V] is ever kept or read - it would be as
// large as the logits - and the logits are requested before the walk, so that it runs while they travel.
#include "common.h"

#include <limits.h>
#include <math.h>
#include <type_traits>

namespace {

constexpr int NT = 256;              // threads per workgroup
constexpr int WAVES = NT / 64;
constexpr float NEG = -__builtin_inff();

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int VEC = 4; };
template <> struct Elem<__bf16> { static constexpr int VEC = 8; };
template <> struct Elem<_Float16> { static constexpr int VEC = 8; };

// 16 bytes of a row at any element's address: rows of an odd width start anywhere.  (Global loads and stores of 4 dwords
// need no more than the element's alignment on this target.)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[Elem<T>::VEC]; };
struct __attribute__((packed, aligned(4))) Float4u { float v[4]; };

struct Args {
    int R, T, V, L, S;
    const void *logits;
    long long ld_b, ld_t;
    const int64_t *history;
    long long ld_history;
    const int32_t *history_len;
    int len_per_row;
    const float *rep_p, *pres_p, *freq_p, *temp_p;
    float rep, pres, freq, temp;
    const float *bias;
    long long ld_bias;
    const int32_t *allowed;
    long long ld_allowed;
    const int32_t *state;
    int state_per_row;
    int units;                       // units per row
};

// What a row needs besides its logits.
template <typename T> struct Row {
    const T *x;
    const int64_t *hist;
    int len;
    float rep, pres, freq, temp;
    const float *bias;
    const uint32_t *mask;            // null: every token allowed
    bool none;                       // no token allowed
};

__device__ __forceinline__ float positive(float v) { return v > 0.f && v < __builtin_inff() ? v : __builtin_nanf(""); }

template <typename T> __device__ __forceinline__ Row<T> row_of(const Args &a, int r) {
    const int b = a.T == 1 ? r : (int)((unsigned)r / (unsigned)a.T), t = r - b * a.T;
    Row<T> w;
    w.x = (const T *)a.logits + b * a.ld_b + t * a.ld_t;
    w.hist = nullptr, w.len = 0;
    if (a.history) {
        w.hist = a.history + b * a.ld_history;
        const int n = a.history_len ? a.history_len[a.len_per_row ? r : b] : a.L;
        w.len = n < 0 ? 0 : (n < a.L ? n : a.L);
    }
    // a repetition or temperature that is not a positive finite number makes what it touches NaN
    w.rep = positive(a.rep_p ? a.rep_p[b] : a.rep);
    w.pres = a.pres_p ? a.pres_p[b] : a.pres;
    w.freq = a.freq_p ? a.freq_p[b] : a.freq;
    w.temp = positive(a.temp_p ? a.temp_p[b] : a.temp);
    w.bias = a.bias ? a.bias + b * a.ld_bias : nullptr;
    w.mask = nullptr, w.none = false;
    if (a.allowed) {
        const int s = a.state ? a.state[a.state_per_row ? r : b] : (a.S == 1 ? 0 : b);
        w.none = s >= a.S;
        if (s >= 0 && s < a.S) w.mask = (const uint32_t *)a.allowed + s * a.ld_allowed;
    }
    return w;
}

// VEC values from p[0 .. left): the whole 16 bytes where they are inside, one by one at a row's end.
template <typename T> __device__ __forceinline__ Pack<T> load_pack(const T *p, int left) {
    Pack<T> v;
    if (left >= Elem<T>::VEC) {
        v = *reinterpret_cast<const Pack<T> *>(p);
    } else {
#pragma unroll
        for (int j = 0; j < Elem<T>::VEC; ++j) v.v[j] = j < left ? p[j] : (T)0.f;
    }
    return v;
}
template <typename T> __device__ __forceinline__ void store_pack(T *p, const Pack<T> &v, int left) {
    if (left >= Elem<T>::VEC) {
        *reinterpret_cast<Pack<T> *>(p) = v;
    } else {
#pragma unroll
        for (int j = 0; j < Elem<T>::VEC; ++j)
            if (j < left) p[j] = v.v[j];
    }
}

// ---- bits.  Bit j of `bits` as a word of ones or zeros: one bit-field extract, and a masked value is then one bit-select
// (a compare and a conditional move per value would be three).
__device__ __forceinline__ int bit_word(uint32_t bits, int j) { return (int)(bits << (31 - j)) >> 31; }
__device__ __forceinline__ float select(int word, float yes, float no) {
    return __int_as_float((word & __float_as_int(yes)) | (~word & __float_as_int(no)));
}
__device__ __forceinline__ double select(int word, double yes, double no) {
    const long long w = word;
    return __longlong_as_double((w & __double_as_longlong(yes)) | (~w & __double_as_longlong(no)));
}

// ---- sums and maxima over the wave in the vector unit's own lane permutes: within rows of 16 lanes, then from row to row.  A lane
// without a source takes `none`.
template <int CTRL, int ROWS> __device__ __forceinline__ float lane_move(float none, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS> __device__ __forceinline__ double lane_move(double none, double v) {
    const long long n = __double_as_longlong(none), x = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp((int)n, (int)x, CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp((int)(n >> 32), (int)(x >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo));
}
constexpr int ROW_SHR1 = 0x111, ROW_SHR2 = 0x112, ROW_SHR4 = 0x114, ROW_SHR8 = 0x118, BCAST15 = 0x142, BCAST31 = 0x143;

__device__ __forceinline__ float from_lane(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ double from_lane(double v, int lane) {
    const long long x = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_readlane((int)x, lane), hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
    return __longlong_as_double((long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo));
}
template <typename C> __device__ __forceinline__ C wave_scan(C v) {   // inclusive, in lane order
    v += lane_move<ROW_SHR1, 0xf>((C)0, v);
    v += lane_move<ROW_SHR2, 0xf>((C)0, v);
    v += lane_move<ROW_SHR4, 0xf>((C)0, v);
    v += lane_move<ROW_SHR8, 0xf>((C)0, v);
    v += lane_move<BCAST15, 0xa>((C)0, v);
    v += lane_move<BCAST31, 0xc>((C)0, v);
    return v;
}
template <typename C> __device__ __forceinline__ C wave_sum(C v) { return from_lane(wave_scan(v), 63); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
template <typename C> __device__ __forceinline__ C wave_max(C v) {
    const C none = (C)NEG;
    v = larger(v, lane_move<ROW_SHR1, 0xf>(none, v));
    v = larger(v, lane_move<ROW_SHR2, 0xf>(none, v));
    v = larger(v, lane_move<ROW_SHR4, 0xf>(none, v));
    v = larger(v, lane_move<ROW_SHR8, 0xf>(none, v));
    v = larger(v, lane_move<BCAST15, 0xa>(none, v));
    v = larger(v, lane_move<BCAST31, 0xc>(none, v));
    return from_lane(v, 63);
}

// 1 / x by Newton's iteration from the unit's estimate (1 ulp; 2^-22 for doubles): a row's few reciprocals cost 3 and 5 instructions
// instead of a division's 10 and 14.
__device__ __forceinline__ float reciprocal(float x) {
    const float r = __builtin_amdgcn_rcpf(x);
    return fmaf(fmaf(-x, r, 1.f), r, r);
}
__device__ __forceinline__ double reciprocal(double x) {
    double r = __builtin_amdgcn_rcp(x);
    r = fma(fma(-x, r, 1.), r, r);
    return fma(fma(-x, r, 1.), r, r);
}

// The penalties and the last factor of a row in type C (float; double for draws).  `unit` scales the result: 1, or log2 e where it goes
// into a power of two.
template <typename C> struct Rule {
    C rep, inv_rep, pres, freq, scale;
    template <typename T> __device__ Rule(const Row<T> &w, C unit)
        : rep((C)w.rep), inv_rep(reciprocal((C)w.rep)), pres((C)w.pres), freq((C)w.freq), scale(unit * reciprocal((C)w.temp)) {}
    __device__ __forceinline__ C factor(C x) const { return x > (C)0 ? inv_rep : rep; }   // what a seen token's logit is multiplied by
    __device__ __forceinline__ C penalised(C x, int c) const { return x * factor(x) - (freq * (C)c + pres); }
};

// y in units of 1 / scale, rounded by itself.  Equal values have to stay equal: fused with the subtraction of the row's maximum that follows, the
// product would keep its unrounded rest, which for values near the type's lowest is far from 0.
template <typename C> __device__ __forceinline__ C scaled(C y, C scale) {
#pragma clang fp contract(off)
    return y * scale;
}

// The bias of VEC elements, zeros past the row's end.
template <int VEC> __device__ __forceinline__ void load_bias(const float *bias, int left, float (&b)[VEC]) {
    if (left >= VEC) {
#pragma unroll
        for (int q = 0; q < VEC / 4; ++q) {
            const Float4u f = *reinterpret_cast<const Float4u *>(bias + 4 * q);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[4 * q + j] = f.v[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) b[j] = j < left ? bias[j] : 0.f;
    }
}

// Where a thread stands: which row, which unit, which elements.
template <typename T, int K, int ROWS> struct Place {
    static constexpr int VEC = Elem<T>::VEC, THREADS = NT / ROWS, SPAN = THREADS * VEC * K;
    int r, unit, tid, lane, wave;    // row; unit of the row; thread, lane and wave inside the row's group
    bool live;
    __device__ Place(const Args &a, int block) {
        tid = threadIdx.x & (THREADS - 1), lane = threadIdx.x & 63, wave = ROWS == 1 ? __builtin_amdgcn_readfirstlane(tid >> 6) : 0;
        if (ROWS == 1) {
            r = a.units == 1 ? block : (int)((unsigned)block / (unsigned)a.units), unit = block - r * a.units;
        } else {
            r = block * ROWS + __builtin_amdgcn_readfirstlane((int)threadIdx.x / THREADS), unit = 0;
        }
        live = r < a.R;
        if (!live) r = a.R - 1;
    }
    __device__ __forceinline__ int base() const { return unit * SPAN; }
    __device__ __forceinline__ int at(int k) const { return ((wave * K + k) * 64 + lane) * VEC; }   // inside the unit
};

// What the past does to a unit: the count of every id in `cell`, and one bit for every id that occurs in `seen`.
template <int SPAN> struct Past {
    int cell[SPAN];
    uint32_t seen[SPAN / 32];
};
struct NoPast {};

// Counts the ids [base, base + n) of the row's history.  Every thread of the workgroup calls it (barriers); the calling group's threads
// number `tid` of `threads`.
template <int SPAN>
__device__ __forceinline__ void count_unit(Past<SPAN> &past, const int64_t *hist, int len, int base, int n, int tid, int threads) {
    for (int i = tid * 4; i < SPAN; i += threads * 4) *reinterpret_cast<int4 *>(past.cell + i) = make_int4(0, 0, 0, 0);
    for (int i = tid; i < SPAN / 32; i += threads) past.seen[i] = 0u;
    __syncthreads();
#pragma unroll 4
    for (int j = tid; j < len; j += threads) {
        const unsigned long long at = (unsigned long long)(hist[j] - base);   // ids outside the vocabulary fall outside every unit
        if (at < (unsigned long long)n) {
            atomicAdd(&past.cell[at], 1);
            atomicOr(&past.seen[at >> 5], 1u << (at & 31));
        }
    }
    __syncthreads();
}

// A thread's part of a unit: K packs of logits with their bias and mask, requested before the history is walked, and what the walk found.
//   PAST 0: no history.  1: counts (and bits).  2: `cell` holds the finished value y of every seen id in place of its count, computed
//   once by one thread; a pack of 64 * VEC ids that has a seen one then costs two instructions an element more, not eight.
template <typename T, int K, int ROWS, int PAST> struct Unit {
    using P = Place<T, K, ROWS>;
    using Lds = std::conditional_t<PAST != 0, Past<P::SPAN>, NoPast>;
    static constexpr int VEC = P::VEC;
    P p;
    Row<T> w;
    Pack<T> x[K];
    float b[K][VEC];
    uint32_t allow[K];               // bit j: element j of the pack is in the row and allowed
    Lds *past;
    int n;                           // elements of the unit that the row has

    __device__ __forceinline__ int left(int k) const { return n - p.at(k); }
    __device__ __forceinline__ int element(int k) const { return p.base() + p.at(k); }
    __device__ Unit(const Args &a, int block, Lds *lds, bool want_logits) : p(a, block), w(row_of<T>(a, p.r)) {
        const int base = p.base();
        n = p.live ? (a.V - base < P::SPAN ? a.V - base : P::SPAN) : 0;
        past = lds + (ROWS == 1 ? 0 : (int)threadIdx.x / P::THREADS);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            allow[k] = 0xffffffffu;
#pragma unroll
            for (int j = 0; j < VEC; ++j) b[k][j] = 0.f;
        }
        if (n == P::SPAN) {          // (no lane's load hangs on a test of its own)
            if (want_logits) {
#pragma unroll
                for (int k = 0; k < K; ++k) x[k] = *reinterpret_cast<const Pack<T> *>(w.x + element(k));
                if (w.bias) {
#pragma unroll
                    for (int k = 0; k < K; ++k) load_bias<VEC>(w.bias + element(k), VEC, b[k]);
                }
            }
            if (w.mask) {
#pragma unroll
                for (int k = 0; k < K; ++k) allow[k] = w.mask[element(k) >> 5] >> (element(k) & 31);   // (whole packs: one word)
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int l = left(k);
                if (want_logits) {
                    x[k] = load_pack(w.x + element(k), l);
                    if (w.bias) load_bias<VEC>(w.bias + element(k), l, b[k]);
                }
                if (w.mask && l > 0) allow[k] = w.mask[element(k) >> 5] >> (element(k) & 31);
                allow[k] &= l >= VEC ? 0xffffffffu : l > 0 ? (1u << l) - 1u : 0u;
            }
        }
        if (w.none) {
#pragma unroll
            for (int k = 0; k < K; ++k) allow[k] = 0u;
        }
        if constexpr (PAST != 0) count_unit(*past, w.hist, p.live ? w.len : 0, base, n, p.tid, P::THREADS);
    }
    // PAST 2: one thread for each seen id - the one that takes its bit - leaves y in its cell; the bits are set again as they are taken.
    __device__ __forceinline__ void finish_seen(const Rule<float> &rule) {
        for (int i = p.tid; i < P::SPAN / 32; i += P::THREADS) past->seen[i] = 0u;
        __syncthreads();
        const int base = p.base(), len = p.live ? w.len : 0;
#pragma unroll 4
        for (int j = p.tid; j < len; j += P::THREADS) {
            const unsigned long long at = (unsigned long long)(w.hist[j] - base);
            if (at < (unsigned long long)n) {
                const uint32_t bit = 1u << (at & 31);
                if (!(atomicOr(&past->seen[at >> 5], bit) & bit)) {
                    const int i = base + (int)at;
                    const float v = rule.penalised((float)w.x[i], past->cell[at]) + (w.bias ? w.bias[i] : 0.f);
                    past->cell[at] = __float_as_int(scaled(v, rule.scale));
                }
            }
        }
        __syncthreads();
    }
    // bit j: element j of pack k has been seen; 0 in every lane unless one of the wave has a bit
    __device__ __forceinline__ uint32_t seen(int k) const {
        if constexpr (PAST == 0) return 0u;
        else return (reinterpret_cast<const uint8_t *>(past->seen)[p.at(k) >> 3] >> (p.at(k) & 7)) & ((1u << VEC) - 1u);
    }
    __device__ __forceinline__ void cells(int k, int (&c)[VEC]) const {
        if constexpr (PAST != 0) {
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
                const int4 v = *reinterpret_cast<const int4 *>(past->cell + p.at(k) + 4 * q);
                c[4 * q] = v.x, c[4 * q + 1] = v.y, c[4 * q + 2] = v.z, c[4 * q + 3] = v.w;
            }
        }
    }
    // y of pack k, before the mask
    __device__ __forceinline__ void values(int k, const Rule<float> &rule, float (&y)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = scaled((float)x[k].v[j] + b[k][j], rule.scale);
        if (PAST == 2) {
            const uint32_t s = seen(k);
            if (__ballot(s != 0)) {
                int c[VEC];
                cells(k, c);
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[j] = select(bit_word(s, j), __int_as_float(c[j]), y[j]);
            }
        }
    }
    __device__ __forceinline__ void values(int k, const Rule<double> &rule, double (&y)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = (double)(float)x[k].v[j];
        if (PAST == 1) {
            const uint32_t s = seen(k);
            if (__ballot(s != 0)) {
                int c[VEC];
                cells(k, c);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (c[j] > 0) y[j] = rule.penalised(y[j], c[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = scaled(y[j] + (double)b[k][j], rule.scale);
    }
};

template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void shape_fwd_kernel(Args a, T *__restrict__ out, long long ld_out) {
    using U = Unit<T, K, ROWS, HIST ? 2 : 0>;
    __shared__ __align__(16) typename U::Lds lds[ROWS];
    U u(a, blockIdx.x, lds, true);
    const Rule<float> rule(u.w, 1.f);
    if constexpr (HIST) u.finish_seen(rule);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float v[U::VEC];
        u.values(k, rule, v);
        Pack<T> y;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) y.v[j] = (T)select(bit_word(u.allow[k], j), v[j], NEG);
        store_pack(out + u.p.r * ld_out + u.element(k), y, u.left(k));
    }
}

// dl = g dy/dl; the logits are read only where the sign of a seen token's decides.
template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void shape_bwd_kernel(Args a, const T *__restrict__ g, long long ld_gb, long long ld_gt,
                                                       T *__restrict__ dx, long long ld_dx) {
    using U = Unit<T, K, ROWS, HIST ? 1 : 0>;
    __shared__ __align__(16) typename U::Lds lds[ROWS];
    U u(a, blockIdx.x, lds, false);
    const Rule<float> rule(u.w, 1.f);
    const int b = a.T == 1 ? u.p.r : (int)((unsigned)u.p.r / (unsigned)a.T), t = u.p.r - b * a.T;
    const T *gr = g + b * ld_gb + t * ld_gt;
#pragma unroll
    for (int k = 0; k < K; ++k) u.x[k] = load_pack(gr + u.element(k), u.left(k));
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = u.element(k);
        float v[U::VEC];
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) v[j] = (float)u.x[k].v[j] * rule.scale;
        if (HIST) {
            const uint32_t s = u.seen(k);
            if (__ballot(s != 0)) {
#pragma unroll
                for (int j = 0; j < U::VEC; ++j)
                    if ((s >> j) & 1u) v[j] *= rule.factor((float)u.w.x[i + j]);
            }
        }
        Pack<T> d;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) d.v[j] = (T)select(bit_word(u.allow[k], j), v[j], 0.f);
        store_pack(dx + u.p.r * ld_dx + i, d, u.left(k));
    }
}

__device__ __forceinline__ float log_prob_of(float y_tok, float m, float s) {
    return m == NEG && s == 0.f ? NEG : y_tok - m - logf(s);   // (nothing allowed: log 0)
}

// a row's token as an element of it, or one that no pack holds
__device__ __forceinline__ int token_of(long long tok, int V) { return tok >= 0 && tok < V ? (int)tok : INT_MIN / 2; }

// exp(y - m) as a power of two.  (The difference first: a row of the type's lowest values - masked by hand - has an m whose multiple of
// log2 e overflows.)  A piece that allows nothing has m = -inf: 0 in its place.
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float reference_of(float m) { return m == NEG ? 0.f : m; }
__device__ __forceinline__ float exp_from(float y, float m) { return __builtin_amdgcn_exp2f((y - m) * LOG2E); }

// Per wave: the maximum and the sum of exponentials of its piece; per row: the shaped value of its token.  ROWS > 1: the wave has the
// whole row and finishes it.  Sums are 32-bit: 64 lanes of at most VEC * K terms each, then 6 levels, so the relative error stays below
// (VEC * K + 6 + pieces) * 2^-24.
template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void log_prob_fwd_kernel(Args a, const int64_t *__restrict__ tokens, float *__restrict__ lp,
                                                          float2 *__restrict__ stats, float2 *__restrict__ part,
                                                          float *__restrict__ target) {
    using U = Unit<T, K, ROWS, HIST ? 2 : 0>;
    __shared__ __align__(16) typename U::Lds lds[ROWS];
    U u(a, blockIdx.x, lds, true);
    const Rule<float> rule(u.w, 1.f);
    if constexpr (HIST) u.finish_seen(rule);
    if (!u.p.live) return;
    const int tok = token_of(tokens[u.p.r], a.V);
    float y[K][U::VEC];
    float m = NEG, yt = 0.f;
    bool mine = false;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        u.values(k, rule, y[k]);
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) {
            y[k][j] = select(bit_word(u.allow[k], j), y[k][j], NEG);
            m = fmaxf(m, y[k][j]);
        }
        const unsigned at = (unsigned)(tok - u.element(k));
        if (at < (unsigned)U::VEC) {
            mine = true;
#pragma unroll
            for (int j = 0; j < U::VEC; ++j)
                if (j == (int)at) yt = y[k][j];
        }
    }
    m = wave_max(m);
    const float from = reference_of(m);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) s += exp_from(y[k][j], from);
    s = wave_sum(s);
    if (ROWS == 1) {
        if (mine) target[u.p.r] = yt;
        if (u.p.lane == 0) part[(long long)u.p.r * a.units * WAVES + u.p.unit * WAVES + u.p.wave] = make_float2(m, s);
        return;
    }
    const unsigned long long owner = __ballot(mine);
    const float v = owner ? log_prob_of(from_lane(yt, __ffsll((long long)owner) - 1), m, s) : 0.f;
    if (u.p.lane == 0) lp[u.p.r] = v, stats[u.p.r] = make_float2(m, s);
}

// One wave per row: the pieces' maxima and sums joined.
__global__ __launch_bounds__(NT) void log_prob_join_kernel(int R, int V, int pieces, const int64_t *__restrict__ tokens,
                                                           const float2 *__restrict__ part, const float *__restrict__ target,
                                                           float *__restrict__ lp, float2 *__restrict__ stats) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (r >= R) return;
    const float2 *p = part + (long long)r * pieces;
    float m = NEG;
    for (int i = lane; i < pieces; i += 64) m = fmaxf(m, p[i].x);
    m = wave_max(m);
    float s = 0.f;
    for (int i = lane; i < pieces; i += 64) {
        const float2 q = p[i];
        s += q.x == NEG ? q.y : q.y * __expf(q.x - m);   // (an empty piece adds its 0, one that holds nothing but NaN its NaN)
    }
    s = wave_sum(s);
    if (lane != 0) return;
    const long long tok = tokens[r];
    lp[r] = tok >= 0 && tok < V ? log_prob_of(target[r], m, s) : 0.f;
    stats[r] = make_float2(m, s);
}

template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void log_prob_bwd_kernel(Args a, const int64_t *__restrict__ tokens, const float2 *__restrict__ stats,
                                                          const float *__restrict__ g, T *__restrict__ dx, long long ld_dx) {
    using U = Unit<T, K, ROWS, HIST ? 2 : 0>;
    __shared__ __align__(16) typename U::Lds lds[ROWS];
    U u(a, blockIdx.x, lds, true);
    const Rule<float> rule(u.w, 1.f);
    if constexpr (HIST) u.finish_seen(rule);
    const int tok = token_of(tokens[u.p.r], a.V);
    const float2 st = stats[u.p.r];
    const bool zero = tok < 0 || (st.x == NEG && st.y == 0.f);   // a row without a token, or with none allowed
    const float at_token = g[u.p.r] * rule.scale, others = -at_token / st.y, from = reference_of(st.x);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = u.element(k);
        float v[U::VEC];
        u.values(k, rule, v);
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) v[j] = others * exp_from(v[j], from);
        const unsigned at = (unsigned)(tok - i);
        if (at < (unsigned)U::VEC) {
#pragma unroll
            for (int j = 0; j < U::VEC; ++j)
                if (j == (int)at) v[j] += at_token;
        }
        if (HIST) {
            const uint32_t s = u.seen(k);
            if (__ballot(s != 0)) {
#pragma unroll
                for (int j = 0; j < U::VEC; ++j) v[j] = select(bit_word(s, j), v[j] * rule.factor((float)u.x[k].v[j]), v[j]);
            }
        }
        const uint32_t bits = zero ? 0u : u.allow[k];
        Pack<T> d;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) d.v[j] = (T)select(bit_word(bits, j), v[j], 0.f);
        store_pack(dx + u.p.r * ld_dx + i, d, u.left(k));
    }
}

// ---- draw.  The pick is a decision: with a running sum in 32 bits, u * total falls on the wrong side of some boundary about once in
// 1e3 .. 1e4 rows at V = 1e5 (V boundaries, each off by ~1e-8), and differently for every tiling.  So values, exponentials and sums are
// 64-bit here: the pick is the one of the exact distribution but for ~1e-9 of the rows, whatever the tiling.
struct Piece {
    double s, m;                     // sum of 2^(z - m), largest z;  z = y log2 e
};
constexpr double NEG64 = -__builtin_inf(), LOG2E64 = 1.4426950408889634;

// 2^z for z <= 0 (0 below 2^-1074): 2^n of the nearest whole number times the series of 2^r = e^(r ln 2), |r| <= 1/2, whose rest after
// the 11th power is below 7e-15 of the value.
__device__ __forceinline__ double power_of_two(double z) {
    z = fmax(z, -1080.);
    const double n = rint(z), r = z - n;
    double p = 4.4455382718708116e-10;
    p = fma(p, r, 7.054911620801123e-09);
    p = fma(p, r, 1.01780860092397e-07);
    p = fma(p, r, 1.321548679014431e-06);
    p = fma(p, r, 1.5252733804059841e-05);
    p = fma(p, r, 0.0001540353039338161);
    p = fma(p, r, 0.0013333558146428443);
    p = fma(p, r, 0.009618129107628477);
    p = fma(p, r, 0.05550410866482158);
    p = fma(p, r, 0.24022650695910072);
    p = fma(p, r, 0.6931471805599453);
    p = fma(p, r, 1.);
    return ldexp(p, (int)n);
}

// e[k][j] = 2^(z - m) of the thread's elements (0 where not allowed), m the wave's largest z, which is returned: NaN if a value that is
// allowed is NaN.
template <typename T, int K, int ROWS, int PAST, int VEC>
__device__ __forceinline__ double exp_values(const Unit<T, K, ROWS, PAST> &u, double (&e)[K][VEC]) {
    const Rule<double> rule(u.w, LOG2E64);
    double m = NEG64;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        u.values(k, rule, e[k]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            e[k][j] = select(bit_word(u.allow[k], j), e[k][j], NEG64);
            bad |= e[k][j] != e[k][j];
            m = fmax(m, e[k][j]);
        }
    }
    m = wave_max(m);
    const double from = m == NEG64 ? 0. : m;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[k][j] = power_of_two(e[k][j] - from);
    return __ballot(bad) ? __builtin_nan("") : m;
}

// The first element, in index order, at which the running sum (starting from `before`) exceeds thr; the last positive one if it never
// does.  Returns whether it did, the element's index inside the wave's piece (-1: nothing positive) and its e.  The whole wave calls it.
struct Pick {
    double value;
    int index;
    bool over;
};
template <int K, int VEC> __device__ __forceinline__ Pick pick_in_wave(const double (&e)[K][VEC], double before, double thr) {
    Pick found = {0., -1, false};
    double cum = before;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        double s = 0.;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += e[k][j];
        const double inc = wave_scan(s);
        const unsigned long long some = __ballot(s > 0.), hit = __ballot(s > 0. && cum + inc > thr);
        if (!found.over && some) {
            // inside each lane: the first positive element past thr, else the last positive one
            int mine = -1;
            double run = cum + (inc - s), v = 0.;
            bool over = false;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (e[k][j] > 0. && !over) run += e[k][j], mine = j, v = e[k][j], over = run > thr;
            const int l = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
            found.index = (k * 64 + l) * VEC + __builtin_amdgcn_readlane(mine, l), found.value = from_lane(v, l), found.over = hit != 0;
        }
        cum += from_lane(inc, 63);
    }
    return found;
}

__device__ __forceinline__ float draw_log_prob(double value, double total) { return (float)log(value / total); }

// a whole row in a wave
template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void draw_row_kernel(Args a, const float *__restrict__ uniforms, long long ld_u, int64_t empty,
                                                      int64_t *__restrict__ out, float *__restrict__ lp) {
    using U = Unit<T, K, ROWS, HIST ? 1 : 0>;
    __shared__ __align__(16) typename U::Lds lds[ROWS];
    U u(a, blockIdx.x, lds, true);
    if (!u.p.live) return;
    double e[K][U::VEC];
    const double m = exp_values(u, e);
    double s = 0.;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) s += e[k][j];
    s = wave_sum(s);
    const Pick pick = pick_in_wave(e, 0., (double)uniforms[u.p.r * ld_u] * s);
    if (u.p.lane == 0) {
        const bool ok = s > 0. && m < __builtin_inf() && pick.index >= 0;
        out[u.p.r] = ok ? pick.index : empty;
        lp[u.p.r] = ok ? draw_log_prob(pick.value, s) : (m == NEG64 ? NEG : __builtin_nanf(""));
    }
}

template <typename T, int K, bool HIST>
__global__ __launch_bounds__(NT) void draw_piece_kernel(Args a, Piece *__restrict__ part) {
    using U = Unit<T, K, 1, HIST ? 1 : 0>;
    __shared__ __align__(16) typename U::Lds lds[1];
    U u(a, blockIdx.x, lds, true);
    double e[K][U::VEC];
    const double m = exp_values(u, e);
    double s = 0.;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) s += e[k][j];
    s = wave_sum(s);
    if (u.p.lane == 0) part[(long long)u.p.r * a.units * WAVES + u.p.unit * WAVES + u.p.wave] = Piece{s, m};
}

// One workgroup per row: the pieces joined in index order, the piece that holds u * total found, and its elements computed and walked
// again, a slab of it for each wave.
template <typename T, int K, bool HIST>
__global__ __launch_bounds__(NT) void draw_join_kernel(Args a, const Piece *__restrict__ part, const float *__restrict__ uniforms,
                                                       long long ld_u, int64_t empty, int64_t *__restrict__ out,
                                                       float *__restrict__ lp) {
    constexpr int VEC = Elem<T>::VEC, SPAN = 64 * VEC * K;             // a piece: what one wave of draw_piece_kernel had
    constexpr int SLABS = K < WAVES ? 1 : K / WAVES, USED = K / SLABS;   // packs for each of the waves that take part
    __shared__ __align__(16) std::conditional_t<HIST, Past<SPAN>, NoPast> past;
    __shared__ double sums[WAVES];
    __shared__ Pick picks[WAVES];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), pieces = a.units * WAVES;
    const Piece *p = part + (long long)r * pieces;
    double m = NEG64;
    bool bad = false;
    for (int i = lane; i < pieces; i += 64) m = fmax(m, p[i].m), bad |= p[i].m != p[i].m;
    m = wave_max(m);
    const bool nan = __ballot(bad) != 0;
    if (nan || !(m > NEG64 && m < __builtin_inf())) {   // (the same in every wave)
        if (threadIdx.x == 0) out[r] = empty, lp[r] = !nan && m == NEG64 ? NEG : __builtin_nanf("");
        return;
    }
    double total = 0.;
    for (int base = 0; base < pieces; base += 64) {
        const int i = base + lane;
        total += wave_sum(i < pieces ? p[i].s * power_of_two(p[i].m - m) : 0.);
    }
    // every wave has the same total and comes to the same piece
    const double thr = (double)uniforms[r * ld_u] * total;
    int found = 0;
    bool over = false;
    double cum = 0., before = 0.;
    for (int base = 0; base < pieces && !over; base += 64) {
        const int i = base + lane;
        const double w = i < pieces ? p[i].s * power_of_two(p[i].m - m) : 0.;
        const double inc = wave_scan(w), ahead = cum + (inc - w);
        const unsigned long long some = __ballot(w > 0.), hit = __ballot(w > 0. && cum + inc > thr);
        if (some) {
            const int l = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
            found = base + l, before = from_lane(ahead, l), over = hit != 0;
        }
        cum += from_lane(inc, 63);
    }
    const Row<T> w = row_of<T>(a, r);
    const int base = found * SPAN, n = a.V - base < SPAN ? a.V - base : SPAN;   // (a piece with a positive sum begins inside the row)
    if constexpr (HIST) count_unit(past, w.hist, w.len, base, n, threadIdx.x, NT);
    double e[SLABS][VEC];
    double s = 0.;
    if (wave < USED) {
        const Rule<double> rule(w, LOG2E64);
#pragma unroll
        for (int k = 0; k < SLABS; ++k) {
            const int at = ((wave * SLABS + k) * 64 + lane) * VEC, left = n - at, i = base + at;
            const Pack<T> x = load_pack(w.x + i, left);
            const uint32_t bits = left > 0 ? (w.mask ? w.mask[i >> 5] >> (i & 31) : 0xffffffffu) : 0u;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                e[k][j] = 0.;
                if (j < left && ((bits >> j) & 1u)) {
                    double y = (double)(float)x.v[j];
                    if constexpr (HIST) {
                        if (past.cell[at + j] > 0) y = rule.penalised(y, past.cell[at + j]);
                    }
                    e[k][j] = power_of_two(scaled(y + (w.bias ? (double)w.bias[i + j] : 0.), rule.scale) - m);
                }
                s += e[k][j];
            }
        }
        s = wave_sum(s);
        if (lane == 0) sums[wave] = s;
    }
    __syncthreads();
    if (wave < USED) {
        for (int v = 0; v < wave; ++v) before += sums[v];
        const Pick pick = pick_in_wave(e, before, thr);
        if (lane == 0) picks[wave] = pick;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Pick best = {0., -1, false};
        for (int v = 0; v < USED && !best.over; ++v)
            if (picks[v].index >= 0) best = picks[v], best.index += v * SLABS * 64 * VEC;
        out[r] = best.index >= 0 ? base + best.index : empty;
        lp[r] = best.index >= 0 ? draw_log_prob(best.value, total) : __builtin_nanf("");
    }
}

// ---- host
constexpr int ROW_MAX = 1024;        // widest vocabulary of the wave-per-row form
constexpr long long MAX_BLOCKS = (1ll << 24) - 1;   // a launch holds fewer than 2^32 threads

int elem_size(int dtype) { return dtype == PSVAE_F32 ? 4 : 2; }

// How a call is cut: rows per workgroup and the loads per thread (as elements per thread, 8 .. 32).
struct Cut {
    bool wave_rows;
    int per_thread, units;
    long long blocks;
};
Cut cut_of(const psvae_shaping *s) {
    Cut c;
    const long long R = (long long)s->B * s->T;
    c.wave_rows = s->V <= ROW_MAX;
    if (c.wave_rows) {
        c.per_thread = s->V <= 512 ? 8 : 16, c.units = 1;
        c.blocks = (R + WAVES - 1) / WAVES;
        return c;
    }
    // units of 8192 elements; of 2048 where those would leave compute units idle
    c.per_thread = R * psvae_cdiv(s->V, NT * 32) < 512 ? 8 : 32;
    c.units = psvae_cdiv(s->V, NT * c.per_thread);
    c.blocks = R * c.units;
    return c;
}

int check_shaping(const char *fn, const psvae_shaping *s, Args *a) {
    PSVAE_REQUIRE(s != nullptr, PSVAE_EINVAL, "%s: null description", fn);
    PSVAE_REQUIRE(s->B >= 0 && s->T >= 1 && s->V >= 1, PSVAE_EINVAL, "%s: bad sizes B=%d T=%d V=%d", fn, s->B, s->T, s->V);
    PSVAE_REQUIRE(s->dtype == PSVAE_F32 || s->dtype == PSVAE_BF16 || s->dtype == PSVAE_F16, PSVAE_EINVAL, "%s: unknown dtype %d", fn,
                  s->dtype);
    PSVAE_REQUIRE(s->V <= (1 << 30) && (long long)s->B * s->T < (1ll << 31), PSVAE_ETOOLARGE, "%s: %d x %d rows of %d", fn, s->B, s->T,
                  s->V);
    PSVAE_REQUIRE(cut_of(s).blocks <= MAX_BLOCKS, PSVAE_ETOOLARGE, "%s: %d x %d rows of %d are more than one launch holds", fn, s->B, s->T,
                  s->V);
    PSVAE_REQUIRE(s->repetition > 0.f && s->repetition < __builtin_inff() && s->temperature > 0.f && s->temperature < __builtin_inff(),
                  PSVAE_EINVAL, "%s: repetition and temperature must be positive and finite", fn);
    PSVAE_REQUIRE(s->presence - s->presence == 0.f && s->frequency - s->frequency == 0.f, PSVAE_EINVAL,
                  "%s: presence and frequency must be finite", fn);
    if (s->B == 0) return PSVAE_OK;
    PSVAE_REQUIRE(s->logits != nullptr, PSVAE_EINVAL, "%s: null logits", fn);
    PSVAE_REQUIRE(((uintptr_t)s->logits & (elem_size(s->dtype) - 1)) == 0, PSVAE_EINVAL, "%s: misaligned logits", fn);
    PSVAE_REQUIRE(s->L >= 0 && s->L <= (1 << 24), PSVAE_EINVAL, "%s: history of %d ids (at most 2^24: counts stay exact in 32 bits)", fn, s->L);
    PSVAE_REQUIRE(s->history != nullptr || (s->L == 0 && s->history_len == nullptr), PSVAE_EINVAL, "%s: history is null", fn);
    PSVAE_REQUIRE(s->allowed == nullptr ? s->state == nullptr : s->S >= 1, PSVAE_EINVAL, "%s: states without a mask table", fn);
    PSVAE_REQUIRE(s->allowed == nullptr || s->ld_allowed >= (s->V + 31) / 32 || s->S == 1, PSVAE_EINVAL, "%s: mask rows are shorter than V bits", fn);
    PSVAE_REQUIRE(s->allowed == nullptr || s->state != nullptr || s->S == 1 || s->S == s->B, PSVAE_EINVAL,
                  "%s: without states the mask table has one row, or one per sequence", fn);
    a->R = s->B * s->T, a->T = s->T, a->V = s->V, a->L = s->L, a->S = s->S;
    a->logits = s->logits, a->ld_b = s->ld_b, a->ld_t = s->ld_t;
    a->history = s->L > 0 ? s->history : nullptr, a->ld_history = s->ld_history;
    a->history_len = s->history_len, a->len_per_row = s->len_per_row;
    a->rep_p = s->repetition_rows, a->pres_p = s->presence_rows, a->freq_p = s->frequency_rows, a->temp_p = s->temperature_rows;
    a->rep = s->repetition, a->pres = s->presence, a->freq = s->frequency, a->temp = s->temperature;
    a->bias = s->bias, a->ld_bias = s->ld_bias;
    a->allowed = s->allowed, a->ld_allowed = s->ld_allowed, a->state = s->state, a->state_per_row = s->state_per_row;
    a->units = cut_of(s).units;
    return PSVAE_OK;
}

// Launches KERNEL<T, K, ROWS, HIST> for the call's type, cut and history.
#define PSVAE_LAUNCH_K(KERNEL, T, K, ROWS, ...)                                                                                     \
    do {                                                                                                                            \
        if (args.history) hipLaunchKernelGGL((KERNEL<T, K, ROWS, true>), dim3((unsigned)cut.blocks), dim3(NT), 0, st, __VA_ARGS__); \
        else hipLaunchKernelGGL((KERNEL<T, K, ROWS, false>), dim3((unsigned)cut.blocks), dim3(NT), 0, st, __VA_ARGS__);             \
    } while (0)
#define PSVAE_LAUNCH_T(KERNEL, T, ...)                                                               \
    do {                                                                                             \
        constexpr int PER = Elem<T>::VEC;                                                            \
        if (cut.wave_rows && cut.per_thread == 8) PSVAE_LAUNCH_K(KERNEL, T, 8 / PER, WAVES, __VA_ARGS__);   \
        else if (cut.wave_rows) PSVAE_LAUNCH_K(KERNEL, T, 16 / PER, WAVES, __VA_ARGS__);             \
        else if (cut.per_thread == 8) PSVAE_LAUNCH_K(KERNEL, T, 8 / PER, 1, __VA_ARGS__);            \
        else PSVAE_LAUNCH_K(KERNEL, T, 32 / PER, 1, __VA_ARGS__);                                    \
    } while (0)

template <typename T, int K> void launch_draw_wide(const Args &args, const Cut &cut, Piece *part, const float *u, long long ld_u,
                                                   int64_t empty, int64_t *out, float *lp, hipStream_t st) {
    if (args.history) {
        hipLaunchKernelGGL((draw_piece_kernel<T, K, true>), dim3((unsigned)cut.blocks), dim3(NT), 0, st, args, part);
        hipLaunchKernelGGL((draw_join_kernel<T, K, true>), dim3((unsigned)args.R), dim3(NT), 0, st, args, part, u, ld_u, empty, out, lp);
    } else {
        hipLaunchKernelGGL((draw_piece_kernel<T, K, false>), dim3((unsigned)cut.blocks), dim3(NT), 0, st, args, part);
        hipLaunchKernelGGL((draw_join_kernel<T, K, false>), dim3((unsigned)args.R), dim3(NT), 0, st, args, part, u, ld_u, empty, out, lp);
    }
}

template <typename T> void launch_draw(const Args &args, const Cut &cut, Piece *part, const float *u, long long ld_u, int64_t empty,
                                       int64_t *out, float *lp, hipStream_t st) {
    constexpr int PER = Elem<T>::VEC;
    if (cut.wave_rows) {
        if (cut.per_thread == 8) PSVAE_LAUNCH_K(draw_row_kernel, T, 8 / PER, WAVES, args, u, ld_u, empty, out, lp);
        else PSVAE_LAUNCH_K(draw_row_kernel, T, 16 / PER, WAVES, args, u, ld_u, empty, out, lp);
    } else if (cut.per_thread == 8) {
        launch_draw_wide<T, 8 / PER>(args, cut, part, u, ld_u, empty, out, lp, st);
    } else {
        launch_draw_wide<T, 32 / PER>(args, cut, part, u, ld_u, empty, out, lp, st);
    }
}

size_t pieces_of(const psvae_shaping *s) {
    if (s == nullptr || s->B <= 0 || s->T < 1 || s->V < 1) return 0;
    const Cut c = cut_of(s);
    return c.wave_rows ? 0 : (size_t)s->B * s->T * c.units * WAVES;
}

}  // namespace

#define PSVAE_BY_TYPE(CALL)                       \
    do {                                          \
        if (shaping->dtype == PSVAE_F32) CALL(float); \
        else if (shaping->dtype == PSVAE_BF16) CALL(__bf16); \
        else CALL(_Float16);                      \
    } while (0)

extern "C" int psvae_shape_logits_fwd(const psvae_shaping *shaping, void *out, int64_t ld_out, void *stream) {
    const char *fn = "psvae_shape_logits_fwd";
    Args args;
    if (int rc = check_shaping(fn, shaping, &args)) return rc;
    if (shaping->B == 0) return PSVAE_OK;
    PSVAE_REQUIRE(out != nullptr && ld_out >= shaping->V, PSVAE_EINVAL, "%s: null output or rows shorter than V", fn);
    PSVAE_REQUIRE(((uintptr_t)out & (elem_size(shaping->dtype) - 1)) == 0, PSVAE_EINVAL, "%s: misaligned output", fn);
    const Cut cut = cut_of(shaping);
    hipStream_t st = (hipStream_t)stream;
#define CALL(T) PSVAE_LAUNCH_T(shape_fwd_kernel, T, args, (T *)out, (long long)ld_out)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" int psvae_shape_logits_bwd(const psvae_shaping *shaping, const void *g, int64_t ld_gb, int64_t ld_gt, void *dlogits,
                                      int64_t ld_dlogits, void *stream) {
    const char *fn = "psvae_shape_logits_bwd";
    Args args;
    if (int rc = check_shaping(fn, shaping, &args)) return rc;
    if (shaping->B == 0) return PSVAE_OK;
    PSVAE_REQUIRE(g != nullptr && dlogits != nullptr && ld_dlogits >= shaping->V, PSVAE_EINVAL, "%s: null gradient or rows shorter than V", fn);
    PSVAE_REQUIRE((((uintptr_t)g | (uintptr_t)dlogits) & (elem_size(shaping->dtype) - 1)) == 0, PSVAE_EINVAL, "%s: misaligned gradient", fn);
    const Cut cut = cut_of(shaping);
    hipStream_t st = (hipStream_t)stream;
#define CALL(T) PSVAE_LAUNCH_T(shape_bwd_kernel, T, args, (const T *)g, (long long)ld_gb, (long long)ld_gt, (T *)dlogits, (long long)ld_dlogits)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" size_t psvae_shaped_log_prob_workspace_bytes(const psvae_shaping *shaping) {
    const size_t pieces = pieces_of(shaping);
    return pieces ? pieces * sizeof(float2) + (size_t)shaping->B * shaping->T * sizeof(float) : 0;
}

extern "C" int psvae_shaped_log_prob_fwd(const psvae_shaping *shaping, const int64_t *tokens, float *log_prob, float *stats,
                                         void *workspace, size_t workspace_bytes, void *stream) {
    const char *fn = "psvae_shaped_log_prob_fwd";
    Args args;
    if (int rc = check_shaping(fn, shaping, &args)) return rc;
    if (shaping->B == 0) return PSVAE_OK;
    PSVAE_REQUIRE(tokens != nullptr && log_prob != nullptr && stats != nullptr, PSVAE_EINVAL, "%s: null pointer", fn);
    PSVAE_REQUIRE(((uintptr_t)stats & 7u) == 0, PSVAE_EINVAL, "%s: stats must be 8-byte aligned", fn);
    const size_t need = psvae_shaped_log_prob_workspace_bytes(shaping);
    PSVAE_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && ((uintptr_t)workspace & 7u) == 0), PSVAE_EWORKSPACE,
                  "%s: workspace too small or not 8-byte aligned", fn);
    const Cut cut = cut_of(shaping);
    hipStream_t st = (hipStream_t)stream;
    float2 *part = (float2 *)workspace, *stat2 = (float2 *)stats;
    float *target = need ? (float *)(part + pieces_of(shaping)) : nullptr;
#define CALL(T) PSVAE_LAUNCH_T(log_prob_fwd_kernel, T, args, tokens, log_prob, stat2, part, target)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    if (!cut.wave_rows) {
        hipLaunchKernelGGL(log_prob_join_kernel, dim3(psvae_cdiv(args.R, WAVES)), dim3(NT), 0, st, args.R, args.V, args.units * WAVES,
                           tokens, part, target, log_prob, stat2);
        PSVAE_CHECK_LAUNCH(fn);
    }
    return PSVAE_OK;
}

extern "C" int psvae_shaped_log_prob_bwd(const psvae_shaping *shaping, const int64_t *tokens, const float *stats, const float *g,
                                         void *dlogits, int64_t ld_dlogits, void *stream) {
    const char *fn = "psvae_shaped_log_prob_bwd";
    Args args;
    if (int rc = check_shaping(fn, shaping, &args)) return rc;
    if (shaping->B == 0) return PSVAE_OK;
    PSVAE_REQUIRE(tokens && stats && g && dlogits && ld_dlogits >= shaping->V, PSVAE_EINVAL, "%s: null pointer or rows shorter than V", fn);
    PSVAE_REQUIRE(((uintptr_t)dlogits & (elem_size(shaping->dtype) - 1)) == 0 && ((uintptr_t)stats & 7u) == 0, PSVAE_EINVAL,
                  "%s: misaligned gradient or stats", fn);
    const Cut cut = cut_of(shaping);
    hipStream_t st = (hipStream_t)stream;
#define CALL(T) PSVAE_LAUNCH_T(log_prob_bwd_kernel, T, args, tokens, (const float2 *)stats, g, (T *)dlogits, (long long)ld_dlogits)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" size_t psvae_shaped_draw_workspace_bytes(const psvae_shaping *shaping) { return pieces_of(shaping) * sizeof(Piece); }

extern "C" int psvae_shaped_draw(const psvae_shaping *shaping, const float *uniforms, int64_t ld_uniforms, int64_t empty_token,
                                 int64_t *tokens, float *log_prob, void *workspace, size_t workspace_bytes, void *stream) {
    const char *fn = "psvae_shaped_draw";
    Args args;
    if (int rc = check_shaping(fn, shaping, &args)) return rc;
    PSVAE_REQUIRE(shaping->T == 1, PSVAE_EINVAL, "%s: one token per sequence is drawn (T = %d)", fn, shaping->T);
    if (shaping->B == 0) return PSVAE_OK;
    PSVAE_REQUIRE(uniforms != nullptr && tokens != nullptr && log_prob != nullptr, PSVAE_EINVAL, "%s: null pointer", fn);
    const size_t need = psvae_shaped_draw_workspace_bytes(shaping);
    PSVAE_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && psvae_aligned16(workspace)), PSVAE_EWORKSPACE,
                  "%s: workspace too small or not 16-byte aligned", fn);
    const Cut cut = cut_of(shaping);
    PSVAE_REQUIRE(args.R <= MAX_BLOCKS, PSVAE_ETOOLARGE, "%s: %d rows", fn, args.R);
    hipStream_t st = (hipStream_t)stream;
#define CALL(T) launch_draw<T>(args, cut, (Piece *)workspace, uniforms, (long long)ld_uniforms, empty_token, tokens, log_prob, st)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}
