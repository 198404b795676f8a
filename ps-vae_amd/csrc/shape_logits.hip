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

#include <math.h>

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

// Counts of the ids [base, base + n) in the row's history, into cnt[0 .. n).  Every thread of the workgroup calls it (barriers);
// the calling group's threads number `tid` of `threads`.
__device__ __forceinline__ void count_unit(int *cnt, int span, const int64_t *hist, int len, int base, int n, int tid, int threads) {
    for (int i = tid * 4; i < span; i += threads * 4) *reinterpret_cast<int4 *>(cnt + i) = make_int4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll 4
    for (int j = tid; j < len; j += threads) {
        const unsigned long long at = (unsigned long long)(hist[j] - base);   // ids outside the vocabulary fall outside every unit
        if (at < (unsigned long long)n) atomicAdd(&cnt[at], 1);
    }
    __syncthreads();
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

// The shaped value in type C (float, double) and, for the gradient, its slope.
template <typename C> struct Rule {
    C rep, pres, freq, inv_temp;
    template <typename T> __device__ Rule(const Row<T> &w)
        : rep((C)w.rep), pres((C)w.pres), freq((C)w.freq), inv_temp((C)1 / (C)w.temp) {}
    __device__ __forceinline__ C value(C x, int c, C bias) const {
        if (c > 0) x = (x > (C)0 ? x / rep : x * rep) - freq * (C)c - pres;
        return (x + bias) * inv_temp;
    }
    __device__ __forceinline__ C slope(C x, int c) const { return c > 0 ? (x > (C)0 ? inv_temp / rep : inv_temp * rep) : inv_temp; }
};

// VEC bits of the mask for the elements i .. i + VEC - 1 (i a multiple of VEC)
template <int VEC> __device__ __forceinline__ uint32_t mask_bits(const uint32_t *mask, int i) {
    return mask ? (mask[i >> 5] >> (i & 31)) : 0xffffffffu;
}
template <int VEC> __device__ __forceinline__ void load_bias(const float *bias, int left, float (&b)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) b[j] = 0.f;
    if (!bias) return;
    if (left >= VEC) {
#pragma unroll
        for (int q = 0; q < VEC / 4; ++q) {
            const Float4u f = *reinterpret_cast<const Float4u *>(bias + 4 * q);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[4 * q + j] = f.v[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < left) b[j] = bias[j];
    }
}

// Where a thread stands: which row, which unit, which elements.
template <typename T, int K, int ROWS> struct Place {
    static constexpr int VEC = Elem<T>::VEC, THREADS = NT / ROWS, SPAN = THREADS * VEC * K;
    int r, unit, tid, lane, wave;    // row; unit of the row; thread, lane and wave inside the row's group
    bool live;
    __device__ Place(const Args &a, int block) {
        tid = threadIdx.x & (THREADS - 1), lane = threadIdx.x & 63, wave = tid >> 6;
        if (ROWS == 1) {
            r = a.units == 1 ? block : (int)((unsigned)block / (unsigned)a.units), unit = block - r * a.units;
        } else {
            r = block * ROWS + (int)threadIdx.x / THREADS, unit = 0;
        }
        live = r < a.R;
        if (!live) r = a.R - 1;
    }
    __device__ __forceinline__ int base() const { return unit * SPAN; }
    __device__ __forceinline__ int at(int k) const { return ((wave * K + k) * 64 + lane) * VEC; }   // inside the unit
};

// Loads a thread's logits, counts the unit, and hands out (element, left, count, bits, bias) per VEC.
template <typename T, int K, int ROWS, bool HIST> struct Unit {
    using P = Place<T, K, ROWS>;
    static constexpr int VEC = P::VEC;
    P p;
    Row<T> w;
    Pack<T> x[K];
    int *cnt;
    int V;
    __device__ Unit(const Args &a, int block, int *lds, bool want_logits) : p(a, block), w(row_of<T>(a, p.r)), V(a.V) {
        const int base = p.base();
        if (want_logits) {
#pragma unroll
            for (int k = 0; k < K; ++k) x[k] = load_pack(w.x + base + p.at(k), p.live ? V - base - p.at(k) : 0);
        }
        cnt = HIST ? lds + (ROWS == 1 ? 0 : (int)threadIdx.x / P::THREADS * P::SPAN) : nullptr;
        if (HIST) {
            const int n = V - base < P::SPAN ? V - base : P::SPAN;
            count_unit(cnt, P::SPAN, w.hist, p.live ? w.len : 0, base, n, p.tid, P::THREADS);
        }
    }
    __device__ __forceinline__ int left(int k) const { return p.live ? V - p.base() - p.at(k) : 0; }
    __device__ __forceinline__ uint32_t bits(int k) const {
        return w.none || left(k) <= 0 ? 0u : mask_bits<VEC>(w.mask, p.base() + p.at(k));
    }
    __device__ __forceinline__ int count(int k, int j) const { return HIST ? cnt[p.at(k) + j] : 0; }
};

template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void shape_fwd_kernel(Args a, T *__restrict__ out, long long ld_out) {
    using U = Unit<T, K, ROWS, HIST>;
    __shared__ __align__(16) int lds[HIST ? U::P::SPAN * ROWS : 4];
    U u(a, blockIdx.x, lds, true);
    if (!u.p.live) return;
    const Rule<float> rule(u.w);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int left = u.left(k);
        if (left <= 0) continue;
        const int i = u.p.base() + u.p.at(k);
        const uint32_t bits = u.bits(k);
        float b[U::VEC];
        load_bias<U::VEC>(u.w.bias ? u.w.bias + i : nullptr, left, b);
        Pack<T> y;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) {
            const float v = rule.value((float)u.x[k].v[j], u.count(k, j), b[j]);
            y.v[j] = (T)((bits >> j) & 1u ? v : NEG);
        }
        store_pack(out + u.p.r * ld_out + i, y, left);
    }
}

// dl = g * slope; the logits are read only where a past token's sign decides the slope (x != null).
template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void shape_bwd_kernel(Args a, const T *__restrict__ g, long long ld_gb, long long ld_gt,
                                                       T *__restrict__ dx, long long ld_dx) {
    using U = Unit<T, K, ROWS, HIST>;
    __shared__ __align__(16) int lds[HIST ? U::P::SPAN * ROWS : 4];
    U u(a, blockIdx.x, lds, false);
    if (!u.p.live) return;
    const Rule<float> rule(u.w);
    const int b = a.T == 1 ? u.p.r : (int)((unsigned)u.p.r / (unsigned)a.T), t = u.p.r - b * a.T;
    const T *gr = g + b * ld_gb + t * ld_gt;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int left = u.left(k);
        if (left <= 0) continue;
        const int i = u.p.base() + u.p.at(k);
        const uint32_t bits = u.bits(k);
        const Pack<T> gv = load_pack(gr + i, left);
        Pack<T> d;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) {
            const int c = u.count(k, j);
            float x = 0.f;
            if (c > 0) x = (float)u.w.x[i + j];
            d.v[j] = (T)((bits >> j) & 1u ? (float)gv.v[j] * rule.slope(x, c) : 0.f);
        }
        store_pack(dx + u.p.r * ld_dx + i, d, left);
    }
}

__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
template <typename C> __device__ __forceinline__ C wave_max(C v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = larger(v, __shfl_xor(v, d));
    return v;
}
template <typename C> __device__ __forceinline__ C wave_sum(C v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
template <typename C> __device__ __forceinline__ C wave_scan(C v, int lane) {   // inclusive, in lane order
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const C up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    return v;
}

__device__ __forceinline__ float log_prob_of(float y_tok, float m, float s) {
    return m == NEG && s == 0.f ? NEG : y_tok - m - logf(s);   // (nothing allowed: log 0)
}

// Per wave: the maximum and the sum of exponentials of its piece; per row: the shaped value of its token.  ROWS > 1: the wave has the
// whole row and finishes it.  Sums are 32-bit: 64 lanes of at most VEC * K terms each, then 6 levels, so the relative error stays below
// (VEC * K + 6 + pieces) * 2^-24.
template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void log_prob_fwd_kernel(Args a, const int64_t *__restrict__ tokens, float *__restrict__ lp,
                                                          float2 *__restrict__ stats, float2 *__restrict__ part,
                                                          float *__restrict__ target) {
    using U = Unit<T, K, ROWS, HIST>;
    __shared__ __align__(16) int lds[HIST ? U::P::SPAN * ROWS : 4];
    U u(a, blockIdx.x, lds, true);
    if (!u.p.live) return;
    const Rule<float> rule(u.w);
    const long long tok = tokens[u.p.r];
    float y[K][U::VEC];
    float m = NEG, yt = 0.f;
    bool mine = false;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int left = u.left(k), i = u.p.base() + u.p.at(k);
        const uint32_t bits = u.bits(k);
        float b[U::VEC];
        load_bias<U::VEC>(u.w.bias ? u.w.bias + i : nullptr, left, b);
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) {
            y[k][j] = j < left && ((bits >> j) & 1u) ? rule.value((float)u.x[k].v[j], u.count(k, j), b[j]) : NEG;
            m = fmaxf(m, y[k][j]);
            if (j < left && i + j == tok) yt = y[k][j], mine = true;
        }
    }
    m = wave_max(m);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) s += y[k][j] == NEG ? 0.f : __expf(y[k][j] - m);
    s = wave_sum(s);
    if (ROWS == 1) {
        if (mine) target[u.p.r] = yt;
        if (u.p.lane == 0) part[(long long)u.p.r * a.units * WAVES + u.p.unit * WAVES + u.p.wave] = make_float2(m, s);
        return;
    }
    const unsigned long long owner = __ballot(mine);
    const float v = owner ? log_prob_of(__shfl(yt, __ffsll((long long)owner) - 1), m, s) : 0.f;
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
    using U = Unit<T, K, ROWS, HIST>;
    __shared__ __align__(16) int lds[HIST ? U::P::SPAN * ROWS : 4];
    U u(a, blockIdx.x, lds, true);
    if (!u.p.live) return;
    const Rule<float> rule(u.w);
    const long long tok = tokens[u.p.r];
    const float2 st = stats[u.p.r];
    const bool zero = tok < 0 || tok >= a.V || (st.x == NEG && st.y == 0.f);   // a row without a token, or with none allowed
    const float gr = g[u.p.r], inv = 1.f / st.y;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int left = u.left(k);
        if (left <= 0) continue;
        const int i = u.p.base() + u.p.at(k);
        const uint32_t bits = zero ? 0u : u.bits(k);
        float b[U::VEC];
        load_bias<U::VEC>(u.w.bias ? u.w.bias + i : nullptr, left, b);
        Pack<T> d;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) {
            const int c = u.count(k, j);
            const float x = (float)u.x[k].v[j];
            const float p = __expf(rule.value(x, c, b[j]) - st.x) * inv;
            d.v[j] = (T)((bits >> j) & 1u ? gr * ((i + j == tok ? 1.f : 0.f) - p) * rule.slope(x, c) : 0.f);
        }
        store_pack(dx + u.p.r * ld_dx + i, d, left);
    }
}

// ---- draw.  The pick is a decision: with a running sum in 32 bits, u * total falls on the wrong side of some boundary about once in
// 1e3 .. 1e4 rows at V = 1e5 (V boundaries, each off by ~1e-8), and differently for every tiling.  So values, exponentials and sums are
// 64-bit here: the pick is the one of the exact distribution but for ~1e-11 of the rows, whatever the tiling.
struct Piece {
    double s, m;
};
constexpr double NEG64 = -__builtin_inf();

// e[k][j] = exp(y - m) of the thread's elements (0 where not allowed); returns m, the wave's largest y.
template <typename T, int K, int ROWS, bool HIST, int VEC>
__device__ __forceinline__ double exp_values(const Unit<T, K, ROWS, HIST> &u, double (&e)[K][VEC]) {
    const Rule<double> rule(u.w);
    double m = NEG64;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int left = u.left(k), i = u.p.base() + u.p.at(k);
        const uint32_t bits = u.bits(k);
        float b[VEC];
        load_bias<VEC>(u.w.bias ? u.w.bias + i : nullptr, left, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            e[k][j] = j < left && ((bits >> j) & 1u) ? rule.value((double)(float)u.x[k].v[j], u.count(k, j), (double)b[j]) : NEG64;
            m = fmax(m, e[k][j]);
        }
    }
    m = wave_max(m);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[k][j] = e[k][j] == NEG64 ? 0. : exp(e[k][j] - m);
    return m;
}

// The first element, in index order, at which the running sum (starting from `before`) exceeds thr; the last positive one if it never
// does.  Returns its index inside the wave's piece (or -1: nothing positive) and its e.  The whole wave calls it.
template <int K, int VEC> __device__ __forceinline__ int pick_in_wave(const double (&e)[K][VEC], int lane, double before, double thr, double *value) {
    int found = -1, last = -1;
    double cum = before, v_found = 0., v_last = 0.;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        double s = 0.;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += e[k][j];
        const double inc = wave_scan(s, lane);
        // inside the lane: the first positive element past thr, else the last positive one
        int mine = -1;
        double run = cum + (inc - s), mine_v = 0.;
        bool over = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (e[k][j] > 0. && !over) run += e[k][j], mine = j, mine_v = e[k][j], over = run > thr;
        const unsigned long long some = __ballot(s > 0.), hit = __ballot(s > 0. && cum + inc > thr);
        if (found < 0 && hit) {
            const int l = __ffsll((long long)hit) - 1;
            found = (k * 64 + l) * VEC + __shfl(mine, l), v_found = __shfl(mine_v, l);
        }
        if (some) {
            const int l = 63 - __clzll((long long)some);
            last = (k * 64 + l) * VEC + __shfl(mine, l), v_last = __shfl(mine_v, l);
        }
        cum += __shfl(inc, 63);
    }
    *value = found >= 0 ? v_found : v_last;
    return found >= 0 ? found : last;
}

// a whole row in a wave
template <typename T, int K, int ROWS, bool HIST>
__global__ __launch_bounds__(NT) void draw_row_kernel(Args a, const float *__restrict__ uniforms, long long ld_u, int64_t empty,
                                                      int64_t *__restrict__ out, float *__restrict__ lp) {
    using U = Unit<T, K, ROWS, HIST>;
    __shared__ __align__(16) int lds[HIST ? U::P::SPAN * ROWS : 4];
    U u(a, blockIdx.x, lds, true);
    if (!u.p.live) return;
    double e[K][U::VEC];
    const double m = exp_values(u, e);
    double s = 0.;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        double t = 0.;
#pragma unroll
        for (int j = 0; j < U::VEC; ++j) t += e[k][j];
        s += wave_sum(t);
    }
    double v;
    const int pick = pick_in_wave(e, u.p.lane, 0., (double)uniforms[u.p.r * ld_u] * s, &v);
    if (u.p.lane == 0) {
        const bool ok = s > 0. && m < __builtin_inf() && pick >= 0;
        out[u.p.r] = ok ? pick : empty;
        lp[u.p.r] = ok ? (float)log(v / s) : (m == NEG64 && s == 0. ? NEG : __builtin_nanf(""));
    }
}

template <typename T, int K, bool HIST>
__global__ __launch_bounds__(NT) void draw_piece_kernel(Args a, Piece *__restrict__ part) {
    using U = Unit<T, K, 1, HIST>;
    __shared__ __align__(16) int lds[HIST ? U::P::SPAN : 4];
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

// One workgroup per row: the pieces joined in index order, the piece that holds u * total found, and its elements walked again (the
// workgroup counts the piece's ids, its first wave walks).
template <typename T, int K, bool HIST>
__global__ __launch_bounds__(NT) void draw_join_kernel(Args a, const Piece *__restrict__ part, const float *__restrict__ uniforms,
                                                       long long ld_u, int64_t empty, int64_t *__restrict__ out,
                                                       float *__restrict__ lp) {
    constexpr int VEC = Elem<T>::VEC, SPAN = 64 * VEC * K;   // a piece: what one wave of draw_piece_kernel had
    __shared__ __align__(16) int cnt[HIST ? SPAN : 4];
    const int r = blockIdx.x, lane = threadIdx.x & 63, pieces = a.units * WAVES;
    const Piece *p = part + (long long)r * pieces;
    double m = NEG64;
    for (int i = lane; i < pieces; i += 64) m = fmax(m, p[i].m);
    m = wave_max(m);
    double total = 0.;
    for (int base = 0; base < pieces; base += 64) {
        const int i = base + lane;
        const double w = i < pieces ? (p[i].m == NEG64 ? p[i].s : p[i].s * exp(p[i].m - m)) : 0.;
        total += wave_sum(w);
    }
    // every wave of the workgroup has the same total and comes to the same piece
    const double thr = (double)uniforms[r * ld_u] * total;
    int found = -1, last = -1;
    double cum = 0., before = 0., before_last = 0.;
    for (int base = 0; base < pieces; base += 64) {
        const int i = base + lane;
        const double w = i < pieces ? (p[i].m == NEG64 ? p[i].s : p[i].s * exp(p[i].m - m)) : 0.;
        const double inc = wave_scan(w, lane);
        const unsigned long long some = __ballot(w > 0.), hit = __ballot(w > 0. && cum + inc > thr);
        const double ahead = cum + (inc - w);
        if (found < 0 && hit) {
            const int l = __ffsll((long long)hit) - 1;
            found = base + l, before = __shfl(ahead, l);
        }
        if (some) {
            const int l = 63 - __clzll((long long)some);
            last = base + l, before_last = __shfl(ahead, l);
        }
        cum += __shfl(inc, 63);
    }
    if (found < 0) found = last, before = before_last;
    if (!(total > 0.) || !(m < __builtin_inf()) || found < 0) {
        if (threadIdx.x == 0) out[r] = empty, lp[r] = m == NEG64 && total == 0. ? NEG : __builtin_nanf("");
        return;   // (the whole workgroup: every thread has the same total, m and found)
    }
    const Row<T> w = row_of<T>(a, r);
    const int base = found * SPAN, n = a.V - base < SPAN ? a.V - base : SPAN;
    if (HIST) count_unit(cnt, SPAN, w.hist, w.len, base, n, threadIdx.x, NT);
    if (threadIdx.x >= 64) return;
    const Rule<double> rule(w);
    double e[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int at = (k * 64 + lane) * VEC, left = n - at, i = base + at;
        const Pack<T> x = load_pack(w.x + i, left);
        const uint32_t bits = left > 0 ? mask_bits<VEC>(w.mask, i) : 0u;
        float b[VEC];
        load_bias<VEC>(w.bias ? w.bias + i : nullptr, left, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            e[k][j] = j < left && ((bits >> j) & 1u)
                          ? exp(rule.value((double)(float)x.v[j], HIST ? cnt[at + j] : 0, (double)b[j]) - m) : 0.;
    }
    double v;
    const int pick = pick_in_wave(e, lane, before, thr, &v);
    if (lane == 0) {
        out[r] = pick >= 0 ? base + pick : empty;
        lp[r] = pick >= 0 ? (float)log(v / total) : __builtin_nanf("");
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
