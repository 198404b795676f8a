// Between the vocabulary layer's logits and the next token: penalties for tokens of the past, a bias, a temperature and a
// grammar's mask (shape), the log-probability of a given token under the result and its gradient (log_prob), and one
// token drawn from it (draw).  For row r = (b, t), with c_i the number of times id i occurs in the first len_r ids of history[b]:
//     a_i = l_i;  c_i > 0:  a_i = (l_i > 0 ? l_i / rep_b : l_i * rep_b) - freq_b c_i - pres_b
//     y_i = (a_i + bias_i) / T_b   where bit i of allowed[state_r] is set (state < 0: every bit; state >= S: no bit), else -inf
//     log_prob = y_tok - m - log s,  m = max y, s = sum exp(y - m);  d log_prob / d l_i = ([i = tok] - exp(y_i - m) / s) dy_i/dl_i
//     draw:  min(#{i : cdf_i <= u cdf_last}, last i of positive probability),  cdf the running sum of exp(y - m) in index order
//
// Bound: one read of the logits (and one write) at large sizes, launches at small ones, with 8 to 14 vector instructions an element in
// between that have to stay under the time of the loads (shape of wide rows: the vector unit 21 % busy; log_prob both ways: 80 %, so
// this bounds it as much as the loads); the draw, whose 25 of 38 are 64-bit, is bound by them (77 %).
//
// Rows of at most 1024 logits: one wave each (Narrow).  Wider rows are cut into runs of up to 32768 elements, a workgroup each, whose
// waves stream through it in steps of 512 or 1024 elements (`stream`).
//
// The penalties need c_i.  No table of counts of [rows, V] is kept or read - it would be as large as the logits.  The
// workgroup walks the row's history itself (8 bytes an entry) and builds in LDS what its elements need: one bit per element says whether the id was
// seen, and the finished values y of the seen ids - computed once by one thread each - lie in a list in the order of the bits.  The
// stream over the elements leaves the seen ones out of its sums, the list's values being added beside it; or takes them as if nothing had been
// seen, the list's values replacing these on their way out (Stage).  So an element that was not seen, which nearly all are not, pays nothing for the question (looked up
// element by element the seen ones cost 8 of 24 instructions).  Counts are sums of integers and every value is computed from them
// alone: the order of the LDS atomics does not show.
#include "common.h"

#include <algorithm>
#include <limits.h>
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
    int run, runs;                   // wide rows: elements of a run, runs of a row
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
    __device__ __forceinline__ bool allows(int i) const { return !none && (!mask || ((mask[i >> 5] >> (i & 31)) & 1u)); }
};

// Repetition and temperature: numbers whose 32-bit reciprocal is a normal number too (beyond, the unit's estimate of it is infinite, or 0).
constexpr float RULE_MIN = 0x1p-126f, RULE_MAX = 0x1p126f;
__device__ __forceinline__ float in_range(float v) { return v >= RULE_MIN && v <= RULE_MAX ? v : __builtin_nanf(""); }
bool is_in_range(float v) { return v >= RULE_MIN && v <= RULE_MAX; }

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
    // a repetition or temperature out of range makes what it touches NaN
    w.rep = in_range(a.rep_p ? a.rep_p[b] : a.rep);
    w.pres = a.pres_p ? a.pres_p[b] : a.pres;
    w.freq = a.freq_p ? a.freq_p[b] : a.freq;
    w.temp = in_range(a.temp_p ? a.temp_p[b] : a.temp);
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
// (Non-temporal: what is written here is read by a later kernel, far more of it than the caches hold.)
typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> __device__ __forceinline__ void store_pack(T *p, const Pack<T> &v, int left) {
    if (left >= Elem<T>::VEC) {
        __builtin_nontemporal_store(__builtin_bit_cast(Words, v), reinterpret_cast<Words *>(p));
    } else {
#pragma unroll
        for (int j = 0; j < Elem<T>::VEC; ++j)
            if (j < left) p[j] = v.v[j];
    }
}

// f(id - base) for every id of a row's history that lies in [base, base + n): the threads `tid` of `threads` take it in turn, BATCH ids
// of each requested at once (one by one, each behind the last one's test, a walk of 4000 ids took 16 memory latencies).  Ids outside
// the vocabulary fall outside every range.
template <int BATCH, typename F> __device__ __forceinline__ void walk(const int64_t *hist, int len, int base, int n, int tid, int threads, F f) {
    for (int first = 0; first < len; first += BATCH * threads) {
        int64_t id[BATCH];
#pragma unroll
        for (int q = 0; q < BATCH; ++q) {
            const int j = first + q * threads + tid;
            if (first + q * threads < len) id[q] = hist[j < len ? j : len - 1];
        }
#pragma unroll
        for (int q = 0; q < BATCH; ++q) {
            if (first + q * threads >= len) break;
            const unsigned long long at = (unsigned long long)id[q] - (unsigned long long)base;
            if (first + q * threads + tid < len && at < (unsigned long long)n) f((int)at);
        }
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

// a row's token as an element of it, or one that no element is
__device__ __forceinline__ int token_of(long long tok, int V) { return tok >= 0 && tok < V ? (int)tok : INT_MIN / 2; }

// exp(y - m) as a power of two.  (The difference first: a row of the type's lowest values - masked by hand - has an m whose multiple of
// log2 e overflows.)  Where nothing is allowed m = -inf: 0 in its place.
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float reference_of(float m) { return m == NEG ? 0.f : m; }
__device__ __forceinline__ float exp_from(float y, float from) { return __builtin_amdgcn_exp2f((y - from) * LOG2E); }
__device__ __forceinline__ float log_prob_of(float y_tok, float m, float s) {
    return m == NEG && s == 0.f ? NEG : y_tok - m - logf(s);   // (nothing allowed: log 0)
}

// ---- 64-bit arithmetic of the draw.  The pick is a decision: with a running sum in 32 bits, u * total falls on the wrong side of some
// boundary about once in 1e3 .. 1e4 rows at V = 1e5 (V boundaries, each off by ~1e-8), and differently for every tiling.  So values,
// exponentials and sums are 64-bit: the pick is the one of the exact distribution but for ~1e-8 of the rows, whatever the tiling.
constexpr double NEG64 = -__builtin_inf(), LOG2E64 = 1.4426950408889634;

// 2^z (0 below 2^-1074): 2^n of the nearest whole number times a polynomial in the rest |r| <= 1/2 - the one of degree 9 that is 1
// at r = 0 and has the smallest largest relative error (Remez exchange: 7.7e-14).
__device__ __forceinline__ double power_of_two(double z) {
    double low = -1080.;
    asm("v_max_f64 %0, %1, %2" : "=v"(z) : "v"(z), "s"(low));   // (fmax would first quieten z in an instruction of its own)
    const double n = rint(z), r = z - n;
    double p = 9.16811938851594e-08;
    p = fma(p, r, 1.3255182784592006e-06);
    p = fma(p, r, 1.5258493063907014e-05);
    p = fma(p, r, 0.0001540345603665657);
    p = fma(p, r, 0.0013333547331461978);
    p = fma(p, r, 0.009618129159172244);
    p = fma(p, r, 0.055504108739712246);
    p = fma(p, r, 0.24022650695813708);
    p = fma(p, r, 0.6931471805585505);
    p = fma(p, r, 1.);
    return ldexp(p, (int)n);
}

// A number in -1080 .. -1080.25 in place of t where the bit is clear: its power of two is 0.  (Only the upper word needs replacing.)
__device__ __forceinline__ double or_nothing(int word, double t) {
    const unsigned long long x = (unsigned long long)__double_as_longlong(t);
    const unsigned hi = ((unsigned)(x >> 32) & (unsigned)word) | (0xc090e000u & ~(unsigned)word);
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | (unsigned)x));
}

// The weights 2^(z - m) of a wave's elements, z = v * scale (scale: log2 e over the temperature), 0 where `allow` has no bit.  fill(k, v) gives
// the v of pack k, take(k, weights) gets its weights, more(f) calls f for further z of this lane.
// Any m will do that leaves the sum in range and comes to the same for equal rows, so m is the `guess` that the caller brings from the wave's
// elements before; if that is no number, the largest of 64 elements, each lane's first - its product with the scale then needs no rounding of
// its own; and the largest of all (exactly: equal z have to give equal weights, however large they are) only where these allow nothing, are not small
// numbers, or turn out to be far from the others.
struct Weights {
    double sum, m;                   // m: NaN if an allowed value is, +inf if one is, -inf if there is none
};
template <int K, int VEC, typename Fill, typename Take, typename More>
__device__ __forceinline__ Weights weigh(const uint32_t (&allow)[K], double scale, double &guess, Fill fill, Take take, More more) {
    double v[VEC];
    fill(0, v);
    if (!(fabs(guess) < 1e6)) guess = (double)wave_max(allow[0] & 1u ? (float)(v[0] * scale) : NEG);
    double m = guess, sum = __builtin_nan("");
    bool bad = false;
    if (fabs(m) < 1e6) {
        sum = 0.;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (k > 0) fill(k, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[j] = or_nothing(bit_word(allow[k], j), fma(v[j], scale, -m));
                bad |= v[j] != v[j];
                v[j] = power_of_two(v[j]);
                sum += v[j];
            }
            take(k, v);
        }
        more([&](double z) { bad |= z != z, sum += power_of_two(z - m); });
        sum = wave_sum(sum);
    }
    if (!(sum < 0x1p500 && sum > 0x1p-500)) {
        double largest = NEG64;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            fill(k, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[j] = select(bit_word(allow[k], j), scaled(v[j], scale), NEG64);
                bad |= v[j] != v[j], largest = fmax(largest, v[j]);
            }
        }
        more([&](double z) { bad |= z != z, largest = fmax(largest, z); });
        m = wave_max(largest);
        const double from = m == NEG64 ? 0. : m;
        sum = 0.;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            fill(k, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = power_of_two(select(bit_word(allow[k], j), scaled(v[j], scale), NEG64) - from), sum += v[j];
            take(k, v);
        }
        more([&](double z) { sum += power_of_two(z - from); });
        sum = wave_sum(sum);
    }
    return {sum, __ballot(bad) ? __builtin_nan("") : m};
}

// The first element, in index order, at which the running sum (starting from `before`) exceeds thr; the last positive one if it never
// does: lane l holds the weights of elements l * N .. l * N + N - 1.  Returns whether it did, the element's index (-1: nothing
// positive) and its weight.  The whole wave calls it.
struct Pick {
    double value;
    int index;
    bool over;
};
template <int N> __device__ __forceinline__ Pick pick_in_wave(const double (&e)[N], double before, double thr) {
    double s = 0.;
#pragma unroll
    for (int j = 0; j < N; ++j) s += e[j];
    const double inc = wave_scan(s);
    const unsigned long long some = __ballot(s > 0.), hit = __ballot(s > 0. && before + inc > thr);
    if (!some) return {0., -1, false};
    // inside each lane: the first positive element past thr, else the last positive one
    int mine = -1;
    double run = before + (inc - s), v = 0.;
    bool over = false;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (e[j] > 0. && !over) run += e[j], mine = j, v = e[j], over = run > thr;
    const int l = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
    return {from_lane(v, l), l * N + __builtin_amdgcn_readlane(mine, l), hit != 0};
}

// log(part / whole) for 0 < part <= whole, the quotient taken apart from the powers of two (it may lie below every double): 2^n f with f in
// [sqrt(1/2), sqrt(2)], log f = 2 artanh(s), s = (f - 1) / (f + 1), |s| < 0.172: the series to s^15 leaves less than 1e-14 of the
// value.  (28 instructions; the library's logarithm and a division are 120, which a narrow row would pay for one number.)
__device__ __forceinline__ float log_of_share(double part, double whole) {
    if (part == whole) return 0.f;
    int n, n_whole;
    double f = frexp(part, &n);
    f *= reciprocal(frexp(whole, &n_whole));
    n -= n_whole;
    if (f < 0.70710678118654752) f *= 2., --n;
    if (f > 1.4142135623730951) f *= 0.5, ++n;
    const double s = (f - 1.) * reciprocal(f + 1.), t = s * s;
    double p = 1. / 15.;
    p = fma(p, t, 1. / 13.);
    p = fma(p, t, 1. / 11.);
    p = fma(p, t, 1. / 9.);
    p = fma(p, t, 1. / 7.);
    p = fma(p, t, 1. / 5.);
    p = fma(p, t, 1. / 3.);
    p = fma(p, t, 1.);
    return (float)fmin(fma((double)n, 0.69314718055994531, 2. * s * p), 0.);
}

// ---- packs: K of them are a thread's share of 64 * VEC * K neighbouring elements, pack k holding elements (k * 64 + lane) * VEC of these.
template <typename T, int K, bool BIAS> struct Packs {
    static constexpr int VEC = Elem<T>::VEC, SPAN = 64 * VEC * K;
    Pack<T> x[K];                    // logits (or what `from` holds)
    float b[BIAS ? K : 1][VEC];
    uint32_t allow[K];               // bit j: element j of the pack is in the row and allowed
    static __device__ __forceinline__ int at(int k) { return (k * 64 + ((int)threadIdx.x & 63)) * VEC; }

    // Elements [base, base + SPAN) of a row, all inside it.  The same loads in every lane and on every path, so that the wait for these packs
    // can leave the next ones in flight: without a mask the word loaded is any word, and is overruled.
    __device__ __forceinline__ void load(const T *from, const Row<T> &w, int base) {
        // (an address in global memory for certain: a load that might be from LDS would be waited for with LDS's own)
        typedef const __attribute__((address_space(1))) uint32_t *Global;
        const Global mask = (Global)(w.mask ? (uintptr_t)w.mask : (uintptr_t)w.x & ~(uintptr_t)3);   // (the 4 bytes that hold the first logit)
        const int which = w.mask ? ~0 : 0;
        const uint32_t all = w.mask ? 0u : 0xffffffffu;
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] = *reinterpret_cast<const Pack<T> *>(from + base + at(k));
        if constexpr (BIAS) {
#pragma unroll
            for (int k = 0; k < K; ++k) load_bias<VEC>(w.bias + base + at(k), VEC, b[k]);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = base + at(k);                      // (whole packs: their bits are in one word)
            allow[k] = ((mask[(i >> 5) & which] >> (i & 31)) | all) & (w.none ? 0u : 0xffffffffu);
        }
    }
    // The same for a row's end: elements of [base, V).
    __device__ __forceinline__ void load_end(const T *from, const Row<T> &w, int base, int V) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = base + at(k), left = V - i;
            x[k] = load_pack(from + i, left);
            if constexpr (BIAS) load_bias<VEC>(w.bias + i, left, b[k]);
            allow[k] = left >= VEC ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
            if (w.mask && left > 0) allow[k] &= w.mask[i >> 5] >> (i & 31);
            if (w.none) allow[k] = 0u;
        }
    }
    // y as if nothing had been seen, before the mask
    __device__ __forceinline__ void raw(int k, const Rule<float> &rule, float (&y)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            y[j] = (float)x[k].v[j];
            if constexpr (BIAS) y[j] += b[k][j];
            y[j] = scaled(y[j], rule.scale);
        }
    }
    // the same before the last factor, in 64 bits
    __device__ __forceinline__ void sums(int k, double (&v)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            v[j] = (double)(float)x[k].v[j];
            if constexpr (BIAS) v[j] += (double)b[k][j];
        }
    }
    __device__ __forceinline__ void masked(int k, float no, float (&y)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = select(bit_word(allow[k], j), y[j], no);
    }
};
template <typename T, int VEC> __device__ __forceinline__ Pack<T> rounded(const float (&v)[VEC]) {
    Pack<T> p;
#pragma unroll
    for (int j = 0; j < VEC; ++j) p.v[j] = (T)v[j];
    return p;
}

// ---- rows of at most ROW_MAX elements: a wave each, a lane holding N neighbouring elements, N = V / 64 rounded up to a form that is
// built.  (One form of 8, its loads aligned, leaves 2 lanes in 5 idle at 300 elements.)  The counts of all ids are a dense array.
constexpr int ROW_MAX = 1024;
template <int SPAN> struct Counts {
    int cell[SPAN];
};
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Few { T v[N]; };

template <typename T, int N> struct Narrow {
    using Lds = Counts<64 * N>;
    int r, lane, i, left;            // i: the lane's first element; left: elements of the row from it on
    bool live;
    Row<T> w;
    Few<T, N> x;                     // logits (or what `from` holds)
    Few<float, N> b;                 // bias, 0 without one
    uint32_t allow;                  // bit j: element i + j is in the row and allowed
    const int *cell;                 // counts of the lane's elements; null: no history
    __device__ Narrow(const Args &a, Lds *all, const T *from, long long ld_b, long long ld_t) {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        lane = threadIdx.x & 63, r = blockIdx.x * WAVES + wave, live = r < a.R, i = lane * N, left = a.V - i;
        if (!live) r = a.R - 1;      // (such a wave only keeps the barriers company)
        w = row_of<T>(a, r);
        const int seq = a.T == 1 ? r : (int)((unsigned)r / (unsigned)a.T), t = r - seq * a.T;
        from += seq * ld_b + t * ld_t;
        allow = w.none || left <= 0 ? 0u : left >= N ? 0xffffffffu : (1u << left) - 1u;
        if (left >= N) {
            x = *reinterpret_cast<const Few<T, N> *>(from + i);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x.v[j] = j < left ? from[i + j] : (T)0.f;
        }
        if (!w.bias) {
#pragma unroll
            for (int j = 0; j < N; ++j) b.v[j] = 0.f;
        } else if (left >= N) {
            b = *reinterpret_cast<const Few<float, N> *>(w.bias + i);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) b.v[j] = j < left ? w.bias[i + j] : 0.f;
        }
        if (w.mask && left > 0) {    // (the bits may lie in two words)
            const int last = (a.V - 1) >> 5, word = i >> 5;
            const unsigned long long two = w.mask[word] | (unsigned long long)w.mask[word < last ? word + 1 : last] << 32;
            allow &= (uint32_t)(two >> (i & 31));
        }
        cell = nullptr;
        if (a.history) {
            int *cells = all[wave].cell;
            for (int q = lane; q < 64 * N; q += 64) cells[q] = 0;
            __syncthreads();
            walk<4>(w.hist, w.len, 0, a.V, lane, 64, [&](int id) { atomicAdd(&cells[id], 1); });
            __syncthreads();
            cell = cells + i;
        }
    }
    // logits with the penalties and the bias: y before the last factor
    template <typename C> __device__ __forceinline__ void sums(const Rule<C> &rule, C (&v)[N]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (C)(float)x.v[j];
        if (cell) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int c = cell[j];
                v[j] = c > 0 ? rule.penalised(v[j], c) : v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += (C)b.v[j];
    }
    __device__ __forceinline__ void values(const Rule<float> &rule, float no, float (&y)[N]) const {
        sums(rule, y);
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = select(bit_word(allow, j), scaled(y[j], rule.scale), no);
    }
    // d y / d l of a seen element's logit l: what its gradient is multiplied by
    __device__ __forceinline__ void times_factor(const Rule<float> &rule, const Few<T, N> &l, float (&v)[N]) const {
        if (cell) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (cell[j] > 0) v[j] *= rule.factor((float)l.v[j]);
        }
    }
    __device__ __forceinline__ void store(T *row, const float (&v)[N]) const {
        if (left >= N) {
            Few<T, N> p;
#pragma unroll
            for (int j = 0; j < N; ++j) p.v[j] = (T)v[j];
            *reinterpret_cast<Few<T, N> *>(row + i) = p;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j < left) row[i + j] = (T)v[j];
        }
    }
};

// ---- wider rows: runs
// What a run's workgroup knows of the row's past.  bits: one for each element of the run; the list of the seen ones in the order of the
// bits, entry rank[i / 32] being the first of word i / 32: id (the element of the run) and its finished value, -inf where the mask forbids it.
template <typename C> struct Seen {
    C *value;
    uint32_t *bits;
    uint16_t *rank, *small;
    int total, cap;                  // entries of the list; room in it
    // Beside entry u's count (which `value` holds first) there are two 16-bit numbers: its id, and - while the list is made - one of the
    // history's ids in the run, in any order.  A double has room for them in itself (the id is not asked for after the value is there).
    static constexpr int BESIDE = sizeof(C) == 8 ? 0 : 4;
    static size_t bytes(int run, int len) {
        const int cap = len < run ? len : run;
        return ((size_t)cap * (sizeof(C) + BESIDE) + 15) / 16 * 16 + (size_t)run / 32 * 6;
    }
    __device__ Seen(char *lds, int run, int len) : total(0), cap(len < run ? len : run) {
        value = reinterpret_cast<C *>(lds), small = reinterpret_cast<uint16_t *>(lds + (BESIDE ? (size_t)cap * sizeof(C) : 0));
        bits = reinterpret_cast<uint32_t *>(lds + ((size_t)cap * (sizeof(C) + BESIDE) + 15) / 16 * 16);
        rank = reinterpret_cast<uint16_t *>(bits + run / 32);
    }
    __device__ __forceinline__ uint16_t &id(int u) const { return small[BESIDE ? u : 4 * u + 2]; }
    __device__ __forceinline__ uint16_t &hit(int u) const { return small[BESIDE ? cap + u : 4 * u + 3]; }
    // (once the list is finished, beside a float: what is left to ask about entry u)
    __device__ __forceinline__ bool allowed(int u) const { return hit(u) & 1; }
    __device__ __forceinline__ bool above_zero(int u) const { return hit(u) & 2; }
    // the entries [x, y) of the run's elements [at, at + span), at and span multiples of 32
    __device__ __forceinline__ int2 among(int at, int span, int n) const {
        const int next = (at + span) >> 5;
        return make_int2(rank[at >> 5], next < (n + 31) >> 5 ? rank[next] : total);
    }
};

constexpr int RUN_MAX = 32768;       // ranks and ids fit 16 bits; 1024 words of bits, 4 for each thread

// Sets the bits of the seen elements of [base, base + n); with LIST also ranks and the list of finished values.  The workgroup calls it.
template <bool LIST, typename T, typename C>
__device__ __forceinline__ void look_back(Seen<C> &seen, const Row<T> &w, const Rule<C> &rule, int base, int n) {
    __shared__ int wave_total[WAVES], hits;
    const int words = (n + 31) >> 5, tid = threadIdx.x;
    const bool kept = LIST && w.len <= seen.cap;   // the ids found are kept, for the second time
    for (int i = tid; i < words; i += NT) seen.bits[i] = 0u;
    if (tid == 0) hits = 0;
    __syncthreads();
    walk<8>(w.hist, w.len, base, n, tid, NT, [&](int at) {
        atomicOr(&seen.bits[at >> 5], 1u << (at & 31));
        if (kept) seen.hit(atomicAdd(&hits, 1)) = (uint16_t)at;
    });
    __syncthreads();
    if constexpr (LIST) {
        // ranks: every thread 4 words, their bits counted and summed over the workgroup
        int here[RUN_MAX / 32 / NT], mine = 0;
#pragma unroll
        for (int q = 0; q < RUN_MAX / 32 / NT; ++q) {
            const int i = tid * (RUN_MAX / 32 / NT) + q;
            here[q] = mine;
            mine += i < words ? __popc(seen.bits[i]) : 0;
        }
        const int upto = (int)wave_scan((float)mine);   // (exact: at most 32768)
        if ((tid & 63) == 63) wave_total[tid >> 6] = upto;
        __syncthreads();
        int first = upto - mine, total = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            if (v < (tid >> 6)) first += wave_total[v];
            total += wave_total[v];
        }
        seen.total = total;
#pragma unroll
        for (int q = 0; q < RUN_MAX / 32 / NT; ++q) {
            const int i = tid * (RUN_MAX / 32 / NT) + q;
            if (i < words) seen.rank[i] = (uint16_t)(first + here[q]);
        }
        int *count = reinterpret_cast<int *>(seen.value);   // entry u: first its count, in the value's first 4 bytes
        constexpr int STEP = sizeof(C) / 4;
        for (int u = tid; u < total; u += NT) count[u * STEP] = 0;
        __syncthreads();
        auto count_one = [&](int at) {
            const uint32_t word = seen.bits[at >> 5];
            const int u = seen.rank[at >> 5] + __popc(word & ((1u << (at & 31)) - 1u));
            atomicAdd(&count[u * STEP], 1);
            seen.id(u) = (uint16_t)at;                       // (the same from every thread that holds the id)
        };
        if (kept) {
            for (int j = tid; j < hits; j += NT) count_one(seen.hit(j));
        } else {
            walk<8>(w.hist, w.len, base, n, tid, NT, count_one);
        }
        __syncthreads();
        for (int u = tid; u < total; u += NT) {
            const int at = seen.id(u), i = base + at;
            const float l = (float)w.x[i];
            const bool allowed = w.allows(i);
            const C v = rule.penalised((C)l, count[u * STEP]) + (w.bias ? (C)w.bias[i] : (C)0);
            seen.value[u] = allowed ? scaled(v, rule.scale) : (C)NEG;
            if (Seen<C>::BESIDE) seen.hit(u) = (uint16_t)((allowed ? 1 : 0) | (l > 0.f ? 2 : 0));
        }
        __syncthreads();
    }
}

// Where a workgroup's run lies.
struct Place {
    int r, base, n;
    __device__ Place(const Args &a, int block) {
        r = a.runs == 1 ? block : (int)((unsigned)block / (unsigned)a.runs);
        base = (block - r * a.runs) * a.run;
        n = a.V - base < a.run ? a.V - base : a.run;
    }
};

// bits of the seen elements of the pack that begins at element `at` of the run
template <int VEC, typename C> __device__ __forceinline__ uint32_t seen_bits(const Seen<C> &seen, int at, int n) {
    return at < n ? (seen.bits[at >> 5] >> (at & 31)) & ((1u << VEC) - 1u) : 0u;
}

// A step's results on their way out: where some of them are replaced (`any`, the same in every lane: by `replace(results of the step)`), the wave
// takes them through LDS, so that whole lines are stored.  (Stores of the replaced elements alone, behind the step's, cost a
// second write of their lines: 119 against 101 us for shape of 4000 rows of 32768 bf16 with histories of up to 500.)
template <typename P, typename T> struct Stage {
    T cell[WAVES][P::SPAN];
    template <typename Packs, typename F> __device__ __forceinline__ void pass(Packs &out, bool any, F replace) {
        if (!any) return;
        constexpr int K = sizeof(out) / sizeof(out[0]);
        T *mine = cell[threadIdx.x >> 6];
        in_order();                  // (the step before has been read)
#pragma unroll
        for (int k = 0; k < K; ++k) *reinterpret_cast<uint4 *>(mine + P::at(k)) = __builtin_bit_cast(uint4, out[k]);
        in_order();
        replace(mine);
        in_order();
#pragma unroll
        for (int k = 0; k < K; ++k) out[k] = __builtin_bit_cast(Pack<T>, *reinterpret_cast<uint4 *>(mine + P::at(k)));
    }
    // one wave's accesses to LDS take place in their order; the compiler keeps to it here
    static __device__ __forceinline__ void in_order() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
};

// Streams through a run: `f(packs, element of the row that they begin at)` for every step of SPAN elements, the steps shared out to the
// waves in turn.  AHEAD: a step's loads are requested while the step before is worked on, the first before `prepare()` runs.  Where
// that costs waves of a SIMD it does not pay: the draw takes 114 registers without and 144 with it (44 against 48 us for 250 rows of 100003), the backward
// of log_prob 56 and 82 (99.6 against 102.9 us for 4000 rows of 32768); shape has 76 with it (58 us for 256 rows of
// 131072, 59 without; 142 and 138 for 4000 of 32768), the forward of log_prob 72 (no difference).
template <typename P, bool AHEAD, typename T, typename Prepare, typename F>
__device__ __forceinline__ void stream(const Args &a, const Place &at, const Row<T> &w, const T *from, Prepare prepare, F f) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), full = at.n / P::SPAN;
    P one;
    int s = wave;
    if (AHEAD && s < full) one.load(from, w, at.base + s * P::SPAN);
    prepare();
    if constexpr (!AHEAD) {
        for (; s < full; s += WAVES) {
            one.load(from, w, at.base + s * P::SPAN);
            f(one, at.base + s * P::SPAN);
        }
    } else if (s < full) {
        P two;
        const int last = full - 1 - ((full - 1 - wave) & (WAVES - 1));   // (after the last step it is requested once more: no path without loads)
        for (;;) {
            two.load(from, w, at.base + std::min(s + WAVES, last) * P::SPAN);
            f(one, at.base + s * P::SPAN);
            s += WAVES;
            if (s >= full) break;
            one.load(from, w, at.base + std::min(s + WAVES, last) * P::SPAN);
            f(two, at.base + s * P::SPAN);
            s += WAVES;
            if (s >= full) break;
        }
    }
    if (s == full && full * P::SPAN < at.n) {
        one.load_end(from, w, at.base + s * P::SPAN, a.V);
        f(one, at.base + s * P::SPAN);
    }
}

extern __shared__ __align__(16) char run_lds[];

// A row's token where it lies in the run: its value as if it had not been seen, requested before the stream.  (Looking for it among the elements
// that stream past would cost 2 instructions for each of them.)
struct Token {
    int i;                           // the element of the row; -1: none in the run
    float y;                         // -inf where the mask forbids it
    template <typename T> __device__ __forceinline__ Token(int tok, const Place &at, const Row<T> &w, const Rule<float> &rule) {
        const bool here = tok >= at.base && tok < at.base + at.n;
        const int j = here ? tok : at.base;
        float v = (float)w.x[j];
        if (w.bias) v += w.bias[j];
        i = here ? tok : -1, y = w.allows(j) ? scaled(v, rule.scale) : NEG;
    }
    __device__ __forceinline__ bool unseen(const Args &a, const Seen<float> &seen, const Place &at) const {
        return i >= 0 && !(a.history && ((seen.bits[(i - at.base) >> 5] >> ((i - at.base) & 31)) & 1u));
    }
};

// ---- shape.  Measured: rows of 302 f32, 25600 of them, 17.4 us forward and 21.0 backward (62 MB each way: 3.6 and 3.0 TB/s, bound by
// the latency of a row's dependent loads); 256 rows of 131072 bf16 with a bias row each 57 us (272 MB: 4.8 TB/s, the rate of a copy is 4.7).
template <typename T, int N> __global__ __launch_bounds__(NT) void shape_rows_kernel(Args a, T *__restrict__ out, long long ld_out) {
    __shared__ typename Narrow<T, N>::Lds lds[WAVES];
    const Narrow<T, N> u(a, lds, (const T *)a.logits, a.ld_b, a.ld_t);
    if (!u.live) return;
    float v[N];
    u.values(Rule<float>(u.w, 1.f), NEG, v);
    u.store(out + u.r * ld_out, v);
}

template <typename T, int K, bool BIAS> __global__ __launch_bounds__(NT) void shape_run_kernel(Args a, T *__restrict__ out, long long ld_out) {
    using P = Packs<T, K, BIAS>;
    const Place at(a, blockIdx.x);
    const Row<T> w = row_of<T>(a, at.r);
    const Rule<float> rule(w, 1.f);
    Seen<float> seen(run_lds, a.run, a.L);
    __shared__ __align__(16) Stage<P, T> stage;
    T *row = out + at.r * ld_out;
    const int lane = threadIdx.x & 63;
    stream<P, true>(a, at, w, w.x, [&] { if (a.history) look_back<true>(seen, w, rule, at.base, at.n); },
                 [&](const P &p, int first) {
        Pack<T> o[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float v[P::VEC];
            p.raw(k, rule, v);
            p.masked(k, NEG, v);
            o[k] = rounded<T>(v);
        }
        if (a.history) {
            const int2 some = seen.among(first - at.base, P::SPAN, at.n);
            stage.pass(o, __builtin_amdgcn_readfirstlane(some.y - some.x) != 0, [&](T *to) {
                for (int u = some.x + lane; u < some.y; u += 64) to[at.base + seen.id(u) - first] = (T)seen.value[u];
            });
        }
#pragma unroll
        for (int k = 0; k < K; ++k) store_pack(row + first + P::at(k), o[k], a.V - first - P::at(k));
    });
}

// dl = g dy/dl; the logits are read only where the sign of a seen token's decides.
template <typename T, int N>
__global__ __launch_bounds__(NT) void shape_rows_bwd_kernel(Args a, const T *__restrict__ g, long long ld_gb, long long ld_gt,
                                                            T *__restrict__ dx, long long ld_dx) {
    __shared__ typename Narrow<T, N>::Lds lds[WAVES];
    a.bias = nullptr;
    const Narrow<T, N> u(a, lds, g, ld_gb, ld_gt);
    if (!u.live) return;
    const Rule<float> rule(u.w, 1.f);
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)u.x.v[j] * rule.scale;
    if (u.cell) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (u.cell[j] > 0) v[j] *= rule.factor((float)u.w.x[u.i + j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = select(bit_word(u.allow, j), v[j], 0.f);
    u.store(dx + u.r * ld_dx, v);
}

template <typename T, int K>
__global__ __launch_bounds__(NT) void shape_run_bwd_kernel(Args a, const T *__restrict__ g, long long ld_gb, long long ld_gt,
                                                           T *__restrict__ dx, long long ld_dx) {
    using P = Packs<T, K, false>;
    const Place at(a, blockIdx.x);
    const Row<T> w = row_of<T>(a, at.r);
    const Rule<float> rule(w, 1.f);
    Seen<float> seen(run_lds, a.run, 0);                 // (bits alone)
    const int b = a.T == 1 ? at.r : (int)((unsigned)at.r / (unsigned)a.T), t = at.r - b * a.T;
    stream<P, true>(a, at, w, g + b * ld_gb + t * ld_gt, [&] { if (a.history) look_back<false>(seen, w, rule, at.base, at.n); },
                 [&](const P &p, int first) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = first + P::at(k);
            float v[P::VEC];
            p.raw(k, rule, v);
            if (a.history) {
                const uint32_t s = seen_bits<P::VEC>(seen, i - at.base, at.n);
                if (s) {
#pragma unroll
                    for (int j = 0; j < P::VEC; ++j)
                        if ((s >> j) & 1u) v[j] *= rule.factor((float)w.x[i + j]);
                }
            }
            p.masked(k, 0.f, v);
            store_pack(dx + at.r * ld_dx + i, rounded<T>(v), a.V - i);
        }
    });
}

// ---- log_prob.  Measured, 4000 rows of 32768 bf16 with histories of up to 500, a bias and masks: forward 84 us (262 MB; 50 us, 5.2 TB/s, with neither
// bias nor history: the bias costs 15, its 4 bytes an element coming from L2, the look back 11), backward 99.6 us (524 MB: 5.3 TB/s).
// Streamed stores took the backward from 163 to 128 us, reading the rows from the end 154 to 128, whole lines (Stage) 122 to 101.
// Sums are 32-bit.  With u = 2^-24, the sum's relative error is at most
//     (3 ln V + 2) u   from the exponentials: three rounded factors in each argument t = y - m, which weighted by the terms themselves averages at
//                      most ln V (what a lane's maximum moved by on the way counts as part of t), and the unit's 1 ulp,
//     3 u              for each rescaling of a partial sum: a lane's steps (8 of 16 elements in a run of 32768) and entries of the list of seen ids
//                      (at most 4096 over 256 threads: 16), then its wave, the workgroup and the row,
//     u                for each addition: 128 terms and 16 entries in a lane's chain, 6 levels over the wave, 4 waves, runs / 64 + 6 over the row's runs:
// under 290 u + u runs / 64 for a row of 32768, and far below it on average.
template <typename T, int N>
__global__ __launch_bounds__(NT) void log_prob_rows_kernel(Args a, const int64_t *__restrict__ tokens, float *__restrict__ lp,
                                                           float2 *__restrict__ stats) {
    __shared__ typename Narrow<T, N>::Lds lds[WAVES];
    const Narrow<T, N> u(a, lds, (const T *)a.logits, a.ld_b, a.ld_t);
    if (!u.live) return;
    const int tok = token_of(tokens[u.r], a.V);
    float y[N], m = NEG, yt = 0.f;
    u.values(Rule<float>(u.w, 1.f), NEG, y);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        m = fmaxf(m, y[j]);
        if (u.i + j == tok) yt = y[j];
    }
    m = wave_max(m);
    const float from = reference_of(m);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += exp_from(y[j], from);
    s = wave_sum(s);
    const float v = tok >= 0 ? log_prob_of(from_lane(yt, tok / N), m, s) : 0.f;
    if (u.lane == 0) lp[u.r] = v, stats[u.r] = make_float2(m, s);
}

// (maximum, sum) pairs joined: the sums in units of the common maximum.  An empty part adds its 0, one that holds nothing but NaN its NaN.
__device__ __forceinline__ float rebased(float2 part, float m) { return part.x == NEG ? part.y : part.y * exp_from(part.x, reference_of(m)); }

template <typename T, int K, bool BIAS>
__global__ __launch_bounds__(NT) void log_prob_run_kernel(Args a, const int64_t *__restrict__ tokens, float *__restrict__ lp,
                                                          float2 *__restrict__ stats, float2 *__restrict__ part, float *__restrict__ target) {
    using P = Packs<T, K, BIAS>;
    __shared__ float2 waves[WAVES];
    __shared__ float at_token;
    const Place at(a, blockIdx.x);
    const Row<T> w = row_of<T>(a, at.r);
    const Rule<float> rule(w, 1.f);
    Seen<float> seen(run_lds, a.run, a.L);
    const int tok = token_of(tokens[at.r], a.V);
    const Token token(tok, at, w, rule);
    float m = NEG, s = 0.f;          // of this lane's elements so far
    stream<P, true>(a, at, w, w.x, [&] { if (a.history) look_back<true>(seen, w, rule, at.base, at.n); },
                 [&](const P &p, int first) {
        float y[K][P::VEC], top = m;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = first + P::at(k);
            p.raw(k, rule, y[k]);
            uint32_t left_out = 0u;
            if (a.history) left_out = seen_bits<P::VEC>(seen, i - at.base, at.n);
            const uint32_t allow = p.allow[k] & ~left_out;
#pragma unroll
            for (int j = 0; j < P::VEC; ++j) y[k][j] = select(bit_word(allow, j), y[k][j], NEG), top = fmaxf(top, y[k][j]);
        }
        const float from = reference_of(top);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < P::VEC; ++j) sum += exp_from(y[k][j], from);
        s = s * exp_from(m, from) + sum, m = top;
    });
    if (threadIdx.x == 0 && token.unseen(a, seen, at)) at_token = token.y;
    if (a.history) {
        for (int u = threadIdx.x; u < seen.total; u += NT) {
            const float y = seen.value[u], top = fmaxf(m, y), from = reference_of(top);
            s = s * exp_from(m, from) + exp_from(y, from), m = top;
            if (at.base + seen.id(u) == tok) at_token = y;
        }
    }
    const float top = wave_max(m);
    s = wave_sum(rebased(make_float2(m, s), top));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = make_float2(top, s);
    __syncthreads();
    if (threadIdx.x != 0) return;
    m = NEG, s = 0.f;
    for (int v = 0; v < WAVES; ++v) m = fmaxf(m, waves[v].x);
    for (int v = 0; v < WAVES; ++v) s += rebased(waves[v], m);
    if (a.runs == 1) {
        lp[at.r] = tok >= 0 ? log_prob_of(at_token, m, s) : 0.f, stats[at.r] = make_float2(m, s);
    } else {
        part[(long long)at.r * a.runs + at.base / a.run] = make_float2(m, s);
        if (tok >= at.base && tok < at.base + at.n) target[at.r] = at_token;
    }
}

// One wave per row: its runs joined.
__global__ __launch_bounds__(NT) void log_prob_join_kernel(int R, int V, int runs, const int64_t *__restrict__ tokens,
                                                           const float2 *__restrict__ part, const float *__restrict__ target,
                                                           float *__restrict__ lp, float2 *__restrict__ stats) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (r >= R) return;
    const float2 *p = part + (long long)r * runs;
    float m = NEG;
    for (int i = lane; i < runs; i += 64) m = fmaxf(m, p[i].x);
    m = wave_max(m);
    float s = 0.f;
    for (int i = lane; i < runs; i += 64) s += rebased(p[i], m);
    s = wave_sum(s);
    if (lane != 0) return;
    const long long tok = tokens[r];
    lp[r] = tok >= 0 && tok < V ? log_prob_of(target[r], m, s) : 0.f;
    stats[r] = make_float2(m, s);
}

// What the backward of a row is made of: dl_i = (others * exp(y_i - from) + [i = tok] at_token) * (factor of a seen token)
struct Slope {
    int tok;
    bool zero;                       // a row without a token, or with none allowed
    float at_token, others, from;
    __device__ Slope(const Args &a, int r, const int64_t *tokens, const float2 *stats, const float *g, const Rule<float> &rule) {
        const float2 st = stats[r];
        tok = token_of(tokens[r], a.V), zero = tok < 0 || (st.x == NEG && st.y == 0.f);
        at_token = g[r] * rule.scale, others = -at_token * reciprocal(st.y), from = reference_of(st.x);
    }
    template <int VEC> __device__ __forceinline__ void of(int i, float (&v)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = others * exp_from(v[j], from);
        const unsigned here = (unsigned)(tok - i);
        if (here < (unsigned)VEC) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j == (int)here) v[j] += at_token;
        }
    }
};

template <typename T, int N>
__global__ __launch_bounds__(NT) void log_prob_rows_bwd_kernel(Args a, const int64_t *__restrict__ tokens, const float2 *__restrict__ stats,
                                                               const float *__restrict__ g, T *__restrict__ dx, long long ld_dx) {
    __shared__ typename Narrow<T, N>::Lds lds[WAVES];
    const Narrow<T, N> u(a, lds, (const T *)a.logits, a.ld_b, a.ld_t);
    if (!u.live) return;
    const Rule<float> rule(u.w, 1.f);
    const Slope slope(a, u.r, tokens, stats, g, rule);
    float v[N];
    u.values(rule, NEG, v);
    slope.of(u.i, v);
    u.times_factor(rule, u.x, v);
    const uint32_t allow = slope.zero ? 0u : u.allow;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = select(bit_word(allow, j), v[j], 0.f);
    u.store(dx + u.r * ld_dx, v);
}

// (The rows are taken from the last one down: what the forward pass read last is what the last-level cache still holds.)
template <typename T, int K, bool BIAS>
__global__ __launch_bounds__(NT) void log_prob_run_bwd_kernel(Args a, const int64_t *__restrict__ tokens, const float2 *__restrict__ stats,
                                                              const float *__restrict__ g, T *__restrict__ dx, long long ld_dx) {
    using P = Packs<T, K, BIAS>;
    const Place at(a, gridDim.x - 1 - blockIdx.x);
    const Row<T> w = row_of<T>(a, at.r);
    const Rule<float> rule(w, 1.f);
    Seen<float> seen(run_lds, a.run, a.L);
    const Slope slope(a, at.r, tokens, stats, g, rule);
    const Token token(slope.tok, at, w, rule);
    const float above = rule.factor(1.f), below = rule.factor(-1.f);
    const bool token_allowed = w.allows(token.i < 0 ? at.base : token.i);
    __shared__ __align__(16) Stage<P, T> stage;
    T *row = dx + at.r * ld_dx;
    const int lane = threadIdx.x & 63;
    stream<P, false>(a, at, w, w.x, [&] { if (a.history) look_back<true>(seen, w, rule, at.base, at.n); },
                 [&](const P &p, int first) {
        Pack<T> o[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float v[P::VEC];
            p.raw(k, rule, v);
            const uint32_t allow = slope.zero ? 0u : p.allow[k];
#pragma unroll
            for (int j = 0; j < P::VEC; ++j) v[j] = select(bit_word(allow, j), slope.others * exp_from(v[j], slope.from), 0.f);
            o[k] = rounded<T>(v);
        }
        const bool holds_token = (unsigned)(token.i - first) < (unsigned)P::SPAN;
        int2 some = make_int2(0, 0);
        if (a.history) some = seen.among(first - at.base, P::SPAN, at.n);
        stage.pass(o, holds_token || __builtin_amdgcn_readfirstlane(some.y - some.x) != 0, [&](T *to) {
            if (holds_token && lane == 0 && token.unseen(a, seen, at)) {
                float v[1] = {token.y};
                slope.of(token.i, v);
                to[token.i - first] = (T)(slope.zero || !token_allowed ? 0.f : v[0]);
            }
            for (int u = some.x + lane; u < some.y; u += 64) {
                const int i = at.base + seen.id(u);
                float v[1] = {seen.value[u]};
                slope.of(i, v);
                to[i - first] = (T)(slope.zero || !seen.allowed(u) ? 0.f : v[0] * (seen.above_zero(u) ? above : below));
            }
        });
#pragma unroll
        for (int k = 0; k < K; ++k) store_pack(row + first + P::at(k), o[k], a.V - first - P::at(k));
    });
}

// ---- draw.  Measured: 10000 rows of 302 f32 13.6 us (vector unit 76 % busy: 500 instructions a row, half of them 64-bit); 250 rows of
// 100003 f16 with histories of up to 4000 44 us for the weights (38 instructions an element, 25 of them 64-bit, about 5 cycles each: 30 us) and
// 9 us for the pick.
template <typename T, int N>
__global__ __launch_bounds__(NT) void draw_rows_kernel(Args a, const float *__restrict__ uniforms, long long ld_u, int64_t empty,
                                                       int64_t *__restrict__ out, float *__restrict__ lp) {
    __shared__ typename Narrow<T, N>::Lds lds[WAVES];
    const Narrow<T, N> u(a, lds, (const T *)a.logits, a.ld_b, a.ld_t);
    if (!u.live) return;
    const Rule<double> rule(u.w, LOG2E64);
    double v[N], e[N];
    u.sums(rule, v);
    const uint32_t allow[1] = {u.allow};
    double guess = NEG64;
    const Weights all = weigh<1, N>(allow, rule.scale, guess, [&](int, double (&to)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) to[j] = v[j];
    }, [&](int, const double (&from)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) e[j] = from[j];
    }, [](auto) {});
    const Pick pick = pick_in_wave(e, 0., (double)uniforms[u.r * ld_u] * all.sum);
    if (u.lane == 0) {
        const bool ok = all.sum > 0. && fabs(all.m) < __builtin_inf() && pick.index >= 0;
        out[u.r] = ok ? pick.index : empty;
        lp[u.r] = ok ? log_of_share(pick.value, all.sum) : (all.m == NEG64 ? NEG : __builtin_nanf(""));
    }
}

// A wide row, first: every step of a run leaves the sum of its weights and its m.
struct Piece {
    double s, m;
};
template <typename T, int K, bool BIAS> __global__ __launch_bounds__(NT) void draw_run_kernel(Args a, Piece *__restrict__ part) {
    using P = Packs<T, K, BIAS>;
    const Place at(a, blockIdx.x);
    const Row<T> w = row_of<T>(a, at.r);
    const Rule<double> rule(w, LOG2E64);
    Seen<double> seen(run_lds, a.run, a.L);
    const int pieces = (a.V + P::SPAN - 1) / P::SPAN, lane = threadIdx.x & 63;
    double guess = NEG64;
    stream<P, false>(a, at, w, w.x, [&] { if (a.history) look_back<true>(seen, w, rule, at.base, at.n); },
                 [&](const P &p, int first) {
        uint32_t allow[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            allow[k] = p.allow[k];
            if (a.history) allow[k] &= ~seen_bits<P::VEC>(seen, first + P::at(k) - at.base, at.n);
        }
        int2 some = make_int2(0, 0);  // the list's entries of this step
        if (a.history) some = seen.among(first - at.base, P::SPAN, at.n);
        const Weights all = weigh<K, P::VEC>(allow, rule.scale, guess, [&](int k, double (&v)[P::VEC]) { p.sums(k, v); }, [](int, auto &) {},
                                             [&](auto f) {
            for (int u = some.x + lane; u < some.y; u += 64) f(seen.value[u]);
        });
        if (lane == 0) part[(long long)at.r * pieces + first / P::SPAN] = Piece{all.sum, all.m};
    });
}

// Then one workgroup per row: the pieces joined in index order, the piece that holds u * total found, and its elements computed and walked
// again, a few for each thread.
template <typename T, int SPAN>
__global__ __launch_bounds__(NT) void draw_join_kernel(Args a, const Piece *__restrict__ part, const float *__restrict__ uniforms,
                                                       long long ld_u, int64_t empty, int64_t *__restrict__ out, float *__restrict__ lp) {
    constexpr int EACH = SPAN / NT;
    __shared__ __align__(16) Counts<SPAN> lds;
    __shared__ double sums[WAVES];
    __shared__ Pick picks[WAVES];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pieces = (a.V + SPAN - 1) / SPAN;
    const Piece *p = part + (long long)r * pieces;
    if (a.history) {
        for (int i = tid; i < SPAN; i += NT) lds.cell[i] = 0;
    }
    double m = NEG64;
    bool bad = false;
    for (int i = lane; i < pieces; i += 64) m = fmax(m, p[i].m), bad |= p[i].m != p[i].m;
    m = wave_max(m);
    const bool nan = __ballot(bad) != 0;
    if (nan || !(m > NEG64 && m < __builtin_inf())) {   // (the same in every wave)
        if (tid == 0) out[r] = empty, lp[r] = !nan && m == NEG64 ? NEG : __builtin_nanf("");
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
        const double s = i < pieces ? p[i].s * power_of_two(p[i].m - m) : 0.;
        const double inc = wave_scan(s), ahead = cum + (inc - s);
        const unsigned long long some = __ballot(s > 0.), hit = __ballot(s > 0. && cum + inc > thr);
        if (some) {
            const int l = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
            found = base + l, before = from_lane(ahead, l), over = hit != 0;
        }
        cum += from_lane(inc, 63);
    }
    const Row<T> w = row_of<T>(a, r);
    const int base = found * SPAN, n = a.V - base < SPAN ? a.V - base : SPAN;
    // this thread's elements, requested before the history is walked
    const int mine = tid * EACH;
    float x[EACH], b[EACH];
    uint32_t allow = 0u;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const bool in = mine + j < n;
        x[j] = in ? (float)w.x[base + mine + j] : 0.f;
        b[j] = in && w.bias ? w.bias[base + mine + j] : 0.f;
        const bool yes = in && (!w.mask || ((w.mask[(base + mine + j) >> 5] >> ((base + mine + j) & 31)) & 1u));
        allow |= (yes ? 1u : 0u) << j;
    }
    if (a.history) {
        __syncthreads();
        walk<8>(w.hist, w.len, base, n, tid, NT, [&](int at) { atomicAdd(&lds.cell[at], 1); });
        __syncthreads();
    }
    const Rule<double> rule(w, LOG2E64);
    double e[EACH], s = 0.;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        double y = (double)x[j];
        if (a.history) {
            const int c = lds.cell[mine + j];
            if (c > 0) y = rule.penalised(y, c);
        }
        e[j] = (allow >> j) & 1u ? power_of_two(scaled(y + (double)b[j], rule.scale) - m) : 0., s += e[j];
    }
    s = wave_sum(s);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    for (int v = 0; v < wave; ++v) before += sums[v];
    const Pick pick = pick_in_wave(e, before, thr);
    if (lane == 0) picks[wave] = pick;
    __syncthreads();
    if (tid == 0) {
        Pick best = {0., -1, false};
        for (int v = 0; v < WAVES && !best.over; ++v)
            if (picks[v].index >= 0) best = picks[v], best.index += v * 64 * EACH;
        out[r] = best.index >= 0 ? base + best.index : empty;
        lp[r] = best.index >= 0 ? log_of_share(best.value, total) : __builtin_nanf("");
    }
}

// ---- host
constexpr long long MAX_BLOCKS = (1ll << 24) - 1;   // a launch holds fewer than 2^32 threads

int elem_size(int dtype) { return dtype == PSVAE_F32 ? 4 : 2; }

// How a call is cut.
struct Cut {
    bool rows;                       // a wave per row
    int per_lane;                    // elements a lane takes at once: of a row 1 to 16, of a run's step 8 or 16
    int run, runs;                   // elements of a run, runs of a row
    long long blocks;
};
Cut cut_of(const psvae_shaping *s) {
    Cut c;
    const long long R = (long long)s->B * s->T;
    c.rows = s->V <= ROW_MAX;
    if (c.rows) {
        c.run = s->V, c.runs = 1;
        for (int n : {1, 2, 3, 4, 5, 6, 8, 12, 16}) {   // (the forms of PSVAE_LAUNCH_ROWS)
            c.per_lane = n;
            if (64 * n >= s->V) break;
        }
        c.blocks = (R + WAVES - 1) / WAVES;
        return c;
    }
    // The longest runs that leave 960 workgroups: a run pays for its walk through the history once, and 4 workgroups for each compute unit, 1024,
    // are in flight at a time.  The number of runs being rounded up, 960 seldom comes to more than 1024, and aiming at 1024 does: draws of 120, 200
    // and 250 rows of 100003 take 30, 38 and 44 us, and 33, 43 and 46; of 32003 16, 20 and 21, and 16, 24 and 24.  The other way round at
    // 64 rows (32003: 14.4 and 13.1 us; 131072: 23 and 22); 16 rows or fewer and 700 or more show no difference.  Down to 2048 elements, in smaller steps, where
    // rows are few.  A long history's list of seen ids has to fit LDS: at most 4096 of them.  So with ROOM for more (L; how many are in use is only
    // known on the device) runs have at most 4096 elements, and every one of them walks the history - twice, where more than 4096 ids are in use, which
    // are then not kept in between: rows * (V / 4096) * 16 * (ids in use) bytes, mostly from L2.  250 rows of 100003 f16, shape / log_prob / draw_run:
    //     500 ids in use, room for 4096: 28 / 22 / 35 us;  room for 4097, or 65536: 42 / 41 / 47
    //     4096 ids: 43 / 31 / 44;  4097: 80 / 72 / 81;  8192: 118 / 104 / 110;  65536: 694 / 566 / 573
    // (16 rows or fewer have short runs anyway: no difference between a room of 4096 and one of 65536.)
    const int longest = s->history != nullptr && s->L > 4096 ? 4096 : RUN_MAX;
    long long runs = std::max<long long>(psvae_cdiv(s->V, longest), std::min<long long>(psvae_cdiv(s->V, 2048), (960 + R - 1) / std::max<long long>(R, 1)));
    c.run = psvae_cdiv(psvae_cdiv(s->V, runs), 1024) * 1024;
    if (c.run < 2048) c.run = 2048;
    c.per_lane = c.run > 2048 ? 16 : 8;
    c.runs = psvae_cdiv(s->V, c.run);
    c.blocks = R * c.runs;
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
    PSVAE_REQUIRE(is_in_range(s->repetition) && is_in_range(s->temperature), PSVAE_EINVAL,
                  "%s: repetition and temperature must lie in 2^-126 .. 2^126", fn);
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
    const Cut c = cut_of(s);
    a->run = c.run, a->runs = c.runs;
    return PSVAE_OK;
}

// Launches a kernel of the call's type, elements per lane and (where it has both forms) with or without a bias.  BYTES: dynamic LDS.
#define PSVAE_LAUNCH_KERNEL(KERNEL, BYTES, ...) \
    hipLaunchKernelGGL((KERNEL), dim3((unsigned)cut.blocks), dim3(NT), args.history ? (BYTES) : 0, st, __VA_ARGS__)
#define PSVAE_LAUNCH(NAME, T, BYTES, ...)                                                                                           \
    do {                                                                                                                            \
        if (cut.per_lane == 8 && args.bias) PSVAE_LAUNCH_KERNEL((NAME<T, 8 / Elem<T>::VEC, true>), BYTES, __VA_ARGS__);             \
        else if (cut.per_lane == 8) PSVAE_LAUNCH_KERNEL((NAME<T, 8 / Elem<T>::VEC, false>), BYTES, __VA_ARGS__);                    \
        else if (args.bias) PSVAE_LAUNCH_KERNEL((NAME<T, 16 / Elem<T>::VEC, true>), BYTES, __VA_ARGS__);                            \
        else PSVAE_LAUNCH_KERNEL((NAME<T, 16 / Elem<T>::VEC, false>), BYTES, __VA_ARGS__);                                          \
    } while (0)
#define PSVAE_LAUNCH_ROWS(NAME, T, ...)                                                      \
    do {                                                                                     \
        switch (cut.per_lane) {                                                              \
            case 1: PSVAE_LAUNCH_KERNEL((NAME<T, 1>), 0, __VA_ARGS__); break;                \
            case 2: PSVAE_LAUNCH_KERNEL((NAME<T, 2>), 0, __VA_ARGS__); break;                \
            case 3: PSVAE_LAUNCH_KERNEL((NAME<T, 3>), 0, __VA_ARGS__); break;                \
            case 4: PSVAE_LAUNCH_KERNEL((NAME<T, 4>), 0, __VA_ARGS__); break;                \
            case 5: PSVAE_LAUNCH_KERNEL((NAME<T, 5>), 0, __VA_ARGS__); break;                \
            case 6: PSVAE_LAUNCH_KERNEL((NAME<T, 6>), 0, __VA_ARGS__); break;                \
            case 8: PSVAE_LAUNCH_KERNEL((NAME<T, 8>), 0, __VA_ARGS__); break;                \
            case 12: PSVAE_LAUNCH_KERNEL((NAME<T, 12>), 0, __VA_ARGS__); break;              \
            default: PSVAE_LAUNCH_KERNEL((NAME<T, 16>), 0, __VA_ARGS__); break;              \
        }                                                                                    \
    } while (0)
#define PSVAE_LAUNCH_NO_BIAS(NAME, T, BYTES, ...)                                                                  \
    do {                                                                                                           \
        if (cut.per_lane == 8) PSVAE_LAUNCH_KERNEL((NAME<T, 8 / Elem<T>::VEC>), BYTES, __VA_ARGS__);               \
        else PSVAE_LAUNCH_KERNEL((NAME<T, 16 / Elem<T>::VEC>), BYTES, __VA_ARGS__);                                \
    } while (0)

template <typename T> void launch_draw(const Args &args, const Cut &cut, Piece *part, const float *u, long long ld_u, int64_t empty,
                                       int64_t *out, float *lp, hipStream_t st) {
    if (cut.rows) {
        PSVAE_LAUNCH_ROWS(draw_rows_kernel, T, args, u, ld_u, empty, out, lp);
        return;
    }
    PSVAE_LAUNCH(draw_run_kernel, T, Seen<double>::bytes(args.run, args.L), args, part);
    if (cut.per_lane == 8)
        hipLaunchKernelGGL((draw_join_kernel<T, 512>), dim3((unsigned)args.R), dim3(NT), 0, st, args, part, u, ld_u, empty, out, lp);
    else
        hipLaunchKernelGGL((draw_join_kernel<T, 1024>), dim3((unsigned)args.R), dim3(NT), 0, st, args, part, u, ld_u, empty, out, lp);
}

// parts of a wide call's rows: runs for a log-probability (none where one run is the row), steps for a draw
bool sized(const psvae_shaping *s) { return s != nullptr && s->B > 0 && s->T >= 1 && s->V >= 1; }
size_t log_prob_parts(const psvae_shaping *s) {
    const Cut c = cut_of(s);
    return c.runs > 1 ? (size_t)s->B * s->T * c.runs : 0;
}
size_t draw_parts(const psvae_shaping *s) {
    const Cut c = cut_of(s);
    return c.rows ? 0 : (size_t)s->B * s->T * psvae_cdiv(s->V, 64 * c.per_lane);
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
    const size_t lds = Seen<float>::bytes(args.run, args.L);
#define CALL(T)                                                                                       \
    do {                                                                                              \
        if (cut.rows) PSVAE_LAUNCH_ROWS(shape_rows_kernel, T, args, (T *)out, (long long)ld_out);     \
        else PSVAE_LAUNCH(shape_run_kernel, T, lds, args, (T *)out, (long long)ld_out);           \
    } while (0)
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
    const size_t lds = Seen<float>::bytes(args.run, 0);
#define SHAPE_BWD(T) args, (const T *)g, (long long)ld_gb, (long long)ld_gt, (T *)dlogits, (long long)ld_dlogits
#define CALL(T)                                                                     \
    do {                                                                            \
        if (cut.rows) PSVAE_LAUNCH_ROWS(shape_rows_bwd_kernel, T, SHAPE_BWD(T));    \
        else PSVAE_LAUNCH_NO_BIAS(shape_run_bwd_kernel, T, lds, SHAPE_BWD(T));          \
    } while (0)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" size_t psvae_shaped_log_prob_workspace_bytes(const psvae_shaping *shaping) {
    const size_t parts = sized(shaping) ? log_prob_parts(shaping) : 0;
    return parts ? parts * sizeof(float2) + (size_t)shaping->B * shaping->T * sizeof(float) : 0;
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
    float *target = need ? (float *)(part + log_prob_parts(shaping)) : nullptr;
    const size_t lds = Seen<float>::bytes(args.run, args.L);
#define CALL(T)                                                                                               \
    do {                                                                                                      \
        if (cut.rows) PSVAE_LAUNCH_ROWS(log_prob_rows_kernel, T, args, tokens, log_prob, stat2);              \
        else PSVAE_LAUNCH(log_prob_run_kernel, T, lds, args, tokens, log_prob, stat2, part, target);      \
    } while (0)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    if (need) {
        hipLaunchKernelGGL(log_prob_join_kernel, dim3(psvae_cdiv(args.R, WAVES)), dim3(NT), 0, st, args.R, args.V, args.runs,
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
    const size_t lds = Seen<float>::bytes(args.run, args.L);
#define LOG_PROB_BWD(T) args, tokens, (const float2 *)stats, g, (T *)dlogits, (long long)ld_dlogits
#define CALL(T)                                                                           \
    do {                                                                                  \
        if (cut.rows) PSVAE_LAUNCH_ROWS(log_prob_rows_bwd_kernel, T, LOG_PROB_BWD(T));    \
        else PSVAE_LAUNCH(log_prob_run_bwd_kernel, T, lds, LOG_PROB_BWD(T));          \
    } while (0)
    PSVAE_BY_TYPE(CALL);
#undef CALL
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" size_t psvae_shaped_draw_workspace_bytes(const psvae_shaping *shaping) { return sized(shaping) ? draw_parts(shaping) * sizeof(Piece) : 0; }

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
