// The 2-norm over a list of gradient tensors of several types, and the list scaled to a largest norm.
//
//     norm = sqrt(sum_i sum_j g_ij^2);   out_ij = g_ij * min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM at large sizes (one read for the norm, one read and one write for the scaling), by launches at small ones.  The list
// travels as kernel arguments (up to 200 tensors a launch for the norm, 140 for the scaling), so nothing is copied to the device, nothing
// outlives the call and a captured graph holds its own copy.  Every tensor is cut into chunks of so many BYTES - half as many elements
// of a type twice as wide, so that the workgroups finish together - and up to 1024 workgroups a launch take the chunks in turn,
// each with one partial sum at its end.  Squares are formed and added in 64 bits: a float's square neither overflows nor vanishes
// there, and the card does a 64-bit multiply-add at the rate of a 32-bit one, so the sum stays under the time of the loads.
#include "common.h"

#include <algorithm>
#include <math.h>
#include <vector>

namespace {

constexpr int NT = 256;
constexpr int GROUPS = 1024;                    // workgroups of a launch at most: 4 for each compute unit
// Bytes of a chunk: 4 loads of a thread; 16 where a list is large, whose workgroups take many chunks (finding a chunk's tensor costs about a
// microsecond's latency): the norm of 400 M elements in bfloat16 takes 211 us with large chunks, 252 with small ones; a list under 64 MB
// would not reach all compute units with large ones.
constexpr int CHUNK_SMALL = NT * 16 * 4, CHUNK_LARGE = NT * 16 * 16;
constexpr long long LARGE = 64ll << 20;         // bytes of a large list

// A list's part for one launch.  `size`: the elements, with the source's type in bits 60, 61 and the output's in bits 62, 63.  `first`: the
// tensor's first chunk, counted from the launch's first; [n]: chunks in all.
template <int N, bool OUT> struct List {
    static constexpr int ROOM = N;
    const void *src[N];
    void *dst[OUT ? N : 1];
    unsigned long long size[N];
    int first[N + 1];
    int n, chunk;                               // tensors; bytes of a chunk
};
using NormList = List<200, false>;              // 20 bytes each of the 4 KB that kernel arguments may take
using ClipList = List<140, true>;               // 28 bytes
// More partial sums than this are added up by a launch of their own before the scaling's launches, whose workgroups would each read all of
// them: no difference at 20000 tensors (the host's 4 ms cover it), 100000 tensors of 64 elements 57 -> 51 ms.
constexpr int FOLD = 8192;
constexpr unsigned long long ELEMENTS = (1ull << 60) - 1;

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int VEC = 4; };
template <> struct Elem<__bf16> { static constexpr int VEC = 8; };
template <> struct Elem<_Float16> { static constexpr int VEC = 8; };

// 16 bytes at any element's address (a slice of a larger buffer may start anywhere)
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

__device__ __forceinline__ double block_sum(double s, double *sh) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    double t = sh[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) t += sh[w];
    return t;
}

// Chunk c of the launch: f(tensor, source type, output type, first element, elements).
template <typename L, typename F> __device__ __forceinline__ void with_chunk(const L &l, int c, F f) {
    int lo = 0, hi = l.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    const unsigned long long size = l.size[lo];
    const int st = (int)(size >> 60) & 3, each = st == PSVAE_F32 ? l.chunk / 4 : l.chunk / 2;
    const long long at = (long long)(c - l.first[lo]) * each, left = (long long)(size & ELEMENTS) - at;
    f(lo, st, (int)(size >> 62), at, left < each ? (int)left : each);
}

template <typename T> __device__ __forceinline__ double sum_squares(const T *g, int n) {
    constexpr int VEC = Elem<T>::VEC, UNROLL = 4;
    double acc[UNROLL] = {0., 0., 0., 0.};
    int i = threadIdx.x * VEC;
    for (; i + (UNROLL - 1) * NT * VEC + VEC <= n; i += UNROLL * NT * VEC) {
        Pack<T, VEC> p[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) p[u] = *reinterpret_cast<const Pack<T, VEC> *>(g + i + u * NT * VEC);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const double d = (double)(float)p[u].v[j];
                acc[u] = fma(d, d, acc[u]);
            }
    }
    for (; i < n; i += NT * VEC) {
        const int left = n - i < VEC ? n - i : VEC;
        if (left == VEC) {
            const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC> *>(g + i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[0] = fma((double)(float)p.v[j], (double)(float)p.v[j], acc[0]);
        } else {
            for (int j = 0; j < left; ++j) acc[0] = fma((double)(float)g[i + j], (double)(float)g[i + j], acc[0]);
        }
    }
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// Measured: 400 M elements (1.14 GB in bfloat16 and float32) 208 us, 5.4 TB/s; the 63 tensors of this package's
// model, 7.6 MB, 5.9 us and 4 us for the sum of the partial sums.
__global__ __launch_bounds__(NT) void grad_squares_kernel(NormList l, double *__restrict__ partial) {
    __shared__ double sh[NT / 64];
    double s = 0.;
    for (int c = blockIdx.x; c < l.first[l.n]; c += gridDim.x)
        with_chunk(l, c, [&](int i, int st, int, long long at, int n) {
            if (st == PSVAE_F32) s += sum_squares((const float *)l.src[i] + at, n);
            else if (st == PSVAE_BF16) s += sum_squares((const __bf16 *)l.src[i] + at, n);
            else s += sum_squares((const _Float16 *)l.src[i] + at, n);
        });
    s = block_sum(s, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The sum of all partials in one fixed order, the same in every workgroup that forms it.
__device__ __forceinline__ double total_of(const double *partial, int n, double *sh) {
    double s = 0.;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += NT) s += partial[i];
    return block_sum(s, sh);
}

__global__ __launch_bounds__(NT) void grad_norm_kernel(const double *__restrict__ partial, int n, float *__restrict__ norm) {
    __shared__ double sh[NT / 64];
    const double s = total_of(partial, n, sh);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// partial[0] = the sum of all, so that the workgroups of many launches need not each read a long list.
__global__ __launch_bounds__(NT) void grad_total_kernel(double *partial, int n) {
    __shared__ double sh[NT / 64];
    const double s = total_of(partial, n, sh);   // (every read comes before its barrier)
    if (threadIdx.x == 0) partial[0] = s;
}

// Loads and stores of at most 16 bytes a lane, so that a wave's store covers whole lines.
// (Non-temporal: the scaled values are read by a later kernel, far more of them than the caches hold.)
typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t Words2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename T, int N> __device__ __forceinline__ void store_streamed(T *p, const Pack<T, N> &v) {
    if constexpr (sizeof(v) == 8) __builtin_nontemporal_store(__builtin_bit_cast(Words2, v), reinterpret_cast<Words2 *>(p));
    else __builtin_nontemporal_store(__builtin_bit_cast(Words4, v), reinterpret_cast<Words4 *>(p));
}

template <typename S, typename D> __device__ __forceinline__ void scale(const S *g, D *out, int n, float coef) {
    constexpr int VEC = 16 / (sizeof(S) > sizeof(D) ? sizeof(S) : sizeof(D)), UNROLL = 64 / (VEC * (int)sizeof(S));
    int i = threadIdx.x * VEC;
    for (; i + (UNROLL - 1) * NT * VEC + VEC <= n; i += UNROLL * NT * VEC) {
        Pack<S, VEC> p[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) p[u] = *reinterpret_cast<const Pack<S, VEC> *>(g + i + u * NT * VEC);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            Pack<D, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = (D)((float)p[u].v[j] * coef);
            store_streamed(out + i + u * NT * VEC, o);
        }
    }
    for (; i < n; i += NT * VEC) {
        const int left = n - i < VEC ? n - i : VEC;
        for (int j = 0; j < left; ++j) out[i + j] = (D)((float)g[i + j] * coef);
    }
}

template <typename S> __device__ __forceinline__ void scale_to(const S *g, void *out, int dt, long long at, int n, float coef) {
    if (dt == PSVAE_F32) scale(g + at, (float *)out + at, n, coef);
    else if (dt == PSVAE_BF16) scale(g + at, (__bf16 *)out + at, n, coef);
    else scale(g + at, (_Float16 *)out + at, n, coef);
}

// The chunks are taken from the list's end: what the norm read last is what the last-level cache still holds.  Measured: 300 M elements in
// two types, into float32, 557 us with the norm (2.65 GB of traffic at 4.7 TB/s, what a large copy reaches).  Ordinary stores: 565 us.
__global__ __launch_bounds__(NT) void clip_grads_kernel(ClipList l, const double *__restrict__ partial, int n_partial, double max_norm,
                                                        float *__restrict__ norm) {
    __shared__ double sh[NT / 64];
    const double v = sqrt(total_of(partial, n_partial, sh));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    const double q = max_norm / (v + 1e-6);
    const float coef = q > 1. ? 1.f : (float)q;   // (a NaN stays one, as torch.clamp keeps it)
    for (int c = l.first[l.n] - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x)
        with_chunk(l, c, [&](int i, int st, int dt, long long at, int n) {
            if (coef == 1.f && l.src[i] == l.dst[i] && st == dt) return;
            if (st == PSVAE_F32) scale_to((const float *)l.src[i], l.dst[i], dt, at, n, coef);
            else if (st == PSVAE_BF16) scale_to((const __bf16 *)l.src[i], l.dst[i], dt, at, n, coef);
            else scale_to((const _Float16 *)l.src[i], l.dst[i], dt, at, n, coef);
        });
}

// ---- host
int type_size(int t) { return t == PSVAE_F32 ? 4 : 2; }

int check_list(const char *fn, int n, const void *const *grads, const int64_t *numel, const int32_t *types) {
    PSVAE_REQUIRE(n >= 0, PSVAE_EINVAL, "%s: %d tensors", fn, n);
    PSVAE_REQUIRE(n == 0 || (grads && numel && types), PSVAE_EINVAL, "%s: null list", fn);
    PSVAE_REQUIRE(n <= (1 << 20), PSVAE_ETOOLARGE, "%s: %d tensors (at most 2^20)", fn, n);
    long long total = 0;             // (at most 2^40 elements: 2^26 chunks)
    for (int i = 0; i < n; ++i) {
        PSVAE_REQUIRE(numel[i] >= 0 && numel[i] <= (1ll << 40) && (total += numel[i]) <= (1ll << 40), PSVAE_EINVAL, "%s: tensor %d has %lld elements", fn, i, (long long)numel[i]);
        PSVAE_REQUIRE(types[i] == PSVAE_F32 || types[i] == PSVAE_BF16 || types[i] == PSVAE_F16, PSVAE_EINVAL, "%s: tensor %d is of an unknown type %d",
                      fn, i, (int)types[i]);
        PSVAE_REQUIRE(numel[i] == 0 || (grads[i] != nullptr && ((uintptr_t)grads[i] & (type_size(types[i]) - 1)) == 0), PSVAE_EINVAL,
                      "%s: tensor %d is null or misaligned", fn, i);
    }
    return PSVAE_OK;
}

// Whether an output shares memory with another output, or with a gradient other than the one that it is.
bool overlaps(int n, const void *const *grads, const int64_t *numel, const int32_t *types, void *const *out, const int32_t *out_types) {
    // slices of one buffer in their order, the gradients elsewhere: no sorting
    uintptr_t low = 0, high = 0;
    bool simple = true;
    for (int i = 0; i < n && simple; ++i) {
        if (numel[i] == 0) continue;
        const uintptr_t o = (uintptr_t)out[i];
        if (high == 0) low = o;
        simple = o >= high, high = o + (uintptr_t)numel[i] * type_size(out_types[i]);
    }
    for (int i = 0; i < n && simple; ++i) {
        const uintptr_t g = (uintptr_t)grads[i];
        simple = numel[i] == 0 || g >= high || g + (uintptr_t)numel[i] * type_size(types[i]) <= low;
    }
    if (simple) return false;
    struct Range {
        uintptr_t begin, end;
        bool out;
    };
    std::vector<Range> all;
    all.reserve(2 * (size_t)n);
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        const uintptr_t o = (uintptr_t)out[i], g = (uintptr_t)grads[i];
        all.push_back({o, o + (uintptr_t)numel[i] * type_size(out_types[i]), true});
        if (o != g || types[i] != out_types[i]) all.push_back({g, g + (uintptr_t)numel[i] * type_size(types[i]), false});
    }
    std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    uintptr_t end = 0, end_out = 0;     // of the ranges so far, of the outputs among them
    for (const Range &r : all) {
        if (r.begin < (r.out ? end : end_out)) return true;
        end = std::max(end, r.end);
        if (r.out) end_out = std::max(end_out, r.end);
    }
    return false;
}

int chunk_of(int n, const int64_t *numel, const int32_t *types) {
    long long bytes = 0;
    for (int i = 0; i < n; ++i) bytes += numel[i] * type_size(types[i]);
    return bytes >= LARGE ? CHUNK_LARGE : CHUNK_SMALL;
}

// Tensors [at, n) into a launch's part, as many that hold anything as it has room for.  Returns where the next part begins.
template <typename L>
int fill(L *l, int at, int n, const void *const *grads, const int64_t *numel, const int32_t *types, void *const *out, const int32_t *out_types, int chunk) {
    l->n = 0, l->chunk = chunk, l->first[0] = 0;
    for (; at < n && l->n < L::ROOM; ++at) {
        if (numel[at] == 0) continue;
        const long long each = chunk / type_size(types[at]), chunks = (numel[at] + each - 1) / each;
        const int k = l->n;
        l->src[k] = grads[at];
        if (out) l->dst[k] = out[at];
        l->size[k] = (unsigned long long)numel[at] | (unsigned long long)types[at] << 60 | (unsigned long long)(out_types ? out_types[at] : 0) << 62;
        l->first[k + 1] = l->first[k] + (int)chunks;
        l->n = k + 1;
    }
    return at;
}
template <typename L> int groups(const L &l) { return std::min(l.first[l.n], GROUPS); }

// the launches that a norm's list takes at most, each with its partial sums
int norm_parts(int n) { return (n + NormList::ROOM - 1) / NormList::ROOM; }

// the partial sums of squares of the whole list; *n_partial: how many
int squares(const char *fn, int n, const void *const *grads, const int64_t *numel, const int32_t *types, double *partial, int *n_partial, hipStream_t st) {
    NormList l;
    const int chunk = chunk_of(n, numel, types);
    *n_partial = 0;
    for (int at = 0; at < n;) {
        at = fill(&l, at, n, grads, numel, types, nullptr, nullptr, chunk);
        if (l.n == 0) break;
        hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)groups(l)), dim3(NT), 0, st, l, partial + *n_partial);
        PSVAE_CHECK_LAUNCH(fn);
        *n_partial += groups(l);
    }
    return PSVAE_OK;
}

}  // namespace

extern "C" size_t psvae_grad_norm_workspace_bytes(int n) { return n <= 0 ? 0 : (size_t)norm_parts(n) * GROUPS * sizeof(double); }

extern "C" int psvae_grad_norm(int n, const void *const *grads_host, const int64_t *numel_host, const int32_t *types_host, float *norm,
                               void *workspace, size_t workspace_bytes, void *stream) {
    const char *fn = "psvae_grad_norm";
    if (int rc = check_list(fn, n, grads_host, numel_host, types_host)) return rc;
    PSVAE_REQUIRE(norm != nullptr, PSVAE_EINVAL, "%s: null norm", fn);
    PSVAE_REQUIRE(n == 0 || (workspace != nullptr && workspace_bytes >= psvae_grad_norm_workspace_bytes(n) && psvae_aligned16(workspace)),
                  PSVAE_EWORKSPACE, "%s: workspace too small or not 16-byte aligned", fn);
    hipStream_t st = (hipStream_t)stream;
    int n_partial = 0;
    if (int rc = squares(fn, n, grads_host, numel_host, types_host, (double *)workspace, &n_partial, st)) return rc;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(NT), 0, st, (const double *)workspace, n_partial, norm);
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" int psvae_clip_grads(int n, const void *const *grads_host, const int64_t *numel_host, const int32_t *types_host,
                                void *const *out_host, const int32_t *out_types_host, double max_norm, float *norm, void *workspace,
                                size_t workspace_bytes, void *stream) {
    const char *fn = "psvae_clip_grads";
    if (int rc = check_list(fn, n, grads_host, numel_host, types_host)) return rc;
    if (int rc = check_list(fn, n, (const void *const *)out_host, numel_host, out_types_host)) return rc;
    PSVAE_REQUIRE(norm != nullptr, PSVAE_EINVAL, "%s: null norm", fn);
    PSVAE_REQUIRE(max_norm >= 0., PSVAE_EINVAL, "%s: max_norm must not be negative", fn);
    bool shared = false;
    try {
        shared = overlaps(n, grads_host, numel_host, types_host, out_host, out_types_host);
    } catch (...) {   // (host memory for the check ran out: no C++ exception leaves a C entry point)
        PSVAE_REQUIRE(false, PSVAE_ETOOLARGE, "%s: out of host memory", fn);
    }
    PSVAE_REQUIRE(!shared, PSVAE_EINVAL, "%s: an output overlaps another output, or a gradient that it is not", fn);
    PSVAE_REQUIRE(n == 0 || (workspace != nullptr && workspace_bytes >= psvae_grad_norm_workspace_bytes(n) && psvae_aligned16(workspace)),
                  PSVAE_EWORKSPACE, "%s: workspace too small or not 16-byte aligned", fn);
    hipStream_t st = (hipStream_t)stream;
    const double *partial = (const double *)workspace;
    int n_partial = 0;
    if (int rc = squares(fn, n, grads_host, numel_host, types_host, (double *)workspace, &n_partial, st)) return rc;
    if (n_partial == 0) {            // no elements
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(NT), 0, st, partial, 0, norm);
        PSVAE_CHECK_LAUNCH(fn);
        return PSVAE_OK;
    }
    if (n_partial > FOLD) {
        hipLaunchKernelGGL(grad_total_kernel, dim3(1), dim3(NT), 0, st, (double *)workspace, n_partial);
        PSVAE_CHECK_LAUNCH(fn);
        n_partial = 1;
    }
    // the parts of the list from its end, for the same reason as the chunks
    const int chunk = chunk_of(n, numel_host, types_host);
    for (int end = n; end > 0;) {
        int begin = end, held = 0;
        while (begin > 0 && held < ClipList::ROOM) held += numel_host[--begin] > 0;
        ClipList l;
        fill(&l, begin, end, grads_host, numel_host, types_host, out_host, out_types_host, chunk);
        end = begin;
        if (l.n == 0) continue;
        hipLaunchKernelGGL(clip_grads_kernel, dim3((unsigned)groups(l)), dim3(NT), 0, st, l, partial, n_partial, max_norm, norm);
        PSVAE_CHECK_LAUNCH(fn);
    }
    return PSVAE_OK;
}
