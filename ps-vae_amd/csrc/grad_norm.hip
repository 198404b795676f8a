// The 2-norm over a list of gradient tensors of several types, and the list scaled to a largest norm.
//
//     norm = sqrt(sum_i sum_j g_ij^2);   out_ij = g_ij * min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM at large sizes (one read for the norm, one read and one write for the scaling), by launches at small ones.  The list
// travels as kernel arguments (up to LIST tensors a launch), so nothing is copied to the device, nothing outlives the call and a captured
// graph holds its own copy.  Every tensor is cut into chunks of one size; a workgroup takes one chunk.  Squares are
// formed and added in 64 bits: a float's square neither overflows nor vanishes there, and the card does a 64-bit multiply-add
// at the rate of a 32-bit one, so the sum stays under the time of the loads.
#include "common.h"

#include <algorithm>
#include <math.h>
#include <vector>

namespace {

constexpr int NT = 256;
constexpr int LIST = 120;                       // tensors per launch: 30 bytes each of the 4 KB that kernel arguments may take
constexpr long long CHUNK_MIN = 4096;           // elements per workgroup: 16 per thread
constexpr int PARTIALS = 2048;                  // workgroups that a large list is cut into (8 per compute unit)

struct List {
    const void *src[LIST];
    void *dst[LIST];
    long long numel[LIST];
    int first[LIST + 1];                        // first chunk of each tensor, counted from the launch's first; [n]: chunks in all
    uint8_t st[LIST], dt[LIST];
    int n;
    long long chunk;
};

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

// the tensor that chunk `c` of the launch belongs to
__device__ __forceinline__ int tensor_of(const List &l, int c) {
    int lo = 0, hi = l.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T> __device__ __forceinline__ double sum_squares(const T *g, long long n) {
    constexpr int VEC = Elem<T>::VEC, UNROLL = 4;
    double acc[UNROLL] = {0., 0., 0., 0.};
    long long i = (long long)threadIdx.x * VEC;
    for (; i + (long long)(UNROLL - 1) * NT * VEC + VEC <= n; i += (long long)UNROLL * NT * VEC) {
        Pack<T, VEC> p[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) p[u] = *reinterpret_cast<const Pack<T, VEC> *>(g + i + (long long)u * NT * VEC);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const double d = (double)(float)p[u].v[j];
                acc[u] = fma(d, d, acc[u]);
            }
    }
    for (; i < n; i += (long long)NT * VEC) {
        const int left = n - i < VEC ? (int)(n - i) : VEC;
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

__global__ __launch_bounds__(NT) void grad_squares_kernel(List l, double *__restrict__ partial) {
    __shared__ double sh[NT / 64];
    const int c = blockIdx.x, i = tensor_of(l, c);
    const long long at = (long long)(c - l.first[i]) * l.chunk, n = l.numel[i] - at < l.chunk ? l.numel[i] - at : l.chunk;
    double s;
    if (l.st[i] == PSVAE_F32) s = sum_squares((const float *)l.src[i] + at, n);
    else if (l.st[i] == PSVAE_BF16) s = sum_squares((const __bf16 *)l.src[i] + at, n);
    else s = sum_squares((const _Float16 *)l.src[i] + at, n);
    s = block_sum(s, sh);
    if (threadIdx.x == 0) partial[c] = s;
}

// The sum of all partials in one fixed order, the same in every workgroup that forms it.
__device__ __forceinline__ double total_of(const double *__restrict__ partial, int n, double *sh) {
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

template <typename S, typename D> __device__ __forceinline__ void scale(const S *g, D *out, long long n, float coef) {
    constexpr int VEC = Elem<S>::VEC, UNROLL = 4;
    long long i = (long long)threadIdx.x * VEC;
    for (; i + (long long)(UNROLL - 1) * NT * VEC + VEC <= n; i += (long long)UNROLL * NT * VEC) {
        Pack<S, VEC> p[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) p[u] = *reinterpret_cast<const Pack<S, VEC> *>(g + i + (long long)u * NT * VEC);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            Pack<D, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = (D)((float)p[u].v[j] * coef);
            *reinterpret_cast<Pack<D, VEC> *>(out + i + (long long)u * NT * VEC) = o;
        }
    }
    for (; i < n; i += (long long)NT * VEC) {
        const int left = n - i < VEC ? (int)(n - i) : VEC;
        for (int j = 0; j < left; ++j) out[i + j] = (D)((float)g[i + j] * coef);
    }
}

template <typename S> __device__ __forceinline__ void scale_to(const S *g, void *out, int dt, long long at, long long n, float coef) {
    if (dt == PSVAE_F32) scale(g + at, (float *)out + at, n, coef);
    else if (dt == PSVAE_BF16) scale(g + at, (__bf16 *)out + at, n, coef);
    else scale(g + at, (_Float16 *)out + at, n, coef);
}

// The chunks are taken from the list's end: what the norm read last is what the last-level cache still holds.
__global__ __launch_bounds__(NT) void clip_grads_kernel(List l, const double *__restrict__ partial, int n_partial, float max_norm,
                                                        float *__restrict__ norm) {
    __shared__ double sh[NT / 64];
    const double v = sqrt(total_of(partial, n_partial, sh));
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    const double q = (double)max_norm / (v + 1e-6);
    const float coef = q > 1. ? 1.f : (float)q;   // (a NaN stays one, as torch.clamp keeps it)
    const int c = (int)gridDim.x - 1 - (int)blockIdx.x;
    const int i = tensor_of(l, c);
    if (coef == 1.f && l.src[i] == l.dst[i] && l.st[i] == l.dt[i]) return;
    const long long at = (long long)(c - l.first[i]) * l.chunk, n = l.numel[i] - at < l.chunk ? l.numel[i] - at : l.chunk;
    if (l.st[i] == PSVAE_F32) scale_to((const float *)l.src[i], l.dst[i], l.dt[i], at, n, coef);
    else if (l.st[i] == PSVAE_BF16) scale_to((const __bf16 *)l.src[i], l.dst[i], l.dt[i], at, n, coef);
    else scale_to((const _Float16 *)l.src[i], l.dst[i], l.dt[i], at, n, coef);
}

// ---- host
// How a list is cut: the chunk length (a multiple of 64 elements) and the chunks.
struct Cut {
    long long chunk, chunks;
};
Cut cut_of(int n, const int64_t *numel) {
    long long total = 0;
    for (int i = 0; i < n; ++i) total += numel[i];
    Cut c;
    c.chunk = std::max(CHUNK_MIN, ((total + PARTIALS - 1) / PARTIALS + 63) / 64 * 64);
    c.chunks = 0;
    for (int i = 0; i < n; ++i) c.chunks += (numel[i] + c.chunk - 1) / c.chunk;
    return c;
}

int type_size(int t) { return t == PSVAE_F32 ? 4 : 2; }

int check_list(const char *fn, int n, const void *const *grads, const int64_t *numel, const int32_t *types) {
    PSVAE_REQUIRE(n >= 0, PSVAE_EINVAL, "%s: %d tensors", fn, n);
    PSVAE_REQUIRE(n == 0 || (grads && numel && types), PSVAE_EINVAL, "%s: null list", fn);
    PSVAE_REQUIRE(n <= (1 << 20), PSVAE_ETOOLARGE, "%s: %d tensors (at most 2^20)", fn, n);
    for (int i = 0; i < n; ++i) {
        PSVAE_REQUIRE(numel[i] >= 0 && numel[i] < (1ll << 40), PSVAE_EINVAL, "%s: tensor %d has %lld elements", fn, i, (long long)numel[i]);
        PSVAE_REQUIRE(types[i] == PSVAE_F32 || types[i] == PSVAE_BF16 || types[i] == PSVAE_F16, PSVAE_EINVAL, "%s: tensor %d is of an unknown type %d",
                      fn, i, (int)types[i]);
        PSVAE_REQUIRE(numel[i] == 0 || (grads[i] != nullptr && ((uintptr_t)grads[i] & (type_size(types[i]) - 1)) == 0), PSVAE_EINVAL,
                      "%s: tensor %d is null or misaligned", fn, i);
    }
    return PSVAE_OK;
}

// Whether an output shares memory with another output, or with a gradient other than the one that it is.
bool overlaps(int n, const void *const *grads, const int64_t *numel, const int32_t *types, void *const *out, const int32_t *out_types) {
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

// The list's next part for one launch: tensors [at, ...), at most LIST that hold anything.  Returns where the next part begins.
int fill(List *l, int at, int n, const void *const *grads, const int64_t *numel, const int32_t *types, void *const *out, const int32_t *out_types,
         long long chunk) {
    l->n = 0, l->chunk = chunk, l->first[0] = 0;
    for (; at < n && l->n < LIST; ++at) {
        if (numel[at] == 0) continue;
        const int k = l->n;
        l->src[k] = grads[at], l->dst[k] = out ? out[at] : nullptr, l->numel[k] = numel[at];
        l->st[k] = (uint8_t)types[at], l->dt[k] = out_types ? (uint8_t)out_types[at] : 0;
        l->first[k + 1] = l->first[k] + (int)((numel[at] + chunk - 1) / chunk);
        l->n = k + 1;
    }
    return at;
}

// the partial sums of squares of the whole list
int squares(const char *fn, int n, const void *const *grads, const int64_t *numel, const int32_t *types, const Cut &cut, double *partial, hipStream_t st) {
    List l;
    long long base = 0;
    for (int at = 0; at < n;) {
        at = fill(&l, at, n, grads, numel, types, nullptr, nullptr, cut.chunk);
        if (l.n == 0) break;
        hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)l.first[l.n]), dim3(NT), 0, st, l, partial + base);
        PSVAE_CHECK_LAUNCH(fn);
        base += l.first[l.n];
    }
    return PSVAE_OK;
}

}  // namespace

extern "C" size_t psvae_grad_norm_workspace_bytes(int n, const int64_t *numel_host) {
    if (n <= 0 || numel_host == nullptr) return 0;
    return (size_t)cut_of(n, numel_host).chunks * sizeof(double);
}

extern "C" int psvae_grad_norm(int n, const void *const *grads_host, const int64_t *numel_host, const int32_t *types_host, float *norm,
                               void *workspace, size_t workspace_bytes, void *stream) {
    const char *fn = "psvae_grad_norm";
    if (int rc = check_list(fn, n, grads_host, numel_host, types_host)) return rc;
    PSVAE_REQUIRE(norm != nullptr, PSVAE_EINVAL, "%s: null norm", fn);
    const Cut cut = cut_of(n, numel_host);
    PSVAE_REQUIRE(cut.chunks == 0 || (workspace != nullptr && workspace_bytes >= (size_t)cut.chunks * sizeof(double) && psvae_aligned16(workspace)),
                  PSVAE_EWORKSPACE, "%s: workspace too small or not 16-byte aligned", fn);
    hipStream_t st = (hipStream_t)stream;
    if (int rc = squares(fn, n, grads_host, numel_host, types_host, cut, (double *)workspace, st)) return rc;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(NT), 0, st, (const double *)workspace, (int)cut.chunks, norm);
    PSVAE_CHECK_LAUNCH(fn);
    return PSVAE_OK;
}

extern "C" int psvae_clip_grads(int n, const void *const *grads_host, const int64_t *numel_host, const int32_t *types_host,
                                void *const *out_host, const int32_t *out_types_host, float max_norm, float *norm, void *workspace,
                                size_t workspace_bytes, void *stream) {
    const char *fn = "psvae_clip_grads";
    if (int rc = check_list(fn, n, grads_host, numel_host, types_host)) return rc;
    if (int rc = check_list(fn, n, (const void *const *)out_host, numel_host, out_types_host)) return rc;
    PSVAE_REQUIRE(norm != nullptr, PSVAE_EINVAL, "%s: null norm", fn);
    PSVAE_REQUIRE(max_norm >= 0.f, PSVAE_EINVAL, "%s: max_norm must not be negative", fn);
    bool shared = false;
    try {
        shared = overlaps(n, grads_host, numel_host, types_host, out_host, out_types_host);
    } catch (...) {   // (host memory for the check ran out: no C++ exception leaves a C entry point)
        PSVAE_REQUIRE(false, PSVAE_ETOOLARGE, "%s: out of host memory", fn);
    }
    PSVAE_REQUIRE(!shared, PSVAE_EINVAL, "%s: an output overlaps another output, or a gradient that it is not", fn);
    const Cut cut = cut_of(n, numel_host);
    PSVAE_REQUIRE(cut.chunks == 0 || (workspace != nullptr && workspace_bytes >= (size_t)cut.chunks * sizeof(double) && psvae_aligned16(workspace)),
                  PSVAE_EWORKSPACE, "%s: workspace too small or not 16-byte aligned", fn);
    hipStream_t st = (hipStream_t)stream;
    const double *partial = (const double *)workspace;
    if (int rc = squares(fn, n, grads_host, numel_host, types_host, cut, (double *)workspace, st)) return rc;
    if (cut.chunks == 0) {
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(NT), 0, st, partial, 0, norm);
        PSVAE_CHECK_LAUNCH(fn);
        return PSVAE_OK;
    }
    // the parts of the list in reverse, for the same reason as the chunks
    for (int end = n; end > 0;) {
        int begin = end, held = 0;
        while (begin > 0 && held < LIST) held += numel_host[--begin] > 0;
        List l;
        fill(&l, begin, end, grads_host, numel_host, types_host, out_host, out_types_host, cut.chunk);
        end = begin;
        if (l.n == 0) continue;
        hipLaunchKernelGGL(clip_grads_kernel, dim3((unsigned)l.first[l.n]), dim3(NT), 0, st, l, partial, (int)cut.chunks, max_norm, norm);
        PSVAE_CHECK_LAUNCH(fn);
    }
    return PSVAE_OK;
}
