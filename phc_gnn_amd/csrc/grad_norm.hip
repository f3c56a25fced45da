// The norm over many tensors together, and the tensors scaled to a bound (fp32 / bf16 / fp16, mixed):
//
//   n = (sum g^2)^(1/2) | sum |g| | max |g|         c = min(1, max_norm / (n + 1e-6))         out = c g
//
// One read of everything for the norm; where something is to be written, a second read (from the Infinity Cache when the tensors fit
// it) and one write.  In place with c = 1 nothing is written and the second pass ends at once.  Squares are summed in fp64: an fp32
// square overflows for |g| > 1.8e19, and the conversion + fma per element hide behind the loads.  Every workgroup sums a fixed set of
// chunks into its own partial, partials are added in a fixed order: the result does not depend on timing.
//
// 536 M fp32 into other fp32 tensors: 371 us for the norm (5.8 TB/s), 831 for the scaling (5.2 TB/s read and written).
// Tensors come by kernel argument, GN_MAX_TENSORS per launch: no table in memory that a captured graph would have to keep alive.
#include <algorithm>
#include <new>
#include <vector>

#include "dtype_io.h"

namespace phc {

constexpr int GN_THREADS = 256;
constexpr int GN_CHUNK = 8192;                // elements of one tensor
constexpr int GN_MAX_TENSORS = 128;
constexpr int GN_MAX_BLOCKS = 2048;           // 8 workgroups on each CU

struct GnTable {
    const void *g[GN_MAX_TENSORS];
    void *out[GN_MAX_TENSORS];
    long long numel[GN_MAX_TENSORS];
    int first_chunk[GN_MAX_TENSORS];          // chunks of the tensors in front
    unsigned char dtype[GN_MAX_TENSORS], out_dtype[GN_MAX_TENSORS];
    int n, chunks;
};

// tensor of a chunk: the last one whose first chunk is not behind it (two lane-wide compares instead of a search)
__device__ __forceinline__ int gn_tensor_of(const GnTable &t, int chunk) {
    const int lane = threadIdx.x & 63;
    const unsigned long long a = __ballot(lane < t.n && t.first_chunk[lane] <= chunk);
    const unsigned long long b = __ballot(lane + 64 < t.n && t.first_chunk[lane + 64 < GN_MAX_TENSORS ? lane + 64 : 0] <= chunk);
    return __builtin_amdgcn_readfirstlane(__popcll(a) + __popcll(b) - 1);
}

// elements at any element-aligned address: one 16-byte access (the hardware takes unaligned addresses)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[16 / sizeof(T)];
};

template <int KIND>
struct GnAcc {
    double s = 0.0;
    float m = 0.f;
    __device__ __forceinline__ void add(float x) {
        if constexpr (KIND == PHC_NORM_L2) {
            const double d = (double)x;
            s = fma(d, d, s);
        } else if constexpr (KIND == PHC_NORM_L1) {
            s += (double)fabsf(x);
        } else {
            const float a = fabsf(x);
            m = (a > m || a != a) ? a : m;          // (a NaN stays)
        }
    }
    __device__ __forceinline__ double value() const { return KIND == PHC_NORM_MAX ? (double)m : s; }
};
template <int KIND>
__device__ __forceinline__ double gn_join(double a, double b) {
    if constexpr (KIND == PHC_NORM_MAX) return (b > a || b != b) ? b : a;
    return a + b;
}

template <int KIND>
__device__ __forceinline__ double gn_block_join(double v, double *red) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = gn_join<KIND>(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) t = gn_join<KIND>(t, red[w]);
    return t;
}

template <int KIND, typename T>
__device__ __forceinline__ void gn_chunk(const T *__restrict__ g, int n, GnAcc<KIND> &acc) {
    constexpr int W = 16 / sizeof(T);
    int i = threadIdx.x * W;
    for (; i + W <= n; i += GN_THREADS * W) {
        const Loose<T> q = *reinterpret_cast<const Loose<T> *>(g + i);
#pragma unroll
        for (int k = 0; k < W; ++k) acc.add(to_f32(q.v[k]));
    }
    for (int k = i; k < n && k < i + W; ++k) acc.add(to_f32(g[k]));
}

template <int KIND>
__global__ __launch_bounds__(GN_THREADS) void grad_norm_partial_kernel(GnTable t, double *__restrict__ partial) {
    __shared__ double red[GN_THREADS / 64];
    GnAcc<KIND> acc;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = gn_tensor_of(t, c);
        const long long off = (long long)(c - t.first_chunk[i]) * GN_CHUNK;
        const int n = (int)min((long long)GN_CHUNK, t.numel[i] - off);
        const int dt = t.dtype[i];
        if (dt == PHC_DTYPE_F32) gn_chunk<KIND, float>(static_cast<const float *>(t.g[i]) + off, n, acc);
        else if (dt == PHC_DTYPE_BF16) gn_chunk<KIND, bf16_t>(static_cast<const bf16_t *>(t.g[i]) + off, n, acc);
        else gn_chunk<KIND, f16_t>(static_cast<const f16_t *>(t.g[i]) + off, n, acc);
    }
    const double v = gn_block_join<KIND>(acc.value(), red);
    if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

template <int KIND>
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double *__restrict__ partial, int n, double max_norm,
                                                               float *__restrict__ norm_coef) {
    __shared__ double red[16];
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) v = gn_join<KIND>(v, partial[i]);
    v = gn_block_join<KIND>(v, red);
    if (threadIdx.x == 0) {
        const double norm = KIND == PHC_NORM_L2 ? sqrt(v) : v;
        const double c = max_norm / (norm + 1e-6);
        norm_coef[0] = (float)norm;
        norm_coef[1] = c >= 1.0 ? 1.f : (float)c;            // (NaN stays NaN, as the gradients then are)
    }
}

// Accesses in flight per thread.  From 16-bit tensors 4 (157 us instead of 184 for 110 M bf16 gradients clipped into fp32 ones); from fp32 one:
// the 32 wavefronts of a CU already keep the memory busy, and more only spread its open pages (1 / 2 / 4 in flight: 1208 / 1224 / 1257 us for
// 536 M; the same holds for the norm's pass, 1208 / 1211 / 1244 us).
template <typename T>
constexpr int GN_AHEAD = sizeof(T) == 2 ? 4 : 1;

// W results at an element-aligned address, past the caches (nothing reads them soon, and the gradients still to be scaled lie there)
template <typename U, int W>
__device__ __forceinline__ void gn_store(U *p, const float (&v)[W]) {
    typedef U vec __attribute__((ext_vector_type(W), aligned(sizeof(U))));
    vec o;
#pragma unroll
    for (int k = 0; k < W; ++k) o[k] = from_f32<U>(v[k]);
    __builtin_nontemporal_store(o, reinterpret_cast<vec *>(p));
}

template <typename T, typename U>
__device__ __forceinline__ void gn_scale_chunk(const T *g, U *out, int n, float c) {
    constexpr int W = 16 / (sizeof(T) > sizeof(U) ? sizeof(T) : sizeof(U)), STEP = GN_THREADS * W, AHEAD = GN_AHEAD<T>;     // (16-byte accesses of the wider type)
    int i = threadIdx.x * W;
    for (; i + (AHEAD - 1) * STEP + W <= n; i += AHEAD * STEP) {
        LoosePack<T, W> q[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) q[a] = *reinterpret_cast<const LoosePack<T, W> *>(g + i + a * STEP);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            float v[W];
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = to_f32(q[a].v[k]) * c;
            gn_store<U, W>(out + i + a * STEP, v);
        }
    }
    for (; i + W <= n; i += STEP) {
        const LoosePack<T, W> q = *reinterpret_cast<const LoosePack<T, W> *>(g + i);
        float v[W];
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = to_f32(q.v[k]) * c;
        gn_store<U, W>(out + i, v);
    }
    for (int k = i; k < n && k < i + W; ++k) out[k] = from_f32<U>(to_f32(g[k]) * c);
}

template <typename T>
__device__ __forceinline__ void gn_scale_to(const void *g, void *out, int out_dtype, long long off, int n, float c) {
    const T *src = static_cast<const T *>(g) + off;
    if (out_dtype == PHC_DTYPE_F32) gn_scale_chunk<T, float>(src, static_cast<float *>(out) + off, n, c);
    else if (out_dtype == PHC_DTYPE_BF16) gn_scale_chunk<T, bf16_t>(src, static_cast<bf16_t *>(out) + off, n, c);
    else gn_scale_chunk<T, f16_t>(src, static_cast<f16_t *>(out) + off, n, c);
}

__global__ __launch_bounds__(GN_THREADS) void grad_scale_kernel(GnTable t, const float *__restrict__ norm_coef, int in_place) {
    const float c = norm_coef[1];
    if (in_place && c == 1.f) return;
    // from the end: what the norm read last is still in the Infinity Cache
    for (int k = t.chunks - 1 - (int)blockIdx.x; k >= 0; k -= gridDim.x) {
        const int i = gn_tensor_of(t, k);
        const long long off = (long long)(k - t.first_chunk[i]) * GN_CHUNK;
        const int n = (int)min((long long)GN_CHUNK, t.numel[i] - off);
        const int dt = t.dtype[i];
        if (dt == PHC_DTYPE_F32) gn_scale_to<float>(t.g[i], t.out[i], t.out_dtype[i], off, n, c);
        else if (dt == PHC_DTYPE_BF16) gn_scale_to<bf16_t>(t.g[i], t.out[i], t.out_dtype[i], off, n, c);
        else gn_scale_to<f16_t>(t.g[i], t.out[i], t.out_dtype[i], off, n, c);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
static int gn_fill(GnTable *t, int first, int n, const void *const *g, void *const *out, const int64_t *numel, const int32_t *dtype,
                   const int32_t *out_dtype) {
    t->n = 0;
    t->chunks = 0;
    int i = first;
    for (; i < n && t->n < GN_MAX_TENSORS; ++i) {
        if (numel[i] == 0) continue;
        const int64_t chunks = (numel[i] + GN_CHUNK - 1) / GN_CHUNK;
        if (t->chunks + chunks > (1 << 30)) break;                  // (chunk numbers stay in 32 bits)
        t->g[t->n] = g[i];
        t->out[t->n] = out ? out[i] : nullptr;
        t->numel[t->n] = numel[i];
        t->first_chunk[t->n] = t->chunks;
        t->dtype[t->n] = (unsigned char)dtype[i];
        t->out_dtype[t->n] = (unsigned char)(out_dtype ? out_dtype[i] : dtype[i]);
        t->chunks += (int)chunks;
        t->n += 1;
    }
    return i;
}
static unsigned gn_blocks(const GnTable &t) { return (unsigned)(t.chunks < GN_MAX_BLOCKS ? t.chunks : GN_MAX_BLOCKS); }

struct GnRange {
    uintptr_t lo, hi;
    int i;
};

// No element is written twice, and none that another tensor still reads is written (the launch orders nothing among its workgroups).
static int gn_check_overlap(const char *who, int n, const void *const *g, void *const *out, const int64_t *numel, const int32_t *dtype,
                            const int32_t *out_dtype) {
    try {
        std::vector<GnRange> w;
        w.reserve(n);
        for (int i = 0; i < n; ++i)
            if (numel[i] > 0) {
                const uintptr_t p = reinterpret_cast<uintptr_t>(out[i]);
                w.push_back({p, p + (uintptr_t)numel[i] * dtype_bytes(out_dtype[i]), i});
            }
        std::sort(w.begin(), w.end(), [](const GnRange &a, const GnRange &b) { return a.lo < b.lo; });
        for (size_t k = 1; k < w.size(); ++k)
            PHC_REQUIRE(w[k].lo >= w[k - 1].hi, PHC_ERR_INVALID_ARG, "%s: tensors %d and %d share memory that both would write", who, w[k - 1].i,
                        w[k].i);
        for (int i = 0; i < n; ++i) {
            if (numel[i] == 0) continue;
            const uintptr_t lo = reinterpret_cast<uintptr_t>(g[i]), hi = lo + (uintptr_t)numel[i] * dtype_bytes(dtype[i]);
            // the written ranges are disjoint and sorted: the first that ends behind lo, and on while they begin in front of hi
            auto it = std::upper_bound(w.begin(), w.end(), lo, [](uintptr_t v, const GnRange &r) { return v < r.hi; });
            for (; it != w.end() && it->lo < hi; ++it)
                PHC_REQUIRE(it->i == i && it->lo == lo && out_dtype[i] == dtype[i], PHC_ERR_INVALID_ARG,
                            "%s: tensor %d reads memory that result %d writes", who, i, it->i);
        }
    } catch (const std::bad_alloc &) {
        PHC_REQUIRE(false, PHC_ERR_INVALID_ARG, "%s: out of host memory", who);
    }
    return PHC_OK;
}

template <int KIND>
static void gn_launch_norm(int n, const void *const *g, const int64_t *numel, const int32_t *dtype, double max_norm, double *partial,
                           float *norm_coef, hipStream_t s) {
    GnTable t;
    int slots = 0;
    for (int i = 0; i < n;) {
        i = gn_fill(&t, i, n, g, nullptr, numel, dtype, nullptr);
        if (t.n == 0) continue;
        PHC_LAUNCH_AS(K_GRAD_NORM, (grad_norm_partial_kernel<KIND>), dim3(gn_blocks(t)), dim3(GN_THREADS), 0, s, t, partial + slots);
        slots += (int)gn_blocks(t);
    }
    PHC_LAUNCH_AS(K_GRAD_NORM, (grad_norm_finish_kernel<KIND>), dim3(1), dim3(1024), 0, s, (const double *)partial, slots, max_norm, norm_coef);
}

}  // namespace phc

using namespace phc;

extern "C" {

size_t phc_grad_norm_ws_bytes(int n, const int64_t *numel) {
    if (n < 0 || (n > 0 && !numel)) return 0;
    size_t slots = 0, in_group = 0;
    long long chunks = 0;
    for (int i = 0; i < n; ++i) {                 // as gn_fill cuts the list
        if (numel[i] <= 0) continue;
        const long long c = (numel[i] + GN_CHUNK - 1) / GN_CHUNK;
        if (in_group == (size_t)GN_MAX_TENSORS || chunks + c > (1 << 30)) {
            slots += (size_t)std::min<long long>(chunks, GN_MAX_BLOCKS);
            in_group = 0;
            chunks = 0;
        }
        chunks += c;
        ++in_group;
    }
    slots += (size_t)std::min<long long>(chunks, GN_MAX_BLOCKS);
    return (slots + 1) * sizeof(double);
}

int phc_grad_norm_clip(int n, const void *const *grads, const int64_t *numel, const int32_t *dtype, int norm_kind, double max_norm,
                       void *const *out, const int32_t *out_dtype, float *norm_coef, void *ws, size_t ws_bytes, void *stream) {
    PHC_REQUIRE(n >= 0 && (n == 0 || (grads && numel && dtype)) && norm_coef && (!out || out_dtype), PHC_ERR_INVALID_ARG,
                "phc_grad_norm_clip: null pointer or negative count");
    PHC_REQUIRE(norm_kind == PHC_NORM_L2 || norm_kind == PHC_NORM_L1 || norm_kind == PHC_NORM_MAX, PHC_ERR_INVALID_ARG,
                "phc_grad_norm_clip: unknown norm %d", norm_kind);
    PHC_REQUIRE(max_norm >= 0.0, PHC_ERR_INVALID_ARG, "phc_grad_norm_clip: max_norm %g", max_norm);
    bool in_place = out != nullptr;
    for (int i = 0; i < n; ++i) {
        PHC_REQUIRE(dtype_bytes(dtype[i]) && (!out || dtype_bytes(out_dtype[i])), PHC_ERR_INVALID_ARG, "phc_grad_norm_clip: tensor %d: unknown dtype", i);
        PHC_REQUIRE(numel[i] >= 0 && numel[i] <= (1ll << 40) && (numel[i] == 0 || (grads[i] && (!out || out[i]))), PHC_ERR_INVALID_ARG,
                    "phc_grad_norm_clip: tensor %d: null pointer or bad size", i);
        PHC_REQUIRE(numel[i] == 0 || (aligned_to(grads[i], dtype_bytes(dtype[i])) && (!out || aligned_to(out[i], dtype_bytes(out_dtype[i])))),
                    PHC_ERR_INVALID_ARG, "phc_grad_norm_clip: tensor %d: address not aligned to its element", i);
        if (out && numel[i] && (out[i] != grads[i] || out_dtype[i] != dtype[i])) in_place = false;
    }
    if (out)
        if (int rc = gn_check_overlap("phc_grad_norm_clip", n, grads, out, numel, dtype, out_dtype)) return rc;
    PHC_REQUIRE(ws && aligned_to(ws, 8) && ws_bytes >= phc_grad_norm_ws_bytes(n, numel), PHC_ERR_WORKSPACE,
                "phc_grad_norm_clip: workspace of %zu bytes, %zu needed", ws_bytes, phc_grad_norm_ws_bytes(n, numel));
    hipStream_t s = static_cast<hipStream_t>(stream);
    {
        double *partial = static_cast<double *>(ws);
        if (norm_kind == PHC_NORM_L2) gn_launch_norm<PHC_NORM_L2>(n, grads, numel, dtype, max_norm, partial, norm_coef, s);
        else if (norm_kind == PHC_NORM_L1) gn_launch_norm<PHC_NORM_L1>(n, grads, numel, dtype, max_norm, partial, norm_coef, s);
        else gn_launch_norm<PHC_NORM_MAX>(n, grads, numel, dtype, max_norm, partial, norm_coef, s);
    }
    if (out) {
        // the launches too go from the end
        GnTable t;
        for (int end = n; end > 0;) {
            int first = 0, next = 0;
            while (next < end) {
                first = next;
                next = gn_fill(&t, first, end, grads, out, numel, dtype, out_dtype);
            }
            if (t.n > 0)
                PHC_LAUNCH_AS(K_GRAD_SCALE, grad_scale_kernel, dim3(gn_blocks(t)), dim3(GN_THREADS), 0, s, t, (const float *)norm_coef, in_place ? 1 : 0);
            end = first;
        }
    }
    return launch_status("phc_grad_norm_clip");
}

}  // extern "C"
