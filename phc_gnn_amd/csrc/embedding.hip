// One embedding table of any size (fp32 / bf16 / fp16): lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale W[t_i]                       dW[v] = scale sum over i with t_i = v, v != pad, of dy[i]
//
// The lookup moves N rows in and N rows out.  The gradient writes all V rows once (rows no token names are zero), and reads dy once:
//   1. sort    the tokens with their positions, stable: equal tokens keep their order, so every sum below has ONE order of its terms,
//              whatever the launch's timing (no floating-point atomics anywhere);
//   2. chunks  of EB_CHUNK sorted positions: every lane group walks one chunk of one column slab with fp32 sums in registers; a run of
//              equal tokens that lies inside a chunk is finished there, a run that crosses a chunk's edge leaves a partial sum.  The
//              chunks are equal pieces of work however the tokens are distributed: one token may own half of all positions;
//   3. joins   the partial sums of a crossing run are added in order by the chunk it starts in.
#include "dtype_io.h"

namespace phc {

constexpr int EB_THREADS = 256;
constexpr int EB_CHUNK = 32;              // sorted positions per chunk
constexpr int EB_RADIX_BITS = 8;
constexpr int EB_BINS = 1 << EB_RADIX_BITS;
constexpr int EB_SORT_ITEMS = 8;          // keys per thread and sort tile
constexpr int EB_SORT_TILE = EB_THREADS * EB_SORT_ITEMS;

// ---- lookup ----------------------------------------------------------------------------------------------------------------------
// A lane group of 2^lg lanes owns a row and walks it in accesses of W elements.
template <typename T, int W>
__global__ __launch_bounds__(EB_THREADS) void embedding_fwd_kernel(const long long *__restrict__ tokens, const T *__restrict__ weight,
                                                                  long long N, long long V, long long ldw, int D, float scale, int lg,
                                                                  T *__restrict__ out, int *err) {
    const long long row = (((long long)blockIdx.x * EB_THREADS + threadIdx.x) >> lg);
    if (row >= N) return;
    const long long tok = checked_index(tokens[row], V, err, PHC_IDX_ERR_TOKEN);
    const T *src = weight + tok * ldw;
    T *dst = out + row * D;
    for (int c = (threadIdx.x & ((1 << lg) - 1)) * W; c < D; c += W << lg) {
        float v[W];
        load_pack<T, W>(src + c, v);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] *= scale;
        store_pack<T, W>(dst + c, v);
    }
}

// ---- stable radix sort of (token, position) -------------------------------------------------------------------------------------------
// One pass: tile histograms, one scan over [digit][tile], stable scatter.  Inside a tile a wavefront ranks its 64 keys by comparing
// digits with ballots (peers = lanes with the same digit); the wavefronts' counts are then added in order.
__global__ __launch_bounds__(EB_THREADS) void embedding_keys_kernel(const long long *__restrict__ tokens, long long N, long long V,
                                                                    int *__restrict__ keys, int *__restrict__ pos) {
    for (long long i = (long long)blockIdx.x * EB_THREADS + threadIdx.x; i < N; i += (long long)gridDim.x * EB_THREADS) {
        keys[i] = (int)safe_index(tokens[i], V);
        pos[i] = (int)i;
    }
}

__global__ __launch_bounds__(EB_THREADS) void embedding_hist_kernel(const int *__restrict__ keys, int N, int shift, int tiles,
                                                                   int *__restrict__ hist) {
    __shared__ int bins[EB_BINS];
    bins[threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * EB_SORT_TILE;
    for (int j = 0; j < EB_SORT_ITEMS; ++j) {
        const int i = base + j * EB_THREADS + threadIdx.x;
        if (i < N) atomicAdd(&bins[(keys[i] >> shift) & (EB_BINS - 1)], 1);
    }
    __syncthreads();
    hist[threadIdx.x * tiles + blockIdx.x] = bins[threadIdx.x];
}

// exclusive scan of n counts, in place, by one workgroup
__global__ __launch_bounds__(1024) void embedding_scan_kernel(int *__restrict__ a, int n) {
    __shared__ int wsum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int base = 0; base < n; base += 1024 * 4) {
        const int i0 = base + threadIdx.x * 4;
        int v[4], s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = i0 + j < n ? a[i0 + j] : 0;
            s += v[j];
        }
        int inc = s;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 63) wsum[wave] = inc;
        __syncthreads();
        int before = carry, total = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) before += wsum[w];
            total += wsum[w];
        }
        int run = before + inc - s;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j < n) a[i0 + j] = run;
            run += v[j];
        }
        carry += total;
        __syncthreads();
    }
}

__global__ __launch_bounds__(EB_THREADS) void embedding_scatter_kernel(const int *__restrict__ keys, const int *__restrict__ pos, int N,
                                                                      int shift, int tiles, const int *__restrict__ offs,
                                                                      int *__restrict__ keys_out, int *__restrict__ pos_out) {
    constexpr int WAVES = EB_THREADS / 64;
    __shared__ int wcount[WAVES][EB_BINS];       // keys of a digit met by each wavefront: then the wavefront's start in the output
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = lane; b < EB_BINS; b += 64) wcount[wave][b] = 0;
    __syncthreads();
    const int base = blockIdx.x * EB_SORT_TILE + wave * (64 * EB_SORT_ITEMS);      // a wavefront owns consecutive keys
    int digit[EB_SORT_ITEMS], rank[EB_SORT_ITEMS];
#pragma unroll
    for (int j = 0; j < EB_SORT_ITEMS; ++j) {
        const int i = base + j * 64 + lane;
        const bool in = i < N;
        digit[j] = in ? (keys[i] >> shift) & (EB_BINS - 1) : -1;
        unsigned long long peers = __ballot(in);
#pragma unroll
        for (int b = 0; b < EB_RADIX_BITS; ++b) {
            const unsigned long long m = __ballot((digit[j] >> b) & 1);
            peers &= ((digit[j] >> b) & 1) ? m : ~m;
        }
        const int below = __popcll(peers & ((1ull << lane) - 1));
        const int before = in ? wcount[wave][digit[j]] : 0;
        rank[j] = before + below;
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) wcount[wave][digit[j]] = before + __popcll(peers);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    {
        const int b = threadIdx.x;
        int run = offs[b * tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int c = wcount[w][b];
            wcount[w][b] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EB_SORT_ITEMS; ++j) {
        const int i = base + j * 64 + lane;
        if (i < N) {
            const int o = wcount[wave][digit[j]] + rank[j];
            keys_out[o] = keys[i];
            pos_out[o] = pos[i];
        }
    }
}

// ---- segmented sums ----------------------------------------------------------------------------------------------------------------
// Workgroups [0, chunk_blocks): lane groups over (chunk, column slab).  The others: 64 rows of the table each, zero where no token is.
template <typename T, int W>
__global__ __launch_bounds__(EB_THREADS) void embedding_bwd_kernel(const int *__restrict__ keys, const int *__restrict__ pos,
                                                                  const T *__restrict__ dy, long long ldy, int N, int V, int D, float scale,
                                                                  int pad, int lg, int chunk_blocks, T *__restrict__ dW,
                                                                  float *__restrict__ partial) {
    if ((int)blockIdx.x >= chunk_blocks) {
        // rows without a token: a search per lane for its row, then whole-row stores by the workgroup
        __shared__ int empty_rows[64];
        __shared__ int n_empty;
        const int row0 = ((int)blockIdx.x - chunk_blocks) * 64;
        if (threadIdx.x < 64) {
            const int r = row0 + threadIdx.x;
            int lo = 0, hi = N;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (keys[mid] < r) lo = mid + 1; else hi = mid;
            }
            const bool empty = r < V && (lo == N || keys[lo] != r || r == pad);
            const unsigned long long m = __ballot(empty);
            if (empty) empty_rows[__popcll(m & ((1ull << threadIdx.x) - 1))] = r;
            if (threadIdx.x == 0) n_empty = __popcll(m);
        }
        __syncthreads();
        float z[W] = {};
        for (int e = threadIdx.x >> 6; e < n_empty; e += EB_THREADS / 64) {
            T *dst = dW + (size_t)empty_rows[e] * D;
            for (int c = (threadIdx.x & 63) * W; c < D; c += 64 * W) store_pack<T, W>(dst + c, z);
        }
        return;
    }
    const int slab_cols = W << lg;
    const int slabs = (D + slab_cols - 1) / slab_cols;
    const long long group = ((long long)blockIdx.x * EB_THREADS + threadIdx.x) >> lg;
    const int chunk = (int)(group / slabs);
    const int col = (int)(group % slabs) * slab_cols + (threadIdx.x & ((1 << lg) - 1)) * W;
    const long long first = (long long)chunk * EB_CHUNK;
    if (first >= N || col >= D) return;
    const int begin = (int)first, end = min(begin + EB_CHUNK, N);
    float acc[W] = {};
    int key = keys[begin];
    bool from_before = begin > 0 && keys[begin - 1] == key;        // the run started in an earlier chunk
    for (int i = begin; i < end; ++i) {
        float v[W];
        load_pack<T, W>(dy + (long long)pos[i] * ldy + col, v);
#pragma unroll
        for (int q = 0; q < W; ++q) acc[q] += v[q];
        const int next = i + 1 < N ? keys[i + 1] : -1;
        if (next == key && i + 1 < end) continue;
        if (from_before || next == key) {
            // part of a crossing run: slot 0 = a run that came from before, slot 1 = one that starts here and goes on
            float *p = partial + ((size_t)chunk * 2 + (from_before ? 0 : 1)) * D + col;
#pragma unroll
            for (int q = 0; q < W; ++q) p[q] = acc[q];
        } else if (key != pad) {
#pragma unroll
            for (int q = 0; q < W; ++q) acc[q] *= scale;
            store_pack<T, W>(dW + (size_t)key * D + col, acc);
        }
#pragma unroll
        for (int q = 0; q < W; ++q) acc[q] = 0.f;
        from_before = false;
        key = next;
    }
}

// the crossing run that starts in a chunk: its parts in order
template <typename T, int W>
__global__ __launch_bounds__(EB_THREADS) void embedding_join_kernel(const int *__restrict__ keys, int N, int D, float scale, int pad, int lg,
                                                                   int chunks, const float *__restrict__ partial, T *__restrict__ dW) {
    const int slab_cols = W << lg;
    const int slabs = (D + slab_cols - 1) / slab_cols;
    const long long group = ((long long)blockIdx.x * EB_THREADS + threadIdx.x) >> lg;
    const int chunk = (int)(group / slabs);
    const int col = (int)(group % slabs) * slab_cols + (threadIdx.x & ((1 << lg) - 1)) * W;
    if (chunk + 1 >= chunks || col >= D) return;                     // (the last chunk's runs end in it)
    const int last = (chunk + 1) * EB_CHUNK - 1;
    const int key = keys[last];
    if (keys[last + 1] != key || key == pad) return;                 // no run crosses this chunk's end
    const int begin = chunk * EB_CHUNK;
    if (keys[begin] == key && begin > 0 && keys[begin - 1] == key) return;      // ... or it started in an earlier chunk
    float acc[W];
#pragma unroll
    for (int q = 0; q < W; ++q) acc[q] = partial[((size_t)chunk * 2 + 1) * D + col + q];
    for (int c = chunk + 1; c < chunks && keys[c * EB_CHUNK] == key; ++c) {
#pragma unroll
        for (int q = 0; q < W; ++q) acc[q] += partial[(size_t)c * 2 * D + col + q];
    }
#pragma unroll
    for (int q = 0; q < W; ++q) acc[q] *= scale;
    store_pack<T, W>(dW + (size_t)key * D + col, acc);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
struct EmbeddingWs {
    int *keys[2], *pos[2], *hist;
    float *partial;
    size_t bytes;
    EmbeddingWs(void *ws, long long N, int D) {
        Carve c(ws);
        const long long tiles = (N + EB_SORT_TILE - 1) / EB_SORT_TILE, chunks = (N + EB_CHUNK - 1) / EB_CHUNK;
        for (int i = 0; i < 2; ++i) {
            keys[i] = c.take<int>(N);
            pos[i] = c.take<int>(N);
        }
        hist = c.take<int>(tiles * EB_BINS);
        partial = c.take<float>((size_t)chunks * 2 * D);
        bytes = c.used;
    }
};

// lanes per row: the smallest power of two that covers a row in one go, at most a wavefront
static int lane_group(int D, int W) {
    int lg = 0;
    while (lg < 6 && (W << lg) < D) ++lg;
    return lg;
}

// widest access that row length, row stride and base addresses allow (bytes of one access: 16, 8, 4 or 2)
static int pack_width(int esize, long long D, long long ld, const void *a, const void *b) {
    for (int w = 16 / esize; w > 1; w >>= 1)
        if (D % w == 0 && ld % w == 0 && aligned_to(a, (size_t)w * esize) && aligned_to(b, (size_t)w * esize)) return w;
    return 1;
}

template <typename T, int W>
static void launch_fwd(const int64_t *tokens, const void *weight, int64_t N, int64_t V, int64_t ldw, int D, float scale, void *out,
                       hipStream_t s) {
    const int lg = lane_group(D, W);
    const long long blocks = ((N << lg) + EB_THREADS - 1) / EB_THREADS;
    PHC_LAUNCH_AS(K_EMBEDDING_FWD, (embedding_fwd_kernel<T, W>), dim3((unsigned)blocks), dim3(EB_THREADS), 0, s, reinterpret_cast<const long long *>(tokens),
               static_cast<const T *>(weight), (long long)N, (long long)V, (long long)ldw, D, scale, lg, static_cast<T *>(out), err_word());
}

template <typename T, int W>
static void launch_bwd(const EmbeddingWs &w, int side, const void *dy, int64_t N, int64_t V, int64_t ldy, int D, float scale, int pad,
                       void *dW, hipStream_t s) {
    const int lg = lane_group(D, W);
    const long long slabs = (D + (W << lg) - 1) / (W << lg), chunks = (N + EB_CHUNK - 1) / EB_CHUNK;
    const long long cb = (((chunks * slabs) << lg) + EB_THREADS - 1) / EB_THREADS, zb = (V + 63) / 64;
    PHC_LAUNCH_AS(K_EMBEDDING_BWD, (embedding_bwd_kernel<T, W>), dim3((unsigned)(cb + zb)), dim3(EB_THREADS), 0, s, (const int *)w.keys[side],
               (const int *)w.pos[side], static_cast<const T *>(dy), (long long)ldy, (int)N, (int)V, D, scale, pad, lg, (int)cb,
               static_cast<T *>(dW), w.partial);
    if (chunks > 1)
        PHC_LAUNCH_AS(K_EMBEDDING_BWD, (embedding_join_kernel<T, W>), dim3((unsigned)cb), dim3(EB_THREADS), 0, s, (const int *)w.keys[side], (int)N, D, scale, pad,
                   lg, (int)chunks, (const float *)w.partial, static_cast<T *>(dW));
}

}  // namespace phc

using namespace phc;

#define EB_DISPATCH(FN, dtype, width, ...)                                   \
    do {                                                                     \
        if ((dtype) == PHC_DTYPE_F32) {                                      \
            if ((width) == 4) FN<float, 4>(__VA_ARGS__);                     \
            else if ((width) == 2) FN<float, 2>(__VA_ARGS__);                \
            else FN<float, 1>(__VA_ARGS__);                                  \
        } else if ((dtype) == PHC_DTYPE_BF16) {                              \
            if ((width) == 8) FN<bf16_t, 8>(__VA_ARGS__);                    \
            else if ((width) == 4) FN<bf16_t, 4>(__VA_ARGS__);               \
            else if ((width) == 2) FN<bf16_t, 2>(__VA_ARGS__);               \
            else FN<bf16_t, 1>(__VA_ARGS__);                                 \
        } else {                                                             \
            if ((width) == 8) FN<f16_t, 8>(__VA_ARGS__);                     \
            else if ((width) == 4) FN<f16_t, 4>(__VA_ARGS__);                \
            else if ((width) == 2) FN<f16_t, 2>(__VA_ARGS__);                \
            else FN<f16_t, 1>(__VA_ARGS__);                                  \
        }                                                                    \
    } while (0)

static int embedding_check(const char *who, int64_t N, int64_t V, int64_t D, int64_t ld, int dtype) {
    PHC_REQUIRE(dtype_bytes(dtype) != 0, PHC_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
    PHC_REQUIRE(N >= 0 && V >= 1 && D >= 1, PHC_ERR_INVALID_ARG, "%s: N=%lld V=%lld D=%lld", who, (long long)N, (long long)V, (long long)D);
    PHC_REQUIRE(N <= (1ll << 28) && V <= (1ll << 30) && D <= (1ll << 20), PHC_ERR_UNSUPPORTED, "%s: N=%lld V=%lld D=%lld is beyond 2^28, 2^30, 2^20",
                who, (long long)N, (long long)V, (long long)D);
    PHC_REQUIRE(ld >= D || N <= 1 || V <= 1, PHC_ERR_INVALID_ARG, "%s: row stride %lld below the row length %lld", who, (long long)ld, (long long)D);
    return PHC_OK;
}

extern "C" {

int phc_embedding_fwd(const int64_t *tokens, const void *weight, int64_t N, int64_t V, int64_t D, int64_t ldw, int dtype, float scale,
                      void *out, void *stream) {
    if (int rc = embedding_check("phc_embedding_fwd", N, V, D, ldw, dtype)) return rc;
    if (N == 0) return PHC_OK;
    PHC_REQUIRE(tokens && weight && out, PHC_ERR_INVALID_ARG, "phc_embedding_fwd: null pointer");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int w = pack_width(dtype_bytes(dtype), D, ldw, weight, out);
    EB_DISPATCH(launch_fwd, dtype, w, tokens, weight, N, V, ldw, (int)D, scale, out, s);
    return launch_status("phc_embedding_fwd");
}

size_t phc_embedding_bwd_ws_bytes(int64_t N, int64_t V, int64_t D) {
    if (N < 0 || N > (1ll << 28) || V < 1 || V > (1ll << 30) || D < 1 || D > (1ll << 20)) return 0;
    return EmbeddingWs(nullptr, N, (int)D).bytes + 256;
}

int phc_embedding_bwd(const int64_t *tokens, const void *dy, int64_t N, int64_t V, int64_t D, int64_t ldy, int dtype, float scale,
                      int64_t padding_idx, void *dW, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = embedding_check("phc_embedding_bwd", N, V, D, ldy, dtype)) return rc;
    PHC_REQUIRE(dW && (N == 0 || (tokens && dy)), PHC_ERR_INVALID_ARG, "phc_embedding_bwd: null pointer");
    PHC_REQUIRE(ws && aligned_to(ws, 16) && ws_bytes >= phc_embedding_bwd_ws_bytes(N, V, D), PHC_ERR_WORKSPACE,
                "phc_embedding_bwd: workspace of %zu bytes, %zu needed", ws_bytes, phc_embedding_bwd_ws_bytes(N, V, D));
    hipStream_t s = static_cast<hipStream_t>(stream);
    EmbeddingWs w(ws, N, (int)D);
    const int pad = padding_idx >= 0 && padding_idx < V ? (int)padding_idx : -1;
    int side = 0;
    if (N > 0) {
        const int tiles = (int)((N + EB_SORT_TILE - 1) / EB_SORT_TILE);
        const unsigned kb = (unsigned)((N + EB_THREADS - 1) / EB_THREADS);
        PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_keys_kernel, dim3(kb < 4096 ? kb : 4096), dim3(EB_THREADS), 0, s, reinterpret_cast<const long long *>(tokens),
                   (long long)N, (long long)V, w.keys[0], w.pos[0]);
        int bits = 0;
        while ((1ll << bits) < V) ++bits;
        for (int shift = 0; shift < bits; shift += EB_RADIX_BITS, side ^= 1) {
            PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_hist_kernel, dim3(tiles), dim3(EB_THREADS), 0, s, (const int *)w.keys[side], (int)N, shift, tiles, w.hist);
            PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_scan_kernel, dim3(1), dim3(1024), 0, s, w.hist, tiles * EB_BINS);
            PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_scatter_kernel, dim3(tiles), dim3(EB_THREADS), 0, s, (const int *)w.keys[side], (const int *)w.pos[side],
                       (int)N, shift, tiles, (const int *)w.hist, w.keys[side ^ 1], w.pos[side ^ 1]);
        }
    }
    const int width = pack_width(dtype_bytes(dtype), D, ldy, dy ? dy : dW, dW);
    EB_DISPATCH(launch_bwd, dtype, width, w, side, dy, N, V, ldy, (int)D, scale, pad, dW, s);
    return launch_status("phc_embedding_bwd");
}

}  // extern "C"
