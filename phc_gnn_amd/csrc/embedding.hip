// One embedding table of any size (fp32 / bf16 / fp16): lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale W[t_i]                       dW[v] = scale sum over i with t_i = v, v != pad, of dy[i]
//
// The lookup moves N rows in and N rows out.  The gradient writes all V rows once (rows no token names are zero), and reads dy once:
//   1. sort    the tokens with their positions, stable: equal tokens keep their order, so every sum below has ONE order of its terms,
//              whatever the launch's timing (no floating-point atomics anywhere);
//   2. chunks  of EB_CHUNK sorted positions: every lane group walks one chunk of one column slab with fp32 sums in registers; a run of
//              equal tokens that lies inside a chunk is finished there, a run that crosses a chunk's edge leaves a partial sum.  The
//              chunks are equal pieces of work however the tokens are distributed; positions of the padding token are summed too, and not
//              stored;
//   3. joins   the partial sums of a crossing run are added in order by the chunk it starts in, a workgroup for each column slab.  This part
//              goes by the longest run: 131072 positions of 2048 bf16 columns 30 us with random tokens, 111 with half of the positions on
//              one token, 216 with all of them (lookup, sort and sums together 460, 420 and 370 us).
#include "dtype_io.h"

namespace phc {

constexpr int EB_THREADS = 256;
constexpr int EB_CHUNK = 32;              // sorted positions per chunk
constexpr int EB_RADIX_BITS = 9;           // (two passes up to 262144 rows)
constexpr int EB_BINS = 1 << EB_RADIX_BITS;
constexpr int EB_SORT_ITEMS = 8;          // keys per thread and sort tile
constexpr int EB_SORT_TILE = EB_THREADS * EB_SORT_ITEMS;

// ---- lookup ----------------------------------------------------------------------------------------------------------------------
// A lane group of 2^lg lanes owns a row and walks it in accesses of W elements: a copy with scattered reads.  131072 rows of 2048 bf16 from a
// table of as many: 155 - 171 us for 1.07 GB = 6.3 - 6.9 TB/s (rows met twice come from the caches).
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
// Digits of at most 9 bits, as many passes as the vocabulary's bits need.  A wavefront ranks its 64 keys by comparing digits with ballots
// (peers = lanes with the same digit); the counts of its earlier keys stand in LDS.  Up to EB_LDS_SORT positions one workgroup sorts in
// LDS, in one launch; beyond that every pass is tile histograms, one scan over [digit][tile] and a stable scatter.  All latency, by the keys a thread
// holds (2, 6 or 16: the fewest that take all positions) and the passes.  32003 rows, two passes: 2048 / 2049 positions 7.6 / 12.4 us, 6144 /
// 6145 14.9 / 25.8, 16384 / 16385 31.6 / 33 (the six launches; LDS ends at 160 KB).  119 rows, one pass: 13568 positions 16.4 us.  131072 positions 44 us.

// rank of this lane's key among the wavefront's keys of the same digit; `count` (this wavefront's, per digit) is moved on
__device__ __forceinline__ int eb_rank(int digit, bool in, int bits, int *count) {
    unsigned long long peers = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long m = __ballot((digit >> b) & 1);
        peers &= ((digit >> b) & 1) ? m : ~m;
    }
    const int below = __popcll(peers & ((1ull << (threadIdx.x & 63)) - 1));
    const int before = in ? count[digit] : 0;
    __builtin_amdgcn_wave_barrier();
    if (in && below == 0) count[digit] = before + __popcll(peers);
    __builtin_amdgcn_wave_barrier();
    return before + below;
}

// One workgroup, everything in LDS: a thread holds PER keys of its wavefront's consecutive 64 PER.
template <int PER>
__global__ __launch_bounds__(1024) void embedding_sort_lds_kernel(const long long *__restrict__ tokens, int N, long long V, int bits, int passes,
                                                                 int *__restrict__ keys_out, int *__restrict__ pos_out) {
    constexpr int WAVES = 16, CAP = 1024 * PER;
    extern __shared__ int smem[];
    int *lkeys = smem;                                            // [CAP]
    int(*count)[EB_BINS] = reinterpret_cast<int(*)[EB_BINS]>(smem + CAP);      // [WAVES]
    int *wsum = smem + CAP + WAVES * EB_BINS;                     // [WAVES]
    unsigned short *lpos = reinterpret_cast<unsigned short *>(wsum + WAVES);   // [CAP]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, base = wave * 64 * PER + lane;
    int key[PER], pos[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = base + j * 64;
        key[j] = i < N ? (int)safe_index(tokens[i], V) : 0;
        pos[j] = i;
    }
    const int width = (bits + passes - 1) / passes, mask = (1 << width) - 1;
    for (int p = 0; p < passes; ++p) {
        for (int b = lane; b < EB_BINS; b += 64) count[wave][b] = 0;
        int rank[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) rank[j] = eb_rank((key[j] >> (p * width)) & mask, base + j * 64 < N, width, count[wave]);
        __syncthreads();
        // exclusive starts: digits in order, the wavefronts of a digit in order (a thread has one digit: EB_BINS <= 1024)
        int total = 0;
        if (threadIdx.x < EB_BINS)
            for (int w = 0; w < WAVES; ++w) total += count[w][threadIdx.x];
        int inc = total;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 63) wsum[wave] = inc;
        __syncthreads();
        if (threadIdx.x < EB_BINS) {
            int run = inc - total;
            for (int w = 0; w < wave; ++w) run += wsum[w];
            for (int w = 0; w < WAVES; ++w) {
                const int c = count[w][threadIdx.x];
                count[w][threadIdx.x] = run;
                run += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (base + j * 64 >= N) continue;
            const int o = count[wave][(key[j] >> (p * width)) & mask] + rank[j];
            lkeys[o] = key[j];
            lpos[o] = (unsigned short)pos[j];
        }
        __syncthreads();
        if (p == passes - 1) break;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = base + j * 64;
            if (i < N) {
                key[j] = lkeys[i];
                pos[j] = lpos[i];
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < N; i += 1024) {
        keys_out[i] = lkeys[i];
        pos_out[i] = lpos[i];
    }
}

// The first pass reads the tokens themselves (keys == nullptr); positions are then the indices.
__device__ __forceinline__ int eb_key(const int *keys, const long long *tokens, long long V, int i) {
    return keys ? keys[i] : (int)safe_index(tokens[i], V);
}

__global__ __launch_bounds__(EB_THREADS) void embedding_hist_kernel(const int *__restrict__ keys, const long long *__restrict__ tokens, long long V,
                                                                   int N, int shift, int mask, int *__restrict__ hist) {
    __shared__ int bins[EB_BINS];
    for (int b = threadIdx.x; b < EB_BINS; b += EB_THREADS) bins[b] = 0;
    __syncthreads();
    const int base = blockIdx.x * EB_SORT_TILE;
#pragma unroll
    for (int j = 0; j < EB_SORT_ITEMS; ++j) {
        const int i = base + j * EB_THREADS + threadIdx.x;
        if (i < N) atomicAdd(&bins[(eb_key(keys, tokens, V, i) >> shift) & mask], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < EB_BINS; b += EB_THREADS) hist[(size_t)blockIdx.x * EB_BINS + b] = bins[b];
}

// hist [tile][digit] -> the first place of every (tile, digit) in the output: digits in order, the tiles of a digit in order.  One workgroup;
// 1024 / EB_BINS thread groups share the tiles.
__global__ __launch_bounds__(1024) void embedding_scan_kernel(int *__restrict__ hist, int tiles) {
    constexpr int GROUPS = 1024 / EB_BINS, AHEAD = 16;
    __shared__ int sums[GROUPS][EB_BINS], wsum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = threadIdx.x % EB_BINS, g = threadIdx.x / EB_BINS;
    const int each = (tiles + GROUPS - 1) / GROUPS, t0 = min(g * each, tiles), t1 = min(t0 + each, tiles);
    int mine = 0;
    for (int t = t0; t < t1; t += AHEAD) {
        int v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) v[q] = t + q < t1 ? hist[(size_t)(t + q) * EB_BINS + b] : 0;
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) mine += v[q];
    }
    sums[g][b] = mine;
    __syncthreads();
    int total = 0;
    if (g == 0)
        for (int k = 0; k < GROUPS; ++k) total += sums[k][b];
    int inc = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    if (g == 0) {
        int run = inc - total;
        for (int w = 0; w < wave; ++w) run += wsum[w];
        for (int k = 0; k < GROUPS; ++k) {
            const int c = sums[k][b];
            sums[k][b] = run;
            run += c;
        }
    }
    __syncthreads();
    int run = sums[g][b];
    for (int t = t0; t < t1; t += AHEAD) {
        int v[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) v[q] = t + q < t1 ? hist[(size_t)(t + q) * EB_BINS + b] : 0;
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (t + q < t1) hist[(size_t)(t + q) * EB_BINS + b] = run;
            run += v[q];
        }
    }
}

__global__ __launch_bounds__(EB_THREADS) void embedding_scatter_kernel(const int *__restrict__ keys, const long long *__restrict__ tokens, long long V,
                                                                      const int *__restrict__ pos, int N, int shift, int width,
                                                                      const int *__restrict__ offs, int *__restrict__ keys_out,
                                                                      int *__restrict__ pos_out) {
    constexpr int WAVES = EB_THREADS / 64;
    __shared__ int count[WAVES][EB_BINS];        // keys of a digit met by each wavefront: then the wavefront's start in the output
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mask = (1 << width) - 1;
    for (int b = lane; b < EB_BINS; b += 64) count[wave][b] = 0;
    const int base = blockIdx.x * EB_SORT_TILE + wave * (64 * EB_SORT_ITEMS) + lane;      // a wavefront owns consecutive keys
    int key[EB_SORT_ITEMS], at[EB_SORT_ITEMS], rank[EB_SORT_ITEMS];
#pragma unroll
    for (int j = 0; j < EB_SORT_ITEMS; ++j) {
        const int i = base + j * 64;
        key[j] = i < N ? eb_key(keys, tokens, V, i) : 0;
        at[j] = i < N && keys ? pos[i] : i;
    }
#pragma unroll
    for (int j = 0; j < EB_SORT_ITEMS; ++j) rank[j] = eb_rank((key[j] >> shift) & mask, base + j * 64 < N, width, count[wave]);
    __syncthreads();
    for (int b = threadIdx.x; b < EB_BINS; b += EB_THREADS) {
        int run = offs[(size_t)blockIdx.x * EB_BINS + b];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int c = count[w][b];
            count[w][b] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EB_SORT_ITEMS; ++j) {
        if (base + j * 64 >= N) continue;
        const int o = count[wave][(key[j] >> shift) & mask] + rank[j];
        keys_out[o] = key[j];
        pos_out[o] = at[j];
    }
}

// ---- segmented sums ----------------------------------------------------------------------------------------------------------------
// Workgroups [0, chunk_blocks): lane groups over (chunk, column slab).  The others: 64 rows of the table each, zero where no token is.  dy is
// read and dW written once: 131072 rows of 2048 bf16 into as many rows 207 - 216 us for 1.07 GB = 5 TB/s.  16-byte accesses although fewer
// wavefronts then share the work (236 us against 251 and 284 with 8 and 4 bytes, 50000 rows of 2048); chunks of 16 positions leave more
// crossing runs (268 us).
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
        for (int e = threadIdx.x >> 6; e < n_empty; e += EB_THREADS / 64) {
            T *dst = dW + (size_t)empty_rows[e] * D;
            for (int c = (threadIdx.x & 63) * W; c < D; c += 64 * W) store_zeros<T, W>(dst + c);
        }
        return;
    }
    // the chunk's keys and positions, one in front and one behind: by the group's lanes, for all of them
    extern __shared__ int staged[];                                // [groups of the workgroup][EB_CHUNK + 2 keys | EB_CHUNK positions]
    const int slab_cols = W << lg, lanes = 1 << lg, me = threadIdx.x & (lanes - 1);
    int *skeys = staged + (threadIdx.x >> lg) * (2 * EB_CHUNK + 2), *spos = skeys + EB_CHUNK + 2;
    const int slabs = (D + slab_cols - 1) / slab_cols;
    const long long group = ((long long)blockIdx.x * EB_THREADS + threadIdx.x) >> lg;
    const int chunk = (int)(group / slabs);
    const int col = (int)(group % slabs) * slab_cols + me * W;
    const long long first = (long long)chunk * EB_CHUNK;
    const int begin = (int)min(first, (long long)N), n = min(EB_CHUNK, N - begin);
    for (int i = me; i < EB_CHUNK + 2; i += lanes) {
        const int at = begin + i - 1;
        skeys[i] = at >= 0 && at < N ? keys[at] : -1;
        if (i < EB_CHUNK) spos[i] = begin + i < N ? pos[begin + i] : 0;
    }
    __syncthreads();
    if (n <= 0 || col >= D) return;
    float acc[W] = {};
    int key = skeys[1];
    bool from_before = skeys[0] == key;                         // the run started in an earlier chunk
    constexpr int AHEAD = 8;                                       // rows in flight
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
        Pack<T, W> row[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)                            // (behind the chunk's end: its last row again, not used)
            row[q] = *reinterpret_cast<const Pack<T, W> *>(dy + (long long)spos[min(i0 + q, n - 1)] * ldy + col);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (i0 + q >= n) break;
#pragma unroll
            for (int c = 0; c < W; ++c) acc[c] += to_f32(row[q].v[c]);
            const int next = skeys[i0 + q + 2];
            if (next == key && i0 + q + 1 < n) continue;
            if (from_before || next == key) {
                // part of a crossing run: slot 0 = a run that came from before, slot 1 = one that starts here and goes on
                store_pack<float, W>(partial + ((size_t)chunk * 2 + (from_before ? 0 : 1)) * D + col, acc);
            } else if (key != pad) {
#pragma unroll
                for (int c = 0; c < W; ++c) acc[c] *= scale;
                store_pack<T, W>(dW + (size_t)key * D + col, acc);
            }
#pragma unroll
            for (int c = 0; c < W; ++c) acc[c] = 0.f;
            from_before = false;
            key = next;
        }
    }
}

// The crossing runs that start in EB_JOIN neighbouring chunks: their parts in order.  A workgroup takes those chunks and a column slab; its
// lane groups share a run's parts (group g the g-th stretch of them) and their sums are added in order.  8 - 10 us with few long runs (119
// tokens, 13568 positions), 31 us with many short ones (131072 positions of 2048 columns).
constexpr int EB_JOIN = 4;
template <typename T, int W>
__global__ __launch_bounds__(EB_THREADS) void embedding_join_kernel(const int *__restrict__ keys, int N, int D, float scale, int pad, int lg,
                                                                   int chunks, int slabs, const float *__restrict__ partial, T *__restrict__ dW) {
    __shared__ float meet[EB_THREADS * W];
    const int first = (int)(blockIdx.x / slabs) * EB_JOIN, count = min(EB_JOIN, chunks - 1 - first);     // (the last chunk's runs end in it)
    const int lanes = 1 << lg, me = threadIdx.x & (lanes - 1), g = threadIdx.x >> lg, groups = EB_THREADS >> lg;
    const int col = (int)(blockIdx.x % slabs) * (W << lg) + me * W;
    // which of the chunks start a crossing run (the same answer in every wavefront)
    bool starts = false;
    if ((int)(threadIdx.x & 63) < count) {
        const int begin = (first + (threadIdx.x & 63)) * EB_CHUNK, key = keys[begin + EB_CHUNK - 1];
        starts = keys[begin + EB_CHUNK] == key && key != pad && !(keys[begin] == key && begin > 0 && keys[begin - 1] == key);
    }
    unsigned long long todo = __ballot(starts);
    for (; todo; todo &= todo - 1) {
        const int chunk = first + __builtin_ctzll(todo), last = (chunk + 1) * EB_CHUNK - 1, key = keys[last];
        int lo = last + 1, hi = N;                                   // the run's end
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (keys[mid] <= key) lo = mid + 1; else hi = mid;
        }
        const int parts = (lo - 1) / EB_CHUNK - chunk;               // in the chunks behind this one
        const int each = (parts + groups - 1) / groups, p0 = min(g * each, parts), p1 = min(p0 + each, parts);
        float acc[W] = {};
        if (col < D) {
            const float *src = partial + (size_t)(chunk + 1) * 2 * D + col;
            constexpr int AHEAD = 8;
            for (int p = p0; p < p1; p += AHEAD) {
                float v[AHEAD][W];
#pragma unroll
                for (int q = 0; q < AHEAD; ++q) load_pack<float, W>(src + (size_t)min(p + q, p1 - 1) * 2 * D, v[q]);
#pragma unroll
                for (int q = 0; q < AHEAD; ++q)
                    if (p + q < p1)
#pragma unroll
                        for (int c = 0; c < W; ++c) acc[c] += v[q][c];
            }
        }
        __syncthreads();                                             // (the run before has been read)
#pragma unroll
        for (int c = 0; c < W; ++c) meet[c * EB_THREADS + threadIdx.x] = acc[c];
        __syncthreads();
        if (g == 0 && col < D) {
            float sum[W];
            load_pack<float, W>(partial + ((size_t)chunk * 2 + 1) * D + col, sum);
            for (int k = 0; k < min(groups, parts); ++k)
#pragma unroll
                for (int c = 0; c < W; ++c) sum[c] += meet[c * EB_THREADS + k * lanes + me];
#pragma unroll
            for (int c = 0; c < W; ++c) sum[c] *= scale;
            store_pack<T, W>(dW + (size_t)key * D + col, sum);
        }
    }
}

// ---- up to 64 positions -----------------------------------------------------------------------------------------------------------------
// A wavefront holds all tokens, one a lane: no sort, one launch.  Workgroups [0, sum_blocks): a wavefront for each (position, column slab); the
// first position of a token adds the token's rows in order.  The others: 64 rows of the table each, zero where no token is.
template <typename T, int W>
__global__ __launch_bounds__(EB_THREADS) void embedding_bwd_few_kernel(const long long *__restrict__ tokens, const T *__restrict__ dy, long long ldy, int N,
                                                                      int V, int D, float scale, int pad, int sum_blocks, T *__restrict__ dW) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int key = lane < N ? (int)safe_index(tokens[lane], V) : -1;
    if ((int)blockIdx.x >= sum_blocks) {
        const int row0 = ((int)blockIdx.x - sum_blocks) * 64, rows = min(64, V - row0);
        unsigned long long used = key >= row0 && key < row0 + 64 && key != pad ? 1ull << (key - row0) : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) used |= __shfl_xor(used, d);
        for (int r = wave; r < rows; r += EB_THREADS / 64) {
            if ((used >> r) & 1) continue;
            T *dst = dW + (size_t)(row0 + r) * D;
            for (int c = lane * W; c < D; c += 64 * W) store_zeros<T, W>(dst + c);
        }
        return;
    }
    const int slabs = (D + 64 * W - 1) / (64 * W), unit = (int)blockIdx.x * (EB_THREADS / 64) + wave, i = unit / slabs;
    if (i >= N) return;
    const int mine = __shfl(key, i);
    unsigned long long todo = __ballot(key == mine);
    const int col = (unit % slabs) * 64 * W + lane * W;
    if (__builtin_ctzll(todo) != i || mine == pad || col >= D) return;
    float acc[W] = {};
    constexpr int AHEAD = 8;                                       // rows in flight
    while (todo) {
        Pack<T, W> row[AHEAD];
        bool in[AHEAD];
        int at = 0;
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {                          // (behind the token's last row: that one again, not used)
            in[q] = todo != 0;
            if (in[q]) at = __builtin_ctzll(todo);
            todo &= todo - 1;
            row[q] = *reinterpret_cast<const Pack<T, W> *>(dy + at * ldy + col);
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            if (in[q])
#pragma unroll
                for (int c = 0; c < W; ++c) acc[c] += to_f32(row[q].v[c]);
    }
#pragma unroll
    for (int c = 0; c < W; ++c) acc[c] *= scale;
    store_pack<T, W>(dW + (size_t)mine * D + col, acc);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
constexpr int EB_LDS_SORT = 16384;
template <int PER>
constexpr size_t eb_lds_sort_bytes() { return (size_t)1024 * PER * 6 + 16 * EB_BINS * 4 + 16 * 4; }

struct EmbeddingWs {
    int *keys[2], *pos[2], *hist;
    float *partial;
    size_t bytes;
    EmbeddingWs(void *ws, long long N, int D) {
        Carve c(ws);
        const long long tiles = (N + EB_SORT_TILE - 1) / EB_SORT_TILE, chunks = (N + EB_CHUNK - 1) / EB_CHUNK;
        for (int i = 0; i < 2; ++i) {
            const bool used = i == 0 || N > EB_LDS_SORT;
            keys[i] = c.take<int>(used ? N : 0);
            pos[i] = c.take<int>(used ? N : 0);
        }
        hist = c.take<int>(N > EB_LDS_SORT ? tiles * EB_BINS : 0);
        partial = c.take<float>((size_t)chunks * 2 * D);
        bytes = c.used;
    }
};

template <int PER>
static bool sort_lds(const int64_t *tokens, int N, int64_t V, int bits, int passes, const EmbeddingWs &w, hipStream_t s) {
    if (!ensure_dynamic_lds(embedding_sort_lds_kernel<PER>, eb_lds_sort_bytes<PER>())) return false;
    PHC_LAUNCH_AS(K_EMBEDDING_SORT, (embedding_sort_lds_kernel<PER>), dim3(1), dim3(1024), eb_lds_sort_bytes<PER>(), s,
                  reinterpret_cast<const long long *>(tokens), N, (long long)V, bits, passes, w.keys[0], w.pos[0]);
    return true;
}

// sorted (token, position) in keys[side], pos[side]; -1: a launch was refused
static int sort_tokens(const int64_t *tokens, int N, int64_t V, const EmbeddingWs &w, hipStream_t s) {
    int bits = 1;
    while ((1ll << bits) < V) ++bits;
    const int passes = (bits + EB_RADIX_BITS - 1) / EB_RADIX_BITS, width = (bits + passes - 1) / passes;
    if (N <= 2048) return sort_lds<2>(tokens, N, V, bits, passes, w, s) ? 0 : -1;
    if (N <= 6144) return sort_lds<6>(tokens, N, V, bits, passes, w, s) ? 0 : -1;
    if (N <= EB_LDS_SORT) return sort_lds<16>(tokens, N, V, bits, passes, w, s) ? 0 : -1;
    const int tiles = (N + EB_SORT_TILE - 1) / EB_SORT_TILE, mask = (1 << width) - 1;
    const long long *t = reinterpret_cast<const long long *>(tokens);
    int side = 1;
    for (int p = 0; p < passes; ++p, side ^= 1) {
        const int *keys = p ? w.keys[side] : nullptr, *pos = p ? w.pos[side] : nullptr;
        PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_hist_kernel, dim3(tiles), dim3(EB_THREADS), 0, s, keys, t, (long long)V, N, p * width, mask, w.hist);
        PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_scan_kernel, dim3(1), dim3(1024), 0, s, w.hist, tiles);
        PHC_LAUNCH_AS(K_EMBEDDING_SORT, embedding_scatter_kernel, dim3(tiles), dim3(EB_THREADS), 0, s, keys, t, (long long)V, pos, N, p * width, width,
                      (const int *)w.hist, w.keys[side ^ 1], w.pos[side ^ 1]);
    }
    return side;
}

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

// threads of one launch (the hardware counts them in 32 bits)
constexpr long long EB_MAX_THREADS = 1ll << 31;

template <typename T, int W>
static void launch_fwd(const int64_t *tokens, const void *weight, int64_t N, int64_t V, int64_t ldw, int D, float scale, void *out,
                       hipStream_t s) {
    const int lg = lane_group(D, W);
    const long long most = EB_MAX_THREADS >> lg;
    for (long long i = 0; i < N; i += most) {
        const long long n = N - i < most ? N - i : most;
        PHC_LAUNCH_AS(K_EMBEDDING_FWD, (embedding_fwd_kernel<T, W>), dim3((unsigned)(((n << lg) + EB_THREADS - 1) / EB_THREADS)), dim3(EB_THREADS), 0, s,
                      reinterpret_cast<const long long *>(tokens) + i, static_cast<const T *>(weight), n, (long long)V, (long long)ldw, D, scale, lg,
                      static_cast<T *>(out) + i * D, err_word());
    }
}

// Sums: a lane for each W columns of a chunk.
static int bwd_lanes(int D, int W) {
    const int lg = lane_group(D, W);
    return lg < 3 ? 3 : lg;                                       // (8 lanes at least: a group stages 66 words)
}
static long long bwd_chunk_blocks(long long N, int D, int W) {
    const int lg = bwd_lanes(D, W);
    const long long slabs = (D + (W << lg) - 1) / (W << lg), chunks = (N + EB_CHUNK - 1) / EB_CHUNK;
    return (((chunks * slabs) << lg) + EB_THREADS - 1) / EB_THREADS;
}

template <typename T, int W>
static void launch_bwd(const EmbeddingWs &w, int side, const void *dy, int64_t N, int64_t V, int64_t ldy, int D, float scale, int pad,
                       void *dW, hipStream_t s) {
    const int lg = bwd_lanes(D, W);
    const long long slabs = (D + (W << lg) - 1) / (W << lg), chunks = (N + EB_CHUNK - 1) / EB_CHUNK;
    const long long cb = bwd_chunk_blocks(N, D, W), zb = (V + 63) / 64;
    PHC_LAUNCH_AS(K_EMBEDDING_BWD, (embedding_bwd_kernel<T, W>), dim3((unsigned)(cb + zb)), dim3(EB_THREADS),
                  (EB_THREADS >> lg) * (2 * EB_CHUNK + 2) * sizeof(int), s, (const int *)w.keys[side],
               (const int *)w.pos[side], static_cast<const T *>(dy), (long long)ldy, (int)N, (int)V, D, scale, pad, lg, (int)cb,
               static_cast<T *>(dW), w.partial);
    if (chunks > 1)
        PHC_LAUNCH_AS(K_EMBEDDING_BWD, (embedding_join_kernel<T, W>), dim3((unsigned)((chunks + EB_JOIN - 2) / EB_JOIN * slabs)), dim3(EB_THREADS), 0, s, (const int *)w.keys[side],
                      (int)N, D, scale, pad, lg, (int)chunks, (int)slabs, (const float *)w.partial, static_cast<T *>(dW));
}

constexpr int EB_FEW = 64;

template <typename T, int W>
static void launch_bwd_few(const int64_t *tokens, const void *dy, int64_t N, int64_t V, int64_t ldy, int D, float scale, int pad, void *dW, hipStream_t s) {
    const long long units = N * ((D + 64 * W - 1) / (64 * W)), sb = (units + EB_THREADS / 64 - 1) / (EB_THREADS / 64);
    PHC_LAUNCH_AS(K_EMBEDDING_BWD, (embedding_bwd_few_kernel<T, W>), dim3((unsigned)(sb + (V + 63) / 64)), dim3(EB_THREADS), 0, s,
                  reinterpret_cast<const long long *>(tokens), static_cast<const T *>(dy), (long long)ldy, (int)N, (int)V, D, scale, pad, (int)sb,
                  static_cast<T *>(dW));
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
    PHC_REQUIRE(N <= (1ll << 28) && V <= (1ll << 29) && D <= (1ll << 20), PHC_ERR_UNSUPPORTED, "%s: N=%lld V=%lld D=%lld is beyond 2^28, 2^29, 2^20",
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
    if (N < 0 || N > (1ll << 28) || V < 1 || V > (1ll << 29) || D < 1 || D > (1ll << 20)) return 0;
    return EmbeddingWs(nullptr, N, (int)D).bytes + 256;
}

int phc_embedding_bwd(const int64_t *tokens, const void *dy, int64_t N, int64_t V, int64_t D, int64_t ldy, int dtype, float scale,
                      int64_t padding_idx, void *dW, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = embedding_check("phc_embedding_bwd", N, V, D, ldy, dtype)) return rc;
    PHC_REQUIRE(dW && (N == 0 || (tokens && dy)), PHC_ERR_INVALID_ARG, "phc_embedding_bwd: null pointer");
    PHC_REQUIRE(ws && aligned_to(ws, 16) && ws_bytes >= phc_embedding_bwd_ws_bytes(N, V, D), PHC_ERR_WORKSPACE,
                "phc_embedding_bwd: workspace of %zu bytes, %zu needed", ws_bytes, phc_embedding_bwd_ws_bytes(N, V, D));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int width = pack_width(dtype_bytes(dtype), D, ldy, dy ? dy : dW, dW);
    PHC_REQUIRE(bwd_chunk_blocks(N, (int)D, width) <= EB_MAX_THREADS / EB_THREADS - (V + 63) / 64, PHC_ERR_UNSUPPORTED,
                "phc_embedding_bwd: N=%lld rows of %lld are beyond one launch", (long long)N, (long long)D);
    const int pad = padding_idx >= 0 && padding_idx < V ? (int)padding_idx : -1;
    if (N <= EB_FEW) {
        EB_DISPATCH(launch_bwd_few, dtype, width, tokens, dy, N, V, ldy, (int)D, scale, pad, dW, s);
        return launch_status("phc_embedding_bwd");
    }
    EmbeddingWs w(ws, N, (int)D);
    const int side = sort_tokens(tokens, (int)N, V, w, s);
    PHC_REQUIRE(side >= 0, PHC_ERR_LAUNCH, "phc_embedding_bwd: the runtime refused the sort's LDS size");
    EB_DISPATCH(launch_bwd, dtype, width, w, side, dy, N, V, ldy, (int)D, scale, pad, dW, s);
    return launch_status("phc_embedding_bwd");
}

}  // extern "C"
