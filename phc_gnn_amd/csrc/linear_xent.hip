// Softmax cross entropy of a linear map over a large vocabulary, without keeping the logits (fp32 / bf16 / fp16).
//
//   l_iv = x_i . w_v + b_v      lse_i = log sum_v exp l_iv      loss_i = lse_i - l_{i, t_i}      (0 where t_i = ignore_index)
//   d_iv = exp(l_iv - lse_i) - [v = t_i]       dx_i = g_i sum_v d_iv w_v       dw_v = sum_i g_i d_iv x_i       db_v = sum_i g_i d_iv
//
// Forward: ONE product whose tiles never leave the registers — every tile leaves the maximum and the sum of exponentials of its part
// of a row and, where the target lies in it, the target's logit; a small kernel joins the parts.  Backward keeps only lse: the
// vocabulary is walked in pieces, a piece's logits are computed again, become d in the tile's registers, are written in 16 bits in
// both orders (N x piece and piece x N) and feed the two gradient products while they lie in the caches.
//
// All products run through one kernel, C[m, n] = sum_k A[m, k] B[n, k] with k contiguous in both operands, on 16-bit matrix
// instructions with fp32 accumulators.  The vocabulary (or the output's contiguous dimension) is always the m side: a lane then holds four
// consecutive m of one n, so row statistics are mostly in-lane and outputs are stored in 16-byte pieces.
//
// fp32 inputs: every value is split into three bf16 terms, a = h + m + l (8 bits each, |a - h - m - l| <= 2^-26 |a|), and the product
// is the sum of the six term products l h, h l, m m, m h, h m, h h (smallest first; the three left out are below 2^-25 |a b|): the same
// kernel walks six (plane of A, plane of B) pairs.  Six 16-bit products cost less than one product on the fp32 matrix instructions,
// whose rate is a sixteenth of the 16-bit one.
#include "dtype_io.h"

namespace phc {

constexpr int XT_BK = 64;                      // k per step: 128 bytes of a row = one line of LDS

// ---- operand layout -------------------------------------------------------------------------------------------------------------------
struct XPlanes {
    void *p[3];
};

__device__ __forceinline__ void split3(float a, bf16_t &h, bf16_t &m, bf16_t &l) {
    h = (bf16_t)a;
    const float r = a - (float)h;
    m = (bf16_t)r;
    l = (bf16_t)(r - (float)m);
}

// value -> the operand planes (one for 16-bit types, three for fp32)
template <typename TIN>
__device__ __forceinline__ void put_planes(const XPlanes &o, size_t at, TIN v) {
    if constexpr (sizeof(TIN) == 4) {
        bf16_t h, m, l;
        split3(v, h, m, l);
        static_cast<bf16_t *>(o.p[0])[at] = h;
        static_cast<bf16_t *>(o.p[1])[at] = m;
        static_cast<bf16_t *>(o.p[2])[at] = l;
    } else {
        static_cast<TIN *>(o.p[0])[at] = v;
    }
}

// rows [R, C] -> operand rows [R, Cp], columns behind C zero
template <typename TIN>
__global__ __launch_bounds__(256) void xent_pack_kernel(const TIN *__restrict__ src, long long ld, long long R, int C, int Cp, XPlanes out) {
    const long long total = R * (long long)Cp;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const long long r = e / Cp;
        const int c = (int)(e - r * Cp);
        put_planes<TIN>(out, (size_t)e, c < C ? src[r * ld + c] : (TIN)0.f);
    }
}

// rows [R, C] -> operand columns [C, Rp], rows behind R zero; `target`: a row whose target is ignored counts as zero, whatever it
// holds (its d is zero, and zero times a NaN is none)
template <typename TIN>
__global__ __launch_bounds__(256) void xent_transpose_kernel(const TIN *__restrict__ src, long long ld, long long R, int C, long long Rp,
                                                            const long long *__restrict__ target, long long ignore, XPlanes out) {
    __shared__ TIN tile[64][65];
    const long long r0 = (long long)blockIdx.x * 64;
    const int c0 = (int)blockIdx.y * 64;
    for (int i = threadIdx.x >> 6; i < 64; i += 4) {
        const long long r = r0 + i;
        const int c = c0 + (threadIdx.x & 63);
        TIN v = (TIN)0.f;
        if (r < R && c < C && !(target && target[r] == ignore)) v = src[r * ld + c];
        tile[i][threadIdx.x & 63] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x >> 6; i < 64; i += 4) {
        const int c = c0 + i;
        const long long r = r0 + (threadIdx.x & 63);
        if (c < C && r < Rp) put_planes<TIN>(out, (size_t)c * Rp + r, tile[threadIdx.x & 63][i]);
    }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void xt_wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void xt_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// One LDS-DMA instruction: every lane's 16 bytes at base + voff land at LDS byte address lds + 16 lane.  In asm because hipcc orders its
// builtin against every later LDS read with s_waitcnt vmcnt(0), which would drain the prefetch; the loop's own waits order it.  M0 is
// the DMA's LDS base, saved and restored inside the statement.
__device__ __forceinline__ void xt_dma16(unsigned lds, unsigned voff, const void *base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds), "v"(voff), "s"(base)
                 : "memory");
}

template <typename T>
struct Mfma16;
template <>
struct Mfma16<bf16_t> {
    typedef bf16x8_t frag;
    static __device__ __forceinline__ f32x4_t mul(frag a, frag b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mfma16<f16_t> {
    typedef f16x8_t frag;
    static __device__ __forceinline__ f32x4_t mul(frag a, frag b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

enum XEpilogue { XE_STATS, XE_DLOGITS, XE_OUT };

struct XGemm {
    const char *A[6], *B[6];       // operand planes of each segment of the k loop
    int segments;                  // 1, or 6 for fp32 inputs
    int ksteps;                    // steps of XT_BK per segment
    unsigned lda, ldb;             // row strides in bytes
    long long rowsA, rowsB;        // valid m, n
    int tilesM, tilesN, splits;
    // XE_STATS / XE_DLOGITS
    const void *bias;              // fp32 or the operand's type (bias_f32), of this piece; may be null
    int bias_f32;
    const long long *target;       // [rowsB]
    long long ignore, first_v, vocab;     // piece begins at first_v
    int *err;
    float *part_max, *part_sum;    // [parts][rowsB]
    float *target_logit;           // [rowsB]
    const float *lse, *row_rel;    // [rowsB]
    XPlanes d, dT;                 // [rowsB][ldd] and [m][lddT]
    long long ldd, lddT;
    float d_scale;                 // 16-bit d are stored times this
    float *db_part;                // [tilesN * WN][rowsA] or null
    // XE_OUT
    const float *row_scale;        // [rowsB] or null
    const float *scale;            // one value, or null
    float out_scale;
    void *out;                     // element (n, m) at n * ldo + m
    long long ldo, slab;           // slab: elements between the splits' partial outputs (fp32), 0 = final output in its own type
    int accumulate, out_dtype, out_vec;
};

// Tile order: the workgroups of an XCD take neighbouring tiles (blockIdx goes round-robin over the 8 XCDs), in bands of 8 m-tiles, so
// that the tiles in flight on an XCD share operand rows in its L2.
__device__ __forceinline__ void xt_tile_of(unsigned b, int tilesM, int tilesN, int &tm, int &tn) {
    const unsigned total = (unsigned)tilesM * tilesN;
    const unsigned per = total / 8, rest = total % 8, x = b % 8, i = b / 8;
    const unsigned t = x * per + (x < rest ? x : rest) + i;
    const unsigned band = t / (8u * tilesN);
    const unsigned height = min(8u, (unsigned)tilesM - band * 8u);
    const unsigned in = t - band * 8u * tilesN;
    tm = (int)(band * 8u + in % height);
    tn = (int)(in / height);
}

template <typename T, int EPI, bool WIDE, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM *WN * 64, 2) void xent_gemm_kernel(XGemm a) {
    typedef typename Mfma16<T>::frag frag;
    constexpr int NW = WM * WN, TM = WM * FM * 16, TN = WN * FN * 16;
    constexpr int LOADS = (TM + TN) / 8 / NW;                   // LDS-DMA instructions per wavefront and step (8 rows each)
    static_assert((TM / 8) % LOADS == 0, "a wavefront loads rows of one operand");
    constexpr unsigned BUF = (TM + TN) * 128;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const unsigned tiles = (unsigned)a.tilesM * a.tilesN;
    const int split = (int)(blockIdx.x / tiles);
    int tm, tn;
    xt_tile_of(blockIdx.x % tiles, a.tilesM, a.tilesN, tm, tn);

    // this split's share of the steps
    const int steps = a.segments * a.ksteps;
    const int s0 = (int)((long long)steps * split / a.splits), s1 = (int)((long long)steps * (split + 1) / a.splits);

    // loader: the wavefront's rows of its operand; 16-byte pieces of a row are stored at piece ^ (row & 7) (bank spread for the reads)
    const bool loads_a = wave * LOADS < TM / 8;
    const long long row0 = loads_a ? (long long)tm * TM : (long long)tn * TN;
    const long long rows = loads_a ? a.rowsA : a.rowsB;
    const unsigned ld = loads_a ? a.lda : a.ldb;
    unsigned voff[LOADS];
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
        const int r = (wave * LOADS + q) * 8 - (loads_a ? 0 : TM) + (lane >> 3);
        const long long row = min(row0 + r, rows - 1) - row0;   // rows behind the operand repeat its last one; their results are dropped
        voff[q] = (unsigned)row * ld + (((lane & 7) ^ (r & 7)) << 4);
    }
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    const unsigned lds_wave = lds0 + wave * LOADS * 1024;
    auto issue = [&](int s, int buf) {
        const int seg = s / a.ksteps, k = s - seg * a.ksteps;
        const char *base = (loads_a ? a.A[seg] : a.B[seg]) + row0 * ld + (size_t)k * (XT_BK * 2);
#pragma unroll
        for (int q = 0; q < LOADS; ++q) xt_dma16(lds_wave + buf * BUF + q * 1024, voff[q], base);
    };

    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int fr = lane & 15, fg = lane >> 4;
    if (s0 < s1) issue(s0, 0);
    for (int s = s0; s < s1; ++s) {
        const int buf = (s - s0) & 1;
        xt_wait_lds();                                          // this wavefront's reads of the other buffer are done
        xt_wait_vm<0>();                                        // and its loads into this one
        __builtin_amdgcn_s_barrier();
        if (s + 1 < s1) issue(s + 1, buf ^ 1);
        const char *la = smem + buf * BUF, *lb = la + TM * 128;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            frag fa[FM], fb[FN];
            const int piece = ((kk * 4 + fg) ^ (fr & 7)) << 4;
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const frag *>(la + (wm * FM * 16 + i * 16 + fr) * 128 + piece);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = *reinterpret_cast<const frag *>(lb + (wn * FN * 16 + j * 16 + fr) * 128 + piece);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = Mfma16<T>::mul(fa[i], fb[j], acc[i][j]);
        }
    }

    // element (i, j, r): m = mbase + i * 16 + r, n = nbase + j * 16
    const long long mbase = (long long)tm * TM + wm * FM * 16 + fg * 4;
    const long long nbase = (long long)tn * TN + wn * FN * 16 + fr;
    if constexpr (EPI == XE_STATS || EPI == XE_DLOGITS) {
        float bias[FM][4];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const long long m = mbase + i * 16 + r;
                float b = 0.f;
                if (a.bias && m < a.rowsA) b = a.bias_f32 ? static_cast<const float *>(a.bias)[m] : to_f32(static_cast<const T *>(a.bias)[m]);
                bias[i][r] = m < a.rowsA ? b : -INFINITY;       // columns behind the vocabulary: exp 0
            }
        float dbs[FM][4] = {};
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const long long n = nbase + j * 16;
            const bool in = n < a.rowsB;
            const long long t = a.target[in ? n : 0];
            const bool kept = in && t != a.ignore;
            const long long hit = (kept ? (EPI == XE_STATS ? checked_index(t, a.vocab, fg == 0 && tm == 0 ? a.err : nullptr, PHC_IDX_ERR_TARGET)
                                                          : safe_index(t, a.vocab))
                                        : -1) - a.first_v - mbase;          // target's m, counted from this lane's first
            if constexpr (EPI == XE_STATS) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float l = acc[i][j][r] + bias[i][r];
                        acc[i][j][r] = l;
                        mx = fmaxf(mx, l);
                        if (hit == i * 16 + r) a.target_logit[n] = l;
                    }
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float shift = mx == -INFINITY ? 0.f : mx;             // nothing but -inf: every exponential is 0
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum += WIDE ? expf(acc[i][j][r] - shift) : __expf(acc[i][j][r] - shift);
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                if (in && fg == 0) {
                    const size_t at = (size_t)(tm * WM + wm) * a.rowsB + n;
                    a.part_max[at] = mx;
                    a.part_sum[at] = sum;
                }
            } else {
                const float lse = in ? a.lse[n] : 0.f, rel = in ? a.row_rel[n] : 0.f;
#pragma unroll
                for (int i = 0; i < FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float l = acc[i][j][r] + bias[i][r];
                        const float p = WIDE ? expf(l - lse) : __expf(l - lse);
                        const long long m = mbase + i * 16 + r;
                        const float d = kept && m < a.rowsA ? p - (hit == i * 16 + r ? 1.f : 0.f) : 0.f;
                        const float dr = kept && m < a.rowsA ? d * rel : 0.f;
                        dbs[i][r] += dr;
                        if (in && m < a.ldd) put_planes<std::conditional_t<WIDE, float, T>>(a.d, (size_t)n * a.ldd + m, (std::conditional_t<WIDE, float, T>)(d * a.d_scale));
                        if (m < a.rowsA && n < a.lddT) put_planes<std::conditional_t<WIDE, float, T>>(a.dT, (size_t)m * a.lddT + n, (std::conditional_t<WIDE, float, T>)(dr * a.d_scale));
                    }
                }
            }
        }
        if (EPI == XE_DLOGITS && a.db_part) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = dbs[i][r];
#pragma unroll
                    for (int x = 1; x < 16; x <<= 1) v += __shfl_xor(v, x);
                    const long long m = mbase + i * 16 + r;
                    if (fr == 0 && m < a.rowsA) a.db_part[(size_t)(tn * WN + wn) * a.rowsA + m] = v;
                }
        }
    } else {
        const float s = a.out_scale * (a.scale ? *a.scale : 1.f);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const long long n = nbase + j * 16;
            if (n >= a.rowsB) continue;
            const float sn = a.row_scale ? a.row_scale[n] * s : s;
            const bool zero = a.row_scale && a.row_scale[n] == 0.f;         // (a row without a gradient: 0 whatever the operands hold)
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const long long m = mbase + i * 16;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = zero ? 0.f : acc[i][j][r] * sn;
                const size_t at = (size_t)n * a.ldo + m;
                if (a.slab || a.out_dtype == PHC_DTYPE_F32) {
                    float *o = static_cast<float *>(a.out) + (a.slab ? (size_t)split * a.slab : 0) + at;
                    if (a.out_vec && m + 4 <= a.rowsA) {
                        float4 q = make_float4(v[0], v[1], v[2], v[3]);
                        if (a.accumulate) {
                            const float4 p = *reinterpret_cast<const float4 *>(o);
                            q.x += p.x, q.y += p.y, q.z += p.z, q.w += p.w;
                        }
                        *reinterpret_cast<float4 *>(o) = q;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < a.rowsA) o[r] = a.accumulate ? o[r] + v[r] : v[r];
                    }
                } else {
                    T *o = static_cast<T *>(a.out) + at;
                    if (a.out_vec && m + 4 <= a.rowsA) store_pack<T, 4>(o, v);
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < a.rowsA) o[r] = from_f32<T>(v[r]);
                }
            }
        }
    }
}

// ---- rows -------------------------------------------------------------------------------------------------------------------------------
// A workgroup joins the parts of 64 rows: 16 wavefronts share the parts, then one adds them up.
__global__ __launch_bounds__(1024) void xent_rows_kernel(const float *__restrict__ part_max, const float *__restrict__ part_sum, int parts,
                                                        long long N, const float *__restrict__ target_logit,
                                                        const long long *__restrict__ target, long long ignore, float *__restrict__ lse,
                                                        float *__restrict__ loss) {
    __shared__ float sm[16][64], ss[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long n = (long long)blockIdx.x * 64 + lane;
    float mx = -INFINITY, sum = 0.f;
    auto join = [&](float m, float s) {
        const float top = fmaxf(mx, m);
        const float shift = top == -INFINITY ? 0.f : top;
        sum = sum * expf(mx - shift) + s * expf(m - shift);
        mx = top;
    };
    if (n < N)
        for (int p = wave; p < parts; p += 16) join(part_max[(size_t)p * N + n], part_sum[(size_t)p * N + n]);
    sm[wave][lane] = mx;
    ss[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && n < N) {
        for (int w = 1; w < 16; ++w) join(sm[w][lane], ss[w][lane]);
        const float l = mx + logf(sum);
        lse[n] = l;
        loss[n] = target[n] == ignore ? 0.f : l - target_logit[n];
    }
}

// sum of the rows' losses and the number of rows that count -> out[0] = sum or mean, stat = {sum, count}
__global__ __launch_bounds__(1024) void xent_reduce_kernel(const float *__restrict__ rows, const long long *__restrict__ target, long long ignore,
                                                          long long N, int mean, float *__restrict__ out, float *__restrict__ stat) {
    __shared__ double red[16], cnt[16];
    double s = 0.0, c = 0.0;
    for (long long i = threadIdx.x; i < N; i += 1024) {
        if (target[i] == ignore) continue;
        s += (double)rows[i];
        c += 1.0;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        s += __shfl_xor(s, d);
        c += __shfl_xor(c, d);
    }
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = s;
        cnt[threadIdx.x >> 6] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) {
            s += red[w];
            c += cnt[w];
        }
        if (out) out[0] = (float)(mean ? s / c : s);          // (no row counts: the mean of nothing is NaN)
        stat[0] = (float)s;
        stat[1] = (float)c;
    }
}

// g_i of every row: row_scale = g_i (dx), top = max |g_i|, row_rel = g_i / top (what the 16-bit d of the weight gradient carry)
__global__ __launch_bounds__(1024) void xent_scales_kernel(const float *__restrict__ dloss, int per_row, int mean, const float *__restrict__ stat,
                                                          const long long *__restrict__ target, long long ignore, long long N,
                                                          float *__restrict__ row_scale, float *__restrict__ row_rel, float *__restrict__ top) {
    __shared__ float red[16];
    const float count = stat[1];
    auto g_of = [&](long long i) {
        if (target[i] == ignore) return 0.f;
        const float g = per_row ? dloss[i] : dloss[0];
        return mean ? g / count : g;
    };
    float m = 0.f;
    for (long long i = threadIdx.x; i < N; i += 1024) m = fmaxf(m, fabsf(g_of(i)));
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int w = 0; w < 16; ++w) m = fmaxf(m, red[w]);
    if (threadIdx.x == 0) *top = m;
    for (long long i = threadIdx.x; i < N; i += 1024) {
        const float g = g_of(i);
        row_scale[i] = g;
        row_rel[i] = g == 0.f ? 0.f : g / m;
    }
}

// out[i] = sum over the slabs, in order
template <typename T>
__global__ __launch_bounds__(256) void xent_sum_slabs_kernel(const float *__restrict__ slabs, long long slab, int n, long long count,
                                                            const float *__restrict__ scale, T *__restrict__ out) {
    const float f = scale ? *scale : 1.f;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < count; e += (long long)gridDim.x * 256) {
        float v = slabs[e];
        for (int s = 1; s < n; ++s) v += slabs[(size_t)s * slab + e];
        out[e] = from_f32<T>(v * f);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
static long long round_up(long long v, long long m) { return (v + m - 1) / m * m; }
static long long ceil_div(long long v, long long m) { return (v + m - 1) / m; }

constexpr long long XT_PIECE_BYTES = 256ll << 20;      // both orders of a piece's d together: what the Infinity Cache holds

struct XPlan {
    bool wide;                 // fp32 inputs
    int planes, segments;
    long long Kp, Np, piece, pieces;
    bool pack_x, pack_w;
    long long parts;
    int splits_dx, splits_dw;
};

constexpr int TILE = 128;

static int splits_for(long long tiles, long long steps) {
    // enough workgroups for the 256 CUs twice over, at least 8 steps each
    long long s = ceil_div(512, tiles);
    if (s > steps / 8) s = steps / 8;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

static XPlan make_plan(const phc_linear_xent_desc *d) {
    XPlan p;
    p.wide = d->dtype == PHC_DTYPE_F32;
    p.planes = p.wide ? 3 : 1;
    p.segments = p.wide ? 6 : 1;
    p.Kp = round_up(d->D, XT_BK);
    p.Np = round_up(d->N, XT_BK);
    // an operand is read where it lies when its rows are whole steps and 16-byte aligned
    p.pack_x = p.wide || d->D % XT_BK || d->ldx % 8 || !aligned_to(d->x, 16);
    p.pack_w = p.wide || d->D % XT_BK || d->ldw % 8 || !aligned_to(d->W, 16);
    p.parts = ceil_div(d->V, TILE) * 2;
    long long piece = XT_PIECE_BYTES / (4 * p.planes * (d->N > 0 ? d->N : 1)) / 256 * 256;
    if (piece < 2048) piece = 2048;
    if (d->piece > 0) piece = round_up(d->piece, 64);
    if (piece >= d->V) piece = round_up(d->V, 64);
    p.pieces = ceil_div(d->V, piece);
    p.piece = d->piece > 0 ? piece : round_up(ceil_div(d->V, p.pieces), 64);
    p.pieces = ceil_div(d->V, p.piece);
    p.splits_dx = splits_for(ceil_div(d->D, TILE) * ceil_div(d->N, TILE), p.segments * (p.piece / XT_BK));
    p.splits_dw = splits_for(ceil_div(d->D, TILE) * ceil_div(p.piece, TILE), p.segments * (p.Np / XT_BK));
    return p;
}

struct XWs {
    XPlanes x{}, w{}, xT{}, wT{}, dl{}, dlT{};
    float *part_max = nullptr, *part_sum = nullptr, *target_logit = nullptr, *rows = nullptr;
    float *row_scale = nullptr, *row_rel = nullptr, *top = nullptr, *dx_slabs = nullptr, *dw_slabs = nullptr, *db_part = nullptr;
    size_t bytes;
    XWs(const phc_linear_xent_desc *d, const XPlan &p, bool backward, void *ws) {
        Carve c(ws);
        auto planes = [&](XPlanes &o, size_t count) {
            for (int i = 0; i < p.planes; ++i) o.p[i] = c.take<unsigned short>(count);
        };
        if (p.pack_x) planes(x, (size_t)d->N * p.Kp);
        if (p.pack_w) planes(w, (size_t)(backward ? p.piece : d->V) * p.Kp);
        if (!backward) {
            part_max = c.take<float>((size_t)p.parts * d->N);
            part_sum = c.take<float>((size_t)p.parts * d->N);
            target_logit = c.take<float>(d->N);
            rows = c.take<float>(d->N);
        } else {
            row_scale = c.take<float>(d->N);
            row_rel = c.take<float>(d->N);
            top = c.take<float>(1);
            planes(dl, (size_t)d->N * p.piece);
            planes(dlT, (size_t)p.piece * p.Np);
            if (d->dx) {
                planes(wT, (size_t)d->D * p.piece);
                if (p.splits_dx > 1 || p.pieces > 1) dx_slabs = c.take<float>((size_t)p.splits_dx * d->N * d->D);
            }
            if (d->dW) {
                planes(xT, (size_t)d->D * p.Np);
                if (p.splits_dw > 1) dw_slabs = c.take<float>((size_t)p.splits_dw * p.piece * d->D);
            }
            if (d->db) db_part = c.take<float>((size_t)ceil_div(d->N, TILE) * 2 * p.piece);
        }
        bytes = c.used;
    }
};

static unsigned flat_grid(long long n) {
    const long long b = ceil_div(n, 256);
    return (unsigned)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

static void pack(const phc_linear_xent_desc *d, const void *src, long long ld, long long R, int C, long long Cp, const XPlanes &out, hipStream_t s) {
    const dim3 g(flat_grid(R * Cp));
    if (d->dtype == PHC_DTYPE_F32)
        PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_pack_kernel<float>), g, dim3(256), 0, s, static_cast<const float *>(src), ld, R, C, (int)Cp, out);
    else if (d->dtype == PHC_DTYPE_BF16)
        PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_pack_kernel<bf16_t>), g, dim3(256), 0, s, static_cast<const bf16_t *>(src), ld, R, C, (int)Cp, out);
    else
        PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_pack_kernel<f16_t>), g, dim3(256), 0, s, static_cast<const f16_t *>(src), ld, R, C, (int)Cp, out);
}

static void transpose(const phc_linear_xent_desc *d, const void *src, long long ld, long long R, int C, long long Rp, const long long *target,
                      const XPlanes &out, hipStream_t s) {
    const dim3 g((unsigned)ceil_div(Rp, 64), (unsigned)ceil_div(C, 64));
    const long long ig = d->ignore_index;
    if (d->dtype == PHC_DTYPE_F32)
        PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_transpose_kernel<float>), g, dim3(256), 0, s, static_cast<const float *>(src), ld, R, C, Rp, target, ig, out);
    else if (d->dtype == PHC_DTYPE_BF16)
        PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_transpose_kernel<bf16_t>), g, dim3(256), 0, s, static_cast<const bf16_t *>(src), ld, R, C, Rp, target, ig, out);
    else
        PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_transpose_kernel<f16_t>), g, dim3(256), 0, s, static_cast<const f16_t *>(src), ld, R, C, Rp, target, ig, out);
}

static void set_planes(const XPlan &p, const XPlanes &A, const XPlanes &B, XGemm *g) {
    static const int ia[6] = {2, 0, 1, 1, 0, 0}, ib[6] = {0, 2, 1, 0, 1, 0};
    g->segments = p.segments;
    for (int i = 0; i < 6; ++i) {
        g->A[i] = static_cast<const char *>(A.p[p.wide ? ia[i] : 0]);
        g->B[i] = static_cast<const char *>(B.p[p.wide ? ib[i] : 0]);
    }
}

template <typename T, int EPI, bool WIDE>
static bool launch_gemm(int kid, XGemm &g, hipStream_t s) {
    constexpr int WM = 2, WN = 2, FM = 4, FN = 4, LDS = 2 * (WM * FM + WN * FN) * 16 * 128;
    g.tilesM = (int)ceil_div(g.rowsA, WM * FM * 16);
    g.tilesN = (int)ceil_div(g.rowsB, WN * FN * 16);
    if (!ensure_dynamic_lds(xent_gemm_kernel<T, EPI, WIDE, WM, WN, FM, FN>, LDS)) return false;
    PHC_LAUNCH_AS(kid, (xent_gemm_kernel<T, EPI, WIDE, WM, WN, FM, FN>), dim3((unsigned)(g.tilesM * g.tilesN * g.splits)), dim3(WM * WN * 64), LDS, s, g);
    return true;
}
template <int EPI>
static bool gemm(const phc_linear_xent_desc *d, int kid, XGemm &g, hipStream_t s) {
    if (d->dtype == PHC_DTYPE_F32) return launch_gemm<bf16_t, EPI, true>(kid, g, s);
    if (d->dtype == PHC_DTYPE_BF16) return launch_gemm<bf16_t, EPI, false>(kid, g, s);
    return launch_gemm<f16_t, EPI, false>(kid, g, s);
}

static void sum_slabs(const phc_linear_xent_desc *d, int kid, const float *slabs, long long slab, int n, long long count, const float *scale, void *out,
                      hipStream_t s) {
    const dim3 g(flat_grid(count));
    if (d->dtype == PHC_DTYPE_F32)
        PHC_LAUNCH_AS(kid, (xent_sum_slabs_kernel<float>), g, dim3(256), 0, s, slabs, slab, n, count, scale, static_cast<float *>(out));
    else if (d->dtype == PHC_DTYPE_BF16)
        PHC_LAUNCH_AS(kid, (xent_sum_slabs_kernel<bf16_t>), g, dim3(256), 0, s, slabs, slab, n, count, scale, static_cast<bf16_t *>(out));
    else
        PHC_LAUNCH_AS(kid, (xent_sum_slabs_kernel<f16_t>), g, dim3(256), 0, s, slabs, slab, n, count, scale, static_cast<f16_t *>(out));
}

static int xent_check(const char *who, const phc_linear_xent_desc *d) {
    PHC_REQUIRE(d, PHC_ERR_INVALID_ARG, "%s: null descriptor", who);
    PHC_REQUIRE(dtype_bytes(d->dtype), PHC_ERR_INVALID_ARG, "%s: unknown dtype %d", who, d->dtype);
    PHC_REQUIRE(d->reduction >= 0 && d->reduction <= 2, PHC_ERR_INVALID_ARG, "%s: unknown reduction %d", who, d->reduction);
    PHC_REQUIRE(d->N >= 1 && d->V >= 1 && d->D >= 1, PHC_ERR_INVALID_ARG, "%s: N=%lld V=%lld D=%lld", who, (long long)d->N, (long long)d->V, (long long)d->D);
    PHC_REQUIRE(d->N <= (1 << 22) && d->V <= (1 << 22) && d->D <= (1 << 20) && d->ldx <= (1 << 22) && d->ldw <= (1 << 22), PHC_ERR_UNSUPPORTED,
                "%s: N=%lld, V=%lld, D=%lld or a row stride is beyond 2^22, 2^22, 2^20, 2^22", who, (long long)d->N, (long long)d->V, (long long)d->D);
    PHC_REQUIRE(d->ldx >= d->D && d->ldw >= d->D, PHC_ERR_INVALID_ARG, "%s: row stride below the row length", who);
    PHC_REQUIRE(d->piece >= 0, PHC_ERR_INVALID_ARG, "%s: piece %lld", who, (long long)d->piece);
    PHC_REQUIRE(d->x && d->W && d->target && d->lse && d->stat, PHC_ERR_INVALID_ARG, "%s: null pointer", who);
    return PHC_OK;
}

}  // namespace phc

using namespace phc;

extern "C" {

size_t phc_linear_xent_ws_bytes(const phc_linear_xent_desc *d, int backward) {
    if (xent_check("phc_linear_xent_ws_bytes", d)) return 0;
    return XWs(d, make_plan(d), backward != 0, nullptr).bytes + 256;
}

int phc_linear_xent_fwd(const phc_linear_xent_desc *d, void *stream) {
    if (int rc = xent_check("phc_linear_xent_fwd", d)) return rc;
    PHC_REQUIRE(d->loss, PHC_ERR_INVALID_ARG, "phc_linear_xent_fwd: null pointer");
    PHC_REQUIRE(d->ws && aligned_to(d->ws, 256) && d->ws_bytes >= phc_linear_xent_ws_bytes(d, 0), PHC_ERR_WORKSPACE,
                "phc_linear_xent_fwd: workspace of %zu bytes, %zu needed", (size_t)d->ws_bytes, phc_linear_xent_ws_bytes(d, 0));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const XPlan p = make_plan(d);
    XWs w(d, p, false, d->ws);
    const int es = dtype_bytes(d->dtype);
    XPlanes X{{const_cast<void *>(d->x)}}, W{{const_cast<void *>(d->W)}};
    long long ldx = d->ldx * es, ldw = d->ldw * es;
    if (p.pack_x) {
        pack(d, d->x, d->ldx, d->N, (int)d->D, p.Kp, w.x, s);
        X = w.x;
        ldx = p.Kp * 2;
    }
    if (p.pack_w) {
        pack(d, d->W, d->ldw, d->V, (int)d->D, p.Kp, w.w, s);
        W = w.w;
        ldw = p.Kp * 2;
    }
    XGemm g{};
    set_planes(p, W, X, &g);
    g.ksteps = (int)(p.Kp / XT_BK);
    g.lda = (unsigned)ldw;
    g.ldb = (unsigned)ldx;
    g.rowsA = d->V;
    g.rowsB = d->N;
    g.splits = 1;
    g.bias = d->bias;
    g.bias_f32 = p.wide;
    g.target = reinterpret_cast<const long long *>(d->target);
    g.ignore = d->ignore_index;
    g.vocab = d->V;
    g.err = err_word();
    g.part_max = w.part_max;
    g.part_sum = w.part_sum;
    g.target_logit = w.target_logit;
    PHC_REQUIRE(gemm<XE_STATS>(d, K_XENT_LOGITS, g, s), PHC_ERR_LAUNCH, "phc_linear_xent_fwd: LDS size refused");
    float *rows = d->reduction == 0 ? d->loss : w.rows;
    PHC_LAUNCH_AS(K_XENT_ROWS, xent_rows_kernel, dim3((unsigned)ceil_div(d->N, 64)), dim3(1024), 0, s, (const float *)w.part_max,
                  (const float *)w.part_sum, (int)p.parts, (long long)d->N, (const float *)w.target_logit, g.target, g.ignore, d->lse, rows);
    PHC_LAUNCH_AS(K_XENT_ROWS, xent_reduce_kernel, dim3(1), dim3(1024), 0, s, (const float *)rows, g.target, g.ignore, (long long)d->N,
                  d->reduction == 2 ? 1 : 0, d->reduction == 0 ? (float *)nullptr : d->loss, d->stat);
    return launch_status("phc_linear_xent_fwd");
}

int phc_linear_xent_bwd(const phc_linear_xent_desc *d, void *stream) {
    if (int rc = xent_check("phc_linear_xent_bwd", d)) return rc;
    PHC_REQUIRE(d->dloss && (!d->db || d->bias), PHC_ERR_INVALID_ARG, "phc_linear_xent_bwd: null pointer");
    PHC_REQUIRE(d->ws && aligned_to(d->ws, 256) && d->ws_bytes >= phc_linear_xent_ws_bytes(d, 1), PHC_ERR_WORKSPACE,
                "phc_linear_xent_bwd: workspace of %zu bytes, %zu needed", (size_t)d->ws_bytes, phc_linear_xent_ws_bytes(d, 1));
    if (!d->dx && !d->dW && !d->db) return PHC_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const XPlan p = make_plan(d);
    XWs w(d, p, true, d->ws);
    const int es = dtype_bytes(d->dtype);
    const long long *target = reinterpret_cast<const long long *>(d->target);
    PHC_LAUNCH_AS(K_XENT_ROWS, xent_scales_kernel, dim3(1), dim3(1024), 0, s, d->dloss, d->reduction == 0 ? 1 : 0, d->reduction == 2 ? 1 : 0,
                  (const float *)d->stat, target, (long long)d->ignore_index, (long long)d->N, w.row_scale, w.row_rel, w.top);
    // fp16 has no normal values below 6e-5, where most probabilities of a large vocabulary lie: its d are stored times 2^14
    const float d_scale = d->dtype == PHC_DTYPE_F16 ? 16384.f : 1.f;
    XPlanes X{{const_cast<void *>(d->x)}};
    long long ldx = d->ldx * es;
    if (p.pack_x) {
        pack(d, d->x, d->ldx, d->N, (int)d->D, p.Kp, w.x, s);
        X = w.x;
        ldx = p.Kp * 2;
    }
    if (d->dW) transpose(d, d->x, d->ldx, d->N, (int)d->D, p.Np, target, w.xT, s);
    for (long long v0 = 0; v0 < d->V; v0 += p.piece) {
        const long long nv = d->V - v0 < p.piece ? d->V - v0 : p.piece, nvp = round_up(nv, XT_BK);
        const char *Wv = static_cast<const char *>(d->W) + (size_t)v0 * d->ldw * es;
        XPlanes W{{const_cast<char *>(Wv)}};
        long long ldw = d->ldw * es;
        if (p.pack_w) {
            pack(d, Wv, d->ldw, nv, (int)d->D, p.Kp, w.w, s);
            W = w.w;
            ldw = p.Kp * 2;
        }
        XGemm g{};
        set_planes(p, W, X, &g);
        g.ksteps = (int)(p.Kp / XT_BK);
        g.lda = (unsigned)ldw;
        g.ldb = (unsigned)ldx;
        g.rowsA = nv;
        g.rowsB = d->N;
        g.splits = 1;
        g.bias = d->bias ? static_cast<const char *>(d->bias) + (size_t)v0 * es : nullptr;
        g.bias_f32 = p.wide;
        g.target = target;
        g.ignore = d->ignore_index;
        g.first_v = v0;
        g.vocab = d->V;
        g.lse = d->lse;
        g.row_rel = w.row_rel;
        g.d = w.dl;
        g.dT = w.dlT;
        g.ldd = nvp;
        g.lddT = p.Np;
        g.d_scale = d_scale;
        g.db_part = d->db ? w.db_part : nullptr;
        PHC_REQUIRE(gemm<XE_DLOGITS>(d, K_XENT_DLOGITS, g, s), PHC_ERR_LAUNCH, "phc_linear_xent_bwd: LDS size refused");
        if (d->db)
            sum_slabs(d, K_XENT_DW, w.db_part, nv, (int)(ceil_div(d->N, TILE) * 2), nv, w.top, static_cast<char *>(d->db) + (size_t)v0 * es, s);
        if (d->dx) {
            transpose(d, Wv, d->ldw, nv, (int)d->D, nvp, nullptr, w.wT, s);
            XGemm o{};
            set_planes(p, w.wT, w.dl, &o);
            o.ksteps = (int)(nvp / XT_BK);
            o.lda = o.ldb = (unsigned)(nvp * 2);
            o.rowsA = d->D;
            o.rowsB = d->N;
            o.splits = p.splits_dx;
            o.row_scale = w.row_scale;
            o.out_scale = 1.f / d_scale;
            o.out = w.dx_slabs ? static_cast<void *>(w.dx_slabs) : d->dx;
            o.ldo = d->D;
            o.slab = w.dx_slabs ? (long long)d->N * d->D : 0;
            o.accumulate = v0 > 0;
            o.out_dtype = d->dtype;
            o.out_vec = d->D % 4 == 0 && (w.dx_slabs || aligned_to(d->dx, 4 * es));
            PHC_REQUIRE(gemm<XE_OUT>(d, K_XENT_DX, o, s), PHC_ERR_LAUNCH, "phc_linear_xent_bwd: LDS size refused");
        }
        if (d->dW) {
            XGemm o{};
            set_planes(p, w.xT, w.dlT, &o);
            o.ksteps = (int)(p.Np / XT_BK);
            o.lda = o.ldb = (unsigned)(p.Np * 2);
            o.rowsA = d->D;
            o.rowsB = nv;
            o.splits = p.splits_dw;
            o.scale = w.top;
            o.out_scale = 1.f / d_scale;
            char *out = static_cast<char *>(d->dW) + (size_t)v0 * d->D * es;
            o.out = w.dw_slabs ? static_cast<void *>(w.dw_slabs) : out;
            o.ldo = d->D;
            o.slab = w.dw_slabs ? nv * d->D : 0;
            o.out_dtype = d->dtype;
            o.out_vec = d->D % 4 == 0 && (w.dw_slabs || aligned_to(d->dW, 4 * es));
            PHC_REQUIRE(gemm<XE_OUT>(d, K_XENT_DW, o, s), PHC_ERR_LAUNCH, "phc_linear_xent_bwd: LDS size refused");
            if (w.dw_slabs) sum_slabs(d, K_XENT_DW, w.dw_slabs, o.slab, p.splits_dw, nv * d->D, nullptr, out, s);
        }
    }
    if (d->dx && w.dx_slabs) sum_slabs(d, K_XENT_DX, w.dx_slabs, (long long)d->N * d->D, p.splits_dx, (long long)d->N * d->D, nullptr, d->dx, s);
    return launch_status("phc_linear_xent_bwd");
}

}  // extern "C"
