// Softmax cross entropy of a linear map over a large vocabulary, without keeping the logits (fp32 / bf16 / fp16).
//
//   l_iv = x_i . w_v + b_v      lse_i = log sum_v exp l_iv      loss_i = lse_i - l_{i, t_i}      (0 where t_i = ignore_index)
//   d_iv = exp(l_iv - lse_i) - [v = t_i]       dx_i = g_i sum_v d_iv w_v       dw_v = sum_i g_i d_iv x_i       db_v = sum_i g_i d_iv
//
// Forward: ONE product whose tiles never leave the registers: every tile leaves the maximum and the sum of exponentials of its part
// of a row and, where the target lies in it, the target's logit; a small kernel joins the parts.  Backward keeps only lse: a piece's
// logits are computed again, become d in the tile's registers, and are written once, [row][column], for the two gradient products.  Four
// products instead of three, and no N x V tensor: both directions walk the vocabulary in pieces.
//
// Roundings.  Logits, statistics, losses, d and all sums are fp32.  For 16-bit inputs d g_i / max |g| is ROUNDED to their type, as an operand of
// the gradient products; two such terms would double two of the four products.  Against 64 bits dx and dW of bf16 are then off by 0.0018 (relative,
// over all elements) where products of unrounded d give 0.0017, those of fp16 by 0.00032 and 0.00032 (4096 x 32000 x 1024; 1021 x 30011 x 770): the
// rounding of the results themselves is most of it.  fp32 keeps 24 bits of d in three terms.  The exponentials of 16-bit inputs are the fast ones: for
// an argument x an error of |x| 2^-24 exp x, below the rounding of d.
//
// All products run through one kernel, C[m, n] = sum_k A[m, k] B[n, k], on 16-bit matrix instructions with fp32 accumulators.  An
// operand lies in memory with k contiguous, or with m (n) contiguous (W in dx; x and d in dW) and is transposed by its LDS reads.  The
// vocabulary (or the output's contiguous dimension) is always the m side: a lane then holds four consecutive m of one n, so row statistics
// are mostly in-lane and outputs are stored in 16-byte pieces.
//
// fp32 inputs: every value is split into three bf16 terms, a = h + m + l (8 bits each, |a - h - m - l| <= 2^-26 |a|), and the product
// is the sum of the six term products l h, h l, m m, m h, h m, h h (smallest first; the three left out are below 2^-25 |a b|): the same
// kernel walks six (plane of A, plane of B) pairs.  Six 16-bit products cost less than one product on the fp32 matrix instructions,
// whose rate is a sixteenth of the 16-bit one; with few rows (XT_NATIVE) it is the other way round.
//
// What bounds it: large products run at 1.25 - 1.33 PFLOP/s (8192 x 131072 x 2048 bf16: 3.5 ms forward, 0.86 - 0.96 ms each for d, dx and dW of
// a piece of 32768 columns), which is the rate of a library product of those sizes and the card's power: on zeros the same launch
// runs 20 % faster.  4096 x 32000 x 1024 bf16: 0.97 - 1.05 ms for a step.  Smaller ones: the beginning and end of each tile's k loop.
#include "dtype_io.h"

namespace phc {

constexpr int XT_ROW = 128;                    // bytes of a k-contiguous operand row per step = one line of LDS: 64 k of 16 bits, 32 of fp32
constexpr int XT_BK = 64;                      // what rows and columns of operands are padded to

// ---- rows that count --------------------------------------------------------------------------------------------------------------------
// Rows whose target is ignored cost nothing: the others are numbered in order ("packed" rows), and every product runs over those.
struct XRows {
    int *count;                // rows that count
    int *from;                 // [packed row] -> row
    int *to;                   // [row] -> packed row, -1 for the ignored ones
    int *target;               // [packed row] -> column, checked
};

__global__ __launch_bounds__(1024) void xent_rows_that_count_kernel(const long long *__restrict__ target, long long ignore, int N, long long V,
                                                                   int *err, XRows r) {
    constexpr int PER = 8;                     // a wavefront takes 8 x 64 consecutive rows at a time
    __shared__ int wsum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int base = 0; base < N; base += 1024 * PER) {
        const int i0 = base + wave * 64 * PER + lane;
        long long t[PER];
        unsigned long long m[PER];
        int mine = 0;
#pragma unroll
        for (int q = 0; q < PER; ++q) t[q] = i0 + q * 64 < N ? target[i0 + q * 64] : ignore;
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            m[q] = __ballot(t[q] != ignore);
            mine += __popcll(m[q]);
        }
        if (lane == 0) wsum[wave] = mine;
        __syncthreads();
        int at = carry;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) at += wsum[w];
            carry += wsum[w];
        }
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int i = i0 + q * 64, k = at + __popcll(m[q] & ((1ull << lane) - 1));
            const bool kept = t[q] != ignore;
            if (i < N) r.to[i] = kept ? k : -1;
            if (kept) {
                r.from[k] = i;
                r.target[k] = (int)checked_index(t[q], V, err, PHC_IDX_ERR_TARGET);
            }
            at += __popcll(m[q]);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *r.count = carry;
}

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

// W consecutive values -> the operand: as they are, or (SPLIT) in three planes
template <bool SPLIT, typename TIN, int W>
__device__ __forceinline__ void put_planes(const XPlanes &o, size_t at, const TIN (&v)[W]) {
    if constexpr (SPLIT) {
        Pack<bf16_t, W> h, m, l;
#pragma unroll
        for (int i = 0; i < W; ++i) split3(v[i], h.v[i], m.v[i], l.v[i]);
        *reinterpret_cast<Pack<bf16_t, W> *>(static_cast<bf16_t *>(o.p[0]) + at) = h;
        *reinterpret_cast<Pack<bf16_t, W> *>(static_cast<bf16_t *>(o.p[1]) + at) = m;
        *reinterpret_cast<Pack<bf16_t, W> *>(static_cast<bf16_t *>(o.p[2]) + at) = l;
    } else {
        constexpr int H = 16 / sizeof(TIN);
#pragma unroll
        for (int k = 0; k < W; k += H) {
            Pack<TIN, H> q;
#pragma unroll
            for (int i = 0; i < H; ++i) q.v[i] = v[k + i];
            *reinterpret_cast<Pack<TIN, H> *>(static_cast<TIN *>(o.p[0]) + at + k) = q;
        }
    }
}

// Rows [R, C] -> operand rows [., Cp] (8 columns a thread), columns behind C zero.  `to`: row i goes to packed row to[i]; an ignored one
// has its row of `zero` (dense [R, C], may be null) cleared instead; the packed rows behind `count` up to a whole step are zero.
template <typename TIN, bool SPLIT>
__global__ __launch_bounds__(256) void xent_pack_kernel(const TIN *__restrict__ src, long long ld, long long R, int C, int Cp,
                                                       const int *__restrict__ to, const int *__restrict__ count, TIN *__restrict__ zero, XPlanes out) {
    const int per = Cp / 8;
    const long long total = (R + (to ? XT_BK : 0)) * (long long)per;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const long long r = e / per;
        const int c = (int)(e - r * per) * 8;
        TIN v[8];
        long long at = r;
        bool fill = false;
        if (to) {
            if (r >= R) {                                         // rows behind the last one
                at = *count + (r - R);
                fill = true;
                if (at >= (*count + XT_BK - 1) / XT_BK * XT_BK) continue;
            } else {
                at = to[r];
                if (at < 0) {
                    if (zero)
                        for (int k = c; k < c + 8 && k < C; ++k) zero[r * C + k] = (TIN)0.f;
                    continue;
                }
            }
        }
        if (!fill && c + 8 <= C) {
            constexpr int H = 16 / sizeof(TIN);                   // 16-byte loads, at element-aligned addresses
#pragma unroll
            for (int k = 0; k < 8; k += H) {
                const LoosePack<TIN, H> q = *reinterpret_cast<const LoosePack<TIN, H> *>(src + r * ld + c + k);
#pragma unroll
                for (int j = 0; j < H; ++j) v[k + j] = q.v[j];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = !fill && c + k < C ? src[r * ld + c + k] : (TIN)0.f;
        }
        put_planes<SPLIT, TIN, 8>(out, (size_t)at * Cp + c, v);
    }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void xt_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int LOADS>
__device__ __forceinline__ void xt_wait_but() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory"); }      // (loads return in order)
__device__ __forceinline__ void xt_wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// Eight (four) LDS-DMA instructions: every lane's 16 bytes at base + voff[q] land at LDS byte address lds + 1024 q + 16 lane.  In asm because hipcc
// orders its builtin against every later LDS read with s_waitcnt vmcnt(0), which would drain the prefetch; the loop's own waits order
// them.  M0 is the DMA's LDS base, saved and restored inside the statement.
__device__ __forceinline__ void xt_dma(unsigned lds, const unsigned (&voff)[8], const void *base) {
    unsigned keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %6, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %7, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %8, %10\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %9, %10\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(lds), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "v"(voff[4]), "v"(voff[5]), "v"(voff[6]), "v"(voff[7]), "s"(base)
        : "memory", "scc");
}

__device__ __forceinline__ void xt_dma(unsigned lds, const unsigned (&voff)[4], const void *base) {
    unsigned keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %6\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(lds), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "s"(base)
        : "memory", "scc");
}

// one of them, for the lanes that are active
__device__ __forceinline__ void xt_dma(unsigned lds, unsigned voff, const void *base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds), "v"(voff), "s"(base)
                 : "memory");
}

// (the same in all lanes; hipcc must know it)
__device__ __forceinline__ const char *uniform(const char *p) {
    const unsigned long long v = reinterpret_cast<unsigned long long>(p);
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return reinterpret_cast<const char *>(((unsigned long long)hi << 32) | lo);
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

// fp32: 16 bytes are 4 k of each of 4 lane groups, product q takes the q-th of each (any order of k will do that both operands share)
template <>
struct Mfma16<float> {
    typedef f32x4_t frag;
    static __device__ __forceinline__ f32x4_t mul(frag a, frag b, f32x4_t c) {
#pragma unroll
        for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[q], c, 0, 0, 0);
        return c;
    }
};

typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(8))) short s16x8_t;
typedef __attribute__((address_space(3))) const char lds_char;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
typedef __attribute__((address_space(3))) const s16x8_t lds_s16x8;

// (maximum, sum of exponentials below it) of two parts of a row; a part of nothing but -inf has sum 0
__device__ __forceinline__ void xt_join(float &mx, float &sum, float m, float s) {
    const float top = fmaxf(mx, m);
    const float shift = top == -INFINITY ? 0.f : top;
    sum = sum * expf(mx - shift) + s * expf(m - shift);
    mx = top;
}

enum XEpilogue { XE_STATS, XE_DLOGITS, XE_DX, XE_DW };

struct XGemm {
    const char *A[6], *B[6];       // operand planes of each segment of the k loop
    int segments;                  // 1, or 6 for fp32 inputs
    long long K;                   // valid k (XE_DW: the count of packed rows instead)
    int kA;                        // the logits: k that A's rows hold, a whole number of 16-byte pieces (B has zeros up to K)
    unsigned lda, ldb;             // row strides in bytes
    int rowsA;                     // valid m
    int rowsB;                     // valid n (where n are the packed rows: at most)
    int colsA;                     // A held as [k][m]: readable columns
    int tilesM, tilesN, max_blocks;
    int split_k;                   // k that the number of splits goes by
    const int *count;              // packed rows
    int big, small;                // the logits' tile sizes to choose from (xt_tile); launched with each, one does the work
    // XE_STATS / XE_DLOGITS
    const void *bias;              // fp32 or the operand's type, of this piece; may be null
    const int *target;             // [packed rows]
    int first_v;                   // the piece begins here
    float *part_max, *part_sum;    // [tilesM][N]
    float *target_logit;           // [packed rows]
    const float *lse, *rel;        // [packed rows]
    XPlanes d;                     // [packed rows][ldd]
    int ldd;
    float d_scale;                 // 16-bit d are stored times this
    float *db_part;                // [tilesN * WN][rowsA] or null
    int N;
    // XE_DX / XE_DW
    const float *top, *dloss;      // g of the products: *top (finite), or (no top) *dloss over the rows that count
    int mean;
    float out_scale;
    const int *row_of;             // XE_DX: packed row -> output row
    void *out;                     // element (n, m) at n * ldo + m
    int ldo;
    float *slabs;                  // fp32 partial outputs [split][rows][ldo]
    int accumulate, pieces;
};

// 256 x 256 tiles need half the operand bytes of 128 x 128 ones per product, and fill the card only with enough of them.
__host__ __device__ inline bool xt_big(int m, int n) {
    return m > 128 && n > 128 && ((m + 255) / 256) * ((n + 255) / 256) >= 192;
}

// The tile size of the logits, by the rows that count, which the device alone knows.  small = 0 (fp32 on its own matrix instructions, which bound
// it): 64 where the last 128 rows would be at most half full (33 rows x 13565 x 1728: 116 -> 41 us), else 128.
__host__ __device__ inline int xt_tile(int big, int small, int m, int count) {
    if (big && xt_big(m, count)) return 256;
    return small ? small : ((count + 63) / 64) % 2 ? 64 : 128;
}

// what the products of d are multiplied by: the largest finite |g_i| where the rows of d carry g_i / that, else the one g
__device__ __forceinline__ float xt_scale(const float *top, const float *dloss, int mean, int count) {
    if (count <= 0) return 0.f;                                 // (a sum over nothing, whatever its factor)
    if (top) return *top;
    return mean ? *dloss / (float)count : *dloss;
}

// Work of a product over `tiles` output tiles: the k loop is split where the tiles alone do not fill the card, never below 4 steps.
__host__ __device__ inline int xt_splits(int tiles, int steps, int max_blocks) {
    int s = tiles > 0 ? max_blocks / tiles : 1;
    if (s > steps / 4) s = steps / 4;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}

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

// One operand's side of the tile: S rows (m or n) by a step's k, in LDS either as it is read k-contiguous, [S][128 bytes], or, where memory
// holds it as [k][m], as [k][S] (16 bits: with the transposing LDS read; fp32: a word for each k).  16-byte pieces of an LDS row are stored at
// piece ^ f(row), which spreads the banks of the rows that are read together.
template <typename T, int S, bool TR, bool PAIR>
struct XSide {
    static constexpr int BK = XT_ROW / sizeof(T);
    static constexpr int PIECES = TR ? S * (int)sizeof(T) / 16 : 8;     // per LDS row
    static __device__ __forceinline__ int f(int row) {
        if constexpr (TR) return sizeof(T) == 4 ? ((row >> 2) & 3) << 2 : ((row & 3) << 1) ^ (((row >> 3) & 1) << 3);
        else return PAIR ? (row & 3) | ((row >> 1) & 4) : row & 7;
    }
    // m (n) of row rho of fragment i.  PAIR: two fragments give a lane 8 consecutive m (it holds rows 4 g .. 4 g + 3 of each).
    static __device__ __forceinline__ int index(int i, int rho) {
        return PAIR ? (i >> 1) * 32 + (rho >> 2) * 8 + (i & 1) * 4 + (rho & 3) : i * 16 + rho;
    }
    // fragment i (from `first` on) of half kk of the step
    template <typename frag>
    static __device__ __forceinline__ frag read(lds_char *tile, int first, int i, int kk, int lane) {
        const int rho = lane & 15, g = lane >> 4;
        if constexpr (TR && sizeof(T) == 4) {
            const int k = kk * 16 + g * 4, piece = ((first + i * 16) >> 2) + (rho >> 2);
            lds_char *at = tile + k * (S * 4) + ((piece ^ f(k)) << 4) + (rho & 3) * 4;          // f(k) .. f(k + 3) are the same
            frag r;
#pragma unroll
            for (int q = 0; q < 4; ++q) r[q] = *(__attribute__((address_space(3))) const float *)(at + q * (S * 4));
            return r;
        } else if constexpr (TR) {
            const int k = kk * 32 + g * 8 + (rho >> 2), piece = ((first + i * 16) >> 3) + ((rho >> 1) & 1);
            lds_char *at = tile + k * (S * 2) + ((piece ^ f(k)) << 4) + (rho & 1) * 8;          // f(k + 4) = f(k)
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)at);
            const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at + 4 * (S * 2)));
            return __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int row = first + index(i, rho);
            return __builtin_bit_cast(frag, *(lds_s16x8 *)(tile + row * XT_ROW + (((kk * 4 + g) ^ f(row)) << 4)));
        }
    }
};

// One workgroup a tile (or a split of its k).  Loads go straight to LDS two steps ahead; 16-byte LDS reads without bank conflicts; the matrix pipes
// are busy 0.52 - 0.63 of the cycles.  256 x 256 by 8 wavefronts reads half the operand bytes of 128 x 128 by 4 (14.5 against 17.1 ms for
// 8192 x 131072 x 2048).  Tried without gain: raised wave priority, all of a step's reads first, workgroups that stay for more tiles.
template <typename T, int EPI, bool WIDE, int WM, int WN, int FM, int FN, int NB>
__global__ __launch_bounds__(WM *WN * 64, 2) void xent_gemm_kernel(XGemm a) {
    typedef typename Mfma16<T>::frag frag;
    constexpr int NW = WM * WN, TM = WM * FM * 16, TN = WN * FN * 16;
    constexpr bool A_TR = EPI == XE_DX || EPI == XE_DW, B_TR = EPI == XE_DW, PAIR = EPI == XE_DLOGITS;
    typedef XSide<T, TM, A_TR, PAIR> SA;
    typedef XSide<T, TN, B_TR, false> SB;
    constexpr int BK = SA::BK, PER = 16 / sizeof(T);            // k of a step, elements of a 16-byte piece
    constexpr int LOADS = (TM + TN) / 8 / NW;                   // LDS-DMA instructions per wavefront and step (1 KiB each)
    static_assert(FN <= FM, "a group of products for each n fragment's read");
    static_assert((TM / 8) % LOADS == 0, "a wavefront loads one operand");
    constexpr unsigned BUF = (TM + TN) * XT_ROW;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // what there is to do goes by the rows that count
    const int count = *a.count;
    if ((EPI == XE_STATS || EPI == XE_DLOGITS) && xt_tile(a.big, a.small, a.rowsA, count) != TM) return;
    const int rowsB = EPI == XE_DW ? a.rowsB : count;
    const int tilesN = (rowsB + TN - 1) / TN, tiles = a.tilesM * tilesN;
    const int ksteps = EPI == XE_DW ? (count + BK - 1) / BK : (int)((a.K + BK - 1) / BK);
    const int steps = a.segments * ksteps;
    int splits = 1;
    if constexpr (EPI == XE_DX || EPI == XE_DW) splits = xt_splits(tiles, a.segments * (EPI == XE_DW ? ksteps : a.split_k / BK), a.max_blocks);
    const int block = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    if (block >= tiles * splits) return;
    const int split = block / tiles;
    int tm, tn;
    xt_tile_of(block - split * tiles, a.tilesM, tilesN, tm, tn);
    const int s0 = (int)((long long)steps * split / splits), n_steps = (int)((long long)steps * (split + 1) / splits) - s0;

    // loader
    const bool loads_a = wave * LOADS < TM / 8;
    const unsigned ld = loads_a ? a.lda : a.ldb;
    const bool tr = loads_a ? A_TR : B_TR;
    const int dma0 = wave * LOADS - (loads_a ? 0 : TM / 8);     // this wavefront's first instruction of its operand
    const unsigned k_bytes = tr ? BK * ld : XT_ROW;
    const unsigned lds_wave = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)smem + wave * LOADS * 1024);
    // memory rows behind an operand's end repeat its last one: their results are dropped, or the other operand has zeros there
    const int rows = tr ? (EPI == XE_DW ? 0x7fffffff : (int)a.K) : loads_a ? a.rowsA : rowsB;

    const int at0 = loads_a ? tm * TM : tn * TN;
    auto offset = [&](int q, int first, int limit) -> unsigned {
        if (tr) {
            const int per = loads_a ? SA::PIECES : SB::PIECES, row = (dma0 + q) * (64 / per) + lane / per;
            const int f = XSide<T, TM, true, false>::f(row);
            const int col = min(at0 + ((lane % per) ^ f) * PER, (loads_a ? a.colsA : (int)(a.ldb / sizeof(T))) - PER);
            return (unsigned)min(row, limit - 1 - first) * ld + (unsigned)col * (unsigned)sizeof(T);
        }
        const int row = (dma0 + q) * 8 + (lane >> 3);
        const int f = loads_a ? XSide<T, TM, false, PAIR>::f(row) : XSide<T, TN, false, false>::f(row);
        return (unsigned)min(row, limit - 1 - first) * ld + ((lane & 7) ^ f) * 16;
    };
    unsigned voff[LOADS];
#pragma unroll
    for (int q = 0; q < LOADS; ++q) voff[q] = offset(q, tr ? 0 : at0, tr ? BK : rows);
    // the step that is loaded next
    int seg = __builtin_amdgcn_readfirstlane(s0 / (ksteps > 0 ? ksteps : 1)), kst = __builtin_amdgcn_readfirstlane(s0 - seg * ksteps);
    auto plane = [&]() { return uniform((loads_a ? a.A[seg] : a.B[seg]) + (tr ? 0 : (size_t)at0 * ld) + (size_t)kst * k_bytes); };
    const char *base = n_steps > 0 ? plane() : nullptr;
    auto issue = [&](int buf) {
        if (A_TR && EPI != XE_DW && tr && (kst + 1) * BK > rows) {           // the last rows of k
            unsigned last[LOADS];
#pragma unroll
            for (int q = 0; q < LOADS; ++q) last[q] = offset(q, kst * BK, rows);
            xt_dma(lds_wave + buf * BUF, last, base);
        } else if (!A_TR && loads_a && (kst + 1) * BK > a.kA) {              // A's rows end inside the step: zeros behind them
            for (int q = 0; q < LOADS; ++q) {
                const int piece = (lane & 7) ^ XSide<T, TM, false, PAIR>::f((dma0 + q) * 8 + (lane >> 3));
                if (kst * BK + piece * PER < a.kA) xt_dma(lds_wave + buf * BUF + q * 1024, voff[q], base);
                else *reinterpret_cast<uint4 *>(smem + wave * LOADS * 1024 + buf * BUF + q * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
            }
        } else {
            xt_dma(lds_wave + buf * BUF, voff, base);
        }
        base += k_bytes;
        if (++kst == ksteps) {
            kst = 0;
            if (++seg < a.segments) base = plane();
        }
    };
    // What the epilogue of the logits needs, {target, logsumexp, g / max g} of the tile's rows and the bias of its columns: loaded by a
    // thread each in front of the first steps (loads return in order), kept in LDS behind the buffers.
    constexpr bool LOGITS = EPI == XE_STATS || EPI == XE_DLOGITS;
    typedef std::conditional_t<WIDE, float, T> TB;              // the inputs' type
    struct Row {
        int hit;
        float lse, rel;
    };
    static_assert(!LOGITS || NW * 64 >= TM + TN, "a thread for each row and column of the tile");
    Row *const row_meta = reinterpret_cast<Row *>(smem + NB * BUF + WM * TN * sizeof(float2));             // [TN]
    float *const bias_meta = reinterpret_cast<float *>(row_meta + TN);                                    // [TM]
    Row my_row{-1, 0.f, 0.f};
    float my_bias = 0.f;
    if constexpr (LOGITS) {
        if ((int)threadIdx.x < TN) {
            const int n = tn * TN + threadIdx.x;
            const int hit = n < count ? a.target[n] - a.first_v : -1;
            if (n < count) my_row = Row{hit < a.rowsA ? hit : -1, EPI == XE_DLOGITS ? a.lse[n] : 0.f, EPI == XE_DLOGITS && a.rel ? a.rel[n] : 1.f};
        } else if ((int)threadIdx.x < TN + TM) {
            const int m = tm * TM + threadIdx.x - TN;
            my_bias = m >= a.rowsA ? -INFINITY : a.bias ? to_f32(static_cast<const TB *>(a.bias)[m]) : 0.f;     // (columns behind the vocabulary: exp 0)
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (n_steps > b) issue(b);
    if constexpr (LOGITS) {
        if ((int)threadIdx.x < TN) row_meta[threadIdx.x] = my_row;
        else if ((int)threadIdx.x < TN + TM) bias_meta[threadIdx.x - TN] = my_bias;
    }

    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int ma = wm * FM * 16, nb = wn * FN * 16;
    auto half = [&](lds_char *tile, int kk, const frag (&a0)[FM], const frag (&b0)[FN], frag (&a1)[FM], frag (&b1)[FN], bool load, int buf = 0) {
        if (load) issue(buf);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            if (i < FN) b1[i] = SB::template read<frag>(tile + TM * XT_ROW, nb, i, kk, lane);
            a1[i] = SA::template read<frag>(tile, ma, i, kk, lane);
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = Mfma16<T>::mul(a0[i], b0[j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);          // (hipcc would gather the reads behind the products)
        }
    };

    // NB LDS buffers, two halves of a step.  While the products of one half run, the fragments of the next are read; the one barrier of a
    // step stands between them: behind it the next step's buffer is complete, and this step's buffer, read to its end, is loaded anew with the
    // step NB further on.
    lds_char *lds = (lds_char *)smem;
    if (n_steps > 0) {
        frag fa[2][FM], fb[2][FN];
        if (NB > 2 && n_steps >= NB) xt_wait_but<(NB - 1) * LOADS>();
        else xt_wait_all();
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[0][j] = SB::template read<frag>(lds + TM * XT_ROW, nb, j, 0, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[0][i] = SA::template read<frag>(lds, ma, i, 0, lane);
        int slot = 0;
        for (int t = 0; t < n_steps; ++t) {
            const int next = NB == 2 ? slot ^ 1 : slot + 1 == NB ? 0 : slot + 1;
            lds_char *cur = lds + slot * BUF, *nxt = lds + next * BUF;
            half(cur, 1, fa[0], fb[0], fa[1], fb[1], false);
            __builtin_amdgcn_sched_barrier(0);
            if (NB > 2 && t + NB <= n_steps) xt_wait_but<(NB - 2) * LOADS>();       // step t + 1; the NB - 2 behind it may still be under way
            else xt_wait_all();
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            // (behind the last step the fragments are read once more and not used)
            half(nxt, 0, fa[1], fb[1], fa[0], fb[0], t + NB < n_steps, slot);
            __builtin_amdgcn_sched_barrier(0);
            slot = next;
        }
    }

    // a lane holds m = m_of(i) + r (r = 0 .. 3) of n = n0 + 16 j
    const int fr = lane & 15, fg = lane >> 4;
    const int m_base = tm * TM + ma, n0 = tn * TN + nb + fr;
    auto m_of = [&](int i) { return m_base + SA::index(i, fg * 4); };
    if constexpr (LOGITS) {
        const Row *row_of = row_meta + nb + fr;
        auto bias = [&](int i, int r) { return bias_meta[ma + SA::index(i, fg * 4) + r]; };
        if constexpr (EPI == XE_STATS) {
            float mx[FN], sum[FN];
            int hit[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                hit[j] = row_of[j * 16].hit;
                mx[j] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float b = bias(i, r);
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        const float l = acc[i][j][r] + b;
                        acc[i][j][r] = l;
                        mx[j] = fmaxf(mx[j], l);
                        if (hit[j] == m_of(i) + r) a.target_logit[n0 + j * 16] = l;
                    }
                }
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                mx[j] = fmaxf(mx[j], __shfl_xor(mx[j], 16));
                mx[j] = fmaxf(mx[j], __shfl_xor(mx[j], 32));
                const float shift = mx[j] == -INFINITY ? 0.f : mx[j];       // nothing but -inf: every exponential is 0
                sum[j] = 0.f;
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[j] += sizeof(TB) == 4 ? expf(acc[i][j][r] - shift) : __expf(acc[i][j][r] - shift);
                sum[j] += __shfl_xor(sum[j], 16);
                sum[j] += __shfl_xor(sum[j], 32);
            }
            // the wavefronts along m, through LDS behind the buffers (a barrier that orders LDS alone)
            float2 *meet = reinterpret_cast<float2 *>(smem + NB * BUF);      // [WM][TN]
            if (fg == 0)
#pragma unroll
                for (int j = 0; j < FN; ++j) meet[wm * TN + nb + j * 16 + fr] = make_float2(mx[j], sum[j]);
            xt_wait_lds();
            __builtin_amdgcn_s_barrier();
            for (int c = threadIdx.x; c < TN; c += NW * 64) {
                const int n = tn * TN + c;
                if (n >= rowsB) continue;
                float m = meet[c].x, s = meet[c].y;
#pragma unroll
                for (int w = 1; w < WM; ++w) {
                    const float2 o = meet[w * TN + c];
                    xt_join(m, s, o.x, o.y);
                }
                a.part_max[(size_t)tm * a.N + n] = m;
                a.part_sum[(size_t)tm * a.N + n] = s;
            }
        } else {
            const int n_end = (count + XT_BK - 1) / XT_BK * XT_BK;          // zero rows up to a whole step of the weight gradient's k
            Row row[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) row[j] = row_of[j * 16];
#pragma unroll
            for (int i = 0; i < FM; i += 2) {
                float b[8], db[8] = {};
#pragma unroll
                for (int e = 0; e < 8; ++e) b[e] = bias(i + e / 4, e % 4);
                const int m0 = m_of(i);                                      // 8 consecutive columns of two fragments
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    const int n = n0 + j * 16;
                    TB d[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float l = acc[i + e / 4][j][e % 4] + b[e];
                        const float p = sizeof(TB) == 4 ? expf(l - row[j].lse) : __expf(l - row[j].lse);
                        const float v = n < count && m0 + e < a.rowsA ? (p - (row[j].hit == m0 + e ? 1.f : 0.f)) * row[j].rel : 0.f;
                        db[e] += v;
                        d[e] = (TB)(v * a.d_scale);
                    }
                    if (n < n_end && m0 < a.ldd) put_planes<WIDE, TB, 8>(a.d, (size_t)n * a.ldd + m0, d);
                }
                if (a.db_part)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float v = db[e];
#pragma unroll
                        for (int x = 1; x < 16; x <<= 1) v += __shfl_xor(v, x);
                        if (fr == 0 && m0 + e < a.rowsA) a.db_part[(size_t)(tn * WN + wn) * a.rowsA + m0 + e] = v;
                    }
                __builtin_amdgcn_sched_barrier(0);                           // (registers: one pair of fragments at a time)
            }
        }
    } else {
        typedef std::conditional_t<WIDE, float, T> TO;
        const float s = a.out_scale * xt_scale(a.top, a.dloss, a.mean, count);
        const bool final = splits == 1 && (EPI == XE_DW || a.pieces == 1);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + j * 16;
            if (n >= rowsB) continue;
            const size_t row = final && EPI == XE_DX ? a.row_of[n] : n;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int m = m_of(i);
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r] * s;
                if (final) {
                    TO *o = static_cast<TO *>(a.out) + row * a.ldo + m;
                    if (m + 4 <= a.rowsA) store_loose<TO, 4>(o, v);
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < a.rowsA) o[r] = from_f32<TO>(v[r]);
                } else {
                    float *o = a.slabs + ((size_t)split * rowsB + row) * a.ldo + m;
                    if (m + 4 <= a.rowsA) {
                        if (a.accumulate) {
                            float p[4];
                            load_loose<float, 4>(o, p);
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[r] += p[r];
                        }
                        store_loose<float, 4>(o, v);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < a.rowsA) o[r] = a.accumulate ? o[r] + v[r] : v[r];
                    }
                }
            }
        }
    }
}

// ---- a few rows -------------------------------------------------------------------------------------------------------------------------
// Up to 64 rows (scoring a few tokens): W is read once and everything else is small, so the launch is W's bytes at the memory's rate and
// latency.  A workgroup takes 16 FM columns at a time; its four wavefronts share the k and meet in LDS.  W and x go from memory straight into
// matrix operands: lane (rho, g) loads 16 bytes of row rho at k = g * 16 bytes, the same for both operands, so any order of k inside a step
// will do.  Two sets of registers: a step is loaded while the one before is multiplied.  fp32 on the fp32 matrix instructions (4 k each).
// bf16, V = 131072, D = 2048 (537 MB): 1 / 16 / 32 / 64 rows 110 / 119 / 133 / 170 us = 4.9 .. 3.2 TB/s (x comes from L2 for every group, as
// many bytes as W at 64 rows); fp32: 214 / 231 / 266 / 405 us (at 64 rows half of it matrix instructions).
struct XFew {
    const void *W, *x, *bias;
    long long ldw, ldx;            // elements
    int N, V, D;
    const long long *target;
    long long ignore;
    int *err;
    float *part_max, *part_sum;    // [workgroup][16 NF]
    float *target_logit;           // [row]
};

template <typename T>
struct XFewStep : Mfma16<T> {
    static constexpr int PER = 16 / sizeof(T), K = 4 * PER;      // k of a lane group, of an operand
};

// 16 bytes at an element-aligned address.  ODD: 16-bit rows that may begin at odd elements are loaded as the words that hold them (each of which
// holds an element of the row) and shifted: accesses that are not word-aligned take several times as long.
template <typename T, bool ODD, typename frag>
__device__ __forceinline__ frag few_load(const T *p) {
    if constexpr (ODD) {
        const bool odd = reinterpret_cast<uintptr_t>(p) & 2;
        const unsigned *at = reinterpret_cast<const unsigned *>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)2);
        const LoosePack<unsigned, 4> w = *reinterpret_cast<const LoosePack<unsigned, 4> *>(at);
        const unsigned last = at[odd ? 4 : 3], shift = odd ? 16 : 0;
        LoosePack<unsigned, 4> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = __builtin_amdgcn_alignbit(e < 3 ? w.v[e + 1] : last, w.v[e], shift);
        return __builtin_bit_cast(frag, o);
    } else {
        return __builtin_bit_cast(frag, *reinterpret_cast<const LoosePack<T, 16 / sizeof(T)> *>(p));
    }
}
// the first `left` elements of it, zeros behind
template <typename T, typename frag>
__device__ __forceinline__ frag few_load_part(const T *p, int left) {
    LoosePack<T, 16 / sizeof(T)> q = {};
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); ++e)
        if (e < left) q.v[e] = p[e];
    return __builtin_bit_cast(frag, q);
}

template <typename T, int FM, int NF, bool ODD>
__global__ __launch_bounds__(256) void xent_few_kernel(XFew a) {
    typedef XFewStep<T> S;
    typedef typename S::frag frag;
    constexpr int COLS = FM * 16, AHEAD = FM == 1 ? (NF > 2 ? 2 : 4) : NF > 1 ? 1 : 2;                       // steps of a set of registers
    __shared__ f32x4_t meet[4][FM][64];
    __shared__ float2 top[FM][NF * 16];
    // (the wavefront's number is the same in all lanes, and hipcc must know it: under a condition that it takes for a lane's it may narrow EXEC and go on,
    // and the matrix instructions do not look at EXEC)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fg = lane >> 4;
    int v0 = blockIdx.x * COLS;
    const T *w[FM], *x[NF];
    auto columns = [&]() {
#pragma unroll
        for (int i = 0; i < FM; ++i) w[i] = static_cast<const T *>(a.W) + (long long)min(v0 + i * 16 + fr, a.V - 1) * a.ldw + fg * S::PER;
    };
    columns();
#pragma unroll
    for (int j = 0; j < NF; ++j) x[j] = static_cast<const T *>(a.x) + (long long)min(j * 16 + fr, a.N - 1) * a.ldx + fg * S::PER;
    f32x4_t acc[FM][NF];
    // a wavefront takes every fourth step; two sets of registers: one is loaded while the other is multiplied
    const int full = a.D / S::K;
    auto load = [&](frag (&fw)[AHEAD][FM], frag (&fx)[AHEAD][NF], int step) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (step + 4 * u >= full) break;
            const long long k = (long long)(step + 4 * u) * S::K;
#pragma unroll
            for (int i = 0; i < FM; ++i) fw[u][i] = few_load<T, ODD, frag>(w[i] + k);
#pragma unroll
            for (int j = 0; j < NF; ++j) fx[u][j] = few_load<T, ODD, frag>(x[j] + k);
        }
    };
    auto multiply = [&](const frag (&fw)[FM], const frag (&fx)[NF]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) acc[i][j] = S::mul(fw[i], fx[j], acc[i][j]);
    };
    auto multiply_all = [&](const frag (&fw)[AHEAD][FM], const frag (&fx)[AHEAD][NF], int step) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (step + 4 * u < full) multiply(fw[u], fx[u]);
    };
    frag fw0[AHEAD][FM], fx0[AHEAD][NF], fw1[AHEAD][FM], fx1[AHEAD][NF];
    int hit[NF];
#pragma unroll
    for (int j = 0; j < NF; ++j) {
        const long long t = j * 16 + fr < a.N ? a.target[j * 16 + fr] : a.ignore;
        hit[j] = t == a.ignore ? -1 : (int)checked_index(t, a.V, blockIdx.x == 0 ? a.err : nullptr, PHC_IDX_ERR_TARGET);
    }
    float row_max = -INFINITY, row_sum = 0.f;                   // of row threadIdx.x, over this workgroup's columns
    load(fw0, fx0, wave);
    while (v0 < a.V) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        for (int step = wave; step < full; step += 8 * AHEAD) {
            load(fw1, fx1, step + 4 * AHEAD);
            __builtin_amdgcn_sched_barrier(0);
            multiply_all(fw0, fx0, step);
            load(fw0, fx0, step + 8 * AHEAD);
            __builtin_amdgcn_sched_barrier(0);
            multiply_all(fw1, fx1, step + 4 * AHEAD);
        }
        if (full * S::K < a.D && wave == full % 4) {            // the rest of the rows
            const int left = min(max(a.D - full * S::K - fg * S::PER, 0), S::PER);
#pragma unroll
            for (int i = 0; i < FM; ++i) fw0[0][i] = few_load_part<T, frag>(w[i] + full * S::K, left);
#pragma unroll
            for (int j = 0; j < NF; ++j) fx0[0][j] = few_load_part<T, frag>(x[j] + full * S::K, left);
            multiply(fw0[0], fx0[0]);
        }
        const int first = v0 + wave * 16 + fg * 4;              // this lane's columns
        v0 += (int)gridDim.x * COLS;
        if (v0 < a.V) {                                         // the next ones are under way while these end
            columns();
            load(fw0, fx0, wave);
        }
        // wavefront w < FM: columns 16 w ..; a lane holds 4 columns of row fr.  16 rows at a time: LDS for all of them would halve the
        // wavefronts on a CU
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < FM; ++i) meet[wave][i][lane] = acc[i][j];
            __syncthreads();
            if (wave >= FM) continue;
            f32x4_t l = meet[0][wave][lane];
#pragma unroll
            for (int q = 1; q < 4; ++q) l += meet[q][wave][lane];
            const int n = j * 16 + fr;
            float mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int v = first + r;
                if (v >= a.V) {
                    l[r] = -INFINITY;
                    continue;
                }
                if (a.bias) l[r] += to_f32(static_cast<const T *>(a.bias)[v]);
                mx = fmaxf(mx, l[r]);
                if (hit[j] == v) a.target_logit[n] = l[r];
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float shift = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += sizeof(T) == 4 ? expf(l[r] - shift) : __expf(l[r] - shift);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (fg == 0) top[wave][n] = make_float2(mx, sum);
        }
        __syncthreads();
        if (threadIdx.x < NF * 16) {
#pragma unroll
            for (int q = 0; q < FM; ++q) xt_join(row_max, row_sum, top[q][threadIdx.x].x, top[q][threadIdx.x].y);
        }
    }
    if (threadIdx.x < NF * 16) {
        a.part_max[(size_t)blockIdx.x * NF * 16 + threadIdx.x] = row_max;
        a.part_sum[(size_t)blockIdx.x * NF * 16 + threadIdx.x] = row_sum;
    }
}

// joins the workgroups' parts; losses, their reduction and the state for the backward: one workgroup, rows in the lanes of a wavefront
__global__ __launch_bounds__(1024) void xent_few_finish_kernel(XFew a, int parts, int cols, int reduction, XRows rows, float *__restrict__ lse,
                                                              float *__restrict__ loss) {
    // the maximum first, then the sums against it: one exponential for each part.  (The fast one: an error of |x| 2^-24 in exp x, weighted with
    // exp x, moves the logarithm by less than log(parts) 2^-24.)
    __shared__ float sm[1024], ss[1024];
    const int c = threadIdx.x % cols, group = threadIdx.x / cols, groups = 1024 / cols;
    constexpr int AHEAD = 8;                                         // parts in flight
    float mx = -INFINITY, sum = 0.f;
    for (int p = group; p < parts; p += groups * AHEAD) {
        float m[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) m[q] = p + q * groups < parts ? a.part_max[(size_t)(p + q * groups) * cols + c] : -INFINITY;
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) mx = fmaxf(mx, m[q]);
    }
    sm[threadIdx.x] = mx;
    for (int half = groups / 2; half >= 1; half /= 2) {              // (groups is a power of two)
        __syncthreads();
        if (group < half) sm[threadIdx.x] = mx = fmaxf(mx, sm[threadIdx.x + half * cols]);
    }
    __syncthreads();
    mx = sm[c];
    const float shift = mx == -INFINITY ? 0.f : mx;
    for (int p = group; p < parts; p += groups * AHEAD) {
        float m[AHEAD], t[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const bool in = p + q * groups < parts;
            m[q] = in ? a.part_max[(size_t)(p + q * groups) * cols + c] : -INFINITY;
            t[q] = in ? a.part_sum[(size_t)(p + q * groups) * cols + c] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) sum += t[q] * __expf(m[q] - shift);
    }
    ss[threadIdx.x] = sum;
    for (int half = groups / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (group < half) ss[threadIdx.x] = sum += ss[threadIdx.x + half * cols];
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int n = threadIdx.x;
    const long long t = n < a.N ? a.target[n] : a.ignore;
    const bool kept = t != a.ignore;
    const unsigned long long m = __ballot(kept);
    float l = 0.f;
    if (kept) {
        const float e = sm[n] + logf(ss[n]);
        l = e - a.target_logit[n];
        const int at = __popcll(m & ((1ull << n) - 1));
        rows.from[at] = n;
        rows.to[n] = at;
        rows.target[at] = (int)safe_index(t, a.V);
        lse[at] = e;
    } else if (n < a.N) {
        rows.to[n] = -1;
    }
    if (n == 0) *rows.count = __popcll(m);
    if (reduction == PHC_REDUCE_NONE) {
        if (n < a.N) loss[n] = l;
        return;
    }
    double s = (double)l;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if (n == 0) loss[0] = (float)(reduction == PHC_REDUCE_MEAN ? s / (double)__popcll(m) : s);
}

// ---- rows -------------------------------------------------------------------------------------------------------------------------------
// The kernels over all rows that are one workgroup (the numbering above, the sum of the losses, the scales of g) are latency: 5 us each up to some
// thousand rows.  They count where rows are very many and the vocabulary small: 2^20 rows, 1000 columns of 64 bf16: 0.43, 0.29 - 0.35 and 1.5 ms
// of 5.0 ms for a step.
//
// A workgroup joins the parts of 16 rows: 64 lane groups share the parts, then one adds them up.  nv: columns of the piece; `run` carries (maximum, sum)
// from piece to piece, the last one ends the rows.
__global__ __launch_bounds__(1024) void xent_rows_kernel(const float *__restrict__ part_max, const float *__restrict__ part_sum, int nv, int big, int small, int N,
                                                        const int *__restrict__ count, const float *__restrict__ target_logit,
                                                        const int *__restrict__ from, float2 *__restrict__ run, int first, int last, float *__restrict__ lse,
                                                        float *__restrict__ row_loss, float *__restrict__ loss) {
    __shared__ float sm[16][16], ss[16][16];
    const int c = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int n = blockIdx.x * 16 + c, kept = *count;
    if (blockIdx.x * 16 >= kept) return;
    const int tile = xt_tile(big, small, nv, kept), parts = (nv + tile - 1) / tile;
    float mx = -INFINITY, sum = 0.f;
    if (n < kept)
        for (int p = group; p < parts; p += 64) xt_join(mx, sum, part_max[(size_t)p * N + n], part_sum[(size_t)p * N + n]);
    // lane groups of a wavefront, then the wavefronts
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) xt_join(mx, sum, __shfl_xor(mx, d), __shfl_xor(sum, d));
    if ((threadIdx.x & 63) < 16) {
        sm[threadIdx.x >> 6][c] = mx;
        ss[threadIdx.x >> 6][c] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    mx = -INFINITY, sum = 0.f;
    for (int w = group; w < 16; w += 4) xt_join(mx, sum, sm[w][c], ss[w][c]);
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) xt_join(mx, sum, __shfl_xor(mx, d), __shfl_xor(sum, d));
    if (group == 0 && n < kept) {
        if (!first) xt_join(mx, sum, run[n].x, run[n].y);
        if (!last) {
            run[n] = make_float2(mx, sum);
            return;
        }
        const float l = mx + logf(sum);
        lse[n] = l;
        row_loss[n] = l - target_logit[n];
        if (loss) loss[from[n]] = l - target_logit[n];
    }
}

// sum of the rows' losses -> out[0] = sum or mean; per row (out is null): zeros for the ignored rows
__global__ __launch_bounds__(1024) void xent_reduce_kernel(const float *__restrict__ row_loss, const int *__restrict__ count, const int *__restrict__ to,
                                                          int N, int mean, float *__restrict__ out, float *__restrict__ loss) {
    __shared__ double red[16];
    if (loss) {
        for (int i = threadIdx.x; i < N; i += 1024)
            if (to[i] < 0) loss[i] = 0.f;
        return;
    }
    const int kept = *count;
    double s = 0.0;
    for (int i = threadIdx.x; i < kept; i += 1024) s += (double)row_loss[i];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += red[w];
        out[0] = (float)(mean ? s / (double)kept : s);          // (no row counts: the mean of nothing is NaN)
    }
}

// A g_i of its own for every packed row: top = max |g_i| of the finite ones, rel = g_i / top (what the rows of d carry; top goes to the products'
// outputs).  An infinite or NaN g_i stays in its row of d: as the factor of every output it would reach all rows of dx.
__global__ __launch_bounds__(1024) void xent_scales_kernel(const float *__restrict__ dloss, const int *__restrict__ count,
                                                          const int *__restrict__ from, float *__restrict__ rel, float *__restrict__ top) {
    __shared__ float red[16];
    const int kept = *count;
    float m = 0.f;
    for (int i = threadIdx.x; i < kept; i += 1024) {
        const float g = fabsf(dloss[from[i]]);
        if (g < INFINITY) m = fmaxf(m, g);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int w = 0; w < 16; ++w) m = fmaxf(m, red[w]);
    if (m == 0.f) m = 1.f;
    if (threadIdx.x == 0) *top = m;
    for (int i = threadIdx.x; i < kept; i += 1024) rel[i] = dloss[from[i]] / m;
}

// The splits' partial outputs in order.  dx: rows go back to their places; dW: nothing to do where one split wrote the result.
template <typename T>
__global__ __launch_bounds__(256) void xent_sum_slabs_kernel(const float *__restrict__ slabs, const int *__restrict__ count, int rows_static, int tilesM,
                                                            int TN, int split_steps, int bk, int segments, int max_blocks, int D, int pieces,
                                                            const int *__restrict__ row_of, T *__restrict__ out) {
    const int rows = row_of ? *count : rows_static;
    const int steps = segments * (row_of ? split_steps : (*count + bk - 1) / bk);
    const int n = xt_splits(tilesM * ((rows + TN - 1) / TN), steps, max_blocks);
    if (n == 1 && (!row_of || pieces == 1)) return;
    const size_t total = (size_t)rows * D;
    const int per = (D + 3) / 4;                                  // 4 elements a thread
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < (long long)rows * per; e += (long long)gridDim.x * 256) {
        const int r = (int)(e / per), c = (int)(e - (long long)r * per) * 4;
        const float *src = slabs + (size_t)r * D + c;
        T *dst = out + (size_t)(row_of ? row_of[r] : r) * D + c;
        if (c + 4 <= D) {
            float v[4];
            load_loose<float, 4>(src, v);
            for (int s = 1; s < n; ++s) {
                float o[4];
                load_loose<float, 4>(src + s * total, o);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += o[k];
            }
            store_loose<T, 4>(dst, v);
        } else {
            for (int k = 0; c + k < D; ++k) {
                float v = src[k];
                for (int s = 1; s < n; ++s) v += src[s * total + k];
                dst[k] = from_f32<T>(v);
            }
        }
    }
}

// db[v] = top sum over the row tiles' partial sums, in order: 16 columns a workgroup, 16 lane groups share the parts
template <typename T>
__global__ __launch_bounds__(256) void xent_db_kernel(const float *__restrict__ part, const int *__restrict__ count, int nv, int big, int small,
                                                     const float *__restrict__ top, const float *__restrict__ dloss, int mean, T *__restrict__ db) {
    __shared__ float meet[16][16];
    const int c = threadIdx.x & 15, group = threadIdx.x >> 4, v = blockIdx.x * 16 + c;
    const int tile = xt_tile(big, small, nv, *count), n = (*count + tile - 1) / tile * (tile == 256 ? 4 : 2);
    float s = 0.f;
    if (v < nv)
        for (int i = group; i < n; i += 16) s += part[(size_t)i * nv + v];
    meet[group][c] = s;
    __syncthreads();
    if (group == 0 && v < nv) {
        for (int w = 1; w < 16; ++w) s += meet[w][c];
        db[v] = from_f32<T>(n > 0 ? s * xt_scale(top, dloss, mean, *count) : 0.f);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
static long long round_up(long long v, long long m) { return (v + m - 1) / m * m; }
static long long ceil_div(long long v, long long m) { return (v + m - 1) / m; }

// A piece's d, and its rows of W where they are laid out.  Pieces are for memory alone: at N = 8192, V = 131072, D = 2048 (bf16) pieces of 8192,
// 16384, 32768 and all columns took 14.4, 14.3, 14.3 and 14.3 ms, smaller ones cost (4096: 15.8 ms), so that 2048 columns are the least.
constexpr long long XT_PIECE_BYTES = 512ll << 20;

// Tiles of 256 x 256 by 8 wavefronts (one workgroup on a CU) or 128 x 128 by 4 (two)
struct Tile256 {
    static constexpr int WM = 2, WN = 4, FM = 8, FN = 4, SIZE = 256, BLOCKS = 256, NB = 2;
};
struct Tile128 {
    static constexpr int WM = 2, WN = 2, FM = 4, FN = 4, SIZE = 128, BLOCKS = 512, NB = 2;
};

// Small problems: four times the workgroups of Tile128 for the logits, which do not split their k loop.  A step is short beside a load's way: three
// buffers (213 x 3320 x 3989 fp16 forward 55 -> 44 us, 100 x 8000 x 2048 bf16 30 -> 25 us), of which three workgroups fit a CU (four buffers:
// 200 x 10000 x 1024 bf16 25 -> 29 us).
struct Tile64 {
    static constexpr int WM = 2, WN = 2, FM = 2, FN = 2, SIZE = 64, BLOCKS = 512, NB = 3;
};

struct XPlan {
    bool wide;                 // fp32 inputs in three planes
    int planes, segments, bytes, bk;       // bytes of an operand's element, k of a step
    long long Kp, Np;
    long long cols;            // columns of a piece of the forward
    long long piece, pieces;   // of the backward
    bool pack_w;
    bool big_fwd, big_d;       // 256 x 256 tiles, if enough rows count (known on the device alone)
    int small_fwd, small_d;    // the other tile size, 0: 64 or 128, as xt_tile says
    bool big_dx, big_dw;       // 256 x 256 tiles
    long long wcols;           // readable columns of W's operand rows
};

// dx and dW split their k loop: few large tiles do
static bool big_split(long long m, long long n) {
    return m > 128 && n > 128 && ceil_div(m, 256) * ceil_div(n, 256) >= 32;
}

static int small_tile(long long m, long long n, bool native) { return ceil_div(m, 128) * ceil_div(n, 128) < 192 ? 64 : native ? 0 : 128; }

// Rows up to which fp32 goes without planes.  A step in us without and with them, all rows counting: N = 256: 13565 x 1728 488 and 561, 32000 x 512
// 337 and 367, 50000 x 1024 993 and 990; N = 128: 285 and 417, 223 and 273, 569 and 770.  With 15 % counting, N = 256: 220 and 446, 166 and 236, 406
// and 662.  (Planes cost 20 bytes of traffic for each element of W and save 8 N products at 130 instead of 200 TFLOP/s, on tiles of 128 rows.)
constexpr long long XT_NATIVE = 256;

static XPlan make_plan(const phc_linear_xent_desc *d) {
    XPlan p;
    // fp32: three planes from XT_NATIVE rows on; below, laying W out costs more than the fp32 matrix instructions lose
    p.wide = d->dtype == PHC_DTYPE_F32 && d->N > XT_NATIVE;
    p.planes = p.wide ? 3 : 1;
    p.segments = p.wide ? 6 : 1;
    p.bytes = p.wide ? 2 : dtype_bytes(d->dtype);
    p.bk = XT_ROW / p.bytes;
    p.Kp = round_up(d->D, p.bk);
    p.Np = round_up(d->N, XT_BK);
    // W is read where it lies when its rows are whole 16-byte pieces, 16-byte aligned (laid out anew, 192 x 31584 x 3448 bf16 took 163 us forward
    // and 514 a step instead of 76 and 367)
    p.pack_w = p.wide || d->D * p.bytes % 16 || d->ldw * p.bytes % 16 || !aligned_to(d->W, 16);
    p.wcols = p.pack_w ? p.Kp : d->D;
    const long long w_column = p.pack_w ? p.Kp * p.bytes * p.planes : 0;     // bytes of W's layout
    long long piece = XT_PIECE_BYTES / (p.bytes * p.planes * d->N + w_column) / 256 * 256;
    if (piece < 2048) piece = 2048;
    if (d->piece > 0) piece = round_up(d->piece < d->V ? d->piece : d->V, 64);
    if (piece >= d->V) piece = round_up(d->V, 64);
    p.pieces = ceil_div(d->V, piece);
    p.piece = d->piece > 0 ? piece : round_up(ceil_div(d->V, p.pieces), 64);
    p.pieces = ceil_div(d->V, p.piece);
    // The forward's pieces are for memory alone too: the row statistics of all tiles (8 bytes for each row and 128 columns) and W's layout
    p.cols = XT_PIECE_BYTES / (w_column + ceil_div(d->N, 16)) / 256 * 256;
    if (p.cols < 2048) p.cols = 2048;
    if (d->piece > 0 && p.pack_w && p.cols > piece) p.cols = piece;
    if (p.cols >= d->V) p.cols = d->V;
    else if (d->piece <= 0) p.cols = round_up(ceil_div(d->V, ceil_div(d->V, p.cols)), 256);
    p.big_fwd = p.bytes == 2 && xt_big((int)p.cols, (int)d->N);
    p.big_d = p.bytes == 2 && xt_big((int)p.piece, (int)d->N);
    p.small_fwd = small_tile(p.cols, d->N, p.bytes == 4);
    p.small_d = small_tile(p.piece, d->N, p.bytes == 4);
    p.big_dx = p.bytes == 2 && big_split(d->D, d->N);
    p.big_dw = p.bytes == 2 && big_split(d->D, p.piece);
    return p;
}

static size_t slab_floats(long long rows, long long D, bool big, bool keeps) {
    // splits exist only while tiles * splits stays within the blocks of one launch
    const size_t tile = big ? Tile256::SIZE : Tile128::SIZE, blocks = big ? Tile256::BLOCKS : Tile128::BLOCKS;
    const size_t most = blocks * tile * tile;
    const size_t all = (size_t)rows * D;
    return keeps ? (all > most ? all : most) : most;
}

// what the forward hands to the backward
struct XState {
    XRows rows{};
    float *lse = nullptr;
    size_t bytes;
    XState(long long N, void *state) {
        Carve c(state);
        rows.count = c.take<int>(1);
        rows.from = c.take<int>(N);
        rows.to = c.take<int>(N);
        rows.target = c.take<int>(N);
        lse = c.take<float>(N);
        bytes = c.used;
    }
};

struct XWs {
    XPlanes x{}, w{}, dl{};
    float *part_max = nullptr, *part_sum = nullptr, *target_logit = nullptr, *row_loss = nullptr;
    float2 *run = nullptr;
    float *rel = nullptr, *top = nullptr, *dx_slabs = nullptr, *dw_slabs = nullptr, *db_part = nullptr;
    size_t bytes;
    XWs(const phc_linear_xent_desc *d, const XPlan &p, bool backward, void *ws) {
        Carve c(ws);
        auto planes = [&](XPlanes &o, size_t count) {
            for (int i = 0; i < p.planes; ++i) o.p[i] = c.take<char>(count * p.bytes);
        };
        planes(x, (size_t)p.Np * p.Kp);
        if (p.pack_w) planes(w, (size_t)(backward ? p.piece : p.cols) * p.Kp);
        if (!backward) {
            const size_t parts = ceil_div(p.cols, p.small_fwd ? p.small_fwd : 64);
            if (p.cols < d->V) run = c.take<float2>(d->N);
            part_max = c.take<float>(parts * d->N);
            part_sum = c.take<float>(parts * d->N);
            target_logit = c.take<float>(d->N);
            row_loss = c.take<float>(d->N);
        } else {
            rel = c.take<float>(d->N);
            top = c.take<float>(1);
            planes(dl, (size_t)p.Np * p.piece);
            if (d->dx) dx_slabs = c.take<float>(slab_floats(d->N, d->D, p.big_dx, p.pieces > 1));
            if (d->dW) dw_slabs = c.take<float>(slab_floats(p.piece, d->D, p.big_dw, false));
            if (d->db) db_part = c.take<float>((size_t)(ceil_div(d->N, 64) * 2 + 2) * p.piece);          // (large tiles: 4 parts of 256 rows, small ones 2 of 128 or 64)
        }
        bytes = c.used;
    }
};

static unsigned flat_grid(long long n) {
    const long long b = ceil_div(n, 256);
    return (unsigned)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

template <typename T, bool SPLIT>
static void pack_as(const void *src, long long ld, long long R, long long C, long long Cp, const XRows *rows, void *zero, const XPlanes &out, hipStream_t s) {
    PHC_LAUNCH_AS(K_XENT_LAYOUT, (xent_pack_kernel<T, SPLIT>), dim3(flat_grid((R + (rows ? XT_BK : 0)) * (Cp / 8))), dim3(256), 0, s, static_cast<const T *>(src),
                  ld, R, (int)C, (int)Cp, rows ? (const int *)rows->to : (const int *)nullptr, rows ? (const int *)rows->count : (const int *)nullptr,
                  static_cast<T *>(zero), out);
}
static void pack(const XPlan &p, int dtype, const void *src, long long ld, long long R, long long C, const XRows *rows, void *zero, const XPlanes &out,
                 hipStream_t s) {
    if (p.wide) pack_as<float, true>(src, ld, R, C, p.Kp, rows, zero, out, s);
    else if (dtype == PHC_DTYPE_F32) pack_as<float, false>(src, ld, R, C, p.Kp, rows, zero, out, s);
    else if (dtype == PHC_DTYPE_BF16) pack_as<bf16_t, false>(src, ld, R, C, p.Kp, rows, zero, out, s);
    else pack_as<f16_t, false>(src, ld, R, C, p.Kp, rows, zero, out, s);
}

static void set_planes(const XPlan &p, const XPlanes &A, const XPlanes &B, XGemm *g) {
    static const int ia[6] = {2, 0, 1, 1, 0, 0}, ib[6] = {0, 2, 1, 0, 1, 0};
    g->segments = p.segments;
    for (int i = 0; i < 6; ++i) {
        g->A[i] = static_cast<const char *>(A.p[p.wide ? ia[i] : 0]);
        g->B[i] = static_cast<const char *>(B.p[p.wide ? ib[i] : 0]);
    }
}

constexpr long long XT_LINE = 1 << 21;         // workgroups in x: a dimension of a launch holds less than 2^32 threads

template <typename T, int EPI, bool WIDE, typename TILE>
static bool launch_gemm(int kid, XGemm &g, hipStream_t s) {
    constexpr int LDS = TILE::NB * 2 * TILE::SIZE * XT_ROW + TILE::SIZE * (TILE::WM * (int)sizeof(float2) + 12 + 4);      // buffers, the wavefronts' meeting place, rows and columns
    g.tilesM = (int)ceil_div(g.rowsA, TILE::SIZE);
    g.tilesN = (int)ceil_div(g.rowsB, TILE::SIZE);
    g.max_blocks = TILE::BLOCKS;
    auto kernel = xent_gemm_kernel<T, EPI, WIDE, TILE::WM, TILE::WN, TILE::FM, TILE::FN, TILE::NB>;
    if (!ensure_dynamic_lds(kernel, LDS)) return false;
    // a workgroup for each tile; dx, dW: or for each split of them
    long long blocks = (long long)g.tilesM * g.tilesN;
    if ((EPI == XE_DX || EPI == XE_DW) && blocks < TILE::BLOCKS) blocks = TILE::BLOCKS;
    const long long line = blocks < XT_LINE ? blocks : XT_LINE;
    PHC_LAUNCH_AS(kid, kernel, dim3((unsigned)line, (unsigned)ceil_div(blocks, line)), dim3(TILE::WM * TILE::WN * 64), LDS, s, g);
    return true;
}
template <typename T, int EPI, bool WIDE>
static bool launch_tile(int kid, int tile, XGemm &g, hipStream_t s) {
    if constexpr (!(sizeof(T) == 4))
        if (tile == 256) return launch_gemm<T, EPI, WIDE, Tile256>(kid, g, s);
    if constexpr (EPI == XE_STATS || EPI == XE_DLOGITS)
        if (tile == 64) return launch_gemm<T, EPI, WIDE, Tile64>(kid, g, s);
    return launch_gemm<T, EPI, WIDE, Tile128>(kid, g, s);
}
template <int EPI>
static int gemm(const XPlan &p, int dtype, int kid, int tile, XGemm &g, hipStream_t s) {
    const bool ok = p.wide ? launch_tile<bf16_t, EPI, true>(kid, tile, g, s) : dtype == PHC_DTYPE_F32 ? launch_tile<float, EPI, false>(kid, tile, g, s)
                    : dtype == PHC_DTYPE_BF16 ? launch_tile<bf16_t, EPI, false>(kid, tile, g, s) : launch_tile<f16_t, EPI, false>(kid, tile, g, s);
    PHC_REQUIRE(ok, PHC_ERR_LAUNCH, "phc_linear_xent: the runtime refused the kernel's LDS size");
    return PHC_OK;
}
// The logits, launched with every tile size that the rows that count may ask for: all but one launch end at once (4 us each; 13 568 rows of which
// 15 % count against 5000 columns would fill 160 of the 256 CUs with large tiles).
template <int EPI>
static int gemm_logits(const XPlan &p, int dtype, int kid, bool big, int small, XGemm &g, hipStream_t s) {
    g.big = big;
    g.small = small;
    if (small != 128)
        if (int rc = gemm<EPI>(p, dtype, kid, 64, g, s)) return rc;
    if (small != 64)
        if (int rc = gemm<EPI>(p, dtype, kid, 128, g, s)) return rc;
    return big ? gemm<EPI>(p, dtype, kid, 256, g, s) : PHC_OK;
}

template <typename T>
static void sum_slabs_as(int kid, const float *slabs, const XGemm &g, int tile, int bk, int pieces, void *out, hipStream_t s) {
    PHC_LAUNCH_AS(kid, (xent_sum_slabs_kernel<T>), dim3(flat_grid((long long)g.rowsB * ceil_div(g.ldo, 4))), dim3(256), 0, s, slabs, g.count, g.rowsB, g.tilesM, tile,
                  g.split_k / bk, bk, g.segments, g.max_blocks, g.ldo, pieces, g.row_of, static_cast<T *>(out));
}
static void sum_slabs(int dtype, int kid, const float *slabs, const XGemm &g, int tile, int bk, int pieces, void *out, hipStream_t s) {
    if (dtype == PHC_DTYPE_F32) sum_slabs_as<float>(kid, slabs, g, tile, bk, pieces, out, s);
    else if (dtype == PHC_DTYPE_BF16) sum_slabs_as<bf16_t>(kid, slabs, g, tile, bk, pieces, out, s);
    else sum_slabs_as<f16_t>(kid, slabs, g, tile, bk, pieces, out, s);
}

template <typename T>
static void db_as(const float *part, const XRows &r, int nv, int big, int small, const float *top, const float *dloss, int mean, void *db, hipStream_t s) {
    PHC_LAUNCH_AS(K_XENT_DW, (xent_db_kernel<T>), dim3((unsigned)ceil_div(nv, 16)), dim3(256), 0, s, part, (const int *)r.count, nv, big, small, top, dloss, mean,
                  static_cast<T *>(db));
}

constexpr int XT_FEW = 64;
static bool few_rows(const phc_linear_xent_desc *d) { return d->N <= XT_FEW; }

// Workgroups: two on a CU, each with every 512th group of 64 columns (64 rows, V = 100000, D = 1024, bf16: 512, 768, 1024 and one workgroup for
// each group took 68, 79, 75 and 81 us; fewer parts to join, and the next group's loads run beside a group's end).
constexpr long long XT_FEW_BLOCKS = 512;
// Columns of a group: 64, or 16 where groups of 64 are few (a CU's own rate bounds them), against more reads of x.  fp32 1193 x 2848: 1 row 29 -> 14 us,
// 64 rows 57 -> 35 us; bf16 5000 x 4096: 1 row 23 -> 17 us, 64 rows 39 -> 48 us.
static int few_columns(long long V, long long N) { return ceil_div(V, 64) < (N <= 16 ? 128 : 40) ? 16 : 64; }
static long long few_parts(long long V, long long N) {
    const long long groups = ceil_div(V, few_columns(V, N));
    return groups < XT_FEW_BLOCKS ? groups : XT_FEW_BLOCKS;
}

template <typename T, int NF, bool ODD>
static void launch_few_as(const XFew &f, hipStream_t s) {
    const dim3 grid((unsigned)few_parts(f.V, f.N));
    if (few_columns(f.V, f.N) == 16) PHC_LAUNCH_AS(K_XENT_LOGITS, (xent_few_kernel<T, 1, NF, ODD>), grid, dim3(256), 0, s, f);
    else PHC_LAUNCH_AS(K_XENT_LOGITS, (xent_few_kernel<T, 4, NF, ODD>), grid, dim3(256), 0, s, f);
}
template <typename T, bool ODD>
static void launch_few_rows(const XFew &f, hipStream_t s) {
    if (f.N <= 16) launch_few_as<T, 1, ODD>(f, s);
    else if (f.N <= 32) launch_few_as<T, 2, ODD>(f, s);
    else launch_few_as<T, 4, ODD>(f, s);
}
template <typename T>
static void launch_few(const XFew &f, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if ((f.ldw | f.ldx) & 1 || !aligned_to(f.W, 4) || !aligned_to(f.x, 4)) return launch_few_rows<T, true>(f, s);
    launch_few_rows<T, false>(f, s);
}

static int forward_few(const phc_linear_xent_desc *d, const XState &st, hipStream_t s) {
    const int cols = d->N <= 16 ? 16 : d->N <= 32 ? 32 : 64, parts = (int)few_parts(d->V, d->N);
    Carve c(d->ws);
    XFew f{d->W, d->x, d->bias, d->ldw, d->ldx, (int)d->N, (int)d->V, (int)d->D, reinterpret_cast<const long long *>(d->target), d->ignore_index, err_word()};
    f.part_max = c.take<float>((size_t)parts * cols);
    f.part_sum = c.take<float>((size_t)parts * cols);
    f.target_logit = c.take<float>(cols);
    if (d->dtype == PHC_DTYPE_F32) launch_few<float>(f, s);
    else if (d->dtype == PHC_DTYPE_BF16) launch_few<bf16_t>(f, s);
    else launch_few<f16_t>(f, s);
    PHC_LAUNCH_AS(K_XENT_ROWS, xent_few_finish_kernel, dim3(1), dim3(1024), 0, s, f, parts, cols, d->reduction, st.rows, st.lse, d->loss);
    return launch_status("phc_linear_xent_fwd");
}

static int xent_check(const char *who, const phc_linear_xent_desc *d) {
    PHC_REQUIRE(d, PHC_ERR_INVALID_ARG, "%s: null descriptor", who);
    PHC_REQUIRE(dtype_bytes(d->dtype), PHC_ERR_INVALID_ARG, "%s: unknown dtype %d", who, d->dtype);
    PHC_REQUIRE(d->reduction >= 0 && d->reduction <= 2, PHC_ERR_INVALID_ARG, "%s: unknown reduction %d", who, d->reduction);
    PHC_REQUIRE(d->N >= 1 && d->V >= 1 && d->D >= 1, PHC_ERR_INVALID_ARG, "%s: N=%lld V=%lld D=%lld", who, (long long)d->N, (long long)d->V, (long long)d->D);
    // (x is read with 64-bit addresses, a tile's rows of W with 32-bit offsets)
    PHC_REQUIRE(d->N <= (1 << 22) && d->V <= (1 << 22) && d->D <= (1 << 20) && d->ldx <= (1ll << 38) && d->ldw <= (1 << 22), PHC_ERR_UNSUPPORTED,
                "%s: N=%lld, V=%lld, D=%lld or the row stride of x (%lld) or W (%lld) is beyond 2^22, 2^22, 2^20, 2^38, 2^22", who, (long long)d->N, (long long)d->V,
                (long long)d->D, (long long)d->ldx, (long long)d->ldw);
    PHC_REQUIRE(d->ldx >= d->D && d->ldw >= d->D, PHC_ERR_INVALID_ARG, "%s: row stride below the row length", who);
    PHC_REQUIRE(d->piece >= 0, PHC_ERR_INVALID_ARG, "%s: piece %lld", who, (long long)d->piece);
    PHC_REQUIRE(d->x && d->W && d->target && d->state && aligned_to(d->state, 256), PHC_ERR_INVALID_ARG, "%s: null pointer, or a state that is not 256-byte aligned", who);
    return PHC_OK;
}

}  // namespace phc

using namespace phc;

extern "C" {

size_t phc_linear_xent_state_bytes(int64_t N) { return N < 0 || N > (1 << 22) ? 0 : XState(N, nullptr).bytes; }

size_t phc_linear_xent_ws_bytes(const phc_linear_xent_desc *d, int backward) {
    if (xent_check("phc_linear_xent_ws_bytes", d)) return 0;
    if (!backward && few_rows(d)) return (size_t)few_parts(d->V, d->N) * 64 * 2 * sizeof(float) + 2048;
    return XWs(d, make_plan(d), backward != 0, nullptr).bytes + 256;
}

int phc_linear_xent_fwd(const phc_linear_xent_desc *d, void *stream) {
    if (int rc = xent_check("phc_linear_xent_fwd", d)) return rc;
    PHC_REQUIRE(d->loss, PHC_ERR_INVALID_ARG, "phc_linear_xent_fwd: null pointer");
    PHC_REQUIRE(d->ws && aligned_to(d->ws, 256) && d->ws_bytes >= phc_linear_xent_ws_bytes(d, 0), PHC_ERR_WORKSPACE,
                "phc_linear_xent_fwd: workspace of %zu bytes, %zu needed", (size_t)d->ws_bytes, phc_linear_xent_ws_bytes(d, 0));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const XState st(d->N, d->state);
    if (few_rows(d)) return forward_few(d, st, s);
    const XPlan p = make_plan(d);
    XWs w(d, p, false, d->ws);
    const int es = dtype_bytes(d->dtype), N = (int)d->N;
    PHC_LAUNCH_AS(K_XENT_ROWS, xent_rows_that_count_kernel, dim3(1), dim3(1024), 0, s, reinterpret_cast<const long long *>(d->target),
                  (long long)d->ignore_index, N, (long long)d->V, err_word(), st.rows);
    pack(p, d->dtype, d->x, d->ldx, d->N, d->D, &st.rows, nullptr, w.x, s);
    float *loss = d->reduction == PHC_REDUCE_NONE ? d->loss : nullptr;
    for (long long v0 = 0; v0 < d->V; v0 += p.cols) {
        const int nv = (int)(d->V - v0 < p.cols ? d->V - v0 : p.cols);
        const char *Wv = static_cast<const char *>(d->W) + (size_t)v0 * d->ldw * es;
        XPlanes W{{const_cast<char *>(Wv)}};
        if (p.pack_w) {
            pack(p, d->dtype, Wv, d->ldw, nv, d->D, nullptr, nullptr, w.w, s);
            W = w.w;
        }
        XGemm g{};
        set_planes(p, W, w.x, &g);
        g.K = p.Kp;
        g.kA = (int)p.wcols;
        g.lda = (unsigned)(p.pack_w ? p.Kp * p.bytes : d->ldw * es);
        g.ldb = (unsigned)(p.Kp * p.bytes);
        g.rowsA = nv;
        g.rowsB = g.N = N;
        g.count = st.rows.count;
        g.bias = d->bias ? static_cast<const char *>(d->bias) + (size_t)v0 * es : nullptr;
        g.target = st.rows.target;
        g.first_v = (int)v0;
        g.part_max = w.part_max;
        g.part_sum = w.part_sum;
        g.target_logit = w.target_logit;
        if (int rc = gemm_logits<XE_STATS>(p, d->dtype, K_XENT_LOGITS, p.big_fwd, p.small_fwd, g, s)) return rc;
        PHC_LAUNCH_AS(K_XENT_ROWS, xent_rows_kernel, dim3((unsigned)ceil_div(N, 16)), dim3(1024), 0, s, (const float *)w.part_max, (const float *)w.part_sum, nv,
                      p.big_fwd ? 1 : 0, p.small_fwd, N, g.count, (const float *)w.target_logit, (const int *)st.rows.from, w.run, v0 == 0 ? 1 : 0,
                      v0 + p.cols >= d->V ? 1 : 0, st.lse, w.row_loss, loss);
    }
    PHC_LAUNCH_AS(K_XENT_ROWS, xent_reduce_kernel, dim3(1), dim3(1024), 0, s, (const float *)w.row_loss, (const int *)st.rows.count, (const int *)st.rows.to, N,
                  d->reduction == PHC_REDUCE_MEAN ? 1 : 0, loss ? (float *)nullptr : d->loss, loss);
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
    const XState st(d->N, d->state);
    const int es = dtype_bytes(d->dtype), N = (int)d->N;
    const bool per_row = d->reduction == PHC_REDUCE_NONE;
    const float *rel = per_row ? w.rel : nullptr, *top = per_row ? w.top : nullptr;
    const int mean = d->reduction == PHC_REDUCE_MEAN ? 1 : 0;
    if (per_row)
        PHC_LAUNCH_AS(K_XENT_ROWS, xent_scales_kernel, dim3(1), dim3(1024), 0, s, d->dloss, (const int *)st.rows.count, (const int *)st.rows.from, w.rel, w.top);
    pack(p, d->dtype, d->x, d->ldx, d->N, d->D, &st.rows, d->dx, w.x, s);
    // fp16 has no normal values below 6e-5, where most probabilities of a large vocabulary lie: its d are stored times 2^14.  With a g_i for each row
    // what is below 2^-28 of the largest |g| is then rounded to multiples of 2^-38 of it, in rows of small g_i too.
    const float d_scale = d->dtype == PHC_DTYPE_F16 ? 16384.f : 1.f;
    XGemm o{};                                                   // (the last piece's dx product: its splits are joined at the end)
    for (long long v0 = 0; v0 < d->V; v0 += p.piece) {
        const int nv = (int)(d->V - v0 < p.piece ? d->V - v0 : p.piece), nvp = (int)round_up(nv, XT_BK);
        const char *Wv = static_cast<const char *>(d->W) + (size_t)v0 * d->ldw * es;
        XPlanes W{{const_cast<char *>(Wv)}};
        if (p.pack_w) {
            pack(p, d->dtype, Wv, d->ldw, nv, d->D, nullptr, nullptr, w.w, s);
            W = w.w;
        }
        const unsigned ldw = (unsigned)(p.pack_w ? p.Kp * p.bytes : d->ldw * es);
        XGemm g{};
        set_planes(p, W, w.x, &g);
        g.K = p.Kp;
        g.kA = (int)p.wcols;
        g.lda = ldw;
        g.ldb = (unsigned)(p.Kp * p.bytes);
        g.rowsA = nv;
        g.rowsB = g.N = N;
        g.count = st.rows.count;
        g.bias = d->bias ? static_cast<const char *>(d->bias) + (size_t)v0 * es : nullptr;
        g.target = st.rows.target;
        g.first_v = (int)v0;
        g.lse = st.lse;
        g.rel = rel;
        g.d = w.dl;
        g.ldd = nvp;
        g.d_scale = d_scale;
        g.db_part = d->db ? w.db_part : nullptr;
        if (int rc = gemm_logits<XE_DLOGITS>(p, d->dtype, K_XENT_DLOGITS, p.big_d, p.small_d, g, s)) return rc;
        if (d->db) {
            char *db = static_cast<char *>(d->db) + (size_t)v0 * es;
            if (d->dtype == PHC_DTYPE_F32) db_as<float>(w.db_part, st.rows, nv, p.big_d, p.small_d, top, d->dloss, mean, db, s);
            else if (d->dtype == PHC_DTYPE_BF16) db_as<bf16_t>(w.db_part, st.rows, nv, p.big_d, p.small_d, top, d->dloss, mean, db, s);
            else db_as<f16_t>(w.db_part, st.rows, nv, p.big_d, p.small_d, top, d->dloss, mean, db, s);
        }
        if (d->dx) {
            o = XGemm{};
            set_planes(p, W, w.dl, &o);
            o.K = nv;
            o.split_k = (int)p.piece;
            o.lda = ldw;
            o.ldb = (unsigned)(nvp * p.bytes);
            o.rowsA = (int)d->D;
            o.colsA = (int)p.wcols;
            o.rowsB = N;
            o.count = st.rows.count;
            o.top = top;
            o.dloss = d->dloss;
            o.mean = mean;
            o.out_scale = 1.f / d_scale;
            o.row_of = st.rows.from;
            o.out = d->dx;
            o.ldo = (int)d->D;
            o.slabs = w.dx_slabs;
            o.accumulate = v0 > 0;
            o.pieces = (int)p.pieces;
            if (int rc = gemm<XE_DX>(p, d->dtype, K_XENT_DX, p.big_dx ? 256 : 128, o, s)) return rc;
        }
        if (d->dW) {
            XGemm q{};
            set_planes(p, w.x, w.dl, &q);
            q.lda = (unsigned)(p.Kp * p.bytes);
            q.ldb = (unsigned)(nvp * p.bytes);
            q.rowsA = (int)d->D;
            q.colsA = (int)p.Kp;
            q.rowsB = nv;
            q.count = st.rows.count;
            q.top = top;
            q.dloss = d->dloss;
            q.mean = mean;
            q.out_scale = 1.f / d_scale;
            q.out = static_cast<char *>(d->dW) + (size_t)v0 * d->D * es;
            q.ldo = (int)d->D;
            q.slabs = w.dw_slabs;
            q.pieces = 1;
            if (int rc = gemm<XE_DW>(p, d->dtype, K_XENT_DW, p.big_dw ? 256 : 128, q, s)) return rc;
            if ((long long)q.tilesM * q.tilesN * 2 <= q.max_blocks)
                sum_slabs(d->dtype, K_XENT_DW, w.dw_slabs, q, p.big_dw ? 256 : 128, p.bk, 1, q.out, s);
        }
    }
    if (d->dx) sum_slabs(d->dtype, K_XENT_DX, w.dx_slabs, o, p.big_dx ? 256 : 128, p.bk, (int)p.pieces, d->dx, s);
    return launch_status("phc_linear_xent_bwd");
}

}  // extern "C"
