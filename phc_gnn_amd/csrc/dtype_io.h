// Loads and stores of the element types that the vocabulary operators take (PHC_DTYPE_*): values are fp32 in registers, 16-bit types
// only in memory.  A store rounds once, to nearest even.
#pragma once

#include "phc_common.h"

namespace phc {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

// W consecutive elements as one access (W * sizeof(T) = 2, 4, 8 or 16 bytes, naturally aligned: the callers choose W by alignment)
template <typename T, int W>
struct alignas(sizeof(T) * W) Pack {
    T v[W];
};
template <typename T, int W>
__device__ __forceinline__ void load_pack(const T *p, float (&out)[W]) {
    const Pack<T, W> q = *reinterpret_cast<const Pack<T, W> *>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = to_f32(q.v[i]);
}
template <typename T, int W>
__device__ __forceinline__ void store_pack(T *p, const float (&in)[W]) {
    Pack<T, W> q;
#pragma unroll
    for (int i = 0; i < W; ++i) q.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<Pack<T, W> *>(p) = q;
}

// (hipcc splits the store of a Pack of zeros into elements)
template <typename T, int W>
__device__ __forceinline__ void store_zeros(T *p) {
    if constexpr (sizeof(T) * W == 16) *reinterpret_cast<uint4 *>(p) = make_uint4(0, 0, 0, 0);
    else if constexpr (sizeof(T) * W == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(0, 0);
    else if constexpr (sizeof(T) * W == 4) *reinterpret_cast<unsigned *>(p) = 0;
    else *reinterpret_cast<unsigned short *>(p) = 0;
}

// ... at any element-aligned address (the hardware takes unaligned global accesses)
template <typename T, int W>
struct __attribute__((packed, aligned(sizeof(T)))) LoosePack {
    T v[W];
};
template <typename T, int W>
__device__ __forceinline__ void load_loose(const T *p, float (&out)[W]) {
    const LoosePack<T, W> q = *reinterpret_cast<const LoosePack<T, W> *>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = to_f32(q.v[i]);
}
template <typename T, int W>
__device__ __forceinline__ void store_loose(T *p, const float (&in)[W]) {
    LoosePack<T, W> q;
#pragma unroll
    for (int i = 0; i < W; ++i) q.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<LoosePack<T, W> *>(p) = q;
}

inline int dtype_bytes(int dtype) { return dtype == PHC_DTYPE_F32 ? 4 : (dtype == PHC_DTYPE_BF16 || dtype == PHC_DTYPE_F16) ? 2 : 0; }
inline bool aligned_to(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// one launch under the profiler (a scope's event pair is stamped by one dispatch)
#define PHC_LAUNCH_AS(kid, kernel, grid, block, shmem, stream, ...)      \
    do {                                                                 \
        phc::ProfScope prof_(kid, stream);                               \
        PHC_LAUNCH(kernel, grid, block, shmem, stream, __VA_ARGS__);     \
    } while (0)

inline int launch_status(const char *who) {
    const hipError_t e = hipGetLastError();
    PHC_REQUIRE(e == hipSuccess, PHC_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
    return PHC_OK;
}

// A caller's workspace cut into aligned parts; with base == nullptr it only adds up what they need.
struct Carve {
    char *base;
    size_t used = 0;
    explicit Carve(void *p) : base(static_cast<char *>(p)) {}
    template <typename T>
    T *take(size_t count) {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

}  // namespace phc
