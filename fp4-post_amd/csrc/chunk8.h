// Eight consecutive elements of a row, bf16 or binary32, as a lane holds them: 16 or 32 bytes in registers, unpacked where they are used.
#pragma once
#include "metis_device.h"

namespace metis {

typedef uint32_t chunk_u32x4_t __attribute__((ext_vector_type(4)));
// 16 bytes with the non-temporal hint: data that nothing will find in a cache again
__device__ __forceinline__ uint4 load_streamed(const void* p, size_t at)
{
    const chunk_u32x4_t v = __builtin_nontemporal_load(static_cast<const chunk_u32x4_t*>(p) + at);
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void store_streamed(void* p, size_t at, uint4 v)
{
    __builtin_nontemporal_store((chunk_u32x4_t){v.x, v.y, v.z, v.w}, static_cast<chunk_u32x4_t*>(p) + at);
}

struct Bf16x8 {
    static constexpr int bytes = 16;
    uint4 v;
    __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, size_t chunk) { v = STREAM ? load_streamed(p, chunk) : static_cast<const uint4*>(p)[chunk]; }
    __device__ __forceinline__ float get(int j) const
    {
        const uint32_t w = (j >> 1) == 0 ? v.x : (j >> 1) == 1 ? v.y : (j >> 1) == 2 ? v.z : v.w;
        return (j & 1) ? bf16_hi(w) : bf16_lo(w);
    }
    __device__ __forceinline__ void set(const float* f)                        // rounds
    {
        v = make_uint4(rb_pair(f[0], f[1]), rb_pair(f[2], f[3]), rb_pair(f[4], f[5]), rb_pair(f[6], f[7]));
    }
    template <bool STREAM = false> __device__ __forceinline__ void store(void* p, size_t chunk) const
    {
        if constexpr (STREAM) store_streamed(p, chunk, v);
        else static_cast<uint4*>(p)[chunk] = v;
    }
};

struct F32x8 {
    static constexpr int bytes = 32;
    float4 a, b;
    __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, size_t chunk)
    {
        if constexpr (STREAM) {
            a = __builtin_bit_cast(float4, load_streamed(p, 2 * chunk));
            b = __builtin_bit_cast(float4, load_streamed(p, 2 * chunk + 1));
        } else {
            a = static_cast<const float4*>(p)[2 * chunk];
            b = static_cast<const float4*>(p)[2 * chunk + 1];
        }
    }
    __device__ __forceinline__ float get(int j) const
    {
        const float4 q = j < 4 ? a : b;
        return (j & 3) == 0 ? q.x : (j & 3) == 1 ? q.y : (j & 3) == 2 ? q.z : q.w;
    }
    __device__ __forceinline__ void set(const float* f)
    {
        a = make_float4(f[0], f[1], f[2], f[3]);
        b = make_float4(f[4], f[5], f[6], f[7]);
    }
    template <bool STREAM = false> __device__ __forceinline__ void store(void* p, size_t chunk) const
    {
        if constexpr (STREAM) {
            store_streamed(p, 2 * chunk, __builtin_bit_cast(uint4, a));
            store_streamed(p, 2 * chunk + 1, __builtin_bit_cast(uint4, b));
        } else {
            static_cast<float4*>(p)[2 * chunk] = a;
            static_cast<float4*>(p)[2 * chunk + 1] = b;
        }
    }
};

}  // namespace metis
