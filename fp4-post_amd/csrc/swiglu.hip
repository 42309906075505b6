// silu(gate) * up between two projections of an MLP, and its gradients:
//   a = g s u,   s = 1 / (1 + exp(-g));     du = da g s,   dg = da u s (1 + g (1 - s))
// in binary32, each result rounded once.  Elementwise and bound by memory: 6 (10) bytes an element in bf16.  gate and up are rows of their own strides
// (the halves of one product's rows as they are; 4096 x 18944 bf16 in halves 72 us forward and 123 backward, 6.4 and 6.3 TB/s); a lane takes eight elements where rows, strides and addresses allow whole 16-byte accesses, else one.
#include "chunk8.h"
#include "metis_host.h"

namespace metis {

constexpr uint64_t kStreamBytes = (uint64_t)256 << 20;         // the memory-side cache

// The sigmoid of a bf16 value needs no more than the hardware's exponential and reciprocal; a binary32 one takes the library's and a true division.
template <bool F32> __device__ __forceinline__ float sigmoid(float g)
{
    if constexpr (F32) return 1.0f / (1.0f + expf(-g));
    else return __builtin_amdgcn_rcpf(1.0f + __expf(-g));
}
template <bool F32> __device__ __forceinline__ float gated(float g, float u) { return g * sigmoid<F32>(g) * u; }
template <bool F32> __device__ __forceinline__ void gated_back(float g, float u, float da, float& dg, float& du)
{
    const float s = sigmoid<F32>(g);
    dg = da * u * s * fmaf(g, 1.0f - s, 1.0f);
    du = da * (g * s);
}

// position of unit `at` (eight elements or one) in rows of `per` units and `ld` units' stride
template <class I> __device__ __forceinline__ size_t strided(I at, uint32_t per, uint64_t ld) { return ld == per ? at : at / per * ld + at % per; }

// STREAM: more bytes than the memory-side cache holds (kStreamBytes) go by it with the non-temporal hint, and the backward takes two chunks a lane at once.
// 4096 x 18944 bf16, halves of one product: 87 us forward and 148 backward without either, 72 and 123 with both; of 1024 rows, which stay in the cache, 19 and 31 us with or without
// the hint, 512 x 8960 8.4 us without and 9.4 with it.
template <class C, bool STREAM>
__global__ __launch_bounds__(256) void swiglu_kernel(const void* __restrict__ gate, uint64_t ldg, const void* __restrict__ up, uint64_t ldu, uint32_t total,
                                                     uint32_t per, void* __restrict__ out)
{
    constexpr bool F32 = C::bytes == 32;
    const uint32_t at = blockIdx.x * 256u + threadIdx.x;
    if (at >= total) return;
    C g, u, o;
    g.template load<STREAM>(gate, strided(at, per, ldg));
    u.template load<STREAM>(up, strided(at, per, ldu));
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = gated<F32>(g.get(j), u.get(j));
    o.set(f);
    o.template store<STREAM>(out, at);
}

template <class C, bool STREAM>
__global__ __launch_bounds__(256) void swiglu_backward_kernel(const void* __restrict__ gate, uint64_t ldg, const void* __restrict__ up, uint64_t ldu,
                                                              const void* __restrict__ grad, uint32_t total, uint32_t per, void* __restrict__ ggate,
                                                              void* __restrict__ gup)
{
    constexpr bool F32 = C::bytes == 32;
    constexpr int N = STREAM ? 2 : 1;                          // chunks of a lane, a workgroup's width apart
    const uint32_t first = blockIdx.x * 256u * N + threadIdx.x;
    C g[N], u[N], a[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t at = first + 256u * k;
        if (at >= total) break;
        g[k].template load<STREAM>(gate, strided(at, per, ldg));
        u[k].template load<STREAM>(up, strided(at, per, ldu));
        a[k].template load<STREAM>(grad, at);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t at = first + 256u * k;
        if (at >= total) break;
        float dg[8], du[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) gated_back<F32>(g[k].get(j), u[k].get(j), a[k].get(j), dg[j], du[j]);
        g[k].set(dg);
        u[k].set(du);
        g[k].template store<STREAM>(ggate, at);
        u[k].template store<STREAM>(gup, at);
    }
}

template <bool F32> __device__ __forceinline__ float element(const void* p, size_t at)
{
    if constexpr (F32) return static_cast<const float*>(p)[at];
    else return bf16_lo(static_cast<const uint16_t*>(p)[at]);
}
template <bool F32> __device__ __forceinline__ void put_element(void* p, size_t at, float v)
{
    if constexpr (F32) static_cast<float*>(p)[at] = v;
    else static_cast<uint16_t*>(p)[at] = (uint16_t)bf16_bits(v);
}
template <bool F32, bool BACK>
__global__ __launch_bounds__(256) void swiglu_single_kernel(const void* __restrict__ gate, uint64_t ldg, const void* __restrict__ up, uint64_t ldu,
                                                            const void* __restrict__ grad, uint64_t total, uint32_t per, void* __restrict__ out, void* __restrict__ gup)
{
    for (uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256u) {
        const float g = element<F32>(gate, strided(at, per, ldg)), u = element<F32>(up, strided(at, per, ldu));
        if constexpr (BACK) {
            float dg, du;
            gated_back<F32>(g, u, element<F32>(grad, at), dg, du);
            put_element<F32>(out, at, dg);
            put_element<F32>(gup, at, du);
        } else {
            put_element<F32>(out, at, gated<F32>(g, u));
        }
    }
}

// grad == nullptr: out = silu(gate) up; else out, gup are the gradients of gate and up
int swiglu(const void* gate, int64_t ldg, const void* up, int64_t ldu, const void* grad, int64_t rows, int64_t cols, int dtype, bool back, void* out, void* gup,
           hipStream_t st)
{
    if (rows < 0 || cols < 0 || ldg < 0 || ldu < 0 || (dtype != METIS_DTYPE_BF16 && dtype != METIS_DTYPE_F32)) return METIS_E_ARG;
    if (rows == 0 || cols == 0) return METIS_OK;
    if (cols > INT32_MAX || rows > ((int64_t)1 << 46) / cols || (rows > 1 && (ldg < cols || ldu < cols))) return METIS_E_ARG;
    if (!gate || !up || !out || (back && (!grad || !gup))) return METIS_E_ARG;
    const bool f32 = dtype == METIS_DTYPE_F32;
    const uintptr_t size = f32 ? 4 : 2, any = (uintptr_t)gate | (uintptr_t)up | (uintptr_t)grad | (uintptr_t)out | (uintptr_t)gup;
    if (any % size) return METIS_E_ARG;
    if (rows == 1) ldg = ldu = cols;
    const bool whole = cols % 8 == 0 && ldg % 8 == 0 && ldu % 8 == 0 && any % 16 == 0;
    const uint64_t unit = whole ? 8 : 1, total = (uint64_t)rows * (uint64_t)cols / unit;
    if (whole && total > (uint64_t)INT32_MAX) return METIS_E_TOO_LARGE;         // (units are counted in 32 bits)
    const bool stream = whole && total * 8 * size * (back ? 5 : 3) > kStreamBytes;
    const uint64_t lane = back && stream ? 2 : 1, need = (total + 256 * lane - 1) / (256 * lane), cap = (uint64_t)device_cus() * 16;
    const dim3 grid((unsigned)(whole || need < cap ? need : cap)), block(256);
    const uint32_t per = (uint32_t)(cols / unit);
    const uint64_t lg = (uint64_t)ldg / unit, lu = (uint64_t)ldu / unit;
#define METIS_SGF(C, S) hipLaunchKernelGGL((swiglu_kernel<C, S>), grid, block, 0, st, gate, lg, up, lu, (uint32_t)total, per, out)
#define METIS_SGB(C, S) hipLaunchKernelGGL((swiglu_backward_kernel<C, S>), grid, block, 0, st, gate, lg, up, lu, grad, (uint32_t)total, per, out, gup)
    if (whole && !back) {
        if (f32) { if (stream) METIS_SGF(F32x8, true); else METIS_SGF(F32x8, false); }
        else { if (stream) METIS_SGF(Bf16x8, true); else METIS_SGF(Bf16x8, false); }
    } else if (whole) {
        if (f32) { if (stream) METIS_SGB(F32x8, true); else METIS_SGB(F32x8, false); }
        else { if (stream) METIS_SGB(Bf16x8, true); else METIS_SGB(Bf16x8, false); }
#undef METIS_SGF
#undef METIS_SGB
    } else {
#define METIS_SG(F, K) hipLaunchKernelGGL((swiglu_single_kernel<F, K>), grid, block, 0, st, gate, lg, up, lu, grad, total, per, out, gup)
        if (f32) { if (back) METIS_SG(true, true); else METIS_SG(true, false); }
        else { if (back) METIS_SG(false, true); else METIS_SG(false, false); }
#undef METIS_SG
    }
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

}  // namespace metis
