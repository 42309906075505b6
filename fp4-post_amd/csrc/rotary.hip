// Queries and keys turned by the angles of their positions, and the same for new tokens with their keys and values written into the pages of a cache:
//   (y1, y2) = f (x1 cos a - x2 sin a, x2 cos a + x1 sin a),   a = position * inv_freq[i]
// for the pairs (i, i + R/2) or (2i, 2i + 1) of a head's first R columns; the columns behind them are copied.  The gradient is the same turn by -a.
// Bound by memory.  The angle is formed in 64 bits and reduced to a part of a turn in [-1/2, 1/2] before anything is rounded to binary32 (a position of 2^20 times a frequency
// near one has 20 bits before the point, so binary32 would leave 4 behind it); its sine and cosine serve all heads of a token that a lane goes through.  8192 tokens of 28 + 4
// heads of 128 bf16 numbers (134 MB) in 27 us, 65536 in 181 (5.9 TB/s, a large copy 4.9 to 6.9); binary32 (268 MB) 48 us by halves, 64 in neighbouring pairs, where a lane has 64
// bytes side by side and each of its four loads takes 16 of every 64 bytes.  A token of 12 + 2 heads into a cache in 2.6, 4099 of 28 + 4 heads (76 MB) in 15 (from memory 19), into an
// e4m3 one 19 (71 MB), 32768 tokens 115 and 112.
#include "chunk8.h"
#include "metis_host.h"

namespace metis {

// A lane's piece of a head: N pairs, 2 N elements.  N = 8 where strides, addresses and sizes allow whole 16-byte accesses, else 1.
struct RotaryArgs {
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;    // strides in elements
    const int64_t *positions, *slots;
    int64_t npos;
    const void* inv_freq;
    void *q_out, *k_out, *v_out;                                   // (k_out, v_out: the cache's keys and values where there is one)
    int64_t tokens, places;                                        // places: pages * page
    int q_heads, k_heads, dim, half, freq64, interleaved;          // half = R / 2
    int head_lanes, tok_lanes, units, turned_units;
    float factor, sign, key_scale, value_scale;
    int page, rotate_blocks;
};

template <bool F32, int N> struct Piece;
template <> struct Piece<false, 8> {
    Bf16x8 c;
    __device__ __forceinline__ void load(const void* p, size_t at) { c.load(static_cast<const uint16_t*>(p) + at, 0); }
    __device__ __forceinline__ float get(int j) const { return c.get(j); }
    __device__ __forceinline__ void put(void* p, size_t at, const float* f) { c.set(f); c.store(static_cast<uint16_t*>(p) + at, 0); }
};
template <> struct Piece<true, 8> {
    F32x8 c;
    __device__ __forceinline__ void load(const void* p, size_t at) { c.load(static_cast<const float*>(p) + at, 0); }
    __device__ __forceinline__ float get(int j) const { return c.get(j); }
    __device__ __forceinline__ void put(void* p, size_t at, const float* f) { c.set(f); c.store(static_cast<float*>(p) + at, 0); }
};
template <> struct Piece<false, 1> {
    float c;
    __device__ __forceinline__ void load(const void* p, size_t at) { c = bf16_lo(static_cast<const uint16_t*>(p)[at]); }
    __device__ __forceinline__ float get(int) const { return c; }
    __device__ __forceinline__ void put(void* p, size_t at, const float* f) { static_cast<uint16_t*>(p)[at] = (uint16_t)bf16_bits(f[0]); }
};
template <> struct Piece<true, 1> {
    float c;
    __device__ __forceinline__ void load(const void* p, size_t at) { c = static_cast<const float*>(p)[at]; }
    __device__ __forceinline__ float get(int) const { return c; }
    __device__ __forceinline__ void put(void* p, size_t at, const float* f) { static_cast<float*>(p)[at] = f[0]; }
};

// value / scale in e4m3, to nearest, with the largest magnitude (448) for everything beyond it; NaN stays NaN
__device__ __forceinline__ float e4m3_range(float v, float scale)
{
    v = v / scale;
    return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }
template <int N> __device__ __forceinline__ void put_e4m3(uint8_t* p, const float* f, float scale)
{
    if constexpr (N == 8) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = e4m3_pair(e4m3_range(f[2 * j], scale), e4m3_range(f[2 * j + 1], scale));
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    } else {
        *p = (uint8_t)e4m3_pair(e4m3_range(f[0], scale), 0.0f);
    }
}

// Sine and cosine of a part of a turn for binary32, rounded once: the nearest quarter turn is taken off in 64 bits, and the series of sin(2 pi t) and cos(2 pi t) for what is left,
// |t| <= 1/8, are added up in 64 bits as well (a 64-bit product takes as long as one in binary32 that is not packed); what is cut off of them is under 2^-33.
__device__ __forceinline__ void sine_cosine(double turns, float& si, float& co)
{
    constexpr double S[6] = {6.283185307179586, -41.34170224039976, 81.60524927607506, -76.70585975306139, 42.058693944897655, -15.09464257682299};
    constexpr double C[6] = {1.0, -19.739208802178716, 64.9393940226683, -85.45681720669373, 60.24464137187666, -26.4262567833744};
    const double magic = fma(turns, 4.0, 0x1.8p52), t = fma(magic - 0x1.8p52, -0.25, turns), t2 = t * t;
    const int quarter = (int)__double_as_longlong(magic);
    double s = S[5], c = C[5];
#pragma unroll
    for (int i = 4; i >= 0; --i) {
        s = fma(s, t2, S[i]);
        c = fma(c, t2, C[i]);
    }
    const float a = (float)(s * t), b = (float)c;
    si = quarter & 1 ? b : a;
    co = quarter & 1 ? a : b;
    si = quarter & 2 ? -si : si;
    co = (quarter + 1) & 2 ? -co : co;
}

// CACHE 0: none; 1: bf16; 2: e4m3.  A workgroup takes tok_lanes tokens, head_lanes of their heads at a time.
template <bool F32, int N, int CACHE>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a)
{
    if (CACHE && (int)blockIdx.x >= a.rotate_blocks) {
        // values: a lane takes eight dimensions of one token, neighbouring lanes neighbouring tokens, whose places lie side by side in a page
        const int64_t i = (int64_t)(blockIdx.x - a.rotate_blocks) * 256 + threadIdx.x;
        const int per = a.dim / (N == 8 ? 8 : 1);
        if (i >= a.tokens * a.k_heads * per) return;
        const int64_t t = i % a.tokens, slot = a.slots[t];
        if (slot < 0 || slot >= a.places) return;
        const int c = (int)(i / a.tokens), h = c / per, d = (c - h * per) * N;
        Piece<false, N> x;
        x.load(a.v, (size_t)(t * a.v_token) + (size_t)(h * a.v_head) + d);
        const size_t at = ((size_t)(slot / a.page) * a.k_heads + h) * a.dim * a.page + (size_t)d * a.page + (size_t)(slot % a.page);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if constexpr (CACHE == 2) {
                const float f = x.get(j);
                put_e4m3<1>(static_cast<uint8_t*>(a.v_out) + at + (size_t)j * a.page, &f, a.value_scale);
            } else {
                static_cast<uint16_t*>(a.v_out)[at + (size_t)j * a.page] = (uint16_t)(__float_as_uint(x.get(j)) >> 16);
            }
        }
        return;
    }
    const int u = threadIdx.x % a.units, rest = threadIdx.x / a.units, first = rest % a.head_lanes, row = rest / a.head_lanes;
    const int64_t t = (int64_t)blockIdx.x * a.tok_lanes + row;
    if (row >= a.tok_lanes || t >= a.tokens) return;
    const bool turned = u < a.turned_units;
    float c[N], s[N];
    if (turned) {
        const double position = (double)a.positions[t % a.npos];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = u * N + j;
            const double f = a.freq64 ? static_cast<const double*>(a.inv_freq)[i] : (double)static_cast<const float*>(a.inv_freq)[i];
            double turns = position * f * 0.15915494309189535;
            turns -= rint(turns);
            float si, co;
            if constexpr (F32) {
                sine_cosine(turns, si, co);
            } else {                                               // (the hardware's sine of a part of a turn is off by less than 2^-20; bf16 has 2^-9)
                si = __builtin_amdgcn_sinf((float)turns);
                co = __builtin_amdgcn_cosf((float)turns);
            }
            c[j] = co * a.factor;
            s[j] = si * a.factor * a.sign;
        }
    }
    int64_t slot = 0;
    if constexpr (CACHE != 0) slot = a.slots[t];
    const int heads = a.q_heads + a.k_heads;
    // the two pieces of a unit: N columns each, half the turned columns apart, or side by side
    const int p0 = turned ? (a.interleaved ? 2 * u * N : u * N) : 2 * a.half + 2 * (u - a.turned_units) * N;
    const int p1 = turned && !a.interleaved ? p0 + a.half : p0 + N;
    for (int h = first; h < heads; h += a.head_lanes) {
        const bool is_q = h < a.q_heads;
        const int hk = h - a.q_heads;
        const void* src = is_q ? a.q : a.k;
        const size_t from = is_q ? (size_t)(t * a.q_token) + (size_t)(h * a.q_head) : (size_t)(t * a.k_token) + (size_t)(hk * a.k_head);
        Piece<F32, N> x0, x1;
        x0.load(src, from + p0);
        x1.load(src, from + p1);
        float y0[N], y1[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            y0[j] = x0.get(j);
            y1[j] = x1.get(j);
        }
        if (turned && !a.interleaved) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float p = y0[j], q = y1[j];
                y0[j] = fmaf(p, c[j], -(q * s[j]));
                y1[j] = fmaf(q, c[j], p * s[j]);
            }
        } else if (turned) {
            if constexpr (N == 1) {
                const float p = y0[0], q = y1[0];
                y0[0] = fmaf(p, c[0], -(q * s[0]));
                y1[0] = fmaf(q, c[0], p * s[0]);
            } else {
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const float p = y0[j], q = y0[j + 1], v = y1[j], w = y1[j + 1];
                    const int e = j / 2, o = N / 2 + j / 2;
                    y0[j] = fmaf(p, c[e], -(q * s[e]));
                    y0[j + 1] = fmaf(q, c[e], p * s[e]);
                    y1[j] = fmaf(v, c[o], -(w * s[o]));
                    y1[j + 1] = fmaf(w, c[o], v * s[o]);
                }
            }
        }
        if (CACHE == 0 || is_q) {
            if (CACHE != 0 && slot >= a.places) {                  // a place that the cache does not have: nothing is written there, and the query says so
#pragma unroll
                for (int j = 0; j < N; ++j) y0[j] = y1[j] = __builtin_nanf("");
            }
            void* out = is_q ? a.q_out : a.k_out;
            const size_t to = is_q ? ((size_t)t * a.q_heads + h) * a.dim : ((size_t)t * a.k_heads + hk) * a.dim;
            x0.put(out, to + p0, y0);
            x1.put(out, to + p1, y1);
        } else if (slot >= 0 && slot < a.places) {
            const size_t to = (((size_t)(slot / a.page) * a.k_heads + hk) * a.page + (size_t)(slot % a.page)) * a.dim;
            if constexpr (CACHE == 2) {
                put_e4m3<N>(static_cast<uint8_t*>(a.k_out) + to + p0, y0, a.key_scale);
                put_e4m3<N>(static_cast<uint8_t*>(a.k_out) + to + p1, y1, a.key_scale);
            } else {
                x0.put(a.k_out, to + p0, y0);
                x1.put(a.k_out, to + p1, y1);
            }
        }
    }
}

// strides of whole elements that keep a row's pieces apart from the next one's
static bool fits(int64_t token, int64_t head, int64_t heads, int64_t tokens)
{
    const int64_t most = (int64_t)1 << 46;
    return token >= 0 && head >= 0 && head <= most / (heads > 0 ? heads : 1) && (tokens <= 1 || token <= most / tokens);
}

int rotary(const void* q, int64_t q_token, int64_t q_head, int64_t q_heads, const void* k, int64_t k_token, int64_t k_head, int64_t k_heads, const void* v, int64_t v_token,
           int64_t v_head, const int64_t* positions, int64_t npos, const void* inv_freq, int freq_dtype, const int64_t* slots, int64_t tokens, int64_t dim, int64_t turned,
           int interleaved, int back, float factor, int dtype, int64_t pages, int64_t page, int cache_dtype, float key_scale, float value_scale, void* q_out, void* k_out,
           void* v_out, bool cached, hipStream_t st)
{
    if (tokens < 0 || q_heads < 0 || k_heads < 0 || q_heads + k_heads > 65536 || q_heads > 65536 || k_heads > 65536 || dim <= 0 || dim > 512 || dim % 2 || turned < 0 ||
        turned > dim || turned % 2 || (dtype != METIS_DTYPE_BF16 && dtype != METIS_DTYPE_F32) || (freq_dtype != METIS_DTYPE_F32 && freq_dtype != METIS_DTYPE_F64))
        return METIS_E_ARG;
    if (cached && (dtype != METIS_DTYPE_BF16 || k_heads == 0 || pages <= 0 || page <= 0 || page > 4096 || (cache_dtype != METIS_DTYPE_BF16 && cache_dtype != METIS_DTYPE_E4M3) ||
                   !(key_scale > 0.0f && key_scale < INFINITY) || !(value_scale > 0.0f && value_scale < INFINITY)))
        return METIS_E_ARG;
    if (tokens == 0 || q_heads + k_heads == 0) return METIS_OK;
    if (tokens > (int64_t)1 << 31 || npos <= 0 || tokens % npos || !positions || (turned && !inv_freq)) return METIS_E_ARG;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || (cached && (!v || !v_out || !slots))) return METIS_E_ARG;
    if (!fits(q_token, q_head, q_heads, tokens) || !fits(k_token, k_head, k_heads, tokens) || (cached && !fits(v_token, v_head, k_heads, tokens))) return METIS_E_ARG;
    if (cached && pages > (((int64_t)1 << 46) / page) / (k_heads * dim)) return METIS_E_ARG;
    const bool f32 = dtype == METIS_DTYPE_F32;
    const uintptr_t size = f32 ? 4 : 2;
    const uintptr_t any = (q_heads ? (uintptr_t)q | (uintptr_t)q_out : 0) | (k_heads ? (uintptr_t)k : 0) | (cached ? (uintptr_t)v : 0) |
                          (k_heads && !(cached && cache_dtype == METIS_DTYPE_E4M3) ? (uintptr_t)k_out | (cached ? (uintptr_t)v_out : 0) : 0);
    if (any % size || (uintptr_t)positions % 8 || (uintptr_t)slots % 8 || (uintptr_t)inv_freq % (freq_dtype == METIS_DTYPE_F64 ? 8 : 4)) return METIS_E_ARG;
    const int64_t strides = (q_heads ? q_token | q_head : 0) | (k_heads ? k_token | k_head : 0) | (cached ? v_token | v_head : 0);
    const bool whole = any % 16 == 0 && strides % (f32 ? 4 : 8) == 0 && turned % 16 == 0 && (dim - turned) % 16 == 0 && (!cached || (uintptr_t)k_out % 8 == 0);
    const int N = whole ? 8 : 1;
    RotaryArgs a = {};
    a.q = q; a.k = k; a.v = v;
    a.q_token = q_token; a.q_head = q_head; a.k_token = k_token; a.k_head = k_head; a.v_token = v_token; a.v_head = v_head;
    a.positions = positions; a.slots = slots; a.npos = npos;
    a.inv_freq = inv_freq; a.q_out = q_out; a.k_out = k_out; a.v_out = v_out;
    a.tokens = tokens; a.places = pages * page;
    a.q_heads = (int)q_heads; a.k_heads = (int)k_heads; a.dim = (int)dim; a.half = (int)(turned / 2); a.freq64 = freq_dtype == METIS_DTYPE_F64; a.interleaved = interleaved;
    a.units = (int)(dim / (2 * N)); a.turned_units = (int)(turned / (2 * N));
    a.factor = factor; a.sign = back ? -1.0f : 1.0f; a.key_scale = key_scale; a.value_scale = value_scale; a.page = (int)page;
    // A lane goes through two heads with one set of sines from two waves' pieces for each of the device's SIMDs on, else every head has lanes of its own (two heads / one / four of
    // each token, 28 + 4 of 128 numbers: 64 tokens 3.9 / 3.5 / 4.7 us, 512 4.3 / 4.5 / 5.2, 4096 12.4 / 14.6 / 11.9, 8192 26.9 / 28.1 / 28.3, 65536 181 / 194 / 195;
    // 12 + 2 heads: 512 tokens 4.0 / 3.6 / 4.8, 1024 4.3 / 4.4 / 5.1, 16384 24.4 / 27.2 / 25.9).
    const int heads = a.q_heads + a.k_heads;
    const bool two = (double)tokens * heads * a.units > (double)device_cus() * 512;
    a.head_lanes = two ? (heads + 1) / 2 : heads;
    if (a.head_lanes > 256 / a.units) a.head_lanes = 256 / a.units;
    a.tok_lanes = 256 / (a.units * a.head_lanes);
    const int64_t blocks = (tokens + a.tok_lanes - 1) / a.tok_lanes, v_items = cached ? tokens * k_heads * (dim / (N == 8 ? 8 : 1)) : 0;
    if (!launch_takes(blocks + (v_items + 255) / 256, 256)) return METIS_E_TOO_LARGE;
    a.rotate_blocks = (int)blocks;
    const dim3 grid((unsigned)(blocks + (v_items + 255) / 256)), block(256);
#define METIS_ROT(F, C) do { if (whole) hipLaunchKernelGGL((rotary_kernel<F, 8, C>), grid, block, 0, st, a); else hipLaunchKernelGGL((rotary_kernel<F, 1, C>), grid, block, 0, st, a); } while (0)
    if (!cached) { if (f32) METIS_ROT(true, 0); else METIS_ROT(false, 0); }
    else if (cache_dtype == METIS_DTYPE_BF16) METIS_ROT(false, 1);
    else METIS_ROT(false, 2);
#undef METIS_ROT
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

}  // namespace metis
