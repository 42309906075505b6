// Attention of one new token of each sequence over the pages of its keys and values, and copies of whole pages:
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q . k_t - m),   m the largest of the scores so far (one pass, the sums rescaled when it grows)
// Bound by reading the cache.  All query heads that share a head of the cache (up to 16 in a tile) go through it together on the matrix cores, each key and value
// read once, from memory straight into the registers that the products take them from:
//   scores^T [tokens, heads] = K q^T        K is the first operand as it lies in its page (a row is a token)
//   o^T [dim, heads] = V^T p^T              V is kept transposed in its page (a row is a dimension, its tokens side by side)
// and the tokens are dealt to the rows of the first product in an order that leaves a lane with exactly the eight (two times eight) neighbouring tokens of one head
// that the second product wants from it: no value crosses lanes but the maximum.  The probabilities enter the second product as two bf16 terms, which
// costs nothing, as the matrix cores are idle most of the time: each is good to 2^-16 of itself and to 2^-126 of the sequence's largest.
// 28 query and 4 cache heads of 128 numbers, keys and values from memory: 64 ragged sequences of up to 4096 tokens in pages of 16 (276 MB) 65 us (in pages of 64 79), one of 131072 (268 MB) 54 with the joining launch's 5 (5.0 TB/s), 48 ragged ones of up to 16384 tokens of 8 e4m3 heads (811 MB) 155
// (5.2 TB/s); a large copy moves 4.9.  One sequence of 411 tokens 8: lengths, table, a block's keys and values one after the other.
#include <cmath>

#include "metis_device.h"
#include "metis_host.h"

namespace metis {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;                                          // waves of a workgroup, each with its own blocks of tokens
constexpr int kHeadTile = 16;

struct AttendArgs {
    const void *q, *keys, *values;
    const int *tables, *lengths;
    void* out;
    float *sums, *stats;                                           // of splits: [seq, head, split][dim], and [seq, head, split][2]: maximum and sum of the weights
    int64_t q_seq, q_head, table_stride;
    int q_heads, kv_heads, group, pages, page_shift, width, splits, chunk, tiles, pairs;
    float scale, value_scale;                                      // scale: of the scores, with log2 e
};

// eight e4m3 bytes as bf16, exactly
__device__ __forceinline__ bf16x8_t widen(uint32_t lo, uint32_t hi)
{
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true),
                   c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return (bf16x8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// DT: dimensions / 32.  F8: the cache is e4m3.  TOK: tokens of a block, 64, or 32 where 64 tokens' keys and values do not fit the registers.
template <int DT, bool F8, int TOK>
__global__ __launch_bounds__(64 * kWaves, 2) void attend_kernel(const AttendArgs a)
{
    constexpr int D = 32 * DT, S = TOK / 32, T = TOK / 16, NV = D / 16;
    constexpr bool WIDE = F8 && TOK == 64;                         // sixteen neighbouring tokens to a lane, one 16-byte load of values for both steps; else eight a step
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    // the splits of all sequences one after the other: neighbouring workgroups, which lie on different XCDs, have the same split of other sequences and heads, so that a
    // ragged batch's late splits, which only the long sequences have, do not leave XCDs without work
    const int split = blockIdx.x / a.pairs;
    int rest = blockIdx.x - split * a.pairs;
    const int tile = rest % a.tiles;
    rest /= a.tiles;
    const int kv = rest % a.kv_heads, seq = rest / a.kv_heads;
    const int capacity = a.width << a.page_shift, said = a.lengths[seq], length = said < 0 ? 0 : said > capacity ? capacity : said;
    const bool lie = said != length;                               // a length that the table cannot have: the result is NaN
    const int begin = split * a.chunk, end = min(length, begin + a.chunk);
    if (split > 0 && begin >= length) return;
    const int heads = min(a.group - tile * kHeadTile, kHeadTile);  // heads of this tile
    const int* table = a.tables + (size_t)seq * a.table_stride;

    // q^T, the second operand: head n, dimensions as the keys' pieces have them
    bf16x8_t q[DT];
    const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + (size_t)seq * a.q_seq + (size_t)(kv * a.group + tile * kHeadTile + n) * a.q_head;
#pragma unroll
    for (int c = 0; c < DT; ++c) {
        const int d = F8 ? 64 * (c / 2) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
        const uint4 w = n < heads ? *reinterpret_cast<const uint4*>(qrow + d) : make_uint4(0u, 0u, 0u, 0u);
        q[c] = __builtin_bit_cast(bf16x8_t, w);
    }

    f32x4_t o[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] = (f32x4_t){0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, sum = 0.0f;

    const size_t unit = F8 ? 1 : 2, head_bytes = ((size_t)D << a.page_shift) * unit, page_bytes = head_bytes * a.kv_heads;
    const char* keys = static_cast<const char*>(a.keys) + kv * head_bytes;
    const char* values = static_cast<const char*>(a.values) + kv * head_bytes;
    const int mask = (1 << a.page_shift) - 1;

    // Three things are on their way at a time: a block's values while its scores are formed, the next block's keys from then on, and the pages of the one after that (PIPE; where
    // keys and values do not fit the registers side by side, the values come after the scores).  The first block's pages are asked for before anything is known of the
    // length.  A run of eight tokens (WIDE: sixteen) lies in one page: KP runs of a lane's keys, VL of its values (loads of a dimension too, of VW words).
    constexpr int KP = WIDE ? 1 : S, VL = WIDE ? 1 : S, VW = F8 && !WIDE ? 2 : 4, KC = F8 ? DT / 2 : DT, STEP = kWaves * TOK;
    constexpr bool PIPE = F8 || DT < 7;
    const int r = n >> 2, last = a.width - 1;
    int kpage[KP], vpage[VL];
    const auto page_of = [&](int tok) { return table[max(min(tok >> a.page_shift, last), 0)]; };
    const auto ask_keys = [&](int t0) {
#pragma unroll
        for (int s = 0; s < KP; ++s) kpage[s] = page_of(t0 + (WIDE ? 16 * r : 32 * s + 8 * r));
    };
    const auto ask_values = [&](int t0) {
#pragma unroll
        for (int s = 0; s < VL; ++s) vpage[s] = page_of(t0 + (WIDE ? 16 * g : 32 * s + 8 * g));
    };
    uint4 kx[T][KC];
    uint32_t vx[NV][VL][VW], bad = 0;                              // bit s of bad: the page of this lane's s-th run of keys is none
    const auto load_keys = [&](int t0) {
        const char* run[KP];
        bad = 0;
#pragma unroll
        for (int s = 0; s < KP; ++s) {
            const int tok = t0 + (WIDE ? 16 * r : 32 * s + 8 * r);
            const bool none = (uint32_t)kpage[s] >= (uint32_t)a.pages;
            if (none && tok < end) bad |= 1u << s;
            run[s] = keys + (size_t)(none || tok >= end ? 0 : kpage[s]) * page_bytes + (size_t)((tok & mask) + (n & 3)) * (D * unit) + 16 * g;
        }
#pragma unroll
        for (int t = 0; t < T; ++t)                                // (the token of row n of score tile t: number n & 3 of four)
#pragma unroll
            for (int c = 0; c < KC; ++c) kx[t][c] = *reinterpret_cast<const uint4*>(run[WIDE ? 0 : t >> 1] + (WIDE ? 4 * t : 4 * (t & 1)) * (int)(D * unit) + 64 * c);
    };
    const auto load_values = [&](int t0) {
#pragma unroll
        for (int s = 0; s < VL; ++s) {
            const int tok = t0 + (WIDE ? 16 * g : 32 * s + 8 * g);
            const char* col = values + (size_t)((uint32_t)vpage[s] >= (uint32_t)a.pages || tok >= end ? 0 : vpage[s]) * page_bytes + (size_t)(tok & mask) * unit + (((size_t)n << a.page_shift) * unit);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const char* at = col + (((size_t)(16 * i) << a.page_shift) * unit);
                if constexpr (VW == 4) {
                    const uint4 w = *reinterpret_cast<const uint4*>(at);
                    vx[i][s][0] = w.x; vx[i][s][1] = w.y; vx[i][s][2] = w.z; vx[i][s][3] = w.w;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(at);
                    vx[i][s][0] = w.x; vx[i][s][1] = w.y;
                }
            }
        }
    };
    int t0 = begin + wave * TOK;
    if (last >= 0) {
        ask_keys(t0);
        ask_values(t0);
    }
    if (PIPE && t0 < end) {
        load_keys(t0);
        ask_keys(t0 + STEP);
    }
    for (; t0 < end; t0 += STEP) {
        if constexpr (PIPE) {
            load_values(t0);
            ask_values(t0 + STEP);
            __builtin_amdgcn_sched_barrier(0);
        } else {
            load_keys(t0);
            ask_keys(t0 + STEP);
        }
        float p[TOK / 4];                                          // scores, then weights, of the lane's tokens in their order
#pragma unroll
        for (int t = 0; t < T; ++t) {
            f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < DT; ++c) {
                bf16x8_t k;
                if constexpr (F8) k = (c & 1) ? widen(kx[t][c / 2].z, kx[t][c / 2].w) : widen(kx[t][c / 2].x, kx[t][c / 2].y);
                else k = __builtin_bit_cast(bf16x8_t, kx[t][c]);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[c], acc, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) p[4 * t + j] = acc[j] * a.scale;
        }
        if (__any(bad != 0)) {                                     // a token whose page is none makes the result NaN
            const uint32_t mine = (uint32_t)__shfl((int)bad, 4 * g, 64);          // (a lane whose keys' rows are this lane's scores)
#pragma unroll
            for (int t = 0; t < T; ++t)
                if (mine >> (WIDE ? 0 : t >> 1) & 1) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[4 * t + j] = __builtin_nanf("");
                }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (PIPE) {
            if (t0 + STEP < end) {
                load_keys(t0 + STEP);
                ask_keys(t0 + 2 * STEP);
            }
        } else {
            load_values(t0);
            ask_values(t0 + STEP);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (t0 + TOK > end) {                                      // tokens behind the end have no weight, and what lies there may be anything: 0 times it has to be 0
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (t0 + (WIDE ? 16 * g + 4 * t + j : 32 * (t >> 1) + 8 * g + 4 * (t & 1) + j) >= end) p[4 * t + j] = -INFINITY;
#pragma unroll
            for (int s = 0; s < VL; ++s) {
                const int left = end - (t0 + (WIDE ? 16 * g : 32 * s + 8 * g));            // tokens of this load that count
                constexpr int PER = F8 ? 4 : 2;                                            // of a word
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const int k = min(max(left - PER * w, 0), PER);
                    const uint32_t keep = k == PER ? ~0u : (1u << (32 / PER * k)) - 1u;
#pragma unroll
                    for (int i = 0; i < NV; ++i) vx[i][s][w] &= keep;
                }
            }
        }
        float top = p[0];
#pragma unroll
        for (int i = 1; i < TOK / 4; ++i) top = fmaxf(top, p[i]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float next = fmaxf(m, top), shift = next == -INFINITY ? 0.0f : next;
        const float shrink = __builtin_amdgcn_exp2f(m - shift);
        m = next;
        sum *= shrink;
#pragma unroll
        for (int i = 0; i < TOK / 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(p[i] - shift);
            sum += p[i];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i] *= shrink;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float x = p[8 * s + 2 * w], y = p[8 * s + 2 * w + 1];
                hi[w] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);      // both cut off
                // What is left of a weight stays positive, so that an infinite value keeps its sign in both products: 2^-126 at least, binary32's smallest step, and nothing
                // where the weight is nothing.
                lo[w] = rb_pair(fmaxf(x - bf16_lo(hi[w]), fminf(x, 0x1p-126f)), fmaxf(y - bf16_hi(hi[w]), fminf(y, 0x1p-126f)));
            }
            const bf16x8_t ph = __builtin_bit_cast(bf16x8_t, make_uint4(hi[0], hi[1], hi[2], hi[3])), pl = __builtin_bit_cast(bf16x8_t, make_uint4(lo[0], lo[1], lo[2], lo[3]));
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                bf16x8_t v;
                if constexpr (WIDE) v = widen(vx[i][0][2 * s], vx[i][0][2 * s + 1]);
                else if constexpr (F8) v = widen(vx[i][s][0], vx[i][s][1]);
                else v = __builtin_bit_cast(bf16x8_t, make_uint4(vx[i][s][0], vx[i][s][1], vx[i][s][2], vx[i][s][3]));
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph, o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl, o[i], 0, 0, 0);
            }
        }
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);

    // the waves' sums together: [wave][head][dim], heads a bank apart
    __shared__ float part[kWaves][kHeadTile][D + 1];
    __shared__ float tops[kWaves][kHeadTile], sums[kWaves][kHeadTile];
    if (g == 0) {
        tops[wave][n] = m;
        sums[wave][n] = sum;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[wave][n][16 * i + 4 * g + j] = o[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < heads * D; e += 64 * kWaves) {
        const int head = e / D, d = e - head * D;
        float top = tops[0][head];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, tops[w][head]);
        const float base = top == -INFINITY ? 0.0f : top;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(tops[w][head] - base);
            num = fmaf(part[w][head][d], f, num);
            den = fmaf(sums[w][head], f, den);
        }
        if (a.splits == 1) {
            // (no token: zero)
            const float v = lie ? __builtin_nanf("") : length == 0 ? 0.0f : num / den * a.value_scale;
            static_cast<uint16_t*>(a.out)[((size_t)seq * a.q_heads + kv * a.group + tile * kHeadTile + head) * D + d] = (uint16_t)bf16_bits(v);
        } else {
            const size_t row = ((size_t)seq * a.q_heads + kv * a.group + tile * kHeadTile + head) * a.splits + split;
            a.sums[row * D + d] = num;
            if (d == 0) {
                a.stats[2 * row] = top;
                a.stats[2 * row + 1] = den;
            }
        }
    }
}

// The splits' sums of one head together: a lane has four dimensions of every G-th split.  Bound by the way to memory and back, twice: the maxima, then the sums, eight splits
// of a lane on their way at once.
constexpr int kJoinThreads = 512;
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void attend_join_kernel(const AttendArgs a)
{
    constexpr int D = 32 * DT, LANES = D / 4, G = kJoinThreads / LANES;
    const int row = blockIdx.x, seq = row / a.q_heads, tid = threadIdx.x;
    const int capacity = a.width << a.page_shift, said = a.lengths[seq], length = said < 0 ? 0 : said > capacity ? capacity : said;
    const int splits = max(1, (length + a.chunk - 1) / a.chunk);
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + (size_t)row * a.splits;
    const float4* sums = reinterpret_cast<const float4*>(a.sums) + (size_t)row * a.splits * LANES;
    __shared__ float tops[kJoinThreads / 64], dens[G];
    __shared__ float4 nums[G][LANES];
    float top = -INFINITY;
    for (int s = tid; s < splits; s += kJoinThreads) top = fmaxf(top, stats[s].x);
    top = wave_max(top);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    top = tops[0];
#pragma unroll
    for (int i = 1; i < kJoinThreads / 64; ++i) top = fmaxf(top, tops[i]);
    const float base = top == -INFINITY ? 0.0f : top;
    const int lane = tid % LANES, k = tid / LANES;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f;
    if (k < G) {
#pragma unroll 8
        for (int s = k; s < splits; s += G) {
            const float2 st = stats[s];
            const float4 v = sums[(size_t)s * LANES + lane];
            const float f = __builtin_amdgcn_exp2f(st.x - base);
            num.x = fmaf(v.x, f, num.x); num.y = fmaf(v.y, f, num.y); num.z = fmaf(v.z, f, num.z); num.w = fmaf(v.w, f, num.w);
            den = fmaf(st.y, f, den);
        }
        nums[k][lane] = num;
        if (lane == 0) dens[k] = den;
    }
    __syncthreads();
    if (tid >= LANES) return;
    const int parts = min(G, splits);
    for (int i = 1; i < parts; ++i) {
        const float4 v = nums[i][lane];
        num.x += v.x; num.y += v.y; num.z += v.z; num.w += v.w;
        den += dens[i];
    }
    const float f = said != length ? __builtin_nanf("") : length == 0 ? 0.0f : a.value_scale / den;
    uint2* out = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (size_t)row * D) + lane;
    *out = length == 0 && said == length ? make_uint2(0u, 0u) : make_uint2(rb_pair(num.x * f, num.y * f), rb_pair(num.z * f, num.w * f));
}

// Tokens of a split: up to 4096, and so many splits that the workgroups fill the rounds that the device's compute units take them in.  A round that is not full costs as
// much as one that is, a split the joining launch (5 to 9 us) and its way through memory (64 sequences of 4096 tokens, 4 heads of the cache: 93 us whole, 102 in halves); so the
// fewest splits that fill 0.85 of the rounds are taken (0.8 where the sequences are cut in any case), or of six more the best.  Uniform and ragged sequences of up to 4096
// tokens, this and in the fewest splits that reach every compute unit, from memory (a GB and more of caches in turn, pages of 64): 48 of them 80 and 79, 68 and 75 us; 65 of them
// 115 and 150, 74 and 111; 80 of them 133 and 154, 97 and 111; 160 of them 246 and 250, 171 and 208; 130 of them 213 and 240, 132 and 124, the one that loses.  512 tokens are never
// cut: two blocks a wave take less than the joining launch.
static int64_t split_tokens(int64_t pairs, int64_t capacity)
{
    const int64_t block = 64 * kWaves, most = 4096, cus = device_cus();
    if (capacity <= 2 * block) return 2 * block;
    const int64_t fewest = (capacity + most - 1) / most;
    const int64_t splits = cus / pairs > fewest ? cus / pairs : fewest;
    int64_t chosen = 0;
    const double enough = fewest > 1 ? 0.8 : 0.85;
    double best = 0.0;
    for (int64_t k = splits; k < splits + 6; ++k) {
        const int64_t chunk = ((capacity + k - 1) / k + block - 1) / block * block;
        if (chosen && (chunk < 3 * block || best >= enough)) break;
        const double rounds = (double)pairs * (double)((capacity + chunk - 1) / chunk) / (double)cus, fill = rounds / ceil(rounds);
        if (!chosen || fill > best) {
            chosen = chunk;
            best = fill;
        }
    }
    return chosen;
}

size_t paged_attention_workspace_bytes(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t capacity)
{
    if (seqs <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || dim <= 0 || capacity <= 0 || capacity > INT32_MAX || seqs > INT32_MAX || q_heads > 65536) return 16;
    const int64_t tiles = (q_heads / kv_heads + kHeadTile - 1) / kHeadTile, chunk = split_tokens(seqs * kv_heads * tiles, capacity), splits = (capacity + chunk - 1) / chunk;
    return splits <= 1 ? 16 : (size_t)seqs * (size_t)q_heads * (size_t)splits * (size_t)(dim + 2) * 4;
}

int paged_attention(const void* q, int64_t q_seq, int64_t q_head, int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim, const void* keys, const void* values, int64_t pages,
                    int64_t page, int cache_dtype, const int* tables, int64_t table_stride, int64_t width, const int* lengths, float scale, float key_scale, float value_scale,
                    void* out, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    const bool f8 = cache_dtype == METIS_DTYPE_E4M3;
    if (seqs < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads > 65536 || q_heads % kv_heads || pages < 0 || pages > INT32_MAX || width < 0 || q_seq < 0 || q_head < 0 || table_stride < 0 ||
        (cache_dtype != METIS_DTYPE_BF16 && !f8))
        return METIS_E_ARG;
    if (!(fabsf(scale) < INFINITY) || !(key_scale > 0.0f && key_scale < INFINITY) || !(value_scale > 0.0f && value_scale < INFINITY)) return METIS_E_ARG;
    if (dim <= 0 || dim > 256 || dim % (f8 ? 64 : 32) || page < 16 || page > 4096 || (page & (page - 1))) return METIS_E_ARG;
    if (seqs == 0) return METIS_OK;
    if (!out || (uintptr_t)out % 8 || !lengths || (uintptr_t)lengths % 4 || (width > 0 && (!tables || (uintptr_t)tables % 4)) || !q || (uintptr_t)q % 16 || q_seq % 8 || q_head % 8)
        return METIS_E_ARG;
    if (pages > 0 ? (!keys || !values || ((uintptr_t)keys | (uintptr_t)values) % 16) : width > 0) return METIS_E_ARG;
    if (width > (INT32_MAX - 65536) / page || seqs > ((int64_t)1 << 46) / q_heads / dim) return METIS_E_ARG;
    const int64_t capacity = width * page, tiles = (q_heads / kv_heads + kHeadTile - 1) / kHeadTile, pairs = seqs * kv_heads * tiles;
    const int64_t chunk = split_tokens(pairs, capacity > 0 ? capacity : 1), splits = capacity > 0 ? (capacity + chunk - 1) / chunk : 1;
    if (pairs > INT32_MAX / splits || !launch_takes(pairs * splits, 64 * kWaves) || (splits > 1 && !launch_takes(seqs * q_heads, kJoinThreads))) return METIS_E_TOO_LARGE;
    if (splits > 1 && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < (size_t)seqs * (size_t)q_heads * (size_t)splits * (size_t)(dim + 2) * 4)) return METIS_E_WORKSPACE;
    AttendArgs a = {};
    a.q = q; a.keys = keys; a.values = values; a.tables = tables; a.lengths = lengths; a.out = out; a.sums = static_cast<float*>(workspace);
    a.q_seq = q_seq; a.q_head = q_head; a.table_stride = table_stride;
    a.q_heads = (int)q_heads; a.kv_heads = (int)kv_heads; a.group = (int)(q_heads / kv_heads); a.pages = (int)pages; a.page_shift = __builtin_ctzll((unsigned long long)page);
    a.width = (int)width; a.splits = (int)splits; a.chunk = (int)chunk; a.tiles = (int)tiles; a.pairs = (int)pairs;
    a.scale = (float)((double)scale * (double)key_scale * 1.4426950408889634);
    a.value_scale = value_scale;
    if (splits > 1) a.stats = a.sums + (size_t)seqs * (size_t)q_heads * (size_t)splits * (size_t)dim;
    const dim3 grid((unsigned)(pairs * splits)), block(64 * kWaves), rows((unsigned)(seqs * q_heads));
#define METIS_ATT(DT, F, TOK) hipLaunchKernelGGL((attend_kernel<DT, F, TOK>), grid, block, 0, st, a)
    if (f8) {
        switch (dim / 32) {
            case 2: METIS_ATT(2, true, 64); break;
            case 4: METIS_ATT(4, true, 64); break;
            case 6: METIS_ATT(6, true, 32); break;
            default: METIS_ATT(8, true, 32);
        }
    } else {
        switch (dim / 32) {
            case 1: METIS_ATT(1, false, 64); break;
            case 2: METIS_ATT(2, false, 64); break;
            case 3: METIS_ATT(3, false, 64); break;
            case 4: METIS_ATT(4, false, 64); break;
            case 5: METIS_ATT(5, false, 32); break;
            case 6: METIS_ATT(6, false, 32); break;
            case 7: METIS_ATT(7, false, 32); break;
            default: METIS_ATT(8, false, 32);
        }
    }
#undef METIS_ATT
    if (splits > 1) {
        switch (dim / 32) {
#define METIS_JOIN(DT) case DT: hipLaunchKernelGGL((attend_join_kernel<DT>), rows, dim3(kJoinThreads), 0, st, a); break
            METIS_JOIN(1); METIS_JOIN(2); METIS_JOIN(3); METIS_JOIN(4); METIS_JOIN(5); METIS_JOIN(6); METIS_JOIN(7); METIS_JOIN(8);
#undef METIS_JOIN
        }
    }
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

// ---------------------------------------------------------------------------------------------- copies of pages
// The pairs travel with the launch: nothing has to be brought to the device first.  256 pages of 28 layers (470 MB read and written) 97 us, 4.8 TB/s, what a large copy reaches;
// 15 pages of 28 layers (7 MB) 4.
constexpr int kCopyPairs = 448;                                    // (a launch's arguments hold 4 KB)
struct CopyArgs {
    char *keys, *values;
    uint64_t page_bytes, layer_bytes;
    int layers, pieces, count;
    int from[kCopyPairs], to[kCopyPairs];
};
constexpr int kCopyPiece = 16384;                                  // bytes of a workgroup, 64 a lane

__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyArgs a)
{
    uint32_t b = blockIdx.x;
    const uint32_t piece = b % a.pieces;
    b /= a.pieces;
    const uint32_t layer = b % a.layers;
    b /= a.layers;
    const uint32_t which = b & 1, pair = b >> 1;
    char* base = (which ? a.values : a.keys) + (size_t)layer * a.layer_bytes;
    const char* from = base + (size_t)a.from[pair] * a.page_bytes;
    char* to = base + (size_t)a.to[pair] * a.page_bytes;
    const uint64_t at = (uint64_t)piece * kCopyPiece + threadIdx.x * 16;
    if ((uint64_t)(piece + 1) * kCopyPiece <= a.page_bytes) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const u32x4* src = reinterpret_cast<const u32x4*>(from + at);
        u32x4* dst = reinterpret_cast<u32x4*>(to + at);
        const u32x4 w0 = src[0], w1 = src[256], w2 = src[512], w3 = src[768];
        dst[0] = w0;
        dst[256] = w1;
        dst[512] = w2;
        dst[768] = w3;
    } else {
        for (int i = 0; i < kCopyPiece / 4096; ++i)
            if (at + 4096 * i < a.page_bytes) *reinterpret_cast<uint4*>(to + at + 4096 * i) = *reinterpret_cast<const uint4*>(from + at + 4096 * i);
    }
}

int copy_pages(void* keys, void* values, int64_t layers, int64_t pages, int64_t page_bytes, const int64_t* from, const int64_t* to, int64_t count, hipStream_t st)
{
    if (layers < 0 || pages < 0 || pages > INT32_MAX || page_bytes <= 0 || page_bytes % 16 || page_bytes > ((int64_t)1 << 31) || count < 0 || count > pages) return METIS_E_ARG;
    if (count == 0 || layers == 0) return METIS_OK;
    if (!keys || !values || ((uintptr_t)keys | (uintptr_t)values) % 16 || !from || !to) return METIS_E_ARG;
    for (int64_t i = 0; i < count; ++i)
        if (from[i] < 0 || from[i] >= pages || to[i] < 0 || to[i] >= pages) return METIS_E_ARG;
    // copies of one launch run side by side: no page is written twice, and none that is written is read
    unsigned char* written = static_cast<unsigned char*>(calloc((size_t)(pages + 7) / 8, 1));
    if (!written) return METIS_E_TOO_LARGE;
    bool apart = true;
    for (int64_t i = 0; i < count && apart; ++i) {
        apart = !(written[to[i] >> 3] >> (to[i] & 7) & 1);
        written[to[i] >> 3] |= (unsigned char)(1u << (to[i] & 7));
    }
    for (int64_t i = 0; i < count && apart; ++i) apart = !(written[from[i] >> 3] >> (from[i] & 7) & 1);
    free(written);
    if (!apart) return METIS_E_ARG;
    CopyArgs a = {};
    a.keys = static_cast<char*>(keys); a.values = static_cast<char*>(values);
    a.page_bytes = (uint64_t)page_bytes; a.layer_bytes = (uint64_t)page_bytes * (uint64_t)pages;
    a.pieces = (int)((page_bytes + kCopyPiece - 1) / kCopyPiece);
    if (layers > INT32_MAX / 2 / a.pieces || !launch_takes(2 * layers * a.pieces, 256)) return METIS_E_TOO_LARGE;
    const int64_t one = 2 * layers * a.pieces;
    a.layers = (int)layers;
    int64_t most = kCopyPairs;                                     // pairs of a launch
    while (!launch_takes(one * most, 256)) most /= 2;
    for (int64_t done = 0; done < count; done += most) {
        a.count = (int)(count - done < most ? count - done : most);
        for (int i = 0; i < a.count; ++i) {
            a.from[i] = (int)from[done + i];
            a.to[i] = (int)to[done + i];
        }
        hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(one * a.count)), dim3(256), 0, st, a);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    return METIS_OK;
}

}  // namespace metis
