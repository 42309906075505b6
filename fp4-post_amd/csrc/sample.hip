// A token of each row's distribution, drawn by a given random number, and its log-probability:
//   w_i = exp((x_i - max x) / T);  the tokens in order of falling logits, of equal ones the lower index first;
//   K1 the first k of them, K2 those of K1 with less than p sum(K1) of weight before them, K3 those of K2 with w >= min_p;
//   the lowest index i of K3 with  sum_{j <= i, j in K3} w_j > u sum(K3),   log p_i = log w_i - log sum_i w_i  (of all tokens, not of K3 alone)
// Nothing is sorted but the few tokens next to a threshold.  A weight is 2^(-n / 64) 2^(-r / 64) with n whole and |r| <= 1/2: n is the token's bin.  One pass counts tokens
// and adds up weights by bins, in whole numbers of 2^-41 of the bin's own, so that the order of the additions does not count; the bin that holds a threshold is then
// taken apart (its tokens sorted where they are few, by digits of their logits and indices where they are many).  The draw adds up kept weights in the order of the
// tokens.  Weights are accurate to 2^-46 and sums are held in 64 bits: with some 10^5 tokens next to each other in the running sum, what binary32 is off would take
// another token now and then.
#include "metis_device.h"
#include "metis_host.h"

namespace metis {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 4096;                                        // 64 octaves; the last one holds everything below them
constexpr int kList = 2048;                                        // tokens that are sorted
constexpr double kUnit = 0x1p41;                                   // a weight of its bin's own, as a whole number

struct SampleArgs {
    const void* logits;
    int64_t ld;
    const float* uniforms;
    const double* row_parameters;                                  // [rows, 4], or nullptr: the four below for all rows
    double temperature, top_k, top_p, min_p;
    int64_t* tokens;
    float* logprobs;
    int rows, vocab;
};

// inclusive sums over the workgroup in the order of the threads; `all`: the sum over all of them
template <class V> __device__ __forceinline__ V scan(V v, V* waves, V& all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    V before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    all = total;
    return v + before;
}

// a row's logits in pieces of eight whose addresses are multiples of 16 bytes: the first and the last may reach beyond the row (those are -inf, with indices >= vocab)
template <bool F32> struct LogitRow {
    const char* base;
    int vocab, shift, pieces;
    __device__ LogitRow(const void* p, int vocab_) : base(static_cast<const char*>(p)), vocab(vocab_)
    {
        shift = (int)(reinterpret_cast<uintptr_t>(p) % (F32 ? 32 : 16)) / (F32 ? 4 : 2);
        pieces = (vocab + shift + 7) / 8;
    }
    __device__ __forceinline__ float one(int i) const
    {
        if ((unsigned)i >= (unsigned)vocab) return -INFINITY;
        if constexpr (F32) return reinterpret_cast<const float*>(base)[i];
        else return bf16_lo(reinterpret_cast<const uint16_t*>(base)[i]);
    }
    // index of the first of the eight
    __device__ __forceinline__ int load(int piece, float* x) const
    {
        const int i = piece * 8 - shift;
        if (i >= 0 && i + 8 <= vocab) {
            if constexpr (F32) {
                const float4 a = *reinterpret_cast<const float4*>(base + (size_t)i * 4), b = *reinterpret_cast<const float4*>(base + (size_t)i * 4 + 16);
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(base + (size_t)i * 2);
                x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x); x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
                x[4] = bf16_lo(a.z); x[5] = bf16_hi(a.z); x[6] = bf16_lo(a.w); x[7] = bf16_hi(a.w);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = one(i + j);
        }
        return i;
    }
};

// 2^(-r / 64) for |r| <= 1/2: the series of exp to the fifth power of 0.0054 (the next term is 2^-54)
__device__ __forceinline__ double bin_part(double r)
{
    constexpr double a = -0.010830424696249145;                    // -log 2 / 64
    double p = a * a * a * a * a / 120;
    p = fma(p, r, a * a * a * a / 24);
    p = fma(p, r, a * a * a / 6);
    p = fma(p, r, a * a / 2);
    p = fma(p, r, a);
    return fma(p, r, 1.0);
}

struct Weigher {
    double top, rate;                                              // the row's maximum; 64 log2(e) / T
    const double* table;                                           // 2^(-i / 64)
    // 64 times the binary logarithm of 1 / w, at most 2^20 (w = 0)
    __device__ __forceinline__ double depth(float x) const
    {
        const double t = fmin((top - (double)x) * rate, 0x1p20);
        return (double)x == top ? 0.0 : t;                         // (an infinite maximum less itself is no number)
    }
    __device__ __forceinline__ static int bin(double whole) { return min((int)whole, kBins - 1); }
    __device__ __forceinline__ double edge(int n) const { return ldexp(table[n & 63], -(n >> 6)); }
    // the weight as a whole number of its bin's units
    __device__ __forceinline__ uint64_t units(double t, double whole, int b) const
    {
        double p = bin_part(t - whole);
        if (b == kBins - 1) p *= edge((int)whole - b);
        return (uint64_t)(p * kUnit + 0.5);
    }
    __device__ __forceinline__ double weight(float x) const
    {
        const double t = depth(x), whole = rint(t);
        return bin_part(t - whole) * edge((int)whole);
    }
};

// falling logits, then rising indices, as rising whole numbers of 56 bits
__device__ __forceinline__ uint32_t falling(float x)
{
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);      // (both zeros are one logit)
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ uint64_t place(float x, int i) { return (uint64_t)falling(x) << 24 | ((uint32_t)i & 0xffffffu); }
__device__ __forceinline__ float logit_at(uint64_t place)
{
    const uint32_t f = (uint32_t)(place >> 24);
    return __uint_as_float(f & 0x80000000u ? f : ~f & 0x7fffffffu);
}

struct SampleShared {
    uint64_t weight[kBins];
    uint32_t count[kBins];
    uint64_t list[kList];
    uint64_t digit_weight[256];
    uint32_t digit_count[256];
    double table[64];
    double waves_d[kSampleWaves];
    uint64_t waves_u[kSampleWaves];
    uint32_t waves_n[kSampleWaves], found_n;
    float tops[kSampleWaves];
    double found_d[2];
    uint64_t found_u[2];
    int found_i;
    uint32_t filled;
};

// The threshold inside bin b: the place of its need-th token (by_weight: of the token with which the bin's weights reach `need_weight`, in its units), and the weight up to it.
template <bool F32>
__device__ void take_apart(SampleShared& s, const LogitRow<F32>& row, const Weigher& w, int b, bool by_weight, uint32_t need, double need_weight, uint64_t& threshold, uint64_t& upto)
{
    const int tid = threadIdx.x;
    uint64_t prefix = 0, base = 0;                                 // base: weight of the tokens in front of those that match the prefix
    int bits = 0;
    uint32_t left = s.count[b], skipped = 0;
    while (left > kList && bits < 56) {
        __syncthreads();
        if (tid < 256) { s.digit_count[tid] = 0; s.digit_weight[tid] = 0; }
        __syncthreads();
        for (int p = tid; p < row.pieces; p += kSampleThreads) {
            float x[8];
            const int i = row.load(p, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double t = w.depth(x[j]), whole = rint(t);
                if (Weigher::bin(whole) != b) continue;
                const uint64_t at = place(x[j], i + j);
                if (bits && (at >> (56 - bits)) != prefix) continue;
                const int digit = (int)(at >> (48 - bits)) & 255;
                atomicAdd(&s.digit_count[digit], 1u);
                atomicAdd((unsigned long long*)&s.digit_weight[digit], (unsigned long long)w.units(t, whole, b));
            }
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t n = skipped;
            uint64_t sum = base;
            int d = 0;
            for (; d < 255; ++d) {
                if (by_weight ? (double)(sum + s.digit_weight[d]) >= need_weight && s.digit_count[d] : n + s.digit_count[d] >= need) break;
                n += s.digit_count[d];
                sum += s.digit_weight[d];
            }
            // (where no token reaches it, the last one that there is)
            if (s.digit_count[d] == 0)
                while (d > 0 && s.digit_count[d] == 0) { --d; n -= s.digit_count[d]; sum -= s.digit_weight[d]; }
            s.found_i = d;
            s.found_n = n;
            s.found_u[0] = sum;
        }
        __syncthreads();
        const int d = s.found_i;
        skipped = s.found_n;
        base = s.found_u[0];
        prefix = prefix << 8 | (uint64_t)d;
        bits += 8;
        left = s.digit_count[d];
    }
    __syncthreads();
    if (tid == 0) s.filled = 0;
    int size = 64;
    while (size < (int)left) size <<= 1;
    for (int e = tid; e < size; e += kSampleThreads) s.list[e] = ~0ull;
    __syncthreads();
    for (int p = tid; p < row.pieces; p += kSampleThreads) {
        float x[8];
        const int i = row.load(p, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (Weigher::bin(rint(w.depth(x[j]))) != b) continue;
            const uint64_t at = place(x[j], i + j);
            if (bits && (at >> (56 - bits)) != prefix) continue;
            const uint32_t e = atomicAdd(&s.filled, 1u);
            if (e < (uint32_t)kList) s.list[e] = at;
        }
    }
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int e = tid; e < size; e += kSampleThreads) {
                const int other = e ^ j;
                if (other > e) {
                    const uint64_t a = s.list[e], c = s.list[other];
                    if ((a > c) == ((e & k) == 0)) { s.list[e] = c; s.list[other] = a; }
                }
            }
            __syncthreads();
        }
    // two neighbours a thread
    uint64_t mine[2] = {0, 0}, all;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int e = 2 * tid + j;
        if (e < (int)left) {
            const double t = w.depth(logit_at(s.list[e])), whole = rint(t);
            mine[j] = w.units(t, whole, b);
        }
    }
    const uint64_t incl = scan<uint64_t>(mine[0] + mine[1], s.waves_u, all);
    const uint64_t sums[2] = {base + incl - mine[1], base + incl};
    if (tid == 0) s.found_i = (int)left - 1;
    __syncthreads();
    if (by_weight) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (2 * tid + j < (int)left && (double)sums[j] >= need_weight) atomicMin(&s.found_i, 2 * tid + j);
    } else if (tid == 0) {
        s.found_i = min((int)(need - skipped) - 1, (int)left - 1);
    }
    __syncthreads();
    const int e = s.found_i;
    if (e >> 1 == tid) s.found_u[0] = sums[e & 1];
    __syncthreads();
    threshold = s.list[e];
    upto = s.found_u[0];
    __syncthreads();
}

template <bool F32>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleArgs a)
{
    __shared__ SampleShared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    const double* own = a.row_parameters ? a.row_parameters + 4 * (size_t)r : nullptr;
    const double temperature = own ? own[0] : a.temperature, top_k = own ? own[1] : a.top_k, top_p = own ? own[2] : a.top_p, min_p = own ? own[3] : a.min_p;
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    const double u = (double)a.uniforms[r];

    // ---- the maximum; a NaN anywhere shows in it
    float top = -INFINITY;
    bool nan = false;
    for (int p = tid; p < row.pieces; p += kSampleThreads) {
        float x[8];
        row.load(p, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            nan |= x[j] != x[j];
            top = fmaxf(top, x[j]);
        }
    }
    top = wave_max(top);
    if (__any(nan)) top = __builtin_nanf("");
    if (lane == 0) s.tops[wave] = top;
    if (tid < 64) s.table[tid] = exp2(-(double)tid / 64);
    for (int b = tid; b < kBins; b += kSampleThreads) { s.weight[b] = 0; s.count[b] = 0; }
    __syncthreads();
    top = s.tops[0];
#pragma unroll
    for (int w = 1; w < kSampleWaves; ++w) {
        const float other = s.tops[w];
        top = top != top || other != other ? __builtin_nanf("") : fmaxf(top, other);
    }
    // nothing to draw from, or no way to
    if (!(top > -INFINITY) || !(temperature > 0.0 && temperature < INFINITY) || !(u >= 0.0 && u < 1.0) || !(top_k >= 0.0) || !(top_p > 0.0) || !(min_p >= 0.0 && min_p <= 1.0)) {
        if (tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = __builtin_nanf("");
        }
        return;
    }
    const Weigher w = {(double)top, 92.33248261893243 / temperature, s.table};

    // ---- tokens and weights by bins
    const bool by_k = top_k >= 1.0 && top_k < (double)a.vocab, by_p = top_p < 1.0;
    for (int p = tid; p < row.pieces; p += kSampleThreads) {
        float x[8];
        row.load(p, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double t = w.depth(x[j]), whole = rint(t);
            const int b = Weigher::bin(whole);
            atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)w.units(t, whole, b));
            if (by_k || by_p) atomicAdd(&s.count[b], 1u);
        }
    }
    __syncthreads();
    constexpr int per = kBins / kSampleThreads;
    double weights[per], sum = 0.0, total;
    uint32_t counts[per], number = 0, tokens_all;
#pragma unroll
    for (int j = 0; j < per; ++j) {
        const int b = per * tid + j;
        weights[j] = (double)s.weight[b] * (1.0 / kUnit) * w.edge(b);
        counts[j] = s.count[b];
        sum += weights[j];
        number += counts[j];
    }
    const double before = scan<double>(sum, s.waves_d, total) - sum;

    // ---- thresholds
    uint64_t threshold = ~0ull;
    double kept = total;                                           // sum(K1)
    int last = kBins;                                              // the bin that K1 ends in
    if (by_k) {
        uint32_t upto = scan<uint32_t>(number, s.waves_n, tokens_all) - number;
        const uint32_t need = (uint32_t)top_k;
        double above = before;
#pragma unroll
        for (int j = 0; j < per; ++j) {
            if (upto < need && upto + counts[j] >= need) {
                s.found_i = per * tid + j;
                s.found_n = upto;
                s.found_d[0] = above;
            }
            upto += counts[j];
            above += weights[j];
        }
        __syncthreads();
        last = s.found_i;
        const uint32_t skipped = s.found_n;
        const double in_front = s.found_d[0];
        __syncthreads();
        uint64_t units;
        take_apart<F32>(s, row, w, last, false, need - skipped, 0.0, threshold, units);
        kept = in_front + (double)units * (1.0 / kUnit) * w.edge(last);
    }
    if (by_p) {
        const double need = top_p * kept;
        if (tid == 0) s.found_i = -1;
        __syncthreads();
        double above = before;
#pragma unroll
        for (int j = 0; j < per; ++j) {
            const int b = per * tid + j;
            const double upto = b == last ? kept : above + weights[j];
            if (b <= last && above < need && upto >= need && weights[j] > 0.0) {   // (one bin at most: the sums rise)
                s.found_i = b;
                s.found_d[0] = above;
            }
            above += weights[j];
        }
        __syncthreads();
        const int b = s.found_i;
        const double in_front = s.found_d[0];
        __syncthreads();
        if (b >= 0) {
            uint64_t place_p, units;
            take_apart<F32>(s, row, w, b, true, 0, (need - in_front) / w.edge(b) * kUnit, place_p, units);
            threshold = place_p < threshold ? place_p : threshold;
        }
    }

    // ---- the draw: kept weights by stretches of 512 tokens in the order of the tokens, then the stretch that the random number falls into
    constexpr int most = kBins;                                    // stretches at a time, in place of the bins' weights
    double* const stretch = reinterpret_cast<double*>(s.weight);
    const int stretches = (row.pieces + 63) / 64;
    double done = 0.0, goal = 0.0;
    int chosen = -1;
    double chosen_front = 0.0;
    for (int round = 0; round < 2; ++round) {                      // the sum first, then the place (once where the stretches fit)
        done = 0.0;
        for (int first = 0; first < stretches; first += most) {
            const int here = min(most, stretches - first);
            if (round == 0 || stretches > most) {
                __syncthreads();
                for (int k = wave; k < here; k += kSampleWaves) {
                    double v = 0.0;
                    const int p = (first + k) * 64 + lane;
                    if (p < row.pieces) {
                        float x[8];
                        const int i = row.load(p, x);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (place(x[j], i + j) <= threshold) {
                                const double wt = w.weight(x[j]);
                                v += wt >= min_p ? wt : 0.0;
                            }
                    }
#pragma unroll
                    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
                    if (lane == 0) stretch[k] = v;
                }
                __syncthreads();
            }
            // four stretches a thread
            double v[per], sum4 = 0.0, all;
#pragma unroll
            for (int j = 0; j < per; ++j) {
                v[j] = per * tid + j < here ? stretch[per * tid + j] : 0.0;
                sum4 += v[j];
            }
            const double incl = scan<double>(sum4, s.waves_d, all);
            if (round == 1) {
                double at = done + (incl - sum4);
#pragma unroll
                for (int j = 0; j < per; ++j) {
                    if (v[j] > 0.0 && at + v[j] > goal) atomicMin(&s.found_i, first + per * tid + j);
                    if (v[j] > 0.0) atomicMax((int*)&s.filled, first + per * tid + j);
                    at += v[j];
                }
                __syncthreads();
                const int f = s.found_i - first;
                if (s.found_i < stretches && chosen < 0) {
                    if (f >= 0 && f / per == tid) {
                        double in_front = done + (incl - sum4);
#pragma unroll
                        for (int j = 0; j < per; ++j)
                            if (j < f % per) in_front += v[j];
                        s.found_d[0] = in_front;
                    }
                    __syncthreads();
                    chosen = s.found_i;
                    chosen_front = s.found_d[0];
                }
            }
            done += all;
        }
        if (round == 0) {
            goal = u * done;
            __syncthreads();
            if (tid == 0) { s.found_i = stretches; s.filled = 0; }
            __syncthreads();
        }
    }
    const bool end = chosen < 0;                                   // (a rounding put the goal behind every weight: the last token that has one)
    if (end) chosen = (int)s.filled;
    if (wave != 0) return;
    const int p = chosen * 64 + lane;
    double v[8], mine = 0.0;
    float x[8];
    int i = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0;
    if (p < row.pieces) {
        i = row.load(p, x);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (place(x[j], i + j) <= threshold) {
                const double wt = w.weight(x[j]);
                v[j] = wt >= min_p ? wt : 0.0;
                mine += v[j];
            }
    }
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double q = __shfl_up(incl, o, 64);
        if (lane >= o) incl += q;
    }
    double at = chosen_front + (incl - mine);
    int found = -1, behind = -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        at += v[j];
        if (v[j] > 0.0) {
            behind = j;
            if (found < 0 && !end && at > goal) found = j;
        }
    }
    const uint64_t hits = __ballot(found >= 0), live = __ballot(behind >= 0);
    const int who = hits ? __ffsll((unsigned long long)hits) - 1 : 63 - __clzll((unsigned long long)live);
    if (lane == who) {
        const int j = hits ? found : behind;
        float xt = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) xt = e == j ? x[e] : xt;
        a.tokens[r] = i + j;
        a.logprobs[r] = (float)(-w.depth(xt) * 0.010830424696249145 - log(total));
    }
}

int sample_tokens(const void* logits, int64_t ld, int dtype, int64_t rows, int64_t vocab, const float* uniforms, const double* parameters, const double* row_parameters, int64_t* tokens,
                  float* logprobs, hipStream_t st)
{
    if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > (int64_t)1 << 22 || (rows > 1 && ld < vocab) || ld < 0 || (rows > 0 && ld > ((int64_t)1 << 46) / rows) ||
        (dtype != METIS_DTYPE_BF16 && dtype != METIS_DTYPE_F32))
        return METIS_E_ARG;
    if (rows == 0) return METIS_OK;
    if (!logits || (uintptr_t)logits % (dtype == METIS_DTYPE_F32 ? 4 : 2) || !uniforms || (uintptr_t)uniforms % 4 || !tokens || (uintptr_t)tokens % 8 || !logprobs || (uintptr_t)logprobs % 4)
        return METIS_E_ARG;
    if (row_parameters ? (uintptr_t)row_parameters % 8 != 0 : !parameters) return METIS_E_ARG;
    SampleArgs a = {logits, ld, uniforms, row_parameters, 1.0, 0.0, 1.0, 0.0, tokens, logprobs, (int)rows, (int)vocab};
    if (!row_parameters) {
        a.temperature = parameters[0]; a.top_k = parameters[1]; a.top_p = parameters[2]; a.min_p = parameters[3];
        if (!(a.temperature > 0.0 && a.temperature < INFINITY) || !(a.top_k >= 0.0) || !(a.top_p > 0.0) || !(a.min_p >= 0.0 && a.min_p <= 1.0)) return METIS_E_ARG;
    }
    if (dtype == METIS_DTYPE_F32) hipLaunchKernelGGL(sample_kernel<true>, dim3((unsigned)rows), dim3(kSampleThreads), 0, st, a);
    else hipLaunchKernelGGL(sample_kernel<false>, dim3((unsigned)rows), dim3(kSampleThreads), 0, st, a);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

}  // namespace metis
