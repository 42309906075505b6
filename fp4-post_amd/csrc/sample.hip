// A token of each row's distribution, drawn by a given random number, and its log-probability:
//   w_i = exp((x_i - max x) / T);  the tokens in order of falling logits, of equal ones the lower index first;
//   K1 the first k of them, K2 those of K1 with less than p sum(K1) of weight before them, K3 those of K2 with w >= min_p;
//   the lowest index i of K3 with  sum_{j <= i, j in K3} w_j > u sum(K3),   log p_i = log w_i - log sum_i w_i  (of all tokens, not of K3 alone)
// The vocabulary is not sorted.  A token's depth is the binary logarithm of 1 / w, its bin the depth in 1/64.  One pass adds up all weights and takes out the tokens of the
// bins down to one that the thresholds lie above of as a rule:
//   k  at least k tokens lie in the bins down to the one that holds the k-th largest of 4096 maxima over disjoint shares of the row;
//   p  some 3000 tokens lie down to the 2130th largest of them, and some 16000 down to the 4013th (where the first are not enough); and with W0 the weights of those maxima (less than all weights), tokens deeper than
//      log2(2 V / ((1 - p) W0)) have together less than half of what K2 leaves out.
// They are sorted where they are few; else they are counted (k) and their weights added up (p) by bins, in whole numbers, so that the order of the additions does not
// count, and the tokens of the bin that holds a threshold are sorted.  What is kept is added up by stretches of 512 indices for the draw, in whole numbers again.  Where
// the thresholds lie deeper (large k, flat rows), further passes over the row do the same with all tokens, and narrow a bin of too many by digits of its logits and indices.
// Weights are accurate to 2^-44 and sums are held in 64 bits: with some 10^5 tokens next to each other in the running sum, what binary32 is off would take another
// token now and then.  Each pass is a chain of some twenty 64-bit operations for each token, and what it must not do is go through LDS for each (one LDS
// operation of a compute unit's sixteen waves costs as much as sixteen of these on its four SIMDs): there are no tables, sums over lanes go by DPP.
// Rows that do not fill the device are shared out to several workgroups for the passes over all tokens, in launches of their own.
#include <type_traits>

#include "metis_device.h"
#include "metis_host.h"

namespace metis {

constexpr int kSampleThreads = 1024;                               // of the workgroup that has a row to itself
constexpr int kPartThreads = 256;                                  // of one that has a part of a row
constexpr int kBins = 4096;                                        // 64 octaves; the last one holds everything below them
constexpr int kTaken = 24576, kPartTaken = 8192;                   // tokens that are taken out of a row, and of a part of one
constexpr int kList = 1024;                                        // tokens that can be sorted
constexpr int kShares = 4096, kSharesDown = 2130, kSharesFar = 4013;   // maxima of a row, and how many of them lie in the bins that p takes tokens out of, first and then
constexpr double kUnit = 0x1p41;                                   // a weight of its bin's octave, as a whole number
constexpr double kKeptUnit = 0x1p50;                               // a kept weight of a stretch

struct SampleArgs {
    const void* logits;
    int64_t ld;
    const float* uniforms;
    const double* row_parameters;                                  // [rows, 4], or nullptr: the four below for all rows
    double temperature, top_k, top_p, min_p;
    int64_t* tokens;
    float* logprobs;
    // of rows in parts: [rows][kShares] maxima, [rows][parts] sums of weights, [rows][kBins] sums of stretches, [rows][kTaken] indices and their numbers
    float* tops;
    double* sums;
    double* stretches;
    uint32_t *taken, *filled;
    int rows, vocab, parts;
};

// The thread's number, anew: comparisons with it are made where they are used. (Kept from one step of a kernel for all later ones, they need more scalar registers than
// there are, and the spilled ones take vector registers.)
__device__ __forceinline__ int thread_anew()
{
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return tid;
}

// Another lane's value through DPP, 0 where there is none.
template <int CTRL, int ROWS = 0xf, class V> __device__ __forceinline__ V from_lane(V v)
{
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "");
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    }
}
template <class V> __device__ __forceinline__ V lane_value(V v, int lane)      // (a lane that all agree on)
{
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane);
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    }
}
// inclusive sums over a wave's lanes: within rows of 16, then the last lane of a row to the next, of the first two rows to the others
template <class V> __device__ __forceinline__ V wave_scan(V v)
{
    v += from_lane<0x111>(v);
    v += from_lane<0x112>(v);
    v += from_lane<0x114>(v);
    v += from_lane<0x118>(v);
    v += from_lane<0x142, 0xa>(v);
    v += from_lane<0x143, 0xc>(v);
    return v;
}
// inclusive sums over the workgroup in the order of the threads; `all`: the sum over all of them
template <int THREADS, class V> __device__ __forceinline__ V scan(V v, V* waves, V& all)
{
    const int tid = thread_anew(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    const V sums = wave_scan(lane < THREADS / 64 ? waves[lane] : (V)0);
    all = lane_value(sums, THREADS / 64 - 1);
    return wave > 0 ? v + lane_value(sums, wave - 1) : v;
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
    // eight logits as they lie in memory
    struct Piece {
        uint4 a, b;                                                // (b: of binary32)
        __device__ __forceinline__ void expand(float* x) const
        {
            if constexpr (F32) {
                x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
                x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
            } else {
                x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x); x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
                x[4] = bf16_lo(a.z); x[5] = bf16_hi(a.z); x[6] = bf16_lo(a.w); x[7] = bf16_hi(a.w);
            }
        }
    };
    __device__ __forceinline__ int index(int piece) const { return piece * 8 - shift; }       // of its first logit
    __device__ __forceinline__ Piece load(int piece) const
    {
        const int i = index(piece);
        Piece v;
        if (i >= 0 && i + 8 <= vocab) {
            v.a = *reinterpret_cast<const uint4*>(base + (size_t)i * (F32 ? 4 : 2));
            if constexpr (F32) v.b = *reinterpret_cast<const uint4*>(base + (size_t)i * 4 + 16);
        } else if constexpr (F32) {
            v.a = make_uint4(bits(i), bits(i + 1), bits(i + 2), bits(i + 3));
            v.b = make_uint4(bits(i + 4), bits(i + 5), bits(i + 6), bits(i + 7));
        } else {
            v.a = make_uint4(bits(i) >> 16 | bits(i + 1), bits(i + 2) >> 16 | bits(i + 3), bits(i + 4) >> 16 | bits(i + 5), bits(i + 6) >> 16 | bits(i + 7));
        }
        return v;
    }
    __device__ __forceinline__ uint32_t bits(int i) const { return __float_as_uint(one(i)); }
    // f(eight logits, piece) for pieces first, first + step, ..; the next is on its way meanwhile: they come from memory or from a cache behind the L2, and a
    // workgroup's waves alone do not cover that way
    template <class F> __device__ __forceinline__ void each(int first, int end, int step, F f) const
    {
        constexpr int AHEAD = 1;
        Piece v[AHEAD] = {};
#pragma unroll 1
        for (int p = first - AHEAD * step; p < end; p += step) {
            const Piece now = v[0];
#pragma unroll
            for (int u = 0; u + 1 < AHEAD; ++u) v[u] = v[u + 1];
            if (p + AHEAD * step < end) v[AHEAD - 1] = load(p + AHEAD * step);
            if (p < first) continue;
            float x[8];
            now.expand(x);
            f(x, p);
        }
    }
};

// Depths and weights of a row.  Where the largest logit is infinite, or 2000 octaves less than a step of it, it alone has weight (and all that equal it): settle() makes
// such a row one of zeros and -inf at T = 1.
struct Weigher {
    double top, rate;                                              // the row's maximum; log2(e) / T
    float least, top32, rate32, cut;                               // what lies 2000 octaves deep or more has no weight: logits below `least` are that
    bool single;
    __device__ Weigher(float top_, double rate_) : top((double)top_), rate(rate_), cut(top_)
    {
        const double deep = top - 2000.0 / rate_;
        single = !(top_ < INFINITY) || !(deep > -3.4e38) || !((float)deep < top_);
        if (single) { top = 0.0; rate = 1.0; }
        least = single ? -2000.0f : (float)deep;
        top32 = (float)top;
        rate32 = (float)rate;
    }
    __device__ __forceinline__ float settled(float x) const { return !single ? x : x < cut ? -INFINITY : 0.0f; }
    __device__ __forceinline__ void settle(float* x) const
    {
        if (single) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] < cut ? -INFINITY : 0.0f;
        }
    }
    // A logit's bin (its depth in 1/64 octaves, to the nearest: read off a sum with 1.5 2^52), the bin's octave (bins 64 o - 32 to 64 o + 31) and what is left, |r| <= 0.508.
    struct Depth {
        double r;
        int bin, octave;
    };
    __device__ __forceinline__ Depth depth(float x) const
    {
        const double d = top - (double)fmaxf(x, least);
        const int bin = (int)__double_as_longlong(fma(d, rate * 64.0, 0x1.8p52)), octave = (bin + 32) >> 6;
        return {fma(d, rate, -(double)octave), bin, octave};
    }
    __device__ __forceinline__ static int octave_of(int bin) { return (bin + 32) >> 6; }
    // p r + c; HOT: for all tokens (as the compiler writes it, it first copies c to where the sum goes; the constants of those for a few stay out of the registers)
    template <bool HOT> __device__ __forceinline__ static double step(double p, double r, double c)
    {
        if constexpr (!HOT) return fma(p, r, c);
        double v;
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(v) : "v"(p), "v"(r), "v"(c));
        return v;
    }
    // 2^-r: a polynomial through 2^-r at nine Chebyshev points of |r| <= 0.508, and 1 at 0; within 2^-44.4
    template <bool HOT = false> __device__ __forceinline__ static double part(double r)
    {
        double p = step<HOT>(-1.020392955712988e-07, r, 1.3256508477029382e-06);
        p = step<HOT>(p, r, -1.52526837656183e-05);
        p = step<HOT>(p, r, 0.0001540345096151519);
        p = step<HOT>(p, r, -0.0013333558182304001);
        p = step<HOT>(p, r, 0.00961812916457961);
        p = step<HOT>(p, r, -0.05550410866475214);
        p = step<HOT>(p, r, 0.24022650695799835);
        p = step<HOT>(p, r, -0.6931471805599453);
        return fma(p, r, 1.0);
    }
    template <bool HOT = false> __device__ __forceinline__ double weight(float x) const
    {
        const Depth d = depth(x);
        return ldexp(part<HOT>(d.r), -d.octave);
    }
    // a weight as a whole number of its bin's units (read off the bits of a sum with 2^52), and the unit
    __device__ __forceinline__ static uint64_t units(double part, Depth d)
    {
        const uint64_t u = (uint64_t)__double_as_longlong(fma(part, kUnit, 0x1p52)) - 0x4330000000000000ull;
        return d.bin < kBins - 1 ? u : u >> min(d.octave - octave_of(kBins - 1), 63);
    }
    __device__ __forceinline__ static double unit(int bin) { return ldexp(1.0 / kUnit, -octave_of(bin)); }
    // logits of bin b and above are not below this; those of bin b and below are not above `highest`
    __device__ __forceinline__ float lowest(int b) const { return b >= kBins - 1 ? -INFINITY : wide(top - ((double)b + 1.0) / (rate * 64.0), -1.0); }
    __device__ __forceinline__ float highest(int b) const { return b <= 0 ? INFINITY : wide(top - ((double)b - 1.0) / (rate * 64.0), 1.0); }
    __device__ __forceinline__ float wide(double x, double way) const { return (float)(x + way * 0x1p-20 * (fabs(x) + fabs(top))); }
    // log of a weight
    __device__ __forceinline__ double log_weight(float x) const { return (x == top32 ? 0.0 : (double)x - top) * rate * 0.6931471805599453; }
};

// falling logits, then rising indices, as rising whole numbers of 56 bits
__device__ __forceinline__ uint32_t falling(float x)
{
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);      // (both zeros are one logit)
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float risen(uint32_t f) { return __uint_as_float(f & 0x80000000u ? f : ~f & 0x7fffffffu); }
__device__ __forceinline__ uint64_t place(float x, int i) { return (uint64_t)falling(x) << 24 | ((uint32_t)i & 0xffffffu); }

struct RowSettings {
    double temperature, top_k, top_p, min_p, u;
    bool by_k, by_p;
    __device__ RowSettings(const SampleArgs& a, int r)
    {
        const double* own = a.row_parameters ? a.row_parameters + 4 * (size_t)r : nullptr;
        temperature = own ? own[0] : a.temperature;
        top_k = own ? own[1] : a.top_k;
        top_p = own ? own[2] : a.top_p;
        min_p = own ? own[3] : a.min_p;
        u = (double)a.uniforms[r];
        by_k = top_k >= 1.0 && top_k < (double)a.vocab;
        by_p = top_p < 1.0;
    }
    __device__ bool fit() const
    {
        return temperature > 0.0 && temperature <= 0x1p64 && u >= 0.0 && u < 1.0 && top_k >= 0.0 && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0;
    }
    __device__ double rate() const { return 1.4426950408889634 / temperature; }
};

// What a workgroup holds of a row or of a part of one.
template <int THREADS, int TAKEN> struct SampleShared {
    static constexpr int WAVES = THREADS / 64;
    uint64_t weight[kBins];
    uint32_t taken[TAKEN];
    double waves_d[WAVES];
    uint64_t waves_u[WAVES];
    uint32_t waves_n[WAVES];
    float tops[WAVES];
    int found_i, found_bins[2];
    uint32_t filled;
};
using PartShared = SampleShared<kPartThreads, kPartTaken>;
struct RowShared : SampleShared<kSampleThreads, kTaken> {
    uint32_t count[kBins];
    uint64_t list[kList];
    uint64_t digit_weight[256];
    uint32_t digit_count[256];
    double found_d[2];
    uint64_t found_u[2];
    uint32_t found_n;
};

// the largest of the workgroup's values; NaN where one is
template <int THREADS> __device__ __forceinline__ float largest(float top, float* waves)
{
    const bool nan = __any(top != top);
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = nan ? __builtin_nanf("") : top;
    __syncthreads();
    top = waves[threadIdx.x & (THREADS / 64 - 1)];
    if (__any(top != top)) return __builtin_nanf("");
    return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(wave_max(top))));
}
// The largest logits of this thread's pieces (first, first + step, ..), dealt to `slots` shares (a power of two up to SLOTS; -inf: of an empty one); NaN where one is.
template <bool F32, int SLOTS> __device__ __forceinline__ void own_largest(const LogitRow<F32>& row, int first, int end, int step, int slots, float (&top)[SLOTS])
{
    bool nan = false;
    int turn = 0;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) top[k] = -INFINITY;
    row.each(first, end, step, [&](const float* x, int) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            nan |= x[j] != x[j];
            most = fmaxf(most, x[j]);
        }
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) top[k] = k == (turn & (slots - 1)) ? fmaxf(top[k], most) : top[k];
        ++turn;
    });
    if (nan) top[0] = __builtin_nanf("");
}

// Bins down to which at least so many of the shares' maxima lie (the last one where there is none).  s.weight is used.
template <int THREADS, class S>
__device__ __forceinline__ void bins_of_shares(S& s, const Weigher& w, const float (&mine)[kShares / THREADS], uint32_t need, uint32_t need_far, int& bin, int& far)
{
    const int tid = threadIdx.x;
    constexpr int per = kBins / THREADS;
    uint32_t* const count = reinterpret_cast<uint32_t*>(s.weight);
    for (int b = tid; b < kBins / 2; b += THREADS) s.weight[b] = 0;
    if (tid < 2) s.found_bins[tid] = kBins - 1;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kShares / THREADS; ++j) atomicAdd(&count[min(w.depth(w.settled(mine[j])).bin, kBins - 1)], 1u);
    __syncthreads();
    uint32_t c[per], n = 0, all;
#pragma unroll
    for (int j = 0; j < per; ++j) {
        c[j] = count[per * tid + j];
        n += c[j];
    }
    uint32_t upto = scan<THREADS>(n, s.waves_n, all) - n;
#pragma unroll
    for (int j = 0; j < per; ++j) {
        if (upto < need && upto + c[j] >= need) s.found_bins[0] = per * tid + j;
        if (upto < need_far && upto + c[j] >= need_far) s.found_bins[1] = per * tid + j;
        upto += c[j];
    }
    __syncthreads();
    bin = s.found_bins[0];
    far = s.found_bins[1];
}
// The deepest bin that p's threshold can lie in.
template <int THREADS, class S> __device__ __forceinline__ int deepest_p(S& s, const RowSettings& set, const Weigher& w, const float (&mine)[kShares / THREADS], int vocab)
{
    double known = 0.0, all;
#pragma unroll
    for (int j = 0; j < kShares / THREADS; ++j) known += w.weight(w.settled(mine[j]));
    scan<THREADS>(known, s.waves_d, all);
    // (W0's tokens are in the row, each once, so W >= W0; two more bins make good what W0 and the bins are rounded by)
    const double bins = (log2(2.0 * (double)vocab) - log2((1.0 - set.top_p) * all)) * 64.0 + 2.0;
    return bins < (double)(kBins - 1) ? max((int)bins, 0) : kBins - 1;
}
// The bins down to which tokens are taken out, first and then (-1: none are: no thresholds, or so large a k that another pass is needed anyhow), and the deepest one that counts.
struct Limits {
    int first = -1, far = -1, deepest = kBins - 1;
    template <int THREADS, class S> __device__ __forceinline__ void find(S& s, const RowSettings& set, const Weigher& w, const float (&mine)[kShares / THREADS], int vocab)
    {
        if (set.by_k ? set.top_k > (double)kSharesFar : !set.by_p) return;
        bins_of_shares<THREADS>(s, w, mine, set.by_k ? (uint32_t)set.top_k : (uint32_t)kSharesDown, (uint32_t)kSharesFar, first, far);
        if (set.by_k) return;
        deepest = deepest_p<THREADS>(s, set, w, mine, vocab);
        first = min(first, deepest);
        far = min(far, deepest);
    }
};

// f(logit, number) for those of eight neighbours that are wanted.  Few are as a rule: each lane goes through its own, one after the other.
template <class W, class F> __device__ __forceinline__ void each_of_eight(const float* x, W wanted, F f)
{
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine |= wanted(x[j]) ? 1u << j : 0u;
    while (mine) {
        const int j = __ffs((int)mine) - 1;
        float y = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y = e == j ? x[e] : y;
        f(y, j);
        mine &= mine - 1;
    }
}

// Takes the indices of the tokens down to bin `limit` (and of some of the next one: those that are not below a bound in binary32; never of -inf) out of pieces first,
// first + step, .., multiples of 64 lanes (s.filled counts them, also those that s.taken has no room for); returns the thread's sum of all weights (SUM).  With k that sum is
// for the log-probability alone, and formed in binary32 by eights (a weight is off by 2^-19 at a depth of 40 octaves, 2^-22 where it counts).
template <bool F32, bool SUM, int TAKEN, class S>
__device__ __forceinline__ double take_down(S& s, const RowSettings& set, const LogitRow<F32>& row, const Weigher& w, int limit, int first, int end, int step)
{
    double sum = 0.0;
    const float lowest = limit < 0 ? INFINITY : fmaxf(w.lowest(limit), -3.4028234e38f);
    const auto take = [&](const float* x, float most, int i) {
        if (!__any(most >= lowest)) return;
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) n += x[j] >= lowest ? 1u : 0u;
        const uint32_t upto = wave_scan(n);
        uint32_t at = 0;
        if ((threadIdx.x & 63) == 63) at = atomicAdd(&s.filled, upto);
        at = lane_value(at, 63) + upto - n;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (x[j] >= lowest) {
                if (at < (uint32_t)TAKEN) s.taken[at] = (uint32_t)(i + j);
                ++at;
            }
    };
    if constexpr (!SUM) {
        row.each(first, end, step, [&](float* x, int p) {
            w.settle(x);
            float most = x[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) most = fmaxf(most, x[j]);
            take(x, most, row.index(p));
        });
    } else if (set.by_k) {
        row.each(first, end, step, [&](float* x, int p) {
            w.settle(x);
            float eight = 0.0f, most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                eight += __builtin_amdgcn_exp2f((x[j] - w.top32) * w.rate32);
                most = fmaxf(most, x[j]);
            }
            sum += (double)eight;
            take(x, most, row.index(p));
        });
    } else {
        row.each(first, end, step, [&](float* x, int p) {
            w.settle(x);
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum += w.template weight<true>(x[j]);
                most = fmaxf(most, x[j]);
                if (j % 2) __builtin_amdgcn_sched_barrier(0);      // (two tokens' chains side by side are enough, and eight want more registers than there are)
            }
            take(x, most, row.index(p));
        });
    }
    return sum;
}

// Weights (p) of the whole row by bins down to `limit`, and tokens (k) by all bins.
template <bool F32> __device__ __forceinline__ void fill_bins(RowShared& s, const RowSettings& set, const LogitRow<F32>& row, const Weigher& w, int limit)
{
    const int tid = threadIdx.x;
    __syncthreads();
    for (int b = tid; b < kBins; b += kSampleThreads) { s.weight[b] = 0; s.count[b] = 0; }
    __syncthreads();
    row.each(tid, row.pieces, kSampleThreads, [&](float* x, int) {
        w.settle(x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const auto d = w.depth(x[j]);
            const int b = min(d.bin, kBins - 1);
            if (set.by_p) {
                const uint64_t units = w.units(w.template part<true>(d.r), d);
                if (b <= limit) atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)units);
            }
            if (set.by_k) atomicAdd(&s.count[b], 1u);
            if (j % 2) __builtin_amdgcn_sched_barrier(0);
        }
    });
    __syncthreads();
}

// f(logit, index) for the n tokens that were taken out of the row, four at a time (their logits are fetched again).
template <bool F32, class F> __device__ __forceinline__ void each_taken(const RowShared& s, const LogitRow<F32>& row, const Weigher& w, uint32_t n, F f)
{
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += 4 * kSampleThreads) {
        int index[4];
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            index[u] = i + u * kSampleThreads < n ? (int)s.taken[i + u * kSampleThreads] : -1;
            x[u] = w.settled(row.one(index[u]));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (index[u] >= 0) f(x[u], index[u]);
    }
}
// Weights and tokens of those by bins down to `limit`.
template <bool F32> __device__ __forceinline__ void fill_bins_again(RowShared& s, const LogitRow<F32>& row, const Weigher& w, uint32_t n, int limit)
{
    const int tid = threadIdx.x;
    __syncthreads();
    for (int b = tid; b < kBins; b += kSampleThreads) { s.weight[b] = 0; s.count[b] = 0; }
    __syncthreads();
    each_taken(s, row, w, n, [&](float x, int) {
        const auto d = w.depth(x);
        const int b = min(d.bin, kBins - 1);
        if (b > limit) return;                                     // (not all of that bin's tokens are here)
        atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)w.units(w.part(d.r), d));
        atomicAdd(&s.count[b], 1u);
    });
    __syncthreads();
}

// The value of the lane that differs in the given bit of its number.
template <int BIT> __device__ __forceinline__ uint32_t other_lane(uint32_t v)
{
    const auto dpp = [](uint32_t x, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, false); };
    if constexpr (BIT == 1) return dpp(v, std::integral_constant<int, 0xb1>());                                                  // quads 1 0 3 2
    else if constexpr (BIT == 2) return dpp(v, std::integral_constant<int, 0x4e>());                                             // quads 2 3 0 1
    else if constexpr (BIT == 4) return dpp(dpp(v, std::integral_constant<int, 0x141>()), std::integral_constant<int, 0x1b>());  // halves of a row turned round, quads turned back
    else if constexpr (BIT == 8) return dpp(v, std::integral_constant<int, 0x128>());                                            // rows by eight
    else if constexpr (BIT == 16) {
        const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);        // {rows 0 0 2 2, rows 1 1 3 3}
        return threadIdx.x & 16 ? both[0] : both[1];
    } else {
        const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);        // {the lower half twice, the upper half twice}
        return threadIdx.x & 32 ? both[0] : both[1];
    }
}
template <int BIT> __device__ __forceinline__ uint64_t other_lane(uint64_t v)
{
    return (uint64_t)other_lane<BIT>((uint32_t)(v >> 32)) << 32 | other_lane<BIT>((uint32_t)v);
}

template <int BIT> __device__ __forceinline__ void exchange(uint64_t& v, int e, bool rising)
{
    const uint64_t other = other_lane<BIT>(v);
    const bool smaller = ((e & BIT) == 0) == rising;
    v = smaller == (other < v) ? other : v;
}
// the last six steps of a merge: within a wave
__device__ __forceinline__ void merge_wave(uint64_t& v, int e, bool rising)
{
    exchange<32>(v, e, rising);
    exchange<16>(v, e, rising);
    exchange<8>(v, e, rising);
    exchange<4>(v, e, rising);
    exchange<2>(v, e, rising);
    exchange<1>(v, e, rising);
}
__device__ __forceinline__ void sort_wave(uint64_t& v, int e)
{
    exchange<1>(v, e, (e & 2) == 0);
    exchange<2>(v, e, (e & 4) == 0); exchange<1>(v, e, (e & 4) == 0);
    exchange<4>(v, e, (e & 8) == 0); exchange<2>(v, e, (e & 8) == 0); exchange<1>(v, e, (e & 8) == 0);
    exchange<8>(v, e, (e & 16) == 0); exchange<4>(v, e, (e & 16) == 0); exchange<2>(v, e, (e & 16) == 0); exchange<1>(v, e, (e & 16) == 0);
    exchange<16>(v, e, (e & 32) == 0); exchange<8>(v, e, (e & 32) == 0); exchange<4>(v, e, (e & 32) == 0); exchange<2>(v, e, (e & 32) == 0); exchange<1>(v, e, (e & 32) == 0);
    merge_wave(v, e, (e & 64) == 0);
}
// Sorts s.list[0 .. size), size a power of two from 64 to kList (bitonic; an element to a thread).  Within a wave partners exchange by DPP, and waves without elements
// take part in the barriers alone.
__device__ __forceinline__ void sort_list(RowShared& s, int size)
{
    static_assert(kList == kSampleThreads, "");
    const int tid = thread_anew();
    const bool mine = tid < size;
    uint64_t v = mine ? s.list[tid] : ~0ull;
    if (mine) sort_wave(v, tid);
#pragma unroll 1
    for (int k = 128; k <= size; k <<= 1) {
#pragma unroll 1
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            if (mine) s.list[tid] = v;
            __syncthreads();
            if (mine) {
                const uint64_t other = s.list[tid ^ j];
                v = (((tid & j) == 0) == ((tid & k) == 0)) == (other < v) ? other : v;
            }
        }
        if (mine) merge_wave(v, tid, (tid & k) == 0);
    }
    __syncthreads();
    if (mine) s.list[tid] = v;
    __syncthreads();
}
__device__ __forceinline__ int list_size(uint32_t n)
{
    int size = 64;
    while (size < (int)n) size <<= 1;
    return size;
}

// Puts the places of the row's tokens of bin b (with bits > 0: with this prefix of their place) into the list, ~0 behind them; returns their number, which may be more than
// the list holds.
template <bool F32> __device__ __forceinline__ uint32_t take_out(RowShared& s, const LogitRow<F32>& row, const Weigher& w, int b, uint64_t prefix, int bits)
{
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) s.filled = 0;
    s.list[tid] = ~0ull;
    __syncthreads();
    const float lo = w.lowest(b), hi = w.highest(b);
    row.each(tid, row.pieces, kSampleThreads, [&](float* x, int p) {
        w.settle(x);
        const int i = row.index(p);
        each_of_eight(x, [&](float y) { return y >= lo && y <= hi; }, [&](float y, int j) {
            const uint64_t at = place(y, i + j);
            if (min(w.depth(y).bin, kBins - 1) != b || (bits && (at >> (56 - bits)) != prefix)) return;
            const uint32_t e = atomicAdd(&s.filled, 1u);
            if (e < (uint32_t)kList) s.list[e] = at;
        });
    });
    __syncthreads();
    return s.filled;
}
// The same from the n tokens that were taken out of the row: those of bin b, or all of them (b < 0).
template <bool F32> __device__ __forceinline__ uint32_t take_again(RowShared& s, const LogitRow<F32>& row, const Weigher& w, uint32_t n, int b)
{
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) s.filled = 0;
    s.list[tid] = ~0ull;
    __syncthreads();
    each_taken(s, row, w, n, [&](float x, int i) {
        if (b >= 0 && min(w.depth(x).bin, kBins - 1) != b) return;
        const uint32_t e = atomicAdd(&s.filled, 1u);
        if (e < (uint32_t)kList) s.list[e] = place(x, i);
    });
    __syncthreads();
    return s.filled;
}

// A threshold inside bin b: its need-th token (by_weight: the token with which the bin's weights reach `need_weight`, in its units).
struct Wanted {
    bool by_weight;
    uint32_t need;
    double need_weight;
};
// Narrows a bin of more tokens than the list holds down to those that share the first `bits` of their places with the threshold.
struct Narrowed {
    uint64_t prefix = 0, base = 0;                                 // base: weight of the tokens in front of those that match the prefix
    uint32_t skipped = 0;                                          // and their number
    int bits = 0;
};
template <bool F32> __device__ __forceinline__ Narrowed narrow(RowShared& s, const LogitRow<F32>& row, const Weigher& w, int b, uint32_t left, const Wanted& want)
{
    const int tid = threadIdx.x;
    Narrowed at;
    const float lo = w.lowest(b), hi = w.highest(b);
#pragma unroll 1
    while (left > kList && at.bits < 56) {
        __syncthreads();
        if (tid < 256) { s.digit_count[tid] = 0; s.digit_weight[tid] = 0; }
        __syncthreads();
        row.each(tid, row.pieces, kSampleThreads, [&](float* x, int p) {
            w.settle(x);
            const int i = row.index(p);
            each_of_eight(x, [&](float y) { return y >= lo && y <= hi; }, [&](float y, int j) {
                const auto d = w.depth(y);
                const uint64_t place_j = place(y, i + j);
                if (min(d.bin, kBins - 1) != b || (at.bits && (place_j >> (56 - at.bits)) != at.prefix)) return;
                const int digit = (int)(place_j >> (48 - at.bits)) & 255;
                atomicAdd(&s.digit_count[digit], 1u);
                atomicAdd((unsigned long long*)&s.digit_weight[digit], (unsigned long long)w.units(w.part(d.r), d));
            });
        });
        __syncthreads();
        if (tid == 0) {
            uint32_t n = at.skipped;
            uint64_t sum = at.base;
            int d = 0;
            for (; d < 255; ++d) {
                if (want.by_weight ? (double)(sum + s.digit_weight[d]) >= want.need_weight && s.digit_count[d] : n + s.digit_count[d] >= want.need) break;
                n += s.digit_count[d];
                sum += s.digit_weight[d];
            }
            // (where no token reaches it, the last one that there is)
            while (d > 0 && s.digit_count[d] == 0) { --d; n -= s.digit_count[d]; sum -= s.digit_weight[d]; }
            s.found_i = d;
            s.found_n = n;
            s.found_u[0] = sum;
        }
        __syncthreads();
        const int d = s.found_i;
        at.skipped = s.found_n;
        at.base = s.found_u[0];
        at.prefix = at.prefix << 8 | (uint64_t)d;
        at.bits += 8;
        left = s.digit_count[d];
    }
    return at;
}
// The threshold among the sorted list's `left` tokens: its place, and the weight of the bin up to it.
__device__ __forceinline__ uint64_t pick_threshold(RowShared& s, const Weigher& w, uint32_t left, const Wanted& want, const Narrowed& at, uint64_t& upto)
{
    const int tid = thread_anew();
    uint64_t mine = 0, all;
    if (tid < (int)left) {
        const auto d = w.depth(risen((uint32_t)(s.list[tid] >> 24)));
        mine = w.units(w.part(d.r), d);
    }
    const uint64_t sum = at.base + scan<kSampleThreads>(mine, s.waves_u, all);
    if (tid == 0) s.found_i = (int)left - 1;
    __syncthreads();
    if (want.by_weight) {
        if (tid < (int)left && (double)sum >= want.need_weight) atomicMin(&s.found_i, tid);
    } else if (tid == 0) {
        s.found_i = min((int)(want.need - at.skipped) - 1, (int)left - 1);
    }
    __syncthreads();
    const int e = s.found_i;
    if (e == tid) s.found_u[0] = sum;
    __syncthreads();
    upto = s.found_u[0];
    const uint64_t threshold = s.list[e];
    __syncthreads();
    return threshold;
}

__device__ __forceinline__ void answer(const SampleArgs& a, int r, int64_t token, double logp)
{
    a.tokens[r] = token;
    a.logprobs[r] = (float)logp;
}

// Kept weights of a row's pieces, and of all (for rows without thresholds in between).
struct Kept {
    uint64_t threshold;
    double min_p;
    float floor, edge;                                             // nothing below `floor` is kept (a wide bound); the threshold's logit
    int edge_index;                                                // and index
    bool whole;                                                    // all tokens are kept
    __device__ Kept(uint64_t threshold_, const RowSettings& set, const Weigher& w) : threshold(threshold_), min_p(set.min_p)
    {
        edge = threshold == ~0ull ? -INFINITY : risen((uint32_t)(threshold >> 24));
        edge_index = threshold == ~0ull ? INT32_MAX : (int)(threshold & 0xffffffu);
        floor = edge;
        if (min_p > 0.0) floor = fmaxf(floor, w.lowest((int)fmin(-log2(min_p) * 64.0 + 1.0, (double)kBins)));
        whole = threshold == ~0ull && !(min_p > 0.0);
    }
    __device__ __forceinline__ bool may(float x, int i) const { return x >= floor && (x > edge || (x == edge && i <= edge_index)); }
    __device__ __forceinline__ double one(const Weigher& w, float x, int i) const
    {
        if (!may(x, i)) return 0.0;
        const double v = w.weight(x);
        return v >= min_p ? v : 0.0;
    }
    // of eight neighbours, i the index of the first
    __device__ __forceinline__ double eight(const Weigher& w, const float* x, int i) const
    {
        double sum = 0.0;
        if (whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum += w.template weight<true>(x[j]);
                if (j % 2) __builtin_amdgcn_sched_barrier(0);
            }
            return sum;
        }
        // (of equal logits only those with lower indices than the threshold's)
        each_of_eight(x, [&](float y) { return y >= floor; }, [&](float y, int j) { sum += one(w, y, i + j); });
        return sum;
    }
};

// K1's and K2's threshold from the sorted list of n tokens, K1's among them.
__device__ __forceinline__ uint64_t threshold_of_list(RowShared& s, const RowSettings& set, const Weigher& w, uint32_t n)
{
    const int tid = thread_anew();
    const uint32_t limit = min((uint32_t)set.top_k, n);
    double all;
    const double v = tid < (int)limit ? w.weight(risen((uint32_t)(s.list[tid] >> 24))) : 0.0;
    const double before = scan<kSampleThreads>(v, s.waves_d, all) - v, goal = set.by_p ? set.top_p * all : INFINITY;
    if (tid == 0) s.found_i = 0;
    __syncthreads();
    if (tid < (int)limit && before < goal) atomicMax(&s.found_i, tid);
    __syncthreads();
    return s.list[s.found_i];
}

// The token from the row's stretches of 512: `chosen` is the one that the goal falls into, `front` the weight in front of it (-1: a rounding put the goal behind every
// weight, and the last token of stretch `end` that has one is meant).
template <bool F32>
__device__ __forceinline__ void draw_from_stretch(const SampleArgs& a, int r, const LogitRow<F32>& row, const Weigher& w, const Kept& kept, int chosen, int end, double front, double goal,
                                                  double total)
{
    const int lane = threadIdx.x & 63;
    if (threadIdx.x >= 64) return;
    const bool last = chosen < 0;
    const int p = (last ? end : chosen) * 64 + lane;
    float x[8];
    row.load(p).expand(x);                                         // (pieces behind the row: -inf)
    w.settle(x);
    const int i = row.index(p);
    const double mine = kept.eight(w, x, i), incl = wave_scan(mine);
    double at = front + (incl - mine);
    int found = -1, behind = -1;
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
        float y = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y = e == j ? x[e] : y;
        const double v = kept.one(w, y, i + j);
        at += v;
        if (v > 0.0) {
            behind = j;
            if (found < 0 && !last && at > goal) found = j;
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
        a.logprobs[r] = (float)(w.log_weight(xt) - log(total));
    }
}

// Thresholds and the draw.  total: the sum of all weights (< 0: it is what is kept); limits.first: the bin down to which s.filled tokens were taken out.  ready: there are no thresholds, and the sums of the stretches are in s.weight.
template <bool F32>
__device__ __forceinline__ void finish_row(RowShared& s, const SampleArgs& a, int r, const RowSettings& set, const LogitRow<F32>& row, const Weigher& w, double total, const Limits& limits,
                                           bool ready)
{
    const int tid = threadIdx.x;
    constexpr int per = kBins / kSampleThreads;
    int limit = limits.first;
    uint32_t filled = s.filled;
    uint64_t threshold = ~0ull;
    double kept_sum = total;                                       // sum(K1)
    int last = kBins;                                              // the bin that K1 ends in
    // what was taken out is all that may be kept, but for p with a threshold further down
    const int stretches = (row.pieces + 63) / 64;
    bool taken = limit >= 0 && stretches <= kBins && filled <= (uint32_t)kTaken;
    if (taken && set.by_k && filled <= (uint32_t)kList) {
        const uint32_t n = take_again(s, row, w, filled, -1);
        sort_list(s, list_size(n));
        threshold = threshold_of_list(s, set, w, n);
    } else {
        bool refill = (set.by_k || set.by_p) && !taken;
        if (taken) fill_bins_again(s, row, w, filled, limit);
        bool far = false;                                          // the second, larger number of tokens was taken out
#pragma unroll 1
        for (int stage = 0; stage < 2; ++stage) {                  // top_k, then top_p
            if (!(stage ? set.by_p : set.by_k)) continue;
            // the bin: k by the bins' counts, p by their weights
            const double goal = stage ? set.top_p * kept_sum : (double)(uint32_t)set.top_k;
            const auto held = [&](int b) { return stage ? (double)s.weight[b] * w.unit(b) : (double)s.count[b]; };
            double sum, above;
            for (;;) {
                sum = 0.0;
#pragma unroll
                for (int j = 0; j < per; ++j) sum += held(per * tid + j);
                if (tid == 0) s.found_i = -1;
                double all;
                above = scan<kSampleThreads>(sum, s.waves_d, all) - sum;
                if (!refill && !(taken && all < goal)) break;
                if (taken && !far && !set.by_k && limits.far > limit) {                  // further down
                    far = true;
                    limit = limits.far;
                    if (tid == 0) s.filled = 0;
                    __syncthreads();
                    take_down<F32, false, kTaken>(s, set, row, w, limit, tid, (row.pieces + 63) / 64 * 64, kSampleThreads);
                    __syncthreads();
                    filled = s.filled;
                    if (filled <= (uint32_t)kTaken) {
                        fill_bins_again(s, row, w, filled, limit);
                        continue;
                    }
                }
                taken = refill = false;                            // by another pass
                fill_bins<F32>(s, set, row, w, limits.deepest);
            }
            double front = above;
#pragma unroll
            for (int j = 0; j < per; ++j) {
                const int b = per * tid + j;
                const double here = held(b), up = stage && b == last ? kept_sum : front + here;
                // (one bin at most: the sums rise)
                if (here > 0.0 && b <= last && front < goal && up >= goal) {
                    s.found_i = b;
                    s.found_d[0] = front;
                }
                front += here;
            }
            __syncthreads();
            const int b = s.found_i;
            const double in_front = s.found_d[0];
            __syncthreads();
            if (b < 0) continue;
            const Wanted want = {stage == 1, stage ? 0 : (uint32_t)goal - (uint32_t)in_front, stage ? (goal - in_front) / w.unit(b) : 0.0};
            uint32_t n = taken ? take_again(s, row, w, filled, b) : take_out<F32>(s, row, w, b, 0, 0);
            Narrowed at;
            if (n > (uint32_t)kList) {
                at = narrow<F32>(s, row, w, b, n, want);
                n = min(take_out<F32>(s, row, w, b, at.prefix, at.bits), (uint32_t)kList);
            }
            sort_list(s, list_size(n));
            uint64_t units;
            const uint64_t found = pick_threshold(s, w, n, want, at, units);
            threshold = found < threshold ? found : threshold;
            if (stage == 0) {
                // sum(K1): with p the weights of the bins in front of this one, else nobody asks
                double before = 0.0;
                if (set.by_p) {
                    double v = 0.0;
#pragma unroll
                    for (int j = 0; j < per; ++j) v += per * tid + j < b ? (double)s.weight[per * tid + j] * w.unit(per * tid + j) : 0.0;
                    scan<kSampleThreads>(v, s.waves_d, before);
                }
                kept_sum = before + (double)units * w.unit(b);
                last = b;
            }
        }
    }

    // the sums of the stretches, in place of the bins: of what was taken out, or by another pass over the row
    const Kept kept(threshold, set, w);
    double* const stretch = reinterpret_cast<double*>(s.weight);
    __syncthreads();
    if (taken) {
        for (int k = tid; k < kBins; k += kSampleThreads) s.weight[k] = 0;
        __syncthreads();
        each_taken(s, row, w, filled, [&](float x, int index) {
            const double v = kept.one(w, x, index);
            // (no less than one unit: the number 0 falls into the first kept token, however little it weighs)
            if (v > 0.0) atomicAdd((unsigned long long*)&s.weight[(index + row.shift) / 512], (unsigned long long)fmax(v * kKeptUnit, 1.0));
        });
        __syncthreads();
    }
    double done = 0.0, goal = 0.0, chosen_front = 0.0;
    int chosen = -1;
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {                      // the sum first, then the place (one pass where the stretches fit)
        done = 0.0;
#pragma unroll 1
        for (int first = 0; first < stretches; first += kBins) {
            const int here = min(kBins, stretches - first);
            if (!taken && ((round == 0 && !ready) || stretches > kBins)) {
                __syncthreads();
                row.each(first * 64 + tid, (first + here) * 64, kSampleThreads, [&](float* x, int p) {
                    w.settle(x);
                    const double sum = wave_scan(kept.eight(w, x, row.index(p)));
                    if ((tid & 63) == 63) stretch[p / 64 - first] = sum;
                });
                __syncthreads();
            }
            double v[per], sum = 0.0, all;
#pragma unroll
            for (int j = 0; j < per; ++j) {
                v[j] = per * tid + j >= here ? 0.0 : taken ? (double)s.weight[per * tid + j] * (1.0 / kKeptUnit) : stretch[per * tid + j];
                sum += v[j];
            }
            const double incl = scan<kSampleThreads>(sum, s.waves_d, all);
            if (round == 1) {
                double at = done + (incl - sum);
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
                        double in_front = done + (incl - sum);
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
            goal = set.u * done;
            __syncthreads();
            if (tid == 0) { s.found_i = stretches; s.filled = 0; }
            __syncthreads();
        }
    }
    draw_from_stretch<F32>(a, r, row, w, kept, chosen, (int)s.filled, chosen_front, goal, total < 0.0 ? done : total);
}

// A workgroup for each row.
template <bool F32>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleArgs a)
{
    __shared__ RowShared s;
    const int tid = threadIdx.x, r = blockIdx.x;
    const RowSettings set(a, r);
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    constexpr int SLOTS = kShares / kSampleThreads;
    float mine[SLOTS];
    own_largest<F32, SLOTS>(row, tid, row.pieces, kSampleThreads, SLOTS, mine);
    float top = mine[0];                                           // (a NaN is there)
#pragma unroll
    for (int k = 1; k < SLOTS; ++k) top = top != top ? top : fmaxf(top, mine[k]);
    top = largest<kSampleThreads>(top, s.tops);
    if (!(top > -INFINITY) || !set.fit()) {                        // nothing to draw from, or no way to
        if (tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = __builtin_nanf("");
        }
        return;
    }
    const Weigher w(top, set.rate());
    Limits limits;
    limits.find<kSampleThreads>(s, set, w, mine, a.vocab);
    if (tid == 0) s.filled = 0;
    __syncthreads();
    double total = -1.0;
    if (set.by_k || set.by_p || set.min_p > 0.0)
        scan<kSampleThreads>(take_down<F32, true, kTaken>(s, set, row, w, limits.first, tid, (row.pieces + 63) / 64 * 64, kSampleThreads), s.waves_d, total);
    finish_row<F32>(s, a, r, set, row, w, total, limits, false);
}

// whether a row's stretches of 512 tokens fit in place of its bins
__device__ __forceinline__ bool stretches_fit(int pieces) { return (pieces + 63) / 64 <= kBins; }

// Rows in parts, three launches.  1: the maxima of the row's shares; the stretches' sums and the number of tokens taken out cleared.
template <bool F32>
__global__ __launch_bounds__(kPartThreads) void sample_tops_kernel(const SampleArgs a)
{
    const int r = blockIdx.x / a.parts, part = blockIdx.x - r * a.parts, tid = threadIdx.x;
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    const int at = part * kPartThreads + tid, all = a.parts * kPartThreads;
    // (a thread's pieces are dealt to several shares, or several threads have one)
    constexpr int SLOTS = kShares / kSampleThreads;
    const int slots = max(kShares / all, 1), per = max(all / kShares, 1);
    float top[SLOTS];
    own_largest<F32, SLOTS>(row, at, row.pieces, all, slots, top);
    for (int o = 1; o < per; o <<= 1) {                            // (one slot then)
        const float other = __shfl_xor(top[0], o, 64);
        top[0] = top[0] != top[0] || other != other ? __builtin_nanf("") : fmaxf(top[0], other);
    }
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
        if (k < slots && at % per == 0) a.tops[(size_t)r * kShares + k * all + at / per] = top[k];
    for (int b = at; b < kBins; b += all) a.stretches[(size_t)r * kBins + b] = 0.0;
    if (at == 0) a.filled[r] = 0;
}

template <int THREADS> __device__ __forceinline__ float row_top(const SampleArgs& a, int r, float (&mine)[kShares / THREADS], float* waves)
{
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < kShares / THREADS; ++j) {
        mine[j] = a.tops[(size_t)r * kShares + threadIdx.x + j * THREADS];
        nan |= mine[j] != mine[j];
        top = fmaxf(top, mine[j]);
    }
    return largest<THREADS>(nan ? __builtin_nanf("") : top, waves);
}

// 2: the sum of all weights, and the tokens that are taken out or the stretches' sums
template <bool F32>
__global__ __launch_bounds__(kPartThreads) void sample_bins_kernel(const SampleArgs a)
{
    __shared__ PartShared s;
    const int r = blockIdx.x / a.parts, part = blockIdx.x - r * a.parts, tid = threadIdx.x;
    const RowSettings set(a, r);
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    float mine[kShares / kPartThreads];
    const float top = row_top<kPartThreads>(a, r, mine, s.tops);
    if (!(top > -INFINITY) || !set.fit()) return;
    const Weigher w(top, set.rate());
    Limits limits;
    limits.find<kPartThreads>(s, set, w, mine, a.vocab);
    const int limit = limits.first;
    if (tid == 0) s.filled = 0;
    __syncthreads();
    double sum = 0.0;
    if (set.by_k || set.by_p || !stretches_fit(row.pieces)) {
        sum = take_down<F32, true, kPartTaken>(s, set, row, w, limit, part * kPartThreads + tid, (row.pieces + 63) / 64 * 64, a.parts * kPartThreads);
    } else {
        // no thresholds: the stretches' sums, in place of the bins
        const Kept kept(~0ull, set, w);
        row.each(part * kPartThreads + tid, (row.pieces + 63) / 64 * 64, a.parts * kPartThreads, [&](float* x, int p) {
            w.settle(x);
            const double some = wave_scan(kept.eight(w, x, row.index(p)));
            if ((tid & 63) == 63) a.stretches[(size_t)r * kBins + p / 64] = some;
            if (!kept.whole) {
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += w.template weight<true>(x[j]);
            }
        });
    }
    double all;
    scan<kPartThreads>(sum, s.waves_d, all);
    if (tid == 0) a.sums[(size_t)r * a.parts + part] = all;
    if (limit < 0) return;
    // (more than there is room for, here or there: the number says so)
    const uint32_t n = s.filled;
    if (tid == 0) s.found_i = (int)atomicAdd(&a.filled[r], n > (uint32_t)kPartTaken ? (uint32_t)kTaken + 1 : n);
    __syncthreads();
    const uint32_t at = (uint32_t)s.found_i;
    for (uint32_t i = tid; i < n && i < (uint32_t)kPartTaken && at + i < (uint32_t)kTaken; i += kPartThreads) a.taken[(size_t)r * kTaken + at + i] = s.taken[i];
}

// 3: thresholds and the draw
template <bool F32>
__global__ __launch_bounds__(kSampleThreads) void sample_finish_kernel(const SampleArgs a)
{
    __shared__ RowShared s;
    const int tid = threadIdx.x, r = blockIdx.x;
    const RowSettings set(a, r);
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    float mine[kShares / kSampleThreads];
    const float top = row_top<kSampleThreads>(a, r, mine, s.tops);
    if (!(top > -INFINITY) || !set.fit()) {
        if (tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = __builtin_nanf("");
        }
        return;
    }
    const Weigher w(top, set.rate());
    const bool ready = !set.by_k && !set.by_p && stretches_fit(row.pieces);
    const uint32_t filled = a.filled[r];
    Limits limits;
    limits.find<kSampleThreads>(s, set, w, mine, a.vocab);         // (as the launch before found them)
    if (tid == 0) s.filled = filled;
    if (ready)
        for (int b = tid; b < kBins; b += kSampleThreads) s.weight[b] = __double_as_longlong(a.stretches[(size_t)r * kBins + b]);
    for (uint32_t i = tid; i < filled && i < (uint32_t)kTaken; i += kSampleThreads) s.taken[i] = a.taken[(size_t)r * kTaken + i];
    double total;
    scan<kSampleThreads>(tid < a.parts ? a.sums[(size_t)r * a.parts + tid] : 0.0, s.waves_d, total);
    finish_row<F32>(s, a, r, set, row, w, ready && !(set.min_p > 0.0) ? -1.0 : total, limits, ready);
}

// Workgroups that share a row, or 0 for one workgroup and one launch: rows that fill a quarter of the device or more, and vocabularies of a few pieces a thread.
static int row_parts(int64_t rows, int64_t vocab)
{
    const int64_t room = (int64_t)device_cus() / rows;
    int parts = 4;                                                 // (as many threads as a row has alone, or more)
    while (parts < 32 && parts * 2 <= room && vocab >= (int64_t)parts * 2 * kPartThreads * 16) parts *= 2;
    return room >= 4 && vocab >= 4 * kPartThreads * 16 ? parts : 0;
}

struct SampleSpace {
    size_t tops, sums, stretches, taken, filled, bytes;
    SampleSpace(int64_t rows, int parts)
    {
        const size_t n = (size_t)rows;
        stretches = 0;
        taken = n * kBins * 8;
        sums = taken + n * kTaken * 4;
        tops = sums + n * (size_t)parts * 8;
        filled = tops + n * kShares * 4;
        bytes = filled + n * 4;
    }
};
size_t sample_tokens_workspace_bytes(int64_t rows, int64_t vocab)
{
    if (rows <= 0 || vocab <= 0) return 0;
    const int parts = row_parts(rows, vocab);
    return parts ? SampleSpace(rows, parts).bytes : 0;
}

int sample_tokens(const void* logits, int64_t ld, int dtype, int64_t rows, int64_t vocab, const float* uniforms, const double* parameters, const double* row_parameters, int64_t* tokens,
                  float* logprobs, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > (int64_t)1 << 22 || (rows > 1 && ld < vocab) || ld < 0 || (rows > 0 && ld > ((int64_t)1 << 46) / rows) ||
        (dtype != METIS_DTYPE_BF16 && dtype != METIS_DTYPE_F32))
        return METIS_E_ARG;
    if (rows == 0) return METIS_OK;
    if (!logits || (uintptr_t)logits % (dtype == METIS_DTYPE_F32 ? 4 : 2) || !uniforms || (uintptr_t)uniforms % 4 || !tokens || (uintptr_t)tokens % 8 || !logprobs || (uintptr_t)logprobs % 4)
        return METIS_E_ARG;
    if (row_parameters ? (uintptr_t)row_parameters % 8 != 0 : !parameters) return METIS_E_ARG;
    SampleArgs a = {};
    a.logits = logits; a.ld = ld; a.uniforms = uniforms; a.row_parameters = row_parameters; a.tokens = tokens; a.logprobs = logprobs;
    a.rows = (int)rows; a.vocab = (int)vocab;
    if (!row_parameters) {
        a.temperature = parameters[0]; a.top_k = parameters[1]; a.top_p = parameters[2]; a.min_p = parameters[3];
        if (!(a.temperature > 0.0 && a.temperature <= 0x1p64) || !(a.top_k >= 0.0) || !(a.top_p > 0.0) || !(a.min_p >= 0.0 && a.min_p <= 1.0)) return METIS_E_ARG;
    }
    a.parts = row_parts(rows, vocab);
    if (a.parts) {
        const SampleSpace space(rows, a.parts);
        if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < space.bytes) return METIS_E_WORKSPACE;
        char* base = static_cast<char*>(workspace);
        a.tops = reinterpret_cast<float*>(base + space.tops);
        a.sums = reinterpret_cast<double*>(base + space.sums);
        a.stretches = reinterpret_cast<double*>(base + space.stretches);
        a.taken = reinterpret_cast<uint32_t*>(base + space.taken);
        a.filled = reinterpret_cast<uint32_t*>(base + space.filled);
    }
    const dim3 grid((unsigned)rows), parts((unsigned)(rows * (a.parts ? a.parts : 1)));
#define METIS_SAMPLE(F)                                                                                                             \
    do {                                                                                                                            \
        if (!a.parts) {                                                                                                             \
            hipLaunchKernelGGL(sample_kernel<F>, grid, dim3(kSampleThreads), 0, st, a);                                             \
        } else {                                                                                                                    \
            hipLaunchKernelGGL(sample_tops_kernel<F>, parts, dim3(kPartThreads), 0, st, a);                                         \
            hipLaunchKernelGGL(sample_bins_kernel<F>, parts, dim3(kPartThreads), 0, st, a);                                         \
            hipLaunchKernelGGL(sample_finish_kernel<F>, grid, dim3(kSampleThreads), 0, st, a);                                      \
        }                                                                                                                           \
    } while (0)
    if (dtype == METIS_DTYPE_F32) METIS_SAMPLE(true);
    else METIS_SAMPLE(false);
#undef METIS_SAMPLE
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

}  // namespace metis
