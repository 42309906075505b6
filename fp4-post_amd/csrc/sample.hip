// A token of each row's distribution, drawn by a given random number, and its log-probability:
//   w_i = exp((x_i - max x) / T);  the tokens in order of falling logits, of equal ones the lower index first;
//   K1 the first k of them, K2 those of K1 with less than p sum(K1) of weight before them, K3 those of K2 with w >= min_p;
//   the lowest index i of K3 with  sum_{j <= i, j in K3} w_j > u sum(K3),   log p_i = log w_i - log sum_i w_i  (of all tokens, not of K3 alone)
// The vocabulary is not sorted.  A token's depth is the binary logarithm of 1 / w, its bin the depth in 1/64.  A first pass finds the row's maximum (with p, also a sum of all
// weights that is good to a few digits) and 8192 maxima over disjoint shares of the row (up to 8192 tokens: each one of them), a second one adds up all weights and takes out the tokens that a threshold lies
// among as a rule:
//   k  those in the bins down to the one that holds the k-th largest of the maxima: at least k;
//   p  those in a window of bins around the one in which the weights reach p of their sum, by a guess: where M of S shares have a maximum in the bins down to one, about
//      V (1 - (1 - M / S)^(S / V)) tokens lie there (to 1.3 percent where that are 12000 of 131072); those above the window are kept, and added up by stretches of 512 indices at once.
// They are sorted where they are few; else they are counted (k) and their weights added up (p) by bins, in whole numbers, so that the order of the additions does not
// count, and the tokens of the bin that holds a threshold are sorted.  What is kept of them is added to the stretches' sums for the draw, in whole numbers again.  Where
// the thresholds lie elsewhere (large k, flat rows), further passes over the row do the same with all tokens, and narrow a bin of too many by digits of its logits and indices.
// A weight is accurate to 2^-44 of itself and sums are held in 64 bits: with some 10^5 tokens next to each other in the running sum, what binary32 is off would take another
// token now and then.  Whole numbers round once more: of the taken tokens each kept weight to 2^-54 of the largest (one below 2^-53 is 2^-53), in the bins, where they only say
// where a threshold lies, to 2^-41.5 of itself (beyond 64 octaves to 2^-105 of the largest).  Each pass is a chain of 25 instructions for each token, 17 of them 64-bit, and an LDS operation beside it
// would cost as much as sixteen of these (a compute unit's sixteen waves share one LDS and have four SIMDs): there are no tables, sums over lanes go by DPP.  An LDS operation in
// place of the chain, a count of a bf16 row's logits by their bits, has not been tried.
// Rows that do not fill the device are shared out to several workgroups for the passes over all tokens, in launches of their own.
// 256 rows of 131072 bf16 logits (67 MB, 14 us at a large copy's rate): no thresholds 43 us, top_k = 50 38, top_p = 0.95 83 to 106 (the row that keeps most, 12000 to 14000 tokens,
// sets the time; most rows take 62 to 72: 12 for the first pass, 5 for the guess of the sum, 7 for the window, 35 for the weights in 64 bits, 4 to 14 for the list, 6 for the
// stretches and the draw).  Rows that keep more than 27000 of them take 150 to 168.  One row of 131072 binary32 logits with all settings 25 us: 3.4 + 11.4 + 11.2 in three launches.
#include <type_traits>

#include "metis_device.h"
#include "metis_host.h"

namespace metis {

constexpr int kSampleThreads = 1024;                               // of the workgroup that has a row to itself
constexpr int kPartThreads = 256;                                  // of one that has a part of a row
constexpr int kBins = 4096;                                        // 64 octaves; the last one holds everything below them
constexpr int kTaken = 16384, kPartTaken = 8192;                   // tokens that are taken out of a row, and of a part of one
constexpr int kList = 1024;                                        // tokens that can be sorted
constexpr int kShares = 8192;                                      // maxima of a row
constexpr double kLowTemperatures = 0x1p100;                       // 1 / T from which depths do not fit binary32
constexpr double kUnit = 0x1p41;                                   // a weight of its bin's octave, as a whole number
constexpr double kKeptUnit = 0x1p53;                               // a kept weight of a stretch (512 of them have room in 64 bits)

struct SampleArgs {
    const void* logits;
    int64_t ld;
    const float* uniforms;
    const double* row_parameters;                                  // [rows, 4], or nullptr: the four below for all rows
    double temperature, top_k, top_p, min_p;
    int64_t* tokens;
    float* logprobs;
    // of rows in parts: [rows][kShares] maxima, [rows][kBins] sums of stretches, [rows][kTaken] indices and their numbers
    float *tops, *guesses, *rests;                                 // (and [rows][parts][2] largest logits and guessed sums, [rows][kShares] what they hold besides the maxima)
    double* sums;                                                  // [rows][parts][2]: of all weights, of those above the window
    double* stretches;
    uint32_t *taken, *filled;
    int* limits;                                                   // [rows][3]: the window's bins, the largest logit
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

// N of them at once: exclusive
template <int THREADS, int N> __device__ __forceinline__ void scan_several(float (&v)[N], float* waves)
{
    const int tid = thread_anew(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float own[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        own[i] = v[i];
        v[i] = wave_scan(v[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane == 63) waves[i * (THREADS / 64) + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float sums = wave_scan(lane < THREADS / 64 ? waves[i * (THREADS / 64) + lane] : 0.0f);
        v[i] = (wave > 0 ? v[i] + lane_value(sums, wave - 1) : v[i]) - own[i];
    }
}

// a row's logits in pieces of eight whose addresses are multiples of 16 bytes: the first and the last may reach beyond the row (those are -inf, with indices >= vocab)
template <bool F32> struct LogitRow {
    const char* base;
    int vocab, shift, pieces;
    __device__ __forceinline__ LogitRow(const void* p, int vocab_) : base(static_cast<const char*>(p)), vocab(vocab_)
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
    double far;                                                    // 2000 octaves
    bool single;
    __device__ __forceinline__ Weigher(float top_, double rate_) : top((double)top_), rate(rate_), cut(top_)
    {
        const double deep = top - 2000.0 / rate_;
        single = !(top_ < INFINITY) || !(deep > -3.4e38) || !((float)deep < top_);
        if (single) { top = 0.0; rate = 1.0; }
        least = single ? -2000.0f : (float)deep;
        far = 2000.0 / rate;
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
    // 2^-r: a polynomial through 2^-r at nine Chebyshev points of |r| <= 0.508, and 1 at 0; within 2^-44.4
    static constexpr double C[9] = {-0.6931471805599453, 0.24022650695799835, -0.05550410866475214, 0.00961812916457961, -0.0013333558182304001, 0.0001540345096151519, -1.52526837656183e-05,
                                    1.3256508477029382e-06, -1.020392955712988e-07};
    __device__ __forceinline__ static double part(double r)
    {
        double p = C[8];
#pragma unroll
        for (int i = 7; i >= 0; --i) p = fma(p, r, C[i]);
        return fma(p, r, 1.0);
    }
    // two of them for the passes over all tokens, side by side, as they are to be issued: the compiler copies each constant to where the sum goes
    __device__ __forceinline__ static void parts(double r, double q, double& a, double& b)
    {
        asm("v_fma_f64 %0, %4, %2, %5\n\tv_fma_f64 %1, %4, %3, %5\n\tv_fma_f64 %0, %0, %2, %6\n\tv_fma_f64 %1, %1, %3, %6\n\tv_fma_f64 %0, %0, %2, %7\n\tv_fma_f64 %1, %1, %3, %7\n\t"
            "v_fma_f64 %0, %0, %2, %8\n\tv_fma_f64 %1, %1, %3, %8\n\tv_fma_f64 %0, %0, %2, %9\n\tv_fma_f64 %1, %1, %3, %9\n\tv_fma_f64 %0, %0, %2, %10\n\tv_fma_f64 %1, %1, %3, %10\n\t"
            "v_fma_f64 %0, %0, %2, %11\n\tv_fma_f64 %1, %1, %3, %11\n\tv_fma_f64 %0, %0, %2, %12\n\tv_fma_f64 %1, %1, %3, %12\n\tv_fma_f64 %0, %0, %2, 1.0\n\tv_fma_f64 %1, %1, %3, 1.0"
            : "=&v"(a), "=&v"(b)
            : "v"(r), "v"(q), "v"(C[8]), "v"(C[7]), "v"(C[6]), "v"(C[5]), "v"(C[4]), "v"(C[3]), "v"(C[2]), "v"(C[1]), "v"(C[0]));
    }
    __device__ __forceinline__ double weight(float x) const
    {
        const double d = fmin(top - (double)x, far), o = fma(d, -rate, 0x1.8p52);
        return ldexp(part(fma(d, rate, o - 0x1.8p52)), (int)__double_as_longlong(o));
    }
    // The same bits for two tokens of a pass over all (a token next to min_p is one of the kept in the sums and in the draw, or in neither): 0 from 2000 octaves on; the octave to
    // the nearest, read off a sum again.
    __device__ __forceinline__ void weights(float x, float y, double& a, double& b) const
    {
        const double d = fmin(top - (double)x, far), e = fmin(top - (double)y, far), o = fma(d, -rate, 0x1.8p52), p = fma(e, -rate, 0x1.8p52);
        parts(fma(d, rate, o - 0x1.8p52), fma(e, rate, p - 0x1.8p52), a, b);
        a = ldexp(a, (int)__double_as_longlong(o));
        b = ldexp(b, (int)__double_as_longlong(p));
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
    __device__ __forceinline__ RowSettings(const SampleArgs& a, int r)
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
    __device__ __forceinline__ bool fit() const
    {
        return temperature > 0.0 && temperature <= 0x1p64 && u >= 0.0 && u < 1.0 && top_k >= 0.0 && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0;
    }
    __device__ __forceinline__ double rate() const { return 1.4426950408889634 / temperature; }
};

// What a workgroup holds of a row or of a part of one.
template <int THREADS, int TAKEN> struct SampleShared {
    static constexpr int WAVES = THREADS / 64;
    uint64_t weight[kBins];
    uint32_t taken[TAKEN];
    double waves_d[WAVES];
    uint64_t waves_u[WAVES];
    uint32_t waves_n[WAVES];
    float waves_f[3 * WAVES];
    float tops[WAVES];
    int found_i, found_bins[2];
    uint32_t filled;
};
using PartShared = SampleShared<kPartThreads, kPartTaken>;
struct RowShared : SampleShared<kSampleThreads, kTaken> {
    double above[kBins];                                           // sums of the stretches: of the tokens above the window
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
// Where a thread has one piece at most, its eight logits are the shares.  guess: with rate > 0 the sum of their weights as seen from the largest of them, `most_of_all`, in binary32.
template <bool F32, int SLOTS>
__device__ __forceinline__ void own_largest(const LogitRow<F32>& row, int first, int end, int step, int slots, float rate, float (&top)[SLOTS], float& most_of_all, float& guess)
{
    bool nan = false;
    int turn = 0;
    guess = 0.0f;
    most_of_all = -INFINITY;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) top[k] = -INFINITY;
    row.each(first, end, step, [&](const float* x, int) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            nan |= x[j] != x[j];
            most = fmaxf(most, x[j]);
        }
        if (SLOTS == 8 && slots == 8 && end <= step) {
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) top[k] = x[k % 8];
        } else {
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) top[k] = k == (turn & (slots - 1)) ? fmaxf(top[k], most) : top[k];
        }
        ++turn;
        if (rate > 0.0f) {
            const float now = fmaxf(most_of_all, most), from = now == -INFINITY ? 0.0f : now;
            guess *= __builtin_amdgcn_exp2f((most_of_all - from) * rate);
#pragma unroll
            for (int j = 0; j < 8; ++j) guess += __builtin_amdgcn_exp2f((x[j] - from) * rate);
            most_of_all = now;
        }
    });
    if (nan) top[0] = __builtin_nanf("");
}
// the rate that weights are guessed with: 0 where nobody asks
__device__ __forceinline__ float guess_rate(const RowSettings& set) { return set.by_p && !set.by_k ? (float)set.rate() : 0.0f; }
// One logit with as much weight as all that a thread guessed but its shares' maxima: where two of the row's largest lie in the same share, the other one.
template <int SLOTS> __device__ __forceinline__ float rest_of(const float (&top)[SLOTS], float most, float guess, float rate)
{
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) guess -= top[k] > -INFINITY ? __builtin_amdgcn_exp2f((top[k] - most) * rate) : 0.0f;
    return guess > 0.0f ? most + __log2f(guess) / rate : -INFINITY;
}
// the row's sum of weights from what was guessed for some of it, as seen from the row's maximum
template <int THREADS> __device__ __forceinline__ float guessed_sum(float most, float guess, float top, float rate, float* waves)
{
    float all;
    scan<THREADS>(guess > 0.0f ? guess * __builtin_amdgcn_exp2f((most - top) * rate) : 0.0f, waves, all);
    return all;
}

// The bins whose tokens are taken out, `first` (0: nothing lies above them) to `last` (-1: none are: no thresholds, or so large a k or so flat a row that further passes are
// needed anyhow).
struct Limits {
    int first = 0, last = -1;
    __device__ __forceinline__ static float bin_weight(int b) { return __builtin_amdgcn_exp2f((float)b * (-1.0f / 64.0f)); }
    // rest: what the guess says besides the maxima (rest_of), of so many threads.  s.weight and s.taken are used
    template <int THREADS, int RESTS, class S>
    __device__ __forceinline__ void find(S& s, const RowSettings& set, const Weigher& w, const float (&mine)[kShares / THREADS], const float (&rest)[RESTS], int rests, float guess, int vocab, int pieces)
    {
        const bool exact = pieces <= THREADS && kShares == 8 * THREADS;        // every token is a share
        const int filled_shares = exact ? vocab : min(pieces, kShares);
        // (k up to 5/6 of the shares: some 14000 of 131072 tokens)
        if (set.by_k ? vocab > kTaken && set.top_k > (double)(filled_shares / 6 * 5) : !set.by_p) return;
        const int tid = threadIdx.x;
        constexpr int per = kBins / THREADS;
        uint32_t* const count = reinterpret_cast<uint32_t*>(s.weight);
        unsigned long long* const weight = reinterpret_cast<unsigned long long*>(s.taken);               // beside what the counts say, in units of 2^-40 (signed)
        static_assert(sizeof s.taken >= kBins * 8, "");
        for (int b = tid; b < kBins / 2; b += THREADS) s.weight[b] = 0;
        for (int b = tid; b < kBins; b += THREADS) weight[b] = 0;
        if (tid < 2) s.found_bins[tid] = tid ? INT32_MAX : kBins - 1;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kShares / THREADS; ++j) {
            // (empty shares: what many lanes add to one place goes there one by one)
            if (pieces >= kShares || mine[j] > -INFINITY) atomicAdd(&count[min(w.depth(w.settled(mine[j])).bin, kBins - 1)], 1u);
        }
        if (!set.by_k) {                                           // of the heavy ones the weight itself, where the bin's is off by up to half a percent
            const float heavy = w.top32 - 9.0f / w.rate32;         // (2^-9 < 0.002; the sum is at least 1)
#pragma unroll
            for (int j = 0; j < kShares / THREADS; ++j) {
                if (!(w.settled(mine[j]) > heavy)) continue;
                const auto d = w.depth(w.settled(mine[j]));
                const float v = __builtin_amdgcn_exp2f(-(float)((double)d.octave + d.r));
                atomicAdd(&weight[min(d.bin, kBins - 1)], (unsigned long long)(long long)((v - bin_weight(d.bin)) * 0x1p40f));
            }
        }
        // A token that is hidden behind a heavier one of its share: what a thread's tokens besides the maxima weigh more than others'.
        float plain = 0.0f;
        if (!set.by_k) {
            float v[RESTS], mean = 0.0f;
#pragma unroll
            for (int j = 0; j < RESTS; ++j) {
                v[j] = rest[j] > -INFINITY ? __builtin_amdgcn_exp2f((fminf(w.settled(rest[j]), w.top32) - w.top32) * w.rate32) : 0.0f;
                mean += v[j];
            }
            scan<THREADS>(mean, reinterpret_cast<float*>(s.waves_n), mean);
            mean /= (float)min(pieces, rests);
            plain = fmaxf(10.0f * mean, 1e-5f * guess);            // a hidden token of more weight is known (what else a thread has may well be twice the mean)
#pragma unroll
            for (int j = 0; j < RESTS; ++j)
                if (v[j] > plain) atomicAdd(&weight[min(max((int)(__log2f(v[j] - mean) * -64.0f), 0), kBins - 1)], (unsigned long long)((v[j] - mean) * 0x1p40f));
        }
        __syncthreads();
        uint32_t c[per], n = 0, all;
#pragma unroll
        for (int j = 0; j < per; ++j) {
            c[j] = count[per * tid + j];
            n += c[j];
        }
        const uint32_t before = scan<THREADS>(n, s.waves_n, all) - n;
        uint32_t m = before;
        if (set.by_k) {
            const uint32_t need = (uint32_t)set.top_k;
#pragma unroll
            for (int j = 0; j < per; ++j) {
                if (m < need && m + c[j] >= need) s.found_bins[0] = per * tid + j;
                m += c[j];
            }
            __syncthreads();
            last = s.found_bins[0];
            return;
        }
        // the weights of the maxima, and of the others that are guessed to lie in the same bins
        const float shares = (float)filled_shares, most = exact ? shares : shares * 0.995f;
        const auto tokens = [&](uint32_t m) __attribute__((always_inline)) { return exact ? (float)m : (float)vocab * (1.0f - __builtin_amdgcn_exp2f(__log2f(1.0f - fminf((float)m, most) / shares) * (shares / (float)vocab))); };
        if (!(guess < INFINITY)) guess = 1.0f;                     // (rows of infinities)
        float known[per], hidden[per], square[per], sum = 0.0f, sum_hidden = 0.0f, sum_square = 0.0f, told = tokens(before);
#pragma unroll
        for (int j = 0; j < per; ++j) {
            m += c[j];
            const float now = c[j] ? tokens(m) : told;
            const float each = bin_weight(per * tid + j);
            known[j] = fmaf((float)c[j], each, (float)(long long)weight[per * tid + j] * 0x1p-40f);
            hidden[j] = each > plain ? 0.0f : fmaxf(now - told - (float)c[j], 0.0f) * each;
            square[j] = hidden[j] * each;
            sum += known[j] + hidden[j];
            sum_hidden += hidden[j];
            sum_square += square[j];
            told = now;
        }
        float fronts[3] = {sum, sum_hidden, sum_square};
        scan_several<THREADS>(fronts, s.waves_f);
        float front = fronts[0], front_hidden = fronts[1], front_square = fronts[2];
        // The window: where the guess is that far from p of the sum that it may be off by that.  (Of n hidden tokens the deviation is sqrt(n) where they are few, 2.1 sqrt(n) where
        // 12000 of 131072 lie down to there.  Of 1200 rows of 131072 the window missed none that keeps up to 27000 tokens.)
        const float goal = (float)set.top_p * guess;
        const auto error = [&]() __attribute__((always_inline)) { return 0.001f * guess + 0.02f * front_hidden + 6.0f * __builtin_amdgcn_sqrtf(fmaxf(front_square, 0.0f)); };
        m = before;
        float off = error();
        bool upper = tid > 0 && front + off >= goal, lower = tid > 0 && front - off >= goal;             // (a bin has passed the goal)
#pragma unroll
        for (int j = 0; j < per; ++j) {
            m += c[j];
            front += known[j] + hidden[j];
            front_hidden += hidden[j];
            front_square += square[j];
            off = error();
            if (!upper && front + off >= goal) { atomicMin(&s.found_bins[0], per * tid + j); upper = true; }
            if (!lower && front - off >= goal && (float)m <= most) { atomicMin(&s.found_bins[1], per * tid + j); lower = true; }
        }
        __syncthreads();
        first = s.found_bins[0];
        last = s.found_bins[1];
        // what a short list holds is taken out from the top on
        if (last < kBins && last / per == tid) {
            m = before;
            for (int j = 0; j <= last % per; ++j) m += c[j];
            s.found_i = (int)tokens(m);
        }
        __syncthreads();
        if (last >= kBins) {                                       // (a guess that ends before it gets there)
            last = vocab <= kTaken ? kBins - 1 : -1;
            first = first == kBins - 1 ? 0 : first;
        } else if (s.found_i < kList / 2) {
            first = 0;
        }
        // (all tokens above the window are kept: none is less than min_p)
        if (set.min_p > 0.0) first = min(first, max((int)(fmin(-log2(set.min_p), 64.0) * 64.0) - 2, 0));
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

// Takes the indices of the tokens of the window's bins (and of some of the next ones: those that are not beyond its bounds in binary32; never of -inf) out of pieces first,
// first + step, .., multiples of 64 lanes (s.filled counts them, also those that s.taken has no room for); returns the thread's sum of all weights, and in `upper` that of the
// tokens above the window, which go into stretches[] as well (by stretches).  With k the sum is for the log-probability alone, and formed in binary32 by eights (a weight is off
// by 2^-19 at a depth of 40 octaves, 2^-22 where it counts).
struct Window {
    float lowest, highest;
    __device__ __forceinline__ Window(const Limits& limits, const Weigher& w)
    {
        lowest = limits.last < 0 ? INFINITY : fmaxf(w.lowest(limits.last), -3.4028234e38f);
        highest = w.highest(limits.first);
    }
};
template <bool F32, int TAKEN, class S>
__device__ __forceinline__ double take_down(S& s, const RowSettings& set, const LogitRow<F32>& row, const Weigher& w, const Limits& limits, int first, int end, int step, double* stretches,
                                            double& upper)
{
    double sum = 0.0;
    upper = 0.0;
    const Window window(limits, w);
    const auto take = [&](const float* x, uint32_t n, int i) __attribute__((always_inline)) {
        if (!__any(n > 0)) return;
        const uint32_t upto = wave_scan(n);
        uint32_t at = 0;
        if ((threadIdx.x & 63) == 63) at = atomicAdd(&s.filled, upto);
        at = lane_value(at, 63) + upto - n;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (x[j] >= window.lowest && x[j] <= window.highest) {
                if (at < (uint32_t)TAKEN) s.taken[at] = (uint32_t)(i + j);
                ++at;
            }
    };
    if (set.by_k && w.rate < kLowTemperatures) {
        row.each(first, end, step, [&](float* x, int p) {
            w.settle(x);
            float eight = 0.0f;
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                eight += __builtin_amdgcn_exp2f((x[j] - w.top32) * w.rate32);
                n += x[j] >= window.lowest ? 1u : 0u;
            }
            sum += (double)eight;
            take(x, n, row.index(p));
        });
    } else {
        row.each(first, end, step, [&](float* x, int p) {
            w.settle(x);
            uint32_t n = 0;
            double over = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                double v[2];
                w.weights(x[j], x[j + 1], v[0], v[1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    sum += v[e];
                    over = fma(v[e], __longlong_as_double((long long)((uint64_t)(x[j + e] > window.highest ? 0x3ff00000u : 0u) << 32)), over);
                    n += x[j + e] >= window.lowest && x[j + e] <= window.highest ? 1u : 0u;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            upper += over;
            if (__any(over > 0.0)) over = wave_scan(over);
            if ((threadIdx.x & 63) == 63 && p / 64 < kBins) stretches[p / 64] = over;
            take(x, n, row.index(p));
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
        for (int j = 0; j < 8; j += 2) {
            const Weigher::Depth d[2] = {w.depth(x[j]), w.depth(x[j + 1])};
            double v[2];
            if (set.by_p) w.parts(d[0].r, d[1].r, v[0], v[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int b = min(d[e].bin, kBins - 1);
                if (set.by_p && b <= limit) atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)w.units(v[e], d[e]));
                if (set.by_k) atomicAdd(&s.count[b], 1u);
            }
            __builtin_amdgcn_sched_barrier(0);                     // (two tokens' chains side by side are enough, and eight want more registers than there are)
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
    __device__ __forceinline__ Kept(uint64_t threshold_, const RowSettings& set, const Weigher& w) : threshold(threshold_), min_p(set.min_p)
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
    // of eight neighbours, i the index of the first; PASS: in a pass over the row
    template <bool PASS> __device__ __forceinline__ double eight(const Weigher& w, const float* x, int i) const
    {
        double sum = 0.0;
        if (whole) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                double v[2];
                w.weights(x[j], x[j + 1], v[0], v[1]);
                sum += v[0] + v[1];
                __builtin_amdgcn_sched_barrier(0);
            }
            return sum;
        }
        float most = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) most = fmaxf(most, x[j]);
        if (PASS && __popcll(__ballot(most >= floor)) > 16) {                        // (many: all weights, side by side, are sooner there)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                double v[2];
                w.weights(x[j], x[j + 1], v[0], v[1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) sum += may(x[j + e], i + j + e) && v[e] >= min_p ? v[e] : 0.0;
                __builtin_amdgcn_sched_barrier(0);
            }
            return sum;
        }
        // (of equal logits only those with lower indices than the threshold's)
        each_of_eight(x, [&](float y) { return y >= floor; }, [&](float y, int j) { sum += one(w, y, i + j); });
        return sum;
    }
};

// K1's and K2's threshold from the sorted list of the window's n tokens, K1's among them; without k, `total` is the sum of all weights and `upper` of those above the window, and
// the answer false where K2 ends elsewhere.
__device__ __forceinline__ bool threshold_of_list(RowShared& s, const RowSettings& set, const Weigher& w, uint32_t n, double total, double upper, uint64_t& threshold)
{
    const int tid = thread_anew();
    const uint32_t limit = set.by_k ? min((uint32_t)set.top_k, n) : n;
    double all;
    const double v = tid < (int)limit ? w.weight(risen((uint32_t)(s.list[tid] >> 24))) : 0.0;
    const double before = upper + (scan<kSampleThreads>(v, s.waves_d, all) - v), goal = set.by_p ? set.top_p * (set.by_k ? all : total) : INFINITY;
    if (!set.by_k && (upper >= goal || upper + all < goal)) return false;
    if (tid == 0) s.found_i = 0;
    __syncthreads();
    if (tid < (int)limit && before < goal) atomicMax(&s.found_i, tid);
    __syncthreads();
    threshold = s.list[s.found_i];
    return true;
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
    const double mine = kept.eight<false>(w, x, i), incl = wave_scan(mine);
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
    const int who = hits ? __ffsll((unsigned long long)hits) - 1 : live ? 63 - __clzll((unsigned long long)live) : 0;
    if (lane != who) return;
    if (!hits && !live) {                                          // (a stretch is chosen for a weight that the draw sees too)
        answer(a, r, -1, __builtin_nan(""));
    } else {
        const int j = hits ? found : behind;
        float xt = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) xt = e == j ? x[e] : xt;
        answer(a, r, i + j, w.log_weight(xt) - log(total));
    }
}

// Thresholds and the draw.  total: the sum of all weights (< 0: it is what is kept); limits: the bins of which s.filled tokens were taken out, `upper` the weights above them.
// ready: there are no thresholds, and the sums of the stretches are in s.weight.
template <bool F32>
__device__ __forceinline__ void finish_row(RowShared& s, const SampleArgs& a, int r, const RowSettings& set, const LogitRow<F32>& row, const Weigher& w, double total, double upper,
                                           const Limits& limits, bool ready)
{
    const int tid = threadIdx.x;
    constexpr int per = kBins / kSampleThreads;
    const uint32_t filled = s.filled;
    uint64_t threshold = ~0ull;
    double kept_sum = total;                                       // sum(K1)
    int last = kBins;                                              // the bin that K1 ends in
    const int stretches = (row.pieces + 63) / 64;
    bool taken = limits.last >= 0 && stretches <= kBins && filled <= (uint32_t)kTaken, found_in_list = false;
    if (taken && filled <= (uint32_t)kList) {
        const uint32_t n = take_again(s, row, w, filled, -1);
        sort_list(s, list_size(n));
        taken = found_in_list = threshold_of_list(s, set, w, n, total, upper, threshold);
    }
    if (!found_in_list && (set.by_k || set.by_p)) {
        // the deepest bin that p's threshold can lie in: V tokens further down have less than half of what K2 leaves out
        const auto pass = [&]() __attribute__((always_inline)) {
            const double bins = (log2(2.0 * (double)a.vocab) - log2((1.0 - set.top_p) * total)) * 64.0 + 2.0;
            taken = false;
            fill_bins<F32>(s, set, row, w, set.by_k || !(bins < (double)(kBins - 1)) ? kBins - 1 : max((int)bins, 0));
        };
        if (taken) fill_bins_again(s, row, w, filled, limits.last);
        else pass();
#pragma unroll 1
        for (int stage = 0; stage < 2; ++stage) {                  // top_k, then top_p
            if (!(stage ? set.by_p : set.by_k)) continue;
            // the bin: k by the bins' counts, p by their weights
            const double goal = stage ? set.top_p * kept_sum : (double)(uint32_t)set.top_k;
            const auto held = [&](int b) __attribute__((always_inline)) { return stage ? (double)s.weight[b] * w.unit(b) : (double)s.count[b]; };
            int b;
            uint32_t n;
            double in_front;
#pragma unroll 1
            for (;;) {
                double sum = 0.0, all;
#pragma unroll
                for (int j = 0; j < per; ++j) sum += held(per * tid + j);
                if (tid == 0) s.found_i = INT32_MAX;
                const double over = taken && !set.by_k ? upper : 0.0;                    // (nothing lies above what k takes out)
                double front = over + (scan<kSampleThreads>(sum, s.waves_d, all) - sum);
                if (taken && (over + all < goal || (over > 0.0 && over >= goal))) {      // the window missed it
                    pass();
                    continue;
                }
                // The first bin that reaches the goal.  (Where a thread's sums begin and where the one before it ended, two roundings of one sum, a goal may lie between them: then
                // it is the latter's bin, or the former's first.)
                int mine = INT32_MAX;
                double mine_front = 0.0;
#pragma unroll
                for (int j = 0; j < per; ++j) {
                    const int at = per * tid + j;
                    const double here = held(at), up = stage && at == last ? kept_sum : front + here;
                    if (mine == INT32_MAX && here > 0.0 && at <= last && up >= goal) {
                        mine = at;
                        mine_front = front;
                    }
                    front += here;
                }
                const uint64_t reach = __ballot(mine != INT32_MAX);
                if (reach && (tid & 63) == __ffsll((unsigned long long)reach) - 1) atomicMin(&s.found_i, mine);
                __syncthreads();
                b = s.found_i == INT32_MAX ? -1 : s.found_i;
                if (mine == b) s.found_d[0] = mine_front;
                __syncthreads();
                in_front = s.found_d[0];
                __syncthreads();
                n = b < 0 ? 0 : taken ? take_again(s, row, w, filled, b) : take_out<F32>(s, row, w, b, 0, 0);
                if (!taken || (b >= 0 && n <= (uint32_t)kList)) break;
                pass();
            }
            if (b < 0) continue;
            const Wanted want = {stage == 1, stage ? 0 : (uint32_t)goal - (uint32_t)in_front, stage ? (goal - in_front) / w.unit(b) : 0.0};
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
        for (int k = tid; k < stretches; k += kSampleThreads) s.weight[k] = 0;
        __syncthreads();
        each_taken(s, row, w, filled, [&](float x, int index) {
            const double v = kept.one(w, x, index);
            // (no less than one unit: the number 0 falls into the first kept token, however little it weighs)
            if (v > 0.0) atomicAdd((unsigned long long*)&s.weight[(index + row.shift) / 512], (unsigned long long)(fmax(v * kKeptUnit, 1.0) + 0.5));
        });
        __syncthreads();
    }
    double done = 0.0, goal = 0.0, chosen_front = 0.0, v[per], sum = 0.0, incl = 0.0, all = 0.0;
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
                    const double sum = wave_scan(kept.template eight<true>(w, x, row.index(p)));
                    if ((tid & 63) == 63) stretch[p / 64 - first] = sum;
                });
                __syncthreads();
            }
            if (round == 0 || stretches > kBins) {
                sum = 0.0;
#pragma unroll
                for (int j = 0; j < per; ++j) {
                    v[j] = per * tid + j >= here ? 0.0
                           : taken               ? (double)s.weight[per * tid + j] * (1.0 / kKeptUnit) + (set.by_k ? 0.0 : s.above[per * tid + j])
                                                 : stretch[per * tid + j];
                    sum += v[j];
                }
                incl = scan<kSampleThreads>(sum, s.waves_d, all);
            }
            if (round == 1) {
                double at = done + (incl - sum);
                int hit = -1, live = -1;
#pragma unroll
                for (int j = 0; j < per; ++j) {
                    at += v[j];
                    if (v[j] > 0.0) {
                        if (hit < 0 && at > goal) hit = first + per * tid + j;
                        live = first + per * tid + j;
                    }
                }
                const uint64_t hits = __ballot(hit >= 0), lives = __ballot(live >= 0);
                hit = lane_value(hit, hits ? __ffsll((unsigned long long)hits) - 1 : 0);
                live = lane_value(live, lives ? 63 - __clzll((unsigned long long)lives) : 0);
                if ((thread_anew() & 63) == 0) {
                    if (hits) atomicMin(&s.found_i, hit);
                    if (lives) atomicMax((int*)&s.filled, live);
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
    const int r = blockIdx.x;
    const RowSettings set(a, r);
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    constexpr int SLOTS = kShares / kSampleThreads;
    float mine[SLOTS], most, guess;
    own_largest<F32, SLOTS>(row, threadIdx.x, row.pieces, kSampleThreads, SLOTS, guess_rate(set), mine, most, guess);
    float top = mine[0];                                           // (a NaN is there)
#pragma unroll
    for (int k = 1; k < SLOTS; ++k) top = top != top ? top : fmaxf(top, mine[k]);
    top = largest<kSampleThreads>(top, s.tops);
    if (!(top > -INFINITY) || !set.fit()) {                        // nothing to draw from, or no way to
        if (thread_anew() == 0) answer(a, r, -1, __builtin_nan(""));
        return;
    }
    const Weigher w(top, set.rate());
    const float rest[1] = {guess_rate(set) > 0.0f ? rest_of(mine, most, guess, guess_rate(set)) : -INFINITY};
    if (guess_rate(set) > 0.0f) guess = guessed_sum<kSampleThreads>(most, guess, top, guess_rate(set), reinterpret_cast<float*>(s.waves_n));
    Limits limits;
    limits.find<kSampleThreads>(s, set, w, mine, rest, kSampleThreads, guess, a.vocab, row.pieces);
    if (thread_anew() == 0) s.filled = 0;
    __syncthreads();
    double total = -1.0, upper = 0.0;
    if (set.by_k || set.by_p || set.min_p > 0.0) {
        double some;
        const double own = take_down<F32, kTaken>(s, set, row, w, limits, thread_anew(), (row.pieces + 63) / 64 * 64, kSampleThreads, s.above, some);
        scan<kSampleThreads>(own, s.waves_d, total);
        scan<kSampleThreads>(some, s.waves_d, upper);
    }
    finish_row<F32>(s, a, r, set, row, w, total, upper, limits, false);
}

// whether a row's stretches of 512 tokens fit in place of its bins
__device__ __forceinline__ bool stretches_fit(int pieces) { return (pieces + 63) / 64 <= kBins; }

// Rows in parts, three launches.  1: the maxima of the row's shares, and the guess of the weights' sum; the number of tokens taken out cleared.
template <bool F32>
__global__ __launch_bounds__(kPartThreads) void sample_tops_kernel(const SampleArgs a)
{
    __shared__ float waves[kPartThreads / 64];
    const int r = blockIdx.x / a.parts, part = blockIdx.x - r * a.parts, tid = threadIdx.x;
    const RowSettings set(a, r);
    const LogitRow<F32> row(static_cast<const char*>(a.logits) + (size_t)r * a.ld * (F32 ? 4 : 2), a.vocab);
    const int at = part * kPartThreads + tid, all = a.parts * kPartThreads;
    constexpr int SLOTS = kShares / (4 * kPartThreads);            // (a thread's pieces are dealt to several shares)
    const int slots = kShares / all;
    const float rate = guess_rate(set);
    float top[SLOTS], most, guess;
    own_largest<F32, SLOTS>(row, at, row.pieces, all, slots, rate, top, most, guess);
    if (rate > 0.0f) {
        const float highest = largest<kPartThreads>(most, waves);
        __syncthreads();
        const float sum = guessed_sum<kPartThreads>(most, guess, highest, rate, waves);
        if (tid < 2) a.guesses[2 * ((size_t)r * a.parts + part) + tid] = tid ? sum : highest;
    }
    if (rate > 0.0f) a.rests[(size_t)r * kShares + at] = rest_of(top, most, guess, rate);
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
        if (k < slots) a.tops[(size_t)r * kShares + k * all + at] = top[k];
    if (at == 0) a.filled[r] = 0;
}

__device__ __forceinline__ float row_top(const SampleArgs& a, int r, float (&mine)[kShares / kPartThreads], float* waves)
{
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < kShares / kPartThreads; ++j) {
        mine[j] = a.tops[(size_t)r * kShares + threadIdx.x + j * kPartThreads];
        nan |= mine[j] != mine[j];
        top = fmaxf(top, mine[j]);
    }
    return largest<kPartThreads>(nan ? __builtin_nanf("") : top, waves);
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
    const float top = row_top(a, r, mine, s.tops);
    if (part == 0 && tid == 0) a.limits[3 * (size_t)r + 2] = __float_as_int(top);
    if (!(top > -INFINITY) || !set.fit()) return;
    const Weigher w(top, set.rate());
    float guess = 0.0f, rest[kShares / kPartThreads];
#pragma unroll
    for (int j = 0; j < kShares / kPartThreads; ++j) rest[j] = guess_rate(set) > 0.0f && j < a.parts ? a.rests[(size_t)r * kShares + j * kPartThreads + tid] : -INFINITY;
    if (guess_rate(set) > 0.0f) {
        const float* const told = a.guesses + 2 * (size_t)r * a.parts;
        guess = guessed_sum<kPartThreads>(tid < a.parts ? told[2 * tid] : -INFINITY, tid < a.parts ? told[2 * tid + 1] : 0.0f, top, guess_rate(set), reinterpret_cast<float*>(s.waves_n));
    }
    Limits limits;
    limits.find<kPartThreads>(s, set, w, mine, rest, a.parts * kPartThreads, guess, a.vocab, row.pieces);
    if (part == 0 && tid == 0) {
        a.limits[3 * (size_t)r] = limits.first;
        a.limits[3 * (size_t)r + 1] = limits.last;
    }
    if (tid == 0) s.filled = 0;
    __syncthreads();
    double sum = 0.0, some = 0.0;
    if (set.by_k || set.by_p || !stretches_fit(row.pieces)) {
        sum = take_down<F32, kPartTaken>(s, set, row, w, limits, part * kPartThreads + tid, (row.pieces + 63) / 64 * 64, a.parts * kPartThreads, a.stretches + (size_t)r * kBins, some);
    } else {
        // no thresholds: the stretches' sums, in place of the bins
        const Kept kept(~0ull, set, w);
        row.each(part * kPartThreads + tid, (row.pieces + 63) / 64 * 64, a.parts * kPartThreads, [&](float* x, int p) {
            w.settle(x);
            const double some = wave_scan(kept.template eight<true>(w, x, row.index(p)));
            if ((tid & 63) == 63) a.stretches[(size_t)r * kBins + p / 64] = some;
            if (!kept.whole) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    double v[2];
                    w.weights(x[j], x[j + 1], v[0], v[1]);
                    sum += v[0] + v[1];
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        });
    }
    double all, upper;
    scan<kPartThreads>(sum, s.waves_d, all);
    scan<kPartThreads>(some, s.waves_d, upper);
    if (tid < 2) a.sums[2 * ((size_t)r * a.parts + part) + tid] = tid ? upper : all;
    if (limits.last < 0) return;
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
    const float top = __int_as_float(a.limits[3 * (size_t)r + 2]);
    if (!(top > -INFINITY) || !set.fit()) {
        if (tid == 0) answer(a, r, -1, __builtin_nan(""));
        return;
    }
    const Weigher w(top, set.rate());
    const bool ready = !set.by_k && !set.by_p && stretches_fit(row.pieces);
    const uint32_t filled = a.filled[r];
    Limits limits;                                                 // (those that the launch before took: sums in another order might give others)
    limits.first = a.limits[3 * (size_t)r];
    limits.last = a.limits[3 * (size_t)r + 1];
    if (tid == 0) s.filled = filled;
    const int stretches = min((row.pieces + 63) / 64, kBins);
    for (int b = tid; b < stretches; b += kSampleThreads) (ready ? reinterpret_cast<double*>(s.weight) : s.above)[b] = a.stretches[(size_t)r * kBins + b];
    for (uint32_t i = tid; i < filled && i < (uint32_t)kTaken; i += kSampleThreads) s.taken[i] = a.taken[(size_t)r * kTaken + i];
    const double* const sums = a.sums + 2 * (size_t)r * a.parts;
    double total, upper;
    scan<kSampleThreads>(tid < a.parts ? sums[2 * tid] : 0.0, s.waves_d, total);
    scan<kSampleThreads>(tid < a.parts ? sums[2 * tid + 1] : 0.0, s.waves_d, upper);
    finish_row<F32>(s, a, r, set, row, w, ready && !(set.min_p > 0.0) ? -1.0 : total, upper, limits, ready);
}

// Workgroups that share a row, or 0 for one workgroup and one launch.  Three launches and the row's sums on their way through memory cost 10 us or so, and a workgroup alone
// needs 35 us (top_k) to 65 and more (top_p) for 131072 tokens: rows are shared out from 65536 tokens on, as long as they fill an eighth of the device or less (from 131072: a
// quarter).  In parts and alone, no thresholds / top_k = 50 / top_p = 0.95: a row of 131072 18 / 27 / 40 and 41 / 37 / 70, of 65536 19 / 27 / 36 and 25 / 28 / 45, of 50000 20 / 27 / 33
// and 21 / 24 / 35, of 32003 21 / 28 / 36 and 18 / 22 / 30; 64 rows of 131072 35 / 40 / 78 and 41 / 37 / 85, of 65536 27 / 33 / 52 and 26 / 28 / 54.
static int row_parts(int64_t rows, int64_t vocab)
{
    const int64_t room = (int64_t)device_cus() / rows;
    if (vocab < 65536 || room < 4 || rows * 131072 > (int64_t)device_cus() / 4 * vocab) return 0;
    int parts = 4;                                                 // (as many threads as a row has alone, or more)
    while (parts < 32 && parts * 2 <= room && vocab >= (int64_t)parts * 2 * kPartThreads * 16) parts *= 2;
    return parts;
}

struct SampleSpace {
    size_t tops, guesses, rests, sums, stretches, taken, filled, limits, bytes;
    SampleSpace(int64_t rows, int parts)
    {
        const size_t n = (size_t)rows;
        stretches = 0;
        sums = n * kBins * 8;
        taken = sums + n * (size_t)parts * 16;
        tops = taken + n * kTaken * 4;
        guesses = tops + n * kShares * 4;
        rests = guesses + n * (size_t)parts * 8;
        filled = rests + n * kShares * 4;
        limits = filled + n * 4;
        bytes = limits + n * 12;
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
        a.guesses = reinterpret_cast<float*>(base + space.guesses);
        a.rests = reinterpret_cast<float*>(base + space.rests);
        a.sums = reinterpret_cast<double*>(base + space.sums);
        a.stretches = reinterpret_cast<double*>(base + space.stretches);
        a.taken = reinterpret_cast<uint32_t*>(base + space.taken);
        a.filled = reinterpret_cast<uint32_t*>(base + space.filled);
        a.limits = reinterpret_cast<int*>(base + space.limits);
    }
    const bool f32 = dtype == METIS_DTYPE_F32;
    if (a.parts) {                                                 // (rows that a small part of the device's compute units takes)
        const dim3 grid((unsigned)rows), parts((unsigned)(rows * a.parts));
#define METIS_SAMPLE_PARTS(F)                                                                   \
    do {                                                                                        \
        hipLaunchKernelGGL(sample_tops_kernel<F>, parts, dim3(kPartThreads), 0, st, a);         \
        hipLaunchKernelGGL(sample_bins_kernel<F>, parts, dim3(kPartThreads), 0, st, a);         \
        hipLaunchKernelGGL(sample_finish_kernel<F>, grid, dim3(kSampleThreads), 0, st, a);      \
    } while (0)
        if (f32) METIS_SAMPLE_PARTS(true);
        else METIS_SAMPLE_PARTS(false);
#undef METIS_SAMPLE_PARTS
        return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
    }
    constexpr int64_t most = (int64_t)UINT32_MAX / kSampleThreads;                    // rows of a launch
    for (int64_t first = 0; first < rows; first += most) {
        SampleArgs some = a;
        some.logits = static_cast<const char*>(logits) + (size_t)first * (size_t)ld * (f32 ? 4 : 2);
        some.uniforms += first;
        if (some.row_parameters) some.row_parameters += 4 * first;
        some.tokens += first;
        some.logprobs += first;
        some.rows = (int)(rows - first < most ? rows - first : most);
        if (f32) hipLaunchKernelGGL(sample_kernel<true>, dim3((unsigned)some.rows), dim3(kSampleThreads), 0, st, some);
        else hipLaunchKernelGGL(sample_kernel<false>, dim3((unsigned)some.rows), dim3(kSampleThreads), 0, st, some);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    return METIS_OK;
}

}  // namespace metis
