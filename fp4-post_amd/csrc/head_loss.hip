// Log-probabilities of given tokens under a large head, without the logits, and their gradients (gfx950).
//
//   l[t, v] = sum_k hidden[t, k] weight[v, k] / temperature
//   lse[t] = log sum_v exp l,   logp[t] = l[t, target] - lse,   H[t] = lse - sum_v p l,   p = exp(l - lse)
// and for gradients g of logp and e of H
//   dl = (g (1[v = target] - p) - e p (l - lse + H)) / temperature
//   grad_hidden = dl weight,   grad_weight = dl^T hidden
//
// All three products run on one tile engine (below).  Forward: every 256-column tile of the logits leaves, per token, its maximum and its sum of
// exponentials (and of p l) from the accumulators; a second launch folds the tiles.  Backward: pieces of the vocabulary one after the other; a piece's
// logits are formed again, turned into dl in the accumulators, rounded to bf16 once (the type in which both products take it: its 2^-9 is that of the
// gradients' own rounding and averages out in the sums) and kept only until the piece's two products have read it.  The gradient of hidden is summed in
// binary32 over the pieces.
//
// Tokens whose target is ignored take no part: a first launch lists the others ("live"), the products run over the listed rows, and what an ignored
// row of hidden holds (padding: anything) is never read into a sum.
#include "gemm_common.h"

namespace metis {

namespace {

constexpr int HL_BN = 256, HL_TN = 2, HL_THREADS = 512;

__host__ __device__ constexpr int hl_stage_bytes(int TM) { return (64 * TM + HL_BN) * 64; }
__host__ __device__ constexpr int hl_slots(int TM) { return 4; }

__host__ __device__ constexpr int hl_waitcnt(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | ((lgkm & 15) << 8); }
#define HL_WAIT(VM, LGKM) __builtin_amdgcn_s_waitcnt(hl_waitcnt(VM, LGKM))

typedef short hl_short4_t __attribute__((ext_vector_type(4)));
typedef short hl_short8_t __attribute__((ext_vector_type(8)));
typedef uint32_t hl_u32x4_t __attribute__((ext_vector_type(4)));
typedef hl_short4_t __attribute__((address_space(3))) * hl_lds_ptr_t;

// ---------------------------------------------------------------------------------------------
// The tile engine: 64 TM x 256 of a product per workgroup, eight waves (2 x 4) of 32 TM x 64, stages of 32 along the contraction in a ring of four
// LDS slots, filled by direct loads three stages ahead; one barrier a stage, waits that never drain the queue.
//
// An operand lies in memory either along the contraction ("plain": [row][k]) or across it ("turned": [k][row]); both go to LDS as they are, 1 KiB per load
// instruction.  Plain: 16 rows of 64 bytes, the four 16-byte pieces of row q in the order c ^ swz(q), read back as ds_read_b128.  Turned: rows of k, whose
// 64-byte segments are exchanged by f(k) so that the four rows which a transposing read (ds_read_b64_tr_b16) takes at once lie in different banks; two
// such reads give a lane its eight consecutive k.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int hl_swz(int q) { return ((q >> 2) & 1) | ((((q >> 1) ^ (q >> 3)) & 1) << 1); }
template <int ROW_BYTES> __device__ __forceinline__ int hl_turn(int k) { return ROW_BYTES >= 256 ? (k & 3) << 6 : ((k >> 1) & 1) << 6; }

struct Operand {
    const uint16_t* base;        // first element of the tile's rows (plain) or of the first k's row (turned)
    int64_t ld;                  // elements between rows (plain) or between k (turned)
    int limit;                   // rows from here on are not there: the last one is read in their place
    const int* index;            // plain: the rows' numbers, or nullptr for rows as they come
    int rest;                    // k of the last stage that are there: 16 or 32 (plain), 1 .. 32 (turned); in place of others some that are there are read
};

// Stages [0, steps) of 32 along the contraction; half: only the first sixteen k of the last one count.  Where fewer count otherwise, one operand holds zeros
// beyond them.
template <int TM, bool AT, bool BT>
__device__ __forceinline__ void hl_main_loop(float16_t (&acc)[TM][HL_TN], uint8_t* lds, const Operand& a, const Operand& b, int steps, bool half)
{
    constexpr int BM = 64 * TM, NA = BM / 16, TOTAL = NA + HL_BN / 16, LPW = (TOTAL + 7) / 8, STAGE = hl_stage_bytes(TM), NS = hl_slots(TM), B_AT = NA * 1024;
    constexpr int A_RB = BM * 2, B_RB = HL_BN * 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3;

    // ---- this wave's load instructions of a stage: where its lanes read in the first one, how far they go per stage, and back in the last
    const uint8_t* src[LPW];
    int64_t inc[LPW];
    uint32_t back[LPW];
    int place[LPW];
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
        int ot = j * 8 + wave;
        if (ot >= TOTAL) ot -= 8;                              // (a piece that another wave loads too: the same bytes to the same place)
        place[j] = ot * 1024;
        const bool is_a = ot < NA;
        const Operand& o = is_a ? a : b;
        const int q = is_a ? ot : ot - NA;
        if (is_a ? AT : BT) {
            const int rb = is_a ? A_RB : B_RB, k = q * (1024 / rb) + lane * 16 / rb, at = lane * 16 % rb;
            int col = (at ^ (is_a ? hl_turn<A_RB>(k) : hl_turn<B_RB>(k))) >> 1;
            if (col >= o.limit) col = 0;                       // (columns in eights: all there or none)
            src[j] = reinterpret_cast<const uint8_t*>(o.base + (int64_t)k * o.ld + col);
            inc[j] = o.ld * 64;
            back[j] = k >= o.rest ? (uint32_t)((k - (o.rest - 1)) * (o.ld * 2)) : 0u;
        } else {
            const int row = q * 16 + (lane >> 2), chunk = (lane & 3) ^ hl_swz(row & 15);
            int r = row < o.limit ? row : o.limit - 1;
            const int64_t at = o.index ? o.index[r] : r;
            src[j] = reinterpret_cast<const uint8_t*>(o.base + at * o.ld + chunk * 8);
            inc[j] = 64;
            back[j] = chunk * 8 >= o.rest ? 32u : 0u;
        }
    }
    auto issue_one = [&](int slot, int j, bool last) {
        const uint8_t* g = src[j] - (last ? back[j] : 0u);
        const uint32_t dst = (uint32_t)(slot * STAGE + place[j]);
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(g), "s"(dst) : "memory");
        src[j] += inc[j];
    };

    // ---- fragments: lane -> row l % 32 of a 32-row tile, k 8 (l / 32) .. + 7 of a half stage
    const int lr = lane & 31, hi = lane >> 5;
    const int plain = (lr >> 4) * 1024 + (lr & 15) * 64 + ((hi ^ hl_swz(lr & 15)) * 16);
    int a_off[AT ? TM : 2], b_off[BT ? HL_TN : 2];
    const int tk = 8 * hi + ((lane & 15) >> 2), tc = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    if constexpr (AT) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a_off[i] = tk * A_RB + (((wm * TM + i) * 64) ^ hl_turn<A_RB>(tk)) + tc;
    } else {
        a_off[0] = wm * TM * 2048 + plain;
        a_off[1] = wm * TM * 2048 + (plain ^ 32);
    }
    if constexpr (BT) {
#pragma unroll
        for (int j = 0; j < HL_TN; ++j) b_off[j] = B_AT + tk * B_RB + (((wn * HL_TN + j) * 64) ^ hl_turn<B_RB>(tk)) + tc;
    } else {
        b_off[0] = B_AT + wn * HL_TN * 2048 + plain;
        b_off[1] = B_AT + wn * HL_TN * 2048 + (plain ^ 32);
    }
    uint4 fa[2][TM], fb[2][HL_TN];
    auto turned = [&](const uint8_t* p, int rb) -> uint4 {
        const hl_short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((hl_lds_ptr_t)p);
        const hl_short4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((hl_lds_ptr_t)(p + 4 * rb));
        const hl_short8_t v = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
        return __builtin_bit_cast(uint4, v);
    };
    auto load_frags = [&](int slot, int ks) {
        const uint8_t* x = lds + slot * STAGE;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if constexpr (AT) fa[ks][i] = turned(x + a_off[i] + ks * 16 * A_RB, A_RB);
            else fa[ks][i] = *reinterpret_cast<const uint4*>(x + a_off[ks] + i * 2048);
        }
#pragma unroll
        for (int j = 0; j < HL_TN; ++j) {
            if constexpr (BT) fb[ks][j] = turned(x + b_off[j] + ks * 16 * B_RB, B_RB);
            else fb[ks][j] = *reinterpret_cast<const uint4*>(x + b_off[ks] + j * 2048);
        }
    };
    auto mfma_one = [&](int ks, int i, int j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, fb[ks][j]), __builtin_bit_cast(bf16x8_t, fa[ks][i]), acc[i][j], 0, 0, 0);
    };
    auto mfmas = [&](int ks) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < HL_TN; ++j) mfma_one(ks, i, j);
    };
    constexpr int NM = TM * HL_TN, NF = TM * (AT ? 2 : 1) + HL_TN * (BT ? 2 : 1);

    if (steps <= 0) return;
#pragma unroll
    for (int p = 0; p < NS; ++p)
        if (p < steps) {
#pragma unroll
            for (int j = 0; j < LPW; ++j) issue_one(p, j, p == steps - 1);
        }
    if (steps >= NS) HL_WAIT((NS - 1) * LPW, 15);
    else HL_WAIT(0, 15);
    __syncthreads();
    load_frags(0, 0);
    int s = 0, slot = 0;
    for (; s + NS < steps; ++s) {
        const int nslot = slot + 1 == NS ? 0 : slot + 1;
        const bool last = s + NS == steps - 1;
        load_frags(slot, 1);
        mfmas(0);
        sched_substep<NM, 0, NF, 0>();
        HL_WAIT((NS - 2) * LPW, 0);                            // own loads of stage s + 1 are there, own reads of stage s done
        __syncthreads();
        load_frags(nslot, 0);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
#pragma unroll
            for (int j = 0; j < LPW; ++j)
                if (j * NM / LPW == m) issue_one(slot, j, last);
            mfma_one(1, m / HL_TN, m % HL_TN);
        }
        slot = nslot;
    }
    for (; s < steps; ++s) {
        const int nslot = slot + 1 == NS ? 0 : slot + 1;
        const bool both = s + 1 < steps || !half;
        if (both) load_frags(slot, 1);
        mfmas(0);
        HL_WAIT(0, 0);
        __syncthreads();
        if (s + 1 < steps) load_frags(nslot, 0);
        if (both) mfmas(1);
        slot = nslot;
    }
    __syncthreads();                                           // the ring is free
}

// acc[i][j][e] of lane l: row 32 (TM wm + i) + l % 32, column 64 wn + 32 j + 8 (e / 4) + 4 (l / 32) + e % 4 of the tile.
// The tile as bf16, rows of `ld` elements from `out` on: through the wave's own part of LDS, 32 rows at a time, so that a store writes 8 rows of 128 bytes.
template <int TM>
__device__ __forceinline__ void hl_store_bf16(const float16_t (&acc)[TM][HL_TN], uint8_t* lds, uint16_t* out, int64_t ld, int rows, int cols)
{
    constexpr int CROW = 72;                                   // 144 bytes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    uint16_t* cw = reinterpret_cast<uint16_t*>(lds) + wave * (32 * CROW);
    const int n = wn * 64 + (lane & 7) * 8;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < HL_TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float16_t& v = acc[i][j];
                *reinterpret_cast<uint2*>(cw + lr * CROW + j * 32 + 8 * g + 4 * hi) =
                    make_uint2(rb_pair(v[4 * g], v[4 * g + 1]), rb_pair(v[4 * g + 2], v[4 * g + 3]));
            }
        __builtin_amdgcn_s_waitcnt(hl_waitcnt(63, 0));         // the wave reads back what it wrote itself
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int ml = it * 8 + (lane >> 3), m = (wm * TM + i) * 32 + ml;
            const uint4 w = *reinterpret_cast<const uint4*>(cw + ml * CROW + (lane & 7) * 8);
            if (m < rows && n < cols) *reinterpret_cast<uint4*>(out + m * ld + n) = w;
        }
        __builtin_amdgcn_s_waitcnt(hl_waitcnt(63, 0));
        __builtin_amdgcn_wave_barrier();
    }
}

// What the launches share about the tokens: index[0] the number of live ones, index[64 ..] their rows in order, index[64 + tokens ..] each row's place
// among them or -1.
struct Tokens {
    const uint16_t* hidden;
    int64_t ld;
    const int64_t* targets;
    const int* index;
    int tokens, H, V;
    float scale2;                // log2(e) / temperature: logits in powers of two
};
__device__ __forceinline__ const int* live_rows(const int* index) { return index + 64; }

// workgroup -> tile, a contiguous range of the tiles per XCD
__device__ __forceinline__ int hl_logical(int total)
{
    const int per = (total + 7) >> 3, logical = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    return (int)(blockIdx.x >> 3) < per && logical < total ? logical : -1;
}
// groups of four tile rows, walked column by column
__device__ __forceinline__ void hl_origin(int logical, int tiles_m, int tiles_n, int& tm, int& tn)
{
    constexpr int GM = 4;
    const int group = logical / (GM * tiles_n), first = group * GM, size = min(tiles_m - first, GM), in = logical - group * GM * tiles_n;
    tm = first + in % size;
    tn = in / size;
}

template <int TM> __device__ __forceinline__ void hl_clear(float16_t (&acc)[TM][HL_TN])
{
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < HL_TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
}

// ---------------------------------------------------------------------------------------------
// Forward: per tile and live token the maximum of its logits (in powers of two), the sum of 2^(l - maximum) and, for the entropy, of
// 2^(l - maximum) (l - maximum); the target's logit from the tile that has it.
// ---------------------------------------------------------------------------------------------
template <int TM, bool ENT>
__global__ __launch_bounds__(HL_THREADS, TM == 1 ? 4 : 2) void head_stats_kernel(const Tokens tk, const uint16_t* __restrict__ weight, int64_t ldw, int stride,
                                                                               float2* __restrict__ part, float* __restrict__ part_e, float* __restrict__ hit)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t hl_lds[];
    constexpr int BM = 64 * TM;
    const int count = tk.index[0], tiles_m = (count + BM - 1) / BM, tiles_n = (tk.V + HL_BN - 1) / HL_BN;
    const int logical = hl_logical(tiles_m * tiles_n);
    if (logical < 0) return;
    int tm, tn;
    hl_origin(logical, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * HL_BN;
    float16_t acc[TM][HL_TN];
    hl_clear<TM>(acc);
    const int rest = tk.H % 32 ? 16 : 32;
    const Operand a = {tk.hidden, tk.ld, count - m0, live_rows(tk.index) + m0, rest}, b = {weight + (int64_t)n0 * ldw, ldw, tk.V - n0, nullptr, rest};
    hl_main_loop<TM, false, false>(acc, hl_lds, a, b, (tk.H + 31) / 32, rest == 16);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    const int there = tk.V - (n0 + wn * 64);                   // columns of this wave that exist
    float* red = reinterpret_cast<float*>(hl_lds);             // [row][wave column][3]
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int row = (wm * TM + i) * 32 + lr, m = m0 + row;
        float top = -INFINITY, sum = 0.0f, ent = 0.0f;
        if (there > 0) {
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float v = acc[i][j][e] * tk.scale2;
                    if (there < 64 && j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3) >= there) v = -INFINITY;
                    acc[i][j][e] = v;
                    top = fmaxf(top, v);
                }
            top = fmaxf(top, __shfl_xor(top, 32, 64));
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float d = acc[i][j][e] - top, p = __builtin_amdgcn_exp2f(d);
                    sum += p;
                    if constexpr (ENT) ent = there < 64 && j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3) >= there ? ent : fmaf(p, d, ent);
                }
            sum += __shfl_xor(sum, 32, 64);
            if constexpr (ENT) ent += __shfl_xor(ent, 32, 64);
            int64_t want = -1;
            if (m < count) want = tk.targets[live_rows(tk.index)[m]] - (n0 + wn * 64);
            if (__any(want >= 0 && want < 64)) {
#pragma unroll
                for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (want == j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3)) hit[m] = acc[i][j][e];
            }
        }
        if (hi == 0) {
            red[(row * 4 + wn) * 3] = top;
            red[(row * 4 + wn) * 3 + 1] = sum;
            red[(row * 4 + wn) * 3 + 2] = ent;
        }
    }
    __syncthreads();
    const int row = threadIdx.x;
    if (row >= BM || m0 + row >= count) return;
    float top = red[row * 12], sum = red[row * 12 + 1], ent = red[row * 12 + 2];   // (the first wave has columns that exist)
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        if (tk.V - n0 <= w * 64) break;
        const float t = red[(row * 4 + w) * 3], s = red[(row * 4 + w) * 3 + 1], e = red[(row * 4 + w) * 3 + 2], up = fmaxf(top, t);
        const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(t - up);
        if constexpr (ENT) ent = f0 * fmaf(top - up, sum, ent) + f1 * fmaf(t - up, s, e);
        sum = f0 * sum + f1 * s;
        top = up;
    }
    part[(size_t)tn * stride + m0 + row] = make_float2(top, sum);
    if constexpr (ENT) part_e[(size_t)tn * stride + m0 + row] = ent;
}

// The tiles of a token folded: 64 chains of every 64th tile, then the chains in order; 16 tokens per workgroup.
template <bool ENT>
__global__ __launch_bounds__(1024) void head_finish_kernel(const int64_t* __restrict__ targets, const int* __restrict__ index, int tokens, int V, int tiles_n, int stride,
                                                           const float2* __restrict__ part, const float* __restrict__ part_e, const float* __restrict__ hit,
                                                           float* __restrict__ logp, float* __restrict__ lse, float* __restrict__ entropy)
{
    __shared__ float red[64][16][3];
    const int r = threadIdx.x & 15, chain = threadIdx.x >> 4, t = blockIdx.x * 16 + r;
    const int pos = t < tokens ? live_rows(index)[tokens + t] : -1;
    float top = -INFINITY, sum = 0.0f, ent = 0.0f;
    auto fold = [&](float t1, float s1, float e1) {
        const float up = fmaxf(top, t1);
        if (up == -INFINITY && s1 == 0.0f) return;             // nothing yet and nothing new
        const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(t1 - up);
        if constexpr (ENT) ent = (sum != 0.0f ? f0 * fmaf(top - up, sum, ent) : 0.0f) + f1 * fmaf(t1 - up, s1, e1);
        sum = (sum != 0.0f ? f0 * sum : 0.0f) + f1 * s1;
        top = up;
    };
    if (pos >= 0)
        for (int k = chain; k < tiles_n; k += 64) {
            const float2 p = part[(size_t)k * stride + pos];
            fold(p.x, p.y, ENT ? part_e[(size_t)k * stride + pos] : 0.0f);
        }
    red[chain][r][0] = top;
    red[chain][r][1] = sum;
    red[chain][r][2] = ent;
    __syncthreads();
    if (chain || t >= tokens) return;
    if (pos < 0) {
        logp[t] = lse[t] = 0.0f;
        if constexpr (ENT) entropy[t] = 0.0f;
        return;
    }
    for (int k = 1; k < 64 && k < tiles_n; ++k) fold(red[k][r][0], red[k][r][1], red[k][r][2]);
    constexpr float kLn2 = 0.693147180559945f;
    const int64_t want = targets[t];
    const bool there = want >= 0 && want < V;                  // (a target outside of the vocabulary shows: everything of its row is NaN)
    const float l2 = __log2f(sum), nan = __uint_as_float(0x7fc00000u);
    lse[t] = there ? (top + l2) * kLn2 : nan;
    logp[t] = there ? ((hit[pos] - top) - l2) * kLn2 : nan;
    if constexpr (ENT) entropy[t] = there ? (l2 - ent / sum) * kLn2 : nan;
}

// The live tokens in order, one workgroup.
__global__ __launch_bounds__(1024) void head_index_kernel(const int64_t* __restrict__ targets, int64_t ignore, int tokens, int* __restrict__ index)
{
    __shared__ int wave_count[2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0, turn = 0;
    for (int t0 = 0; t0 < tokens; t0 += 1024, turn ^= 1) {
        const int t = t0 + threadIdx.x;
        const bool live = t < tokens && targets[t] != ignore;
        const uint64_t mask = __ballot(live);
        if (lane == 0) wave_count[turn][wave] = __popcll(mask);
        __syncthreads();
        int before = base, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int n = wave_count[turn][w];
            if (w < wave) before += n;
            all += n;
        }
        const int at = before + __popcll(mask & ((1ull << lane) - 1ull));
        if (live) index[64 + at] = t;
        if (t < tokens) index[64 + tokens + t] = live ? at : -1;
        base += all;
    }
    if (threadIdx.x == 0) index[0] = base;
}

// ---------------------------------------------------------------------------------------------
// Backward, first launch of a piece: dl of the vocabulary's columns v0 .. v0 + width - 1 as bf16 [live tokens, padded to the tile][ld], zero where tokens or
// columns are not there.
// ---------------------------------------------------------------------------------------------
struct RowGrads {
    const float *lse, *entropy, *g_logp, *g_entropy;           // by token; entropy and g_entropy may be nullptr
};
template <int TM>
__global__ __launch_bounds__(HL_THREADS, 2) void head_dlogits_kernel(const Tokens tk, const uint16_t* __restrict__ weight, int64_t ldw, int v0, int width, const RowGrads rg,
                                                                     uint16_t* __restrict__ dl, int64_t ld)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t hl_lds[];
    constexpr int BM = 64 * TM;
    constexpr float kLn2 = 0.693147180559945f, kLog2e = 1.44269504088896f;
    const int count = tk.index[0], tiles_m = (count + BM - 1) / BM, tiles_n = (width + HL_BN - 1) / HL_BN;
    const int logical = hl_logical(tiles_m * tiles_n);
    if (logical < 0) return;
    int tm, tn;
    hl_origin(logical, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * HL_BN;
    float16_t acc[TM][HL_TN];
    hl_clear<TM>(acc);
    const int* live = live_rows(tk.index);
    const int rest = tk.H % 32 ? 16 : 32;
    const Operand a = {tk.hidden, tk.ld, count - m0, live + m0, rest}, b = {weight + (int64_t)(v0 + n0) * ldw, ldw, width - n0, nullptr, rest};
    hl_main_loop<TM, false, false>(acc, hl_lds, a, b, (tk.H + 31) / 32, rest == 16);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    const int there = width - (n0 + wn * 64);
    const float inv_t = tk.scale2 * kLn2;                      // 1 / temperature
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = m0 + (wm * TM + i) * 32 + lr;
        float lse2 = 0.0f, g = 0.0f, ge = 0.0f, h = 0.0f;
        int want = -1;
        const bool on = m < count;
        if (on) {
            const int t = live[m];
            lse2 = rg.lse[t] * kLog2e;
            if (rg.g_logp) g = rg.g_logp[t] * inv_t;
            if (rg.g_entropy) {
                ge = rg.g_entropy[t] * inv_t;
                h = rg.entropy[t];
            }
            const int64_t w = tk.targets[t] - (v0 + n0 + wn * 64);
            want = w >= 0 && w < 64 ? (int)w : -1;
        }
#pragma unroll
        for (int j = 0; j < HL_TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3);
                const float d = acc[i][j][e] * tk.scale2 - lse2, p = __builtin_amdgcn_exp2f(d);
                const float f = rg.g_entropy ? fmaf(ge, fmaf(d, kLn2, h), g) : g;
                const float v = n == want ? fmaf(-p, f, g) : -p * f;
                acc[i][j][e] = on && n < there ? v : 0.0f;
            }
    }
    hl_store_bf16<TM>(acc, hl_lds, dl + (int64_t)m0 * ld + n0, ld, BM, HL_BN);
}

// The live rows of hidden side by side, then zero rows up to a multiple of 32.
__global__ __launch_bounds__(256) void head_gather_kernel(const Tokens tk, uint4* __restrict__ out)
{
    const int count = tk.index[0], rows = (count + 31) & ~31, cpr = tk.H / 8;
    for (int m = blockIdx.x; m < rows; m += gridDim.x) {
        const uint4* src = m < count ? reinterpret_cast<const uint4*>(tk.hidden + (int64_t)live_rows(tk.index)[m] * tk.ld) : nullptr;
        for (int c = threadIdx.x; c < cpr; c += 256) out[(int64_t)m * cpr + c] = src ? src[c] : make_uint4(0u, 0u, 0u, 0u);
    }
}

// ---------------------------------------------------------------------------------------------
// Second launch of a piece: both products that read dl.  The tiles of grad_hidden (long contractions, over the piece's columns) start first, in `splits`
// ranges of it each, and those of grad_weight (over the tokens) fill the compute units beside and behind them.
//   grad_hidden: slabs [split][live tokens, padded][H] in binary32, this piece's share added to that of the ones before
//   grad_weight: rows v0 .. of the gradient, complete
// ---------------------------------------------------------------------------------------------
struct Products {
    const uint16_t* dl;          // [padded tokens][ld]
    int64_t ld;
    const uint16_t* weight;      // the piece's first row
    int64_t ldw;
    const uint16_t* gathered;    // live rows of hidden
    float* slabs;                // nullptr: grad_hidden is not wanted
    uint16_t* grad_weight;       // nullptr: grad_weight is not wanted
    const int* index;
    int width, H, splits, first; // first: the slabs hold nothing yet
    int64_t slab_rows;
};
__global__ __launch_bounds__(HL_THREADS, 2) void head_products_kernel(const Products p)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t hl_lds[];
    constexpr int TM = 4, BM = 256;
    const int count = p.index[0], tiles_t = (count + BM - 1) / BM, tiles_h = (p.H + HL_BN - 1) / HL_BN, tiles_v = (p.width + BM - 1) / BM;
    const int xcd = blockIdx.x & 7;
    int li = blockIdx.x >> 3;
    const int hidden_jobs = p.slabs ? tiles_t * tiles_h * p.splits : 0, hidden_x = (hidden_jobs + 7) >> 3;
    float16_t acc[TM][HL_TN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    if (li < hidden_x) {
        const int job = xcd * hidden_x + li;
        if (job >= hidden_jobs) return;
        const int split = job / (tiles_t * tiles_h);
        int tm, tn;
        hl_origin(job - split * tiles_t * tiles_h, tiles_t, tiles_h, tm, tn);
        const int m0 = tm * BM, n0 = tn * HL_BN, kt = (p.width + 31) / 32;
        const int begin = (int)((int64_t)split * kt / p.splits), end = (int)((int64_t)(split + 1) * kt / p.splits);
        float* slab = p.slabs + ((int64_t)split * p.slab_rows + m0) * p.H + n0;
        if (p.first) {
            hl_clear<TM>(acc);
        } else {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int n = wn * 64 + j * 32 + 8 * g + 4 * hi;
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (n0 + n < p.H) v = *reinterpret_cast<const float4*>(slab + (int64_t)((wm * TM + i) * 32 + lr) * p.H + n);
                        acc[i][j][4 * g] = v.x; acc[i][j][4 * g + 1] = v.y; acc[i][j][4 * g + 2] = v.z; acc[i][j][4 * g + 3] = v.w;
                    }
        }
        const Operand a = {p.dl + (int64_t)m0 * p.ld + begin * 32, p.ld, BM, nullptr, 32};
        const Operand b = {p.weight + (int64_t)begin * 32 * p.ldw + n0, p.ldw, p.H - n0, nullptr, end == kt && p.width % 32 ? p.width % 32 : 32};
        hl_main_loop<TM, false, true>(acc, hl_lds, a, b, end - begin, false);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = wn * 64 + j * 32 + 8 * g + 4 * hi;
                    if (n0 + n < p.H)
                        *reinterpret_cast<float4*>(slab + (int64_t)((wm * TM + i) * 32 + lr) * p.H + n) =
                            make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
                }
        return;
    }
    if (!p.grad_weight) return;
    li -= hidden_x;
    const int jobs = tiles_v * tiles_h, per = (jobs + 7) >> 3, job = xcd * per + li;
    if (li >= per || job >= jobs) return;
    int tm, tn;
    hl_origin(job, tiles_v, tiles_h, tm, tn);
    const int m0 = tm * BM, n0 = tn * HL_BN;
    hl_clear<TM>(acc);
    const Operand a = {p.dl + m0, p.ld, BM, nullptr, 32}, b = {p.gathered + n0, p.H, p.H - n0, nullptr, 32};
    hl_main_loop<TM, true, true>(acc, hl_lds, a, b, (count + 31) / 32, false);
    hl_store_bf16<TM>(acc, hl_lds, p.grad_weight + (int64_t)m0 * p.H + n0, p.H, p.width - m0, p.H - n0);
}

// grad_hidden of every token: the slabs of a live one added in order, zero for the others.
__global__ __launch_bounds__(256) void head_hidden_kernel(const float* __restrict__ slabs, int splits, int64_t slab_rows, const int* __restrict__ index, int tokens, int H,
                                                          uint16_t* __restrict__ out)
{
    const int quads = H / 4;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < (int64_t)tokens * quads; at += (int64_t)gridDim.x * 256) {
        const int t = (int)(at / quads), c = (int)(at - (int64_t)t * quads), pos = live_rows(index)[tokens + t];
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (pos >= 0)
            for (int s = 0; s < splits; ++s) {
                const float4 q = *reinterpret_cast<const float4*>(slabs + ((int64_t)s * slab_rows + pos) * H + c * 4);
                v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
            }
        *reinterpret_cast<uint2*>(out + (int64_t)t * H + c * 4) = make_uint2(rb_pair(v.x, v.y), rb_pair(v.z, v.w));
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
int row_tiles(int64_t tokens) { return tokens <= 64 ? 1 : tokens <= 128 ? 2 : 4; }    // TM of the products over hidden
int64_t padded(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

bool sizes_ok(int64_t tokens, int64_t H, int64_t V)
{
    return tokens >= 0 && tokens <= (1 << 24) && H > 0 && H <= 65536 && H % 16 == 0 && V > 0 && V <= (1 << 22);
}

struct BackwardPlan {
    int64_t rows, width;         // padded tokens, columns of a piece
    int splits;
};
// Pieces: as many columns as 256 MiB of dl hold, or twice the bytes of the binary32 gradient of hidden where that is more (what a piece costs apart from its
// products is one pass over that gradient).  Splits of grad_hidden's contraction: as many as leave none of its tiles longer than a compute unit's
// share of the launch.
BackwardPlan backward_plan(int64_t tokens, int64_t H, int64_t V, bool want_weight)
{
    BackwardPlan p;
    p.rows = padded(tokens, 256);
    int64_t bytes = 8 * p.rows * H;
    if (bytes < ((int64_t)256 << 20)) bytes = (int64_t)256 << 20;
    int64_t most = bytes / (2 * p.rows) / 256 * 256;
    if (most < 256) most = 256;
    const int64_t pieces = (V + most - 1) / most;
    p.width = padded((V + pieces - 1) / pieces, 256);
    const int64_t tiles_h = (H + 255) / 256, tiles = p.rows / 256 * tiles_h, stages = p.width / 32;
    const int64_t all = tiles * stages + (want_weight ? p.width / 256 * tiles_h * (p.rows / 32) : 0), cus = device_cus();
    int64_t share = (all + cus - 1) / cus;
    if (share < 16) share = 16;
    int64_t s = (stages + share - 1) / share;
    if (s > 64) s = 64;
    p.splits = (int)(s < 1 ? 1 : s);
    return p;
}
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

template <int TM, bool ENT>
int launch_stats(const Tokens& tk, const void* weight, int64_t ldw, int stride, float2* part, float* part_e, float* hit, hipStream_t st)
{
    static bool done[64] = {};
    const size_t lds = (size_t)hl_slots(TM) * hl_stage_bytes(TM);
    if (const int rc = allow_dynamic_lds((const void*)head_stats_kernel<TM, ENT>, lds, done)) return rc;
    const int64_t tiles = ((tk.tokens + 64 * TM - 1) / (64 * TM)) * (int64_t)((tk.V + HL_BN - 1) / HL_BN);
    hipLaunchKernelGGL((head_stats_kernel<TM, ENT>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(HL_THREADS), lds, st, tk, (const uint16_t*)weight, ldw, stride, part, part_e, hit);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

template <int TM>
int launch_dlogits(const Tokens& tk, const void* weight, int64_t ldw, int v0, int width, const RowGrads& rg, uint16_t* dl, int64_t ld, hipStream_t st)
{
    static bool done[64] = {};
    const size_t lds = (size_t)hl_slots(TM) * hl_stage_bytes(TM);
    if (const int rc = allow_dynamic_lds((const void*)head_dlogits_kernel<TM>, lds, done)) return rc;
    const int64_t tiles = ((tk.tokens + 64 * TM - 1) / (64 * TM)) * (int64_t)((width + HL_BN - 1) / HL_BN);
    hipLaunchKernelGGL((head_dlogits_kernel<TM>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(HL_THREADS), lds, st, tk, (const uint16_t*)weight, ldw, v0, width, rg, dl, ld);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

Tokens tokens_of(const void* hidden, int64_t ld, const void* targets, const void* index, int64_t tokens, int64_t H, int64_t V, float temperature)
{
    return Tokens{(const uint16_t*)hidden, ld, (const int64_t*)targets, (const int*)index, (int)tokens, (int)H, (int)V, 1.44269504088896f / temperature};
}
bool operands_ok(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const void* targets, const void* index, int64_t H, float temperature)
{
    if (!hidden || !weight || !targets || !index || ldh < H || ldw < H || ldh % 8 || ldw % 8 || ldw > INT32_MAX / 128) return false;
    if ((uintptr_t)hidden % 16 || (uintptr_t)weight % 16 || (uintptr_t)targets % 8 || (uintptr_t)index % 256) return false;
    return temperature > 0.0f && temperature < INFINITY;
}

}  // namespace

size_t head_index_bytes(int64_t tokens) { return tokens < 0 || tokens > (1 << 24) ? 0 : align256((size_t)(64 + 2 * tokens) * sizeof(int)); }

size_t head_logprobs_workspace_bytes(int64_t tokens, int64_t H, int64_t V, int entropy)
{
    if (tokens <= 0 || !sizes_ok(tokens, H, V)) return 0;
    const size_t rows = (size_t)padded(tokens, 16), tiles = (size_t)(V + HL_BN - 1) / HL_BN;
    return align256(rows * tiles * 8) + align256(rows * 4) + (entropy ? align256(rows * tiles * 4) : 0);
}

int head_logprobs(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const void* targets, int64_t ignore, int64_t tokens, int64_t H, int64_t V, float temperature,
                  float* logp, float* lse, float* entropy, void* index, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (!sizes_ok(tokens, H, V)) return METIS_E_ARG;
    if (tokens == 0) return METIS_OK;
    if (!operands_ok(hidden, ldh, weight, ldw, targets, index, H, temperature) || !logp || !lse) return METIS_E_ARG;
    if (((uintptr_t)logp | (uintptr_t)lse | (uintptr_t)entropy) % 4) return METIS_E_ARG;
    if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < head_logprobs_workspace_bytes(tokens, H, V, entropy != nullptr)) return METIS_E_WORKSPACE;
    const int stride = (int)padded(tokens, 16), tiles_n = (int)((V + HL_BN - 1) / HL_BN);
    float2* part = static_cast<float2*>(workspace);
    float* hit = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256((size_t)stride * tiles_n * 8));
    float* part_e = entropy ? reinterpret_cast<float*>(reinterpret_cast<char*>(hit) + align256((size_t)stride * 4)) : nullptr;
    hipLaunchKernelGGL(head_index_kernel, dim3(1), dim3(1024), 0, st, (const int64_t*)targets, ignore, (int)tokens, (int*)index);
    if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    const Tokens tk = tokens_of(hidden, ldh, targets, index, tokens, H, V, temperature);
    const int tm = row_tiles(tokens);
    int rc;
    if (entropy) rc = tm == 1 ? launch_stats<1, true>(tk, weight, ldw, stride, part, part_e, hit, st) : tm == 2 ? launch_stats<2, true>(tk, weight, ldw, stride, part, part_e, hit, st)
                                                                                                       : launch_stats<4, true>(tk, weight, ldw, stride, part, part_e, hit, st);
    else rc = tm == 1 ? launch_stats<1, false>(tk, weight, ldw, stride, part, part_e, hit, st) : tm == 2 ? launch_stats<2, false>(tk, weight, ldw, stride, part, part_e, hit, st)
                                                                                                 : launch_stats<4, false>(tk, weight, ldw, stride, part, part_e, hit, st);
    if (rc != METIS_OK) return rc;
    const dim3 grid((unsigned)((tokens + 15) / 16));
    if (entropy)
        hipLaunchKernelGGL((head_finish_kernel<true>), grid, dim3(1024), 0, st, (const int64_t*)targets, (const int*)index, (int)tokens, (int)V, tiles_n, stride, part, part_e, hit, logp, lse, entropy);
    else
        hipLaunchKernelGGL((head_finish_kernel<false>), grid, dim3(1024), 0, st, (const int64_t*)targets, (const int*)index, (int)tokens, (int)V, tiles_n, stride, part, part_e, hit, logp, lse, entropy);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

size_t head_logprobs_backward_workspace_bytes(int64_t tokens, int64_t H, int64_t V, int want_hidden, int want_weight)
{
    if (tokens <= 0 || !sizes_ok(tokens, H, V)) return 0;
    const BackwardPlan p = backward_plan(tokens, H, V, want_weight != 0);
    return align256((size_t)p.rows * p.width * 2) + (want_weight ? align256((size_t)p.rows * H * 2) : 0) + (want_hidden ? align256((size_t)p.splits * p.rows * H * 4) : 0);
}

int head_logprobs_backward(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, const void* targets, int64_t tokens, int64_t H, int64_t V, float temperature,
                           const float* lse, const float* entropy, const float* g_logp, const float* g_entropy, const void* index, void* grad_hidden, void* grad_weight,
                           void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (!sizes_ok(tokens, H, V) || tokens == 0) return METIS_E_ARG;
    if (!operands_ok(hidden, ldh, weight, ldw, targets, index, H, temperature) || !lse || (g_entropy && !entropy)) return METIS_E_ARG;
    if (((uintptr_t)grad_hidden | (uintptr_t)grad_weight) % 16 || ((uintptr_t)lse | (uintptr_t)entropy | (uintptr_t)g_logp | (uintptr_t)g_entropy) % 4) return METIS_E_ARG;
    if (!grad_hidden && !grad_weight) return METIS_OK;
    if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < head_logprobs_backward_workspace_bytes(tokens, H, V, grad_hidden != nullptr, grad_weight != nullptr))
        return METIS_E_WORKSPACE;
    const BackwardPlan p = backward_plan(tokens, H, V, grad_weight != nullptr);
    char* at = static_cast<char*>(workspace);
    uint16_t* dl = reinterpret_cast<uint16_t*>(at);
    at += align256((size_t)p.rows * p.width * 2);
    uint16_t* gathered = nullptr;
    if (grad_weight) {
        gathered = reinterpret_cast<uint16_t*>(at);
        at += align256((size_t)p.rows * H * 2);
    }
    float* slabs = grad_hidden ? reinterpret_cast<float*>(at) : nullptr;
    const Tokens tk = tokens_of(hidden, ldh, targets, index, tokens, H, V, temperature);
    const RowGrads rg = {lse, entropy, g_logp, g_entropy};
    const int cus = device_cus();
    if (grad_weight) {
        hipLaunchKernelGGL(head_gather_kernel, dim3((unsigned)(tokens + 31 < 8 * (int64_t)cus ? tokens + 31 : 8 * (int64_t)cus)), dim3(256), 0, st, tk, (uint4*)gathered);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    static bool done[64] = {};
    const size_t lds = (size_t)hl_slots(4) * hl_stage_bytes(4);
    if (const int rc = allow_dynamic_lds((const void*)head_products_kernel, lds, done)) return rc;
    const int tm = row_tiles(tokens);
    const int64_t tiles_h = (H + 255) / 256;
    for (int64_t v0 = 0; v0 < V; v0 += p.width) {
        const int width = (int)(V - v0 < p.width ? V - v0 : p.width);
        const int rc = tm == 1 ? launch_dlogits<1>(tk, weight, ldw, (int)v0, width, rg, dl, p.width, st)
                     : tm == 2 ? launch_dlogits<2>(tk, weight, ldw, (int)v0, width, rg, dl, p.width, st) : launch_dlogits<4>(tk, weight, ldw, (int)v0, width, rg, dl, p.width, st);
        if (rc != METIS_OK) return rc;
        const Products pr = {dl, p.width, (const uint16_t*)weight + v0 * ldw, ldw, gathered, slabs, grad_weight ? (uint16_t*)grad_weight + v0 * H : nullptr, (const int*)index, width, (int)H,
                             p.splits, v0 == 0, p.rows};
        const int64_t hidden_jobs = slabs ? p.rows / 256 * tiles_h * p.splits : 0, weight_jobs = grad_weight ? (width + 255) / 256 * tiles_h : 0;
        const unsigned grid = 8u * (unsigned)((hidden_jobs + 7) / 8 + (weight_jobs + 7) / 8);
        hipLaunchKernelGGL(head_products_kernel, dim3(grid), dim3(HL_THREADS), lds, st, pr);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    if (grad_hidden) {
        const int64_t need = (tokens * (H / 4) + 255) / 256, cap = (int64_t)cus * 16;
        hipLaunchKernelGGL(head_hidden_kernel, dim3((unsigned)(need < cap ? need : cap)), dim3(256), 0, st, (const float*)slabs, p.splits, p.rows, (const int*)index, (int)tokens, (int)H,
                           (uint16_t*)grad_hidden);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    return METIS_OK;
}

}  // namespace metis
