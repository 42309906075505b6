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
// logits are formed again, turned into dl in the accumulators, rounded to bf16 once and kept only until the piece's two products have read it.  The gradient of
// hidden is summed in binary32 over the pieces.
//
// That rounding is a choice: bf16 is the type in which the matrix units take both products at their full rate (dl in two parts would be two more products,
// 6 ms beside 12.5 at 4096 x 3584 against 131072), and the one in which a bf16 model's gradient of its logits is held anyway.  It is made good where it would not average
// out, at the target, whose element makes most of a token's row (AtTarget).  Errors against 64 bits, relative to the norm (411 x 1536 against 32003, 600 x 2048 against
// 65537; the results' own rounding to bf16 alone is 0.0017): both gradients 0.0017 where the targets' elements are most of them; where the mass lies on other
// tokens, 0.0018; the entropy's alone under peaked distributions, and the rows of the weight's gradient that are no token's target, 0.0024.
//
// Tokens whose target is ignored take no part: a first launch lists the others ("live"), the products run over the listed rows, and what an ignored
// row of hidden holds (padding: anything) is never read into a sum.
#include "gemm_common.h"
#include <type_traits>

namespace metis {

namespace {

constexpr int HL_BN = 256, HL_TN = 2, HL_THREADS = 512;

__host__ __device__ constexpr int hl_stage_bytes(int TM) { return (64 * TM + HL_BN) * 64; }
constexpr int HL_NS = 5;

__host__ __device__ constexpr int hl_waitcnt(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | ((lgkm & 15) << 8); }
#define HL_WAIT(VM, LGKM) __builtin_amdgcn_s_waitcnt(hl_waitcnt(VM, LGKM))

typedef short hl_short4_t __attribute__((ext_vector_type(4)));
typedef short hl_short8_t __attribute__((ext_vector_type(8)));
typedef uint32_t hl_u32x4_t __attribute__((ext_vector_type(4)));
typedef hl_short4_t __attribute__((address_space(3))) * hl_lds_ptr_t;

// ---------------------------------------------------------------------------------------------
// The tile engine: 64 TM x 256 of a product per workgroup, eight waves (2 x 4) of 32 TM x 64, stages of 32 along the contraction in a ring of five
// LDS slots, filled by direct loads three stages ahead; one barrier a stage, waits that never drain the queue.  Loads go out for two stages at a time (a
// plain operand's 64 bytes of either are the halves of one 128-byte line) and spread over both iterations between the products.
//
// An operand lies in memory either along the contraction ("plain": [row][k]) or across it ("turned": [k][row]); both go to LDS as they are, 1 KiB per load
// instruction.  Plain: 16 rows of 64 bytes, the four 16-byte pieces of row q in the order c ^ swz(q), read back as ds_read_b128.  Turned: rows of k, whose
// 64-byte segments are exchanged by f(k) so that the four rows which a transposing read (ds_read_b64_tr_b16) takes at once lie in different banks; two
// such reads give a lane its eight consecutive k.
//
// 4096 x 3584 against 131072 rows, 3686 live: forward 2.85 ms (1213 TFLOP/s of the live tokens' products, 1293 with all live), dl 4 x 0.79, the two other
// products 4 x 1.59; a library's product of the same operands reaches 1285, 884 and 1011 TFLOP/s, 1538 at 8192^3.  The matrix units are busy 72, 67 and
// 64 % of the cycles; without its loads the loop would reach 1525.  Few tokens: the head's bytes (5 x 1536: 5.3 TB/s).  Five slots and loads by pairs of stages
// took the forward from 3.27 to 2.94 ms; two slots of twice the stage, hints off, wave priorities and other groups of tiles gained nothing.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int hl_swz(int q) { return ((q >> 2) & 1) | ((((q >> 1) ^ (q >> 3)) & 1) << 1); }
template <int ROW_BYTES> __device__ __forceinline__ int hl_turn(int k) { return ROW_BYTES >= 256 ? (k & 3) << 6 : ((k >> 1) & 1) << 6; }

// The thread's number, as a value of its own at each place: what follows from it is formed again for every tile and not kept in registers across its products
// (kept, the kernels that go through several tiles need more than there are).
__device__ __forceinline__ int hl_thread()
{
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

struct Operand {
    const uint16_t* base;        // first element of the tile's rows (plain) or of the first k's row (turned)
    int64_t ld;                  // elements between rows (plain) or between k (turned)
    int limit;                   // rows from here on are not there: the last one is read in their place
    const int* index;            // plain: the rows' numbers, or nullptr for rows as they come
    int rest;                    // k of the last stage that are there: 16 or 32 (plain), 1 .. 32 (turned); in place of others some that are there are read
    int64_t panel;               // A in panels: elements between panels of 64 columns of the stored matrix, whose rows are then 64 long (ld 64)
};

// One wave's view of it.  aim() at a tile: stages [0, steps) along the contraction; half: only the first sixteen k of the last one count.  Where fewer
// count otherwise, one operand holds zeros beyond them.  PANELS: A is stored in panels.  Then request(0), request(2) and multiply(): the first pair of stages
// goes to slots 0 and 1, the second to 2 and 3, so that the next tile's first pair can be under way while this one's results leave through the
// rest of the ring.
template <int TM, bool AT, bool BT, bool PANELS> struct Pipe {
    static constexpr int BM = 64 * TM, NA = BM / 16, TOTAL = NA + HL_BN / 16, LPW = (TOTAL + 7) / 8, STAGE = hl_stage_bytes(TM), NS = HL_NS, B_AT = NA * 1024;
    static constexpr int A_RB = BM * 2, B_RB = HL_BN * 2;
    uint8_t* lds;
    const uint8_t* src[LPW];     // this wave's load instructions of a stage: where the lane reads next,
    int64_t inc[LPW], inc_odd[LPW];   // how far it goes behind even and odd stages (64 bytes where both operands are plain),
    uint32_t back[LPW];          // and how far back in the last one
    int steps;
    bool half;

    __device__ __forceinline__ void aim(const Operand& a, const Operand& b, int count, bool half_last)
    {
        const int thread = hl_thread(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
        steps = count;
        half = half_last;
#pragma unroll
        for (int j = 0; j < LPW; ++j) {
            int ot = j * 8 + wave;
            if (ot >= TOTAL) ot -= 8;                              // (a piece that another wave loads too: the same bytes to the same place)
            const bool is_a = ot < NA;
            const Operand& o = is_a ? a : b;
            const int q = is_a ? ot : ot - NA;
            if (is_a ? AT : BT) {
                const int rb = is_a ? A_RB : B_RB, k = q * (1024 / rb) + lane * 16 / rb, at = lane * 16 % rb;
                int col = (at ^ (is_a ? hl_turn<A_RB>(k) : hl_turn<B_RB>(k))) >> 1;
                if (col >= o.limit) col = 0;                       // (columns in eights: all there or none)
                src[j] = reinterpret_cast<const uint8_t*>(o.base + (int64_t)k * o.ld + (PANELS && is_a ? (col >> 6) * o.panel + (col & 63) : col));
                inc[j] = inc_odd[j] = o.ld * 64;
                back[j] = k >= o.rest ? (uint32_t)((k - (o.rest - 1)) * (o.ld * 2)) : 0u;
            } else {
                const int row = q * 16 + (lane >> 2), chunk = (lane & 3) ^ hl_swz(row & 15);
                int r = row < o.limit ? row : o.limit - 1;
                const int64_t at = o.index ? o.index[r] : r;
                src[j] = reinterpret_cast<const uint8_t*>(o.base + at * o.ld + chunk * 8);
                inc[j] = 64;
                inc_odd[j] = PANELS && is_a ? o.panel * 2 - 64 : 64;
                back[j] = chunk * 8 >= o.rest ? 32u : 0u;
            }
        }
    }
    __device__ __forceinline__ void issue_one(int slot, int j, bool odd, bool last)
    {
        const uint8_t* g = src[j] - (last ? back[j] : 0u);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = j * 8 + wave, ot = at < TOTAL ? at : at - 8;
        const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(slot * STAGE + ot * 1024));
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(g), "s"(dst) : "memory");
        if constexpr (!AT && !BT && !PANELS) src[j] += 64;
        else if constexpr (!AT && PANELS) src[j] += odd ? inc_odd[j] : inc[j];
        else src[j] += inc[j];
    }
    // Two stages are requested together, piece by piece: a plain operand's two pieces are the halves of the same 128-byte lines.
    __device__ __forceinline__ void issue_pair(int slot0, int slot1, int j, int stage0)
    {
        if (stage0 < steps) issue_one(slot0, j, false, stage0 == steps - 1);
        if (stage0 + 1 < steps) issue_one(slot1, j, true, stage0 + 1 == steps - 1);
    }
    __device__ __forceinline__ void request(int stage0)
    {
#pragma unroll
        for (int j = 0; j < LPW; ++j) issue_pair(stage0, stage0 + 1, j, stage0);
    }

    // adds the tile's products; behind it every slot is free
    __device__ __forceinline__ void multiply(float16_t (&acc)[TM][HL_TN])
    {
        if (steps <= 0) return;
        const int thread = hl_thread(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), wm = wave >> 2, wn = wave & 3;
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

        if (steps >= 4) HL_WAIT(2 * LPW + 1, 15);
        else HL_WAIT(0, 15);
        __syncthreads();
        load_frags(0, 0);
        int s = 0, slot = 0;
        auto next_of = [](int k) { return k + 1 == NS ? 0 : k + 1; };
        auto before = [](int k) { return k == 0 ? NS - 1 : k - 1; };
        // Stage s in `slot`.  FIRST (s even): half of the load instructions of stages s + 4 and s + 5, into the slots before `slot` and `slot` itself, whose
        // stages every wave has in registers behind this barrier; the iteration after it the other half, EARLY pairs of them before its own barrier: with turned
        // operands, whose fragments take twice the reads, the queue is evener so (both products of 4096 x 3584 against 32768 columns 1.74 -> 1.70 ms; grad_hidden
        // alone likes two early, grad_weight alone one).  At a barrier at most `most` loads are outstanding.
        constexpr int EARLY = !BT ? 0 : AT ? 1 : 2;
        auto iterate = [&](auto first, auto most) {
            constexpr bool FIRST = decltype(first)::value;
            constexpr int H0 = LPW / 2, E = FIRST ? 0 : EARLY < LPW - H0 ? EARLY : LPW - H0, J0 = FIRST ? 0 : H0 + E, COUNT = FIRST ? H0 : LPW - H0 - E;
            const int slot1 = FIRST ? slot : before(slot), slot0 = before(slot1);
            const bool last = (FIRST ? s + 5 : s + 4) == steps - 1;
            auto loads = [&](int m, int from, int count) {         // between the products: instruction m of NM
#pragma unroll
                for (int j = from; j < from + count; ++j)
                    if ((j - from) * NM / count == m) {
                        issue_one(slot0, j, false, false);
                        issue_one(slot1, j, true, last);
                    }
            };
            load_frags(slot, 1);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                if constexpr (E > 0) loads(m, H0, E);
                mfma_one(0, m / HL_TN, m % HL_TN);
            }
            if constexpr (E == 0) sched_substep<NM, 0, NF, 0>();
            HL_WAIT(decltype(most)::value, 0);                     // own loads of stage s + 1 are there, own reads of stage s done
            __syncthreads();
            load_frags(next_of(slot), 0);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                if constexpr (COUNT > 0) loads(m, J0, COUNT);
                mfma_one(1, m / HL_TN, m % HL_TN);
            }
            slot = next_of(slot);
            ++s;
        };
        // when stage s + 1 has to be there: s even, all of its pair (all but the next pair); s odd, the even half of its pair (all but the last load of it,
        // the first half of the next pair and what went out early)
        constexpr int SENT = LPW / 2 + (EARLY < LPW - LPW / 2 ? EARLY : LPW - LPW / 2);
        while (s + 5 < steps) {
            iterate(std::true_type{}, std::integral_constant<int, 2 * LPW>{});
            iterate(std::false_type{}, std::integral_constant<int, 2 * SENT + 1>{});
        }
        for (; s < steps; ++s) {
            const bool both = s + 1 < steps || !half;
            if (both) load_frags(slot, 1);
            mfmas(0);
            HL_WAIT(0, 0);
            __syncthreads();
            if (s + 1 < steps) load_frags(next_of(slot), 0);
            if ((s & 1) == 0) {
#pragma unroll
                for (int j = 0; j < LPW; ++j) issue_pair(before(slot), slot, j, s + 4);
            }
            if (both) mfmas(1);
            slot = next_of(slot);
        }
        __syncthreads();                                           // the ring is free
    }
};

// acc[i][j][e] of lane l: row 32 (TM wm + i) + l % 32, column 64 wn + 32 j + 8 (e / 4) + 4 (l / 32) + e % 4 of the tile.
// The tile as bf16, the wave's 64 columns in rows of `ld` elements from `out` on: through the wave's own part of LDS, 32 rows at a time, so that a store
// writes 8 rows of 128 bytes.
template <int TM>
__device__ __forceinline__ void hl_store_bf16(const float16_t (&acc)[TM][HL_TN], uint8_t* lds, uint16_t* out, int64_t ld, int rows, int cols)
{
    constexpr int CROW = 72;                                   // 144 bytes
    const int thread = hl_thread(), lane = thread & 63, wave = thread >> 6, wm = wave >> 2, lr = lane & 31, hi = lane >> 5;
    uint16_t* cw = reinterpret_cast<uint16_t*>(lds) + wave * (32 * CROW);
    const int n = (lane & 7) * 8;
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
// among them or -1, index[64 + 2 tokens ..] by place the target's log-probability in powers of two, as the forward's own sums give it.
struct Tokens {
    const uint16_t* hidden;
    int64_t ld;
    const int64_t* targets;
    const int* index;
    int tokens, H, V;
    float scale2;                // log2(e) / temperature: logits in powers of two
};
__device__ __forceinline__ const int* live_rows(const int* index) { return index + 64; }
__host__ __device__ constexpr int64_t index_words(int64_t tokens) { return 64 + 3 * tokens; }

// the k-th tile of this workgroup's XCD, which has a contiguous range of the tiles; -1 behind it
__device__ __forceinline__ int hl_logical(int total, int k)
{
    const int per = (total + 7) >> 3, logical = (blockIdx.x & 7) * per + k;
    return k < per && logical < total ? logical : -1;
}
// groups of up to five tile rows, as even as they come, walked column by column: 32 compute units of an XCD share the operands of a few rows and columns.
// (Groups of up to 6, 8, 16 rows: 16 rows of tiles, all three products, 1 to 6 % slower.)
__device__ __forceinline__ void hl_origin(int logical, int tiles_m, int tiles_n, int& tm, int& tn)
{
    constexpr int MOST = 5;
    const int groups = (tiles_m + MOST - 1) / MOST, gm = (tiles_m + groups - 1) / groups;
    const int group = logical / (gm * tiles_n), first = group * gm, size = min(tiles_m - first, gm), in = logical - group * gm * tiles_n;
    tm = first + in % size;
    tn = in / size;
}

// Rows of a tile over tokens, 64 TM, by the live tokens' number.  A tile takes 57, 80, 100 parts of time with TM = 2, 3, 4 (65536 x 2048: 33, 46, 58 us each),
// so fewer rows pay only where the last tile of more would be mostly empty: 300 tokens 119 -> 101 us, 540 176 -> 147, 100 63 -> 51; but 400 stay (124,
// 142 with TM = 3).  The number is known on the device alone: the launches for up to kFewTokens tokens hold all three, beyond that it is always 4.
constexpr int kListTokens = 64, kFewTokens = 2048;
__host__ __device__ __forceinline__ int hl_row_tiles(int count)
{
    if (count <= 128) return 2;
    return (count + 191) / 192 * 80 < (count + 255) / 256 * 100 ? 3 : 4;
}
enum Rows { kList, kFew, kMany };                              // up to kListTokens tokens (TM = 1), up to kFewTokens, more
// f with the TM that counts
template <int ROWS, class F> __device__ __forceinline__ void with_row_tiles(int count, F&& f)
{
    if constexpr (ROWS == kList) f(std::integral_constant<int, 1>{});
    else if constexpr (ROWS == kMany) f(std::integral_constant<int, 4>{});
    else {
        const int tm = hl_row_tiles(count);
        if (tm == 2) f(std::integral_constant<int, 2>{});
        else if (tm == 3) f(std::integral_constant<int, 3>{});
        else f(std::integral_constant<int, 4>{});
    }
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
// 2^(l - maximum) (l - maximum); the target's sum of products from the tile that has it.
// ---------------------------------------------------------------------------------------------
// What a tile leaves, from its accumulators; `red`: LDS.
template <int TM, bool ENT>
__device__ __forceinline__ void hl_stats_out(float16_t (&acc)[TM][HL_TN], float* red, const Tokens& tk, int count, const int* live, int m0, int tn, int stride, float2* part, float* part_e,
                                             float* hit)
{
    constexpr int BM = 64 * TM;
    const int n0 = tn * HL_BN;
    const int thread = hl_thread(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    const int there = tk.V - (n0 + wn * 64);                   // columns of this wave that exist
    // red: [row][wave column][3]
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int row = (wm * TM + i) * 32 + lr, m = m0 + row;
        float top = -INFINITY, sum = 0.0f, ent = 0.0f;
        if (there > 0) {
            if (there < 64) {                                  // columns that do not exist
#pragma unroll
                for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3) >= there) acc[i][j][e] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
            top = fmaxf(top, __shfl_xor(top, 32, 64)) * tk.scale2;
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float d = fmaf(acc[i][j][e], tk.scale2, -top), p = __builtin_amdgcn_exp2f(d);
                    sum += p;
                    if constexpr (ENT) ent = fmaf(p, there < 64 ? fmaxf(d, -1e30f) : d, ent);      // (0 * -infinity of a column that does not exist)
                }
            sum += __shfl_xor(sum, 32, 64);
            if constexpr (ENT) ent += __shfl_xor(ent, 32, 64);
            int64_t want = -1;
            if (m < count) want = tk.targets[live[m]] - (n0 + wn * 64);
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
    const int row = thread;
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

// A workgroup per compute unit (their LDS holds no second) goes through its tiles, the next one's first stages under way while one's results leave: 64 tokens
// x 3584 against 131072 rows 180 -> 172 us, of many tokens 0 to 2 %.  (dl's tiles and those of grad_weight gain nothing by it: their stores have to be done
// before the next tile's stages can be waited for.)
template <int TM, bool ENT>
__device__ __forceinline__ void hl_stats_tiles(uint8_t* hl_lds, const Tokens& tk, int count, const int* live, const uint16_t* weight, int64_t ldw, int stride, float2* part, float* part_e,
                                               float* hit)
{
    constexpr int BM = 64 * TM;
    const int tiles_m = (count + BM - 1) / BM, tiles_n = (tk.V + HL_BN - 1) / HL_BN, total = tiles_m * tiles_n, rest = tk.H % 32 ? 16 : 32;
    int k = blockIdx.x >> 3, logical = hl_logical(total, k), tm, tn;
    if (logical < 0) return;
    Pipe<TM, false, false, false> pipe;
    pipe.lds = hl_lds;
    auto begin = [&]() {
        hl_origin(logical, tiles_m, tiles_n, tm, tn);
        const int m0 = tm * BM, n0 = tn * HL_BN;
        pipe.aim(Operand{tk.hidden, tk.ld, count - m0, live + m0, rest, 0}, Operand{weight + (int64_t)n0 * ldw, ldw, tk.V - n0, nullptr, rest, 0}, (tk.H + 31) / 32, rest == 16);
        pipe.request(0);
    };
    begin();
    while (true) {
        pipe.request(2);
        float16_t acc[TM][HL_TN];
        hl_clear<TM>(acc);
        pipe.multiply(acc);
        const int m0 = tm * BM, at_n = tn;
        k += gridDim.x >> 3;
        logical = hl_logical(total, k);
        if (logical >= 0) begin();
        hl_stats_out<TM, ENT>(acc, reinterpret_cast<float*>(hl_lds + 2 * hl_stage_bytes(TM)), tk, count, live, m0, at_n, stride, part, part_e, hit);
        if (logical < 0) return;
        __syncthreads();
    }
}

// kList: every workgroup lists the live tokens for itself, in LDS behind the ring, and the first writes the list down for the launches to come: a launch less
// (5 x 1536 against 131072: 91 -> 83 us with the fold of the tiles in fewer steps).
template <int ROWS, bool ENT>
__global__ __launch_bounds__(HL_THREADS, 2) void head_stats_kernel(const Tokens tk, const uint16_t* __restrict__ weight, int64_t ldw, int stride,
                                                                 float2* __restrict__ part, float* __restrict__ part_e, float* __restrict__ hit, int64_t ignore,
                                                                 int* __restrict__ list)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t hl_lds[];
    int count;
    const int* live;
    if constexpr (ROWS == kList) {
        int* own = reinterpret_cast<int*>(hl_lds + HL_NS * hl_stage_bytes(1));
        const int t = threadIdx.x & 63;
        const bool on = t < tk.tokens && tk.targets[t] != ignore;
        const uint64_t mask = __ballot(on);
        const int at = __popcll(mask & ((1ull << t) - 1ull));
        count = __popcll(mask);
        if (threadIdx.x < 64) {
            if (on) own[at] = t;
            if (blockIdx.x == 0) {
                if (t == 0) list[0] = count;
                if (on) list[64 + at] = t;
                if (t < tk.tokens) list[64 + tk.tokens + t] = on ? at : -1;
            }
        }
        __syncthreads();
        live = own;
    } else {
        count = tk.index[0];
        live = live_rows(tk.index);
    }
    with_row_tiles<ROWS>(count, [&](auto tm) { hl_stats_tiles<decltype(tm)::value, ENT>(hl_lds, tk, count, live, weight, ldw, stride, part, part_e, hit); });
}

// A maximum with its sum of 2^(l - maximum) and, for the entropy, of 2^(l - maximum) (l - maximum); empty: -infinity, 0, 0.
struct Fold {
    float top, sum, ent;
};
template <bool ENT> __device__ __forceinline__ Fold fold(const Fold& a, const Fold& b)
{
    Fold r;
    r.top = fmaxf(a.top, b.top);
    const float da = a.sum != 0.0f ? a.top - r.top : 0.0f, db = b.sum != 0.0f ? b.top - r.top : 0.0f;     // (nothing in it: no infinity less infinity)
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    r.sum = fa * a.sum + fb * b.sum;
    r.ent = ENT ? fa * fmaf(da, a.sum, a.ent) + fb * fmaf(db, b.sum, b.ent) : 0.0f;
    return r;
}

// The tiles of a token folded, 16 tokens per workgroup: 64 chains of every 64th tile, eight requested together, then the four chains of a wave by lanes and
// the sixteen waves in order.
template <bool ENT>
__global__ __launch_bounds__(1024) void head_finish_kernel(const int64_t* __restrict__ targets, int* __restrict__ index, int tokens, int V, int tiles_n, int stride, float scale2,
                                                           const float2* __restrict__ part, const float* __restrict__ part_e, const float* __restrict__ hit,
                                                           float* __restrict__ logp, float* __restrict__ lse, float* __restrict__ entropy)
{
    __shared__ float red[16][16][3];
    const int r = threadIdx.x & 15, chain = threadIdx.x >> 4, wave = threadIdx.x >> 6, t = blockIdx.x * 16 + r;
    const int pos = t < tokens ? live_rows(index)[tokens + t] : -1;
    Fold mine = {-INFINITY, 0.0f, 0.0f};
    for (int k0 = chain; k0 < tiles_n; k0 += 8 * 64) {
        float2 p[8];
        float e[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            p[b] = make_float2(-INFINITY, 0.0f);
            e[b] = 0.0f;
            const int k = k0 + b * 64;
            if (pos >= 0 && k < tiles_n) {
                p[b] = part[(size_t)k * stride + pos];
                if constexpr (ENT) e[b] = part_e[(size_t)k * stride + pos];
            }
        }
#pragma unroll
        for (int b = 0; b < 8; ++b) mine = fold<ENT>(mine, Fold{p[b].x, p[b].y, e[b]});
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1)
        mine = fold<ENT>(mine, Fold{__shfl_xor(mine.top, o, 64), __shfl_xor(mine.sum, o, 64), ENT ? __shfl_xor(mine.ent, o, 64) : 0.0f});
    if ((threadIdx.x & 63) < 16) {
        red[wave][r][0] = mine.top;
        red[wave][r][1] = mine.sum;
        red[wave][r][2] = mine.ent;
    }
    __syncthreads();
    if (chain || t >= tokens) return;
    if (pos < 0) {
        logp[t] = lse[t] = 0.0f;
        if constexpr (ENT) entropy[t] = 0.0f;
        return;
    }
#pragma unroll
    for (int k = 1; k < 16; ++k) mine = fold<ENT>(mine, Fold{red[k][r][0], red[k][r][1], red[k][r][2]});
    constexpr float kLn2 = 0.693147180559945f;
    const int64_t want = targets[t];
    const bool there = want >= 0 && want < V;                  // (a target outside of the vocabulary shows: everything of its row is NaN)
    const float l2 = __log2f(mine.sum), nan = __uint_as_float(0x7fc00000u);
    // The target's logit is compared with the maximum as the sums compared each of theirs: one fma from its sum of products.  Where it is the maximum, what is left
    // is the sum's distance from one, with nothing of the size of the logits in it.
    float lp2 = there ? fmaf(hit[pos], scale2, -mine.top) - l2 : nan;
    lp2 = lp2 > 0.0f ? 0.0f : lp2;                             // (a rounding above zero; NaN stays)
    lse[t] = there ? (mine.top + l2) * kLn2 : nan;
    logp[t] = lp2 * kLn2;
    reinterpret_cast<float*>(index)[64 + 2 * tokens + pos] = lp2;
    if constexpr (ENT) entropy[t] = there ? (l2 - mine.ent / mine.sum) * kLn2 : nan;
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
// Backward, first launch of a piece: dl of the vocabulary's columns v0 .. v0 + width - 1 as bf16, in panels of 64 columns, [panel][live tokens, padded][64]
// (whole lines that lie side by side for both products; rows of a whole piece would be a power of two apart), zero where tokens of a tile or columns are not there.
// ---------------------------------------------------------------------------------------------
struct RowGrads {
    const float *lse, *entropy, *g_logp, *g_entropy;           // by token; entropy and g_entropy may be nullptr
};
// dl at the targets, by place among the live tokens: the value as bf16, what that leaves out, the target (-1: not in the vocabulary).  This one element makes
// most of a token's gradient, so its rounding (up to 2^-8) would be a common factor of a whole row: the products take `rounded`, and `left` goes into both
// gradients in binary32.  (Gradients against 64 bits, 411 x 1536 against 32003: 0.0025 of their norm with the rounding left as it is.)
struct AtTarget {
    float *rounded, *left;
    int* column;
};
// dl of a tile from its accumulators; `area`: LDS.
template <int TM>
__device__ __forceinline__ void hl_dlogits_out(float16_t (&acc)[TM][HL_TN], uint8_t* area, const Tokens& tk, int count, int m0, int n0, int v0, int width, const RowGrads& rg, const AtTarget& target,
                                               uint16_t* dl, int64_t panel)
{
    constexpr int BM = 64 * TM;
    constexpr float kLn2 = 0.693147180559945f, kLog2e = 1.44269504088896f;
    const int* live = live_rows(tk.index);
    const int thread = hl_thread(), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6), wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    const int there = width - (n0 + wn * 64);
    const float inv_t = tk.scale2 * kLn2;                      // 1 / temperature
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = m0 + (wm * TM + i) * 32 + lr;
        float lse2 = 0.0f, g = 0.0f, ge = 0.0f, h = 0.0f, at_target = 0.0f;
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
            const int w = target.column[m] - (v0 + n0 + wn * 64);
            if (w >= 0 && w < 64) {
                want = w;
                at_target = target.rounded[m];
            }
        }
        // -p f everywhere, then the target's, then zero where nothing is: the last two in few tiles
        const float ge2 = ge * kLn2;
        if (rg.g_entropy) {
            g = fmaf(ge, h, g);                                // f = g + ge (d ln 2 + h)
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float d = fmaf(acc[i][j][e], tk.scale2, -lse2);
                    acc[i][j][e] = -__builtin_amdgcn_exp2f(d) * fmaf(ge2, d, g);
                }
        } else {
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = -__builtin_amdgcn_exp2f(fmaf(acc[i][j][e], tk.scale2, -lse2)) * g;
        }
        if (__any(want >= 0)) {
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3) == want ? at_target : acc[i][j][e];
        }
        if (__any(!on) || there < 64) {
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!on || j * 32 + 8 * (e >> 2) + 4 * hi + (e & 3) >= there) acc[i][j][e] = 0.0f;
        }
    }
    hl_store_bf16<TM>(acc, area, dl + (int64_t)(n0 / 64 + wn) * panel + m0 * 64, 64, BM, 64);
}

template <int TM>
__device__ __forceinline__ void hl_dlogits_tile(uint8_t* hl_lds, const Tokens& tk, int count, const uint16_t* weight, int64_t ldw, int v0, int width, const RowGrads& rg,
                                                const AtTarget& target, uint16_t* dl, int64_t panel)
{
    constexpr int BM = 64 * TM;
    const int tiles_m = (count + BM - 1) / BM, tiles_n = (width + HL_BN - 1) / HL_BN, rest = tk.H % 32 ? 16 : 32, logical = hl_logical(tiles_m * tiles_n, blockIdx.x >> 3);
    if (logical < 0) return;
    int tm, tn;
    hl_origin(logical, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * HL_BN;
    float16_t acc[TM][HL_TN];
    hl_clear<TM>(acc);
    Pipe<TM, false, false, false> pipe;
    pipe.lds = hl_lds;
    pipe.aim(Operand{tk.hidden, tk.ld, count - m0, live_rows(tk.index) + m0, rest, 0}, Operand{weight + (int64_t)(v0 + n0) * ldw, ldw, width - n0, nullptr, rest, 0}, (tk.H + 31) / 32,
             rest == 16);
    pipe.request(0);
    pipe.request(2);
    pipe.multiply(acc);
    hl_dlogits_out<TM>(acc, hl_lds, tk, count, m0, n0, v0, width, rg, target, dl, panel);
}

template <int ROWS>
__global__ __launch_bounds__(HL_THREADS, 2) void head_dlogits_kernel(const Tokens tk, const uint16_t* __restrict__ weight, int64_t ldw, int v0, int width, const RowGrads rg,
                                                                     const AtTarget target, uint16_t* __restrict__ dl, int64_t panel)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t hl_lds[];
    const int count = tk.index[0];
    with_row_tiles<ROWS>(count, [&](auto tm) { hl_dlogits_tile<decltype(tm)::value>(hl_lds, tk, count, weight, ldw, v0, width, rg, target, dl, panel); });
}

// Before the pieces: dl at the targets, and for grad_weight (`out`) the live rows of hidden side by side, then zero rows up to a multiple of 32.
//   dl = g (1 - p) - e p (log p + H)  at the target, with the forward's log p: 1 - p is what the other tokens' p add up to but for the rounding of sums of about one.
// (With p from a product of its own and the log-sum-exp 1 - p was off by their roundings, 2^-24 of the logits: where a model is sure, 1 - p under 1e-3, by
// a tenth and more of these tokens' gradients.)
__global__ __launch_bounds__(256) void head_gather_kernel(const Tokens tk, const RowGrads rg, const AtTarget target, uint4* __restrict__ out)
{
    constexpr float kLn2 = 0.693147180559945f;
    const int count = tk.index[0], cpr = tk.H / 8;
    const float inv_t = tk.scale2 * kLn2;                      // 1 / temperature
    for (int m = blockIdx.x * 256 + threadIdx.x; m < count; m += gridDim.x * 256) {
        const int t = live_rows(tk.index)[m];
        const int64_t want = tk.targets[t];
        const bool there = want >= 0 && want < tk.V;
        const float lp = reinterpret_cast<const float*>(tk.index)[64 + 2 * tk.tokens + m] * kLn2;
        float v = rg.g_logp ? rg.g_logp[t] * inv_t * -expm1f(lp) : 0.0f;
        if (rg.g_entropy) v = fmaf(-expf(lp), rg.g_entropy[t] * inv_t * (lp + rg.entropy[t]), v);
        const float r = __uint_as_float(rb_pair(v, 0.0f) << 16);
        target.rounded[m] = r;
        target.left[m] = there && fabsf(r) < INFINITY ? v - r : 0.0f;
        target.column[m] = there ? (int)want : -1;
    }
    if (!out) return;
    const int rows = (count + 31) & ~31;
    for (int m = blockIdx.x; m < rows; m += gridDim.x) {
        const uint4* x = reinterpret_cast<const uint4*>(tk.hidden + (int64_t)live_rows(tk.index)[m < count ? m : 0] * tk.ld);
        for (int c = threadIdx.x; c < cpr; c += 256) out[(int64_t)m * cpr + c] = m < count ? x[c] : make_uint4(0u, 0u, 0u, 0u);
    }
}

// Per 256 rows of the vocabulary: which rows of grad_weight are targets' (`row_of`: the first live token with that target, or -1) and, as the row of that
// token, what `left` of all tokens with that target gives, in their order.  (Its own rounding to bf16 is 2^-8 of at most 2^-8 of the gradient.)  A wave takes
// 512 columns of one such row; where the vocabulary has few rows, gridDim.y workgroups share its columns.
__global__ __launch_bounds__(1024) void head_targets_kernel(const int* __restrict__ index, const AtTarget target, const uint16_t* __restrict__ gathered, int H, int* __restrict__ row_of,
                                                            uint16_t* __restrict__ rest)
{
    __shared__ int first[256], times[256], list[256], listed[4];
    const int count = index[0], v0 = blockIdx.x * 256, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x < 256) {
        first[threadIdx.x] = INT32_MAX;
        times[threadIdx.x] = 0;
    }
    __syncthreads();
    for (int m = threadIdx.x; m < count; m += 1024) {
        const int row = target.column[m] - v0;
        if (row >= 0 && row < 256) {
            atomicMin(&first[row], m);
            atomicAdd(&times[row], 1);
        }
    }
    __syncthreads();
    const bool has = threadIdx.x < 256 && times[threadIdx.x & 255] > 0;
    const uint64_t mask = __ballot(has);
    if (wave < 4 && lane == 0) listed[wave] = __popcll(mask);
    if (blockIdx.y == 0 && threadIdx.x < 256) row_of[v0 + threadIdx.x] = has ? first[threadIdx.x] : -1;
    __syncthreads();
    int at = __popcll(mask & ((1ull << lane) - 1ull));
#pragma unroll
    for (int w = 0; w < 3; ++w) at += w < wave ? listed[w] : 0;
    if (has) list[at] = threadIdx.x;
    __syncthreads();
    const int chunks = ((H + 511) / 512 - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y, jobs = (listed[0] + listed[1] + listed[2] + listed[3]) * chunks;
    for (int job = wave; job < jobs; job += 16) {
        const int row = list[job / chunks], c = ((int)blockIdx.y + job % chunks * (int)gridDim.y) * 512 + lane * 8, begin = __builtin_amdgcn_readfirstlane(first[row]);
        int to_come = __builtin_amdgcn_readfirstlane(times[row]);
        float sum[8] = {};
        for (int m0 = begin; m0 < count && to_come > 0; m0 += 64) {
            uint64_t same = to_come == 1 && m0 == begin ? 1ull : __ballot(m0 + lane < count && target.column[m0 + lane] == v0 + row);
            to_come -= __popcll(same);
            while (same) {                                     // eight rows requested together
                uint4 x[8];
                float left[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int m = m0 + (same ? __builtin_ctzll(same) : 0);
                    left[k] = same ? target.left[m] : 0.0f;
                    x[k] = make_uint4(0u, 0u, 0u, 0u);
                    if (same && c < H) x[k] = *reinterpret_cast<const uint4*>(gathered + (int64_t)m * H + c);
                    same &= same - 1;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sum[2 * e] = fmaf(left[k], __uint_as_float(w[e] << 16), sum[2 * e]);
                        sum[2 * e + 1] = fmaf(left[k], __uint_as_float(w[e] & 0xffff0000u), sum[2 * e + 1]);
                    }
                }
            }
        }
        if (c < H)
            *reinterpret_cast<uint4*>(rest + (int64_t)begin * H + c) = make_uint4(rb_pair(sum[0], sum[1]), rb_pair(sum[2], sum[3]), rb_pair(sum[4], sum[5]), rb_pair(sum[6], sum[7]));
    }
}

// ---------------------------------------------------------------------------------------------
// Second launch of a piece: both products that read dl.  The tiles of grad_hidden (long contractions, over the piece's columns) start first, in `splits`
// ranges of it each, and those of grad_weight (over the tokens) fill the compute units beside and behind them.
//   grad_hidden: slabs [split][live tokens, padded][H] in binary32, this piece's share added to that of the ones before
//   grad_weight: rows v0 .. of the gradient, complete
// ---------------------------------------------------------------------------------------------
struct Products {
    const uint16_t* dl;
    int64_t rows;                // of its panels, and of a slab: the tokens, padded to grad_hidden's tiles
    const uint16_t* weight;      // the piece's first row
    int64_t ldw;
    const uint16_t* gathered;    // live rows of hidden
    float* slabs;                // nullptr: grad_hidden is not wanted
    uint16_t* grad_weight;       // nullptr: grad_weight is not wanted
    const int* index;
    const int* row_of;           // by the piece's rows, and
    const uint16_t* rest;        // what they are to have added (head_targets_kernel)
    int width, H, splits, first; // first: the slabs hold nothing yet
};
// Tile `job` of grad_hidden.
template <int TMX>
__device__ __forceinline__ void hl_hidden_tile(uint8_t* hl_lds, const Products& p, int count, int job, int tiles_t, int tiles_h)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3, lr = lane & 31, hi = lane >> 5;
    const int split = job / (tiles_t * tiles_h);
    int tm, tn;
    hl_origin(job - split * tiles_t * tiles_h, tiles_t, tiles_h, tm, tn);
    const int m0 = tm * 64 * TMX, n0 = tn * HL_BN, kt = (p.width + 31) / 32, pairs = (kt + 1) / 2;
    const int begin = 2 * (int)((int64_t)split * pairs / p.splits), end = min(kt, 2 * (int)((int64_t)(split + 1) * pairs / p.splits));
    float* slab = p.slabs + ((int64_t)split * p.rows + m0) * p.H + n0;
    float16_t acc[TMX][HL_TN];
    hl_clear<TMX>(acc);
    // the lane's places in the slab, four columns at a time
    auto each = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < TMX; ++i) {
            const int row = (wm * TMX + i) * 32 + lr;
            if (m0 + row >= count) continue;
#pragma unroll
            for (int j = 0; j < HL_TN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = wn * 64 + j * 32 + 8 * g + 4 * hi;
                    if (n0 + n < p.H) f(acc[i][j], 4 * g, reinterpret_cast<float4*>(slab + (int64_t)row * p.H + n));
                }
        }
    };
    if (!p.first)
        each([](float16_t& v, int e, const float4* q) {
            const float4 x = *q;
            v[e] = x.x; v[e + 1] = x.y; v[e + 2] = x.z; v[e + 3] = x.w;
        });
    const Operand a = {p.dl + (int64_t)(begin / 2) * p.rows * 64 + m0 * 64, 64, 64 * TMX, nullptr, 32, p.rows * 64};
    const Operand b = {p.weight + (int64_t)begin * 32 * p.ldw + n0, p.ldw, p.H - n0, nullptr, end == kt && p.width % 32 ? p.width % 32 : 32, 0};
    Pipe<TMX, false, true, true> pipe;
    pipe.lds = hl_lds;
    pipe.aim(a, b, end - begin, false);
    pipe.request(0);
    pipe.request(2);
    pipe.multiply(acc);
    each([](const float16_t& v, int e, float4* q) { *q = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]); });
}

template <int ROWS>
__global__ __launch_bounds__(HL_THREADS, 2) void head_products_kernel(const Products p)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t hl_lds[];
    const int count = p.index[0], tmx = ROWS == kList ? 1 : ROWS == kMany ? 4 : hl_row_tiles(count);
    const int tiles_t = (count + 64 * tmx - 1) / (64 * tmx), tiles_h = (p.H + HL_BN - 1) / HL_BN, tiles_v = (p.width + 255) / 256;
    const int xcd = blockIdx.x & 7;
    int li = blockIdx.x >> 3;
    const int hidden_jobs = p.slabs ? tiles_t * tiles_h * p.splits : 0, hidden_x = (hidden_jobs + 7) >> 3;
    if (li < hidden_x) {
        const int job = xcd * hidden_x + li;
        if (job < hidden_jobs)
            with_row_tiles<ROWS>(count, [&](auto tm) { hl_hidden_tile<decltype(tm)::value>(hl_lds, p, count, job, tiles_t, tiles_h); });
        return;
    }
    if (!p.grad_weight) return;
    li -= hidden_x;
    const int jobs = tiles_v * tiles_h, per = (jobs + 7) >> 3, job = xcd * per + li;
    if (li >= per || job >= jobs) return;
    int tm, tn;
    hl_origin(job, tiles_v, tiles_h, tm, tn);
    const int m0 = tm * 256, n0 = tn * HL_BN, wn = (threadIdx.x >> 6) & 3;
    const int thread = hl_thread(), lane = thread & 63, wm = thread >> 8, lr = lane & 31, hi = lane >> 5;
    // Sums begin with what the targets' rows are to have added: which rows, asked for before the ring's stages (5 x 1536 against 131072, both gradients: 305 us;
    // behind the products 313, and 297 without the targets' remainders), the values behind them.
    float16_t acc[4][HL_TN];
    hl_clear<4>(acc);
    int from[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) from[i] = p.row_of[m0 + (wm * 4 + i) * 32 + lr];
    Pipe<4, true, true, true> pipe;
    pipe.lds = hl_lds;
    pipe.aim(Operand{p.dl + (int64_t)(m0 / 64) * p.rows * 64, 64, 256, nullptr, 32, p.rows * 64}, Operand{p.gathered + n0, p.H, p.H - n0, nullptr, 32, 0}, (count + 31) / 32, false);
    pipe.request(0);
    pipe.request(2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (from[i] < 0) continue;
        const uint16_t* rest = p.rest + (int64_t)from[i] * p.H + n0 + wn * 64 + 4 * hi;
#pragma unroll
        for (int j = 0; j < HL_TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (n0 + wn * 64 + j * 32 + 8 * g + 4 * hi >= p.H) continue;
                const uint2 r = *reinterpret_cast<const uint2*>(rest + j * 32 + 8 * g);
                acc[i][j][4 * g] = __uint_as_float(r.x << 16);
                acc[i][j][4 * g + 1] = __uint_as_float(r.x & 0xffff0000u);
                acc[i][j][4 * g + 2] = __uint_as_float(r.y << 16);
                acc[i][j][4 * g + 3] = __uint_as_float(r.y & 0xffff0000u);
            }
    }
    pipe.multiply(acc);
    hl_store_bf16<4>(acc, hl_lds, p.grad_weight + (int64_t)m0 * p.H + n0 + wn * 64, p.H, p.width - m0, p.H - (n0 + wn * 64));
}

// grad_hidden of every token: the slabs of a live one added in order, then what its dl at the target left, zero for the others.
__global__ __launch_bounds__(256) void head_hidden_kernel(const float* __restrict__ slabs, int splits, int64_t slab_rows, const int* __restrict__ index, int tokens, int H,
                                                          const uint16_t* __restrict__ weight, int64_t ldw, const AtTarget target, uint16_t* __restrict__ out)
{
    const int quads = H / 4;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < (int64_t)tokens * quads; at += (int64_t)gridDim.x * 256) {
        const int t = (int)(at / quads), c = (int)(at - (int64_t)t * quads), pos = live_rows(index)[tokens + t];
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (pos >= 0) {
            const int column = target.column[pos];
            const float left = target.left[pos];
            uint2 w = make_uint2(0u, 0u);
            if (column >= 0) w = *reinterpret_cast<const uint2*>(weight + (int64_t)column * ldw + c * 4);
            for (int s = 0; s < splits; ++s) {
                const float4 q = *reinterpret_cast<const float4*>(slabs + ((int64_t)s * slab_rows + pos) * H + c * 4);
                v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
            }
            v.x = fmaf(left, __uint_as_float(w.x << 16), v.x);
            v.y = fmaf(left, __uint_as_float(w.x & 0xffff0000u), v.y);
            v.z = fmaf(left, __uint_as_float(w.y << 16), v.z);
            v.w = fmaf(left, __uint_as_float(w.y & 0xffff0000u), v.w);
        }
        *reinterpret_cast<uint2*>(out + (int64_t)t * H + c * 4) = make_uint2(rb_pair(v.x, v.y), rb_pair(v.z, v.w));
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
int rows_kind(int64_t tokens) { return tokens <= kListTokens ? kList : tokens <= kFewTokens ? kFew : kMany; }
// the most tiles over tokens that a launch may have
int64_t most_row_tiles(int64_t tokens) { return tokens <= kListTokens ? 1 : tokens <= kFewTokens ? (tokens + 191) / 192 : (tokens + 255) / 256; }
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
// products is one pass over that gradient).  Splits of grad_hidden's contraction: beside grad_weight, whose tiles fill the launch up, as many as leave none of
// its tiles longer than a compute unit's share; by itself those with the fewest stages in a row, a tile's beginning and end counted as eight and a pass over the
// slabs as its bytes (in a stage's 0.8 us 4 MB go), for tokens that are all live.  (By itself with the share's rule 540 x 2048 against 65536 had 11 splits of 24
// tiles, a second round of eight: 442 us, now 352; 5 x 1536 against 131072 222 and 174, 64 x 3584 499 and 373, 4096 x 3584 7.0 and 6.7 ms.)
BackwardPlan backward_plan(int64_t tokens, int64_t H, int64_t V, bool want_weight)
{
    BackwardPlan p;
    p.rows = tokens <= kListTokens ? 64 : tokens <= kFewTokens ? padded(tokens, 64) + 192 : padded(tokens, 256);      // (a tile begins with a token)
    int64_t bytes = 8 * p.rows * H;
    if (bytes < ((int64_t)256 << 20)) bytes = (int64_t)256 << 20;
    int64_t most = bytes / (2 * p.rows) / 256 * 256;
    if (most < 256) most = 256;
    const int64_t pieces = (V + most - 1) / most;
    p.width = padded((V + pieces - 1) / pieces, 256);
    const int64_t tiles_h = (H + 255) / 256, stages = p.width / 32;
    const int64_t rows = tokens <= kListTokens ? 64 : 64 * (tokens <= kFewTokens ? hl_row_tiles((int)tokens) : 4), tiles = (tokens + rows - 1) / rows * tiles_h;
    const int64_t all = tiles * stages + (want_weight ? p.width / 256 * tiles_h * ((tokens + 31) / 32) : 0), cus = device_cus();
    int64_t share = (all + cus - 1) / cus;
    if (share < 16) share = 16;
    int64_t s = (stages + share - 1) / share;
    if (s > 64) s = 64;
    p.splits = (int)(s < 1 ? 1 : s);
    if (want_weight) return p;
    double least = 0.0;
    for (int n = 1; n <= 64 && (n == 1 || n * 16 <= stages); ++n) {
        const double rounds = (double)((tiles * n + cus - 1) / cus), cost = rounds * ((double)stages / n + 8.0) + (double)n * (double)p.rows * (double)H * 8.0 / 4e6;
        if (n == 1 || cost < least) {
            least = cost;
            p.splits = n;
        }
    }
    return p;
}
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// f with the kind of launch
template <class F> int with_rows(int64_t tokens, F&& f)
{
    switch (rows_kind(tokens)) {
        case kList: return f(std::integral_constant<int, kList>{});
        case kFew: return f(std::integral_constant<int, kFew>{});
        default: return f(std::integral_constant<int, kMany>{});
    }
}
// a workgroup for each tile, alike on all XCDs
unsigned tile_grid(int64_t tiles) { return (unsigned)((tiles + 7) / 8 * 8); }
// LDS of a kernel whose tiles have at most 64 TM rows
constexpr size_t ring_bytes(int TM) { return (size_t)HL_NS * hl_stage_bytes(TM); }

template <int ROWS, bool ENT>
int launch_stats(const Tokens& tk, const void* weight, int64_t ldw, int stride, float2* part, float* part_e, float* hit, int64_t ignore, int* list, hipStream_t st)
{
    static bool done[64] = {};
    const size_t lds = ROWS == kList ? ring_bytes(1) + kListTokens * sizeof(int) : ring_bytes(4);
    if (const int rc = allow_dynamic_lds((const void*)head_stats_kernel<ROWS, ENT>, lds, done)) return rc;
    const unsigned tiles = tile_grid(most_row_tiles(tk.tokens) * ((tk.V + HL_BN - 1) / HL_BN)), cus = (unsigned)(device_cus() + 7) / 8 * 8;
    hipLaunchKernelGGL((head_stats_kernel<ROWS, ENT>), dim3(tiles < cus ? tiles : cus), dim3(HL_THREADS), lds, st, tk, (const uint16_t*)weight, ldw, stride, part, part_e, hit,
                       ignore, list);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

template <int ROWS>
int launch_dlogits(const Tokens& tk, const void* weight, int64_t ldw, int v0, int width, const RowGrads& rg, const AtTarget& target, uint16_t* dl, int64_t panel, hipStream_t st)
{
    static bool done[64] = {};
    const size_t lds = ring_bytes(ROWS == kList ? 1 : 4);
    if (const int rc = allow_dynamic_lds((const void*)head_dlogits_kernel<ROWS>, lds, done)) return rc;
    hipLaunchKernelGGL((head_dlogits_kernel<ROWS>), dim3(tile_grid(most_row_tiles(tk.tokens) * ((width + HL_BN - 1) / HL_BN))), dim3(HL_THREADS), lds, st, tk, (const uint16_t*)weight, ldw, v0,
                       width, rg, target, dl, panel);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

template <int ROWS>
int launch_products(const Products& p, unsigned grid, hipStream_t st)
{
    static bool done[64] = {};
    const size_t lds = ring_bytes(4);
    if (const int rc = allow_dynamic_lds((const void*)head_products_kernel<ROWS>, lds, done)) return rc;
    hipLaunchKernelGGL((head_products_kernel<ROWS>), dim3(grid), dim3(HL_THREADS), lds, st, p);
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
    return temperature > 0.0f && temperature < INFINITY && 1.44269504088896f / temperature < INFINITY;
}

}  // namespace

size_t head_index_bytes(int64_t tokens) { return tokens < 0 || tokens > (1 << 24) ? 0 : align256((size_t)index_words(tokens) * sizeof(int)); }

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
    if (tokens > kListTokens) {
        hipLaunchKernelGGL(head_index_kernel, dim3(1), dim3(1024), 0, st, (const int64_t*)targets, ignore, (int)tokens, (int*)index);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    const Tokens tk = tokens_of(hidden, ldh, targets, index, tokens, H, V, temperature);
    const int rc = with_rows(tokens, [&](auto rows) {
        return entropy ? launch_stats<decltype(rows)::value, true>(tk, weight, ldw, stride, part, part_e, hit, ignore, (int*)index, st)
                       : launch_stats<decltype(rows)::value, false>(tk, weight, ldw, stride, part, part_e, hit, ignore, (int*)index, st);
    });
    if (rc != METIS_OK) return rc;
    const dim3 grid((unsigned)((tokens + 15) / 16));
    if (entropy)
        hipLaunchKernelGGL((head_finish_kernel<true>), grid, dim3(1024), 0, st, (const int64_t*)targets, (int*)index, (int)tokens, (int)V, tiles_n, stride, tk.scale2, part, part_e, hit, logp, lse, entropy);
    else
        hipLaunchKernelGGL((head_finish_kernel<false>), grid, dim3(1024), 0, st, (const int64_t*)targets, (int*)index, (int)tokens, (int)V, tiles_n, stride, tk.scale2, part, part_e, hit, logp, lse, entropy);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

size_t head_logprobs_backward_workspace_bytes(int64_t tokens, int64_t H, int64_t V, int want_hidden, int want_weight)
{
    if (tokens <= 0 || !sizes_ok(tokens, H, V)) return 0;
    const BackwardPlan p = backward_plan(tokens, H, V, want_weight != 0);
    return align256((size_t)p.rows * p.width * 2) + 3 * align256((size_t)p.rows * 4) + (want_weight ? 2 * align256((size_t)p.rows * H * 2) + (size_t)padded(V, 256) * 4 : 0) + (want_hidden ? align256((size_t)p.splits * p.rows * H * 4) : 0);
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
    auto take = [&](size_t bytes) {
        char* here = at;
        at += align256(bytes);
        return here;
    };
    const size_t by_row = (size_t)p.rows * 4;
    AtTarget target;
    target.rounded = reinterpret_cast<float*>(take(by_row));
    target.left = reinterpret_cast<float*>(take(by_row));
    target.column = reinterpret_cast<int*>(take(by_row));
    uint16_t *gathered = nullptr, *rest = nullptr;
    int* row_of = nullptr;
    if (grad_weight) {
        gathered = reinterpret_cast<uint16_t*>(take((size_t)p.rows * H * 2));
        rest = reinterpret_cast<uint16_t*>(take((size_t)p.rows * H * 2));
        row_of = reinterpret_cast<int*>(take((size_t)padded(V, 256) * 4));
    }
    float* slabs = grad_hidden ? reinterpret_cast<float*>(at) : nullptr;
    const Tokens tk = tokens_of(hidden, ldh, targets, index, tokens, H, V, temperature);
    const RowGrads rg = {lse, entropy, g_logp, g_entropy};
    const int cus = device_cus();
    const int64_t teams = gathered ? tokens + 31 : (tokens + 255) / 256;
    hipLaunchKernelGGL(head_gather_kernel, dim3((unsigned)(teams < 8 * (int64_t)cus ? teams : 8 * (int64_t)cus)), dim3(256), 0, st, tk, rg, target, (uint4*)gathered);
    if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    if (grad_weight) {
        const int64_t fit = 2 * (int64_t)cus / ((V + 255) / 256), chunks = (H + 511) / 512;
        const unsigned share = (unsigned)(fit < 1 ? 1 : fit < chunks ? fit : chunks);
        hipLaunchKernelGGL(head_targets_kernel, dim3((unsigned)((V + 255) / 256), share), dim3(1024), 0, st, (const int*)index, target, (const uint16_t*)gathered, (int)H,
                           row_of, rest);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    const int64_t tiles_h = (H + 255) / 256;
    for (int64_t v0 = 0; v0 < V; v0 += p.width) {
        const int width = (int)(V - v0 < p.width ? V - v0 : p.width);
        int rc = with_rows(tokens, [&](auto rows) { return launch_dlogits<decltype(rows)::value>(tk, weight, ldw, (int)v0, width, rg, target, dl, p.rows * 64, st); });
        if (rc != METIS_OK) return rc;
        const Products pr = {dl, p.rows, (const uint16_t*)weight + v0 * ldw, ldw, gathered, slabs, grad_weight ? (uint16_t*)grad_weight + v0 * H : nullptr, (const int*)index,
                             row_of ? row_of + v0 : nullptr, rest, width, (int)H, p.splits, v0 == 0};
        const int64_t hidden_jobs = slabs ? most_row_tiles(tokens) * tiles_h * p.splits : 0, weight_jobs = grad_weight ? (width + 255) / 256 * tiles_h : 0;
        const unsigned grid = 8u * (unsigned)((hidden_jobs + 7) / 8 + (weight_jobs + 7) / 8);
        rc = with_rows(tokens, [&](auto rows) { return launch_products<decltype(rows)::value>(pr, grid, st); });
        if (rc != METIS_OK) return rc;
    }
    if (grad_hidden) {
        const int64_t need = (tokens * (H / 4) + 255) / 256, cap = (int64_t)cus * 16;
        hipLaunchKernelGGL(head_hidden_kernel, dim3((unsigned)(need < cap ? need : cap)), dim3(256), 0, st, (const float*)slabs, p.splits, p.rows, (const int*)index, (int)tokens, (int)H,
                           (const uint16_t*)weight, ldw, target, (uint16_t*)grad_hidden);
        if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    }
    return METIS_OK;
}

}  // namespace metis
