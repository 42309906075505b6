// The residual sum behind a block with the norms before and after it, and its gradients.
//
//   z = y            or   y rstd(y) post_weight
//   h = x + scale gate z                    stored in x's type
//   n = h rstd(h) weight                    of h as it is stored, rounded once
//   rstd(t) = 1 / sqrt(mean(t^2) + eps)
//
// and with gh, gn the gradients of h and n, hh = h rstd(h), yh = y rstd(y), all in binary32:
//   d     = gh + rstd(h) (gn weight - hh mean(gn weight hh))                       the gradient of x
//   dz    = scale gate d                                                           the gradient of y, or
//   gy    = rstd(y) (dz post_weight - yh mean(dz post_weight yh))
//   gweight = sum gn hh,   gpost = sum dz yh,   ggate = sum over the rows of a gate's row of scale d z
//
// A row belongs to W waves (one per 512 columns up to 2048, then four or eight), lane l of wave w holding the chunks of eight elements
// (i W + w) 64 + l: every access instruction of a wave covers consecutive bytes, the row is read once, its sums are folded across the lanes with
// DPP moves and across the waves through LDS.  Bound by memory: 8192 x 3584 bf16 forward 40 us and backward 40, both 5.9 TB/s of 8 bytes an element (x, y
// read, h, n written; h, gh, gn read, gx written, which is gy too where nothing lies between the sum and y), and 4 us for the columns' sums.
#include "chunk8.h"
#include "metis_host.h"

namespace metis {

template <int CTRL> __device__ __forceinline__ float rn_dpp(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// sum over the 64 lanes, the same value in every lane
__device__ __forceinline__ float rn_wave_sum(float v)
{
    v += rn_dpp<0xB1>(v);
    v += rn_dpp<0x4E>(v);
    v += rn_dpp<0x141>(v);
    v += rn_dpp<0x140>(v);
    const int b = __builtin_bit_cast(int, v);
    const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0)), r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
    const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32)), r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
    return (r0 + r1) + (r2 + r3);
}

// Sums of up to three numbers over the waves of a row.  Two areas in turn: a wave writes an area again only behind the barrier of the
// other one, which every wave passes after it has read the first.
template <int W> struct RowSums {
    static constexpr int kWords = W > 1 ? 2 * 3 * W : 1;       // for the waves of one row
    float* area;
    int turn = 0;
    template <int N> __device__ __forceinline__ void operator()(float (&v)[N], int wave)
    {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = rn_wave_sum(v[k]);
        if constexpr (W > 1) {
            float* a = area + turn * 3 * W;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int k = 0; k < N; ++k) a[k * W + wave] = v[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) s += a[k * W + w];
                v[k] = s;
            }
        }
    }
};

template <class R, class B, int NL, int W, bool POST>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void residual_norm_kernel(const void* __restrict__ x, const void* __restrict__ y, const void* __restrict__ weight,
                                                                             const void* __restrict__ post, const void* __restrict__ gate, uint32_t gate_every,
                                                                             float scale, float eps, uint32_t rows, uint32_t cols, void* __restrict__ h,
                                                                             void* __restrict__ n)
{
    constexpr int WAVES = W > 4 ? W : 4, ROWS = WAVES / W;
    __shared__ float area[ROWS][RowSums<W>::kWords];
    const uint32_t cpr = cols / 8u, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, part = wave % W, team = wave / W;
    RowSums<W> fold{area[team]};
    const float fcols = (float)cols;
    B wt[NL], pw[POST ? NL : 1];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const uint32_t c = (i * W + part) * 64u + lane;
        wt[i].zero();
        if (c < cpr) wt[i].load(weight, c);
        if constexpr (POST) {
            pw[i].zero();
            if (c < cpr) pw[i].load(post, c);
        }
    }
    // (all teams go round as often as the first: the folds hold barriers for all of them)
    for (uint32_t row0 = blockIdx.x * ROWS; row0 < rows; row0 += gridDim.x * ROWS) {
        const uint32_t row = row0 + team;
        const bool live = row < rows;
        R xr[NL];
        B yr[NL], gr[NL];
        const size_t at = (size_t)row * cpr, gate_at = gate && live ? (size_t)(row / gate_every) * cpr : 0;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t c = (i * W + part) * 64u + lane;
            xr[i].zero();
            yr[i].zero();
            gr[i].zero();
            if (live && c < cpr) {
                yr[i].load(y, at + c);
                xr[i].load(x, at + c);
                if (gate) gr[i].load(gate, gate_at + c);
            }
        }
        float ry = 1.0f;
        if constexpr (POST) {
            float ss[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < NL; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) ss[0] = fmaf(yr[i].get(j), yr[i].get(j), ss[0]);
            fold(ss, part);
            ry = 1.0f / sqrtf(ss[0] / fcols + eps);
        }
        float ss[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float z = yr[i].get(j);
                if constexpr (POST) z = z * ry * pw[i].get(j);
                f[j] = fmaf(gate ? scale * gr[i].get(j) : scale, z, xr[i].get(j));
            }
            xr[i].set(f);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss[0] = fmaf(xr[i].get(j), xr[i].get(j), ss[0]);
        }
        fold(ss, part);
        const float rh = 1.0f / sqrtf(ss[0] / fcols + eps);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t c = (i * W + part) * 64u + lane;
            if (!live || c >= cpr) continue;
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = xr[i].get(j) * rh * wt[i].get(j);
            B out;
            out.set(f);
            xr[i].store(h, at + c);
            out.store(n, at + c);
        }
    }
}

// Gradients.  A workgroup owns every slabs-th row (set of ROWS) of one gate row's rows and keeps the column sums of its rows in registers; they go to
// partial rows of the workspace, [sum][gate row][slab][column], which residual_norm_sums_kernel adds in order.  No gate: one gate row for all rows.
// Where there are more gate rows than workgroups a workgroup takes several, one after the other, and writes the gate's gradient itself.
//
// The sums' registers leave room for two waves per SIMD, one workgroup of eight per compute unit: two of four leave twice the partial rows (512 x 3584 bf16 12.8 us,
// now 10.6, 2048 x 3584 17.3 and 16.1, 4099 x 3584 39.6 and 38.8; 2103 x 4096 with a norm behind the block and gates, binary32 stream, is the one that loses,
// 42.1 and 43.7 with the sums).  A row's reads have to be under way while the one before is worked on: the next row is requested before the folds (AHEAD; where
// the registers hold it).  weight, post_weight and the gate stay in LDS, every lane reading what it put there itself.
template <class R, class B> struct RowIn {                    // one chunk of the lane's share of a row
    R h, gh;
    B gn, y;
};
template <class R, class B, int NL, int W, bool POST>
__global__ __launch_bounds__(512, 2) void residual_norm_backward_kernel(
    const void* __restrict__ h, const void* __restrict__ y, const void* __restrict__ weight, const void* __restrict__ post, const void* __restrict__ gate,
    uint32_t groups, uint32_t group_rows, uint32_t slabs, float scale, float eps, uint32_t cols, const void* __restrict__ gh, const void* __restrict__ gn,
    void* __restrict__ gx, void* __restrict__ gy, float* __restrict__ sum_w, float* __restrict__ sum_p, float* __restrict__ sum_g, void* __restrict__ ggate)
{
    constexpr int ROWS = 8 / W, THREADS = 512;                 // rows at once
    constexpr bool AHEAD = !(POST && NL == 2 && R::bytes == 32 && (W != 4 || B::bytes == 32));
    __shared__ float area[ROWS][RowSums<W>::kWords];
    __shared__ float turn[ROWS > 1 ? W * NL * 64 * 8 : 1];
    __shared__ B vec_w[NL][THREADS], vec_p[POST ? NL : 1][POST ? THREADS : 1], vec_g[NL][THREADS];
    const uint32_t cpr = cols / 8u, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, part = wave % W, team = wave / W;
    RowSums<W> fold{area[team]};
    const float inv_cols = 1.0f / (float)cols, fcols = (float)cols;
    float acc_w[NL][8], acc_p[POST ? NL : 1][8], acc_g[NL][8];
    auto clear = [](float(&a)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = 0.0f;
    };
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const uint32_t c = (i * W + part) * 64u + lane;
        clear(acc_w[i]);
        clear(acc_g[i]);
        if constexpr (POST) clear(acc_p[i]);
        B v;
        v.zero();
        if (c < cpr) v.load(weight, c);
        vec_w[i][threadIdx.x] = v;
        if constexpr (POST) {
            v.zero();
            if (c < cpr) v.load(post, c);
            vec_p[i][threadIdx.x] = v;
        }
    }
    // the sums of a workgroup: those of its teams in order
    auto write_sums = [&](float(&a)[NL][8], float* out, void* rounded) {
        if constexpr (ROWS > 1) {
            float* mine = turn + part * (NL * 64 * 8) + lane;
            for (uint32_t v = 0; v < (uint32_t)ROWS; ++v) {
                if (team == v) {
#pragma unroll
                    for (int i = 0; i < NL; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float* t = mine + (i * 8 + j) * 64;
                            *t = v ? *t + a[i][j] : a[i][j];
                        }
                }
                __syncthreads();
            }
            if (team == 0) {
#pragma unroll
                for (int i = 0; i < NL; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[i][j] = mine[(i * 8 + j) * 64];
            }
            __syncthreads();
            if (team) return;
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t c = (i * W + part) * 64u + lane;
            if (c >= cpr) continue;
            if (rounded) {
                B o;
                o.set(a[i]);
                o.store(rounded, c);
            } else {
                F32x8 o;
                o.set(a[i]);
                o.store(out, c);
            }
        }
    };
    const uint32_t slab = blockIdx.x % slabs;
    for (uint32_t group = blockIdx.x / slabs; group < groups; group += gridDim.x / slabs) {
        RowIn<R, B> in[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t c = (i * W + part) * 64u + lane;
            B v;
            v.zero();
            if (gate && c < cpr) v.load(gate, (size_t)group * cpr + c);
            vec_g[i][threadIdx.x] = v;
            in[i].h.zero();
            in[i].gh.zero();
            in[i].gn.zero();
            in[i].y.zero();
        }
        auto request = [&](uint32_t r) {
            const size_t at = ((size_t)group * group_rows + r) * cpr;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint32_t c = (i * W + part) * 64u + lane;
                if (c < cpr) {
                    in[i].h.load(h, at + c);
                    if (gn) in[i].gn.load(gn, at + c);
                    if (gh) in[i].gh.load(gh, at + c);
                    if (y) in[i].y.load(y, at + c);
                }
            }
        };
        // (all teams go round as often as the first: the folds hold barriers for all; one without a row adds nothing)
        const uint32_t step = slabs * ROWS;
        if (AHEAD && slab * ROWS + team < group_rows) request(slab * ROWS + team);
        for (uint32_t r0 = slab * ROWS; r0 < group_rows; r0 += step) {
            const uint32_t r = r0 + team;
            const bool live = r < group_rows;
            const size_t at = ((size_t)group * group_rows + r) * cpr;
            if (!AHEAD && live) request(r);
            RowIn<R, B> cur[NL];
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                cur[i] = in[i];
                if (ROWS > 1 && !live) {
                    cur[i].h.zero();
                    cur[i].gh.zero();
                    cur[i].gn.zero();
                    cur[i].y.zero();
                }
            }
            float s[POST ? 3 : 2] = {};                        // sum h^2, sum (gn weight) h, sum y^2
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const B wt = vec_w[i][threadIdx.x];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float hv = cur[i].h.get(j);
                    s[0] = fmaf(hv, hv, s[0]);
                    s[1] = fmaf(cur[i].gn.get(j) * wt.get(j), hv, s[1]);
                    if constexpr (POST) s[2] = fmaf(cur[i].y.get(j), cur[i].y.get(j), s[2]);
                }
            }
            if (AHEAD && r + step < group_rows) request(r + step);
            fold(s, part);
            const float rh = live ? 1.0f / sqrtf(s[0] / fcols + eps) : 0.0f, mean = s[1] * rh * inv_cols;
            float ry = live ? 1.0f : 0.0f;
            if constexpr (POST) ry = live ? 1.0f / sqrtf(s[2] / fcols + eps) : 0.0f;
            float dz[NL][8], dot[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint32_t c = (i * W + part) * 64u + lane;
                const B wt = vec_w[i][threadIdx.x], gt = vec_g[i][threadIdx.x], pw = vec_p[POST ? i : 0][POST ? threadIdx.x : 0];
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float hh = cur[i].h.get(j) * rh, gv = cur[i].gn.get(j);
                    acc_w[i][j] = fmaf(gv, hh, acc_w[i][j]);
                    d[j] = fmaf(rh, fmaf(gv, wt.get(j), -hh * mean), cur[i].gh.get(j));
                    const float sd = scale * d[j], yh = cur[i].y.get(j) * ry;
                    dz[i][j] = gate ? sd * gt.get(j) : sd;
                    if constexpr (POST) {
                        acc_g[i][j] = fmaf(sd, yh * pw.get(j), acc_g[i][j]);
                        acc_p[i][j] = fmaf(dz[i][j], yh, acc_p[i][j]);
                        dot[0] = fmaf(dz[i][j] * pw.get(j), yh, dot[0]);
                    } else {
                        acc_g[i][j] = fmaf(sd, yh, acc_g[i][j]);
                    }
                }
                if (gx && live && c < cpr) {
                    R o;
                    o.set(d);
                    o.store(gx, at + c);
                }
            }
            if constexpr (POST) fold(dot, part);
            if (!gy) continue;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint32_t c = (i * W + part) * 64u + lane;
                if (!live || c >= cpr) continue;
                const B pw = vec_p[POST ? i : 0][POST ? threadIdx.x : 0];
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    f[j] = dz[i][j];
                    if constexpr (POST) f[j] = ry * fmaf(dz[i][j], pw.get(j), -(cur[i].y.get(j) * ry) * (dot[0] * inv_cols));
                }
                B o;
                o.set(f);
                o.store(gy, at + c);
            }
        }
        if (sum_g || ggate) {                                  // this gate row's share
            write_sums(acc_g, sum_g ? sum_g + ((size_t)group * slabs + slab) * cols : nullptr, ggate ? static_cast<char*>(ggate) + (size_t)group * cpr * B::bytes : nullptr);
#pragma unroll
            for (int i = 0; i < NL; ++i) clear(acc_g[i]);
        }
    }
    if (sum_w) write_sums(acc_w, sum_w + (size_t)blockIdx.x * cols, nullptr);
    if constexpr (POST) {
        if (sum_p) write_sums(acc_p, sum_p + (size_t)blockIdx.x * cols, nullptr);
    }
}

// Partial rows added in a fixed order: output row 0 is weight's gradient, 1 post_weight's, 2 .. the gates'.  Sixteen chains of a column, each of every
// sixteenth partial row in order with eight requested together, then the chains in order.
template <class B>
__global__ __launch_bounds__(1024) void residual_norm_sums_kernel(const float* __restrict__ sum_w, const float* __restrict__ sum_p, const float* __restrict__ sum_g,
                                                                  uint32_t all, uint32_t slabs, uint32_t cols, void* __restrict__ gw, void* __restrict__ gp,
                                                                  void* __restrict__ gg)
{
    __shared__ float part[16][64];
    const uint32_t lane = threadIdx.x & 63u, chain = threadIdx.x >> 6, c = blockIdx.x * 64u + lane;
    const float* src = blockIdx.y == 0 ? sum_w : blockIdx.y == 1 ? sum_p : sum_g ? sum_g + (size_t)(blockIdx.y - 2) * slabs * cols : nullptr;
    if (!src) return;
    const uint32_t count = blockIdx.y < 2 ? all : slabs;
    float s = 0.0f;
    for (uint32_t k0 = chain; k0 < count; k0 += 128u) {
        float v[8];
#pragma unroll
        for (uint32_t b = 0; b < 8u; ++b) v[b] = (k0 + 16u * b < count && c < cols) ? src[(size_t)(k0 + 16u * b) * cols + c] : 0.0f;
#pragma unroll
        for (uint32_t b = 0; b < 8u; ++b) s += v[b];
    }
    part[chain][lane] = s;
    __syncthreads();
    if (chain || c >= cols) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += part[k][lane];
    void* out = blockIdx.y == 0 ? gw : blockIdx.y == 1 ? gp : gg;
    const size_t at = (blockIdx.y < 2 ? 0 : (size_t)(blockIdx.y - 2) * cols) + c;
    if constexpr (B::bytes == 16) static_cast<uint16_t*>(out)[at] = (uint16_t)bf16_bits(s);
    else static_cast<float*>(out)[at] = s;
}

namespace {

// waves of a row; a workgroup has eight, forward four where these are enough
int row_waves(int64_t cols, int y_dtype) { return cols <= 512 ? 1 : cols <= 1024 ? 2 : cols <= 2048 || (cols <= 4096 && y_dtype == METIS_DTYPE_BF16) ? 4 : 8; }

struct BackwardPlan {
    uint32_t groups, group_rows, slabs, grid;
    bool direct;                                               // more gate rows than workgroups: each writes its gate's gradient itself
};
BackwardPlan backward_plan(int64_t rows, int64_t cols, int y_dtype, int64_t gate_rows)
{
    BackwardPlan p;
    p.groups = gate_rows > 0 ? (uint32_t)gate_rows : 1u;
    p.group_rows = (uint32_t)(rows / p.groups);
    const uint32_t cap = (uint32_t)device_cus(), at_once = 8u / (uint32_t)row_waves(cols, y_dtype), need = (p.group_rows + at_once - 1) / at_once;
    p.slabs = p.groups >= cap ? 1u : cap / p.groups;
    if (p.slabs > need) p.slabs = need;
    p.grid = p.slabs * (p.groups < cap ? p.groups : cap);
    p.direct = p.slabs == 1;
    return p;
}

bool sizes_ok(int64_t rows, int64_t cols, int x_dtype, int y_dtype, int64_t gate_rows)
{
    if (rows < 0 || rows > INT32_MAX || cols <= 0 || cols > 8192 || cols % 8 || gate_rows < 0) return false;
    if ((x_dtype != METIS_DTYPE_BF16 && x_dtype != METIS_DTYPE_F32) || (y_dtype != METIS_DTYPE_BF16 && y_dtype != METIS_DTYPE_F32)) return false;
    if (x_dtype == METIS_DTYPE_BF16 && y_dtype == METIS_DTYPE_F32) return false;        // the residual stream is the wider of the two
    return gate_rows == 0 || rows % gate_rows == 0;
}
bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

// calls F with the kernel's types and widths
#define METIS_RN_WIDTH(F, R, B, P)                                                                                              \
    do {                                                                                                                        \
        if (cols <= 512) F(R, B, 1, 1, P);                                                                                      \
        else if (cols <= 1024) F(R, B, 1, 2, P);                                                                                \
        else if (cols <= 2048) F(R, B, 1, 4, P);                                                                                \
        else if (cols <= 4096) F(R, B, (B::bytes == 16 ? 2 : 1), (B::bytes == 16 ? 4 : 8), P);                                  \
        else F(R, B, 2, 8, P);                                                                                                  \
    } while (0)
#define METIS_RN_TYPES(F, P)                                                                    \
    do {                                                                                        \
        if (x_dtype == METIS_DTYPE_BF16) METIS_RN_WIDTH(F, Bf16x8, Bf16x8, P);                  \
        else if (y_dtype == METIS_DTYPE_BF16) METIS_RN_WIDTH(F, F32x8, Bf16x8, P);              \
        else METIS_RN_WIDTH(F, F32x8, F32x8, P);                                                \
    } while (0)

int residual_norm(const void* x, int x_dtype, const void* y, int y_dtype, const void* weight, const void* post, const void* gate, int64_t gate_rows, float scale,
                  float eps, int64_t rows, int64_t cols, void* h, void* n, hipStream_t st)
{
    if (!sizes_ok(rows, cols, x_dtype, y_dtype, gate_rows)) return METIS_E_ARG;
    if (rows == 0) return METIS_OK;
    if (!x || !y || !weight || !h || !n || (gate_rows > 0) != (gate != nullptr)) return METIS_E_ARG;
    if (!aligned(x) || !aligned(y) || !aligned(weight) || !aligned(post) || !aligned(gate) || !aligned(h) || !aligned(n)) return METIS_E_ARG;
    const int waves = row_waves(cols, y_dtype);
    const int64_t at_once = waves == 8 ? 1 : 4 / waves, need = (rows + at_once - 1) / at_once, cap = (int64_t)device_cus() * (waves == 8 ? 4 : 8);
    const unsigned grid = (unsigned)(need < cap ? need : cap), threads = waves == 8 ? 512 : 256;
    const uint32_t every = gate ? (uint32_t)(rows / gate_rows) : 1u;
#define METIS_RN_FWD(R, B, NL, W, P) hipLaunchKernelGGL((residual_norm_kernel<R, B, NL, W, P>), dim3(grid), dim3(threads), 0, st, x, y, weight, post, gate, every, \
                                                        scale, eps, (uint32_t)rows, (uint32_t)cols, h, n)
    if (post) METIS_RN_TYPES(METIS_RN_FWD, true);
    else METIS_RN_TYPES(METIS_RN_FWD, false);
#undef METIS_RN_FWD
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

size_t residual_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_rows)
{
    if (rows <= 0 || !sizes_ok(rows, cols, METIS_DTYPE_F32, METIS_DTYPE_F32, gate_rows)) return 0;
    const BackwardPlan p = backward_plan(rows, cols, METIS_DTYPE_F32, gate_rows);       // (its rows take the most waves: the most workgroups of the two types)
    return (size_t)p.grid * (size_t)cols * sizeof(float) * (gate_rows > 0 && !p.direct ? 3 : 2);
}

int residual_norm_backward(const void* h, int x_dtype, const void* y, int y_dtype, const void* weight, const void* post, const void* gate, int64_t gate_rows,
                           float scale, float eps, int64_t rows, int64_t cols, const void* gh, const void* gn, void* gx, void* gy, void* gweight, void* gpost,
                           void* ggate, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (!sizes_ok(rows, cols, x_dtype, y_dtype, gate_rows) || rows == 0) return METIS_E_ARG;
    if (!h || !weight || (gate_rows > 0) != (gate != nullptr) || (gpost && !post) || (ggate && !gate) || ((post || ggate) && !y)) return METIS_E_ARG;
    if (!aligned(h) || !aligned(y) || !aligned(weight) || !aligned(post) || !aligned(gate) || !aligned(gh) || !aligned(gn) || !aligned(gx) || !aligned(gy) ||
        !aligned(gweight) || !aligned(gpost) || !aligned(ggate))
        return METIS_E_ARG;
    if (!workspace || !aligned(workspace) || workspace_bytes < residual_norm_backward_workspace_bytes(rows, cols, gate_rows)) return METIS_E_WORKSPACE;
    const BackwardPlan p = backward_plan(rows, cols, y_dtype, gate_rows);
    float* sum_w = static_cast<float*>(workspace);
    float* sum_p = sum_w + (size_t)p.grid * cols;
    float* sum_g = ggate && !p.direct ? sum_p + (size_t)p.grid * cols : nullptr;
    if (!gweight) sum_w = nullptr;
    if (!gpost) sum_p = nullptr;
    const void* yy = (post || ggate) ? y : nullptr;
    void* direct = p.direct ? ggate : nullptr;
#define METIS_RN_BWD(R, B, NL, W, P) hipLaunchKernelGGL((residual_norm_backward_kernel<R, B, NL, W, P>), dim3(p.grid), dim3(512), 0, st, h, yy, weight, post, gate, \
                                                        p.groups, p.group_rows, p.slabs, scale, eps, (uint32_t)cols, gh, gn, gx, gy, sum_w, sum_p, sum_g, direct)
    if (post) METIS_RN_TYPES(METIS_RN_BWD, true);
    else METIS_RN_TYPES(METIS_RN_BWD, false);
#undef METIS_RN_BWD
    if (hipGetLastError() != hipSuccess) return METIS_E_LAUNCH;
    if (!sum_w && !sum_p && !sum_g) return METIS_OK;
    const dim3 g((unsigned)((cols + 63) / 64), sum_g ? 2u + p.groups : sum_p ? 2u : 1u);
    if (y_dtype == METIS_DTYPE_BF16)
        hipLaunchKernelGGL((residual_norm_sums_kernel<Bf16x8>), g, dim3(1024), 0, st, sum_w, sum_p, sum_g, p.grid, p.slabs, (uint32_t)cols, gweight, gpost, ggate);
    else
        hipLaunchKernelGGL((residual_norm_sums_kernel<F32x8>), g, dim3(1024), 0, st, sum_w, sum_p, sum_g, p.grid, p.slabs, (uint32_t)cols, gweight, gpost, ggate);
    return hipGetLastError() == hipSuccess ? METIS_OK : METIS_E_LAUNCH;
}

}  // namespace metis
