// The norms around a residual block, fused with its gate, its residual scale and the next block's norm, and their backward pass
// (include/lego_hip.h: lego_block_norm_*).  A row of `width` channels:
//
//   oh = o (mean o^2 + eps)^-1/2      y = x + scale act(gate) oh post_w      yh = y (mean y^2 + eps)^-1/2      n = yh next_w
//
// in one pass: x, o and gate are read once, y and n written once.  Without a block (o = NULL) y = x and only n is written.  HBM-bound: a row
// lives in the registers of 1 to 16 waves (16- / 8-byte loads, 4 channels a lane), the weights of a lane's channels stay in registers over the rows
// of a persistent workgroup, and the next row's loads are in flight while a row is summed -- without that the two dependent sums of a row left the
// memory idle (65536 x 1024 bf16, backward: 454 us, 212 with it; 5.1 TB/s, as a copy of that size).
//
// That holds for widths of 256 to 4096 that 4 divides.  Others are right, and slower than memory (32 M channels, fp32, TB/s of
// what a pass has to move; forward / backward of both halves, at 1024 5.5 / 5.0):
//   narrow rows leave lanes of their one wave idle                                            32: 2.6 / 1.7     64: 4.3 / 3.0
//   widths that 4 does not divide load single elements, in the widest form of their waves    257: 2.9 / 2.2   1001: 4.3 / 4.3   1025: 4.3 / 3.9
//   above 4096 a row takes 1024 lanes, which have 128 registers each: two rows spill        5120: 5.1 / 1.8   8192: 5.2 / 2.4  16384: 2.2 / 1.2
//   both                                                                                    4099: 0.7 / 0.3   8193: 1.1 / 0.5
//
// Backward, with d = dy + rms_y^-1 (dn next_w - yh mean(dn next_w yh)) the gradient of y:  dx = d,  e = d scale act post_w,
//   do = rms_o^-1 (e - oh mean(e oh)),  dgate = d scale oh post_w act'(gate),
//   z = sum_rows d act oh:  dpost_w = z scale, dscale = z post_w;  dnext_w = sum_rows dn yh.
// y is formed again in fp32 from x, o and gate (the stored y may be rounded to 16 bits); the two root mean squares are kept from the forward
// pass, so a row needs two sums.  Column sums: registers over a workgroup's rows, LDS over its waves, one partial row a workgroup, and a
// second launch adds those in a fixed order (no atomics: the same bits every time).
#include "seq_common.hpp"

namespace lego {

constexpr int BN_BLOCK = 1, BN_NEXT = 2;                               // which of the two halves a call computes

struct Rows { const void* p; int64_t ld; };
struct BlockNorm {
    Rows x, o, gate;
    const float *post_w, *scale, *next_w;
    float eps;
    int act, rows, width;
};

// act(g) and act'(g): 0 none, 1 sigmoid, 2 silu
__device__ __forceinline__ float gate_act(int act, float g, float& slope) {
    if (act == 0) { slope = 0.f; return 1.f; }
    // sigmoid(g) and 1 - sigmoid(g) = sigmoid(-g) from one exponential, the smaller one without a difference
    const float e = __builtin_amdgcn_exp2f(-1.44269504088896340736f * fabsf(g)), q = __builtin_amdgcn_rcpf(1.f + e), small = e * q;
    const float s = g < 0.f ? small : q, r = g < 0.f ? q : small;
    if (act == 1) { slope = s * r; return s; }
    const float v = g * s;
    slope = s + v * r;
    return v;
}

// sum over the row's waves; `red` is one of two buffers in turn, so that one barrier a sum is enough
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[16], int& turn) {
    v = wave_total(v);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[turn][0];
#pragma unroll
        for (int w = 1; w < WPR; ++w) v += red[turn][w];
        turn ^= 1;
    }
    return v;
}

// a lane's channels of a row's tensors, as they lie in memory
template <typename T, int N, int NJ, bool FULL>
struct Line {
    vec<T, 4> v[N][NJ];
    __device__ __forceinline__ void fetch(const Rows (&src)[N], int64_t row, int c0, int width) {
#pragma unroll
        for (int q = 0; q < N; ++q)
#pragma unroll
            for (int j = 0; j < NJ; ++j) v[q][j] = load_some<T, 4, FULL>((const T*)src[q].p + row * src[q].ld, c0 + 256 * j, width);
    }
    __device__ __forceinline__ f32x4 at(int q, int j) const { return __builtin_convertvector(v[q][j], f32x4); }
};

// the sum of a lane's 4 channels of f, without those behind the row
template <bool FULL>
__device__ __forceinline__ float in_row(f32x4 f, int c, int width) {
    if constexpr (FULL) return c < width ? (f[0] + f[1]) + (f[2] + f[3]) : 0.f;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) s += c + k < width ? f[k] : 0.f;
    return s;
}

template <int WPR> constexpr int kWaves = WPR == 1 ? 4 : WPR;          // one-wave rows: four of them a workgroup

template <typename T, int MODE, int WPR, int NJ, bool FULL>
__global__ __launch_bounds__(64 * kWaves<WPR>) void block_norm_fwd_kernel(BlockNorm p, T* __restrict__ y, T* __restrict__ next, float* __restrict__ stat) {
    __shared__ float red[2][16];
    constexpr int RPW = WPR == 1 ? 4 : 1;                              // rows a workgroup holds at a time
    constexpr int N = MODE & BN_BLOCK ? 3 : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int c0 = 4 * (lane + (WPR == 1 ? 0 : 64 * NJ * wave)), W = p.width;
    const float inv = 1.f / (float)W;
    Rows src[N];
    src[0] = p.x;
    if constexpr (MODE & BN_BLOCK) { src[1] = p.o; src[2] = p.act != 0 ? p.gate : p.x; }
    f32x4 wp[NJ], ws[NJ], wn[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int c = c0 + 256 * j;
        if constexpr (MODE & BN_BLOCK) { wp[j] = load<float, 4, FULL>(p.post_w, c, W); ws[j] = load<float, 4, FULL>(p.scale, c, W); }
        if constexpr (MODE & BN_NEXT) wn[j] = load<float, 4, FULL>(p.next_w, c, W);
    }
    int turn = 0;
    const int64_t step = (int64_t)gridDim.x * RPW;
    int64_t row = (int64_t)blockIdx.x * RPW + (WPR == 1 ? wave : 0);
    Line<T, N, NJ, FULL> in, ahead;
    in.fetch(src, row < p.rows ? row : p.rows - 1, c0, W);
    for (; row < p.rows; row += step) {
        ahead.fetch(src, row + step < p.rows ? row + step : p.rows - 1, c0, W);
        f32x4 v[NJ];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] = in.at(0, j);
        if constexpr (MODE & BN_BLOCK) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) s += in_row<FULL>(in.at(1, j) * in.at(1, j), c0 + 256 * j, W);
            const float ro = rsqrtf(row_sum<WPR>(s, red, turn) * inv + p.eps);
            if (stat != nullptr && threadIdx.x % (64 * WPR) == 0) stat[row] = ro;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f32x4 o = in.at(1, j), g = in.at(2, j);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float slope;
                    v[j][k] += ws[j][k] * gate_act(p.act, g[k], slope) * (o[k] * ro * wp[j][k]);
                }
                store<T, 4, FULL>(y + row * W, c0 + 256 * j, W, v[j]);
            }
        }
        if constexpr (MODE & BN_NEXT) {
            s = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) s += in_row<FULL>(v[j] * v[j], c0 + 256 * j, W);
            const float ry = rsqrtf(row_sum<WPR>(s, red, turn) * inv + p.eps);
            if (stat != nullptr && threadIdx.x % (64 * WPR) == 0) stat[(MODE & BN_BLOCK ? p.rows : 0) + row] = ry;
#pragma unroll
            for (int j = 0; j < NJ; ++j) store<T, 4, FULL>(next + row * W, c0 + 256 * j, W, v[j] * ry * wn[j]);
        }
        in = ahead;
    }
}

template <typename T, int MODE, int WPR, int NJ, bool FULL>
__global__ __launch_bounds__(64 * kWaves<WPR>) void block_norm_bwd_kernel(BlockNorm p, Rows dy, Rows dn, const float* __restrict__ stat,
                                                                         T* __restrict__ dx, T* __restrict__ dout, T* __restrict__ dgate,
                                                                         float* __restrict__ parts) {
    __shared__ float red[2][16];
    constexpr int RPW = WPR == 1 ? 4 : 1;
    constexpr int N = MODE == (BN_BLOCK | BN_NEXT) ? 5 : 3;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int c0 = 4 * (lane + (WPR == 1 ? 0 : 64 * NJ * wave)), W = p.width;
    const float inv = 1.f / (float)W;
    const f32x4 zero{0.f, 0.f, 0.f, 0.f};
    // what a row reads: dy first (any tensor in its place where there is none), then x and dn of the norm, o and the gate of the block
    constexpr int X = 1, DN = 2, O = MODE & BN_NEXT ? 3 : 1, G = O + 1;
    const bool has_dy = dy.p != nullptr;
    Rows src[N];
    src[0] = has_dy ? dy : p.x;
    if constexpr (MODE & BN_NEXT) { src[X] = p.x; src[DN] = dn; }
    if constexpr (MODE & BN_BLOCK) { src[O] = p.o; src[G] = p.act != 0 ? p.gate : p.o; }
    f32x4 wp[NJ], ws[NJ], wn[NJ], z[NJ], zn[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int c = c0 + 256 * j;
        if constexpr (MODE & BN_BLOCK) { wp[j] = load<float, 4, FULL>(p.post_w, c, W); ws[j] = load<float, 4, FULL>(p.scale, c, W); }
        if constexpr (MODE & BN_NEXT) wn[j] = load<float, 4, FULL>(p.next_w, c, W);
        z[j] = zn[j] = zero;
    }
    int turn = 0;
    const int64_t step = (int64_t)gridDim.x * RPW;
    int64_t row = (int64_t)blockIdx.x * RPW + (WPR == 1 ? wave : 0);
    Line<T, N, NJ, FULL> in, ahead;
    in.fetch(src, row < p.rows ? row : p.rows - 1, c0, W);
    for (; row < p.rows; row += step) {
        const float ro = MODE & BN_BLOCK ? stat[row] : 0.f, ry = MODE & BN_NEXT ? stat[(MODE & BN_BLOCK ? p.rows : 0) + row] : 0.f;
        ahead.fetch(src, row + step < p.rows ? row + step : p.rows - 1, c0, W);
        f32x4 oh[NJ], act[NJ], slope[NJ], d[NJ], t[NJ];
        if constexpr (MODE & BN_BLOCK) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f32x4 g = in.at(G, j);
                oh[j] = in.at(O, j) * ro;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float sl;
                    act[j][k] = gate_act(p.act, g[k], sl);
                    slope[j][k] = sl;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) d[j] = has_dy ? in.at(0, j) : zero;
        if constexpr (MODE & BN_NEXT) {
            f32x4 v[NJ];
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f32x4 g = in.at(DN, j);
                v[j] = in.at(X, j);
                if constexpr (MODE & BN_BLOCK) v[j] += ws[j] * act[j] * (oh[j] * wp[j]);
                v[j] *= ry;                                            // yh
                zn[j] += g * v[j];
                t[j] = g * wn[j];
                s += in_row<FULL>(t[j] * v[j], c0 + 256 * j, W);
            }
            const float m = row_sum<WPR>(s, red, turn) * inv;
#pragma unroll
            for (int j = 0; j < NJ; ++j) d[j] += ry * (t[j] - v[j] * m);
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) store<T, 4, FULL>(dx + row * W, c0 + 256 * j, W, d[j]);
        if constexpr (MODE & BN_BLOCK) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                z[j] += d[j] * act[j] * oh[j];
                const f32x4 e = d[j] * ws[j] * wp[j];
                t[j] = e * act[j];
                s += in_row<FULL>(t[j] * oh[j], c0 + 256 * j, W);
                if (p.act != 0) store<T, 4, FULL>(dgate + row * W, c0 + 256 * j, W, e * oh[j] * slope[j]);
            }
            const float m = row_sum<WPR>(s, red, turn) * inv;
#pragma unroll
            for (int j = 0; j < NJ; ++j) store<T, 4, FULL>(dout + row * W, c0 + 256 * j, W, ro * (t[j] - oh[j] * m));
        }
        in = ahead;
    }
    // this workgroup's partial column sums: parts[workgroup][0] = z, [1] = zn
    float* mine = parts + (int64_t)blockIdx.x * 2 * W;
    if constexpr (WPR > 1) {                                           // each wave holds columns of its own
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (MODE & BN_BLOCK) store<float, 4, FULL>(mine, c0 + 256 * j, W, z[j]);
            if constexpr (MODE & BN_NEXT) store<float, 4, FULL>(mine + W, c0 + 256 * j, W, zn[j]);
        }
    } else {
        __shared__ f32x4 fold[4][64 * NJ];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (!(MODE & (half == 0 ? BN_BLOCK : BN_NEXT))) continue;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NJ; ++j) fold[wave][lane + 64 * j] = half == 0 ? z[j] : zn[j];
            __syncthreads();
            for (int q = threadIdx.x; q < 64 * NJ; q += 256)
                store<float, 4, FULL>(mine + half * W, 4 * q, W, (fold[0][q] + fold[1][q]) + (fold[2][q] + fold[3][q]));
        }
    }
}

// the partial rows of all workgroups: 16 columns x 64 row lanes a workgroup, 8 rows of a lane in flight
__global__ __launch_bounds__(1024) void block_norm_weights_kernel(const float* __restrict__ parts, int n_parts, int mode, const float* __restrict__ post_w,
                                                                  const float* __restrict__ scale, float* __restrict__ dpost_w,
                                                                  float* __restrict__ dscale, float* __restrict__ dnext_w, int width) {
    __shared__ float red[2][64][17];
    const int col = threadIdx.x & 15, lane = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (!(mode & (half == 0 ? BN_BLOCK : BN_NEXT))) continue;
        float s = 0.f;
        if (c < width)
            for (int q = lane; q < n_parts; q += 64 * 8) {
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = q + 64 * u < n_parts ? parts[((int64_t)(q + 64 * u) * 2 + half) * width + c] : 0.f;
#pragma unroll
                for (int u = 0; u < 8; ++u) s += v[u];
            }
        red[half][lane][col] = s;
    }
    __syncthreads();
    if (threadIdx.x < 32 && c < width) {
        const int half = threadIdx.x >> 4;
        if (mode & (half == 0 ? BN_BLOCK : BN_NEXT)) {
            float s = 0.f;
            for (int q = 0; q < 64; ++q) s += red[half][q][col];
            if (half == 0) { dpost_w[c] = s * scale[c]; dscale[c] = s * post_w[c]; }
            else dnext_w[c] = s;
        }
    }
}

// Waves a row and 4-channel groups a lane: one wave to 1024 channels (no barrier in its sums), then 4, 8 and 16 waves of two groups, as many lanes as
// the width needs; four groups in 16 waves above 8192.  Measured backwards, bf16, TB/s: 1024 channels in 1 x 4 / 2 x 2 / 4 x 1 (waves x groups)
// 4.8 / 3.9-5.1 / 4.7-5.1, 512 channels in 1 x 2 / 2 x 1 5.1 / 2.9-4.7, 4096 channels in 8 x 2 / 16 x 1 4.8 / 4.8.
static void block_norm_shape(int width, int& wpr, int& nj) {
    wpr = width <= 1024 ? 1 : width <= 2048 ? 4 : width <= 4096 ? 8 : 16;
    nj = wpr == 1 ? (width + 255) / 256 : width <= 8192 ? 2 : 4;
}

static int block_norm_grid(int rows, int wpr, int cap) {
    const int rpw = wpr == 1 ? 4 : 1;
    const int64_t wgs = ((int64_t)rows + rpw - 1) / rpw;
    return (int)(wgs < cap ? wgs : cap);
}

// workgroups at most (they then take rows in turn): forward 2048 -- 4096 and 1024 are 2 to 6 % slower at 29600 x 768 fp32 --, backward 512, where
// more cost partial rows of column sums and weights that are loaded again (65536 x 512 bf16: 104 us, 125 with 1024)
constexpr int BN_FWD_CAP = 2048, BN_BWD_CAP = 512;

}  // namespace lego

using namespace lego;
#define ST ((hipStream_t)stream)

// one instantiation for the row's shape; widths that are no multiple of 4 take the widest form of their wave count
#define BY_SHAPE(GO, T, MODE)                                                                                                                      \
    do {                                                                                                                                           \
        if (!full) { if (wpr == 1) GO(T, MODE, 1, 4, false); else if (wpr == 4) GO(T, MODE, 4, 2, false);                                           \
                     else if (wpr == 8) GO(T, MODE, 8, 2, false); else GO(T, MODE, 16, 4, false); }                                                 \
        else if (wpr == 1) { if (nj == 1) GO(T, MODE, 1, 1, true); else if (nj == 2) GO(T, MODE, 1, 2, true);                                       \
                             else if (nj == 3) GO(T, MODE, 1, 3, true); else GO(T, MODE, 1, 4, true); }                                             \
        else if (wpr == 4) GO(T, MODE, 4, 2, true);                                                                                                \
        else if (wpr == 8) GO(T, MODE, 8, 2, true);                                                                                                \
        else if (nj == 2) GO(T, MODE, 16, 2, true);                                                                                                \
        else GO(T, MODE, 16, 4, true);                                                                                                             \
    } while (0)
#define BY_MODE(GO, T) do { if (mode == 3) BY_SHAPE(GO, T, 3); else if (mode == BN_BLOCK) BY_SHAPE(GO, T, 1); else BY_SHAPE(GO, T, 2); } while (0)

static int block_norm_check(const char* who, const BlockNorm& p, int dtype, int mode) {
    LEGO_REQUIRE(dtype == LEGO_F32 || dtype == LEGO_BF16 || dtype == LEGO_F16, "%s: unknown dtype %d", who, dtype);
    LEGO_REQUIRE(p.rows >= 0 && p.width > 0 && p.width <= LEGO_BLOCK_NORM_MAX_WIDTH, "%s: bad sizes rows=%d, width=%d (1 .. %d)", who, p.rows, p.width,
                 LEGO_BLOCK_NORM_MAX_WIDTH);
    LEGO_REQUIRE(mode != 0, "%s: neither a block (o) nor a norm after it (next_w)", who);
    LEGO_REQUIRE(p.act >= 0 && p.act <= 2, "%s: unknown activation %d of the gate", who, p.act);
    if (p.rows == 0) return 0;
    LEGO_REQUIRE(p.x.p != nullptr && (!(mode & BN_BLOCK) || (p.post_w && p.scale && (p.act == 0 || p.gate.p))), "%s: NULL operand", who);
    return 0;
}

extern "C" int64_t lego_block_norm_workspace(int rows, int width) {
    if (rows <= 0 || width <= 0) return 0;
    int wpr, nj;
    block_norm_shape(width, wpr, nj);
    return (int64_t)block_norm_grid(rows, wpr, BN_BWD_CAP) * 2 * width;
}

extern "C" int lego_block_norm_fwd(const void* x, int64_t ldx, const void* o, int64_t ldo, const void* gate, int64_t ldg, int dtype, int act,
                                   const float* post_w, const float* scale, const float* next_w, float eps, void* y, void* next, float* stat, int rows,
                                   int width, void* stream) {
    const BlockNorm p{{x, ldx}, {o, ldo}, {gate, ldg}, post_w, scale, next_w, eps, act, rows, width};
    const int mode = (o != nullptr ? BN_BLOCK : 0) | (next_w != nullptr ? BN_NEXT : 0);
    if (int rc = block_norm_check("lego_block_norm_fwd", p, dtype, mode)) return rc;
    if (rows == 0) return 0;
    LEGO_REQUIRE((!(mode & BN_BLOCK) || y) && (!(mode & BN_NEXT) || next), "lego_block_norm_fwd: NULL output");
    int wpr, nj;
    block_norm_shape(width, wpr, nj);
    const bool full = width % 4 == 0;
    const dim3 grid(block_norm_grid(rows, wpr, BN_FWD_CAP)), block(64 * (wpr == 1 ? 4 : wpr));
#define GO(T, M, W, J, F) hipLaunchKernelGGL((block_norm_fwd_kernel<T, M, W, J, F>), grid, block, 0, ST, p, (T*)y, (T*)next, stat)
    LEGO_BY_TYPE(dtype, BY_MODE(GO, T));
#undef GO
    return check_launch("lego_block_norm_fwd");
}

extern "C" int lego_block_norm_bwd(const void* x, int64_t ldx, const void* o, int64_t ldo, const void* gate, int64_t ldg, int dtype, int act,
                                   const float* post_w, const float* scale, const float* next_w, float eps, const void* dy, int64_t lddy,
                                   const void* dn, int64_t lddn, const float* stat, void* dx, void* dout, void* dgate, float* dpost_w, float* dscale,
                                   float* dnext_w, float* workspace, int64_t workspace_floats, int rows, int width, void* stream) {
    const BlockNorm p{{x, ldx}, {o, ldo}, {gate, ldg}, post_w, scale, next_w, eps, act, rows, width};
    const int mode = (o != nullptr ? BN_BLOCK : 0) | (next_w != nullptr ? BN_NEXT : 0);
    if (int rc = block_norm_check("lego_block_norm_bwd", p, dtype, mode)) return rc;
    LEGO_REQUIRE(rows > 0, "lego_block_norm_bwd: no rows: nothing to differentiate");
    LEGO_REQUIRE(stat && dx && ((mode & BN_NEXT) ? dn && dnext_w : dy != nullptr) && (!(mode & BN_BLOCK) || (dout && dpost_w && dscale && (act == 0 || dgate))),
                 "lego_block_norm_bwd: NULL operand");
    LEGO_REQUIRE(workspace != nullptr && workspace_floats >= lego_block_norm_workspace(rows, width),
                 "lego_block_norm_bwd: workspace of %lld floats, lego_block_norm_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_block_norm_workspace(rows, width));
    int wpr, nj;
    block_norm_shape(width, wpr, nj);
    const Rows gy{dy, lddy}, gn{dn, lddn};
    const bool full = width % 4 == 0;
    const int wgs = block_norm_grid(rows, wpr, BN_BWD_CAP);
    const dim3 grid(wgs), block(64 * (wpr == 1 ? 4 : wpr));
#define GO(T, M, W, J, F) hipLaunchKernelGGL((block_norm_bwd_kernel<T, M, W, J, F>), grid, block, 0, ST, p, gy, gn, stat, (T*)dx, (T*)dout, (T*)dgate, workspace)
    LEGO_BY_TYPE(dtype, BY_MODE(GO, T));
#undef GO
    if (int rc = check_launch("lego_block_norm_bwd")) return rc;
    hipLaunchKernelGGL(block_norm_weights_kernel, dim3((width + 15) / 16), dim3(1024), 0, ST, workspace, wgs, mode, post_w, scale, dpost_w, dscale, dnext_w, width);
    return check_launch("lego_block_norm_bwd (weights)");
}
