// Gated linear recurrence over sequences, its backward pass and its single step (include/lego_hip.h: lego_gated_scan_*).
//
//   l_t = -c softplus(lam) sigmoid(r_t)      a_t = e^l_t      b_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t       h_t = a_t h_(t-1) + b_t
//
// Steps compose: (A2, H2) after (A1, H1) is (A2 A1, A2 H1 + H2).  A workgroup owns 64 channels of one sequence and walks it in tiles of 64
// steps: a lane holds 4 channels x 4 steps in registers, composes them, the 4 groups of a wave join by shuffles, the 4 waves through LDS
// (one barrier a tile), and each lane then replays its 4 steps from the state that reaches it -- every input is read once.  Few sequences
// that are long are cut into chunks: a first launch composes each chunk, the second starts every chunk from the chunks before it.
//
// The backward pass keeps no h: the forward pass saves the fp32 state at the head of every tile (1/64 of the cells), the tile's states are
// formed again from it in fp32, and G_t = dh_t + a_(t+1) G_(t+1) is the same composition from the other end.
#include "seq_common.hpp"

namespace lego {

constexpr int SC_TILE = LEGO_SCAN_TILE, SC_STEPS = 4, SC_CH = 64, SC_THREADS = 256;      // 16 time groups x 16 channel lanes
static_assert(SC_TILE == SC_STEPS * (SC_THREADS / 16), "a tile is 16 groups of SC_STEPS steps");

struct Seq { const void* p; int64_t sn, sl; };                     // [n, length, width] with its strides; channels are contiguous

// 1 - e^l for l <= 0: the series where 1 - e^l would cancel (truncation 0.5^8 / 9! = 1e-8 of the value), else the exponential
__device__ __forceinline__ float one_minus_exp(float l, float& e) {
    float s = 1.f / 40320.f;
    s = __builtin_fmaf(s, l, 1.f / 5040.f);
    s = __builtin_fmaf(s, l, 1.f / 720.f);
    s = __builtin_fmaf(s, l, 1.f / 120.f);
    s = __builtin_fmaf(s, l, 1.f / 24.f);
    s = __builtin_fmaf(s, l, 1.f / 6.f);
    s = __builtin_fmaf(s, l, 0.5f);
    s = __builtin_fmaf(s, l, 1.f);
    const float near = -l * s, far = __builtin_amdgcn_exp2f(1.44269504088896340736f * l);
    const bool small = l > -0.5f;
    e = small ? 1.f - near : far;
    return small ? near : 1.f - far;
}

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }

// l = k sigmoid(r), a = e^l, beta = sqrt(1 - a^2) = sqrt((1 - a)(1 + a))
__device__ __forceinline__ void decay(float k, float sr, float& l, float& a, float& beta) {
    l = k * sr;
    const float p = one_minus_exp(l, a);
    beta = __builtin_amdgcn_sqrtf(p * (1.f + a));
}

__device__ __forceinline__ f32x4 shuffle_up(f32x4 v, int by) {
    return f32x4{__shfl_up(v[0], by, 64), __shfl_up(v[1], by, 64), __shfl_up(v[2], by, 64), __shfl_up(v[3], by, 64)};
}
__device__ __forceinline__ f32x4 shuffle_down(f32x4 v, int by) {
    return f32x4{__shfl_down(v[0], by, 64), __shfl_down(v[1], by, 64), __shfl_down(v[2], by, 64), __shfl_down(v[3], by, 64)};
}

// -c softplus(lam) of this lane's channels
__device__ __forceinline__ f32x4 rates(const float* __restrict__ lam, float sharpness, int c, int width) {
    f32x4 k;
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = c + j < width ? -sharpness * softplus(lam[c + j]) : 0.f;
    return k;
}

struct Totals { f32x4 a[2][4][16], h[2][4][16]; };                 // two tiles in turn, so that one barrier a tile is enough

// Compose the 16 time groups of a tile, first step first.  In: this lane's composition (A, H) and the state before the tile.  Out: the
// state before this lane's steps; `carry` becomes the state after the tile.
__device__ __forceinline__ f32x4 join_forward(Totals& tot, int buf, int wave, int group, int cl, f32x4 A, f32x4 H, f32x4& carry) {
#pragma unroll
    for (int by = 1; by < 4; by <<= 1) {
        const f32x4 pa = shuffle_up(A, 16 * by), ph = shuffle_up(H, 16 * by);
        if (group >= by) { H = A * ph + H; A = A * pa; }
    }
    if (group == 3) { tot.a[buf][wave][cl] = A; tot.h[buf][wave][cl] = H; }
    const f32x4 pa = shuffle_up(A, 16), ph = shuffle_up(H, 16);
    __syncthreads();
    f32x4 at = carry;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w == wave) at = carry;
        carry = tot.a[buf][w][cl] * carry + tot.h[buf][w][cl];
    }
    return group == 0 ? at : pa * at + ph;
}

// One workgroup: channels [64 blockIdx.x, + 64) of sequence blockIdx.y, tiles [chunk * per, + per).
//   SUMMARY: only the chunk's composition goes to `sums` [n, chunks, 2, width]
template <typename T, bool ALIGNED, bool SUMMARY>
__global__ __launch_bounds__(SC_THREADS) void scan_fwd_kernel(Seq x, Seq r, Seq i, const float* __restrict__ lam, float sharpness,
                                                              const uint8_t* __restrict__ mask, int64_t mask_sn, const float* __restrict__ state,
                                                              T* __restrict__ h, float* __restrict__ last, float* __restrict__ tiles,
                                                              float* __restrict__ sums, int length, int width, int chunks, int per) {
    __shared__ Totals tot;
    const int cl = threadIdx.x & 15, tg = threadIdx.x >> 4, group = tg & 3, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int c = blockIdx.x * SC_CH + 4 * cl, chunk = blockIdx.z;
    const int64_t n = blockIdx.y;
    const int n_tiles = (length + SC_TILE - 1) / SC_TILE, t_end = min(n_tiles, (chunk + 1) * per);
    const T *xp = (const T*)x.p + n * x.sn, *rp = (const T*)r.p + n * r.sn, *ip = (const T*)i.p + n * i.sn;
    const f32x4 k = rates(lam, sharpness, c, width);
    f32x4 carry{0.f, 0.f, 0.f, 0.f}, through{1.f, 1.f, 1.f, 1.f};
    if constexpr (!SUMMARY) {
        if (state != nullptr) carry = load4<float, ALIGNED>(state + n * width, c, width);
        for (int q = 0; q < chunk; ++q) {
            const float* s = sums + ((n * chunks + q) * 2) * width;
            carry = load4<float, ALIGNED>(s, c, width) * carry + load4<float, ALIGNED>(s + width, c, width);
        }
    }
    for (int tile = chunk * per; tile < t_end; ++tile) {
        f32x4 xs[SC_STEPS], rs[SC_STEPS], is[SC_STEPS], a[SC_STEPS], b[SC_STEPS];
        bool live[SC_STEPS];
        const int t0 = tile * SC_TILE + tg * SC_STEPS;
#pragma unroll
        for (int s = 0; s < SC_STEPS; ++s) live[s] = t0 + s < length && (mask == nullptr || mask[n * mask_sn + t0 + s] != 0);
#pragma unroll
        for (int s = 0; s < SC_STEPS; ++s) {
            if (!live[s]) continue;
            xs[s] = load4<T, ALIGNED>(xp + (t0 + s) * x.sl, c, width);
            rs[s] = load4<T, ALIGNED>(rp + (t0 + s) * r.sl, c, width);
            is[s] = load4<T, ALIGNED>(ip + (t0 + s) * i.sl, c, width);
        }
        f32x4 A{1.f, 1.f, 1.f, 1.f}, H{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < SC_STEPS; ++s) {
            a[s] = f32x4{1.f, 1.f, 1.f, 1.f};
            b[s] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (live[s])
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float l, av, beta;
                    decay(k[j], sigmoid(rs[s][j]), l, av, beta);
                    a[s][j] = av;
                    b[s][j] = beta * (sigmoid(is[s][j]) * xs[s][j]);
                }
            H = a[s] * H + b[s];
            A = A * a[s];
        }
        if (!SUMMARY && tiles != nullptr && tg == 0) store4<float, ALIGNED>(tiles + (n * n_tiles + tile) * width, c, width, carry);
        if constexpr (SUMMARY) {
            f32x4 unit = through;                                     // the product of the decays rides along as a recurrence without inputs
            f32x4 now = join_forward(tot, tile & 1, wave, group, cl, A, H, carry);
            (void)now;
#pragma unroll
            for (int w = 0; w < 4; ++w) unit = tot.a[tile & 1][w][cl] * unit;
            through = unit;
        } else {
            f32x4 now = join_forward(tot, tile & 1, wave, group, cl, A, H, carry);
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) {
                now = a[s] * now + b[s];
                if (t0 + s < length) store4<T, ALIGNED>(h + (n * length + t0 + s) * (int64_t)width, c, width, live[s] ? now : f32x4{0.f, 0.f, 0.f, 0.f});
            }
        }
    }
    if (tg == 0) {
        if constexpr (SUMMARY) {
            float* s = sums + ((n * chunks + chunk) * 2) * width;
            store4<float, ALIGNED>(s, c, width, through);
            store4<float, ALIGNED>(s + width, c, width, carry);
        } else if (t_end == n_tiles) store4<float, ALIGNED>(last + n * width, c, width, carry);
    }
}

// Backward.  C_t = a_t G_t is what step t hands to step t - 1: C_t = a_t C_(t+1) + a_t dh_t, G_t = dh_t + C_(t+1).
//   SUMMARY: the chunk's composition of the C recurrence (reads r and dh only)
template <typename T, bool ALIGNED, bool SUMMARY>
__global__ __launch_bounds__(SC_THREADS) void scan_bwd_kernel(Seq x, Seq r, Seq i, Seq gh, const float* __restrict__ lam, float sharpness,
                                                              const uint8_t* __restrict__ mask, int64_t mask_sn, const float* __restrict__ tiles,
                                                              const float* __restrict__ glast, T* __restrict__ dx, T* __restrict__ dr,
                                                              T* __restrict__ di, float* __restrict__ dstate, float* __restrict__ qsum,
                                                              float* __restrict__ sums, int seqs, int length, int width, int chunks, int per) {
    __shared__ Totals tot, fwd;
    __shared__ f32x4 fold[16][16];
    const int cl = threadIdx.x & 15, tg = threadIdx.x >> 4, group = tg & 3, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int c = blockIdx.x * SC_CH + 4 * cl, chunk = blockIdx.z;
    const int n_tiles = (length + SC_TILE - 1) / SC_TILE, t_end = min(n_tiles, (chunk + 1) * per);
    const f32x4 k = rates(lam, sharpness, c, width), zero{0.f, 0.f, 0.f, 0.f};
    f32x4 q_all = zero;
    int buf = 0;
    for (int64_t n = blockIdx.y; n < seqs; n += gridDim.y) {
        const T *xp = (const T*)x.p + n * x.sn, *rp = (const T*)r.p + n * r.sn, *ip = (const T*)i.p + n * i.sn, *gp = (const T*)gh.p + n * gh.sn;
        f32x4 carry = zero, through{1.f, 1.f, 1.f, 1.f};
        if constexpr (!SUMMARY) {
            if (glast != nullptr) carry = load4<float, ALIGNED>(glast + n * width, c, width);
            for (int q = chunks - 1; q > chunk; --q) {
                const float* s = sums + ((n * chunks + q) * 2) * width;
                carry = load4<float, ALIGNED>(s, c, width) * carry + load4<float, ALIGNED>(s + width, c, width);
            }
        }
        for (int tile = t_end - 1; tile >= chunk * per; --tile, buf ^= 1) {
            f32x4 xs[SC_STEPS], sr[SC_STEPS], si[SC_STEPS], g[SC_STEPS], a[SC_STEPS], beta[SC_STEPS];
            bool live[SC_STEPS];
            const int t0 = tile * SC_TILE + tg * SC_STEPS;
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) live[s] = t0 + s < length && (mask == nullptr || mask[n * mask_sn + t0 + s] != 0);
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) {
                xs[s] = sr[s] = si[s] = g[s] = zero;
                if (!live[s]) continue;
                sr[s] = load4<T, ALIGNED>(rp + (t0 + s) * r.sl, c, width);
                g[s] = load4<T, ALIGNED>(gp + (t0 + s) * gh.sl, c, width);
                if constexpr (!SUMMARY) {
                    xs[s] = load4<T, ALIGNED>(xp + (t0 + s) * x.sl, c, width);
                    si[s] = load4<T, ALIGNED>(ip + (t0 + s) * i.sl, c, width);
                }
            }
            f32x4 head = zero;
            if constexpr (!SUMMARY) head = load4<float, ALIGNED>(tiles + (n * n_tiles + tile) * width, c, width);
            f32x4 A{1.f, 1.f, 1.f, 1.f}, H = zero, C = zero;
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) {
                a[s] = f32x4{1.f, 1.f, 1.f, 1.f};
                beta[s] = zero;
                if (live[s])
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float l, av, bv;
                        sr[s][j] = sigmoid(sr[s][j]);
                        decay(k[j], sr[s][j], l, av, bv);
                        a[s][j] = av;
                        beta[s][j] = bv;
                        if constexpr (!SUMMARY) si[s][j] = sigmoid(si[s][j]);
                    }
                A = A * a[s];
                if constexpr (!SUMMARY) H = a[s] * H + beta[s] * (si[s] * xs[s]);
            }
#pragma unroll
            for (int s = SC_STEPS - 1; s >= 0; --s) C = a[s] * (C + g[s]);
            // join from the last group to the first: (A, C) of the steps from this group on to the end of the wave
            f32x4 Ar = A;
#pragma unroll
            for (int by = 1; by < 4; by <<= 1) {
                const f32x4 na = shuffle_down(Ar, 16 * by), nc = shuffle_down(C, 16 * by);
                if (group + by < 4) { C = Ar * nc + C; Ar = Ar * na; }
            }
            if (group == 0) { tot.a[buf][wave][cl] = Ar; tot.h[buf][wave][cl] = C; }
            const f32x4 na = shuffle_down(Ar, 16), nc = shuffle_down(C, 16);
            f32x4 now = zero;
            if constexpr (!SUMMARY) now = join_forward(fwd, buf, wave, group, cl, A, H, head);     // its barrier covers `tot` too
            else __syncthreads();
            f32x4 at = carry;
#pragma unroll
            for (int w = 3; w >= 0; --w) {
                if (w == wave) at = carry;
                carry = tot.a[buf][w][cl] * carry + tot.h[buf][w][cl];
                if constexpr (SUMMARY) through = tot.a[buf][w][cl] * through;
            }
            if constexpr (!SUMMARY) {
                f32x4 back = group == 3 ? at : na * at + nc;                                        // C of the step after this lane's last
                f32x4 before[SC_STEPS];
#pragma unroll
                for (int s = 0; s < SC_STEPS; ++s) {
                    before[s] = now;
                    now = a[s] * now + beta[s] * (si[s] * xs[s]);
                }
#pragma unroll
                for (int s = SC_STEPS - 1; s >= 0; --s) {
                    const f32x4 G = g[s] + back;
                    back = a[s] * G;
                    if (t0 + s >= length) continue;
                    f32x4 vx = zero, vr = zero, vi = zero;
                    if (live[s])
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float l = k[j] * sr[s][j], bv = beta[s][j], u = si[s][j] * xs[s][j];
                            // l / beta tends to 0 with l (as -sqrt(-l / 2)): where beta has become 0, so has l
                            const float lb = bv > 0.f ? l * __builtin_amdgcn_rcpf(bv) : 0.f;
                            const float q = G[j] * a[s][j] * (before[s][j] * l - u * a[s][j] * lb), du = G[j] * bv;
                            q_all[j] += q;
                            vx[j] = du * si[s][j];
                            vr[j] = q * (1.f - sr[s][j]);
                            vi[j] = du * u * (1.f - si[s][j]);
                        }
                    const int64_t at_row = (n * length + t0 + s) * (int64_t)width;
                    store4<T, ALIGNED>(dx + at_row, c, width, vx);
                    store4<T, ALIGNED>(dr + at_row, c, width, vr);
                    store4<T, ALIGNED>(di + at_row, c, width, vi);
                }
            }
        }
        if (tg == 0) {
            if constexpr (SUMMARY) {
                float* s = sums + ((n * chunks + chunk) * 2) * width;
                store4<float, ALIGNED>(s, c, width, through);
                store4<float, ALIGNED>(s + width, c, width, carry);
            } else if (chunk == 0 && dstate != nullptr) store4<float, ALIGNED>(dstate + n * width, c, width, carry);
        }
    }
    if constexpr (!SUMMARY) {                                          // this workgroup's part of sum q, in a fixed order
        fold[tg][cl] = q_all;
        __syncthreads();
        if (tg == 0) {
            f32x4 s = fold[0][cl];
#pragma unroll
            for (int w = 1; w < 16; ++w) s += fold[w][cl];
            store4<float, ALIGNED>(qsum + ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * width, c, width, s);
        }
    }
}

// dlam = sum q sigmoid(lam) / softplus(lam): `parts` rows of partial sums, 16 columns x 16 row lanes a workgroup, fixed order
__global__ __launch_bounds__(256) void scan_dlam_kernel(const float* __restrict__ qsum, int parts, const float* __restrict__ lam, float* __restrict__ dlam,
                                                        int width) {
    __shared__ float red[16][17];
    const int col = threadIdx.x & 15, lane = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
    float s = 0.f;
    if (c < width)
        for (int p = lane; p < parts; p += 16) s += qsum[(int64_t)p * width + c];
    red[lane][col] = s;
    __syncthreads();
    if (lane == 0 && c < width) {
#pragma unroll
        for (int w = 1; w < 16; ++w) s += red[w][col];
        const float v = lam[c], sp = softplus(v);
        // sigmoid / softplus -> 1 - e^lam / 2 for lam -> -inf, where both underflow together
        dlam[c] = s * (v < -15.f ? 1.f : 1.f / ((1.f + expf(-v)) * sp));
    }
}

// one step for n states: 4 channels a thread, every input read once
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void scan_step_kernel(Seq x, Seq r, Seq i, const float* __restrict__ lam, float sharpness,
                                                        const uint8_t* __restrict__ mask, const float* __restrict__ state, T* __restrict__ h,
                                                        float* __restrict__ next, int seqs, int width) {
    const int groups = (width + 3) / 4;
    for (int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; at < (int64_t)seqs * groups; at += (int64_t)gridDim.x * blockDim.x) {
        const int64_t n = at / groups;
        const int c = 4 * (int)(at - n * groups);
        f32x4 now = load4<float, ALIGNED>(state + n * width, c, width), out{0.f, 0.f, 0.f, 0.f};
        if (mask == nullptr || mask[n] != 0) {
            const f32x4 xs = load4<T, ALIGNED>((const T*)x.p + n * x.sn, c, width), rs = load4<T, ALIGNED>((const T*)r.p + n * r.sn, c, width),
                        is = load4<T, ALIGNED>((const T*)i.p + n * i.sn, c, width), k = rates(lam, sharpness, c, width);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float l, a, beta;
                decay(k[j], sigmoid(rs[j]), l, a, beta);
                now[j] = a * now[j] + beta * (sigmoid(is[j]) * xs[j]);
            }
            out = now;
        }
        store4<T, ALIGNED>(h + n * width, c, width, out);
        store4<float, ALIGNED>(next + n * width, c, width, now);
    }
}

struct ScanPlan { int slices, tiles, chunks, per, rows; };

// chunks of a sequence and workgroup rows of the backward pass: one workgroup a (sequence, 64 channels) fills the 256 CUs from about 512
// workgroups on; below that long sequences are cut until about 1024 are in flight, at least 2 tiles each
static ScanPlan scan_plan(int n, int length, int width) {
    ScanPlan p;
    p.slices = (width + SC_CH - 1) / SC_CH;
    p.tiles = (length + SC_TILE - 1) / SC_TILE;
    const int64_t wgs = (int64_t)n * p.slices;
    p.chunks = 1;
    if (wgs < 512 && p.tiles >= 4) {
        const int64_t want = (1024 + wgs - 1) / wgs;
        p.chunks = (int)(want < p.tiles / 2 ? want : p.tiles / 2);
    }
    p.per = p.tiles > 0 ? (p.tiles + p.chunks - 1) / p.chunks : 1;
    p.chunks = p.tiles > 0 ? (p.tiles + p.per - 1) / p.per : 1;
    const int cap = 2048 / p.slices > 0 ? 2048 / p.slices : 1;         // partial rows of sum q
    p.rows = n < cap ? n : cap;
    return p;
}

}  // namespace lego

using namespace lego;
#define ST ((hipStream_t)stream)

static int scan_sizes(const char* who, int dtype, int n, int length, int width) {
    LEGO_REQUIRE(dtype == LEGO_F32 || dtype == LEGO_BF16 || dtype == LEGO_F16, "%s: unknown dtype %d", who, dtype);
    LEGO_REQUIRE(n >= 0 && n <= 65535 && length >= 0 && width >= 0 && length <= (1 << 30) && width <= (1 << 20),
                 "%s: bad sizes n=%d (at most 65535), length=%d, width=%d", who, n, length, width);
    return 0;
}

extern "C" int64_t lego_gated_scan_workspace(int n, int length, int width) {
    if (n <= 0 || length <= 0 || width <= 0) return 0;
    const ScanPlan p = scan_plan(n, length, width);
    return (p.chunks > 1 ? 2 * (int64_t)n * p.chunks * width : 0) + (int64_t)p.rows * p.chunks * width;
}

extern "C" int lego_gated_scan_fwd(const void* x, int64_t x_sn, int64_t x_sl, const void* r, int64_t r_sn, int64_t r_sl, const void* i, int64_t i_sn,
                                   int64_t i_sl, int dtype, const float* lam, float sharpness, const uint8_t* mask, int64_t mask_sn,
                                   const float* state, void* h, float* last, float* tiles, float* workspace, int64_t workspace_floats, int n,
                                   int length, int width, void* stream) {
    if (int rc = scan_sizes("lego_gated_scan_fwd", dtype, n, length, width)) return rc;
    if (n == 0 || width == 0) return 0;
    LEGO_REQUIRE(length > 0, "lego_gated_scan_fwd: length 0 (the state is the answer)");
    LEGO_REQUIRE(x && r && i && lam && h && last, "lego_gated_scan_fwd: NULL operand");
    const ScanPlan p = scan_plan(n, length, width);
    LEGO_REQUIRE(p.chunks == 1 || (workspace != nullptr && workspace_floats >= lego_gated_scan_workspace(n, length, width)),
                 "lego_gated_scan_fwd: workspace of %lld floats, lego_gated_scan_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_gated_scan_workspace(n, length, width));
    const Seq sx{x, x_sn, x_sl}, sr{r, r_sn, r_sl}, si{i, i_sn, i_sl};
    const bool al = width % 4 == 0 && (x_sn | x_sl | r_sn | r_sl | i_sn | i_sl) % 4 == 0 && aligned4(x, dtype) && aligned4(r, dtype) && aligned4(i, dtype) &&
                    aligned4(h, dtype) && aligned4(state, LEGO_F32) && aligned4(last, LEGO_F32) && aligned4(tiles, LEGO_F32) && aligned4(workspace, LEGO_F32);
    const dim3 grid(p.slices, n, p.chunks);
#define GO(AL, SUM) hipLaunchKernelGGL((scan_fwd_kernel<T, AL, SUM>), grid, dim3(SC_THREADS), 0, ST, sx, sr, si, lam, sharpness, mask, mask_sn, state, \
                                       (T*)h, last, tiles, workspace, length, width, p.chunks, p.per)
    LEGO_BY_TYPE(dtype, {
        if (p.chunks > 1) { if (al) GO(true, true); else GO(false, true); }
        if (al) GO(true, false); else GO(false, false);
    });
#undef GO
    return check_launch("lego_gated_scan_fwd");
}

extern "C" int lego_gated_scan_bwd(const void* x, int64_t x_sn, int64_t x_sl, const void* r, int64_t r_sn, int64_t r_sl, const void* i, int64_t i_sn,
                                   int64_t i_sl, const void* gh, int64_t gh_sn, int64_t gh_sl, int dtype, const float* lam, float sharpness,
                                   const uint8_t* mask, int64_t mask_sn, const float* tiles, const float* glast, void* dx, void* dr, void* di,
                                   float* dlam, float* dstate, float* workspace, int64_t workspace_floats, int n, int length, int width, void* stream) {
    if (int rc = scan_sizes("lego_gated_scan_bwd", dtype, n, length, width)) return rc;
    LEGO_REQUIRE(n > 0 && length > 0, "lego_gated_scan_bwd: n=%d, length=%d: nothing to differentiate", n, length);
    if (width == 0) return 0;
    LEGO_REQUIRE(x && r && i && gh && lam && tiles && dx && dr && di && dlam, "lego_gated_scan_bwd: NULL operand");
    const ScanPlan p = scan_plan(n, length, width);
    LEGO_REQUIRE(workspace != nullptr && workspace_floats >= lego_gated_scan_workspace(n, length, width),
                 "lego_gated_scan_bwd: workspace of %lld floats, lego_gated_scan_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_gated_scan_workspace(n, length, width));
    const Seq sx{x, x_sn, x_sl}, sr{r, r_sn, r_sl}, si{i, i_sn, i_sl}, sg{gh, gh_sn, gh_sl};
    const bool al = width % 4 == 0 && (x_sn | x_sl | r_sn | r_sl | i_sn | i_sl | gh_sn | gh_sl) % 4 == 0 && aligned4(x, dtype) && aligned4(r, dtype) &&
                    aligned4(i, dtype) && aligned4(gh, dtype) && aligned4(dx, dtype) && aligned4(dr, dtype) && aligned4(di, dtype) &&
                    aligned4(tiles, LEGO_F32) && aligned4(glast, LEGO_F32) && aligned4(dstate, LEGO_F32) && aligned4(workspace, LEGO_F32);
    float* qsum = workspace;
    float* sums = workspace + (int64_t)p.rows * p.chunks * width;
    const dim3 all(p.slices, n, p.chunks), grid(p.slices, p.rows, p.chunks);
#define GO(AL, SUM, GRID) hipLaunchKernelGGL((scan_bwd_kernel<T, AL, SUM>), GRID, dim3(SC_THREADS), 0, ST, sx, sr, si, sg, lam, sharpness, mask, mask_sn, \
                                             tiles, glast, (T*)dx, (T*)dr, (T*)di, dstate, qsum, sums, n, length, width, p.chunks, p.per)
    LEGO_BY_TYPE(dtype, {
        if (p.chunks > 1) { if (al) GO(true, true, all); else GO(false, true, all); }
        if (al) GO(true, false, grid); else GO(false, false, grid);
    });
#undef GO
    if (int rc = check_launch("lego_gated_scan_bwd")) return rc;
    hipLaunchKernelGGL(scan_dlam_kernel, dim3((width + 15) / 16), dim3(256), 0, ST, qsum, p.rows * p.chunks, lam, dlam, width);
    return check_launch("lego_gated_scan_bwd (dlam)");
}

extern "C" int lego_gated_scan_step(const void* x, int64_t x_sn, const void* r, int64_t r_sn, const void* i, int64_t i_sn, int dtype, const float* lam,
                                    float sharpness, const uint8_t* mask, const float* state, void* h, float* next, int n, int width, void* stream) {
    LEGO_REQUIRE(dtype == LEGO_F32 || dtype == LEGO_BF16 || dtype == LEGO_F16, "lego_gated_scan_step: unknown dtype %d", dtype);
    LEGO_REQUIRE(n >= 0 && width >= 0 && width <= (1 << 20), "lego_gated_scan_step: bad sizes n=%d, width=%d", n, width);
    if (n == 0 || width == 0) return 0;
    LEGO_REQUIRE(x && r && i && lam && state && h && next, "lego_gated_scan_step: NULL operand");
    const Seq sx{x, x_sn, 0}, sr{r, r_sn, 0}, si{i, i_sn, 0};
    const bool al = width % 4 == 0 && (x_sn | r_sn | i_sn) % 4 == 0 && aligned4(x, dtype) && aligned4(r, dtype) && aligned4(i, dtype) &&
                    aligned4(h, dtype) && aligned4(state, LEGO_F32) && aligned4(next, LEGO_F32);
    const int64_t wgs = ((int64_t)n * ((width + 3) / 4) + 255) / 256;
    const dim3 grid((unsigned)(wgs < 4096 ? wgs : 4096));
#define GO(AL) hipLaunchKernelGGL((scan_step_kernel<T, AL>), grid, dim3(256), 0, ST, sx, sr, si, lam, sharpness, mask, state, (T*)h, next, n, width)
    LEGO_BY_TYPE(dtype, { if (al) GO(true); else GO(false); });
#undef GO
    return check_launch("lego_gated_scan_step");
}
