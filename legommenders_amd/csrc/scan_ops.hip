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
#include <type_traits>

#include "seq_common.hpp"

namespace lego {

// A lane holds SC_VC channels x SC_STEPS steps; SC_LANES lanes span the channels, the other lanes and the waves the tile's steps.
constexpr int SC_VC = 2, SC_STEPS = 4, SC_LANES = 32, SC_WAVES = 8, SC_TILE = LEGO_SCAN_TILE;
constexpr int SC_CH = SC_VC * SC_LANES, SC_GROUPS = 64 / SC_LANES, SC_RUNS = SC_GROUPS * SC_WAVES, SC_THREADS = 64 * SC_WAVES;
static_assert(SC_TILE == SC_STEPS * SC_RUNS, "a tile is SC_RUNS runs of SC_STEPS steps");
using fv = vec<float, SC_VC>;

struct Seq { const void* p; int64_t sn, sl; };                     // [n, length, width] with its strides; channels are contiguous

// softplus to about 1e-7 relative on the hardware exponential and logarithm: ln(1 + t) = ln(u) t / (u - 1) with u = 1 + t rounded takes the
// rounding of u back out; e^v = 2^hi (1 + lo ln 2) keeps the part of v log2(e) that one fp32 number drops
__device__ __forceinline__ float softplus(float v) {
    const float hi = v * 1.44269504088896340736f, lo = __builtin_fmaf(v, 1.44269504088896340736f, -hi) + v * 1.92596299112661746887e-8f;
    const float e = __builtin_amdgcn_exp2f(hi), t = __builtin_fmaf(e, lo * 0.69314718055994530942f, e), u = 1.f + t, d = u - 1.f;
    const float s = d > 0.f ? 0.69314718055994530942f * __builtin_amdgcn_logf(u) * (t * __builtin_amdgcn_rcpf(d)) : t;
    return v > 20.f ? v : s;
}

// l = k sigmoid(r) <= 0, a = e^l, beta = sqrt(1 - a^2) = sqrt((1 - a)(1 + a)), 4 channels.  1 - a would cancel near 1: for l >= -0.5
// (e^l - 1) / l is the degree-5 polynomial through its Chebyshev points there (3e-9 relative), else the hardware exponential.  NEAR: |k| <= 0.5
// for every channel of the wave, so that no l is below -0.5 (decays that start at 0.6 and more -- the usual initialisation is 0.9 to 0.999).
template <bool NEAR>
__device__ __forceinline__ void decay(fv k, fv sr, fv& l, fv& a, fv& beta) {
    fv m;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) {
        l[j] = k[j] * sr[j];
        float s = 0.0011234042467549443f;
        s = __builtin_fmaf(s, l[j], 0.008189613930881023f);
        s = __builtin_fmaf(s, l[j], 0.04163007438182831f);
        s = __builtin_fmaf(s, l[j], 0.16666242480278015f);
        s = __builtin_fmaf(s, l[j], 0.4999998211860657f);
        s = __builtin_fmaf(s, l[j], 1.f);
        m[j] = l[j] * s;
        a[j] = 1.f + m[j];
    }
    if constexpr (!NEAR)
#pragma unroll
        for (int j = 0; j < SC_VC; ++j) {
            const float far = __builtin_amdgcn_exp2f(1.44269504088896340736f * l[j]);
            if (l[j] < -0.5f) { a[j] = far; m[j] = far - 1.f; }
        }
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) beta[j] = __builtin_amdgcn_sqrtf(-m[j] * (1.f + a[j]));
}

__device__ __forceinline__ fv sigmoid_of(fv v) {
    fv s;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) s[j] = sigmoid(v[j]);
    return s;
}

__device__ __forceinline__ bool all_near(fv k) {
    bool near = true;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) near &= k[j] >= -0.5f;
    return __all(near);
}

__device__ __forceinline__ fv shuffle_up(fv v, int lanes) {
    fv s;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) s[j] = __shfl_up(v[j], lanes, 64);
    return s;
}
__device__ __forceinline__ fv shuffle_down(fv v, int lanes) {
    fv s;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) s[j] = __shfl_down(v[j], lanes, 64);
    return s;
}

// -c softplus(lam) of this lane's channels
template <bool FULL>
__device__ __forceinline__ fv rates(const float* __restrict__ lam, float sharpness, int c, int width) {
    const fv v = load<float, SC_VC, FULL>(lam, c, width);
    fv k;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) k[j] = c + j < width ? -sharpness * softplus(v[j]) : 0.f;
    return k;
}

struct Totals { fv a[2][SC_WAVES][SC_LANES], h[2][SC_WAVES][SC_LANES]; };   // two tiles in turn, so that one barrier a tile is enough

// Compose the runs of a tile, first step first.  In: this lane's composition (A, H) and the state before the tile.  Out: the state before this
// lane's steps; `carry` becomes the state after the tile, and `through` (where given) takes the tile's product of decays.
__device__ __forceinline__ fv join_forward(Totals& tot, int buf, int wave, int group, int cl, fv A, fv H, fv& carry, fv* through = nullptr) {
#pragma unroll
    for (int by = 1; by < SC_GROUPS; by <<= 1) {
        const fv pa = shuffle_up(A, SC_LANES * by), ph = shuffle_up(H, SC_LANES * by);
        if (group >= by) { H = A * ph + H; A = A * pa; }
    }
    if (group == SC_GROUPS - 1) { tot.a[buf][wave][cl] = A; tot.h[buf][wave][cl] = H; }
    const fv pa = shuffle_up(A, SC_LANES), ph = shuffle_up(H, SC_LANES);
    __syncthreads();
    fv at = carry;
#pragma unroll 4
    for (int w = 0; w < SC_WAVES; ++w) {
        const fv a = tot.a[buf][w][cl], h = tot.h[buf][w][cl];
        if (w == wave) at = carry;
        carry = a * carry + h;
        if (through != nullptr) *through = a * *through;
    }
    return group == 0 ? at : pa * at + ph;
}

// the same from the last step to the first, of the recurrence C_t = a_t (C_(t+1) + g_t): returns the C of the step behind this lane's last.  The
// barrier is the caller's, between the two halves.
__device__ __forceinline__ void join_backward_put(Totals& tot, int buf, int wave, int group, int cl, fv& A, fv& C, fv& na, fv& nc) {
#pragma unroll
    for (int by = 1; by < SC_GROUPS; by <<= 1) {
        const fv a = shuffle_down(A, SC_LANES * by), c = shuffle_down(C, SC_LANES * by);
        if (group + by < SC_GROUPS) { C = A * c + C; A = A * a; }
    }
    if (group == 0) { tot.a[buf][wave][cl] = A; tot.h[buf][wave][cl] = C; }
    na = shuffle_down(A, SC_LANES), nc = shuffle_down(C, SC_LANES);
}
__device__ __forceinline__ fv join_backward_get(const Totals& tot, int buf, int wave, int group, int cl, fv na, fv nc, fv& carry, fv* through = nullptr) {
    fv at = carry;
#pragma unroll 4
    for (int w = SC_WAVES - 1; w >= 0; --w) {
        const fv a = tot.a[buf][w][cl], c = tot.h[buf][w][cl];
        if (w == wave) at = carry;
        carry = a * carry + c;
        if (through != nullptr) *through = a * *through;
    }
    return group == SC_GROUPS - 1 ? at : na * at + nc;
}

// `carry` through the compositions of `count` chunks from chunk `first` on, in the direction DIR: the SC_RUNS groups of lanes take a run of them each
template <bool FULL, int DIR>
__device__ __forceinline__ void join_chunks(Totals& tot, const float* __restrict__ sums, int first, int count, int wave, int group, int tg, int cl, int c,
                                            int width, fv& carry) {
    fv A(1.f), H(0.f);
    const int run = (count + SC_RUNS - 1) / SC_RUNS, end = min(count, (tg + 1) * run);
#pragma unroll 4
    for (int q = tg * run; q < end; ++q) {
        const float* s = sums + (int64_t)(first + DIR * q) * 2 * width;
        const fv a = load<float, SC_VC, FULL>(s, c, width), h = load<float, SC_VC, FULL>(s + width, c, width);
        H = a * H + h;
        A = A * a;
    }
    join_forward(tot, 0, wave, group, cl, A, H, carry);
    __syncthreads();                                                   // the tiles use the same buffers
}

// N inputs of a sequence, tile by tile: scalar pointers to the tile's head, 32-bit lane offsets into it.
template <typename T, int N, bool FULL>
struct Rows {
    const T* head[N];
    int64_t tile[N];                                                   // elements between tiles
    uint32_t step[N], at[N], idle[N];                                  // bytes: between steps, of this lane's first step, of its channels in the head row
    __device__ __forceinline__ void set(int q, const Seq& s, int64_t n, int first_tile, int t, int c, int width) {
        tile[q] = SC_TILE * s.sl;
        head[q] = (const T*)s.p + n * s.sn + first_tile * tile[q];
        step[q] = (uint32_t)(s.sl * (int)sizeof(T));
        idle[q] = (uint32_t)(min(c, width - (FULL ? SC_VC : 1)) * (int)sizeof(T));       // a lane behind the row reads the row's end
        at[q] = (uint32_t)t * step[q] + idle[q];
    }
    __device__ __forceinline__ void move(int tiles) {
#pragma unroll
        for (int q = 0; q < N; ++q) head[q] += tiles * tile[q];
    }
};

// A lane's steps of N inputs as they lie in memory.  Every load is issued, without a branch between them (the compiler then knows how many are in
// flight, and a tile's wait leaves the next tile's loads alone); what is not live reads the tile's head row again, which costs no traffic.
template <typename T, int N, bool FULL>
struct Steps {
    vec<T, SC_VC> v[N][SC_STEPS];
    uint32_t live;                                                     // bit s: step s exists and is not masked
    // t: this lane's first step in the tile, left: steps from the tile's head to the end (at least 1), mask: of the tile's head
    __device__ __forceinline__ void fetch(const Rows<T, N, FULL>& rows, const uint8_t* __restrict__ mask, int t, int left, int c, int width) {
        live = 0;
#pragma unroll
        for (int s = 0; s < SC_STEPS; ++s) live |= (t + s < left ? 1u : 0u) << s;
        if (mask != nullptr) {
            uint8_t m[SC_STEPS];
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) m[s] = mask[(uint32_t)min(t + s, left - 1)];
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) live &= ~((m[s] == 0 ? 1u : 0u) << s);
        }
#pragma unroll
        for (int s = 0; s < SC_STEPS; ++s)
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const uint32_t at = live >> s & 1u ? rows.at[q] + s * rows.step[q] : rows.idle[q];
                const char* p = reinterpret_cast<const char*>(rows.head[q]) + at;
                if constexpr (FULL) __builtin_memcpy(&v[q][s], p, sizeof(v[q][s]));
                else
#pragma unroll
                    for (int k = 0; k < SC_VC; ++k) v[q][s][k] = *reinterpret_cast<const T*>(p + (c + k < width ? k * (int)sizeof(T) : 0));
            }
    }
    __device__ __forceinline__ fv at(int q, int s) const { return __builtin_convertvector(v[q][s], fv); }
    // hides from the compiler that the values are still the same: what is cheap to form from them is formed again, not kept in registers
    __device__ __forceinline__ void renew() {
        using Bits = typename std::conditional<SC_VC * sizeof(T) == 4, uint32_t, uint64_t>::type;
#pragma unroll
        for (int q = 0; q < N; ++q)
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) {
                Bits b = __builtin_bit_cast(Bits, v[q][s]);
                asm volatile("" : "+v"(b));
                v[q][s] = __builtin_bit_cast(decltype(v[q][s] + v[q][s]), b);
            }
    }
};

constexpr int ONE_TILE = 0, TILES = 1, SUMMARY = 2;                    // sequences of one tile need no next one fetched ahead

// the byte offset of step t, channel c in a tile of a contiguous output
template <typename T>
__device__ __forceinline__ uint32_t lane_offset(int t, int width, int c) { return (uint32_t)((t * width + c) * (int)sizeof(T)); }

// a and b of a lane's steps; a step that is not live is a = 1, b = 0 whatever was read for it
template <bool NEAR, typename In>
__device__ __forceinline__ void gates_forward(const In& in, fv k, fv (&a)[SC_STEPS], fv (&b)[SC_STEPS]) {
#pragma unroll
    for (int s = 0; s < SC_STEPS; ++s) {
        fv l, beta;
        decay<NEAR>(k, sigmoid_of(in.at(1, s)), l, a[s], beta);
        b[s] = beta * (sigmoid_of(in.at(2, s)) * in.at(0, s));
        const bool live = in.live >> s & 1u;
#pragma unroll
        for (int j = 0; j < SC_VC; ++j) { a[s][j] = live ? a[s][j] : 1.f; b[s][j] = live ? b[s][j] : 0.f; }
    }
}

// One workgroup: channels [64 blockIdx.x, + 64) of sequence blockIdx.y, tiles [chunk * per, + per).  The next tile's loads are in flight
// while a tile is computed.  SUMMARY: only the chunk's composition goes to `sums` [n, chunks, 2, width].
template <typename T, bool FULL, int MODE>
__global__ __launch_bounds__(SC_THREADS, 4) void scan_fwd_kernel(Seq x, Seq r, Seq i, const float* __restrict__ lam, float sharpness,
                                                                 const uint8_t* __restrict__ mask, int64_t mask_sn, const float* __restrict__ state,
                                                                 T* __restrict__ h, float* __restrict__ last, float* __restrict__ tiles,
                                                                 float* __restrict__ sums, int length, int width, int chunks, int per) {
    __shared__ Totals tot;
    const int cl = threadIdx.x & (SC_LANES - 1), tg = threadIdx.x / SC_LANES, group = tg & (SC_GROUPS - 1);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int c = blockIdx.x * SC_CH + SC_VC * cl, chunk = blockIdx.z, t = tg * SC_STEPS;
    const int64_t n = blockIdx.y;
    const int n_tiles = (length + SC_TILE - 1) / SC_TILE, t_begin = chunk * per, t_end = min(n_tiles, t_begin + per);
    if (t_begin >= t_end) return;
    Rows<T, 3, FULL> rows;
    rows.set(0, x, n, t_begin, t, c, width);
    rows.set(1, r, n, t_begin, t, c, width);
    rows.set(2, i, n, t_begin, t, c, width);
    const uint8_t* m = mask != nullptr ? mask + n * mask_sn + t_begin * SC_TILE : nullptr;
    int left = length - t_begin * SC_TILE;
    Steps<T, 3, FULL> in, ahead;
    in.fetch(rows, m, t, left, c, width);
    const fv k = rates<FULL>(lam, sharpness, c, width), zero(0.f);
    const bool near = all_near(k);
    const uint32_t at_h = lane_offset<T>(t, width, c);
    fv carry(0.f), through(1.f);
    if constexpr (MODE != SUMMARY) {
        if (state != nullptr) carry = load<float, SC_VC, FULL>(state + n * width, c, width);
        if (MODE == TILES && chunk > 0) join_chunks<FULL, 1>(tot, sums + n * chunks * 2 * width, 0, chunk, wave, group, tg, cl, c, width, carry);
    }
    for (int tile = t_begin; tile < t_end; ++tile, left -= SC_TILE) {
        if (MODE != ONE_TILE && tile + 1 < t_end) {
            rows.move(1);
            if (m != nullptr) m += SC_TILE;
            ahead.fetch(rows, m, t, left - SC_TILE, c, width);
        }
        fv a[SC_STEPS], b[SC_STEPS], A(1.f), H(0.f);
        if (__any(in.live != 0)) {
            if (near) gates_forward<true>(in, k, a, b);
            else gates_forward<false>(in, k, a, b);
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) {
                H = a[s] * H + b[s];
                A = A * a[s];
            }
        }
        if constexpr (MODE == SUMMARY) join_forward(tot, tile & 1, wave, group, cl, A, H, carry, &through);
        else {
            if (tiles != nullptr && tg == 0) store<float, SC_VC, FULL>(tiles + (n * n_tiles + tile) * width, c, width, carry);
            fv now = join_forward(tot, tile & 1, wave, group, cl, A, H, carry);
            T* head = h + (n * length + (int64_t)tile * SC_TILE) * width;
#pragma unroll
            for (int s = 0; s < SC_STEPS; ++s) {
                fv out = zero;
                if (in.live >> s & 1u) out = now = a[s] * now + b[s];
                if (t + s < left) store_at<T, SC_VC, FULL>(head + s * width, at_h, c, width, out);
            }
        }
        if constexpr (MODE != ONE_TILE) in = ahead;
    }
    if (tg == 0) {
        if constexpr (MODE == SUMMARY) {
            float* s = sums + ((n * chunks + chunk) * 2) * width;
            store<float, SC_VC, FULL>(s, c, width, through);
            store<float, SC_VC, FULL>(s + width, c, width, carry);
        } else if (t_end == n_tiles) store<float, SC_VC, FULL>(last + n * width, c, width, carry);
    }
}

template <bool NEAR, bool ALL, typename In>
__device__ __forceinline__ void gates_backward(const In& in, fv k, fv (&sr)[SC_STEPS], fv (&si)[SC_STEPS], fv (&a)[SC_STEPS], fv (&beta)[SC_STEPS]) {
#pragma unroll
    for (int s = 0; s < SC_STEPS; ++s) {
        fv l;
        sr[s] = sigmoid_of(in.at(0, s));
        decay<NEAR>(k, sr[s], l, a[s], beta[s]);
        if constexpr (ALL) si[s] = sigmoid_of(in.at(3, s));
        const bool live = in.live >> s & 1u;
#pragma unroll
        for (int j = 0; j < SC_VC; ++j) a[s][j] = live ? a[s][j] : 1.f;
    }
}

// Backward.  C_t = a_t G_t is what step t hands to step t - 1: C_t = a_t (C_(t+1) + dh_t), G_t = dh_t + C_(t+1).
//   SUMMARY: the chunk's composition of the C recurrence (reads r and dh only)
template <typename T, bool FULL, int MODE>
__global__ __launch_bounds__(SC_THREADS, 4) void scan_bwd_kernel(Seq x, Seq r, Seq i, Seq gh, const float* __restrict__ lam, float sharpness,
                                                                 const uint8_t* __restrict__ mask, int64_t mask_sn, const float* __restrict__ tiles,
                                                                 const float* __restrict__ glast, T* __restrict__ dx, T* __restrict__ dr,
                                                                 T* __restrict__ di, float* __restrict__ dstate, float* __restrict__ qsum,
                                                                 float* __restrict__ sums, int seqs, int length, int width, int chunks, int per) {
    __shared__ Totals tot, fwd;
    __shared__ fv fold[SC_RUNS][SC_LANES];
    constexpr int N = MODE == SUMMARY ? 2 : 4;
    constexpr bool AHEAD = MODE == SUMMARY;                            // four inputs leave no registers for a second tile
    const int cl = threadIdx.x & (SC_LANES - 1), tg = threadIdx.x / SC_LANES, group = tg & (SC_GROUPS - 1);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int c = blockIdx.x * SC_CH + SC_VC * cl, chunk = blockIdx.z, t = tg * SC_STEPS;
    const int n_tiles = (length + SC_TILE - 1) / SC_TILE, t_begin = chunk * per, t_end = min(n_tiles, t_begin + per);
    const fv k = rates<FULL>(lam, sharpness, c, width), zero(0.f);
    const bool near = all_near(k);
    const uint32_t at_d = lane_offset<T>(t, width, c);
    fv q_all(0.f);
    int buf = 0;
    for (int64_t n = blockIdx.y; n < seqs && t_begin < t_end; n += gridDim.y) {
        Rows<T, N, FULL> rows;
        rows.set(0, r, n, t_end - 1, t, c, width);
        rows.set(1, gh, n, t_end - 1, t, c, width);
        if constexpr (MODE != SUMMARY) {
            rows.set(2, x, n, t_end - 1, t, c, width);
            rows.set(3, i, n, t_end - 1, t, c, width);
        }
        const uint8_t* m = mask != nullptr ? mask + n * mask_sn + (t_end - 1) * SC_TILE : nullptr;
        int left = length - (t_end - 1) * SC_TILE;
        Steps<T, N, FULL> in, ahead;
        in.fetch(rows, m, t, left, c, width);
        fv carry(0.f), through(1.f);
        if constexpr (MODE != SUMMARY) {
            if (glast != nullptr) carry = load<float, SC_VC, FULL>(glast + n * width, c, width);
            if (MODE == TILES && chunk < chunks - 1)
                join_chunks<FULL, -1>(tot, sums + n * chunks * 2 * width, chunks - 1, chunks - 1 - chunk, wave, group, tg, cl, c, width, carry);
        }
        for (int tile = t_end - 1; tile >= t_begin; --tile, buf ^= 1, left += SC_TILE) {
            fv head(0.f);
            if constexpr (MODE != SUMMARY) head = load<float, SC_VC, FULL>(tiles + (n * n_tiles + tile) * width, c, width);
            if (MODE != ONE_TILE && tile > t_begin) {
                rows.move(-1);
                if (m != nullptr) m -= SC_TILE;
                if constexpr (AHEAD) ahead.fetch(rows, m, t, left + SC_TILE, c, width);
            }
            fv sr[SC_STEPS], si[SC_STEPS], a[SC_STEPS], beta[SC_STEPS], A(1.f), H(0.f), C(0.f);
            if (__any(in.live != 0)) {
                if (near) gates_backward<true, MODE != SUMMARY>(in, k, sr, si, a, beta);
                else gates_backward<false, MODE != SUMMARY>(in, k, sr, si, a, beta);
#pragma unroll
                for (int s = 0; s < SC_STEPS; ++s) {
                    if constexpr (MODE != SUMMARY)
                        if (in.live >> s & 1u) H = a[s] * H + beta[s] * (si[s] * in.at(2, s));
                    A = A * a[s];
                }
#pragma unroll
                for (int s = SC_STEPS - 1; s >= 0; --s)
                    if (in.live >> s & 1u) C = a[s] * (C + in.at(1, s));
            }
            fv Ar = A, na, nc, now(0.f);
            join_backward_put(tot, buf, wave, group, cl, Ar, C, na, nc);
            if constexpr (MODE != SUMMARY) now = join_forward(fwd, buf, wave, group, cl, A, H, head);     // its barrier covers `tot` too
            else __syncthreads();
            fv back = join_backward_get(tot, buf, wave, group, cl, na, nc, carry, MODE == SUMMARY ? &through : nullptr);
            if constexpr (MODE != SUMMARY) {
                const int64_t row = (n * length + (int64_t)tile * SC_TILE) * width;
                in.renew();
#pragma unroll
                for (int s = 0; s < SC_STEPS; ++s) asm volatile("" : "+v"(sr[s]), "+v"(si[s]), "+v"(beta[s]));
                fv before[SC_STEPS];
#pragma unroll
                for (int s = 0; s < SC_STEPS; ++s) {
                    before[s] = now;
                    if (in.live >> s & 1u) now = a[s] * now + beta[s] * (si[s] * in.at(2, s));
                }
#pragma unroll
                for (int s = SC_STEPS - 1; s >= 0; --s) {
                    if (t + s >= left) continue;
                    fv vx = zero, vr = zero, vi = zero;
                    if (in.live >> s & 1u) {
                        const fv G = in.at(1, s) + back, xs = in.at(2, s);
                        back = a[s] * G;
#pragma unroll
                        for (int j = 0; j < SC_VC; ++j) {
                            const float l = k[j] * sr[s][j], bv = beta[s][j], u = si[s][j] * xs[j];
                            // l / beta tends to 0 with l (as -sqrt(-l / 2)): where beta has become 0, so has l
                            const float lb = bv > 0.f ? l * __builtin_amdgcn_rcpf(bv) : 0.f;
                            const float q = back[j] * (before[s][j] * l - u * a[s][j] * lb), du = G[j] * bv;
                            q_all[j] += q;
                            vx[j] = du * si[s][j];
                            vr[j] = q * (1.f - sr[s][j]);
                            vi[j] = du * u * (1.f - si[s][j]);
                        }
                    }
                    store_at<T, SC_VC, FULL>(dx + row + s * width, at_d, c, width, vx);
                    store_at<T, SC_VC, FULL>(dr + row + s * width, at_d, c, width, vr);
                    store_at<T, SC_VC, FULL>(di + row + s * width, at_d, c, width, vi);
                }
            }
            if constexpr (AHEAD) in = ahead;
            else if (MODE != ONE_TILE && tile > t_begin) in.fetch(rows, m, t, left + SC_TILE, c, width);
        }
        if (tg == 0) {
            if constexpr (MODE == SUMMARY) {
                float* s = sums + ((n * chunks + chunk) * 2) * width;
                store<float, SC_VC, FULL>(s, c, width, through);
                store<float, SC_VC, FULL>(s + width, c, width, carry);
            } else if (chunk == 0 && dstate != nullptr) store<float, SC_VC, FULL>(dstate + n * width, c, width, carry);
        }
    }
    if constexpr (MODE != SUMMARY) {                                   // this workgroup's part of sum q, in a fixed order
        fold[tg][cl] = q_all;
        __syncthreads();
        if (tg == 0) {
            fv s = fold[0][cl];
#pragma unroll
            for (int w = 1; w < SC_RUNS; ++w) s += fold[w][cl];
            store<float, SC_VC, FULL>(qsum + ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * width, c, width, s);
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

// one step for n states: SC_VC channels a thread, every input read once
template <typename T, bool FULL>
__global__ __launch_bounds__(256) void scan_step_kernel(Seq x, Seq r, Seq i, const float* __restrict__ lam, float sharpness,
                                                        const uint8_t* __restrict__ mask, const float* __restrict__ state, T* __restrict__ h,
                                                        float* __restrict__ next, int seqs, int width) {
    const int groups = (width + SC_VC - 1) / SC_VC;
    for (int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; at < (int64_t)seqs * groups; at += (int64_t)gridDim.x * blockDim.x) {
        const int64_t n = at / groups;
        const int c = SC_VC * (int)(at - n * groups);
        fv now = load<float, SC_VC, FULL>(state + n * width, c, width), out(0.f);
        if (mask == nullptr || mask[n] != 0) {
            const fv xs = load<T, SC_VC, FULL>((const T*)x.p + n * x.sn, c, width), rs = load<T, SC_VC, FULL>((const T*)r.p + n * r.sn, c, width),
                        is = load<T, SC_VC, FULL>((const T*)i.p + n * i.sn, c, width), k = rates<FULL>(lam, sharpness, c, width);
            fv l, a, beta;
            decay<false>(k, sigmoid_of(rs), l, a, beta);
            now = a * now + beta * (sigmoid_of(is) * xs);
            out = now;
        }
        store<T, SC_VC, FULL>(h + n * width, c, width, out);
        store<float, SC_VC, FULL>(next + n * width, c, width, now);
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

static int scan_strides(const char* who, int64_t a, int64_t b, int64_t c, int64_t d) {
    const int64_t most = 1 << 24;                                      // a tile's 64 steps of 4 bytes fit a 32-bit offset
    LEGO_REQUIRE(a >= 0 && b >= 0 && c >= 0 && d >= 0 && a < most && b < most && c < most && d < most,
                 "%s: strides between steps have to be below %lld elements", who, (long long)most);
    return 0;
}

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
    if (int rc = scan_strides("lego_gated_scan_fwd", x_sl, r_sl, i_sl, 0)) return rc;
    const ScanPlan p = scan_plan(n, length, width);
    LEGO_REQUIRE(p.chunks == 1 || (workspace != nullptr && workspace_floats >= lego_gated_scan_workspace(n, length, width)),
                 "lego_gated_scan_fwd: workspace of %lld floats, lego_gated_scan_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_gated_scan_workspace(n, length, width));
    const Seq sx{x, x_sn, x_sl}, sr{r, r_sn, r_sl}, si{i, i_sn, i_sl};
    const bool full = width % SC_VC == 0;
    const dim3 grid(p.slices, n, p.chunks);
#define GO(F, MODE) hipLaunchKernelGGL((scan_fwd_kernel<T, F, MODE>), grid, dim3(SC_THREADS), 0, ST, sx, sr, si, lam, sharpness, mask, mask_sn, state, \
                                       (T*)h, last, tiles, workspace, length, width, p.chunks, p.per)
    LEGO_BY_TYPE(dtype, {
        if (p.chunks > 1) { if (full) GO(true, SUMMARY); else GO(false, SUMMARY); }
        if (p.tiles > 1) { if (full) GO(true, TILES); else GO(false, TILES); }
        else if (full) GO(true, ONE_TILE); else GO(false, ONE_TILE);
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
    if (int rc = scan_strides("lego_gated_scan_bwd", x_sl, r_sl, i_sl, gh_sl)) return rc;
    const ScanPlan p = scan_plan(n, length, width);
    LEGO_REQUIRE(workspace != nullptr && workspace_floats >= lego_gated_scan_workspace(n, length, width),
                 "lego_gated_scan_bwd: workspace of %lld floats, lego_gated_scan_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_gated_scan_workspace(n, length, width));
    const Seq sx{x, x_sn, x_sl}, sr{r, r_sn, r_sl}, si{i, i_sn, i_sl}, sg{gh, gh_sn, gh_sl};
    const bool full = width % SC_VC == 0;
    float* qsum = workspace;
    float* sums = workspace + (int64_t)p.rows * p.chunks * width;
    const dim3 all(p.slices, n, p.chunks), grid(p.slices, p.rows, p.chunks);
#define GO(F, MODE, GRID) hipLaunchKernelGGL((scan_bwd_kernel<T, F, MODE>), GRID, dim3(SC_THREADS), 0, ST, sx, sr, si, sg, lam, sharpness, mask, mask_sn, \
                                             tiles, glast, (T*)dx, (T*)dr, (T*)di, dstate, qsum, sums, n, length, width, p.chunks, p.per)
    LEGO_BY_TYPE(dtype, {
        if (p.chunks > 1) { if (full) GO(true, SUMMARY, all); else GO(false, SUMMARY, all); }
        if (p.tiles > 1) { if (full) GO(true, TILES, grid); else GO(false, TILES, grid); }
        else if (full) GO(true, ONE_TILE, grid); else GO(false, ONE_TILE, grid);
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
    const bool full = width % SC_VC == 0;
    const int64_t wgs = ((int64_t)n * ((width + SC_VC - 1) / SC_VC) + 255) / 256;
    const dim3 grid((unsigned)(wgs < 4096 ? wgs : 4096));
#define GO(F) hipLaunchKernelGGL((scan_step_kernel<T, F>), grid, dim3(256), 0, ST, sx, sr, si, lam, sharpness, mask, state, (T*)h, next, n, width)
    LEGO_BY_TYPE(dtype, { if (full) GO(true); else GO(false); });
#undef GO
    return check_launch("lego_gated_scan_step");
}
