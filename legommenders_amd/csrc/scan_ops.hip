// Gated linear recurrence over sequences, its backward pass and its single step (include/lego_hip.h: lego_gated_scan_*).
//
//   l_t = -c softplus(lam) sigmoid(r_t)      a_t = e^l_t      b_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t       h_t = a_t h_(t-1) + b_t
//
// Steps compose: (A2, H2) after (A1, H1) is (A2 A1, A2 H1 + H2).  A workgroup owns 64 channels of one sequence and walks it in tiles of 64
// steps: a lane holds 2 channels x a few steps in registers and composes them, the two halves of a wave join by a shuffle, the waves through LDS
// (one barrier a tile), and each lane then replays its steps from the state that reaches it -- every input is read once.  Few sequences
// that are long are cut into chunks: a first launch composes each chunk, the second starts every chunk from the chunks before it.
//
// The backward pass keeps no h: the forward pass saves the fp32 state at the head of every tile (1/64 of the cells), the tile's states are
// formed again from it in fp32, and G_t = dh_t + a_(t+1) G_(t+1) is the same composition from the other end.
//
// What bounds it: in fp32 memory (64 x 2048 x 256: forward 114 us, 4.7 TB/s; backward 214 us, 4.4 TB/s); in 16 bits, with half the bytes, the vector
// units (the same cells: forward 65 us, backward 155; a copy of their bytes 54 and 94; forward 50 instructions a cell, 5 of them transcendental, backward two more
// of those).  Cut into chunks, 2 x 32768 x 768 bf16: forward 160 us, backward 225 (one call after another; 180 and 252 after other work has taken the
// cache).  512 x 50 x 256 fp32 with ragged lengths, a tile a workgroup, most of whose waves have no live step: 17 us forward of 12, 38 backward of 24.
#include <float.h>

#include <type_traits>

#include "seq_common.hpp"

namespace lego {

// A lane holds SC_VC channels x STEPS steps; SC_LANES lanes span the channels, the other lanes and the waves the tile's runs of STEPS steps.
constexpr int SC_VC = 2, SC_LANES = 32, SC_TILE = LEGO_SCAN_TILE, SC_CH = SC_VC * SC_LANES, SC_GROUPS = 64 / SC_LANES;
template <int WAVES_, int STEPS_> struct Shape {
    static constexpr int WAVES = WAVES_, STEPS = STEPS_, RUNS = SC_GROUPS * WAVES, THREADS = 64 * WAVES;
    static_assert(STEPS * RUNS == SC_TILE && SC_VC == 2, "a tile is RUNS runs of STEPS steps");
};
// (This and what follows was compared before rest_of's exponential, which adds 2 to 7 % to every backward form alike; scan_plan's table is with it.)
// Measured (us): forward 8 x 4 / 4 x 8, 64 x 2048 x 256 fp32 115 / 117, 1 x 10007 x 301 fp16 42 / 48; backward, which has the registers of 16 cells a
// lane only in workgroups of 4 waves, 512 x 50 x 256 fp32 84 / 54, 64 x 2048 x 256 fp32 231 / 211.
using Fwd = Shape<8, 4>;
using Bwd = Shape<4, 8>;
using fv = vec<float, SC_VC>;

struct Seq { const void* p; int64_t sn, sl; };                     // [n, length, width] with its strides; channels are contiguous

// softplus to about 1e-7 relative on the hardware exponential and logarithm: ln(1 + t) = ln(u) t / (u - 1) with u = 1 + t rounded takes the
// rounding of u back out; e^v = 2^hi (1 + lo ln 2) keeps the part of v log2(e) that one fp32 number drops.  Below -104 it is 0 in fp32 (for v = -inf the
// two parts would be inf - inf)
__device__ __forceinline__ float softplus(float v) {
    const float hi = v * 1.44269504088896340736f, lo = __builtin_fmaf(v, 1.44269504088896340736f, -hi) + v * 1.92596299112661746887e-8f;
    const float e = __builtin_amdgcn_exp2f(hi), t = __builtin_fmaf(e, lo * 0.69314718055994530942f, e), u = 1.f + t, d = u - 1.f;
    const float s = d > 0.f ? 0.69314718055994530942f * __builtin_amdgcn_logf(u) * (t * __builtin_amdgcn_rcpf(d)) : t;
    return v > 20.f ? v : v < -104.f ? 0.f : s;
}

// l = k sigmoid(r) <= 0, a = e^l, beta = sqrt(1 - a^2) = sqrt((1 - a)(1 + a)), 2 channels.  1 - a would cancel near 1: for l >= -0.5
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
    for (int j = 0; j < SC_VC; ++j) beta[j] = __builtin_amdgcn_sqrtf(__builtin_fmaf(-m[j], a[j], -m[j]));
}

__device__ __forceinline__ fv sigmoid_of(fv v) {
    fv s;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) s[j] = sigmoid(v[j]);
    return s;
}

// 1 - s of s = sigmoid(v) as e^-v s: its bits are there for open gates too, where the difference has lost them.  (From v = -88 on s is 0, and so is what
// is multiplied by this; the argument is kept below where e^-v overflows, for no 0 * inf.)  What the exponential costs, us: 64 x 2048 x 256 fp32
// 210 -> 214, bf16 147 -> 157, 2 x 32768 x 768 bf16 217 -> 226.  The plain difference for waves in which no gate is open far enough to matter
// in 16 bits was slower than both, 169 and 240: the branch parts loads from arithmetic.
__device__ __forceinline__ fv rest_of(fv v, fv s) {
    fv o;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) o[j] = __builtin_amdgcn_exp2f(fminf(-1.44269504088896340736f * v[j], 126.f)) * s[j];
    return o;
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

// -c softplus(lam) of this lane's channels; finite where it overflows, so that a gate that is shut (sigmoid 0: every step that is not live) decays by 1
template <bool FULL>
__device__ __forceinline__ fv rates(const float* __restrict__ lam, float sharpness, int c, int width) {
    const fv v = load<float, SC_VC, FULL>(lam, c, width);
    fv k;
#pragma unroll
    for (int j = 0; j < SC_VC; ++j) {
        const float q = -sharpness * softplus(v[j]);
        k[j] = c + j < width ? (q < -FLT_MAX ? -FLT_MAX : q) : 0.f;    // (NaN stays NaN)
    }
    return k;
}

// where a lane is: channels [c, + SC_VC), steps [t, + STEPS) of a tile, which is run `run` of it
template <typename S> struct Lane {
    int cl = threadIdx.x & (SC_LANES - 1), run = threadIdx.x / SC_LANES, group = run & (SC_GROUPS - 1);
    int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), c = blockIdx.x * SC_CH + SC_VC * cl, t = run * S::STEPS;
    __device__ __forceinline__ Lane() {}
};

template <typename S> struct Totals { fv a[2][S::WAVES][SC_LANES], h[2][S::WAVES][SC_LANES]; };      // two tiles in turn: one barrier a tile is enough

// A tile's runs, in the order DIR (1: from the first run, -1: from the last).  put: this lane's (A, H), a barrier; then before: the state that enters this
// lane's run, if `carry` enters the tile -- it moves on to what leaves it -- or past, for a chunk's composition (through, carry).  The waves pass on a
// state, two multiply-adds each; composing them as the lanes are composed took 64 instructions more a tile, of 400 (64 x 2048 x 256 bf16 forward 87
// -> 79 us, 2 x 32768 x 768 177 -> 170).
template <typename S, int DIR>
struct Join {
    fv pa, ph;                                                         // the composition of the wave's runs before this lane's
    static __device__ __forceinline__ fv shifted(fv v, int groups) { return DIR > 0 ? shuffle_up(v, SC_LANES * groups) : shuffle_down(v, SC_LANES * groups); }
    __device__ __forceinline__ void put(Totals<S>& tot, int buf, const Lane<S>& at, fv A, fv H) {
        const int place = DIR > 0 ? at.group : SC_GROUPS - 1 - at.group;
#pragma unroll
        for (int by = 1; by < SC_GROUPS; by <<= 1) {
            const fv a = shifted(A, by), h = shifted(H, by);
            if (place >= by) { H = A * h + H; A = A * a; }
        }
        if (place == SC_GROUPS - 1) { tot.a[buf][at.wave][at.cl] = A; tot.h[buf][at.wave][at.cl] = H; }
        pa = shifted(A, 1), ph = shifted(H, 1);
        if (place == 0) { pa = fv(1.f); ph = fv(0.f); }
    }
    __device__ __forceinline__ fv before(const Totals<S>& tot, int buf, const Lane<S>& at, fv& carry) const {
        fv mine = carry;
#pragma unroll
        for (int q = 0; q < S::WAVES; ++q) {
            const int w = DIR > 0 ? q : S::WAVES - 1 - q;
            if (w == at.wave) mine = carry;
            carry = tot.a[buf][w][at.cl] * carry + tot.h[buf][w][at.cl];
        }
        return pa * mine + ph;
    }
    static __device__ __forceinline__ void past(const Totals<S>& tot, int buf, const Lane<S>& at, fv& through, fv& carry) {
#pragma unroll
        for (int q = 0; q < S::WAVES; ++q) {
            const int w = DIR > 0 ? q : S::WAVES - 1 - q;
            const fv a = tot.a[buf][w][at.cl];
            carry = a * carry + tot.h[buf][w][at.cl];
            through = a * through;
        }
    }
};

// Widths.  Two channels are one load each way: in a row of odd width the last lane loads the last two and takes the second (1 x 10007 x 301 fp16, forward +
// backward: 110 us with an element a load, 70 so, in chunks of two tiles).
enum Width { EVEN, ODD, SINGLE };

// N inputs of a sequence, tile by tile: scalar pointers to the tile's head, 32-bit lane offsets into it.
template <typename T, int N, Width W>
struct Rows {
    const T* head[N];
    int64_t tile[N];                                                   // elements between tiles
    uint32_t step[N], at[N], idle[N];                                  // bytes: between steps, of this lane's first step, of its channels in the head row
    __device__ __forceinline__ void set(int q, const Seq& s, int64_t n, int first_tile, int t, int c, int width) {
        tile[q] = SC_TILE * s.sl;
        head[q] = (const T*)s.p + n * s.sn + first_tile * tile[q];
        step[q] = (uint32_t)(s.sl * (int)sizeof(T));
        idle[q] = (uint32_t)(min(c, width - (W == SINGLE ? 1 : SC_VC)) * (int)sizeof(T));       // a lane behind the row reads the row's end
        at[q] = (uint32_t)t * step[q] + idle[q];
    }
    __device__ __forceinline__ void move(int tiles) {
#pragma unroll
        for (int q = 0; q < N; ++q) head[q] += tiles * tile[q];
    }
};

// A lane's steps of N inputs as they lie in memory.  Every load is issued, without a branch between them (the compiler then knows how many are in
// flight, and a tile's wait leaves the next tile's loads alone); what is not live reads the tile's head row again, which costs no traffic.
template <typename T, int N, int STEPS, Width W>
struct Steps {
    using Pair = vec<T, SC_VC>;
    using Bits = typename std::conditional<sizeof(Pair) == 4, uint32_t, uint64_t>::type;
    Pair v[N][STEPS];
    uint32_t live;                                                     // bit s: step s exists and is not masked (looked at where !whole only)
    bool whole;                                                        // every step of the wave is live
    bool second;                                                       // (ODD) of what was loaded, only the second is a channel of this lane
    static __device__ __forceinline__ void one(Pair& to, const char* p) { __builtin_memcpy(&to, p, (W == SINGLE ? 1 : SC_VC) * sizeof(T)); }
    // t: this lane's first step in the tile, left: steps from the tile's head to the end (at least 1), mask: of the tile's head
    __device__ __forceinline__ void fetch(const Rows<T, N, W>& rows, const uint8_t* __restrict__ mask, int t, int left, int c, int width) {
        second = c + 1 == width;
        if (mask == nullptr && left >= SC_TILE) {                      // all live: one lane offset an input, the steps in the scalar address
            whole = true;
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int q = 0; q < N; ++q) one(v[q][s], reinterpret_cast<const char*>(rows.head[q]) + s * (uint64_t)rows.step[q] + rows.at[q]);
            return;
        }
        live = 0;
        whole = false;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) live |= (t + s < left ? 1u : 0u) << s;
        if (mask != nullptr) {
            uint8_t m[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) m[s] = mask[(uint32_t)min(t + s, left - 1)];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) live &= ~((m[s] == 0 ? 1u : 0u) << s);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const uint32_t at = live >> s & 1u ? rows.at[q] + s * rows.step[q] : rows.idle[q];
                one(v[q][s], reinterpret_cast<const char*>(rows.head[q]) + at);
            }
        whole = __all(live == (1u << STEPS) - 1u);                     // (of this wave's steps: then nothing has to be cleaned)
    }
    __device__ __forceinline__ fv at(int q, int s) const { return __builtin_convertvector(v[q][s], fv); }
    // A step that is not live: the recurrence gate's logit R becomes -inf -- sigmoid 0, decay 1, beta 0 exactly -- and the other inputs 0, so that
    // nothing after this asks again whether a step is live, but for what is written
    template <int R>
    // (64 x 2048 x 256 bf16 with a mask: 92 us with selects of single channels and every tile of a mask cleaned, 77 so)
    __device__ __forceinline__ void clean() {
        if constexpr (W == ODD)
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const Bits b = __builtin_bit_cast(Bits, v[q][s]);
                    v[q][s] = __builtin_bit_cast(Pair, second ? b >> 8 * sizeof(T) : b);
                }
        if (whole) return;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const bool on = live >> s & 1u;
#pragma unroll
            for (int q = 0; q < N; ++q)                                // both channels at once
                v[q][s] = __builtin_bit_cast(Pair, on ? __builtin_bit_cast(Bits, v[q][s]) : q == R ? __builtin_bit_cast(Bits, Pair((T)-INFINITY)) : (Bits)0);
        }
    }
    __device__ __forceinline__ fv kept(int s, fv f) const {            // what is written, or summed over steps
        return whole || (live >> s & 1u) ? f : fv(0.f);
    }
    // hides from the compiler that the values are still the same: what is cheap to form from them is formed again, not kept in registers
    __device__ __forceinline__ void renew() {
#pragma unroll
        for (int q = 0; q < N; ++q)
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                Bits b = __builtin_bit_cast(Bits, v[q][s]);
                asm volatile("" : "+v"(b));
                v[q][s] = __builtin_bit_cast(Pair, b);
            }
    }
};

// A sequence's chunks of tiles, each with its composition [2, width] in `sums`: the state that enters after `count` chunks from `first` on, in the order
// DIR, if `edge` enters the first.  The runs of a workgroup share the chunks out.
template <bool FULL, int DIR, typename S>
__device__ __forceinline__ fv entering(Totals<S>& tot, const float* __restrict__ sums, int first, int count, fv edge, const Lane<S>& at, int width) {
    fv A(1.f), H(0.f);
    const int each = (count + S::RUNS - 1) / S::RUNS, end = min(count, (at.run + 1) * each);
#pragma unroll 4
    for (int q = at.run * each; q < end; ++q) {
        const float* s = sums + (int64_t)(first + DIR * q) * 2 * width;
        const fv a = load<float, SC_VC, FULL>(s, at.c, width), h = load<float, SC_VC, FULL>(s + width, at.c, width);
        H = a * H + h;
        A = A * a;
    }
    Join<S, 1> j;
    j.put(tot, 1, at, A, H);                                           // (the first tile uses the other half)
    __syncthreads();
    j.before(tot, 1, at, edge);
    return edge;
}

// the byte offset of step t, channel c in a tile of a contiguous output
template <typename T>
__device__ __forceinline__ uint32_t lane_offset(int t, int width, int c) { return (uint32_t)((t * width + c) * (int)sizeof(T)); }

// a and b of a lane's steps
template <bool NEAR, int STEPS, typename In>
__device__ __forceinline__ void gates_forward(const In& in, fv k, fv (&a)[STEPS], fv (&b)[STEPS]) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        fv l, beta;
        decay<NEAR>(k, sigmoid_of(in.at(1, s)), l, a[s], beta);
        b[s] = beta * (sigmoid_of(in.at(2, s)) * in.at(0, s));
    }
}

// a, b of a lane's steps and their composition; false if the wave has none that is live
template <typename In, int STEPS>
__device__ __forceinline__ bool compose(In& in, bool near, fv k, fv (&a)[STEPS], fv (&b)[STEPS], fv& A, fv& H) {
    A = fv(1.f), H = fv(0.f);
    if (!in.whole && !__any(in.live != 0)) return false;               // (a wave past the end of its sequence has nothing to do)
    in.template clean<1>();
    if (near) gates_forward<true>(in, k, a, b);
    else gates_forward<false>(in, k, a, b);
    A = a[0], H = b[0];
#pragma unroll
    for (int s = 1; s < STEPS; ++s) {
        H = a[s] * H + b[s];
        A = A * a[s];
    }
    return true;
}

// h of a lane's steps from the state before them
template <typename T, bool FULL, int STEPS>
__device__ __forceinline__ void replay(bool whole, uint32_t live, bool some, const fv (&a)[STEPS], const fv (&b)[STEPS], fv now, T* head, uint32_t at_h, int t,
                                       int left, int c, int width) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (some) now = a[s] * now + b[s];
        if (whole || t + s < left) store_at<T, SC_VC, FULL>(head + s * width, at_h, c, width, whole || (live >> s & 1u) ? now : fv(0.f));
    }
}

// Workgroup: channels [64 blockIdx.x, + 64) of sequence blockIdx.y, tiles [per blockIdx.z, + per) one after the other; the next tile's loads are in flight
// while a tile is computed.  ONE: sequences of one tile, which need no registers for a next one.  SUM: only the chunk's composition, to `sums`
// [n, chunks, 2, width]; chunks after the first start from those.
enum class Pass { ONE, TILES, SUM };
template <typename T, Width W, Pass PASS>
__global__ __launch_bounds__(Fwd::THREADS, 4) void scan_fwd_kernel(Seq x, Seq r, Seq i, const float* __restrict__ lam, float sharpness,
                                                                   const uint8_t* __restrict__ mask, int64_t mask_sn, const float* __restrict__ state,
                                                                   T* __restrict__ h, float* __restrict__ last, float* __restrict__ tiles,
                                                                   float* __restrict__ sums, int length, int width, int per) {
    using S = Fwd;
    constexpr bool FULL = W == EVEN;
    __shared__ Totals<S> tot;
    const Lane<S> at;
    const int64_t n = blockIdx.y;
    const int c = at.c, t = at.t, n_tiles = PASS == Pass::ONE ? 1 : (length + SC_TILE - 1) / SC_TILE;
    const int first = PASS == Pass::ONE ? 0 : blockIdx.z * per, end = min(n_tiles, first + per);        // (every chunk has a tile)
    Rows<T, 3, W> rows;
    rows.set(0, x, n, first, t, c, width);
    rows.set(1, r, n, first, t, c, width);
    rows.set(2, i, n, first, t, c, width);
    if (mask != nullptr) mask += n * mask_sn;
    Steps<T, 3, S::STEPS, W> in, ahead;
    in.fetch(rows, mask != nullptr ? mask + (int64_t)first * SC_TILE : nullptr, t, length - first * SC_TILE, c, width);
    const fv k = rates<FULL>(lam, sharpness, c, width);
    const bool near = all_near(k);
    const uint32_t at_h = lane_offset<T>(t, width, c);
    fv carry(0.f), through(1.f);
    if (PASS != Pass::SUM && state != nullptr) carry = load<float, SC_VC, FULL>(state + n * width, c, width);
    if (PASS == Pass::TILES && blockIdx.z > 0) carry = entering<FULL, 1>(tot, sums + n * gridDim.z * 2 * width, 0, blockIdx.z, carry, at, width);
    for (int tile = first, buf = 0;; ++tile, buf ^= 1) {
        const int left = length - tile * SC_TILE;
        if (PASS != Pass::ONE && tile + 1 < end) {
            rows.move(1);
            ahead.fetch(rows, mask != nullptr ? mask + (int64_t)(tile + 1) * SC_TILE : nullptr, t, left - SC_TILE, c, width);
        }
        fv a[S::STEPS], b[S::STEPS], A, H;
        const bool some = compose(in, near, k, a, b, A, H);
        Join<S, 1> j;
        j.put(tot, buf, at, A, H);
        __syncthreads();
        if constexpr (PASS == Pass::SUM) j.past(tot, buf, at, through, carry);
        else {
            if (tiles != nullptr && at.run == 0) store<float, SC_VC, FULL>(tiles + (n * n_tiles + tile) * width, c, width, carry);
            replay<T, FULL>(in.whole, in.live, some, a, b, j.before(tot, buf, at, carry), h + (n * length + (int64_t)tile * SC_TILE) * width, at_h, t, left, c, width);
        }
        if (PASS == Pass::ONE || tile + 1 == end) break;
        in = ahead;
    }
    if (at.run != 0) return;
    if constexpr (PASS == Pass::SUM) {
        float* s = sums + (n * gridDim.z + blockIdx.z) * 2 * width;
        store<float, SC_VC, FULL>(s, c, width, through);
        store<float, SC_VC, FULL>(s + width, c, width, carry);
    } else if (end == n_tiles) store<float, SC_VC, FULL>(last + n * width, c, width, carry);
}

template <bool NEAR, int STEPS, typename In>
__device__ __forceinline__ void gates_backward(const In& in, fv k, fv (&sr)[STEPS], fv (&si)[STEPS], fv (&a)[STEPS], fv (&beta)[STEPS]) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        fv l;
        sr[s] = sigmoid_of(in.at(0, s));
        decay<NEAR>(k, sr[s], l, a[s], beta[s]);
        si[s] = sigmoid_of(in.at(3, s));
    }
}

// Backward.  C_t = a_t G_t is what step t hands to step t - 1: C_t = a_t (C_(t+1) + dh_t), G_t = dh_t + C_(t+1).  Tiles from the last to the first.
// inputs of `in`: 0 r, 1 dh, 2 x, 3 i
template <typename In, int STEPS>
__device__ __forceinline__ bool compose_both(In& in, bool near, fv k, fv (&sr)[STEPS], fv (&si)[STEPS], fv (&a)[STEPS], fv (&beta)[STEPS], fv& A, fv& H,
                                             fv& C) {
    A = fv(1.f), H = fv(0.f), C = fv(0.f);
    if (!in.whole && !__any(in.live != 0)) return false;
    in.template clean<0>();
    if (near) gates_backward<true>(in, k, sr, si, a, beta);
    else gates_backward<false>(in, k, sr, si, a, beta);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        H = a[s] * H + beta[s] * (si[s] * in.at(2, s));
        A = A * a[s];
    }
#pragma unroll
    for (int s = STEPS - 1; s >= 0; --s) C = a[s] * (C + in.at(1, s));
    return true;
}

template <typename T> struct Grads { T *dx, *dr, *di; };
template <typename T> Grads<T> grads(void* dx, void* dr, void* di) { return {(T*)dx, (T*)dr, (T*)di}; }

// the gradients of a lane's steps: `now` the state before them, `back` the C of the step behind them
template <typename T, bool FULL, typename In, int STEPS>
__device__ __forceinline__ void gradients(In& in, bool some, fv k, fv (&sr)[STEPS], fv (&si)[STEPS], fv (&a)[STEPS], fv (&beta)[STEPS], fv now, fv back,
                                          fv& q_all, Grads<T> d, int64_t row, uint32_t at_d, int t, int left, int c, int width) {
    if (some) {
        in.renew();
#pragma unroll
        for (int s = 0; s < STEPS; ++s) asm volatile("" : "+v"(sr[s]), "+v"(si[s]), "+v"(beta[s]));
        fv before[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            before[s] = now;
            now = a[s] * now + beta[s] * (si[s] * in.at(2, s));
        }
#pragma unroll
        for (int s = STEPS - 1; s >= 0; --s) {
            const fv G = in.at(1, s) + back, xs = in.at(2, s), du = G * beta[s], u = si[s] * xs, l = k * sr[s];
            back = a[s] * G;
            // l / beta tends to 0 with l (as -sqrt(-l / 2)): where beta has become 0, so has l.  l comes last: it may be as large as fp32 goes, where back is 0
            fv rb;
#pragma unroll
            for (int q = 0; q < SC_VC; ++q) rb[q] = beta[s][q] > 0.f ? __builtin_amdgcn_rcpf(beta[s][q]) : 0.f;
            const fv q = in.kept(s, back * (before[s] - u * a[s] * rb) * l);
            q_all += q;
            if (!in.whole && t + s >= left) continue;
            store_at<T, SC_VC, FULL>(d.dx + row + s * width, at_d, c, width, in.kept(s, du * si[s]));
            store_at<T, SC_VC, FULL>(d.dr + row + s * width, at_d, c, width, in.kept(s, q * rest_of(in.at(0, s), sr[s])));
            store_at<T, SC_VC, FULL>(d.di + row + s * width, at_d, c, width, in.kept(s, du * u * rest_of(in.at(3, s), si[s])));
        }
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (t + s >= left) continue;
            store_at<T, SC_VC, FULL>(d.dx + row + s * width, at_d, c, width, fv(0.f));
            store_at<T, SC_VC, FULL>(d.dr + row + s * width, at_d, c, width, fv(0.f));
            store_at<T, SC_VC, FULL>(d.di + row + s * width, at_d, c, width, fv(0.f));
        }
    }
}

// a part of sum q, its lanes in a fixed order
template <bool FULL, typename S>
__device__ __forceinline__ void fold_q(fv (&fold)[S::RUNS][SC_LANES], fv q_all, float* qsum, const Lane<S>& at, int width) {
    fold[at.run][at.cl] = q_all;
    __syncthreads();
    if (at.run != 0) return;
    fv s = fold[0][at.cl];
#pragma unroll
    for (int w = 1; w < S::RUNS; ++w) s += fold[w][at.cl];
    store<float, SC_VC, FULL>(qsum, at.c, width, s);
}

// The composition of a chunk's C recurrence, for few sequences (r and dh alone are read), to `sums` [n, chunks, 2, width]
template <typename T, Width W>
__global__ __launch_bounds__(Bwd::THREADS, 2) void scan_bwd_sum_kernel(Seq r, Seq gh, const float* __restrict__ lam, float sharpness,
                                                                       const uint8_t* __restrict__ mask, int64_t mask_sn, float* __restrict__ sums,
                                                                       int length, int width, int per) {
    using S = Bwd;
    constexpr bool FULL = W == EVEN;
    __shared__ Totals<S> tot;
    const Lane<S> at;
    const int64_t n = blockIdx.y;
    const int c = at.c, t = at.t, n_tiles = (length + SC_TILE - 1) / SC_TILE, first = blockIdx.z * per, end = min(n_tiles, first + per);
    Rows<T, 2, W> rows;
    rows.set(0, r, n, end - 1, t, c, width);
    rows.set(1, gh, n, end - 1, t, c, width);
    if (mask != nullptr) mask += n * mask_sn;
    Steps<T, 2, S::STEPS, W> in, ahead;
    in.fetch(rows, mask != nullptr ? mask + (int64_t)(end - 1) * SC_TILE : nullptr, t, length - (end - 1) * SC_TILE, c, width);
    const fv k = rates<FULL>(lam, sharpness, c, width);
    const bool near = all_near(k);
    fv carry(0.f), through(1.f);
    for (int tile = end - 1, buf = 0;; --tile, buf ^= 1) {
        if (tile > first) {
            rows.move(-1);
            ahead.fetch(rows, mask != nullptr ? mask + (int64_t)(tile - 1) * SC_TILE : nullptr, t, length - (tile - 1) * SC_TILE, c, width);
        }
        fv A(1.f), C(0.f);
        in.template clean<0>();
#pragma unroll
        for (int s = S::STEPS - 1; s >= 0; --s) {
            fv l, a, beta;
            if (near) decay<true>(k, sigmoid_of(in.at(0, s)), l, a, beta);
            else decay<false>(k, sigmoid_of(in.at(0, s)), l, a, beta);
            C = a * (C + in.at(1, s));
            A = A * a;
        }
        Join<S, -1> j;
        j.put(tot, buf, at, A, C);
        __syncthreads();
        j.past(tot, buf, at, through, carry);
        if (tile == first) break;
        in = ahead;
    }
    if (at.run != 0) return;
    float* s = sums + (n * gridDim.z + blockIdx.z) * 2 * width;
    store<float, SC_VC, FULL>(s, c, width, through);
    store<float, SC_VC, FULL>(s + width, c, width, carry);
}

// Workgroup: channels [64 blockIdx.x, + 64) of sequences blockIdx.y, + gridDim.y, .., tiles [per blockIdx.z, + per) from the last one on.
// AHEAD: the next tile's loads are in flight while a tile is computed.  Its registers are there for 16-bit inputs only, and it pays from 4 tiles a
// workgroup on: bf16 without and with, 64 x 2048 x 256 166 / 150 us, 2 x 32768 x 768 250 / 228, 512 x 50 x 256 35.6 / 37.3; 1 x 10007 x 301 fp16, 2 tiles
// a workgroup, 33.8 / 36.0.
template <typename T, Width W, bool AHEAD>
__global__ __launch_bounds__(Bwd::THREADS, 2) void scan_bwd_kernel(Seq x, Seq r, Seq i, Seq gh, const float* __restrict__ lam, float sharpness,
                                                                   const uint8_t* __restrict__ mask, int64_t mask_sn, const float* __restrict__ tiles,
                                                                   const float* __restrict__ glast, Grads<T> d, float* __restrict__ dstate,
                                                                   float* __restrict__ qsum, const float* __restrict__ sums, int seqs, int length,
                                                                   int width, int per) {
    using S = Bwd;
    constexpr bool FULL = W == EVEN;
    __shared__ Totals<S> tot, fwd;
    __shared__ fv fold[S::RUNS][SC_LANES];
    const Lane<S> at;
    const int c = at.c, t = at.t, n_tiles = (length + SC_TILE - 1) / SC_TILE, chunks = gridDim.z, first = blockIdx.z * per, end = min(n_tiles, first + per);
    const fv k = rates<FULL>(lam, sharpness, c, width);
    const bool near = all_near(k);
    const uint32_t at_d = lane_offset<T>(t, width, c);
    fv q_all(0.f), carry(0.f);
    Rows<T, 4, W> rows;
    Steps<T, 4, S::STEPS, W> in, ahead;
    const auto fetch = [&](int64_t n, int tile, Steps<T, 4, S::STEPS, W>& to) {
        rows.set(0, r, n, tile, t, c, width);
        rows.set(1, gh, n, tile, t, c, width);
        rows.set(2, x, n, tile, t, c, width);
        rows.set(3, i, n, tile, t, c, width);
        to.fetch(rows, mask != nullptr ? mask + n * mask_sn + (int64_t)tile * SC_TILE : nullptr, t, length - tile * SC_TILE, c, width);
    };
    int tile = end - 1;
    int64_t n = blockIdx.y;
    if (glast != nullptr) carry = load<float, SC_VC, FULL>(glast + n * width, c, width);
    if (end < n_tiles) carry = entering<FULL, -1>(tot, sums + n * chunks * 2 * width, chunks - 1, chunks - 1 - (int)blockIdx.z, carry, at, width);
    // (Sequences that are cut have a workgroup each: what follows takes no second one of them.)  One loop over sequences and tiles: nested, the compiler
    // spills 45 registers.
    if constexpr (AHEAD) fetch(n, tile, in);
    for (int buf = 0; n < seqs; buf ^= 1) {
        const int left = length - tile * SC_TILE;
        // (behind the last tile some tile again, rather than a branch: with one the compiler spills)
        if constexpr (AHEAD) fetch(tile > first ? n : min(n + (int64_t)gridDim.y, (int64_t)seqs - 1), tile > first ? tile - 1 : end - 1, ahead);
        else fetch(n, tile, in);
        fv head = load<float, SC_VC, FULL>(tiles + (n * n_tiles + tile) * width, c, width);
        fv sr[S::STEPS], si[S::STEPS], a[S::STEPS], beta[S::STEPS], A, H, C;
        const bool some = compose_both(in, near, k, sr, si, a, beta, A, H, C);
        Join<S, 1> f;
        Join<S, -1> j;
        f.put(fwd, buf, at, A, H);
        j.put(tot, buf, at, A, C);
        __syncthreads();
        const fv now = f.before(fwd, buf, at, head), back = j.before(tot, buf, at, carry);
        if (tile == 0 && at.run == 0 && dstate != nullptr) store<float, SC_VC, FULL>(dstate + n * width, c, width, carry);
        gradients<T, FULL>(in, some, k, sr, si, a, beta, now, back, q_all, d, (n * length + (int64_t)tile * SC_TILE) * width, at_d, t, left, c, width);
        if constexpr (AHEAD) in = ahead;
        if (--tile < first) {
            tile = end - 1;
            n += gridDim.y;
            carry = fv(0.f);
            if (glast != nullptr && n < seqs) carry = load<float, SC_VC, FULL>(glast + n * width, c, width);
        }
    }
    fold_q<FULL>(fold, q_all, qsum + ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * width, at, width);
}

// dlam = sum q sigmoid(lam) / softplus(lam): `parts` rows of partial sums, 16 columns x 64 row lanes a workgroup, 8 rows of a lane in flight, in a fixed
// order (512 x 50 x 256, 512 rows: 16 lanes, one row in flight 8.2 us, this 4.4)
__global__ __launch_bounds__(1024) void scan_dlam_kernel(const float* __restrict__ qsum, int parts, const float* __restrict__ lam, float* __restrict__ dlam,
                                                         int width) {
    __shared__ float red[64][17];
    const int col = threadIdx.x & 15, lane = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
    float s = 0.f;
    if (c < width)
        for (int p = lane; p < parts; p += 64 * 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p + 64 * u < parts ? qsum[(int64_t)(p + 64 * u) * width + c] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    red[lane][col] = s;
    __syncthreads();
    if (lane == 0 && c < width) {
        for (int w = 1; w < 64; ++w) s += red[w][col];
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

// A workgroup a (sequence, 64 channels) reads every input once, and from some number of them on is as fast as memory or the vector units allow; fewer
// leave the GPU idle, and sequences of 4 tiles and more are then cut into chunks, which read their inputs twice.  n x 2048 x 256, us uncut / cut:
//   workgroups        64         128         160         192         224         256
//   forward   fp32   71 / 47    76 / 94     82 / 120    88 / 143    97 / 176   108 / 188      cut below  96
//   forward   bf16   61 / 36    63 / 62     64 / 76     64 / 82     65 / 101    65 / 107                128
//   backward  fp32  156 / 70   172 / 135   178 / 168   184 / 192   193 / 232   205 / 255                160
//   backward  bf16  135 / 49   146 / 91    147 / 113   149 / 124   152 / 151   153 / 158                224
// They are cut until about CUT_TO workgroups are in flight, a tile each at least.  Forward + backward (us) for 512 / 768 / 1024: 2 x 32768 x 768 bf16
// 430 / 432 / 442, 8 x 4096 x 768 bf16 250 / 224 / 225; at least 1 / 2 / 4 tiles: 1 x 10007 x 301 fp16 62 / 70 / 78, 1 x 2048 x 256 fp32 26 / 34 / 51.
// (A single pass over the chunks, each waiting for the one before it, was no faster: 184 us forward and 284 backward at 2 x 32768 x 768, 181 and 250 in two
// passes at the time.  What a tile waits for others costs more than its second reading.)
constexpr int CUT_MOST = 224, CUT_TO = 768;
static int cut_below(int dtype, bool backward) { return dtype == LEGO_F32 ? (backward ? 160 : 96) : (backward ? CUT_MOST : 128); }
static ScanPlan scan_plan(int n, int length, int width, int below) {
    ScanPlan p;
    p.slices = (width + SC_CH - 1) / SC_CH;
    p.tiles = (length + SC_TILE - 1) / SC_TILE;
    const int64_t wgs = (int64_t)n * p.slices;
    p.chunks = 1;
    if (wgs < below && p.tiles >= 4) {
        const int64_t want = (CUT_TO + wgs - 1) / wgs;
        p.chunks = (int)(want < p.tiles ? want : p.tiles);
    }
    p.per = p.tiles > 0 ? (p.tiles + p.chunks - 1) / p.chunks : 1;
    p.chunks = p.tiles > 0 ? (p.tiles + p.per - 1) / p.per : 1;        // (none is empty)
    const int cap = 2048 / p.slices > 0 ? 2048 / p.slices : 1;         // backward: workgroups that take sequences one after the other
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

// floats: the partial rows of sum q, then the chunks' compositions, of whichever call cuts
extern "C" int64_t lego_gated_scan_workspace(int n, int length, int width) {
    if (n <= 0 || length <= 0 || width <= 0) return 0;
    const ScanPlan p = scan_plan(n, length, width, CUT_MOST);
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
    const ScanPlan p = scan_plan(n, length, width, cut_below(dtype, false));
    LEGO_REQUIRE(p.chunks == 1 || (workspace != nullptr && workspace_floats >= lego_gated_scan_workspace(n, length, width)),
                 "lego_gated_scan_fwd: workspace of %lld floats, lego_gated_scan_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_gated_scan_workspace(n, length, width));
    const Seq sx{x, x_sn, x_sl}, sr{r, r_sn, r_sl}, si{i, i_sn, i_sl};
    const dim3 grid(p.slices, n, p.chunks);
#define GO(W, PASS) hipLaunchKernelGGL((scan_fwd_kernel<T, W, PASS>), grid, dim3(Fwd::THREADS), 0, ST, sx, sr, si, lam, sharpness, mask, mask_sn, state, \
                                       (T*)h, last, tiles, workspace, length, width, p.per)
#define BY_WIDTH(PASS)                          \
    do {                                        \
        if (width % 2 == 0) GO(EVEN, PASS);     \
        else if (width > 1) GO(ODD, PASS);      \
        else GO(SINGLE, PASS);                  \
    } while (0)
    LEGO_BY_TYPE(dtype, {
        if (p.chunks > 1) BY_WIDTH(Pass::SUM);
        if (p.tiles > 1) BY_WIDTH(Pass::TILES);
        else BY_WIDTH(Pass::ONE);
    });
#undef BY_WIDTH
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
    const ScanPlan p = scan_plan(n, length, width, cut_below(dtype, true));
    LEGO_REQUIRE(workspace != nullptr && workspace_floats >= lego_gated_scan_workspace(n, length, width),
                 "lego_gated_scan_bwd: workspace of %lld floats, lego_gated_scan_workspace says %lld", (long long)workspace_floats,
                 (long long)lego_gated_scan_workspace(n, length, width));
    const Seq sx{x, x_sn, x_sl}, sr{r, r_sn, r_sl}, si{i, i_sn, i_sl}, sg{gh, gh_sn, gh_sl};
    float *qsum = workspace, *sums = workspace + (int64_t)p.rows * p.chunks * width;
    const dim3 all(p.slices, n, p.chunks), grid(p.slices, p.rows, p.chunks);
#define SUM(W) hipLaunchKernelGGL((scan_bwd_sum_kernel<T, W>), all, dim3(Bwd::THREADS), 0, ST, sr, sg, lam, sharpness, mask, mask_sn, sums, length, width, p.per)
#define GO(W) hipLaunchKernelGGL((scan_bwd_kernel<T, W, ahead>), grid, dim3(Bwd::THREADS), 0, ST, sx, sr, si, sg, lam, sharpness, mask, mask_sn, tiles, glast, d, \
                                 dstate, qsum, sums, n, length, width, p.per)
#define BY_WIDTH(LAUNCH)                   \
    do {                                   \
        if (width % 2 == 0) LAUNCH(EVEN);  \
        else if (width > 1) LAUNCH(ODD);   \
        else LAUNCH(SINGLE);               \
    } while (0)
    LEGO_BY_TYPE(dtype, {
        const Grads<T> d = grads<T>(dx, dr, di);
        if (p.chunks > 1) BY_WIDTH(SUM);
        const auto run = [&](auto with) {
            constexpr bool ahead = decltype(with)::value;
            BY_WIDTH(GO);
        };
        if (sizeof(T) == 2 && p.per >= 4) run(std::integral_constant<bool, sizeof(T) == 2>());
        else run(std::false_type());
    });
#undef BY_WIDTH
#undef GO
#undef SUM
    if (int rc = check_launch("lego_gated_scan_bwd")) return rc;
    hipLaunchKernelGGL(scan_dlam_kernel, dim3((width + 15) / 16), dim3(1024), 0, ST, qsum, p.rows * p.chunks, lam, dlam, width);
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
