// Log probabilities over a catalogue or vocabulary: one read of a row of logits gives the log probability of a wanted item, the entropy and
// the k likeliest items; the backward pass reads the logits once and writes their gradient once (include/lego_hip.h: lego_token_logprobs_*).
//
//   m = max x_j   S = sum e^(x_j - m)   T = sum e^(x_j - m) (x_j - m):   lse = m + ln S   entropy = ln S - T / S   logp_t = x_t - lse
//   d x_j = -p_j (G + g_entropy (ln p_j + entropy)) + g_logp [j = t] + g_top_q [j = index_q]      G = g_logp + sum_q g_top_q
//
// A lane keeps m, S, T of its 16-byte vectors with the running maximum (T' = e^(m - m') (T + (m - m') S)), all in fp32.  m and ln S stay two
// numbers to the end: x - m is exact where x - (m + ln S) would round ln S away (logits of thousands, or all of a mask's lowest value).
//
// HBM-bound: the rest is to keep the selection off that one read.  A key orders an element by (value, lower index first) and is unique; while it
// reads, a lane keeps its largest key only.  The k-th largest of 64 (k <= 16) or 256 groups of lanes' keys is a lower bound of the k-th largest
// element, so only the few lanes at or above it can own one of the k: the workgroup reads those lanes' vectors again (about k lanes' shares of
// the row, from the caches), collects what reaches the bound and ranks it by counting.  If more than the list holds reach it, the k are taken one
// at a time instead, a reading of the row each.  That takes lanes that own very many large elements, or ties: in a row of equal elements all that the first
// k - 1 groups' lanes own come before the k-th group's first (512 x 65536, 1024 lanes: from k = 10 in bf16 -- 150 us there, 1690 for k = 128, against 20
// and 30 of ordinary rows --, from k = 65 in fp32).  Few rows are cut into chunks, and a second launch joins the chunks' statistics and keys.
#include <float.h>

#include <algorithm>

#include "seq_common.hpp"

namespace lego {

constexpr int LP_GROUPS = 256, LP_FEW = 64, LP_LIST = 1024, LP_MAX_K = LEGO_LOGPROBS_MAX_K;
static_assert(LP_MAX_K < LP_GROUPS, "the bound comes from one key a group");
constexpr float LOG2E = 1.44269504088896340736f;
using u64 = unsigned long long;

// larger for larger (value, lower index); -0 equals +0; 0 is "no element" (no element that takes part is NaN or -inf)
__device__ __forceinline__ u64 make_key(float v, uint32_t index) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return ((u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(u64 key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ int key_index(u64 key) { return (int)~(uint32_t)key; }

// A row's elements as 16-byte vectors on 16-byte boundaries: vector j holds elements [j VEC - shift, + VEC); the first and the last may be partial,
// [lo, hi) are whole.
template <typename T, bool MASK>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    struct Raw { vec<T, VEC> v; vec<uint8_t, VEC> live; };
    const T* x;
    const uint8_t* mask;
    int n, shift, lo, hi, vectors;
    __device__ Row(const T* row, const uint8_t* m, int items) : x(row), mask(m), n(items), shift((int)(((uintptr_t)row & 15) / sizeof(T))) {
        vectors = (int)(((int64_t)shift + n + VEC - 1) / VEC);
        lo = shift > 0 ? 1 : 0;
        hi = (int)(((int64_t)shift + n) / VEC);
    }
    __device__ __forceinline__ Raw whole(int j) const {
        Raw r;
        r.v = *reinterpret_cast<const vec<T, VEC>*>(x + (j * VEC - shift));
        if constexpr (MASK) __builtin_memcpy(&r.live, mask + (j * VEC - shift), VEC);
        return r;
    }
    // masked elements read as -inf
    __device__ __forceinline__ void values(const Raw& r, float (&f)[VEC]) const {
#pragma unroll
        for (int k = 0; k < VEC; ++k) f[k] = !MASK || r.live[k] ? (float)r.v[k] : -INFINITY;
    }
    // any vector; elements that are outside the row read as -inf too
    __device__ __forceinline__ void load(int j, float (&f)[VEC]) const {
        if (j >= lo && j < hi) { values(whole(j), f); return; }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int e = j * VEC - shift + k;
            f[k] = e >= 0 && e < n && (!MASK || mask[e]) ? (float)x[e] : -INFINITY;
        }
    }
};

// running maximum, sum and weighted sum; m starts at the lowest finite value, so that -inf only ever gives e^-inf = 0
struct Stat { float m, s, t; };
__device__ __forceinline__ float not_below(float v, float lo) { return v < lo ? lo : v; }         // NaN stays NaN
__device__ __forceinline__ void rescale(Stat& a, float m) {
    const float d = not_below(a.m - m, -1000.f), e = __builtin_amdgcn_exp2f(LOG2E * d);
    a.t = e * (a.t + a.s * d);
    a.s *= e;
    a.m = m;
}
__device__ __forceinline__ void add(Stat& a, float v) {
    const float d = v - a.m, e = __builtin_amdgcn_exp2f(LOG2E * d);
    a.s += e;
    a.t += e * fmaxf(d, -200.f);                                                                   // e^-200 is 0 in fp32: no 0 * -inf (a NaN is in e)
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

struct alignas(16) Shared {
    u64 list[LP_LIST];
    uint32_t high[LP_GROUPS];
    uint16_t owner[1024];
    float red[3][16];
    u64 best[16];
    u64 bound;
    int owners, found, picked;
};

// the workgroup's statistics from its lanes'
template <int NT>
__device__ __forceinline__ Stat join(Shared& sh, Stat a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = wave_max(a.m);
    if (lane == 0) sh.red[0][wave] = m;
    __syncthreads();
    m = sh.red[0][0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) m = fmaxf(m, sh.red[0][w]);
    rescale(a, m);
    const float s = wave_sum(a.s), t = wave_sum(a.t);
    if (lane == 0) { sh.red[1][wave] = s; sh.red[2][wave] = t; }
    __syncthreads();
    Stat all{m, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { all.s += sh.red[1][w]; all.t += sh.red[2][w]; }
    return all;
}

// The k largest keys of the workgroup, largest first (0 behind the last), through `put(rank, key)`.  `mine`: the largest key of this lane;
// src.each(lane, it, f): f(key) for the keys of lane `lane` in its it-th vector, it < src.iters.
template <int NT, typename Src, typename Put>
__device__ void largest(Shared& sh, const Src& src, u64 mine, int k, Put put) {
    const int tid = threadIdx.x;
    // the groups' keys: 64 groups while k is small against them, else 256
    const int groups = k <= LP_FEW / 4 ? LP_FEW : LP_GROUPS, lanes = NT / groups;
    u64 top = mine;
    for (int o = 1; o < lanes; o <<= 1) {
        const u64 other = __shfl_xor(top, o, 64);
        top = other > top ? other : top;
    }
    // A group's place among them goes by the upper 24 bits of its value, made different by the group's number: whichever groups the k first are, they
    // are k different elements, and the smallest of them is a bound.  The group's lanes share the comparisons.
    const int group = tid / lanes, part = tid % lanes, share = groups / lanes;
    const uint32_t high = ((uint32_t)(top >> 32) & 0xFFFFFF00u) | (uint32_t)(LP_GROUPS - 1 - group);
    if (tid == 0) { sh.bound = ~0ull; sh.owners = sh.found = sh.picked = 0; }
    if (part == 0) sh.high[group] = high;
    __syncthreads();
    int place = 0;
#pragma unroll 4
    for (int u = part * share; u < (part + 1) * share; u += 4) {
        const uint4 h = *reinterpret_cast<const uint4*>(&sh.high[u]);
        place += (h.x > high) + (h.y > high) + (h.z > high) + (h.w > high);
    }
    for (int o = 1; o < lanes; o <<= 1) place += __shfl_xor(place, o, 64);
    if (part == 0 && top != 0 && place < k) {
        atomicMin(&sh.bound, top);
        atomicAdd(&sh.picked, 1);
    }
    __syncthreads();
    const u64 bound = sh.picked < k ? 1ull : sh.bound;                  // fewer than k groups own anything: every element takes part
    if (mine >= bound && mine != 0) sh.owner[atomicAdd(&sh.owners, 1)] = (uint16_t)tid;
    __syncthreads();
    const int owners = sh.owners;
    const int work = owners * src.iters;                                // vectors to read again, dealt to all lanes (at most 2^28 + 1024)
    for (int w = tid; w < work; w += NT) {
        const int it = (int)((uint32_t)w / (uint32_t)owners);
        src.each(sh.owner[w - it * owners], it, [&](u64 key) {
            if (key >= bound) {
                const int at = atomicAdd(&sh.found, 1);
                if (at < LP_LIST) sh.list[at] = key;
            }
        });
    }
    __syncthreads();
    const int found = sh.found;
    if (found <= LP_LIST) {
        for (int q = tid; q < found; q += NT) {
            const u64 key = sh.list[q];
            int rank = 0;
            for (int u = 0; u < found; ++u) rank += sh.list[u] > key;
            if (rank < k) put(rank, key);
        }
        for (int q = found + tid; q < k; q += NT) put(q, 0ull);
        return;
    }
    u64 last = ~0ull;
    for (int q = 0; q < k; ++q) {                                       // one at a time: the largest key below the last one
        u64 now = 0;
        for (int it = 0; it < src.iters; ++it) src.each(tid, it, [&](u64 key) { now = key < last && key > now ? key : now; });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const u64 other = __shfl_xor(now, o, 64);
            now = other > now ? other : now;
        }
        if ((tid & 63) == 0) sh.best[tid >> 6] = now;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) now = sh.best[w] > now ? sh.best[w] : now;
        __syncthreads();
        if (tid == 0) put(q, now);
        last = now;                                                     // 0: nothing is below it, and the rest are 0 too
    }
}

template <typename T, bool MASK, int NT>
struct RowSource {
    Row<T, MASK> row;
    int v0, v1, iters;
    template <typename F>
    __device__ __forceinline__ void each(int lane, int it, F f) const {
        const int64_t j = (int64_t)v0 + lane + (int64_t)it * NT;
        if (j >= v1) return;
        float v[Row<T, MASK>::VEC];
        row.load((int)j, v);
#pragma unroll
        for (int k = 0; k < Row<T, MASK>::VEC; ++k)
            if (v[k] > -INFINITY) f(make_key(v[k], (uint32_t)((int)j * Row<T, MASK>::VEC - row.shift + k)));
    }
};

template <int NT>
struct KeySource {                                                      // the chunks' keys, dealt to the lanes one by one
    const u64* keys;
    int n, iters;
    template <typename F>
    __device__ __forceinline__ void each(int lane, int it, F f) const {
        const int64_t at = lane + (int64_t)it * NT;
        if (at < n && keys[at] != 0) f(keys[at]);
    }
};

struct Wanted { const void* p; int wide; };                             // the wanted items, int32 or int64 (NULL, or outside [0, items): none)
__device__ __forceinline__ int64_t wanted(const Wanted& w, int64_t row) {
    return w.p == nullptr ? -1 : w.wide ? ((const int64_t*)w.p)[row] : ((const int32_t*)w.p)[row];
}

static Wanted wanted_from(const void* targets, int wide, int64_t row) {
    return {targets == nullptr ? nullptr : wide ? (const void*)((const int64_t*)targets + row) : (const void*)((const int32_t*)targets + row), wide};
}

struct Outputs { float *logp, *entropy, *stat, *top; int32_t* index; };

// the wanted item's logit, -inf where a mask hides it (asked for before the row is read: its latency is then hidden)
template <typename T>
__device__ __forceinline__ float wanted_logit(const T* x, const uint8_t* mask, int64_t t, int items) {
    return t >= 0 && t < items && (mask == nullptr || mask[t]) ? (float)x[t] : -INFINITY;
}

// the row's numbers, and m and ln S as they are kept; a row with nothing left has m = -inf and log probabilities -inf, one with NaN or +inf has NaN
struct Norm { float m, ln_s; };
__device__ __forceinline__ Norm row_numbers(const Outputs& out, int64_t row, int64_t t, float xt, int items, Stat a) {
    const bool empty = a.s == 0.f;
    const Norm r{empty ? -INFINITY : a.m, empty ? 0.f : logf(a.s)};
    if (threadIdx.x == 0) {
        out.stat[2 * row] = r.m;
        out.stat[2 * row + 1] = r.ln_s;
        out.entropy[row] = empty ? 0.f : r.ln_s - a.t / a.s;
        out.logp[row] = t < 0 || t >= items ? 0.f : empty || xt == -INFINITY ? -INFINITY + (empty ? 0.f : 0.f * r.ln_s) : (xt - r.m) - r.ln_s;
    }
    return r;
}

__device__ __forceinline__ void put_top(const Outputs& out, int64_t at, u64 key, Norm r) {
    out.top[at] = key ? (key_value(key) - r.m) - r.ln_s : -INFINITY;
    out.index[at] = key ? key_index(key) : -1;
}
template <int NT>
__device__ __forceinline__ void put_undefined(const Outputs& out, int64_t row, int k) {
    for (int q = threadIdx.x; q < k; q += NT) { out.top[row * k + q] = NAN; out.index[row * k + q] = -1; }
}

// Workgroup: chunk `blockIdx.x % chunks` of row `blockIdx.x / chunks`, vectors [chunk per, + per).  Chunks leave their statistics and keys behind.
template <typename T, bool MASK, int NT>
__global__ __launch_bounds__(NT) void logprobs_fwd_kernel(const T* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask, int64_t mask_ld,
                                                          Wanted w, Outputs out, float4* __restrict__ stats, u64* __restrict__ keys, int items, int k, int chunks,
                                                          int per) {
    __shared__ Shared sh;
    constexpr int VEC = 16 / sizeof(T), UNROLL = 4;
    const int64_t row = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x - row * chunks), tid = threadIdx.x;
    const T* xr = logits + row * ld;
    const uint8_t* mr = MASK ? mask + row * mask_ld : nullptr;
    const Row<T, MASK> src(xr, mr, items);
    const int v0 = chunk * per, v1 = min(src.vectors, v0 + per), lo = max(v0, src.lo), hi = min(v1, src.hi);
    const int64_t t = chunks == 1 ? wanted(w, row) : -1;
    const float xt = wanted_logit(xr, mr, t, items);
    Stat a{-FLT_MAX, 0.f, 0.f};
    float best = -INFINITY;
    int best_at = 0;
    const auto take = [&](int j, const float (&f)[VEC]) {
        float top = f[0];
#pragma unroll
        for (int q = 1; q < VEC; ++q) top = fmaxf(top, f[q]);
        if (top > best) {
            int at = VEC - 1;
#pragma unroll
            for (int q = VEC - 2; q >= 0; --q) at = f[q] == top ? q : at;
            best = top;
            best_at = j * VEC - src.shift + at;
            rescale(a, top);
        }
#pragma unroll
        for (int q = 0; q < VEC; ++q) add(a, f[q]);
    };
    // vector j belongs to lane (j - v0) mod NT.  The whole ones: UNROLL loads in flight, without a branch between them (what is behind the end
    // loads the last whole vector again and does not count)
    if (src.lo > v0 && tid == 0) {
        float f[VEC];
        src.load(v0, f);
        take(v0, f);
    }
    for (int j = v0 + tid; lo < hi && j < hi; j += NT * UNROLL) {
        typename Row<T, MASK>::Raw raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) raw[u] = src.whole(min(max(j + u * NT, lo), hi - 1));
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int at = j + u * NT;
            if (at < lo || at >= hi) continue;
            float f[VEC];
            src.values(raw[u], f);
            take(at, f);
        }
    }
    if (v1 > v0 && v1 > hi && v1 > src.lo && (v1 - 1 - v0) % NT == tid) {          // the partial one at the row's end
        float f[VEC];
        src.load(v1 - 1, f);
        take(v1 - 1, f);
    }
    a = join<NT>(sh, a);
    const u64 mine = best > -INFINITY ? make_key(best, (uint32_t)best_at) : 0ull;
    const RowSource<T, MASK, NT> source{src, v0, v1, (max(v1 - v0, 0) + NT - 1) / NT};
    const bool defined = a.s == a.s;
    if (chunks > 1) {
        const int64_t at = row * chunks + chunk;
        if (tid == 0) stats[at] = make_float4(a.m, a.s, a.t, 0.f);
        if (k > 0 && defined) largest<NT>(sh, source, mine, k, [&](int q, u64 key) { keys[at * k + q] = key; });
        return;
    }
    const Norm norm = row_numbers(out, row, t, xt, items, a);
    if (k == 0) return;
    if (defined) largest<NT>(sh, source, mine, k, [&](int q, u64 key) { put_top(out, row * k + q, key, norm); });
    else put_undefined<NT>(out, row, k);
}

// one workgroup a row: the chunks' statistics and keys
template <typename T, int NT>
__global__ __launch_bounds__(NT) void logprobs_join_kernel(const T* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask, int64_t mask_ld, Wanted w,
                                                           Outputs out, const float4* __restrict__ stats, const u64* __restrict__ keys, int items, int k,
                                                           int chunks) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const int64_t t = wanted(w, row);
    const float xt = wanted_logit(logits + row * ld, mask != nullptr ? mask + row * mask_ld : nullptr, t, items);
    const KeySource<NT> source{keys + row * chunks * k, chunks * k, (chunks * k + NT - 1) / NT};
    u64 mine = 0;                                                       // (of a row that is not a distribution these are not keys, and not used)
    for (int q = tid; q < source.n; q += NT) mine = source.keys[q] > mine ? source.keys[q] : mine;
    Stat a{-FLT_MAX, 0.f, 0.f};
    for (int c = tid; c < chunks; c += NT) {
        const float4 s = stats[row * chunks + c];
        Stat b{s.x, s.y, s.z};
        const float m = fmaxf(a.m, b.m);
        rescale(a, m);
        rescale(b, m);
        a.s += b.s;
        a.t += b.t;
    }
    a = join<NT>(sh, a);
    const Norm norm = row_numbers(out, row, t, xt, items, a);
    if (k == 0) return;
    if (a.s == a.s) largest<NT>(sh, source, mine, k, [&](int q, u64 key) { put_top(out, row * k + q, key, norm); });
    else put_undefined<NT>(out, row, k);
}

struct Grads { const float *logp, *entropy, *top; };

template <typename T, bool MASK>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const T* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask, int64_t mask_ld,
                                                                  Wanted w, const float* __restrict__ stat, const float* __restrict__ entropy_,
                                                                  const int32_t* __restrict__ index, Grads g, T* __restrict__ dlogits, int items, int k,
                                                                  int chunks, int per) {
    __shared__ float red[4];
    constexpr int VEC = 16 / sizeof(T);
    using V = T __attribute__((ext_vector_type(VEC)));
    const int64_t row = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x - row * chunks), tid = threadIdx.x;
    const uint8_t* mr = MASK ? mask + row * mask_ld : nullptr;
    const Row<T, MASK> src(logits + row * ld, mr, items);
    T* dr = dlogits + row * items;
    const Row<T, false> dst(dr, nullptr, items);                        // the vectors lie on the output's 16-byte boundaries
    const bool same = src.shift == dst.shift;
    const float top = stat[2 * row], ln_s = stat[2 * row + 1], entropy = entropy_[row], ge = g.entropy != nullptr ? g.entropy[row] : 0.f;
    const int64_t t = wanted(w, row);
    const float gl = g.logp != nullptr && t >= 0 && t < items ? g.logp[row] : 0.f;
    float all = gl;
    if (g.top != nullptr) {
        float s = 0.f;
        for (int q = tid; q < k; q += 256) s += index[row * k + q] >= 0 ? g.top[row * k + q] : 0.f;
        s = wave_sum(s);
        if ((tid & 63) == 0) red[tid >> 6] = s;
        __syncthreads();
        all += (red[0] + red[1]) + (red[2] + red[3]);
    }
    const bool empty = top == -INFINITY;
    const auto value = [&](float v, int e) {                            // d logits[e], without the top's own share
        const float lp = not_below((v - top) - ln_s, -200.f), p = __builtin_amdgcn_exp2f(LOG2E * lp);
        const float d = -p * (all + ge * (lp + entropy));
        return e == t ? d + gl : d;
    };
    const int v0 = chunk * per, v1 = min(dst.vectors, v0 + per);
    for (int j = v0 + tid; j < v1; j += 256) {
        const int e0 = j * VEC - dst.shift;
        if (e0 >= 0 && e0 <= items - VEC) {
            float f[VEC];
            bool live[VEC];
            if (same) {
                const V v = *reinterpret_cast<const V*>(src.x + e0);
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] = (float)v[q];
            } else
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] = (float)src.x[e0 + q];
            if constexpr (MASK) {
                uint8_t m[VEC];
                __builtin_memcpy(m, mr + e0, VEC);
#pragma unroll
                for (int q = 0; q < VEC; ++q) live[q] = m[q] != 0;
            } else
#pragma unroll
                for (int q = 0; q < VEC; ++q) live[q] = true;
            V o;
#pragma unroll
            for (int q = 0; q < VEC; ++q) o[q] = (T)(live[q] && !empty ? value(f[q], e0 + q) : 0.f);
            *reinterpret_cast<V*>(dr + e0) = o;
        } else
            for (int q = 0; q < VEC; ++q) {
                const int e = e0 + q;
                if (e >= 0 && e < items) dr[e] = (T)((!MASK || mr[e]) && !empty ? value((float)src.x[e], e) : 0.f);
            }
    }
    if (g.top == nullptr || empty) return;
    __syncthreads();                                                    // every store of this chunk is done: the k places are written again, whole
    for (int q = tid; q < k; q += 256) {
        const int e = index[row * k + q];
        if (e < 0 || e >= items || (MASK && !mr[e])) continue;
        const int j = (e + dst.shift) / VEC;
        if (j >= v0 && j < v1) dr[e] = (T)(value((float)src.x[e], e) + g.top[row * k + q]);
    }
}

struct LogprobPlan { int chunks, per, threads; };

// A launch has fewer than 2^32 lanes: more rows than that go in several, one after the other (forward, only rows that are one chunk: fewer than 512 rows
// are cut, into 512 workgroups and some)
static int rows_a_launch(const LogprobPlan& p) { return (int)(((1ll << 32) - 1) / p.threads / p.chunks); }

// Forward: a workgroup a row, of 1024 lanes where a row has 8192 vectors (of 16 bytes) and more, else of 256 (2048 x 30522 bf16: 33 us with 256 lanes, 50
// with 1024, whose ends are too much of so short a row, one call after another; 45 with 256 behind a backward pass, which leaves none of the logits in the
// cache; 512 x 65238 fp32, 50 alternatives: 47 and 37 us).  Fewer than 512 rows do not fill
// the 256 CUs: they are cut into chunks of at least 2048 vectors until there are about 512 workgroups, and joined by a second launch.
static LogprobPlan fwd_plan(int rows, int items, int dtype) {
    const int vec = dtype == LEGO_F32 ? 4 : 8;
    const int64_t vectors = ((int64_t)items + 2 * vec - 2) / vec;       // of a row at the worst alignment
    LogprobPlan p;
    p.threads = vectors >= 8192 ? 1024 : 256;
    int64_t want = (512 + (int64_t)rows - 1) / rows, most = vectors / 2048;
    if (want > most) want = most;
    if (want < 1) want = 1;
    p.per = (int)((vectors + want - 1) / want);
    p.chunks = (int)((vectors + p.per - 1) / p.per);
    return p;
}
static LogprobPlan bwd_plan(int items, int dtype) {
    const int vec = dtype == LEGO_F32 ? 4 : 8;
    const int64_t vectors = ((int64_t)items + 2 * vec - 2) / vec;
    LogprobPlan p;
    p.threads = 256;
    p.per = 2048;
    p.chunks = (int)((vectors + p.per - 1) / p.per);
    return p;
}

}  // namespace lego

using namespace lego;
#define ST ((hipStream_t)stream)

static int logprobs_check(const char* who, int dtype, int rows, int items, int k) {
    LEGO_REQUIRE(dtype == LEGO_F32 || dtype == LEGO_BF16 || dtype == LEGO_F16, "%s: unknown dtype %d", who, dtype);
    LEGO_REQUIRE(rows >= 0 && items > 0 && items <= (1 << 30), "%s: bad sizes rows=%d, items=%d", who, rows, items);
    LEGO_REQUIRE(k >= 0 && k <= LP_MAX_K && k <= items, "%s: k=%d (at most %d, and at most items=%d)", who, k, LP_MAX_K, items);
    return 0;
}

extern "C" int64_t lego_token_logprobs_workspace(int rows, int items, int dtype, int k) {
    if (rows <= 0 || items <= 0) return 0;
    const LogprobPlan p = fwd_plan(rows, items, dtype);
    return p.chunks > 1 ? (int64_t)rows * p.chunks * (2 + (int64_t)k) : 0;      // statistics (16 bytes) and k keys a chunk
}

extern "C" int lego_token_logprobs_fwd(const void* logits, int64_t ld, int dtype, const uint8_t* mask, int64_t mask_ld, const void* targets, int targets_64,
                                       int k, float* logp, float* entropy, float* stat, float* top, int32_t* index, uint64_t* workspace,
                                       int64_t workspace_words, int rows, int items, void* stream) {
    if (int rc = logprobs_check("lego_token_logprobs_fwd", dtype, rows, items, k)) return rc;
    if (rows == 0) return 0;
    LEGO_REQUIRE(logits && logp && entropy && stat && (k == 0 || (top && index)), "lego_token_logprobs_fwd: NULL operand");
    const LogprobPlan p = fwd_plan(rows, items, dtype);
    LEGO_REQUIRE(p.chunks == 1 || (workspace != nullptr && workspace_words >= lego_token_logprobs_workspace(rows, items, dtype, k)),
                 "lego_token_logprobs_fwd: workspace of %lld words, lego_token_logprobs_workspace says %lld", (long long)workspace_words,
                 (long long)lego_token_logprobs_workspace(rows, items, dtype, k));
    float4* stats = (float4*)workspace;
    u64* keys = (u64*)workspace + 2 * (int64_t)rows * p.chunks;
    const int most = rows_a_launch(p);
#define GO(MASK, NT) hipLaunchKernelGGL((logprobs_fwd_kernel<T, MASK, NT>), grid, dim3(NT), 0, ST, x, ld, m, mask_ld, w, out, stats, keys, items, k, p.chunks, p.per)
#define JOIN(NT) hipLaunchKernelGGL((logprobs_join_kernel<T, NT>), dim3(rows), dim3(NT), 0, ST, x, ld, m, mask_ld, w, out, stats, keys, items, k, p.chunks)
    LEGO_BY_TYPE(dtype, {
        for (int64_t r = 0; r < rows; r += most) {
            const dim3 grid((unsigned)(std::min<int64_t>(most, rows - r) * p.chunks));
            const T* x = (const T*)logits + r * ld;
            const uint8_t* m = mask != nullptr ? mask + r * mask_ld : nullptr;
            const Wanted w = wanted_from(targets, targets_64, r);
            const Outputs out{logp + r, entropy + r, stat + 2 * r, top != nullptr ? top + r * k : nullptr, index != nullptr ? index + r * k : nullptr};
            if (p.threads == 1024) { if (mask != nullptr) GO(true, 1024); else GO(false, 1024); }
            else if (mask != nullptr) GO(true, 256); else GO(false, 256);
            if (p.chunks > 1) { if ((int64_t)p.chunks * k > 256) JOIN(1024); else JOIN(256); }
        }
    });
#undef GO
#undef JOIN
    return check_launch("lego_token_logprobs_fwd");
}

extern "C" int lego_token_logprobs_bwd(const void* logits, int64_t ld, int dtype, const uint8_t* mask, int64_t mask_ld, const void* targets, int targets_64,
                                       int k, const float* stat, const float* entropy, const int32_t* index, const float* g_logp, const float* g_entropy,
                                       const float* g_top, void* dlogits, int rows, int items, void* stream) {
    if (int rc = logprobs_check("lego_token_logprobs_bwd", dtype, rows, items, k)) return rc;
    if (rows == 0) return 0;
    LEGO_REQUIRE(logits && stat && entropy && dlogits && (g_top == nullptr || (k > 0 && index)), "lego_token_logprobs_bwd: NULL operand");
    const LogprobPlan p = bwd_plan(items, dtype);
    const int most = rows_a_launch(p);
#define GO(MASK) hipLaunchKernelGGL((logprobs_bwd_kernel<T, MASK>), grid, dim3(256), 0, ST, (const T*)logits + r * ld, ld, m, mask_ld, w, stat + 2 * r, entropy + r, \
                                    i, g, (T*)dlogits + r * items, items, k, p.chunks, p.per)
    LEGO_BY_TYPE(dtype, {
        for (int64_t r = 0; r < rows; r += most) {
            const dim3 grid((unsigned)(std::min<int64_t>(most, rows - r) * p.chunks));
            const uint8_t* m = mask != nullptr ? mask + r * mask_ld : nullptr;
            const Wanted w = wanted_from(targets, targets_64, r);
            const Grads g{g_logp != nullptr ? g_logp + r : nullptr, g_entropy != nullptr ? g_entropy + r : nullptr, g_top != nullptr ? g_top + r * k : nullptr};
            const int32_t* i = index != nullptr ? index + r * k : nullptr;
            if (mask != nullptr) GO(true); else GO(false);
        }
    });
#undef GO
    return check_launch("lego_token_logprobs_bwd");
}
