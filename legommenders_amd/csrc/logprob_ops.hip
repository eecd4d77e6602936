// Log probabilities over a catalogue or vocabulary: one read of a row of logits gives the log probability of a wanted item, the entropy and
// the k likeliest items; the backward pass reads the logits once and writes their gradient once (include/lego_hip.h: lego_token_logprobs_*).
//
//   m = max x_j   S = sum e^(x_j - m)   T = sum e^(x_j - m) (x_j - m):   lse = m + ln S   entropy = ln S - T / S   logp_t = x_t - lse
//   d x_j = -p_j (G + g_entropy (ln p_j + entropy)) + g_logp [j = t] + g_top_q [j = index_q]      G = g_logp + sum_q g_top_q
//
// A lane keeps m, S, T of its 16-byte vectors with the running maximum (T' = e^(m - m') (T + (m - m') S)), all in fp32.  HBM-bound: the rest is
// to keep the selection off that one read.  A key orders an element by (value, lower index first) and is unique; while it reads, a lane keeps
// its largest key only.  The k-th largest of the 256 lanes' keys is a lower bound of the k-th largest element, so only the few lanes at or
// above it can own one of the k: the workgroup reads those lanes' vectors again (about k of 256 shares of the row, mostly from the caches),
// collects what reaches the bound and ranks it by counting.  If more than the list holds reach it (lanes that own very many large elements),
// the k are taken one at a time instead.  Few rows are cut into chunks, and a second launch joins the chunks' statistics and keys.
#include <float.h>

#include "seq_common.hpp"

namespace lego {

constexpr int LP_THREADS = 256, LP_LIST = 1024, LP_MAX_K = LEGO_LOGPROBS_MAX_K;
static_assert(LP_MAX_K < LP_THREADS, "the bound comes from one key a lane");
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

// A row's elements as 16-byte vectors on 16-byte boundaries: vector j holds elements [j VEC - shift, + VEC); the first and the last may be partial.
template <typename T, bool MASK>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    const T* x;
    const uint8_t* mask;
    int n, shift;
    __device__ Row(const T* row, const uint8_t* m, int items) : x(row), mask(m), n(items), shift((int)(((uintptr_t)row & 15) / sizeof(T))) {}
    __device__ int vectors() const { return (int)(((int64_t)shift + n + VEC - 1) / VEC); }
    // elements that are outside the row or masked read as -inf
    __device__ __forceinline__ void load(int j, float (&f)[VEC]) const {
        const int e0 = j * VEC - shift;
        if (e0 >= 0 && e0 <= n - VEC) {
            using V = T __attribute__((ext_vector_type(VEC)));
            const V v = *reinterpret_cast<const V*>(x + e0);
#pragma unroll
            for (int k = 0; k < VEC; ++k) f[k] = (float)v[k];
            if constexpr (MASK) {
                uint8_t live[VEC];
                __builtin_memcpy(live, mask + e0, VEC);
#pragma unroll
                for (int k = 0; k < VEC; ++k) f[k] = live[k] ? f[k] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const int e = e0 + k;
                f[k] = e >= 0 && e < n && (!MASK || mask[e]) ? (float)x[e] : -INFINITY;
            }
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
    const float d = not_below(v - a.m, -200.f), e = __builtin_amdgcn_exp2f(LOG2E * d);            // e^-200 is 0 in fp32
    a.s += e;
    a.t += e * d;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

struct alignas(16) Shared {
    u64 list[LP_LIST];
    uint32_t high[LP_THREADS];
    uint16_t owner[LP_THREADS];
    float red[3][4];
    u64 best[4];
    u64 bound;
    int owners, found, picked;
};

// the workgroup's statistics from its lanes'
__device__ __forceinline__ Stat join(Shared& sh, Stat a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = wave_max(a.m);
    if (lane == 0) sh.red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh.red[0][0], sh.red[0][1]), fmaxf(sh.red[0][2], sh.red[0][3]));
    rescale(a, m);
    const float s = wave_sum(a.s), t = wave_sum(a.t);
    if (lane == 0) { sh.red[1][wave] = s; sh.red[2][wave] = t; }
    __syncthreads();
    return Stat{m, (sh.red[1][0] + sh.red[1][1]) + (sh.red[1][2] + sh.red[1][3]), (sh.red[2][0] + sh.red[2][1]) + (sh.red[2][2] + sh.red[2][3])};
}

// The k largest keys of the workgroup, largest first (0 behind the last), through `put(rank, key)`.  `mine`: the largest key of this lane;
// src.each(owner, it, f): f(key) for the keys of lane `owner` in its it-th vector, it < src.iters.
template <typename Src, typename Put>
__device__ void largest(Shared& sh, const Src& src, u64 mine, int k, Put put) {
    const int tid = threadIdx.x;
    if (tid == 0) { sh.bound = ~0ull; sh.owners = sh.found = sh.picked = 0; }
    const uint32_t high = (uint32_t)(mine >> 32);
    sh.high[tid] = high;
    __syncthreads();
    // this lane's place among the 256 (equal values by lane): the k first hold k different elements, the smallest of which is the bound
    int place = 0;
    for (int u = 0; u < LP_THREADS; u += 4) {
        const uint4 h = *reinterpret_cast<const uint4*>(&sh.high[u]);
        place += (h.x > high || (h.x == high && u < tid)) + (h.y > high || (h.y == high && u + 1 < tid)) + (h.z > high || (h.z == high && u + 2 < tid)) +
                 (h.w > high || (h.w == high && u + 3 < tid));
    }
    if (mine != 0 && place < k) {
        atomicMin(&sh.bound, mine);
        atomicAdd(&sh.picked, 1);
    }
    __syncthreads();
    const u64 bound = sh.picked < k ? 1ull : sh.bound;                  // fewer than k lanes own anything: every element takes part
    if (mine >= bound && mine != 0) sh.owner[atomicAdd(&sh.owners, 1)] = (uint16_t)tid;
    __syncthreads();
    const int owners = sh.owners;
    const int64_t work = (int64_t)owners * src.iters;
    for (int64_t w = tid; w < work; w += LP_THREADS) {
        const int it = (int)(w / owners);
        src.each(sh.owner[w - (int64_t)it * owners], it, [&](u64 key) {
            if (key >= bound) {
                const int at = atomicAdd(&sh.found, 1);
                if (at < LP_LIST) sh.list[at] = key;
            }
        });
    }
    __syncthreads();
    const int found = sh.found;
    if (found <= LP_LIST) {
        for (int q = tid; q < found; q += LP_THREADS) {
            const u64 key = sh.list[q];
            int rank = 0;
            for (int u = 0; u < found; ++u) rank += sh.list[u] > key;
            if (rank < k) put(rank, key);
        }
        for (int q = found + tid; q < k; q += LP_THREADS) put(q, 0ull);
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
        for (int w = 0; w < 4; ++w) now = sh.best[w] > now ? sh.best[w] : now;
        __syncthreads();
        if (tid == 0) put(q, now);
        last = now;                                                     // 0: nothing is below it, and the rest are 0 too
    }
}

template <typename T, bool MASK>
struct RowSource {
    Row<T, MASK> row;
    int v0, v1, iters;
    template <typename F>
    __device__ __forceinline__ void each(int owner, int it, F f) const {
        const int64_t j = (int64_t)v0 + owner + (int64_t)it * LP_THREADS;
        if (j >= v1) return;
        float v[Row<T, MASK>::VEC];
        row.load((int)j, v);
#pragma unroll
        for (int k = 0; k < Row<T, MASK>::VEC; ++k)
            if (v[k] > -INFINITY) f(make_key(v[k], (uint32_t)((int)j * Row<T, MASK>::VEC - row.shift + k)));
    }
};

struct KeySource {                                                      // the chunks' keys, dealt to the lanes one by one
    const u64* keys;
    int n, iters;
    template <typename F>
    __device__ __forceinline__ void each(int owner, int it, F f) const {
        const int64_t at = owner + (int64_t)it * LP_THREADS;
        if (at < n && keys[at] != 0) f(keys[at]);
    }
};

struct Wanted { const void* p; int wide; };                             // the wanted items, int32 or int64 (NULL, or outside [0, items): none)
__device__ __forceinline__ int64_t wanted(const Wanted& w, int64_t row) {
    return w.p == nullptr ? -1 : w.wide ? ((const int64_t*)w.p)[row] : ((const int32_t*)w.p)[row];
}

struct Outputs { float *logp, *entropy, *lse, *top; int32_t* index; };

// the row's numbers; a row with nothing left has log probabilities -inf and entropy 0, one with NaN or +inf has NaN
template <typename T>
__device__ __forceinline__ void row_numbers(const Outputs& out, int64_t row, const T* x, const uint8_t* mask, int items, const Wanted& w, Stat a, float& lse) {
    const bool empty = a.s == 0.f;
    lse = empty ? -INFINITY : a.m + logf(a.s);
    if (threadIdx.x == 0) {
        out.lse[row] = lse;
        out.entropy[row] = empty ? 0.f : logf(a.s) - a.t / a.s;
        const int64_t t = wanted(w, row);
        float lp = 0.f;
        if (t >= 0 && t < items) lp = empty || (mask != nullptr && !mask[t]) ? -INFINITY : (float)x[t] - lse;
        out.logp[row] = lp;
    }
}

// workgroup: chunk `blockIdx.x % chunks` of row `blockIdx.x / chunks`, vectors [chunk per, + per)
template <typename T, bool MASK>
__global__ __launch_bounds__(LP_THREADS) void logprobs_fwd_kernel(const T* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask, int64_t mask_ld,
                                                                  Wanted w, Outputs out, u64* __restrict__ work, int items, int k, int chunks, int per) {
    __shared__ Shared sh;
    constexpr int VEC = 16 / sizeof(T), UNROLL = 4;
    const int64_t row = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x - row * chunks), tid = threadIdx.x;
    const T* xr = logits + row * ld;
    const uint8_t* mr = MASK ? mask + row * mask_ld : nullptr;
    const Row<T, MASK> src(xr, mr, items);
    const int v0 = chunk * per, v1 = min(src.vectors(), v0 + per);
    Stat a{-FLT_MAX, 0.f, 0.f};
    float best = -INFINITY;
    int best_at = 0;
    for (int j = v0 + tid; j < v1; j += LP_THREADS * UNROLL) {
        float f[UNROLL][VEC];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (j + u * LP_THREADS < v1) src.load(j + u * LP_THREADS, f[u]);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (j + u * LP_THREADS >= v1) break;
            float top = f[u][0];
#pragma unroll
            for (int q = 1; q < VEC; ++q) top = fmaxf(top, f[u][q]);
            if (top > best) {
                int at = VEC - 1;
#pragma unroll
                for (int q = VEC - 2; q >= 0; --q) at = f[u][q] == top ? q : at;
                best = top;
                best_at = (j + u * LP_THREADS) * VEC - src.shift + at;
                rescale(a, top);
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) add(a, f[u][q]);
        }
    }
    a = join(sh, a);
    const u64 mine = best > -INFINITY ? make_key(best, (uint32_t)best_at) : 0ull;
    const RowSource<T, MASK> keys{src, v0, v1, (max(v1 - v0, 0) + LP_THREADS - 1) / LP_THREADS};
    const bool defined = a.s == a.s;
    if (chunks > 1) {
        u64* mywork = work + (row * chunks + chunk) * (2 + k);
        if (tid == 0) {
            reinterpret_cast<float*>(mywork)[0] = a.m;
            reinterpret_cast<float*>(mywork)[1] = a.s;
            reinterpret_cast<float*>(mywork)[2] = a.t;
        }
        if (k > 0 && defined) largest(sh, keys, mine, k, [&](int q, u64 key) { mywork[2 + q] = key; });
        return;
    }
    float lse;
    row_numbers(out, row, xr, mr, items, w, a, lse);
    if (k == 0) return;
    if (defined)
        largest(sh, keys, mine, k, [&](int q, u64 key) {
            out.top[row * k + q] = key ? key_value(key) - lse : -INFINITY;
            out.index[row * k + q] = key ? key_index(key) : -1;
        });
    else
        for (int q = tid; q < k; q += LP_THREADS) { out.top[row * k + q] = NAN; out.index[row * k + q] = -1; }
}

// one workgroup a row: the chunks' statistics and keys
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_join_kernel(const T* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask, int64_t mask_ld,
                                                                   Wanted w, Outputs out, u64* __restrict__ work, u64* __restrict__ keys, int items, int k, int chunks) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const u64* mywork = work + row * chunks * (2 + k);
    Stat a{-FLT_MAX, 0.f, 0.f};
    for (int c = tid; c < chunks; c += LP_THREADS) {
        const float* s = reinterpret_cast<const float*>(mywork + (int64_t)c * (2 + k));
        Stat b{s[0], s[1], s[2]};
        const float m = fmaxf(a.m, b.m);
        rescale(a, m);
        rescale(b, m);
        a.s += b.s;
        a.t += b.t;
    }
    a = join(sh, a);
    float lse;
    row_numbers(out, row, logits + row * ld, mask != nullptr ? mask + row * mask_ld : nullptr, items, w, a, lse);
    if (k == 0) return;
    if (!(a.s == a.s)) {
        for (int q = tid; q < k; q += LP_THREADS) { out.top[row * k + q] = NAN; out.index[row * k + q] = -1; }
        return;
    }
    // the keys of all chunks in one run
    u64* mykeys = keys + row * chunks * k;
    u64 mine = 0;
    for (int q = tid; q < chunks * k; q += LP_THREADS) {
        const int c = q / k;
        const u64 key = mywork[(int64_t)c * (2 + k) + 2 + (q - c * k)];
        mykeys[q] = key;
        mine = key > mine ? key : mine;
    }
    __syncthreads();
    const KeySource src{mykeys, chunks * k, (chunks * k + LP_THREADS - 1) / LP_THREADS};
    largest(sh, src, mine, k, [&](int q, u64 key) {
        out.top[row * k + q] = key ? key_value(key) - lse : -INFINITY;
        out.index[row * k + q] = key ? key_index(key) : -1;
    });
}

struct Grads { const float *logp, *entropy, *top; };

template <typename T, bool MASK>
__global__ __launch_bounds__(LP_THREADS) void logprobs_bwd_kernel(const T* __restrict__ logits, int64_t ld, const uint8_t* __restrict__ mask, int64_t mask_ld,
                                                                  Wanted w, const float* __restrict__ lse_, const float* __restrict__ entropy_,
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
    const float lse = lse_[row], entropy = entropy_[row], ge = g.entropy != nullptr ? g.entropy[row] : 0.f;
    const int64_t t = wanted(w, row);
    const float gl = g.logp != nullptr && t >= 0 && t < items ? g.logp[row] : 0.f;
    float all = gl;
    if (g.top != nullptr) {
        float s = 0.f;
        for (int q = tid; q < k; q += LP_THREADS) s += index[row * k + q] >= 0 ? g.top[row * k + q] : 0.f;
        s = wave_sum(s);
        if ((tid & 63) == 0) red[tid >> 6] = s;
        __syncthreads();
        all += (red[0] + red[1]) + (red[2] + red[3]);
    }
    const bool empty = lse == -INFINITY;
    const auto value = [&](float v, int e) {                            // d logits[e], without the top's own share
        const float lp = not_below(v - lse, -200.f), p = __builtin_amdgcn_exp2f(LOG2E * lp);
        const float d = -p * (all + ge * (lp + entropy));
        return e == t ? d + gl : d;
    };
    const int v0 = chunk * per, v1 = min(dst.vectors(), v0 + per);
    for (int j = v0 + tid; j < v1; j += LP_THREADS) {
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
    for (int q = tid; q < k; q += LP_THREADS) {
        const int e = index[row * k + q];
        if (e < 0 || e >= items || (MASK && !mr[e])) continue;
        const int j = (e + dst.shift) / VEC;
        if (j >= v0 && j < v1) dr[e] = (T)(value((float)src.x[e], e) + g.top[row * k + q]);
    }
}

struct LogprobPlan { int chunks, per; };

// forward: one workgroup a row from about 2048 rows on; below, chunks of at least 1024 vectors until there are as many workgroups
static LogprobPlan fwd_plan(int rows, int items, int dtype) {
    const int vec = dtype == LEGO_F32 ? 4 : 8;
    const int64_t vectors = ((int64_t)items + 2 * vec - 2) / vec;       // of a row at the worst alignment
    int64_t want = (2048 + (int64_t)rows - 1) / rows, most = (vectors + 1023) / 1024;
    if (want > most) want = most;
    if (want < 1) want = 1;
    LogprobPlan p;
    p.per = (int)((vectors + want - 1) / want);
    p.chunks = (int)((vectors + p.per - 1) / p.per);
    return p;
}
static LogprobPlan bwd_plan(int items, int dtype) {
    const int vec = dtype == LEGO_F32 ? 4 : 8;
    const int64_t vectors = ((int64_t)items + 2 * vec - 2) / vec;
    LogprobPlan p;
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
    return p.chunks > 1 ? (int64_t)rows * p.chunks * (2 + 2 * (int64_t)k) : 0;
}

extern "C" int lego_token_logprobs_fwd(const void* logits, int64_t ld, int dtype, const uint8_t* mask, int64_t mask_ld, const void* targets, int targets_64,
                                       int k, float* logp, float* entropy, float* lse, float* top, int32_t* index, uint64_t* workspace,
                                       int64_t workspace_words, int rows, int items, void* stream) {
    if (int rc = logprobs_check("lego_token_logprobs_fwd", dtype, rows, items, k)) return rc;
    if (rows == 0) return 0;
    LEGO_REQUIRE(logits && logp && entropy && lse && (k == 0 || (top && index)), "lego_token_logprobs_fwd: NULL operand");
    const LogprobPlan p = fwd_plan(rows, items, dtype);
    LEGO_REQUIRE(p.chunks == 1 || (workspace != nullptr && workspace_words >= lego_token_logprobs_workspace(rows, items, dtype, k)),
                 "lego_token_logprobs_fwd: workspace of %lld words, lego_token_logprobs_workspace says %lld", (long long)workspace_words,
                 (long long)lego_token_logprobs_workspace(rows, items, dtype, k));
    LEGO_REQUIRE((int64_t)rows * p.chunks < (1ll << 31), "lego_token_logprobs_fwd: %d rows in %d chunks", rows, p.chunks);
    const Wanted w{targets, targets_64};
    const Outputs out{logp, entropy, lse, top, index};
    u64* work = (u64*)workspace;
    const dim3 grid((unsigned)((int64_t)rows * p.chunks));
#define GO(MASK) hipLaunchKernelGGL((logprobs_fwd_kernel<T, MASK>), grid, dim3(LP_THREADS), 0, ST, (const T*)logits, ld, mask, mask_ld, w, out, work, items, k, \
                                    p.chunks, p.per)
    LEGO_BY_TYPE(dtype, {
        if (mask != nullptr) GO(true); else GO(false);
        if (p.chunks > 1)
            hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3(rows), dim3(LP_THREADS), 0, ST, (const T*)logits, ld, mask, mask_ld, w, out, work,
                               work + (int64_t)rows * p.chunks * (2 + k), items, k, p.chunks);
    });
#undef GO
    return check_launch("lego_token_logprobs_fwd");
}

extern "C" int lego_token_logprobs_bwd(const void* logits, int64_t ld, int dtype, const uint8_t* mask, int64_t mask_ld, const void* targets, int targets_64,
                                       int k, const float* lse, const float* entropy, const int32_t* index, const float* g_logp, const float* g_entropy,
                                       const float* g_top, void* dlogits, int rows, int items, void* stream) {
    if (int rc = logprobs_check("lego_token_logprobs_bwd", dtype, rows, items, k)) return rc;
    if (rows == 0) return 0;
    LEGO_REQUIRE(logits && lse && entropy && dlogits && (g_top == nullptr || (k > 0 && index)), "lego_token_logprobs_bwd: NULL operand");
    const LogprobPlan p = bwd_plan(items, dtype);
    LEGO_REQUIRE((int64_t)rows * p.chunks < (1ll << 31), "lego_token_logprobs_bwd: %d rows in %d chunks", rows, p.chunks);
    const Wanted w{targets, targets_64};
    const Grads g{g_logp, g_entropy, g_top};
    const dim3 grid((unsigned)((int64_t)rows * p.chunks));
#define GO(MASK) hipLaunchKernelGGL((logprobs_bwd_kernel<T, MASK>), grid, dim3(LP_THREADS), 0, ST, (const T*)logits, ld, mask, mask_ld, w, lse, entropy, index, g, \
                                    (T*)dlogits, items, k, p.chunks, p.per)
    LEGO_BY_TYPE(dtype, { if (mask != nullptr) GO(true); else GO(false); });
#undef GO
    return check_launch("lego_token_logprobs_bwd");
}
