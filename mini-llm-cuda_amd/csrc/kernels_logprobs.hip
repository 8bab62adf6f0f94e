// Log probabilities of given tokens, entropy and most likely tokens of rows of logits (mlh_logprobs_device).
//
// One pass over a row.  A thread keeps its running maximum m, the sum s of exp((x - m) / T) and the sum t of that times its exponent; a larger maximum scales both.  Threads, waves and
// parts of a row are joined by the same rule.  For the top tokens a thread also notes the largest of every 32 elements it has seen (a group).  The k-th largest of the threads' maxima is
// a bound that k tokens reach, so only groups that reach it can hold one of the k most likely: about as many groups as tokens are asked for.  Those are read again, their elements
// that reach the bound are ranked by counting how many are larger, and the row is done.
// A row is a workgroup's, or, few and long ones, cut into parts, whose sums and groups a second launch takes up with a workgroup a row.
#include <math.h>

#include <algorithm>

#include "kv_cache.h"

#define LP_WG 256
#define LP_WAVES (LP_WG / 64)
#define LP_CHUNK 16                            // elements a thread takes at once
#define LP_FLUSH 8                             // chunks whose share of the entropy's sum is one in fp32
#define LP_GROUP 32                            // ... and whose largest it notes
#define LP_UNIT (LP_WG * LP_GROUP)             // elements of which every thread has a group; parts are whole units
#define LP_GROUPS 16                           // groups of a thread, at most, where one workgroup has a row
#define LP_TOP 64
#define LP_CANDS (LP_TOP * LP_GROUP)           // elements that are ranked, at most
#define LP_PAD 8
#define LP_PARTS 64                            // of a row, at most

struct LpArgs {
    const void* logits;
    long long stride;
    const int32_t* tokens;
    float *logProb, *entropy;
    int32_t* topIds;
    float* topLogProb;
    int rows, vocab, given, top;
    double inv;  // 1 / temperature
    float scale; // ... times log2(e)
    int parts, partGranules, units; // units: of a row, at most
    unsigned char* work;            // with parts: what they leave
};
struct LpSums { double s; float m, t; }; // of a part; behind those of all parts the ranks of the groups, [rows][units][LP_WG]
__device__ __forceinline__ uint32_t* lp_ranks(const LpArgs& A, int row) { return reinterpret_cast<uint32_t*>(A.work + (size_t)A.rows * A.parts * sizeof(LpSums)) + (size_t)row * A.units * LP_WG; }

template <typename T> struct LpType;
template <> struct LpType<float> { static constexpr int V = 4; };
template <> struct LpType<bf16_t> { static constexpr int V = 8; };
template <> struct LpType<f16_t> { static constexpr int V = 8; };

__device__ __forceinline__ float lp_get(const float* p) { return *p; }
__device__ __forceinline__ float lp_get(const bf16_t* p) { return kv_bf16(*p); }
__device__ __forceinline__ float lp_get(const f16_t* p) { return kv_half(p->bits); }
// element i of 16 bytes
__device__ __forceinline__ float lp_elem(const kv_u32x4& v, int i, float) { return __uint_as_float(v[i]); }
__device__ __forceinline__ float lp_elem(const kv_u32x4& v, int i, bf16_t) { return i & 1 ? __uint_as_float(v[i >> 1] & 0xffff0000u) : kv_bf16(v[i >> 1] & 0xffffu); }
__device__ __forceinline__ float lp_elem(const kv_u32x4& v, int i, f16_t) { return kv_half(i & 1 ? v[i >> 1] >> 16 : v[i >> 1] & 0xffffu); }

// What a token is ranked by: the larger the likelier, of equal logits the lower id.  NaN counts as -infinity, and the zeros are equal.  0 is no token.
__device__ __forceinline__ uint32_t lp_rank(float x) {
    if (!(x > -INFINITY)) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t lp_key(uint32_t rank, int id) { return (uint64_t)rank << 32 | (uint32_t)~id; }
__device__ __forceinline__ int lp_id(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float lp_value(uint64_t key) {
    const uint32_t r = (uint32_t)(key >> 32);
    return __uint_as_float((r & 0x80000000u) ? r & 0x7fffffffu : ~r);
}

// (m, s, t) as seen from a maximum `to` that is not smaller; the factor.  Nothing seen: m is -infinity and s and t are 0.
template <typename E> __device__ __forceinline__ float lp_scale(float& m, double& s, E& t, float to, float scale) {
    if (!(m < to)) return 1.f;
    const float d = fmaxf((m - to) * scale, -1e4f), f = __builtin_amdgcn_exp2f(d); // (2^-1e4 is 0; an infinity would make NaN of 0)
    t = f * fma((E)s, (E)d, t);
    s *= f;
    m = to;
    return f;
}

// A row's granules of 16 bytes; the first and the last may hold elements of other rows.
struct LpRow {
    const kv_u32x4* at;
    int lead, granules, vocab;
};
template <typename T> __device__ __forceinline__ LpRow lp_row(const LpArgs& A, int row) {
    constexpr int V = LpType<T>::V;
    const T* x = (const T*)A.logits + (size_t)row * A.stride;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));
    return {(const kv_u32x4*)(x - lead), lead, (A.vocab + lead + V - 1) / V, A.vocab};
}

// Sums and maxima over a wave, in its last lane: row_shr 1, 2, 4, 8, then row_bcast 15 and 31.  `none`: what a lane without a partner takes.
template <typename T, int CTRL, typename F> __device__ __forceinline__ T lp_step(T v, T none, F f) {
    T o;
    if constexpr (sizeof(T) == 8) {
        const uint64_t x = __builtin_bit_cast(uint64_t, v), n = __builtin_bit_cast(uint64_t, none);
        const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)n, (int)(uint32_t)x, CTRL, 0xf, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp((int)(n >> 32), (int)(x >> 32), CTRL, 0xf, 0xf, false);
        o = __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else
        o = __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
    return f(v, o);
}
template <typename T, typename F> __device__ __forceinline__ T lp_wave(T v, T none, F f) {
    v = lp_step<T, 0x111>(v, none, f);
    v = lp_step<T, 0x112>(v, none, f);
    v = lp_step<T, 0x114>(v, none, f);
    v = lp_step<T, 0x118>(v, none, f);
    v = lp_step<T, 0x142>(v, none, f);
    return lp_step<T, 0x143>(v, none, f);
}
__device__ __forceinline__ uint32_t lp_last(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ float lp_last(float v) { return __uint_as_float(lp_last(__float_as_uint(v))); }
__device__ __forceinline__ float lp_wave_max(float v) { return lp_last(lp_wave(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); })); }
template <typename T> __device__ __forceinline__ T lp_wave_sum(T v) { return lp_wave(v, T(0), [](T a, T b) { return a + b; }); } // (in lane 63)

// The sum of the threads' counts.  Two calls in a row take different slots.
__device__ __forceinline__ int lp_count(int mine, int* slot) {
    const int sum = lp_wave_sum(mine);
    if ((threadIdx.x & 63) == 63) slot[threadIdx.x >> 6] = sum;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int i = 0; i < LP_WAVES; i++) n += slot[i];
    return n;
}

// Ranks the n keys in cand (all different; written before a barrier; with room for LP_PAD more) and puts the first `top` of them into best, in order.  More than LP_WG are first cut down to few more than top, by
// bisection.  All threads; best is whole after a barrier.
__device__ void lp_best(uint64_t* cand, int n, int top, int (*slot)[LP_WAVES], uint64_t* best) {
    uint64_t least = 0;
    if (threadIdx.x < LP_PAD) cand[n + threadIdx.x] = 0;
    __syncthreads();
    if (n > LP_WG) {
        uint64_t lo = 0, hi = ~0ull; // as many as top reach lo, not hi
        for (int step = 0, seen = n; seen > top + 32 && hi - lo > 1; step++) {
            const uint64_t mid = lo + (hi - lo) / 2;
            int mine = 0;
            for (int i = threadIdx.x; i < n; i += LP_WG) mine += cand[i] >= mid;
            const int c = lp_count(mine, slot[step & 1]);
            if (c >= top) { lo = mid; seen = c; } else hi = mid;
        }
        least = lo;
    }
    for (int i = threadIdx.x; i < n; i += LP_WG) {
        const uint64_t key = cand[i];
        if (key < least) continue;
        int r = 0;
        for (int j = 0; j < n; j += LP_PAD) { // (one after the other, each would wait for the LDS by itself)
            uint64_t other[LP_PAD];
#pragma unroll
            for (int q = 0; q < LP_PAD; q++) other[q] = cand[j + q];
#pragma unroll
            for (int q = 0; q < LP_PAD; q++) r += other[q] > key;
        }
        if (r < top) best[r] = key;
    }
}

template <int GROUPS> struct LpTops {
    union {
        uint32_t group[GROUPS][LP_WG];    // rank of the largest of every group; 0: none
        uint64_t cand[LP_CANDS + LP_PAD]; // (once the groups that matter are known)
    };
    uint32_t most[LP_WG];
    uint64_t best[LP_TOP];
    int list[LP_TOP];
    int count, found, seen;
    uint32_t bound;
    int slot[2][LP_WAVES];
};

// The elements of granule g of a row that belong to it
template <typename T, typename F> __device__ __forceinline__ void lp_granule(const LpRow& R, int g, F f) {
    constexpr int V = LpType<T>::V;
    const kv_u32x4 v = R.at[g];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int id = g * V - R.lead + i;
        if (id >= 0 && id < R.vocab) f(lp_elem(v, i, T{}), id, i);
    }
}

// sh.best: the row's most likely tokens.  group: the ranks of its groups, [groups][LP_WG] (in LDS they are sh.group, and lost), of which a thread has every LP_WG-th, or (WIDE) four
// in every 4 * LP_WG; `mine`: the largest of this thread's.  All threads; whole after a barrier.  (Few workgroups run this, once each, so that fetching the code counts: loops are not unrolled
// but where loads have to be on their way together.)
template <typename T, bool WIDE, int GROUPS> __device__ void lp_tops(LpTops<GROUPS>& sh, const LpRow& R, int groups, const uint32_t* group, uint32_t mine, int top) {
    constexpr int V = LpType<T>::V, U = LP_GROUP / V; // granules of a group
    const int t = threadIdx.x;
    sh.most[t] = mine;
    if (t == 0) sh.count = sh.found = 0;
    __syncthreads();
    if (t < 64) { // a bound that at least top threads reach, and not many more
        uint32_t b[LP_WAVES], lo = ~0u, hi = 0u;
#pragma unroll
        for (int i = 0; i < LP_WAVES; i++) { b[i] = sh.most[i * 64 + t]; lo = min(lo, b[i]); hi = max(hi, b[i]); }
        hi = lp_last(lp_wave(hi, 0u, [](uint32_t a, uint32_t c) { return max(a, c); })) + 1;
        lo = lp_last(lp_wave(lo, ~0u, [](uint32_t a, uint32_t c) { return min(a, c); }));
        const auto reach = [&](uint32_t least) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < LP_WAVES; i++) c += __builtin_popcountll(__ballot(b[i] >= least));
            return c;
        };
        if (top == 1) lo = hi - 1;
        if (reach(lo + 1) < top) hi = lo + 1; // (masked tokens fill most threads, or top is 1)
        int seen = reach(lo);
        while (seen > top + top / 4 && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int c = reach(mid);
            if (c >= top) { lo = mid; seen = c; } else hi = mid;
        }
        if (t == 0) {
            sh.bound = max(lo, 1u);
            sh.seen = lo ? seen : 0;
        }
    }
    __syncthreads();
    uint32_t bound = sh.bound;
    const auto each = [&](auto f) { // four of this thread's groups at a time: f(ranks, index of the first, from one to the next)
        if constexpr (WIDE) {
#pragma unroll 1
            for (int at = t * 4; at < groups * LP_WG; at += LP_WG * 4) f(*reinterpret_cast<const kv_u32x4*>(group + at), at, 1);
        } else {
#pragma unroll 1
            for (int at = t; at < groups * LP_WG; at += LP_WG * 4) {
                kv_u32x4 r;
#pragma unroll
                for (int e = 0; e < 4; e++) r[e] = at + e * LP_WG < groups * LP_WG ? group[at + e * LP_WG] : 0u;
                f(r, at, LP_WG);
            }
        }
    };
    const auto list = [&](uint32_t least) { // this thread's groups that reach it
        each([&](kv_u32x4 r, int at, int by) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (r[e] >= least) {
                    const int i = atomicAdd(&sh.count, 1);
                    if (i < LP_TOP) sh.list[i] = at + e * by;
                }
        });
    };
    bool many = sh.seen > LP_TOP; // (threads that are equal at the bound)
    if (!many) {
        if (mine >= bound) list(bound);
        __syncthreads();
        many = sh.count > LP_TOP;
    }
    if (many) { // a bound that at least top groups reach and at most LP_TOP; if there is none, the top-th largest group itself: fewer than top are larger
        uint32_t lo = bound, hi = ~0u;
        for (int step = 0; many && hi - lo > 1; step++) {
            const uint32_t mid = step == 0 ? lo + 1 : lo + (hi - lo) / 2; // (most often masked tokens are what is at the bound)
            int c = 0;
            if (mine >= mid)
                each([&](kv_u32x4 r, int, int) {
#pragma unroll
                    for (int e = 0; e < 4; e++) c += r[e] >= mid;
                });
            c = lp_count(c, sh.slot[step & 1]);
            if (c >= top) lo = mid; else hi = mid;
            many = c < top || c > LP_TOP;
        }
        bound = lo;
        if (t == 0) sh.count = 0;
        __syncthreads();
        if (mine >= bound) list(many ? bound + 1 : bound);
        __syncthreads();
    }
    const int listed = sh.count;
    for (int i = t; i < listed * U; i += LP_WG) {
        const int where = sh.list[i / U], g = ((where >> 8) * U + i % U) * LP_WG + (where & 255);
        if (g < R.granules) {
            uint64_t keys[V];
            uint32_t those = 0;
            lp_granule<T>(R, g, [&](float x, int id, int e) {
                const uint32_t r = lp_rank(x);
                keys[e] = lp_key(r, id);
                those |= (uint32_t)(r >= bound + many) << e; // (no rank is 2^32 - 1)
            });
            if (those) {
                int at = atomicAdd(&sh.found, __builtin_popcount(those));
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (those >> e & 1) sh.cand[at++] = keys[e];
            }
        }
    }
    __syncthreads();
    int n = sh.found;
    if (many && n < top) { // of those that equal the bound the first ones: granule by granule in the order of ids
        int need = top - n;
        for (int g0 = 0, step = 0; g0 < R.granules && need > 0; g0 += LP_WG, step++) {
            const int g = g0 + t;
            uint32_t equal = 0;
            if (g < R.granules) lp_granule<T>(R, g, [&](float x, int, int e) { equal |= (uint32_t)(lp_rank(x) == bound) << e; });
            int before = __builtin_popcount(equal);
            const int own = before;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(before, o, 64);
                if ((t & 63) >= o) before += v;
            }
            if ((t & 63) == 63) sh.slot[step & 1][t >> 6] = before;
            before -= own;
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int i = 0; i < LP_WAVES; i++) {
                if (i < t >> 6) before += sh.slot[step & 1][i];
                all += sh.slot[step & 1][i];
            }
            while (equal && before < need) {
                const int i = __builtin_ctz(equal);
                equal &= equal - 1;
                sh.cand[n + before++] = lp_key(bound, g * V - R.lead + i);
            }
            const int took = min(all, need);
            n += took;
            need -= took;
        }
        __syncthreads();
    }
    lp_best(sh.cand, n, top, sh.slot, sh.best);
}

// What a row's maximum and sums come to: its entropy, its given tokens, and the logarithm of its sum, which its most likely tokens need.  One wave.
__device__ __forceinline__ double lp_finish(const LpArgs& A, int row, float m, double s, float ent, int token, float given) {
    const int lane = threadIdx.x & 63;
    const double logz = m > -INFINITY ? log(s) : NAN;
    if (lane == 0 && A.entropy) A.entropy[row] = (float)(logz - (double)ent * 0.69314718055994530942 / s);
    if (lane < A.given) A.logProb[(size_t)row * A.given + lane] = token < 0 ? 0.f : token >= A.vocab ? NAN : (float)(((double)given - (double)m) * A.inv - logz);
    return logz;
}
// Its most likely tokens: the first wave, one thread a token.
__device__ __forceinline__ void lp_finish_top(const LpArgs& A, int row, float m, double logz, const uint64_t* best) {
    const int t = threadIdx.x;
    if (t < A.top) {
        const uint64_t key = best[t];
        A.topIds[(size_t)row * A.top + t] = lp_id(key);
        A.topLogProb[(size_t)row * A.top + t] = (float)(((double)lp_value(key) - (double)m) * A.inv - logz);
    }
}

// What bounds it: many rows memory (8192 of 50257 in bf16, 823 MB: 148 to 153 us, 5.4 to 5.6 TB/s), with the instructions for 16 exponentials a chunk close behind (162 with a maximum over the wave for every chunk); few rows the latencies of one workgroup (a row
// of 8192 in fp32, five tokens: 6 us, of which the launch is 2).  Workgroups of 512 and 1024 threads were no faster: a compute unit takes 0.1 us for 1000 elements however they are dealt.
// Rows in parts: 64 of 131075 in bf16 15.0 to 15.5 us, of which the parts take 8.0 and the join 7.5, a row alone 3.8 and 6.9: the join waits for memory three times (ranks, groups, given tokens' logits) and for
// its own code.  Parts that picked their own top tokens took 14 + 5 us; joined by the last part to end, counted by atomics, 25 to 52.
enum { LP_SUMS, LP_WHOLE, LP_PARTLY }; // no top tokens; with them, of rows that are one workgroup's; the groups left in work
template <typename T, int KIND>
__global__ void __launch_bounds__(LP_WG, sizeof(T) == 4 ? 5 : 6) k_logprobs(LpArgs A) {
    constexpr int V = LpType<T>::V, U = LP_CHUNK / V;
    __shared__ LpTops<KIND == LP_WHOLE ? LP_GROUPS : 1> sh;
    __shared__ LpSums of[LP_WAVES];
    __shared__ double logz;
    __shared__ float rowMax, given[64];
    __shared__ int token[64];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const unsigned items = (unsigned)A.rows * A.parts; // (2^30 at most)
    for (unsigned item = blockIdx.x; item < items; item += gridDim.x) {
        const int row = (int)(item / A.parts), part = (int)(item % A.parts);
        const LpRow R = lp_row<T>(A, row);
        const int first = min(part * A.partGranules, R.granules), end = min(first + A.partGranules, R.granules);
        const int chunks = (end - first + LP_WG * U - 1) / (LP_WG * U);
        kv_u32x4 next[U];
        const auto load = [&](int j) {
            const int g0 = first + j * LP_WG * U + t;
#pragma unroll
            for (int u = 0; u < U; u++) next[u] = R.at[min(g0 + u * LP_WG, end - 1)]; // (behind the end the last one again)
        };
        load(0);
        const bool whole = KIND == LP_WHOLE || (KIND == LP_SUMS && A.parts == 1);
        if (whole && wave == LP_WAVES - 1 && lane < A.given) { // (kept in LDS: the loop has no registers left)
            const int id = A.tokens[(size_t)row * A.given + lane];
            token[lane] = id;
            given[lane] = id >= 0 && id < A.vocab ? lp_get((const T*)A.logits + (size_t)row * A.stride + id) : 0.f;
        }
        uint32_t* const ranks = KIND == LP_PARTLY ? lp_ranks(A, row) + first / (LP_UNIT / V) * LP_WG + t : nullptr;
        float m = -INFINITY, ent = 0.f; // m: the wave's
        // ent's sum of the chunks before the last LP_FLUSH, where there can be more (up to 1024: of equal logits all would be rounded the same way)
        double s = 0.0, before = 0.0;
        uint32_t mine = 0;
        float grp = -INFINITY; // a group's largest, and whether it has any
        bool some = false;
        for (int j = 0; j < chunks; j++) {
            const int g0 = first + j * LP_WG * U;
            kv_u32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = next[u];
            load(j + 1);
            float x[LP_CHUNK];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < V; i++) x[u * V + i] = lp_elem(v[u], i, T{});
            bool any = true;
            if ((g0 == 0 && R.lead) || g0 + LP_WG * U >= R.granules || g0 + LP_WG * U > end) { // an end of the row or of the part
                any = g0 + t < end;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int g = g0 + u * LP_WG + t, id = g * V - R.lead, room = g < end ? R.vocab - id : 0;
#pragma unroll
                    for (int i = 0; i < V; i++) x[u * V + i] = i >= -id && i < room ? x[u * V + i] : -INFINITY;
                }
            }
            float c = x[0];
#pragma unroll
            for (int i = 1; i < LP_CHUNK; i++) c = fmaxf(c, x[i]);
            if (!(c > -INFINITY)) c = -INFINITY; // (NaN alone)
            if (KIND != LP_SUMS) {
                grp = j & 1 ? fmaxf(grp, c) : c;
                some = any || (j & 1 && some);
                if (j & 1 || j + 1 == chunks) {
                    const uint32_t rank = some ? lp_rank(grp) : 0u;
                    if (KIND == LP_WHOLE) {
                        sh.group[j / 2][t] = rank;
                        mine = max(mine, rank);
                    } else
                        ranks[j / 2 * LP_WG] = rank;
                }
            }
            const bool less = __ballot(c >= m) == 0; // (most often)
            if (!less) {
                const float cw = lp_wave_max(c);
                if (cw > m) {
                    if (KIND == LP_WHOLE) lp_scale(m, s, ent, cw, A.scale);
                    else ent *= lp_scale(m, s, before, cw, A.scale);
                }
            }
            const float from = m > -INFINITY ? m : 0.f;
            if (less) {
                float e4[2] = {}, t4[2] = {};
#pragma unroll
                for (int i = 0; i < LP_CHUNK; i++) {
                    const float d = (x[i] - from) * A.scale, e = __builtin_amdgcn_exp2f(d);
                    e4[i & 1] += e;
                    t4[i & 1] = fmaf(e, fmaxf(d, -1e4f), t4[i & 1]);
                }
                s += (double)(e4[0] + e4[1]);
                ent += t4[0] + t4[1];
            } else { // the maximum's 1 is among them, beside which fp32 would lose the others
#pragma unroll
                for (int i = 0; i < LP_CHUNK; i++) {
                    const float d = (x[i] - from) * A.scale, e = __builtin_amdgcn_exp2f(d);
                    s += (double)e;
                    ent = fmaf(e, fmaxf(d, -1e4f), ent);
                }
            }
            if (KIND != LP_WHOLE && j % LP_FLUSH == LP_FLUSH - 1) {
                before += (double)ent;
                ent = 0.f;
            }
        }
        s = lp_wave_sum(s);
        ent = lp_wave_sum(KIND == LP_WHOLE ? ent : (float)(before + (double)ent));
        if (lane == 63) of[wave] = LpSums{s, m, ent};
        if (KIND == LP_WHOLE) lp_tops<T, false>(sh, R, (chunks + 1) / 2, &sh.group[0][0], mine, A.top); // (with the barrier that the sums need)
        else __syncthreads();
        if (wave == LP_WAVES - 1) { // (it has less to rank than the first, or nothing)
            LpSums all = {0.0, -INFINITY, 0.f};
#pragma unroll
            for (int i = 0; i < LP_WAVES; i++) all.m = fmaxf(all.m, of[i].m);
#pragma unroll
            for (int i = 0; i < LP_WAVES; i++) {
                LpSums one = of[i];
                lp_scale(one.m, one.s, one.t, all.m, A.scale);
                all.s += one.s;
                all.t += one.t;
            }
            if (whole) {
                const double z = lp_finish(A, row, all.m, all.s, all.t, token[lane], given[lane]);
                if (KIND == LP_WHOLE && lane == 0) { rowMax = all.m; logz = z; }
            } else if (lane == 0)
                reinterpret_cast<LpSums*>(A.work)[item] = all;
        }
        if (KIND == LP_WHOLE) {
            __syncthreads();
            lp_finish_top(A, row, rowMax, logz, sh.best);
        }
        if (item + gridDim.x < items) __syncthreads();
    }
}

// One workgroup a row: the parts' sums, and the tokens out of the groups' ranks.
template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_WG) k_logprobs_join(LpArgs A) {
    __shared__ LpTops<1> sh;
    __shared__ double logz;
    __shared__ float rowMax;
    const int t = threadIdx.x, lane = t & 63, row = blockIdx.x;
    const bool last = t >= LP_WG - 64; // the wave that takes the sums, while the first ranks
    float given = 0.f;
    int token = -1;
    LpSums mine = {0.0, -INFINITY, 0.f};
    if (last && lane < A.given) {
        token = A.tokens[(size_t)row * A.given + lane];
        if (token >= 0 && token < A.vocab) given = lp_get((const T*)A.logits + (size_t)row * A.stride + token);
    }
    if (last && lane < A.parts) mine = reinterpret_cast<const LpSums*>(A.work)[(size_t)row * A.parts + lane];
    if (TOP) {
        constexpr int V = LpType<T>::V;
        const LpRow R = lp_row<T>(A, row);
        const int groups = (R.granules + LP_UNIT / V - 1) / (LP_UNIT / V);
        const uint32_t* ranks = lp_ranks(A, row);
        uint32_t most = 0;
        for (int at = t * 4; at < groups * LP_WG; at += LP_WG * 32) {
            kv_u32x4 r[8];
#pragma unroll
            for (int j = 0; j < 8; j++) r[j] = *reinterpret_cast<const kv_u32x4*>(ranks + min(at + j * LP_WG * 4, groups * LP_WG - 4));
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) most = max(most, at + j * LP_WG * 4 < groups * LP_WG ? r[j][e] : 0u);
        }
        lp_tops<T, true>(sh, R, groups, ranks, most, A.top);
    }
    if (last) {
        const float m = lp_wave_max(mine.m);
        lp_scale(mine.m, mine.s, mine.t, m, A.scale);
        const double s = __shfl(lp_wave_sum(mine.s), 63, 64);
        const double z = lp_finish(A, row, m, s, lp_last(lp_wave_sum(mine.t)), token, given);
        if (lane == 0) { rowMax = m; logz = z; }
    }
    if (TOP) {
        __syncthreads();
        lp_finish_top(A, row, rowMax, logz, sh.best);
    }
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
static std::string lp_check_sizes(const mlh_logprobs* a) { // what the workspace goes by
    if (!a) return "null arguments";
    if (a->type != MLH_DTYPE_F32 && a->type != MLH_DTYPE_BF16 && a->type != MLH_DTYPE_F16) return "unknown type of logits";
    if (a->rows < 0 || a->rows > (1 << 24)) return "rows must be 0 to 2^24";
    if (a->vocab < 1 || a->vocab > (1 << 22)) return "vocab must be 1 to 2^22";
    if (a->stride < a->vocab || a->stride > (1ll << 32)) return "stride smaller than vocab, or beyond 2^32";
    if (a->given < 0 || a->given > 64 || a->top < 0 || a->top > 64 || a->top > a->vocab) return "given and top must be 0 to 64, top at most vocab";
    return "";
}
static std::string lp_check(const mlh_logprobs* a) {
    const std::string bad = lp_check_sizes(a);
    if (!bad.empty()) return bad;
    if (!a->logits || (a->given && (!a->tokens || !a->logProb)) || (a->top && (!a->topIds || !a->topLogProb))) return "null pointer";
    if ((uintptr_t)a->logits % kv_elem_bytes(a->type)) return "logits must be aligned to their elements";
    if (((a->given ? (uintptr_t)a->tokens | (uintptr_t)a->logProb : 0) | (uintptr_t)a->entropy | (a->top ? (uintptr_t)a->topIds | (uintptr_t)a->topLogProb : 0)) % 4) return "tokens and results must be 4-byte aligned";
    if (a->temperature != 0.f && !(a->temperature >= 1e-4f && a->temperature <= 1e4f)) return "temperature must be 0 or 1e-4 to 1e4";
    return "";
}

// How rows are cut.  A row is one workgroup's where it can be (LP_GROUPS): a second launch costs about 4 us, and many rows fill the chip.  Few and long rows are cut into parts of as many whole
// units as keep them within 1024 workgroups (512: up to 1 us more; 64 rows of 131075 are 17 units each, two a part: 576 workgroups), since one compute unit takes 0.1 us for 1000 elements.  bf16 with the 20 most likely, us whole / cut: 1 row of 32768 10.5 / 10.7, 40000 11.9 / 10.6,
// 100000 20.6 / 11.2; 64 rows 11.2 / 11.9, 12.3 / 12.2, 21.3 / 14.3; 128 rows of 32768 11.3 / 13.1, 50000 14.4 / 13.8, 100000 21.8 / 17.1; 256 rows of 50000 14.5 / 16.9, 100000 22.8 / 23.3.
struct LpCut { int units, parts, per; bool join; }; // units: of a row; per: of a part
static LpCut lp_cut(const mlh_logprobs* a) {
    const int V = 16 / (int)kv_elem_bytes(a->type), units = (a->vocab + V - 1 + LP_UNIT - 1) / LP_UNIT;
    const bool few = a->rows <= 128 && a->vocab >= 40960;
    LpCut c = {units, 1, units, (a->top && units > LP_GROUPS) || few};
    if (c.join) {
        const int parts = std::min(std::max(1024 / std::max(a->rows, 1), 1), LP_PARTS);
        c.per = (units + parts - 1) / parts;
        c.parts = (units + c.per - 1) / c.per;
    }
    return c;
}

extern "C" uint64_t mlh_logprobs_work_bytes(const mlh_logprobs* a) {
    if (!lp_check_sizes(a).empty()) return 0;
    const LpCut c = lp_cut(a);
    return c.join ? (uint64_t)a->rows * (c.parts * sizeof(LpSums) + (a->top ? (uint64_t)c.units * LP_WG * 4 : 0)) : 0;
}

template <typename T> static int lp_go(const LpArgs& A, bool join, void* stream) {
    const dim3 grid((unsigned)std::min<long long>((long long)A.rows * A.parts, 1 << 22)), rows((unsigned)A.rows);
    const int rc = kv_launch(!A.top ? &k_logprobs<T, LP_SUMS> : join ? &k_logprobs<T, LP_PARTLY> : &k_logprobs<T, LP_WHOLE>, grid, LP_WG, 0, stream, A);
    if (rc || !join) return rc;
    return kv_launch(A.top ? &k_logprobs_join<T, true> : &k_logprobs_join<T, false>, rows, LP_WG, 0, stream, A);
}

extern "C" int mlh_logprobs_device(const mlh_logprobs* a, void* stream) {
    const std::string bad = lp_check(a);
    if (!bad.empty()) return kv_fail(bad);
    if (a->rows == 0) return 0;
    const uint64_t need = mlh_logprobs_work_bytes(a);
    if (need && (!a->work || (uintptr_t)a->work % 16 || a->workBytes < need)) return kv_fail("work must be 16-byte aligned and have mlh_logprobs_work_bytes");
    const double inv = a->temperature == 0.f ? 1.0 : 1.0 / (double)a->temperature;
    const LpCut c = lp_cut(a);
    LpArgs A = {a->logits, a->stride, a->tokens, a->logProb, a->entropy, a->topIds, a->topLogProb, a->rows, a->vocab, a->given, a->top, inv, (float)(inv * 1.4426950408889634074),
                c.parts, c.per * (LP_UNIT / (16 / (int)kv_elem_bytes(a->type))), c.units, (unsigned char*)a->work};
    if (a->type == MLH_DTYPE_F32) return lp_go<float>(A, c.join, stream);
    if (a->type == MLH_DTYPE_BF16) return lp_go<bf16_t>(A, c.join, stream);
    return lp_go<f16_t>(A, c.join, stream);
}
