// Attention over a caller's paged K/V cache (mlh_attention_device): causal, with a sliding window and first positions that stay visible, over pages of 32, 16 or 4
// bits.  Three kernels and one that joins:
//   k_kvattn_f32   rows in fp32, 16 of them a workgroup, on the fp32 matrix cores
//   k_kvattn_few   rows in 16 bits, few a sequence (single tokens): 16 a workgroup (4 or 8 over 4-bit pages, a column for each group), its waves take key tiles in turn
//   k_kvattn_many  rows in 16 bits, many a sequence (prompts): 32 a wave, key tiles through LDS
//   k_kvattn_join  the shares of workgroups that split a sequence's keys
//
// A "row" here is a query head's query: the heads of one K/V head are rows of one workgroup, so that a key is fetched once for all of them.  Row r of a sequence is
// head r % G of its query r / G, G = heads / kvHeads.
//
// All of them keep, per row, the running maximum m of the scores (times log2 e) and the sums l of 2^(s - m) and acc of 2^(s - m) v, in fp32.  What a row does not see
// has weight zero whatever the memory holds: scores are replaced by a selection, and where a tile is hidden from some row, elements of v that are no numbers are taken out of
// the product and added for the rows that see them alone (repair, below), as zero times infinity would be NaN.
#include <math.h>

#include <algorithm>

#include "kv_cache.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct KvAttnArgs {
    const void *poolK, *poolV;
    const int32_t *table, *start, *len;
    const void* q;
    void* out;
    float* part; // shares of split keys: acc [nsplit, rows * heads, HD], then (m, l) pairs [nsplit, rows * heads]
    long long qStride, outStride;
    int nseq, rows, heads, kvHeads, group, pagesPerSeq, numPages, window, sinks, nsplit;
    float scale2; // scale * log2 e
};

#define KV_NAN __uint_as_float(0x7fc00000u)

// The rows of a workgroup: nr of them from row r0 of sequence s.
struct KvBlock {
    int s, r0, nr, row0; // row0: the call's row of the sequence's first query
    int pos0;            // its position
    int minPos, maxPos;  // of the block's rows; maxPos inside the page table
    int cap;             // positions that the page table has
};

// Blocks of QB rows: those of sequence s begin at number start[s] G / QB + s, which leaves every sequence enough of them.
template <int QB> __device__ __forceinline__ bool kv_block(const KvAttnArgs& A, int blk, KvBlock& B) {
    auto first = [&](int i) { return A.start[i] * A.group / QB + i; };
    const int s = kv_find(A.nseq, blk, first);
    const int b = kv_uniform(A.start, s), e = kv_uniform(A.start, s + 1), end = min(e, A.rows);
    if (b < 0 || end <= b) return false;
    const int r0 = (blk - (b * A.group / QB + s)) * QB, all = (end - b) * A.group;
    if (r0 < 0 || r0 >= all) return false;
    B.s = s; B.r0 = r0; B.nr = min(QB, all - r0); B.row0 = b;
    B.pos0 = (int)((unsigned)kv_uniform(A.len, s) - (unsigned)e + (unsigned)b);
    B.cap = A.pagesPerSeq * MLH_KV_PAGE;
    B.minPos = max(B.pos0 + r0 / A.group, -1);
    B.maxPos = min(B.pos0 + (r0 + B.nr - 1) / A.group, B.cap - 1);
    return true;
}

// The same for calls of at most 64 sequences, the longest ones' blocks first: what starts last is short then, and the numbers without rows come behind all others
// (64 tokens over 100 to 12000 positions 316 -> 292 us, 60 chunks of up to 120 rows behind up to 2000 139 -> 108).  Beyond 64 it is the caller's order: 65 of those tokens take 342 us
// in the order of the 64, 332 when the shortest come first and 297 when the longest do.  LAST: of a sequence the last rows first, which see most.  A lane a sequence: the blocks of longer ones are before its own.  From nine on, each of the four waves looks at a quarter of them (64 tokens over 300
// each: 20 us where every wave looks at all, 17).  For workgroups of four waves, all together.
template <int QB, bool LAST = false> __device__ __forceinline__ bool kv_block_longest_first(const KvAttnArgs& A, int blk, KvBlock& B) {
    __shared__ int parts[4][64];
    if (A.nseq > 64) return kv_block<QB>(A, LAST ? (gridDim.x - 1) / A.kvHeads - blk : blk, B);
    const int lane = threadIdx.x & 63, own = min(lane, A.nseq - 1);
    const int b = A.start[own], e = A.start[own + 1], len = A.len[own];
    const int all = b < 0 || lane >= A.nseq ? 0 : max(min(e, A.rows) - b, 0) * A.group, blocks = (all + QB - 1) / QB;
    const int key = min(max(len, 0), (1 << 25) - 1) << 6 | (63 - lane); // (each another)
    const bool shared = A.nseq > 8;
    int before = 0;
    auto look = [&](int t) {
        const int k = __builtin_amdgcn_readlane(key, t), n = __builtin_amdgcn_readlane(blocks, t);
        before += k > key ? n : 0;
    };
    if (!shared) {
        for (int t = 0; t < A.nseq; t++) look(t);
    } else {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < 16; i++) look(16 * wave + i); // (lanes without a sequence have no blocks)
        parts[wave][lane] = before;
        __syncthreads();
        before = parts[0][lane] + parts[1][lane] + parts[2][lane] + parts[3][lane];
    }
    const unsigned long long who = __ballot(blk >= before && blk < before + blocks);
    if (!who) return false;
    const int s = __builtin_ctzll(who);
    const int nth = blk - __builtin_amdgcn_readlane(before, s), r0 = (LAST ? __builtin_amdgcn_readlane(blocks, s) - 1 - nth : nth) * QB;
    B.s = s; B.r0 = r0; B.nr = min(QB, __builtin_amdgcn_readlane(all, s) - r0); B.row0 = __builtin_amdgcn_readlane(b, s);
    B.pos0 = (int)((unsigned)__builtin_amdgcn_readlane(len, s) - (unsigned)__builtin_amdgcn_readlane(e, s) + (unsigned)B.row0);
    B.cap = A.pagesPerSeq * MLH_KV_PAGE;
    B.minPos = max(B.pos0 + r0 / A.group, -1);
    B.maxPos = min(B.pos0 + (r0 + B.nr - 1) / A.group, B.cap - 1);
    return true;
}

// The key tiles of TK positions that a block's rows see something of: the first positions' and the window's.
template <int TK> struct KvTiles {
    int firsts, skip, n;
    __device__ __forceinline__ KvTiles(const KvAttnArgs& A, const KvBlock& B) {
        const int low = A.window ? max(B.minPos + 1 - A.window, 0) / TK : 0;
        firsts = A.window ? min(low, (min(A.sinks, B.maxPos + 1) + TK - 1) / TK) : 0;
        firsts = max(firsts, 0);
        skip = low - firsts;
        n = B.maxPos < 0 ? 0 : max(B.maxPos / TK + 1 - skip, 0);
    }
    __device__ __forceinline__ int at(int i) const { return i < firsts ? i : i + skip; }
};

// what a row sees: positions up to `pos`, above `below` or among the first `sinks`
struct KvSight {
    int pos, below, sinks;
    int low;       // without the first ones: positions low .. low + span
    unsigned span;
    __device__ __forceinline__ KvSight(const KvAttnArgs& A, int p) : pos(p), below(A.window ? max(p, -1) - A.window : -1), sinks(A.sinks) {
        const int l = max(below + 1, 0);
        low = p < l ? 0x7fffffff : l;
        span = p < l ? 0u : (unsigned)(p - l);
    }
    __device__ __forceinline__ bool sees(int j) const { return (j <= pos) & ((j > below) | (j < sinks)); } // (without branches)
};
// do all rows of [minPos, maxPos] see all of a tile's n positions from j0?
__device__ __forceinline__ bool kv_all_see(const KvAttnArgs& A, int minPos, int maxPos, int j0, int n) {
    return j0 + n - 1 <= minPos && (!A.window || j0 > maxPos - A.window || j0 + n <= A.sinks);
}

__device__ __forceinline__ bool kv_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float kv_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
// The larger of two (as a median: fmaxf would first quiet both, an instruction each; where one is no number, either, and the row's sum is none then)
__device__ __forceinline__ float kv_max(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }
// The running maximum follows when a weight is 2^8 times beyond that of the last one and not before: with every new maximum, of 32 rows some have one in most tiles, and sums and
// result are multiplied again (the prompts below: 1071 and 171 us for 1017 and 158).
#define KV_SLACK 8.f
// m is the maximum less KvRaise: a weight is 2^KvRaise at a new maximum, and up to 2^(KvRaise + KV_SLACK) before there is another.
// Halves: 2^7, the largest then 2^15, so that half of their smallest step, which is what a weight is off by at least, is 2^-32 of the largest weight.  (With 1 for 2^7, of one key and 60000
// others whose scores are 17 lower, 0.0025 of the result in all, each counted 1.4 times or not at all.)  bf16, which has room below: 2^-8, no weight above one, so that
// sums stay as far from the end of fp32's range as they can.
template <bool BF> struct KvRaise { static constexpr float value = BF ? -KV_SLACK : 7.f; };
__device__ __forceinline__ float kv_halves_max(float v) { // of a lane and the one 32 further
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return kv_max(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float kv_quad_max(float v) { // over the four lanes that hold a column of a 16 x 16 product
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return kv_halves_max(kv_max(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float kv_quad_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ void kv_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void kv_put(bf16_t* p, float v) { *p = (bf16_t)kv_to_bf16(v); }
__device__ __forceinline__ void kv_put(f16_t* p, float v) { p->bits = (uint16_t)kv_to_half(v); }

template <typename T> __device__ __forceinline__ void kv_put4(T* p, const f32x4& v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else if constexpr (KvType<T>::code == MLH_DTYPE_BF16) *reinterpret_cast<uint2*>(p) = make_uint2(kv_to_bf16(v.x) | kv_to_bf16(v.y) << 16, kv_to_bf16(v.z) | kv_to_bf16(v.w) << 16);
    else *reinterpret_cast<uint2*>(p) = make_uint2(kv_to_half(v.x) | kv_to_half(v.y) << 16, kv_to_half(v.z) | kv_to_half(v.w) << 16);
}

// one element of a page, as a float
template <typename CT, int HD> __device__ __forceinline__ float kv_one(const void* pool, int page, int at, int kvHeads, int kh, int d) {
    if constexpr (KvType<CT>::code == MLH_CACHE_Q4) {
        const uint8_t* tile = (const uint8_t*)pool + ((size_t)page * kvHeads + kh) * kv_tile_bytes(HD);
        const uint32_t code = (uint32_t)tile[at * (HD / 2) + d / 2] >> (4 * (d & 1)) & 15u;
        const uint32_t par = *reinterpret_cast<const uint32_t*>(tile + kv_param_at(HD) + (at * (HD / KV_GROUP) + d / KV_GROUP) * 4);
        return fmaf((float)code, kv_half(par >> 16), kv_half(par & 0xffffu));
    } else {
        const CT* p = (const CT*)pool + (((size_t)page * MLH_KV_PAGE + at) * kvHeads + kh) * HD + d;
        if constexpr (sizeof(CT) == 4) return *p;
        else if constexpr (KvType<CT>::code == MLH_DTYPE_BF16) return kv_bf16(*p);
        else return kv_half(p->bits);
    }
}

// The elements of a row of V that are no numbers, zeros for the others, as floats into HD places of the wave's own: for the repair of a tile, by one key at a time.
template <typename CT, int HD, bool HALVES> __device__ __forceinline__ void kv_odd_row(const KvAttnArgs& A, int page, int at, int kh, float* place) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int d = threadIdx.x & 63; d < HD; d += 64) {
        float x = kv_one<CT, HD>(A.poolV, page, at, A.kvHeads, kh, d);
        if (HALVES) x = (float)(_Float16)x;
        place[d] = kv_finite(x) ? 0.f : x;
    }
    __builtin_amdgcn_wave_barrier(); // (LDS serves a wave's accesses in order)
}

// The end of the 16-row kernels: acc of every wave (block b, element i of lane 16 g + n: row n, element dim(b, 4 g + i)), its m and l (of row n), joined over the waves, and
// written as the row's result or, with split keys, as this workgroup's share.  lds: NW * 16 * (HD + 4 + 2) floats.  SP: columns of a row, all alike.
template <typename IT, int HD, int NW, int SP, typename F>
__device__ __forceinline__ void kv_finish16(const KvAttnArgs& A, const KvBlock& B, int kh, int split, const f32x4 (&acc)[HD / 16], float m, float l, float* lds, F dim4) {
    constexpr int LDO = HD + 4;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = lane & 15, g = lane >> 4;
    float (*part)[16][LDO] = reinterpret_cast<float (*)[16][LDO]>(lds);
    float (*stat)[2][16] = reinterpret_cast<float (*)[2][16]>(lds + NW * 16 * LDO);
    if (g == 0 && n % SP == 0) { stat[wave][0][n / SP] = m; stat[wave][1][n / SP] = l; }
    dim4([&](int d, const f32x4& v) { *reinterpret_cast<f32x4*>(&part[wave][n / SP][d]) = v; });
    __syncthreads();
    for (int i = tid; i < B.nr * (HD / 4); i += NW * 64) {
        const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
        float M = -INFINITY, den = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, stat[w][0][r]);
        const float ref = M == -INFINITY ? 0.f : M;
        f32x4 o = (f32x4)(0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = kv_exp2(stat[w][0][r] - ref);
            den = fmaf(stat[w][1][r], f, den);
            o += *reinterpret_cast<const f32x4*>(&part[w][r][d]) * f;
        }
        const int qi = (B.r0 + r) / A.group, h = kh * A.group + (B.r0 + r) % A.group, row = B.row0 + qi;
        if (B.pos0 + qi >= B.cap) { den = KV_NAN; M = 0.f; } // (its own position is behind the page table)
        if (B.pos0 + qi < 0) { den = 1.f; M = 0.f; } // sees nothing: o is zero.  (Every other row sees itself: no weight at all means that each score is -infinity, and 0 / 0 is what that is)
        if (A.nsplit > 1) {
            const size_t rh = (size_t)split * A.rows * A.heads + (size_t)row * A.heads + h;
            *reinterpret_cast<f32x4*>(A.part + rh * HD + d) = o;
            if (d == 0) *reinterpret_cast<float2*>(A.part + (size_t)A.nsplit * A.rows * A.heads * HD + rh * 2) = make_float2(M, den);
        } else {
            if constexpr (sizeof(IT) == 4) o = f32x4{o.x / den, o.y / den, o.z / den, o.w / den}; // (a division's rounding, not a product's with a rounded inverse)
            else o = o * (1.0f / den);
            kv_put4((IT*)A.out + (size_t)row * A.outStride + (size_t)h * HD + d, o);
        }
    }
}

// ----------------------------------------------------------------------------
// fp32 rows.  Products on v_mfma_f32_16x16x4_f32: S^T[key, row] = K . Q^T, then O^T += V^T . P^T, K and V from the pages straight into registers in 16-byte pieces:
// lane 16 g + n holds elements [g HD/4, (g + 1) HD/4) of key n (the order of a contraction is free), the product leaves it the scores of keys 4 g .. 4 g + 3 of row n,
// which is the second product's operand as it stands; row m of V's operand of block b is element m HD/16 + b.  The waves take tiles of 16 keys in turn, the next tile's loads
// go out before this one's products.
// Three sequences of 100, 308 and 517 rows, 6 heads of 128, window 200: 19 us, of which 4 are products (348 workgroups on 256 compute units: what a workgroup waits for,
// start, page, first tile, bounds it).  One token over 256 positions of 12 heads of 64: 8 us, the same latencies.  Eight waves a workgroup: 24 and 8 us.
// ----------------------------------------------------------------------------
// Keeps a lane's 32-bit offset one: widened outside of the loop, it would be added to each page's base in vector registers, and these wait for the loads that use them.
__device__ __forceinline__ void kv_offset(unsigned& o) { asm volatile("" : "+v"(o)); }
template <typename CT, int HD> struct KvTile32 { // a lane's part of 16 keys
    static constexpr int KC = HD / 4, VB = HD / 16;
    f32x4 k[KC / 4], v[4][VB / 4];
    struct Lane {
        unsigned ko, vo;
        __device__ __forceinline__ Lane(const KvAttnArgs& A, int n, int g) : ko(n * (unsigned)A.kvHeads * HD * 4 + g * KC * 4), vo(4 * g * (unsigned)A.kvHeads * HD * 4 + n * VB * 4) {}
    };
    // (a page's base is the same for all lanes and a lane's offset the same for all tiles: no address arithmetic in vector registers.  Rows behind the last position
    // are read as they are, a page being whole, and weigh nothing.)
    __device__ __forceinline__ void fetch(const KvAttnArgs& A, int page, int at, int kh, Lane& lane) {
        const unsigned row = (unsigned)A.kvHeads * HD * 4;
        kv_offset(lane.ko); kv_offset(lane.vo);
        const size_t base = ((size_t)page * MLH_KV_PAGE + at) * row + (size_t)kh * HD * 4;
        const char *bk = (const char*)A.poolK + base, *bv = (const char*)A.poolV + base;
#pragma unroll
        for (int c = 0; c < KC / 4; c++) k[c] = *reinterpret_cast<const f32x4*>(bk + lane.ko + 16 * c);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < VB / 4; c++) v[i][c] = *reinterpret_cast<const f32x4*>(bv + (size_t)i * row + lane.vo + 16 * c);
    }
    __device__ __forceinline__ void values(f32x4 (&ko)[KC / 4], f32x4 (&vo)[4][VB / 4]) const {
#pragma unroll
        for (int c = 0; c < KC / 4; c++) ko[c] = k[c];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < VB / 4; c++) vo[i][c] = v[i][c];
    }
};
template <int HD> struct KvTile32<q4_t, HD> {
    static constexpr int KC = HD / 4, VB = HD / 16;
    uint32_t k[KC / 8], kp, v[4], vp[4];
    struct Lane {
        unsigned ko, kpo, vo, vpo;
        __device__ __forceinline__ Lane(const KvAttnArgs&, int n, int g)
            : ko(n * (HD / 2) + g * (KC / 2)), kpo((n * (HD / KV_GROUP) + g * KC / KV_GROUP) * 4), vo(4 * g * (HD / 2) + n * (VB / 2)), vpo((4 * g * (HD / KV_GROUP) + n * VB / KV_GROUP) * 4) {}
    };
    __device__ __forceinline__ void fetch(const KvAttnArgs& A, int page, int at, int kh, Lane& lane) {
        const size_t base = ((size_t)page * A.kvHeads + kh) * kv_tile_bytes(HD);
        const uint8_t *tk = (const uint8_t*)A.poolK + base + at * (HD / 2), *tv = (const uint8_t*)A.poolV + base + at * (HD / 2);
        const uint8_t *pk = (const uint8_t*)A.poolK + base + kv_param_at(HD) + at * (HD / KV_GROUP) * 4, *pv = (const uint8_t*)A.poolV + base + kv_param_at(HD) + at * (HD / KV_GROUP) * 4;
        kv_offset(lane.ko); kv_offset(lane.kpo); kv_offset(lane.vo); kv_offset(lane.vpo);
#pragma unroll
        for (int c = 0; c < KC / 8; c += 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(tk + lane.ko + 4 * c);
            k[c] = w.x; k[c + 1] = w.y;
        }
        kp = *reinterpret_cast<const uint32_t*>(pk + lane.kpo);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (HD == 128) v[i] = *reinterpret_cast<const uint32_t*>(tv + lane.vo + i * (HD / 2));
            else v[i] = *reinterpret_cast<const uint16_t*>(tv + lane.vo + i * (HD / 2));
            vp[i] = *reinterpret_cast<const uint32_t*>(pv + lane.vpo + i * (HD / KV_GROUP) * 4);
        }
    }
    __device__ __forceinline__ void values(f32x4 (&ko)[KC / 4], f32x4 (&vo)[4][VB / 4]) const {
#pragma unroll
        for (int c = 0; c < KC / 8; c++) {
            float x[8];
            kv_values8(k[c], kp, x);
#pragma unroll
            for (int i = 0; i < 8; i++) ko[2 * c + i / 4][i % 4] = x[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float x[8];
            kv_values8(v[i], vp[i], x);
#pragma unroll
            for (int j = 0; j < VB; j++) vo[i][j / 4][j % 4] = x[j];
        }
    }
};

#define KV_F32_WAVES 4
template <typename CT, int HD>
__global__ void __launch_bounds__(KV_F32_WAVES * 64, 2) k_kvattn_f32(KvAttnArgs A) {
    constexpr int NW = KV_F32_WAVES, KC = HD / 4, VB = HD / 16;
    __shared__ __attribute__((aligned(16))) float lds[NW * 16 * (HD + 4 + 2)];
    __shared__ float odds[NW][HD];
    const int kh = blockIdx.x % A.kvHeads, block = blockIdx.x / A.kvHeads / A.nsplit, split = blockIdx.x / A.kvHeads % A.nsplit;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    KvBlock B;
    if (!kv_block_longest_first<16>(A, block, B)) return;
    const int r = B.r0 + min(n, B.nr - 1), h = kh * A.group + r % A.group;
    const KvSight sight(A, B.pos0 + r / A.group);
    f32x4 q[KC / 4];
    {
        const float* qr = (const float*)A.q + (size_t)(B.row0 + r / A.group) * A.qStride + (size_t)h * HD + g * KC;
#pragma unroll
        for (int c = 0; c < KC / 4; c++) q[c] = *reinterpret_cast<const f32x4*>(qr + 4 * c);
    }
    f32x4 acc[VB];
#pragma unroll
    for (int b = 0; b < VB; b++) acc[b] = (f32x4)(0.f);
    float m = -INFINITY, l = 0.f; // of row n; l: over this lane's keys
    const KvTiles<16> tiles(A, B);
    KvTile32<CT, HD> raw[2];
    typename KvTile32<CT, HD>::Lane offsets(A, n, g);
    int page[2];
    int next = 0; // page of the tile to be fetched next
    auto look = [&](int i) { next = kv_page(A.table, A.pagesPerSeq, A.numPages, B.s, tiles.at(min(i, tiles.n - 1)) * 16 >> 6); };
    auto fetch = [&](int i, int set) __attribute__((always_inline)) {
        const int j0 = tiles.at(i) * 16;
        page[set] = next;
        raw[set].fetch(A, max(page[set], 0), j0 & 63, kh, offsets);
    };
    auto tile = [&](int i, int set) __attribute__((always_inline)) {
        const int j0 = tiles.at(i) * 16, key = j0 + 4 * g;
        f32x4 k[KC / 4], v[4][VB / 4];
        raw[set].values(k, v);
        f32x4 s0 = (f32x4)(0.f), s1 = (f32x4)(0.f); // two chains
#pragma unroll
        for (int c = 0; c < KC / 4; c++) {
            s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c].x, q[c].x, s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c].y, q[c].y, s1, 0, 0, 0);
            s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c].z, q[c].z, s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c].w, q[c].w, s1, 0, 0, 0);
        }
        const bool whole = kv_all_see(A, B.minPos, B.maxPos, j0, 16) && page[set] >= 0;
        float p[4], mt = m;
        bool see[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            see[e] = whole || sight.sees(key + e);
            p[e] = (s0[e] + s1[e]) * A.scale2;
            if (!whole) p[e] = !see[e] ? -INFINITY : page[set] < 0 ? KV_NAN : p[e];
            mt = kv_max(mt, p[e]);
        }
        mt = kv_quad_max(mt);
        const float ref = mt == -INFINITY ? 0.f : mt, corr = kv_exp2(m - ref);
        m = mt;
        l *= corr;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            p[e] = see[e] ? kv_exp2(p[e] - ref) : 0.f;
            l += p[e];
        }
        if (__any(corr != 1.f)) { // (a maximum that moves gets rare)
#pragma unroll
            for (int b = 0; b < VB; b++) acc[b] *= corr;
        }
        if (!whole) { // repair
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int b = 0; b < VB; b++) odd = odd || !kv_finite(v[e][b / 4][b % 4]);
            if (__ballot(odd)) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    bool odd_ = false;
#pragma unroll
                    for (int b = 0; b < VB; b++) {
                        odd_ = odd_ || !kv_finite(v[e][b / 4][b % 4]);
                        v[e][b / 4][b % 4] = kv_finite(v[e][b / 4][b % 4]) ? v[e][b / 4][b % 4] : 0.f;
                    }
                    const unsigned long long who = __ballot(odd_);
#pragma unroll 1
                    for (int gk = 0; gk < 4; gk++) {
                        const int j = j0 + 4 * gk + e;
                        if (j > B.maxPos || page[set] < 0 || !(who >> (16 * gk) & 0xffffu)) continue;
                        kv_odd_row<CT, HD, false>(A, page[set], j & 63, kh, odds[wave]);
                        const float w = __shfl(p[e], 16 * gk + n, 64);
                        const bool see_ = sight.sees(j);
#pragma unroll
                        for (int b = 0; b < VB; b++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                if (i == 0) __builtin_amdgcn_sched_barrier(0); // (few registers for what hardly happens)
                                const float x = odds[wave][(4 * g + i) * VB + b];
                                acc[b][i] += see_ && x != 0.f ? w * x : 0.f;
                            }
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int b = 0; b < VB; b++) acc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e][b / 4][b % 4], p[e], acc[b], 0, 0, 0);
    };
    const int step = NW * A.nsplit;
    int t = split * NW + wave;
    if (t < tiles.n) {
        look(t);
        fetch(t, 0);
        look(t + step);
    }
    while (t < tiles.n) { // (no further tile: the same loads again, dropped)
        fetch(min(t + step, tiles.n - 1), 1);
        look(t + 2 * step);
        __builtin_amdgcn_sched_barrier(0); // (the compiler would put the loads behind the products)
        tile(t, 0);
        t += step;
        if (t >= tiles.n) break;
        fetch(min(t + step, tiles.n - 1), 0);
        look(t + 2 * step);
        __builtin_amdgcn_sched_barrier(0);
        tile(t, 1);
        t += step;
    }
    l = kv_quad_sum(l);
    kv_finish16<float, HD, NW, 1>(A, B, kh, split, acc, m, l, lds, [&](auto put) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int b = 0; b < VB; b += 4) put((4 * g + i) * VB + b, f32x4{acc[b][i], acc[b + 1][i], acc[b + 2][i], acc[b + 3][i]});
    });
}

// ----------------------------------------------------------------------------
// Few 16-bit rows of a sequence.  A wave takes 32 keys at a time: S^T[key, row] = K . Q^T on 16x16x32 products, K from the pages straight into registers; V's
// rows go through the wave's own piece of LDS, which hands them back transposed (ds_read_b64_tr_b16: lane i of 16 gets column i of four rows), so that
// O^T += V^T . P^T takes the weights from the registers that the first product left them in.  4-bit pages: codes become halves on the way (the values
// are minimum + code * scale in halves, one rounding), all products are in halves, and rows are scaled by a power of two first.
// 16-bit pages are bound by memory: 64 tokens over 100 to 12000 positions, 32 heads on 8 of 128 in bf16, 1.59 GB, 288 us (5.5 TB/s; reads alone reach 6.1); 64 over 3000
// each 150 us.  Eight waves a workgroup, one of them a compute unit then, before the longest came first: 307 and 170 us for 316 and 156, one token over 4000 17 for 12.  4-bit
// pages by the instructions that unpack them: one token over 65000 positions, bf16, 21 us (83 MB, 3.9 TB/s; the vector ALU busy in 0.58 of the cycles, the rest is the start of 768
// workgroups of five turns); eight waves a workgroup 146 us for 116 (48 tokens, before the spread below).
// Weights are rounded to 16 bits for the second product, and summed as rounded: errors against the results' norm 2.1e-3 (bf16) and 2.8e-4 (fp16) where rounding the results alone gives
// 1.7e-3 and 2.1e-4.  In two parts they would take a second product of each; only the few rows in halves over 4-bit pages, which keep K as it is, do.
// ----------------------------------------------------------------------------
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <bool BF> __device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF> __device__ __forceinline__ uint32_t kv_pack(float a, float b) {
    if constexpr (BF) { typedef __bf16 bf16x2 __attribute__((ext_vector_type(2))); return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b}); }
    else return pack_f16(a, b);
}
template <bool BF> __device__ __forceinline__ float kv_add2(uint32_t w, float sum) { // two 16-bit numbers onto a sum
    if constexpr (BF) { typedef __bf16 bf16x2 __attribute__((ext_vector_type(2))); return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{(__bf16)1.f, (__bf16)1.f}, sum, false); }
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.f, (_Float16)1.f}, sum, false);
}
__device__ __forceinline__ u32x2 lds_transposed(const void* p) { // 4 rows x 16 columns of 16 bits from 16 lanes' addresses
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
template <bool BF> __device__ __forceinline__ bool kv_odd(const u32x4& a) { // is one of eight elements no number?
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = __builtin_bit_cast(u16x2, a.x & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, a[i] & 0x7fff7fffu));
    return __builtin_elementwise_max(m.x, m.y) >= (BF ? 0x7f80 : 0x7c00);
}
template <bool BF> __device__ __forceinline__ u32x4 kv_without_odd(u32x4 a) { // zeros instead of those
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] = ((a[i] & E) == E ? 0u : a[i] & 0xffffu) | ((a[i] >> 16 & E) == E ? 0u : a[i] & 0xffff0000u);
    return a;
}
template <int PERM> __device__ __forceinline__ float kv_neighbour(float v) { // among four lanes
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), PERM, 0xf, 0xf, true));
}
// eight codes -> halves that are whole numbers, or the values; pairs come out as elements (0, 4), (1, 5), (2, 6), (3, 7)
// (code | 1024 with the code in the lowest bits, code | 64 with it four bits higher, where a unit is sixteen of the last place: both exact, and so is taking 1024 and 64 off; the
// constants in vector registers, as one instruction masks and joins then)
__device__ __forceinline__ u32x4 kv_codes(uint32_t codes) {
    uint32_t k = 0x64006400u, j = 0x54005400u;
    asm("" : "+v"(k), "+v"(j));
    const uint32_t up = codes >> 8;
    const uint32_t w[4] = {(codes & 0x000f000fu) | k, (codes & 0x00f000f0u) | j, (up & 0x000f000fu) | k, (up & 0x00f000f0u) | j};
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const _Float16 off = i & 1 ? (_Float16)-64.f : (_Float16)-1024.f;
        o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w[i]) + f16x2{off, off});
    }
    return o;
}
// The same without taking anything off: halves below the normal ones, code * 2^-24, -20, -24, -20, which the matrix cores take as what they are.
__device__ __forceinline__ u32x4 kv_tiny(uint32_t codes) {
    const uint32_t up = codes >> 8;
    return u32x4{codes & 0x000f000fu, codes & 0x00f000f0u, up & 0x000f000fu, up & 0x00f000f0u};
}
__device__ __forceinline__ u32x4 kv_halves(uint32_t codes, uint32_t params) {
    const _Float16 base = __builtin_bit_cast(_Float16, (uint16_t)(params & 0xffffu)), scale = __builtin_bit_cast(_Float16, (uint16_t)(params >> 16));
    const f16x2 b = {base, base}, s = {scale, scale};
    u32x4 o = kv_codes(codes);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = o[i]; // (a bit cast of an element of a vector reads the first)
        o[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, w), s, b));
    }
    return o;
}

// one, two or four words
__device__ __forceinline__ void kv_words(const uint8_t* p, uint32_t (&w)[1]) { w[0] = *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ void kv_words(const uint8_t* p, uint32_t (&w)[2]) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    w[0] = x.x; w[1] = x.y;
}
__device__ __forceinline__ void kv_words(const uint8_t* p, uint32_t (&w)[4]) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = x[i];
}

// A row's power of two: largest |q| into [1, 2), so that halves hold it, as long as the scale divided by it stays above 2^-100 (what halves then lose of a row moves no
// score by 2^-70).  (0: the row holds an infinity or NaN and stays as it is.)
__device__ __forceinline__ int kv_row_exp(float most, float scale) {
    const int e = __float_as_uint(most) >> 23 & 255u;
    return e == 255 ? 0 : min(127 - max(e, 1), (int)(__float_as_uint(scale) >> 23) - 27);
}

template <typename IT, typename CT, int HD> struct KvRaw16 { // a lane's part of 32 keys: key 16 b + n, elements 32 t + 8 g ..; of V the same
    static constexpr int KS = HD / 32;
    u32x4 k[2][KS], v[2][KS];
    struct Lane {
        unsigned o;
        __device__ __forceinline__ Lane(const KvAttnArgs& A, int n, int g) : o(n * (unsigned)A.kvHeads * HD * 2 + g * 16) {}
    };
    __device__ __forceinline__ void fetch(const KvAttnArgs& A, int page, int at, int kh, Lane& lane) { // (addresses: as in KvTile32)
        const unsigned row = (unsigned)A.kvHeads * HD * 2;
        kv_offset(lane.o);
        const size_t base = ((size_t)page * MLH_KV_PAGE + at) * row + (size_t)kh * HD * 2;
        const char *bk = (const char*)A.poolK + base, *bv = (const char*)A.poolV + base;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int t = 0; t < KS; t++) k[b][t] = *reinterpret_cast<const u32x4*>(bk + (size_t)(16 * b) * row + lane.o + 64 * t);
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int t = 0; t < KS; t++) v[b][t] = *reinterpret_cast<const u32x4*>(bv + (size_t)(16 * b) * row + lane.o + 64 * t);
    }
    __device__ __forceinline__ u32x4 key(int b, int t) const { return k[b][t]; }
    __device__ __forceinline__ u32x4 val(int b, int t) const { return v[b][t]; }
};
// Rows in halves over 4-bit pages (16 rows a workgroup): rounding K's values to halves costs such rows more than all else together, so that they are multiplied as what they are, minimum +
// (high + low part of the scale) * code: parts of six and five bits times a code of four are exact in halves, two products instead of one, and the minima meet the sum of
// the row's elements (as two halves) in one product more.  (15 times a scale may be beyond the halves' range where the values are not: of the high part, whose last place is 2^-19 at
// least, a sixteenth is multiplied, exact as well, and the sum is 16 times as much; the low part is below a 32nd of the scale.)  The weights are two halves as well.  (Error of a result, normal values, 4000 keys, against its norm: 4.4e-4 with
// K, V and weights each rounded to halves, 2.8e-4 so, 2.1e-4 the rounding of the result alone.)  Rows in bf16 round their results eight times as far.
template <typename IT, typename CT> constexpr bool kv_in_parts() { return KvType<CT>::code == MLH_CACHE_Q4 && KvType<IT>::code == MLH_DTYPE_F16; }
__device__ __forceinline__ u32x4 kv_times(const u32x4& codes, uint32_t scaleBits) {
    const _Float16 f = __builtin_bit_cast(_Float16, (uint16_t)scaleBits);
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = codes[i]; // (a bit cast of an element of a vector reads the first)
        o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) * f16x2{f, f});
    }
    return o;
}
template <typename IT, int HD> struct KvRaw16<IT, q4_t, HD> { // the same, elements (HD / 4) g + 8 t .. (one group of 32, or half of one)
    static constexpr int KS = HD / 32;
    uint32_t k[2][KS], v[2][KS], kp[2], vp[2];
    struct Lane {
        unsigned o, p;
        __device__ __forceinline__ Lane(const KvAttnArgs&, int n, int g) : o(n * (HD / 2) + g * (HD / 8)), p((n * (HD / KV_GROUP) + g * (HD / 4) / KV_GROUP) * 4) {}
    };
    __device__ __forceinline__ void fetch(const KvAttnArgs& A, int page, int at, int kh, Lane& lane) {
        const size_t base = ((size_t)page * A.kvHeads + kh) * kv_tile_bytes(HD);
        kv_offset(lane.o); kv_offset(lane.p);
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint8_t *tk = (const uint8_t*)A.poolK + base + (at + 16 * b) * (HD / 2), *tv = (const uint8_t*)A.poolV + base + (at + 16 * b) * (HD / 2);
            const uint8_t *pk = (const uint8_t*)A.poolK + base + kv_param_at(HD) + (at + 16 * b) * (HD / KV_GROUP) * 4, *pv = (const uint8_t*)A.poolV + base + kv_param_at(HD) + (at + 16 * b) * (HD / KV_GROUP) * 4;
            kp[b] = *reinterpret_cast<const uint32_t*>(pk + lane.p);
            vp[b] = *reinterpret_cast<const uint32_t*>(pv + lane.p);
            kv_words(tk + lane.o, k[b]);
            kv_words(tv + lane.o, v[b]);
        }
    }
    __device__ __forceinline__ u32x4 key(int b, int t) const { return kv_halves(k[b][t], kp[b]); }
    __device__ __forceinline__ u32x4 val(int b, int t) const { return kv_halves(v[b][t], vp[b]); }
};

// SP > 1 (fp16 rows over 4-bit pages, at most 16 / SP of them a sequence): column n of the first product is row n / SP with the elements of group n % SP alone.  A sum's codes
// then share minimum and scale: codes go in as they are (kv_tiny), the scale is one multiplication a key and group in fp32 behind them, exact where the 16-row form
// needs two products, and the groups' sums meet in the neighbouring columns.  The minima meet the row's sums of elements in one product more.
// 48 tokens over up to 9000 positions, window 4096, 16 heads of 128, 389 MB: 79 us (4.9 TB/s).  48 over 4000 each: 103 us, 120 in the 16-row form; bf16 rows, whose
// 16-row form has one product, 98, and spread 4 % more.
#define KV_FEW_WAVES 4
template <typename IT, typename CT, int HD, int SP>
__global__ void __launch_bounds__(KV_FEW_WAVES * 64, KvType<CT>::code == MLH_CACHE_Q4 ? 3 : 2) k_kvattn_few(KvAttnArgs A) {
    constexpr bool FOUR = KvType<CT>::code == MLH_CACHE_Q4, BF = !FOUR && KvType<IT>::code == MLH_DTYPE_BF16; // products in bf16
    constexpr bool PARTS = kv_in_parts<IT, CT>();
    constexpr float RAISE = KvRaise<BF>::value;
    constexpr int NW = KV_FEW_WAVES, KS = HD / 32, VB = HD / 16;
    static_assert(SP == 1 || (PARTS && SP == HD / KV_GROUP), "a column for each group of a row");
    constexpr int VP = HD * 2 + 16; // bytes of a row of V in LDS: four rows start in different banks
    constexpr int LV = NW * 32 * VP, LF = NW * 16 * (HD + 4 + 2) * 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[LV > LF ? LV : LF];
    __shared__ float odds[NW][HD];
    __shared__ __attribute__((aligned(16))) uint32_t params[SP > 1 ? NW : 1][SP][36]; // of 32 keys (four more words, so that the groups' rows start in different banks)
    const int kh = blockIdx.x % A.kvHeads, block = blockIdx.x / A.kvHeads / A.nsplit, split = blockIdx.x / A.kvHeads % A.nsplit;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    KvBlock B;
    if (!kv_block_longest_first<16 / SP>(A, block, B)) return;
    const int r = B.r0 + min(n / SP, B.nr - 1), h = kh * A.group + r % A.group;
    const KvSight sight(A, B.pos0 + r / A.group);
    // the row, on its way before the first tile and looked at behind it
    u32x4 q[KS], qsum = (u32x4)(0u);
    float scale = A.scale2, x[FOUR ? KS : 1][8];
    float zero = 0.f;
    asm volatile("" : "+v"(zero)); // (a product with a half on it is one instruction)
    {
        const IT* qr = (const IT*)A.q + (size_t)(B.row0 + r / A.group) * A.qStride + (size_t)h * HD;
#pragma unroll
        for (int t = 0; t < KS; t++) {
            if constexpr (FOUR) kv_load8(qr + (HD / 4) * g + 8 * t, x[t]);
            else q[t] = *reinterpret_cast<const u32x4*>(qr + 32 * t + 8 * g);
        }
    }
    f32x4 acc[VB];
#pragma unroll
    for (int b = 0; b < VB; b++) acc[b] = (f32x4)(0.f);
    float m = -INFINITY, l = 0.f;
    unsigned char* const vt = lds + wave * 32 * VP;
    const KvTiles<32> tiles(A, B);
    KvRaw16<IT, CT, HD> raw[2];
    typename KvRaw16<IT, CT, HD>::Lane offsets(A, n, g);
    int page[2];
    int next = 0; // page of the tile to be fetched next
    auto look = [&](int i) { next = kv_page(A.table, A.pagesPerSeq, A.numPages, B.s, tiles.at(min(i, tiles.n - 1)) * 32 >> 6); };
    auto fetch = [&](int i, int set) __attribute__((always_inline)) {
        const int j0 = tiles.at(i) * 32;
        page[set] = next;
        raw[set].fetch(A, max(page[set], 0), j0 & 63, kh, offsets);
    };
    auto tile = [&](int i, int set) __attribute__((always_inline)) {
        const int j0 = tiles.at(i) * 32;
        const bool whole = kv_all_see(A, B.minPos, B.maxPos, j0, 32) && page[set] >= 0;
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            s[b] = (f32x4)(0.f);
            if constexpr (SP > 1) {
                const uint32_t own = raw[set].kp[b];
                params[wave][g * (HD / 4) / KV_GROUP][16 * b + n] = own;
#pragma unroll
                for (int t = 0; t < KS; t++) s[b] = mfma16<false>(kv_tiny(raw[set].k[b][t]), q[t], s[b]);
                const f32x4 base = mfma16<false>(u32x4{(own & 0xffffu) | own << 16, 0u, 0u, 0u}, qsum, (f32x4)(0.f));
                const u32x4 par = *reinterpret_cast<const u32x4*>(&params[wave][n % SP][16 * b + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t w = par[e]; // (a bit cast of an element of a vector reads the first)
                    float v = fmaf(kv_half(w >> 16), s[b][e], zero);
                    v += kv_neighbour<0xb1>(v);
                    if constexpr (SP == 4) v += kv_neighbour<0x4e>(v);
                    s[b][e] = fmaf(v, 1024.f, base[e]);
                }
            } else if constexpr (PARTS) {
                const uint32_t par = raw[set].kp[b];
                const _Float16 top = __builtin_bit_cast(_Float16, (uint16_t)(par >> 16 & 0xffe0u));
                const _Float16 low = __builtin_bit_cast(_Float16, (uint16_t)(par >> 16)) - top, high = top * (_Float16)0.0625f;
                f32x4 most = (f32x4)(0.f); // a sixteenth of the high part's sum
                s[b] = mfma16<false>(u32x4{(par & 0xffffu) | par << 16, 0u, 0u, 0u}, qsum, s[b]);
#pragma unroll
                for (int t = 0; t < KS; t++) {
                    const u32x4 codes = kv_codes(raw[set].k[b][t]);
                    most = mfma16<false>(kv_times(codes, __builtin_bit_cast(uint16_t, high)), q[t], most);
                    s[b] = mfma16<false>(kv_times(codes, __builtin_bit_cast(uint16_t, low)), q[t], s[b]);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[b][e] = fmaf(most[e], 16.f, s[b][e]);
            } else {
#pragma unroll
                for (int t = 0; t < KS; t++) s[b] = mfma16<BF>(raw[set].key(b, t), q[t], s[b]);
            }
        }
        bool odd[2] = {false, false}; // does this lane hold an element of V that is no number?
        if (!whole) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int t = 0; t < KS; t++) odd[b] |= kv_odd<BF>(raw[set].val(b, t));
        }
        const bool repair = __any(odd[0] | odd[1]);
        // V's rows: columns in the order that the pieces come in (4-bit pages: (0, 4), (1, 5) ... of every eight)
        unsigned char* const place = vt + n * VP + (FOUR ? (HD / 4) * g : 8 * g) * 2;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int t = 0; t < KS; t++) {
                u32x4 x = raw[set].val(b, t);
                if (repair) x = kv_without_odd<BF>(x);
                *reinterpret_cast<u32x4*>(place + 16 * b * VP + (FOUR ? 8 * t : 32 * t) * 2) = x;
            }
        if (!whole) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[b][e] = !sight.sees(j0 + 16 * b + 4 * g + e) ? -INFINITY : page[set] < 0 ? KV_NAN : s[b][e];
        }
        float mx = -INFINITY, p[2][4];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = kv_max(mx, s[b][e]);
        const float mt = kv_quad_max(mx) * scale;
        if (__any(mt > m + (RAISE + KV_SLACK))) {
            const float mn = mt > m + (RAISE + KV_SLACK) ? mt - RAISE : m, corr = m == -INFINITY ? 0.f : kv_exp2(m - mn); // (each row for itself)
            m = mn;
            l *= corr;
#pragma unroll
            for (int b = 0; b < VB; b++) acc[b] *= corr;
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) p[b][e] = kv_exp2(fmaf(s[b][e], scale, -ref)); // (hidden: 2^-inf)
        if (repair) {
#pragma unroll
            for (int b = 0; b < 2; b++) {
                unsigned long long hit = __ballot(odd[b]);
                uint32_t keys = (uint32_t)((hit | hit >> 16 | hit >> 32 | hit >> 48) & 0xffffu);
                while (keys) {
                    const int k = __builtin_ctz(keys), j = j0 + 16 * b + k;
                    keys &= keys - 1;
                    if (j > B.maxPos) break;
                    float w = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; e++) w = fmaf(e == (k & 3) ? 1.f : 0.f, p[b][e], w); // (a selection would go through memory)
                    w = __shfl(w, 16 * (k >> 2) + n, 64);
                    if (page[set] >= 0) kv_odd_row<CT, HD, FOUR>(A, page[set], j & 63, kh, odds[wave]);
                    const bool see_ = page[set] >= 0 && sight.sees(j);
#pragma unroll
                    for (int c = 0; c < VB; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (e == 0) __builtin_amdgcn_sched_barrier(0); // (few registers for what hardly happens)
                            const int at = 16 * c + 4 * g + e, d = FOUR ? (at & ~7) + (at & 7) / 2 + 4 * (at & 1) : at;
                            const float x = odds[wave][d];
                            acc[c][e] += see_ && x != 0.f ? w * x : 0.f;
                        }
                }
            }
        }
        const u32x4 pw = {kv_pack<BF>(p[0][0], p[0][1]), kv_pack<BF>(p[0][2], p[0][3]), kv_pack<BF>(p[1][0], p[1][1]), kv_pack<BF>(p[1][2], p[1][3])};
        u32x4 rest = (u32x4)(0u); // what the halves leave of the weights
        if constexpr (PARTS) {
            auto left = [&](uint32_t w, float a, float b) { return pack_f16(a - kv_half(w & 0xffffu), b - kv_half(w >> 16)); };
            rest = u32x4{left(pw.x, p[0][0], p[0][1]), left(pw.y, p[0][2], p[0][3]), left(pw.z, p[1][0], p[1][1]), left(pw.w, p[1][2], p[1][3])};
        }
#pragma unroll
        for (int i = 0; i < 4; i++) { // (the weights as the products have them)
            l = kv_add2<BF>(pw[i], l);
            if constexpr (PARTS) l = kv_add2<BF>(rest[i], l);
        }
        // lane i of a group of 16 gives the address of row i / 4, columns 4 (i % 4) ..
        const unsigned char* va = vt + (4 * g + (n >> 2)) * VP + (n & 3) * 8;
#pragma unroll
        for (int b = 0; b < VB; b++) {
            const u32x2 lo = lds_transposed(va + 32 * b), hi = lds_transposed(va + 16 * VP + 32 * b);
            acc[b] = mfma16<BF>(u32x4{lo.x, lo.y, hi.x, hi.y}, pw, acc[b]);
            if constexpr (PARTS) acc[b] = mfma16<BF>(u32x4{lo.x, lo.y, hi.x, hi.y}, rest, acc[b]);
        }
    };
    const int step = NW * A.nsplit;
    int t = split * NW + wave;
    if (t < tiles.n) {
        look(t);
        fetch(t, 0);
        look(t + step);
    }
    if constexpr (FOUR) {
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < KS; t++)
#pragma unroll
            for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(x[t][i]));
        const int e = kv_row_exp(kv_quad_max(most), A.scale2);
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < KS; t++) sum += ((x[t][0] + x[t][1]) + (x[t][2] + x[t][3])) + ((x[t][4] + x[t][5]) + (x[t][6] + x[t][7]));
        sum = ldexpf(sum, e);
        scale = ldexpf(scale, -e);
        if constexpr (SP > 1) {
            // column n: this row's elements of group n % SP, zeros elsewhere; largest into [2^14, 2^15), that of the odd words 2^-4 of it; the product is 2^-10 of the sum then
            const bool own = g * (HD / 4) / KV_GROUP == n % SP;
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) q[t][i] = own ? pack_f16(ldexpf(x[t][i], e + (i & 1 ? 10 : 14)), ldexpf(x[t][i + 4], e + (i & 1 ? 10 : 14))) : 0u;
        } else {
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) q[t][i] = pack_f16(ldexpf(x[t][i], e), ldexpf(x[t][i + 4], e));
        }
        if constexpr (SP > 1 || PARTS) {
            const uint32_t first = kv_to_half(sum);
            qsum.x = first | kv_to_half(sum - kv_half(first)) << 16;
        }
    }
    while (t < tiles.n) { // (no further tile: the same loads again, dropped)
        fetch(min(t + step, tiles.n - 1), 1);
        look(t + 2 * step);
        __builtin_amdgcn_sched_barrier(0);
        tile(t, 0);
        t += step;
        if (t >= tiles.n) break;
        fetch(min(t + step, tiles.n - 1), 0);
        look(t + 2 * step);
        __builtin_amdgcn_sched_barrier(0);
        tile(t, 1);
        t += step;
    }
    l = kv_quad_sum(l);
    __syncthreads(); // the waves' V tiles become the place where they meet
    kv_finish16<IT, HD, NW, SP>(A, B, kh, split, acc, m, l, reinterpret_cast<float*>(lds), [&](auto put) {
        if (n % SP != 0) return;
#pragma unroll
        for (int b = 0; b < VB; b++) {
            if constexpr (!FOUR) put(16 * b + 4 * g, acc[b]);
            else { // columns (0, 4, 1, 5) or (2, 6, 3, 7) of every eight
                float* f = reinterpret_cast<float*>(lds) + ((size_t)wave * 16 + n / SP) * (HD + 4) + 16 * b + 8 * (g >> 1) + 2 * (g & 1);
                f[0] = acc[b].x; f[4] = acc[b].y; f[1] = acc[b].z; f[5] = acc[b].w;
            }
        }
    });
}

// ----------------------------------------------------------------------------
// Many 16-bit rows of a sequence: 32 a wave, NW waves a workgroup, a page (64 keys) at a time through LDS, double-buffered.  S^T[key, row] = K . Q^T on 32x32x16
// products: every lane owns one row (element i of lane l: key 8 (i / 4) + 4 (l / 32) + i % 4, row l % 32), so maximum and sum run down registers, with one
// exchange between the lane halves; O^T += V^T . P^T takes the weights as they lie and V through the transposing LDS read.  Pages of 16 bits go straight to LDS
// (the 16-byte pieces of a row in an order that keeps both readings free of bank conflicts), those of 4 bits through registers, where codes become halves; fp16 rows too
// meet K and V rounded to halves here (error against the result's norm 4.4e-4, 2.1e-4 the rounding of the result).  Weights are rounded to 16 bits as above: in two parts the
// products would be half as many again.
// Bound by the matrix cores at the clock that their power leaves (1.8 GHz) and the vector ALU's exponentials between them: 16384 rows, 32 heads of 128 in fp16, window 4096
// 1.02 to 1.10 ms on different cards, 0.95 to 0.89 PFLOP/s of what is seen (a library product of 8192 cubed: 1.07).  Eight prompts of 2048, window 1024: 0.16 to 0.18 ms, 0.64 to
// 0.57 PFLOP/s: of 19 tiles that a workgroup's rows touch 16 are seen whole, and every workgroup starts with a lookup and a tile that nothing hides; matrix cores and vector ALU
// are busy in 0.35 and 0.41 of the cycles.  1289 rows behind 3000 to 7000 positions in 4 bits, heads of 64: 101 us, 0.51 PFLOP/s: the vector ALU, busy in 0.64 of the cycles to the
// matrix cores' 0.28, unpacks every tile for 128 rows.
// ----------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <bool BF> __device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// place of 16-byte piece c of row r: K's operand takes the same piece of 32 rows at once, V's takes four pieces of four rows
template <int HD> __device__ __forceinline__ int kv_place_k(int r, int c) { return r * (HD * 2) + 16 * (c ^ (HD == 128 ? r & 15 : (r >> 1) & 7)); }
template <int HD> __device__ __forceinline__ int kv_place_v(int r, int c) { return r * (HD * 2) + 16 * (c ^ (HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1))); }

template <typename IT, typename CT, int HD, int NW>
__global__ void __launch_bounds__(NW * 64, HD == 64 ? 3 : 2) k_kvattn_many(KvAttnArgs A) {
    constexpr bool FOUR = KvType<CT>::code == MLH_CACHE_Q4, BF = !FOUR && KvType<IT>::code == MLH_DTYPE_BF16;
    constexpr float RAISE = KvRaise<BF>::value;
    constexpr int KS = HD / 16, MB = HD / 32, TB = 64 * HD * 2, QB = NW * 32; // TB: bytes of a tile of K or V
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[]; // K, V of two tiles; keys to repair; a row of V for each wave
    uint32_t* const flags = reinterpret_cast<uint32_t*>(lds + 4 * TB);
    float (*const odds)[HD] = reinterpret_cast<float (*)[HD]>(lds + 4 * TB + 32);
    const int kh = blockIdx.x % A.kvHeads, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, half = lane >> 5;
    KvBlock B;
    if (!kv_block_longest_first<QB, true>(A, blockIdx.x / A.kvHeads, B)) return;
    const bool active = wave * 32 < B.nr;
    const int wr0 = B.r0 + min(wave * 32, B.nr - 1), wr1 = B.r0 + min(wave * 32 + 31, B.nr - 1); // this wave's rows
    const int wMin = max(B.pos0 + wr0 / A.group, -1), wMax = min(B.pos0 + wr1 / A.group, B.cap - 1);
    const int r = B.r0 + min(wave * 32 + n, B.nr - 1), h = kh * A.group + r % A.group;
    const KvSight sight(A, B.pos0 + r / A.group);
    u32x4 q[KS];
    float scale = A.scale2;
    {
        const IT* qr = (const IT*)A.q + (size_t)(B.row0 + r / A.group) * A.qStride + (size_t)h * HD + 8 * half;
        if constexpr (!FOUR) {
#pragma unroll
            for (int t = 0; t < KS; t++) q[t] = *reinterpret_cast<const u32x4*>(qr + 16 * t);
        } else {
            float most = 0.f;
            if (KvType<IT>::code == MLH_DTYPE_BF16) {
                for (int t = 0; t < KS; t++) {
                    float x[8];
                    kv_load8(qr + 16 * t, x);
#pragma unroll
                    for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(x[i]));
                }
                most = fmaxf(most, __shfl_xor(most, 32, 64));
            }
            const int e = KvType<IT>::code == MLH_DTYPE_BF16 ? kv_row_exp(most, A.scale2) : 0;
            scale = ldexpf(scale, -e);
#pragma unroll
            for (int t = 0; t < KS; t++) {
                float x[8];
                kv_load8(qr + 16 * t, x);
#pragma unroll
                for (int i = 0; i < 4; i++) q[t][i] = pack_f16(ldexpf(x[i], e), ldexpf(x[i + 4], e));
            }
        }
    }
    f32x16 acc[MB];
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[b][i] = 0.f;
    float m = -INFINITY, l = 0.f; // (of the scores times scale)
    const KvTiles<64> tiles(A, B);
    const int split = blockIdx.y, t0 = (int)((long long)tiles.n * split / A.nsplit), t1 = (int)((long long)tiles.n * (split + 1) / A.nsplit); // this workgroup's

    // ---- a tile into LDS ----
    constexpr int EPT = HD / NW; // 4-bit pages: elements a thread takes of K and of V
    uint32_t kc[FOUR ? EPT / 8 : 1], vc[FOUR ? EPT / 8 : 1], kp = 0, vp = 0;
    const int qRow = tid / NW, qAt = (tid % NW) * EPT;
    constexpr int RPI = 512 / HD, CPR = HD / 8; // 16-bit pages: rows an instruction, pieces a row
    auto page_of = [&](int i) { return kv_page(A.table, A.pagesPerSeq, A.numPages, B.s, tiles.at(i)); };
    auto fetch = [&](int found, int buf) __attribute__((always_inline)) { // the tile of that page
        const int page = max(found, 0);
        if constexpr (FOUR) {
            const size_t base = ((size_t)page * A.kvHeads + kh) * kv_tile_bytes(HD);
            const unsigned o = qRow * (HD / 2) + qAt / 2, p = kv_param_at(HD) + (qRow * (HD / KV_GROUP) + qAt / KV_GROUP) * 4;
            const uint8_t *tk = (const uint8_t*)A.poolK + base, *tv = (const uint8_t*)A.poolV + base;
            kp = *reinterpret_cast<const uint32_t*>(tk + p);
            vp = *reinterpret_cast<const uint32_t*>(tv + p);
            kv_words(tk + o, kc);
            kv_words(tv + o, vc);
        } else { // 1 KiB an instruction: lane i's 16 bytes go to the i-th place of it
            const size_t base = (((size_t)page * MLH_KV_PAGE) * A.kvHeads + kh) * HD * 2;
            const int lr = lane / CPR, lc = lane % CPR;
#pragma unroll
            for (int j = 0; j < 64 / RPI / NW; j++) {
                const int r0 = (j * NW + wave) * RPI, row = r0 + lr;
                const unsigned ko = (unsigned)(row * A.kvHeads * HD * 2) + ((kv_place_k<HD>(row, lc) - row * (HD * 2)));
                const unsigned vo = (unsigned)(row * A.kvHeads * HD * 2) + ((kv_place_v<HD>(row, lc) - row * (HD * 2)));
                const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds + buf * 2 * TB + r0 * (HD * 2);
                const unsigned char *sk = (const unsigned char*)A.poolK + base, *sv = (const unsigned char*)A.poolV + base;
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(ko), "s"(sk) : "memory", "m0");
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(__builtin_amdgcn_readfirstlane(to + TB)), "v"(vo), "s"(sv) : "memory", "m0");
            }
        }
    };
    // Before tile i counts as landed: 4-bit pages are written from what fetch left in registers; and where some row does not see all of the tile, elements of V that are no
    // numbers leave it, and their keys are noted (each wave: what it brought itself; a place to note three tiles long, so that it is cleared two barriers before).
    auto land = [&](int i, int page, int buf, int slot) __attribute__((always_inline)) {
        const int j0 = tiles.at(i) * 64;
        const bool part = !kv_all_see(A, B.minPos, B.maxPos, j0, 64) || page < 0;
        auto note = [&](int row) { if (j0 + row <= B.maxPos && page >= 0) atomicOr(&flags[2 * slot + (row >> 5)], 1u << (row & 31)); };
        if constexpr (FOUR) {
#pragma unroll
            for (int e = 0; e < EPT / 8; e++) {
                *reinterpret_cast<u32x4*>(lds + buf * 2 * TB + kv_place_k<HD>(qRow, qAt / 8 + e)) = kv_halves(kc[e], kp);
                u32x4 x = kv_halves(vc[e], vp);
                if (part && kv_odd<BF>(x)) { x = kv_without_odd<BF>(x); note(qRow); }
                *reinterpret_cast<u32x4*>(lds + buf * 2 * TB + TB + kv_place_v<HD>(qRow, qAt / 8 + e)) = x;
            }
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (part) {
#pragma unroll
                for (int j = 0; j < 64 / RPI / NW; j++) {
                    const int r0 = (j * NW + wave) * RPI;
                    u32x4* p = reinterpret_cast<u32x4*>(lds + buf * 2 * TB + TB + r0 * (HD * 2)) + lane;
                    const u32x4 x = *p;
                    if (kv_odd<BF>(x)) { *p = kv_without_odd<BF>(x); note(r0 + lane / CPR); }
                }
            }
        }
    };

    auto tile = [&](int i, int page, int buf, int slot) __attribute__((always_inline)) {
        const int j0 = tiles.at(i) * 64;
        if (!active || j0 > wMax || (A.window && j0 + 63 <= wMin - A.window && j0 >= A.sinks)) return;
        const unsigned char *kt = lds + buf * 2 * TB, *vt = kt + TB;
        const bool whole = kv_all_see(A, wMin, wMax, j0, 64) && page >= 0;
        f32x16 s[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
#pragma unroll
            for (int e = 0; e < 16; e++) s[b][e] = 0.f;
#pragma unroll
            for (int t = 0; t < KS; t++) s[b] = mfma32<BF>(*reinterpret_cast<const u32x4*>(kt + kv_place_k<HD>(32 * b + n, 2 * t + half)), q[t], s[b]);
        }
        float mx = -INFINITY;
        if (!whole) {
            if (page < 0) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[b][e] = KV_NAN;
            }
            const int j = j0 + 4 * half;
            if (A.window && j0 < A.sinks) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[b][e] = sight.sees(j + 32 * b + 8 * (e >> 2) + (e & 3)) ? s[b][e] : -INFINITY;
            } else {
                const unsigned from = j - sight.low;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[b][e] = from + (32 * b + 8 * (e >> 2) + (e & 3)) <= sight.span ? s[b][e] : -INFINITY;
            }
        }
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) mx = kv_max(mx, s[b][e]);
        const float mt = kv_halves_max(mx) * scale;
        if (__any(mt > m + (RAISE + KV_SLACK))) {
            const float mn = mt > m + (RAISE + KV_SLACK) ? mt - RAISE : m, corr = m == -INFINITY ? 0.f : kv_exp2(m - mn); // (each row for itself)
            m = mn;
            l *= corr;
#pragma unroll
            for (int b = 0; b < MB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[b][e] *= corr;
        }
        const float ref = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) { // (hidden: 2^-inf)
                s[b][e] = kv_exp2(fmaf(s[b][e], scale, ref));
            }
        uint32_t odd[2] = {0, 0};
        if (!kv_all_see(A, B.minPos, B.maxPos, j0, 64)) { odd[0] = __builtin_amdgcn_readfirstlane(flags[2 * slot]); odd[1] = __builtin_amdgcn_readfirstlane(flags[2 * slot + 1]); }
        if (odd[0] | odd[1]) { // repair
#pragma unroll
            for (int b = 0; b < 2; b++)
                for (uint32_t keys = odd[b]; keys; keys &= keys - 1) {
                    const int k = __builtin_ctz(keys), j = j0 + 32 * b + k, at = 4 * (k >> 3) + (k & 3);
                    float w = 0.f;
#pragma unroll
                    for (int e = 0; e < 16; e++) w = e == at ? s[b][e] : w;
                    w = __shfl(w, n + 32 * ((k >> 2) & 1), 64);
                    const bool see = sight.sees(j);
                    kv_odd_row<CT, HD, FOUR>(A, page, j & 63, kh, odds[wave]);
#pragma unroll
                    for (int c = 0; c < MB; c++)
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            if (e % 4 == 0) __builtin_amdgcn_sched_barrier(0); // (few registers for what hardly happens)
                            const int col = 32 * c + 8 * (e >> 2) + 4 * half + (e & 3), d = FOUR ? (col & ~7) + (col & 7) / 2 + 4 * (col & 1) : col;
                            const float x = odds[wave][d];
                            acc[c][e] += see && x != 0.f ? w * x : 0.f;
                        }
                }
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int b = t >> 1, e0 = 8 * (t & 1);
            const u32x4 pw = {kv_pack<BF>(s[b][e0], s[b][e0 + 1]), kv_pack<BF>(s[b][e0 + 2], s[b][e0 + 3]), kv_pack<BF>(s[b][e0 + 4], s[b][e0 + 5]), kv_pack<BF>(s[b][e0 + 6], s[b][e0 + 7])};
#pragma unroll
            for (int i = 0; i < 4; i++) l = kv_add2<BF>(pw[i], l); // (the weights as the product has them)
            const int row = 16 * t + 4 * half + ((lane & 15) >> 2), piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), rest = 8 * (lane & 1);
#pragma unroll
            for (int c = 0; c < MB; c++) {
                const u32x2 lo = lds_transposed(vt + kv_place_v<HD>(row, 4 * c + piece) + rest), hi = lds_transposed(vt + kv_place_v<HD>(row + 8, 4 * c + piece) + rest);
                acc[c] = mfma32<BF>(u32x4{lo.x, lo.y, hi.x, hi.y}, pw, acc[c]);
            }
        }
    };

    if (tid < 6) flags[tid] = 0;
    int page = 0, next = 0; // of tiles i and i + 1; looked up two tiles ahead
    if (t0 < t1) {
        page = page_of(t0);
        next = page_of(min(t0 + 1, t1 - 1));
        fetch(page, 0);
    }
    __syncthreads();
    for (int i = t0, slot = 0; i < t1; i++) {
        const int buf = (i - t0) & 1;
        land(i, page, buf, slot);
        __syncthreads(); // for every wave, and every wave is done with tile i - 1
        if (i + 1 < t1) fetch(next, buf ^ 1);
        const int later = page_of(min(i + 2, t1 - 1));
        __builtin_amdgcn_sched_barrier(0);
        if (tid < 2) flags[2 * (slot == 0 ? 2 : slot - 1) + tid] = 0; // tile i - 1's, and i + 2's
        tile(i, page, buf, slot);
        slot = slot == 2 ? 0 : slot + 1;
        page = next;
        next = later;
    }
    if (!active || wave * 32 + n >= B.nr) return;
    l += __shfl_xor(l, 32, 64);
    const int qi = r / A.group;
    const bool beyond = B.pos0 + qi >= B.cap, none = B.pos0 + qi < 0; // its own position is behind the page table; it sees nothing (as in kv_finish16)
    const float inv = A.nsplit > 1 || none ? 1.f : beyond ? KV_NAN : 1.0f / l;
    IT* out = (IT*)A.out + (size_t)(B.row0 + qi) * A.outStride + (size_t)h * HD;
    const size_t shares = (size_t)A.rows * A.heads, rh = split * shares + (size_t)(B.row0 + qi) * A.heads + h;
    float* part = A.part + rh * HD;
    if (A.nsplit > 1 && half == 0) *reinterpret_cast<float2*>(A.part + A.nsplit * shares * HD + rh * 2) = beyond ? make_float2(0.f, KV_NAN) : none ? make_float2(0.f, 1.f) : make_float2(m, l);
#pragma unroll
    for (int c = 0; c < MB; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f32x4 o = f32x4{acc[c][4 * e], acc[c][4 * e + 1], acc[c][4 * e + 2], acc[c][4 * e + 3]} * inv;
            if (FOUR) { // columns (0, 4, 1, 5) here, (2, 6, 3, 7) in the other half: four neighbours each
                const float a = __shfl_xor(half ? o.x : o.y, 32, 64), b = __shfl_xor(half ? o.z : o.w, 32, 64);
                o = half ? f32x4{a, b, o.y, o.w} : f32x4{o.x, o.z, a, b};
            }
            if (A.nsplit > 1) *reinterpret_cast<f32x4*>(part + 32 * c + 8 * e + 4 * half) = o;
            else kv_put4(out + 32 * c + 8 * e + 4 * half, o);
        }
}

// ----------------------------------------------------------------------------
// The shares of nsplit workgroups of a row and head, MOST at most: a lane a share (or several) for the factors, 256 / (HD / 4) groups of threads for the sums.
// ----------------------------------------------------------------------------
// (32 of 64 shares: 4 us, latency)
#define KV_MAX_SPLIT 256 // (one token over 200000 positions in 4 bits, one K/V head: 23 us; 128: 30, 64: 49)
template <typename IT, int HD, int MOST>
__global__ void __launch_bounds__(256) k_kvattn_join(KvAttnArgs A) {
    constexpr int T = HD / 4, G = 256 / T, L = MOST / 64; // L: shares of a lane, lane + 64 i
    __shared__ f32x4 sum[G][T];
    const size_t rh = blockIdx.x, n = (size_t)A.rows * A.heads;
    const int row = (int)(rh / A.heads), h = (int)(rh % A.heads), lane = threadIdx.x & 63, t = threadIdx.x % T, g = threadIdx.x / T;
    const float2* stat = reinterpret_cast<const float2*>(A.part + (size_t)A.nsplit * n * HD);
    float2 ml[L];
#pragma unroll
    for (int i = 0; i < L; i++) ml[i] = lane + 64 * i < A.nsplit ? stat[(lane + 64 * i) * n + rh] : make_float2(-INFINITY, 0.f);
    f32x4 v[MOST / G]; // (everything on its way before anything is waited for)
#pragma unroll
    for (int i = 0; i < MOST / G; i++) v[i] = *reinterpret_cast<const f32x4*>(A.part + (min(i * G + g, A.nsplit - 1) * n + rh) * HD + 4 * t);
    if (row < A.start[0] || row >= A.start[A.nseq]) return;
    float M = -INFINITY, den = 0.f, f[L];
#pragma unroll
    for (int i = 0; i < L; i++) M = fmaxf(M, ml[i].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
#pragma unroll
    for (int i = 0; i < L; i++) {
        f[i] = kv_exp2(ml[i].x - (M == -INFINITY ? 0.f : M));
        den = fmaf(ml[i].y, f[i], den);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o, 64);
    f32x4 o = (f32x4)(0.f);
#pragma unroll
    for (int i = 0; i < MOST / G; i++) {
        const float w = __shfl(f[i * G / 64], (i * G + g) % 64, 64); // (of a share that is not there: 2^-inf)
        if (i * G + g < A.nsplit) o += v[i] * w;
    }
    sum[g][t] = o;
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int i = 1; i < G; i++) o += sum[i][t];
    o = f32x4{o.x / den, o.y / den, o.z / den, o.w / den};
    kv_put4((IT*)A.out + (size_t)row * A.outStride + (size_t)h * HD + 4 * t, o);
}

// The same of few shares (KV_JOIN_FEW at most): a thread for four elements.  (41248 rows of 4 shares of 64: 9 us, 4.6 TB/s; k_kvattn_join 43.)
#define KV_JOIN_FEW 8
template <typename IT, int HD>
__global__ void __launch_bounds__(256) k_kvattn_join_few(KvAttnArgs A) {
    constexpr int T = HD / 4;
    const size_t rh = (size_t)blockIdx.x * (256 / T) + threadIdx.x / T, n = (size_t)A.rows * A.heads;
    if (rh >= n) return;
    const int row = (int)(rh / A.heads), h = (int)(rh % A.heads), d = threadIdx.x % T * 4;
    const float2* stat = reinterpret_cast<const float2*>(A.part + (size_t)A.nsplit * n * HD);
    float2 ml[KV_JOIN_FEW];
    f32x4 v[KV_JOIN_FEW], o = (f32x4)(0.f);
    float M = -INFINITY, den = 0.f;
#pragma unroll
    for (int s = 0; s < KV_JOIN_FEW; s++) {
        const size_t i = (size_t)min(s, A.nsplit - 1) * n + rh;
        ml[s] = stat[i];
        v[s] = *reinterpret_cast<const f32x4*>(A.part + i * HD + d);
        M = fmaxf(M, ml[s].x);
    }
    if (row < A.start[0] || row >= A.start[A.nseq]) return;
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int s = 0; s < KV_JOIN_FEW; s++) {
        if (s >= A.nsplit) continue;
        const float f = kv_exp2(ml[s].x - ref);
        den = fmaf(ml[s].y, f, den);
        o += v[s] * f;
    }
    o = f32x4{o.x / den, o.y / den, o.z / den, o.w / den};
    kv_put4((IT*)A.out + (size_t)row * A.outStride + (size_t)h * HD + d, o);
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
static std::string attn_check(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_attention* a) {
    std::string bad = kv_check(c, b, false);
    if (!bad.empty()) return bad;
    if (!a) return "null arguments";
    const long long width = (long long)b->heads * c->headDim;
    bad = kv_check_rows("q", a->q, a->qStride, width, b->type);
    if (bad.empty()) bad = kv_check_rows("out", a->out, a->outStride, width, b->type);
    if (!bad.empty()) return bad;
    if (a->q == a->out) return "out must not be q";
    if (a->window < 0 || a->sinks < 0 || a->maxLen < 0 || a->maxNew < 0) return "window, sinks, maxLen and maxNew must not be negative";
    if (a->scale != 0.f && (!(a->scale >= 1.0e-30f) || !(a->scale <= 1.0e30f))) return "scale must be 0 or 1e-30 to 1e30";
    return "";
}

// Which kernel (32 query heads on 8, heads of 128, bf16, 4000 positions; "rows" are a sequence's, over the heads of one K/V head):
//   16-bit pages: k_kvattn_many from 17 rows on.  16 sequences of 4, 16, 32, 64 rows: k_kvattn_few 49, 59, 111, 174 us, k_kvattn_many 50, 53, 57, 73; one sequence: 12, 12, 19, 19
//     and 15, 15, 16, 18; 64 of 4 rows over 100 to 12000 positions: 290 and 377 (it splits less).
//   4-bit pages: from 65 on.  16 sequences of 32, 64, 96 rows: k_kvattn_few 44, 68, 95 us, k_kvattn_many 53, 69, 77 (its tiles pass through LDS as halves).  fp16 rows, whose
//     products are two there: 44 and 76 for 50 and 58 us at 32 and 64, for the keys that it keeps.
//   fp16 rows over 4-bit pages that leave a column for each of their groups: spread (above).
// How keys are split, a second kernel joining the shares:
#define KV_SPLIT_WGS 768 // k_kvattn_few, k_kvattn_f32: until a call has this many workgroups of at least four turns each, or two until each compute unit has one
                         // (64 tokens over 100 to 12000, 64 over 3000 positions, 48 over up to 9000 in 4 bits: 291, 150, 87 us; 512: 339, 141, 87; 1536: 293, 152, 90;
                         // four turns always: one token over 4000 15 us for 12; two always: 64 over 300 30 for 17)
#define KV_SPLIT_MANY 1024 // k_kvattn_many: the same (512 to 3000: no difference within 3 of 118 us) ...
#define KV_SPLIT_LEAST 8   // ... of at least eight tiles each, four until each compute unit has a workgroup (one sequence, 32 rows: 16 us, 21 with eight; two: 14, but 512 rows 44 for 32)
struct AttnPlan {         // which kernel, and how the keys are split
    int many;             // waves of a workgroup of k_kvattn_many; 0: the kernels of 16 rows
    int rowsPer;          // rows of a workgroup
    int blocks, nsplit;
    long long wgs;        // workgroups with rows, per split
    size_t bytes;
};
static AttnPlan attn_plan(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_attention* a) {
    AttnPlan P;
    const int group = b->heads / c->heads;
    const long long cap = (long long)c->pagesPerSeq * MLH_KV_PAGE, rows = (long long)b->rows * group;
    const long long maxLen = a->maxLen ? std::min<long long>(a->maxLen, cap) : cap;
    const long long maxNew = a->maxNew ? std::min(a->maxNew, b->rows) : b->rows;
    P.many = b->type != MLH_DTYPE_F32 && maxNew * group > (c->type == MLH_CACHE_Q4 ? 64 : 16) ? 4 : 0;
    const int spread = 16 * KV_GROUP / c->headDim; // rows that leave a column for each of their groups
    P.rowsPer = P.many ? P.many * 32 : c->type == MLH_CACHE_Q4 && b->type == MLH_DTYPE_F16 && maxNew * group <= spread ? spread : 16;
    const int qb = P.rowsPer;
    P.blocks = (int)((rows + qb - 1) / qb + c->nseq - 1); // (floor(a) + ceil(b) <= ceil(a + b))
    P.wgs = ((rows + qb - 1) / qb + std::min(c->nseq, b->rows) - 1) * c->heads;
    // positions that a row sees, in turns of a workgroup: four waves of 32 keys, or a page
    const long long seen = a->window ? std::min<long long>(maxLen, (long long)a->window + std::min<long long>(a->sinks, maxLen) + 64) : maxLen;
    const int turn = P.many ? 64 : 128;
    const long long rounds = (seen + turn - 1) / turn;
    auto each = [&](long long most) { return (most + P.wgs - 1) / P.wgs; };
    const long long n = P.many ? std::min(each(KV_SPLIT_MANY), std::max(rounds / KV_SPLIT_LEAST, std::min(rounds / (KV_SPLIT_LEAST / 2), each(256)))) : std::min(each(KV_SPLIT_WGS), std::max(rounds / 4, std::min(rounds / 2, each(256))));
    P.nsplit = (int)std::max<long long>(1, std::min<long long>(n, KV_MAX_SPLIT));
    P.bytes = P.nsplit > 1 ? (size_t)P.nsplit * b->rows * b->heads * (c->headDim + 2) * 4 : 0;
    return P;
}

// A workgroup has 16 rows at most, and nsplit times their number is below KV_SPLIT_WGS and once more their own, which is below that where keys are split.
size_t mlh_attention_work_most(int headDim) { return (size_t)2 * KV_SPLIT_WGS * 16 * (headDim + 2) * 4; }

template <typename IT, typename CT, int HD, int NW> static int launch_many(dim3 grid, void* stream, const KvAttnArgs& A) {
    constexpr int bytes = 4 * 64 * HD * 2 + 32 + NW * HD * 4;
    if (bytes > 65536) { // (asked for on every call: the attribute belongs to the device that is current)
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_kvattn_many<IT, CT, HD, NW>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return kv_status(e);
    }
    return kv_launch(&k_kvattn_many<IT, CT, HD, NW>, grid, NW * 64, bytes, stream, A);
}

template <typename IT, int HD> static int launch_join(void* stream, const KvAttnArgs& A) {
    const unsigned n = (unsigned)(A.rows * A.heads), per = 256 / (HD / 4);
    if (A.nsplit <= KV_JOIN_FEW) return kv_launch(&k_kvattn_join_few<IT, HD>, dim3((n + per - 1) / per), 256, 0, stream, A);
    return kv_launch(A.nsplit <= 64 ? &k_kvattn_join<IT, HD, 64> : &k_kvattn_join<IT, HD, KV_MAX_SPLIT>, dim3(n), 256, 0, stream, A);
}
static int launch_join(void* stream, int type, int hd, const KvAttnArgs& A) {
    if (A.nsplit == 1) return 0;
#define JOIN(IT_) return hd == 64 ? launch_join<IT_, 64>(stream, A) : launch_join<IT_, 128>(stream, A)
    if (type == MLH_DTYPE_F32) JOIN(float);
    if (type == MLH_DTYPE_BF16) JOIN(bf16_t);
    JOIN(f16_t);
#undef JOIN
}

extern "C" uint64_t mlh_attention_work_bytes(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_attention* a) {
    return attn_check(c, b, a).empty() ? attn_plan(c, b, a).bytes : 0;
}

extern "C" int mlh_attention_device(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_attention* a, void* stream) {
    const std::string bad = attn_check(c, b, a);
    if (!bad.empty()) return kv_fail(bad);
    if (b->rows == 0) return 0;
    const AttnPlan P = attn_plan(c, b, a);
    if (P.bytes > 0 && (!a->work || a->workBytes < P.bytes)) return kv_fail("work is smaller than mlh_attention_work_bytes() = " + std::to_string(P.bytes));
    if (P.bytes > 0 && (uintptr_t)a->work % 16) return kv_fail("work must be 16-byte aligned");
    if ((long long)P.blocks * c->heads * P.nsplit * 512 > 0xffffffffll) return kv_fail("too many rows or sequences for one call");
    const int hd = c->headDim;
    const KvAttnArgs A = {c->k, c->v, c->table, b->start, b->len, a->q, a->out, (float*)a->work, a->qStride, a->outStride, c->nseq, b->rows, b->heads, c->heads, b->heads / c->heads,
                          c->pagesPerSeq, c->numPages, a->window, a->sinks, P.nsplit, (a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)hd)) * 1.44269504088896341f};
    const dim3 grid = P.many ? dim3(c->heads * P.blocks, P.nsplit) : dim3(c->heads * P.blocks * P.nsplit);
    int rc;
    if (P.many) {
#define MANY(IT_, CT_) (hd == 64 ? launch_many<IT_, CT_, 64, 4>(grid, stream, A) : launch_many<IT_, CT_, 128, 4>(grid, stream, A))
        if (b->type == MLH_DTYPE_BF16) rc = c->type == MLH_CACHE_Q4 ? MANY(bf16_t, q4_t) : MANY(bf16_t, bf16_t);
        else rc = c->type == MLH_CACHE_Q4 ? MANY(f16_t, q4_t) : MANY(f16_t, f16_t);
#undef MANY
    } else if (b->type == MLH_DTYPE_F32) {
#define F32_ROWS(CT_) kv_launch(hd == 64 ? &k_kvattn_f32<CT_, 64> : &k_kvattn_f32<CT_, 128>, grid, KV_F32_WAVES * 64, 0, stream, A)
        rc = c->type == MLH_CACHE_Q4 ? F32_ROWS(q4_t) : F32_ROWS(float);
#undef F32_ROWS
    } else {
#define FEW(IT_, CT_, SP64_) kv_launch(hd == 64 ? &k_kvattn_few<IT_, CT_, 64, SP64_> : &k_kvattn_few<IT_, CT_, 128, SP64_ * SP64_>, grid, KV_FEW_WAVES * 64, 0, stream, A)
        if (P.rowsPer < 16) rc = FEW(f16_t, q4_t, 2); // (spread: a column for each of 2 groups, 4 for heads of 128)
        else if (b->type == MLH_DTYPE_BF16) rc = c->type == MLH_CACHE_Q4 ? FEW(bf16_t, q4_t, 1) : FEW(bf16_t, bf16_t, 1);
        else rc = c->type == MLH_CACHE_Q4 ? FEW(f16_t, q4_t, 1) : FEW(f16_t, f16_t, 1);
#undef FEW
    }
    return rc ? rc : launch_join(stream, b->type, hd, A);
}
