// Attention over a caller's paged K/V cache (mlh_attention_device): causal, with a sliding window and first positions that stay visible, over pages of 32, 16 or 4
// bits.
#include <math.h>

#include <algorithm>

#include "kv_cache.h"

struct KvAttnArgs {
    const void *poolK, *poolV;
    const int32_t *table, *start, *len;
    const void* q;
    void* out;
    long long qStride, outStride;
    int nseq, rows, heads, kvHeads, pagesPerSeq, numPages, window, sinks;
    float scale;
};

// One wave per row and head: lanes take a key each for the scores, then the output's elements.
template <typename IT, typename CT, int HD>
__global__ void __launch_bounds__(64) k_kv_attn(KvAttnArgs A) {
    __shared__ float q[HD];
    const int h = blockIdx.x % A.heads, row = blockIdx.x / A.heads, lane = threadIdx.x, kh = h / (A.heads / A.kvHeads);
    const int s = kv_find(A.nseq, row, [&](int i) { return A.start[i]; });
    const int b = A.start[s], e = A.start[s + 1];
    if (row < b || row >= e) return;
    const long long pos = (long long)A.len[s] - e + row;
    if (lane < HD / 8) {
        float x[8];
        kv_load8((const IT*)A.q + (size_t)row * A.qStride + (size_t)h * HD + lane * 8, x);
        for (int i = 0; i < 8; i++) q[lane * 8 + i] = x[i];
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[HD / 64] = {};
    auto row8 = [&](const void* pool, int page, int at, int d, float (&x)[8]) {
        if constexpr (KvType<CT>::code != MLH_CACHE_Q4) {
            kv_load8((const CT*)pool + (((size_t)page * MLH_KV_PAGE + at) * A.kvHeads + kh) * HD + d, x);
        } else {
            const uint8_t* tile = (const uint8_t*)pool + ((size_t)page * A.kvHeads + kh) * kv_tile_bytes(HD);
            kv_values8(*reinterpret_cast<const uint32_t*>(tile + at * (HD / 2) + d / 2), *reinterpret_cast<const uint32_t*>(tile + kv_param_at(HD) + (at * (HD / KV_GROUP) + d / KV_GROUP) * 4), x);
        }
    };
    const long long w0 = A.window ? std::max<long long>(0, pos + 1 - A.window) : 0;
    for (long long j0 = 0; j0 <= pos; j0 += 64) {
        if (A.window && j0 >= A.sinks && j0 + 64 <= w0) continue;
        const int page = kv_page(A.table, A.pagesPerSeq, A.numPages, s, (int)(j0 >> 6));
        const long long j = j0 + lane;
        const bool seen = j <= pos && (j >= w0 || j < A.sinks);
        float sc = -INFINITY;
        if (seen && page < 0) sc = __uint_as_float(0x7fc00000u);
        else if (seen) {
            sc = 0.f;
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                row8(A.poolK, page, lane, d, x);
                for (int i = 0; i < 8; i++) sc = fmaf(x[i], q[d + i], sc);
            }
            sc *= A.scale;
        }
        float mt = fmaxf(m, sc);
        for (int o = 32; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor(mt, o, 64));
        const float ref = mt == -INFINITY ? 0.f : mt, corr = expf(m - ref), p = seen ? expf(sc - ref) : 0.f;
        m = mt;
        float ps = p;
        for (int o = 32; o > 0; o >>= 1) ps += __shfl_xor(ps, o, 64);
        l = l * corr + ps;
        for (int i = 0; i < HD / 64; i++) acc[i] *= corr;
        for (int k = 0; k < 64; k++) {
            const float pk = __shfl(p, k, 64);
            if (!((__ballot(seen) >> k) & 1)) continue;
            float x[8];
            for (int i = 0; i < HD / 64; i++) {
                const int d = lane + 64 * i;
                if (page >= 0) row8(A.poolV, page, k, d & ~7, x);
                float v = 0.f;
                for (int t = 0; t < 8; t++) v = page >= 0 && t == (d & 7) ? x[t] : v;
                acc[i] = fmaf(pk, v, acc[i]);
            }
        }
    }
    for (int i = 0; i < HD / 64; i++) {
        float o = l == 0.f ? 0.f : acc[i] / l;
        IT* p = (IT*)A.out + (size_t)row * A.outStride + (size_t)h * HD + lane + 64 * i;
        if constexpr (KvType<IT>::code == MLH_DTYPE_F32) *p = o;
        else if constexpr (KvType<IT>::code == MLH_DTYPE_BF16) *p = (bf16_t)kv_to_bf16(o);
        else p->bits = (uint16_t)kv_to_half(o);
    }
}

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
    if (!(a->scale >= 0.f) || !(a->scale <= 3.0e38f)) return "scale must be finite and not negative";
    return "";
}

extern "C" uint64_t mlh_attention_work_bytes(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_attention* a) {
    return attn_check(c, b, a).empty() ? 0 : 0;
}

extern "C" int mlh_attention_device(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_attention* a, void* stream) {
    const std::string bad = attn_check(c, b, a);
    if (!bad.empty()) return kv_fail(bad);
    if (b->rows == 0) return 0;
    const KvAttnArgs A = {c->k, c->v, c->table, b->start, b->len, a->q, a->out, a->qStride, a->outStride, c->nseq, b->rows, b->heads, c->heads, c->pagesPerSeq, c->numPages, a->window, a->sinks,
                          a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)c->headDim)};
    const dim3 grid((unsigned)b->rows * b->heads);
#define GO(IT_, CT_) \
    do { \
        if (c->headDim == 64) hipLaunchKernelGGL((k_kv_attn<IT_, CT_, 64>), grid, dim3(64), 0, (hipStream_t)stream, A); \
        else hipLaunchKernelGGL((k_kv_attn<IT_, CT_, 128>), grid, dim3(64), 0, (hipStream_t)stream, A); \
    } while (0)
    if (c->type == MLH_CACHE_Q4) {
        if (b->type == MLH_DTYPE_F32) GO(float, q4_t);
        else if (b->type == MLH_DTYPE_BF16) GO(bf16_t, q4_t);
        else GO(f16_t, q4_t);
    } else if (b->type == MLH_DTYPE_F32) GO(float, float);
    else if (b->type == MLH_DTYPE_BF16) GO(bf16_t, bf16_t);
    else GO(f16_t, f16_t);
#undef GO
    return kv_launched();
}
