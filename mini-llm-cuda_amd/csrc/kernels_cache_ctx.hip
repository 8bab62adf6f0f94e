// A context's attention layers on the operators of a paged cache (kernels_cache.hip, kernels_cache_attn.hip): with a sliding window, or with pages of 4 bits.
// A layer is then two or three launches where it is one otherwise: the rows go into the pages, attention reads them, and the result is put where
// the output projection expects it.
#include <algorithm>

#include "kv_cache.h"

bool mlh_cache_ops(const mlh_ctx* c) {
    if (c->window == 0 && c->kvType == MLH_DTYPE_F32) return false;
    for (const LayerDev& L : c->layers) // (a model of gated-delta-net layers alone has neither)
        if (L.kind == MLH_KIND_ATTENTION) return true;
    return false;
}

// Where the rows of a call stand, once for all layers: workgroup s has sequence seqs[s].  segStart null: a decode step, one row each.
__global__ void __launch_bounds__(256) k_cache_begin(const int* pageTable, int pagesPerSeq, int n, int rows, const int* seqs, const int* pos, const int* segStart, const int* segLen, const int* segPos0,
                                                     int* start, int* len, int* table) {
    const int s = blockIdx.x, seq = seqs[s];
    for (int j = threadIdx.x; j < pagesPerSeq; j += 256) table[(size_t)s * pagesPerSeq + j] = pageTable[(size_t)seq * pagesPerSeq + j];
    if (threadIdx.x == 0) {
        start[s] = segStart ? segStart[s] : s;
        len[s] = segStart ? segPos0[s] + segLen[s] : pos[seq] + 1;
        if (s == n - 1) start[n] = rows;
    }
}

static int* cache_start(const mlh_ctx* c) { return c->cacheMeta; }
static int* cache_len(const mlh_ctx* c) { return c->cacheMeta + c->hp.maxSeqs + 1; }
static int* cache_table(const mlh_ctx* c) { return c->cacheMeta + 2 * c->hp.maxSeqs + 1; }

// Tables of the calls, and room for the shares of split keys: each is kept from its first need on (a second try after a failure finds what the first one got).
static int prepare(mlh_ctx* c, bool attention) {
    const size_t S = c->hp.maxSeqs;
    void* p = nullptr;
    if (!c->cacheMeta) {
        if (const int rc = mlh_dev_alloc_bytes(c, &p, (2 * S + 1 + S * c->pagesPerSeq) * 4)) return rc;
        c->cacheMeta = (int*)p;
    }
    if (attention && !c->cacheWork) {
        if (const int rc = mlh_dev_alloc_bytes(c, &p, mlh_attention_work_most(c->hp.headDim))) return rc;
        c->cacheWork = p;
    }
    return 0;
}

// (no allocation, no synchronisation: can be captured)
int mlh_cache_begin(mlh_ctx* c, int n, int rows, const int* seqs, const int* segStart, const int* segLen, const int* segPos0) {
    if (!mlh_cache_ops(c)) return 0;
    hipLaunchKernelGGL(k_cache_begin, dim3(n), dim3(256), 0, c->stream, c->d_pageTable, c->pagesPerSeq, n, rows, seqs, c->d_pos, segStart, segLen, segPos0, cache_start(c), cache_len(c), cache_table(c));
    MLH_CHECK(c, hipGetLastError());
    return 0;
}

static mlh_kv_cache cache_of(const mlh_ctx* c, const LayerDev& L, const int* table, int nseq) {
    return {L.K, L.V, table, c->kvType, c->hp.attnHeads, c->hp.headDim, c->hp.maxSeqs * c->pagesPerSeq, c->pagesPerSeq, nseq};
}

// Rows [q | k | v | ..] of n sequences, `rows` of them `ld` floats apart: norm and rotation (q in place), into the pages, attention into out [rows, dim].
int mlh_cache_layer(mlh_ctx* c, const LayerDev& L, int n, int rows, float* qkv, int ld, float* out) {
    const mlh_hparams& hp = c->hp;
    const mlh_kv_cache cache = cache_of(c, L, cache_table(c), n);
    const mlh_kv_batch batch = {cache_start(c), cache_len(c), rows, MLH_DTYPE_F32, hp.attnHeads};
    mlh_kv_append in = {};
    in.q = qkv; in.qOut = qkv; in.k = qkv + L.offK; in.v = qkv + L.offV;
    in.qStride = in.qOutStride = in.kStride = in.vStride = ld;
    in.rope = c->rope; in.ropeRows = hp.maxL;
    in.qGain = hp.qkRmsNorm ? L.gq : nullptr; in.kGain = hp.qkRmsNorm ? L.gk : nullptr;
    mlh_attention at = {};
    at.q = qkv; at.out = out; at.qStride = ld; at.outStride = hp.dim;
    at.window = c->window; at.sinks = c->sinks; at.maxLen = hp.maxL;
    at.work = c->cacheWork; at.workBytes = mlh_attention_work_most(hp.headDim);
    int rc = mlh_kv_append_device(&cache, &batch, &in, c->stream);
    if (rc == 0) rc = mlh_attention_device(&cache, &batch, &at, c->stream);
    if (rc) c->err = std::string("paged attention: ") + mlh_last_error(nullptr);
    return rc;
}

// A decode step's result to the output projection: gated (inference.cu:241-250) and, with the PLE columns, as the planes of the row step; or as
// the first of the GEMV's partial results.  Grid: slots x pieces of the row.
__global__ void __launch_bounds__(256) k_cache_put(StepArgs a, LayerDev L, const float* out) {
    const int slot = blockIdx.x, i = blockIdx.y * 256 + threadIdx.x;
    const float* qkv = a.qkv + (size_t)slot * a.qkvStride;
    if (!a.mixRows) {
        if (i >= L.ad) return;
        const int h = i / a.hd, e = i - h * a.hd;
        for (int s = 0; s < a.nsplit; s++) {
            float* p = a.part + (((size_t)slot * a.nsplit + s) * a.heads + h) * (a.hd + 2);
            p[e] = s == 0 ? out[(size_t)slot * a.dim + i] : 0.f;
            if (e == 0) { p[a.hd] = s == 0 ? 0.f : -1.0e30f; p[a.hd + 1] = s == 0 ? 1.f : 0.f; } // maximum, sum
        }
        return;
    }
    const bool half = a.wbytes == 2;
    if (i < L.ad) {
        float v = out[(size_t)slot * a.dim + i];
        if (a.gating) v = v / (1.0f + expf(-qkv[L.offG + i]));
        rows_put(a.mixRows, i, slot, a.mixLay, half, v);
    } else if (i - L.ad < a.ple) {
        const int j = i - L.ad;
        const size_t t = (size_t)a.tok[slot] * a.ple + j;
        const float g = qkv[L.offPle + j], p = half ? kv_bf16(((const bf16_t*)L.pleTable)[t]) : ((const float*)L.pleTable)[t];
        rows_put(a.mixRows, i, slot, a.mixLay, half, g / (1.0f + expf(-g)) * p);
    }
}

// The mixing part of an attention layer of a decode step.
int mlh_cache_step(mlh_ctx* c, const StepArgs& a, const LayerDev& L) {
    if (const int rc = mlh_cache_layer(c, L, a.nseq, a.nseq, a.qkv, a.qkvStride, c->h1)) return rc; // (h1 is written by the output projection only)
    hipLaunchKernelGGL(k_cache_put, dim3(a.nseq, (L.ad + a.ple + 255) / 256), dim3(256), 0, c->stream, a, L, c->h1);
    return 0;
}

// ----------------------------------------------------------------------------
// settings
// ----------------------------------------------------------------------------
extern "C" int mlh_set_attention_window(mlh_ctx* c, int window, int sinks) {
    if (!c) return -1;
    if (window < 0 || sinks < 0) { c->err = "window and sinks must not be negative"; return -1; }
    (void)hipSetDevice(c->device);
    if (const int rc = window ? prepare(c, true) : 0) return rc;
    mlh_drop_graphs(c); // recorded launches hold the old values
    c->window = window;
    c->sinks = window ? sinks : 0;
    return 0;
}

extern "C" int mlh_set_kv_type(mlh_ctx* c, int type) {
    if (!c) return -1;
    if (type != MLH_DTYPE_F32 && type != MLH_CACHE_Q4) { c->err = "a context's pages are MLH_DTYPE_F32 or MLH_CACHE_Q4"; return -1; }
    if (type == c->kvType) return 0;
    for (int n : c->h_len)
        if (n > 0) { c->err = "the type of the pages can be changed while all sequences are empty (mlh_reset)"; return -1; }
    (void)hipSetDevice(c->device);
    if (const int rc = type == MLH_CACHE_Q4 ? prepare(c, true) : 0) return rc;
    const size_t bytes = (size_t)c->hp.maxSeqs * c->pagesPerSeq * mlh_kv_page_bytes(type, c->hp.attnHeads, c->hp.headDim);
    std::vector<void*> fresh; // the new pools first: the context stays as it is when they do not fit
    auto drop = [&]() { for (void* p : fresh) (void)hipFree(p); };
    for (const LayerDev& L : c->layers) {
        if (L.kind != MLH_KIND_ATTENTION) continue;
        for (int k = 0; k < 2; k++) {
            void* p = nullptr;
            hipError_t e = hipMalloc(&p, bytes);
            if (e == hipSuccess) { fresh.push_back(p); e = hipMemset(p, 0, bytes); }
            if (e != hipSuccess) { drop(); (void)hipGetLastError(); c->err = std::string("pages: ") + hipGetErrorString(e); return -2; }
        }
    }
    const hipError_t e = hipDeviceSynchronize();
    if (e != hipSuccess) { drop(); c->err = std::string("hipDeviceSynchronize: ") + hipGetErrorString(e); return -2; }
    mlh_drop_graphs(c);
    size_t at = 0;
    for (LayerDev& L : c->layers) {
        if (L.kind != MLH_KIND_ATTENTION) continue;
        for (float** pool : {&L.K, &L.V}) {
            std::replace(c->allocs.begin(), c->allocs.end(), (void*)*pool, fresh[at]); // (the context owns them)
            (void)hipFree(*pool);
            *pool = (float*)fresh[at++];
        }
    }
    c->kvType = type;
    MLH_CHECK(c, hipMemcpy(c->d_layers, c->layers.data(), c->layers.size() * sizeof(LayerDev), hipMemcpyHostToDevice)); // (once more in finalize)
    return 0;
}

extern "C" int mlh_read_kv(mlh_ctx* c, int layer, int seq, int pos, int n, float* k, float* v) {
    if (!c) return -1;
    if (layer < 0 || layer >= c->hp.transformers || c->layers[layer].kind != MLH_KIND_ATTENTION) { c->err = "layer is not an attention layer"; return -1; }
    if (seq < 0 || seq >= c->hp.maxSeqs) { c->err = "sequence index out of range"; return -1; }
    if (!k || !v || pos < 0 || n <= 0 || n > c->h_len[seq] || pos > c->h_len[seq] - n) { c->err = "positions beyond what the sequence holds, or a null output"; return -1; }
    (void)hipSetDevice(c->device);
    if (const int rc = prepare(c, false)) return rc;
    const size_t d = c->hp.dim, bytes = (size_t)n * d * 4;
    float* tmp = nullptr;
    MLH_CHECK(c, hipStreamSynchronize(c->stream));
    MLH_CHECK(c, hipMalloc((void**)&tmp, 2 * bytes));
    const int head[2] = {0, n}, len = pos + n; // (the metadata's place is free between calls)
    hipError_t e = hipMemcpy(cache_start(c), head, 8, hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMemcpy(cache_len(c), &len, 4, hipMemcpyHostToDevice);
    int rc = 0;
    if (e == hipSuccess) {
        const mlh_kv_cache cache = cache_of(c, c->layers[layer], c->d_pageTable + (size_t)seq * c->pagesPerSeq, 1);
        const mlh_kv_batch batch = {cache_start(c), cache_len(c), n, MLH_DTYPE_F32, c->hp.attnHeads};
        const mlh_kv_read args = {tmp, tmp + (size_t)n * d, (int64_t)d};
        rc = mlh_kv_read_device(&cache, &batch, &args, c->stream);
        if (rc) c->err = std::string("reading pages: ") + mlh_last_error(nullptr);
        else {
            e = hipStreamSynchronize(c->stream);
            if (e == hipSuccess) e = hipMemcpy(k, tmp, bytes, hipMemcpyDeviceToHost);
            if (e == hipSuccess) e = hipMemcpy(v, tmp + (size_t)n * d, bytes, hipMemcpyDeviceToHost);
        }
    }
    (void)hipFree(tmp);
    if (e != hipSuccess) { c->err = std::string("reading pages: ") + hipGetErrorString(e); rc = -2; }
    return rc;
}
