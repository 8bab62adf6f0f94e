// Rows into and out of a caller's paged K/V cache: mlh_kv_append_device (per-head norm, rotation, conversion to the pages' type, 4-bit quantisation
// in one pass over the rows) and mlh_kv_read_device.
#include <math.h>

#include <algorithm>

#include "kv_cache.h"

#define KV_WG 256
// workgroups along the rows: with `pieces` of a row each below 2^32 threads, which is what a launch can have; beyond, they take several turns
static unsigned kv_grid(int rows, int pieces) { return (unsigned)std::min(rows, std::max(1, (1 << 22) / pieces)); }

struct KvRows { // what the kernels need of cache and batch
    const int32_t *start, *len, *table;
    int nseq, rows, pagesPerSeq, numPages, heads, kvHeads;
};

// sequence and position of a row; false: behind the last sequence
__device__ __forceinline__ bool kv_row(const KvRows& R, int row, int& seq, int& pos) {
    const int s = kv_find(R.nseq, row, [&](int i) { return R.start[i]; });
    const int b = kv_uniform(R.start, s), e = kv_uniform(R.start, s + 1);
    seq = s;
    pos = (int)((unsigned)kv_uniform(R.len, s) - (unsigned)e + (unsigned)row);
    return row >= b && row < e;
}

struct KvAppendArgs {
    KvRows R;
    void *poolK, *poolV;
    const void *q, *k, *v;
    void* qOut;
    long long qStride, qOutStride, kStride, vStride;
    const float *rope, *qGain, *kGain;
    int ropeRows;
};

// The code of x: the nearest whole number to (x - base) / scale.  The fp32 quotient, up to 16 where it is not clamped, is off by less than 2^-18 (three roundings: difference, inverse
// and product): only within 1e-4 of a half, 26 times that, is it done again in 64 bits.
__device__ __forceinline__ uint32_t kv_code(float x, float base, float scale, float inv) {
    const float u = (x - base) * inv;
    float c = rintf(u);
    if (fabsf(u - c) > 0.4999f) c = (float)rint(((double)x - (double)base) / (double)scale);
    return (uint32_t)fminf(fmaxf(c, 0.f), 15.f);
}

// One thread: eight elements of a head's row of q, k or v.  HD / 8 neighbouring threads hold the row (norm), four a group of 32 (4-bit codes).  Grid: rows x pieces of the
// heads.  Norm and rotation are in 64 bits and rounded once, as the plain form's products of fp32 numbers are exact there.
// Bound by memory: 17435 rows of 32 + 8 + 8 heads of 128 in bf16, 429 MB read and written, 80 us (5.4 TB/s; a copy of 1 GiB: 5.2).  11071 rows of the same heads in fp16
// into 4-bit pages 57 to 59 us (240 MB, 4.2 TB/s): the vector ALU, busy in 0.84 of the cycles.  With gains 127 and 85 us, by the norm's arithmetic in 64 bits (a division an element).
// A single token: 2.2 us, the latency of start, table and row in turn.  Streaming stores (NT) for
// calls that write more than the L2s hold: 112 us without.  Two, four and eight rows a workgroup, their loads together: 95, 107 and 149 us against 91 for one (all before the row
// was loaded ahead of the lookup).
template <typename IT, typename CT, int HD, bool NT>
__global__ void __launch_bounds__(KV_WG) k_kv_append(KvAppendArgs A) {
    constexpr int T = HD / 8;
    const int u = blockIdx.y * KV_WG + threadIdx.x;
    const int units = (A.R.heads + 2 * A.R.kvHeads) * T, qUnits = A.R.heads * T, kUnits = A.R.kvHeads * T;
    const int kind = u < qUnits ? 0 : u < qUnits + kUnits ? 1 : 2; // q, k, v
    const int w = u - (kind == 0 ? 0 : kind == 1 ? qUnits : qUnits + kUnits), h = w / T, d = (w % T) * 8;
    const bool live = u < units && (kind != 0 || A.q); // (whole heads' threads: HD / 8 divides 64)
    const IT* const src = (const IT*)(kind == 0 ? A.q : kind == 1 ? A.k : A.v) + (size_t)h * HD + d;
    const long long stride = kind == 0 ? A.qStride : kind == 1 ? A.kStride : A.vStride;
    const float* const gain = kind == 0 ? A.qGain : kind == 1 ? A.kGain : nullptr;
    for (int row = blockIdx.x; row < A.R.rows; row += gridDim.x) {
        float x[8], cs[8];
        int seq, pos;
        if (live) kv_load8(src + (size_t)row * stride, x); // (on its way while the row's sequence and page are looked up)
        const bool mine = kv_row(A.R, row, seq, pos);
        int page = pos < 0 ? -1 : kv_page(A.R.table, A.R.pagesPerSeq, A.R.numPages, seq, pos >> 6);
        if (A.rope && pos >= A.ropeRows) page = -1;
        if (!live || !mine || (page < 0 && kind != 0)) continue;
        if (A.rope && kind != 2) kv_load8(A.rope + (size_t)(page < 0 ? 0 : pos) * HD + d, cs);
        if (gain) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < 8; i++) s += (double)x[i] * (double)x[i];
#pragma unroll
            for (int o = 1; o < T; o <<= 1) s += __shfl_xor(s, o, 64);
            const double r = sqrt(s / (double)HD + 1e-8);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = (float)((double)gain[h * HD + d + i] * ((double)x[i] / r));
        }
        if (A.rope && kind != 2) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) { // (products of two fp32 values are exact in 64 bits)
                const double a = x[i], c = x[i + 1], co = cs[i], si = cs[i + 1];
                x[i] = (float)(co * a - si * c);
                x[i + 1] = (float)(si * a + co * c);
            }
        }
        if (kind == 0) {
            if (page < 0) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = __uint_as_float(0x7fc00000u);
            }
            kv_store8<NT>((IT*)A.qOut + (size_t)row * A.qOutStride + (size_t)h * HD + d, x);
            continue;
        }
        void* pool = kind == 1 ? A.poolK : A.poolV;
        if constexpr (KvType<CT>::code != MLH_CACHE_Q4) {
            kv_store8<NT>((CT*)pool + (((size_t)page * MLH_KV_PAGE + (pos & 63)) * A.R.kvHeads + h) * HD + d, x);
        } else {
            float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); bad += x[i] * 0.f; } // (bad: NaN with an infinity or NaN among them)
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) { lo = fminf(lo, __shfl_xor(lo, o, 64)); hi = fmaxf(hi, __shfl_xor(hi, o, 64)); bad += __shfl_xor(bad, o, 64); }
            float step = (hi - lo) * (1.0f / 15.0f);
            asm volatile("" : "+v"(step)); // (rounded to fp32 first; in one instruction with the conversion the product is not)
            uint32_t minBits = kv_to_half(__builtin_amdgcn_fmed3f(lo, -65504.f, 65504.f)), scaleBits = kv_to_half(step);
            const float base = kv_half(minBits), scale = kv_half(scaleBits);
            uint32_t codes = 0;
            if (!(bad == 0.f) || scaleBits == 0x7c00u) { minBits = 0x7e00u; scaleBits = 0; }
            else if (scale > 0.f) {
                const float inv = 1.0f / scale;
#pragma unroll
                for (int i = 0; i < 8; i++) codes |= kv_code(x[i], base, scale, inv) << (4 * i);
            }
            uint8_t* tile = (uint8_t*)pool + ((size_t)page * A.R.kvHeads + h) * kv_tile_bytes(HD);
            *reinterpret_cast<uint32_t*>(tile + (pos & 63) * (HD / 2) + d / 2) = codes;
            if (d % KV_GROUP == 0) *reinterpret_cast<uint32_t*>(tile + kv_param_at(HD) + ((pos & 63) * (HD / KV_GROUP) + d / KV_GROUP) * 4) = minBits | scaleBits << 16;
        }
    }
}

struct KvReadArgs {
    KvRows R;
    const void *poolK, *poolV;
    void *k, *v;
    long long stride;
};

// The same places read: a thread eight elements of k or v.  Bound by what it writes: 11071 rows of 8 heads of 128 from 4 bits into fp32, 14 MB in, 91 MB out, 24 us (4.4 TB/s);
// 64 rows of 16 heads 3.2 us.
template <typename OT, typename CT, int HD>
__global__ void __launch_bounds__(KV_WG) k_kv_read(KvReadArgs A) {
    constexpr int T = HD / 8;
    const int units = 2 * A.R.kvHeads * T, kUnits = A.R.kvHeads * T;
    const int u = blockIdx.y * KV_WG + threadIdx.x;
    for (int row = blockIdx.x; row < A.R.rows; row += gridDim.x) {
        int seq, pos;
        if (!kv_row(A.R, row, seq, pos)) continue;
        if (u >= units) continue;
        const bool val = u >= kUnits;
        const int w = val ? u - kUnits : u, h = w / T, d = (w % T) * 8;
        const int page = pos < 0 ? -1 : kv_page(A.R.table, A.R.pagesPerSeq, A.R.numPages, seq, pos >> 6);
        const void* pool = val ? A.poolV : A.poolK;
        float x[8];
        if (page < 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __uint_as_float(0x7fc00000u);
        } else if constexpr (KvType<CT>::code != MLH_CACHE_Q4) {
            kv_load8((const CT*)pool + (((size_t)page * MLH_KV_PAGE + (pos & 63)) * A.R.kvHeads + h) * HD + d, x);
        } else {
            const uint8_t* tile = (const uint8_t*)pool + ((size_t)page * A.R.kvHeads + h) * kv_tile_bytes(HD);
            kv_values8(*reinterpret_cast<const uint32_t*>(tile + (pos & 63) * (HD / 2) + d / 2),
                       *reinterpret_cast<const uint32_t*>(tile + kv_param_at(HD) + ((pos & 63) * (HD / KV_GROUP) + d / KV_GROUP) * 4), x);
        }
        kv_store8<false>((OT*)(val ? A.v : A.k) + (size_t)row * A.stride + (size_t)h * HD + d, x);
    }
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
int kv_fail(const std::string& msg) {
    mlh_set_thread_error(msg);
    return -1;
}

static bool kv_float_type(int t) { return t == MLH_DTYPE_F32 || t == MLH_DTYPE_BF16 || t == MLH_DTYPE_F16; }

std::string kv_check(const mlh_kv_cache* c, const mlh_kv_batch* b, bool anyType) {
    if (!c || !b) return "null cache or batch";
    if (!c->k || !c->v || !c->table || !b->start || !b->len) return "null pointer in cache or batch";
    if (!kv_float_type(c->type) && c->type != MLH_CACHE_Q4) return "unknown cache type";
    if (!kv_float_type(b->type)) return "unknown row type";
    if (!anyType && c->type != MLH_CACHE_Q4 && c->type != b->type) return "rows must have the type of the cache's pages";
    if (c->headDim != 64 && c->headDim != 128) return "headDim must be 64 or 128";
    if (c->heads < 1 || c->heads > 4096) return "a cache has 1 to 4096 heads";
    if (!anyType && (b->heads < c->heads || b->heads % c->heads || b->heads / c->heads > 32)) return "query heads must be a multiple of the cache's heads, at most 32 times as many";
    if (c->numPages < 1 || c->nseq < 1 || c->nseq > (1 << 20)) return "numPages and nseq must be positive (nseq at most 2^20)";
    if (c->pagesPerSeq < 1 || c->pagesPerSeq > (1 << 24)) return "pagesPerSeq must be 1 to 2^24";
    if (b->rows < 0 || b->rows > (1 << 24)) return "rows must be 0 to 2^24";
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 || ((uintptr_t)c->table | (uintptr_t)b->start | (uintptr_t)b->len) % 4) return "a pool must be 16-byte aligned, tables and lengths 4-byte aligned";
    return "";
}

std::string kv_check_rows(const char* what, const void* p, long long stride, long long width, int type) {
    if (!p) return std::string("null pointer: ") + what;
    if ((uintptr_t)p % 16 || (stride * (long long)kv_elem_bytes(type)) % 16) return std::string(what) + ": rows must be 16-byte aligned";
    if (stride < width || stride > (1ll << 32)) return std::string(what) + ": stride smaller than a row, or beyond 2^32";
    return "";
}

static KvRows kv_rows_of(const mlh_kv_cache* c, const mlh_kv_batch* b) {
    return {b->start, b->len, c->table, c->nseq, b->rows, c->pagesPerSeq, c->numPages, b->heads, c->heads};
}

extern "C" uint64_t mlh_kv_page_bytes(int type, int heads, int headDim) {
    if (heads < 1 || heads > 4096 || (headDim != 64 && headDim != 128)) return 0;
    if (type == MLH_CACHE_Q4) return (uint64_t)heads * kv_tile_bytes(headDim);
    return kv_float_type(type) ? (uint64_t)MLH_KV_PAGE * heads * headDim * kv_elem_bytes(type) : 0;
}

int kv_status(hipError_t e) {
    if (e == hipSuccess) return 0;
    (void)hipGetLastError(); // (reported here)
    mlh_set_thread_error(std::string("launch failed: ") + hipGetErrorString(e));
    return -2;
}

extern "C" int mlh_kv_append_device(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_kv_append* a, void* stream) {
    std::string bad = kv_check(c, b, false);
    if (bad.empty() && !a) bad = "null arguments";
    if (!bad.empty()) return kv_fail(bad);
    const int hd = c->headDim;
    if (!a->q != !a->qOut) return kv_fail("q and qOut must both be given, or neither");
    if (a->q) {
        bad = kv_check_rows("q", a->q, a->qStride, (long long)b->heads * hd, b->type);
        if (bad.empty()) bad = kv_check_rows("qOut", a->qOut, a->qOutStride, (long long)b->heads * hd, b->type);
        if (bad.empty() && a->q == a->qOut && a->qStride != a->qOutStride) bad = "q rotated in place must keep its stride";
    } else if (a->qGain) bad = "a gain for q without q";
    if (bad.empty()) bad = kv_check_rows("k", a->k, a->kStride, (long long)c->heads * hd, b->type);
    if (bad.empty()) bad = kv_check_rows("v", a->v, a->vStride, (long long)c->heads * hd, b->type);
    if (bad.empty() && (uintptr_t)a->rope % 16) bad = "rope must be 16-byte aligned";
    if (bad.empty() && a->rope && a->ropeRows < 1) bad = "ropeRows must be positive";
    if (bad.empty() && ((uintptr_t)a->qGain | (uintptr_t)a->kGain) % 4) bad = "gains must be 4-byte aligned";
    if (!bad.empty()) return kv_fail(bad);
    if (b->rows == 0) return 0;
    KvAppendArgs A = {kv_rows_of(c, b), c->k, c->v, a->q, a->k, a->v, a->qOut, a->qStride, a->qOutStride, a->kStride, a->vStride, a->rope, a->qGain, a->kGain, a->ropeRows};
    const int pieces = ((b->heads + 2 * c->heads) * (hd / 8) + KV_WG - 1) / KV_WG;
    const dim3 grid(kv_grid(b->rows, pieces), pieces);
    const bool nt = (double)b->rows * (b->heads + 2 * c->heads) * hd * kv_elem_bytes(b->type) > 32e6; // eight L2s of 4 MB
#define KV_GO(IT_, CT_) \
    return kv_launch(hd == 64 ? (nt ? &k_kv_append<IT_, CT_, 64, true> : &k_kv_append<IT_, CT_, 64, false>) \
                              : (nt ? &k_kv_append<IT_, CT_, 128, true> : &k_kv_append<IT_, CT_, 128, false>), grid, KV_WG, 0, stream, A)
    if (c->type == MLH_CACHE_Q4) {
        if (b->type == MLH_DTYPE_F32) KV_GO(float, q4_t);
        if (b->type == MLH_DTYPE_BF16) KV_GO(bf16_t, q4_t);
        KV_GO(f16_t, q4_t);
    }
    if (b->type == MLH_DTYPE_F32) KV_GO(float, float);
    if (b->type == MLH_DTYPE_BF16) KV_GO(bf16_t, bf16_t);
    KV_GO(f16_t, f16_t);
#undef KV_GO
}

extern "C" int mlh_kv_read_device(const mlh_kv_cache* c, const mlh_kv_batch* b, const mlh_kv_read* a, void* stream) {
    std::string bad = kv_check(c, b, true);
    if (bad.empty() && !a) bad = "null arguments";
    if (!bad.empty()) return kv_fail(bad);
    const int hd = c->headDim;
    bad = kv_check_rows("k", a->k, a->stride, (long long)c->heads * hd, b->type);
    if (bad.empty()) bad = kv_check_rows("v", a->v, a->stride, (long long)c->heads * hd, b->type);
    if (!bad.empty()) return kv_fail(bad);
    if (b->rows == 0) return 0;
    KvReadArgs A = {kv_rows_of(c, b), c->k, c->v, a->k, a->v, a->stride};
    const int pieces = (2 * c->heads * (hd / 8) + KV_WG - 1) / KV_WG;
    const dim3 grid(kv_grid(b->rows, pieces), pieces);
#define KV_GO2(OT_, CT_) return kv_launch(hd == 64 ? &k_kv_read<OT_, CT_, 64> : &k_kv_read<OT_, CT_, 128>, grid, KV_WG, 0, stream, A)
#define KV_GO(CT_) \
    do { \
        if (b->type == MLH_DTYPE_F32) KV_GO2(float, CT_); \
        if (b->type == MLH_DTYPE_BF16) KV_GO2(bf16_t, CT_); \
        KV_GO2(f16_t, CT_); \
    } while (0)
    if (c->type == MLH_CACHE_Q4) KV_GO(q4_t);
    if (c->type == MLH_DTYPE_F32) KV_GO(float);
    if (c->type == MLH_DTYPE_BF16) KV_GO(bf16_t);
    KV_GO(f16_t);
#undef KV_GO
#undef KV_GO2
}
