// What the kernels on a caller's paged K/V cache (mlh_kv_cache) share: element types, places of rows, values of 4-bit pages.
#pragma once
#include "mlh_internal.h"

typedef float kv_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_u32x4 __attribute__((ext_vector_type(4)));
struct q4_t { uint8_t byte; }; // two codes

template <typename T> struct KvType;
template <> struct KvType<float> { static constexpr int code = MLH_DTYPE_F32; };
template <> struct KvType<bf16_t> { static constexpr int code = MLH_DTYPE_BF16; };
template <> struct KvType<f16_t> { static constexpr int code = MLH_DTYPE_F16; };
template <> struct KvType<q4_t> { static constexpr int code = MLH_CACHE_Q4; };

#define KV_GROUP 32 // elements of a row that share a minimum and a scale
__host__ __device__ constexpr int kv_tile_bytes(int hd) { return MLH_KV_PAGE * hd / 2 + MLH_KV_PAGE * (hd / KV_GROUP) * 4; } // 4-bit pages: one head's
__host__ __device__ constexpr int kv_param_at(int hd) { return MLH_KV_PAGE * hd / 2; }                                     // ... minima and scales in it

__device__ __forceinline__ float kv_half(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
__device__ __forceinline__ float kv_bf16(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ uint32_t kv_to_bf16(float v) { // to nearest even; NaN stays NaN
    typedef __bf16 kv_bf16x2 __attribute__((ext_vector_type(2)));
    return (uint16_t)(__builtin_bit_cast(uint32_t, kv_bf16x2{(__bf16)v, (__bf16)0.0f}));
}
__device__ __forceinline__ uint32_t kv_to_half(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

// eight consecutive elements <-> floats
__device__ __forceinline__ void kv_load8(const float* p, float (&x)[8]) {
    const kv_f32x4 a = *reinterpret_cast<const kv_f32x4*>(p), b = *reinterpret_cast<const kv_f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) { x[i] = a[i]; x[4 + i] = b[i]; }
}
__device__ __forceinline__ void kv_load8(const bf16_t* p, float (&x)[8]) {
    const kv_u32x4 a = *reinterpret_cast<const kv_u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) { x[2 * i] = kv_bf16(a[i] & 0xffffu); x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u); }
}
__device__ __forceinline__ void kv_load8(const f16_t* p, float (&x)[8]) {
    const kv_u32x4 a = *reinterpret_cast<const kv_u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) { x[2 * i] = kv_half(a[i] & 0xffffu); x[2 * i + 1] = kv_half(a[i] >> 16); }
}
template <bool NT, typename T> __device__ __forceinline__ void kv_store16(void* p, const T& v) { // NT: not to be kept in the caches
    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<T*>(p));
    else *reinterpret_cast<T*>(p) = v;
}
template <bool NT> __device__ __forceinline__ void kv_store8(float* p, const float (&x)[8]) {
    kv_store16<NT>(p, kv_f32x4{x[0], x[1], x[2], x[3]});
    kv_store16<NT>(p + 4, kv_f32x4{x[4], x[5], x[6], x[7]});
}
template <bool NT> __device__ __forceinline__ void kv_store8(bf16_t* p, const float (&x)[8]) {
    kv_u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] = kv_to_bf16(x[2 * i]) | kv_to_bf16(x[2 * i + 1]) << 16;
    kv_store16<NT>(p, a);
}
template <bool NT> __device__ __forceinline__ void kv_store8(f16_t* p, const float (&x)[8]) {
    kv_u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] = kv_to_half(x[2 * i]) | kv_to_half(x[2 * i + 1]) << 16;
    kv_store16<NT>(p, a);
}

// Largest s in [0, nseq) with key(s) <= b, for keys that do not decrease (0 if there is none).  All lanes of a wave together, for one b: 64 places a load, since what a
// search costs is a memory latency a step.
template <typename F> __device__ __forceinline__ int kv_find(int nseq, int b, F key) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = nseq;
    while (n > 1) {
        const int step = (n + 63) >> 6, i = lane * step;
        const int below = __builtin_popcountll(__ballot(i < n && key(lo + min(i, n - 1)) <= b));
        const int skip = max(below - 1, 0) * step;
        lo += skip;
        n = min(step, n - skip);
    }
    return lo;
}

// A word at an index that all lanes share, of memory that no kernel of the call writes: through the scalar cache.  (As a vector load, which the compiler takes where it
// sees stores around, it waits for every load on its way before it.)
__device__ __forceinline__ int kv_uniform(const int32_t* p, size_t i) { return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(p + i); }

// Pool page of page j of sequence s; -1: beyond the table, or not in the pool.
__device__ __forceinline__ int kv_page(const int32_t* table, int pagesPerSeq, int numPages, int s, int j) {
    if (j < 0 || j >= pagesPerSeq) return -1;
    const int p = kv_uniform(table, (size_t)s * pagesPerSeq + j);
    return (unsigned)p < (unsigned)numPages ? p : -1;
}

// A group's parameters and codes (16 bits each: minimum, scale)
__device__ __forceinline__ void kv_values8(uint32_t codes, uint32_t params, float (&x)[8]) {
    const float base = kv_half(params & 0xffffu), scale = kv_half(params >> 16);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = fmaf((float)((codes >> (4 * i)) & 15u), scale, base);
}

// The code of x: the nearest whole number to (x - base) / scale.  The fp32 quotient, up to 16 where it is not clamped, is off by less than 2^-18 (three roundings: difference, inverse
// and product): only within 1e-4 of a half, 26 times that, is it done again in 64 bits.
__device__ __forceinline__ uint32_t kv_code(float x, float base, float scale, float inv) {
    const float u = (x - base) * inv;
    float c = rintf(u);
    if (fabsf(u - c) > 0.4999f) c = (float)rint(((double)x - (double)base) / (double)scale);
    return (uint32_t)fminf(fmaxf(c, 0.f), 15.f);
}

// mlh_kv_append_device's and its fellows' checks, also made by the context's calls: empty, or what is wrong
std::string kv_check(const mlh_kv_cache* cache, const mlh_kv_batch* batch, bool anyType);
std::string kv_check_rows(const char* what, const void* p, long long stride, long long width, int type);
int kv_fail(const std::string& msg); // -1, with the text for mlh_last_error(NULL)
int kv_status(hipError_t e);         // of a launch: 0, or -2, with the text
// What this launch returned, and not hipGetLastError, which also gives what an earlier call of the program left.
template <typename Args> int kv_launch(void (*kernel)(Args), dim3 grid, int threads, size_t lds, void* stream, const Args& a) {
    void* args[] = {const_cast<Args*>(&a)};
    return kv_status(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), args, lds, (hipStream_t)stream));
}
inline size_t kv_elem_bytes(int type) { return type == MLH_DTYPE_F32 ? 4 : 2; }
