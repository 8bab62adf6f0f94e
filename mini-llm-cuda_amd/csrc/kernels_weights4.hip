// Matrices in 4 bits: laid out and read back (mlh_weights4_*), and the product of few rows with them (mlh_gemm4_device).
#include <math.h>

#include <algorithm>

#include "p3.h"
#include "weights4.h"

typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 w4_f16x8 __attribute__((ext_vector_type(8)));

#define W4_WG 256   // threads of the kernels that lay out and read
#define W4_WAVES 8  // waves of a product's workgroup

// ----------------------------------------------------------------------------
// laying out
// ----------------------------------------------------------------------------
struct W4Args {
    uint8_t* data;
    int N, K, rows; // rows: N up to whole tiles
    const void* src;
    const uint32_t* params;
    void* dst;
    long long stride;
};

// A thread: eight columns of a row.  group / 8 neighbouring threads share a pair (whole tiles of 128 columns are gone through, so they are of one wave); those behind K bring no value.
template <typename T, int G>
__global__ void __launch_bounds__(W4_WG) k_w4_pack(W4Args A) {
    constexpr int L = G / 8;
    const int perRow = w4_tiles(A.K) * (W4_COLS / 8);
    const size_t units = (size_t)A.rows * perRow;
    for (size_t u = (size_t)blockIdx.x * W4_WG + threadIdx.x; u < units; u += (size_t)gridDim.x * W4_WG) {
        const int n = (int)(u / perRow), k = (int)(u % perRow) * 8;
        const bool live = n < A.N && k < A.K;
        float x[8], lo = INFINITY, hi = -INFINITY, bad = 0.f;
        if (live) {
            kv_load8((const T*)A.src + (size_t)n * A.stride + k, x);
#pragma unroll
            for (int i = 0; i < 8; i++) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); bad += x[i] * 0.f; }
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) { lo = fminf(lo, __shfl_xor(lo, o, 64)); hi = fmaxf(hi, __shfl_xor(hi, o, 64)); bad += __shfl_xor(bad, o, 64); }
        float step = (hi - lo) * (1.0f / 15.0f);
        asm volatile("" : "+v"(step)); // (rounded to fp32 first; in one instruction with the conversion the product is not)
        uint32_t minBits = kv_to_half(__builtin_amdgcn_fmed3f(lo, -65504.f, 65504.f)), scaleBits = kv_to_half(step);
        const float base = kv_half(minBits), scale = kv_half(scaleBits);
        uint32_t codes = 0;
        if (lo > hi && bad == 0.f) minBits = scaleBits = 0; // (nobody brought a value)
        else if (!(bad == 0.f) || scaleBits == 0x7c00u) { minBits = 0x7e00u; scaleBits = 0; }
        else if (live && scale > 0.f) {
            const float inv = 1.0f / scale;
#pragma unroll
            for (int i = 0; i < 8; i++) codes |= kv_code(x[i], base, scale, inv) << (4 * i);
        }
        *reinterpret_cast<uint32_t*>(A.data + w4_code_at(n, k, A.K, G)) = w4_spread(codes);
        if (k % G == 0) *reinterpret_cast<uint32_t*>(A.data + w4_param_at(n, k, A.K, G)) = minBits | scaleBits << 16;
    }
}

template <int G>
__global__ void __launch_bounds__(W4_WG) k_w4_set(W4Args A) {
    const int perRow = w4_tiles(A.K) * (W4_COLS / 8);
    const size_t units = (size_t)A.rows * perRow;
    for (size_t u = (size_t)blockIdx.x * W4_WG + threadIdx.x; u < units; u += (size_t)gridDim.x * W4_WG) {
        const int n = (int)(u / perRow), k = (int)(u % perRow) * 8;
        const bool live = n < A.N && k < A.K;
        *reinterpret_cast<uint32_t*>(A.data + w4_code_at(n, k, A.K, G)) = live ? w4_spread(((const uint32_t*)A.src)[((size_t)n * A.K + k) / 8]) : 0u;
        if (k % G == 0) *reinterpret_cast<uint32_t*>(A.data + w4_param_at(n, k, A.K, G)) = live ? A.params[(size_t)n * ((A.K + G - 1) / G) + k / G] : 0u;
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(W4_WG) k_w4_read(W4Args A) {
    const int perRow = A.K / 8;
    const size_t units = (size_t)A.N * perRow;
    for (size_t u = (size_t)blockIdx.x * W4_WG + threadIdx.x; u < units; u += (size_t)gridDim.x * W4_WG) {
        const int n = (int)(u / perRow), k = (int)(u % perRow) * 8;
        float x[8];
        kv_values8(w4_gather(*reinterpret_cast<const uint32_t*>(A.data + w4_code_at(n, k, A.K, G))), *reinterpret_cast<const uint32_t*>(A.data + w4_param_at(n, k, A.K, G)), x);
        kv_store8<false>((T*)A.dst + (size_t)n * A.stride + k, x);
    }
}

// ----------------------------------------------------------------------------
// product
// ----------------------------------------------------------------------------
struct Gemm4Args {
    const uint8_t* w;
    const void *a, *r;
    void* c;
    long long aStride, rStride, cStride;
    int M, N, K, swiglu;
};

// How codes and activations meet on the matrix cores, exactly.  PLANES: of an activation.  codes(x, i): eight codes of a word as an operand that stands for UNIT * (code + SHIFT).
template <typename T> struct W4Mul;
template <> struct W4Mul<f16_t> { // codes as the smallest halves, code * 2^-24
    static constexpr int PLANES = 1;
    static constexpr float UNIT = 0x1p-24f, SHIFT = 0.f;
    typedef w4_f16x8 V;
    static __device__ __forceinline__ V codes(uint32_t x) {
        return __builtin_bit_cast(V, w4_u32x4{x & 0x000f000fu, x >> 4 & 0x000f000fu, x >> 8 & 0x000f000fu, x >> 12 & 0x000f000fu});
    }
    static __device__ __forceinline__ V ones() { return V{1, 1, 1, 1, 1, 1, 1, 1}; }
    static __device__ __forceinline__ w4_f32x4 mul(V a, V b, w4_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct W4Mul<bf16_t> { // codes behind 16: 16 + code is a bf16 with the code in bits 3 to 6
    static constexpr int PLANES = 1;
    static constexpr float UNIT = 1.f, SHIFT = 16.f;
    typedef w4_bf16x8 V;
    static __device__ __forceinline__ V codes(uint32_t x) {
        return __builtin_bit_cast(V, w4_u32x4{(x << 3 & 0x00780078u) | 0x41804180u, (x >> 1 & 0x00780078u) | 0x41804180u, (x >> 5 & 0x00780078u) | 0x41804180u, (x >> 9 & 0x00780078u) | 0x41804180u});
    }
    static __device__ __forceinline__ V ones() { return __builtin_bit_cast(V, w4_u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}); }
    static __device__ __forceinline__ w4_f32x4 mul(V a, V b, w4_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct W4Mul<float> { // the same with activations as three planes (p3.h): every product exact
    static constexpr int PLANES = 3;
    static constexpr float UNIT = 1.f, SHIFT = 16.f;
    typedef w4_bf16x8 V;
    static __device__ __forceinline__ V codes(uint32_t x) { return W4Mul<bf16_t>::codes(x); }
    static __device__ __forceinline__ V ones() { return W4Mul<bf16_t>::ones(); }
    static __device__ __forceinline__ w4_f32x4 mul(V a, V b, w4_f32x4 c) { return W4Mul<bf16_t>::mul(a, b, c); }
};

__device__ __forceinline__ float w4_get(const float* p) { return *p; }
__device__ __forceinline__ float w4_get(const bf16_t* p) { return kv_bf16(*p); }
__device__ __forceinline__ float w4_get(const f16_t* p) { return kv_half(p->bits); }
__device__ __forceinline__ void w4_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void w4_put(bf16_t* p, float v) { *p = (bf16_t)kv_to_bf16(v); }
__device__ __forceinline__ void w4_put(f16_t* p, float v) { p->bits = (uint16_t)kv_to_half(v); }

// Eight neighbouring elements of a row of A on their way into LDS: raw, then as the planes that are multiplied
template <typename T> struct W4Raw {
    w4_u32x4 x;
    __device__ __forceinline__ void load(const T* p) { x = *reinterpret_cast<const w4_u32x4*>(p); }
    __device__ __forceinline__ void zero() { x = w4_u32x4{}; }
    __device__ __forceinline__ void put(w4_u32x4* at, int) const { *at = x; }
};
template <> struct W4Raw<float> {
    w4_u32x4 x[2];
    __device__ __forceinline__ void load(const float* p) { x[0] = *reinterpret_cast<const w4_u32x4*>(p); x[1] = *reinterpret_cast<const w4_u32x4*>(p + 4); }
    __device__ __forceinline__ void zero() { x[0] = x[1] = w4_u32x4{}; }
    __device__ __forceinline__ void put(w4_u32x4* at, int plane) const {
        uint32_t s[4][3];
#pragma unroll
        for (int i = 0; i < 4; i++) p3_split2(__uint_as_float(x[i / 2][i % 2 * 2]), __uint_as_float(x[i / 2][i % 2 * 2 + 1]), s[i]);
#pragma unroll
        for (int pl = 0; pl < 3; pl++) at[pl * plane] = w4_u32x4{s[0][pl], s[1][pl], s[2][pl], s[3][pl]};
    }
};

// A workgroup of WN x WK waves: WN * NT * 16 rows of W against all rows of A, K in blocks of WK * TPW tiles.  A block of A goes through LDS, once for all waves (asked for a block ahead,
// into registers); wave (wn, wk) multiplies TPW tiles of it with its NT times 16 rows, whose codes it asks for a block ahead, too.  Sums over K stay in registers; those of the WK waves are
// added up in LDS at the end, in order.
// With sum over a group of a (min + scale code) = (scale / UNIT) D + (min - scale SHIFT) S, D the sum of a (UNIT (code + SHIFT)) and S the sum of a: both come from the matrix cores, S as a product with ones.
// Lane l of a result holds column l % 16 (a row of W) and the instruction's rows 4 (l / 16) + i, i = 0 .. 3.  RG of the four are used: row m of A is row m / RG * 4 + m % RG of the
// instruction, so that few rows cost few multiplications by scales.
template <typename T, int G, int MT, int RG, int WN, int WK, int NT, int TPW>
__global__ void __launch_bounds__(W4_WAVES * 64) k_gemm4(Gemm4Args A) {
    typedef W4Mul<T> X;
    static_assert(WN * WK == W4_WAVES && (MT == 1 || RG == 4), "waves, rows");
    constexpr int S = G / 32, TG = w4_groups(G), KB = WK * TPW * W4_COLS, THREADS = W4_WAVES * 64, ROWS = MT * 4 * RG, UPT = (ROWS * KB / 8 + THREADS - 1) / THREADS;
    typedef uint32_t Pairs __attribute__((ext_vector_type(TG)));
    extern __shared__ w4_u32x4 lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave / WK, wk = wave % WK, row = lane & 15, quad = lane >> 4;
    const int tiles = w4_tiles(A.K), blocks = (tiles + WK * TPW - 1) / (WK * TPW), bands = (A.N + W4_ROWS - 1) / W4_ROWS;
    const int held = MT == 1 ? A.M : ROWS; // rows of A in LDS
    const int plane = KB / 32 * held * 4;  // pieces of 16 bytes of a plane: [KB / 32][held][4], the four of a row's 32 columns swapped so that the lanes' reads meet no bank twice
    const uint8_t* w[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) w[nt] = A.w + (size_t)min((int)(blockIdx.x * WN + wn) * NT + nt, bands - 1) * tiles * w4_tile(G);

    w4_u32x4 codes[TPW][NT];
    Pairs pairs[TPW][NT];
    const auto ask = [&](int b, int j) {
        const int t = min((b * WK + wk) * TPW + j, tiles - 1);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            codes[j][nt] = *reinterpret_cast<const w4_u32x4*>(w[nt] + (size_t)t * w4_tile(G) + lane * 16);
            pairs[j][nt] = *reinterpret_cast<const Pairs*>(w[nt] + (size_t)t * w4_tile(G) + W4_CODES + row * (TG * 4));
        }
    };
    W4Raw<T> raw[UPT];
    const auto ask_a = [&](int b) { // unit u: piece u % 4 of row u / 4 % held of 32 columns u / (4 held)
#pragma unroll
        for (int i = 0; i < UPT; i++) {
            const int u = i * THREADS + threadIdx.x, m = u / 4 % held, k = b * KB + u / (4 * held) * 32 + u % 4 * 8;
            if (u < plane) {
                if (k < A.K) raw[i].load((const T*)A.a + (size_t)min(m, A.M - 1) * A.aStride + k);
                else raw[i].zero();
            }
        }
    };
    const auto put_a = [&]() {
#pragma unroll
        for (int i = 0; i < UPT; i++) {
            const int u = i * THREADS + threadIdx.x, m = u / 4 % held;
            if (u < plane) raw[i].put(lds + (u ^ (m >> 2 & 3)), plane);
        }
    };
    ask_a(0);
#pragma unroll
    for (int j = 0; j < TPW; j++) ask(0, j);

    const typename X::V one = X::ones();
    w4_f32x4 acc[NT][MT] = {};
    const w4_u32x4* mine[MT]; // this lane's piece of the first 32 columns
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int m = MT == 1 ? min(row / 4 * RG + min(row % 4, RG - 1), held - 1) : mt * 16 + row;
        mine[mt] = lds + m * 4 + (quad ^ (m >> 2 & 3));
    }
    for (int b = 0; b < blocks; b++) {
        if (b) __syncthreads();
        put_a();
        __syncthreads();
        if (b + 1 < blocks) ask_a(b + 1);
#pragma unroll
        for (int j = 0; j < TPW; j++) {
            if ((b * WK + wk) * TPW + j < tiles) {
#pragma unroll
                for (int g = 0; g < TG; g++) {
                    w4_f32x4 d[NT][MT] = {}, s[MT] = {};
#pragma unroll
                    for (int q = 0; q < S; q++) {
                        const int step = g * S + q;
                        typename X::V c[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) c[nt] = X::codes(codes[j][nt][step]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
                            for (int p = X::PLANES - 1; p >= 0; p--) {
                                const typename X::V a = __builtin_bit_cast(typename X::V, mine[mt][p * plane + ((wk * TPW + j) * 4 + step) * held * 4]);
                                s[mt] = X::mul(a, one, s[mt]);
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) d[nt][mt] = X::mul(a, c[nt], d[nt][mt]);
                            }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const float sc = kv_half(pairs[j][nt][g] >> 16), scale = sc * (1.f / X::UNIT), low = kv_half(pairs[j][nt][g] & 0xffffu) - sc * X::SHIFT;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int i = 0; i < RG; i++) acc[nt][mt][i] = fmaf(scale, d[nt][mt][i], fmaf(low, s[mt][i], acc[nt][mt][i]));
                    }
                }
            }
            if (b + 1 < blocks) ask(b + 1, j);
        }
    }
    // [WK][WN * NT][ROWS][16]
    __syncthreads();
    float* part = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < RG; i++) part[((wk * WN * NT + wn * NT + nt) * ROWS + mt * 16 + quad * RG + i) * 16 + row] = acc[nt][mt][i];
    __syncthreads();
    const auto sum = [&](int m, int n) { // element (m, n) of this workgroup's columns
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < WK; q++) v += part[((q * WN * NT + n / 16) * ROWS + m) * 16 + n % 16];
        return v;
    };
    constexpr int COLS = WN * NT * 16;
    if (A.swiglu) {
        for (int u = threadIdx.x; u < A.M * (COLS / 2); u += THREADS) {
            const int m = u / (COLS / 2), j = u % (COLS / 2), n = (int)blockIdx.x * (COLS / 2) + j;
            if (n >= A.N / 2) continue;
            const float gate = sum(m, 2 * j), up = sum(m, 2 * j + 1);
            w4_put((T*)A.c + (size_t)m * A.cStride + n, gate / (1.f + expf(-gate)) * up);
        }
    } else {
        for (int u = threadIdx.x; u < A.M * COLS; u += THREADS) {
            const int m = u / COLS, j = u % COLS, n = (int)blockIdx.x * COLS + j;
            if (n >= A.N) continue;
            float v = sum(m, j);
            if (A.r) v += w4_get((const T*)A.r + (size_t)m * A.rStride + n);
            w4_put((T*)A.c + (size_t)m * A.cStride + n, v);
        }
    }
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
static bool w4_type(int t) { return t == MLH_DTYPE_F32 || t == MLH_DTYPE_BF16 || t == MLH_DTYPE_F16; }

extern "C" uint64_t mlh_weights4_bytes(int N, int K, int group) {
    if (N < 1 || N > (1 << 20) || K < 32 || K > (1 << 17) || K % 32 || (group != 32 && group != 64 && group != 128)) return 0;
    return (uint64_t)((N + W4_ROWS - 1) / W4_ROWS) * w4_tiles(K) * w4_tile(group);
}

static std::string w4_check(const mlh_weights4* w) {
    if (!w) return "null weights";
    if (!mlh_weights4_bytes(w->N, w->K, w->group)) return "N must be 1 to 2^20, K a multiple of 32 up to 2^17, group 32, 64 or 128";
    if (!w->data || (uintptr_t)w->data % 16) return "data must be given and 16-byte aligned";
    return "";
}

static unsigned w4_grid(size_t units) { return (unsigned)std::min<size_t>((units + W4_WG - 1) / W4_WG, 1 << 20); }
static W4Args w4_args(const mlh_weights4* w) { return {(uint8_t*)w->data, w->N, w->K, (w->N + W4_ROWS - 1) / W4_ROWS * W4_ROWS, nullptr, nullptr, nullptr, 0}; }

#define W4_BY_GROUP(KERNEL_, ...) (w->group == 32 ? &KERNEL_<__VA_ARGS__ 32> : w->group == 64 ? &KERNEL_<__VA_ARGS__ 64> : &KERNEL_<__VA_ARGS__ 128>)
#define W4_COMMA ,

extern "C" int mlh_weights4_pack_device(const mlh_weights4* w, int type, const void* src, int64_t stride, void* stream) {
    std::string bad = w4_check(w);
    if (bad.empty() && !w4_type(type)) bad = "unknown type";
    if (bad.empty()) bad = kv_check_rows("src", src, stride, w->K, type);
    if (!bad.empty()) return kv_fail(bad);
    W4Args A = w4_args(w);
    A.src = src;
    A.stride = stride;
    const unsigned grid = w4_grid((size_t)A.rows * w4_tiles(A.K) * (W4_COLS / 8));
    if (type == MLH_DTYPE_F32) return kv_launch(W4_BY_GROUP(k_w4_pack, float W4_COMMA), dim3(grid), W4_WG, 0, stream, A);
    if (type == MLH_DTYPE_BF16) return kv_launch(W4_BY_GROUP(k_w4_pack, bf16_t W4_COMMA), dim3(grid), W4_WG, 0, stream, A);
    return kv_launch(W4_BY_GROUP(k_w4_pack, f16_t W4_COMMA), dim3(grid), W4_WG, 0, stream, A);
}

extern "C" int mlh_weights4_set_device(const mlh_weights4* w, const uint8_t* codes, const uint16_t* params, void* stream) {
    std::string bad = w4_check(w);
    if (bad.empty() && (!codes || !params)) bad = "null pointer: codes or params";
    if (bad.empty() && ((uintptr_t)codes | (uintptr_t)params) % 16) bad = "codes and params must be 16-byte aligned";
    if (!bad.empty()) return kv_fail(bad);
    W4Args A = w4_args(w);
    A.src = codes;
    A.params = (const uint32_t*)params;
    return kv_launch(W4_BY_GROUP(k_w4_set, ), dim3(w4_grid((size_t)A.rows * w4_tiles(A.K) * (W4_COLS / 8))), W4_WG, 0, stream, A);
}

extern "C" int mlh_weights4_read_device(const mlh_weights4* w, int type, void* dst, int64_t stride, void* stream) {
    std::string bad = w4_check(w);
    if (bad.empty() && !w4_type(type)) bad = "unknown type";
    if (bad.empty()) bad = kv_check_rows("dst", dst, stride, w->K, type);
    if (!bad.empty()) return kv_fail(bad);
    W4Args A = w4_args(w);
    A.dst = dst;
    A.stride = stride;
    const unsigned grid = w4_grid((size_t)A.N * (A.K / 8));
    if (type == MLH_DTYPE_F32) return kv_launch(W4_BY_GROUP(k_w4_read, float W4_COMMA), dim3(grid), W4_WG, 0, stream, A);
    if (type == MLH_DTYPE_BF16) return kv_launch(W4_BY_GROUP(k_w4_read, bf16_t W4_COMMA), dim3(grid), W4_WG, 0, stream, A);
    return kv_launch(W4_BY_GROUP(k_w4_read, f16_t W4_COMMA), dim3(grid), W4_WG, 0, stream, A);
}

static std::string gemm4_check(const mlh_weights4* w, const mlh_gemm4* a) {
    std::string bad = w4_check(w);
    if (!bad.empty()) return bad;
    if (!a) return "null arguments";
    if (!w4_type(a->type)) return "unknown row type";
    if (a->M < 0 || a->M > 64) return "M must be 0 to 64";
    if (a->swiglu != 0 && a->swiglu != 1) return "swiglu must be 0 or 1";
    if (a->swiglu && (w->N % 2 || a->r)) return "swiglu: N must be even, and there is no R";
    const int cols = a->swiglu ? w->N / 2 : w->N;
    bad = kv_check_rows("a", a->a, a->aStride, w->K, a->type);
    if (!bad.empty()) return bad;
    if (!a->c || (uintptr_t)a->c % kv_elem_bytes(a->type) || (uintptr_t)a->r % kv_elem_bytes(a->type)) return "c must be given, c and r aligned to their elements";
    if (a->cStride < cols || a->cStride > (1ll << 32)) return "c: stride smaller than a row, or beyond 2^32";
    if (a->r && ((a->rStride != 0 && a->rStride < cols) || a->rStride > (1ll << 32))) return "r: stride smaller than a row, or beyond 2^32";
    if (a->r == a->c && a->rStride != a->cStride) return "a residual in place must have the stride of c";
    if (a->a == a->c) return "c must not be a";
    return "";
}

extern "C" uint64_t mlh_gemm4_work_bytes(const mlh_weights4* w, const mlh_gemm4* a) { return 0; }

template <typename T, int G, int MT, int RG, int WN, int WK, int NT, int TPW> static int gemm4_run(const Gemm4Args& A, void* stream) {
    constexpr int planes = W4Mul<T>::PLANES, rows = MT * 4 * RG;
    const int held = MT == 1 ? A.M : rows;
    const size_t lds = std::max<size_t>((size_t)WK * TPW * W4_COLS * held * 2 * planes, (size_t)WK * WN * NT * rows * 16 * 4);
    const unsigned grid = ((A.N + W4_ROWS - 1) / W4_ROWS + WN * NT - 1) / (WN * NT);
    if (lds > 65536) { // (asked for on every call: the attribute belongs to the device that is current)
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_gemm4<T, G, MT, RG, WN, WK, NT, TPW>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return kv_status(e);
    }
    return kv_launch(&k_gemm4<T, G, MT, RG, WN, WK, NT, TPW>, dim3(grid), W4_WAVES * 64, lds, stream, A);
}

template <typename T, int G> static int gemm4_go(const Gemm4Args& A, void* stream) {
    static const int cfg = getenv("G4") ? atoi(getenv("G4")) : 0;
    if constexpr (sizeof(T) == 2) {
        if (A.M <= 4) return cfg == 1 ? gemm4_run<T, G, 1, 1, 1, 8, 1, 2>(A, stream) : cfg == 2 ? gemm4_run<T, G, 1, 1, 1, 8, 2, 2>(A, stream) : cfg == 3 ? gemm4_run<T, G, 1, 1, 2, 4, 1, 4>(A, stream) : gemm4_run<T, G, 1, 1, 1, 8, 1, 4>(A, stream);
        if (A.M <= 8) return cfg == 1 ? gemm4_run<T, G, 1, 2, 1, 8, 1, 2>(A, stream) : cfg == 2 ? gemm4_run<T, G, 1, 2, 1, 8, 2, 2>(A, stream) : cfg == 3 ? gemm4_run<T, G, 1, 2, 2, 4, 1, 4>(A, stream) : gemm4_run<T, G, 1, 2, 1, 8, 1, 4>(A, stream);
        if (A.M <= 16) return cfg == 1 ? gemm4_run<T, G, 1, 4, 1, 8, 1, 2>(A, stream) : cfg == 2 ? gemm4_run<T, G, 1, 4, 1, 8, 2, 2>(A, stream) : cfg == 3 ? gemm4_run<T, G, 1, 4, 2, 4, 2, 2>(A, stream) : gemm4_run<T, G, 1, 4, 1, 8, 2, 1>(A, stream);
        if (A.M <= 32) return cfg == 1 ? gemm4_run<T, G, 2, 4, 1, 8, 1, 1>(A, stream) : cfg == 2 ? gemm4_run<T, G, 2, 4, 2, 4, 1, 2>(A, stream) : cfg == 3 ? gemm4_run<T, G, 2, 4, 4, 2, 2, 2>(A, stream) : gemm4_run<T, G, 2, 4, 2, 4, 2, 2>(A, stream);
        return cfg == 1 ? gemm4_run<T, G, 4, 4, 2, 4, 1, 1>(A, stream) : cfg == 2 ? gemm4_run<T, G, 4, 4, 4, 2, 2, 2>(A, stream) : cfg == 3 ? gemm4_run<T, G, 4, 4, 4, 2, 1, 2>(A, stream) : gemm4_run<T, G, 4, 4, 2, 4, 2, 1>(A, stream);
    } else {
        if (A.M <= 4) return gemm4_run<T, G, 1, 1, 1, 8, 1, 2>(A, stream);
        if (A.M <= 16) return gemm4_run<T, G, 1, 4, 1, 8, 1, 1>(A, stream);
        if (A.M <= 32) return gemm4_run<T, G, 2, 4, 4, 2, 1, 1>(A, stream);
        return gemm4_run<T, G, 4, 4, 4, 2, 1, 1>(A, stream);
    }
}

extern "C" int mlh_gemm4_device(const mlh_weights4* w, const mlh_gemm4* a, void* stream) {
    const std::string bad = gemm4_check(w, a);
    if (!bad.empty()) return kv_fail(bad);
    if (a->M == 0) return 0;
    const Gemm4Args A = {(const uint8_t*)w->data, a->a, a->r, a->c, a->aStride, a->rStride, a->cStride, a->M, w->N, w->K, a->swiglu};
#define W4_GO(T_) return w->group == 32 ? gemm4_go<T_, 32>(A, stream) : w->group == 64 ? gemm4_go<T_, 64>(A, stream) : gemm4_go<T_, 128>(A, stream)
    if (a->type == MLH_DTYPE_F32) W4_GO(float);
    if (a->type == MLH_DTYPE_BF16) W4_GO(bf16_t);
    W4_GO(f16_t);
#undef W4_GO
}
