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
#define W4_WAVES 8   // waves of a product's workgroup that multiply

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

// A wave: a tile, as the lanes of a product hold it: lane l row l % 16, eight columns of each of the four steps.  The columns of a group are those of 1, 2 or 4 steps in the four lanes of a row.
// Bound by memory.  28672 columns of 8192 rows, groups of 32: codes laid out in 70 to 75 us, 3.9 to 4.2 TB/s (read four bytes at a time 99 us, and written so, 64 apart, 142), packed from bf16 in 153, 4.0 TB/s, read back in 170, 3.6.
struct W4Place { int n, k, lane; }; // row and first column of step 0
__device__ __forceinline__ W4Place w4_place(const W4Args& A, size_t tile) {
    const int perBand = w4_tiles(A.K), lane = threadIdx.x & 63;
    return {(int)(tile / perBand) * W4_ROWS + (lane & 15), (int)(tile % perBand) * W4_COLS + (lane >> 4) * 8, lane};
}
#define W4_EACH_TILE(PLACE_) \
    for (size_t tile = (size_t)blockIdx.x * (W4_WG / 64) + (threadIdx.x >> 6), tiles = (size_t)(A.rows / W4_ROWS) * w4_tiles(A.K); tile < tiles; tile += (size_t)gridDim.x * (W4_WG / 64)) \
        if (const W4Place PLACE_ = w4_place(A, tile); true)

template <typename T, int G>
__global__ void __launch_bounds__(W4_WG) k_w4_pack(W4Args A) {
    constexpr int S = G / 32, TG = w4_groups(G);
    W4_EACH_TILE(P) {
        float x[4][8];
        bool live[4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            live[s] = P.n < A.N && P.k + s * 32 < A.K;
            if (live[s]) kv_load8((const T*)A.src + (size_t)P.n * A.stride + P.k + s * 32, x[s]);
        }
        uint32_t pairs[TG], words[4];
#pragma unroll
        for (int g = 0; g < TG; g++) {
            float lo = INFINITY, hi = -INFINITY, bad = 0.f;
#pragma unroll
            for (int s = g * S; s < g * S + S; s++)
                if (live[s]) {
#pragma unroll
                    for (int i = 0; i < 8; i++) { lo = fminf(lo, x[s][i]); hi = fmaxf(hi, x[s][i]); bad += x[s][i] * 0.f; }
                }
#pragma unroll
            for (int o = 16; o < 64; o <<= 1) { lo = fminf(lo, __shfl_xor(lo, o, 64)); hi = fmaxf(hi, __shfl_xor(hi, o, 64)); bad += __shfl_xor(bad, o, 64); }
            float step = (hi - lo) * (1.0f / 15.0f);
            asm volatile("" : "+v"(step)); // (rounded to fp32 first; in one instruction with the conversion the product is not)
            uint32_t minBits = kv_to_half(__builtin_amdgcn_fmed3f(lo, -65504.f, 65504.f)), scaleBits = kv_to_half(step);
            const float base = kv_half(minBits), scale = kv_half(scaleBits);
            const bool none = lo > hi && bad == 0.f, odd = !none && (!(bad == 0.f) || scaleBits == 0x7c00u); // (nobody brought a value; a value is no number)
            if (none) minBits = scaleBits = 0;
            if (odd) { minBits = 0x7e00u; scaleBits = 0; }
            const float inv = 1.0f / scale;
#pragma unroll
            for (int s = g * S; s < g * S + S; s++) {
                uint32_t codes = 0;
                if (live[s] && !odd && scale > 0.f) {
#pragma unroll
                    for (int i = 0; i < 8; i++) codes |= kv_code(x[s][i], base, scale, inv) << (4 * i);
                }
                words[s] = w4_spread(codes);
            }
            pairs[g] = minBits | scaleBits << 16;
        }
        uint8_t* at = A.data + tile * w4_tile(G);
        *reinterpret_cast<w4_u32x4*>(at + P.lane * 16) = w4_u32x4{words[0], words[1], words[2], words[3]};
        if (P.lane < W4_ROWS) {
#pragma unroll
            for (int g = 0; g < TG; g++) *reinterpret_cast<uint32_t*>(at + W4_CODES + (P.lane * TG + g) * 4) = pairs[g];
        }
    }
}

template <int G>
__global__ void __launch_bounds__(W4_WG) k_w4_set(W4Args A) {
    constexpr int TG = w4_groups(G);
    W4_EACH_TILE(P) {
        // lane (row, q) loads the 32 columns of step q; its word of step s is word q of lane (row, s)
        const int q = P.lane >> 4, k = P.k - q * 8 + q * 32;
        w4_u32x4 step = {}, words = {};
        if (P.n < A.N && k < A.K) step = *reinterpret_cast<const w4_u32x4*>((const uint8_t*)A.src + ((size_t)P.n * A.K + k) / 2);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = q ^ i;
            const uint32_t give = p & 2 ? (p & 1 ? step[3] : step[2]) : (p & 1 ? step[1] : step[0]), take = w4_spread((uint32_t)__shfl_xor((int)give, 16 * i, 64));
#pragma unroll
            for (int s = 0; s < 4; s++) words[s] = s == p ? take : words[s];
        }
        uint8_t* at = A.data + tile * w4_tile(G);
        *reinterpret_cast<w4_u32x4*>(at + P.lane * 16) = words;
        if (P.lane < W4_ROWS) {
#pragma unroll
            for (int g = 0; g < TG; g++)
                *reinterpret_cast<uint32_t*>(at + W4_CODES + (P.lane * TG + g) * 4) = P.n < A.N && P.k + g * G < A.K ? A.params[(size_t)P.n * ((A.K + G - 1) / G) + (P.k + g * G) / G] : 0u;
        }
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(W4_WG) k_w4_read(W4Args A) {
    constexpr int S = G / 32, TG = w4_groups(G);
    W4_EACH_TILE(P) {
        const uint8_t* at = A.data + tile * w4_tile(G);
        const w4_u32x4 words = *reinterpret_cast<const w4_u32x4*>(at + P.lane * 16);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            float x[8];
            kv_values8(w4_gather(words[s]), *reinterpret_cast<const uint32_t*>(at + W4_CODES + ((P.lane & 15) * TG + s / S) * 4), x);
            if (P.n < A.N && P.k + s * 32 < A.K) kv_store8<false>((T*)A.dst + (size_t)P.n * A.stride + P.k + s * 32, x);
        }
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

// Columns 2j and 2j + 1 of a word of codes, each in bits 3 to 6 of a half
template <int J> __device__ __forceinline__ uint32_t w4_turn(uint32_t x) { return J == 0 ? x : J == 3 ? __builtin_amdgcn_alignbit(x, x, 12) : x >> (4 * J); }

// How codes and activations meet on the matrix cores; every product there is exact.  PLANES: of an activation.  codes(x): a word of eight codes as an operand that stands for UNIT * (code + SHIFT); unit(): one of UNIT.
template <typename T> struct W4Mul;
template <> struct W4Mul<f16_t> { // codes as halves below 2^-14, code * 2^-21
    static constexpr int PLANES = 1;
    static constexpr float UNIT = 0x1p-21f, SHIFT = 0.f;
    typedef w4_f16x8 V;
    static __device__ __forceinline__ V codes(uint32_t x) {
        return __builtin_bit_cast(V, w4_u32x4{w4_turn<0>(x) & 0x00780078u, w4_turn<1>(x) & 0x00780078u, w4_turn<2>(x) & 0x00780078u, w4_turn<3>(x) & 0x00780078u});
    }
    static __device__ __forceinline__ V unit(bool on = true) { const uint32_t u = on ? 0x00080008u : 0u; return __builtin_bit_cast(V, w4_u32x4{u, u, u, u}); }
    static __device__ __forceinline__ w4_f32x4 mul(V a, V b, w4_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct W4Mul<bf16_t> { // codes behind 16: a bf16 of 16 + code has the code in bits 3 to 6
    static constexpr int PLANES = 1;
    static constexpr float UNIT = 1.f, SHIFT = 16.f;
    typedef w4_bf16x8 V;
    static __device__ __forceinline__ V codes(uint32_t x) {
        uint32_t base = 0x41804180u;
        asm("" : "+v"(base)); // (a register: with two literals the mask and the base would take an instruction each)
        return __builtin_bit_cast(V, w4_u32x4{(w4_turn<0>(x) & 0x00780078u) | base, (w4_turn<1>(x) & 0x00780078u) | base, (w4_turn<2>(x) & 0x00780078u) | base, (w4_turn<3>(x) & 0x00780078u) | base});
    }
    static __device__ __forceinline__ V unit(bool on = true) { const uint32_t u = on ? 0x3f803f80u : 0u; return __builtin_bit_cast(V, w4_u32x4{u, u, u, u}); }
    static __device__ __forceinline__ w4_f32x4 mul(V a, V b, w4_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct W4Mul<float> : W4Mul<bf16_t> { // the same with activations as three planes (p3.h): every product exact
    static constexpr int PLANES = 3;
};

__device__ __forceinline__ float w4_get(const float* p) { return *p; }
__device__ __forceinline__ float w4_get(const bf16_t* p) { return kv_bf16(*p); }
__device__ __forceinline__ float w4_get(const f16_t* p) { return kv_half(p->bits); }
__device__ __forceinline__ void w4_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void w4_put(bf16_t* p, float v) { *p = (bf16_t)kv_to_bf16(v); }
__device__ __forceinline__ void w4_put(f16_t* p, float v) { p->bits = (uint16_t)kv_to_half(v); }

// Eight neighbouring elements of a row of A: as loaded, and as the operands that are multiplied
template <typename T> struct W4Raw {
    w4_u32x4 x;
    __device__ __forceinline__ void load(const T* p) { x = *reinterpret_cast<const w4_u32x4*>(p); }
    __device__ __forceinline__ void zero() { x = w4_u32x4{}; }
    __device__ __forceinline__ void split(w4_u32x4 (&v)[1]) const { v[0] = x; }
};
template <> struct W4Raw<float> {
    w4_u32x4 x[2];
    __device__ __forceinline__ void load(const float* p) { x[0] = *reinterpret_cast<const w4_u32x4*>(p); x[1] = *reinterpret_cast<const w4_u32x4*>(p + 4); }
    __device__ __forceinline__ void zero() { x[0] = x[1] = w4_u32x4{}; }
    __device__ __forceinline__ void split(w4_u32x4 (&v)[3]) const {
        uint32_t s[4][3];
#pragma unroll
        for (int i = 0; i < 4; i++) p3_split2(__uint_as_float(x[i / 2][i % 2 * 2]), __uint_as_float(x[i / 2][i % 2 * 2 + 1]), s[i]);
#pragma unroll
        for (int pl = 0; pl < 3; pl++) v[pl] = w4_u32x4{s[0][pl], s[1][pl], s[2][pl], s[3][pl]};
    }
};

// The epilogue of BANDS times 16 columns: sum(m, n) is their element (m, n)
template <typename T, int BANDS, int THREADS, typename F> __device__ __forceinline__ void w4_finish(const Gemm4Args& A, F sum) {
    constexpr int COLS = BANDS * 16;
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

// This workgroup's rows of A, ROWS at most.
template <typename T, int ROWS> __device__ __forceinline__ void w4_rows(Gemm4Args& A) {
    const int first = (int)blockIdx.y * ROWS;
    A.M = min(A.M - first, ROWS);
    A.a = (const T*)A.a + first * A.aStride;
    if (A.r) A.r = (const T*)A.r + first * A.rStride;
    A.c = (T*)A.c + first * A.cStride;
}

// Products with minimum and scale behind the sums: the sum over a group of a (min + scale code) is (scale D + (min - scale SHIFT) S) / UNIT, D the sum of a UNIT (code + SHIFT) and S that of
// a UNIT; both come from the matrix cores, S as a product with UNIT.  All of it is fp32.  With SHIFT 16 the roundings of min - 16 scale and of its product
// with S are up to 2^-19 of the scale in a weight, those of D (fp32 rows: a (16 + code) has up to 29 bits) and its product with the scale 62 2^-24, where quantising leaves half the scale; codes that
// stand for themselves would take another instruction a pair, min and 16 scale applied apart another matrix instruction of 32 cycles for every 128 of 16-bit products.  Lane l of a result holds column l % 16 (a row of W) and the instruction's rows 4 (l / 16) + i, i = 0 .. 3.
//
// Few rows, four in an operand: the instruction's row 4 m + s is row m of A in the s-th 32 columns of a tile, so that one load brings a tile's share of A to the lanes that multiply it and the product with
// the s-th step's codes has that step's sums, of row m, in element s of lanes 16 m to 16 m + 15.  (The other elements are of rows and codes that do not belong together.)  One product with UNIT gives the S of
// all four steps.  No LDS and no barrier but for the sums of WK waves at the end.
// A workgroup is WN x WK waves, WN * NT * 16 rows of W; a wave has TPW tiles of its share of K on their way.
// Bound by memory where W is large (5 rows, N 8192, K 28672, groups of 32, fp16: 147 MB in 28 us, 5.2 TB/s), else by the latency of a start, of a wave's first tiles and of its last sums (1 row, N 11264,
// K 2048, groups of 64, bf16: 13 MB in 4.9 us).
template <typename T, int G, int MR, int WN, int WK, int NT, int TPW>
__global__ void __launch_bounds__(W4_WAVES * 64) k_gemm4_few(Gemm4Args A) {
    typedef W4Mul<T> X;
    constexpr int S = G / 32, TG = w4_groups(G);
    static_assert(WN * WK == W4_WAVES, "waves");
    typedef uint32_t Pairs __attribute__((ext_vector_type(TG)));
    __shared__ float part[WK][WN * NT][MR][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave / WK, wk = wave % WK, row = lane & 15, quad = lane >> 4;
    w4_rows<T, MR * 4>(A);
    const int tiles = w4_tiles(A.K), bands = (A.N + W4_ROWS - 1) / W4_ROWS, k0 = (row & 3) * 32 + quad * 8;
    const uint8_t* w[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) w[nt] = A.w + (size_t)min((int)(blockIdx.x * WN + wn) * NT + nt, bands - 1) * tiles * w4_tile(G);
    const T* from[MR];
#pragma unroll
    for (int r = 0; r < MR; r++) from[r] = (const T*)A.a + (size_t)min(r * 4 + (row >> 2), A.M - 1) * A.aStride;

    w4_u32x4 codes[TPW][NT];
    Pairs pairs[TPW][NT];
    W4Raw<T> raw[TPW][MR];
    const auto ask = [&](int t, int j) { // (behind the end the last tile again, so that there is always as much on its way)
        t = min(t, tiles - 1);
        const int k = min(t * W4_COLS + k0, A.K - 8);
#pragma unroll
        for (int r = 0; r < MR; r++) raw[j][r].load(from[r] + k);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint8_t* at = w[nt] + (size_t)t * w4_tile(G);
            codes[j][nt] = *reinterpret_cast<const w4_u32x4*>(at + lane * 16);
            pairs[j][nt] = *reinterpret_cast<const Pairs*>(at + W4_CODES + row * (TG * 4));
        }
    };
#pragma unroll
    for (int j = 0; j < TPW; j++) ask(j * WK + wk, j);
    const typename X::V unit = X::unit();
    float acc[NT][MR] = {};
    for (int t0 = wk; t0 < tiles; t0 += WK * TPW) {
#pragma unroll
        for (int j = 0; j < TPW; j++) {
            const int t = t0 + j * WK;
            if (t < tiles) {
                if (t * W4_COLS + W4_COLS > A.K && t * W4_COLS + k0 >= A.K) {
#pragma unroll
                    for (int r = 0; r < MR; r++) raw[j][r].zero();
                }
                w4_u32x4 a[MR][X::PLANES];
                w4_f32x4 s[MR] = {};
#pragma unroll
                for (int r = 0; r < MR; r++) {
                    raw[j][r].split(a[r]);
#pragma unroll
                    for (int p = X::PLANES - 1; p >= 0; p--) s[r] = X::mul(__builtin_bit_cast(typename X::V, a[r][p]), unit, s[r]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int step = 0; step < 4; step++) {
                        const int g = step / S;
                        const typename X::V c = X::codes(codes[j][nt][step]);
                        const float scale = kv_half(pairs[j][nt][g] >> 16), low = kv_half(pairs[j][nt][g] & 0xffffu) - scale * X::SHIFT;
#pragma unroll
                        for (int r = 0; r < MR; r++) {
                            w4_f32x4 d = {};
#pragma unroll
                            for (int p = X::PLANES - 1; p >= 0; p--) d = X::mul(__builtin_bit_cast(typename X::V, a[r][p]), c, d);
                            acc[nt][r] = fmaf(scale, d[step], acc[nt][r]);
                            if (step % S == S - 1) {
                                float sum = s[r][g * S];
#pragma unroll
                                for (int q = 1; q < S; q++) sum += s[r][g * S + q];
                                acc[nt][r] = fmaf(low, sum, acc[nt][r]);
                            }
                        }
                    }
                }
            }
            ask(t + WK * TPW, j);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int r = 0; r < MR; r++) part[wk][wn * NT + nt][r][lane] = acc[nt][r] * (1.f / X::UNIT);
    __syncthreads();
    w4_finish<T, WN * NT, W4_WAVES * 64>(A, [&](int m, int n) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < WK; q++) v += part[q][n / 16][m / 4][m % 4 * 16 + n % 16];
        return v;
    });
}

// More rows, MT times 16 of them a workgroup: the instruction's rows are rows of A.  A goes through LDS, once for all waves of a workgroup, a block of WK * TPW tiles of K at a time and two blocks in turn; LOADERS
// further waves bring it there, since loads come back in the order they were asked for: a wave that waits for A, which is near, would wait for codes that are far and not needed yet.  Wave (wn, wk) of the
// others multiplies TPW tiles of every block with its NT times 16 rows of W, whose codes it asks for AHEAD blocks ahead.
// S does not depend on W: the loaders take it, with UNIT in the four rows of the instruction that belong to a group and zeros in the others, so that four groups add up in one result and stand where
// v_mfma_f32_16x16x4_f32 wants them, which multiplies four groups' S with their minima at once, in fp32.  (With S and its products in every multiplying wave fp32 took 5 to 12 % longer, groups of 32 up to 15 %.)
// Groups of 128 are two of 64 here, for fewer registers.  Eight loaders where the registers of 16 waves hold the shape (S and A in time: fp32, 16 rows, 7.8 us for 8.8 at 128 bands), four elsewhere.
// 64 rows, N 28672, K 8192, groups of 64, fp16 take 50 us, 600 TFLOP/s, twice what the matrix cores alone need.  Left out in turn (before the loaders took S, of 55 to 60 us), the loads of W saved 13 us, A's out of LDS 6,
// the loaders 2, and all three half the time: the three wait for each other; two and three blocks of codes ahead, other waves and shares were no faster.
// In LDS piece q (eight columns) of step s (32 columns) of row m stands at [m][s ^ (m / 4 % 4)][q ^ (m % 4)], so that neither the lanes of a store, which share a row, nor those of a load, which share
// step and piece, meet in a bank.
__host__ __device__ constexpr int w4_sums_at(int buf, int part) { return 2 * buf > part ? 2 * buf : part; } // bytes in front of the sums: two blocks of A, later the waves' results
template <typename T, int G, int MT, int WN, int WK, int NT, int TPW, int AHEAD, int LOADERS>
__global__ void __launch_bounds__((W4_WAVES + LOADERS) * 64) k_gemm4_many(Gemm4Args A) {
    typedef W4Mul<T> X;
    constexpr int S = G < 64 ? 1 : 2, TG = 4 / S, LOADED = w4_groups(G), ROWS = MT * 16, STEPS = WK * TPW * 4, PIECES = STEPS * 4, PLANE = ROWS * PIECES, BUF = PLANE * X::PLANES;
    constexpr int FOURS = (TPW * TG + 3) / 4; // groups of a wave's share of a block, by four
    typedef uint32_t Pairs __attribute__((ext_vector_type(LOADED)));
    extern __shared__ w4_u32x4 lds[];
    w4_rows<T, ROWS>(A);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = w4_tiles(A.K), blocks = (tiles + WK * TPW - 1) / (WK * TPW);
    const int wn = wave / WK, wk = wave % WK, row = lane & 15, quad = lane >> 4;
    float* part = reinterpret_cast<float*>(lds); // [WK][WN * NT][ROWS][16], at the end
    float* sums = reinterpret_cast<float*>(lds) + w4_sums_at(BUF * 16, WK * WN * NT * ROWS * 64) / 4; // of blocks in turn, [2][WK][MT][FOURS][64]
    int at[4]; // this lane's piece of step s of a block's first tile, in its first 16 rows
#pragma unroll
    for (int s = 0; s < 4; s++) at[s] = (row * STEPS + (s ^ (row >> 2 & 3))) * 4 + (quad ^ (row & 3));
    if (wave >= W4_WAVES) {
        constexpr int THREADS = LOADERS * 64, UNITS = PLANE / THREADS, EVERY = THREADS / PIECES; // EVERY: rows from one of a thread's pieces to the next
        static_assert(WN * WK == W4_WAVES && PIECES <= THREADS && PLANE % THREADS == 0, "waves, pieces of A");
        const int thread = threadIdx.x - W4_WAVES * 64, row0 = PIECES < 64 ? thread / PIECES : (wave - W4_WAVES) * 64 / PIECES, piece = thread % PIECES;
        W4Raw<T> raw[UNITS];
        const T* from[UNITS]; // rows, the last one again behind the end
#pragma unroll
        for (int i = 0; i < UNITS; i++) from[i] = (const T*)A.a + (size_t)min(row0 + i * EVERY, A.M - 1) * A.aStride;
        const auto ask = [&](int b) { // (behind the end of a row its last piece again)
            const unsigned k = min(b * (STEPS * 32) + piece * 8, A.K - 8);
#pragma unroll
            for (int i = 0; i < UNITS; i++) raw[i].load(from[i] + k);
        };
        // the place of row m's piece: EVERY divides or is a multiple of 4, so that the bits of m that are swapped in are those of row0 and of i * EVERY put together
        const int place = row0 * PIECES + (((piece >> 2) ^ (row0 >> 2 & 3)) * 4 | ((piece & 3) ^ (row0 & 3)));
        const auto put = [&](int b) {
            w4_u32x4* const buf = lds + (b & 1) * BUF;
            if ((b + 1) * (STEPS * 32) > A.K && b * (STEPS * 32) + piece * 8 >= A.K) {
#pragma unroll
                for (int i = 0; i < UNITS; i++) raw[i].zero();
            }
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                w4_u32x4 v[X::PLANES];
                raw[i].split(v);
#pragma unroll
                for (int p = 0; p < X::PLANES; p++) buf[(place ^ ((i * EVERY >> 2 & 3) * 4 | (i * EVERY & 3))) + (p * PLANE + i * EVERY * PIECES)] = v[p];
            }
        };
        // S of block b, four groups in a result: the instruction's rows of UNIT are where the group's lanes are, the others zero
        const auto take = [&](int b) {
            const w4_u32x4* const buf = lds + (b & 1) * BUF;
            for (int u = wave - W4_WAVES; u < WK * MT * FOURS; u += LOADERS) { // [WK][MT][FOURS]
                const w4_u32x4* const from = buf + u / FOURS % MT * 16 * PIECES + (u / FOURS / MT * TPW + u % FOURS * 4 / TG) * 16;
                w4_f32x4 s[4] = {};
#pragma unroll
                for (int g = 0; g < 4 && g < TPW * TG; g++) {
                    const typename X::V unit = X::unit(row >> 2 == g);
#pragma unroll
                    for (int q = 0; q < S; q++)
#pragma unroll
                        for (int p = X::PLANES - 1; p >= 0; p--) s[g] = X::mul(unit, __builtin_bit_cast(typename X::V, from[p * PLANE + at[g % TG * S + q] + g / TG * 16]), s[g]);
                }
                sums[((b & 1) * WK * MT * FOURS + u) * 64 + lane] = (s[0][0] + s[1][0]) + (s[2][0] + s[3][0]);
            }
        };
        ask(0);
        put(0);
        ask(1);
        __syncthreads();
        for (int b = 0; b < blocks; b++) { // (while the others multiply block b)
            take(b);
            if (b + 1 < blocks) put(b + 1);
            ask(b + 2);
            __syncthreads();
        }
    } else {
        const int bands = (A.N + W4_ROWS - 1) / W4_ROWS;
        const uint8_t* w[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) w[nt] = A.w + (size_t)min((int)(blockIdx.x * WN + wn) * NT + nt, bands - 1) * tiles * w4_tile(G);
        w4_u32x4 codes[AHEAD][TPW][NT];
        Pairs pairs[AHEAD][TPW][NT];
        const auto ask = [&](int b, int a, int j) { // (behind the end the last tile again, so that there is always as much on its way)
            const int t = min((b * WK + wk) * TPW + j, tiles - 1);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint8_t* at = w[nt] + (size_t)t * w4_tile(G);
                codes[a][j][nt] = *reinterpret_cast<const w4_u32x4*>(at + lane * 16);
                pairs[a][j][nt] = *reinterpret_cast<const Pairs*>(at + W4_CODES + row * (LOADED * 4));
            }
        };
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
#pragma unroll
            for (int j = 0; j < TPW; j++) ask(a, a, j);
        w4_f32x4 acc[NT][MT] = {};
        uint32_t lows[NT][FOURS] = {}; // the pair of this lane's row and group of each four
        // S times (min - scale SHIFT) for the block behind the last barrier: four groups in an instruction of fp32.  What it reads, and its products: with few rows at
        // the end of the next block, where nothing waits for the LDS (16 rows, 1792 bands 28 us for 31), with more at once, for want of registers
        float low[NT][FOURS], s[MT][FOURS];
        const auto minima = [&](int b) {
#pragma unroll
            for (int f = 0; f < FOURS; f++) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) s[mt][f] = sums[((((b & 1) * WK + wk) * MT + mt) * FOURS + f) * 64 + lane];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) low[nt][f] = kv_half(lows[nt][f] & 0xffffu) - kv_half(lows[nt][f] >> 16) * X::SHIFT;
            }
        };
        const auto multiply = [&] {
#pragma unroll
            for (int f = 0; f < FOURS; f++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) acc[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[mt][f], low[nt][f], acc[nt][mt], 0, 0, 0);
        };
        __syncthreads();
        for (int b0 = 0; b0 < blocks; b0 += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const int b = b0 + u;
                if (b < blocks) {
                    const w4_u32x4* const buf = lds + (b & 1) * BUF;

                    // Sixteen rows of A by a group of columns at a time; A's pieces for the next ones are asked for in front of the products, between which the scales of the last ones are applied.
                    // (Behind the last tile A is zero.)
                    constexpr int PARTS = TPW * TG * MT;
                    typename X::V a[2][S][X::PLANES];
                    const auto fetch = [&](int i) {
#pragma unroll
                        for (int q = 0; q < S; q++)
#pragma unroll
                            for (int p = 0; p < X::PLANES; p++)
                                a[i & 1][q][p] = __builtin_bit_cast(typename X::V, buf[p * PLANE + at[i / MT % TG * S + q] + i % MT * 16 * PIECES + (wk * TPW + i / MT / TG) * 16]);
                    };
                    fetch(0);
                    typename X::V c[S][NT];
                    float scale[2][NT];
                    w4_f32x4 d[2][NT];
                    if (b > 0) {
                        minima(b - 1);
                        if (MT > 1) multiply();
                    }
                    const auto apply = [&](int i) {
                        const int mt = i % MT, h = i / MT & 1;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[nt][mt][e] = fmaf(scale[h][nt], d[i & 1][nt][e], acc[nt][mt][e]);
                    };
#pragma unroll
                    for (int i = 0; i < PARTS; i++) {
                        const int mt = i % MT, g = i / MT % TG, j = i / MT / TG, h = i / MT & 1;
                        if (i + 1 < PARTS) fetch(i + 1);
                        if (mt == 0) {
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                                for (int q = 0; q < S; q++) c[q][nt] = X::codes(codes[u][j][nt][g * S + q]);
                                scale[h][nt] = kv_half(pairs[u][j][nt][g * LOADED / TG] >> 16);
                                lows[nt][(j * TG + g) / 4] = quad == (j * TG + g) % 4 ? pairs[u][j][nt][g * LOADED / TG] : (j * TG + g) % 4 ? lows[nt][(j * TG + g) / 4] : 0u;
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) d[i & 1][nt] = w4_f32x4{};
#pragma unroll
                        for (int q = 0; q < S; q++)
#pragma unroll
                            for (int p = X::PLANES - 1; p >= 0; p--) {
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) d[i & 1][nt] = X::mul(a[i & 1][q][p], c[q][nt], d[i & 1][nt]);
                            }
                        if (i > 0) apply(i - 1);
                        if (mt == MT - 1 && g == TG - 1) ask(b + AHEAD, u, j);
                    }
                    if (MT == 1 && b > 0) multiply();
                    apply(PARTS - 1);
                    __syncthreads();
                }
            }
        }
        minima(blocks - 1);
        multiply();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) part[((wk * WN * NT + wn * NT + nt) * ROWS + mt * 16 + quad * 4 + i) * 16 + row] = acc[nt][mt][i] * (1.f / X::UNIT);
    }
    __syncthreads();
    w4_finish<T, WN * NT, (W4_WAVES + LOADERS) * 64>(A, [&](int m, int n) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < WK; q++) v += part[((q * WN * NT + n / 16) * ROWS + m) * 16 + n % 16];
        return v;
    });
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

static unsigned w4_grid(const W4Args& A) { return (unsigned)std::min<size_t>(((size_t)(A.rows / W4_ROWS) * w4_tiles(A.K) + W4_WG / 64 - 1) / (W4_WG / 64), 1 << 20); }
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
    const unsigned grid = w4_grid(A);
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
    return kv_launch(W4_BY_GROUP(k_w4_set, ), dim3(w4_grid(A)), W4_WG, 0, stream, A);
}

extern "C" int mlh_weights4_read_device(const mlh_weights4* w, int type, void* dst, int64_t stride, void* stream) {
    std::string bad = w4_check(w);
    if (bad.empty() && !w4_type(type)) bad = "unknown type";
    if (bad.empty()) bad = kv_check_rows("dst", dst, stride, w->K, type);
    if (!bad.empty()) return kv_fail(bad);
    W4Args A = w4_args(w);
    A.dst = dst;
    A.stride = stride;
    const unsigned grid = w4_grid(A);
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

template <typename T, int G, int MR, int WN, int WK, int NT, int TPW> static int gemm4_few(const Gemm4Args& A, void* stream) {
    const unsigned grid = ((A.N + W4_ROWS - 1) / W4_ROWS + WN * NT - 1) / (WN * NT);
    return kv_launch(&k_gemm4_few<T, G, MR, WN, WK, NT, TPW>, dim3(grid, (A.M + MR * 4 - 1) / (MR * 4)), W4_WAVES * 64, 0, stream, A);
}
template <typename T, int G, int MT, int WN, int WK, int NT, int TPW, int AHEAD, int LOADERS> static int gemm4_many(const Gemm4Args& A, void* stream) {
    constexpr int rows = MT * 16, lds = w4_sums_at(WK * TPW * 4 * rows * 64 * W4Mul<T>::PLANES, WK * WN * NT * rows * 16 * 4) + 2 * WK * MT * ((TPW * (G < 64 ? 4 : 2) + 3) / 4) * 256;
    static_assert(lds <= 163840, "LDS of a compute unit");
    const unsigned grid = ((A.N + W4_ROWS - 1) / W4_ROWS + WN * NT - 1) / (WN * NT);
    if (lds > 65536) { // (asked for on every call: the attribute belongs to the device that is current)
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_gemm4_many<T, G, MT, WN, WK, NT, TPW, AHEAD, LOADERS>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return kv_status(e);
    }
    return kv_launch(&k_gemm4_many<T, G, MT, WN, WK, NT, TPW, AHEAD, LOADERS>, dim3(grid, (A.M + rows - 1) / rows), (W4_WAVES + LOADERS) * 64, lds, stream, A);
}

// A workgroup's share of a product of more than four rows: rows of A times 16-row bands of W, and what a round of such workgroups, one a compute unit, takes (tenths of a us at N 2048, K 8192, fp32 or
// fp16, groups of 64).  Large shares read A and W less often, small ones fill the chip when there are few: taken is the share whose rounds take least.  With every share
// forced in turn, 5 to 64 rows of 48 to 1792 bands, fp16 and fp32, groups of 32 to 128, the one taken was within 7 % of the fastest at K 2048 and 4096, 10 % at 8192 and 16384, 15 % at 32768; where K is shorter
// than 2048, starts count for more than these times say: up to 18 % at K 1024, 30 % at 512, half more at 256 (fp32, 64 rows, 1280 bands 14.6 for 9.8).  For instance, us with the share taken / the next ones, fp16, K 4096: 64 rows, 256 bands 16 x 4 8.8 / 32 x 4 10.9, 16 x 8 11.8; 1024 bands 32 x 8 18.6 / 32 x 4 25.4, 64 x 8 26.8;
// 1280 bands 64 x 8 27.4 / 32 x 8 31.9; 32 rows, 1024 bands 32 x 4 14.9 / 16 x 8 15.2, 32 x 8 18.0; 16 rows, 256 bands 16 x 1 5.6 / 16 x 2 7.0, 16 x 4 8.1; fp32: 8 rows, 256 bands 8 x 1 7.7 / 8 x 2 9.1,
// 16 x 2 10.7; 64 rows, 256 bands 16 x 4 13.4 / 16 x 8 17.5,
// 16 x 2 20.0, 32 x 8 26.3.  (64 x 4 takes longer than 32 x 8 everywhere: 21.1 for 18.6.)
struct W4Share { int rows, bands, us; };
static int w4_share(const W4Share* s, int n, int M, int bands) {
    int best = 0;
    long long least = -1;
    for (int i = 0; i < n; i++) {
        const long long groups = (long long)((M + s[i].rows - 1) / s[i].rows) * ((bands + s[i].bands - 1) / s[i].bands), us = (groups + 255) / 256 * s[i].us;
        if (least < 0 || us < least) { least = us; best = i; }
    }
    return best;
}

// Up to four rows a band is a workgroup's eight waves; four bands where there are many and their last round over the compute units is not mostly empty: fewer starts, but fewer codes on their way, which
// counts with long K of 16-bit types.  Us, one band / four, fp16, groups of 32: 1024 bands, K 4096 10.6 / 10.8; 1280, K 4096 13.2 / 15.5; 1792, K 8192 29.8 / 30.7; 2000, K 2048 11.2 / 10.5; 256, K 4096
// 4.7 / 8.1; fp32 the same five 15.6 / 14.2, 19.0 / 20.0, 44.7 / 39.7, 19.2 / 13.5, 6.2 / 11.8.
template <typename T, int G> static int gemm4_go(const Gemm4Args& A, void* stream) {
    constexpr bool f32 = sizeof(T) == 4;
    const int bands = (A.N + W4_ROWS - 1) / W4_ROWS;
    if (A.M <= 4) return bands >= 1024 && bands >= (bands + 1023) / 1024 * 768 && (f32 || A.K <= 4096) ? gemm4_few<T, G, 1, 2, 4, 2, 2>(A, stream) : gemm4_few<T, G, 1, 1, 8, 1, 2>(A, stream);
    if constexpr (f32) {
        static const W4Share shares[] = {{8, 1, 120}, {8, 2, 141}, {16, 2, 174}, {16, 4, 209}, {16, 8, 304}, {32, 8, 488}};
        switch (w4_share(shares, 6, A.M, bands)) {
        case 0: return gemm4_few<T, G, 2, 1, 8, 1, 2>(A, stream);
        case 1: return gemm4_few<T, G, 2, 1, 8, 2, 2>(A, stream);
        case 2: return gemm4_many<T, G, 1, 2, 4, 1, 1, 2, 8>(A, stream);
        case 3: return gemm4_many<T, G, 1, 2, 4, 2, 1, 2, 8>(A, stream);
        case 4: return gemm4_many<T, G, 1, 4, 2, 2, 2, 1, 4>(A, stream);
        default: return gemm4_many<T, G, 2, 4, 2, 2, 1, 1, 8>(A, stream);
        }
    } else {
        static const W4Share shares[] = {{8, 1, 77}, {8, 2, 94}, {16, 1, 80}, {16, 2, 103}, {16, 4, 124}, {16, 8, 192}, {32, 4, 171}, {32, 8, 264}, {64, 8, 406}};
        switch (w4_share(shares, 9, A.M, bands)) {
        case 0: return gemm4_few<T, G, 2, 1, 8, 1, 2>(A, stream);
        case 1: return gemm4_few<T, G, 2, 1, 8, 2, 2>(A, stream);
        case 2: return gemm4_few<T, G, 4, 1, 8, 1, 2>(A, stream);
        case 3: return gemm4_few<T, G, 4, 1, 8, 2, 2>(A, stream);
        case 4: return gemm4_many<T, G, 1, 2, 4, 2, 2, 1, 8>(A, stream);
        case 5: return gemm4_many<T, G, 1, 4, 2, 2, 2, 2, G == 64 ? 8 : 4>(A, stream);
        case 6: return gemm4_many<T, G, 2, 2, 4, 2, 2, 1, 8>(A, stream);
        case 7: return gemm4_many<T, G, 2, 4, 2, 2, 2, 1, 4>(A, stream);
        default: return gemm4_many<T, G, 4, 4, 2, 2, 2, 1, 4>(A, stream);
        }
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
