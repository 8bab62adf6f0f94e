// Rotary positions of a caller's rows (mlh_rotate_device).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"

#define ROT_WG 256
#define ROT_LDS 8192 // bytes of cosines and sines: two rows of 512 turned elements in 64 bits

struct RotateArgs {
    const void *q, *k;
    void *qOut, *kOut;
    long long qStride, qOutStride, kStride, kOutStride;
    const int32_t* pos;
    const double* freq;
    int rows, heads, kvHeads, hd, rotated, rowsAtOnce;
    bool copy; // elements behind the turned ones
    double amplitude;
};

// V neighbouring elements, which stand on a multiple of their size, <-> floats
__device__ __forceinline__ float rot_get(float v) { return v; }
__device__ __forceinline__ float rot_get(bf16_t v) { return kv_bf16(v); }
__device__ __forceinline__ float rot_get(f16_t v) { return kv_half(v.bits); }
__device__ __forceinline__ void rot_put(float& p, float v) { p = v; }
__device__ __forceinline__ void rot_put(bf16_t& p, float v) { p = (bf16_t)kv_to_bf16(v); }
__device__ __forceinline__ void rot_put(f16_t& p, float v) { p.bits = (uint16_t)kv_to_half(v); }
template <typename T, int V> struct __align__(sizeof(T) * V) RotVec { T v[V]; };
template <int V, typename T> __device__ __forceinline__ void rot_load(const T* p, float (&x)[V]) {
    if constexpr (V == 8) kv_load8(p, x);
    else {
        const RotVec<T, V> r = *reinterpret_cast<const RotVec<T, V>*>(p);
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = rot_get(r.v[i]);
    }
}
template <bool NT, int V, typename T> __device__ __forceinline__ void rot_store(T* p, const float (&x)[V]) {
    if constexpr (V == 8) kv_store8<NT>(p, x);
    else {
        RotVec<T, V> r;
#pragma unroll
        for (int i = 0; i < V; i++) rot_put(r.v[i], x[i]);
        *reinterpret_cast<RotVec<T, V>*>(p) = r;
    }
}

// A workgroup takes a few rows at a time: their cosines and sines once, into LDS, for all heads, then the heads.  The angle is counted in half turns, of which sincospi takes the whole ones off exactly.
// A piece is V elements of a head: with halves the two times V that are V pairs, with pairs V neighbours, or V elements behind the turned ones.
// Bound by memory: 16384 rows of 32 + 8 heads of 128 in bf16, 336 MB read and written, 58 us (5.8 TB/s; a copy of 1 GiB 5.2), fp32 rows 63 us for as many bytes (5.3).  Narrower pieces take longer: 8192 rows of the same heads in bf16, halves, 20 turned
// of 80 (two elements a piece) 50 us, 2.1 TB/s, 24 of 96 (four) 41, 3.1, 62 of 128 (one) 104, 1.6.  A single token 2.6 us, the latency
// of position, angle and LDS in turn.  Rows at once: about as many as give every thread a piece; of 40 heads one, two and four 58, 62 and 65 us, of 3 heads one, four and eight 18, 11 and 9.5.
template <typename T, bool HALVES, int V, bool NT>
__global__ void __launch_bounds__(ROT_WG) k_rotate(RotateArgs A) {
    typedef std::conditional_t<sizeof(T) == 4, double, float> C; // (64-bit products of fp32 rows)
    __shared__ __align__(16) C cs[ROT_LDS / sizeof(C)]; // [rows][half] pairs
    const int half = A.rotated / 2, rest = A.hd - A.rotated, heads = A.heads + A.kvHeads;
    const int turned = (HALVES ? half : A.rotated) / V, pieces = turned + (A.copy ? rest / V : 0); // of a head
    for (int row0 = blockIdx.x * A.rowsAtOnce; row0 < A.rows; row0 += gridDim.x * A.rowsAtOnce) {
        const int rows = min(A.rowsAtOnce, A.rows - row0);
        if (row0 != (int)blockIdx.x * A.rowsAtOnce) __syncthreads();
        for (int u = threadIdx.x; u < rows * half; u += ROT_WG) {
            const int t = u % half;
            // pos freq / pi, off by 0.78 2^-52 of itself: what freq / pi loses when it is rounded goes with it, 1 / pi as a double is off by 0.28 2^-52, the last rounding is half of 2^-52
            const double pos = (double)A.pos[row0 + u / half], freq = A.freq[t], f = freq * 0.31830988618379067154, turns = fma(pos, f, pos * fma(freq, 0.31830988618379067154, -f));
            double s, c;
            sincospi(turns, &s, &c);
            cs[2 * u] = (C)(c * A.amplitude);
            cs[2 * u + 1] = (C)(s * A.amplitude);
        }
        __syncthreads();
        for (int u = threadIdx.x; u < rows * heads * pieces; u += ROT_WG) {
            const int p = u % pieces, g = u / pieces, h = g % heads, r = g / heads;
            const bool isK = h >= A.heads;
            const size_t row = row0 + r;
            const T* x = (const T*)(isK ? A.k : A.q) + row * (isK ? A.kStride : A.qStride) + (size_t)(isK ? h - A.heads : h) * A.hd;
            T* y = (T*)(isK ? A.kOut : A.qOut) + row * (isK ? A.kOutStride : A.qOutStride) + (size_t)(isK ? h - A.heads : h) * A.hd;
            float a[V], b[V];
            if (p >= turned) {
                const int i = A.rotated + (p - turned) * V;
                rot_load<V>(x + i, a);
                rot_store<NT, V>(y + i, a);
            } else if constexpr (HALVES) {
                const int i = p * V, j = half + p * V;
                const C* w = cs + 2 * ((size_t)r * half + p * V);
                rot_load<V>(x + i, a);
                rot_load<V>(x + j, b);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const C c = w[2 * e], s = w[2 * e + 1], f = a[e], g2 = b[e];
                    a[e] = (float)(c * f - s * g2);
                    b[e] = (float)(s * f + c * g2);
                }
                rot_store<NT, V>(y + i, a);
                rot_store<NT, V>(y + j, b);
            } else {
                const C* w = cs + (size_t)r * half * 2 + p * V;
                rot_load<V>(x + p * V, a);
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const C c = w[e], s = w[e + 1], f = a[e], g2 = a[e + 1];
                    a[e] = (float)(c * f - s * g2);
                    a[e + 1] = (float)(s * f + c * g2);
                }
                rot_store<NT, V>(y + p * V, a);
            }
        }
    }
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
static std::string rot_check(const mlh_rotate* a) {
    if (!a) return "null arguments";
    if (a->type != MLH_DTYPE_F32 && a->type != MLH_DTYPE_BF16 && a->type != MLH_DTYPE_F16) return "unknown row type";
    if (a->rows < 0 || a->rows > (1 << 24)) return "rows must be 0 to 2^24";
    if (a->heads < 1 || a->heads > 4096 || (a->k && (a->kvHeads < 1 || a->kvHeads > 4096))) return "rows have 1 to 4096 heads";
    if (a->headDim < 8 || a->headDim > 512 || a->headDim % 8) return "headDim must be a multiple of 8 up to 512";
    if (a->rotated < 2 || a->rotated > a->headDim || a->rotated % 2) return "rotated must be even, 2 to headDim";
    if (a->layout != MLH_ROTATE_PAIRS && a->layout != MLH_ROTATE_HALVES) return "unknown layout";
    if (a->amplitude != 0.f && !(a->amplitude >= 1e-30f && a->amplitude <= 1e30f)) return "amplitude must be 0 or 1e-30 to 1e30";
    if (!a->pos || !a->freq) return "null pointer: pos or freq";
    if ((uintptr_t)a->pos % 4 || (uintptr_t)a->freq % 8) return "pos must be 4-byte aligned, freq 8-byte aligned";
    if (!a->k != !a->kOut) return "k and kOut must both be given, or neither";
    std::string bad = kv_check_rows("q", a->q, a->qStride, (long long)a->heads * a->headDim, a->type);
    if (bad.empty()) bad = kv_check_rows("qOut", a->qOut, a->qOutStride, (long long)a->heads * a->headDim, a->type);
    if (bad.empty() && a->k) bad = kv_check_rows("k", a->k, a->kStride, (long long)a->kvHeads * a->headDim, a->type);
    if (bad.empty() && a->k) bad = kv_check_rows("kOut", a->kOut, a->kOutStride, (long long)a->kvHeads * a->headDim, a->type);
    if (bad.empty() && ((a->q == a->qOut && a->qStride != a->qOutStride) || (a->k && a->k == a->kOut && a->kStride != a->kOutStride))) bad = "rows rotated in place must keep their stride";
    return bad;
}

extern "C" int mlh_rotate_device(const mlh_rotate* a, void* stream) {
    const std::string bad = rot_check(a);
    if (!bad.empty()) return kv_fail(bad);
    if (a->rows == 0) return 0;
    const int kvHeads = a->k ? a->kvHeads : 0;
    const bool halves = a->layout == MLH_ROTATE_HALVES;
    const bool copy = a->rotated < a->headDim && (a->q != a->qOut || (a->k && a->k != a->kOut));
    const size_t bytes = (size_t)a->rows * (a->heads + kvHeads) * a->headDim * kv_elem_bytes(a->type);
    int v = 8; // elements of a piece
    while (v > 1 && (halves ? a->rotated / 2 : a->rotated) % v) v /= 2;
    const int pieces = (a->heads + kvHeads) * ((halves ? a->rotated / 2 : a->rotated) + (copy ? a->headDim - a->rotated : 0)) / v; // of a row
    const int most = ROT_LDS / (a->rotated * (a->type == MLH_DTYPE_F32 ? 8 : 4)), atOnce = std::max(1, std::min(most, ROT_WG / pieces));
    RotateArgs A = {a->q, a->k, a->qOut, a->kOut, a->qStride, a->qOutStride, a->kStride, a->kOutStride, a->pos, a->freq, a->rows, a->heads, kvHeads, a->headDim, a->rotated, atOnce, copy,
                    a->amplitude == 0.f ? 1.0 : (double)a->amplitude};
    const dim3 grid((unsigned)std::min((a->rows + atOnce - 1) / atOnce, 1 << 20));
    const bool nt = bytes > 32e6; // streaming stores for calls that write more than the L2s hold
#define ROT_GO(T_) \
    do { \
        if (v == 8) return kv_launch(halves ? (nt ? &k_rotate<T_, true, 8, true> : &k_rotate<T_, true, 8, false>) : (nt ? &k_rotate<T_, false, 8, true> : &k_rotate<T_, false, 8, false>), grid, ROT_WG, 0, stream, A); \
        if (v == 4) return kv_launch(halves ? &k_rotate<T_, true, 4, false> : &k_rotate<T_, false, 4, false>, grid, ROT_WG, 0, stream, A); \
        if (v == 2) return kv_launch(halves ? &k_rotate<T_, true, 2, false> : &k_rotate<T_, false, 2, false>, grid, ROT_WG, 0, stream, A); \
        return kv_launch(&k_rotate<T_, true, 1, false>, grid, ROT_WG, 0, stream, A); \
    } while (0)
    if (a->type == MLH_DTYPE_F32) ROT_GO(float);
    if (a->type == MLH_DTYPE_BF16) ROT_GO(bf16_t);
    ROT_GO(f16_t);
#undef ROT_GO
}
