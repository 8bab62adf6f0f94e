// Rotary positions of a caller's rows (mlh_rotate_device).
#include <math.h>

#include <algorithm>

#include "kv_cache.h"

#define ROT_WG 256

struct RotateArgs {
    const void *q, *k;
    void *qOut, *kOut;
    long long qStride, qOutStride, kStride, kOutStride;
    const int32_t* pos;
    const double* freq;
    int rows, heads, kvHeads, hd, rotated;
    double amplitude;
};

__device__ __forceinline__ double rot_get(const float* p) { return *p; }
__device__ __forceinline__ double rot_get(const bf16_t* p) { return kv_bf16(*p); }
__device__ __forceinline__ double rot_get(const f16_t* p) { return kv_half(p->bits); }
__device__ __forceinline__ void rot_put(float* p, double v) { *p = (float)v; }
__device__ __forceinline__ void rot_put(bf16_t* p, double v) { *p = (bf16_t)kv_to_bf16((float)v); }
__device__ __forceinline__ void rot_put(f16_t* p, double v) { p->bits = (uint16_t)kv_to_half((float)v); }

// One workgroup a row: cosines and sines of its pairs once, into LDS, then its heads.  The angle is counted in half turns, whose whole ones are taken off in 64 bits.
template <typename T, bool HALVES>
__global__ void __launch_bounds__(ROT_WG) k_rotate(RotateArgs A) {
    __shared__ double cs[2 * 256];
    const int half = A.rotated / 2, rest = A.hd - A.rotated;
    for (int row = blockIdx.x; row < A.rows; row += gridDim.x) {
        __syncthreads();
        for (int t = threadIdx.x; t < half; t += ROT_WG) {
            const double turns = (double)A.pos[row] * (A.freq[t] * 0.31830988618379067154);
            double s, c;
            sincospi(turns - 2.0 * rint(turns * 0.5), &s, &c);
            cs[2 * t] = c * A.amplitude;
            cs[2 * t + 1] = s * A.amplitude;
        }
        __syncthreads();
        for (int u = threadIdx.x; u < (A.heads + A.kvHeads) * (half + rest); u += ROT_WG) {
            const int g = u / (half + rest), t = u % (half + rest);
            const bool isK = g >= A.heads;
            const int h = isK ? g - A.heads : g;
            const T* x = (const T*)(isK ? A.k : A.q) + (size_t)row * (isK ? A.kStride : A.qStride) + (size_t)h * A.hd;
            T* y = (T*)(isK ? A.kOut : A.qOut) + (size_t)row * (isK ? A.kOutStride : A.qOutStride) + (size_t)h * A.hd;
            if (t >= half) {
                y[A.rotated + t - half] = x[A.rotated + t - half];
                continue;
            }
            const int i = HALVES ? t : 2 * t, j = HALVES ? t + half : 2 * t + 1;
            const double a = rot_get(x + i), b = rot_get(x + j), c = cs[2 * t], s = cs[2 * t + 1];
            rot_put(y + i, c * a - s * b);
            rot_put(y + j, s * a + c * b);
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
    RotateArgs A = {a->q, a->k, a->qOut, a->kOut, a->qStride, a->qOutStride, a->kStride, a->kOutStride, a->pos, a->freq, a->rows, a->heads, a->k ? a->kvHeads : 0, a->headDim, a->rotated,
                    a->amplitude == 0.f ? 1.0 : (double)a->amplitude};
    const dim3 grid((unsigned)std::min(a->rows, 1 << 20));
    const bool halves = a->layout == MLH_ROTATE_HALVES;
#define ROT_GO(T_) return kv_launch(halves ? &k_rotate<T_, true> : &k_rotate<T_, false>, grid, ROT_WG, 0, stream, A)
    if (a->type == MLH_DTYPE_F32) ROT_GO(float);
    if (a->type == MLH_DTYPE_BF16) ROT_GO(bf16_t);
    ROT_GO(f16_t);
#undef ROT_GO
}
