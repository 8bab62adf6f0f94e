// Log probabilities of given tokens, entropy and most likely tokens of rows of logits (mlh_logprobs_device).
#include <math.h>

#include <algorithm>

#include "kv_cache.h"

#define LP_WG 256

struct LpArgs {
    const void* logits;
    long long stride;
    const int32_t* tokens;
    float *logProb, *entropy;
    int32_t* topIds;
    float* topLogProb;
    int rows, vocab, given, top;
    double inv; // 1 / temperature
};

__device__ __forceinline__ float lp_get(const float* p) { return *p; }
__device__ __forceinline__ float lp_get(const bf16_t* p) { return kv_bf16(*p); }
__device__ __forceinline__ float lp_get(const f16_t* p) { return kv_half(p->bits); }

// What a token is ranked by: the larger the likelier, of equal logits the lower id.  NaN counts as -infinity, and the zeros are equal.
__device__ __forceinline__ uint64_t lp_key(float x, int id) {
    if (!(x > -INFINITY)) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.f);
    return (uint64_t)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (uint32_t)~id;
}

// One workgroup a row, the row again for each of its top tokens.
template <typename T>
__global__ void __launch_bounds__(LP_WG) k_logprobs(LpArgs A) {
    __shared__ float best[LP_WG];
    __shared__ double sums[2 * LP_WG];
    __shared__ uint64_t keys[LP_WG];
    const int t = threadIdx.x;
    for (int row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const T* x = (const T*)A.logits + (size_t)row * A.stride;
        float m = -INFINITY;
        for (int i = t; i < A.vocab; i += LP_WG) m = fmaxf(m, lp_get(x + i));
        __syncthreads();
        best[t] = m;
        __syncthreads();
        for (int i = 0; i < LP_WG; i++) m = fmaxf(m, best[i]);
        double z = 0, e = 0;
        for (int i = t; i < A.vocab; i += LP_WG) {
            const double d = ((double)lp_get(x + i) - (double)m) * A.inv, p = exp(d);
            z += p;
            e += p > 0 ? p * d : 0;
        }
        sums[t] = z;
        sums[LP_WG + t] = e;
        __syncthreads();
        z = e = 0;
        for (int i = 0; i < LP_WG; i++) { z += sums[i]; e += sums[LP_WG + i]; }
        const double logz = log1p(z - 1.0);
        if (t == 0 && A.entropy) A.entropy[row] = (float)(logz - e / z);
        if (t < A.given) {
            const int id = A.tokens[(size_t)row * A.given + t];
            A.logProb[(size_t)row * A.given + t] = id < 0 ? 0.f : id >= A.vocab ? NAN : (float)(((double)lp_get(x + id) - (double)m) * A.inv - logz);
        }
        uint64_t last = ~0ull;
        for (int j = 0; j < A.top; j++) {
            uint64_t k = 0;
            for (int i = t; i < A.vocab; i += LP_WG) {
                const uint64_t y = lp_key(lp_get(x + i), i);
                if (y < last && y > k) k = y;
            }
            __syncthreads();
            keys[t] = k;
            __syncthreads();
            for (int i = 0; i < LP_WG; i++) k = keys[i] > k ? keys[i] : k;
            last = k;
            const int id = (int)~(uint32_t)k;
            if (t == 0) {
                A.topIds[(size_t)row * A.top + j] = id;
                A.topLogProb[(size_t)row * A.top + j] = (float)(((double)lp_get(x + id) - (double)m) * A.inv - logz);
            }
        }
    }
}

// ----------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------
static std::string lp_check(const mlh_logprobs* a) {
    if (!a) return "null arguments";
    if (a->type != MLH_DTYPE_F32 && a->type != MLH_DTYPE_BF16 && a->type != MLH_DTYPE_F16) return "unknown type of logits";
    if (a->rows < 0 || a->rows > (1 << 24)) return "rows must be 0 to 2^24";
    if (a->vocab < 1 || a->vocab > (1 << 22)) return "vocab must be 1 to 2^22";
    if (a->stride < a->vocab || a->stride > (1ll << 32)) return "stride smaller than vocab, or beyond 2^32";
    if (a->given < 0 || a->given > 64 || a->top < 0 || a->top > 64 || a->top > a->vocab) return "given and top must be 0 to 64, top at most vocab";
    if (!a->logits || (a->given && (!a->tokens || !a->logProb)) || (a->top && (!a->topIds || !a->topLogProb))) return "null pointer";
    if ((uintptr_t)a->logits % kv_elem_bytes(a->type)) return "logits must be aligned to their elements";
    if (((a->given ? (uintptr_t)a->tokens | (uintptr_t)a->logProb : 0) | (uintptr_t)a->entropy | (a->top ? (uintptr_t)a->topIds | (uintptr_t)a->topLogProb : 0)) % 4) return "tokens and results must be 4-byte aligned";
    if (a->temperature != 0.f && !(a->temperature >= 1e-4f && a->temperature <= 1e4f)) return "temperature must be 0 or 1e-4 to 1e4";
    return "";
}

extern "C" uint64_t mlh_logprobs_work_bytes(const mlh_logprobs* a) { return 0; }

extern "C" int mlh_logprobs_device(const mlh_logprobs* a, void* stream) {
    const std::string bad = lp_check(a);
    if (!bad.empty()) return kv_fail(bad);
    if (a->rows == 0) return 0;
    LpArgs A = {a->logits, a->stride, a->tokens, a->logProb, a->entropy, a->topIds, a->topLogProb, a->rows, a->vocab, a->given, a->top, a->temperature == 0.f ? 1.0 : 1.0 / (double)a->temperature};
    const dim3 grid((unsigned)std::min(a->rows, 1 << 20));
    if (a->type == MLH_DTYPE_F32) return kv_launch(&k_logprobs<float>, grid, LP_WG, 0, stream, A);
    if (a->type == MLH_DTYPE_BF16) return kv_launch(&k_logprobs<bf16_t>, grid, LP_WG, 0, stream, A);
    return kv_launch(&k_logprobs<f16_t>, grid, LP_WG, 0, stream, A);
}
