// k_logprobs.hip — log probabilities of given tokens under rows of logits, the rows' entropies and
// their likeliest tokens.
//
// With m the largest logit of a row, e_i = exp(l_i - m), S = sum e_i and W = sum e_i (l_i - m):
//   log p_i = l_i - m - log S,   H = -sum p_i log p_i = log S - W / S.
// An entry of -inf weighs nothing (0 log 0 = 0). A row whose largest logit is not finite has no
// distribution: its scores are NaN. NaN entries order as -inf, as in the sampler; a row that holds
// one has no distribution either.
#include "hip_common.h"
#include "kernels.h"

namespace {

constexpr int LP_THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f;

// ascending order key of a float; -0 and +0 share a key, NaN takes the key of -inf
__device__ __forceinline__ uint32_t okey(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float okey_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// descending order is descending value, then ascending id
__device__ __forceinline__ uint64_t ckey(float v, int id) { return ((uint64_t) okey(v) << 32) | (uint32_t) ~id; }

template <class T, class F>
__device__ T block_reduce(T v, T * s, F f) {
    const int t = threadIdx.x;
    s[t] = v;
    __syncthreads();
    for (int n = LP_THREADS / 2; n > 0; n /= 2) {
        if (t < n) s[t] = f(s[t], s[t + n]);
        __syncthreads();
    }
    v = s[0];
    __syncthreads();
    return v;
}

__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(logprobs_launch L) {
    __shared__ uint64_t sk[LP_THREADS];
    __shared__ float sf[LP_THREADS];
    const int r = blockIdx.x, t = threadIdx.x;
    const int64_t row = L.row0 + r, i1 = row % L.ne1, i2 = row / L.ne1 % L.ne2, i3 = row / (L.ne1 * L.ne2);
    const float * x = (const float *) (L.base + i1 * L.nb1 + i2 * L.nb2 + i3 * L.nb3);
    float * out = L.out + (int64_t) r * (2 + 2 * L.k);
    float m = -INFINITY, bad = 0.0f;
    for (int i = t; i < L.n; i += LP_THREADS) {
        m = fmaxf(m, x[i]);
        if (x[i] != x[i]) bad = 1.0f;
    }
    m = block_reduce(m, sf, [](float a, float b) { return fmaxf(a, b); });
    bad = block_reduce(bad, sf, [](float a, float b) { return fmaxf(a, b); });
    float sum = 0.0f, wsum = 0.0f;
    for (int i = t; i < L.n; i += LP_THREADS) {
        const float z = x[i] - m, e = exp2f(z * LOG2E);
        sum += e;
        if (e > 0.0f) wsum = fmaf(e, z, wsum);
    }
    sum = block_reduce(sum, sf, [](float a, float b) { return a + b; });
    wsum = block_reduce(wsum, sf, [](float a, float b) { return a + b; });
    const bool none = bad != 0.0f || !(fabsf(m) < INFINITY);
    const float ls = none ? NAN : logf(sum);
    if (t == 0) {
        out[0] = L.tokens ? x[L.tokens[r]] - m - ls : 0.0f;
        out[1] = ls - wsum / sum;
    }
    uint64_t last = ~(uint64_t) 0;
    for (int j = 0; j < L.k; j++) {
        uint64_t best = 0;
        for (int i = t; i < L.n; i += LP_THREADS) {
            const uint64_t k = ckey(x[i], i);
            if (k < last && k > best) best = k;
        }
        best = block_reduce(best, sk, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        last = best;
        if (t == 0) {
            ((int32_t *) out)[2 + j] = (int32_t) ~(uint32_t) best;
            out[2 + L.k + j] = okey_value((uint32_t) (best >> 32)) - m - ls;
        }
    }
}

} // namespace

void launch_logprobs(const logprobs_launch & L, hipStream_t st) {
    launch(logprobs_kernel, dim3((unsigned) L.n_rows), dim3(LP_THREADS), 0, st, L);
}
