// k_ssm.hip — the state space mixers' operators: the short causal convolution and the selective scan
// (model.cpp:1156-1196).
#include "hip_common.h"
#include "kernels.h"

#include <algorithm>

namespace {

// e^x by the hardware's 2^x: x * log2(e) rounds once (2^-24 of it) and v_exp_f32 is off by one unit
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// log(1 + e^x); above 20 the sum rounds to e^x, so x itself (the unary op's rule)
__device__ __forceinline__ float softplus(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// ---------------------------------------------------------------------------------------------
// short causal convolution

// one thread per output, the channel fastest
__global__ __launch_bounds__(256) void ssm_conv_kernel(ssm_conv_launch L) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= L.D * L.T * L.S) return;
    const int64_t d = i % L.D, t = i / L.D % L.T, s = i / (L.D * L.T);
    const float * w = L.w + d * L.w_d;
    const float * sp = L.state + d * L.st_d + s * L.st_s;
    const float * xp = L.x + d * L.x_d + s * L.x_s;
    float v = L.bias ? L.bias[d] : 0.0f;
    for (int k = 0; k < L.K; k++) {
        const int64_t j = t + k;
        v = fmaf(w[k * L.w_k], j < L.K - 1 ? sp[j * L.st_j] : xp[(j - L.K + 1) * L.x_t], v);
    }
    if (L.silu) v = v / (1.0f + expf(-v));
    L.y[i] = v;
}

// ---------------------------------------------------------------------------------------------
// selective scan

// One row (sequence, head, channel) per group of LANES lanes, R states per lane, the tokens in order.
template <int LANES, int R>
__global__ __launch_bounds__(256) void ssm_scan_rows_kernel(ssm_scan_launch L) {
    const int64_t row = ((int64_t) blockIdx.x * 256 + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t rows = (int64_t) L.P * L.H * L.S;
    // lanes past the last row compute it again and store nothing, so that every lane takes part in the sums
    const int64_t r = row < rows ? row : rows - 1;
    const bool mine = row < rows;
    const int p = (int) (r % L.P), h = (int) (r / L.P % L.H);
    const int64_t s = r / ((int64_t) L.P * L.H);
    const int g = h / (L.H / L.G);
    int64_t id = L.ids[s * L.ids_s];
    id = id < 0 ? 0 : id >= L.pool ? L.pool - 1 : id;
    const float * s0 = L.s + p * L.s_p + h * L.s_h + id * L.s_row;
    const float * A = L.A + h * L.a_h;
    float st[R], a[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int n = lane + i * LANES;
        st[i] = n < L.N ? s0[n] : 0.0f;
        a[i] = (n < L.N ? A[L.a_scalar ? 0 : n] : 0.0f) * LOG2E;
    }
    const float * x = L.x + p + h * L.x_h + s * L.x_s;
    const float * dt = L.dt + h + s * L.dt_s;
    const float * B = L.B + g * L.b_g + s * L.b_s;
    const float * C = L.C + g * L.c_g + s * L.c_s;
    float * y = L.y + p + (int64_t) L.P * (h + (int64_t) L.H * L.T * s);
    for (int64_t t = 0; t < L.T; t++) {
        const float d = softplus(dt[t * L.dt_t]);
        const float dx = d * x[t * L.x_t];
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int n = lane + i * LANES;
            const float b = n < L.N ? B[t * L.b_t + n] : 0.0f, c = n < L.N ? C[t * L.c_t + n] : 0.0f;
            st[i] = fmaf(st[i], exp2_hw(d * a[i]), dx * b);
            v = fmaf(st[i], c, v);
        }
        v = group_sum<LANES>(v);
        if (mine && lane == 0) y[t * L.P * L.H] = v;
    }
    if (!mine) return;
    float * so = L.s_out + (int64_t) L.N * r;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int n = lane + i * LANES;
        if (n < L.N) so[n] = st[i];
    }
}

template <int LANES, int R>
void launch_rows(const ssm_scan_launch & L, hipStream_t st) {
    const int64_t rows = (int64_t) L.P * L.H * L.S, per = 256 / LANES;
    launch(ssm_scan_rows_kernel<LANES, R>, dim3((unsigned) ((rows + per - 1) / per)), dim3(256), 0, st, L);
}

} // namespace

void launch_ssm_conv(const ssm_conv_launch & L, hipStream_t st) {
    const int64_t n = L.D * L.T * L.S;
    if (n == 0) return;
    launch(ssm_conv_kernel, dim3((unsigned) ((n + 255) / 256)), dim3(256), 0, st, L);
}

void launch_ssm_scan(const ssm_scan_launch & L, hipStream_t st) {
    if ((int64_t) L.P * L.H * L.S == 0) return;
    if (L.N <= 16) launch_rows<16, 1>(L, st);
    else if (L.N <= 32) launch_rows<32, 1>(L, st);
    else if (L.N <= 64) launch_rows<64, 1>(L, st);
    else if (L.N <= 128) launch_rows<64, 2>(L, st);
    else launch_rows<64, 4>(L, st);
}
