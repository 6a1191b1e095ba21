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

// The operator reads each row and writes each output once, so it is bound by memory. Two kernels, by
// the order of the rows: channels next to each other (a projection's rows, as the executor's fused
// form has them) need no exchange between lanes; steps next to each other (the joined rows of the
// plain node) are turned round in LDS. A step of one token is latency: one round of loads.

__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + exp2_hw(-v * LOG2E)); }

template <int V> struct chunk { float v[V]; };
template <int V> __device__ __forceinline__ chunk<V> ldv(const float * p) {
    chunk<V> c;
    if constexpr (V == 4) {
        const float4 f = *(const float4 *) p;
        c.v[0] = f.x; c.v[1] = f.y; c.v[2] = f.z; c.v[3] = f.w;
    } else {
        c.v[0] = *p;
    }
    return c;
}
template <int V> __device__ __forceinline__ void stv(float * p, const chunk<V> & c) {
    if constexpr (V == 4) *(float4 *) p = make_float4(c.v[0], c.v[1], c.v[2], c.v[3]);
    else *p = c.v[0];
}

// Channels contiguous (x_d == 1), K taps, V channels and TT tokens per thread, all rows of a tile in
// flight at once. The first tile's threads, the only ones that touch the state, write the new one:
// it may be the old one's own memory.
// PACK: filters and states contiguous and 16-byte aligned, so that a thread's four of each are whole
// float4s (K or K - 1 of them) instead of a dword per value.
template <int K, int V, int TT, bool PACK>
__global__ __launch_bounds__(256) void ssm_conv_rows_kernel(ssm_conv_launch L, int blocks) {
    const int cb = (int) (blockIdx.x % (unsigned) blocks);
    const int64_t t0 = (int64_t) (blockIdx.x / (unsigned) blocks) * TT;
    const int64_t d = ((int64_t) cb * blockDim.x + threadIdx.x) * V;
    if (d >= L.D) return;
    float w[V][K];
    if constexpr (PACK) {
#pragma unroll
        for (int q = 0; q < K; q++) {
            const chunk<4> c = ldv<4>(L.w + d * K + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; i++) w[(4 * q + i) / K][(4 * q + i) % K] = c.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
#pragma unroll
            for (int k = 0; k < K; k++) w[i][k] = L.w[(d + i) * L.w_d + k * L.w_k];
        }
    }
    chunk<V> b{};
    if (L.bias) b = ldv<V>(L.bias + d);
    for (int64_t s = blockIdx.y; s < L.S; s += gridDim.y) {
        const float * xp = L.x + d + s * L.x_s;
        const float * sp = L.state + d * L.st_d + s * L.st_s;
        chunk<V> r[TT + K - 1];
#pragma unroll
        for (int j = 0; j < TT + K - 1; j++) {
            const int64_t t = t0 + j - (K - 1);   // a row past the last is the last again, and not used
            r[j] = ldv<V>(xp + (t < 0 ? 0 : t < L.T ? t : L.T - 1) * L.x_t);
        }
        if (K > 1 && t0 == 0) {
            float old[V][K > 1 ? K - 1 : 1];      // rows 0 .. K - 2
            if constexpr (PACK) {
#pragma unroll
                for (int q = 0; q < K - 1; q++) {
                    const chunk<4> c = ldv<4>(sp + 4 * q);
#pragma unroll
                    for (int i = 0; i < 4; i++) old[(4 * q + i) / (K - 1)][(4 * q + i) % (K - 1)] = c.v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) {
#pragma unroll
                    for (int j = 0; j < K - 1; j++) old[i][j] = sp[i * L.st_d + j * L.st_j];
                }
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
#pragma unroll
                for (int j = 0; j < K - 1; j++) r[j].v[i] = old[i][j];
            }
            if (L.new_state) {
                float last[V][K > 1 ? K - 1 : 1];
#pragma unroll
                for (int j = 0; j < K - 1; j++) {
                    const int64_t t = L.T + j - (K - 1);
                    const chunk<V> c = ldv<V>(xp + (t < 0 ? 0 : t) * L.x_t);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        last[i][j] = c.v[i];
#pragma unroll
                        for (int o = 0; o < K - 1; o++) last[i][j] = L.T + j == o ? old[i][o] : last[i][j];
                    }
                }
                float * np = L.new_state + (s * L.D + d) * (K - 1);
                if constexpr (PACK) {
#pragma unroll
                    for (int q = 0; q < K - 1; q++) {
                        chunk<4> c;
#pragma unroll
                        for (int i = 0; i < 4; i++) c.v[i] = last[(4 * q + i) / (K - 1)][(4 * q + i) % (K - 1)];
                        stv<4>(np + 4 * q, c);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) {
#pragma unroll
                        for (int j = 0; j < K - 1; j++) np[i * (K - 1) + j] = last[i][j];
                    }
                }
            }
        }
        float * y = L.y + d + L.D * (t0 + L.T * s);
#pragma unroll
        for (int j = 0; j < TT; j++) {
            if (t0 + j >= L.T) break;
            chunk<V> o;
#pragma unroll
            for (int i = 0; i < V; i++) {
                float v = b.v[i];
#pragma unroll
                for (int k = 0; k < K; k++) v = fmaf(w[i][k], r[j + k].v[i], v);
                o.v[i] = L.silu ? silu(v) : v;
            }
            stv<V>(y + j * L.D, o);
        }
    }
}

// Rows in any order: 64 channels by 64 tokens and the K - 1 rows before them through LDS, read with
// the steps across the lanes and used with the channels across them. An odd row length keeps the
// lanes' reads on different banks.
__global__ __launch_bounds__(256) void ssm_conv_tile_kernel(ssm_conv_launch L, int blocks) {
    extern __shared__ float rows[];
    const int width = 64 + L.K - 1, stride = width | 1, tid = threadIdx.x;
    const int64_t d0 = (int64_t) (blockIdx.x % (unsigned) blocks) * 64, t0 = (int64_t) (blockIdx.x / (unsigned) blocks) * 64;
    const int nd = (int) min((int64_t) 64, L.D - d0), nt = (int) min((int64_t) 64, L.T - t0);
    for (int64_t s = blockIdx.y; s < L.S; s += gridDim.y) {
        __syncthreads();
        for (int i = tid; i < nd * width; i += 256) {
            const int d = i / width, j = i - d * width;
            const int64_t r = t0 + j;
            if (j >= nt + L.K - 1) continue;
            rows[d * stride + j] = r < L.K - 1 ? L.state[(d0 + d) * L.st_d + r * L.st_j + s * L.st_s]
                                               : L.x[(d0 + d) * L.x_d + (r - L.K + 1) * L.x_t + s * L.x_s];
        }
        if (L.new_state && t0 == 0) {
            // read before the barrier, written after it, by the one tile that reads the state at all
            for (int i = tid; i < nd * (L.K - 1); i += 256) {
                const int d = i / (L.K - 1), j = i - d * (L.K - 1);
                const int64_t r = L.T + j;
                rows[64 * stride + i] = r < L.K - 1 ? L.state[(d0 + d) * L.st_d + r * L.st_j + s * L.st_s]
                                                    : L.x[(d0 + d) * L.x_d + (r - L.K + 1) * L.x_t + s * L.x_s];
            }
        }
        __syncthreads();
        if (L.new_state && t0 == 0) {
            for (int i = tid; i < nd * (L.K - 1); i += 256) L.new_state[(s * L.D + d0) * (L.K - 1) + i] = rows[64 * stride + i];
        }
        const int d = tid % 64, tw = tid / 64 * 16;
        if (d < nd) {
            const float bias = L.bias ? L.bias[d0 + d] : 0.0f;
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; j++) v[j] = bias;
            for (int k = 0; k < L.K; k++) {
                const float w = L.w[(d0 + d) * L.w_d + k * L.w_k];
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = fmaf(w, rows[d * stride + tw + j + k], v[j]);
            }
            float * y = L.y + d0 + d + L.D * (t0 + L.T * s);
#pragma unroll
            for (int j = 0; j < 16; j++) {
                if (tw + j < nt) y[(tw + j) * L.D] = L.silu ? silu(v[j]) : v[j];
            }
        }
    }
}

template <int K, int V, bool PACK>
void launch_conv_rows(const ssm_conv_launch & L, hipStream_t st) {
    const int64_t groups = (L.D + V - 1) / V;
    const int threads = (int) std::min<int64_t>(256, (groups + 63) / 64 * 64);
    const int blocks = (int) ((groups + threads - 1) / threads);
    const unsigned gy = (unsigned) std::min<int64_t>(L.S, 65535);
    // eight rows per thread read 11 for 8 outputs (4 taps); one token takes its own rows only
    if (L.T == 1) launch(ssm_conv_rows_kernel<K, V, 1, PACK>, dim3((unsigned) blocks, gy), dim3(threads), 0, st, L, blocks);
    else launch(ssm_conv_rows_kernel<K, V, 8, PACK>, dim3((unsigned) (blocks * ((L.T + 7) / 8)), gy), dim3(threads), 0, st, L, blocks);
}

template <int K>
void launch_conv_rows(const ssm_conv_launch & L, hipStream_t st) {
    const bool wide = L.D % 4 == 0 && L.x_t % 4 == 0 && L.x_s % 4 == 0 && ((uintptr_t) L.x | (uintptr_t) L.y | (uintptr_t) L.bias) % 16 == 0;
    const bool pack = wide && L.w_k == 1 && L.w_d == K && (K == 1 || (L.st_j == 1 && L.st_d == K - 1 && L.st_s % 4 == 0)) &&
                      ((uintptr_t) L.w | (K == 1 ? 0 : (uintptr_t) L.state | (uintptr_t) L.new_state)) % 16 == 0;
    if (pack) launch_conv_rows<K, 4, true>(L, st);
    else if (wide) launch_conv_rows<K, 4, false>(L, st);
    else launch_conv_rows<K, 1, false>(L, st);
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
    if (L.D == 0 || L.S == 0) return;
    if (L.T == 0) return;
    if (L.x_d == 1 && L.K <= 4) {
        switch (L.K) {
            case 1: launch_conv_rows<1>(L, st); return;
            case 2: launch_conv_rows<2>(L, st); return;
            case 3: launch_conv_rows<3>(L, st); return;
            default: launch_conv_rows<4>(L, st); return;
        }
    }
    const int blocks = (int) ((L.D + 63) / 64);
    const size_t lds = sizeof(float) * (64 * ((64 + L.K - 1) | 1) + 64 * (L.K - 1));
    launch(ssm_conv_tile_kernel, dim3((unsigned) (blocks * ((L.T + 63) / 64)), (unsigned) std::min<int64_t>(L.S, 65535)), dim3(256), lds, st,
           L, blocks);
}

void launch_ssm_scan(const ssm_scan_launch & L, hipStream_t st) {
    if ((int64_t) L.P * L.H * L.S == 0) return;
    if (L.N <= 16) launch_rows<16, 1>(L, st);
    else if (L.N <= 32) launch_rows<32, 1>(L, st);
    else if (L.N <= 64) launch_rows<64, 1>(L, st);
    else if (L.N <= 128) launch_rows<64, 2>(L, st);
    else launch_rows<64, 4>(L, st);
}
