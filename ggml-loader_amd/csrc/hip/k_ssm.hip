// k_ssm.hip — the state space mixers' operators: the short causal convolution and the selective scan
// (model.cpp:1156-1196).
#include "hip_common.h"
#include "kernels.h"
#include "ssm_ops.h"

#include <algorithm>

namespace {

// ---------------------------------------------------------------------------------------------
// short causal convolution

// The operator reads each row and writes each output once, so it is bound by memory. Two kernels, by
// the order of the rows: channels next to each other (a projection's rows, as the executor's fused
// form has them) need no exchange between lanes; steps next to each other (the joined rows of the
// plain node) are turned round in LDS. A step of one token is latency: one round of loads. 4096 tokens of 10240
// channels and 4 taps, which are read and written once: 66.3 us by rows (5.06 TB/s; 63 on the same rows again), 146
// by tiles, which divide by the rows' width for each value and load four bytes at a time.

__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + exp2_hw(-v * LOG2E)); }

template <int V> struct chunk { float v[V]; };
template <int V> __device__ __forceinline__ chunk<V> ldv(const float * p) {
    chunk<V> c;
    if constexpr (V == 4) {
        const float4 f = load4(p);
        c.v[0] = f.x; c.v[1] = f.y; c.v[2] = f.z; c.v[3] = f.w;
    } else {
        c.v[0] = *p;
    }
    return c;
}
template <int V> __device__ __forceinline__ void stv(float * p, const chunk<V> & c) {
    if constexpr (V == 4) store4(p, make_float4(c.v[0], c.v[1], c.v[2], c.v[3]));
    else *p = c.v[0];
}

// Channels contiguous (x_d == 1), K taps, V channels and TT tokens per thread, all rows of a tile in
// flight at once. The first tile's threads, the only ones that touch the state, write the new one:
// it may be the old one's own memory.
// PACK: filters and a sequence's states contiguous, so that a thread's four of each are K or K - 1 float4s. Four
// channels a thread only where they are: 64 tokens of 5120 channels take 5.2 us so, 5.5 with a channel each,
// and 8.9 with four of which each loads its filter and state by dwords; 4096 tokens of 10240 62.9, 73.4
// and 76.1, each on the same rows again.
template <int K, int V, int TT, bool PACK>
__device__ __forceinline__ void conv_rows(const ssm_conv_launch & L, int64_t t0, int64_t d) {
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

// V channels a thread; the ones that are left over have a thread each, in a wave of their own: in the last
// wave of the others they would wait for those (777 tokens of 2558 channels 7.9 us, and 7.0 with a thread a channel)
template <int K, int V, int TT, bool PACK>
__global__ __launch_bounds__(256) void ssm_conv_rows_kernel(ssm_conv_launch L, int blocks) {
    const int64_t t0 = (int64_t) (blockIdx.x / (unsigned) blocks) * TT;
    const int64_t i = (int64_t) (blockIdx.x % (unsigned) blocks) * blockDim.x + threadIdx.x, whole = L.D / V, rest = (whole + 63) / 64 * 64;
    if (i < whole) conv_rows<K, V, TT, PACK>(L, t0, i * V);
    else if (V > 1 && i >= rest && i < rest + L.D % V) conv_rows<K, 1, TT, false>(L, t0, i - rest + whole * V);
}

// Rows in any order: 64 channels by 64 tokens and the K - 1 rows before them through LDS, read with
// the steps across the lanes and used with the channels across them. An odd row length keeps the
// lanes' reads on different banks.
__global__ __launch_bounds__(256) void ssm_conv_tile_kernel(ssm_conv_launch L, int blocks) {
    extern __shared__ float rows[];
    const int width = 64 + L.K - 1, stride = width | 1, tid = threadIdx.x;
    const unsigned tile = blockIdx.z * gridDim.x + blockIdx.x;
    const int64_t d0 = (int64_t) (tile % (unsigned) blocks) * 64, t0 = (int64_t) (tile / (unsigned) blocks) * 64;
    if (t0 >= L.T) return;                                     // past the last tile
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
    const int64_t groups = L.D % V ? (L.D / V + 63) / 64 * 64 + L.D % V : L.D / V;
    const int threads = (int) std::min<int64_t>(256, (groups + 63) / 64 * 64);
    const int blocks = (int) ((groups + threads - 1) / threads);
    const unsigned gy = (unsigned) std::min<int64_t>(L.S, 65535);
    // eight rows per thread read 11 for 8 outputs (4 taps); one token takes its own rows only
    if (L.T == 1) launch(ssm_conv_rows_kernel<K, V, 1, PACK>, dim3((unsigned) blocks, gy), dim3(threads), 0, st, L, blocks);
    else launch(ssm_conv_rows_kernel<K, V, 8, PACK>, dim3((unsigned) (blocks * ((L.T + 7) / 8)), gy), dim3(threads), 0, st, L, blocks);
}

template <int K>
void launch_conv_rows(const ssm_conv_launch & L, hipStream_t st) {
    const bool pack = L.w_k == 1 && L.w_d == K && (K == 1 || (L.st_j == 1 && L.st_d == K - 1));
    if (pack) launch_conv_rows<K, 4, true>(L, st);
    else launch_conv_rows<K, 1, false>(L, st);
}

// ---------------------------------------------------------------------------------------------
// selective scan

__device__ __forceinline__ int64_t pool_row(const ssm_scan_launch & L, int64_t s) {
    const int64_t id = L.ids[s * L.ids_s];
    return id < 0 ? 0 : id >= L.pool ? L.pool - 1 : id;
}

// Any operands: one row (sequence, head, channel) per group of LANES lanes, R states per lane, the tokens
// in order.
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
    const float * s0 = L.s + p * L.s_p + h * L.s_h + pool_row(L, s) * L.s_row;
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

// A few tokens (decoding): the states are most of what is read and written, so a lane takes them 16 bytes
// at a time and STEP_ROWS channels at once. LANES lanes hold a channel's 4 LANES states; the group's channels
// share B and C, and (ONE_HEAD) the time step and the decay. 32 sequences of 80 heads of 64 channels and 128
// states: 35 us a token, 4.8 TB/s of states; on the same states again 26.6, and 75 by the kernel for any operands.
constexpr int STEP_ROWS = 4;

template <int LANES, bool ONE_HEAD>
__global__ __launch_bounds__(256) void ssm_scan_step_kernel(ssm_scan_launch L, int64_t groups) {
    const int64_t group = ((int64_t) blockIdx.x * 256 + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES, n = 4 * lane;
    if (group >= groups) return;                               // whole groups only
    const int64_t per = (int64_t) L.P * L.H, in_seq = (per + STEP_ROWS - 1) / STEP_ROWS, s = group / in_seq;
    const int q0 = (int) (group - s * in_seq) * STEP_ROWS;
    const bool on = n < L.N;
    // past a sequence's last channel that one again: its values are stored twice
    int q[STEP_ROWS], p[STEP_ROWS], h[STEP_ROWS];
#pragma unroll
    for (int k = 0; k < STEP_ROWS; k++) {
        q[k] = ONE_HEAD ? q0 + k : min(q0 + k, (int) per - 1);
        h[k] = ONE_HEAD ? q0 / L.P : q[k] / L.P;
        p[k] = q[k] - h[k] * L.P;
    }
    const int g = h[0] / (L.H / L.G);
    const int64_t id = pool_row(L, s);
    const float4 zero = make_float4(0, 0, 0, 0);
    float4 st[STEP_ROWS], a[ONE_HEAD ? 1 : STEP_ROWS];
#pragma unroll
    for (int k = 0; k < STEP_ROWS; k++) st[k] = on ? load4(L.s + p[k] * L.s_p + h[k] * L.s_h + id * L.s_row + n) : zero;
#pragma unroll
    for (int k = 0; k < (ONE_HEAD ? 1 : STEP_ROWS); k++) {
        const float * A = L.A + h[k] * L.a_h;
        if (L.a_scalar) a[k] = make_float4(A[0], A[0], A[0], A[0]);
        else a[k] = on ? load4(A + n) : zero;
        a[k] = make_float4(a[k].x * LOG2E, a[k].y * LOG2E, a[k].z * LOG2E, a[k].w * LOG2E);
    }
    const float * B = L.B + g * L.b_g + s * L.b_s + n, * C = L.C + g * L.c_g + s * L.c_s + n;
    float * y = L.y + per * L.T * s;
    for (int64_t t = 0; t < L.T; t++) {
        float d[ONE_HEAD ? 1 : STEP_ROWS], x[STEP_ROWS], v[STEP_ROWS];
#pragma unroll
        for (int k = 0; k < (ONE_HEAD ? 1 : STEP_ROWS); k++) d[k] = L.dt[h[k] + t * L.dt_t + s * L.dt_s];
#pragma unroll
        for (int k = 0; k < STEP_ROWS; k++) x[k] = L.x[p[k] + h[k] * L.x_h + t * L.x_t + s * L.x_s];
        const float4 b = on ? load4(B + t * L.b_t) : zero, c = on ? load4(C + t * L.c_t) : zero;
        float4 e = zero;
#pragma unroll
        for (int k = 0; k < STEP_ROWS; k++) {
            if (!ONE_HEAD || k == 0) {
                float & dk = d[ONE_HEAD ? 0 : k];
                const float4 ak = a[ONE_HEAD ? 0 : k];
                dk = softplus(dk);
                e.x = exp2_hw(dk * ak.x);
                if (ONE_HEAD && L.a_scalar) e.y = e.z = e.w = e.x;
                else { e.y = exp2_hw(dk * ak.y); e.z = exp2_hw(dk * ak.z); e.w = exp2_hw(dk * ak.w); }
            }
            const float dx = d[ONE_HEAD ? 0 : k] * x[k];
            st[k].x = fmaf(st[k].x, e.x, dx * b.x);
            st[k].y = fmaf(st[k].y, e.y, dx * b.y);
            st[k].z = fmaf(st[k].z, e.z, dx * b.z);
            st[k].w = fmaf(st[k].w, e.w, dx * b.w);
            v[k] = group_sum<LANES>(fmaf(st[k].x, c.x, st[k].y * c.y) + fmaf(st[k].z, c.z, st[k].w * c.w));
        }
#pragma unroll
        for (int k = 0; k < STEP_ROWS; k++) {
            if (lane == k % LANES) y[t * per + q[k]] = v[k];
        }
    }
    if (!on) return;
#pragma unroll
    for (int k = 0; k < STEP_ROWS; k++) store4(L.s_out + (int64_t) L.N * (q[k] + per * s) + n, st[k]);
}

bool step_takes(const ssm_scan_launch & L) {
    return L.N % 4 == 0 && (L.G == 1 || ((int64_t) L.H / L.G * L.P) % STEP_ROWS == 0);
}

template <int LANES>
void launch_step(const ssm_scan_launch & L, hipStream_t st) {
    const int64_t groups = ((int64_t) L.P * L.H + STEP_ROWS - 1) / STEP_ROWS * L.S, per = 256 / LANES;
    const dim3 grid((unsigned) ((groups + per - 1) / per));
    if (L.P % STEP_ROWS == 0) launch(ssm_scan_step_kernel<LANES, true>, grid, dim3(256), 0, st, L, groups);
    else launch(ssm_scan_step_kernel<LANES, false>, grid, dim3(256), 0, st, L, groups);
}

// Heads of one channel: a lane per channel with all of its N states in registers, so that no sum crosses lanes
// and B and C, the same for the wave's 64 channels, are scalar operands. Every state takes an exponential and
// four more operations per token, which bounds it over many tokens; the states' bytes do over few, and they go
// through LDS so that lanes next to each other read 16 bytes next to each other (without it 81 sequences of 5120
// channels and 16 states took 32 us a token, with it 12.1, 4.8 TB/s; the kernel for few tokens took 15.7).
// Where channels alone are too few waves the tokens are split into segments: `local` finds each segment's final
// state from nothing and its sum of time steps, `join` the state that each begins with, and the last launch the
// outputs (74.7 us at 1500 tokens of 5120 channels: 29, 10 and 37). The first pass repeats 7/8 of the work;
// carrying its outputs over would take as many exponentials again.
struct chan_plan {
    ssm_scan_launch L;
    float * part;          // [S, n_seg, H, N]: segments' states, then what each begins with
    float * sums;          // [S, n_seg, H]
    int     seg, n_seg;    // tokens per segment, segments
};

typedef const __attribute__((address_space(4))) float * scalar_ptr;

template <int N, bool OUT>
__global__ __launch_bounds__(64) void ssm_scan_channels_kernel(chan_plan P) {
    const ssm_scan_launch & L = P.L;
    // decays and states lie by channels in memory: LANES lanes read a channel's, and LDS turns them
    constexpr int LANES = N / 4, PITCH = N + 4;
    __shared__ __align__(16) float turn[64 * PITCH];
    const int h0 = blockIdx.x * 64, h = h0 + threadIdx.x, hc = min(h, L.H - 1), sg = blockIdx.y;
    const int c0 = threadIdx.x / LANES, n4 = threadIdx.x % LANES * 4;
    const int64_t s = blockIdx.z;
    const int g = h0 / (L.H / L.G);
    const int64_t t0 = (int64_t) sg * P.seg, t1 = min(L.T, t0 + P.seg);
    float a[N], st[N];
    float4 part[LANES];
    auto rows = [&](const float * p, int64_t step) {
#pragma unroll
        for (int i = 0; i < LANES; i++) part[i] = load4(p + min(h0 + c0 + i * (64 / LANES), L.H - 1) * step + n4);
    };
    auto turned = [&](float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < LANES; i++) *(float4 *) (turn + (c0 + i * (64 / LANES)) * PITCH + n4) = part[i];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; n += 4) {
            const float4 f = *(const float4 *) (turn + threadIdx.x * PITCH + n);
            v[n] = f.x; v[n + 1] = f.y; v[n + 2] = f.z; v[n + 3] = f.w;
        }
        __syncthreads();
    };
    if (L.a_scalar) {
        const float a0 = L.A[hc * L.a_h];
#pragma unroll
        for (int n = 0; n < N; n++) a[n] = a0;
    } else {
        rows(L.A, L.a_h);
        turned(a);
    }
#pragma unroll
    for (int n = 0; n < N; n++) a[n] *= LOG2E;
    if (!OUT) {
#pragma unroll
        for (int n = 0; n < N; n++) st[n] = 0.0f;
    } else if (P.n_seg == 1) {
        rows(L.s + pool_row(L, s) * L.s_row, L.s_h);
        turned(st);
    } else {
        rows(P.part + (s * P.n_seg + sg) * N * L.H, N);
        turned(st);
    }
    const float * x = L.x + hc * L.x_h + s * L.x_s + t0 * L.x_t, * dt = L.dt + hc + s * L.dt_s + t0 * L.dt_t;
    scalar_ptr B = (scalar_ptr) (uintptr_t) (L.B + g * L.b_g + s * L.b_s + t0 * L.b_t);
    scalar_ptr C = (scalar_ptr) (uintptr_t) (L.C + g * L.c_g + s * L.c_s + t0 * L.c_t);
    float * y = L.y + hc + (int64_t) L.H * (t0 + L.T * s);
    // the segment's time steps, added with what each sum rounds away: a decay over many tokens rounds as one over few
    float sum = 0.0f, lost = 0.0f, plain = 0.0f;
    auto token = [&](float raw, float xt) {
        const float d = softplus(raw), dx = d * xt;
        float v = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++) {
            st[n] = fmaf(dx, B[n], st[n] * exp2_hw(d * a[n]));
            if (OUT) v = fmaf(st[n], C[n], v);
        }
        if (!OUT) {
            const float part = d - lost, next = sum + part;
            lost = (next - sum) - part;
            sum = next;
            plain += d;
        }
        if (OUT) {
            *y = v;                                            // lanes past the last channel store its value again
            y += L.H;
            C += L.c_t;
        }
        B += L.b_t;
    };
    // four tokens at a time, the next four's inputs on their way (past the segment, its last token's)
    float xn[4], dn[4];
    auto fetch = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t k = min(t + i, t1 - 1) - t0;
            xn[i] = x[k * L.x_t];
            dn[i] = dt[k * L.dt_t];
        }
    };
    fetch(t0);
    int64_t t = t0;
    for (; t + 4 <= t1; t += 4) {
        float xt[4], raw[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            xt[i] = xn[i];
            raw[i] = dn[i];
        }
        fetch(t + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) token(raw[i], xt[i]);
    }
    for (int i = 0; t + i < t1; i++) token(i == 0 ? dn[0] : i == 1 ? dn[1] : dn[2], i == 0 ? xn[0] : i == 1 ? xn[1] : xn[2]);
    if (OUT && sg != P.n_seg - 1) return;
    float * q = OUT ? L.s_out + (int64_t) N * L.H * s : P.part + (s * P.n_seg + sg) * N * L.H;
#pragma unroll
    for (int n = 0; n < N; n += 4) *(float4 *) (turn + threadIdx.x * PITCH + n) = make_float4(st[n], st[n + 1], st[n + 2], st[n + 3]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LANES; i++) {
        const int c = c0 + i * (64 / LANES);
        if (h0 + c < L.H) store4(q + (int64_t) N * (h0 + c) + n4, *(const float4 *) (turn + c * PITCH + n4));
    }
    if (!OUT && h < L.H) P.sums[(s * P.n_seg + sg) * L.H + h] = plain < INFINITY ? sum : plain;   // past float's range nothing is lost but all
}

// a thread per channel and state: the segments in order
__global__ __launch_bounds__(256) void ssm_scan_join_kernel(chan_plan P) {
    const ssm_scan_launch & L = P.L;
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x, step = (int64_t) L.N * L.H, s = blockIdx.y;
    if (i >= step) return;
    const int h = (int) (i / L.N), n = (int) (i - (int64_t) h * L.N);
    const float a = L.A[h * L.a_h + (L.a_scalar ? 0 : n)] * LOG2E;
    float st = L.s[n + h * L.s_h + pool_row(L, s) * L.s_row];
    float * q = P.part + s * P.n_seg * step + i;
    const float * sum = P.sums + s * P.n_seg * L.H + h;
    // sixteen segments' loads in flight
    for (int k0 = 0; k0 < P.n_seg; k0 += 16) {
        float own[16], d[16];
#pragma unroll
        for (int k = 0; k < 16; k++) {
            if (k0 + k < P.n_seg - 1) {
                own[k] = q[(k0 + k) * step];
                d[k] = sum[(int64_t) (k0 + k) * L.H];
            }
        }
#pragma unroll
        for (int k = 0; k < 16; k++) {
            if (k0 + k >= P.n_seg) break;
            q[(k0 + k) * step] = st;
            st = fmaf(st, exp2_hw(d[k] * a), own[k]);
        }
    }
}

bool channels_take(const ssm_scan_launch & L) {
    return L.P == 1 && (L.N == 8 || L.N == 16 || L.N == 32) && L.T >= 1 && (L.G == 1 || L.H / L.G % 64 == 0) && L.S <= 65535;
}

// One segment, or enough for four waves of every SIMD, of 8 tokens at least. With w waves of channels a token
// takes 0.4 us in one piece (up to a wave per SIMD); split, about w / 820 of that, the first pass's work included,
// and 12 us more. 80 waves (5120 channels): 32 tokens 15.7 us in one piece and 17.0 split, 48 tokens 21.9 and
// 17.5; 640 waves: 54 tokens 26.6 and 40.1. Two, three, four and six waves of every SIMD: 1500 tokens of 5120 channels
// 82, 73.5, 75 and 79 us, of 8192 117, 104, 99 and 102.
void chan_segments(const ssm_scan_launch & L, chan_plan & P) {
    const int64_t waves = (L.H + 63) / 64 * L.S;
    int64_t n = 1;
    if (L.T * (820 - waves) > 32 * 820) n = std::min<int64_t>({ (4096 + waves - 1) / waves, L.T / 8, 4096 });
    P.seg = (int) ((L.T + n - 1) / n);
    P.n_seg = (int) ((L.T + P.seg - 1) / P.seg);
}

template <int N>
void launch_channels(const chan_plan & P, hipStream_t st) {
    const ssm_scan_launch & L = P.L;
    const unsigned hx = (unsigned) ((L.H + 63) / 64);
    if (P.n_seg > 1) {
        launch(ssm_scan_channels_kernel<N, false>, dim3(hx, (unsigned) P.n_seg - 1, (unsigned) L.S), dim3(64), 0, st, P);
        launch(ssm_scan_join_kernel, dim3((unsigned) (((int64_t) N * L.H + 255) / 256), (unsigned) L.S), dim3(256), 0, st, P);
    }
    launch(ssm_scan_channels_kernel<N, true>, dim3(hx, (unsigned) P.n_seg, (unsigned) L.S), dim3(64), 0, st, P);
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
    // up to 2^25 tiles; a dimension of the grid has less than 2^32 threads
    const int64_t tiles = blocks * ((L.T + 63) / 64), across = std::min<int64_t>(tiles, 1 << 22);
    launch(ssm_conv_tile_kernel, dim3((unsigned) across, (unsigned) std::min<int64_t>(L.S, 65535), (unsigned) ((tiles + across - 1) / across)),
           dim3(256), lds, st, L, blocks);
}

int64_t ssm_scan_scratch_bytes(const ssm_scan_launch & L) {
    if (L.S == 0) return 0;                                    // nothing to launch, and no workgroups to share segments
    if (!channels_take(L)) return ssm_scan_mm_takes(L) ? ssm_scan_mm_scratch_bytes(L) : 0;
    chan_plan P{};
    chan_segments(L, P);
    return P.n_seg == 1 ? 0 : L.S * P.n_seg * (int64_t) L.H * (L.N + 1) * 4;
}

void launch_ssm_scan(const ssm_scan_launch & L, void * ws, hipStream_t st) {
    if ((int64_t) L.P * L.H * L.S == 0) return;
    if (channels_take(L)) {
        chan_plan P{};
        P.L = L;
        chan_segments(L, P);
        P.part = (float *) ws;
        P.sums = P.part + L.S * P.n_seg * (int64_t) L.H * L.N;
        if (L.N == 8) launch_channels<8>(P, st);
        else if (L.N == 16) launch_channels<16>(P, st);
        else launch_channels<32>(P, st);
        return;
    }
    if (ssm_scan_mm_takes(L)) {
        launch_ssm_scan_mm(L, ws, st);
        return;
    }
    if (step_takes(L)) {
        if (L.N <= 16) launch_step<4>(L, st);
        else if (L.N <= 32) launch_step<8>(L, st);
        else if (L.N <= 64) launch_step<16>(L, st);
        else if (L.N <= 128) launch_step<32>(L, st);
        else launch_step<64>(L, st);
        return;
    }
    if (L.N <= 16) launch_rows<16, 1>(L, st);
    else if (L.N <= 32) launch_rows<32, 1>(L, st);
    else if (L.N <= 64) launch_rows<64, 1>(L, st);
    else if (L.N <= 128) launch_rows<64, 2>(L, st);
    else launch_rows<64, 4>(L, st);
}
