// k_ssm_mm.hip — the selective scan with one decay per head over many tokens, as matrix products.
//
// Over a chunk of 64 tokens, with d_j = softplus(dt_j), c_t = sum_{j <= t} d_j A, S the state at the
// chunk's start [n, p] and X_j = d_j x_j:
//   y_t = exp(c_t) C_t S + sum_{j <= t} (C_t . B_j) exp(c_t - c_j) X_j
//   S'  = exp(c_63) S + sum_j B_j (exp(c_63 - c_j) X_j)^T
// which is 4 N P operations per token beside the 64 P of the sum over the chunk, where the recurrence
// itself is three vector operations per state and token (330 us for 4096 tokens of 128 heads x 64 x
// 128 at the vector rate, which no layout can go below).
//
// The products run on the F16 matrix cores. Every operand is scaled by a power of two that puts its
// largest magnitude at 2^12 and split as x = hi + lo, two halves: 22 bits, and values down to 2^-26 of
// the largest lose none of them. hi hi + hi lo + lo hi is then a float32 product to within 2^-22, at
// 16/3 times the rate of the float32 matrix instructions. Sums and states are float32. The running
// sums c are formed in double and kept as two floats, so that their differences keep 24 bits.
//
// Three launches. `prepare`, per (sequence, chunk, group): C and B split into the order in which the
// lanes of a matrix instruction hold them, and the products C_t . B_j, which the group's heads share;
// per (sequence, chunk, 16 heads): c and its exponentials. `scan<false>`, where the tokens are split
// into segments for want of heads: each segment's state from nothing. `scan<true>`: the segments
// before joined, then the chunks one after another. A wave holds the states of 16 or 32 channels of a
// head in registers for its whole segment: the instruction that updates them leaves state n of
// channel p in the lane that the next chunk's product reads it from, when the k index of that product
// runs n = 4 g + i, then 16 + 4 g + i over lane group g, the order that C is prepared in.
//
// A value that is not finite must not reach earlier tokens of its chunk through 0 times it: X is
// cleared of such values, and the channel's outputs from that token on, and its state, are NaN. (B, C
// and dt enter rows and columns of their own only.)
#include "hip_common.h"
#include "kernels.h"

#include <algorithm>

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int Q = 64;                        // tokens per chunk
constexpr int STEP_WORDS = 5 * Q;            // exp(c), exp(c_63 - c), d, c as two floats
constexpr int M_BYTES = 6 * 1024;            // one plane of a head's 64 x 64 lower triangle, in 16 x 32 blocks
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// the power of two that takes a largest magnitude to 2^12 .. 2^13, and its inverse
__device__ __forceinline__ float scale_of(float most) {
    const int e = (int) (__float_as_uint(most) >> 23 & 255);
    return __uint_as_float((uint32_t) min(266 - e, 247) << 23);
}
__device__ __forceinline__ float inverse_of(float scale) { return __uint_as_float((254u - (__float_as_uint(scale) >> 23)) << 23); }
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }

// eight scaled values as hi + lo
__device__ __forceinline__ void split8(const float (&v)[8], half8 & hi, half8 & lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const half2v h = __builtin_convertvector(float2v{ v[i], v[i + 1] }, half2v);
        const half2v l = __builtin_convertvector(float2v{ fmaf((float) h[0], -1.0f, v[i]), fmaf((float) h[1], -1.0f, v[i + 1]) }, half2v);
        hi[i] = h[0]; hi[i + 1] = h[1];
        lo[i] = l[0]; lo[i + 1] = l[1];
    }
}

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float4v mfma3(half8 ah, half8 al, half8 bh, half8 bl, float4v c) {
    return mfma(ah, bh, mfma(ah, bl, mfma(al, bh, c)));
}

// log(1 + e^x); above 20 the sum rounds to e^x, so x itself (the unary op's rule)
__device__ __forceinline__ float softplus(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// what the launches share; offsets into the scratch in bytes
struct mm_plan {
    ssm_scan_launch L;
    char *          ws;
    int64_t         planes, gmat, scales, steps, parts, decays;
    const float *   s0;           // initial states: the pool (ids) or, for later blocks of tokens, [N, P, H, S]
    float *         s1;           // final states [N, P, H, S]
    int64_t         t0;           // first token
    int             T;            // tokens
    int             nc;           // chunks
    int             n_seg, seg;   // segments, chunks per segment
    int             pooled;       // s0 is the pool
    int             vec_bc, vec_s0, vec_s1;
    int             hw, slices, head_blocks, p_blocks;   // heads per workgroup, waves per head, ...
};

template <int NK> constexpr int64_t rec_bytes() { return (int64_t) NK * 16 * 1024; }   // C and B of a chunk and group: two planes each

// ---------------------------------------------------------------------------------------------
// prepare

// eight states of a token in the order of the products' k index: 4 from n, 4 from n + 16
__device__ __forceinline__ void load_perm(const float * row, int n, int N, bool vec, float (&v)[8]) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const int k = n + 16 * q;
        if (vec && k + 3 < N) {
            const float4 f = *(const float4 *) (row + k);
            v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * q + i] = k + i < N ? row[k + i] : 0.0f;
        }
    }
}

__device__ __forceinline__ float block_max(float v, float * s) {
    v = wave_max(v);
    if (threadIdx.x % WAVE == 0) s[threadIdx.x / WAVE] = v;
    __syncthreads();
    v = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    __syncthreads();
    return v;
}

template <int NK>
__device__ void prepare_operands(const mm_plan & P, int s, int c, int g, char * lds) {
    const ssm_scan_launch & L = P.L;
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int left = P.T - c * Q;             // tokens from the chunk's first on
    float * red = (float *) (lds + 16 * 1024 * NK);
    constexpr int PLANE = 4 * 1024 * NK;
    const int64_t rec = ((int64_t) s * P.nc + c) * L.G + g;
    char * out = P.ws + P.planes + rec * rec_bytes<NK>();
    const float * src[2] = { L.C + g * L.c_g + s * L.c_s + (P.t0 + c * Q) * L.c_t, L.B + g * L.b_g + s * L.b_s + (P.t0 + c * Q) * L.b_t };
    const int64_t stride[2] = { L.c_t, L.b_t };
    float inv[2];
#pragma unroll
    for (int o = 0; o < 2; o++) {
        float v[NK][8], most = 0.0f;
#pragma unroll
        for (int q = 0; q < NK; q++) {
            const int it = tid + 256 * q, tt = it / (64 * NK), ks = it / 64 % NK;
            const int t = 16 * tt + lane % 16;
            load_perm(src[o] + (int64_t) min(t, left - 1) * stride[o], 32 * ks + 4 * (lane / 16), L.N, P.vec_bc, v[q]);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[q][i] = t < left ? v[q][i] : 0.0f;
                most = fmaxf(most, finite_abs(v[q][i]));
            }
        }
        const float sc = scale_of(block_max(most, red));
        inv[o] = inverse_of(sc);
#pragma unroll
        for (int q = 0; q < NK; q++) {
            const int it = tid + 256 * q;
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i++) v[q][i] *= sc;
            split8(v[q], hi, lo);
            char * at = lds + o * 2 * PLANE + it * 16;
            *(half8 *) at = hi;
            *(half8 *) (at + PLANE) = lo;
            if (o == 0) {
                *(half8 *) (out + it * 16) = hi;
                *(half8 *) (out + PLANE + it * 16) = lo;
            }
        }
    }
    __syncthreads();
    // C_t . B_j for the blocks of 16 x 16 on and below the diagonal
    float * G = (float *) (P.ws + P.gmat) + rec * Q * Q;
    float most = 0.0f;
    for (int q = wave; q < 10; q += 4) {
        const int tt = q < 1 ? 0 : q < 3 ? 1 : q < 6 ? 2 : 3, jt = q - tt * (tt + 1) / 2;
        float4v acc = { 0, 0, 0, 0 };
#pragma unroll
        for (int ks = 0; ks < NK; ks++) {
            const char * a = lds + ((tt * NK + ks) * 64 + lane) * 16, * b = lds + 2 * PLANE + ((jt * NK + ks) * 64 + lane) * 16;
            acc = mfma3(*(const half8 *) a, *(const half8 *) (a + PLANE), *(const half8 *) b, *(const half8 *) (b + PLANE), acc);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = acc[i] * inv[0] * inv[1];
            G[(16 * tt + 4 * (lane / 16) + i) * Q + 16 * jt + lane % 16] = v;
            most = fmaxf(most, finite_abs(v));
        }
    }
    most = block_max(most, red);
    if (tid == 0) {
        float * sc = (float *) (P.ws + P.scales) + rec * 4;
        sc[0] = inv[0]; sc[1] = inv[1]; sc[2] = most;
    }
    // B with the tokens as its k index: row n, eight tokens per lane
    const uint16_t * bh = (const uint16_t *) (lds + 2 * PLANE);
#pragma unroll
    for (int q = 0; q < NK; q++) {
        const int it = tid + 256 * q, nt = it / 128, ks = it / 64 % 2;
        const int n = 16 * nt + lane % 16, j0 = 32 * ks + 8 * (lane / 16), m = n % 32;
        const int at = (n / 32 * 64 + 16 * (m % 16 / 4)) * 8 + m / 16 * 4 + m % 4;
        uint32_t w[2][4];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = j0 + i, k = at + (j / 16 * NK * 64 + j % 16) * 8;
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const uint32_t u = bh[k + p * (PLANE / 2)];
                w[p][i / 2] = i % 2 ? w[p][i / 2] | u << 16 : u;
            }
        }
#pragma unroll
        for (int p = 0; p < 2; p++) *(uint4 *) (out + (2 + p) * PLANE + it * 16) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
}

// 16 heads' running sums over a chunk: a wave per head, a lane per token
__device__ void prepare_steps(const mm_plan & P, int s, int c, int h0, float * lds) {
    const ssm_scan_launch & L = P.L;
    const int tid = threadIdx.x, lane = tid % WAVE, left = P.T - c * Q;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int t = 16 * i + tid / 16, h = h0 + tid % 16;
        lds[t * 17 + tid % 16] = t < left && h < L.H ? L.dt[h + (P.t0 + c * Q + t) * L.dt_t + s * L.dt_s] : 0.0f;
    }
    __syncthreads();
    for (int k = tid / WAVE; k < 16; k += 4) {
        const int h = h0 + k;
        if (h >= L.H) break;
        // a token past the last neither decays nor adds
        const float d = lane < left ? softplus(lds[lane * 17 + k]) : 0.0f;
        double sum = (double) d * ((double) L.A[h * L.a_h] * 1.4426950408889634074);
        if (lane >= left) sum = 0.0;
#pragma unroll
        for (int o = 1; o < WAVE; o *= 2) {
            const double u = __shfl_up(sum, o, WAVE);
            sum += lane >= o ? u : 0.0;
        }
        const double rest = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(sum), 63),
                                             __builtin_amdgcn_readlane(__double2loint(sum), 63)) - sum;
        const float hi = (float) sum, lo = fabsf(hi) < INFINITY ? (float) (sum - (double) hi) : 0.0f;
        const float rh = (float) rest, rl = fabsf(rh) < INFINITY ? (float) (rest - (double) rh) : 0.0f;
        float * o = (float *) (P.ws + P.steps) + (((int64_t) s * P.nc + c) * L.H + h) * STEP_WORDS + lane;
        o[0] = exp2_hw(hi) * fmaf(lo, LN2, 1.0f);
        o[Q] = exp2_hw(rh) * fmaf(rl, LN2, 1.0f);
        o[2 * Q] = d;
        o[3 * Q] = hi;
        o[4 * Q] = lo;
    }
}

template <int NK>
__global__ __launch_bounds__(256) void ssm_prepare_kernel(mm_plan P) {
    extern __shared__ __align__(16) char lds[];
    const int c = blockIdx.x, y = blockIdx.y, s = blockIdx.z;
    if (y < P.L.G) prepare_operands<NK>(P, s, c, y, lds);
    else prepare_steps(P, s, c, (y - P.L.G) * 16, (float *) lds);
}

// ---------------------------------------------------------------------------------------------
// scan

// NK: steps of 32 states; PT: tiles of 16 channels per wave; OUT: outputs and final states, else the
// segment's state from nothing
template <int NK, int PT, bool OUT>
__global__ __launch_bounds__(256, 2) void ssm_scan_mm_kernel(mm_plan P) {
    extern __shared__ __align__(16) char lds[];
    const ssm_scan_launch & L = P.L;
    constexpr int PLANE = 4 * 1024 * NK;
    char * buf = lds;                                          // C's planes, then B's
    float * steps = (float *) (lds + 2 * PLANE);               // per head
    char * mats = (char *) (steps + P.hw * STEP_WORDS);        // per head: the two planes of (C_t . B_j) exp(c_t - c_j)
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE, col = lane % 16, grp = lane / 16;

    // the workgroups that read the same operands take turns on one XCD (consecutive ids go to different ones)
    const int members = P.head_blocks * P.p_blocks, units = (int) (gridDim.x / (unsigned) members);
    int u, m;
    if (units % 8 == 0) {
        const int q = (int) blockIdx.x / 8;
        u = (int) blockIdx.x % 8 + 8 * (q / members);
        m = q % members;
    } else {
        u = (int) blockIdx.x / members;
        m = (int) blockIdx.x % members;
    }
    const int g = u % L.G, sg = u / L.G % P.n_seg, s = u / (L.G * P.n_seg);
    const int per = L.H / L.G;
    const int hl = P.p_blocks > 1 ? 0 : wave / P.slices, slice = P.p_blocks > 1 ? m % P.p_blocks * 4 + wave : wave % P.slices;
    if (!OUT && sg == P.n_seg - 1) return;                     // nobody starts from the last segment's state
    const int hb = m / P.p_blocks * P.hw;
    const int heads = min(P.hw, per - hb);                     // heads of this workgroup
    const bool active = hl < heads && slice < P.slices;
    const int h = g * per + hb + (active ? hl : 0);
    const int c0 = sg * P.seg, c1 = min(P.nc, c0 + P.seg);

    // the wave's states: tile nt, channel tile pt, i: state 16 nt + 4 grp + i of channel 16 (slice PT + pt) + col
    float4v S[2 * NK][PT];
    int pch[PT];
    bool pok[PT];
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
        const int p = 16 * (slice * PT + pt) + col;
        pok[pt] = active && p < L.P;
        pch[pt] = min(p, L.P - 1);
    }
#pragma unroll
    for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
        for (int pt = 0; pt < PT; pt++) S[nt][pt] = float4v{ 0, 0, 0, 0 };
    }
    if (OUT && active) {
        int64_t row = s;
        if (P.pooled) {
            row = L.ids[s * L.ids_s];
            row = row < 0 ? 0 : row >= L.pool ? L.pool - 1 : row;
        }
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
            const float * s0 = P.s0 + (P.pooled ? pch[pt] * L.s_p + h * L.s_h + row * L.s_row
                                                : (int64_t) L.N * (pch[pt] + (int64_t) L.P * (h + (int64_t) L.H * s)));
#pragma unroll
            for (int nt = 0; nt < 2 * NK; nt++) {
                const int n = 16 * nt + 4 * grp;
                if (P.vec_s0 && n + 3 < L.N) {
                    const float4 f = *(const float4 *) (s0 + n);
                    S[nt][pt] = float4v{ f.x, f.y, f.z, f.w };
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) S[nt][pt][i] = n + i < L.N ? s0[n + i] : 0.0f;
                }
            }
        }
    }
    // segments' states: in the order the lanes hold them
    auto part_at = [&](int k) {
        return (float4v *) (P.ws + P.parts) + ((((int64_t) s * P.n_seg + k) * L.H + h) * P.slices + slice) * (2 * NK * PT * WAVE) + lane;
    };
    if (OUT && active) {
        for (int k = 0; k < sg; k++) {
            const float dec = ((const float *) (P.ws + P.decays))[((int64_t) s * P.n_seg + k) * L.H + h];
            const float4v * q = part_at(k);
#pragma unroll
            for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                for (int pt = 0; pt < PT; pt++) {
                    const float4v f = q[(nt * PT + pt) * WAVE];
#pragma unroll
                    for (int i = 0; i < 4; i++) S[nt][pt][i] = fmaf(S[nt][pt][i], dec, f[i]);
                }
            }
        }
    }

    uint4v stage[2 * NK];                                      // a thread's share of an operand's planes on their way to LDS
    auto fetch = [&](int c, int which) {
        const char * src = P.ws + P.planes + (((int64_t) s * P.nc + c) * L.G + g) * rec_bytes<NK>() + which * 2 * PLANE + tid * 16;
#pragma unroll
        for (int q = 0; q < 2 * NK; q++) stage[q] = *(const uint4v *) (src + q * 4096);
    };
    auto put = [&]() {
#pragma unroll
        for (int q = 0; q < 2 * NK; q++) *(uint4v *) (buf + tid * 16 + q * 4096) = stage[q];
    };

    float decay = 1.0f;                                        // of the segment so far
    fetch(c0, OUT ? 0 : 1);
    for (int c = c0; c < c1; c++) {
        const int left = P.T - c * Q;
        // X's inputs: token 32 ks + 8 grp + i of the wave's channels
        float x[PT][2][8];
        {
            // one lane offset for all of them: the rest of each address is the wave's
            const float * xp = L.x + h * L.x_h + s * L.x_s + (P.t0 + c * Q) * L.x_t;
            if (left >= Q) {
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float * xi = xp + (32 * ks + i) * L.x_t;
#pragma unroll
                        for (int pt = 0; pt < PT; pt++) x[pt][ks][i] = xi[(uint32_t) (8 * grp * (int) L.x_t + pch[pt])];
                    }
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int t = min(32 * ks + 8 * grp + i, left - 1);
#pragma unroll
                        for (int pt = 0; pt < PT; pt++) x[pt][ks][i] = xp[(uint32_t) (t * (int) L.x_t + pch[pt])];
                    }
                }
            }
        }
        __syncthreads();                                       // the last chunk's reads of LDS are done
        put();
        {
            const float * sp = (const float *) (P.ws + P.steps) + (((int64_t) s * P.nc + c) * L.H + g * per + hb) * STEP_WORDS;
            for (int i = tid; i < heads * (STEP_WORDS / 4); i += 256) ((float4 *) steps)[i] = ((const float4 *) sp)[i];
        }
        const float * scales = (const float *) (P.ws + P.scales) + (((int64_t) s * P.nc + c) * L.G + g) * 4;
        const float inv_c = scales[0], inv_b = scales[1], gmost = scales[2];
        if (OUT) fetch(c, 1);
        __syncthreads();
        const float * my = steps + (active ? hl : 0) * STEP_WORDS;
        const float e_last = my[Q - 1];
        if (OUT) {
            // (C_t . B_j) exp(c_t - c_j) below the diagonal, split, in the order of the A operand: thread's row t, eight j
            const float * G = (const float *) (P.ws + P.gmat) + (((int64_t) s * P.nc + c) * L.G + g) * Q * Q;
            for (int it = tid; it < heads * 384; it += 256) {
                const int k = it / 384, e = it - k * 384;
                const int t = e < 128 ? e / 4 : 32 + (e - 128) / 8, jb = e < 128 ? e % 4 : e % 8;
                const float * st = steps + k * STEP_WORDS;
                const float sm = scale_of(gmost * fmaxf(1.0f, st[Q - 1]));
                const float ht = st[3 * Q + t], lt = st[4 * Q + t];
                const float4 g0 = *(const float4 *) (G + t * Q + 8 * jb), g1 = *(const float4 *) (G + t * Q + 8 * jb + 4);
                const float4 h0 = *(const float4 *) (st + 3 * Q + 8 * jb), h1 = *(const float4 *) (st + 3 * Q + 8 * jb + 4);
                const float4 l0 = *(const float4 *) (st + 4 * Q + 8 * jb), l1 = *(const float4 *) (st + 4 * Q + 8 * jb + 4);
                const float gg[8] = { g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w };
                const float hh[8] = { h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w };
                const float ll[8] = { l0.x, l0.y, l0.z, l0.w, l1.x, l1.y, l1.z, l1.w };
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float w = gg[i] * sm * exp2_hw((ht - hh[i]) + (lt - ll[i]));
                    v[i] = 8 * jb + i <= t ? w : 0.0f;
                }
                half8 hi, lo;
                split8(v, hi, lo);
                const int tt = t / 16, blk = tt < 2 ? tt : 2 * tt - 2 + jb / 4;
                char * at = mats + k * 2 * M_BYTES + blk * 1024 + (t % 16 + 16 * (jb % 4)) * 16;
                *(half8 *) at = hi;
                *(half8 *) (at + M_BYTES) = lo;
            }
        }
        // X = d x, cleared of tokens past the last and of values that are not finite
        int bad[PT];                                           // the channel's first token with such a value
        float sx[PT];
        {
            float odd = 0.0f;
#pragma unroll
            for (int pt = 0; pt < PT; pt++) {
                float most = 0.0f;
                bad[pt] = Q;
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    const float4 d0 = *(const float4 *) (my + 2 * Q + 32 * ks + 8 * grp), d1 = *(const float4 *) (my + 2 * Q + 32 * ks + 8 * grp + 4);
                    const float dd[8] = { d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w };
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float v = pok[pt] && 32 * ks + 8 * grp + i < left ? x[pt][ks][i] * dd[i] : 0.0f;
                        x[pt][ks][i] = v;
                        odd = fmaf(v, 0.0f, odd);
                        most = fmaxf(most, fabsf(v));
                    }
                }
                sx[pt] = most;
            }
            if (__any(odd != 0.0f)) {
#pragma unroll
                for (int pt = 0; pt < PT; pt++) {
                    sx[pt] = 0.0f;
#pragma unroll
                    for (int ks = 1; ks >= 0; ks--) {
#pragma unroll
                        for (int i = 7; i >= 0; i--) {
                            const bool fine = fabsf(x[pt][ks][i]) < INFINITY;
                            if (!fine) bad[pt] = 32 * ks + 8 * grp + i;
                            x[pt][ks][i] = fine ? x[pt][ks][i] : 0.0f;
                            sx[pt] = fmaxf(sx[pt], fabsf(x[pt][ks][i]));
                        }
                    }
                    bad[pt] = min(bad[pt], __shfl_xor(bad[pt], 16, WAVE));
                    bad[pt] = min(bad[pt], __shfl_xor(bad[pt], 32, WAVE));
                }
            }
#pragma unroll
            for (int pt = 0; pt < PT; pt++) {
                sx[pt] = fmaxf(sx[pt], __shfl_xor(sx[pt], 16, WAVE));
                sx[pt] = fmaxf(sx[pt], __shfl_xor(sx[pt], 32, WAVE));
            }
        }
        if (OUT) {
            // exp(c_t) C_t S
            float4v acc[4][PT];
            float inv_s[PT];
            if (active) {
                float ss[PT];
#pragma unroll
                for (int pt = 0; pt < PT; pt++) {
                    float most = 0.0f;
#pragma unroll
                    for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(S[nt][pt][i]));
                    }
                    most = fmaxf(most, __shfl_xor(most, 16, WAVE));
                    most = fmaxf(most, __shfl_xor(most, 32, WAVE));
                    if (__any(!(most < INFINITY))) {
                        most = 0.0f;
#pragma unroll
                        for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                            for (int i = 0; i < 4; i++) most = fmaxf(most, finite_abs(S[nt][pt][i]));
                        }
                        most = fmaxf(most, __shfl_xor(most, 16, WAVE));
                        most = fmaxf(most, __shfl_xor(most, 32, WAVE));
                    }
                    ss[pt] = scale_of(most);
                    inv_s[pt] = inverse_of(ss[pt]) * inv_c;
                }
#pragma unroll
                for (int tt = 0; tt < 4; tt++) {
#pragma unroll
                    for (int pt = 0; pt < PT; pt++) acc[tt][pt] = float4v{ 0, 0, 0, 0 };
                }
#pragma unroll
                for (int ks = 0; ks < NK; ks++) {
                    half8 bh[PT], bl[PT];
#pragma unroll
                    for (int pt = 0; pt < PT; pt++) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = as_f32(S[2 * ks + i / 4][pt][i % 4] * ss[pt]);
                        split8(v, bh[pt], bl[pt]);
                    }
#pragma unroll
                    for (int tt = 0; tt < 4; tt++) {
                        const char * a = buf + ((tt * NK + ks) * 64 + lane) * 16;
                        const half8 ah = *(const half8 *) a, al = *(const half8 *) (a + PLANE);
#pragma unroll
                        for (int pt = 0; pt < PT; pt++) acc[tt][pt] = mfma3(ah, al, bh[pt], bl[pt], acc[tt][pt]);
                    }
                }
            }
            __syncthreads();                                   // C is read, the matrices are written
            put();
            if (active) {
                half8 xh[PT][2], xl[PT][2];
                float inv_x[PT];
                const float inv_m = inverse_of(scale_of(gmost * fmaxf(1.0f, e_last)));
#pragma unroll
                for (int pt = 0; pt < PT; pt++) {
                    const float sc = scale_of(sx[pt]);
                    inv_x[pt] = inverse_of(sc);
#pragma unroll
                    for (int ks = 0; ks < 2; ks++) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = as_f32(x[pt][ks][i] * sc);
                        split8(v, xh[pt][ks], xl[pt][ks]);
                    }
                }
                const char * mine = mats + hl * 2 * M_BYTES + lane * 16;
                float * y = L.y + h * L.P + (int64_t) L.P * L.H * (P.t0 + c * Q + L.T * s);
#pragma unroll
                for (int tt = 0; tt < 4; tt++) {
                    float4v sum[PT];
#pragma unroll
                    for (int pt = 0; pt < PT; pt++) sum[pt] = float4v{ 0, 0, 0, 0 };
#pragma unroll
                    for (int ks = 0; ks <= tt / 2; ks++) {
                        const char * a = mine + (tt < 2 ? tt : 2 * tt - 2 + ks) * 1024;
                        const half8 ah = *(const half8 *) a, al = *(const half8 *) (a + M_BYTES);
#pragma unroll
                        for (int pt = 0; pt < PT; pt++) sum[pt] = mfma3(ah, al, xh[pt][ks], xl[pt][ks], sum[pt]);
                    }
                    const float4 e4 = *(const float4 *) (my + 16 * tt + 4 * grp);
                    const float e[4] = { e4.x, e4.y, e4.z, e4.w };
#pragma unroll
                    for (int pt = 0; pt < PT; pt++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int t = 16 * tt + 4 * grp + i;
                            float v = fmaf(acc[tt][pt][i] * inv_s[pt], e[i], sum[pt][i] * inv_m * inv_x[pt]);
                            v = t < bad[pt] ? v : NAN;
                            if (pok[pt] && t < left) (y + (16 * tt + i) * L.P * L.H)[(uint32_t) (4 * grp * L.P * L.H + pch[pt])] = v;
                        }
                    }
                }
            }
            if (c + 1 < c1) fetch(c + 1, 0);
            __syncthreads();                                   // B is in place
        } else if (c + 1 < c1) {
            fetch(c + 1, 1);
        }
        // the state at the chunk's end
        if (active) {
            half8 xh[PT][2], xl[PT][2];
            float inv_x[PT];
            const float grow = fmaxf(1.0f, my[Q]);
#pragma unroll
            for (int pt = 0; pt < PT; pt++) {
                const float sc = scale_of(sx[pt] * grow);
                inv_x[pt] = inverse_of(sc) * inv_b;
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    const float4 w0 = *(const float4 *) (my + Q + 32 * ks + 8 * grp), w1 = *(const float4 *) (my + Q + 32 * ks + 8 * grp + 4);
                    const float ww[8] = { w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w };
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = as_f32(x[pt][ks][i] * ww[i] * sc);
                    split8(v, xh[pt][ks], xl[pt][ks]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < 2 * NK; nt++) {
                float4v sum[PT];
#pragma unroll
                for (int pt = 0; pt < PT; pt++) sum[pt] = float4v{ 0, 0, 0, 0 };
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    const char * a = buf + ((nt * 2 + ks) * 64 + lane) * 16;
                    const half8 ah = *(const half8 *) a, al = *(const half8 *) (a + PLANE);
#pragma unroll
                    for (int pt = 0; pt < PT; pt++) sum[pt] = mfma3(ah, al, xh[pt][ks], xl[pt][ks], sum[pt]);
                }
#pragma unroll
                for (int pt = 0; pt < PT; pt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float v = fmaf(S[nt][pt][i], e_last, sum[pt][i] * inv_x[pt]);
                        S[nt][pt][i] = bad[pt] < Q ? NAN : v;
                    }
                }
            }
            decay *= e_last;
        }
    }
    if (!active) return;
    if (!OUT) {
        if (lane == 0 && slice == 0) ((float *) (P.ws + P.decays))[((int64_t) s * P.n_seg + sg) * L.H + h] = decay;
        float4v * q = part_at(sg);
#pragma unroll
        for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
            for (int pt = 0; pt < PT; pt++) q[(nt * PT + pt) * WAVE] = S[nt][pt];
        }
    } else if (c1 == P.nc) {
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
            if (!pok[pt]) continue;
            float * s1 = P.s1 + (int64_t) L.N * (pch[pt] + (int64_t) L.P * (h + (int64_t) L.H * s));
#pragma unroll
            for (int nt = 0; nt < 2 * NK; nt++) {
                const int n = 16 * nt + 4 * grp;
                if (P.vec_s1 && n + 3 < L.N) {
                    *(float4 *) (s1 + n) = make_float4(S[nt][pt][0], S[nt][pt][1], S[nt][pt][2], S[nt][pt][3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (n + i < L.N) s1[n + i] = S[nt][pt][i];
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------

int steps_of(int N) { return N <= 32 ? 1 : N <= 64 ? 2 : N <= 128 ? 4 : 8; }
// two tiles of channels per wave read each operand from LDS once for both; eight steps of states leave no registers for that
int tiles_of(int N, int P) { return steps_of(N) == 8 || P <= 16 ? 1 : 2; }

struct mm_sizes {
    int     nk, pt, slices, hw, head_blocks, p_blocks;
    int64_t chunks, block, n_seg, seg;      // chunks in all and per block of tokens, segments of a block
    int64_t planes, gmat, scales, steps, parts, decays, state, total;
};

mm_sizes mm_size(const ssm_scan_launch & L) {
    mm_sizes z;
    z.nk = steps_of(L.N);
    z.pt = tiles_of(L.N, L.P);
    z.slices = (L.P + 16 * z.pt - 1) / (16 * z.pt);
    z.hw = z.slices == 1 ? 4 : z.slices == 2 ? 2 : 1;
    z.p_blocks = (z.slices + 3) / 4;
    z.head_blocks = (L.H / L.G + z.hw - 1) / z.hw;
    z.chunks = (L.T + Q - 1) / Q;
    const int64_t rec = (int64_t) z.nk * 16384 + Q * Q * 4 + 16, per = L.S * (L.G * rec + (int64_t) L.H * STEP_WORDS * 4);
    // prepared operands of at most 64 MiB: the tokens go through in blocks
    z.block = std::max<int64_t>(1, std::min<int64_t>({ z.chunks, ((int64_t) 64 << 20) / per, 65535 }));
    // segments until two workgroups of every CU have work, of at least two chunks
    const int64_t base = L.S * L.G * z.head_blocks * z.p_blocks;
    const int64_t part = L.S * L.H * (int64_t) z.slices * (2 * z.nk * z.pt * WAVE * 16 + 4);
    z.n_seg = std::max<int64_t>(1, std::min<int64_t>({ (512 + base - 1) / base, z.block / 2, ((int64_t) 32 << 20) / part }));
    z.seg = (z.block + z.n_seg - 1) / z.n_seg;
    z.n_seg = (z.block + z.seg - 1) / z.seg;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
    z.planes = take(L.S * z.block * L.G * (int64_t) z.nk * 16384);
    z.gmat = take(L.S * z.block * L.G * Q * Q * 4);
    z.scales = take(L.S * z.block * L.G * 16);
    z.steps = take(L.S * z.block * (int64_t) L.H * STEP_WORDS * 4);
    z.parts = take(z.n_seg > 1 ? L.S * z.n_seg * (int64_t) L.H * z.slices * 2 * z.nk * z.pt * WAVE * 16 : 0);
    z.decays = take(z.n_seg > 1 ? L.S * z.n_seg * (int64_t) L.H * 4 : 0);
    // states between blocks of tokens, one read while the next is written
    z.state = take(z.block < z.chunks ? 2 * L.S * (int64_t) L.N * L.P * L.H * 4 : 0);
    z.total = at;
    return z;
}

template <int NK, int PT>
void launch_mm(const ssm_scan_launch & L, const mm_sizes & z, void * ws, hipStream_t st) {
    mm_plan P{};
    P.L = L;
    P.ws = (char *) ws;
    P.planes = z.planes; P.gmat = z.gmat; P.scales = z.scales; P.steps = z.steps; P.parts = z.parts; P.decays = z.decays;
    P.hw = z.hw; P.slices = z.slices; P.head_blocks = z.head_blocks; P.p_blocks = z.p_blocks;
    static const bool lds_set = [] {
        HIP_CHECK(hipFuncSetAttribute((const void *) ssm_prepare_kernel<NK>, hipFuncAttributeMaxDynamicSharedMemorySize, NK * 16384 + 64));
        HIP_CHECK(hipFuncSetAttribute((const void *) ssm_scan_mm_kernel<NK, PT, true>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                      NK * 8192 + 4 * (STEP_WORDS * 4 + 2 * M_BYTES)));
        return true;
    }();
    (void) lds_set;
    auto rows16 = [](const void * p, int64_t a, int64_t b, int64_t c) { return (uintptr_t) p % 16 == 0 && a % 4 == 0 && b % 4 == 0 && c % 4 == 0; };
    P.vec_bc = rows16(L.B, L.b_g, L.b_t, L.b_s) && rows16(L.C, L.c_g, L.c_t, L.c_s);
    float * hold = (float *) ((char *) ws + z.state);
    const int64_t states = L.S * (int64_t) L.N * L.P * L.H;
    for (int64_t c = 0, turn = 0; c < z.chunks; c += z.block, turn ^= 1) {
        P.nc = (int) std::min(z.block, z.chunks - c);
        P.t0 = c * Q;
        P.T = (int) std::min<int64_t>(L.T - P.t0, (int64_t) P.nc * Q);
        P.seg = (int) z.seg;
        P.n_seg = (P.nc + P.seg - 1) / P.seg;
        P.pooled = c == 0;
        P.s0 = c == 0 ? L.s : hold + (turn ^ 1) * states;
        P.s1 = c + z.block < z.chunks ? hold + turn * states : L.s_out;
        P.vec_s0 = c == 0 ? rows16(L.s, L.s_p, L.s_h, L.s_row) : L.N % 4 == 0 && (uintptr_t) P.s0 % 16 == 0;
        P.vec_s1 = L.N % 4 == 0 && (uintptr_t) P.s1 % 16 == 0;
        const size_t planes = (size_t) NK * 8192;
        launch(ssm_prepare_kernel<NK>, dim3((unsigned) P.nc, (unsigned) (L.G + (L.H + 15) / 16), (unsigned) L.S), dim3(256),
               std::max<size_t>(2 * planes + 64, Q * 17 * 4), st, P);
        const size_t lds = planes + (size_t) z.hw * STEP_WORDS * 4;
        const unsigned members = (unsigned) (z.head_blocks * z.p_blocks);
        if (P.n_seg > 1) launch(ssm_scan_mm_kernel<NK, PT, false>, dim3((unsigned) (L.S * L.G * P.n_seg) * members), dim3(256), lds, st, P);
        launch(ssm_scan_mm_kernel<NK, PT, true>, dim3((unsigned) (L.S * L.G * P.n_seg) * members), dim3(256), lds + (size_t) z.hw * 2 * M_BYTES, st, P);
    }
}

} // namespace

bool ssm_scan_mm_takes(const ssm_scan_launch & L) {
    // the grids' limits: one dimension each for the sequences and for groups and heads
    return L.a_scalar && L.T >= SSM_MM_MIN_TOKENS && L.S <= 65535 && L.G + (L.H + 15) / 16 <= 65535 &&
           L.S * (int64_t) L.H * L.P < INT32_MAX &&
           // 32-bit offsets within a chunk
           L.x_t >= 0 && L.x_t <= 1 << 24 && (int64_t) L.H * L.P <= 1 << 24 && L.P <= 1 << 24;
}

int64_t ssm_scan_mm_scratch_bytes(const ssm_scan_launch & L) { return mm_size(L).total; }

void launch_ssm_scan_mm(const ssm_scan_launch & L, void * ws, hipStream_t st) {
    const mm_sizes z = mm_size(L);
    if (z.nk == 8) launch_mm<8, 1>(L, z, ws, st);
    else if (z.nk == 4) z.pt == 2 ? launch_mm<4, 2>(L, z, ws, st) : launch_mm<4, 1>(L, z, ws, st);
    else if (z.nk == 2) z.pt == 2 ? launch_mm<2, 2>(L, z, ws, st) : launch_mm<2, 1>(L, z, ws, st);
    else z.pt == 2 ? launch_mm<1, 2>(L, z, ws, st) : launch_mm<1, 1>(L, z, ws, st);
}
