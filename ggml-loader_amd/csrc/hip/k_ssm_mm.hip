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
// largest magnitude at 2^14 and split as x = hi + 2^-12 lo, two halves: 22 bits down to 2^-30 of the
// largest, and below that an error of 2^-52 of the largest (2^-25 and 2^-12 of it: half a step of the
// smallest halves). hi hi + 2^-12 (hi lo + lo hi), two sums of matrix products, is then a float32
// product to within 2^-21, at 16/3 times the rate of the float32 matrix instructions. Sums and states are
// float32. The running sums c are formed in double and kept as two floats, so that their differences
// keep 24 bits.
//
// One power serves a chunk's C, one its B, one a row of the decayed products C_t . B_j, one a channel's X, its
// states, and its decayed X. So values that differ by more than 2^33 within one of these would lose bits to
// the largest, earlier tokens' outputs to later ones among them: a chunk in which they do, or in which one is
// not finite, is done by its recurrence instead (by_tokens), by the waves of its group for C and B, of its 16 channels
// for X and the states. Of the decayed products, which reach any depth, it is the row's largest against its own
// token's that counts, with the spread of X: outputs are wrong by 2^-52 of the largest |C_t . B_j| |X_j| before
// decay at most, which shows only where all inputs but zeros have decayed by more than 2^30.
// (With one sum for all three products and 2^12 for the largest, halves held 22 bits down to 2^-15 and a later
// value of 1e8 put the outputs before it off by 1e-3; that took 180 us instead of 196 at the first size below.)
//
// Three launches. ssm_prepare_kernel, per (sequence, chunk, group): C and B split into the order in which the
// lanes of a matrix instruction hold them, and the products C_t . B_j, which the group's heads share; per
// (sequence, chunk, 16 heads): c and its exponentials. ssm_scan_mm_kernel<NK, false>, where the tokens are split
// into segments for want of heads: each segment's state from nothing. ssm_scan_mm_kernel<NK, true>: the segments
// before joined, then the chunks one after another. A wave holds the states of 16 channels of a head in registers
// for its whole segment: the instruction that updates them leaves state n of channel p in the lane that the next
// chunk's product reads it from, when the k index of that product runs n = 4 g + i, then 16 + 4 g + i over lane
// group g, the order that C is prepared in. Eight waves share a chunk's operands.
//
// 4096 tokens of 128 heads x 64 x 128, 8 groups: 196 us (1.59 TB/s of what must be read and written, whose floor
// is 61 us; 22 + 46 + 130 in a trace), 333 tokens of 24 heads 35. Before the halves' range was widened these were 180
// and 32, and then nothing was saturated: the matrix cores were busy for a fifth of the time, the vector units for two
// fifths and LDS for a quarter, and leaving any one part out (the loads of x or of the operands, the update of the
// state, the stores) saved a tenth each, so a chunk's barriers and the latency between its parts were what was left.
// Against 119 to 126 us of the last launch then, two tiles of channels a wave took 166, workgroups of four waves 159,
// half the waves a step ahead of the others 149; four waves a SIMD with one buffer spilled.
#include "hip_common.h"
#include "kernels.h"
#include "ssm_ops.h"

#include <algorithm>
#include <atomic>

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int Q = 64;                        // tokens per chunk
// exp(c), exp(c_63 - c), d, c as two floats, exp(c at the end of its 16 tokens - c)
constexpr int STEP_WORDS = 6 * Q;
// per (sequence, chunk, group): the exponents of C's and B's powers of two; how far a row's largest |C_t . B_j|
// exceeds what its own token adds, at most (infinite where C, B or a product is out of range); the largest |C_t . B_j|;
// that of each row
constexpr int SCALE_WORDS = 4 + Q;
// C_t . B_j of a chunk: ten tiles of 16 x 16, the diagonal's and then, row by row, those below it, each as the
// matrices' lanes load it: two parts of 32 lanes (row + 16 (column / 8)) by four columns
constexpr int G_WORDS = 10 * 256;
constexpr int M_BYTES = 6 * 1024;            // one plane of a head's 64 x 64 lower triangle, in 16 x 32 blocks

// the exponent of the power of two that takes a largest magnitude to 2^14 .. 2^15, and that power
__device__ __forceinline__ int shift_of(float most) { return min(141 - (int) (__float_as_uint(most) >> 23 & 255), 126); }
__device__ __forceinline__ float power_of(int shift) { return __uint_as_float((uint32_t) (shift + 127) << 23); }
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }
// The smallest magnitude other than 0 is that of the least key, a NaN where there is none (and less a unit).
__device__ __forceinline__ uint32_t least_key(float x) { return (__float_as_uint(x) << 1) - 1; }
__device__ __forceinline__ float least_value(uint32_t key) { return __uint_as_float(key >> 1); }
// the larger one of a magnitude so far and another, and a NaN where there is one
__device__ __forceinline__ float most_of(float most, float x) { return __builtin_elementwise_maximum(most, fabsf(x)); }
// whether values are finite and the smallest other than 0 so near the largest that halves hold each to 2^-19
__device__ __forceinline__ bool in_range(float least, float most) { return most < INFINITY && !(least * 0x1p33f < most); }

// eight values times a power of two as hi + 2^-12 lo. The product is exact, so hi comes from one mixed-precision
// multiply-add, the rest from another and lo from a third.
__device__ __forceinline__ void split8(const float (&v)[8], float scale, half8 & hi, half8 & lo) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const _Float16 h = (_Float16) fmaf(v[i], scale, 0.0f);
        hi[i] = h;
        lo[i] = (_Float16) fmaf(fmaf(v[i], scale, -(float) h), 0x1p12f, 0.0f);
    }
}

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// a sum of products hi hi and the one of hi lo + lo hi, which stands 2^12 above it
__device__ __forceinline__ void mfma3(half8 ah, half8 al, half8 bh, half8 bl, float4v & sum, float4v & cross) {
    cross = mfma(al, bh, cross);
    sum = mfma(ah, bh, sum);
    cross = mfma(ah, bl, cross);
}
__device__ __forceinline__ float4v joined(float4v sum, float4v cross) {
#pragma unroll
    for (int i = 0; i < 4; i++) sum[i] = fmaf(cross[i], 0x1p-12f, sum[i]);
    return sum;
}

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
    int             hw, slices, head_blocks, p_blocks;   // heads per workgroup, waves per head, ...
};

template <int NK> constexpr int64_t rec_bytes() { return (int64_t) NK * 16 * 1024; }   // C and B of a chunk and group: two planes each

// ---------------------------------------------------------------------------------------------
// prepare

// eight states of a token in the order of the products' k index: 4 from n, 4 from n + 16
__device__ __forceinline__ void load_perm(const float * row, int n, int N, float (&v)[8]) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const int k = n + 16 * q;
        if (k + 3 < N) {
            const float4 f = load4(row + k);
            v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * q + i] = k + i < N ? row[k + i] : 0.0f;
        }
    }
}

constexpr int PREPARE_WORDS = 16 + 2 * Q;    // of LDS beside B's planes

template <int NK>
__device__ __forceinline__ void prepare_operands(const mm_plan & P, int c, int g, int s, char * lds) {
    const ssm_scan_launch & L = P.L;                           // lds: B's planes, blocks of 16 tokens by 32 states
    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int left = P.T - c * Q;             // tokens from the chunk's first on
    constexpr int PLANE = 4 * 1024 * NK;
    float * red = (float *) (lds + 2 * PLANE), * row_most = red + 16, * row_own = red + 16 + Q;
    const int64_t rec = ((int64_t) s * P.nc + c) * L.G + g;
    char * out = P.ws + P.planes + rec * rec_bytes<NK>();
    // a wave's 16 tokens of both, all states
    const int t = 16 * wave + lane % 16;
    const int64_t row = P.t0 + c * Q + min(t, left - 1);
    const float * cp = L.C + g * L.c_g + s * L.c_s + row * L.c_t, * bp = L.B + g * L.b_g + s * L.b_s + row * L.b_t;
    float v[2][NK][8], own = 0.0f;
#pragma unroll
    for (int q = 0; q < NK; q++) {
        load_perm(cp, 32 * q + 4 * (lane / 16), L.N, v[0][q]);
        load_perm(bp, 32 * q + 4 * (lane / 16), L.N, v[1][q]);
    }
#pragma unroll
    for (int o = 0; o < 2; o++) {
        uint32_t key = ~0u;
        float m = 0.0f;
#pragma unroll
        for (int q = 0; q < NK; q++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[o][q][i] = t < left ? v[o][q][i] : 0.0f;
                m = most_of(m, v[o][q][i]);
                key = min(key, least_key(v[o][q][i]));
            }
        }
        const float most = wave_max(m < INFINITY ? m : INFINITY), least = -wave_max(-least_value(key));
        if (lane == 0) {
            red[o * 4 + wave] = most;
            red[8 + o * 4 + wave] = least;
        }
    }
    // what a token's row adds to its own output, at most
#pragma unroll
    for (int q = 0; q < NK; q++) {
#pragma unroll
        for (int i = 0; i < 8; i++) own += fabsf(v[0][q][i] * v[1][q][i]);
    }
    own += __shfl_xor(own, 16, WAVE);
    own += __shfl_xor(own, 32, WAVE);
    if (lane < 16) row_own[t] = own;
    __syncthreads();
    int shift[2];
    bool fine = true;
    half8 ch[NK], cl[NK];
#pragma unroll
    for (int o = 0; o < 2; o++) {
        const float * r = red + o * 4;
        const float most = fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
        fine = fine && in_range(fminf(fminf(r[8], r[9]), fminf(r[10], r[11])), most);
        shift[o] = shift_of(most);
        const float sc = power_of(shift[o]);
#pragma unroll
        for (int q = 0; q < NK; q++) {
            half8 hi, lo;
            const int at = ((wave * NK + q) * 64 + lane) * 16;
            split8(v[o][q], sc, hi, lo);
            if (o == 0) {
                ch[q] = hi;
                cl[q] = lo;
                *(half8 *) (out + at) = hi;
                *(half8 *) (out + PLANE + at) = lo;
            } else {
                *(half8 *) (lds + at) = hi;
                *(half8 *) (lds + PLANE + at) = lo;
            }
        }
    }
    __syncthreads();
    // C_t . B_j of the wave's tokens, up to the diagonal
    const int gcol = lane % 16;
    float * G = (float *) (P.ws + P.gmat) + rec * G_WORDS + (gcol % 8 / 4) * 128 + (gcol / 8 * 16 + 4 * (lane / 16)) * 4 + gcol % 4;
    float top[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
    for (int jt = 0; jt <= wave; jt++) {
        float4v acc = { 0, 0, 0, 0 }, cross = { 0, 0, 0, 0 };
#pragma unroll
        for (int ks = 0; ks < NK; ks++) {
            const char * b = lds + ((jt * NK + ks) * 64 + lane) * 16;
            mfma3(ch[ks], cl[ks], *(const half8 *) b, *(const half8 *) (b + PLANE), acc, cross);
        }
        acc = joined(acc, cross);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float w = ldexpf(acc[i], -(shift[0] + shift[1]));
            G[(jt == wave ? wave : 4 + wave * (wave - 1) / 2 + jt) * 256 + 4 * i] = w;
            // no later token's
            if (jt < wave || gcol <= 4 * (lane / 16) + i) top[i] = fmaxf(top[i], fabsf(w) < INFINITY ? fabsf(w) : INFINITY);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        top[i] = group_max<16>(top[i]);
        if (gcol == 0) row_most[16 * wave + 4 * (lane / 16) + i] = top[i];
    }
    // B with the tokens as its k index: row n, eight tokens per lane
    const uint16_t * bh = (const uint16_t *) lds;
#pragma unroll
    for (int q = 0; q < NK; q++) {
        const int it = tid + 256 * q, nt = it / 128, ks = it / 64 % 2;
        const int n = 16 * nt + lane % 16, j0 = 32 * ks + 8 * (lane / 16), m = n % 32;
        const int at = ((j0 / 16 * NK + n / 32) * 64 + 16 * (m % 16 / 4) + j0 % 16) * 8 + m / 16 * 4 + m % 4;
        uint32_t w[2][4];
#pragma unroll
        for (int p = 0; p < 2; p++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t a = bh[at + 16 * i + p * (PLANE / 2)], b = bh[at + 16 * i + 8 + p * (PLANE / 2)];
                w[p][i] = a | b << 16;
            }
        }
#pragma unroll
        for (int p = 0; p < 2; p++) *(uint4v *) (out + (2 + p) * PLANE + it * 16) = uint4v{ w[p][0], w[p][1], w[p][2], w[p][3] };
    }
    __syncthreads();
    if (wave == 0) {
        const float row = row_most[lane], mine = row_own[lane];
        const float ratio = row < INFINITY ? (row > 0.0f && mine > 0.0f ? row / mine : 0.0f) : INFINITY;
        const float spread = fmaxf(wave_max(ratio), 1.0f), all = wave_max(row);
        float * sc = (float *) (P.ws + P.scales) + rec * SCALE_WORDS;
        sc[4 + lane] = row;
        if (lane == 0) {
            sc[0] = __int_as_float(shift[0]);
            sc[1] = __int_as_float(shift[1]);
            sc[2] = fine ? spread : INFINITY;
            sc[3] = all;
        }
    }
}

// 16 heads' running sums over a chunk: a wave per four heads, a lane per token
__device__ __forceinline__ void prepare_steps(const mm_plan & P, int c, int h0, int s, float * lds) {
    const ssm_scan_launch & L = P.L;
    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), left = P.T - c * Q;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int t = 16 * i + tid / 16, h = h0 + tid % 16;
        lds[t * 17 + tid % 16] = t < left && h < L.H ? L.dt[h + (P.t0 + c * Q + t) * L.dt_t + s * L.dt_s] : 0.0f;
    }
    float a[4];
#pragma unroll
    for (int k = 0; k < 4; k++) a[k] = L.A[min(h0 + 4 * wave + k, L.H - 1) * L.a_h];
    __syncthreads();
    float d[4];
    double sum[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        // a token past the last neither decays nor adds
        d[k] = lane < left ? softplus(lds[lane * 17 + 4 * wave + k]) : 0.0f;
        // 2^-1024 leaves nothing of a float and 2^1024 overflows, so a step beyond either is as good as that one; the
        // sums stay below 2^16 and the differences over other tokens keep their bits
        const double e = (double) d[k] * ((double) a[k] * 1.4426950408889634074);
        sum[k] = lane >= left ? 0.0 : e < -1024.0 ? -1024.0 : e > 1024.0 ? 1024.0 : e;   // a NaN stays one
    }
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double u = __shfl_up(sum[k], o, WAVE);
            sum[k] += lane >= o ? u : 0.0;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int h = h0 + 4 * wave + k;
        const double tile = __shfl(sum[k], lane | 15, WAVE) - sum[k];
        const double rest = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(sum[k]), 63),
                                             __builtin_amdgcn_readlane(__double2loint(sum[k]), 63)) - sum[k];
        const float hi = (float) sum[k], lo = fabsf(hi) < INFINITY ? (float) (sum[k] - (double) hi) : 0.0f;
        const float rh = (float) rest, rl = fabsf(rh) < INFINITY ? (float) (rest - (double) rh) : 0.0f;
        const float th = (float) tile, tl = fabsf(th) < INFINITY ? (float) (tile - (double) th) : 0.0f;
        if (h >= L.H) break;
        float * o = (float *) (P.ws + P.steps) + (((int64_t) s * P.nc + c) * L.H + h) * STEP_WORDS + lane;
        o[0] = exp2_hw(hi) * fmaf(lo, LN2, 1.0f);
        o[Q] = exp2_hw(rh) * fmaf(rl, LN2, 1.0f);
        o[2 * Q] = d[k];
        o[3 * Q] = hi;
        o[4 * Q] = lo;
        o[5 * Q] = exp2_hw(th) * fmaf(tl, LN2, 1.0f);
    }
}

template <int NK>
__global__ __launch_bounds__(256) void ssm_prepare_kernel(mm_plan P) {
    extern __shared__ __align__(16) char lds[];
    const int y = blockIdx.y;
    if (y < P.L.G) prepare_operands<NK>(P, blockIdx.x, y, blockIdx.z, lds);
    else prepare_steps(P, blockIdx.x, (y - P.L.G) * 16, blockIdx.z, (float *) lds);
}

// ---------------------------------------------------------------------------------------------
// scan

constexpr int WAVES = 8;                                       // per workgroup, each with 16 channels of a head
constexpr int THREADS = WAVES * WAVE;
// B's buffers: the next chunk's beside this one's, where they fit 160 KiB with C's and the matrices
constexpr int b_slots(int nk) { return nk == 8 ? 1 : 2; }

// An offset that is formed where it is used: kept for the whole loop, with the fifteen that follow from it,
// it would take the registers that the loop is short of.
__device__ __forceinline__ uint32_t here(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ int here_s(int x) {
    asm volatile("" : "+s"(x));
    return x;
}
// likewise the arguments, read again from where the launch put them
typedef const __attribute__((address_space(4))) mm_plan * plan_ptr;
__device__ __forceinline__ plan_ptr plan_here() {
    plan_ptr p = (plan_ptr) __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// states n .. n + 3 of a row of N
__device__ __forceinline__ float4v states4(const float * row, int n, int N) {
    float4v v;
    if (n + 3 < N) {
        const float4 f = load4(row + n);
        v = float4v{ f.x, f.y, f.z, f.w };
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = n + i < N ? row[n + i] : 0.0f;
    }
    return v;
}

// the largest value of a column's four lanes
__device__ __forceinline__ float column_max(float m) {
    m = fmaxf(m, __shfl_xor(m, 16, WAVE));
    return fmaxf(m, __shfl_xor(m, 32, WAVE));
}

// NK: steps of 32 states; OUT: outputs and final states, else the segment's state from nothing.
// What a chunk reads is loaded into registers while the chunk before it is computed: its operands'
// planes (EARLY; on to LDS at the chunk's end: C's over the last one's, B's beside it), the inputs, C_t . B_j and the
// heads' exponentials. Two barriers a chunk: LDS is written; C is read and the matrices are written.
template <int NK, bool OUT>
__global__ __launch_bounds__(THREADS, 2) void ssm_scan_mm_kernel(mm_plan P) {
    extern __shared__ __align__(16) char lds[];
    const ssm_scan_launch & L = P.L;
    constexpr int PLANE = 4 * 1024 * NK, OPERAND = 2 * PLANE, STAGE = OPERAND / (THREADS * 16), SLOTS = b_slots(NK);
    static_assert(STAGE >= 1, "a thread moves whole 16-byte pieces");
    char * cbuf = lds;                                         // C's planes
    char * bbuf = lds + (OUT ? OPERAND : 0);                   // B's, of this chunk and the next
    float * steps = (float *) (bbuf + SLOTS * OPERAND);        // per head, of this chunk and the next
    char * mats = (char *) (steps + 2 * P.hw * STEP_WORDS);    // per head: the two planes of (C_t . B_j) exp(c_t - c_j)
    int * row_shift = (int *) (mats + P.hw * 2 * M_BYTES);     // per head: the exponents of their rows' powers of two
    // the wave's number as the scalar that it is: what depends on it alone stays out of the vector registers
    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), col = lane % 16, grp = lane / 16;

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
    if (!OUT && sg == P.n_seg - 1) return;                     // nobody starts from the last segment's state
    const int per = L.H / L.G;
    const int hl = P.p_blocks > 1 ? 0 : wave / P.slices, slice = P.p_blocks > 1 ? m % P.p_blocks * WAVES + wave : wave % P.slices;
    const int hb = m / P.p_blocks * P.hw;
    const int heads = min(P.hw, per - hb);                     // heads of this workgroup
    const bool active = hl < heads && slice < P.slices;
    const int h = g * per + hb + (active ? hl : 0);
    const int c0 = sg * P.seg, c1 = min(P.nc, c0 + P.seg);
    const bool pok = active && 16 * slice + col < L.P;
    const int pch = min(16 * slice + col, L.P - 1);

    // the wave's states: tile nt, i: state 16 nt + 4 grp + i of channel 16 slice + col
    float4v S[2 * NK];
#pragma unroll
    for (int nt = 0; nt < 2 * NK; nt++) S[nt] = float4v{ 0, 0, 0, 0 };
    // segments' states: in the order the lanes hold them
    auto part_at = [&](int k) {
        return (float4v *) (P.ws + P.parts) + ((((int64_t) s * P.n_seg + k) * L.H + h) * P.slices + slice) * (2 * NK * WAVE) + lane;
    };
    if (OUT && active) {
        int64_t row = s;
        if (P.pooled) {
            row = L.ids[s * L.ids_s];
            row = row < 0 ? 0 : row >= L.pool ? L.pool - 1 : row;
        }
        const float * s0 = P.s0 + (P.pooled ? pch * L.s_p + h * L.s_h + row * L.s_row
                                            : (int64_t) L.N * (pch + (int64_t) L.P * (h + (int64_t) L.H * s)));
#pragma unroll
        for (int nt = 0; nt < 2 * NK; nt++) S[nt] = states4(s0, 16 * nt + 4 * grp, L.N);
        // two segments' loads in flight
        for (int k = 0; k < sg; k += 2) {
            const int k1 = min(k + 1, sg - 1);
            const float * dp = (const float *) (P.ws + P.decays) + (int64_t) s * P.n_seg * L.H + h;
            const float d0 = dp[(int64_t) k * L.H], d1 = dp[(int64_t) k1 * L.H];
            const float4v * q0 = part_at(k), * q1 = part_at(k1);
            float4v f0[2 * NK], f1[2 * NK];
#pragma unroll
            for (int nt = 0; nt < 2 * NK; nt++) {
                f0[nt] = q0[nt * WAVE];
                f1[nt] = q1[nt * WAVE];
            }
#pragma unroll
            for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) S[nt][i] = fmaf(S[nt][i], d0, f0[nt][i]);
            }
            if (k + 1 < sg) {
#pragma unroll
                for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) S[nt][i] = fmaf(S[nt][i], d1, f1[nt][i]);
                }
            }
        }
    }

    // what the next chunk reads
    // The operands' planes a chunk ahead too, or only once the chunk before is done: the registers that hold them are
    // those that outputs of 256 states lack: 4096 tokens of 128 x 64 x 256 464 us late and 702 ahead, 3 x 586 of 30 x
    // 128 x 256 110 and 152. 128 states don't care (196 and 198 us; 77 both at 1402 of 64 x 80), 64 and fewer have
    // the registers.
    constexpr bool EARLY = !OUT || NK < 4;
    uint4v stage_c[OUT && EARLY ? STAGE : 1], stage_b[EARLY ? STAGE : 1];
    float4v gg[2][2];
    float gr[2], x[2][8], sc_next[4], st_next[(4 * STEP_WORDS + THREADS - 1) / THREADS];
    // The matrices' tiles of 16 x 16, two per wave and turn: a head has four on the diagonal, which need an
    // exponential per element, and six below it, where exp(c_t - c_j) is exp(c_t - c_b) exp(c_b - c_j), b the last
    // of the tile's columns: one exponential per row beside prepared ones. A turn is (head, pair of tiles); the
    // diagonal ones come first, and a second turn goes to the waves that had the cheaper first.
    const int turns = 5 * heads;
    struct tile_place { int k, tt, jt; };
    auto place = [&](int turn) {
        tile_place w;
        if (turn < 2 * heads) {
            w.k = turn / 2;
            w.tt = w.jt = turn % 2 * 2 + lane / 32;
        } else {
            const int q = turn - 2 * heads, i = q % 3 * 2 + lane / 32;
            w.k = q / 3;
            w.tt = i < 1 ? 1 : i < 3 ? 2 : 3;
            w.jt = i < 1 ? 0 : i < 3 ? i - 1 : i - 3;
        }
        return w;
    };
    auto turn_of = [&](int r) { return WAVES * r + (wave + WAVES / 2 * r) % WAVES; };
    // the lane's row of a tile and its eight columns
    const int tr = lane % 16, th = lane / 16 % 2;
    auto load_g = [&](const char * G, const char * scales, int turn, float4v (&v)[2], float & most) {
        most = ((const float *) scales)[4 + 16 * place(turn).tt + tr];
        const int pair = turn < 2 * heads ? turn % 2 : 2 + (turn - 2 * heads) % 3;
        const uint32_t at = here(lane / 32 * 1024 + lane % 32 * 16);
        v[0] = *(const float4v *) (G + pair * 2048 + at);
        v[1] = *(const float4v *) (G + pair * 2048 + 512 + at);
    };
    if (OUT) {
        // the tiles above the diagonal that the products read: blocks 0 and 3, columns 16 to 31
        for (int i = tid; i < heads * 2 * 2 * 32; i += THREADS)
            *(uint4v *) (mats + i / 64 * M_BYTES + (i / 32 % 2 ? 3 : 0) * 1024 + (32 + i % 32) * 16) = uint4v{ 0, 0, 0, 0 };
    }
    // where the next chunk's are, and how far on each lies in the chunk after
    const char * at_planes, * at_steps, * at_scales, * at_g, * at_x;
    {
        const int64_t rec = ((int64_t) s * P.nc + c0) * L.G + g;
        at_planes = P.ws + P.planes + rec * rec_bytes<NK>();
        at_scales = P.ws + P.scales + rec * (SCALE_WORDS * 4);
        at_g = P.ws + P.gmat + rec * (G_WORDS * 4);
        at_steps = P.ws + P.steps + (((int64_t) s * P.nc + c0) * L.H + g * per + hb) * (STEP_WORDS * 4);
        at_x = (const char *) (L.x + h * L.x_h + s * L.x_s + (P.t0 + c0 * Q) * L.x_t);
    }
    const int64_t x_on = Q * 4 * L.x_t, steps_on = (int64_t) L.H * (STEP_WORDS * 4);
    auto fetch = [&](int c) {
        const int left = P.T - c * Q;
        if constexpr (EARLY) {
            const uint32_t piece = here(tid * 16);
#pragma unroll
            for (int q = 0; q < STAGE; q++) {
                if (OUT) stage_c[q] = *(const uint4v *) (at_planes + q * THREADS * 16 + piece);
                stage_b[q] = *(const uint4v *) (at_planes + OPERAND + q * THREADS * 16 + piece);
            }
        }
#pragma unroll
        for (int q = 0; q < (4 * STEP_WORDS + THREADS - 1) / THREADS; q++)
            st_next[q] = *(const float *) (at_steps + 4 * (uint32_t) min(tid + q * THREADS, heads * STEP_WORDS - 1));
#pragma unroll
        for (int i = 0; i < 4; i++) sc_next[i] = ((const float *) at_scales)[i];
        if (OUT) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                if (turn_of(r) < turns) load_g(at_g, at_scales, turn_of(r), gg[r], gr[r]);
            }
        }
        // token 32 ks + 8 grp + i of the wave's channels; past the last token it is the last again, and cleared
        const uint32_t row = 4 * (uint32_t) L.x_t;
        if (left >= Q) {
            uint32_t at = here(8 * grp * row + 4 * (uint32_t) pch);
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                for (int i = 0; i < 8; i++, at += row) x[ks][i] = *(const float *) (at_x + at);
                at += 24 * row;
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[ks][i] = *(const float *) (at_x + (min(32 * ks + 8 * grp + i, left - 1) * row + 4 * (uint32_t) pch));
            }
        }
        at_planes += L.G * rec_bytes<NK>();
        at_scales += L.G * (SCALE_WORDS * 4);
        at_g += L.G * (G_WORDS * 4);
        at_steps += steps_on;
        at_x += x_on;
    };
    // and on to LDS
    auto put = [&](int turn) {
        if constexpr (EARLY) {
#pragma unroll
            for (int q = 0; q < STAGE; q++) {
                if (OUT) *(uint4v *) (cbuf + (tid + q * THREADS) * 16) = stage_c[q];
                *(uint4v *) (bbuf + turn % SLOTS * OPERAND + (tid + q * THREADS) * 16) = stage_b[q];
            }
        } else {
            // C's planes, then B's, in the record
            static_assert(2 * STAGE % 8 == 0, "eight pieces at a time");
            const char * planes = at_planes - L.G * rec_bytes<NK>() + tid * 16;
            char * to[2] = { cbuf + tid * 16, bbuf + turn % SLOTS * OPERAND - OPERAND + tid * 16 };
#pragma unroll
            for (int q0 = 0; q0 < 2 * STAGE; q0 += 8) {
                uint4v piece[8];
#pragma unroll
                for (int q = 0; q < 8; q++) piece[q] = *(const uint4v *) (planes + (q0 + q) * THREADS * 16);
#pragma unroll
                for (int q = 0; q < 8; q++) *(uint4v *) (to[q0 + q >= STAGE] + (q0 + q) * THREADS * 16) = piece[q];
            }
        }
#pragma unroll
        for (int q = 0; q < (4 * STEP_WORDS + THREADS - 1) / THREADS; q++) {
            const int i = tid + q * THREADS;
            if (i < heads * STEP_WORDS) steps[turn * P.hw * STEP_WORDS + i] = st_next[q];
        }
    };

    // The chunk by its recurrence, in float32 throughout: for operands whose halves would lose a value beside a larger
    // one. 16 states after another go through all tokens, a lane's four of its channel, whose output so far stays in
    // memory; the next ones take their registers' place, so that this takes one loop's code and few registers beside
    // the main path's. Where every chunk comes here, 4096 tokens of 128 x 64 x 128 take 8.3 ms, as the kernel for
    // any operands does.
    auto by_tokens = [&](int c, const float * my) {
        const plan_ptr K = plan_here();
        const uint32_t n0 = here(4 * grp), p0 = here(pch);
        const int h1 = here_s(h), s1 = here_s(s), g1 = here_s(g);
        const float a = K->L.A[h1 * K->L.a_h] * LOG2E;
        const int64_t row = K->t0 + c * Q;
        const int n_t = min(Q, K->T - c * Q);
#pragma unroll 1
        for (int nt = 0; nt < 2 * NK; nt++) {
            float4v st = S[0];
            const float * xp = K->L.x + h1 * K->L.x_h + s1 * K->L.x_s + row * K->L.x_t;
            const float * bp = K->L.B + g1 * K->L.b_g + s1 * K->L.b_s + row * K->L.b_t + 16 * nt;
            const float * cp = K->L.C + g1 * K->L.c_g + s1 * K->L.c_s + row * K->L.c_t + 16 * nt;
            float * y = K->L.y + (int64_t) K->L.P * (h1 + (int64_t) K->L.H * (row + K->L.T * s1));
            const int left = K->L.N - 16 * nt;
#pragma unroll 1
            for (int t = 0; t < n_t && left > 0; t++, xp += K->L.x_t, bp += K->L.b_t, cp += K->L.c_t, y += (int64_t) K->L.P * K->L.H) {
                const float d = my[2 * Q + t], e = exp2_hw(d * a), dx = d * xp[p0];
                const float4v b = states4(bp, (int) n0, left), f = OUT ? states4(cp, (int) n0, left) : b;
#pragma unroll
                for (int i = 0; i < 4; i++) st[i] = fmaf(st[i], e, dx * b[i]);
                if (OUT) {
                    float v = fmaf(st[0], f[0], st[1] * f[1]) + fmaf(st[2], f[2], st[3] * f[3]);
                    v += __shfl_xor(v, 16, WAVE);
                    v += __shfl_xor(v, 32, WAVE);
                    if (pok && grp == 0) y[p0] = nt == 0 ? v : y[p0] + v;
                }
            }
#pragma unroll
            for (int i = 0; i + 1 < 2 * NK; i++) S[i] = S[i + 1];
            S[2 * NK - 1] = st;
        }
    };

    float decay = 1.0f;                                        // of the segment so far
    fetch(c0);
    put(0);
    for (int c = c0; c < c1; c++) {
        const int turn = (c - c0) & 1, left = P.T - c * Q;
        const bool whole = left >= Q && 16 * (slice + 1) <= L.P;   // every lane's tokens and channels
        const int shift_c = __float_as_int(sc_next[0]), shift_b = __float_as_int(sc_next[1]);
        const float spread = sc_next[2], gmost = sc_next[3];
        const char * B = bbuf + turn % SLOTS * OPERAND + lane * 16;
        __syncthreads();                                       // this chunk's LDS is written
        const float * head_steps = steps + turn * P.hw * STEP_WORDS, * my = head_steps + (active ? hl : 0) * STEP_WORDS;
        const float e_last = my[Q - 1];
        if (OUT) {
            // (C_t . B_j) exp(c_t - c_j) below the diagonal, split, in the order of the A operand
#pragma unroll 1
            for (int r = 0; turn_of(r) < turns; r++) {
                const int now = turn_of(r);
                const tile_place w = place(now);
                if (r == 1) {
                    gg[0][0] = gg[1][0];
                    gg[0][1] = gg[1][1];
                    gr[0] = gr[1];
                } else if (r > 1) {
                    const int64_t rec = ((int64_t) s * P.nc + c) * L.G + g;
                    load_g(P.ws + P.gmat + rec * (G_WORDS * 4), P.ws + P.scales + rec * (SCALE_WORDS * 4), now, gg[0], gr[0]);
                }
                const float g8[8] = { gg[0][0][0], gg[0][0][1], gg[0][0][2], gg[0][0][3], gg[0][1][0], gg[0][1][1], gg[0][1][2], gg[0][1][3] };
                const float * st = head_steps + w.k * STEP_WORDS;
                const int t = 16 * w.tt + tr, j0 = 16 * w.jt + 8 * th;
                // no element of the row is larger, and what later tokens hold does not matter to it
                const int shift = shift_of(gr[0] * fmaxf(1.0f, st[t]));
                float v[8];
                if (now < 2 * heads) {
                    if (th == 0) row_shift[w.k * Q + t] = shift;
                    const float ht = st[3 * Q + t], lt = st[4 * Q + t];
                    const float4 h0 = *(const float4 *) (st + 3 * Q + j0), h1 = *(const float4 *) (st + 3 * Q + j0 + 4);
                    const float4 l0 = *(const float4 *) (st + 4 * Q + j0), l1 = *(const float4 *) (st + 4 * Q + j0 + 4);
                    const float hh[8] = { h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w };
                    const float ll[8] = { l0.x, l0.y, l0.z, l0.w, l1.x, l1.y, l1.z, l1.w };
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float e = g8[i] * exp2_hw((ht - hh[i]) + (lt - ll[i]));
                        v[i] = 8 * th + i <= tr ? e : 0.0f;
                    }
                } else {
                    const int b = 16 * w.jt + 15;
                    const float row = exp2_hw((st[3 * Q + t] - st[3 * Q + b]) + (st[4 * Q + t] - st[4 * Q + b]));
                    const float4 f0 = *(const float4 *) (st + 5 * Q + j0), f1 = *(const float4 *) (st + 5 * Q + j0 + 4);
                    const float ff[8] = { f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w };
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = g8[i] * ff[i] * row;
                }
                half8 hi, lo;
                split8(v, power_of(shift), hi, lo);
                char * o = mats + w.k * 2 * M_BYTES + (w.tt < 2 ? w.tt : 2 * w.tt - 2 + w.jt / 2) * 1024 + (tr + 16 * (w.jt % 2 * 2 + th)) * 16;
                *(half8 *) o = hi;
                *(half8 *) (o + M_BYTES) = lo;
            }
        }
        // X = d x, cleared of tokens past the last
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const float4 d0 = *(const float4 *) (my + 2 * Q + 32 * ks + 8 * grp), d1 = *(const float4 *) (my + 2 * Q + 32 * ks + 8 * grp + 4);
            const float dd[8] = { d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w };
#pragma unroll
            for (int i = 0; i < 8; i++) x[ks][i] *= dd[i];
        }
        if (!whole) {
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[ks][i] = pok && 32 * ks + 8 * grp + i < left ? x[ks][i] : 0.0f;
            }
        }
        // whether halves do for the wave's channels
        float own = 0.0f;
        uint32_t key = ~0u;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                own = most_of(own, x[ks][i]);
                key = min(key, least_key(x[ks][i]));
            }
        }
        const float most = column_max(own < INFINITY ? own : INFINITY);
        const float growth = fmaxf(1.0f, e_last);              // a decay above 1 grows all through a chunk
        bool fine = in_range(least_value(key), most * (spread * growth)) && gmost * growth < INFINITY;
        half8 xh[2], xl[2];
        if (OUT) {
            // C_t S
            float4v acc[4];
            int shift_s = 0;
            float stop = 0.0f;
            if (active) {
                uint32_t skey = ~0u;
#pragma unroll
                for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        stop = fmaxf(stop, fabsf(S[nt][i]));
                        skey = min(skey, least_key(S[nt][i]));
                    }
                }
                stop = column_max(stop);
                if (__any(!(stop < INFINITY))) {
                    // a state that is not finite: its channel's outputs are not either, and no other's are touched
                    stop = 0.0f;
#pragma unroll
                    for (int nt = 0; nt < 2 * NK; nt++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) stop = fmaxf(stop, finite_abs(S[nt][i]));
                    }
                    stop = column_max(stop);
                }
                fine = fine && in_range(least_value(skey), stop);
            }
            fine = !__any(!fine);
            if (active && fine) {
                shift_s = shift_of(stop);
                const float ss = power_of(shift_s);
                float4v cross[4];
#pragma unroll
                for (int tt = 0; tt < 4; tt++) acc[tt] = cross[tt] = float4v{ 0, 0, 0, 0 };
#pragma unroll
                for (int ks = 0; ks < NK; ks++) {
                    half8 ah[4], al[4], bh, bl;
#pragma unroll
                    for (int tt = 0; tt < 4; tt++) {
                        const char * a = cbuf + ((tt * NK + ks) * 64 + lane) * 16;
                        ah[tt] = *(const half8 *) a;
                        al[tt] = *(const half8 *) (a + PLANE);
                    }
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = S[2 * ks + i / 4][i % 4];
                    split8(v, ss, bh, bl);
#pragma unroll
                    for (int tt = 0; tt < 4; tt++) cross[tt] = mfma(al[tt], bh, cross[tt]);
#pragma unroll
                    for (int tt = 0; tt < 4; tt++) acc[tt] = mfma(ah[tt], bh, acc[tt]);
#pragma unroll
                    for (int tt = 0; tt < 4; tt++) cross[tt] = mfma(ah[tt], bl, cross[tt]);
                }
#pragma unroll
                for (int tt = 0; tt < 4; tt++) acc[tt] = joined(acc[tt], cross[tt]);
            }
            __syncthreads();                                   // C is read, the matrices are written
            if (active && fine) {
                const char * mine = mats + hl * 2 * M_BYTES + lane * 16;
                const int shift_x = shift_of(most);
                float4v sum[4];
#pragma unroll
                for (int ks = 0; ks < 2; ks++) split8(x[ks], power_of(shift_x), xh[ks], xl[ks]);
#pragma unroll
                for (int t2 = 0; t2 < 4; t2 += 2) {
                    // tiles 0 and 1 end within the first 32 tokens
                    half8 ah[2][2], al[2][2];
#pragma unroll
                    for (int ks = 0; ks <= t2 / 2; ks++) {
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            const char * a = mine + (t2 == 0 ? q : 2 + 2 * q + ks) * 1024;
                            ah[q][ks] = *(const half8 *) a;
                            al[q][ks] = *(const half8 *) (a + M_BYTES);
                        }
                    }
                    float4v own[2], cross[2];
#pragma unroll
                    for (int q = 0; q < 2; q++) own[q] = cross[q] = float4v{ 0, 0, 0, 0 };
#pragma unroll
                    for (int ks = 0; ks <= t2 / 2; ks++) {
#pragma unroll
                        for (int q = 0; q < 2; q++) mfma3(ah[q][ks], al[q][ks], xh[ks], xl[ks], own[q], cross[q]);
                    }
#pragma unroll
                    for (int q = 0; q < 2; q++) sum[t2 + q] = joined(own[q], cross[q]);
                }
#pragma unroll
                for (int tt = 0; tt < 4; tt++) {
                    const float4 e4 = *(const float4 *) (my + 16 * tt + 4 * grp);
                    const int4 r4 = *(const int4 *) (row_shift + (active ? hl : 0) * Q + 16 * tt + 4 * grp);
                    const float e[4] = { e4.x, e4.y, e4.z, e4.w };
                    const int rs[4] = { r4.x, r4.y, r4.z, r4.w };
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[tt][i] = ldexpf(acc[tt][i] * e[i], -(shift_s + shift_c)) + ldexpf(sum[tt][i], -(shift_x + rs[i]));
                }
                char * y = (char *) (L.y + h * L.P + (int64_t) L.P * L.H * (P.t0 + c * Q + L.T * s));
                const uint32_t row = 4 * (uint32_t) L.P * (uint32_t) L.H;
                uint32_t at = here(4 * grp * row + 4 * (uint32_t) pch);
#pragma unroll
                for (int tt = 0; tt < 4; tt++) {
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 4; i++, at += row) *(float *) (y + at) = acc[tt][i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++, at += row) {
                            if (pok && 16 * tt + 4 * grp + i < left) *(float *) (y + at) = acc[tt][i];
                        }
                    }
                    at += 12 * row;
                }
            }
        } else {
            fine = !__any(!fine);
        }
        // the state at the chunk's end
        int shift_u = 0;
        if (active && fine) {
            float v[2][8], wmost = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const float4 w0 = *(const float4 *) (my + Q + 32 * ks + 8 * grp), w1 = *(const float4 *) (my + Q + 32 * ks + 8 * grp + 4);
                const float ww[8] = { w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w };
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    v[ks][i] = x[ks][i] * ww[i];
                    wmost = fmaxf(wmost, fabsf(v[ks][i]));
                }
            }
            // by the largest that the decays leave, not by one that they have taken away
            const int shift_w = shift_of(column_max(wmost));
            shift_u = shift_w + shift_b;
#pragma unroll
            for (int ks = 0; ks < 2; ks++) split8(v[ks], power_of(shift_w), xh[ks], xl[ks]);
        }
        if (active && !fine) by_tokens(c, my);
        if (c + 1 < c1) fetch(c + 1);
        if (active && fine) {
#pragma unroll
            for (int n0 = 0; n0 < 2 * NK; n0 += 2) {
                float4v sum[2], cross[2];
                half8 ah[2][2], al[2][2];
#pragma unroll
                for (int q = 0; q < 2; q++) {
#pragma unroll
                    for (int ks = 0; ks < 2; ks++) {
                        ah[q][ks] = *(const half8 *) (B + ((n0 + q) * 2 + ks) * 1024);
                        al[q][ks] = *(const half8 *) (B + ((n0 + q) * 2 + ks) * 1024 + PLANE);
                    }
                }
#pragma unroll
                for (int q = 0; q < 2; q++) sum[q] = cross[q] = float4v{ 0, 0, 0, 0 };
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                    for (int q = 0; q < 2; q++) mfma3(ah[q][ks], al[q][ks], xh[ks], xl[ks], sum[q], cross[q]);
                }
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    sum[q] = joined(sum[q], cross[q]);
#pragma unroll
                    for (int i = 0; i < 4; i++) S[n0 + q][i] = fmaf(S[n0 + q][i], e_last, ldexpf(sum[q][i], -shift_u));
                }
            }
        }
        decay *= e_last;
        if (SLOTS == 1) __syncthreads();                       // B is read
        if (c + 1 < c1) put(turn ^ 1);
    }
    if (!active) return;
    if (!OUT) {
        if (lane == 0 && slice == 0) ((float *) (P.ws + P.decays))[((int64_t) s * P.n_seg + sg) * L.H + h] = decay;
        float4v * q = part_at(sg);
#pragma unroll
        for (int nt = 0; nt < 2 * NK; nt++) q[nt * WAVE] = S[nt];
    } else if (c1 == P.nc && pok) {
        float * s1 = P.s1 + (int64_t) L.N * (pch + (int64_t) L.P * (h + (int64_t) L.H * s));
#pragma unroll
        for (int nt = 0; nt < 2 * NK; nt++) {
            const int n = 16 * nt + 4 * grp;
            if (n + 3 < L.N) {
                store4(s1 + n, make_float4(S[nt][0], S[nt][1], S[nt][2], S[nt][3]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (n + i < L.N) s1[n + i] = S[nt][i];
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------

int steps_of(int N) { return N <= 32 ? 1 : N <= 64 ? 2 : N <= 128 ? 4 : 8; }

struct mm_sizes {
    int     nk, slices, hw, head_blocks, p_blocks;
    int64_t seqs, chunks, block, n_seg, seg;   // sequences at once, chunks in all and per block of tokens, segments of a block
    int64_t planes, gmat, scales, steps, parts, decays, state, total;
};

// prepared operands (with the rounding of their offsets) and segments' states of at most so many bytes: sequences and
// tokens go through in blocks
constexpr int64_t MOST_OPERANDS = ((int64_t) 64 << 20) - 4096, MOST_PARTS = (int64_t) 32 << 20;

// those of one chunk of one sequence
int64_t chunk_bytes(const ssm_scan_launch & L) {
    return L.G * ((int64_t) steps_of(L.N) * 16384 + (G_WORDS + SCALE_WORDS) * 4) + (int64_t) L.H * STEP_WORDS * 4;
}

mm_sizes mm_size(const ssm_scan_launch & L) {
    mm_sizes z;
    z.nk = steps_of(L.N);
    z.slices = (L.P + 15) / 16;
    z.p_blocks = (z.slices + WAVES - 1) / WAVES;
    // heads of a workgroup: as its waves allow, and their matrices' 15 KiB each beside the operands
    z.hw = z.p_blocks > 1 ? 1 : std::min(WAVES / z.slices, z.nk == 8 ? 2 : 4);
    z.head_blocks = (L.H / L.G + z.hw - 1) / z.hw;
    z.chunks = (L.T + Q - 1) / Q;
    // as many sequences at once as one chunk of each leaves room for, in even passes
    const int64_t fit = std::max<int64_t>(1, std::min<int64_t>(L.S, MOST_OPERANDS / chunk_bytes(L))), passes = (L.S + fit - 1) / fit;
    z.seqs = (L.S + passes - 1) / passes;
    z.block = std::max<int64_t>(1, std::min<int64_t>({ z.chunks, MOST_OPERANDS / (z.seqs * chunk_bytes(L)), 65535 }));
    // segments until every CU has a workgroup, of one chunk if need be (333 tokens of 24 heads: 41 us with two
    // chunks at least, 37 with one)
    const int64_t base = z.seqs * L.G * z.head_blocks * z.p_blocks;
    const int64_t part = z.seqs * L.H * (int64_t) z.slices * (2 * z.nk * WAVE * 16) + z.seqs * L.H * 4;
    z.n_seg = std::max<int64_t>(1, std::min<int64_t>({ 256 / base, z.block, MOST_PARTS / part }));
    z.seg = (z.block + z.n_seg - 1) / z.n_seg;
    z.n_seg = (z.block + z.seg - 1) / z.seg;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
    z.planes = take(z.seqs * z.block * L.G * (int64_t) z.nk * 16384);
    z.gmat = take(z.seqs * z.block * L.G * G_WORDS * 4);
    z.scales = take(z.seqs * z.block * L.G * SCALE_WORDS * 4);
    z.steps = take(z.seqs * z.block * (int64_t) L.H * STEP_WORDS * 4);
    z.parts = take(z.n_seg > 1 ? z.seqs * z.n_seg * (int64_t) L.H * z.slices * 2 * z.nk * WAVE * 16 : 0);
    z.decays = take(z.n_seg > 1 ? z.seqs * z.n_seg * (int64_t) L.H * 4 : 0);
    // states between blocks of tokens, one read while the next is written
    z.state = take(z.block < z.chunks ? 2 * z.seqs * (int64_t) L.N * L.P * L.H * 4 : 0);
    z.total = at;
    return z;
}

template <int NK>
void launch_mm(const ssm_scan_launch & L, const mm_sizes & z, void * ws, hipStream_t st) {
    mm_plan P{};
    P.L = L;
    P.ws = (char *) ws;
    P.planes = z.planes; P.gmat = z.gmat; P.scales = z.scales; P.steps = z.steps; P.parts = z.parts; P.decays = z.decays;
    P.hw = z.hw; P.slices = z.slices; P.head_blocks = z.head_blocks; P.p_blocks = z.p_blocks;
    constexpr int OPERAND = NK * 8192;
    auto lds_of = [](int hw, bool out) {
        return (size_t) OPERAND * (b_slots(NK) + (out ? 1 : 0)) + (size_t) hw * (2 * STEP_WORDS * 4 + (out ? 2 * M_BYTES + Q * 4 : 0));
    };
    static std::atomic<uint64_t> lds_set{ 0 };                 // devices, a bit each
    int device = 0;
    HIP_CHECK(hipGetDevice(&device));
    if (device > 63 || !(lds_set.load(std::memory_order_relaxed) >> device & 1)) {
        const int hw = NK == 8 ? 2 : 4;
        HIP_CHECK(hipFuncSetAttribute((const void *) ssm_prepare_kernel<NK>, hipFuncAttributeMaxDynamicSharedMemorySize, OPERAND + PREPARE_WORDS * 4));
        HIP_CHECK(hipFuncSetAttribute((const void *) ssm_scan_mm_kernel<NK, false>, hipFuncAttributeMaxDynamicSharedMemorySize, (int) lds_of(hw, false)));
        HIP_CHECK(hipFuncSetAttribute((const void *) ssm_scan_mm_kernel<NK, true>, hipFuncAttributeMaxDynamicSharedMemorySize, (int) lds_of(hw, true)));
        if (device < 64) lds_set.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    float * hold = (float *) ((char *) ws + z.state);
    const int64_t states = z.seqs * (int64_t) L.N * L.P * L.H;
    for (int64_t c = 0, turn = 0; c < z.chunks; c += z.block, turn ^= 1) {
        P.nc = (int) std::min(z.block, z.chunks - c);
        P.t0 = c * Q;
        P.T = (int) std::min<int64_t>(L.T - P.t0, (int64_t) P.nc * Q);
        P.seg = (int) z.seg;
        P.n_seg = (P.nc + P.seg - 1) / P.seg;
        P.pooled = c == 0;
        P.s0 = c == 0 ? L.s : hold + (turn ^ 1) * states;
        P.s1 = c + z.block < z.chunks ? hold + turn * states : L.s_out;
        launch(ssm_prepare_kernel<NK>, dim3((unsigned) P.nc, (unsigned) (L.G + (L.H + 15) / 16), (unsigned) L.S), dim3(256),
               std::max<size_t>(OPERAND + PREPARE_WORDS * 4, Q * 17 * 4), st, P);
        const dim3 grid((unsigned) (L.S * L.G * P.n_seg * z.head_blocks * z.p_blocks));
        if (P.n_seg > 1) launch(ssm_scan_mm_kernel<NK, false>, grid, dim3(THREADS), lds_of(z.hw, false), st, P);
        launch(ssm_scan_mm_kernel<NK, true>, grid, dim3(THREADS), lds_of(z.hw, true), st, P);
    }
}

// Up to so many tokens the recurrence itself is faster: products need an operand's preparation and a chunk's latency, 14
// us with 32 states, 17 with 64, 22 with 128 and 38 with 256, and a step takes 0.5 to 0.7 us (24 heads of 64 channels and 32
// states: 20 tokens 13.1 us by steps and 14.1 by products, 22 14.2 both; 80 heads of 64 states 24 15.9 and 17.0, 28 18.0
// and 17.1; of 128 28 20.3 and 22.1, 32 22.5 and 22.3; of 256 44 36.4 and 38.0, 48 39.1 and 37.6). Where channels fill the
// chip a step takes longer and the latency doesn't count, whatever the states: 163840 channels of 128 states 18 tokens
// 94.5 and 97.8, 20 99.8 and 97.7; of 64 16 52 and 65 with 2.4 a step; 81920 of 256 26 127.5 and 99.9 with 4.
int step_tokens(const ssm_scan_launch & L) {
    const int few = L.N <= 32 ? 21 : L.N <= 64 ? 26 : L.N <= 128 ? 31 : 46;
    return L.S * (int64_t) L.H * L.P > 65536 ? std::min(few, 19) : few;
}

} // namespace

bool ssm_scan_mm_takes(const ssm_scan_launch & L) {
    // the grids' limits: one dimension each for the sequences and for groups and heads, 2^32 threads in all
    return L.a_scalar && L.T > step_tokens(L) && L.S <= 65535 && L.G + (L.H + 15) / 16 <= 65535 &&
           L.S * (int64_t) L.H * ((L.P + 127) / 128) < 1 << 22 &&
           // one sequence's chunk fits the scratch (512 groups of 256 states do not)
           chunk_bytes(L) <= MOST_OPERANDS &&
           // 32-bit offsets within a chunk
           L.x_t >= 0 && L.x_t <= 1 << 24 && (int64_t) L.H * L.P <= 1 << 24 && L.P <= 1 << 24;
}

int64_t ssm_scan_mm_scratch_bytes(const ssm_scan_launch & L) { return mm_size(L).total; }

void launch_ssm_scan_mm(const ssm_scan_launch & L0, void * ws, hipStream_t st) {
    const mm_sizes z = mm_size(L0);
    const int64_t channels = (int64_t) L0.P * L0.H;
    for (int64_t s = 0; s < L0.S; s += z.seqs) {
        ssm_scan_launch L = L0;
        L.S = std::min(z.seqs, L0.S - s);
        L.x += s * L.x_s; L.dt += s * L.dt_s; L.B += s * L.b_s; L.C += s * L.c_s; L.ids += s * L.ids_s;
        L.y += s * channels * L.T; L.s_out += s * channels * L.N;
        if (z.nk == 8) launch_mm<8>(L, z, ws, st);
        else if (z.nk == 4) launch_mm<4>(L, z, ws, st);
        else if (z.nk == 2) launch_mm<2>(L, z, ws, st);
        else launch_mm<1>(L, z, ws, st);
    }
}
