// k_verify.hip — drafted tokens against the target's probabilities, from given random numbers.
//
// A sequence has n drafted tokens x_1 .. x_n, the target's probabilities p_1 .. p_{n+1} (row i for the token
// behind i - 1 of them), the draft's q_1 .. q_n and numbers u_1 .. u_{n+1} in [0, 1). x_i is accepted while
// u_i q_i(x_i) < p_i(x_i). The first that is not is replaced by a draw from the weights max(p_i - q_i, 0) (from p_i
// where all of them are 0), all accepted are followed by one from p_{n+1}: the first token whose weight, added to
// those before it, exceeds u_{n+1} times their sum. So the tokens are distributed as the target's own.
// Without q the draft is certain of its tokens: q_i is 1 at x_i.
//
// Sums are formed in 64 bits: with 32, the place where a sum of 10^5 probabilities passes a given number
// is off by several tokens' weights. Two launches: every workgroup finds the row by itself (a few
// scattered reads) and adds up a segment; then a workgroup a sequence looks for the segment, and in it for the token.
#include "kernels.h"

#include <algorithm>

namespace {

constexpr int VERIFY_WG = 256;
constexpr int VERIFY_PER = VERIFY_SEGMENT / VERIFY_WG;

struct verify_row {
    const float * p, * q;      // q: nullptr where nothing is taken off
    int without;               // the token without weight, or -1
};

__device__ __forceinline__ const float * row_of(const verify_rows & R, int64_t i) {
    const int64_t i1 = i % R.ne1, r = i / R.ne1;
    return (const float *) (R.base + i1 * R.nb1 + (r % R.ne2) * R.nb2 + (r / R.ne2) * R.nb3);
}

// tokens of sequence s that are accepted, by the whole workgroup
__device__ __forceinline__ int accepted(const verify_launch & L, int s, int first, int n, int * s_first) {
    const int t = threadIdx.x;
    if (t == 0) *s_first = n;
    __syncthreads();
    for (int i = t; i < n; i += VERIFY_WG) {
        const int x = L.tokens[first + i];
        const double p = row_of(L.p, L.row0 + L.seq0 + first + s + i)[x];
        const double q = L.q.base ? (double) row_of(L.q, L.row0 + first + i)[x] : 1.0;
        if (!(L.u[first + s + i] * q < p)) atomicMin(s_first, i);
    }
    __syncthreads();
    return *s_first;
}

__device__ __forceinline__ verify_row drawn_row(const verify_launch & L, int s, int first, int n, int k) {
    verify_row r{ row_of(L.p, L.row0 + L.seq0 + first + s + k), nullptr, -1 };
    if (k < n) {
        if (L.q.base) r.q = row_of(L.q, L.row0 + first + k);
        else r.without = L.tokens[first + k];
    }
    return r;
}

// the weight of token i in the draw (a NaN stays one)
__device__ __forceinline__ double weight(const verify_row & r, float p, float q, int i) {
    const double d = i == r.without ? 0.0 : (double) p - (double) q;
    return d > 0.0 || d != d ? d : 0.0;
}

__device__ __forceinline__ double wg_sum(double v, double * s_part) {
    v = wave_sum_d(v);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) s_part[threadIdx.x / WAVE] = v;
    __syncthreads();
    return ((s_part[0] + s_part[1]) + s_part[2]) + s_part[3];
}

// weights' sums of one segment: parts[s][segment] = (of the draw, of p alone)
__global__ __launch_bounds__(VERIFY_WG) void verify_sums_kernel(const verify_launch L) {
    __shared__ int s_first;
    __shared__ double s_part[VERIFY_WG / WAVE];
    const int s = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const int first = L.first[s], n = L.first[s + 1] - first;
    const int k = accepted(L, s, first, n, &s_first);
    const verify_row r = drawn_row(L, s, first, n, k);
    double sum = 0.0, alone = 0.0;
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j++) {
        const int i = seg * VERIFY_SEGMENT + j * VERIFY_WG + t;
        if (i >= L.n) continue;
        const float p = r.p[i];
        sum += weight(r, p, r.q ? r.q[i] : 0.0f, i);
        alone += p > 0.0f || p != p ? (double) p : 0.0;
    }
    sum = wg_sum(sum, s_part);
    alone = wg_sum(alone, s_part);
    if (t == 0) {
        L.parts[(int64_t) s * L.segments + seg] = make_double2(sum, alone);
        if (seg == 0) L.out[2 * s] = k;
    }
}

// inclusive sums over the workgroup's threads in order; all: of everything
__device__ __forceinline__ double wg_scan(double v, double * s_part, double & all) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
#pragma unroll
    for (int k = 1; k < WAVE; k *= 2) {
        const double o = __shfl_up(v, k);
        if (lane >= k) v += o;
    }
    __syncthreads();
    if (lane == WAVE - 1) s_part[wave] = v;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
    for (int w = 0; w < VERIFY_WG / WAVE; w++) {
        if (w < wave) before += s_part[w];
        all += s_part[w];
    }
    return before + v;
}

__global__ __launch_bounds__(VERIFY_WG) void verify_pick_kernel(const verify_launch L) {
    __shared__ int s_first, s_seg, s_at, s_last;
    __shared__ double s_part[VERIFY_WG / WAVE], s_before;
    const int s = blockIdx.x, t = threadIdx.x;
    const int first = L.first[s], n = L.first[s + 1] - first;
    const int k = accepted(L, s, first, n, &s_first);
    verify_row r = drawn_row(L, s, first, n, k);
    const double2 * parts = L.parts + (int64_t) s * L.segments;
    // the sum, and whether p alone is drawn from
    double total = 0.0, alone = 0.0;
    for (int i = t; i < L.segments; i += VERIFY_WG) { total += parts[i].x; alone += parts[i].y; }
    total = wg_sum(total, s_part);
    alone = wg_sum(alone, s_part);
    const bool only_p = total == 0.0;
    if (only_p) {
        r.q = nullptr;
        r.without = -1;
        total = alone;
    }
    if (!(total > 0.0) || isinf(total)) {
        if (t == 0) L.out[2 * s + 1] = -1;
        return;
    }
    const double goal = L.u[first + s + n] * total;
    // the first segment that passes it (the last with any weight where rounding lets none)
    if (t == 0) { s_seg = L.segments; s_last = 0; s_at = L.n; }
    __syncthreads();
    double before = 0.0;
    for (int i0 = 0; i0 < L.segments; i0 += VERIFY_WG) {
        const int i = i0 + t;
        const double v = i < L.segments ? (only_p ? parts[i].y : parts[i].x) : 0.0;
        double all;
        const double up = before + wg_scan(v, s_part, all);
        if (v > 0.0) atomicMax(&s_last, i);
        if (v > 0.0 && up > goal) atomicMin(&s_seg, i);
        __syncthreads();
        if (s_seg == i) s_before = up - v;
        if (s_seg < L.segments) break;
        before += all;
        __syncthreads();
    }
    __syncthreads();
    const bool past = s_seg == L.segments;
    const int seg = past ? s_last : s_seg;
    before = past ? 0.0 : s_before;
    __syncthreads();
    if (t == 0) s_last = 0;
    __syncthreads();
    // its values, VERIFY_PER in a row for each thread
    double w[VERIFY_PER], sum = 0.0, all;
    const int i0 = seg * VERIFY_SEGMENT + t * VERIFY_PER;
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j++) {
        const int i = i0 + j;
        w[j] = i < L.n ? weight(r, r.p[i], r.q ? r.q[i] : 0.0f, i) : 0.0;
        sum += w[j];
    }
    double up = before + wg_scan(sum, s_part, all) - sum;
    int last = -1;
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j++) {
        up += w[j];
        if (w[j] > 0.0) {
            last = i0 + j;
            if (!past && up > goal) atomicMin(&s_at, i0 + j);
        }
    }
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (t == 0) L.out[2 * s + 1] = s_at < L.n ? s_at : s_last;
}

} // namespace

void launch_verify(const verify_launch & L, hipStream_t st) {
    if (L.n_seqs == 0) return;
    launch(verify_sums_kernel, dim3((unsigned) L.segments, (unsigned) L.n_seqs), dim3(VERIFY_WG), 0, st, L);
    launch(verify_pick_kernel, dim3((unsigned) L.n_seqs), dim3(VERIFY_WG), 0, st, L);
}
