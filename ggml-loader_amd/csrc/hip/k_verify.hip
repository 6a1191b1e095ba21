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
// is off by several tokens' weights. Three launches: a workgroup a sequence finds the row that is drawn from (the
// numbers come from host memory, whose reads the segments' many workgroups would queue for), a workgroup a segment
// adds up its weights, and one a sequence looks for the segment, and in it for the token. (The last segment's
// workgroup to end could do that: but to make its sums visible to it every workgroup writes its die's cache back,
// 130 us for 64 sequences of 128256 tokens.)
// Bound by latency: 4.7 + 2.8 + 3.8 us for one sequence of 151936 tokens, 7 + 10.4 + 4.3 for 64 of 128256 (66 MB of
// probabilities at 6.3 TB/s, out of the memory-side cache), of calls of 28 and 38.
#include "kernels.h"

#include <algorithm>

namespace {

constexpr int VERIFY_WG = 256;
constexpr int VERIFY_PER = VERIFY_SEGMENT / VERIFY_WG;

__device__ __forceinline__ const float * row_of(const verify_rows & R, int64_t i) {
    const int64_t i1 = i % R.ne1, r = i / R.ne1;
    return (const float *) (R.base + i1 * R.nb1 + (r % R.ne2) * R.nb2 + (r / R.ne2) * R.nb3);
}

// the tokens that are accepted, and the row behind them
__global__ __launch_bounds__(VERIFY_WG) void verify_heads_kernel(const verify_launch L) {
    __shared__ int s_first;
    const int s = blockIdx.x, t = threadIdx.x;
    const int first = L.first[s], n = L.first[s + 1] - first;
    if (t == 0) s_first = n;
    __syncthreads();
    for (int i = t; i < n; i += VERIFY_WG) {
        const int x = L.tokens[first + i];
        const double u = L.u[first + s + i];
        const double p = row_of(L.p, L.row0 + L.seq0 + first + s + i)[x];
        const double q = L.q.base ? (double) row_of(L.q, L.row0 + first + i)[x] : 1.0;
        if (!(u * q < p)) atomicMin(&s_first, i);
    }
    __syncthreads();
    if (t != 0) return;
    const int k = s_first;
    verify_head r{ row_of(L.p, L.row0 + L.seq0 + first + s + k), nullptr, L.u[first + s + n], -1 };
    if (k < n) {
        if (L.q.base) r.q = row_of(L.q, L.row0 + first + k);
        else r.without = L.tokens[first + k];
    }
    L.heads[s] = r;
    L.out[2 * s] = k;
}

// the weight of token i in the draw (a NaN stays one)
__device__ __forceinline__ double weight(double p, double q) {
    const double d = p - q;
    return d > 0.0 || d != d ? d : 0.0;
}

// Four values of the segment, 0 past the row's end. wide: rows of fours on 16 bytes
__device__ __forceinline__ void four_of(const float * x, int i, int n, bool wide, float * v) {
    if (wide) {
        const float4 a = i < n ? *(const float4 *) (x + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = i + j < n ? x[i + j] : 0.0f;
}

// the weights of four tokens from i on
__device__ __forceinline__ void weights_of(const float * p, const float * q, int without, int i, double * w) {
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = i + j == without ? 0.0 : weight(p[j], q[j]);
}

// a segment's sums: of the draw's weights, and of p alone
__global__ __launch_bounds__(VERIFY_WG) void verify_sums_kernel(const verify_launch L) {
    __shared__ double s_part[2][VERIFY_WG / WAVE];
    const int s = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const verify_head r = L.heads[s];
    double sum = 0.0, alone = 0.0;
    float p[VERIFY_PER], q[VERIFY_PER];
    const int i0 = seg * VERIFY_SEGMENT + t * 4;
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j += 4) {
        four_of(r.p, i0 + j * VERIFY_WG, L.n, L.wide, p + j);
        if (r.q) four_of(r.q, i0 + j * VERIFY_WG, L.n, L.wide, q + j);
        else q[j] = q[j + 1] = q[j + 2] = q[j + 3] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j += 4) {
        double w[4];
        weights_of(p + j, q + j, r.without, i0 + j * VERIFY_WG, w);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            sum += w[k];
            alone += weight(p[j + k], 0.0);
        }
    }
    sum = wave_sum_d(sum);
    alone = wave_sum_d(alone);
    if (t % WAVE == 0) { s_part[0][t / WAVE] = sum; s_part[1][t / WAVE] = alone; }
    __syncthreads();
    if (t != 0) return;
    auto all = [&](int k) { return ((s_part[k][0] + s_part[k][1]) + s_part[k][2]) + s_part[k][3]; };
    L.parts[(int64_t) s * L.segments + seg] = make_double2(all(0), all(1));
}

// inclusive sums over the workgroup's threads in order, of two values; all: of everything
__device__ __forceinline__ double2 wg_scan(double2 v, double2 * s_part, double2 & all) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
#pragma unroll
    for (int k = 1; k < WAVE; k *= 2) {
        const double x = __shfl_up(v.x, k), y = __shfl_up(v.y, k);
        if (lane >= k) { v.x += x; v.y += y; }
    }
    __syncthreads();
    if (lane == WAVE - 1) s_part[wave] = v;
    __syncthreads();
    double2 before = make_double2(0.0, 0.0);
    all = before;
#pragma unroll
    for (int w = 0; w < VERIFY_WG / WAVE; w++) {
        if (w < wave) { before.x += s_part[w].x; before.y += s_part[w].y; }
        all.x += s_part[w].x;
        all.y += s_part[w].y;
    }
    return make_double2(before.x + v.x, before.y + v.y);
}

// the first lane of the wave with it, or the last, or -1
__device__ __forceinline__ int first_lane(bool b) { return __ffsll((unsigned long long) __ballot(b)) - 1; }
__device__ __forceinline__ int last_lane(bool b) { return WAVE - 1 - __clzll((long long) __ballot(b)); }

// The token of a sequence from its segments' sums (of the draw's weights, and of p alone). p is drawn from where no
// token has a weight.
__global__ __launch_bounds__(VERIFY_WG) void verify_pick_kernel(const verify_launch L) {
    __shared__ int s_seg, s_at, s_last;
    __shared__ double2 s_part[VERIFY_WG / WAVE];
    __shared__ double s_before;
    const int s = blockIdx.x, t = threadIdx.x, lane = t % WAVE;
    const verify_head r = L.heads[s];
    const double2 * parts = L.parts + (int64_t) s * L.segments;
    auto part_of = [&](int i) { return i < L.segments ? parts[i] : make_double2(0.0, 0.0); };
    double2 mine = part_of(t), all, up = wg_scan(mine, s_part, all), total = all;
    for (int i0 = VERIFY_WG; i0 < L.segments; i0 += VERIFY_WG) {
        wg_scan(part_of(i0 + t), s_part, all);
        total.x += all.x;
        total.y += all.y;
    }
    const bool only_p = total.x == 0.0;
    const double sum = only_p ? total.y : total.x;
    if (!(sum > 0.0) || isinf(sum)) {
        if (t == 0) L.out[2 * s + 1] = -1;
        return;
    }
    const double goal = r.u * sum;
    // the first segment that passes it (the last with any weight where rounding lets none)
    if (t == 0) { s_seg = L.segments; s_last = 0; s_at = L.n; s_before = 0.0; }
    __syncthreads();
    double2 before = make_double2(0.0, 0.0);
    for (int i0 = 0;;) {
        const int i = i0 + t;
        const double v = only_p ? mine.y : mine.x, to = only_p ? before.y + up.y : before.x + up.x;
        const int some = last_lane(v > 0.0), passed = first_lane(v > 0.0 && to > goal);
        if (lane == 0 && some >= 0) atomicMax(&s_last, i + some);
        if (lane == 0 && passed >= 0) atomicMin(&s_seg, i + passed);
        __syncthreads();
        if (s_seg == i) s_before = to - v;
        i0 += VERIFY_WG;
        if (s_seg < L.segments || i0 >= L.segments) break;
        if (i0 > VERIFY_WG) { before.x += all.x; before.y += all.y; }
        else {
            wg_scan(mine, s_part, all);
            before = all;
        }
        mine = part_of(i0 + t);
        up = wg_scan(mine, s_part, all);
    }
    __syncthreads();
    const bool past = s_seg == L.segments;
    const int seg = past ? s_last : s_seg;
    // its values, VERIFY_PER in a row for each thread
    const float * q = only_p ? nullptr : r.q;
    const int without = only_p ? -1 : r.without, i0 = seg * VERIFY_SEGMENT + t * VERIFY_PER;
    double w[VERIFY_PER], own = 0.0;
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j += 4) {
        float p4[4], q4[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
        four_of(r.p, i0 + j, L.n, L.wide, p4);
        if (q) four_of(q, i0 + j, L.n, L.wide, q4);
        weights_of(p4, q4, without, i0 + j, w + j);
    }
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j++) own += w[j];
    const double start = s_before;
    double to = start + wg_scan(make_double2(own, 0.0), s_part, all).x - own;
    if (t == 0) s_last = 0;
    __syncthreads();
    int last = -1, at = -1;
#pragma unroll
    for (int j = 0; j < VERIFY_PER; j++) {
        to += w[j];
        if (w[j] > 0.0) {
            last = i0 + j;
            if (!past && at < 0 && to > goal) at = i0 + j;
        }
    }
    if (lane == first_lane(at >= 0)) atomicMin(&s_at, at);
    if (lane == last_lane(last >= 0)) atomicMax(&s_last, last);
    __syncthreads();
    if (t == 0) L.out[2 * s + 1] = s_at < L.n ? s_at : s_last;
}

} // namespace

void launch_verify(verify_launch L, hipStream_t st) {
    if (L.n_seqs == 0) return;
    L.wide = L.n % 4 == 0;
    for (const verify_rows * R : { &L.p, &L.q }) {
        if (((uintptr_t) R->base | (uintptr_t) R->nb1 | (uintptr_t) R->nb2 | (uintptr_t) R->nb3) % 16 && R->base) L.wide = 0;
    }
    launch(verify_heads_kernel, dim3((unsigned) L.n_seqs), dim3(VERIFY_WG), 0, st, L);
    launch(verify_sums_kernel, dim3((unsigned) L.segments, (unsigned) L.n_seqs), dim3(VERIFY_WG), 0, st, L);
    launch(verify_pick_kernel, dim3((unsigned) L.n_seqs), dim3(VERIFY_WG), 0, st, L);
}
