// k_logprobs.hip — log probabilities of given tokens under rows of logits, the rows' entropies and
// their likeliest tokens.
//
// With m the largest logit of a row, e_i = exp(l_i - m), S = sum e_i and W = sum e_i (l_i - m):
//   log p_i = l_i - m - log S,   H = -sum p_i log p_i = log S - W / S.
// An entry of -inf weighs nothing (0 log 0 = 0). A row whose largest logit is not finite has no
// distribution: its scores are NaN. NaN entries order as -inf, as in the sampler; a row that holds
// one has no distribution either.
//
// A row is read once: it is split into segments of up to LP_SEG logits that a workgroup holds in its
// registers (32 per thread), where the maximum, the sums and the selection all read them. Segments
// join as S = sum S_j exp(m_j - m), W = sum exp(m_j - m) (W_j + S_j (m_j - m)), and their k best
// entries merge by rank. So many rows are bound by memory, and one row by two launches' latency.
#include "hip_common.h"
#include "kernels.h"

#include <algorithm>

namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_WAVES = LP_THREADS / WAVE;
constexpr int LP_PER = 32;                        // logits per thread, in groups of 4
constexpr int LP_SEG = LP_THREADS * LP_PER;
constexpr int LP_CAND = 1024;                     // entries a selection sorts
constexpr float LOG2E = 1.4426950408889634f;

// ascending order key of a float; -0 and +0 share a key
__device__ __forceinline__ uint32_t okey(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float okey_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// descending order is descending value, then ascending id; no entry's key is 0
__device__ __forceinline__ uint64_t ckey(float v, int id) { return ((uint64_t) okey(v) << 32) | (uint32_t) ~id; }

__device__ __forceinline__ float wave_sum(float v) { return group_sum<64>(v); }
__device__ __forceinline__ int wave_sum(int v) {
    v += dpp_i<0xB1>(v);
    v += dpp_i<0x4E>(v);
    v += dpp_i<0x141>(v);
    v += dpp_i<0x140>(v);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
           __builtin_amdgcn_readlane(v, 48);
}

struct lp_shared {
    uint64_t key[LP_CAND];
    float f[2][LP_WAVES];
    int n[2][LP_WAVES];
    int count;
};

// The k best of a workgroup's LP_SEG values (v[4 j + c] is entry j * 1024 + thread * 4 + c), in order,
// to out(rank, key): every rank below k, key 0 where there are fewer entries.
// A threshold first: M >= k groups of threads each have a largest value, so the smallest of those, t,
// has at least k entries at or above it (for normally distributed logits and k = 20 about 110 of 8192).
// The entries above t are listed and each finds its rank by comparing with all; where they are fewer
// than k, entries equal to t follow in the order of their ids. Were the list too long (values that the
// groups do not share evenly, such as a block of -inf), t becomes the k-th largest value itself, found
// by bisection: fewer than k entries lie above it.
template <class F>
__device__ void select_top(const float (&v)[LP_PER], int valid, int id0, int k, lp_shared & S, F out) {
    const int tid = threadIdx.x, wave = tid / WAVE;
    auto index = [&](int i) { return (i / 4) * (LP_THREADS * 4) + tid * 4 + i % 4; };
    float t = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP_PER; i++) t = fmaxf(t, v[i]);
    if (k > 64) t = group_max<2>(t);
    else if (k > 32) t = group_max<4>(t);
    else if (k > 16) t = group_max<8>(t);
    else if (k > 8) t = group_max<16>(t);
    else if (k > 4) t = group_max<32>(t);
    else t = group_max<64>(t);
    t = -wave_max(-t);
    if (tid % WAVE == 0) S.f[0][wave] = t;
    __syncthreads();
    t = fminf(fminf(S.f[0][0], S.f[0][1]), fminf(S.f[0][2], S.f[0][3]));
    // entries that satisfy f, over the workgroup; `turn` alternates the words that it uses
    auto count = [&](int turn, auto f) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < LP_PER; i++) n += index(i) < valid && f(v[i]) ? 1 : 0;
        n = wave_sum(n);
        if (tid % WAVE == 0) S.n[turn][wave] = n;
        __syncthreads();
        return S.n[turn][0] + S.n[turn][1] + S.n[turn][2] + S.n[turn][3];
    };
    int above = count(0, [&](float x) { return x > t; });
    if (above > LP_CAND) {
        // the largest value with k entries at or above it; okey(t) has them
        uint32_t lo = okey(t), hi = 0xffffffffu;
        int turn = 1;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (count(turn, [&](float x) { return okey(x) >= mid; }) >= k) lo = mid;
            else hi = mid - 1;
            turn ^= 1;
        }
        t = okey_value(lo);
        above = count(turn, [&](float x) { return x > t; });
    }
    if (tid == 0) S.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LP_PER; i++) {
        if (index(i) < valid && v[i] > t) S.key[atomicAdd(&S.count, 1)] = ckey(v[i], id0 + index(i));
    }
    __syncthreads();
    for (int i = tid; i < above; i += LP_THREADS) {
        const uint64_t mine = S.key[i];
        int rank = 0;
        for (int j = 0; j < above; j++) rank += S.key[j] > mine ? 1 : 0;
        if (rank < k) out(rank, mine);
    }
    // entries equal to the threshold, row of 1024 by row in the order of their ids
    for (int row = 0, at = above; row < LP_PER / 4 && at < k; row++) {
        int n = 0, before = 0, all = 0;
        bool eq[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            float x = v[c];
#pragma unroll
            for (int j = 1; j < LP_PER / 4; j++) x = row == j ? v[4 * j + c] : x;
            eq[c] = row * (LP_THREADS * 4) + tid * 4 + c < valid && x == t;
            const uint64_t m = __ballot(eq[c]);
            before += __popcll(m & ((1ull << (tid % WAVE)) - 1));
            all += __popcll(m);
        }
        __syncthreads();
        if (tid % WAVE == 0) S.n[0][wave] = all;
        __syncthreads();
        for (int w = 0; w < wave; w++) before += S.n[0][w];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int rank = at + before + n;
            if (eq[c] && rank < k) out(rank, ckey(t, id0 + row * (LP_THREADS * 4) + tid * 4 + c));
            n += eq[c] ? 1 : 0;
        }
        at += S.n[0][0] + S.n[0][1] + S.n[0][2] + S.n[0][3];
        if (row == LP_PER / 4 - 1) {
            for (int i = at + tid; i < k; i += LP_THREADS) out(i, 0);
        }
    }
}

__device__ __forceinline__ const float * row_of(const logprobs_launch & L, int r) {
    const int64_t row = L.row0 + r, i1 = row % L.ne1, i2 = row / L.ne1 % L.ne2, i3 = row / (L.ne1 * L.ne2);
    return (const float *) (L.base + i1 * L.nb1 + i2 * L.nb2 + i3 * L.nb3);
}

// a segment's (or a row's) maximum, sums and whether it holds a NaN
struct lp_stats { float m, s, w, bad; };

// the log of the sum of a row's exponentials above its maximum: NaN where it has no distribution
__device__ __forceinline__ float log_sum(const lp_stats & a) { return a.bad != 0.0f || !(fabsf(a.m) < INFINITY) ? NAN : logf(a.s); }

// A row's results, gathered in LDS and then stored as one run of words: they go straight to host
// memory, where each separate store would be a bus transfer of its own.
struct lp_out { float w[2 + 2 * LOGPROBS_MAX_TOP]; };

__device__ __forceinline__ void put_scores(const logprobs_launch & L, int r, const float * x, const lp_stats & a, float ls, lp_out & o) {
    o.w[0] = L.tokens ? x[L.tokens[r]] - a.m - ls : 0.0f;
    o.w[1] = ls - a.w / a.s;
}
__device__ __forceinline__ void put_top(const logprobs_launch & L, float m, float ls, lp_out & o, int rank, uint64_t key) {
    o.w[2 + rank] = __int_as_float((int) ~(uint32_t) key);
    o.w[2 + L.k + rank] = okey_value((uint32_t) (key >> 32)) - m - ls;
}
__device__ __forceinline__ void store_row(const logprobs_launch & L, int r, const lp_out & o) {
    __syncthreads();
    const int n = 2 + 2 * L.k;
    for (int i = threadIdx.x; i < n; i += LP_THREADS) L.out[(int64_t) r * n + i] = o.w[i];
}

// One segment of one row. Where it is the whole row the results are final, else they go to the scratch.
template <bool VEC>
__global__ __launch_bounds__(LP_THREADS) void logprobs_segment_kernel(logprobs_launch L) {
    __shared__ lp_shared S;
    __shared__ lp_out o;
    const int seg = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, wave = tid / WAVE;
    const int id0 = seg * L.seg, valid = min(L.seg, L.n - id0);
    const float * x = row_of(L, r) + id0;
    float v[LP_PER];
#pragma unroll
    for (int j = 0; j < LP_PER / 4; j++) {
        const int i = j * (LP_THREADS * 4) + tid * 4;
        if (VEC && i + 3 < valid) {
            const float4 f = *(const float4 *) (x + i);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) v[4 * j + c] = i + c < valid ? x[i + c] : -INFINITY;
        }
    }
    lp_stats a{ -INFINITY, 0.0f, 0.0f, 0.0f };
#pragma unroll
    for (int i = 0; i < LP_PER; i++) {
        if (v[i] != v[i]) { a.bad = 1.0f; v[i] = -INFINITY; }
        a.m = fmaxf(a.m, v[i]);
    }
    a.m = wave_max(a.m);
    a.bad = wave_max(a.bad);
    if (tid % WAVE == 0) { S.f[0][wave] = a.m; S.f[1][wave] = a.bad; }
    __syncthreads();
    a.m = fmaxf(fmaxf(S.f[0][0], S.f[0][1]), fmaxf(S.f[0][2], S.f[0][3]));
    a.bad = fmaxf(fmaxf(S.f[1][0], S.f[1][1]), fmaxf(S.f[1][2], S.f[1][3]));
    __syncthreads();
    // nothing but -inf: every weight is 0, not exp(-inf + inf)
    const float m = a.m == -INFINITY ? 0.0f : a.m;
#pragma unroll
    for (int i = 0; i < LP_PER; i++) {
        const float z = v[i] - m, e = __builtin_amdgcn_exp2f(z * LOG2E);
        a.s += e;
        a.w = fmaf(e, fmaxf(z, -3e38f), a.w);     // 0 times -inf is no weight
    }
    a.s = wave_sum(a.s);
    a.w = wave_sum(a.w);
    if (tid % WAVE == 0) { S.f[0][wave] = a.s; S.f[1][wave] = a.w; }
    __syncthreads();
    a.s = (S.f[0][0] + S.f[0][1]) + (S.f[0][2] + S.f[0][3]);
    a.w = (S.f[1][0] + S.f[1][1]) + (S.f[1][2] + S.f[1][3]);
    __syncthreads();
    if (L.n_seg == 1) {
        const float ls = log_sum(a);
        if (tid == 0) put_scores(L, r, x, a, ls, o);
        if (L.k) select_top(v, valid, 0, L.k, S, [&](int rank, uint64_t key) { put_top(L, a.m, ls, o, rank, key); });
        store_row(L, r, o);
        return;
    }
    const int64_t at = (int64_t) r * L.n_seg + seg;
    if (tid == 0) ((lp_stats *) L.part)[at] = a;
    uint64_t * keys = (uint64_t *) ((lp_stats *) L.part + (int64_t) L.n_rows * L.n_seg) + at * L.k;
    if (L.k) select_top(v, valid, id0, L.k, S, [&](int rank, uint64_t key) { keys[rank] = key; });
}

// A row's segments joined. Each segment's list is in descending order, so an entry's rank is its own
// place plus, for each other segment, the number of entries above it: a bisection per segment.
__global__ __launch_bounds__(LP_THREADS) void logprobs_join_kernel(logprobs_launch L) {
    extern __shared__ uint64_t staged[];
    __shared__ lp_out o;
    const int r = blockIdx.x, tid = threadIdx.x, total = L.n_seg * L.k;
    const lp_stats * part = (const lp_stats *) L.part + (int64_t) r * L.n_seg;
    const uint64_t * keys = (const uint64_t *) ((const lp_stats *) L.part + (int64_t) L.n_rows * L.n_seg) + (int64_t) r * total;
    // lists of very long rows stay where they are
    const uint64_t * list = L.stage ? staged : keys;
    if (L.stage) {
        for (int i = tid; i < total; i += LP_THREADS) staged[i] = keys[i];
    }
    lp_stats a{ -INFINITY, 0.0f, 0.0f, 0.0f };
    for (int j = 0; j < L.n_seg; j++) {
        a.m = fmaxf(a.m, part[j].m);
        a.bad = fmaxf(a.bad, part[j].bad);
    }
    for (int j = 0; j < L.n_seg; j++) {
        if (part[j].s == 0.0f) continue;          // a segment of -inf alone
        const float z = part[j].m - a.m, e = __builtin_amdgcn_exp2f(z * LOG2E);
        a.s = fmaf(part[j].s, e, a.s);
        if (e > 0.0f) a.w = fmaf(fmaf(part[j].s, z, part[j].w), e, a.w);
    }
    const float ls = log_sum(a);
    if (tid == 0) put_scores(L, r, row_of(L, r), a, ls, o);
    __syncthreads();
    for (int i = tid; i < total; i += LP_THREADS) {
        const uint64_t mine = list[i];
        const int own = i / L.k;
        int rank = i - own * L.k;
        for (int s = 0; s < L.n_seg; s++) {
            if (s == own) continue;
            const uint64_t * l = list + s * L.k;
            int lo = 0, hi = L.k;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (l[mid] > mine) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (mine && rank < L.k) put_top(L, a.m, ls, o, rank, mine);
    }
    store_row(L, r, o);
}

int segments(int n) { return (n + LP_SEG - 1) / LP_SEG; }

} // namespace

int64_t logprobs_scratch_bytes(int n, int k, int n_rows) {
    return segments(n) == 1 ? 0 : (int64_t) n_rows * segments(n) * ((int64_t) sizeof(lp_stats) + 8 * k);
}

void launch_logprobs(const logprobs_launch & L0, hipStream_t st) {
    logprobs_launch L = L0;
    L.n_seg = segments(L.n);
    // even segments, of whole rows of 1024 entries
    L.seg = std::min(LP_SEG, ((L.n + L.n_seg - 1) / L.n_seg + LP_THREADS * 4 - 1) / (LP_THREADS * 4) * (LP_THREADS * 4));
    L.n_seg = (L.n + L.seg - 1) / L.seg;
    const bool vec = ((uintptr_t) L.base | (uintptr_t) L.nb1 | (uintptr_t) L.nb2 | (uintptr_t) L.nb3) % 16 == 0;
    launch(vec ? logprobs_segment_kernel<true> : logprobs_segment_kernel<false>, dim3((unsigned) L.n_seg, (unsigned) L.n_rows),
           dim3(LP_THREADS), 0, st, L);
    if (L.n_seg > 1) {
        const size_t lds = (size_t) L.n_seg * L.k * 8;
        L.stage = lds <= 60 << 10;
        launch(logprobs_join_kernel, dim3((unsigned) L.n_rows), dim3(LP_THREADS), L.stage ? lds : 0, st, L);
    }
}
