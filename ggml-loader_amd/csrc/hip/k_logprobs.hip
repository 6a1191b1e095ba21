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
// entries merge by rank. So many rows are bound by memory, and one row by two launches' latency:
// 512 rows of 128256 logits take 51 us (5.1 TB/s) with 20 entries each and 41 with none, and 10 to join; one
// row of 151936 takes 7 and 7, in a call that waits for its results and takes 19 us with nothing to do.
#include "hip_common.h"
#include "kernels.h"

#include <algorithm>

namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_WAVES = LP_THREADS / WAVE;
constexpr int LP_PER = 32;                        // logits per thread, in groups of 4
constexpr int LP_SEG = LP_THREADS * LP_PER;
constexpr int LP_CAND = 1024;                     // entries a selection sorts
constexpr int LP_KEPT = 6144;                     // entries a join sorts: 48 KiB
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

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
    alignas(16) uint64_t key[LP_CAND];
    alignas(16) float best[LP_THREADS];
    float f[2][LP_WAVES], w[LP_WAVES];
    int n[2][LP_WAVES];
};

// keys[0 .. n) to out(rank, key), every rank below k: each key's rank is the number of keys above it.
// keys is padded with zeros to a multiple of 4 entries; all threads must call it.
template <class F>
__device__ __forceinline__ void rank_keys(const uint64_t * keys, int n, int k, F out) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const uint64_t mine = keys[i];
        int rank = 0;
        const ulonglong2 * kk = (const ulonglong2 *) keys;
#pragma unroll 4
        for (int j = 0; j < (n + 3) / 4 * 2; j++) {
            const ulonglong2 u = kk[j];
            rank += (u.x > mine ? 1 : 0) + (u.y > mine ? 1 : 0);
        }
        if (rank < k) out(rank, mine);
    }
}

// The k best of a workgroup's LP_SEG values (v[4 j + c] is entry j * 1024 + thread * 4 + c; the ones
// from `valid` on are -inf), in order, to out(rank, key): every rank below k, key 0 where there are
// fewer entries. best: the thread's largest value.
// A threshold first: of M groups of threads, each with its largest value, the k-th largest, t, has k entries at or
// above it and few more (with evenly spread values and k = 20 of 64 groups about 24). M is 64 up to k = 32 and 256
// above; up to k = 8 it is 8 or 4, at least k, and t the least of all, which takes no comparing. The entries
// from t on are listed and each finds its rank by comparing with all. Were the list too long (values that the
// groups do not share evenly, such as a block of -inf, or many equal ones), t becomes the k-th largest value
// itself, found by bisection: fewer than k entries lie above it, and ones equal to it follow in the order of
// their ids. (With the least of M >= k groups' values for t, as it was, 110 entries were listed for k = 20,
// and ranking them was a quarter of the pass: 65 us at 512 rows of 128256 instead of 51.)
template <class F>
__device__ __forceinline__ void select_top(const float (&v)[LP_PER], float best, int valid, int id0, int k, lp_shared & S, F out) {
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    float t;
    // `groups` values lie in S.best; of those with fewer than k above them the least one
    auto kth = [&](float own, int groups) {
        int above = 0;
#pragma unroll 16
        for (int i = 0; i < groups; i += 4) {
            const float4 g = *(const float4 *) (S.best + i);
            above += (g.x > own ? 1 : 0) + (g.y > own ? 1 : 0) + (g.z > own ? 1 : 0) + (g.w > own ? 1 : 0);
        }
        return -wave_max(above < k ? -own : -INFINITY);
    };
    // the least of a value per wave
    auto least = [&](float v) {
        if (lane == 0) S.f[0][wave] = v;
        __syncthreads();
        return fminf(fminf(S.f[0][0], S.f[0][1]), fminf(S.f[0][2], S.f[0][3]));
    };
    if (k <= 8) {
        // 8 or 4 groups and the least of all: about 22 or 8 entries
        t = k > 4 ? group_max<32>(best) : group_max<64>(best);
        t = least(-wave_max(-t));
    } else if (k <= 32) {
        // every wave for itself
        const float g = group_max<4>(best);
        if (lane % 4 == 0) S.best[tid / 4] = g;
        __syncthreads();
        t = kth(S.best[lane], 64);
    } else {
        S.best[tid] = best;
        __syncthreads();
        t = least(kth(best, LP_THREADS));
    }
    // entries that satisfy f, of this thread (mine) and of the workgroup; `turn` alternates the words that it uses
    int mine;
    auto count = [&](int turn, auto f) {
        mine = 0;
#pragma unroll
        for (int i = 0; i < LP_PER; i++) mine += f(v[i]) ? 1 : 0;
        const int n = wave_sum(mine);
        if (lane == 0) S.n[turn][wave] = n;
        __syncthreads();
        return S.n[turn][0] + S.n[turn][1] + S.n[turn][2] + S.n[turn][3];
    };
    // entries above `t` are listed: with the float before t that is t's too, but for the -inf that also fill a segment
    const float kt = t;
    bool ties = t == -INFINITY;
    if (!ties) t = okey_value(okey(t) - (t == 0.0f ? 2 : 1));     // -0 is no less than 0
    int turn = 0, above = count(0, [&](float x) { return x > t; });
    if (above > LP_CAND) {
        // the largest value with k entries at or above it; kt has them
        uint32_t lo = okey(kt), hi = 0xffffffffu;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (count(turn ^= 1, [&](float x) { return okey(x) >= mid; }) >= k) lo = mid;
            else hi = mid - 1;
        }
        t = okey_value(lo);
        above = count(turn ^= 1, [&](float x) { return x > t; });
        ties = true;
    }
    // the thread's place in the list: those of the waves and lanes before it
    int scan = mine;
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) {
        const int u = __shfl_up(scan, o, WAVE);
        scan += lane >= o ? u : 0;
    }
    int at = scan - mine;
    for (int w = 0; w < wave; w++) at += S.n[turn][w];
    if (mine) {
#pragma unroll
        for (int i = 0; i < LP_PER; i++) {
            if (v[i] > t) S.key[at++] = ckey(v[i], id0 + (i / 4) * (LP_THREADS * 4) + tid * 4 + i % 4);
        }
    }
    if (tid < (-above & 3)) S.key[above + tid] = 0;
    __syncthreads();
    rank_keys(S.key, above, k, out);
    if (!ties) return;
    // entries equal to the threshold, row of 1024 by row in the order of their ids
    for (int row = 0, got = above; row < LP_PER / 4 && got < k; row++) {
        int n = 0, before = 0, all = 0;
        bool eq[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            float x = v[c];
#pragma unroll
            for (int j = 1; j < LP_PER / 4; j++) x = row == j ? v[4 * j + c] : x;
            eq[c] = row * (LP_THREADS * 4) + tid * 4 + c < valid && x == t;
            const uint64_t m = __ballot(eq[c]);
            before += __popcll(m & ((1ull << lane) - 1));
            all += __popcll(m);
        }
        __syncthreads();
        if (lane == 0) S.n[0][wave] = all;
        __syncthreads();
        for (int w = 0; w < wave; w++) before += S.n[0][w];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int rank = got + before + n;
            if (eq[c] && rank < k) out(rank, ckey(t, id0 + row * (LP_THREADS * 4) + tid * 4 + c));
            n += eq[c] ? 1 : 0;
        }
        got += S.n[0][0] + S.n[0][1] + S.n[0][2] + S.n[0][3];
        if (row == LP_PER / 4 - 1) {
            for (int i = got + tid; i < k; i += LP_THREADS) out(i, 0);
        }
    }
}

__device__ __forceinline__ const float * row_of(const logprobs_launch & L, int r) {
    const int64_t row = L.row0 + r, i1 = row % L.ne1, i2 = row / L.ne1 % L.ne2, i3 = row / (L.ne1 * L.ne2);
    return (const float *) (L.base + i1 * L.nb1 + i2 * L.nb2 + i3 * L.nb3);
}

// a segment's (or a row's) maximum, sums and whether it holds a NaN
struct lp_stats { float m, s, w, bad; };

__device__ __forceinline__ lp_stats join(const lp_stats & a, const lp_stats & b) {
    lp_stats c{ fmaxf(a.m, b.m), 0.0f, 0.0f, fmaxf(a.bad, b.bad) };
    if (a.s > 0.0f) {                              // not a part of -inf alone
        const float z = a.m - c.m, e = __builtin_amdgcn_exp2f(z * LOG2E);
        c.s = a.s * e;
        c.w = e > 0.0f ? fmaf(a.s, z, a.w) * e : 0.0f;
    }
    if (b.s > 0.0f) {
        const float z = b.m - c.m, e = __builtin_amdgcn_exp2f(z * LOG2E);
        c.s = fmaf(b.s, e, c.s);
        c.w += e > 0.0f ? fmaf(b.s, z, b.w) * e : 0.0f;
    }
    return c;
}

// the log of the sum of a row's exponentials above its maximum: NaN where it has no distribution
__device__ __forceinline__ float log_sum(const lp_stats & a) { return a.bad != 0.0f || !(fabsf(a.m) < INFINITY) ? NAN : logf(a.s); }

// A row's results, gathered in LDS and then stored as one run of words: they go straight to host
// memory, where each separate store would be a bus transfer of its own.
struct lp_out { float w[2 + 2 * LOGPROBS_MAX_TOP]; };

__device__ __forceinline__ void put_scores(float tok, const lp_stats & a, float ls, lp_out & o) {
    o.w[0] = tok - a.m - ls;
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
__global__ __launch_bounds__(LP_THREADS) void logprobs_segment_kernel(logprobs_launch L) {
    __shared__ lp_shared S;
    __shared__ lp_out o;
    const int seg = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int id0 = seg * L.seg, valid = min(L.seg, L.n - id0);
    const float * x = row_of(L, r) + id0;
    float v[LP_PER];
#pragma unroll
    for (int j = 0; j < LP_PER / 4; j++) {
        const int i = j * (LP_THREADS * 4) + tid * 4;
        if (i + 3 < valid) {
            const float4 f = load4(x + i);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) v[4 * j + c] = i + c < valid ? x[i + c] : -INFINITY;
        }
    }
    lp_stats a{ -INFINITY, 0.0f, 0.0f, 0.0f };
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP_PER; i++) best = fmaxf(best, v[i]);     // a NaN is never the larger one
    a.m = wave_max(best);
    if (lane == 0) S.f[0][wave] = a.m;
    __syncthreads();
    a.m = fmaxf(fmaxf(S.f[0][0], S.f[0][1]), fmaxf(S.f[0][2], S.f[0][3]));
    // nothing but -inf: every weight is 0, not exp(-inf + inf)
    const float m = a.m == -INFINITY ? 0.0f : a.m;
#pragma unroll
    for (int i = 0; i < LP_PER; i++) {
        const float z = (v[i] - m) * LOG2E, e = __builtin_amdgcn_exp2f(z);
        a.s += e;
        a.w = fmaf(e, fmaxf(z, -3e38f), a.w);     // 0 times -inf is no weight
    }
    a.s = wave_sum(a.s);
    a.w = wave_sum(a.w);
    if (lane == 0) { S.f[1][wave] = a.s; S.w[wave] = a.w; }
    __syncthreads();
    a.s = (S.f[1][0] + S.f[1][1]) + (S.f[1][2] + S.f[1][3]);
    a.w = ((S.w[0] + S.w[1]) + (S.w[2] + S.w[3])) * LN2;
    if (a.s != a.s) {
        // a NaN, or +inf less itself: no distribution. A NaN orders as -inf.
        a.bad = 1.0f;
#pragma unroll
        for (int i = 0; i < LP_PER; i++) v[i] = v[i] != v[i] ? -INFINITY : v[i];
    }
    if (L.n_seg == 1) {
        const float ls = log_sum(a);
        if (tid == 0) put_scores(L.tokens ? x[L.tokens[r]] : 0.0f, a, ls, o);
        if (L.k) select_top(v, best, valid, 0, L.k, S, [&](int rank, uint64_t key) { put_top(L, a.m, ls, o, rank, key); });
        store_row(L, r, o);
        return;
    }
    const int64_t at = (int64_t) r * L.n_seg + seg;
    if (tid == 0) ((lp_stats *) L.part)[at] = a;
    uint64_t * keys = (uint64_t *) ((lp_stats *) L.part + (int64_t) L.n_rows * L.n_seg) + at * L.k;
    if (L.k) select_top(v, best, valid, id0, L.k, S, [&](int rank, uint64_t key) { keys[rank] = key; });
}

// A row's segments joined. Their lists hold n_seg * k entries in descending order; the q best of each,
// q = ceil(k / n_seg), are at least k, so entries below the smallest of the lists' q-th are out (about
// 50 of 380 stay for 19 segments and k = 20). What stays is ranked by comparing each with all.
__global__ __launch_bounds__(LP_THREADS) void logprobs_join_kernel(logprobs_launch L) {
    extern __shared__ __align__(16) uint64_t kept[];
    __shared__ lp_out o;
    __shared__ lp_stats all[LP_WAVES];
    __shared__ uint64_t least[LP_WAVES];
    __shared__ int count;
    const int r = blockIdx.x, tid = threadIdx.x, total = L.n_seg * L.k;
    const lp_stats * part = (const lp_stats *) L.part + (int64_t) r * L.n_seg;
    const uint64_t * keys = (const uint64_t *) ((const lp_stats *) L.part + (int64_t) L.n_rows * L.n_seg) + (int64_t) r * total;
    const float tok = L.tokens ? row_of(L, r)[L.tokens[r]] : 0.0f;
    // the thread's first entries, on their way while the sums join
    uint64_t first[2];
#pragma unroll
    for (int i = 0; i < 2; i++) first[i] = tid + i * LP_THREADS < total ? keys[tid + i * LP_THREADS] : 0;
    uint64_t t = ~(uint64_t) 0;
    if (L.k) {
        const int q = (L.k + L.n_seg - 1) / L.n_seg;
        for (int j = tid; j < L.n_seg; j += LP_THREADS) t = min(t, keys[(int64_t) j * L.k + q - 1]);
    }
    // the sums of this thread's segments, then of the threads' by halves
    lp_stats a{ -INFINITY, 0.0f, 0.0f, 0.0f };
    for (int j = tid; j < L.n_seg; j += LP_THREADS) a = join(a, part[j]);
#pragma unroll
    for (int h = 1; h < WAVE; h *= 2) {
        a = join(a, lp_stats{ __shfl_xor(a.m, h, WAVE), __shfl_xor(a.s, h, WAVE), __shfl_xor(a.w, h, WAVE), __shfl_xor(a.bad, h, WAVE) });
        t = min(t, (uint64_t) __shfl_xor((unsigned long long) t, h, WAVE));
    }
    if (tid % WAVE == 0) {
        all[tid / WAVE] = a;
        least[tid / WAVE] = t;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    a = join(join(all[0], all[1]), join(all[2], all[3]));
    t = min(min(least[0], least[1]), min(least[2], least[3]));
    const float ls = log_sum(a);
    if (tid == 0) put_scores(tok, a, ls, o);
    auto put = [&](int rank, uint64_t key) { put_top(L, a.m, ls, o, rank, key); };
    auto keep = [&](uint64_t key) {
        if (key < t) return;
        const int i = atomicAdd(&count, 1);
        if (i < LP_KEPT) kept[i] = key;
    };
    if (tid < total) keep(first[0]);
    if (tid + LP_THREADS < total) keep(first[1]);
    for (int i = tid + 2 * LP_THREADS; i < total; i += LP_THREADS) keep(keys[i]);
    __syncthreads();
    if (count > LP_KEPT) {
        // too many to compare each with all (a very long row, or one of whose segments nothing is left): t becomes the
        // k-th largest, by bisection; the entries differ by their ids, so k are kept
        uint64_t hi = ~(uint64_t) 0;
        int * parts = (int *) kept;
        for (int turn = 0; t < hi; turn ^= LP_WAVES) {
            const uint64_t mid = t + (hi - t) / 2 + 1;
            int n = 0;
            for (int i = tid; i < total; i += LP_THREADS) n += keys[i] >= mid ? 1 : 0;
            n = wave_sum(n);
            if (tid % WAVE == 0) parts[turn + tid / WAVE] = n;
            __syncthreads();
            n = (parts[turn] + parts[turn + 1]) + (parts[turn + 2] + parts[turn + 3]);
            if (n >= L.k) t = mid;
            else hi = mid - 1;
        }
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        for (int i = tid; i < total; i += LP_THREADS) keep(keys[i]);
        __syncthreads();
    }
    const int n = count;
    if (tid < (-n & 3)) kept[n + tid] = 0;
    __syncthreads();
    rank_keys(kept, n, L.k, put);
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
    // even segments: a short one's best entries would let the join keep most of the others' lists (5 rows of 132883,
    // 42 entries: 40 us, and 33 so)
    L.seg = ((L.n + L.n_seg - 1) / L.n_seg + 3) / 4 * 4;
    L.n_seg = (L.n + L.seg - 1) / L.seg;
    launch(logprobs_segment_kernel, dim3((unsigned) L.n_seg, (unsigned) L.n_rows),
           dim3(LP_THREADS), 0, st, L);
    if (L.n_seg > 1) {
        const size_t lds = (std::min<size_t>((size_t) L.n_seg * L.k, LP_KEPT) + 3) * 8;
        launch(logprobs_join_kernel, dim3((unsigned) L.n_rows), dim3(LP_THREADS), lds, st, L);
    }
}
