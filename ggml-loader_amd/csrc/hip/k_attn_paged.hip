// k_attn_paged.hip — causal attention of the new tokens of several sequences over a 4-bit cache on pages.
//
// Token t of sequence s, the i-th of its n, sees positions 0 .. p = kv_len[s] - n + i:
//   o = sum_j e^(z_j - m) v_j / sum_j e^(z_j - m),  z_j = scale q . k_j,  m = max_j z_j,
// with k_j = d (c - 8) for each block of 32 codes c under one scale d, and v_j likewise.
#include "kernels.h"
#include "ssm_ops.h"

namespace {

// the sequence that token t belongs to, or -1, and its range of tokens
__device__ __forceinline__ int sequence_of(const paged_attn & A, int t, int & first, int & n) {
    for (int s = 0; s < A.n_seqs; s++) {
        const int a = min(max(A.q_start[s], 0), A.n_tokens), b = min(max(A.q_start[s + 1], a), A.n_tokens);
        if (t >= a && t < b) { first = a; n = b - a; return s; }
    }
    return -1;
}

template <int D>
__global__ __launch_bounds__(64) void attn_paged_kernel(const paged_attn A) {
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int kvh = h / (A.n_head / A.n_head_kv);
    int first, n;
    const int s = sequence_of(A, t, first, n);
    if (s < 0) return;
    const int len = min(A.kv_len[s], A.max_pages * A.page);
    const int see = min(A.kv_len[s] - n + (t - first) + 1, len);
    __shared__ float q[D];
    for (int i = lane; i < D; i += 64) q[i] = A.q[t * A.q_t + h * A.q_h + i] * A.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[(D + 63) / 64] = {};
    for (int j0 = 0; j0 < see; j0 += 64) {
        const int j = j0 + lane;
        int64_t page = -1;
        if (j < see) page = A.pages[s * A.pages_s + j / A.page];
        float z = -INFINITY;
        const bool there = page >= 0 && page < A.n_pages;
        const int64_t row = there ? page : 0;
        if (there) {
            const int64_t b0 = page * A.k_page + (j % A.page) * A.k_pos + kvh * A.k_head;
            z = 0.0f;
            for (int b = 0; b < D / 32; b++) {
                float part = 0.0f;
                for (int i = 0; i < 16; i++) {
                    const int c = A.kq[(b0 + b) * 16 + i];
                    part += q[32 * b + i] * (float) ((c & 15) - 8) + q[32 * b + 16 + i] * (float) ((c >> 4) - 8);
                }
                z += part * __half2float(A.kd[b0 + b]);
            }
        }
        const float big = fmaxf(m, wave_max(z));
        if (big == -INFINITY) continue;
        const float p = there ? exp2_hw((z - big) * LOG2E) : 0.0f, keep = exp2_hw((m - big) * LOG2E);
        l = l * keep + group_sum<64>(p);
        m = big;
        for (int k = 0; k < (D + 63) / 64; k++) o[k] *= keep;
        for (int i = 0; i < 64; i++) {
            const float w = lane_f(p, i);
            if (w == 0.0f) continue;
            const int64_t pg = __shfl(row, i);
            const int64_t b0 = pg * A.v_page + ((j0 + i) % A.page) * A.v_pos + kvh * A.v_head;
            for (int k = 0; k < (D + 63) / 64; k++) {
                const int e = lane + 64 * k;
                if (e >= D) continue;
                const int c = A.vq[(b0 + e / 32) * 16 + e % 16], code = e % 32 < 16 ? c & 15 : c >> 4;
                o[k] += w * (float) (code - 8) * __half2float(A.vd[b0 + e / 32]);
            }
        }
    }
    for (int k = 0; k < (D + 63) / 64; k++) {
        const int e = lane + 64 * k;
        if (e < D) A.out[((int64_t) t * A.n_head + h) * D + e] = l > 0.0f ? o[k] / l : l == 0.0f ? 0.0f : l;
    }
}

} // namespace

int64_t paged_attn_scratch_bytes(const paged_attn & A) { (void) A; return 0; }

void launch_paged_attn(const paged_attn & A, hipStream_t st) {
    if (A.n_tokens == 0 || A.n_seqs == 0 || A.n_head == 0) return;
    const dim3 grid(A.n_tokens, A.n_head);
    if (A.D == 64) launch(attn_paged_kernel<64>, grid, dim3(64), 0, st, A);
    else if (A.D == 96) launch(attn_paged_kernel<96>, grid, dim3(64), 0, st, A);
    else if (A.D == 128) launch(attn_paged_kernel<128>, grid, dim3(64), 0, st, A);
    else HIP_ABORT("flash_attn_paged: heads of %d values", A.D);
}
