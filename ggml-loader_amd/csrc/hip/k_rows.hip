// k_rows.hip — rows rotated by positions (of one axis or several) and stored where an index says: the
// rotation of queries, and the append of keys and values to a paged cache.
//
// Pair i of a row turns by the angle t = pos[axis(i)] f(i): (a, b) -> (a cos t - b sin t, a sin t + b cos t).
// For several axes t is formed as turns, t / 2 pi = pos * (f / 2 pi), in 64 bits, so that only its fraction
// meets the sine: a position of 10^6 keeps 10 digits of it, where a 32-bit product keeps two. The rotation is
// formed in 64 bits too and rounded once. (ggml_rope_ext's rows, whose floats are ggml-cpu's, keep its
// 32-bit steps.)
//
// A thread holds four values of a row and its pair's other four (read twice, the second time from the
// cache), eight threads one block of a quantized row; a workgroup 1024 values, whose tokens' cosines its
// threads form once for all heads. Bound by launch and load latency for a few tokens (4096 tokens of 8 heads
// of 128, K rotated and both into 4 bits: see the figures at launch_rows).
//
// Of rows with one index the last is stored: a workgroup looks its indices up among the later ones of its
// pass (at most ROWS_PASS rows; passes follow one another on the stream).
#include "kernels.h"
#include "tview_ops.h"

#include <algorithm>

namespace {

constexpr int ROWS_WG = 256;
constexpr int ROWS_MAX_PER_WG = 32;               // rows of 8 threads
constexpr int ROWS_MAX_CS = 512;                  // rows x pairs of a workgroup: a row has at least pairs / 2 threads

__device__ __forceinline__ int64_t row_index(const rows_job & J, int64_t at) {
    return J.idx64 ? ((const int64_t *) J.idx)[at] : (int64_t) ((const int32_t *) J.idx)[at];
}

// value w of a head, rotated: a and b are the pair's values, first says whether w is the pair's first
__device__ __forceinline__ float rotated(double a, double b, bool first, double2 cs) {
    return (float) (first ? a * cs.x - b * cs.y : a * cs.y + b * cs.x);
}
__device__ __forceinline__ float rotated_f32(float a, float b, bool first, double2 cs) {
    const float c = (float) cs.x, s = (float) cs.y;
    return first ? a * c - b * s : a * s + b * c;
}

__device__ __forceinline__ int min8_dpp(int v) {
    v = min(v, dpp_i<0xB1>(v));
    v = min(v, dpp_i<0x4E>(v));
    return min(v, dpp_i<0x141>(v));
}

// A block of 32 values over eight threads as Q4_0: the scale is the value of largest magnitude (the first of
// equals) over -8, so that it takes the code 0; codes round half up and stop at 15. A NaN makes the scale one.
__device__ __forceinline__ void store_q4_0(const rows_job & J, int64_t block, const float * v, int lane8) {
    float big = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    big = max8_dpp(big);
    int key = 64, nan = 0;
#pragma unroll
    for (int i = 3; i >= 0; i--) {
        if (fabsf(v[i]) == big) key = (lane8 * 4 + i) * 2 + (v[i] < 0.0f);
        nan |= v[i] != v[i];
    }
    key = min8_dpp(key);
    nan = sum8_dpp(nan);
    const float d = ((key & 1) ? -big : big) / -8.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = as_f32(v[i] * id) + 8.5f;
        packed |= (uint32_t) min(max((int) x, 0), 15) << (8 * i);
    }
    // byte j of a block holds values j (low) and j + 16 (high): threads 0 to 3 take the codes of 4 to 7
    const uint32_t high = (uint32_t) dpp_i<0x1B>(dpp_i<0x141>((int) packed));
    if (lane8 < 4) *(uint32_t *) (J.qs + block * Q4_0_QS + lane8 * 4) = packed | (high << 4);
    if (lane8 == 0) J.d[block] = nan ? __ushort_as_half(0x7e00) : __float2half_rn(as_f32(d));
}

// as Q8_0: the scale is the largest magnitude over 127, codes round half away from zero
__device__ __forceinline__ void store_q8_0(const rows_job & J, int64_t block, const float * v, int lane8) {
    float big = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    big = max8_dpp(big);
    int nan = 0;
    const float d = big / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        nan |= v[i] != v[i];
        packed |= (uint32_t) (min(max((int) roundf(as_f32(v[i] * id)), -127), 127) & 0xff) << (8 * i);
    }
    nan = sum8_dpp(nan);
    *(uint32_t *) (J.qs + block * Q8_0_QS + lane8 * 4) = packed;
    if (lane8 == 0) J.d[block] = nan ? __ushort_as_half(0x7e00) : __float2half_rn(as_f32(d));
}

__global__ __launch_bounds__(ROWS_WG) void rows_kernel(const rows_batch B) {
    __shared__ double2 s_cs[ROWS_MAX_CS];
    __shared__ int64_t s_at[ROWS_MAX_PER_WG];
    __shared__ int s_dead[ROWS_MAX_PER_WG];
    int j = 0;
#pragma unroll
    for (int k = 1; k < ROWS_MAX_JOBS; k++) if (k < B.n_jobs && (int64_t) blockIdx.x >= B.job[k].first_wg) j = k;
    const rows_job & J = B.job[j];
    const int t = threadIdx.x, wg = (int) (blockIdx.x - J.first_wg);
    const int64_t i2 = blockIdx.y, i3 = blockIdx.z;
    // the thread's row of the workgroup's, and its quad of values in it
    int lr = 0, quad;
    int64_t row0;
    if (J.chunks > 1) {
        row0 = wg / J.chunks;
        quad = (wg % J.chunks) * ROWS_WG + t;
    } else {
        row0 = (int64_t) wg * J.per_wg;
        lr = t / J.threads;
        quad = t % J.threads;
    }
    const int n_rows = (int) min((int64_t) J.per_wg, J.rows - row0);
    const int64_t row = J.row0 + row0 + min(lr, n_rows - 1);
    const bool mine = lr < n_rows && quad * 4 < J.width;
    const int e0 = mine ? quad * 4 : 0;

    // the row's values, and the other values of their pairs
    const char * src = J.src + row * J.s1 + i2 * J.s2 + i3 * J.s3;
    const int head = e0 / J.head, w0 = e0 - head * J.head;
    const float * x = (const float *) (src + head * J.s_head);
    float own[4], other[4] = { 0, 0, 0, 0 };
    const int n = min(4, J.width - e0);
    const bool apart = J.rope && J.dist > 1;                      // pairs (i, i + dist), else neighbours
    if (J.quads) {
        const float4 a = load4(x + w0);
        own[0] = a.x; own[1] = a.y; own[2] = a.z; own[3] = a.w;
        if (apart && w0 < 2 * J.pairs) {
            const float4 b = load4(x + (w0 < J.pairs ? w0 + J.dist : w0 - J.dist));
            other[0] = b.x; other[1] = b.y; other[2] = b.z; other[3] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = e0 + min(i, n - 1), h = e / J.head, w = e - h * J.head;
            const float * xh = (const float *) (src + h * J.s_head);
            own[i] = xh[w];
            if (J.rope && w < 2 * J.pairs) other[i] = xh[apart ? (w < J.pairs ? w + J.dist : w - J.dist) : w ^ 1];
        }
    }

    int64_t to = row;
    if (J.idx) {
        if (t < n_rows) {
            s_at[t] = row_index(J, J.row0 + row0 + t + (i2 % J.c_n2) * J.c2 + (i3 % J.c_n3) * J.c3);
            s_dead[t] = s_at[t] < 0 || s_at[t] >= J.to_rows;
        }
        __syncthreads();
        to = s_at[min(lr, n_rows - 1)];
        // a later row of the pass with the same index
        const int64_t base = J.row0 + (i2 % J.c_n2) * J.c2 + (i3 % J.c_n3) * J.c3;
        for (int64_t r = row0 + 1 + t; r < J.rows; r += ROWS_WG) {
            const int64_t at = row_index(J, base + r);
            for (int k = 0; k < n_rows && row0 + k < r; k++) if (at == s_at[k]) s_dead[k] = 1;
        }
    }
    if (J.rope) {
        for (int k = t; k < n_rows * J.pairs; k += ROWS_WG) {
            const int r = k / J.pairs, p = k - r * J.pairs;
            const int64_t tok = J.row0 + row0 + r;
            double2 cs;
            if (J.rope == ROWS_ROPE_MULTI) {
                double turns = (double) J.pos[B.axis[p] * J.n_pos + tok] * B.turns[p];
                if (J.ff) turns /= (double) J.ff[p];
                turns -= rint(turns);
                double s, c;
                sincospi(2.0 * turns, &s, &c);
                cs = make_double2(c * B.scale, s * B.scale);
            } else if (J.cs) {
                const float2 f = J.cs[tok * J.pairs + p];
                cs = make_double2(f.x, f.y);
            } else {
                float c, s;
                rope_pair_cs(B.p, J.ff, J.pos[tok], p, c, s);
                cs = make_double2(c, s);
            }
            s_cs[k] = cs;
        }
    }
    if (J.idx || J.rope) __syncthreads();

    const double2 * cs = s_cs + min(lr, n_rows - 1) * J.pairs;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[i] = own[i];
        if (!J.rope) continue;
        const int w = J.quads ? w0 + i : (e0 + min(i, n - 1)) % J.head;
        if (w >= 2 * J.pairs) continue;
        const float mate = apart || !J.quads ? other[i] : own[i ^ 1];
        const bool first = apart ? w < J.pairs : !(w & 1);
        const double2 c = cs[apart ? (first ? w : w - J.dist) : w / 2];
        const float a = first ? v[i] : mate, b = first ? mate : v[i];
        v[i] = J.rope == ROWS_ROPE_MULTI ? rotated(a, b, first, c) : rotated_f32(a, b, first, c);
    }

    if (!mine || (J.idx && s_dead[lr])) return;
    if (J.type == GGML_TYPE_Q4_0 || J.type == GGML_TYPE_Q8_0) {
        const int64_t block = J.first_block + to * J.d1 + i2 * J.d2 + i3 * J.d3 + e0 / 32;
        if (J.type == GGML_TYPE_Q4_0) store_q4_0(J, block, v, t % 8);
        else store_q8_0(J, block, v, t % 8);
        return;
    }
    char * out = J.dst + to * J.d1 + i2 * J.d2 + i3 * J.d3;
    if (J.wide && n == 4) {
        if (J.type == GGML_TYPE_F32) {
            *(float4 *) (out + (int64_t) e0 * 4) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint16_t h[4];
#pragma unroll
            for (int i = 0; i < 4; i++) st((char *) &h[i], J.type, v[i]);
            *(uint2 *) (out + (int64_t) e0 * 2) = make_uint2(h[0] | (uint32_t) h[1] << 16, h[2] | (uint32_t) h[3] << 16);
        }
    } else {
        const int size = J.type == GGML_TYPE_F32 ? 4 : 2;
#pragma unroll
        for (int i = 0; i < 4; i++) if (i < n) st(out + (int64_t) (e0 + i) * size, J.type, v[i]);
    }
}

} // namespace

void rows_shape(rows_job & J) {
    const int quads = (int) ((J.width + 3) / 4);
    J.chunks = (quads + ROWS_WG - 1) / ROWS_WG;
    J.threads = J.chunks > 1 ? ROWS_WG : (quads + 7) / 8 * 8;
    J.per_wg = J.chunks > 1 ? 1 : ROWS_WG / J.threads;
    J.quads = J.width % 4 == 0 && J.head % 4 == 0 && (!J.rope || (J.dist > 1 ? J.pairs % 4 == 0 && J.dist % 4 == 0 : J.pairs % 2 == 0));
    if (J.type == GGML_TYPE_Q4_0 || J.type == GGML_TYPE_Q8_0) return;
    const int size = J.type == GGML_TYPE_F32 ? 16 : 8;
    J.wide = ((uintptr_t) J.dst | (uintptr_t) J.d1 | (uintptr_t) J.d2 | (uintptr_t) J.d3) % size == 0;
}

// One launch for jobs of up to ROWS_PASS rows that have no third and fourth extent; else a job and a pass at a time.
void launch_rows(rows_batch & B, hipStream_t st) {
    bool together = true;
    for (int k = 0; k < B.n_jobs; k++) {
        rows_shape(B.job[k]);
        together = together && B.job[k].n2 == 1 && B.job[k].n3 == 1 && (!B.job[k].idx || B.job[k].rows <= ROWS_PASS);
    }
    auto wgs = [](const rows_job & J) { return J.chunks > 1 ? J.rows * J.chunks : (J.rows + J.per_wg - 1) / J.per_wg; };
    if (together) {
        int64_t all = 0;
        for (int k = 0; k < B.n_jobs; k++) {
            B.job[k].first_wg = all;
            all += wgs(B.job[k]);
        }
        if (all > 0 && all <= INT32_MAX) {
            launch(rows_kernel, dim3((unsigned) all), dim3(ROWS_WG), 0, st, B);
            return;
        }
    }
    for (int k = 0; k < B.n_jobs; k++) {
        rows_batch one = B;
        one.n_jobs = 1;
        one.job[0] = B.job[k];
        rows_job & J = one.job[0];
        J.first_wg = 0;
        const int64_t n = J.rows;
        for (int64_t r = 0; r < n && J.n2 * J.n3 > 0; r += ROWS_PASS) {
            J.row0 = r;
            J.rows = std::min<int64_t>(ROWS_PASS, n - r);
            launch(rows_kernel, dim3((unsigned) wgs(J), (unsigned) J.n2, (unsigned) J.n3), dim3(ROWS_WG), 0, st, one);
        }
    }
}
