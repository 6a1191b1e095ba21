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
// threads form once for all heads. Bound by launch and load latency for a few tokens (16 tokens' 40 heads of 128
// rotated: 6 us with their launch); 2100 tokens of 32 + 8 heads of 128 rotate in 26 us, 3.3 TB/s; 4096 tokens of 8 heads
// of 128, K rotated and both into 4 bits, take 25 us in two rounds of workgroups (34 KB of LDS and 128 registers: four a CU), whose
// waves wait for 55 % of their cycles: loads, indices, cosines and stores follow one another.
//
// Of rows with one index the last is stored: a workgroup looks its indices up among the later ones of its
// pass (at most ROWS_PASS rows; passes follow one another on the stream).
#include "kernels.h"
#include "tview_ops.h"

#include <algorithm>

namespace {

constexpr int ROWS_WG = ROWS_PIECE / 4;
constexpr int ROWS_MAX_PER_WG = 32;               // rows of 8 threads

__device__ __forceinline__ int64_t row_index(const rows_job & J, int64_t at) {
    return J.idx64 ? ((const int64_t *) J.idx)[at] : (int64_t) ((const int32_t *) J.idx)[at];
}

// A value of a pair, rotated: x cos -+ mate sin, minus for the pair's first. (In 32 bits the steps are rope_ext's, whose
// second values add the products in the other order.)
__device__ __forceinline__ float rotated(double x, double mate, bool first, double2 cs) {
    return (float) fma(x, cs.x, (first ? -cs.y : cs.y) * mate);
}
__device__ __forceinline__ float rotated_f32(float x, float mate, bool first, double2 cs) {
    const float c = (float) cs.x, s = (float) cs.y;
    return x * c + mate * (first ? -s : s);
}

// a value's 16 bits as F16 or BF16
__device__ __forceinline__ uint32_t bits16(int type, float v) {
    if (type == GGML_TYPE_F16) return __half_as_ushort(__float2half_rn(as_f32(v)));
    const uint32_t u = __float_as_uint(as_f32(v));
    return (u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 64u : (u + (0x7fffu + ((u >> 16) & 1u))) >> 16;
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

// UNITS: pieces of 256 threads' values that a workgroup takes: of one row where rows are longer, else rows
template <int UNITS>
__global__ __launch_bounds__(ROWS_WG, 4) void rows_kernel(const rows_batch args) {
    __shared__ double2 s_cs[UNITS * ROWS_MAX_CS];
    __shared__ int64_t s_at[UNITS * ROWS_MAX_PER_WG];
    __shared__ int s_dead[UNITS * ROWS_MAX_PER_WG];
    const rows_batch & B = kernargs_prefetched(args);
    const int t = threadIdx.x;
    int j = 0;
#pragma unroll
    for (int k = 1; k < ROWS_MAX_JOBS; k++) if (k < B.n_jobs && (int64_t) blockIdx.x >= B.job[k].first_wg) j = k;
    const rows_job & J = B.job[j];
    const int wg = (int) (blockIdx.x - J.first_wg);
    const int64_t i2 = blockIdx.y, i3 = blockIdx.z;
    // the workgroup's rows, and the thread's row and quad of values of each unit
    const bool pieces = J.chunks > 1;
    const int parts = (J.chunks + UNITS - 1) / UNITS, per = pieces ? 1 : UNITS * J.per_wg;
    const int64_t row0 = pieces ? wg / parts : (int64_t) wg * per;
    const int n_rows = (int) min((int64_t) per, J.rows - row0);
    const int chunk0 = pieces ? (wg - (int) row0 * parts) * UNITS : 0, lr0 = pieces ? 0 : t / J.threads, quad0 = pieces ? t : t - lr0 * J.threads;
    const bool apart = J.rope && J.dist > 1;                      // pairs (i, i + dist), else neighbours
    auto row_of = [&](int u) { return pieces ? 0 : lr0 < J.per_wg ? u * J.per_wg + lr0 : n_rows; };
    auto quad_of = [&](int u) { return pieces ? (chunk0 + u) * ROWS_WG + t : quad0; };
    auto mine_of = [&](int u) { return row_of(u) < n_rows && quad_of(u) * 4 < J.width; };

    // the rows' values, and the other values of their pairs
    float own[UNITS][4], other[UNITS][4];
    int w0[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const int e0 = mine_of(u) ? quad_of(u) * 4 : 0;
        const int64_t row = J.row0 + row0 + min(row_of(u), n_rows - 1);
        const char * src = J.src + row * J.s1 + i2 * J.s2 + i3 * J.s3;
        const int head = J.rope ? quotient(J.by_head, e0) : 0;
        w0[u] = e0 - head * J.head;
        const float * x = (const float *) (src + head * J.s_head);
        const int n = min(4, J.width - e0);
        if (J.quads) {
            const float4 a = load4(x + w0[u]);
            own[u][0] = a.x; own[u][1] = a.y; own[u][2] = a.z; own[u][3] = a.w;
            if (apart) {
                // (values that have no pair read their own again)
                const float4 b = load4(x + (w0[u] < 2 * J.pairs ? (w0[u] < J.pairs ? w0[u] + J.dist : w0[u] - J.dist) : w0[u]));
                other[u][0] = b.x; other[u][1] = b.y; other[u][2] = b.z; other[u][3] = b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = e0 + min(i, n - 1), h = e / J.head, w = e - h * J.head;
                const float * xh = (const float *) (src + h * J.s_head);
                own[u][i] = xh[w];
                other[u][i] = xh[J.rope && w < 2 * J.pairs ? (apart ? (w < J.pairs ? w + J.dist : w - J.dist) : w ^ 1) : w];
            }
        }
    }

    if (J.idx) {
        const int64_t idx0 = J.row0 + (i2 % J.c_n2) * J.c2 + (i3 % J.c_n3) * J.c3;
        if (t < n_rows) {
            s_at[t] = row_index(J, idx0 + row0 + t);
            s_dead[t] = s_at[t] < 0 || s_at[t] >= J.to_rows;
        }
        __syncthreads();
        // a later row of the pass with the same index: of the workgroup's own, and of those behind them, whose lookups
        // go eight at a time where they are many (a pass has fewer than 2^31 rows)
        if (t < n_rows) {
            for (int k = 0; k < t; k++) if (s_at[k] == s_at[t]) s_dead[k] = 1;
        }
        const int last = (int) J.rows - 1;
        int r = (int) row0 + n_rows + t;
        for (const bool many = last - r + t >= 8 * ROWS_WG; many && r <= last; r += 8 * ROWS_WG) {
            int64_t at[8];
#pragma unroll
            for (int i = 0; i < 8; i++) at[i] = row_index(J, idx0 + min(r + i * ROWS_WG, last));
            for (int k = 0; k < n_rows; k++) {
                const int64_t mine = s_at[k];
                bool same = false;
#pragma unroll
                for (int i = 0; i < 8; i++) same |= at[i] == mine;
                if (same) s_dead[k] = 1;
            }
        }
        for (; r <= last; r += ROWS_WG) {
            const int64_t at = row_index(J, idx0 + r);
            for (int k = 0; k < n_rows; k++) if (s_at[k] == at) s_dead[k] = 1;
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

#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const bool mine = mine_of(u);
        const int lr = min(row_of(u), n_rows - 1), e0 = mine ? quad_of(u) * 4 : 0, n = min(4, J.width - e0);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = own[u][i];
        if (J.rope) {
            const double2 * cs = s_cs + lr * J.pairs;
            const bool multi = J.rope == ROWS_ROPE_MULTI;
            if (J.quads) {
                // a quad lies in one half of the pairs, in pairs of neighbours, or past them
                if (w0[u] < 2 * J.pairs) {
                    const bool first = w0[u] < J.pairs;
                    const double2 * at = cs + (apart ? (first ? w0[u] : w0[u] - J.dist) : w0[u] / 2);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const double2 c = at[apart ? i : i / 2];
                        const float mate = apart ? other[u][i] : own[u][i ^ 1];
                        const bool f = apart ? first : !(i & 1);
                        v[i] = multi ? rotated(own[u][i], mate, f, c) : rotated_f32(own[u][i], mate, f, c);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int w = (e0 + min(i, n - 1)) % J.head;
                    if (w >= 2 * J.pairs) continue;
                    const bool first = apart ? w < J.pairs : !(w & 1);
                    const double2 c = cs[apart ? (first ? w : w - J.dist) : w / 2];
                    v[i] = multi ? rotated(own[u][i], other[u][i], first, c) : rotated_f32(own[u][i], other[u][i], first, c);
                }
            }
        }
        if (!mine || (J.idx && s_dead[lr])) continue;
        const int64_t to = J.idx ? s_at[lr] : J.row0 + row0 + lr;
        if (J.type == GGML_TYPE_Q4_0 || J.type == GGML_TYPE_Q8_0) {
            const int64_t block = J.first_block + to * J.d1 + i2 * J.d2 + i3 * J.d3 + e0 / 32;
            if (J.type == GGML_TYPE_Q4_0) store_q4_0(J, block, v, t % 8);
            else store_q8_0(J, block, v, t % 8);
            continue;
        }
        char * out = J.dst + to * J.d1 + i2 * J.d2 + i3 * J.d3;
        if (J.wide && n == 4) {
            if (J.type == GGML_TYPE_F32) {
                *(float4 *) (out + (int64_t) e0 * 4) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; i++) h[i] = bits16(J.type, v[i]);
                *(uint2 *) (out + (int64_t) e0 * 2) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
            }
        } else {
            const int size = J.type == GGML_TYPE_F32 ? 4 : 2;
#pragma unroll
            for (int i = 0; i < 4; i++) if (i < n) st(out + (int64_t) (e0 + i) * size, J.type, v[i]);
        }
    }
}

} // namespace

static void rows_shape(rows_job & J) {
    if (J.rope && (J.pairs > ROWS_MAX_CS || J.pairs * 2 > J.head)) HIP_ABORT("rows: %d pairs of heads of %d values", J.pairs, J.head);
    const int quads = (int) (((int64_t) J.width + 3) / 4);
    J.chunks = (quads + ROWS_WG - 1) / ROWS_WG;
    J.threads = J.chunks > 1 ? ROWS_WG : std::max((quads + 7) / 8 * 8, 8);
    J.per_wg = J.chunks > 1 ? 1 : ROWS_WG / J.threads;
    J.by_head = divisor::by(std::max(J.head, 1));
    J.quads = J.width % 4 == 0 && J.head % 4 == 0 && (!J.rope || (J.dist > 1 ? J.pairs % 4 == 0 && J.dist % 4 == 0 : J.pairs % 2 == 0));
    if (J.type == GGML_TYPE_Q4_0 || J.type == GGML_TYPE_Q8_0) return;
    const int size = J.type == GGML_TYPE_F32 ? 16 : 8;
    J.wide = ((uintptr_t) J.dst | (uintptr_t) J.d1 | (uintptr_t) J.d2 | (uintptr_t) J.d3) % size == 0;
}

static int64_t rows_wgs(const rows_job & J, int units) {
    if (J.width == 0) return 0;
    if (J.chunks > 1) return J.rows * ((J.chunks + units - 1) / units);
    const int64_t per = (int64_t) units * J.per_wg;
    return (J.rows + per - 1) / per;
}

static void launch_units(const rows_batch & B, int units, dim3 grid, hipStream_t st) {
    if (units == 1) launch(rows_kernel<1>, grid, dim3(ROWS_WG), 0, st, B);
    else launch(rows_kernel<4>, grid, dim3(ROWS_WG), 0, st, B);
}

// One launch for jobs of up to ROWS_PASS rows that have no third and fourth extent; else a job and a pass at a time.
// Four units a workgroup where one would give more than ROWS_MANY workgroups: a token's cosines and the search for equal
// indices then serve four times the values (2100 tokens of 40 heads of 128 rotate in 26 us, by one unit in 38); of few tokens
// one, so that all CUs have some (96 tokens' append into F16 5.5 us, by four 9.2).
constexpr int64_t ROWS_MANY = 2048;
void launch_rows(rows_batch & B, hipStream_t st) {
    bool together = true;
    int64_t all = 0;
    for (int k = 0; k < B.n_jobs; k++) {
        rows_shape(B.job[k]);
        together = together && B.job[k].n2 == 1 && B.job[k].n3 == 1 && (!B.job[k].idx || B.job[k].rows <= ROWS_PASS);
        all += rows_wgs(B.job[k], 1);
    }
    const int units = all > ROWS_MANY ? 4 : 1;
    all = 0;
    for (int k = 0; k < B.n_jobs; k++) {
        B.job[k].first_wg = all;
        all += rows_wgs(B.job[k], units);
    }
    if (together && all <= INT32_MAX) {
        if (all > 0) launch_units(B, units, dim3((unsigned) all), st);
        return;
    }
    for (int k = 0; k < B.n_jobs; k++) {
        rows_batch one = B;
        one.n_jobs = 1;
        one.job[0] = B.job[k];
        rows_job & J = one.job[0];
        J.first_wg = 0;
        const int64_t n = J.rows;
        for (int64_t r = 0; r < n && J.width > 0 && J.n2 * J.n3 > 0; r += ROWS_PASS) {
            J.row0 = r;
            J.rows = std::min<int64_t>(ROWS_PASS, n - r);
            launch_units(one, units, dim3((unsigned) rows_wgs(J, units), (unsigned) J.n2, (unsigned) J.n3), st);
        }
    }
}
