// k_attn_paged.hip — causal attention of the new tokens of several sequences over a 4-bit cache on pages.
//
// Token t of sequence s, the i-th of its n, sees positions 0 .. p = kv_len[s] - n + i:
//   o = sum_j e^(z_j - m) v_j / sum_j e^(z_j - m),  z_j = scale q . k_j,  m = max_j z_j,
// with k_j = d (c - 8) for each block of 32 codes c under one scale d, and v_j likewise.
//
// Both products run on the F16 matrix cores: the codes are small integers, exact in F16, and the other operand goes in
// as two halves (two products), which hold 22 of its 24 bits.
//   z: A = codes - 8 of 16 positions, B = 16 rows (query, head) of one KV head, a block of 32 values at a time;
//      the block's sum times the block's scale, in 32 bits.
//   o: A = codes - 8 of 16 values' columns at 32 positions, B = p d, with the scale of each position's block.
// The rows of z land in the registers as o's operand B wants them, so p never leaves its lane.
// K's dwords are exchanged between lanes so that a lane has the four values of a block that its k-index
// wants; V passes through LDS, whose transposing read gives a lane one value's codes at 16 positions.
//
// What has fewer bits than a sum of 32-bit products (half the smallest F16, 2^-25, is where halves end):
//   q: 22 bits, of values below 2^-16 of their row's largest fewer, none below 2^-38 of it;
//   few rows: p d, 22 bits, fewer below 2^-12 of the largest finite scale d that the wave has met (at positions that its
//     rows see or not), none below 2^-34 of it;
//   many: p, 22 bits, fewer below 2^-14, none below 2^-36; V in all its 15 bits, but for scales below 2^-25 of the largest
//     so far in the same place of their heads; of the four products of halves the least, at most 2^-22 p |v|, is left out.
// Errors against 64 bits are 2e-7 to 8e-7 of the output; the formula in 32-bit steps has 5e-7 to 2e-6.
//
// Few rows: 32 sequences of up to 16384 positions, 24 heads over 8 of 128, 52.4 us, 3.2 TB/s of the cache, where a copy
// reaches 4.7. Of the first launch's cycles (46 us) the vector unit has 57 % (decoding, exponentials, p's halves: some 360
// instructions a step of 32 positions), the matrix cores 15 and LDS 18; the rest is waiting, with three waves a SIMD. A
// single sequence is bound by latency (4113 positions, 32 heads over 8: 8 us and 5 for the join). Many rows: parts of 700
// tokens of two prompts over 8192 positions, 32 heads over 8 of 128, 402 us, 367 TFLOP/s of the formula's products, five
// matrix products for each two of it. The matrix cores have 38 % of the cycles, the vector unit 50, LDS 41: none is full, and
// a step's reads, products and exponentials follow one another within a wave.
#include "kernels.h"
#include "ssm_ops.h"

#include <algorithm>

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 32;               // positions of a step, few rows
constexpr int TILE_STEP = 64;          // and many
constexpr int SPLIT_WG = 256;
constexpr float M_NONE = -1.7e38f;     // the maximum of no scores: finite, so that differences are no NaN
// The maximum that p = 2^(z - m) goes by follows the scores only where they pass it by 2^SLACK: with 16 rows, one of them
// finds a new maximum in every second step, but such a one in every twentieth. What p's halves lose by it is their
// range, from below 2^-38 of the largest to below 2^-34.
constexpr int SLACK = 4;

// a value that every lane holds, as a scalar
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t) v), hi = __builtin_amdgcn_readfirstlane((uint32_t) (v >> 32));
    return (int64_t) (((uint64_t) hi << 32) | lo);
}
__device__ __forceinline__ int64_t from_lane(int64_t v, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t) v, l), hi = __builtin_amdgcn_readlane((uint32_t) (v >> 32), l);
    return (int64_t) (((uint64_t) hi << 32) | lo);
}

__device__ __forceinline__ int page_index(const paged_attn & A, int pos) { return quotient(A.by_page, pos); }

// ---- what each sequence asks for ----
struct seq_info { int first, n, len, last; };   // tokens, positions in the table; the last token sees up to `last`

__device__ __forceinline__ seq_info seq_of(const paged_attn & A, int s) {
    seq_info q;
    const int a = A.q_start[s], b = A.q_start[s + 1], kv = A.kv_len[s];
    q.first = min(max(a, 0), A.n_tokens);
    q.n = min(max(b, q.first), A.n_tokens) - q.first;
    q.len = min(max(kv, 0), A.max_pages * A.page);
    q.last = max(kv, 0) - 1;
    return q;
}

// Few rows: the steps of a sequence's whole length for each of its tiles of `rows` rows and teams of heads; of more rows
// than most, none (another launch's).
__device__ __forceinline__ int steps_of(const seq_info & q) { return max((q.len + STEP - 1) / STEP, 1); }
__device__ __forceinline__ int64_t split_units(const paged_attn & A, const seq_info & q, int rows) {
    const int n = q.n * A.group;
    return n > A.split_most ? 0 : (int64_t) ((n + rows - 1) / rows) * A.head_teams * steps_of(q);
}

// Many: of each tile, the steps that its last token sees.
__device__ __forceinline__ int tile_steps(const paged_attn & A, const seq_info & q, int rows, int tile) {
    const int i = min(quotient(A.by_group, (tile + 1) * rows - 1), q.n - 1);     // (rows are fewer than 2^30)
    const int sees = min(q.last - (q.n - 1) + i + 1, q.len);
    return max((sees + TILE_STEP - 1) / TILE_STEP, 1);
}
__device__ __forceinline__ int tiles_of(const paged_attn & A, const seq_info & q, int rows) {
    const int64_t n = (int64_t) q.n * A.group;
    return n < A.tile_least ? 0 : (int) ((n + rows - 1) / rows);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    const int lane = threadIdx.x % WAVE;
#pragma unroll
    for (int k = 1; k < WAVE; k *= 2) {
        const int64_t o = __shfl_up(v, k);
        if (lane >= k) v += o;
    }
    return v;
}

// The units of sequence s0 + lane: by each lane over its tiles, or where one has more than three times as many as there are
// sequences, by the whole wave over each sequence's (a prompt of 8192 tokens in 256 tiles, 32 heads: 1.77 ms for 1.79).
__device__ __forceinline__ int64_t tile_units(const paged_attn & A, int s0, int rows) {
    const int lane = threadIdx.x % WAVE, n = min(A.n_seqs - s0, WAVE);
    seq_info q{ 0, 0, 0, 0 };
    if (lane < n) q = seq_of(A, s0 + lane);
    const int tiles = lane < n ? tiles_of(A, q, rows) : 0;
    int64_t sum = 0;
    if (!__any(tiles > 3 * n)) {
        for (int k = 0; k < tiles; k++) sum += tile_steps(A, q, rows, k);
        return sum * A.n_head_kv;
    }
    for (int i = 0; i < n; i++) {
        const seq_info one{ 0, __builtin_amdgcn_readlane(q.n, i), __builtin_amdgcn_readlane(q.len, i), __builtin_amdgcn_readlane(q.last, i) };
        const int all = __builtin_amdgcn_readlane(tiles, i);
        int64_t mine = 0;
        for (int k = lane; k < all; k += WAVE) mine += tile_steps(A, one, rows, k);
        mine = from_lane(wave_scan(mine), WAVE - 1);
        if (lane == i) sum = mine;
    }
    return sum * A.n_head_kv;
}

// All sequences' tiles, heads and steps in one line of units; teams (of A.team waves, a KV head each) take equal
// runs of it, so that no mixture of lengths leaves a wave idle.
struct plan {
    int64_t units, base, rem;
    int teams;
    __device__ __forceinline__ void deal(int64_t all, int most) {
        units = all;
        teams = (int) max((int64_t) 1, min((int64_t) most, all));
        if (all < ((int64_t) 1 << 31)) {
            base = uniform((int) ((uint32_t) all / (uint32_t) teams));
            rem = (uint32_t) all - (uint32_t) base * (uint32_t) teams;
        } else {
            base = all / teams;
            rem = all % teams;
        }
    }
    __device__ __forceinline__ int64_t begin(int64_t t) const { return t * base + min(t, rem); }
    __device__ __forceinline__ int64_t team_of(int64_t u) const {
        const int64_t big = rem * (base + 1);
        const int64_t v = u < big ? u : u - big, d = u < big ? base + 1 : base;
        const int64_t q = v < ((int64_t) 1 << 31) && d < ((int64_t) 1 << 31) ? (int64_t) ((uint32_t) v / (uint32_t) d) : v / d;
        return u < big ? q : rem + q;
    }
};


// ---- operands ----
__device__ __forceinline__ h8 as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u4 v = { a, b, c, d };
    return __builtin_bit_cast(h8, v);
}

// codes - 8, nibbles (0, 4), (1, 5), (2, 6), (3, 7): 1024 + c or 64 + c in F16, less 1032 or 72. (The codes as F16
// subnormals, with a term for the 8, would take half as many instructions, but the matrix cores' sums of
// subnormals are exact to 1e-5 only.)
struct code_bits {
    uint32_t low = 0x64006400u, high = 0x54005400u;
    // in registers, not literals: an instruction takes a mask or them from elsewhere, not both
    __device__ __forceinline__ code_bits() { asm("" : "+v"(low), "+v"(high)); }
};
__device__ __forceinline__ h8 signed_of(uint32_t x, const code_bits & K) {
    const uint32_t y = x >> 8;
    auto low = [&](uint32_t v) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (v & 0x000F000Fu) | K.low) - h2{ 1032, 1032 }); };
    auto high = [&](uint32_t v) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (v & 0x00F000F0u) | K.high) - h2{ 72, 72 }); };
    return as_h8(low(x), high(x), low(y), high(y));
}

#define LANE_SWAP(op, a, b)                                         \
    do {                                                            \
        const auto v_ = __builtin_amdgcn_##op(a, b, false, false);  \
        a = v_[0];                                                  \
        b = v_[1];                                                  \
    } while (0)

// register k of lane group c to register c of lane group k
__device__ __forceinline__ void transpose4(uint32_t (&r)[4]) {
    LANE_SWAP(permlane32_swap, r[0], r[2]);
    LANE_SWAP(permlane32_swap, r[1], r[3]);
    LANE_SWAP(permlane16_swap, r[0], r[1]);
    LANE_SWAP(permlane16_swap, r[2], r[3]);
}

// over the four lane groups of one column
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
    uint32_t a = __float_as_uint(v), b = a;
    LANE_SWAP(permlane32_swap, a, b);
    v = f(__uint_as_float(a), __uint_as_float(b));
    a = b = __float_as_uint(v);
    LANE_SWAP(permlane16_swap, a, b);
    return f(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float column_max(float v) { return over_groups(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float column_sum(float v) { return over_groups(v, [](float a, float b) { return a + b; }); }

// the scales of a position's blocks, as loaded
template <int NB> struct scales {
    typedef uint32_t u1 __attribute__((aligned(2)));
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
    uint32_t w[2];
    __device__ __forceinline__ void load(const _Float16 * p) {
        if (NB == 4) {
            const u2 v = *(const u2 *) p;
            w[0] = v[0];
            w[1] = v[1];
        } else {
            w[0] = *(const u1 *) p;
            if (NB == 3) w[1] = ((const uint16_t *) p)[2];
        }
    }
    __device__ __forceinline__ float at(int b) const { return (float) __builtin_bit_cast(h2, w[b / 2])[b % 2]; }
};
template <bool B> struct flag { static constexpr bool value = B; };

// nothing in particular, for what is not used again
template <typename T> __device__ __forceinline__ void forget(T & v) { asm volatile("" : "=v"(v)); }

// the value of the lane N further in its row of 16, cyclically
template <int N> __device__ __forceinline__ float row_ror(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
}

// Few rows a sequence: a wave takes steps of one KV head by itself.
//
// Wide: the 16 columns of a tile are 16 rows (query, head). Narrow, for up to 16 / NB rows (4 for
// heads of 96): a column is a row and a block. A lane takes its own block's sums of each product, scales them and
// adds its neighbours', and forms p d for its own block only, which serves all blocks' products (a quarter of that
// work where a KV head has four query heads).
//
// P16: pages of whole sixteens of rows, so that a load's 16 positions are on one page, found by scalar loads.
template <int NB, bool NARROW, bool P16>
__global__ __launch_bounds__(SPLIT_WG, NARROW ? 3 : 2) void paged_split_kernel(const paged_attn args) {
    constexpr int D = NB * 32, RT = 1, COLS = NARROW ? (NB == 2 ? 8 : 4) : 16, ROWS = COLS;
    constexpr int QB = NARROW ? 1 : NB;               // blocks of a column's values: narrow, its own
    constexpr int LOADS = NB == 2 ? 1 : 2;            // 16-byte loads a lane of a step's K or V
    constexpr int SROW = STEP + 4;                    // scales of a block over a step's positions, in 32 bits
    __shared__ __align__(16) uint8_t s_v[SPLIT_WG / WAVE][STEP * NB * 16];
    __shared__ __align__(16) float s_d[SPLIT_WG / WAVE][2][NB * SROW];
    const paged_attn & A = kernargs_prefetched(args);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int col = lane % 16, c = lane / 16;         // the lane's column of a tile, its lane group
    const int own = NARROW ? min(col / COLS, NB - 1) : 0;                  // narrow: the column's block
    const bool spare = NARROW && col / COLS >= NB;
    const int team = (int) blockIdx.x * ((SPLIT_WG / WAVE) >> A.team_bits) + (wave >> A.team_bits);
    const int in_team = wave & (A.team - 1);
    const code_bits K;

    // ---- the team's run: from unit u of sequence seq on, `left` units ----
    plan P;
    int seq = 0;
    int64_t u = 0, left;
    {
        // sequences by lanes, 64 at a time; of few, one look is enough
        int64_t n = lane < A.n_seqs ? split_units(A, seq_of(A, lane), ROWS) : 0, up = wave_scan(n), all = from_lane(up, WAVE - 1);
        for (int s0 = WAVE; s0 < A.n_seqs; s0 += WAVE) {
            const int s = s0 + lane;
            all += from_lane(wave_scan(s < A.n_seqs ? split_units(A, seq_of(A, s), ROWS) : 0), WAVE - 1);
        }
        P.deal(all, A.teams);
        if (team >= P.teams) return;
        u = P.begin(team);
        left = P.begin(team + 1) - u;
        if (left <= 0) return;
        int64_t before = 0;
        uint64_t past = __ballot(up > u);
        for (int s0 = WAVE; !past && s0 < A.n_seqs; s0 += WAVE) {
            before = from_lane(up, WAVE - 1);
            const int s = s0 + lane;
            n = s < A.n_seqs ? split_units(A, seq_of(A, s), ROWS) : 0;
            up = before + wave_scan(n);
            past = __ballot(up > u);
            seq = s0;
        }
        const int l = past ? __builtin_ctzll(past) : 0;
        seq += l;
        u -= from_lane(up - n, l);
    }

    while (left > 0 && seq < A.n_seqs) {
        const seq_info Q = seq_of(A, seq);
        const int steps = steps_of(Q);
        const int tiles = Q.n * A.group > A.split_most ? 0 : (Q.n * A.group + ROWS - 1) / ROWS;
        if (u >= (int64_t) tiles * A.head_teams * steps) { seq++; u = 0; continue; }
        const int item = uniform(u < ((int64_t) 1 << 32) ? (int) ((uint32_t) u / (uint32_t) steps) : (int) (u / steps));
        const int step0 = (int) (u - (int64_t) item * steps);
        const int tile = uniform((int) ((uint32_t) item / (uint32_t) A.head_teams)), head = (item - tile * A.head_teams) * A.team + in_team;
        const int step1 = (int) min((int64_t) steps, step0 + left);
        u += step1 - step0;
        left -= step1 - step0;

        // ---- a step's operands: the rows of its positions, their bytes and scales ----
        const int32_t * table = A.pages + (int64_t) seq * A.pages_s;
        const uint8_t * kq = A.kq + (int64_t) head * A.k_head * 16, * vq = A.vq + (int64_t) head * A.v_head * 16;
        // K and V: lane (col, c) loads block c of position 16 j + col (of two blocks, 16 (c / 2) + col and c % 2)
        auto lane_of = [&](int j) { return NB == 2 ? 16 * (c >> 1) + col : 16 * j + col; };
        const int blk = NB == 2 ? (c & 1) : min(c, NB - 1);
        // scales: K's of position lane, V's of position lane - 32
        const int dpos = lane % STEP;
        const bool dv = lane >= STEP;
        const _Float16 * dp = dv ? (const _Float16 *) A.vd + (int64_t) head * A.v_head : (const _Float16 *) A.kd + (int64_t) head * A.k_head;
        const int64_t n_pages = A.n_pages, k_page = A.k_page, k_pos = A.k_pos, v_page = A.v_page, v_pos = A.v_pos;
        const int rows_page = A.page;
        // P16: a lane's place in a sixteen
        const uint32_t k_off = (uint32_t) (col * (int) k_pos + blk) * 16, v_off = (uint32_t) (col * (int) v_pos + blk) * 16;
        if (P16) dp += col * (int) (dv ? v_pos : k_pos);
        // Pages. P16: 64 table entries at a time in a register, one a lane; the next sixteen's place in the table and
        // in its page go along as scalars. Else each lane looks up its scales' position, two steps ahead.
        int held = 0, at_page = 0, at_row = 0, first_held = 0, page = -1;
        const int sixteens = rows_page >> 4, entries = (Q.len + rows_page - 1) / rows_page;
        auto hold = [&](int from) {
            first_held = from;
            held = from + lane < entries ? table[from + lane] : -1;
        };
        auto page_of = [&](int step) {
            const int pos = step * STEP + dpos;
            page = pos < Q.len && step < step1 ? table[page_index(A, pos)] : -1;
        };
        int64_t krow[2], vrow[2];    // first block of a sixteen's rows, or of the lane's
        bool there;                  // the lane's scales' position is in the cache
        uint32_t missing_next;       // positions whose page is not there
        auto locate = [&](int step) {
            const int live = Q.len - step * STEP;        // positions of the step
            uint32_t bad = 0;
            there = dpos < live;
            if (P16) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if (at_page - first_held == WAVE) hold(at_page);
                    const int id = __builtin_amdgcn_readlane(held, at_page - first_held);
                    const bool ok = (uint32_t) id < (uint32_t) n_pages;
                    if (!ok) bad |= 0xFFFFu << (16 * j);
                    const uint32_t pg = ok ? id : 0, off = ok ? at_row : 0;
                    krow[j] = (int64_t) ((uint64_t) pg * (uint32_t) k_page + (uint64_t) off * (uint32_t) k_pos);
                    vrow[j] = (int64_t) ((uint64_t) pg * (uint32_t) v_page + (uint64_t) off * (uint32_t) v_pos);
                    at_row += 16;
                    if (at_row == rows_page) { at_row = 0; at_page++; }
                }
                there = there && !((bad >> dpos) & 1);
                if (live < STEP) bad &= (1u << max(live, 0)) - 1;
            } else {
                const int p0 = step * STEP + dpos;
                const bool ok = page >= 0 && page < n_pages;
                const int off = p0 - page_index(A, p0) * rows_page;
                krow[0] = ok ? (int64_t) page * k_page + (int64_t) off * k_pos : 0;
                vrow[0] = ok ? (int64_t) page * v_page + (int64_t) off * v_pos : 0;
                bad = (uint32_t) __ballot(there && !ok);
                there = there && ok;
            }
            missing_next = bad;
        };
        auto bytes_of = [&](const uint8_t * base, const int64_t (&row)[2], uint32_t off, int j) -> const uint8_t * {
            if (!P16) return base + (__shfl(row[0], lane_of(j)) + blk) * 16;
            if (NB == 2) {
                const int64_t r0 = uniform(row[0]), r1 = uniform(row[1]);
                return base + ((c >> 1) ? r1 : r0) * 16 + off;
            }
            return base + row[j] * 16 + off;
        };
        u4 kraw[LOADS], vraw[LOADS];
        scales<NB> sd;
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < LOADS; j++) vraw[j] = *(const u4 *) bytes_of(vq, vrow, v_off, j);
            if (P16) {
                // (rows of scales are within 32 bits)
                const uint32_t k0 = uniform((int) krow[0]), k1 = uniform((int) krow[1]), v0 = uniform((int) vrow[0]), v1 = uniform((int) vrow[1]);
                const uint32_t k = (c & 1) ? k1 : k0, v = (c & 1) ? v1 : v0;
                sd.load(dp + (dv ? v : k));
            } else {
                sd.load(dp + (dv ? vrow[0] : krow[0]));
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int j = 0; j < LOADS; j++) kraw[j] = *(const u4 *) bytes_of(kq, krow, k_off, j);
        };
        if (P16) {
            const int first = step0 * (STEP / 16);
            at_page = uniform((int) ((uint32_t) first / (uint32_t) sixteens));
            at_row = (first - at_page * sixteens) * 16;
            hold(at_page);
        } else {
            page_of(step0);
        }

        // ---- the rows: two halves of each value, scaled so that a row's largest is near 2^14 ----
        h8 qh[RT][QB], ql[RT][QB];
        float fac[RT], m[RT], l[RT];
        int lim[RT];
        f4 o[RT][NB][2];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int row = tile * ROWS + t * 16 + (NARROW ? col % COLS : col);
            const bool real = row < Q.n * A.group;
            const int i = real ? quotient(A.by_group, row) : 0, g = real ? row - i * A.group : 0;
            const float * q = A.q + (int64_t) (Q.first + i) * A.q_t + (int64_t) (head * A.group + g) * A.q_h;
            // rows that are not there see what the last one sees
            lim[t] = min(Q.last - (Q.n - 1) + (real ? i : Q.n - 1), Q.len - 1);
            float big = 0.0f;
            auto values_of = [&](int b, float (&v)[8]) {
                const float4 lo = load4(q + 32 * b + 4 * c), hi = load4(q + 32 * b + 16 + 4 * c);
                const float w[8] = { lo.x, lo.z, hi.x, hi.z, lo.y, lo.w, hi.y, hi.w };
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = real && !spare ? w[k] : 0.0f;
            };
            // the row's largest value: of its own block in each column, narrow
            float v[8];
#pragma unroll
            for (int b = 0; b < QB; b++) {
                values_of(NARROW ? own : b, v);
#pragma unroll
                for (int k = 0; k < 8; k++) big = fmaxf(big, fabsf(v[k]));
            }
            if (t == 0) {
                // (behind the queries' loads)
                locate(step0);
                load_k();
                load_v();
                if (!P16) page_of(step0 + 1);
            }
            if (NARROW) {
                big = fmaxf(big, row_ror<8>(big));
                if (NB > 2) big = fmaxf(big, row_ror<4>(big));
            }
            big = column_max(big);
            const int e = big > 0.0f && big < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(big) : 0;
            const float sign = A.scale < 0.0f ? -1.0f : 1.0f;       // the factor of the sums is not negative
#pragma unroll
            for (int b = 0; b < QB; b++) {
                if (!NARROW) values_of(b, v);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float x = __builtin_amdgcn_ldexpf(v[k] * sign, e);
                    qh[t][b][k] = (_Float16) x;
                    ql[t][b][k] = (_Float16) (x - (float) qh[t][b][k]);
                }
            }
            fac[t] = fabsf(A.scale) * LOG2E * __builtin_amdgcn_ldexpf(1.0f, -e);
            m[t] = M_NONE;
            l[t] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[t][b][0] = o[t][b][1] = f4{ 0, 0, 0, 0 };
        }
        // p d is formed times 2^shift, so that the largest scale seen gives 2^13 to 2^15 times the largest p
        int shift = 38;
        // positions up to here are seen by all rows (a length may be past the table)
        const int sure = min(Q.last - (Q.n - 1) + quotient(A.by_group, tile * ROWS), Q.len - 1);

        for (int step = step0; step < step1; step++) {
            const bool more = step + 1 < step1;
            const uint32_t missing = missing_next;
            // ---- V and the scales into LDS, the next ones on their way ----
#pragma unroll
            for (int j = 0; j < LOADS; j++) *(u4 *) &s_v[wave][(lane_of(j) * NB + blk) * 16] = vraw[j];
            float dmax = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float d = there ? sd.at(b) : 0.0f;
                s_d[wave][dv][b * SROW + dpos] = d;
                dmax = fmaxf(dmax, fabsf(d));
            }
            if (!dv) dmax = 0.0f;
            if (more) {
                locate(step + 1);
                load_v();
            } else {
#pragma unroll
                for (int j = 0; j < LOADS; j++) forget(vraw[j]);
                forget(sd.w[0]);
                forget(sd.w[1]);
            }

            // ---- scores ----
            f4 s[RT][2];
#pragma unroll
            for (int j = 0; j < LOADS; j++) {
                uint32_t r[4] = { kraw[j].x, kraw[j].y, kraw[j].z, kraw[j].w };
                transpose4(r);
#pragma unroll
                for (int half = 0; half < 2 / LOADS; half++) {
                    const int t = 2 / LOADS * j + half;
                    f4 mine = { 0, 0, 0, 0 };
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const h8 a = signed_of(r[half * 2 + b], K);
                        f4 d;
                        if (!NARROW) d = *(const f4 *) &s_d[wave][0][b * SROW + 16 * t + 4 * c];
#pragma unroll
                        for (int x = 0; x < RT; x++) {
                            f4 acc = { 0, 0, 0, 0 };
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[x][NARROW ? 0 : b], acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[x][NARROW ? 0 : b], acc, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                if (NARROW) mine[i] = b == 0 || b == own ? acc[i] : mine[i];
                                else s[x][t][i] = b == 0 ? acc[i] * d[i] : fmaf(acc[i], d[i], s[x][t][i]);
                            }
                        }
                    }
                    if (NARROW) {
                        const f4 d = *(const f4 *) &s_d[wave][0][own * SROW + 16 * t + 4 * c];
#pragma unroll
                        for (int i = 0; i < 4; i++) s[0][t][i] = spare ? 0.0f : mine[i] * d[i];
                    }
                    if (NARROW) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            s[0][t][i] += row_ror<8>(s[0][t][i]);
                            if (NB > 2) s[0][t][i] += row_ror<4>(s[0][t][i]);
                        }
                    }
                }
            }
            if (more) {
                load_k();
            } else {
#pragma unroll
                for (int j = 0; j < LOADS; j++) forget(kraw[j]);
            }
            if (!P16) page_of(step + 2);
            // the largest scale of V so far
            if (__any(dmax >= __builtin_amdgcn_ldexpf(1.0f, 15 - SLACK - shift))) {
                // of those that are finite (others make the rows that see them NaN, and cost the rest no bits); 2^-24, the
                // smallest F16, where none is
                float big = 0x1p-24f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float d = fabsf(s_d[wave][1][b * SROW + dpos]);
                    if (d < INFINITY) big = fmaxf(big, d);
                }
                const int now = min(shift, 14 - SLACK - __builtin_amdgcn_frexp_expf(wave_max(big)));
                const float keep = __builtin_amdgcn_ldexpf(1.0f, now - shift);
                shift = now;
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    l[x] *= keep;
#pragma unroll
                    for (int b = 0; b < NB; b++) { o[x][b][0] *= keep; o[x][b][1] *= keep; }
                }
            }
            const bool edge = step * STEP + STEP - 1 > sure || missing;
            uint32_t hidden[RT];
#pragma unroll
            for (int x = 0; x < RT; x++) {
                hidden[x] = 0;
                if (edge) {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int k = 16 * t + 4 * c + i;
                            if (step * STEP + k > lim[x] || ((missing >> k) & 1)) {
                                s[x][t][i] = -INFINITY;
                                hidden[x] |= 1u << (4 * t + i);
                            }
                        }
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; t++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) top = fmaxf(top, s[x][t][i]);
                }
                if (__any(top * fac[x] > m[x] + SLACK)) {
                    top = column_max(top) * fac[x];
                    const float now = top > m[x] + SLACK ? top : m[x], keep = exp2_hw(m[x] - now);
                    m[x] = now;
                    l[x] *= keep;
#pragma unroll
                    for (int b = 0; b < NB; b++) { o[x][b][0] *= keep; o[x][b][1] *= keep; }
                }
                const float at = (float) shift - m[x];
#pragma unroll
                for (int t = 0; t < 2; t++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) s[x][t][i] = exp2_hw(fmaf(s[x][t][i], fac[x], at));
                }
                if (edge) {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) if ((hidden[x] >> (4 * t + i)) & 1) s[x][t][i] = 0.0f;
                    }
                }
                l[x] += ((s[x][0][0] + s[x][0][1]) + (s[x][0][2] + s[x][0][3])) + ((s[x][1][0] + s[x][1][1]) + (s[x][1][2] + s[x][1][3]));
            }

            // ---- o += p d (codes - 8), a block at a time ----
            // The transposing read takes 16 rows of 8 bytes from a lane group: its 8 positions' first halves of a
            // block, then their second; register h is half h's column of the lane at those positions.
            const uint8_t * vrow16 = &s_v[wave][(16 * ((col >> 2) & 1) + 4 * c + (col & 3)) * NB * 16 + (col >> 3) * 8];
            auto products = [&](auto at_edge) {
                constexpr bool EDGE = decltype(at_edge)::value;
                h8 ph[RT], pl[RT];
                auto weights = [&](int b) {
                    const f4 d0 = *(const f4 *) &s_d[wave][1][b * SROW + 4 * c], d1 = *(const f4 *) &s_d[wave][1][b * SROW + 16 + 4 * c];
#pragma unroll
                    for (int x = 0; x < RT; x++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                float d = t ? d1[i] : d0[i];
                                if (EDGE) d = (hidden[x] >> (4 * t + i)) & 1 ? 0.0f : d;
                                // (one product for both halves: see as_f32)
                                const float w = as_f32(s[x][t][i] * d);
                                ph[x][2 * i + t] = (_Float16) w;
                                pl[x][2 * i + t] = (_Float16) fmaf(s[x][t][i], d, -(float) ph[x][2 * i + t]);
                            }
                        }
                    }
                };
                if (NARROW) weights(own);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (!NARROW) weights(b);
                    const i2 codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i2 *) (vrow16 + b * 16));
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const h8 a = signed_of(codes[h], K);
#pragma unroll
                        for (int x = 0; x < RT; x++) {
                            o[x][b][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[x], o[x][b][h], 0, 0, 0);
                            o[x][b][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[x], o[x][b][h], 0, 0, 0);
                        }
                    }
                }
            };
            if (edge) products(flag<true>());
            else products(flag<false>());
        }

        // ---- the rows' results, or this run's part of them ----
        const bool whole = step0 == 0 && step1 == steps;
        const int64_t slot = (((int64_t) team * 2 + (step0 == 0)) * A.team + in_team) * ROWS;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const int at_row = x * 16 + (NARROW ? col % COLS : col), row = tile * ROWS + at_row;
            const float sum = column_sum(l[x]);
            if (row >= Q.n * A.group || spare) continue;
            const int i = quotient(A.by_group, row), g = row - i * A.group;
            // no positions: 0; a NaN stays one
            const float inv = whole ? (sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum) : 1.0f;
            float * out = whole ? A.out + ((int64_t) (Q.first + i) * A.n_head + head * A.group + g) * D
                                : A.part + (slot + at_row) * D;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (NARROW && b != own) continue;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    // the codes' column 4 c + r of eight bytes: value (4 c + r) / 2 of them, or 16 further
                    float * at = out + 32 * b + 8 * h + 2 * c;
                    *(float2 *) at = make_float2(o[x][b][h][0] * inv, o[x][b][h][2] * inv);
                    *(float2 *) (at + 16) = make_float2(o[x][b][h][1] * inv, o[x][b][h][3] * inv);
                }
            }
            if (!whole && c == 0 && own == 0) A.part_ml[slot + at_row] = make_float2(m[x] - (float) shift, sum);
        }
    }
}

// ---- many rows a sequence: the waves of a workgroup share a step's operands ----
//
// A workgroup takes 64 or 128 rows of one KV head, a wave 16 of them, in steps of 64 positions. Each wave decodes a block of
// the step's keys or values (of four waves, both) for all: codes - 8 of K as A wants them, and V's values
// d (codes - 8) as two halves (15 bits: exact but for the smallest scales), so that p is split once for all blocks (three products: hi hi,
// lo hi, hi lo). V's scales are taken times 2^s of each block, so that the largest so far is at 2^11 to 2^12; a scale that
// is not finite counts as 0, and makes the results of the rows that see it NaN.
template <int NB, int WAVES>
__global__ __launch_bounds__(WAVES * WAVE, WAVES == 8 ? 4 : 3) void paged_tile_kernel(const paged_attn args) {
    constexpr int D = NB * 32, RT = 1, ROWS = 16 * WAVES;
    constexpr int SROW = TILE_STEP + 4, P_UP = 15 - SLACK;
    __shared__ __align__(16) u4 s_k[NB][4][WAVE];             // block, sixteen of positions, lane
    __shared__ __align__(16) u4 s_v[NB][2][2][2][WAVE];       // block, 32 positions, half of the block, hi and lo, lane
    __shared__ __align__(16) float s_kd[NB][SROW];
    __shared__ __align__(16) _Float16 s_vd[NB][TILE_STEP];
    __shared__ int s_shift[NB];
    __shared__ uint64_t s_odd[NB], s_gone;                    // positions whose V scale is not finite; whose page is not there
    const paged_attn & A = kernargs_prefetched(args);
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int col = lane % 16, c = lane / 16;
    const code_bits K;
    const int block = wave & 3;                               // the wave's block: of K, of V, or of both
    const bool keys = wave < NB, values = (WAVES == 4 ? wave : wave - 4) >= 0 && block < NB && (WAVES == 4 || wave >= 4);
    const bool decodes = keys || values;
    float one = 1.0f;                                         // a product with it takes an F16 operand as it is
    asm("" : "+v"(one));

    plan P;
    int seq = 0;
    int64_t u = 0, left;
    {
        int64_t n = tile_units(A, 0, ROWS), up = wave_scan(n), all = from_lane(up, WAVE - 1);
        for (int s0 = WAVE; s0 < A.n_seqs; s0 += WAVE) all += from_lane(wave_scan(tile_units(A, s0, ROWS)), WAVE - 1);
        P.deal(all, A.tile_teams);
        if ((int) blockIdx.x >= P.teams) return;
        u = P.begin(blockIdx.x);
        left = P.begin(blockIdx.x + 1) - u;
        if (left <= 0) return;
        int64_t before = 0;
        uint64_t past = __ballot(up > u);
        for (int s0 = WAVE; !past && s0 < A.n_seqs; s0 += WAVE) {
            before = from_lane(up, WAVE - 1);
            n = tile_units(A, s0, ROWS);
            up = before + wave_scan(n);
            past = __ballot(up > u);
            seq = s0;
        }
        const int l = past ? __builtin_ctzll(past) : 0;
        seq += l;
        u -= from_lane(up - n, l);
    }
    // the tile of the sequence, and the unit in it (heads by steps)
    int tile = 0;
    {
        const seq_info Q = seq_of(A, seq);
        const int tiles = tiles_of(A, Q, ROWS);
        for (int k0 = 0; k0 < tiles; k0 += WAVE) {
            const int k = k0 + lane;
            const int64_t n = k < tiles ? (int64_t) tile_steps(A, Q, ROWS, k) * A.n_head_kv : 0, up = wave_scan(n);
            const uint64_t past = __ballot(up > u);
            if (past) {
                const int l = __builtin_ctzll(past);
                tile = k0 + l;
                u -= from_lane(up - n, l);
                break;
            }
            u -= from_lane(up, WAVE - 1);
        }
    }

    while (left > 0 && seq < A.n_seqs) {
        const seq_info Q = seq_of(A, seq);
        if (tile >= tiles_of(A, Q, ROWS)) { seq++; tile = 0; u = 0; continue; }
        const int steps = tile_steps(A, Q, ROWS, tile);
        if (u >= (int64_t) steps * A.n_head_kv) { tile++; u = 0; continue; }
        const int head = uniform((int) ((uint32_t) u / (uint32_t) steps)), step0 = (int) u - head * steps;
        const int step1 = (int) min((int64_t) steps, step0 + left);
        u += step1 - step0;
        left -= step1 - step0;

        // ---- the step's operands: lane l of wave b takes block b of position l ----
        const int32_t * table = A.pages + (int64_t) seq * A.pages_s;
        const int64_t k_first = (int64_t) head * A.k_head + block, v_first = (int64_t) head * A.v_head + block;
        const int n_pages = (int) min(A.n_pages, (int64_t) INT32_MAX), rows_page = A.page;
        const int64_t k_page = A.k_page, k_pos = A.k_pos, v_page = A.v_page, v_pos = A.v_pos;
        int page = -1;
        auto page_of = [&](int step) {
            const int pos = step * TILE_STEP + lane;
            page = decodes && pos < Q.len && step < step1 ? table[page_index(A, pos)] : -1;
        };
        // (of eight waves, none has both)
        u4 raw[WAVES == 8 ? 1 : 2];
        uint16_t rd[WAVES == 8 ? 1 : 2];
        u4 & kraw = raw[0], & vraw = raw[WAVES == 8 ? 0 : 1];
        uint16_t & kd = rd[0], & vd = rd[WAVES == 8 ? 0 : 1];
        bool there;
        auto load = [&](int step) {
            const int pos = step * TILE_STEP + lane;
            there = page >= 0 && page < n_pages;
            const int off = pos - page_index(A, pos) * rows_page;
            // (a cache of 2^32 blocks is 64 GiB; two prompts' parts 422 us, in 64 bits 425)
            auto row = [&](int64_t per_page, int64_t per_pos) {
                if (A.rows32) return (int64_t) (there ? (uint32_t) page * (uint32_t) per_page + (uint32_t) off * (uint32_t) per_pos : 0);
                return there ? (int64_t) page * per_page + (int64_t) off * per_pos : 0;
            };
            if (keys) {
                const int64_t at = k_first + row(k_page, k_pos);
                kraw = *(const u4 *) (A.kq + at * 16);
                kd = ((const uint16_t *) A.kd)[at];
            }
            if (values) {
                const int64_t at = v_first + row(v_page, v_pos);
                vraw = *(const u4 *) (A.vq + at * 16);
                vd = ((const uint16_t *) A.vd)[at];
            }
        };
        page_of(step0);

        // ---- the wave's rows ----
        h8 qh[RT][NB], ql[RT][NB];
        float fac[RT], m[RT], l[RT];
        int lim[RT];
        f4 o[RT][NB][2];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int row = tile * ROWS + (wave * RT + t) * 16 + col;
            const bool real = row < Q.n * A.group;
            const int i = real ? quotient(A.by_group, row) : 0, g = real ? row - i * A.group : 0;
            const float * q = A.q + (int64_t) (Q.first + i) * A.q_t + (int64_t) (head * A.group + g) * A.q_h;
            lim[t] = min(Q.last - (Q.n - 1) + (real ? i : Q.n - 1), Q.len - 1);
            float v[NB][8], big = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float4 lo = load4(q + 32 * b + 4 * c), hi = load4(q + 32 * b + 16 + 4 * c);
                const float w[8] = { lo.x, lo.z, hi.x, hi.z, lo.y, lo.w, hi.y, hi.w };
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    v[b][k] = real ? w[k] : 0.0f;
                    big = fmaxf(big, fabsf(v[b][k]));
                }
            }
            if (t == 0 && decodes) {
                load(step0);
                page_of(step0 + 1);
            }
            big = column_max(big);
            const int e = big > 0.0f && big < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(big) : 0;
            const float sign = A.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float x = __builtin_amdgcn_ldexpf(v[b][k] * sign, e);
                    qh[t][b][k] = (_Float16) x;
                    ql[t][b][k] = (_Float16) (x - (float) qh[t][b][k]);
                }
            }
            fac[t] = fabsf(A.scale) * LOG2E * __builtin_amdgcn_ldexpf(1.0f, -e);
            m[t] = M_NONE;
            l[t] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[t][b][0] = o[t][b][1] = f4{ 0, 0, 0, 0 };
        }
        const int first_row = tile * ROWS + wave * RT * 16;
        const int sure = min(Q.last - (Q.n - 1) + min(quotient(A.by_group, first_row), Q.n - 1), Q.len - 1);
        int own_shift = 38, shift[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) shift[b] = 38;

        for (int step = step0; step < step1; step++) {
            __syncthreads();                              // the operands before these are read
            if (keys) {
                s_kd[block][lane] = there ? (float) __builtin_bit_cast(_Float16, kd) : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) s_k[block][lane / 16][k * 16 + col] = __builtin_bit_cast(u4, signed_of(kraw[k], K));
                const uint64_t gone = __ballot(step * TILE_STEP + lane < Q.len && !there);
                if (wave == 0 && lane == 0) s_gone = gone;
            }
            if (values) {
                const float dr = (float) __builtin_bit_cast(_Float16, vd);
                const bool finite = fabsf(dr) < INFINITY;
                const float dv = there && finite ? fabsf(dr) : 0.0f;
                if (__any(dv >= __builtin_amdgcn_ldexpf(1.0f, 12 - own_shift))) {
                    const float big = wave_max(dv);
                    own_shift = min(own_shift, 12 - __builtin_amdgcn_frexp_expf(big));
                }
                // scales of positions 16 t + 4 c + r side by side over t
                s_vd[block][(lane & 32) + ((lane >> 2) & 3) * 8 + (lane & 3) * 2 + ((lane >> 4) & 1)] =
                    there && finite ? (_Float16) __builtin_amdgcn_ldexpf(dr, own_shift) : (_Float16) 0.0f;
                const uint64_t odd = __ballot(there && !finite);
                if (lane == 0) {
                    s_shift[block] = own_shift;
                    s_odd[block] = odd;
                }
                // V's bytes where its values will be, read again by the transposing read
                uint8_t * bytes = (uint8_t *) &s_v[block][0][0][0][0];
                *(u4 *) (bytes + lane * 16) = vraw;
                i2 codes[2];
#pragma unroll
                for (int hs = 0; hs < 2; hs++) {
                    codes[hs] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                        (__attribute__((address_space(3))) i2 *) (bytes + (32 * hs + 16 * ((col >> 2) & 1) + 4 * c + (col & 3)) * 16 + (col >> 3) * 8));
                }
                u4 d[2];
#pragma unroll
                for (int hs = 0; hs < 2; hs++) d[hs] = *(const u4 *) &s_vd[block][32 * hs + c * 8];
                // (these reads are before the writes: one wave's LDS operations keep their order)
#pragma unroll
                for (int hs = 0; hs < 2; hs++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const h8 a = signed_of(codes[hs][h], K), dd = __builtin_bit_cast(h8, d[hs]);
                        const h8 hi = a * dd, lo = __builtin_elementwise_fma(a, dd, -hi);
                        s_v[block][hs][h][0][lane] = __builtin_bit_cast(u4, hi);
                        s_v[block][hs][h][1][lane] = __builtin_bit_cast(u4, lo);
                    }
                }
            }
            if (decodes && step + 1 < step1) {
                load(step + 1);
                page_of(step + 2);
            }
            __syncthreads();                              // the step's operands are there

            if (first_row >= Q.n * A.group) continue;     // no rows: the wave only decodes
            uint64_t odd = 0;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                odd |= (uint64_t) uniform((int64_t) s_odd[b]);
                const int now = uniform(s_shift[b]);
                if (now != shift[b]) {
                    const float keep = __builtin_amdgcn_ldexpf(1.0f, now - shift[b]);
                    shift[b] = now;
#pragma unroll
                    for (int x = 0; x < RT; x++) { o[x][b][0] *= keep; o[x][b][1] *= keep; }
                }
            }
#pragma unroll 1
            for (int hs = 0; hs < 2; hs++) {
                const int at = step * TILE_STEP + 32 * hs;
                f4 s[RT][2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    __builtin_amdgcn_sched_barrier(0);       // (16 reads at once would not leave their registers)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const h8 a = __builtin_bit_cast(h8, s_k[b][2 * hs + t][lane]);
                        const f4 d = *(const f4 *) &s_kd[b][32 * hs + 16 * t + 4 * c];
#pragma unroll
                        for (int x = 0; x < RT; x++) {
                            f4 acc = { 0, 0, 0, 0 };
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[x][b], acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[x][b], acc, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 4; i++) s[x][t][i] = b == 0 ? acc[i] * d[i] : fmaf(acc[i], d[i], s[x][t][i]);
                        }
                    }
                }
                // positions on missing pages have scales of 0 but scores all the same: their rows' bits
                const uint32_t missing = (uint32_t) ((uint64_t) uniform((int64_t) s_gone) >> (32 * hs));
                const bool edge = at + 31 > sure || missing;
                uint32_t hidden[RT];
                h8 ph[RT], pl[RT];
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    hidden[x] = 0;
                    if (edge) {
#pragma unroll
                        for (int t = 0; t < 2; t++) {
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int k = 16 * t + 4 * c + i;
                                if (at + k > lim[x] || ((missing >> k) & 1)) {
                                    s[x][t][i] = -INFINITY;
                                    hidden[x] |= 1u << (4 * t + i);
                                }
                            }
                        }
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 2; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) top = fmaxf(top, s[x][t][i]);
                    }
                    if (__any(top * fac[x] > m[x] + SLACK)) {
                        top = column_max(top) * fac[x];
                        const float now = top > m[x] + SLACK ? top : m[x], keep = exp2_hw(m[x] - now);
                        m[x] = now;
                        l[x] *= keep;
#pragma unroll
                        for (int b = 0; b < NB; b++) { o[x][b][0] *= keep; o[x][b][1] *= keep; }
                    }
                    // p times 2^P_UP, so that the largest is below 2^15
                    const float up = (float) P_UP - m[x];
#pragma unroll
                    for (int t = 0; t < 2; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) s[x][t][i] = exp2_hw(fmaf(s[x][t][i], fac[x], up));
                    }
                    if (edge) {
#pragma unroll
                        for (int t = 0; t < 2; t++) {
#pragma unroll
                            for (int i = 0; i < 4; i++) if ((hidden[x] >> (4 * t + i)) & 1) s[x][t][i] = 0.0f;
                        }
                    }
                    l[x] += ((s[x][0][0] + s[x][0][1]) + (s[x][0][2] + s[x][0][3])) + ((s[x][1][0] + s[x][1][1]) + (s[x][1][2] + s[x][1][3]));
#pragma unroll
                    for (int i = 0; i < 4; i++) {
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            ph[x][2 * i + t] = (_Float16) s[x][t][i];
                            pl[x][2 * i + t] = (_Float16) fmaf(s[x][t][i], one, -(float) ph[x][2 * i + t]);
                        }
                    }
                }
                if (odd) {
                    // a scale that is not finite at a position that the row sees
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint32_t bits = (uint32_t) (s_odd[b] >> (32 * hs));
#pragma unroll
                        for (int x = 0; x < RT; x++) {
                            bool sees = false;
#pragma unroll
                            for (int t = 0; t < 2; t++) {
#pragma unroll
                                for (int i = 0; i < 4; i++) sees |= ((bits >> (16 * t + 4 * c + i)) & 1) && !((hidden[x] >> (4 * t + i)) & 1);
                            }
                            if (column_max(sees ? 1.0f : 0.0f) > 0.0f) o[x][b][0] = o[x][b][1] = f4{ NAN, NAN, NAN, NAN };
                        }
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (b == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const h8 hi = __builtin_bit_cast(h8, s_v[b][hs][h][0][lane]), lo = __builtin_bit_cast(h8, s_v[b][hs][h][1][lane]);
#pragma unroll
                        for (int x = 0; x < RT; x++) {
                            o[x][b][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, ph[x], o[x][b][h], 0, 0, 0);
                            o[x][b][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pl[x], o[x][b][h], 0, 0, 0);
                            o[x][b][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ph[x], o[x][b][h], 0, 0, 0);
                        }
                    }
                }
            }
        }

        // ---- the rows' results, or this run's part of them ----
        const bool whole = step0 == 0 && step1 == steps;
        const int64_t slot = ((int64_t) blockIdx.x * 2 + (step0 == 0)) * ROWS;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const int at_row = (wave * RT + x) * 16 + col, row = tile * ROWS + at_row;
            const float sum = __builtin_amdgcn_ldexpf(column_sum(l[x]), -P_UP);
            if (row >= Q.n * A.group) continue;
            const int i = quotient(A.by_group, row), g = row - i * A.group;
            const float inv = whole ? (sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum) : 1.0f;
            float * out = whole ? A.out + ((int64_t) (Q.first + i) * A.n_head + head * A.group + g) * D
                                : A.tile_part + (slot + at_row) * D;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                // (in two steps: 2^-(P_UP + shift) may be below the range where inv is large)
                const float w = __builtin_amdgcn_ldexpf(inv, -P_UP);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float r[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) r[k] = __builtin_amdgcn_ldexpf(o[x][b][h][k], -shift[b]) * w;
                    float * at = out + 32 * b + 8 * h + 2 * c;
                    *(float2 *) at = make_float2(r[0], r[2]);
                    *(float2 *) (at + 16) = make_float2(r[1], r[3]);
                }
            }
            if (!whole && c == 0) A.tile_ml[slot + at_row] = make_float2(m[x], sum);
        }
    }
}

// parts of one row, four values of it: o = sum_k 2^(m_k - m) o_k, l likewise
struct part_sum {
    float m = M_NONE, l = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    // parts from, from + by, .. up to last, N of them loaded at a time; at(k): row of part k
    template <int N, typename F>
    __device__ __forceinline__ void add(const float * part, const float2 * part_ml, F at, int D, int e, int64_t from, int64_t last, int by) {
        for (int64_t k0 = from; k0 <= last; k0 += N * by) {
            float2 ml[N];
            float4 v[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int64_t r = at(min(k0 + i * by, last));
                ml[i] = part_ml[r];
                v[i] = *(const float4 *) (part + r * D + 4 * e);
            }
            float now = m;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (k0 + i * by > last) ml[i] = make_float2(M_NONE, 0.0f);
                now = fmaxf(now, ml[i].x);
            }
            const float was = exp2_hw(m - now);
            l *= was;
            o.x *= was;
            o.y *= was;
            o.z *= was;
            o.w *= was;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (k0 + i * by > last) continue;
                const float is = exp2_hw(ml[i].x - now);
                l = fmaf(ml[i].y, is, l);
                o.x = fmaf(v[i].x, is, o.x);
                o.y = fmaf(v[i].y, is, o.y);
                o.z = fmaf(v[i].z, is, o.z);
                o.w = fmaf(v[i].w, is, o.w);
            }
            m = now;
        }
    }
};

// The same by teams: of many tokens few rows have parts. A workgroup looks at the item that its team ends in (its first wave
// does, for all), and joins the item's rows if the team began it and did not finish it. in_team: the team's wave, or of
// TILE's rows the sixteens that it starts with, `by` apart.
struct item_parts { int seq, tile, head; int64_t last; };
template <int SPLIT, int TILE>
__device__ __forceinline__ bool parts_of(const paged_attn & A, int64_t me, int in_team, item_parts & I) {
    constexpr int ROWS = SPLIT ? SPLIT : TILE;
    const int lane = threadIdx.x % WAVE;
    auto units = [&](int s0) {
        if (!SPLIT) return tile_units(A, s0, ROWS);
        return s0 + lane < A.n_seqs ? split_units(A, seq_of(A, s0 + lane), ROWS) : (int64_t) 0;
    };
    int64_t n = units(0), up = wave_scan(n), all = from_lane(up, WAVE - 1);
    for (int s0 = WAVE; s0 < A.n_seqs; s0 += WAVE) all += from_lane(wave_scan(units(s0)), WAVE - 1);
    plan P;
    P.deal(all, SPLIT ? A.teams : A.tile_teams);
    if (me >= P.teams) return false;
    const int64_t begin = P.begin(me), end = P.begin(me + 1);
    if (begin >= end) return false;
    const int64_t u = end - 1;
    uint64_t past = __ballot(up > u);
    int s0 = 0;
    while (!past && s0 + WAVE < A.n_seqs) {
        s0 += WAVE;
        n = units(s0);
        up = from_lane(up, WAVE - 1) + wave_scan(n);
        past = __ballot(up > u);
    }
    if (!past) return false;
    I.seq = s0 + __builtin_ctzll(past);
    int64_t before = from_lane(up - n, __builtin_ctzll(past));
    const seq_info Q = seq_of(A, I.seq);
    auto over = [](int64_t a, int b) { return a < ((int64_t) 1 << 32) ? (int) ((uint32_t) a / (uint32_t) b) : (int) (a / b); };
    int steps;
    if (SPLIT) {
        steps = steps_of(Q);
        const int item = over(u - before, steps);
        I.tile = item / A.head_teams;
        I.head = (item - I.tile * A.head_teams) * A.team + in_team;
        before += (int64_t) item * steps;
    } else {
        const int tiles = tiles_of(A, Q, ROWS);
        I.tile = 0;
        for (int k0 = 0; k0 < tiles; k0 += WAVE) {
            n = k0 + lane < tiles ? (int64_t) tile_steps(A, Q, ROWS, k0 + lane) * A.n_head_kv : 0;
            up = before + wave_scan(n);
            past = __ballot(up > u);
            if (past) {
                I.tile = k0 + __builtin_ctzll(past);
                before = from_lane(up - n, __builtin_ctzll(past));
                break;
            }
            before = from_lane(up, WAVE - 1);
        }
        steps = tile_steps(A, Q, ROWS, I.tile);
        I.head = over(u - before, steps);
        before += (int64_t) I.head * steps;
    }
    if (before < begin || before + steps <= end) return false;
    I.last = P.team_of(before + steps - 1);
    return true;
}
template <int NB, int SPLIT, int TILE>
__device__ __forceinline__ void join_team(const paged_attn & A, int64_t me, int in_team, int by) {
    constexpr int D = NB * 32, PER = D / 4, GROUPS = 256 / PER, ROWS = SPLIT ? SPLIT : TILE;
    __shared__ item_parts s_item;
    __shared__ bool s_any;
    const int t = threadIdx.x;
    if (t < WAVE) {
        item_parts I;
        const bool any = parts_of<SPLIT, TILE>(A, me, in_team, I);
        if (t == 0) { s_any = any; s_item = I; }
    }
    __syncthreads();
    if (!s_any) return;
    const item_parts I = s_item;
    const seq_info Q = seq_of(A, I.seq);
    const float * part = SPLIT ? A.part : A.tile_part;
    const float2 * part_ml = SPLIT ? A.part_ml : A.tile_ml;
    const int group = t / PER, e = t % PER, rows = min(ROWS, Q.n * A.group - I.tile * ROWS), team = SPLIT ? A.team : 1;
    for (int r = group + (SPLIT ? 0 : in_team * GROUPS); group < GROUPS && r < rows; r += GROUPS * (SPLIT ? 1 : by)) {
        part_sum S;
        S.add<4>(part, part_ml, [&](int64_t k) { return ((k * 2 + (k == me)) * team + (SPLIT ? in_team : 0)) * ROWS + r; }, D, e, me, I.last, 1);
        const int row = I.tile * ROWS + r, i = quotient(A.by_group, row), g = row - i * A.group;
        const float inv = S.l > 0.0f ? 1.0f / S.l : S.l == 0.0f ? 0.0f : S.l;
        *(float4 *) (A.out + ((int64_t) (Q.first + i) * A.n_head + I.head * A.group + g) * D + 4 * e) =
            make_float4(S.o.x * inv, S.o.y * inv, S.o.z * inv, S.o.w * inv);
    }
}
// BY workgroups a tile launch's team, and (SPLIT) one a wave of a split launch's behind them
template <int NB, int SPLIT, int TILE, int BY>
__global__ __launch_bounds__(256) void paged_join_teams_kernel(const paged_attn args) {
    const paged_attn & A = kernargs_prefetched(args);
    if ((int) blockIdx.y < BY) join_team<NB, 0, TILE>(A, blockIdx.x, blockIdx.y, BY);
    else if (SPLIT) join_team<NB, SPLIT ? SPLIT : 16, 0>(A, blockIdx.x, blockIdx.y - BY, 0);
}

// Rows whose steps several teams took: their parts joined, a workgroup a row (or COLS columns of it), COLS / 4 threads
// a part. A row is a split launch's (SPLIT rows a tile) or a tile launch's (TILE rows), by its sequence's rows.
template <int NB, int SPLIT, int TILE, int COLS>
__global__ __launch_bounds__(256) void paged_join_kernel(const paged_attn args) {
    const paged_attn & A = kernargs_prefetched(args);
    constexpr int D = NB * 32, PER = COLS / 4, GROUPS = 256 / PER;
    constexpr int SUMS = COLS < D ? 256 / WAVE : GROUPS;      // groups whose sums meet in shared memory
    __shared__ float4 s_o[SUMS][PER];
    __shared__ float2 s_ml[SUMS];
    const int token = blockIdx.x, head = blockIdx.y, t = threadIdx.x, lane = t % WAVE;
    // the token's sequence, and the units before it in either line
    int seq = -1;
    int64_t all_s = 0, all_t = 0, begin_s = 0, begin_t = 0;
    for (int s0 = 0; s0 < A.n_seqs; s0 += WAVE) {
        const int s = s0 + lane;
        bool mine = false;
        int64_t ns = 0, nt = 0;
        if (s < A.n_seqs) {
            const seq_info q = seq_of(A, s);
            mine = token >= q.first && token < q.first + q.n;
            if (SPLIT) ns = split_units(A, q, SPLIT);
        }
        if (TILE) nt = tile_units(A, s0, TILE);
        const uint64_t b = __ballot(mine);
        const int l = b ? __builtin_ctzll(b) : 0;
        const bool first = b && seq < 0;
        if (first) seq = s0 + l;
        if (SPLIT) {
            const int64_t up = wave_scan(ns);
            if (first) begin_s = all_s + from_lane(up - ns, l);
            all_s += from_lane(up, WAVE - 1);
        }
        if (TILE) {
            const int64_t up = wave_scan(nt);
            if (first) begin_t = all_t + from_lane(up - nt, l);
            all_t += from_lane(up, WAVE - 1);
        }
    }
    if (seq < 0) return;
    const seq_info Q = seq_of(A, seq);
    const bool tiled = TILE && (!SPLIT || (int64_t) Q.n * A.group >= A.tile_least);
    const int kvh = quotient(A.by_group, head), row = (token - Q.first) * A.group + head - kvh * A.group;
    const int rows = tiled ? TILE : SPLIT, tile = row / rows, team = tiled ? 1 : A.team;
    plan P;
    P.deal(tiled ? all_t : all_s, tiled ? A.tile_teams : A.teams);
    int64_t a;
    int steps;
    if (tiled) {
        steps = tile_steps(A, Q, rows, tile);
        a = begin_t + (int64_t) kvh * steps;
        for (int k = 0; k < tile; k++) a += (int64_t) tile_steps(A, Q, rows, k) * A.n_head_kv;
    } else {
        steps = steps_of(Q);
        a = begin_s + ((int64_t) tile * A.head_teams + kvh / team) * steps;
    }
    const int64_t t0 = P.team_of(a), t1 = P.team_of(a + steps - 1);
    if (t0 == t1) return;                               // written whole
    const float * part = tiled ? A.tile_part : A.part;
    const float2 * part_ml = tiled ? A.tile_ml : A.part_ml;
    const int group = t / PER, e = t % PER, e0 = COLS < D ? (int) blockIdx.z * PER : 0;
    part_sum S;
    if (group < GROUPS) {
        S.add<COLS < D ? 8 : 4>(part, part_ml, [&](int64_t k) { return ((k * 2 + (k == t0)) * team + kvh % team) * rows + row - tile * rows; }, D, e0 + e, t0 + group, t1, GROUPS);
        if (COLS < D) {                                 // a wave's groups first
#pragma unroll
            for (int k = PER; k < WAVE; k *= 2) {
                const float m = __shfl_xor(S.m, k), now = fmaxf(S.m, m), was = exp2_hw(S.m - now), is = exp2_hw(m - now);
                S.l = fmaf(S.l, was, __shfl_xor(S.l, k) * is);
                S.o.x = fmaf(S.o.x, was, __shfl_xor(S.o.x, k) * is);
                S.o.y = fmaf(S.o.y, was, __shfl_xor(S.o.y, k) * is);
                S.o.z = fmaf(S.o.z, was, __shfl_xor(S.o.z, k) * is);
                S.o.w = fmaf(S.o.w, was, __shfl_xor(S.o.w, k) * is);
                S.m = now;
            }
        }
        const int at = COLS < D ? t / WAVE : group;
        if (COLS == D || lane < PER) {
            s_o[at][e] = S.o;
            if (e == 0) s_ml[at] = make_float2(S.m, S.l);
        }
    }
    __syncthreads();
    if (t >= PER) return;
    float top = M_NONE, l = 0.0f;
    for (int k = 0; k < SUMS; k++) top = fmaxf(top, s_ml[k].x);
    float4 o = make_float4(0, 0, 0, 0);
    for (int k = 0; k < SUMS; k++) {
        const float w = exp2_hw(s_ml[k].x - top);
        const float4 v = s_o[k][t];
        l += s_ml[k].y * w;
        o.x += v.x * w;
        o.y += v.y * w;
        o.z += v.z * w;
        o.w += v.w * w;
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    *(float4 *) (A.out + ((int64_t) token * A.n_head + head) * D + 4 * (e0 + t)) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// Rows a sequence on average. Up to 8 (of heads of 64) or 4 go narrow (32 sequences of 4096 positions, 32 heads over 8 of
// 128: 43 us, wide 50), up to 16 wide, a wave by itself (3 tokens each of 16 such sequences: 37 us, in tiles of 64 53), more
// in tiles: of 64, and of 128 where there are many (8 sequences' 50 tokens 119 us in tiles of 64 and 123 of 128, 150 254 and
// 227, one's 200 71 and 90). Past 64 rows the sequences among them that have 16 or fewer go by waves: 31 single tokens beside
// a prompt of 700 109 us, 319 all in tiles; what it costs where there are none is two launches' 8 us.
// The lengths are the device's, so the average is all that the host knows of a mixture, and below 64 rows it chooses badly
// where a prompt's part is among many single tokens. Over 4000 positions, 32 heads over 8, the part's and the tokens' nodes by
// themselves for one of both: 31 tokens and 512 161 us for 170 (by waves and in tiles), 34 and 512 164 for 207 and 48 and
// 512 176 for 239 (all in tiles), 199 and 500 357 for 438 (all by waves).
struct paged_ways { int split, tile; };      // rows of a tile, 0: no such launch
paged_ways ways_of(const paged_attn & A) {
    const int narrow = A.D == 64 ? 8 : 4;
    const int64_t rows = (int64_t) A.n_tokens * A.group, per = A.n_seqs;
    if (rows <= narrow * per && A.group <= narrow) return { narrow, 0 };
    if (rows <= 16 * per) return { 16, 0 };
    if (rows <= 64 * per) return { 0, 64 };
    return { per > 1 ? 16 : 0, (int64_t) A.n_tokens * A.n_head <= 24576 ? 64 : 128 };
}
// workgroups that the CUs hold at once: more would run behind the first
int split_wgs(int rows) { return rows < 16 ? 768 : 512; }
int tile_wgs(int rows) { return rows == 64 ? 768 : 512; }

template <int NB, bool NARROW>
void split(const paged_attn & A, hipStream_t st) {
    // A sixteen of positions on one page, its rows within 32-bit offsets: wide, 3 tokens of 8 sequences over 4000 positions
    // 28.6 us for 30.0; narrow, a lane's own look-up is as fast or faster (one token of 8 sequences, 32 heads of 96: 17.2
    // for 18.4).
    const int64_t reach = 16 * 16 * std::max(A.k_pos, A.v_pos);
    const dim3 grid(split_wgs(NARROW ? 4 : 16));
    if (!NARROW && A.page % 16 == 0 && A.rows32 && reach <= INT32_MAX) launch(paged_split_kernel<NB, NARROW, !NARROW>, grid, dim3(SPLIT_WG), 0, st, A);
    else launch(paged_split_kernel<NB, NARROW, false>, grid, dim3(SPLIT_WG), 0, st, A);
}

constexpr int64_t JOIN_FEW = 512;
constexpr int JOIN_BY = 4, JOIN_MANY = 4096;
template <int NB>
void attend(const paged_attn & A, const paged_ways & W, hipStream_t st) {
    constexpr int narrow = NB == 2 ? 8 : 4;
    if (W.tile == 64) launch(paged_tile_kernel<NB, 4>, dim3(tile_wgs(64)), dim3(4 * WAVE), 0, st, A);
    else if (W.tile == 128) launch(paged_tile_kernel<NB, 8>, dim3(tile_wgs(128)), dim3(8 * WAVE), 0, st, A);
    if (W.split == narrow) split<NB, true>(A, st);
    else if (W.split == 16) split<NB, false>(A, st);
    const dim3 grid(A.n_tokens, A.n_head);
    // By teams, where rows are many: of 32 heads over 8 of 128, 250 tokens over 250 positions take 25 us with all launches, and
    // joined by rows, whose workgroups take 2 us even where they find nothing to join, 41; 60 tokens over 4000, with few rows
    // and many parts, 75 and 45.
    if (W.tile && ((int64_t) A.n_tokens * A.n_head > JOIN_MANY || W.tile == 128)) {
        const int most = std::max(A.teams, A.tile_teams);
        if (W.tile == 64 && W.split) launch(paged_join_teams_kernel<NB, 16, 64, JOIN_BY>, dim3(most, JOIN_BY + A.team), dim3(256), 0, st, A);
        else if (W.tile == 64) launch(paged_join_teams_kernel<NB, 0, 64, JOIN_BY>, dim3(A.tile_teams, JOIN_BY), dim3(256), 0, st, A);
        else if (W.split) launch(paged_join_teams_kernel<NB, 16, 128, JOIN_BY>, dim3(most, JOIN_BY + A.team), dim3(256), 0, st, A);
        else launch(paged_join_teams_kernel<NB, 0, 128, JOIN_BY>, dim3(A.tile_teams, JOIN_BY), dim3(256), 0, st, A);
        return;
    }
    // Of few rows, whose parts are many, a workgroup joins 32 columns: one sequence of 30000 positions, 32 heads of 128,
    // 21.8 us with both launches for 28.4 by rows; of 16 sequences (2048 such workgroups) by rows 18.6 for 22.9.
    constexpr int D = NB * 32;
    if (!(W.split && W.tile) && (int64_t) A.n_tokens * A.n_head * NB <= JOIN_FEW) {
        const dim3 columns(A.n_tokens, A.n_head, NB);
        if (W.split == narrow) launch(paged_join_kernel<NB, narrow, 0, 32>, columns, dim3(256), 0, st, A);
        else if (W.split) launch(paged_join_kernel<NB, 16, 0, 32>, columns, dim3(256), 0, st, A);
        else launch(paged_join_kernel<NB, 0, 64, 32>, columns, dim3(256), 0, st, A);
        return;
    }
    if (W.split == narrow) launch(paged_join_kernel<NB, narrow, 0, D>, grid, dim3(256), 0, st, A);
    else if (!W.tile) launch(paged_join_kernel<NB, 16, 0, D>, grid, dim3(256), 0, st, A);
    else if (W.split) launch(paged_join_kernel<NB, 16, 64, D>, grid, dim3(256), 0, st, A);
    else launch(paged_join_kernel<NB, 0, 64, D>, grid, dim3(256), 0, st, A);
}

// rows of parts: two a team of waves, or a workgroup
int64_t split_rows(const paged_ways & W) { return W.split ? (int64_t) split_wgs(W.split) * (SPLIT_WG / WAVE) * 2 * W.split : 0; }
int64_t tile_rows(const paged_ways & W) { return W.tile ? (int64_t) tile_wgs(W.tile) * 2 * W.tile : 0; }

} // namespace

int64_t paged_attn_scratch_bytes(const paged_attn & A) {
    if (A.n_tokens == 0 || A.n_seqs == 0 || A.n_head == 0) return 0;
    const paged_ways W = ways_of(A);
    return (split_rows(W) + tile_rows(W)) * (A.D * 4 + 8);
}

void launch_paged_attn(paged_attn A, hipStream_t st) {
    if (A.n_tokens == 0 || A.n_seqs == 0 || A.n_head == 0) return;
    const paged_ways W = ways_of(A);
    A.team = A.n_head_kv % 4 == 0 ? 4 : A.n_head_kv % 2 == 0 ? 2 : 1;
    A.team_bits = A.team / 2;
    A.head_teams = A.n_head_kv / A.team;
    A.teams = W.split ? split_wgs(W.split) * (SPLIT_WG / WAVE) / A.team : 0;
    A.tile_teams = W.tile ? tile_wgs(W.tile) : 0;
    A.split_most = W.tile ? 16 : INT32_MAX;
    A.tile_least = W.split ? 17 : 0;
    // a row's first block as a 32-bit number
    const int64_t most = std::max({ A.k_page, A.v_page, A.k_pos * A.page, A.v_pos * A.page });
    A.rows32 = most <= UINT32_MAX && A.n_pages <= (int64_t) UINT32_MAX / std::max<int64_t>(most, 1) - 1;
    A.by_page = divisor::by(A.page);
    A.by_group = divisor::by(A.group);
    A.part = (float *) A.scratch;
    A.part_ml = (float2 *) (A.part + split_rows(W) * A.D);
    A.tile_part = (float *) (A.part_ml + split_rows(W));
    A.tile_ml = (float2 *) (A.tile_part + tile_rows(W) * A.D);
    if (A.D == 64) attend<2>(A, W, st);
    else if (A.D == 96) attend<3>(A, W, st);
    else if (A.D == 128) attend<4>(A, W, st);
    else HIP_ABORT("flash_attn_paged: heads of %d values", A.D);
}
