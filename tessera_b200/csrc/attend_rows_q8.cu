// Ragged attention over kept rows in 8 bits, whole slots or listed blocks.
//
// A tile is up to 16 query rows, (token, head) pairs: the G heads of a kv head's group times up to T = 16 / G neighbouring
// rows that are the next positions of one slot (drafted tokens, a part of a prompt).  Both products run on warp MMAs with
// the keys, then the channels, as the 16 rows and the queries as the 8 columns:
//     S^T[16 keys x 8 queries] = K Q^T        m16n8k32, s8 in, s32 out
//     O^T[16 channels x 8 queries] += V^T P^T m16n8k16, f16 in, f32 out
// so that a decode row of up to eight heads wastes nothing of the accumulators, and a second eight of queries shares the
// loaded K and the converted V.  (With the queries as rows, half of every accumulator quad of a decode row is padding.)
//
// K goes into its product as it lies, without a conversion: a query row becomes whole numbers of 15 bits and a sign,
// Q = round(q * 32639 / max |q|), in two signed digits Q = 256 q1 + q0, each a product of its own; the sums are exact in 32
// bits (256 * 32639 * 127 < 2^31) and rounded once.  What it saves is half of all instructions (two conversions for every pair of codes).
// What it costs is the rounding of q to 2^-16 of the row's largest magnitude, which so sets the error of every element: with
// keys of unit variance and a scale of 1 / sqrt(W) a score is off by 9e-6 max |q| (one sigma).  That is less than f16 costs a
// probability (2e-4) up to 24 times the others' root mean square, and less than bf16 costs the output (1e-3) up to 120 times.
// After a per-head norm the largest is at most sqrt(W) <= 16 times it, gains aside.  V's codes become f16, which holds them exactly: the bytes are set as the low bits of 1024 + (128 + code) and
// 1152 is subtracted.
//
// The scales leave the products alone.  With s = raw * scale * k_scale in powers of two and
//     x = s + log2(v_scale),   M ~ max x - 7,   P = 2^(x - M)   (f16 operand of P V)
// the output is sum(P code) / sum(P / v_scale): the block's value scale rides in the exponent, so that P needs no second
// factor and stays within f16's range whatever the scales are, and M cancels.  A scale of zero counts as 2^-60, the
// smallest that append writes.  (The second sum is f32: a block whose value scale is below 2^-126 of another's, with
// values of 10^38 beside ordinary ones, drops out of it.)
//
// What feeds it.  Every warp is a worker of its own: it streams a step's codes (4 KB of K, 4 KB of V: 32 keys of width
// 128) into its own ring with TMA, so that no warp waits for another and the only barrier is the one a copy completes on.
// Lanes look up the pool's blocks and their scales 32 blocks at a time, one group ahead.  TMA swizzles the tiles (16-byte
// pieces XORed with the row), which makes every ldmatrix read free of bank conflicts: K as it lies, V transposed in
// 16-bit units (two channels), whose bytes the conversion separates.
//
// How the work is shared out.  The steps of all tiles, laid end to end, are cut into equal runs, one a worker: lengths
// may be as uneven as they like.  A run has at most one tile that began before it and one that goes on after it, so a
// worker leaves at most two partial results (M, sum, output) in the workspace; tiles that lie within a run go straight
// to the output.  A second kernel folds the partials of a tile in the order of their keys: no atomics, the same bits on
// every run.
//
// What bounds it, measured with width 128.  Many decode rows: the codes' bytes (64 rows of up to 8192 keys, 8 kv heads of 2
// heads: 139 us, 0.89 of the copy rate; 4 rows of up to 100003 keys, 8 kv heads of 4: 112 us, 0.88; 140 and 113 where the
// board's power limit holds the clock at 1.67 GHz).  Listed blocks: the same, in blocks that lie scattered, with a merge (64 rows x 4 kv heads x 64 blocks of 64: 58 us, 0.70).
// Drafted tokens, where 16 queries share each key: the instructions around the products (16 slots x 7 rows of up to 4099 keys,
// 4 kv heads of 8: 53 us, 0.15 of the copy rate, an instruction in a third of the cycles from two warps a scheduler, which
// is what their registers leave).  Fewer instructions a step also draw less power: at the board's limit, where the clock
// gives way, 64 x 8192 went from 150 us to 142 with one look-up, copy and scale a step and two stages.
// Width 256: sixteen queries' accumulators and digits do not fit 255 registers (840 and 932 bytes spill, in the cluster's
// kernel 148 and 156).  A decode batch, which has one group of eight, is still bound by its bytes (32 rows of up to 8192
// keys, 8 kv heads of 2: 145 us, 0.86); two groups are not (2 kv heads of 16: 83 us, 0.38; 16 x 7 drafted rows of up to
// 4099 keys, 4 kv heads of 8: 114 us, 0.15).
#include <cmath>

#include "rows_q8.cuh"
#include "ts_ptx.cuh"

namespace ts {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kHalfStage = 4096, kStage = 2 * kHalfStage;  // K codes, then V codes
__device__ constexpr uint32_t kRuns[6] = {1, 2, 3, 4, 6, 8};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kScaleFloor = 8.673617379884035e-19f;  // 2^-60

// Eight warps, with two stages each, have 128 KB an SM under way, several times what the memory's latency asks for.  A third
// stage made the reads less orderly and slower (64 rows x 8192 positions: 145 us against 140).  Twelve warps leave 168
// registers a thread, which spills (156 us), six warps hide too little of a step's arithmetic (149).  Runs at the end that
// whoever is done first claims from a counter even out the SMs' shares of the memory's rate, but cost what they gain.
constexpr int kBlocks = 2, kStages = 2;

struct AttendParams {
    const uint16_t *q;
    RowsQ8Dev kv;
    const uint32_t *ids;  // NULL: whole slots
    uint16_t *out;
    const uint32_t *slots, *positions;
    uint32_t rows, keys, heads, kv_heads, back, count;
    uint32_t group, part, parts;  // heads per kv head; heads of it in a tile, tiles it takes
    uint32_t tokens;              // rows a tile may hold
    uint32_t most;                // tile rows a partial has room for: tokens * part
    uint32_t workers;
    int merged;                   // whether the second kernel runs
    uint32_t whole;               // without it: every tile counts as this many steps and is never cut
    uint32_t cluster;             // blocks of a cluster that has a row and kv head to itself; 0: the other kernels
    float scale;
    float *part_o;    // [workers, 2, most, W]
    float *part_ml;   // [workers, 2, most, 2]
    uint4 *places;    // [rows, kv_heads * parts]: first and last worker of the row's tile, slot of the first, tile row
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t v;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
    uint32_t v;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
    uint32_t v;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Two of the four biased codes (code + 128) as f16: bytes 0, 2 (0x4240) or 1, 3 (0x4341).
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t sel) {
    return sub_f16x2(__byte_perm(biased, 0x64646464u, sel), 0x64806480u);  // 1152 = 0x6480
}

// ---- a tile: which rows, which keys ----
struct Tile {
    uint32_t row, tokens, slot;
    uint32_t from, to;  // keys that any of its rows sees (from >= to: none)
    uint32_t base;      // the first block of positions it reads (whole slots)
    uint32_t entries;   // blocks it reads, or listed blocks
    uint32_t steps;     // at least one, so that every row's result is somebody's work
};

template <int W>
struct Step {
    static constexpr int KEYS = kHalfStage / W, UNITS = KEYS / 16;  // 64, 32, 16 keys; units of 16
    static constexpr int HALVES = W == 256 ? 2 : 1, COLS = W == 64 ? 64 : 128;
};

__device__ __forceinline__ void seen(const AttendParams &p, uint32_t pos, uint32_t *lo, uint32_t *hi) {
    *lo = pos > p.back ? pos - p.back : 0;
    *hi = pos < p.keys ? pos + 1 : p.keys;
}

// Consecutive rows, one a lane, and the tiles that begin at them.  A lane whose row lies in a tile that begins before it
// has steps = 0.  `width` rows are looked at together, a multiple of the rows a tile may hold, so that no tile lies
// across: tiles begin at multiples of `tokens` and where a row is not the next position of the slot before it (or the
// same again).
struct RowGroup {
    uint32_t slot, tokens, from, to, steps;
};

__device__ __forceinline__ uint32_t rows_together(const AttendParams &p) { return 32 - 32 % p.tokens; }

struct RawRow {
    uint32_t slot, pos;
};

__device__ __forceinline__ RawRow row_at(const AttendParams &p, uint32_t first, uint32_t lane) {
    RawRow raw = {0, 0};
    if (lane < rows_together(p) && first + lane < p.rows) raw = {p.slots[first + lane], p.positions[first + lane]};
    return raw;
}

template <int W, bool LIST>
__device__ __forceinline__ RowGroup rows_from(const AttendParams &p, const RawRow &raw, uint32_t first, uint32_t lane) {
    RowGroup g = {raw.slot, 1, 0, 0, 0};
    const uint32_t row = first + lane, pos = raw.pos;
    const bool here = lane < rows_together(p) && row < p.rows;
    uint32_t last = pos;
    bool begins = here;
    if (!LIST && p.tokens > 1) {
        const uint32_t slot0 = __shfl_up_sync(0xFFFFFFFFu, g.slot, 1), pos0 = __shfl_up_sync(0xFFFFFFFFu, pos, 1);
        const bool follows = here && row % p.tokens != 0 && g.slot == slot0 && pos >= pos0 && pos - pos0 <= 1u;
        const uint32_t mask = __ballot_sync(0xFFFFFFFFu, follows);
        begins = here && !follows;
        g.tokens = lane == 31 ? 1 : __ffs(~(mask >> (lane + 1)));  // this row and those that follow without a break
        last = __shfl_sync(0xFFFFFFFFu, pos, min(lane + g.tokens - 1, 31u));
    }
    // positions ascend within a tile: its first row sees the earliest key, its last one the latest
    uint32_t x;
    seen(p, pos, &g.from, &x);
    seen(p, last, &x, &g.to);
    if (g.from >= g.to) g.from = g.to = 0;
    if (begins) {
        if (LIST) g.steps = ((p.count << (p.kv.shift - 4)) + Step<W>::UNITS - 1) / Step<W>::UNITS;
        else g.steps = g.from < g.to ? (g.to - 1 - (g.from >> p.kv.shift << p.kv.shift)) / Step<W>::KEYS + 1 : 1;
    }
    return g;
}

template <bool LIST>
__device__ __forceinline__ Tile tile_at(const AttendParams &p, const RowGroup &g, uint32_t first, uint32_t l) {
    Tile t;
    t.row = first + l;
    t.tokens = __shfl_sync(0xFFFFFFFFu, g.tokens, l);
    t.slot = __shfl_sync(0xFFFFFFFFu, g.slot, l);
    t.from = __shfl_sync(0xFFFFFFFFu, g.from, l);
    t.to = __shfl_sync(0xFFFFFFFFu, g.to, l);
    t.steps = __shfl_sync(0xFFFFFFFFu, g.steps, l);
    t.base = LIST ? 0 : t.from >> p.kv.shift;
    t.entries = LIST ? p.count : t.from < t.to ? ((t.to - 1) >> p.kv.shift) + 1 - t.base : 0;
    return t;
}

__device__ __forceinline__ uint32_t warp_total(uint32_t v) { return __reduce_add_sync(0xFFFFFFFFu, v); }

// ---- the query operand: column r of eight is tile row 8 t + r; thread j of its four has channels 16 s + 4 j + 0..3 ----
constexpr float kQueryMost = 32639.0f;  // 127 * 256 + 127

template <int W, int NT>
struct Queries {
    uint32_t b[NT][W / 32][2][2];   // step of 32 channels; digit 256s, digit ones; channels 0-15 and 16-31 of the step
    float f[NT][2];                 // raw score -> power-of-two exponent, without the key scale, for columns 2 j, 2 j + 1
    uint32_t lo[NT][2], hi[NT][2];  // keys those columns see
};

// As they lie in memory, asked for early.
template <int W, int NT>
struct RawQueries {
    uint2 v[NT][W / 16];
};

template <int W, int NT>
__device__ __forceinline__ RawQueries<W, NT> fetch_queries(const AttendParams &p, const Tile &tile, uint32_t head0, uint32_t part, uint32_t lane) {
    RawQueries<W, NT> raw;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const uint32_t m = 8 * t + (lane >> 2), token = m / part, head = m - token * part;
        const uint16_t *q = p.q + ((size_t)(tile.row + token) * p.heads + head0 + head) * W + 4 * (lane & 3);
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            raw.v[t][s] = make_uint2(0, 0);
            if (token < tile.tokens) raw.v[t][s] = *reinterpret_cast<const uint2 *>(q + 16 * s);
        }
    }
    return raw;
}

template <int W, int NT>
__device__ __forceinline__ void load_queries(const AttendParams &p, const Tile &tile, const RawQueries<W, NT> &raw, uint32_t part,
                                             uint32_t lane, Queries<W, NT> &qs) {
    const uint32_t j = lane & 3;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const uint2 (&v)[W / 16] = raw.v[t];
        float most = 0.0f, bad = 0.0f;  // bad: NaN once an element is infinite or NaN
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            const float x[4] = {bf16_lo(v[s].x), bf16_hi(v[s].x), bf16_lo(v[s].y), bf16_hi(v[s].y)};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                most = fmaxf(most, fabsf(x[i]));
                bad = fmaf(x[i], 0.0f, bad);
            }
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
            bad += __shfl_xor_sync(0xFFFFFFFFu, bad, o);
        }
        // 2^-e first, so that neither the smallest nor the largest magnitudes leave f32 on the way
        uint32_t e = __float_as_uint(most) >> 23;
        e = e < 1 ? 1 : e > 253 ? 253 : e;
        const float down = __uint_as_float((254 - e) << 23), unit = most * down / kQueryMost;
        const float inv = most > 0.0f ? kQueryMost / (most * down) : 0.0f;
        const float f = __uint_as_float(e << 23) * unit * (p.scale * kLog2e) + bad;
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            const float x[4] = {bf16_lo(v[s].x), bf16_hi(v[s].x), bf16_lo(v[s].y), bf16_hi(v[s].y)};
            uint32_t high = 0, low = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int q = __float2int_rn(x[i] * down * inv), q1 = (q + 128) >> 8;
                high |= (uint32_t)(q1 & 255) << (8 * i);
                low |= (uint32_t)((q - (q1 << 8)) & 255) << (8 * i);
            }
            qs.b[t][s / 2][0][s % 2] = high;
            qs.b[t][s / 2][1][s % 2] = low;
        }
#pragma unroll
        for (int e2 = 0; e2 < 2; e2++) {
            qs.f[t][e2] = __shfl_sync(0xFFFFFFFFu, f, (2 * j + e2) * 4);
            const uint32_t tok = (8 * t + 2 * j + e2) / part;
            qs.lo[t][e2] = 1;
            qs.hi[t][e2] = 0;
            if (tok < tile.tokens) seen(p, p.positions[tile.row + tok], &qs.lo[t][e2], &qs.hi[t][e2]);
        }
    }
}

// ---- running softmax and output: columns 2 j + e; o[i][t][e], [2 + e]: channels 16 i + 2 r and 16 i + 2 r + 1 ----
template <int W, int NT>
struct Running {
    float o[W / 16][NT][4];
    float m[NT][2], l[NT][2];
};

// Shared-memory address of this lane's row for an ldmatrix.x4 of pieces c and c + 1 (c even) of unit u: matrices are
// (keys 0-7, c), (keys 8-15, c), (keys 0-7, c + 1), (keys 8-15, c + 1).
// Rows of 64 bytes (W = 64): piece ^ (key / 2 % 4); of 128 bytes: piece ^ (key % 8); W = 256: two such tiles.
template <int W>
__device__ __forceinline__ uint32_t piece_at(uint32_t tile, int u, int c, uint32_t lane) {
    const uint32_t key = 16 * u + (lane & 15), side = lane >> 4;
    if constexpr (W == 64) return tile + key * 64 + (((c + side) ^ (key >> 1 & 3)) << 4);
    else return tile + (c >> 3) * (Step<W>::KEYS * 128) + key * 128 + ((((c & 7) + side) ^ (key & 7)) << 4);
}

// A step's scores in powers of two with the value scale's exponent.  EDGE: some key of the step is not seen by some row.  A
// unit without keys has key0 past every row's.  N: the blocks a step may lie in, one (all its units) or one a unit.
template <int W, int NT, int N, bool EDGE>
__device__ __forceinline__ void score_step(const Queries<W, NT> &qs, uint32_t tile, const float (&ks)[N], const float (&vs)[N],
                                           const uint32_t (&key0)[N], float (&x)[Step<W>::UNITS][NT][4], uint32_t lane) {
    constexpr int U = Step<W>::UNITS;
    const uint32_t r = lane >> 2;
    float lv[N];
#pragma unroll
    for (int n = 0; n < N; n++) lv[n] = log2_approx(max_nan(vs[n], kScaleFloor));  // NaN stays NaN: it shows in rows that see the block
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int n = N == 1 ? 0 : u;
        int high[NT][4], low[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) high[t][i] = low[t][i] = 0;
#pragma unroll
        for (int c = 0; c < W / 16; c += 2) {
            uint32_t a[4];
            ldsm_x4(piece_at<W>(tile, u, c, lane), a);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                mma_s8(high[t], a, qs.b[t][c / 2][0]);
                mma_s8(low[t], a, qs.b[t][c / 2][1]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float f = qs.f[t][e] * ks[n];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float y = fmaf(__int2float_rn(high[t][2 * k + e] * 256 + low[t][2 * k + e]), f, lv[n]);
                    if (EDGE) {
                        const uint32_t key = key0[n] + (N == 1 ? 16 * u : 0) + 8 * k + r;
                        if (key < qs.lo[t][e] || key >= qs.hi[t][e]) y = -INFINITY;
                    }
                    x[u][t][2 * k + e] = y;
                }
            }
    }
}

// The probabilities of a step's scores, as the second product's operand b, and their sum.  M need not be the maximum so
// far: it stays until a score passes it by kSlack, so that most steps neither bring the maximum together across lanes nor
// touch the output (16 rows found a new maximum in every other step: 61 us for 16 x 7 rows of up to 4099 keys, 58.5 so).
//
// P = 2^(x - M + kLift) reaches 2^15 then, the last power of two within f16.  The factor of 2^kLift is in both sums and in
// every partial result alike, so it cancels; without it a weight below 2^-14 of the largest lost digits in the first sum
// and was gone below 2^-25 of it, but not in the second (8192 keys with 1.5 * 2^-24 each beside one whose value is zero:
// the output was off by a third).  Now that begins at 2^-21 and 2^-32, at no cost that can be measured.
constexpr float kSlack = 8.0f, kLift = 7.0f;

template <int W, int NT, int N>
__device__ __forceinline__ void soften(Running<W, NT> &run, const float (&x)[Step<W>::UNITS][NT][4], const float (&vs)[N],
                                       uint32_t (&b)[Step<W>::UNITS][NT][2]) {
    constexpr int U = Step<W>::UNITS;
    float most[NT][2];
    bool past = false;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            most[t][e] = fmaxf(x[0][t][e], x[0][t][2 + e]);
#pragma unroll
            for (int u = 1; u < U; u++) most[t][e] = fmaxf(most[t][e], fmaxf(x[u][t][e], x[u][t][2 + e]));
            past = past || most[t][e] > run.m[t][e] + kSlack;
        }
    if (__any_sync(0xFFFFFFFFu, past)) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) most[t][e] = fmaxf(most[t][e], __shfl_xor_sync(0xFFFFFFFFu, most[t][e], o));
                const float now = fmaxf(run.m[t][e], most[t][e]);
                const float scale = exp2_approx(run.m[t][e] - (now == -INFINITY ? 0.0f : now));
                run.m[t][e] = now;
                run.l[t][e] *= scale;
#pragma unroll
                for (int i = 0; i < W / 16; i++) {
                    run.o[i][t][e] *= scale;
                    run.o[i][t][2 + e] *= scale;
                }
            }
    }
    float top[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) top[t][e] = run.m[t][e] == -INFINITY ? 0.0f : run.m[t][e] - kLift;  // nothing seen yet: 2^(-inf - 0) = 0
    float inv[N];
#pragma unroll
    for (int n = 0; n < N; n++) inv[n] = __fdividef(1.0f, fmaxf(vs[n], kScaleFloor));  // no NaN here: rows that see nothing of the block have P = 0
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                p[e] = exp2_approx(x[u][t][e] - top[t][e]);
                p[2 + e] = exp2_approx(x[u][t][2 + e] - top[t][e]);
                run.l[t][e] = fmaf(p[e] + p[2 + e], inv[N == 1 ? 0 : u], run.l[t][e]);
            }
            b[u][t][0] = transpose_8x8(pack_f16(p[0], p[1]));
            b[u][t][1] = transpose_8x8(pack_f16(p[2], p[3]));
        }
    }
}

template <int W, int NT>
__device__ __forceinline__ void value_step(Running<W, NT> &run, uint32_t tile, const uint32_t (&b)[Step<W>::UNITS][NT][2], uint32_t lane) {
#pragma unroll
    for (int u = 0; u < Step<W>::UNITS; u++)
#pragma unroll
        for (int c = 0; c < W / 16; c += 2) {
            uint32_t w[4];
            ldsm_x4_trans(piece_at<W>(tile, u, c, lane), w);
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] ^= 0x80808080u;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t a0 = codes_f16(w[2 * i], 0x4240), a1 = codes_f16(w[2 * i], 0x4341), a2 = codes_f16(w[2 * i + 1], 0x4240),
                               a3 = codes_f16(w[2 * i + 1], 0x4341);
#pragma unroll
                for (int t = 0; t < NT; t++) mma_f16(run.o[c + i][t], a0, a1, a2, a3, b[u][t]);
            }
        }
}

// 32 blocks' places in the pool and scales, one a lane: entry `first` + lane of the tile's blocks.
constexpr uint32_t kNoKeys = 0xFFFFFF00u;  // a unit's first key where there is no block: rows see less (attend_q8 sees to it)

struct Group {
    uint32_t blk, id;  // pool block or kNoBlock; which block of the slot's positions it is
    float ks, vs;
};

template <bool LIST>
__device__ __forceinline__ Group group_of(const AttendParams &p, const Tile &t, uint32_t kvh, uint32_t first, uint32_t lane) {
    Group g = {kNoBlock, 0, 0.0f, 0.0f};
    const uint32_t e = first + lane;
    if (e < t.entries) {
        g.id = LIST ? p.ids[((size_t)t.row * p.kv_heads + kvh) * p.count + e] : t.base + e;
        if (((uint64_t)g.id << p.kv.shift) < t.to) g.blk = block_of(p.kv, t.slot, g.id);
        if (g.blk != kNoBlock) {
            const size_t at = (size_t)g.blk * p.kv_heads + kvh;
            g.ks = p.kv.k_scale[at];
            g.vs = p.kv.v_scale[at];
        }
    }
    return g;
}

// A warp's ring: the next stage to complete and the parity each completes with.  K and V of a stage complete, and are
// asked for again, each by itself: while one is computed on, the other and the other stages are under way.
struct Ring {
    uint32_t tiles;  // shared-memory address
    uint64_t *full;  // K of every stage, then V of every stage
    uint32_t stage, parity;
    bool ok;  // false: a wait ran out, nothing is copied or computed any more
};

// A part of a worker's run: steps [begin, end) of a tile for one kv head and part of its heads.
struct Segment {
    Tile tile;
    uint32_t unit, kvh, head0, part;  // unit: kv head and part of its heads as one number
    uint32_t begin, end;
    uint32_t start;    // where the tile's steps begin in all steps
    bool partial;      // another worker has the rest of them
    uint32_t slot;     // of the worker's two partial results
    float *part_o, *part_ml;  // where a partial result goes: [tile rows][W] and [tile rows][2]
};

// What follows a segment, so that its first steps' copies leave while the segment's last steps are computed.
struct Following {
    Group group;
    uint32_t begin, steps, kvh;  // steps: how many may be asked for early; 0: nothing follows
};

// Computes a segment, `asked` of whose steps are already on their way, and returns how many of the following one's are.
// ONE: every step lies within one block.  follow() fills `then` in; it is called once the segment's own copies have all been
// asked for, so that its look-ups wait while they are under way.
template <int W, int NT, bool LIST, bool ONE, class Follow>
__device__ __forceinline__ uint32_t attend_steps(const AttendParams &p, const CUtensorMap *map_k, const CUtensorMap *map_v, const Segment &seg,
                                                 Group now, uint32_t asked, const Following &then, Follow &&follow, Ring &ring,
                                                 int *status, uint32_t lane) {
    using namespace ptx;
    constexpr int KEYS = Step<W>::KEYS, U = Step<W>::UNITS, HALVES = Step<W>::HALVES, COLS = Step<W>::COLS, STAGES = kStages;
    constexpr int N = ONE ? 1 : U, SPAN = U / N;  // blocks a step may lie in, units of each
    const Tile &tile = seg.tile;
    const uint32_t kvh = seg.kvh, head0 = seg.head0, part = seg.part, begin = seg.begin, end = seg.end;
    const uint32_t in_block = p.kv.shift - 4;  // log2 of a block's 16-key units
    Running<W, NT> run;
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int i = 0; i < W / 16; i++) run.o[i][t][0] = run.o[i][t][1] = run.o[i][t][2] = run.o[i][t][3] = 0.0f;
        run.m[t][0] = run.m[t][1] = -INFINITY;
        run.l[t][0] = run.l[t][1] = 0.0f;
    }
    uint32_t early = 0;  // steps of what follows that are on their way
    if (tile.from < tile.to) {
        uint32_t first = (begin * U) >> in_block;  // entry of lane 0 of the current group
        const RawQueries<W, NT> raw = fetch_queries<W, NT>(p, tile, head0, part, lane);
        Group next = now;  // the first copies lie in the current group
        const uint32_t per = 1u << in_block, span = ONE ? U : per < (uint32_t)U ? per : U;  // units of one copy
        constexpr bool CHAIN = NT == 1;  // with sixteen rows its registers cost more than it saves (56.7 us for 53.4)
        uint32_t last = end;
        bool followed = !CHAIN;
        // Step s's units as rows of the tensor maps, -1 where there is no block; the current or the next group has its
        // blocks, or what follows does.
        auto find = [&](uint32_t s, int32_t (&y)[N]) {
            const bool mine = !CHAIN || s < end;
            const uint32_t unit = (mine ? s : then.begin + (s - end)) * U, head = mine ? kvh : then.kvh;
            const uint32_t from = mine ? first : (then.begin * U) >> in_block;
#pragma unroll
            for (int n = 0; n < N; n++) {
                y[n] = -1;
                if (!ONE && (n & (span - 1)) != 0) continue;  // lies in the copy of the unit before it
                const uint32_t e = ((unit + n) >> in_block) - from;
                const uint32_t blk = __shfl_sync(0xFFFFFFFFu, !mine ? then.group.blk : e < 32 ? now.blk : next.blk, e & 31);
                if (blk != kNoBlock) y[n] = (int32_t)(((blk * p.kv_heads + head) << p.kv.shift) + (((unit + n) & (per - 1)) << 4));
            }
        };
        // Copies of a step's K (values = 0) or V (1) into stage `at`.
        auto copy = [&](uint32_t at, const int32_t (&y)[N], const CUtensorMap *map, int values) {
            if (lane == 0) {
                uint64_t *bar = &ring.full[values * STAGES + at];
                const uint32_t dst = ring.tiles + at * kStage + values * kHalfStage;
                uint32_t bytes = 0;
#pragma unroll
                for (int n = 0; n < N; n++)
                    if (y[n] >= 0) bytes += span * 16 * W;
                mbar_expect_tx(bar, bytes);
#pragma unroll
                for (int n = 0; n < N; n++) {
                    if (y[n] < 0) continue;
#pragma unroll
                    for (int h = 0; h < HALVES; h++) copy_codes(dst + (h * KEYS + 16 * n) * COLS, map, smem_addr(bar), h * COLS, y[n]);
                }
            }
        };
        int32_t y[N];
        uint32_t ahead = begin + asked;  // the next step to ask for; from `end` on, of what follows
        auto fill = [&](uint32_t s) {  // the stages that are free at step s
            for (; ahead < last && ahead < s + STAGES; ahead++) {
                const uint32_t at = (ring.stage + (ahead - s)) % STAGES;
                find(ahead, y);
                copy(at, y, map_k, 0);
                copy(at, y, map_v, 1);
            }
        };
        fill(begin);
        next = group_of<LIST>(p, tile, kvh, first + 32, lane);
        Queries<W, NT> qs;
        load_queries<W, NT>(p, tile, raw, part, lane, qs);
        uint32_t all_lo = 0, all_hi = 0;  // keys that every row of the tile sees
        {
            uint32_t x;
            seen(p, p.positions[tile.row], &x, &all_hi);
            seen(p, p.positions[tile.row + tile.tokens - 1], &all_lo, &x);
        }
        // Keys [k, k + 16 SPAN) are all seen where k - inner_lo <= inner; nowhere: k is a multiple of 16, never 1.
        const bool any_inner = all_hi >= 16 * SPAN && all_lo <= all_hi - 16 * SPAN;
        const uint32_t inner_lo = any_inner ? all_lo : 1, inner = any_inner ? all_hi - 16 * SPAN - all_lo : 0;
        for (uint32_t s = begin; s < end; s++) {
            if (((s * U) >> in_block) - first >= 32) {
                first += 32;
                now = next;
                next = group_of<LIST>(p, tile, kvh, first + 32, lane);
            }
            if (!followed && ahead >= end) {
                follow();
                followed = true;
                last = end + then.steps;
                fill(s);
            }
            float ks[N], vs[N];
            uint32_t key0[N];
            bool edge = false;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const uint32_t unit = s * U + n;
                if (n == 0 || (unit & (per - 1)) == 0) {  // another block
                    const uint32_t e = ((unit >> in_block) - first) & 31;
                    ks[n] = __shfl_sync(0xFFFFFFFFu, now.ks, e);
                    vs[n] = __shfl_sync(0xFFFFFFFFu, now.vs, e);
                    const uint32_t id = __shfl_sync(0xFFFFFFFFu, now.blk == kNoBlock ? kNoBlock : now.id, e);
                    key0[n] = id == kNoBlock ? kNoKeys : (id << p.kv.shift) + ((unit & (per - 1)) << 4);
                } else {
                    ks[n] = ks[n - (n > 0)];
                    vs[n] = vs[n - (n > 0)];
                    key0[n] = key0[n - (n > 0)] == kNoKeys ? kNoKeys : key0[n - (n > 0)] + 16;
                }
                edge = edge || key0[n] - inner_lo > inner;
            }
            const uint32_t at = ring.tiles + ring.stage * kStage, odd = ring.parity >> ring.stage & 1;
            ring.parity ^= 1u << ring.stage;
            // A wait that runs out ends the warp's work once the copies still under way have been waited for, as long:
            // V of this step and both of the steps from s + 1 up to `ahead`.
            auto give_up = [&](bool k_too) {
                ring.ok = false;
                if (!k_too) mbar_wait(&ring.full[STAGES + ring.stage], odd);
                for (uint32_t i = s + 1; i < ahead; i++) {
                    const uint32_t stage = (ring.stage + (i - s)) % STAGES;
                    mbar_wait(&ring.full[stage], ring.parity >> stage & 1);
                    mbar_wait(&ring.full[STAGES + stage], ring.parity >> stage & 1);
                }
                if (k_too && ahead < last) mbar_wait(&ring.full[ring.stage], odd ^ 1);
                if (lane == 0) atomicExch(status, TS_ERR_TIMEOUT);
            };
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(&ring.full[ring.stage], odd))) {
                give_up(false);
                return 0;
            }
            float x[U][NT][4];
            if (edge) score_step<W, NT, N, true>(qs, at, ks, vs, key0, x, lane);
            else score_step<W, NT, N, false>(qs, at, ks, vs, key0, x, lane);
            __syncwarp();
            if (ahead < last) {
                find(ahead, y);
                copy(ring.stage, y, map_k, 0);
            }
            uint32_t b[U][NT][2];
            soften<W, NT, N>(run, x, vs, b);
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(&ring.full[STAGES + ring.stage], odd))) {
                give_up(true);
                return 0;
            }
            value_step<W, NT>(run, at + kHalfStage, b, lane);
            __syncwarp();
            if (ahead < last) {
                copy(ring.stage, y, map_v, 1);
                ahead++;
            }
            ring.stage = (ring.stage + 1) % STAGES;
        }
        early = ahead - end;
    }
    // ---- this thread's channels of tile rows 8 t + 2 j + e ----
    const uint32_t r = lane >> 2, j = lane & 3;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float l = run.l[t][e];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
            const uint32_t m = 8 * t + 2 * j + e;
            if (m >= tile.tokens * part) continue;
            if (!seg.partial) {
                const uint32_t token = m / part;
                uint16_t *out = p.out + ((size_t)(tile.row + token) * p.heads + head0 + m - token * part) * W + 2 * r;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int i = 0; i < W / 16; i++)
                    *reinterpret_cast<uint32_t *>(out + 16 * i) = pack_bf16(run.o[i][t][e] * inv, run.o[i][t][2 + e] * inv);
            } else {
                float *o = seg.part_o + m * W + 2 * r;
#pragma unroll
                for (int i = 0; i < W / 16; i++) *reinterpret_cast<float2 *>(o + 16 * i) = make_float2(run.o[i][t][e], run.o[i][t][2 + e]);
                if (r == 0) *reinterpret_cast<float2 *>(seg.part_ml + m * 2) = make_float2(run.m[t][e], l);
            }
        }
    return early;
}

template <int W, bool LIST, bool ONE>
__global__ void __launch_bounds__(kThreads, kBlocks)
attend_q8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttendParams p, int *status) {
    using namespace ptx;
    constexpr int STAGES = kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][2 * STAGES];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t worker = warp * gridDim.x + blockIdx.x;  // few workers spread over the SMs
    Ring ring = {smem_addr(smem) + warp * (STAGES * kStage), bars[warp], 0, 0, true};
    if (lane == 0) {
        for (int s = 0; s < 2 * STAGES; s++) mbar_init(&ring.full[s], 1);
        fence_barrier_init();
        if (warp == 0) {
            prefetch_tensormap(&map_k);
            prefetch_tensormap(&map_v);
        }
    }
    __syncwarp();
    pdl_wait();
    if (worker < p.workers) {
        // ---- the steps of all tiles, and this worker's run of them ----
        const uint32_t per_row = p.kv_heads * p.parts, width = rows_together(p);
        uint32_t first = 0, total = 0;
        // Pieces if every tile is cut by itself into pieces of 1, 2, 3, 4, 6 or 8 steps.
        uint32_t pieces[6] = {};
        RawRow raw = row_at(p, 0, lane);
        RowGroup rows;
        if (LIST) {
            rows = rows_from<W, LIST>(p, raw, 0, lane);
            total = __shfl_sync(0xFFFFFFFFu, rows.steps, 0);
#pragma unroll
            for (int i = 0; i < 6; i++) pieces[i] = (total + kRuns[i] - 1) / kRuns[i] * p.rows;
            total *= p.rows;
        } else {
            for (uint32_t f = 0; f < p.rows; f += width) {
                const RawRow next = row_at(p, f + width, lane);  // on its way during the sums
                const RowGroup g = rows_from<W, LIST>(p, raw, f, lane);
                total += warp_total(g.steps);
#pragma unroll
                for (int i = 1; i < 6; i++) pieces[i] += warp_total((g.steps + kRuns[i] - 1) / kRuns[i]);
                if (f == 0) rows = g;
                raw = next;
            }
            pieces[0] = total;
        }
        total *= per_row;
        // A worker's run: an equal share of the steps laid end to end, or, where that is eight steps at most, the shortest
        // piece for which there are workers enough (a run that ends one tile and begins the next pays for two starts).
        uint32_t run = max(1u, (total + p.workers - 1) / p.workers), by = 1;  // by: tiles take multiples of it
        if (!p.merged) {
            by = p.whole;
        } else if (run <= 8) {
#pragma unroll
            for (int i = 5; i >= 0; i--)
                if (pieces[i] * per_row <= p.workers) by = run = kRuns[i];
        }
        auto taken = [&](uint32_t steps) { return (steps + by - 1) / by * by; };
        if (by > 1) {
#pragma unroll
            for (int i = 1; i < 6; i++)
                if (by == kRuns[i]) total = pieces[i] * kRuns[i] * per_row;
        }
        if (!p.merged) run = (total + p.workers * by - 1) / (p.workers * by) * by;
        uint32_t at = worker * run;
        const uint32_t end = min(total, at + run);
        if (at < end) {
            uint32_t before = 0, l = 0;  // steps of earlier rows, all kv heads; the lane whose row holds `at`
            if (LIST) {
                const uint32_t each = total / p.rows, row = at / each;
                before = row * each;
                first = row;
                rows = rows_from<W, LIST>(p, row_at(p, first, lane), first, lane);
            } else {
                for (;;) {
                    uint32_t sum = taken(rows.steps) * per_row;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                        if (lane >= (uint32_t)o) sum += other;
                    }
                    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + sum > at);
                    if (hit) {
                        l = __ffs(hit) - 1;
                        before += __shfl_sync(0xFFFFFFFFu, sum - taken(rows.steps) * per_row, l);
                        break;
                    }
                    before += __shfl_sync(0xFFFFFFFFu, sum, 31);
                    first += width;
                    if (first >= p.rows) return;  // not reached: at < total
                    rows = rows_from<W, LIST>(p, row_at(p, first, lane), first, lane);
                }
            }
            // The run's segments, one after another.
            Tile tile = tile_at<LIST>(p, rows, first, l);
            uint32_t n = taken(tile.steps), unit = (at - before) / n, start = before + unit * n, count = 0;
            auto next_segment = [&](Segment *seg) {
                if (at >= end) return false;
                if (unit == per_row) {  // the next tile
                    before += n * per_row;
                    const uint32_t later = __ballot_sync(0xFFFFFFFFu, rows.steps != 0 && lane > l);
                    if (later) {
                        l = __ffs(later) - 1;
                    } else {
                        first += width;
                        if (first >= p.rows) return false;
                        rows = rows_from<W, LIST>(p, row_at(p, first, lane), first, lane);
                        l = 0;
                    }
                    tile = tile_at<LIST>(p, rows, first, l);
                    n = taken(tile.steps);
                    unit = 0;
                    start = before;
                }
                const uint32_t kvh = p.parts == 1 ? unit : unit / p.parts, hp = unit - kvh * p.parts;
                seg->tile = tile;
                seg->unit = unit;
                seg->kvh = kvh;
                seg->head0 = kvh * p.group + hp * p.part;
                seg->part = min(p.part, p.group - hp * p.part);
                seg->begin = at - start;
                seg->end = min(tile.steps, end - start);
                seg->start = start;
                seg->partial = seg->begin > 0 || seg->end < tile.steps;
                seg->slot = count++ ? 1 : 0;
                seg->part_o = p.part_o + ((size_t)worker * 2 + seg->slot) * p.most * W;
                seg->part_ml = p.part_ml + ((size_t)worker * 2 + seg->slot) * p.most * 2;
                unit++;
                start += n;
                at = start;
                return true;
            };
            auto group_for = [&](const Segment &seg) {
                return group_of<LIST>(p, seg.tile, seg.kvh, (seg.begin * Step<W>::UNITS) >> (p.kv.shift - 4), lane);
            };
            Segment now;
            bool any = next_segment(&now);
            Group group = group_for(now);
            uint32_t asked = 0;
            while (any && ring.ok) {
                Segment next;
                bool more = false, followed = false;
                Following then = {{kNoBlock, 0, 0.0f, 0.0f}, 0, 0, 0};
                auto follow = [&] {
                    followed = true;
                    more = next_segment(&next);
                    if (more) {
                        then.group = group_for(next);
                        then.begin = next.begin;
                        then.steps = next.tile.from < next.tile.to ? min(next.end - next.begin, (uint32_t)kStages) : 0;
                        then.kvh = next.kvh;
                    }
                };
                if (now.tile.tokens * now.part <= 8)
                    asked = attend_steps<W, 1, LIST, ONE>(p, &map_k, &map_v, now, group, asked, then, follow, ring, status, lane);
                else
                    asked = attend_steps<W, 2, LIST, ONE>(p, &map_k, &map_v, now, group, asked, then, follow, ring, status, lane);
                if (!followed) follow();
                // who has a tile's first step says where its partials are
                if (now.begin == 0 && p.merged && lane < now.tile.tokens)
                    p.places[(size_t)(now.tile.row + lane) * per_row + now.unit] =
                        make_uint4(worker, (now.start + now.tile.steps - 1) / run, now.slot, lane * now.part);
                now = next;
                group = then.group;
                any = more;
            }
        }
    }
    pdl_launch_dependents();
}

// One block per (row, head): folds the partials of its tile in the order of their keys.  Threads take partials side by
// side for their weights, then W / 4 threads read a partial's output, THREADS * 4 / W partials side by side.  Few rows and
// heads have many partials each and get 256 threads; many have few, and 64 let all of them be resident at once (3584 rows
// and heads: 13 us with 256).
template <int W, int kMergeThreads>
__global__ void __launch_bounds__(kMergeThreads) attend_q8_merge_kernel(const AttendParams p) {
    constexpr uint32_t COLS = W / 4, SETS = kMergeThreads / COLS;
    extern __shared__ float weight[];  // [partials]
    __shared__ float sm_top[kMergeThreads / 32], sm_l[kMergeThreads / 32];
    __shared__ float4 sm_o[SETS][COLS];
    pdl_wait();
    const uint32_t row = blockIdx.x / p.heads, head = blockIdx.x % p.heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t kvh = head / p.group, in = head % p.group, hp = in / p.part;
    const uint4 place = p.places[((size_t)row * p.kv_heads + kvh) * p.parts + hp];
    const uint32_t m = place.w + in % p.part;
    // else its one worker wrote it (or gave up)
    if (place.x < place.y && place.y < p.workers && place.z < 2 && m < p.most) {
        const uint32_t n = place.y - place.x + 1;
        auto slot = [&](uint32_t i) { return ((size_t)(place.x + i) * 2 + (i == 0 ? place.z : 0)) * p.most + m; };
        // the first outputs are asked for before their weights are known
        constexpr int EARLY = 4;
        const uint32_t set = threadIdx.x / COLS, col = threadIdx.x % COLS;
        float4 early[EARLY];
#pragma unroll
        for (int k = 0; k < EARLY; k++)
            if (set + k * SETS < n) early[k] = *reinterpret_cast<const float4 *>(p.part_o + slot(set + k * SETS) * W + col * 4);
        float top = -INFINITY;
        for (uint32_t i = threadIdx.x; i < n; i += kMergeThreads) {
            weight[i] = p.part_ml[slot(i) * 2];
            top = fmaxf(top, weight[i]);
        }
        top = warp_max(top);
        if (lane == 0) sm_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kMergeThreads / 32; w++) top = fmaxf(top, sm_top[w]);
        if (top == -INFINITY) top = 0.0f;
        float l = 0.0f;
        for (uint32_t i = threadIdx.x; i < n; i += kMergeThreads) {
            const float f = exp2_approx(weight[i] - top);
            weight[i] = f;
            l = fmaf(p.part_ml[slot(i) * 2 + 1], f, l);
        }
        l = warp_sum(l);
        if (lane == 0) sm_l[warp] = l;
        __syncthreads();
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](const float4 &v, float f) {
            o.x = fmaf(v.x, f, o.x);
            o.y = fmaf(v.y, f, o.y);
            o.z = fmaf(v.z, f, o.z);
            o.w = fmaf(v.w, f, o.w);
        };
#pragma unroll
        for (int k = 0; k < EARLY; k++)
            if (set + k * SETS < n) add(early[k], weight[set + k * SETS]);
#pragma unroll 4
        for (uint32_t i = set + EARLY * SETS; i < n; i += SETS)
            add(*reinterpret_cast<const float4 *>(p.part_o + slot(i) * W + col * 4), weight[i]);
        sm_o[set][col] = o;
        __syncthreads();
        if (threadIdx.x < COLS) {
            float4 sum = sm_o[0][threadIdx.x];
            l = sm_l[0];
#pragma unroll
            for (int i = 1; i < (int)SETS; i++) {
                const float4 v = sm_o[i][threadIdx.x];
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
#pragma unroll
            for (int w = 1; w < kMergeThreads / 32; w++) l += sm_l[w];
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            *reinterpret_cast<uint2 *>(p.out + ((size_t)row * p.heads + head) * W + threadIdx.x * 4) =
                make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
        }
    }
    pdl_launch_dependents();
}

// Few and short rows: a cluster of blocks has one row and kv head (or part of its heads), its warps cut the steps among them,
// and the partial results meet through distributed shared memory: one launch, no pass over the rows, no workspace.  One row
// of 517 keys: 9.0 us, 8 rows x 32 listed blocks of 16: 9.9; both wait for one load after another (position, page, scale, codes).
template <int W, bool LIST, bool ONE>
__global__ void __launch_bounds__(kThreads, kBlocks)
attend_q8_cluster_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttendParams p, int *status) {
    using namespace ptx;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][2 * kStages];
    __shared__ float2 sm_ml[kWarps][16];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster_ctarank(), blocks = p.cluster;
    Ring ring = {smem_addr(smem) + warp * (kStages * kStage), bars[warp], 0, 0, true};
    if (lane == 0) {
        for (int s = 0; s < 2 * kStages; s++) mbar_init(&ring.full[s], 1);
        fence_barrier_init();
        if (warp == 0) {
            prefetch_tensormap(&map_k);
            prefetch_tensormap(&map_v);
        }
    }
    __syncwarp();
    pdl_wait();
    const uint32_t per_row = p.kv_heads * p.parts, job = blockIdx.x / blocks, worker = warp * blocks + rank;
    Segment seg;
    Tile &t = seg.tile;
    t.row = job / per_row;
    t.tokens = 1;
    t.slot = p.slots[t.row];
    seen(p, p.positions[t.row], &t.from, &t.to);
    if (t.from >= t.to) t.from = t.to = 0;
    t.base = LIST ? 0 : t.from >> p.kv.shift;
    t.entries = LIST ? p.count : t.from < t.to ? ((t.to - 1) >> p.kv.shift) + 1 - t.base : 0;
    t.steps = LIST            ? ((p.count << (p.kv.shift - 4)) + Step<W>::UNITS - 1) / Step<W>::UNITS
              : t.from < t.to ? (t.to - 1 - (t.base << p.kv.shift)) / Step<W>::KEYS + 1 : 0;
    seg.unit = job - t.row * per_row;
    seg.kvh = p.parts == 1 ? seg.unit : seg.unit / p.parts;
    const uint32_t hp = seg.unit - seg.kvh * p.parts;
    seg.head0 = seg.kvh * p.group + hp * p.part;
    seg.part = min(p.part, p.group - hp * p.part);
    const uint32_t each = (t.steps + kWarps * blocks - 1) / (kWarps * blocks);
    seg.begin = worker * each;
    seg.end = min(t.steps, seg.begin + each);
    seg.partial = true;
    static_assert(16 * W * sizeof(float) <= kStages * kStage, "a warp's ring holds its partial results");
    seg.part_o = reinterpret_cast<float *>(smem + warp * (kStages * kStage));  // its ring is empty by then
    seg.part_ml = reinterpret_cast<float *>(sm_ml[warp]);
    if (lane < 16) sm_ml[warp][lane] = make_float2(-INFINITY, 0.0f);
    __syncwarp();
    if (seg.begin < seg.end && t.from < t.to) {
        const Group group = group_of<LIST>(p, t, seg.kvh, (seg.begin * Step<W>::UNITS) >> (p.kv.shift - 4), lane);
        const Following none = {{kNoBlock, 0, 0.0f, 0.0f}, 0, 0, 0};
        if (seg.part <= 8) attend_steps<W, 1, LIST, ONE>(p, &map_k, &map_v, seg, group, 0, none, [] {}, ring, status, lane);
        else attend_steps<W, 2, LIST, ONE>(p, &map_k, &map_v, seg, group, 0, none, [] {}, ring, status, lane);
    }
    cluster_sync();
    // Block `rank` folds its share of the row's heads' channels, four at a time, in the order of the keys: worker = warp *
    // blocks + rank.
    for (uint32_t i = (rank * kThreads + threadIdx.x) * 4; i < seg.part * W; i += blocks * kThreads * 4) {
        const uint32_t m = i / W, d = i % W;
        const uint32_t ml_at = smem_addr(&sm_ml[0][m]), o_at = smem_addr(smem) + (m * W + d) * 4;
        float top = -INFINITY;
        for (uint32_t w = 0; w < kWarps; w++)
#pragma unroll 4
            for (uint32_t b = 0; b < blocks; b++) top = fmaxf(top, ld_cluster_f32x2(map_to_rank(ml_at + w * (uint32_t)sizeof(sm_ml[0]), b)).x);
        if (top == -INFINITY) top = 0.0f;
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t w = 0; w < kWarps; w++)
#pragma unroll 4
            for (uint32_t b = 0; b < blocks; b++) {
                const float2 ml = ld_cluster_f32x2(map_to_rank(ml_at + w * (uint32_t)sizeof(sm_ml[0]), b));
                const float4 v = ld_cluster_f32x4(map_to_rank(o_at + w * (kStages * kStage), b));
                const float f = exp2_approx(ml.x - top);
                l = fmaf(ml.y, f, l);
                if (ml.x != -INFINITY) {  // else nobody wrote there (NaN scores leave -infinity too, and NaN in l)
                    o.x = fmaf(v.x, f, o.x);
                    o.y = fmaf(v.y, f, o.y);
                    o.z = fmaf(v.z, f, o.z);
                    o.w = fmaf(v.w, f, o.w);
                }
            }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint2 *>(p.out + ((size_t)t.row * p.heads + seg.head0 + m) * W + d) =
            make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
    pdl_launch_dependents();
    cluster_sync();  // the other blocks have read this one's shared memory
}

__device__ int g_attend_status = 0;

struct Plan {
    uint32_t part, parts, tokens, workers, together, whole, cluster;
    bool merged;
    size_t o_bytes, ml_bytes, places_bytes;
    size_t bytes() const { return merged && !cluster ? o_bytes + ml_bytes + places_bytes : 0; }
};

Plan plan_of(uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t back, uint32_t count,
             uint32_t block) {
    Plan s;
    const uint32_t group = heads / kv_heads, step = kHalfStage / width;
    s.part = group < 16 ? group : 16;
    s.parts = ceil_div(group, s.part);
    s.tokens = count || s.parts > 1 ? 1 : 16 / s.part;
    uint64_t span = keys;  // keys a tile may see; the first of them is anywhere in its block of 64 at most
    if (!count && (uint64_t)back + s.tokens < span) span = (uint64_t)back + s.tokens;
    const uint64_t offset = !count && span < keys ? 63 : 0;
    const uint64_t steps = count ? ((uint64_t)count * block + step - 1) / step : (span + offset + step - 1) / step;
    const uint64_t most = (uint64_t)sm_count() * kBlocks * kWarps;
    const uint64_t each = (uint64_t)kv_heads * s.parts * steps;  // steps of a row at most
    // The kernel counts steps in 32 bits: more rows than that allows go in several launches, whole tiles each.
    uint64_t together = 0x7FFFFFFFull / each / s.tokens * s.tokens;
    s.together = (uint32_t)(rows < together ? rows : together);
    // A tile of up to four steps is not worth cutting: a worker does it in less time than a second kernel takes.
    s.merged = steps > 4;
    s.whole = steps <= 1 ? 1 : (uint32_t)(steps < 4 ? steps : 4);
    // (Where not even one tile's steps fit, the call reads less, its slots' room, or is refused: workspace as for one tile.)
    const uint64_t planned = s.together ? s.together : min(rows, s.tokens);
    const uint64_t jobs = s.merged ? planned * each : planned * (each / steps);
    s.workers = (uint32_t)(jobs < most ? jobs : most);
    // A cluster for each row and kv head, as small as leaves a warp two steps, or four: where all of them are resident at once.
    s.cluster = 0;
    const uint64_t rows_heads = (uint64_t)rows * kv_heads * s.parts;
    for (uint32_t most_steps = 2; most_steps <= 4 && !s.cluster; most_steps += 2)
        for (uint32_t c = 1; c <= 8 && !s.cluster; c *= 2)
            if (rows_heads * c <= (uint64_t)sm_count() * kBlocks && steps <= (uint64_t)most_steps * kWarps * c) s.cluster = c;
    s.o_bytes = (size_t)s.workers * 2 * s.tokens * s.part * width * sizeof(float);
    s.ml_bytes = align_up((size_t)s.workers * 2 * s.tokens * s.part * 2 * sizeof(float), 16);
    s.places_bytes = (size_t)rows * kv_heads * s.parts * sizeof(uint4);
    return s;
}

template <int W, bool LIST, bool ONE>
int launch_attend(const AttendParams &p, cudaStream_t stream) {
    constexpr size_t smem = kWarps * kStages * kStage;
    static OncePerDevice configured;
    if (configured.needs()) {
        TS_CUDA(cudaFuncSetAttribute(attend_q8_kernel<W, LIST, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        configured.done();
    }
    int *status = nullptr;
    TS_CUDA(cudaGetSymbolAddress((void **)&status, g_attend_status));
    // Codes as rows of `width` bytes; a copy takes up to a block's rows of one kv head.
    CUtensorMap map_k, map_v;
    const uint64_t rows = ((uint64_t)p.kv.blocks * p.kv_heads) << p.kv.shift;
    const uint32_t box = min(1u << p.kv.shift, (uint32_t)Step<W>::KEYS);
    int rc = make_tensor_map_codes(&map_k, p.kv.k, rows, W, Step<W>::COLS, box);
    if (rc == TS_OK) rc = make_tensor_map_codes(&map_v, p.kv.v, rows, W, Step<W>::COLS, box);
    if (rc != TS_OK) return rc;
    if (p.cluster) {
        static OncePerDevice ready;
        if (ready.needs()) {
            TS_CUDA(cudaFuncSetAttribute(attend_q8_cluster_kernel<W, LIST, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            ready.done();
        }
        cudaLaunchAttribute attr[2] = {};
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = p.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(p.rows * p.kv_heads * p.parts * p.cluster);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, attend_q8_cluster_kernel<W, LIST, ONE>, map_k, map_v, p, status);
        if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of attend (q8, cluster) failed: %s", cudaGetErrorString(e));
        return TS_OK;
    }
    const uint32_t grid = min(p.workers, (uint32_t)sm_count() * kBlocks);
    cudaError_t e = launch(attend_q8_kernel<W, LIST, ONE>, dim3(grid), dim3(kThreads), smem, stream, pdl_enabled(), map_k, map_v, p, status);
    if (e == cudaSuccess && p.merged)  // always as a dependent launch: it waits for the partials itself
        e = p.rows * p.heads > (uint32_t)sm_count() * 8
                ? launch(attend_q8_merge_kernel<W, 64>, dim3(p.rows * p.heads), dim3(64), p.workers * sizeof(float), stream, true, p)
                : launch(attend_q8_merge_kernel<W, 256>, dim3(p.rows * p.heads), dim3(256), p.workers * sizeof(float), stream, true, p);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of attend (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

// Blocks that hold whole steps of keys need one look-up, copy and scale a step.
template <int W>
int launch_attend(const AttendParams &p, cudaStream_t stream) {
    if (Step<W>::UNITS == 1 || (1u << p.kv.shift) >= (uint32_t)Step<W>::KEYS)
        return p.ids ? launch_attend<W, true, true>(p, stream) : launch_attend<W, false, true>(p, stream);
    if constexpr (Step<W>::UNITS > 1)
        return p.ids ? launch_attend<W, true, false>(p, stream) : launch_attend<W, false, false>(p, stream);
}

}  // namespace

int attend_q8_take_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attend_status, sizeof(int)) != cudaSuccess) return TS_ERR_CUDA;
    if (v != 0) cudaMemcpyToSymbol(g_attend_status, &zero, sizeof(int));
    return v;
}

size_t attend_q8_workspace_bytes(uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t back,
                                 uint32_t count, uint32_t block) {
    if (rows == 0 || keys == 0 || heads == 0 || kv_heads == 0 || heads % kv_heads) return 0;
    if (width != 64 && width != 128 && width != 256) return 0;
    // sizes that the calls refuse (a count of blocks and keys past 32 bits would overflow the plan's steps)
    if ((block != 16 && block != 32 && block != 64) || count > kMostListed || kv_heads > 65535) return 0;
    return plan_of(rows, keys, heads, kv_heads, width, back, count, block).bytes();
}

int attend_q8(const void *q, const RowsQ8Dev &kv, const uint32_t *ids, void *out, const uint32_t *slots,
              const uint32_t *positions, uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width,
              uint32_t back, uint32_t count, float scale, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    // A slot has no keys past what its stride or its pages hold (and fewer keys never ask for a larger workspace).
    const uint64_t room = (uint64_t)kv.scalar << (kv.per_shift + kv.shift);
    if (room < keys) keys = (uint32_t)room;
    if (keys > kNoKeys) keys = kNoKeys;
    const Plan s = plan_of(rows, keys, heads, kv_heads, width, back, count, 1u << kv.shift);
    const size_t need = s.bytes();
    TS_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && aligned16(workspace))),
               "attend (q8): workspace of %zu bytes is smaller than the %zu needed, or not 16-byte aligned", workspace_bytes, need);
    TS_REQUIRE(q != out, "attend (q8): out is where q lies, which other blocks still read");
    TS_REQUIRE((uint64_t)rows * heads < 0x7FFFFFFFull, "attend (q8): %u rows are too many for one launch", rows);
    TS_REQUIRE((((uint64_t)kv.blocks * kv_heads) << kv.shift) < 0x7FFFFFFFull, "attend (q8): a pool of %u blocks is too large", kv.blocks);
    TS_REQUIRE(s.together > 0, "attend (q8): %u keys of %u kv heads are too many for one launch", keys, kv_heads);
    AttendParams p = {};
    p.q = (const uint16_t *)q;
    p.kv = kv;
    p.ids = ids;
    p.out = (uint16_t *)out;
    p.slots = slots;
    p.positions = positions;
    p.rows = rows;
    p.keys = keys;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.back = back;
    p.count = count;
    p.group = heads / kv_heads;
    p.part = s.part;
    p.parts = s.parts;
    p.tokens = s.tokens;
    p.most = s.tokens * s.part;
    p.workers = s.workers;
    p.merged = s.merged;
    p.whole = s.whole;
    p.cluster = s.cluster;
    p.scale = scale;
    if (need) {
        p.part_o = (float *)workspace;
        p.part_ml = (float *)((uint8_t *)workspace + s.o_bytes);
        p.places = (uint4 *)((uint8_t *)workspace + s.o_bytes + s.ml_bytes);
    }
    for (uint32_t row = 0; row < rows; row += s.together) {
        p.q = (const uint16_t *)q + (size_t)row * heads * width;
        p.out = (uint16_t *)out + (size_t)row * heads * width;
        p.ids = ids ? ids + (size_t)row * kv_heads * count : nullptr;
        p.slots = slots + row;
        p.positions = positions + row;
        p.rows = min(s.together, rows - row);
        const int rc = width == 64    ? launch_attend<64>(p, stream)
                       : width == 128 ? launch_attend<128>(p, stream)
                                      : launch_attend<256>(p, stream);
        if (rc != TS_OK) return rc;
    }
    return TS_OK;
}

}  // namespace ts
