// Ragged attention over kept rows in 8 bits, whole slots or listed blocks.
//
// A tile is up to 16 query rows, (token, head) pairs: the G heads of a kv head's group times up to T = 16 / G neighbouring
// rows that are the next positions of one slot (drafted tokens, a part of a prompt).  Both products run on warp MMAs
// (m16n8k16, f16 in, f32 out) with the keys, then the channels, as the 16 rows and the queries as the 8 columns:
//     S^T[16 keys x 8 queries] = K Q^T,      O^T[16 channels x 8 queries] += V^T P^T
// so that a decode row of up to eight heads wastes nothing of the accumulators, and a second eight of queries shares the
// converted K and V.  (With the queries as rows, half of every accumulator quad of a decode row is padding: 64 more
// registers and twice the MMAs.)  A code is exact in f16: the bytes are set as the low bits of 1024 + (128 + code) and 1152
// is subtracted; a query row is brought into f16's range by a power of two, which is exact for bf16 (values below 2^-24
// of the row's largest lose digits that no sum would keep).
//
// The scales leave the products alone.  With s = raw * scale * k_scale in powers of two and
//     x = s + log2(v_scale),   M = max x,   P = 2^(x - M)  <= 1   (f16 operand of P V)
// the output is sum P code / sum P / v_scale: the block's value scale rides in the exponent, so that P needs no second
// factor and stays within f16's range whatever the scales are, and M cancels.  A scale of zero counts as 2^-60, the
// smallest that append writes.
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
// every run.  With little work every tile is cut into pieces of four steps instead.
#include <cmath>

#include "rows_q8.cuh"
#include "ts_ptx.cuh"

namespace ts {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kHalfStage = 4096, kStage = 2 * kHalfStage;  // K codes, then V codes
constexpr int kPiece = 4;                                  // steps of a worker's run at least
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kScaleFloor = 8.673617379884035e-19f;  // 2^-60

// Blocks an SM holds and stages a warp has.  Twelve warps keep the issue slots busy where registers allow it (width
// 256 needs up to 255 of them).
template <int W>
struct Shape {
    static constexpr int CTAS = W == 256 ? 2 : 3, STAGES = W == 256 ? 3 : 2;
};

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
// Two of the four biased codes (code + 128) as f16: bytes 0, 1 (0x4140), 2, 3 (0x4342), 0, 2 (0x4240) or 1, 3 (0x4341).
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

// The tile that begins at `row`; false if the row lies in a tile that begins before it.
template <int W, bool LIST>
__device__ __forceinline__ bool tile_of(const AttendParams &p, uint32_t row, Tile *t) {
    t->row = row;
    t->tokens = 1;
    t->slot = p.slots[row];
    if (!LIST && p.tokens > 1) {
        // Tiles begin at multiples of `tokens` and where a row is not the next position of the slot before it (or the same
        // again).
        auto follows = [&](uint32_t r) {
            if (r % p.tokens == 0 || p.slots[r] != p.slots[r - 1]) return false;  // also: row 0 has none before it
            const uint32_t was = p.positions[r - 1], is = p.positions[r];
            return is >= was && is - was <= 1u;
        };
        if (follows(row)) return false;
        while (row + t->tokens < p.rows && follows(row + t->tokens)) t->tokens++;
    }
    // positions ascend within a tile: the first row sees the earliest key, the last one the latest
    uint32_t a, b;
    seen(p, p.positions[row], &t->from, &b);
    seen(p, p.positions[row + t->tokens - 1], &a, &t->to);
    if (t->from >= t->to) t->from = t->to = 0;
    if (LIST) {
        t->base = 0;
        t->entries = p.count;
        t->steps = ((p.count << (p.kv.shift - 4)) + Step<W>::UNITS - 1) / Step<W>::UNITS;
    } else {
        t->base = t->from >> p.kv.shift;
        t->entries = t->from < t->to ? ((t->to - 1) >> p.kv.shift) + 1 - t->base : 0;
        t->steps = t->from < t->to ? (t->to - 1 - (t->base << p.kv.shift)) / Step<W>::KEYS + 1 : 1;
    }
    return true;
}

__device__ __forceinline__ uint32_t warp_total(uint32_t v) { return __reduce_add_sync(0xFFFFFFFFu, v); }

// ---- the query operand: column r of eight is tile row 8 t + r; thread j of its four has channels 16 s + 4 j + 0..3 ----
template <int W, int NT>
struct Queries {
    uint32_t b[NT][W / 16][2];
    float f[NT][2];            // raw score -> power-of-two exponent, without the key scale, for columns 2 j, 2 j + 1
    uint32_t lo[NT][2], hi[NT][2];  // keys those columns see
};

template <int W, int NT>
__device__ __forceinline__ void load_queries(const AttendParams &p, const Tile &tile, uint32_t head0, uint32_t part, uint32_t lane,
                                             Queries<W, NT> &qs) {
    const uint32_t r = lane >> 2, j = lane & 3;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const uint32_t m = 8 * t + r, token = m / part, head = m - token * part;
        uint2 v[W / 16];
        float most = 0.0f;
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            v[s] = make_uint2(0, 0);
            if (token < tile.tokens) v[s] = *reinterpret_cast<const uint2 *>(p.q + ((size_t)(tile.row + token) * p.heads + head0 + head) * W + 16 * s + 4 * j);
        }
#pragma unroll
        for (int s = 0; s < W / 16; s++)
            most = fmaxf(most, fmaxf(fmaxf(fabsf(bf16_lo(v[s].x)), fabsf(bf16_hi(v[s].x))), fmaxf(fabsf(bf16_lo(v[s].y)), fabsf(bf16_hi(v[s].y)))));
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
        uint32_t e = __float_as_uint(most) >> 23;  // the largest magnitude's exponent; 255: infinity
        e = e < 1 ? 1 : e > 253 ? 253 : e;
        const float down = __uint_as_float((254 - e) << 23), f = __uint_as_float(e << 23) * (p.scale * kLog2e);
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            qs.b[t][s][0] = pack_f16(bf16_lo(v[s].x) * down, bf16_hi(v[s].x) * down);
            qs.b[t][s][1] = pack_f16(bf16_lo(v[s].y) * down, bf16_hi(v[s].y) * down);
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

// One step.  EDGE: some key of it is not seen by some row.  A unit without keys has key0 past every row's.
template <int W, int NT, bool EDGE>
__device__ __forceinline__ void step(const Queries<W, NT> &qs, Running<W, NT> &run, uint32_t tile, const float (&ks)[Step<W>::UNITS],
                                     const float (&vs)[Step<W>::UNITS], const uint32_t (&key0)[Step<W>::UNITS], uint32_t lane) {
    constexpr int U = Step<W>::UNITS;
    const uint32_t r = lane >> 2;
    float x[U][NT][4], most[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++) most[t][0] = most[t][1] = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int t = 0; t < NT; t++) x[u][t][0] = x[u][t][1] = x[u][t][2] = x[u][t][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < W / 16; c += 2) {
            uint32_t w[4];
            ldsm_x4(piece_at<W>(tile, u, c, lane), w);
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] ^= 0x80808080u;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t a0 = codes_f16(w[2 * i], 0x4140), a1 = codes_f16(w[2 * i + 1], 0x4140), a2 = codes_f16(w[2 * i], 0x4342),
                               a3 = codes_f16(w[2 * i + 1], 0x4342);
#pragma unroll
                for (int t = 0; t < NT; t++) mma_f16(x[u][t], a0, a1, a2, a3, qs.b[t][c + i]);
            }
        }
        const float lv = log2_approx(fmaxf(vs[u], kScaleFloor));
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float f = qs.f[t][e] * ks[u];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float &y = x[u][t][2 * k + e];
                    y = fmaf(y, f, lv);
                    if (EDGE) {
                        const uint32_t key = key0[u] + 8 * k + r;
                        if (key < qs.lo[t][e] || key >= qs.hi[t][e]) y = -INFINITY;
                    }
                    most[t][e] = fmaxf(most[t][e], y);
                }
            }
    }
    float scale[NT][2], top[NT][2];
    bool same = true;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) most[t][e] = fmaxf(most[t][e], __shfl_xor_sync(0xFFFFFFFFu, most[t][e], o));
            const float now = fmaxf(run.m[t][e], most[t][e]);
            top[t][e] = now == -INFINITY ? 0.0f : now;  // nothing seen yet: 2^(-inf - 0) = 0
            scale[t][e] = exp2_approx(run.m[t][e] - top[t][e]);
            same = same && scale[t][e] == 1.0f;
            run.m[t][e] = now;
            run.l[t][e] *= scale[t][e];
        }
    if (!__all_sync(0xFFFFFFFFu, same)) {
#pragma unroll
        for (int i = 0; i < W / 16; i++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    run.o[i][t][e] *= scale[t][e];
                    run.o[i][t][2 + e] *= scale[t][e];
                }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const float inv = __fdividef(1.0f, fmaxf(vs[u], kScaleFloor));
        uint32_t b[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                p[e] = exp2_approx(x[u][t][e] - top[t][e]);
                p[2 + e] = exp2_approx(x[u][t][2 + e] - top[t][e]);
                run.l[t][e] = fmaf(p[e] + p[2 + e], inv, run.l[t][e]);
            }
            b[t][0] = transpose_8x8(pack_f16(p[0], p[1]));
            b[t][1] = transpose_8x8(pack_f16(p[2], p[3]));
        }
#pragma unroll
        for (int c = 0; c < W / 16; c += 2) {
            uint32_t w[4];
            ldsm_x4_trans(piece_at<W>(tile + kHalfStage, u, c, lane), w);
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] ^= 0x80808080u;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t a0 = codes_f16(w[2 * i], 0x4240), a1 = codes_f16(w[2 * i], 0x4341), a2 = codes_f16(w[2 * i + 1], 0x4240),
                               a3 = codes_f16(w[2 * i + 1], 0x4341);
#pragma unroll
                for (int t = 0; t < NT; t++) mma_f16(run.o[c + i][t], a0, a1, a2, a3, b[t]);
            }
        }
    }
}

// 32 blocks' places in the pool and scales, one a lane: entry `first` + lane of the tile's blocks.
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

// A warp's ring: the next stage to complete and the parity each completes with.
struct Ring {
    uint32_t tiles;  // shared-memory address
    uint64_t *full;
    uint32_t stage, parity;
    bool ok;  // false: a wait ran out, nothing is copied or computed any more
};

// Where a tile's result goes: the output, or a partial.
struct Target {
    bool partial;
    size_t slot;  // worker * 2 + 0 or 1
};

template <int W, int NT, bool LIST>
__device__ __forceinline__ void attend_steps(const AttendParams &p, const CUtensorMap *map_k, const CUtensorMap *map_v, const Tile &tile,
                                             uint32_t kvh, uint32_t head0, uint32_t part, uint32_t begin, uint32_t end, Target to,
                                             Ring &ring, int *status, uint32_t lane) {
    using namespace ptx;
    constexpr int KEYS = Step<W>::KEYS, U = Step<W>::UNITS, HALVES = Step<W>::HALVES, COLS = Step<W>::COLS, STAGES = Shape<W>::STAGES;
    const uint32_t in_block = p.kv.shift - 4;  // log2 of a block's 16-key units
    Running<W, NT> run;
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int i = 0; i < W / 16; i++) run.o[i][t][0] = run.o[i][t][1] = run.o[i][t][2] = run.o[i][t][3] = 0.0f;
        run.m[t][0] = run.m[t][1] = -INFINITY;
        run.l[t][0] = run.l[t][1] = 0.0f;
    }
    if (tile.from < tile.to) {
        uint32_t first = (begin * U) >> in_block;  // entry of lane 0 of the current group
        Group now = group_of<LIST>(p, tile, kvh, first, lane);
        Group next = group_of<LIST>(p, tile, kvh, first + 32, lane);
        // Copies of step s into stage `at`; the current or the next group has its blocks.
        auto copy = [&](uint32_t s, uint32_t at) {
            const uint32_t dst = ring.tiles + at * kStage, bar = smem_addr(&ring.full[at]);
            uint32_t blk[U], bytes = 0;
            const uint32_t per = 1u << in_block, span = per < (uint32_t)U ? per : U;  // units of one copy
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t e = ((s * U + u) >> in_block) - first;
                const uint32_t a = __shfl_sync(0xFFFFFFFFu, now.blk, e & 31), b = __shfl_sync(0xFFFFFFFFu, next.blk, e & 31);
                blk[u] = e < 32 ? a : b;
                if ((u & (span - 1)) == 0 && blk[u] != kNoBlock) bytes += span * 16 * W * 2;
            }
            if (lane == 0) {
                mbar_expect_tx(&ring.full[at], bytes);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if ((u & (span - 1)) != 0 || blk[u] == kNoBlock) continue;
                    const int32_t y = (int32_t)(((blk[u] * p.kv_heads + kvh) << p.kv.shift) + (((s * U + u) & (per - 1)) << 4));
#pragma unroll
                    for (int h = 0; h < HALVES; h++) {
                        copy_codes(dst + (h * KEYS + 16 * u) * COLS, map_k, bar, h * COLS, y);
                        copy_codes(dst + kHalfStage + (h * KEYS + 16 * u) * COLS, map_v, bar, h * COLS, y);
                    }
                }
            }
        };
        uint32_t ahead = begin;
        for (; ahead < end && ahead < begin + STAGES; ahead++) copy(ahead, (ring.stage + (ahead - begin)) % STAGES);
        Queries<W, NT> qs;
        load_queries<W, NT>(p, tile, head0, part, lane, qs);
        uint32_t all_lo = 0, all_hi = 0;  // keys that every row of the tile sees
        {
            uint32_t x;
            seen(p, p.positions[tile.row], &x, &all_hi);
            seen(p, p.positions[tile.row + tile.tokens - 1], &all_lo, &x);
        }
        for (uint32_t s = begin; s < end; s++) {
            if (((s * U) >> in_block) - first >= 32) {
                first += 32;
                now = next;
                next = group_of<LIST>(p, tile, kvh, first + 32, lane);
            }
            float ks[U], vs[U];
            uint32_t key0[U];
            bool edge = false;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t unit = s * U + u, e = ((unit >> in_block) - first) & 31;
                ks[u] = __shfl_sync(0xFFFFFFFFu, now.ks, e);
                vs[u] = __shfl_sync(0xFFFFFFFFu, now.vs, e);
                const uint32_t blk = __shfl_sync(0xFFFFFFFFu, now.blk, e), id = __shfl_sync(0xFFFFFFFFu, now.id, e);
                key0[u] = blk == kNoBlock ? 0xFFFFFFF0u : (id << p.kv.shift) + ((unit & ((1u << in_block) - 1)) << 4);
                edge = edge || key0[u] < all_lo || key0[u] + 16 > all_hi || blk == kNoBlock;
            }
            ring.ok = mbar_wait(&ring.full[ring.stage], ring.parity >> ring.stage & 1);
            ring.parity ^= 1u << ring.stage;
            if (!__all_sync(0xFFFFFFFFu, ring.ok)) {
                ring.ok = false;  // the other copies are waited for, as long, before the block may end
                for (uint32_t i = s + 1; i < ahead; i++) {
                    ring.stage = (ring.stage + 1) % STAGES;
                    mbar_wait(&ring.full[ring.stage], ring.parity >> ring.stage & 1);
                }
                if (lane == 0) atomicExch(status, TS_ERR_TIMEOUT);
                return;
            }
            const uint32_t at = ring.tiles + ring.stage * kStage;
            if (edge) step<W, NT, true>(qs, run, at, ks, vs, key0, lane);
            else step<W, NT, false>(qs, run, at, ks, vs, key0, lane);
            __syncwarp();
            if (ahead < end) {
                copy(ahead, ring.stage);
                ahead++;
            }
            ring.stage = (ring.stage + 1) % STAGES;
        }
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
            if (!to.partial) {
                const uint32_t token = m / part;
                uint16_t *out = p.out + ((size_t)(tile.row + token) * p.heads + head0 + m - token * part) * W + 2 * r;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int i = 0; i < W / 16; i++)
                    *reinterpret_cast<uint32_t *>(out + 16 * i) = pack_bf16(run.o[i][t][e] * inv, run.o[i][t][2 + e] * inv);
            } else {
                float *o = p.part_o + (to.slot * p.most + m) * W + 2 * r;
#pragma unroll
                for (int i = 0; i < W / 16; i++) *reinterpret_cast<float2 *>(o + 16 * i) = make_float2(run.o[i][t][e], run.o[i][t][2 + e]);
                if (r == 0) *reinterpret_cast<float2 *>(p.part_ml + (to.slot * p.most + m) * 2) = make_float2(run.m[t][e], l);
            }
        }
}

template <int W, bool LIST>
__global__ void __launch_bounds__(kThreads, Shape<W>::CTAS)
attend_q8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttendParams p, int *status) {
    using namespace ptx;
    constexpr int STAGES = Shape<W>::STAGES;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][STAGES];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t worker = warp * gridDim.x + blockIdx.x;  // few workers spread over the SMs
    Ring ring = {smem_addr(smem) + warp * (STAGES * kStage), bars[warp], 0, 0, true};
    if (lane == 0) {
        for (int s = 0; s < STAGES; s++) mbar_init(&ring.full[s], 1);
        fence_barrier_init();
    }
    __syncwarp();
    pdl_wait();
    if (worker < p.workers) {
        // ---- the steps of all tiles, and this worker's run of them ----
        const uint32_t per_row = p.kv_heads * p.parts;
        auto steps_of = [&](uint32_t row) {
            Tile t;
            return row < p.rows && tile_of<W, LIST>(p, row, &t) ? t.steps : 0u;
        };
        uint64_t steps = 0, pieces = 0;
        if (LIST) {
            const uint32_t n = steps_of(0);
            steps = (uint64_t)n * p.rows;
            pieces = (uint64_t)((n + kPiece - 1) / kPiece) * p.rows;
        } else {
            for (uint32_t base = 0; base < p.rows; base += 32) {
                const uint32_t n = steps_of(base + lane);
                steps += warp_total(n);
                pieces += warp_total((n + kPiece - 1) / kPiece);
            }
        }
        const bool padded = pieces * per_row <= p.workers;  // every tile in pieces of its own
        const uint64_t total = (padded ? pieces * kPiece : steps) * per_row;
        const uint32_t run = padded ? kPiece : (uint32_t)((total + p.workers - 1) / p.workers);
        uint64_t at = (uint64_t)worker * run;
        const uint64_t end = at + run < total ? at + run : total;
        // the row in whose steps the run begins
        uint64_t before = 0;  // steps of earlier rows, all kv heads
        uint32_t row = 0;
        if (at < end) {
            auto taken = [&](uint32_t n) { return (uint64_t)(padded ? (n + kPiece - 1) / kPiece * kPiece : n) * per_row; };
            if (LIST) {
                const uint64_t each = taken(steps_of(0));
                row = (uint32_t)(at / each);
                before = row * each;
            } else {
                for (uint32_t base = 0; base < p.rows; base += 32) {
                    const uint32_t n = steps_of(base + lane);
                    uint64_t mine = taken(n), sum = mine;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint64_t other = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                        if (lane >= (uint32_t)o) sum += other;
                    }
                    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + sum > at);
                    if (hit) {
                        const int l = __ffs(hit) - 1;
                        row = base + l;
                        before += __shfl_sync(0xFFFFFFFFu, sum - mine, l);
                        break;
                    }
                    before += __shfl_sync(0xFFFFFFFFu, sum, 31);
                }
            }
            bool begun = false;  // whether the run has had a tile already
            while (at < end && row < p.rows && ring.ok) {
                Tile tile;
                if (!tile_of<W, LIST>(p, row, &tile)) {
                    row++;
                    continue;
                }
                const uint32_t n = padded ? (tile.steps + kPiece - 1) / kPiece * kPiece : tile.steps;
                while (at < end && at < before + (uint64_t)n * per_row && ring.ok) {
                    const uint32_t h = (uint32_t)((at - before) / n), s0 = (uint32_t)((at - before) % n);
                    const uint64_t start = at - s0;
                    const uint32_t s1 = (uint32_t)min((uint64_t)n, end - start);
                    const uint32_t kvh = h / p.parts, hp = h % p.parts;
                    const uint32_t head0 = kvh * p.group + hp * p.part, part = min(p.part, p.group - hp * p.part);
                    const uint32_t w0 = (uint32_t)(start / run), w1 = (uint32_t)((start + tile.steps - 1) / run);
                    if (s0 == 0 && p.merged && lane < tile.tokens)
                        p.places[(size_t)(row + lane) * per_row + h] = make_uint4(w0, w1, start % run != 0, lane * part);
                    const Target to = {w0 != w1, (size_t)worker * 2 + begun};
                    const uint32_t stop = min(s1, tile.steps);
                    if (tile.tokens * part <= 8)
                        attend_steps<W, 1, LIST>(p, &map_k, &map_v, tile, kvh, head0, part, s0, stop, to, ring, status, lane);
                    else
                        attend_steps<W, 2, LIST>(p, &map_k, &map_v, tile, kvh, head0, part, s0, stop, to, ring, status, lane);
                    begun = true;
                    at = start + s1;
                }
                before += (uint64_t)n * per_row;
                row++;
            }
        }
    }
    pdl_launch_dependents();
}

// One block per (row, head): folds the partials of its tile in the order of their keys.
template <int W>
__global__ void __launch_bounds__(W) attend_q8_merge_kernel(const AttendParams p) {
    pdl_wait();
    const uint32_t row = blockIdx.x / p.heads, head = blockIdx.x % p.heads, d = threadIdx.x;
    const uint32_t kvh = head / p.group, in = head % p.group, hp = in / p.part;
    const uint4 place = p.places[((size_t)row * p.kv_heads + kvh) * p.parts + hp];
    const uint32_t m = place.w + in % p.part;
    if (place.x < place.y && place.y < p.workers && place.z < 2 && m < p.most) {  // else its one worker wrote it (or gave up)
        auto slot = [&](uint32_t w) { return ((size_t)w * 2 + (w == place.x ? place.z : 0)) * p.most + m; };
        float top = -INFINITY;
        for (uint32_t w = place.x; w <= place.y; w++) top = fmaxf(top, p.part_ml[slot(w) * 2]);
        const float z = top == -INFINITY ? 0.0f : top;
        float l = 0.0f, o = 0.0f;
        for (uint32_t w = place.x; w <= place.y; w++) {
            const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + slot(w) * 2);
            const float f = exp2_approx(ml.x - z);
            l = fmaf(ml.y, f, l);
            o = fmaf(p.part_o[slot(w) * W + d], f, o);
        }
        p.out[((size_t)row * p.heads + head) * W + d] = l == 0.0f ? (uint16_t)0 : bf16_bits(o / l);
    }
    pdl_launch_dependents();
}

__device__ int g_attend_status = 0;

struct Plan {
    uint32_t part, parts, tokens, workers;
    bool merged;
    size_t o_bytes, ml_bytes, places_bytes;
    size_t bytes() const { return merged ? o_bytes + ml_bytes + places_bytes : 0; }
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
    const uint64_t steps = count ? ((uint64_t)count * block + step - 1) / step : (span + 63 + step - 1) / step;
    const uint64_t most = (uint64_t)sm_count() * (width == 256 ? Shape<256>::CTAS : Shape<128>::CTAS) * kWarps;
    const uint64_t pieces = (uint64_t)rows * kv_heads * s.parts * ((steps + kPiece - 1) / kPiece);
    s.workers = (uint32_t)(pieces < most ? pieces : most);
    // Without a second kernel only where no tile can be cut: each fits one piece and there is a worker for every piece.
    s.merged = steps > kPiece || pieces > most;
    s.o_bytes = (size_t)s.workers * 2 * s.tokens * s.part * width * sizeof(float);
    s.ml_bytes = align_up((size_t)s.workers * 2 * s.tokens * s.part * 2 * sizeof(float), 16);
    s.places_bytes = (size_t)rows * kv_heads * s.parts * sizeof(uint4);
    return s;
}

template <int W, bool LIST>
int launch_attend(const AttendParams &p, cudaStream_t stream) {
    constexpr size_t smem = kWarps * Shape<W>::STAGES * kStage;
    static OncePerDevice configured;
    if (configured.needs()) {
        TS_CUDA(cudaFuncSetAttribute(attend_q8_kernel<W, LIST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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
    const uint32_t grid = min(p.workers, (uint32_t)sm_count() * Shape<W>::CTAS);
    cudaError_t e = launch(attend_q8_kernel<W, LIST>, dim3(grid), dim3(kThreads), smem, stream, pdl_enabled(), map_k, map_v, p, status);
    if (e == cudaSuccess && p.merged)  // always as a dependent launch: it waits for the partials itself
        e = launch(attend_q8_merge_kernel<W>, dim3(p.rows * p.heads), dim3(W), 0, stream, true, p);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of attend (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
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
    return plan_of(rows, keys, heads, kv_heads, width, back, count, block).bytes();
}

int attend_q8(const void *q, const RowsQ8Dev &kv, const uint32_t *ids, void *out, const uint32_t *slots,
              const uint32_t *positions, uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width,
              uint32_t back, uint32_t count, float scale, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const Plan s = plan_of(rows, keys, heads, kv_heads, width, back, count, 1u << kv.shift);
    const size_t need = s.bytes();
    TS_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && aligned16(workspace))),
               "attend (q8): workspace of %zu bytes is smaller than the %zu needed, or not 16-byte aligned", workspace_bytes, need);
    TS_REQUIRE((uint64_t)rows * heads < 0x7FFFFFFFull, "attend (q8): %u rows are too many for one launch", rows);
    TS_REQUIRE((((uint64_t)kv.blocks * kv_heads) << kv.shift) < 0x7FFFFFFFull, "attend (q8): a pool of %u blocks is too large", kv.blocks);
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
    p.scale = scale;
    if (s.merged) {
        p.part_o = (float *)workspace;
        p.part_ml = (float *)((uint8_t *)workspace + s.o_bytes);
        p.places = (uint4 *)((uint8_t *)workspace + s.o_bytes + s.ml_bytes);
    }
    return width == 64    ? (ids ? launch_attend<64, true>(p, stream) : launch_attend<64, false>(p, stream))
           : width == 128 ? (ids ? launch_attend<128, true>(p, stream) : launch_attend<128, false>(p, stream))
                          : (ids ? launch_attend<256, true>(p, stream) : launch_attend<256, false>(p, stream));
}

}  // namespace ts
