// Kept rows in 8 bits: append (norm, rotation, block scales, key bounds) and reading rows back.
//
// Append.  A block of B positions has one scale per kv head, so the rows of a call that fall into one block are one
// unit of work: run = the neighbouring rows of a (slot, block), in a call of few rows all of them wherever they stand.  A
// long run (a prompt's) belongs to a team of warps for each kv head's keys and values: they take the block's positions in
// turn, keep the prepared values in shared memory and agree there on the largest magnitude.  A short run (a step's row)
// belongs to one warp, which keeps them in registers.  Either way every value is read once and rounded once.  Held codes are
// read and rewritten only when the scale grows (a new largest value: for values without a trend once in i rows at the
// block's i-th row).  Query heads go to warps of their own, eight heads of a row each when there are many.
//
// W / 8 lanes hold a head: lane i of them the four pairs 4 i .. 4 i + 3, elements 4 i + e and W / 2 + 4 i + e, so that
// loads are 8 bytes and stores of codes 4 a lane.
#include <cmath>
#include <type_traits>

#include "rows_q8.cuh"

namespace ts {

int rows_q8_to_dev(const char *what, const ts_rows_q8 *kv, const ts_kept *kept, uint32_t kv_heads, uint32_t width,
                   RowsQ8Dev *out) {
    TS_REQUIRE(kv && kept, "%s: the rows' record or the kept layout is NULL", what);
    TS_REQUIRE(kv->k && kv->v && kv->k_scale && kv->v_scale, "%s: codes or scales are NULL", what);
    TS_REQUIRE(aligned16(kv->k) && aligned16(kv->v) && (kv->k_bounds == nullptr || aligned16(kv->k_bounds)),
               "%s: codes and bounds must be 16-byte aligned", what);
    TS_REQUIRE(aligned4(kv->k_scale, kv->v_scale), "%s: scales must be 4-byte aligned", what);
    TS_REQUIRE(kv->block == 16 || kv->block == 32 || kv->block == 64, "%s: a block of %u positions is not 16, 32 or 64", what,
               kv->block);
    TS_REQUIRE(kv->blocks > 0 && kv->blocks < kNoBlock, "%s: the pool has no block count", what);
    TS_REQUIRE(width == 64 || width == 128 || width == 256, "%s: width %u is not 64, 128 or 256", what, width);
    TS_REQUIRE(kv_heads > 0 && kv_heads <= 65535, "%s: %u kv heads", what, kv_heads);
    TS_REQUIRE(kept->kind == TS_KEPT_DENSE || kept->kind == TS_KEPT_PAGED,
               "%s: 8-bit rows take a dense or a paged layout (kind %d)", what, kept->kind);
    RowsQ8Dev d = {};
    d.k = (int8_t *)kv->k;
    d.v = (int8_t *)kv->v;
    d.k_scale = kv->k_scale;
    d.v_scale = kv->v_scale;
    d.bounds = (int8_t *)kv->k_bounds;
    d.shift = kv->block == 16 ? 4 : kv->block == 32 ? 5 : 6;
    d.blocks = kv->blocks;
    if (kept->kind == TS_KEPT_DENSE) {
        TS_REQUIRE(kept->kept_scalar > 0 && kept->kept_scalar % kv->block == 0,
                   "%s: a slot's stride of %u rows is not a multiple of the block of %u", what, kept->kept_scalar, kv->block);
        d.scalar = kept->kept_scalar >> d.shift;
    } else {
        TS_REQUIRE(kept->page >= kv->block && (kept->page & (kept->page - 1)) == 0,
                   "%s: pages of %u rows do not hold whole blocks of %u", what, kept->page, kv->block);
        TS_REQUIRE(kept->table != nullptr && kept->table_len > 0 && kept->kept_scalar > 0,
                   "%s: a paged layout needs its page table, table_len and pages per slot", what);
        TS_REQUIRE(aligned4(kept->table), "%s: the page table must be 4-byte aligned", what);
        while ((kv->block << d.per_shift) < kept->page) d.per_shift++;
        d.scalar = kept->kept_scalar;
        d.table = kept->table;
        d.table_len = kept->table_len;
    }
    *out = d;
    return TS_OK;
}

namespace {

constexpr float kScaleFloor = 8.673617379884035e-19f;  // 2^-60
constexpr float kLargest = 3.3895313892515355e38f;    // the largest finite bf16

// Two f32 at a time: one instruction each on sm_100.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Cosine and sine of pos * f.  In 32 bits the product would be off by 0.006 radians at position 100000, so the angle is
// kept in turns as a 64-bit fraction: pos * round(2^64 f / 2 pi) modulo 2^64, whose rounding is below 1e-7 turns at any
// position.  The upper 32 bits, less whole quarters, are an angle within pi / 4, where the series of sine to the ninth
// and of cosine to the eighth power are off by 2e-9 and 3e-8.
__device__ __forceinline__ uint64_t turns_of(float f) {
    const double v = (double)f * 0.15915494309189535;  // 1 / 2 pi
    return __double2ull_rn((v - floor(v)) * 18446744073709551616.0);
}

// Of two pairs.
__device__ __forceinline__ void sine_cosine(uint32_t pos, uint64_t turns0, uint64_t turns1, float2 *s, float2 *c) {
    const uint32_t t[2] = {(uint32_t)((pos * turns0) >> 32), (uint32_t)((pos * turns1) >> 32)};
    const uint32_t quarter[2] = {(t[0] + (1u << 29)) >> 30, (t[1] + (1u << 29)) >> 30};
    const float2 x = mul2(make_float2((float)(int32_t)(t[0] - (quarter[0] << 30)), (float)(int32_t)(t[1] - (quarter[1] << 30))),
                          both(1.4629180792671596e-9f));  // 2 pi / 2^32
    const float2 x2 = mul2(x, x);
    float2 sine = fma2(x2, both(2.7557319e-6f), both(-1.9841270e-4f));
    sine = fma2(x2, sine, both(8.3333333e-3f));
    sine = fma2(x2, sine, both(-1.6666667e-1f));
    sine = fma2(mul2(x, x2), sine, x);
    float2 cosine = fma2(x2, both(2.4801587e-5f), both(-1.3888889e-3f));
    cosine = fma2(x2, cosine, both(4.1666667e-2f));
    cosine = fma2(x2, cosine, both(-0.5f));
    cosine = fma2(x2, cosine, both(1.0f));
    auto settle = [](float sine, float cosine, uint32_t quarter, float *s, float *c) {
        const bool swap = quarter & 1;
        const uint32_t a = __float_as_uint(swap ? cosine : sine), b = __float_as_uint(swap ? sine : cosine);
        *s = __uint_as_float(a ^ (quarter & 2) << 30);
        *c = __uint_as_float(b ^ ((quarter + 1) & 2) << 30);
    };
    settle(sine.x, cosine.x, quarter[0], &s->x, &c->x);
    settle(sine.y, cosine.y, quarter[1], &s->y, &c->y);
}

// What a lane holds of a head: lane i of the W / 8.
template <int W>
struct Lanes {
    static constexpr int PER_HEAD = W / 8, TOGETHER = 32 / PER_HEAD;  // lanes of a head; heads a warp holds at once
};

struct Raw {
    uint2 a, b;  // bf16 elements 4 i .. 4 i + 3 and W / 2 + 4 i ..
};

template <int W>
__device__ __forceinline__ Raw load_head(const uint16_t *src, uint32_t i) {
    return {*reinterpret_cast<const uint2 *>(src + 4 * i), *reinterpret_cast<const uint2 *>(src + W / 2 + 4 * i)};
}

// A lane's eight values as pairs: x[0], x[1] are elements 4 i .., x[2], x[3] elements W / 2 + 4 i ..
__device__ __forceinline__ void widen(const Raw &raw, float2 (&x)[4]) {
    const uint32_t w[4] = {raw.a.x, raw.a.y, raw.b.x, raw.b.y};
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = make_float2(bf16_lo(w[i]), bf16_hi(w[i]));
}

// 1 / rms of a head, from every lane's values.
template <int W>
__device__ __forceinline__ float inverse_rms(const float2 (&x)[4], float eps) {
    float2 sum = mul2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; i++) sum = fma2(x[i], x[i], sum);
    float ss = sum.x + sum.y;
#pragma unroll
    for (int o = 1; o < Lanes<W>::PER_HEAD; o <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    return rsqrtf(fmaf(ss, 1.0f / (float)W, eps));
}

// Norm (g: the lane's gains) and rotation, in 32 bits.
template <int W>
__device__ __forceinline__ void norm_turn(float2 (&x)[4], bool normed, const float2 (&g)[4], const float2 (&sn)[2], const float2 (&cs)[2],
                                          float eps) {
    if (normed) {
        const float2 inv = both(inverse_rms<W>(x, eps));
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = mul2(x[i], mul2(inv, g[i]));
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float2 a = x[e], b = x[2 + e];
        x[e] = fma2(a, cs[e], mul2(b, make_float2(-sn[e].x, -sn[e].y)));
        x[2 + e] = fma2(a, sn[e], mul2(b, cs[e]));
    }
}

template <int W>
__device__ __forceinline__ void load_gains(const float *gain, uint32_t i, float2 (&g)[4]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float *from = gain + h * (W / 2) + 4 * i;  // gains are as aligned as a float array is
        g[2 * h] = gain ? make_float2(from[0], from[1]) : both(1.0f);
        g[2 * h + 1] = gain ? make_float2(from[2], from[3]) : both(1.0f);
    }
}

struct AppendParams {
    const uint16_t *qkv;
    const float *q_norm, *k_norm, *inv_freq;
    const uint32_t *slots, *positions;
    uint16_t *q_out;
    RowsQ8Dev kv;
    uint32_t rows, heads, kv_heads;
    float eps;
    uint32_t window;    // rows whose runs one thread block looks after
    uint32_t q_ctas, stride;  // thread blocks for queries, one in every `stride`
    uint32_t per_warp, q_rows;  // query heads, and rows, that a warp takes
};

__device__ __forceinline__ float min_nan(float a, float b) {  // NaN if either is
    float v;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
    return v;
}
// What is kept of an infinity and of NaN.
__device__ __forceinline__ float tame(float x) { return x != x ? 0.0f : fminf(fmaxf(x, -kLargest), kLargest); }

// round(x / s) for |x / s| < 2^22 in the low bits: the last place of a sum with 1.5 * 2^23 is one.  1 / s comes in two parts,
// so that the quotient is rounded to f32 as a division's is.  With 1 / s alone its error decided where x / s is half-way
// between two codes, which is common for values (they are bf16, and s is a bf16 over 127): one code in 1500 was the other one.
constexpr float kCodeBits = 12582912.0f;
struct Factor {
    float high, low;
};
__device__ __forceinline__ uint32_t code_bits(float x, Factor f) {
    return __float_as_uint(__fadd_rn(fmaf(x, f.high, __fmul_rn(x, f.low)), kCodeBits));
}
__device__ __forceinline__ uint32_t pack_bits(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Code i of four: sign extension by a byte permutation (a conversion straight from a byte runs at a quarter of the rate).
__device__ __forceinline__ float code_at(uint32_t w, int i) {
    int v;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(v) : "r"(w), "r"(i | (i | 8) * 0x1110));  // bit 3 of a selector: the sign
    return __int2float_rn(v);
}

// A block's scale before and after, and how its codes follow.
struct Scales {
    Factor inv, ratio;
    float now;
    bool fresh;
};

__device__ __forceinline__ Scales grow(float was, bool fresh, float most) {
    const float old = fresh ? 0.0f : was;
    Scales s;
    s.now = fmaxf(old, fmaxf(most / 127.0f, kScaleFloor));
    s.inv.high = 1.0f / s.now;
    s.inv.low = fmaf(-s.inv.high, s.now, 1.0f) * s.inv.high;
    s.ratio = {1.0f, 0.0f};
    if (!fresh) {
        s.ratio.high = old / s.now;  // within [0, 1] for every scale that append writes
        s.ratio.low = fmaf(-s.ratio.high, s.now, old) * s.inv.high;
    }
    s.fresh = fresh;
    return s;
}

// |x| <= most, so that no code passes 127.
template <int W>
__device__ __forceinline__ void write_row(int8_t *row, uint32_t i, const float2 (&x)[4], Factor f) {
    auto codes = [&](float2 v) { return __fadd2_rn(fma2(v, both(f.high), mul2(v, both(f.low))), both(kCodeBits)); };
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float2 a = codes(x[2 * h]), b = codes(x[2 * h + 1]);
        *reinterpret_cast<uint32_t *>(row + h * (W / 2) + 4 * i) =
            pack_bits(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    }
}

// A held row's codes follow the scale (a code of -128, which append never writes, becomes -127 at most).
__device__ __forceinline__ uint32_t follow(uint32_t w, Factor ratio) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; e++) c[e] = code_bits(fmaxf(code_at(w, e), -127.0f), ratio);
    return pack_bits(c[0], c[1], c[2], c[3]);
}

template <int W>
__device__ __forceinline__ void follow_row(int8_t *row, uint32_t i, Factor ratio) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t *at = reinterpret_cast<uint32_t *>(row + h * (W / 2) + 4 * i);
        *at = follow(*at, ratio);
    }
}

// Bounds of four channels from the least and the largest new value (rounding keeps their order), joined with those the
// block had unless it is fresh.
template <int W>
__device__ __forceinline__ void write_bounds(int8_t *bounds, uint32_t first, uint32_t was_lo, uint32_t was_hi, const float *low,
                                             const float *high, const Scales &sc) {
    uint32_t *lo = reinterpret_cast<uint32_t *>(bounds + first), *hi = reinterpret_cast<uint32_t *>(bounds + W + first);
    was_lo = follow(was_lo, sc.ratio);
    was_hi = follow(was_hi, sc.ratio);
    uint32_t a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        int l = (int8_t)code_bits(low[e], sc.inv), h = (int8_t)code_bits(high[e], sc.inv);
        if (!sc.fresh) {
            l = min(l, (int)(int8_t)(was_lo >> (8 * e)));
            h = max(h, (int)(int8_t)(was_hi >> (8 * e)));
        }
        a[e] = (uint32_t)l;
        b[e] = (uint32_t)h;
    }
    *lo = pack_bits(a[0], a[1], a[2], a[3]);
    *hi = pack_bits(b[0], b[1], b[2], b[3]);
}

constexpr uint32_t kShort = 4;  // rows of a run that one warp takes
constexpr int kAppendWarps = 4, kAppendThreads = kAppendWarps * 32;
// Rows of a call up to which a block's rows may stand anywhere in it (drafted tokens laid out draft by draft): thread
// blocks then look after kAppendWarps rows and compare every row of the call with them, which at 1024 rows is 33 MB from
// L2 in all, and grows with the rows' square: 64 single rows take 12.9 us for 12.6 without, 512 take 43.3 for 40.7, a
// prompt's 1000 rows 21.6 for 18.9.  A kernel of its own (GATHERS): 8165 rows took 42.7 us for 40.7 when one kernel did both.
constexpr uint32_t kGathered = 1024;

// Measured over stores that are each written once: 64 single rows with 16 + 8 + 8 heads of 128 in blocks of 16 take 12.9 us
// (about half of the scales grow), 6.4 where no scale grows, 13.3 where all do: one load after another (slot, page, scale,
// row, then the block whose codes follow).  8165 rows of three prompts take 40.6 us for 119 MB, 0.45 of the copy rate, whether
// scales grow or not: the angles, norms and roundings of 260,000 heads keep the schedulers busier than the memory.  Two
// values an instruction brought it there from 43, five thread blocks an SM (96 registers, 24 to 64 bytes spilled at width
// 128) from 41 with six (80 registers).
template <int W, int B, bool GATHERS>
__global__ void __launch_bounds__(kAppendThreads, W == 256 ? 4 : 5) append_q8_kernel(const AppendParams p) {
    constexpr int L = Lanes<W>::PER_HEAD, T = Lanes<W>::TOGETHER;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, li = lane % L, which = lane / L;
    const uint32_t per_row = p.heads + 2 * p.kv_heads;
    __shared__ uint64_t sm_turns[W / 2];  // each pair's, computed once: its 64-bit arithmetic is slow
    pdl_wait();
    // Query blocks are spread among the others (which wait for one load after another, while they are bound by their
    // traffic): every p.stride-th block as long as there are any.
    const uint32_t turn_q = blockIdx.x / p.stride;
    const bool queries = blockIdx.x % p.stride == p.stride - 1 && turn_q < p.q_ctas;
    const uint32_t kv_block = blockIdx.x - min(turn_q, p.q_ctas);
    const float freq = threadIdx.x < W / 2 ? p.inv_freq[threadIdx.x] : 0.0f;
    // ---- keys, values: the runs that begin among this block's rows, at most 32 of them, one a lane ----
    const uint32_t units = 2 * p.kv_heads, unit = kv_block % units;
    const uint32_t r0 = kv_block / units * p.window, r1 = min(p.rows, r0 + p.window);
    uint32_t slot = 0, blk_pos = 0xFFFFFFFFu, starts = 0;
    __shared__ uint32_t sm_rows[kAppendWarps], sm_last[kAppendWarps], sm_earlier;  // by run: see below
    bool odd = false;  // another run of the block of one of this thread block's runs begins somewhere in the call
    if (!queries) {
        uint32_t some = 0;
        if (GATHERS && threadIdx.x < p.rows) some = p.slots[threadIdx.x];
        if (r0 + lane < r1) {
            slot = p.slots[r0 + lane];
            blk_pos = p.positions[r0 + lane] >> p.kv.shift;
        }
        uint32_t slot_was = __shfl_up_sync(0xFFFFFFFFu, slot, 1), pos_was = __shfl_up_sync(0xFFFFFFFFu, blk_pos, 1);
        if (lane == 0 && r0 > 0) {
            slot_was = p.slots[r0 - 1];
            pos_was = p.positions[r0 - 1] >> p.kv.shift;
        }
        const bool begins = r0 + lane < r1 && ((r0 == 0 && lane == 0) || slot != slot_was || blk_pos != pos_was);
        starts = __ballot_sync(0xFFFFFFFFu, begins);
        if (starts == 0) {
            pdl_launch_dependents();
            return;
        }
        if constexpr (GATHERS) {
            uint32_t s[kAppendWarps], b[kAppendWarps];
#pragma unroll
            for (int w = 0; w < kAppendWarps; w++) {
                s[w] = __shfl_sync(0xFFFFFFFFu, slot, w);
                b[w] = __shfl_sync(0xFFFFFFFFu, starts >> lane & 1 ? blk_pos : 0xFFFFFFFFu, w);  // no row's block
            }
#pragma unroll
            for (int w = 0; w + 1 < kAppendWarps; w++) odd |= begins & lane > w & slot == s[w] & blk_pos == b[w];
            for (uint32_t i = threadIdx.x; i < p.rows; i += kAppendThreads) {
                if (i >= (uint32_t)kAppendThreads) some = p.slots[i];
                if ((some == s[0] | some == s[1] | some == s[2] | some == s[3]) & i - r0 >= (uint32_t)kAppendWarps) {
                    const uint32_t block = p.positions[i] >> p.kv.shift, before = max(i, 1u) - 1;
                    const bool goes_on = i > 0 & p.slots[before] == some & p.positions[before] >> p.kv.shift == block;
#pragma unroll
                    for (int w = 0; w < kAppendWarps; w++) odd |= !goes_on & some == s[w] & block == b[w];
                }
            }
            if (threadIdx.x < kAppendWarps) sm_rows[threadIdx.x] = sm_last[threadIdx.x] = 0;
            if (threadIdx.x == 0) sm_earlier = 0;
        }
    }
    if (threadIdx.x < W / 2) sm_turns[threadIdx.x] = turns_of(freq);
    __syncthreads();
    uint64_t turns[4];
#pragma unroll
    for (int e = 0; e < 4; e++) turns[e] = sm_turns[4 * li + e];
    if (queries) {
        // ---- queries: a warp takes up to `per_warp` heads of `q_rows` rows, T of them side by side ----
        const uint32_t parts = (p.heads + p.per_warp - 1) / p.per_warp;
        const uint32_t job = turn_q * kAppendWarps + warp;
        const uint32_t h0 = job % parts * p.per_warp, h1 = min(p.heads, h0 + p.per_warp);
        const uint32_t first = job / parts * p.q_rows;
        const bool full = h1 - h0 == 8, normed = p.q_norm != nullptr;
        float2 g[4];
        load_gains<W>(p.q_norm, li, g);
        for (uint32_t r = first; r < min(first + p.q_rows, p.rows); r++) {
            constexpr int PASSES = 8 / T;
            const uint16_t *from = p.qkv + ((size_t)r * per_row + h0 + which) * W;
            uint16_t *to = p.q_out + ((size_t)r * p.heads + h0 + which) * W + 4 * li;
            Raw raw[PASSES];
            if (full) {
#pragma unroll
                for (int k = 0; k < PASSES; k++) raw[k] = load_head<W>(from + k * T * W, li);
            } else {
#pragma unroll
                for (int k = 0; k < PASSES; k++) {
                    raw[k] = {make_uint2(0, 0), make_uint2(0, 0)};
                    if (h0 + k * T + which < h1) raw[k] = load_head<W>(from + k * T * W, li);
                }
            }
            // the row's turn with the gains: first half a (g c) - b (g s), second half a (g s) + b (g c)
            const uint32_t pos = p.positions[r];
            float2 ac[2], as[2], bc[2], bs[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float2 sn, cs;
                sine_cosine(pos, turns[2 * e], turns[2 * e + 1], &sn, &cs);
                ac[e] = mul2(g[e], cs);
                as[e] = mul2(g[e], sn);
                bc[e] = mul2(g[2 + e], cs);
                bs[e] = mul2(g[2 + e], make_float2(-sn.x, -sn.y));
            }
            auto turned = [&](const Raw &raw, uint2 (&out)[2]) {
                float2 x[4];
                widen(raw, x);
                if (normed) {
                    const float2 inv = both(inverse_rms<W>(x, p.eps));
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = mul2(x[i], inv);
                }
                uint32_t w[2][2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float2 y = fma2(x[e], ac[e], mul2(x[2 + e], bs[e])), z = fma2(x[e], as[e], mul2(x[2 + e], bc[e]));
                    w[0][e] = pack_bf16(y.x, y.y);
                    w[1][e] = pack_bf16(z.x, z.y);
                }
                out[0] = make_uint2(w[0][0], w[0][1]);
                out[1] = make_uint2(w[1][0], w[1][1]);
            };
            if (full) {
#pragma unroll
                for (int k = 0; k < PASSES; k++) {
                    uint2 out[2];
                    turned(raw[k], out);
                    *reinterpret_cast<uint2 *>(to + k * T * W) = out[0];
                    *reinterpret_cast<uint2 *>(to + k * T * W + W / 2) = out[1];
                }
            } else {
#pragma unroll
                for (int k = 0; k < PASSES; k++) {
                    if (h0 + k * T >= h1) break;
                    uint2 out[2];
                    turned(raw[k], out);
                    if (h0 + k * T + which < h1) {
                        *reinterpret_cast<uint2 *>(to + k * T * W) = out[0];
                        *reinterpret_cast<uint2 *>(to + k * T * W + W / 2) = out[1];
                    }
                }
            }
        }
        pdl_launch_dependents();
        return;
    }

    // Long runs belong to a team of warps: all four for 64 positions, else two.
    constexpr int TEAM = B == 64 ? 4 : 2, TEAMS = kAppendWarps / TEAM, STEP = TEAM * T, PASSES = B > STEP ? B / STEP : 1;
    const uint32_t team = warp / TEAM, tid = threadIdx.x - team * TEAM * 32;  // the thread's number in its team
    const uint32_t mine = tid / L;                                            // it has positions mine + STEP u
    auto team_sync = [&] {
        if (TEAMS == 1) __syncthreads();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TEAM * 32) : "memory");
    };
    __shared__ int all_src[TEAMS][B];  // the row that writes each position of the block, or -1
    __shared__ uint32_t all_stop[TEAMS];
    __shared__ uint32_t sm_max[kAppendWarps];
    __shared__ float4 sm_step[W / 4];  // sines and cosines of STEP positions, of two pairs
    int *src = all_src[team];
    uint32_t &stop = all_stop[team];
    // Long runs: a thread's prepared values wait here for the scale (in registers they would leave room for 12 warps an SM,
    // 54 us for 8165 rows), then the block's bounds are put together in the same place.
    extern __shared__ __align__(16) float4 all_kept[];  // [teams][passes][2][threads]
    float4 *kept = all_kept + team * (PASSES * 2 * TEAM * 32);
    const bool is_v = unit >= p.kv_heads;
    const uint32_t h = is_v ? unit - p.kv_heads : unit;
    const uint16_t *heads = p.qkv + (size_t)(p.heads + unit) * W;  // this unit's head of row 0
    const bool bounded = !is_v && p.kv.bounds != nullptr, normed = !is_v && p.k_norm != nullptr;
    float2 g[4];
    load_gains<W>(normed ? p.k_norm : nullptr, li, g);
    if (!is_v && threadIdx.x < W / 4) {
        float2 sn, cs;
        sine_cosine(STEP, sm_turns[2 * threadIdx.x], sm_turns[2 * threadIdx.x + 1], &sn, &cs);
        sm_step[threadIdx.x] = make_float4(sn.x, sn.y, cs.x, cs.y);
    }
    bool gather = false;
    if constexpr (GATHERS) {
        gather = __syncthreads_or(odd);
        if (gather) {
            // Of each run's block: whether rows before the run fall into it (then it is not this run's), how many do from the
            // run's start on, and the last of them.
#pragma unroll 1
            for (uint32_t i = threadIdx.x; i < p.rows; i += kAppendThreads)
#pragma unroll 1
                for (uint32_t m = starts; m; m &= m - 1) {
                    const uint32_t w = __ffs(m) - 1, at = r0 + w;
                    if (p.slots[i] != p.slots[at] || (p.positions[i] ^ p.positions[at]) >> p.kv.shift) continue;
                    if (i < at) {
                        atomicOr(&sm_earlier, 1u << w);
                    } else {
                        atomicAdd(&sm_rows[w], 1u);
                        atomicMax(&sm_last[w], i);
                    }
                }
            __syncthreads();
        }
    } else {
        __syncthreads();
    }
    for (uint32_t turn = 0; starts; turn++) {
        const uint32_t first = __ffs(starts) - 1;
        starts &= starts - 1;
        if (gather && (sm_earlier >> first & 1)) continue;  // belongs to the block's first row
        const uint32_t s = r0 + first, run_slot = __shfl_sync(0xFFFFFFFFu, slot, first), b = __shfl_sync(0xFFFFFFFFu, blk_pos, first);
        const uint32_t blk = block_of(p.kv, run_slot, b);
        auto same = [&](uint32_t i) { return i < p.rows && p.slots[i] == run_slot && (p.positions[i] >> p.kv.shift) == b; };
        // rows of the run, as far as kShort + 1: the next run's start tells, or the rows past this block's do
        uint32_t n = starts ? __ffs(starts) - 1 - first : r1 - s;
        if (!starts && n <= kShort) {
            const uint32_t out = ~__ballot_sync(0xFFFFFFFFu, lane < n || (lane <= kShort && same(s + lane)));
            n = __ffs(out) - 1;
        }
        const bool apart = gather && sm_last[first] - s + 1 != sm_rows[first];  // other rows stand between the block's
        const size_t at = (size_t)(blk == kNoBlock ? 0 : blk) * p.kv_heads + h;
        float *scale = (is_v ? p.kv.v_scale : p.kv.k_scale) + at;
        int8_t *codes = (is_v ? p.kv.v : p.kv.k) + at * B * W;
        int8_t *bounds = p.kv.bounds + at * 2 * W;
        const float was = *scale;  // asked for before it is needed
        if (n <= kShort && !apart) {
            // ---- a warp's run ----
            if (turn % kAppendWarps != warp || blk == kNoBlock) continue;
            constexpr int PASSES = kShort / T > 0 ? kShort / T : 1;
            uint32_t held[4] = {};  // the bounds of this lane's channels
            if (bounded && which == 0) {
#pragma unroll
                for (int i = 0; i < 4; i++) held[i] = *reinterpret_cast<const uint32_t *>(bounds + (i & 1) * W + (i >> 1) * (W / 2) + 4 * li);
            }
            uint64_t written = 0;
            for (uint32_t k = 0; k < n; k++) written |= 1ull << (p.positions[s + k] & (B - 1));
            float2 x[PASSES][4];
            float low[8], high[8];
            int8_t *row[PASSES];
#pragma unroll
            for (int e = 0; e < 8; e++) low[e] = INFINITY, high[e] = -INFINITY;
#pragma unroll
            for (int k = 0; k < PASSES; k++) {
                const uint32_t j = k * T + which;
                uint32_t pos = 0;
                bool live = j < n;
                Raw raw = {make_uint2(0, 0), make_uint2(0, 0)};
                if (live) {
                    raw = load_head<W>(heads + (size_t)(s + j) * per_row * W, li);
                    pos = p.positions[s + j];
                    for (uint32_t later = j + 1; later < n; later++) live = live && p.positions[s + later] != pos;
                }
                widen(raw, x[k]);
                if (!is_v && k * T < n) {
                    float2 sn[2], cs[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) sine_cosine(pos, turns[2 * e], turns[2 * e + 1], &sn[e], &cs[e]);
                    norm_turn<W>(x[k], normed, g, sn, cs, p.eps);
                }
                row[k] = live ? codes + (pos & (B - 1)) * W : nullptr;
                if (live) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[k][e] = make_float2(tame(x[k][e].x), tame(x[k][e].y));
                        low[2 * e] = fminf(low[2 * e], x[k][e].x);
                        low[2 * e + 1] = fminf(low[2 * e + 1], x[k][e].y);
                        high[2 * e] = fmaxf(high[2 * e], x[k][e].x);
                        high[2 * e + 1] = fmaxf(high[2 * e + 1], x[k][e].y);
                    }
                }
            }
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (high[e] >= low[e]) most = fmaxf(most, fmaxf(fabsf(low[e]), fabsf(high[e])));
            most = warp_max(most);
            const Scales sc = grow(was, written & 1, most);
#pragma unroll
            for (int k = 0; k < PASSES; k++)
                if (row[k]) write_row<W>(row[k], li, x[k], sc.inv);
            if (sc.ratio.high < 1.0f)
                for (uint32_t i = which; i < (uint32_t)B; i += T)
                    if (!(written >> i & 1)) follow_row<W>(codes + i * W, li, sc.ratio);
            if (bounded) {
#pragma unroll
                for (int o = L; o < 32; o <<= 1)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        low[e] = fminf(low[e], __shfl_xor_sync(0xFFFFFFFFu, low[e], o));
                        high[e] = fmaxf(high[e], __shfl_xor_sync(0xFFFFFFFFu, high[e], o));
                    }
                if (which == 0) {
                    write_bounds<W>(bounds, 4 * li, held[0], held[1], low, high, sc);
                    write_bounds<W>(bounds, W / 2 + 4 * li, held[2], held[3], low + 4, high + 4, sc);
                }
            }
            __syncwarp();  // every lane has read the old scale
            if (lane == 0) *scale = sc.now;
            continue;
        }
        // ---- a team's run: which row writes which position ----
        if (turn % TEAMS != team) continue;
        team_sync();
        if (tid < B) src[tid] = -1;
        if (tid == 0) stop = p.rows;
        team_sync();
        for (uint32_t base = s; base < p.rows; base += TEAM * 32) {
            const uint32_t i = base + tid;
            const bool in = same(i);
            if (!in && i < p.rows && !apart) atomicMin(&stop, i);
            team_sync();
            const uint32_t end = stop;  // later passes only bring it down to rows past this one's
            if (in && i < end) atomicMax(&src[p.positions[i] & (B - 1)], (int)i);
            if (end < base + TEAM * 32) break;
        }
        team_sync();
        if (blk == kNoBlock) continue;
        auto row_of = [&](int u) { return mine + STEP * u < B ? src[mine + STEP * u] : -1; };
        if (is_v) {
            // ---- values: bf16 as they come, kept as such; magnitudes compare as whole numbers ----
            Raw raw[PASSES];
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < PASSES; u++) {
                const int row = row_of(u);
                raw[u] = {make_uint2(0, 0), make_uint2(0, 0)};
                if (row >= 0) raw[u] = load_head<W>(heads + (size_t)row * per_row * W, li);
            }
#pragma unroll
            for (int u = 0; u < PASSES; u++) {
                top = __vmaxu2(top, __vmaxu2(raw[u].a.x & 0x7FFF7FFFu, raw[u].a.y & 0x7FFF7FFFu));
                top = __vmaxu2(top, __vmaxu2(raw[u].b.x & 0x7FFF7FFFu, raw[u].b.y & 0x7FFF7FFFu));
            }
            top = __reduce_max_sync(0xFFFFFFFFu, max(top & 0xFFFFu, top >> 16));
            if (lane == 0) sm_max[warp] = top;
            team_sync();
            top = sm_max[team * TEAM];
#pragma unroll
            for (int w = 1; w < TEAM; w++) top = max(top, sm_max[team * TEAM + w]);
            const bool wild = top > 0x7F7Fu;  // an infinity or NaN among them: the largest of the others counts, see `tame`
            float most = __uint_as_float(top << 16);
            if (wild) {
                most = 0.0f;
#pragma unroll
                for (int u = 0; u < PASSES; u++) {
                    float2 x[4];
                    widen(raw[u], x);
#pragma unroll
                    for (int e = 0; e < 4; e++) most = fmaxf(most, fmaxf(fabsf(tame(x[e].x)), fabsf(tame(x[e].y))));
                }
                top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most));
                team_sync();
                if (lane == 0) sm_max[warp] = top;
                team_sync();
#pragma unroll
                for (int w = 0; w < TEAM; w++) most = fmaxf(most, __uint_as_float(sm_max[team * TEAM + w]));
            }
            const Scales sc = grow(was, src[0] >= 0, most);
#pragma unroll
            for (int u = 0; u < PASSES; u++) {
                const uint32_t i = mine + STEP * u;
                if (row_of(u) >= 0) {
                    float2 x[4];
                    widen(raw[u], x);
                    if (wild) {
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = make_float2(tame(x[e].x), tame(x[e].y));
                    }
                    write_row<W>(codes + i * W, li, x, sc.inv);
                } else if (i < B && sc.ratio.high < 1.0f) {
                    follow_row<W>(codes + i * W, li, sc.ratio);
                }
            }
            team_sync();  // every thread has read the old scale
            if (tid == 0) *scale = sc.now;
            continue;
        }
        // ---- keys ----
        uint32_t held_lo = 0, held_hi = 0;  // the bounds of channels 4 tid ..
        if (bounded && tid < W / 4) {
            held_lo = *reinterpret_cast<const uint32_t *>(bounds + 4 * tid);
            held_hi = *reinterpret_cast<const uint32_t *>(bounds + W + 4 * tid);
        }
        // Least and largest of each of the lane's channels; NaN stays, so that one comparison finds what is to be tamed.
        float low[8], high[8];
#pragma unroll
        for (int e = 0; e < 8; e++) low[e] = INFINITY, high[e] = -INFINITY;
        float2 sn[2], cs[2];
#pragma unroll
        for (int e = 0; e < 2; e++) sine_cosine((b << p.kv.shift) + mine, turns[2 * e], turns[2 * e + 1], &sn[e], &cs[e]);
        bool any = false;
        constexpr int GROUP = PASSES < 4 ? PASSES : 4;  // passes whose loads are under way together
        for (int u0 = 0; u0 < PASSES; u0 += GROUP) {
            Raw raw[GROUP];
#pragma unroll
            for (int k = 0; k < GROUP; k++) {
                const int row = row_of(u0 + k);
                raw[k] = {make_uint2(0, 0), make_uint2(0, 0)};
                if (row >= 0) raw[k] = load_head<W>(heads + (size_t)row * per_row * W, li);
            }
#pragma unroll
            for (int k = 0; k < GROUP; k++) {
                float2 x[4];
                widen(raw[k], x);
                norm_turn<W>(x, normed, g, sn, cs, p.eps);
                // the next pass is STEP positions on: a turn by a fixed angle (at most 15 of them, 2^-24 each)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float4 by = sm_step[2 * li + e];
                    const float2 s1 = make_float2(by.x, by.y), c1 = make_float2(by.z, by.w), s0 = sn[e], c0 = cs[e];
                    cs[e] = fma2(c0, c1, mul2(s0, make_float2(-by.x, -by.y)));
                    sn[e] = fma2(s0, c1, mul2(c0, s1));
                }
                if (row_of(u0 + k) >= 0) {
                    any = true;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        low[2 * e] = min_nan(low[2 * e], x[e].x);
                        low[2 * e + 1] = min_nan(low[2 * e + 1], x[e].y);
                        high[2 * e] = max_nan(high[2 * e], x[e].x);
                        high[2 * e + 1] = max_nan(high[2 * e + 1], x[e].y);
                    }
                }
                kept[(2 * (u0 + k)) * (TEAM * 32) + tid] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
                kept[(2 * (u0 + k) + 1) * (TEAM * 32) + tid] = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
            }
        }
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) most = max_nan(most, max_nan(fabsf(low[e]), fabsf(high[e])));
        if (any && !(most <= kLargest)) {  // an infinity or NaN among them
            most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) low[e] = INFINITY, high[e] = -INFINITY;
            for (int u = 0; u < PASSES; u++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    float4 &v = kept[(2 * u + half) * (TEAM * 32) + tid];
                    float x[4] = {tame(v.x), tame(v.y), tame(v.z), tame(v.w)};
                    v = make_float4(x[0], x[1], x[2], x[3]);
                    if (row_of(u) < 0) continue;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        low[4 * half + e] = fminf(low[4 * half + e], x[e]);
                        high[4 * half + e] = fmaxf(high[4 * half + e], x[e]);
                        most = fmaxf(most, fabsf(x[e]));
                    }
                }
        }
        most = warp_max(any ? most : 0.0f);
        if (lane == 0) sm_max[warp] = __float_as_uint(most);
        team_sync();
#pragma unroll
        for (int w = 0; w < TEAM; w++) most = fmaxf(most, __uint_as_float(sm_max[team * TEAM + w]));
        const Scales sc = grow(was, src[0] >= 0, most);
#pragma unroll 2
        for (int u = 0; u < PASSES; u++) {
            const uint32_t i = mine + STEP * u;
            if (row_of(u) >= 0) {
                const float4 v = kept[(2 * u) * (TEAM * 32) + tid], w = kept[(2 * u + 1) * (TEAM * 32) + tid];
                const float2 x[4] = {make_float2(v.x, v.y), make_float2(v.z, v.w), make_float2(w.x, w.y), make_float2(w.z, w.w)};
                write_row<W>(codes + i * W, li, x, sc.inv);
            } else if (i < B && sc.ratio.high < 1.0f) {
                follow_row<W>(codes + i * W, li, sc.ratio);
            }
        }
        team_sync();  // every thread has read the old scale and its kept values
        if (tid == 0) *scale = sc.now;
        if (bounded) {
            // lanes that hold the same channels meet in shared memory: [STEP][low, high][W]
            float *sm = reinterpret_cast<float *>(kept) + mine * 2 * W;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t d = half * (W / 2) + 4 * li;
                *reinterpret_cast<float4 *>(sm + d) = make_float4(low[4 * half], low[4 * half + 1], low[4 * half + 2], low[4 * half + 3]);
                *reinterpret_cast<float4 *>(sm + W + d) = make_float4(high[4 * half], high[4 * half + 1], high[4 * half + 2], high[4 * half + 3]);
            }
            team_sync();
            if (tid < W / 4) {
                const float *all = reinterpret_cast<const float *>(kept) + 4 * tid;
                float lo[4], hi[4];
#pragma unroll
                for (int e = 0; e < 4; e++) lo[e] = INFINITY, hi[e] = -INFINITY;
#pragma unroll 4
                for (int k = 0; k < STEP; k++) {
                    const float4 l = *reinterpret_cast<const float4 *>(all + k * 2 * W), m = *reinterpret_cast<const float4 *>(all + k * 2 * W + W);
                    lo[0] = fminf(lo[0], l.x); lo[1] = fminf(lo[1], l.y); lo[2] = fminf(lo[2], l.z); lo[3] = fminf(lo[3], l.w);
                    hi[0] = fmaxf(hi[0], m.x); hi[1] = fmaxf(hi[1], m.y); hi[2] = fmaxf(hi[2], m.z); hi[3] = fmaxf(hi[3], m.w);
                }
                write_bounds<W>(bounds, 4 * tid, held_lo, held_hi, lo, hi, sc);
            }
        }
    }
    pdl_launch_dependents();
}

// Reading rows back is a copy that widens: the codes once, twice as many bytes out.  A thread has its 8 channels of a kv
// head's keys or values (a warp's stores then fill whole lines) and goes over ROWS rows: `pieces` threads hold a row (all of
// K, then V), `together` rows lie side by side.  The block first looks all its rows up, then every thread asks for the codes
// of all its rows before it writes the first.  2 x 16001 rows of 8 heads of 128: 30.4 us, 5.5 TB/s, 0.84 of the copy rate;
// 160 rows: 2.4 us, a launch and two loads that wait for each other.
template <int W, int ROWS>
__global__ void __launch_bounds__(512) unpack_q8_kernel(const RowsQ8Dev kv, const uint32_t *slots, const uint32_t *positions,
                                                        uint4 *k_out, uint4 *v_out, uint32_t rows, uint32_t kv_heads, uint32_t pieces,
                                                        uint32_t together) {
    constexpr uint32_t PIECES = W / 8;
    __shared__ uint2 place[256];  // block and position in it
    pdl_wait();
    const uint32_t first = blockIdx.x * together * ROWS;
    for (uint32_t i = threadIdx.x; i < together * ROWS; i += blockDim.x) {
        uint2 at = make_uint2(kNoBlock, 0);
        if (first + i < rows) {
            const uint32_t pos = positions[first + i];
            at = make_uint2(block_of(kv, slots[first + i], pos >> kv.shift), pos & ((1u << kv.shift) - 1u));
        }
        place[i] = at;
    }
    __syncthreads();
    const uint32_t sub = threadIdx.x / pieces, rest = blockIdx.y * pieces + threadIdx.x - sub * pieces;
    if (rest < 2 * kv_heads * PIECES) {
        const bool is_v = rest >= kv_heads * PIECES;
        const uint32_t at = is_v ? rest - kv_heads * PIECES : rest, h = at / PIECES, piece = at % PIECES;
        const int8_t *codes = (is_v ? kv.v : kv.k) + piece * 8;
        const float *scales = is_v ? kv.v_scale : kv.k_scale;
        uint4 *to = (is_v ? v_out : k_out) + ((size_t)(first + sub) * kv_heads * PIECES + at);
        const size_t stride = (size_t)together * kv_heads * PIECES;
        uint2 c[ROWS];
        float s[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
            const uint2 where = place[sub + u * together];
            c[u] = make_uint2(0, 0);
            s[u] = 0.0f;
            if (where.x != kNoBlock) {
                const size_t head = (size_t)where.x * kv_heads + h;
                s[u] = scales[head];
                c[u] = *reinterpret_cast<const uint2 *>(codes + ((head << kv.shift) + where.y) * W);
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS; u++) {
            if (first + sub + u * together >= rows) break;
            const uint32_t w[2] = {c[u].x, c[u].y};
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                out[2 * j] = pack_bf16(code_at(w[j], 0) * s[u], code_at(w[j], 1) * s[u]);
                out[2 * j + 1] = pack_bf16(code_at(w[j], 2) * s[u], code_at(w[j], 3) * s[u]);
            }
            to[u * stride] = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
    pdl_launch_dependents();
}

// Shared memory of the teams: a block of positions' values in f32 each, or what the bounds need, which is less.
template <int W, int B>
constexpr size_t append_smem() {
    constexpr int team = B == 64 ? 4 : 2, step = team * Lanes<W>::TOGETHER, passes = B > step ? B / step : 1;
    static_assert(passes * team * 32 * 8 >= step * 2 * W, "the bounds fit where the values were");
    return (size_t)(kAppendWarps / team) * passes * 2 * team * 32 * sizeof(float4);
}

template <int W, int B, bool GATHERS>
cudaError_t launch_append(const AppendParams &p, uint32_t grid, cudaStream_t stream) {
    constexpr size_t smem = append_smem<W, B>();
    static OncePerDevice configured;
    if (smem > 48 * 1024 && configured.needs()) {
        const cudaError_t e = cudaFuncSetAttribute(append_q8_kernel<W, B, GATHERS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        configured.done();
    }
    return launch(append_q8_kernel<W, B, GATHERS>, dim3(grid), dim3(kAppendThreads), smem, stream, pdl_enabled(), p);
}

template <int W>
cudaError_t launch_append(const AppendParams &p, uint32_t grid, cudaStream_t stream) {
    auto go = [&](auto gathers) {
        constexpr bool GATHERS = decltype(gathers)::value;
        return p.kv.shift == 4   ? launch_append<W, 16, GATHERS>(p, grid, stream)
               : p.kv.shift == 5 ? launch_append<W, 32, GATHERS>(p, grid, stream)
                                 : launch_append<W, 64, GATHERS>(p, grid, stream);
    };
    return p.rows <= kGathered ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

int append_q8(const void *qkv, const float *q_norm, const float *k_norm, const float *inv_freq, const uint32_t *slots,
              const uint32_t *positions, void *q_out, const RowsQ8Dev &kv, uint32_t rows, uint32_t heads, uint32_t kv_heads,
              uint32_t width, float eps, cudaStream_t stream) {
    AppendParams p = {};
    p.qkv = (const uint16_t *)qkv;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.inv_freq = inv_freq;
    p.slots = slots;
    p.positions = positions;
    p.q_out = (uint16_t *)q_out;
    p.kv = kv;
    p.rows = rows;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.eps = eps;
    // A step's rows each have a run of their own: four of them keep the warps of a thread block busy.  A prompt's
    // rows come in runs of up to a block: looking at 32 rows leaves few thread blocks without a run to start.
    p.window = rows <= kGathered ? kAppendWarps : 32;
    // Eight heads a warp compute a row's angles once and have their loads under way together, four rows share what a warp
    // sets up; a step's few heads go to as many warps as there are.
    const bool many = (uint64_t)rows * heads > 32768;
    p.per_warp = many ? 8 : 32 / (width / 8);
    p.q_rows = many ? 4 : 1;
    const uint64_t kv_ctas = (uint64_t)ceil_div(rows, p.window) * 2 * kv_heads;
    const uint64_t q_ctas = ((uint64_t)ceil_div(rows, p.q_rows) * ceil_div(heads, p.per_warp) + kAppendWarps - 1) / kAppendWarps;
    TS_REQUIRE(qkv != q_out, "append (q8): q_out is where qkv lies");
    TS_REQUIRE(kv_ctas + q_ctas < 0x1FFFFFFFull, "append (q8): %u rows of %u heads are too many for one launch", rows, heads);
    const uint32_t grid = (uint32_t)(kv_ctas + q_ctas);
    p.q_ctas = (uint32_t)q_ctas;
    p.stride = grid / p.q_ctas;
    const cudaError_t e = width == 64    ? launch_append<64>(p, grid, stream)
                          : width == 128 ? launch_append<128>(p, grid, stream)
                                         : launch_append<256>(p, grid, stream);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of append (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

int unpack_q8(const RowsQ8Dev &kv, const uint32_t *slots, const uint32_t *positions, void *k_out, void *v_out, uint32_t rows,
              uint32_t kv_heads, uint32_t width, cudaStream_t stream) {
    const uint32_t all = 2 * kv_heads * (width / 8);
    const uint32_t pieces = min(all, 512u), together = pieces < 256 ? 256 / pieces : 1;
    // Eight rows a thread once that still leaves a block for every place on the GPU.
    const bool many = (uint64_t)rows * all >= (uint64_t)sm_count() * 2048 * 8;
    const uint32_t each = together * (many ? 8 : 2);
    const dim3 grid((uint32_t)(((uint64_t)rows + each - 1) / each), ceil_div(all, pieces)), block(pieces * together);
    TS_REQUIRE(grid.y <= 65535, "rows_unpack (q8): %u kv heads are too many", kv_heads);
    auto go = [&](auto kernel) {
        return launch(kernel, grid, block, 0, stream, pdl_enabled(), kv, slots, positions, (uint4 *)k_out, (uint4 *)v_out, rows, kv_heads,
                      pieces, together);
    };
    const cudaError_t e = width == 64    ? (many ? go(unpack_q8_kernel<64, 8>) : go(unpack_q8_kernel<64, 2>))
                          : width == 128 ? (many ? go(unpack_q8_kernel<128, 8>) : go(unpack_q8_kernel<128, 2>))
                                         : (many ? go(unpack_q8_kernel<256, 8>) : go(unpack_q8_kernel<256, 2>));
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of unpack (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

}  // namespace ts
