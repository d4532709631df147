// Ragged attention over kept rows in 8 bits, whole slots or listed blocks.
//
// A tile of 16 query rows is (token, head) pairs: the G heads of a kv head's group times the T = 16 / G neighbouring
// rows that share a slot (drafted tokens, a part of a prompt); the other rows of the tile repeat nothing and are never
// stored.  Both products run on warp MMAs (m16n8k16, f16 in, f32 out): a code is exact in f16, a query row is brought
// into f16's range by a power of two, which is exact for bf16 (values below 2^-24 of the row's largest lose digits that
// no sum would keep).  Codes become f16 by setting them as the low bits of 1024 + 128 + code and subtracting 1152.
//
// The scales leave the products alone.  With s = raw * scale * k_scale in powers of two and
//     x = s + log2(v_scale),   M = max x,   P = 2^(x - M)  <= 1   (f16 operand of P V)
// the output is sum P code / sum P / v_scale: the block's value scale rides in the exponent, so that P needs no second
// factor and stays within f16's range whatever the scales are, and M cancels.  A scale of zero counts as 2^-60, the
// smallest that append writes.
#include <cmath>

#include "rows_q8.cuh"

namespace ts {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kScaleFloor = 8.673617379884035e-19f;  // 2^-60

struct AttendParams {
    const uint16_t *q;
    RowsQ8Dev kv;
    const uint32_t *ids;  // NULL: whole slots
    uint16_t *out;
    const uint32_t *slots, *positions;
    uint32_t rows, keys, heads, kv_heads, back, count;
    uint32_t group, part, parts;  // heads per kv head; heads of it in a tile, tiles it takes
    uint32_t tokens;              // rows a tile may hold
    uint32_t chunk, chunks;       // 16-key steps per item, items per tile
    float scale;
    float *part_o;   // [rows, heads, chunks, W]
    float *part_ml;  // [rows, heads, chunks, 2]
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
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes 0, 1 (sel 0x4140) or 2, 3 (sel 0x4342) of biased codes (code + 128) as two f16.
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t sel) {
    return sub_f16x2(__byte_perm(biased, 0x64646464u, sel), 0x64806480u);  // 1152 = 0x6480
}

// What a thread holds of the query tile: rows r0 = lane / 4 and r0 + 8.  The k index of an MMA step is permuted so that
// a thread's bytes of a key are contiguous: in 64-wide chunk c, step s, thread j = lane % 4 has dims 64 c + 16 j + 4 s + 0..3.
template <int W>
struct QueryTile {
    uint32_t a[W / 16][4];
    float f0, f1;  // raw score -> power-of-two exponent, without the key scale
};

// Row m of the tile: token m / part, head m % part.
template <int W>
__device__ __forceinline__ void load_query(const AttendParams &p, uint32_t row, uint32_t tokens, uint32_t head0, uint32_t part,
                                           uint32_t lane, QueryTile<W> &t) {
    const uint32_t j = lane & 3;
    float f[2];
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const uint32_t m = (lane >> 2) + 8 * half, token = m / part, head = m % part;
        uint2 v[W / 16];
        float most = 0.0f;
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            v[s] = make_uint2(0, 0);
            if (token < tokens)
                v[s] = *reinterpret_cast<const uint2 *>(p.q + ((size_t)(row + token) * p.heads + head0 + head) * W + (s / 4) * 64 + j * 16 + (s % 4) * 4);
            most = fmaxf(most, fmaxf(fmaxf(fabsf(bf16_lo(v[s].x)), fabsf(bf16_hi(v[s].x))), fmaxf(fabsf(bf16_lo(v[s].y)), fabsf(bf16_hi(v[s].y)))));
        }
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
        uint32_t e = __float_as_uint(most) >> 23;  // the largest magnitude's exponent; 255: infinity
        e = e < 1 ? 1 : e > 253 ? 253 : e;
        const float down = __uint_as_float((254 - e) << 23);
        f[half] = __uint_as_float(e << 23) * (p.scale * kLog2e);
#pragma unroll
        for (int s = 0; s < W / 16; s++) {
            t.a[s][half] = pack_f16(bf16_lo(v[s].x) * down, bf16_hi(v[s].x) * down);
            t.a[s][2 + half] = pack_f16(bf16_lo(v[s].y) * down, bf16_hi(v[s].y) * down);
        }
    }
    t.f0 = f[0];
    t.f1 = f[1];
}

template <int N>
__device__ __forceinline__ void load_codes(const int8_t *p, uint32_t (&w)[N]) {
    if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) w[i] ^= 0x80808080u;
}

// Running softmax and output of a tile: rows r0 and r0 + 8, dims [lane % 4 * W / 4, + W / 4) of each.
// o[i][0], [1]: row r0, dims 2 j * W / 8 + i and (2 j + 1) * W / 8 + i; [2], [3]: row r0 + 8.
template <int W>
struct Running {
    float o[W / 8][4];
    float m0, m1, l0, l1;
};

// Sixteen keys: k, v point at their codes (row pitch W), the first key's position is `key0`; row r0 sees [lo0, hi0).
template <int W>
__device__ __forceinline__ void step16(const QueryTile<W> &t, Running<W> &run, const int8_t *k, const int8_t *v, float k_scale,
                                       float v_scale, uint32_t key0, uint32_t lo0, uint32_t hi0, uint32_t lo1, uint32_t hi1,
                                       uint32_t lane) {
    const uint32_t r = lane >> 2, j = lane & 3;
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; n++) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < W / 64; c++) {
            uint32_t w[4];
            load_codes<4>(k + (8 * n + r) * W + c * 64 + j * 16, w);
#pragma unroll
            for (int i = 0; i < 4; i++)
                mma_f16(s[n], t.a[4 * c + i][0], t.a[4 * c + i][1], t.a[4 * c + i][2], t.a[4 * c + i][3], codes_f16(w[i], 0x4140),
                        codes_f16(w[i], 0x4342));
        }
    }
    const float vs = fmaxf(v_scale, kScaleFloor), lvs = log2_approx(vs), ivs = 1.0f / vs;
    const float f0 = t.f0 * k_scale, f1 = t.f1 * k_scale;
    float x[2][4], most0 = -INFINITY, most1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t key = key0 + 8 * n + 2 * j + e;
            x[n][e] = key >= lo0 && key < hi0 ? fmaf(s[n][e], f0, lvs) : -INFINITY;
            x[n][2 + e] = key >= lo1 && key < hi1 ? fmaf(s[n][2 + e], f1, lvs) : -INFINITY;
            most0 = fmaxf(most0, x[n][e]);
            most1 = fmaxf(most1, x[n][2 + e]);
        }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        most0 = fmaxf(most0, __shfl_xor_sync(0xFFFFFFFFu, most0, o));
        most1 = fmaxf(most1, __shfl_xor_sync(0xFFFFFFFFu, most1, o));
    }
    const float n0 = fmaxf(run.m0, most0), n1 = fmaxf(run.m1, most1);
    const float z0 = n0 == -INFINITY ? 0.0f : n0, z1 = n1 == -INFINITY ? 0.0f : n1;  // nothing seen yet: 2^(-inf - 0) = 0
    const float a0 = exp2_approx(run.m0 - z0), a1 = exp2_approx(run.m1 - z1);
    run.m0 = n0;
    run.m1 = n1;
    float p[2][4], sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            p[n][e] = exp2_approx(x[n][e] - z0);
            p[n][2 + e] = exp2_approx(x[n][2 + e] - z1);
            sum0 += p[n][e];
            sum1 += p[n][2 + e];
        }
    run.l0 = fmaf(sum0, ivs, run.l0 * a0);
    run.l1 = fmaf(sum1, ivs, run.l1 * a1);
    if (!__all_sync(0xFFFFFFFFu, a0 == 1.0f && a1 == 1.0f)) {
#pragma unroll
        for (int i = 0; i < W / 8; i++) {
            run.o[i][0] *= a0;
            run.o[i][1] *= a0;
            run.o[i][2] *= a1;
            run.o[i][3] *= a1;
        }
    }
    const uint32_t pa0 = pack_f16(p[0][0], p[0][1]), pa1 = pack_f16(p[0][2], p[0][3]), pa2 = pack_f16(p[1][0], p[1][1]),
                   pa3 = pack_f16(p[1][2], p[1][3]);
    uint32_t w[4][W / 32];  // keys 2 j, 2 j + 1, 2 j + 8, 2 j + 9, this thread's W / 8 dims
#pragma unroll
    for (int i = 0; i < 4; i++) load_codes<W / 32>(v + (2 * j + (i & 1) + 8 * (i >> 1)) * W + r * (W / 8), w[i]);
#pragma unroll
    for (int i = 0; i < W / 32; i++) {
        const uint32_t ab = __byte_perm(w[0][i], w[1][i], 0x5140), AB = __byte_perm(w[0][i], w[1][i], 0x7362);
        const uint32_t cd = __byte_perm(w[2][i], w[3][i], 0x5140), CD = __byte_perm(w[2][i], w[3][i], 0x7362);
        mma_f16(run.o[4 * i], pa0, pa1, pa2, pa3, codes_f16(ab, 0x4140), codes_f16(cd, 0x4140));
        mma_f16(run.o[4 * i + 1], pa0, pa1, pa2, pa3, codes_f16(ab, 0x4342), codes_f16(cd, 0x4342));
        mma_f16(run.o[4 * i + 2], pa0, pa1, pa2, pa3, codes_f16(AB, 0x4140), codes_f16(CD, 0x4140));
        mma_f16(run.o[4 * i + 3], pa0, pa1, pa2, pa3, codes_f16(AB, 0x4342), codes_f16(CD, 0x4342));
    }
}

// An item: (first row of a tile, kv head, heads' part, chunk).  `first_row` false: another item covers this row.
struct Item {
    uint32_t row, tokens, kvh, head0, part, chunk, slot;
};

__device__ __forceinline__ bool item_of(const AttendParams &p, uint32_t index, Item *it) {
    it->chunk = index % p.chunks;
    index /= p.chunks;
    const uint32_t hp = index % p.parts;
    index /= p.parts;
    it->kvh = index % p.kv_heads;
    it->row = index / p.kv_heads;
    it->head0 = it->kvh * p.group + hp * p.part;
    it->part = min(p.part, p.group - hp * p.part);
    it->slot = p.slots[it->row];
    it->tokens = 1;
    if (p.tokens == 1) return true;
    // Tiles begin at multiples of `tokens` and where a row is not the next position of the slot before it (or the same
    // again): what a tile sees then spans at most back + tokens keys, which the number of chunks counts on.
    auto follows = [&](uint32_t r) {
        return r % p.tokens != 0 && p.slots[r] == p.slots[r - 1] && p.positions[r] - p.positions[r - 1] <= 1u;
    };
    if (follows(it->row)) return false;
    while (it->row + it->tokens < p.rows && follows(it->row + it->tokens)) it->tokens++;
    return true;
}

__device__ __forceinline__ void seen(const AttendParams &p, uint32_t pos, uint32_t *lo, uint32_t *hi) {
    *lo = pos > p.back ? pos - p.back : 0;
    *hi = pos < p.keys ? pos + 1 : p.keys;
}

template <int W>
__global__ void __launch_bounds__(kThreads) attend_q8_kernel(const AttendParams p) {
    extern __shared__ float sm[];  // o [kWarps][16][W], then m, l [kWarps][16][2]
    float *sm_o = sm, *sm_ml = sm + kWarps * 16 * W;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    Item it;
    if (!item_of(p, blockIdx.x, &it)) {
        pdl_launch_dependents();
        return;
    }
    const uint32_t B = 1u << p.kv.shift;
    uint32_t lo0 = 1, hi0 = 0, lo1 = 1, hi1 = 0, lo = 0xFFFFFFFFu, hi = 0;
    for (uint32_t t = 0; t < it.tokens; t++) {
        uint32_t a, b;
        seen(p, p.positions[it.row + t], &a, &b);
        if (a < b) {
            lo = min(lo, a);
            hi = max(hi, b);
        }
        if ((lane >> 2) / it.part == t) lo0 = a, hi0 = b;
        if (((lane >> 2) + 8) / it.part == t) lo1 = a, hi1 = b;
    }
    QueryTile<W> tile;
    load_query<W>(p, it.row, it.tokens, it.head0, it.part, lane, tile);
    Running<W> run;
#pragma unroll
    for (int i = 0; i < W / 8; i++) run.o[i][0] = run.o[i][1] = run.o[i][2] = run.o[i][3] = 0.0f;
    run.m0 = run.m1 = -INFINITY;
    run.l0 = run.l1 = 0.0f;
    // 16-key steps [begin, end) of this item
    const uint32_t base = p.ids ? 0 : lo >> 4, steps = p.ids ? p.count << (p.kv.shift - 4) : lo < hi ? ((hi + 15) >> 4) - base : 0;
    const uint32_t begin = it.chunk * p.chunk, end = min(steps, begin + p.chunk);
    const uint32_t *list = p.ids ? p.ids + ((size_t)it.row * p.kv_heads + it.kvh) * p.count : nullptr;
    for (uint32_t s = begin + warp; s < end; s += kWarps) {
        uint32_t key0;
        if (p.ids) {
            const uint32_t b = list[s >> (p.kv.shift - 4)];
            if (((uint64_t)b << p.kv.shift) >= hi) continue;
            key0 = (b << p.kv.shift) + ((s << 4) & (B - 1));
            if (key0 >= hi) continue;
        } else {
            key0 = (base + s) << 4;
        }
        const uint32_t blk = block_of(p.kv, it.slot, key0 >> p.kv.shift);
        if (blk == kNoBlock) continue;
        const size_t at = (size_t)blk * p.kv_heads + it.kvh;
        const size_t off = ((at << p.kv.shift) + (key0 & (B - 1))) * W;
        step16<W>(tile, run, p.kv.k + off, p.kv.v + off, p.kv.k_scale[at], p.kv.v_scale[at], key0, lo0, hi0, lo1, hi1, lane);
    }
    // ---- fold the warps ----
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        run.l0 += __shfl_xor_sync(0xFFFFFFFFu, run.l0, o);
        run.l1 += __shfl_xor_sync(0xFFFFFFFFu, run.l1, o);
    }
    {
        const uint32_t r = lane >> 2, j = lane & 3;
        float *o0 = sm_o + (warp * 16 + r) * W + j * (W / 4), *o1 = o0 + 8 * W;
#pragma unroll
        for (int i = 0; i < W / 8; i++) {
            o0[i] = run.o[i][0];
            o0[W / 8 + i] = run.o[i][1];
            o1[i] = run.o[i][2];
            o1[W / 8 + i] = run.o[i][3];
        }
        if (j == 0) {
            float *ml = sm_ml + (warp * 16 + r) * 2;
            ml[0] = run.m0;
            ml[1] = run.l0;
            ml[16] = run.m1;
            ml[17] = run.l1;
        }
    }
    __syncthreads();
    const uint32_t live = it.tokens * it.part;
    for (uint32_t i = threadIdx.x; i < live * W; i += kThreads) {
        const uint32_t m = i / W, d = i % W;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) top = fmaxf(top, sm_ml[(w * 16 + m) * 2]);
        const float z = top == -INFINITY ? 0.0f : top;
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = exp2_approx(sm_ml[(w * 16 + m) * 2] - z);
            l = fmaf(sm_ml[(w * 16 + m) * 2 + 1], f, l);
            o = fmaf(sm_o[(w * 16 + m) * W + d], f, o);
        }
        const size_t head = (size_t)(it.row + m / it.part) * p.heads + it.head0 + m % it.part;
        if (p.chunks == 1) {
            p.out[head * W + d] = l == 0.0f ? (uint16_t)0 : bf16_bits(o / l);
        } else {
            const size_t at = head * p.chunks + it.chunk;
            p.part_o[at * W + d] = o;
            if (d == 0) {
                p.part_ml[at * 2] = top;
                p.part_ml[at * 2 + 1] = l;
            }
        }
    }
    pdl_launch_dependents();
}

// One block per (row, head): folds the chunks in ascending order.
template <int W>
__global__ void __launch_bounds__(W) attend_q8_merge_kernel(const AttendParams p) {
    pdl_wait();
    const size_t head = blockIdx.x, at = head * p.chunks;
    float top = -INFINITY;
    for (uint32_t c = 0; c < p.chunks; c++) top = fmaxf(top, p.part_ml[(at + c) * 2]);
    const float z = top == -INFINITY ? 0.0f : top;
    float l = 0.0f, o = 0.0f;
    for (uint32_t c = 0; c < p.chunks; c++) {
        const float f = exp2_approx(p.part_ml[(at + c) * 2] - z);
        l = fmaf(p.part_ml[(at + c) * 2 + 1], f, l);
        o = fmaf(p.part_o[(at + c) * W + threadIdx.x], f, o);
    }
    pdl_launch_dependents();
    p.out[head * W + threadIdx.x] = l == 0.0f ? (uint16_t)0 : bf16_bits(o / l);
}

struct Plan {
    uint32_t part, parts, tokens, chunk, chunks;
};

Plan plan_of(uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t back, uint32_t count, uint32_t block) {
    Plan s;
    const uint32_t group = heads / kv_heads;
    s.part = group < 16 ? group : 16;
    s.parts = ceil_div(group, s.part);
    s.tokens = count || s.parts > 1 ? 1 : 16 / s.part;
    uint64_t span = keys;  // keys a tile may see, in 16-key steps below
    if (!count && (uint64_t)back + s.tokens < span) span = (uint64_t)back + s.tokens;
    const uint64_t steps = count ? (uint64_t)count * (block / 16) : (span + 15) / 16 + 1;
    const uint64_t tiles = (uint64_t)rows * kv_heads * s.parts;
    const uint64_t want = ((uint64_t)sm_count() * 4 + tiles - 1) / tiles;
    uint64_t chunk = (steps + want - 1) / want;
    if (chunk < 16) chunk = 16;
    if (chunk > steps) chunk = steps;
    s.chunk = (uint32_t)(chunk ? chunk : 1);
    s.chunks = (uint32_t)((steps + s.chunk - 1) / s.chunk);
    if (s.chunks == 0) s.chunks = 1;
    return s;
}

template <int W>
int launch_attend(const AttendParams &p, uint32_t items, cudaStream_t stream) {
    const size_t smem = (size_t)kWarps * 16 * (W + 2) * sizeof(float);
    static OncePerDevice configured;
    if (configured.needs()) {
        TS_CUDA(cudaFuncSetAttribute(attend_q8_kernel<W>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        configured.done();
    }
    cudaError_t e = launch(attend_q8_kernel<W>, dim3(items), dim3(kThreads), smem, stream, pdl_enabled(), p);
    if (e == cudaSuccess && p.chunks > 1)
        e = launch(attend_q8_merge_kernel<W>, dim3(p.rows * p.heads), dim3(W), 0, stream, pdl_enabled(), p);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of attend (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

}  // namespace

size_t attend_q8_workspace_bytes(uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t back,
                                 uint32_t count, uint32_t block) {
    if (rows == 0 || keys == 0 || heads == 0 || kv_heads == 0 || heads % kv_heads) return 0;
    const Plan s = plan_of(rows, keys, heads, kv_heads, back, count, block);
    return s.chunks > 1 ? (size_t)rows * heads * s.chunks * (width + 2) * sizeof(float) : 0;
}

int attend_q8(const void *q, const RowsQ8Dev &kv, const uint32_t *ids, void *out, const uint32_t *slots,
              const uint32_t *positions, uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width,
              uint32_t back, uint32_t count, float scale, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const Plan s = plan_of(rows, keys, heads, kv_heads, back, count, 1u << kv.shift);
    const size_t need = s.chunks > 1 ? (size_t)rows * heads * s.chunks * (width + 2) * sizeof(float) : 0;
    TS_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && aligned16(workspace))),
               "attend (q8): workspace of %zu bytes is smaller than the %zu needed, or not 16-byte aligned", workspace_bytes, need);
    const uint64_t items = (uint64_t)rows * kv_heads * s.parts * s.chunks;
    TS_REQUIRE(items < 0x7FFFFFFFull && (uint64_t)rows * heads < 0x7FFFFFFFull, "attend (q8): %u rows are too many for one launch", rows);
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
    p.chunk = s.chunk;
    p.chunks = s.chunks;
    p.scale = scale;
    p.part_o = (float *)workspace;
    p.part_ml = p.part_o ? p.part_o + (size_t)rows * heads * s.chunks * width : nullptr;
    return width == 64    ? launch_attend<64>(p, (uint32_t)items, stream)
           : width == 128 ? launch_attend<128>(p, (uint32_t)items, stream)
                          : launch_attend<256>(p, (uint32_t)items, stream);
}

}  // namespace ts
