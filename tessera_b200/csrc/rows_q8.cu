// Kept rows in 8 bits: append (norm, rotation, block scales, key bounds) and reading rows back.
//
// Append.  A block of B positions has one scale per kv head, so the rows of a call that fall into one block are one
// unit of work: run = the neighbouring rows of a (slot, block).  One thread block per (run, kv head, k or v): its four
// warps take the block's positions in turn, keep the prepared values of their B / 4 positions in registers, agree on the
// largest magnitude through shared memory, and write codes once, so that every value is read once and rounded once.
// Held codes are read and rewritten only when the scale grows (a new largest value: for values without a trend once in
// i rows at the block's i-th row).  Query heads go to warps of their own.
#include <cmath>

#include "rows_q8.cuh"

namespace ts {

int rows_q8_to_dev(const char *what, const ts_rows_q8 *kv, const ts_kept *kept, uint32_t kv_heads, uint32_t width,
                   RowsQ8Dev *out) {
    TS_REQUIRE(kv && kept, "%s: the rows' record or the kept layout is NULL", what);
    TS_REQUIRE(kv->k && kv->v && kv->k_scale && kv->v_scale, "%s: codes or scales are NULL", what);
    TS_REQUIRE(aligned16(kv->k) && aligned16(kv->v) && (kv->k_bounds == nullptr || aligned16(kv->k_bounds)),
               "%s: codes and bounds must be 16-byte aligned", what);
    TS_REQUIRE(((reinterpret_cast<uintptr_t>(kv->k_scale) | reinterpret_cast<uintptr_t>(kv->v_scale)) & 3u) == 0,
               "%s: scales must be 4-byte aligned", what);
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

// Cosine and sine of pos * f, the product and its reduction to [-pi, pi] in 64 bits: in 32 bits position 100000 would
// leave an error of 100000 * 2^-24 = 0.006 radians.  Two constants: 2 pi and what its 64-bit form leaves out.
__device__ __forceinline__ void turn_of(uint32_t pos, float f, float *s, float *c) {
    double a = (double)pos * (double)f;
    const double n = rint(a * 0.15915494309189535);
    a = fma(n, -6.283185307179586, a);
    a = fma(n, -2.4492935982947064e-16, a);
    sincosf((float)a, s, c);
}

// A head's row on a warp: lane l owns the pairs j = l * PER + e (e < PER = W / 64): x[e] is element j, x[PER + e]
// element j + W / 2.
template <int W>
__device__ __forceinline__ void load_head(const uint16_t *src, uint32_t lane, uint32_t (&raw)[W / 64]) {
    constexpr int PER = W / 64;
    if constexpr (PER == 1) {
        raw[0] = (uint32_t)src[lane] | ((uint32_t)src[lane + W / 2] << 16);  // low half: element j, high half: j + W / 2
    } else if constexpr (PER == 2) {
        raw[0] = *reinterpret_cast<const uint32_t *>(src + lane * 2);
        raw[1] = *reinterpret_cast<const uint32_t *>(src + W / 2 + lane * 2);
    } else {
        const uint2 a = *reinterpret_cast<const uint2 *>(src + lane * 4), b = *reinterpret_cast<const uint2 *>(src + W / 2 + lane * 4);
        raw[0] = a.x; raw[1] = a.y; raw[2] = b.x; raw[3] = b.y;
    }
}

// The head's values in raw order (widened): x[i], i < W / 32, elements lane * PER + i, then W / 2 + lane * PER + i - PER.
template <int W>
__device__ __forceinline__ void widen(const uint32_t (&raw)[W / 64], float (&x)[W / 32]) {
#pragma unroll
    for (int i = 0; i < W / 64; i++) {
        x[2 * i] = bf16_lo(raw[i]);
        x[2 * i + 1] = bf16_hi(raw[i]);
    }
}

template <int W>
__device__ __forceinline__ void norm_turn(float (&x)[W / 32], const float *gain, const float (&sn)[W / 64],
                                          const float (&cs)[W / 64], float eps, uint32_t lane) {
    constexpr int PER = W / 64;
    if (gain) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < W / 32; i++) ss = fmaf(x[i], x[i], ss);
        const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)W + eps);
#pragma unroll
        for (int e = 0; e < PER; e++) {
            x[e] *= inv * gain[lane * PER + e];
            x[PER + e] *= inv * gain[lane * PER + e + W / 2];
        }
    }
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const float a = x[e], b = x[PER + e];
        x[e] = a * cs[e] - b * sn[e];
        x[PER + e] = a * sn[e] + b * cs[e];
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
    uint32_t kv_ctas;   // thread blocks [0, kv_ctas) do keys and values, the others queries
    uint32_t per_warp;  // query heads a warp takes
};

__device__ __forceinline__ int to_code(float x) {  // NaN converts to 0, infinities to the ends of the integer range
    return max(-127, min(127, __float2int_rn(x)));
}

template <int W, int B>
__global__ void __launch_bounds__(128) append_q8_kernel(const AppendParams p) {
    constexpr int PER = W / 64, N = W / 32, MINE = B / 4;  // positions of a block per warp
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t per_row = p.heads + 2 * p.kv_heads;
    pdl_wait();
    if (blockIdx.x >= p.kv_ctas) {
        // ---- queries: a warp takes `per_warp` heads of a row, the row's angles are computed once ----
        const uint32_t parts = (p.heads + p.per_warp - 1) / p.per_warp;
        const uint64_t unit = (uint64_t)(blockIdx.x - p.kv_ctas) * 4 + warp;
        if (unit < (uint64_t)p.rows * parts) {
            const uint32_t r = unit / parts, h0 = unit % parts * p.per_warp, h1 = min(p.heads, h0 + p.per_warp);
            const uint32_t pos = p.positions[r];
            float sn[PER], cs[PER];
#pragma unroll
            for (int e = 0; e < PER; e++) turn_of(pos, p.inv_freq[lane * PER + e], &sn[e], &cs[e]);
            for (uint32_t h = h0; h < h1; h++) {
                uint32_t raw[PER];
                load_head<W>(p.qkv + ((size_t)r * per_row + h) * W, lane, raw);
                float x[N];
                widen<W>(raw, x);
                norm_turn<W>(x, p.q_norm, sn, cs, p.eps, lane);
                uint16_t *dst = p.q_out + ((size_t)r * p.heads + h) * W;
                if constexpr (PER == 1) {
                    dst[lane] = bf16_bits(x[0]);
                    dst[lane + W / 2] = bf16_bits(x[1]);
                } else {
#pragma unroll
                    for (int e = 0; e < PER; e += 2) {
                        *reinterpret_cast<uint32_t *>(dst + lane * PER + e) = pack_bf16(x[e], x[e + 1]);
                        *reinterpret_cast<uint32_t *>(dst + W / 2 + lane * PER + e) = pack_bf16(x[PER + e], x[PER + e + 1]);
                    }
                }
            }
        }
        pdl_launch_dependents();
        return;
    }

    __shared__ int src[B];          // the row that writes each position of the block, or -1
    __shared__ uint32_t stop;
    __shared__ float sm_max[4];
    __shared__ int8_t sm_low[4][W], sm_high[4][W];
    const uint32_t units = 2 * p.kv_heads, unit = blockIdx.x % units;
    const bool is_v = unit >= p.kv_heads;
    const uint32_t h = is_v ? unit - p.kv_heads : unit;
    const uint32_t r0 = blockIdx.x / units * p.window, r1 = min(p.rows, r0 + p.window);
    for (uint32_t r = r0; r < r1; r++) {
        const uint32_t slot = p.slots[r], b = p.positions[r] >> p.kv.shift;
        if (r > 0 && p.slots[r - 1] == slot && (p.positions[r - 1] >> p.kv.shift) == b) continue;  // not a run's first row
        const uint32_t blk = block_of(p.kv, slot, b);
        if (blk == kNoBlock) continue;
        // ---- the run: which row writes which position ----
        __syncthreads();
        if (threadIdx.x < B) src[threadIdx.x] = -1;
        if (threadIdx.x == 0) stop = p.rows;
        __syncthreads();
        for (uint32_t base = r; base < p.rows; base += 128) {
            const uint32_t i = base + threadIdx.x;
            const uint32_t pos = i < p.rows ? p.positions[i] : 0;
            const bool in = i < p.rows && p.slots[i] == slot && (pos >> p.kv.shift) == b;
            if (!in && i < p.rows) atomicMin(&stop, i);
            __syncthreads();
            const uint32_t end = stop;
            if (in && i < end) atomicMax(&src[pos & (B - 1)], (int)i);
            if (end < base + 128) break;
        }
        __syncthreads();
        const bool fresh = src[0] >= 0;
        // ---- this warp's positions: warp, warp + 4, ... ----
        uint32_t raw[MINE][PER];
#pragma unroll
        for (int u = 0; u < MINE; u++) {
            const int row = src[warp + 4 * u];
#pragma unroll
            for (int e = 0; e < PER; e++) raw[u][e] = 0;
            if (row >= 0) load_head<W>(p.qkv + ((size_t)row * per_row + p.heads + unit) * W, lane, raw[u]);
        }
        float x[MINE][N];
        float most = 0.0f;
#pragma unroll
        for (int u = 0; u < MINE; u++) {
            widen<W>(raw[u], x[u]);
            if (!is_v && src[warp + 4 * u] >= 0) {
                float sn[PER], cs[PER];
#pragma unroll
                for (int e = 0; e < PER; e++)
                    turn_of((b << p.kv.shift) + warp + 4 * u, p.inv_freq[lane * PER + e], &sn[e], &cs[e]);
                norm_turn<W>(x[u], p.k_norm, sn, cs, p.eps, lane);
            }
#pragma unroll
            for (int i = 0; i < N; i++) most = fmaxf(most, fabsf(x[u][i]));  // fmaxf passes over NaN
        }
        most = warp_max(most);
        if (lane == 0) sm_max[warp] = most;
        __syncthreads();
        most = fminf(fmaxf(fmaxf(sm_max[0], sm_max[1]), fmaxf(sm_max[2], sm_max[3])), kLargest);
        const size_t at = (size_t)blk * p.kv_heads + h;
        float *scale = (is_v ? p.kv.v_scale : p.kv.k_scale) + at;
        const float s_old = fresh ? 0.0f : *scale;
        const float s_new = fmaxf(s_old, fmaxf(most / 127.0f, kScaleFloor));
        const float inv = 1.0f / s_new, ratio = fresh ? 1.0f : s_old / s_new;
        int8_t *codes = (is_v ? p.kv.v : p.kv.k) + at * B * W;
        int low[N], high[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            low[i] = 127;
            high[i] = -127;
        }
#pragma unroll
        for (int u = 0; u < MINE; u++) {
            int8_t *row = codes + (warp + 4 * u) * W;
            const bool written = src[warp + 4 * u] >= 0;
            if (!written && !(ratio < 1.0f)) continue;
            int c[N];
            if (written) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    c[i] = to_code(x[u][i] * inv);
                    low[i] = min(low[i], c[i]);
                    high[i] = max(high[i], c[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++)
                    c[i] = to_code((float)row[(i < PER ? 0 : W / 2 - PER) + lane * PER + i] * ratio);
            }
            if constexpr (PER == 1) {
                row[lane] = (int8_t)c[0];
                row[W / 2 + lane] = (int8_t)c[1];
            } else if constexpr (PER == 2) {
                *reinterpret_cast<uint16_t *>(row + lane * 2) = (uint16_t)((c[0] & 255) | (c[1] & 255) << 8);
                *reinterpret_cast<uint16_t *>(row + W / 2 + lane * 2) = (uint16_t)((c[2] & 255) | (c[3] & 255) << 8);
            } else {
                *reinterpret_cast<uint32_t *>(row + lane * 4) =
                    (c[0] & 255) | (c[1] & 255) << 8 | (c[2] & 255) << 16 | (uint32_t)(c[3] & 255) << 24;
                *reinterpret_cast<uint32_t *>(row + W / 2 + lane * 4) =
                    (c[4] & 255) | (c[5] & 255) << 8 | (c[6] & 255) << 16 | (uint32_t)(c[7] & 255) << 24;
            }
        }
        if (!is_v && p.kv.bounds) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int d = (i < PER ? 0 : W / 2 - PER) + lane * PER + i;
                sm_low[warp][d] = (int8_t)low[i];
                sm_high[warp][d] = (int8_t)high[i];
            }
        }
        __syncthreads();  // also: every thread has read the old scale
        if (!is_v && p.kv.bounds) {
            int8_t *bounds = p.kv.bounds + at * 2 * W;
            for (uint32_t d = threadIdx.x; d < W; d += 128) {
                int lo = min(min(sm_low[0][d], sm_low[1][d]), min(sm_low[2][d], sm_low[3][d]));
                int hi = max(max(sm_high[0][d], sm_high[1][d]), max(sm_high[2][d], sm_high[3][d]));
                if (!fresh) {
                    lo = min(lo, to_code((float)bounds[d] * ratio));
                    hi = max(hi, to_code((float)bounds[W + d] * ratio));
                }
                bounds[d] = (int8_t)lo;
                bounds[W + d] = (int8_t)hi;
            }
        }
        if (threadIdx.x == 0) *scale = s_new;
    }
    pdl_launch_dependents();
}

// One thread per 16 codes; a row's K and V pieces lie side by side in the grid.
template <int W>
__global__ void __launch_bounds__(256) unpack_q8_kernel(const RowsQ8Dev kv, const uint32_t *slots, const uint32_t *positions,
                                                        uint4 *k_out, uint4 *v_out, uint32_t rows, uint32_t kv_heads) {
    constexpr uint32_t PIECES = W / 16;
    pdl_wait();
    const uint32_t per_row = 2 * kv_heads * PIECES;
    const uint64_t total = (uint64_t)rows * per_row;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t r = i / per_row, rest = i % per_row;
        const bool is_v = rest >= kv_heads * PIECES;
        const uint32_t at = is_v ? rest - kv_heads * PIECES : rest, h = at / PIECES, piece = at % PIECES;
        const uint32_t pos = positions[r];
        const uint32_t blk = block_of(kv, slots[r], pos >> kv.shift);
        uint32_t out[8] = {};
        if (blk != kNoBlock) {
            const size_t head = (size_t)blk * kv_heads + h;
            const float s = (is_v ? kv.v_scale : kv.k_scale)[head];
            const int8_t *from = (is_v ? kv.v : kv.k) + ((head << kv.shift) + (pos & ((1u << kv.shift) - 1u))) * W + piece * 16;
            const int4 c = *reinterpret_cast<const int4 *>(from);
            const int w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                out[2 * j] = pack_bf16((float)(int8_t)w[j] * s, (float)(int8_t)(w[j] >> 8) * s);
                out[2 * j + 1] = pack_bf16((float)(int8_t)(w[j] >> 16) * s, (float)(int8_t)(w[j] >> 24) * s);
            }
        }
        uint4 *to = (is_v ? v_out : k_out) + ((size_t)r * kv_heads * PIECES + at) * 2;
        to[0] = make_uint4(out[0], out[1], out[2], out[3]);
        to[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
    pdl_launch_dependents();
}

template <int W>
cudaError_t launch_append(const AppendParams &p, uint32_t block, uint32_t grid, cudaStream_t stream) {
    return block == 16   ? launch(append_q8_kernel<W, 16>, dim3(grid), dim3(128), 0, stream, pdl_enabled(), p)
           : block == 32 ? launch(append_q8_kernel<W, 32>, dim3(grid), dim3(128), 0, stream, pdl_enabled(), p)
                         : launch(append_q8_kernel<W, 64>, dim3(grid), dim3(128), 0, stream, pdl_enabled(), p);
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
    // A step's rows each have a run of their own: a thread block for each.  A prompt's rows come in runs of up to a
    // block: looking at eight rows saves seven of eight thread blocks that would find no run to start.
    p.window = rows <= 256 ? 1 : 8;
    p.per_warp = (uint64_t)rows * heads > 8192 ? 4 : 1;
    const uint64_t kv_ctas = (uint64_t)ceil_div(rows, p.window) * 2 * kv_heads;
    const uint64_t q_ctas = ((uint64_t)rows * ceil_div(heads, p.per_warp) + 3) / 4;
    TS_REQUIRE(kv_ctas + q_ctas < 0x7FFFFFFFull, "append (q8): %u rows of %u heads are too many for one launch", rows, heads);
    p.kv_ctas = (uint32_t)kv_ctas;
    const uint32_t grid = (uint32_t)(kv_ctas + q_ctas), block = 1u << kv.shift;
    const cudaError_t e = width == 64    ? launch_append<64>(p, block, grid, stream)
                          : width == 128 ? launch_append<128>(p, block, grid, stream)
                                         : launch_append<256>(p, block, grid, stream);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of append (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

int unpack_q8(const RowsQ8Dev &kv, const uint32_t *slots, const uint32_t *positions, void *k_out, void *v_out, uint32_t rows,
              uint32_t kv_heads, uint32_t width, cudaStream_t stream) {
    const uint64_t threads = (uint64_t)rows * 2 * kv_heads * (width / 16);
    const uint64_t most = (uint64_t)sm_count() * 8 * 4;
    const uint64_t want = (threads + 255) / 256;
    const dim3 grid((uint32_t)(want < most ? want : most));
    const cudaError_t e =
        width == 64    ? launch(unpack_q8_kernel<64>, grid, dim3(256), 0, stream, pdl_enabled(), kv, slots, positions, (uint4 *)k_out, (uint4 *)v_out, rows, kv_heads)
        : width == 128 ? launch(unpack_q8_kernel<128>, grid, dim3(256), 0, stream, pdl_enabled(), kv, slots, positions, (uint4 *)k_out, (uint4 *)v_out, rows, kv_heads)
                       : launch(unpack_q8_kernel<256>, grid, dim3(256), 0, stream, pdl_enabled(), kv, slots, positions, (uint4 *)k_out, (uint4 *)v_out, rows, kv_heads);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of unpack (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

}  // namespace ts
