// Which blocks of 8-bit kept rows a query should read: an upper bound of q . k for each block from the lowest and the
// highest key code of every channel, then the `count` best.
//
// With the query as whole numbers c_g (one scale for the group's heads) the sum over the heads of
// max(c hi, c lo) is max(c, 0) hi + min(c, 0) lo summed over heads first: one dot product of 2 * width whole numbers a
// block whatever the group's size, taken with dp2a (16-bit weights, 8-bit bounds).  Nothing is rounded before the one
// multiplication by the block's key scale, so any order of summation gives the same scores and the same choice.
#include <cmath>

#include "rows_q8.cuh"

namespace ts {
namespace {

struct SelectParams {
    const uint16_t *q;
    RowsQ8Dev kv;
    uint32_t *ids;
    const uint32_t *slots, *positions;
    uint32_t rows, keys, heads, kv_heads, count, first, recent;
    uint32_t most;    // blocks a row may have: the scores' row length
    float *scores;    // [rows, kv_heads, most]
};

__device__ __forceinline__ int dp2a_lo(int a, int b, int c) {  // a: two s16, b: four s8, its low two
    int d;
    asm("dp2a.lo.s32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ int dp2a_hi(int a, int b, int c) {
    int d;
    asm("dp2a.hi.s32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

constexpr int kScore = 128;  // threads of a scoring thread block, and the blocks it scores

// Blocks that hold a position a row sees: 1 + min(pos, keys - 1) / B.
__device__ __forceinline__ uint32_t blocks_of(const SelectParams &p, uint32_t row) {
    return (min(p.positions[row], p.keys - 1) >> p.kv.shift) + 1;
}

// Order of a score as a whole number: larger scores larger, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float score) {
    const uint32_t u = __float_as_uint(score + 0.0f);  // -0 and 0 rank alike
    return score != score ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A warp scores 32 blocks: its lanes look them up side by side, W / 8 lanes then hold a block's 2 W bounds, 16 a lane, and
// several blocks' bounds are under way before the weights are ready.
template <int W>
__global__ void __launch_bounds__(kScore) score_blocks_kernel(const SelectParams p) {
    constexpr uint32_t LANES = W / 8, AT_ONCE = 32 / LANES, LOADS = 32 / AT_ONCE;  // loads for 32 blocks
    constexpr uint32_t EARLY = LOADS < 8 ? LOADS : 8;
    __shared__ __align__(16) int16_t weight[2][W];  // for the lowest codes, for the highest
    __shared__ float sm_max[kScore / 32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    const uint32_t row = blockIdx.z, h = blockIdx.y, n = blocks_of(p, row), b0 = blockIdx.x * kScore;
    if (n <= p.count || b0 >= n) {
        pdl_launch_dependents();
        return;
    }
    const uint32_t mine = b0 + warp * 32 + lane, part = lane % LANES, which = lane / LANES;
    const uint32_t blk = mine < n ? block_of(p.kv, p.slots[row], mine) : kNoBlock;
    const uint32_t group = p.heads / p.kv_heads;
    const uint16_t *q = p.q + ((size_t)row * p.heads + h * group) * W;
    // channels threadIdx.x, + kScore: the group's largest magnitude
    float most = 0.0f;
    for (uint32_t i = threadIdx.x; i < group * W / 2; i += kScore) {
        const uint32_t v = reinterpret_cast<const uint32_t *>(q)[i];
        most = fmaxf(most, fmaxf(fabsf(bf16_lo(v)), fabsf(bf16_hi(v))));
    }
    int4 c[EARLY];
    auto bounds_at = [&](uint32_t k) {  // of the block that load k has for this lane
        const uint32_t b = __shfl_sync(0xFFFFFFFFu, blk, k * AT_ONCE + which);
        return b == kNoBlock ? make_int4(0, 0, 0, 0) : *reinterpret_cast<const int4 *>(p.kv.bounds + ((size_t)b * p.kv_heads + h) * 2 * W + part * 16);
    };
#pragma unroll
    for (uint32_t k = 0; k < EARLY; k++) c[k] = bounds_at(k);
    const float scale = blk == kNoBlock ? 0.0f : p.kv.k_scale[(size_t)blk * p.kv_heads + h];
    most = warp_max(most);
    if (lane == 0) sm_max[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScore / 32; w++) most = fmaxf(most, sm_max[w]);
    for (uint32_t d = threadIdx.x; d < W; d += kScore) {
        int up = 0, down = 0;
        for (uint32_t g = 0; g < group; g++) {
            const float x = bf16_lo(q[g * W + d]);
            // NaN and infinity over infinity convert to 0
            const int code = most > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x * 127.0f, most)))) : 0;
            up += max(code, 0);
            down += min(code, 0);
        }
        weight[0][d] = (int16_t)down;
        weight[1][d] = (int16_t)up;
    }
    __syncthreads();
    int w[8];  // of this lane's 16 channels
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = reinterpret_cast<const int *>(&weight[0][0])[part * 8 + i];
    int total = 0;  // of this lane's own block
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) {
        const int4 v = k < EARLY ? c[k < EARLY ? k : 0] : bounds_at(k);
        const int b[4] = {v.x, v.y, v.z, v.w};
        int sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sum = dp2a_lo(w[2 * i], b[i], sum);
            sum = dp2a_hi(w[2 * i + 1], b[i], sum);
        }
#pragma unroll
        for (uint32_t o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const int got = __shfl_sync(0xFFFFFFFFu, sum, (lane % AT_ONCE) * LANES);  // block k * AT_ONCE + lane % AT_ONCE
        if (lane / AT_ONCE == k) total = got;
    }
    if (mine < n)
        p.scores[((size_t)row * p.kv_heads + h) * p.most + mine] = blk == kNoBlock ? -INFINITY : __fmul_rn(__int2float_rn(total), scale);
    pdl_launch_dependents();
}

constexpr int kPick = 256;
constexpr uint32_t kHeld = 4;

// One thread block per (row, kv head): the rank of the count-th best by four passes over 8-bit digits, then the blocks
// above it, and the lowest of those at it, in ascending order.
__global__ void __launch_bounds__(kPick) pick_blocks_kernel(const SelectParams p) {
    __shared__ uint32_t hist[256], sm_gt[kPick / 32], sm_eq[kPick / 32], sm_digit, sm_left;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    const uint32_t row = blockIdx.y, h = blockIdx.x, n = blocks_of(p, row);
    uint32_t *ids = p.ids + ((size_t)row * p.kv_heads + h) * p.count;
    if (n <= p.count) {
        for (uint32_t i = threadIdx.x; i < p.count; i += kPick) ids[i] = i < n ? i : 0xFFFFFFFFu;
        pdl_launch_dependents();
        return;
    }
    const float *scores = p.scores + ((size_t)row * p.kv_heads + h) * p.most;
    auto ranked = [&](uint32_t i) { return i < p.first || i >= n - p.recent ? 0xFFFFFFFFu : min(rank_of(scores[i]), 0xFFFFFFFEu); };
    // the first kHeld of a thread's blocks stay in registers over the passes
    uint32_t held[kHeld];
#pragma unroll
    for (uint32_t k = 0; k < kHeld; k++) held[k] = threadIdx.x + k * kPick < n ? ranked(threadIdx.x + k * kPick) : 0;
    uint32_t prefix = 0, left = p.count;  // the digits found so far; how many are still to come among those that share them
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[threadIdx.x] = 0;
        __syncthreads();
        auto count = [&](uint32_t u) {
            if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1u);
        };
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++)
            if (threadIdx.x + k * kPick < n) count(held[k]);
        for (uint32_t i = threadIdx.x + kHeld * kPick; i < n; i += kPick) count(ranked(i));
        __syncthreads();
        if (warp == 0) {
            // lane l: digits 255 - 8 l downwards
            uint32_t mine = 0;
            for (int i = 0; i < 8; i++) mine += hist[255 - 8 * lane - i];
            uint32_t before = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, before, o);
                if (lane >= (uint32_t)o) before += other;
            }
            before -= mine;
            if (before < left && before + mine >= left) {
                uint32_t at = before, d = 255 - 8 * lane;
                while (at + hist[d] < left) at += hist[d--];
                sm_digit = d;
                sm_left = left - at;
            }
        }
        __syncthreads();
        prefix |= sm_digit << shift;
        left = sm_left;
    }
    // ranks above `prefix` are in; of those equal to it the first `left`
    uint32_t out = 0, equal = 0;  // taken so far, seen at the border so far
    for (uint32_t base = 0; base < n && out < p.count; base += kPick) {
        const uint32_t i = base + threadIdx.x;
        uint32_t u = 0;
        if (base < kHeld * kPick) {
#pragma unroll
            for (uint32_t k = 0; k < kHeld; k++)
                if (base == k * kPick) u = held[k];
        } else if (i < n) {
            u = ranked(i);
        }
        const bool gt = i < n && u > prefix, eq = i < n && u == prefix;
        const uint32_t m_gt = __ballot_sync(0xFFFFFFFFu, gt), m_eq = __ballot_sync(0xFFFFFFFFu, eq);
        __syncthreads();
        if (lane == 0) {
            sm_gt[warp] = __popc(m_gt);
            sm_eq[warp] = __popc(m_eq);
        }
        __syncthreads();
        uint32_t gt_before = __popc(m_gt & ((1u << lane) - 1)), eq_before = equal + __popc(m_eq & ((1u << lane) - 1));
        uint32_t gts = 0, eqs = 0;
        for (uint32_t w = 0; w < kPick / 32; w++) {
            if (w < warp) {
                gt_before += sm_gt[w];
                eq_before += sm_eq[w];
            }
            gts += sm_gt[w];
            eqs += sm_eq[w];
        }
        // taken before this one: the larger ones, and of the equal ones at most `left`
        const uint32_t at = out + gt_before + min(eq_before, left) - min(equal, left);
        if (gt || (eq && eq_before < left)) ids[at] = i;
        out += gts + min(equal + eqs, left) - min(equal, left);
        equal += eqs;
    }
    pdl_launch_dependents();
}

}  // namespace

size_t select_q8_workspace_bytes(uint32_t rows, uint32_t keys, uint32_t kv_heads, uint32_t block, uint32_t count) {
    if (rows == 0 || keys == 0 || block == 0) return 0;
    const uint32_t most = (uint32_t)(((uint64_t)keys + block - 1) / block);
    return most <= count ? 0 : (size_t)rows * kv_heads * most * sizeof(float);
}

int select_q8(const void *q, const RowsQ8Dev &kv, uint32_t *ids, const uint32_t *slots, const uint32_t *positions, uint32_t rows,
              uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t count, uint32_t first,
              uint32_t recent, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    SelectParams p = {};
    p.q = (const uint16_t *)q;
    p.kv = kv;
    p.ids = ids;
    p.slots = slots;
    p.positions = positions;
    p.rows = rows;
    p.keys = keys;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.count = count;
    p.first = first;
    p.recent = recent;
    p.most = (uint32_t)(((uint64_t)keys + (1u << kv.shift) - 1) >> kv.shift);
    p.scores = (float *)workspace;
    const size_t need = select_q8_workspace_bytes(rows, keys, kv_heads, 1u << kv.shift, count);
    TS_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && aligned16(workspace))),
               "select_blocks (q8): workspace of %zu bytes is smaller than the %zu needed, or not 16-byte aligned",
               workspace_bytes, need);
    TS_REQUIRE(rows <= 65535, "select_blocks (q8): %u rows are more than 65535", rows);
    cudaError_t e = cudaSuccess;
    if (need) {
        const dim3 grid(ceil_div(p.most, kScore), kv_heads, rows);
        e = width == 64    ? launch(score_blocks_kernel<64>, grid, dim3(kScore), 0, stream, pdl_enabled(), p)
            : width == 128 ? launch(score_blocks_kernel<128>, grid, dim3(kScore), 0, stream, pdl_enabled(), p)
                           : launch(score_blocks_kernel<256>, grid, dim3(kScore), 0, stream, pdl_enabled(), p);
    }
    if (e == cudaSuccess) e = launch(pick_blocks_kernel, dim3(kv_heads, rows), dim3(kPick), 0, stream, need ? true : pdl_enabled(), p);
    if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of select_blocks (q8) failed: %s", cudaGetErrorString(e));
    return TS_OK;
}

}  // namespace ts
