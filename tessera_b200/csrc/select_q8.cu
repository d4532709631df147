// Which blocks of 8-bit kept rows a query should read: an upper bound of q . k for each block from the lowest and the
// highest key code of every channel, then the `count` best.
//
// With the query as whole numbers c_g (one scale for the group's heads) the sum over the heads of
// max(c hi, c lo) is max(c, 0) hi + min(c, 0) lo summed over heads first: one dot product of 2 * width whole numbers a
// block whatever the group's size, taken with dp2a (16-bit weights, 8-bit bounds).  Nothing is rounded before the one
// multiplication by the block's key scale, so any order of summation gives the same scores and the same choice.
//
// 64 rows x 4 kv heads x up to 512 blocks of width 128 take 13.3 us, of which the bounds' bytes would need 4: the pick's
// passes over the ranks follow the last score.  8 rows x 8 kv heads x 256 blocks take 6.9 us, one load after another.
// Thousands of blocks, in two launches: 1 row x 8 kv heads x 6000 28 us, 8 rows 45, 64 rows 170 (of which the bounds' bytes 120).
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

// The group's query codes as weights: weight[0] for the lowest codes (the negative ones summed), weight[1] for the highest.
// The queries pass through shared memory where they fit, so that each is read once.
constexpr uint32_t kQueryWords = 2048;  // pairs of bf16: up to 16 heads of 256, 32 of 128, 64 of 64

template <int W, int THREADS>
__device__ __forceinline__ void weigh(const uint16_t *q, uint32_t group, int16_t (&weight)[2][W], float (&sm_max)[THREADS / 32]) {
    __shared__ __align__(16) uint32_t sm_q[kQueryWords];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, words = group * W / 2;
    const bool fits = words <= kQueryWords;
    float most = 0.0f;
    for (uint32_t i = threadIdx.x * 4; i < words; i += THREADS * 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(q + 2 * i);
        if (fits) *reinterpret_cast<uint4 *>(sm_q + i) = v;
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) most = fmaxf(most, fmaxf(fabsf(bf16_lo(x[k])), fabsf(bf16_hi(x[k]))));
    }
    most = warp_max(most);
    if (lane == 0) sm_max[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) most = fmaxf(most, sm_max[w]);
    for (uint32_t d = threadIdx.x; d < W / 2; d += THREADS) {  // two channels
        int up[2] = {0, 0}, down[2] = {0, 0};
#pragma unroll 4
        for (uint32_t g = 0; g < group; g++) {
            const uint32_t v = fits ? sm_q[g * (W / 2) + d] : reinterpret_cast<const uint32_t *>(q)[g * (W / 2) + d];
            const float x[2] = {bf16_lo(v), bf16_hi(v)};
#pragma unroll
            for (int k = 0; k < 2; k++) {
                // NaN and infinity over infinity convert to 0
                const int code = most > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x[k] * 127.0f, most)))) : 0;
                up[k] += max(code, 0);
                down[k] += min(code, 0);
            }
        }
        reinterpret_cast<uint32_t *>(weight[0])[d] = (uint32_t)(down[0] & 0xFFFF) | (uint32_t)down[1] << 16;
        reinterpret_cast<uint32_t *>(weight[1])[d] = (uint32_t)(up[0] & 0xFFFF) | (uint32_t)up[1] << 16;
    }
    __syncthreads();
}

// A warp scores 32 blocks, `blk` a lane: W / 8 lanes hold a block's 2 W bounds, 16 a lane, so that a load instruction has
// AT_ONCE blocks.  The first EARLY loads may be asked for before the weights are ready.
template <int W>
struct Scorer {
    static constexpr uint32_t LANES = W / 8, AT_ONCE = 32 / LANES, LOADS = LANES, EARLY = LOADS < 8 ? LOADS : 8;
    int4 c[EARLY];

    __device__ __forceinline__ int4 bounds_at(const SelectParams &p, uint32_t h, uint32_t blk, uint32_t k, uint32_t lane) {
        const uint32_t b = __shfl_sync(0xFFFFFFFFu, blk, k * AT_ONCE + lane / LANES);
        if (b == kNoBlock) return make_int4(0, 0, 0, 0);
        return *reinterpret_cast<const int4 *>(p.kv.bounds + ((size_t)b * p.kv_heads + h) * 2 * W + lane % LANES * 16);
    }
    __device__ __forceinline__ void ask(const SelectParams &p, uint32_t h, uint32_t blk, uint32_t lane) {
#pragma unroll
        for (uint32_t k = 0; k < EARLY; k++) c[k] = bounds_at(p, h, blk, k, lane);
    }
    // The lane's own block's sum; w: the weights of this lane's 16 channels.
    __device__ __forceinline__ int total(const SelectParams &p, uint32_t h, uint32_t blk, const int (&w)[8], uint32_t lane) {
        int sum[LOADS];
#pragma unroll
        for (uint32_t k = 0; k < LOADS; k++) {
            const int4 v = k < EARLY ? c[k < EARLY ? k : 0] : bounds_at(p, h, blk, k, lane);
            const int b[4] = {v.x, v.y, v.z, v.w};
            sum[k] = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sum[k] = dp2a_lo(w[2 * i], b[i], sum[k]);
                sum[k] = dp2a_hi(w[2 * i + 1], b[i], sum[k]);
            }
        }
        // LANES sums over LANES lanes, halved with each exchange: lane l of them ends with load l's
#pragma unroll
        for (uint32_t o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
            for (uint32_t i = 0; i < o; i++) {
                const bool upper = lane & o;
                const int give = upper ? sum[i] : sum[i + o], keep = upper ? sum[i + o] : sum[i];
                sum[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
            }
        return __shfl_sync(0xFFFFFFFFu, sum[0], lane % AT_ONCE * LANES + lane / AT_ONCE);
    }
};

__device__ __forceinline__ float score_of(const SelectParams &p, uint32_t h, uint32_t blk, int total, float scale) {
    return blk == kNoBlock ? -INFINITY : __fmul_rn(__int2float_rn(total), scale);
}

template <int W>
__global__ void __launch_bounds__(kScore) score_blocks_kernel(const SelectParams p) {
    __shared__ __align__(16) int16_t weight[2][W];
    __shared__ float sm_max[kScore / 32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    const uint32_t row = blockIdx.z, h = blockIdx.y, n = blocks_of(p, row), b0 = blockIdx.x * kScore;
    if (n <= p.count || b0 >= n) {
        pdl_launch_dependents();
        return;
    }
    const uint32_t mine = b0 + warp * 32 + lane, group = p.heads / p.kv_heads;
    const uint32_t blk = mine < n ? block_of(p.kv, p.slots[row], mine) : kNoBlock;
    Scorer<W> scorer;
    scorer.ask(p, h, blk, lane);
    const float scale = blk == kNoBlock ? 0.0f : p.kv.k_scale[(size_t)blk * p.kv_heads + h];
    weigh<W, kScore>(p.q + ((size_t)row * p.heads + h * group) * W, group, weight, sm_max);
    int w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = reinterpret_cast<const int *>(&weight[0][0])[lane % Scorer<W>::LANES * 8 + i];
    const int total = scorer.total(p, h, blk, w, lane);
    if (mine < n) p.scores[((size_t)row * p.kv_heads + h) * p.most + mine] = score_of(p, h, blk, total, scale);
    pdl_launch_dependents();
}

constexpr int kPick = 256;
constexpr uint32_t kHeld = 4;  // blocks whose ranks a thread keeps: threadIdx.x, + kPick, ...

struct PickShared {
    uint32_t hist[256], gt[kPick / 32], eq[kPick / 32], digit, left;
};

// The ids of the p.count best of n blocks by a thread block: the rank of the count-th best by four passes over 8-bit
// digits, then the blocks above it, and the lowest of those at it, in ascending order.  rank(i) for the blocks past those
// whose ranks are held.
template <typename Rank>
__device__ __forceinline__ void pick(const SelectParams &p, uint32_t n, uint32_t *ids, const uint32_t (&held)[kHeld], PickShared &sm, Rank rank) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t prefix = 0, left = p.count;  // the digits found so far; how many are still to come among those that share them
    for (int shift = 24; shift >= 0; shift -= 8) {
        sm.hist[threadIdx.x] = 0;
        __syncthreads();
        auto count = [&](uint32_t u) {
            if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sm.hist[(u >> shift) & 255], 1u);
        };
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++)
            if (threadIdx.x + k * kPick < n) count(held[k]);
        for (uint32_t i = threadIdx.x + kHeld * kPick; i < n; i += kPick) count(rank(i));
        __syncthreads();
        if (warp == 0) {
            // lane l: digits 255 - 8 l downwards
            uint32_t mine = 0;
            for (int i = 0; i < 8; i++) mine += sm.hist[255 - 8 * lane - i];
            uint32_t before = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, before, o);
                if (lane >= (uint32_t)o) before += other;
            }
            before -= mine;
            if (before < left && before + mine >= left) {
                uint32_t at = before, d = 255 - 8 * lane;
                while (at + sm.hist[d] < left) at += sm.hist[d--];
                sm.digit = d;
                sm.left = left - at;
            }
        }
        __syncthreads();
        prefix |= sm.digit << shift;
        left = sm.left;
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
            u = rank(i);
        }
        const bool gt = i < n && u > prefix, eq = i < n && u == prefix;
        const uint32_t m_gt = __ballot_sync(0xFFFFFFFFu, gt), m_eq = __ballot_sync(0xFFFFFFFFu, eq);
        __syncthreads();
        if (lane == 0) {
            sm.gt[warp] = __popc(m_gt);
            sm.eq[warp] = __popc(m_eq);
        }
        __syncthreads();
        uint32_t gt_before = __popc(m_gt & ((1u << lane) - 1)), eq_before = equal + __popc(m_eq & ((1u << lane) - 1));
        uint32_t gts = 0, eqs = 0;
        for (uint32_t w = 0; w < kPick / 32; w++) {
            if (w < warp) {
                gt_before += sm.gt[w];
                eq_before += sm.eq[w];
            }
            gts += sm.gt[w];
            eqs += sm.eq[w];
        }
        // taken before this one: the larger ones, and of the equal ones at most `left`
        const uint32_t at = out + gt_before + min(eq_before, left) - min(equal, left);
        if (gt || (eq && eq_before < left)) ids[at] = i;
        out += gts + min(equal + eqs, left) - min(equal, left);
        equal += eqs;
    }
}

__device__ __forceinline__ uint32_t rank_at(const SelectParams &p, uint32_t n, uint32_t i, float score) {
    return i < p.first || i >= n - p.recent ? 0xFFFFFFFFu : min(rank_of(score), 0xFFFFFFFEu);
}

// Every block taken: no more of them than asked for.
__device__ __forceinline__ bool take_all(const SelectParams &p, uint32_t n, uint32_t *ids) {
    if (n > p.count) return false;
    for (uint32_t i = threadIdx.x; i < p.count; i += kPick) ids[i] = i < n ? i : 0xFFFFFFFFu;
    return true;
}

// One thread block per (row, kv head), over the scores of another launch.
__global__ void __launch_bounds__(kPick) pick_blocks_kernel(const SelectParams p) {
    __shared__ PickShared sm;
    pdl_wait();
    const uint32_t row = blockIdx.y, h = blockIdx.x, n = blocks_of(p, row);
    uint32_t *ids = p.ids + ((size_t)row * p.kv_heads + h) * p.count;
    if (!take_all(p, n, ids)) {
        const float *scores = p.scores + ((size_t)row * p.kv_heads + h) * p.most;
        auto rank = [&](uint32_t i) { return rank_at(p, n, i, scores[i]); };
        uint32_t held[kHeld];
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) held[k] = threadIdx.x + k * kPick < n ? rank(threadIdx.x + k * kPick) : 0;
        pick(p, n, ids, held, sm, rank);
    }
    pdl_launch_dependents();
}

// Scores and choice of up to kHeld * kPick blocks by one thread block per (row, kv head): the scores stay in the
// registers of the threads that pick.
template <int W>
__global__ void __launch_bounds__(kPick) select_blocks_kernel(const SelectParams p) {
    __shared__ PickShared sm;
    __shared__ __align__(16) int16_t weight[2][W];
    __shared__ float sm_max[kPick / 32];
    const uint32_t lane = threadIdx.x & 31;
    pdl_wait();
    const uint32_t row = blockIdx.y, h = blockIdx.x, n = blocks_of(p, row);
    uint32_t *ids = p.ids + ((size_t)row * p.kv_heads + h) * p.count;
    if (!take_all(p, n, ids)) {
        const uint32_t group = p.heads / p.kv_heads, slot = p.slots[row];
        uint32_t blk[kHeld];
        float scale[kHeld];
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) blk[k] = threadIdx.x + k * kPick < n ? block_of(p.kv, slot, threadIdx.x + k * kPick) : kNoBlock;
        Scorer<W> scorer;
        scorer.ask(p, h, blk[0], lane);
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) scale[k] = blk[k] == kNoBlock ? 0.0f : p.kv.k_scale[(size_t)blk[k] * p.kv_heads + h];
        weigh<W, kPick>(p.q + ((size_t)row * p.heads + h * group) * W, group, weight, sm_max);
        int w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = reinterpret_cast<const int *>(&weight[0][0])[lane % Scorer<W>::LANES * 8 + i];
        uint32_t held[kHeld] = {};
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) {
            if ((threadIdx.x & ~31u) + k * kPick >= n) break;  // the whole warp's blocks
            const int total = scorer.total(p, h, blk[k], w, lane);
            if (k + 1 < kHeld) scorer.ask(p, h, blk[k + 1 < kHeld ? k + 1 : 0], lane);
            held[k] = rank_at(p, n, threadIdx.x + k * kPick, score_of(p, h, blk[k], total, scale[k]));
        }
        pick(p, n, ids, held, sm, [](uint32_t) { return 0u; });
    }
    pdl_launch_dependents();
}

// Whether one kernel scores and picks.  It has a thread block for a (row, kv head), two of them fit an SM, and each goes over
// its bounds by itself; of the two launches, the first one spreads them over the GPU.  Measured in us, one kernel / two
// launches, width 128 where no other is given:
//   up to two thread blocks an SM, up to 256 blocks: 1 x 8 (rows x kv heads) 6.5 / 7.1, 37 x 8 8.0 / 9.0, 64 x 4 8.7 / 9.6
//   more of them than that, whatever the blocks: 64 x 8 12.9 / 9.4 (128 blocks), 26.2 / 21.3 (512), 512 x 8 99 / 42 (70)
//   more blocks: few thread blocks leave SMs idle for long, 1 x 8 8.3 / 7.6 (512), 8 x 4 9.3 / 8.8; from 128 of them on one
//   kernel is as good or better up to 512 blocks, 16 x 8 8.9 / 9.2, 64 x 4 14.7 / 15.6 (24 x 8 11.0 / 10.5), but at width
//   256, 16 x 8 22.0 / 13.7; at 768 blocks 64 x 4 19.9 / 19.2, at 1024 8 x 8 12.0 / 10.3
bool together(uint64_t jobs, uint32_t blocks, uint32_t width) {
    if (jobs > 2ull * sm_count()) return false;
    return blocks <= 256 || (blocks <= 512 && jobs >= 128 && width <= 128);
}
static_assert(512 <= kHeld * kPick, "the scores are held in registers");

size_t scores_bytes(uint32_t rows, uint32_t most, uint32_t kv_heads, uint32_t count, uint32_t width) {
    if (most <= count || together((uint64_t)rows * kv_heads, most, width)) return 0;
    return (size_t)rows * kv_heads * most * sizeof(float);
}

}  // namespace

size_t select_q8_workspace_bytes(uint32_t rows, uint32_t keys, uint32_t kv_heads, uint32_t block, uint32_t count) {
    if (rows == 0 || keys == 0 || block == 0) return 0;
    const uint32_t most = (uint32_t)(((uint64_t)keys + block - 1) / block);
    return scores_bytes(rows, most, kv_heads, count, 256);  // what suffices at any width
}

int select_q8(const void *q, const RowsQ8Dev &kv, uint32_t *ids, const uint32_t *slots, const uint32_t *positions, uint32_t rows,
              uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t count, uint32_t first,
              uint32_t recent, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    // A slot has no keys past what its stride or its pages hold (and fewer keys never ask for a larger workspace).
    const uint64_t room = (uint64_t)kv.scalar << (kv.per_shift + kv.shift);
    if (room < keys) keys = (uint32_t)room;
    SelectParams p = {};
    p.kv = kv;
    p.keys = keys;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.count = count;
    p.first = first;
    p.recent = recent;
    p.most = (uint32_t)(((uint64_t)keys + (1u << kv.shift) - 1) >> kv.shift);
    const size_t need = scores_bytes(rows, p.most, kv_heads, count, width);
    TS_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && aligned16(workspace))),
               "select_blocks (q8): workspace of %zu bytes is smaller than the %zu needed, or not 16-byte aligned",
               workspace_bytes, need);
    constexpr uint32_t kTogetherRows = 65535;  // a launch's
    for (uint32_t row = 0; row < rows; row += kTogetherRows) {
        const uint32_t n = min(kTogetherRows, rows - row);
        p.rows = n;
        p.q = (const uint16_t *)q + (size_t)row * heads * width;
        p.ids = ids + (size_t)row * kv_heads * count;
        p.slots = slots + row;
        p.positions = positions + row;
        p.scores = need ? (float *)workspace + (size_t)row * kv_heads * p.most : nullptr;
        const dim3 each(kv_heads, n);
        cudaError_t e;
        if (need) {
            const dim3 grid(ceil_div(p.most, kScore), kv_heads, n);
            e = width == 64    ? launch(score_blocks_kernel<64>, grid, dim3(kScore), 0, stream, pdl_enabled(), p)
                : width == 128 ? launch(score_blocks_kernel<128>, grid, dim3(kScore), 0, stream, pdl_enabled(), p)
                               : launch(score_blocks_kernel<256>, grid, dim3(kScore), 0, stream, pdl_enabled(), p);
            if (e == cudaSuccess) e = launch(pick_blocks_kernel, each, dim3(kPick), 0, stream, true, p);
        } else {
            e = width == 64    ? launch(select_blocks_kernel<64>, each, dim3(kPick), 0, stream, pdl_enabled(), p)
                : width == 128 ? launch(select_blocks_kernel<128>, each, dim3(kPick), 0, stream, pdl_enabled(), p)
                               : launch(select_blocks_kernel<256>, each, dim3(kPick), 0, stream, pdl_enabled(), p);
        }
        if (e != cudaSuccess) return fail(TS_ERR_CUDA, "launch of select_blocks (q8) failed: %s", cudaGetErrorString(e));
    }
    return TS_OK;
}

}  // namespace ts
