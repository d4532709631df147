// Kept rows in 8 bits (ts_rows_q8): the walk from (slot, block of positions) to the pool's block, and the host-side
// check of the two records that describe it.
#pragma once

#include "ts_common.cuh"

namespace ts {

constexpr uint32_t kNoBlock = 0xFFFFFFFFu;
constexpr uint32_t kMostListed = 1u << 24;  // blocks that a row and kv head may list

struct RowsQ8Dev {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int8_t *bounds;
    uint32_t shift;      // log2 of the positions a block covers
    uint32_t blocks;     // blocks in the pool
    uint32_t per_shift;  // paged: log2 of the blocks a page holds
    uint32_t scalar;     // dense: blocks per slot; paged: pages per slot
    uint32_t table_len;
    const uint32_t *table;  // NULL: dense
};

// The pool's block with block `b` of `slot`'s positions, or kNoBlock when slot, position or table lead outside it.
__device__ __forceinline__ uint32_t block_of(const RowsQ8Dev &p, uint32_t slot, uint32_t b) {
    uint64_t at;
    if (p.table == nullptr) {
        if (b >= p.scalar) return kNoBlock;
        at = (uint64_t)slot * p.scalar + b;
    } else {
        const uint32_t page = b >> p.per_shift;
        const uint64_t entry = (uint64_t)slot * p.scalar + page;
        if (page >= p.scalar || entry >= p.table_len) return kNoBlock;
        at = ((uint64_t)p.table[entry] << p.per_shift) | (b & ((1u << p.per_shift) - 1u));
    }
    return at < p.blocks ? (uint32_t)at : kNoBlock;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
    return v;
}

// Arrays of f32 or u32 that a kernel reads an element at a time (NULL is as aligned as any).
inline bool aligned4(const void *a, const void *b = nullptr, const void *c = nullptr) {
    return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & 3u) == 0;
}

// TS_OK, or the recorded failure; `what` names the entry point.
int rows_q8_to_dev(const char *what, const ts_rows_q8 *kv, const ts_kept *kept, uint32_t kv_heads, uint32_t width,
                   RowsQ8Dev *out);

int append_q8(const void *qkv, const float *q_norm, const float *k_norm, const float *inv_freq, const uint32_t *slots,
              const uint32_t *positions, void *q_out, const RowsQ8Dev &kv, uint32_t rows, uint32_t heads,
              uint32_t kv_heads, uint32_t width, float eps, cudaStream_t stream);
int unpack_q8(const RowsQ8Dev &kv, const uint32_t *slots, const uint32_t *positions, void *k_out, void *v_out, uint32_t rows,
              uint32_t kv_heads, uint32_t width, cudaStream_t stream);
// ids NULL: rows [max(0, pos - back), min(pos + 1, keys)) of the slot; else the `count` listed blocks per row and kv head.
size_t attend_q8_workspace_bytes(uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t back,
                                 uint32_t count, uint32_t block);
int attend_q8_take_status();
int attend_q8(const void *q, const RowsQ8Dev &kv, const uint32_t *ids, void *out, const uint32_t *slots,
              const uint32_t *positions, uint32_t rows, uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width,
              uint32_t back, uint32_t count, float scale, void *workspace, size_t workspace_bytes, cudaStream_t stream);
size_t select_q8_workspace_bytes(uint32_t rows, uint32_t keys, uint32_t kv_heads, uint32_t block, uint32_t count);
int select_q8(const void *q, const RowsQ8Dev &kv, uint32_t *ids, const uint32_t *slots, const uint32_t *positions, uint32_t rows,
              uint32_t keys, uint32_t heads, uint32_t kv_heads, uint32_t width, uint32_t count, uint32_t first,
              uint32_t recent, void *workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace ts
