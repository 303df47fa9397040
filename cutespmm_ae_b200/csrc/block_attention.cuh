// What the kernels that walk queries share: a tile of neighbouring queries, the union of the blocks they name, and the ring that
// brings the keys and values of those blocks into shared memory once for all of them.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "pattern_ops.hpp"
#include "ptx.cuh"
#include "tc16.cuh"

namespace cutespmm {

constexpr uint32_t kTileQueries = 32;  // at most: a bit of a word each
constexpr float kLog2e = 1.4426950408889634f;

// How many keys query t of sequence b sees.
__device__ __forceinline__ uint32_t visible_keys(const AttentionArgs &a, uint32_t b, uint32_t t)
{
    const int64_t see = a.visible ? (int64_t)a.visible[(uint64_t)b * a.queries + t] : (int64_t)a.keys - a.queries + 1 + t;
    return (uint32_t)min(max(see, (int64_t)0), (int64_t)a.keys);
}
// Whether block j holds keys that a query seeing `visible` keys may look at (a page that does not exist holds none).
__device__ __forceinline__ bool block_counts(const AttentionArgs &a, uint32_t b, int32_t j, uint32_t visible)
{
    if (j < 0 || (uint32_t)j >= a.num_blocks || (uint64_t)j * a.block >= visible) return false;
    if (!a.pages) return true;
    const int32_t page = a.pages[(uint64_t)b * a.page_cols + j];
    return page >= 0 && (uint32_t)page < a.num_pages;
}

// The union of the blocks that `queries` queries from t0 on name, ascending, each with a bit per query that names it.
struct BlockUnion {
    uint32_t *blocks, *names;  // up to kTileQueries * count
    uint32_t *visible;         // per query of the tile
    uint32_t *bits, *before;   // a bit per block of the sequence, and the blocks in front of each word
    uint32_t *size;

    static __host__ __device__ uint32_t words(uint32_t num_blocks) { return (num_blocks + 31) / 32; }
    static __host__ __device__ uint32_t slots(uint32_t queries, uint32_t count, uint32_t num_blocks)
    {
        const uint32_t n = queries * count;
        return n < num_blocks ? n : num_blocks;
    }
    static __host__ __device__ uint32_t bytes(uint32_t queries, uint32_t count, uint32_t num_blocks)
    {
        return (2 * slots(queries, count, num_blocks) + kTileQueries + 2 * words(num_blocks) + 4) * 4;
    }
    __device__ BlockUnion(unsigned char *p, uint32_t queries, uint32_t count, uint32_t num_blocks)
    {
        uint32_t *w = reinterpret_cast<uint32_t *>(p);
        size = w;
        visible = w + 4;
        bits = visible + kTileQueries;
        before = bits + words(num_blocks);
        blocks = before + words(num_blocks);
        names = blocks + slots(queries, count, num_blocks);
    }
    // every thread of the block; ends with a barrier
    __device__ void build(const AttentionArgs &a, uint32_t b, uint32_t kv, uint32_t t0, uint32_t queries)
    {
        const uint32_t w = words(a.num_blocks), n = queries * a.count;
        const int32_t *src = a.blocks + (((uint64_t)b * a.kv_heads + kv) * a.queries + t0) * a.count;
        for (uint32_t i = threadIdx.x; i < w; i += blockDim.x) bits[i] = 0;
        for (uint32_t i = threadIdx.x; i < queries; i += blockDim.x) visible[i] = visible_keys(a, b, t0 + i);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
            const int32_t j = src[i];
            if (block_counts(a, b, j, visible[i / a.count])) atomicOr(&bits[j >> 5], 1u << (j & 31));
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            uint32_t sum = 0;
            for (uint32_t i = 0; i < w; i += 32) {
                const uint32_t mine = i + threadIdx.x < w ? __popc(bits[i + threadIdx.x]) : 0u;
                uint32_t scan = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t up = __shfl_up_sync(~0u, scan, d);
                    if (threadIdx.x >= (uint32_t)d) scan += up;
                }
                if (i + threadIdx.x < w) before[i + threadIdx.x] = sum + scan - mine;
                sum += __shfl_sync(~0u, scan, 31);
            }
            if (threadIdx.x == 0) *size = sum;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < *size; i += blockDim.x) names[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
            const int32_t j = src[i];
            if (!block_counts(a, b, j, visible[i / a.count])) continue;
            const uint32_t at = before[j >> 5] + __popc(bits[j >> 5] & ((1u << (j & 31)) - 1u));
            blocks[at] = (uint32_t)j;
            atomicOr(&names[at], 1u << (i / a.count));
        }
        __syncthreads();
    }
};

// Where unit `sub` (of `unit` keys) of block j of sequence b lies: coordinates of the tensor maps over k and v.
__device__ __forceinline__ void unit_place(const AttentionArgs &a, uint32_t b, uint32_t j, uint32_t first, int &row, int &outer)
{
    if (a.pages) {
        row = (int)first;
        outer = a.pages[(uint64_t)b * a.page_cols + j];
    } else {
        row = (int)(j * a.block + first);
        outer = (int)b;
    }
}

// Columns: the products are formed transposed, keys (then dims) as rows and (query, head) pairs as columns, eight columns to a
// tensor-core tile.  The heads of a group take `stride` columns: 1, 2, 4 or a multiple of 8.
__host__ __device__ inline uint32_t column_stride(uint32_t heads) { return heads <= 1 ? 1 : heads <= 2 ? 2 : heads <= 4 ? 4 : (heads + 7) / 8 * 8; }
constexpr uint32_t kHeadChunk = 64;  // query heads of a group that one block of threads takes

// masks the 16-bit pair of keys k, k + 1 in a register: only keys below `limit` stay
__device__ __forceinline__ uint32_t keep_keys(uint32_t pair, int k, int limit)
{
    return pair & ((k < limit ? 0xffffu : 0u) | (k + 1 < limit ? 0xffff0000u : 0u));
}

}  // namespace cutespmm
