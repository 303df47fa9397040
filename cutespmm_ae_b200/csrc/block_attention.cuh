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

constexpr uint32_t kTileQueries = 128;  // at most: a row each
constexpr uint32_t kHeadChunk = 64;     // query heads of a group that one block of threads takes, at most
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

// Where the keys from the `first`-th of block j of sequence b on lie: coordinates of the tensor maps over k and v.
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

// ---- tiles of 64 keys ----------------------------------------------------------------------------------------------------
// The tcgen05 kernels walk keys 64 at a time whatever the blocks are: a block of 128 is two tiles, four blocks of 16 are one.
constexpr uint32_t kKeyTile = 64;
__host__ __device__ inline uint32_t parts_of_tile(uint32_t block) { return block < kKeyTile ? kKeyTile / block : 1; }
__host__ __device__ inline uint32_t tiles_of_block(uint32_t block) { return block > kKeyTile ? block / kKeyTile : 1; }

// The union of the tiles of keys that hold a block which some of `queries` queries from t0 on name, ascending; for each part (block) of
// each tile a bit per query that names it.
struct TileUnion {
    uint32_t *tiles, *names;  // names: (slot * parts + part) * sets + query / 32
    uint32_t *visible, *bits, *before, *size;
    uint32_t parts, sets;     // sets of 32 queries

    static __host__ __device__ uint32_t words(uint32_t keys) { return (keys + kKeyTile * 32 - 1) / (kKeyTile * 32); }
    static __host__ __device__ uint32_t slots(uint32_t queries, uint32_t count, uint32_t block, uint32_t keys)
    {
        const uint32_t n = queries * count * tiles_of_block(block), all = (keys + kKeyTile - 1) / kKeyTile;
        return n < all ? n : all;
    }
    static __host__ __device__ uint32_t bytes(uint32_t queries, uint32_t count, uint32_t block, uint32_t keys)
    {
        return (slots(queries, count, block, keys) * (1 + parts_of_tile(block) * ((queries + 31) / 32)) + queries + 2 * words(keys) + 4) * 4;
    }
    __device__ TileUnion(unsigned char *p, uint32_t queries, const AttentionArgs &a)
    {
        uint32_t *w = reinterpret_cast<uint32_t *>(p);
        parts = parts_of_tile(a.block);
        sets = (queries + 31) / 32;
        size = w;
        visible = w + 4;
        bits = visible + queries;
        before = bits + words(a.keys);
        tiles = before + words(a.keys);
        names = tiles + slots(queries, a.count, a.block, a.keys);
    }
    // every thread of the block; ends with a barrier.  size[1]: the most keys that one of the queries sees
    __device__ void build(const AttentionArgs &a, uint32_t b, uint32_t kv, uint32_t t0, uint32_t queries)
    {
        const uint32_t w = words(a.keys), n = queries * a.count, per = tiles_of_block(a.block);
        const int32_t *src = a.blocks + (((uint64_t)b * a.kv_heads + kv) * a.queries + t0) * a.count;
        const uint32_t most_names = slots(queries, a.count, a.block, a.keys) * parts * sets;
        for (uint32_t i = threadIdx.x; i < w; i += blockDim.x) bits[i] = 0;
        for (uint32_t i = threadIdx.x; i < most_names; i += blockDim.x) names[i] = 0;
        for (uint32_t i = threadIdx.x; i < queries; i += blockDim.x) visible[i] = visible_keys(a, b, t0 + i);
        auto each = [&](uint32_t i, int32_t j, uint32_t see, auto &&fn) {  // fn(tile, part, query) for what entry i names and its query sees a part of
            if (!block_counts(a, b, j, see)) return;
            const uint64_t first = (uint64_t)j * a.block;
            for (uint32_t x = 0; x < per; ++x)
                if (first + x * kKeyTile < see) fn((uint32_t)(first / kKeyTile) + x, (uint32_t)(first % kKeyTile) / a.block, i / a.count);
        };
        const int32_t mine = threadIdx.x < n ? src[threadIdx.x] : -1;  // on its way during the barrier
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
            each(i, i == threadIdx.x ? mine : src[i], visible[i / a.count], [&](uint32_t tile, uint32_t, uint32_t) { atomicOr(&bits[tile >> 5], 1u << (tile & 31)); });
        __syncthreads();
        if (threadIdx.x < 32) {
            uint32_t sum = 0, most = 0;
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
            for (uint32_t i = threadIdx.x; i < queries; i += 32) most = max(most, visible[i]);
            most = __reduce_max_sync(~0u, most);
            if (threadIdx.x == 0) {
                size[0] = sum;
                size[1] = most;
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
            each(i, i == threadIdx.x ? mine : src[i], visible[i / a.count], [&](uint32_t tile, uint32_t part, uint32_t q) {
                const uint32_t at = before[tile >> 5] + __popc(bits[tile >> 5] & ((1u << (tile & 31)) - 1u));
                tiles[at] = tile;
                atomicOr(&names[(at * parts + part) * sets + (q >> 5)], 1u << (q & 31));
            });
        __syncthreads();
    }
    // the keys of a tile that query q looks at, a bit each
    __device__ uint64_t seen(uint32_t slot, uint32_t q, uint32_t block) const
    {
        const int64_t limit = (int64_t)visible[q] - (int64_t)tiles[slot] * kKeyTile;
        const uint64_t below = limit >= 64 ? ~0ull : limit > 0 ? (1ull << limit) - 1ull : 0ull;
        const uint32_t *word = names + slot * parts * sets + (q >> 5), bit = 1u << (q & 31);
        if (parts == 1) return *word & bit ? below : 0ull;
        uint64_t named = 0;
        for (uint32_t i = 0; i < parts; ++i)
            if (word[i * sets] & bit) named |= ((1ull << block) - 1ull) << (i * block);
        return named & below;
    }
};

// What a thread block of the tcgen05 kernels that walk queries takes: 128 rows, (query, head of the group) pairs.
struct TcShape {
    uint32_t heads, queries, chunks, box_rows;  // rows of a query, queries of a tile, chunks of a group's heads, rows of a box of k and v
};
inline TcShape tc_shape(uint32_t group, uint32_t box_rows)
{
    TcShape s;
    s.heads = group < kHeadChunk ? group : kHeadChunk;
    s.queries = 128 / s.heads < kTileQueries ? 128 / s.heads : kTileQueries;
    s.chunks = (group + s.heads - 1) / s.heads;
    s.box_rows = box_rows;
    return s;
}
constexpr uint32_t kSmemMost = 227 * 1024;
constexpr uint32_t kTcPolls = 1u << 24;  // of a role that looks at two barriers in turn, before it gives up

// One warp brings the keys (or values) of a tile into shared memory: DP / 64 tiles of 64 rows x 128 bytes, swizzled.  Rows that none of the
// queries sees become zeros: whatever a cache holds behind the last key, 0 times it has to be 0.  box_rows: rows of a box of the map (64,
// or the size of a page).  Returns false when a wait gave up.
template <int DP>
__device__ __forceinline__ bool load_key_tile(unsigned char *to, const CUtensorMap *map, const AttentionArgs &a, uint32_t b, uint32_t kv, uint32_t tile, uint32_t visible, uint32_t box_rows,
                                              uint64_t *full, uint64_t *landed, uint32_t &landed_phase)
{
    const uint32_t lane = threadIdx.x & 31, first = tile * kKeyTile;
    const bool cut = first + kKeyTile > visible;
    uint64_t *bar = cut ? landed : full;
    if (lane == 0) {
        ptx::mbar_expect_tx(bar, DP / 64 * kKeyTile * 128);
        for (uint32_t r = 0; r < kKeyTile; r += box_rows) {
            int row = (int)(first + r), outer = (int)b;
            if (a.pages) {
                const uint32_t j = (first + r) / a.block;
                row = (int)((first + r) % a.block);
                outer = j < a.page_cols ? a.pages[(uint64_t)b * a.page_cols + j] : -1;  // what is no page arrives as zeros
            }
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) tc::tma_load4(to + h * kKeyTile * 128 + r * 128, map, h * 64, (int)kv, row, outer, bar);
        }
    }
    __syncwarp();
    if (!cut) return true;
    const bool ok = ptx::mbar_wait_warp(landed, landed_phase);
    landed_phase ^= 1u;
    constexpr uint32_t kPieces = DP / 8;  // 16-byte pieces of a row
    unsigned char *at = to + lane % kPieces / 8 * kKeyTile * 128 + lane % 8 * 16;
    for (uint32_t row = (visible > first ? visible - first : 0u) + lane / kPieces; row < kKeyTile; row += 32 / kPieces) *reinterpret_cast<uint4 *>(at + row * 128) = make_uint4(0, 0, 0, 0);
    ptx::fence_async_smem();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(full);
    return ok;
}

template <class T> __device__ __forceinline__ const T *key_row(const AttentionArgs &a, const void *base, int64_t s_batch, int64_t s_key, int64_t s_head, uint32_t b, uint32_t kv, uint32_t key)
{
    const T *p = static_cast<const T *>(base) + (int64_t)kv * s_head;
    if (!a.pages) return p + (int64_t)b * s_batch + (int64_t)key * s_key;
    return p + (int64_t)a.pages[(uint64_t)b * a.page_cols + key / a.block] * s_batch + (int64_t)(key % a.block) * s_key;
}

// masks the 16-bit pair of keys k, k + 1 in a register: only keys below `limit` stay
__device__ __forceinline__ uint32_t keep_keys(uint32_t pair, int k, int limit)
{
    return pair & ((k < limit ? 0xffffu : 0u) | (k + 1 < limit ? 0xffff0000u : 0u));
}

}  // namespace cutespmm
