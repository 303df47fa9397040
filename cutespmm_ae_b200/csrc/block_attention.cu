// Attention over selected blocks, forward: out = softmax(scale q K^T) V over the visible keys of the blocks that each query names.
//
// Two kernels.  A tile of neighbouring queries shares the blocks that several of them name: block_attention_kernel.  A single token (or
// few) has its blocks split over the warps of up to eight thread blocks: block_attention_split_kernel.
//
// Both form the transposed products S^T = K Q^T and O^T = V^T P^T, so that keys and dims are the 16 rows of a tensor-core
// instruction and (query, head) pairs its eight columns: with eight heads to a group a column tile is one query, and a query that does
// not name a block costs nothing there.  (A tcgen05 tile of 128 rows would multiply every query of the tile with every block of the union.)
// Softmax with a running maximum and sum per column, in fp32; P is rounded to the 16-bit type for the second product, the sum is
// taken before that rounding.  A masked key never touches a result, whatever stands there: its score is replaced, and its value is cut out of the
// second product's operand (0 times infinity would not be 0).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "block_attention.cuh"
#include "device_plan.hpp"
#include "num.cuh"
#include "pattern_ops.hpp"
#include "ptx.cuh"
#include "tc16.cuh"

namespace cutespmm {
namespace {

__device__ uint32_t g_status;  // set to 1 when a bounded wait gives up

constexpr int kRingBytes = 128 * 1024;  // keys and values in flight per thread block of the tile kernel

// A unit of keys in shared memory: DP / 64 tiles of UNIT rows x 128 bytes (swizzled) of keys, then the same of values.
template <int DP, int UNIT> constexpr int kHalfBytes = DP / 64 * UNIT * 128;
template <int DP, int UNIT> constexpr int kUnitBytes = 2 * kHalfBytes<DP, UNIT>;
template <int DP, int UNIT> constexpr int kRing = kRingBytes / kUnitBytes<DP, UNIT> < 8 ? kRingBytes / kUnitBytes<DP, UNIT> : 8;

template <int DP, int UNIT>
__device__ __forceinline__ void load_unit(unsigned char *stage, const CUtensorMap *k_map, const CUtensorMap *v_map, int kv, int row, int outer, uint64_t *bar)
{
    ptx::mbar_expect_tx(bar, kUnitBytes<DP, UNIT>);
#pragma unroll
    for (int h = 0; h < DP / 64; ++h) tc::tma_load4(stage + h * UNIT * 128, k_map, h * 64, kv, row, outer, bar);
#pragma unroll
    for (int h = 0; h < DP / 64; ++h) tc::tma_load4(stage + kHalfBytes<DP, UNIT> + h * UNIT * 128, v_map, h * 64, kv, row, outer, bar);
}

// Softmax state and accumulator of one tile of eight columns in the registers of a warp.  A lane holds columns 2 (lane % 4) and
// the next one; of each 16 x 8 tile rows lane / 4 and lane / 4 + 8.
template <class T, int DP> struct ColumnTile {
    uint32_t q[DP / 16][2];   // operand B of the first product
    float o[DP / 16][4];      // O^T
    float top[2], sum[2];     // running maximum (times scale and log2 e) and this lane's share of the running sum

    // `row`: the query-head row of q that column lane / 4 holds, or nullptr
    __device__ void start(const T *row, uint32_t dim, uint32_t lane)
    {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t d = s * 16 + h * 8 + 2 * (lane & 3);
                q[s][h] = row && d < dim ? *reinterpret_cast<const uint32_t *>(row + d) : 0u;
            }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[s][j] = 0.f;
        top[0] = top[1] = -INFINITY;
        sum[0] = sum[1] = 0.f;
    }
    // scores of a unit -> P^T as operand B of the second product
    template <int KT> __device__ void softmax(float (&s)[KT][4], uint32_t (&p)[KT][2], float scale_log2)
    {
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            m0 = fmaxf(m0, fmaxf(s[k][0], s[k][2]));
            m1 = fmaxf(m1, fmaxf(s[k][1], s[k][3]));
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(~0u, m0, x));
            m1 = fmaxf(m1, __shfl_xor_sync(~0u, m1, x));
        }
        m0 = fmaxf(top[0], m0 * scale_log2);
        m1 = fmaxf(top[1], m1 * scale_log2);
        if (__any_sync(~0u, m0 > top[0] || m1 > top[1])) {
            const float f0 = top[0] == m0 ? 1.f : tc::exp2_fast(top[0] - m0), f1 = top[1] == m1 ? 1.f : tc::exp2_fast(top[1] - m1);
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                o[d][0] *= f0;
                o[d][1] *= f1;
                o[d][2] *= f0;
                o[d][3] *= f1;
            }
            sum[0] *= f0;
            sum[1] *= f1;
            top[0] = m0;
            top[1] = m1;
        }
        const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;  // nothing visible yet: every exponential is 0
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const float e0 = tc::exp2_fast(fmaf(s[k][0], scale_log2, -b0)), e1 = tc::exp2_fast(fmaf(s[k][1], scale_log2, -b1));
            const float e2 = tc::exp2_fast(fmaf(s[k][2], scale_log2, -b0)), e3 = tc::exp2_fast(fmaf(s[k][3], scale_log2, -b1));
            sum[0] += e0 + e2;
            sum[1] += e1 + e3;
            p[k][0] = tc::transpose8x8(tc::round2<T>(e0, e1));
            p[k][1] = tc::transpose8x8(tc::round2<T>(e2, e3));
        }
    }
    __device__ void finish_sum()
    {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            sum[0] += __shfl_xor_sync(~0u, sum[0], x);
            sum[1] += __shfl_xor_sync(~0u, sum[1], x);
        }
    }
};

// Operand A of the first product: rows 16 k of the keys, dims 16 s.
__device__ __forceinline__ uint32_t keys_at(uint32_t keys, int unit, int k, int s, uint32_t lane)
{
    return keys + (s >> 2) * unit * 128 + tc::swizzled(k * 16 + (lane & 15), (s & 3) * 2 + (lane >> 4));
}
// Operand A of the second product, transposed on the way: dims 16 d, keys 16 k.
__device__ __forceinline__ uint32_t values_at(uint32_t values, int unit, int k, int d, uint32_t lane)
{
    return values + (d >> 2) * unit * 128 + tc::swizzled(k * 16 + ((lane >> 4) << 3) + (lane & 7), (d & 3) * 2 + ((lane >> 3) & 1));
}

// ---- a tile of queries -------------------------------------------------------------------------------------------------
// WARPS warps of NT column tiles each, and one that loads.  The warps of a block take a unit when it has landed and leave it when they are
// done, without waiting for each other; a unit that none of a warp's queries names is passed over.
struct TileShape {
    uint32_t stride, queries, chunks;  // columns of a query's heads, queries of a thread block, chunks of a group's heads
};

template <class T, int DP, int UNIT, int WARPS, int NT>
__global__ void __launch_bounds__((WARPS + 1) * 32, 1) block_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, AttentionArgs a, TileShape shape)
{
    constexpr int KT = UNIT / 16, STAGES = kRing<DP, UNIT>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + STAGES * kUnitBytes<DP, UNIT>), *empty = full + STAGES;
    volatile uint32_t *gave_up = reinterpret_cast<volatile uint32_t *>(empty + STAGES);
    BlockUnion u(reinterpret_cast<unsigned char *>(empty + STAGES + 2), shape.queries, a.count, a.num_blocks);
    const uint32_t t0 = blockIdx.x * shape.queries, b = blockIdx.z;
    const uint32_t kv = blockIdx.y / shape.chunks, group = a.heads / a.kv_heads, head0 = blockIdx.y % shape.chunks * kHeadChunk;
    const uint32_t heads = min(kHeadChunk, group - head0), queries = min(shape.queries, a.queries - t0);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], WARPS);
        }
        *gave_up = 0;
        ptx::fence_mbar_init();
    }
    ptx::grid_wait();
    ptx::grid_release();
    u.build(a, b, kv, t0, queries);  // its barriers also cover the ones above
    const uint32_t per_block = a.block / UNIT, units = *u.size * per_block;

    if (warp == WARPS) {
        if (lane == 0) {
            uint32_t i = 0;
            for (; i < units && !*gave_up; ++i) {
                const uint32_t s = i % STAGES;
                if (!ptx::mbar_wait(&empty[s], ((i / STAGES) & 1u) ^ 1u)) {
                    *gave_up = 1;
                    break;
                }
                int row, outer;
                unit_place(a, b, u.blocks[i / per_block], i % per_block * UNIT, row, outer);
                load_unit<DP, UNIT>(smem + s * kUnitBytes<DP, UNIT>, &k_map, &v_map, (int)kv, row, outer, &full[s]);
            }
            if (*gave_up) {
                atomicExch(&g_status, 1u);
                for (uint32_t j = i > STAGES ? i - STAGES : 0; j < i; ++j) ptx::mbar_wait(&full[j % STAGES], (j / STAGES) & 1u);  // no copy stays in flight
            }
        }
        return;
    }

    ColumnTile<T, DP> tile[NT];
    uint32_t asks[NT];          // the queries of a column tile, a bit each
    uint32_t query[NT][2];      // of this lane's two columns (32: none)
    int sees[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t c0 = (warp * NT + i) * 8;
        const uint32_t c = c0 + lane / 4, ct = c / shape.stride, ch = c % shape.stride;
        const T *row = nullptr;
        if (ct < queries && ch < heads)
            row = static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)(t0 + ct) * a.q_query + (int64_t)(kv * group + head0 + ch) * a.q_head;
        tile[i].start(row, a.dim, lane);
        asks[i] = 0;
        for (uint32_t j = c0 / shape.stride; j <= (c0 + 7) / shape.stride; ++j)
            if (j < queries && c0 - min(c0, j * shape.stride) < heads) asks[i] |= 1u << j;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t col = c0 + 2 * (lane & 3) + h, t = col / shape.stride;
            const bool on = t < queries && col % shape.stride < heads;
            query[i][h] = on ? t : 32u;
            sees[i][h] = on ? (int)u.visible[t] : 0x7fffffff;
        }
    }
    const float scale_log2 = a.scale * kLog2e;

    for (uint32_t n = 0; n < units; ++n) {
        const uint32_t s = n % STAGES, slot = n / per_block, names = u.names[slot];
        const int first = (int)(u.blocks[slot] * a.block + n % per_block * UNIT);
        if (!ptx::mbar_wait(&full[s], (n / STAGES) & 1u)) {
            *gave_up = 1;
            if (lane == 0) atomicExch(&g_status, 1u);
            return;
        }
        bool on[NT], any = false;
#pragma unroll
        for (int i = 0; i < NT; ++i) any |= on[i] = (names & asks[i]) != 0;
        if (any) {
            const uint32_t keys = ptx::smem_u32(smem + s * kUnitBytes<DP, UNIT>), values = keys + kHalfBytes<DP, UNIT>;
            float sc[NT][KT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[i][k][j] = 0.f;
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t f[4];
                    tc::ldmatrix4(f, keys_at(keys, UNIT, k, d, lane));
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        if (on[i]) tc::mma16<T>(sc[i][k], f, tile[i].q[d][0], tile[i].q[d][1]);
                }
            uint32_t p[NT][KT][2];
            bool whole[NT], slow = false;
            int limit[NT][2];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                whole[i] = true;
                if (!on[i]) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) limit[i][h] = query[i][h] == 32u ? UNIT : (names >> query[i][h]) & 1u ? sees[i][h] - first : 0;
                whole[i] = __all_sync(~0u, limit[i][0] >= UNIT && limit[i][1] >= UNIT);
                if (!whole[i]) {
                    slow = true;
                    const int r = (int)(lane >> 2);
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        if (k * 16 + r >= limit[i][0]) sc[i][k][0] = -INFINITY;
                        if (k * 16 + r >= limit[i][1]) sc[i][k][1] = -INFINITY;
                        if (k * 16 + r + 8 >= limit[i][0]) sc[i][k][2] = -INFINITY;
                        if (k * 16 + r + 8 >= limit[i][1]) sc[i][k][3] = -INFINITY;
                    }
                }
                tile[i].softmax(sc[i], p[i], scale_log2);
            }
            if (!slow) {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        uint32_t f[4];
                        tc::ldmatrix4_trans(f, values_at(values, UNIT, k, d, lane));
#pragma unroll
                        for (int i = 0; i < NT; ++i)
                            if (on[i]) tc::mma16<T>(tile[i].o[d], f, p[i][k][0], p[i][k][1]);
                    }
            } else {
                // Queries of one column tile that see different parts of the unit: a pass for those that see all of it, one for each
                // other; a pass changes its own columns only.
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (!on[i]) continue;
                    uint32_t left = names & asks[i];
                    bool all = true;  // first the pass over whole units
                    while (left) {
                        int cut = UNIT;
                        uint32_t taken = 0;
                        if (all) {
                            for (uint32_t m = left; m; m &= m - 1) {
                                const uint32_t t = __ffs(m) - 1;
                                if ((int)u.visible[t] - first >= UNIT) taken |= 1u << t;
                            }
                            all = false;
                        } else {
                            const uint32_t t = __ffs(left) - 1;
                            taken = 1u << t;
                            cut = (int)u.visible[t] - first;
                        }
                        left &= ~taken;
                        if (!taken || cut <= 0) continue;
                        const bool mine0 = (taken >> query[i][0]) & (query[i][0] < 32u), mine1 = (taken >> query[i][1]) & (query[i][1] < 32u);
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) {
                            float o[4] = {tile[i].o[d][0], tile[i].o[d][1], tile[i].o[d][2], tile[i].o[d][3]};
#pragma unroll
                            for (int k = 0; k < KT; ++k) {
                                uint32_t f[4];
                                tc::ldmatrix4_trans(f, values_at(values, UNIT, k, d, lane));
                                if (cut < UNIT) {
                                    const int at = k * 16 + 2 * (int)(lane & 3);
                                    f[0] = keep_keys(f[0], at, cut);
                                    f[1] = keep_keys(f[1], at, cut);
                                    f[2] = keep_keys(f[2], at + 8, cut);
                                    f[3] = keep_keys(f[3], at + 8, cut);
                                }
                                tc::mma16<T>(o, f, p[i][k][0], p[i][k][1]);
                            }
                            if (mine0) {
                                tile[i].o[d][0] = o[0];
                                tile[i].o[d][2] = o[2];
                            }
                            if (mine1) {
                                tile[i].o[d][1] = o[1];
                                tile[i].o[d][3] = o[3];
                            }
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&empty[s]);
    }

#pragma unroll
    for (int i = 0; i < NT; ++i) {
        tile[i].finish_sum();
        const float f0 = tile[i].sum[0] > 0.f ? 1.f / tile[i].sum[0] : 0.f, f1 = tile[i].sum[1] > 0.f ? 1.f / tile[i].sum[1] : 0.f;
        const uint32_t c = (warp * NT + i) * 8 + lane / 4, t = c / shape.stride, h = c % shape.stride;
        const bool row_on = t < queries && h < heads;
        T *row = static_cast<T *>(a.out) + (((uint64_t)b * a.queries + t0 + t) * a.heads + kv * group + head0 + h) * a.dim;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            const uint32_t lo = tc::transpose8x8(tc::round2<T>(tile[i].o[d][0] * f0, tile[i].o[d][1] * f1));
            const uint32_t hi = tc::transpose8x8(tc::round2<T>(tile[i].o[d][2] * f0, tile[i].o[d][3] * f1));
            const uint32_t at = d * 16 + 2 * (lane & 3);
            if (row_on && at < a.dim) *reinterpret_cast<uint32_t *>(row + at) = lo;
            if (row_on && at + 8 < a.dim) *reinterpret_cast<uint32_t *>(row + at + 8) = hi;
        }
        if (lane < 4)
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                const uint32_t col = (warp * NT + i) * 8 + 2 * lane + h2, ct = col / shape.stride, ch = col % shape.stride;
                if (ct < queries && ch < heads)
                    a.lse[((uint64_t)b * a.heads + kv * group + head0 + ch) * a.queries + t0 + ct] =
                        tile[i].sum[h2] > 0.f ? (tile[i].top[h2] + log2f(tile[i].sum[h2])) * 0.6931471805599453f : -INFINITY;
            }
    }
}

// ---- a single token ----------------------------------------------------------------------------------------------------
// One query's heads of one head of keys: its blocks, in pieces of 16 keys, are dealt over the warps of a cluster of thread blocks.  A
// warp fills a ring of its own (its lane 0 issues the loads) and keeps its own softmax state; the states are joined in the
// order of the warps, first inside a thread block, then over the cluster through distributed shared memory: no scratch, no counters, one
// launch.  Bound: HBM (the named blocks once) in batches, a chain of latencies for one sequence.
constexpr int kSplitWarps = 4, kSplitUnit = 16;
template <int DP> constexpr int kSplitStages = DP == 128 ? 4 : 8;
constexpr uint32_t kSplitCount = 128;  // most blocks of a query

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 peer_load4(const float *p, uint32_t rank)
{
    float4 v;
    asm volatile(
        "{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\tld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [r];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(ptx::smem_u32(p)), "r"(rank)
        : "memory");
    return v;
}
__device__ __forceinline__ float peer_load(const float *p, uint32_t rank)
{
    float v;
    asm volatile("{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}" : "=f"(v) : "r"(ptx::smem_u32(p)), "r"(rank) : "memory");
    return v;
}

template <int DP, int NT> struct SplitSmem {
    static constexpr int kStage = kUnitBytes<DP, kSplitUnit>;
    static constexpr int kRings = kSplitWarps * kSplitStages<DP> * kStage;
    static constexpr int kPitch = DP + 4;                                      // floats of a column of a partial result
    static constexpr int kPartial = kRings;                                    // per warp 8 NT columns; the thread block's own join lies in warp 0's
    static constexpr int kStats = kPartial + kSplitWarps * 8 * NT * kPitch * 4;  // per warp and column: maximum, sum
    static constexpr int kBars = kStats + kSplitWarps * 8 * NT * 8;
    static constexpr int kList = kBars + kSplitWarps * kSplitStages<DP> * 8;
    static constexpr int kBytes = kList + kSplitCount * 8 + 16;
};

template <class T, int DP, int NT>
__global__ void __launch_bounds__(kSplitWarps * 32) block_attention_split_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, AttentionArgs a, uint32_t chunks)
{
    using S = SplitSmem<DP, NT>;
    constexpr int STAGES = kSplitStages<DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x, ranks = gridDim.x;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::kBars) + warp * STAGES;
    uint32_t *list = reinterpret_cast<uint32_t *>(smem + S::kList), *first_of = list + kSplitCount, *size = first_of + kSplitCount;
    const uint32_t t = blockIdx.z % a.queries, b = blockIdx.z / a.queries;
    const uint32_t kv = blockIdx.y / chunks, group = a.heads / a.kv_heads, head0 = blockIdx.y % chunks * (8 * NT), heads = min(8u * NT, group - head0);
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) ptx::mbar_init(&full[s], 1);
        ptx::fence_mbar_init();
    }
    ptx::grid_wait();
    ptx::grid_release();
    // the query's blocks, in its order, each once: thread i looks at entry i
    const uint32_t visible = visible_keys(a, b, t);
    const int32_t *src = a.blocks + (((uint64_t)b * a.kv_heads + kv) * a.queries + t) * a.count;
    const int32_t mine = threadIdx.x < a.count ? src[threadIdx.x] : -1;
    list[threadIdx.x] = (uint32_t)mine;
    static_assert(kSplitWarps * 32 == (int)kSplitCount, "a thread per entry");
    __syncthreads();
    bool counts = threadIdx.x < a.count && block_counts(a, b, mine, visible);
    if (counts)
        for (uint32_t i = 0; i < threadIdx.x; ++i) counts = counts && list[i] != (uint32_t)mine;
    const uint32_t votes = __ballot_sync(~0u, counts);
    if (lane == 0) first_of[warp] = votes;
    __syncthreads();
    uint32_t at = __popc(votes & ((1u << lane) - 1u)), total = 0;
    for (uint32_t w = 0; w < (uint32_t)kSplitWarps; ++w) {
        if (w < warp) at += __popc(first_of[w]);
        total += __popc(first_of[w]);
    }
    __syncthreads();
    if (counts) list[at] = (uint32_t)mine;
    (void)size;
    __syncthreads();

    const uint32_t per_block = a.block / kSplitUnit, units = total * per_block;
    const uint32_t walkers = ranks * kSplitWarps, me = warp * ranks + rank;  // neighbouring units go to different thread blocks
    const uint32_t mine_units = units > me ? (units - me + walkers - 1) / walkers : 0u;
    unsigned char *ring = smem + warp * STAGES * S::kStage;
    auto issue = [&](uint32_t i) {
        const uint32_t n = me + i * walkers;
        int row, outer;
        unit_place(a, b, list[n / per_block], n % per_block * kSplitUnit, row, outer);
        load_unit<DP, kSplitUnit>(ring + i % STAGES * S::kStage, &k_map, &v_map, (int)kv, row, outer, &full[i % STAGES]);
    };
    if (lane == 0)
        for (uint32_t i = 0; i < mine_units && i < (uint32_t)STAGES; ++i) issue(i);

    ColumnTile<T, DP> tile[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t h = i * 8 + lane / 4;
        tile[i].start(h < heads ? static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)t * a.q_query + (int64_t)(kv * group + head0 + h) * a.q_head : nullptr, a.dim, lane);
    }
    const float scale_log2 = a.scale * kLog2e;
    for (uint32_t i = 0; i < mine_units; ++i) {
        const uint32_t n = me + i * walkers, s = i % STAGES;
        if (!ptx::mbar_wait(&full[s], (i / STAGES) & 1u)) {  // later loads of this ring land before the block ends, or their waits give up too
            if (lane == 0) atomicExch(&g_status, 1u);
            continue;
        }
        const int limit = (int)visible - (int)(list[n / per_block] * a.block + n % per_block * kSplitUnit);
        if (limit > 0) {
            const uint32_t keys = ptx::smem_u32(ring + s * S::kStage), values = keys + kHalfBytes<DP, kSplitUnit>;
            float sc[NT][1][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) sc[j][0][0] = sc[j][0][1] = sc[j][0][2] = sc[j][0][3] = 0.f;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t f[4];
                tc::ldmatrix4(f, keys_at(keys, kSplitUnit, 0, d, lane));
#pragma unroll
                for (int j = 0; j < NT; ++j) tc::mma16<T>(sc[j][0], f, tile[j].q[d][0], tile[j].q[d][1]);
            }
            uint32_t p[NT][1][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if ((int)(lane >> 2) >= limit) sc[j][0][0] = sc[j][0][1] = -INFINITY;
                if ((int)(lane >> 2) + 8 >= limit) sc[j][0][2] = sc[j][0][3] = -INFINITY;
                tile[j].softmax(sc[j], p[j], scale_log2);
            }
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t f[4];
                tc::ldmatrix4_trans(f, values_at(values, kSplitUnit, 0, d, lane));
                if (limit < kSplitUnit) {
                    const int k = 2 * (int)(lane & 3);
                    f[0] = keep_keys(f[0], k, limit);
                    f[1] = keep_keys(f[1], k, limit);
                    f[2] = keep_keys(f[2], k + 8, limit);
                    f[3] = keep_keys(f[3], k + 8, limit);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) tc::mma16<T>(tile[j].o[d], f, p[j][0][0], p[j][0][1]);
            }
        }
        __syncwarp();
        if (lane == 0 && i + STAGES < mine_units) issue(i + STAGES);
    }

    // this warp's columns: maximum, sum and O, not divided
    float *partial = reinterpret_cast<float *>(smem + S::kPartial), *stats = reinterpret_cast<float *>(smem + S::kStats);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        tile[j].finish_sum();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t col = j * 8 + 2 * (lane & 3) + h;
            if (lane < 4) {
                stats[(warp * 8 * NT + col) * 2] = tile[j].top[h];
                stats[(warp * 8 * NT + col) * 2 + 1] = tile[j].sum[h];
            }
            float *o = partial + (warp * 8 * NT + col) * S::kPitch + lane / 4;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                o[d * 16] = tile[j].o[d][h];
                o[d * 16 + 8] = tile[j].o[d][h + 2];
            }
        }
    }
    // join over the warps and thread blocks: four dims of a column at a time, dealt over the threads of the cluster
    if (ranks > 1) cluster_sync(); else __syncthreads();
    constexpr uint32_t kParts = DP / 4;
    for (uint32_t i = rank * blockDim.x + threadIdx.x; i < heads * kParts; i += ranks * blockDim.x) {
        const uint32_t col = i / kParts, d = i % kParts * 4;
        float top = -INFINITY;
        for (uint32_t r = 0; r < ranks; ++r)
            for (uint32_t w = 0; w < (uint32_t)kSplitWarps; ++w) top = fmaxf(top, peer_load(stats + (w * 8 * NT + col) * 2, r));
        const float base = top == -INFINITY ? 0.f : top;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
        for (uint32_t r = 0; r < ranks; ++r)
            for (uint32_t w = 0; w < (uint32_t)kSplitWarps; ++w) {
                const uint32_t c = w * 8 * NT + col;
                const float f = tc::exp2_fast(peer_load(stats + c * 2, r) - base);
                const float4 x = peer_load4(partial + c * S::kPitch + d, r);
                sum = fmaf(f, peer_load(stats + c * 2 + 1, r), sum);
                o.x = fmaf(f, x.x, o.x);
                o.y = fmaf(f, x.y, o.y);
                o.z = fmaf(f, x.z, o.z);
                o.w = fmaf(f, x.w, o.w);
            }
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        const uint32_t head = kv * group + head0 + col;
        if (d < a.dim) {
            uint2 v;
            v.x = tc::round2<T>(o.x * inv, o.y * inv);
            v.y = tc::round2<T>(o.z * inv, o.w * inv);
            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + (((uint64_t)b * a.queries + t) * a.heads + head) * a.dim + d) = v;
        }
        if (d == 0) a.lse[((uint64_t)b * a.heads + head) * a.queries + t] = sum > 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
    if (ranks > 1) cluster_sync();  // a peer may still be reading this block's shared memory
}

template <class T, int DP, int NT> cudaError_t launch_split(const CUtensorMap &k_map, const CUtensorMap &v_map, const AttentionArgs &a, int sm_count, cudaStream_t s)
{
    using S = SplitSmem<DP, NT>;
    cudaError_t e = allow_dynamic_smem<block_attention_split_kernel<T, DP, NT>>(S::kBytes);
    if (e != cudaSuccess) return e;
    const uint32_t group = a.heads / a.kv_heads, chunks = (group + 8 * NT - 1) / (8 * NT);
    const uint64_t rows = (uint64_t)a.batch * a.queries * a.kv_heads * chunks, units = (uint64_t)a.count * (a.block / kSplitUnit);
    // thread blocks per query: as many as keep the machine busy, while each warp has two pieces of 16 keys
    uint32_t ranks = 1;
    while (ranks < 8 && rows * ranks < (uint64_t)sm_count && units >= 4ull * ranks * kSplitWarps) ranks *= 2;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ranks, a.kv_heads * chunks, a.batch * a.queries);
    cfg.blockDim = dim3(kSplitWarps * 32);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, block_attention_split_kernel<T, DP, NT>, k_map, v_map, a, chunks);
}

template <class T, int DP, int UNIT, int WARPS, int NT>
cudaError_t launch_tile(const CUtensorMap &k_map, const CUtensorMap &v_map, const AttentionArgs &a, cudaStream_t s)
{
    const uint32_t group = a.heads / a.kv_heads, heads = group < kHeadChunk ? group : kHeadChunk;
    TileShape shape;
    shape.stride = column_stride(heads);
    shape.queries = WARPS * NT * 8 / shape.stride;
    if (shape.queries > kTileQueries) shape.queries = kTileQueries;
    shape.chunks = (group + kHeadChunk - 1) / kHeadChunk;
    constexpr int kFixed = kRing<DP, UNIT> * (kUnitBytes<DP, UNIT> + 16) + 16;
    const uint32_t bytes = kFixed + BlockUnion::bytes(shape.queries, a.count, a.num_blocks);
    cudaError_t e = allow_dynamic_smem<block_attention_kernel<T, DP, UNIT, WARPS, NT>>(227 * 1024);
    if (e != cudaSuccess) return e;
    const dim3 grid((a.queries + shape.queries - 1) / shape.queries, a.kv_heads * shape.chunks, a.batch);
    return launch_overlapped(block_attention_kernel<T, DP, UNIT, WARPS, NT>, grid, dim3((WARPS + 1) * 32), bytes, s, k_map, v_map, a, shape);
}

template <class T, int DP> cudaError_t launch_d(const CUtensorMap &k_map, const CUtensorMap &v_map, const AttentionArgs &a, bool split, int sm_count, cudaStream_t s)
{
    const uint32_t group = a.heads / a.kv_heads;
    if (split) return group <= 8 ? launch_split<T, DP, 1>(k_map, v_map, a, sm_count, s) : launch_split<T, DP, 2>(k_map, v_map, a, sm_count, s);
    auto unit = [&](auto u) {
        constexpr int U = decltype(u)::value;
        // a tile has at most 32 queries: groups of one or two heads fill fewer columns
        if (group == 1) return launch_tile<T, DP, U, 4, 1>(k_map, v_map, a, s);
        if (group == 2) return launch_tile<T, DP, U, 4, 2>(k_map, v_map, a, s);
        return launch_tile<T, DP, U, 8, 2>(k_map, v_map, a, s);
    };
    if (a.block == 16) return unit(std::integral_constant<int, 16>());
    if (a.block == 32) return unit(std::integral_constant<int, 32>());
    return unit(std::integral_constant<int, 64>());
}

}  // namespace

cudaError_t launch_block_attention(const AttentionArgs &a, int sm_count, cudaStream_t s)
{
    if (!a.batch || !a.queries || !a.heads || !a.dim) return cudaSuccess;
    const bool bf16 = a.dtype == CUTESPMM_BF16;
    // few queries: a thread block per query and head of keys, its blocks split over warps
    const bool split = a.queries <= 4;
    const uint32_t rows = a.pages ? a.block : a.keys, outer = a.pages ? a.num_pages : a.batch;
    const uint32_t box = split ? (uint32_t)kSplitUnit : a.block < 64 ? a.block : 64;
    CUtensorMap k_map{}, v_map{};
    if (rows && outer) {  // without keys no block counts and nothing is loaded
        cudaError_t e = tc::make_map(&k_map, bf16, a.k, a.dim, a.kv_heads, rows, outer, a.k_head, a.k_key, a.k_batch, box);
        if (e == cudaSuccess) e = tc::make_map(&v_map, bf16, a.v, a.dim, a.kv_heads, rows, outer, a.v_head, a.v_key, a.v_batch, box);
        if (e != cudaSuccess) return e;
    }
    if (bf16)
        return a.dim <= 64 ? launch_d<__nv_bfloat16, 64>(k_map, v_map, a, split, sm_count, s) : launch_d<__nv_bfloat16, 128>(k_map, v_map, a, split, sm_count, s);
    return a.dim <= 64 ? launch_d<__half, 64>(k_map, v_map, a, split, sm_count, s) : launch_d<__half, 128>(k_map, v_map, a, split, sm_count, s);
}

cudaError_t block_attention_status(uint32_t *word) { return read_status(g_status, word); }

}  // namespace cutespmm
