// Which blocks of keys a query attends to: the mean key of every block, the score of every query against every mean, and per query
// the blocks of the highest scores.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "device_plan.hpp"
#include "num.cuh"
#include "pattern_ops.hpp"
#include "ptx.cuh"
#include "tc16.cuh"
#include "tmap.hpp"

namespace cutespmm {
namespace {

__device__ uint32_t g_status;  // set to 1 when a bounded wait of the score kernel gives up

// ---- means -------------------------------------------------------------------------------------------------------------
// A block of threads takes 32 groups of eight columns (of all heads side by side) of one block of keys: eight warps walk its rows,
// every load is 512 contiguous bytes where the heads are.  Sums in fp32, one rounding.  Bound: HBM (the keys once).
constexpr int kMeanWarps = 8;

template <class T> __global__ void __launch_bounds__(kMeanWarps * 32) block_means_kernel(MeansArgs a)
{
    __shared__ float part[kMeanWarps][32][9];
    ptx::grid_wait();
    ptx::grid_release();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, packs = a.dim / 8;
    const uint32_t col = blockIdx.y * 32 + lane, blk = blockIdx.x, b = blockIdx.z;
    const uint32_t head = col / packs, d = col % packs * 8;
    const bool on = head < a.kv_heads;
    const uint32_t keys = a.lengths ? (uint32_t)min(max(a.lengths[b], 0), (int)a.keys) : a.keys;
    const uint32_t first = blk * a.block, n = first < keys ? min(a.block, keys - first) : 0u;
    const T *src = static_cast<const T *>(a.k) + (int64_t)b * a.k_batch + (int64_t)head * a.k_head + d + (int64_t)first * a.k_key;
    float acc[8] = {};
#pragma unroll 4
    for (uint32_t r = warp; r < n; r += kMeanWarps)
        if (on) {
            const Pack<T, 8> p = load_pack<T, 8>(src + (int64_t)r * a.k_key);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += to_f32(p.x[j]);
        }
#pragma unroll
    for (int j = 0; j < 8; ++j) part[warp][lane][j] = acc[j];
    __syncthreads();
    // thread t adds column t of the 256 over the warps
    const uint32_t l = threadIdx.x >> 3, j = threadIdx.x & 7, out_col = blockIdx.y * 32 + l;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMeanWarps; ++w) sum += part[w][l][j];
    if (out_col < a.kv_heads * packs)
        static_cast<T *>(a.means)[((uint64_t)b * a.blocks + blk) * a.kv_heads * a.dim + (uint64_t)out_col * 8 + j] = from_f32<T>(n ? sum / (float)n : 0.f);
}

// ---- scores ------------------------------------------------------------------------------------------------------------
// scores[t, n] = sum over the heads h of a group of q[t, h] . means[n]: one product with heads and dims side by side as K, so that the
// sum over heads costs no additions of its own; the products of 16-bit values are exact and are added in fp32 in tensor memory.  A thread block per
// SM walks jobs of 128 queries x up to 512 means: q comes from memory once, through a ring of TMA tiles, each multiplied with two tiles of 256 means that
// stay in shared memory (they are the same operand for every head).  Eight warps write the two accumulators out.  With up to 256 means a job uses one
// accumulator, in turn, and the ring is twice as deep.  Bound: HBM (q and the scores) and the tensor cores about equally (32768 queries, 32 heads, 512 blocks:
// 82 and 70 us); it takes 131 us (121 in an ncu capture), because the write-out of a job with two accumulators is not hidden.  A thread block per 128 x 256 tile, two on an SM: 140 us.
constexpr int kScoreRows = 128, kScoreCols = 256, kScoreMaxStages = 8;
constexpr int kScoreStageBytes = kScoreRows * 128;
constexpr int kScoreMeansBytes = 2 * kScoreCols * 128;                       // 256 rows of up to 128 dims
constexpr int kScoreOut = 2 * kScoreMeansBytes + 4 * kScoreStageBytes;       // behind 4 stages and two tiles of means, or 8 and one: 32 x 32 floats per writing warp
constexpr int kScoreBars = kScoreOut + 8 * 32 * 32 * 4;
constexpr int kScoreSmem = kScoreBars + 208;
constexpr int kScoreThreads = 320;  // warps 0-7 write (four an accumulator), warp 8 loads, warp 9 multiplies

// Job i of all: which sequence and head of keys, which queries, which tiles of means.
struct ScoreJob {
    uint32_t z, t, n, width;
    __device__ ScoreJob(uint32_t i, uint32_t across, uint32_t down)
    {
        const uint32_t pairs = (across + 1) / 2;
        z = i / (pairs * down);
        n = i % (pairs * down) / down * 2;
        t = i % down;
        width = min(2u, across - n);
    }
};

template <class T> __global__ void __launch_bounds__(kScoreThreads, 1) block_scores_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap m_map, ScoresArgs a, uint32_t jobs)
{
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + kScoreBars), *empty = full + kScoreMaxStages, *means_in = empty + kScoreMaxStages, *summed = means_in + 2, *written = summed + 2;
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(written + 2);  // [0] tensor memory, [1] gave up
    const uint32_t across = (a.blocks + kScoreCols - 1) / kScoreCols, down = (a.queries + kScoreRows - 1) / kScoreRows;
    const uint32_t stages = across == 1 ? 8u : 4u, means_at = stages * kScoreStageBytes;
    const uint32_t begin = (uint32_t)((uint64_t)jobs * blockIdx.x / gridDim.x), end = (uint32_t)((uint64_t)jobs * (blockIdx.x + 1) / gridDim.x);
    const uint32_t group = a.heads / a.kv_heads, halves = (a.dim + 63) / 64, steps = group * halves;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kScoreMaxStages; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(&means_in[s], 1);
            ptx::mbar_init(&summed[s], 1);
            ptx::mbar_init(&written[s], 4);
        }
        misc[1] = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 0) tc::alloc(const_cast<uint32_t *>(&misc[0]), 2 * kScoreCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = misc[0];
    ptx::grid_wait();
    ptx::grid_release();
    bool ok = true;
    if (warp == 8) {
        if (lane == 0) {
            uint32_t k = 0, loads = 0, holds = ~0u;  // tiles of q so far; the means that are there: (z, n)
            for (uint32_t i = begin; i < end && ok; ++i) {
                const ScoreJob x(i, across, down);
                const uint32_t b = x.z / a.kv_heads, kv = x.z % a.kv_heads;
                if (holds != x.z * across + x.n) {
                    holds = x.z * across + x.n;
                    for (uint32_t j = k > stages ? k - stages : 0; j < k && ok; ++j) ok = ptx::mbar_wait(&empty[j % stages], (j / stages) & 1u);  // nothing reads the old ones any more
                    if (!ok) break;
                    for (uint32_t m = 0; m < x.width; ++m) {
                        ptx::mbar_expect_tx(&means_in[m], halves * kScoreCols * 128);
                        for (uint32_t h = 0; h < halves; ++h)
                            tc::tma_load4(smem + means_at + m * kScoreMeansBytes + h * kScoreCols * 128, &m_map, (int)(h * 64), (int)kv, (int)((x.n + m) * kScoreCols), (int)b, &means_in[m]);
                        loads += m ? 1u << 16 : 1u;
                    }
                }
                for (uint32_t j = 0; j < steps; ++j, ++k) {
                    const uint32_t s = k % stages;
                    if (!(ok = ptx::mbar_wait(&empty[s], ((k / stages) & 1u) ^ 1u))) break;
                    ptx::mbar_expect_tx(&full[s], kScoreStageBytes);
                    tc::tma_load4(smem + s * kScoreStageBytes, &q_map, (int)(j % halves * 64), (int)(kv * group + j / halves), (int)(x.t * kScoreRows), (int)b, &full[s]);
                }
            }
            if (!ok) {
                misc[1] = 1;
                // no copy stays in flight
                if (loads & 0xffffu) ptx::mbar_wait(&means_in[0], (loads - 1) & 1u);
                if (loads >> 16) ptx::mbar_wait(&means_in[1], ((loads >> 16) - 1) & 1u);
                for (uint32_t j = k > stages ? k - stages : 0; j < k; ++j) ptx::mbar_wait(&full[j % stages], (j / stages) & 1u);
            }
        }
    } else if (warp == 9) {
        if (lane == 0) {
            constexpr uint32_t id = tc::idesc(std::is_same<T, __nv_bfloat16>::value, kScoreRows, kScoreCols);
            const uint64_t q_k = tc::desc_k(ptx::smem_u32(smem)), m_k = tc::desc_k(ptx::smem_u32(smem) + means_at);
            uint32_t k = 0, holds = ~0u, loads[2] = {0, 0}, uses[2] = {0, 0};
            for (uint32_t i = begin; i < end && ok; ++i) {
                const ScoreJob x(i, across, down);
                const uint32_t first = x.width == 2 ? 0u : (i - begin) & 1u, last = x.width == 2 ? 1u : first;  // accumulators of the job
                if (holds != x.z * across + x.n) {
                    holds = x.z * across + x.n;
                    for (uint32_t m = 0; m < x.width && ok; ++m) ok = ptx::mbar_wait(&means_in[m], loads[m]++ & 1u);
                }
                for (uint32_t c = first; c <= last && ok; ++c) ok = ptx::mbar_wait(&written[c], (uses[c]++ & 1u) ^ 1u);
                if (!ok) break;
                for (uint32_t j = 0; j < steps; ++j, ++k) {
                    const uint32_t s = k % stages;
                    if (!(ok = ptx::mbar_wait(&full[s], (k / stages) & 1u))) break;
                    tc::fence_after();
                    const uint64_t ad = q_k + s * (kScoreStageBytes >> 4);
                    for (uint32_t c = first; c <= last; ++c) {
                        const uint64_t bd = m_k + ((c - first) * (kScoreMeansBytes >> 4) + j % halves * (kScoreCols * 128 >> 4));
#pragma unroll
                        for (int d = 0; d < 4; ++d) tc::mma(tmem + c * kScoreCols, ad + 2 * d, bd + 2 * d, id, j || d);
                    }
                    tc::commit(&empty[s]);
                }
                for (uint32_t c = first; c <= last; ++c) tc::commit(&summed[c]);
            }
            if (!ok) misc[1] = 1;
        }
    } else {
        // accumulator -> rows of scores, 32 x 32 at a time through shared memory, so that a store is whole 128-byte pieces of rows: 16 bytes a
        // lane where rows allow that, 4 otherwise (a loop that stored what it had just read took 17000 cycles a job, as long as the products)
        unsigned char *part = smem + kScoreOut + warp * 32 * 128;
        auto piece = [&](uint32_t row, uint32_t p) { return part + row * 128 + ((p ^ (row & 7)) << 4); };
        const bool wide = a.blocks % 4 == 0 && reinterpret_cast<uintptr_t>(a.scores) % 16 == 0;
        const uint32_t acc = warp >> 2;
        uint32_t uses = 0;
        for (uint32_t i = begin; i < end; ++i) {
            const ScoreJob x(i, across, down);
            if (x.width == 1 && ((i - begin) & 1u) != acc) continue;
            const uint32_t t0 = x.t * kScoreRows + (warp & 3) * 32, n0 = (x.n + (x.width == 2 ? acc : 0u)) * kScoreCols;
            if (!(ok = ptx::mbar_wait_warp(&summed[acc], uses++ & 1u))) break;
            tc::fence_after();
            float *out = a.scores + ((uint64_t)x.z * a.queries + t0) * a.blocks + n0;
            const uint32_t rows = t0 < a.queries ? min(32u, a.queries - t0) : 0u;
            for (uint32_t c = 0; c < kScoreCols && n0 + c < a.blocks; c += 32) {
                uint32_t v[32];
                tc::ld32(tmem + (((warp & 3) * 32) << 16) + acc * kScoreCols + c, v);
                tc::wait_ld();
                __syncwarp();
#pragma unroll
                for (int p = 0; p < 8; ++p) *reinterpret_cast<uint4 *>(piece(lane, p)) = make_uint4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
                __syncwarp();
                if (wide) {
                    const uint32_t p = lane & 7, col = c + 4 * p;
                    uint4 y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = *reinterpret_cast<const uint4 *>(piece(4 * k + lane / 8, p));
                    if (n0 + col < a.blocks) {
                        float *to = out + (uint64_t)(lane / 8) * a.blocks + col;
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (4 * k + lane / 8 < rows) __stcs(reinterpret_cast<uint4 *>(to + (uint64_t)(4 * k) * a.blocks), y[k]);
                    }
                } else if (n0 + c + lane < a.blocks) {
                    float *to = out + c + lane;
#pragma unroll
                    for (uint32_t r = 0; r < 32; r += 16) {
                        float y[16];
#pragma unroll
                        for (uint32_t k = 0; k < 16; ++k) y[k] = *reinterpret_cast<const float *>(piece(r + k, lane >> 2) + (lane & 3) * 4);
#pragma unroll
                        for (uint32_t k = 0; k < 16; ++k)
                            if (r + k < rows) __stcs(to + (uint64_t)(r + k) * a.blocks, y[k]);
                    }
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&written[acc]);
        }
        if (!ok) misc[1] = 1;
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && misc[1]) atomicExch(&g_status, 1u);
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tmem, 2 * kScoreCols);
    }
}

// ---- selection ---------------------------------------------------------------------------------------------------------
// WARPS warps take one row of scores, 32 * R consecutive ones each, in registers as unsigned integers of the same order (0: not to be
// chosen; all ones: chosen in any case).  The count-th largest is found by halving an interval of integers -- how many are at least this
// candidate? -- until a candidate leaves exactly `count`; with up to 32 to choose the interval begins at the least of the lanes' largest
// keys, of which there are 32, and takes some eight halvings instead of twenty from the top bit down (16384 x 4 rows of 256, 16 to choose:
// 58 us that way).  Then the chosen indices are written in ascending order, equal scores from the lowest index on.  Bound: instructions in large calls,
// latency in small ones.
template <int R, int WARPS> __device__ __forceinline__ void select_row(const SelectArgs &a, const float *src, uint32_t n, int32_t *out, uint32_t (*counts)[2])
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = WARPS == 1 ? 0 : warp;
    const uint32_t i0 = part * R * 32 + lane;
    uint32_t key[R];
    uint32_t any = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t i = i0 + r * 32;
        key[r] = 0;
        if (i < n) {
            const float f = __ldg(src + i) + 0.f;  // -0 becomes 0: they are equal scores
            const uint32_t bits = __float_as_uint(f);
            if (f > -INFINITY) key[r] = (bits >> 31) ? ~bits : bits | 0x80000000u;  // neither NaN nor -infinity
            if (i < a.first || i + a.last >= n) key[r] = ~0u;
        }
        any += key[r] != 0;
    }
    // how many of the row
    auto total = [&](uint32_t v) {
        v = __reduce_add_sync(~0u, v);
        if constexpr (WARPS > 1) {
            __syncthreads();
            if (lane == 0) counts[warp][0] = v;
            __syncthreads();
            v = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += counts[w][0];
        }
        return v;
    };
    uint32_t limit = 0;     // chosen: every key above it, and the first `ties` that equal it (never keys of 0)
    uint32_t ties = 0;
    if (total(any) > a.count) {
        uint32_t top = 0, least = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) top = max(top, key[r]);
        if (a.count <= 32) least = __reduce_min_sync(~0u, top);
        top = __reduce_max_sync(~0u, top);
        if constexpr (WARPS > 1) {
            __syncthreads();
            if (lane == 0) {
                counts[warp][0] = top;
                counts[warp][1] = least;
            }
            __syncthreads();
            least = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                top = max(top, counts[w][0]);
                least = max(least, counts[w][1]);  // any warp's 32 lanes will do
            }
        }
        // at least `lo` are count keys and more, at least `hi` are fewer than count, or exactly that many (hi found)
        uint32_t lo = max(least, 1u), hi = top;
        uint32_t c = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) c += key[r] >= hi;
        uint32_t above = total(c);  // keys of at least hi
        if (above > a.count) {      // so many equal ones at the top
            lo = hi;
            above = 0;
        } else
            while (above != a.count && hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                c = 0;
#pragma unroll
                for (int r = 0; r < R; ++r) c += key[r] >= mid;
                c = total(c);
                if (c <= a.count) {
                    hi = mid;
                    above = c;
                } else
                    lo = mid;
            }
        if (above == a.count) limit = hi - 1;
        else {
            limit = lo;
            ties = a.count - above;
        }
    }
    uint32_t before = 0, ties_before = 0;  // chosen, and equal to the limit, at lower indices
    if constexpr (WARPS > 1) {
        uint32_t above = 0, equal = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            above += key[r] > limit;
            equal += ties && key[r] == limit;
        }
        above = __reduce_add_sync(~0u, above);
        equal = __reduce_add_sync(~0u, equal);
        __syncthreads();
        if (lane == 0) {
            counts[warp][0] = above;
            counts[warp][1] = equal;
        }
        __syncthreads();
        for (uint32_t w = 0; w < part; ++w) {
            before += counts[w][0];
            ties_before += counts[w][1];
        }
        before += min(ties_before, ties);
    }
    const uint32_t below = (1u << lane) - 1u;
    if (ties) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t equal = __ballot_sync(~0u, key[r] == limit);
            const uint32_t chosen = __ballot_sync(~0u, key[r] > limit || (key[r] == limit && ties_before + __popc(equal & below) < ties));
            if ((chosen >> lane) & 1u) out[before + __popc(chosen & below)] = (int32_t)(i0 + r * 32);
            before += __popc(chosen);
            ties_before += __popc(equal);
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool mine = key[r] > limit;
            const uint32_t chosen = __ballot_sync(~0u, mine);
            if (mine) out[before + __popc(chosen & below)] = (int32_t)(i0 + r * 32);
            before += __popc(chosen);
        }
    }
    if (part == WARPS - 1)
        for (uint32_t i = before + lane; i < a.count; i += 32) out[i] = -1;
}

template <int R, int WARPS> __global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) select_blocks_kernel(SelectArgs a)
{
    constexpr int kRowsPerBlock = WARPS == 1 ? 4 : 1;
    __shared__ uint32_t counts[WARPS][2];
    ptx::grid_wait();
    ptx::grid_release();
    const uint32_t t = blockIdx.x * kRowsPerBlock + (WARPS == 1 ? threadIdx.x >> 5 : 0), bh = blockIdx.y, b = bh / a.kv_heads;
    if (t >= a.queries) return;
    const int64_t see = a.visible ? a.visible[(uint64_t)b * a.queries + t] : (int64_t)a.keys - a.queries + 1 + t;
    const uint32_t visible = (uint32_t)min(max(see, (int64_t)0), (int64_t)a.keys);
    const uint32_t n = min((visible + a.block - 1) / a.block, a.blocks);
    const float *src = a.scores + (int64_t)b * a.s_batch + (int64_t)(bh % a.kv_heads) * a.s_head + (int64_t)t * a.s_query;
    int32_t *out = a.out + ((uint64_t)bh * a.queries + t) * a.count;
    // a row that sees a half or a quarter of the blocks takes as many instructions less
    if constexpr (WARPS == 1 && R >= 4) {
        if (n <= R * 8) select_row<R / 4, 1>(a, src, n, out, counts);
        else if (n <= R * 16) select_row<R / 2, 1>(a, src, n, out, counts);
        else select_row<R, 1>(a, src, n, out, counts);
    } else
        select_row<R, WARPS>(a, src, n, out, counts);
}

}  // namespace

cudaError_t launch_block_means(const MeansArgs &a, cudaStream_t s)
{
    if (!a.batch || !a.blocks || !a.kv_heads || !a.dim) return cudaSuccess;
    const dim3 grid(a.blocks, (a.kv_heads * (a.dim / 8) + 31) / 32, a.batch);
    return a.dtype == CUTESPMM_BF16 ? launch_overlapped(block_means_kernel<__nv_bfloat16>, grid, dim3(kMeanWarps * 32), 0, s, a)
                                    : launch_overlapped(block_means_kernel<__half>, grid, dim3(kMeanWarps * 32), 0, s, a);
}

cudaError_t launch_block_scores(const ScoresArgs &a, int sm_count, cudaStream_t s)
{
    if (!a.batch || !a.queries || !a.kv_heads || !a.blocks) return cudaSuccess;
    if (!a.heads) return cudaMemsetAsync(a.scores, 0, (uint64_t)a.batch * a.kv_heads * a.queries * a.blocks * 4, s);  // sums of nothing
    const bool bf16 = a.dtype == CUTESPMM_BF16;
    CUtensorMap q_map, m_map;
    cudaError_t e = tc::make_map(&q_map, bf16, a.q, a.dim, a.heads, a.queries, a.batch, a.q_head, a.q_query, a.q_batch, kScoreRows);
    if (e == cudaSuccess) e = tc::make_map(&m_map, bf16, a.means, a.dim, a.kv_heads, a.blocks, a.batch, a.m_head, a.m_block, a.m_batch, kScoreCols);
    if (e == cudaSuccess) e = bf16 ? allow_dynamic_smem<block_scores_kernel<__nv_bfloat16>>(kScoreSmem) : allow_dynamic_smem<block_scores_kernel<__half>>(kScoreSmem);
    if (e != cudaSuccess) return e;
    const uint64_t jobs = (uint64_t)((a.blocks + 2 * kScoreCols - 1) / (2 * kScoreCols)) * ((a.queries + kScoreRows - 1) / kScoreRows) * a.batch * a.kv_heads;
    if (jobs >> 31) return cudaErrorInvalidConfiguration;
    const unsigned grid = (unsigned)(jobs < (uint64_t)sm_count ? jobs : (uint64_t)sm_count);
    return bf16 ? launch_overlapped(block_scores_kernel<__nv_bfloat16>, dim3(grid), dim3(kScoreThreads), kScoreSmem, s, q_map, m_map, a, (uint32_t)jobs)
                : launch_overlapped(block_scores_kernel<__half>, dim3(grid), dim3(kScoreThreads), kScoreSmem, s, q_map, m_map, a, (uint32_t)jobs);
}

cudaError_t launch_select_blocks(const SelectArgs &a, int sm_count, cudaStream_t s)
{
    const uint64_t rows = (uint64_t)a.batch * a.kv_heads * a.queries;
    if (!rows || !a.count) return cudaSuccess;
    const unsigned heads = a.batch * a.kv_heads;
    auto one = [&](auto kernel) { return launch_overlapped(kernel, dim3((a.queries + 3) / 4, heads), dim3(128), 0, s, a); };
    auto eight = [&](auto kernel) { return launch_overlapped(kernel, dim3(a.queries, heads), dim3(256), 0, s, a); };
    // eight warps a row where there are too few rows to fill the machine with a warp each, or too many scores for one warp's registers.  One warp / eight, us, the
    // launches of a graph: rows of 1024 scores 256: 9.8 / 5.4, 1000: 10.2 / 11.4, 2400: 13.8 / 21; of 256 scores 8: 4.0 / 4.0, 1000: 4.5 / 9.2, 2400: 5.2 / 16, 65536: 58 / 349
    if (a.blocks <= 1024 && (a.blocks <= 32 || rows > (uint64_t)sm_count * 8)) {
        if (a.blocks <= 32) return one(select_blocks_kernel<1, 1>);
        if (a.blocks <= 64) return one(select_blocks_kernel<2, 1>);
        if (a.blocks <= 128) return one(select_blocks_kernel<4, 1>);
        if (a.blocks <= 256) return one(select_blocks_kernel<8, 1>);
        if (a.blocks <= 512) return one(select_blocks_kernel<16, 1>);
        return one(select_blocks_kernel<32, 1>);
    }
    if (a.blocks <= 256) return eight(select_blocks_kernel<1, 8>);
    if (a.blocks <= 1024) return eight(select_blocks_kernel<4, 8>);
    if (a.blocks <= 4096) return eight(select_blocks_kernel<16, 8>);
    return eight(select_blocks_kernel<64, 8>);
}

namespace tc {

cudaError_t make_map(CUtensorMap *out, bool bf16, const void *p, uint32_t dim, uint32_t heads, uint32_t rows, uint32_t outer, int64_t head_stride, int64_t row_stride,
                     int64_t outer_stride, uint32_t box_rows, uint32_t box_heads)
{
    // the stride of an extent of one is never used, but has to be one that a map can hold
    auto bytes = [](int64_t stride, uint32_t extent) { return (cuuint64_t)(extent > 1 ? stride * 2 : 16); };
    const cuuint64_t dims[4] = {dim, heads, rows, outer};
    const cuuint64_t strides[3] = {bytes(head_stride, heads), bytes(row_stride, rows), bytes(outer_stride, outer)};
    const cuuint32_t box[4] = {64, box_heads, box_rows, 1};
    return encode_tiled(out, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

}  // namespace tc

cudaError_t block_select_status(uint32_t *word) { return read_status(g_status, word); }

}  // namespace cutespmm
