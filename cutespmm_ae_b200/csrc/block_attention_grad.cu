// Gradients of attention over selected blocks.  With P = exp(scale q K^T - lse), D = dout V^T and delta = <dout, out> per row:
//   dS = P (D - delta),   dq = scale dS K,   dk = scale dS^T q,   dv = P^T dout.
//
// Two walks over the pattern, each with sums of its own and in a fixed order, so nothing is added by atomics:
//   * dq by tiles of neighbouring queries over the union of their blocks, like the forward kernel (block_attention_dq_kernel);
//   * dk and dv by tiles of 64 keys over the queries that name them (block_attention_dkv_kernel).  That needs the pattern turned round:
//     a bit per (block, query), from which the kernel reads a tile's queries in ascending order.
// P is formed again in each of the two from lse; nothing of size queries x keys is stored.
//
// Roundings to 16 bits, each half a step u: dS as operand of dq and dk, P as operand of dv (the tensor cores multiply 16-bit values by 16-bit
// values only), out, which delta is formed from, and the results.  Against 64 bits dq is 2.6e-3 to 3.1e-3 off in bf16 where fp32 throughout is 1.7e-3, dk 2.4e-3.
// The roundings one by one in 64 bits give exactly that: dS and the result 2.5e-3, delta from an exact out rounded once 2.7e-3 to 3.0e-3, from the forward
// pass's out, which has P's rounding, 2.8e-3 to 3.1e-3 (dk 2.3e-3, 2.4e-3, 2.4e-3); fp16 3.4e-4 to 4.2e-4 where 2.1e-4.  dS makes most of it and has no other form here; for
// the rest the forward pass would have to leave a second copy of out, as large as the first, for every step.
// dS beyond fp16's range is infinite, and what it enters is formed again in fp32 (exact_dq_row, exact_key).
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

__device__ uint32_t g_status;  // set to 1 (dq) or 2 (dk, dv) when a bounded wait gives up

// ---- dq ----------------------------------------------------------------------------------------------------------------
// The forward kernel's 128 rows and union of key tiles.  Per tile S = Q K^T and D = dO V^T (128 x 64, two buffers of tensor memory), dS from
// registers back into S's columns as 16-bit operand, dQ += dS K with the same bytes of K.  Q and dO stay in tensor memory for the whole kernel: an
// operand A in shared memory would be read again for every 16 dims, 6 KB for 32 cycles of multiplying.  Eight warps form dS: a row's lse and
// delta are one value each, two threads share a row.  Warp 8 loads, warp 9 issues S and D, warp 10 dQ.  Measured: 8192 queries, 32 heads of dim 128 over 4,
// 16 blocks of 64: 585 us (q and dout in shared memory, one issuing warp: 713), tensor pipe 39 % busy; bound by the round trip of a tile through its two buffers.  A row whose dq is not finite is formed again from
// what its query looks at.
constexpr int kDqWarps = 8, kDqThreads = (kDqWarps + 3) * 32, kDqStages = 4;
constexpr uint32_t kDqBuffer = 128, kDqSum = 256, kDqQ = 384, kDqDo = 448, kDqCols = 512;

template <int DP> struct DqSmem {
    static constexpr int kTile = DP / 64 * 64 * 128;
    static constexpr int kKeys = 0, kValues = kDqStages * kTile;
    static constexpr int kDelta = 2 * kDqStages * kTile;  // two shares of delta per row
    static constexpr int kBars = kDelta + 2 * 128 * 4;
    static constexpr int kLists = kBars + 192;
};

// dq of one row by itself: a warp, four dims a lane.  Dims first to end - 1 are written: the others are another warp's, and what it has stored
// there, or forms again by itself, stays.
template <class T>
__device__ void exact_dq_row(const AttentionArgs &a, const TileUnion &u, uint32_t b, uint32_t kv, uint32_t t, uint32_t q_of_tile, uint32_t head, float delta, uint32_t first, uint32_t end)
{
    const uint32_t lane = threadIdx.x & 31, d = lane * 4;
    const bool on = d < a.dim;
    const T *qr = static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)t * a.q_query + (int64_t)head * a.q_head + d;
    const T *gr = static_cast<const T *>(a.dout) + (int64_t)b * a.do_batch + (int64_t)t * a.do_query + (int64_t)head * a.do_head + d;
    float q[4] = {}, g[4] = {}, sum[4] = {};
    if (on)
        for (int j = 0; j < 4; ++j) {
            q[j] = to_f32(qr[j]);
            g[j] = to_f32(gr[j]);
        }
    const float lse = a.lse[((uint64_t)b * a.heads + head) * a.queries + t];
    for (uint32_t slot = 0; slot < *u.size; ++slot)
        for (uint64_t seen = u.seen(slot, q_of_tile, a.block); seen; seen &= seen - 1) {
            const uint32_t key = u.tiles[slot] * kKeyTile + __ffsll((long long)seen) - 1;
            const T *kr = key_row<T>(a, a.k, a.k_batch, a.k_key, a.k_head, b, kv, key) + d, *vr = key_row<T>(a, a.v, a.v_batch, a.v_key, a.v_head, b, kv, key) + d;
            float s = 0.f, dp = 0.f;
            if (on)
                for (int j = 0; j < 4; ++j) {
                    s = fmaf(q[j], to_f32(kr[j]), s);
                    dp = fmaf(g[j], to_f32(vr[j]), dp);
                }
#pragma unroll
            for (int x = 16; x; x >>= 1) {
                s += __shfl_xor_sync(~0u, s, x);
                dp += __shfl_xor_sync(~0u, dp, x);
            }
            const float ds = exp2f((s * a.scale - lse) * kLog2e) * (dp - delta);
            if (on)
                for (int j = 0; j < 4; ++j) sum[j] = fmaf(ds, to_f32(kr[j]), sum[j]);
        }
    if (on && d >= first && d < end)
        for (int j = 0; j < 4; ++j) static_cast<T *>(a.dq)[(((uint64_t)b * a.queries + t) * a.heads + head) * a.dim + d + j] = from_f32<T>(a.scale * sum[j]);
}

// 8 V columns of tensor memory from V 16-byte pieces of a row
template <class T, int V> __device__ __forceinline__ void row_to_tmem(uint32_t taddr, const T *src, uint32_t dims)
{
    uint32_t w[4 * V];
#pragma unroll
    for (int x = 0; x < V; ++x) {
        const uint4 u = 8 * x < (int)dims ? __ldg(reinterpret_cast<const uint4 *>(src) + x) : make_uint4(0, 0, 0, 0);
        w[4 * x] = u.x;
        w[4 * x + 1] = u.y;
        w[4 * x + 2] = u.z;
        w[4 * x + 3] = u.w;
    }
    if constexpr (V == 8) tc::st32(taddr, w);
    else tc::st16(taddr, w);
}

template <class T, int DP>
__global__ void __launch_bounds__(kDqThreads, 1) block_attention_dq_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, AttentionArgs a, TcShape shape)
{
    using S = DqSmem<DP>;
    constexpr uint32_t kHalfDims = DP / 2;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a stage's values are given back when S and D are complete (scored), its keys when dQ is (summed)
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + S::kBars), *v_full = k_full + kDqStages, *scored = v_full + kDqStages, *formed = scored + kDqStages, *summed = formed + kDqStages, *rows_in = summed + kDqStages, *landed = rows_in + 1;
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(landed + 1);  // [0] tensor memory, [1] gave up
    TileUnion u(smem + S::kLists, shape.queries, a);
    const uint32_t t0 = blockIdx.x * shape.queries, b = blockIdx.z;
    const uint32_t kv = blockIdx.y / shape.chunks, group = a.heads / a.kv_heads, head0 = blockIdx.y % shape.chunks * shape.heads;
    const uint32_t heads = min(shape.heads, group - head0), queries = min(shape.queries, a.queries - t0);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kDqStages; ++s) {
            ptx::mbar_init(&k_full[s], 1);
            ptx::mbar_init(&v_full[s], 1);
            ptx::mbar_init(&scored[s], 1);
            ptx::mbar_init(&formed[s], kDqWarps);
            ptx::mbar_init(&summed[s], 1);
        }
        ptx::mbar_init(rows_in, kDqWarps);
        ptx::mbar_init(landed, 1);
        misc[1] = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 0) tc::alloc(const_cast<uint32_t *>(&misc[0]), kDqCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = misc[0];
    ptx::grid_wait();
    ptx::grid_release();
    u.build(a, b, kv, t0, queries);
    const uint32_t units = *u.size;

    bool ok = true;
    if (warp == kDqWarps) {
        uint32_t phase = 0, i = 0;
        for (; i < units; ++i) {
            const uint32_t s = i % kDqStages, parity = ((i / kDqStages) & 1u) ^ 1u;
            ok = ptx::mbar_wait_warp(&summed[s], parity) &&
                 load_key_tile<DP>(smem + S::kKeys + s * S::kTile, &k_map, a, b, kv, u.tiles[i], u.size[1], shape.box_rows, &k_full[s], landed, phase) &&
                 load_key_tile<DP>(smem + S::kValues + s * S::kTile, &v_map, a, b, kv, u.tiles[i], u.size[1], shape.box_rows, &v_full[s], landed, phase);
            if (!ok) break;
        }
        if (!ok) {
            misc[1] = 1;
            if (lane == 0)  // no copy stays in flight
                for (uint32_t j = i > kDqStages ? i - kDqStages : 0; j <= i && j < units; ++j) {
                    ptx::mbar_wait(&k_full[j % kDqStages], (j / kDqStages) & 1u);
                    ptx::mbar_wait(&v_full[j % kDqStages], (j / kDqStages) & 1u);
                }
        }
    } else if (warp == kDqWarps + 1) {
        if (lane == 0) {
            constexpr uint32_t id = tc::idesc(std::is_same<T, __nv_bfloat16>::value, 128, 64);
            const uint64_t k_k = tc::desc_k(ptx::smem_u32(smem) + S::kKeys), v_k = tc::desc_k(ptx::smem_u32(smem) + S::kValues);
            ok = ptx::mbar_wait(rows_in, 0);
            for (uint32_t i = 0; ok && i < units; ++i) {
                const uint32_t s = i % kDqStages, parity = (i / kDqStages) & 1u, at = s * (S::kTile >> 4), buffer = tmem + (i & 1u) * kDqBuffer;
                // the buffer held dS two tiles ago
                if (!(ok = ptx::mbar_wait(&k_full[s], parity) && ptx::mbar_wait(&v_full[s], parity) && (i < 2 || ptx::mbar_wait(&summed[(i - 2) % kDqStages], ((i - 2) / kDqStages) & 1u)))) break;
                tc::fence_after();
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) tc::mma_ta(buffer, tmem + kDqQ + d * 8, k_k + (at + (d >> 2) * 512 + (d & 3) * 2), id, d != 0);
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) tc::mma_ta(buffer + 64, tmem + kDqDo + d * 8, v_k + (at + (d >> 2) * 512 + (d & 3) * 2), id, d != 0);
                tc::commit(&scored[s]);
            }
            if (!ok) misc[1] = 1;
        }
    } else if (warp == kDqWarps + 2) {
        if (lane == 0) {
            constexpr uint32_t id = tc::idesc(std::is_same<T, __nv_bfloat16>::value, 128, DP, false, true);
            const uint64_t k_mn = tc::desc_mn(ptx::smem_u32(smem) + S::kKeys, 64 * 128);
            for (uint32_t i = 0; i < units; ++i) {
                const uint32_t s = i % kDqStages, at = s * (S::kTile >> 4), ds = tmem + (i & 1u) * kDqBuffer;
                if (!(ok = ptx::mbar_wait(&formed[s], (i / kDqStages) & 1u))) break;
                tc::fence_after();
                // the two threads of a row leave 16 columns each, where they read S
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma_ta(tmem + kDqSum, ds + (k >> 1) * 32 + (k & 1) * 8, k_mn + (at + k * 128), id, i || k);
                tc::commit(&summed[s]);
            }
            if (!ok) misc[1] = 1;
        }
    } else {
        const uint32_t r = threadIdx.x & 127, half = threadIdx.x >> 7, q = r / shape.heads, h = r % shape.heads, head = kv * group + head0 + h;
        const bool real = q < queries && h < heads;
        const uint32_t tq = real ? t0 + q : t0, th = real ? head : kv * group;  // rows that are none read a row that is
        const uint64_t row = ((uint64_t)b * a.queries + tq) * a.heads + th, stat = ((uint64_t)b * a.heads + th) * a.queries + tq;
        const uint32_t lanes_in = tmem + (((warp & 3) * 32) << 16), dims = !real || a.dim <= half * kHalfDims ? 0u : min(a.dim - half * kHalfDims, kHalfDims);
        const T *dout = static_cast<const T *>(a.dout) + (int64_t)b * a.do_batch + (int64_t)tq * a.do_query + (int64_t)th * a.do_head + half * kHalfDims;
        row_to_tmem<T, DP / 16>(lanes_in + kDqQ + half * (DP / 4), static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)tq * a.q_query + (int64_t)th * a.q_head + half * kHalfDims, dims);
        row_to_tmem<T, DP / 16>(lanes_in + kDqDo + half * (DP / 4), dout, dims);
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(rows_in);
        // delta = <dout, out>, while the first tiles are on their way
        float part = 0.f;
        const T *out = static_cast<const T *>(a.out) + row * a.dim + half * kHalfDims;
#pragma unroll
        for (uint32_t x = 0; x < kHalfDims / 8; ++x)
            if (8 * x < dims) {
                const Pack<T, 8> o = load_pack<T, 8>(out + 8 * x), g = load_pack<T, 8>(dout + 8 * x);
#pragma unroll
                for (int j = 0; j < 8; ++j) part = fmaf(to_f32(o.x[j]), to_f32(g.x[j]), part);
            }
        float *shares = reinterpret_cast<float *>(smem + S::kDelta);
        shares[half * 128 + r] = part;
        asm volatile("bar.sync 1, %0;" ::"n"(kDqWarps * 32) : "memory");
        const float delta = shares[r] + shares[128 + r], lse = real ? a.lse[stat] * kLog2e : 0.f, scale_log2 = a.scale * kLog2e;
        if (real && half == 0) a.delta[stat] = delta;
        const uint32_t lanes = tmem + (((warp & 3) * 32) << 16);
        for (uint32_t i = 0; i < units; ++i) {
            const uint64_t both = real ? u.seen(i, q, a.block) : 0ull;
            const uint32_t seen = half ? (uint32_t)(both >> 32) : (uint32_t)both;
            const uint32_t s = i % kDqStages, buffer = lanes + (i & 1u) * kDqBuffer + half * 32;
            if (!(ok = ptx::mbar_wait_warp(&scored[s], (i / kDqStages) & 1u))) break;
            tc::fence_after();
            uint32_t ds[16];
            if (__any_sync(~0u, seen != 0)) {
                uint32_t sv[32], dv[32];
                tc::ld32(buffer, sv);
                tc::ld32(buffer + 64, dv);
                tc::wait_ld();
                // a row that does not name the tile: P is 0 (where D is no number dq is none, and that is formed again)
                const float minus = seen ? -lse : -INFINITY;
                const uint64_t scale2 = ptx::pack2(scale_log2, scale_log2), minus2 = ptx::pack2(minus, minus), delta2 = ptx::pack2(-delta, -delta);
                const bool plain = __all_sync(~0u, seen == 0 || seen == ~0u);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float2 x = ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), scale2, minus2));
                    const uint64_t e = ptx::pack2(tc::exp2_fast(x.x), tc::exp2_fast(x.y)), d = ptx::add2(ptx::pack2(__uint_as_float(dv[2 * c]), __uint_as_float(dv[2 * c + 1])), delta2);
                    const float2 y = ptx::unpack2(ptx::mul2(e, d));
                    ds[c] = tc::round2<T>(y.x, y.y);
                }
                if (!plain) {
#pragma unroll
                    for (int c = 0; c < 16; ++c) ds[c] &= ((seen >> (2 * c)) & 1u ? 0xffffu : 0u) | ((seen >> (2 * c + 1)) & 1u ? 0xffff0000u : 0u);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 16; ++c) ds[c] = 0;
            }
            __syncwarp();
            tc::st16(buffer, ds);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&formed[s]);
        }
        if (ok && units) ok = ptx::mbar_wait_warp(&summed[(units - 1) % kDqStages], ((units - 1) / kDqStages) & 1u);
        tc::fence_after();
        if (!ok) misc[1] = 1;
        T *dst = static_cast<T *>(a.dq) + row * a.dim;
        bool finite = true;
#pragma unroll 1
        for (uint32_t c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
            uint32_t o[32];
            if (units) {
                tc::ld32(lanes + kDqSum + c, o);
                tc::wait_ld();
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float o0 = units ? __uint_as_float(o[8 * x + 2 * y]) * a.scale : 0.f, o1 = units ? __uint_as_float(o[8 * x + 2 * y + 1]) * a.scale : 0.f;
                    finite = finite && fabsf(o0) < INFINITY && fabsf(o1) < INFINITY;
                    w[y] = tc::round2<T>(o0, o1);
                }
                if (real && c + 8 * x < a.dim) *reinterpret_cast<uint4 *>(dst + c + 8 * x) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        for (uint32_t left = __ballot_sync(~0u, real && !finite); left && !misc[1]; left &= left - 1) {
            const uint32_t from = __ffs(left) - 1, rq = __shfl_sync(~0u, q, from), rh = __shfl_sync(~0u, head, from);
            const float rd = __shfl_sync(~0u, delta, from);
            __syncwarp();
            exact_dq_row<T>(a, u, b, kv, t0 + rq, rq, rh, rd, half * (DP / 2), (half + 1) * (DP / 2));
        }
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && misc[1]) atomicExch(&g_status, 1u);
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tmem, kDqCols);
    }
}

// ---- the pattern turned round ------------------------------------------------------------------------------------------
constexpr uint32_t kItemRows = 4096;   // (query, head) rows that one work item takes at least, unless the tile has fewer

// Where the parts of the workspace begin (bytes), and the sizes they follow from.
struct GradLayout {
    uint32_t words, tiles;  // words of a block's bits over the queries; key tiles of a sequence
    uint64_t tile_rows;     // key tiles of all sequences and heads of keys
    uint32_t item_queries;  // queries of a work item
    uint64_t max_items, max_slots;
    uint64_t delta, bits, bits_bytes, counts, items, totals, partial, total;
    explicit GradLayout(const AttentionArgs &a)
    {
        const uint32_t group = a.heads / a.kv_heads;
        words = (a.queries + 31) / 32;
        tiles = (a.keys + kKeyTile - 1) / kKeyTile;
        tile_rows = (uint64_t)a.batch * a.kv_heads * tiles;
        // every pair of a query and a block it names is in one tile, in two where a block is two tiles
        const uint64_t pairs = (uint64_t)a.batch * a.kv_heads * a.queries * a.count * (a.block > kKeyTile ? 2 : 1);
        uint64_t rows = pairs * group / 4096;  // about 4096 items in large jobs
        if (rows < kItemRows) rows = kItemRows;
        const uint32_t per_tile = 128 / group;  // queries of 128 rows
        uint64_t n = rows / group < a.queries ? rows / group : a.queries;
        item_queries = (uint32_t)((n + per_tile - 1) / per_tile * per_tile);
        max_items = pairs / item_queries + tile_rows;
        max_slots = 2 * (pairs / item_queries) + 1;  // a tile with two items or more has more than half of them full
        uint64_t at = 0;
        auto take = [&](uint64_t bytes) { const uint64_t p = at; at += (bytes + 255) / 256 * 256; return p; };
        delta = take((uint64_t)a.batch * a.heads * a.queries * 4);
        bits_bytes = (uint64_t)a.batch * a.kv_heads * a.num_blocks * words * 4;
        bits = take(bits_bytes);
        counts = take(tile_rows * 16);  // of each tile: queries, then the first item, then the first slot, then whether sums are formed again
        items = take(max_items * 8);
        totals = take(8);
        partial = take(max_slots * 2 * kKeyTile * (a.dim <= 64 ? 64 : 128) * 4);
        total = at;
    }
};

struct TurnArgs {
    AttentionArgs a;
    uint32_t words, tiles, item_queries;
    uint64_t tile_rows;
    uint32_t *bits, *counts, *first_item, *first_slot, *redo;
    uint2 *items;      // (tile row, which of its items)
    uint32_t *totals;  // items
    float *partial;
};

// A warp per 32 queries: lane i sets query i's bit in the blocks it names.
__global__ void __launch_bounds__(256) pattern_bits_kernel(TurnArgs p)
{
    ptx::grid_wait();
    ptx::grid_release();
    const AttentionArgs &a = p.a;
    const uint64_t w = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31;
    if (w >= (uint64_t)a.batch * a.kv_heads * p.words) return;
    const uint32_t word = (uint32_t)(w % p.words), bh = (uint32_t)(w / p.words), b = bh / a.kv_heads, t = word * 32 + lane;
    if (t >= a.queries) return;
    const uint32_t visible = visible_keys(a, b, t);
    const int32_t *src = a.blocks + ((uint64_t)bh * a.queries + t) * a.count;
    for (uint32_t i = 0; i < a.count; ++i) {
        const int32_t j = src[i];
        if (block_counts(a, b, j, visible)) atomicOr(p.bits + ((uint64_t)bh * a.num_blocks + j) * p.words + word, 1u << lane);
    }
}

// The queries that name some block of a key tile, 32 of them.
__device__ __forceinline__ uint32_t tile_word(const TurnArgs &p, uint64_t tile_row, uint32_t word)
{
    const AttentionArgs &a = p.a;
    const uint32_t tile = (uint32_t)(tile_row % p.tiles);
    const uint64_t bh = tile_row / p.tiles;
    const uint32_t b0 = tile * kKeyTile / a.block, b1 = min((tile * kKeyTile + kKeyTile - 1) / a.block, a.num_blocks - 1);
    uint32_t any = 0;
    for (uint32_t j = b0; j <= b1; ++j) any |= p.bits[(bh * a.num_blocks + j) * p.words + word];
    return any;
}

__global__ void __launch_bounds__(256) pattern_count_kernel(TurnArgs p)
{
    ptx::grid_wait();
    ptx::grid_release();
    const uint64_t row = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.tile_rows) return;
    uint32_t n = 0;
    for (uint32_t w = threadIdx.x & 31; w < p.words; w += 32) n += __popc(tile_word(p, row, w));
    n = __reduce_add_sync(~0u, n);
    if ((threadIdx.x & 31) == 0) {
        p.counts[row] = n;
        p.redo[row] = 0;
    }
}

// Work item it: its first query, as a rank among those that name the tile, and how many it takes -- equal parts, whole tiles of rows.
__device__ __forceinline__ uint2 item_part(const TurnArgs &p, uint2 it)
{
    const uint32_t n = p.counts[it.x], parts = (n + p.item_queries - 1) / p.item_queries, per_tile = 128 / (p.a.heads / p.a.kv_heads);
    const uint32_t each = ((n + parts - 1) / parts + per_tile - 1) / per_tile * per_tile, first = it.y * each;
    return make_uint2(first, min(each, n - first));
}
__device__ __forceinline__ void copy16(uint32_t saddr, uint64_t src, uint32_t bytes)  // what is behind `bytes` becomes zeros
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(src), "r"(bytes) : "memory");
}

// One block: the work items of every tile, in order; slots for partial sums where a tile has several.
__global__ void __launch_bounds__(1024) pattern_items_kernel(TurnArgs p)
{
    __shared__ uint2 warp_sum[32];
    ptx::grid_wait();
    ptx::grid_release();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t items_before = 0, slots_before = 0;
    for (uint64_t r0 = 0; r0 < p.tile_rows; r0 += 1024) {
        const uint64_t row = r0 + threadIdx.x;
        const uint32_t n = row < p.tile_rows ? (p.counts[row] + p.item_queries - 1) / p.item_queries : 0u, slots = n > 1 ? n : 0u;
        uint32_t si = n, ss = slots;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t ui = __shfl_up_sync(~0u, si, d), us = __shfl_up_sync(~0u, ss, d);
            if (lane >= (uint32_t)d) {
                si += ui;
                ss += us;
            }
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = make_uint2(si, ss);
        __syncthreads();
        uint32_t bi = items_before + si - n, bs = slots_before + ss - slots;
        for (uint32_t w = 0; w < 32; ++w) {
            if (w < warp) {
                bi += warp_sum[w].x;
                bs += warp_sum[w].y;
            }
            items_before += warp_sum[w].x;
            slots_before += warp_sum[w].y;
        }
        if (row < p.tile_rows) {
            p.first_item[row] = bi;
            p.first_slot[row] = bs;
            for (uint32_t i = 0; i < n; ++i) p.items[bi + i] = make_uint2((uint32_t)row, i);
        }
    }
    if (threadIdx.x == 0) p.totals[0] = items_before;
}

// ---- dk and dv ---------------------------------------------------------------------------------------------------------
// One thread block per SM walks work items: 64 keys and a range of the queries that name them.  The queries' rows of q and dout are
// gathered into tiles of 128 rows (16 bytes a lane; a TMA box per query and 64 dims took 9100 cycles a tile, a hundred each to issue); per tile
//     S  = Q K^T   and  D = dO V^T       (128 x 64 each, tensor memory, two buffers)
//     P, dS in registers of eight warps (thread = row: lse, delta and the limit of the row are one value each), written as 16-bit operands
//     dV^T += dO^T P  and  dK^T += Q^T dS  (dims x 64 keys, accumulators in tensor memory for the whole item)
// with the same shared-memory bytes of Q and dO serving as row-major operand of the first pair and as transposed operand of the second.
// The tile after is multiplied while this one's P and dS are formed.  Every query names its keys by choice, so no row of a tile is
// wasted, however little neighbouring queries agree; this is what makes the 128-row instruction the right one here.
// Measured: 8192 queries, 32 heads of dim 128 over 4, 16 blocks of 64: 505 us, 3800 cycles a tile, of which the products take 2000: 62 each for 32 of
// arithmetic, because both operands come from shared memory (6 KB at 128 bytes a cycle).  Bound: a stage's round trip (gather 2200 cycles, S and D 1000, P and dS 1100, sums
// 1000) over the two stages that shared memory holds.
constexpr int kDkvWarps = 8, kDkvLoaders = 8;  // warps 0-7 form P and dS, 8-15 load, warp 16 multiplies
constexpr int kDkvThreads = (kDkvWarps + kDkvLoaders + 1) * 32;
constexpr int kDkvStages = 2;
constexpr uint32_t kTmemS = 0, kTmemD = 64, kTmemBuffer = 128, kTmemDv = 256, kTmemDk = 320, kTmemCols = 512;

template <int DP> struct DkvSmem {
    static constexpr int kHalves = DP / 64;
    static constexpr int kKeys = 0;                                     // 64 rows x 128 bytes per 64 dims
    static constexpr int kValues = kKeys + kHalves * 64 * 128;
    static constexpr int kTileBytes = kHalves * 128 * 128;              // 128 rows of q (or dout)
    static constexpr int kStage = kValues + kHalves * 64 * 128;         // per stage q, then dout
    static constexpr int kP = kStage + kDkvStages * 2 * kTileBytes;     // 128 rows x 64 keys
    static constexpr int kDs = kP + 128 * 128;
    static constexpr int kRows = kDs + 128 * 128;                       // per stage and row: lse log2 e, delta, a bit per key that it looks at
    static constexpr int kBars = kRows + kDkvStages * 128 * 16;
    static constexpr int kBytes = kBars + 16 * 8 + 16;
};

template <class T, int DP>
__global__ void __launch_bounds__(kDkvThreads, 1)
    block_attention_dkv_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, TurnArgs p)
{
    using S = DkvSmem<DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const AttentionArgs &a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::kBars);  // q, dout and the rows of a stage are there
    uint64_t *empty = full + kDkvStages;                             // the products that read the stage are done
    uint64_t *kv_full = empty + kDkvStages;
    uint64_t *scored = kv_full + 1;                                  // S and D of a buffer are complete (2)
    uint64_t *formed = scored + 2;                                   // P and dS are written
    uint64_t *used = formed + 1;                                     // the products that read P and dS are done
    uint64_t *summed = used + 1;                                     // an item's accumulators are complete
    uint64_t *read = summed + 1;                                     // ... and have been read
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + S::kBars + 16 * 8);  // [0] tensor memory, [1] gave up
    if (threadIdx.x == 0) {
        for (int s = 0; s < kDkvStages; ++s) {
            ptx::mbar_init(&full[s], kDkvLoaders);
            ptx::mbar_init(&empty[s], 1);
        }
        ptx::mbar_init(kv_full, 1);
        ptx::mbar_init(&scored[0], 1);
        ptx::mbar_init(&scored[1], 1);
        ptx::mbar_init(formed, kDkvWarps);
        ptx::mbar_init(used, 1);
        ptx::mbar_init(summed, 1);
        ptx::mbar_init(read, kDkvWarps);
        misc[1] = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 0) tc::alloc(const_cast<uint32_t *>(&misc[0]), kTmemCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = misc[0];
    ptx::grid_wait();
    ptx::grid_release();

    const uint32_t group = a.heads / a.kv_heads, per_tile = 128 / group;
    const uint32_t items = p.totals[0];
    uint32_t tile_count = 0;  // tiles of all items so far
    bool ok = true;
    auto tiles_of = [&](uint2 it) { return (item_part(p, it).y + per_tile - 1) / per_tile; };

    if (warp >= kDkvWarps && warp < kDkvWarps + kDkvLoaders) {
        // ================= loads: warps w and w + 4 look up rows 32 w .. 32 w + 31 of every tile, one brings q, one dout =================
        const uint32_t w = (warp - kDkvWarps) & 3, r = w * 32 + lane, entry = r / group, head = r % group;
        const bool is_q = warp - kDkvWarps < 4;
        const int64_t row_stride = is_q ? a.q_query : a.do_query;
        const uint32_t blocks_per_tile = a.block < kKeyTile ? kKeyTile / a.block : 1;
        uint32_t issued = 0, announced = 0;  // tiles whose copies are queued, and those the others know of
        // Announces the tile whose copies are in flight, if there is one.  Always before this warp waits for anything: what it waits for
        // comes from products that are queued behind those of that tile.
        auto announce = [&]() {
            if (issued == announced) return;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            ptx::fence_async_smem();  // the tensor cores read what this thread's copies wrote
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&full[announced % kDkvStages]);
            ++announced;
        };
        for (uint32_t k = 0, i = blockIdx.x; i < items && ok; i += gridDim.x, ++k) {
            const uint2 it = p.items[i];
            const uint32_t tile = it.x % p.tiles, bh = it.x / p.tiles, b = bh / a.kv_heads, kv = bh % a.kv_heads;
            const uint2 part = item_part(p, it);  // ranks among the queries that name the tile
            const uint32_t n_tiles = (part.y + per_tile - 1) / per_tile;
            announce();
            if (warp == kDkvWarps) {
                if (k && !(ok = ptx::mbar_wait_warp(summed, (k - 1) & 1u))) break;
                if (lane == 0) {
                    ptx::mbar_expect_tx(kv_full, 2 * S::kHalves * 64 * 128);
                    for (int h = 0; h < S::kHalves; ++h) {
                        tc::tma_load4(smem + S::kKeys + h * 64 * 128, &k_map, h * 64, (int)kv, (int)(tile * kKeyTile), (int)b, kv_full);
                        tc::tma_load4(smem + S::kValues + h * 64 * 128, &v_map, h * 64, (int)kv, (int)(tile * kKeyTile), (int)b, kv_full);
                    }
                }
                __syncwarp();
            }
            // a window of 32 words of the tile's bits, one per lane: `before` queries in front of this lane's word, `ranks` in front of the window
            uint32_t window = 0, word = 0, before = 0, size = 0, ranks = 0;
            auto take_window = [&]() {
                word = window + lane < p.words ? tile_word(p, it.x, window + lane) : 0u;
                before = __popc(word);
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t up = __shfl_up_sync(~0u, before, d);
                    if (lane >= (uint32_t)d) before += up;
                }
                size = __shfl_sync(~0u, before, 31);
                before -= __popc(word);
            };
            take_window();
            const T *row0 = is_q ? static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)(kv * group + head) * a.q_head
                                 : static_cast<const T *>(a.dout) + (int64_t)b * a.do_batch + (int64_t)(kv * group + head) * a.do_head;
            const uint64_t stat0 = ((uint64_t)b * a.heads + kv * group + head) * a.queries;
            for (uint32_t j = 0; j < n_tiles; ++j, ++tile_count) {
                // this lane's row: the query of rank part.x + j per_tile + entry
                const uint32_t local = j * per_tile + entry, rank = part.x + local;
                uint32_t t = a.queries;
                bool pending = entry < per_tile && local < part.y;
                for (;;) {
                    const bool here = pending && rank < ranks + size;
                    if (__any_sync(~0u, here)) {
                        const uint32_t at = here ? rank - ranks : 0u;
                        uint32_t l = 0;
#pragma unroll
                        for (int d = 16; d; d >>= 1)
                            if (__shfl_sync(~0u, before, l + d) <= at) l += d;
                        uint32_t bits = __shfl_sync(~0u, word, l), nth = at - __shfl_sync(~0u, before, l), bit = 0;
#pragma unroll
                        for (int d = 16; d; d >>= 1) {
                            const uint32_t c = __popc(bits & ((1u << d) - 1u));
                            if (nth >= c) {
                                nth -= c;
                                bits >>= d;
                                bit += d;
                            }
                        }
                        if (here) {
                            t = (window + l) * 32 + bit;
                            pending = false;
                        }
                    }
                    if (!__any_sync(~0u, pending) || window + 32 >= p.words) break;
                    ranks += size;
                    window += 32;
                    take_window();
                }
                const bool on = t < a.queries;
                float lse = 0.f, delta = 0.f;
                uint64_t sees = 0;
                if (on && is_q) {
                    lse = a.lse[stat0 + t] * kLog2e;
                    delta = a.delta[stat0 + t];
                    const int limit = (int)visible_keys(a, b, t) - (int)(tile * kKeyTile);
                    sees = limit >= 64 ? ~0ull : limit > 0 ? (1ull << limit) - 1ull : 0ull;
                    if (blocks_per_tile > 1) {
                        uint64_t named = 0;
                        const uint64_t one = (1ull << a.block) - 1ull;
                        for (uint32_t n = 0; n < blocks_per_tile && tile * blocks_per_tile + n < a.num_blocks; ++n)
                            if ((p.bits[((uint64_t)bh * a.num_blocks + tile * blocks_per_tile + n) * p.words + (t >> 5)] >> (t & 31)) & 1u) named |= one << (n * a.block);
                        sees &= named;
                    }
                }
                announce();  // the tile before has had all of this one's look-up to land
                const uint32_t s = tile_count % kDkvStages;
                if (!(ok = ptx::mbar_wait_warp(&empty[s], ((tile_count / kDkvStages) & 1u) ^ 1u))) break;
                if (is_q) reinterpret_cast<uint4 *>(smem + S::kRows)[s * 128 + r] = make_uint4(__float_as_uint(lse), __float_as_uint(delta), (uint32_t)sees, (uint32_t)(sees >> 32));
                const uint64_t row_at = reinterpret_cast<uint64_t>(row0 + (int64_t)(on ? t : 0u) * row_stride);
                const uint32_t to = ptx::smem_u32(smem + S::kStage) + (2 * s + (is_q ? 0 : 1)) * S::kTileBytes;
                constexpr uint32_t kPieces = DP / 8, kAtOnce = 32 / kPieces;  // 16-byte pieces of a row, rows of an instruction
                const uint32_t piece = lane % kPieces;
                const uint32_t rows_on = __ballot_sync(~0u, on);
#pragma unroll
                for (uint32_t x = 0; x < 32; x += kAtOnce) {
                    const uint32_t from = x + lane / kPieces;
                    const uint64_t src = __shfl_sync(~0u, row_at, from);
                    const uint32_t bytes = ((rows_on >> from) & 1u) && piece * 8 < a.dim ? 16u : 0u;  // 0: zeros
                    copy16(to + (piece >> 3) * 128 * 128 + tc::swizzled(w * 32 + from, piece & 7), bytes ? src + piece * 16 : reinterpret_cast<uint64_t>(a.q), bytes);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                ++issued;
            }
        }
        announce();
        if (!ok) {
            misc[1] = 1;
            if (warp == kDkvWarps && lane == 0)  // no copy stays in flight
                for (uint32_t x = 0; x < 2; ++x) ptx::mbar_wait(kv_full, x);
        }
    } else if (warp == kDkvWarps + kDkvLoaders) {
        // ================= products =================
        if (lane == 0) {
            constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
            constexpr uint32_t id_s = tc::idesc(bf16, 128, 64), id_t = tc::idesc(bf16, 128, 64, true, true);
            const uint32_t base = ptx::smem_u32(smem);
            // dims as rows: with 64 of them the second block of the 128-row instruction is the first once more, and its rows are left alone
            constexpr uint32_t block_bytes = DP == 128 ? 128 * 128 : 0;
            // every descriptor is one of these plus a constant
            const uint64_t q_k = tc::desc_k(base + S::kStage), k_k = tc::desc_k(base + S::kKeys), v_k = tc::desc_k(base + S::kValues);
            const uint64_t q_mn = tc::desc_mn(base + S::kStage, block_bytes), p_mn = tc::desc_mn(base + S::kP, 0), d_mn = tc::desc_mn(base + S::kDs, 0);
            constexpr uint32_t kTile = S::kTileBytes >> 4;
            uint32_t scores = 0, sums = 0;  // tiles whose first and second products are issued, over all items
            for (uint32_t k = 0, i = blockIdx.x; i < items && ok; i += gridDim.x, ++k) {
                const uint32_t first = scores, end = first + tiles_of(p.items[i]);
                if (!(ok = ptx::mbar_wait(kv_full, k & 1u))) break;
                // whichever is ready: the second products of a tile give its stage back, so they go first
                for (uint32_t idle = 0; sums < end;) {
                    if (sums < scores && ptx::mbar_test(formed, sums & 1u)) {
                        if (sums == first && k && !(ok = ptx::mbar_wait(read, (k - 1) & 1u))) break;
                        tc::fence_after();
                        const uint32_t s = sums % kDkvStages, at = s * 2 * kTile;
#pragma unroll
                        for (int r = 0; r < 8; ++r) tc::mma(tmem + kTmemDv, q_mn + (at + kTile + r * 128), p_mn + r * 128, id_t, sums != first || r);
#pragma unroll
                        for (int r = 0; r < 8; ++r) tc::mma(tmem + kTmemDk, q_mn + (at + r * 128), d_mn + r * 128, id_t, sums != first || r);
                        tc::commit(&empty[s]);
                        tc::commit(used);
                        if (++sums == end) tc::commit(summed);
                        idle = 0;
                    } else if (scores < end && scores < sums + 2 && ptx::mbar_test(&full[scores % kDkvStages], (scores / kDkvStages) & 1u)) {
                        tc::fence_after();
                        const uint32_t at = scores % kDkvStages * 2 * kTile, buffer = tmem + (scores & 1u) * kTmemBuffer;
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) tc::mma(buffer + kTmemS, q_k + (at + (d >> 2) * 1024 + (d & 3) * 2), k_k + ((d >> 2) * 512 + (d & 3) * 2), id_s, d != 0);
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) tc::mma(buffer + kTmemD, q_k + (at + kTile + (d >> 2) * 1024 + (d & 3) * 2), v_k + ((d >> 2) * 512 + (d & 3) * 2), id_s, d != 0);
                        tc::commit(&scored[scores & 1u]);
                        ++scores;
                        idle = 0;
                    } else if (++idle == kTcPolls) {
                        ok = false;
                        break;
                    }
                }
            }
            if (!ok) misc[1] = 1;
        }
    } else {
        // ================= P and dS =================
        const uint32_t r = (warp & 3) * 32 + lane, half = warp >> 2;
        const float scale_log2 = a.scale * kLog2e;
        const uint32_t lanes = tmem + (((warp & 3) * 32) << 16);
        for (uint32_t k = 0, i = blockIdx.x; i < items && ok; i += gridDim.x, ++k) {
            const uint2 it = p.items[i];
            const uint32_t tile = it.x % p.tiles, bh = it.x / p.tiles, b = bh / a.kv_heads, kv = bh % a.kv_heads;
            const uint32_t n_tiles = tiles_of(it);
            for (uint32_t j = 0; j < n_tiles; ++j, ++tile_count) {
                const uint32_t s = tile_count % kDkvStages;
                if (!(ok = ptx::mbar_wait_warp(&full[s], (tile_count / kDkvStages) & 1u))) break;
                const uint4 info = reinterpret_cast<const uint4 *>(smem + S::kRows)[s * 128 + r];
                const float lse = __uint_as_float(info.x), delta = __uint_as_float(info.y);
                const uint32_t sees = half ? info.w : info.z;  // a bit per key of this thread's half
                const uint32_t buffer = lanes + (tile_count & 1u) * kTmemBuffer + half * 32;
                if (!(ok = ptx::mbar_wait_warp(&scored[tile_count & 1u], (tile_count >> 1) & 1u))) break;
                tc::fence_after();
                uint32_t sv[32], dv[32];
                tc::ld32(buffer + kTmemS, sv);
                tc::ld32(buffer + kTmemD, dv);
                tc::wait_ld();
                uint32_t pp[16], dd[16];
                const uint64_t scale2 = ptx::pack2(scale_log2, scale_log2), minus2 = ptx::pack2(-lse, -lse), delta2 = ptx::pack2(-delta, -delta);
                const bool plain = __all_sync(~0u, sees == ~0u);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float2 x = ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), scale2, minus2));
                    const float2 e = make_float2(tc::exp2_fast(x.x), tc::exp2_fast(x.y));
                    const float2 y = ptx::unpack2(ptx::mul2(ptx::pack2(e.x, e.y), ptx::add2(ptx::pack2(__uint_as_float(dv[2 * c]), __uint_as_float(dv[2 * c + 1])), delta2)));
                    pp[c] = tc::round2<T>(e.x, e.y);
                    dd[c] = tc::round2<T>(y.x, y.y);
                }
                if (!plain) {  // keys that a row does not look at: zeros, whatever stands there
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const uint32_t keep = ((sees >> (2 * c)) & 1u ? 0xffffu : 0u) | ((sees >> (2 * c + 1)) & 1u ? 0xffff0000u : 0u);
                        pp[c] &= keep;
                        dd[c] &= keep;
                    }
                }
                if (tile_count && !(ok = ptx::mbar_wait_warp(used, (tile_count - 1) & 1u))) break;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t at = tc::swizzled(r, half * 4 + c);
                    *reinterpret_cast<uint4 *>(smem + S::kP + at) = make_uint4(pp[4 * c], pp[4 * c + 1], pp[4 * c + 2], pp[4 * c + 3]);
                    *reinterpret_cast<uint4 *>(smem + S::kDs + at) = make_uint4(dd[4 * c], dd[4 * c + 1], dd[4 * c + 2], dd[4 * c + 3]);
                }
                ptx::fence_async_smem();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(formed);
            }
            if (!ok) break;
            // ---- the item's sums: warps 0-3 dv, warps 4-7 dk; thread = dim ----
            if (!(ok = ptx::mbar_wait_warp(summed, k & 1u))) break;
            tc::fence_after();
            const bool is_dk = half != 0;
            const uint32_t d = r, n_items = (p.counts[it.x] + p.item_queries - 1) / p.item_queries;
            const float f = is_dk ? a.scale : 1.f;
            bool finite = true;
#pragma unroll 1
            for (uint32_t c = 0; c < 64; c += 32) {
                uint32_t v[32];
                tc::ld32(lanes + (is_dk ? kTmemDk : kTmemDv) + c, v);
                tc::wait_ld();
                if (d >= a.dim) continue;
#pragma unroll
                for (int x = 0; x < 32; ++x) finite = finite && fabsf(__uint_as_float(v[x])) < INFINITY;
                if (n_items == 1) {
                    T *dst = static_cast<T *>(is_dk ? a.dk : a.dv) + (((uint64_t)b * a.keys + tile * kKeyTile + c) * a.kv_heads + kv) * a.dim + d;
                    const uint32_t n = a.keys > tile * kKeyTile + c ? min(32u, a.keys - tile * kKeyTile - c) : 0u;
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if ((uint32_t)x < n) dst[(uint64_t)x * a.kv_heads * a.dim] = from_f32<T>(f * __uint_as_float(v[x]));
                } else {
                    float *dst = p.partial + (((uint64_t)p.first_slot[it.x] + it.y) * 2 + (is_dk ? 1 : 0)) * kKeyTile * DP + c * DP + d;
#pragma unroll
                    for (int x = 0; x < 32; ++x) __stcs(dst + x * DP, f * __uint_as_float(v[x]));
                }
            }
            if (__any_sync(~0u, !finite) && lane == 0) p.redo[it.x] = 1;
            tc::fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(read);
        }
        if (!ok) misc[1] = 1;
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && misc[1]) atomicExch(&g_status, 2u);
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tmem, kTmemCols);
    }
}

// dk and dv of one key by themselves: a warp, four dims a lane, over the queries that look at the key, in ascending order.
template <class T> __device__ __forceinline__ void exact_key(const TurnArgs &p, uint32_t b, uint32_t kv, uint32_t key, float (&dk)[4], float (&dv)[4])
{
    const AttentionArgs &a = p.a;
    const uint32_t lane = threadIdx.x & 31, d = lane * 4, group = a.heads / a.kv_heads;
    const bool on = d < a.dim;
    const T *kr = key_row<T>(a, a.k, a.k_batch, a.k_key, a.k_head, b, kv, key) + d, *vr = key_row<T>(a, a.v, a.v_batch, a.v_key, a.v_head, b, kv, key) + d;
    float k[4] = {}, v[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        dk[j] = dv[j] = 0.f;
        if (on) {
            k[j] = to_f32(kr[j]);
            v[j] = to_f32(vr[j]);
        }
    }
    const uint32_t *bits = p.bits + (((uint64_t)b * a.kv_heads + kv) * a.num_blocks + key / a.block) * p.words;
    for (uint32_t w = 0; w < p.words; w += 32) {
        const uint32_t mine = w + lane < p.words ? bits[w + lane] : 0u;
        for (uint32_t some = __ballot_sync(~0u, mine != 0); some; some &= some - 1) {
            const uint32_t l = __ffs(some) - 1;
            for (uint32_t word = __shfl_sync(~0u, mine, l); word; word &= word - 1) {
                const uint32_t t = (w + l) * 32 + __ffs(word) - 1;
                if (key >= visible_keys(a, b, t)) continue;
                for (uint32_t head = kv * group; head < (kv + 1) * group; ++head) {
                    const T *qr = static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)t * a.q_query + (int64_t)head * a.q_head + d;
                    const T *gr = static_cast<const T *>(a.dout) + (int64_t)b * a.do_batch + (int64_t)t * a.do_query + (int64_t)head * a.do_head + d;
                    float q[4] = {}, g[4] = {}, s = 0.f, dp = 0.f;
                    if (on)
                        for (int j = 0; j < 4; ++j) {
                            q[j] = to_f32(qr[j]);
                            g[j] = to_f32(gr[j]);
                            s = fmaf(q[j], k[j], s);
                            dp = fmaf(g[j], v[j], dp);
                        }
#pragma unroll
                    for (int x = 16; x; x >>= 1) {
                        s += __shfl_xor_sync(~0u, s, x);
                        dp += __shfl_xor_sync(~0u, dp, x);
                    }
                    const uint64_t stat = ((uint64_t)b * a.heads + head) * a.queries + t;
                    const float e = exp2f((s * a.scale - a.lse[stat]) * kLog2e), ds = a.scale * e * (dp - a.delta[stat]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dk[j] = fmaf(ds, q[j], dk[j]);
                        dv[j] = fmaf(e, g[j], dv[j]);
                    }
                }
                bool lost = true;  // what is no number stays none
                for (int j = 0; j < 4; ++j) lost = lost && dk[j] != dk[j] && dv[j] != dv[j];
                if (__all_sync(~0u, lost || !on)) return;
            }
        }
    }
}

// Key tiles that no query names are zero; the partial sums of those with several work items are added in order.  Eight blocks of threads a tile.
// In a tile that has a sum which is not finite, a warp takes a key: the products multiply every gathered row of q and dout with all 64 keys, and 0 times
// a row that is no number is not 0, so such a key is formed again from the queries that look at it.
template <class T, int DP> __global__ void __launch_bounds__(256) dkv_join_kernel(TurnArgs p)
{
    ptx::grid_wait();
    ptx::grid_release();
    const AttentionArgs &a = p.a;
    const uint32_t row = blockIdx.x, items = (p.counts[row] + p.item_queries - 1) / p.item_queries;
    const bool redo = p.redo[row] != 0;
    if (items == 1 && !redo) return;
    const uint32_t tile = row % p.tiles, bh = row / p.tiles, b = bh / a.kv_heads, kv = bh % a.kv_heads;
    const uint32_t n = min(kKeyTile, a.keys - tile * kKeyTile);
    const float *src = p.partial + (uint64_t)p.first_slot[row] * 2 * kKeyTile * DP;
    if (redo) {
        const uint32_t d = (threadIdx.x & 31) * 4;
        for (uint32_t key = blockIdx.y * 8 + (threadIdx.x >> 5); key < n; key += 8 * gridDim.y) {
            const uint64_t at = (((uint64_t)b * a.keys + tile * kKeyTile + key) * a.kv_heads + kv) * a.dim + d;
            T *to_dk = static_cast<T *>(a.dk) + at, *to_dv = static_cast<T *>(a.dv) + at;
            float dk[4] = {}, dv[4] = {};
            if (d < a.dim && items == 1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    dk[j] = to_f32(to_dk[j]);
                    dv[j] = to_f32(to_dv[j]);
                }
            } else if (d < a.dim)
                for (uint32_t k = 0; k < items; ++k) {
                    const float *part = src + (uint64_t)k * 2 * kKeyTile * DP + key * DP + d;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dv[j] += part[j];
                        dk[j] += part[kKeyTile * DP + j];
                    }
                }
            bool finite = true;
#pragma unroll
            for (int j = 0; j < 4; ++j) finite = finite && fabsf(dk[j]) < INFINITY && fabsf(dv[j]) < INFINITY;
            if (!__all_sync(~0u, finite)) exact_key<T>(p, b, kv, tile * kKeyTile + key, dk, dv);
            if (d < a.dim) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    to_dk[j] = from_f32<T>(dk[j]);
                    to_dv[j] = from_f32<T>(dv[j]);
                }
            }
        }
        return;
    }
    for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < 2 * n * (DP / 4); i += 256 * gridDim.y) {
        const uint32_t d = i % (DP / 4) * 4, key = i / (DP / 4) % n, is_dk = i / (DP / 4) / n;
        if (d >= a.dim) continue;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t k = 0; k < items; ++k) {
            const float4 x = __ldcs(reinterpret_cast<const float4 *>(src + ((uint64_t)k * 2 + is_dk) * kKeyTile * DP + key * DP + d));
            sum.x += x.x;
            sum.y += x.y;
            sum.z += x.z;
            sum.w += x.w;
        }
        T *dst = static_cast<T *>(is_dk ? a.dk : a.dv) + (((uint64_t)b * a.keys + tile * kKeyTile + key) * a.kv_heads + kv) * a.dim + d;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(tc::round2<T>(sum.x, sum.y), tc::round2<T>(sum.z, sum.w));
    }
}

template <class T, int DP> cudaError_t launch_dq(const AttentionArgs &a, cudaStream_t s)
{
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    TcShape shape = tc_shape(a.heads / a.kv_heads, 64);
    uint32_t bytes = 0;  // fewer queries where their lists are too long
    for (;; shape.queries /= 2)
        if ((bytes = DqSmem<DP>::kLists + TileUnion::bytes(shape.queries, a.count, a.block, a.keys)) <= kSmemMost || shape.queries == 1) break;
    CUtensorMap k_map{}, v_map{};
    cudaError_t e = cudaSuccess;
    if (a.keys) {
        e = tc::make_map(&k_map, bf16, a.k, a.dim, a.kv_heads, a.keys, a.batch, a.k_head, a.k_key, a.k_batch, 64);
        if (e == cudaSuccess) e = tc::make_map(&v_map, bf16, a.v, a.dim, a.kv_heads, a.keys, a.batch, a.v_head, a.v_key, a.v_batch, 64);
    }
    if (e == cudaSuccess) e = allow_dynamic_smem<block_attention_dq_kernel<T, DP>>(kSmemMost);
    if (e != cudaSuccess) return e;
    const dim3 grid((a.queries + shape.queries - 1) / shape.queries, a.kv_heads * shape.chunks, a.batch);
    return launch_overlapped(block_attention_dq_kernel<T, DP>, grid, dim3(kDqThreads), bytes, s, k_map, v_map, a, shape);
}

template <class T, int DP> cudaError_t launch_grad(AttentionArgs a, int sm_count, cudaStream_t s)
{
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const GradLayout l(a);
    char *w = static_cast<char *>(a.workspace);
    a.delta = reinterpret_cast<float *>(w + l.delta);
    cudaError_t e = launch_dq<T, DP>(a, s);
    if (e != cudaSuccess || !a.keys) return e;
    TurnArgs p{};
    p.a = a;
    p.words = l.words;
    p.tiles = l.tiles;
    p.item_queries = l.item_queries;
    p.tile_rows = l.tile_rows;
    p.bits = reinterpret_cast<uint32_t *>(w + l.bits);
    p.counts = reinterpret_cast<uint32_t *>(w + l.counts);
    p.first_item = p.counts + l.tile_rows;
    p.first_slot = p.first_item + l.tile_rows;
    p.redo = p.first_slot + l.tile_rows;
    p.items = reinterpret_cast<uint2 *>(w + l.items);
    p.totals = reinterpret_cast<uint32_t *>(w + l.totals);
    p.partial = reinterpret_cast<float *>(w + l.partial);
    if ((e = cudaMemsetAsync(p.bits, 0, l.bits_bytes, s)) != cudaSuccess) return e;
    const uint64_t bit_warps = (uint64_t)a.batch * a.kv_heads * l.words;
    if ((e = launch_overlapped(pattern_bits_kernel, dim3((unsigned)((bit_warps + 7) / 8)), dim3(256), 0, s, p)) != cudaSuccess) return e;
    if ((e = launch_overlapped(pattern_count_kernel, dim3((unsigned)((l.tile_rows + 7) / 8)), dim3(256), 0, s, p)) != cudaSuccess) return e;
    if ((e = launch_overlapped(pattern_items_kernel, dim3(1), dim3(1024), 0, s, p)) != cudaSuccess) return e;
    CUtensorMap k_map, v_map;
    if ((e = tc::make_map(&k_map, bf16, a.k, a.dim, a.kv_heads, a.keys, a.batch, a.k_head, a.k_key, a.k_batch, kKeyTile)) != cudaSuccess) return e;
    if ((e = tc::make_map(&v_map, bf16, a.v, a.dim, a.kv_heads, a.keys, a.batch, a.v_head, a.v_key, a.v_batch, kKeyTile)) != cudaSuccess) return e;
    if ((e = allow_dynamic_smem<block_attention_dkv_kernel<T, DP>>(DkvSmem<DP>::kBytes)) != cudaSuccess) return e;
    const uint64_t blocks = l.max_items < (uint64_t)sm_count ? l.max_items : (uint64_t)sm_count;
    if ((e = launch_overlapped(block_attention_dkv_kernel<T, DP>, dim3((unsigned)blocks), dim3(kDkvThreads), DkvSmem<DP>::kBytes, s, k_map, v_map, p)) != cudaSuccess) return e;
    return launch_overlapped(dkv_join_kernel<T, DP>, dim3((unsigned)l.tile_rows, 8), dim3(256), 0, s, p);
}

}  // namespace

// Whether some query may look at some key; without one there is no pattern to turn round, and sizes that the layout divides by are zero.
static bool has_pairs(const AttentionArgs &a) { return a.batch && a.queries && a.heads && a.count; }

uint64_t block_attention_grad_workspace(const AttentionArgs &a) { return has_pairs(a) ? GradLayout(a).total : 0; }

cudaError_t launch_block_attention_grad(const AttentionArgs &a, int sm_count, cudaStream_t s)
{
    if (!has_pairs(a)) {  // nobody looks at any key
        const uint64_t kv_bytes = (uint64_t)a.batch * a.keys * a.kv_heads * a.dim * 2, q_bytes = (uint64_t)a.batch * a.queries * a.heads * a.dim * 2;
        cudaError_t e = cudaSuccess;
        if (kv_bytes && (e = cudaMemsetAsync(a.dk, 0, kv_bytes, s)) == cudaSuccess) e = cudaMemsetAsync(a.dv, 0, kv_bytes, s);
        if (e == cudaSuccess && q_bytes) e = cudaMemsetAsync(a.dq, 0, q_bytes, s);
        return e;
    }
    if (a.dtype == CUTESPMM_BF16) return a.dim <= 64 ? launch_grad<__nv_bfloat16, 64>(a, sm_count, s) : launch_grad<__nv_bfloat16, 128>(a, sm_count, s);
    return a.dim <= 64 ? launch_grad<__half, 64>(a, sm_count, s) : launch_grad<__half, 128>(a, sm_count, s);
}

cudaError_t block_attention_grad_status(uint32_t *word) { return read_status(g_status, word); }

}  // namespace cutespmm
