// Attention over selected blocks, forward: out = softmax(scale q K^T) V over the visible keys of the blocks that each query names.
//
// Two kernels.  A tile of neighbouring queries shares the blocks that several of them name: block_attention_kernel, on tcgen05.  A single
// token (or few) has its blocks split over the warps of up to eight thread blocks: block_attention_split_kernel, on mma.sync.
//
// Softmax with a running maximum and sum per row, in fp32.  P is rounded to the 16-bit type for the second product, because the tensor cores
// multiply 16-bit values by 16-bit values only (as tf32 the product would run at half the rate and V would have to be widened): half a step
// per term, u sum p |v| at most beside the u |out| of the result's own rounding; the sum is taken before it.  Against 64 bits out is 2.2e-3 off in
// bf16 where fp32 throughout is 1.6e-3 (16384 queries, 32 blocks of 64), 2.6e-4 for 2.0e-4 in fp16.  A key that a query does not look at never touches its result, whatever stands there.
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

// A unit of keys of the single-token kernel in shared memory: DP / 64 tiles of 16 rows x 128 bytes (swizzled) of keys, then the same of values.
constexpr int kSplitUnit = 16;
template <int DP> constexpr int kHalfBytes = DP / 64 * kSplitUnit * 128;
template <int DP> constexpr int kUnitBytes = 2 * kHalfBytes<DP>;

template <int DP>
__device__ __forceinline__ void load_unit(unsigned char *stage, const CUtensorMap *k_map, const CUtensorMap *v_map, int kv, int row, int outer, uint64_t *bar)
{
    ptx::mbar_expect_tx(bar, kUnitBytes<DP>);
#pragma unroll
    for (int h = 0; h < DP / 64; ++h) tc::tma_load4(stage + h * kSplitUnit * 128, k_map, h * 64, kv, row, outer, bar);
#pragma unroll
    for (int h = 0; h < DP / 64; ++h) tc::tma_load4(stage + kHalfBytes<DP> + h * kSplitUnit * 128, v_map, h * 64, kv, row, outer, bar);
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
    __device__ void softmax(const float (&s)[4], uint32_t (&p)[2], float scale_log2)
    {
        float m0 = fmaxf(s[0], s[2]), m1 = fmaxf(s[1], s[3]);
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
        const float e0 = tc::exp2_fast(fmaf(s[0], scale_log2, -b0)), e1 = tc::exp2_fast(fmaf(s[1], scale_log2, -b1));
        const float e2 = tc::exp2_fast(fmaf(s[2], scale_log2, -b0)), e3 = tc::exp2_fast(fmaf(s[3], scale_log2, -b1));
        sum[0] += e0 + e2;
        sum[1] += e1 + e3;
        p[0] = tc::transpose8x8(tc::round2<T>(e0, e1));
        p[1] = tc::transpose8x8(tc::round2<T>(e2, e3));
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

// Operand A of the first product: the 16 keys of a unit, dims 16 s.
__device__ __forceinline__ uint32_t keys_at(uint32_t keys, int s, uint32_t lane) { return keys + (s >> 2) * kSplitUnit * 128 + tc::swizzled(lane & 15, (s & 3) * 2 + (lane >> 4)); }
// Operand A of the second product, transposed on the way: dims 16 d.
__device__ __forceinline__ uint32_t values_at(uint32_t values, int d, uint32_t lane)
{
    return values + (d >> 2) * kSplitUnit * 128 + tc::swizzled(((lane >> 4) << 3) + (lane & 7), (d & 3) * 2 + ((lane >> 3) & 1));
}

// ---- a tile of queries -------------------------------------------------------------------------------------------------
// 128 rows -- neighbouring queries with all heads of a group (or a chunk of them) -- against the union of the tiles of 64 keys that they name:
//     S = Q K^T (128 x 64, two buffers in tensor memory);  P from registers back into S's columns as 16-bit operand;  O += P V.
// Warps 0-3 hold a row each lane (a row's maximum and sum need no other lane), warp 4 loads, warp 5 issues S, warp 6 O: one warp for both
// spent a third of a tile's time between them.
// Rows whose query does not name a tile have P = 0 there.  Multiplying only what is named, on mma.sync with a query's eight heads as the columns of
// an instruction, was slower for every group, block size and dim tried with the blocks of a selection: 8192 queries, 32 heads, 16 blocks of 64, where
// 16 neighbouring queries name 241 blocks, 40 of them distinct, 1290 us against 407 (in ncu captures 1183 against 341); 4096 queries, one head to a group, 16 blocks of 16 302 against 94.
// The maximum is raised only when a score exceeds it by 8 (of the base-2 exponent), so that O is rescaled in tensor memory a few times per row instead of once per
// tile; P is then at most 256 and out, a quotient, the same.  Two blocks of threads share an SM while their lists
// leave room (17 KB each for dims beyond 64, 66 KB below): one multiplies while the other's rows are at work.  Many short blocks a query in a long cache take more --
// one head to a group, 16 blocks of 16 among 32768 keys: 35 KB -- and then a block has its SM to itself; a tile gets smaller only where its lists would not fit at all.
// 0 times a value that is no number is not 0: rows of V behind the last visible key are zeroed as they land, and a row whose result is
// not finite is formed again, key by key, from what its query looks at (exact_row).
// Measured, forward alone: 8192 queries, 32 heads of dim 128 over 4 heads of keys, 16 blocks of 64: 354 to 410 us (tensor pipe 45 % busy, issue slots 36 %);
// 16384 queries, 16 heads over 2, 32 blocks: 717 us.  Bound: a row's way from S to P (1100 cycles a tile, half of it exponentials), twice on an SM.
constexpr int kTcThreads = 224;
constexpr int kTcStages = 2;  // of keys, of values, and of S in tensor memory
constexpr uint32_t kTcO = 128, kTcCols = 256;  // columns of tensor memory: two buffers of S, O
constexpr float kRaise = 8.f;                  // log2

template <int DP> struct TcSmem {
    static constexpr int kHalves = DP / 64;
    static constexpr int kQ = 0;
    static constexpr int kRing = kHalves * 128 * 128;
    static constexpr int kTile = kHalves * 64 * 128;      // keys of a stage, or its values
    static constexpr int kBars = kRing + 2 * kTcStages * kTile;  // stages of keys, then of values
    static constexpr int kLists = kBars + 144;
};

// One row by itself: a warp, four dims a lane, over the keys its query looks at.
template <class T> __device__ void exact_row(const AttentionArgs &a, const TileUnion &u, uint32_t b, uint32_t kv, uint32_t t, uint32_t q_of_tile, uint32_t head)
{
    const uint32_t lane = threadIdx.x & 31, d = lane * 4;
    const bool on = d < a.dim;
    const T *qr = static_cast<const T *>(a.q) + (int64_t)b * a.q_batch + (int64_t)t * a.q_query + (int64_t)head * a.q_head + d;
    float q[4] = {}, o[4] = {}, top = -INFINITY, sum = 0.f;
    if (on)
        for (int j = 0; j < 4; ++j) q[j] = to_f32(qr[j]);
    for (uint32_t slot = 0; slot < *u.size; ++slot)
        for (uint64_t seen = u.seen(slot, q_of_tile, a.block); seen; seen &= seen - 1) {
            const uint32_t key = u.tiles[slot] * kKeyTile + __ffsll((long long)seen) - 1;
            const T *kr = key_row<T>(a, a.k, a.k_batch, a.k_key, a.k_head, b, kv, key) + d, *vr = key_row<T>(a, a.v, a.v_batch, a.v_key, a.v_head, b, kv, key) + d;
            float s = 0.f;
            if (on)
                for (int j = 0; j < 4; ++j) s = fmaf(q[j], to_f32(kr[j]), s);
#pragma unroll
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
            s *= a.scale * kLog2e;
            const float m = fmaxf(top, s), base = m == -INFINITY ? 0.f : m, f = exp2f(top - base), p = exp2f(s - base);
            sum = sum * f + p;
            for (int j = 0; j < 4; ++j) o[j] = o[j] * f + (on ? p * to_f32(vr[j]) : 0.f);
            top = m;
        }
    const uint64_t row = ((uint64_t)b * a.queries + t) * a.heads + head;
    if (on)
        for (int j = 0; j < 4; ++j) static_cast<T *>(a.out)[row * a.dim + d + j] = from_f32<T>(sum != 0.f ? o[j] / sum : 0.f);
    if (lane == 0) a.lse[((uint64_t)b * a.heads + head) * a.queries + t] = sum != 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

template <class T, int DP>
__global__ void __launch_bounds__(kTcThreads, 2) block_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap q_map, AttentionArgs a, TcShape shape)
{
    using S = TcSmem<DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // keys are given back when S is complete, values when O is: a tile's keys are on their way while the one before is summed
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + S::kBars), *v_full = k_full + kTcStages, *scored = v_full + kTcStages, *formed = scored + kTcStages, *summed = formed + kTcStages, *q_full = summed + kTcStages, *landed = q_full + 1;
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(landed + 1);  // [0] tensor memory, [1] gave up
    TileUnion u(smem + S::kLists, shape.queries, a);
    const uint32_t t0 = blockIdx.x * shape.queries, b = blockIdx.z;
    const uint32_t kv = blockIdx.y / shape.chunks, group = a.heads / a.kv_heads, head0 = blockIdx.y % shape.chunks * shape.heads;
    const uint32_t heads = min(shape.heads, group - head0), queries = min(shape.queries, a.queries - t0);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kTcStages; ++s) {
            ptx::mbar_init(&k_full[s], 1);
            ptx::mbar_init(&v_full[s], 1);
            ptx::mbar_init(&scored[s], 1);
            ptx::mbar_init(&formed[s], 4);  // per buffer: a warp without work may be a tile ahead of the others
            ptx::mbar_init(&summed[s], 1);
        }
        ptx::mbar_init(q_full, 1);
        ptx::mbar_init(landed, 1);
        misc[1] = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 0) tc::alloc(const_cast<uint32_t *>(&misc[0]), kTcCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = misc[0];
    ptx::grid_wait();
    ptx::grid_release();
    if (warp == 4 && lane == 0) {
        ptx::mbar_expect_tx(q_full, S::kHalves * shape.queries * shape.heads * 128);
        for (int h = 0; h < S::kHalves; ++h) tc::tma_load4(smem + S::kQ + h * 128 * 128, &q_map, h * 64, (int)(kv * group + head0), (int)t0, (int)b, q_full);
    }
    u.build(a, b, kv, t0, queries);
    const uint32_t units = *u.size;

    bool ok = true;
    if (warp == 4) {
        uint32_t phase = 0, i = 0;
        for (; i < units; ++i) {
            const uint32_t s = i % kTcStages;
            const uint32_t parity = ((i / kTcStages) & 1u) ^ 1u;
            unsigned char *keys = smem + S::kRing + s * S::kTile;
            if (!(ok = ptx::mbar_wait_warp(&scored[s], parity) && load_key_tile<DP>(keys, &k_map, a, b, kv, u.tiles[i], u.size[1], shape.box_rows, &k_full[s], landed, phase))) break;
            if (!(ok = ptx::mbar_wait_warp(&summed[s], parity) && load_key_tile<DP>(keys + kTcStages * S::kTile, &v_map, a, b, kv, u.tiles[i], u.size[1], shape.box_rows, &v_full[s], landed, phase))) break;
        }
        if (!ok) {
            misc[1] = 1;
            if (lane == 0) {  // no copy stays in flight
                ptx::mbar_wait(q_full, 0);
                for (uint32_t j = i > kTcStages ? i - kTcStages : 0; j <= i && j < units; ++j) {  // of tile i perhaps the keys alone: that wait runs out
                    ptx::mbar_wait(&k_full[j % kTcStages], (j / kTcStages) & 1u);
                    if (j < i) ptx::mbar_wait(&v_full[j % kTcStages], (j / kTcStages) & 1u);
                }
            }
        } else if (!units && lane == 0)
            ok = ptx::mbar_wait(q_full, 0);
    } else if (warp == 5) {
        if (lane == 0 && units) {
            constexpr uint32_t id = tc::idesc(std::is_same<T, __nv_bfloat16>::value, 128, 64);
            const uint32_t base = ptx::smem_u32(smem);
            const uint64_t q_k = tc::desc_k(base + S::kQ), k_k = tc::desc_k(base + S::kRing);
            ok = ptx::mbar_wait(q_full, 0);
            for (uint32_t i = 0; ok && i < units; ++i) {
                const uint32_t s = i % kTcStages, parity = (i / kTcStages) & 1u;
                // the buffer held P two tiles ago
                if (!(ok = ptx::mbar_wait(&k_full[s], parity) && ptx::mbar_wait(&summed[s], parity ^ 1u))) break;
                tc::fence_after();
                const uint32_t at = s * (S::kTile >> 4);
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) tc::mma(tmem + s * 64, q_k + ((d >> 2) * 1024 + (d & 3) * 2), k_k + (at + (d >> 2) * 512 + (d & 3) * 2), id, d != 0);
                tc::commit(&scored[s]);
            }
            if (!ok) misc[1] = 1;
        }
    } else if (warp == 6) {
        if (lane == 0) {
            constexpr uint32_t id = tc::idesc(std::is_same<T, __nv_bfloat16>::value, 128, DP, false, true);
            const uint64_t v_mn = tc::desc_mn(ptx::smem_u32(smem) + S::kRing + kTcStages * S::kTile, 64 * 128);
            for (uint32_t i = 0; i < units; ++i) {
                const uint32_t s = i % kTcStages, parity = (i / kTcStages) & 1u, at = s * (S::kTile >> 4);
                if (!(ok = ptx::mbar_wait(&v_full[s], parity) && ptx::mbar_wait(&formed[s], parity))) break;
                tc::fence_after();
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma_ta(tmem + kTcO, tmem + s * 64 + k * 8, v_mn + (at + k * 128), id, i || k);
                tc::commit(&summed[s]);
            }
            if (!ok) misc[1] = 1;
        }
    } else {
        const uint32_t r = threadIdx.x, q = r / shape.heads, h = r % shape.heads, head = kv * group + head0 + h;
        const bool real = q < queries && h < heads;
        const uint32_t lanes = tmem + ((warp * 32) << 16);
        const float scale_log2 = a.scale * kLog2e;
        float top = -INFINITY, sum = 0.f;
        for (uint32_t i = 0; i < units; ++i) {
            const uint64_t seen = real ? u.seen(i, q, a.block) : 0ull;
            const uint32_t buffer = lanes + (i & 1u) * 64;
            if (!(ok = ptx::mbar_wait_warp(&scored[i & 1u], (i >> 1) & 1u))) break;
            tc::fence_after();
            uint32_t p[32];
            if (__any_sync(~0u, seen != 0)) {
                uint32_t v[64];
                tc::ld32(buffer, reinterpret_cast<uint32_t(&)[32]>(v[0]));
                tc::ld32(buffer + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
                tc::wait_ld();
                const bool plain = __all_sync(~0u, seen == 0 || seen == ~0ull);
                if (!plain) {
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (!((uint32_t)(seen >> (c & 32)) & (1u << (c & 31)))) v[c] = 0xff800000u;
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains: one of 64 would be the latency of 64 instructions
#pragma unroll
                for (int c = 0; c < 64; c += 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) m4[x] = ptx::max3(m4[x], __uint_as_float(v[c + 2 * x]), __uint_as_float(v[c + 2 * x + 1]));
                float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                m *= scale_log2;
                bool raise = false;
                float f = 1.f;
                if (seen) {
                    if (top == -INFINITY) top = m;  // nothing summed yet
                    else if (m > top + kRaise) {
                        raise = true;
                        f = tc::exp2_fast(top - m);
                        top = m;
                        sum *= f;
                    }
                }
                if (__any_sync(~0u, raise)) {
                    if (!(ok = ptx::mbar_wait_warp(&summed[(i - 1) & 1u], ((i - 1) >> 1) & 1u))) break;  // the products in flight add to O
                    tc::fence_after();
#pragma unroll 1
                    for (uint32_t c = 0; c < DP; c += 32) {
                        uint32_t o[32];
                        tc::ld32(lanes + kTcO + c, o);
                        tc::wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        tc::st32(lanes + kTcO + c, o);
                    }
                }
                // a row that does not name the tile: every exponential is 0 (a score that is no number makes its result none, and that is formed again)
                const float minus = !seen ? -INFINITY : top == -INFINITY ? 0.f : -top;
                const uint64_t scale2 = ptx::pack2(scale_log2, scale_log2), minus2 = ptx::pack2(minus, minus);
                uint64_t part[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    const float2 x = ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), scale2, minus2));
                    const float e0 = tc::exp2_fast(x.x), e1 = tc::exp2_fast(x.y);
                    part[c & 1] = ptx::add2(part[c & 1], ptx::pack2(e0, e1));
                    p[c] = tc::round2<T>(e0, e1);
                }
                const float2 both = ptx::unpack2(ptx::add2(part[0], part[1]));
                sum += both.x + both.y;
                __syncwarp();
            } else {
#pragma unroll
                for (int c = 0; c < 32; ++c) p[c] = 0;
            }
            tc::st32(buffer, p);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&formed[i & 1u]);
        }
        if (ok && units) ok = ptx::mbar_wait_warp(&summed[(units - 1) & 1u], ((units - 1) >> 1) & 1u);
        tc::fence_after();
        if (!ok) misc[1] = 1;
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        T *row = static_cast<T *>(a.out) + (((uint64_t)b * a.queries + t0 + q) * a.heads + head) * a.dim;
        bool finite = sum < INFINITY;
#pragma unroll 1
        for (uint32_t c = 0; c < DP; c += 32) {
            uint32_t o[32];
            if (units) {
                tc::ld32(lanes + kTcO + c, o);
                tc::wait_ld();
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float o0 = units ? __uint_as_float(o[8 * x + 2 * y]) : 0.f, o1 = units ? __uint_as_float(o[8 * x + 2 * y + 1]) : 0.f;
                    finite = finite && fabsf(o0) < INFINITY && fabsf(o1) < INFINITY;
                    w[y] = tc::round2<T>(o0 * inv, o1 * inv);
                }
                if (real && c + 8 * x < a.dim) *reinterpret_cast<uint4 *>(row + c + 8 * x) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if (real) a.lse[((uint64_t)b * a.heads + head) * a.queries + t0 + q] = sum > 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        for (uint32_t left = __ballot_sync(~0u, real && !finite); left && !misc[1]; left &= left - 1) {
            const uint32_t from = __ffs(left) - 1, rq = __shfl_sync(~0u, q, from), rh = __shfl_sync(~0u, head, from);
            __syncwarp();
            exact_row<T>(a, u, b, kv, t0 + rq, rq, rh);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && misc[1]) atomicExch(&g_status, 1u);
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tmem, kTcCols);
    }
}

// ---- a single token ----------------------------------------------------------------------------------------------------
// The products are formed transposed, S^T = K Q^T and O^T = V^T P^T: keys and dims are the 16 rows of an instruction and the group's heads its eight columns.
// One query's heads of one head of keys: its blocks, in pieces of 16 keys, are dealt over the warps of a cluster of thread blocks.  A
// warp fills a ring of its own (its lane 0 issues the loads) and keeps its own softmax state; the states are joined in the
// order of the warps, first inside a thread block, then over the cluster through distributed shared memory: no scratch, no counters, one
// launch.  Bound: HBM (the named blocks once) in batches: 64 tokens, 64 heads over 8, 48 blocks of 64 keys of a paged cache 148 us, 5.4 TB/s (one thread block
// an SM with rings twice as deep: 214 us).  A chain of latencies for one sequence: 8 us.
constexpr int kSplitWarps = 4;
template <int DP> constexpr int kSplitStages = DP == 128 ? 2 : 4;  // 64 KB of keys and values: three thread blocks share an SM
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
    static constexpr int kStage = kUnitBytes<DP>;
    static constexpr int kRings = kSplitWarps * kSplitStages<DP> * kStage;
    static constexpr int kPitch = DP + 4;                                      // floats of a column of a partial result
    static constexpr int kRing = kSplitStages<DP> * kStage;                    // of a warp; its partial result takes the ring's place
    static_assert(8 * NT * kPitch * 4 <= kRing, "a warp's partial result fits its ring");
    static constexpr int kStats = kRings;                                      // per warp and column: maximum, sum
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
    uint32_t *list = reinterpret_cast<uint32_t *>(smem + S::kList), *first_of = list + kSplitCount;
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
    __syncthreads();

    const uint32_t per_block = a.block / kSplitUnit, units = total * per_block;
    const uint32_t walkers = ranks * kSplitWarps, me = warp * ranks + rank;  // neighbouring units go to different thread blocks
    const uint32_t mine_units = units > me ? (units - me + walkers - 1) / walkers : 0u;
    unsigned char *ring = smem + warp * S::kRing;
    auto issue = [&](uint32_t i) {
        const uint32_t n = me + i * walkers;
        int row, outer;
        unit_place(a, b, list[n / per_block], n % per_block * kSplitUnit, row, outer);
        load_unit<DP>(ring + i % STAGES * S::kStage, &k_map, &v_map, (int)kv, row, outer, &full[i % STAGES]);
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
        if (!ptx::mbar_wait_warp(&full[s], (i / STAGES) & 1u)) {  // later loads of this ring land before the block ends, or their waits give up too
            if (lane == 0) atomicExch(&g_status, 1u);
            continue;
        }
        const int limit = (int)visible - (int)(list[n / per_block] * a.block + n % per_block * kSplitUnit);
        if (limit > 0) {
            const uint32_t keys = ptx::smem_u32(ring + s * S::kStage), values = keys + kHalfBytes<DP>;
            float sc[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t f[4];
                tc::ldmatrix4(f, keys_at(keys, d, lane));
#pragma unroll
                for (int j = 0; j < NT; ++j) tc::mma16<T>(sc[j], f, tile[j].q[d][0], tile[j].q[d][1]);
            }
            uint32_t p[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if ((int)(lane >> 2) >= limit) sc[j][0] = sc[j][1] = -INFINITY;
                if ((int)(lane >> 2) + 8 >= limit) sc[j][2] = sc[j][3] = -INFINITY;
                tile[j].softmax(sc[j], p[j], scale_log2);
            }
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t f[4];
                tc::ldmatrix4_trans(f, values_at(values, d, lane));
                if (limit < kSplitUnit) {
                    const int k = 2 * (int)(lane & 3);
                    f[0] = keep_keys(f[0], k, limit);
                    f[1] = keep_keys(f[1], k, limit);
                    f[2] = keep_keys(f[2], k + 8, limit);
                    f[3] = keep_keys(f[3], k + 8, limit);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) tc::mma16<T>(tile[j].o[d], f, p[j][0], p[j][1]);
            }
        }
        __syncwarp();
        if (lane == 0 && i + STAGES < mine_units) issue(i + STAGES);
    }

    // this warp's columns: maximum, sum and O, not divided
    __syncwarp();  // every lane is done with the ring
    auto partial = [&](uint32_t w, uint32_t col) { return reinterpret_cast<float *>(smem + w * S::kRing) + col * S::kPitch; };
    float *stats = reinterpret_cast<float *>(smem + S::kStats);
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
            float *o = partial(warp, col) + lane / 4;
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
                const float4 x = peer_load4(partial(w, col) + d, r);
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
        // a sum that is no number (a seen key that is none) makes lse none, as it makes out
        if (d == 0) a.lse[((uint64_t)b * a.heads + head) * a.queries + t] = sum != 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
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
    // thread blocks per query: enough for a few rounds of three on each SM, so that the last round costs little, while a warp has four pieces
    // of 16 keys (two where the machine would not be full otherwise).  One / this rule / always eight, us, the launches of a graph, dim 128, 8 heads of keys, blocks of 64: 1 token with
    // 16 blocks 18 / 7.5 / 7.5, with 48 50 / 12 / 12; 4 tokens 51 / 17 / 17, 16 52 / 54 / 55, 64 152 / 141 / 187
    uint32_t ranks = 1;
    while (ranks < 8 && rows * ranks < 12ull * sm_count && units >= (rows * ranks < (uint64_t)sm_count ? 4ull : 8ull) * ranks * kSplitWarps) ranks *= 2;
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

template <class T, int DP> cudaError_t launch_tile(const CUtensorMap &k_map, const CUtensorMap &v_map, const AttentionArgs &a, uint32_t box_rows, cudaStream_t s)
{
    TcShape shape = tc_shape(a.heads / a.kv_heads, box_rows);
    uint32_t bytes = 0;  // fewer queries where their lists are too long (tens of blocks for each of 128 queries)
    for (;; shape.queries /= 2)
        if ((bytes = TcSmem<DP>::kLists + TileUnion::bytes(shape.queries, a.count, a.block, a.keys)) <= kSmemMost || shape.queries == 1) break;
    CUtensorMap q_map;
    cudaError_t e = tc::make_map(&q_map, std::is_same<T, __nv_bfloat16>::value, a.q, a.dim, a.heads, a.queries, a.batch, a.q_head, a.q_query, a.q_batch, shape.queries, shape.heads);
    if (e == cudaSuccess) e = allow_dynamic_smem<block_attention_kernel<T, DP>>(kSmemMost);
    if (e != cudaSuccess) return e;
    const dim3 grid((a.queries + shape.queries - 1) / shape.queries, a.kv_heads * shape.chunks, a.batch);
    return launch_overlapped(block_attention_kernel<T, DP>, grid, dim3(kTcThreads), bytes, s, k_map, v_map, q_map, a, shape);
}

template <class T, int DP> cudaError_t launch_d(const CUtensorMap &k_map, const CUtensorMap &v_map, const AttentionArgs &a, bool split, uint32_t box_rows, int sm_count, cudaStream_t s)
{
    if (!split) return launch_tile<T, DP>(k_map, v_map, a, box_rows, s);
    return a.heads / a.kv_heads <= 8 ? launch_split<T, DP, 1>(k_map, v_map, a, sm_count, s) : launch_split<T, DP, 2>(k_map, v_map, a, sm_count, s);
}

}  // namespace

cudaError_t launch_block_attention(const AttentionArgs &a, int sm_count, cudaStream_t s)
{
    if (!a.batch || !a.queries || !a.heads || !a.dim) return cudaSuccess;
    const bool bf16 = a.dtype == CUTESPMM_BF16;
    // Few queries: a thread block or a cluster per query and head of keys, its blocks split over warps.  Split / tile in us at 1, 4, 5, 16 and 64 queries a sequence, caches of 32768 keys,
    // dim 128, neighbours agreeing on most blocks:
    //   1 sequence, 8 heads of keys, groups of 4, 16 blocks of 64:    8.5 / 19   12 / 40    11 / 42     21 / 56     52 / 61
    //   8 sequences, groups of 8, 16 blocks of 64:                     14 / 19   35 / 43    43 / 50     76 / 69    219 / 77
    //   64 sequences, groups of 8, 48 blocks of 64:                  147 / 131  335 / 262  403 / 284  1119 / 361  4315 / 1116
    // Where each is the better depends on the thread blocks a call makes, not on the queries alone: the limit of 4 is right for single tokens and for eight sequences and more, and gives away
    // a factor of two to four for 5 to 32 queries of one sequence.
    const bool split = a.queries <= 4;
    const uint32_t rows = a.pages ? a.block : a.keys, outer = a.pages ? a.num_pages : a.batch;
    const uint32_t box = split ? (uint32_t)kSplitUnit : a.pages && a.block < 64 ? a.block : 64u;
    CUtensorMap k_map{}, v_map{};
    if (rows && outer) {  // without keys no block counts and nothing is loaded
        cudaError_t e = tc::make_map(&k_map, bf16, a.k, a.dim, a.kv_heads, rows, outer, a.k_head, a.k_key, a.k_batch, box);
        if (e == cudaSuccess) e = tc::make_map(&v_map, bf16, a.v, a.dim, a.kv_heads, rows, outer, a.v_head, a.v_key, a.v_batch, box);
        if (e != cudaSuccess) return e;
    }
    if (bf16)
        return a.dim <= 64 ? launch_d<__nv_bfloat16, 64>(k_map, v_map, a, split, box, sm_count, s) : launch_d<__nv_bfloat16, 128>(k_map, v_map, a, split, box, sm_count, s);
    return a.dim <= 64 ? launch_d<__half, 64>(k_map, v_map, a, split, box, sm_count, s) : launch_d<__half, 128>(k_map, v_map, a, split, box, sm_count, s);
}

cudaError_t block_attention_status(uint32_t *word) { return read_status(g_status, word); }

}  // namespace cutespmm
