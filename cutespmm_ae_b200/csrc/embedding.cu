// Embedding: out[i] = scale * table[token_i], the product of a one-hot matrix with a table, and its gradient
// dtable[v] = scale * sum over the i with token_i = v of dout[i], the product with the transposed one-hot matrix.
//
// Both move rows and do next to no arithmetic: what bounds them is HBM (65536 tokens, 131072 x 4096 bf16: forward 158 us, 5.4 TB/s; gradient 370 us, of which the sort
// takes 25 and the sums, which write 1 GB, 347 at 4.5 TB/s).  The forward kernel copies; the gradient needs the
// transposed pattern, which is made in the call: a stable radix sort of the tokens (their positions stay in order inside a token,
// so sums are added in one fixed order and results do not change from run to run), then one kernel that writes every row of
// dtable exactly once -- a sum in fp32, rounded once, where a token names the row, zeros where none does.  fp32 also where the table is
// fp32: a sum of n terms is off by at most (n + 2) 2^-24 of their magnitudes, 6.1e-8 in all on a step of 8191 tokens where sums in 64 bits are off by 2.5e-8
// (the rounding of the result).  The terms are fp32 results of other kernels with errors of that size themselves, so wider sums were not taken.
#include <cuda_runtime.h>

#include <cstdint>

#include "device_plan.hpp"
#include "num.cuh"
#include "pattern_ops.hpp"
#include "ptx.cuh"

namespace cutespmm {
namespace {

constexpr int kWarps = 8;
constexpr int kInFlight = 4;  // loads of a lane in flight

// The row a token names, `vocab` for a token outside [0, vocab).
__device__ __forceinline__ uint32_t row_of_token(const void *tokens, int token_bytes, uint64_t i, uint64_t vocab)
{
    const uint64_t t = token_bytes == 8 ? (uint64_t)static_cast<const int64_t *>(tokens)[i] : (uint64_t)(int64_t)static_cast<const int32_t *>(tokens)[i];
    return (uint32_t)(t < vocab ? t : vocab);  // negative ones are large
}

template <class T, int V> __global__ void __launch_bounds__(kWarps * 32) embedding_kernel(EmbeddingArgs a)
{
    ptx::grid_wait();
    ptx::grid_release();
    const uint32_t lane = threadIdx.x & 31, span = 32u * V * kInFlight;
    const uint32_t spans = (a.dim + span - 1) / span;
    const uint64_t items = a.count * spans, step = (uint64_t)gridDim.x * kWarps;
    const T *table = static_cast<const T *>(a.src);
    T *out = static_cast<T *>(a.dst);
    for (uint64_t w = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); w < items; w += step) {
        const uint64_t i = w / spans;
        const uint32_t c0 = (uint32_t)(w % spans) * span + lane * V;
        const uint32_t row = row_of_token(a.tokens, a.token_bytes, i, a.vocab);
        const bool named = row < a.vocab;
        Pack<T, V> p[kInFlight];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u)
            if (named && c0 + u * 32 * V < a.dim) p[u] = load_pack<T, V>(table + row * a.ld_src + c0 + u * 32 * V);
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            const uint32_t c = c0 + u * 32 * V;
            if (c >= a.dim) break;
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = named ? a.scale * to_f32(p[u].x[j]) : 0.f;
            store_pack<T, V>(out + i * a.ld_dst + c, f);
        }
    }
}

// ---- the stable sort ---------------------------------------------------------------------------------------------------
// Least significant digit first, at most nine bits a pass (two passes up to 262 143 words, where eight would take three).  A pass is two kernels: every
// block counts the digits of its keys, then places them behind what the blocks in front of it counted.  kMaxBlocks bounds what a
// block has to add up; longer inputs give a block more keys.

constexpr int kMaxDigitBits = 9, kMaxBins = 1 << kMaxDigitBits;
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32;
constexpr uint32_t kMaxSortBlocks = 256;

struct SortArgs {
    const void *tokens;  // first pass: keys are made from the tokens
    int token_bytes;
    uint64_t vocab;
    uint32_t n, per_warp;          // keys, and keys of a warp (a multiple of 32)
    uint32_t shift, bins;
    const uint32_t *keys, *order;  // later passes
    uint32_t *keys_out, *order_out;
    uint32_t *counts;              // blocks x bins
    uint32_t *named;               // bit per row: some token names it (set by the first pass)
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, uint32_t i)
{
    return a.keys ? a.keys[i] : row_of_token(a.tokens, a.token_bytes, i, a.vocab);
}

// Digits of this block's keys, per warp, into shared memory.
__device__ __forceinline__ void count_digits(const SortArgs &a, uint32_t (*bins)[kMaxBins], bool mark)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t i = threadIdx.x; i < kSortWarps * kMaxBins; i += kSortThreads) (&bins[0][0])[i] = 0;
    __syncthreads();
    const uint64_t first = ((uint64_t)blockIdx.x * kSortWarps + warp) * a.per_warp;
    for (uint32_t k = lane; k < a.per_warp; k += 32) {
        if (first + k >= a.n) break;
        const uint32_t key = sort_key(a, (uint32_t)(first + k));
        atomicAdd(&bins[warp][(key >> a.shift) & (a.bins - 1)], 1u);
        if (mark && key < a.vocab) atomicOr(a.named + (key >> 5), 1u << (key & 31));
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a)
{
    __shared__ uint32_t bins[kSortWarps][kMaxBins];
    ptx::grid_wait();
    ptx::grid_release();
    count_digits(a, bins, a.keys == nullptr);
    for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) sum += bins[w][b];
        a.counts[(uint64_t)blockIdx.x * a.bins + b] = sum;
    }
}

__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortArgs a)
{
    __shared__ uint32_t bins[kSortWarps][kMaxBins];
    __shared__ uint32_t warp_sum[kSortWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ptx::grid_wait();
    ptx::grid_release();
    count_digits(a, bins, false);
    // per digit: keys of all blocks, and of the blocks in front of this one; two digits a thread
    static_assert(kMaxBins == 2 * kSortThreads, "two digits per thread");
    uint32_t before[2] = {0, 0}, all[2] = {0, 0};
    if (2 * threadIdx.x < a.bins) {
#pragma unroll 16
        for (uint32_t k = 0; k < gridDim.x; ++k) {
            const uint2 c = *reinterpret_cast<const uint2 *>(a.counts + (uint64_t)k * a.bins + 2 * threadIdx.x);  // at least two bins: a pass has a bit or more
            all[0] += c.x;
            all[1] += c.y;
            before[0] += k < blockIdx.x ? c.x : 0u;
            before[1] += k < blockIdx.x ? c.y : 0u;
        }
    }
    // keys of smaller digits: a scan over the threads
    const uint32_t mine = all[0] + all[1];
    uint32_t scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, scan, d);
        if (lane >= (uint32_t)d) scan += up;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    uint32_t base = scan - mine;
    for (uint32_t w = 0; w < warp; ++w) base += warp_sum[w];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t b = 2 * threadIdx.x + h;
        if (b >= a.bins) continue;
        uint32_t at = base + (h ? all[0] : 0u) + before[h];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = bins[w][b];
            bins[w][b] = at;  // where this warp's first key of the digit goes
            at += c;
        }
    }
    __syncthreads();
    const uint64_t first = ((uint64_t)blockIdx.x * kSortWarps + warp) * a.per_warp;
    for (uint32_t k = 0; k < a.per_warp; k += 32) {
        if (first + k >= a.n) break;
        const bool has = first + k + lane < a.n;
        const uint32_t i = has ? (uint32_t)(first + k + lane) : 0u;
        const uint32_t key = has ? sort_key(a, i) : 0u;
        const uint32_t digit = has ? (key >> a.shift) & (a.bins - 1) : kMaxBins;
        const uint32_t same = __match_any_sync(~0u, digit);
        const uint32_t rank = __popc(same & ((1u << lane) - 1u));
        uint32_t at = 0;
        if (has) at = bins[warp][digit] + rank;
        __syncwarp();
        if (has && rank == 0) bins[warp][digit] += __popc(same);
        __syncwarp();
        if (has) {
            a.keys_out[at] = key;
            a.order_out[at] = a.keys ? a.order[i] : i;
        }
    }
}

// ---- the rows of dtable ------------------------------------------------------------------------------------------------
// The sorted positions are cut into chunks; a block takes the tokens whose first position lies in its chunk and goes on to the end of
// the last one, so that sums of up to kLong positions stay in one block's registers.  Longer ones are cut at multiples of kPiece: each
// piece leaves a partial sum, and the block that finishes a token's last piece adds them in order (a counter per token and column
// slab; nobody waits).  The blocks behind those fill the rows that no token names.

constexpr uint32_t kChunk = 16, kPiece = 256, kLong = 2 * kPiece;
constexpr int kRowsInFlight = 8;  // rows of dout whose loads a thread has in flight
constexpr uint32_t kZeroRows = 32;  // rows of a block that fills: one word of `named`

struct SumArgs {
    EmbeddingArgs e;
    const uint32_t *keys, *order, *named;
    uint32_t *arrivals;  // window of kPiece positions x slab
    float *partial;      // 2 x windows x dim
    uint32_t n, chunks, slabs;
};

// The first position in (lo, hi] whose key is not `key`, given that key(lo) is.
__device__ __forceinline__ uint32_t end_of(const uint32_t *keys, uint32_t lo, uint32_t hi, uint32_t key)
{
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] == key) lo = mid; else hi = mid;
    }
    return hi;
}
__device__ __forceinline__ uint32_t start_of(const uint32_t *keys, uint32_t at, uint32_t key)
{
    uint32_t lo = 0, hi = at;  // keys[hi] == key; the first such position is in [lo, hi]
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] == key) hi = mid; else lo = mid + 1;
    }
    return lo;
}

template <class T, int V> struct Rows {
    const SumArgs &a;
    const uint32_t c;    // this thread's first column
    const bool on;
    float acc[V];

    __device__ Rows(const SumArgs &a_, uint32_t c_) : a(a_), c(c_), on(c_ < a_.e.dim) { clear(); }
    __device__ void clear()
    {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.f;
    }
    __device__ void flush(uint32_t row)
    {
        if (on) {
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] *= a.e.scale;
            store_pack<T, V>(static_cast<T *>(a.e.dst) + row * a.e.ld_dst + c, acc);
        }
        clear();
    }
    // Adds the rows of positions [b, e) in order; where EACH, a row of dtable is written at the end of each token, else the sum stays.
    // The lanes of a warp hold 32 positions' keys and places, the next 32 on their way, so that loads of rows wait for no index.
    template <bool EACH> __device__ void walk(uint32_t b, uint32_t e)
    {
        if (b >= e) return;
        const T *src = static_cast<const T *>(a.e.src) + c;
        const uint32_t lane = threadIdx.x & 31;
        uint32_t place = b + lane < e ? a.order[b + lane] : 0u, key = EACH && b + lane < e ? a.keys[b + lane] : 0u;
        uint32_t row = __shfl_sync(~0u, key, 0);
        for (uint32_t w = b; w < e; w += 32) {
            const uint32_t n = min(32u, e - w);
            const uint32_t next_place = w + 32 + lane < e ? a.order[w + 32 + lane] : 0u, next_key = EACH && w + 32 + lane < e ? a.keys[w + 32 + lane] : 0u;
            for (uint32_t x = 0; x < n; x += kRowsInFlight) {
                Pack<T, V> p[kRowsInFlight];
#pragma unroll
                for (int u = 0; u < kRowsInFlight; ++u) {
                    const uint32_t at = __shfl_sync(~0u, place, x + u);
                    if (on && x + u < n) p[u] = load_pack<T, V>(src + at * a.e.ld_src);
                }
#pragma unroll
                for (int u = 0; u < kRowsInFlight; ++u) {
                    const uint32_t token = __shfl_sync(~0u, key, x + u);
                    if (x + u >= n) break;
                    if (EACH && token != row) {
                        flush(row);
                        row = token;
                    }
                    if (on) {
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] += to_f32(p[u].x[j]);
                    }
                }
            }
            place = next_place;
            key = next_key;
        }
        if (EACH) flush(row);
    }
};

template <class T, int V> __global__ void embedding_sum_kernel(SumArgs a)
{
    ptx::grid_wait();
    ptx::grid_release();
    __shared__ uint32_t last;
    T *dst = static_cast<T *>(a.e.dst);
    if (blockIdx.x >= a.chunks * a.slabs) {  // rows that no token names
        const uint64_t row0 = (uint64_t)(blockIdx.x - a.chunks * a.slabs) * kZeroRows;
        const uint32_t named = a.named[row0 / 32];
        const float zero[V] = {};
        for (uint32_t r = 0; r < kZeroRows && row0 + r < a.e.vocab; ++r)
            if (!((named >> r) & 1u))
                for (uint32_t c = threadIdx.x * V; c < a.e.dim; c += blockDim.x * V) store_pack<T, V>(dst + (row0 + r) * a.e.ld_dst + c, zero);
        return;
    }
    const uint32_t chunk = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs, lane = threadIdx.x & 31;
    const uint32_t i0 = chunk * kChunk, i1 = min(i0 + kChunk, a.n);
    Rows<T, V> rows(a, (slab * blockDim.x + threadIdx.x) * V);

    // which positions of the chunk begin a token: lane l looks at position i0 + l
    const uint32_t at = i0 + lane;
    const uint32_t key = at < i1 ? a.keys[at] : (uint32_t)a.e.vocab;
    uint32_t prev = __shfl_up_sync(~0u, key, 1);
    if (lane == 0) prev = i0 ? a.keys[i0 - 1] : ~0u;
    const uint32_t heads = __ballot_sync(~0u, at < i1 && key < a.e.vocab && key != prev);
    const uint32_t key0 = __shfl_sync(~0u, key, 0);

    // the sum of a piece [b, e) of a long token that starts at position s
    auto piece = [&](uint32_t b, uint32_t e, uint32_t s, uint32_t token) {
        rows.template walk<false>(b, e);
        const uint32_t slot = 2 * (b / kPiece) + (b == s ? 1u : 0u);
        if (rows.on) {
#pragma unroll
            for (int j = 0; j < V; ++j) __stcg(a.partial + (uint64_t)slot * a.e.dim + rows.c + j, rows.acc[j]);
        }
        rows.clear();
        __threadfence();
        __syncthreads();
        const uint32_t end = end_of(a.keys, s, a.n, token), pieces = 1 + (end - 1) / kPiece - s / kPiece;
        if (threadIdx.x == 0) last = atomicAdd(a.arrivals + (uint64_t)(s / kPiece) * a.slabs + slab, 1u) == pieces - 1;
        __syncthreads();
        if (last) {
            __threadfence();
            if (rows.on) {
                for (uint32_t k = 0; k < pieces; ++k) {
                    const uint32_t from = k ? 2 * (s / kPiece + k) : 2 * (s / kPiece) + 1;
#pragma unroll
                    for (int j = 0; j < V; ++j) rows.acc[j] += __ldcg(a.partial + (uint64_t)from * a.e.dim + rows.c + j);
                }
            }
            rows.flush(token);
        }
        __syncthreads();  // `last` is read before it is written again
    };

    if (i0 % kPiece == 0 && key0 < a.e.vocab && !(heads & 1u)) {
        const uint32_t s = start_of(a.keys, i0, key0);
        if ((uint64_t)s + kLong < a.n && a.keys[s + kLong] == key0) piece(i0, end_of(a.keys, i0, min(i0 + kPiece, a.n), key0), s, key0);
    }
    if (!heads) return;
    const uint32_t b = i0 + __ffs(heads) - 1, tail = i0 + 31 - __clz(heads), tail_key = a.keys[tail];
    if ((uint64_t)tail + kLong < a.n && a.keys[tail + kLong] == tail_key) {
        rows.template walk<true>(b, tail);
        piece(tail, (tail / kPiece + 1) * kPiece, tail, tail_key);
    } else
        rows.template walk<true>(b, end_of(a.keys, tail, min(tail + kLong, a.n), tail_key));
}

template <class T> bool wide(const EmbeddingArgs &a)
{
    const uint64_t bytes = reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst) | (a.ld_src | a.ld_dst | a.dim) * sizeof(T);
    return bytes % 16 == 0;
}

// Where the parts of the gradient's workspace begin (bytes).
struct GradLayout {
    uint64_t keys[2], order[2], counts, named, arrivals, partial, cleared, total;
    uint32_t slabs_most;
    GradLayout(uint64_t n, uint64_t vocab, uint32_t dim)
    {
        uint64_t at = 0;
        auto take = [&](uint64_t bytes) { const uint64_t p = at; at += (bytes + 255) / 256 * 256; return p; };
        for (int i = 0; i < 2; ++i) {
            keys[i] = take(n * 4);
            order[i] = take(n * 4);
        }
        counts = take((uint64_t)kMaxSortBlocks * kMaxBins * 4);
        const uint64_t windows = (n + kPiece - 1) / kPiece;
        slabs_most = (dim + 31) / 32;  // one column per thread, 32 threads: never more slabs than this
        named = take((vocab + 31) / 32 * 4);
        arrivals = take(windows * slabs_most * 4);
        cleared = at - named;
        partial = take(2 * windows * dim * 4);
        total = at;
    }
};

}  // namespace

cudaError_t launch_embedding(const EmbeddingArgs &a, int sm_count, cudaStream_t s)
{
    if (a.count == 0 || a.dim == 0) return cudaSuccess;
    return for_dtype(a.dtype, [&](auto zero) {
        using T = decltype(zero);
        auto go = [&](auto kernel, uint32_t v) {
            const uint64_t spans = (a.dim + 32ull * v * kInFlight - 1) / (32ull * v * kInFlight), blocks = (a.count * spans + kWarps - 1) / kWarps;
            const uint64_t cap = (uint64_t)sm_count * 64;
            return launch_overlapped(kernel, dim3((unsigned)(blocks < cap ? blocks : cap)), dim3(kWarps * 32), 0, s, a);
        };
        return wide<T>(a) ? go(embedding_kernel<T, kVec<T>>, kVec<T>) : go(embedding_kernel<T, 1>, 1);
    });
}

uint64_t embedding_grad_workspace(uint64_t count, uint64_t vocab, uint32_t dim) { return GradLayout(count, vocab, dim).total; }

cudaError_t launch_embedding_grad(const EmbeddingArgs &a, void *workspace, cudaStream_t s)
{
    if (a.vocab == 0 || a.dim == 0) return cudaSuccess;
    const GradLayout l(a.count, a.vocab, a.dim);
    char *w = static_cast<char *>(workspace);
    auto words = [&](uint64_t at) { return reinterpret_cast<uint32_t *>(w + at); };
    cudaError_t e = cudaMemsetAsync(w + l.named, 0, l.cleared, s);
    if (e != cudaSuccess) return e;
    SumArgs sum{};
    sum.e = a;
    sum.n = (uint32_t)a.count;
    if (a.count) {
        int bits = 1;
        while ((a.vocab >> bits) != 0) ++bits;  // the largest key is vocab itself
        const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits, digit = (bits + passes - 1) / passes;
        SortArgs p{};
        p.tokens = a.tokens;
        p.token_bytes = a.token_bytes;
        p.vocab = a.vocab;
        p.n = sum.n;
        // 64 keys a warp: a pass is a chain of latencies; more where that would make too many blocks (65536 tokens 30 us a pass with 256)
        p.per_warp = 64;
        while ((a.count + (uint64_t)p.per_warp * kSortWarps - 1) / ((uint64_t)p.per_warp * kSortWarps) > kMaxSortBlocks) p.per_warp *= 2;
        const unsigned blocks = (unsigned)((a.count + (uint64_t)p.per_warp * kSortWarps - 1) / ((uint64_t)p.per_warp * kSortWarps));
        p.bins = 1u << digit;
        p.counts = words(l.counts);
        p.named = words(l.named);
        for (int i = 0; i < passes; ++i) {
            p.shift = (uint32_t)(i * digit);
            p.keys = i ? words(l.keys[(i + 1) & 1]) : nullptr;
            p.order = i ? words(l.order[(i + 1) & 1]) : nullptr;
            p.keys_out = words(l.keys[i & 1]);
            p.order_out = words(l.order[i & 1]);
            if ((e = launch_overlapped(sort_count_kernel, dim3(blocks), dim3(kSortThreads), 0, s, p)) != cudaSuccess) return e;
            if ((e = launch_overlapped(sort_place_kernel, dim3(blocks), dim3(kSortThreads), 0, s, p)) != cudaSuccess) return e;
        }
        sum.keys = p.keys_out;
        sum.order = p.order_out;
    }
    sum.named = words(l.named);
    sum.arrivals = words(l.arrivals);
    sum.partial = reinterpret_cast<float *>(w + l.partial);
    return for_dtype(a.dtype, [&](auto zero) {
        using T = decltype(zero);
        auto go = [&](auto kernel, uint32_t v) {
            const uint32_t packs = (a.dim + v - 1) / v;
            const uint32_t threads = packs <= 32 ? 32 : packs <= 64 ? 64 : 128;
            sum.slabs = (packs + threads - 1) / threads;
            sum.chunks = (uint32_t)((a.count + kChunk - 1) / kChunk);
            const uint64_t blocks = (uint64_t)sum.chunks * sum.slabs + (a.vocab + kZeroRows - 1) / kZeroRows;
            if (blocks > 0x7fffffffull) return cudaErrorInvalidConfiguration;
            return launch_overlapped(kernel, dim3((unsigned)blocks), dim3(threads), 0, s, sum);
        };
        return wide<T>(a) ? go(embedding_sum_kernel<T, kVec<T>>, kVec<T>) : go(embedding_sum_kernel<T, 1>, 1);
    });
}

}  // namespace cutespmm
