// The extern "C" surface of the operators whose sparse pattern the data choose in each call (include/cutespmm.h): checks of arguments,
// then the launchers of pattern_ops.hpp.  Nothing here allocates, waits or throws.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_plan.hpp"
#include "nvtx.hpp"
#include "pattern_ops.hpp"
#include "plan_object.hpp"
#include "../../include/cutespmm.h"

using namespace cutespmm;

namespace {

int refuse(int status, const char *msg) { return fail_status(status, msg); }
int launched(cudaError_t e, const char *what) { return e == cudaSuccess ? CUTESPMM_OK : fail_cuda_status(e, what); }
cudaStream_t stream_of(void *s) { return static_cast<cudaStream_t>(s); }

bool aligned(const void *p, const int64_t *strides)
{
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    for (int i = 0; i < 3; ++i)
        if (strides[i] < 0 || strides[i] % 8 || strides[i] >= (int64_t)1 << 39) return false;
    return true;
}
// Kernels load and store 16 bytes at a time in results as well; every other array has to lie on its elements' own grid.
bool on_grid(const void *p, uint32_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
uint32_t bytes_of(int dtype) { return dtype == CUTESPMM_F32 ? 4 : 2; }
const char *const kOffElements = "a pointer is not aligned to its elements";
bool fits_grid(uint64_t n) { return n <= 65535; }

int check_embedding(int dtype, uint64_t vocab, uint32_t dim, const void *a, uint64_t ld_a, const void *b, uint64_t ld_b, const void *tokens, int token_bytes, uint64_t count)
{
    if (dtype != CUTESPMM_F32 && dtype != CUTESPMM_F16 && dtype != CUTESPMM_BF16) return refuse(CUTESPMM_EINVAL, "dtype must be CUTESPMM_F32, CUTESPMM_F16 or CUTESPMM_BF16");
    if (token_bytes != 4 && token_bytes != 8) return refuse(CUTESPMM_EINVAL, "tokens must be int32 or int64 (token_bytes 4 or 8)");
    if (ld_a < dim || ld_b < dim) return refuse(CUTESPMM_EINVAL, "leading dimension smaller than dim");
    if (vocab >> 31 || count >> 31) return refuse(CUTESPMM_EUNSUPPORTED, "more than 2^31 - 1 rows or tokens");
    if (dim >> 30) return refuse(CUTESPMM_EUNSUPPORTED, "dim must be below 2^30");
    if (count && !tokens) return refuse(CUTESPMM_EINVAL, "tokens is NULL");
    if (!on_grid(a, bytes_of(dtype)) || !on_grid(b, bytes_of(dtype)) || !on_grid(tokens, (uint32_t)token_bytes)) return refuse(CUTESPMM_EINVAL, kOffElements);
    return CUTESPMM_OK;
}

int check_blocks(int dtype, uint32_t batch, uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t dim)
{
    if (dtype != CUTESPMM_F16 && dtype != CUTESPMM_BF16) return refuse(CUTESPMM_EINVAL, "dtype must be CUTESPMM_F16 or CUTESPMM_BF16");
    if (dim == 0 || dim % 8 || dim > 128) return refuse(CUTESPMM_EUNSUPPORTED, "dim must be a multiple of 8, at most 128");
    if (kv_heads == 0 || heads % kv_heads) return refuse(CUTESPMM_EINVAL, "heads must be a multiple of kv_heads");
    if (!fits_grid((uint64_t)batch * kv_heads)) return refuse(CUTESPMM_EUNSUPPORTED, "batch * kv_heads must be at most 65535");
    if (rows >> 28) return refuse(CUTESPMM_EUNSUPPORTED, "more than 2^28 - 1 queries or keys");
    return CUTESPMM_OK;
}
bool block_size_ok(uint32_t block) { return block == 16 || block == 32 || block == 64 || block == 128; }
constexpr uint32_t kMostBlocks = 65536;
const char *const kTooManyBlocks = "at most 65536 blocks of keys";
const char *const kBlockSizes = "block must be 16, 32, 64 or 128";

// Checks a call's description and turns it into the kernels' arguments.
int to_args(const cutespmm_block_attention_t *d, AttentionArgs &a)
{
    if (!d) return refuse(CUTESPMM_EINVAL, "args is NULL");
    if (d->struct_size != sizeof *d) return refuse(CUTESPMM_EINVAL, "struct_size does not match cutespmm_block_attention_t");
    int st = check_blocks((int)d->dtype, d->batch, d->queries, d->heads, d->kv_heads, d->dim);
    if (st != CUTESPMM_OK) return st;
    if (!block_size_ok(d->block)) return refuse(CUTESPMM_EINVAL, kBlockSizes);
    if (!(d->scale > 0.f && d->scale < INFINITY)) return refuse(CUTESPMM_EINVAL, "scale must be positive and finite");
    if (d->count > 128) return refuse(CUTESPMM_EUNSUPPORTED, "at most 128 blocks per query");
    if (d->keys >> 28) return refuse(CUTESPMM_EUNSUPPORTED, "more than 2^28 - 1 keys");
    if (d->heads / d->kv_heads > 128) return refuse(CUTESPMM_EUNSUPPORTED, "at most 128 query heads for each head of keys");
    if (!fits_grid((uint64_t)d->batch * 4)) return refuse(CUTESPMM_EUNSUPPORTED, "batch must be at most 16383");
    if (!fits_grid((uint64_t)d->kv_heads * ((d->heads / d->kv_heads + 7) / 8))) return refuse(CUTESPMM_EUNSUPPORTED, "too many heads: kv_heads for every eight of a group must be at most 65535");
    const uint32_t blocks = (d->keys + d->block - 1) / d->block;
    if (blocks > kMostBlocks) return refuse(CUTESPMM_EUNSUPPORTED, kTooManyBlocks);
    if (d->pages && (uint64_t)d->page_cols * d->block != d->keys) return refuse(CUTESPMM_EINVAL, "keys must be page_cols * block for a paged cache");
    if (d->pages && d->num_pages >> 31) return refuse(CUTESPMM_EUNSUPPORTED, "more than 2^31 - 1 pages");
    const bool work = d->batch && d->queries && d->heads;
    if (work && !d->q) return refuse(CUTESPMM_EINVAL, "q is NULL");
    if (work && d->keys && (!d->pages || d->num_pages) && (!d->k || !d->v)) return refuse(CUTESPMM_EINVAL, "k or v is NULL");
    if (work && d->count && !d->blocks) return refuse(CUTESPMM_EINVAL, "blocks is NULL");
    if (!aligned(d->q, d->q_strides) || !aligned(d->k, d->k_strides) || !aligned(d->v, d->v_strides))
        return refuse(CUTESPMM_EINVAL, "q, k and v must be 16-byte aligned, their strides multiples of 8 elements");
    if (!on_grid(d->blocks, 4) || !on_grid(d->visible, 4) || !on_grid(d->pages, 4)) return refuse(CUTESPMM_EINVAL, kOffElements);
    a = AttentionArgs{};
    a.dtype = (int)d->dtype;
    a.q = d->q; a.k = d->k; a.v = d->v;
    a.q_batch = d->q_strides[0]; a.q_query = d->q_strides[1]; a.q_head = d->q_strides[2];
    a.k_batch = d->k_strides[0]; a.k_key = d->k_strides[1]; a.k_head = d->k_strides[2];
    a.v_batch = d->v_strides[0]; a.v_key = d->v_strides[1]; a.v_head = d->v_strides[2];
    a.blocks = d->blocks; a.visible = d->visible; a.pages = d->pages;
    a.batch = d->batch; a.queries = d->queries; a.heads = d->heads; a.kv_heads = d->kv_heads; a.dim = d->dim;
    a.keys = d->keys; a.block = d->block; a.count = d->count; a.num_blocks = blocks;
    a.page_cols = d->pages ? d->page_cols : 0; a.num_pages = d->pages ? d->num_pages : 0;
    a.scale = d->scale;
    return CUTESPMM_OK;
}

}  // namespace

extern "C" {

int cutespmm_embedding(int dtype, const void *table_dev, uint64_t ld_table, uint64_t vocab, uint32_t dim, const void *tokens_dev, int token_bytes, uint64_t count, float scale,
                       void *out_dev, uint64_t ld_out, void *stream)
{
    int st = check_embedding(dtype, vocab, dim, table_dev, ld_table, out_dev, ld_out, tokens_dev, token_bytes, count);
    if (st != CUTESPMM_OK) return st;
    if (count && dim && ((vocab && !table_dev) || !out_dev)) return refuse(CUTESPMM_EINVAL, "table or out is NULL");
    int dev = -1, sms = 0;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: embedding");
    const EmbeddingArgs a{dtype, tokens_dev, token_bytes, count, vocab, dim, scale, table_dev, ld_table, out_dev, ld_out};
    return launched(launch_embedding(a, sms, stream_of(stream)), "embedding");
}

uint64_t cutespmm_embedding_grad_workspace(uint64_t count, uint64_t vocab, uint32_t dim) { return embedding_grad_workspace(count, vocab, dim); }

int cutespmm_embedding_grad(int dtype, const void *dout_dev, uint64_t ld_dout, const void *tokens_dev, int token_bytes, uint64_t count, uint64_t vocab, uint32_t dim, float scale,
                            void *dtable_dev, uint64_t ld_dtable, void *workspace_dev, uint64_t workspace_bytes, void *stream)
{
    int st = check_embedding(dtype, vocab, dim, dout_dev, ld_dout, dtable_dev, ld_dtable, tokens_dev, token_bytes, count);
    if (st != CUTESPMM_OK) return st;
    if (vocab == 0 || dim == 0) return CUTESPMM_OK;
    if ((count && !dout_dev) || !dtable_dev) return refuse(CUTESPMM_EINVAL, "dout or dtable is NULL");
    if (!workspace_dev || reinterpret_cast<uintptr_t>(workspace_dev) % 256 || workspace_bytes < embedding_grad_workspace(count, vocab, dim))
        return refuse(CUTESPMM_EINVAL, "workspace must be 256-byte aligned and hold cutespmm_embedding_grad_workspace() bytes");
    int dev = -1, sms = 0;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: embedding gradient");
    const EmbeddingArgs a{dtype, tokens_dev, token_bytes, count, vocab, dim, scale, dout_dev, ld_dout, dtable_dev, ld_dtable};
    return launched(launch_embedding_grad(a, workspace_dev, stream_of(stream)), "embedding gradient");
}

int cutespmm_block_means(int dtype, const void *k_dev, const int64_t k_strides[3], const int32_t *lengths_dev, uint32_t batch, uint32_t keys, uint32_t kv_heads, uint32_t dim,
                         uint32_t block, void *means_dev, void *stream)
{
    int st = check_blocks(dtype, batch, keys, kv_heads, kv_heads, dim);
    if (st != CUTESPMM_OK) return st;
    if (!block_size_ok(block)) return refuse(CUTESPMM_EINVAL, kBlockSizes);
    const uint32_t blocks = (keys + block - 1) / block;
    if (blocks > kMostBlocks) return refuse(CUTESPMM_EUNSUPPORTED, kTooManyBlocks);
    if (!k_strides || !aligned(k_dev, k_strides)) return refuse(CUTESPMM_EINVAL, "k must be 16-byte aligned, its strides multiples of 8 elements");
    if (batch && blocks && (!k_dev || !means_dev)) return refuse(CUTESPMM_EINVAL, "k or means is NULL");
    if (!on_grid(lengths_dev, 4) || !on_grid(means_dev, 2)) return refuse(CUTESPMM_EINVAL, kOffElements);
    int dev = -1, sms = 0;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: block means");
    const MeansArgs a{dtype, k_dev, k_strides[0], k_strides[1], k_strides[2], lengths_dev, means_dev, batch, keys, blocks, block, kv_heads, dim};
    return launched(launch_block_means(a, stream_of(stream)), "block means");
}

int cutespmm_block_scores(int dtype, const void *q_dev, const int64_t q_strides[3], const void *means_dev, const int64_t means_strides[3], uint32_t batch, uint32_t queries,
                          uint32_t heads, uint32_t kv_heads, uint32_t blocks, uint32_t dim, float *scores_dev, void *stream)
{
    int st = check_blocks(dtype, batch, queries, heads, kv_heads, dim);
    if (st != CUTESPMM_OK) return st;
    if (!q_strides || !means_strides || !aligned(q_dev, q_strides) || !aligned(means_dev, means_strides))
        return refuse(CUTESPMM_EINVAL, "q and means must be 16-byte aligned, their strides multiples of 8 elements");
    if (blocks > kMostBlocks) return refuse(CUTESPMM_EUNSUPPORTED, kTooManyBlocks);
    if (((uint64_t)(blocks + 255) / 256 * ((queries + 127) / 128) * batch * kv_heads) >> 31) return refuse(CUTESPMM_EUNSUPPORTED, "too many queries and blocks for one call");
    if (batch && queries && blocks && ((heads && (!q_dev || !means_dev)) || !scores_dev)) return refuse(CUTESPMM_EINVAL, "q, means or scores is NULL");
    if (!on_grid(scores_dev, 4)) return refuse(CUTESPMM_EINVAL, kOffElements);
    int dev = -1, sms = 0;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: block scores");
    const ScoresArgs a{dtype, q_dev, means_dev, q_strides[0], q_strides[1], q_strides[2], means_strides[0], means_strides[1], means_strides[2], scores_dev, batch, queries, heads,
                       kv_heads, blocks, dim};
    return launched(launch_block_scores(a, sms, stream_of(stream)), "block scores");
}

int cutespmm_select_blocks(const float *scores_dev, const int64_t s_strides[3], const int32_t *visible_dev, uint32_t batch, uint32_t kv_heads, uint32_t queries, uint32_t blocks,
                           uint32_t keys, uint32_t block, uint32_t count, uint32_t first, uint32_t last, int32_t *blocks_dev, void *stream)
{
    if (!block_size_ok(block)) return refuse(CUTESPMM_EINVAL, kBlockSizes);
    if ((keys + (uint64_t)block - 1) / block != blocks) return refuse(CUTESPMM_EINVAL, "scores must have a column per block of keys");
    if ((uint64_t)first + last > count) return refuse(CUTESPMM_EINVAL, "first + last must not exceed count");
    if (blocks > 16384) return refuse(CUTESPMM_EUNSUPPORTED, "at most 16384 blocks");
    if (keys >> 28 || queries >> 28 || count >> 16) return refuse(CUTESPMM_EUNSUPPORTED, "too many keys, queries or blocks per query");
    if (!fits_grid((uint64_t)batch * kv_heads)) return refuse(CUTESPMM_EUNSUPPORTED, "batch * kv_heads must be at most 65535");
    if (batch && kv_heads && queries && count && ((blocks && (!scores_dev || !s_strides)) || !blocks_dev)) return refuse(CUTESPMM_EINVAL, "scores, strides or blocks is NULL");
    if (!on_grid(scores_dev, 4) || !on_grid(visible_dev, 4) || !on_grid(blocks_dev, 4)) return refuse(CUTESPMM_EINVAL, kOffElements);
    int dev = -1, sms = 0, st;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: block selection");
    SelectArgs a{scores_dev, 0, 0, 0, visible_dev, blocks_dev, batch, kv_heads, queries, blocks, keys, block, count, first, last};
    if (s_strides) {
        a.s_batch = s_strides[0];
        a.s_head = s_strides[1];
        a.s_query = s_strides[2];
    }
    return launched(launch_select_blocks(a, sms, stream_of(stream)), "block selection");
}

int cutespmm_block_attention(const cutespmm_block_attention_t *args, void *out_dev, float *lse_dev, void *stream)
{
    AttentionArgs a;
    int st = to_args(args, a);
    if (st != CUTESPMM_OK) return st;
    if (a.batch && a.queries && a.heads && (!out_dev || !lse_dev)) return refuse(CUTESPMM_EINVAL, "out or lse is NULL");
    if (!on_grid(out_dev, 16) || !on_grid(lse_dev, 4)) return refuse(CUTESPMM_EINVAL, "out must be 16-byte aligned, lse aligned to its elements");
    int dev = -1, sms = 0;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: block attention");
    a.out = out_dev;
    a.lse = lse_dev;
    return launched(launch_block_attention(a, sms, stream_of(stream)), "block attention");
}

uint64_t cutespmm_block_attention_grad_workspace(const cutespmm_block_attention_t *args)
{
    AttentionArgs a;
    return to_args(args, a) == CUTESPMM_OK ? block_attention_grad_workspace(a) : 0;
}

int cutespmm_block_attention_grad(const cutespmm_block_attention_t *args, const void *dout_dev, const int64_t dout_strides[3], const void *out_dev, const float *lse_dev, void *dq_dev,
                                  void *dk_dev, void *dv_dev, void *workspace_dev, uint64_t workspace_bytes, void *stream)
{
    AttentionArgs a;
    int st = to_args(args, a);
    if (st != CUTESPMM_OK) return st;
    if (a.pages) return refuse(CUTESPMM_EUNSUPPORTED, "a paged cache has no gradient");
    if (!dout_strides || !aligned(dout_dev, dout_strides)) return refuse(CUTESPMM_EINVAL, "dout must be 16-byte aligned, its strides multiples of 8 elements");
    if (a.batch && a.queries && a.heads && (!dout_dev || !out_dev || !lse_dev || !dq_dev)) return refuse(CUTESPMM_EINVAL, "dout, out, lse or dq is NULL");
    if (a.batch && a.keys && (!dk_dev || !dv_dev)) return refuse(CUTESPMM_EINVAL, "dk or dv is NULL");
    if (!on_grid(out_dev, 16) || !on_grid(dq_dev, 16) || !on_grid(dk_dev, 16) || !on_grid(dv_dev, 16) || !on_grid(lse_dev, 4))
        return refuse(CUTESPMM_EINVAL, "out, dq, dk and dv must be 16-byte aligned, lse aligned to its elements");
    const uint64_t need = block_attention_grad_workspace(a);
    if (need && (!workspace_dev || reinterpret_cast<uintptr_t>(workspace_dev) % 256 || workspace_bytes < need))
        return refuse(CUTESPMM_EINVAL, "workspace must be 256-byte aligned and hold cutespmm_block_attention_grad_workspace() bytes");
    int dev = -1, sms = 0;
    if ((st = cutespmm_internal_usable_device(&dev, &sms)) != CUTESPMM_OK) return st;
    NvtxRange range("cutespmm: block attention gradient");
    a.out = const_cast<void *>(out_dev);
    a.lse = const_cast<float *>(lse_dev);
    a.dout = dout_dev;
    a.do_batch = dout_strides[0]; a.do_query = dout_strides[1]; a.do_head = dout_strides[2];
    a.dq = dq_dev; a.dk = dk_dev; a.dv = dv_dev;
    a.workspace = workspace_dev;
    return launched(launch_block_attention_grad(a, sms, stream_of(stream)), "block attention gradient");
}

int cutespmm_pattern_status(uint32_t *status)
{
    if (!status) return refuse(CUTESPMM_EINVAL, "status is NULL");
    int dev = -1, sms = 0;
    const int st = cutespmm_internal_usable_device(&dev, &sms);
    if (st != CUTESPMM_OK) return st;
    *status = 0;
    for (auto read : {block_select_status, block_attention_status, block_attention_grad_status}) {
        uint32_t word = 0;
        const cudaError_t e = read(&word);
        if (e != cudaSuccess) return fail_cuda_status(e, "reading the status words");
        *status |= word;
    }
    return CUTESPMM_OK;
}

}  // extern "C"
