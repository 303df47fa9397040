// Argument blocks and launcher prototypes of the operators whose sparse pattern the data choose in each call: embedding (a
// one-hot matrix times a table) and its gradient, and attention over blocks of keys that a score selects for each query.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace cutespmm {

// ---- embedding.cu ----
struct EmbeddingArgs {
    int dtype;            // cutespmm_dtype_t of the table, the output and both gradients
    const void *tokens;   // count indices of token_bytes (4 or 8) each
    int token_bytes;
    uint64_t count, vocab;
    uint32_t dim;
    float scale;
    const void *src;      // forward: the table; gradient: dout
    uint64_t ld_src;      // elements
    void *dst;            // forward: out; gradient: dtable
    uint64_t ld_dst;
};
cudaError_t launch_embedding(const EmbeddingArgs &a, int sm_count, cudaStream_t s);
uint64_t embedding_grad_workspace(uint64_t count, uint64_t vocab, uint32_t dim);
cudaError_t launch_embedding_grad(const EmbeddingArgs &a, void *workspace, cudaStream_t s);

// ---- block_select.cu ----
struct MeansArgs {
    int dtype;
    const void *k;
    int64_t k_batch, k_key, k_head;  // strides in elements
    const int32_t *lengths;          // per sequence, or nullptr: every key counts
    void *means;                     // batch x blocks x kv_heads x dim
    uint32_t batch, keys, blocks, block, kv_heads, dim;
};
cudaError_t launch_block_means(const MeansArgs &a, cudaStream_t s);

struct ScoresArgs {
    int dtype;
    const void *q, *means;
    int64_t q_batch, q_query, q_head, m_batch, m_block, m_head;
    float *scores;  // batch x kv_heads x queries x blocks
    uint32_t batch, queries, heads, kv_heads, blocks, dim;
};
cudaError_t launch_block_scores(const ScoresArgs &a, int sm_count, cudaStream_t s);

struct SelectArgs {
    const float *scores;     // batch x kv_heads x queries x blocks, rows contiguous
    int64_t s_batch, s_head, s_query;
    const int32_t *visible;  // batch x queries, or nullptr: query i sees keys - queries + 1 + i
    int32_t *out;            // batch x kv_heads x queries x count
    uint32_t batch, kv_heads, queries, blocks, keys, block, count, first, last;
};
cudaError_t launch_select_blocks(const SelectArgs &a, int sm_count, cudaStream_t s);

// ---- block_attention.cu, block_attention_grad.cu ----
struct AttentionArgs {
    int dtype;
    const void *q, *k, *v;
    int64_t q_batch, q_query, q_head, k_batch, k_key, k_head, v_batch, v_key, v_head;  // elements; k_batch, v_batch: of a page in a paged cache
    const int32_t *blocks;   // batch x kv_heads x queries x count
    const int32_t *visible;  // batch x queries, or nullptr
    const int32_t *pages;    // batch x page_cols, or nullptr
    void *out;               // batch x queries x heads x dim
    float *lse;              // batch x heads x queries
    uint32_t batch, queries, heads, kv_heads, dim, keys, block, count, num_blocks, page_cols, num_pages;
    float scale;
    // gradient
    const void *dout;
    int64_t do_batch, do_query, do_head;
    float *delta;            // batch x heads x queries
    void *dq, *dk, *dv;      // contiguous, like q, k and v
    void *workspace;
};
cudaError_t launch_block_attention(const AttentionArgs &a, int sm_count, cudaStream_t s);
uint64_t block_attention_grad_workspace(const AttentionArgs &a);
cudaError_t launch_block_attention_grad(const AttentionArgs &a, int sm_count, cudaStream_t s);

// What a bounded wait that gave up has written on the current device, cleared.  Waits for the device.
cudaError_t block_select_status(uint32_t *word);
cudaError_t block_attention_status(uint32_t *word);
cudaError_t block_attention_grad_status(uint32_t *word);

}  // namespace cutespmm
