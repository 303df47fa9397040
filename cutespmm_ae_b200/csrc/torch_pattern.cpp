// The operators whose sparse pattern the data choose in each call, on torch tensors: checks, outputs and scratch from torch's
// allocator (so calls can be captured and overlap), the current stream and the tensors' own device, gradients.
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "torch_common.hpp"

namespace {

using namespace bind;
using OptTensor = std::optional<Tensor>;

int dtype_of(const Tensor &t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return CUTESPMM_F32;
        case at::kHalf: return CUTESPMM_F16;
        case at::kBFloat16: return CUTESPMM_BF16;
        default: return -1;
    }
}
uint32_t u32(int64_t v)
{
    TORCH_CHECK_VALUE(v >= 0 && v <= (int64_t)UINT32_MAX, "a size of ", v, " is beyond 32 bits");
    return (uint32_t)v;
}
Tensor empty_like_of(at::IntArrayRef sizes, const Tensor &like, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false).memory_format(at::MemoryFormat::Contiguous)); }
Tensor empty_like_of(at::IntArrayRef sizes, const Tensor &like) { return empty_like_of(sizes, like, like.scalar_type()); }
Tensor scratch(uint64_t bytes, const Tensor &like) { return bytes ? empty_like_of({(int64_t)bytes}, like, at::kByte) : Tensor(); }
void *pointer_of(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
template <class T> T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(const_cast<void *>(t.const_data_ptr())) : nullptr; }
void want_cuda(const Tensor &first, std::initializer_list<Tensor> others)
{
    TORCH_CHECK_VALUE(first.is_cuda(), "operands must be CUDA tensors");
    for (const Tensor &t : others) TORCH_CHECK_VALUE(!t.defined() || t.device() == first.device(), "all operands must live on one device");
}

// ---- embedding -------------------------------------------------------------------------------------------------------

void check_tokens(const Tensor &tokens) { TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens must be int32 or int64"); }
Tensor unit_stride(const Tensor &t) { return t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous(); }
uint64_t ld(const Tensor &t) { return t.size(0) > 1 ? (uint64_t)t.stride(0) : (uint64_t)t.size(1); }

Tensor op_embedding(const Tensor &tokens, const Tensor &table, double scale)
{
    check_tokens(tokens);
    TORCH_CHECK_VALUE(table.dim() == 2 && dtype_of(table) >= 0, "table must be a 2-D tensor of float32, float16 or bfloat16");
    want_cuda(table, {tokens});
    const c10::cuda::CUDAGuard guard(table.device());
    const Tensor ids = tokens.contiguous(), rows = unit_stride(table);
    std::vector<int64_t> sizes = ids.sizes().vec();
    sizes.push_back(rows.size(1));
    Tensor out = empty_like_of(sizes, rows);
    check_status(cutespmm_embedding(dtype_of(rows), ptr<void>(rows), ld(rows), (uint64_t)rows.size(0), u32(rows.size(1)), ptr<void>(ids), (int)ids.element_size(), (uint64_t)ids.numel(),
                                    (float)scale, pointer_of(out), (uint64_t)rows.size(1), stream_of(rows)));
    return out;
}

Tensor op_embedding_grad(const Tensor &tokens, const Tensor &dout, int64_t vocab, double scale)
{
    check_tokens(tokens);
    TORCH_CHECK_VALUE(dout.dim() >= 1 && dtype_of(dout) >= 0 && dout.dim() == tokens.dim() + 1 && dout.sizes().slice(0, tokens.dim()) == tokens.sizes(),
                      "dout must be a tensor of float32, float16 or bfloat16 with a row for each token");
    TORCH_CHECK_VALUE(vocab >= 0, "vocab must not be negative");
    want_cuda(dout, {tokens});
    const c10::cuda::CUDAGuard guard(dout.device());
    const int64_t dim = dout.size(-1);
    const Tensor ids = tokens.contiguous(), rows = unit_stride(dout.reshape({tokens.numel(), dim}));
    Tensor table = empty_like_of({vocab, dim}, rows);
    const Tensor work = scratch(cutespmm_embedding_grad_workspace((uint64_t)ids.numel(), (uint64_t)vocab, u32(dim)), rows);
    check_status(cutespmm_embedding_grad(dtype_of(rows), ptr<void>(rows), ld(rows), ptr<void>(ids), (int)ids.element_size(), (uint64_t)ids.numel(), (uint64_t)vocab, u32(dim), (float)scale,
                                         pointer_of(table), (uint64_t)dim, pointer_of(work), work.defined() ? (uint64_t)work.numel() : 0, stream_of(rows)));
    return table;
}

// ---- attention over selected blocks ----------------------------------------------------------------------------------

// An operand [batch][row][head][dim] with strides the kernels take, copied only where it has others.
struct Operand {
    Tensor t;
    int64_t strides[3];
    explicit Operand(const Tensor &x) : t(x)
    {
        if (!fits()) {
            t = x.contiguous();
            if (!fits()) t = x.clone(at::MemoryFormat::Contiguous);  // contiguous, but off the 16-byte grid
        }
        for (int i = 0; i < 3; ++i) strides[i] = t.numel() && t.size(i) > 1 ? t.stride(i) : 0;  // without elements any strides will do
    }
    bool fits() const
    {
        if (t.numel() == 0) return true;
        if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 || (t.stride(3) != 1 && t.size(3) > 1)) return false;
        for (int i = 0; i < 3; ++i)
            if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8)) return false;
        return true;
    }
};
bool half_type(const Tensor &t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
void check_4d(const Tensor &t, const char *name)
{
    TORCH_CHECK_VALUE(t.dim() == 4 && half_type(t), name, " must be a [batch, row, head, dim] tensor of float16 or bfloat16");
    TORCH_CHECK_VALUE(t.size(3) % 8 == 0 && t.size(3) > 0 && t.size(3) <= 128, name, ": dim must be a multiple of 8, at most 128");
}
void check_block(int64_t block) { TORCH_CHECK_VALUE(block == 16 || block == 32 || block == 64 || block == 128, "block must be 16, 32, 64 or 128"); }
void check_visible(const Tensor &v, int64_t batch, int64_t queries)
{
    TORCH_CHECK_VALUE(!v.defined() || (v.scalar_type() == at::kInt && v.dim() == 2 && v.size(0) == batch && v.size(1) == queries), "visible must be an int32 tensor [batch, queries]");
}
Tensor defined_or_not(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
Tensor contiguous_or_not(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

Tensor op_block_means(const Tensor &k, int64_t block, const OptTensor &lengths_)
{
    const Tensor lengths = contiguous_or_not(defined_or_not(lengths_));
    check_4d(k, "k");
    check_block(block);
    TORCH_CHECK_VALUE(!lengths.defined() || (lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == k.size(0)), "lengths must be an int32 tensor [batch]");
    want_cuda(k, {lengths});
    const c10::cuda::CUDAGuard guard(k.device());
    const Operand x(k);
    Tensor means = empty_like_of({k.size(0), (k.size(1) + block - 1) / block, k.size(2), k.size(3)}, k);
    if (means.numel() == 0) return means;
    check_status(cutespmm_block_means(dtype_of(k), ptr<void>(x.t), x.strides, ptr<int32_t>(lengths), u32(k.size(0)), u32(k.size(1)), u32(k.size(2)), u32(k.size(3)), u32(block),
                                      pointer_of(means), stream_of(k)));
    return means;
}

Tensor op_block_scores(const Tensor &q, const Tensor &means)
{
    check_4d(q, "q");
    check_4d(means, "means");
    TORCH_CHECK_VALUE(q.scalar_type() == means.scalar_type() && q.size(0) == means.size(0) && q.size(3) == means.size(3), "q and means must have the same type, batch and dim");
    TORCH_CHECK_VALUE(means.size(2) > 0 && q.size(2) % means.size(2) == 0, "the heads of q must be a multiple of those of the means");
    want_cuda(q, {means});
    const c10::cuda::CUDAGuard guard(q.device());
    const Operand x(q), m(means);
    Tensor scores = empty_like_of({q.size(0), means.size(2), q.size(1), means.size(1)}, q, at::kFloat);
    if (scores.numel() == 0) return scores;
    check_status(cutespmm_block_scores(dtype_of(q), ptr<void>(x.t), x.strides, ptr<void>(m.t), m.strides, u32(q.size(0)), u32(q.size(1)), u32(q.size(2)), u32(means.size(2)),
                                       u32(means.size(1)), u32(q.size(3)), ptr<float>(scores), stream_of(q)));
    return scores;
}

Tensor op_select_blocks(const Tensor &scores, int64_t count, int64_t block, int64_t keys, const OptTensor &visible_, int64_t first, int64_t last)
{
    const Tensor visible = contiguous_or_not(defined_or_not(visible_));
    TORCH_CHECK_VALUE(scores.dim() == 4 && scores.scalar_type() == at::kFloat, "scores must be a [batch, kv_heads, queries, blocks] float32 tensor");
    check_block(block);
    TORCH_CHECK_VALUE(keys >= 0 && keys < (int64_t)1 << 28 && scores.size(3) == (keys + block - 1) / block, "scores must have a column per block of the ", keys, " keys");
    TORCH_CHECK_VALUE(count >= 0 && first >= 0 && last >= 0 && first <= count && last <= count - first, "first + last must not exceed count");
    check_visible(visible, scores.size(0), scores.size(2));
    want_cuda(scores, {visible});
    const c10::cuda::CUDAGuard guard(scores.device());
    const Tensor s = scores.size(3) <= 1 || scores.stride(3) == 1 ? scores : scores.contiguous();
    Tensor blocks = empty_like_of({s.size(0), s.size(1), s.size(2), count}, s, at::kInt);
    const int64_t strides[3] = {s.stride(0), s.stride(1), s.stride(2)};
    check_status(cutespmm_select_blocks(ptr<float>(s), strides, ptr<int32_t>(visible), u32(s.size(0)), u32(s.size(1)), u32(s.size(2)), u32(s.size(3)), u32(keys), u32(block), u32(count),
                                        u32(first), u32(last), ptr<int32_t>(blocks), stream_of(s)));
    return blocks;
}

// The checked operands of an attention call, alive while it is queued.
struct Attention {
    Operand q, k, v;
    Tensor blocks, visible, pages;
    cutespmm_block_attention_t args{};

    static const Tensor &checked(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block, const Tensor &visible, double scale, const Tensor &pages)
    {
        check_4d(q, "q");
        check_4d(k, "k");
        check_4d(v, "v");
        check_block(block);
        TORCH_CHECK_VALUE((float)scale > 0.f && (float)scale < INFINITY, "scale must be positive and finite");
        TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must have the same type");
        TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "k and v must have the same shape");
        TORCH_CHECK_VALUE(q.size(3) == k.size(3), "q and k must have the same dim");
        TORCH_CHECK_VALUE(k.size(2) > 0 && q.size(2) % k.size(2) == 0, "the heads of q must be a multiple of those of k");
        if (pages.defined()) {
            TORCH_CHECK_VALUE(k.size(1) == block, "a paged cache has pages of `block` keys: k must be [pages, block, kv_heads, dim]");
            TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt && pages.dim() == 2 && pages.size(0) == q.size(0), "pages must be an int32 tensor [batch, pages of a sequence]");
            TORCH_CHECK_VALUE(visible.defined(), "a paged cache needs `visible`: how many of a sequence's keys are written");
        } else
            TORCH_CHECK_VALUE(q.size(0) == k.size(0), "q and k must have the same batch");
        TORCH_CHECK_VALUE(blocks.scalar_type() == at::kInt && blocks.dim() == 4 && blocks.size(0) == q.size(0) && blocks.size(1) == k.size(2) && blocks.size(2) == q.size(1),
                          "blocks must be an int32 tensor [batch, kv_heads, queries, count]");
        check_visible(visible, q.size(0), q.size(1));
        want_cuda(q, {k, v, blocks, visible, pages});
        return q;
    }
    Attention(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &blocks_, int64_t block, const Tensor &visible_, double scale, const Tensor &pages_)
        : q(checked(q_, k_, v_, blocks_, block, visible_, scale, pages_)), k(k_), v(v_), blocks(blocks_.contiguous()), visible(contiguous_or_not(visible_)), pages(contiguous_or_not(pages_))
    {
        const int64_t keys = pages.defined() ? pages.size(1) * block : k_.size(1);
        TORCH_CHECK_VALUE(keys < (int64_t)1 << 28 && q_.size(1) < (int64_t)1 << 28, "more than 2^28 - 1 queries or keys");
        args.struct_size = sizeof args;
        args.dtype = (uint32_t)dtype_of(q_);
        args.batch = u32(q_.size(0)); args.queries = u32(q_.size(1)); args.heads = u32(q_.size(2)); args.kv_heads = u32(k_.size(2)); args.dim = u32(q_.size(3));
        args.keys = u32(keys); args.block = u32(block); args.count = u32(blocks.size(3));
        args.q = ptr<void>(q.t); args.k = ptr<void>(k.t); args.v = ptr<void>(v.t);
        for (int i = 0; i < 3; ++i) {
            args.q_strides[i] = q.strides[i];
            args.k_strides[i] = k.strides[i];
            args.v_strides[i] = v.strides[i];
        }
        args.blocks = ptr<int32_t>(blocks);
        args.visible = ptr<int32_t>(visible);
        args.pages = ptr<int32_t>(pages);
        if (pages.defined()) {
            args.page_cols = u32(pages.size(1));
            args.num_pages = u32(k_.size(0));
        }
        args.scale = (float)scale;
    }
};

std::tuple<Tensor, Tensor> op_block_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block, const OptTensor &visible, double scale, const OptTensor &pages)
{
    c10::cuda::OptionalCUDAGuard guard;
    if (q.is_cuda()) guard.set_device(q.device());
    const Attention at(q, k, v, blocks, block, defined_or_not(visible), scale, defined_or_not(pages));
    Tensor out = empty_like_of(q.sizes(), q), lse = empty_like_of({q.size(0), q.size(2), q.size(1)}, q, at::kFloat);
    if (out.numel()) check_status(cutespmm_block_attention(&at.args, pointer_of(out), ptr<float>(lse), stream_of(q)));
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> op_block_attention_grad(const Tensor &dout, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &out, const Tensor &lse, const Tensor &blocks,
                                                           int64_t block, const OptTensor &visible, double scale)
{
    c10::cuda::OptionalCUDAGuard guard;
    if (q.is_cuda()) guard.set_device(q.device());
    const Attention at(q, k, v, blocks, block, defined_or_not(visible), scale, Tensor());
    TORCH_CHECK_VALUE(dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(),
                      "dout and out must have the shape and type of q");
    TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.sizes() == at::IntArrayRef({q.size(0), q.size(2), q.size(1)}), "lse must be a float32 tensor [batch, heads, queries]");
    want_cuda(q, {dout, out, lse});
    const Operand g(dout);
    Tensor o = out.contiguous();
    if (o.numel() && reinterpret_cast<uintptr_t>(o.const_data_ptr()) % 16) o = o.clone(at::MemoryFormat::Contiguous);  // a view off the 16-byte grid
    const Tensor l = lse.contiguous();
    Tensor dq = empty_like_of(q.sizes(), q), dk = empty_like_of(k.sizes(), k), dv = empty_like_of(v.sizes(), v);
    if (!dq.numel()) return {dq, dk.zero_(), dv.zero_()};
    const Tensor work = scratch(cutespmm_block_attention_grad_workspace(&at.args), q);
    check_status(cutespmm_block_attention_grad(&at.args, ptr<void>(g.t), g.strides, ptr<void>(o), ptr<float>(l), pointer_of(dq), pointer_of(dk), pointer_of(dv), pointer_of(work),
                                               work.defined() ? (uint64_t)work.numel() : 0, stream_of(q)));
    return {dq, dk, dv};
}

// ---- gradients -------------------------------------------------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor call_embedding(const Tensor &tokens, const Tensor &table, double scale)
{
    static auto h = handle<Tensor(const Tensor &, const Tensor &, double)>("cutespmm::embedding");
    return h.call(tokens, table, scale);
}
Tensor call_embedding_grad(const Tensor &tokens, const Tensor &dout, int64_t vocab, double scale)
{
    static auto h = handle<Tensor(const Tensor &, const Tensor &, int64_t, double)>("cutespmm::embedding_grad");
    return h.call(tokens, dout, vocab, scale);
}
Tensor call_block_means(const Tensor &k, int64_t block, const OptTensor &lengths)
{
    static auto h = handle<Tensor(const Tensor &, int64_t, const OptTensor &)>("cutespmm::block_means");
    return h.call(k, block, lengths);
}
Tensor call_block_scores(const Tensor &q, const Tensor &means)
{
    static auto h = handle<Tensor(const Tensor &, const Tensor &)>("cutespmm::block_scores");
    return h.call(q, means);
}
Tensor call_select_blocks(const Tensor &scores, int64_t count, int64_t block, int64_t keys, const OptTensor &visible, int64_t first, int64_t last)
{
    static auto h = handle<Tensor(const Tensor &, int64_t, int64_t, int64_t, const OptTensor &, int64_t, int64_t)>("cutespmm::select_blocks");
    return h.call(scores, count, block, keys, visible, first, last);
}
using AttentionSig = std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t, const OptTensor &, double, const OptTensor &);
std::tuple<Tensor, Tensor> call_block_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block, const OptTensor &visible, double scale, const OptTensor &pages)
{
    static auto h = handle<AttentionSig>("cutespmm::block_attention");
    return h.call(q, k, v, blocks, block, visible, scale, pages);
}

// The two are each other's gradient: a row is copied to each of its tokens, or collected from them.
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
    static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &table, double scale)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        ctx->saved_data["vocab"] = table.dim() ? table.size(0) : 0;
        ctx->saved_data["scale"] = scale;
        ctx->save_for_backward({tokens});
        return call_embedding(tokens, table, scale);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g)
    {
        return {Tensor(), call_embedding_grad(ctx->get_saved_variables()[0], g[0], ctx->saved_data["vocab"].toInt(), ctx->saved_data["scale"].toDouble()), Tensor()};
    }
};
struct EmbeddingGradGrad : torch::autograd::Function<EmbeddingGradGrad> {
    static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &dout, int64_t vocab, double scale)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        ctx->saved_data["scale"] = scale;
        ctx->save_for_backward({tokens});
        return call_embedding_grad(tokens, dout, vocab, scale);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g)
    {
        return {Tensor(), call_embedding(ctx->get_saved_variables()[0], g[0], ctx->saved_data["scale"].toDouble()), Tensor(), Tensor()};
    }
};

struct AttentionGrad : torch::autograd::Function<AttentionGrad> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block, const OptTensor &visible, double scale)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [out, lse] = call_block_attention(q, k, v, blocks, block, visible, scale, std::nullopt);
        ctx->saved_data["block"] = block;
        ctx->saved_data["scale"] = scale;
        ctx->save_for_backward({q, k, v, blocks, defined_or_not(visible), out, lse});
        ctx->mark_non_differentiable({lse});
        return {out, lse};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g)
    {
        static auto h = handle<std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, int64_t,
                                                                  const OptTensor &, double)>("cutespmm::block_attention_grad");
        const variable_list s = ctx->get_saved_variables();
        // it has no gradient of its own: unless a graph of this pass is asked for (and has to name it), go past the kernel that says so
        std::optional<at::AutoDispatchBelowADInplaceOrView> guard;
        if (!c10::GradMode::is_enabled()) guard.emplace();
        const OptTensor visible = s[4].defined() ? OptTensor(s[4]) : std::nullopt;
        auto [dq, dk, dv] = h.call(g[0], s[0], s[1], s[2], s[5], s[6], s[3], ctx->saved_data["block"].toInt(), visible, ctx->saved_data["scale"].toDouble());
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};
std::tuple<Tensor, Tensor> autograd_block_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block, const OptTensor &visible, double scale, const OptTensor &pages)
{
    const bool graph = c10::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    // a tensor with a tangent need not require a gradient: below here it would lose the tangent without a word
    for (const Tensor *t : {&q, &k, &v})
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "block_attention has no forward-mode derivative");
    if (!graph) {
        at::AutoDispatchBelowADInplaceOrView guard;
        return call_block_attention(q, k, v, blocks, block, visible, scale, pages);
    }
    TORCH_CHECK_VALUE(!pages.has_value() || !pages->defined(), "a paged cache has no gradient: call under torch.no_grad(), or with tensors that need none");
    auto r = AttentionGrad::apply(q, k, v, blocks, block, visible, scale);
    return {r[0], r[1]};
}

TORCH_LIBRARY_FRAGMENT(cutespmm, m)
{
    m.def("embedding(Tensor tokens, Tensor table, float scale) -> Tensor");
    m.def("embedding_grad(Tensor tokens, Tensor dout, int vocab, float scale) -> Tensor");
    m.def("block_means(Tensor k, int block, Tensor? lengths) -> Tensor");
    m.def("block_scores(Tensor q, Tensor means) -> Tensor");
    m.def("select_blocks(Tensor scores, int count, int block, int keys, Tensor? visible, int first, int last) -> Tensor");
    m.def("block_attention(Tensor q, Tensor k, Tensor v, Tensor blocks, int block, Tensor? visible, float scale, Tensor? pages) -> (Tensor, Tensor)");
    m.def("block_attention_grad(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor blocks, int block, Tensor? visible, float scale) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(cutespmm, CompositeExplicitAutograd, m)
{
    m.impl("embedding", op_embedding);
    m.impl("embedding_grad", op_embedding_grad);
    m.impl("block_means", op_block_means);
    m.impl("block_scores", op_block_scores);
    m.impl("select_blocks", op_select_blocks);
    m.impl("block_attention", op_block_attention);
    m.impl("block_attention_grad", op_block_attention_grad);
}
TORCH_LIBRARY_IMPL(cutespmm, Autograd, m)
{
    m.impl("embedding", [](const Tensor &tokens, const Tensor &table, double scale) { return EmbeddingGrad::apply(tokens, table, scale); });
    m.impl("embedding_grad", [](const Tensor &tokens, const Tensor &dout, int64_t vocab, double scale) { return EmbeddingGradGrad::apply(tokens, dout, vocab, scale); });
    m.impl("block_attention", autograd_block_attention);
    // without one of these a backward pass through them would go on with zeros and a warning
    m.impl("block_means", torch::autograd::autogradNotImplementedFallback());
    m.impl("block_scores", torch::autograd::autogradNotImplementedFallback());
    m.impl("select_blocks", torch::autograd::autogradNotImplementedFallback());
    m.impl("block_attention_grad", torch::autograd::autogradNotImplementedFallback());
}

// ---- calls without the packet lookup of torch.ops ----------------------------------------------------------------------

int64_t signed_integer(PyObject *o)
{
    const int64_t v = (int64_t)PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double number(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
OptTensor optional_tensor(PyObject *o, const char *what) { return o == Py_None ? OptTensor() : OptTensor(tensor(o, what)); }

PyObject *py_embedding(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    want_args(n, 3);
    const Tensor tokens = tensor(a[0], "tokens"), table = tensor(a[1], "table");
    const double scale = number(a[2]);
    return THPVariable_Wrap(without_gil([&] { return call_embedding(tokens, table, scale); }));
    END_HANDLE_TH_ERRORS
}
PyObject *py_block_means(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    want_args(n, 3);
    const Tensor k = tensor(a[0], "k");
    const int64_t block = signed_integer(a[1]);
    const OptTensor lengths = optional_tensor(a[2], "lengths");
    return THPVariable_Wrap(without_gil([&] { return call_block_means(k, block, lengths); }));
    END_HANDLE_TH_ERRORS
}
PyObject *py_block_scores(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    want_args(n, 2);
    const Tensor q = tensor(a[0], "q"), means = tensor(a[1], "means");
    return THPVariable_Wrap(without_gil([&] { return call_block_scores(q, means); }));
    END_HANDLE_TH_ERRORS
}
PyObject *py_select_blocks(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    want_args(n, 7);
    const Tensor scores = tensor(a[0], "scores");
    const int64_t count = signed_integer(a[1]), block = signed_integer(a[2]), keys = signed_integer(a[3]), first = signed_integer(a[5]), last = signed_integer(a[6]);
    const OptTensor visible = optional_tensor(a[4], "visible");
    return THPVariable_Wrap(without_gil([&] { return call_select_blocks(scores, count, block, keys, visible, first, last); }));
    END_HANDLE_TH_ERRORS
}
PyObject *py_block_attention(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    want_args(n, 8);
    const Tensor q = tensor(a[0], "q"), k = tensor(a[1], "k"), v = tensor(a[2], "v"), blocks = tensor(a[3], "blocks");
    const int64_t block = signed_integer(a[4]);
    const OptTensor visible = optional_tensor(a[5], "visible"), pages = optional_tensor(a[7], "pages");
    const double scale = number(a[6]);
    return THPVariable_Wrap(without_gil([&] { return std::get<0>(call_block_attention(q, k, v, blocks, block, visible, scale, pages)); }));
    END_HANDLE_TH_ERRORS
}
PyObject *py_pattern_status(PyObject *, PyObject *const *, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    want_args(n, 0);
    uint32_t status = 0;
    without_gil([&] { check_status(cutespmm_pattern_status(&status)); });
    return PyLong_FromUnsignedLong(status);
    END_HANDLE_TH_ERRORS
}

#define FAST(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_pattern_methods[] = {FAST("op_embedding", py_embedding), FAST("op_block_means", py_block_means), FAST("op_block_scores", py_block_scores),
                                   FAST("op_select_blocks", py_select_blocks), FAST("op_block_attention", py_block_attention), FAST("pattern_status", py_pattern_status),
                                   {nullptr, nullptr, 0, nullptr}};

}  // namespace

int bind::add_pattern_calls(PyObject *module) { return PyModule_AddFunctions(module, g_pattern_methods); }
