"""Operators whose sparse pattern the data choose in each call (cutespmm_ae_b200/torch_ops.py): embedding and its gradient, mean keys,
scores, selection, attention over the selected blocks and its gradients, against plain forms in 64 bits.

Tolerances.  Inputs are given in the tested type, so the plain form starts from the same numbers.  u = eps / 2 is half a step of the type,
u32 that of float32.
  * A sum of n float32 terms is off by at most (n + 2) u32 times the sum of their magnitudes; one rounding to the type adds u times the
    result.
  * Attention: P is rounded to the type before the product with V (u each, the sum is taken before that), out is rounded once (u): at most
    2 u sum(p |v|), and the float32 parts: a score s is off by (dim + 2) u32 sum |q k| scale, so p by that much relatively (and as much
    again through the sum), the exponential itself by 4 u32 and its argument by u32 |s|.
  * Gradients: dS = P (D - delta) with P unrounded, D off by (dim + 2) u32 sum |dout v|, delta formed from the rounded out: off by
    u sum |dout out|; dS is rounded to the type (u), P is rounded for dv (u), results once (u).
The bounds below are these, element by element, computed in 64 bits next to the reference."""
import math

import numpy as np
import pytest
import torch

import cutespmm_ae_b200 as cs
from cutespmm_ae_b200 import torch_ops as ops

U32 = torch.finfo(torch.float32).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of the smallest numbers: what a rounding near zero is off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, bound):
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {float(((got - want).abs() / bound.clamp(min=1e-300))[bad].max()):.3g} times the bound"


@pytest.fixture(autouse=True)
def _no_wait_gave_up(request):
    yield
    if request.node.get_closest_marker("gpu"):
        assert ops.pattern_status() == 0


# ---- embedding -----------------------------------------------------------------------------------------------------


def embedding_reference(tokens, table, scale):
    named = (tokens >= 0) & (tokens < table.shape[0])
    return table.double()[torch.where(named, tokens, 0).long()] * scale * named[..., None]


def check_embedding(tokens, table, scale, dout=None):
    u = half_step(table.dtype)
    x = table.detach().clone().requires_grad_(True)
    out = ops.embedding(tokens, x, scale)
    want = embedding_reference(tokens, table, scale)
    assert out.dtype == table.dtype and out.shape == want.shape
    within(out, want, want.abs() * (u + 3 * U32) + tiny(table.dtype))
    if dout is None:
        dout = torch.randn(out.shape, device="cuda").to(table.dtype)
    (got,) = torch.autograd.grad(out, x, dout)
    named = ((tokens >= 0) & (tokens < table.shape[0])).flatten()
    row = tokens.flatten()[named].long()
    g = dout.reshape(-1, table.shape[1])[named].double()
    want = torch.zeros(table.shape, device="cuda", dtype=torch.float64).index_add_(0, row, g) * scale
    size = torch.zeros(table.shape, device="cuda", dtype=torch.float64).index_add_(0, row, g.abs()) * abs(scale)
    n = torch.bincount(row, minlength=table.shape[0])[:, None]
    assert got.dtype == table.dtype and got.shape == table.shape
    within(got, want, size * (n + 3) * U32 + want.abs() * u + tiny(table.dtype) * (n > 0))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 8), (1, 1000, 4096), (37, 5, 24), (4097, 511, 72), (2048, 512, 1000), (3001, 513, 33), (700, 262144, 16), (5000, 300001, 7), (9000, 3, 520)])
def test_embedding_and_its_gradient(dtype, tokens, vocab, dim):
    """Tables from one row on, vocabularies on both sides of a digit of the sort (512, 262144), rows off the 16-byte grid, words that
    nearly every token names (pieces of a long sum), padded positions on both sides of the vocabulary."""
    torch.manual_seed(tokens + vocab)
    ids = torch.randint(-1, vocab + 1, (tokens,), device="cuda")
    ids[torch.rand(tokens, device="cuda") < 0.2] = vocab // 2
    check_embedding(ids, torch.randn(vocab, dim, device="cuda").to(dtype), 1.7)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [(511,), (512,), (513,), (257, 600, 1, 5000, 300), (100, 513, 14, 2000, 1, 1, 1025)])
def test_embedding_gradient_of_long_sums(lengths):
    """Words named by so many tokens that their sum is cut into pieces, beginning at every place of a chunk and a piece."""
    torch.manual_seed(len(lengths))
    ids = torch.cat([torch.full((n,), 3 * i + 1, device="cuda", dtype=torch.int32) for i, n in enumerate(lengths)])
    ids = ids[torch.randperm(len(ids), device="cuda")]
    a = check_embedding(ids, torch.randn(40, 136, device="cuda"), 0.5, torch.randn(len(ids), 136, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    b = check_embedding(ids, torch.randn(40, 136, device="cuda"), 0.5, torch.randn(len(ids), 136, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    assert torch.equal(a, b)  # the same bits in every run


@pytest.mark.gpu
def test_embedding_shapes_views_and_empties():
    torch.manual_seed(2)
    table = torch.randn(100, 48, device="cuda")
    ids = torch.randint(0, 100, (3, 5, 2), device="cuda", dtype=torch.int32)
    assert check_embedding(ids, table, -2.0).shape == table.shape
    wide = torch.randn(100, 100, device="cuda")
    assert torch.equal(ops.embedding(ids, wide[:, 1:50], 1.0), wide[:, 1:50][ids.long()])  # rows off the 16-byte grid
    assert torch.equal(ops.embedding(ids, wide.t(), 1.0), wide.t()[ids.long()])            # columns apart
    assert torch.equal(ops.embedding(ids.transpose(0, 2), table), table[ids.transpose(0, 2).long()])
    assert torch.equal(ops.embedding(torch.full((4,), -1, device="cuda"), table), torch.zeros(4, 48, device="cuda"))
    assert torch.equal(ops.embedding(torch.tensor([2**40, 2**31, -(2**40), 99], device="cuda"), table)[:3], torch.zeros(3, 48, device="cuda"))
    assert ops.embedding(ids[:0], table).shape == (0, 5, 2, 48)
    assert ops.embedding(ids, table[:, :0]).shape == (3, 5, 2, 0)
    assert torch.equal(ops.embedding(ids, table[:0]), torch.zeros(3, 5, 2, 48, device="cuda"))
    x = table.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.embedding(ids[:0], x).sum(), x)
    assert torch.equal(g, torch.zeros_like(table))
    (g,) = torch.autograd.grad(ops.embedding(ids, x, 3.0).sum(), x)  # a gradient that is one number everywhere
    assert torch.equal(g, 3.0 * torch.bincount(ids.flatten().long(), minlength=100)[:, None].expand(100, 48))
    assert not torch.isnan(ops.embedding(ids, torch.full((100, 48), math.nan, device="cuda"))).logical_not().any()


@pytest.mark.gpu
def test_embedding_second_derivative():
    """The gradient is linear in dout; its own gradient is the embedding again."""
    torch.manual_seed(3)
    ids = torch.tensor([1, 1, 4, -1, 0], device="cuda")
    x = torch.randn(6, 8, device="cuda").requires_grad_(True)
    (ops.embedding(ids, x, 2.0) ** 3).sum().backward(create_graph=True)
    g, x.grad = x.grad, None
    (g * g).sum().backward()
    y = x.detach().double().requires_grad_(True)
    loss = ((2.0 * y[ids.clamp(min=0)] * (ids >= 0)[:, None]) ** 3).sum()
    (h,) = torch.autograd.grad(loss, y, create_graph=True)
    (want,) = torch.autograd.grad((h * h).sum(), y)
    within(x.grad, want, want.abs() * 40 * U32 + 1e-30)


# ---- means, scores, selection --------------------------------------------------------------------------------------


def blocks_of(keys, block):
    return (keys + block - 1) // block


def means_reference(k, block, lengths=None):
    batch, keys, kv, dim = k.shape
    mean = torch.zeros(batch, blocks_of(keys, block), kv, dim, device=k.device, dtype=torch.float64)
    size = torch.zeros_like(mean)
    for b in range(batch):
        n = keys if lengths is None else min(max(int(lengths[b]), 0), keys)
        for j in range(blocks_of(n, block)):
            part = k[b, j * block : min((j + 1) * block, n)].double()
            mean[b, j], size[b, j] = part.mean(0), part.abs().mean(0)
    return mean, size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,keys,kv,dim,block", [(1, 1, 1, 8, 16), (2, 63, 3, 64, 64), (3, 130, 2, 128, 32), (1, 1000, 5, 104, 128), (2, 77, 1, 72, 16)])
def test_block_means(dtype, batch, keys, kv, dim, block):
    torch.manual_seed(keys)
    k = torch.randn(batch, keys, kv, dim, device="cuda").to(dtype)
    want, size = means_reference(k, block)
    within(ops.block_means(k, block), want, want.abs() * half_step(dtype) + size * (block + 3) * U32 + tiny(dtype))
    lengths = torch.tensor([0, keys // 2, keys + 5][:batch], device="cuda", dtype=torch.int32)
    for b in range(batch):
        k[b, min(int(lengths[b]), keys) :] = math.nan  # keys that are not written yet
    want, size = means_reference(k, block, lengths)
    within(ops.block_means(k, block, lengths), want, want.abs() * half_step(dtype) + size * (block + 3) * U32 + tiny(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,queries,kv,group,dim,blocks", [(1, 1, 1, 1, 64, 1), (2, 129, 2, 3, 72, 33), (1, 300, 1, 8, 128, 257), (3, 64, 4, 2, 8, 100), (1, 40, 2, 16, 80, 600), (2, 1400, 3, 1, 64, 1300), (7, 260, 3, 2, 128, 530)])
def test_block_scores(dtype, batch, queries, kv, group, dim, blocks):
    torch.manual_seed(queries)
    q = torch.randn(batch, queries, kv * group, dim, device="cuda").to(dtype)
    means = torch.randn(batch, blocks, kv, dim, device="cuda").to(dtype)
    q5 = q.double().view(batch, queries, kv, group, dim)
    want = torch.einsum("btkgd,bnkd->bktn", q5, means.double())
    size = torch.einsum("btkgd,bnkd->bktn", q5.abs(), means.double().abs())
    within(ops.block_scores(q, means), want, size * (group * dim + 2) * U32)
    # rows with gaps, and operands that have to be copied
    wide = torch.randn(batch, queries, kv * group, dim + 24, device="cuda").to(dtype)
    assert torch.equal(ops.block_scores(wide[..., 8 : dim + 8], means), ops.block_scores(wide[..., 8 : dim + 8].contiguous(), means))
    assert torch.equal(ops.block_scores(wide[..., 3 : dim + 3], means), ops.block_scores(wide[..., 3 : dim + 3].contiguous(), means))
    assert torch.equal(ops.block_scores(q.transpose(1, 2).contiguous().transpose(1, 2), means), ops.block_scores(q, means))


def selection_reference(scores, count, block, keys, visible, first, last):
    """Row by row, by sorting (score descending, index ascending)."""
    batch, kv, queries, blocks = scores.shape
    out = np.full((batch, kv, queries, count), -1, dtype=np.int32)
    s = scores.cpu().numpy()
    for b in range(batch):
        for t in range(queries):
            v = keys - queries + 1 + t if visible is None else int(visible[b, t])
            n = min(blocks_of(min(max(v, 0), keys), block), blocks)
            forced = [j for j in range(n) if j < first or j >= n - last]
            for h in range(kv):
                row = s[b, h, t]
                rest = sorted((j for j in range(n) if j not in forced and row[j] > -math.inf), key=lambda j: (-row[j], j))
                chosen = sorted((forced + rest)[:count])
                out[b, h, t, : len(chosen)] = chosen
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("batch,kv,queries,keys,block,count,first,last", [(1, 1, 1, 1, 16, 1, 0, 0), (2, 3, 65, 65, 16, 3, 1, 1), (1, 2, 37, 1000, 16, 8, 2, 3), (2, 1, 5, 4000, 32, 128, 0, 1),
                                                                          (1, 2, 1500, 1500, 64, 4, 1, 2), (1, 1, 3, 20000, 16, 16, 1, 1), (2, 2, 2, 70000, 16, 33, 0, 0), (1, 1, 1, 262144, 16, 128, 5, 7),
                                                                          (1, 1, 2400, 3000, 128, 30, 1, 1), (1, 4, 600, 8000, 16, 20, 1, 1), (3, 1, 900, 5000, 16, 40, 0, 0)])
def test_select_blocks(batch, kv, queries, keys, block, count, first, last):
    """Every size class of the kernel, ties, equal scores of both signs, infinities, NaN, rows that see nothing and rows that see less than count."""
    torch.manual_seed(keys + count)
    blocks = blocks_of(keys, block)
    for kind in range(3):
        scores = torch.randn(batch, kv, queries, blocks, device="cuda")
        visible = None
        if kind == 1:  # few distinct values
            scores = (scores * 1.5).round() * torch.where(torch.rand_like(scores) < 0.5, -1.0, 1.0)
            visible = torch.randint(0, keys + 1, (batch, queries), device="cuda", dtype=torch.int32)
        if kind == 2:
            r = torch.rand_like(scores)
            scores = torch.where(r < 0.3, math.nan, torch.where(r < 0.6, -math.inf, torch.where(r < 0.62, math.inf, torch.where(r < 0.7, torch.finfo(torch.float32).min, scores))))
            visible = torch.randint(-3, keys + 9, (batch, queries), device="cuda", dtype=torch.int32)
            visible[:, 0] = 0
        got = ops.select_blocks(scores, count, block, keys, visible, first, last)
        assert got.dtype == torch.int32
        assert np.array_equal(got.cpu().numpy(), selection_reference(scores, count, block, keys, visible, first, last))
    assert torch.equal(ops.select_blocks(scores.transpose(1, 2).contiguous().transpose(1, 2), count, block, keys, visible, first, last), got)


# ---- attention -----------------------------------------------------------------------------------------------------


def default_visible(batch, queries, keys):
    return (torch.arange(queries, device="cuda", dtype=torch.int32) + (keys - queries + 1)).expand(batch, queries).contiguous()


def pattern_of(blocks, block, keys, visible):
    """[batch, kv, queries, keys]: whether the query looks at the key."""
    n = blocks_of(keys, block)
    names = torch.zeros(*blocks.shape[:3], n + 1, device="cuda", dtype=torch.bool)
    names.scatter_(3, torch.where((blocks >= 0) & (blocks < n), blocks, n).long(), True)
    seen = torch.arange(keys, device="cuda") < visible.clamp(0, keys)[:, None, :, None]
    return names[..., :n].repeat_interleave(block, 3)[..., :keys] & seen


def attention_reference(q, k, v, pattern, scale, dout=None):
    """(out, its bound) and, with dout, the gradients and their bounds, in 64 bits."""
    dtype = q.dtype
    u = half_step(dtype)
    batch, queries, heads, dim = q.shape
    kv = k.shape[2]
    group = heads // kv
    q5 = q.double().view(batch, queries, kv, group, dim).permute(0, 2, 3, 1, 4)
    some = pattern.any(2)[..., None]  # keys that nobody looks at may hold anything
    k5, v5 = (torch.where(some, t.double().permute(0, 2, 1, 3), 0.0)[:, :, None] for t in (k, v))
    m = pattern[:, :, None]
    s = (q5 @ k5.transpose(3, 4)) * scale
    s_err = (q5.abs() @ k5.abs().transpose(3, 4)) * abs(scale) * (dim + 2) * U32 + s.abs() * 3 * U32 + 8 * U32
    s = s.masked_fill(~m, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total.clamp(min=1e-300), 0.0)
    s_err = torch.where(m, s_err, 0.0)
    p_err = p * (s_err + (p * s_err).sum(-1, keepdim=True) + pattern.shape[-1] * U32 + 8 * U32)  # of P in float32, to first order
    out = p @ v5
    pv = p @ v5.abs()
    out_err = 2.05 * (p_err @ v5.abs()) + u * pv * 1.02 + u * out.abs() * 1.02 + pv * (pattern.shape[-1] + 4) * U32
    back = lambda t: t.permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, -1)  # noqa: E731
    near0 = tiny(dtype) * 4
    result = [(back(out), back(out_err) + near0)]
    if dout is not None:
        d5 = dout.double().view(batch, queries, kv, group, dim).permute(0, 2, 3, 1, 4)
        rows = p.sum(-1, keepdim=True) > 0
        d5 = torch.where(rows, d5, 0.0)
        dp = d5 @ v5.transpose(3, 4)
        delta = (d5 * out).sum(-1, keepdim=True)
        dp_err = (d5.abs() @ v5.abs().transpose(3, 4)) * (dim + 2) * U32
        delta_err = (d5.abs() * (out_err + near0)).sum(-1, keepdim=True) + (d5 * out).abs().sum(-1, keepdim=True) * (dim + 2) * U32
        ds = p * (dp - delta)
        ds_err = 1.05 * (p_err * (dp - delta).abs() + p * (dp_err + delta_err)) + 1.02 * u * ds.abs() + tiny(dtype)
        ds_err = torch.where(m, ds_err, 0.0)
        n = max(pattern.shape[-1], queries * group)
        shared = lambda t: t.sum(2).permute(0, 2, 1, 3)  # noqa: E731
        dq, dq_err = scale * (ds @ k5), abs(scale) * (ds_err @ k5.abs() + (ds.abs() @ k5.abs()) * (n + 4) * U32)
        dk, dk_err = scale * (ds.transpose(3, 4) @ q5), abs(scale) * (ds_err.transpose(3, 4) @ q5.abs() + (ds.abs().transpose(3, 4) @ q5.abs()) * (n + 4) * U32)
        pw = torch.where(m, p_err * 1.05 + 1.02 * u * p + tiny(dtype), 0.0)
        dv, dv_err = p.transpose(3, 4) @ d5, pw.transpose(3, 4) @ d5.abs() + (p.transpose(3, 4) @ d5.abs()) * (n + 4) * U32
        result += [(back(dq), back(dq_err + u * dq.abs()) + near0)]
        result += [(shared(dk), shared(dk_err) + u * shared(dk).abs() * 1.02 + near0), (shared(dv), shared(dv_err) + u * shared(dv).abs() * 1.02 + near0)]
    return result


def random_blocks(batch, kv, queries, count, keys, block, share=0.6):
    """Neighbouring queries share some of their blocks; entries in any order, some empty, some outside, some twice."""
    n = blocks_of(keys, block)
    common = torch.randint(-1, n + 1, (batch, kv, (queries + 7) // 8, count), device="cuda").repeat_interleave(8, 2)[:, :, :queries]
    own = torch.randint(-1, n + 1, (batch, kv, queries, count), device="cuda")
    return torch.where(torch.rand(own.shape, device="cuda") < share, common, own).int()


def attention_inputs(dtype, batch, queries, keys, kv, group, dim):
    q = torch.randn(batch, queries, kv * group, dim, device="cuda").to(dtype)
    k, v = (torch.randn(batch, keys, kv, dim, device="cuda").to(dtype) for _ in range(2))
    return q, k, v


def check_attention(q, k, v, blocks, block, visible=None, scale=None, grad=True, dout=None):
    keys = k.shape[1]
    see = default_visible(q.shape[0], q.shape[1], keys) if visible is None else visible
    pattern = pattern_of(blocks, block, keys, see)
    dout = torch.randn(q.shape, device="cuda").to(q.dtype) if grad and dout is None else dout
    want = attention_reference(q, k, v, pattern, 1 / math.sqrt(q.shape[3]) if scale is None else scale, dout if grad else None)
    leaves = [t.detach().requires_grad_(grad) for t in (q, k, v)]
    out = ops.block_attention(*leaves, blocks, block, visible, scale)
    assert out.dtype == q.dtype and out.shape == q.shape
    got = [out, *torch.autograd.grad(out, leaves, dout)] if grad else [out]
    for g, (w, bound) in zip(got, want):
        within(g, w, bound)
    return got


FORMS = [  # batch, queries, keys, kv, group, dim, block, count
    (1, 1, 1, 1, 1, 64, 16, 1),
    (1, 5, 5, 1, 8, 128, 64, 1),
    (2, 70, 70, 2, 8, 128, 64, 2),
    (1, 200, 200, 1, 1, 64, 16, 5),
    (2, 130, 130, 3, 2, 72, 32, 3),
    (1, 150, 333, 2, 4, 128, 128, 2),
    (1, 97, 400, 1, 3, 80, 16, 9),
    (1, 90, 260, 2, 16, 128, 64, 4),
    (1, 40, 300, 1, 12, 96, 32, 6),
    (1, 33, 129, 1, 65, 64, 64, 3),
    (1, 20, 100, 1, 128, 128, 32, 3),
    (1, 300, 2000, 1, 8, 64, 16, 128),
    (1, 600, 600, 1, 7, 8, 64, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", FORMS)
def test_attention_and_its_gradients(dtype, form):
    batch, queries, keys, kv, group, dim, block, count = form
    torch.manual_seed(queries + dim)
    q, k, v = attention_inputs(dtype, batch, queries, keys, kv, group, dim)
    check_attention(q, k, v, random_blocks(batch, kv, queries, count, keys, block), block)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,group,dim,block,count", [(1, 1, 8, 16, 128), (1, 2, 128, 32, 100), (2, 8, 64, 16, 60)])
def test_many_blocks_of_a_long_cache(kv, group, dim, block, count):
    """Queries whose blocks lie all over a cache of 150000 keys: tiles of queries get smaller where their lists would not fit."""
    torch.manual_seed(group)
    q, k, v = attention_inputs(torch.bfloat16, 1, 130, 150000, kv, group, dim)
    check_attention(q, k, v, random_blocks(1, kv, 130, count, 150000, block, share=0.1), block, grad=group < 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", [(2, 65, 300, 2, 8, 128, 64, 4), (2, 65, 300, 2, 1, 64, 16, 8), (3, 40, 100, 1, 4, 64, 32, 3), (2, 50, 256, 1, 2, 128, 128, 2)])
def test_rows_that_see_nothing_and_keys_that_nobody_sees(dtype, form):
    """visible of 0 and below, beyond the keys, and keys behind it that hold NaN and infinities: no trace of them in any result."""
    batch, queries, keys, kv, group, dim, block, count = form
    torch.manual_seed(7)
    q, k, v = attention_inputs(dtype, batch, queries, keys, kv, group, dim)
    visible = torch.randint(-2, keys // 2, (batch, queries), device="cuda", dtype=torch.int32)
    visible[0] = keys + 100
    visible[0, ::3] = 0
    visible[-1, queries // 2 :] = 0
    top = visible.amax(1).clamp(max=keys)
    for b in range(batch):
        k[b, top[b] :] = math.nan
        v[b, top[b] :] = math.inf
    blocks = random_blocks(batch, kv, queries, count, keys, block)
    blocks[0, :, 5] = -1
    dout = torch.randn(q.shape, device="cuda").to(dtype)
    dout[visible <= 0] = math.nan  # padded positions: nothing of them reaches a gradient
    got = check_attention(q, k, v, blocks, block, visible, dout=dout)
    assert not got[0][visible <= 0].any() and not got[1][visible <= 0].any()
    assert not got[0][0, 5].any()
    # a key that later queries see may hold anything as far as earlier ones are concerned, and so may a block that others name
    late = default_visible(batch, queries, keys)
    q, k, v = attention_inputs(dtype, batch, queries, keys, kv, group, dim)
    blocks[:, :, : queries // 2] = torch.where(blocks[:, :, : queries // 2] == 0, -1, blocks[:, :, : queries // 2])
    pattern = pattern_of(blocks, block, keys, late)
    clean = ~pattern[..., [0, -1]].any(-1).any(1)  # queries that look at neither key 0 nor the last
    dout = torch.randn(q.shape, device="cuda").to(dtype)
    (want, bound), (want_dq, bound_dq) = attention_reference(q, k, v, pattern, 1 / math.sqrt(dim), dout)[:2]
    k[:, -1], v[:, -1] = math.nan, math.inf
    k[:, 0], v[:, 0] = -math.inf, math.nan
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = ops.block_attention(*leaves, blocks, block, late)
    within(out[clean], want[clean], bound[clean])
    (dq,) = torch.autograd.grad(out, q, dout)
    within(dq[clean], want_dq[clean], bound_dq[clean])
    few = slice(queries - 4, queries)
    with torch.no_grad():
        out = ops.block_attention(q[:, few], k, v, blocks[:, :, few].contiguous(), block, late[:, few].contiguous())
    within(out[clean[:, few]], want[:, few][clean[:, few]], bound[:, few][clean[:, few]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,queries,keys,kv,group,dim,block,count", [(1, 1, 1, 1, 1, 64, 16, 1), (3, 1, 700, 2, 8, 128, 64, 6), (2, 4, 5000, 1, 4, 64, 16, 128), (1, 2, 3000, 2, 12, 128, 128, 20),
                                                                         (2, 1, 4000, 1, 40, 96, 32, 64), (5, 3, 200, 3, 1, 72, 16, 7), (40, 1, 900, 4, 8, 128, 64, 8)])
def test_single_tokens(dtype, batch, queries, keys, kv, group, dim, block, count):
    """One to four queries over a long cache of different lengths, contiguous and paged: the same result, and pages that do not exist are as if
    their keys were not there."""
    torch.manual_seed(keys)
    q, k, v = attention_inputs(dtype, batch, queries, keys, kv, group, dim)
    visible = torch.randint(0, keys + 1, (batch, queries), device="cuda", dtype=torch.int32)
    blocks = random_blocks(batch, kv, queries, count, keys, block)
    (out,) = check_attention(q, k, v, blocks, block, visible, scale=0.2, grad=False)
    n = blocks_of(keys, block)
    pages = torch.randperm(batch * n + 3, device="cuda")[: batch * n].view(batch, n).int()
    cache = []
    for t in (k, v):
        c = torch.full((batch * n + 3, block, kv, dim), math.nan, device="cuda", dtype=dtype)
        padded = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, n * block - keys))
        c[pages.long().flatten()] = padded.view(batch * n, block, kv, dim)
        cache.append(c)
    assert torch.equal(ops.block_attention(q, *cache, blocks, block, visible, 0.2, pages), out)
    # pages that do not exist
    gone = torch.rand(pages.shape, device="cuda") < 0.4
    broken = torch.where(gone, torch.where(torch.rand(pages.shape, device="cuda") < 0.5, -5, batch * n + 3), pages).int()
    kept = torch.where((blocks >= 0) & (blocks < n), blocks, 0).long()
    lost = torch.gather(gone[:, None, None].expand(batch, kv, queries, n), 3, kept)
    fewer = torch.where(lost, -1, blocks)
    assert torch.equal(ops.block_attention(q, *cache, blocks, block, visible, 0.2, broken), ops.block_attention(q, *cache, fewer, block, visible, 0.2, pages))


@pytest.mark.gpu
def test_a_paged_prompt():
    torch.manual_seed(11)
    batch, queries, keys, kv, group, dim, block, count = 2, 70, 320, 2, 8, 128, 64, 3
    q, k, v = attention_inputs(torch.bfloat16, batch, queries, keys, kv, group, dim)
    blocks, visible = random_blocks(batch, kv, queries, count, keys, block), default_visible(batch, queries, keys)
    n = keys // block
    pages = torch.randperm(batch * n, device="cuda").view(batch, n).int()
    cache = []
    for t in (k, v):
        c = torch.empty(batch * n, block, kv, dim, device="cuda", dtype=t.dtype)
        c[pages.long().flatten()] = t.view(batch * n, block, kv, dim)
        cache.append(c)
    assert torch.equal(ops.block_attention(q, *cache, blocks, block, visible, None, pages), ops.block_attention(q, k, v, blocks, block, visible))
    with pytest.raises(ValueError, match="no gradient"):
        ops.block_attention(q.requires_grad_(True), *cache, blocks, block, visible, None, pages)


@pytest.mark.gpu
def test_attention_views_and_extreme_scores():
    torch.manual_seed(12)
    q, k, v = attention_inputs(torch.bfloat16, 2, 60, 60, 2, 4, 64)
    blocks = random_blocks(2, 2, 60, 3, 60, 16)
    want = check_attention(q, k, v, blocks, 16)
    packed = torch.cat([t.reshape(2, 60, -1) for t in (q, k, v)], 2)  # one tensor that holds the three
    a, b, c = packed[..., :512].view(2, 60, 8, 64), packed[..., 512:640].view(2, 60, 2, 64), packed[..., 640:].view(2, 60, 2, 64)
    assert torch.equal(ops.block_attention(a, b, c, blocks, 16), want[0])
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(ops.block_attention(*heads_first, blocks, 16), want[0])
    off = [torch.cat([torch.zeros(2, 60, t.shape[2], 3, device="cuda", dtype=t.dtype), t], 3)[..., 3:] for t in (q, k, v)]
    assert torch.equal(ops.block_attention(*off, blocks, 16), want[0])
    check_attention(q, k[:, :, :1].expand(2, 60, 2, 64), v[:, :1].expand(2, 60, 2, 64), blocks, 16)
    # scores so far apart that all but one exponential vanish, and so large that a sum of them would overflow
    check_attention(q * 12, k * 12, v, blocks, 16, grad=False)
    check_attention(q, k, v, blocks, 16, scale=3.0)
    check_attention(q, k, v, blocks, 16, scale=1e-6)
    # a gradient with strides of its own, and one that is the same number everywhere
    check_attention(q, k, v, blocks, 16, dout=torch.randn(2, 8, 60, 64, device="cuda").bfloat16().transpose(1, 2))
    check_attention(q, k, v, blocks, 16, dout=torch.ones(1, 1, 1, 1, device="cuda", dtype=torch.bfloat16).expand(2, 60, 8, 64))


@pytest.mark.gpu
def test_empty_attention():
    q, k, v = attention_inputs(torch.float16, 2, 9, 32, 1, 2, 64)
    blocks = torch.zeros(2, 1, 9, 2, device="cuda", dtype=torch.int32)
    for i in ((slice(0, 0), slice(None)), (slice(None), slice(0, 0))):
        out = ops.block_attention(q[i], k[i[0]], v[i[0]], blocks[i[0], :, i[1]], 16)
        assert out.shape == q[i].shape
    leaves = [t.requires_grad_(True) for t in (q, k[:, :0].detach().clone(), v[:, :0].detach().clone())]
    out = ops.block_attention(*leaves, blocks, 16)
    grads = torch.autograd.grad(out.sum(), leaves)
    assert not out.any() and not grads[0].any() and grads[1].shape == (2, 0, 1, 64)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.block_attention(*leaves, blocks[..., :0], 16)
    assert not out.any() and not any(g.any() for g in torch.autograd.grad(out.sum(), leaves))


@pytest.mark.gpu
def test_gradients_against_differences():
    """<gradient, direction> against a difference of the plain form in 64 bits along that direction."""
    torch.manual_seed(13)
    q, k, v = attention_inputs(torch.bfloat16, 1, 64, 64, 2, 8, 64)
    blocks = random_blocks(1, 2, 64, 3, 64, 16)
    pattern = pattern_of(blocks, 16, 64, default_visible(1, 64, 64))
    dout = torch.randn(q.shape, device="cuda").bfloat16()
    grads = check_attention(q, k, v, blocks, 16, dout=dout)[1:]
    want = attention_reference(q, k, v, pattern, 0.125, dout)[1:]

    def loss(*x):
        q5 = x[0].view(1, 64, 2, 8, 64).permute(0, 2, 3, 1, 4)
        k5, v5 = (t.permute(0, 2, 1, 3)[:, :, None] for t in x[1:])
        s = (q5 @ k5.transpose(3, 4) * 0.125).masked_fill(~pattern[:, :, None], -math.inf)
        p = torch.softmax(s, -1).nan_to_num()
        return ((p @ v5).permute(0, 3, 1, 2, 4).reshape(1, 64, 16, 64) * dout.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i in range(3):
        direction = torch.randn(x[i].shape, device="cuda", dtype=torch.float64)
        h = 1e-5
        plus, minus = ([t + s * h * direction if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        slope = float(loss(*plus) - loss(*minus)) / (2 * h)
        allowed = float((want[i][1] * direction.abs()).sum()) + 1e-6 * abs(slope) + 1e-6
        assert abs(float((grads[i].double() * direction).sum()) - slope) <= allowed


@pytest.mark.gpu
def test_results_are_the_same_in_every_run():
    torch.manual_seed(14)
    q, k, v = attention_inputs(torch.bfloat16, 1, 1500, 1500, 1, 8, 64)  # block 0 is named by every query: several work items
    blocks = random_blocks(1, 1, 1500, 6, 1500, 64)
    blocks[..., 0] = 0
    dout = torch.randn(q.shape, device="cuda").bfloat16()
    first = check_attention(q, k, v, blocks, 64, dout=dout)
    for _ in range(3):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops.block_attention(*leaves, blocks, 64)
        for a, b in zip(first, [out, *torch.autograd.grad(out, leaves, dout)]):
            assert torch.equal(a, b)


# ---- together, streams, graphs, refusals ---------------------------------------------------------------------------


def layer(tokens, table, wq, wk, wv, heads, kv, block, count):
    """Tokens to attention output, as a model would call the operators."""
    batch, length = tokens.shape
    x = ops.embedding(tokens, table, math.sqrt(table.shape[1]))
    q, k, v = (torch.matmul(x, w).view(batch, length, -1, 64) for w in (wq, wk, wv))
    with torch.no_grad():
        blocks = ops.select_blocks(ops.block_scores(q, ops.block_means(k, block)), count, block, length)
    return ops.block_attention(q, k, v, blocks, block), blocks, (x, q, k, v)


@pytest.mark.gpu
def test_a_training_step_through_all_of_them():
    torch.manual_seed(15)
    vocab, dim, heads, kv, block, count = 300, 96, 8, 2, 16, 4
    tokens = torch.randint(0, vocab, (2, 150), device="cuda")
    table = (torch.randn(vocab, dim, device="cuda") / 10).bfloat16().requires_grad_(True)
    weights = [(torch.randn(dim, h * 64, device="cuda") / 10).bfloat16().requires_grad_(True) for h in (heads, kv, kv)]
    out, blocks, (x, q, k, v) = layer(tokens, table, *weights, heads, kv, block, count)
    assert torch.equal(blocks, ops.select_blocks(ops.block_scores(q, ops.block_means(k, block)), count, block, 150))
    dout = torch.randn(out.shape, device="cuda").bfloat16()
    grads = torch.autograd.grad(out, (table, *weights, q, k, v, x), dout, retain_graph=True)
    pattern = pattern_of(blocks, block, 150, default_visible(2, 150, 150))
    want = attention_reference(q.detach(), k.detach(), v.detach(), pattern, 0.125, dout)
    within(out, *want[0])
    for g, w in zip(grads[4:7], want[1:]):
        within(g, *w)
    size = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, tokens.flatten(), grads[7].reshape(-1, dim).double().abs()) * math.sqrt(dim)
    sums = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, tokens.flatten(), grads[7].reshape(-1, dim).double()) * math.sqrt(dim)
    within(grads[0], sums, size * 400 * U32 + sums.abs() * half_step(torch.bfloat16) + tiny(torch.bfloat16))
    # the last token alone, over a cache of the keys in front of it, is the last row of the prompt
    last = torch.full((2, 1), 150, device="cuda", dtype=torch.int32)
    one = ops.select_blocks(ops.block_scores(q[:, -1:], ops.block_means(k, block)), count, block, 150, last)
    assert torch.equal(one, blocks[:, :, -1:])
    with torch.no_grad():
        got = ops.block_attention(q[:, -1:], k, v, one, block, last)
    within(got, want[0][0][:, -1:], want[0][1][:, -1:])


@pytest.mark.gpu
def test_other_streams_and_two_calls_at_once():
    torch.manual_seed(16)
    q, k, v = attention_inputs(torch.bfloat16, 1, 400, 400, 2, 8, 128)
    blocks = random_blocks(1, 2, 400, 4, 400, 64)
    ids, table = torch.randint(0, 1000, (3000,), device="cuda"), torch.randn(1000, 256, device="cuda")

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        out = ops.block_attention(*leaves[:3], blocks, 64)
        emb = ops.embedding(ids, leaves[3], 2.0)
        return [out, emb, *torch.autograd.grad((out.float() ** 2).sum() + (emb ** 2).sum(), leaves)]

    want = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_and_replayed():
    """Two graphs of a whole step, replayed in turn with new inputs."""
    torch.manual_seed(17)
    state = dict(ids=torch.randint(0, 500, (700,), device="cuda"), table=torch.randn(500, 64, device="cuda"), k=torch.randn(1, 200, 2, 64, device="cuda").bfloat16(),
                 v=torch.randn(1, 200, 2, 64, device="cuda").bfloat16(), q=torch.randn(1, 200, 8, 64, device="cuda").bfloat16())

    def step(ids, table, q, k, v):
        blocks = ops.select_blocks(ops.block_scores(q, ops.block_means(k, 16)), 4, 16, 200)
        out, lse = torch.ops.cutespmm.block_attention(q, k, v, blocks, 16, None, 0.125, None)
        grads = torch.ops.cutespmm.block_attention_grad(out, q, k, v, out, lse, blocks, 16, None, 0.125)
        emb = ops.embedding(ids, table)
        one = ops.block_attention(q[:, -1:], k, v, blocks[:, :, -1:].contiguous(), 16)
        return [blocks, out, *grads, emb, torch.ops.cutespmm.embedding_grad(ids, emb, 500, 1.5), one]

    with torch.no_grad():
        step(**state)
        graphs = []
        for _ in range(2):
            own = {n: t.clone() for n, t in state.items()}
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(**own)
            graphs.append((graph, own, out))
        for i in range(4):
            graph, own, out = graphs[i % 2]
            own["ids"].copy_(torch.randint(-1, 500, (700,), device="cuda"))
            for n in ("q", "k", "v"):
                own[n].copy_(torch.randn(own[n].shape, device="cuda"))
            graph.replay()
            graphs[(i + 1) % 2][0].replay()
            want = step(**{n: t.clone() for n, t in own.items()})
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_operator_registrations():
    torch.manual_seed(18)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    ids, table = torch.randint(0, 50, (30,), device="cuda"), torch.randn(50, 16, device="cuda").requires_grad_(True)
    q, k, v = (t.requires_grad_(True) for t in attention_inputs(torch.bfloat16, 1, 40, 40, 2, 2, 64))
    blocks = random_blocks(1, 2, 40, 3, 40, 16)
    torch.library.opcheck(torch.ops.cutespmm.embedding.default, (ids, table, 2.0), test_utils=tests)
    torch.library.opcheck(torch.ops.cutespmm.embedding_grad.default, (ids, torch.randn(30, 16, device="cuda"), 50, 2.0), test_utils=tests)
    torch.library.opcheck(torch.ops.cutespmm.block_means.default, (k.detach(), 16, None), test_utils=tests)
    torch.library.opcheck(torch.ops.cutespmm.block_scores.default, (q.detach(), k.detach()), test_utils=tests)
    torch.library.opcheck(torch.ops.cutespmm.select_blocks.default, (torch.randn(1, 2, 40, 3, device="cuda"), 2, 16, 40, None, 1, 1), test_utils=tests)
    torch.library.opcheck(torch.ops.cutespmm.block_attention.default, (q, k, v, blocks, 16, None, 0.1, None), test_utils=tests)
    with pytest.raises(RuntimeError):  # a selection has no gradient
        ops.block_scores(q, k).sum().backward()
    out = ops.block_attention(q, k, v, blocks, 16)
    (dq,) = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):  # nor has the gradient
        dq.sum().backward()


def refused(match, fn, *a, **kw):
    with pytest.raises((ValueError, cs.CuteSpmmError), match=match):
        fn(*a, **kw)


def test_refusals():
    """Arguments are checked before anything is asked of a device."""
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    refused("int32 or int64", ops.embedding, torch.zeros(3), torch.zeros(4, 8))
    refused("2-D", ops.embedding, i(3), torch.zeros(8))
    refused("2-D", ops.embedding, i(3), torch.zeros(4, 8, dtype=torch.float64))
    refused("CUDA", ops.embedding, i(3), torch.zeros(4, 8))
    refused("a row for each token", torch.ops.cutespmm.embedding_grad, i(3), torch.zeros(4, 8), 9, 1.0)
    refused("vocab", torch.ops.cutespmm.embedding_grad, i(4), torch.zeros(4, 8), -1, 1.0)
    refused("float16 or bfloat16", ops.block_means, torch.zeros(1, 16, 1, 64), 16)
    refused("multiple of 8", ops.block_means, h(1, 16, 1, 60), 16)
    refused("at most 128", ops.block_means, h(1, 16, 1, 136), 16)
    refused("block must be", ops.block_means, h(1, 16, 1, 64), 48)
    refused("lengths", ops.block_means, h(1, 16, 1, 64), 16, i(2))
    refused("CUDA", ops.block_means, h(1, 16, 1, 64), 16)
    refused("same type", ops.block_scores, h(1, 4, 2, 64), torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16))
    refused("multiple", ops.block_scores, h(1, 4, 3, 64), h(1, 3, 2, 64))
    refused("column per block", ops.select_blocks, torch.zeros(1, 1, 4, 3), 2, 16, 64)
    refused("first \\+ last", ops.select_blocks, torch.zeros(1, 1, 4, 4), 1, 16, 64)
    refused("float32", ops.select_blocks, h(1, 1, 4, 4), 2, 16, 64)
    refused("visible", ops.select_blocks, torch.zeros(1, 1, 4, 4), 2, 16, 64, i(1, 3))
    q, k, b = h(2, 5, 4, 64), h(2, 32, 2, 64), i(2, 2, 5, 3)
    refused("same type", ops.block_attention, q, k.bfloat16(), k, b, 16)
    refused("same shape", ops.block_attention, q, k, h(2, 31, 2, 64), b, 16)
    refused("same batch", ops.block_attention, q, h(1, 32, 2, 64), h(1, 32, 2, 64), b, 16)
    refused("same dim", ops.block_attention, q, h(2, 32, 2, 72), h(2, 32, 2, 72), b, 16)
    refused("multiple", ops.block_attention, q, h(2, 32, 3, 64), h(2, 32, 3, 64), i(2, 3, 5, 3), 16)
    refused("block must be", ops.block_attention, q, k, k, b, 20)
    refused("scale must be", ops.block_attention, q, k, k, b, 16, None, 0.0)
    refused("scale must be", ops.block_attention, q, k, k, b, 16, None, math.nan)
    refused("blocks must be", ops.block_attention, q, k, k, b.long(), 16)
    refused("blocks must be", ops.block_attention, q, k, k, b[:, :1], 16)
    refused("visible", ops.block_attention, q, k, k, b, 16, i(5))
    refused("pages of `block` keys", ops.block_attention, q, k, k, b, 16, i(2, 5), None, i(2, 2))
    refused("needs `visible`", ops.block_attention, q, h(9, 16, 2, 64), h(9, 16, 2, 64), b, 16, None, None, i(2, 2))
    refused("pages must be", ops.block_attention, q, h(9, 16, 2, 64), h(9, 16, 2, 64), b, 16, i(2, 5), None, i(3, 2))
    refused("CUDA", ops.block_attention, q, k, k, b, 16)


def test_refusals_of_the_c_abi():
    import ctypes as C

    lib, EINVAL, EUNSUPPORTED = cs.lib, -1, -4
    s3 = (C.c_int64 * 3)(64, 64, 64)
    p = C.c_void_p(1 << 20)  # never read: every call below is refused
    assert lib.cutespmm_embedding(3, p, 8, 4, 8, p, 4, 2, 1.0, p, 8, None) == EINVAL
    assert lib.cutespmm_embedding(0, p, 8, 4, 8, p, 2, 2, 1.0, p, 8, None) == EINVAL
    assert lib.cutespmm_embedding(0, p, 7, 4, 8, p, 4, 2, 1.0, p, 8, None) == EINVAL
    assert lib.cutespmm_embedding(0, p, 8, 1 << 31, 8, p, 4, 2, 1.0, p, 8, None) == EUNSUPPORTED
    assert lib.cutespmm_embedding(0, p, 8, 4, 8, None, 4, 2, 1.0, p, 8, None) == EINVAL
    need = lib.cutespmm_embedding_grad_workspace(100, 50, 64)
    assert need > 100 * 16
    assert lib.cutespmm_embedding_grad(0, p, 64, p, 4, 100, 50, 64, 1.0, p, 64, p, need - 1, None) == EINVAL
    assert lib.cutespmm_embedding_grad(0, p, 64, p, 4, 100, 50, 64, 1.0, p, 64, C.c_void_p((1 << 20) + 16), need, None) == EINVAL
    assert lib.cutespmm_block_means(0, p, s3, None, 1, 16, 1, 64, 16, p, None) == EINVAL
    assert lib.cutespmm_block_means(1, p, s3, None, 1, 16, 1, 60, 16, p, None) == EUNSUPPORTED
    assert lib.cutespmm_block_means(1, p, s3, None, 1, 16, 1, 64, 24, p, None) == EINVAL
    assert lib.cutespmm_block_means(1, C.c_void_p((1 << 20) + 8), s3, None, 1, 16, 1, 64, 16, p, None) == EINVAL
    assert lib.cutespmm_block_scores(1, p, (C.c_int64 * 3)(4, 8, 8), p, s3, 1, 2, 4, 2, 3, 64, p, None) == EINVAL
    assert lib.cutespmm_block_scores(1, p, s3, p, s3, 1, 2, 3, 2, 3, 64, p, None) == EINVAL
    assert lib.cutespmm_select_blocks(p, s3, None, 1, 1, 1, 3, 64, 16, 2, 1, 1, p, None) == EINVAL
    assert lib.cutespmm_select_blocks(p, s3, None, 1, 1, 1, 16385, 16385 * 16, 16, 2, 1, 1, p, None) == EUNSUPPORTED
    assert lib.cutespmm_select_blocks(None, s3, None, 1, 1, 1, 4, 64, 16, 2, 1, 1, p, None) == EINVAL
    assert lib.cutespmm_block_attention(None, p, p, None) == EINVAL
    assert lib.cutespmm_pattern_status(None) == EINVAL
    buf = (C.c_uint8 * 4096)()  # a description with struct_size 0
    assert lib.cutespmm_block_attention(buf, p, p, None) == EINVAL
    assert lib.cutespmm_block_attention_grad_workspace(buf) == 0


def test_fake_kernels_give_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = torch.empty(2, 5, 4, 64, dtype=torch.float16), torch.empty(2, 40, 2, 64, dtype=torch.float16)
        assert torch.ops.cutespmm.embedding(torch.empty(3, 4, dtype=torch.int64), torch.empty(10, 6), 1.0).shape == (3, 4, 6)
        assert torch.ops.cutespmm.embedding_grad(torch.empty(3, dtype=torch.int64), torch.empty(3, 6), 10, 1.0).shape == (10, 6)
        means = torch.ops.cutespmm.block_means(k, 16, None)
        scores = torch.ops.cutespmm.block_scores(q, means)
        assert means.shape == (2, 3, 2, 64) and scores.shape == (2, 2, 5, 3) and scores.dtype == torch.float32
        blocks = torch.ops.cutespmm.select_blocks(scores, 2, 16, 40, None, 1, 1)
        assert blocks.shape == (2, 2, 5, 2) and blocks.dtype == torch.int32
        out, lse = torch.ops.cutespmm.block_attention(q, k, k, blocks, 16, None, 1.0, None)
        assert out.shape == q.shape and lse.shape == (2, 4, 5)
        assert [g.shape for g in torch.ops.cutespmm.block_attention_grad(out, q, k, k, out, lse, blocks, 16, None, 1.0)] == [q.shape, k.shape, k.shape]


@pytest.mark.gpu
def test_no_forward_mode_derivatives():
    """Refused for all of them, whatever a tangent hangs on: nothing goes on with a tangent of zeros."""
    torch.manual_seed(19)
    q, k, v = attention_inputs(torch.bfloat16, 1, 40, 40, 2, 2, 64)
    blocks = random_blocks(1, 2, 40, 3, 40, 16)
    ids, table = torch.randint(0, 50, (30,), device="cuda"), torch.randn(50, 16, device="cuda")
    calls = [(lambda x: ops.block_attention(x, k, v, blocks, 16), q), (lambda x: ops.block_attention(q, x, v, blocks, 16), k), (lambda x: ops.block_attention(q, k, x, blocks, 16), v),
             (lambda x: ops.embedding(ids, x), table), (lambda x: ops.block_means(x, 16), k), (lambda x: ops.block_scores(x, k), q)]
    for fn, x in calls:
        with pytest.raises(RuntimeError):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
            fn(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    pages = torch.arange(3, device="cuda", dtype=torch.int32)[None]
    cache = torch.randn(3, 16, 2, 64, device="cuda").bfloat16()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        ops.block_attention(torch.autograd.forward_ad.make_dual(q, q), cache, cache, blocks, 16, torch.full((1, 40), 40, device="cuda", dtype=torch.int32), None, pages)
    with torch.autograd.forward_ad.dual_level():  # without a tangent there is nothing to lose
        assert torch.equal(ops.block_attention(q, k, v, blocks, 16), ops.block_attention(q, k, v, blocks, 16))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_dims_of_a_key_that_is_no_number_do_not_touch_the_others(dim):
    """An unseen key that is no number in the upper half of its dims: only those dims of dq are formed again."""
    torch.manual_seed(dim)
    q, k, v = attention_inputs(torch.bfloat16, 1, 64, 64, 2, 8, dim)
    blocks = torch.randint(0, 4, (1, 2, 64, 2), device="cuda", dtype=torch.int32)
    dout = torch.randn(q.shape, device="cuda").bfloat16()
    pattern = pattern_of(blocks, 16, 64, default_visible(1, 64, 64))
    rows = ~pattern[..., 40].any(1)[0]  # queries that do not look at key 40
    want = attention_reference(q, k, v, pattern, 1 / math.sqrt(dim), dout)[1]

    def dq(k):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(ops.block_attention(*leaves, blocks, 16), leaves[0], dout)[0]

    clean = dq(k)
    k[0, 40, :, dim // 2 + 5] = math.nan
    runs = [dq(k) for _ in range(8)]
    for g in runs:
        assert torch.equal(g[:, rows, :, : dim // 2], clean[:, rows, :, : dim // 2])
        assert torch.equal(g[:, rows], runs[0][:, rows])
        within(g[:, rows], want[0][:, rows], want[1][:, rows])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", [(1, 70, 128, 2, 4, 64, 16, 3), (1, 300, 300, 1, 8, 128, 64, 2), (2, 90, 130, 2, 3, 72, 32, 2), (1, 130, 256, 1, 1, 128, 128, 1), (1, 1500, 1500, 1, 8, 64, 64, 4)])
@pytest.mark.parametrize("what", ["q", "dout", "both"])
def test_rows_that_are_no_numbers_reach_no_key_they_do_not_look_at(dtype, form, what):
    """NaN and infinities in q or dout of two queries: dk and dv of the keys they do not look at are those without them, also inside a tile of
    64 keys -- another block of it, or the keys behind the last that they see -- and where a tile's sums come in parts."""
    batch, queries, keys, kv, group, dim, block, count = form
    torch.manual_seed(queries + dim)
    q, k, v = attention_inputs(dtype, batch, queries, keys, kv, group, dim)
    blocks = random_blocks(batch, kv, queries, count, keys, block)
    blocks[..., 0] = 0  # many work items for the first tile of the longest form
    bad = [40, 700] if queries > 1000 else [queries // 2, queries // 2 + 1]
    for t in bad:
        blocks[:, :, t] = -1
        blocks[:, :, t, 0] = (keys - queries + t) // block  # the block that holds the last key it sees
    pattern = pattern_of(blocks, block, keys, default_visible(batch, queries, keys))
    dout = torch.randn(q.shape, device="cuda").to(dtype)
    want = attention_reference(q, k, v, pattern, 1 / math.sqrt(dim), dout)
    if what != "dout":
        q[:, bad[0], :, dim // 3] = math.nan
        q[:, bad[1], 0, 0] = math.inf
    if what != "q":
        dout[:, bad[0], -1] = math.nan
        dout[:, bad[1], :, 1] = -math.inf
    free = ~pattern[:, :, bad].any(2).transpose(1, 2)  # [batch, keys, kv]
    tiles = [(keys - queries + t) // 64 * 64 for t in bad]
    assert any(free[:, i : i + 64].any() and not free[:, i : i + 64].all() for i in tiles)  # a tile of 64 keys of which they see a part
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(ops.block_attention(*leaves, blocks, block), leaves, dout)
    others = torch.ones(queries, device="cuda", dtype=torch.bool)
    others[bad] = False
    within(grads[0][:, others], want[1][0][:, others], want[1][1][:, others])
    for g, (w, bound) in zip(grads[1:], want[2:]):
        within(g[free], w[free], bound[free])
    assert not torch.isfinite(grads[1][~free]).all() and not torch.isfinite(grads[2][~free]).all()  # while what they look at shows it
    again = torch.autograd.grad(ops.block_attention(*leaves, blocks, block), leaves, dout)
    for a, b in zip(grads, again):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.gpu
def test_gradients_whose_inner_products_leave_the_range_of_half():
    """dout v beyond 65504, as a scaled loss makes it: dS has no fp16 form there, but dq, dk and dv do."""
    torch.manual_seed(23)
    q, k, v = attention_inputs(torch.float16, 1, 200, 200, 2, 4, 64)
    blocks = random_blocks(1, 2, 200, 3, 200, 16)
    got = check_attention(q, k, v * 100, blocks, 16, scale=1e-3, dout=(torch.randn(q.shape, device="cuda") * 300).half())
    assert all(torch.isfinite(g).all() for g in got)


@pytest.mark.gpu
def test_the_status_read_waits_for_every_stream():
    side = torch.cuda.Stream()
    done = torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        done.record()
    assert ops.pattern_status() == 0
    assert done.query()


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported_once(tmp_path):
    """The kernels' wait with a limit of a few polls on a barrier that nothing arrives at: it ends, the word is read behind it, and cleared."""
    import subprocess
    from conftest import ROOT

    exe = tmp_path / "status_driver"
    subprocess.run([cs._build.NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{cs._build.CSRC}", str(ROOT / "tests" / "cpp" / "status_driver.cu"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout.strip() == "ran out 1, read again 0, arrived 0", res.stdout + res.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [1, 4, 5])
def test_a_seen_key_that_is_no_number_shows(queries):
    """Few queries and many give the same for a row whose scores are no numbers: out, lse and dq of that row are none either."""
    torch.manual_seed(20)
    q, k, v = attention_inputs(torch.bfloat16, 1, queries, 64, 1, 4, 64)
    blocks = torch.zeros(1, 1, queries, 2, device="cuda", dtype=torch.int32)
    blocks[..., 1] = 2
    visible = torch.full((1, queries), 64, device="cuda", dtype=torch.int32)
    k[0, 3, 0, 7] = math.nan
    out, lse = torch.ops.cutespmm.block_attention(q, k, v, blocks, 16, visible, 0.125, None)
    assert out.isnan().all() and lse.isnan().all()
    dq, dk, dv = torch.ops.cutespmm.block_attention_grad(torch.ones_like(q), q, k, v, out, lse, blocks, 16, visible, 0.125)
    named = torch.zeros(64, device="cuda", dtype=torch.bool)
    named[0:16] = named[32:48] = True
    assert dq.isnan().all() and dk[0, named].isnan().all() and dv[0, named].isnan().all()
    assert not dk[0, ~named].any() and not dv[0, ~named].any()


@pytest.mark.gpu
def test_numbers_beyond_32_bits_are_refused():
    """Not cut down to what is left of them: a result without rows shows it without memory."""
    none = torch.zeros(0, 1, 1, 4, device="cuda")
    refused("beyond 32 bits", ops.select_blocks, none, 2**32 + 5, 16, 64)
    refused("first \\+ last", ops.select_blocks, none, 3, 16, 64, None, 2**62, 2**62)
    refused("beyond 32 bits|2\\^31", torch.ops.cutespmm.embedding_grad, torch.zeros(3, device="cuda", dtype=torch.int32), torch.zeros(3, 0, device="cuda"), 2**40, 1.0)


@pytest.mark.gpu
def test_empty_operands_off_the_grid():
    """Slices without elements, of tensors whose strides are no multiples of 8."""
    q, wide = (torch.randn(2, n, h, 75, device="cuda").half() for n, h in ((9, 2), (33, 1)))
    k = wide[:, :0, :, 3:67]
    blocks = torch.zeros(2, 1, 9, 2, device="cuda", dtype=torch.int32)
    assert k.stride(0) % 8 and not ops.block_attention(q[..., 3:67], k, k, blocks, 16).any()
    leaves = [t.detach().requires_grad_(True) for t in (q[..., 3:67], k, k)]
    grads = torch.autograd.grad(ops.block_attention(*leaves, blocks, 16).sum(), leaves)
    assert not grads[0].any() and grads[1].shape == grads[2].shape == (2, 0, 1, 64)
    assert ops.block_means(k, 16).shape == (2, 0, 1, 64)
    assert ops.block_scores(q[:, :0, :, 3:67], wide[..., 3:67]).shape == (2, 1, 0, 33)
    assert ops.block_scores(q[..., 3:67], k).shape == (2, 1, 9, 0)


def in_a_new_thread(fn):
    import threading

    got = []

    def body():
        try:
            got.append(fn())
        except Exception as e:  # noqa: BLE001 -- shown by the thread that waits
            got.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.gpu
def test_the_first_call_of_a_thread():
    """A thread that has asked nothing of the device before, with memory that torch's allocator holds already."""
    torch.manual_seed(26)
    q, k, v = attention_inputs(torch.bfloat16, 1, 70, 70, 2, 8, 64)
    blocks = random_blocks(1, 2, 70, 3, 70, 16)
    out, lse = torch.ops.cutespmm.block_attention(q, k, v, blocks, 16, None, 0.125, None)
    dout = torch.randn_like(q)
    table, ids = torch.randn(50, 16, device="cuda"), torch.randint(0, 50, (30,), device="cuda")
    calls = [lambda: ops.block_attention(q, k, v, blocks, 16), lambda: ops.block_attention(q[:, :2], k, v, blocks[:, :, :2].contiguous(), 16), lambda: ops.block_scores(q, k),
             lambda: ops.block_means(k, 16), lambda: ops.select_blocks(ops.block_scores(q, ops.block_means(k, 16)), 3, 16, 70), lambda: ops.embedding(ids, table),
             lambda: torch.cat([g.flatten() for g in torch.ops.cutespmm.block_attention_grad(dout, q, k, v, out, lse, blocks, 16, None, 0.125)]),
             lambda: torch.ops.cutespmm.embedding_grad(ids, torch.ones(30, 16, device="cuda"), 50, 1.0)]
    for fn in calls:
        want = fn()
        fn()  # its memory is in torch's cache
        assert torch.equal(in_a_new_thread(fn), want)


@pytest.mark.gpu
def test_compiled():
    """torch.compile through all of them, forward and backward, is the eager call."""
    torch.manual_seed(21)
    tokens = torch.randint(0, 300, (2, 150), device="cuda")
    table = (torch.randn(300, 96, device="cuda") / 10).bfloat16().requires_grad_(True)
    weights = [(torch.randn(96, h * 64, device="cuda") / 10).bfloat16().requires_grad_(True) for h in (8, 2, 2)]

    def step(tokens, table, *weights):
        return layer(tokens, table, *weights, 8, 2, 16, 4)[0]

    want = step(tokens, table, *weights)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(tokens, table, *weights)
    dout = torch.randn(want.shape, device="cuda").bfloat16()
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, (table, *weights), dout), torch.autograd.grad(want, (table, *weights), dout)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_compiled_single_token_over_pages():
    """The branch that a decoding program compiles: kept means, a selection, attention over a paged cache."""
    torch.manual_seed(25)
    cache = [torch.randn(40, 64, 2, 64, device="cuda").bfloat16() for _ in range(2)]
    pages, see = torch.randperm(40, device="cuda").view(2, 20).int(), torch.tensor([[1200], [77]], device="cuda", dtype=torch.int32)
    q = torch.randn(2, 1, 8, 64, device="cuda").bfloat16()
    means = ops.block_means(cache[0][pages.long()].view(2, 1280, 2, 64), 64, see[:, 0].contiguous())

    def step(q, k, v, means, see, pages):
        blocks = ops.select_blocks(ops.block_scores(q, means), 5, 64, 1280, see)
        return blocks, ops.block_attention(q, k, v, blocks, 64, see, None, pages)

    with torch.no_grad():
        want = step(q, *cache, means, see, pages)
        got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, *cache, means, see, pages)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- calls of the C ABI that the torch operators do not make ---------------------------------------------------------


def attention_call(q, k, v, blocks, block, queries, heads, *, batch=1, kv_heads=2, dim=64, keys=64, count=2, visible=None, pages=None, page_cols=0):
    """The C ABI's description of a call (cutespmm_block_attention_t), operands contiguous."""
    import ctypes as C

    class Call(C.Structure):
        _fields_ = [(n, C.c_uint32) for n in "struct_size dtype batch queries heads kv_heads dim keys block count".split()]
        _fields_ += [(n, C.c_void_p) for n in ("q", "k", "v")] + [(n, C.c_int64 * 3) for n in ("q_strides", "k_strides", "v_strides")]
        _fields_ += [(n, C.c_void_p) for n in ("blocks", "visible", "pages")] + [("page_cols", C.c_uint32), ("num_pages", C.c_uint32), ("scale", C.c_float)]

    c = Call(C.sizeof(Call), 1, batch, queries, heads, kv_heads, dim, keys, block, count, q, k, v)
    c.q_strides[:] = queries * heads * dim, heads * dim, dim
    c.k_strides[:] = c.v_strides[:] = keys * kv_heads * dim, kv_heads * dim, dim
    c.blocks, c.visible, c.pages, c.scale = blocks, visible, pages, 0.125
    c.page_cols = c.num_pages = page_cols
    return c


def test_pointers_off_their_grid_are_refused():
    """Kernels store and load 16 bytes at a time in out and the gradients; the rest lies on its elements' grid.  Checked before a device is asked."""
    import ctypes as C

    lib, p, EINVAL = cs.lib, 1 << 20, -1
    s3 = (C.c_int64 * 3)(64, 64, 64)
    call = C.byref(attention_call(p, p, p, p, 16, 4, 4))
    assert lib.cutespmm_block_attention(call, p + 8, p, None) == EINVAL
    assert lib.cutespmm_block_attention(call, p, p + 2, None) == EINVAL
    need = lib.cutespmm_block_attention_grad_workspace(call)
    assert need
    for i in range(5):  # out, lse, dq, dk, dv
        at = [p] * 5
        at[i] += 2 if i == 1 else 8
        assert lib.cutespmm_block_attention_grad(call, p, s3, at[0], at[1], at[2], at[3], at[4], p, need, None) == EINVAL
    for bad in (dict(visible=p + 2), dict(pages=p + 1, page_cols=4), dict(blocks=p + 2)):
        assert lib.cutespmm_block_attention(C.byref(attention_call(p, p, p, bad.pop("blocks", p), 16, 4, 4, **bad)), p, p, None) == EINVAL
    for table, tokens, out in ((p + 1, p, p), (p, p + 2, p), (p, p, p + 1)):
        assert lib.cutespmm_embedding(2, table, 8, 4, 8, tokens, 4, 2, 1.0, out, 8, None) == EINVAL
        assert lib.cutespmm_embedding_grad(2, table, 8, tokens, 4, 2, 4, 8, 1.0, out, 8, p, 1 << 30, None) == EINVAL
    assert lib.cutespmm_embedding(0, p + 2, 8, 4, 8, p, 4, 2, 1.0, p, 8, None) == EINVAL
    assert lib.cutespmm_embedding(0, p, 8, 4, 8, p + 4, 8, 2, 1.0, p, 8, None) == EINVAL
    assert lib.cutespmm_block_means(1, p, s3, p + 2, 1, 16, 1, 64, 16, p, None) == EINVAL
    assert lib.cutespmm_block_means(1, p, s3, None, 1, 16, 1, 64, 16, p + 1, None) == EINVAL
    assert lib.cutespmm_block_scores(1, p, s3, p, s3, 1, 2, 4, 2, 3, 64, p + 2, None) == EINVAL
    for scores, visible, blocks in ((p + 2, p, p), (p, p + 1, p), (p, p, p + 2)):
        assert lib.cutespmm_select_blocks(scores, s3, visible, 1, 1, 1, 4, 64, 16, 2, 1, 1, blocks, None) == EINVAL


@pytest.mark.gpu
def test_gradient_from_an_output_off_the_grid():
    """`out` as a view that begins two bytes behind the 16-byte grid is copied; the gradients are the same."""
    torch.manual_seed(22)
    q, k, v = attention_inputs(torch.bfloat16, 1, 40, 40, 2, 2, 64)
    blocks = random_blocks(1, 2, 40, 3, 40, 16)
    out, lse = torch.ops.cutespmm.block_attention(q, k, v, blocks, 16, None, 0.125, None)
    off = torch.cat([out.new_zeros(1), out.flatten()])[1:].view(out.shape)
    assert off.data_ptr() % 16 == 2 and off.is_contiguous()
    dout = torch.randn(q.shape, device="cuda").bfloat16()
    for a, b in zip(torch.ops.cutespmm.block_attention_grad(dout, q, k, v, off, lse, blocks, 16, None, 0.125), torch.ops.cutespmm.block_attention_grad(dout, q, k, v, out, lse, blocks, 16, None, 0.125)):
        assert torch.equal(a, b)


EMPTY = [dict(queries=0), dict(heads=0), dict(batch=0), dict(count=0), dict(keys=0), dict(queries=0, keys=0)]


def empty_call(empty, q=1 << 20, k=1 << 20, v=1 << 20, blocks=1 << 20):
    sizes = dict(dict(queries=4, heads=4), **empty)
    return attention_call(q, k, v, blocks, 16, sizes.pop("queries"), sizes.pop("heads"), **sizes)


@pytest.mark.parametrize("empty", EMPTY)
def test_workspace_of_an_empty_gradient(empty):
    """In a process of its own: sizes of zero ended it."""
    import subprocess
    import sys
    from conftest import ROOT

    code = ("import ctypes as C, test_pattern_ops as t; n = t.cs.lib.cutespmm_block_attention_grad_workspace(C.byref(t.empty_call(%r))); "
            "print(n); assert (n > 0) == %r") % (empty, set(empty) == {"keys"})  # dq alone takes delta
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**__import__("os").environ, "PYTHONPATH": f"{ROOT}:{ROOT / 'tests'}"}, capture_output=True, text=True)
    assert res.returncode == 0, (res.returncode, res.stdout, res.stderr)


@pytest.mark.gpu
@pytest.mark.parametrize("empty", EMPTY)
def test_empty_gradients_of_the_c_abi(empty):
    """Without queries, heads or blocks nobody looks at any key: the gradients that have elements become zero."""
    import ctypes as C

    q, k, v, out = (torch.randn(4096, device="cuda").half() for _ in range(4))
    blocks, lse = torch.zeros(64, device="cuda", dtype=torch.int32), torch.zeros(64, device="cuda")
    grads = [torch.full((64 * 2 * 64 + 8,), 3.0, device="cuda", dtype=torch.float16) for _ in range(3)]
    work = torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
    c = empty_call(empty, q.data_ptr(), k.data_ptr(), v.data_ptr(), blocks.data_ptr())
    need = cs.lib.cutespmm_block_attention_grad_workspace(C.byref(c))
    assert need <= work.numel()
    st = cs.lib.cutespmm_block_attention_grad(C.byref(c), q.data_ptr(), c.q_strides, out.data_ptr(), lse.data_ptr(), *(g.data_ptr() for g in grads), work.data_ptr() if need else None, need, None)
    assert st == 0
    torch.cuda.synchronize()
    sizes = [c.batch * c.queries * c.heads * c.dim] + [c.batch * c.keys * c.kv_heads * c.dim] * 2
    for g, n in zip(grads, sizes):
        assert not g[:n].any() and (g[n:] == 3.0).all()


@pytest.mark.gpu
def test_scores_of_no_heads_are_zero():
    import ctypes as C

    s3 = (C.c_int64 * 3)(64, 64, 64)
    means, scores = torch.randn(384, device="cuda").half(), torch.full((2 * 5 * 3 + 2,), 7.0, device="cuda")
    assert cs.lib.cutespmm_block_scores(1, None, s3, means.data_ptr(), s3, 2, 5, 0, 1, 3, 64, scores.data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert not scores[:30].any() and (scores[30:] == 7.0).all()
    assert not ops.block_scores(torch.zeros(2, 5, 0, 64, device="cuda").half(), means.view(2, 3, 1, 64)).any()


@pytest.mark.gpu
def test_as_many_blocks_as_scores_and_attention_take():
    """65536 blocks have means, scores and attention; one more is refused by all three."""
    torch.manual_seed(24)
    k = torch.randn(1, 65536 * 16, 1, 8, device="cuda").half()
    means = ops.block_means(k, 16)
    parts = k.double().view(65536, 16, 8)
    within(means[0, :, 0], parts.mean(1), parts.mean(1).abs() * half_step(k.dtype) + parts.abs().mean(1) * 19 * U32 + tiny(k.dtype))
    q = torch.randn(1, 6, 1, 8, device="cuda").half()
    assert ops.block_scores(q, means).shape == (1, 1, 6, 65536)
    blocks = torch.tensor([65535, 0, 40000], device="cuda", dtype=torch.int32).expand(1, 1, 6, 3)
    see = torch.full((1, 6), k.shape[1], device="cuda", dtype=torch.int32)
    keys = torch.cat([k[:, j * 16 : j * 16 + 16] for j in (0, 40000, 65535)], 1)
    few = torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32).expand(1, 1, 6, 3)
    (want,) = attention_reference(q, keys, keys, pattern_of(few, 16, 48, torch.full((1, 6), 48, device="cuda")), 1 / math.sqrt(8))
    within(ops.block_attention(q, k, k, blocks, 16, see), *want)
    more = torch.zeros(1, 65536 * 16 + 1, 1, 8, device="cuda").half()
    refused("65536", ops.block_means, more, 16)
    refused("65536", ops.block_scores, q, torch.zeros(1, 65537, 1, 8, device="cuda").half())
    refused("65536", ops.block_attention, q, more, more, blocks, 16, see)


def test_grids_that_are_too_large_are_refused():
    import ctypes as C

    p = 1 << 20
    many = attention_call(p, p, p, p, 16, 4, 9000 * 64, kv_heads=9000)
    assert cs.lib.cutespmm_block_attention(C.byref(many), p, p, None) == -4
    assert cs.lib.cutespmm_block_attention_grad_workspace(C.byref(many)) == 0
