"""The operators whose sparse pattern the data choose in each step, as they are timed: one case is one call (or one training
step) that a user's program makes through `cutespmm_ae_b200.torch_ops`.

A case is a dict of plain values:

    op      what is called
              embed         out = scale * table[tokens]                                             embedding
              embed_train   the same and the gradient of the table                                  embedding, autograd
              scores        mean key of every block; scores of every query against kept means       block_means, block_scores
              select        the blocks of the highest scores for every query                        select_blocks
              attend        attention of a prompt over the blocks selected for each query           block_attention
              attend_train  the same and the gradients of q, k and v                                block_attention, autograd
              decode        attention of one token per sequence over a cache, contiguous or paged   block_attention
    dtype   float32, float16 or bfloat16
    and the sizes: tokens, vocab, dim; batch, length (queries and keys of a prompt, longest cache of a decode), heads, kv_heads,
    dim, block (keys per block), count (blocks per query)

The attention cases take blocks that a real selection made, from queries and keys with topics: a block of keys has a topic, a
query looks for one for a while, so that neighbouring queries name some of the same blocks and not others.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # the next token of 64 sequences that are served together
        {"name": "embed-64-tokens", "op": "embed", "dtype": "bfloat16", "tokens": 64, "vocab": 128000, "dim": 4096},
        # a training step of a small model: odd numbers of tokens, words and columns
        {"name": "embed-train-odd", "op": "embed_train", "dtype": "float32", "tokens": 8191, "vocab": 50021, "dim": 1000},
        # a training step of a large model with a padded batch: the table's gradient is 1 GB
        {"name": "embed-train-64k", "op": "embed_train", "dtype": "bfloat16", "tokens": 65536, "vocab": 131072, "dim": 4096},
        # a batch of two short prompts, small blocks
        {"name": "scores-3000", "op": "scores", "dtype": "float16", "batch": 2, "length": 3000, "heads": 8, "kv_heads": 2, "dim": 64, "block": 32},
        # a long prompt
        {"name": "scores-32k", "op": "scores", "dtype": "bfloat16", "batch": 1, "length": 32768, "heads": 32, "kv_heads": 4, "dim": 128, "block": 64},
        # one token each of 32 sequences, caches of up to 65536 keys
        {"name": "select-32-tokens", "op": "select", "batch": 32, "length": 1, "keys": 65536, "kv_heads": 8, "block": 64, "count": 32},
        # every query of a long prompt
        {"name": "select-16k", "op": "select", "batch": 1, "length": 16384, "keys": 16384, "kv_heads": 4, "block": 64, "count": 16},
        # a training step of a small model: odd length, one query head for each head of keys, small blocks
        {"name": "attend-train-517", "op": "attend_train", "dtype": "float16", "batch": 3, "length": 517, "heads": 6, "kv_heads": 6, "dim": 64, "block": 16, "count": 8},
        # a training step on a long text, eight query heads for each head of keys
        {"name": "attend-train-8k", "op": "attend_train", "dtype": "bfloat16", "batch": 1, "length": 8192, "heads": 32, "kv_heads": 4, "dim": 128, "block": 64, "count": 16},
        # a long prompt
        {"name": "attend-16k", "op": "attend", "dtype": "bfloat16", "batch": 1, "length": 16384, "heads": 16, "kv_heads": 2, "dim": 128, "block": 64, "count": 32},
        # one token of one sequence: latency counts
        {"name": "decode-one", "op": "decode", "dtype": "bfloat16", "batch": 1, "length": 9001, "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "count": 16, "paged": False},
        # one token each of 64 sequences of different lengths over a paged cache
        {"name": "decode-64-paged", "op": "decode", "dtype": "bfloat16", "batch": 64, "length": 32768, "heads": 64, "kv_heads": 8, "dim": 128, "block": 64, "count": 48, "paged": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embed", "embed_train", "scores", "select", "attend", "attend_train", "attend_train", "decode", "decode"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "embed":
        return {"op": op, "dtype": rng.choice(list(_DTYPES)), "tokens": _log_int(rng, 1, 60000), "vocab": _log_int(rng, 1000, 130000), "dim": _log_int(rng, 64, 4096)}
    if op == "embed_train":
        return {"op": op, "dtype": rng.choice(list(_DTYPES)), "tokens": _log_int(rng, 16, 60000), "vocab": _log_int(rng, 1000, 130000), "dim": _log_int(rng, 64, 2048)}
    dim, block = rng.choice([64, 80, 96, 128]), rng.choice([16, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 3, 4, 6, 8])
    if op == "scores":
        length = _log_int(rng, 64, 16000)
        return {"op": op, "dtype": dtype, "batch": 1 if length > 4000 else rng.choice([1, 2, 5]), "length": length, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "block": max(block, 64) if length > 4000 else block}
    if op == "select":
        keys, count = _log_int(rng, 200, 60000), rng.choice([4, 13, 16, 32, 64])
        length = 1 if rng.random() < 0.3 else min(keys, _log_int(rng, 1, 4000))
        return {"op": op, "batch": rng.choice([1, 2, 7]), "length": length, "keys": keys, "kv_heads": kv_heads, "block": 64 if keys > 8000 else block, "count": count}
    if op == "decode":
        return {"op": op, "dtype": dtype, "batch": rng.choice([1, 2, 5, 16, 33]), "length": _log_int(rng, 2, 20000), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "block": block,
                "count": rng.choice([2, 5, 16, 31, 48]), "paged": rng.random() < 0.5}
    length = _log_int(rng, 40, 5000)
    return {"op": op, "dtype": dtype, "batch": 1 if length > 1500 else rng.choice([1, 2, 3]), "length": length, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "block": block,
            "count": rng.choice([3, 4, 8, 16, 20])}


# ---- inputs -------------------------------------------------------------------------------------------------------


def _word_share(vocab):
    """Probability of the i-th most frequent word: a few words make up much of a text, most are rare."""
    edges = (torch.arange(vocab + 1, dtype=torch.float64) / vocab) ** (1 / 3)
    return edges[1:] - edges[:-1]


def _padding(case):
    return case["tokens"] // 50 if case["op"] == "embed_train" else 0


def _tokens(case, g):
    vocab = case["vocab"]
    u = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
    word = (u ** 3 * vocab).long().clamp_(max=vocab - 1)
    word = torch.randperm(vocab, generator=g, device="cuda")[word]
    pad = _padding(case)
    if pad:
        word[-pad:] = -1
    return word


def _topics(case, g, blocks):
    """Queries and keys [batch, length, heads, dim] with topics."""
    batch, length, heads, kv, dim = (case[n] for n in ("batch", "length", "heads", "kv_heads", "dim"))
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    topic = rand(batch, blocks, kv, dim)
    k = rand(batch, length, kv, dim) + 0.7 * topic.repeat_interleave(case["block"], 1)[:, :length]
    stretch = 24  # queries that look for the same thing
    spans = (length + stretch - 1) // stretch
    wanted = rand(batch, spans, kv, 1, dim).repeat_interleave(stretch, 1)[:, :length]
    q = (0.5 * wanted + rand(batch, length, kv, heads // kv, dim)).reshape(batch, length, heads, dim)
    return q, k


def _selection(scores, count, block, visible):
    """First and last visible block and the visible ones of the highest scores, ascending, -1 behind the last.  scores
    [batch, kv_heads, queries, blocks], visible [batch, queries] keys."""
    blocks = scores.shape[-1]
    n = ((visible + block - 1) // block)[:, None, :, None]
    at = torch.arange(blocks, device=scores.device)
    s = torch.where(at < n, scores.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf), -math.inf)
    s = torch.where((at < n) & ((at < 1) | (at >= n - 1)), math.inf, s)
    order = torch.argsort(s, dim=-1, descending=True, stable=True)[..., : min(count, blocks)]
    kept = torch.gather(s, -1, order) > -math.inf
    got = torch.where(kept, order, blocks).sort(-1).values
    got = torch.where(got < blocks, got, -1).int()
    return torch.nn.functional.pad(got, (0, count - got.shape[-1]), value=-1)


def _mean_of_blocks(k, block):
    batch, length, kv, dim = k.shape
    blocks = (length + block - 1) // block
    padded = torch.nn.functional.pad(k.float(), (0, 0, 0, 0, 0, blocks * block - length)).view(batch, blocks, block, kv, dim).sum(2)
    keys = (length - block * torch.arange(blocks, device=k.device)).clamp(max=block)
    return padded / keys[None, :, None, None]


def _scores_of(q, means):
    """[batch, kv_heads, queries, blocks]: q summed over the heads of a group, times the mean keys."""
    batch, length, heads, dim = q.shape
    kv = means.shape[2]
    s = q.float().view(batch, length, kv, heads // kv, dim).sum(3)
    return torch.matmul(s.transpose(1, 2), means.float().permute(0, 2, 3, 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if op in ("embed", "embed_train"):
        dtype = _DTYPES[case["dtype"]]
        table = torch.empty(case["vocab"], case["dim"], device="cuda", dtype=dtype).normal_(0, 0.02, generator=g)
        s = {"op": op, "tokens": _tokens(case, g), "table": table, "scale": math.sqrt(case["dim"])}
        if op == "embed_train":
            s["dout"] = (rand(case["tokens"], case["dim"]) * 1e-2).to(dtype)
            s["table"].requires_grad_(True)
        return s
    if op == "select":
        batch, length, keys, kv, block = (case[n] for n in ("batch", "length", "keys", "kv_heads", "block"))
        blocks = (keys + block - 1) // block
        scores = rand(batch, kv, length, blocks) * 8 + 4 * rand(batch, kv, 1, blocks)
        visible = None if length > 1 else torch.randint(keys // 2 + 1, keys + 1, (batch, 1), generator=g, device="cuda", dtype=torch.int32)
        return {"op": op, "scores": scores, "keys": keys, "block": block, "count": case["count"], "visible": visible}
    dtype, block = _DTYPES[case["dtype"]], case["block"]
    blocks = (case["length"] + block - 1) // block
    if op == "scores":
        q, k = _topics(case, g, blocks)
        q, k = q.to(dtype), k.to(dtype)
        return {"op": op, "q": q, "k": k, "block": block, "means": _mean_of_blocks(k, block).to(dtype)}
    batch, length, heads, kv, dim = (case[n] for n in ("batch", "length", "heads", "kv_heads", "dim"))
    if op == "decode":
        pages = batch * blocks
        shape = (pages, block, kv, dim) if case["paged"] else (batch, length, kv, dim)
        k, v = (torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g) for _ in range(2))
        q = rand(batch, 1, heads, dim).to(dtype)
        lengths = torch.randint(length // 2 + 1, length + 1, (batch, 1), generator=g, device="cuda", dtype=torch.int32)
        table = torch.randperm(pages, generator=g, device="cuda").view(batch, blocks).int() if case["paged"] else None
        picked = _selection(rand(batch, kv, 1, blocks), case["count"], block, lengths)
        return {"op": op, "q": q, "k": k, "v": v, "blocks": picked, "block": block, "visible": lengths, "pages": table}
    q, k = _topics(case, g, blocks)
    q, k, v = q.to(dtype), k.to(dtype), rand(batch, length, kv, dim).to(dtype)
    visible = torch.arange(1, length + 1, device="cuda", dtype=torch.int32).expand(batch, length)
    picked = _selection(_scores_of(q, _mean_of_blocks(k, block).to(dtype)), case["count"], block, visible)
    s = {"op": op, "q": q, "k": k, "v": v, "blocks": picked, "block": block}
    if op == "attend_train":
        s["dout"] = rand(batch, length, heads, dim).to(dtype)
        s["q"], s["k"], s["v"] = (t.requires_grad_(True) for t in (q, k, v))
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from cutespmm_ae_b200 import torch_ops as ops

    op = s["op"]
    if op == "embed":
        return {"out": ops.embedding(s["tokens"], s["table"], s["scale"])}
    if op == "embed_train":
        out = ops.embedding(s["tokens"], s["table"], s["scale"])
        (dtable,) = torch.autograd.grad(out, s["table"], s["dout"])
        return {"out": out.detach(), "dtable": dtable}
    if op == "scores":
        return {"means": ops.block_means(s["k"], s["block"]), "scores": ops.block_scores(s["q"], s["means"])}
    if op == "select":
        return {"blocks": ops.select_blocks(s["scores"], s["count"], s["block"], s["keys"], s["visible"])}
    if op == "decode":
        return {"out": ops.block_attention(s["q"], s["k"], s["v"], s["blocks"], s["block"], visible=s["visible"], pages=s["pages"])}
    out = ops.block_attention(s["q"], s["k"], s["v"], s["blocks"], s["block"])
    if op == "attend":
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


@torch.no_grad()
def _run_plain(s):
    op = s["op"]
    if op in ("embed", "embed_train"):
        tokens, table, scale = s["tokens"], s["table"], s["scale"]
        named = (tokens >= 0) & (tokens < table.shape[0])
        row = torch.where(named, tokens, 0)
        out = {"out": (table[row].float() * (named[:, None] * scale)).to(table.dtype)}
        if op == "embed_train":
            # 64 bits: the most frequent word's gradient is a long sum
            total = torch.zeros(table.shape, device="cuda", dtype=torch.float64 if table.dtype == torch.float32 else torch.float32)
            total.index_add_(0, row, s["dout"].to(total.dtype) * named[:, None])
            out["dtable"] = (total * scale).to(table.dtype)
        return out
    if op == "scores":
        return {"means": _mean_of_blocks(s["k"], s["block"]).to(s["k"].dtype), "scores": _scores_of(s["q"], s["means"])}
    if op == "select":
        return {"blocks": _plain_select(s)}
    return _plain_decode(s) if op == "decode" else _plain_attend(s)


def _plain_select(s):
    scores, visible = s["scores"], s["visible"]
    if visible is None:
        queries = scores.shape[2]
        visible = (torch.arange(queries, device="cuda", dtype=torch.int32) + (s["keys"] - queries + 1)).expand(scores.shape[0], queries)
    return _selection(scores, s["count"], s["block"], visible)


def _plain_decode(s):
    q, k, v, blocks, block = s["q"], s["k"], s["v"], s["blocks"], s["block"]
    batch, _, heads, dim = q.shape
    kv, count = k.shape[2], blocks.shape[3]
    b = blocks[:, :, 0, :].long()  # batch, kv, count
    key = (b.clamp(min=0)[..., None] * block + torch.arange(block, device="cuda")).reshape(batch, kv, count * block)
    seen = (b >= 0).repeat_interleave(block, -1) & (key < s["visible"][:, :, None])
    key = torch.where(seen, key, 0)
    head = torch.arange(kv, device="cuda")[None, :, None]
    if s["pages"] is None:
        row = torch.arange(batch, device="cuda")[:, None, None]
        keys, values = k[row, key, head], v[row, key, head]
    else:
        page = torch.gather(s["pages"].long()[:, None].expand(-1, kv, -1), 2, key // block)
        keys, values = k[page, key % block, head], v[page, key % block, head]
    score = torch.matmul(q.float().view(batch, kv, heads // kv, dim), keys.float().transpose(2, 3)) / math.sqrt(dim)
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, values.float()) / p.sum(-1, keepdim=True)
    return {"out": out.view(batch, 1, heads, dim).to(q.dtype)}


def _plain_attend(s):
    q, k, v, blocks, block = s["q"], s["k"], s["v"], s["blocks"], s["block"]
    batch, length, heads, dim = q.shape
    kv = k.shape[2]
    group, dtype, scale = heads // kv, q.dtype, 1 / math.sqrt(dim)
    names = torch.zeros(batch, kv, length, (length + block - 1) // block + 1, device="cuda", dtype=torch.bool)
    names.scatter_(3, torch.where(blocks >= 0, blocks, names.shape[3] - 1).long(), True)
    at = torch.arange(length, device="cuda")
    hidden = ~names[..., :-1].repeat_interleave(block, -1)[..., :length] | (at > at[:, None])
    q5 = q.float().view(batch, length, kv, group, dim).permute(0, 2, 3, 1, 4)
    k5, v5 = (t.float().permute(0, 2, 1, 3)[:, :, None] for t in (k, v))
    p = torch.matmul(q5, k5.transpose(3, 4)).mul_(scale).masked_fill_(hidden[:, :, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    out5 = torch.matmul(p, v5)
    back = lambda t: t.permute(0, 3, 1, 2, 4).reshape(batch, length, heads, dim).to(dtype)  # noqa: E731
    out = {"out": back(out5)}
    if s["op"] == "attend_train":
        d5 = s["dout"].float().view(batch, length, kv, group, dim).permute(0, 2, 3, 1, 4)
        shared = lambda t: t.sum(2).permute(0, 2, 1, 3).to(dtype)  # noqa: E731
        out["dv"] = shared(torch.matmul(p.transpose(3, 4), d5))
        ds = torch.matmul(d5, v5.transpose(3, 4)).sub_((d5 * out5).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"], out["dk"] = back(torch.matmul(ds, k5)), shared(torch.matmul(ds.transpose(3, 4), q5))
        out = {n: out[n] for n in ("out", "dq", "dk", "dv")}
    return out


# ---- in 64 bits ---------------------------------------------------------------------------------------------------


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("embed", "embed_train"):
        got = torch.zeros(case["tokens"], case["dim"], device="cuda", dtype=torch.float64)
        real = (s["tokens"] >= 0).nonzero()[:, 0]
        got[real] = s["table"].double().index_select(0, s["tokens"][real]) * s["scale"]
        if op == "embed":
            return {"out": got}
        grad = torch.zeros(case["vocab"], case["dim"], device="cuda", dtype=torch.float64)
        for i in range(0, len(real), 8192):
            at = real[i : i + 8192]
            grad.index_put_((s["tokens"][at],), s["dout"][at].double() * s["scale"], accumulate=True)
        return {"out": got, "dtable": grad}
    if op == "select":
        return None
    if op == "scores":
        q, means, k, block = s["q"].double(), s["means"].double(), s["k"].double(), case["block"]
        group = case["heads"] // case["kv_heads"]
        total = sum(torch.einsum("bthd,bnhd->bhtn", q[:, :, i::group], means) for i in range(group))
        pooled = torch.stack([k[:, i : i + block].mean(1) for i in range(0, case["length"], block)], 1)
        return {"means": pooled, "scores": total}
    heads, kv, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    group, out, grads = heads // kv, torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64), {}
    if op == "attend_train":
        grads = {n: torch.zeros(s[n[1:]].shape, device="cuda", dtype=torch.float64) for n in ("dq", "dk", "dv")}
    queries = s["q"].shape[1]
    for b in range(case["batch"]):
        for h in range(kv):
            heads_of = slice(h * group, (h + 1) * group)
            if s.get("pages") is not None:
                rows = s["pages"][b].long()
                k, v = (t[rows, :, h].reshape(-1, dim) for t in (s["k"], s["v"]))
            else:
                k, v = s["k"][b, :, h], s["v"][b, :, h]
            step = max(1, 2 ** 26 // (case["count"] * block * dim))
            for i in range(0, queries, step):
                at = torch.arange(i, min(i + step, queries), device="cuda")
                last = at if op != "decode" else s["visible"][b].long() - 1
                chosen = s["blocks"][b, h, at].long()
                key = (chosen[:, :, None] * block + torch.arange(block, device="cuda")).flatten(1)
                key = torch.where((chosen < 0).repeat_interleave(block, 1) | (key > last[:, None]), -1, key)
                near, values, q = k[key.clamp(min=0)].double(), v[key.clamp(min=0)].double(), s["q"][b, at, heads_of].double()
                logits = torch.einsum("tgd,tkd->tgk", q, near) / math.sqrt(dim)
                weight = torch.softmax(logits.masked_fill((key < 0)[:, None], -math.inf), -1)
                o = torch.einsum("tgk,tkd->tgd", weight, values)
                out[b, at, heads_of] = o
                if grads:
                    d = s["dout"][b, at, heads_of].double()
                    slope = weight * (torch.einsum("tgd,tkd->tgk", d, values) - (d * o).sum(-1, keepdim=True)) / math.sqrt(dim)
                    grads["dq"][b, at, heads_of] = torch.einsum("tgk,tkd->tgd", slope, near)
                    spread = key.clamp(min=0).flatten()
                    grads["dk"][b, :, h].index_add_(0, spread, torch.einsum("tgk,tgd->tkd", slope, q).flatten(0, 1))
                    grads["dv"][b, :, h].index_add_(0, spread, torch.einsum("tgk,tgd->tkd", weight, d).flatten(0, 1))
    return {"out": out, **grads}


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op in ("embed", "embed_train"):
        size, tokens, dim = _DTYPES[case["dtype"]].itemsize, case["tokens"], case["dim"]
        real = tokens - _padding(case)
        named = float((1 - (1 - _word_share(case["vocab"])) ** real).sum())
        moved = 8 * tokens + named * dim * size + tokens * dim * size
        if op == "embed":
            return {"bytes": moved, "flops": tokens * dim}
        return {"bytes": moved + real * dim * size + case["vocab"] * dim * size, "flops": 2 * tokens * dim}
    if op == "select":
        rows, blocks = case["batch"] * case["kv_heads"], (case["keys"] + case["block"] - 1) // case["block"]
        if case["length"] == 1:
            seen = 0.75 * blocks  # caches are half full to full
        else:
            seen = sum((case["keys"] - case["length"] + t) // case["block"] + 1 for t in range(case["length"]))
        return {"bytes": rows * (4 * seen + 4 * case["count"] * case["length"]), "flops": rows * seen}
    size = 2
    batch, length, heads, kv, dim, block = (case[n] for n in ("batch", "length", "heads", "kv_heads", "dim", "block"))
    blocks = (length + block - 1) // block
    if op == "scores":
        moved = size * batch * dim * (length * (heads + kv) + 2 * blocks * kv) + 4 * batch * kv * length * blocks
        return {"bytes": moved, "flops": batch * dim * (length * (heads + kv) + 2 * kv * length * blocks)}
    per = case["count"] * block
    if op == "decode":
        pairs = batch * min(per, 0.75 * length)
        moved = size * dim * (2 * kv * pairs + 2 * batch * heads) + 4 * batch * kv * case["count"]
        return {"bytes": moved, "flops": 4 * dim * heads * pairs}
    pairs = batch * sum(min(t + 1, per) for t in range(length))
    moved = size * dim * batch * length * (2 * heads + 2 * kv) + 4 * batch * kv * length * case["count"]
    if op == "attend":
        return {"bytes": moved, "flops": 4 * dim * heads * pairs}
    return {"bytes": moved + size * dim * batch * length * (2 * heads + 2 * kv), "flops": 14 * dim * heads * pairs}
