"""The operators of a decoding step that verifies drafted tokens over a paged key/value cache, as
cases that can be measured: their inputs, their plain form in elementary torch operations, the calls
of this package that replace it, and their definition in 64 bits.

One step of such a program takes the rows of the q|k|v projection, normalises and rotates the heads
and puts keys and values into the cache (``rope``), attends over the cache with a tree of drafted
tokens per sequence (``tree``), draws a token for each node from the logits (``sample``), keeps the
accepted branch's entries (``compact``), and forks sequences by copying pages (``copy``).

The head layout (16 query heads, 8 key/value heads of 128), the vocabulary of 151936 rows and the
context of 2304 positions are those of the decode benchmark; the other sizes are generic.
"""
import math

import numpy as np
import torch

own = False

VOCAB = 151936
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the single-sequence decode step: one token, its heads rotated into an f32 cache
        dict(name="rope one token f32", op="rope", tokens=1, hq=16, hkv=8, hd=128, rot=128, inter=False, norm=True,
             dtype="f32", page=16, factor=1.0),
        # a prefill chunk of 16384 positions, half of each head rotated in pairs, context scaled by 4
        dict(name="rope prefill bf16", op="rope", tokens=16384, hq=16, hkv=8, hd=128, rot=64, inter=True, norm=True,
             dtype="bf16", page=64, factor=4.0),
        # one sequence, one token, a short f32 cache: the latency of a plain decode step
        dict(name="tree 1x1 ctx 152 f32", op="tree", seqs=1, tree=1, ctx=152, hq=16, hkv=8, hd=128, dtype="f32", page=16),
        # 64 sequences, single tokens, the benchmark's contexts in f32
        dict(name="tree 64x1 ctx 2303 f32", op="tree", seqs=64, tree=1, ctx=2303, hq=16, hkv=8, hd=128, dtype="f32", page=16),
        # 16 sequences with drafts of up to 16 nodes in bf16
        dict(name="tree 16x16 ctx 2303 bf16", op="tree", seqs=16, tree=16, ctx=2303, hq=16, hkv=8, hd=128, dtype="bf16", page=16),
        # one long document with the widest tree
        dict(name="tree 1x64 ctx 131000 bf16", op="tree", seqs=1, tree=64, ctx=131000, hq=16, hkv=8, hd=128, dtype="bf16", page=64),
        # forks of 2 and of 96 sequences: the last, partly filled page of each is copied in all layers
        dict(name="copy 2 pages f32", op="copy", pairs=2, layers=28, hkv=8, hd=128, page=16, dtype="f32"),
        dict(name="copy 96 pages bf16", op="copy", pairs=96, layers=28, hkv=8, hd=128, page=16, dtype="bf16"),
        # the accepted branches of one wide tree, and of 64 trees, move to the front of their drafts in all layers
        dict(name="compact 1x64 f32", op="compact", seqs=1, tree=64, layers=28, hkv=8, hd=128, page=16, dtype="f32"),
        dict(name="compact 64x16 bf16", op="compact", seqs=64, tree=16, layers=28, hkv=8, hd=128, page=16, dtype="bf16"),
        # one sequence's next token; 64 nodes of drafted trees at once
        dict(name="sample 1 row f32", op="sample", rows=1, n=VOCAB, top_k=0, top_p=0.9, min_p=0.0, dtype="f32"),
        dict(name="sample 64 rows bf16", op="sample", rows=64, n=VOCAB, top_k=50, top_p=0.9, min_p=0.05, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "tree", "tree", "copy", "compact", "sample", "sample"])
    hkv = rng.choice([1, 2, 4, 8])
    heads = dict(hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv, hd=rng.choice([64, 128]))
    dtype, page = rng.choice(["f32", "bf16"]), rng.choice([16, 32, 64])
    if op == "rope":
        per = (heads["hq"] + 2 * hkv) * heads["hd"] * 2
        tokens = min(_log(rng, 1, 16384), 16384 * 8192 // per)
        return dict(op=op, tokens=tokens, **heads, rot=rng.choice([heads["hd"], heads["hd"] // 2, 32]),
                    inter=rng.random() < 0.5, norm=rng.random() < 0.7, dtype=dtype, page=page,
                    factor=rng.choice([1.0, 2.0, 8.0]))
    if op == "tree":
        tree, seqs = rng.choice([1, 2, 5, 8, 13, 24, 32, 47, 64]), _log(rng, 1, 64)
        most = min(131000, 131000 * 8 // (seqs * hkv), 131000 * 64 * 16 // (seqs * tree * heads["hq"]))
        return dict(op=op, seqs=seqs, tree=tree, ctx=_log(rng, 1, max(2, most)), **heads, dtype=dtype, page=page)
    if op == "copy":
        return dict(op=op, pairs=_log(rng, 1, 48), layers=rng.randint(1, 28), hkv=hkv, hd=heads["hd"], page=page if page < 64 else 16,
                    dtype=dtype)
    if op == "compact":
        return dict(op=op, seqs=_log(rng, 1, 48), tree=rng.choice([4, 7, 16, 33, 64]), layers=rng.randint(1, 28), hkv=hkv,
                    hd=heads["hd"], page=16, dtype=dtype)
    return dict(op=op, rows=_log(rng, 1, 64), n=rng.choice([VOCAB, _log(rng, 100, VOCAB)]), top_k=rng.choice([0, 1, 20, 50, 1000]),
                top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.05, 0.2]), dtype=dtype)


# ----------------------------------------------------------------------------------------- inputs
def _spread(case, most, least):
    """Whole numbers in [least, most], one per sequence, the first the largest: the same for every seed."""
    r = np.random.RandomState(case["seqs"] * 7919 + case["tree"] * 31 + most)
    v = r.randint(least, most + 1, case["seqs"])
    v[0] = most
    return v


def _lengths(case):
    """Contexts in [3/4 ctx, ctx] and tree sizes in [1/2 tree, tree] of a case's sequences."""
    ctx = case.get("ctx", 100)
    return _spread(case, ctx, max(1, 3 * ctx // 4)), _spread(case, case["tree"], max(1, case["tree"] // 2))


def _trees(rng, trees):
    """Random trees: every node's ancestors and itself as bits, node j's parent among the nodes before it
    (the newest more often).  Returns int64 [sequences, most nodes]."""
    most = int(trees.max())
    mask = np.zeros((len(trees), most), np.uint64)
    rows = np.arange(len(trees))
    for j in range(most):
        if j == 0:
            mask[:, 0] = 1
            continue
        back = np.minimum(rng.geometric(0.5, len(trees)), j)
        mask[:, j] = mask[rows, j - back] | np.uint64(1 << j)
    return mask.view(np.int64)


def _accepted(case):
    """The accepted branch of each tree of a case, as node bits: the same for every seed."""
    _, trees = _lengths(case)
    rng = np.random.RandomState(case["seqs"] + 97 * case["tree"])
    mask = _trees(rng, trees)
    return mask[np.arange(len(trees)), trees - 1 - rng.randint(0, (trees + 1) // 2)]


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    dt = DTYPES[case["dtype"]]
    s = dict(case=dict(case))
    op = case["op"]
    if op == "rope":
        n, hq, hkv, hd, page = case["tokens"], case["hq"], case["hkv"], case["hd"], case["page"]
        pages = -(-n // page) + 2
        s["qkv"] = _randn(g, (n, (hq + 2 * hkv) * hd), dt)
        # a few long documents: positions run on from somewhere below a million
        s["positions"] = _dev((rng.randint(0, 1000000) + np.arange(n)).astype(np.int32))
        slots = rng.permutation(pages)[: -(-n // page)][np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
        if n > 8:
            slots[rng.randint(0, n, n // 64 + 1)] = -1  # padded rows have no place in the cache
        s["slots"] = _dev(slots.astype(np.int32))
        s["inv_freq"] = _dev(1e6 ** (-np.arange(0, case["rot"], 2, dtype=np.float64) / case["rot"]) / case["factor"])
        s["scale"] = 0.1 * math.log(case["factor"]) + 1.0
        if case["norm"]:
            s["q_norm"] = 1 + 0.1 * _randn(g, (hd,), torch.float32)
            s["k_norm"] = 1 + 0.1 * _randn(g, (hd,), torch.float32)
        s["k"] = _randn(g, (pages, page, hkv, hd), dt)
        s["v"] = _randn(g, (pages, page, hkv, hd), dt)
    elif op == "tree":
        ctx, trees = _lengths(case)
        hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
        need = -(-(ctx + trees) // page)
        pages = int(need.sum())
        table = np.zeros((len(ctx), int(need.max())), np.int32)
        order, at = rng.permutation(pages).astype(np.int32), 0
        for i, c in enumerate(need):
            table[i, :c] = order[at : at + c]
            at += c
        mask = _trees(rng, trees)
        s["mask"] = _dev(np.concatenate([mask[i, :t] for i, t in enumerate(trees)]))
        s["table"], s["ctx"] = _dev(table), _dev(ctx.astype(np.int32))
        s["start"] = _dev(np.concatenate([[0], np.cumsum(trees)]).astype(np.int32))
        s["q"] = 1.5 * _randn(g, (int(trees.sum()), hq, hd), dt)
        s["k"] = _randn(g, (pages, page, hkv, hd), dt)
        s["v"] = _randn(g, (pages, page, hkv, hd), dt)
        s["max_tree"], s["max_ctx"] = int(trees.max()), int(ctx.max())
    elif op == "copy":
        pages = 2 * case["pairs"] + 8
        order = rng.permutation(pages).astype(np.int32)
        s["src"], s["dst"] = _dev(order[: case["pairs"]]), _dev(order[case["pairs"] : 2 * case["pairs"]])
        shape = (case["layers"], pages, case["page"], case["hkv"], case["hd"])
        s["k"], s["v"] = _randn(g, shape, dt), _randn(g, shape, dt)
    elif op == "compact":
        ctx, trees = _lengths(case)
        page = case["page"]
        per = -(-int((ctx + trees).max()) // page)
        pages = per * len(ctx)
        s["table"], s["ctx"] = _dev(rng.permutation(pages).astype(np.int32).reshape(len(ctx), per)), _dev(ctx.astype(np.int32))
        s["accepted"] = _dev(_accepted(case))
        s["new_len"] = torch.zeros(len(ctx), dtype=torch.int32, device="cuda")
        shape = (case["layers"], pages, page, case["hkv"], case["hd"])
        s["k"], s["v"] = _randn(g, shape, dt), _randn(g, shape, dt)
    else:
        m, n = case["rows"], case["n"]
        # logits of a language model: most of them low, a few far above the rest
        x = 2.0 * _randn(g, (m, n), torch.float32)
        x += 6.0 * (torch.rand((m, n), generator=g, device="cuda") < 20.0 / n) * torch.rand((m, n), generator=g, device="cuda")
        s["logits"] = x.to(dt)
        s["u"] = torch.rand((m,), generator=g, device="cuda")
        s["temperature"] = _dev(rng.choice([0.7, 1.0, 1.3], m).astype(np.float32))
    return s


# ----------------------------------------------------------------------------------- plain forms
def _plain_rope(s):
    c = s["case"]
    n, hq, hkv, hd, rot = c["tokens"], c["hq"], c["hkv"], c["hd"], c["rot"]
    x = s["qkv"].float().view(n, hq + 2 * hkv, hd)
    q, k, v = x[:, :hq], x[:, hq : hq + hkv], x[:, hq + hkv :]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["scale"]).float()[:, None], (angle.sin() * s["scale"]).float()[:, None]

    def norm_rotate(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r, rest = x[..., :rot], x[..., rot:]
        if c["inter"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = r[..., : rot // 2], r[..., rot // 2 :]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((r, rest), -1)

    q, k = norm_rotate(q, s.get("q_norm")), norm_rotate(k, s.get("k_norm"))
    kc, vc = s["k"].view(-1, hkv, hd), s["v"].view(-1, hkv, hd)
    kept = (s["slots"] >= 0).nonzero()[:, 0]
    at = s["slots"].long()[kept]
    kc[at], vc[at] = k[kept].to(kc.dtype), v[kept].to(vc.dtype)
    return dict(q=q.to(s["qkv"].dtype), k=s["k"], v=s["v"])


def _plain_tree(s):
    c = s["case"]
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    seqs, most, dev = len(s["ctx"]), s["max_tree"], s["q"].device
    start, ctx = s["start"].long(), s["ctx"].long()
    counts = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(seqs, device=dev), counts, output_size=len(s["q"]))
    node = torch.arange(len(s["q"]), device=dev) - start[seq]
    q = torch.zeros((seqs, most, hq, hd), device=dev)
    q[seq, node] = s["q"].float()
    mask = torch.zeros((seqs, most), dtype=torch.int64, device=dev)
    mask[seq, node] = s["mask"]
    k = s["k"][s["table"].long()].flatten(1, 2).float()  # [sequence, position, head, hd]
    v = s["v"][s["table"].long()].flatten(1, 2).float()
    pos = torch.arange(k.shape[1], device=dev)
    draft = pos[None] - ctx[:, None]  # the draft that a position holds, if 0 <= it < counts
    bit = (mask[:, :, None] >> draft.clamp(0, 63)[:, None]) & 1
    seen = (draft < 0)[:, None] | ((draft < counts[:, None])[:, None] & (bit == 1) & (draft >= 0)[:, None])
    q = q.view(seqs, most, hkv, hq // hkv, hd).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, most * (hq // hkv), hd)
    score = (q / math.sqrt(hd)) @ k.permute(0, 2, 3, 1)
    score = score.view(seqs, hkv, most, hq // hkv, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top.clamp_min(-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(seqs, hkv, most * (hq // hkv), -1) @ v.permute(0, 2, 1, 3)
    o = o.view(seqs, hkv, most, hq // hkv, hd) / total.clamp_min(1e-30)
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, most, hq, hd)[seq, node]
    return o.to(s["q"].dtype)


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return dict(k=s["k"], v=s["v"])


def _plain_compact(s):
    c = s["case"]
    page, dev = c["page"], s["k"].device
    bit = (s["accepted"][:, None] >> torch.arange(64, device=dev)) & 1
    rank = bit.cumsum(1) - bit
    seq, j = bit.nonzero(as_tuple=True)
    src, dst = s["ctx"].long()[seq] + j, s["ctx"].long()[seq] + rank[seq, j]
    table = s["table"].long()
    src, dst = table[seq, src // page] * page + src % page, table[seq, dst // page] * page + dst % page
    for x in (s["k"], s["v"]):
        flat = x.view(c["layers"], -1, c["hkv"], c["hd"])
        flat[:, dst] = flat[:, src]
    s["new_len"].copy_(s["ctx"] + bit.sum(1))
    return dict(k=s["k"], v=s["v"], new_len=s["new_len"])


def _plain_sample(s):
    c = s["case"]
    x = s["logits"].double()
    x, index = x.sort(dim=-1, descending=True, stable=True)  # equal logits keep their order: lowest index first
    w = ((x - x[:, :1]) / s["temperature"].double()[:, None]).exp()
    if c["top_k"]:
        w[:, c["top_k"] :] = 0
    cum = w.cumsum(-1)
    keep = (cum - w < c["top_p"] * cum[:, -1:]) if c["top_p"] < 1 else torch.ones_like(w, dtype=torch.bool)
    w = w * (keep & (w >= c["min_p"]))
    cum = w.cumsum(-1)
    total = cum[:, -1:]
    at = (cum <= s["u"].double()[:, None] * total).sum(-1, keepdim=True)
    at = at.clamp_max(c["n"] - 1)
    return dict(idx=index.gather(1, at)[:, 0].int(), prob=(w.gather(1, at) / total)[:, 0].float())


# -------------------------------------------------------------------------------------------- run
def _own(s):
    import pyxis_b200 as px

    c = s["case"]
    op = c["op"]
    if op == "rope":
        q = px.qk_norm_rope_dev(s["qkv"], s["positions"], s["inv_freq"], c["hq"], c["hkv"], c["hd"], q_norm=s.get("q_norm"),
                                k_norm=s.get("k_norm"), eps=1e-6, interleaved=c["inter"], rope_scale=s["scale"],
                                k_pages=s["k"], v_pages=s["v"], slots=s["slots"])
        return dict(q=q, k=s["k"], v=s["v"])
    if op == "tree":
        return px.tree_attention_dev(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["start"], s["mask"],
                                     max_tree=s["max_tree"], max_context=s["max_ctx"])
    if op == "copy":
        px.kv_copy_pages_dev(s["k"], s["v"], s["src"], s["dst"])
        return dict(k=s["k"], v=s["v"])
    if op == "compact":
        px.kv_compact_dev(s["k"], s["v"], s["table"], s["ctx"], s["accepted"], new_len=s["new_len"])
        return dict(k=s["k"], v=s["v"], new_len=s["new_len"])
    idx, prob = px.sample_dev(s["logits"], s["u"], temperature=s["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
    return dict(idx=idx, prob=prob)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    plain = dict(rope=_plain_rope, tree=_plain_tree, copy=_plain_copy, compact=_plain_compact, sample=_plain_sample)
    return plain[op](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    op, e = case["op"], 4 if case["dtype"] == "f32" else 2
    if op == "rope":
        row = (case["hq"] + 2 * case["hkv"]) * case["hd"]
        pairs = (case["hq"] + case["hkv"]) * case["rot"] // 2
        flops = 6 * pairs + (4 * (case["hq"] + case["hkv"]) * case["hd"] if case["norm"] else 0)
        return dict(bytes=case["tokens"] * (2 * row * e + 8) + 4 * case["rot"], flops=case["tokens"] * flops)
    if op == "tree":
        ctx, trees = _lengths(case)
        keys = int((ctx + trees).sum()) * case["hkv"] * case["hd"] * 2 * e
        rows = 2 * int(trees.sum()) * case["hq"] * case["hd"] * e
        pairs = int((trees * (ctx + trees)).sum()) * case["hq"]
        return dict(bytes=keys + rows + 4 * int((-(-(ctx + trees) // case["page"])).sum()) + 8 * int(trees.sum()),
                    flops=4 * case["hd"] * pairs)
    if op == "copy":
        return dict(bytes=case["pairs"] * (case["layers"] * case["page"] * case["hkv"] * case["hd"] * 2 * 2 * e + 8), flops=0)
    if op == "compact":
        # an accepted node that is not in its place yet is read and written once
        bits = (_accepted(case)[:, None] >> np.arange(64)) & 1
        moved = int(((bits == 1) & (bits.cumsum(1) - 1 != np.arange(64))).sum())
        return dict(bytes=moved * case["layers"] * case["hkv"] * case["hd"] * 2 * 2 * e + 24 * case["seqs"], flops=0)
    return dict(bytes=case["rows"] * (case["n"] * e + 16), flops=4 * case["rows"] * case["n"])


# ------------------------------------------------------------------- the definitions in 64 bits
def _exact_rope(s):
    c = s["case"]
    hq, hkv, hd, rot = c["hq"], c["hkv"], c["hd"], c["rot"]
    x = s["qkv"].double().reshape(c["tokens"], -1, hd)
    z = torch.polar(torch.full_like(s["inv_freq"], s["scale"]).expand(c["tokens"], -1).contiguous(),
                    torch.remainder(s["positions"].double()[:, None] * s["inv_freq"], 2 * math.pi))
    first = torch.arange(0, rot, 2, device=x.device) if c["inter"] else torch.arange(rot // 2, device=x.device)
    second = first + (1 if c["inter"] else rot // 2)
    heads = x[:, : hq + hkv].clone()
    if c["norm"]:
        heads /= (heads.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        heads[:, :hq] *= s["q_norm"].double()
        heads[:, hq:] *= s["k_norm"].double()
    turned = torch.complex(heads[..., first], heads[..., second]) * z[:, None]
    heads[..., first], heads[..., second] = turned.real, turned.imag
    k, v = s["k"].double(), s["v"].double()
    at = s["slots"].long()
    k.view(-1, hkv, hd)[at[at >= 0]] = heads[at >= 0, hq:]
    v.view(-1, hkv, hd)[at[at >= 0]] = x[at >= 0, hq + hkv :]
    return dict(q=heads[:, :hq], k=k, v=v)


def _exact_tree(s):
    c = s["case"]
    hkv, group, page = c["hkv"], c["hq"] // c["hkv"], c["page"]
    start, ctx, mask = s["start"].tolist(), s["ctx"].tolist(), s["mask"].cpu().numpy().view(np.uint64)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(ctx):
        lo, hi = start[i], start[i + 1]
        total = length + hi - lo
        pages = s["table"][i, : -(-total // page)].long()
        k, v = (x[pages].reshape(-1, hkv, c["hd"])[:total].double() for x in (s["k"], s["v"]))
        bits = (mask[lo:hi, None] >> np.arange(hi - lo, dtype=np.uint64)) & np.uint64(1)
        seen = torch.from_numpy(np.concatenate([np.ones((hi - lo, length), bool), bits.astype(bool)], 1)).cuda()
        for h in range(hkv):
            q = s["q"][lo:hi, h * group : (h + 1) * group].double()
            score = torch.einsum("tgd,ld->tgl", q, k[:, h]) / math.sqrt(c["hd"])
            p = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1)
            out[lo:hi, h * group : (h + 1) * group] = torch.einsum("tgl,ld->tgd", p, v[:, h])
    return out


def _exact_sample(s):
    """Row by row on the host: sorts, walks the tokens from the most likely one, drops and draws."""
    c = s["case"]
    probs, tokens = [], []
    logits, t, u = s["logits"].double().cpu().numpy(), s["temperature"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    for x, temperature, r in zip(logits, t, u):
        order = np.argsort(-x, kind="stable")
        w = np.exp((x[order] - x[order[0]]) / temperature)
        w = w[: c["top_k"]] if c["top_k"] else w
        if c["top_p"] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            w = w[: np.count_nonzero(before < c["top_p"] * w.sum())]
        w = w[: np.count_nonzero(w >= c["min_p"])]
        at = min(int(np.searchsorted(np.cumsum(w), r * w.sum(), side="right")), len(w) - 1)
        tokens.append(order[at])
        probs.append(w[at] / w.sum())
    return dict(idx=torch.tensor(np.array(tokens), dtype=torch.int32), prob=torch.tensor(probs, dtype=torch.float64))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_rope(s)
    if op == "tree":
        return _exact_tree(s)
    if op == "copy":
        src, dst = s["src"].tolist(), s["dst"].tolist()
        k, v = s["k"].double(), s["v"].double()
        for a, b in zip(src, dst):
            k[:, b], v[:, b] = s["k"][:, a].double(), s["v"][:, a].double()
        return dict(k=k, v=v)
    if op == "compact":
        k, v = s["k"].double(), s["v"].double()
        table, ctx, accepted, page = s["table"].tolist(), s["ctx"].tolist(), s["accepted"].tolist(), case["page"]
        lens = []
        for i, at in enumerate(ctx):
            rank = at
            for j in range(64):
                if accepted[i] >> j & 1:
                    to, of = (table[i][rank // page], rank % page), (table[i][(at + j) // page], (at + j) % page)
                    k[:, to[0], to[1]], v[:, to[0], to[1]] = s["k"][:, of[0], of[1]].double(), s["v"][:, of[0], of[1]].double()
                    rank += 1
            lens.append(rank)
        return dict(k=k, v=v, new_len=torch.tensor(lens, dtype=torch.int32))
    return _exact_sample(s)
