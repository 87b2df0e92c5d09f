"""The serving operators (include/pyxis_serve.h) on the GPU against plain 64-bit forms.

Tolerances (u = 2^-24, half a step of f32; h = half a step of the output type relative to the value:
u for f32, 2^-8 for bf16) bound the rounding of the formulas as the kernels evaluate them and were
written down before the first run; beside each stands what it counts."""
import math

import numpy as np
import pytest
import torch

import pyxis_b200 as px

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def half_step(dt):
    return U if dt == F32 else 2.0 ** -8


def dev(a, dt=None):
    t = torch.as_tensor(np.ascontiguousarray(a)).cuda()
    return t if dt is None else t.to(dt)


def rand(g, *shape, dt=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, dtype=F32) * scale).to(dt).cuda()


def new_pages(g, layers, num, size, heads, hd, dt, order="nd"):
    """K and V pages [layers, num, size, heads, hd] in some memory order, filled with NaN: what no call
    writes must stay what it is, and what no row sees must not matter."""
    def one():
        if order == "nd":
            return torch.full((layers, num, size, heads, hd), math.nan, dtype=dt, device="cuda")
        if order == "hd":  # heads before slots
            return torch.full((layers, num, heads, size, hd), math.nan, dtype=dt, device="cuda").transpose(2, 3)
        wide = torch.full((num, layers, size, heads, 2, hd), math.nan, dtype=dt, device="cuda")
        return wide.transpose(0, 1)[..., 1, :]  # layers inside pages, heads apart
    return one(), one()


# --------------------------------------------------------------------------- norm, rotation, append
def rope_reference(qkv, pos, inv_freq, hq, hkv, hd, qn, kn, eps, inter, m):
    x = qkv.double().cpu().reshape(qkv.shape[0], -1, hd)
    heads = x[:, : hq + hkv].clone()
    for lo, hi, w in ((0, hq, qn), (hq, hq + hkv, kn)):
        if w is not None:
            heads[:, lo:hi] = heads[:, lo:hi] / (heads[:, lo:hi].square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
    mag = heads.abs().clone()
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        a = pos.double().cpu()[:, None] * inv_freq.cpu()
        c, s = a.cos()[:, None] * m, a.sin()[:, None] * m
        i = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
        j = i + 1 if inter else i + rot // 2
        xi, xj = heads[..., i].clone(), heads[..., j].clone()
        heads[..., i], heads[..., j] = xi * c - xj * s, xj * c + xi * s
        mag[..., i] = mag[..., j] = (xi.abs() + xj.abs()) * m
    return heads[:, :hq], heads[:, hq:], x[:, hq + hkv:], mag


def check_rope(got, want, mag, hd, dt):
    # norm: the sum of hd squares is off by at most hd u relative (half of it in the root), 4 more
    # operations; cos and sin by u of rounding the angle times 1 and 2 u of sincosf's own 1.5 ulp, the
    # scale and the products 3 u: (hd / 2 + 12) u of the magnitudes that are added; then the type's step
    tol = (hd / 2 + 12) * U * mag + half_step(dt) * want.abs() * (1 + 2.0 ** -7) + 1e-30
    bad = (got.double().cpu() - want).abs() - tol
    assert bad.max() <= 0, bad.max()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n,hq,hkv,hd,rot,inter,norm,order", [
    (1, 16, 8, 128, 128, False, True, "nd"), (1, 1, 1, 64, 64, True, False, "hd"), (7, 6, 2, 64, 32, False, True, "lay"),
    (33, 5, 1, 128, 64, True, True, "hd"), (130, 8, 8, 128, 0, False, True, "nd"), (5, 3, 3, 64, 16, True, True, "nd"),
    (1501, 4, 2, 64, 48, False, False, "lay"), (1300, 16, 8, 128, 128, True, True, "nd")])
def test_qk_norm_rope(dt, n, hq, hkv, hd, rot, inter, norm, order):
    g = torch.Generator().manual_seed(n * 31 + rot)
    qkv = rand(g, n, (hq + 2 * hkv) * hd, dt=dt, scale=2.0)
    kp, vp = new_pages(g, 1, (n + 15) // 16 + 3, 16, hkv, hd, dt, order)
    kp, vp = kp[0], vp[0]
    perm = torch.randperm(kp.shape[0] * 16, generator=g)[:n]
    slots = perm.clone()
    if n > 4:
        slots[2], slots[n - 1], slots[3] = -1, kp.shape[0] * 16, -(1 << 31)  # none of them is a place
    pos = torch.randint(0, 1 << 20, (n,), generator=g, dtype=torch.int32).cuda()
    f, m = (None, 1.0) if rot == 0 else px.rope_frequencies(rot, 1e6, "yarn", factor=4.0, original_context=4096)
    f = None if f is None else dev(f)
    qn, kn = (1 + 0.2 * rand(g, hd), 1 + 0.2 * rand(g, hd)) if norm else (None, None)
    q = px.qk_norm_rope_dev(qkv, pos, f, hq, hkv, hd, k_pages=kp, v_pages=vp, slots=slots.int().cuda(), q_norm=qn, k_norm=kn,
                            eps=1e-5, interleaved=inter, rope_scale=m)
    wq, wk, wv, mag = rope_reference(qkv, pos, f, hq, hkv, hd, qn, kn, 1e-5, inter, float(np.float32(m)))
    check_rope(q, wq, mag[:, :hq], hd, dt)
    ok = ((slots >= 0) & (slots < kp.shape[0] * 16)).nonzero()[:, 0]
    flat_k, flat_v = kp.reshape(-1, hkv, hd).cpu(), vp.reshape(-1, hkv, hd).cpu()
    check_rope(flat_k[slots[ok]], wk[ok], mag[ok, hq:], hd, dt)
    assert torch.equal(flat_v[slots[ok]].double(), wv[ok])
    rest = torch.ones(len(flat_k), dtype=torch.bool)
    rest[slots[ok]] = False
    assert flat_k[rest].isnan().all() and flat_v[rest].isnan().all()


@pytest.mark.parametrize("pos", [0, 1, 4095, 131071, 1 << 24, (1 << 31) - 1, -5])
def test_rope_angles_hold_at_far_positions(pos):
    g = torch.Generator().manual_seed(3)
    qkv = rand(g, 1, 3 * 128)
    kp, vp = new_pages(g, 1, 1, 16, 1, 128, F32)
    f, _ = px.rope_frequencies(128, 1e4)
    f = dev(f)
    p = torch.tensor([pos], dtype=torch.int32).cuda()
    q = px.qk_norm_rope_dev(qkv, p, f, 1, 1, 128, k_pages=kp[0], v_pages=vp[0], slots=torch.zeros(1, dtype=torch.int32).cuda())
    want, _, _, mag = rope_reference(qkv, p, f, 1, 1, 128, None, None, 0, False, 1.0)
    check_rope(q, want, mag[:, :1], 128, F32)


def test_rope_in_place_and_into_a_wider_buffer():
    g = torch.Generator().manual_seed(4)
    n, hq, hkv, hd = 9, 4, 2, 64
    qkv = rand(g, n, (hq + 2 * hkv) * hd)
    f, _ = px.rope_frequencies(64, 1e4)
    f, pos, slots = dev(f), torch.arange(n, dtype=torch.int32).cuda(), torch.arange(n, dtype=torch.int32).cuda()
    kp, vp = new_pages(g, 1, 1, 16, hkv, hd, F32)
    want = px.qk_norm_rope_dev(qkv, pos, f, hq, hkv, hd, k_pages=kp[0], v_pages=vp[0], slots=slots)
    wide = torch.full((n, 2 * hq, hd), 7.0, device="cuda")
    px.qk_norm_rope_dev(qkv, pos, f, hq, hkv, hd, k_pages=kp[0], v_pages=vp[0], slots=slots, q=wide[:, :hq])
    assert torch.equal(wide[:, :hq], want) and (wide[:, hq:] == 7).all()
    mine = qkv.clone()
    q = px.qk_norm_rope_dev(mine, pos, f, hq, hkv, hd, k_pages=kp[0], v_pages=vp[0], slots=slots,
                            q=mine.view(n, -1, hd)[:, :hq])
    assert torch.equal(q, want) and torch.equal(mine[:, hq * hd:], qkv[:, hq * hd:])
    with pytest.raises(px.PyxisError):
        px.qk_norm_rope_dev(mine, pos, f, hq, hkv, hd, k_pages=kp[0], v_pages=vp[0], slots=slots,
                            q=mine.view(n, -1, hd)[:, 1:hq + 1])


# --------------------------------------------------------------------------------- tree attention
def tree_masks(rng, n):
    mask = np.zeros(n, np.uint64)
    for j in range(n):
        mask[j] = np.uint64(1 << j) | (mask[rng.integers(0, j)] if j else np.uint64(0))
    return mask


class Tree:
    """A batch: pages with NaN wherever no sequence has written, ragged contexts and trees."""

    def __init__(self, seed, ctx, trees, hq, hkv, hd, dt, page=16, order="nd", q_scale=1.0, chain=False):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.ctx, self.trees, self.hq, self.hkv, self.hd, self.dt, self.page = ctx, trees, hq, hkv, hd, dt, page
        need = [-(-(c + t) // page) for c, t in zip(ctx, trees)]
        num = sum(need) + 2
        k, v = new_pages(g, 1, num, page, hkv, hd, dt, order)
        self.k, self.v = k[0], v[0]
        order_ = rng.permutation(num)
        self.table = np.full((len(ctx), max(max(need), 1)), -7, np.int32)  # -7: never looked at
        at = 0
        self.keys, self.vals = [], []
        for i, c in enumerate(need):
            self.table[i, :c] = order_[at : at + c]
            at += c
            n = ctx[i] + trees[i]
            kk, vv = rand(g, n, hkv, hd, dt=dt), rand(g, n, hkv, hd, dt=dt)
            self.keys.append(kk.double().cpu())
            self.vals.append(vv.double().cpu())
            pos = np.arange(n)
            if n:
                pages, slots = dev(self.table[i][pos // page].astype(np.int64)), dev(pos % page)
                self.k[pages, slots], self.v[pages, slots] = kk, vv
        self.start = np.concatenate([[0], np.cumsum(trees)]).astype(np.int32)
        self.mask = np.concatenate([tree_masks(rng, t) for t in trees] + [np.zeros(0, np.uint64)])
        if chain:
            self.mask = np.concatenate([np.array([(2 << j) - 1 for j in range(t)], np.uint64) for t in trees])
        self.q = rand(g, int(self.start[-1]), hq, hd, dt=dt, scale=q_scale)

    def args(self):
        return (self.q, self.k, self.v, dev(self.table), dev(np.array(self.ctx, np.int32)), dev(self.start),
                dev(self.mask.view(np.int64)))

    def run(self, **kw):
        kw.setdefault("max_tree", max(1, max(self.trees)))
        return px.tree_attention_dev(*self.args(), **kw)

    def check(self, out, scale=None):
        scale = self.hd ** -0.5 if scale is None else scale
        G, h, worst = self.hq // self.hkv, half_step(self.dt), -1.0
        q, out = self.q.double().cpu(), out.double().cpu()
        for i, (c, t) in enumerate(zip(self.ctx, self.trees)):
            if t == 0:
                continue
            lo = int(self.start[i])
            bits = (self.mask[lo : lo + t, None] >> np.arange(t, dtype=np.uint64)) & np.uint64(1)
            seen = torch.from_numpy(np.concatenate([np.ones((t, c), bool), bits.astype(bool)], 1))
            for head in range(self.hq):
                qq, kk, vv = q[lo : lo + t, head], self.keys[i][:, head // G], self.vals[i][:, head // G]
                s = (qq @ kk.T) * scale
                s = s.masked_fill(~seen, -math.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)  # a row that sees nothing is zero
                vv = torch.where(seen.any(0)[:, None], vv, 0.0)
                want, A = p @ vv, p @ vv.abs()
                # a score is off by delta: (hd + 3) u of sum |q k| (the products' sum, q times scale),
                # and 2 u of it in log2 units and its difference to the maximum; exp2 is off by 2 ulp; a
                # weight by e = 2 delta + 4 u; the sums of n terms by n u; numerator and sum both: twice.
                # bf16 may round each weight to bf16 before P V: 2^-8 of A, twice with its sum.
                mag = (qq.abs() @ kk.abs().T).where(seen, torch.zeros(())).amax(-1, keepdim=True) * abs(scale)
                e = 2 * (self.hd + 7) * U * mag + 4 * U
                if self.dt == BF16:
                    e = e + 2.0 ** -8
                tol = 2 * (e + (c + t) * U) * A * 1.05 + h * want.abs() * 1.05 + 1e-30
                err = (out[lo : lo + t, head] - want).abs()
                worst = max(worst, float((err / tol).nan_to_num(nan=math.inf).max()))
        assert worst <= 1.0, worst


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("ctx,trees,hq,hkv,hd,page,order", [
    ([1], [1], 1, 1, 64, 16, "nd"), ([0], [1], 2, 1, 128, 16, "nd"), ([0, 5], [3, 0], 2, 2, 64, 16, "hd"),
    ([31, 32, 33, 0], [1, 1, 1, 1], 16, 8, 128, 16, "nd"), ([127, 128, 129], [2, 2, 2], 4, 2, 128, 64, "lay"),
    ([152], [1], 16, 8, 128, 16, "nd"), ([700, 3, 64], [8, 5, 13], 8, 2, 128, 16, "hd"),
    ([90, 1000], [64, 33], 8, 4, 64, 32, "nd"), ([257], [64], 8, 1, 128, 16, "lay"), ([0], [64], 3, 1, 128, 16, "nd"),
    ([2303, 40, 1500], [16, 16, 7], 16, 8, 128, 16, "nd"), ([5000], [3], 6, 2, 64, 1, "nd"), ([300], [47], 21, 3, 64, 7, "hd")])
def test_tree_attention(dt, ctx, trees, hq, hkv, hd, page, order):
    t = Tree(sum(ctx) + 7, ctx, trees, hq, hkv, hd, dt, page, order)
    t.check(t.run())
    t.check(t.run(max_context=max(ctx)))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_chain_is_the_causal_mask(dt):
    t = Tree(11, [70, 0], [20, 9], 4, 2, 64, dt, chain=True)
    a = t.args()
    out = px.tree_attention_dev(*a[:6], None, max_tree=20)
    t.check(out)
    assert torch.equal(out, t.run())


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd,ctx", [(64, 0), (128, 0), (128, 200), (64, 1000)])
def test_rows_that_see_nothing_and_hidden_non_finite_drafts(dt, hd, ctx):
    t = Tree(12, [ctx, ctx], [9, 5], 4, 2, hd, dt)
    t.mask[3] = 0  # sees the context alone: nothing at all where ctx is 0
    for bad in (2, 4):  # drafts of the first sequence that some rows see and some do not
        pos = ctx + bad
        pg, sl = int(t.table[0, pos // t.page]), pos % t.page
        t.v[pg, sl, 0, 5] = math.inf if bad == 2 else math.nan
        t.v[pg, sl, 1] = -math.inf
        t.k[pg, sl, :, 0] = math.nan if bad == 4 else 1.0
    out = t.run()
    hidden = (t.mask & np.uint64((1 << 2) | (1 << 4))) == 0
    hidden[9:] = True
    rows = torch.from_numpy(np.nonzero(hidden)[0])
    assert len(rows) > 6 and out.cpu()[rows].isfinite().all()
    sees = torch.from_numpy(np.nonzero(~hidden)[0])
    assert len(sees) > 0 and not out.cpu()[sees][:, :2, 5].isfinite().any()  # heads 0, 1 read kv head 0
    # the finite rows are those of the same batch without the bad values
    clean = Tree(12, [ctx, ctx], [9, 5], 4, 2, hd, dt)
    clean.mask[3] = 0
    ref = clean.run()
    clean.check(ref)
    assert torch.equal(out.cpu()[rows], ref.cpu()[rows])
    if ctx == 0:
        assert (out[3] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_rows_outside_the_sequences_are_left_alone(dt):
    t = Tree(13, [50, 20], [4, 3], 4, 2, 64, dt)
    q, k, v, table, ctx, start, mask = t.args()
    pad = torch.cat([torch.zeros_like(q[:2]), q, torch.full_like(q[:5], math.nan)])
    out = torch.full((len(pad), 6, 64), 3.0, dtype=dt, device="cuda")
    m = torch.cat([mask[:2], mask, mask[:5]])
    px.tree_attention_dev(pad, k, v, table, ctx, start + 2, m, max_tree=4, out=out[:, 1:5])
    t.check(out[2:9, 1:5])
    assert (out[:2] == 3).all() and (out[9:] == 3).all() and (out[:, 0] == 3).all() and (out[:, 5] == 3).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_bad_pages_and_lengths_stay_inside_the_cache(dt):
    t = Tree(14, [100, 60], [4, 3], 4, 2, 64, dt)
    t.table[0, 2], t.table[0, 3] = -(1 << 31), (1 << 31) - 1
    q, k, v, table, ctx, start, mask = t.args()
    out = px.tree_attention_dev(q, k, v, table, ctx, start, mask, max_tree=4)
    good = Tree(14, [100, 60], [4, 3], 4, 2, 64, dt)
    assert torch.equal(out[4:], good.run()[4:])
    # contexts beyond the table, below zero; rows beyond the buffer
    for c, s in (([1 << 30, 60], [0, 4, 7]), ([-3, 60], [0, 4, 7]), ([100, 60], [0, 4, 1 << 30]), ([100, 60], [-9, 4, 2])):
        px.tree_attention_dev(q, k, v, dev(good.table), dev(np.array(c, np.int32)), dev(np.array(s, np.int32)), mask, max_tree=4)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_large_scores_and_an_explicit_scale(dt):
    t = Tree(15, [400, 33], [6, 2], 8, 4, 128, dt, q_scale=12.0)  # scores to about +-150: few keys have weight
    t.check(t.run())
    t.check(t.run(scale=0.02), scale=0.02)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_cache_past_32_bit_offsets(dt):
    hkv, hd, page = 1, 128, 64
    num = (1 << 32) // (page * hd) + 40 if dt == BF16 else (1 << 31) // (page * hd) + 40
    k = torch.empty((num, page, hkv, hd), dtype=dt, device="cuda")
    v = torch.empty_like(k)
    t = Tree(16, [700], [3], 2, 1, hd, dt, page)
    table = (num - 1 - np.arange(t.table.shape[1])).astype(np.int32)[None]
    for i, p in enumerate(t.table[0]):
        k[int(table[0, i])], v[int(table[0, i])] = t.k[int(p)], t.v[int(p)]
    a = t.args()
    out = px.tree_attention_dev(t.q, k, v, dev(table), *a[4:], max_tree=3)
    t.check(out)
    slots = torch.tensor([num * page - 1], dtype=torch.int32).cuda()
    px.qk_norm_rope_dev(torch.ones((1, 4 * hd), dtype=dt, device="cuda"), None, None, 2, 1, hd, k_pages=k, v_pages=v, slots=slots)
    assert (k[-1, -1] == 1).all() and (v[-1, -1] == 1).all()


def test_tree_workspace_is_checked_and_enough():
    t = Tree(17, [3000], [3], 2, 1, 64, F32)
    want = t.run()
    with pytest.raises(px.PyxisError):
        t.run(workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    assert torch.equal(t.run(workspace=torch.empty(4 << 20, dtype=torch.uint8, device="cuda")), want)


def relaid(x, pad=0, slots=0, order="nd"):
    """The same pages [num, size, heads, hd] in other strides, NaN between."""
    num, size, heads, hd = x.shape
    if order == "heads":  # heads outermost
        wide = torch.full((heads, num, size + slots, hd + pad), math.nan, dtype=x.dtype, device="cuda").permute(1, 2, 0, 3)
    else:
        wide = torch.full((num, size + slots, heads, hd + pad), math.nan, dtype=x.dtype, device="cuda")
    y = wide[:, :size, :, :hd]
    y.copy_(x)
    return y


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("trees", [[20, 5], [2, 1]])
def test_cache_strides(dt, hd, trees):
    t = Tree(30, [700, 131], trees, 8, 4, hd, dt)
    want = t.run()
    t.check(want)
    a = t.args()
    for pad, slots, order in ((8, 0, "nd"), (16, 3, "nd"), (64, 0, "nd"), (0, 0, "heads"), (24, 1, "heads")):
        k, v = relaid(t.k, pad, slots, order), relaid(t.v, pad, slots, order)
        assert torch.equal(px.tree_attention_dev(a[0], k, v, *a[3:], max_tree=max(trees)), want)
    # one kv head; keys and values in one buffer
    t = Tree(31, [300], [trees[0]], 4, 1, hd, dt)
    a, both = t.args(), torch.stack([t.k, t.v], 2)
    assert torch.equal(px.tree_attention_dev(a[0], relaid(t.k, 8), relaid(t.v, 8), *a[3:], max_tree=trees[0]), t.run())
    out = px.tree_attention_dev(a[0], both[:, :, 0], both[:, :, 1], *a[3:], max_tree=trees[0])
    t.check(out)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("trees", [[40, 3, 0, 17], [2, 1, 1, 2]])
@pytest.mark.parametrize("page", [1, 8, 24, 64, 128, 256, 384])
def test_page_sizes(dt, hd, trees, page):
    t = Tree(page, [700, 127, 385, 0], trees, 6, 3, hd, dt, page)
    t.check(t.run())


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("nodes", [1, 12])
def test_many_ragged_sequences(dt, nodes):
    rng = np.random.default_rng(nodes)
    n = 1100
    ctx, trees = rng.integers(0, 70, n), rng.integers(0, nodes + 1, n)
    ctx[::97] = rng.integers(0, 600, len(ctx[::97]))
    t = Tree(nodes, ctx.tolist(), trees.tolist(), 4, 2, 64, dt)
    t.check(t.run())
    t.check(t.run(max_context=600))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("trees", [[40, 9], [8, 3], [2, 1]])
def test_odd_strides_of_rows_and_negative_scales(dt, trees):
    t = Tree(33, [333, 90], trees, 8, 4, 64, dt)
    a, n = t.args(), sum(trees)
    want = t.run()
    q = torch.full((n, 9, 67), math.nan, dtype=dt, device="cuda")[:, 1:, 3:]
    q.copy_(t.q)
    buf = torch.full((n, 9, 65), 7.0, dtype=dt, device="cuda")
    got = px.tree_attention_dev(q, *a[1:], max_tree=max(trees), out=buf[:, :8, 1:])
    assert torch.equal(got, want)
    assert (buf[:, 8] == 7).all() and (buf[:, :, 0] == 7).all()
    for scale in (-0.11, 0.0, 1e-3):
        t.check(t.run(scale=scale), scale=scale)
        assert torch.equal(px.tree_attention_dev(q, *a[1:], max_tree=max(trees), scale=scale, out=buf[:, :8, 1:]), t.run(scale=scale))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("group,nodes", [(1, 64), (2, 10), (16, 3)])
def test_nodes_past_max_tree_and_masks_past_the_tree(dt, group, nodes):
    hq = 2 * group
    t = Tree(34, [150, 40], [nodes, 2], hq, 2, 128, dt)
    t.check(t.run())
    if nodes < 64:  # bits of nodes that are not there count for nothing
        want = t.run()
        t.mask |= np.uint64((1 << 63) | (1 << nodes))
        assert torch.equal(t.run(), want)
    most = max(2, nodes // 2)
    out = torch.full_like(t.q, 5.0)
    t.run(max_tree=most, out=out)
    assert (out[most:nodes] == 5).all() and (out[:most] != 5).any()
    part = Tree(34, [150, 40], [nodes, 2], hq, 2, 128, dt)
    part.mask[:] &= np.uint64((1 << most) - 1)  # the nodes left out are no keys either
    part.check(torch.cat([out[:most], part.run()[most:]]))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_every_tensor_on_a_side_stream_and_uint64_masks(dt):
    t = Tree(35, [900, 4, 60], [30, 1, 64], 4, 1, 128, dt)
    a = t.args()
    want = t.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = [x.clone() for x in a[:6]] + [a[6].view(torch.uint64).clone()]
        out = px.tree_attention_dev(*b, max_tree=64)
    s.synchronize()
    assert torch.equal(out, want)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")  # two calls at once: a workspace each
    out2 = torch.empty_like(out)
    with torch.cuda.stream(s):
        px.tree_attention_dev(*b, max_tree=64, out=out2, workspace=ws)
    out3 = t.run()
    torch.cuda.synchronize()
    assert torch.equal(out2, want) and torch.equal(out3, want)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e18])
def test_tree_attention_of_very_small_and_large_values(dt, size):
    # scores of an ordinary size from keys far from 1, values far from 1, and one tile much larger than the rest
    t = Tree(36, [500, 70], [20, 40], 4, 2, 128, dt)
    t.k *= size
    t.v *= size
    t.v[int(t.table[0, 20])] *= 64.0
    t.q /= size
    for i in range(2):
        n = t.ctx[i] + t.trees[i]
        pos = np.arange(n)
        pages, slots = t.table[i][pos // t.page].astype(np.int64), pos % t.page
        t.keys[i], t.vals[i] = t.k[pages, slots].double().cpu(), t.v[pages, slots].double().cpu()
    t.check(t.run())


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ctx,nodes", [(0, 6), (200, 6), (0, 20), (200, 20), (60, 64), (0, 64), (192, 20), (192, 64), (180, 64)])
@pytest.mark.parametrize("size", [1e-30, 1e20, 3.3e38])
def test_hidden_drafts_of_any_size(dt, hd, ctx, nodes, size):
    t, clean = (Tree(40, [ctx, 77], [nodes, 3], 4, 2, hd, dt) for _ in range(2))
    for x in (t, clean):  # every node sees its own and node 1, and nodes 2 and 5 are seen by few
        x.mask[:nodes] = [np.uint64(1 << j | 2 | (4 if j % 5 == 0 else 0)) for j in range(nodes)]
    for d, sign in ((2, 1.0), (5, -1.0)):
        pos = ctx + d
        pg, sl = int(t.table[0, pos // t.page]), pos % t.page
        t.k[pg, sl] = sign * size
        t.v[pg, sl] = -sign * size
    hidden = (t.mask & np.uint64(4 | 32)) == 0
    hidden[nodes:] = True
    rows = torch.from_numpy(np.nonzero(hidden)[0]).cuda()
    assert 0 < len(rows) < len(hidden)
    want, out = clean.run(), t.run()
    clean.check(want)
    mixed = want.clone()
    mixed[rows] = out[rows]
    clean.check(mixed)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ctx,nodes", [(0, 6), (200, 6), (0, 20), (200, 20), (60, 64), (0, 64), (192, 20), (192, 64), (180, 64)])
def test_drafts_with_values_of_any_size(dt, hd, ctx, nodes):
    t = Tree(41, [ctx, 77], [nodes, 3], 4, 2, hd, dt)
    t.mask[5] = 1 << 5  # sees its own alone
    for d, size in ((0, 1e3), (2, 1e20), (5, 1e-20), (3, 0.0)):
        pos = ctx + d
        pg, sl = int(t.table[0, pos // t.page]), pos % t.page
        t.v[pg, sl] *= size
        t.vals[0][pos] = t.v[pg, sl].double().cpu()
    t.check(t.run())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_keys_and_values_that_change_size_along_the_cache(dt):
    # tiles of 64 keys far apart in size, up and down; the columns of V apart, too
    t = Tree(42, [900, 320], [24, 5], 4, 2, 128, dt)
    cols = torch.logspace(-2, 2, 128, device="cuda").to(dt)
    for i in range(2):
        n = t.ctx[i] + t.trees[i]
        pos = np.arange(n)
        pages, slots = t.table[i][pos // t.page].astype(np.int64), pos % t.page
        f = torch.tensor([(1.0, 300.0, 1e-3, 1e4)[(x // 64) % 4] for x in pos], device="cuda").to(dt)
        t.k[pages, slots] *= (f ** 0.25).to(dt)[:, None, None]
        t.v[pages, slots] *= f[:, None, None] * cols
        t.keys[i], t.vals[i] = t.k[pages, slots].double().cpu(), t.v[pages, slots].double().cpu()
    t.check(t.run())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_trees_over_a_cache_past_32_bit_offsets(dt):
    hkv, hd, page = 1, 128, 64
    num = ((1 << 32) if dt == BF16 else (1 << 31)) // (page * hd) + 40
    k = torch.full((num, page, hkv, hd), math.nan, dtype=dt, device="cuda")
    v = torch.full_like(k, math.nan)
    for nodes, ctx in ((6, 700), (40, 1000), (64, 0)):  # 12, 80 and 128 rows
        t = Tree(44, [ctx], [nodes], 2, 1, hd, dt, page)
        table = (num - 1 - np.arange(t.table.shape[1])).astype(np.int32)[None]
        for i, p in enumerate(t.table[0]):
            k[int(table[0, i])], v[int(table[0, i])] = t.k[int(p)], t.v[int(p)]
        a = t.args()
        t.check(px.tree_attention_dev(t.q, k, v, dev(table), *a[4:], max_tree=nodes))
    # pages copied and compacted there, too
    far = dev(np.array([num - 3], np.int32))
    px.kv_copy_pages_dev(k[None], v[None], far, dev(np.array([num - 30], np.int32)))
    assert torch.equal(k[num - 30].nan_to_num(), k[num - 3].nan_to_num())
    before = k[num - 30].clone()
    px.kv_compact_dev(k[None], v[None], dev(np.array([[num - 30]], np.int32)), dev(np.array([10], np.int32)),
                      dev(np.array([0b1010], np.int64)))
    assert torch.equal(k[num - 30, 10].nan_to_num(), before[11].nan_to_num())
    assert torch.equal(k[num - 30, 11].nan_to_num(), before[13].nan_to_num())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_few_nodes_in_a_long_buffer_of_rows(dt):
    t = Tree(45, [9000], [2], 8, 4, 64, dt)
    a = t.args()
    q = torch.zeros((200000, 8, 64), dtype=dt, device="cuda")
    q[150000:150002] = t.q
    mask = torch.zeros(200000, dtype=torch.int64, device="cuda")
    mask[150000:150002] = a[6]
    free = torch.cuda.mem_get_info()[0]
    out = torch.full_like(q, 2.0)
    px.tree_attention_dev(q, *a[1:5], a[5] + 150000, mask, max_tree=2, out=out)
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] < 2 << 30
    t.check(out[150000:150002])
    assert (out[:150000] == 2).all() and (out[150002:] == 2).all()


# ------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("layers,size,heads,hd,order", [(1, 16, 1, 64, "nd"), (3, 16, 8, 128, "nd"), (2, 5, 3, 64, "hd"), (4, 64, 2, 128, "lay")])
def test_copy_pages(dt, layers, size, heads, hd, order):
    g = torch.Generator().manual_seed(size)
    k, v = new_pages(g, layers, 12, size, heads, hd, dt, order)
    k.copy_(rand(g, *k.shape, dt=dt))
    v.copy_(rand(g, *v.shape, dt=dt))
    wk, wv = k.clone(), v.clone()
    src, dst = [3, 0, 11, 0, 4, -1, 12, 5], [1, 2, 6, 8, 4, 9, 9, 1 << 30]  # the last three name no page
    for a, b in list(zip(src, dst))[:5]:
        wk[:, b], wv[:, b] = k[:, a], v[:, a]
    px.kv_copy_pages_dev(k, v, dev(np.array(src, np.int32)), dev(np.array(dst, np.int32)))
    assert torch.equal(k, wk) and torch.equal(v, wv)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("layers,size,heads,hd,order", [(1, 16, 1, 64, "nd"), (3, 16, 8, 128, "nd"), (2, 5, 3, 64, "hd"), (2, 64, 2, 128, "lay")])
def test_compact(dt, layers, size, heads, hd, order):
    rng, g = np.random.default_rng(size), torch.Generator().manual_seed(size)
    acc = [0, 1, 0b10, 0b1011, 0b110100, (1 << 64) - 1, (1 << 64) - 2, 1 << 63, (1 << 64) // 3, 0b111]
    ctx = [0, 3, 15, 16, 17, 1, 40, 7, 33, 5]
    n, width = len(acc), -(-(40 + 64) // size)
    num = n * width
    k, v = new_pages(g, layers, num, size, heads, hd, dt, order)
    k.copy_(rand(g, *k.shape, dt=dt))
    v.copy_(rand(g, *v.shape, dt=dt))
    table = rng.permutation(num).astype(np.int32).reshape(n, width)
    wk, wv, lens = k.clone(), v.clone(), []
    for i in range(n):
        to = ctx[i]
        for j in range(64):
            if acc[i] >> j & 1:
                a, b = ctx[i] + j, to
                wk[:, table[i, b // size], b % size] = k[:, table[i, a // size], a % size]
                wv[:, table[i, b // size], b % size] = v[:, table[i, a // size], a % size]
                to += 1
        lens.append(to)
    bits = dev(np.array(acc, np.uint64).view(np.int64))
    new = px.kv_compact_dev(k, v, dev(table), dev(np.array(ctx, np.int32)), bits)
    assert new.tolist() == lens
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_compact_leaves_out_places_past_the_table():
    g = torch.Generator().manual_seed(1)
    k, v = new_pages(g, 1, 4, 16, 1, 64, F32)
    k.copy_(rand(g, *k.shape))
    v.copy_(rand(g, *v.shape))
    wk = k.clone()
    table = torch.tensor([[2, 99], [1, -1]], dtype=torch.int32).cuda()
    bits = torch.tensor([(1 << 4) | (1 << 9), (1 << 2) | (1 << 20) | (1 << 40)], dtype=torch.int64).cuda()
    new = px.kv_compact_dev(k, v, table, torch.tensor([10, 3], dtype=torch.int32).cuda(), bits)
    wk[:, 2, 10] = wk[:, 2, 14].clone()
    wk[:, 1, 3] = wk[:, 1, 5].clone()
    assert new.tolist() == [12, 6] and torch.equal(k, wk)


# --------------------------------------------------------------------------------------- sampling
def sample_reference(x, u, t, k, p, m):
    """One row by the definition, in 64 bits: (token, probability)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    if not t > 0:
        return order[0], 1.0
    x = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(x == x[0], 1.0, np.where(np.isinf(x), 0.0, np.exp((x - x[0]) / t)))
    if k > 0:
        w = w[:k]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        w = w[: max(1, np.count_nonzero(before < p * w.sum()))]
    w = w[: max(1, np.count_nonzero(w >= min(m, 1.0)))]
    u = min(max(u, 0.0), 1.0)
    c = np.cumsum(w)
    at = np.searchsorted(c, u * c[-1], side="right")
    if at >= len(w):
        at = np.nonzero(w)[0][-1]
    return order[at], w[at] / c[-1]


def check_sample(x, u, t, k, p, m, **kw):
    idx, prob = px.sample_dev(x, dev(np.asarray(u, np.float32)), t, k, p, m, **kw)
    xs, per = x.float().cpu().numpy(), lambda v, i: float(v[i]) if isinstance(v, torch.Tensor) else v  # noqa: E731
    for i in range(len(xs)):
        want = sample_reference(xs[i], float(np.float32(u[i])), per(t, i), int(per(k, i)), per(p, i), per(m, i))
        got = int(idx[i]), float(prob[i])
        assert got[0] == want[0], (i, got, want)
        # weights are 2^-44 steps of the largest (a share is off by less than 1e-9 of itself where it
        # can be drawn from so few numbers), the quotient rounds to f32
        assert abs(got[1] - want[1]) <= U * want[1] * 1.01 + 1e-12, (i, got, want)
    return idx, prob


def logits(seed, m, n, dt=F32, sigma=2.0, peaks=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g) * sigma
    if peaks:
        x += 6 * (torch.rand(m, n, generator=g) < 20.0 / n) * torch.rand(m, n, generator=g)
    return x.to(dt).cuda()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 2), (5, 31), (4, 1000), (3, 4097), (2, 40001), (4, 151936)])
@pytest.mark.parametrize("t,k,p,mp", [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 50, 1.0, 0.0), (1.0, 50, 0.9, 0.05), (0.7, 0, 1.0, 0.1),
                                      (1.0, 1, 1.0, 0.0), (2.0, 3000, 0.5, 0.0), (0.0, 7, 0.5, 0.1)])
def test_sample(dt, m, n, t, k, p, mp):
    u = np.random.default_rng(n + k).random(m)
    u[0] = 0.0
    if m > 2:
        u[2] = 1 - 2.0 ** -24
    check_sample(logits(n + m, m, n, dt), u, t, k, p, mp)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("kind", ["equal", "two", "steps", "flat", "cold", "hot"])
def test_sample_ties_and_flat_rows(dt, kind):
    m, n, t = 6, 20011, 1.0
    g = torch.Generator().manual_seed(9)
    if kind == "equal":
        x = torch.zeros(m, n)
        x[:, ::2] = -0.0
    elif kind == "two":
        x = (torch.rand(m, n, generator=g) < 0.3).float() * 3
    elif kind == "steps":
        x = torch.randint(0, 12, (m, n), generator=g).float() / 8
    elif kind == "flat":
        x = torch.randn(m, n, generator=g) * 1e-3
    else:
        x, t = torch.randn(m, n, generator=g), 1e-3 if kind == "cold" else 1e4
    x = x.to(dt).cuda()
    u = np.array([0.0, 0.1, 0.5, 0.77, 0.999, 0.3])
    check_sample(x, u, t, 0, 1.0, 0.0)
    check_sample(x, u, t, 5000, 1.0, 0.0)
    check_sample(x, u, t, 7000, 0.6, 0.0)
    check_sample(x, u, t, 0, 0.3, 0.5)


def test_sample_infinities_nan_and_empty_rows():
    n = 5000
    x = logits(3, 8, n).cpu()
    x[0, 100:] = -math.inf
    x[1, :] = -math.inf
    x[2, :] = math.nan
    x[3, ::2] = math.nan
    x[4, 17] = x[4, 3000] = math.inf
    x[5, :] = -math.inf
    x[5, 4999] = -3e38
    x[6, 7], x[6, 8] = 3.0e38, -3.0e38
    x[7, :] = torch.finfo(F32).min
    u = np.array([0.9, 0.5, 0.5, 0.7, 0.6, 0.2, 0.99, 0.5])
    check_sample(x.cuda(), u, 1.0, 0, 1.0, 0.0)
    check_sample(x.cuda(), u, 0.7, 20, 0.9, 0.01)
    idx, prob = check_sample(x.cuda(), u, 0.0, 0, 1.0, 0.0)
    assert idx.tolist()[1:3] == [-1, -1] and prob.tolist()[1:3] == [0.0, 0.0]


def test_sample_parameters_per_row_and_odd_values():
    m, n = 12, 9000
    t = torch.tensor([1.0, 0.0, -1.0, math.nan, 0.5, math.inf, 1e-30, 2.0, 1.0, 1.0, 1.0, 1.0])
    k = torch.tensor([0, 5, 5, 5, 1, 300, 2, -4, 1 << 30, 10, 0, 3], dtype=torch.int32)
    p = torch.tensor([1.0, 0.5, 0.5, 0.5, 0.9, 0.7, 0.9, 2.0, 0.0, -1.0, 1e-9, 0.999])
    mp = torch.tensor([0.0, 0.1, 0.0, 0.0, 0.0, 0.0, 0.0, -1.0, 0.0, 0.0, 0.0, 2.0])
    u = np.array([0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, -2.0, 1.0, 5.0, 0.5, 0.999])
    check_sample(logits(5, m, n), u, t.cuda(), k.cuda(), p.cuda(), mp.cuda())
    x = logits(5, 2, n)
    idx, _ = px.sample_dev(x, torch.tensor([math.nan, 0.0], device="cuda"))  # NaN draws like 0: the first token
    assert idx.tolist() == x.argmax(1).tolist()


def test_sample_rows_with_a_stride_and_odd_alignment():
    for dt in (F32, BF16):
        wide = logits(6, 5, 10003, dt)
        for lo in (0, 1, 3, 5):
            check_sample(wide[:, lo : lo + 9001], np.linspace(0, 0.99, 5), 0.9, 0, 0.95, 0.0)


def test_sample_rows_longer_than_shared_memory():
    check_sample(logits(7, 2, 700001, F32), [0.3, 0.9], 1.0, 0, 0.9, 0.0)
    check_sample(logits(8, 1, 2100000, BF16), [0.6], 1.5, 100000, 1.0, 0.0)


def test_greedy_rows_are_the_argmax():
    x = logits(10, 7, 151936)
    idx, _ = px.sample_dev(x, torch.rand(7, device="cuda"), temperature=0.0)
    assert idx.tolist() == px.argmax_dev(x)[0].tolist()


def test_many_rows_draw_with_the_right_frequencies():
    """20000 draws from one small distribution: each count within 6 standard deviations."""
    n, m = 8, 20000
    x = torch.tensor([[2.0, 1.0, 0.5, 0.0, 0.0, -1.0, -2.0, -8.0]]).cuda()
    u = torch.rand(m, generator=torch.Generator().manual_seed(2)).cuda()
    idx, prob = px.sample_dev(x.expand(m, n).contiguous(), u)
    p = torch.softmax(x[0].double(), 0)
    count = torch.bincount(idx.long(), minlength=n).double()
    assert ((count - m * p).abs() <= 6 * (m * p * (1 - p)).sqrt() + 1).all()
    assert torch.allclose(prob.double(), p[idx.long()], rtol=1e-6)


# ------------------------------------------------------------------------- streams, graphs, the step
def test_calls_on_another_stream_and_in_a_graph():
    t = Tree(20, [500, 90], [5, 3], 4, 2, 64, F32)
    a = t.args()
    x, u = logits(4, 8, 30000), torch.rand(8, device="cuda")
    want, (wi, wp) = t.run(), px.sample_dev(x, u, 0.8, 40, 0.9)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = px.tree_attention_dev(*a, max_tree=5)
        idx, prob = px.sample_dev(x, u, 0.8, 40, 0.9)
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(idx, wi) and torch.equal(prob, wp)
    out.zero_()
    idx.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        px.tree_attention_dev(*a, max_tree=5, out=out)
        px.sample_dev(x, u, 0.8, 40, 0.9, idx=idx, prob=prob)
    for _ in range(3):
        out.zero_()
        idx.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(idx, wi) and torch.equal(prob, wp)
    # a workspace that grows later leaves the graph's own in place
    big = Tree(21, [60000], [64], 16, 1, 64, F32)
    big.run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_verified_tree_continues_as_if_decoded_token_by_token(dt):
    """Two sequences, one a fork of the other: a tree of drafts is rotated, appended, attended and sampled;
    the accepted branch is compacted; the next token then gives what a token-by-token decode of the
    same branch gives."""
    g, page, hq, hkv, hd, vocab = torch.Generator().manual_seed(30), 16, 4, 2, 64, 500
    f, _ = px.rope_frequencies(hd, 1e4)
    f, head = dev(f), rand(g, vocab, hq * hd)
    qn, kn = 1 + 0.1 * rand(g, hd), 1 + 0.1 * rand(g, hd)
    pool = px.PagePool(32, page)
    k, v = new_pages(g, 2, 32, page, hkv, hd, dt)
    layer = 1

    def slots(table, pos):
        return torch.tensor([table[p // page] * page + p % page for p in pos], dtype=torch.int32).cuda()

    def step(tables, ctx, qkv, pos, masks, counts):
        width = max(len(t) for t in tables)
        bt = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32).cuda()
        place = torch.cat([slots(t, range(c, c + n)) for t, c, n in zip(tables, ctx, counts)])
        q = px.qk_norm_rope_dev(qkv, torch.tensor(pos, dtype=torch.int32).cuda(), f, hq, hkv, hd, k_pages=k[layer], v_pages=v[layer],
                                slots=place, q_norm=qn, k_norm=kn)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()
        out = px.tree_attention_dev(q, k[layer], v[layer], bt, torch.tensor(ctx, dtype=torch.int32).cuda(), cu,
                                    torch.tensor(masks, dtype=torch.int64).cuda(), max_tree=max(counts))
        x = out.float().reshape(len(qkv), -1) @ head.T
        idx, _ = px.sample_dev(x, torch.full((len(qkv),), 0.4, device="cuda"), 0.9, 40, 0.95)
        return out, idx, bt

    # a prompt of 37 tokens as chains of up to 64
    prompt = rand(g, 37, (hq + 2 * hkv) * hd, dt=dt)
    a = pool.allocate(37)
    step([a], [0], prompt, list(range(37)), [(2 << j) - 1 for j in range(37)], [37])
    b, src, dst = pool.fork(a, 37)
    px.kv_copy_pages_dev(k, v, torch.tensor(src, dtype=torch.int32).cuda(), torch.tensor(dst, dtype=torch.int32).cuda())
    c, src, dst = pool.fork(a, 37)  # the token-by-token one
    px.kv_copy_pages_dev(k, v, torch.tensor(src, dtype=torch.int32).cuda(), torch.tensor(dst, dtype=torch.int32).cuda())
    for t in (a, b, c):
        pool.grow(t, 37 + 8)
    # a tree: 0 - 1 - 3 - 6, 0 - 2 - 4, 2 - 5
    parent = [-1, 0, 0, 1, 2, 2, 3]
    depth, mask = [], []
    for j, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        mask.append((1 << j) | (0 if p < 0 else mask[p]))
    drafts = rand(g, 7, (hq + 2 * hkv) * hd, dt=dt)
    out, idx, bt = step([a, b], [37, 37], drafts.repeat(2, 1), [37 + d for d in depth] * 2, mask * 2, [7, 7])
    assert torch.equal(out[:7], out[7:]) and torch.equal(idx[:7], idx[7:])
    # a accepts 0 - 2 - 5, b accepts 0 - 1 - 3 - 6
    acc = torch.tensor([mask[5], mask[6]], dtype=torch.int64).cuda()
    new = px.kv_compact_dev(k, v, bt, torch.tensor([37, 37], dtype=torch.int32).cuda(), acc)
    assert new.tolist() == [40, 41]
    nxt = rand(g, 1, (hq + 2 * hkv) * hd, dt=dt)
    after, idx_after, _ = step([a], [40], nxt, [40], [1], [1])
    tol = 2e-5 if dt == F32 else 0.03  # other split of the same sums: (n + hd) u, a step of bf16 on top
    for i, j in enumerate((0, 2, 5)):
        one, tok, _ = step([c], [37 + i], drafts[j : j + 1], [37 + i], [1], [1])
        assert torch.allclose(one[0].float(), out[j].float(), atol=tol, rtol=tol)
    one, tok, _ = step([c], [40], nxt, [40], [1], [1])
    assert torch.allclose(one.float(), after.float(), atol=tol, rtol=tol) and tok.tolist() == idx_after.tolist()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("nodes", [5, 24])
def test_a_captured_verify_step_replays_as_the_calls_do(dt, nodes):
    """A padded batch of three (the last has no nodes) steps forward five times, by calls and by two
    captured graphs in turn that share the context's workspace; lengths and accepted nodes change."""
    g, page, hq, hkv, hd, vocab, n = torch.Generator().manual_seed(50), 16, 8, 4, 128, 3001, 3
    rng = np.random.default_rng(nodes)
    f, _ = px.rope_frequencies(hd, 1e6)
    f, head = dev(f), rand(g, vocab, hq * hd, scale=0.05)
    k0, v0 = rand(g, 2, 120, page, hkv, hd, dt=dt), rand(g, 2, 120, page, hkv, hd, dt=dt)
    width = 38
    table = dev(rng.permutation(120)[: n * width].reshape(n, width).astype(np.int32))
    mask = dev(np.concatenate([tree_masks(rng, nodes) for _ in range(n)]).view(np.int64))
    start = torch.tensor([0, nodes, 2 * nodes, 2 * nodes], dtype=torch.int32).cuda()
    rows = n * nodes  # the last third is padding
    qkv = rand(g, 5, rows, (hq + 2 * hkv) * hd, dt=dt)
    uni, accepted = torch.rand(5, rows, generator=g).cuda(), torch.from_numpy(rng.integers(0, 1 << nodes, (5, n))).cuda()
    accepted[:, 2] = 0
    node = torch.arange(nodes, device="cuda").repeat(n)
    seq = torch.arange(n, device="cuda").repeat_interleave(nodes)

    class State:
        def __init__(self):
            self.k, self.v = k0.clone(), v0.clone()
            self.ctx = torch.tensor([37, 500, 0], dtype=torch.int32).cuda()
            self.qkv, self.uni, self.acc = torch.empty_like(qkv[0]), torch.empty_like(uni[0]), torch.empty_like(accepted[0])
            self.q = torch.empty((rows, hq, hd), dtype=dt, device="cuda")
            self.out, self.new = torch.zeros_like(self.q), torch.zeros_like(self.ctx)
            self.idx, self.prob = torch.zeros(rows, dtype=torch.int32).cuda(), torch.zeros(rows).cuda()

        def feed(self, i):
            self.qkv.copy_(qkv[i]), self.uni.copy_(uni[i]), self.acc.copy_(accepted[i])

        def step(self):
            pos = (self.ctx.long()[seq] + node)
            slots = (table[seq, pos // page].long() * page + pos % page).int()
            slots[2 * nodes :] = -1
            for layer in range(2):
                px.qk_norm_rope_dev(self.qkv, pos.int(), f, hq, hkv, hd, k_pages=self.k[layer], v_pages=self.v[layer], slots=slots,
                                    q=self.q)
                px.tree_attention_dev(self.q, self.k[layer], self.v[layer], table, self.ctx, start, mask, max_tree=nodes, out=self.out)
            px.sample_dev(self.out.float().reshape(rows, -1) @ head.T, self.uni, 0.8, 50, 0.95, idx=self.idx, prob=self.prob)
            px.kv_compact_dev(self.k, self.v, table, self.ctx, self.acc, new_len=self.new)
            self.ctx.copy_(self.new)

    a, b = State(), State()
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # (warm-up on a state of its own)
        w = State()
        w.feed(0)
        w.step()
    side.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.step()
        graphs.append(graph)
    for i in range(5):
        a.feed(i)
        a.step()
        b.feed(i)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        for x in ("ctx", "out", "idx", "prob", "k", "v", "q"):
            assert torch.equal(getattr(a, x), getattr(b, x)), (i, x)
        assert (a.out[2 * nodes :] == 0).all() and int(a.ctx[2]) == 0
    assert a.out[: 2 * nodes].isfinite().all()
