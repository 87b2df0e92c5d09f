"""Precision and edge cases of the serving operators (include/pyxis_serve.h) on the GPU: how many bits the
weights of the attention keep, infinities in the cache, results on a stream of the caller's, weights next to
a border, the context's workspace.

Tolerances (u = 2^-24, half a step of f32; half_step of the output type relative to the value) were written
down before the first run; beside each stands what it counts."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import pyxis_b200 as px
from pyxis_b200 import _native
from test_serve_gpu import BF16, F32, U, Tree, dev, half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _waits_ended():
    """No kernel of the test gave up a bounded wait."""
    yield
    _native.check(_native.lib().pyxis_cuda_check_device_error(px.get_cuda(0).handle))


# ------------------------------------------------------------------------------ bits of the weights
def attention(t):
    """Per sequence: the sum p v, the sum p |v| and the largest sum |q k| of a row, in 64 bits."""
    q, G, scale = t.q.double().cpu(), t.hq // t.hkv, t.hd ** -0.5
    for i, (c, n) in enumerate(zip(t.ctx, t.trees)):
        if n == 0:
            continue
        lo = int(t.start[i])
        bits = (t.mask[lo : lo + n, None] >> np.arange(n, dtype=np.uint64)) & np.uint64(1)
        seen = torch.from_numpy(np.concatenate([np.ones((n, c), bool), bits.astype(bool)], 1))
        for head in range(t.hq):
            qq, kk, vv = q[lo : lo + n, head], t.keys[i][:, head // G], t.vals[i][:, head // G]
            p = torch.softmax(((qq @ kk.T) * scale).masked_fill(~seen, -math.inf), -1)
            mag = (qq.abs() @ kk.abs().T).where(seen, torch.zeros(())).amax(-1, keepdim=True) * scale
            yield slice(lo, lo + n), head, c + n, p @ vv, p @ vv.abs(), mag


@pytest.mark.parametrize("ctx,trees,hq,hkv,hd,page", [
    ([700, 3, 64], [8, 5, 13], 8, 2, 128, 16), ([90, 1000], [64, 33], 8, 4, 64, 32), ([2303, 40, 1500], [16, 16, 7], 16, 8, 128, 16),
    ([300], [5], 3, 3, 128, 64), ([5000], [64], 4, 2, 128, 64)])
def test_bf16_weights_are_not_rounded_to_bf16(ctx, trees, hq, hkv, hd, page):
    # As the f32 form's bound: scores off by (hd + 7) u of sum |q k|, twice, in their weights, 4 u of the
    # weights' own, n u of the sums, numerator and sum both; a weight as two bf16 terms is off by 2^-16; one
    # rounding of the output to bf16, at most 2^-8 of it.  (Weights rounded to bf16 would add 2^-8 of A.)
    t = Tree(51, ctx, trees, hq, hkv, hd, BF16, page)
    out, worst = t.run().double().cpu(), 0.0
    for rows, head, n, want, A, mag in attention(t):
        e = 2 * (hd + 7) * U * mag + 4 * U + 2.0 ** -16
        tol = 2 * (e + n * U) * A * 1.05 + half_step(BF16) * want.abs() * 1.05 + 1e-30
        worst = max(worst, float(((out[rows, head] - want).abs() / tol).nan_to_num(nan=math.inf).max()))
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [2, 6, 24, 64])  # a form of the f32 kernels each
@pytest.mark.parametrize("gap", [12.0, 17.25, 24.0])
def test_many_light_keys_behind_a_heavy_one(dt, hd, nodes, gap):
    """One key far above all others, whose weights (2^-17, 2^-24.9, 2^-34.6 of its own) are small, many and
    alike: each of them has to keep its bits, as their sum is a part in 10^1 to 10^6 of the result."""
    ctx = 40000
    t = Tree(52, [ctx], [nodes], 2, 1, hd, dt)
    pos = np.arange(ctx + nodes)
    pages, slots = dev(t.table[0][pos // t.page].astype(np.int64)), dev(pos % t.page)
    t.q.zero_()
    t.q[..., 0] = 4.0
    k, v = t.keys[0], t.vals[0].abs()
    k[:, :, 0] = 0.0
    k[0, :, 0] = 2 * gap  # exact in bf16; times q's 4 and the scale: the gap
    v[0] = 2.0 ** -14    # so that the light keys' part is seen beside the heavy one's
    t.k[pages, slots], t.v[pages, slots] = k.to(dt).cuda(), v.to(dt).cuda()
    t.vals[0] = v
    out = t.run(scale=0.125).double().cpu()
    seen = np.concatenate([np.ones((nodes, ctx)), ((t.mask[:, None] >> np.arange(nodes, dtype=np.uint64)) & np.uint64(1)).astype(float)], 1)
    w = torch.from_numpy(seen)
    w[:, 1:] *= math.exp(-gap)
    num, den = w @ t.vals[0][:, 0], w.sum(1, keepdim=True)
    # The score is one product: q, its scale in log2 units and the product round, 4 u of 1.44 gap; exp2 2 u;
    # two terms of a weight leave 2^-22 (f32 pages) or 2^-16 (bf16) of it; values of two terms 2^-22.  Sums
    # run over at most 64 keys a tile, then over the ctx / 64 tiles (in halves of a row, of a tensor-core
    # accumulation that cuts off: 2 u an addition), numerator and sum both.  All values are positive.
    e = 4 * U * 1.45 * gap + 2 * U + (2.0 ** -21 if dt == F32 else 2.0 ** -16) + 2 * (2 * U * (64 + ctx / 64))
    want = num / den
    bad = (out - want[:, None]).abs() / want[:, None] / (e * 1.05 + half_step(dt) * 1.05)
    assert bad.max() <= 1.0, bad.max()


# ------------------------------------------------------------------------------ infinities in the cache
def place(t, pos):
    return int(t.table[0, pos // t.page]), pos % t.page


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [2, 6, 24, 64])
@pytest.mark.parametrize("ctx,at", [(300, 100), (300, 299), (40, 3), (2000, 1999)])  # in a tile of context alone, in the drafts' tile
def test_a_key_with_an_infinity_reaches_rows_by_its_sign(dt, hd, nodes, ctx, at):
    """Its score is -inf where q is negative there: weight 0, a row like any other; +inf elsewhere: NaN."""
    t = Tree(53, [ctx, 70], [nodes, 3], 2, 1, hd, dt)
    t.q = t.q.to(BF16).to(dt)  # queries of few bits, so that a second term of theirs is zero
    pg, sl = place(t, at)
    t.k[pg, sl, 0, 3] = math.inf
    out = t.run(scale=1.0 / 16).cpu()
    below = (t.q[:nodes, :, 3] < 0).cpu()
    assert nodes == 2 or (below.any() and not below.all())
    got = out[:nodes]
    assert got[below].isfinite().all() and got[~below].isnan().all()
    # the rows with a score of -inf: softmax over the other keys
    q, keys, vals = t.q.double().cpu(), t.keys[0][:, 0], t.vals[0][:, 0]
    bits = (t.mask[:nodes, None] >> np.arange(nodes, dtype=np.uint64)) & np.uint64(1)
    seen = torch.from_numpy(np.concatenate([np.ones((nodes, ctx), bool), bits.astype(bool)], 1))
    seen[:, at] = False
    for h in range(2):
        p = torch.softmax((q[:nodes, h] @ keys.T / 16).masked_fill(~seen, -math.inf), -1)
        mag = (q[:nodes, h].abs() @ keys.abs().T).amax(-1, keepdim=True) / 16
        e = 2 * (hd + 7) * U * mag + 4 * U + (2.0 ** -16 if dt == BF16 else 2.0 ** -21)
        tol = 2 * (e + (ctx + nodes) * U) * (p @ vals.abs()) * 1.05 + half_step(dt) * (p @ vals).abs() * 1.05
        rows = below[:, h]
        assert ((got[rows, h].double() - p[rows] @ vals).abs() <= tol[rows]).all()
    assert out[nodes:].isfinite().all()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [2, 6, 24, 64])
@pytest.mark.parametrize("ctx,at", [(300, 100), (300, 299), (40, 3), (1, 0), (7000, 6000)])
def test_infinite_and_nan_values_stay_in_their_columns(dt, hd, nodes, ctx, at):
    t, clean = (Tree(54, [ctx, 70], [nodes, 3], 2, 1, hd, dt) for _ in range(2))
    pg, sl = place(t, at)
    for x in (t, clean):  # the key of that place has most of the weight: its weight's second term may be zero
        x.k[pg, sl, 0] = 0.3 * x.q[0, 0]
    t.v[pg, sl, 0, 5], t.v[pg, sl, 0, 7], t.v[pg, sl, 0, hd - 1] = math.inf, -math.inf, math.nan
    if ctx > 1:
        pg2, sl2 = place(t, at - 1)  # both signs in one column
        t.v[pg2, sl2, 0, 9], t.v[pg, sl, 0, 9] = math.inf, -math.inf
    out, ref = t.run().cpu(), clean.run().cpu()
    got = out[:nodes]
    assert (got[..., 5] == math.inf).all() and (got[..., 7] == -math.inf).all() and got[..., hd - 1].isnan().all()
    assert ctx == 1 or got[..., 9].isnan().all()
    cols = [c for c in range(hd) if c not in (5, 7, 9, hd - 1)]
    assert torch.equal(got[..., cols], ref[:nodes][..., cols])
    assert torch.equal(out[nodes:], ref[nodes:])


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n", [4097, 4104, 8193, 8200])
def test_short_segments_of_a_cluster(dt, n):
    """Rows a little longer than one CTA's share: each CTA of a cluster has little to load before it writes its
    maximum into the others' memory.  The largest logit lies in each CTA's segment once."""
    m = 96
    g = torch.Generator().manual_seed(n)
    x = torch.randn(m, n, generator=g)
    at = (torch.arange(m) * n) // m
    x[torch.arange(m), at] = 30.0  # has all the weight that f32 shows
    for _ in range(20):
        idx, prob = px.sample_dev(x.to(dt).cuda(), torch.full((m,), 0.5, device="cuda"))
        assert torch.equal(idx.cpu().long(), at) and (prob > 0.999).all()


# --------------------------------------------------------------------------------------- sampling
def test_weights_next_to_min_p():
    """min_p 1.6 steps of 2^-44 below a token's weight keeps the token.  The weight is exp() rounded to such a
    step, half a step at most, and off by less than 0.05 of one before that (a few u of 64 bits, 2^-54.5 of
    the polynomial); min_p rounds up to a step: below 1.1 steps of the two together."""
    rng = np.random.default_rng(3)
    x = -np.concatenate([(np.arange(1, 200) + f) * math.log(2) / 256 for f in (0.46, 0.49, 0.5, 0.51, 0.54)] + [rng.random(500) * 0.7])
    x = x.astype(np.float32)
    drop = []
    for v in x:
        w = math.exp(float(v))
        idx, _ = px.sample_dev(torch.tensor([[0.0, float(v)]]).cuda(), torch.tensor([1 - 2.0 ** -24], device="cuda"),
                               min_p=w - 1.6 * 2.0 ** -44)
        drop.append(idx)
        idx, _ = px.sample_dev(torch.tensor([[0.0, float(v)]]).cuda(), torch.tensor([1 - 2.0 ** -24], device="cuda"),
                               min_p=w + 1.6 * 2.0 ** -44)
        drop.append(1 - idx)
    assert (torch.cat(drop) == 1).all()


# ----------------------------------------------------------------------------------------- streams
def outputs_on(stream, call):
    """The call's results, made on `stream` without an output of the caller's while the current stream still
    reads memory that it has given back; those reads must see what was there."""
    want = call(None)
    sizes = [w.untyped_storage().nbytes() for w in want]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(2)]
    copies = [torch.empty_like(h) for h in held]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)  # about 0.1 s
    for h, c in zip(held, copies):
        c.copy_(h)
    del held, h
    got = call(stream)
    stream.synchronize()
    torch.cuda.synchronize()
    for c in copies:
        assert (c == 7).all()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_outputs_for_another_stream_are_its_own():
    s = torch.cuda.Stream()
    t = Tree(60, [500, 90], [5, 3], 16, 2, 128, F32)
    a = t.args()
    outputs_on(s, lambda st: (px.tree_attention_dev(*a, max_tree=5, stream=st),))
    x, u = torch.randn(300, 200, device="cuda"), torch.rand(300, device="cuda")
    outputs_on(s, lambda st: px.sample_dev(x, u, stream=st))
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(9, 8 * 64, generator=g).cuda()
    pages, vpages = (torch.zeros(2, 16, 2, 64, device="cuda") for _ in range(2))
    slots = torch.arange(9, dtype=torch.int32, device="cuda")
    outputs_on(s, lambda st: (px.qk_norm_rope_dev(qkv, None, None, 4, 2, 64, k_pages=pages, v_pages=vpages, slots=slots, stream=st),))
    table = torch.zeros(300, 1, dtype=torch.int32, device="cuda")
    ctx, acc = torch.arange(300, dtype=torch.int32, device="cuda") % 9, torch.zeros(300, dtype=torch.int64, device="cuda")
    outputs_on(s, lambda st: (px.kv_compact_dev(pages[None], vpages[None], table, ctx, acc, stream=st),))


# --------------------------------------------------------------------------------------- arguments
def test_numbers_past_32_bits_are_refused_or_mean_what_they_say():
    x, u = torch.tensor([[0.0, 1.0, 2.0]]).cuda(), torch.tensor([0.99], device="cuda")
    keep = px.sample_dev(x, u)[0].tolist()
    assert keep == [0]
    assert px.sample_dev(x, u, top_k=(1 << 32) + 1)[0].tolist() == keep  # more than the row: all of it
    assert px.sample_dev(x, u, top_k=(1 << 31))[0].tolist() == keep
    assert px.sample_dev(x, u, top_k=-(1 << 40) + 1)[0].tolist() == keep
    t = Tree(61, [20], [3], 2, 1, 64, F32)
    for bad in ((1 << 32) + 3, -(1 << 32) + 3):
        with pytest.raises(px.PyxisError):
            t.run(max_tree=bad)
    assert torch.equal(t.run(max_context=1 << 80), t.run())  # a bound that bounds nothing
    with pytest.raises(px.PyxisError):
        t.run(max_context=-(1 << 64) + 5)


def test_outputs_of_products_and_argmax_for_another_stream_are_its_own():
    s = torch.cuda.Stream()
    w = px.Weights.quantize_int8(px.synth_normal_bf16(3, 512 * 256, 0.02), 256)
    x = torch.randn(5, 256, device="cuda")
    outputs_on(s, lambda st: (px.matmul_dev(x, w, 512, 256, stream=st),))
    v = torch.randn(300, 1000, device="cuda")
    outputs_on(s, lambda st: px.argmax_dev(v, stream=st))


# --------------------------------------------------------------------------------- context workspace
class Context:
    def __enter__(self):
        self.handle = C.c_void_p()
        _native.check(_native.lib().pyxis_cuda_init(0, C.byref(self.handle)))
        return self.handle

    def __exit__(self, *_):
        torch.cuda.synchronize()
        _native.check(_native.lib().pyxis_cuda_destroy(self.handle))


def leave_free(nbytes):
    """Takes the GPU's memory but for about nbytes."""
    torch.cuda.empty_cache()
    return torch.empty(torch.cuda.mem_get_info()[0] - nbytes, dtype=torch.uint8, device="cuda")


GB = 1 << 30


def test_the_workspace_grows_into_what_memory_there_is():
    L = _native.lib()
    with Context() as ctx:
        _native.check(L.pyxis_cuda_reserve_workspace(ctx, 2 * GB))
        rest = leave_free(GB)
        # 2.5 GB fit once the old 2 GB are given back, which no captured graph names; 1.5 times the old does not fit beside it
        _native.check(L.pyxis_cuda_reserve_workspace(ctx, 5 * GB // 2))
        free = torch.cuda.mem_get_info()[0]
        assert free < GB
        _native.check(L.pyxis_cuda_reserve_workspace(ctx, GB))  # has it
        assert torch.cuda.mem_get_info()[0] == free
        assert L.pyxis_cuda_reserve_workspace(ctx, 400 * GB) != 0  # an error, and no more than that
        del rest
        torch.cuda.empty_cache()
        _native.check(L.pyxis_cuda_reserve_workspace(ctx, 3 * GB))


def test_a_captured_call_keeps_its_workspace_when_the_context_grows():
    t = Tree(62, [9000], [3], 2, 1, 64, F32)
    want = t.run()
    out = torch.empty_like(want)
    a = t.args()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        px.tree_attention_dev(*a, max_tree=3, out=out)
    L, ctx = _native.lib(), px.get_cuda(0).handle
    _native.check(L.pyxis_cuda_reserve_workspace(ctx, 256 << 20))
    junk = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")  # where a freed workspace might have been
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert (junk == 255).all()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("nodes", [6, 24])
def test_pages_without_a_finite_number_in_long_contexts(dt, nodes):
    """Sequences that fill a CTA each, whose last context page holds nothing finite: no wait runs out while the
    columns are taken from the values."""
    n_seq, ctx, hd, page = 150, 50000, 128, 64
    per = -(-(ctx + nodes) // page)
    k = torch.randn(n_seq * per, page, 1, hd, device="cuda", dtype=dt)
    v = torch.randn(n_seq * per, page, 1, hd, device="cuda", dtype=dt)
    table = torch.arange(n_seq * per, dtype=torch.int32, device="cuda").view(n_seq, per)
    last = table[:, (ctx - 1) // page].long()
    fill = v[last].clone()
    q = torch.randn(n_seq * nodes, 2, hd, device="cuda", dtype=dt)
    start = torch.arange(n_seq + 1, dtype=torch.int32, device="cuda") * nodes
    lens = torch.full((n_seq,), ctx, dtype=torch.int32, device="cuda")

    def run():
        return px.tree_attention_dev(q, k, v, table, lens, start, max_tree=nodes, max_context=ctx)

    v[last] = math.inf
    assert (run() == math.inf).all()
    v[last] = math.nan
    assert run().isnan().all()
    v[last] = fill
    k[last] = math.nan
    assert run().isnan().all()
    k[last] = math.inf  # inf times both signs of q
    assert run().isnan().all()
