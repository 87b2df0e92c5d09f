"""The serving operators (include/pyxis_serve.h) without a GPU: argument checks, which come before the
context is looked at, the rotary frequencies, and the page bookkeeping."""
import ctypes as C
import math
import random

import numpy as np
import pytest

import pyxis_b200 as px
from pyxis_b200 import _native, serve

EINVAL = _native.PYXIS_EINVAL
A = 1 << 20  # an address that is never read: every check below fails before any launch


def pages(**kw):
    d = dict(k=A, v=2 * A, dtype=1, n_layers=2, num_pages=8, page_size=16, n_kv_heads=2, head_dim=128,
             layer_stride=8 * 16 * 256, page_stride=16 * 256, slot_stride=256, head_stride=128)
    d.update(kw)
    return serve._Pages(*[d[n] for n, _ in serve._Pages._fields_])


def rope_args(**kw):
    d = dict(qkv=A, q=8 * A, n_tokens=3, ld_qkv=1024, ld_q=512, positions=A, slots=A, inv_freq=A, q_norm=A, k_norm=A,
             n_q_heads=4, rotary_dim=128, interleaved=0, eps=1e-6, rope_scale=1.0)
    d.update(kw)
    return serve._RopeArgs(*[d[n] for n, _ in serve._RopeArgs._fields_])


def tree_args(**kw):
    d = dict(q=A, out=8 * A, q_row=512, q_head=128, out_row=512, out_head=128, n_rows=4, n_seq=2, q_start=A, context_len=A,
             block_table=A, tree_mask=A, table_stride=4, table_width=4, n_q_heads=4, max_tree=2, max_context=10, scale=0.1)
    d.update(kw)
    return serve._TreeArgs(*[d[n] for n, _ in serve._TreeArgs._fields_])


def refused(rc, text):
    assert rc == EINVAL
    assert text in _native.lib().pyxis_cuda_last_error().decode()


BAD_PAGES = [(dict(k=None), "null cache"), (dict(dtype=3), "dtype"), (dict(head_dim=96), "head_dim"),
             (dict(num_pages=0), "pages"), (dict(page_size=-1), "pages"), (dict(n_kv_heads=0), "heads"),
             (dict(num_pages=1 << 27, page_size=16), "2^31"), (dict(v=A + 8), "aligned"), (dict(slot_stride=254), "slot stride"),
             (dict(head_stride=64), "head stride"), (dict(page_stride=0), "page stride"), (dict(dtype=2, slot_stride=260), "slot stride")]


@pytest.mark.parametrize("kw,text", BAD_PAGES)
def test_bad_pages_are_refused_everywhere(kw, text):
    L, kv = _native.lib(), pages(**kw)
    refused(L.pyxis_cuda_qk_norm_rope_dev(None, C.byref(rope_args()), C.byref(kv), None), text)
    refused(L.pyxis_cuda_tree_attention_dev(None, C.byref(tree_args()), C.byref(kv), None, 0, None), text)
    refused(L.pyxis_cuda_kv_copy_pages_dev(None, C.byref(kv), A, A, 1, None), text)
    refused(L.pyxis_cuda_kv_compact_dev(None, C.byref(kv), A, 4, 4, A, A, 2, 2 * A, None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(qkv=None), "null qkv"), (dict(slots=None), "null qkv"), (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=144), "rotary_dim"),
    (dict(positions=None), "positions"), (dict(inv_freq=None), "positions"), (dict(ld_qkv=1020), "rows of qkv"),
    (dict(ld_qkv=1026), "rows of qkv"), (dict(ld_q=508), "rows of qkv"), (dict(qkv=A + 4), "aligned"), (dict(q=A + 512 * 4), "overlaps"),
    (dict(q=A), "overlaps"), (dict(n_q_heads=0), "query heads"), (dict(n_tokens=1 << 31), "too many")])
def test_rope_arguments(kw, text):
    refused(_native.lib().pyxis_cuda_qk_norm_rope_dev(None, C.byref(rope_args(**kw)), C.byref(pages()), None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(n_q_heads=3), "query heads"), (dict(max_tree=0), "max_tree"), (dict(max_tree=65), "max_tree"), (dict(max_context=-1), "max_context"),
    (dict(table_stride=3), "block table"), (dict(q=None), "null q"), (dict(q_start=None), "null q"), (dict(block_table=None), "null q"),
    (dict(out_head=64), "strides"), (dict(out=A), "overlaps"), (dict(out=A + 2), "aligned"), (dict(n_rows=1 << 31), "too many")])
def test_tree_arguments(kw, text):
    refused(_native.lib().pyxis_cuda_tree_attention_dev(None, C.byref(tree_args(**kw)), C.byref(pages()), None, 0, None), text)


def test_more_rows_than_a_grid_holds_are_refused():
    args = tree_args(max_tree=64, n_q_heads=1024, q_row=1 << 17, out_row=1 << 17)
    refused(_native.lib().pyxis_cuda_tree_attention_dev(None, C.byref(args), C.byref(pages()), None, 0, None), "too many query heads")


def test_page_operator_arguments():
    L, kv = _native.lib(), C.byref(pages())
    refused(L.pyxis_cuda_kv_copy_pages_dev(None, kv, None, A, 1, None), "null src")
    refused(L.pyxis_cuda_kv_compact_dev(None, kv, A, 4, 4, A, None, 2, 2 * A, None), "null block_table")
    refused(L.pyxis_cuda_kv_compact_dev(None, kv, A, 3, 4, A, A, 2, 2 * A, None), "block table")
    refused(L.pyxis_cuda_kv_compact_dev(None, kv, A, 4, 4, A, A, 2, A + 4, None), "overlaps")
    refused(L.pyxis_cuda_kv_compact_dev(None, kv, A, 4, 4, A, A, 65536, 2 * A, None), "65535")


def test_sample_arguments():
    L, p = _native.lib(), serve._SampleParams(None, None, None, None, 1.0, 0, 1.0, 0.0)
    call = lambda x=A, t=1, M=2, n=10, ld=10, u=A, params=C.byref(p), idx=A: L.pyxis_cuda_sample_dev(  # noqa: E731
        None, x, t, M, n, ld, u, params, idx, None, None)
    refused(call(params=None), "null params")
    refused(call(t=4), "dtype")
    refused(call(n=0), "empty row")
    refused(call(n=1 << 31, ld=1 << 31), "too long")
    refused(call(M=65536), "65535")
    refused(call(ld=9), "stride")
    refused(call(x=None), "null logits")
    refused(call(u=None), "null logits")
    refused(call(x=A + 2), "aligned")
    refused(call(), "null context")  # all else in order


def test_nothing_to_do_is_no_error():
    L, kv = _native.lib(), C.byref(pages())
    assert L.pyxis_cuda_qk_norm_rope_dev(None, C.byref(rope_args(n_tokens=0)), kv, None) == 0
    assert L.pyxis_cuda_tree_attention_dev(None, C.byref(tree_args(n_seq=0)), kv, None, 0, None) == 0
    assert L.pyxis_cuda_kv_copy_pages_dev(None, kv, None, None, 0, None) == 0
    assert L.pyxis_cuda_kv_compact_dev(None, kv, None, 0, 0, None, None, 0, None, None) == 0


# ---------------------------------------------------------------------------------- frequencies
@pytest.mark.parametrize("rot,theta", [(2, 1e4), (64, 1e4), (128, 1e6)])
def test_plain_and_linear_frequencies(rot, theta):
    f, m = px.rope_frequencies(rot, theta)
    want = theta ** (-np.arange(0, rot, 2) / rot)
    np.testing.assert_allclose(f, want, rtol=1e-15 * 4)
    assert m == 1.0
    g, m = px.rope_frequencies(rot, theta, "linear", factor=4.0)
    np.testing.assert_allclose(g, want / 4, rtol=1e-15 * 4)
    assert m == 1.0


def test_ntk_stretches_the_lowest_frequency_by_the_factor():
    f, _ = px.rope_frequencies(64, 1e4)
    g, m = px.rope_frequencies(64, 1e4, "ntk", factor=8.0)
    assert g[0] == 1.0 and m == 1.0
    assert g[-1] == pytest.approx(f[-1] / 8.0, rel=1e-12)


def test_yarn_keeps_fast_and_divides_slow_frequencies():
    f, _ = px.rope_frequencies(128, 1e6)
    g, m = px.rope_frequencies(128, 1e6, "yarn", factor=4.0, original_context=32768)
    assert m == pytest.approx(0.1 * math.log(4.0) + 1.0, rel=1e-15)
    turns = 32768 * f / (2 * math.pi)
    fast, slow = turns > 32 * 2, turns < 0.5  # well outside the ramp
    assert fast.any() and slow.any()
    np.testing.assert_array_equal(g[fast], f[fast])
    np.testing.assert_allclose(g[slow], f[slow] / 4, rtol=1e-14)
    assert np.all(g <= f) and np.all(g >= f / 4 * (1 - 1e-14)) and np.all(np.diff(g) < 0)


@pytest.mark.parametrize("args,kw", [((3, 1e4), {}), ((0, 1e4), {}), ((64, -1.0), {}), ((64, 1e4), dict(kind="linear", factor=0.5)),
                                     ((2, 1e4), dict(kind="ntk", factor=2.0)), ((64, 1e4), dict(kind="yarn", factor=2.0)),
                                     ((64, 1e4), dict(kind="yarn", factor=2.0, original_context=100.0, beta_fast=1.0, beta_slow=1.0)),
                                     ((64, 1e4), dict(kind="other")), ((64, float("nan")), {})])
def test_frequency_refusals(args, kw):
    with pytest.raises(px.PyxisError) as e:
        px.rope_frequencies(*args, **kw)
    assert e.value.code == EINVAL


# ------------------------------------------------------------------------------------- page pool
def test_pool_shares_full_pages_and_copies_the_partial_one():
    pool = px.PagePool(8, 16)
    t = pool.allocate(40)
    assert len(t) == 3 and pool.available == 5
    child, src, dst = pool.fork(t, 40)
    assert child[:2] == t[:2] and src == [t[2]] and dst == [child[2]] and child[2] not in t and pool.available == 4
    at_edge, src, dst = pool.fork(t, 32)
    assert at_edge == t[:2] and src == [] and dst == [] and pool.available == 4
    pool.free(t)
    assert pool.available == 5  # only the third page was its own
    pool.free(child)
    pool.free(at_edge)
    assert pool.available == 8 and t == [] and child == []


def test_pool_refuses_without_taking_pages():
    pool = px.PagePool(4, 16)
    t = pool.allocate(33)
    with pytest.raises(px.PyxisError) as e:
        pool.allocate(17)
    assert e.value.code == _native.PYXIS_ENOMEM and pool.available == 1
    with pytest.raises(px.PyxisError):
        pool.grow(t, 100)
    assert pool.available == 1 and len(t) == 3
    pool.grow(t, 60)
    assert len(t) == 4 and pool.available == 0
    with pytest.raises(px.PyxisError):
        pool.fork(t, 65)
    with pytest.raises(px.PyxisError):
        pool.fork(t, 63)  # its partial page needs a free one
    pool.shrink(t, 16)
    assert len(t) == 1 and pool.available == 3
    twice = list(t)
    pool.free(t)
    with pytest.raises(px.PyxisError):
        pool.free(twice)
    assert pool.available == 4


def test_pool_refuses_bad_tables_without_giving_pages_back():
    pool = px.PagePool(4, 16)
    t = pool.allocate(48)
    free = (set(range(4)) - set(t)).pop()
    for bad in (t + [free], t + [t[0]], [t[0], -1], [t[0], 4]):
        with pytest.raises(px.PyxisError):
            pool.free(list(bad))
        assert pool.available == 1
    pool.free(t)
    assert pool.available == 4


def test_pool_refuses_to_cut_into_a_shared_page():
    pool = px.PagePool(4, 16)
    t = pool.allocate(32)
    child, _, _ = pool.fork(t, 32)
    with pytest.raises(px.PyxisError):
        pool.shrink(child, 20)
    pool.shrink(child, 16)  # whole pages go back
    assert len(child) == 1


def test_pool_random_walk_never_hands_out_a_page_twice():
    rng, pool, tables = random.Random(5), px.PagePool(64, 4), []
    for _ in range(3000):
        what = rng.random()
        try:
            if what < 0.3 or not tables:
                tables.append((pool.allocate(rng.randint(0, 40)), 0))
            elif what < 0.5:
                i = rng.randrange(len(tables))
                t, _ = tables[i]
                tables.append((pool.fork(t, rng.randint(0, len(t) * 4))[0], 0))
            elif what < 0.7:
                pool.grow(rng.choice(tables)[0], rng.randint(0, 60))
            else:
                pool.free(tables.pop(rng.randrange(len(tables)))[0])
        except px.PyxisError as e:
            assert e.code == _native.PYXIS_ENOMEM
        named = set(p for t, _ in tables for p in t)
        assert len(named) + pool.available == 64
        assert all(len(set(t)) == len(t) for t, _ in tables)
