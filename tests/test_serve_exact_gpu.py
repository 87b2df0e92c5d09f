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
