"""Operators of a decoding step that verifies drafted tokens over a paged KV cache
(include/pyxis_serve.h), over torch CUDA tensors:

  qk_norm_rope_dev     QK-RMSNorm, rotary positions and the append to the cache's pages in one pass
                       over the q|k|v rows (src/attention.rs:81-100, :144-162)
  tree_attention_dev   attention of a tree of drafted tokens per sequence over the pages
                       (src/attention.rs:107-135); a tree of one node is a plain decode step
  sample_dev           temperature, top-k, top-p and min-p from given uniform numbers
                       (src/sampler.rs:23-110)
  kv_copy_pages_dev    pages copied in all layers (forks)
  kv_compact_dev       the accepted branch of each tree moved to the front of its drafts
  PagePool             which pages are free and how many tables share each (host side)

Pages are two tensors of one shape and layout, ``[..., num_pages, page_size, n_kv_heads, head_dim]``
with any strides whose last is 1, float32 or bfloat16; the page operators take a leading axis of
layers.  Calls are asynchronous on ``stream`` (default: torch's current stream of the tensors'
device) and raise PyxisError on bad arguments.  Where a ``stream`` is given, it has to come after
the work that makes the inputs, and outputs that the call makes itself belong to that stream: use
them there, or elsewhere after waiting for it (and ``record_stream``).

The attention's kernels never wait without a limit: where a wait runs out, the launch ends with its
outputs partly unwritten and sets the context's error flag, which ``get_cuda(device).check_device_error()``
reads (it waits for the device: once per some steps, not per call).
"""
from __future__ import annotations

import ctypes as C
from operator import index as _index

import numpy as np

from . import CUDA_STREAM_LEGACY, _native, _require_cuda
from ._native import DTYPE_BF16, DTYPE_F32, PYXIS_EINVAL, PyxisError, check

_vp, _sz, _i64 = C.c_void_p, C.c_size_t, C.c_int64


class _Pages(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("dtype", C.c_int), ("n_layers", C.c_int), ("num_pages", C.c_int),
                ("page_size", C.c_int), ("n_kv_heads", C.c_int), ("head_dim", C.c_int), ("layer_stride", _i64),
                ("page_stride", _i64), ("slot_stride", _i64), ("head_stride", _i64)]


class _RopeArgs(C.Structure):
    _fields_ = [("qkv", _vp), ("q", _vp), ("n_tokens", _sz), ("ld_qkv", _sz), ("ld_q", _sz), ("positions", _vp),
                ("slots", _vp), ("inv_freq", _vp), ("q_norm", _vp), ("k_norm", _vp), ("n_q_heads", C.c_int),
                ("rotary_dim", C.c_int), ("interleaved", C.c_int), ("eps", C.c_float), ("rope_scale", C.c_float)]


class _TreeArgs(C.Structure):
    _fields_ = [("q", _vp), ("out", _vp), ("q_row", _i64), ("q_head", _i64), ("out_row", _i64), ("out_head", _i64),
                ("n_rows", _sz), ("n_seq", _sz), ("q_start", _vp), ("context_len", _vp), ("block_table", _vp),
                ("tree_mask", _vp), ("table_stride", _sz), ("table_width", _sz), ("n_q_heads", C.c_int),
                ("max_tree", C.c_int), ("max_context", _i64), ("scale", C.c_float)]


class _SampleParams(C.Structure):
    _fields_ = [("temperature", _vp), ("top_k", _vp), ("top_p", _vp), ("min_p", _vp), ("temperature_all", C.c_double),
                ("top_k_all", C.c_int32), ("top_p_all", C.c_double), ("min_p_all", C.c_double)]


def _fail(msg: str):
    raise PyxisError(PYXIS_EINVAL, msg)


def _int32(value, what: str) -> int:
    value = _index(value)
    if not -(1 << 31) <= value < 1 << 31:
        _fail(f"{what} {value} is out of range")
    return value


class _Torch:
    """What the calls use of torch and of the library, looked up once: a call is a few microseconds,
    and the kernels of a small step are no longer."""

    def __init__(self):
        import torch
        self.Tensor = torch.Tensor
        self.f32, self.f64, self.i32, self.i64 = torch.float32, torch.float64, torch.int32, torch.int64
        self.masks = (torch.int64, torch.uint64)
        self.types = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16}
        self.on_stream = torch.cuda.stream
        self.contexts: dict = {}
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.raw_stream = raw or (lambda device: torch.cuda.current_stream(device).cuda_stream)
        L = _native.lib()
        self.rope, self.tree = L.pyxis_cuda_qk_norm_rope_dev, L.pyxis_cuda_tree_attention_dev
        self.copy, self.compact, self.sample = (L.pyxis_cuda_kv_copy_pages_dev, L.pyxis_cuda_kv_compact_dev,
                                                L.pyxis_cuda_sample_dev)


_torch = None


def _begin(t):
    """(what the calls use, the tensor's device, its context) of a CUDA tensor."""
    global _torch
    if _torch is None:
        _torch = _Torch()
    d = t.get_device()
    if d < 0:
        _fail(f"a CUDA tensor is needed, not one on {t.device}")
    ctx = _torch.contexts.get(d)
    if ctx is None:
        ctx = _torch.contexts[d] = _require_cuda(d)
    return _torch, d, ctx.handle


def _stream(stream, device: int) -> int:
    # torch's default stream is 0, which the library reads as its own: name the legacy stream instead
    return (_torch.raw_stream(device) if stream is None else stream.cuda_stream) or CUDA_STREAM_LEGACY


def _empty(like, shape, dtype, stream):
    """An output of the call, from the memory of the stream that writes it."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch.on_stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _array(t, what: str, dtype, n: int, device: int) -> int:
    """Address of a contiguous device array of at least n elements."""
    if t.get_device() != device:
        _fail(f"{what} must be on cuda:{device}")
    if t.dtype is not dtype and (dtype is not _torch.i64 or t.dtype not in _torch.masks):
        _fail(f"{what} must be {dtype}, not {t.dtype}")
    if t.numel() < n or not t.is_contiguous():
        _fail(f"{what} must hold {n} contiguous elements")
    return t.data_ptr()


def _table(t, what: str, device: int):
    if t.dim() != 2 or t.stride(1) != 1 or t.dtype is not _torch.i32 or t.get_device() != device:
        _fail(f"{what} must be int32 [sequences, pages] with contiguous rows on cuda:{device}")
    return t.shape


def _pages(k, v, device: int, layers: bool) -> _Pages:
    n, s = k.shape, k.stride()
    if len(n) != (5 if layers else 4) or n != v.shape or s != v.stride() or k.dtype is not v.dtype:
        _fail(f"k_pages and v_pages must be {5 if layers else 4}-dimensional tensors of one shape, layout and type")
    if k.get_device() != device or v.get_device() != device:
        _fail(f"cache pages must be on cuda:{device}")
    kind = _torch.types.get(k.dtype)
    if kind is None or s[-1] != 1:
        _fail(f"cache pages of {k.dtype}: float32 or bfloat16 with contiguous heads are needed")
    if layers:
        return _Pages(k.data_ptr(), v.data_ptr(), kind, n[0], n[1], n[2], n[3], n[4], s[0], s[1], s[2], s[3])
    return _Pages(k.data_ptr(), v.data_ptr(), kind, 1, n[0], n[1], n[2], n[3], 0, s[0], s[1], s[2])


ROPE_KINDS = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3}


def rope_frequencies(rotary_dim: int, theta: float, kind: str = "plain", factor: float = 1.0,
                     original_context: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(frequencies [rotary_dim / 2] float64, scale of cos and sin) on the host
    (pyxis_rope_frequencies): kind "plain", "linear", "ntk" or "yarn"."""
    if kind not in ROPE_KINDS:
        _fail(f"unknown frequency scaling {kind!r}")
    if _int32(rotary_dim, "rotary_dim") <= 0:
        _fail(f"rotary_dim {rotary_dim} is not even and positive")
    freq = np.empty(rotary_dim // 2, np.float64)
    scale = C.c_double()
    check(_native.lib().pyxis_rope_frequencies(ROPE_KINDS[kind], theta, rotary_dim, factor, original_context, beta_fast,
                                               beta_slow, freq.ctypes.data_as(_vp), C.addressof(scale)))
    return freq, scale.value


def qk_norm_rope_dev(qkv, positions, inv_freq, n_q_heads: int, n_kv_heads: int, head_dim: int, *, k_pages, v_pages, slots,
                     q_norm=None, k_norm=None, eps: float = 1e-6, interleaved: bool = False, rope_scale: float = 1.0,
                     q=None, stream=None):
    """Normalises and rotates the heads of ``qkv`` [tokens, (n_q + 2 n_kv) * head_dim], puts keys and
    values into ``k_pages`` / ``v_pages`` [pages, page_size, n_kv, head_dim] at ``slots`` (int32; page
    * page_size + place, -1: none) and returns the queries [tokens, n_q, head_dim]
    (pyxis_cuda_qk_norm_rope_dev).  ``positions`` int32 [tokens]; ``inv_freq`` float64 [rotary_dim / 2]
    on the device, or None for no rotation; ``q_norm`` / ``k_norm`` float32 [head_dim] or None;
    ``q``: a [tokens, n_q, head_dim] tensor with contiguous heads to write, ``qkv``'s own rows
    included."""
    T, dev, ctx = _begin(qkv)
    shape, ld, dtype = qkv.shape, qkv.stride(), qkv.dtype
    if len(shape) != 2 or shape[1] != (n_q_heads + 2 * n_kv_heads) * head_dim or ld[1] != 1:
        _fail("qkv must be [tokens, (n_q + 2 n_kv) * head_dim] with contiguous rows")
    n = shape[0]
    kv = _pages(k_pages, v_pages, dev, False)
    if kv.n_kv_heads != n_kv_heads or kv.head_dim != head_dim or k_pages.dtype is not dtype:
        _fail("the cache's heads or type differ from qkv's")
    if q is None:
        q = _empty(qkv, (n, n_q_heads, head_dim), dtype, stream)
        ld_q = n_q_heads * head_dim
    else:
        if q.shape != (n, n_q_heads, head_dim) or q.dtype is not dtype or q.get_device() != dev or q.stride(2) != 1 or (
                n_q_heads > 1 and q.stride(1) != head_dim):
            _fail("q must be [tokens, n_q, head_dim] of qkv's type and device with contiguous heads")
        ld_q = q.stride(0)
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    a = _RopeArgs(qkv.data_ptr(), q.data_ptr(), n, ld[0], ld_q, _array(positions, "positions", T.i32, n, dev) if rot else None,
                  _array(slots, "slots", T.i32, n, dev), _array(inv_freq, "inv_freq", T.f64, rot // 2, dev) if rot else None,
                  None if q_norm is None else _array(q_norm, "q_norm", T.f32, head_dim, dev),
                  None if k_norm is None else _array(k_norm, "k_norm", T.f32, head_dim, dev),
                  n_q_heads, rot, 1 if interleaved else 0, eps, rope_scale)
    rc = T.rope(ctx, C.byref(a), C.byref(kv), _stream(stream, dev))
    if rc:
        check(rc)
    return q


def tree_attention_dev(q, k_pages, v_pages, block_table, context_len, q_start, tree_mask=None, *, max_tree: int,
                       max_context: int | None = None, scale: float | None = None, out=None, workspace=None, stream=None):
    """Attention of ``q`` [rows, n_q, head_dim] over the pages (pyxis_cuda_tree_attention_dev):
    sequence s owns rows ``q_start[s]`` .. ``q_start[s + 1] - 1`` (at most ``max_tree`` <= 64), whose
    row j sees positions below ``context_len[s]`` and the drafts i with bit i of ``tree_mask`` (int64
    or uint64 [rows]; None: drafts 0 .. j) at positions ``context_len[s]`` + i of the pages in
    ``block_table`` [sequences, width].  ``max_context`` bounds the contexts, for the split of the work
    (default: what the table holds); ``scale`` defaults to 1 / sqrt(head_dim).  Rows outside every
    sequence are left as they are (in a new ``out``: uninitialised).  Partial sums lie in the device
    context's memory, so calls without a ``workspace`` must not overlap on the GPU; a call that may
    overlap others brings its own (256-byte aligned; one too small is refused with the size needed)."""
    T, dev, ctx = _begin(q)
    kv = _pages(k_pages, v_pages, dev, False)
    shape, s, dtype = q.shape, q.stride(), q.dtype
    if len(shape) != 3 or shape[2] != kv.head_dim or s[2] != 1 or dtype is not k_pages.dtype:
        _fail("q must be [rows, n_q, head_dim] of the cache's type")
    rows, n_q, hd = shape
    if out is None:
        out = _empty(q, (rows, n_q, hd), dtype, stream)
    elif out.shape != shape or out.dtype is not dtype or out.get_device() != dev or out.stride(2) != 1:
        _fail("out must have q's shape, type and device")
    o = out.stride()
    n_seq, width = _table(block_table, "block_table", dev)
    a = _TreeArgs(q.data_ptr(), out.data_ptr(), s[0], s[1], o[0], o[1], rows, n_seq,
                  _array(q_start, "q_start", T.i32, n_seq + 1, dev), _array(context_len, "context_len", T.i32, n_seq, dev),
                  block_table.data_ptr(), None if tree_mask is None else _array(tree_mask, "tree_mask", T.i64, rows, dev),
                  block_table.stride(0), width, n_q, _int32(max_tree, "max_tree"),
                  width * kv.page_size if max_context is None else max(-1, min(_index(max_context), (1 << 62))),
                  hd ** -0.5 if scale is None else scale)
    if workspace is None:
        rc = T.tree(ctx, C.byref(a), C.byref(kv), None, 0, _stream(stream, dev))
    else:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            _fail(f"the workspace must be contiguous on cuda:{dev}")
        rc = T.tree(ctx, C.byref(a), C.byref(kv), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                    _stream(stream, dev))
    if rc:
        check(rc)
    return out


def kv_copy_pages_dev(k_pages, v_pages, src, dst, stream=None) -> None:
    """Copies pages ``src[i]`` to ``dst[i]`` (int32) of ``k_pages`` / ``v_pages`` [layers, pages,
    page_size, n_kv, head_dim] in every layer (pyxis_cuda_kv_copy_pages_dev)."""
    T, dev, ctx = _begin(k_pages)
    kv = _pages(k_pages, v_pages, dev, True)
    n = src.numel()
    if dst.numel() != n:
        _fail("src and dst differ in length")
    rc = T.copy(ctx, C.byref(kv), _array(src, "src", T.i32, n, dev), _array(dst, "dst", T.i32, n, dev), n, _stream(stream, dev))
    if rc:
        check(rc)


def kv_compact_dev(k_pages, v_pages, block_table, context_len, accepted, new_len=None, stream=None):
    """Moves the cache entries of each sequence's ``accepted`` nodes (bits, int64 or uint64
    [sequences]) to positions ``context_len[s]``, ``context_len[s]`` + 1, ... in every layer and
    returns ``new_len`` int32 [sequences] = context_len + their number (pyxis_cuda_kv_compact_dev)."""
    T, dev, ctx = _begin(k_pages)
    kv = _pages(k_pages, v_pages, dev, True)
    n_seq, width = _table(block_table, "block_table", dev)
    if new_len is None:
        new_len = _empty(context_len, (n_seq,), T.i32, stream)
    rc = T.compact(ctx, C.byref(kv), block_table.data_ptr(), block_table.stride(0), width,
                   _array(context_len, "context_len", T.i32, n_seq, dev), _array(accepted, "accepted", T.i64, n_seq, dev), n_seq,
                   _array(new_len, "new_len", T.i32, n_seq, dev), _stream(stream, dev))
    if rc:
        check(rc)
    return new_len


def sample_dev(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, idx=None, prob=None, stream=None):
    """One token per row of ``logits`` [M, n] (float32 or bfloat16) from ``uniforms`` float32 [M] in
    [0, 1) (pyxis_cuda_sample_dev).  Each parameter is a number for all rows or a device tensor [M]
    (float32; ``top_k`` int32).  Temperature 0 is the greedy choice.  Returns (idx int32 [M],
    prob float32 [M]: the token's share of the kept weights)."""
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
    T, dev, ctx = _begin(logits)
    M, n = logits.shape
    kind = T.types.get(logits.dtype)
    if kind is None or (n > 1 and logits.stride(1) != 1):
        _fail(f"logits of {logits.dtype}: float32 or bfloat16 with contiguous rows are needed")

    def per_row(value, what, dtype):
        return _array(value, what, dtype, M, dev) if isinstance(value, T.Tensor) else None

    t, k, p, m = (per_row(temperature, "temperature", T.f32), per_row(top_k, "top_k", T.i32), per_row(top_p, "top_p", T.f32),
                  per_row(min_p, "min_p", T.f32))
    params = _SampleParams(t, k, p, m, temperature if t is None else 1.0,
                           max(0, min(_index(top_k), n)) if k is None else 0, top_p if p is None else 1.0,
                           min_p if m is None else 0.0)
    if idx is None:
        idx = _empty(logits, (M,), T.i32, stream)
    if prob is None:
        prob = _empty(logits, (M,), T.f32, stream)
    rc = T.sample(ctx, logits.data_ptr(), kind, M, n, logits.stride(0), _array(uniforms, "uniforms", T.f32, M, dev), C.byref(params),
                  _array(idx, "idx", T.i32, M, dev), _array(prob, "prob", T.f32, M, dev), _stream(stream, dev))
    if rc:
        check(rc)
    return idx, prob


class PagePool:
    """Host-side bookkeeping of a cache's pages: the block tables of sequences over ``num_pages`` pages
    of ``page_size`` slots, each page counted by the tables that name it.

        table = pool.allocate(tokens)          pages for a new sequence
        pool.grow(table, tokens)               more of them, in place
        child, src, dst = pool.fork(table, n)  a table sharing the full pages of the first n tokens; the
                                               partly filled one is copied: kv_copy_pages_dev(.., src, dst)
        pool.shrink(table, tokens)             gives back the pages past the first ``tokens`` slots
        pool.free(table)

    Raises PyxisError (PYXIS_ENOMEM) when too few pages are free, without taking any."""

    def __init__(self, num_pages: int, page_size: int):
        if num_pages <= 0 or page_size <= 0:
            _fail(f"{num_pages} pages of {page_size} slots")
        self.num_pages, self.page_size = num_pages, page_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._uses = [0] * num_pages

    @property
    def available(self) -> int:
        return len(self._free)

    def _pages_for(self, tokens: int) -> int:
        if tokens < 0:
            _fail(f"{tokens} tokens")
        return -(-tokens // self.page_size)

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise PyxisError(_native.PYXIS_ENOMEM, f"{n} pages needed, {len(self._free)} free")
        got = [self._free.pop() for _ in range(n)]
        for p in got:
            self._uses[p] = 1
        return got

    def _check(self, pages) -> None:
        if len(set(pages)) < len(pages):
            _fail("a page stands twice in a table")
        for p in pages:
            if not 0 <= p < self.num_pages or self._uses[p] <= 0:
                _fail(f"page {p} is free already" if 0 <= p < self.num_pages else f"no page {p}")

    def _drop(self, pages) -> None:
        self._check(pages)  # (all checks first: a refusal leaves the pool as it was)
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                self._free.append(p)

    def allocate(self, tokens: int) -> list[int]:
        return self._take(self._pages_for(tokens))

    def grow(self, table: list[int], tokens: int) -> None:
        table.extend(self._take(max(0, self._pages_for(tokens) - len(table))))

    def shrink(self, table: list[int], tokens: int) -> None:
        keep = self._pages_for(tokens)
        if tokens % self.page_size and keep <= len(table) and self._uses[table[keep - 1]] > 1:
            _fail(f"page {table[keep - 1]} is shared and would be written again: fork at {tokens} tokens instead")
        self._drop(table[keep:])
        del table[keep:]

    def free(self, table: list[int]) -> None:
        self._drop(table)
        table.clear()

    def fork(self, table: list[int], tokens: int) -> tuple[list[int], list[int], list[int]]:
        if self._pages_for(tokens) > len(table):
            _fail(f"a fork at {tokens} tokens of a table of {len(table)} pages")
        self._check(table)
        full = tokens // self.page_size
        new = self._take(self._pages_for(tokens) - full)
        for p in table[:full]:
            self._uses[p] += 1
        return table[:full] + new, table[full : full + len(new)], list(new)
