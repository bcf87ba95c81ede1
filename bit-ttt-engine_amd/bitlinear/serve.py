"""Serving a batch of sequences (include/bitserve.h): a Q8 KV cache in pages of a
shared pool, its append, its reading back, the attention over it, and the choice of
next tokens.

One-sequence counterparts: KVCacheQ8 and BitLlamaHip (bitlinear/model.py) over
btl_rope_kv_append, btl_attention and btl_greedy_next.  Reference
(imonoonoko/Bit-TTT-Engine, crates/rust_engine/src): layers/kv_cache.rs:14-128,
layers/attention.rs:149-239, model/llama.rs:496-530 (the pick at a temperature).

    cache = PagedKVCacheQ8(n_pages, 64, n_kv_heads, head_dim, "cuda")     # one a layer
    batch = PagedBatch(row_start, pos, pages, rows, max_rows, max_len)    # one a step
    q = paged_rope_append(q, k, v, cache, batch, rope_cos, rope_sin)
    o = paged_attention(q, cache, batch)
    ids, probs = sample(logits, u, temperature=0.8, top_k=50, top_p=0.95)
"""
import ctypes
import functools

import torch

from ._lib import (
    BTL_ERR_ARG, BTL_ERR_DEVICE, BTL_ERR_DTYPE, BTL_ERR_LAYOUT, BTL_ERR_SHAPE, BitLinearError, BtlKvPaged, BtlPagedBatch,
    check, lib,
)
from .layer import _DT, _dtype_code, _on_gpu

# A decoded token's calls take microseconds on the GPU: the checks around them look at
# what is right first and only then for what is wrong.
_current_device = torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _on_its_device(f):
    """The library works on the current device: make it the first argument's."""

    @functools.wraps(f)
    def call(x, *args, **kw):
        dev = x.device
        if dev.type == "cuda" and dev.index != _current_device():
            with torch.cuda.device(dev):
                return f(x, *args, **kw)
        return f(x, *args, **kw)

    return call


def _tensor(t, what, dtype, shape, device):
    """A contiguous tensor on `device` of this dtype and shape (None in the shape: any)."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.is_cuda and t.is_contiguous() \
            and t.device == device:
        return t
    if not torch.is_tensor(t):
        raise BitLinearError(BTL_ERR_ARG, "%s must be a tensor" % what)
    _on_gpu(t, what)
    if t.device != device:
        raise BitLinearError(BTL_ERR_DEVICE, "%s is on %s, not on %s" % (what, t.device, device))
    if t.dtype != dtype:
        raise BitLinearError(BTL_ERR_DTYPE, "%s must be %s, got %s" % (what, dtype, t.dtype))
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        raise BitLinearError(BTL_ERR_SHAPE, "%s must be %s, got %s" % (what, list(shape), list(t.shape)))
    return t


class Scratch:
    """A caller-owned workspace of so many bytes."""

    def __init__(self, nbytes, device):
        self.nbytes = int(nbytes)
        self.buf = torch.empty(max(self.nbytes, 256), dtype=torch.uint8, device=device)
        self.device = self.buf.device
        self._args = self.buf.data_ptr(), self.nbytes

    def args(self):
        return self._args


def _ws_args(ws, device):
    if ws is None:
        return None, 0
    if ws.device != device:
        raise BitLinearError(BTL_ERR_DEVICE, "the workspace is on %s, not on %s" % (ws.device, device))
    return ws.args()


class PagedKVCacheQ8:
    """btl_kv_paged_t: one layer's keys and values, quantised to 8 bits, in n_pages pages
    of page_size tokens that any sequences share.  k [n_pages, n_kv_heads, page_size,
    head_dim] u8; v in blocks of 16 tokens, [n_pages, n_kv_heads, page_size / 16,
    head_dim, 16] u8; k_scale, v_scale [n_pages, n_kv_heads, page_size] f32."""

    def __init__(self, n_pages, page_size, n_kv_heads, head_dim, device="cuda"):
        if page_size < 16 or page_size % 16 or head_dim < 16 or head_dim % 16 or head_dim > 128:
            raise BitLinearError(BTL_ERR_SHAPE, "page_size a multiple of 16, head_dim a multiple of 16 up to 128 "
                                 "(got %d, %d)" % (page_size, head_dim))
        u8 = dict(dtype=torch.uint8, device=device)
        k = torch.zeros((n_pages, n_kv_heads, page_size, head_dim), **u8)
        v = torch.zeros((n_pages, n_kv_heads, page_size // 16, head_dim, 16), **u8)
        ks = torch.zeros((n_pages, n_kv_heads, page_size), dtype=torch.float32, device=device)
        self._hold(k, v, ks, torch.zeros_like(ks))

    @staticmethod
    def of(k, v, k_scale, v_scale):
        """The cache that lies in these tensors."""
        c = PagedKVCacheQ8.__new__(PagedKVCacheQ8)
        c._hold(k, v, k_scale, v_scale)
        return c

    def _hold(self, k, v, k_scale, v_scale):
        if not torch.is_tensor(k) or k.dim() != 4:
            raise BitLinearError(BTL_ERR_SHAPE, "k must be [n_pages, n_kv_heads, page_size, head_dim]")
        n, h, ps, hd = k.shape
        self.device = k.device
        self.k = _tensor(k, "k", torch.uint8, (n, h, ps, hd), k.device)
        self.v = _tensor(v, "v", torch.uint8, (n, h, ps // 16, hd, 16), k.device)
        self.k_scale = _tensor(k_scale, "k_scale", torch.float32, (n, h, ps), k.device)
        self.v_scale = _tensor(v_scale, "v_scale", torch.float32, (n, h, ps), k.device)
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n, h, ps, hd
        self.c = BtlKvPaged(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, h, ps, hd)
        self._ref = ctypes.byref(self.c)


class PagedBatch:
    """btl_paged_batch_t: the sequences of one call.  row_start [n_seqs + 1], pos [n_seqs]
    and pages [n_seqs, max_pages] are int32 tensors on the GPU, read when the kernels
    run; sequence s has the rows row_start[s] .. row_start[s + 1] - 1 of the call's
    `rows`, at positions from pos[s] on.  max_rows and max_len: no sequence has more
    rows, or more tokens with them (default: as many as rows and pages allow)."""

    def __init__(self, row_start, pos, pages, rows, max_rows=None, max_len=None):
        if not torch.is_tensor(pos) or pos.dim() != 1:
            raise BitLinearError(BTL_ERR_SHAPE, "pos must be [n_seqs]")
        n = pos.shape[0]
        self.device = pos.device
        self.pos = _tensor(pos, "pos", torch.int32, (n,), pos.device)
        self.row_start = _tensor(row_start, "row_start", torch.int32, (n + 1,), pos.device)
        self.pages = _tensor(pages, "pages", torch.int32, (n, None), pos.device)
        self.rows = int(rows)
        max_rows = self.rows if max_rows is None else int(max_rows)
        max_len = 1 << 30 if max_len is None else int(max_len)
        self.c = BtlPagedBatch(row_start.data_ptr(), pos.data_ptr(), pages.data_ptr() if pages.numel() else None, n,
                               pages.shape[1], self.rows, max_rows, max_len)
        self._ref = ctypes.byref(self.c)


def _heads(q, cache, batch):
    """q's dtype code, heads and device."""
    if not q.is_cuda or not q.is_contiguous():
        _on_gpu(q, "q")
    shape, device, dt = q.shape, q.device, _DT.get(q.dtype)
    if len(shape) != 2 or shape[0] != batch.rows or shape[1] % cache.head_dim:
        raise BitLinearError(BTL_ERR_SHAPE, "q must be [%d, n_heads * %d], got %s"
                             % (batch.rows, cache.head_dim, list(shape)))
    if cache.device != device or batch.device != device:
        raise BitLinearError(BTL_ERR_DEVICE, "q on %s, cache on %s, batch on %s" % (device, cache.device, batch.device))
    return _dtype_code(q, "q") if dt is None else dt, shape[1] // cache.head_dim, device


@_on_its_device
def paged_rope_append(q, k, v, cache, batch, rope_cos, rope_sin, q_out=None):
    """btl_paged_rope_append: RoPE of the rows q [rows, n_heads * head_dim] and k [rows,
    n_kv * head_dim], k and v quantised into the cache.  Returns the rotated q (q_out,
    which may be q).  rope_cos, rope_sin: float32 [positions, head_dim / 2]."""
    dt, nh, dev = _heads(q, cache, batch)
    kv = (batch.rows, cache.n_kv_heads * cache.head_dim)
    _tensor(k, "k", q.dtype, kv, dev)
    _tensor(v, "v", q.dtype, kv, dev)
    length = rope_cos.shape[0] if rope_cos.dim() == 2 else -1
    _tensor(rope_cos, "rope_cos", torch.float32, (length, cache.head_dim // 2), dev)
    _tensor(rope_sin, "rope_sin", torch.float32, (length, cache.head_dim // 2), dev)
    if q_out is None:
        q_out = torch.empty_like(q)
    else:
        _tensor(q_out, "q_out", q.dtype, q.shape, dev)
    check(lib.btl_paged_rope_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, nh, cache._ref, batch._ref,
                                    rope_cos.data_ptr(), rope_sin.data_ptr(), length, q_out.data_ptr(),
                                    _stream(dev)))
    return q_out


@_on_its_device
def paged_read(cache, batch, dtype=torch.float32, k_out=None, v_out=None):
    """btl_paged_read: the rows' keys and values out of the cache, each [rows, n_kv *
    head_dim] of `dtype` (or of k_out's and v_out's).  Whole contexts are a batch at
    pos = 0 with as many rows as tokens."""
    shape, dev = (batch.rows, cache.n_kv_heads * cache.head_dim), cache.device
    if dev != batch.device:
        raise BitLinearError(BTL_ERR_DEVICE, "cache on %s, batch on %s" % (dev, batch.device))
    first = k_out if k_out is not None else v_out
    dtype = dtype if first is None else first.dtype
    k_out = torch.empty(shape, dtype=dtype, device=cache.device) if k_out is None else k_out
    v_out = torch.empty(shape, dtype=dtype, device=cache.device) if v_out is None else v_out
    _tensor(k_out, "k_out", dtype, shape, dev)
    _tensor(v_out, "v_out", dtype, shape, dev)
    check(lib.btl_paged_read(cache._ref, batch._ref, k_out.data_ptr(), v_out.data_ptr(), _dtype_code(k_out, "output"),
                             _stream(dev)))
    return k_out, v_out


@_on_its_device
def paged_attention(q, cache, batch, out=None, workspace=None):
    """btl_paged_attention: causal attention of the rotated rows q [rows, n_heads *
    head_dim] over their sequences' pages.  Returns out, of q's dtype."""
    dt, nh, dev = _heads(q, cache, batch)
    if out is None:
        out = torch.empty_like(q)
    else:
        _tensor(out, "out", q.dtype, q.shape, dev)
    wsp, wsn = _ws_args(workspace, dev)
    check(lib.btl_paged_attention(q.data_ptr(), dt, nh, cache._ref, batch._ref, out.data_ptr(), wsp, wsn,
                                  _stream(dev)))
    return out


def paged_attention_workspace(cache, batch, n_heads):
    """A workspace for paged_attention calls of this cache's and batch's sizes."""
    return Scratch(lib.btl_paged_attention_workspace_bytes(n_heads, cache._ref, batch._ref), cache.device)


def _per_row(v, what, dtype, rows, device):
    """One value a row: a tensor, a number for all of them, or None."""
    if v is None:
        return None
    if torch.is_tensor(v):
        return _tensor(v, what, dtype, (rows,), device)
    return torch.full((rows,), v, dtype=dtype, device=device)


@_on_its_device
def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, ids=None, probs=None, workspace=None):
    """btl_sample: next tokens of logits [rows, n] float32 (rows may be strided) from
    given random numbers u [rows] in [0, 1).  temperature, top_p, min_p (float32) and
    top_k (int32): tensors [rows], numbers, or None.  Returns (ids int32 [rows], probs
    float32 [rows]: each token's probability among those the filters left)."""
    if not logits.is_cuda:
        _on_gpu(logits, "logits")
    if logits.dtype is not torch.float32:
        raise BitLinearError(BTL_ERR_DTYPE, "logits must be float32, got %s" % logits.dtype)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise BitLinearError(BTL_ERR_LAYOUT, "logits must be [rows, n], each row contiguous")
    rows, n = logits.shape
    dev = logits.device
    f = torch.float32
    ld = logits.stride(0) if rows > 1 else n
    _tensor(u, "u", f, (rows,), dev)
    row = [_per_row(temperature, "temperature", f, rows, dev), _per_row(top_k, "top_k", torch.int32, rows, dev),
           _per_row(top_p, "top_p", f, rows, dev), _per_row(min_p, "min_p", f, rows, dev)]
    ids = torch.empty((rows,), dtype=torch.int32, device=dev) if ids is None \
        else _tensor(ids, "ids", torch.int32, (rows,), dev)
    probs = torch.empty((rows,), dtype=f, device=dev) if probs is None else _tensor(probs, "probs", f, (rows,), dev)
    wsp, wsn = _ws_args(workspace, dev)
    check(lib.btl_sample(logits.data_ptr(), rows, n, ld, *[None if t is None else t.data_ptr() for t in row],
                         u.data_ptr(), ids.data_ptr(), probs.data_ptr(), wsp, wsn, _stream(dev)))
    return ids, probs


def sample_workspace(rows, n, device="cuda"):
    """A workspace for sample calls of up to these sizes."""
    return Scratch(lib.btl_sample_workspace_bytes(rows, n), device)
