"""CPU tests of the batched serving ops (include/bitserve.h): argument checks before any
device work, workspace sizes, and the plain implementations that the GPU tests use."""
import ctypes
import math

import numpy as np
import pytest
import torch

import bitlinear as bl
import serve_ref as ref

A = 4096  # an address, never read


def cache(**change):
    c = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=10, n_kv_heads=2, page_size=16, head_dim=64)
    c.update(change)
    return bl.BtlKvPaged(*c.values())


def batch(**change):
    b = dict(row_start=A, pos=A, pages=A, n_seqs=3, max_pages=4, rows=5, max_rows=2, max_len=50)
    b.update(change)
    return bl.BtlPagedBatch(*b.values())


def append(c=None, b=None, q=A, k=2 * A, v=3 * A, dt=0, nh=4, cos=A, sin=A, length=64, out=16 * A):
    c, b = c or cache(), b or batch()
    return bl.lib.btl_paged_rope_append(q, k, v, dt, nh, ctypes.byref(c), ctypes.byref(b), cos, sin, length, out, None)


def read(c=None, b=None, k=A, v=4 * A, dt=0):
    c, b = c or cache(), b or batch()
    return bl.lib.btl_paged_read(ctypes.byref(c), ctypes.byref(b), k, v, dt, None)


def attention(c=None, b=None, q=A, out=16 * A, dt=0, nh=4, ws=None, wsn=0):
    c, b = c or cache(), b or batch()
    return bl.lib.btl_paged_attention(q, dt, nh, ctypes.byref(c), ctypes.byref(b), out, ws, wsn, None)


CALLS = [append, read, attention]


@pytest.mark.parametrize("call", CALLS)
def test_cache_and_batch_are_checked(call):
    for bad in (dict(n_pages=0), dict(n_kv_heads=0), dict(page_size=0), dict(page_size=8), dict(page_size=24),
                dict(page_size=1 << 17), dict(head_dim=0), dict(head_dim=8), dict(head_dim=72), dict(head_dim=144),
                dict(n_pages=1 << 29)):
        assert call(c=cache(**bad)) == bl.BTL_ERR_SHAPE, bad
        assert bl.lib.btl_last_error() != b""
    for bad in (dict(n_seqs=-1), dict(rows=-1), dict(max_pages=-1), dict(max_rows=-1), dict(max_len=-1),
                dict(rows=(1 << 23) + 1), dict(n_seqs=1 << 21)):
        assert call(b=batch(**bad)) == bl.BTL_ERR_SHAPE, bad
    for bad in (dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=A + 8), dict(v=A + 4),
                dict(k_scale=A + 8), dict(v_scale=A + 4)):
        assert call(c=cache(**bad)) == bl.BTL_ERR_LAYOUT, bad
    for bad in (dict(row_start=None), dict(pos=None), dict(pages=None), dict(pos=A + 2), dict(row_start=A + 1),
                dict(pages=A + 3)):
        assert call(b=batch(**bad)) == bl.BTL_ERR_LAYOUT, bad
    assert call(dt=2) == bl.BTL_ERR_DTYPE
    # no rows or no sequences: nothing to do, nothing looked at
    assert call(b=batch(rows=0, row_start=None)) == bl.BTL_OK
    assert call(b=batch(n_seqs=0, pos=None)) == bl.BTL_OK


def test_null_structs():
    c, b = cache(), batch()
    assert bl.lib.btl_paged_read(None, ctypes.byref(b), A, A, 0, None) == bl.BTL_ERR_ARG
    assert bl.lib.btl_paged_read(ctypes.byref(c), None, A, A, 0, None) == bl.BTL_ERR_ARG
    assert bl.lib.btl_paged_attention_workspace_bytes(4, None, ctypes.byref(b)) == 0


def test_append_refusals():
    for nh in (0, 3, 34, -2):  # none, no multiple of 2, 17 a KV head
        assert append(nh=nh) == bl.BTL_ERR_SHAPE
    assert append(length=-1) == bl.BTL_ERR_SHAPE
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cos=None), dict(sin=None),
                dict(q=A + 2), dict(out=16 * A + 1), dict(cos=A + 2)):
        assert append(**bad) == bl.BTL_ERR_LAYOUT, bad
    # q_out over part of q, k or v (5 rows of 4 * 64 and of 2 * 64 floats)
    assert append(q=A, out=A + 5 * 1024 - 4) == bl.BTL_ERR_LAYOUT
    assert append(k=16 * A + 4) == bl.BTL_ERR_LAYOUT
    assert append(v=16 * A - 4) == bl.BTL_ERR_LAYOUT


def test_read_refusals():
    assert read(k=A, v=A) == bl.BTL_ERR_LAYOUT
    assert read(k=A + 2) == bl.BTL_ERR_LAYOUT
    assert read(k=None, v=None) == bl.BTL_OK


def test_attention_refusals():
    for nh in (0, 3, 34):
        assert attention(nh=nh) == bl.BTL_ERR_SHAPE
    for bad in (dict(q=None), dict(out=None), dict(q=A + 8), dict(out=16 * A + 4), dict(out=A), dict(out=A + 16)):
        assert attention(**bad) == bl.BTL_ERR_LAYOUT, bad
    # one grid's workgroups
    assert attention(b=batch(n_seqs=1 << 20, max_len=1 << 30, max_pages=1 << 24),
                     c=cache(n_kv_heads=1024, page_size=1 << 16), nh=1024) == bl.BTL_ERR_SHAPE


def test_sample_refusals():
    def call(logits=A, rows=2, n=100, ld=100, t=A, k=A, p=A, m=A, u=A, ids=A, probs=A):
        return bl.lib.btl_sample(logits, rows, n, ld, t, k, p, m, u, ids, probs, None, 0, None)
    for bad in (dict(rows=-1), dict(rows=65536), dict(n=0), dict(n=(1 << 22) + 1, ld=1 << 23), dict(ld=99)):
        assert call(**bad) == bl.BTL_ERR_SHAPE, bad
    for bad in (dict(logits=None), dict(u=None), dict(ids=None), dict(logits=A + 2), dict(t=A + 1), dict(k=A + 2),
                dict(p=A + 3), dict(m=A + 2), dict(probs=A + 1), dict(ids=A + 2)):
        assert call(**bad) == bl.BTL_ERR_LAYOUT, bad
    assert call(rows=0, logits=None) == bl.BTL_OK
    size = bl.lib.btl_sample_workspace_bytes
    assert size(0, 10) == 0 and size(1, 0) == 0 and size(1, 1 << 23) == 0 and 0 < size(1, 10) <= size(2, 10) <= size(2, 10 ** 5)


def test_workspace_grows_with_the_split():
    def size(**b):
        c, b = cache(n_kv_heads=8, n_pages=10000, page_size=64, head_dim=128), batch(**b)
        return bl.lib.btl_paged_attention_workspace_bytes(32, ctypes.byref(c), ctypes.byref(b))
    assert size(n_seqs=1, rows=1, max_rows=1, max_len=16, max_pages=1) == 0  # one chunk: no parts
    assert size(n_seqs=1, rows=1, max_rows=1, max_len=10 ** 5, max_pages=2000) > 0
    assert size(n_seqs=0) == 0


def test_python_refusals():
    with pytest.raises(bl.BitLinearError):
        bl.PagedKVCacheQ8(4, 24, 2, 64, "cpu")
    with pytest.raises(bl.BitLinearError):
        bl.PagedKVCacheQ8(4, 16, 2, 64, "cpu")  # no kernels there
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(bl.BitLinearError):
        bl.PagedBatch(i, i[:2], torch.zeros((2, 4), dtype=torch.int32), 3)
    with pytest.raises(bl.BitLinearError):
        bl.sample(torch.zeros((2, 5)), torch.zeros(2))


def test_reference_attention_is_softmax():
    rng = np.random.default_rng(0)
    sizes = [(3, 20), (1, 0)]
    table, n_pages = ref.pages_for(sizes, 16, rng)
    c = ref.rand_cache(rng, n_pages, 2, 16, 32)
    q = rng.standard_normal((4, 4, 32))
    out, bound = ref.attention(q, c, table, sizes, [0, 3], False)
    k, v = ref.rows_of(c, table, 0, 23)
    for i in range(3):
        for h in range(4):
            s = [float(q[i, h] @ k[j, h // 2]) / math.sqrt(32) for j in range(21 + i)]
            w = [math.exp(x - max(s)) for x in s]
            o = sum(x * v[j, h // 2] for j, x in enumerate(w)) / sum(w)
            assert np.abs(out[i, h] - o).max() < 1e-12
    assert np.abs(out[3, 2] - ref.rows_of(c, table, 1, 1)[1][0, 1]).max() < 1e-12
    assert (bound > 0).all() and bound.max() < 1e-3


def test_reference_sample_by_hand():
    w = np.log(np.array([1, 4, 2, 1], np.float32))
    assert ref.sample_one(w, u=0.0)[0] == 1 and ref.sample_one(w, u=0.49)[0] == 1
    assert ref.sample_one(w, u=0.51)[0] == 2 and ref.sample_one(w, u=0.76)[0] == 0 and ref.sample_one(w, u=0.99)[0] == 3
    assert ref.sample_one(w, k=2, u=0.99)[0] == 2 and ref.sample_one(w, p=0.4, u=0.99)[0] == 1
    assert ref.sample_one(w, m=0.4, u=0.99)[0] == 2 and ref.sample_one(w, t=0.0)[0] == 1
    assert abs(ref.sample_one(w, k=3, u=0.99)[1] - 1 / 7) < 1e-9 and ref.sample_one(w, k=3, u=0.99)[0] == 0
