"""CPU tests of what long contexts ask for (include/bitserve.h): argument checks before any
device work, workspace sizes, and the plain implementations that the GPU tests use."""
import ctypes
import math

import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_serve_host import A, batch, cache

FAR = 1 << 20


def account(**change):
    a = dict(weight=FAR, token=2 * FAR, filled=3 * FAR, shift=4 * FAR, ld=64)
    a.update(change)
    return bl.BtlKvAccount(*a.values())


def by(x):
    return None if x is None else ctypes.byref(x)


def prefixed(c=None, b=None, p=0, q=A, out=16 * A, dt=0, nh=4, ws=None, wsn=0):
    c, b, p = c or cache(), b or batch(), batch(n_seqs=2, max_rows=5) if p == 0 else p
    return bl.lib.btl_paged_attention_prefix(q, dt, nh, by(c), by(b), by(p), out, ws, wsn, None)


def accounted(c=None, b=None, p=0, a=0, q=A, out=16 * A, dt=0, nh=4, ws=None, wsn=0):
    c, b, p = c or cache(), b or batch(), batch(n_seqs=2, max_rows=5) if p == 0 else p
    a = account() if a == 0 else a
    return bl.lib.btl_paged_attention_account(q, dt, nh, by(c), by(b), by(p), by(a), out, ws, wsn, None)


def evict(c=None, b=None, a=0, keep=5 * FAR, sink=6 * FAR, recent=7 * FAR, most=32, to=None, held=8 * FAR, ws=None, wsn=0):
    c, b, a = c or cache(), b or batch(), account() if a == 0 else a
    return bl.lib.btl_paged_evict(by(c), by(b), by(a), keep, sink, recent, most, by(to), held, ws, wsn, None)


def shifted(c=None, b=None, shift=A, dt=0, nh=4):
    c, b = c or cache(), b or batch()
    return bl.lib.btl_paged_rope_append_shifted(A, 2 * A, 3 * A, dt, nh, by(c), by(b), shift, A, A, 64, 16 * A, None)


@pytest.mark.parametrize("call", [prefixed, accounted, evict, shifted])
def test_cache_and_batch_are_checked(call):
    for bad in (dict(n_pages=0), dict(n_kv_heads=0), dict(page_size=24), dict(head_dim=72), dict(head_dim=144)):
        assert call(c=cache(**bad)) == bl.BTL_ERR_SHAPE, bad
    for bad in (dict(n_seqs=-1), dict(rows=-1), dict(max_pages=-1), dict(max_rows=-1), dict(max_len=-1), dict(n_seqs=1 << 21)):
        assert call(b=batch(**bad)) == bl.BTL_ERR_SHAPE, bad
    for bad in (dict(k=None), dict(v=A + 4), dict(k_scale=None), dict(v_scale=A + 8)):
        assert call(c=cache(**bad)) == bl.BTL_ERR_LAYOUT, bad
    for bad in (dict(row_start=None), dict(pos=None), dict(pages=None), dict(pos=A + 2)):
        assert call(b=batch(**bad)) == bl.BTL_ERR_LAYOUT, bad
    assert call(b=batch(n_seqs=0, pos=None)) == bl.BTL_OK


@pytest.mark.parametrize("call", [prefixed, accounted])
def test_attention_refusals(call):
    assert call(dt=2) == bl.BTL_ERR_DTYPE
    for nh in (0, 3, 34):
        assert call(nh=nh) == bl.BTL_ERR_SHAPE
    assert call(p=batch(rows=4)) == bl.BTL_ERR_SHAPE  # other rows than the batch's
    assert b"rows" in bl.lib.btl_last_error()
    assert call(p=batch(n_seqs=-1)) == bl.BTL_ERR_SHAPE
    for bad in (dict(row_start=None), dict(pos=A + 1), dict(pages=None)):
        assert call(p=batch(**bad)) == bl.BTL_ERR_LAYOUT, bad
    for bad in (dict(q=None), dict(out=None), dict(q=A + 8), dict(out=16 * A + 4), dict(out=A + 16)):
        assert call(**bad) == bl.BTL_ERR_LAYOUT, bad
    assert call(b=batch(rows=0), p=batch(rows=0, pos=None)) == bl.BTL_OK
    # one grid's workgroups, of the batch and of the prefix
    huge = dict(n_seqs=1 << 20, max_len=1 << 30, max_pages=1 << 24)
    wide = dict(c=cache(n_kv_heads=1024, page_size=1 << 16), nh=1024)
    a = dict(a=account(ld=1 << 24)) if call is accounted else {}
    assert call(b=batch(**huge), **wide, **a) == bl.BTL_ERR_SHAPE
    assert call(p=batch(**huge), **wide, **a) == bl.BTL_ERR_SHAPE


def test_prefix_is_asked_for():
    assert prefixed(p=None) == bl.BTL_ERR_ARG
    c, b = cache(), batch()
    assert bl.lib.btl_paged_attention_prefix_workspace_bytes(4, by(c), by(b), None) == 0


def test_account_refusals():
    assert accounted(a=None) == bl.BTL_ERR_ARG and evict(a=None) == bl.BTL_ERR_ARG
    # fewer positions than a sequence may have (50)
    for call in (accounted, evict):
        assert call(a=account(ld=49)) == bl.BTL_ERR_SHAPE
        assert call(a=account(ld=(1 << 32) + 1)) == bl.BTL_ERR_SHAPE
        assert call(a=account(weight=None)) == bl.BTL_ERR_LAYOUT
        assert call(a=account(weight=FAR + 2)) == bl.BTL_ERR_LAYOUT
    assert accounted(a=account(weight=A)) == bl.BTL_ERR_LAYOUT           # over q
    assert accounted(a=account(weight=16 * A + 4)) == bl.BTL_ERR_LAYOUT  # over out
    # one over the largest grid of positions
    assert accounted(b=batch(n_seqs=1 << 20, max_len=4096, max_pages=1 << 10), c=cache(n_kv_heads=2),
                     a=account(ld=4096), p=None) == bl.BTL_ERR_SHAPE


def test_evict_refusals():
    assert evict(most=-1) == bl.BTL_ERR_SHAPE
    for name in ("token", "filled", "shift"):
        assert evict(a=account(**{name: None})) == bl.BTL_ERR_LAYOUT, name
        assert evict(a=account(**{name: FAR * 9 + 2})) == bl.BTL_ERR_LAYOUT, name
        to = dict(weight=20 * FAR, token=21 * FAR, filled=22 * FAR, shift=23 * FAR)
        to[name] = None
        assert evict(to=account(**to)) == bl.BTL_ERR_LAYOUT, name
    for bad in (dict(keep=None), dict(held=None), dict(keep=5 * FAR + 2), dict(sink=6 * FAR + 1), dict(recent=7 * FAR + 3),
                dict(held=8 * FAR + 2)):
        assert evict(**bad) == bl.BTL_ERR_LAYOUT, bad
    # what is put out lies over what others read: held over keep, pos or the account, one account's filled over
    # the other's shift, weights shifted by one, two arrays over each other
    for bad in (dict(held=5 * FAR), dict(held=A), dict(held=4 * FAR + 8), dict(held=3 * FAR),
                dict(to=account(weight=20 * FAR, token=21 * FAR, filled=4 * FAR, shift=23 * FAR)),
                dict(to=account(weight=FAR + 4, token=21 * FAR, filled=22 * FAR, shift=23 * FAR)),
                dict(to=account(weight=FAR, ld=65)),
                dict(to=account(weight=20 * FAR, token=20 * FAR, filled=22 * FAR, shift=23 * FAR)),
                dict(held=22 * FAR, to=account(weight=20 * FAR, token=21 * FAR, filled=22 * FAR, shift=23 * FAR))):
        assert evict(**bad) == bl.BTL_ERR_LAYOUT, bad
    assert evict(to=account(ld=49)) == bl.BTL_ERR_SHAPE
    assert evict(b=batch(n_seqs=1 << 20, max_len=50), c=cache(n_kv_heads=8)) == bl.BTL_ERR_SHAPE


def test_shift_refusals():
    assert shifted(shift=A + 2) == bl.BTL_ERR_LAYOUT


def test_workspaces():
    def size(n_heads=32, prefix=None, what="account", **b):
        c = cache(n_kv_heads=8, n_pages=10000, page_size=64, head_dim=128)
        b = batch(**dict(dict(max_pages=200), **b))
        f = getattr(bl.lib, "btl_paged_attention_%s_workspace_bytes" % what)
        return f(n_heads, by(c), by(b), by(prefix))
    p = batch(n_seqs=1, rows=5, max_rows=5, max_len=5000, max_pages=100)
    assert size(what="prefix", prefix=p) > 0 and size(what="prefix") == 0
    assert size() > 0 and size(prefix=p) > size()
    assert size(n_seqs=0) == 0 and size(rows=0) == 0 and size(n_heads=3) == 0
    assert size(prefix=batch(rows=4)) == 0
    # scores of 2^28 and more are not kept: the workspace stays small
    assert size(n_seqs=64, rows=64, max_rows=1, max_len=1 << 20, max_pages=1 << 17) < 1 << 32
    c, b = cache(), batch()
    assert bl.lib.btl_paged_evict_workspace_bytes(by(c), by(b)) >= 3 * 2 * 50 * 4
    assert bl.lib.btl_paged_evict_workspace_bytes(by(cache()), by(batch(max_len=10 ** 5, max_pages=10 ** 4))) >= 3 * 3 * 2 * 10 ** 5 * 4
    assert bl.lib.btl_paged_evict_workspace_bytes(None, by(b)) == 0


def test_python_refusals():
    with pytest.raises(bl.BitLinearError):
        bl.KVAccount(2, 2, 10, "cpu")  # no kernels there
    with pytest.raises(bl.BitLinearError):
        bl.KVAccount.of(torch.zeros((2, 10)))


def test_reference_weights_and_choice_by_hand():
    rng = np.random.default_rng(0)
    sizes, lists = [(2, 5), (1, 0)], [(1, 2, 9)]
    table, n_pages = ref.pages_for(sizes + [(0, 9)], 16, rng)
    c = ref.rand_cache(rng, n_pages, 1, 16, 32)
    q = rng.standard_normal((3, 2, 32))
    out, _, w, _ = cref.attention(q, c, table[:2], sizes, [0, 2], False, lists, table[2:])
    k, v = ref.rows_of(c, table, 0, 7)
    pk, pv = ref.rows_of(c, table, 2, 9)
    total = np.zeros(7)
    for i in range(2):
        for h in range(2):
            kk = [x[0] for x in (list(pk) if i else [])] + [k[j, 0] for j in range(6 + i)]
            vv = [x[0] for x in (list(pv) if i else [])] + [v[j, 0] for j in range(6 + i)]
            e = [math.exp(float(q[i, h] @ x) / math.sqrt(32)) for x in kk]
            p = [x / sum(e) for x in e]
            assert np.abs(out[i, h] - sum(a * b for a, b in zip(p, vv))).max() < 1e-12
            total[:6 + i] += p[9 * i:]
    assert np.abs(w[0][0] - total).max() < 1e-12 and w[1].shape == (1, 1)
    come, place = cref.choose([5, 1, 7, 1, 2, 1], [0] * 6, 0, 10, 6, 3, 0, 1)
    assert come == [0, 5, 2] and place == [10, 15, 12]  # the last, and the heaviest two
    come, place = cref.choose([5, 1, float("nan"), 1, 1, 2], [40, 3, 41, 44], 4, 100, 6, 4, 4, 0)
    assert come == [0, 1, 5, 3] and place == [40, 3, 105, 44]
