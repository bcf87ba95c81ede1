"""GPU tests of the batched serving ops (include/bitserve.h) against plain implementations
in 64 bits (serve_ref.py) and, for what is written into the cache, the CPU oracle.

Codes, scales and rows read back are compared bit for bit; attention within the bound that
serve_ref.attention derives; tokens exactly."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import serve_ref as ref
from oracle import oracle as orc

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.detach().float().cpu().numpy()


def batch_of(table, sizes, rows=None, max_rows=None, max_len=None, first=0):
    starts = first + np.concatenate([[0], np.cumsum([r for r, _ in sizes])])
    b = bl.PagedBatch(dev(starts.astype(np.int32)), dev(np.array([p for _, p in sizes], np.int32)), dev(table),
                      int(starts[-1]) if rows is None else rows,
                      max([r for r, _ in sizes]) if max_rows is None else max_rows,
                      max([r + p for r, p in sizes]) if max_len is None else max_len)
    return b, starts


def rope(hd, size):
    c, s = orc.rope_table(10000.0, hd, size)
    return c, s, dev(c), dev(s)


def same(a, b, what=""):
    a, b = np.ascontiguousarray(a, np.float32), np.ascontiguousarray(b, np.float32)
    assert a.shape == b.shape
    ok = (a.view(np.uint32) == b.view(np.uint32)) | (np.isnan(a) & np.isnan(b))
    assert ok.all(), "%s: %d of %d differ, first %r vs %r" % (what, (~ok).sum(), ok.size, a[~ok][0], b[~ok][0])


# ------------------------------------------------------------------ append and read

APPENDS = [
    # (heads, kv heads, hd, page, [(rows, pos)])
    (4, 2, 64, 16, [(1, 0)]),
    (32, 8, 128, 16, [(1, 37), (0, 5), (3, 0), (1, 15), (17, 16)]),
    (3, 1, 16, 48, [(50, 1), (2, 47)]),
    (10, 2, 80, 64, [(70, 60), (1, 128)]),
    (8, 8, 112, 256, [(33, 240)]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", APPENDS)
def test_append_writes_the_oracles_codes_and_nothing_else(nh, nkv, hd, ps, sizes, dtype):
    print("append", nh, nkv, hd, ps, sizes, dtype, flush=True)
    rng = np.random.default_rng(hd + ps)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    first, behind = 2, 3  # rows of no sequence on both sides
    rows = first + sum(r for r, _ in sizes) + behind
    q, k, v = (dev(rng.standard_normal((rows, n * hd)).astype(np.float32) * 3, DT[dtype]) for n in (nh, nkv, nkv))
    k[first, :hd] = 0  # a head of zeros
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    for t, x in ((cache.k, 7), (cache.v, 9), (cache.k_scale, 0.5), (cache.v_scale, 0.25)):
        t.fill_(x)
    batch, starts = batch_of(table, sizes, rows=rows, first=first)
    cos, sin, dc, ds = rope(hd, 400)
    out = torch.full_like(q, 5)
    got = bl.paged_rope_append(q, k, v, cache, batch, dc, ds, q_out=out)
    assert got is out
    ek, ev = np.full(cache.k.shape, 7, np.uint8), np.full(cache.v.shape, 9, np.uint8)
    eks, evs = np.full(cache.k_scale.shape, 0.5, np.float32), np.full(cache.v_scale.shape, 0.25, np.float32)
    eq = np.full((rows, nh * hd), 5, np.float32)
    qh, kh, vh = host(q), host(k), host(v)
    for s, (r, p) in enumerate(sizes):
        for i in range(r):
            t, at = starts[s] + i, p + i
            pg, sl = table[s, at // ps], at % ps
            eq[t] = orc.rope_apply(qh[t].reshape(nh, hd), cos[at], sin[at]).reshape(-1)
            ek[pg, :, sl], eks[pg, :, sl] = orc.q8_quant(orc.rope_apply(kh[t].reshape(nkv, hd), cos[at], sin[at]))
            c, evs[pg, :, sl] = orc.q8_quant(vh[t].reshape(nkv, hd))
            ev[pg, :, sl // 16, :, sl % 16] = c
    same(host(out), ref.bf16_round(eq) if dtype == "bf16" else eq, "q")
    assert np.array_equal(cache.k.cpu().numpy(), ek) and np.array_equal(cache.v.cpu().numpy(), ev)
    same(host(cache.k_scale), eks, "k scale")
    same(host(cache.v_scale), evs, "v scale")
    # in place over q
    bl.paged_rope_append(q, k, v, cache, batch, dc, ds, q_out=q)
    keep = torch.ones(rows, dtype=torch.bool)
    keep[first:rows - behind] = False
    same(host(q)[~keep.numpy()], host(out)[~keep.numpy()], "q in place")
    same(host(q)[keep.numpy()], qh[keep.numpy()], "rows of no sequence")
    # what was written, read back
    kr, vr = bl.paged_read(cache, batch, dtype=DT[dtype], k_out=torch.full_like(k, 3), v_out=torch.full_like(v, 3))
    xk, xv = np.full(k.shape, 3, np.float32), np.full(v.shape, 3, np.float32)
    for s, (r, p) in enumerate(sizes):
        if r:
            a, b = ref.rows_of((ek, ev, eks, evs), table, s, r + p)
            xk[starts[s]:starts[s] + r] = a[p:].reshape(r, -1).astype(np.float32)
            xv[starts[s]:starts[s] + r] = b[p:].reshape(r, -1).astype(np.float32)
    if dtype == "bf16":
        xk, xv = ref.bf16_round(xk), ref.bf16_round(xv)
    same(np.abs(host(kr)), np.abs(xk), "k read")  # a zero head's sign is not asked for
    same(np.abs(host(vr)), np.abs(xv), "v read")
    assert np.array_equal(host(kr), xk) and np.array_equal(host(vr), xv)


def test_append_equals_the_contiguous_caches_bytes():
    nh, nkv, hd, ps, m, pos = 32, 8, 128, 32, 70, 45
    rng = np.random.default_rng(5)
    q, k, v = (dev(rng.standard_normal((m, n * hd)).astype(np.float32)) for n in (nh, nkv, nkv))
    _, _, dc, ds = rope(hd, 256)
    from bitlinear.model import KVCacheQ8
    import ctypes
    flat = KVCacheQ8(nkv, 128, hd, DEV)
    qf = torch.empty_like(q)
    bl.check(bl.lib.btl_rope_kv_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), m, nh, ctypes.byref(flat.c), pos, None,
                                       dc.data_ptr(), ds.data_ptr(), qf.data_ptr(),
                                       torch.cuda.current_stream().cuda_stream))
    table, n_pages = ref.pages_for([(m, pos)], ps, rng)
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    batch, _ = batch_of(table, [(m, pos)])
    qp = bl.paged_rope_append(q, k, v, cache, batch, dc, ds)
    assert torch.equal(qp, qf)
    at = torch.arange(pos, pos + m)
    pg, sl = torch.from_numpy(table[0]).long()[at // ps], at % ps
    assert torch.equal(cache.k.cpu()[pg, :, sl].transpose(0, 1), flat.k.cpu()[:, pos:pos + m])
    assert torch.equal(cache.v.cpu()[pg, :, sl // 16, :, sl % 16].transpose(0, 1), flat.v.cpu()[:, pos:pos + m])
    assert torch.equal(cache.k_scale.cpu()[pg, :, sl].t(), flat.k_scale.cpu()[:, pos:pos + m])
    assert torch.equal(cache.v_scale.cpu()[pg, :, sl].t(), flat.v_scale.cpu()[:, pos:pos + m])


def test_what_the_device_refuses_is_nan_and_not_stored():
    """Sequences that break a bound, pages outside the pool, positions past the RoPE table."""
    nh, nkv, hd, ps = 4, 2, 64, 16
    sizes = [(2, 3), (2, -1), (3, 40), (5, 0), (2, 14), (2, 30)]
    rng = np.random.default_rng(1)
    table, n_pages = ref.pages_for([(r, max(p, 0)) for r, p in sizes], ps, rng, wide_extra=0)
    table[4, 0] = n_pages  # one past the pool; positions 14, 15
    max_rows, max_len = 4, 40  # sequence 2 has too many tokens, 3 too many rows
    starts = np.concatenate([[0], np.cumsum([r for r, _ in sizes])])
    rows = int(starts[-1])
    batch = bl.PagedBatch(dev(starts.astype(np.int32)), dev(np.array([p for _, p in sizes], np.int32)), dev(table), rows,
                          max_rows, max_len)
    q, k, v = (dev(rng.standard_normal((rows, n * hd)).astype(np.float32)) for n in (nh, nkv, nkv))
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    cache.k_scale.fill_(-1)
    _, _, dc, ds = rope(hd, 31)  # positions 31 and later have no table: sequence 5's second row
    out = host(bl.paged_rope_append(q, k, v, cache, batch, dc, ds))
    kr, vr = bl.paged_read(cache, batch)
    o = host(bl.paged_attention(q, cache, batch))
    refused = [2, 3, 4, 5, 6, 7, 8, 9, 10, 11]
    lost = refused + [rows - 1]
    assert np.isnan(out[lost]).all() and np.isfinite(np.delete(out, lost, 0)).all()
    written = {(table[0, 0], 3), (table[0, 0], 4), (table[5, 1], 14)}
    got = {(int(p), int(s)) for p, s in zip(*np.nonzero((host(cache.k_scale) >= 0).any(1)))}
    assert got == written
    bad_page = [12, 13]  # positions 14 and 15 of sequence 4
    for x in (host(kr), host(vr)):
        assert np.isnan(x[refused + bad_page]).all() and np.isfinite(np.delete(x, refused + bad_page, 0)).all()
    assert np.isnan(o[refused + bad_page]).all() and np.isfinite(o[:2]).all()


# ------------------------------------------------------------------ attention

ATTENTIONS = [
    # (heads, kv heads, hd, page, [(rows, pos)])
    (1, 1, 16, 16, [(1, 0)]),
    (4, 2, 64, 16, [(1, 0), (1, 15), (1, 16), (1, 63), (1, 64), (1, 255), (1, 256), (1, 300)]),
    (32, 8, 128, 64, [(1, 776), (0, 3), (1, 1023), (2, 511)]),
    (16, 1, 128, 32, [(1, 100), (1, 5)]),          # a group of 16: one token fills the tile
    (5, 5, 80, 48, [(16, 0), (3, 200), (1, 47)]),  # no groups, odd width, pages of 48
    (10, 2, 96, 16, [(40, 0), (7, 77), (1, 130), (0, 0), (26, 250)]),
    (8, 2, 112, 256, [(200, 60)]),
    (8, 1, 32, 32, [(129, 0), (1, 400), (128, 384)]),
    (12, 4, 48, 16, [(65, 511), (1, 1), (2, 700)]),
    # many weights in short sums, where the bound is near two f16 parts' own error
    (16, 4, 32, 16, [(12, 0)] * 60),
]


def check_attention(nh, nkv, hd, ps, sizes, dtype, seed=0, change=None, **bounds):
    rng = np.random.default_rng(seed + hd + ps)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    # slots that no sequence reaches hold anything
    used = np.zeros((n_pages, ps), bool)
    for s, (r, p) in enumerate(sizes):
        for j in range(r + p):
            used[table[s, j // ps], j % ps] = True
    for scales, x in ((cache[2], np.nan), (cache[3], np.inf)):
        scales.transpose(0, 2, 1)[~used] = x
    rows = sum(r for r, _ in sizes)
    q = (rng.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    if change:
        change(q, cache, table)
    if dtype == "bf16":
        q = ref.bf16_round(q)
    batch, starts = batch_of(table, sizes, **bounds)
    dq = dev(q.reshape(rows, -1), DT[dtype])
    paged = bl.PagedKVCacheQ8.of(*[dev(x) for x in cache])
    out = bl.paged_attention(dq, paged, batch)
    again = bl.paged_attention(dq, paged, batch, workspace=bl.paged_attention_workspace(paged, batch, nh))
    assert torch.equal(out.nan_to_num(7), again.nan_to_num(7)), "two runs differ"
    exp, bound = ref.attention(q, cache, table, sizes, starts, dtype == "bf16")
    got = host(out).reshape(exp.shape).astype(np.float64)
    off = np.abs(got - exp)
    worst = float((off / bound).max())
    print("attention", nh, nkv, hd, ps, sizes, dtype, "worst %.3f of the bound" % worst, flush=True)
    assert np.isfinite(got).all() and worst <= 1.0
    return got, exp


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", ATTENTIONS)
def test_attention(nh, nkv, hd, ps, sizes, dtype):
    check_attention(nh, nkv, hd, ps, sizes, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_with_loose_bounds(dtype):
    # the host's bounds are far above the sizes: other launches and splits, the same results
    check_attention(8, 2, 64, 32, [(1, 100), (9, 300), (1, 0)], dtype, max_rows=4096, max_len=100000)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_large_and_small_numbers(dtype):
    """Queries and scales over many powers of two, peaked rows, zero scales."""
    def change(q, cache, table):
        q[0] *= 2.0 ** 60
        cache[2][...] *= np.float32(2.0 ** -60)  # scores of row 0 as they were, 0 of the others
        q[1] = 0
        q[2] *= np.float32(2.0 ** -100)
        cache[3][table[0, 0], :, :8] *= np.float32(2.0 ** 20)
        cache[3][table[0, 1], :, 3] = 0
        cache[3][table[1][:6]] *= np.float32(2.0 ** -90)
        q[3] *= np.float32(2.0 ** -90)
        cache[2][table[1][:6]] *= np.float32(2.0 ** 120)  # the second sequence's scores: as large as ever
        cache[2][table[1][:6]] *= np.float32(2.0 ** 30)
    check_attention(8, 2, 64, 16, [(3, 40), (1, 90)], dtype, change=change)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("power", [10, 30, 60])
def test_attention_of_one_key(dtype, power):
    """Scores so far apart that each row is its best key's value, of either sign, over several steps
    and chunks (no rounding of a score changes which is best: they are whole multiples of one)."""
    nh, nkv, hd, ps, sizes = 8, 2, 64, 16, [(1, 1300), (20, 90), (2, 3)]
    rng = np.random.default_rng(power)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    cache[0][...] = 128
    cache[0][..., 0] = rng.integers(1, 256, cache[0].shape[:3])
    cache[2][...] = np.float32(2.0 ** power)
    rows = sum(r for r, _ in sizes)
    q = np.zeros((rows, nh, hd), np.float32)
    q[..., 0] = np.where(rng.random((rows, nh)) < 0.5, 1024, -1024)
    batch, starts = batch_of(table, sizes)
    got = host(bl.paged_attention(dev(q.reshape(rows, -1), DT[dtype]), bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]),
                                  batch)).reshape(rows, nh, hd)
    exp, _ = ref.attention(q, cache, table, sizes, starts, dtype == "bf16")
    # equal best keys are averaged: their weights are alike, off by the f16 parts and the sums alone
    most = 0.032 * 127
    tol = (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24) * np.abs(exp) + ((2.0 ** -11 if dtype == "bf16" else 2.0 ** -22)
                                                                       + 1400 * 2.0 ** -24) * most
    assert np.isfinite(got).all() and (np.abs(got - exp) <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_places_have_no_effect(dtype):
    """A later row's key with a scale that is huge, infinite or NaN: earlier rows do not see it."""
    nh, nkv, hd, ps, sizes = 8, 2, 64, 16, [(40, 30)]
    rng = np.random.default_rng(9)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    q = (rng.standard_normal((40, nh, hd)) * 2).astype(np.float32)
    batch, starts = batch_of(table, sizes)
    dq = dev(q.reshape(40, -1), DT[dtype])
    clean = host(bl.paged_attention(dq, bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]), batch))
    at = 30 + 25  # row 25's own key
    for ks, vs in ((np.nan, 1.0), (1.0, np.nan), (np.inf, 1.0), (1.0, np.inf), (1.0, 2.0 ** 100), (3e38, 3e38)):
        bad = [x.copy() for x in cache]
        bad[2][table[0, at // ps], :, at % ps] = ks
        bad[3][table[0, at // ps], :, at % ps] = vs
        got = host(bl.paged_attention(dq, bl.PagedKVCacheQ8.of(*[dev(x) for x in bad]), batch))
        same(got[:25], clean[:25], "rows before the key, scales %g %g" % (ks, vs))
        if not np.isfinite([ks, vs]).all():
            assert not np.isfinite(got[25:]).all(1).any()
    q2 = q.copy()
    q2[7, 3, 5], q2[8, 0, 0] = np.nan, np.inf
    got = host(bl.paged_attention(dev(q2.reshape(40, -1), DT[dtype]),
                                  bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]), batch)).reshape(40, nh, hd)
    bad = np.zeros((40, nh), bool)
    bad[7, 3] = bad[8, 0] = True
    assert np.isnan(got[bad]).all()
    same(got[~bad], clean.reshape(40, nh, hd)[~bad], "the other queries")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_leaves_other_rows(dtype):
    sizes = [(2, 20), (0, 0), (1, 9)]
    rng = np.random.default_rng(2)
    table, n_pages = ref.pages_for(sizes, 16, rng)
    cache = ref.rand_cache(rng, n_pages, 2, 16, 64)
    batch, starts = batch_of(table, sizes, rows=9, first=1)
    q = dev(rng.standard_normal((9, 4 * 64)).astype(np.float32), DT[dtype])
    out = torch.full_like(q, 3)
    bl.paged_attention(q, bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]), batch, out=out)
    got = host(out)
    assert (got[[0, 4, 5, 6, 7, 8]] == 3).all() and (got[1:4] != 3).any(1).all()


def test_attention_shares_pages_and_matches_the_contiguous_form():
    """Two sequences over the same prefix pages; the one-sequence attention as a check."""
    import ctypes
    from bitlinear.model import KVCacheQ8
    nh, nkv, hd, ps, n = 8, 2, 128, 16, 75
    rng = np.random.default_rng(3)
    table = np.stack([rng.permutation(8)[:5]] * 2).astype(np.int32)
    cache = ref.rand_cache(rng, 8, nkv, ps, hd)
    paged = bl.PagedKVCacheQ8.of(*[dev(x) for x in cache])
    q = dev(rng.standard_normal((2, nh * hd)).astype(np.float32))
    batch, _ = batch_of(table, [(1, n - 1), (1, 40)])
    got = host(bl.paged_attention(q, paged, batch))
    flat = KVCacheQ8(nkv, 80, hd, DEV)
    at = np.arange(80)
    flat.k.copy_(dev(cache[0][table[0][at // ps], :, at % ps].transpose(1, 0, 2)))
    flat.v.copy_(dev(cache[1][table[0][at // ps], :, at % ps // 16, :, at % 16].transpose(1, 0, 2)))
    flat.k_scale.copy_(dev(cache[2][table[0][at // ps], :, at % ps].T))
    flat.v_scale.copy_(dev(cache[3][table[0][at // ps], :, at % ps].T))
    out = torch.empty_like(q)
    for i, p in enumerate((n - 1, 40)):
        bl.check(bl.lib.btl_attention(q[i].data_ptr(), 1, nh, ctypes.byref(flat.c), p, None, out[i].data_ptr(), None, 0,
                                      torch.cuda.current_stream().cuda_stream))
    _, bound = ref.attention(host(q).reshape(2, nh, hd), cache, table, [(1, n - 1), (1, 40)], [0, 1], False)
    assert (np.abs(got - host(out)) <= 2 * bound.reshape(2, -1)).all()


def test_caches_past_32_bits():
    """Pages whose codes lie more than 4 GiB into the pool."""
    nh, nkv, hd, ps = 8, 8, 128, 64
    n_pages = 2 ** 32 // (nkv * ps * hd) + 40
    rng = np.random.default_rng(4)
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    _, _, dc, ds = rope(hd, 256)
    sizes = [(100, 0), (1, 0)]
    table = np.array([[n_pages - 1, n_pages - 30], [0, 0]], np.int32)
    q, k, v = (dev(rng.standard_normal((101, n * hd)).astype(np.float32)) for n in (nh, nkv, nkv))
    batch, starts = batch_of(table, sizes)
    rot = bl.paged_rope_append(q, k, v, cache, batch, dc, ds)
    o = host(bl.paged_attention(rot, cache, batch)).reshape(101, nh, hd)
    kr, vr = bl.paged_read(cache, batch)
    small = np.array([0, n_pages - 30, n_pages - 1])
    c = [t[dev(small)].cpu().numpy() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    near = np.array([[2, 1], [0, 0]])
    exp, bound = ref.attention(host(rot).reshape(101, nh, hd), c, near, sizes, starts, False)
    assert (np.abs(o - exp) <= bound).all()
    for s, (r, p) in enumerate(sizes):
        a, b = ref.rows_of(c, near, s, r)
        assert np.array_equal(host(kr)[starts[s]:starts[s] + r], a.reshape(r, -1).astype(np.float32))
        assert np.array_equal(host(vr)[starts[s]:starts[s] + r], b.reshape(r, -1).astype(np.float32))
    assert (np.abs(host(kr)[:100] - host(k)[:100]).max() > 0)


def test_many_sequences():
    # more than 64 of them: the search for a row's sequence takes a second step
    check_attention(4, 2, 32, 16, [(1, 3 + i % 40) if i % 7 else (0, 2) for i in range(200)], "f32")
    check_attention(4, 2, 32, 16, [(1 + 30 * (i % 50 == 0), 3 + i % 40) for i in range(150)], "f32")


# ------------------------------------------------------------------ sampling

def check_sample(logits, **f):
    """Rows against the definition; f: lists of one value a row."""
    rows, n = logits.shape
    full = dict(t=[1.0] * rows, k=[0] * rows, p=[1.0] * rows, m=[0.0] * rows, u=[0.5] * rows)
    full.update(f)
    args = [dev(np.array(full[x], np.float32)) for x in "tpmu"]
    k = dev(np.array(full["k"], np.int32))
    x = dev(logits.astype(np.float32))
    ids, probs = bl.sample(x, args[3], args[0], k, args[1], args[2], workspace=bl.sample_workspace(rows, n, DEV))
    i2, p2 = bl.sample(x, args[3], args[0], k, args[1], args[2])
    assert torch.equal(ids, i2) and torch.equal(probs, p2)
    for r in range(rows):
        e, p = ref.sample_one(logits[r], *[full[c][r] for c in "tkpmu"])
        got = (int(ids[r]), float(probs[r]))
        # one f64 division and one rounding to f32; the weights, whole numbers from 2^-1 on, may differ by
        # one where the two exponentials do
        assert got[0] == e and abs(got[1] - p) <= 2.0 ** -23 * p + 2.0 ** -39, (r, n, {c: full[c][r] for c in "tkpmu"}, got, e, p)


FILTERS = [dict(), dict(t=0.7), dict(k=1), dict(k=40), dict(p=0.9), dict(p=0.5, t=1.3), dict(m=0.05), dict(m=1.0),
           dict(k=50, p=0.95, m=0.02, t=0.8), dict(t=0.0), dict(k=3000, p=0.99), dict(p=0.0), dict(p=1e-6),
           dict(k=7, p=0.3), dict(t=100.0), dict(t=1e-6), dict(k=10 ** 9), dict(k=-1, p=2.0, m=-3.0), dict(m=2.0)]


@pytest.mark.parametrize("n", [1, 2, 7, 300, 4096, 4097, 32003, 128256])
@pytest.mark.parametrize("flat", [False, True])
def test_sample(n, flat):
    print("sample", n, flat, flush=True)
    rng = np.random.default_rng(n)
    rows = len(FILTERS)
    logits = rng.standard_normal((rows, n)) * (1.5 if flat else 0.7)
    if not flat:
        logits -= 1.4 * np.log1p(rng.permuted(np.tile(np.arange(n), (rows, 1)), axis=1))
    base = dict(t=1.0, k=0, p=1.0, m=0.0)
    cols = {c: [dict(base, **f)[c] for f in FILTERS] for c in base}
    for u in (rng.random(rows), np.zeros(rows), np.full(rows, 1 - 2.0 ** -24)):
        check_sample(logits.astype(np.float32), u=u.astype(np.float32).tolist(), **cols)


@pytest.mark.parametrize("n", [5000, 100003])
def test_sample_ties(n):
    """Equal logits: more of them in one bin than are ordered at once; cuts inside a tie."""
    print("sample ties", n, flush=True)
    rng = np.random.default_rng(n)
    rows = 8
    logits = np.zeros((rows, n), np.float32)
    logits[1] = -0.0
    logits[2] = rng.integers(0, 2, n)
    logits[3] = rng.integers(0, 40, n) / 1024.0
    logits[4] = np.nextafter(np.float32(1), np.float32(2)) - (rng.integers(0, 2, n) * 2.0 ** -23).astype(np.float32)
    logits[5, ::2] = -0.0
    logits[6] = rng.standard_normal(n) * 1e-4
    logits[7] = rng.integers(0, 3, n) * 50.0
    for f in (dict(), dict(k=3333), dict(p=0.37), dict(k=4000, p=0.71), dict(m=0.9, k=4999), dict(k=700), dict(k=1024, p=0.4)):
        cols = {c: [x] * rows for c, x in f.items()}
        check_sample(logits, u=rng.random(rows).astype(np.float32).tolist(), **cols)


def test_sample_odd_rows():
    """Infinities, NaN, rows with nothing, numbers outside their range."""
    inf, nan, n = np.inf, np.nan, 50
    rng = np.random.default_rng(0)
    a = rng.standard_normal((12, n)).astype(np.float32)
    a[0] = -inf
    a[1] = nan
    a[2, ::2] = nan
    a[3, 7] = a[3, 40] = inf
    a[4] = -inf
    a[4, 49] = -3e38
    a[5] = np.where(np.arange(n) % 2, 3e38, -3e38)
    a[6, 3:] = -inf
    a[7] = np.float32(1e-45) * np.arange(n)
    t = [1, 1, 1, 1, 1, 1e38, 1, 1e-45, nan, inf, 1, -2.0]
    for u in (0.0, 0.3, 0.999, 1.0, 7.0, -1.0, nan):
        print("sample odd", u, flush=True)
        check_sample(a, t=t, u=[u] * 12)
        check_sample(a, t=t, k=[2] * 12, p=[0.7] * 12, u=[u] * 12)
    check_sample(a, t=t, p=[nan] * 12, m=[nan] * 12, u=[0.6] * 12)
    check_sample(a, t=[1e38] * 12, k=[40] * 12, u=[0.6] * 12)  # every finite logit weighs the same
    ids, probs = bl.sample(dev(a), dev(np.full(12, 0.4, np.float32)))
    assert int(ids[0]) == -1 and int(ids[1]) == -1 and float(probs[0]) == 0


def test_sample_strides_and_numbers():
    rng = np.random.default_rng(6)
    wide = dev(rng.standard_normal((5, 1003)).astype(np.float32))
    u = dev(rng.random(5).astype(np.float32))
    for lo, hi in ((0, 1000), (1, 1000), (3, 900)):  # rows that do not begin on 16 bytes
        x = wide[:, lo:hi]
        ids, probs = bl.sample(x, u, temperature=0.9, top_k=30, top_p=0.9, min_p=0.01)
        for r in range(5):
            e, p = ref.sample_one(host(x)[r], 0.9, 30, 0.9, 0.01, float(u[r]))
            assert int(ids[r]) == e and abs(float(probs[r]) - p) <= 2.0 ** -23 * p + 2.0 ** -39


def test_sample_follows_the_weights():
    """All random numbers of a grid: each token as often as its weight says, to one step of the grid."""
    logits = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625], np.float32))[None].repeat(4096, 0)
    u = (np.arange(4096) / 4096).astype(np.float32)
    ids, probs = bl.sample(dev(logits), dev(u))
    got = np.bincount(ids.cpu().numpy(), minlength=5) / 4096
    assert np.abs(got - [0.5, 0.25, 0.125, 0.0625, 0.0625]).max() <= 2 / 4096


# ------------------------------------------------------------------ together

def serve_step(h, state, cache, batch, tabs, weights, u, spaces):
    """A layer's attention and the pick of each sequence's next token."""
    q, k, v = (h @ w for w in weights[:3])
    rot = bl.paged_rope_append(q, k, v, cache, batch, *tabs)
    o = bl.paged_attention(rot, cache, batch, workspace=spaces[0])
    logits = o @ weights[3]
    return o, logits, bl.sample(logits, u, temperature=0.8, top_k=20, top_p=0.9, workspace=spaces[1])


def test_a_step_captured_and_replayed_as_sequences_grow():
    """append -> attention -> sample in a HIP graph; positions, pages and random numbers change
    between replays; every replay against the eager calls on a cache of its own."""
    nh, nkv, hd, ps, n, vocab = 8, 2, 64, 16, 5, 700
    rng = np.random.default_rng(8)
    g = torch.Generator(device=DEV).manual_seed(1)
    weights = [torch.randn((64, w * hd), generator=g, device=DEV) * 0.1 for w in (nh, nkv, nkv)]
    weights.append(torch.randn((nh * hd, vocab), generator=g, device=DEV) * 0.5)
    _, _, dc, ds = rope(hd, 512)
    table, n_pages = ref.pages_for([(1, 200)] * n, ps, rng)
    start = [0, 15, 30, 100, 180]
    init = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    caches = [bl.PagedKVCacheQ8.of(*[dev(x) for x in init]) for _ in range(2)]
    h, u = torch.randn((n, 64), generator=g, device=DEV), torch.rand((n,), generator=g, device=DEV)
    pos = dev(np.array(start, np.int32))
    batch = bl.PagedBatch(dev(np.arange(n + 1, dtype=np.int32)), pos, dev(table), n, 1, 300)
    spaces = (bl.paged_attention_workspace(caches[0], batch, nh), bl.sample_workspace(n, vocab, DEV))
    eager_spaces = (bl.paged_attention_workspace(caches[1], batch, nh), bl.sample_workspace(n, vocab, DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # library handles and code are loaded before the capture
        serve_step(h, None, bl.PagedKVCacheQ8.of(*[dev(x) for x in init]), batch, (dc, ds), weights, u, spaces)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = serve_step(h, None, caches[0], batch, (dc, ds), weights, u, spaces)
    for step in range(6):
        h.copy_(torch.randn((n, 64), generator=g, device=DEV))
        u.copy_(torch.rand((n,), generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        exp = serve_step(h, None, caches[1], batch, (dc, ds), weights, u, eager_spaces)
        torch.cuda.synchronize()
        assert torch.equal(got[0], exp[0]) and torch.equal(got[2][0], exp[2][0]) and torch.equal(got[2][1], exp[2][1])
        for a, b in zip((caches[0].k, caches[0].v, caches[0].k_scale, caches[0].v_scale),
                        (caches[1].k, caches[1].v, caches[1].k_scale, caches[1].v_scale)):
            assert torch.equal(a, b)
        lg = host(got[1])
        for r in range(n):
            assert int(got[2][0][r]) == ref.sample_one(lg[r], 0.8, 20, 0.9, 0.0, float(u[r]))[0]
        pos.add_(1)
        if step == 3:  # one sequence leaves, another starts over in its pages
            pos[3] = 0


def test_a_prompt_in_chunks_equals_the_prompt_at_once():
    nh, nkv, hd, ps, n = 8, 2, 64, 16, 130
    rng = np.random.default_rng(11)
    q, k, v = (dev(rng.standard_normal((n, w * hd)).astype(np.float32)) for w in (nh, nkv, nkv))
    _, _, dc, ds = rope(hd, 256)
    table, n_pages = ref.pages_for([(n, 0)], ps, rng)
    outs, caches = [], []
    for chunks in ([n], [1, 16, 33, 50, 30]):
        cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
        got, at = [], 0
        for c in chunks:
            batch, _ = batch_of(table, [(c, at)])
            rot = bl.paged_rope_append(q[at:at + c], k[at:at + c], v[at:at + c], cache, batch, dc, ds)
            got.append(bl.paged_attention(rot, cache, batch))
            at += c
        outs.append(host(torch.cat(got)))
        caches.append([t.cpu().numpy() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    for a, b in zip(*caches):
        assert np.array_equal(a, b)
    rot = host(bl.paged_rope_append(q, k, v, cache, batch_of(table, [(n, 0)])[0], dc, ds)).reshape(n, nh, hd)
    exp, bound = ref.attention(rot, caches[0], table, [(n, 0)], [0], False)
    for o in outs:
        assert (np.abs(o.reshape(exp.shape) - exp) <= bound).all()


def test_on_another_stream():
    nh, nkv, hd, ps, sizes = 8, 2, 64, 16, [(1, 700), (1, 90)]
    rng = np.random.default_rng(12)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    paged = bl.PagedKVCacheQ8.of(*[dev(x) for x in ref.rand_cache(rng, n_pages, nkv, ps, hd)])
    batch, _ = batch_of(table, sizes)
    q = dev(rng.standard_normal((2, nh * hd)).astype(np.float32))
    exp = bl.paged_attention(q, paged, batch)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:  # two at once, a workspace each
        with torch.cuda.stream(s):
            ws = bl.paged_attention_workspace(paged, batch, nh)
            outs.append((bl.paged_attention(q, paged, batch, workspace=ws), ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, exp) for o, _ in outs)


def test_the_decoder_samples():
    """BitLlamaHip.generate at a temperature: every token is the definition's pick of the logits of
    the tokens before it, captured or not; temperature 0 stays the greedy pick."""
    from test_gpu_model import gpu_model
    from test_model_oracle import TinyCfg, tiny_weights
    cfg = TinyCfg()
    model = gpu_model(cfg, tiny_weights(cfg, 3), max_rows=8)
    prompt, n = [3, 9, 27, 5], 20
    greedy = model.generate(prompt, n)
    u = np.random.default_rng(2).random(n).astype(np.float32)
    f = dict(temperature=0.9, top_k=12, top_p=0.9, min_p=0.01)
    got = model.generate(prompt, n, u=u, **f)
    assert np.array_equal(got, model.generate(prompt, n, use_graph=False, u=u, **f))
    model.reset()
    logits = host(model.prefill(prompt)).copy()
    for i in range(n):
        assert got[i] == ref.sample_one(logits, 0.9, 12, 0.9, 0.01, float(u[i]))[0], i
        assert model.sample(u[i], **f) == got[i]
        logits = host(model.forward_one(int(got[i]))).copy()
    assert not np.array_equal(got, greedy) and np.array_equal(model.generate(prompt, n), greedy)
    with pytest.raises(ValueError):
        model.generate(prompt, n, u=u[:-1], **f)
