"""GPU tests of accounted weights over scales that are not finite (include/bitserve.h): a row
that sees one comes back as NaN and adds nothing, in the token form and in tiles, over its own
positions and over a prefix; the other rows' weights are as in 64 bits (context_ref.py)."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_gpu_contexts import lists_of, on_gpu, within
from test_gpu_serve import DEV, DT, batch_of, dev, host, same
from test_gpu_serve_scales import FORMS, SCALES

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

HEAD = 1  # the KV head of the bad key


def check(nh, nkv, hd, sizes, lists, lost, put, dtype, seed):
    """Weights and outputs with each of SCALES in one place.  lost(s, i): row i of sequence s sees it;
    put(table, prefix table): its page and slot, of 32 positions a page."""
    ps, g = 32, nh // nkv
    rng = np.random.default_rng(seed)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    rows = sum(r for r, _ in sizes)
    prefix = ptable = None
    if lists:
        prefix, ptable, n_pages = lists_of(lists, ps, rng, n_pages, rows)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    batch, starts = batch_of(table, sizes)
    q = dev((rng.standard_normal((rows, nh * hd)) * 2).astype(np.float32), DT[dtype])
    hq = host(q).reshape(rows, nh, hd)
    before = rng.random((len(sizes), nkv, max(r + p for r, p in sizes))).astype(np.float32)
    bf = dtype == "bf16"
    out, bound, w, wb = cref.attention(hq, cache, table, sizes, starts, bf, lists, ptable)
    # rows see positions in order, so those that do not see the key are a sequence's first
    good = [sum(not lost(s, i) for i in range(r)) for s, (r, _) in enumerate(sizes)]
    _, _, w1, wb1 = cref.attention(hq, cache, table, [(n, p) for n, (_, p) in zip(good, sizes)], starts, bf, lists, ptable)
    gone = np.zeros((rows, nh), bool)
    for s, (r, p) in enumerate(sizes):
        gone[starts[s] + good[s]:starts[s] + r, HEAD * g:(HEAD + 1) * g] = True
        for x, y in ((w, w1), (wb, wb1)):
            x[s][HEAD] = 0
            x[s][HEAD, :good[s] + p] = y[s][HEAD]
        w[s][:, :p] += before[s, :, :p]
    assert gone.any()
    page, slot = put(table, ptable)
    for ks, vs in SCALES:
        print("weights", nh, nkv, hd, sizes[:3], lists, dtype, ks, vs, flush=True)
        bad = [x.copy() for x in cache]
        bad[2][page, HEAD, slot], bad[3][page, HEAD, slot] = ks, vs
        account = bl.KVAccount.of(dev(before))
        got = host(bl.paged_attention_account(q, on_gpu(bad), batch, account, prefix=prefix)).reshape(hq.shape)
        assert np.isnan(got[gone]).all()
        within(got[~gone], out[~gone], bound[~gone], "outputs")
        weight = host(account.weight)
        for s, (r, p) in enumerate(sizes):
            if r:
                within(weight[s, :, :r + p].astype(np.float64), w[s], wb[s] + cref.U * w[s], "weights of sequence %d" % s)
            else:
                same(weight[s], before[s])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,sizes,at", FORMS)
def test_rows_that_see_a_scale_that_is_not_finite_add_nothing(nh, nkv, hd, sizes, at, dtype):
    check(nh, nkv, hd, sizes, (), lambda s, i: s == 0 and sizes[0][1] + i >= at,
          lambda table, _: (table[0, at // 32], at % 32), dtype, hd + at)


# (heads, kv heads, hd, [(rows, pos)], [(first row, rows, prefix length)], position of the bad key of list 0)
BEHIND = [
    (8, 2, 64, [(1, 3 * n) for n in range(6)], [(0, 4, 300), (4, 2, 40)], 150),           # the token form
    (8, 2, 64, [(1, 3 * n) for n in range(24)], [(0, 20, 300), (20, 4, 40)], 150),        # tiles, of single tokens
    (8, 2, 112, [(1, 9 * n) for n in range(24)], [(0, 20, 2100), (20, 4, 40)], 2099),     # the same in chunks
    (8, 2, 80, [(40, 130), (0, 7), (1, 20), (9, 0)], [(0, 40, 64), (40, 10, 33)], 0),     # tiles of both
    (32, 8, 128, [(380, 30), (25, 100)], [(0, 380, 330), (380, 25, 70)], 64),             # tiles of 128 rows in 16 bits
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,sizes,lists,at", BEHIND)
def test_rows_behind_a_prefix_with_such_a_scale_add_nothing(nh, nkv, hd, sizes, lists, at, dtype):
    n = sum(r for r, _ in sizes)
    first = np.cumsum([0] + [r for r, _ in sizes])
    assert n == lists[-1][0] + lists[-1][1]
    check(nh, nkv, hd, sizes, lists, lambda s, i: first[s] + i < lists[0][1],
          lambda _, ptable: (ptable[0, at // 32], at % 32), dtype, hd + at)
