"""GPU tests of many sequences and lists (include/bitserve.h): a row's sequence and list are
looked up 64 at a time, so counts on both sides of that and past twice of it."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_gpu_contexts import check_evict, lists_of, on_gpu, random_account, within
from test_gpu_serve import DEV, DT, batch_of, dev, host, same

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

COUNTS = [63, 64, 65, 130, 200]


def case_of(form, n):
    """(sizes, lists) of n sequences."""
    if form == "lists":      # a list a sequence, some of no positions and some of no rows
        sizes = [(int(s % 9 != 4), (7 * s) % 50) for s in range(n)]
        start = np.cumsum([0] + [r for r, _ in sizes])
        return sizes, [(int(start[s]), sizes[s][0], (11 * s) % 70) for s in range(n)]
    if form == "one list":   # of few rows, in many chunks
        return [(1, (5 * s) % 90) for s in range(n)], [(n - 8, 8, 9000)]
    if form == "long list":  # lists of one row, behind them one of many: tiles
        sizes = [(1, (3 * s) % 40) for s in range(n)] + [(12, 5)] * 2
        return sizes, [(s, 1, 20 + s % 5) for s in range(n)] + [(n, 24, 130)]
    if form == "rows":       # many rows here and there, the last far behind
        return [(40 if s in (1, n - 2, n - 1) else s % 3, (s * 13) % 300) for s in range(n)], []
    return [(20 if s % 50 == 3 else 1, (s * 13) % 200) for s in range(n)], [(0, n // 2, 40), (n // 2, n // 3, 300)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", COUNTS)
@pytest.mark.parametrize("form", ["lists", "one list", "long list", "rows", "both"])
def test_rows_of_many_sequences_and_lists(form, n, dtype):
    nh, nkv, hd, ps = 8, 2, 32, 32
    print("many", form, n, dtype, flush=True)
    rng = np.random.default_rng(n)
    sizes, lists = case_of(form, n)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    rows = sum(r for r, _ in sizes)
    prefix = ptable = None
    if lists:
        prefix, ptable, n_pages = lists_of(lists, ps, rng, n_pages, rows)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    gpu = on_gpu(cache)
    batch, starts = batch_of(table, sizes)
    q = dev(rng.standard_normal((rows, nh * hd)).astype(np.float32) * 2, DT[dtype])
    before = rng.random((len(sizes), nkv, max(r + p for r, p in sizes) + 3)).astype(np.float32)
    want, bound, w, wb = cref.attention(host(q).reshape(rows, nh, hd), cache, table, sizes, starts, dtype == "bf16", lists,
                                        ptable)
    if lists:
        alone = bl.paged_attention_prefix(q, gpu, batch, prefix)
        within(host(alone).reshape(rows, nh, hd), want, bound, "outputs beside a prefix")
    account = bl.KVAccount.of(dev(before))
    got = bl.paged_attention_account(q, gpu, batch, account, prefix=prefix)
    within(host(got).reshape(rows, nh, hd), want, bound, "outputs")
    weight = host(account.weight)
    for s, (r, p) in enumerate(sizes):
        if r == 0:
            same(weight[s], before[s], "a sequence without rows")
            continue
        w[s][:, :p] += before[s, :, :p]
        within(weight[s, :, :r + p].astype(np.float64), w[s], wb[s] + cref.U * w[s], "weights of sequence %d" % s)
        same(weight[s, :, r + p:], before[s, :, r + p:], "behind the sequence")
    again = bl.KVAccount.of(dev(before))
    assert torch.equal(bl.paged_attention_account(q, gpu, batch, again, prefix=prefix), got)
    assert torch.equal(again.weight, account.weight)


@pytest.mark.parametrize("n", COUNTS)
@pytest.mark.parametrize("long", [0, 9000])
def test_eviction_of_many_sequences(n, long):
    rng = np.random.default_rng(n)
    size = [(s * 37) % 150 for s in range(n)]
    size[-1] = max(size[-1], long)  # in one launch a head, or by spans
    keep = [(s * 11) % 90 - 1 for s in range(n)]
    table, n_pages = ref.pages_for([(0, x) for x in size], 16, rng)
    cache = ref.rand_cache(rng, n_pages, 2, 16, 16)
    account = random_account(rng, size, 2, max(size), keep, True)
    check_evict(cache, table, size, account, keep, [3] * n, [5] * n, in_place=True)
