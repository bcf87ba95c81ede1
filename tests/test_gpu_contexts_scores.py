"""GPU tests of accounted weights (include/bitserve.h) whose scores are made a second time: each
row's weights are those of the softmax that the attention took, however large its scores are."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_gpu_contexts import on_gpu
from test_gpu_serve import DEV, DT, batch_of, dev, host

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

FAR = 1 << 23  # a bound on the lengths that leaves few rows' scores unkept


@pytest.mark.parametrize("sizes", [[(1, 100), (3, 700)], [(4, 60), (2, 0)], [(1, 300), (40, 100)]])
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1.0, 1e6, 1e12, 1e30])
def test_scores_of_any_size_that_are_not_kept(size, dtype, hd, sizes):
    nh, nkv, ps = 8, 2, 16
    print("scores", size, dtype, hd, sizes, flush=True)
    rng = np.random.default_rng(41)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    table = np.concatenate([table, np.full((len(sizes), FAR // ps - table.shape[1]), -1, np.int32)], axis=1)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    batch, _ = batch_of(table, sizes, max_len=FAR)
    rows = sum(r for r, _ in sizes)
    q = dev((rng.standard_normal((rows, nh * hd)) * size).astype(np.float32), DT[dtype])
    account = bl.KVAccount.of(torch.zeros((len(sizes), nkv, FAR), device=DEV))
    out = host(bl.paged_attention_account(q, on_gpu(cache), batch, account))
    assert np.isfinite(out).all()
    for s, (r, p) in enumerate(sizes):
        w = host(account.weight[s, :, :p + r]).astype(np.float64)
        assert np.isfinite(w).all() and (w >= 0).all()
        n = r * nh // nkv  # softmaxes of a KV head, each 1 in all but for the roundings of its terms and sums
        assert np.abs(w.sum(axis=1) - n).max() <= n * (2 * (p + r) + n + 8) * cref.U
        if size >= 1e12:  # every softmax is one key's
            assert (np.abs(w - np.rint(w)) <= n * 8 * cref.U).all()


@pytest.mark.parametrize("rows,far", [(1, 0), (4, FAR), (40, 0), (400, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_far_below_one_that_meets_only_zeros(dtype, rows, far):
    """The attention scales a row by its largest query and loses bits of those far below it.  Where that one
    meets zeros alone, the scores are what is lost: a position's weight is still at most 1 a row and head."""
    nh, nkv, hd, ps, pos = 16, 4, 64, 16, 100
    rng = np.random.default_rng(43)
    table, n_pages = ref.pages_for([(rows, pos)], ps, rng)
    table = np.concatenate([table, np.full((1, max(1, far // ps - table.shape[1])), -1, np.int32)], axis=1)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    cache[0][..., 5] = 128
    batch, _ = batch_of(table, [(rows, pos)], max_len=far or None)
    q = (rng.standard_normal((rows, nh, hd)) * 2.0 ** 40).astype(np.float32)
    q[..., 5] = 2.0 ** 90
    ld = far or rows + pos
    account = bl.KVAccount.of(torch.zeros((1, nkv, ld), device=DEV))
    out = host(bl.paged_attention_account(dev(q.reshape(rows, -1), DT[dtype]), on_gpu(cache), batch, account))
    assert np.isfinite(out).all()
    w = host(account.weight[0, :, :pos + rows])
    n = rows * nh // nkv
    assert np.isfinite(w).all() and (w >= 0).all() and (w <= n * (1 + n * cref.U)).all()
