"""GPU tests of how exact the paged attention of single tokens is in 16 bits: what is rounded
to bf16 at the end is as exact as the f32 form's result."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import serve_ref as ref
from test_gpu_serve import DT, batch_of, dev, host

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", [
    (8, 2, 64, 16, [(1, 300), (4, 75), (1, 0), (2, 500)]),
    (32, 8, 128, 64, [(1, 1500), (1, 15), (1, 776)]),
    (16, 1, 96, 32, [(1, 700)]),
    (5, 5, 32, 16, [(16, 9), (3, 200)]),
])
def test_single_tokens_are_rounded_once(nh, nkv, hd, ps, sizes):
    """Rounding keeps the order: a result within b of the exact one e lies, rounded, between the
    roundings of e - b and e + b.  b is the f32 form's bound, in which queries and weights are off by
    2^-22 of themselves; weights of 11 bits would leave it."""
    rng = np.random.default_rng(hd)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    rows = sum(r for r, _ in sizes)
    q = ref.bf16_round((rng.standard_normal((rows, nh, hd)) * 2).astype(np.float32))
    batch, starts = batch_of(table, sizes)
    out = bl.paged_attention(dev(q.reshape(rows, -1), DT["bf16"]), bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]), batch)
    got = host(out).reshape(q.shape)
    exp, b = ref.attention(q, cache, table, sizes, starts, False)
    low, high = (torch.from_numpy(x).to(torch.bfloat16).float().numpy() for x in (exp - b, exp + b))
    off = (got < low) | (got > high)
    print("single tokens", nh, nkv, hd, sizes, "%d of %d outside" % (off.sum(), off.size), flush=True)
    assert not off.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[(1, 700), (2, 80)], [(30, 300), (1, 9)]])
@pytest.mark.parametrize("query,scale", [(0, 105), (10, 105), (60, 60), (-40, 60), (-89, 105), (-109, 119), (-20, 40)])
def test_products_up_to_the_stated_size(query, scale, sizes, dtype):
    """Queries of 2^query and key scales of 2^scale, products of up to 127 times as much, below
    2^(114 + query) (2^18 from 2^-96 down): each row is its best key's value.  Scores are exact multiples
    of 2^(query + scale) / sqrt(64), 2^10 and more apart after the factor of log2 e, so a rounding of one
    (2^-23 of 127 such steps) changes no order and every other weight is 0."""
    e = max(query, -96)
    assert query + scale + 7 <= 114 + e and query + scale >= 10
    nh, nkv, hd, ps = 8, 2, 64, 16
    rng = np.random.default_rng(abs(query) + scale)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    cache[0][...] = 128
    cache[0][..., 0] = rng.integers(1, 256, cache[0].shape[:3])
    cache[2][...] = np.float32(2.0 ** scale)
    rows = sum(r for r, _ in sizes)
    q = np.zeros((rows, nh, hd), np.float32)
    q[..., 0] = np.where(rng.random((rows, nh)) < 0.5, 1, -1) * np.float32(2.0 ** query)
    batch, starts = batch_of(table, sizes)
    got = host(bl.paged_attention(dev(q.reshape(rows, -1), DT[dtype]), bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]),
                                  batch)).reshape(rows, nh, hd)
    exp, _ = ref.attention(q, cache, table, sizes, starts, dtype == "bf16")
    # equal best keys are averaged: weights off by the parts (2^-11 where they are one), sums of n terms
    most = 0.032 * 127
    tol = (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24) * np.abs(exp) \
        + ((2.0 ** -11 if dtype == "bf16" else 2.0 ** -22) + 800 * 2.0 ** -24) * most
    assert np.isfinite(got).all() and (np.abs(got - exp) <= tol).all()


@pytest.mark.parametrize("sizes", [[(1, 700), (2, 80)], [(30, 300), (1, 9)]])
@pytest.mark.parametrize("ratio", [4, 8, 20])
def test_a_large_value_scale_that_weighs_nothing(ratio, sizes):
    """Each sequence's first key has a value scale 2^ratio times the others' largest and a score so
    low that its weight is 0.  Of the others at most 2^-33 of that scale is lost, of 127 codes each, beside
    the ordinary error, which goes by their own sizes."""
    nh, nkv, hd, ps = 8, 2, 64, 16
    rng = np.random.default_rng(ratio)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    rows = sum(r for r, _ in sizes)
    q = (rng.standard_normal((rows, nh, hd)) * 0.5).astype(np.float32)
    q[..., 0] = 8
    for s in range(len(sizes)):
        cache[0][table[s, 0], :, 0] = 128
        cache[0][table[s, 0], :, 0, 0] = 1  # the product is -127 * 8 times its scale
        cache[2][table[s, 0], :, 0] = 4.0   # a score of -508: e^-400 of the others' at most
    batch, starts = batch_of(table, sizes)
    low = [x.copy() for x in cache]
    big = np.float32(0.032 * 2.0 ** ratio)
    for s in range(len(sizes)):
        cache[3][table[s, 0], :, 0] = big
        low[3][table[s, 0], :, 0] = 0.0
    got = host(bl.paged_attention(dev(q.reshape(rows, -1)), bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]), batch))
    exp, bound = ref.attention(q, low, table, sizes, starts, False)
    n = max(r + p for r, p in sizes)
    off = np.abs(got.reshape(exp.shape) - exp)
    assert (off <= bound + n * 127 * 2.0 ** -33 * big).all()
    assert ratio > 8 or (off <= 2 * bound).all()
