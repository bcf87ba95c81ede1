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
