"""GPU tests of paged attention over batches in which sequences break a bound of the call:
their rows are NaN, and every other sequence's are what they are without them."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import serve_ref as ref
from test_gpu_serve import DEV, DT, batch_of, dev, host

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

REFUSED = [
    # (heads, kv heads, hd, most rows, most tokens, [(rows, pos)], the sequences that break a bound)
    # 64-row tiles: more rows than the bound allows, ahead of others, between them, behind them
    (8, 2, 64, 20, 500, [(980, 0), (20, 5)], [0]),
    (8, 2, 64, 20, 500, [(40, 0), (20, 3), (20, 40)], [0]),
    (8, 2, 64, 20, 900, [(20, 0), (300, 7), (1, 30), (20, 700), (90, 0)], [1, 4]),
    # one row more than the bound; tokens past theirs; a position below 0; beside single tokens
    (8, 2, 96, 33, 400, [(34, 0), (33, 100), (1, 399), (33, 368), (1, 400), (5, -1), (33, 367)], [0, 3, 4, 5]),
    # every sequence refused but the last; a group of one
    (4, 4, 32, 17, 300, [(200, 0), (18, 0), (70, 5), (17, 80)], [0, 1, 2]),
    # rows enough for tiles of 128 in 16 bits
    (8, 2, 128, 100, 600, [(1500, 0), (100, 3), (7, 560), (100, 500)], [0]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,max_rows,max_len,sizes,refused", REFUSED)
def test_a_refused_sequence_costs_no_other_its_rows(nh, nkv, hd, max_rows, max_len, sizes, refused, dtype):
    print("refused", nh, nkv, hd, max_rows, max_len, sizes, dtype, flush=True)
    rng = np.random.default_rng(hd + len(sizes))
    ps = 32
    table, n_pages = ref.pages_for([(r, max(p, 0)) for r, p in sizes], ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    rows = sum(r for r, _ in sizes)
    q = (rng.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    if dtype == "bf16":
        q = ref.bf16_round(q)
    batch, starts = batch_of(table, sizes, max_rows=max_rows, max_len=max_len)
    paged = bl.PagedKVCacheQ8.of(*[dev(x) for x in cache])
    dq = dev(q.reshape(rows, -1), DT[dtype])
    # a workspace that holds no numbers of an earlier call
    space = bl.paged_attention_workspace(paged, batch, nh)
    space.buf.fill_(0x7F)
    got = host(bl.paged_attention(dq, paged, batch, out=torch.full_like(dq, 3), workspace=space)).reshape(q.shape)
    taken = [(0 if s in refused else r, p) for s, (r, p) in enumerate(sizes)]
    exp, bound = ref.attention(q, cache, table, taken, starts, dtype == "bf16")
    for s, (r, _) in enumerate(sizes):
        a = slice(starts[s], starts[s] + r)
        if s in refused:
            assert np.isnan(got[a]).all(), "sequence %d is refused" % s
        else:
            off = np.abs(got[a] - exp[a]) / bound[a]
            assert np.isfinite(got[a]).all() and off.max() <= 1.0, "sequence %d: %g of the bound" % (s, off.max())
