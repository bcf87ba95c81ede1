"""GPU tests of paged attention over scales that are not finite: a row that sees one is NaN
in every head of the key's KV head and every value, and no other row is touched."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import serve_ref as ref
from test_gpu_serve import DEV, DT, batch_of, dev, host, rope, same

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

INF, NAN = np.inf, np.nan
SCALES = [(INF, 1.0), (-INF, 1.0), (NAN, 1.0), (1.0, INF), (1.0, -INF), (1.0, NAN), (INF, INF), (0.0, INF), (INF, 0.0)]
FORMS = [
    # (heads, kv heads, hd, [(rows, pos)], position of the bad key of sequence 0)
    (8, 2, 64, [(1, 70), (1, 90)], 33),            # the token form, a step in which every row sees every key
    (8, 2, 64, [(4, 70), (2, 90)], 72),            # the same, a key that rows 0 and 1 do not see
    (8, 2, 80, [(1, 1300), (1, 2)], 1100),         # the same in chunks
    (8, 2, 64, [(40, 130), (1, 90)], 20),          # the tile form, a step in which every row sees every key
    (8, 2, 96, [(40, 30), (20, 90)], 55),          # the same, a key that rows up to 24 do not see
    (8, 2, 128, [(30, 1300), (20, 90)], 1310),     # the same in chunks
    (16, 2, 128, [(800, 100), (1, 9)], 300),       # tiles of 128 rows in 16 bits
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,sizes,at", FORMS)
def test_a_seen_scale_that_is_not_finite_is_nan(nh, nkv, hd, sizes, at, dtype):
    ps, g = 32, nh // nkv
    rng = np.random.default_rng(hd + at)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    rows = sum(r for r, _ in sizes)
    q = (rng.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    dq = dev(q.reshape(rows, -1), DT[dtype])
    batch, _ = batch_of(table, sizes)
    clean = host(bl.paged_attention(dq, bl.PagedKVCacheQ8.of(*[dev(x) for x in cache]), batch)).reshape(q.shape)
    assert np.isfinite(clean).all()
    r, p = sizes[0]
    sees = np.zeros((rows, nh), bool)
    head = 1  # the key's KV head; the other's rows stay as they are
    sees[max(0, at - p):r, head * g:(head + 1) * g] = True
    for ks, vs in SCALES:
        print("scales", nh, nkv, hd, sizes, at, dtype, ks, vs, flush=True)
        bad = [x.copy() for x in cache]
        bad[2][table[0, at // ps], head, at % ps] = ks
        bad[3][table[0, at // ps], head, at % ps] = vs
        got = host(bl.paged_attention(dq, bl.PagedKVCacheQ8.of(*[dev(x) for x in bad]), batch)).reshape(q.shape)
        assert np.isnan(got[sees]).all(), (ks, vs, int(np.isfinite(got[sees]).sum()), int(np.isinf(got[sees]).sum()))
        same(got[~sees], clean[~sees], "rows that do not see it")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[(40, 8)], [(1, 47)]])
def test_an_appended_infinity_is_nan_for_the_rows_that_see_it(sizes, dtype):
    """A key, or a value, with one infinite element: its scale is infinite and its code 0, whatever its sign."""
    nh, nkv, hd, ps, n, at = 8, 2, 64, 16, 48, 20
    rng = np.random.default_rng(7)
    _, _, dc, ds = rope(hd, 64)
    table, n_pages = ref.pages_for([(n, 0)], ps, rng)
    rows, pos = sizes[0]
    q = dev(rng.standard_normal((n, nh * hd)).astype(np.float32), DT[dtype])
    k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
    for which in ("k", "v"):
        for bad in (INF, -INF):
            x = dict(k=k.copy(), v=v.copy())
            x[which][at, 0, 3] = bad
            cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
            rot = bl.paged_rope_append(q, dev(x["k"].reshape(n, -1), DT[dtype]), dev(x["v"].reshape(n, -1), DT[dtype]),
                                       cache, batch_of(table, [(n, 0)])[0], dc, ds)
            scale = host(cache.k_scale if which == "k" else cache.v_scale)
            assert scale[table[0, at // ps], 0, at % ps] == INF
            out = bl.paged_attention(rot[n - rows:], cache, batch_of(table, sizes)[0])
            got = host(out).reshape(rows, nkv, nh // nkv, hd)
            sees = pos + np.arange(rows) >= at
            assert np.isnan(got[sees, 0]).all(), (which, bad)
            assert np.isfinite(got[~sees]).all() and np.isfinite(got[:, 1]).all()
