"""GPU tests of the batched serving ops at the sizes that take their larger forms: appends of
many rows, 128-row tiles, merges of more than eight chunks, chunks of more than 1024 keys."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import serve_ref as ref
from launches import launched
from test_gpu_serve import (DEV, DT, batch_of, check_attention, check_sample, dev, host, rope, same,
                            test_append_writes_the_oracles_codes_and_nothing_else as check_append)

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


# ------------------------------------------------------------------ append

# rows * (heads + 2 kv heads) > 8192 and at least 8 rows a sequence: k and v by groups of 16
# positions.  Runs that begin and end anywhere in a group, of one row, of none.
RUNS = [
    # (heads, kv heads, hd, page, [(rows, pos)])
    (6, 2, 64, 16, [(380, 5), (0, 7), (300, 77), (1, 31), (333, 50), (1, 32)]),
    (32, 8, 128, 64, [(150, 13), (61, 120)]),
    (3, 1, 16, 48, [(390, 1), (17, 47), (399, 0), (398, 2), (15, 33), (385, 15), (40, 8)]),
    (10, 2, 80, 32, [(256, 16), (14, 2), (331, 69)]),
    (9, 9, 112, 256, [(309, 3), (2, 14)]),  # an odd number of heads: a wave of no q head
    (5, 1, 32, 16, [(160 + i, i) for i in range(8)]),
]
# as many rows of fewer than 8 a sequence: several heads a wave
SHORT = [
    (32, 8, 128, 16, [(1, i) for i in range(180)]),
    (10, 2, 80, 64, [(1 + i % 3, 2 * i) for i in range(190)] + [(0, 0)] * 3 + [(7, 45)] * 32),
    (7, 7, 48, 32, [(3, i) for i in range(135)]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", RUNS + SHORT)
def test_append_of_many_rows(nh, nkv, hd, ps, sizes, dtype):
    rows = sum(r for r, _ in sizes)
    assert rows * (nh + 2 * nkv) > 8192 and (rows + 5 >= 8 * len(sizes)) == ((nh, nkv, hd, ps, sizes) in RUNS)
    check_append(nh, nkv, hd, ps, sizes, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_of_runs_leaves_out_what_the_device_refuses(dtype):
    """Refused sequences, pages outside the pool and the end of the RoPE table among long runs: what
    the appends of a few rows at a time do."""
    nh, nkv, hd, ps = 8, 2, 64, 32
    sizes = [(300, 9), (250, -2), (310, 0), (400, 0), (1, 210), (200, 215), (60, 401)]
    rng = np.random.default_rng(2)
    table, n_pages = ref.pages_for([(r, max(p, 0)) for r, p in sizes], ps, rng, wide_extra=0)
    table[0, 3], table[2, 1], table[2, 8] = -1, n_pages, 2 ** 31 - 1
    max_rows, max_len, length = 390, 460, 303  # the fourth has too many rows, the last too many tokens
    rows = sum(r for r, _ in sizes)
    q, k, v = (dev(rng.standard_normal((rows, n * hd)).astype(np.float32), DT[dtype]) for n in (nh, nkv, nkv))
    _, _, dc, ds = rope(hd, length)
    caches, outs = [], []
    for few in (False, True):
        cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
        for t, x in ((cache.k, 7), (cache.v, 9), (cache.k_scale, 0.5), (cache.v_scale, 0.25)):
            t.fill_(x)
        batch, starts = batch_of(table, sizes, max_rows=max_rows, max_len=max_len)
        out = torch.full_like(q, 5)
        if not few:
            bl.paged_rope_append(q, k, v, cache, batch, dc, ds, q_out=out)
        else:
            for s, (r, p) in enumerate(sizes):
                for a in range(0, r, 50):
                    n = min(50, r - a)
                    at = slice(starts[s] + a, starts[s] + a + n)
                    # a refused sequence's pieces keep what it is refused for
                    refused = p < 0 or r > max_rows or r + p > max_len
                    one = bl.PagedBatch(dev(np.array([0, n], np.int32)), dev(np.array([-1 if refused else p + a], np.int32)),
                                        dev(table[s:s + 1]), n, n, max_len)
                    bl.paged_rope_append(q[at], k[at], v[at], cache, one, dc, ds, q_out=out[at])
        caches.append([t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
        outs.append(host(out))
    same(outs[0], outs[1], "q")
    for a, b in zip(*caches):
        assert torch.equal(a, b)
    lost = np.zeros(rows, bool)
    for s, (r, p) in enumerate(sizes):
        lost[starts[s]:starts[s] + r] = s in (1, 3, 6) or (p + np.arange(r) >= length)
    assert np.array_equal(np.isnan(outs[0]).all(1), lost) and np.array_equal(np.isnan(outs[0]).any(1), lost)


def test_append_of_millions_of_rows():
    """One sequence near the most tokens that a sequence may have: past 2^24 heads the append is by
    rows again.  The same bytes as in pieces that go by groups."""
    nh, nkv, hd, ps, n = 1, 1, 16, 65536, 5_600_000
    assert n * (nh + 2 * nkv) >= 2 ** 24 > 1_000_000 * (nh + 2 * nkv)
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn((n, hd), generator=g, device=DEV) for _ in range(3))
    angle = torch.rand((n, hd // 2), generator=g, device=DEV) * 6
    dc, ds = angle.cos(), angle.sin()
    pages = -(-n // ps)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(DEV)[None]
    i32 = dict(dtype=torch.int32, device=DEV)
    caches, outs = [], []
    for step in (n, 1_000_000):
        cache = bl.PagedKVCacheQ8(pages, ps, nkv, hd, DEV)
        out = torch.empty_like(q)
        for a in range(0, n, step):
            m = min(step, n - a)
            batch = bl.PagedBatch(torch.tensor([0, m], **i32), torch.tensor([a], **i32), table, m, m, n)
            bl.paged_rope_append(q[a:a + m], k[a:a + m], v[a:a + m], cache, batch, dc, ds, q_out=out[a:a + m])
        caches.append(cache)
        outs.append(out)
    assert torch.equal(*outs)
    for x in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0], x), getattr(caches[1], x))
    x1, x2 = q[:, :hd // 2], q[:, hd // 2:]
    assert torch.equal(outs[0], torch.cat((x1 * dc - x2 * ds, x1 * ds + x2 * dc), 1))
    _, vr = bl.paged_read(caches[0], bl.PagedBatch(torch.tensor([0, n], **i32), torch.tensor([0], **i32), table, n))
    # a code is the nearest: half a step, 1 / 254 of the largest value, and the roundings of x / s and code * s
    assert bool(((vr - v).abs() <= v.abs().amax(1, keepdim=True) * (0.5 / 127 + 2.0 ** -22)).all())


# ------------------------------------------------------------------ attention

# rows * heads >= 96 * 128: tiles of 128 query rows in 16 bits
TILES = [
    (8, 2, 64, 32, [(1537, 100)]),
    (16, 2, 128, 64, [(500, 300), (269, 3), (1, 50)]),
    (48, 8, 80, 48, [(257, 40)]),
    (16, 16, 32, 16, [(640, 0), (130, 77)]),
    (12, 4, 96, 16, [(900, 500), (0, 3), (129, 0)]),
    (32, 2, 16, 256, [(17, 9), (380, 250)]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", TILES)
def test_attention_of_many_rows(nh, nkv, hd, ps, sizes, dtype):
    assert sum(r for r, _ in sizes) * nh >= 96 * 128
    check_attention(nh, nkv, hd, ps, sizes, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", [
    (8, 2, 64, 64, [(1, 2599)]),             # eleven chunks of 256
    (8, 2, 128, 64, [(1, 2304), (1, 2303), (1, 255), (1, 256), (3, 2558)]),
    (4, 4, 16, 16, [(2, 5000)]),
    (8, 2, 80, 32, [(30, 2600)]),            # the tile form
    (8, 2, 128, 32, [(20, 2290), (1, 2700), (17, 0)]),
])
def test_attention_of_many_chunks(nh, nkv, hd, ps, sizes, dtype):
    check_attention(nh, nkv, hd, ps, sizes, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [
    [(1, 3000), (2, 2900), (1, 5), (1, 2303)],  # the token form, chunks of 2304 keys
    [(200, 2500)],                              # the tile form, one chunk of all keys
    [(150, 2500), (60, 1100), (1, 2400)],       # both
])
def test_attention_of_long_chunks(sizes, dtype):
    """The host's bound on the lengths, far above them, makes chunks of more than 1024 keys."""
    check_attention(8, 2, 32, 65536, sizes, dtype, max_len=131072)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_thousands_of_sequences(dtype):
    """More than 64 * 64 of them: the search for a row's sequence takes a third step."""
    sizes = [(1 + (i % 97 == 0), 1 + i % 11) if i % 5 else (0, 3) for i in range(4500)] + [(0, 0)] * 3
    check_append(2, 1, 16, 16, sizes, dtype)
    check_attention(2, 1, 16, 16, sizes, dtype)
    sizes[4321] = (30, 50)  # a tile of one among them
    check_attention(2, 1, 16, 16, sizes, dtype)


@pytest.mark.parametrize("rows,dtype", [(1, "f32"), (1, "bf16"), (21, "f32"), (21, "bf16")])
def test_attention_over_the_most_tokens(rows, dtype):
    """2^23 tokens, the most that a sequence may have, and one more, which is refused.

    Sums of weights: a lane's 16 keys a step over at most 66 steps of a chunk, then lanes, waves and some
    512 chunks, 64 a set: below 1200 additions in a row, each off by 2^-24, above and below the line; scores
    off as in serve_ref.attention; weights in bf16 tiles by 2^-11.  Values lie on one side of 0, so every
    chunk counts: one that is left out moves the result by a five hundredth of itself."""
    nh = nkv = 1
    hd, ps, n = 16, 65536, 2 ** 23
    g = torch.Generator(device=DEV).manual_seed(3)
    pages = n // ps
    cache = bl.PagedKVCacheQ8(pages, ps, nkv, hd, DEV)
    cache.k.random_(1, 256, generator=g)
    cache.v.random_(160, 256, generator=g)
    cache.k_scale.uniform_(0.002, 0.032, generator=g)
    cache.v_scale.uniform_(0.002, 0.032, generator=g)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(4)).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    q = (torch.randn((rows, hd), generator=g, device=DEV) * 2).to(DT[dtype])
    batch = bl.PagedBatch(torch.tensor([0, rows], **i32), torch.tensor([n - rows], **i32),
                          order.to(torch.int32)[None].contiguous(), rows)
    got = bl.paged_attention(q, cache, batch).double()
    k = (cache.k[order].view(n, hd).double() - 128) * cache.k_scale[order].view(n, 1).double()
    v = cache.v[order].view(n // 16, hd, 16).transpose(1, 2).reshape(n, hd).double() - 128
    v = v * cache.v_scale[order].view(n, 1).double()
    u = 2.0 ** -24
    for i in range(rows):
        seen = n - rows + i + 1
        x = q[i].double()
        sc = (k[:seen] * x).sum(1) / hd ** 0.5
        size = float((k[:seen].abs() * x.abs()).sum(1).max()) / hd ** 0.5
        w = torch.softmax(sc, 0)
        e = (w[:, None] * v[:seen]).sum(0)
        rel = 2 * ((2.0 ** -22 + (hd + 4) * u) * size + 6 * u * size) + 2 * 1200 * u \
            + (2.0 ** -11 if dtype == "bf16" and rows > 16 else 2.0 ** -22) + (2.0 ** -8 if dtype == "bf16" else u)
        off = float(((got[i] - e).abs() / e).max())
        print("most tokens", rows, dtype, i, "off by %.3g of %.3g" % (off, rel), flush=True)
        assert off <= rel
    past = bl.PagedBatch(batch.row_start, torch.tensor([n - rows + 1], **i32), batch.pages, rows)
    assert bool(torch.isnan(bl.paged_attention(q, cache, past)).all())


# ------------------------------------------------------------------ sampling

def test_sample_of_the_longest_rows():
    """2^22 logits: running weights up to 2^62, every token alike, and rows with a spread."""
    n = 2 ** 22
    u = np.array([0.0, 0.25, 0.7, 1 - 2.0 ** -24], np.float32)
    ids, probs = bl.sample(torch.zeros((4, n), device=DEV), dev(u))
    # floor(u W) of W = 2^62, over 2^40 a token
    assert ids.tolist() == [int(float(x) * 2 ** 62) >> 40 for x in u] and probs.tolist() == [2.0 ** -22] * 4
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((2, n)) * 1.5).astype(np.float32)
    check_sample(logits, t=[0.9, 1.0], p=[0.95, 1.0], k=[0, 3000000], u=[0.93, 0.9999])


# ------------------------------------------------------------------ which form runs

def step_of(nh, nkv, hd, ps, sizes, dtype, max_len=None):
    rng = np.random.default_rng(0)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    batch, starts = batch_of(table, sizes, max_len=max_len)
    q, k, v = (torch.zeros((int(starts[-1]), n * hd), dtype=DT[dtype], device=DEV) for n in (nh, nkv, nkv))
    _, _, dc, ds = rope(hd, 400)
    out, space = torch.empty_like(q), bl.paged_attention_workspace(cache, batch, nh)
    return (lambda: bl.paged_rope_append(q, k, v, cache, batch, dc, ds, q_out=q),
            lambda: bl.paged_attention(q, cache, batch, out=out, workspace=space))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_larger_forms_are_the_ones_that_run(dtype):
    """The cases above are here for these kernels: a rule that moves past them shows here."""
    bf = int(dtype == "bf16")

    def has(f, name):
        return any(name in n for n in launched(f))
    for case in RUNS:
        assert has(step_of(*case, dtype)[0], "k_paged_append_runs"), case
    for case in SHORT:
        assert has(step_of(*case, dtype)[0], "k_paged_appendILb%dELi6E" % bf), case
    for case in TILES:
        tiles = -(-case[2] // 32) * 2  # of 16 values, in twos
        assert has(step_of(*case, dtype)[1], "k_paged_tileILi%dELi%dELb%dE" % (tiles, 1 + bf, bf)), case
    assert has(step_of(8, 2, 64, 64, [(1, 2599)], dtype)[1], "k_paged_mergeILi4E")
    assert has(step_of(8, 2, 80, 32, [(30, 2600)], dtype)[1], "k_paged_mergeILi4E")
