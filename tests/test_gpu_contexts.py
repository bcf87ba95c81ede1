"""GPU tests of what long contexts ask for (include/bitserve.h): attention beside a shared
prefix, accounted weights, eviction, rows at shifted RoPE positions, and a run of them
together, against plain implementations in 64 bits (context_ref.py).

Attention and weights are held to the bounds that context_ref derives; what eviction moves is
compared bit for bit."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_gpu_serve import DEV, DT, batch_of, dev, host, rope, same

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


def lists_of(lists, ps, rng, n_pages, rows, max_rows=None, max_len=None):
    """A prefix: (PagedBatch, page table, pages in the pool with it); its pages come behind n_pages."""
    table, more = ref.pages_for([(0, n) for _, _, n in lists], ps, rng, extra=0)
    table = np.where(table >= 0, table + n_pages, -1).astype(np.int32)
    # rows of no list lie between lists only where a list of none stands for them
    starts = np.array([f for f, _, _ in lists] + [lists[-1][0] + lists[-1][1]], np.int32)
    p = bl.PagedBatch(dev(starts), dev(np.array([n for _, _, n in lists], np.int32)), dev(table), rows,
                      max(c for _, c, _ in lists) if max_rows is None else max_rows,
                      max(n for _, _, n in lists) if max_len is None else max_len)
    return p, table, n_pages + more


def on_gpu(cache):
    return bl.PagedKVCacheQ8.of(*[dev(x) for x in cache])


def within(got, want, bound, what=""):
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= bound).all(), "%s: %.3g over the bound, %d of %d" % (
        what, (off / np.maximum(bound, 1e-300)).max(), (off > bound).sum(), off.size)


# (heads, kv heads, hd, page, [(rows, pos)], [(first row, rows, prefix length)])
PREFIXES = [
    (1, 1, 16, 16, [(1, 0)], [(0, 1, 1)]),
    (4, 2, 64, 16, [(1, 5), (1, 0), (1, 33)], [(0, 3, 70)]),
    # lists of one to many rows, one of no positions, rows behind the last list
    (8, 2, 64, 32, [(1, 20), (1, 3), (2, 40), (1, 100), (1, 7), (1, 1)], [(0, 2, 300), (2, 2, 0), (4, 1, 15)]),
    # one list over many tokens: the tile form; lengths that end in no page, step or chunk
    (32, 8, 128, 64, [(1, 3 * n) for n in range(24)], [(0, 24, 1001)]),
    (16, 1, 128, 48, [(1, 0), (1, 31)], [(0, 2, 777)]),       # a group of 16: two rows are 32
    (5, 5, 80, 16, [(40, 0), (3, 20)], [(0, 43, 130)]),       # prompts behind a prefix
    (10, 2, 96, 16, [(33, 64), (1, 130), (7, 7)], [(0, 20, 65), (20, 21, 257)]),  # a list ends inside a sequence
    (8, 2, 112, 256, [(70, 0)], [(0, 70, 2049)]),             # chunks of the prefix
    (12, 4, 48, 32, [(2, 600), (1, 511), (1, 512)], [(0, 4, 512)]),               # chunks of both
    (3, 1, 32, 16, [(0, 9), (1, 0), (0, 0), (150, 3)], [(0, 151, 64)]),           # sequences without rows
    (4, 2, 16, 128, [(1, 40), (1, 3000)], [(0, 1, 6001), (1, 1, 5)]),             # many chunks of few tokens
    (32, 8, 128, 64, [(395, 30), (5, 100)], [(0, 400, 330)]),                     # tiles of 128 rows in bf16
    (2, 2, 64, 16, [(9, 2)], [(0, 3, 40), (3, 0, 9), (3, 6, 80)]),                # a list without rows
    (6, 2, 48, 32, [(1, 9 * n) for n in range(11)], [(0, 7, 700), (7, 1, 300), (8, 2, 31)]),  # tiles of 16 rows: 21 of 32
    (16, 2, 128, 16, [(2, 30), (2, 0)], [(0, 4, 1500)]),                          # two full ones
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(PREFIXES)))
def test_attention_beside_a_prefix(case, dtype):
    nh, nkv, hd, ps, sizes, lists = PREFIXES[case]
    print("prefix", PREFIXES[case][:4], dtype, flush=True)
    rng = np.random.default_rng(case)
    table, n_own = ref.pages_for(sizes, ps, rng)
    rows = sum(r for r, _ in sizes)
    prefix, ptable, n_pages = lists_of(lists, ps, rng, n_own, rows + 2)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    batch, starts = batch_of(table, sizes, rows=rows + 2)
    q = dev(rng.standard_normal((rows + 2, nh * hd)).astype(np.float32) * 2, DT[dtype])
    out = torch.full_like(q, 7)
    got = bl.paged_attention_prefix(q, on_gpu(cache), batch, prefix, out=out)
    assert got is out and (out[rows:] == 7).all()  # rows of no sequence
    want, bound, _, _ = cref.attention(host(q)[:rows].reshape(rows, nh, hd), cache, table, sizes, starts, dtype == "bf16",
                                       lists, ptable)
    within(host(got)[:rows].reshape(rows, nh, hd), want, bound)
    again = bl.paged_attention_prefix(q, on_gpu(cache), batch, prefix,
                                      workspace=bl.paged_attention_prefix_workspace(on_gpu(cache), batch, prefix, nh))
    assert torch.equal(again[:rows], got[:rows])


def test_a_prefix_that_is_part_of_every_sequence():
    """The same contexts as one page table a sequence: the outputs of paged_attention."""
    nh, nkv, hd, ps, n, own, shared = 8, 2, 64, 16, 5, 21, 96
    rng = np.random.default_rng(3)
    table, n_own = ref.pages_for([(1, own - 1)] * n, ps, rng)
    prefix, ptable, n_pages = lists_of([(0, n, shared)], ps, rng, n_own, n)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    gpu = on_gpu(cache)
    whole = np.concatenate([np.repeat(ptable[:, :shared // ps], n, axis=0), table], axis=1)
    q = dev(rng.standard_normal((n, nh * hd)).astype(np.float32))
    batch, starts = batch_of(table, [(1, own - 1)] * n)
    both, _ = batch_of(whole, [(1, shared + own - 1)] * n)
    a, b = bl.paged_attention_prefix(q, gpu, batch, prefix), bl.paged_attention(q, gpu, both)
    want, bound = ref.attention(host(q).reshape(n, nh, hd), cache, whole, [(1, shared + own - 1)] * n, starts, False)
    for x in (a, b):
        within(host(x).reshape(n, nh, hd), want, bound)


def test_lists_that_the_device_refuses():
    """NaN in the rows of the list, and the others as without it."""
    nh, nkv, hd, ps = 4, 2, 32, 16
    rng = np.random.default_rng(4)
    sizes = [(1, n) for n in (3, 17, 40, 8, 60, 1)]
    table, n_own = ref.pages_for(sizes, ps, rng)
    lists = [(0, 1, 30), (1, 1, 50), (2, 1, 20), (3, 2, 33), (5, 1, 16)]
    prefix, ptable, n_pages = lists_of(lists, ps, rng, n_own, 6)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    gpu = on_gpu(cache)
    batch, starts = batch_of(table, sizes)
    q = dev(rng.standard_normal((6, nh * hd)).astype(np.float32))
    good = host(bl.paged_attention_prefix(q, gpu, batch, prefix))
    want, bound, _, _ = cref.attention(host(q).reshape(6, nh, hd), cache, table, sizes, starts, False, lists, ptable)
    within(good.reshape(6, nh, hd), want, bound)
    pos = np.array([30, 51, -1, 33, 16], np.int32)  # one past max_len, one negative
    bad_table = ptable.copy()
    bad_table[4, 0] = n_pages                       # one past the pool
    bad = bl.PagedBatch(prefix.row_start, dev(pos), dev(bad_table), 6, 1, 50)  # list 3 has two rows
    account = bl.KVAccount(6, nkv, 64, DEV)
    for got in (host(bl.paged_attention_prefix(q, gpu, batch, bad)),
                host(bl.paged_attention_account(q, gpu, batch, account, prefix=bad))):
        assert np.isnan(got[1:]).all()
        same(got[:1], good[:1])
    w = host(account.weight)
    assert (w[1:] == 0).all() and (w[0, :, :4] > 0).all() and (w[0, :, 4:] == 0).all()


def test_row_starts_and_pages_of_anything():
    """Arrays that no caller should give: no row is written that is not the batch's."""
    nh, nkv, hd, ps = 4, 2, 32, 16
    rng = np.random.default_rng(5)
    table, n_own = ref.pages_for([(2, 10), (3, 40)], ps, rng)
    cache = ref.rand_cache(rng, n_own, nkv, ps, hd)
    batch, _ = batch_of(table, [(2, 10), (3, 40)], rows=6)
    q = dev(rng.standard_normal((6, nh * hd)).astype(np.float32))
    big = 2 ** 31 - 1
    for starts in ([-5, 3, big], [4, 2, 1], [big, big, big], [0, -big, 6]):
        prefix = bl.PagedBatch(dev(np.array(starts, np.int32)), dev(np.array([40, 17], np.int32)),
                               dev(np.array([[0, -1, n_own], [big, 1, -big]], np.int32)), 6, 6, 48)
        out = torch.full_like(q, 3)
        account = bl.KVAccount(2, nkv, 64, DEV)
        bl.paged_attention_account(q, on_gpu(cache), batch, account, prefix=prefix, out=out)
        assert (out[5:] == 3).all()


# (heads, kv heads, hd, page, [(rows, pos)], lists)
ACCOUNTS = [
    (1, 1, 16, 16, [(1, 0)], []),
    (4, 2, 64, 16, [(1, 0), (1, 15), (1, 64), (1, 255), (0, 40), (1, 256), (1, 300)], []),
    (32, 8, 128, 64, [(1, 776), (0, 3), (1, 1023), (2, 511)], []),
    (16, 1, 128, 32, [(1, 100), (1, 5)], []),
    (5, 5, 80, 48, [(16, 0), (3, 200), (17, 47)], []),         # 17 rows: the tile form beside the token form
    (10, 2, 96, 16, [(40, 0), (7, 77), (1, 130), (0, 0), (26, 250)], []),
    (8, 2, 112, 256, [(200, 60)], []),                         # one sequence: shares of its rows
    (8, 1, 32, 32, [(129, 0), (1, 400), (128, 384)], []),
    (12, 4, 48, 16, [(65, 511), (1, 1), (2, 700)], [(0, 65, 100), (65, 3, 31)]),
    (8, 2, 64, 32, [(1, 20), (1, 3), (2, 40), (1, 100)], [(0, 2, 300), (2, 2, 0)]),
    (2, 2, 128, 16, [(100, 1)], [(0, 50, 17)]),                # rows of no list
    (8, 2, 64, 128, [(1, 5003)], []),                          # many chunks
    (4, 2, 32, 64, [(2, 3100), (1, 7)], []),                   # of two rows, and of some
    (32, 8, 128, 64, [(390, 300), (20, 0)], [(0, 390, 150)]),  # tiles of 128 rows in bf16
    (15, 1, 112, 16, [(1, 200), (1, 0), (3, 64)], [(0, 2, 100)]),  # groups of 15
    # many rows, whose merges wait for nothing: of up to 8 chunks, up to 16, more
    (8, 2, 64, 64, [(40, 1500), (1, 33)], []),
    (8, 2, 64, 64, [(40, 2400), (1, 33)], []),
    (8, 2, 64, 64, [(40, 5000), (1, 33)], []),
    (80, 5, 16, 16, [(2, 700), (3, 10), (0, 9), (1, 600)], [(0, 5, 20)]),  # more heads than a wave has lanes
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(ACCOUNTS)))
def test_accounted_weights(case, dtype):
    nh, nkv, hd, ps, sizes, lists = ACCOUNTS[case]
    print("account", ACCOUNTS[case][:4], dtype, flush=True)
    rng = np.random.default_rng(100 + case)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    rows = sum(r for r, _ in sizes)
    prefix = ptable = None
    if lists:
        prefix, ptable, n_pages = lists_of(lists, ps, rng, n_pages, rows)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    batch, starts = batch_of(table, sizes)
    q = dev(rng.standard_normal((rows, nh * hd)).astype(np.float32) * 2, DT[dtype])
    ld = max(r + p for r, p in sizes) + 5
    before = (rng.random((len(sizes), nkv, ld)) * 2).astype(np.float32)
    # what a position of this call's rows held before is not looked at
    for s, (r, p) in enumerate(sizes):
        before[s, :, p:p + r] = np.nan
    account = bl.KVAccount.of(dev(before))
    got = bl.paged_attention_account(q, on_gpu(cache), batch, account, prefix=prefix)
    want, bound, w, wb = cref.attention(host(q).reshape(rows, nh, hd), cache, table, sizes, starts, dtype == "bf16", lists,
                                        ptable)
    within(host(got).reshape(rows, nh, hd), want, bound, "outputs")
    weight = host(account.weight).astype(np.float64)
    for s, (r, p) in enumerate(sizes):
        if r == 0:
            same(weight[s], before[s], "a sequence without rows")
            continue
        w[s][:, :p] += before[s, :, :p]
        within(weight[s, :, :r + p], w[s], wb[s] + cref.U * w[s], "weights of sequence %d" % s)
        same(weight[s, :, r + p:], before[s, :, r + p:], "behind the sequence")
    other = bl.KVAccount.of(dev(before))
    space = bl.paged_attention_account_workspace(on_gpu(cache), batch, nh, prefix=prefix)
    again = bl.paged_attention_account(q, on_gpu(cache), batch, other, prefix=prefix, workspace=space)
    assert torch.equal(again, got) and torch.equal(other.weight, account.weight)


def test_weights_of_bounds_far_above_the_lengths():
    """Scores are not kept where the bounds would make them a large workspace."""
    nh, nkv, hd, ps = 16, 1, 16, 65536
    rng = np.random.default_rng(9)
    sizes = [(1, 70), (1, 0), (1, 333)]
    table = np.full((3, 128), -1, np.int32)
    table[:, 0] = [1, 3, 0]
    cache = ref.rand_cache(rng, 4, nkv, ps, hd)
    batch, starts = batch_of(table, sizes, max_len=1 << 23)
    q = dev(rng.standard_normal((3, nh * hd)).astype(np.float32))
    account = bl.KVAccount(3, nkv, 1 << 23, DEV)
    got = bl.paged_attention_account(q, on_gpu(cache), batch, account)
    want, bound, w, wb = cref.attention(host(q).reshape(3, nh, hd), cache, table, sizes, starts, False)
    within(host(got).reshape(3, nh, hd), want, bound)
    for s, (r, p) in enumerate(sizes):
        within(host(account.weight[s, :, :r + p]), w[s], wb[s] + cref.U * w[s])
        assert (account.weight[s, :, r + p:] == 0).all()


def test_weights_beside_more_rows_than_a_grid_merges():
    """2^21 rows of 64 heads, all but two behind the last sequence: their merges alone are 2^24
    workgroups of 256 threads, one more than a grid has."""
    nh, nkv, hd, ps, rows = 64, 4, 16, 16, 1 << 21
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of free memory")
    rng = np.random.default_rng(12)
    sizes = [(1, 900), (1, 300)]
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    batch, starts = batch_of(table, sizes, rows=rows)
    q = torch.empty((rows, nh * hd), dtype=torch.bfloat16, device=DEV)
    q[:2] = dev(rng.standard_normal((2, nh * hd)).astype(np.float32), torch.bfloat16)
    out = torch.empty_like(q)
    out[2:4], out[-1] = 7, 7
    account = bl.KVAccount(2, nkv, 901, DEV)
    workspace = bl.paged_attention_account_workspace(on_gpu(cache), batch, nh)
    bl.paged_attention_account(q, on_gpu(cache), batch, account, out=out, workspace=workspace)
    assert (out[2:4] == 7).all() and (out[-1] == 7).all()
    want, bound, weights, wbounds = cref.attention(host(q[:2]).reshape(2, nh, hd), cache, table, sizes, starts, True)
    within(host(out[:2]).reshape(2, nh, hd), want, bound)
    for s, (r, p) in enumerate(sizes):
        within(host(account.weight)[s, :, :r + p], weights[s], wbounds[s] + cref.U * weights[s])



@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-30, 1e6, 1e12, 1e30])
def test_weights_of_scores_of_any_size(size, dtype, rows):
    """Scores whose roundings are far above one: each row's weights still are a softmax's, and of one
    key far above the others' all of it."""
    nh, nkv, hd, ps, pos = 4, 2, 64, 16, 100
    rng = np.random.default_rng(11)
    sizes = [(rows, pos)]
    table, n_pages = ref.pages_for(sizes, ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    batch, _ = batch_of(table, sizes)
    q = dev((rng.standard_normal((rows, nh * hd)) * size).astype(np.float32), DT[dtype])
    account = bl.KVAccount(1, nkv, pos + rows, DEV)
    out = host(bl.paged_attention_account(q, on_gpu(cache), batch, account))
    w = host(account.weight).astype(np.float64)
    assert np.isfinite(out).all() and np.isfinite(w).all() and (w >= 0).all()
    n = rows * nh // nkv  # softmaxes of a KV head, each 1 in all but for the roundings of its terms and sums
    assert np.abs(w.sum(axis=2) - n).max() <= n * (2 * (pos + rows) + n + 8) * cref.U
    if size >= 1e12:  # every softmax is one key's
        assert (np.abs(w - np.rint(w)) <= n * 8 * cref.U).all()


def test_what_a_mask_hides_and_rows_that_are_nan():
    """Infinities and NaN behind a sequence change nothing; a row that is NaN adds nothing."""
    nh, nkv, hd, ps = 4, 2, 64, 16
    rng = np.random.default_rng(12)
    for sizes, bad in (([(1, 20), (1, 40)], 0), ([(30, 20), (2, 40)], 5)):
        table, n_pages = ref.pages_for(sizes, ps, rng, wide_extra=0)
        rows = sum(r for r, _ in sizes)
        cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
        batch, starts = batch_of(table, sizes)
        q = rng.standard_normal((rows, nh * hd)).astype(np.float32)
        clean = bl.KVAccount(2, nkv, 80, DEV)
        a = bl.paged_attention_account(dev(q), on_gpu(cache), batch, clean)
        for s, (r, p) in enumerate(sizes):  # the slots behind the last position
            last = r + p - 1
            for j in range(last + 1, (last // ps + 1) * ps):
                for x in (2, 3):
                    cache[x][table[s, j // ps], :, j % ps] = [np.inf, np.nan]
        dirty = bl.KVAccount(2, nkv, 80, DEV)
        b = bl.paged_attention_account(dev(q), on_gpu(cache), batch, dirty)
        assert torch.equal(a, b) and torch.equal(clean.weight, dirty.weight)
        q[bad, :hd] = np.inf  # the first head of one row
        some = bl.KVAccount(2, nkv, 80, DEV)
        c = host(bl.paged_attention_account(dev(q), on_gpu(cache), batch, some))
        assert np.isnan(c[bad, :hd]).all() and np.isfinite(np.delete(c, bad, 0)).all() and np.isfinite(c[bad, hd:]).all()
        q[bad, :hd] = 0
        want, _, w, wb = cref.attention(q.reshape(rows, nh, hd), cache, table, sizes, starts, False)
        w[0][0, :sizes[0][1] + bad + 1] -= 1.0 / (sizes[0][1] + bad + 1)  # a row of zeros gives each the same
        for s, (r, p) in enumerate(sizes):
            within(host(some.weight[s, :, :r + p]), w[s], wb[s] + 4 * cref.U * (w[s] + 1))


# (kv heads, hd, page, [positions], [keep], sink, recent, filled before)
EVICTS = [
    (1, 16, 16, [1], [0], 0, 0, False),
    (2, 64, 16, [0, 5, 17, 33, 64], [3, 5, 16, 1, 63], 0, 0, False),
    (8, 128, 64, [700, 300, 1025, 64], [256, 299, 1024, 64], 4, 32, True),
    (2, 80, 48, [200, 201, 202], [-1, 500, 0], 2, 5, False),
    (1, 112, 32, [100, 90], [10, 20], 30, 40, True),          # more of them first than are kept
    (3, 96, 256, [2000, 1], [999, 1], 0, 2000, False),        # all of them among the last
    (1, 32, 128, [20000, 8192, 8193], [5000, 100, 8191], 4, 100, True),  # several spans
    (4, 48, 16, [50] * 7, [25] * 7, 0, 3, True),
    # spans: keep at their ends and beside them, whole and empty sequences among long ones, few that go
    (1, 16, 64, [30000, 24577, 16384, 8192, 100], [24576, 8192, 16383, 1, 50], 0, 0, False),
    (2, 32, 256, [9000, 20001, 0, 8200], [-1, 0, 5, 9000], 10, 7, True),
    (1, 16, 128, [50000], [49999], 3, 1000, True),
    (1, 16, 128, [40000, 40000], [8193, 33000], 20000, 9000, False),
    # both sizes of the workgroups that hold a head: the most of each, and one more than the smaller's
    (2, 32, 64, [8192, 4097, 8191, 40], [4096, 2049, 1, 8], 4, 50, True),
    (2, 48, 32, [4096, 4095, 3], [2048, 4094, 1], 4, 50, True),
    (1, 16, 128, [4097, 4096], [4096, 2048], 0, 0, False),
]


def random_account(rng, sizes, nkv, ld, keep, again):
    """Weights with equals, zeros, infinities, NaN and negatives among them; tokens in no order."""
    w = np.exp(2 * rng.standard_normal((len(sizes), nkv, ld))).astype(np.float32)
    w = np.where(rng.random(w.shape) < 0.4, np.round(w * 8) / 8, w).astype(np.float32)
    for x, v in ((0.03, 0.0), (0.02, -0.0), (0.02, np.nan), (0.02, np.inf), (0.02, -1.5), (0.01, -np.inf), (0.01, 1e-45)):
        w[rng.random(w.shape) < x] = v
    token = rng.integers(-5, 5, w.shape).astype(np.int32)
    filled = np.array([min(n, max(k, 0)) if again else 0 for n, k in zip(sizes, keep)], np.int32)
    shift = np.array([3 * n if again else 0 for n in range(len(sizes))], np.int32)
    for s in range(len(sizes)):
        for h in range(nkv):
            token[s, h, :filled[s]] = rng.permutation(filled[s] + shift[s])[:filled[s]]
    return w, token, filled, shift


def same_bits(got, want, what):
    g, w = np.ascontiguousarray(got), np.ascontiguousarray(want)
    assert g.dtype == w.dtype and g.shape == w.shape
    if g.dtype == np.float32:
        ok = (g.view(np.uint32) == w.view(np.uint32)) | (np.isnan(g) & np.isnan(w))
    else:
        ok = g == w
    assert ok.all(), "%s: %d of %d differ, first at %s" % (what, (~ok).sum(), ok.size, np.argwhere(~ok)[0])


def check_evict(cache, table, sizes, account, keep, sink, recent, ok=None, in_place=False, **batch):
    n = len(sizes)
    gpu = on_gpu(cache)
    b = bl.PagedBatch(dev(np.zeros(n + 1, np.int32)), dev(np.array(batch.get("pos", sizes), np.int32)), dev(table),
                      0, 0, batch.get("max_len", max(sizes)))
    acc = bl.KVAccount.of(*[dev(x) for x in account])
    rng = np.random.default_rng(0)
    start = [rng.integers(0, 9, x.shape).astype(x.dtype) for x in account]
    out = acc if in_place else bl.KVAccount.of(*[dev(x) for x in start])
    per = [dev(np.array(x, np.int32)) for x in (keep, sink, recent)]
    held = bl.paged_evict(gpu, b, acc, per[0], sink=per[1], recent=per[2], out=out, max_keep=batch.get("max_keep"))
    want_cache, want, want_held = cref.evict(cache, table, sizes, account, keep, sink, recent, ok)
    assert held.tolist() == want_held
    for name, g, w in zip(("k", "v", "k scale", "v scale"), (gpu.k, gpu.v, gpu.k_scale, gpu.v_scale), want_cache):
        same_bits(g.cpu().numpy(), w, name)
    got = [x.cpu().numpy() for x in (out.weight, out.token, out.filled, out.shift)]
    for i, name in enumerate(("weight", "token", "filled", "shift")):
        w = want[i].copy() if in_place else start[i]
        for s, left in enumerate(want_held):
            if left < 0:
                continue
            if i < 2:
                w[s, :, :left] = want[i][s, :, :left]
            else:
                w[s] = want[i][s]
        same_bits(got[i], w, name)
    if not in_place:  # what came in is as it was
        for t, x in zip((acc.weight, acc.token, acc.filled, acc.shift), account):
            same_bits(t.cpu().numpy(), x, "the account that came in")
    return gpu, b, acc, out


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_eviction(case, in_place):
    nkv, hd, ps, sizes, keep, sink, recent, again = EVICTS[case]
    print("evict", EVICTS[case], flush=True)
    rng = np.random.default_rng(200 + case)
    table, n_pages = ref.pages_for([(0, n) for n in sizes], ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    account = random_account(rng, sizes, nkv, max(sizes) + 3, keep, again)
    n = len(sizes)
    check_evict(cache, table, sizes, account, keep, [sink] * n, [recent] * n, in_place=in_place)


def test_eviction_of_equal_weights_keeps_the_first():
    rng = np.random.default_rng(7)
    sizes, keep = [9000, 300], [4000, 100]
    table, n_pages = ref.pages_for([(0, n) for n in sizes], 16, rng)
    cache = ref.rand_cache(rng, n_pages, 1, 16, 16)
    account = [np.full((2, 1, 9000), 0.25, np.float32), np.zeros((2, 1, 9000), np.int32), np.zeros(2, np.int32),
               np.zeros(2, np.int32)]
    gpu, _, _, out = check_evict(cache, table, sizes, account, keep, [0, 0], [0, 0])
    assert out.token[0, 0, :4000].tolist() == list(range(4000))
    check_evict(cache, table, sizes, account, keep, [0, 0], [50, 1])


def test_evictions_that_the_device_refuses():
    """A position out of bounds, keep above max_keep: held is -1 and nothing else changes; pages outside the
    pool: what would come from them has NaN scales, what would go to them is lost."""
    nkv, hd, ps = 2, 32, 16
    rng = np.random.default_rng(8)
    sizes, keep = [60, -3, 90, 50, 61, 64], [20, 5, 30, 41, 30, 20]
    table, n_pages = ref.pages_for([(0, max(n, 0)) for n in sizes], ps, rng)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    account = random_account(rng, [80] * 6, nkv, 90, [0] * 6, False)
    table[4, 0] = n_pages       # some of its first sixteen go
    table[4, 3] = -7            # its last stay
    account[0][4, :, 48:61] = 1e9
    table[5, 3] = 2 ** 31 - 1
    account[0][5, :, 48:64] = 1e9
    gpu, *_ = check_evict(cache, table, sizes, account, keep, [0] * 6, [0] * 6, ok=[True, False, False, False, True, True],
                          max_len=80, max_keep=40)
    assert torch.isnan(gpu.k_scale).any()


def test_an_eviction_leaves_positions_below_sink_where_they_are():
    """Sequences that share the pages of their first tokens may keep them by sink."""
    nkv, hd, ps, n = 2, 64, 16, 3
    rng = np.random.default_rng(13)
    table, n_pages = ref.pages_for([(0, 200)] * n, ps, rng)
    table[1:, :4] = table[0, :4]
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    account = random_account(rng, [200] * n, nkv, 200, [0] * n, False)
    gpu, *_ = check_evict(cache, table, [200] * n, account, [100] * n, [64] * n, [0] * n)
    first = table[0, :4]
    for t, x in zip((gpu.k, gpu.v, gpu.k_scale, gpu.v_scale), cache):
        same_bits(t.cpu().numpy()[first], x[first], "the shared pages")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,sizes", [
    (4, 2, 64, 16, [(1, 0), (3, 20)]),
    (32, 8, 128, 64, [(200, 30), (0, 5), (150, 0)]),   # by runs
    (6, 3, 80, 48, [(9, 40), (1, 7), (40, 0)]),
])
def test_append_at_shifted_rope_positions(nh, nkv, hd, ps, sizes, dtype):
    """The bytes of an append at the RoPE position, in the slots of the position."""
    rng = np.random.default_rng(hd)
    table, n_pages = ref.pages_for(sizes, ps, rng)
    rows = sum(r for r, _ in sizes)
    q, k, v = (dev(rng.standard_normal((rows, n * hd)).astype(np.float32), DT[dtype]) for n in (nh, nkv, nkv))
    _, _, dc, ds = rope(hd, 400)
    batch, starts = batch_of(table, sizes)
    shift = np.array([7, 300, 133][:len(sizes)], np.int32)
    shift[-1] = -sizes[-1][1] + 133
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    got = bl.paged_rope_append(q, k, v, cache, batch, dc, ds, rope_shift=dev(shift))
    kr, vr = bl.paged_read(cache, batch)
    moved = [(r, p + int(d)) for (r, p), d in zip(sizes, shift)]
    far, n_far = ref.pages_for(moved, ps, rng)
    other = bl.PagedKVCacheQ8(n_far, ps, nkv, hd, DEV)
    there, _ = batch_of(far, moved)
    want = bl.paged_rope_append(q, k, v, other, there, dc, ds)
    kw, vw = bl.paged_read(other, there)
    # rows past the table are NaN in both
    same(host(got), host(want), "q")
    inside = [starts[s] + i for s, (r, p) in enumerate(moved) for i in range(r) if p + i < 400]
    assert len(inside) >= rows - 50
    assert torch.equal(kr[inside], kw[inside]) and torch.equal(vr[inside], vw[inside])
    none = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    zero = bl.paged_rope_append(q, k, v, none, batch, dc, ds, rope_shift=dev(np.zeros(len(sizes), np.int32)))
    plain = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    same(host(zero), host(bl.paged_rope_append(q, k, v, plain, batch, dc, ds)))
    assert torch.equal(none.k, plain.k) and torch.equal(none.v, plain.v)


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("shift", [-2 ** 31, 2 ** 31 - 1, -12, 60])
def test_append_past_the_rope_table_stores_nothing(shift, rows):
    nh, nkv, hd, ps, pos, size = 32, 8, 32, 16, 10, 64
    rng = np.random.default_rng(1)
    table, n_pages = ref.pages_for([(rows, pos)], ps, rng)
    q, k, v = (dev(rng.standard_normal((rows, n * hd)).astype(np.float32)) for n in (nh, nkv, nkv))
    _, _, dc, ds = rope(hd, size)
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    cache.k_scale.fill_(-1)
    cache.v_scale.fill_(-1)
    batch, _ = batch_of(table, [(rows, pos)])
    out = host(bl.paged_rope_append(q, k, v, cache, batch, dc, ds, rope_shift=dev(np.array([shift], np.int32))))
    inside = [i for i in range(rows) if 0 <= pos + i + shift < size]
    assert np.isfinite(out[inside]).all() and np.isnan(np.delete(out, inside, 0)).all()
    want = {(int(table[0, (pos + i) // ps]), (pos + i) % ps) for i in inside}
    for t in (cache.k_scale, cache.v_scale):
        assert {(int(p), int(s)) for p, s in zip(*np.nonzero((host(t) >= 0).any(1)))} == want


def test_steps_within_a_budget_behind_a_shared_prompt():
    """Prompt pages shared by four answers; each step appends, attends, accounts and evicts, and is
    compared with a model of the cache in 64 bits; one graph of a step, replayed."""
    nh, nkv, hd, ps, n, prompt, budget = 8, 2, 64, 16, 4, 75, 24
    rng = np.random.default_rng(21)
    _, _, dc, ds = rope(hd, 400)
    per = 3  # pages of an answer: budget and the rows of a step
    n_pages = 5 + n * per
    cache = bl.PagedKVCacheQ8(n_pages, ps, nkv, hd, DEV)
    ptable = np.arange(5, dtype=np.int32)[None]
    table = (5 + rng.permutation(n * per)).reshape(n, per).astype(np.int32)
    # the prompt's keys, by one sequence
    first = bl.PagedBatch(dev(np.array([0, prompt], np.int32)), dev(np.zeros(1, np.int32)), dev(ptable), prompt)
    q, k, v = (dev(rng.standard_normal((prompt, m * hd)).astype(np.float32)) for m in (nh, nkv, nkv))
    bl.paged_rope_append(q, k, v, cache, first, dc, ds)
    pos = torch.zeros(n, dtype=torch.int32, device=DEV)
    batch = bl.PagedBatch(dev(np.arange(n + 1, dtype=np.int32)), pos, dev(table), n, 1, budget + 1)
    prefix = bl.PagedBatch(dev(np.array([0, n], np.int32)), dev(np.array([prompt], np.int32)), dev(ptable), n, n, prompt)
    account = bl.KVAccount(n, nkv, budget + 4, DEV, shift=prompt)
    keep, recent = (dev(np.full(n, x, np.int32)) for x in (budget, 4))
    held = torch.zeros_like(pos)
    spaces = (bl.paged_attention_account_workspace(cache, batch, nh, prefix=prefix), bl.paged_evict_workspace(cache, batch))
    qs, ks, vs = (torch.empty((n, m * hd), device=DEV) for m in (nh, nkv, nkv))
    qr, out = torch.empty_like(qs), torch.empty_like(qs)

    def step():
        bl.paged_rope_append(qs, ks, vs, cache, batch, dc, ds, q_out=qr, rope_shift=account.shift)
        bl.paged_attention_account(qr, cache, batch, account, prefix=prefix, out=out, workspace=spaces[0])
        bl.paged_evict(cache, batch, account, keep, recent=recent, max_keep=budget, held=held, workspace=spaces[1])
        pos.copy_(held)

    graph = None
    for t in range(60):
        new = [rng.standard_normal((n, m * hd)).astype(np.float32) for m in (nh, nkv, nkv)]
        for x, y in zip((qs, ks, vs), new):
            x.copy_(torch.from_numpy(y))
        was = [x.cpu().numpy().copy() for x in (account.weight, account.token, account.filled, account.shift, pos)]
        size = min(t, budget)
        assert was[4].tolist() == [size] * n and was[3].tolist() == [prompt + max(0, t - budget)] * n
        if t == 30:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        if t in (0, 1, 5, 23, 24, 25, 29, 30, 31, 45, 59):
            # the rows' rotation is at the token's number
            lone = bl.PagedKVCacheQ8(n * 30, ps, nkv, hd, DEV)
            far = bl.PagedBatch(dev(np.arange(n + 1, dtype=np.int32)), torch.full_like(pos, prompt + t),
                                dev(np.arange(n * 30, dtype=np.int32).reshape(n, 30)), n, 1)
            same(host(qr), host(bl.paged_rope_append(qs, ks, vs, lone, far, dc, ds)), "q")
            # outputs against what the step's attention saw: the cache before its eviction, known from the sources
            now = [x.cpu().numpy() for x in (account.token, account.filled, account.shift)]
            assert now[1].tolist() == [min(t + 1, budget)] * n and now[2].tolist() == [prompt + max(0, t + 1 - budget)] * n
            for s in range(n):
                for h in range(nkv):
                    mine = now[0][s, h, :now[1][s]].tolist()
                    assert len(set(mine)) == len(mine) and set(range(prompt + max(0, t - 3), prompt + t + 1)) <= set(mine)
        assert torch.isfinite(out).all()
    # the last attention again, from the cache as it is: the tokens held, each head's own
    sizes = [(1, budget - 1)] * n
    last = bl.PagedBatch(dev(np.arange(n + 1, dtype=np.int32)), torch.full_like(pos, budget - 1), dev(table), n, 1, budget)
    fresh = bl.KVAccount(n, nkv, budget, DEV)
    got = bl.paged_attention_account(qr, cache, last, fresh, prefix=prefix)
    arrays = [x.cpu().numpy() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    want, bound, w, wb = cref.attention(host(qr).reshape(n, nh, hd), arrays, table, sizes, list(range(n)), False,
                                        [(0, n, prompt)], ptable)
    within(host(got).reshape(n, nh, hd), want, bound)
    for s in range(n):
        within(host(fresh.weight[s]), w[s], wb[s] + cref.U * w[s])


def test_calls_on_a_stream_and_in_two_graphs_of_one_workspace():
    """Another stream than the current one's default, and two captured calls that share a workspace,
    replayed in turn with other lengths and pages."""
    nh, nkv, hd, ps, n = 8, 2, 64, 16, 3
    rng = np.random.default_rng(31)
    tables = [ref.pages_for([(1, 90)] * n, ps, rng, wide_extra=0)[0] for _ in range(2)]
    n_pages = int(max(t.max() for t in tables)) + 1
    ptable = np.arange(6, dtype=np.int32)[None] + n_pages
    cache = ref.rand_cache(rng, n_pages + 6, nkv, ps, hd)
    gpu = on_gpu(cache)
    q = dev(rng.standard_normal((n, nh * hd)).astype(np.float32))
    pos, pages, p_len = dev(np.zeros(n, np.int32)), dev(tables[0]), dev(np.zeros(1, np.int32))
    batch = bl.PagedBatch(dev(np.arange(n + 1, dtype=np.int32)), pos, pages, n, 1, 91)
    prefix = bl.PagedBatch(dev(np.array([0, n], np.int32)), p_len, dev(ptable), n, n, 96)
    accounts = [bl.KVAccount(n, nkv, 96, DEV) for _ in range(2)]
    space = bl.paged_attention_account_workspace(gpu, batch, nh, prefix=prefix)
    outs = [torch.empty_like(q) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for a, o in zip(accounts, outs):
            bl.paged_attention_account(q, gpu, batch, a, prefix=prefix, out=o, workspace=space)
            g = torch.cuda.CUDAGraph()
            side.synchronize()
            with torch.cuda.graph(g, stream=side):
                bl.paged_attention_account(q, gpu, batch, a, prefix=prefix, out=o, workspace=space)
            graphs.append(g)
        for step, (at, size) in enumerate([(0, 1), (40, 96), (89, 0), (90, 33)]):
            pos.fill_(at)
            p_len.fill_(size)
            pages.copy_(dev(tables[step % 2]))
            for a in accounts:
                a.weight.zero_()
            graphs[0].replay()
            graphs[1].replay()
            side.synchronize()
            want, bound, w, wb = cref.attention(host(q).reshape(n, nh, hd), cache, tables[step % 2], [(1, at)] * n,
                                                list(range(n)), False, [(0, n, size)], ptable)
            for a, o in zip(accounts, outs):
                within(host(o).reshape(n, nh, hd), want, bound)
                for s in range(n):
                    within(host(a.weight[s, :, :at + 1]), w[s], wb[s] + cref.U * w[s])
                assert (a.weight[:, :, at + 1:] == 0).all()
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_captured_step_whose_rows_change_hands(dtype):
    """Attention with weights behind a prefix and the eviction after it in one graph: between its
    replays rows go from one sequence to another, so that each is once of many rows, of few and of
    none, and lists end elsewhere."""
    nh, nkv, hd, ps, rows, keep = 8, 2, 64, 32, 60, 150
    rng = np.random.default_rng(77)
    table, n_own = ref.pages_for([(60, 400)] * 3, ps, rng, wide_extra=0)
    ptable = np.arange(n_own, n_own + 16, dtype=np.int32).reshape(2, 8)
    cache = ref.rand_cache(rng, n_own + 16, nkv, ps, hd)
    gpu, fresh = on_gpu(cache), [dev(x) for x in cache]
    q = dev(rng.standard_normal((rows, nh * hd)).astype(np.float32), DT[dtype])
    start, pos = dev(np.array([0, 20, 40, 60], np.int32)), dev(np.zeros(3, np.int32))
    p_start, p_pos = dev(np.array([0, 30, 60], np.int32)), dev(np.zeros(2, np.int32))
    batch = bl.PagedBatch(start, pos, dev(table), rows, 60, 460)
    prefix = bl.PagedBatch(p_start, p_pos, dev(ptable), rows, 60, 250)
    account, left = bl.KVAccount(3, nkv, 460, DEV), bl.KVAccount(3, nkv, 460, DEV)
    out, held = torch.empty_like(q), dev(np.zeros(3, np.int32))
    recent = dev(np.full(3, 10, np.int32))
    keeps = dev(np.full(3, keep, np.int32))
    space = bl.paged_attention_account_workspace(gpu, batch, nh, prefix=prefix)
    more = bl.paged_evict_workspace(gpu, batch)

    def step():
        bl.paged_attention_account(q, gpu, batch, account, prefix=prefix, out=out, workspace=space)
        bl.paged_evict(gpu, batch, account, keeps, recent=recent, max_keep=keep, out=left, held=held, workspace=more)

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for starts, at, p_starts, p_at in (([0, 20, 40, 60], [0, 100, 400], [0, 30, 60], [250, 3]),
                                       ([0, 57, 58, 60], [300, 400, 0], [0, 1, 59], [64, 250]),
                                       ([0, 0, 1, 60], [222, 399, 90], [0, 0, 60], [250, 100]),
                                       ([0, 60, 60, 60], [400, 149, 151], [10, 20, 50], [0, 250]),
                                       ([0, 20, 40, 60], [0, 100, 400], [0, 30, 60], [250, 3])):
        for x, y in zip((start, pos, p_start, p_pos), (starts, at, p_starts, p_at)):
            x.copy_(dev(np.array(y, np.int32)))
        for x, y in zip((gpu.k, gpu.v, gpu.k_scale, gpu.v_scale), fresh):
            x.copy_(y)
        account.weight.fill_(0.25)
        graph.replay()
        sizes = [(b - a, p) for a, b, p in zip(starts, starts[1:], at)]
        lists = [(a, b - a, p) for a, b, p in zip(p_starts, p_starts[1:], p_at)]
        want, bound, w, wb = cref.attention(host(q).reshape(rows, nh, hd), cache, table, sizes, starts, dtype == "bf16", lists,
                                            ptable)
        within(host(out).reshape(rows, nh, hd), want, bound)
        for s, (r, p) in enumerate(sizes):
            if r:
                w[s][:, :p] += 0.25
                within(host(account.weight[s, :, :r + p]), w[s], wb[s] + cref.U * w[s])
                assert (account.weight[s, :, r + p:] == 0.25).all()
            else:
                assert (account.weight[s] == 0.25).all()
        arrays = [x.cpu().numpy() for x in (account.weight, account.token, account.filled, account.shift)]
        want_cache, kept, want_held = cref.evict(cache, table, [r + p for r, p in sizes], arrays, [keep] * 3, [0] * 3, [10] * 3)
        assert held.tolist() == want_held
        for name, g, x in zip(("k", "v", "k scale", "v scale"), (gpu.k, gpu.v, gpu.k_scale, gpu.v_scale), want_cache):
            same_bits(g.cpu().numpy(), x, name)
        for s, n in enumerate(want_held):
            same_bits(left.weight[s, :, :n].cpu().numpy(), kept[0][s, :, :n], "weights")
            same_bits(left.token[s, :, :n].cpu().numpy(), kept[1][s, :, :n], "tokens")
