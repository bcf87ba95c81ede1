"""GPU tests of eviction (include/bitserve.h) at the ends of its numbers' ranges, against
context_ref.evict bit for bit."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_gpu_contexts import check_evict, on_gpu, random_account, same_bits
from test_gpu_serve import DEV, dev

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

MOST = 2 ** 31 - 1


@pytest.mark.filterwarnings("ignore:overflow")  # 2^31 on the way to shift + size - keep
@pytest.mark.parametrize("size,keep", [(20, 10), (9000, 4000)])
@pytest.mark.parametrize("recent", [0, 1, 3, MOST])
@pytest.mark.parametrize("sink", [0, -5, MOST])
@pytest.mark.parametrize("end", ["first", "last"])
def test_tokens_at_the_ends_of_int32(size, keep, recent, sink, end):
    """The last token is 2^31 - 1, or the first -2^31: recent ones are those from len + shift - recent on, also
    where that is 2^31 or below -2^31."""
    rng = np.random.default_rng(size)
    table, n_pages = ref.pages_for([(0, size)] * 2, 16, rng)
    cache = ref.rand_cache(rng, n_pages, 2, 16, 16)
    account = list(random_account(rng, [size] * 2, 2, size + 1, [0, 0], False))
    account[0][:, :, size - 1] = -1e30  # the last position goes where nothing keeps it
    account[3][:] = MOST - (size - 1) if end == "last" else -2 ** 31
    check_evict(cache, table, [size] * 2, account, [keep] * 2, [sink] * 2, [recent] * 2)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_captured_eviction_of_long_heads_whose_lengths_change(in_place):
    """One graph, replayed as sequences grow past a workgroup's positions and fall below them, stay
    whole, are empty or are refused, in the account itself or in another."""
    nkv, hd, ps, cap, n = 2, 16, 32, 20000, 4
    rng = np.random.default_rng(61)
    table, n_pages = ref.pages_for([(0, cap)] * n, ps, rng, wide_extra=0)
    cache = ref.rand_cache(rng, n_pages, nkv, ps, hd)
    gpu, fresh = on_gpu(cache), [dev(x) for x in cache]
    pos, keep, sink, recent = (dev(np.zeros(n, np.int32)) for _ in range(4))
    batch = bl.PagedBatch(dev(np.zeros(n + 1, np.int32)), pos, dev(table), 0, 0, cap)
    account, other, held = bl.KVAccount(n, nkv, cap, DEV), bl.KVAccount(n, nkv, cap, DEV), dev(np.zeros(n, np.int32))
    out = account if in_place else other
    space = bl.paged_evict_workspace(gpu, batch)

    def call():
        bl.paged_evict(gpu, batch, account, keep, sink=sink, recent=recent, max_keep=9000, out=out, held=held, workspace=space)

    call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    for sizes, keeps in (([20000, 100, 8193, 0], [9000, 50, 8192, 3]), ([300, 20000, 8192, 16385], [-1, 8192, 9000, 1]),
                         ([cap + 1, 12000, 12000, -1], [5, 9001, 9000, 5]), ([9000, 9001, 17, 20000], [0, 9000, 16, 9000]),
                         ([20000, 100, 8193, 0], [9000, 50, 8192, 3])):
        print("evict", sizes, keeps, flush=True)
        ok = [0 <= s <= cap and (k < 0 or k >= s or k <= 9000) for s, k in zip(sizes, keeps)]
        lens = [min(max(s, 0), cap) for s in sizes]
        came = random_account(rng, lens, nkv, cap, keeps, True)
        for x, y in zip((pos, keep, sink, recent), (sizes, keeps, [4] * n, [70] * n)):
            x.copy_(dev(np.array(y, np.int32)))
        for x, y in zip((account.weight, account.token, account.filled, account.shift), came):
            x.copy_(dev(y))
        for x, y in zip((gpu.k, gpu.v, gpu.k_scale, gpu.v_scale), fresh):
            x.copy_(y)
        graph.replay()
        want_cache, want, want_held = cref.evict(cache, table, lens, came, keeps, [4] * n, [70] * n, ok)
        assert held.tolist() == want_held
        for x, y in zip((gpu.k, gpu.v, gpu.k_scale, gpu.v_scale), want_cache):
            same_bits(x.cpu().numpy(), y, "cache")
        got = [x.cpu().numpy() for x in (out.weight, out.token, out.filled, out.shift)]
        for s, left in enumerate(want_held):
            if left < 0:
                continue
            same_bits(got[0][s, :, :left], want[0][s, :, :left], "weights")
            same_bits(got[1][s, :, :left], want[1][s, :, :left], "tokens")
            assert got[2][s] == want[2][s] and got[3][s] == want[3][s]
