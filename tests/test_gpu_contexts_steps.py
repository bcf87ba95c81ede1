"""GPU test of steps within a budget behind a shared prompt (include/bitserve.h): each step's
append, attention with weights and eviction against a model of the cache that is carried along
in 64 bits (context_ref.py), first by calls and then by graphs that are replayed."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import context_ref as cref
import serve_ref as ref
from test_gpu_contexts import same_bits, within
from test_gpu_serve import DEV, DT, dev, host, rope, same

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

NAMES = ("k", "v", "k scale", "v scale"), ("weight", "token", "filled", "shift")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,rows,keep,sink,recent", [
    (8, 2, 1, [24, 10, 24, 7], 0, 4),
    (8, 2, 3, [24, 10, 31, 7], 79, 3),     # drafts; the first tokens behind the prompt stay
    (6, 3, 9, [40, 33, 9, 64], 0, 0),      # tiles
])
def test_steps_within_a_budget_and_a_model_of_them(nh, nkv, rows, keep, sink, recent, dtype):
    hd, ps, n, prompt, steps = 64, 16, len(keep), 75, 36
    rng = np.random.default_rng(nh + rows)
    _, _, dc, ds = rope(hd, prompt + steps * rows)
    cap = max(keep) + rows
    per = -(-cap // ps)
    cache = bl.PagedKVCacheQ8(5 + n * per, ps, nkv, hd, DEV)
    ptable = np.arange(5, dtype=np.int32)[None]
    table = (5 + rng.permutation(n * per)).reshape(n, per).astype(np.int32)
    first = bl.PagedBatch(dev(np.array([0, prompt], np.int32)), dev(np.zeros(1, np.int32)), dev(ptable), prompt)
    bl.paged_rope_append(*[dev(rng.standard_normal((prompt, m * hd)).astype(np.float32), DT[dtype]) for m in (nh, nkv, nkv)],
                         cache, first, dc, ds)
    pos = dev(np.zeros(n, np.int32))
    starts = rows * np.arange(n + 1, dtype=np.int32)
    batch = bl.PagedBatch(dev(starts), pos, dev(table), n * rows, rows, cap)
    prefix = bl.PagedBatch(dev(np.array([0, n * rows], np.int32)), dev(np.array([prompt], np.int32)), dev(ptable), n * rows,
                           n * rows, prompt)
    account = bl.KVAccount(n, nkv, cap + 1, DEV, shift=prompt)
    keeps, sinks, recents = (dev(np.array(x, np.int32)) for x in (keep, [sink] * n, [recent] * n))
    held = torch.zeros_like(pos)
    spaces = bl.paged_attention_account_workspace(cache, batch, nh, prefix=prefix), bl.paged_evict_workspace(cache, batch)
    new = [torch.empty((n * rows, m * hd), device=DEV, dtype=DT[dtype]) for m in (nh, nkv, nkv)]
    qr, out = torch.empty_like(new[0]), torch.empty_like(new[0])
    now = [cache.k, cache.v, cache.k_scale, cache.v_scale], [account.weight, account.token, account.filled, account.shift]

    def attend():
        bl.paged_rope_append(*new, cache, batch, dc, ds, q_out=qr, rope_shift=account.shift)
        bl.paged_attention_account(qr, cache, batch, account, prefix=prefix, out=out, workspace=spaces[0])

    def evict():
        bl.paged_evict(cache, batch, account, keeps, sink=sinks, recent=recents, max_keep=max(keep), held=held,
                       workspace=spaces[1])

    def captured(f):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            f()
        return graph.replay

    def arrays(of):
        return [x.cpu().numpy().copy() for x in of]

    rows_of = {}  # (sequence, head, token) -> its codes and scales as they were appended
    at = [0] * n
    for t in range(steps):
        print("step", t, at, flush=True)
        for x in new:
            x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        if t == steps // 2:
            attend, evict = captured(attend), captured(evict)
        was, had = arrays(now[0]), arrays(now[1])
        attend()
        mid, got = arrays(now[0]), arrays(now[1])
        # the append: what a cache has that holds the same tokens at their RoPE positions, and nothing else
        lone = bl.PagedKVCacheQ8(n * (prompt + steps * rows) // 16 + 2 * n, 16, nkv, hd, DEV)
        lone_table = np.arange(lone.n_pages // n * n, dtype=np.int32).reshape(n, -1)
        far = bl.PagedBatch(dev(starts), dev(np.full(n, prompt + t * rows, np.int32)), dev(lone_table), n * rows, rows)
        same(host(qr), host(bl.paged_rope_append(*new, lone, far, dc, ds)), "q")
        there = arrays([lone.k, lone.v, lone.k_scale, lone.v_scale])

        def row(c, page, h, slot):
            return (c[0][page, h, slot].tobytes(), c[1][page, h, slot // 16, :, slot % 16].tobytes(),
                    c[2][page, h, slot].tobytes(), c[3][page, h, slot].tobytes())

        for s in range(n):
            for i in range(rows):
                token, j = prompt + t * rows + i, at[s] + i
                for h in range(nkv):
                    mine = row(there, lone_table[s, token // 16], h, token % 16)
                    rows_of[s, h, token] = mine
                    page, slot = table[s, j // ps], j % ps
                    assert row(mid, page, h, slot) == mine
                    was[0][page, h, slot], was[2][page, h, slot] = mid[0][page, h, slot], mid[2][page, h, slot]
                    was[1][page, h, slot // 16, :, slot % 16] = mid[1][page, h, slot // 16, :, slot % 16]
                    was[3][page, h, slot] = mid[3][page, h, slot]
        for x, y, name in zip(mid, was, NAMES[0]):
            same_bits(x, y, "appended " + name)
        # the attention and the weights, added to those of before the step
        sizes = [(rows, p) for p in at]
        want, bound, w, wb = cref.attention(host(qr).reshape(n * rows, nh, hd), mid, table, sizes, starts, dtype == "bf16",
                                            [(0, n * rows, prompt)], ptable)
        within(host(out).reshape(n * rows, nh, hd), want, bound, "outputs")
        for s, (r, p) in enumerate(sizes):
            w[s][:, :p] += had[0][s, :, :p]
            within(got[0][s, :, :p + r].astype(np.float64), w[s], wb[s] + cref.U * w[s], "weights")
            same_bits(got[0][s, :, p + r:], had[0][s, :, p + r:], "behind")
        for x, y, name in zip(got[1:], had[1:], NAMES[1][1:]):
            same_bits(x, y, "kept " + name)
        # the eviction, from the weights that the attention left
        evict()
        size = [p + rows for p in at]
        want_cache, want, want_held = cref.evict(mid, table, size, got, keep, [sink] * n, [recent] * n)
        for x, y, name in zip(arrays(now[0]), want_cache, NAMES[0]):
            same_bits(x, y, name)
        after = arrays(now[1])
        for x, y, name in zip(after, want, NAMES[1]):
            same_bits(x, y, name)
        assert held.tolist() == want_held == [min(k, x) for k, x in zip(keep, size)]
        pos.copy_(held)
        at = want_held
        # each position holds the codes of the token that is recorded for it
        end = arrays(now[0])
        for s in range(n):
            for h in range(nkv):
                for j in range(at[s]):
                    assert row(end, table[s, j // ps], h, j % ps) == rows_of[s, h, int(after[1][s, h, j])]
    assert after[3].tolist() == [prompt + steps * rows - k for k in keep]
