"""Plain implementations of the batched serving ops (include/bitserve.h) in 64 bits, on
the CPU, and small paged caches to run them on."""
import math

import numpy as np
import torch


def pages_for(sizes, ps, rng, extra=3, wide_extra=1):
    """A page table (rows of shuffled ids, -1 behind a sequence's last page) for sequences of
    sizes [(rows, pos)], and the pool's page count."""
    per = [max(0, -(-(r + p) // ps)) for r, p in sizes]
    n_pages = sum(per) + extra
    order = rng.permutation(n_pages)
    table = np.full((len(sizes), max(per + [1]) + wide_extra), -1, np.int32)
    at = 0
    for s, c in enumerate(per):
        table[s, :c] = order[at:at + c]
        at += c
    return table, n_pages


def rand_cache(rng, n_pages, nkv, ps, hd):
    """Random codes and scales in the paged layout: k, v (blocked), k_scale, v_scale."""
    k = rng.integers(1, 256, (n_pages, nkv, ps, hd)).astype(np.uint8)
    v = rng.integers(1, 256, (n_pages, nkv, ps // 16, hd, 16)).astype(np.uint8)
    ks = (rng.random((n_pages, nkv, ps)) * 0.03 + 0.002).astype(np.float32)
    vs = (rng.random((n_pages, nkv, ps)) * 0.03 + 0.002).astype(np.float32)
    return k, v, ks, vs


def rows_of(cache, table, s, size):
    """Sequence s's first `size` keys and values in 64 bits: [size, nkv, hd]."""
    k, v, ks, vs = cache
    n_pages, nkv, ps, hd = k.shape
    kk, vv = np.empty((size, nkv, hd)), np.empty((size, nkv, hd))
    for p in range(size):
        pg, sl = table[s, p // ps], p % ps
        kk[p] = (k[pg, :, sl].astype(np.float64) - 128) * ks[pg, :, sl].astype(np.float64)[:, None]
        vv[p] = (v[pg, :, sl // 16, :, sl % 16].astype(np.float64) - 128) * vs[pg, :, sl].astype(np.float64)[:, None]
    return kk, vv


def attention(q, cache, table, sizes, starts, bf16):
    """(outputs, bound) [rows, nh, hd] in 64 bits: softmax attention of each row over its
    sequence, and how far a result may be from it.

    The bound, from the arithmetic that include/bitserve.h states.  u = 2^-24.  A query in f16
    parts is off by e_q of itself (2^-22 in two parts, 0 for bf16 in one); a product of hd terms
    summed in f32, scaled by the key's scale and the row's, is off by (hd + 4) u of the sum of
    the terms' sizes A: ds = (e_q + (hd + 4) u) A.  The exponent's argument is formed and rounded
    at the size of the scores in log2 units, S: another 4 u S; exp2 and the sums of n weights:
    (n + 8) u.  Every weight is then off by the factor 1 +- (2 (ds + 4 u S) + 2 (n + 8) u) in the
    ratio of the two sums, and by e_p (2^-22, 2^-11 for one part) as the matrix product takes it;
    the output, a mean of values of size V at most, by that many V; and by the final rounding."""
    rows, nh, hd = q.shape
    u = 2.0 ** -24
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    nkv = cache[0].shape[1]
    g = nh // nkv
    for s, (r, p) in enumerate(sizes):
        if not r:
            continue
        k, v = rows_of(cache, table, s, r + p)
        for h in range(nkv):
            qs = q[starts[s]:starts[s] + r, h * g:(h + 1) * g].astype(np.float64)  # [r, g, hd]
            sc = np.einsum("igd,jd->igj", qs, k[:, h]) / math.sqrt(hd)
            size = np.einsum("igd,jd->igj", np.abs(qs), np.abs(k[:, h])) / math.sqrt(hd)
            late = np.arange(r + p)[None] > (p + np.arange(r))[:, None]
            sc = np.where(late[:, None], -np.inf, sc)
            w = np.exp(sc - sc.max(axis=2, keepdims=True))
            o = np.einsum("igj,jd->igd", w / w.sum(axis=2, keepdims=True), v[:, h])
            seen = np.where(late[:, None], 0.0, size).max(axis=2)
            most = np.where(late[:, :, None], 0.0, np.abs(v[None, :, h])).max(axis=1)  # [r, hd]
            ds = ((0 if bf16 else 2.0 ** -22) + (hd + 4) * u) * seen + 4 * u * 1.5 * seen
            rel = 2 * ds + 2 * (r + p + 8) * u + (2.0 ** -11 if bf16 else 2.0 ** -22)
            out[starts[s]:starts[s] + r, h * g:(h + 1) * g] = o
            bound[starts[s]:starts[s] + r, h * g:(h + 1) * g] = \
                rel[:, :, None] * most[:, None].max(axis=2, keepdims=True) + (2.0 ** -8 if bf16 else u) * np.abs(o)
    return out, bound


def sample_one(logits, t=1.0, k=0, p=1.0, m=0.0, u=0.0):
    """(id, probability) of one row, from the definition: whole weights in Python integers."""
    l = np.asarray(logits, np.float32).astype(np.float64).copy()
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(l)), 1.0
    if top == np.inf:
        w = np.where(l == np.inf, 2.0 ** 40, 0.0)
    else:
        with np.errstate(over="ignore", invalid="ignore"):
            w = np.rint(np.exp((l - top) / np.float64(np.float32(t))) * 2.0 ** 40)
        w[l == -np.inf] = 0
    order = np.argsort(-l, kind="stable")
    w = [int(x) for x in w[order]]
    m = min(max(float(np.float32(m)), 0.0), 1.0) if m == m else 0.0
    w = [x for x in w if x >= max(1, math.ceil(m * 2 ** 40))]
    if 0 < k < len(w):
        w = w[:k]
    p = float(np.float32(p))
    if p < 1:
        goal, run, n = max(1, math.ceil(max(p, 0.0) * float(sum(w)))), 0, 0
        while run < goal and n < len(w):
            run += w[n]
            n += 1
        w = w[:n]
    total = sum(w)
    u = float(np.float32(u))
    r = min(int((u if u > 0 else 0.0) * float(total)), total - 1)
    run = 0
    for i, x in enumerate(w):
        run += x
        if run > r:
            return int(order[i]), x / total
    raise AssertionError


def bf16_round(x):
    """f32 array -> the nearest bf16 values (ties to even), as f32."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).float().numpy()
