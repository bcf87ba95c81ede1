"""Plain implementations in 64 bits, on the CPU, of attention beside a shared prefix, of the
weights that rows give positions, and of eviction (include/bitserve.h)."""
import math

import numpy as np

import serve_ref as ref

U = 2.0 ** -24


def attention(q, cache, table, sizes, starts, bf16, lists=(), list_table=None):
    """(out, bound, weights, weight bounds) for rows q [rows, nh, hd]: of each row its softmax
    attention over its list's prefix and its sequence's positions, and per sequence the
    weights [nkv, rows + pos] that its rows gave its own positions.  lists: (first row, rows,
    prefix length).

    The bounds are those of serve_ref.attention for the row's terms, with u = 2^-24: scores off by
    ds = (e_q + (hd + 4) u) A + 4 u S, a softmax weight by the factor 1 +- (2 ds + 2 (n + 8) u).
    The sum of R such weights in f32 is off by another R u of itself, and its addition to what a
    position had by u of the result (added by the caller, who knows that)."""
    rows, nh, hd = q.shape
    nkv = cache[0].shape[1]
    g = nh // nkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    weights, wbounds = [], []
    behind = [None] * rows
    for n, (first, count, size) in enumerate(lists):
        kv = ref.rows_of(cache, list_table, n, size)
        for t in range(first, first + count):
            behind[t] = kv
    for s, (r, p) in enumerate(sizes):
        w_s, b_s = np.zeros((nkv, r + p)), np.zeros((nkv, r + p))
        k, v = ref.rows_of(cache, table, s, r + p)
        for i in range(r):
            t = starts[s] + i
            kk, vv = k[:p + i + 1], v[:p + i + 1]
            np_ = 0
            if behind[t] is not None:
                np_ = len(behind[t][0])
                kk, vv = np.concatenate([behind[t][0], kk]), np.concatenate([behind[t][1], vv])
            for h in range(nkv):
                qs = q[t, h * g:(h + 1) * g].astype(np.float64)
                sc = qs @ kk[:, h].T / math.sqrt(hd)
                size = (np.abs(qs) @ np.abs(kk[:, h]).T).max(axis=1) / math.sqrt(hd)
                w = np.exp(sc - sc.max(axis=1, keepdims=True))
                w /= w.sum(axis=1, keepdims=True)
                o = w @ vv[:, h]
                ds = ((0 if bf16 else 2.0 ** -22) + (hd + 4) * U) * size + 4 * U * 1.5 * size
                rel = 2 * ds + 2 * (len(kk) + 8) * U  # of a weight
                most = np.abs(vv[:, h]).max()
                out[t, h * g:(h + 1) * g] = o
                bound[t, h * g:(h + 1) * g] = (rel + (2.0 ** -11 if bf16 else 2.0 ** -22))[:, None] * most \
                    + (2.0 ** -8 if bf16 else U) * np.abs(o)
                w_s[h, :p + i + 1] += w[:, np_:].sum(axis=0)
                b_s[h, :p + i + 1] += ((rel + (r * g + 4) * U)[:, None] * w[:, np_:]).sum(axis=0)
        weights.append(w_s)
        wbounds.append(b_s)
    return out, bound, weights, wbounds


def choose(weight, token, filled, shift, size, keep, sink, recent):
    """Per (sequence, KV head): (source of each held position, its token); weight, token: the
    head's rows."""
    place = [int(token[j]) if j < filled else j + int(shift) for j in range(size)]
    if keep < 0 or keep >= size:
        return list(range(size)), place
    late = size + int(shift) - max(recent, 0)

    def order(j):
        if place[j] < sink or place[j] >= late:
            return (0, 0.0, j)
        w = float(weight[j])
        return (2, 0.0, j) if math.isnan(w) else (1, -w, j)

    stay = set(sorted(range(size), key=order)[:keep])
    movers = iter(sorted(j for j in stay if j >= keep))
    come = [j if j in stay else next(movers) for j in range(keep)]
    return come, [place[j] for j in come]


def evict(cache, table, sizes, account, keep, sink, recent, ok=None):
    """The caches' arrays and the account after an eviction, and held.  account: weight, token,
    filled, shift (numpy); ok: sequences that are not refused."""
    k, v, ks, vs = (x.copy() for x in cache)
    n_pages, nkv, ps, _ = k.shape
    weight, token, filled, shift = (x.copy() for x in account)
    held = []
    for s, size in enumerate(sizes):
        if ok is not None and not ok[s]:
            held.append(-1)
            continue
        left = size if keep[s] < 0 else min(keep[s], size)
        for h in range(nkv):
            come, place = choose(account[0][s, h], account[1][s, h], account[2][s], account[3][s], size, keep[s], sink[s],
                                 recent[s])
            weight[s, h, :left] = account[0][s, h, come]
            token[s, h, :left] = place
            for j, c in enumerate(come):
                if c == j:
                    continue
                tp, ts, fp, fs = table[s, j // ps], j % ps, table[s, c // ps], c % ps
                if not 0 <= tp < n_pages:
                    continue
                if not 0 <= fp < n_pages:
                    ks[tp, h, ts] = vs[tp, h, ts] = np.nan
                    continue
                k[tp, h, ts] = cache[0][fp, h, fs]
                v[tp, h, ts // 16, :, ts % 16] = cache[1][fp, h, fs // 16, :, fs % 16]
                ks[tp, h, ts], vs[tp, h, ts] = cache[2][fp, h, fs], cache[3][fp, h, fs]
        filled[s], shift[s] = left, account[3][s] + size - left
        held.append(left)
    return (k, v, ks, vs), (weight, token, filled, shift), held
