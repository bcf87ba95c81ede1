"""The operators of a batch of sequences that are served together, as cases that can be timed and compared.

`store`: the new rows' RoPE, their keys and values quantised into the pages of a shared cache, and
what was written read back.  `read`: whole contexts read back from the pages.  `attention`: the new
rows of every sequence over its pages.  `sample`: the next tokens from logits and given random numbers.
With `own` false each is computed by elementary torch operations, else by the package's kernels.
Head counts and widths are those of bench.py and of the tests (32 heads over 8 of 128), and generic ones.
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ONE = float(2 ** 40)  # the weight of the likeliest token

own = False


def listed():
    return [
        # One decoded token of one sequence: the smallest append, where latency counts.
        {"name": "store_token", "kind": "store", "seqs": 1, "rows": 1, "len": 200, "ragged": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 16, "dtype": "f32"},
        # 64 sequences decoded together.
        {"name": "store_batch", "kind": "store", "seqs": 64, "rows": 1, "len": 1500, "ragged": 1, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 64, "dtype": "f32"},
        # Prompts of four sequences in chunks of up to 1001 tokens that begin and end inside pages.
        {"name": "store_prompts", "kind": "store", "seqs": 4, "rows": 1001, "len": 1700, "ragged": 1, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 32, "dtype": "bf16"},
        # A short context read back.
        {"name": "read_short", "kind": "read", "seqs": 1, "rows": 300, "len": 300, "ragged": 0, "heads": 8,
         "kv_heads": 4, "hd": 64, "page": 16, "dtype": "f32"},
        # Sixteen contexts of up to 4099 tokens taken out of the cache.
        {"name": "read_contexts", "kind": "read", "seqs": 16, "rows": 4099, "len": 4099, "ragged": 1, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # One token over a short context: the attention's latency.
        {"name": "attention_token", "kind": "attention", "seqs": 1, "rows": 1, "len": 777, "ragged": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 16, "dtype": "f32"},
        # 32 sequences of up to 8192 tokens decoded together: bound by the cache's bytes.
        {"name": "attention_batch", "kind": "attention", "seqs": 32, "rows": 1, "len": 8192, "ragged": 1, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # One token over a very long context: few rows, a long axis.
        {"name": "attention_long", "kind": "attention", "seqs": 1, "rows": 1, "len": 100001, "ragged": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 128, "dtype": "f32"},
        # The last 512 tokens of an 8192-token prompt that is taken in chunks: bound by the products.
        {"name": "attention_chunk", "kind": "attention", "seqs": 1, "rows": 512, "len": 8192, "ragged": 0, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # A step that mixes two prompt chunks with decoded tokens, in 32 bits, heads of 96.
        {"name": "attention_mixed", "kind": "attention", "seqs": 14, "rows": 201, "len": 1900, "ragged": 2, "heads": 16,
         "kv_heads": 4, "hd": 96, "page": 32, "dtype": "f32"},
        # One sequence's next token, all filters on.
        {"name": "sample_one", "kind": "sample", "rows": 1, "n": 128256, "filters": "all", "flat": False},
        # 64 sequences' next tokens; every request has filters of its own.
        {"name": "sample_batch", "kind": "sample", "rows": 64, "n": 128256, "filters": "mixed", "flat": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: the listed kinds over the sizes they stand for, costs bounded by the listed ones'."""
    kind = rng.choice(["store", "read", "attention", "attention", "attention", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 96)
        return {"kind": kind, "rows": rows, "n": min(_log(rng, 300, 150000), 8_000_000 // rows),
                "filters": rng.choice(["all", "mixed", "mixed", "none", "top_k", "top_p", "min_p"]),
                "flat": rng.random() < 0.3}
    kv = rng.choice([1, 2, 4, 8, 8])
    case = {"kind": kind, "heads": kv * rng.choice([1, 2, 4, 4, 5, 8]), "kv_heads": kv,
            "hd": rng.choice([32, 64, 80, 96, 112, 128, 128]), "page": rng.choice([16, 32, 48, 64, 128, 256]),
            "dtype": rng.choice(["f32", "bf16"])}
    if kind == "store":
        seqs = _log(rng, 1, 128)
        rows = rng.choice([1, _log(rng, 1, max(1, 2500 // seqs))])
        return dict(case, seqs=seqs, rows=rows, len=rows + _log(rng, 1, 2000), ragged=rng.choice([0, 1]))
    if kind == "read":
        seqs = _log(rng, 1, 24)
        rows = _log(rng, 1, 24000 // seqs)
        return dict(case, seqs=seqs, rows=rows, len=rows + rng.choice([0, 0, 17]), ragged=rng.choice([0, 1]))
    form = rng.choice(["tokens", "tokens", "chunk", "mixed"])
    if form == "tokens":  # one to a few new tokens of each sequence
        seqs, rows = _log(rng, 1, 48), rng.choice([1, 1, 1, 2, 5])
        return dict(case, seqs=seqs, rows=rows, len=rows + _log(rng, 1, min(100000, 150000 // seqs)), ragged=rng.choice([0, 1]))
    if form == "chunk":
        rows = _log(rng, 6, 512)
        return dict(case, seqs=rng.choice([1, 1, 2]), rows=rows, len=rows + rng.choice([0, _log(rng, 1, 1500)]),
                    ragged=rng.choice([0, 1]))
    rows = _log(rng, 6, 220)
    return dict(case, seqs=rng.randint(2, 14), rows=rows, len=rows + _log(rng, 1, 1600), ragged=2)


# ------------------------------------------------------------------ inputs

def _sizes(case):
    """(rows, positions before them) of each sequence.  ragged 0: all alike; 1: contexts down to a
    quarter of the longest, rows down to a third; 2: one or two chunks, then single tokens."""
    n, got = case["seqs"], []
    for i in range(n):
        size, rows = case["len"], case["rows"]
        if case["ragged"]:
            size = max(1, round(size * (1 - 0.75 * i / n)))
            rows = max(1, round(rows * (1 - 0.67 * i / n))) if case["ragged"] == 1 else (rows if i == 0 else max(1, rows // 3) if i == 1 else 1)
        rows = min(rows, size)
        got.append((rows, size - rows))
    return got


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _paged(case, g, seed):
    """The page pool with quantised rows in it, each sequence's pages in no order, and the batch."""
    sizes, ps, kv, hd = _sizes(case), case["page"], case["kv_heads"], case["hd"]
    per = [-(-(r + p) // ps) for r, p in sizes]
    wide, n_pages = max(per), sum(per) + 3
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for c in per:
        table.append(order[at:at + c] + [0] * (wide - c))
        at += c
    starts = [0]
    for r, _ in sizes:
        starts.append(starts[-1] + r)
    i32 = dict(dtype=torch.int32, device=DEV)

    def codes():
        """Codes of values near a normal distribution, three deviations wide."""
        x = torch.randn((n_pages, kv, ps, hd), generator=g, device=DEV)
        return x.mul_(40).round_().clamp_(-127, 127).add_(128).to(torch.uint8)

    def scales():
        return torch.rand((n_pages, kv, ps), generator=g, device=DEV) * 0.03 + 0.01

    k = codes()
    # values lie in blocks of 16 slots, the slots innermost
    v = codes().view(n_pages, kv, ps // 16, 16, hd).transpose(3, 4).contiguous()
    seq = torch.tensor([s for s, (r, _) in enumerate(sizes) for _ in range(r)], device=DEV)
    i = torch.tensor([j for r, _ in sizes for j in range(r)], device=DEV)
    pos = torch.tensor([p for _, p in sizes], **i32)
    return {"case": dict(case), "k_codes": k, "v_codes": v, "k_scale": scales(), "v_scale": scales(),
            "pages": torch.tensor(table, **i32), "row_start": torch.tensor(starts, **i32), "pos": pos,
            "max_rows": max(r for r, _ in sizes), "max_len": max(r + p for r, p in sizes),
            "row_seq": seq, "row_i": i, "row_pos": pos.long()[seq] + i, "sizes": sizes}


def _rope(size, hd):
    """Tables of cos and sin, one row a position."""
    inv = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    a = torch.arange(size, dtype=torch.float64, device=DEV)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _filters(case):
    """Each row's temperature, top_k, top_p and min_p; 0 or 1 where one is off."""
    mixes = {"all": [(0.8, 50, 0.95, 0.02)], "none": [(1.0, 0, 1.0, 0.0)], "top_k": [(0.7, 40, 1.0, 0.0)],
             "top_p": [(0.9, 0, 0.9, 0.0)], "min_p": [(1.1, 0, 1.0, 0.05)],
             "mixed": [(0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.1),
                       (1.0, 0, 1.0, 0.0), (0.6, 1000, 0.8, 0.01), (0.9, 5, 1.0, 0.0)]}[case["filters"]]
    return [mixes[i % len(mixes)] for i in range(case["rows"])]


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "sample":
        rows, n = case["rows"], case["n"]
        logits = torch.randn((rows, n), generator=g, device=DEV)
        if case["flat"]:  # an untrained model's
            logits.mul_(1.5)
        else:  # a model's: they fall with the logarithm of a token's rank
            rank = torch.argsort(torch.rand((rows, n), generator=g, device=DEV), dim=1)
            logits.mul_(0.7).add_(-1.4 * torch.log1p(rank.float()))
        f = _filters(case)
        col = lambda i, t: torch.tensor([x[i] for x in f], dtype=t, device=DEV)  # noqa: E731
        return {"case": dict(case), "logits": logits, "temperature": col(0, torch.float32), "top_k": col(1, torch.int32),
                "top_p": col(2, torch.float32), "min_p": col(3, torch.float32),
                "u": torch.rand((rows,), generator=g, device=DEV),
                "ids": torch.empty((rows,), dtype=torch.int32, device=DEV),
                "probs": torch.empty((rows,), device=DEV), "space": _space(case)}
    s = _paged(case, g, seed)
    rows, kv, hd, dt = s["row_seq"].numel(), case["kv_heads"], case["hd"], DTYPES[case["dtype"]]
    if case["kind"] != "read":
        s["q"] = (torch.randn((rows, case["heads"] * hd), generator=g, device=DEV) * 2).to(dt)
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] == "store":
        s["k"] = (torch.randn((rows, kv * hd), generator=g, device=DEV) * 2).to(dt)
        s["v"] = torch.randn((rows, kv * hd), generator=g, device=DEV).to(dt)
        s["cos"], s["sin"] = _rope(s["max_len"], hd)
    if case["kind"] != "attention":
        back = torch.float32 if case["kind"] == "store" else dt
        s["k_out"] = torch.empty((rows, kv * hd), dtype=back, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    if own:
        bl = _engine()
        s["cache"] = bl.PagedKVCacheQ8.of(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        s["batch"] = bl.PagedBatch(s["row_start"], s["pos"], s["pages"], rows, s["max_rows"], s["max_len"])
        if case["kind"] == "attention":
            s["space"] = bl.paged_attention_workspace(s["cache"], s["batch"], case["heads"])
    return s


def _engine():
    where = os.path.join(ROOT, "bit-ttt-engine_amd")
    if where not in sys.path:
        sys.path.insert(1, where)
    import bitlinear
    return bitlinear


def _space(case):
    return _engine().sample_workspace(case["rows"], case["n"], DEV) if own else None


# ------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if kind == "sample":
        return _sample(s)
    if kind == "attention":
        return _attention(s)
    if kind == "read":
        return _read(s)
    return _store(s)


def _slots(s):
    """Page and slot of each row's position."""
    ps = s["case"]["page"]
    return s["pages"][s["row_seq"], s["row_pos"] // ps].long(), s["row_pos"] % ps


def _turn(s, x, heads):
    """RoPE of rows, every product and sum rounded to 32 bits."""
    half = s["case"]["hd"] // 2
    x = x.float().view(x.shape[0], heads, 2, half)
    c, t = s["cos"][s["row_pos"]][:, None], s["sin"][s["row_pos"]][:, None]
    a, b = x[:, :, 0], x[:, :, 1]
    return torch.cat((a * c - b * t, a * t + b * c), dim=2)


def _quantise(x):
    """Codes about 128 and the scale of each head's row; halves go away from zero (in 64 bits: 0.5 less one
    step must not become 1)."""
    scale = x.abs().amax(dim=2) * (1.0 / 127.0)
    y = (x / scale[:, :, None]).double()
    code = torch.sign(y) * torch.floor(y.abs() + 0.5) + 128
    return torch.nan_to_num(code, nan=0.0).clamp(0, 255).to(torch.uint8), scale


def _store(s):
    case = s["case"]
    if own:
        bl = _engine()
        bl.paged_rope_append(s["q"], s["k"], s["v"], s["cache"], s["batch"], s["cos"], s["sin"], q_out=s["out"])
        bl.paged_read(s["cache"], s["batch"], k_out=s["k_out"], v_out=s["v_out"])
        return s["out"], s["k_out"], s["v_out"]
    rows, kv, hd = s["q"].shape[0], case["kv_heads"], case["hd"]
    q = _turn(s, s["q"], case["heads"]).reshape(rows, -1).to(s["q"].dtype)
    page, slot = _slots(s)
    page, slot, head = page[:, None], slot[:, None], torch.arange(kv, device=DEV)[None]
    kc, ks = _quantise(_turn(s, s["k"], kv))
    vc, vs = _quantise(s["v"].float().view(rows, kv, hd))
    s["k_codes"][page, head, slot] = kc
    s["v_codes"][page, head, slot // 16, :, slot % 16] = vc
    s["k_scale"][page, head, slot] = ks
    s["v_scale"][page, head, slot] = vs
    k, v = _read(s)
    return q, k, v


def _read(s):
    if own:
        return _engine().paged_read(s["cache"], s["batch"], k_out=s["k_out"], v_out=s["v_out"])
    page, slot = _slots(s)
    head = torch.arange(s["case"]["kv_heads"], device=DEV)[None]
    page, slot = page[:, None], slot[:, None]
    k = (s["k_codes"][page, head, slot].float() - 128) * s["k_scale"][page, head, slot][:, :, None]
    v = (s["v_codes"][page, head, slot // 16, :, slot % 16].float() - 128) * s["v_scale"][page, head, slot][:, :, None]
    shape, dt = s["k_out"].shape, s["k_out"].dtype
    return k.reshape(shape).to(dt), v.reshape(shape).to(dt)


def _attention(s):
    case = s["case"]
    if own:
        return _engine().paged_attention(s["q"], s["cache"], s["batch"], out=s["out"], workspace=s["space"])
    kv, hd, ps = case["kv_heads"], case["hd"], case["page"]
    group, seqs, rows, size = case["heads"] // kv, case["seqs"], s["max_rows"], s["max_len"]
    # every sequence's keys and values, padded to the longest: [sequence, head, position, value]
    j = torch.arange(size, device=DEV)
    page, slot = s["pages"][:, j // ps].long()[:, None], (j % ps)[None, None]
    head = torch.arange(kv, device=DEV)[None, :, None]
    k = (s["k_codes"][page, head, slot].float() - 128) * s["k_scale"][page, head, slot][..., None]
    v = (s["v_codes"][page, head, slot // 16, :, slot % 16].float() - 128) * s["v_scale"][page, head, slot][..., None]
    # the rows, padded likewise: [sequence, head, row and query head of the group, value]
    i = torch.arange(rows, device=DEV)
    at = (s["row_start"][:-1, None].long() + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[at].view(seqs, rows, kv, group, hd).transpose(1, 2).reshape(seqs, kv, rows * group, hd)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    seen = j <= (s["pos"].long()[:, None] + i)[..., None]  # [sequence, row, position]
    w = w.view(seqs, kv, rows, group, size).masked_fill_(~seen[:, None, :, None], -math.inf)
    w = torch.exp(w - w.amax(dim=4, keepdim=True))
    total = w.sum(dim=4)
    o = torch.matmul(w.view(seqs, kv, rows * group, size), v).view(seqs, kv, rows, group, hd) / total[..., None]
    return o.transpose(1, 2)[s["row_seq"], s["row_i"]].reshape(s["q"].shape).to(s["q"].dtype)


def _sample(s):
    if own:
        return _engine().sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                                ids=s["ids"], probs=s["probs"], workspace=s["space"])
    n = s["logits"].shape[1]
    logit, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    # whole weights in 64 bits: sums are exact, and a token at a border is the same one in any order of them
    x = (logit.double() - logit[:, :1].double()) / torch.where(t > 0, t, 1.0)
    w = torch.round(torch.exp(x) * ONE).to(torch.int64)
    place = torch.arange(n, device=DEV)[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], n)[:, None]
    w = torch.where((w >= s["min_p"].double()[:, None] * ONE) & (place < torch.where(t > 0, k, 1)), w, 0)
    total = torch.cumsum(w, dim=1)
    p = s["top_p"].double()[:, None]
    goal = torch.where(p < 1, torch.ceil(p * total[:, -1:].double()).to(torch.int64).clamp(min=1), total[:, -1:])
    w = torch.where(total - w < goal, w, 0)
    total = torch.cumsum(w, dim=1)
    left = total[:, -1:]
    r = torch.minimum((s["u"].double()[:, None] * left.double()).to(torch.int64), left - 1)
    at = torch.searchsorted(total, r, right=True)
    prob = w.gather(1, at).double() / left.double()
    return order.gather(1, at)[:, 0].to(torch.int32), prob[:, 0].float()


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["n"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 2 * n}
    sizes, kv, hd = _sizes(case), case["kv_heads"], case["hd"]
    rows, size = sum(r for r, _ in sizes), 4 if case["dtype"] == "f32" else 2
    held = kv * (2 * hd + 8)  # a position's codes and scales
    if case["kind"] == "store":  # q in and out; k, v in; the cache written; it read back and put out in 32 bits
        return {"bytes": rows * (2 * size * case["heads"] * hd + 2 * size * kv * hd + 2 * held + 8 * kv * hd + 4 * hd),
                "flops": rows * hd * (3 * case["heads"] + 7 * kv)}
    if case["kind"] == "read":
        return {"bytes": rows * (held + 2 * size * kv * hd), "flops": 4 * rows * kv * hd}
    seen = sum(r * p + r * (r + 1) // 2 for r, p in sizes)
    return {"bytes": sum(r + p for r, p in sizes) * held + 2 * rows * case["heads"] * hd * size,
            "flops": 4 * seen * case["heads"] * hd}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return None, torch.tensor([_chance(s, r) for r in range(case["rows"])], dtype=torch.float64)
    kv, hd, ps = case["kv_heads"], case["hd"], case["page"]
    if case["kind"] == "store":
        # a code next to a border has no one value in more bits: only the rotated rows have
        rows, half = s["q"].shape[0], hd // 2
        z = torch.view_as_complex(s["q"].double().view(rows, -1, 2, half).transpose(2, 3).contiguous())
        at = torch.cat([torch.arange(p, p + r, device=DEV) for r, p in s["sizes"]])
        z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        return torch.view_as_real(z).transpose(2, 3).reshape(rows, -1), None, None
    ks, vs, os_ = [], [], []
    for n, (r, p) in enumerate(s["sizes"]):
        pages = s["pages"][n, :-(-(r + p) // ps)].long()
        # [head, position, value] of this sequence
        k = ((s["k_codes"][pages].double() - 128) * s["k_scale"][pages].double().unsqueeze(-1)).transpose(0, 1).reshape(kv, -1, hd)
        v = s["v_codes"][pages].transpose(3, 4).reshape(len(pages), kv, ps, hd).double() - 128
        v = (v * s["v_scale"][pages].double().unsqueeze(-1)).transpose(0, 1).reshape(kv, -1, hd)
        if case["kind"] == "read":
            ks.append(k[:, p:p + r].transpose(0, 1).reshape(r, -1))
            vs.append(v[:, p:p + r].transpose(0, 1).reshape(r, -1))
            continue
        a = int(s["row_start"][n])
        q = s["q"][a:a + r].double().view(r, kv, -1, hd)
        o = torch.empty_like(q)
        late = torch.arange(r + p, device=DEV)[None] > torch.arange(p, p + r, device=DEV)[:, None]
        for h in range(kv):
            for e in range(q.shape[2]):
                w = (q[:, h, e] @ k[h, :r + p].t().contiguous()) / math.sqrt(hd)
                w = torch.softmax(w.masked_fill(late, -math.inf), dim=1)
                o[:, h, e] = w @ v[h, :r + p]
        os_.append(o.reshape(r, -1))
    return torch.cat(os_) if os_ else (torch.cat(ks), torch.cat(vs))


def _chance(s, r):
    """The drawn token's probability among those that the filters leave."""
    t, k, top, low = (float(s[c][r]) for c in ("temperature", "top_k", "top_p", "min_p"))
    if t <= 0:
        return 1.0
    l = s["logits"][r].double()
    p = torch.sort(torch.softmax(l / t, 0), descending=True).values
    p = p[p >= low * p[0]]
    p = p[:int(k)] if k > 0 else p
    if 0 < top < 1:
        before = torch.cumsum(p, 0) - p
        p = p[before < top * p.sum()]
    c = torch.cumsum(p, 0)
    at = min(int(torch.searchsorted(c, float(s["u"][r]) * c[-1].item(), right=True)), p.numel() - 1)
    return (p[at] / c[-1]).item()
