"""Operators of long contexts in a paged cache, as cases that can be timed and compared.

`prefix`: attention of a batch whose sequences share a long prefix, which is gone through once for all
of them.  `account`: attention that also adds up, for every position of the cache, the weight that the
rows gave it.  `evict`: each sequence cut down to its positions of most weight, and what is left read
back.  With `own` false each is computed by elementary torch operations, else by the package's kernels.
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

own = False


def listed():
    return [
        # Four answers to one short prompt, decoded together: the smallest, where latency counts.
        {"name": "prefix_token", "kind": "prefix", "seqs": 4, "rows": 1, "len": 70, "ragged": 1, "prefix": 515,
         "groups": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 16, "dtype": "f32"},
        # 64 conversations behind one long system prompt, decoded together.
        {"name": "prefix_batch", "kind": "prefix", "seqs": 64, "rows": 1, "len": 700, "ragged": 1, "prefix": 8192,
         "groups": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # Six answers to each of five prompts, three drafted tokens of each looked at; heads of 96, in 32 bits.
        {"name": "prefix_groups", "kind": "prefix", "seqs": 30, "rows": 3, "len": 400, "ragged": 1, "prefix": 2999,
         "groups": 5, "heads": 16, "kv_heads": 4, "hd": 96, "page": 32, "dtype": "f32"},
        # Twelve questions of up to 130 tokens about one document, taken in at once: bound by the products.
        {"name": "prefix_questions", "kind": "prefix", "seqs": 12, "rows": 130, "len": 130, "ragged": 1,
         "prefix": 16001, "groups": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # One decoded token over a short context, its weights added up: latency.
        {"name": "account_token", "kind": "account", "seqs": 1, "rows": 1, "len": 777, "ragged": 0, "prefix": 0,
         "groups": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 16, "dtype": "f32"},
        # 32 sequences of up to 8192 tokens decoded together: bound by the cache's bytes.
        {"name": "account_batch", "kind": "account", "seqs": 32, "rows": 1, "len": 8192, "ragged": 1, "prefix": 0,
         "groups": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # The last 1000 tokens of a prompt of 4099, whose weights choose what is kept of it.
        {"name": "account_prompt", "kind": "account", "seqs": 1, "rows": 1000, "len": 4099, "ragged": 0, "prefix": 0,
         "groups": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # Two prompt chunks and decoded tokens behind two shared prefixes; heads of 64, in 32 bits.
        {"name": "account_mixed", "kind": "account", "seqs": 14, "rows": 201, "len": 1500, "ragged": 2, "prefix": 500,
         "groups": 2, "heads": 16, "kv_heads": 4, "hd": 64, "page": 32, "dtype": "f32"},
        # Eight sequences at their budget, each with one token too many after a step: latency.
        {"name": "evict_step", "kind": "evict", "seqs": 8, "len": 1025, "ragged": 0, "keep": 1024, "sink": 4,
         "recent": 64, "again": True, "kv_heads": 8, "hd": 128, "page": 16, "dtype": "bf16"},
        # A batch's contexts of up to 8192 tokens cut down to 2048.
        {"name": "evict_batch", "kind": "evict", "seqs": 32, "len": 8192, "ragged": 1, "keep": 2048, "sink": 4,
         "recent": 256, "again": False, "kv_heads": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # One very long prompt cut down to 4097 positions: few heads, a long choice.
        {"name": "evict_long", "kind": "evict", "seqs": 1, "len": 100001, "ragged": 0, "keep": 4097, "sink": 16,
         "recent": 1000, "again": False, "kv_heads": 8, "hd": 128, "page": 128, "dtype": "bf16"},
        # Five middling contexts of two heads of 64, evicted from for another time, read back in 32 bits.
        {"name": "evict_again", "kind": "evict", "seqs": 5, "len": 2001, "ragged": 1, "keep": 700, "sink": 0,
         "recent": 100, "again": True, "kv_heads": 2, "hd": 64, "page": 48, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: the listed kinds over the sizes they stand for, costs bounded by the listed ones'."""
    kind = rng.choice(["prefix", "account", "evict"])
    kv = rng.choice([1, 2, 4, 8, 8])
    case = {"kind": kind, "kv_heads": kv, "hd": rng.choice([32, 64, 80, 96, 112, 128, 128]),
            "page": rng.choice([16, 32, 48, 64, 128, 256]), "dtype": rng.choice(["f32", "bf16"])}
    if kind == "evict":
        seqs = _log(rng, 1, 32)
        size = _log(rng, 20, min(100000, 160000 // seqs))
        keep = rng.choice([size - 1, _log(rng, 1, size), max(1, size // 4), max(1, size // 2)])
        return dict(case, seqs=seqs, len=size, ragged=rng.choice([0, 1]), keep=max(1, keep), sink=rng.choice([0, 4, 16]),
                    recent=rng.choice([0, max(1, keep // 8), 1]), again=rng.random() < 0.4)
    case["heads"] = kv * rng.choice([1, 2, 4, 4, 5, 8])
    form = rng.choice(["tokens", "tokens", "chunk", "mixed"])
    if form == "tokens":  # one to a few new tokens of each sequence
        seqs, rows, ragged = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5]), rng.choice([0, 1])
        most = min(8000, 120000 // seqs)
    elif form == "chunk":
        seqs, rows, ragged = rng.choice([1, 1, 2, 6]), _log(rng, 6, 130), rng.choice([0, 1])
        most = 1500
    else:
        seqs, rows, ragged = rng.randint(2, 14), _log(rng, 6, 200), 2
        most = 1500
    case.update(seqs=seqs, rows=rows, len=rows + rng.choice([0, _log(rng, 1, most), _log(rng, 1, most)]), ragged=ragged)
    if kind == "account":
        return dict(case, prefix=rng.choice([0, 0, _log(rng, 1, 2000)]), groups=rng.randint(1, min(seqs, 3)))
    return dict(case, prefix=_log(rng, 16, 16000), groups=rng.choice([1, 1, rng.randint(1, min(seqs, 8))]))


# ------------------------------------------------------------------ inputs

def _sizes(case):
    """(rows, own positions before them) of each sequence.  ragged 0: all alike; 1: contexts down to a
    quarter of the longest, rows down to a third; 2: one or two chunks, then single tokens."""
    n, got = case["seqs"], []
    for i in range(n):
        size, rows = case["len"], case.get("rows", 0)
        if case["ragged"]:
            size = max(1, round(size * (1 - 0.75 * i / n)))
            rows = max(1, round(rows * (1 - 0.67 * i / n))) if case["ragged"] == 1 else (rows if i == 0 else max(1, rows // 3) if i == 1 else 1)
        rows = min(rows, size) if case["kind"] != "evict" else 0
        got.append((rows, size - rows))
    return got


def _shared(case):
    """(first sequence of each group and behind the last, prefix length of each): the lengths go down to half."""
    n, groups = case["seqs"], case.get("groups", 1) if case.get("prefix", 0) else 0
    return [g * n // groups for g in range(groups + 1)] if groups else [0], \
        [max(1, round(case["prefix"] * (1 - 0.5 * g / groups))) for g in range(groups)]


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _paged(case, g, seed):
    """The page pool with quantised rows in it, the pages of sequences and prefixes in no order, and the batch."""
    sizes, (first, prefix), ps, kv, hd = _sizes(case), _shared(case), case["page"], case["kv_heads"], case["hd"]
    per = [-(-(r + p) // ps) for r, p in sizes]
    per_prefix = [-(-p // ps) for p in prefix]
    n_pages = sum(per) + sum(per_prefix) + 3
    order = list(range(n_pages - 1))
    random.Random(seed).shuffle(order)
    at = 0

    def table(counts):
        nonlocal at
        rows = []
        for c in counts:  # behind a sequence's pages stands one that is nobody's
            rows.append(order[at:at + c] + [n_pages - 1] * (max(counts) - c))
            at += c
        return torch.tensor(rows, dtype=torch.int32, device=DEV).view(len(counts), -1)

    i32 = dict(dtype=torch.int32, device=DEV)
    starts = [0]
    for r, _ in sizes:
        starts.append(starts[-1] + r)

    def codes():
        """Codes of values near a normal distribution, three deviations wide."""
        x = torch.randn((n_pages, kv, ps, hd), generator=g, device=DEV)
        return x.mul_(40).round_().clamp_(-127, 127).add_(128).to(torch.uint8)

    def scales():
        return torch.rand((n_pages, kv, ps), generator=g, device=DEV) * 0.03 + 0.01

    k = codes()
    # values lie in blocks of 16 slots, the slots innermost
    v = codes().view(n_pages, kv, ps // 16, 16, hd).transpose(3, 4).contiguous()
    s = {"case": dict(case), "k_codes": k, "v_codes": v, "k_scale": scales(), "v_scale": scales(), "sizes": sizes,
         "pages": table(per), "pos": torch.tensor([p for _, p in sizes], **i32),
         "row_start": torch.tensor(starts, **i32), "max_rows": max(r for r, _ in sizes),
         "max_len": max(r + p for r, p in sizes), "rows": starts[-1]}
    s["row_seq"] = torch.tensor([n for n, (r, _) in enumerate(sizes) for _ in range(r)], dtype=torch.long, device=DEV)
    s["row_i"] = torch.tensor([j for r, _ in sizes for j in range(r)], dtype=torch.long, device=DEV)
    if prefix:
        s["p_pages"], s["p_len"] = table(per_prefix), torch.tensor(prefix, **i32)
        g_start = [starts[f] for f in first]
        s["p_row_start"], s["p_max_len"] = torch.tensor(g_start, **i32), max(prefix)
        s["p_max_rows"] = max(b - a for a, b in zip(g_start, g_start[1:]))
        s["row_group"] = torch.tensor([n for n in range(len(prefix)) for _ in range(g_start[n], g_start[n + 1])], dtype=torch.long, device=DEV)
        s["row_in_group"] = torch.tensor([j for a, b in zip(g_start, g_start[1:]) for j in range(b - a)], dtype=torch.long, device=DEV)
        s["prefix_of"] = [n for n, (a, b) in enumerate(zip(first, first[1:])) for _ in range(a, b)]
    return s


def _weights(case, g, ld):
    """Accumulated weights: a few heavy positions, many light ones, some equal, some never seen."""
    shape = (case["seqs"], case["kv_heads"], ld)
    w = torch.exp(2 * torch.randn(shape, generator=g, device=DEV) - 3)
    w = torch.where(torch.rand(shape, generator=g, device=DEV) < 0.3, (w * 256).round() / 256, w)
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.05, 0.0, w)


def prepare(case, seed):
    g = _gen(seed)
    s = _paged(case, g, seed)
    kv, hd, dt, seqs, ld = case["kv_heads"], case["hd"], DTYPES[case["dtype"]], case["seqs"], s["max_len"] + 8
    if case["kind"] != "prefix":
        s["weight"] = _weights(case, g, ld)
    i32 = dict(dtype=torch.int32, device=DEV)
    if case["kind"] != "evict":
        s["q"] = (torch.randn((s["rows"], case["heads"] * hd), generator=g, device=DEV) * 2).to(dt)
        s["out"] = torch.empty_like(s["q"])
    else:
        size = [p for _, p in s["sizes"]]
        # positions that earlier evictions left, in no order, and how many they dropped
        s["filled"] = torch.tensor([min(n, case["keep"]) if case["again"] else 0 for n in size], **i32)
        s["shift"] = torch.tensor([n // 3 if case["again"] else 0 for n in size], **i32)
        s["token"] = torch.zeros((seqs, kv, ld), **i32)
        if case["again"]:
            for n in range(seqs):
                f, d = min(size[n], case["keep"]), size[n] // 3
                s["token"][n, :, :f] = torch.rand((kv, f + d), generator=g, device=DEV).argsort(dim=1)[:, :f].int()
        for name in ("keep", "sink", "recent"):
            s[name] = torch.full((seqs,), case[name], **i32)
        s["weight_out"], s["token_out"] = torch.zeros_like(s["weight"]), torch.zeros_like(s["token"])
        s["filled_out"], s["shift_out"] = torch.zeros_like(s["filled"]), torch.zeros_like(s["shift"])
        s["held"] = torch.zeros_like(s["filled"])
        left = [min(n, case["keep"]) for n in size]
        s["left"] = sum(left)
        s["left_start"] = torch.tensor([sum(left[:n]) for n in range(seqs + 1)], **i32)
        s["left_seq"] = torch.tensor([n for n in range(seqs) for _ in range(left[n])], dtype=torch.long, device=DEV)
        s["left_j"] = torch.cat([torch.arange(n, device=DEV) for n in left])
        s["zero"] = torch.zeros((seqs,), **i32)
        s["k_out"] = torch.empty((s["left"], kv * hd), dtype=dt, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    if own:
        _handles(s)
    return s


def _engine():
    where = os.path.join(ROOT, "bit-ttt-engine_amd")
    if where not in sys.path:
        sys.path.insert(1, where)
    import bitlinear
    return bitlinear


def _handles(s):
    """The cache, batches, accounts and workspace that a program keeps."""
    bl, case = _engine(), s["case"]
    s["cache"] = bl.PagedKVCacheQ8.of(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    s["batch"] = bl.PagedBatch(s["row_start"], s["pos"], s["pages"], s["rows"], s["max_rows"], s["max_len"])
    s["prefix"] = bl.PagedBatch(s["p_row_start"], s["p_len"], s["p_pages"], s["rows"], s["p_max_rows"],
                                s["p_max_len"]) if "p_len" in s else None
    if case["kind"] == "prefix":
        s["space"] = bl.paged_attention_prefix_workspace(s["cache"], s["batch"], s["prefix"], case["heads"])
    elif case["kind"] == "account":
        s["account"] = bl.KVAccount.of(s["weight"])
        s["space"] = bl.paged_attention_account_workspace(s["cache"], s["batch"], case["heads"], prefix=s["prefix"])
    else:
        s["account"] = bl.KVAccount.of(s["weight"], s["token"], s["filled"], s["shift"])
        s["account_out"] = bl.KVAccount.of(s["weight_out"], s["token_out"], s["filled_out"], s["shift_out"])
        s["space"] = bl.paged_evict_workspace(s["cache"], s["batch"])
        s["left_batch"] = bl.PagedBatch(s["left_start"], s["zero"], s["pages"], s["left"], case["keep"], case["keep"])


# ------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if kind == "prefix":
        if own:
            return _engine().paged_attention_prefix(s["q"], s["cache"], s["batch"], s["prefix"], out=s["out"],
                                                    workspace=s["space"])
        return _attention(s)[0]
    if kind == "account":
        if own:
            o = _engine().paged_attention_account(s["q"], s["cache"], s["batch"], s["account"], prefix=s["prefix"],
                                                  out=s["out"], workspace=s["space"])
            return o, s["weight"]
        return _account(s)
    return _evict(s)


def _gather(s, pages, size):
    """The first `size` keys and values of each row of a page table: [row, head, position, value]."""
    ps = s["case"]["page"]
    j = torch.arange(size, device=DEV)
    page, slot = pages[:, j // ps].long()[:, None], (j % ps)[None, None]
    head = torch.arange(s["case"]["kv_heads"], device=DEV)[None, :, None]
    k = (s["k_codes"][page, head, slot].float() - 128) * s["k_scale"][page, head, slot][..., None]
    v = (s["v_codes"][page, head, slot // 16, :, slot % 16].float() - 128) * s["v_scale"][page, head, slot][..., None]
    return k, v


def _part(s, row_start, pages, rows, size, seen):
    """Softmax parts of row lists (row_start) over the positions of a page table, seen [list, row, position]:
    the largest score, the weights against it, their sum and the values they weigh, [list, head, row, group, ...]."""
    case = s["case"]
    kv, hd = case["kv_heads"], case["hd"]
    group, lists = case["heads"] // kv, pages.shape[0]
    k, v = _gather(s, pages, size)
    at = (row_start[:-1, None].long() + torch.arange(rows, device=DEV)).clamp(max=s["rows"] - 1)
    q = s["q"].float()[at].view(lists, rows, kv, group, hd).transpose(1, 2).reshape(lists, kv, rows * group, hd)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    w = w.view(lists, kv, rows, group, size).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = w.amax(dim=4)
    w = torch.exp(w - top.clamp(min=-1e30)[..., None])
    o = torch.matmul(w.view(lists, kv, rows * group, size), v).view(lists, kv, rows, group, hd)
    return top, w, w.sum(dim=4), o


def _attention(s):
    """(outputs; the own positions' softmax weights [sequence, head, row, group, position])."""
    case = s["case"]
    i, j = torch.arange(s["max_rows"], device=DEV), torch.arange(s["max_len"], device=DEV)
    seen = j <= (s["pos"].long()[:, None] + i)[..., None]
    top, w, total, o = _part(s, s["row_start"], s["pages"], s["max_rows"], s["max_len"], seen)
    at = s["row_seq"], slice(None), s["row_i"]
    t, n, x = top[at], total[at], o[at]
    if "p_len" in s:
        j = torch.arange(s["p_max_len"], device=DEV)
        seen = (j < s["p_len"].long()[:, None])[:, None].expand(-1, s["p_max_rows"], -1)
        p_top, _, p_total, p_o = _part(s, s["p_row_start"], s["p_pages"], s["p_max_rows"], s["p_max_len"], seen)
        p = s["row_group"], slice(None), s["row_in_group"]
        both = torch.maximum(t, p_top[p])
        a, b = torch.exp(t - both), torch.exp(p_top[p] - both)
        n, x = a * n + b * p_total[p], a[..., None] * x + b[..., None] * p_o[p]
        total = torch.ones_like(total)
        total[at] = n / a.clamp(min=1e-37)  # the sum against the own positions' largest score
    out = (x / n[..., None]).reshape(s["q"].shape).to(s["q"].dtype)
    return out, w.div_(total[..., None]) if case["kind"] == "account" else None


def _account(s):
    out, w = _attention(s)
    there = torch.arange(s["max_rows"], device=DEV) < (s["row_start"][1:] - s["row_start"][:-1])[:, None]
    w = (w * there[:, None, :, None, None]).sum(dim=(2, 3))
    j = torch.arange(s["max_len"], device=DEV)[None, None]
    pos, end = s["pos"][:, None, None], (s["pos"] + s["row_start"][1:] - s["row_start"][:-1])[:, None, None]
    before = s["weight"][:, :, :s["max_len"]]
    # a row's own position begins with this call; those behind the sequence stay as they are
    before.copy_(torch.where(j < end, torch.where(j < pos, before, 0.0) + w, before))
    return out, s["weight"]


def _evict(s):
    case = s["case"]
    kv, ps, most = case["kv_heads"], case["page"], min(case["keep"], s["max_len"])
    if own:
        bl = _engine()
        bl.paged_evict(s["cache"], s["batch"], s["account"], s["keep"], sink=s["sink"], recent=s["recent"],
                       max_keep=case["keep"], out=s["account_out"], held=s["held"], workspace=s["space"])
        k, v = bl.paged_read(s["cache"], s["left_batch"], k_out=s["k_out"], v_out=s["v_out"])
        return s["held"], s["filled_out"], s["shift_out"], s["weight_out"], s["token_out"], k, v
    size = s["max_len"]
    j = torch.arange(size, device=DEV)[None, None]
    n, keep, shift = s["pos"][:, None, None], s["keep"][:, None, None], s["shift"][:, None, None]
    weight = s["weight"][:, :, :size]
    token = torch.where(j < s["filled"][:, None, None], s["token"][:, :, :size], (j + shift).int())
    safe = (token < s["sink"][:, None, None]) | (token >= n + shift - s["recent"][:, None, None])
    key = torch.where(j < n, torch.where(safe, math.inf, weight), -1.0)
    order = torch.argsort(key, dim=2, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(2, order, j.expand_as(order).contiguous())
    kept = (rank < keep) & (j < n)
    hole, source = ~kept & (j < torch.minimum(keep, n)), kept & (j >= keep)
    # the n-th hole takes the n-th source
    nth = torch.where(source, torch.cumsum(source, dim=2) - 1, size)
    which = torch.zeros((*order.shape[:2], size + 1), dtype=torch.long, device=DEV).scatter_(2, nth, j.expand_as(order).contiguous())
    come = torch.where(hole, which.gather(2, (torch.cumsum(hole, dim=2) - 1).clamp(min=0)), j)[:, :, :most]
    held = torch.minimum(s["keep"], s["pos"])
    there = j[:, :, :most] < held[:, None, None]
    s["weight_out"][:, :, :most] = torch.where(there, weight.gather(2, come), s["weight_out"][:, :, :most])
    s["token_out"][:, :, :most] = torch.where(there, token.gather(2, come), s["token_out"][:, :, :most])
    s["held"].copy_(held)
    s["filled_out"].copy_(held)
    s["shift_out"].copy_(s["shift"] + s["pos"] - held)
    # every position that stays, from where it was to where it is to be
    seq, head = torch.arange(case["seqs"], device=DEV)[:, None, None], torch.arange(kv, device=DEV)[None, :, None]
    come = torch.where(there, come, j[:, :, :most])
    fp, fs = s["pages"][seq, come // ps].long(), come % ps
    tp, ts = s["pages"][seq, j[:, :, :most] // ps].long(), (j[:, :, :most] % ps).expand_as(come)
    s["k_codes"][tp, head, ts] = s["k_codes"][fp, head, fs]
    s["v_codes"][tp, head, ts // 16, :, ts % 16] = s["v_codes"][fp, head, fs // 16, :, fs % 16]
    s["k_scale"][tp, head, ts] = s["k_scale"][fp, head, fs]
    s["v_scale"][tp, head, ts] = s["v_scale"][fp, head, fs]
    page, slot = s["pages"][s["left_seq"], s["left_j"] // ps].long()[:, None], (s["left_j"] % ps)[:, None]
    head = torch.arange(kv, device=DEV)[None]
    k = (s["k_codes"][page, head, slot].float() - 128) * s["k_scale"][page, head, slot][..., None]
    v = (s["v_codes"][page, head, slot // 16, :, slot % 16].float() - 128) * s["v_scale"][page, head, slot][..., None]
    shape, dt = s["k_out"].shape, s["k_out"].dtype
    return s["held"], s["filled_out"], s["shift_out"], s["weight_out"], s["token_out"], k.reshape(shape).to(dt), v.reshape(shape).to(dt)


def work(case):
    sizes, kv, hd, size = _sizes(case), case["kv_heads"], case["hd"], 4 if case["dtype"] == "f32" else 2
    held = kv * (2 * hd + 8)  # a position's codes and scales
    if case["kind"] == "evict":
        bytes_ = 0
        for _, n in sizes:
            left = min(n, case["keep"])
            moved = left * (n - left) / n  # of weights in no order
            # weights read, and recorded positions; both written; rows moved; what is left read and put out
            bytes_ += kv * (4 * n + (4 * left if case["again"] else 0) + 8 * left) + 2 * moved * held
            bytes_ += left * (held + 2 * size * kv * hd)
        return {"bytes": bytes_, "flops": 4 * kv * sum(min(n, case["keep"]) for _, n in sizes) * hd}
    first, prefix = _shared(case)
    rows = sum(r for r, _ in sizes)
    seen = sum(r * p + r * (r + 1) // 2 for r, p in sizes)
    seen += sum(p * sum(r for r, _ in sizes[a:b]) for p, a, b in zip(prefix, first, first[1:]))
    bytes_ = (sum(r + p for r, p in sizes) + sum(prefix)) * held + 2 * rows * case["heads"] * hd * size
    if case["kind"] == "account":  # weights read where they are added to, and written
        bytes_ += 4 * kv * sum(r + 2 * p for r, p in sizes)
    return {"bytes": bytes_, "flops": 4 * seen * case["heads"] * hd}


# ------------------------------------------------------------------ in 64 bits

def _dense(s, table, n):
    """[head, position, value] of the first n positions of a row of a page table."""
    ps, kv, hd = s["case"]["page"], s["case"]["kv_heads"], s["case"]["hd"]
    pages = table[:-(-n // ps)].long()
    k = (s["k_codes"][pages].double() - 128) * s["k_scale"][pages].double().unsqueeze(-1)
    v = s["v_codes"][pages].transpose(3, 4).reshape(len(pages), kv, ps, hd).double() - 128
    v = v * s["v_scale"][pages].double().unsqueeze(-1)
    return [x.transpose(0, 1).reshape(kv, -1, hd)[:, :n] for x in (k, v)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(s)
    kv, hd = case["kv_heads"], case["hd"]
    _, prefix = _shared(case)
    os_, weight = [], s["weight"].double() if case["kind"] == "account" else None
    for n, (r, p) in enumerate(s["sizes"]):
        k, v = _dense(s, s["pages"][n], r + p)
        behind = prefix[s["prefix_of"][n]] if prefix else 0
        if behind:
            pk, pv = _dense(s, s["p_pages"][s["prefix_of"][n]], behind)
            k, v = torch.cat((pk, k), dim=1), torch.cat((pv, v), dim=1)
        a = int(s["row_start"][n])
        q = s["q"][a:a + r].double().view(r, kv, -1, hd)
        o = torch.empty_like(q)
        late = torch.arange(behind + r + p, device=DEV)[None] > torch.arange(behind + p, behind + p + r, device=DEV)[:, None]
        for h in range(kv):
            if weight is not None:
                weight[n, h, p:p + r] = 0
            for e in range(q.shape[2]):
                w = (q[:, h, e] @ k[h].t().contiguous()) / math.sqrt(hd)
                w = torch.softmax(w.masked_fill(late, -math.inf), dim=1)
                o[:, h, e] = w @ v[h]
                if weight is not None:
                    weight[n, h, :r + p] += w[:, behind:].sum(dim=0)
        os_.append(o.reshape(r, -1))
    return torch.cat(os_) if weight is None else (torch.cat(os_), weight)


def _exact_evict(s):
    """The choice by sorting each head's positions on the host."""
    case = s["case"]
    weight = s["weight"].cpu().numpy()
    token, filled, shift = (s[x].cpu().numpy() for x in ("token", "filled", "shift"))
    out = torch.zeros(s["weight"].shape, dtype=torch.float64)
    ks, vs = [], []
    for n, (_, size) in enumerate(s["sizes"]):
        k, v = _dense(s, s["pages"][n], size)
        left, come = min(size, case["keep"]), []
        for h in range(case["kv_heads"]):
            place = [int(token[n, h, j]) if j < filled[n] else j + int(shift[n]) for j in range(size)]
            late = size + int(shift[n]) - case["recent"]
            w = weight[n, h, :size].tolist()
            ranked = sorted(range(size), key=lambda j: (not (place[j] < case["sink"] or place[j] >= late),
                                                        0.0 if place[j] < case["sink"] or place[j] >= late else -w[j], j))
            stay = set(ranked[:left])
            movers = iter(sorted(j for j in stay if j >= left))
            come.append([j if j in stay else next(movers) for j in range(left)])
            out[n, h, :left] = torch.tensor([w[j] for j in come[-1]], dtype=torch.float64)
        at = torch.tensor(come, device=DEV)[..., None].expand(-1, -1, case["hd"])
        ks.append(k.gather(1, at).transpose(0, 1).reshape(left, -1))
        vs.append(v.gather(1, at).transpose(0, 1).reshape(left, -1))
    return None, None, None, out, None, torch.cat(ks), torch.cat(vs)
