"""Performance cases of the paged-cache operators: rotary positions, the append to the pages, attention of new
tokens and of prompts over them, and the pages' own bookkeeping.

listed() are the cases, draw() gives more of the same ranges. With `own` false run() computes a case with
elementary torch operations on the documented layouts; with `own` true it makes the calls of velox_amd.paged.
exact() recomputes the numbers in float64, sequence by sequence.

A page holds `page` positions of one layer: for every KV head the K rows [page][d], then for every KV head the
V blocks [page / 32][d][32], position r of a block at slot 8 ((r % 16) / 4) + 4 (r / 16) + r % 4 -- the layout
of an arena's KV cache. The pool is [layers][pages][2 * hkv * page * d]; table [sequences][max_pages] holds page
numbers, -1 where there is none; lens the positions of each sequence; refs how many table entries name a page.
"""
from __future__ import annotations

import math

import torch

own = False

# head shapes of the builtin configurations: q heads, KV heads, head size
HEADS = {"smollm_135m": (9, 3, 64), "llama3_8b": (32, 8, 128), "qwen2_5_7b": (28, 4, 128), "qwen2_72b": (64, 8, 128)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------------

def listed():
    return [
        # one user of the smallest model at a short context: the decode step's own fp32 activations, launch latency
        {"name": "token_smollm_b1_len700", "op": "token", "model": "smollm_135m", "seqs": 1, "len": 700, "spread": 0,
         "page": 32, "q": "f32", "kv": "bf16", "window": 0, "sinks": 0},
        # serving: 32 sequences of unequal length, q a slice of the fused q/k/v rows
        {"name": "token_qwen7b_b32_len2100", "op": "token", "model": "qwen2_5_7b", "seqs": 32, "len": 2100, "spread": 1500,
         "page": 64, "q": "f32", "kv": "bf16", "window": 0, "sinks": 0},
        # a few very long contexts: the cache's bytes are all that counts
        {"name": "token_llama8b_b4_len131000", "op": "token", "model": "llama3_8b", "seqs": 4, "len": 131000,
         "spread": 40000, "page": 128, "q": "bf16", "kv": "bf16", "window": 0, "sinks": 0},
        # short prompts of unequal length, some of one token, with a small window and sinks
        {"name": "prompt_smollm_ragged", "op": "prompt", "model": "smollm_135m", "seqs": 7, "rows": 70, "before": 0,
         "spread": 69, "page": 32, "q": "f32", "kv": "f16", "window": 33, "sinks": 4},
        # a long prompt in one call through a window
        {"name": "prompt_llama8b_8192_window", "op": "prompt", "model": "llama3_8b", "seqs": 1, "rows": 8192, "before": 0,
         "spread": 0, "page": 64, "q": "bf16", "kv": "bf16", "window": 4096, "sinks": 4},
        # chunks of four prompts behind earlier positions, everything visible
        {"name": "prompt_qwen7b_chunks", "op": "prompt", "model": "qwen2_5_7b", "seqs": 4, "rows": 500, "before": 4000,
         "spread": 120, "page": 64, "q": "bf16", "kv": "bf16", "window": 0, "sinks": 0},
        # the append of a batched decode step: one fp32 row of q, k and v for each sequence
        {"name": "append_qwen7b_decode32", "op": "append", "model": "qwen2_5_7b", "seqs": 32, "rows": 1, "before": 2000,
         "spread": 0, "pad": 0, "page": 64, "q": "f32", "kv": "bf16", "rot": 128, "layout": "half", "scaling": "none",
         "theta": 1e6, "factor": 1.0, "orig": 8192},
        # the append of prompts: bf16 rows, frequencies scaled in bands, padding behind the last sequence
        {"name": "append_llama8b_prompts", "op": "append", "model": "llama3_8b", "seqs": 5, "rows": 2047, "before": 100,
         "spread": 900, "pad": 37, "page": 128, "q": "bf16", "kv": "bf16", "rot": 128, "layout": "half", "scaling": "bands",
         "theta": 5e5, "factor": 8.0, "orig": 8192},
        # rotation alone, interleaved over half of each head, at far positions of a stretched context
        {"name": "rope_72b_far_partial", "op": "rope", "model": "qwen2_72b", "rows": 4001, "far": 1000000, "q": "f16",
         "rot": 64, "layout": "interleaved", "scaling": "yarn", "theta": 1e6, "factor": 32.0, "orig": 32768},
        # two users' samples forked and extended by one token: latency
        {"name": "pages_small_fork", "op": "pages", "model": "smollm_135m", "layers": 30, "users": 2, "width": 4, "len": 75,
         "page": 32, "add": 1, "spare": 8},
        # sixteen users with four samples each at unequal lengths: shared last pages are copied in every layer
        {"name": "pages_qwen7b_fork64", "op": "pages", "model": "qwen2_5_7b", "layers": 28, "users": 16, "width": 4,
         "len": 900, "page": 64, "add": 1, "spare": 100},
        # half of the sequences end, the rest moves to the front of the pool
        {"name": "compact_llama8b", "op": "compact", "model": "llama3_8b", "layers": 32, "users": 40, "width": 1, "len": 1000,
         "page": 128, "add": 0, "spare": 30},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("token", "token", "prompt", "prompt", "rope", "append", "pages", "compact"))
    model = rng.choice(tuple(HEADS))
    page = rng.choice((32, 64, 96, 128, 256))
    q, kv = rng.choice((("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")))
    window = rng.choice((0, 0, _log(rng, 1, 5000)))
    mask = {"window": window, "sinks": rng.randint(0, 8) if window else 0}
    if op == "token":
        seqs = _log(rng, 1, 64)
        length = _log(rng, 1, 200000 // seqs)
        return {"op": op, "model": model, "seqs": seqs, "len": length, "spread": rng.randint(0, length), "page": page,
                "q": q, "kv": kv, **mask}
    if op == "prompt":
        seqs = _log(rng, 1, 8)
        rows = _log(rng, 1, 2800 // seqs)
        return {"op": op, "model": model, "seqs": seqs, "rows": rows, "before": rng.choice((0, _log(rng, 1, 3000))),
                "spread": rng.randint(0, rows), "page": page, "q": q, "kv": kv, **mask}
    if op in ("pages", "compact"):
        width = rng.randint(1, 6) if op == "pages" else 1
        return {"op": op, "model": model, "layers": rng.randint(1, 8), "users": _log(rng, 1, 24), "width": width,
                "len": _log(rng, 1, 1000), "page": page, "add": rng.choice((1, 1, _log(rng, 1, 100))) if op == "pages" else 0,
                "spare": rng.randint(0, 60)}
    d = HEADS[model][2]
    turn = {"rot": rng.choice((d, d, d // 2, d // 4 + 2)), "layout": rng.choice(("half", "interleaved")),
            "scaling": rng.choice(("none", "linear", "bands", "yarn")), "theta": rng.choice((1e4, 5e5, 1e6)),
            "factor": rng.choice((2.0, 8.0, 32.0)), "orig": rng.choice((2048, 8192, 32768))}
    if op == "rope":
        return {"op": op, "model": model, "rows": _log(rng, 1, 8000), "far": _log(rng, 10, 2000000), "q": rng.choice(("f32", "f16", "bf16")), **turn}
    seqs = _log(rng, 1, 64)
    return {"op": op, "model": model, "seqs": seqs, "rows": _log(rng, 1, 8000 // seqs), "before": rng.choice((0, _log(rng, 1, 3000))),
            "spread": rng.choice((0, 5)), "pad": rng.choice((0, 3)), "page": page, "q": q, "kv": kv, **turn}


# ---- what a case's numbers say --------------------------------------------------------------------

def _ragged(n, base, spread):
    """n whole numbers of [base - spread, base], at least 1, the first of them base."""
    return [max(1, base - (i * 7919) % (spread + 1)) for i in range(n)]


def _lengths(case):
    """(new rows, positions with them) of every sequence."""
    n = case["seqs"]
    if case["op"] == "token":
        return [1] * n, _ragged(n, case["len"], case["spread"])
    rows = _ragged(n, case["rows"], case["spread"])
    return rows, [r + case["before"] for r in rows]


def _visible(rows, length, window, sinks):
    """(row, position) pairs that the mask leaves of one sequence, and positions that some row sees."""
    first = length - rows
    pairs = 0
    for t in range(first, length):
        near = min(t + 1, window) if window else t + 1
        pairs += near + min(sinks, t + 1 - near)
    low = max(0, first - window + 1) if window else 0
    return pairs, length - low + min(sinks, low)


def _families(case):
    """For "pages" and "compact": each sequence's parent, length and, for "pages", new length; user u's
    sequences share the pages of its first three quarters."""
    users, width = case["users"], case["width"]
    lens = [x for x in _ragged(users, case["len"], case["len"] // 2) for _ in range(width)]
    src = [s - s % width + (s * s + 1) % width for s in range(users * width)]
    if users > 1 and case["op"] == "pages":
        src[-1] = -1  # the last sequence ends
    return src, lens


def _layout(case):
    """(page numbers [sequence][page] before the permutation, pages in all) of a "pages" or "compact" pool."""
    _, lens = _families(case)
    width, page = case["width"], case["page"]
    rows, used = [], 0
    for s, n in enumerate(lens):
        whole = (n * 3 // 4) // page if width > 1 else 0
        if s % width == 0:
            shared = list(range(used, used + whole))
            used += whole
        own_pages = -(-n // page) - whole
        rows.append(shared + list(range(used, used + own_pages)))
        used += own_pages
    new = sum(-(-(n + case["add"]) // page) - -(-n // page) + 1 for n in lens)
    return rows, used + new + case["spare"]


def work(case):
    hq, hkv, d = HEADS[case["model"]]
    if case["op"] in ("token", "prompt"):
        rows, lens = _lengths(case)
        seen = [_visible(r, n, case["window"], case["sinks"]) for r, n in zip(rows, lens)]
        return {"bytes": sum(s for _, s in seen) * 2 * hkv * d * SIZE[case["kv"]] + 2 * sum(rows) * hq * d * SIZE[case["q"]],
                "flops": 4 * hq * d * sum(p for p, _ in seen)}
    if case["op"] == "rope":
        n = case["rows"] * hq * d
        return {"bytes": 2 * n * SIZE[case["q"]] + 4 * case["rows"], "flops": 3 * case["rows"] * hq * case["rot"]}
    if case["op"] == "append":
        t = sum(_lengths(case)[0])
        return {"bytes": t * d * ((2 * hq + 2 * hkv) * SIZE[case["q"]] + 2 * hkv * SIZE[case["kv"]]),
                "flops": 3 * t * (hq + hkv) * case["rot"]}
    src, lens = _families(case)
    page_bytes = case["layers"] * 2 * hkv * case["page"] * d * 2
    rows, n_pages = _layout(case)
    if case["op"] == "compact":
        live = sum(len(r) for s, r in enumerate(rows) if s % 2)  # the others end
        moved = live * (n_pages - live) // n_pages               # of pages spread evenly
    else:
        last = [rows[p][-1] if p >= 0 and lens[p] % case["page"] else None for p in src]
        moved = sum(p is not None for p in last) - len({p for p in last if p is not None})
    return {"bytes": 2 * moved * page_bytes + 8 * sum(len(r) for r in rows) + 4 * n_pages, "flops": 0}


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + tag) % (1 << 61))


def _randn(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _fill(shape, g, dtype):
    """Random values of a large pool, made in slices."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda", dtype=torch.float32 if n < 1 << 20 else dtype)
    return t


def _paged(case, seed, lens):
    """pool, table and lens of a cache of one layer whose pages lie in random order."""
    _, hkv, d = HEADS[case["model"]]
    page = case["page"]
    need = [-(-n // page) for n in lens]
    n_pages, width = sum(need) + 3, max(need) + 1
    order = torch.randperm(n_pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    pool = _fill((1, n_pages, 2 * hkv * page * d), _gen(seed, 2), TYPES[case["kv"]])
    return {"pool": pool, "table": table, "lens": _ints(lens)}


def _frequencies(case):
    """Radians per position of each pair, and the factor on the rotated values."""
    r, theta, factor, orig = case["rot"], case["theta"], case["factor"], case["orig"]
    f = [theta ** (-2.0 * j / r) for j in range(r // 2)]
    if case["scaling"] == "linear":
        return [x / factor for x in f], 1.0
    if case["scaling"] == "bands":  # long waves are stretched, short ones kept, between 1 and 4 turns mixed
        out = []
        for x in f:
            turns = orig * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / 3.0))
            out.append(x * (keep + (1 - keep) / factor))
        return out, 1.0
    if case["scaling"] == "yarn":  # a ramp over the pairs between 32 turns and one turn in `orig` positions
        def pair(turns):
            return r * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
        out = []
        for j, x in enumerate(f):
            stretch = min(1.0, max(0.0, (j - low) / max(high - low, 0.001)))
            out.append(x * (1 - stretch) + x / factor * stretch)
        return out, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rope_handle(case):
    from velox_amd import paged
    return paged.Rope(case["rot"], theta=case["theta"], layout=case["layout"], scaling=case["scaling"], factor=case["factor"],
                      original_len=case["orig"])


def _cache_handle(case, s):
    from velox_amd import paged
    _, hkv, d = HEADS[case["model"]]
    return paged.PagedCache.over(s["pool"], s["table"], s["lens"], page_size=case["page"], num_kv_heads=hkv, head_dim=d,
                                 refs=s.get("refs"))


def prepare(case, seed):
    hq, hkv, d = HEADS[case["model"]]
    s = {"case": case}
    if case["op"] == "rope":
        s["x"] = _randn((case["rows"], hq, d), _gen(seed, 3), TYPES[case["q"]])
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=_gen(seed, 4), device="cuda", dtype=torch.int32)
        s["freq"], s["amp"] = torch.tensor(_frequencies(case)[0], dtype=torch.float64, device="cuda"), _frequencies(case)[1]
        if own:
            s["rope"] = _rope_handle(case)
        return s
    if case["op"] in ("pages", "compact"):
        src, lens = _families(case)
        rows, n_pages = _layout(case)
        order = torch.randperm(n_pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
        width = max(len(r) for r in rows) + -(-case["add"] // case["page"]) + 1
        flat = [r + [-1] * (width - len(r)) for r in rows]
        table = _ints(flat)
        table = torch.where(table >= 0, order[table.clamp(min=0).long()], table)
        refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        refs.index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
        s["pool"] = _fill((case["layers"], n_pages, 2 * hkv * case["page"] * d), _gen(seed, 2), torch.bfloat16)
        s["before"] = (table, _ints(lens), refs)
        s["table"], s["lens"], s["refs"] = (t.clone() for t in s["before"])
        s["src"], s["add"] = _ints(src), torch.full((len(src),), case["add"], dtype=torch.int32, device="cuda")
        s["ended"] = _ints(list(range(0, len(src), 2)))
        if own:
            s["cache"] = _cache_handle(case, s)
        return s
    rows, lens = _lengths(case)
    s.update(_paged(case, seed, lens))
    total, pad = sum(rows), case.get("pad", 0)
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    # q, k and v as slices of the rows that one product leaves
    s["qkv"] = _randn((total + pad, (hq + 2 * hkv) * d), _gen(seed, 3), TYPES[case["q"]])
    s["q"] = s["qkv"][:, :hq * d].unflatten(1, (hq, d))
    s["start"], s["rows"], s["most"], s["last"] = _ints(start), total, max(rows), max(lens)
    if case["op"] == "append":
        s["k"] = s["qkv"][:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        s["v"] = s["qkv"][:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        s["out"] = torch.zeros(total + pad, hq, d, dtype=TYPES[case["q"]], device="cuda")
        s["freq"], s["amp"] = torch.tensor(_frequencies(case)[0], dtype=torch.float64, device="cuda"), _frequencies(case)[1]
        if own:
            s["rope"] = _rope_handle(case)
    if own:
        s["cache"] = _cache_handle(case, s)
        if case["op"] == "token":
            s["space"] = s["cache"].attention_workspace(hq, max_len=s["last"])
        elif case["op"] == "prompt":
            s["space"] = s["cache"].prompt_workspace(hq, max_len=s["last"], max_rows=s["most"], total_rows=total)
    return s


# ---- one pass -------------------------------------------------------------------------------------

SLOT = [8 * ((r % 16) // 4) + 4 * (r // 16) + r % 4 for r in range(32)]  # of position r in a V block


def _gathered(s, hkv, d, page):
    """K and V of every table entry's positions, fp32 [sequence][KV head][position][d]; entries without a page
    give page 0, which the mask leaves out."""
    table = s["table"]
    n, m = table.shape
    pages = s["pool"][0][table.clamp(min=0).long()].view(n, m, 2, hkv, page * d)
    k = pages[:, :, 0].view(n, m, hkv, page, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, m * page, d)
    slot = torch.tensor(SLOT, device=table.device)
    v = pages[:, :, 1].view(n, m, hkv, page // 32, d, 32)[..., slot].permute(0, 2, 1, 3, 5, 4).reshape(n, hkv, m * page, d)
    return k.float(), v.float()


def _plain_attention(s, q):
    """q [sequence][row][q head][d] padded in front to the longest, so that the last row is the last position."""
    case = s["case"]
    hq, hkv, d = HEADS[case["model"]]
    k, v = _gathered(s, hkv, d, case["page"])
    n, rows = q.shape[:2]
    span = k.shape[2]
    at = s["lens"].view(n, 1, 1) - rows + torch.arange(rows, device=q.device).view(1, rows, 1)
    j = torch.arange(span, device=q.device).view(1, 1, span)
    seen = j <= at
    if case["window"]:
        seen &= (j > at - case["window"]) | (j < case["sinks"])
    seen &= (s["table"] >= 0).repeat_interleave(case["page"], 1).view(n, 1, span)
    g = hq // hkv
    q = q.float().view(n, rows, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * rows, d)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(n, hkv, g, rows, span)
    p.masked_fill_(~seen.view(n, 1, 1, rows, span), float("-inf"))
    top = p.amax(4, keepdim=True)
    p.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(4, keepdim=True)
    o = torch.matmul(p.view(n, hkv, g * rows, span), v).view(n, hkv, g, rows, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(n, rows, hq, d)


def _plain_turn(x, positions, s):
    """x [row][head][d] with the first rot values of every head rotated, fp32."""
    case = s["case"]
    angle = positions.double().unsqueeze(1) * s["freq"]
    c, n = ((f(angle) * s["amp"]).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    x = x.float()
    r = case["rot"]
    if case["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * c - b * n, b * c + a * n), 2)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * c - b * n, b * c + a * n), 3).flatten(2)
    return torch.cat((turned, x[..., r:]), 2)


def _row_places(s):
    """Sequence and position of every row of a ragged batch."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["start"], row, right=True) - 1
    return seq, s["lens"][seq] - s["start"][seq + 1] + row


def _plain_append(s):
    case = s["case"]
    _, hkv, d = HEADS[case["model"]]
    page, kv = case["page"], TYPES[case["kv"]]
    n = s["rows"]
    seq, at = _row_places(s)
    s["out"][:n] = _plain_turn(s["q"][:n], at, s).to(s["out"].dtype)
    where = s["table"][seq, (at // page).long()].long().unsqueeze(1)
    inside = (at % page).long().unsqueeze(1)
    head = torch.arange(hkv, device="cuda").unsqueeze(0)
    pages = s["pool"][0].view(-1, 2, hkv, page * d)
    k = pages[:, 0].view(-1, hkv, page, d)
    k[where, head, inside] = _plain_turn(s["k"][:n], at, s).to(kv)
    v = pages[:, 1].view(-1, hkv, page // 32, d, 32)
    slot = torch.tensor(SLOT, device="cuda")[inside % 32]
    v[where, head, inside // 32, :, slot] = s["v"][:n].to(kv)
    return s["out"], s["pool"]


def _plain_fork(s):
    table, lens, refs, src = s["table"], s["lens"], s["refs"], s["src"].long()
    gone = (src < 0)
    new = torch.where(gone.unsqueeze(1), -1, table[src.clamp(min=0)])
    n_pages = refs.numel()
    for t, sign in ((new, 1), (table, -1)):
        hot = t.flatten().long()
        count = torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda")
        refs += count.index_add_(0, torch.where(hot < 0, n_pages, hot), torch.full_like(hot, sign, dtype=torch.int32))[:n_pages]
    lens.copy_(torch.where(gone, 0, lens[src.clamp(min=0)]))
    table.copy_(new)


def _plain_extend(s):
    case = s["case"]
    page = case["page"]
    table, lens, refs, add, pool = s["table"], s["lens"], s["refs"], s["add"], s["pool"]
    n, m = table.shape
    n_pages = refs.numel()
    grows = add > 0
    old, new = (lens + page - 1) // page, (lens + add + page - 1) // page
    fits = grows & (new <= m)
    last = table.gather(1, (old - 1).clamp(min=0).long().unsqueeze(1)).squeeze(1).long()
    shared = fits & (lens % page != 0) & (refs[last.clamp(min=0)] > 1)
    # of the sequences that share a page and all go on, the last one keeps it
    spot = torch.where(shared, last, n_pages)
    wants = torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda").index_add_(0, spot, torch.ones_like(add))
    keeper = torch.full((n_pages + 1,), -1, dtype=torch.int64, device="cuda")
    me = torch.arange(n, device="cuda")
    keeper.scatter_reduce_(0, spot, me, "amax")
    copies = shared & ~((wants[spot] == torch.cat((refs, refs.new_zeros(1)))[spot]) & (keeper[spot] == me))
    need = torch.where(fits, new - old + copies.int(), 0)
    upto = need.cumsum(0)
    done = fits & (upto <= (refs == 0).sum())
    first = upto - need
    free = torch.argsort((refs != 0).int(), stable=True)
    copies &= done
    col = torch.arange(m, device="cuda").unsqueeze(0)
    fresh = done.unsqueeze(1) & (col >= old.unsqueeze(1)) & (col < new.unsqueeze(1))
    swap = copies.unsqueeze(1) & (col == (old - 1).unsqueeze(1))
    rank = (first + copies.int()).unsqueeze(1) + col - old.unsqueeze(1)
    rank = torch.where(swap, first.unsqueeze(1), rank).clamp(0, n_pages - 1).long()
    table.copy_(torch.where(fresh | swap, free[rank].to(torch.int32), table))
    taken = torch.where(fresh | swap, table, n_pages).flatten().long()
    refs += torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda").index_add_(0, taken, torch.ones_like(taken, dtype=torch.int32))[:n_pages]
    left = torch.where(copies, last, n_pages)
    refs -= torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda").index_add_(0, left, torch.ones_like(add))[:n_pages]
    lens += torch.where(done, add, 0)
    a = last[copies]
    pool[:, table.gather(1, (old - 1).clamp(min=0).long().unsqueeze(1)).squeeze(1)[copies].long()] = pool[:, a]


def _plain_compact(s):
    table, lens, refs, pool, ended = s["table"], s["lens"], s["refs"], s["pool"], s["ended"].long()
    n_pages = refs.numel()
    hot = table[ended].flatten().long()
    refs -= torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda").index_add_(
        0, torch.where(hot < 0, n_pages, hot), torch.ones_like(hot, dtype=torch.int32))[:n_pages]
    table[ended], lens[ended] = -1, 0
    live = refs > 0
    page = torch.arange(n_pages, device="cuda")
    front = page < live.sum()
    holes, moved = (front & ~live).nonzero().squeeze(1), (~front & live).nonzero().squeeze(1)
    pool[:, holes] = pool[:, moved]
    page[moved] = holes
    refs[holes] = refs[moved]
    refs[moved] = 0
    table.copy_(torch.where(table >= 0, page[table.clamp(min=0).long()].to(torch.int32), table))


def run(s):
    case = s["case"]
    op = case["op"]
    if op in ("pages", "compact"):
        for t, saved in zip((s["table"], s["lens"], s["refs"]), s["before"]):
            t.copy_(saved)
        if own and op == "pages":
            s["cache"].fork(s["src"])
            s["cache"].extend(s["add"])
        elif own:
            s["cache"].free(s["ended"])
            s["cache"].compact()
        elif op == "pages":
            _plain_fork(s)
            _plain_extend(s)
        else:
            _plain_compact(s)
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "pool": s["pool"]}
    if own:
        from velox_amd import paged
        if op == "rope":
            return paged.rope(s["rope"], s["x"], s["positions"])
        if op == "append":
            paged.rope_append(s["cache"], 0, s["rope"], s["q"], s["k"], s["v"], s["out"], q_start=s["start"])
            return s["out"], s["pool"]
        if op == "token":
            return paged.attention(s["cache"], 0, s["q"], window=case["window"], sinks=case["sinks"], max_len=s["last"],
                                   workspace=s["space"])
        return paged.prompt_attention(s["cache"], 0, s["q"], s["start"], max_rows=s["most"], window=case["window"],
                                      sinks=case["sinks"], max_len=s["last"], workspace=s["space"])
    if op == "rope":
        return _plain_turn(s["x"], s["positions"], s).to(s["x"].dtype)
    if op == "append":
        return _plain_append(s)
    if op == "token":
        return _plain_attention(s, s["q"].unsqueeze(1)).squeeze(1).to(s["q"].dtype)
    n, most = s["lens"].numel(), s["most"]
    counts = s["start"][1:] - s["start"][:-1]
    row = torch.arange(most, device="cuda").unsqueeze(0) - (most - counts).unsqueeze(1)  # padded in front
    flat = (s["start"][:-1].unsqueeze(1) + row).clamp(min=0).long()
    o = _plain_attention(s, s["q"][flat])
    seq = torch.searchsorted(s["start"], torch.arange(s["rows"], device="cuda", dtype=torch.int32), right=True) - 1
    inside = torch.arange(s["rows"], device="cuda") - s["start"][seq] + (most - counts)[seq]
    return o[seq, inside.long()].to(s["q"].dtype)


# ---- the same in 64 bits --------------------------------------------------------------------------

def _exact_turn(x, positions, case):
    freq, amp = _frequencies(case)
    out = x.double().clone()
    half = case["rot"] // 2
    for j in range(half):
        i, k = (j, j + half) if case["layout"] == "half" else (2 * j, 2 * j + 1)
        z = torch.complex(x[:, :, i].double(), x[:, :, k].double())
        z = z * torch.polar(torch.full_like(positions, amp, dtype=torch.float64), positions.double() * freq[j]).unsqueeze(1)
        out[:, :, i], out[:, :, k] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d = HEADS[case["model"]]
    page = case.get("page")
    if case["op"] == "rope":
        return _exact_turn(s["x"], s["positions"], case)
    if case["op"] in ("pages", "compact"):
        return None  # numbers are moved here, not computed
    rows, lens = _lengths(case)
    table = s["table"].tolist()
    start = s["start"].tolist()
    if case["op"] == "append":
        out, pool = s["out"].double(), s["pool"].double()
        for b, n in enumerate(lens):
            lo, hi = start[b], start[b + 1]
            at = torch.arange(n - rows[b], n, device="cuda")
            out[lo:hi] = _exact_turn(s["q"][lo:hi], at, case)
            k, v = _exact_turn(s["k"][lo:hi], at, case), s["v"][lo:hi].double()
            for p, number in enumerate(table[b]):
                here = (at // page == p).nonzero().flatten()
                if here.numel():
                    r = at[here] % page
                    kk = pool[0, number][:hkv * page * d].view(hkv, page, d)
                    kk[:, r] = k[here].transpose(0, 1)
                    vv = pool[0, number][hkv * page * d:].view(hkv, page // 32, d, 32)
                    for h in range(hkv):
                        vv[h, r // 32, :, torch.tensor(SLOT, device="cuda")[r % 32]] = v[here, h]
        return out, pool
    result = torch.zeros(s["rows"], hq, d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        mine = [p for p in table[b] if p >= 0]
        cells = s["pool"][0][torch.tensor(mine, device="cuda")]
        k = cells[:, :hkv * page * d].reshape(-1, hkv, page, d)
        v = cells[:, hkv * page * d:].reshape(-1, hkv, page // 32, d, 32)
        lo, hi = start[b], start[b + 1]
        t = torch.arange(n - rows[b], n, device="cuda").unsqueeze(1)
        j = torch.arange(n, device="cuda").unsqueeze(0)
        seen = j <= t
        if case["window"]:
            seen = seen & ((t - j < case["window"]) | (j < case["sinks"]))
        for h in range(hq):
            g = h * hkv // hq
            kh = k[:, g].reshape(-1, d)[:n].double()
            vh = v[:, g].transpose(2, 3)[:, :, torch.tensor(SLOT, device="cuda")].reshape(-1, d)[:n].double()
            x = (s["q"][lo:hi, h].double() @ kh.T) / math.sqrt(d)
            x = x.masked_fill(~seen, float("-inf"))
            result[lo:hi, h] = torch.softmax(x, 1) @ vh
    return result
