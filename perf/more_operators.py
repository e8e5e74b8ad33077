"""Performance cases of the 8-bit integer products and the experts: products with a scale for each token and channel,
the choice of experts, the grouping of rows by expert, and the experts' feed-forward products.

listed() are the cases, draw() gives more of the same ranges. With `own` false run() computes a case with
elementary torch operations on plain row-major weights; with `own` true it makes the calls of velox_amd.int8 and
velox_amd.experts. exact() recomputes the numbers in float64.

A row x is held as s * c with s = fl32(max |x| / 127) and whole numbers c = x / s to nearest (ties to even); a weight
row likewise, by its own scale. A product is (c . w) * scale of the weight row * scale of the row. An expert's answer is
down(silu(gate(x)) * up(x)), the inner row held in 8 bits too; a row's answer is the sum of its experts' by weight.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------------

def listed():
    return [
        # one token's output projection with the residual stream: fp32 activations, launch latency
        {"name": "product_llama8b_o_row1", "op": "product", "rows": 1, "n": 4096, "k": 4096, "type": "f32", "paired": False,
         "bias": False, "residual": True},
        # a decode step of 32 sequences: gate and up with SwiGLU, the weights' bytes count
        {"name": "product_qwen7b_gate_up_rows32", "op": "product", "rows": 32, "n": 2 * 18944, "k": 3584, "type": "f32", "paired": True,
         "bias": False, "residual": False},
        # a short prompt of the smallest model: odd rows, q, k and v with biases
        {"name": "product_smollm_qkv_prompt", "op": "product", "rows": 1037, "n": 960, "k": 576, "type": "f16", "paired": False,
         "bias": True, "residual": False},
        # a long prompt through the largest matrix: the matrix cores' rate
        {"name": "product_72b_down_prompt8192", "op": "product", "rows": 8192, "n": 8192, "k": 29568, "type": "bf16", "paired": False,
         "bias": False, "residual": False},
        # one token among 256 experts in 8 groups, sigmoid scores with a bias for balance: latency
        {"name": "route_256_row1", "op": "route", "rows": 1, "experts": 256, "top": 8, "scores": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "by": "two", "renormalize": True, "scale": 2.5, "type": "f32", "masked": 0.0},
        # the same for a long prompt
        {"name": "route_256_prompt16384", "op": "route", "rows": 16384, "experts": 256, "top": 8, "scores": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "by": "two", "renormalize": True, "scale": 2.5, "type": "f32", "masked": 0.0},
        # softmax scores of 16-bit logits (many of them equal), some experts masked, rows of padding wholly
        {"name": "route_60_masked", "op": "route", "rows": 4001, "experts": 60, "top": 6, "scores": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "by": "max", "renormalize": False, "scale": 1.0, "type": "f16", "masked": 0.1},
        # one token of a small mixture: six of 64 experts, latency
        {"name": "ffn_64_row1", "op": "ffn", "rows": 1, "experts": 64, "total": 64, "first": 0, "top": 6, "hidden": 2048, "inter": 1408,
         "type": "bf16", "pad": 0},
        # a decode batch of 32 rows on a rank that holds 64 of 256 experts: the bytes of the experts that were chosen
        {"name": "ffn_64of256_rows32", "op": "ffn", "rows": 32, "experts": 64, "total": 256, "first": 64, "top": 8, "hidden": 7168,
         "inter": 2048, "type": "bf16", "pad": 0},
        # few small experts, odd rows, a padded batch
        {"name": "ffn_5_odd_padded", "op": "ffn", "rows": 257, "experts": 5, "total": 5, "first": 0, "top": 2, "hidden": 576, "inter": 1100,
         "type": "f16", "pad": 31},
        # a prompt through eight large experts, two for each row
        {"name": "ffn_8_prompt1000", "op": "ffn", "rows": 1000, "experts": 8, "total": 8, "first": 0, "top": 2, "hidden": 4096,
         "inter": 14336, "type": "f16", "pad": 0},
        # a long prompt on a rank that holds 64 of 256 experts, unequal numbers of rows for each
        {"name": "ffn_64of256_prompt4096", "op": "ffn", "rows": 4096, "experts": 64, "total": 256, "first": 128, "top": 8, "hidden": 7168,
         "inter": 2048, "type": "bf16", "pad": 0},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("product", "product", "route", "ffn", "ffn"))
    if op == "product":
        rows, k = _log(rng, 1, 8192), _log(rng, 32, 30000)
        n = _log(rng, 16, min(40000, int(1.9e12) // (rows * k)))
        paired = rng.random() < 0.3
        return {"op": op, "rows": rows, "n": n // 2 * 2 if paired else n, "k": k, "type": rng.choice(tuple(TYPES)), "paired": paired,
                "bias": not paired and rng.random() < 0.5, "residual": not paired and rng.random() < 0.5}
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * _log(rng, 2, 512 // groups)
        top_groups = rng.randint(1, groups)
        sigmoid = rng.random() < 0.5
        return {"op": op, "rows": _log(rng, 1, 16384), "experts": experts, "top": rng.randint(1, min(16, experts // groups * top_groups)),
                "scores": "sigmoid" if sigmoid else "softmax", "bias": sigmoid and rng.random() < 0.7, "groups": groups,
                "top_groups": top_groups, "by": rng.choice(("max", "two")), "renormalize": rng.random() < 0.6,
                "scale": rng.choice((1.0, 2.5, 16.0)), "type": rng.choice(tuple(TYPES)), "masked": rng.choice((0.0, 0.0, 0.1))}
    experts = _log(rng, 1, 64)
    total = experts * rng.choice((1, 1, 4))
    hidden = _log(rng, 64, 7168)
    inter = _log(rng, 32, min(14336, 2900 * 1000 * 1000 // (3 * hidden * experts)))
    top = rng.randint(1, min(8, total))
    rows = _log(rng, 1, max(1, min(4096, int(3.2e11) // (hidden * inter * top))))
    return {"op": op, "rows": rows, "experts": experts, "total": total, "first": rng.randint(0, total - experts), "top": top,
            "hidden": hidden, "inter": inter, "type": rng.choice(("f16", "bf16")), "pad": rng.choice((0, 0, 3))}


# ---- what a case's numbers say --------------------------------------------------------------------

def _choices(case):
    """Which experts the rows of an "ffn" case go to, the same for every seed but for the experts' numbers: some are
    in demand, others hardly; the last `pad` rows are padding (-1)."""
    g = torch.Generator().manual_seed(11)
    liked = torch.randn(case["total"], generator=g) * 0.7
    ids = (torch.randn(case["rows"], case["total"], generator=g) + liked).topk(case["top"], 1).indices
    if case["pad"]:
        ids[max(0, case["rows"] - case["pad"]):] = -1
    return ids


def work(case):
    if case["op"] == "product":
        m, n, k, e = case["rows"], case["n"], case["k"], SIZE[case["type"]]
        cols = n // 2 if case["paired"] else n
        return {"bytes": n * k + 4 * n * (2 if case["bias"] else 1) + m * e * (k + cols * (2 if case["residual"] else 1)), "flops": 2 * m * n * k}
    if case["op"] == "route":
        m, e = case["rows"], case["experts"]
        return {"bytes": m * e * SIZE[case["type"]] + 12 * m * case["top"] + 4 * e, "flops": 8 * m * e}
    ids = _choices(case)
    here = ids[(ids >= case["first"]) & (ids < case["first"] + case["experts"])]
    h, f = case["hidden"], case["inter"]
    return {"bytes": here.unique().numel() * (3 * h * f + 4 * (2 * f + h)) + case["rows"] * (2 * h * SIZE[case["type"]] + 8 * case["top"]),
            "flops": 6 * here.numel() * h * f}


# ---- inputs ---------------------------------------------------------------------------------------

def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + tag) % (1 << 61))


def _activations(rows, k, g, dtype):
    """Rows of unequal size with a few channels far above the others, as hidden states have."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= 1.0 + 8.0 * (torch.rand(k, generator=g, device="cuda") < 0.004)
    return (x * (0.25 + 2 * torch.rand(rows, 1, generator=g, device="cuda"))).to(dtype)


def _weights(shape, g):
    """Whole numbers and scales of matrices [...][n][k], made in slices."""
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = codes.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        n = min(1 << 28, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=g, device="cuda", dtype=torch.float16 if n > 1 << 20 else torch.float32) * 31).round_().clamp_(-127, 127)
    scales = (0.5 + torch.rand(shape[:-1], generator=g, device="cuda")) / (31 * math.sqrt(shape[-1]))
    return codes, scales


def prepare(case, seed):
    s = {"case": case}
    if case["op"] == "product":
        t = TYPES[case["type"]]
        cols = case["n"] // 2 if case["paired"] else case["n"]
        s["x"] = _activations(case["rows"], case["k"], _gen(seed, 1), t)
        s["w"], s["sw"] = _weights((case["n"], case["k"]), _gen(seed, 2))
        s["bias"] = torch.randn(case["n"], generator=_gen(seed, 3), device="cuda") if case["bias"] else None
        s["residual"] = torch.randn(case["rows"], cols, generator=_gen(seed, 4), device="cuda").to(t) if case["residual"] else None
        if own:
            from velox_amd import int8
            s["matrix"] = int8.Int8Matrix(s["w"], s["sw"], paired=case["paired"])
            s["space"] = int8.product_workspace(s["matrix"], case["rows"])
        return s
    if case["op"] == "route":
        m, e = case["rows"], case["experts"]
        x = torch.randn(m, e, generator=_gen(seed, 1), device="cuda") * 1.5 + torch.randn(e, generator=_gen(seed, 2), device="cuda") * 0.5
        if case["masked"]:
            x[torch.rand(m, e, generator=_gen(seed, 3), device="cuda") < case["masked"]] = -math.inf
            x[m - m // 50:] = -math.inf
        s["logits"] = x.to(TYPES[case["type"]])
        s["bias"] = torch.randn(e, generator=_gen(seed, 4), device="cuda") * 0.1 if case["bias"] else None
        if own:
            from velox_amd import experts
            s["space"] = experts.group_workspace(m * case["top"], e)
        return s
    first, count, total = case["first"], case["experts"], case["total"]
    inside = first + torch.randperm(count, generator=_gen(seed, 5), device="cuda")
    away = torch.cat((torch.arange(first, device="cuda"), torch.arange(first + count, total, device="cuda")))
    names = torch.cat((away[:first], inside, away[first:], torch.full((1,), -1, device="cuda")))
    s["ids"] = names[_choices(case).cuda()].to(torch.int32)
    s["share"] = torch.softmax(torch.randn(case["rows"], case["top"], generator=_gen(seed, 6), device="cuda"), 1)
    s["x"] = _activations(case["rows"], case["hidden"], _gen(seed, 1), TYPES[case["type"]])
    s["up"], s["sup"] = _weights((count, 2 * case["inter"], case["hidden"]), _gen(seed, 2))
    s["down"], s["sdown"] = _weights((count, case["hidden"], case["inter"]), _gen(seed, 3))
    # the most rows of an expert: what the plain form pads to
    seen = _choices(case)
    seen = seen[(seen >= first) & (seen < first + count)] - first
    s["most"] = max(1, int(torch.bincount(seen, minlength=count).max()))
    if own:
        from velox_amd import experts, int8
        s["gate_up"] = int8.Int8Matrix(s["up"], s["sup"], paired=True)
        s["out_matrix"] = int8.Int8Matrix(s["down"], s["sdown"])
        s["space"] = experts.ffn_workspace(s["gate_up"], s["out_matrix"], case["rows"], case["top"])
    return s


# ---- one pass -------------------------------------------------------------------------------------

def _held(x):
    """Rows in whole numbers (as fp32) and their scales."""
    scale = (x.abs().amax(-1, keepdim=True).double() / 127).float()  # rounded once
    codes = torch.where(scale > 0, x.double() / scale.double(), 0.0).round_()  # to the nearest of exact quotients
    return codes.float(), scale


def _silu_product(g, u):
    return g / (1 + torch.exp(-g)) * u


def _plain_product(s):
    x = s["x"].float()
    c, scale = _held(x)
    y = torch.matmul(c, s["w"].float().t()).mul_(s["sw"]).mul_(scale)
    if s["bias"] is not None:
        y += s["bias"]
    if s["case"]["paired"]:
        half = y.shape[1] // 2
        y = _silu_product(y[:, :half], y[:, half:])
    if s["residual"] is not None:
        y += s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_route(s):
    case = s["case"]
    m, e, groups, top = case["rows"], case["experts"], case["groups"], case["top"]
    x = s["logits"].double()  # in 64 bits: which of two nearly equal scores is larger
    there = x > -math.inf
    x = torch.where(there, x, -math.inf)
    if case["scores"] == "softmax":
        p = torch.exp(x - torch.where(there.any(1, keepdim=True), x.amax(1, keepdim=True), 0.0))
        score = p / p.sum(1, keepdim=True).clamp(min=1.0)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score + s["bias"].double() if s["bias"] is not None else score
    choice = torch.where(there, choice, -math.inf)
    if groups > 1:
        best = choice.view(m, groups, -1).sort(dim=2, descending=True).values
        mark = best[:, :, 0]
        if case["by"] == "two" and best.shape[2] > 1:
            mark = mark + torch.where(best[:, :, 1] > -math.inf, best[:, :, 1], 0.0)
        kept = mark.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_ = torch.zeros(m, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        choice = torch.where(open_.repeat_interleave(e // groups, 1), choice, -math.inf)
    value, ids = choice.sort(dim=1, descending=True, stable=True)
    value, ids = value[:, :top], ids[:, :top]
    weights = torch.where(value > -math.inf, score.gather(1, ids), 0.0)
    if case["renormalize"]:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
    ids = torch.where(value > -math.inf, ids, -1).to(torch.int32)
    return ids, (weights * case["scale"]).float()


def _plain_group(ids, count, first):
    """The slots of `ids` in the order of their experts, -1 behind them, and where each expert's begin."""
    e = ids.flatten().long() - first
    e = torch.where((e >= 0) & (e < count), e, count)
    order = torch.argsort(e, stable=True)
    where = torch.searchsorted(e[order], torch.arange(count + 1, device="cuda")).to(torch.int32)
    return torch.where(e[order] < count, order, -1).to(torch.int32), where


def _plain_ffn(s):
    """Every expert's rows padded to the most that one has; where there are fewer slots than experts, a matrix for
    each slot."""
    case = s["case"]
    count, most, top, f = case["experts"], s["most"], case["top"], case["inter"]
    slots = case["rows"] * top
    matrices = [s[name] for name in ("up", "sup", "down", "sdown")]
    if slots < count:
        expert = s["ids"].flatten().long() - case["first"]
        filled = ((expert >= 0) & (expert < count)).unsqueeze(1)
        matrices = [t[expert.clamp(0, count - 1)] for t in matrices]
        count, most = slots, 1
        slot = torch.arange(slots, device="cuda").unsqueeze(1)
    else:
        order, begin = _plain_group(s["ids"], count, case["first"])
        begin = begin.long()
        place = begin[:-1].unsqueeze(1) + torch.arange(most, device="cuda")
        filled = place < begin[1:].unsqueeze(1)
        slot = torch.where(filled, order[place.clamp(max=slots - 1)].long(), 0)
    up, sup, down, sdown = matrices
    c, scale = _held(s["x"].float())
    row = slot // top
    gu = torch.bmm(up.float(), c[row].transpose(1, 2).contiguous())
    gu.mul_(sup.unsqueeze(2)).mul_(scale[row].view(count, 1, most))
    h, hscale = _held(_silu_product(gu[:, :f], gu[:, f:]).transpose(1, 2))
    del gu
    y = torch.bmm(down.float(), h.transpose(1, 2).contiguous())
    y.mul_(sdown.unsqueeze(2)).mul_(hscale.view(count, 1, most))
    y.mul_(torch.where(filled, s["share"].flatten()[slot], 0.0).unsqueeze(1))
    # the answers back to their slots, then summed over a row's experts
    back = torch.zeros(slots + 1, case["hidden"], device="cuda")
    back[torch.where(filled, slot, slots).flatten()] = y.transpose(1, 2).reshape(count * most, -1)
    back[slots] = 0
    return back[:-1].view(case["rows"], top, -1).sum(1).to(s["x"].dtype)


def run(s):
    case = s["case"]
    if own:
        from velox_amd import experts, int8
        if case["op"] == "product":
            return int8.product(s["x"], s["matrix"], bias=s["bias"], residual=s["residual"], workspace=s["space"])
        if case["op"] == "route":
            ids, weights = experts.route(s["logits"], case["top"], scores=case["scores"], bias=s["bias"], groups=case["groups"],
                                         top_groups=case["top_groups"], group_by=case["by"], renormalize=case["renormalize"],
                                         scale=case["scale"])
            return ids, weights, *experts.group(ids, case["experts"], workspace=s["space"])
        return experts.ffn(s["x"], s["ids"], s["share"], s["gate_up"], s["out_matrix"], first=case["first"], workspace=s["space"])
    if case["op"] == "product":
        return _plain_product(s)
    if case["op"] == "route":
        ids, weights = _plain_route(s)
        return ids, weights, *_plain_group(ids, case["experts"], 0)
    return _plain_ffn(s)


# ---- the same in 64 bits --------------------------------------------------------------------------

def _exact_rows(x):
    """(whole numbers, scale) of every row, in float64; the scale is a 32-bit number by definition."""
    top = x.float().abs().max(dim=1).values
    scale = (top.double() / 127.0).float().double()
    return torch.where(scale.unsqueeze(1) == 0, 0.0, torch.round(x.double() / scale.unsqueeze(1))), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        c, scale = _exact_rows(s["x"])
        parts = []
        for at in range(0, case["n"], 4096):  # in strips of the weights
            w = s["w"][at:at + 4096].double() * s["sw"][at:at + 4096].double().unsqueeze(1)
            parts.append((w @ c.T).T * scale.unsqueeze(1))
        y = torch.cat(parts, 1)
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if case["paired"]:
            gate, up = y.chunk(2, 1)
            y = gate * torch.sigmoid(gate) * up
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "route":
        x = s["logits"].double()
        score = torch.nan_to_num(torch.softmax(x, 1)) if case["scores"] == "softmax" else torch.sigmoid(x)
        pick = score if s["bias"] is None else score + s["bias"].double()
        pick = pick.masked_fill(x == -math.inf, -math.inf)
        e, groups = case["experts"], case["groups"]
        if groups > 1:
            a = pick.unflatten(1, (groups, e // groups))
            mark = a.amax(2)
            if case["by"] == "two" and e > groups:
                second = a.topk(2, 2).values[:, :, 1]
                mark = mark + second.masked_fill(second == -math.inf, 0.0)
            shut = torch.ones_like(mark, dtype=torch.bool)
            for _ in range(case["top_groups"]):  # one group after the other, the first of equal ones
                at = mark.argmax(1, keepdim=True)
                shut.scatter_(1, at, False)
                mark = mark.scatter(1, at, -math.inf)
            pick = pick.unflatten(1, (groups, e // groups)).masked_fill(shut.unsqueeze(2), -math.inf).flatten(1)
        chosen = []
        for _ in range(case["top"]):
            value, at = pick.max(1, keepdim=True)
            chosen.append(score.gather(1, at).masked_fill(value == -math.inf, 0.0))
            pick = pick.scatter(1, at, -math.inf)
        w = torch.cat(chosen, 1)
        if case["renormalize"]:
            w = torch.nan_to_num(w / w.sum(1, keepdim=True))
        return None, w * case["scale"], None, None
    c, scale = _exact_rows(s["x"])
    out = torch.zeros(case["rows"], case["hidden"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        row, j = (s["ids"] == case["first"] + e).nonzero(as_tuple=True)
        if row.numel():
            gate, up = ((s["up"][e].double() * s["sup"][e].double().unsqueeze(1)) @ c[row].T * scale[row]).T.chunk(2, 1)
            inner = gate * torch.sigmoid(gate) * up
            step = inner.abs().amax(1, keepdim=True) / 127
            inner = torch.where(step > 0, torch.round(inner / step), 0.0) * step
            y = ((s["down"][e].double() * s["sdown"][e].double().unsqueeze(1)) @ inner.T).T
            out.index_add_(0, row, y * s["share"][row, j].double().unsqueeze(1))
    return out
