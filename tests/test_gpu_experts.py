"""The choice of experts, the grouping and the experts' products on the GPU against float64.

Choices and orders have to be equal; routing weights are off by the rounding to fp32 and by what 64-bit scores leave (1e-13).
The experts' products: u = 2^-24. A hidden value h = silu(g) up is off by at most e_h = |h| 11 u + |up| |g| 3.3 u (three
roundings each of g and up, silu's slope below 1.1, the exponential, a sum, a quotient, a product), its row's scale by what
the largest value is off and 2 u. So a code can be another one only where its exact quotient lies within that of a half:
each such place may move the product by one step of the code, |w| scale. A product then is off by 3 u, its weighted sum over
the row's experts in fp32 by (top + 1) u of the sum of sizes, and the output by half a step of its type.
"""
import math

import numpy as np
import pytest
import torch

from velox_amd import experts, int8
from velox_amd.engine import MlaEngine

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- routing ----

def route_by_rule(x, top, scores="softmax", bias=None, groups=1, top_groups=1, group_by="max", renormalize=False, scale=1.0):
    """(ids, weights) of one row of numbers, by the rule's words."""
    n, scale = len(x), float(np.float32(scale))  # (the C ABI's scale is fp32)
    big = float(np.finfo(np.float32).max)
    x = [min(v, big) if v == v else -math.inf for v in map(float, x)]
    if scores == "softmax":
        most = max(x)
        p = [math.exp(v - most) if v > -math.inf else 0.0 for v in x]
        total = math.fsum(p)
        score = [v / total if total else 0.0 for v in p]
    else:
        score = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in x]
    if scores == "softmax" and bias is None and group_by == "max":
        choice = list(x)
    else:
        choice = [s if v > -math.inf else -math.inf for s, v in zip(score, x)]
    if bias is not None:
        choice = [c + float(b) if c > -math.inf and math.isfinite(b) else -math.inf for c, b in zip(choice, bias)]
    size = n // groups
    if groups > 1:
        marks = []
        for g in range(groups):
            best = sorted(choice[g * size:(g + 1) * size], reverse=True)
            marks.append(best[0] + best[1] if group_by == "two" and size > 1 and best[1] > -math.inf else best[0])
        kept = sorted(range(groups), key=lambda g: (-marks[g], g))[:top_groups]
        choice = [c if e // size in kept else -math.inf for e, c in enumerate(choice)]
    order = sorted((e for e in range(n) if choice[e] > -math.inf), key=lambda e: (-choice[e], e))[:top]
    w = [score[e] for e in order]
    if renormalize:
        total = math.fsum(w)
        w = [v / total if total else 0.0 for v in w]
    return order + [-1] * (top - len(order)), [v * scale for v in w] + [0.0] * (top - len(order))


def check_route(x, top, **kw):
    b = kw.get("bias")
    ids, w = experts.route(x, top, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (x.shape[0], top)
    rule = dict(kw, bias=b.tolist() if b is not None else None)
    for r, row in enumerate(x.double().tolist()):
        want, share = route_by_rule(row, top, **rule)
        assert ids[r].tolist() == want, (r, ids[r].tolist(), want)
        for a, v in zip(w[r].tolist(), share):
            assert abs(a - v) <= U * abs(v) + 1e-13 * abs(v) + 2.0 ** -149, (r, a, v)


@pytest.mark.parametrize("n,experts_,top,groups,top_groups", [(1, 1, 1, 1, 1), (3, 2, 2, 1, 1), (5, 63, 7, 1, 1), (70, 64, 8, 8, 3), (33, 65, 6, 1, 1), (9, 256, 8, 8, 4),
                                                              (41, 160, 6, 8, 3), (7, 512, 10, 1, 1), (6, 1024, 64, 64, 5), (4, 1000, 33, 4, 1), (12, 60, 6, 60, 9),
                                                              (130, 8, 2, 1, 1), (5, 257, 3, 1, 1), (3, 320, 9, 10, 10)])
@pytest.mark.parametrize("scores,biased,by", [("softmax", False, "max"), ("softmax", True, "max"), ("softmax", False, "two"), ("sigmoid", True, "two"),
                                              ("sigmoid", False, "max")])
def test_route(n, experts_, top, groups, top_groups, scores, biased, by):
    for i, dtype in enumerate(T):
        x = (torch.randn(n, experts_, generator=gen(n + i), device="cuda") * 2).to(T[dtype])
        bias = torch.randn(experts_, generator=gen(5), device="cuda") * 0.2 if biased else None
        check_route(x, top, scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_by=by, renormalize=i % 2 == 0, scale=(1.0, 2.5, 0.3)[i])


def test_route_equal_scores_go_by_index():
    x = torch.zeros(5, 64, device="cuda")
    x[1, 40:] = 1.0
    x[2, ::3] = 2.0
    x[3] = torch.arange(64, device="cuda") // 9
    x[4] = -torch.arange(64, device="cuda") // 9
    for kw in (dict(), dict(scores="sigmoid"), dict(groups=8, top_groups=3), dict(groups=8, top_groups=3, group_by="two"),
               dict(bias=torch.full((64,), 0.25, device="cuda"))):
        check_route(x, 9, **kw)


def test_route_masks_and_what_is_no_number():
    inf, nan = math.inf, math.nan
    low = torch.finfo(torch.float32).min
    x = torch.randn(12, 16, generator=gen(3), device="cuda")
    x[0] = -inf
    x[1, 3:] = -inf
    x[2] = nan
    x[3, :14] = nan
    x[4] = low
    x[5, 4:] = low
    x[6, 2], x[6, 9] = inf, inf
    x[7] = inf
    x[8, ::2], x[8, 1] = -inf, nan
    x[9, 8:] = -inf
    x[10, :9] = -inf
    x[11, 5] = 1000.0
    bias = torch.zeros(16, device="cuda")
    odd = torch.tensor([0.1, -inf, nan, inf] + [0.0] * 12, device="cuda")
    for kw in (dict(), dict(renormalize=True), dict(scores="sigmoid"), dict(scores="sigmoid", renormalize=True), dict(groups=4, top_groups=2),
               dict(groups=4, top_groups=2, group_by="two", scores="sigmoid"), dict(bias=bias), dict(bias=odd), dict(bias=odd, scores="sigmoid", groups=2)):
        check_route(x, 4, **kw)
    x16 = x.clamp(min=-6e4).half()
    check_route(x16, 4, renormalize=True)
    ids, w = experts.route(x, 4)
    assert (ids[0] == -1).all() and (w[0] == 0).all() and ids[1].tolist()[3] == -1


def test_route_scores_next_to_each_other():
    """Scores that fp32 cannot tell apart keep the order that their logits and biases give."""
    step = 2.0 ** -20
    x = torch.zeros(3, 128, device="cuda")
    x[0] = 12 + torch.arange(128, device="cuda") * step      # sigmoid: 1 - 6e-6 (1 - ...): far below an fp32 step apart
    x[1] = 12 - torch.arange(128, device="cuda") * step
    x[2] = torch.randn(128, generator=gen(1), device="cuda") * step + 9
    check_route(x, 16, scores="sigmoid")
    check_route(x, 16, scores="sigmoid", bias=torch.full((128,), 0.125, device="cuda"), renormalize=True)
    check_route(x, 16)
    check_route(x, 16, bias=torch.full((128,), 0.125, device="cuda"))


@pytest.mark.parametrize("n", [64, 200, 256, 1024])
def test_route_a_few_or_many_too_near_to_tell(n):
    """Logits with clusters of 2 to 100 neighbours that differ by less than fp32 scores show, some of them equal; groups
    whose marks do as well."""
    g = gen(n)
    x = torch.randn(40, n, generator=g, device="cuda")
    for r in range(40):
        size = (2, 3, 10, 63, 64, 65, 100, n)[r % 8]
        at = torch.randperm(n, generator=g, device="cuda")[:size]
        x[r, at] = 3.0 + (r % 5) * 0.5 + torch.randint(0, 8, (len(at),), generator=g, device="cuda") * 2.0 ** -21
    bias = torch.zeros(n, device="cuda")
    some = torch.randint(0, 2, (n,), generator=g, device="cuda") * 0.25
    for kw in (dict(bias=bias, scores="sigmoid"), dict(bias=some, scores="sigmoid", renormalize=True), dict(bias=bias), dict(bias=some, renormalize=True),
               dict(bias=bias, scores="sigmoid", groups=4, top_groups=2, group_by="two"), dict(groups=4, top_groups=2, group_by="two"),
               dict(bias=some, groups=8, top_groups=3)):
        for top in (1, 8) if "groups" in kw else (1, 8, 64):
            check_route(x, top, **kw)


def test_route_groups_whose_marks_cancel():
    """Marks of two values far larger than their sum are off by more than the marks beside them are apart: a group in the
    middle of the order, or one that is out, may be the one that is wrong."""
    score = torch.tensor([0.6, 0.2, 0.5, 0.4, 0.45, 0.4, 0.1, 0.1], dtype=torch.float64)  # marks 0.8, 0.9, 0.85, 0.2
    x = torch.log(score / (1 - score)).float().cuda().unsqueeze(0)
    bias = torch.zeros(8, device="cuda")
    bias[0], bias[1] = 1e7, -1e7
    kw = dict(scores="sigmoid", bias=bias, groups=4, group_by="two")
    check_route(x, 4, top_groups=2, **kw)
    assert sorted(experts.route(x, 4, top_groups=2, **kw)[0][0].tolist()) == [2, 3, 4, 5]
    for n, groups in ((8, 4), (64, 8), (256, 8), (60, 20), (512, 64), (1024, 16)):
        size = n // groups
        x = torch.randn(24, n, generator=gen(n), device="cuda")
        x[5, :size], x[6, 2 * size:] = -math.inf, -math.inf  # groups without an expert
        for large in (3e4, 1e5, 1e7, 1e12):
            bias = torch.randn(n, generator=gen(n + 1), device="cuda") * 0.05
            for g in range(0, groups, 3):
                bias[g * size], bias[g * size + 1] = large, -large
                bias[g * size + 2:(g + 1) * size] = -2 * large  # (the two are the group's mark)
            for scores in ("sigmoid", "softmax"):
                for top_groups in {1, 2, groups // 2, groups - 1}:
                    check_route(x, min(4, size * top_groups), scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_by="two")


def test_route_marks_past_fp32():
    """Two biases next to the largest number: their sum is a number in 64 bits, and above that of a group without an expert."""
    most = torch.finfo(torch.float32).max
    x = torch.randn(20, 24, generator=gen(7), device="cuda")
    x[4, :4] = -math.inf
    x[5, 4:8] = -math.inf
    x[6, 4:] = -math.inf
    x[7, :20] = -math.inf
    x[8] = -math.inf
    for signs in ((-1, -1), (1, 1), (1, -1)):
        for at in (0, 1, 5):  # the group
            bias = torch.zeros(24, device="cuda")
            bias[4 * at:4 * at + 4] = -most
            bias[4 * at], bias[4 * at + 1] = signs[0] * most, signs[1] * most
            both = bias.clone()
            both[8:12] = -most
            for b in (bias, both, torch.full_like(bias, -most), torch.full_like(bias, most)):
                for scores in ("sigmoid", "softmax"):
                    for top_groups in (1, 2, 5, 6):
                        check_route(x, 4, scores=scores, bias=b, groups=6, top_groups=top_groups, group_by="two")
                        check_route(x, 4, scores=scores, bias=b, groups=6, top_groups=top_groups)


def test_route_strided_rows_and_given_outputs():
    wide = torch.randn(20, 100, generator=gen(2), device="cuda").bfloat16()
    x = wide[:, 13:77]
    check_route(x, 5, renormalize=True)
    ids, w = torch.full((20, 5), 77, dtype=torch.int32, device="cuda"), torch.zeros(20, 5, device="cuda")
    a, b = experts.route(x, 5, ids=ids, weights=w)
    assert a is ids and b is w and (ids != 77).all()
    none = experts.route(x[:0], 5)
    assert none[0].shape == (0, 5)


# ---- grouping ----

def check_group(ids, count, first=0):
    order, offsets = experts.group(ids, count, first)
    e = ids.flatten().cpu().numpy().astype(np.int64) - first
    e = np.where((e >= 0) & (e < count), e, count)
    want = np.argsort(e, kind="stable")
    want = np.where(e[want] < count, want, -1)
    assert np.array_equal(order.cpu().numpy(), want)
    assert np.array_equal(offsets.cpu().numpy(), np.searchsorted(np.sort(e), np.arange(count + 1)))


@pytest.mark.parametrize("rows,top,total,first,count", [(0, 1, 4, 0, 4), (1, 1, 1, 0, 1), (1, 8, 256, 0, 256), (3, 2, 5, 1, 3), (63, 1, 64, 0, 64), (65, 6, 64, 0, 64),
                                                        (341, 6, 100, 40, 60), (1024, 2, 8, 0, 8), (1025, 2, 1024, 0, 1024), (4001, 8, 256, 64, 64),
                                                        (16384, 8, 256, 0, 256), (5000, 1, 2, 0, 1), (131072, 8, 1000, 3, 900)])
def test_group(rows, top, total, first, count):
    ids = torch.randint(-1, total, (rows, top), generator=gen(rows + total), device="cuda", dtype=torch.int32)
    check_group(ids, count, first)
    if rows:
        check_group(torch.full_like(ids, first), count, first)       # one expert has all
        check_group(torch.full_like(ids, -1), count, first)          # nobody any
        check_group(torch.full_like(ids, first + count), count, first)
        check_group(torch.full_like(ids, -2 ** 31), count, first)


@pytest.mark.parametrize("n", [7, 1024, 1025, 9000])
def test_group_memory_side_by_side_and_overlapping(n):
    """Neighbours in one piece of memory are apart; a call in the ids' own place is refused at every size."""
    room = torch.full((2 * n + 5,), -7, dtype=torch.int32, device="cuda")
    ids, order, offsets = room[:n], room[n:2 * n], room[2 * n:]
    ids.copy_(torch.randint(-1, 4, (n,), generator=gen(n), device="cuda", dtype=torch.int32))
    want = experts.group(ids.clone(), 4)
    got = experts.group(ids, 4, order=order, offsets=offsets)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    before = room.clone()
    for call in (lambda: experts.group(ids, 4, order=ids), lambda: experts.group(ids, 4, order=room[1:n + 1]), lambda: experts.group(ids, 4, offsets=room[n - 1:n + 4])):
        with pytest.raises(RuntimeError):
            call()
    assert torch.equal(room, before)


def test_route_memory_side_by_side_and_overlapping():
    """ids and weights between strided rows of logits, which they do not touch; where they do, the call is refused."""
    room = torch.randn(9, 200, generator=gen(3), device="cuda")
    x = room[:, :64]
    want = experts.route(x.contiguous(), 4)
    ids, w = room[2, 64:100].view(torch.int32).view(9, 4), room[5, 164:200].view(9, 4)
    got = experts.route(x, 4, ids=ids, weights=w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for kw in (dict(ids=room[2, 63:99].view(torch.int32).view(9, 4)), dict(weights=room.flatten()[1165:1201].view(9, 4)), dict(ids=ids, weights=ids.view(torch.float32))):
        with pytest.raises(RuntimeError):
            experts.route(x, 4, **kw)


# ---- the experts' products ----

class Mixture:
    def __init__(self, count, hidden, inner, seed=1, first=0):
        g = gen(seed)

        def made(n, k):
            w = torch.randint(-127, 128, (count, n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
            return w, (0.2 + torch.rand(count, n, generator=g, device="cuda")) / (70 * math.sqrt(k))

        self.count, self.hidden, self.inner, self.first = count, hidden, inner, first
        self.up, self.sup = made(2 * inner, hidden)
        self.down, self.sdown = made(hidden, inner)
        self.gate_up, self.out = int8.Int8Matrix(self.up, self.sup, paired=True), int8.Int8Matrix(self.down, self.sdown)

    def __call__(self, x, ids, w, **kw):
        return experts.ffn(x, ids, w, self.gate_up, self.out, first=self.first, **kw)

    def check(self, x, ids, w, got, residual=None):
        n, top = ids.shape
        xd = x.double()
        most = xd.abs().amax(1)
        s = (most / 127).float().double()
        bad = ~torch.isfinite(most)
        c = torch.where((bad | (s == 0)).unsqueeze(1), 0.0, torch.round(xd / s.unsqueeze(1)))
        s = torch.where(bad, math.nan, s)
        want = torch.zeros(n, self.hidden, dtype=torch.float64, device="cuda")
        size, tol = torch.zeros_like(want), torch.zeros_like(want)
        for e in range(self.count):
            r, j = (ids == self.first + e).nonzero(as_tuple=True)
            if not r.numel():
                continue
            y = (c[r] @ self.up[e].double().T) * self.sup[e].double() * s[r].unsqueeze(1)
            g, u = y[:, :self.inner], y[:, self.inner:]
            h = g * torch.sigmoid(g) * u
            eh = h.abs() * 11 * U + u.abs() * g.abs() * 3.3 * U + 1e-37
            hmost = h.abs().amax(1, keepdim=True)
            hs = (hmost / 127).float().double()
            off = (eh.amax(1, keepdim=True) / hmost).nan_to_num(0.0) + 2 * U
            q = torch.where(hs > 0, h / hs, 0.0)
            near = torch.where(hs > 0, eh / hs, 0.0) + q.abs() * off
            swing = ((q - torch.floor(q) - 0.5).abs() <= near).double()  # codes that may be the next one
            dn = self.down[e].double() * self.sdown[e].double().unsqueeze(1)
            a = (torch.round(q) @ dn.T) * hs
            wj = w[r, j].double().unsqueeze(1)
            a_tol = a.abs() * (3 * U + off) + (swing @ dn.abs().T) * hs * (1 + 4 * U)
            want.index_add_(0, r, a * wj)
            size.index_add_(0, r, (a * wj).abs())
            tol.index_add_(0, r, a_tol * wj.abs())
        if residual is not None:
            want = want + residual.double()
            tol = tol + U * want.abs()
        t = got.dtype
        tol = (tol + (top + 1) * U * size + 1e-36) * (1 + half_step(t)) * (1 + 1e-4) + half_step(t) * want.abs() + (2.0 ** -25 if t == torch.float16 else 0)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        miss = ~((got.double() - want).abs() <= tol) & ~torch.isnan(want)
        assert not miss.any(), (miss.nonzero()[:4].tolist(), (got.double() - want).abs().nan_to_num().max().item(), miss.sum().item())


def rows(n, k, dtype, seed):
    return (torch.randn(n, k, generator=gen(seed), device="cuda") * torch.logspace(-1, 1, n, device="cuda").unsqueeze(1)).to(T[dtype])


def choice(n, top, total, seed, low=0):
    ids = torch.randint(low, total, (n, top), generator=gen(seed), device="cuda", dtype=torch.int32)
    return ids, torch.rand(n, top, generator=gen(seed + 1), device="cuda")


@pytest.mark.parametrize("n,top,count,total,first,hidden,inner", [
    (1, 1, 1, 1, 0, 16, 16), (1, 6, 64, 64, 0, 256, 176), (1, 8, 16, 64, 16, 512, 256), (2, 2, 4, 4, 0, 130, 70), (3, 4, 8, 8, 0, 1, 1), (5, 8, 300, 300, 0, 64, 48),
    (7, 1, 2, 9, 4, 640, 1000), (16, 2, 8, 8, 0, 1024, 513), (17, 3, 5, 5, 0, 576, 1100), (32, 8, 16, 64, 32, 700, 300), (33, 2, 1, 1, 0, 256, 130),
    (64, 4, 3, 3, 0, 300, 256), (100, 2, 8, 8, 0, 384, 500), (257, 2, 5, 5, 0, 576, 1100), (300, 8, 32, 64, 0, 256, 256), (513, 1, 4, 5, 1, 1030, 640),
    (1000, 2, 8, 8, 0, 512, 700), (2049, 6, 64, 64, 0, 256, 128)])
@pytest.mark.parametrize("dtype", T)
def test_ffn(n, top, count, total, first, hidden, inner, dtype):
    m = Mixture(count, hidden, inner, seed=n + top, first=first)
    x = rows(n, hidden, dtype, 3)
    ids, w = choice(n, top, total, 5, low=-1)  # some places empty, the same expert twice in a row at times
    got = m(x, ids, w)
    assert got.dtype == x.dtype and got.shape == x.shape
    m.check(x, ids, w, got)


@pytest.mark.parametrize("n", [1, 4, 5])
@pytest.mark.parametrize("inner", [2047, 2048, 2049])
@pytest.mark.parametrize("hidden", [96, 100])
def test_ffn_where_slots_stop_being_done_one_by_one(n, inner, hidden):
    """Up to four rows of whole vectors whose hidden rows have up to 2048 values, and just behind."""
    m = Mixture(5, hidden, inner, seed=n)
    ids, w = choice(n, 64, 5, 5, low=-1)  # the most places of a row
    for dtype in T:
        x = rows(n, hidden, dtype, 3)
        m.check(x, ids, w, m(x, ids, w))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("count,top,hidden,inner", [(40, 16, 96, 2047), (40, 16, 100, 2048), (40, 16, 104, 2049), (40, 17, 96, 2048), (300, 16, 64, 48), (4, 4, 4096, 1024),
                                                    (2, 2, 2048, 2048), (1, 1, 4096, 2048), (1, 2, 4096, 2048), (3, 8, 1024, 1500), (5, 16, 96, 2048)])
def test_ffn_slot_by_slot_and_by_groups(count, top, hidden, inner, n):
    """A few rows, on both sides of where slots are no longer done one by one: by the places, by how often an expert's weights
    would be read. The same bits as in a larger batch, which goes by groups."""
    m = Mixture(count, hidden, inner, seed=count + top)
    ids, w = choice(40, top, count, 5, low=-1)
    for dtype in T:
        x = rows(40, hidden, dtype, 3)
        got = m(x[:n], ids[:n], w[:n])
        m.check(x[:n], ids[:n], w[:n], got)
        assert torch.equal(got, m(x, ids, w)[:n])
        kept = x[:n].clone()
        m(kept, ids[:n], w[:n], residual=kept, out=kept)
        assert torch.equal(kept, m(x, ids, w, residual=x)[:n])


@pytest.mark.parametrize("n,hidden,inner", [(100, 256, 14336), (65, 100, 16001), (600, 48, 14336), (1500, 300, 8200)])
def test_ffn_of_very_unequal_products(n, hidden, inner):
    """A wide first product by large blocks, a narrow second one by parts of them, the last part partly filled or empty."""
    m = Mixture(4, hidden, inner, seed=n)
    x = rows(n, hidden, "bf16", 3)
    ids, w = choice(n, 2, 4, 5, low=-1)
    m.check(x, ids, w, m(x, ids, w))
    ids[:, 0] = 2  # all rows to one expert
    m.check(x, ids, w, m(x, ids, w))


@pytest.mark.parametrize("hidden,inner", [(131072, 48), (48, 131072), (131072, 2048)])
def test_ffn_of_the_longest_rows(hidden, inner):
    m = Mixture(2, hidden, inner)
    for n in (1, 3, 6, 40, 200):
        for dtype in ("f32", "bf16"):
            x = rows(n, hidden, dtype, n)
            ids, w = choice(n, 2, 2, 5, low=-1)
            m.check(x, ids, w, m(x, ids, w))


def test_ffn_of_the_most_experts():
    m = Mixture(1024, 64, 32)
    for n, top in ((1, 8), (4, 64), (100, 8), (700, 64)):
        x = rows(n, 64, "f16", n)
        ids, w = choice(n, top, 1024, 5, low=-1)
        m.check(x, ids, w, m(x, ids, w))


def test_ffn_weights_past_32_bits():
    """18 experts of 8192 x 16384: the last one's gate and up lie 4.5 GB in."""
    m = Mixture(18, 8192, 16384)
    for n in (1, 40, 200):
        x = rows(n, 8192, "bf16", n)
        ids = torch.full((n, 2), 17, dtype=torch.int32, device="cuda")
        ids[:, 1] = -1
        w = torch.rand(n, 2, generator=gen(1), device="cuda")
        m.check(x, ids, w, m(x, ids, w))


def test_ffn_all_rows_to_one_expert_and_none():
    for n in (1, 15, 16, 130, 600):
        m = Mixture(7, 320, 200, seed=n)
        x = rows(n, 320, "f32", 3)
        w = torch.rand(n, 2, generator=gen(1), device="cuda")
        for e in (0, 6):
            ids = torch.full((n, 2), e, dtype=torch.int32, device="cuda")
            m.check(x, ids, w, m(x, ids, w))
        none = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
        assert (m(x, none, w) == 0).all()
        assert torch.equal(m(x, none, w, residual=x), x)


@pytest.mark.parametrize("dtype", T)
@pytest.mark.parametrize("n", [1, 9, 200])
def test_ffn_residual_in_place_strides_and_padding(n, dtype):
    m = Mixture(6, 200, 96, seed=2)
    ids, w = choice(n, 3, 6, 4)
    ids[n - n // 4:] = -1  # a padded batch
    wide = torch.randn(n, 230, generator=gen(8), device="cuda").to(T[dtype])
    kept = wide.clone()
    x = wide[:, 11:211]
    res = rows(n, 200, "f32", 9)
    room = torch.full((n, 215), 3.0, device="cuda")
    out = m(x, ids, w, residual=res, out=room[:, 7:207])
    m.check(x, ids, w, out, residual=res)
    assert (room[:, :7] == 3).all() and (room[:, 207:] == 3).all()
    before = x.clone()
    m(x, ids, w, residual=x, out=x)  # the rows' own place
    m.check(before, ids, w, x, residual=before)
    assert torch.equal(wide[:, :11], kept[:, :11]) and torch.equal(wide[:, 211:], kept[:, 211:])


def test_ffn_what_is_no_number_stays_in_its_row():
    for n in (4, 40, 300):
        m = Mixture(3, 128, 64, seed=3)
        ids, w = choice(n, 2, 3, 4)
        x = rows(n, 128, "bf16", 5)
        x[0, 5], x[2, 127] = math.nan, math.inf
        got = m(x, ids, w)
        assert torch.isnan(got).all(1).nonzero().flatten().tolist() == [0, 2] and not torch.isnan(got[1]).any()
        m.check(x, ids, w, got)
        w[1, 0] = math.nan  # a weight
        ids[3] = -1
        w[3] = math.nan     # of no expert: not looked at
        got = m(x, ids, w)
        assert torch.isnan(got[1]).all() and (got[3] == 0).all()


def test_ffn_large_and_small_values():
    """Hidden values beyond what 16 bits hold, and next to nothing."""
    for scale in (1e-18, 300.0, 1e4):
        m = Mixture(4, 256, 160, seed=6)
        x = rows(50, 256, "f32", 7) * scale
        ids, w = choice(50, 2, 4, 8)
        m.check(x, ids, w, m(x, ids, w))
        y = m(x, ids, w, out=torch.empty(50, 256, dtype=torch.bfloat16, device="cuda"))
        m.check(x, ids, w, y)


def test_ffn_gives_the_same_bits_every_time_and_in_any_batch():
    """Sums in a fixed order: a row's answer does not depend on the rows beside it, nor on the run."""
    m = Mixture(8, 384, 256, seed=4)
    x = rows(200, 384, "f32", 5)
    ids, w = choice(200, 3, 8, 6)
    whole = m(x, ids, w)
    for _ in range(3):
        assert torch.equal(m(x, ids, w), whole)
    for lo, hi in ((0, 1), (5, 21), (100, 200)):
        assert torch.equal(m(x[lo:hi], ids[lo:hi], w[lo:hi]), whole[lo:hi])


# ---- together ----

def layer(x, gate, m, bias, out=None, **space):
    """Routing, grouping and products of one layer, as a model calls them."""
    ids, w = experts.route(x @ gate, 4, scores="sigmoid", bias=bias, groups=4, top_groups=2, group_by="two", renormalize=True, scale=2.5,
                           **{k: space[k] for k in ("ids", "weights") if k in space})
    return ids, w, m(x, ids, w, residual=x, out=out, workspace=space.get("workspace"))


@pytest.mark.parametrize("n", [1, 24, 300])
def test_a_layer_captured_and_replayed(n):
    hidden, total = 512, 32
    m = Mixture(total, hidden, 192, seed=2)
    gate = torch.randn(hidden, total, generator=gen(1), device="cuda") / 8
    bias = torch.randn(total, generator=gen(2), device="cuda") * 0.1
    x = rows(n, hidden, "f32", 3)
    given = dict(out=torch.empty_like(x), ids=torch.empty(n, 4, dtype=torch.int32, device="cuda"), weights=torch.empty(n, 4, device="cuda"),
                 workspace=experts.ffn_workspace(m.gate_up, m.out, n, 4))
    layer(x, gate, m, bias, **given)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, gate, m, bias, **given)
    other = torch.cuda.Stream()
    for seed in range(4):
        x.copy_(rows(n, hidden, "f32", 50 + seed))
        given["out"].zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            ids, w, y = layer(x, gate, m, bias)
        torch.cuda.synchronize()
        assert torch.equal(ids, given["ids"]) and torch.equal(w, given["weights"]) and torch.equal(y, given["out"])
        m.check(x, ids, w, y, residual=x)
        check_group(ids, total)


def test_ranks_of_experts_add_up_to_the_whole():
    """Experts dealt to four holders: each adds its own to the sum so far."""
    whole = Mixture(16, 256, 128, seed=7)
    x = rows(60, 256, "f32", 8)
    ids, w = choice(60, 4, 16, 9)
    out = torch.zeros(60, 256, device="cuda")
    for r in range(4):
        part = [int8.Int8Matrix(c[4 * r:4 * r + 4], s[4 * r:4 * r + 4], paired=p) for c, s, p in ((whole.up, whole.sup, True), (whole.down, whole.sdown, False))]
        out = experts.ffn(x, ids, w, *part, first=4 * r, residual=out, out=out)
    whole.check(x, ids, w, out)


def test_shared_expert_of_rows_quantized_once():
    """A shared expert beside the routed ones: two products of rows already in 8 bits, then the routed experts on top."""
    m = Mixture(8, 256, 128, seed=7)
    one = Mixture(1, 256, 320, seed=8)
    x = rows(33, 256, "bf16", 9)
    held = int8.quantize(x)
    up = int8.Int8Matrix(one.up[0], one.sup[0], paired=True)
    down = int8.Int8Matrix(one.down[0], one.sdown[0])
    shared = int8.product(int8.product(held, up), down)
    one.check(x, torch.zeros(33, 1, dtype=torch.int32, device="cuda"), torch.ones(33, 1, device="cuda"), shared)
    ids, w = choice(33, 2, 8, 1)
    m.check(x, ids, w, m(x, ids, w, residual=shared, out=shared.clone()), residual=shared)


class _Rows:
    """Device memory of another owner as an array."""

    def __init__(self, address, shape):
        self.__cuda_array_interface__ = dict(shape=shape, typestr="<f4", data=(address, False), version=2)


def test_between_the_attention_layers_of_a_stack():
    """The feed-forward half of a layer on the attention stack's own hidden rows, between two layer steps."""
    batch, hidden, total = 3, 256, 16
    small = dict(hidden_dim=hidden, num_heads=16, q_lora_rank=128, kv_lora_rank=128, qk_nope_dim=128, qk_rope_dim=64, v_head_dim=128, kv_norm=1,
                 rms_norm_eps=1e-6, rope_theta=10000.0)
    m = Mixture(total, hidden, 96, seed=3)
    gate = torch.randn(hidden, total, generator=gen(1), device="cuda") / 8
    bias = torch.randn(total, generator=gen(2), device="cuda") * 0.1
    start = np.random.default_rng(5).standard_normal((batch, hidden)).astype(np.float32)
    stacks = [MlaEngine(small, max_seq_len=64, max_batch=batch, num_layers=2, seed=7, norm_sigma=0.1) for _ in range(2)]
    for s in stacks:
        for layer_ in range(2):
            for b in range(batch):
                s.fill_cache(layer_, b, 5 + b, seed=9, sigma=1.0)
                s.set_position(b, 5 + b)
        s.set_hidden(start)
        s.step(0, batch)
    h = torch.as_tensor(_Rows(stacks[0].buf.hidden, (batch, hidden)), device="cuda")
    before = h.clone()
    ids, w, y = layer(h, gate, m, bias, out=h)
    torch.cuda.synchronize()
    assert y.data_ptr() == stacks[0].buf.hidden
    m.check(before, ids, w, h, residual=before)
    stacks[1].set_hidden(h.cpu().numpy())
    for s in stacks:
        s.step(1, batch)
    a, b = (s.hidden(batch) for s in stacks)
    assert np.array_equal(a, b) and not np.array_equal(a, before.cpu().numpy())
    for s in stacks:
        s.close()


def test_refusals():
    m = Mixture(4, 64, 32)
    x, (ids, w) = torch.zeros(5, 64, device="cuda"), choice(5, 2, 4, 1)
    grad = torch.zeros(5, 64, device="cuda", requires_grad=True)
    lg = torch.zeros(5, 8, device="cuda")
    for call in (lambda: m(x[:, :63], ids, w), lambda: m(x.double(), ids, w), lambda: m(x.cpu(), ids, w), lambda: m(grad, ids, w), lambda: m(x, ids[:4], w),
                 lambda: m(x, ids.long(), w), lambda: m(x, ids, w.half()), lambda: m(x, ids, w[:, :1]), lambda: m(x, ids, w, out=x[:4]),
                 lambda: m(x, ids, w, residual=x[:, :60]), lambda: m(x, ids.t().contiguous().t(), w), lambda: m(x, ids, w.requires_grad_()),
                 lambda: experts.ffn(x, ids, w, m.out, m.gate_up), lambda: experts.ffn(x, ids, w, m.gate_up, Mixture(3, 64, 32).out),
                 lambda: experts.ffn(x, ids, w.detach(), m.gate_up, m.out, first=-1),
                 lambda: experts.route(lg, 9), lambda: experts.route(lg, 0), lambda: experts.route(lg, 2, scores="none"), lambda: experts.route(lg, 2, group_by="x"),
                 lambda: experts.route(lg, 2, groups=3), lambda: experts.route(lg, 3, groups=4), lambda: experts.route(lg, 2, groups=2, top_groups=3),
                 lambda: experts.route(lg[0], 2), lambda: experts.route(lg.long(), 2), lambda: experts.route(lg, 2, bias=torch.zeros(7, device="cuda")),
                 lambda: experts.route(lg, 2, ids=ids[:, :1]), lambda: experts.route(torch.zeros(1, 1025, device="cuda"), 2),
                 lambda: experts.route(lg.requires_grad_(), 2), lambda: experts.group(ids.long(), 4), lambda: experts.group(ids, 0), lambda: experts.group(ids, 1025),
                 lambda: experts.group(ids, 4, -1), lambda: experts.group(ids, 4, order=ids.flatten()[:3]), lambda: experts.group(ids.t(), 4)):
        with pytest.raises(ValueError):
            call()
    w = w.detach()
    for call in (lambda: m(x, ids, w, workspace=torch.empty(100, dtype=torch.uint8, device="cuda")),
                 lambda: experts.group(torch.zeros(9000, 1, dtype=torch.int32, device="cuda"), 4, workspace=torch.empty(4, dtype=torch.uint8, device="cuda")),
                 lambda: experts.route(lg.detach(), 2, scale=math.inf), lambda: experts.ffn_workspace(m.out, m.out, 3, 2)):
        with pytest.raises(RuntimeError):
            call()
