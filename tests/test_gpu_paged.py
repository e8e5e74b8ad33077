"""The paged cache on the GPU against plain float64 computations of the same inputs.

Tolerances are derived from the roundings: u(t) = finfo(t).eps / 2 is half a step of a type. An output o of
attention may be off by its own rounding u(out) |o| and by c A, A = sum_j p_j |v_j|, where c collects the relative
errors of the weights p: twice the error of a score (a product of d terms summed in fp32: (d + 8) u(f32) times
its absolute sum, plus 2^-22 times the largest score for the exponential's argument), the rounding of p to the
cache's type where q is of that type too (u(kv); 2^-20 where it is not, and p is kept in several terms), and the
sum over n weights in fp32 (n + 64) u(f32).
"""
import math

import numpy as np
import pytest
import torch

from velox_amd import _lib as L
from velox_amd import paged

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SLOT = np.array([8 * ((r % 16) // 4) + 4 * (r // 16) + r % 4 for r in range(32)])


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(list(map(int, x)), dtype=torch.int32, device="cuda")


class Filled:
    """A cache of one layer whose places are NaN but for K and V of each sequence's positions, in pages of a
    random order; hidden positions' pages can be taken away."""

    def __init__(self, lens, hkv, d, page, kv, seed=1, spare=2, amp=1.0):
        g = gen(seed)
        self.hkv, self.d, self.page, self.lens = hkv, d, page, list(lens)
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g, device="cuda").tolist()
        table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
        self.pool = torch.full((1, total, 2 * hkv * page * d), float("nan"), dtype=T[kv], device="cuda")
        self.k, self.v = [], []
        slot = torch.tensor(SLOT, device="cuda")
        at = 0
        for s, n in enumerate(lens):
            k = (torch.randn(n, hkv, d, generator=g, device="cuda") * amp).to(T[kv])
            v = torch.randn(n, hkv, d, generator=g, device="cuda").to(T[kv])
            self.k.append(k)
            self.v.append(v)
            for j in range(need[s]):
                number = order[at]
                at += 1
                table[s, j] = number
                lo, hi = j * page, min(n, (j + 1) * page)
                cell = self.pool[0, number]
                cell[:hkv * page * d].view(hkv, page, d)[:, :hi - lo] = k[lo:hi].transpose(0, 1)
                vv = cell[hkv * page * d:].view(hkv, page // 32, d, 32)
                r = torch.arange(hi - lo, device="cuda")
                for h in range(hkv):
                    vv[h, r // 32, :, slot[r % 32]] = v[lo:hi, h]
        self.table = table.cuda()
        self.cache = paged.PagedCache.over(self.pool, self.table, ints(lens), page_size=page, num_kv_heads=hkv, head_dim=d)

    def no_page(self, s, j, value=-1):
        self.table[s, j] = value

    def check(self, q, out, seq, row0, window, sinks, same_type, scale=None, gone=()):
        """Rows row0 .. of sequence `seq` (the last one its newest position) against the formula."""
        hq, d = q.shape[1], self.d
        n = self.lens[seq]
        rows = q.shape[0]
        scale = scale or 1 / math.sqrt(d)
        t = torch.arange(n - rows, n, device="cuda").unsqueeze(1)
        j = torch.arange(n, device="cuda").unsqueeze(0)
        seen = j <= t
        if window:
            seen = seen & ((j > t - window) | (j < sinks))
        for p in gone:
            seen = seen & (j // self.page != p)
        k, v = self.k[seq].double(), self.v[seq].double()
        for h in range(hq):
            g = h // (hq // self.hkv)
            x = q[:, h].double()
            s = torch.where(seen, x @ k[:, g].T * scale, -math.inf)
            big = torch.where(seen, x.abs() @ k[:, g].abs().T * abs(scale), 0.0).amax(1, keepdim=True) if n else torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
            any_ = seen.any(1, keepdim=True) if n else torch.zeros(rows, 1, dtype=torch.bool, device="cuda")
            p = torch.where(any_, torch.softmax(torch.where(any_, s, 0.0), 1), 0.0) if n else s
            o = p @ v[:, g] if n else torch.zeros(rows, d, dtype=torch.float64, device="cuda")
            a = p @ v[:, g].abs() if n else torch.zeros_like(o)
            u = half_step(torch.float32)
            c = 2 * ((d + 8) * u * big + 2 ** -22 * big) + (half_step(self.pool.dtype) if same_type else 2 ** -20) + (n + 64) * u
            got = out[:, h].double()
            tol = half_step(out.dtype) * o.abs() * (1 + c) + c * a * (1 + half_step(out.dtype)) + 1e-30
            if out.dtype == torch.float16:
                tol = tol + 2.0 ** -25  # its least positive step
            bad = ~((got - o).abs() <= tol)
            assert not bad.any(), (seq, h, bad.nonzero()[:4].tolist(), (got - o).abs().max().item(), tol.min().item())


def queries(rows, hq, hkv, d, dtype, seed=7):
    """q as a slice of fused q/k/v rows."""
    x = torch.randn(rows, (hq + 2 * hkv) * d, generator=gen(seed), device="cuda").to(T[dtype])
    return x[:, :hq * d].unflatten(1, (hq, d))


LENS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1023, 1500]


@pytest.mark.parametrize("hq,hkv,d,page,q,kv", [(9, 3, 64, 32, "f32", "bf16"), (32, 8, 128, 64, "bf16", "bf16"), (28, 4, 128, 96, "f32", "f16"),
                                                (4, 4, 64, 256, "f16", "f16"), (40, 2, 128, 32, "f32", "bf16"), (17, 1, 64, 64, "bf16", "f16"),
                                                (16, 1, 128, 64, "f16", "bf16")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 3), (33, 70), (600, 4)])
def test_token_attention(hq, hkv, d, page, q, kv, window, sinks):
    f = Filled(LENS, hkv, d, page, kv)
    x = queries(len(LENS), hq, hkv, d, q)
    for max_len in (0, 1500):
        out = paged.attention(f.cache, 0, x, window=window, sinks=sinks, max_len=max_len)
        assert out.dtype == x.dtype
        for s in range(len(LENS)):
            f.check(x[s:s + 1], out[s:s + 1], s, s, window, sinks, q == kv)


def test_token_attention_long_and_planned_short():
    """One long sequence (split over workgroups), also where the bound it is planned by is far too low."""
    f = Filled([20011], 2, 128, 64, "bf16")
    x = queries(1, 8, 2, 128, "f32")
    for max_len in (0, 20011, 100):
        for window, sinks in ((0, 0), (5000, 4), (19990, 40)):
            f.check(x, paged.attention(f.cache, 0, x, window=window, sinks=sinks, max_len=max_len), 0, 0, window, sinks, False)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_token_attention_output_types_strides_and_scale(out):
    f = Filled([300, 7], 2, 64, 32, "bf16")
    x = queries(2, 6, 2, 64, "f32")
    room = torch.full((2, 6, 80), 9.0, dtype=T[out], device="cuda")
    o = paged.attention(f.cache, 0, x, out=room[:, :, 8:72], scale=0.3)
    assert o.data_ptr() == room[:, :, 8:72].data_ptr() and (room[:, :, :8] == 9).all() and (room[:, :, 72:] == 9).all()
    for s in range(2):
        f.check(x[s:s + 1], o[s:s + 1], s, s, 0, 0, False, scale=0.3)
    odd = torch.randn(2 * 6 * 65 + 1, device="cuda")[1:].unflatten(0, (2, 6, 65))[:, :, :64]  # no 16-byte alignment
    o = paged.attention(f.cache, 0, odd)
    for s in range(2):
        f.check(odd[s:s + 1], o[s:s + 1], s, s, 0, 0, False)


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("bf16", "f16")])
def test_attention_in_place_at_any_alignment_with_a_negative_scale(q, kv):
    lens, start = [70, 33], [0, 40, 45]
    f = Filled(lens, 2, 64, 32, kv)
    flat = torch.randn(45 * 6 * 65 + 1, generator=gen(4), device="cuda").to(T[q])
    for shift in (0, 1):
        x = flat[shift:shift + 45 * 6 * 65].unflatten(0, (45, 6, 65))[:, :, :64]
        for scale in (0.2, -0.2):
            room = flat.clone()
            y = room[shift:shift + 45 * 6 * 65].unflatten(0, (45, 6, 65))[:, :, :64]
            assert paged.prompt_attention(f.cache, 0, y, ints(start), scale=scale, out=y) is y
            for s in range(2):
                f.check(x[start[s]:start[s + 1]], y[start[s]:start[s + 1]], s, 0, 0, 0, q == kv, scale=scale)
            assert torch.equal(room[:shift], flat[:shift])
            y = room[shift:shift + 45 * 6 * 65].unflatten(0, (45, 6, 65))[:, :, :64]
            y.copy_(x)
            assert paged.attention(f.cache, 0, y[:2], scale=scale, out=y[:2]).data_ptr() == y.data_ptr()
            for s in range(2):
                f.check(x[s:s + 1], y[s:s + 1], s, 0, 0, 0, q == kv, scale=scale)


def test_weights_far_below_the_largest():
    """One position holds most of the weight, thousands of others 2^-20 of it each: fp16 weights would lose bits."""
    n, d = 8000, 64
    for q, kv in (("f16", "f16"), ("f32", "f16"), ("bf16", "bf16")):
        f = Filled([n], 1, d, 32, kv)
        f.pool[0].view(-1, 2, 32 * d)[:, 0] = 0
        for s, k in enumerate(f.k):
            k.zero_()
        number, r = int(f.table[0, 40 // 32]), 40 % 32
        f.pool[0, number, r * d] = 8.0
        f.k[0][40, 0, 0] = 8.0
        x = torch.zeros(3, 2, d, device="cuda").to(T[q])
        x[:, :, 0] = 20 * math.log(2)  # times 8 / 8
        f.check(x[:1], paged.attention(f.cache, 0, x[:1]), 0, 0, 0, 0, q == kv)
        f.check(x, paged.prompt_attention(f.cache, 0, x, ints([0, 3])), 0, 0, 0, 0, q == kv)


def test_token_attention_large_values():
    """Scores of several hundred: the weights fall to nothing but for a few."""
    f = Filled([900, 40], 1, 128, 32, "bf16", amp=30.0)
    x = queries(2, 4, 1, 128, "f32") * 5
    out = paged.attention(f.cache, 0, x)
    assert torch.isfinite(out).all()
    for s in range(2):
        f.check(x[s:s + 1], out[s:s + 1], s, s, 0, 0, False)


@pytest.mark.parametrize("q,kv", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("value", [-1, 1 << 30])
def test_positions_without_a_page_are_left_out(q, kv, value):
    f = Filled([200, 96, 32], 2, 64, 32, kv)
    f.no_page(0, 2, value)
    f.no_page(0, 6, value)  # the newest position's own
    f.no_page(2, 0, value)  # all there is
    x = queries(3, 4, 2, 64, q)
    gone = [(2, 6), (), (0,)]
    out = paged.attention(f.cache, 0, x)
    for s in range(3):
        f.check(x[s:s + 1], out[s:s + 1], s, s, 0, 0, q == kv, gone=gone[s])
    assert (out[2] == 0).all()
    x = queries(40, 4, 2, 64, q)
    out = paged.prompt_attention(f.cache, 0, x, ints([0, 20, 30, 40]))
    for s, (lo, hi) in enumerate(((0, 20), (20, 30), (30, 40))):
        f.check(x[lo:hi], out[lo:hi], s, lo, 0, 0, q == kv, gone=gone[s])


def test_lengths_past_the_table_are_left_out():
    f = Filled([64], 2, 64, 32, "bf16")
    n = f.table.shape[1] * 32
    x = queries(1, 4, 2, 64, "f32")
    for more in (1000, 2 ** 31 - 1 - n):
        f.cache.lens.fill_(n + more)
        f.check(x, paged.attention(f.cache, 0, x), 0, 0, 0, 0, False)
        f.check(x, paged.prompt_attention(f.cache, 0, x, ints([0, 1])), 0, 0, 0, 0, False)
        assert (paged.attention(f.cache, 0, x, window=500) == 0).all()
        assert (paged.prompt_attention(f.cache, 0, x, ints([0, 1]), window=500) == 0).all()
        f.lens[0] = 40  # of a window that lies behind the table the sinks are left
        k, v = f.k[0], f.v[0]
        f.k[0], f.v[0] = k[:40], v[:40]
        f.check(x, paged.attention(f.cache, 0, x, window=500, sinks=40), 0, 0, 0, 0, False)
        f.check(x, paged.prompt_attention(f.cache, 0, x, ints([0, 1]), window=500, sinks=40), 0, 0, 0, 0, False)
        f.lens[0], f.k[0], f.v[0] = 64, k, v


@pytest.mark.parametrize("hq,hkv,d,page,q,kv", [(9, 3, 64, 32, "f32", "f16"), (8, 2, 128, 64, "bf16", "bf16"), (28, 4, 128, 96, "f16", "f16"),
                                                (6, 6, 64, 128, "f32", "bf16"), (33, 1, 64, 32, "bf16", "bf16"), (4, 1, 128, 64, "f16", "bf16")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 3), (100, 70)])
def test_prompt_attention(hq, hkv, d, page, q, kv, window, sinks):
    lens = [300, 5, 0, 64, 129, 1, 700, 33]
    rows = [300, 5, 0, 1, 100, 1, 37, 2]
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    f = Filled(lens, hkv, d, page, kv)
    x = queries(start[-1] + 5, hq, hkv, d, q)
    out = torch.full((start[-1] + 5, hq, d), 7.0, dtype=x.dtype, device="cuda")
    paged.prompt_attention(f.cache, 0, x, ints(start), window=window, sinks=sinks, out=out, max_rows=300, max_len=700)
    assert (out[start[-1]:] == 7).all()  # behind the last sequence
    for s in range(len(lens)):
        f.check(x[start[s]:start[s + 1]], out[start[s]:start[s + 1]], s, start[s], window, sinks, q == kv)


def test_prompt_attention_few_rows_behind_a_long_context():
    lens, start = [9000, 4100], [0, 3, 20]
    f = Filled(lens, 2, 128, 64, "bf16")
    for q in ("bf16", "f32"):
        x = queries(20, 8, 2, 128, q)
        for window, sinks in ((0, 0), (4000, 5)):
            out = paged.prompt_attention(f.cache, 0, x, ints(start), window=window, sinks=sinks, max_rows=17, max_len=9000)
            for s in range(2):
                f.check(x[start[s]:start[s + 1]], out[start[s]:start[s + 1]], s, 0, window, sinks, q == "bf16")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows, n", [(1100, 8000), (2000, 2100), (40, 1700), (9, 40000)])
def test_prompt_attention_in_few_and_many_splits(d, rows, n):
    f = Filled([n], 2, d, 64, "bf16")
    x = queries(rows, 4, 2, d, "bf16")
    space = f.cache.prompt_workspace(4, total_rows=rows)
    assert space is not None
    out = paged.prompt_attention(f.cache, 0, x, ints([0, rows]), workspace=space)
    f.check(x, out, 0, 0, 0, 0, True)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[2000] * 6, [1000] * 40, [30000, 7], [3000] * 30])
def test_token_attention_in_few_and_many_splits(d, lens):
    f = Filled(lens, 2, d, 64, "bf16")
    x = queries(len(lens), 4, 2, d, "f32")
    out = paged.attention(f.cache, 0, x)
    for s in range(len(lens)):
        f.check(x[s:s + 1], out[s:s + 1], s, 0, 0, 0, False)


def test_prompt_rows_in_front_of_position_0_stay():
    f = Filled([4], 2, 64, 32, "bf16")
    x = queries(10, 4, 2, 64, "bf16")
    out = torch.full((10, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    paged.prompt_attention(f.cache, 0, x, ints([0, 10]), out=out)
    assert (out[:6] == 7).all()
    f.check(x[6:], out[6:], 0, 6, 0, 0, True)


@pytest.mark.parametrize("lens", [(9000, 7000), (40, 30)], ids=["split", "whole"])
def test_prompt_rows_of_no_sequence_stay(lens):
    f = Filled(lens, 2, 64, 32, "bf16")
    x = queries(20, 4, 2, 64, "bf16")
    out = torch.full((20, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    space = f.cache.prompt_workspace(4, total_rows=20)
    assert (space is None) == (lens[0] < 1000)
    if space is not None:
        space.zero_()
    paged.prompt_attention(f.cache, 0, x, ints([3, 8, 15]), out=out, workspace=space)
    assert (out[:3] == 7).all() and (out[15:] == 7).all()
    f.check(x[3:8], out[3:8], 0, 0, 0, 0, True)
    f.check(x[8:15], out[8:15], 1, 0, 0, 0, True)


@pytest.mark.parametrize("q,kv", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_rows_do_not_see_what_later_or_left_positions_hold(q, kv, value):
    """A K or V value that is no number reaches the rows that see its position and no others."""
    d, window, sinks, n, rows = 64, 50, 2, 400, 300
    for where in (1, 130, 199, 300, 399):
        f = Filled([n], 1, d, 64, kv)
        cell = f.pool[0, int(f.table[0, where // 64])]
        v = cell[64 * d:].view(2, d, 32)
        v[where % 64 // 32, 5, int(SLOT[where % 32])] = value
        x = queries(rows, 3, 1, d, q)
        t = torch.arange(n - rows, n, device="cuda")
        sees = (t >= where) & ((t < where + window) | (where < sinks))
        out = paged.prompt_attention(f.cache, 0, x, ints([0, rows]), window=window, sinks=sinks)
        # the seeing rows get no number: infinity, or NaN where a weight is held in terms of both signs (p0 inf + p1 inf)
        assert torch.equal(torch.isfinite(out[:, :, 5]), ~sees.view(-1, 1).expand(rows, 3))
        keep = [e for e in range(d) if e != 5]
        other = out.clone()
        other[:, :, 5] = 0
        f.v[0][:, 0, 5] = 0  # that dimension is looked at above
        f.check(x, other, 0, 0, window, sinks, q == kv)
        assert torch.isfinite(out[:, :, keep]).all()
        one = paged.attention(f.cache, 0, x[-1:], window=window, sinks=sinks)
        assert torch.isfinite(one[0, :, 5]).all() == (not bool(sees[-1])) and torch.isfinite(one[:, :, keep]).all()
        f = Filled([n], 1, d, 64, kv)
        cell = f.pool[0, int(f.table[0, where // 64])]
        cell[:64 * d].view(64, d)[where % 64, 9] = value
        out = paged.prompt_attention(f.cache, 0, x, ints([0, rows]), window=window, sinks=sinks)
        assert torch.isfinite(out[~sees]).all()
        for i in (~sees).nonzero().flatten()[::37].tolist():  # a few rows by themselves
            g = Filled([n], 1, d, 64, kv)
            g.lens[0] = n - rows + i + 1
            g.k[0], g.v[0] = g.k[0][:g.lens[0]], g.v[0][:g.lens[0]]
            g.check(x[i:i + 1], out[i:i + 1], 0, i, window, sinks, q == kv)


def test_prompt_attention_many_sequences():
    """More sequences than a wave counts at once, most of them without rows."""
    lens = [(i * 13) % 70 for i in range(150)]
    rows = [n if i % 3 == 0 else 0 for i, n in enumerate(lens)]
    start = np.concatenate([[0], np.cumsum(rows)]).tolist()
    f = Filled(lens, 1, 64, 32, "bf16")
    x = queries(start[-1], 2, 1, 64, "bf16")
    out = paged.prompt_attention(f.cache, 0, x, ints(start), window=20, sinks=2)
    for s in range(150):
        if rows[s]:
            f.check(x[start[s]:start[s + 1]], out[start[s]:start[s + 1]], s, 0, 20, 2, True)


def test_attention_past_32_bit_offsets():
    """Pages whose elements lie past 2^32."""
    hkv, d, page = 8, 128, 256
    f = Filled([700, 300], hkv, d, page, "bf16")
    elements = 2 * hkv * page * d
    n_pages = (1 << 32) // elements + 40
    pool = torch.empty(1, n_pages, elements, dtype=torch.bfloat16, device="cuda")
    far = n_pages - f.pool.shape[1]
    pool[0, far:] = f.pool[0]
    table = torch.where(f.table >= 0, f.table + far, f.table)
    cache = paged.PagedCache.over(pool, table, f.cache.lens, page_size=page, num_kv_heads=hkv, head_dim=d)
    x = queries(2, 16, hkv, d, "bf16")
    out = paged.attention(cache, 0, x)
    start = ints([0, 1, 2])
    out2 = paged.prompt_attention(cache, 0, x, start)
    for s in range(2):
        f.check(x[s:s + 1], out[s:s + 1], s, s, 0, 0, True)
        f.check(x[s:s + 1], out2[s:s + 1], s, s, 0, 0, True)


def test_attention_over_an_arenas_layout(hiplib):
    """A layer cache of velox_hip_attention_decode is one page: the same answer over it."""
    hq, hkv, d, s_max, pos = 32, 8, 128, 512, 300
    cap = 512
    g = gen(3)
    kv = torch.randn(2 * hkv * cap * d, generator=g, device="cuda").to(torch.bfloat16)
    qkv = torch.randn((hq + 2 * hkv) * d, generator=g, device="cuda")
    want = torch.empty(hq * d, device="cuda")
    L.check(hiplib.velox_hip_attention_decode(qkv.data_ptr(), kv.data_ptr(), hq, hkv, d, s_max, pos, 10000.0, 4, want.data_ptr(), None))
    turned = paged.rope(paged.Rope(d), qkv[:hq * d].view(1, hq, d), ints([pos]))
    cache = paged.PagedCache.over(kv.view(1, 1, -1), ints([0]).view(1, 1), ints([pos + 1]), page_size=cap, num_kv_heads=hkv, head_dim=d)
    got = paged.attention(cache, 0, turned)
    # k was rounded to bf16 from fp32 angles there and here from one rotation: the newest position may differ
    # by the angle's fp32 rounding, pos 2^-24 radians on values of up to about 4
    assert (got.view(-1) - want).abs().max().item() < 4 * pos * 2 ** -23 * 4


# ---- rotation and append ----------------------------------------------------------------------------

def turned(x, positions, turn, interleaved):
    """float64 rotation and the absolute sums that its tolerance takes."""
    freq, amp = turn.frequencies()
    r = turn.rot_dim
    y, size = x.double().clone(), x.double().abs()
    a = positions.double().unsqueeze(1) * torch.tensor(freq, dtype=torch.float64, device="cuda")
    c, s = torch.cos(a).unsqueeze(1) * amp, torch.sin(a).unsqueeze(1) * amp
    i0 = slice(0, r, 2) if interleaved else slice(0, r // 2)
    i1 = slice(1, r, 2) if interleaved else slice(r // 2, r)
    p, q = x[..., i0].double(), x[..., i1].double()
    y[..., i0], y[..., i1] = p * c - q * s, q * c + p * s
    both = (p.abs() + q.abs()) * amp
    size[..., i0], size[..., i1] = both, both
    return y, size


def close_turn(got, want, size, dtype):
    # cos and sin: the angle's fraction of a turn is rounded to fp32 (pi 2^-24 rad) and the functions are
    # good to a few steps; two products and a sum in fp32
    tol = half_step(dtype) * want.abs() + size * (math.pi * 2 ** -24 + 8 * half_step(torch.float32)) * (1 + half_step(dtype))
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max().item()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot,scaling", [(64, 64, "none"), (128, 128, "bands"), (128, 64, "yarn"), (64, 18, "linear"), (65, 6, "none"),
                                           (256, 256, "none"), (128, 2, "yarn"), (96, 80, "none")])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rope_rows(layout, d, rot, scaling, dtype):
    turn = paged.Rope(rot, theta=5e5, layout=layout, scaling=scaling, factor=8.0, original_len=8192)
    for rows, heads in ((1, 1), (5, 9), (37, 3)):
        x = torch.randn(rows, heads, d, generator=gen(rows), device="cuda").to(T[dtype])
        at = torch.randint(0, 2 ** 31 - 1, (rows,), generator=gen(5), device="cuda", dtype=torch.int32)
        at[0] = 0
        if rows > 2:
            at[1:3] = ints([1, 1000003])
        want, size = turned(x, at, turn, layout == "interleaved")
        got = paged.rope(turn, x, at)
        close_turn(got, want, size, T[dtype])
        same = x.clone()  # in place
        assert paged.rope(turn, same, at, out=same) is same
        assert torch.equal(same, got)
        wide = torch.zeros(rows, heads * d + 3, dtype=T[dtype], device="cuda")  # rows without 16-byte alignment
        view = wide[:, 1:1 + heads * d].unflatten(1, (heads, d))
        view.copy_(x)
        out = torch.zeros(heads, rows, d + 8, dtype=T[dtype], device="cuda")
        paged.rope(turn, view, at, out=out.transpose(0, 1)[:, :, :d])
        assert torch.equal(out.transpose(0, 1)[:, :, :d], got) and (out[:, :, d:] == 0).all()


def test_rope_no_rows():
    x = torch.zeros(0, 4, 64, device="cuda")
    assert paged.rope(paged.Rope(64), x, ints([])).shape == (0, 4, 64)


def unpacked(pool, hkv, page, d):
    """K and V of a layer's pages, [page][KV head][position][d]."""
    n = pool.shape[0]
    cells = pool.view(n, 2, hkv, page * d)
    k = cells[:, 0].view(n, hkv, page, d)
    v = cells[:, 1].view(n, hkv, page // 32, d, 32)[..., torch.tensor(SLOT, device="cuda")].transpose(3, 4).reshape(n, hkv, page, d)
    return k, v


@pytest.mark.parametrize("hq,hkv,d,page,rot,layout,q,kv", [(9, 3, 64, 32, 64, "half", "f32", "bf16"), (8, 2, 128, 64, 128, "half", "bf16", "bf16"),
                                                           (4, 4, 128, 96, 34, "interleaved", "f16", "f16"), (2, 1, 64, 32, 32, "half", "f32", "f16"),
                                                           (6, 2, 64, 64, 64, "interleaved", "bf16", "f16")])
@pytest.mark.parametrize("rows,before", [([1, 1, 1, 1], [0, 31, 32, 100]), ([70, 0, 5, 33], [0, 4, 30, 17]), ([200, 1, 64, 32], [1, 63, 32, 0])])
def test_append(hq, hkv, d, page, rot, layout, q, kv, rows, before):
    lens = [r + b for r, b in zip(rows, before)]
    start = np.concatenate([[0], np.cumsum(rows)]).tolist()
    total = start[-1]
    f = Filled(lens, hkv, d, page, kv)
    before_pool = f.pool.clone()
    x = torch.randn(total + 3, (hq + 2 * hkv) * d, generator=gen(2), device="cuda").to(T[q])
    xq, xk, xv = (x[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    turn = paged.Rope(rot, layout=layout, theta=1e6)
    out = torch.full((total + 3, hq, d), 5.0, dtype=T[q], device="cuda")
    paged.rope_append(f.cache, 0, turn, xq, xk, xv, out, q_start=ints(start))
    assert (out[total:] == 5).all()
    k, v = unpacked(f.pool[0], hkv, page, d)
    k0, v0 = unpacked(before_pool[0].clone(), hkv, page, d)
    for s, n in enumerate(lens):
        lo, hi = start[s], start[s + 1]
        at = torch.arange(before[s], n, device="cuda")
        want, size = turned(xq[lo:hi], at, turn, layout == "interleaved")
        close_turn(out[lo:hi], want, size, T[q])
        number, r = f.table[s, at // page].long(), at % page
        want, size = turned(xk[lo:hi], at, turn, layout == "interleaved")
        close_turn(k[number, :, r], want, size, T[kv])
        assert torch.equal(v[number, :, r], xv[lo:hi].to(T[kv]))
        k0[number, :, r], v0[number, :, r] = k[number, :, r], v[number, :, r]
    bits = torch.int16
    assert torch.equal(k.contiguous().view(bits), k0.contiguous().view(bits)) and torch.equal(v.contiguous().view(bits), v0.contiguous().view(bits))
    # the same in place, and k and v alone
    pool = f.pool.clone()
    f.pool.copy_(before_pool)
    paged.rope_append(f.cache, 0, turn, xq, xk, xv, xq, q_start=ints(start))
    assert torch.equal(xq[:total], out[:total]) and torch.equal(f.pool.view(bits), pool.view(bits))
    f.pool.copy_(before_pool)
    assert paged.rope_append(f.cache, 0, turn, None, xk, xv, q_start=ints(start)) is None
    assert torch.equal(f.pool.view(bits), pool.view(bits))


def test_append_one_row_each_without_rotation_and_without_pages():
    f = Filled([40, 5, 64], 2, 64, 32, "bf16")
    f.no_page(1, 0)
    f.no_page(2, 1, 1 << 29)
    before = f.pool.clone()
    x = torch.randn(3, 8, 64, generator=gen(1), device="cuda")
    out = paged.rope_append(f.cache, 0, None, x[:, :4], x[:, 4:6], x[:, 6:])
    assert torch.equal(out, x[:, :4])
    k, v = unpacked(f.pool[0], 2, 32, 64)
    number = int(f.table[0, 1])
    assert torch.equal(k[number, :, 7], x[0, 4:6].bfloat16()) and torch.equal(v[number, :, 7], x[0, 6:].bfloat16())
    k0, v0 = unpacked(before[0], 2, 32, 64)
    same = [p for p in range(f.pool.shape[1]) if p != number]
    assert torch.equal(f.pool[0, same].view(torch.int16), before[0, same].view(torch.int16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_many_sequences_of_few_rows(dtype, ragged):
    """130 sequences at once give, bit for bit, what 13 batches of ten give."""
    n, hq, hkv, d, page = 130, 6, 2, 128, 32
    rng = np.random.default_rng(3)
    count = rng.integers(0, 4, n) if ragged else np.ones(n, int)
    a = paged.PagedCache(n * 4, n, 4, page_size=page, num_kv_heads=hkv, head_dim=d)
    a.extend(ints(rng.integers(1, 60, n).tolist()))
    a.extend(ints(count.tolist()))
    b = torch.zeros_like(a.pool)
    start = np.concatenate([[0], np.cumsum(count)])
    x = torch.randn(int(start[-1]), hq + 2 * hkv, d, generator=gen(4), device="cuda").to(dtype)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    turn = paged.Rope(d, layout="interleaved" if ragged else "half")
    out = paged.rope_append(a, 0, turn, q, k, v, q_start=ints(start.tolist()) if ragged else None)
    parts = []
    for s in range(0, n, 10):
        c = paged.PagedCache.over(b, a.table[s:s + 10], a.lens[s:s + 10], page_size=page, num_kv_heads=hkv, head_dim=d)
        r = slice(int(start[s]), int(start[s + 10]))
        own = ints((start[s:s + 11] - start[s]).tolist()) if ragged else None
        parts.append(paged.rope_append(c, 0, turn, q[r], k[r], v[r], q_start=own))
    assert torch.equal(out, torch.cat(parts)) and torch.equal(a.pool, b)


def test_append_more_rows_than_positions_leaves_the_front_ones():
    f = Filled([3], 1, 64, 32, "bf16")
    x = torch.randn(10, 4, 64, device="cuda")
    out = torch.full((10, 2, 64), 5.0, device="cuda")
    paged.rope_append(f.cache, 0, None, x[:, :2], x[:, 2:3], x[:, 3:], out, q_start=ints([0, 10]))
    assert (out[:7] == 5).all() and torch.equal(out[7:], x[7:, :2])
    k, _ = unpacked(f.pool[0], 1, 32, 64)
    assert torch.equal(k[int(f.table[0, 0]), 0, :3], x[7:, 2].bfloat16())


# ---- pages ----------------------------------------------------------------------------------------

class Model:
    """The page rules, sequence by sequence; a page's data is a number that goes wherever it is copied."""

    def __init__(self, n_pages, n_seqs, max_pages, page):
        self.n, self.m, self.page = n_pages, max_pages, page
        self.table = [[-1] * max_pages for _ in range(n_seqs)]
        self.lens, self.refs = [0] * n_seqs, [0] * n_pages
        self.data = list(range(n_pages))

    def free(self):
        return [p for p in range(self.n) if self.refs[p] == 0]

    def extend(self, add):
        up = lambda x: -(-x // self.page)  # noqa: E731
        want = {}
        for s, a in enumerate(add):
            n = self.lens[s]
            if a and up(n + a) <= self.m:
                p = self.table[s][up(n) - 1] if n % self.page else -1
                want[s] = p if p >= 0 and self.refs[p] > 1 else -1
        copies = {}
        for s, p in want.items():
            if p >= 0:
                sharing = [x for x, y in want.items() if y == p]
                copies[s] = not (len(sharing) == self.refs[p] and s == sharing[-1])
        free, refused, out = self.free(), 0, False
        for s, a in enumerate(add):
            if not a:
                continue
            n = self.lens[s]
            if s not in want:
                refused += 1
                continue
            need = up(n + a) - up(n) + copies.get(s, False)
            if out or need > len(free):
                refused += 1
                out = True
                continue
            if copies.get(s):
                p = free.pop(0)
                self.data[p] = self.data[want[s]]
                self.refs[want[s]] -= 1
                self.refs[p] = 1
                self.table[s][up(n) - 1] = p
            for j in range(up(n), up(n + a)):
                self.table[s][j] = p = free.pop(0)
                self.refs[p] = 1
            self.lens[s] += a
        return refused

    def fork(self, src):
        old = [r[:] for r in self.table]
        lens = self.lens[:]
        for r in old:
            for p in r:
                if p >= 0:
                    self.refs[p] -= 1
        for s, f in enumerate(src):
            ok = 0 <= f < len(old)
            self.table[s] = old[f][:] if ok else [-1] * self.m
            self.lens[s] = lens[f] if ok else 0
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] += 1

    def drop(self, s, j):
        p = self.table[s][j]
        if p >= 0:
            self.refs[p] -= 1
            self.table[s][j] = -1

    def end(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.table):
                for j in range(self.m):
                    self.drop(s, j)
                self.lens[s] = 0

    def trim(self, window, sinks):
        for s, n in enumerate(self.lens):
            for j in range(self.m):
                if j * self.page >= sinks and (j + 1) * self.page <= n + 1 - window:
                    self.drop(s, j)

    def compact(self):
        live = [p for p in range(self.n) if self.refs[p]]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for a, b in to.items():
            self.refs[b], self.refs[a], self.data[b] = self.refs[a], 0, self.data[a]
        self.table = [[to.get(p, p) for p in r] for r in self.table]

    def check(self, c):
        assert c.lens.tolist() == self.lens
        assert c.table.tolist() == self.table
        assert c.refs.tolist() == self.refs
        live = [p for p in range(self.n) if self.refs[p]]
        got = c.pool[:, live].float()
        want = torch.tensor([self.data[p] for p in live], dtype=torch.float32, device="cuda")
        layer = torch.arange(c.pool.shape[0], device="cuda").view(-1, 1, 1)
        assert torch.equal(got, (want.view(1, -1, 1) + 512 * layer).expand_as(got).to(c.pool.dtype).float())


def marked(cache):
    """Every page of layer l holds its number + 512 l (whole numbers below 2048 are exact in fp16)."""
    n_layers, n_pages, _ = cache.pool.shape
    cache.pool.copy_((torch.arange(n_pages, device="cuda").view(1, -1, 1) + 512 * torch.arange(n_layers, device="cuda").view(-1, 1, 1)).to(cache.pool.dtype))


@pytest.mark.parametrize("n_pages,n_seqs,max_pages,page,layers", [(40, 6, 9, 32, 2), (500, 33, 20, 64, 1), (7, 3, 4, 32, 3), (300, 100, 6, 32, 1),
                                                                  (1, 1, 1, 32, 1)])
def test_pages_follow_the_rules(n_pages, n_seqs, max_pages, page, layers):
    import random

    c = paged.PagedCache(n_pages, n_seqs, max_pages, page_size=page, num_kv_heads=1, head_dim=64, n_layers=layers, dtype=torch.float16)
    marked(c)
    m = Model(n_pages, n_seqs, max_pages, page)
    rng = random.Random(n_pages)
    for step in range(60):
        op = rng.choice(("extend", "extend", "extend", "fork", "fork", "free", "trim", "compact"))
        if op == "extend":
            most = rng.choice((1, 3, page, 3 * page, max_pages * page + 5))
            add = [rng.randint(0, most) if rng.random() < 0.7 else 0 for _ in range(n_seqs)]
            c.extend(ints(add))
            refused = m.extend(add)
            assert c.status() == (refused, len(m.free())), (step, add)
        elif op == "fork":
            src = [rng.choice((s, s, rng.randrange(n_seqs), rng.randrange(n_seqs), -1 if rng.random() < 0.1 else s)) for s in range(n_seqs)]
            c.fork(ints(src))
            m.fork(src)
        elif op == "free":
            seqs = [rng.randrange(-1, n_seqs + 1) for _ in range(rng.randint(0, max(1, n_seqs // 3)))]
            seqs += seqs[:1]
            c.free(ints(seqs))
            m.end(seqs)
        elif op == "trim":
            window, sinks = rng.choice((1, page, 2 * page + 1, 1 << 33)), rng.choice((0, 1, page, page + 1))
            c.trim(window, sinks)
            m.trim(window, sinks)
        else:
            c.compact()
            m.compact()
        m.check(c)


def test_pages_of_many_sequences():
    """The largest number of sequences, with more pages than one pass of the scan takes."""
    n, pages = 4096, 20000
    c = paged.PagedCache(pages, n, 5, page_size=32, num_kv_heads=1, head_dim=64, dtype=torch.float16)
    c.pool.zero_()
    m = Model(pages, n, 5, 32)
    for step in range(4):
        add = [(s * 37 + step * 11) % 60 for s in range(n)]
        c.extend(ints(add))
        m.extend(add)
        src = [(s * 5 + step) % n if s % 3 else s for s in range(n)]
        c.fork(ints(src))
        m.fork(src)
        assert c.lens.tolist() == m.lens and c.table.tolist() == m.table and c.refs.tolist() == m.refs
    c.free(ints(range(0, n, 2)))
    m.end(range(0, n, 2))
    c.compact()
    m.compact()
    assert c.lens.tolist() == m.lens and c.table.tolist() == m.table and c.refs.tolist() == m.refs


def test_pages_with_a_holder_outside_the_table_and_a_strided_table():
    words = dict(dtype=torch.int32, device="cuda")
    wide = torch.full((3, 9), 77, **words)
    c = paged.PagedCache.over(torch.zeros(2, 10, 2 * 32 * 64, dtype=torch.float16, device="cuda"), wide[:, 2:6], torch.zeros(3, **words),
                              page_size=32, num_kv_heads=1, head_dim=64, refs=torch.zeros(10, **words))
    c.reset()
    marked(c)
    c.extend(ints([40, 0, 0]))
    c.refs[1] += 1  # the second page is kept by someone
    c.extend(ints([1, 0, 0]))  # so its own is copied
    assert c.table.tolist()[0] == [0, 2, -1, -1] and c.refs.tolist()[:3] == [1, 1, 1] and (c.pool[0, 2] == 1).all()
    assert (wide[:, :2] == 77).all() and (wide[:, 6:] == 77).all()
    c.free(ints([0]))
    assert c.refs.tolist() == [0, 1] + [0] * 8 and c.status() == (0, 9)


# ---- together -------------------------------------------------------------------------------------

def test_serving_run_with_forks_a_window_and_trims():
    """Prompts appended and attended, samples forked, one token after another with old pages given back:
    every step against the sequences' own histories."""
    hq, hkv, d, page, layers, window, sinks = 8, 2, 64, 32, 2, 60, 3
    c = paged.PagedCache(60, 4, 12, page_size=page, num_kv_heads=hkv, head_dim=d, n_layers=layers)
    c.pool.fill_(float("nan"))
    turn = paged.Rope(d, scaling="yarn", factor=4.0, original_len=64)
    g = gen(11)
    past = [[(torch.zeros(0, hkv, d), torch.zeros(0, hkv, d)) for _ in range(layers)] for _ in range(4)]

    def step(rows):
        total = sum(rows)
        start = np.concatenate([[0], np.cumsum(rows)]).tolist()
        c.extend(ints(rows))
        assert c.status()[0] == 0
        for layer in range(layers):
            x = torch.randn(total, hq + 2 * hkv, d, generator=g, device="cuda")
            one = all(r == 1 for r in rows)
            q = paged.rope_append(c, layer, turn, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q_start=None if one else ints(start))
            if one:
                out = paged.attention(c, layer, q, window=window, sinks=sinks)
            else:
                out = paged.prompt_attention(c, layer, q, ints(start), window=window, sinks=sinks)
            for s in range(4):
                lo, hi = start[s], start[s + 1]
                k0, v0 = past[s][layer]
                at = torch.arange(len(k0), len(k0) + hi - lo, device="cuda")
                k = torch.cat((k0, turned(x[lo:hi, hq:hq + hkv], at, turn, False)[0].bfloat16().cpu().float()))
                v = torch.cat((v0, x[lo:hi, hq + hkv:].bfloat16().cpu().float()))
                past[s][layer] = (k, v)
                y = turned(x[lo:hi, :hq], at, turn, False)[0].cpu()
                for i in range(hi - lo):
                    t = int(at[i])
                    seen = torch.tensor([j for j in range(t + 1) if j > t - window or j < sinks])
                    for h in range(hq):
                        kk, vv = k[seen, h // 4].double(), v[seen, h // 4].double()
                        p = torch.softmax(kk @ y[i, h] / math.sqrt(d), 0)
                        # k is rounded to bf16 from angles a little apart: where one falls on the other side
                        # of a step a score moves by u(bf16) |q k| / sqrt(d) of one element (below 4 * 4)
                        tol = 2 * 2 * half_step(torch.bfloat16) * 16 / math.sqrt(d) * (p @ vv.abs())
                        assert ((out[lo + i, h].cpu().double() - p @ vv).abs() <= tol + 1e-5).all()
        c.trim(window, sinks)

    step([100, 1, 0, 37])
    c.fork(ints([0, 0, 3, 3]))
    past[:] = [[tuple(t.clone() for t in layer) for layer in past[s]] for s in (0, 0, 3, 3)]
    for i in range(40):
        step([1, 1, 1, 1])
        if i == 20:
            c.fork(ints([1, 1, 2, 0]))
            past[:] = [[tuple(t.clone() for t in layer) for layer in past[s]] for s in (1, 1, 2, 0)]
            c.compact()
    step([5, 0, 40, 1])


def test_a_captured_step_crosses_pages():
    """extend, append and attention of a decode step in one graph, replayed across page borders with eager
    work between, against the same steps run eagerly on a second cache."""
    hq, hkv, d, page = 4, 2, 64, 32

    def make():
        c = paged.PagedCache(40, 3, 8, page_size=page, num_kv_heads=hkv, head_dim=d)
        c.extend(ints([30, 64, 1]))
        c.pool.copy_(torch.randn(c.pool.shape, generator=gen(5), device="cuda"))
        c.fork(ints([0, 1, 0]))
        return c

    a, b = make(), make()
    turn = paged.Rope(d)
    x = torch.zeros(3, hq + 2 * hkv, d, device="cuda")
    one = ints([1, 1, 1])
    q, out = torch.empty(3, hq, d, device="cuda"), torch.empty(3, hq, d, device="cuda")
    space = a.attention_workspace(hq)

    def step(c, q, out):
        c.extend(one)
        paged.rope_append(c, 0, turn, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q)
        paged.attention(c, 0, q, out=out, workspace=space)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(a, q, out)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(40):
        x.copy_(torch.randn(x.shape, generator=gen(100 + i), device="cuda"))
        graph.replay()
        q2, out2 = torch.empty_like(q), torch.empty_like(out)
        step(b, q2, out2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(a.table, b.table) and torch.equal(a.lens, b.lens) and torch.equal(a.refs, b.refs)
    assert a.lens.tolist() == [70, 104, 70]


def test_captured_page_operations_and_prompts():
    """A serving turn (free, prompts, fork, trim, compact) in one graph, replayed with other inputs and eager work
    between, against the same turns run eagerly on a second cache."""
    hq, hkv, d, page, n, window = 4, 2, 64, 32, 4, 50

    def make():
        # 40 pages of 32 positions: parts of 512 at least are split off, so that the workspace is used
        c = paged.PagedCache(120, n, 40, page_size=page, num_kv_heads=hkv, head_dim=d, n_layers=2)
        c.extend(ints([700, 5, 64, 200]))
        c.pool.copy_(torch.randn(c.pool.shape, generator=gen(5), device="cuda"))
        return c

    a, b = make(), make()
    turn = paged.Rope(d)
    x = torch.zeros(20, hq + 2 * hkv, d, device="cuda")
    rows, start, src, gone = ints([5, 0, 9, 1]), ints([0, 5, 5, 14, 15]), ints([0, 1, 2, 3]), ints([-1, -1])
    q, out = torch.zeros(20, hq, d, device="cuda"), torch.zeros(20, hq, d, device="cuda")
    space = a.prompt_workspace(hq, total_rows=20)
    assert space is not None

    def step(c, q, out):
        c.free(gone)
        c.fork(src)
        c.extend(rows)
        for layer in range(2):
            paged.rope_append(c, layer, turn, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q, q_start=start)
            paged.prompt_attention(c, layer, q, start, sinks=4, window=window * layer, out=out, workspace=space)
        c.trim(700)
        c.compact()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(a, q, out)
    torch.cuda.current_stream().wait_stream(side)
    q2, out2 = torch.zeros_like(q), torch.zeros_like(out)
    for i, (s, g) in enumerate([([0, 1, 2, 3], [-1, -1]), ([0, 0, 2, 2], [-1, -1]), ([0, 1, 0, 3], [1, 1]), ([3, 1, 2, -1], [-1, 2]),
                                ([0, 2, 2, 0], [7, -1]), ([0, 1, 2, 3], [0, 2])]):
        x.copy_(torch.randn(x.shape, generator=gen(100 + i), device="cuda"))
        src.copy_(ints(s))
        gone.copy_(ints(g))
        graph.replay()
        torch.cuda.synchronize()
        step(b, q2, out2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(q, q2)
        for u, w in ((a.table, b.table), (a.lens, b.lens), (a.refs, b.refs), (a.pool, b.pool)):
            assert torch.equal(u, w)
        assert a.status() == b.status()


def test_a_prompt_workspace_serves_fewer_rows():
    f = Filled([2100], 2, 64, 64, "bf16")
    space = f.cache.prompt_workspace(8, total_rows=900)
    for n in (900, 300, 33, 1):
        q, start = queries(n, 8, 2, 64, "bf16"), ints([0, n])
        got = paged.prompt_attention(f.cache, 0, q, start, workspace=space)
        assert torch.equal(got, paged.prompt_attention(f.cache, 0, q, start))


def test_calls_run_on_the_current_stream():
    f = Filled([500, 90], 2, 64, 32, "bf16")
    x = torch.zeros(2, 4, 64, device="cuda")
    want_x = torch.randn(2, 4, 64, generator=gen(1), device="cuda")
    busy = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            busy = busy @ busy * 1e-4
        x.copy_(want_x)  # after the products, so a call on another stream would read zeros
        out = paged.attention(f.cache, 0, x)
    side.synchronize()
    for s in range(2):
        f.check(want_x[s:s + 1], out[s:s + 1], s, s, 0, 0, False)


def test_calls_repeat_bit_for_bit():
    f = Filled([3000, 700, 33], 2, 128, 64, "bf16")
    x = queries(3, 8, 2, 128, "f32")
    first = paged.attention(f.cache, 0, x)
    y = queries(60, 8, 2, 128, "bf16")
    start = ints([0, 20, 40, 60])
    again = paged.prompt_attention(f.cache, 0, y, start)
    for _ in range(3):
        assert torch.equal(paged.attention(f.cache, 0, x), first)
        assert torch.equal(paged.prompt_attention(f.cache, 0, y, start), again)


def test_python_calls_refuse_what_does_not_fit():
    f = Filled([64, 3], 2, 64, 32, "bf16")
    x = torch.zeros(2, 4, 64, device="cuda")
    c = f.cache
    for call in (lambda: paged.attention(c, 0, x[:1]), lambda: paged.attention(c, 0, x.double()), lambda: paged.attention(c, 0, x.cpu()),
                 lambda: paged.attention(c, 0, torch.zeros(2, 4, 128, device="cuda")), lambda: paged.attention(c, 0, x[..., ::2]),
                 lambda: paged.attention(c, 0, x, window=-1), lambda: paged.attention(c, -1, x),
                 lambda: paged.attention(c, 0, x, out=torch.zeros(2, 2, 64, device="cuda")),
                 lambda: paged.prompt_attention(c, 0, x, ints([0, 1])), lambda: paged.prompt_attention(c, 0, x, torch.zeros(3, device="cuda")),
                 lambda: paged.rope(paged.Rope(64), x, ints([0])), lambda: paged.rope(paged.Rope(64), x, ints([0, 1]), out=x.half()),
                 lambda: paged.rope_append(c, 0, None, x, x, x), lambda: paged.rope_append(c, 0, None, x, x[:, :2], x[:1, :2])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: paged.attention(c, 1, x), lambda: paged.attention(c, 0, x[:, :3]), lambda: paged.rope(paged.Rope(128), x, ints([0, 0])),
                 lambda: paged.rope_append(c, 0, paged.Rope(128), None, x[:, :2], x[:, 2:]), lambda: c.extend(ints([1, 1])), lambda: c.compact()):
        with pytest.raises(RuntimeError):
            call()
