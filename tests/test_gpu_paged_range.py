"""The paged cache's operators at the sizes that only long or many rows reach, and to the precision that they state,
against plain float64 computations of the same inputs (tolerances: test_gpu_paged.py's, with the weights' rounding given).
"""
import math

import pytest
import torch

from velox_amd import paged
from test_gpu_paged import SLOT, T, Filled, close_turn, gen, half_step, ints, queries, turned
from test_gpu_paged import test_append as check_append

pytestmark = pytest.mark.gpu


def near(f, q, out, seq, weights, window=0, sinks=0, scale=None, small=0.0):
    """Rows q of sequence seq, the last one its newest position. weights: how far a softmax weight may be off, relative
    to itself; small: and relative to the row's largest."""
    n, rows, d = f.lens[seq], q.shape[0], f.d
    scale = scale or 1 / math.sqrt(d)
    t = torch.arange(n - rows, n, device="cuda").unsqueeze(1)
    j = torch.arange(n, device="cuda").unsqueeze(0)
    hidden = j > t
    if window:
        hidden |= (j <= t - window) & (j >= sinks)
    u, ou = half_step(torch.float32), half_step(out.dtype)
    for h in range(q.shape[1]):
        g = h // (q.shape[1] // f.hkv)
        x, k, v = q[:, h].double(), f.k[seq][:, g].double(), f.v[seq][:, g].double()
        big = (x.abs() @ k.abs().T * abs(scale)).masked_fill_(hidden, 0.0).amax(1, keepdim=True)
        p = torch.softmax((x @ k.T * scale).masked_fill_(hidden, -math.inf), 1)
        o, a = p @ v, p @ v.abs()
        c = 2 * ((d + 8) * u * big + 2 ** -22 * big) + weights + (n + 64) * u
        tol = ou * o.abs() * (1 + c) + (c * a + small * n * v.abs().amax()) * (1 + ou) + 1e-30
        bad = ~((out[:, h].double() - o).abs() <= tol)
        assert not bad.any(), (seq, h, int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 4)])
def test_weights_are_held_in_two_terms(t, d, window, sinks):
    """q of the cache's type, an fp32 output: two terms leave u^2 of a weight (of fp16 weights, times 2^7 against a
    maximum that is at most 2^8 too low, no less than 2^-25 of that), one would leave u."""
    lens, rows = [40, 33, 2, 700, 6000], [40, 33, 2, 200, 5]
    start = [sum(rows[:i]) for i in range(len(rows) + 1)]
    f = Filled(lens, 2, d, 32, t)
    x = queries(start[-1], 6, 2, d, t)
    weights, small = half_step(T[t]) ** 2, 2.0 ** -32 if t == "f16" else 0.0
    out = torch.empty(start[-1], 6, d, device="cuda")
    paged.prompt_attention(f.cache, 0, x, ints(start), window=window, sinks=sinks, out=out)
    last = ints(start[1:]).long() - 1
    one = paged.attention(f.cache, 0, x[last], window=window, sinks=sinks, out=torch.empty(len(lens), 6, d, device="cuda"))
    for s in range(len(lens)):
        near(f, x[start[s]:start[s + 1]], out[start[s]:start[s + 1]], s, weights, window, sinks, small=small)
        near(f, x[last[s]:last[s] + 1], one[s:s + 1], s, weights, window, sinks, small=small)


def test_calls_refuse_tensors_that_require_a_gradient():
    f = Filled([64, 3], 2, 64, 32, "bf16")
    c, turn = f.cache, paged.Rope(64)
    x = torch.randn(2, 4, 64, device="cuda")
    g = x.clone().requires_grad_()
    calls = [lambda g: paged.attention(c, 0, g), lambda g: paged.attention(c, 0, x, out=g), lambda g: paged.prompt_attention(c, 0, g, ints([0, 1, 2])),
             lambda g: paged.rope(turn, g, ints([0, 1])), lambda g: paged.rope_append(c, 0, turn, g, x[:, :2], x[:, 2:]),
             lambda g: paged.rope_append(c, 0, turn, x, g[:, :2], x[:, 2:]), lambda g: paged.rope_append(c, 0, turn, x, x[:, :2], g[:, 2:])]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(g)
    pool = torch.zeros_like(f.pool).requires_grad_()
    over = lambda: paged.PagedCache.over(pool, f.table, f.cache.lens, page_size=32, num_kv_heads=2, head_dim=64)  # noqa: E731
    with pytest.raises(ValueError, match="gradient"):
        over()
    with torch.no_grad():
        over()
        assert torch.equal(paged.rope(turn, g, ints([0, 1])), paged.rope(turn, x, ints([0, 1])))
        for call in calls:
            call(g)


@pytest.mark.parametrize("hq,hkv,d,t", [(8, 2, 64, "f32"), (16, 8, 128, "bf16")])
def test_short_rows_of_many_sequences(hq, hkv, d, t):
    """The bound on a sequence's rows decides the splits and nothing else, also where it is too low."""
    lens, rows = [600 + 37 * i for i in range(40)], [2 + i * 5 % 7 for i in range(40)]
    start = [sum(rows[:i]) for i in range(41)]
    f = Filled(lens, hkv, d, 64, "bf16")
    x = queries(start[-1], hq, hkv, d, t)
    for max_rows in (0, 8, 1):
        space = f.cache.prompt_workspace(hq, total_rows=start[-1], max_rows=max_rows, max_len=lens[-1])
        out = paged.prompt_attention(f.cache, 0, x, ints(start), max_rows=max_rows, max_len=lens[-1], workspace=space)
        for s in range(40):
            near(f, x[start[s]:start[s + 1]], out[start[s]:start[s + 1]], s, 2 ** -16 if t == "bf16" else 2 ** -20)


def test_calls_refuse_numbers_past_32_bits():
    f = Filled([64, 3], 2, 64, 32, "bf16")
    c, x, wrap = f.cache, torch.randn(2, 4, 64, device="cuda"), 1 << 32
    for call in (lambda: paged.attention(c, wrap, x), lambda: paged.attention(c, 0, x, max_len=wrap), lambda: c.attention_workspace(wrap + 4),
                 lambda: c.attention_workspace(4, max_len=wrap + 1), lambda: paged.prompt_attention(c, wrap, x, ints([0, 1, 2])),
                 lambda: paged.prompt_attention(c, 0, x, ints([0, 1, 2]), max_rows=wrap + 1), lambda: c.prompt_workspace(4, total_rows=wrap + 2),
                 lambda: c.prompt_workspace(4, total_rows=-1), lambda: paged.prompt_attention(c, 0, x, ints([0, 1, 2]), max_len=wrap),
                 lambda: paged.rope_append(c, wrap, None, x, x[:, :2], x[:, 2:])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("q,kv", [("f32", "f16"), ("bf16", "f16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("amp,scale", [(1e-30, 1e-20), (1.0, 1e-43), (1e-30, -1e-12)])
def test_scales_next_to_nothing(q, kv, amp, scale):
    """Scores that vanish leave the mean of what a row sees."""
    f = Filled([300, 70], 2, 64, 32, kv)
    x = (queries(120, 4, 2, 64, "f32") * amp).to(T[q])
    out = torch.empty(120, 4, 64, device="cuda")
    paged.prompt_attention(f.cache, 0, x, ints([0, 70, 120]), scale=scale, window=100, sinks=3, out=out)
    one = paged.attention(f.cache, 0, x[:2], scale=scale, window=100, sinks=3, out=torch.empty(2, 4, 64, device="cuda"))
    weights = half_step(T[kv]) ** 2 + 2 ** -20
    for s, (lo, hi) in enumerate(((0, 70), (70, 120))):
        near(f, x[lo:hi], out[lo:hi], s, weights, 100, 3, scale=scale, small=2.0 ** -32)
        near(f, x[s:s + 1], one[s:s + 1], s, weights, 100, 3, scale=scale, small=2.0 ** -32)


@pytest.mark.parametrize("hq,hkv,d,q,kv", [(32, 8, 128, "bf16", "bf16"), (16, 8, 128, "f32", "f16"), (16, 8, 128, "f32", "bf16"), (24, 8, 64, "f16", "f16"),
                                           (16, 8, 64, "f32", "bf16")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 70)])
def test_long_prompt_behind_a_long_context(hq, hkv, d, q, kv, window, sinks):
    """Workgroups that walk 2500 to 4600 positions whole: their pages are looked up several times."""
    n, rows = 4637, 2101
    f = Filled([n], hkv, d, 64, kv)
    assert f.cache.prompt_workspace(hq, total_rows=rows) is not None and -(-rows * (hq // hkv) // 128) * hkv >= 256  # not split
    x = queries(rows, hq, hkv, d, q)
    near(f, x, paged.prompt_attention(f.cache, 0, x, ints([0, rows]), window=window, sinks=sinks), 0,
         half_step(T[kv]) ** 2 if q == kv else 2 ** -20, window, sinks, small=2.0 ** -32)


@pytest.mark.parametrize("q,kv", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,n,rows,where,window,sinks", [(32, 8, 4637, 2101, 4600, 0, 0), (32, 8, 4637, 2101, 3000, 1500, 3), (32, 8, 4637, 2101, 5, 3000, 9),
                                                              (2, 1, 1700, 40, 1690, 0, 0), (2, 1, 9000, 90, 3, 4000, 5)],
                         ids=["late", "window", "sink", "split", "split-sink"])
def test_infinities_in_long_walks_and_splits(d, q, kv, hq, hkv, n, rows, where, window, sinks):
    """What is no number in V reaches the rows that see its position, far along a walk and in one of several splits."""
    f = Filled([n], hkv, d, 64, kv)
    x = queries(rows, hq, hkv, d, q)
    space = f.cache.prompt_workspace(hq, total_rows=rows)
    assert space is not None  # (of 2101 rows: for fewer)
    t = torch.arange(n - rows, n, device="cuda")
    sees = (t >= where) & ((t < where + window) | (where < sinks) if window else True)
    assert sees.any() and (window or not sees.all())
    h, e, r = hkv - 1, d - 3, where % 64
    cell = f.pool[0, int(f.table[0, where // 64])][hkv * 64 * d:].view(hkv, 2, d, 32)
    g = hq // hkv
    for value in (math.nan, math.inf, -math.inf):
        cell[h, r // 32, e, int(SLOT[r % 32])] = value
        out = paged.prompt_attention(f.cache, 0, x, ints([0, rows]), window=window, sinks=sinks, workspace=space)
        assert torch.equal(torch.isfinite(out[:, h * g:, e]), ~sees.view(-1, 1).expand(rows, g))
        out[:, h * g:, e] = 0
        assert torch.isfinite(out).all()
    f.v[0][:, h, e] = 0  # that dimension is looked at above
    near(f, x, out, 0, half_step(T[kv]) ** 2 if q == kv else 2 ** -20, window, sinks, small=2.0 ** -32)


@pytest.mark.parametrize("q", ["f32", "bf16"])
def test_token_attention_past_the_caches(q):
    """K and V of more than 256 MiB: loads that leave nothing in the caches."""
    f = Filled([70011], 8, 128, 256, "bf16")
    assert f.table.shape[1] * 256 * 8 * 128 * 4 > 256 << 20
    x = queries(1, 16, 8, 128, q)
    out = torch.empty(1, 16, 128, device="cuda")
    near(f, x, paged.attention(f.cache, 0, x, out=out), 0, 2 ** -16 if q == "bf16" else 2 ** -20)
    near(f, x, paged.attention(f.cache, 0, x, window=69000, sinks=33, out=out), 0, 2 ** -16 if q == "bf16" else 2 ** -20, 69000, 33)


@pytest.mark.parametrize("rows,heads", [(2049, 70), (4001, 70), (4001, 3)])
@pytest.mark.parametrize("layout,rot", [("half", 128), ("interleaved", 128), ("half", 64), ("interleaved", 64)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rope_of_many_rows(rows, heads, layout, rot, dtype):
    """Several rows a workgroup and fewer in the last one, more heads than are requested at once, and more bytes than the caches."""
    x = torch.randn(rows, heads, 128, generator=gen(rows), device="cuda").to(T[dtype])
    at = torch.randint(0, 2 ** 31 - 1, (rows,), generator=gen(5), device="cuda", dtype=torch.int32)
    turn = paged.Rope(rot, theta=5e5, layout=layout)
    want, size = turned(x, at, turn, layout == "interleaved")
    got = paged.rope(turn, x, at)
    close_turn(got, want, size, T[dtype])
    paged.rope(turn, x, at, out=x)
    assert torch.equal(x, got)


@pytest.mark.parametrize("hq,hkv,q,kv,rows,layout", [(32, 8, "bf16", "bf16", [2700, 33, 70], "half"), (64, 8, "f32", "bf16", [800, 1, 70], "half"),
                                                     (64, 8, "f16", "f16", [1600, 33, 70], "interleaved"), (32, 8, "f32", "f16", [1300, 1, 75], "interleaved"),
                                                     (64, 8, "bf16", "bf16", [70, 33, 1], "half"), (32, 8, "f32", "bf16", [70, 33, 1], "half")])
def test_append_of_many_heads_and_bytes(hq, hkv, q, kv, rows, layout):
    """More heads than a thread requests at once, and rows past the caches; blocks of fewer than 32 rows among them."""
    if rows[0] > 70:
        assert (sum(rows) + 3) * (hq + 2 * hkv) * 128 * T[q].itemsize > 32 << 20
    check_append(hq, hkv, 128, 64, 128, layout, q, kv, rows, [17, 5, 64])


def test_a_captured_step_of_split_token_attention():
    """A decode step whose attention is split and joined, in a graph that is replayed with eager steps on a second cache
    between, against those."""
    hq, hkv, d = 4, 2, 64

    def make():
        c = paged.PagedCache(160, 3, 64, page_size=32, num_kv_heads=hkv, head_dim=d)
        c.extend(ints([1500, 2, 700]))
        c.pool.copy_(torch.randn(c.pool.shape, generator=gen(5), device="cuda"))
        return c

    a, b = make(), make()
    turn, one = paged.Rope(d), ints([1, 1, 1])
    x = torch.zeros(3, hq + 2 * hkv, d, device="cuda")
    sets = [(torch.empty(3, hq, d, device="cuda"), torch.empty(3, hq, d, device="cuda"), a.attention_workspace(hq)) for _ in range(2)]
    assert sets[0][2] is not None

    def step(c, q, out, space):
        c.extend(one)
        paged.rope_append(c, 0, turn, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q)
        paged.attention(c, 0, q, out=out, workspace=space)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(a, *sets[0])
    torch.cuda.current_stream().wait_stream(side)
    for i in range(40):
        x.copy_(torch.randn(x.shape, generator=gen(100 + i), device="cuda"))
        sets[0][2].fill_(255 if i % 2 else 0)  # nothing of an earlier call is needed: all bits set are NaN
        graph.replay()
        step(b, *sets[1])
        torch.cuda.synchronize()
        assert torch.isfinite(sets[0][1]).all() and torch.equal(sets[0][1], sets[1][1]) and torch.equal(a.lens, b.lens)


@pytest.mark.parametrize("d,rot", [(2048, 256), (1040, 256), (4099, 34)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rope_of_wide_heads(d, rot, layout, dtype):
    """Heads of more units than a workgroup has threads."""
    x = torch.randn(7, 3, d, generator=gen(d), device="cuda").to(T[dtype])
    at, turn = ints([0, 1, 5, 100, 4096, 99999, 2 ** 31 - 1]), paged.Rope(rot, theta=5e5, layout=layout)
    want, size = turned(x, at, turn, layout == "interleaved")
    got = paged.rope(turn, x, at)
    close_turn(got, want, size, T[dtype])
    assert torch.equal(paged.rope(turn, x, at, out=x), got)


@pytest.mark.parametrize("q,k,v,kv", [("f32", "bf16", "bf16", "bf16"), ("bf16", "f32", "f16", "f16"), ("f16", "f16", "f32", "bf16")])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_of_mixed_types_at_any_address(q, k, v, kv, odd, ragged):
    """Each of q, k and v by itself against the same rows in one type, whose roundings come last."""
    n, hq, hkv, d = 6, 5, 2, 64
    rows = [3, 0, 40, 1, 7, 2] if ragged else [1] * 5  # one row each of the first five of six sequences
    start = [sum(rows[:i]) for i in range(len(rows) + 1)]
    f = Filled([70, 33, 90, 1, 64, 128], hkv, d, 32, kv)
    turn, total = paged.Rope(d, layout="interleaved" if odd else "half"), start[-1]

    def made(heads, dtype, seed):
        room = torch.empty(total * heads * d + 1, dtype=T[dtype], device="cuda")
        x = room[odd:odd + total * heads * d].view(total, heads, d)
        return x.copy_(torch.randn(total, heads, d, generator=gen(seed), device="cuda"))

    xq, xk, xv = made(hq, q, 1), made(hkv, k, 2), made(hkv, v, 3)
    at = ints(start) if ragged else None
    pool = f.pool.clone()
    out = paged.rope_append(f.cache, 0, turn, xq, xk, xv, q_start=at)
    got = f.pool.clone()
    f.pool.copy_(pool)
    wide = paged.rope_append(f.cache, 0, turn, xq.float(), xk.float(), xv.float(), q_start=at)
    assert out.dtype == T[q] and torch.equal(out, wide.to(T[q])) and torch.equal(got.view(torch.int16), f.pool.view(torch.int16))
    assert not torch.equal(f.pool.view(torch.int16), pool.view(torch.int16))


@pytest.mark.parametrize("q,kv", [("bf16", "bf16"), ("f32", "f16")])
def test_prompts_in_place_of_split_rows_and_of_many_heads(q, kv):
    weights = half_step(T[kv]) ** 2 if q == kv else 2 ** -20
    for hq, hkv, n, rows in ((4, 2, 3000, 50), (300, 1, 90, 40), (300, 1, 2500, 3)):
        f = Filled([n], hkv, 64, 32, kv)
        x = queries(rows, hq, hkv, 64, q)
        y = x.clone()
        assert (f.cache.prompt_workspace(hq, total_rows=rows) is None) == (n < 1000)
        assert paged.prompt_attention(f.cache, 0, y, ints([0, rows]), out=y) is y
        near(f, x, y, 0, weights, small=2.0 ** -32)
        one = x[-1:].clone()
        paged.attention(f.cache, 0, one, out=one)
        near(f, x[-1:], one, 0, weights, small=2.0 ** -32)


def test_layers_of_a_larger_pool():
    """A cache over every second layer and the first pages of a pool, in the rows of a wider table."""
    hkv, d, page = 2, 64, 32
    f = Filled([100, 40], hkv, d, page, "bf16")
    n_pages = f.pool.shape[1]
    pool = torch.full((5, n_pages + 3, f.pool.shape[2]), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool[2, :n_pages] = f.pool[0]
    table = torch.full((2, 11), -1, dtype=torch.int32, device="cuda")
    table[:, 3:3 + f.table.shape[1]] = f.table
    c = paged.PagedCache.over(pool[::2, :n_pages], table[:, 3:8], f.cache.lens, page_size=page, num_kv_heads=hkv, head_dim=d)
    x = queries(30, 4, hkv, d, "f32")
    for out, rows in ((paged.prompt_attention(c, 1, x, ints([0, 20, 30])), ((0, 20), (20, 30))), (paged.attention(c, 1, x[:2]), ((0, 1), (1, 2)))):
        for s, (lo, hi) in enumerate(rows):
            near(f, x[lo:hi], out[lo:hi], s, 2 ** -20)
    before = pool.clone()
    paged.rope_append(c, 2, None, None, x[:2, :2], x[:2, 2:])
    same = torch.ones(5, n_pages + 3, dtype=torch.bool, device="cuda")
    same[4, table[:, 3:8].max(1).values.new_tensor([int(f.table[0, 3]), int(f.table[1, 1])]).long()] = False
    assert torch.equal(pool[same].view(torch.int16), before[same].view(torch.int16)) and not torch.equal(pool[4].view(torch.int16), before[4].view(torch.int16))


def test_in_place_rows_lie_as_q_does():
    f = Filled([40, 7], 2, 64, 32, "bf16")
    x = queries(2, 4, 2, 64, "f32")
    flat = x.as_strided((2, 4, 64), (256, 64, 1))
    for call in (lambda: paged.attention(f.cache, 0, x, out=flat), lambda: paged.prompt_attention(f.cache, 0, x, ints([0, 1, 2]), out=flat)):
        with pytest.raises(RuntimeError):
            call()
    f = Filled([40], 2, 64, 32, "bf16")
    for run in (lambda a, o: paged.attention(f.cache, 0, a, out=o), lambda a, o: paged.prompt_attention(f.cache, 0, a, ints([0, 1]), out=o)):
        y = x[:1].clone()
        run(y, y.as_strided((1, 4, 64), (1000, 64, 1)))  # of one row there is no stride
        near(f, x[:1], y, 0, 2 ** -20)
