"""The 8-bit integer products on the GPU against float64.

Tolerances are derived from the roundings, u = 2^-24 half a step of fp32, u(t) = finfo(t).eps / 2 that of an output type. Codes
have to be equal: the rule rounds exact quotients. A product is an exact sum S in whole numbers: fl(S), times the weight
row's scale, times the row's: three roundings, 3 u |y|; a bias and a residual one each of what they give. silu(g) up: g
and up off by 3 u each; the exponential by 2^-22 of itself besides what its argument's error makes of it, a sum, a
quotient and a product: |h| (3 + 8) u and |up| |g| 1.1 * 3 u (the largest slope of silu is below 1.1).
"""
import math

import pytest
import torch

from velox_amd import _lib as L
from velox_amd import int8

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    """Half of the type's smallest step."""
    return {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[t]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def held(x):
    """(codes, scales) in float64 of rows x: the definition."""
    x = x.double()
    top = x.abs().amax(1)
    s = (top / 127).float().double()
    bad = ~torch.isfinite(top)
    none = s < 2.0 ** -126
    c = torch.where((none | bad).unsqueeze(1), 0.0, torch.round(x / s.unsqueeze(1)))
    return c, torch.where(bad, math.nan, torch.where(none, 0.0, s))


def weights(n, k, seed, count=0, lowest=-127):
    shape = (count, n, k) if count else (n, k)
    w = torch.randint(lowest, 128, shape, generator=gen(seed), device="cuda", dtype=torch.int32).to(torch.int8)
    return w, (0.2 + torch.rand(shape[:-1], generator=gen(seed + 1), device="cuda")) / (70 * math.sqrt(k))


def rows(n, k, dtype, seed, odd=False):
    """Rows of unequal size, next to each other or (odd) as slices of wider ones at any alignment."""
    x = torch.randn(n, k + (7 if odd else 0), generator=gen(seed), device="cuda") * torch.logspace(-2, 2, n, device="cuda").unsqueeze(1)
    x = x.to(T[dtype])
    return x[:, 3:3 + k] if odd else x


def check(x, w, sw, got, paired=False, bias=None, residual=None):
    c, s = held(x)
    y = (c @ w.double().T) * sw.double() * s.unsqueeze(1)
    if paired:
        half = y.shape[1] // 2
        g, up = y[:, :half], y[:, half:]
        want = g * torch.sigmoid(g) * up
        tol = want.abs() * 11 * U + 3.3 * U * up.abs() * g.abs()
    else:
        want, tol = y, 3 * U * y.abs()
        for t in (bias, residual):
            if t is not None:
                want = want + t.double()
                tol = tol + U * want.abs()
    tol = (tol * (1 + 16 * U) + 1e-36) * (1 + half_step(got.dtype)) + half_step(got.dtype) * want.abs() + least(got.dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    over = want.abs() > torch.finfo(got.dtype).max  # (rounds to infinity)
    bad = ~((got.double() - want).abs() <= tol) & ~torch.isnan(want) & ~over
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (got.double() - want).abs().nan_to_num().max().item(), bad.sum().item())
    assert torch.equal(got[over].double(), torch.sign(want[over]) * math.inf)


@pytest.mark.parametrize("dtype", T)
@pytest.mark.parametrize("n,k", [(1, 1), (2, 127), (3, 128), (5, 129), (70, 1000), (9, 4096), (4, 30001), (1, 131072), (300, 64), (17, 2048)])
def test_quantize(dtype, n, k):
    for odd in (False, True):
        x = rows(n, k, dtype, n * 1000 + k, odd)
        q = int8.quantize(x)
        c, s = held(x)
        assert torch.equal(q.scales.double(), s)
        assert torch.equal(q.codes[:, :k].double(), c)
        assert not q.codes[:, k:].any()


def test_quantize_ties_and_borders():
    """Quotients of exactly a half, and next to it by one step of x either way; the largest and least numbers."""
    s = torch.tensor([1.0, 0.7, 3.3e-20, 1.1e30, 2.0 ** -120], device="cuda")
    half = torch.arange(-126, 127, device="cuda") + 0.5
    for step in (-1, 0, 1):
        x = (half.double().unsqueeze(0) * s.double().unsqueeze(1)).float()
        x = torch.nextafter(x, torch.full_like(x, math.inf if step > 0 else -math.inf)) if step else x
        x = torch.cat((x, (127 * s).unsqueeze(1)), 1)
        q = int8.quantize(x)
        c, want = held(x)
        assert torch.equal(q.scales.double(), want) and torch.equal(q.codes[:, :x.shape[1]].double(), c)
    tiny = torch.tensor([[0.0, -0.0], [1e-45, -1e-45], [2.0 ** -119, 0.0], [127 * 2.0 ** -126, 2.0 ** -126], [3.4028234e38, -1.0]], device="cuda")
    q = int8.quantize(tiny)
    c, want = held(tiny)
    assert torch.equal(q.scales.double(), want) and torch.equal(q.codes[:, :2].double(), c)
    assert want[:2].eq(0).all() and want[2:].gt(0).all()  # (2^-119 / 127 is above 2^-126)
    assert int8.quantize(torch.full((1, 9), 2.0 ** -120, device="cuda")).scales.item() == 0


@pytest.mark.parametrize("dtype", T)
def test_what_is_no_number_stays_in_its_row(dtype):
    x = rows(6, 300, dtype, 5)
    x[1, 299], x[3, 0], x[4, 17] = math.nan, math.inf, -math.inf
    q = int8.quantize(x)
    assert torch.isnan(q.scales).tolist() == [False, True, False, True, True, False] and not q.codes[1].any()
    w, sw = weights(40, 300, 1)
    for m in (int8.Int8Matrix(w, sw), int8.Int8Matrix(w, sw, paired=True)):
        y = int8.product(x, m)
        check(x, w, sw, y, paired=m.paired)
        assert torch.isnan(y).all(1).tolist() == [False, True, False, True, True, False]


SHAPES = [(1, 16, 128), (1, 1, 1), (1, 4096, 4096), (2, 960, 576), (3, 47, 130), (15, 100, 1000), (16, 33, 64), (17, 2050, 257), (31, 512, 3584), (32, 1000, 2048),
          (33, 130, 4000), (48, 258, 640), (64, 64, 64), (65, 300, 300), (100, 1030, 511), (128, 128, 128), (129, 257, 513), (255, 500, 700),
          (257, 1000, 1408), (300, 3, 5000), (513, 777, 129), (1000, 2000, 384), (1037, 960, 576)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k):
    for i, dtype in enumerate(T):
        x = rows(m, k, dtype, m + n + k + i, odd=i == 1)
        w, sw = weights(n, k, 3 + i, lowest=-128)
        bias = torch.randn(n, generator=gen(9), device="cuda") if i != 1 else None
        res = rows(m, n, dtype, 10, odd=True) if i else None
        got = int8.product(x, int8.Int8Matrix(w, sw), bias=bias, residual=res)
        assert got.dtype == x.dtype and got.shape == (m, n)
        check(x, w, sw, got, bias=bias, residual=res)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_swiglu(m, n, k):
    for i, dtype in enumerate(T):
        x = rows(m, k, dtype, m + n + k + i, odd=i == 2)
        w, sw = weights(2 * n, k, 3 + i)
        check(x, w, sw, int8.product(x, int8.Int8Matrix(w, sw, paired=True)), paired=True)


def test_product_at_the_largest_sums():
    """Every product 127 * 127 or 127 * -128 over the longest rows: the sum needs 31 bits."""
    k = 131072
    x = torch.ones(3, k, device="cuda")
    w = torch.full((20, k), -128, dtype=torch.int8, device="cuda")
    w[7:] = 127
    sw = torch.ones(20, device="cuda")
    check(x, w, sw, int8.product(x, int8.Int8Matrix(w, sw)))
    x = torch.ones(300, k, device="cuda")
    check(x, w, sw, int8.product(x, int8.Int8Matrix(w, sw)))


@pytest.mark.parametrize("m", [1, 3, 17, 40, 100, 300])
def test_product_of_the_most_outputs(m):
    """2^20 weight rows; paired, 2^19 gate and up rows."""
    n, k = 1 << 20, 72
    x = rows(m, k, "bf16", m)
    w, sw = weights(n, k, 3)
    check(x, w, sw, int8.product(x, int8.Int8Matrix(w, sw)))
    check(x, w, sw, int8.product(x, int8.Int8Matrix(w, sw, paired=True)), paired=True)


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_product_of_rows_already_in_8_bits_any_output_type_and_place(m):
    k, n = 500, 70
    x = rows(m, k, "bf16", 2)
    q = int8.quantize(x)
    for i, dtype in enumerate(T):
        w, sw = weights(n, k, 20 + i)
        mat = int8.Int8Matrix(w, sw)
        room = torch.full((m, n + 9), 5.0, device="cuda").to(T[dtype])
        out = room[:, 5:5 + n]
        assert int8.product(q, mat, out=out) is out
        check(x, w, sw, out)
        assert (room[:, :5] == 5).all() and (room[:, 5 + n:] == 5).all()
        assert torch.equal(int8.product(q, mat, dtype=T[dtype]), out) and torch.equal(int8.product(x, mat, dtype=T[dtype]), out)
        # the residual's own place
        before = out.clone()
        res = int8.product(q, mat, residual=out, out=out)
        check(x, w, sw, res, residual=before)


@pytest.mark.parametrize("m", [1, 2, 3, 20, 40, 100, 700])
def test_product_in_the_rows_place(m):
    """out begins where x does: every row is in 8 bits before the first output is written."""
    for i, dtype in enumerate(T):
        w, sw = weights(256, 256, 5 + i)
        mat = int8.Int8Matrix(w, sw)
        x = rows(m, 256, dtype, 4)
        before = x.clone()
        apart = int8.product(x, mat, residual=x)
        assert int8.product(x, mat, residual=x, out=x) is x
        assert torch.equal(x, apart)
        check(before, w, sw, x, residual=before)


@pytest.mark.parametrize("m,step", [(2, 2 ** 31 + 8), (20, 2 ** 28 + 8), (100, 2 ** 26 + 8), (300, 2 ** 24 + 3)])
def test_rows_that_lie_past_32_bits(m, step):
    n, k = 80, 144
    x, res, room = (torch.empty((m - 1) * step + 160, device="cuda", dtype=torch.float16) for _ in range(3))
    xr, rr, out = x.as_strided((m, k), (step, 1)), res.as_strided((m, n), (step, 1)), room.as_strided((m, n), (step, 1))
    xr.copy_(rows(m, k, "f16", 1))
    rr.copy_(rows(m, n, "f16", 2))
    w, sw = weights(n, k, 3)
    mat = int8.Int8Matrix(w, sw)
    int8.product(xr, mat, residual=rr, out=out)
    check(xr.clone(), w, sw, out, residual=rr.clone())
    q = int8.quantize(xr)
    assert torch.equal(int8.product(q, mat, residual=rr, dtype=torch.float16), out)


@pytest.mark.parametrize("dtype", T)
@pytest.mark.parametrize("n,k", [(96, 320), (1030, 200), (66, 2056)])
def test_a_row_gives_the_same_bits_in_any_batch(n, k, dtype):
    """Rows alone, among few and among many go through different kernels: the same sums, scales and roundings in each."""
    x, w, sw = rows(1200, k, dtype, 3), *weights(2 * n, k, 4)
    bias, res = torch.randn(2 * n, generator=gen(5), device="cuda"), rows(1200, 2 * n, dtype, 6)
    plain, paired = int8.Int8Matrix(w, sw), int8.Int8Matrix(w, sw, paired=True)
    calls = (lambda r: int8.product(x[r], plain), lambda r: int8.product(x[r], plain, bias=bias), lambda r: int8.product(x[r], plain, residual=res[r]),
             lambda r: int8.product(x[r], plain, bias=bias, residual=res[r]), lambda r: int8.product(x[r], paired),
             lambda r: int8.product(x[r], plain, residual=res[r], dtype=torch.float32), lambda r: int8.product(x[r], plain, bias=bias, residual=res[r].double().float()))
    for call in calls:
        whole = call(slice(0, 1200))
        for m in (1, 2, 3, 16, 17, 20, 33, 40, 64, 65, 100, 300):
            for at in (0, 1200 - m):
                assert torch.equal(call(slice(at, at + m)), whole[at:at + m]), (m, at)


def test_rows_behind_the_last_are_left_as_they_were():
    for m in (1, 7, 16, 33, 130, 257):
        x = rows(m, 256, "f32", 2)
        w, sw = weights(96, 256, 3)
        room = torch.full((m + 300, 96), 7.0, device="cuda")
        int8.product(x, int8.Int8Matrix(w, sw), out=room[:m])
        assert (room[m:] == 7).all()
        check(x, w, sw, room[:m])


def test_layout_of_strided_codes_and_quantized_weights():
    full = torch.randint(-127, 128, (3, 50, 333), generator=gen(1), device="cuda", dtype=torch.int32).to(torch.int8)
    part = full[:, 5:39, 7:307]  # rows at any alignment
    s = torch.rand(3, 34, generator=gen(2), device="cuda")
    x = rows(9, 300, "f32", 4)
    for i in range(3):
        check(x, part[i], s[i], int8.product(x, int8.Int8Matrix(part[i], s[i])))
    w = torch.randn(60, 200, generator=gen(3), device="cuda").bfloat16()
    m = int8.Int8Matrix.quantized(w)
    c, sw = held(w)
    x = rows(9, 200, "f32", 4)
    check(x, c, sw, int8.product(x, m))


def test_outputs_whose_rows_overlap_are_refused():
    w, sw = weights(48, 200, 1)
    mat = int8.Int8Matrix(w, sw)
    x, room = rows(3, 200, "f32", 2), torch.full((200,), 4.0, device="cuda")
    for stride in (0, 47):
        with pytest.raises(ValueError):
            int8.product(x, mat, out=room.as_strided((3, 48), (stride, 1)))
    assert (room == 4).all()
    int8.product(x[:1], mat, out=room.as_strided((1, 48), (0, 1)))  # one row has no other
    check(x[:1], w, sw, room[:48].view(1, 48))


def test_weights_of_more_rows_than_a_call_takes():
    """1024 matrices of 16385 rows, 2^24 + 1024 in all: as the last matrices alone."""
    w = torch.randn(1024, 16385, 3, generator=gen(1), device="cuda", dtype=torch.float16)
    many = int8.Int8Matrix.quantized(w)
    for at in (0, 511, 1023):
        one = int8.Int8Matrix.quantized(w[at])
        assert torch.equal(many._codes.view(1024, -1)[at], one._codes) and torch.equal(many._scales.view(1024, -1)[at], one._scales)


def test_captured_and_replayed_beside_eager_calls_on_another_stream():
    k, n = 1000, 300
    w, sw = weights(n, k, 1)
    mat = int8.Int8Matrix(w, sw)
    other = torch.cuda.Stream()
    for m in (1, 20, 300):
        x = rows(m, k, "bf16", 3)
        space, out = int8.product_workspace(mat, m), torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        int8.product(x, mat, out=out, workspace=space)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            int8.product(x, mat, out=out, workspace=space)
        for seed in range(3):
            x.copy_(rows(m, k, "bf16", 30 + seed))
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            with torch.cuda.stream(other):
                y = int8.product(x, mat)  # (a workspace of its own)
            torch.cuda.synchronize()
            assert torch.equal(y, out)
            check(x, w, sw, out)


def test_a_workspace_for_more_rows_serves_fewer():
    w, sw = weights(64, 256, 1)
    mat = int8.Int8Matrix(w, sw)
    space = int8.product_workspace(mat, 500)
    for m in (0, 1, 33, 500):
        x = rows(m, 256, "f32", 3) if m else torch.empty(0, 256, device="cuda")
        y = int8.product(x, mat, workspace=space)
        assert y.shape == (m, 64)
        if m:
            check(x, w, sw, y)


def test_refusals():
    w, sw = weights(40, 200, 1)
    m, p = int8.Int8Matrix(w, sw), int8.Int8Matrix(w, sw, paired=True)
    x = torch.zeros(3, 200, device="cuda")
    many = int8.Int8Matrix(w.unsqueeze(0).repeat(2, 1, 1), sw.repeat(2, 1))
    grad = torch.zeros(3, 200, device="cuda", requires_grad=True)
    for call in (lambda: int8.product(x[:, :199], m), lambda: int8.product(x.cpu(), m), lambda: int8.product(x.double(), m), lambda: int8.product(x.t(), m),
                 lambda: int8.product(x[0], m), lambda: int8.product(x, many), lambda: int8.product(grad, m), lambda: int8.quantize(grad),
                 lambda: int8.product(x, m, bias=torch.zeros(39, device="cuda")), lambda: int8.product(x, m, bias=torch.zeros(40, device="cuda").half()),
                 lambda: int8.product(x, p, bias=torch.zeros(40, device="cuda")), lambda: int8.product(x, p, residual=torch.zeros(3, 20, device="cuda")),
                 lambda: int8.product(x, m, residual=torch.zeros(2, 40, device="cuda")), lambda: int8.product(x, m, out=torch.zeros(3, 41, device="cuda")),
                 lambda: int8.product(x, m, out=torch.zeros(4, 40, device="cuda")), lambda: int8.product(x, m, out=torch.zeros(3, 40, device="cuda"), dtype=torch.float16),
                 lambda: int8.product(int8.quantize(x[:, :100]), m), lambda: int8.Int8Matrix(w[:39], sw[:39], paired=True), lambda: int8.Int8Matrix(w, sw[:39]),
                 lambda: int8.Int8Matrix(w.to(torch.int16), sw), lambda: int8.Int8Matrix(w.t(), sw), lambda: int8.Int8Matrix(w[:0], sw[:0]),
                 lambda: int8.quantize(x, int8.Int8Rows(3, 199)), lambda: int8.quantize(x, int8.Int8Rows(2, 200)),
                 lambda: int8.product_workspace(m, 1 << 32)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        int8.product(x, m, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    with torch.no_grad():
        int8.product(grad, m)
