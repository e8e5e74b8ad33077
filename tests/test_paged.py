"""CPU tests of the paged cache's entry points: sizes, rotary frequencies against their formulas, refusals
(every one is made on the host, before anything is launched)."""
import ctypes as C
import math

import pytest

from velox_amd import _lib as L

P = 1 << 20  # an address that is aligned and never followed


def desc(**kw):
    d = dict(pool=P, layer_stride=1 << 30, dtype=L.DT_BF16, num_layers=2, num_kv_heads=2, head_dim=64, n_pages=10, page_size=32,
             n_seqs=3, max_pages=4, table_stride=5, reserved=0, table=P, lens=P, refs=P, scratch=P)
    d.update(kw)
    return L.PagedCacheDesc(**d)


def rows(heads=4, dtype=L.DT_F32, data=P, rs=1024, hs=64):
    return L.Rows(data, dtype, heads, rs, hs)


def test_sizes(hiplib):
    v = [C.c_uint64() for _ in range(5)]
    assert hiplib.velox_hip_paged_bytes(C.byref(desc()), *[C.byref(x) for x in v]) == 0
    page, pool, table, refs, scratch = (x.value for x in v)
    assert page == 2 * 2 * 32 * 64 * 2
    assert pool == (1 << 30) + 10 * page and table == 3 * 5 * 4 and refs == 40
    assert scratch >= 4 * (3 * 10)
    assert hiplib.velox_hip_paged_bytes(C.byref(desc(num_layers=1, layer_stride=0)), None, C.byref(v[1]), None, None, None) == 0
    assert v[1].value == 10 * page


BAD = [dict(dtype=L.DT_F32), dict(dtype=7), dict(head_dim=96), dict(head_dim=0), dict(num_kv_heads=0), dict(num_layers=0),
       dict(n_pages=0), dict(page_size=0), dict(page_size=48), dict(page_size=1 << 25), dict(n_seqs=0), dict(n_seqs=4097),
       dict(max_pages=0), dict(table_stride=3), dict(reserved=1), dict(n_pages=1 << 31),
       dict(n_seqs=4096, max_pages=1 << 20, table_stride=1 << 20)]
BAD_MEMORY = [dict(pool=None), dict(pool=P + 8), dict(layer_stride=10 * 16384 - 16), dict(layer_stride=(1 << 30) + 8),
              dict(table=None), dict(lens=None), dict(table=P + 2)]


def attention(lib, d, q=None, out=None, layer=0, window=0, scale=0.0, max_len=128, space=P, size=1 << 40):
    return lib.velox_hip_paged_attention(C.byref(d), layer, C.byref(q or rows()), C.byref(out or rows()), L.AttnMask(window, 0),
                                         scale, max_len, space, size, None)


def prompt(lib, d, q=None, out=None, layer=0, start=P, n=7, scale=0.0):
    return lib.velox_hip_paged_prompt_attention(C.byref(d), layer, C.byref(q or rows()), C.byref(out or rows()), start, n,
                                                L.AttnMask(0, 0), scale, 0, 0, P, 1 << 40, None)


def append(lib, d, q=None, k=None, v=None, qo=None, layer=0, rope=None, start=P, n=2):
    ref = lambda r: C.byref(r) if r is not None else None  # noqa: E731
    return lib.velox_hip_rope_append(C.byref(d), layer, rope, ref(q), ref(k or rows(2)), ref(v or rows(2)), ref(qo), start, n, None)


@pytest.mark.parametrize("bad", BAD + BAD_MEMORY, ids=str)
def test_refuses_descriptions(hiplib, bad):
    d = desc(**bad)
    assert attention(hiplib, d) == L.EINVAL
    assert prompt(hiplib, d) == L.EINVAL
    assert append(hiplib, d) == L.EINVAL
    assert hiplib.velox_hip_pages_extend(C.byref(d), P, None) == L.EINVAL
    if bad in BAD:
        assert hiplib.velox_hip_paged_bytes(C.byref(d), None, None, None, None, None) == L.EINVAL
        n = C.c_uint64()
        assert hiplib.velox_hip_paged_attention_bytes(C.byref(d), 4, 0, C.byref(n)) == L.EINVAL
        assert hiplib.velox_hip_paged_prompt_attention_bytes(C.byref(d), 4, 5, 0, 0, C.byref(n)) == L.EINVAL


def test_refuses_attention_arguments(hiplib):
    d = desc()
    for kw in (dict(layer=2), dict(q=rows(3), out=rows(3)), dict(q=rows(4), out=rows(2)), dict(q=rows(0), out=rows(0)),
               dict(q=rows(data=None)), dict(out=rows(data=P + 2)), dict(q=rows(dtype=3)), dict(scale=math.inf), dict(scale=math.nan),
               dict(q=rows(data=P + 1, dtype=L.DT_F16))):
        assert attention(hiplib, d, **kw) == L.EINVAL, kw
        assert prompt(hiplib, d, **kw) == L.EINVAL, kw
    assert prompt(hiplib, d, start=None) == L.EINVAL
    assert prompt(hiplib, d, start=P + 1) == L.EINVAL
    assert prompt(hiplib, d, n=0) == 0
    n = C.c_uint64(5)
    assert hiplib.velox_hip_paged_attention_bytes(C.byref(d), 3, 0, C.byref(n)) == L.EINVAL
    assert hiplib.velox_hip_paged_attention_bytes(C.byref(d), 4, 0, None) == L.EINVAL
    assert hiplib.velox_hip_paged_prompt_attention_bytes(C.byref(d), 4, 0, 0, 0, C.byref(n)) == 0 and n.value == 0


def test_refuses_a_small_workspace(hiplib):
    d = desc(n_seqs=1, max_pages=5000, table_stride=5000, n_pages=5000, num_layers=1)
    n = C.c_uint64()
    assert hiplib.velox_hip_paged_attention_bytes(C.byref(d), 4, 0, C.byref(n)) == 0
    if n.value:
        for space, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
            assert attention(hiplib, d, max_len=0, space=space, size=size) == L.EINVAL


def test_workspace_grows_with_its_bounds(hiplib):
    """A windowed call plans by a shorter span: the size for the whole length has to be enough for it."""
    d = desc(n_seqs=1, max_pages=5000, table_stride=5000, n_pages=5000, num_layers=1)
    last = 0
    for max_len in (1, 31, 32, 33, 100, 255, 256, 511, 700, 1024, 2000, 4096, 5000, 10000, 30000, 80000, 160000):
        n = C.c_uint64()
        assert hiplib.velox_hip_paged_attention_bytes(C.byref(d), 4, max_len, C.byref(n)) == 0
        assert n.value >= last
        last = n.value


@pytest.mark.parametrize("heads, hkv", [(4, 2), (32, 8), (28, 4), (9, 3), (128, 1), (300, 1), (8, 8)])
def test_prompt_workspace_grows_with_its_rows(hiplib, heads, hkv):
    """Fewer rows are split more, yet the size for a number of rows is enough for any smaller one; the largest of
    the sizes that the numbers up to it need."""
    d = desc(num_kv_heads=hkv, n_seqs=1, max_pages=500, table_stride=500, n_pages=500, num_layers=1, layer_stride=0)

    def size(n):
        v = C.c_uint64()
        assert hiplib.velox_hip_paged_prompt_attention_bytes(C.byref(d), heads, n, 0, 0, C.byref(v)) == 0
        return v.value

    last = 0
    for n in list(range(1, 700)) + [1000, 2048, 4096, 8192, 100000, (1 << 24) - 1]:
        assert size(n) >= last
        last = size(n)
    assert size(1) and last == size(200000)


def test_refuses_too_many_rows(hiplib):
    from velox_amd.paged import Rope

    d, turn, n = desc(), Rope(64), C.c_uint64()
    for many in (1 << 24, (1 << 32) - 1):
        assert prompt(hiplib, d, n=many) == L.EINVAL
        assert append(hiplib, d, n=many) == L.EINVAL
        assert hiplib.velox_hip_rope_rows(turn.handle, C.byref(rows()), C.byref(rows()), many, 64, P, None) == L.EINVAL
        assert hiplib.velox_hip_paged_prompt_attention_bytes(C.byref(d), 4, many, 0, 0, C.byref(n)) == L.EINVAL


def test_refuses_append_arguments(hiplib):
    d = desc()
    for kw in (dict(layer=2), dict(k=rows(3)), dict(v=rows(1)), dict(q=rows(4)), dict(qo=rows(4)), dict(q=rows(4), qo=rows(3)),
               dict(q=rows(4), qo=rows(4, dtype=L.DT_F16)), dict(q=rows(4), qo=rows(4, rs=512)), dict(start=None, n=4),
               dict(start=P + 2)):
        assert append(hiplib, d, **kw) == L.EINVAL, kw
    assert append(hiplib, d, n=0) == 0


def test_refuses_page_calls(hiplib):
    for bad in (dict(refs=None), dict(scratch=None), dict(refs=P + 4), dict(table=None)):
        d = C.byref(desc(**bad))
        assert hiplib.velox_hip_pages_reset(d, None) == L.EINVAL
        assert hiplib.velox_hip_pages_extend(d, P, None) == L.EINVAL
        assert hiplib.velox_hip_pages_fork(d, P, None) == L.EINVAL
        assert hiplib.velox_hip_pages_free(d, P, 1, None) == L.EINVAL
        assert hiplib.velox_hip_pages_trim(d, 5, 0, None) == L.EINVAL
        assert hiplib.velox_hip_pages_compact(d, None) == L.EINVAL
        assert hiplib.velox_hip_pages_status(d, None, None, None) == L.EINVAL
    d = C.byref(desc())
    assert hiplib.velox_hip_pages_extend(d, None, None) == L.EINVAL
    assert hiplib.velox_hip_pages_fork(d, None, None) == L.EINVAL
    assert hiplib.velox_hip_pages_free(d, None, 1, None) == L.EINVAL
    assert hiplib.velox_hip_pages_free(d, None, 0, None) == 0
    assert hiplib.velox_hip_pages_trim(d, 0, 0, None) == L.EINVAL


def test_rope_frequencies(hiplib):
    from velox_amd.paged import Rope

    for r, theta in ((64, 1e4), (128, 5e5), (18, 1e6), (2, 1e4), (256, 1e6)):
        f0 = [theta ** (-2 * j / r) for j in range(r // 2)]
        f, a = Rope(r, theta=theta).frequencies()
        assert a == 1.0 and f == pytest.approx(f0, rel=1e-14)
        f, a = Rope(r, theta=theta, scaling="linear", factor=8).frequencies()
        assert a == 1.0 and f == pytest.approx([x / 8 for x in f0], rel=1e-14)
        # by wave lengths: kept up to 8192 / 4 positions, stretched from 8192 / 1 on
        f, a = Rope(r, theta=theta, scaling="bands", factor=8, original_len=8192).frequencies()
        for x, y in zip(f0, f):
            wave = 2 * math.pi / x
            want = x if wave < 2048 else x / 8 if wave > 8192 else None
            if want is None:
                mix = (8192 / wave - 1) / 3
                want = (1 - mix) * x / 8 + mix * x
            assert y == pytest.approx(want, rel=1e-12)
        f, a = Rope(r, theta=theta, scaling="yarn", factor=32, original_len=4096, amplitude=0.0).frequencies()
        assert a == pytest.approx(0.1 * math.log(32) + 1, rel=1e-14)
        assert all(x / 32 * (1 - 1e-12) <= y <= x * (1 + 1e-12) for x, y in zip(f0, f))
        assert f[0] == f0[0] or r == 2
    assert Rope(64, scaling="yarn", factor=4, original_len=4096, amplitude=1.0).frequencies()[1] == 1.0


@pytest.mark.parametrize("r, theta, length, low, high", [(128, 1e6, 4096, 0, 0), (64, 1e4, 32768, 0, 0), (64, 1e4, 4096, 2.0, 16.0),
                                                       (18, 5e5, 100, 0, 0), (128, 1e4, 5, 0, 0)])
def test_yarn_frequencies(r, theta, length, low, high):
    from velox_amd.paged import Rope

    turn = Rope(r, theta=theta, scaling="yarn", factor=16, original_len=length, low_turns=low, high_turns=high)
    got, _ = turn.frequencies()
    # the pair that turns n times within the length: theta^(-2 j / r) length = 2 pi n, solved for j
    pair = lambda n: r * math.log(length / (2 * math.pi * n)) / (2 * math.log(theta))  # noqa: E731
    a, b = max(math.floor(pair(high or 32)), 0), min(math.ceil(pair(low or 1)), r - 1)
    for j, y in enumerate(got):
        f = theta ** (-2 * j / r)
        ramp = 0.0 if j <= a else 1.0 if j >= b else (j - a) / (b - a)
        assert y == pytest.approx((1 - ramp) * f + ramp * f / 16, rel=1e-12)


def test_refuses_rope_configurations(hiplib):
    def status(**kw):
        d = dict(rot_dim=64, layout=0, scaling=0, original_len=0, theta=1e4, factor=1.0, low_turns=0.0, high_turns=0.0, amplitude=0.0)
        d.update(kw)
        h = C.c_void_p()
        rc = hiplib.velox_hip_rope_create(C.byref(L.RopeConfig(**d)), C.byref(h))
        if rc == 0:
            hiplib.velox_hip_rope_destroy(h)
        return rc

    assert status() == 0
    for kw in (dict(rot_dim=0), dict(rot_dim=63), dict(rot_dim=258), dict(layout=2), dict(scaling=4), dict(theta=0.0), dict(theta=-1.0),
               dict(theta=math.nan), dict(scaling=1, factor=0.5), dict(scaling=1, factor=math.inf), dict(scaling=2, factor=8.0),
               dict(scaling=2, factor=8.0, original_len=10, low_turns=4.0, high_turns=1.0), dict(scaling=3, factor=2.0, original_len=0),
               dict(scaling=3, factor=2.0, original_len=10, theta=1.0), dict(amplitude=-1.0), dict(amplitude=math.nan),
               dict(scaling=2, factor=8.0, original_len=10, low_turns=0.0, high_turns=4.0)):
        assert status(**kw) == L.EINVAL, kw
    assert hiplib.velox_hip_rope_create(None, None) == L.EINVAL
    assert hiplib.velox_hip_rope_frequencies(None, None, None) == L.EINVAL


def test_refuses_rope_rows(hiplib):
    from velox_amd.paged import Rope

    h = Rope(64).handle

    def status(x=None, out=None, n=3, d=64, at=P, rope=h):
        return hiplib.velox_hip_rope_rows(rope, C.byref(x or rows()), C.byref(out or rows()), n, d, at, None)

    turn = Rope(64)
    h = turn.handle
    for kw in (dict(rope=None), dict(d=62), dict(at=None), dict(at=P + 2), dict(out=rows(3)), dict(out=rows(dtype=L.DT_F16)),
               dict(out=rows(rs=512)), dict(x=rows(data=None)), dict(x=rows(heads=0), out=rows(heads=0))):
        kw.setdefault("rope", h)
        assert status(**kw) == L.EINVAL, kw
    assert status(n=0, rope=h) == 0


def test_python_calls_refuse_cpu_tensors():
    import torch

    from velox_amd import paged

    with pytest.raises(ValueError):
        paged.PagedCache.over(torch.zeros(1, 4, 2 * 2 * 32 * 64, dtype=torch.bfloat16), torch.zeros(1, 4, dtype=torch.int32),
                              torch.zeros(1, dtype=torch.int32), page_size=32, num_kv_heads=2, head_dim=64)
    with pytest.raises(ValueError):
        paged.rope(paged.Rope(64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        paged.Rope(64, layout="other")
    with pytest.raises(RuntimeError):
        paged.Rope(63)


def test_rows_that_require_a_gradient_are_refused():
    """No gradient would reach them: an error, not a result without a graph."""
    import torch

    from velox_amd import paged

    cpu = torch.device("cpu")
    x = torch.zeros(2, 3, 64, requires_grad=True)
    for t in (x, x * 2, (x * 2)[:, :2]):
        with pytest.raises(ValueError, match="gradient"):
            paged._rows(t, cpu, "x")
        with torch.no_grad():
            assert paged._rows(t, cpu, "x")[1] == 2
        with torch.inference_mode():
            assert paged._rows(t, cpu, "x")[1] == 2
        assert paged._rows(t.detach(), cpu, "x")[1] == 2


def prompt_bytes(lib, d, heads, n, max_rows, max_len=0):
    v = C.c_uint64()
    assert lib.velox_hip_paged_prompt_attention_bytes(C.byref(d), heads, n, max_rows, max_len, C.byref(v)) == 0
    return v.value


def test_short_rows_of_many_sequences_are_not_split(hiplib):
    """Every sequence has workgroups of its own, a KV head each: where those are 512 at least nothing is split."""
    d = desc(num_kv_heads=8, head_dim=128, n_seqs=80, max_pages=64, table_stride=64, n_pages=4096, page_size=64, num_layers=1)
    for m in (0, 1, 2, 3, 4, 8, 100, 256, 300):
        most = 0
        for n in range(1, 400):
            tiles = 8 * -(-n * 4 // 128)  # of 128 (row, head) pairs
            splits = max(1, min(-(-512 // tiles) if tiles < 256 else 1, 4096 // 512))
            if m and 8 * -(-n // m) >= 512:
                splits = 1
            most = max(most, n * 32 * splits * (128 + 2) * 4 if splits > 1 else 0)
            assert prompt_bytes(hiplib, d, 32, n, m) == most, (n, m)


@pytest.mark.parametrize("heads, hkv", [(4, 2), (28, 4), (9, 3), (300, 1)])
@pytest.mark.parametrize("max_rows", [1, 5, 64])
def test_prompt_workspace_of_short_rows_grows_with_them(hiplib, heads, hkv, max_rows):
    d = desc(num_kv_heads=hkv, n_seqs=4096, max_pages=500, table_stride=500, n_pages=500, num_layers=1, layer_stride=0)
    last = 0
    for n in list(range(1, 400)) + [1000, 2048, 4096, 100000]:
        size = prompt_bytes(hiplib, d, heads, n, max_rows)
        assert last <= size <= prompt_bytes(hiplib, d, heads, n, 0)
        last = size


def test_numbers_past_32_bits_are_refused():
    """ctypes takes a number modulo 2^32: layer 2^32 would be layer 0."""
    import torch

    from velox_amd import paged

    cpu = torch.device("cpu")
    for call in (lambda: paged.Rope((1 << 32) + 64), lambda: paged.Rope(64, scaling="yarn", factor=2.0, original_len=(1 << 32) + 4096),
                 lambda: paged.Rope(64, original_len=-1), lambda: paged._rows(torch.zeros(1, 1, 2).expand((1 << 32) + 1, 1, 2), cpu, "x")):
        with pytest.raises(ValueError):
            call()
    assert paged._rows(torch.zeros(1, 1, 2).expand(1 << 20, 1, 2), cpu, "x")[1] == 1 << 20


def test_refuses_a_workspace_that_a_long_cache_needs_and_is_not_given(hiplib):
    d = desc(n_seqs=1, max_pages=5000, table_stride=5000, n_pages=5000, num_layers=1)
    n = C.c_uint64()
    assert hiplib.velox_hip_paged_attention_bytes(C.byref(d), 4, 0, C.byref(n)) == 0 and n.value
    for space, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
        assert attention(hiplib, d, max_len=0, space=space, size=size) == L.EINVAL
    assert hiplib.velox_hip_paged_prompt_attention_bytes(C.byref(d), 4, 7, 0, 0, C.byref(n)) == 0 and n.value
    for space, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
        assert hiplib.velox_hip_paged_prompt_attention(C.byref(d), 0, C.byref(rows()), C.byref(rows()), P, 7, L.AttnMask(0, 0), 0.0, 0, 0, space,
                                                       size, None) == L.EINVAL


def test_attention_refuses_rows_at_one_address_that_lie_otherwise(hiplib):
    """out may be q; other rows from the same address on would be written while q's are read."""
    d = desc()
    for out in (rows(rs=512), rows(hs=128), rows(dtype=L.DT_BF16)):
        assert attention(hiplib, d, out=out) == L.EINVAL
        assert prompt(hiplib, d, out=out) == L.EINVAL
