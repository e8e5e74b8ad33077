"""CPU tests of the entry points of the 8-bit products and the experts: sizes and refusals (every one is made on the host,
before anything is launched)."""
import ctypes as C
import math

import pytest

from velox_amd import _lib as L

P = 1 << 20  # an address that is aligned and never followed


def matrix(**kw):
    d = dict(codes=P, scales=P, n=48, k=200, count=1, paired=0)
    d.update(kw)
    return L.Int8MatrixDesc(**d)


def rows(dtype=L.DT_F32, data=P, rs=1024, heads=1):
    return L.Rows(data, dtype, heads, rs, 0)


def held(codes=P, scales=P, rs=256):
    return L.Int8RowsDesc(codes, scales, rs)


def ref(s):
    return C.byref(s) if s is not None else None


def u64(fn, *args):
    v = C.c_uint64(12345)
    return fn(*args, C.byref(v)), v.value


@pytest.mark.parametrize("n,k,count,paired,tiles,k_tiles", [(1, 1, 1, 0, 1, 2), (48, 200, 1, 0, 3, 4), (49, 128, 5, 0, 4, 2), (34, 129, 2, 1, 4, 4),
                                                            (1 << 20, 1 << 17, 1, 0, 1 << 16, 1 << 11), (2, 64, 1024, 1, 2, 2)])
def test_sizes(hiplib, n, k, count, paired, tiles, k_tiles):
    codes, scales = C.c_uint64(), C.c_uint64()
    m = matrix(n=n, k=k, count=count, paired=paired, codes=None, scales=None)
    assert hiplib.velox_hip_int8_layout(C.byref(m), C.byref(codes), C.byref(scales)) == 0
    assert codes.value == count * tiles * k_tiles * 1024 and scales.value == count * tiles * 64
    assert hiplib.velox_hip_int8_layout(C.byref(m), None, None) == 0
    if count == 1:
        rc, size = u64(hiplib.velox_hip_int8_product_bytes, C.byref(m), 7)
        assert rc == 0 and size >= 7 * k_tiles * 64 + 28
        assert u64(hiplib.velox_hip_int8_product_bytes, C.byref(m), 0)[0] == 0


BAD = [dict(n=0), dict(k=0), dict(count=0), dict(paired=2), dict(n=47, paired=1), dict(k=(1 << 17) + 1), dict(n=(1 << 20) + 1), dict(count=1025)]
BAD_MEMORY = [dict(codes=None), dict(scales=None), dict(codes=P + 8), dict(scales=P + 4)]


def product(lib, m, x=None, q=None, n=3, bias=None, res=None, out=None, mode=L.GEMV_STORE, space=P, size=1 << 40):
    if x is None and q is None:
        x = rows()
    return lib.velox_hip_int8_product(C.byref(m), ref(x), ref(q), n, bias, ref(res), ref(out or rows()), mode, space, size, None)


@pytest.mark.parametrize("bad", BAD + BAD_MEMORY, ids=str)
def test_refuses_matrices(hiplib, bad):
    m = matrix(**bad)
    assert product(hiplib, m, mode=L.GEMV_SWIGLU if bad.get("paired") else L.GEMV_STORE) == L.EINVAL
    assert hiplib.velox_hip_int8_pack(C.byref(m), 0, 1, P, 0, 200, P, 0, None) == L.EINVAL
    if bad in BAD:
        assert hiplib.velox_hip_int8_layout(C.byref(m), None, None) == L.EINVAL
        assert u64(hiplib.velox_hip_int8_product_bytes, C.byref(m), 3)[0] == L.EINVAL


def test_refuses_pack_arguments(hiplib):
    m = matrix(count=4)
    pack = lambda first, number, codes=P, scales=P: hiplib.velox_hip_int8_pack(C.byref(m), first, number, codes, 9600, 200, scales, 48, None)  # noqa: E731
    for args in ((5, 0), (4, 1), (0, 5), (0xFFFFFFFF, 2), (0, 1, None), (0, 1, P, None), (0, 1, P, P + 2)):
        assert pack(*args) == L.EINVAL, args
    assert pack(4, 0) == 0


def test_refuses_product_arguments(hiplib):
    m = matrix()
    for kw in (dict(x=rows(), q=held()), dict(x=rows(data=None)), dict(x=rows(dtype=3)), dict(x=rows(heads=2)), dict(x=rows(data=P + 2)),
               dict(q=held(codes=None)), dict(q=held(codes=P + 8)), dict(q=held(scales=None)), dict(q=held(scales=P + 1)), dict(q=held(rs=128)),
               dict(q=held(rs=300)), dict(n=1 << 24), dict(out=rows(data=None)), dict(out=rows(heads=0)), dict(out=rows(dtype=L.DT_BF16, data=P + 1)),
               dict(mode=3), dict(mode=-1), dict(mode=L.GEMV_SWIGLU), dict(mode=L.GEMV_RESIDUAL), dict(res=rows()),
               dict(res=rows(data=P + 64, heads=3), mode=L.GEMV_RESIDUAL), dict(res=rows(rs=2048), mode=L.GEMV_RESIDUAL),
               dict(res=rows(dtype=L.DT_F16), mode=L.GEMV_RESIDUAL), dict(bias=P + 2), dict(space=None), dict(space=P + 8), dict(size=100)):
        assert product(hiplib, m, **kw) == L.EINVAL, kw
    p = matrix(paired=1)
    for kw in (dict(), dict(mode=L.GEMV_RESIDUAL, res=rows()), dict(mode=L.GEMV_SWIGLU, bias=P), dict(mode=L.GEMV_SWIGLU, res=rows())):
        assert product(hiplib, p, **kw) == L.EINVAL, kw
    assert product(hiplib, matrix(count=2)) == L.EINVAL
    assert hiplib.velox_hip_int8_product(C.byref(m), None, None, 3, None, None, C.byref(rows()), 0, P, 1 << 40, None) == L.EINVAL
    assert product(hiplib, m, n=0) == 0 and product(hiplib, m, q=held(), n=0) == 0


def test_refuses_quantize_arguments(hiplib):
    call = lambda x=rows(), n=2, k=200, out=held(): hiplib.velox_hip_int8_quantize(ref(x), n, k, ref(out), None)  # noqa: E731
    for kw in (dict(x=None), dict(x=rows(dtype=9)), dict(x=rows(heads=2)), dict(k=0), dict(k=(1 << 17) + 1), dict(n=1 << 24), dict(out=None),
               dict(out=held(rs=128)), dict(out=held(rs=257)), dict(out=held(codes=P + 4)), dict(out=held(scales=None))):
        assert call(**kw) == L.EINVAL, kw
    assert call(n=0) == 0


def route_config(**kw):
    d = dict(n_experts=64, top_k=4, scores=0, groups=1, top_groups=1, group_by=0, renormalize=0, scale=1.0)
    d.update(kw)
    return L.RouteConfig(**d)


def test_refuses_route_arguments(hiplib):
    call = lambda cfg, x=rows(), bias=None, n=3, ids=P, w=P: hiplib.velox_hip_expert_route(ref(cfg), ref(x), bias, n, ids, w, None)  # noqa: E731
    for kw in (dict(n_experts=0), dict(n_experts=1025), dict(top_k=0), dict(top_k=65), dict(scores=2), dict(groups=0), dict(groups=65, n_experts=130),
               dict(groups=3), dict(groups=4, top_groups=5), dict(top_groups=0), dict(group_by=2), dict(renormalize=2), dict(scale=math.inf),
               dict(scale=math.nan), dict(groups=32, top_groups=1, top_k=3), dict(n_experts=3)):
        assert call(route_config(**kw)) == L.EINVAL, kw
    c = route_config()
    for kw in (dict(x=None), dict(x=rows(heads=2)), dict(x=rows(dtype=5)), dict(x=rows(data=P + 2)), dict(bias=P + 1), dict(n=1 << 24), dict(ids=None),
               dict(w=None), dict(ids=P + 2), dict(w=P + 2)):
        assert call(c, **kw) == L.EINVAL, kw
    assert call(c, n=0) == 0
    assert hiplib.velox_hip_expert_route(None, ref(rows()), None, 3, P, P, None) == L.EINVAL


def test_refuses_group_arguments(hiplib):
    call = lambda ids=P, n=100, first=0, count=8, order=P, offsets=P, space=P, size=1 << 30: hiplib.velox_hip_expert_group(  # noqa: E731
        ids, n, first, count, order, offsets, space, size, None)
    for kw in (dict(ids=None), dict(ids=P + 1), dict(n=(1 << 20) + 1), dict(count=0), dict(count=1025), dict(first=0xFFFFFFFF), dict(first=0xFFFFFFF8),
               dict(order=None), dict(order=P + 2), dict(offsets=None), dict(offsets=P + 3), dict(n=1 << 20, space=None), dict(n=1 << 20, space=P + 8),
               dict(n=1 << 20, size=10)):
        assert call(**kw) == L.EINVAL, kw
    for args in (((1 << 20) + 1, 8), (5, 0), (5, 1025)):
        assert u64(hiplib.velox_hip_expert_group_bytes, *args)[0] == L.EINVAL
    last = 0
    for n in (0, 1, 100, 2048, 2049, 5000, 100000, 1 << 20):  # a workspace for many slots serves fewer
        rc, size = u64(hiplib.velox_hip_expert_group_bytes, n, 256)
        assert rc == 0 and size >= last
        last = size


def test_refuses_group_memory_that_overlaps(hiplib):
    """Several workgroups read ids while others write order: every pair of the four has to be apart, by a byte at least."""
    n, count = 5000, 8
    rc, need = u64(hiplib.velox_hip_expert_group_bytes, n, count)
    assert rc == 0 and need > 0
    own = dict(ids=P, order=2 * P, offsets=3 * P, space=4 * P)
    size = dict(ids=4 * n, order=4 * n, offsets=4 * (count + 1), space=need)
    for a in own:
        for b in own:
            if a == b:
                continue
            ends = [0, 16, size[b] - 4, 4 - size[a]]  # where a begins, from b on: its start, inside, its last word, a's last word
            for at in ends if "space" not in (a, b) else [0, 16, (size[b] - 1) // 16 * 16, -((size[a] - 1) // 16 * 16)]:
                kw = dict(own, **{a: own[b] + at})
                assert hiplib.velox_hip_expert_group(kw["ids"], n, 0, count, kw["order"], kw["offsets"], kw["space"], need, None) == L.EINVAL, (a, b, at)
    for m in (1, 1024):  # one workgroup too
        assert hiplib.velox_hip_expert_group(P, m, 0, count, P, 2 * P, None, 0, None) == L.EINVAL
        assert hiplib.velox_hip_expert_group(P, m, 0, count, 2 * P, P + 4 * m - 4, None, 0, None) == L.EINVAL


def test_refuses_route_memory_that_overlaps(hiplib):
    n, c = 40, route_config()  # 64 experts, 4 of them
    bytes_ = 4 * n * 4

    def call(x=rows(), bias=None, ids=3 * P, w=4 * P):
        return hiplib.velox_hip_expert_route(ref(c), ref(x), bias, n, ids, w, None)

    for at in (0, 4, bytes_ - 4, 4 - bytes_):
        assert call(w=3 * P + at) == L.EINVAL, at
    last = P + 4 * 1024 * (n - 1)  # the last row's logits
    for at in (P, P + 4 * 63, P + 4 * 1024 - 4 * 100, last, last + 4 * 63, P - bytes_ + 4):
        for kw in (dict(ids=at), dict(w=at)):
            assert call(**kw) == L.EINVAL, (at, kw)
    half = rows(dtype=L.DT_BF16)
    for at in (P, P + 124, P + 2 * 1024 * 7 + 124, P + 2 * 1024 * (n - 1) + 124):
        assert call(x=half, ids=at) == L.EINVAL, at
    for at in (5 * P, 5 * P + 252, 5 * P - bytes_ + 4):
        assert call(bias=5 * P, ids=at) == L.EINVAL and call(bias=5 * P, w=at) == L.EINVAL, at


def test_refuses_ffn_arguments(hiplib):
    gu, dn = matrix(n=128, k=256, count=4, paired=1), matrix(n=256, k=64, count=4)

    def call(g=gu, d=dn, first=0, x=rows(), ids=P, w=P, n=3, top=2, res=None, out=rows(data=1 << 24), space=P, size=1 << 50):
        return hiplib.velox_hip_expert_ffn(ref(g), ref(d), first, ref(x), ids, w, n, top, ref(res), ref(out), space, size, None)

    shapes = [dict(g=matrix(n=128, k=256, count=4)), dict(d=matrix(n=256, k=64, count=4, paired=1)), dict(d=matrix(n=256, k=64, count=3)),
              dict(d=matrix(n=256, k=128, count=4)), dict(d=matrix(n=255, k=64, count=4)), dict(top=0), dict(top=65), dict(n=(1 << 19) + 1)]
    for kw in shapes + [dict(g=matrix(n=128, k=256, count=4, paired=1, codes=None)), dict(d=matrix(n=256, k=64, count=4, scales=P + 4)), dict(x=None),
                        dict(x=rows(heads=4)), dict(out=None), dict(out=rows(dtype=3)), dict(first=0xFFFFFFFF), dict(ids=None), dict(w=None),
                        dict(ids=P + 2), dict(w=P + 1), dict(res=rows(data=1 << 24, rs=2048)), dict(res=rows(heads=2)), dict(out=rows(rs=2048)),
                        dict(out=rows(dtype=L.DT_F16)), dict(space=None), dict(space=P + 8), dict(size=1000)]:
        assert call(**kw) == L.EINVAL, kw
    for kw in shapes:
        assert u64(hiplib.velox_hip_expert_ffn_bytes, ref(kw.get("g", gu)), ref(kw.get("d", dn)), kw.get("n", 3), kw.get("top", 2))[0] == L.EINVAL
    assert call(n=0) == 0


def test_ffn_workspace_grows_with_its_rows(hiplib):
    """The size for a number of rows is enough for any smaller one."""
    for hidden, inner, count, top in ((256, 64, 4, 2), (7168, 2048, 64, 8), (100, 33, 1, 1), (2048, 1408, 64, 6)):
        gu, dn = matrix(n=2 * inner, k=hidden, count=count, paired=1), matrix(n=hidden, k=inner, count=count)
        last = 0
        for n in list(range(0, 70)) + [100, 128, 255, 256, 257, 511, 512, 1000, 1024, 4096, 10000]:
            rc, size = u64(hiplib.velox_hip_expert_ffn_bytes, ref(gu), ref(dn), n, top)
            assert rc == 0 and size >= last, n
            last = size


def test_python_refuses_tensors_of_the_host():
    torch = pytest.importorskip("torch")
    from velox_amd import experts, int8
    with pytest.raises(ValueError):
        int8.quantize(torch.zeros(2, 4))
    with pytest.raises(ValueError):
        int8.Int8Matrix(torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2))
    with pytest.raises(ValueError):
        experts.route(torch.zeros(2, 4), 1)
    with pytest.raises(ValueError):
        experts.group(torch.zeros(2, 4, dtype=torch.int32), 3)


@pytest.mark.parametrize("stride", [0, 1, 47])
def test_refuses_outputs_whose_rows_overlap(hiplib, stride):
    assert product(hiplib, matrix(), out=rows(data=1 << 24, rs=stride)) == L.EINVAL
    assert product(hiplib, matrix(), q=held(), out=rows(data=1 << 24, rs=stride)) == L.EINVAL
    assert product(hiplib, matrix(n=96, paired=1), out=rows(data=1 << 24, rs=stride), mode=L.GEMV_SWIGLU) == L.EINVAL
    out = rows(data=1 << 24, rs=stride)  # (the residual's own place does not help)
    assert product(hiplib, matrix(), out=out, res=out, mode=L.GEMV_RESIDUAL) == L.EINVAL
    gu, dn = matrix(n=128, k=48, count=4, paired=1), matrix(n=48, k=64, count=4)
    assert hiplib.velox_hip_expert_ffn(ref(gu), ref(dn), 0, ref(rows()), P, P, 2, 2, None, ref(out), P, 1 << 50, None) == L.EINVAL


def test_python_refuses_outputs_whose_rows_overlap():
    torch = pytest.importorskip("torch")
    from velox_amd import int8
    cpu, room = torch.device("cpu"), torch.zeros(100)
    for stride in (0, 1, 7):
        with pytest.raises(ValueError):
            int8._result(room.as_strided((3, 8), (stride, 1)), cpu, 8, 3)
        assert int8._result(room.as_strided((1, 8), (stride, 1)), cpu, 8, 1).row_stride == stride
    assert int8._result(room.as_strided((3, 8), (8, 1)), cpu, 8, 3).row_stride == 8


def test_python_refuses_rows_and_lengths_past_32_bits():
    """ctypes would hand them on modulo 2^32, and all but the first rows, or the first values, would be left out."""
    torch = pytest.importorskip("torch")
    from velox_amd import int8
    cpu = torch.device("cpu")
    for t in (torch.zeros(1, 8).expand((1 << 32) + 5, 8), torch.zeros(1, 8, dtype=torch.bfloat16).expand(1 << 32, 8),
              torch.empty(0).as_strided((0, (1 << 32) + 8), (1, 1))):
        with pytest.raises(ValueError):
            int8._plain(t, cpu, "x")
        with pytest.raises(ValueError):
            int8._plain(t, cpu, "x", t.shape[1])
    assert int8._plain(torch.zeros(1, 8).expand((1 << 32) - 1, 8), cpu, "x")[1] == (1 << 32) - 1  # (the C ABI refuses these)
