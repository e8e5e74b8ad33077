"""The paged KV cache and its operators on torch tensors: rotary positions, append, attention, pages.

Thin calls of the C ABI (include/velox_hip.h, "paged KV cache"): a call checks types, shapes and devices
(ValueError), launches on the current stream of the cache's device and returns without waiting; a status other
than 0 raises as everywhere in this package. Tensors of whole numbers are int32 and hold the C ABI's unsigned
values: -1 is VELOX_HIP_NO_PAGE / VELOX_HIP_NO_SEQ. The operators have no backward pass: with gradients enabled, tensors
that require one are refused. Calls can be captured into a graph once `out` and
`workspace` are given. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.DT_F32, torch.float16: L.DT_F16, torch.bfloat16: L.DT_BF16}
_LAYOUTS = {"half": L.ROPE_HALF, "interleaved": L.ROPE_INTERLEAVED}
_SCALINGS = {"none": L.ROPE_PLAIN, "linear": L.ROPE_LINEAR, "bands": L.ROPE_BANDS, "yarn": L.ROPE_YARN}


# the current device and a device's current stream as plain numbers: torch.cuda.current_stream builds an object for
# every call, a good part of a small operator's host time
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _numbers(what: str, *values: int) -> None:
    """Whole numbers that the C ABI's 32 bits hold: ctypes would take others modulo 2^32."""
    for v in values:
        if not 0 <= v <= 0xFFFFFFFF:
            raise ValueError(f"{what}: whole numbers of [0, 2^32) are wanted, got {v}")


def _no_gradient(t: torch.Tensor, what: str) -> None:
    _need(not (t.requires_grad and torch.is_grad_enabled()),
          f"{what}: requires a gradient, and none is formed here (detach it, or call under torch.no_grad())")


def _gpu(t: torch.Tensor, what: str) -> torch.device:
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{what}: a tensor on the GPU is wanted")
    return t.device


def _call(fn, index: int, *args) -> None:
    """fn(*args, stream) on device `index`, its current stream."""
    if _device() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        L.check(rc, fn.__name__)


def _like(t: torch.Tensor, r: L.Rows, dim: int) -> tuple[torch.Tensor, L.Rows]:
    """A new tensor of t's shape and type, and its rows; r: t's."""
    out = torch.empty_like(t, memory_format=torch.contiguous_format)
    h = r.heads
    return out, L.Rows(out.data_ptr(), r.dtype, h, h * dim, dim)


def _words(t: torch.Tensor, n: int, device: torch.device, what: str) -> int:
    """The address of an int32 vector of n elements (n < 0: any length)."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 vector on {device} is wanted")
    if n >= 0 and t.numel() != n:
        raise ValueError(f"{what}: {n} elements are wanted, got {t.numel()}")
    return t.data_ptr()


def _rows(t: torch.Tensor, device: torch.device, what: str, heads: int = 0, dim: int = 0) -> tuple[L.Rows, int]:
    """[row][head][element] as VeloxHipRows, and its rows; the elements of a head are next to each other."""
    code = _DTYPES.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if code is None or t.device != device or t.dim() != 3:
        raise ValueError(f"{what}: a float32, float16 or bfloat16 tensor [row][head][element] on {device} is wanted")
    if t.requires_grad:
        _no_gradient(t, what)
    n, h, d = t.shape
    if (n | h | d) >> 32:
        _numbers(what, n, h, d)
    if (heads and h != heads) or (dim and d != dim):
        raise ValueError(f"{what}: heads and head size {heads, dim} are wanted, got {h, d}")
    rs, hs, es = t.stride()
    if es != 1 and d != 1:
        raise ValueError(f"{what}: a head's elements have to be next to each other")
    return L.Rows(t.data_ptr(), code, h, rs, hs), n


class PagedCache:
    """A paged KV cache of `n_seqs` sequences: pool [layers][pages][2 * KV heads * page size * head size], table
    [sequences][max_pages] (page numbers, -1: none), lens [sequences], refs [pages].

    PagedCache(...) allocates and empties one; over() takes tensors the caller has (refs None: the caller keeps
    the pages itself and extend .. compact refuse). The tensors stay the caller's to read and write between calls.
    """

    def __init__(self, n_pages: int, n_seqs: int, max_pages: int, *, page_size: int, num_kv_heads: int, head_dim: int,
                 n_layers: int = 1, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        _need(min(n_pages, n_seqs, max_pages, page_size, num_kv_heads, head_dim, n_layers) > 0, "sizes have to be positive")
        words = dict(dtype=torch.int32, device=device)
        pool = torch.zeros(n_layers, n_pages, 2 * num_kv_heads * page_size * head_dim, dtype=dtype, device=device)
        self._bind(pool, torch.full((n_seqs, max_pages), -1, **words), torch.zeros(n_seqs, **words), page_size,
                   num_kv_heads, head_dim, torch.zeros(n_pages, **words))
        self.reset()

    @classmethod
    def over(cls, pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *, page_size: int, num_kv_heads: int,
             head_dim: int, refs: torch.Tensor | None = None) -> "PagedCache":
        self = cls.__new__(cls)
        self._bind(pool, table, lens, page_size, num_kv_heads, head_dim, refs)
        return self

    def _bind(self, pool, table, lens, page_size, num_kv_heads, head_dim, refs) -> None:
        device = _gpu(pool, "pool")
        _no_gradient(pool, "pool")
        _need(pool.dim() == 3 and pool.dtype in (torch.float16, torch.bfloat16), "pool: float16 or bfloat16 [layer][page][element]")
        n_layers, n_pages, elements = pool.shape
        _need(elements == 2 * num_kv_heads * page_size * head_dim, "pool: a page holds 2 * KV heads * page size * head size elements")
        _need(pool.stride(2) == 1 and (n_pages == 1 or pool.stride(1) == elements), "pool: the pages of a layer have to be next to each other")
        _need(_gpu(table, "table") == device and table.dim() == 2 and table.dtype == torch.int32 and table.stride(1) == 1,
              "table: int32 [sequence][page] on the pool's device")
        self.lib = L.load()
        self.device, self.head_dim, self.num_kv_heads, self.page_size = device, head_dim, num_kv_heads, page_size
        self.n_seqs, self.max_pages = table.shape
        self.pool, self.table, self.lens, self.refs = pool, table, lens, refs
        stride = table.stride(0) if self.n_seqs > 1 else self.max_pages
        _numbers("table", self.max_pages, stride)
        d = L.PagedCacheDesc(pool.data_ptr(), pool.stride(0) * 2, _DTYPES[pool.dtype], n_layers, num_kv_heads, head_dim, n_pages,
                             page_size, self.n_seqs, self.max_pages, stride, 0, table.data_ptr(),
                             _words(lens, self.n_seqs, device, "lens"), None, None)
        scratch = C.c_uint64()
        L.check(self.lib.velox_hip_paged_bytes(C.byref(d), None, None, None, None, C.byref(scratch)), "paged_bytes")
        self._scratch = None
        if refs is not None:
            d.refs = _words(refs, n_pages, device, "refs")
            self._scratch = torch.zeros(scratch.value // 4, dtype=torch.int32, device=device)
            d.scratch = self._scratch.data_ptr()
        self.desc = d
        self._ref, self._index = C.byref(d), device.index

    # -- pages ----------------------------------------------------------------------------------
    def _pages(self, name: str, *args) -> None:
        _call(getattr(self.lib, "velox_hip_pages_" + name), self._index, self._ref, *args)

    def reset(self) -> None:
        """No sequence has a page, every page is free."""
        self._pages("reset")

    def extend(self, add: torch.Tensor) -> None:
        """lens += add (int32 [sequence]), with the pages that takes; a shared last page is copied first."""
        self._pages("extend", _words(add, self.n_seqs, self.device, "add"))

    def fork(self, src: torch.Tensor) -> None:
        """Every sequence s becomes what src[s] was (int32 [sequence], -1: empty), its pages shared."""
        self._pages("fork", _words(src, self.n_seqs, self.device, "src"))

    def free(self, seqs: torch.Tensor) -> None:
        """The sequences listed (int32) are empty."""
        listed = _words(seqs, -1, self.device, "seqs")
        _numbers("seqs", seqs.numel())
        self._pages("free", listed, seqs.numel())

    def trim(self, window: int, sinks: int = 0) -> None:
        """Frees the whole pages that no later row of a window sees."""
        _need(window >= 1 and sinks >= 0, "trim: window >= 1 and sinks >= 0 are wanted")
        self._pages("trim", min(window, 0xFFFFFFFF), min(sinks, 0xFFFFFFFF))

    def compact(self) -> None:
        """The live pages move to the front of the pool."""
        self._pages("compact")

    def status(self) -> tuple[int, int]:
        """(sequences that the last extend refused, free pages now); waits for the stream."""
        refused, free = C.c_uint32(), C.c_uint32()
        self._pages("status", C.byref(refused), C.byref(free))
        return int(refused.value), int(free.value)

    # -- workspaces -----------------------------------------------------------------------------
    def attention_workspace(self, heads: int, *, max_len: int = 0) -> torch.Tensor | None:
        """What attention() needs with these bounds, whatever its mask (None: nothing)."""
        n = C.c_uint64()
        _numbers("heads and max_len", heads, max_len)
        L.check(self.lib.velox_hip_paged_attention_bytes(self._ref, heads, max_len, C.byref(n)), "paged_attention_bytes")
        return torch.empty(n.value, dtype=torch.uint8, device=self.device) if n.value else None

    def prompt_workspace(self, heads: int, *, total_rows: int, max_rows: int = 0, max_len: int = 0) -> torch.Tensor | None:
        """What prompt_attention() needs for up to total_rows rows with these bounds (None: nothing)."""
        n = C.c_uint64()
        _numbers("heads, total_rows, max_rows and max_len", heads, total_rows, max_rows, max_len)
        L.check(self.lib.velox_hip_paged_prompt_attention_bytes(self._ref, heads, total_rows, max_rows, max_len, C.byref(n)),
                "paged_prompt_attention_bytes")
        return torch.empty(n.value, dtype=torch.uint8, device=self.device) if n.value else None


class Rope:
    """Rotary positions of the first rot_dim values of a head (velox_hip_rope_create)."""

    def __init__(self, rot_dim: int, *, theta: float = 10000.0, layout: str = "half", scaling: str = "none", factor: float = 1.0,
                 original_len: int = 0, low_turns: float = 0.0, high_turns: float = 0.0, amplitude: float = 0.0):
        _need(layout in _LAYOUTS and scaling in _SCALINGS, f"layout is one of {tuple(_LAYOUTS)}, scaling one of {tuple(_SCALINGS)}")
        _need(rot_dim > 0, "rot_dim has to be positive")
        _numbers("rot_dim and original_len", rot_dim, original_len)
        self.lib = L.load()
        self.handle = C.c_void_p()
        self.rot_dim = rot_dim
        cfg = L.RopeConfig(rot_dim, _LAYOUTS[layout], _SCALINGS[scaling], original_len, theta, factor, low_turns, high_turns, amplitude)
        L.check(self.lib.velox_hip_rope_create(C.byref(cfg), C.byref(self.handle)), "rope_create")

    def frequencies(self) -> tuple[list[float], float]:
        """Radians per position of every pair, and the factor on the rotated values."""
        f, amplitude = (C.c_double * (self.rot_dim // 2))(), C.c_double()
        L.check(self.lib.velox_hip_rope_frequencies(self.handle, f, C.byref(amplitude)), "rope_frequencies")
        return list(f), amplitude.value

    def close(self) -> None:
        if self.handle:
            self.lib.velox_hip_rope_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def rope(turn: Rope, x: torch.Tensor, positions: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [row][head][element] turned by positions (int32 [row]); out: x itself, or a tensor of its shape and type."""
    device = _gpu(x, "x")
    _need(bool(turn.handle), "rope: the handle is closed")
    xr, n = _rows(x, device, "x")
    if out is None:
        out, o = _like(x, xr, x.shape[2])
    else:
        o, _ = _rows(out, device, "out")
        _need(out.shape == x.shape and out.dtype == x.dtype, "out: the shape and type of x are wanted")
    at = _words(positions, n, device, "positions")
    if x.numel():
        _call(turn.lib.velox_hip_rope_rows, device.index, turn.handle, xr, o, n, x.shape[2], at)
    return out


def rope_append(cache: PagedCache, layer: int, turn: Rope | None, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                q_out: torch.Tensor | None = None, *, q_start: torch.Tensor | None = None) -> torch.Tensor | None:
    """The new rows of `layer`: q turned into q_out (default: a new tensor; may be q), k turned and v into the pages.
    q_start (int32 [sequences + 1]) gives the sequences' rows; None: row s is sequence s's."""
    device, d = cache.device, cache.head_dim
    _need(turn is None or bool(turn.handle), "rope_append: the handle is closed")
    if layer >> 32:
        _numbers("layer", layer)
    kr, n = _rows(k, device, "k", cache.num_kv_heads, d)
    vr, vn = _rows(v, device, "v", cache.num_kv_heads, d)
    _need(vn == n, "k and v: as many rows of each are wanted")
    qr = qo = None
    if q is not None:
        qr, qn = _rows(q, device, "q", 0, d)
        if q_out is None:
            on = qn
            q_out, qo = _like(q, qr, d)
        else:
            qo, on = _rows(q_out, device, "q_out", qr.heads, d)
        _need(qn == n and on == n, "q and q_out: as many rows as k are wanted")
    else:
        _need(q_out is None, "q_out without q")
    start = _words(q_start, cache.n_seqs + 1, device, "q_start") if q_start is not None else None
    if n:
        _call(cache.lib.velox_hip_rope_append, cache._index, cache._ref, layer, turn.handle if turn is not None else None, qr, kr, vr,
              qo, start, n)
    return q_out


_WHOLE = L.AttnMask(0, 0)


def _mask(window: int, sinks: int) -> L.AttnMask:
    if window == 0 and sinks >= 0:
        return _WHOLE  # sinks do nothing without a window
    _need(window >= 0 and sinks >= 0, "window and sinks have to be at least 0")
    return L.AttnMask(min(window, 0xFFFFFFFF), min(sinks, 0xFFFFFFFF))


def _space(workspace: torch.Tensor | None, device: torch.device) -> tuple[int | None, int]:
    if workspace is None:
        return None, 0
    if not isinstance(workspace, torch.Tensor) or workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace: contiguous memory on {device} is wanted")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def attention(cache: PagedCache, layer: int, q: torch.Tensor, *, window: int = 0, sinks: int = 0, scale: float = 0.0,
              max_len: int = 0, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every sequence's newest position: q [sequence][q head][head size], already in the cache.
    max_len bounds lens for planning; workspace: cache.attention_workspace of the same bounds (None: made here)."""
    device = cache.device
    if (layer | max_len) >> 32:
        _numbers("layer and max_len", layer, max_len)
    qr, n = _rows(q, device, "q", 0, cache.head_dim)
    _need(n == cache.n_seqs, f"q: {cache.n_seqs} rows are wanted")
    if out is None:
        out, o = _like(q, qr, cache.head_dim)
    else:
        o, on = _rows(out, device, "out", qr.heads, cache.head_dim)
        _need(on == n, "out: as many rows as q are wanted")
    if workspace is None:
        workspace = cache.attention_workspace(qr.heads, max_len=max_len)
    space, size = _space(workspace, device)
    _call(cache.lib.velox_hip_paged_attention, cache._index, cache._ref, layer, qr, o, _mask(window, sinks), scale, max_len, space, size)
    return out


def prompt_attention(cache: PagedCache, layer: int, q: torch.Tensor, q_start: torch.Tensor, *, window: int = 0, sinks: int = 0,
                     scale: float = 0.0, max_rows: int = 0, max_len: int = 0, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged batch's rows, q [row][q head][head size]; sequence s has rows q_start[s] .. q_start[s + 1],
    the last of them its newest position. Rows of no sequence are not written."""
    device = cache.device
    if (layer | max_rows | max_len) >> 32:
        _numbers("layer, max_rows and max_len", layer, max_rows, max_len)
    qr, n = _rows(q, device, "q", 0, cache.head_dim)
    if out is None:
        out, o = _like(q, qr, cache.head_dim)
    else:
        o, on = _rows(out, device, "out", qr.heads, cache.head_dim)
        _need(on == n, "out: as many rows as q are wanted")
    start = _words(q_start, cache.n_seqs + 1, device, "q_start")
    if n == 0:
        return out
    if workspace is None:
        workspace = cache.prompt_workspace(qr.heads, total_rows=n, max_rows=max_rows, max_len=max_len)
    space, size = _space(workspace, device)
    _call(cache.lib.velox_hip_paged_prompt_attention, cache._index, cache._ref, layer, qr, o, start, n, _mask(window, sinks), scale,
          max_rows, max_len, space, size)
    return out
