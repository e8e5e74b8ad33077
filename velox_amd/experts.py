"""Experts on torch tensors: the choice of experts for each token, the grouping of tokens by expert, the experts' products.

Thin calls of the C ABI (include/velox_hip.h, "experts"), in the manner of velox_amd.paged: a call checks types, shapes and
devices (ValueError), launches on the current stream of its tensors' device and returns without waiting; a status other than
0 raises. ids are int32 and hold the C ABI's unsigned values: -1 is VELOX_HIP_NO_EXPERT. No backward pass: with gradients
enabled, tensors that require one are refused. Calls can be captured into a graph once their outputs and `workspace` are
given. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib as L
from .int8 import Int8Matrix, _floats, _memory, _plain, _result
from .paged import _call, _gpu, _need, _numbers, _space, _words

_lib = L.load  # (the library is looked up by the calls, not where this module is read)
_SCORES = {"softmax": L.ROUTE_SOFTMAX, "sigmoid": L.ROUTE_SIGMOID}
_MARKS = {"max": L.GROUP_LARGEST, "two": L.GROUP_TWO}


def _whole(t: torch.Tensor, shape: tuple, device: torch.device, what: str) -> int:
    """The address of a contiguous int32 tensor of a shape."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 tensor of shape {shape} on {device} is wanted")
    return t.data_ptr()


def route(logits: torch.Tensor, top_k: int, *, scores: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          top_groups: int = 1, group_by: str = "max", renormalize: bool = False, scale: float = 1.0,
          ids: torch.Tensor | None = None, weights: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(ids int32, weights float32), both [row][top_k]: the experts with the largest score (+ bias) of logits [row][expert], of
    the top_groups best groups where there are several; weights are the scores (renormalize: divided by their sum) times
    scale. -infinity masks an expert; a row without enough experts ends in -1 with weight 0. ids and weights are memory of
    their own."""
    device = _gpu(logits, "logits")
    how, mark = _SCORES.get(scores), _MARKS.get(group_by)
    if how is None or mark is None:
        raise ValueError(f"scores is one of {tuple(_SCORES)}, group_by one of {tuple(_MARKS)}")
    xr, n = _plain(logits, device, "logits")
    experts = logits.shape[1]
    if not (1 <= groups <= 64 and 1 <= experts <= 1024 and experts % groups == 0 and 1 <= top_groups <= groups):
        raise ValueError("1 to 1024 experts in up to 64 groups of one size are wanted, and 1 to `groups` of the groups")
    if not 1 <= top_k <= min(64, experts // groups * top_groups):
        raise ValueError("top_k: 1 to 64, no more than there are experts in top_groups groups")
    if ids is None:
        ids = torch.empty((n, top_k), dtype=torch.int32, device=device)
        i = ids.data_ptr()
    else:
        i = _whole(ids, (n, top_k), device, "ids")
    if weights is None:
        weights = torch.empty((n, top_k), dtype=torch.float32, device=device)
        w = weights.data_ptr()
    else:
        w = _floats(weights, (n, top_k), device, "weights")
    b = _floats(bias, (experts,), device, "bias") if bias is not None else None
    if n:
        cfg = L.RouteConfig(experts, top_k, how, groups, top_groups, mark, 1 if renormalize else 0, scale)
        _call(_lib().velox_hip_expert_route, device.index, cfg, xr, b, n, i, w)
    return ids, weights


def _device_index(device) -> torch.device:
    device = torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


@functools.lru_cache(maxsize=1024)
def _group_bytes(slots: int, count: int) -> int:
    n = C.c_uint64()
    L.check(_lib().velox_hip_expert_group_bytes(slots, count, C.byref(n)), "expert_group_bytes")
    return n.value


def group_workspace(slots: int, count: int, device="cuda") -> torch.Tensor | None:
    """What group() needs for up to `slots` slots of `count` experts (None: nothing)."""
    _numbers("slots and count", slots, count)
    n = _group_bytes(slots, count)
    return _memory(n, device if isinstance(device, torch.device) else _device_index(device)) if n else None


def group(ids: torch.Tensor, count: int, first: int = 0, *, order: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
          workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(order int32 [slot], offsets int32 [count + 1]): the slots of ids (row * top_k + place) by expert first .. first +
    count - 1, an expert's in their own order at order[offsets[e] : offsets[e + 1]]; -1 behind the last. ids, order, offsets
    and workspace are memory of their own."""
    device = _gpu(ids, "ids")
    slots = ids.numel()
    at = _whole(ids, ids.shape, device, "ids")
    if (first | count) >> 32:
        _numbers("first and count", first, count)
    if not 1 <= count <= 1024 or slots > 1 << 20:
        raise ValueError("1 to 1024 experts and up to 2^20 slots are wanted")
    if order is None:
        order = torch.empty(slots, dtype=torch.int32, device=device)
        o = order.data_ptr()
    else:
        o = _words(order, slots, device, "order")
    if offsets is None:
        offsets = torch.empty(count + 1, dtype=torch.int32, device=device)
        f = offsets.data_ptr()
    else:
        f = _words(offsets, count + 1, device, "offsets")
    if workspace is None:
        workspace = group_workspace(slots, count, device)
    space, size = _space(workspace, device)
    _call(_lib().velox_hip_expert_group, device.index, at, slots, first, count, o, f, space, size)
    return order, offsets


def ffn_workspace(gate_up: Int8Matrix, down: Int8Matrix, rows: int, top_k: int) -> torch.Tensor | None:
    """What ffn() needs for up to `rows` rows of top_k experts (None: nothing)."""
    n = C.c_uint64()
    _numbers("rows and top_k", rows, top_k)
    L.check(gate_up.lib.velox_hip_expert_ffn_bytes(gate_up._ref, down._ref, rows, top_k, C.byref(n)), "expert_ffn_bytes")
    return _memory(n.value, gate_up.device)


def ffn(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate_up: Int8Matrix, down: Int8Matrix, *, first: int = 0,
        residual: torch.Tensor | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Row r of x [row][hidden]: the sum over j of weights[r][j] * down_e(silu(gate_e(x)) * up_e(x)), e = ids[r][j] (int32
    [row][top_k]), plus the residual's row. gate_up (paired) and down hold the experts first .. first + count - 1; other
    ids add nothing. out: a new tensor of x's type, or the one given (may be x or the residual). workspace: ffn_workspace
    (None: made here)."""
    device = gate_up.device
    if not (gate_up.paired and not down.paired and down.device == device and gate_up.count == down.count and gate_up.outputs == down.k and
            gate_up.k == down.n):
        raise ValueError("gate_up (paired) [2 inner][hidden] and down [hidden][inner] of as many experts are wanted")
    xr, n = _plain(x, device, "x", gate_up.k)
    top = ids.shape[1] if isinstance(ids, torch.Tensor) and ids.dim() == 2 else 0
    if not 1 <= top <= 64 or n * top > 1 << 20:
        raise ValueError("ids: [row][1 to 64] is wanted, up to 2^20 slots in all")
    if first >> 32:
        _numbers("first", first)
    i, w = _whole(ids, (n, top), device, "ids"), _floats(weights, (n, top), device, "weights")
    if out is None:
        out = torch.empty((n, gate_up.k), dtype=x.dtype, device=device)
        o = L.Rows(out.data_ptr(), xr.dtype, 1, gate_up.k, 0)
    else:
        o = _result(out, device, gate_up.k, n)
    res = _plain(residual, device, "residual", gate_up.k, n)[0] if residual is not None else None
    if n == 0:
        return out
    if workspace is None:
        workspace = ffn_workspace(gate_up, down, n, top)
    space, size = _space(workspace, device)
    _call(gate_up.lib.velox_hip_expert_ffn, gate_up._index, gate_up._ref, down._ref, first, xr, i, w, n, top, res, o, space, size)
    return out
