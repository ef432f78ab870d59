"""Operators of a gated recurrent mixer beside the GDN-2 layer, over the C ABI
of include/gdn2_mixer.h (no reference counterpart):

  gated_scan, gated_scan_backward           h_t = e^{g_t} h_{t-1} + w_t v_t per channel
  group_norm_act, group_norm_act_backward   group norm over channels-last rows with
                                            an activation or an activated gate

Tensors as in ops.py, of any strides with contiguous channels, in float32 or
bfloat16; log decays, states, weights and their gradients are
float32.  A call runs on its tensors' device, on torch's current stream there;
workspaces come from torch's allocator, so a call may be captured into a graph.
No autograd graph is recorded: a torch.autograd.Function calls the backward with
what it kept of the forward.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _capi as C
from .ops import _stream_of

_SUFFIX = {torch.float32: "_f32", torch.bfloat16: "_bf16"}


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The index of every operand's device; TypeError off the GPU, ValueError for
    several devices."""
    if not first.is_cuda:
        raise TypeError("gdn2_amd operators take device tensors")
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            if not t.is_cuda:
                raise TypeError("gdn2_amd operators take device tensors")
            raise ValueError("the operands are on several devices")
    return index


def _call(fn, args, index: int) -> None:
    if torch.cuda.current_device() == index:
        status = fn(args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            status = fn(args, _stream_of(index))
    if status:
        C.check(status)


def _workspace(args, workspace: Optional[torch.Tensor], need: int, like: torch.Tensor):
    """Sets the workspace of `args`, a new one where none or too small a one is
    given; returns the tensor, to be kept until the call is made."""
    if workspace is not None and (workspace.get_device() != like.get_device() or not workspace.is_contiguous()):
        raise ValueError("workspace must be a contiguous tensor on the operands' device")
    if need == 0:
        return None
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=like.device)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return workspace


# A new result is laid out like its operand; where that would take more than so many
# times the elements' memory (the last token of every sequence of a prompt), like a
# contiguous copy of the operand, which costs two more passes over few elements.
_MOST_GAPS = 4


def _dense_rows(t: torch.Tensor, most: Optional[int] = None) -> torch.Tensor:
    """t, or a copy of it, with contiguous channels, no element of memory in two
    places and, with `most`, elements apart by at most so many times their number
    (what the gradients are laid out like)."""
    if t.is_contiguous():
        return t
    if t.dim() == 4:  # [B, T, H, V] seen as [B, H, T, V]
        (B, H, T, V), st = t.shape, t.stride()
        if st == (T * H * V, V, H * V, 1):
            return t
    if t.shape[-1] != 1 and t.stride(-1) != 1:
        return t.contiguous()
    span = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda x: x[1]):
        if s < span:
            return t.contiguous()
        span = s * n
    return t if most is None or span <= most * t.numel() else t.contiguous()


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """A tensor of t's shape, type and strides."""
    r = torch.empty_like(t)  # (t's strides where no memory is left out between its rows)
    if r.stride() == t.stride():
        return r
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device)


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether tensors of one shape have the same strides (a dimension of one has none
    to speak of)."""
    return a.stride() == b.stride() or all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _in_layout(t: torch.Tensor, ref: torch.Tensor) -> torch.Tensor:
    if _same_layout(t, ref):
        return t
    return _empty_like(ref).copy_(t)


# -- gated scan -----------------------------------------------------------------

def _scan_check(g, v, w, state, cu_seqlens, others=(), states=()):
    """The checks of both directions; the shape of the states.  others: (name,
    tensor) of v's shape and type; states: (name, tensor) beside `state`."""
    ty, shape = v.dtype, v.shape
    if len(shape) != 4:
        raise ValueError("v must be [B, H, T, V]")
    if ty not in _SUFFIX:
        raise TypeError("v must be float32 or bfloat16")
    if g.dtype is not torch.float32:
        raise TypeError("g must be float32")
    gs = g.shape
    if gs != shape and (len(gs) != 4 or gs[:3] != shape[:3] or gs[3] != 1):
        raise ValueError("g must be [B, H, T, V] or [B, H, T, 1]")
    for name, t in (("w", w), *others):
        if t is not None:
            if t.dtype is not ty:
                raise TypeError(f"{name} must have v's type")
            if t.shape != shape:
                raise ValueError(f"{name} must have v's shape")
    n = shape[0]
    if cu_seqlens is not None:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous():
            raise TypeError("cu_seqlens must be a contiguous int32 vector")
        if n != 1:
            raise ValueError("packed sequences need a batch of 1")
        n = cu_seqlens.shape[0] - 1
        if n < 0:
            raise ValueError("cu_seqlens needs at least one offset")
    of_states = (n, shape[1], shape[3])
    for name, t in (("state", state), *states):
        if t is not None:
            if t.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32")
            if t.shape != of_states:
                raise ValueError(f"{name} must be [{n}, H, V]")
    return of_states


def _scan_args(g, v, w, state, new_state, out, cu_seqlens, n):
    B, H, T, V = v.shape
    gb, gh, gt, _ = g.stride()
    vb, vh, vt, _ = v.stride()
    ob, oh, ot, _ = out.stride()
    return C.GatedScanArgs(g.data_ptr(), v.data_ptr(), _p(w), _p(state), _p(new_state), out.data_ptr(), _p(cu_seqlens), B,
                           H, T, V, n, g.shape[3] == 1, gb, gh, gt, vb, vh, vt, ob, oh, ot, None, 0)


_WALK = 12  # tokens without offsets that never need a workspace (gdn2_mixer.h)


def _channels(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def gated_scan(g, v, w=None, state=None, cu_seqlens=None, out=None, new_state=None,
               workspace=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """h_t = e^{g_t} h_{t-1} + w_t v_t for every channel; returns (h [B, H, T, V],
    the state after the last token [N, H, V]).

    g [B, H, T, V], or [B, H, T, 1] for one log decay per head and token; w None
    means 1, state None zeros.  With cu_seqlens (int32 on the device, N + 1 token
    offsets) the one row of the batch holds N sequences, each with its own state;
    rows of out outside all of them are left as they were (as allocated, in a new
    one).  Otherwise N = B.  T = 1 is the serving step.  `out` (no input of the call)
    and `new_state` (which may be `state`) take the results where given."""
    of_states = _scan_check(g, v, w, state, cu_seqlens, (("out", out),) if out is not None else (),
                            (("new_state", new_state),) if new_state is not None else ())
    index = _device(v, g, w, state, cu_seqlens, out, new_state)
    v, g = _channels(v), _channels(g)
    if w is not None and not _same_layout(w, v):
        v = _dense_rows(v, _MOST_GAPS)
        w = _in_layout(w, v)
    if state is not None:
        state = state.contiguous()
    if out is None:
        out = torch.empty_like(v)
    elif _dense_rows(out) is not out:
        raise ValueError("out's channels must be contiguous and its rows apart")
    if new_state is None:
        new_state = v.new_empty(of_states, dtype=torch.float32) if state is None else torch.empty_like(state)
    elif not new_state.is_contiguous():
        raise ValueError("new_state must be contiguous")
    a = _scan_args(g, v, w, state, new_state, out, cu_seqlens, of_states[0])
    L = C.lib()
    keep = None
    if v.shape[2] > _WALK or cu_seqlens is not None:
        keep = _workspace(a, workspace, L.gdn2_gated_scan_workspace_bytes(a), v)
    _call(L.gdn2_gated_scan_fwd_f32 if v.dtype is torch.float32 else L.gdn2_gated_scan_fwd_bf16, a, index)
    del keep
    return out, new_state


def gated_scan_backward(g, v, w, out, d_out, state=None, d_state=None, cu_seqlens=None, workspace=None) -> dict:
    """The gradients of L = <d_out, out> + <d_state, new_state> for gated_scan's
    arguments and its `out`: dict dg (g's shape), dv, dw (v's; dw None without w)
    and dS0 (the state's gradient, also for state None).  Rows outside every
    sequence of cu_seqlens have no gradient: dg, dv and dw are zero there."""
    of_states = _scan_check(g, v, w, state, cu_seqlens, (("out", out), ("d_out", d_out)), (("d_state", d_state),))
    index = _device(v, g, w, state, cu_seqlens, out, d_out, d_state)
    v, g = _dense_rows(v, _MOST_GAPS), _dense_rows(g, _MOST_GAPS)
    if w is not None:
        w = _in_layout(w, v)
    out = _dense_rows(out, _MOST_GAPS)
    d_out = _in_layout(d_out, out)
    state = None if state is None else state.contiguous()
    d_state = None if d_state is None else d_state.contiguous()
    dg, dv, dw = _empty_like(g), _empty_like(v), None if w is None else _empty_like(v)
    like = d_state if state is None else state
    dS0 = v.new_empty(of_states, dtype=torch.float32) if like is None else torch.empty_like(like)
    a = C.GatedScanBwdArgs(_scan_args(g, v, w, state, None, out, cu_seqlens, of_states[0]), d_out.data_ptr(), _p(d_state),
                           dg.data_ptr(), dv.data_ptr(), _p(dw), dS0.data_ptr(), None, 0)
    L = C.lib()
    keep = _workspace(a, workspace, L.gdn2_gated_scan_bwd_workspace_bytes(a), v)
    _call(L.gdn2_gated_scan_bwd_f32 if v.dtype is torch.float32 else L.gdn2_gated_scan_bwd_bf16, a, index)
    del keep
    return {"dg": dg, "dv": dv, "dw": dw, "dS0": dS0}


# -- group norm -------------------------------------------------------------------

_ACTS = {"none": C.ACT_NONE, "silu": C.ACT_SILU, "gelu": C.ACT_GELU}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[N, C] as it is, [N, ..., C] as [N, S, C]."""
    return t if t.dim() <= 3 else t.reshape(t.shape[0], math.prod(t.shape[1:-1]), t.shape[-1])


def _norm_check(x, groups, weight, bias, activation, gate, others=()):
    ty, shape = x.dtype, x.shape
    if len(shape) < 2:
        raise ValueError("x must be [N, C] or [N, ..., C]")
    if ty not in _SUFFIX:
        raise TypeError("x must be float32 or bfloat16")
    if activation not in _ACTS:
        raise ValueError(f"activation must be one of {sorted(_ACTS)}, got {activation!r}")
    if groups < 1 or shape[-1] % groups:
        raise ValueError("the channels must be a multiple of groups")
    for name, t in (("gate", gate), *others):
        if t is not None:
            if t.dtype is not ty:
                raise TypeError(f"{name} must have x's type")
            if t.shape != shape:
                raise ValueError(f"{name} must have x's shape")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            if t.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32")
            if t.shape != shape[-1:]:
                raise ValueError(f"{name} must be [C]")


def _contig(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


def _norm_args(x, groups, weight, bias, eps, activation, gate, y, stats):
    N, S, Ch = x.shape if x.dim() == 3 else (x.shape[0], 1, x.shape[1])
    xs, gs = x.stride(), (0, 0) if gate is None else gate.stride()  # ([N, C]: the one row has no stride to speak of)
    return C.GroupNormArgs(x.data_ptr(), _p(gate), _p(weight), _p(bias), _p(y), _p(stats), N, S, Ch, groups, xs[0], xs[1], gs[0],
                           gs[1], eps, _ACTS[activation], None, 0)


def group_norm_act(x, groups: int, weight=None, bias=None, eps: float = 1e-5, activation: str = "silu", gate=None,
                   return_stats: bool = False, out=None, workspace=None):
    """act(z), or z act(gate) with a gate, of z = group_norm(x) weight + bias.

    x [N, ..., C] with its channels in `groups` runs; a group is normalised over
    the run and all of the dimensions between, for each of the N samples alone.
    [M, C]: each row for itself, as a norm over the heads of a token takes it.
    activation: "silu", "gelu" (with erf) or "none".  weight, bias [C].
    With return_stats also stats [N, groups, 2] (mean, 1 / sqrt(variance + eps)),
    which the backward takes.  `out` takes the result where given (it may be x)."""
    _norm_check(x, groups, weight, bias, activation, gate, (("out", out),) if out is not None else ())
    index = _device(x, weight, bias, gate, out)
    shape, x = x.shape, _dense_rows(_rows(x), _MOST_GAPS if out is None else None)
    gate = None if gate is None else _dense_rows(_rows(gate))
    weight, bias = _contig(weight), _contig(bias)
    y = _empty_like(x) if out is None else _rows(out)
    if out is not None and (y.data_ptr() != out.data_ptr() or not _same_layout(y, x)):
        raise ValueError("out must have x's layout")
    stats = x.new_empty((x.shape[0], groups, 2), dtype=torch.float32) if return_stats else None
    a = _norm_args(x, groups, weight, bias, eps, activation, gate, y, stats)
    L = C.lib()
    keep = _workspace(a, workspace, L.gdn2_group_norm_act_workspace_bytes(a), x)
    _call(L.gdn2_group_norm_act_f32 if x.dtype is torch.float32 else L.gdn2_group_norm_act_bf16, a, index)
    del keep
    y = out if out is not None else y.view(shape) if len(shape) > 3 else y
    return (y, stats) if return_stats else y


def group_norm_act_backward(x, groups: int, stats, d_out, weight=None, bias=None, activation: str = "silu", gate=None,
                            workspace=None) -> dict:
    """The gradients of <d_out, y> for group_norm_act's arguments and the stats it
    returned: dict dx, dgate (None without a gate), dweight and dbias [C] (also for
    weight or bias None: of ones and zeros)."""
    _norm_check(x, groups, weight, bias, activation, gate, (("d_out", d_out),))
    if stats.dtype is not torch.float32:
        raise TypeError("stats must be float32")
    if stats.shape != (x.shape[0], groups, 2):
        raise ValueError("stats must be [N, groups, 2]")
    index = _device(x, weight, bias, gate, d_out, stats)
    shape, x = x.shape, _dense_rows(_rows(x), _MOST_GAPS)
    gate = None if gate is None else _dense_rows(_rows(gate), _MOST_GAPS)
    d_out = _in_layout(_rows(d_out), x)
    weight, bias, stats = _contig(weight), _contig(bias), stats.contiguous()
    dx, dgate = _empty_like(x), None if gate is None else _empty_like(gate)
    dweight = x.new_empty(shape[-1], dtype=torch.float32) if weight is None else torch.empty_like(weight)
    dbias = torch.empty_like(dweight)
    a = C.GroupNormBwdArgs(_norm_args(x, groups, weight, bias, 0.0, activation, gate, None, stats), d_out.data_ptr(),
                           dx.data_ptr(), _p(dgate), dweight.data_ptr(), dbias.data_ptr(), None, 0)
    L = C.lib()
    keep = _workspace(a, workspace, L.gdn2_group_norm_act_bwd_workspace_bytes(a), x)
    _call(L.gdn2_group_norm_act_bwd_f32 if x.dtype is torch.float32 else L.gdn2_group_norm_act_bwd_bf16, a, index)
    del keep
    if len(shape) > 3:
        dx, dgate = dx.view(shape), None if dgate is None else dgate.view(shape)
    return {"dx": dx, "dgate": dgate, "dweight": dweight, "dbias": dbias}
