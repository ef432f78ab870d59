"""What stands around the mixer in a block that is trained and served, over the C
ABI of include/gdn2_block.h (no reference counterpart):

  dropout, dropout_backward              a mask from a counter-based generator that
                                         is formed where it is needed, never stored
  residual_norm, residual_norm_backward  the norm behind a block, its gate, dropout,
                                         the scaled residual and the norm before the
                                         next block
  low_rank_add, low_rank_add_backward    every request's own low-rank adapter beside a
                                         projection that all of them share

Tensors as in mixer.py: any strides with contiguous channels (others are copied),
float32 or bfloat16; weights, statistics and the weights' gradients are float32.  A
call runs on its tensors' device, on torch's current stream there; workspaces come
from torch's allocator, so a call may be captured into a graph.  No autograd graph is
recorded: a torch.autograd.Function calls the backward with what it kept.

A call with dropout takes rows * ceil(C / 4) counters from `offset` on; the same seed
and offset give the same mask in every operator here, for any strides and types.
`rng`, an int64 tensor of two on the device, gives the seed in place of `seed` and is
added to `offset`: a captured graph replayed after a change of it draws another mask.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _capi as C
from .mixer import _SUFFIX, _contig, _call, _device, _p, _same_layout, _workspace
from .ops import _stream_of

_U64 = (1 << 64) - 1


def _drop(p: float, seed: int, offset: int, rng: Optional[torch.Tensor]) -> C.Dropout:
    if not 0.0 <= p <= 1.0:
        raise ValueError("the share to drop must be between 0 and 1")
    if rng is not None and (rng.dtype is not torch.int64 or rng.shape != (2,) or not rng.is_contiguous()):
        raise TypeError("rng must be a contiguous int64 tensor of two: seed and offset")
    return C.Dropout(p, seed & _U64, offset & _U64, _p(rng))


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """The first byte of t's elements and the one behind the last."""
    lo = hi = 0
    for n, s in zip(t.shape, t.stride()):
        lo, hi = (lo, hi + (n - 1) * s) if s >= 0 else (lo + (n - 1) * s, hi)
    e = t.element_size()
    return t.data_ptr() + lo * e, t.data_ptr() + (hi + 1) * e


def _clash(a: Optional[torch.Tensor], b: Optional[torch.Tensor]) -> bool:
    """Whether a write to a may change b: their memory meets, and they are not other
    columns of the same rows."""
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.shape == b.shape and _same_layout(a, b) and a.element_size() == b.element_size():
        n, e = a.shape[-1], a.element_size()
        rows = [s for m, s in zip(a.shape[:-1], a.stride()[:-1]) if m > 1]
        row = math.gcd(*rows) if rows else 0
        if row and (b.data_ptr() - a.data_ptr()) % e == 0:
            return not n <= (b.data_ptr() - a.data_ptr()) // e % row <= row - n
    return True


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no element of memory is in two places of t, by a rule that no dense or
    padded layout fails."""
    span = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n != 1):
        if s < span:
            return False
        span += s * (n - 1)
    return True


def _takes(name: str, t: torch.Tensor, like: torch.Tensor, dtype, own: Optional[torch.Tensor], others) -> None:
    """The checks of a tensor that the caller gives for a result: own, where not None,
    is an operand that it may be; none of the others may share its memory."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}")
    if t.shape != like.shape:
        raise ValueError(f"{name} must have the operand's shape")
    if t.numel() and (t.shape[-1] != 1 and t.stride(-1) != 1 or not _rows_apart(t)):
        raise ValueError(f"{name}'s channels must be contiguous and its rows apart")
    if own is not None and t.data_ptr() == own.data_ptr() and _same_layout(t, own):
        own = None
    if any(_clash(t, o) for o in (own, *others)):
        raise ValueError(f"{name} must not share memory with another operand")


# -- dropout ----------------------------------------------------------------------

def _dropout_check(x, out) -> None:
    if x.dtype not in _SUFFIX:
        raise TypeError("x must be float32 or bfloat16")
    if x.dim() < 1:
        raise ValueError("x must be [..., C]")
    if out is not None:
        _takes("out", out, x, x.dtype, x, ())


def dropout(x, p: float, seed: int = 0, offset: int = 0, rng=None, out=None) -> torch.Tensor:
    """x / (1 - p) where the element is kept, 0 where it is dropped (a share p of them,
    to the nearest 2^-24; p = 1 drops all), for the rows of x [..., C].  `out` takes the
    result where given (it may be x)."""
    d = _drop(p, seed, offset, rng)
    _dropout_check(x, out)
    index = _device(x, rng, out)
    shape, n, ch = x.shape, x.numel(), x.shape[-1]
    if n == 0:
        return torch.empty_like(x) if out is None else out
    if out is not None and _pitch(out) is None:  # rows not evenly apart
        return out.copy_(dropout(x, p, seed, offset, rng))
    sx = _pitch(x)
    if sx is None:
        x, sx = x.contiguous(), ch
    y = torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else out
    fn = C.lib().gdn2_dropout_f32 if x.dtype is torch.float32 else C.lib().gdn2_dropout_bf16
    _call(lambda a, s: fn(x.data_ptr(), y.data_ptr(), n // ch, ch, sx, ch if out is None else _pitch(y), a, s), d, index)
    return y


def _pitch(t: torch.Tensor) -> Optional[int]:
    """How far t's rows are apart, where they are evenly and their channels contiguous."""
    ch = t.shape[-1]
    if t.is_contiguous():
        return ch
    if ch != 1 and t.stride(-1) != 1:
        return None
    dims = [(m, s) for m, s in zip(t.shape[:-1], t.stride()[:-1]) if m != 1]
    for (_, s), (m, inner) in zip(dims, dims[1:]):
        if s != m * inner:
            return None
    return dims[-1][1] if dims else ch


def dropout_backward(d_out, p: float, seed: int = 0, offset: int = 0, rng=None, out=None) -> torch.Tensor:
    """The gradient of x for <d_out, dropout(x, ...)>: the same elements of d_out, by
    the same factor."""
    return dropout(d_out, p, seed, offset, rng, out)


# -- the residual path ----------------------------------------------------------------

_GATES = {"none": C.GATE_NONE, "silu": C.GATE_SILU, "sigmoid": C.GATE_SIGMOID}
_TYPES = {(torch.float32, torch.float32): "_f32", (torch.bfloat16, torch.bfloat16): "_bf16",
          (torch.float32, torch.bfloat16): "_f32_bf16"}


def _residual_check(x, y, gate, post_weight, pre_weight, activation, branch, others) -> int:
    """The checks of both directions; which rows the gate has.  others: (name, tensor,
    type) of x's shape."""
    shape = x.shape
    if len(shape) < 2:
        raise ValueError("x must be [N, C] or [N, ..., C]")
    if (x.dtype, branch) not in _TYPES:
        raise TypeError("the stream and the branch must be float32 or bfloat16, a bfloat16 stream with a bfloat16 branch")
    if activation not in _GATES:
        raise ValueError(f"activation must be one of {sorted(_GATES)}, got {activation!r}")
    for name, t, ty in others:
        if t is not None:
            if t.dtype is not ty:
                raise TypeError(f"{name} must be {ty}")
            if t.shape != shape:
                raise ValueError(f"{name} must have x's shape")
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None:
            if t.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32")
            if t.shape != shape[-1:]:
                raise ValueError(f"{name} must be [C]")
    if y is None and (gate is not None or post_weight is not None):
        raise ValueError("a gate or post_weight needs y")
    if gate is None:
        return C.GATE_ROW
    if gate.dtype is not branch:
        raise TypeError("gate must have y's type")
    gs = gate.shape
    if gs == shape:
        return C.GATE_ROW
    if gs == shape[-1:]:
        return C.GATE_ALL
    if len(shape) > 2 and len(gs) == len(shape) and gs[0] == shape[0] and gs[-1] == shape[-1] and all(n == 1 for n in gs[1:-1]):
        return C.GATE_SAMPLE
    raise ValueError("gate must be [N, ..., C], [N, 1, ..., C] or [C]")


def _three(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """[N, C] as it is, [N, ..., C] as [N, S, C], with contiguous channels."""
    if t is None:
        return None
    if t.dim() > 3:
        t = t.reshape(t.shape[0], math.prod(t.shape[1:-1]), t.shape[-1])
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _ns(t: Optional[torch.Tensor]) -> Tuple[int, int]:
    """The strides of sample and row ([N, C]: one sample's rows)."""
    if t is None:
        return 0, 0
    s = t.stride()
    return (s[0], s[1]) if len(s) == 3 else (0, s[0]) if len(s) == 2 else (0, 0)


def _gate_ns(gate: Optional[torch.Tensor], kind: int) -> Tuple[int, int]:
    return _ns(gate) if kind == C.GATE_ROW else (gate.stride(0), 0) if kind == C.GATE_SAMPLE else (0, 0)


def _sizes(t: torch.Tensor) -> Tuple[int, int, int]:
    s = t.shape
    return (s[0], s[1], s[2]) if len(s) == 3 else (1, s[0], s[1])


def _new(t: torch.Tensor, dtype=None) -> torch.Tensor:
    """A dense tensor of t's shape with contiguous channels, in t's order of rows."""
    r = torch.empty_like(t, dtype=dtype)
    return r if t.shape[-1] == 1 or r.stride(-1) == 1 else torch.empty(t.shape, dtype=r.dtype, device=t.device)


def _seen(t: Optional[torch.Tensor], shape) -> Optional[torch.Tensor]:
    return t if t is None or t.shape == shape else t.view(shape)


def _in_place(t: torch.Tensor) -> torch.Tensor:
    """A caller's tensor for a result as [N, S, C] of the same memory."""
    if t.dim() <= 3:
        return t
    try:
        return t.view(t.shape[0], math.prod(t.shape[1:-1]), t.shape[-1])
    except RuntimeError:
        raise ValueError("a result's rows must be evenly apart within a sample") from None


def residual_norm(x, y=None, gate=None, post_weight=None, pre_weight=None, eps: float = 1e-5, activation: str = "none",
                  residual_scale: float = 1.0, branch_scale: float = 1.0, dropout_p: float = 0.0, seed: int = 0,
                  offset: int = 0, rng=None, return_stats: bool = False, out=None, normed=None):
    """The residual path between two blocks; returns (out, normed):
      p      = y rstd(y) post_weight            (y itself without post_weight)
      out    = residual_scale x + branch_scale dropout(act(gate) p)
      normed = out rstd(out) pre_weight         (None without pre_weight)
      rstd(t) = 1 / sqrt(mean(t^2) + eps), for each row of C channels.

    x [N, ..., C] is the residual stream, y the block's output (None before the first
    block: out is residual_scale x).  gate: like y, [N, 1, ..., C] (one row a sample) or
    [C]; activation of it: "none", "sigmoid" or "silu".  The stream may be float32 with y,
    gate and normed in bfloat16.  normed is formed from out before its rounding.  With
    return_stats also stats [N, ..., 2] (rstd(y), rstd(out); 0 where not taken), which
    the backward takes.  `out` and `normed` take the results where given (out may be x,
    normed may be y; without y, normed's type is that of the branch)."""
    branch = y.dtype if y is not None else normed.dtype if normed is not None else x.dtype
    kind = _residual_check(x, y, gate, post_weight, pre_weight, activation, branch, (("y", y, branch),))
    drop = _drop(dropout_p, seed, offset, rng)
    if y is None and dropout_p:
        raise ValueError("dropout needs y")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if normed is not None and pre_weight is None:
        raise ValueError("normed needs pre_weight")
    if out is not None:
        _takes("out", out, x, x.dtype, x, (y, gate, normed, post_weight, pre_weight))
    if normed is not None:
        _takes("normed", normed, x, branch, y, (x, gate, out, post_weight, pre_weight))
    index = _device(x, y, gate, post_weight, pre_weight, rng, out, normed)
    shape = x.shape
    x, y, gate = _three(x), _three(y), _three(gate)
    post_weight, pre_weight = _contig(post_weight), _contig(pre_weight)
    o = _new(x) if out is None else _in_place(out)
    n = None if pre_weight is None else _new(x if y is None else y, branch) if normed is None else _in_place(normed)
    stats = x.new_empty((*shape[:-1], 2), dtype=torch.float32) if return_stats else None
    if x.numel():
        a = C.ResidualNormArgs(x.data_ptr(), _p(y), _p(gate), _p(post_weight), _p(pre_weight), o.data_ptr(), _p(n), _p(stats),
                               *_sizes(x), *_ns(x), *_ns(y), *_gate_ns(gate, kind), *_ns(o), *_ns(n), eps, residual_scale,
                               branch_scale, _GATES[activation], kind, drop)
        _call(getattr(C.lib(), "gdn2_residual_norm" + _TYPES[x.dtype, branch]), a, index)
    elif stats is not None and stats.numel():  # rows of no channels: the mean of nothing
        for i, taken in enumerate((post_weight is not None, pre_weight is not None)):
            stats[..., i] = math.nan if taken else 0.0
    o = out if out is not None else _seen(o, shape)
    n = normed if normed is not None else _seen(n, shape)
    return (o, n, stats) if return_stats else (o, n)


def residual_norm_backward(out, y, stats, d_out=None, d_normed=None, gate=None, post_weight=None, pre_weight=None,
                           activation: str = "none", residual_scale: float = 1.0, branch_scale: float = 1.0,
                           dropout_p: float = 0.0, seed: int = 0, offset: int = 0, rng=None, workspace=None) -> dict:
    """The gradients of <d_out, out> + <d_normed, normed> for residual_norm's arguments
    and the out and stats it returned: dict dx, dy, dgate (in gate's shape: where rows
    share one, the sum over them), dpost and dpre [C]; None for what was not given.
    d_out None: zero.  d_normed comes with pre_weight and only then."""
    branch = y.dtype if y is not None else d_normed.dtype if d_normed is not None else out.dtype
    kind = _residual_check(out, y, gate, post_weight, pre_weight, activation, branch,
                           (("y", y, branch), ("d_out", d_out, out.dtype), ("d_normed", d_normed, branch)))
    drop = _drop(dropout_p, seed, offset, rng)
    if y is None and dropout_p:
        raise ValueError("dropout needs y")
    if (d_normed is None) != (pre_weight is None):
        raise ValueError("d_normed and pre_weight go together")
    if stats is not None:
        if stats.dtype is not torch.float32:
            raise TypeError("stats must be float32")
        if stats.shape != (*out.shape[:-1], 2):
            raise ValueError("stats must be [N, ..., 2]")
    elif pre_weight is not None or post_weight is not None:
        raise ValueError("a norm's backward needs stats")
    index = _device(out, y, stats, d_out, d_normed, gate, post_weight, pre_weight, rng)
    shape, gate_shape = out.shape, None if gate is None else gate.shape
    out, y, gate, d_out, d_normed = _three(out), _three(y), _three(gate), _three(d_out), _three(d_normed)
    post_weight, pre_weight, stats = _contig(post_weight), _contig(pre_weight), _contig(stats)
    dx, dy, dgate = _new(out), None if y is None else _new(y), None if gate is None else _new(gate)
    dpost = None if post_weight is None else torch.empty_like(post_weight)
    dpre = None if pre_weight is None else torch.empty_like(pre_weight)
    if out.numel():
        f = C.ResidualNormArgs(None, _p(y), _p(gate), _p(post_weight), _p(pre_weight), out.data_ptr(), None, _p(stats),
                               *_sizes(out), 0, 0, *_ns(y), *_gate_ns(gate, kind), *_ns(out), 0, 0, 0.0, residual_scale,
                               branch_scale, _GATES[activation], kind, drop)
        a = C.ResidualNormBwdArgs(f, _p(d_out), _p(d_normed), dx.data_ptr(), _p(dy), _p(dgate), _p(dpost), _p(dpre),
                                  *_ns(d_out), *_ns(d_normed), *_ns(dx), *_ns(dy), *_gate_ns(dgate, kind), None, 0)
        L = C.lib()
        keep = _workspace(a, workspace, L.gdn2_residual_norm_bwd_workspace_bytes(a), out)
        _call(getattr(L, "gdn2_residual_norm_bwd" + _TYPES[out.dtype, branch]), a, index)
        del keep
    else:
        for t in (dgate, dpost, dpre):
            if t is not None:
                t.zero_()
    return {"dx": _seen(dx, shape), "dy": _seen(dy, shape), "dgate": _seen(dgate, gate_shape), "dpost": dpost, "dpre": dpre}


# -- low-rank adapters ----------------------------------------------------------------

def _adapters_check(x, a, b, adapters, scale, cu_seqlens, others) -> None:
    """The checks of both directions.  others: (name, tensor, channels, type)."""
    ty, shape = x.dtype, x.shape
    if len(shape) not in (2, 3):
        raise ValueError("x must be [N, D] or [B, T, D]")
    if ty not in _SUFFIX:
        raise TypeError("x must be float32 or bfloat16")
    for name, t, ch in (("a", a, shape[-1]), ("b", b, None)):
        if t.dtype is not ty:
            raise TypeError(f"{name} must have x's type")
        if t.dim() != 3 or ch is not None and t.shape[2] != ch:
            raise ValueError(f"{name} must be [L, R, {'D' if ch is not None else 'O'}]")
    if a.shape[:2] != b.shape[:2]:
        raise ValueError("a and b must have the same adapters and ranks")
    for name, t, ch, dtype in others:
        if t is not None:
            if t.dtype is not dtype:
                raise TypeError(f"{name} must be {dtype}")
            if t.shape != (*shape[:-1], ch):
                raise ValueError(f"{name} must be {tuple((*shape[:-1], ch))}")
    n = shape[0]
    if cu_seqlens is not None:
        if cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous():
            raise TypeError("cu_seqlens must be a contiguous int32 vector")
        if len(shape) != 3 or n != 1:
            raise ValueError("packed requests need a batch of 1")
        n = cu_seqlens.shape[0] - 1
        if n < 0:
            raise ValueError("cu_seqlens needs at least one offset")
    if adapters.dtype is not torch.int32 or not adapters.is_contiguous():
        raise TypeError("adapters must be a contiguous int32 vector")
    if adapters.shape != (n,):
        raise ValueError(f"adapters must be [{n}], one of each request")
    if scale is not None:
        if scale.dtype is not torch.float32:
            raise TypeError("scale must be float32")
        if scale.shape != a.shape[:1]:
            raise ValueError("scale must be [L]")


def _rowed(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy, with contiguous channels and its rows no further apart than the
    kernels take."""
    near = t.dim() == 2 or t.shape[1] <= 1 or t.stride(1) < 1 << 24
    return t if near and (t.shape[-1] == 1 or t.stride(-1) == 1) else t.contiguous()


def _bt(t: Optional[torch.Tensor]) -> Tuple[int, int]:
    """The strides of batch and token ([N, D]: a token each)."""
    if t is None:
        return 0, 0
    s = t.stride()
    return (s[0], s[1] if t.shape[1] > 1 else 0) if len(s) == 3 else (s[0], 0)


def _low_rank_args(x, a, b, y, out, adapters, scale, cu_seqlens, hidden):
    B, T = x.shape[0], x.shape[1] if x.dim() == 3 else 1
    L, R, D = a.shape
    return C.LowRankArgs(_p(x), _p(a), _p(b), _p(y), _p(out), _p(adapters), _p(cu_seqlens), _p(scale), _p(hidden), B, T, D,
                         b.shape[2], R, L, 0 if cu_seqlens is None else cu_seqlens.shape[0] - 1, *_bt(x), *_bt(y), *_bt(out),
                         a.stride(0), a.stride(1) if R > 1 else 0, b.stride(0), b.stride(1) if R > 1 else 0, None, 0)


def low_rank_add(y, x, a, b, adapters, scale=None, cu_seqlens=None, return_hidden: bool = False, out=None, workspace=None):
    """y + scale_l (x a_l^T) b_l, with l the adapter of each row's request: what the
    low-rank adapters of many requests add to the output y of a projection that they
    share.

    x [B, T, D] (or [N, D], a token each), y [B, T, O]; a [L, R, D], b [L, R, O]: the
    adapters' vectors, rank by rank (an adapter of fewer ranks is padded with zeros).
    adapters: int32 on the device, one of each request; outside [0, L) none, and the
    row is y's.  scale [L] or None (1).  The requests are the batch entries, or with
    cu_seqlens (int32 on the device, N + 1 token offsets) runs of the one row; rows
    outside all of them have no adapter.  x a_l^T is not rounded to x's type on its way.
    With return_hidden also it, [B, T, R] float32 (0 without an adapter), which the
    backward takes.  `out` takes the result where given (it may be y)."""
    _adapters_check(x, a, b, adapters, scale, cu_seqlens, (("y", y, b.shape[2], x.dtype),))
    if out is not None:
        _takes("out", out, y, x.dtype, y, (x, a, b, adapters, scale, cu_seqlens))
    index = _device(x, y, a, b, adapters, scale, cu_seqlens, out)
    x, y, a, b, scale = _rowed(x), _rowed(y), _rowed(a), _rowed(b), _contig(scale)
    o = _new(y) if out is None else out
    hidden = x.new_empty((*x.shape[:-1], a.shape[1]), dtype=torch.float32) if return_hidden else None
    if x.shape[:-1].numel():
        args = _low_rank_args(x, a, b, y, o, adapters, scale, cu_seqlens, hidden)
        L = C.lib()
        keep = _workspace(args, workspace, L.gdn2_low_rank_add_workspace_bytes(args), x)
        _call(L.gdn2_low_rank_add_f32 if x.dtype is torch.float32 else L.gdn2_low_rank_add_bf16, args, index)
        del keep
    return (o, hidden) if return_hidden else o


def low_rank_add_backward(x, a, b, adapters, hidden, d_out, scale=None, cu_seqlens=None, dx=None, workspace=None) -> dict:
    """The gradients of <d_out, low_rank_add(y, x, ...)> for its arguments and the hidden
    it returned (y's is d_out itself): dict dx (0 in rows without an adapter; where a
    `dx` is given, the shared projection's gradient of x, it is added to that, in place),
    da [L, R, D] and db [L, R, O] in float32."""
    _adapters_check(x, a, b, adapters, scale, cu_seqlens,
                    (("d_out", d_out, b.shape[2], x.dtype), ("hidden", hidden, a.shape[1], torch.float32)))
    if dx is not None:
        _takes("dx", dx, x, x.dtype, None, (x, a, b, adapters, hidden, d_out, scale, cu_seqlens))
    index = _device(x, a, b, adapters, hidden, d_out, scale, cu_seqlens, dx)
    x, a, b, d_out, scale, hidden = _rowed(x), _rowed(a), _rowed(b), _rowed(d_out), _contig(scale), hidden.contiguous()
    into = _new(x) if dx is None else dx
    da, db = (torch.empty(t.shape, dtype=torch.float32, device=t.device) for t in (a, b))
    if x.shape[:-1].numel() or da.numel() or db.numel():
        args = C.LowRankBwdArgs(_low_rank_args(x, a, b, None, None, adapters, scale, cu_seqlens, hidden), _p(d_out), _p(into),
                                _p(da), _p(db), dx is not None, *_bt(d_out), *_bt(into), None, 0)
        L = C.lib()
        keep = _workspace(args, workspace, L.gdn2_low_rank_add_bwd_workspace_bytes(args), x)
        _call(L.gdn2_low_rank_add_bwd_f32 if x.dtype is torch.float32 else L.gdn2_low_rank_add_bwd_bf16, args, index)
        del keep
    return {"dx": into, "da": da, "db": db}
