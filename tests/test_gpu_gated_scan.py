"""gated_scan and gated_scan_backward against their plain 64-bit forms, from one
token to several tiles a sequence, every form of their arguments."""
import itertools

import numpy as np
import pytest

import mixer_testutil as M

pytestmark = pytest.mark.gpu


def _types(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _np(t):
    return t.detach().double().cpu().numpy()


def _make(gpu, seed, B, T, H, V, ty, per_head, w, state, N=None, slow=False):
    """Operands in the layout a projection leaves ([B, T, H, V] seen as [B, H, T, V])."""
    import torch

    r = torch.Generator().manual_seed(seed)
    tt = _types(ty)
    rows = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    lo, hi = (-9.0, -4.0) if slow else (-7.0, 1.0)
    g = -torch.exp(torch.rand(B, T, H, 1 if per_head else V, generator=r) * (hi - lo) + lo)
    d = {"g": g.to(gpu).transpose(1, 2), "v": rows(B, T, H, V).to(gpu, tt).transpose(1, 2),
         "w": torch.sigmoid(rows(B, T, H, V)).to(gpu, tt).transpose(1, 2) if w else None,
         "state": rows(N or B, H, V).to(gpu) if state else None}
    return d


def _flat(t):
    """[B, H, T, V] -> numpy [B, T, H, V]"""
    return _np(t).transpose(0, 2, 1, 3)


def _scan64(d, N, bounds=None):
    H, V = d["v"].shape[1], d["v"].shape[3]
    u = _flat(d["v"]) * (_flat(d["w"]) if d["w"] is not None else 1.0)
    g = np.broadcast_to(_flat(d["g"]), u.shape)
    h0 = _np(d["state"]) if d["state"] is not None else np.zeros((N, H, V))
    return M.scan64(g, u, h0, bounds)


def _check_forward(d, out, new, N, ty, bounds=None):
    h, last, err, last_err = _scan64(d, N, bounds)
    got = _flat(out)
    inside = ~np.isnan(h)
    a = M.worst(got[inside], h[inside], err[inside], M.HALF[ty])
    b = M.worst(_np(new), last, last_err, 0)
    assert a <= 1 and b <= 1, (a, b)
    return inside


CASES = [  # B, T, H, V
    (1, 1, 1, 1), (3, 1, 2, 128), (2, 7, 3, 5), (2, 8, 2, 4), (1, 9, 2, 64), (2, 31, 1, 33), (1, 64, 2, 36),
    (2, 65, 3, 12), (1, 127, 1, 100), (1, 128, 2, 32), (1, 129, 4, 96), (2, 256, 1, 128), (1, 257, 2, 40),
    (1, 1000, 1, 7), (2, 1025, 2, 36), (1, 2500, 1, 64), (5, 300, 2, 1), (1, 3000, 3, 128), (2, 2400, 1, 96), (1, 4500, 1, 40),
]


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,H,V", CASES)
def test_forward(gpu, B, T, H, V, ty):
    import torch

    import gdn2_amd as G

    for k, (per_head, w, state) in enumerate(itertools.product((False, True), repeat=3)):
        print("forward", B, T, H, V, ty, per_head, w, state, flush=True)
        d = _make(gpu, 100 * T + V + k, B, T, H, V, ty, per_head, w, state, slow=k % 3 == 0)
        out, new = G.gated_scan(**d)
        torch.cuda.synchronize()
        assert out.dtype == _types(ty) and out.shape == (B, H, T, V) and new.shape == (B, H, V)
        assert _check_forward(d, out, new, B, ty).all()


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,T", [(1, 12), (1, 13), (80, 13), (80, 32), (80, 33)])
def test_few_tokens(gpu, B, T, ty):
    """Lengths at which the walk over the tokens gives way to tiles, with few rows
    and with more than run at once."""
    import torch

    import gdn2_amd as G

    for per_head, V in ((False, 128), (True, 128), (False, 127)):
        d = _make(gpu, T + B, B, T, 16, V, ty, per_head, True, True)
        out, new = G.gated_scan(**d)
        torch.cuda.synchronize()
        assert _check_forward(d, out, new, B, ty).all()


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,H,V", CASES)
def test_backward(gpu, B, T, H, V, ty):
    import torch

    import gdn2_amd as G

    for k, (per_head, w, state) in enumerate(itertools.product((False, True), repeat=3)):
        print("backward", B, T, H, V, ty, per_head, w, state, flush=True)
        d = _make(gpu, 100 * T + V + k, B, T, H, V, ty, per_head, w, state, slow=k % 3 == 0)
        out, _ = G.gated_scan(**d)
        d_out = torch.randn(B, T, H, V, device=gpu).to(_types(ty)).transpose(1, 2)
        d_state = torch.randn(B, H, V, device=gpu) if state else None
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=d_state)
        torch.cuda.synchronize()
        _check_backward(d, out, d_out, d_state, r, B, ty)


def _check_backward(d, out, d_out, d_state, r, N, ty, bounds=None):
    H, V = d["v"].shape[1], d["v"].shape[3]
    zeros = np.zeros((N, H, V))
    v, w = _flat(d["v"]), _flat(d["w"]) if d["w"] is not None else None
    g = np.broadcast_to(_flat(d["g"]), v.shape)
    want, err = M.scan_bwd64(g, v, w, _flat(out), _flat(d_out), _np(d["state"]) if d["state"] is not None else zeros,
                             _np(d_state) if d_state is not None else zeros, bounds)
    if d["g"].shape[3] == 1:  # a sum of V terms: V roundings of their magnitudes at most
        err["dg"] = (err["dg"] + V * M.EPS * np.abs(want["dg"])).sum(3, keepdims=True)
        want["dg"] = want["dg"].sum(3, keepdims=True)
    assert r["dg"].shape == d["g"].shape and r["dv"].shape == d["v"].shape
    assert (r["dw"] is None) == (w is None)
    for n in ("dg", "dv", "dw", "dS0"):
        if r[n] is None:
            continue
        got = _np(r[n]) if n == "dS0" else _flat(r[n])
        e = M.worst(got, want[n], err[n], M.HALF[ty] if n in ("dv", "dw") else 0)
        assert e <= 1, (n, e)


PACKED = [  # offsets, T: empty sequences, rows before and behind them, many in a tile, one over many tiles
    ([0, 5], 5), ([0, 1, 2, 3, 4], 4), ([0, 0, 3, 3, 10, 10], 10), ([2, 9, 40], 50), ([0, 700], 1000),
    ([0, 63, 64, 65, 300, 301, 900], 901), ([0, 256, 512, 513], 513), ([0, 1, 1300], 1400), ([0] * 5, 20),
    ([17, 17, 17], 30), (list(range(0, 401, 2)), 403),
]


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("bounds,T", PACKED)
def test_packed(gpu, bounds, T, ty):
    """Forward and backward of packed sequences.  What lies outside the sequences
    is NaN in every input and must reach nothing; rows of out there stay."""
    import torch

    import gdn2_amd as G

    N = len(bounds) - 1
    cu = torch.tensor(bounds, dtype=torch.int32, device=gpu)
    outside = torch.ones(T, dtype=torch.bool)
    outside[bounds[0]:bounds[-1]] = False
    outside = outside.to(gpu)
    for k, (per_head, w, state, V) in enumerate([(False, True, True, 40), (True, True, False, 36), (True, False, True, 128),
                                                 (False, False, True, 7), (True, True, True, 3)]):
        print("packed", bounds[:8], T, ty, per_head, w, state, V, flush=True)
        d = _make(gpu, 31 * T + k, 1, T, 2, V, ty, per_head, w, state, N=N)
        for n in ("g", "v", "w"):
            if d[n] is not None:
                d[n][:, :, outside] = float("nan")
        out = torch.full((1, T, 2, V), 7.0, device=gpu, dtype=_types(ty)).transpose(1, 2)
        res, new = G.gated_scan(**d, cu_seqlens=cu, out=out)
        torch.cuda.synchronize()
        assert res is out and new.shape == (N, 2, V)
        inside = _check_forward(d, out, new, N, ty, bounds)
        assert (_flat(out)[~inside] == 7.0).all()

        d_out = torch.randn(1, T, 2, V, device=gpu).to(_types(ty)).transpose(1, 2)
        d_out[:, :, outside] = float("nan")
        out[:, :, outside] = float("nan")
        d_state = torch.randn(N, 2, V, device=gpu) if state else None
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=d_state, cu_seqlens=cu)
        torch.cuda.synchronize()
        for n in ("dg", "dv", "dw"):
            assert r[n] is None or (r[n][:, :, outside] == 0).all()
        _check_backward(d, out, d_out, d_state, r, N, ty, bounds)


def test_packed_equals_separate_calls(gpu):
    """The rows of packed sequences equal those of one call each, to rounding."""
    import torch

    import gdn2_amd as G

    bounds = [0, 300, 301, 900]
    d = _make(gpu, 5, 1, 900, 2, 64, "f32", False, True, True, N=3)
    cu = torch.tensor(bounds, dtype=torch.int32, device=gpu)
    out, new = G.gated_scan(**d, cu_seqlens=cu)
    for n in range(3):
        part = {k: (x[:, :, bounds[n]:bounds[n + 1]] if k != "state" else x[n:n + 1]) for k, x in d.items()}
        o, s = G.gated_scan(**part)
        h, last, err, last_err = _scan64(part, 1)
        assert M.worst(_flat(o), _flat(out[:, :, bounds[n]:bounds[n + 1]]), 2 * err, 0) <= 1
        assert M.worst(_np(s), _np(new[n:n + 1]), 2 * last_err, 0) <= 1


def test_steps_equal_one_call(gpu):
    """Token by token with the state handed on in place = one call over the prompt."""
    import torch

    import gdn2_amd as G

    d = _make(gpu, 6, 3, 40, 2, 96, "f32", True, True, True)
    out, new = G.gated_scan(**d)
    h, last, err, last_err = _scan64(d, 3)
    state, got = d["state"].clone(), []
    for t in range(40):
        o, s = G.gated_scan(d["g"][:, :, t:t + 1], d["v"][:, :, t:t + 1], d["w"][:, :, t:t + 1], state, new_state=state)
        assert s is state
        got.append(o)
    assert M.worst(_flat(torch.cat(got, 2)), h, err, 0) <= 1 and M.worst(_np(state), last, last_err, 0) <= 1
    assert M.worst(_flat(out), h, err, 0) <= 1


@pytest.mark.parametrize("T", [5, 70, 3000])
def test_state_in_place(gpu, T):
    import torch

    import gdn2_amd as G

    d = _make(gpu, 8, 2, T, 2, 64, "f32", False, True, True)
    out, new = G.gated_scan(**d)
    state = d["state"].clone()
    o2, s2 = G.gated_scan(d["g"], d["v"], d["w"], state, new_state=state)
    assert s2 is state and torch.equal(out, o2) and torch.equal(new, state)


def test_same_bits_every_time(gpu):
    """Tiles join in one order whatever their timing: 160 tiles a chain, with and
    without other work on the device."""
    import torch

    import gdn2_amd as G

    d = _make(gpu, 9, 1, 40000, 2, 64, "bf16", True, True, True)
    out, new = G.gated_scan(**d)
    d_out = torch.randn_like(out)
    first = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=new)
    side, a = torch.cuda.Stream(), torch.randn(4096, 4096, device=gpu)
    for i in range(6):
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(4):
                    a = torch.tanh(a)
        o, s = G.gated_scan(**d)
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=new)
        torch.cuda.synchronize()
        assert torch.equal(o, out) and torch.equal(s, new)
        assert all(torch.equal(r[n], first[n]) for n in first)


def test_special_values(gpu):
    """g = -inf forgets the state, infinities and NaN included; a NaN stays in its
    channel and sequence; a growing run whose decay overflows keeps zeros zero."""
    import torch

    import gdn2_amd as G

    T, V = 700, 8
    z = lambda *s: torch.zeros(*s, device=gpu)  # noqa: E731
    for bounds in (None, [0, 290, 310, 700]):
        g, v = z(1, 1, T, V) - 0.01, z(1, 1, T, V) + 1.0
        v[0, 0, 3, 1] = float("nan")
        v[0, 0, 4, 2] = float("inf")
        g[0, 0, 600] = float("-inf")
        st = z(1 if bounds is None else 3, 1, V)
        st[:, 0, 3] = float("inf")
        cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu)
        out, new = G.gated_scan(g, v, None, st, cu_seqlens=cu)
        torch.cuda.synchronize()
        assert torch.isnan(out[0, 0, 3:290, 1]).all() and torch.isinf(out[0, 0, 4:290, 2]).all()
        assert (out[0, 0, 600] == 1).all() and torch.isfinite(out[0, 0, 600:]).all()
        if bounds is None:
            assert torch.isnan(out[0, 0, 3:600, 1]).all()
        else:  # the next sequences
            assert torch.isfinite(out[0, 0, 290:, 1:3]).all() and torch.isinf(out[0, 0, :600, 3]).all()
        assert torch.isfinite(out[0, 0, :, 0]).all() and torch.isfinite(out[0, 0, :, 4:]).all()
        assert torch.isfinite(new[-1]).all()
    out, new = G.gated_scan(z(1, 1, T, V) + 2.0, z(1, 1, T, V))
    assert (out == 0).all() and (new == 0).all()
    # e^{2 t} of a state that starts at 1e-38: finite for 87 tokens
    out, _ = G.gated_scan(z(1, 1, 80, V) + 2.0, z(1, 1, 80, V), None, z(1, 1, V) + 1e-38)
    want = 1e-38 * np.exp(2.0 * np.arange(1, 81))
    assert np.abs(_np(out)[0, 0, :, 0] / want - 1).max() < 1e-4


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("T", [3, 40, 700])
def test_decays_at_the_borders(gpu, T, ty):
    """Log decays of either zero, the smallest numbers, and both sides of where the
    decay's form changes, among ordinary ones; values and gradients."""
    import torch

    import gdn2_amd as G

    edge = torch.tensor([-0.0, 0.0, -1e-45, -1e-38, -2e-30, -1e-9, -0.125, -0.12499999, -0.12500001, -1e-3], device=gpu)
    for per_head, V in ((False, 64), (True, 64), (False, 5), (True, 36)):
        d = _make(gpu, 31 + T, 2, T, 3, V, ty, per_head, True, True)
        g = d["g"].clone()
        pick = torch.randint(0, 2 * len(edge), g.shape, device=gpu)
        d["g"] = torch.where(pick < len(edge), edge[pick.clamp(max=len(edge) - 1)], g)
        out, new = G.gated_scan(**d)
        assert _check_forward(d, out, new, 2, ty).all()
        d_out, d_state = torch.randn_like(out), torch.randn_like(new)
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=d_state)
        _check_backward(d, out, d_out, d_state, r, 2, ty)
        keep = {n: t for n, t in d.items() if n != "g"}
        zeros = G.gated_scan(torch.zeros_like(d["g"]), **keep), G.gated_scan(-torch.zeros_like(d["g"]), **keep)
        assert all(torch.equal(a, b) for a, b in zip(*zeros))


def test_slow_decay_keeps_its_digits(gpu):
    """A constant log decay of -2^-13 over 30000 tokens.  The state's own rounding
    is half a step of it a token, which decays too: after many tokens at most
    2^13 half steps if all were of one sign (their random sum is 2^6.5).  A rounded
    e^g would be off by up to 2^-24 at every token, the same way: 2^-11 of h."""
    import torch

    import gdn2_amd as G

    T = 30000
    g = torch.full((1, 1, T, 4), -2.0 ** -13, device=gpu)
    v = torch.randn(1, 1, T, 4, device=gpu).abs()
    out, _ = G.gated_scan(g, v)
    h, _, _, _ = M.scan64(_flat(g), _flat(v), np.zeros((1, 1, 4)))
    rel = np.abs(_flat(out) - h) / h
    assert rel.max() < 2.0 ** -24 * 2 ** 6.5 * 6, rel.max()  # (six deviations of that random sum)


def test_layouts(gpu):
    """Head-major, sliced, unaligned and broadcast operands give what contiguous
    ones give, and nothing outside out's view is written."""
    import torch

    import gdn2_amd as G

    B, T, H, V = 2, 150, 3, 32
    d = _make(gpu, 12, B, T, H, V, "f32", False, True, True)
    out, new = G.gated_scan(**d)
    d_out = torch.randn_like(out)
    ref = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"])

    def inside(x, lead):  # x within a larger buffer, `lead` elements from an aligned place
        big = torch.full((B, H, T, V + 9), 3.0, device=gpu, dtype=x.dtype)
        view = big[..., lead:lead + V]
        view.copy_(x)
        return view

    forms = {
        "head-major": {n: d[n].contiguous() for n in "gvw"},
        "aligned slice": {n: inside(d[n], 0) for n in "gvw"},
        "unaligned slice": {n: inside(d[n], 1) for n in "gvw"},
        "mixed": {"g": d["g"], "v": d["v"].contiguous(), "w": inside(d["w"], 3)},
        "channels strided": {"g": d["g"], "v": torch.stack([d["v"]] * 2, -1)[..., 0], "w": d["w"]},
    }
    for name, f in forms.items():
        o, s = G.gated_scan(f["g"], f["v"], f["w"], d["state"])
        _check_forward({**f, "state": d["state"]}, o, s, B, "f32")
        r = G.gated_scan_backward(f["g"], f["v"], f["w"], o, d_out, d["state"])
        _check_backward({**f, "state": d["state"]}, o, d_out, None, r, B, "f32")
    big = torch.full((B, T + 4, H, V + 8), 5.0, device=gpu)
    view = big[:, 2:T + 2, :, 4:V + 4].transpose(1, 2)
    o, s = G.gated_scan(**d, out=view)
    assert o is view and torch.equal(o, out) and torch.equal(s, new)
    view.fill_(5.0)
    assert (big == 5.0).all()
    one = torch.randn(B, 1, T, V, device=gpu).expand(B, H, T, V)  # one v for all heads
    o, s = G.gated_scan(d["g"], one, None, d["state"])
    _check_forward({"g": d["g"], "v": one, "w": None, "state": d["state"]}, o, s, B, "f32")
    r = G.gated_scan_backward(d["g"], one, None, o, d_out, d["state"])
    _check_backward({"g": d["g"], "v": one, "w": None, "state": d["state"]}, o, d_out, None, r, B, "f32")
    assert ref["dg"].stride() == d["g"].stride()


def test_offsets_past_32_bits(gpu):
    """Token rows further apart than 2^31 elements."""
    import torch

    import gdn2_amd as G

    T, V, st = 12, 64, (1 << 28) + 64
    view, res = (torch.as_strided(torch.empty((T - 1) * st + V, dtype=torch.bfloat16, device=gpu), (1, 1, T, V),
                                  (st, st, st, 1)) for _ in range(2))
    v = torch.randn(1, 1, T, V, device=gpu).bfloat16()
    view.copy_(v)
    g = -torch.rand(1, 1, T, 1, device=gpu)
    o1, s1 = G.gated_scan(g, v)
    o2, s2 = G.gated_scan(g, view, out=res)
    assert torch.equal(o1, o2) and torch.equal(s1, s2)


def test_no_tokens(gpu):
    import torch

    import gdn2_amd as G

    v = torch.empty(2, 3, 0, 8, device=gpu)
    st = torch.randn(2, 3, 8, device=gpu)
    out, new = G.gated_scan(v, v, v, st)
    assert out.shape == v.shape and torch.equal(new, st)
    _, new = G.gated_scan(v, v)
    assert (new == 0).all()
    r = G.gated_scan_backward(v, v, v, v, v, st, d_state=st)
    assert torch.equal(r["dS0"], st) and r["dw"].shape == v.shape
    v = torch.empty(0, 3, 5, 8, device=gpu)
    assert G.gated_scan(v, v)[1].shape == (0, 3, 8)
    v = torch.randn(1, 3, 5, 8, device=gpu)
    out, new = G.gated_scan(v, v, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=gpu), out=v.clone())
    assert torch.equal(out, v) and new.shape == (0, 3, 8)


@pytest.mark.parametrize("T", [5, 700])
def test_gradients_of_nothing_are_zero(gpu, T):
    """No sequence, and heads of no channels: the gradients that there are are zero."""
    import torch

    import gdn2_amd as G

    for g_channels in (1, 8):
        v, g = torch.randn(1, 3, T, 8, device=gpu), -torch.rand(1, 3, T, g_channels, device=gpu)
        torch.empty(1 << 22, device=gpu).fill_(7.0)  # (what the results' memory held before)
        cu = torch.zeros(1, dtype=torch.int32, device=gpu)
        r = G.gated_scan_backward(g, v, v, v, v, cu_seqlens=cu)
        assert all((r[n] == 0).all() for n in ("dg", "dv", "dw")) and r["dS0"].shape == (0, 3, 8)
    none, g = torch.empty(2, 3, T, 0, device=gpu), -torch.rand(2, T, 3, 1, device=gpu).transpose(1, 2)
    torch.empty(1 << 22, device=gpu).fill_(7.0)
    assert G.gated_scan(g, none)[0].shape == none.shape
    r = G.gated_scan_backward(g, none, None, none, none)
    assert r["dg"].shape == g.shape and (r["dg"] == 0).all()


@pytest.mark.parametrize("T", [5, 200])
def test_expanded_operands(gpu, T):
    """Operands that several batches or tokens share in memory."""
    import torch

    import gdn2_amd as G

    for per_head in (False, True):
        d = _make(gpu, 17, 3, T, 2, 64, "f32", per_head, True, True)
        for share in (("v",), ("w",), ("g",), ("v", "w"), ("g", "v", "w")):
            for dim in (0, 2):
                e = {n: t.narrow(dim, 0, 1).expand(t.shape) if n in share else t for n, t in d.items()}
                c = {n: t.contiguous() for n, t in e.items()}
                got, want = G.gated_scan(**e), G.gated_scan(**c)
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (share, dim)
                dy = want[0][:1].expand(want[0].shape)
                got = G.gated_scan_backward(e["g"], e["v"], e["w"], want[0], dy, e["state"])
                want = G.gated_scan_backward(c["g"], c["v"], c["w"], want[0], dy.contiguous(), c["state"])
                assert all(torch.equal(got[n], want[n]) for n in want), (share, dim)
        h = G.gated_scan(**d)[0]
        dy = torch.randn_like(h)
        same = h[:1].expand(h.shape)  # (an `out` of equal batches)
        got = G.gated_scan_backward(d["g"], d["v"], d["w"], same, dy)
        want = G.gated_scan_backward(d["g"], d["v"], d["w"], same.contiguous(), dy)
        assert all(torch.equal(got[n], want[n]) for n in want)
        for out in (h[:1].expand(h.shape), h.transpose(2, 3).contiguous().transpose(2, 3), d["v"]):
            with pytest.raises((ValueError, RuntimeError)):
                G.gated_scan(**d, out=out)


def test_workspaces_that_do_not_fit(gpu):
    """Too small: another is taken.  Not of this device, or not contiguous: refused."""
    import torch

    import gdn2_amd as G

    d = _make(gpu, 18, 1, 3000, 2, 64, "f32", True, True, True)
    want = G.gated_scan(**d)[0]
    x = torch.randn(1, 3000, 64, device=gpu)
    y, stats = G.group_norm_act(x, 2, return_stats=True)
    w = torch.randn(64, 4, device=gpu)
    calls = [lambda ws: G.gated_scan(**d, workspace=ws)[0],
             lambda ws: G.gated_scan_backward(d["g"], d["v"], d["w"], want, want, workspace=ws)["dv"],
             lambda ws: G.group_norm_act(x, 2, workspace=ws),
             lambda ws: G.group_norm_act_backward(x, 2, stats, x, workspace=ws)["dx"],
             lambda ws: G.short_conv_1d_backward(x, w, x, workspace=ws)["dx"]]
    small, large = torch.empty(8, dtype=torch.uint8, device=gpu), torch.empty(1 << 24, dtype=torch.uint8, device=gpu)
    for call in calls:
        assert torch.equal(call(small), call(None)) and torch.equal(call(large), call(None))
        for bad in (torch.empty(1 << 24, dtype=torch.uint8), small[:1].expand(1 << 24), large[::2]):
            with pytest.raises(ValueError):
                call(bad)


def test_bad_offsets_stay_in_bounds(gpu):
    """Offsets outside the row or decreasing: unspecified results, the buffers
    around the tensors untouched."""
    import torch

    import gdn2_amd as G

    T, H, V = 300, 2, 36
    big = torch.full((T + 200, H, V), 5.0, device=gpu)
    out = big[100:100 + T].unsqueeze(0).transpose(1, 2)
    d = _make(gpu, 13, 1, T, H, V, "f32", False, True, True, N=4)
    states = torch.full((8, H, V), 5.0, device=gpu)
    for bounds in ([-5, 10, 400, 1000, 2 ** 31 - 1], [300, 200, 100, 50, 0], [0, 200, 100, 250, 300], [-9, -8, -7, -6, -5]):
        cu = torch.tensor(bounds, dtype=torch.int32, device=gpu)
        G.gated_scan(**d, cu_seqlens=cu, out=out, new_state=states[2:6])
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, out, d["state"], cu_seqlens=cu)
        torch.cuda.synchronize()
        assert (big[:100] == 5).all() and (big[100 + T:] == 5).all() and (states[:2] == 5).all() and (states[6:] == 5).all()
        assert r["dS0"].shape == (4, H, V)


def test_streams_and_graphs(gpu):
    """Two calls at once on two streams; a captured forward and backward replayed
    with new inputs between eager calls."""
    import torch

    import gdn2_amd as G

    d = [_make(gpu, 20 + i, 1, 5000, 2, 64, "f32", True, True, True) for i in range(2)]
    want = [G.gated_scan(**x) for x in d]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = G.gated_scan(**d[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])

    x = {n: t.clone() for n, t in d[0].items()}
    d_out = torch.randn_like(want[0][0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o, n = G.gated_scan(**x)
        G.gated_scan_backward(x["g"], x["v"], x["w"], o, d_out, x["state"], d_state=n)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, n = G.gated_scan(**x)
        r = G.gated_scan_backward(x["g"], x["v"], x["w"], o, d_out, x["state"], d_state=n)
    for k in range(4):
        for name in x:
            x[name].copy_(d[k % 2][name])
        graph.replay()
        torch.cuda.synchronize()
        e, en = want[k % 2]
        er = G.gated_scan_backward(x["g"], x["v"], x["w"], e, d_out, x["state"], d_state=en)
        assert torch.equal(o, e) and torch.equal(n, en) and all(torch.equal(r[m], er[m]) for m in r)
