"""gated_scan and gated_scan_backward with values that are not finite, decays of
zero and states that overflow, in full tiles (the form of a tile whose tokens are
all of one sequence) and in the others: what a token by token pass in f32 does."""
import itertools

import numpy as np
import pytest

import mixer_testutil as M

pytestmark = pytest.mark.gpu

MOST = 2.0 ** 128  # (f32 ends half a step below)


def _type(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _flat(t):
    """[B, H, T, V] -> numpy [B, T, H, V]"""
    return t.detach().double().cpu().numpy().transpose(0, 2, 1, 3)


def _spans(T, B, bounds):
    if bounds is None:
        return [(b, b, 0, T) for b in range(B)]
    return [(0, n, bounds[n], bounds[n + 1]) for n in range(len(bounds) - 1)]


def _f32(x):
    return np.where(np.abs(x) >= MOST, np.sign(x) * np.inf, x)


def _gone(a):
    """Decays that f32 has as zero."""
    return a < 2.0 ** -150


# What a log decay's own rounding costs the state that it is of, in half steps of |g|
# of it (M.scan64 counts it against the state and what is added, of ordinary decays; a
# state that nothing is added to keeps all of it).  e^g is 2^(g log2 e) with a rounded
# product and constant: 1.3.  Of a run it is 2^G, G a sum of its tokens' in f32, whose
# every partial sum is off by half a step of itself, and so of |g| of each token in it:
# 8 tokens a thread, 2 to 4 steps over lanes and 8 waves, of which no form has more
# than 18.
SUMS = 20


def forward64(g, u, h0, bounds=None):
    """h_t = e^{g_t} h_{t-1} + u_t, nothing of h passing an e^g that is zero in f32 and
    what leaves f32 infinite; the final states; the bound of f32 arithmetic (the
    roundings of M.scan64)."""
    B, T = u.shape[:2]
    h, err, last = np.zeros(u.shape), np.zeros(u.shape), np.array(h0)
    with np.errstate(invalid="ignore", over="ignore"):
        for row, n, t0, t1 in _spans(T, B, bounds):
            x, xa, e = last[n].copy(), np.abs(last[n]), np.zeros(last[n].shape)
            for t in range(t0, t1):
                a = np.exp(g[row, t])
                gone, ut = _gone(a), u[row, t]
                x = _f32(np.where(gone, 0, a * x) + ut)
                e = np.where(gone, 0, a * e + SUMS * M.EPS * np.abs(g[row, t]) * a * xa)
                xa = np.where(gone, 0, a * xa) + np.abs(ut)
                e = e + 8 * M.EPS * xa
                h[row, t], err[row, t] = x, e
            last[n] = x
    return h, last, err


def backward64(g, v, w, h, dy, h0, ds, bounds=None):
    """The gradients for given h, by the same rules: nothing of the gradient passes an
    e^g of zero, nor has g_t one there; the bounds of M.scan_bwd64."""
    B, T = v.shape[:2]
    out = {n: np.zeros(v.shape) for n in ("dg", "dv", "dw")}
    err = {n: np.zeros(v.shape) for n in out}
    dS0 = np.array(ds)
    with np.errstate(invalid="ignore", over="ignore"):
        for row, n, t0, t1 in _spans(T, B, bounds):
            E, Ea, e = dS0[n].copy(), np.abs(dS0[n]), np.zeros(dS0[n].shape)
            for t in range(t1 - 1, t0 - 1, -1):
                a = np.exp(g[row, t])
                gone = _gone(a)
                D, Da = _f32(dy[row, t] + E), np.abs(dy[row, t]) + Ea
                de = e + M.EPS * Da
                out["dv"][row, t], out["dw"][row, t] = _f32(w[row, t] * D), _f32(v[row, t] * D)
                err["dv"][row, t] = np.abs(w[row, t]) * (de + 2 * M.EPS * Da)
                err["dw"][row, t] = np.abs(v[row, t]) * (de + 2 * M.EPS * Da)
                E, Ea = np.where(gone, 0, a * D), np.where(gone, 0, a * Da)
                e = np.where(gone, 0, a * de) + (8 + SUMS * np.where(gone, 0, np.abs(g[row, t]))) * M.EPS * Ea
                before = h0[n] if t == t0 else h[row, t - 1]
                out["dg"][row, t] = np.where(gone, 0, E * before)
                err["dg"][row, t] = np.where(gone, 0, np.abs(before) * (e + M.EPS * Ea))
            dS0[n] = E
    out["dS0"], err["dS0"] = dS0, None
    return out, err


def same(name, got, want, err, half):
    """NaN where NaN is due, infinities of the same sign, the rest within its bound."""
    got = np.asarray(got)
    assert got.shape == want.shape
    for what, a, b in (("NaN", np.isnan(got), np.isnan(want)), ("inf", np.isposinf(got), np.isposinf(want)),
                       ("-inf", np.isneginf(got), np.isneginf(want))):
        bad = np.argwhere(a != b)
        assert len(bad) == 0, f"{name}: {what} differs at {len(bad)} places, the first {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"
    if err is None:
        return
    ok = np.isfinite(want)
    e = M.worst(got[ok], want[ok], np.nan_to_num(err[ok], posinf=0), half)
    assert e <= 1, (name, e)


FORMS = [  # T, H, V, offsets: one tile, several, several chains of some tiles, packed
    (40, 1, 128, None), (420, 1, 128, None), (300, 2, 256, None), (420, 1, 128, [0, 64, 420]),
]
KINDS = [("f32", False, True), ("f32", True, False), ("bf16", False, False), ("bf16", True, True)]


def _operands(gpu, T, H, V, ty, per_head, w, bounds, seed=0):
    import torch

    r = torch.Generator().manual_seed(1000 + seed)
    N = 1 if bounds is None else len(bounds) - 1
    d = {"g": -0.005 - 0.2 * torch.rand(1, T, H, 1 if per_head else V, generator=r),
         "v": torch.randn(1, T, H, V, generator=r) + 3.0,  # (no zeros: an infinity times it is one)
         "w": 0.5 + torch.rand(1, T, H, V, generator=r) if w else None, "state": torch.randn(N, H, V, generator=r) + 3.0}
    return d, N


def _on(gpu, d, ty):
    import torch

    return {n: None if t is None else t.to(gpu, _type(ty) if n in "vw" else torch.float32) if n == "state" else
            t.to(gpu, _type(ty) if n in "vw" else torch.float32).transpose(1, 2) for n, t in d.items()}


def _check(gpu, d, N, ty, bounds, d_out=None):
    """Both directions of the operands d [1, T, H, .] on the host."""
    import torch

    import gdn2_amd as G

    x = _on(gpu, d, ty)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu)
    out, new = G.gated_scan(x["g"], x["v"], x["w"], x["state"], cu_seqlens=cu)
    torch.cuda.synchronize()
    v, w = _flat(x["v"]), _flat(x["w"]) if x["w"] is not None else np.ones(d["v"].shape)
    g, h0 = np.broadcast_to(_flat(x["g"]), v.shape), x["state"].double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        h, last, err = forward64(g, _f32(v * w), h0, bounds)
    same("out", _flat(out), h, err, M.HALF[ty])
    same("state", new.double().cpu().numpy(), last, None, 0)
    if d_out is None:
        return
    dy = d_out.to(gpu, _type(ty)).transpose(1, 2)
    ds = torch.ones_like(x["state"])
    # (finite states: those of a call without the values that are not)
    calm = {n: None if t is None else torch.nan_to_num(t, nan=1.0, posinf=1.0, neginf=-0.1) for n, t in x.items()}
    h = G.gated_scan(calm["g"], calm["v"], calm["w"], calm["state"], cu_seqlens=cu)[0]
    r = G.gated_scan_backward(x["g"], calm["v"], calm["w"], h, dy, calm["state"], d_state=ds, cu_seqlens=cu)
    torch.cuda.synchronize()
    cv, cw = _flat(calm["v"]), _flat(calm["w"]) if x["w"] is not None else np.ones(v.shape)
    want, err = backward64(g, cv, cw, _flat(h), _flat(dy), calm["state"].double().cpu().numpy(), ds.double().cpu().numpy(), bounds)
    if x["g"].shape[3] == 1:
        with np.errstate(invalid="ignore"):
            V = v.shape[3]
            err["dg"] = (err["dg"] + V * M.EPS * np.abs(want["dg"])).sum(3, keepdims=True)
            want["dg"] = want["dg"].sum(3, keepdims=True)
    for n in ("dg", "dv", "dw"):
        if r[n] is not None:
            same(n, _flat(r[n]), want[n], err[n], M.HALF[ty] if n != "dg" else 0)
    same("dS0", r["dS0"].double().cpu().numpy(), want["dS0"], None, 0)


def _gradient(T, H, V, seed=0):
    import torch

    return torch.rand(1, T, H, V, generator=torch.Generator().manual_seed(7 + seed)) + 0.5


@pytest.mark.parametrize("ty,per_head,w", KINDS)
@pytest.mark.parametrize("T,H,V,bounds", FORMS)
def test_states_that_are_not_finite(gpu, T, H, V, bounds, ty, per_head, w):
    """An infinity or a NaN in some channels' initial state (in the adjoint: gradient of
    the last one) reaches every token's row of these channels, and no row stays as it
    was."""
    import torch

    import gdn2_amd as G

    d, N = _operands(gpu, T, H, V, ty, per_head, w, bounds)
    d["state"][:, :, 3::32], d["state"][:, :, 17::64] = float("inf"), float("nan")
    d["state"][:, :, 20::64] = float("-inf")
    _check(gpu, d, N, ty, bounds)
    x = _on(gpu, d, ty)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu)
    ones, dy = torch.ones_like(x["v"]), torch.ones_like(x["v"])
    r = G.gated_scan_backward(x["g"], ones, None, ones, dy, None, d_state=x["state"], cu_seqlens=cu)
    torch.cuda.synchronize()
    one = np.ones((1, T, H, V))
    want, err = backward64(np.broadcast_to(_flat(x["g"]), one.shape), one, one, one, one, np.zeros((N, H, V)),
                           x["state"].double().cpu().numpy(), bounds)
    same("dv", _flat(r["dv"]), want["dv"], err["dv"], M.HALF[ty])
    same("dS0", r["dS0"].double().cpu().numpy(), want["dS0"], None, 0)


@pytest.mark.parametrize("ty,per_head,w", KINDS)
@pytest.mark.parametrize("T,H,V,bounds", FORMS)
def test_values_that_are_not_finite(gpu, T, H, V, bounds, ty, per_head, w):
    """An infinity or a NaN at another token in every channel, so at every place of a
    wave's tokens, and a log decay of -inf some tokens later (in the adjoint: before):
    they reach every token up to there, and none beyond."""
    for bad, after in itertools.product((float("inf"), float("-inf"), float("nan")), (1, 2, 3, 9, None)):
        print("values", T, H, V, bounds, ty, per_head, w, bad, after, flush=True)
        d, N = _operands(gpu, T, H, V, ty, per_head, w, bounds)
        dy = _gradient(T, H, V)
        for c in range(V):
            t = (T // 3 + c) % T
            d["v"][0, t, :, c] = bad
            dy[0, t, :, c] = bad
            if after and not per_head:
                d["g"][0, (t + after) % T, :, c] = float("-inf")
                d["g"][0, (t - after) % T, :, c] = float("-inf")
        if after and per_head:
            d["g"][0, after::11] = float("-inf")
        _check(gpu, d, N, ty, bounds, dy)


def _overflowing(name, got, wide, step, err, half):
    """States that leave f32.  wide: the recurrence in 64 bits, whose range holds all of
    them; step: token by token, infinite from the first that f32 does not hold.  Both
    are right where they differ: e^G h + X over a run of tokens can be finite again
    where a state inside the run is not.  So: infinite where `wide` is out of range,
    else either of the two, and never a NaN."""
    either = np.isinf(step) & (got == step)
    same(name, np.where(either, step, got), np.where(either, step, _f32(wide)), err, half)


@pytest.mark.parametrize("ty,per_head,w", KINDS)
def test_states_that_overflow(gpu, ty, per_head, w):
    """States that leave f32 at some token, another one in every channel, and with them
    the gradients: infinite, of that sign, and no NaN behind them."""
    import torch

    import gdn2_amd as G

    T, H, V = 300, 1, 128
    for reset in (False, True):
        d, N = _operands(gpu, T, H, V, ty, per_head, w, None)
        dy = _gradient(T, H, V)
        big = 1.5 * 2.0 ** 127  # two of them, hardly decayed between, overflow
        for c in range(V):
            sign = 1 - 2 * (c % 2)
            for i in (0, 1):
                d["v"][0, 70 + c + i, :, c] = sign * big
                dy[0, 70 + c + i, :, c] = sign * big
        d["g"][:, 60:210] = -0.01
        if w:
            d["w"][...] = 1.0
        if reset:
            d["g"][0, 3::17] = float("-inf")
        x = _on(gpu, d, ty)
        out, new = G.gated_scan(x["g"], x["v"], x["w"], x["state"])
        ones = torch.ones_like(x["v"])
        r = G.gated_scan_backward(x["g"], ones, None, ones, dy.to(gpu, _type(ty)).transpose(1, 2), x["state"])
        torch.cuda.synchronize()
        g = np.broadcast_to(_flat(x["g"]), (1, T, H, V))
        h0, v = x["state"].double().cpu().numpy(), _flat(x["v"])
        step, _, err = forward64(g, v, h0)
        with np.errstate(invalid="ignore"):
            wide = M.scan64(g, v, h0)[0]
        _overflowing("out", _flat(out), wide, step, err, M.HALF[ty])
        one, zeros, dy = np.ones((1, T, H, V)), np.zeros((1, H, V)), _flat(dy.to(_type(ty)).transpose(1, 2))
        step, err = backward64(g, one, one, one, dy, h0, zeros)
        with np.errstate(invalid="ignore"):
            wide = M.scan_bwd64(g, one, one, one, dy, h0, zeros)[0]
        _overflowing("dv", _flat(r["dv"]), wide["dv"], step["dv"], err["dv"], M.HALF[ty])


@pytest.mark.parametrize("ty,per_head,w", KINDS)
@pytest.mark.parametrize("T,H,V,bounds", FORMS)
def test_zero_decays_of_finite_logs(gpu, T, H, V, bounds, ty, per_head, w):
    """A log decay whose e^g is zero in f32 forgets a state that is not finite as -inf
    does, wherever the borders of runs, waves and tiles fall; so does one behind a log
    decay that is NaN itself."""
    import torch

    for reset, bad in itertools.product((-110.0, -130.0, -170.0, -1e30, float("-inf")), ("state", "nan decay")):
        print("zero decays", T, H, V, bounds, ty, per_head, w, reset, bad, flush=True)
        d, N = _operands(gpu, T, H, V, ty, per_head, w, bounds)
        d["state"][:, :, 1::2] = float("inf")
        d["state"][:, :, 2::4] = float("nan")
        for c in range(1 if per_head else V):
            d["g"][0, (7 + 5 * c) % T::29, :, c] = reset
            if bad == "nan decay" and c % 2 == 0:
                d["g"][0, (6 + 5 * c) % T::29, :, c] = float("nan")
        _check(gpu, d, N, ty, bounds)
        # the adjoint: the last state's gradient comes from behind
        import gdn2_amd as G

        x = _on(gpu, d, ty)
        cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu)
        ones, dy = torch.ones_like(x["v"]), torch.ones_like(x["v"])
        r = G.gated_scan_backward(x["g"], ones, None, ones, dy, None, d_state=x["state"], cu_seqlens=cu)
        torch.cuda.synchronize()
        one = np.ones((1, T, H, V))
        want, err = backward64(np.broadcast_to(_flat(x["g"]), one.shape), one, one, one, one, np.zeros((N, H, V)),
                               x["state"].double().cpu().numpy(), bounds)
        same("dv", _flat(r["dv"]), want["dv"], err["dv"], M.HALF[ty])
        same("dS0", r["dS0"].double().cpu().numpy(), want["dS0"], None, 0)


@pytest.mark.parametrize("ty,per_head,w", KINDS)
def test_the_smallest_decays_count_the_same_in_tiles_and_steps(gpu, ty, per_head, w):
    """e^g between 2^-150 and 2^-126 may count as zero: then in every form of the call.
    A prompt in tiles and its tokens one by one are infinite and NaN at the same places."""
    import torch

    import gdn2_amd as G

    T, V = 200, 128
    for reset in (-87.2, -87.5, -95.0, -100.0, -103.0):
        d, N = _operands(gpu, T, 1, V, ty, per_head, w, None)
        d["state"][:, :, 1::2] = float("inf")
        d["state"][:, :, 2::4] = float("nan")
        for c in range(1 if per_head else V):
            d["g"][0, 20 + c, :, c] = reset
        x = _on(gpu, d, ty)
        out, new = G.gated_scan(**x)
        state, steps = x["state"], []
        for t in range(T):
            o, state = G.gated_scan(*(None if x[n] is None else x[n][:, :, t:t + 1] for n in "gvw"), state)
            steps.append(o)
        steps = torch.cat(steps, 2)
        torch.cuda.synchronize()
        for a, b in ((out, steps), (new, state)):
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b)), reset


@pytest.mark.parametrize("ty,per_head,w", KINDS)
@pytest.mark.parametrize("T,H,V,bounds", FORMS)
def test_long_decays_keep_what_is_not_finite(gpu, T, H, V, bounds, ty, per_head, w):
    """An infinite state stays infinite and a NaN one NaN through any number of decays
    that are not zero, also where their product is below f32's range; a finite one
    of any size leaves nothing there."""
    import torch

    import gdn2_amd as G

    for pace in (2.0, 60.0):
        d, N = _operands(gpu, T, H, V, ty, per_head, w, bounds)
        d["g"] *= pace / 0.1
        d["g"].clamp_(min=-85.0)
        d["state"][:, :, 1::4], d["state"][:, :, 2::4], d["state"][:, :, 3::8] = float("inf"), float("nan"), float("-inf")
        d["state"][:, :, 7::8] = 3e38
        _check(gpu, d, N, ty, bounds)
        x = _on(gpu, d, ty)
        cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu)
        ones, dy = torch.ones_like(x["v"]), torch.ones_like(x["v"])
        r = G.gated_scan_backward(x["g"], ones, None, ones, dy, None, d_state=x["state"], cu_seqlens=cu)
        torch.cuda.synchronize()
        one = np.ones((1, T, H, V))
        want, err = backward64(np.broadcast_to(_flat(x["g"]), one.shape), one, one, one, one, np.zeros((N, H, V)),
                               x["state"].double().cpu().numpy(), bounds)
        same("dv", _flat(r["dv"]), want["dv"], err["dv"], M.HALF[ty])
        same("dS0", r["dS0"].double().cpu().numpy(), want["dS0"], None, 0)


@pytest.mark.parametrize("ty,per_head,w", KINDS)
@pytest.mark.parametrize("T,H,V,bounds", FORMS)
def test_gradient_of_a_zero_decay_is_zero(gpu, T, H, V, bounds, ty, per_head, w):
    """Padding that holds NaN or infinities, shut off by a log decay of -inf behind it:
    out does not depend on that decay, and its gradient is zero (the gradients behind
    it, and those of the tokens before the padding, are those of a clean call)."""
    import torch

    import gdn2_amd as G

    for bad, reset in itertools.product((float("nan"), float("inf")), (float("-inf"), -150.0)):
        d, N = _operands(gpu, T, H, V, ty, per_head, w, bounds)
        dy = _gradient(T, H, V)
        pads = [(a, a + 5) for a in range(9, T - 8, 14)]
        inside = np.zeros(T, bool)
        for a, b in pads:
            d["v"][0, a:b] = bad
            d["g"][0, a], d["g"][0, b] = -0.3, reset
            dy[0, a:b] = 0
            inside[a:b] = True
        x = _on(gpu, d, ty)
        cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=gpu)
        out, _ = G.gated_scan(x["g"], x["v"], x["w"], x["state"], cu_seqlens=cu)
        r = G.gated_scan_backward(x["g"], x["v"], x["w"], out, dy.to(gpu, _type(ty)).transpose(1, 2), x["state"], cu_seqlens=cu)
        torch.cuda.synchronize()
        v, w_ = _flat(x["v"]), _flat(x["w"]) if x["w"] is not None else np.ones(d["v"].shape)
        g = np.broadcast_to(_flat(x["g"]), v.shape)
        want, err = backward64(g, v, w_, _flat(out), _flat(dy.to(_type(ty)).transpose(1, 2)),
                               x["state"].double().cpu().numpy(), np.zeros((N, H, V)), bounds)
        if per_head:
            with np.errstate(invalid="ignore"):
                err["dg"] = (err["dg"] + V * M.EPS * np.abs(want["dg"])).sum(3, keepdims=True)
                want["dg"] = want["dg"].sum(3, keepdims=True)
        dg = _flat(r["dg"])
        assert all((dg[0, b] == 0).all() for _, b in pads)
        for n in ("dg", "dv", "dw"):
            if r[n] is not None:
                same(n, _flat(r[n])[:, ~inside], want[n][:, ~inside], err[n][:, ~inside], M.HALF[ty] if n != "dg" else 0)
