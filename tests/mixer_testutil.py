"""Plain 64-bit forms of the mixer operators (numpy), and what f32 arithmetic
may be off by.  Operands are [B, T, C]-like numpy arrays: the callers flatten
heads."""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24  # half a step of f32
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}  # half a step of a result's type


def scan64(g, u, h0, bounds=None):
    """h_t = e^{g_t} h_{t-1} + u_t over axis 1 of [B, T, ...]; bounds: token
    offsets of the sequences in row 0.  Returns h (NaN outside), final states,
    and the bound on an f32 result's error (see scan_error)."""
    B, T = u.shape[:2]
    h, err = np.full(u.shape, np.nan), np.full(u.shape, np.nan)
    last = np.array(h0, np.float64)
    last_err = np.zeros_like(last)
    spans = [(b, b, 0, T) for b in range(B)] if bounds is None else [
        (0, n, bounds[n], bounds[n + 1]) for n in range(len(bounds) - 1)]
    for row, n, t0, t1 in spans:
        x, xa, e = np.array(h0[n], np.float64), np.abs(np.array(h0[n], np.float64)), np.zeros_like(h0[n], np.float64)
        for t in range(t0, t1):
            a = np.exp(g[row, t])
            with np.errstate(invalid="ignore"):
                keep = a != 0
                x = np.where(keep, a * x, 0) + u[row, t]
                xa = np.where(keep, a * xa, 0) + np.abs(u[row, t])
                # a token costs at most 8 roundings of what it adds up: w v, the decay
                # (series or exponential: two, and |g| e^g < 0.37 of its argument), the
                # product and sum of the two forms, and its share of the joins, one for
                # four tokens or more, of four roundings and those of G (|G| e^G < 0.37)
                e = np.where(keep, a * e, 0) + 8 * EPS * xa
            h[row, t], err[row, t] = x, e
        last[n], last_err[n] = x, e
    return h, last, err, last_err


def scan_bwd64(g, v, w, h, dy, h0, ds, bounds=None):
    """The gradients for given h; each with the bound on its error.  Arrays as in
    scan64 (w None: 1)."""
    B, T = v.shape[:2]
    names = ("dg", "dv", "dw")
    out = {n: np.zeros(v.shape) for n in names}
    err = {n: np.zeros(v.shape) for n in names}
    dh0, dh0_err = np.array(ds, np.float64), np.zeros(ds.shape)
    ww = np.ones(v.shape) if w is None else w
    spans = [(b, b, 0, T) for b in range(B)] if bounds is None else [
        (0, n, bounds[n], bounds[n + 1]) for n in range(len(bounds) - 1)]
    for row, n, t0, t1 in spans:
        E, Ea, e = np.array(ds[n], np.float64), np.abs(ds[n]), np.zeros(ds[n].shape)
        for t in range(t1 - 1, t0 - 1, -1):
            a = np.exp(g[row, t])
            D, Da = dy[row, t] + E, np.abs(dy[row, t]) + Ea
            de = e + EPS * Da
            out["dv"][row, t], out["dw"][row, t] = ww[row, t] * D, v[row, t] * D
            err["dv"][row, t] = np.abs(ww[row, t]) * (de + 2 * EPS * Da)
            err["dw"][row, t] = np.abs(v[row, t]) * (de + 2 * EPS * Da)
            E, Ea, e = a * D, a * Da, a * de + 8 * EPS * a * Da
            before = h0[n] if t == t0 else h[row, t - 1]
            out["dg"][row, t] = E * before
            err["dg"][row, t] = np.abs(before) * (e + EPS * Ea)
        dh0[n], dh0_err[n] = E, e
    out["dS0"], err["dS0"] = dh0, dh0_err
    return out, err


def worst(got, want, err, half):
    """The largest error in units of what it may be: `err` of the f32 arithmetic
    and half a step of the result's type (1 = at the bound)."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    if got.size == 0:
        return 0.0
    bound = err + half * (np.abs(want) + err) + 1e-37  # (and the range of f32)
    return float(np.max(np.abs(got - want) / bound))
