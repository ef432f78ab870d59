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


# -- group norm -------------------------------------------------------------------

def act64(z, act):
    """act(z) and its first derivative."""
    from scipy.special import erf, expit

    if act == "silu":
        s = expit(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + erf(z / np.sqrt(2)))
        return z * c, c + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    return z, np.ones_like(z)


def _act_err(z, z_err, a):
    """The error of act(z) and of its derivative in f32: those of z (|act'| < 1.13,
    |act''| < 0.8), the exponential's argument (2 |z| roundings of the factor it
    makes), erf's two units in the last place of 1, and a few products."""
    return 1.13 * z_err + (np.abs(a) * (2 * np.abs(z) + 8) + 4 * np.abs(z)) * EPS, 0.8 * z_err + (4 * np.abs(z) + 12) * EPS


SUM = 80  # roundings of a sum of a group: 64 terms one after the other, then a tree


def norm64(x, groups, weight, bias, eps, act, gate=None, stats=None):
    """[N, S, C]: dict y, stats, and what the backward needs; *_err bounds on f32
    errors.  With `stats` these are taken as given."""
    N, S, C = x.shape
    r = x.reshape(N, S, groups, C // groups)
    full = lambda v: np.broadcast_to(v, r.shape).reshape(N, S, C)  # noqa: E731
    if stats is None:
        mean, var = r.mean((1, 3), keepdims=True), r.var((1, 3), keepdims=True)
        rstd = 1 / np.sqrt(var + eps)
        mean_err = SUM * EPS * np.abs(r).mean((1, 3), keepdims=True)
        # the variance about a shifted point loses what the shift adds to the squares
        spread = 1 + ((r - mean) ** 2).max((1, 3), keepdims=True) * rstd ** 2
        rel = 0.5 * (SUM * EPS * spread + (mean_err * rstd) ** 2) + 4 * EPS
    else:
        mean, rstd = stats[:, None, :, 0:1], stats[:, None, :, 1:2]
        mean_err, rel = np.zeros_like(mean), np.zeros_like(mean)
    n = full((r - mean) * rstd)
    n_err = np.abs(n) * full(rel + 3 * EPS) + full(mean_err * rstd)
    w, b = (np.ones(C) if weight is None else weight), (np.zeros(C) if bias is None else bias)
    z = n * w + b
    z_err = np.abs(w) * n_err + 2 * EPS * (np.abs(n * w) + np.abs(b))
    p = z if gate is None else gate  # what the activation is of
    a, d = act64(p, act)
    a_err, d_err = _act_err(p, z_err if gate is None else 0.0, a)
    y, y_err = (a, a_err) if gate is None else (z * a, z_err * np.abs(a) + np.abs(z) * a_err + EPS * np.abs(z * a))
    st = np.concatenate([mean, rstd], -1).reshape(N, groups, 2)
    st_err = np.concatenate([mean_err, rel * rstd], -1).reshape(N, groups, 2)
    return dict(y=y, y_err=y_err, stats=st, stats_err=st_err, n=n, n_err=n_err, z=z, z_err=z_err, a=a, a_err=a_err, d=d,
                d_err=d_err, w=w, rstd=full(rstd))


def norm_bwd64(x, groups, weight, bias, act, gate, stats, dy, sum_terms=200):
    """The gradients for given stats, and the bounds on their errors.  sum_terms:
    roundings of a sum over samples and rows (a thread's rows one after the other,
    then its workgroup's and the others')."""
    N, S, C = x.shape
    f = norm64(x, groups, weight, bias, 0.0, act, gate, stats)
    k, k_err = (f["d"], f["d_err"]) if gate is None else (f["a"], f["a_err"])
    dz = dy * k
    dz_err = np.abs(dy) * k_err + EPS * np.abs(dz)
    dn, dn_err = dz * f["w"], np.abs(f["w"]) * dz_err + EPS * np.abs(dz * f["w"])
    grp = lambda v: np.broadcast_to(v.reshape(N, S, groups, -1).mean((1, 3), keepdims=True),  # noqa: E731
                                    (N, S, groups, C // groups)).reshape(N, S, C)
    n, n_err = f["n"], f["n_err"]
    s1, s2 = grp(dn), grp(dn * n)
    s1_err = grp(dn_err + (SUM + sum_terms) * EPS * np.abs(dn))
    s2_err = grp(dn_err * np.abs(n) + np.abs(dn) * n_err + (SUM + sum_terms) * EPS * np.abs(dn * n))
    out = {"dx": f["rstd"] * (dn - s1 - n * s2), "dweight": (dz * n).sum((0, 1)), "dbias": dz.sum((0, 1)), "dgate": None}
    err = {"dx": f["rstd"] * (dn_err + s1_err + n_err * np.abs(s2) + np.abs(n) * s2_err
                              + 4 * EPS * (np.abs(dn) + np.abs(s1) + np.abs(n * s2))),
           "dweight": (dz_err * np.abs(n) + np.abs(dz) * n_err + sum_terms * EPS * np.abs(dz * n)).sum((0, 1)),
           "dbias": (dz_err + sum_terms * EPS * np.abs(dz)).sum((0, 1)), "dgate": None}
    if gate is not None:
        out["dgate"] = dy * f["z"] * f["d"]
        err["dgate"] = np.abs(dy) * (f["z_err"] * np.abs(f["d"]) + np.abs(f["z"]) * f["d_err"]) + 2 * EPS * np.abs(out["dgate"])
    return out, err


# -- short conv -------------------------------------------------------------------

def conv64(x, w, cache):
    """x [B, T, C], w [C, 4], cache [B, 3, C] or None: out, new cache."""
    B, T, C = x.shape
    xp = np.concatenate([cache if cache is not None else np.repeat(x[:, :1], 3, 1), x], 1)
    z = sum(xp[:, i:i + T] * w[:, i] for i in range(4))
    return act64(z, "silu")[0], xp[:, T:], xp, z


def conv_bwd64(x, w, cache, dy, dc, sum_terms=120):
    """The gradients and the bounds on their f32 errors.  sum_terms: roundings of a
    sum over tokens (32 of a thread, its workgroup's waves, 16 threads over the
    workgroups' sums and these)."""
    B, T, C = x.shape
    _, _, xp, z = conv64(x, w, cache)
    d = act64(z, "silu")[1]
    z_err = 5 * EPS * sum(np.abs(xp[:, i:i + T] * w[:, i]) for i in range(4))
    dz = dy * d
    dz_err = np.abs(dy) * _act_err(z, z_err, z)[1] + EPS * np.abs(dz)
    dp, dp_err = np.zeros_like(xp), np.zeros_like(xp)
    for i in range(4):
        dp[:, i:i + T] += dz * w[:, i]
        dp_err[:, i:i + T] += (dz_err + 6 * EPS * np.abs(dz)) * np.abs(w[:, i])
    if dc is not None:
        dp[:, T:] += dc
        dp_err[:, T:] += 3 * EPS * np.abs(dc)
    out = {"dweight": np.stack([(dz * xp[:, i:i + T]).sum((0, 1)) for i in range(4)], 1), "dx": dp[:, 3:].copy(), "dcache": None}
    err = {"dweight": np.stack([((dz_err + sum_terms * EPS * np.abs(dz)) * np.abs(xp[:, i:i + T])).sum((0, 1))
                                for i in range(4)], 1), "dx": dp_err[:, 3:] + 4 * EPS * np.abs(dp[:, 3:]), "dcache": None}
    if cache is None:
        if T:
            out["dx"][:, 0] += dp[:, :3].sum(1)
            err["dx"][:, 0] += (dp_err[:, :3] + 4 * EPS * np.abs(dp[:, :3])).sum(1)
    else:
        out["dcache"], err["dcache"] = dp[:, :3], dp_err[:, :3]
    return out, err
