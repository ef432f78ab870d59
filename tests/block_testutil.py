"""Plain 64-bit forms of the block operators (torch on the CPU), and what f32
arithmetic may be off by.  Rows are [M, C]: the callers flatten what stands before."""
from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -24  # half a step of f32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # of a result's type (bf16: 2^-8 relative at most)
F64 = torch.float64


def words(rows, C, seed, offset=0):
    """uint32 words of [rows, C]: Philox-4x32, 7 rounds, counter offset + row ceil(C/4) + c/4."""
    q = -(-C // 4)
    n = (np.arange(rows * q, dtype=np.uint64) + np.uint64(offset % 2 ** 64))  # (wraps)
    return philox(n & np.uint64(0xFFFFFFFF), n >> np.uint64(32), 0 * n, 0 * n, seed % 2 ** 64).reshape(rows, 4 * q)[:, :C]


def philox(c0, c1, c2, c3, key, rounds=7):
    m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    for i in range(rounds):
        k0, k1 = (np.uint64(((key >> sh) + i * w) & 0xFFFFFFFF) for sh, w in ((0, 0x9E3779B9), (32, 0xBB67AE85)))
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> s) ^ c1 ^ k0, b & m, (a >> s) ^ c3 ^ k1, a & m
    return np.stack([c0, c1, c2, c3], -1)


def kept(rows, C, p, seed, offset=0):
    """bool [rows, C]."""
    return torch.from_numpy((words(rows, C, seed, offset) >> np.uint64(8)) >= np.uint64(np.floor(p * 2 ** 24 + 0.5)))


def drop_factor(M, C, p, seed=0, offset=0):
    if p == 0:
        return torch.ones(M, C, dtype=F64)
    return kept(M, C, p, seed, offset).double() / (1 - p if p < 1 else 1)


def _act(z, act):
    s = torch.sigmoid(z)
    if act == "none":
        return z, torch.ones_like(z)
    return (z * s, s * (1 + z * (1 - s))) if act == "silu" else (s, s * (1 - s))


def _act_err(z, act):
    """Of act(z) relative to it, and of act'(z): the exponential's argument costs 2 |z|
    half steps, it, the sum and the reciprocal 5, a product or two the rest."""
    if act == "none":
        return torch.zeros_like(z), torch.zeros_like(z)
    a = (2 * z.abs() + 8) * U
    return a, a * (1 + z.abs())


def residual64(x, y, gate, post, pre, eps, act, alpha, sigma, factor):
    """(out, normed, stats) and the errors of an f32 result.  gate: of every row.  A
    mean of squares takes at most 16 products a lane, 6 joins of lanes and 8 of waves,
    then 1 / C and eps: 33 half steps, halved by the root, and 2 for it: 20."""
    sy = sr = None
    r, err = alpha * x, 2 * U * (alpha * x).abs()
    if y is not None:
        b, rel = y, torch.full_like(y, 3 * U)
        if post is not None:
            sy = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
            b, rel = y * sy * post, rel + 22 * U
        if gate is not None:
            b, rel = b * _act(gate, act)[0], rel + U + _act_err(gate, act)[0]
        b = sigma * factor * b
        r = r + b
        err = err + rel * b.abs()
    err = err + U * r.abs()
    n = n_err = None
    stats = torch.zeros(x.shape[0], 2, dtype=F64)
    stats_err = torch.zeros_like(stats)
    if sy is not None:
        stats[:, :1], stats_err[:, :1] = sy, 20 * U * sy
    if pre is not None:
        sr = (r.square().mean(-1, keepdim=True) + eps).rsqrt()
        rel = 20 * U + err.norm(dim=-1, keepdim=True) / r.norm(dim=-1, keepdim=True).clamp_min(1e-300)
        n = r * sr * pre
        n_err = n.abs() * (rel + 2 * U) + err * sr * pre.abs()
        stats[:, 1:], stats_err[:, 1:] = sr, rel * sr
    return (r, n, stats), (err, n_err, stats_err)


def residual_bwd64(r, y, gate, post, pre, stats, dr, dn, act, alpha, sigma, factor):
    """The gradients for given r and stats, dgate of every row, and the errors."""
    sy, sr = stats[:, :1], stats[:, 1:]
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    sums = (128 + 256 + 3) * U  # a column: 128 rows a thread, then at most 256 threads, then 64 bits
    g, e = {}, {}
    d = dr if dr is not None else torch.zeros_like(r)
    err = U * d.abs()
    if pre is not None:
        rn, f = r * sr, dn * pre
        g["dpre"], e["dpre"] = (dn * rn).sum(0), sums * (dn * rn).abs().sum(0)
        d = d + sr * (f - rn * mean(f * rn))
        err = err + U * (d.abs() + sr * (4 * f.abs() + 40 * rn.abs() * mean((f * rn).abs())))
    g["dx"], e["dx"] = alpha * d, abs(alpha) * err + 2 * U * (alpha * d).abs()
    if y is None:
        return g, e
    d, err = sigma * factor * d, (abs(sigma) * factor) * err + 3 * U * (sigma * factor * d).abs()
    yn = y * sy
    if gate is not None:
        a, da = _act(gate, act)
        ra, ea = _act_err(gate, act)
        p = yn * post if post is not None else y
        g["dgate"] = d * p * da
        e["dgate"] = (p * da).abs() * err + (d * p).abs() * ea + 4 * U * g["dgate"].abs()
        d, err = d * a, a.abs() * err + (ra + U) * (d * a).abs()
    if post is not None:
        g["dpost"], e["dpost"] = (d * yn).sum(0), (yn.abs() * err).sum(0) + sums * (d * yn).abs().sum(0)
        d, err = d * post, post.abs() * err + U * (d * post).abs()
        m, em = mean(d * yn), mean(yn.abs() * err) + 40 * U * mean((d * yn).abs())
        err = sy * (err + yn.abs() * em + 3 * U * (d.abs() + yn.abs() * mean((d * yn).abs())))
        d = sy * (d - yn * m)
        err = err + 2 * U * d.abs()
    g["dy"], e["dy"] = d, err
    return g, e


def near(got, want, err, what=""):
    """got (a tensor of any device) within err of want, and half a step of its type."""
    got64 = got.detach().cpu().double().reshape(want.shape)
    bound = err + HALF[got.dtype] * (want.abs() + err)
    off = (got64 - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp_min(1e-300))[bad].max()))


def requests(B, T, cu):
    """(first row, behind the last) of each request among all rows."""
    return [(i * T, (i + 1) * T) for i in range(B)] if cu is None else list(zip(cu, cu[1:]))


def low_rank64(y, x, a, b, ids, scale, B, T, cu=None):
    """(out, h), both with the errors of f32 sums: a sum of n products is off by at most n
    half steps of the terms' magnitudes (however it is arranged, exact products, fewer
    joins than terms), the product with the scale and the last sum by three."""
    M, L, R, D = x.shape[0], *a.shape
    out, h = y.clone(), torch.zeros(M, R, dtype=F64)
    err, h_err = torch.zeros_like(y), torch.zeros_like(h)
    for n, (r0, r1) in enumerate(requests(B, T, cu)):
        l = int(ids[n])
        if not 0 <= l < L or r1 <= r0:
            continue
        s = float(scale[l]) if scale is not None else 1.0
        at = slice(r0, r1)
        h[at] = x[at] @ a[l].t()
        h_err[at] = (D + 8) * U * (x[at].abs() @ a[l].abs().t())
        e = s * (h[at] @ b[l])
        out[at] = y[at] + e
        err[at] = abs(s) * (h_err[at] @ b[l].abs() + (R + 2) * U * (h[at].abs() @ b[l].abs())) + U * out[at].abs()
    return (out, h), (err, h_err)


def low_rank_bwd64(x, a, b, ids, hidden, dy, scale, B, T, cu=None, dx=None):
    M, L, R, D = x.shape[0], *a.shape
    O = b.shape[2]
    g = {"dx": torch.zeros_like(x) if dx is None else dx.clone(), "da": torch.zeros_like(a), "db": torch.zeros_like(b)}
    e = {k: torch.zeros_like(v) for k, v in g.items()}
    for n, (r0, r1) in enumerate(requests(B, T, cu)):
        l = int(ids[n])
        if not 0 <= l < L or r1 <= r0:
            continue
        s = float(scale[l]) if scale is not None else 1.0
        at, rows = slice(r0, r1), r1 - r0
        dh = s * (dy[at] @ b[l].t())
        dh_err = (O + 9) * U * abs(s) * (dy[at].abs() @ b[l].abs().t())
        g["dx"][at] += dh @ a[l]
        e["dx"][at] = dh_err @ a[l].abs() + (R + 2) * U * (dh.abs() @ a[l].abs()) + U * g["dx"][at].abs()
        g["da"][l] += dh.t() @ x[at]
        e["da"][l] += dh_err.t() @ x[at].abs() + (min(rows, 4096) + 4) * U * (dh.abs().t() @ x[at].abs())
        g["db"][l] += s * (hidden[at].t() @ dy[at])
        e["db"][l] += (min(rows, 4096) + 4) * U * abs(s) * (hidden[at].abs().t() @ dy[at].abs())
    return g, e


def alike(got, want, what=""):
    """All of got as one vector: its error against want's length.  The roundings of sums
    have either sign, so that n of them come to about the square root of n half steps of
    sums like the result: 32 of them stand for 1024 terms' sums in two products one after
    the other; a result's own rounding is at most half a step, and of many results
    (uniform in it, and half a step at most of each value) 1/sqrt(3) of that."""
    off = float((got.detach().cpu().double().reshape(want.shape) - want).norm())
    size = float(want.norm())
    half = HALF[got.dtype] / (3 ** 0.5 if got.numel() >= 1000 else 1)  # (one result's is half a step, whatever the others')
    assert off <= (2 * 32 * U + half) * size, (what, off / max(size, 1e-300))
