"""The operators of a gated recurrent mixer beside GDN-2, as cases that can be timed.

Kinds (each one call of the package, and its plain form in elementary torch
operations):

  scan        gated_scan: h_t = e^{g_t} h_{t-1} + w_t v_t for every channel of
              [B, H, T, V], a state in and out, one token to long packed rows
  scan_bwd    gated_scan_backward: the gradients of g, v, w and the state
  norm        group_norm_act: group norm over channels-last rows, an activation
              or an activated gate in the same pass
  norm_bwd    group_norm_act_backward: the gradients of x, gate, weight, bias
  conv_bwd    short_conv_1d_backward: the gradients of the 4-tap causal conv
              with SiLU (x, weight, cache)

Sizes are those of the repository's configurations, benchmark and tests
(hidden 2048 with 16 heads of 128, heads of 64, 96 and 256, 8 x 4096 and
4 x 2048 tokens, 65536 tokens of one row), and odd ones between.
"""
import math
import os
import sys

import torch

own = False  # False: the plain forms; True: the package's operators

DEV = "cuda"
BF = torch.bfloat16


# -- cases ---------------------------------------------------------------------

def _scan_case(kind, name, B, T, H, V, bf16=False, per_head=False, w=True, state=True, seqs=0):
    c = {"kind": kind, "B": B, "T": T, "H": H, "V": V, "bf16": bf16, "per_head": per_head, "w": w, "state": state,
         "seqs": seqs}
    return dict(c, name=name) if name else c


def _norm_case(kind, name, N, S, C, groups, bf16=False, gate=False, act="silu"):
    c = {"kind": kind, "N": N, "S": S, "C": C, "groups": groups, "bf16": bf16, "gate": gate, "act": act}
    return dict(c, name=name) if name else c


def _conv_case(name, B, T, C, cache=True):
    c = {"kind": "conv_bwd", "B": B, "T": T, "C": C, "cache": cache}
    return dict(c, name=name) if name else c


def listed():
    return [
        # serving: 64 sequences take one token each into their carried states
        _scan_case("scan", "scan_step_b64", 64, 1, 16, 128),
        # a batch of prompts, the headline prefill size
        _scan_case("scan", "scan_prefill_b8_t4096", 8, 4096, 16, 128, state=False),
        # one row of packed documents in 16 bits, a decay for each head and token
        _scan_case("scan", "scan_packed_t65536", 1, 65536, 16, 128, bf16=True, per_head=True, seqs=37),
        # a training step's backward at the layer's training size
        _scan_case("scan_bwd", "scan_bwd_b4_t2048", 4, 2048, 16, 128, state=False),
        # the backward of packed documents in 16 bits, a decay for each head and token
        _scan_case("scan_bwd", "scan_bwd_packed_t32767", 1, 32767, 16, 128, bf16=True, per_head=True, seqs=19),
        # the norm of 64 decoded tokens per head, gated
        _norm_case("norm", "norm_step_b64", 64, 1, 2048, 16, gate=True),
        # ... of a batch of prompts in 16 bits
        _norm_case("norm", "norm_tokens_b8_t4096", 32768, 1, 2048, 16, bf16=True, gate=True),
        # whole sequences normalised as one sample each: a convolutional front end's norm
        _norm_case("norm", "norm_samples_b8_s4096", 8, 4096, 1024, 32),
        # training: the gated per-token norm at the layer's training size
        _norm_case("norm_bwd", "norm_bwd_tokens_b4_t2048", 8192, 1, 2048, 16, gate=True),
        # ... a front end's narrow groups in 16 bits, ragged
        _norm_case("norm_bwd", "norm_bwd_samples_s1999", 4, 1999, 320, 32, bf16=True),
        # training: the short conv before the recurrence
        _conv_case("conv_bwd_b4_t2048", 4, 2048, 2048, cache=False),
        # ... continuing from a cache, a few channels and a ragged length
        _conv_case("conv_bwd_c1536_t777", 3, 777, 1536),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan"] * 3 + ["scan_bwd"] * 2 + ["norm"] * 2 + ["norm_bwd"] * 2 + ["conv_bwd"])
    bf16 = rng.random() < 0.5
    if kind in ("scan", "scan_bwd"):
        V, H = rng.choice([33, 64, 64, 96, 100, 128, 128, 128, 256]), rng.choice([1, 2, 4, 8, 16])
        per_head, w, state = rng.random() < 0.4, rng.random() < 0.7, rng.random() < 0.6
        if kind == "scan" and rng.random() < 0.25:
            return _scan_case(kind, None, _log_int(rng, 1, 256), 1, H, V, bf16, per_head, w, True)
        M = _log_int(rng, 16, 65536 if kind == "scan" else 32768)
        if M >= 64 and rng.random() < 0.4:
            return _scan_case(kind, None, 1, M, H, V, bf16, per_head, w, state, rng.randint(1, min(64, M // 8)))
        B = min(M, _log_int(rng, 1, 16))
        return _scan_case(kind, None, B, M // B, H, V, bf16, per_head, w, state)
    if kind in ("norm", "norm_bwd"):
        groups, D = rng.choice([(1, 512), (4, 64), (8, 33), (8, 128), (16, 96), (16, 128), (32, 10), (32, 32), (2, 250)])
        act = rng.choice(["silu", "silu", "gelu", "none"])
        gate = rng.random() < 0.5
        M = _log_int(rng, 16, 32768)
        if rng.random() < 0.6:
            return _norm_case(kind, None, M, 1, groups * D, groups, bf16, gate, act)
        N = min(M // 2, _log_int(rng, 1, 16))
        return _norm_case(kind, None, N, M // N, groups * D, groups, bf16, gate, act)
    M = _log_int(rng, 16, 8192)
    B = min(M, _log_int(rng, 1, 8))
    return _conv_case(None, B, M // B, rng.choice([96, 250, 512, 1024, 1537, 2048]), rng.random() < 0.5)


# -- inputs ---------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 29)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _rand(g, lo, hi, *shape):
    return torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo


def _bounds(c, seed):
    """Token offsets of the packed sequences, [seqs + 1]: ragged, none empty."""
    g = torch.Generator()
    g.manual_seed(7 * int(seed) + 3)
    cuts = (torch.randperm(c["T"] - 1, generator=g)[:c["seqs"] - 1] + 1).sort().values
    return [0] + cuts.tolist() + [c["T"]]


def _prepare_scan(c, seed):
    g = _gen(seed)
    B, T, H, V = c["B"], c["T"], c["H"], c["V"]
    ty = BF if c["bf16"] else torch.float32
    # the layout that a projection leaves, [B, T, H, V], seen as [B, H, T, V]
    rows = lambda x: x.transpose(1, 2)  # noqa: E731
    # decays that remember between 2 and 1000 tokens
    s = {"g": rows(-torch.exp(_rand(g, math.log(1e-3), math.log(0.5), B, T, H, 1 if c["per_head"] else V))),
         "v": rows(_randn(g, B, T, H, V).to(ty)),
         "w": rows(torch.sigmoid(_randn(g, B, T, H, V)).to(ty)) if c["w"] else None,
         "state": _randn(g, c["seqs"] or B, H, V) if c["state"] else None, "cu": None}
    if c["seqs"]:
        s["cu"] = torch.tensor(_bounds(c, seed), dtype=torch.int32, device=DEV)
    if c["kind"] == "scan_bwd":
        s["out"] = _plain_scan(s)[0]
        s["d_out"] = rows(_randn(g, B, T, H, V).to(ty))
        s["d_state"] = _randn(g, c["seqs"] or B, H, V) if c["state"] else None
    return s


def _prepare_norm(c, seed):
    g = _gen(seed)
    N, S, C = c["N"], c["S"], c["C"]
    ty = BF if c["bf16"] else torch.float32
    x = _randn(g, N, S, C)
    x.mul_(_rand(g, 0.5, 2.0, C)).add_(_randn(g, C))
    s = {"x": x.to(ty), "gate": _randn(g, N, S, C).to(ty) if c["gate"] else None, "weight": _rand(g, 0.5, 1.5, C),
         "bias": _randn(g, C) * 0.2, "groups": c["groups"], "act": c["act"]}
    if c["kind"] == "norm_bwd":
        s["stats"] = _plain_stats(s["x"], c["groups"])
        s["d_out"] = _randn(g, N, S, C).to(ty)
    return s


def _prepare_conv(c, seed):
    g = _gen(seed)
    B, T, C = c["B"], c["T"], c["C"]
    return {"x": _randn(g, B, T, C), "weight": _rand(g, -0.5, 0.5, C, 4),
            "cache": _randn(g, B, 3, C) if c["cache"] else None, "d_out": _randn(g, B, T, C),
            "d_cache": _randn(g, B, 3, C) if c["cache"] else None}


def prepare(case, seed):
    c = dict(case)
    f = _prepare_scan if c["kind"] in ("scan", "scan_bwd") else _prepare_conv if c["kind"] == "conv_bwd" else _prepare_norm
    return dict(f(c, seed), kind=c["kind"])


# -- the plain forms ----------------------------------------------------------------

EPS = 1e-5


def _recurrence(a, x):
    """y_t = a_t y_{t-1} + x_t along dim 2 (y_{-1} = 0): spans of 1, 2, 4, ...
    tokens are joined, y_t += (a_t .. a_{t-d+1}) y_{t-d}.  Overwrites both."""
    d, T = 1, x.shape[2]
    while d < T:
        x[:, :, d:] += a[:, :, d:] * x[:, :, :-d]
        if 2 * d < T:
            a[:, :, d:] = a[:, :, d:] * a[:, :, :-d]
        d *= 2
    return x


def _full(g, v):
    return g.expand(v.shape)


def _plain_scan(s):
    g, v, w, h0, cu = s["g"], s["v"], s["w"], s["state"], s["cu"]
    B, H, T, V = v.shape
    a = _full(g, v).float().exp()
    x = v.float() * w.float() if w is not None else v.float().clone()
    if cu is not None:
        first, last = cu[:-1].long(), cu[1:].long() - 1
        if h0 is not None:
            x[0, :, first] += a[0, :, first] * h0.transpose(0, 1)
        a[0, :, first] = 0
    elif h0 is not None:
        x[:, :, 0] += a[:, :, 0] * h0
    h = _recurrence(a, x)
    state = h[0, :, last].transpose(0, 1).contiguous() if cu is not None else h[:, :, -1].clone()
    return h.to(v.dtype), state


def _plain_scan_bwd(s):
    g, v, w, h0, cu, dS = s["g"], s["v"], s["w"], s["state"], s["cu"], s["d_state"]
    B, H, T, V = v.shape
    a = _full(g, v).float().exp()
    d = s["d_out"].float().clone()
    before = torch.zeros_like(d)  # the state before each token
    before[:, :, 1:] = s["out"].float()[:, :, :-1]
    nxt = torch.zeros_like(d)  # the decay after each token
    nxt[:, :, :-1] = a[:, :, 1:]
    if cu is not None:
        first, last = cu[:-1].long(), cu[1:].long() - 1
        before[0, :, first] = h0.transpose(0, 1) if h0 is not None else 0.0
        nxt[0, :, last] = 0
        if dS is not None:
            d[0, :, last] += dS.transpose(0, 1)
    else:
        first = None
        if h0 is not None:
            before[:, :, 0] = h0
        if dS is not None:
            d[:, :, -1] += dS
    d = _recurrence(nxt.flip(2), d.flip(2)).flip(2)  # dL/dh_t
    e = a * d
    dh0 = e[0, :, first].transpose(0, 1).contiguous() if cu is not None else e[:, :, 0].clone()
    dg = e * before
    if g.shape[3] == 1:
        dg = dg.sum(3, keepdim=True)
    return {"dg": dg, "dv": (d * w.float() if w is not None else d).to(v.dtype),
            "dw": (d * v.float()).to(v.dtype) if w is not None else None, "dS0": dh0}


def _plain_stats(x, groups):
    """[N, groups, 2]: the mean and 1 / sqrt(variance + eps) of each group."""
    N, S, C = x.shape
    r = x.float().view(N, S, groups, C // groups)
    mean = r.mean((1, 3), keepdim=True)
    var = ((r - mean) ** 2).mean((1, 3), keepdim=True)
    return torch.stack([mean, (var + EPS).rsqrt()], -1).view(N, groups, 2)


def _act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _d_act(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _normalised(x, stats, groups):
    N, S, C = x.shape
    r = x.float().view(N, S, groups, C // groups)
    return ((r - stats[:, None, :, 0:1]) * stats[:, None, :, 1:2]).view(N, S, C)


def _plain_norm(s):
    x, act = s["x"], s["act"]
    z = _normalised(x, _plain_stats(x, s["groups"]), s["groups"]) * s["weight"] + s["bias"]
    return (z * _act(s["gate"].float(), act) if s["gate"] is not None else _act(z, act)).to(x.dtype)


def _plain_norm_bwd(s):
    x, act, groups = s["x"], s["act"], s["groups"]
    N, S, C = x.shape
    n = _normalised(x, s["stats"], groups)
    z = n * s["weight"] + s["bias"]
    dy, dgate = s["d_out"].float(), None
    if s["gate"] is not None:
        gate = s["gate"].float()
        dz, dgate = dy * _act(gate, act), (dy * z * _d_act(gate, act)).to(x.dtype)
    else:
        dz = dy * _d_act(z, act)
    dn = (dz * s["weight"]).view(N, S, groups, C // groups)
    n4 = n.view(N, S, groups, C // groups)
    dx = dn - dn.mean((1, 3), keepdim=True) - n4 * (dn * n4).mean((1, 3), keepdim=True)
    dx = dx * s["stats"][:, None, :, 1:2]
    return {"dx": dx.view(N, S, C).to(x.dtype), "dgate": dgate, "dweight": (dz * n).sum((0, 1)), "dbias": dz.sum((0, 1))}


def _plain_conv_bwd(s):
    x, w, cache = s["x"], s["weight"], s["cache"]
    B, T, C = x.shape
    pad = cache if cache is not None else x[:, :1].expand(B, 3, C)
    xp = torch.cat([pad, x], 1)
    z = xp[:, 0:T] * w[:, 0] + xp[:, 1:T + 1] * w[:, 1] + xp[:, 2:T + 2] * w[:, 2] + xp[:, 3:T + 3] * w[:, 3]
    dz = s["d_out"] * _d_act(z, "silu")
    dw = torch.stack([(dz * xp[:, 0:T]).sum((0, 1)), (dz * xp[:, 1:T + 1]).sum((0, 1)),
                      (dz * xp[:, 2:T + 2]).sum((0, 1)), (dz * xp[:, 3:T + 3]).sum((0, 1))], 1)
    dp = torch.zeros_like(xp)
    dp[:, 0:T] += dz * w[:, 0]
    dp[:, 1:T + 1] += dz * w[:, 1]
    dp[:, 2:T + 2] += dz * w[:, 2]
    dp[:, 3:T + 3] += dz * w[:, 3]
    if s["d_cache"] is not None:
        dp[:, T:] += s["d_cache"]
    dx = dp[:, 3:].contiguous()
    if cache is None:
        dx[:, 0] += dp[:, :3].sum(1)
        return {"dx": dx, "dweight": dw, "dcache": None}
    return {"dx": dx, "dweight": dw, "dcache": dp[:, :3].contiguous()}


# -- a pass ---------------------------------------------------------------------------

def _package():
    pkg = os.path.join(os.getcwd(), "burn-gdn2_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gdn2_amd

    return gdn2_amd


def _own(s):
    G, kind = _package(), s["kind"]
    if kind == "scan":
        return G.gated_scan(s["g"], s["v"], s["w"], s["state"], cu_seqlens=s["cu"])
    if kind == "scan_bwd":
        return G.gated_scan_backward(s["g"], s["v"], s["w"], s["out"], s["d_out"], s["state"], d_state=s["d_state"],
                                     cu_seqlens=s["cu"])
    if kind == "norm":
        return G.group_norm_act(s["x"], s["groups"], s["weight"], s["bias"], EPS, s["act"], gate=s["gate"])
    if kind == "norm_bwd":
        return G.group_norm_act_backward(s["x"], s["groups"], s["stats"], s["d_out"], s["weight"], s["bias"], s["act"],
                                         gate=s["gate"])
    return G.short_conv_1d_backward(s["x"], s["weight"], s["d_out"], s["cache"], d_cache=s["d_cache"])


_PLAIN = {"scan": _plain_scan, "scan_bwd": _plain_scan_bwd, "norm": _plain_norm, "norm_bwd": _plain_norm_bwd,
          "conv_bwd": _plain_conv_bwd}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["kind"]](state)


# -- what a pass cannot do without ------------------------------------------------------

def work(case):
    c = case
    if c["kind"] in ("scan", "scan_bwd"):
        rows = c["B"] * c["T"] * c["H"]
        n, e, gb = rows * c["V"], 2 if c["bf16"] else 4, 4 * rows * (1 if c["per_head"] else c["V"])
        st = 4 * (c["seqs"] or c["B"]) * c["H"] * c["V"]
        w = n * e if c["w"] else 0
        if c["kind"] == "scan":  # g, v, w, the state; h and the new state.  An exponential, two products, a sum
            return {"bytes": gb + 2 * n * e + w + st + (st if c["state"] else 0), "flops": 4 * n}
        # g, v (for dw alone), w, h, dh, both states; dg, dv, dw, dS0
        v = n * e if c["w"] else 0
        return {"bytes": 2 * gb + 3 * n * e + 2 * w + v + st + (2 * st if c["state"] else 0), "flops": 7 * n}
    if c["kind"] in ("norm", "norm_bwd"):
        n, e = c["N"] * c["S"] * c["C"], 2 if c["bf16"] else 4
        if c["kind"] == "norm":
            return {"bytes": n * e * (3 if c["gate"] else 2) + 8 * c["C"], "flops": n * 12}
        return {"bytes": n * e * (5 if c["gate"] else 3) + 16 * c["C"] + 8 * c["N"] * c["groups"], "flops": n * 24}
    n = c["B"] * c["T"] * c["C"]
    return {"bytes": 4 * (3 * n + 8 * c["C"] + (9 * c["B"] * c["C"] if c["cache"] else 0)), "flops": n * 32}


# -- 64 bits, from the definitions --------------------------------------------------------

def _exact_scan(c, s):
    """Token by token."""
    g, v = s["g"].double(), s["v"].double()
    u = v * s["w"].double() if s["w"] is not None else v
    B, H, T, V = v.shape
    cu = _list(s["cu"])
    rows = cu is not None and {t: n for n, t in enumerate(cu[:-1])}
    a, h0 = g.exp().unbind(2), s["state"].double() if s["state"] is not None else torch.zeros(
        c["seqs"] or B, H, V, dtype=torch.float64, device=DEV)
    h, out, ends = h0, torch.empty(T, B, H, V, dtype=torch.float64, device=DEV), []
    for t, ut in enumerate(u.unbind(2)):
        if cu is not None and t in rows:
            if t:
                ends.append(h)
            h = h0[rows[t]:rows[t] + 1]
        h = torch.addcmul(ut, a[t], h)
        out[t] = h
    ends.append(h)
    return out.permute(1, 2, 0, 3), torch.cat(ends) if cu is not None else h


def _exact_scan_bwd(c, s):
    """Token by token, from the last."""
    g, v, out, dy = s["g"].double(), s["v"].double(), s["out"].double(), s["d_out"].double()
    B, H, T, V = v.shape
    N = c["seqs"] or B
    zeros = torch.zeros(N, H, V, dtype=torch.float64, device=DEV)
    h0 = s["state"].double() if s["state"] is not None else zeros
    dS = s["d_state"].double() if s["d_state"] is not None else zeros
    cu = _list(s["cu"])
    starts = {t: n for n, t in enumerate(cu[:-1])} if cu is not None else {0: None}
    ends = {t - 1: n for n, t in enumerate(cu[1:])} if cu is not None else {T - 1: None}
    pick = lambda x, n: x if n is None else x[n:n + 1]  # noqa: E731
    D, E = torch.empty(T, B, H, V, dtype=torch.float64, device=DEV), torch.empty(T, B, H, V, dtype=torch.float64, device=DEV)
    a, dh0, e = g.exp().unbind(2), torch.empty_like(zeros), None
    dyt = dy.unbind(2)
    for t in range(T - 1, -1, -1):
        if t in ends:
            e = pick(dS, ends[t])
        d = dyt[t] + e
        D[t] = d
        e = d * a[t]
        E[t] = e
        if t in starts:
            pick(dh0, starts[t]).copy_(e)
    D, E = D.permute(1, 2, 0, 3), E.permute(1, 2, 0, 3)
    before = out.roll(1, 2)
    for t, n in starts.items():
        before[:, :, t] = pick(h0, n)
    dg = E * before
    return {"dg": dg.sum(3, keepdim=True) if g.shape[3] == 1 else dg,
            "dv": D * s["w"].double() if s["w"] is not None else D, "dw": D * v if s["w"] is not None else None,
            "dS0": dh0}


def _list(cu):
    return None if cu is None else cu.tolist()


def _norm64(x, gate, weight, bias, groups, act):
    import torch.nn.functional as F

    N, S, C = x.shape
    f = {"silu": F.silu, "gelu": F.gelu, "none": lambda z: z}[act]
    var, mean = torch.var_mean(x.view(N, S, groups, C // groups), (1, 3), unbiased=False, keepdim=True)
    z = torch.addcmul(bias, ((x.view(N, S, groups, C // groups) - mean) / (var + EPS).sqrt()).view(N, S, C), weight)
    return z * f(gate) if gate is not None else f(z)


def _exact_norm(c, s):
    d = lambda x: None if x is None else x.double()  # noqa: E731
    return _norm64(d(s["x"]), d(s["gate"]), d(s["weight"]), d(s["bias"]), c["groups"], c["act"])


def _exact_norm_bwd(c, s):
    leaf = lambda x: None if x is None else x.double().requires_grad_()  # noqa: E731
    x, gate, weight, bias = leaf(s["x"]), leaf(s["gate"]), leaf(s["weight"]), leaf(s["bias"])
    y = _norm64(x, gate, weight, bias, c["groups"], c["act"])
    y.backward(s["d_out"].double())
    return {"dx": x.grad, "dgate": None if gate is None else gate.grad, "dweight": weight.grad, "dbias": bias.grad}


def _exact_conv_bwd(c, s):
    import torch.nn.functional as F

    leaf = lambda x: None if x is None else x.double().requires_grad_()  # noqa: E731
    x, w, cache = leaf(s["x"]), leaf(s["weight"]), leaf(s["cache"])
    B, T, C = x.shape
    xp = torch.cat([cache if cache is not None else x[:, :1].expand(B, 3, C), x], 1)
    z = sum(xp[:, i:i + T] * w[:, i] for i in range(4))
    loss = (F.silu(z) * s["d_out"].double()).sum()
    if s["d_cache"] is not None:
        loss = loss + (xp[:, T:] * s["d_cache"].double()).sum()
    loss.backward()
    return {"dx": x.grad, "dweight": w.grad, "dcache": None if cache is None else cache.grad}


_EXACT = {"scan": _exact_scan, "scan_bwd": _exact_scan_bwd, "norm": _exact_norm, "norm_bwd": _exact_norm_bwd,
          "conv_bwd": _exact_conv_bwd}


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))
