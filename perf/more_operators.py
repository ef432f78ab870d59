"""What stands around the mixer in a block that is trained and served, as cases
that can be timed.

Kinds (each one call of the package, and its plain form in elementary torch
operations):

  drop       dropout and dropout_backward: a mask from a counter-based
             generator, formed where it is needed and never stored
  res        residual_norm: the norm behind a block, its gate, dropout, the
             scaled residual and the norm before the next block, one pass
  res_bwd    residual_norm_backward: the gradients of x, y, gate and both weights
  lora       low_rank_add: every request's own low-rank adapter beside a
             projection that all requests share
  lora_bwd   low_rank_add_backward: the gradients of x and of the adapters

Sizes are those of the repository's configurations, benchmark and tests
(hidden 2048, 8 x 4096 and 4 x 2048 tokens, 64 decoded tokens, front ends of
320 channels), and odd ones between.
"""
import math
import os
import sys

import numpy as np
import torch

own = False  # False: the plain forms; True: the package's operators

DEV = "cuda"
BF = torch.bfloat16
EPS = 1e-5


# -- cases ---------------------------------------------------------------------

def _drop_case(name, rows, C, bf16=False, p=0.1, bwd=False):
    c = {"kind": "drop", "rows": rows, "C": C, "bf16": bf16, "p": p, "bwd": bwd}
    return dict(c, name=name) if name else c


def _res_case(kind, name, N, S, C, ty, gate="none", act="none", post=True, pre=True, p=0.0, alpha=1.0, sigma=1.0):
    c = {"kind": kind, "N": N, "S": S, "C": C, "ty": ty, "gate": gate, "act": act, "post": post, "pre": pre, "p": p,
         "alpha": alpha, "sigma": sigma}
    return dict(c, name=name) if name else c


def _lora_case(kind, name, B, T, D, O, R, L, bf16=False, seqs=0):
    c = {"kind": kind, "B": B, "T": T, "D": D, "O": O, "R": R, "L": L, "bf16": bf16, "seqs": seqs}
    return dict(c, name=name) if name else c


def listed():
    return [
        # training: the activations of a batch of prompts in 16 bits
        _drop_case("drop_b8_t4096", 32768, 2048, bf16=True),
        # the gradient's pass over odd rows in 32 bits
        _drop_case("drop_bwd_c1537_t777", 3 * 777, 1537, p=0.25, bwd=True),
        # serving: 64 decoded tokens between two blocks
        _res_case("res", "res_step_b64", 64, 1, 2048, "f32"),
        # ... a batch of prompts in 16 bits, the block's output gated per channel and token
        _res_case("res", "res_b8_t4096", 8, 4096, 2048, "bf16", gate="full", act="silu"),
        # training: a 32-bit residual stream, blocks in 16 bits, dropout and a learned scale for each channel
        _res_case("res", "res_train_b4_t2048", 4, 2048, 2048, "mixed", gate="channel", p=0.1, sigma=0.5),
        # the backward at the training size, gated and with dropout
        _res_case("res_bwd", "res_bwd_b4_t2048", 4, 2048, 2048, "bf16", gate="full", act="silu", p=0.1),
        # ... of a narrow front end, one gate a sample
        _res_case("res_bwd", "res_bwd_s1999_c320", 4, 1999, 320, "f32", gate="sample", act="sigmoid", alpha=0.8),
        # serving: 64 requests take one token each through 16 adapters
        _lora_case("lora", "lora_step_b64", 64, 1, 2048, 2048, 16, 16),
        # ... their prompts, the headline prefill size
        _lora_case("lora", "lora_b8_t4096", 8, 4096, 2048, 2048, 16, 4),
        # ... packed prompts in 16 bits, larger adapters
        _lora_case("lora", "lora_packed_t32767", 1, 32767, 2048, 2048, 64, 8, bf16=True, seqs=37),
        # training an adapter at the layer's training size
        _lora_case("lora_bwd", "lora_bwd_b4_t2048", 4, 2048, 2048, 2048, 16, 1, bf16=True),
        # ... several at once on packed documents, ragged
        _lora_case("lora_bwd", "lora_bwd_packed_t3001", 1, 3001, 1537, 1000, 24, 5, seqs=19),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["drop", "res", "res", "res_bwd", "res_bwd", "lora", "lora", "lora", "lora_bwd", "lora_bwd"])
    bf16 = rng.random() < 0.5
    if kind == "drop":
        return _drop_case(None, _log_int(rng, 16, 32768), rng.choice([96, 250, 320, 1024, 1537, 2048]), bf16,
                          rng.choice([0.05, 0.1, 0.25, 0.5]), rng.random() < 0.5)
    if kind in ("res", "res_bwd"):
        C = rng.choice([64, 96, 250, 320, 512, 1000, 1024, 1537, 2048, 2048, 4096])
        M = _log_int(rng, 1 if kind == "res" else 16, 32768 * 2048 // max(C, 2048) // (1 if kind == "res" else 4))
        N = min(M, _log_int(rng, 1, 64))
        gate = rng.choice(["none", "full", "full", "sample", "channel"])
        return _res_case(kind, None, N, M // N, C, rng.choice(["f32", "bf16", "bf16", "mixed"]), gate,
                         rng.choice(["none", "sigmoid", "silu"]) if gate != "none" else "none",
                         rng.random() < 0.7, rng.random() < 0.8, rng.choice([0.0, 0.1, 0.25]),
                         rng.choice([1.0, 0.8]), rng.choice([1.0, 0.5]))
    D, O = rng.choice([64, 250, 512, 1024, 1537, 2048, 2048]), rng.choice([64, 333, 1000, 1024, 2048, 2048])
    R, L = rng.choice([1, 4, 8, 16, 16, 24, 32, 64]), rng.choice([1, 2, 5, 16])
    if kind == "lora" and rng.random() < 0.3:
        return _lora_case(kind, None, _log_int(rng, 1, 256), 1, D, O, R, L, bf16)
    M = _log_int(rng, 16, 32768 if kind == "lora" else 8192)
    if M >= 64 and rng.random() < 0.5:
        return _lora_case(kind, None, 1, M, D, O, R, L, bf16, rng.randint(1, min(64, M // 8)))
    B = min(M, _log_int(rng, 1, 16))
    return _lora_case(kind, None, B, M // B, D, O, R, L, bf16)


# -- inputs ---------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 41)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _rand(g, lo, hi, *shape):
    return torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo


def _counters(seed):
    """The generator's seed and first counter of a step: 64 bits, and past 32."""
    return (int(seed) * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63), (1 << 33) + int(seed) % 1000003


def _prepare_drop(c, seed):
    x = _randn(_gen(seed), c["rows"], c["C"])
    key, offset = _counters(seed)
    return {"x": x.to(BF) if c["bf16"] else x, "p": c["p"], "seed": key, "offset": offset, "bwd": c["bwd"]}


def _prepare_res(c, seed):
    g = _gen(seed)
    N, S, C = c["N"], c["S"], c["C"]
    stream, branch = {"f32": (torch.float32,) * 2, "bf16": (BF, BF), "mixed": (torch.float32, BF)}[c["ty"]]
    x = _randn(g, N, S, C).mul_(_rand(g, 0.5, 2.0, C))
    y = _randn(g, N, S, C).mul_(_rand(g, 0.2, 1.0, C))
    gate = {"none": None, "full": (N, S, C), "sample": (N, 1, C), "channel": (C,)}[c["gate"]]
    if gate is not None:
        gate = _randn(g, *gate).to(branch)
    key, offset = _counters(seed)
    s = {"x": x.to(stream), "y": y.to(branch), "gate": gate, "act": c["act"], "alpha": c["alpha"], "sigma": c["sigma"],
         "post": _rand(g, 0.5, 1.5, C) if c["post"] else None, "pre": _rand(g, 0.5, 1.5, C) if c["pre"] else None,
         "p": c["p"], "seed": key, "offset": offset}
    if c["kind"] == "res_bwd":
        s["out"] = _plain_res(s)["out"]
        s["stats"] = _stats(s, _rstd(s["y"].float()), _rstd(s["out"].float()))
        s["d_out"] = _randn(g, N, S, C).to(stream)
        s["d_normed"] = _randn(g, N, S, C).to(branch) if c["pre"] else None
        del s["x"]
    return s


def _bounds(c, seed):
    """Token offsets of the packed requests, [seqs + 1]: ragged, none empty."""
    g = torch.Generator()
    g.manual_seed(11 * int(seed) + 5)
    cuts = (torch.randperm(c["T"] - 1, generator=g)[:c["seqs"] - 1] + 1).sort().values
    return [0] + cuts.tolist() + [c["T"]]


def _prepare_lora(c, seed):
    g = _gen(seed)
    B, T, D, O, R, L = c["B"], c["T"], c["D"], c["O"], c["R"], c["L"]
    ty = BF if c["bf16"] else torch.float32
    n = c["seqs"] or B
    bounds = _bounds(c, seed) if c["seqs"] else None
    s = {"x": _randn(g, B, T, D).to(ty), "a": (_randn(g, L, R, D) * D ** -0.5).to(ty),
         "b": (_randn(g, L, R, O) * R ** -0.5).to(ty), "scale": _rand(g, 0.5, 2.0, L),
         "ids": torch.randint(0, L, (n,), generator=g, device=DEV, dtype=torch.int32),
         "cu": torch.tensor(bounds, dtype=torch.int32, device=DEV) if bounds else None,
         "longest": max(v - u for u, v in zip(bounds, bounds[1:])) if bounds else T}
    if c["kind"] == "lora":
        s["y"] = _randn(g, B, T, O).to(ty)
    else:
        s["d_out"] = _randn(g, B, T, O).to(ty)
        s["hidden"] = _rows_back(s, torch.bmm(_by_request(s, s["x"]), s["a"].float()[s["ids"].long()].transpose(1, 2).contiguous()))
    return s


def prepare(case, seed):
    c = dict(case)
    f = {"drop": _prepare_drop, "res": _prepare_res, "res_bwd": _prepare_res}.get(c["kind"], _prepare_lora)
    return dict(f(c, seed), kind=c["kind"])


# -- the plain forms ----------------------------------------------------------------

_LOW = 0xFFFFFFFF


def _words(rows, C, seed, offset):
    """The generator's 32-bit words of [rows, C]: Philox-4x32 of 7 rounds (Salmon,
    Moraes, Dror, Shaw 2011), counter offset + row ceil(C / 4) + c / 4, word c % 4."""
    q = -(-C // 4)
    n = torch.arange(rows * q, dtype=torch.int64, device=DEV) + offset
    c0, c1, c2, c3 = n & _LOW, (n >> 32) & _LOW, torch.zeros_like(n), torch.zeros_like(n)
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(7):
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (the low 64 bits)
        c0, c1, c2, c3 = ((m1 >> 32) & _LOW) ^ c1 ^ k0, m1 & _LOW, ((m0 >> 32) & _LOW) ^ c3 ^ k1, m0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack([c0, c1, c2, c3], -1).view(rows, 4 * q)[:, :C]


def _dropped(x, p, seed, offset):
    """x in 32 bits with a share p of it 0 and the rest over 1 - p."""
    if p == 0:
        return x
    rows, C = x.numel() // x.shape[-1], x.shape[-1]
    keep = (_words(rows, C, seed, offset) >> 8) >= int(p * 2 ** 24 + 0.5)
    return torch.where(keep.view(x.shape), x * (1 / (1 - p)), 0.0)


def _plain_drop(s):
    return _dropped(s["x"].float(), s["p"], s["seed"], s["offset"]).to(s["x"].dtype)


def _rstd(x):
    return ((x * x).mean(-1) + EPS).rsqrt()


def _act(z, act):
    s = torch.sigmoid(z)
    return {"none": z, "sigmoid": s, "silu": z * s}[act]


def _d_act(z, act):
    s = torch.sigmoid(z)
    return {"none": torch.ones_like(z), "sigmoid": s * (1 - s), "silu": s * (1 + z * (1 - s))}[act]


def _plain_res(s):
    x, y = s["x"], s["y"].float()
    sy = _rstd(y)
    b = y * sy[..., None] * s["post"] if s["post"] is not None else y
    if s["gate"] is not None:
        b = b * _act(s["gate"].float(), s["act"])
    r = s["alpha"] * x.float() + s["sigma"] * _dropped(b, s["p"], s["seed"], s["offset"])
    sr = _rstd(r)
    n = (r * sr[..., None] * s["pre"]).to(s["y"].dtype) if s["pre"] is not None else None
    return {"out": r.to(x.dtype), "normed": n, "stats": _stats(s, sy, sr)}


def _stats(s, sy, sr):
    """0 where a norm is not taken."""
    return torch.stack([sy * (s["post"] is not None), sr * (s["pre"] is not None)], -1)


def _plain_res_bwd(s):
    out, y, gate = s["out"], s["y"].float(), s["gate"]
    sy, sr = s["stats"][..., 0:1], s["stats"][..., 1:2]
    d, dpre, dpost, dgate = s["d_out"].float(), None, None, None
    if s["pre"] is not None:
        rn, dn = out.float() * sr, s["d_normed"].float()
        dpre = (dn * rn).sum((0, 1))
        dn = dn * s["pre"]
        d = d + sr * (dn - rn * (dn * rn).mean(-1, keepdim=True))
    db = _dropped(s["sigma"] * d, s["p"], s["seed"], s["offset"])
    yn = y * sy
    p = yn * s["post"] if s["post"] is not None else y
    if gate is not None:
        z = gate.float()
        dgate = db * p * _d_act(z, s["act"])
        if gate.dim() == 1:
            dgate = dgate.sum((0, 1))
        elif gate.shape[1] != y.shape[1]:
            dgate = dgate.sum(1, keepdim=True)
        dgate = dgate.to(gate.dtype)
        db = db * _act(z, s["act"])
    if s["post"] is not None:
        dpost = (db * yn).sum((0, 1))
        db = db * s["post"]
        db = sy * (db - yn * (db * yn).mean(-1, keepdim=True))
    return {"dx": (s["alpha"] * d).to(out.dtype), "dy": db.to(s["y"].dtype), "dgate": dgate, "dpost": dpost, "dpre": dpre}


def _by_request(s, t):
    """The rows of each request in 32 bits, [requests, longest, ...], zeros behind its last."""
    if s["cu"] is None:
        return t.float()
    at, ok = _places(s)
    return t[0].float()[at] * ok[..., None]


def _places(s):
    cu = s["cu"].long()
    at = cu[:-1, None] + torch.arange(s["longest"], device=DEV)
    ok = at < cu[1:, None]
    return torch.where(ok, at, 0), ok


def _rows_back(s, t):
    """_by_request's rows back at their places."""
    if s["cu"] is None:
        return t
    at, ok = _places(s)
    r = torch.zeros((1, s["x"].shape[1], t.shape[2]), device=DEV)
    r[0, at[ok]] = t[ok]
    return r


def _plain_lora(s):
    ids = s["ids"].long()
    h = torch.bmm(_by_request(s, s["x"]), s["a"].float()[ids].transpose(1, 2).contiguous())
    e = torch.bmm(h, s["b"].float()[ids]) * s["scale"][ids][:, None, None]
    return (s["y"].float() + _rows_back(s, e)).to(s["y"].dtype)


def _plain_lora_bwd(s):
    ids, L = s["ids"].long(), s["a"].shape[0]
    dy = _by_request(s, s["d_out"]) * s["scale"][ids][:, None, None]
    x, h = _by_request(s, s["x"]), _by_request(s, s["hidden"])
    dh = torch.bmm(dy, s["b"].float()[ids].transpose(1, 2).contiguous())
    dx = torch.bmm(dh, s["a"].float()[ids])
    da, db = torch.bmm(dh.transpose(1, 2).contiguous(), x), torch.bmm(h.transpose(1, 2).contiguous(), dy)
    of = (torch.arange(L, device=DEV)[:, None] == ids).float()  # the requests of each adapter
    return {"dx": _rows_back(s, dx).to(s["x"].dtype), "da": (of @ da.flatten(1)).view(L, *da.shape[1:]),
            "db": (of @ db.flatten(1)).view(L, *db.shape[1:])}


# -- a pass ---------------------------------------------------------------------------

def _package():
    pkg = os.path.join(os.getcwd(), "burn-gdn2_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gdn2_amd

    return gdn2_amd


def _own(s):
    G, kind = _package(), s["kind"]
    if kind == "drop":
        f = G.dropout_backward if s["bwd"] else G.dropout
        return f(s["x"], s["p"], s["seed"], s["offset"])
    if kind == "res":
        out, normed, stats = G.residual_norm(s["x"], s["y"], s["gate"], s["post"], s["pre"], EPS, s["act"], s["alpha"],
                                             s["sigma"], s["p"], s["seed"], s["offset"], return_stats=True)
        return {"out": out, "normed": normed, "stats": stats}
    if kind == "res_bwd":
        return G.residual_norm_backward(s["out"], s["y"], s["stats"], s["d_out"], s["d_normed"], s["gate"], s["post"],
                                        s["pre"], s["act"], s["alpha"], s["sigma"], s["p"], s["seed"], s["offset"])
    if kind == "lora":
        return G.low_rank_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scale"], cu_seqlens=s["cu"])
    return G.low_rank_add_backward(s["x"], s["a"], s["b"], s["ids"], s["hidden"], s["d_out"], s["scale"], cu_seqlens=s["cu"])


_PLAIN = {"drop": _plain_drop, "res": _plain_res, "res_bwd": _plain_res_bwd, "lora": _plain_lora,
          "lora_bwd": _plain_lora_bwd}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["kind"]](state)


# -- what a pass cannot do without ------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "drop":
        n = c["rows"] * c["C"]
        return {"bytes": 2 * n * (2 if c["bf16"] else 4), "flops": n}
    if c["kind"] in ("res", "res_bwd"):
        M = c["N"] * c["S"]
        n = M * c["C"]
        es, eb = {"f32": (4, 4), "bf16": (2, 2), "mixed": (4, 2)}[c["ty"]]
        gate = {"none": 0, "full": n, "sample": c["N"] * c["C"], "channel": c["C"]}[c["gate"]]
        weights = 4 * c["C"] * (c["post"] + c["pre"])
        if c["kind"] == "res":  # x, y, the gate, the weights; out, normed, two statistics a row
            return {"bytes": n * (2 * es + eb + (eb if c["pre"] else 0)) + gate * eb + weights + 8 * M, "flops": 12 * n}
        # out, y, the gate, d_out, d_normed, the statistics; dx, dy, dgate and the weights' gradients
        return {"bytes": n * (2 * es + 2 * eb + ((es + eb) if c["pre"] else 0)) + 2 * gate * eb + 2 * weights + 8 * M,
                "flops": 24 * n}
    M, R, e = c["B"] * c["T"], c["R"], 2 if c["bf16"] else 4
    used = min(c["L"], c["seqs"] or c["B"])
    w = used * R * (c["D"] + c["O"])
    if c["kind"] == "lora":
        return {"bytes": e * (M * (c["D"] + 2 * c["O"]) + w), "flops": 2 * M * R * (c["D"] + c["O"])}
    return {"bytes": e * (M * (2 * c["D"] + c["O"]) + w) + 4 * (M * R + c["L"] * R * (c["D"] + c["O"])),
            "flops": 4 * M * R * (c["D"] + c["O"])}


# -- 64 bits, from the definitions --------------------------------------------------------

def _mask64(rows, C, p, seed, offset):
    """The factors of [rows, C], 0 or 1 / (1 - p)."""
    q = (C + 3) // 4
    n = np.arange(rows * q, dtype=np.uint64) + np.uint64(offset)
    mask, half = np.uint64(_LOW), np.uint64(32)
    v = [n & mask, n >> half, np.zeros_like(n), np.zeros_like(n)]
    for i in range(7):
        key = [np.uint64((seed + i * 0x9E3779B9) & _LOW), np.uint64(((seed >> 32) + i * 0xBB67AE85) & _LOW)]
        a, b = v[0] * np.uint64(0xD2511F53), v[2] * np.uint64(0xCD9E8D57)
        v = [(b >> half) ^ v[1] ^ key[0], b & mask, (a >> half) ^ v[3] ^ key[1], a & mask]
    w = np.stack(v, -1).reshape(rows, 4 * q)[:, :C]
    keep = (w >> np.uint64(8)) >= np.uint64(math.floor(p * (1 << 24) + 0.5))
    return torch.from_numpy(keep).to(DEV).double() / (1 - p)


def _exact_drop(c, s):
    return s["x"].double() * _mask64(c["rows"], c["C"], c["p"], s["seed"], s["offset"])


def _branch64(c, s, y, gate, post):
    b = y
    if post is not None:
        b = post * y / (y.square().mean(-1, keepdim=True) + EPS).sqrt()
    if gate is not None:
        b = b * {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[c["act"]](gate)
    if c["p"]:
        b = b * _mask64(c["N"] * c["S"], c["C"], c["p"], s["seed"], s["offset"]).view(y.shape)
    return b * c["sigma"]


def _dbl(t):
    return None if t is None else t.double()


def _exact_res(c, s):
    y = s["y"].double()
    r = s["x"].double() * c["alpha"] + _branch64(c, s, y, _dbl(s["gate"]), _dbl(s["post"]))
    norm = lambda t: 1 / (t.square().mean(-1) + EPS).sqrt()  # noqa: E731
    return {"out": r, "normed": r * norm(r)[..., None] * s["pre"].double() if s["pre"] is not None else None,
            "stats": torch.stack([norm(y) * (s["post"] is not None), norm(r) * (s["pre"] is not None)], -1)}


def _exact_res_bwd(c, s):
    leaf = lambda t: None if t is None else t.double().requires_grad_()  # noqa: E731
    r, y, gate, post, pre = leaf(s["out"]), leaf(s["y"]), leaf(s["gate"]), leaf(s["post"]), leaf(s["pre"])
    d = s["d_out"].double()
    if pre is not None:
        (r * pre / (r.square().mean(-1, keepdim=True) + EPS).sqrt() * s["d_normed"].double()).sum().backward()
        d = d + r.grad
    (_branch64(c, s, y, gate, post) * d).sum().backward()
    grad = lambda t: None if t is None else t.grad  # noqa: E731
    return {"dx": c["alpha"] * d, "dy": y.grad, "dgate": grad(gate), "dpost": grad(post), "dpre": grad(pre)}


def _requests(c, s):
    """(batch row, first token, behind the last, adapter) of each request."""
    ids = s["ids"].tolist()
    if s["cu"] is None:
        return [(i, 0, c["T"], ids[i]) for i in range(c["B"])]
    cu = s["cu"].tolist()
    return [(0, cu[i], cu[i + 1], ids[i]) for i in range(len(ids))]


def _exact_lora(c, s):
    out = s["y"].double()
    for i, t0, t1, n in _requests(c, s):
        h = s["x"][i, t0:t1].double() @ s["a"][n].double().t()
        out[i, t0:t1] += s["scale"][n].double() * (h @ s["b"][n].double())
    return out


def _exact_lora_bwd(c, s):
    dx = torch.zeros(s["x"].shape, dtype=torch.float64, device=DEV)
    da, db = (torch.zeros(s[k].shape, dtype=torch.float64, device=DEV) for k in ("a", "b"))
    for i, t0, t1, n in _requests(c, s):
        dy = s["d_out"][i, t0:t1].double() * s["scale"][n].double()
        dh = dy @ s["b"][n].double().t()
        dx[i, t0:t1] = dh @ s["a"][n].double()
        da[n] += dh.t() @ s["x"][i, t0:t1].double()
        db[n] += s["hidden"][i, t0:t1].double().t() @ dy
    return {"dx": dx, "da": da, "db": db}


_EXACT = {"drop": _exact_drop, "res": _exact_res, "res_bwd": _exact_res_bwd, "lora": _exact_lora,
          "lora_bwd": _exact_lora_bwd}


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))
