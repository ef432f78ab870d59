"""residual_norm and its backward against their 64-bit forms, within what f32
arithmetic may be off by (block_testutil)."""
import pytest
import torch

import block_testutil as K

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
TYPES = {"f32": (F32, F32), "bf16": (BF, BF), "mixed": (F32, BF)}


def make(M, C, ty, gate=True, post=True, pre=True, seed=0, N=None, gate_shape=None):
    g = torch.Generator().manual_seed(seed * 1000 + M + C)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    stream, branch = TYPES[ty]
    shape = (M, C) if N is None else (N, M // N, C)
    t = {"x": rnd(*shape).to(stream) * 1.5, "y": rnd(*shape).to(branch) * 0.5,
         "gate": (rnd(*(gate_shape or shape)) * 2).to(branch) if gate else None, "post": 0.5 + torch.rand(C, generator=g) if post else None,
         "pre": 0.5 + torch.rand(C, generator=g) if pre else None, "d_out": rnd(*shape).to(stream),
         "d_normed": rnd(*shape).to(branch) if pre else None}
    return t


def dbl(t, M, C, shape=None):
    return None if t is None else t.double().expand(shape or t.shape).reshape(M, C)


def check(gpu, t, M, C, act="silu", alpha=0.8, sigma=0.5, p=0.0, seed=3, offset=7):
    """Both directions."""
    import gdn2_amd as G

    shape = t["x"].shape
    d = {k: None if v is None else v.to(gpu) for k, v in t.items()}
    factor = K.drop_factor(M, C, p, seed, offset)
    gate64 = dbl(t["gate"], M, C, shape)
    w = [None if t[k] is None else t[k].double() for k in ("post", "pre")]
    want, err = K.residual64(dbl(t["x"], M, C), dbl(t["y"], M, C), gate64, *w, 1e-5, act, alpha, sigma, factor)
    out, normed, stats = G.residual_norm(d["x"], d["y"], d["gate"], d["post"], d["pre"], 1e-5, act, alpha, sigma, p, seed, offset,
                                         return_stats=True)
    assert out.shape == shape and out.dtype == t["x"].dtype and stats.shape == (*shape[:-1], 2)
    K.near(out, want[0], err[0], "out")
    K.near(stats, want[2], err[2], "stats")
    if t["pre"] is not None:
        assert normed.dtype == t["y"].dtype
        K.near(normed, want[1], err[1], "normed")
    else:
        assert normed is None
    # the backward, of the out and stats that were written
    st = stats.cpu().double().reshape(M, 2)
    g, e = K.residual_bwd64(dbl(out.cpu(), M, C), dbl(t["y"], M, C), gate64, *w, st, dbl(t["d_out"], M, C),
                            dbl(t["d_normed"], M, C), act, alpha, sigma, factor)
    got = G.residual_norm_backward(out, d["y"], stats, d["d_out"], d["d_normed"], d["gate"], d["post"], d["pre"], act, alpha, sigma,
                                   p, seed, offset)
    if t["gate"] is not None and t["gate"].shape != shape:
        for r in (g, e):  # the sums over the rows that share a gate
            v = r["dgate"].view(shape)
            r["dgate"] = v.sum(1, keepdim=True) if t["gate"].dim() > 1 else v.sum((0, 1))
        share = K.residual_bwd64(dbl(out.cpu(), M, C), dbl(t["y"], M, C), gate64, *w, st, dbl(t["d_out"], M, C),
                                 dbl(t["d_normed"], M, C), act, alpha, sigma, factor)[0]["dgate"].abs().view(shape)
        e["dgate"] = e["dgate"] + (128 + 256 + 3) * K.U * (share.sum(1, keepdim=True) if t["gate"].dim() > 1 else share.sum((0, 1)))
    for name in ("dx", "dy", "dgate", "dpost", "dpre"):
        if name in g:
            assert got[name].shape == {"dx": shape, "dy": shape, "dgate": t["gate"].shape if t["gate"] is not None else None,
                                       "dpost": (C,), "dpre": (C,)}[name]
            K.near(got[name], g[name], e[name], name)
        else:
            assert got[name] is None
    return d, out, normed, stats, got


@pytest.mark.parametrize("ty", list(TYPES))
@pytest.mark.parametrize("M,C", [(1, 1), (3, 2), (70, 5), (1, 8), (130, 8), (33, 64), (5, 96), (129, 250), (300, 320), (9, 512),
                                 (2, 513), (7, 1537), (64, 2048), (2, 2049), (3, 4096), (2, 8191), (1, 8192)])
def test_sizes(gpu, ty, M, C):
    check(gpu, make(M, C, ty), M, C, p=0.1)


@pytest.mark.parametrize("ty", list(TYPES))
@pytest.mark.parametrize("C", [2100, 2051, 4096, 4104])
@pytest.mark.parametrize("shared", [False, True])
def test_wide_rows(gpu, ty, C, shared):
    """More rows than workgroups, of channels that eight waves hold."""
    check(gpu, make(1602, C, ty, N=2, gate_shape=(2, 1, C) if shared else None), 1602, C, p=0.1)


@pytest.mark.parametrize("ty", list(TYPES))
@pytest.mark.parametrize("post,pre,gate", [(a, b, c) for a in (False, True) for b in (False, True) for c in (False, True)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_forms(gpu, ty, post, pre, gate, p):
    for C in (40, 700):
        check(gpu, make(19, C, ty, gate, post, pre), 19, C, p=p)


@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("ty", list(TYPES))
def test_activations(gpu, act, ty):
    t = make(17, 96, ty)
    t["gate"] *= 8  # into their flat parts
    check(gpu, t, 17, 96, act=act)


@pytest.mark.parametrize("ty", list(TYPES))
@pytest.mark.parametrize("N,S,C", [(1, 1, 8), (3, 1, 40), (5, 37, 40), (2, 300, 96), (40, 3, 320), (3, 50, 700), (2, 9, 3000), (700, 2, 16)])
def test_shared_gates(gpu, ty, N, S, C):
    for shape in ((N, 1, C), (C,)):
        check(gpu, make(N * S, C, ty, N=N, gate_shape=shape), N * S, C, act="sigmoid", p=0.1)


@pytest.mark.parametrize("C", [24, 600])
def test_sums_over_many_rows(gpu, C):
    """More rows than the f32 sums take; the column sums keep their digits where every
    term has the same sign."""
    M = 150000 if C == 24 else 140000
    t = make(M, C, "f32", N=4, gate_shape=(C,))
    for k in ("d_out", "d_normed"):
        t[k] = t[k].abs()
    check(gpu, t, M, C, act="none")


@pytest.mark.parametrize("ty", list(TYPES))
def test_no_branch(gpu, ty):
    """y None: the norm before the first block."""
    import gdn2_amd as G

    M, C = 21, 250
    t = make(M, C, ty, gate=False, post=False)
    x, w = t["x"].to(gpu), t["pre"].to(gpu)
    normed = torch.empty_like(x, dtype=TYPES[ty][1])
    out, n, stats = G.residual_norm(x, pre_weight=w, residual_scale=0.5, normed=normed, return_stats=True)
    assert n is normed
    want, err = K.residual64(dbl(t["x"], M, C), None, None, None, t["pre"].double(), 1e-5, "none", 0.5, 1.0, 1.0)
    for got, a, b in zip((out, n, stats), want, err):
        K.near(got, a, b)
    g, e = K.residual_bwd64(dbl(out.cpu(), M, C), None, None, None, t["pre"].double(), stats.cpu().double(), dbl(t["d_out"], M, C),
                            dbl(t["d_normed"], M, C), "none", 0.5, 1.0, 1.0)
    got = G.residual_norm_backward(out, None, stats, t["d_out"].to(gpu), t["d_normed"].to(gpu), pre_weight=w, residual_scale=0.5)
    assert got["dy"] is None
    for name in ("dx", "dpre"):
        K.near(got[name], g[name], e[name], name)


def test_no_d_out(gpu):
    import gdn2_amd as G

    t = make(9, 96, "bf16")
    d = {k: v.to(gpu) for k, v in t.items()}
    out, _, st = G.residual_norm(d["x"], d["y"], d["gate"], d["post"], d["pre"], return_stats=True)
    a = G.residual_norm_backward(out, d["y"], st, None, d["d_normed"], d["gate"], d["post"], d["pre"])
    b = G.residual_norm_backward(out, d["y"], st, torch.zeros_like(out), d["d_normed"], d["gate"], d["post"], d["pre"])
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("ty", list(TYPES))
def test_layouts(gpu, ty):
    """Operands of any strides give the bits of contiguous ones."""
    import gdn2_amd as G

    N, S, C = 3, 5, 40
    t = {k: None if v is None else v.to(gpu) for k, v in make(N * S, C, ty, N=N).items()}

    def call(f=lambda v: v):
        a = {k: f(v) if v.dim() == 3 else v for k, v in t.items()}
        o, n, st = G.residual_norm(a["x"], a["y"], a["gate"], a["post"], a["pre"], 1e-5, "silu", 0.8, 0.5, 0.2, 4, return_stats=True)
        r = G.residual_norm_backward(f(o), a["y"], st, a["d_out"], a["d_normed"], a["gate"], a["post"], a["pre"], "silu", 0.8, 0.5,
                                     0.2, 4)
        return [o, n, st, *r.values()]

    ref = call()
    for f in (lambda v: v.transpose(0, 1).contiguous().transpose(0, 1), lambda v: torch.cat([v, v], 2)[..., 40:],
              lambda v: torch.cat([v, v, v], 2)[..., 40:80], lambda v: v.transpose(1, 2).contiguous().transpose(1, 2),
              lambda v: torch.cat([v, v[..., :3]], 2)[..., :40], lambda v: torch.cat([v, v], 1)[:, :5]):
        for a, b in zip(call(f), ref):
            assert a.shape == b.shape and torch.equal(a, b)
    four = [v.view(N, S, 1, C) if v is not None and v.dim() == 3 else v for v in (t["x"], t["y"], t["gate"])]
    o, n = G.residual_norm(*four, t["post"], t["pre"], 1e-5, "silu", 0.8, 0.5, 0.2, 4)
    assert o.shape == (N, S, 1, C) and torch.equal(o.view(N, S, C), ref[0]) and torch.equal(n.view(N, S, C), ref[1])


@pytest.mark.parametrize("ty", list(TYPES))
@pytest.mark.parametrize("M,C", [(130, 24), (7, 1000), (2, 5000)])
def test_in_place(gpu, ty, M, C):
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(M, C, ty).items()}
    a = (t["gate"], t["post"], t["pre"])
    o, n = G.residual_norm(t["x"], t["y"], *a)
    x, y = t["x"].clone(), t["y"].clone()
    o2, n2 = G.residual_norm(x, y, *a, out=x, normed=y)
    assert o2 is x and n2 is y and torch.equal(x, o) and torch.equal(y, n)
    buf = torch.full((M, C + 5), 9.0, dtype=o.dtype, device=gpu)
    o3, _ = G.residual_norm(t["x"], t["y"], *a, out=buf[:, 2:2 + C])
    assert torch.equal(o3, o) and (buf[:, :2] == 9).all() and (buf[:, 2 + C:] == 9).all()


def test_dropout_is_that_of_dropout(gpu):
    """The mask of the fused pass is dropout's at the same counters."""
    import gdn2_amd as G

    for C in (250, 2048):
        x, y = torch.randn(11, C, device=gpu), torch.randn(11, C, device=gpu)
        out, _ = G.residual_norm(x, y, dropout_p=0.3, seed=8, offset=2 ** 34)
        assert torch.equal(out, x + G.dropout(y, 0.3, 8, 2 ** 34))


def test_values_that_are_not_finite(gpu):
    """A row with them does not reach its neighbours; dropped ones do not reach the row."""
    import gdn2_amd as G

    for C in (40, 700, 3000):
        t = {k: v.to(gpu) for k, v in make(9, C, "f32").items()}
        f = lambda: G.residual_norm(t["x"], t["y"], t["gate"], None, t["pre"], 1e-5, "sigmoid", 1.0, 1.0, 0.5, 6)  # noqa: E731
        o, n = f()
        k = K.kept(9, C, 0.5, 6)
        gone = int((~k[4]).nonzero()[0])
        t["y"][4, gone] = float("nan")
        assert all(torch.equal(a, b) for a, b in zip(f(), (o, n)))
        t["y"][4, int(k[4].nonzero()[0])] = float("inf")
        o2, n2 = f()
        rest = [i for i in range(9) if i != 4]
        assert torch.equal(o2[rest], o[rest]) and torch.equal(n2[rest], n[rest]) and o2[4].isinf().any() and n2[4].isnan().any()
    x = torch.zeros(4, 96, device=gpu)  # rows of zeros: eps alone
    o, n, st = G.residual_norm(x, x, post_weight=torch.ones(96, device=gpu), pre_weight=torch.ones(96, device=gpu), return_stats=True)
    assert (n == 0).all() and torch.allclose(st, torch.full_like(st, 1e5 ** 0.5), rtol=1e-6)


def test_nothing(gpu):
    import gdn2_amd as G

    w = torch.ones(8, device=gpu)
    for s in ((0, 8), (2, 0, 8), (0, 3, 8)):
        x = torch.empty(s, device=gpu)
        gate = torch.empty((s[0], 1, 8), device=gpu) if len(s) == 3 else torch.ones(8, device=gpu)
        o, n, st = G.residual_norm(x, x, gate, w, w, return_stats=True)
        assert o.shape == n.shape == s and st.shape == (*s[:-1], 2)
        r = G.residual_norm_backward(o, x, st, o, n, gate, w, w)
        assert (r["dpre"] == 0).all() and (r["dpost"] == 0).all() and (r["dgate"] == 0).all() and r["dgate"].shape == gate.shape
        assert r["dx"].shape == s


def test_workspace_of_the_caller(gpu):
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(50, 96, "f32").items()}
    o, n, st = G.residual_norm(t["x"], t["y"], t["gate"], t["post"], t["pre"], return_stats=True)
    a = (o, t["y"], st, t["d_out"], t["d_normed"], t["gate"], t["post"], t["pre"])
    ref = G.residual_norm_backward(*a)
    ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device=gpu)
    for w in (ws, ws[:256]):
        got = G.residual_norm_backward(*a, workspace=w)
        assert all(torch.equal(got[k], ref[k]) for k in ref)
    with pytest.raises(ValueError):
        G.residual_norm_backward(*a, workspace=torch.empty(1 << 20, dtype=torch.uint8))
    with pytest.raises(TypeError):
        G.residual_norm_backward(*a[:1], a[1].cpu(), *a[2:])


def test_captured(gpu):
    """A training step's two calls, replayed with new inputs and another mask."""
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(60, 2048, "mixed", N=4, gate_shape=(4, 1, 2048)).items()}
    rng = torch.tensor([5, 0], dtype=torch.int64, device=gpu)

    def step(rng=rng, seed=0, offset=0):
        o, n, st = G.residual_norm(t["x"], t["y"], t["gate"], t["post"], t["pre"], 1e-5, "silu", 1.0, 1.0, 0.1, seed, offset, rng,
                                   return_stats=True)
        r = G.residual_norm_backward(o, t["y"], st, t["d_out"], t["d_normed"], t["gate"], t["post"], t["pre"], "silu", 1.0, 1.0, 0.1,
                                     seed, offset, rng)
        return [o, n, st, *r.values()]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for k in ("x", "y", "gate"):
            t[k].copy_(torch.randn(t[k].shape, generator=torch.Generator().manual_seed(i)))
        rng.copy_(torch.tensor([5 + i, i << 33]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(None, 5 + i, i << 33)):
            assert torch.equal(a, b)


def test_on_another_stream(gpu):
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(64, 2048, "bf16").items()}
    ref = G.residual_norm(t["x"], t["y"], t["gate"], t["post"], t["pre"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = G.residual_norm(t["x"], t["y"], t["gate"], t["post"], t["pre"])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
