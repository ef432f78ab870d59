"""The mixer operators together, as a block of them is used: short conv -> gated
scan -> group norm with an activated gate, trained (forward, then backward through
all three) and served (a prompt, then token by token with the states handed on)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _block64(p, x, f, gate, state, H, heads_decay):
    """The block in float64 with torch's autograd, token by token."""
    import torch
    import torch.nn.functional as F

    B, T, C = x.shape
    V = C // H
    xp = torch.cat([x[:, :1].expand(B, 3, C), x], 1)
    v = F.silu(sum(xp[:, i:i + T] * p["conv"][:, i] for i in range(4))).view(B, T, H, V)
    g = -F.softplus(f).view(B, T, H, 1 if heads_decay else V)
    h, out = state, []
    for t in range(T):
        h = torch.exp(g[:, t]) * h + v[:, t]
        out.append(h)
    o = torch.stack(out, 1)
    n = (o - o.mean(3, keepdim=True)) / torch.sqrt(o.var(3, unbiased=False, keepdim=True) + EPS)
    z = n.reshape(B, T, C) * p["weight"] + p["bias"]
    return z * F.silu(gate), h


def _block(G, p, x, f, gate, state, H, heads_decay, cache=None):
    import torch.nn.functional as F

    B, T, C = x.shape
    v, new_cache = G.short_conv_1d(x, p["conv"], cache)
    g = -F.softplus(f).view(B, T, H, -1).transpose(1, 2)
    o, new_state = G.gated_scan(g, v.view(B, T, H, C // H).transpose(1, 2), None, state)
    rows = o.transpose(1, 2).reshape(B * T, C)
    y, stats = G.group_norm_act(rows, H, p["weight"], p["bias"], EPS, "silu", gate=gate.reshape(B * T, C), return_stats=True)
    return y.view(B, T, C), new_state, new_cache, (g, v, o, rows, stats)


@pytest.mark.parametrize("heads_decay", [False, True])
@pytest.mark.parametrize("B,T,H,V", [(2, 300, 2, 32), (1, 45, 3, 20)])
def test_training_through_the_block(gpu, B, T, H, V, heads_decay):
    """Gradients of every input and weight against float64 autograd.  Tolerance: the
    block is a few hundred f32 roundings of sums whose terms are not far larger than
    the result; 2^-24 x 512 of the largest gradient of the tensor."""
    import torch
    import torch.nn.functional as F

    import gdn2_amd as G

    r = torch.Generator().manual_seed(T)
    C = H * V
    rand = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    cpu = {"x": rand(B, T, C), "f": rand(B, T, H if heads_decay else C) - 2, "gate": rand(B, T, C), "state": rand(B, H, V),
           "conv": torch.rand(C, 4, generator=r) - 0.5, "weight": torch.rand(C, generator=r) + 0.5, "bias": rand(C) * 0.2}
    dy, ds = rand(B, T, C), rand(B, H, V)
    leaf = {n: t.double().requires_grad_() for n, t in cpu.items()}
    y64, s64 = _block64(leaf, leaf["x"], leaf["f"], leaf["gate"], leaf["state"], H, heads_decay)
    ((y64 * dy.double()).sum() + (s64 * ds.double()).sum()).backward()

    d = {n: t.to(gpu) for n, t in cpu.items()}
    y, s, _, (g, v, o, rows, stats) = _block(G, d, d["x"], d["f"], d["gate"], d["state"], H, heads_decay)
    n = G.group_norm_act_backward(rows, H, stats, dy.to(gpu).view(B * T, C), d["weight"], d["bias"], "silu",
                                  gate=d["gate"].view(B * T, C))
    c = G.gated_scan_backward(g, v.view(B, T, H, V).transpose(1, 2), None, o,
                              n["dx"].view(B, T, H, V).transpose(1, 2), d["state"], d_state=ds.to(gpu))
    k = G.short_conv_1d_backward(d["x"], d["conv"], c["dv"].transpose(1, 2).reshape(B, T, C))
    df = (-c["dg"].transpose(1, 2).reshape(d["f"].shape)) * torch.sigmoid(d["f"])
    got = {"x": k["dx"], "conv": k["dweight"], "f": df, "gate": n["dgate"].view(B, T, C), "weight": n["dweight"],
           "bias": n["dbias"], "state": c["dS0"]}
    torch.cuda.synchronize()
    tol = 512 * 2.0 ** -24
    for name, a, b in [("y", y, y64), ("new state", s, s64)] + [(m, got[m], leaf[m].grad) for m in got]:
        b = b.detach()
        e = float((a.double().cpu() - b).abs().max() / b.abs().max())
        assert e <= tol, (name, e)


@pytest.mark.parametrize("heads_decay", [False, True])
def test_prompt_then_tokens(gpu, heads_decay):
    """A prompt of 70 tokens in one call, then 6 tokens one by one, equals 76 tokens
    at once (same arithmetic but for the joins of tiles: 2^-24 x 256)."""
    import torch

    import gdn2_amd as G

    B, T, H, V = 3, 76, 2, 64
    C = H * V
    p = {"conv": torch.rand(C, 4, device=gpu) - 0.5, "weight": torch.rand(C, device=gpu), "bias": torch.randn(C, device=gpu)}
    x, gate = torch.randn(B, T, C, device=gpu), torch.randn(B, T, C, device=gpu)
    f = torch.randn(B, T, H if heads_decay else C, device=gpu)
    whole, s_end, c_end, _ = _block(G, p, x, f, gate, None, H, heads_decay)
    parts, state, cache = [], None, None
    for a, b in [(0, 70)] + [(t, t + 1) for t in range(70, 76)]:
        y, state, cache, _ = _block(G, p, x[:, a:b], f[:, a:b], gate[:, a:b], state, H, heads_decay, cache)
        parts.append(y)
    got = torch.cat(parts, 1)
    assert torch.equal(cache, c_end)
    for a, b in ((got, whole), (state, s_end)):
        assert float((a - b).abs().max()) <= 256 * 2.0 ** -24 * float(b.abs().max())


def test_captured_training_step(gpu):
    """Forward and backward of the block in one graph, replayed on other inputs
    between eager steps."""
    import torch

    import gdn2_amd as G

    B, T, H, V = 2, 400, 2, 32
    C = H * V
    p = {"conv": torch.rand(C, 4, device=gpu) - 0.5, "weight": torch.rand(C, device=gpu), "bias": torch.randn(C, device=gpu)}
    ins = [{"x": torch.randn(B, T, C, device=gpu), "f": torch.randn(B, T, H, device=gpu),
            "gate": torch.randn(B, T, C, device=gpu), "dy": torch.randn(B * T, C, device=gpu)} for _ in range(2)]

    def step(i):
        y, s, _, (g, v, o, rows, stats) = _block(G, p, i["x"], i["f"], i["gate"], None, H, True)
        n = G.group_norm_act_backward(rows, H, stats, i["dy"], p["weight"], p["bias"], "silu", gate=i["gate"].view(B * T, C))
        c = G.gated_scan_backward(g, v.view(B, T, H, V).transpose(1, 2), None, o, n["dx"].view(B, T, H, V).transpose(1, 2))
        k = G.short_conv_1d_backward(i["x"], p["conv"], c["dv"].transpose(1, 2).reshape(B, T, C))
        return [y, s, n["dgate"], n["dweight"], n["dbias"], c["dg"], c["dS0"], k["dx"], k["dweight"]]

    cur = {n: t.clone() for n, t in ins[0].items()}
    want = [step(i) for i in ins]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cur)
    for k in range(4):
        for n in cur:
            cur[n].copy_(ins[k % 2][n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 2]))
        step(ins[1 - k % 2])


def test_captured_decoding(gpu):
    """One token through scan and norm in a graph that hands the state on in place,
    replayed token after token, equals the eager steps."""
    import torch

    import gdn2_amd as G

    B, H, V, steps = 5, 2, 64, 6
    C = H * V
    g, v = -torch.rand(steps, B, H, 1, 1, device=gpu), torch.randn(steps, B, H, 1, V, device=gpu)
    z, weight = torch.randn(steps, B, C, device=gpu), torch.rand(C, device=gpu)
    start = torch.randn(B, H, V, device=gpu)
    cur = {"g": g[0].clone(), "v": v[0].clone(), "z": z[0].clone(), "state": start.clone()}

    def step(i):
        o, _ = G.gated_scan(i["g"], i["v"], None, i["state"], new_state=i["state"])
        return G.group_norm_act(o.view(B, C), H, weight, None, EPS, "silu", gate=i["z"])

    step(cur)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(cur)
    cur["state"].copy_(start)
    eager = {"state": start.clone()}
    for t in range(steps):
        for n, x in (("g", g), ("v", v), ("z", z)):
            cur[n].copy_(x[t])
            eager[n] = x[t].clone()
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(cur["state"], eager["state"]), t


def test_graphs_that_share_a_workspace(gpu):
    """Two graphs captured with one workspace, replayed in turn, and an eager call
    with it between them."""
    import torch

    import gdn2_amd as G

    ws = torch.empty(1 << 24, dtype=torch.uint8, device=gpu)
    ins = [{"g": -torch.rand(1, 2, T, 64, device=gpu), "v": torch.randn(1, 2, T, 64, device=gpu),
            "x": torch.randn(1, T, 128, device=gpu), "w": torch.randn(128, 4, device=gpu)} for T in (3000, 1700)]

    def all_of(i, ws):
        o, s = G.gated_scan(i["g"], i["v"], workspace=ws)
        r = G.gated_scan_backward(i["g"], i["v"], None, o, o, workspace=ws)
        y, stats = G.group_norm_act(i["x"], 4, return_stats=True, workspace=ws)
        n = G.group_norm_act_backward(i["x"], 4, stats, y, workspace=ws)
        c = G.short_conv_1d_backward(i["x"], i["w"], y, workspace=ws)
        return [o, s, r["dg"], r["dv"], r["dS0"], y, n["dx"], n["dweight"], n["dbias"], c["dx"], c["dweight"]]

    want = [all_of(i, None) for i in ins]
    graphs, got = [], []
    for i in ins:
        all_of(i, ws)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(all_of(i, ws))
    for k in (0, 1, 1, 0, 1, 0):
        for t in got[k]:
            t.zero_()
        graphs[k].replay()
        eager = all_of(ins[1 - k], ws)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k])), k
        assert all(torch.equal(a, b) for a, b in zip(eager, want[1 - k])), k
