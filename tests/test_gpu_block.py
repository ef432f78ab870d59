"""The block operators together, as a training step and a serving loop use them."""
import pytest
import torch

import block_testutil as K

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
B, T, D, O, R, L = 3, 40, 96, 96, 8, 2
ALPHA, SIGMA, P, SEED = 0.9, 0.5, 0.2, 77


def inputs(ty):
    g = torch.Generator().manual_seed(21)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": rnd(B, T, D), "w": rnd(D, O) * D ** -0.5, "a": rnd(L, R, D) * D ** -0.5, "b": rnd(L, R, O) * R ** -0.5,
         "gate": rnd(B, 1, O), "pre0": 0.5 + torch.rand(D, generator=g), "post": 0.5 + torch.rand(O, generator=g),
         "pre": 0.5 + torch.rand(O, generator=g), "d_out": rnd(B, T, D), "d_normed": rnd(B, T, O)}
    for k in ("a", "b", "gate", "d_normed", "w"):
        t[k] = t[k].to(ty)
    return t, torch.tensor([1, 0, 1], dtype=torch.int32), torch.tensor([0.7, 1.6])


def step(t, ids, scale, ty, rng=None, seed=SEED):
    """Norm, a shared projection with adapters whose input is dropped out, the residual
    path; then everything's gradient."""
    import gdn2_amd as G

    q = 0 if rng is not None else seed
    normed_in = torch.empty_like(t["x"], dtype=ty)
    _, n0, st0 = G.residual_norm(t["x"], pre_weight=t["pre0"], normed=normed_in, return_stats=True)
    xd = G.dropout(n0, P, q, 0, rng=rng)
    y0 = (n0.float().view(-1, D) @ t["w"].float()).view(B, T, O).to(ty)  # the shared projection
    y, h = G.low_rank_add(y0, xd, t["a"], t["b"], ids, scale, return_hidden=True)
    first = B * T * (D // 4)  # counters behind the first mask's
    a = ("silu", ALPHA, SIGMA, P, q, first)
    out, n, st = G.residual_norm(t["x"], y, t["gate"], t["post"], t["pre"], 1e-5, *a, rng=rng, return_stats=True)
    r = G.residual_norm_backward(out, y, st, t["d_out"], t["d_normed"], t["gate"], t["post"], t["pre"], *a, rng=rng)
    dl = G.low_rank_add_backward(xd, t["a"], t["b"], ids, h, r["dy"], scale)
    dn0 = G.dropout_backward(dl["dx"], P, q, 0, rng=rng).float()
    dn0 = (dn0 + (r["dy"].float().view(-1, O) @ t["w"].float().t()).view(B, T, D)).to(ty)
    dw = n0.float().view(-1, D).t() @ r["dy"].float().view(-1, O)
    last = G.residual_norm_backward(t["x"], None, st0, r["dx"], dn0, pre_weight=t["pre0"])
    return {"out": out, "normed": n, "x": last["dx"], "pre0": last["dpre"], "w": dw, "a": dl["da"], "b": dl["db"],
            "gate": r["dgate"], "post": r["dpost"], "pre": r["dpre"]}


def step64(t, ids, scale, seed):
    """The same from the formulas, in 64 bits, the gradients by autograd."""
    leaf = {k: t[k].double().requires_grad_() for k in ("x", "w", "a", "b", "gate", "pre0", "post", "pre")}
    norm = lambda v, w: v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w  # noqa: E731
    n0 = norm(leaf["x"], leaf["pre0"])
    xd = n0 * K.drop_factor(B * T, D, P, seed).view(B, T, D)
    y = n0 @ leaf["w"] + torch.stack([float(scale[l]) * (xd[i] @ leaf["a"][l].t()) @ leaf["b"][l] for i, l in enumerate(ids.tolist())])
    gate = torch.nn.functional.silu(leaf["gate"])
    out = ALPHA * leaf["x"] + SIGMA * gate * norm(y, leaf["post"]) * K.drop_factor(B * T, O, P, seed, B * T * (D // 4)).view(B, T, O)
    n = norm(out, leaf["pre"])
    ((out * t["d_out"].double()).sum() + (n * t["d_normed"].double()).sum()).backward()
    return {"out": out.detach(), "normed": n.detach(), **{k: v.grad for k, v in leaf.items()}}


@pytest.mark.parametrize("ty", [torch.float32, BF])
def test_training_step(gpu, ty):
    """Each result as one vector.  f32: a chain of at most eight operators, each within
    2^-20 of its result's length (32 half steps twice, as in block_testutil.alike; sums of
    these sizes are far from cancelling).  bf16: twelve roundings of a half step, 2^-8/sqrt(3),
    on the way (six tensors are rounded, forward and backward)."""
    t, ids, scale = inputs(ty)
    got = step({k: v.to(gpu) for k, v in t.items()}, ids.to(gpu), scale.to(gpu), ty)
    want = step64(t, ids, scale, SEED)
    bound = 8 * 2.0 ** -20 if ty is torch.float32 else 12 * 2.0 ** -8 / 3 ** 0.5
    for k, w in want.items():
        g = got[k].cpu().double()
        assert g.shape == w.shape and float((g - w).norm()) <= bound * float(w.norm()), (k, float((g - w).norm() / w.norm()))


@pytest.mark.parametrize("ty", [torch.float32, BF])
def test_captured_training_step(gpu, ty):
    """Replayed with other inputs, adapters and masks beside the eager step."""
    t, ids, scale = inputs(ty)
    t, ids, scale = {k: v.to(gpu) for k, v in t.items()}, ids.to(gpu), scale.to(gpu)
    rng = torch.tensor([SEED, 0], dtype=torch.int64, device=gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(t, ids, scale, ty, rng)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(t, ids, scale, ty, rng)
    for i in range(4):
        t["x"].copy_(torch.randn(B, T, D, generator=torch.Generator().manual_seed(i)))
        ids.copy_(torch.tensor([i % 2, 1, -1 if i == 3 else 0]))
        rng.copy_(torch.tensor([SEED + i, 0]))
        graph.replay()
        torch.cuda.synchronize()
        want = step(t, ids, scale, ty, None, SEED + i)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), k


def test_serving_loop(gpu):
    """Two layers with adapters and the residual path between them: a prompt and single
    tokens give what one pass over all of them does."""
    import gdn2_amd as G

    layers = [G.GatedDeltaNet2(G.Gdn2Config(hidden_size=128, num_heads=2, head_dim=64, mode="chunk"), seed=s) for s in (1, 2)]
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g).to(gpu)  # noqa: E731
    ads = [G.Gdn2Adapters(m, {n: (rnd(3, 4, 128) * 0.05, rnd(3, 4, 128) * 0.05) for n in ("q_proj", "o_proj")}) for m in layers]
    ids = torch.tensor([0, 2, -1], dtype=torch.int32, device=gpu)
    w = [[rnd(128).abs() + 0.5 for _ in range(2)] for _ in range(2)]
    x = rnd(3, 80, 128)

    def run(x, states):
        r, n = G.residual_norm(x, pre_weight=w[0][0])
        for i, (m, ad) in enumerate(zip(layers, ads)):
            y, states[i] = m.forward(n, states[i], ad, ids)
            r, n = G.residual_norm(r, y, None, w[i][1], w[1][0])
        return torch.cat([r, n], -1)

    whole = run(x, [None, None])
    states, parts = [None, None], []
    for t0, t1 in ((0, 70), *((i, i + 1) for i in range(70, 80))):
        parts.append(run(x[:, t0:t1].contiguous(), states))
    got = torch.cat(parts, 1)
    # the layer's own bound between its forms, 1e-4 of the largest output, through two of them
    assert float((got - whole).abs().max()) <= 2e-4 * float(whole.abs().max())
