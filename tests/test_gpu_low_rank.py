"""low_rank_add and its backward against their 64-bit forms."""
import pytest
import torch

import block_testutil as K

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def make(B, T, D, O, R, L, ty, seed=0, cu=None):
    g = torch.Generator().manual_seed(seed * 77 + B + T + D + O + R + L)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    n = B if cu is None else len(cu) - 1
    return {"x": rnd(B, T, D).to(ty), "y": rnd(B, T, O).to(ty), "a": (rnd(L, R, D) * D ** -0.5).to(ty),
            "b": (rnd(L, R, O) * R ** -0.5).to(ty), "ids": torch.randint(-1, L + 1, (n,), generator=g, dtype=torch.int32),
            "scale": 0.5 + torch.rand(L, generator=g), "d_out": rnd(B, T, O).to(ty), "dx": rnd(B, T, D).to(ty)}


def check(gpu, t, cu=None, scale=True, dx=True):
    """Both directions; the device's tensors and results."""
    import gdn2_amd as G

    B, T, D = t["x"].shape
    O, M = t["y"].shape[2], B * T
    d = {k: v.to(gpu) for k, v in t.items()}
    dcu = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=gpu)
    s = d["scale"] if scale else None
    flat = {k: v.double().reshape(-1, v.shape[-1]) if k in ("x", "y", "d_out", "dx") else v.double() for k, v in t.items()}
    w64 = (flat["a"], flat["b"], t["ids"], flat["scale"] if scale else None)
    (out64, h64), (err, h_err) = K.low_rank64(flat["y"], flat["x"], *w64, B, T, cu)
    out, h = G.low_rank_add(d["y"], d["x"], d["a"], d["b"], d["ids"], s, cu_seqlens=dcu, return_hidden=True)
    K.near(h, h64, h_err, "hidden")
    K.near(out, out64, err, "out")
    K.alike(out, out64, "out")
    assert torch.equal(out, G.low_rank_add(d["y"], d["x"], d["a"], d["b"], d["ids"], s, cu_seqlens=dcu))
    into = d["dx"].clone() if dx else None
    got = G.low_rank_add_backward(d["x"], d["a"], d["b"], d["ids"], h, d["d_out"], s, cu_seqlens=dcu, dx=into)
    assert into is None or got["dx"] is into
    g, e = K.low_rank_bwd64(flat["x"], *w64[:3], h.cpu().double().reshape(M, -1), flat["d_out"], w64[3], B, T, cu,
                            flat["dx"] if dx else None)
    for k in ("dx", "da", "db"):
        assert got[k].dtype == (t["x"].dtype if k == "dx" else F32)
        K.near(got[k], g[k], e[k], k)
        K.alike(got[k], g[k], k)
    return d, out, h, got


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("B,T,D,O,R,L", [
    (1, 1, 1, 1, 1, 1), (3, 1, 5, 7, 2, 2), (64, 1, 256, 192, 16, 16), (2, 17, 33, 250, 3, 2), (5, 16, 96, 64, 16, 3),
    (2, 100, 250, 333, 24, 2), (1, 129, 1537, 100, 17, 1), (3, 64, 512, 1024, 33, 2), (1, 200, 128, 129, 64, 1),
    (2, 70, 64, 96, 100, 2), (1, 40, 300, 200, 129, 1), (7, 9, 2048, 520, 8, 5), (1, 33, 640, 640, 512, 1)])
def test_sizes(gpu, ty, B, T, D, O, R, L):
    check(gpu, make(B, T, D, O, R, L, ty))


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("B,T,R", [(1100, 5, 8), (1100, 5, 24), (1100, 5, 40), (2, 16500, 24), (2, 16500, 40), (1, 33000, 65)])
def test_many_tiles(gpu, ty, B, T, R):
    """Short and long requests that fill the card, by the number of ranks."""
    check(gpu, make(B, T, 72, 70, R, 3, ty))


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [1, 16, 24, 40, 64])
def test_long_requests(gpu, ty, R):
    """The tiles of 64 rows, ragged ends, several blocks of rows for an adapter."""
    check(gpu, make(3, 3001, 160, 144, R, 2, ty, seed=R))


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("cu", [[0, 50], [0, 0, 50], [3, 3, 20, 20, 47], [0, 1, 2, 3, 50], [10, 40], [0, 16, 32, 48, 50], [50, 50], [0]])
def test_packed(gpu, ty, cu):
    """Requests of no tokens, of one, that end inside a tile; rows outside all of them."""
    d, out, h, got = check(gpu, make(1, 50, 96, 80, 8, 3, ty, cu=cu), cu)
    outside = [r for r in range(50) if not cu[0] <= r < cu[-1]]
    assert torch.equal(out[0, outside], d["y"][0, outside]) and (h[0, outside] == 0).all()
    assert torch.equal(got["dx"][0, outside], d["dx"][0, outside])


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("N", [61, 62, 63, 64, 65, 300])
def test_many_packed(gpu, ty, N):
    g = torch.Generator().manual_seed(N)
    cu = [2] + (torch.randint(2, 9000, (N - 1,), generator=g).sort().values.tolist() if N < 300 else
                torch.randint(2, 2000, (N - 1,), generator=g).sort().values.tolist()) + [9000 if N < 300 else 2001]
    check(gpu, make(1, cu[-1] + 3, 64, 72, 16, 4, ty, cu=cu), cu)


@pytest.mark.parametrize("ty", [F32, BF])
def test_many_rows(gpu, ty):
    """Enough rows for one share of the wide dimension, with and without hidden."""
    check(gpu, make(2, 16500, 200, 100, 4, 2, ty), dx=False)


@pytest.mark.parametrize("ty", [F32, BF])
def test_no_scale_and_no_dx(gpu, ty):
    check(gpu, make(3, 40, 64, 64, 4, 2, ty), scale=False, dx=False)


@pytest.mark.parametrize("ty", [F32, BF])
def test_rows_of_two_dimensions(gpu, ty):
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(70, 1, 96, 40, 8, 5, ty).items()}
    a = (t["a"], t["b"], t["ids"], t["scale"])
    ref, h = G.low_rank_add(t["y"], t["x"], *a, return_hidden=True)
    got, h2 = G.low_rank_add(t["y"][:, 0], t["x"][:, 0], *a, return_hidden=True)
    assert got.shape == (70, 40) and h2.shape == (70, 8) and torch.equal(got, ref[:, 0]) and torch.equal(h, h2[:, None])
    r = G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], h, t["d_out"], t["scale"])
    r2 = G.low_rank_add_backward(t["x"][:, 0], t["a"], t["b"], t["ids"], h2, t["d_out"][:, 0], t["scale"])
    assert torch.equal(r["dx"][:, 0], r2["dx"]) and torch.equal(r["da"], r2["da"]) and torch.equal(r["db"], r2["db"])


@pytest.mark.parametrize("ty", [F32, BF])
def test_layouts_and_places(gpu, ty):
    """Any strides, columns of wider rows at odd places, in place: the bits of contiguous
    operands, and nothing beside the results is written."""
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(3, 50, 96, 40, 8, 5, ty).items()}

    def call(f=lambda v: v, w=lambda v: v):
        a = {k: f(t[k]) for k in ("x", "y", "d_out")}
        o, h = G.low_rank_add(a["y"], a["x"], w(t["a"]), w(t["b"]), t["ids"], t["scale"], return_hidden=True)
        r = G.low_rank_add_backward(a["x"], w(t["a"]), w(t["b"]), t["ids"], h, a["d_out"], t["scale"])
        return [o, h, *r.values()]

    ref = call()
    wide = lambda v: torch.cat([v[..., :3], v, v[..., :2]], -1)[..., 3:-2]  # noqa: E731
    for f, w in ((wide, wide), (lambda v: v.transpose(0, 1).contiguous().transpose(0, 1), lambda v: v.transpose(0, 1).contiguous().transpose(0, 1)),
                 (lambda v: v.transpose(1, 2).contiguous().transpose(1, 2), lambda v: v.transpose(1, 2).contiguous().transpose(1, 2))):
        for a, b in zip(call(f, w), ref):
            assert a.shape == b.shape and torch.equal(a, b)
    y = t["y"].clone()
    assert G.low_rank_add(y, t["x"], t["a"], t["b"], t["ids"], t["scale"], out=y) is y and torch.equal(y, ref[0])
    buf = torch.full((3, 50, 47), 9.0, dtype=ty, device=gpu)
    out = buf[..., 5:45]
    G.low_rank_add(t["y"], t["x"], t["a"], t["b"], t["ids"], t["scale"], out=out)
    assert torch.equal(out, ref[0]) and (buf[..., :5] == 9).all() and (buf[..., 45:] == 9).all()


@pytest.mark.parametrize("ty", [F32, BF])
def test_values_that_are_not_finite(gpu, ty):
    """A request's infinities and NaN stay in its rows (and its adapter's gradients), an
    adapter's in its requests; rows without an adapter are copied."""
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(4, 20, 96, 40, 8, 3, ty).items()}
    t["ids"].copy_(torch.tensor([0, 1, -1, 1]))
    a = lambda: G.low_rank_add(t["y"], t["x"], t["a"], t["b"], t["ids"], t["scale"], return_hidden=True)  # noqa: E731
    ref, h = a()
    ref_g = G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], h, t["d_out"], t["scale"])
    for bad in (float("nan"), float("inf")):
        x = t["x"].clone()
        t["x"][0, 7, 11] = bad
        t["x"][2, 3] = bad
        t["y"][2, 4, 5] = bad
        t["a"][2] = bad  # nobody's
        got, h2 = a()
        g = G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], h, t["d_out"], t["scale"])
        rest = [i for i in range(20) if i != 7]
        assert torch.equal(got[0, rest], ref[0, rest]) and torch.equal(got[1], ref[1]) and torch.equal(got[3], ref[3])
        assert not got[0, 7].isfinite().any() and torch.equal(torch.nan_to_num(got[2]), torch.nan_to_num(t["y"][2]))
        assert torch.equal(g["da"][1], ref_g["da"][1]) and torch.equal(g["db"], ref_g["db"]) and torch.equal(g["dx"][1], ref_g["dx"][1])
        assert (g["dx"][2] == 0).all() and (g["da"][2] == 0).all()
        t["x"].copy_(x)
    # an infinite h: infinite where b is not zero, of b's sign
    t["x"].zero_()
    t["x"][1, 0, 0] = float("inf")
    t["a"].zero_()
    t["a"][1, 0, 0] = 1
    t["a"][1, 1:, 1] = 1  # the other ranks' h stay 0 ...
    t["x"][1, 0, 1] = 0
    t["a"][1, 0, 1:] = 0
    out, h = a()
    assert h[1, 0].isnan().sum() + h[1, 0].isinf().sum() >= 1 and out[1, 1:].isfinite().all()


@pytest.mark.parametrize("ty", [F32, BF])
def test_nothing(gpu, ty):
    import gdn2_amd as G

    ids = torch.zeros(2, dtype=torch.int32, device=gpu)
    for B, T, D, O, R, L in ((0, 4, 8, 8, 2, 1), (2, 0, 8, 8, 2, 1), (2, 3, 0, 8, 2, 1), (2, 3, 8, 0, 2, 1), (2, 3, 8, 8, 0, 1), (2, 3, 8, 8, 2, 0)):
        x, y = torch.randn(B, T, D, device=gpu).to(ty), torch.randn(B, T, O, device=gpu).to(ty)
        a, b = torch.ones(L, R, D, device=gpu).to(ty), torch.ones(L, R, O, device=gpu).to(ty)
        out, h = G.low_rank_add(y, x, a, b, ids[:B], return_hidden=True)
        assert out.shape == y.shape and h.shape == (B, T, R)
        if D == 0 or R == 0 or L == 0:
            assert torch.equal(out, y) and (h == 0).all()
        r = G.low_rank_add_backward(x, a, b, ids[:B], h, y)
        if B * T == 0 or D * O == 0:
            assert (r["da"] == 0).all() and (r["db"] == 0).all()
        if R == 0 or L == 0:
            assert (r["dx"] == 0).all()


def test_workspace_of_the_caller(gpu):
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(3, 50, 1024, 40, 8, 5, F32).items()}
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device=gpu)
    f = lambda **kw: G.low_rank_add(t["y"], t["x"], t["a"], t["b"], t["ids"], t["scale"], return_hidden=True, **kw)  # noqa: E731
    ref, h = f()
    g = lambda **kw: G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], h, t["d_out"], t["scale"], **kw)  # noqa: E731
    ref_g = g()
    for w in (ws, ws[:256]):
        got, h2 = f(workspace=w)
        assert torch.equal(got, ref) and torch.equal(h2, h)
        assert all(torch.equal(v, ref_g[k]) for k, v in g(workspace=w).items())


@pytest.mark.parametrize("ty", [F32, BF])
def test_captured(gpu, ty):
    """A serving step and a training step, replayed with other inputs, adapters and bounds."""
    import gdn2_amd as G

    t = {k: v.to(gpu) for k, v in make(1, 300, 512, 200, 16, 4, ty, cu=[0, 100, 180, 300]).items()}
    cu = torch.tensor([0, 100, 180, 300], dtype=torch.int32, device=gpu)

    def step():
        o, h = G.low_rank_add(t["y"], t["x"], t["a"], t["b"], t["ids"], t["scale"], cu_seqlens=cu, return_hidden=True)
        r = G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], h, t["d_out"], t["scale"], cu_seqlens=cu)
        return [o, h, *r.values()]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, (ids, b) in enumerate((([0, 1, 2], [0, 100, 180, 300]), ([3, 3, -1], [5, 5, 250, 299]), ([1, 0, 1], [0, 1, 2, 3]))):
        t["ids"].copy_(torch.tensor(ids))
        cu.copy_(torch.tensor(b))
        t["x"].copy_(torch.randn(t["x"].shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, step()):
            assert torch.equal(p, q)


def test_offsets_past_32_bits(gpu):
    """Rows more than 2^32 elements into their tensor."""
    import gdn2_amd as G

    T, D = 2 ** 21 + 70, 2048
    x = torch.zeros(1, T, D, dtype=BF, device=gpu)
    t = make(1, 64, D, 24, 4, 1, BF)
    x[0, -64:] = t["x"][0].to(gpu)
    y = torch.zeros(1, T, 24, dtype=BF, device=gpu)
    a, b, ids = t["a"].to(gpu), t["b"].to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    out, h = G.low_rank_add(y, x, a, b, ids, return_hidden=True)
    (want, h64), (err, h_err) = K.low_rank64(torch.zeros(64, 24, dtype=K.F64), t["x"][0].double(), t["a"].double(), t["b"].double(),
                                             torch.zeros(1), None, 1, 64)
    K.near(out[0, -64:], want, err)
    K.near(h[0, -64:], h64, h_err)
    assert (out[0, :-64] == 0).all()
    dy = torch.zeros_like(y)
    dy[0, -64:] = t["d_out"][0].to(gpu)
    got = G.low_rank_add_backward(x, a, b, ids, h, dy)
    g, e = K.low_rank_bwd64(t["x"][0].double(), t["a"].double(), t["b"].double(), torch.zeros(1), h[0, -64:].cpu().double(),
                            t["d_out"][0].double(), None, 1, 64)
    K.near(got["dx"][0, -64:], g["dx"], e["dx"])
    K.near(got["da"], g["da"], e["da"])
    K.near(got["db"], g["db"], e["db"])
