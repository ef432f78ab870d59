"""low_rank_add and its backward where the kernels' loops over features run several
times: wide rows in every shape of tile, many ranks over many and packed rows, workspaces
that hold anything, infinite products.  The 64-bit forms are formed on the device."""
import pytest
import torch

import block_testutil as K

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def make(gpu, B, T, D, O, R, L, ty, cu=None, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed * 77 + B + T + D + O + R + L)
    rnd = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    n = B if cu is None else len(cu) - 1
    return {"x": rnd(B, T, D).to(ty), "y": rnd(B, T, O).to(ty), "a": (rnd(L, R, D) * D ** -0.5).to(ty),
            "b": (rnd(L, R, O) * R ** -0.5).to(ty),
            "ids": (torch.arange(n, device=gpu) % (L + 1)).int(),  # (L: none)
            "scale": 0.5 + torch.rand(L, generator=g, device=gpu), "d_out": rnd(B, T, O).to(ty), "dx": rnd(B, T, D).to(ty)}


def both(t, cu=None, dx=None, **kw):
    import gdn2_amd as G

    out, h = G.low_rank_add(t["y"], t["x"], t["a"], t["b"], t["ids"], t["scale"], cu_seqlens=cu, return_hidden=True, **kw)
    return {"out": out, "hidden": h, **G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], h, t["d_out"], t["scale"],
                                                               cu_seqlens=cu, dx=dx, **kw)}


def check(gpu, B, T, D, O, R, ty, L=2, cu=None):
    """Bounds of every value, and (block_testutil.alike) of each result as a whole: n terms
    of either sign, added one after the other, come to about (n / 6)^1/2 half steps of a sum
    of their size (partial sums grow as a square root, a rounding's deviation is 1 / 3^1/2
    of half a step); 2100 features and then 4096 rows to 32, below its 64."""
    t = make(gpu, B, T, D, O, R, L, ty, cu)
    got = both(t, None if cu is None else torch.tensor(cu, dtype=torch.int32, device=gpu), t["dx"].clone())
    flat = {k: v.double().reshape(-1, v.shape[-1]) if k in ("x", "y", "d_out", "dx") else v.double() for k, v in t.items()}
    with gpu:
        (out, h), (err, h_err) = K.low_rank64(flat["y"], flat["x"], flat["a"], flat["b"], t["ids"], flat["scale"], B, T, cu)
        want, errs = K.low_rank_bwd64(flat["x"], flat["a"], flat["b"], t["ids"], got["hidden"].double().reshape(B * T, R),
                                      flat["d_out"], flat["scale"], B, T, cu, flat["dx"])
    want, errs = dict(want, out=out, hidden=h), dict(errs, out=err, hidden=h_err)
    for k, v in got.items():
        K.near(v, want[k].cpu(), errs[k].cpu(), k)
        K.alike(v, want[k].cpu(), k)


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("B,T", [
    (1, 1000),   # 16 rows a tile, eight waves
    (600, 13),   # ... four waves, short requests
    (1, 6150),   # 193 tiles of 32 rows
    (1, 8200),   # 257 of 32, 513 of 16
    (1, 10300),  # 322 of 32
    (3, 11000)])  # 1032 of 32
@pytest.mark.parametrize("R", [16, 24, 64])
def test_wide_features(gpu, ty, B, T, R):
    """Two and more chunks of features a wave, two and more steps over the columns; features
    that end in fewer columns than a lane holds (2051) and in part of a tile (1549)."""
    check(gpu, B, T, 2051, 1549, R, ty)


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [65, 130])
@pytest.mark.parametrize("B,T", [(2, 500), (1, 8200)])  # tiles of 16 rows; 129 of 64
def test_many_ranks(gpu, ty, B, T, R):
    check(gpu, B, T, 1301, 1100, R, ty)


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [65, 130])
@pytest.mark.parametrize("cu", [[5, 5, 6, 40, 40, 333, 1000, 1017, 1017], [0, 1, 1, 70, 4096, 4099, 8000, 8333]])
def test_many_ranks_packed(gpu, ty, R, cu):
    """Requests of no tokens, of one, ragged ones; rows before and behind all of them.  The
    longer ones in tiles of 64 rows for the first product and of 32 for the second."""
    check(gpu, 1, cu[-1] + 3, 700, 645, R, ty, L=4, cu=cu)


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [16, 64])
def test_wide_features_packed(gpu, ty, R):
    g = torch.Generator().manual_seed(R)
    cu = [1] + torch.randint(1, 8300, (17,), generator=g).sort().values.tolist() + [8301]
    check(gpu, 1, 8307, 2051, 1549, R, ty, L=4, cu=cu)


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [8, 65, 100])
@pytest.mark.parametrize("packed", [False, True])
def test_workspaces_that_hold_anything(gpu, ty, R, packed):
    """NaN in the caller's workspace reach no result; too small a one is not used."""
    cu = [3, 3, 50, 51, 140] if packed else None
    t = make(gpu, 1 if packed else 4, 150, 200, 90, R, 3, ty, cu)
    t["ids"].copy_(torch.tensor([1, -1, 2, 0]))
    dcu = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=gpu)
    ref = both(t, dcu)
    assert all(v.isfinite().all() for v in ref.values())
    for n in (1 << 26, 256):
        ws = torch.full((n,), 255, dtype=torch.uint8, device=gpu)
        got = both(t, dcu, workspace=ws)
        assert all(torch.equal(got[k], v) for k, v in ref.items())


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [1, 8, 40, 100])
def test_infinite_products(gpu, ty, R):
    """An infinite h gives infinities of b's sign, NaN where b is zero, and so dh of dx;
    other rows stay finite."""
    t = make(gpu, 2, 20, 96, 80, R, 1, ty)
    t["ids"].zero_()
    t["x"][:, :, 0] = 0
    t["x"][1, 3] = 0
    t["x"][1, 3, 0] = float("inf")
    sign = torch.where(torch.arange(R, device=gpu) % 2 == 0, 1.0, -1.0)
    t["a"][0] = t["a"][0].abs() + 0.1
    t["a"][0] *= sign[:, None].to(ty)
    cols = torch.where(torch.arange(80, device=gpu) % 3 == 0, -1.0, 1.0)
    t["b"][0] = ((0.5 + torch.rand(R, 80, device=gpu)) * sign[:, None] * cols).to(ty)
    t["b"][0, 0, 7] = 0
    got = both(t)
    out, h = got["out"], got["hidden"]
    assert torch.equal(h[1, 3], sign * float("inf"))
    want = cols * float("inf")
    want[7] = float("nan")
    assert torch.equal(out[1, 3].float().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
    keep = torch.ones(2, 20, dtype=torch.bool, device=gpu)
    keep[1, 3] = False
    assert out[keep].isfinite().all() and h[keep].isfinite().all()
    # the gradients: an infinite row of d_out in one place whose b has one sign in all ranks
    t["x"][1, 3, 0] = 1
    t["b"][0, :, 5] = sign.to(ty)
    t["d_out"][0, 2] = 0
    t["d_out"][0, 2, 5] = -float("inf")
    got = both(t)
    assert torch.equal(got["dx"][0, 2].float(), torch.full((96,), -float("inf"), device=gpu))
    keep = torch.ones(2, 20, dtype=torch.bool, device=gpu)
    keep[0, 2] = False
    assert got["dx"][keep].isfinite().all()


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("R", [8, 100])
def test_scales_that_are_not_finite(gpu, ty, R):
    """db is the scale times a sum, of zero too; an adapter without requests has zeros,
    whatever its scale."""
    import gdn2_amd as G

    t = make(gpu, 3, 40, 96, 80, R, 3, ty)
    t["ids"].copy_(torch.tensor([0, 2, 0]))
    t["d_out"][..., 3] = 0
    hidden = torch.randn(3, 40, R, device=gpu)
    grads = lambda: G.low_rank_add_backward(t["x"], t["a"], t["b"], t["ids"], hidden, t["d_out"], t["scale"])  # noqa: E731
    ref = grads()
    t["scale"][0], t["scale"][1] = float("inf"), float("nan")
    got = grads()
    want = ref["db"].sign() * float("inf")
    want[:, :, 3] = float("nan")
    assert torch.equal(got["db"][0].nan_to_num(nan=7.0), want[0].nan_to_num(nan=7.0))
    assert (got["db"][1] == 0).all() and (got["da"][1] == 0).all()
    assert all(torch.equal(got[k][2], ref[k][2]) for k in ("da", "db")) and torch.equal(got["dx"][1], ref["dx"][1])
