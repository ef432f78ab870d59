"""The block operators' edges on the device: C entries without rows, sums whose terms
differ much in size, large shapes of constant rows."""
import ctypes

import pytest
import torch

import block_testutil as K

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


@pytest.mark.parametrize("ty", ["f32", "bf16", "f32_bf16"])
@pytest.mark.parametrize("samples,rows", [(0, 3), (0, 0), (2, 0)])
@pytest.mark.parametrize("gate_rows", [0, 1, 2])
def test_residual_backward_entry_without_rows(gpu, ty, samples, rows, gate_rows):
    """The weights' gradients, and those of gates that no row takes, are zeros."""
    from gdn2_amd import _capi as C

    n = 40
    w, dpre, dpost = (torch.full((n,), 9.0, device=gpu) for _ in range(3))
    gate, dgate, some = (torch.full((4, n), 9.0, dtype=F32 if ty == "f32" else BF, device=gpu) for _ in range(3))
    b = C.ResidualNormBwdArgs()
    for k, v in dict(y=some, gate=gate, post_weight=w, pre_weight=w, out=some).items():
        setattr(b.fwd, k, v.data_ptr())
    for k, v in dict(samples=samples, rows=rows, channels=n, stride_gate_n=n, eps=1e-5, residual_scale=1.0, branch_scale=1.0,
                     gate_rows=gate_rows).items():
        setattr(b.fwd, k, v)
    for k, v in dict(dx=some, dy=some, dgate=dgate, dpost=dpost, dpre=dpre).items():
        setattr(b, k, v.data_ptr())
    b.stride_dgate_n = n
    assert getattr(C.lib(), "gdn2_residual_norm_bwd_" + ty)(ctypes.byref(b), torch.cuda.current_stream().cuda_stream) == C.GDN2_OK
    torch.cuda.synchronize()
    assert (dpre == 0).all() and (dpost == 0).all() and (some == 9).all()
    written = {0: 0, 1: samples, 2: 1}[gate_rows]
    assert (dgate[:written] == 0).all() and (dgate[written:] == 9).all()


@pytest.mark.parametrize("ty", [F32, BF])
def test_in_place_by_other_strides_of_dimensions_of_one(gpu, ty):
    import gdn2_amd as G

    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g).to(ty).to(gpu)  # noqa: E731
    x, y, a, b = rnd(64, 1, 40), rnd(64, 1, 40), rnd(3, 4, 40), rnd(3, 4, 40)
    w, ids = torch.rand(40, generator=g).to(gpu), (torch.arange(64, dtype=torch.int32) % 4).to(gpu)
    one = lambda t: t.as_strided(t.shape, (40, 512, 1))  # noqa: E731
    ref = G.dropout(x, 0.5, 3)
    t = x.clone()
    assert torch.equal(G.dropout(t, 0.5, 3, out=one(t)), ref) and torch.equal(t, ref)
    ref = G.residual_norm(x, y, None, w, w)
    t, u = x.clone(), y.clone()
    got = G.residual_norm(t, u, None, w, w, out=one(t), normed=one(u))
    assert all(torch.equal(p, q) for p, q in zip(got, ref)) and torch.equal(t, ref[0]) and torch.equal(u, ref[1])
    ref = G.low_rank_add(y, x, a, b, ids)
    t = y.clone()
    assert torch.equal(G.low_rank_add(t, x, a, b, ids, out=one(t)), ref) and torch.equal(t, ref)


@pytest.mark.parametrize("C,M", [(8, 2 ** 29 + 300), (520, 2 ** 21 + 5), (2056, 2 ** 21 + 5)])
def test_residual_norm_over_more_rows_than_a_launch(gpu, C, M):
    """A second turn of the workgroups' row loop, and places past 2^32 elements: the bits of
    calls on those rows alone, and in the backward the sums over all rows."""
    import gdn2_amd as G

    g = torch.Generator(device=gpu).manual_seed(C)
    rnd = lambda: torch.empty(M, C, dtype=BF, device=gpu).normal_(generator=g)  # noqa: E731
    x, y = rnd(), rnd()
    post, pre = (0.5 + torch.rand(C, generator=g, device=gpu) for _ in range(2))
    a = (None, post, pre, 1e-5, "none", 0.8, 0.5, 0.1, 7)
    out, normed, stats = G.residual_norm(x, y, *a, offset=11, return_stats=True)
    spans = [slice(r, min(r + 9, M)) for r in (0, M // 2, 2 ** 32 // C, M - 310, M - 9)]
    for at in spans:
        ref = G.residual_norm(x[at], y[at], *a, offset=11 + at.start * (C // 4), return_stats=True)
        assert all(torch.equal(p[at], q) for p, q in zip((out, normed, stats), ref))
    if M >= 2 ** 28:  # (the backward's limit)
        return
    del normed
    b = (None, post, pre, "none", 0.8, 0.5, 0.1, 7)
    got = G.residual_norm_backward(out, y, stats, x, y, *b, offset=11)  # (x and y stand for the results' gradients)
    for at in spans:
        ref = G.residual_norm_backward(out[at], y[at], stats[at], x[at], y[at], *b, offset=11 + at.start * (C // 4))
        assert all(torch.equal(got[k][at], ref[k]) for k in ("dx", "dy"))
    want = torch.zeros(C, dtype=K.F64, device=gpu)
    size = torch.zeros_like(want)
    for r in range(0, M, 2 ** 17):
        t = y[r:r + 2 ** 17].double() * out[r:r + 2 ** 17].double() * stats[r:r + 2 ** 17, 1:].double()
        want += t.sum(0)
        size += t.abs().sum(0)
    K.near(got["dpre"], want.cpu(), ((128 + 3) * K.U * size).cpu())


@pytest.mark.parametrize("ty", [F32, BF])
@pytest.mark.parametrize("C", [8, 24, 40, 320, 512])
def test_column_sums_of_narrow_rows(gpu, ty, C):
    """The rows that a workgroup holds at once (256 of 8 channels, 4 of 512) are added in 64
    bits: one of 2^24, ones, and as many rows again with -2^24 among zeros.  Each lane has
    one row; a workgroup's sum is rounded to f32, half a step of 2^24 (1) off at most."""
    import gdn2_amd as G

    lanes = 1
    while lanes * 8 < C:
        lanes *= 2
    n = 256 // lanes
    v = torch.zeros(2 * n, C, dtype=ty, device=gpu)
    v[0], v[1:n - 1], v[n] = 2.0 ** 24, 1, -2.0 ** 24
    one, w = torch.ones_like(v), torch.ones(C, device=gpu)
    stats = torch.ones(2 * n, 2, device=gpu)
    got = G.residual_norm_backward(one, one, stats, None, v, pre_weight=w)["dpre"]
    assert float((got - (n - 2)).abs().max()) <= 1
    r = G.residual_norm_backward(one, one, stats, v, None, torch.ones(C, dtype=ty, device=gpu), w)
    for k in ("dpost", "dgate"):
        assert float((r[k].float() - (n - 2)).abs().max()) <= 1, k


@pytest.mark.parametrize("C", [96, 2048])
@pytest.mark.parametrize("size", [1.2e-19, 1e-19, 1e-20, 2.0 ** -70])
def test_rows_whose_squares_are_subnormal(gpu, C, size):
    """Without eps: both statistics are finite.  A square, and the mean, are each off by half
    of 2^-149 at most, halved by the root; the rest as in block_testutil."""
    import gdn2_amd as G

    x = torch.full((3, C), size, device=gpu)
    x[1] *= -1
    x[2] = 0
    w = torch.ones(C, device=gpu)
    got, n, stats = G.residual_norm(torch.zeros_like(x), x, None, w, w, eps=0.0, return_stats=True)
    rel = 2.0 ** -150 / size ** 2 + 25 * K.U
    assert float((stats[:2, 0].double() * x[0, 0].double() - 1).abs().max()) <= rel
    assert float((got[:2].double() - torch.tensor([[1.0], [-1.0]], device=gpu)).abs().max()) <= rel
    assert stats[2, 0].isinf() and got[2].isnan().all()  # 1 / 0, and 0 times it
    _, n, stats = G.residual_norm(x, pre_weight=w, eps=0.0, return_stats=True)
    assert float((stats[:2, 1].double() * x[0, 0].double() - 1).abs().max()) <= rel
    assert float((n[:2].double() - torch.tensor([[1.0], [-1.0]], device=gpu)).abs().max()) <= rel


@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False), (False, False)])
def test_statistics_of_rows_of_no_channels(gpu, post, pre):
    """NaN, the mean of nothing, for a norm that is taken, else 0: never what memory held."""
    import gdn2_amd as G

    x, w = torch.empty(2, 3, 0, device=gpu), torch.empty(0, device=gpu)
    for _ in range(3):
        del_me = torch.full((12,), 7.0, device=gpu)  # what the allocator gives out next
        del del_me
        o, n, st = G.residual_norm(x, x, None, w if post else None, w if pre else None, return_stats=True)
        assert st.shape == (2, 3, 2) and o.shape == x.shape
        for i, taken in enumerate((post, pre)):
            assert st[..., i].isnan().all() if taken else (st[..., i] == 0).all()
    r = G.residual_norm_backward(o, x, st, o, o if pre else None, None, w if post else None, w if pre else None)
    assert r["dx"].shape == r["dy"].shape == x.shape
