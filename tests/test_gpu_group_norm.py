"""group_norm_act and group_norm_act_backward against their plain 64-bit forms:
groups from one channel to thousands, one row to many, every form of their
arguments."""
import numpy as np
import pytest

import mixer_testutil as M

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _types(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _make(gpu, seed, N, S, C, ty, gate, affine=True, shift=0.5):
    import torch

    r = torch.Generator().manual_seed(seed)
    x = torch.randn(N, S, C, generator=r) * (torch.rand(C, generator=r) + 0.5) + shift * torch.randn(C, generator=r)
    d = {"x": x.to(gpu, _types(ty)), "gate": torch.randn(N, S, C, generator=r).to(gpu, _types(ty)) if gate else None,
         "weight": (torch.rand(C, generator=r) + 0.5).to(gpu) if affine else None,
         "bias": (torch.randn(C, generator=r) * 0.3).to(gpu) if affine else None}
    return d, torch.randn(N, S, C, generator=r).to(gpu, _types(ty))


def _check_forward(d, groups, act, y, stats, ty, shape=None):
    x = _np(d["x"])
    shape = shape or x.shape
    gate = None if d["gate"] is None else _np(d["gate"]).reshape(shape)
    f = M.norm64(x.reshape(shape), groups, _np(d["weight"]), _np(d["bias"]), EPS, act, gate)
    e = M.worst(_np(y).reshape(shape), f["y"], f["y_err"], M.HALF[ty])
    assert e <= 1, ("y", e)
    if stats is not None:
        e = M.worst(_np(stats), f["stats"], f["stats_err"], 0)
        assert e <= 1, ("stats", e)


def _check_backward(d, groups, act, stats, dy, r, ty, shape=None):
    x = _np(d["x"])
    shape = shape or x.shape
    gate = None if d["gate"] is None else _np(d["gate"]).reshape(shape)
    want, err = M.norm_bwd64(x.reshape(shape), groups, _np(d["weight"]), _np(d["bias"]), act, gate, _np(stats),
                             _np(dy).reshape(shape))
    assert (r["dgate"] is None) == (gate is None) and r["dx"].shape == d["x"].shape
    for n in ("dx", "dgate", "dweight", "dbias"):
        if r[n] is not None:
            got = _np(r[n]).reshape(want[n].shape)
            e = M.worst(got, want[n], err[n], M.HALF[ty] if n in ("dx", "dgate") else 0)
            assert e <= 1, (n, e)


CASES = [  # N, S, C, groups
    (1, 1, 1, 1), (5, 1, 7, 7), (9, 1, 128, 1), (33, 1, 256, 2), (17, 1, 2048, 16), (6, 1, 96, 3), (7, 1, 330, 10),
    (70, 1, 320, 32), (5, 1, 500, 2), (3, 1, 2048, 1), (4, 1, 4096, 1), (3, 1, 5000, 2), (2, 1, 8192, 1), (3, 1, 1001, 1),
    (2, 1, 1500, 1), (600, 1, 64, 4), (3, 2, 64, 4), (2, 5, 10, 2), (1, 9, 33, 3), (2, 100, 320, 32), (1, 257, 1024, 32),
    (3, 64, 7, 1), (4, 1000, 64, 8), (1, 5000, 12, 3), (2, 33, 1100, 4), (300, 3, 40, 4),
    # a group held by several workgroups: by rows, by channels, by both; too many for that; odd widths
    (2, 513, 128, 4), (1, 4096, 128, 1), (2, 4097, 64, 2), (1, 2100, 512, 1), (2, 40, 4100, 1), (1, 700, 1500, 3),
    (2, 600, 264, 8), (2, 90, 500, 2), (3, 37, 65, 5), (1, 3100, 96, 32), (1, 9000, 24, 2), (2, 17, 130, 2), (5, 8, 9, 9),
]


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("N,S,C,groups", CASES)
def test_both_ways(gpu, N, S, C, groups, ty):
    import torch

    import gdn2_amd as G

    for k, (act, gate, affine) in enumerate([("silu", False, True), ("silu", True, True), ("gelu", False, True),
                                             ("gelu", True, False), ("none", False, False), ("none", True, True)]):
        print("norm", N, S, C, groups, ty, act, gate, affine, flush=True)
        d, dy = _make(gpu, 10 * C + k, N, S, C, ty, gate, affine)
        if C // groups * S == 1:
            d["x"][...] = 1.25  # a group of one: variance zero
        y, stats = G.group_norm_act(d["x"], groups, d["weight"], d["bias"], EPS, act, gate=d["gate"], return_stats=True)
        y2 = G.group_norm_act(d["x"], groups, d["weight"], d["bias"], EPS, act, gate=d["gate"])
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and y.dtype == _types(ty) and stats.shape == (N, groups, 2)
        _check_forward(d, groups, act, y, stats, ty)
        r = G.group_norm_act_backward(d["x"], groups, stats, dy, d["weight"], d["bias"], act, gate=d["gate"])
        r2 = G.group_norm_act_backward(d["x"], groups, stats, dy, d["weight"], d["bias"], act, gate=d["gate"])
        torch.cuda.synchronize()
        assert all(r[n] is None or torch.equal(r[n], r2[n]) for n in r)  # sums in one order
        _check_backward(d, groups, act, stats, dy, r, ty)


def test_many_rows_and_samples(gpu):
    """Sums over tens of thousands of rows."""
    import gdn2_amd as G

    for N, S, C, groups in ((20000, 1, 64, 2), (2, 20000, 64, 4), (5000, 4, 32, 2)):
        print("rows", N, S, C, flush=True)
        d, dy = _make(gpu, N, N, S, C, "f32", True)
        y, stats = G.group_norm_act(d["x"], groups, d["weight"], d["bias"], EPS, "silu", gate=d["gate"], return_stats=True)
        _check_forward(d, groups, "silu", y, stats, "f32")
        r = G.group_norm_act_backward(d["x"], groups, stats, dy, d["weight"], d["bias"], "silu", gate=d["gate"])
        _check_backward(d, groups, "silu", stats, dy, r, "f32")


@pytest.mark.parametrize("looks", [0, 3])
def test_parts_formed_by_those_who_wait(gpu, looks):
    """A workgroup that stops waiting for another's sums forms them itself: the same
    bits, whichever parts that were."""
    import torch

    import gdn2_amd as G
    from gdn2_amd import _capi as C

    for N, S, C_, groups, ty in ((3, 700, 128, 4, "f32"), (2, 333, 320, 32, "bf16"), (1, 40, 2048, 1, "f32"), (2, 900, 33, 11, "f32")):
        for gate in (False, True):
            d, dy = _make(gpu, S, N, S, C_, ty, gate)

            def both():
                y, st = G.group_norm_act(d["x"], groups, d["weight"], d["bias"], EPS, "silu", gate=d["gate"], return_stats=True)
                r = G.group_norm_act_backward(d["x"], groups, st, dy, d["weight"], d["bias"], "silu", gate=d["gate"])
                return [y, st] + [t for t in r.values() if t is not None]

            want = both()
            torch.cuda.synchronize()
            before = C.lib().gdn2_group_norm_patience(looks)
            try:
                got = both()
                torch.cuda.synchronize()
            finally:
                assert C.lib().gdn2_group_norm_patience(before) == looks
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (N, S, C_, groups, gate)


@pytest.mark.parametrize("N,S", [(8, 1), (2, 300)])
def test_large_mean(gpu, N, S):
    """A mean of 1000 standard deviations: sums of raw squares would leave nothing
    of the variance.  The mean's own rounding, half a step of 1000, is 2^-14 of a
    standard deviation, which the bound counts."""
    import torch

    import gdn2_amd as G

    x = torch.randn(N, S, 256, device=gpu) + 1000.0
    y, stats = G.group_norm_act(x, 4, eps=EPS, activation="none", return_stats=True)
    r = x.double().view(N, S, 4, 64)
    var, mean = torch.var_mean(r, (1, 3), unbiased=False)
    assert ((stats[..., 0] - mean).abs() <= 1000 * (M.SUM + 8) * M.EPS).all()
    rel = (stats[..., 1].double() * torch.sqrt(var + EPS) - 1).abs()
    # squares about a point at most 1000 M.SUM EPS off the mean, and their own roundings
    assert (rel <= 0.5 * ((1000 * (M.SUM + 8) * M.EPS) ** 2 + 20 * M.SUM * M.EPS) + 4 * M.EPS).all()


def test_zero_and_extreme_rows(gpu):
    """Constant groups give act(bias); zeros too; a NaN or an infinity stays in its
    sample's group."""
    import torch

    import gdn2_amd as G

    for N, S in ((6, 1), (6, 50)):
        x = torch.randn(N, S, 64, device=gpu)
        x[0] = 0.0
        x[1] = 3.0
        bias = torch.randn(64, device=gpu)
        x[2, 0, 3] = float("nan")
        x[3, 0, 20] = float("inf")
        y, stats = G.group_norm_act(x, 4, None, bias, EPS, "none", return_stats=True)
        want = bias.expand(S, 64)
        assert torch.equal(y[0], want) and (y[1] - want).abs().max() <= 3 * M.SUM * M.EPS / EPS ** 0.5
        assert torch.isnan(y[2, :, :16]).all() and torch.isfinite(y[2, :, 16:]).all()
        assert not torch.isfinite(y[3, 0, 16:32]).all() and torch.isfinite(y[3, :, :16]).all()
        assert torch.isfinite(y[3, :, 32:]).all() and torch.isfinite(y[4:]).all()
        dy = torch.randn_like(x)
        r = G.group_norm_act_backward(x, 4, stats, dy, None, bias, "none")
        assert torch.isfinite(r["dx"][4:]).all() and torch.isfinite(r["dx"][2, :, 16:]).all()


def test_layouts_and_shapes(gpu):
    """Rows of a wider buffer, unaligned ones, [M, C] and [N, H, W, C], results in
    given buffers and in place."""
    import torch

    import gdn2_amd as G

    for N, S in ((5, 1), (3, 40)):
        d, dy = _make(gpu, 77, N, S, 64, "f32", True)
        y, stats = G.group_norm_act(d["x"], 4, d["weight"], d["bias"], EPS, "silu", gate=d["gate"], return_stats=True)
        for lead in (0, 1, 4):
            big = torch.full((N, S, 80), 9.0, device=gpu)
            x = big[..., lead:lead + 64]
            x.copy_(d["x"])
            e = dict(d, x=x)
            o, st = G.group_norm_act(x, 4, d["weight"], d["bias"], EPS, "silu", gate=d["gate"], return_stats=True)
            _check_forward(e, 4, "silu", o, st, "f32")
            r = G.group_norm_act_backward(x, 4, st, dy, d["weight"], d["bias"], "silu", gate=d["gate"])
            _check_backward(e, 4, "silu", st, dy, r, "f32")
            o = G.group_norm_act(x, 4, d["weight"], d["bias"], EPS, "silu", gate=d["gate"], out=x)  # in place
            assert o is x
            _check_forward(d, 4, "silu", x, None, "f32")
            assert (big[..., :lead] == 9).all() and (big[..., lead + 64:] == 9).all()
        turned = {n: (t.transpose(0, 1).contiguous().transpose(0, 1) if t is not None and t.dim() == 3 else t)
                  for n, t in d.items()}
        o, st = G.group_norm_act(turned["x"], 4, d["weight"], d["bias"], EPS, "silu", gate=turned["gate"], return_stats=True)
        _check_forward(d, 4, "silu", o, st, "f32")
        strided = torch.stack([d["x"]] * 2, -1)[..., 0]
        o = G.group_norm_act(strided, 4, d["weight"], d["bias"], EPS, "silu", gate=d["gate"])
        assert torch.equal(o, y)
    d, dy = _make(gpu, 78, 6, 1, 64, "f32", False)
    two = {n: (t[:, 0] if t is not None and t.dim() == 3 else t) for n, t in d.items()}
    o, st = G.group_norm_act(two["x"], 4, d["weight"], d["bias"], EPS, "gelu", return_stats=True)
    assert o.shape == (6, 64)
    _check_forward(d, 4, "gelu", o, st, "f32", (6, 1, 64))
    r = G.group_norm_act_backward(two["x"], 4, st, dy[:, 0], d["weight"], d["bias"], "gelu")
    _check_backward(two, 4, "gelu", st, dy, r, "f32", (6, 1, 64))
    d, dy = _make(gpu, 79, 2, 30, 64, "f32", True)
    four = {n: (t.view(2, 5, 6, 64) if t is not None and t.dim() == 3 else t) for n, t in d.items()}
    o, st = G.group_norm_act(four["x"], 8, d["weight"], d["bias"], EPS, "silu", gate=four["gate"], return_stats=True)
    assert o.shape == (2, 5, 6, 64)
    _check_forward(d, 8, "silu", o, st, "f32", (2, 30, 64))
    r = G.group_norm_act_backward(four["x"], 8, st, dy.view(2, 5, 6, 64), d["weight"], d["bias"], "silu", gate=four["gate"])
    _check_backward(four, 8, "silu", st, dy, r, "f32", (2, 30, 64))


def test_nothing(gpu):
    import torch

    import gdn2_amd as G

    for shape in ((0, 3, 64), (4, 0, 64), (0, 64), (0, 3, 5, 64), (2, 0, 5, 64)):
        x = torch.empty(shape, device=gpu)
        y, stats = G.group_norm_act(x, 4, return_stats=True)
        assert y.shape == shape
        r = G.group_norm_act_backward(x, 4, stats, x)
        assert r["dx"].shape == shape and (r["dweight"] == 0).all() and (r["dbias"] == 0).all()


def test_offsets_past_32_bits(gpu):
    """Samples further apart than 2^31 elements."""
    import torch

    import gdn2_amd as G

    for S in (1, 20):
        st = (1 << 30) + 64
        wide = [torch.as_strided(torch.empty(2 * st + 64 * S, dtype=torch.bfloat16, device=gpu), (3, S, 64), (st, 64, 1))
                for _ in range(2)]
        d, dy = _make(gpu, 5, 3, S, 64, "bf16", False)
        wide[0].copy_(d["x"])
        y, stats = G.group_norm_act(d["x"], 2, d["weight"], d["bias"], EPS, return_stats=True)
        assert torch.equal(G.group_norm_act(wide[0], 2, d["weight"], d["bias"], EPS, out=wide[1]), y)


def test_streams_and_graphs(gpu):
    import torch

    import gdn2_amd as G

    for N, S in ((500, 1), (3, 700)):
        d = [_make(gpu, 40 + i, N, S, 256, "f32", True) for i in range(2)]

        def both(x, dy):
            y, st = G.group_norm_act(x["x"], 4, x["weight"], x["bias"], EPS, "silu", gate=x["gate"], return_stats=True)
            r = G.group_norm_act_backward(x["x"], 4, st, dy, x["weight"], x["bias"], "silu", gate=x["gate"])
            return [y, st] + [r[n] for n in ("dx", "dgate", "dweight", "dbias")]

        want = [both(*x) for x in d]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[i] = both(*d[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
        x, dy = {n: t.clone() for n, t in d[0][0].items()}, d[0][1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(x, dy)
        for k in range(4):
            for n in x:
                x[n].copy_(d[k % 2][0][n])
            dy.copy_(d[k % 2][1])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, both(*d[k % 2]))), (N, S, k)
