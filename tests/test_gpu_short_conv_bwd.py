"""short_conv_1d_backward against its plain 64-bit form."""
import numpy as np
import pytest

import mixer_testutil as M

pytestmark = pytest.mark.gpu


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


CASES = [(1, 1, 1), (2, 2, 4), (2, 3, 96), (1, 4, 250), (3, 7, 256), (1, 8, 33), (2, 9, 64), (1, 31, 128), (1, 33, 300),
         (2, 65, 12), (1, 130, 1537), (3, 200, 512), (2, 777, 96), (40, 5, 260), (1, 3000, 64)]


def _make(gpu, seed, B, T, C, cache):
    import torch

    r = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=r).to(gpu)  # noqa: E731
    return {"x": rand(B, T, C), "weight": (torch.rand(C, 4, generator=r) - 0.5).to(gpu), "d_out": rand(B, T, C),
            "cache": rand(B, 3, C) if cache else None, "d_cache": rand(B, 3, C)}


def _check(d, r):
    want, err = M.conv_bwd64(*(_np(d[n]) for n in ("x", "weight", "cache", "d_out", "d_cache")))
    assert (r["dcache"] is None) == (d["cache"] is None)
    for n in ("dx", "dweight", "dcache"):
        if r[n] is not None:
            e = M.worst(_np(r[n]), want[n], err[n], 0)
            assert e <= 1, (n, e)


@pytest.mark.parametrize("B,T,C", CASES)
def test_matches_the_plain_form(gpu, B, T, C):
    import torch

    import gdn2_amd as G

    for cache in (False, True):
        for dc in (False, True):
            print("conv backward", B, T, C, cache, dc, flush=True)
            d = _make(gpu, T + C, B, T, C, cache)
            if not dc:
                d["d_cache"] = None
            r = G.short_conv_1d_backward(**d)
            r2 = G.short_conv_1d_backward(**d)
            torch.cuda.synchronize()
            assert all(r[n] is None or torch.equal(r[n], r2[n]) for n in r)  # sums in one order
            _check(d, r)


def test_no_tokens(gpu):
    import torch

    import gdn2_amd as G

    x, w, c = torch.empty(2, 0, 8, device=gpu), torch.randn(8, 4, device=gpu), torch.randn(2, 3, 8, device=gpu)
    r = G.short_conv_1d_backward(x, w, x, c, d_cache=c)
    assert torch.equal(r["dcache"], c) and (r["dweight"] == 0).all() and r["dx"].shape == x.shape
    r = G.short_conv_1d_backward(x, w, x, c)
    assert (r["dcache"] == 0).all()
    x = torch.empty(0, 5, 8, device=gpu)
    assert (G.short_conv_1d_backward(x, w, x)["dweight"] == 0).all()


def test_layouts(gpu):
    """Strided and unaligned operands (copied, as the forward copies them)."""
    import gdn2_amd as G

    d = _make(gpu, 3, 2, 70, 64, True)
    e = dict(d, x=d["x"].transpose(0, 1).contiguous().transpose(0, 1), d_out=d["d_out"].expand(2, 70, 64))
    _check(d, G.short_conv_1d_backward(**e))
    flat = d["x"].new_empty(2 * 70 * 64 + 1)[1:].view(2, 70, 64)  # 4 bytes from an aligned place
    flat.copy_(d["x"])
    _check(d, G.short_conv_1d_backward(**dict(d, x=flat)))


def test_streams_and_graphs(gpu):
    import torch

    import gdn2_amd as G

    d = [_make(gpu, 50 + i, 2, 900, 128, True) for i in range(2)]
    want = [G.short_conv_1d_backward(**x) for x in d]
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = G.short_conv_1d_backward(**d[i])
    torch.cuda.synchronize()
    assert all(torch.equal(got[i][n], want[i][n]) for i in range(2) for n in want[i])
    x = {n: t.clone() for n, t in d[0].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = G.short_conv_1d_backward(**x)
    for k in range(4):
        for n in x:
            x[n].copy_(d[k % 2][n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(r[n], want[k % 2][n]) for n in r)
        G.short_conv_1d_backward(**d[k % 2])
