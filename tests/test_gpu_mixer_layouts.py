"""The mixer operators' results for operands that lie apart in a larger tensor."""
import pytest

pytestmark = pytest.mark.gpu


def _small(*tensors):
    for t in tensors:
        if t is not None:
            held, needed = t.untyped_storage().nbytes(), t.numel() * t.element_size()
            assert held <= 4 * needed + 512, (tuple(t.shape), t.stride())


def test_results_take_little_memory(gpu):
    """The last token of every sequence, every eighth head: results are of the operands'
    size, whatever lies between those."""
    import torch

    import gdn2_amd as G

    big = torch.randn(6, 500, 16, 64, device=gpu)
    x = big.view(6, 500, 1024)[:, -1]
    print("norm", flush=True)
    y, stats = G.group_norm_act(x, 16, return_stats=True)
    want, want_stats = G.group_norm_act(x.contiguous(), 16, return_stats=True)
    r = G.group_norm_act_backward(x, 16, stats, x.clone(), gate=x)
    want_r = G.group_norm_act_backward(x.contiguous(), 16, stats, x.clone(), gate=x.contiguous())
    assert torch.equal(y, want) and torch.equal(stats, want_stats)
    assert all(torch.equal(r[n], want_r[n]) for n in r)
    _small(y, r["dx"], r["dgate"])

    v, g = big[:, :, ::8].transpose(1, 2), -big[:, :, 1::8, :1].abs().transpose(1, 2)
    w = big[:, :, 2::8].transpose(1, 2)
    for ww in (None, w, w.contiguous()):
        print("scan", None if ww is None else ww.stride(), flush=True)
        out, new = G.gated_scan(g, v, ww)
        r = G.gated_scan_backward(g, v, ww, out, torch.ones_like(out))
        c = [None if t is None else t.contiguous() for t in (g, v, ww)]
        want, _ = G.gated_scan(*c)
        want_r = G.gated_scan_backward(*c, want, torch.ones_like(want))
        assert torch.equal(out, want) and all(r[n] is None or torch.equal(r[n], want_r[n]) for n in r)
        _small(out, new, *r.values())


def test_strides_of_one_element_do_not_count(gpu):
    """`out` that differs from x in the stride of a dimension of one alone is taken."""
    import torch

    import gdn2_amd as G

    for shape, strides in (((1, 40, 64), (99999, 64, 1)), ((5, 1, 64), (64, 7, 1)), ((1, 64), (3, 1))):
        x, out = torch.randn(shape, device=gpu), torch.empty_strided(shape, strides, device=gpu)
        y = G.group_norm_act(x, 4, out=out)
        assert y is out and torch.equal(y, G.group_norm_act(x, 4))
        y, stats = G.group_norm_act(x, 4, return_stats=True)
        dy = torch.randn(shape, device=gpu)
        r = G.group_norm_act_backward(x, 4, stats, torch.empty_strided(shape, strides, device=gpu).copy_(dy))
        want = G.group_norm_act_backward(x, 4, stats, dy)
        assert all(r[n] is None or torch.equal(r[n], want[n]) for n in r)
    v, w = torch.randn(2, 1, 16, 128, device=gpu).transpose(1, 2), torch.rand(2, 16, 1, 128, device=gpu)
    g = -torch.rand(2, 16, 1, 1, device=gpu)
    out, new = G.gated_scan(g, v, w)
    want, last = G.gated_scan(g, v.contiguous(), w)
    r, want_r = (G.gated_scan_backward(g, v, w, out, d) for d in (torch.ones_like(out), torch.ones(2, 16, 1, 128, device=gpu)))
    assert torch.equal(out, want) and torch.equal(new, last) and all(torch.equal(r[n], want_r[n]) for n in r)


def test_statistics_of_nothing(gpu):
    """Groups of no rows have no mean: their statistics are NaN, not what the memory
    held before."""
    import torch

    import gdn2_amd as G

    for shape in ((4, 0, 64), (2, 0, 5, 64), (3, 5, 0), (7, 0)):
        junk = [torch.full((n,), 7.0, device=gpu) for n in (128, 256, 512)]
        del junk
        y, stats = G.group_norm_act(torch.empty(shape, device=gpu), 4, return_stats=True)
        assert y.shape == shape and stats.shape == (shape[0], 4, 2) and torch.isnan(stats).all()
