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
