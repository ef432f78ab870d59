"""dropout against the generator's words formed on the host: the same bits."""
import pytest
import torch

import block_testutil as K

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def want(x, p, seed, offset=0):
    """On the host: one product in f32, rounded once."""
    C = x.shape[-1]
    k = K.kept(x.numel() // C, C, p, seed, offset).reshape(x.shape)
    s = torch.tensor(1 / (1 - p) if p < 1 else 0.0, dtype=torch.float32)
    return torch.where(k, x.float() * s, torch.zeros(())).to(x.dtype)


def same(a, b):
    return a.dtype == b.dtype and torch.equal(a.cpu().view(torch.int16 if a.dtype == BF else torch.int32),
                                               b.contiguous().view(torch.int16 if a.dtype == BF else torch.int32))


@pytest.mark.parametrize("ty", [torch.float32, BF])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 1), (5, 3), (4, 8), (7, 12), (2, 33, 250), (1, 2048), (64, 2048),
                                   (777, 1537), (3, 5, 7, 96), (4097, 24), (1, 100003)])
def test_rows(gpu, ty, shape):
    import gdn2_amd as G

    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g).to(ty)
    for p, seed, offset in ((0.1, 7, 0), (0.5, 2 ** 63 + 12345, 2 ** 32 - 3), (0.25, -1, 2 ** 64 - 2)):
        y = G.dropout(x.to(gpu), p, seed, offset)
        assert y.shape == x.shape and same(y.contiguous(), want(x, p, seed, offset)), (p, seed, offset)
        assert torch.equal(y, G.dropout_backward(x.to(gpu), p, seed, offset))


@pytest.mark.parametrize("ty", [torch.float32, BF])
def test_shares_of_nothing_and_all(gpu, ty):
    import gdn2_amd as G

    x = torch.randn(9, 40).to(ty)
    x[0, 0], x[1, 1], x[2, 2] = float("nan"), float("inf"), -float("inf")
    assert same(G.dropout(x.to(gpu), 0.0), x)
    assert same(G.dropout(x.to(gpu), 1.0), torch.zeros_like(x))  # whatever x holds
    y = G.dropout(x.to(gpu), 0.5, 3).cpu()
    k = K.kept(9, 40, 0.5, 3)
    assert (y[~k] == 0).all() and torch.equal(y[k].isnan(), x[k].isnan())


@pytest.mark.parametrize("ty", [torch.float32, BF])
def test_layouts(gpu, ty):
    """The mask goes by place, whatever the strides; memory beside the rows is left alone."""
    import gdn2_amd as G

    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 10, 40, generator=g).to(ty)
    d = x.to(gpu)
    ref = want(x, 0.3, 5, 11)
    for v in (d.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([d, d], 2)[..., 40:], torch.cat([d, d], 2)[..., :40],
              d.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([d, d], 1)[:, 10:]):
        assert not v.is_contiguous() and same(G.dropout(v, 0.3, 5, 11).contiguous(), ref)
    e = d[0, 0, :1].expand(4, 8)
    assert same(G.dropout(e, 0.3, 5).contiguous(), want(e.cpu().contiguous(), 0.3, 5))
    for n in (0, 1, 2):  # rows in a wider buffer, of odd starts, too
        buf = torch.full((60, 83), 9.0, dtype=ty, device=gpu)
        out = buf[:, n:n + 40]
        assert G.dropout(d.view(60, 40), 0.3, 5, 11, out=out) is out
        assert same(out.contiguous(), ref.view(60, 40)) and (buf[:, :n] == 9).all() and (buf[:, n + 40:] == 9).all()
    out = torch.empty(10, 6, 40, dtype=ty, device=gpu).transpose(0, 1)  # rows not evenly apart
    assert G.dropout(d, 0.3, 5, 11, out=out) is out and same(out.contiguous(), ref)
    assert G.dropout(d, 0.3, 5, 11, out=d) is d and same(d, ref)  # in place


def test_nothing(gpu):
    import gdn2_amd as G

    for s in ((0, 8), (3, 0), (0,)):
        x = torch.empty(s, device=gpu)
        assert G.dropout(x, 0.5).shape == s and G.dropout(x, 0.5, out=x) is x


def test_large_offsets_of_elements(gpu):
    """More than 2^32 elements in one call: the last ones' counters and places."""
    import gdn2_amd as G

    rows, C = 2 ** 21 + 3, 2048
    x = torch.ones(rows, C, dtype=BF, device=gpu)
    G.dropout(x, 0.5, 4, out=x)
    for r in (0, 2 ** 20, 2 ** 21, rows - 1):
        ref = want(torch.ones(1, C, dtype=BF), 0.5, 4, r * (C // 4))
        assert same(x[r:r + 1].contiguous(), ref), r


def test_replays_draw_by_the_device_words(gpu):
    """A captured call: the seed and offset of the moment, added to the call's offset."""
    import gdn2_amd as G

    x = torch.randn(33, 250, device=gpu)
    rng = torch.tensor([5, 0], dtype=torch.int64, device=gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        G.dropout(x, 0.4, 0, 17, rng=rng)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = G.dropout(x, 0.4, 0, 17, rng=rng)
    for seed, offset in ((5, 0), (5, 1000), (-3, 2 ** 40), (5, 0)):
        rng.copy_(torch.tensor([seed, offset]))
        graph.replay()
        torch.cuda.synchronize()
        assert same(y, want(x.cpu(), 0.4, seed, offset + 17))
        assert torch.equal(y, G.dropout(x, 0.4, seed, offset + 17))
