"""Sums of group_norm_act and its backward where ordinary f32 ones would lose digits:
a value far from all others, very many rows, terms of one sign."""
import pytest

import mixer_testutil as M

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _stats64(x, groups):
    """[N, groups] mean and variance in 64 bits."""
    import torch

    N, S, C = x.shape
    r = x.double().view(N, S, groups, C // groups)
    return torch.var_mean(r, (1, 3), unbiased=False)


@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("N,S,C,groups", [(6, 1, 512, 2), (3, 40, 64, 4), (2, 4096, 64, 2), (2, 700, 33, 1), (1, 600, 1500, 1),
                                          (2, 90, 500, 2), (1, 200000, 64, 2), (1, 50000, 2048, 1)])
def test_one_value_far_from_the_others(gpu, N, S, C, groups, ty, at):
    """One value of a group is 10^4 standard deviations off, as a sequence's first token
    may be.  The group's mean and variance keep their digits: moments about a value
    are not taken about that one at the cost of the others'.  Tolerance: a sum's SUM
    roundings, of the variance and, for the mean, of the mean magnitude."""
    import torch

    import gdn2_amd as G

    x = torch.randn(N, S, C, generator=torch.Generator(device=gpu).manual_seed(S + C), device=gpu)
    row, col = {"first": (0, 0), "middle": (S // 2, C // groups // 2), "last": (S - 1, C // groups - 1)}[at]
    x[:, row, col::C // groups] += 1e4
    x = x.to({"f32": torch.float32, "bf16": torch.bfloat16}[ty])
    y, stats = G.group_norm_act(x, groups, eps=EPS, activation="none", return_stats=True)
    torch.cuda.synchronize()
    var, mean = _stats64(x, groups)
    size = x.double().abs().view(N, S, groups, C // groups).mean((1, 3))
    assert ((stats[..., 0] - mean).abs() <= M.SUM * M.EPS * size).all()
    rel = (stats[..., 1].double() * torch.sqrt(var + EPS) - 1).abs().max().item()
    print("rstd off by", rel, flush=True)
    assert rel <= M.SUM * M.EPS, rel
