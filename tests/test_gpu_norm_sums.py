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


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("N,S,C,groups", [(6, 1, 512, 2), (2, 50, 64, 4), (2, 4096, 64, 2), (8, 1000, 1024, 32), (1, 700, 33, 1),
                                          (1, 600, 1500, 1), (1, 50000, 2048, 1), (1, 200000, 64, 2)])
def test_large_means(gpu, N, S, C, groups, inplace):
    """Values around 1000 that differ by 0.01, and constants: the mean is right to the
    last digit that f32 has for it, and the variance of the values about it too.
    Tolerance, of the mean: a step of 1000, 2^-14 (half of one is its own rounding).
    Of the variance: those of the means m_r that are joined, off by d_r of half a step
    at most, sum n_r (m_r + d_r - m)^2 / n - sum n_r (m_r - m)^2 / n
    <= 2 (step / 2) sum n_r |m_r - m| / n + step^2 / 4 <= step sd + step^2 / 4 (the mean
    magnitude of m_r - m is at most its root mean square, and that at most sd); and
    SUM roundings.  Groups of one row sum the values themselves: their mean is off by
    SUM roundings of 1000, as in test_gpu_group_norm's test_large_mean, and the variance
    by the square of that."""
    import torch

    import gdn2_amd as G

    step = 2.0 ** -14  # of values from 512 to 1024 (x stays below)
    for spread in (0.0, 0.01):
        r = torch.Generator(device=gpu).manual_seed(S + C)
        x = 1000.1 + spread * torch.randn(N, S, C, generator=r, device=gpu).clamp(-5, 5)
        var, mean = _stats64(x, groups)
        y, stats = G.group_norm_act(x, groups, eps=EPS, activation="none", return_stats=True, out=x if inplace else None)
        torch.cuda.synchronize()
        off = (stats[..., 0] - mean).abs().max().item()
        rel = (stats[..., 1].double() * torch.sqrt(var + EPS) - 1).abs().max().item()
        print("mean off by", off / step, "steps, rstd by", rel, flush=True)
        far = step if S > 1 else M.SUM * M.EPS * 1001
        assert off <= far
        extra = step * var.sqrt() + step ** 2 / 4 if S > 1 else far ** 2
        bound = 0.5 * (extra / (var + EPS)).max().item() + M.SUM * M.EPS
        assert rel <= bound, (rel, bound)


# Sums of one sign: a serial f32 sum of n equal terms is off by up to n / 4 half steps
# (its partial sums' roundings are all the same way within a power of two), one in
# pieces by its longest chain's.  SUM_TERMS as in M.norm_bwd64; the terms are constants
# whose sums f32 does not hold.
SUM_TERMS = 200


@pytest.mark.parametrize("N,S,C,groups", [(1 << 22, 1, 64, 1), (1 << 20, 4, 16, 1), (1, 100000, 2048, 1), (1, 1 << 22, 32, 1)])
def test_gradients_of_weights_over_very_many_rows(gpu, N, S, C, groups):
    """A loss that is a mean: d_out the same everywhere."""
    import torch

    import gdn2_amd as G

    r = torch.Generator(device=gpu).manual_seed(3)
    x = torch.randn(N, S, C, generator=r, device=gpu)
    y, stats = G.group_norm_act(x, groups, eps=EPS, activation="none", return_stats=True)
    del y
    dy = torch.tensor(0.1, device=gpu).expand(C).contiguous().expand(N, S, C)
    g = G.group_norm_act_backward(x, groups, stats, dy, activation="none")
    torch.cuda.synchronize()
    c = float(torch.tensor(0.1))
    off = (g["dbias"].double() / (N * S * c) - 1).abs().max().item()
    print("dbias off by", off / M.EPS, "half steps", flush=True)
    assert off <= SUM_TERMS * M.EPS, off / M.EPS
    # dn is the same everywhere: what is left of it, dn - mean(dn) - n mean(dn n), are roundings
    n = C // groups * S
    mean_n = (SUM_TERMS + 8) * M.EPS  # mean(n) is zero but for the statistics' roundings, of mean |n| < 1
    left = g["dx"].abs().max().item()
    bound = stats[..., 1].max().item() * c * ((SUM_TERMS + 8) * M.EPS + 7 * (mean_n + SUM_TERMS * M.EPS))  # (|n| < 7)
    print("dx", left, "of", bound, n, flush=True)
    assert left <= bound, (left, bound)


def test_gradients_of_conv_weights_over_very_many_tokens(gpu):
    import torch

    import gdn2_amd as G

    T, C = 1 << 22, 16
    x, w = torch.full((1, T, C), 0.7, device=gpu), torch.full((C, 4), 0.1, device=gpu)
    r = G.short_conv_1d_backward(x, w, torch.full_like(x, 0.1))
    torch.cuda.synchronize()
    a, d = float(torch.tensor(0.7)), float(torch.tensor(0.1))
    z = 4 * a * d
    s = 1 / (1 + 2.718281828459045 ** -z)
    want = T * d * s * (1 + z * (1 - s)) * a
    off = (r["dweight"].double() / want - 1).abs().max().item()
    print("dweight off by", off / M.EPS, "half steps", flush=True)
    assert off <= 120 * M.EPS, off / M.EPS  # (as M.conv_bwd64; the terms' own few roundings among them)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("N,S,C,groups", [(1, 9000, 520, 1), (1, 9000, 521, 1), (2, 5000, 1040, 2), (1, 300, 33000, 1),
                                          (1, 40000, 64, 1)])
def test_large_groups(gpu, N, S, C, groups, ty):
    """Groups whose chunks of rows are joined in several spans, one of them shorter."""
    import test_gpu_group_norm as B

    import gdn2_amd as G

    for act, gate in (("silu", True), ("gelu", False)):
        d, dy = B._make(gpu, C + S, N, S, C, ty, gate)
        y, stats = G.group_norm_act(d["x"], groups, d["weight"], d["bias"], EPS, act, gate=d["gate"], return_stats=True)
        B._check_forward(d, groups, act, y, stats, ty)
        r = G.group_norm_act_backward(d["x"], groups, stats, dy, d["weight"], d["bias"], act, gate=d["gate"])
        B._check_backward(d, groups, act, stats, dy, r, ty)
