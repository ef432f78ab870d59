"""gated_scan and gated_scan_backward over chains of wide tiles that are longer than
one look: more than four chains, more than eight tiles each (fewer chains take narrow
tiles).  The sizes where that matters most are those of full prompts."""
import pytest

import test_gpu_gated_scan as S

pytestmark = pytest.mark.gpu

# B, T, H, V: tiles of 64 to 256 tokens by 128 channels (64 where V is a multiple of 4
# alone in 16 bits, 32 where it is odd), so 12 to 47 of them a chain
CHAINS = [(5, 3000, 2, 128), (1, 3000, 10, 132), (6, 1100, 1, 33)]


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,H,V", CHAINS)
def test_both_ways(gpu, B, T, H, V, ty):
    import torch

    import gdn2_amd as G

    for k, (per_head, w, state) in enumerate([(False, True, True), (True, True, False), (False, False, False), (True, False, True)]):
        print("chains", B, T, H, V, ty, per_head, w, state, flush=True)
        d = S._make(gpu, 1000 + T + k, B, T, H, V, ty, per_head, w, state, slow=k < 2)
        out, new = G.gated_scan(**d)
        torch.cuda.synchronize()
        assert S._check_forward(d, out, new, B, ty).all()
        d_out = torch.randn(B, T, H, V, device=gpu).to(S._types(ty)).transpose(1, 2)
        d_state = torch.randn(B, H, V, device=gpu) if state else None
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=d_state)
        torch.cuda.synchronize()
        S._check_backward(d, out, d_out, d_state, r, B, ty)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("per_head", [False, True])
def test_packed(gpu, per_head, ty):
    """One row, six and more chains: a sequence over all tiles but a few, short ones
    before and behind it, empty ones, and rows of no sequence at both ends."""
    import torch

    import gdn2_amd as G

    T, H, V = 4200, 6, 128
    bounds = [3, 20, 20, 90, 3900, 3901, 4150]
    N = len(bounds) - 1
    cu = torch.tensor(bounds, dtype=torch.int32, device=gpu)
    d = S._make(gpu, 77, 1, T, H, V, ty, per_head, True, True, N=N, slow=True)
    out = torch.full((1, T, H, V), 7.0, device=gpu, dtype=S._types(ty)).transpose(1, 2)
    out, new = G.gated_scan(**d, cu_seqlens=cu, out=out)
    torch.cuda.synchronize()
    inside = S._check_forward(d, out, new, N, ty, bounds)
    assert (S._flat(out)[~inside] == 7.0).all()
    d_out, d_state = torch.randn_like(out), torch.randn_like(new)
    r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=d_state, cu_seqlens=cu)
    torch.cuda.synchronize()
    S._check_backward(d, out, d_out, d_state, r, N, ty, bounds)


@pytest.mark.parametrize("ty,per_head", [("f32", False), ("bf16", True), ("bf16", False)])
def test_same_bits_every_time(gpu, ty, per_head):
    """79 to 313 tiles a chain, 16 chains and more, with and without other work on
    the device: one order of joins whatever their timing."""
    import torch

    import gdn2_amd as G

    d = S._make(gpu, 9, 1, 20000, 16, 128, ty, per_head, True, True, slow=True)
    out, new = G.gated_scan(**d)
    d_out = torch.randn_like(out)
    first = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=new)
    side, a = torch.cuda.Stream(), torch.randn(4096, 4096, device=gpu)
    for i in range(6):
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(4):
                    a = torch.tanh(a)
        o, s = G.gated_scan(**d)
        r = G.gated_scan_backward(d["g"], d["v"], d["w"], out, d_out, d["state"], d_state=new)
        torch.cuda.synchronize()
        assert torch.equal(o, out) and torch.equal(s, new)
        assert all(torch.equal(r[n], first[n]) for n in first)


def test_what_is_not_finite_along_a_chain(gpu):
    """An infinite state and a NaN one over 47 tiles of two joining waves, and a decay
    of zero half way."""
    import torch

    import gdn2_amd as G

    T, V = 3000, 128
    d = S._make(gpu, 5, 5, T, 2, V, "f32", False, True, True, slow=True)
    d["state"][:, :, 1::2], d["state"][:, :, 2::4] = float("inf"), float("nan")
    d["g"][:, :, 1500, ::3] = float("-inf")
    out, new = G.gated_scan(**d)
    torch.cuda.synchronize()
    o, s = out.cpu(), new.cpu()
    for c in range(V):
        due = torch.isinf if c % 2 else torch.isnan if c % 4 == 2 else torch.isfinite
        end = 1500 if c % 3 == 0 else T
        assert due(o[:, :, :end, c]).all() and torch.isfinite(o[:, :, end:, c]).all(), c
        assert (torch.isfinite if c % 3 == 0 else due)(s[:, :, c]).all(), c
