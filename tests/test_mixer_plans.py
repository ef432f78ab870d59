"""What the mixer operators plan for a call, without a GPU."""
import ctypes

import pytest


@pytest.mark.parametrize("S,C,groups,tiles", [(32768, 512, 1, 2), (50000, 2048, 1, 8), (20000, 16384, 1, 64), (20000, 1024, 1, 4)])
def test_large_groups_are_spread_over_the_device(S, C, groups, tiles):
    """A group in three passes is read by 512 workgroups or more, two a compute unit,
    whatever its channels (the workspace holds a pair for each chunk of rows and
    channel)."""
    from gdn2_amd import _capi as C_

    a = C_.GroupNormArgs()
    for k, v in dict(x=256, y=256, samples=1, rows=S, channels=C, groups=groups, eps=1e-5, activation=1, stride_x_n=S * C,
                     stride_x_s=C).items():
        setattr(a, k, v)
    for size in (C_.lib().gdn2_group_norm_act_workspace_bytes(ctypes.byref(a)),
                 C_.lib().gdn2_group_norm_act_bwd_workspace_bytes(ctypes.byref(C_.GroupNormBwdArgs(a)))):
        chunks = size // (8 * C)
        assert 500 <= chunks * tiles <= 4096, chunks


def test_strides_of_one_element_do_not_count():
    """A dimension of one has no stride to speak of: at T = 1 the v that a projection
    leaves, [B, 1, H, V] seen as [B, H, 1, V], and a contiguous w are laid out alike, and
    a decoding step copies neither."""
    torch = pytest.importorskip("torch")
    from gdn2_amd import mixer

    v, w = torch.zeros(2, 1, 16, 128).transpose(1, 2), torch.zeros(2, 16, 1, 128)
    assert v.stride() != w.stride()
    assert mixer._in_layout(w, v) is w and mixer._in_layout(v, w) is v
    one = torch.zeros(1, 7, 64)
    assert mixer._in_layout(torch.zeros(9, 7, 64)[:1], one) is not one  # (equal strides, another tensor)
    odd = torch.empty_strided((1, 7, 64), (12345, 64, 1))
    assert mixer._in_layout(odd, one) is odd
    other = torch.zeros(2, 64, 7).transpose(1, 2)
    assert mixer._in_layout(other, torch.zeros(2, 7, 64)) is not other


def test_imports_without_torchs_private_names():
    """A torch built without a GPU lacks some; the package imports all the same."""
    import os
    import subprocess
    import sys

    pytest.importorskip("torch")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys; sys.path.insert(0, 'burn-gdn2_amd')\n"
            "import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, n)\n"
            "import gdn2_amd\n"
            "assert gdn2_amd.gated_scan")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_few_tokens_need_no_workspace():
    """Up to mixer._WALK tokens the Python entry asks for none, at any size."""
    from gdn2_amd import _capi as C, mixer

    for T in (1, mixer._WALK, mixer._WALK + 1):
        for B, H, V in ((1, 1, 1), (1, 16, 128), (64, 16, 128), (300, 16, 131)):
            a = C.GatedScanArgs()
            for k, v in dict(g=256, v=256, out=256, batch=B, num_heads=H, seq_len=T, head_v_dim=V).items():
                setattr(a, k, v)
            n = C.lib().gdn2_gated_scan_workspace_bytes(ctypes.byref(a))
            assert n == 0 or T > mixer._WALK
