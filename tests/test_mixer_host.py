"""The mixer operators without a GPU: their 64-bit forms against differences,
and what they refuse."""
import ctypes
import os
import re
import subprocess
import sys

import numpy as np
import pytest

import mixer_testutil as M


@pytest.mark.parametrize("bounds", [None, [0, 3, 3, 7], [1, 4, 6]])
@pytest.mark.parametrize("w", [False, True])
def test_scan_gradients_against_differences(bounds, w):
    """The plain backward against central differences of the plain forward."""
    r = np.random.default_rng(3)
    B, T, C = (1, 7, 2) if bounds else (2, 7, 2)
    N = len(bounds) - 1 if bounds else B
    x = {"g": -r.uniform(0.01, 1.5, (B, T, C)), "v": r.standard_normal((B, T, C)), "w": r.standard_normal((B, T, C)),
         "h0": r.standard_normal((N, C))}
    dy, ds = r.standard_normal((B, T, C)), r.standard_normal((N, C))

    def loss(y):
        h, last, _, _ = M.scan64(y["g"], y["v"] * (y["w"] if w else 1), y["h0"], bounds)
        return np.nansum(h * dy) + (last * ds).sum()

    h = M.scan64(x["g"], x["v"] * (x["w"] if w else 1), x["h0"], bounds)[0]
    got, _ = M.scan_bwd64(x["g"], x["v"], x["w"] if w else None, h, dy, x["h0"], ds, bounds)
    for name, key in (("g", "dg"), ("v", "dv"), ("w", "dw"), ("h0", "dS0")):
        if name == "w" and not w:
            continue
        for i in np.ndindex(x[name].shape):
            up, down = dict(x, **{name: x[name].copy()}), dict(x, **{name: x[name].copy()})
            up[name][i] += 1e-6
            down[name][i] -= 1e-6
            d = (loss(up) - loss(down)) / 2e-6
            assert abs(d - got[key][i]) <= 1e-7 * (1 + abs(d)), (name, i)


def _scan_struct(**kw):
    from gdn2_amd import _capi as C

    a = C.GatedScanArgs()
    for k, v in dict(g=256, v=256, out=256, batch=1, num_heads=2, seq_len=4, head_v_dim=8).items():
        setattr(a, k, v)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_scan_refusals_of_the_c_entry():
    """Invalid arguments come back as a status with a message, before any launch."""
    from gdn2_amd import _capi as C

    L = C.lib()
    for fn in (L.gdn2_gated_scan_fwd_f32, L.gdn2_gated_scan_fwd_bf16):
        assert fn(None, None) == C.GDN2_EINVAL
        for bad in (dict(batch=-1), dict(seq_len=-1), dict(g=None), dict(v=None), dict(out=None),
                    dict(cu_seqlens=256, num_seqs=2, batch=2), dict(num_seqs=-1), dict(seq_len=5000),
                    dict(seq_len=5000, workspace=256, workspace_bytes=8),
                    dict(seq_len=5000, workspace=264, workspace_bytes=1 << 40),
                    dict(cu_seqlens=256, num_seqs=2)):
            assert fn(ctypes.byref(_scan_struct(**bad)), None) == C.GDN2_EINVAL, bad
            assert b"gdn2_gated_scan_fwd" in L.gdn2_last_error()
        for big in (dict(seq_len=1 << 30), dict(num_heads=1 << 30), dict(head_v_dim=1 << 20, num_heads=1 << 20),
                    dict(batch=1 << 29, head_v_dim=1 << 10), dict(batch=1 << 20, seq_len=1 << 20)):
            assert fn(ctypes.byref(_scan_struct(**big)), None) == C.GDN2_NOT_APPLICABLE, big
        for nothing in (dict(batch=0), dict(num_heads=0), dict(head_v_dim=0), dict(cu_seqlens=256, num_seqs=0)):
            assert fn(ctypes.byref(_scan_struct(**nothing)), None) == C.GDN2_OK, nothing
    for fn in (L.gdn2_gated_scan_bwd_f32, L.gdn2_gated_scan_bwd_bf16):
        assert fn(None, None) == C.GDN2_EINVAL
        b = C.GatedScanBwdArgs(_scan_struct(), 256, None, 256, 256, None, None, None, 0)
        b.fwd.w = 256  # dw missing
        assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL
        b.fwd.w, b.dw = None, 256  # dw without w
        assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL
        b.dw, b.dv = None, None
        assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL
        b.dv, b.fwd.seq_len = 256, 5000  # workspace missing
        assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL


def test_scan_workspace_sizes():
    from gdn2_amd import _capi as C

    size = lambda **kw: C.lib().gdn2_gated_scan_workspace_bytes(ctypes.byref(_scan_struct(**kw)))  # noqa: E731
    assert size(seq_len=1) == size(seq_len=8) == size(seq_len=0) == size(batch=0) == size(batch=-1) == 0
    assert C.lib().gdn2_gated_scan_workspace_bytes(None) == 0 and C.lib().gdn2_gated_scan_bwd_workspace_bytes(None) == 0
    assert 0 < size(seq_len=5000) <= 4 * 5000 * 16  # less than one operand
    assert size(seq_len=5, cu_seqlens=256, num_seqs=1) >= 4 * 7


def test_scan_refusals_in_python():
    torch = pytest.importorskip("torch")
    import gdn2_amd as G

    v = torch.zeros(2, 3, 5, 8)
    g1 = torch.zeros(2, 3, 5, 1)
    st = torch.zeros(2, 3, 8)
    cu = torch.tensor([0, 5], dtype=torch.int32)
    for err, args, kw in [
        (TypeError, (v, v), {}),  # not on a device
        (TypeError, (v, v.half()), {}), (TypeError, (v.bfloat16(), v.bfloat16()), {}),
        (ValueError, (v, v[0]), {}), (ValueError, (v[:, :, :4], v), {}), (ValueError, (torch.zeros(2, 3, 5, 2), v), {}),
        (TypeError, (g1, v, v.bfloat16()), {}), (ValueError, (g1, v, v[:1]), {}),
        (ValueError, (g1, v, None, st[:1]), {}), (TypeError, (g1, v, None, st.double()), {}),
        (ValueError, (g1, v, None, None, cu), {}), (TypeError, (g1[:1], v[:1], None, None, cu.long()), {}),
        (ValueError, (g1[:1], v[:1], None, st, cu), {}), (ValueError, (g1[:1], v[:1], None, None, cu[:0]), {}),
        (ValueError, (g1, v), {"out": v[:1]}), (TypeError, (g1, v), {"out": v.bfloat16()}),
        (ValueError, (g1, v), {"new_state": st[:1]}),
    ]:
        with pytest.raises(err):
            G.gated_scan(*args, **kw)
    for err, args, kw in [(TypeError, (g1, v, None, v, v), {}), (ValueError, (g1, v, None, v[:1], v), {}),
                          (TypeError, (g1, v, None, v, v.bfloat16()), {}),
                          (ValueError, (g1, v, None, v, v), {"d_state": st[:1]})]:
        with pytest.raises(err):
            G.gated_scan_backward(*args, **kw)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("gate", [False, True])
def test_norm_gradients_against_differences(act, gate):
    """The plain backward against central differences of the plain forward."""
    r = np.random.default_rng(4)
    N, S, C, groups = 2, 3, 6, 2
    x = {"x": r.standard_normal((N, S, C)), "weight": r.uniform(0.5, 1.5, C), "bias": r.standard_normal(C),
         "gate": r.standard_normal((N, S, C))}
    dy = r.standard_normal((N, S, C))

    def run(y):
        return M.norm64(y["x"], groups, y["weight"], y["bias"], 1e-5, act, y["gate"] if gate else None)

    got, _ = M.norm_bwd64(x["x"], groups, x["weight"], x["bias"], act, x["gate"] if gate else None, run(x)["stats"], dy)
    for name in ("x", "weight", "bias") + (("gate",) if gate else ()):
        for i in np.ndindex(x[name].shape):
            up, down = dict(x, **{name: x[name].copy()}), dict(x, **{name: x[name].copy()})
            up[name][i] += 1e-5
            down[name][i] -= 1e-5
            d = ((run(up)["y"] - run(down)["y"]) * dy).sum() / 2e-5
            assert abs(d - got["d" + name][i]) <= 1e-7 * (1 + abs(d)), (name, i)


def _norm_struct(**kw):
    from gdn2_amd import _capi as C

    a = C.GroupNormArgs()
    for k, v in dict(x=256, y=256, samples=2, rows=9000, channels=8, groups=2, eps=1e-5, activation=1, workspace=256,
                     workspace_bytes=1 << 40).items():
        setattr(a, k, v)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_norm_refusals_of_the_c_entry():
    from gdn2_amd import _capi as C

    L = C.lib()
    for fn in (L.gdn2_group_norm_act_f32, L.gdn2_group_norm_act_bf16):
        assert fn(None, None) == C.GDN2_EINVAL
        for bad in (dict(samples=-1), dict(rows=-1), dict(channels=-8), dict(groups=3), dict(groups=0), dict(x=None),
                    dict(y=None), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(activation=3),
                    dict(activation=-1), dict(workspace=None), dict(workspace_bytes=8), dict(workspace=264)):
            assert fn(ctypes.byref(_norm_struct(**bad)), None) == C.GDN2_EINVAL, bad
            assert b"gdn2_group_norm_act" in L.gdn2_last_error()
        for big in (dict(samples=1 << 24), dict(rows=1 << 30), dict(channels=1 << 24), dict(samples=1 << 20, groups=8, channels=8 * 4, rows=1) | dict(samples=1 << 22)):
            assert fn(ctypes.byref(_norm_struct(**big)), None) == C.GDN2_NOT_APPLICABLE, big
        for nothing in (dict(samples=0), dict(rows=0), dict(channels=0)):
            assert fn(ctypes.byref(_norm_struct(**nothing)), None) == C.GDN2_OK, nothing
    for fn in (L.gdn2_group_norm_act_bwd_f32, L.gdn2_group_norm_act_bwd_bf16):
        assert fn(None, None) == C.GDN2_EINVAL
        for bad in (dict(stats=None), dict(x=None), dict(gate=256), dict(activation=9)):
            b = C.GroupNormBwdArgs(_norm_struct(**{"stats": 256, **bad}), 256, 256, None, None, None, 256, 1 << 40)
            assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL, bad
        for bad in (dict(d_y=None), dict(dx=None), dict(dgate=256), dict(workspace=None), dict(workspace_bytes=8)):
            b = C.GroupNormBwdArgs(_norm_struct(stats=256), 256, 256, None, None, None, 256, 1 << 40)
            for k, v in bad.items():
                setattr(b, k, v)
            assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL, bad


def test_norm_workspace_sizes():
    from gdn2_amd import _capi as C

    size = lambda **kw: C.lib().gdn2_group_norm_act_workspace_bytes(ctypes.byref(_norm_struct(**kw)))  # noqa: E731
    assert size(rows=1, channels=2048, groups=16) == size(samples=0) == size(groups=3) == 0
    assert 0 < size(samples=8, rows=4096, channels=1024, groups=32) < 8 * 4096 * 1024
    assert C.lib().gdn2_group_norm_act_workspace_bytes(None) == 0
    assert C.lib().gdn2_group_norm_act_bwd_workspace_bytes(None) == 0


def test_norm_refusals_in_python():
    torch = pytest.importorskip("torch")
    import gdn2_amd as G

    x, w, st = torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(2, 2, 2)
    for err, args, kw in [
        (TypeError, (x, 2), {}),  # not on a device
        (TypeError, (x.half(), 2), {}), (ValueError, (x[0, 0], 2), {}), (ValueError, (x, 3), {}), (ValueError, (x, 0), {}),
        (ValueError, (x, 2, w[:4]), {}), (TypeError, (x, 2, w.double()), {}), (ValueError, (x, 2, w, w[:4]), {}),
        (ValueError, (x, 2), {"activation": "relu"}), (ValueError, (x, 2), {"gate": x[:1]}),
        (TypeError, (x, 2), {"gate": x.bfloat16()}), (ValueError, (x, 2), {"out": x[:1]}),
    ]:
        with pytest.raises(err):
            G.group_norm_act(*args, **kw)
    for err, args in [(TypeError, (x, 2, st, x)), (ValueError, (x, 2, st[:1], x)), (TypeError, (x, 2, st.double(), x)),
                      (ValueError, (x, 2, st, x[:1])), (TypeError, (x, 2, st, x.bfloat16()))]:
        with pytest.raises(err):
            G.group_norm_act_backward(*args)


@pytest.mark.parametrize("T,cache", [(1, False), (2, True), (5, False), (6, True)])
def test_conv_gradients_against_differences(T, cache):
    r = np.random.default_rng(5)
    B, C = 2, 3
    x = {"x": r.standard_normal((B, T, C)), "weight": r.uniform(-0.5, 0.5, (C, 4)), "cache": r.standard_normal((B, 3, C))}
    dy, dc = r.standard_normal((B, T, C)), r.standard_normal((B, 3, C))

    def loss(y):
        out, new, _, _ = M.conv64(y["x"], y["weight"], y["cache"] if cache else None)
        return (out * dy).sum() + (new * dc).sum()

    got, _ = M.conv_bwd64(x["x"], x["weight"], x["cache"] if cache else None, dy, dc)
    for name in ("x", "weight") + (("cache",) if cache else ()):
        for i in np.ndindex(x[name].shape):
            up, down = dict(x, **{name: x[name].copy()}), dict(x, **{name: x[name].copy()})
            up[name][i] += 1e-6
            down[name][i] -= 1e-6
            d = (loss(up) - loss(down)) / 2e-6
            assert abs(d - got["d" + name][i]) <= 1e-7 * (1 + abs(d)), (name, i)


def test_conv_refusals():
    torch = pytest.importorskip("torch")
    import gdn2_amd as G
    from gdn2_amd import _capi as C

    L = C.lib()
    ok = dict(x=256, w=256, cache=None, dy=256, dc=None, dx=1 << 20, dw=256, dci=None, B=2, T=5, C=8, ws=256, n=1 << 40)
    call = lambda **kw: L.gdn2_short_conv_bwd_f32(*{**ok, **kw}.values(), None)  # noqa: E731
    for bad in (dict(B=-1), dict(T=-1), dict(C=-1), dict(x=None), dict(w=None), dict(dy=None), dict(dx=None), dict(dw=None),
                dict(dci=256), dict(ws=None), dict(n=8), dict(ws=264), dict(dx=256), dict(dx=260)):
        assert call(**bad) == C.GDN2_EINVAL, bad
        assert b"gdn2_short_conv_bwd_f32" in L.gdn2_last_error()
    for big in (dict(C=1 << 22), dict(B=1 << 24), dict(T=1 << 30)):
        assert call(**big) == C.GDN2_NOT_APPLICABLE, big
    assert call(C=0) == C.GDN2_OK
    size = L.gdn2_short_conv_bwd_workspace_bytes
    assert size(0, 5, 8) == size(2, 0, 8) == size(2, 5, 0) == size(-1, 5, 8) == 0 and size(2, 5, 8) > 0
    x, w, c = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(2, 3, 8)
    for err, args, kw in [(TypeError, (x, w, x), {}), (ValueError, (x, w[:4], x), {}), (ValueError, (x, w, x[:1]), {}),
                          (ValueError, (x, w, x, c[:1]), {}), (ValueError, (x[0], w, x), {}),
                          (ValueError, (x, w, x), {"d_cache": c[:, :2]})]:
        with pytest.raises(err):
            G.short_conv_1d_backward(*args, **kw)


def test_operands_that_are_one_another():
    """A result that is an input, where that is not allowed, comes back as EINVAL."""
    from gdn2_amd import _capi as C

    L = C.lib()
    ptr = dict(g=1 << 20, v=2 << 20, w=3 << 20, out=4 << 20)
    for fn in (L.gdn2_gated_scan_fwd_f32, L.gdn2_gated_scan_fwd_bf16):
        for name in "gvw":
            assert fn(ctypes.byref(_scan_struct(**{**ptr, "out": ptr[name]})), None) == C.GDN2_EINVAL, name
            assert b"out must not be" in L.gdn2_last_error()
    for fn in (L.gdn2_gated_scan_bwd_f32, L.gdn2_gated_scan_bwd_bf16):
        for name in ("dg", "dv", "dw"):
            for to in (*ptr.values(), 5 << 20):
                b = C.GatedScanBwdArgs(_scan_struct(**ptr), 5 << 20, None, 6 << 20, 7 << 20, 8 << 20, None, None, 0)
                setattr(b, name, to)
                assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL, (name, to)
                assert b"must not be inputs" in L.gdn2_last_error()
    for fn in (L.gdn2_group_norm_act_f32, L.gdn2_group_norm_act_bf16):
        a = _norm_struct(x=1 << 20, y=2 << 20, gate=2 << 20, stride_x_n=72000, stride_x_s=8, stride_gate_n=144000, stride_gate_s=16)
        assert fn(ctypes.byref(a), None) == C.GDN2_EINVAL and b"strides" in L.gdn2_last_error()
    norm = dict(x=1 << 20, gate=2 << 20, stats=256)
    for fn in (L.gdn2_group_norm_act_bwd_f32, L.gdn2_group_norm_act_bwd_bf16):
        for name, to in (("dx", 1), ("dx", 2), ("dx", 5), ("dgate", 1), ("dgate", 2), ("dgate", 3), ("dgate", 4)):
            b = C.GroupNormBwdArgs(_norm_struct(**norm), 3 << 20, 4 << 20, 5 << 20, None, None, 256, 1 << 40)
            setattr(b, name, to << 20)
            assert fn(ctypes.byref(b), None) == C.GDN2_EINVAL and b"must not be" in L.gdn2_last_error(), (name, to)
    conv = lambda dci, dc: L.gdn2_short_conv_bwd_f32(1 << 20, 256, 2 << 20, 3 << 20, dc, 4 << 20, 256, dci, 2, 5, 8, 256, 1 << 40, None)  # noqa: E731
    for dci, dc in ((2 << 20, None), ((2 << 20) + 16, None), (5 << 20, 5 << 20), ((5 << 20) - 16, 5 << 20)):
        assert conv(dci, dc) == C.GDN2_EINVAL and b"d_cache_in" in L.gdn2_last_error()


def test_layouts_of_results():
    """Results never share memory between elements; no elements have a shape."""
    torch = pytest.importorskip("torch")
    from gdn2_amd import mixer

    one = torch.zeros(1, 2, 3, 4)
    wide = one.expand(5, 2, 3, 4)
    assert mixer._dense_rows(wide) is not wide and mixer._dense_rows(wide).is_contiguous()
    gaps = torch.zeros(5, 2, 3, 8)[..., :4]
    assert mixer._dense_rows(gaps) is gaps and mixer._empty_like(gaps).stride() == gaps.stride()
    assert mixer._rows(torch.zeros(0, 3, 5, 8)).shape == (0, 15, 8)
    assert mixer._rows(torch.zeros(2, 0, 5, 8)).shape == (2, 0, 8)
    assert mixer._rows(torch.zeros(2, 3, 5, 0)).shape == (2, 15, 0)


@pytest.mark.parametrize("source", ["gated_scan", "group_norm", "short_conv_bwd"])
def test_no_kernel_keeps_registers_in_memory(source, tmp_path):
    """What the forms of the kernels were chosen by (see FormOf in gated_scan.hip)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "burn-gdn2_amd"))
    import build

    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    flags = [f for f in build.FLAGS if f != "-shared"]
    r = subprocess.run([build.HIPCC, *flags, "--offload-device-only", "-Rpass-analysis=kernel-resource-usage", "-c",
                        os.path.join(root, "burn-gdn2_amd", "csrc", source + ".hip"), "-o", str(tmp_path / "device.o")],
                       capture_output=True, text=True, check=True)
    names = re.findall(r"Function Name: (\S+)", r.stderr)
    scratch = [int(n) for n in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)]
    assert names and len(names) == len(scratch)
    assert not [n for n, size in zip(names, scratch) if size]
