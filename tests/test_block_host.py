"""The block operators without a GPU: their 64-bit forms against differences, the
generator against its published values, and what they refuse."""
import ctypes

import numpy as np
import pytest
import torch

import block_testutil as K


@pytest.mark.parametrize("c,key,want", [
    (0, 0, (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
    (0xFFFFFFFF, 2 ** 64 - 1, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662))])
def test_generator(c, key, want):
    """Seven rounds at counters and keys of zeros and of ones: the generator's published
    answers."""
    n = np.array([c], np.uint64)
    assert tuple(int(v) for v in K.philox(n, n, n, n, key)[0]) == want


def test_generator_shares():
    """Shares of dropped elements within five standard deviations, rows and neighbours
    unlike."""
    for p in (0.1, 0.5, 0.9):
        k = K.kept(256, 1000, p, 12345, 2 ** 40).double()
        assert abs(float(k.mean()) - (1 - p)) < 5 * (p * (1 - p) / k.numel()) ** 0.5
        for a, b in ((k[1:], k[:-1]), (k[:, 1:], k[:, :-1])):
            both = float((a * b).mean())
            assert abs(both - (1 - p) ** 2) < 6 * (1 / a.numel()) ** 0.5


@pytest.mark.parametrize("post,pre,gate,act,p", [(True, True, True, "silu", 0.3), (True, False, True, "sigmoid", 0.0),
                                                 (False, True, True, "none", 0.3), (True, True, False, "none", 0.0)])
def test_residual_gradients_against_differences(post, pre, gate, act, p):
    g = torch.Generator().manual_seed(5)
    M, C, alpha, sigma = 3, 7, 0.8, 0.5
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=K.F64)  # noqa: E731
    t = {"x": rnd(M, C), "y": rnd(M, C), "gate": rnd(M, C) if gate else None, "post": rnd(C) if post else None,
         "pre": rnd(C) if pre else None}
    dr, dn, factor = rnd(M, C), rnd(M, C), K.drop_factor(M, C, p, 9)

    def loss(t):
        (r, n, _), _ = K.residual64(t["x"], t["y"], t["gate"], t["post"], t["pre"], 1e-5, act, alpha, sigma, factor)
        return float((r * dr).sum() + ((n * dn).sum() if pre else 0))

    (r, _, stats), _ = K.residual64(t["x"], t["y"], t["gate"], t["post"], t["pre"], 1e-5, act, alpha, sigma, factor)
    got, _ = K.residual_bwd64(r, t["y"], t["gate"], t["post"], t["pre"], stats, dr, dn if pre else None, act, alpha, sigma, factor)
    for name, v in t.items():
        if v is None:
            assert "d" + name not in got
            continue
        for i in np.ndindex(*v.shape):
            lo, hi = dict(t, **{name: v.clone()}), dict(t, **{name: v.clone()})
            lo[name][i] -= 1e-6
            hi[name][i] += 1e-6
            d = (loss(hi) - loss(lo)) / 2e-6
            assert abs(d - float(got["d" + name][i])) <= 1e-7 * (1 + abs(d)), (name, i)


def test_dropout_refusals_of_the_c_entry():
    from gdn2_amd import _capi as C

    L = C.lib()
    ok = C.Dropout(0.5, 1, 0, None)
    for fn in (L.gdn2_dropout_f32, L.gdn2_dropout_bf16):
        assert fn(256, 512, 2, 8, 8, 8, None, None) == C.GDN2_EINVAL
        for p in (-0.1, 1.5, float("nan")):
            assert fn(256, 512, 2, 8, 8, 8, C.Dropout(p, 0, 0, None), None) == C.GDN2_EINVAL
        assert fn(None, 512, 2, 8, 8, 8, ok, None) == fn(256, None, 2, 8, 8, 8, ok, None) == C.GDN2_EINVAL
        assert fn(256, 512, -1, 8, 8, 8, ok, None) == fn(256, 512, 2, -8, 8, 8, ok, None) == C.GDN2_EINVAL
        assert fn(256, 256, 2, 8, 8, 16, ok, None) == C.GDN2_EINVAL  # in place with another stride
        assert b"gdn2_dropout" in L.gdn2_last_error()
        assert fn(256, 512, 0, 8, 8, 8, ok, None) == fn(None, None, 2, 0, 8, 8, ok, None) == C.GDN2_OK
        assert fn(256, 512, 1, 1 << 31, 8, 8, ok, None) == C.GDN2_NOT_APPLICABLE
        assert fn(256, 512, 1 << 33, 5, 5, 5, ok, None) == C.GDN2_NOT_APPLICABLE


def _res(**kw):
    from gdn2_amd import _capi as C

    a = C.ResidualNormArgs()
    for k, v in dict(dict(x=256, y=256, out=256, samples=2, rows=3, channels=8, eps=1e-5, residual_scale=1.0,
                          branch_scale=1.0), **kw).items():
        setattr(a, k, v)
    return a


def test_residual_refusals_of_the_c_entry():
    from gdn2_amd import _capi as C

    L = C.lib()
    for fn in (L.gdn2_residual_norm_f32, L.gdn2_residual_norm_bf16, L.gdn2_residual_norm_f32_bf16):
        assert fn(None, None) == C.GDN2_EINVAL
        for bad in (dict(samples=-1), dict(rows=-1), dict(channels=-1), dict(x=None), dict(out=None), dict(activation=3),
                    dict(activation=-1), dict(gate_rows=3), dict(eps=-1.0), dict(eps=float("nan")), dict(pre_weight=256),
                    dict(normed=256), dict(y=None, gate=256), dict(y=None, post_weight=256),
                    dict(dropout=C.Dropout(2.0, 0, 0, None)), dict(y=None, dropout=C.Dropout(0.1, 0, 0, None))):
            assert fn(_res(**bad), None) == C.GDN2_EINVAL, bad
            assert b"gdn2_residual_norm" in L.gdn2_last_error()
        for big in (dict(channels=8193), dict(samples=1 << 30), dict(samples=1 << 20, rows=1 << 20)):
            assert fn(_res(**big), None) == C.GDN2_NOT_APPLICABLE, big
        for nothing in (dict(samples=0), dict(rows=0), dict(channels=0)):
            assert fn(_res(**nothing), None) == C.GDN2_OK
    for fn in (L.gdn2_residual_norm_bwd_f32, L.gdn2_residual_norm_bwd_bf16, L.gdn2_residual_norm_bwd_f32_bf16):
        assert fn(None, None) == C.GDN2_EINVAL

        def bwd(fwd, **kw):
            b = C.ResidualNormBwdArgs()
            b.fwd = _res(stats=256, **fwd)
            for k, v in dict(dict(d_out=256, dx=256, dy=256), **kw).items():
                setattr(b, k, v)
            return fn(ctypes.byref(b), None)

        pre, post = dict(pre_weight=256), dict(post_weight=256)
        for fwd, kw in ((pre, {}), (pre, dict(dpre=256)), (pre, dict(d_normed=256)), ({}, dict(d_normed=256)), (post, {}),
                        ({}, dict(dpost=256)), (dict(gate=256), {}), ({}, dict(dgate=256)), ({}, dict(dy=None)),
                        (dict(y=None), {}), (dict(out=None, **pre), dict(dpre=256, d_normed=256)),
                        (pre, dict(dpre=256, d_normed=256)),  # workspace missing
                        (pre, dict(dpre=256, d_normed=256, workspace=256, workspace_bytes=8)),
                        (pre, dict(dpre=256, d_normed=256, workspace=264, workspace_bytes=1 << 30))):
            assert bwd(fwd, **kw) == C.GDN2_EINVAL, (fwd, kw)
        assert bwd(dict(channels=8193)) == C.GDN2_NOT_APPLICABLE
        assert bwd(dict(channels=0)) == C.GDN2_OK


def test_sizes_at_the_limits_of_the_c_entries():
    """Refused before anything runs, and no sooner than the header says (there the next
    check, of the workspace or a pointer, refuses)."""
    from gdn2_amd import _capi as C

    L = C.lib()
    for fn in (L.gdn2_residual_norm_bwd_f32, L.gdn2_residual_norm_bwd_bf16, L.gdn2_residual_norm_bwd_f32_bf16):

        def bwd(**kw):
            b = C.ResidualNormBwdArgs()
            b.fwd = _res(gate=256, **kw)
            b.d_out = b.dx = b.dy = b.dgate = 256
            return fn(ctypes.byref(b), None)

        one = dict(gate_rows=C.GATE_SAMPLE)
        assert bwd(samples=1 << 16, rows=2, channels=8192, **one) == C.GDN2_NOT_APPLICABLE
        assert bwd(samples=(1 << 15) - 1, rows=2, channels=8192, **one) == C.GDN2_EINVAL
        assert bwd(samples=1 << 22, rows=1, channels=64, **one) == C.GDN2_NOT_APPLICABLE
        assert bwd(samples=(1 << 21) - 1, rows=100, channels=64, **one) == C.GDN2_EINVAL
        assert bwd(samples=1, rows=1 << 29, channels=2048, gate_rows=C.GATE_ALL) == C.GDN2_NOT_APPLICABLE
        assert bwd(samples=1, rows=(1 << 28) - 1, channels=2048, gate_rows=C.GATE_ALL) == C.GDN2_EINVAL
    for fn in (L.gdn2_low_rank_add_f32, L.gdn2_low_rank_add_bf16):
        for rank in (16, 64):
            assert fn(_lora(batch=1 << 22, seq_len=1, rank=rank), None) == C.GDN2_NOT_APPLICABLE
            assert fn(_lora(batch=1 << 21, seq_len=33, rank=rank), None) == C.GDN2_NOT_APPLICABLE
        assert fn(_lora(batch=(1 << 20) - 1, seq_len=64, rank=128, out_features=1024, workspace=None), None) == C.GDN2_EINVAL
        assert fn(_lora(batch=1 << 20, seq_len=64, rank=128, out_features=4096, workspace=None), None) == C.GDN2_NOT_APPLICABLE


def test_residual_workspace_sizes():
    from gdn2_amd import _capi as C

    L = C.lib()

    def size(**kw):
        b = C.ResidualNormBwdArgs()
        b.fwd = _res(**kw)
        return L.gdn2_residual_norm_bwd_workspace_bytes(b)

    assert L.gdn2_residual_norm_bwd_workspace_bytes(None) == 0
    assert size() == size(pre_weight=256, rows=0) == size(pre_weight=256, channels=8193) == 0
    one = size(pre_weight=256, samples=8, rows=4096, channels=2048)
    assert one == 768 * 2048 * 4 and size(pre_weight=256, post_weight=256, samples=8, rows=4096, channels=2048) == 2 * one
    # no f32 sum over more than 128 rows
    assert size(pre_weight=256, samples=1, rows=1 << 20, channels=2048) == (1 << 13) * 2048 * 4
    # a gate a sample: at least a workgroup each
    assert size(gate=256, gate_rows=1, samples=5000, rows=2, channels=64) == 5000 * 64 * 4


def test_refusals_in_python():
    import gdn2_amd as G

    x, w = torch.zeros(2, 3, 8), torch.zeros(8)
    b = x.bfloat16()
    st = torch.zeros(2, 3, 2)
    for err, f, args, kw in [
        (TypeError, G.dropout, (x, 0.5), {}),  # not on a device
        (TypeError, G.dropout, (x.half(), 0.5), {}), (ValueError, G.dropout, (x, -0.1), {}), (ValueError, G.dropout, (x, 1.1), {}),
        (ValueError, G.dropout, (torch.zeros(()), 0.5), {}), (TypeError, G.dropout, (x, 0.5), dict(out=b)),
        (ValueError, G.dropout, (x, 0.5), dict(out=x[:1])), (TypeError, G.dropout, (x, 0.5), dict(rng=torch.zeros(2))),
        (ValueError, G.dropout, (x, 0.5), dict(out=torch.zeros(8).expand(2, 3, 8))),
        (ValueError, G.dropout, (torch.zeros(3, 8), 0.5), dict(out=torch.zeros(4, 8).as_strided((3, 8), (4, 1)))),
        (TypeError, G.dropout, (x, 0.5), dict(rng=torch.zeros(3, dtype=torch.int64))),
        (TypeError, G.residual_norm, (x, x), {}), (ValueError, G.residual_norm, (w, w), {}),
        (TypeError, G.residual_norm, (b, x), {}), (TypeError, G.residual_norm, (x.half(), x.half()), {}),
        (ValueError, G.residual_norm, (x, x[:1]), {}), (ValueError, G.residual_norm, (x, x), dict(activation="gelu")),
        (TypeError, G.residual_norm, (x, x, b), {}), (ValueError, G.residual_norm, (x, x, x[:, :2]), {}),
        (ValueError, G.residual_norm, (x, x, x[:1]), {}), (ValueError, G.residual_norm, (x, None, x), {}),
        (ValueError, G.residual_norm, (x, None), dict(post_weight=w)), (ValueError, G.residual_norm, (x, None), dict(dropout_p=0.1)),
        (TypeError, G.residual_norm, (x, x), dict(pre_weight=w.bfloat16())), (ValueError, G.residual_norm, (x, x), dict(pre_weight=w[:4])),
        (ValueError, G.residual_norm, (x, x), dict(eps=-1.0)), (ValueError, G.residual_norm, (x, x), dict(normed=x.clone())),
        (ValueError, G.residual_norm, (x, x.clone()), dict(out=torch.zeros(2, 3, 9)[..., 1:].transpose(0, 1))),
        (TypeError, G.residual_norm, (x, x), dict(pre_weight=w, normed=b)),
        (ValueError, G.residual_norm_backward, (x, x, None), dict(pre_weight=w, d_normed=x)),
        (ValueError, G.residual_norm_backward, (x, x, st[:1]), {}), (TypeError, G.residual_norm_backward, (x, x, st.double()), {}),
        (ValueError, G.residual_norm_backward, (x, x, st), dict(pre_weight=w)), (ValueError, G.residual_norm_backward, (x, x, st), dict(d_normed=x)),
        (TypeError, G.residual_norm_backward, (x, x, st), dict(d_out=b)),
    ]:
        with pytest.raises(err):
            f(*args, **kw)


def test_results_that_share_memory_are_refused():
    """Before anything else is asked of the operands (these are not on a device)."""
    import gdn2_amd as G

    buf = torch.zeros(3, 32)
    x, y, gate = buf[:, :8], buf[:, 8:16], buf[:, 16:24]
    w = torch.zeros(8)
    for kw in (dict(out=y), dict(out=gate), dict(out=buf[:, 4:12]), dict(pre_weight=w, normed=x), dict(pre_weight=w, normed=gate),
               dict(pre_weight=w, out=buf[:, 24:], normed=buf[:, 24:]), dict(out=buf.view(-1)[1:25].view(3, 8))):
        with pytest.raises(ValueError):
            G.residual_norm(x, y, gate, **kw)
    for kw in (dict(out=x), dict(out=buf[:, 24:]), dict(pre_weight=w, normed=y, out=x)):  # other columns, or in place
        with pytest.raises(TypeError, match="device"):
            G.residual_norm(x, y, gate, **kw)
    with pytest.raises(ValueError):
        G.dropout(x, 0.5, out=buf[:, 1:9])


def test_low_rank_gradients_against_differences():
    g = torch.Generator().manual_seed(8)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=K.F64)  # noqa: E731
    t = {"x": rnd(7, 3), "a": rnd(2, 2, 3), "b": rnd(2, 2, 4)}
    y, dy, ids, scale, cu = rnd(7, 4), rnd(7, 4), [1, 0, 1, -1], [0.7, 1.3], [1, 3, 3, 5, 6]
    loss = lambda t: float((K.low_rank64(y, t["x"], t["a"], t["b"], ids, scale, 1, 7, cu)[0][0] * dy).sum())  # noqa: E731
    h = K.low_rank64(y, t["x"], t["a"], t["b"], ids, scale, 1, 7, cu)[0][1]
    got = K.low_rank_bwd64(t["x"], t["a"], t["b"], ids, h, dy, scale, 1, 7, cu)[0]
    for name, v in t.items():
        for i in np.ndindex(*v.shape):
            lo, hi = dict(t, **{name: v.clone()}), dict(t, **{name: v.clone()})
            lo[name][i] -= 1e-6
            hi[name][i] += 1e-6
            d = (loss(hi) - loss(lo)) / 2e-6
            assert abs(d - float(got["d" + name][i])) <= 1e-7 * (1 + abs(d)), (name, i)


def _lora(**kw):
    from gdn2_amd import _capi as C

    a = C.LowRankArgs()
    for k, v in dict(dict(x=256, a=256, b=256, y=256, out=512, adapters=256, batch=2, seq_len=3, in_features=8, out_features=8,
                          rank=2, num_adapters=2, workspace=256, workspace_bytes=1 << 30), **kw).items():
        setattr(a, k, v)
    return a


def test_low_rank_refusals_of_the_c_entry():
    from gdn2_amd import _capi as C

    L = C.lib()
    for fn in (L.gdn2_low_rank_add_f32, L.gdn2_low_rank_add_bf16):
        assert fn(None, None) == C.GDN2_EINVAL
        for bad in (dict(batch=-1), dict(seq_len=-1), dict(in_features=-1), dict(out_features=-1), dict(rank=-1), dict(num_adapters=-1),
                    dict(x=None), dict(a=None), dict(b=None), dict(y=None), dict(out=None), dict(adapters=None),
                    dict(cu_seqlens=256, num_seqs=1), dict(cu_seqlens=256, batch=1, num_seqs=-1), dict(rank=65, workspace=None),
                    dict(rank=65, workspace=264), dict(rank=65, workspace_bytes=8), dict(out=256, stride_out_t=8)):
            assert fn(_lora(**bad), None) == C.GDN2_EINVAL, bad
            assert b"gdn2_low_rank_add" in L.gdn2_last_error()
        for big in (dict(rank=513), dict(in_features=1 << 24), dict(out_features=1 << 24), dict(batch=1 << 20, seq_len=1 << 20),
                    dict(num_adapters=1 << 24), dict(batch=1 << 24, seq_len=1), dict(seq_len=1 << 29, out_features=1 << 20)):
            assert fn(_lora(**big), None) == C.GDN2_NOT_APPLICABLE, big
        for nothing in (dict(batch=0), dict(seq_len=0), dict(out_features=0)):
            assert fn(_lora(**nothing), None) == C.GDN2_OK
    for fn in (L.gdn2_low_rank_add_bwd_f32, L.gdn2_low_rank_add_bwd_bf16):
        assert fn(None, None) == C.GDN2_EINVAL

        def bwd(fwd={}, **kw):
            b = C.LowRankBwdArgs()
            b.fwd = _lora(hidden=256, **fwd)
            for k, v in dict(dict(d_out=256, dx=256, da=256, db=256, workspace=256, workspace_bytes=1 << 30), **kw).items():
                setattr(b, k, v)
            return fn(ctypes.byref(b), None)

        for fwd, kw in ((dict(rank=-1), {}), (dict(x=None), {}), (dict(a=None), {}), (dict(b=None), {}), (dict(adapters=None), {}),
                        ({}, dict(d_out=None)), ({}, dict(workspace=None)), ({}, dict(workspace=264)), ({}, dict(workspace_bytes=8))):
            assert bwd(fwd, **kw) == C.GDN2_EINVAL, (fwd, kw)
        b = C.LowRankBwdArgs(_lora(), 256, 256, 256, 256, 0, 0, 0, 0, 0, 256, 1 << 30)  # hidden missing
        assert fn(b, None) == C.GDN2_EINVAL
        assert bwd(dict(rank=513)) == C.GDN2_NOT_APPLICABLE


def test_low_rank_workspace_sizes():
    from gdn2_amd import _capi as C

    L = C.lib()
    size = lambda **kw: L.gdn2_low_rank_add_workspace_bytes(_lora(**kw))  # noqa: E731
    assert L.gdn2_low_rank_add_workspace_bytes(None) == L.gdn2_low_rank_add_bwd_workspace_bytes(None) == 0
    assert size(batch=0) == size(rank=0) == size(rank=513) == size(seq_len=-1) == 0
    # more than 64 ranks: h in f32, rows of a multiple of 16
    assert size(batch=8, seq_len=4096, rank=64) == 0 and size(batch=64, seq_len=1, rank=65) == 4 * 64 * 80


def test_low_rank_refusals_in_python():
    import gdn2_amd as G

    x, y, a, b = torch.zeros(2, 3, 8), torch.zeros(2, 3, 6), torch.zeros(4, 2, 8), torch.zeros(4, 2, 6)
    ids, sc, cu = torch.zeros(2, dtype=torch.int32), torch.zeros(4), torch.tensor([0, 2, 3], dtype=torch.int32)
    h, w = torch.zeros(2, 3, 2), torch.zeros(2, 3, 14)
    for err, args, kw in [
        (TypeError, (y, x, a, b, ids), {}),  # not on a device
        (TypeError, (y.half(), x.half(), a.half(), b.half(), ids), {}), (TypeError, (y, x, a.bfloat16(), b, ids), {}),
        (TypeError, (y.bfloat16(), x, a, b, ids), {}), (ValueError, (y, x[0, 0], a, b, ids), {}), (ValueError, (y, x, a[0], b, ids), {}),
        (ValueError, (y, x, a[..., :4], b, ids), {}), (ValueError, (y, x, a[:, :1], b, ids), {}), (ValueError, (y, x, a[:2], b, ids), {}),
        (ValueError, (y[:1], x, a, b, ids), {}), (ValueError, (y, x, a, b[..., :5], ids), {}), (TypeError, (y, x, a, b, ids.long()), {}),
        (ValueError, (y, x, a, b, ids[:1]), {}), (TypeError, (y, x, a, b, ids, sc.double()), {}), (ValueError, (y, x, a, b, ids, sc[:2]), {}),
        (ValueError, (y, x, a, b, ids), dict(cu_seqlens=cu)), (TypeError, (y[:1], x[:1], a, b, ids), dict(cu_seqlens=cu.long())),
        (ValueError, (y[:1], x[:1], a, b, ids), dict(cu_seqlens=cu[:0])), (ValueError, (y[:1], x[:1], a, b, ids), dict(cu_seqlens=cu[:2])),
        (ValueError, (y, x, a, b, ids), dict(out=y[..., :5])), (TypeError, (y, x, a, b, ids), dict(out=y.bfloat16())),
        (ValueError, (w[..., 8:], w[..., :8], a, b, ids), dict(out=w[..., 2:8])),
        (ValueError, (y, x, a, b, ids), dict(out=torch.zeros(6).expand(2, 3, 6))),
    ]:
        with pytest.raises(err):
            G.low_rank_add(*args, **kw)
    for err, args, kw in [
        (TypeError, (x, a, b, ids, h, y), {}), (ValueError, (x, a, b, ids, h[..., :1], y), {}), (TypeError, (x, a, b, ids, h.bfloat16(), y), {}),
        (ValueError, (x, a, b, ids, h, x), {}), (ValueError, (x, a, b, ids, h, y), dict(dx=x)), (ValueError, (x, a, b, ids, h, y), dict(dx=y)),
    ]:
        with pytest.raises(err):
            G.low_rank_add_backward(*args, **kw)


def test_layer_adapters_of_the_c_entry():
    """Invalid adapters come back before any launch (a layer is not needed to see that)."""
    from gdn2_amd import _capi as C

    L = C.lib()
    assert L.gdn2_layer_forward_adapted_f32(None, 256, 1, 1, None, 512, None, None) == C.GDN2_EINVAL
    assert b"gdn2_layer_forward_adapted_f32" in L.gdn2_last_error()
