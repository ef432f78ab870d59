"""What the block operators do at their edges without a GPU: empty batches and sizes
whose products pass 64 bits.  No call here gets as far as a launch."""
import ctypes

import pytest
import torch

from gdn2_amd import _capi as C


def _res(**kw):
    a = C.ResidualNormArgs()
    for k, v in dict(dict(x=256, y=256, out=256, samples=2, rows=3, channels=8, eps=1e-5, residual_scale=1.0,
                          branch_scale=1.0), **kw).items():
        setattr(a, k, v)
    return a


def _res_bwd(fwd, **kw):
    b = C.ResidualNormBwdArgs()
    b.fwd = _res(**fwd)
    for k, v in dict(dict(d_out=256, dx=256, dy=256), **kw).items():
        setattr(b, k, v)
    return ctypes.byref(b)


def test_residual_backward_of_no_samples():
    """A gate a sample and no samples: an empty dgate, and nothing to launch."""
    L = C.lib()
    for fn in (L.gdn2_residual_norm_bwd_f32, L.gdn2_residual_norm_bwd_bf16, L.gdn2_residual_norm_bwd_f32_bf16):
        for rows in (0, 3):
            assert fn(_res_bwd(dict(gate=256, gate_rows=C.GATE_SAMPLE, samples=0, rows=rows), dgate=256), None) == C.GDN2_OK
        assert fn(_res_bwd(dict(samples=0)), None) == C.GDN2_OK
    assert L.gdn2_residual_norm_bwd_workspace_bytes(_res_bwd(dict(gate=256, gate_rows=C.GATE_SAMPLE, samples=0), dgate=256)) == 0


def test_sizes_whose_product_passes_64_bits():
    """2^32 samples of 2^32 rows are not none."""
    L = C.lib()
    for fn in (L.gdn2_residual_norm_f32, L.gdn2_residual_norm_bf16, L.gdn2_residual_norm_f32_bf16):
        for samples, rows in ((1 << 32, 1 << 32), (1 << 62, 4), (1 << 33, 1 << 30)):
            assert fn(_res(samples=samples, rows=rows), None) == C.GDN2_NOT_APPLICABLE
    for fn in (L.gdn2_residual_norm_bwd_f32, L.gdn2_residual_norm_bwd_bf16, L.gdn2_residual_norm_bwd_f32_bf16):
        assert fn(_res_bwd(dict(samples=1 << 32, rows=1 << 32)), None) == C.GDN2_NOT_APPLICABLE
    for fn in (L.gdn2_dropout_f32, L.gdn2_dropout_bf16):
        assert fn(256, 512, 1 << 39, 1 << 30, 1 << 30, 1 << 30, C.Dropout(0.5, 0, 0, None), None) == C.GDN2_NOT_APPLICABLE
    big = dict(batch=1 << 32, seq_len=1 << 32)
    for fn in (L.gdn2_low_rank_add_f32, L.gdn2_low_rank_add_bf16):
        a = C.LowRankArgs()
        for k, v in dict(x=256, a=256, b=256, y=256, out=512, adapters=256, in_features=8, out_features=8, rank=2, num_adapters=2,
                         **big).items():
            setattr(a, k, v)
        assert fn(a, None) == C.GDN2_NOT_APPLICABLE


def _one(t, *strides):
    """t's memory by other strides of its dimensions of one."""
    return t.as_strided(t.shape, strides)


def test_strides_of_dimensions_of_one_do_not_count():
    """In place is in place, and other columns of the same rows are other columns (these
    operands are not on a device: the next check refuses)."""
    import gdn2_amd as G

    x, y, w = torch.zeros(64, 1, 8), torch.zeros(64, 1, 8), torch.zeros(8)
    out, normed = _one(x, 8, 512, 1), _one(y, 8, 3, 1)
    one = torch.zeros(5, 1)
    buf = torch.zeros(4, 1, 32)
    left, right = buf[..., :8], _one(buf[..., 8:], 32, 77, 1)[..., :8]
    ids, a = torch.zeros(64, dtype=torch.int32), torch.zeros(1, 2, 8)
    for f, args, kw in ((G.dropout, (x, 0.5), dict(out=out)), (G.dropout, (one, 0.5), dict(out=_one(one, 1, 9))),
                        (G.residual_norm, (x, y), dict(out=out)), (G.residual_norm, (x, y, None, w, w), dict(out=out, normed=normed)),
                        (G.residual_norm, (left, torch.zeros(4, 1, 8)), dict(out=right)),
                        (G.low_rank_add, (y, x, a, a, ids), dict(out=normed))):
        with pytest.raises(TypeError, match="device"):
            f(*args, **kw)
    with pytest.raises(ValueError):  # still refused: another place of the same memory
        G.dropout(buf[..., :8], 0.5, out=_one(buf[..., 4:], 32, 5, 1)[..., :8])


def test_limits_of_dropout():
    """Rows that lie together: from 2^24 workgroups of 1024 (f32) or 2048 (bf16) elements on."""
    L = C.lib()
    half = C.Dropout(0.5, 0, 0, None)
    for fn, per in ((L.gdn2_dropout_f32, 1024), (L.gdn2_dropout_bf16, 2048)):
        for rows, ch in (((1 << 24) * per // 2048, 2048), (((1 << 24) - 1) * per // 8 + 1, 8), ((1 << 40), 8)):
            assert fn(256, 512, rows, ch, ch, ch, half, None) == C.GDN2_NOT_APPLICABLE
        assert fn(256, 512, (1 << 32) - 256, 4, 8, 8, half, None) == C.GDN2_NOT_APPLICABLE  # counters of rows apart
