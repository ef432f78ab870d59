"""GatedDeltaNet2.forward with adapters: every request against the oracle's layer whose
weights are the shared ones plus that request's low-rank products."""
import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu


def make(layer, names, L, R, seed):
    import gdn2_amd as G

    r = np.random.default_rng(seed)
    return {n: tuple((r.standard_normal((L, R, d)) * (0.5 / np.sqrt(d * R)) ** 0.5).astype(np.float32)
                     for d in G.layer.param_shape(layer.config, n)) for n in names}


def merged(params, host, scale, l):
    """The weights that a request with adapter l sees."""
    w = dict(params)
    for n, (a, b) in host.items():
        if 0 <= l < a.shape[0]:
            w[n] = (params[n].astype(np.float64) + float(scale[l]) * (a[l].astype(np.float64).T @ b[l].astype(np.float64))).astype(np.float32)
    return w


CONFIGS = {
    "chunk": dict(hidden_size=256, num_heads=4, head_dim=64, mode="chunk"),
    "recurrent_gva": dict(hidden_size=128, num_heads=2, num_v_heads=4, head_dim=32, mode="fused_recurrent"),
    "no_conv": dict(hidden_size=192, num_heads=3, head_dim=64, use_short_conv=False, mode="chunk"),
}


@pytest.mark.parametrize("case", list(CONFIGS))
@pytest.mark.parametrize("names,R", [(("q_proj", "v_proj"), 8), (("q_proj", "k_proj", "b_proj", "v_proj", "w_proj", "f_proj_0", "g_proj_0", "o_proj"), 5),
                                     (("o_proj",), 64)])
def test_prefill_and_decode(gpu, case, names, R):
    """A prompt of 70 tokens, three single ones, then five at once: outputs and states."""
    import torch

    import gdn2_amd as G

    cfg = G.Gdn2Config(**CONFIGS[case])
    layer = G.GatedDeltaNet2(cfg, seed=11)
    L, ids = 3, [2, -1, 0, 2, 7]
    host = make(layer, names, L, R, 5)
    scale = np.array([0.5, 3.0, 1.5], np.float32)
    dev = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(gpu)  # noqa: E731
    ad = G.Gdn2Adapters(layer, {n: (dev(a), dev(b)) for n, (a, b) in host.items()}, dev(scale))
    dids = torch.tensor(ids, dtype=torch.int32, device=gpu)
    xh = np.random.default_rng(3).standard_normal((len(ids), 78, cfg.hidden_size)).astype(np.float32)
    x, outs, st = dev(xh), [], None
    for t0, t1 in ((0, 70), (70, 71), (71, 72), (72, 73), (73, 78)):
        o, st = layer.forward(x[:, t0:t1], st, adapters=ad, adapter_ids=dids)
        outs.append(o)
    got = torch.cat(outs, 1).cpu().numpy()
    params = layer.params()
    plain = layer.forward(x)[0].cpu().numpy()
    for i, l in enumerate(ids):
        ref, rst = O.layer_forward(cfg, merged(params, host, scale, l), xh[i:i + 1])
        size = np.abs(ref.out).max()
        # the merged weight is rounded to f32 (2^-24 of each of up to 256 terms), the layer's
        # own bound is 1e-4 of the largest output
        assert np.abs(got[i] - ref.out[0]).max() <= 1e-4 * size, (i, l)
        assert np.abs(st.recurrent[i] - rst.recurrent[0]).max() <= 1e-4 * max(1.0, np.abs(rst.recurrent).max())
        if 0 <= l < L:
            assert np.abs(plain[i] - ref.out[0]).max() > 1e-2 * size  # (the adapters matter)
        else:
            assert np.abs(plain[i] - ref.out[0]).max() <= 1e-4 * size


def test_captured_step(gpu):
    """A decoding step recorded once, replayed after the requests' adapters changed."""
    import torch

    import gdn2_amd as G

    cfg = G.Gdn2Config(hidden_size=256, num_heads=4, head_dim=64)
    layer = G.GatedDeltaNet2(cfg, seed=2)
    host = make(layer, ("q_proj", "o_proj"), 4, 16, 9)
    ad = G.Gdn2Adapters(layer, {n: tuple(torch.from_numpy(v).to(gpu) for v in ab) for n, ab in host.items()})
    B = 6
    x, ids = torch.randn(B, 1, 256, device=gpu), torch.zeros(B, dtype=torch.int32, device=gpu)
    rec, ref = G.Gdn2State.zeros(layer, B), G.Gdn2State.zeros(layer, B)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):  # (the conv caches alternate between two buffers: an even number of steps a graph)
            layer.forward(x, rec, ad, ids)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o1, _ = layer.forward(x, rec, ad, ids)
        o2, _ = layer.forward(x, rec, ad, ids)
    for _ in range(2):
        layer.forward(x, ref, ad, ids)
    for i in range(3):
        ids.copy_(torch.tensor([(i + j) % 5 for j in range(B)]))
        x.copy_(torch.randn(B, 1, 256, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        for o in (o1, o2):
            want, _ = layer.forward(x, ref, ad, ids)
            assert torch.equal(o, want)


def test_refusals(gpu):
    import torch

    import gdn2_amd as G

    cfg = G.Gdn2Config(hidden_size=64, num_heads=1, head_dim=32)
    layer, other = G.GatedDeltaNet2(cfg), G.GatedDeltaNet2(cfg)
    a, b = torch.zeros(2, 4, 64, device=gpu), torch.zeros(2, 4, 32, device=gpu)
    ids, x = torch.zeros(3, dtype=torch.int32, device=gpu), torch.zeros(3, 2, 64, device=gpu)
    for err, w, scale in [(ValueError, {"f_proj_1": (b, b)}, None), (ValueError, {"q_proj": (b, a)}, None), (TypeError, {"q_proj": (a.cpu(), b)}, None),
                          (TypeError, {"q_proj": (a.double(), b)}, None), (ValueError, {"q_proj": (a, b[:1])}, None),
                          (ValueError, {"q_proj": (a, b), "k_proj": (a[:1], b[:1])}, None),
                          (ValueError, {"q_proj": (torch.zeros(2, 65, 64, device=gpu), torch.zeros(2, 65, 32, device=gpu))}, None),
                          (ValueError, {"q_proj": (a, b)}, torch.ones(3, device=gpu)), (TypeError, {"q_proj": (a, b)}, torch.ones(2))]:
        with pytest.raises(err):
            G.Gdn2Adapters(layer, w, scale)
    ad = G.Gdn2Adapters(layer, {"q_proj": (a, b)})
    for err, args in [(ValueError, (ad, None)), (ValueError, (None, ids)), (TypeError, (ad, ids.long())), (ValueError, (ad, ids[:2])),
                      (ValueError, (ad, ids.cpu())), (ValueError, (G.Gdn2Adapters(other, {"q_proj": (a, b)}), ids))]:
        with pytest.raises(err):
            layer.forward(x, None, *args)
    got, _ = layer.forward(x, None, G.Gdn2Adapters(layer, {}), ids)  # none at all
    assert torch.equal(got, layer.forward(x)[0])
