"""Decode on 4-bit weights (set_decode_bits): against the oracle run on the weights that the
codes stand for, across the attention forms, graph and eager; the switch itself."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import oracle as orc
from test_gpu_four_bit import ref_weight

pytestmark = pytest.mark.gpu


def _model(gpu, seed, **kw):
    from larynx_amd.llm import Qwen2Config, Qwen2LM, qwen2_param_shapes
    cfg = Qwen2Config(n_layers=2, text_vocab=2000, **kw)
    params = orc.make_params(qwen2_param_shapes(cfg), seed)
    for k in params:
        if k.endswith("layernorm.weight") or k == "norm.weight":
            params[k] = (params[k] + 1.0).astype(np.float32)
    lm = Qwen2LM({k: torch.from_numpy(v).to(gpu) for k, v in params.items()}, cfg, max_ctx=320)
    return cfg, params, lm


@pytest.fixture(scope="module")
def lm4(gpu):
    cfg, params, lm = _model(gpu, 91)
    yield cfg, params, lm
    lm.close()


def _stand_for(params, group):
    """The model's weights with those decode holds in 4 bits replaced by what they stand for."""
    out = dict(params)
    for k, v in params.items():
        if any(n in k for n in ("q_proj.weight", "k_proj.weight", "v_proj.weight", "mlp.",
                                "llm_decoder")):
            out[k] = ref_weight(v, group)[0].astype(np.float32)
    return out


def _fill(lm, o, cfg, n, gpu):
    for layer in range(cfg.n_layers):
        kd, vd = lm.cache_views(layer)
        kd.fill_(float("nan"))
        vd.fill_(float("nan"))
        for cache, dev, part in ((o.k_cache, kd, 1), (o.v_cache, vd, 2)):
            c = orc.normal((n, kd.shape[1]), 700 + layer, part, 1.0)
            cache[layer, :n] = c
            dev[:n].copy_(torch.from_numpy(c))
    o.cache_len = n
    lm.set_cache_len(n)


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 63, 64, 200])
def test_decode_on_4_bit_weights_vs_oracle(gpu, lm4, n, group, graph):
    """The bar of the fp32 decode (test_gpu_decode_short): sums of at most 4864 products with
    errors of fp32's level, through two layers.  Three steps, so that appended rows are read."""
    cfg, params, lm = lm4
    announce(f"4-bit decode n={n} group={group} graph={graph}")
    lm.set_decode_bits(4, group)
    lm.set_decode_graph(graph)
    o = orc.Qwen2(_stand_for(params, group), cfg, cap=320)
    _fill(lm, o, cfg, n, gpu)
    for tok in (4321, 17, 6560):
        lg, fn = lm.decode(tok, final_norm=True)
        torch.cuda.synchronize()
        rlg, rfn = o.decode(tok)
        assert orc.rel_err(fn.cpu().numpy(), rfn) < 1e-5
        assert orc.rel_err(lg.cpu().numpy(), rlg) < 1e-5


def test_switching_back_gives_the_fp32_bits(gpu, lm4):
    cfg, params, lm = lm4
    announce("4-bit decode switched on and off")
    o = orc.Qwen2(params, cfg, cap=320)
    lm.set_decode_graph(True)
    got = []
    for bits in (32, 4, 32, 4):
        lm.set_decode_bits(bits)
        _fill(lm, o, cfg, 100, gpu)
        got.append([lm.decode(t) for t in (5, 6)])
    torch.cuda.synchronize()
    for a, b in ((0, 2), (1, 3)):
        for x, y in zip(got[a], got[b]):
            assert torch.equal(x, y)
    assert not torch.equal(got[0][0], got[1][0])
    # the prefill does not see the switch
    x = lm.build_lm_input([1, 2, 3], [4, 5])
    p4 = lm.prefill(x)
    lm.set_decode_bits(32)
    assert torch.equal(p4, lm.prefill(x))


@pytest.mark.parametrize("kw", [dict(hidden=320, intermediate=1100, n_heads=5, n_kv_heads=1),
                                dict(hidden=1024, intermediate=132, n_heads=16, n_kv_heads=8),
                                dict(hidden=1536, intermediate=2048, n_heads=24, n_kv_heads=4)])
def test_other_geometries(gpu, kw):
    """Widths that are no multiple of a group or a block, one to eight kv heads, and one past the
    eight blocks that a wave requests at once."""
    announce(f"4-bit decode {kw}")
    cfg, params, lm = _model(gpu, 92, **kw)
    lm.set_decode_bits(4, 64)
    o = orc.Qwen2(_stand_for(params, 64), cfg, cap=320)
    for n in (5, 150):
        _fill(lm, o, cfg, n, gpu)
        lg = lm.decode(999)
        torch.cuda.synchronize()
        assert orc.rel_err(lg.cpu().numpy(), o.decode(999)[0]) < 1e-5
    lm.close()


def test_refusals(gpu, lm4):
    from larynx_amd import LxError
    lm = lm4[2]
    announce("set_decode_bits refusals")
    for bits, group in ((8, 64), (4, 16), (0, 0), (-4, 64)):
        with pytest.raises(LxError):
            lm.set_decode_bits(bits, group)
