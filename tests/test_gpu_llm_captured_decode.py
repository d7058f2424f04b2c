"""Decode steps that the caller captured (set_decode_graph(False)) across set_decode_bits."""
import pytest
import torch

from conftest import announce
from test_gpu_llm_four_bit import _model

pytestmark = pytest.mark.gpu


def _captured(lm, gpu):
    """A decode step at row 40 captured into a graph of the caller's: (graph, its logits)."""
    lm.set_cache_len(40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lm.decode(11)
    torch.cuda.current_stream().wait_stream(side)
    lm.set_cache_len(40)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logits = lm.decode(11)
    return g, logits


@pytest.mark.parametrize("first", [32, 64, 128])
def test_captured_steps_outlive_a_change_of_group(gpu, first):
    """A captured step gives the logits of the weights it was captured on, whatever decode runs on
    since: another group, fp32, and the first again."""
    announce(f"captured decode, groups of {first} first")
    cfg, params, lm = _model(gpu, 93)
    for layer in range(cfg.n_layers):
        for i, c in enumerate(lm.cache_views(layer)):
            g = torch.Generator(device=gpu).manual_seed(10 * layer + i)
            c[:40].copy_(torch.randn(c[:40].shape, device=gpu, generator=g))
    lm.set_decode_graph(False)
    lm.set_decode_bits(4, first)
    graph, logits = _captured(lm, gpu)
    graph.replay()
    torch.cuda.synchronize()
    want = logits.clone()
    for bits, group in ((4, 32), (4, 64), (4, 128), (32, 0), (4, first)):
        lm.set_decode_bits(bits, group)
        lm.set_cache_len(40)
        eager = lm.decode(11)
        logits.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want), (bits, group)
        assert torch.equal(eager, want) == ((bits, group) == (4, first))
    lm.close()
