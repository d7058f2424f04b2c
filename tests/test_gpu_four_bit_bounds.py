"""The four-bit operators against the bounds of four_bit_bounds (test_four_bit_bounds plants
mistakes that these see), and attention that counts every key once."""
import numpy as np
import pytest
import torch

import four_bit_bounds as fb
from conftest import announce
from test_four_bit_bounds import LINEAR
from test_gpu_four_bit import CASES, _attn_case, _dev, _gen, ref_cache, ref_weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
def test_attention_within_bounds(gpu, case, causal):
    from larynx_amd import ops
    B, Tq, heads, kv, hd, rows, lens, max_len = case
    announce(f"kv4 attention bounds {case} causal={causal}")
    rng = _gen(sum(case[:6]) + 1)
    q, k, v, cache = _attn_case(gpu, rng, B, Tq, heads, kv, hd, rows, lens)
    want, bound = fb.attention(q, ref_cache(k), ref_cache(v), lens, heads, hd ** -0.5, causal)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    got = ops.attention_kv4(_dev(q, gpu), cache, n, heads, causal=causal, max_len=max_len)
    fb.check(got.cpu().numpy().reshape(want.shape) - want, bound)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES + [
    (1, 1, 2, 2, 64, 9000, [8191], 0), (1, 1, 32, 8, 128, 20000, [19999], 0),
    (64, 1, 14, 2, 64, 700, list(range(1, 705, 11)), 700), (1, 300, 14, 2, 64, 2000, [2000], 0)],
    ids=lambda c: "-".join(map(str, c[:6])))
def test_attention_counts_every_key_once(gpu, case, causal):
    """A query of zeros weighs all keys alike: an output is the mean of its values.  These are whole
    numbers 0 .. 15 that the cache holds exactly, so that weights, sums and counts are exact in fp32
    and only the quotient rounds (its reciprocal and the product: 2 U); a key lost, doubled or taken
    for another moves the mean by 1 / n of a step and more."""
    from larynx_amd import ops
    B, Tq, heads, kv, hd, rows, lens, max_len = case
    announce(f"kv4 attention counts {case} causal={causal}")
    rng = _gen(sum(case[:6]))
    v = rng.integers(0, 16, (B, rows, kv, hd)).astype(np.float32)
    v[..., ::64], v[..., 1::64] = 0, 15
    k = rng.standard_normal((B, rows, kv, hd)).astype(np.float32)
    cache = ops.kv4_cache(B, kv, rows, hd)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, _dev(k.reshape(B, rows, -1), gpu), _dev(v.reshape(B, rows, -1), gpu),
                   zero)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    got = ops.attention_kv4(torch.zeros(B, Tq, heads * hd, device=gpu), cache, n, heads,
                            causal=causal, max_len=max_len).cpu().numpy().astype(np.float64)
    sums = np.concatenate([np.zeros((B, 1, kv, hd)), np.cumsum(v, 1, dtype=np.float64)], 1)
    for b in range(B):
        for t in range(Tq):
            seen = max(0, lens[b] - Tq + t + 1) if causal else lens[b]
            want = np.repeat(sums[b, seen] / max(seen, 1), heads // kv, 0).ravel()
            assert (np.abs(got[b, t] - want) <= 3 * fb.U * want).all(), (b, t)


def test_attention_large_scores_within_bounds(gpu):
    """Scores in the hundreds, rising and falling along the keys."""
    from larynx_amd import ops
    announce("kv4 attention large scores, bounds")
    rng = _gen(20)
    for rows, hd, heads in ((300, 64, 1), (700, 128, 4)):
        k = rng.standard_normal((2, rows, 1, hd)).astype(np.float32) * np.float32(0.1)
        ramp = np.linspace(0, 40, rows, dtype=np.float32)
        k += np.stack([ramp, ramp[::-1]])[:, :, None, None]
        v = rng.standard_normal((2, rows, 1, hd)).astype(np.float32)
        q = (1 + 0.1 * rng.standard_normal((2, 1, heads * hd))).astype(np.float32)
        cache = ops.kv4_cache(2, 1, rows, hd)
        zero = torch.zeros(2, dtype=torch.int32, device=gpu)
        ops.kv4_append(cache, _dev(k.reshape(2, rows, -1), gpu), _dev(v.reshape(2, rows, -1), gpu),
                       zero)
        got = ops.attention_kv4(_dev(q, gpu), cache, zero + rows, heads).cpu().numpy()
        want, bound = fb.attention(q, ref_cache(k), ref_cache(v), [rows] * 2, heads, hd ** -0.5,
                                   True)
        fb.check(got.reshape(want.shape) - want, bound)


@pytest.mark.parametrize("M,N,K,G", LINEAR + [(2, 1152, 896, 64), (8, 896, 4864, 64),
                                              (1, 896, 4864, 128), (33, 300, 8192, 128)])
def test_projections_within_bounds(gpu, M, N, K, G):
    from larynx_amd import ops
    announce(f"q4 linear bounds M={M} N={N} K={K} G={G}")
    rng = _gen(M + N + K)
    W = (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0] *= 1e3
    x[:, K // 2] *= 50  # a channel that stands out
    want, bound = fb.linear(x, *ref_weight(W, G), G)
    got = ops.linear_q4(_dev(x, gpu), ops.q4_pack(_dev(W, gpu), G)).cpu().numpy()
    fb.check(got - want, bound)
