"""Attention over the 4-bit cache where the cached values differ much in scale.

What a row contributes is its weight times its values: a row of large values and next to no weight
must not cost the others their precision, nor one that does count, nor the size of all of them."""
import numpy as np
import pytest
import torch

import four_bit_bounds as fb
from conftest import announce
from test_gpu_four_bit import ref_cache

pytestmark = pytest.mark.gpu

SHAPES = [(2, 1, 2, 2, 64, 70), (2, 1, 14, 2, 64, 150), (1, 1, 32, 8, 128, 64),
          (1, 9, 14, 2, 64, 100), (1, 5, 8, 2, 128, 97), (1, 1, 14, 2, 64, 2500)]


def _attend(gpu, q, k, v, heads):
    from larynx_amd import ops
    B, rows, kv, hd = k.shape
    cache = ops.kv4_cache(B, kv, rows, hd)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    kd, vd = (torch.from_numpy(a.reshape(B, rows, -1)).to(gpu) for a in (k, v))
    ops.kv4_append(cache, kd, vd, zero)
    o = ops.attention_kv4(torch.from_numpy(q).to(gpu), cache, zero + rows, heads, causal=False)
    return o.cpu().numpy().reshape(*q.shape[:2], heads, hd)


@pytest.mark.parametrize("gap", [0.0, 20.0, 60.0])
@pytest.mark.parametrize("ratio", [10, 16, 24, 30, -30])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_rows_of_other_scales(gpu, shape, ratio, gap):
    """Rows 2^ratio as large in value and e^-gap of the weight, first and last and in between."""
    announce(f"kv4 value scales {shape} 2^{ratio} gap {gap}")
    B, Tq, heads, kv, hd, rows = shape
    rng = np.random.default_rng(sum(shape) + ratio + 64)
    for at in ([0], [rows - 1], [3, rows // 2]):
        q, k, v = fb.value_scale_case(rng, B, Tq, heads, kv, hd, rows, 2.0 ** ratio, at, gap)
        want, bound = fb.attention(q, ref_cache(k), ref_cache(v), [rows] * B, heads, hd ** -0.5,
                                   False)
        fb.check(_attend(gpu, q, k, v, heads) - want, bound)


@pytest.mark.parametrize("big", [0, 1])
@pytest.mark.parametrize("ratio", [16, 30])
def test_groups_of_other_scales(gpu, ratio, big):
    """Heads of 128: one of a row's two groups 2^ratio as large, in one row and in all of them."""
    announce(f"kv4 value scales of groups 2^{ratio} group {big}")
    rng = np.random.default_rng(ratio + big)
    for at in ([0], list(range(80))):
        q, k, v = fb.value_scale_case(rng, 2, 1, 8, 2, 128, 80, 2.0 ** ratio, at, 0.0, [big])
        want, bound = fb.attention(q, ref_cache(k), ref_cache(v), [80] * 2, 8, 128 ** -0.5, False)
        fb.check(_attend(gpu, q, k, v, 8) - want, bound)


@pytest.mark.parametrize("power", [-60, 60, 100, 108])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_all_values_of_another_size(gpu, shape, power):
    """Values times a power of two: outputs times the same, to the bit (scores within 15, so that no
    product of a weight and a scale leaves fp32's normal range)."""
    announce(f"kv4 value size {shape} 2^{power}")
    B, Tq, heads, kv, hd, rows = shape
    rng = np.random.default_rng(sum(shape))
    q = rng.standard_normal((B, Tq, heads * hd)).astype(np.float32)
    k, v = (rng.standard_normal((B, rows, kv, hd)).astype(np.float32) for _ in range(2))
    k *= 2
    one = _attend(gpu, q, k, v, heads)
    assert np.abs(v).max() < 32
    got = _attend(gpu, q, k, v * np.float32(2.0 ** power), heads)
    assert np.array_equal(got, one * np.float32(2.0 ** power))


def test_rows_without_range_and_large(gpu):
    """Rows whose channels are all alike (codes without a scale) beside ordinary ones, and nothing
    but such rows, up to 2^115."""
    announce("kv4 values without range")
    rng = np.random.default_rng(5)
    for power, every in ((0, 3), (30, 5), (100, 1), (115, 1)):
        q, k, v = fb.value_scale_case(rng, 2, 1, 14, 2, 64, 90, 1.0, [], 0.0)
        v[:, ::every] = np.float32(2.0 ** power) * np.float32(
            rng.uniform(1, 1.9, v[:, ::every, :, :1].shape))
        want, bound = fb.attention(q, ref_cache(k), ref_cache(v), [90] * 2, 14, 0.125, False)
        fb.check(_attend(gpu, q, k, v, 14) - want, bound)
