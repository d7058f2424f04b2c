"""The bounds of four_bit_bounds on the CPU: the operators' arithmetic restated in numpy stays
within them, and each mistake planted in it does not."""
import numpy as np
import pytest

import four_bit_bounds as fb
from test_gpu_four_bit import ref_cache, ref_weight


def _run(q, k, v, **kw):
    """Head by head, one query each."""
    kc, vc = ref_cache(k), ref_cache(v)
    heads, hd = q.shape[2] // k.shape[3], k.shape[3]
    want, bound = fb.attention(q, kc, vc, [k.shape[1]], heads, hd ** -0.5, False)
    rep = heads // k.shape[2]
    got = np.stack([fb.emulate(q[0, 0, h * hd:(h + 1) * hd], [a[0, :, h // rep] for a in kc],
                               [a[0, :, h // rep] for a in vc], hd ** -0.5, **kw)
                    for h in range(heads)])
    return got - want[0, 0], bound[0, 0]


@pytest.mark.parametrize("gap", [0.0, 20.0, 60.0])
@pytest.mark.parametrize("ratio", [10, 16, 24, 30, -30])
@pytest.mark.parametrize("hd", [64, 128])
def test_parts_that_follow_the_weights_stay_within(hd, ratio, gap):
    rng = np.random.default_rng(hd + ratio + 64)
    for at in ([0], [149], [3, 75]):
        q, k, v = fb.value_scale_case(rng, 1, 1, 8, 2, hd, 150, 2.0 ** ratio, at, gap)
        fb.check(*_run(q, k, v))


@pytest.mark.parametrize("ratio", [16, 24, 30])
@pytest.mark.parametrize("hd", [64, 128])
def test_parts_that_follow_the_scales_are_seen(hd, ratio):
    rng = np.random.default_rng(hd + ratio)
    q, k, v = fb.value_scale_case(rng, 1, 1, 8, 2, hd, 150, 2.0 ** ratio, [0], 60.0)
    with pytest.raises(AssertionError):
        fb.check(*_run(q, k, v, lift="scales"))


def _plain_case(rng, hd, rows):
    q = (2 * rng.standard_normal((1, 1, 8 * hd))).astype(np.float32)
    k, v = (rng.standard_normal((1, rows, 2, hd)).astype(np.float32) for _ in range(2))
    k[..., ::16] += 4.0
    return q, k, v


@pytest.mark.parametrize("hd,rows", [(64, 33), (64, 2001), (128, 1055)])
def test_a_query_of_one_part_is_seen(hd, rows):
    q, k, v = _plain_case(np.random.default_rng(hd + rows), hd, rows)
    fb.check(*_run(q, k, v))
    with pytest.raises(AssertionError):
        fb.check(*_run(q, k, v, parts=1))


@pytest.mark.parametrize("rows", [70, 1055, 4000])
def test_a_lost_key_is_seen(rows):
    """A key that weighs less than nine tenths of the others."""
    q, k, v = _plain_case(np.random.default_rng(rows), 64, rows)
    s = ref_cache(k)[0][0, :, 0] @ q[0, 0, :64]
    with pytest.raises(AssertionError):
        fb.check(*_run(q, k, v, skip=int(np.argsort(s)[rows // 10])))


LINEAR = [(1, 9728, 896, 64), (3, 6762, 896, 32), (4, 896, 4864, 64), (5, 70, 1000, 128),
          (16, 384, 2048, 128), (29, 46, 772, 64), (64, 258, 516, 32)]


@pytest.mark.parametrize("M,N,K,G", LINEAR)
def test_projections_of_one_part_are_seen(M, N, K, G):
    rng = np.random.default_rng(M + N + K)
    W = (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0] *= 1e3
    want, bound = fb.linear(x, *ref_weight(W, G), G)
    for parts in (2, 1):
        xp = np.zeros(x.shape)
        for k in range(0, K, 128):
            f = 2.0 ** np.floor(np.log2(np.abs(x[:, k:k + 128]).max(1, keepdims=True)))
            xp[:, k:k + 128] = fb.two_parts(x[:, k:k + 128] / f, parts) * f
        err = (xp @ ref_weight(W, G)[0].T).astype(np.float32) - want
        if parts == 2:
            fb.check(err, bound)
        else:
            with pytest.raises(AssertionError):
                fb.check(err, bound)
