"""The four-bit operators on the GPU against plain 64-bit forms.

What is held in 4 bits must equal the definition's value exactly (both sides form the quotient
in 64 bits).  Projections are also checked bit for bit on small whole numbers, whose fp32 sums
are exact in any order; elsewhere the tolerances count roundings: a sum of R terms whose partial
sums stay below A is off by at most about 2^-24 A sqrt(R) (independent roundings of half a step
each, two standard deviations of slack in the constants below), never by a whole code step.
"""
import math

import numpy as np
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative


def _gen(seed):
    return np.random.default_rng(seed)


def _dev(a, gpu):
    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


# ---- plain forms ------------------------------------------------------------------------


def _bf16_steps(x, how):
    """x (float64) on the bf16 grid (8 significant bits, steps of 2^-133 at least), rounded by
    `how`."""
    _, e = np.frexp(x)
    e = np.maximum(e, -125) - 8
    return np.ldexp(how(np.ldexp(x, -e)), e)


def ref_weight(W, G):
    """What the codes and scales of W (N, K) stand for: (W~ float64, scales (N, K) float64)."""
    out, sc = np.zeros(W.shape), np.zeros(W.shape)
    with np.errstate(all="ignore"):
        for k in range(0, W.shape[1], G):
            w = W[:, k:k + G].astype(np.float64)
            v = np.take_along_axis(w, np.argmax(np.abs(w), 1)[:, None], 1)
            s = _bf16_steps(v / -8.0, np.rint)
            q = np.where(s != 0, np.clip(np.rint(w / np.where(s != 0, s, 1.0)), -8, 7), 0.0)
            s = np.where(np.isfinite(w).all(1, keepdims=True), s, np.nan)
            out[:, k:k + G], sc[:, k:k + G] = q * s, s
    return out, sc


def ref_cache(x):
    """What the cache holds of x (..., hd): (x~, s, z), float64, per channel."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, 64)
    with np.errstate(all="ignore"):
        z = _bf16_steps(g.min(-1, keepdims=True), np.floor)
        s = _bf16_steps((g.max(-1, keepdims=True) - z) / 15.0, np.ceil)
        q = np.where(s > 0, np.clip(np.rint((g - z) / np.where(s > 0, s, 1.0)), 0, 15), 0.0)
        bad = ~np.isfinite(g).all(-1, keepdims=True) | ~(np.abs(z) + 16 * s < 3.4e38)
        v = np.where(bad, np.nan, z + s * q)
    full = np.ones_like(g)
    return tuple((a * full).reshape(x.shape) for a in (v, s, z))


def ref_attention(q, k, v, lens, heads, scale, causal):
    """q (B, Tq, heads * hd), k / v (B, rows, kv, hd) float64."""
    B, Tq = q.shape[:2]
    kv, hd = k.shape[2:]
    rep = heads // kv
    o = np.zeros((B, Tq, heads, hd))
    qh = q.astype(np.float64).reshape(B, Tq, heads, hd)
    for b in range(B):
        for t in range(Tq):
            n = max(0, lens[b] - Tq + t + 1) if causal else lens[b]
            for h in range(heads if n else 0):
                s = scale * (k[b, :n, h // rep] @ qh[b, t, h])
                p = np.exp(s - s.max())
                o[b, t, h] = (p / p.sum()) @ v[b, :n, h // rep]
    return o.reshape(B, Tq, heads * hd)


def _weights(rng, N, K, G):
    """A layer's weights with what a quantiser can trip over: a zero group, equal magnitudes of
    both signs, a lone large value, tiny and huge groups."""
    W = (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32)
    W[0, :G] = 0.0
    if N > 3:
        W[1, :G] = 0.25
        W[1, :G:2] = -0.25
        W[2] *= 1e-42 / 0.01
        W[3] *= 1e37
    W[-1, -1] = 7.0
    return W


# ---- weights ----------------------------------------------------------------------------


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 4), (5, 60), (16, 128), (17, 132), (33, 896), (6761, 36)])
def test_pack_unpack_equal_the_definition(gpu, N, K, G):
    from larynx_amd import ops
    announce(f"q4 pack N={N} K={K} G={G}")
    W = _weights(_gen(N + K + G), N, K, G)
    w = ops.q4_pack(_dev(W, gpu), G)
    got = ops.q4_unpack(w).cpu().numpy()
    ref, _ = ref_weight(W, G)
    assert np.array_equal(got.astype(np.float64), ref)


def test_pack_groups_with_infinities_stand_for_nan(gpu):
    from larynx_amd import ops
    announce("q4 pack non-finite")
    W = _gen(3).standard_normal((18, 256)).astype(np.float32)
    W[2, 70], W[5, 3], W[17, 255] = np.inf, np.nan, -np.inf
    got = ops.q4_unpack(ops.q4_pack(_dev(W, gpu), 64)).cpu().numpy().astype(np.float64)
    ref, _ = ref_weight(W, 64)
    assert np.array_equal(got, ref, equal_nan=True)
    assert np.isnan(got).sum() == 3 * 64


def _exact_weights(rng, N, K, G):
    """Whole multiples -8 .. 7 of a power of two per group, -8 first in each: packed exactly."""
    W = np.zeros((N, K), np.float32)
    for k in range(0, K, G):
        n = min(G, K - k)
        q = rng.integers(-8, 8, (N, n))
        q[:, 0] = -8
        W[:, k:k + n] = q * 2.0 ** rng.integers(-3, 1, (N, 1))
    return W


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 5, 6, 16, 17, 33, 48, 64])
@pytest.mark.parametrize("N,K", [(1, 4), (15, 60), (16, 128), (130, 132), (1152, 896),
                                 (97, 4864)])
def test_linear_bit_exact_on_whole_numbers(gpu, M, N, K, G):
    """x in -3 .. 3: every partial sum is a multiple of 1/8 below 2^21 (31 * 3 * 4864 with the
    offset), so fp32 holds it exactly whatever the order.  x and out are views with padding."""
    from larynx_amd import ops
    announce(f"q4 linear exact M={M} N={N} K={K} G={G}")
    rng = _gen(M * N + K + G)
    W = _exact_weights(rng, N, K, G)
    x = rng.integers(-3, 4, (M, K)).astype(np.float32)
    xd = torch.full((M + 1, K + 8), float("nan"), device=gpu)
    xd[:M, :K] = _dev(x, gpu)
    out = torch.full((M + 2, N + 3), -77.0, device=gpu)
    b = rng.integers(-9, 10, N).astype(np.float32)
    w = ops.q4_pack(_dev(W, gpu), G)
    ops.linear_q4(xd[:M, :K], w, _dev(b, gpu), out=out[:M, :N])
    got = out.cpu().numpy()
    assert np.array_equal(got[:M, :N], (x.astype(np.float64) @ W.T.astype(np.float64)) + b)
    assert (got[M:] == -77).all() and (got[:, N:] == -77).all()


@pytest.mark.parametrize("M,N,K,G", [
    (1, 90004, 896, 64), (4, 151936, 896, 32), (7, 33000, 700, 128),   # few rows, many tiles
    (3, 70000, 1100, 64), (8, 9000, 2500, 64), (6, 3000, 2500, 32),    # and past 1024 inputs
    (5, 40000, 1100, 64),
    (16, 9999, 896, 64), (12, 300, 4100, 32), (16, 2500, 8192, 128), (9, 17, 1028, 128),
    (31, 70, 8192, 64), (17, 40001, 260, 64), (32, 5000, 2000, 128),
    (40, 33, 1028, 32), (48, 4097, 1500, 64), (64, 3000, 3000, 32), (64, 20000, 512, 64),
    (64, 130, 8192, 128)])
def test_linear_bit_exact_on_larger_shapes(gpu, M, N, K, G):
    """As above, on the shapes of the kernel that shares x: whole numbers, against torch in 64 bits
    on the device; columns past N and rows past M untouched."""
    from larynx_amd import ops
    announce(f"q4 linear exact, larger M={M} N={N} K={K} G={G}")
    g = torch.Generator(device=gpu).manual_seed(M + N + K)
    W = torch.randint(-8, 8, (N, K), device=gpu, generator=g).float()
    W[:, ::G] = -8
    x = torch.randint(-3, 4, (M, K), device=gpu, generator=g).float()
    b = torch.randint(-9, 10, (N,), device=gpu, generator=g).float()
    out = torch.full((M + 1, N + 5), -77.0, device=gpu)
    ops.linear_q4(x, ops.q4_pack(W, G), b, out=out[:M, :N])
    want = (x.double() @ W.t().contiguous().double() + b).float()
    assert torch.equal(out[:M, :N], want)
    assert (out[M:] == -77).all() and (out[:, N:] == -77).all()


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 4, 7, 8, 16, 33, 64])
@pytest.mark.parametrize("N,K", [(200, 132), (1152, 896), (97, 4864), (60000, 900)])
def test_linear_every_bit_of_x(gpu, M, N, K, G):
    """Whole numbers of 20 bits and both signs, a single weight a row: each output is one product,
    exact in fp32, and x's two fp16 parts hold it exactly (11 bits each, and 2^-24 of the largest of
    a block is below 1)."""
    from larynx_amd import ops
    announce(f"q4 linear bits of x M={M} N={N} K={K} G={G}")
    g = torch.Generator(device=gpu).manual_seed(M * N + K + G)
    at = torch.randint(0, K, (N,), device=gpu, generator=g)
    val = -8.0 * 2.0 ** torch.randint(-3, 4, (N,), device=gpu, generator=g)
    W = torch.zeros(N, K, device=gpu)
    W[torch.arange(N, device=gpu), at] = val
    x = torch.randint(-2 ** 20 + 1, 2 ** 20, (M, K), device=gpu, generator=g).float()
    got = ops.linear_q4(x, ops.q4_pack(W, G))
    assert torch.equal(got, x[:, at] * val)


@pytest.mark.parametrize("M", [2, 20])
def test_linear_far_offsets(gpu, M):
    """A weight of 4.3 GB of codes (34 GB in fp32), the last rows other than zero: offsets past 32
    bits in packing and in the product."""
    from larynx_amd import ops
    announce(f"q4 far offsets M={M}")
    N, K, n = (1 << 20) + 24, 8192, 40
    g = torch.Generator(device=gpu).manual_seed(M)
    W = torch.zeros(N, K, device=gpu)
    W[-n:] = torch.randint(-8, 8, (n, K), device=gpu, generator=g).float()
    W[-n:, ::64] = -8
    w = ops.q4_pack(W, 64)
    assert w.data.numel() > 1 << 32
    x = torch.randint(-3, 4, (M, K), device=gpu, generator=g).float()
    got = ops.linear_q4(x, w)
    want = (x.double() @ W[-n:].t().contiguous().double()).float()
    del W
    assert torch.equal(got[:, -n:], want)
    assert not got[:, :-n].any()


def _linear_tolerance(x, sc, G):
    """Per output: the group sums run through 4 G / 8 accumulations (three parts and the sum of
    x) of partial sums below (24 + 31) sum |x| times the scale, then over the groups."""
    K = x.shape[1]
    A = 55.0 * (np.abs(x).astype(np.float64) @ np.abs(sc).T)
    return 4.0 * U * A * math.sqrt(4 * G + K / G) / math.sqrt(K / min(G, K))


@pytest.mark.parametrize("epi", ["none", "gelu", "resid", "swiglu"])
@pytest.mark.parametrize("M,N,K,G", [(1, 9728, 896, 64), (3, 6762, 896, 32), (4, 896, 4864, 64),
                                     (5, 70, 1000, 128), (16, 384, 2048, 128), (29, 46, 772, 64),
                                     (64, 258, 516, 32)])
def test_linear_epilogues(gpu, epi, M, N, K, G):
    from larynx_amd import ops
    announce(f"q4 linear {epi} M={M} N={N} K={K} G={G}")
    rng = _gen(M + N + K)
    W = (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0] *= 1e3
    b = rng.standard_normal(N).astype(np.float32)
    y = rng.standard_normal((M, N)).astype(np.float32)
    ref, sc = ref_weight(W, G)
    acc = x.astype(np.float64) @ ref.T + b
    tol = _linear_tolerance(x, sc, G) + 2 * U * np.abs(acc)
    out, e = None, None
    if epi == "gelu":
        # derivative within 1.13, and 8 roundings in the formula
        e = ops.Epilogue(kind=ops.LX_EPI_GELU_TANH)
        want = 0.5 * acc * (1 + np.tanh(0.7978845608028654 * (acc + 0.044715 * acc ** 3)))
        # exponents up to 2 |u|: a rounding of u moves the factor by u |u| while it is not 0 or 1
        tol = 1.13 * tol + 64 * U * (np.abs(acc) + 1)
    elif epi == "resid":
        e, out = ops.Epilogue(kind=ops.LX_EPI_RESID), _dev(y, gpu)
        want = y + acc
        tol = tol + U * np.abs(want)
    elif epi == "swiglu":
        e = ops.Epilogue(kind=ops.LX_EPI_SWIGLU_PAIRED)
        g, u = acc[:, 0::2], acc[:, 1::2]
        sg = 1 / (1 + np.exp(-np.clip(g, -700, None)))
        want = g * sg * u
        tol = (1.1 * tol[:, 0::2] * np.abs(u) + np.abs(g * sg) * tol[:, 1::2] +
               64 * U * (np.abs(want) + np.abs(u)))
    else:
        want = acc
    got = ops.linear_q4(_dev(x, gpu), ops.q4_pack(_dev(W, gpu), G), _dev(b, gpu), epilogue=e,
                        out=out).cpu().numpy()
    err = np.abs(got - want)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("M", [3, 7, 40])
def test_linear_nan_stays_in_its_row(gpu, M):
    from larynx_amd import ops
    announce(f"q4 linear NaN row M={M}")
    rng = _gen(M)
    W = rng.standard_normal((40, 256)).astype(np.float32)
    x = rng.standard_normal((M, 256)).astype(np.float32)
    w = ops.q4_pack(_dev(W, gpu))
    clean = ops.linear_q4(_dev(x, gpu), w)
    for bad in (np.nan, np.inf):
        x2 = x.copy()
        x2[1, 9] = bad
        got = ops.linear_q4(_dev(x2, gpu), w)
        assert torch.isnan(got[1]).all()
        keep = [m for m in range(M) if m != 1]
        assert torch.equal(got[keep], clean[keep])


# ---- cache ------------------------------------------------------------------------------


def _rows(rng, *shape):
    """Rows with offset channels, and what a quantiser can trip over."""
    x = rng.standard_normal(shape).astype(np.float32)
    x[..., ::16] += 30.0
    flat = x.reshape(-1, shape[-1])
    flat[0] = 3.14159       # no range
    if len(flat) > 4:
        flat[1] = 0.0
        flat[2] = np.linspace(-1.0, 1.0, shape[-1])  # ties
        flat[3] *= 1e-40
        flat[4] *= 1e35
    return x


@pytest.mark.parametrize("hd,kv", [(64, 2), (64, 5), (128, 1), (128, 3)])
@pytest.mark.parametrize("T,pos", [(1, [0, 7]), (1, [31, 32]), (3, [30, 95]), (40, [0, 17]),
                                   (97, [3, 31])])
def test_append_equals_the_definition_and_leaves_other_rows(gpu, hd, kv, T, pos):
    from larynx_amd import ops
    announce(f"kv4 append hd={hd} kv={kv} T={T} pos={pos}")
    rng = _gen(hd + kv + T)
    B, rows = 2, 130
    cache = ops.kv4_cache(B, kv, rows, hd)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    old_k, old_v = _rows(rng, B, rows, kv * hd), _rows(rng, B, rows, kv * hd)
    ops.kv4_append(cache, _dev(old_k, gpu), _dev(old_v, gpu), zero)
    # strided views: k and v as column ranges of one fused row
    fused = np.concatenate([_rows(rng, B, T, kv * hd), _rows(rng, B, T, kv * hd)], -1)
    fd = _dev(fused, gpu)
    ops.kv4_append(cache, fd[..., :kv * hd], fd[..., kv * hd:], torch.tensor(
        pos, dtype=torch.int32, device=gpu))
    k, v = (a.cpu().numpy() for a in ops.kv4_read(cache, zero, rows))
    for b in range(B):
        n = min(T, rows - pos[b])
        old_k[b, pos[b]:pos[b] + n] = fused[b, :n, :kv * hd]
        old_v[b, pos[b]:pos[b] + n] = fused[b, :n, kv * hd:]
    for got, src in ((k, old_k), (v, old_v)):
        ref = ref_cache(src.reshape(B, rows, kv, hd))[0].reshape(B, rows, kv * hd)
        assert np.array_equal(got.astype(np.float64), ref.astype(np.float32))


def test_append_codes_next_to_borders(gpu):
    """Values on the borders between codes and one step of fp32 to either side, under scales of
    many sizes, subnormal ones too: where a quotient taken in 32 bits could fall either way."""
    from larynx_amd import ops
    announce("kv4 append borders")
    rng = _gen(21)
    rows = 2000
    s = (2.0 ** rng.integers(-20, 20, (rows, 1)) * (1 + rng.integers(0, 128, (rows, 1)) / 128))
    s[-200:] = 2.0 ** -133 * rng.integers(1, 200, (200, 1))
    z = np.float32(s * rng.integers(-128, 128, (rows, 1)) * 2.0 ** rng.integers(-3, 3, (rows, 1)))
    z = np.float32(_bf16_steps(z.astype(np.float64), np.floor))
    q = rng.integers(0, 15, (rows, 64)) + rng.choice([0.0, 0.5, 0.5], (rows, 64))
    x = np.float32(z + s * q)
    x = np.where(rng.random(x.shape) < 0.3, np.nextafter(x, np.float32(np.inf)), x)
    x = np.where(rng.random(x.shape) < 0.3, np.nextafter(x, np.float32(-np.inf)), x)
    x[:, 0], x[:, 1] = z[:, 0], np.float32(z + 15 * s)[:, 0]
    x = x.astype(np.float32)[None]
    cache = ops.kv4_cache(1, 1, rows)
    zero = torch.zeros(1, dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, _dev(x, gpu), _dev(-x, gpu), zero)
    for got, src in zip(ops.kv4_read(cache, zero, rows), (x, -x)):
        ref = ref_cache(src.reshape(1, rows, 1, 64))[0].reshape(1, rows, 64)
        assert np.array_equal(got.cpu().numpy(), ref.astype(np.float32))


def test_append_outside_the_cache_writes_nothing(gpu):
    from larynx_amd import ops
    announce("kv4 append outside")
    rng = _gen(4)
    cache = ops.kv4_cache(4, 2, 50)
    cache.data.fill_(0x5A)
    before = cache.data.clone()
    x = _dev(_rows(rng, 4, 3, 128), gpu)
    far = torch.tensor([-3, 64, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, x, x, far)
    assert torch.equal(cache.data, before)
    # rows 50 .. 63 exist in the last record but not in the cache; a row before the first
    edge = torch.tensor([49, 50, -2, -3], dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, x, x, edge)
    k, _ = ops.kv4_read(cache, edge, 3)
    ref = ref_cache(x.cpu().numpy().reshape(4, 3, 2, 64))[0].reshape(4, 3, 128)
    got = k.cpu().numpy()
    assert np.array_equal(got[0, 0], ref[0, 0].astype(np.float32)) and not got[0, 1:].any()
    assert not got[1].any()
    assert np.array_equal(got[2, 2], ref[2, 2].astype(np.float32)) and not got[2, :2].any()
    rec = cache.data.view(4, -1)
    assert torch.equal(rec[1], before.view(4, -1)[1])
    assert torch.equal(rec[3], before.view(4, -1)[3])


def test_append_groups_with_infinities_stand_for_nan(gpu):
    from larynx_amd import ops
    announce("kv4 append non-finite")
    rng = _gen(5)
    x = rng.standard_normal((1, 40, 128)).astype(np.float32)
    x[0, 3, 5], x[0, 4, 127], x[0, 5, 64] = np.inf, np.nan, -np.inf
    x[0, 6, 0], x[0, 6, 1] = 3.4e38, -3.3e38    # |z| + 16 s passes fp32
    x[0, 7, 0] = -3.4028e38                     # no bf16 below it
    x[0, 8, 0], x[0, 8, 1] = 1.0e38, -1.0e38    # 3.1e38: all of it below fp32's largest
    cache = ops.kv4_cache(1, 2, 40)
    zero = torch.zeros(1, dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, _dev(x, gpu), _dev(x, gpu), zero)
    ref = ref_cache(x.reshape(1, 40, 2, 64))[0].reshape(1, 40, 128).astype(np.float32)
    for got in ops.kv4_read(cache, zero, 40):
        assert np.array_equal(got.cpu().numpy(), ref, equal_nan=True)
    assert np.isnan(ref).sum() == 5 * 64


# ---- attention --------------------------------------------------------------------------


def _attn_case(gpu, rng, B, Tq, heads, kv, hd, rows, lens):
    from larynx_amd import ops
    k = rng.standard_normal((B, rows, kv * hd)).astype(np.float32)
    v = rng.standard_normal((B, rows, kv * hd)).astype(np.float32)
    k[..., ::16] += 4.0
    q = rng.standard_normal((B, Tq, heads * hd)).astype(np.float32) * 2
    cache = ops.kv4_cache(B, kv, rows, hd)
    cache.data.fill_(0xFF)  # rows never appended: scales that are NaN
    for b in range(B):      # only the rows in use
        if lens[b]:
            one = ops.Kv4Cache(cache.data.view(B, -1)[b], 1, kv, hd, rows)
            ops.kv4_append(one, _dev(k[b:b + 1, :lens[b]], gpu), _dev(v[b:b + 1, :lens[b]], gpu),
                           torch.zeros(1, dtype=torch.int32, device=gpu))
    return q, k.reshape(B, rows, kv, hd), v.reshape(B, rows, kv, hd), cache


def _attn_tolerance(q, k, v, heads, scale, splits_roundings=64):
    """Scores: sums of hd products of three parts whose partial sums stay below B; a score off by
    d scales its weight by 1 + d; weights, scales and the joined sums round about 64 times."""
    kt, ks, kz = ref_cache(k)
    vt, vs, vz = ref_cache(v)
    hd = k.shape[-1]
    qa = np.abs(q).reshape(q.shape[0], q.shape[1], heads, hd)
    top = (np.abs(kz) + 47 * ks).max((0, 1))                       # (kv, hd)
    Bd = scale * (qa * np.repeat(top, heads // k.shape[2], 0)).sum(-1).max()
    vmax = (np.abs(vz) + 47 * vs).max()
    return vmax * U * (2 * 4 * Bd * math.sqrt(3 * hd / 8) / math.sqrt(hd / 8) +
                       splits_roundings)


CASES = [
    # B, Tq, heads, kv, hd, rows, lens, max_len
    (1, 1, 14, 2, 64, 2100, [2001], 0),
    (1, 1, 14, 2, 64, 40, [1], 0),
    (3, 1, 14, 2, 64, 70, [0, 33, 64], 70),
    (2, 1, 16, 16, 64, 200, [200, 31], 0),
    (2, 1, 8, 1, 128, 300, [257, 32], 300),
    (1, 1, 32, 8, 128, 1100, [1055], 0),
    (2, 3, 14, 2, 64, 90, [90, 2], 0),        # two queries of the second see nothing
    (1, 5, 48, 3, 64, 130, [129], 130),       # 16 heads a group, 80 query rows
    (2, 40, 14, 2, 64, 129, [129, 40], 0),
    (1, 177, 14, 2, 64, 400, [333], 0),
    (1, 33, 4, 4, 128, 64, [33], 0),
    (2, 70, 2, 2, 64, 65, [65, 65], 0),       # more queries than rows
    (9, 1, 14, 2, 64, 5000, [5000, 0, 1, 31, 32, 33, 64, 4999, 2500], 5000),
    (2, 1, 14, 2, 64, 3000, [3000, 2999], 10),  # a hint far too small
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
def test_attention(gpu, case, causal):
    from larynx_amd import ops
    B, Tq, heads, kv, hd, rows, lens, max_len = case
    announce(f"kv4 attention {case} causal={causal}")
    rng = _gen(sum(case[:6]))
    q, k, v, cache = _attn_case(gpu, rng, B, Tq, heads, kv, hd, rows, lens)
    buf = torch.full((B, Tq, heads * hd + 8), -77.0, device=gpu)
    ld = torch.tensor(lens, dtype=torch.int32, device=gpu)
    qd = torch.full((B, Tq, heads * hd + 4), float("nan"), device=gpu)
    qd[..., :heads * hd] = _dev(q, gpu)
    ops.attention_kv4(qd[..., :heads * hd], cache, ld, heads, causal=causal,
                      out=buf[..., :heads * hd], max_len=max_len)
    got = buf.cpu().numpy()
    want = ref_attention(q, ref_cache(k)[0], ref_cache(v)[0], lens, heads, hd ** -0.5, causal)
    err = np.abs(got[..., :heads * hd] - want).max()
    tol = _attn_tolerance(q, k, v, heads, hd ** -0.5)
    assert err <= tol, (err, tol)
    assert (got[..., heads * hd:] == -77).all()
    for b in range(B):
        for t in range(Tq):
            if (lens[b] - Tq + t + 1 if causal else lens[b]) <= 0:
                assert not got[b, t, :heads * hd].any()


def test_attention_does_not_see_later_rows(gpu):
    """NaN in a key and a value a later query sees: the queries before it keep their bits."""
    from larynx_amd import ops
    announce("kv4 attention NaN ahead")
    rng = _gen(8)
    B, Tq, heads, kv, hd, rows = 1, 6, 14, 2, 64, 64
    q, k, v, cache = _attn_case(gpu, rng, B, Tq, heads, kv, hd, rows, [50])
    n = torch.tensor([50], dtype=torch.int32, device=gpu)
    clean = ops.attention_kv4(_dev(q, gpu), cache, n, heads)
    bad = torch.full((1, 1, kv * hd), float("nan"), device=gpu)
    ops.kv4_append(cache, bad, bad, torch.tensor([47], dtype=torch.int32, device=gpu))
    got = ops.attention_kv4(_dev(q, gpu), cache, n, heads)
    assert torch.equal(got[:, :3], clean[:, :3])
    assert torch.isnan(got[:, 3:]).all()


@pytest.mark.parametrize("rows,Tq", [(40, 1), (4000, 1), (700, 30)])
def test_attention_nan_stays_in_its_query(gpu, rows, Tq):
    """A query with a NaN or an infinity makes NaN of its row and head, split keys or not, and of
    nothing else."""
    from larynx_amd import ops
    announce(f"kv4 attention NaN query rows={rows} Tq={Tq}")
    rng = _gen(rows)
    q, k, v, cache = _attn_case(gpu, rng, 2, Tq, 14, 2, 64, rows, [rows, rows])
    n = torch.tensor([rows, rows], dtype=torch.int32, device=gpu)
    clean = ops.attention_kv4(_dev(q, gpu), cache, n, 14)
    for bad in (np.nan, np.inf):
        q2 = q.copy()
        q2[1, Tq // 2, 5 * 64 + 3] = bad
        got = ops.attention_kv4(_dev(q2, gpu), cache, n, 14)
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[1, Tq // 2, 5 * 64:6 * 64] = True
        assert torch.isnan(got[hit]).all()
        assert torch.equal(got[~hit], clean[~hit])


def test_attention_lengths_outside_the_cache(gpu):
    from larynx_amd import ops
    announce("kv4 attention lengths clamped")
    rng = _gen(9)
    q, k, v, cache = _attn_case(gpu, rng, 2, 1, 4, 2, 64, 50, [50, 50])
    a = ops.attention_kv4(_dev(q, gpu), cache, torch.tensor([50, 0], dtype=torch.int32,
                                                            device=gpu), 4)
    b = ops.attention_kv4(_dev(q, gpu), cache, torch.tensor(
        [2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=gpu), 4)
    assert torch.equal(a, b) and not a[1].any()


@pytest.mark.parametrize("hd,heads,kv,Tq", [(64, 64, 8, 200), (128, 32, 8, 100), (64, 14, 2, 1),
                                            (64, 16, 16, 3), (128, 32, 8, 1)])
def test_attention_every_weight(gpu, hd, heads, kv, Tq):
    """Six keys with scores within 2 of each other, so that each weight of each row counts in the
    output: scores are off by 2^-24 of sums below 8 sqrt(3 hd) roundings at most, a weight's two
    parts by 2^-22, the rest by some ten roundings.  (A weight that lost its second part would be
    off by up to 2^-11.)"""
    from larynx_amd import ops
    announce(f"kv4 attention every weight hd={hd} heads={heads}/{kv} Tq={Tq}")
    rng = _gen(hd + heads)
    B, rows = (8, 6) if Tq > 1 else (64, 6)
    k = (rng.standard_normal((B, rows, kv, hd)) * 0.2).astype(np.float32)
    v = rng.standard_normal((B, rows, kv, hd)).astype(np.float32)
    q = rng.standard_normal((B, Tq, heads * hd)).astype(np.float32)
    cache = ops.kv4_cache(B, kv, rows, hd)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, _dev(k.reshape(B, rows, -1), gpu), _dev(v.reshape(B, rows, -1), gpu),
                   zero)
    got = ops.attention_kv4(_dev(q, gpu), cache, zero + rows, heads, causal=False).cpu().numpy()
    kt, vt = ref_cache(k)[0], ref_cache(v)[0]
    rep = heads // kv
    s = np.einsum("btgrc,bkgc->btgrk", q.astype(np.float64).reshape(B, Tq, kv, rep, hd),
                  kt) * hd ** -0.5
    p = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("btgrk,bkgc->btgrc", p / p.sum(-1, keepdims=True), vt).reshape(got.shape)
    assert np.abs(s).max() < 2.5
    vmax = np.abs(vt).max()
    tol = vmax * (U * (2 * 8 * math.sqrt(3 * hd) / math.sqrt(hd) + 16) + 2.0 ** -22)
    assert np.abs(got - want).max() < tol, (np.abs(got - want).max(), tol)


@pytest.mark.parametrize("hd,heads,kv,Tq,rows", [(64, 14, 2, 1, 37), (64, 16, 16, 1, 600),
                                                 (128, 32, 8, 3, 200), (64, 14, 2, 50, 300),
                                                 (128, 8, 1, 1, 3000)])
def test_attention_does_not_drift(gpu, hd, heads, kv, Tq, rows):
    """Weights of all sizes, down to e^-20.  The bound of test_attention_every_weight, for scores up
    to S, is eight times what roundings that go either way come to: their root mean square is an
    eighth of it, and their mean over N outputs sqrt(N) times less.  Sums that drop bits on one
    side are off by little, but everywhere and alike."""
    from larynx_amd import ops
    announce(f"kv4 attention drift hd={hd} heads={heads}/{kv} Tq={Tq} rows={rows}")
    rng = _gen(hd + heads + rows)
    B = 2 if Tq > 1 else 6
    k = rng.standard_normal((B, rows, kv, hd)).astype(np.float32)
    v = rng.standard_normal((B, rows, kv, hd)).astype(np.float32)
    q = (2 * rng.standard_normal((B, Tq, heads * hd))).astype(np.float32)
    cache = ops.kv4_cache(B, kv, rows, hd)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    ops.kv4_append(cache, _dev(k.reshape(B, rows, -1), gpu), _dev(v.reshape(B, rows, -1), gpu),
                   zero)
    got = ops.attention_kv4(_dev(q, gpu), cache, zero + rows, heads, causal=False).cpu().numpy()
    kt, vt = ref_cache(k)[0], ref_cache(v)[0]
    want = ref_attention(q, kt, vt, [rows] * B, heads, hd ** -0.5, False)
    S = np.abs(np.einsum("btgrc,bkgc->btgrk", q.astype(np.float64).reshape(
        B, Tq, kv, heads // kv, hd), kt)).max() * hd ** -0.5
    one = np.abs(vt).max() * (U * (28 * S + 16) + 2.0 ** -22)
    err = got - want
    assert math.sqrt((err ** 2).mean()) < one / 8, (math.sqrt((err ** 2).mean()), one)
    assert abs(err.mean()) < one / math.sqrt(err.size), (err.mean(), one, err.size)


def test_attention_large_scores(gpu):
    """Scores in the hundreds, rising along the keys: the running maximum moves in every record."""
    from larynx_amd import ops
    announce("kv4 attention large scores")
    rng = _gen(10)
    rows, hd = 300, 64
    k = rng.standard_normal((1, rows, hd)).astype(np.float32) * 0.1
    k += np.linspace(0, 40, rows, dtype=np.float32)[None, :, None]
    v = rng.standard_normal((1, rows, hd)).astype(np.float32)
    q = np.full((1, 1, hd), 1.0, np.float32)
    cache = ops.kv4_cache(1, 1, rows, hd)
    ops.kv4_append(cache, _dev(k, gpu), _dev(v, gpu), torch.zeros(1, dtype=torch.int32,
                                                                  device=gpu))
    got = ops.attention_kv4(_dev(q, gpu), cache, torch.tensor([rows], dtype=torch.int32,
                                                              device=gpu), 1).cpu().numpy()
    k4, v4 = k.reshape(1, rows, 1, hd), v.reshape(1, rows, 1, hd)
    want = ref_attention(q, ref_cache(k4)[0], ref_cache(v4)[0], [rows], 1, hd ** -0.5, True)
    assert np.abs(got - want).max() <= _attn_tolerance(q, k4, v4, 1, hd ** -0.5)


def test_far_offsets(gpu):
    """The last sequence of a 9.7 GB cache, near its last row: offsets past 32 bits."""
    from larynx_amd import ops
    announce("kv4 far offsets")
    rng = _gen(11)
    B, kv, hd, rows = 8, 8, 128, 1 << 20
    cache = ops.kv4_cache(B, kv, rows, hd)
    assert cache.data.numel() > 1 << 33
    T = 70
    k = rng.standard_normal((B, T, kv * hd)).astype(np.float32)
    v = rng.standard_normal((B, T, kv * hd)).astype(np.float32)
    pos = torch.full((B,), rows - T, dtype=torch.int32, device=gpu)
    pos[0] = 0
    ops.kv4_append(cache, _dev(k, gpu), _dev(v, gpu), pos)
    gk, gv = ops.kv4_read(cache, pos, T)
    for got, src in ((gk, k), (gv, v)):
        ref = ref_cache(src.reshape(B, T, kv, hd))[0].reshape(B, T, kv * hd)
        assert np.array_equal(got.cpu().numpy().astype(np.float64), ref.astype(np.float32))
    # attention over the whole of the last sequence, the rows before holding zeros
    last = ops.Kv4Cache(cache.data.view(B, -1)[B - 1], 1, kv, hd, rows)
    heads = last.data.view(kv, -1)  # each head's records are a run of their own
    heads[:, :heads.shape[1] // rows * (rows - 128)].zero_()
    z = torch.zeros(1, 128 - T, kv * hd, device=gpu)
    ops.kv4_append(last, z, z, torch.tensor([rows - 128], dtype=torch.int32, device=gpu))
    q = rng.standard_normal((B, 1, kv * hd)).astype(np.float32)
    lens = torch.zeros(B, dtype=torch.int32, device=gpu)
    lens[B - 1] = rows
    got = ops.attention_kv4(_dev(q, gpu), cache, lens, kv, scale=2.0).cpu().numpy()
    kt, vt = (ref_cache(a[B - 1].reshape(T, kv, hd))[0] for a in (k, v))
    for h in range(kv):
        s = 2.0 * (kt[:, h] @ q[B - 1, 0, h * hd:(h + 1) * hd].astype(np.float64))
        top = max(s.max(), 0.0)
        p = np.exp(s - top)
        want = p @ vt[:, h] / (p.sum() + (rows - T) * np.exp(-top))
        assert np.abs(got[B - 1, 0, h * hd:(h + 1) * hd] - want).max() < 2e-4 * np.abs(want).max()
    assert not got[:B - 1].any()


# ---- together ---------------------------------------------------------------------------


def _layer(ops, st, x, pos, lens, Tq):
    """One attention layer of a decoder: projection -> append -> attention -> o_proj + residual."""
    qkv = ops.linear_q4(x, st["qkv"], st["b"])
    B = pos.numel()
    H, KV = st["heads"] * 64, st["kv"] * 64
    rows = qkv.view(B, Tq, H + 2 * KV)
    ops.kv4_append(st["cache"], rows[..., H:H + KV], rows[..., H + KV:], pos)
    att = ops.attention_kv4(rows[..., :H], st["cache"], lens, st["heads"])
    ops.linear_q4(att.view(B * Tq, H), st["o"], epilogue=st["resid"], out=x)
    return x


def _layer_state(gpu, rng, B, rows, heads=14, kv=2):
    from larynx_amd import ops
    H = heads * 64
    Wq = (rng.standard_normal((H + 2 * kv * 64, H)) * H ** -0.5).astype(np.float32)
    Wo = (rng.standard_normal((H, H)) * H ** -0.5).astype(np.float32)
    b = (rng.standard_normal(H + 2 * kv * 64) * 0.1).astype(np.float32)
    st = dict(heads=heads, kv=kv, qkv=ops.q4_pack(_dev(Wq, gpu)), o=ops.q4_pack(_dev(Wo, gpu)),
              b=_dev(b, gpu), cache=ops.kv4_cache(B, kv, rows),
              resid=ops.Epilogue(kind=ops.LX_EPI_RESID))
    return st, ref_weight(Wq, 64)[0], ref_weight(Wo, 64)[0], b


def test_layer_together(gpu):
    """A prompt of 20 rows, then single tokens, two sequences: each step against 64 bits, fed with
    the GPU's own projected rows (a rounding next to a code's border is a whole step of the
    cache, so the cache's input is taken as given)."""
    from larynx_amd import ops
    announce("four-bit layer, prompt and tokens")
    rng = _gen(12)
    B, rows = 2, 64
    st, Wq, Wo, b = _layer_state(gpu, rng, B, rows)
    H, KV = 896, 128
    ck, cv = np.zeros((B, rows, 2, 64)), np.zeros((B, rows, 2, 64))
    at = 0
    for Tq in (20, 1, 1, 3, 1):
        x0 = rng.standard_normal((B * Tq, H)).astype(np.float32)
        x = _dev(x0, gpu)
        got_qkv = ops.linear_q4(x, st["qkv"], st["b"]).cpu().numpy()
        want = x0.astype(np.float64) @ Wq.T + b
        assert np.abs(got_qkv - want).max() < 1e-5 * np.abs(want).max()
        pos = torch.full((B,), at, dtype=torch.int32, device=gpu)
        at += Tq
        y = _layer(ops, st, x, pos, pos + Tq, Tq).cpu().numpy()
        r = got_qkv.reshape(B, Tq, -1)
        ck[:, at - Tq:at] = ref_cache(r[..., H:H + KV].reshape(B, Tq, 2, 64))[0]
        cv[:, at - Tq:at] = ref_cache(r[..., H + KV:].reshape(B, Tq, 2, 64))[0]
        att = ref_attention(r[..., :H], ck, cv, [at] * B, 14, 0.125, True).reshape(B * Tq, H)
        want = x0 + att @ Wo.T
        assert np.abs(y - want).max() < 1e-5 * np.abs(want).max()


def test_layer_in_a_graph(gpu):
    """The layer captured once and replayed over growing lengths (device counters), with eager work
    between: every replay gives the eager bits."""
    from larynx_amd import ops
    announce("four-bit layer in a graph")
    rng = _gen(13)
    B, rows = 3, 2500
    st, *_ = _layer_state(gpu, rng, B, rows)
    ref = dict(st, cache=ops.kv4_cache(B, 2, rows))
    fill = _dev(_rows(rng, B, 2100, 128), gpu)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    for c in (st["cache"], ref["cache"]):
        ops.kv4_append(c, fill, fill, zero)
    x = torch.zeros(B, 896, device=gpu)
    pos = torch.tensor([2000, 5, 31], dtype=torch.int32, device=gpu)
    lens = pos + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(ops, st, x.clone(), pos, lens, 1)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = _layer(ops, st, x, pos, lens, 1)
    for step in range(5):
        x0 = torch.from_numpy(rng.standard_normal((B, 896)).astype(np.float32)).to(gpu)
        want = _layer(ops, ref, x0.clone(), pos, lens, 1)
        x.copy_(x0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), step
        pos += 1
        lens += 1


@pytest.mark.parametrize("M,N,K,G", [(2, 300, 2000, 64), (48, 520, 2052, 32), (64, 9000, 500, 128),
                                     (7, 33000, 1028, 64)])
def test_products_in_two_graphs(gpu, M, N, K, G):
    """Two graphs of the same weight, captured without a call before them, replayed in turn with
    eager calls between: each replay gives the eager bits, splits and residual included."""
    from larynx_amd import ops
    announce(f"q4 linear in two graphs M={M} N={N} K={K} G={G}")
    g = torch.Generator(device=gpu).manual_seed(M + N)
    w = ops.q4_pack(torch.randn(N, K, device=gpu, generator=g), G)
    resid = ops.Epilogue(kind=ops.LX_EPI_RESID)
    xs = [torch.empty(M, K, device=gpu) for _ in range(2)]
    ys = [torch.zeros(M, N, device=gpu) for _ in range(2)]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, x, y in zip(graphs, xs, ys):
        with torch.cuda.graph(graph):
            ops.linear_q4(x, w, epilogue=resid, out=y)
    for step in range(4):
        want = []
        for x, y in zip(xs, ys):
            x.copy_(torch.randn(M, K, device=gpu, generator=g))
            want.append(ops.linear_q4(x, w, epilogue=resid, out=y.clone()))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for y, b in zip(ys, want):
            assert torch.equal(y, b), step


def test_two_streams_at_once(gpu):
    """Calls of two streams over one cache, both reading, and one weight."""
    from larynx_amd import ops
    announce("four-bit calls on two streams")
    rng = _gen(14)
    q, k, v, cache = _attn_case(gpu, rng, 2, 1, 14, 2, 64, 4000, [4000, 2777])
    lens = torch.tensor([4000, 2777], dtype=torch.int32, device=gpu)
    W = ops.q4_pack(_dev(rng.standard_normal((896, 896)).astype(np.float32), gpu))
    qs = [_dev(q * f, gpu) for f in (1.0, 0.5)]
    want = [ops.linear_q4(ops.attention_kv4(a, cache, lens, 14).view(2, 896), W) for a in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear_q4(ops.attention_kv4(qs[i], cache, lens, 14).view(2, 896),
                                            W))
    torch.cuda.synchronize()
    for i in range(2):
        for a in got[i]:
            assert torch.equal(a, want[i])


def test_python_argument_checks(gpu):
    from larynx_amd import LxError, ops
    announce("four-bit argument checks")
    W = torch.zeros(32, 64, device=gpu)
    with pytest.raises(ValueError):
        ops.q4_pack(W.t())
    with pytest.raises(ValueError):
        ops.q4_pack(W, 48)
    with pytest.raises(ValueError):
        ops.q4_pack(W.half())
    w = ops.q4_pack(W)
    for x in (torch.zeros(1, 60, device=gpu), torch.zeros(1, 64, device=gpu).half(),
              torch.zeros(64, device=gpu), torch.zeros(64, 2, device=gpu).t()):
        with pytest.raises(ValueError):
            ops.linear_q4(x, w)
    with pytest.raises(LxError):
        ops.linear_q4(torch.zeros(65, 64, device=gpu), w)
    with pytest.raises(LxError):
        ops.linear_q4(torch.zeros(0, 64, device=gpu), w)
    x = torch.zeros(2, 64, device=gpu)
    with pytest.raises(ValueError):
        ops.linear_q4(x, w, epilogue=ops.Epilogue(kind=ops.LX_EPI_RESID))
    with pytest.raises(ValueError):
        ops.linear_q4(x, w, b=torch.zeros(31, device=gpu))
    with pytest.raises(ValueError):
        ops.linear_q4(x, w, out=torch.zeros(3, 32, device=gpu))
    cache = ops.kv4_cache(2, 2, 40)
    kv = torch.zeros(2, 1, 128, device=gpu)
    n = torch.zeros(2, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError):
        ops.kv4_append(cache, kv, kv[:, :, :64], n)
    with pytest.raises(ValueError):
        ops.kv4_append(cache, kv, kv, n.long())
    with pytest.raises(ValueError):
        ops.kv4_append(cache, kv[:1], kv[:1], n)
    with pytest.raises(ValueError):
        ops.attention_kv4(kv, cache, n[:1], 2)
    with pytest.raises(ValueError):
        ops.attention_kv4(kv, cache, n, 4)
    with pytest.raises(ValueError):
        ops.attention_kv4(kv, cache, n, 2, out=torch.zeros(2, 2, 128, device=gpu))
    with pytest.raises((ValueError, LxError)):
        ops.kv4_append(cache, kv[:, :0], kv[:, :0], n)
