"""Error bounds of the four-bit operators for the tests, and their arithmetic restated in numpy.

The bounds count roundings of half a step, U = 2^-24 relative, of the partial sums that the
operators form, taken to go either way (root sums of squares).  Errors are divided by the bound of
their own output: their root mean square has to stay below 1 and the largest below 8."""
import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative


def check(err, bound, far=8.0):
    """err and bound, alike in shape.  Outputs whose bound is zero have to be exact."""
    assert np.isfinite(err).all()
    assert not err[bound == 0].any()
    r = (np.abs(err) / np.where(bound == 0, 1.0, bound)).ravel()
    rms = float(np.sqrt((r ** 2).mean()))
    assert rms <= 1.0 and r.max() <= far, (rms, float(r.max()))


def attention(q, k, v, lens, heads, scale, causal):
    """Outputs in 64 bits and their bounds, (B, Tq, heads, hd).  q (B, Tq, heads * hd); k, v: what
    ref_cache gives for (B, rows, kv, hd).

    A score is (8 s + z) sum(q) + s sum(q (code - 8)) a group: every element of q meets at most A =
    |z| + 16 s, in sums of some 60 roundings (8 U); the query's two parts are off by 2^-25 of its
    largest element.  A weight is off by its score's error, by U of its exponent's size twice, by
    the hardware's exp2 and its own rounding (4 U); it moves an output by its value's distance from
    it.  p s, its parts and 8 s + z are off by 2 U of p A.  Outputs are (8 s + z) sum(p) +
    sum(p s (code - 8)), in some 64 + n / 2 roundings of partial sums that go either way; weights
    whose p s is small beside the column's largest end 2^-31 of it apart, times codes up to 8."""
    (kt, ks, kz), (vt, vs, vz) = k, v
    B, Tq = q.shape[:2]
    kv, hd = kt.shape[2:]
    rep = heads // kv
    want, bound = (np.zeros((B, Tq, heads, hd)) for _ in range(2))
    qh = q.astype(np.float64).reshape(B, Tq, heads, hd)
    for b in range(B):
        for g in range(kv):
            ka, va = (np.abs(z[b, :, g]) + 16 * s[b, :, g] for s, z in ((ks, kz), (vs, vz)))
            for t in range(Tq):
                n = min(max(0, lens[b] - Tq + t + 1 if causal else lens[b]), kt.shape[1])
                for h in range(g * rep, (g + 1) * rep if n else 0):
                    x = qh[b, t, h]
                    s = scale * (kt[b, :n, g] @ x)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    e = (8 * U * scale * np.sqrt(ka[:n] ** 2 @ x ** 2) +
                         2.0 ** -25 * scale * np.abs(x).max() * np.sqrt((kt[b, :n, g] ** 2).sum(1)) +
                         2 * U * (s.max() - s) + 4 * U)
                    o = w @ vt[b, :n, g]
                    each = w[:, None] * va[:n]
                    sums = np.abs(o) + np.sqrt((each ** 2).sum(0))
                    want[b, t, h] = o
                    bound[b, t, h] = np.sqrt(
                        (((w * e)[:, None] * (vt[b, :n, g] - o)) ** 2 + (2 * U * each) ** 2).sum(0) +
                        U * U * (64 + n / 2) * sums ** 2 +
                        n * (2.0 ** -28 * (w[:, None] * vs[b, :n, g]).max(0)) ** 2)
    return want, bound


def two_parts(x, parts=2):
    """x as so many fp16 parts, in 64 bits."""
    x = x.astype(np.float32)
    p0 = x.astype(np.float16).astype(np.float32)
    p1 = (x - p0).astype(np.float16) if parts == 2 else np.zeros_like(x)
    return p0.astype(np.float64) + p1.astype(np.float64)


def emulate(q, k, v, scale, parts=2, lift="weights", skip=None):
    """One query row q (hd) over all rows of one head, steps of 32 keys, as a wave forms it: fp32
    statistics and sums, two fp16 parts of the query and of the weights p s.  k, v: (x~, s, z),
    each (n, hd).  lift: what the power of two of the weights' parts follows, the largest product
    ("weights") or the largest scale whatever its weight ("scales").  skip: a key left out."""
    f32 = np.float32
    (_, ks, kz), (_, vs, vz) = k, v
    kq, vq = (np.where(s > 0, np.rint((t - z) / np.where(s > 0, s, 1)), 0) - 8
              for t, s, z in (k, v))
    n, hd = vs.shape
    x = (q.astype(f32) * f32(scale * 1.4426950408889634)).astype(f32)
    f = 2.0 ** np.floor(np.log2(np.abs(x).max()))
    xp = two_parts(x / f32(f), parts)
    s = np.zeros(n, f32)
    for g in range(0, hd, 64):
        c = slice(g, g + 64)
        sg, zg = ks[:, g].astype(f32), kz[:, g].astype(f32)
        dot = (kq[:, c] @ xp[c]).astype(f32)
        s = (s + (sg * dot + (f32(8) * sg + zg) * f32(x[c].sum() / f))).astype(f32)
    if skip is not None:
        s[skip] = -np.inf
    m, l = f32(-np.inf), f32(0)
    o, zsum = np.zeros(hd, f32), np.zeros(hd, f32)
    top = np.zeros(hd // 64)  # of p s (or of s), a group
    lg = np.zeros(hd // 64)
    for j in range(0, n, 32):
        sj, sc = s[j:j + 32], vs[j:j + 32, ::64]
        mn = max(m, sj.max())
        if mn == -np.inf:
            continue
        al = f32(2.0 ** (f * (float(m) - float(mn))))
        m = mn
        p = np.exp2((f * (sj - m)).astype(f32)).astype(f32)
        l = f32(l * al + p.sum(dtype=f32))
        for g in range(hd // 64):
            c = slice(64 * g, 64 * g + 64)
            ps = (p * sc[:, g].astype(f32)).astype(f32)
            if lift == "weights":
                top[g] = max(top[g] * float(al), float(ps.max()))
            else:
                top[:] = max(top.max(), sc.max())
            new = 6 - np.floor(np.log2(top[g])) if top[g] > 0 else 0.0
            o[c] = o[c] * al * f32(2.0 ** (new - lg[g]))
            lg[g] = new
            w = two_parts(ps * f32(2.0 ** new))
            o[c] = (o[c] + w @ vq[j:j + 32, c]).astype(f32)
            mid = (8 * sc[:, g] + vz[j:j + 32, 64 * g]).astype(f32)
            zsum[c] = zsum[c] * al + f32((p * mid).sum(dtype=f32))
    out = (o * 2.0 ** -np.repeat(lg, 64) + zsum) / l
    return out.astype(np.float64)


def value_scale_case(rng, B, Tq, heads, kv, hd, rows, ratio, at, gap, groups=None):
    """q (B, Tq, heads * hd), k and v (B, rows, kv, hd) fp32.  Scores within about 1 of each other
    but those of the rows `at`, which lie `gap` lower and whose values are `ratio` times as large
    (groups: in these groups of 64 channels only)."""
    q = (1 + 0.1 * rng.standard_normal((B, Tq, heads * hd))).astype(np.float32)
    k = (0.05 * rng.standard_normal((B, rows, kv, hd))).astype(np.float32)
    v = rng.standard_normal((B, rows, kv, hd)).astype(np.float32)
    k[:, at] -= np.float32(gap * hd ** -0.5)  # q k / sqrt(hd) of such a row: -gap
    for g in range(hd // 64) if groups is None else groups:
        v[:, at, :, 64 * g:64 * g + 64] *= np.float32(ratio)
    return q, k, v


def linear(x, weight, scales, G, blocks_of=128):
    """Outputs x @ weight^T in 64 bits and their bounds, (M, N).  weight and scales (N, K) as
    ref_weight gives them.

    A group's sum runs over both parts of x in G / 2 roundings, of partial sums of signed codes:
    below B = 8 |s x| (root sum of squares); over the groups, the waves and the splits come K / G +
    24 of the sum so far.  x's two parts are off by 2^-23 of an element, or 2^-25 of the largest of
    its block."""
    K = x.shape[1]
    x = x.astype(np.float64)
    want = x @ weight.T
    B = 8 * np.sqrt(x ** 2 @ (scales ** 2).T)
    top = np.zeros_like(want)
    for k in range(0, K, blocks_of):
        t = np.abs(x[:, k:k + blocks_of]).max(1)
        top += t[:, None] ** 2 * (weight[:, k:k + blocks_of] ** 2).sum(1)
    bound = np.sqrt(U * U * (G / 2 * B ** 2 + (K / G + 24) * (np.abs(want) + B) ** 2) +
                    (2.0 ** -23 * B) ** 2 + 2.0 ** -50 * top)
    return want, bound
