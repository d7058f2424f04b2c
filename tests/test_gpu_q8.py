"""Matrices in 8 bits on the GPU: codes against the format in 64 bits (bit for bit), the norm that
feeds them, products against 64-bit sums over what the codes stand for."""
import math

import pytest
import torch

from conftest import announce
from larynx_amd import ops
from larynx_amd._lib import LxError
from q8_reference import E4M3, held

pytestmark = pytest.mark.gpu
EPS = 1e-6
INF, MAX = float("inf"), torch.finfo(torch.float32).max


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(a, b):
    """Equal, NaN where the other is."""
    a, b = a.double().cpu(), b.double().cpu()
    assert a.shape == b.shape
    bad = ~((a == b) | (a.isnan() & b.isnan()))
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:4].tolist(), a[bad][:4], b[bad][:4])


def _fp32(v):
    """The fp32 that stands for a held value: exact, but for numbers past its range."""
    return v.float()


# ---- codes ----------------------------------------------------------------------------


@pytest.mark.parametrize("scale", [-127, -126, -60, -1, 0, 3, 119])
def test_every_code_and_border(gpu, scale):
    """All e4m3 numbers, the borders between them and the fp32 numbers beside these, at one scale."""
    announce(f"q8 codes at 2^{scale}")
    t = E4M3.float()
    mid = (t[1:] + t[:-1]) / 2
    inf = torch.tensor(float("inf"))
    v = torch.cat([t, mid, torch.nextafter(mid, inf), torch.nextafter(mid, -inf)])
    v = torch.cat([v, -v])
    v = torch.nn.functional.pad(v, (0, -v.numel() % 127)).view(-1, 127)
    v = torch.cat([v, torch.full((v.shape[0], 1), 448.0)], 1)  # each block at this scale
    x = (v.double() * 2.0 ** scale).float()
    want, powers = held(x)
    assert (powers == 2.0 ** scale).all()
    _same(ops.q8_unpack(ops.q8_pack(x.to(gpu))), _fp32(want))


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 127), (2, 128), (3, 129), (15, 500), (16, 896),
                                    (17, 1001), (37, 4864), (300, 13)])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_pack_sizes_and_strides(gpu, rows, K, pad):
    announce(f"q8 pack {rows} x {K} stride +{pad}")
    x = torch.randn(rows, K, generator=_gen(rows * K)) * torch.exp(
        3 * torch.randn(rows, 1, generator=_gen(7)))
    wide = torch.full((rows, K + pad), float("nan"))  # what lies between rows counts for nothing
    wide[:, :K] = x
    q = ops.q8_pack(wide.to(gpu)[:, :K])
    assert (q.rows, q.K) == (rows, K)
    _same(ops.q8_unpack(q), _fp32(held(x)[0]))


def test_pack_extremes(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(8, 300, generator=_gen(3))
    x[0] = 0.0
    x[1] = 1e-42          # subnormal numbers of fp32
    x[2, :128] = 3.4e38   # the largest: stands for 2^128, infinity in fp32
    x[3, 5] = nan
    x[4, 130] = inf
    x[4, 131] = -inf
    x[5] = nan
    x[6] = -0.0
    x[7, 128:256] = torch.tensor([2.0 ** -149, 448 * 2.0 ** -127] * 64)
    _same(ops.q8_unpack(ops.q8_pack(x.to(gpu))), _fp32(held(x)[0]))


def test_pack_into_a_given_matrix(gpu):
    """The rows of the matrix are written whole, whatever it held: nothing of a row's tail stays."""
    q = ops.q8_pack(torch.full((20, 300), float("nan"), device=gpu))
    data = q.data
    x, w = torch.randn(20, 300, generator=_gen(4)), torch.randn(24, 300, generator=_gen(5))
    assert ops.q8_pack(x.to(gpu), out=q) is q and q.data is data
    y = ops.linear_q8(q, ops.q8_pack(w.to(gpu)))
    assert not y.isnan().any()
    with pytest.raises(ValueError, match="out must hold"):
        ops.q8_pack(x[:19].to(gpu), out=q)


# ---- norm -----------------------------------------------------------------------------


def _norm64(h, w, eps=EPS):
    h = h.double()
    eps = float(torch.tensor(eps, dtype=torch.float32))
    return h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()


NORMS = [(1, 896), (5, 1), (3, 128), (33, 1001), (64, 1024), (7, 1025), (130, 2047), (9, 2049),
         (4, 4096), (5, 4100), (6, 8192), (3, 8193), (2, 20000), (37, 2100), (50, 5000), (33, 8300)]


@pytest.mark.parametrize("rows,D", NORMS)
def test_norm_codes(gpu, rows, D):
    announce(f"rms_norm_q8 {rows} x {D}")
    g = _gen(D)
    x = torch.randn(rows, D, generator=g)
    x[:, ::97] *= 20
    w = 1 + 0.2 * torch.randn(D, generator=g)
    q = ops.rms_norm_q8(x.to(gpu), w.to(gpu))
    _same(ops.q8_unpack(q), _fp32(held(_norm64(x, w))[0]))


@pytest.mark.parametrize("rows,D", NORMS)
@pytest.mark.parametrize("where", ["x", "add", "apart"])
def test_norm_with_residual(gpu, rows, D, where):
    announce(f"rms_norm_q8 {rows} x {D} sum in {where}")
    g = _gen(D + 1)
    x, add = torch.randn(rows, D, generator=g), torch.randn(rows, D, generator=g)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    h = x + add
    xd, ad = x.to(gpu), add.to(gpu)
    out = {"x": None, "add": ad, "apart": torch.full((rows, D), 7.0, device=gpu)}[where]
    q = ops.rms_norm_q8(xd, w.to(gpu), add=ad, sum_out=out)
    _same(xd if out is None else out, h)
    if where != "x":
        _same(xd, x)
    if where != "add":
        _same(ad, add)
    _same(ops.q8_unpack(q), _fp32(held(_norm64(h, w))[0]))


@pytest.mark.parametrize("rows,D", [(2048, 4100), (2049, 8192), (2063, 5001)])
@pytest.mark.parametrize("where", ["x", "add", "apart"])
def test_norm_of_many_long_rows(gpu, rows, D, where):
    test_norm_with_residual(gpu, rows, D, where)


@pytest.mark.parametrize("rows,D,where", [(3500, 4480, "x"), (3101, 5001, "add"),
                                          (1901, 8192, "apart"), (3434, 4479, "apart")])
def test_norm_of_rows_from_memory(gpu, rows, D, where):
    """Two rows a workgroup and, just below, one."""
    test_norm_with_residual(gpu, rows, D, where)


def test_norm_strides(gpu):
    """Rows of unequal strides at odd offsets; what lies between them stays."""
    g = _gen(9)
    rows, D = 21, 515
    buf = [torch.randn(rows, D + p, generator=g) for p in (1, 2, 6)]
    w = torch.randn(D + 1, generator=g)
    dev = [b.to(gpu) for b in buf]
    q = ops.rms_norm_q8(dev[0][:, 1:], w.to(gpu)[1:], add=dev[1][:, 2:], sum_out=dev[2][:, 3:-3])
    h = buf[0][:, 1:] + buf[1][:, 2:]
    want = buf[2].clone()
    want[:, 3:-3] = h
    _same(dev[2], want)
    _same(ops.q8_unpack(q), _fp32(held(_norm64(h, w[1:]))[0]))


def test_norm_extremes(gpu):
    """Rows of zeros, of very large and very small numbers, with infinities and NaN."""
    g = _gen(11)
    x = torch.randn(7, 896, generator=g)
    x[0] = 0.0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 17] = float("inf")
    x[4, 600] = float("nan")
    x[5, 895] = 3e38
    x[6] = 2.0 ** -149
    w = torch.randn(896, generator=g)
    _same(ops.q8_unpack(ops.rms_norm_q8(x.to(gpu), w.to(gpu))), _fp32(held(_norm64(x, w))[0]))


def test_norm_refusals(gpu):
    x, w = torch.zeros(4, 256, device=gpu), torch.ones(256, device=gpu)
    for kw in [dict(w=w[:255]), dict(w=w.double()), dict(w=w.cpu()), dict(sum_out=x),
               dict(add=x[:3]), dict(add=x.cpu()), dict(add=x.double()),
               dict(add=torch.zeros_like(x), sum_out=x[:, :255]),
               dict(out=ops.q8_pack(x[:3]))]:
        with pytest.raises(ValueError):
            ops.rms_norm_q8(**{"x": x, "w": w, **kw})
    both = torch.zeros(4, 260, device=gpu)
    with pytest.raises(LxError):
        ops.rms_norm_q8(both[:, :256], w, add=x, sum_out=both[:, 4:])


# ---- products -------------------------------------------------------------------------


def _pair(M, N, K, seed, gpu):
    g = _gen(seed)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) * K ** -0.5
    x[:, ::31] *= 6
    xq, wq = ops.q8_pack(x.to(gpu)), ops.q8_pack(w.to(gpu))
    return xq, wq, ops.q8_unpack(xq).double().cpu(), ops.q8_unpack(wq).double().cpu()


def _bound(X, W):
    """Exact products, at most K + 16 fp32 additions of partial sums below S = sum |x w|, each off
    by less than its last place (2^-23), in the instruction as between them."""
    K = X.shape[1]
    return (K + 16) * 2.0 ** -23 * (X.abs() @ W.abs().t())


LINEARS = [(1, 1, 1), (1, 16, 128), (1, 1152, 896), (2, 17, 129), (4, 6761, 896), (15, 33, 1000),
           (16, 100, 4864), (17, 64, 300), (31, 9, 256), (33, 130, 896), (64, 64, 640),
           (65, 257, 500), (100, 1152, 896), (128, 256, 128), (129, 895, 1280), (177, 6761, 896),
           (256, 9728, 896), (300, 896, 4864), (513, 300, 2000), (1531, 896, 896),
           (1025, 1030, 130), (3, 900, 8192), (2000, 1500, 1100), (2049, 2305, 257),
           (2100, 4100, 384),
           # each tile size with one block of K, a short one, or a long and ragged one
           (9, 4100, 8192), (300, 896, 100), (300, 898, 2100), (1531, 896, 64), (500, 1500, 1600),
           (300, 1600, 4864), (1531, 900, 1600), (1400, 1000, 2177), (256, 9728, 100),
           (2049, 2305, 100), (3600, 3800, 100), (3500, 3590, 700),
           # several blocks a wave on the smallest tiles
           (200, 700, 4864), (40, 900, 2200), (130, 800, 1200),
           # and on the largest that have K to themselves
           (1900, 1000, 3000), (2290, 890, 4864), (20, 17000, 300), (80, 18000, 1600)]


@pytest.mark.parametrize("M,N,K", LINEARS)
def test_products(gpu, M, N, K):
    announce(f"linear_q8 {M} x {N} x {K}")
    xq, wq, X, W = _pair(M, N, K, M + N + K, gpu)
    y = ops.linear_q8(xq, wq).double().cpu()
    want = X @ W.t()
    err = (y - want).abs()
    assert (err <= _bound(X, W)).all(), (err / _bound(X, W)).max()
    # the sums of a whole call: rounding errors average out, a lost product would not
    rel = (err.square().sum() / want.square().sum()).sqrt()
    assert rel <= 2.0 ** -24 * (2 + math.sqrt(K)), rel


@pytest.mark.parametrize("M,N,K", LINEARS)
def test_every_product_counts(gpu, M, N, K):
    """Whole numbers with exact fp32 sums (below 2^24): no product is lost, doubled or moved."""
    announce(f"linear_q8 whole numbers {M} x {N} x {K}")
    g = _gen(M * 7 + N * 3 + K)
    x = torch.randint(-15, 16, (M, K), generator=g).float()
    w = torch.randint(-15, 16, (N, K), generator=g).float()
    x[:, 0] = 15  # |x| <= 15 and steps of 1: held as they are at any scale up to 2^0
    w[:, 0] = 15
    xq, wq = ops.q8_pack(x.to(gpu)), ops.q8_pack(w.to(gpu))
    X, W = ops.q8_unpack(xq).double().cpu(), ops.q8_unpack(wq).double().cpu()
    assert torch.equal(X, x.double()) and torch.equal(W, w.double())
    _same(ops.linear_q8(xq, wq), X @ W.t())


@pytest.mark.parametrize("M,N,K", [(3, 40, 1157), (40, 33, 1157), (300, 900, 1157),
                                   (500, 1500, 1700), (1400, 900, 1700), (1100, 1300, 1157),
                                   (1531, 1152, 300), (2100, 2100, 1157), (3590, 3598, 700),
                                   (60, 200, 2300), (60, 6100, 2300), (1900, 990, 3000)])
def test_scales_of_every_row_and_block(gpu, M, N, K):
    """Blocks at powers of two of their own, one element each: every product has its scales."""
    g = _gen(M)
    kb = (K + 127) // 128
    ex = torch.randint(-40, 40, (M, kb), generator=g)
    ew = torch.randint(-40, 40, (N, kb), generator=g)
    at = torch.randint(0, 5, (kb,), generator=g) + 128 * torch.arange(kb)
    x, w = torch.zeros(M, K), torch.zeros(N, K)
    x[:, at] = torch.ldexp(torch.ones(()), ex)
    # one block a row of w: its product stands alone
    one = torch.arange(N) % kb
    w[torch.arange(N), at[one]] = torch.ldexp(torch.ones(()), ew[torch.arange(N), one])
    y = ops.linear_q8(ops.q8_pack(x.to(gpu)), ops.q8_pack(w.to(gpu)))
    _same(y, x.double() @ w.double().t())


@pytest.mark.parametrize("M,N,K", [(3, 40, 1157), (40, 33, 1157), (300, 900, 1157),
                                   (500, 1500, 1700), (1400, 900, 1700), (1100, 1300, 1157),
                                   (1531, 1152, 900), (2100, 2100, 1157), (3590, 3598, 900),
                                   (60, 200, 2300), (60, 6100, 2300), (1900, 990, 3000)])
def test_ends_of_the_scales(gpu, M, N, K):
    """Blocks at the smallest and the largest powers of two, the other operand's at the opposite:
    whole numbers, exact sums."""
    announce(f"linear_q8 ends of the scales {M} x {N} x {K}")
    g = _gen(M + K)
    ends = torch.tensor([-127, -126, -125, 120, 119, 118, 0])
    e = ends[torch.arange((K + 127) // 128) % len(ends)]
    ex = e.repeat_interleave(128)[:K].double()
    a = torch.randint(-15, 16, (M, K), generator=g).double()
    b = torch.randint(-15, 16, (N, K), generator=g).double()
    # 240 sets its block's power; the other operand is zero there
    a[:, 0::128], b[:, 0::128] = 240, 0
    a[:, 1::128], b[:, 1::128] = 0, 240
    x, w = a * 2.0 ** ex, b * 2.0 ** (-7 - ex)
    assert torch.equal(x.float().double(), x) and torch.equal(w.float().double(), w)
    if M == 3:
        assert torch.equal(held(x)[1], (2.0 ** e.double()).expand(M, -1))
    y = ops.linear_q8(ops.q8_pack(x.float().to(gpu)), ops.q8_pack(w.float().to(gpu)))
    _same(y, a @ b.t() * 2.0 ** -7)


@pytest.mark.parametrize("M", [3, 40, 300, 1531])
def test_smallest_elements(gpu, M):
    """One element a row from 2^-119 down to the smallest, 2^-136: whole from 2^-126 on, the nearest
    multiple of 2^-133 (bf16's subnormal numbers) below."""
    codes = E4M3[1:].float().double()
    K, N = 130, 1152
    x = torch.zeros(M, K, dtype=torch.float64)
    x[:, 1] = codes[torch.arange(M) % len(codes)] * 2.0 ** -127
    w = torch.zeros(N, K)
    w[:, 1] = 2.0 ** 100
    for flip in (False, True):
        p, q = (w, x.float()) if flip else (x.float(), w)
        y = ops.linear_q8(ops.q8_pack(p.to(gpu)), ops.q8_pack(q.to(gpu))).double().cpu()
        y = (y.t() if flip else y) * 2.0 ** -100
        v = x[:, 1:2]
        assert torch.equal(y[v[:, 0] >= 2.0 ** -126], v.expand(-1, N)[v[:, 0] >= 2.0 ** -126])
        assert ((y - v).abs() <= 2.0 ** -134).all()
        assert ((y * 2.0 ** 133).frac() == 0).all()


@pytest.mark.parametrize("M,N", [(3, 40), (40, 33), (300, 900), (1531, 1152)])
def test_past_the_largest_number(gpu, M, N):
    """An element that stands for 2^128 is infinity in a product as in the read-back."""
    x, w = torch.ones(M, 300), torch.ones(N, 300)
    x[M // 2, 200] = 3.4e38
    w[N - 1, 5] = -3.4e38
    y = ops.linear_q8(ops.q8_pack(x.to(gpu)), ops.q8_pack(w.to(gpu))).cpu()
    assert (y[M // 2, :N - 1] == INF).all() and y[M // 2, N - 1].isnan()
    rest = torch.arange(M) != M // 2
    assert (y[rest, N - 1] == -INF).all() and torch.isfinite(y[rest, :N - 1]).all()


def _epi(kind, acc, b=None, r=None):
    if b is not None:
        acc = acc + b.double()
    if kind == "gelu":
        return 0.5 * acc * (1 + torch.tanh(0.7978845608028654 * (acc + 0.044715 * acc ** 3)))
    if kind == "resid":
        return r.double() + acc
    if kind == "swiglu":
        return acc[:, 0::2] / (1 + torch.exp(-acc[:, 0::2])) * acc[:, 1::2]
    return acc


KINDS = {"none": None, "gelu": ops.LX_EPI_GELU_TANH, "resid": ops.LX_EPI_RESID,
         "swiglu": ops.LX_EPI_SWIGLU_PAIRED}
EPI_SHAPES = [(1, 66, 896), (9, 68, 200), (40, 130, 300), (70, 1152, 896), (257, 514, 896),
              (1030, 1026, 150), (300, 898, 260), (500, 1502, 1600), (1531, 898, 1600),
              (1531, 1152, 300), (2100, 2050, 130), (3590, 3598, 130), (1900, 990, 3000)]


@pytest.mark.parametrize("M,N,K", EPI_SHAPES)
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("bias", [False, True])
def test_epilogues(gpu, M, N, K, kind, bias):
    announce(f"linear_q8 {kind} bias {bias} {M} x {N} x {K}")
    xq, wq, X, W = _pair(M, N, K, M + K, gpu)
    g = _gen(5)
    b = torch.randn(N, generator=g) if bias else None
    r = torch.randn(M, N, generator=g) if kind == "resid" else None
    epi = None if KINDS[kind] is None else ops.Epilogue(kind=KINDS[kind])
    y = ops.linear_q8(xq, wq, None if b is None else b.to(gpu), epilogue=epi,
                      resid=None if r is None else r.to(gpu)).double().cpu()
    acc = X @ W.t()
    want = _epi(kind, acc, b, r)
    # the sums' bound, carried through the epilogue (slopes: GELU and SiLU at most 1.13; a SwiGLU
    # output's other factor), and its own fp32 steps: bias and residual additions 2^-24 of what
    # they give, the activations a few 2^-23 of their result (hardware exponentials and
    # reciprocals, arguments off by 2^-22 of themselves: |u| e^-|u| <= 1/2 of it, times |acc|)
    e = _bound(X, W) + 2.0 ** -24 * (acc.abs() + (b.abs().double() if bias else 0.0))
    if kind == "resid":
        tol = e + 2.0 ** -24 * want.abs() + 1e-45
    elif kind == "gelu":
        tol = 1.13 * e + 2.0 ** -20 * (acc + (b.double() if bias else 0.0)).abs()
    elif kind == "swiglu":
        full = acc + (b.double() if bias else 0.0)
        gate, up = full[:, 0::2], full[:, 1::2]
        tol = 1.13 * e[:, 0::2] * (up.abs() + e[:, 1::2]) + gate.abs() * e[:, 1::2] + \
            2.0 ** -20 * (gate * up).abs()
    else:
        tol = e + 2.0 ** -24 * want.abs()
    assert ((y - want).abs() <= tol + 1e-37).all(), ((y - want).abs() / tol).max()


GATES = [0.0, 1e-30, 0.5, 7.0, 20.0, 60.0, 86.9, 87.2, 88.5, 88.8, 90.0, 100.0, 104.0, 105.5, 130.0,
         1e4, 1e30, 2.3e38, 2.4e38, MAX]


@pytest.mark.parametrize("M,N,K", EPI_SHAPES)
def test_swiglu_of_any_gate(gpu, M, N, K):
    """Gates from the type's lowest value to its largest, and past it, through the bias."""
    announce(f"linear_q8 SwiGLU of any gate {M} x {N} x {K}")
    gates = torch.tensor(GATES + [-v for v in GATES] + [INF, -INF, float("nan")])
    up = torch.tensor([1.0, -3.5, 1e-3, 700.0])[torch.arange(N // 2) // 3 % 4]
    xq = ops.q8_pack(torch.zeros(M, K, device=gpu))
    wq = ops.q8_pack(torch.zeros(N, K, device=gpu))
    for roll in (0, 33):  # few columns take two calls
        gate = gates[(torch.arange(N // 2) + roll) % len(gates)]
        y = ops.linear_q8(xq, wq, torch.stack([gate, up], 1).reshape(-1).to(gpu),
                          epilogue=ops.Epilogue(kind=ops.LX_EPI_SWIGLU_PAIRED)).double().cpu()
        g, u = gate.double(), up.double()
        want = g * torch.sigmoid(g) * u
        fin = torch.isfinite(want) & (want.abs() <= MAX)
        # the exponential's square off by two last places (2^-22), the reciprocal by one or two, four
        # roundings of 2^-24: below 2^-20 of the result; a subnormal sigmoid is off by 2^-149, a
        # subnormal result once more
        tol = 2.0 ** -20 * want.abs() + 2.0 ** -149 * (1 + (g * u).abs())
        assert ((y - want).abs() <= tol)[:, fin].all(), (gate[fin], (y - want)[0, fin])
        over = want.isinf() | (want.abs() > MAX)
        assert torch.equal(y[:, over], (torch.sign(want[over]) * INF).expand(M, -1))
        assert y[:, want.isnan()].isnan().all()


@pytest.mark.parametrize("M,N,K", EPI_SHAPES)
@pytest.mark.parametrize("pad", [0, 1, 3, 4])
def test_outputs_in_place_and_strided(gpu, M, N, K, pad):
    """Residual in place, rows of y apart: what lies behind and between them stays."""
    announce(f"linear_q8 in place {M} x {N} x {K} pad {pad}")
    xq, wq, X, W = _pair(M, N, K, K, gpu)
    g = _gen(6)
    buf = torch.randn(M + 3, N + pad, generator=g)
    y = buf.to(gpu)
    out = y[:M, pad:]
    ops.linear_q8(xq, wq, epilogue=ops.Epilogue(kind=ops.LX_EPI_RESID), out=out)
    plain = ops.linear_q8(xq, wq)
    want = buf.clone()
    want[:M, pad:] += plain.cpu()
    _same(y, want)
    z = torch.full_like(y, 3.0)
    ops.linear_q8(xq, wq, out=z[:M, pad:])
    want = torch.full((M + 3, N + pad), 3.0)
    want[:M, pad:] = plain.cpu()
    _same(z, want)


@pytest.mark.parametrize("M,N,K", [(5, 40, 300), (70, 200, 300), (300, 900, 300), (500, 1500, 1600),
                                   (1400, 900, 1600), (1100, 1300, 300), (2100, 2100, 300),
                                   (3590, 3598, 300)])
def test_nan_stays_in_its_rows(gpu, M, N, K):
    g = _gen(8)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    clean = ops.linear_q8(ops.q8_pack(x.to(gpu)), ops.q8_pack(w.to(gpu))).cpu()
    x[M // 2, 7] = float("nan")
    x[0, 299] = float("inf")
    w[N - 1, 130] = -float("inf")
    y = ops.linear_q8(ops.q8_pack(x.to(gpu)), ops.q8_pack(w.to(gpu))).cpu()
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[[0, M // 2]] = True
    bad[:, N - 1] = True
    assert y[bad].isnan().all()
    # the non-finite elements do not change their block's scale here: the rest is as before
    same = ~bad
    assert torch.equal(y[same], clean[same])


def test_rows_past_the_last(gpu):
    """The last tile's memory behind the last row of x and w holds NaN codes: nothing shows."""
    for M, N, K in [(3, 21, 300), (37, 70, 300), (261, 900, 300), (499, 1501, 1600),
                    (1401, 901, 1600), (1029, 1100, 300), (2101, 2101, 300), (3587, 3587, 200)]:
        xq, wq, X, W = _pair(M, N, K, 12, gpu)
        y = ops.linear_q8(xq, wq)
        held_x = ops.q8_pack(torch.full((-(-M // 16) * 16, K), float("nan"), device=gpu))
        held_w = ops.q8_pack(torch.full((-(-N // 16) * 16, K), float("nan"), device=gpu))
        x2 = ops.q8_pack(ops.q8_unpack(xq), out=ops.Q8Matrix(held_x.data, M, K))
        w2 = ops.q8_pack(ops.q8_unpack(wq), out=ops.Q8Matrix(held_w.data, N, K))
        assert torch.equal(ops.linear_q8(x2, w2), y)


def test_past_32_bits(gpu):
    """Matrices of more than 2^31 bytes, as rows and as a weight: whole numbers, exact sums."""
    announce("8-bit matrices past 2^31 bytes")
    g = _gen(21)
    n, K = 270000, 8192  # 2.2 GB of codes
    base = torch.randint(-15, 16, (1000, K), generator=g).float()
    few = torch.randint(-15, 16, (48, K), generator=g).float()
    want = base.double() @ few.double().t()
    big = ops.q8_pack(base.to(gpu).repeat(n // 1000, 1))
    for M in (3, 48):
        q = ops.q8_pack(few[:M].to(gpu))
        _same(ops.linear_q8(big, q)[-1000:], want[:, :M])
        _same(ops.linear_q8(q, big)[:, -1000:], want[:, :M].t())
    x = ops.q8_unpack(big)
    assert torch.equal(x[-1000:].cpu(), base) and torch.equal(x[:1000].cpu(), base)
    h = ops.rms_norm_q8(x, torch.ones(K, device=gpu), add=torch.zeros_like(x), out=big)
    small = ops.q8_unpack(ops.rms_norm_q8(base.to(gpu), torch.ones(K, device=gpu)))
    assert torch.equal(ops.q8_unpack(h)[-1000:], small)


def test_linear_refusals(gpu):
    xq, wq = ops.q8_pack(torch.zeros(4, 256, device=gpu)), ops.q8_pack(torch.zeros(6, 256, device=gpu))
    other = ops.q8_pack(torch.zeros(6, 255, device=gpu))
    with pytest.raises(LxError):
        ops.linear_q8(xq, other)
    resid = ops.Epilogue(kind=ops.LX_EPI_RESID)
    y = torch.zeros(4, 6, device=gpu)
    for kw in [dict(b=torch.zeros(5, device=gpu)), dict(b=torch.zeros(6)), dict(epilogue=resid),
               dict(epilogue=resid, resid=y[:3]), dict(epilogue=resid, resid=y.cpu()),
               dict(out=y[:, :5]), dict(out=y.cpu()), dict(out=y.double())]:
        with pytest.raises(ValueError):
            ops.linear_q8(xq, wq, **kw)
    for kw in [dict(epilogue=ops.Epilogue(kind=ops.LX_EPI_GATED_RESID)), dict(resid=y),
               dict(epilogue=ops.Epilogue(kind=17))]:
        with pytest.raises(LxError):
            ops.linear_q8(xq, wq, **kw)


# ---- streams and graphs ---------------------------------------------------------------


@pytest.mark.parametrize("M", [1, 40, 300])
def test_captured_with_an_eager_call_between(gpu, M):
    """A norm and its projection captured and replayed over changing inputs, eager calls of the
    same sizes between the replays."""
    announce(f"q8 graph {M}")
    D, N = 896, 300
    g = _gen(M)
    xs = [torch.randn(M, D, generator=g).to(gpu) for _ in range(4)]
    w = torch.rand(D, generator=g).to(gpu) + 0.5
    wq = ops.q8_pack(torch.randn(N, D, generator=g).to(gpu))
    want = [ops.linear_q8(ops.rms_norm_q8(x, w), wq) for x in xs]
    x = xs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.linear_q8(ops.rms_norm_q8(x, w), wq)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_q8(ops.rms_norm_q8(x, w), wq)
    for i in [1, 2, 3, 0]:
        x.copy_(xs[i])
        graph.replay()
        eager = ops.linear_q8(ops.rms_norm_q8(xs[(i + 1) % 4], w), wq)
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(eager, want[(i + 1) % 4])


def test_two_streams(gpu):
    g = _gen(2)
    x = [torch.randn(200, 896, generator=g).to(gpu) for _ in range(2)]
    wq = ops.q8_pack(torch.randn(500, 896, generator=g).to(gpu))
    want = [ops.linear_q8(ops.q8_pack(v), wq) for v in x]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.linear_q8(ops.q8_pack(x[i]), wq))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
