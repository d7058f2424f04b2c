"""Log probabilities, entropy and alternatives on the GPU against 64 bits."""
import pytest
import torch

from conftest import announce
from larynx_amd import ops

pytestmark = pytest.mark.gpu
INF = float("inf")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _reference(x, t, top):
    """In 64 bits: logp, entropy, top_logp, top_ids (equal logits by the lower id)."""
    d = x.double()
    lp = d - torch.logsumexp(d, 1, keepdim=True)
    given = torch.where(t < 0, torch.zeros_like(lp[:, 0]),
                        lp.gather(1, t.long().clamp(min=0)[:, None])[:, 0])
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    v, i = torch.sort(x + 0.0, dim=1, descending=True, stable=True)
    return given, H, lp.gather(1, i[:, :top]), i[:, :top].int()


def _check(x, t, top, gpu, pad=0):
    rows, V = x.shape
    wide = torch.full((rows, V + pad), 1e30)  # what lies between rows counts for nothing
    wide[:, :V] = x
    got = ops.token_logprobs(wide.to(gpu)[:, :V], t.to(gpu), top=top)
    logp, H, tl, ti = _reference(x, t, top)
    # s and the sum of products: at most 60 fp32 additions along a path (32 to 128 in a lane,
    # trees above), each exponential off by |d| 2^-24 + 2^-22 of itself: relative error of the
    # sums E = 200 * 2^-24 + 2^-24 * 30; log1p carries it as E / (1 + s) * s <= E; the result is
    # rounded once; an entropy term e^d |d| is off by the same E of itself, and the sum of these
    # is at most H
    E = 230 * 2.0 ** -24
    fin = torch.isfinite(logp)
    assert torch.equal(got.logp.cpu()[~fin].double(), logp[~fin])
    e = (got.logp.cpu().double() - logp).abs()[fin]
    assert (e <= E + 2.0 ** -24 * logp[fin].abs()).all(), e.max()
    e = (got.entropy.cpu().double() - H).abs()
    assert (e <= 4 * E * H + 2.0 ** -24 * H + 1e-30).all(), (e / (E * H)).max()
    if not top:
        assert got.top_logp is None and got.top_ids is None
        return got
    assert torch.equal(got.top_ids.cpu(), ti), (got.top_ids.cpu() != ti).nonzero()[:4]
    fin = torch.isfinite(tl)
    assert torch.equal(got.top_logp.cpu()[~fin].double(), tl[~fin])
    e = (got.top_logp.cpu().double() - tl).abs()[fin]
    assert (e <= E + 2.0 ** -24 * tl[fin].abs()).all(), e.max()
    return got


SIZES = [(1, 1, 1), (1, 2, 2), (3, 64, 64), (5, 100, 7), (1, 6761, 5), (40, 6761, 0), (33, 6761, 20),
         (7, 2048, 64), (7, 2049, 1), (5, 4097, 33), (5, 8192, 64), (4, 8193, 64), (3, 16385, 20),
         (2, 151936, 64), (9, 151936, 20), (3, 151936, 0), (1, 700001, 64), (2, 30003, 1)]


@pytest.mark.parametrize("rows,V,top", SIZES)
@pytest.mark.parametrize("pad", [0, 3])
def test_sizes(gpu, rows, V, top, pad):
    announce(f"token_logprobs {rows} x {V} top {top} pad {pad}")
    g = _gen(rows + V)
    x = 3 * torch.randn(rows, V, generator=g)
    t = torch.randint(0, V, (rows,), generator=g).int()
    t[2::3] = -1
    _check(x, t, top, gpu, pad)


@pytest.mark.parametrize("V", [500, 6761, 20000])
def test_masks(gpu, V):
    """Masked logits, few and many, fewer left than alternatives asked for."""
    announce(f"token_logprobs masks {V}")
    g = _gen(V)
    x = 3 * torch.randn(6, V, generator=g)
    x[0, 3:] = -INF
    x[1, :V - 2] = -INF
    x[2, torch.rand(V, generator=g) < 0.9] = -INF
    x[3, V // 2:] = -INF
    x[4, 1:] = -INF
    x[5, ::2] = torch.finfo(torch.float32).min  # the type's lowest value, as masks often are
    t = torch.tensor([1, 5, 7, V - 1, 0, 1]).int()
    _check(x, t, 64, gpu)


@pytest.mark.parametrize("V", [64, 130, 2048, 2500, 6761, 20000, 151936])
@pytest.mark.parametrize("open_", [0, 1, 5, 63, 64, 200, 1500])
def test_few_open_among_masked(gpu, V, open_):
    """Logits open at the end, the start or anywhere of a masked row; the rest by lowest index."""
    if open_ > V:
        open_ = V // 2
    announce(f"token_logprobs {open_} open of {V}")
    g = _gen(V + open_)
    x = torch.full((4, V), -INF)
    for r, at in enumerate([torch.arange(open_), V - 1 - torch.arange(open_),
                            torch.randperm(V, generator=g)[:open_],
                            torch.randperm(V, generator=g)[:open_]]):
        x[r, at] = torch.randn(open_, generator=g)
    x[3, torch.randperm(V, generator=g)[:min(3, V)]] = float("nan")  # the largest logits
    for top in (3, min(64, V)):
        got = ops.token_logprobs(x.to(gpu), top=top)
        key = torch.where(x.isnan(), torch.full_like(x, INF), x)
        ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_ids.cpu().long(), ids)
        assert got.top_logp[3].isnan().all()
        if open_:
            lp = torch.log_softmax(x[:3].double(), 1).gather(1, ids[:3])
            fin = torch.isfinite(lp)
            tl = got.top_logp[:3].cpu().double()
            assert torch.equal(tl[~fin], lp[~fin])
            assert ((tl - lp).abs()[fin] <= 2.0 ** -16 + 2.0 ** -24 * lp.abs()[fin]).all()
        else:
            assert (got.top_logp[:3] == -INF).all()


@pytest.mark.parametrize("V", [70, 6761, 9000])
def test_rows_of_nothing(gpu, V):
    x = torch.full((3, V), -INF)
    x[1] = torch.randn(V, generator=_gen(1))
    got = ops.token_logprobs(x.to(gpu), torch.tensor([4, 4, -1]).int().to(gpu), top=5)
    assert got.logp[0] == -INF and got.logp[2] == 0 and torch.isfinite(got.logp[1])
    assert got.entropy[0] == 0 and got.entropy[2] == 0
    assert (got.top_logp[[0, 2]] == -INF).all()
    assert got.top_ids[0].tolist() == [0, 1, 2, 3, 4] == got.top_ids[2].tolist()


@pytest.mark.parametrize("V", [70, 6761, 9000])
def test_nan_and_infinity(gpu, V):
    """They make NaN of their row alone; NaN counts as the largest logit."""
    g = _gen(V)
    x = torch.randn(5, V, generator=g)
    x[1, V - 3] = float("nan")
    x[2, 11] = INF
    x[4] = float("nan")
    t = torch.arange(5).int()
    got = ops.token_logprobs(x.to(gpu), t.to(gpu), top=3)
    bad = torch.tensor([False, True, True, False, True])
    assert got.logp.cpu().isnan().tolist() == bad.tolist()
    assert got.entropy.cpu().isnan().tolist() == bad.tolist()
    assert got.top_logp.cpu().isnan().all(1).tolist() == bad.tolist()
    assert got.top_ids[1, 0] == V - 3 and got.top_ids[2, 0] == 11
    assert got.top_ids[4].tolist() == [0, 1, 2]
    _check(x[[0, 3]], t[[0, 3]], 3, gpu)


def test_tokens_outside(gpu):
    x = torch.randn(5, 100, generator=_gen(3)).to(gpu)
    t = torch.tensor([-1, -2, 100, 99, 2 ** 31 - 1]).int().to(gpu)
    got = ops.token_logprobs(x, t).logp.cpu()
    assert got[0] == 0 and got[[1, 2, 4]].isnan().all() and torch.isfinite(got[3])


@pytest.mark.parametrize("V", [200, 6761, 25000, 151936])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "steps", "lane", "zeros"])
def test_order(gpu, V, kind):
    """Ties and orders that crowd the largest logits into few threads."""
    announce(f"token_logprobs order {kind} {V}")
    i = torch.arange(V)
    x = {"equal": torch.full((V,), 2.5), "rising": i * 1e-3, "falling": -i * 1e-3,
         "steps": (i * 7 % 5).float(),
         # the logits of four threads' loads above all others
         "lane": torch.where(i % 1024 < 16, 5.0 + torch.sin(i.float()), torch.sin(i.float())),
         "zeros": torch.where(i % 2 == 0, 0.0, -0.0)}[kind].float()
    x = torch.stack([x, x.flip(0)])
    _check(x, torch.tensor([0, V - 1]).int(), 64, gpu)
    _check(x, torch.tensor([V // 2, 1]).int(), 3, gpu)


@pytest.mark.parametrize("V", [6761, 20000])
@pytest.mark.parametrize("gap", [10.0, 20.0, 60.0, 200.0])
def test_one_likely_token(gpu, V, gap):
    """The probability of the rest is not lost beside one: logp and entropy near zero keep their
    digits."""
    x = torch.randn(4, V, generator=_gen(int(gap)))
    x[:, 17] = x.amax(1) + gap
    t = torch.tensor([17, 17, 3, 17]).int()
    got = ops.token_logprobs(x.to(gpu), t.to(gpu))
    d = (x - x[:, 17:18]).double()  # the differences as fp32 has them: off by 2^-24 of the gap
    others = torch.cat([d[:, :17], d[:, 18:]], 1)
    s = others.exp().sum(1)
    logp = -torch.log1p(s)
    rel = 230 * 2.0 ** -24 + (gap + 10) * 2.0 ** -23
    e = (got.logp.cpu().double() - logp).abs()[[0, 1, 3]]
    assert (e <= rel * logp.abs()[[0, 1, 3]] + 1e-45).all(), e
    H = torch.log1p(s) - (others.exp() * others).sum(1) / (1 + s)
    e = (got.entropy.cpu().double() - H).abs()
    assert (e <= 4 * rel * H + 1e-38).all(), (e / H)


@pytest.mark.parametrize("V", [2, 700, 6761, 20000, 151936])
@pytest.mark.parametrize("gap", [45.0, 50.0, 70.0, 85.0, 87.0, 88.0, 95.0, 100.0, 103.0, 110.0,
                                 1e30])
def test_one_token_far_ahead(gpu, V, gap):
    """All others below 2^-126 of the maximum each: their sum keeps its digits."""
    announce(f"token_logprobs one of {V} ahead by {gap}")
    x = torch.randn(6, V, generator=_gen(V))
    x[1] = x[1].round()
    x[2] = 0.25
    x[3, V // 2:] = -INF
    at = torch.tensor([0, V - 1, V // 2, 0, V // 3, V - 1])
    one = torch.nn.functional.one_hot(at, V).bool()
    x[one] = x.amax(1) + gap
    if V > 2:
        x[4, (V // 3 + 1) % V] = x[4].amax() - gap / 2  # another one between
    got = ops.token_logprobs(x.to(gpu), at.int().to(gpu), top=2)
    d = (x - x[one][:, None]).double()  # as fp32 has them: off by 2^-24 of the gap
    d = torch.where(one, torch.full_like(d, -INF), d)
    p = d.exp()
    s = p.sum(1)
    logp = -torch.log1p(s)
    H = torch.log1p(s) - torch.where(p > 0, p * d, torch.zeros_like(p)).sum(1) / (1 + s)
    # a term below 2^-61 is scaled, its argument carried to 2^-40: 2^-22 of it by the exponential;
    # the others' arguments (up to 62 log2(e)) are off by 2^-24 of themselves.  Sums: as everywhere
    rel = 230 * 2.0 ** -24 + 110 * 2.0 ** -23
    e = (got.logp.cpu().double() - logp).abs()
    assert (e <= rel * logp.abs() + 2.0 ** -149).all(), (e, logp)
    assert torch.equal(got.top_logp[:, 0], got.logp)
    e = (got.entropy.cpu().double() - H).abs()
    assert (e <= 4 * rel * H + 2.0 ** -147).all(), (e, H)


def test_parts_left_out(gpu):
    x = torch.randn(6, 9000, generator=_gen(5)).to(gpu)
    t = torch.arange(6).int().to(gpu)
    full = ops.token_logprobs(x, t, top=4)
    a = ops.token_logprobs(x, t, entropy=False)
    assert torch.equal(a.logp, full.logp) and a.entropy is a.top_ids is a.top_logp is None
    b = ops.token_logprobs(x, top=4, entropy=False)
    assert b.logp is b.entropy is None
    assert torch.equal(b.top_ids, full.top_ids) and torch.equal(b.top_logp, full.top_logp)
    c = ops.token_logprobs(x)
    assert c.logp is None and torch.equal(c.entropy, full.entropy)


def test_refusals(gpu):
    x, t = torch.zeros(4, 100, device=gpu), torch.zeros(4, dtype=torch.int32, device=gpu)
    for kw in [dict(tokens=t.long()), dict(tokens=t[:3]), dict(tokens=t.cpu()),
               dict(logits=x.double()), dict(logits=x.t()), dict(logits=x[0])]:
        with pytest.raises(ValueError):
            ops.token_logprobs(**{"logits": x, "tokens": t, **kw})
    from larynx_amd._lib import LxError
    for kw in [dict(top=65), dict(top=-1), dict(logits=x[:, :3], top=4),
               dict(tokens=None, entropy=False)]:
        with pytest.raises(LxError):
            ops.token_logprobs(**{"logits": x, "tokens": t, **kw})


def test_past_32_bits(gpu):
    """Rows whose offsets pass 2^31 elements, by their stride alone."""
    rows, V, ld = 3, 6761, 1 << 30
    buf = torch.empty((rows - 1) * ld + V, device=gpu)
    x = torch.randn(rows, V, generator=_gen(7))
    view = buf.as_strided((rows, V), (ld, 1))
    view.copy_(x)
    t = torch.tensor([1, 2, 3]).int()
    got = ops.token_logprobs(view, t.to(gpu), top=5)
    ref = ops.token_logprobs(x.to(gpu), t.to(gpu), top=5)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("V", [6761, 20000])
def test_captured(gpu, V):
    g = _gen(V)
    xs = [(3 * torch.randn(5, V, generator=g)).to(gpu) for _ in range(4)]
    t = torch.arange(5).int().to(gpu)
    want = [ops.token_logprobs(x, t, top=8) for x in xs]
    x = xs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.token_logprobs(x, t, top=8)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.token_logprobs(x, t, top=8)
    for i in [1, 2, 3, 0]:
        x.copy_(xs[i])
        graph.replay()
        eager = ops.token_logprobs(xs[(i + 1) % 4], t, top=8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(y, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 4]))
