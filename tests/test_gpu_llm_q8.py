"""The prefill on 8-bit weights (set_prefill_bits) and the scoring of tokens: each layer against 64
bits over what the weights and the quantised rows stand for, the switch, captured prefills."""
import numpy as np
import pytest
import torch

from conftest import announce
from larynx_amd import ops
from oracle import oracle as orc
from q8_reference import held
from test_gpu_llm_four_bit import _model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm8(gpu):
    cfg, params, lm = _model(gpu, 95)
    yield cfg, params, lm
    lm.close()


def _t(a):
    return torch.from_numpy(np.asarray(a)).double()


def _norm(x, w, eps):
    return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * w


def _rope(v, cfg):
    """NEOX rotary of (L, heads, 64)."""
    inv = 1.0 / cfg.rope_theta ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    ang = torch.arange(v.shape[0], dtype=torch.float64)[:, None, None] * inv
    a, b = v[..., :32], v[..., 32:]
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def _layer(x, p, cfg, params):
    """One layer in 64 bits, its projections over 8-bit rows and weights: (x, k, v)."""
    W = lambda n: held(torch.from_numpy(params[p + n]))[0]  # noqa: E731
    q8 = lambda v: held(v)[0]  # noqa: E731
    L, H = x.shape
    hn = q8(_norm(x, _t(params[p + "input_layernorm.weight"]), cfg.rms_eps))
    q, k, v = (hn @ W(f"self_attn.{n}_proj.weight").t() + _t(params[p + f"self_attn.{n}_proj.bias"])
               for n in "qkv")
    q, k = (_rope(t.view(L, -1, 64), cfg) for t in (q, k))
    rep = cfg.n_heads // cfg.n_kv_heads
    kk, vv = k.repeat_interleave(rep, 1), v.view(L, -1, 64).repeat_interleave(rep, 1)
    s = torch.einsum("qhd,khd->hqk", q, kk) / 8
    s = s.masked_fill(torch.triu(torch.ones(L, L, dtype=torch.bool), 1), float("-inf"))
    o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), vv).reshape(L, H)
    x = x + q8(o) @ W("self_attn.o_proj.weight").t()
    hn = q8(_norm(x, _t(params[p + "post_attention_layernorm.weight"]), cfg.rms_eps))
    g = hn @ W("mlp.gate_proj.weight").t()
    a = g / (1 + torch.exp(-g)) * (hn @ W("mlp.up_proj.weight").t())
    return x + q8(a) @ W("mlp.down_proj.weight").t(), k.reshape(L, -1), v


# An activation whose fp32 value (off by 1e-6 of itself) lies next to a border takes the
# neighbouring code: one in 2^-3 / 1e-6, some 1e-5 of them, each moving its products by up to 2^-3
# of themselves; of a sum of K products of equal size, one in sqrt(K) of it.  Root mean square
# over a layer: sqrt(1e-5) * 2^-3 = 4e-4 at most, 1e-3 taken; the largest: a few such products of
# the largest factors, 2^-3 * 4 * 4 / (4 * sqrt(320)) = 3e-2 of the largest sum.
RMS, MOST = 1e-3, 3e-2


def _near(got, want, what):
    got = got.double().cpu()
    rms = ((got - want).square().mean() / want.square().mean()).sqrt()
    assert rms < RMS, (what, rms)
    assert orc.rel_err(got.numpy(), want.numpy()) < MOST, what


@pytest.mark.parametrize("L", [1, 5, 16, 17, 70, 200])
def test_layers(gpu, lm8, L):
    cfg, params, lm = lm8
    announce(f"8-bit prefill, {L} rows")
    lm.set_prefill_bits(8)
    x = torch.randn(L, cfg.hidden, generator=torch.Generator().manual_seed(L)) * 0.5
    logits, hidden, final = lm.prefill(x.to(gpu), capture=True)
    torch.cuda.synchronize()
    assert lm.cache_len == L
    h = x.double()
    for i in range(cfg.n_layers):
        want, k, v = _layer(h, f"layers.{i}.", cfg, params)
        h = hidden[i].double().cpu()  # the next layer from what this one gave
        _near(hidden[i], want, f"layer {i}")
        kd, vd = lm.cache_views(i)
        # one projection of exact codes: fp32 level
        assert orc.rel_err(kd[:L].cpu().numpy(), k.numpy()) < 1e-5
        assert orc.rel_err(vd[:L].cpu().numpy(), v.numpy()) < 1e-5
    fn = _norm(h, _t(params["norm.weight"]), cfg.rms_eps)
    assert orc.rel_err(final.cpu().numpy(), fn.numpy()) < 1e-6
    want = held(fn)[0] @ held(torch.from_numpy(params["llm_decoder.weight"]))[0].t()
    assert orc.rel_err(logits.cpu().numpy(), want.numpy()) < 1e-5
    assert torch.equal(lm.prefill(x.to(gpu)), logits)


@pytest.mark.parametrize("kw", [dict(hidden=320, intermediate=1100, n_heads=5, n_kv_heads=1),
                                dict(hidden=1024, intermediate=132, n_heads=16, n_kv_heads=8)])
def test_other_geometries(gpu, kw):
    """Widths that are no multiple of a block."""
    announce(f"8-bit prefill {kw}")
    cfg, params, lm = _model(gpu, 96, **kw)
    lm.set_prefill_bits(8)
    x = torch.randn(33, cfg.hidden, generator=torch.Generator().manual_seed(1)) * 0.5
    _, hidden, _ = lm.prefill(x.to(gpu), capture=True)
    h = x.double()
    for i in range(cfg.n_layers):
        want = _layer(h, f"layers.{i}.", cfg, params)[0]
        h = hidden[i].double().cpu()
        _near(hidden[i], want, f"layer {i}")
    lm.close()


@pytest.mark.parametrize("L", [600, 1531])
def test_long_prompts(gpu, L):
    """Gate/up on 128 x 128 and 256 x 256 tiles, down on the tiles of long K."""
    announce(f"8-bit prefill of {L} rows")
    from larynx_amd.llm import Qwen2Config, Qwen2LM, qwen2_param_shapes
    cfg = Qwen2Config(n_layers=1, text_vocab=2000, hidden=320, intermediate=4864, n_heads=5,
                      n_kv_heads=1)
    params = orc.make_params(qwen2_param_shapes(cfg), 97)
    for k in params:
        if k.endswith("layernorm.weight") or k == "norm.weight":
            params[k] = (params[k] + 1.0).astype(np.float32)
    lm = Qwen2LM({k: torch.from_numpy(v).to(gpu) for k, v in params.items()}, cfg, max_ctx=1600)
    lm.set_prefill_bits(8)
    x = torch.randn(L, cfg.hidden, generator=torch.Generator().manual_seed(L)) * 0.5
    logits, hidden, final = lm.prefill(x.to(gpu), capture=True)
    want, k, v = _layer(x.double(), "layers.0.", cfg, params)
    _near(hidden[0], want, "layer 0")
    kd, vd = lm.cache_views(0)
    # the rotary angles are fp32: a frequency below 1 is off by two roundings of itself, its product
    # with the position by one more, so the angle by 3 L 2^-24 (2.7e-4 at 1531), and a rotated pair
    # by that of its length, at most sqrt(2) of the largest element
    assert orc.rel_err(kd[:L].cpu().numpy(), k.numpy()) < 1e-5 + 1.5 * 3 * L * 2.0 ** -24
    assert orc.rel_err(vd[:L].cpu().numpy(), v.numpy()) < 1e-5
    fn = _norm(hidden[0].double().cpu(), _t(params["norm.weight"]), cfg.rms_eps)
    assert orc.rel_err(final.cpu().numpy(), fn.numpy()) < 1e-6
    head = held(fn)[0] @ held(torch.from_numpy(params["llm_decoder.weight"]))[0].t()
    assert orc.rel_err(logits.cpu().numpy(), head.numpy()) < 1e-5
    lm.close()


def test_switching_back_gives_the_fp32_bits(gpu, lm8):
    cfg, params, lm = lm8
    x = lm.build_lm_input([1, 2, 3], list(range(60)))
    got = []
    for bits in (32, 8, 32, 8):
        lm.set_prefill_bits(bits)
        got.append(lm.prefill(x))
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    assert not torch.equal(got[0], got[1])
    # eight bits of weights and rows: a few percent a projection
    assert ((got[0] - got[1]).norm() / got[0].norm()).item() < 0.3


def test_decode_goes_on(gpu, lm8):
    """Decode over the cache that an 8-bit prefill left, against the oracle over the same cache."""
    cfg, params, lm = lm8
    lm.set_prefill_bits(8)
    L = lm.build_lm_input([5, 6, 7], list(range(40)))
    lm.prefill(L)
    o = orc.Qwen2(params, cfg, cap=320)
    for i in range(cfg.n_layers):
        for cache, dev in zip((o.k_cache, o.v_cache), lm.cache_views(i)):
            cache[i, :L.shape[0]] = dev[:L.shape[0]].cpu().numpy()
    o.cache_len = L.shape[0]
    for tok in (99, 6560):
        lg = lm.decode(tok)
        torch.cuda.synchronize()
        assert orc.rel_err(lg.cpu().numpy(), o.decode(tok)[0]) < 1e-5


@pytest.mark.parametrize("bits", [32, 8])
def test_score(gpu, lm8, bits):
    cfg, params, lm = lm8
    announce(f"score {bits} bits")
    lm.set_prefill_bits(bits)
    text, prompt, toks = [11, 12, 13], [100, 200], [7, 6560, 3, 3, 42]
    got = lm.score(text, prompt, toks, top=6)
    x = lm.build_lm_input(text, prompt + toks[:-1])
    logits = lm.prefill(x)[-len(toks):].double().cpu()
    assert lm.cache_len == 2 + 3 + 2 + 4
    lp = torch.log_softmax(logits, 1)
    ids = torch.tensor(toks)
    # fp32 logits alike: the scores' own rounding (test_gpu_logprobs), 230 * 2^-24 and a last place
    tol = 230 * 2.0 ** -24 + 2.0 ** -24 * 20
    assert ((got.logp.cpu().double() - lp[torch.arange(5), ids]).abs() <= tol).all()
    top = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :6]
    assert torch.equal(got.top_ids.cpu().long(), top)
    H = -(lp.exp() * lp).sum(1)
    assert ((got.entropy.cpu().double() - H).abs() <= 4 * tol * H).all()
    # as the tokens decoded one by one: the row before each gives its score
    one = lm.score(text, prompt + toks[:2], toks[2:3])
    assert (one.logp - got.logp[2]).abs().item() < (1e-3 if bits == 8 else 1e-4)


def test_score_refusals(gpu, lm8):
    from larynx_amd import LxError
    lm = lm8[2]
    with pytest.raises(ValueError):
        lm.score([1], [2], [])
    for toks in ([6761], [-1], [3, 7000]):
        with pytest.raises(ValueError):
            lm.score([1], [2], toks)
    with pytest.raises(LxError):
        lm.score([1], [2], [7000, 3])


def test_captured_prefills_outlive_the_switch(gpu, lm8):
    """A captured prefill gives what it was captured on, whatever runs between its replays."""
    announce("captured 8-bit prefill")
    cfg, params, lm = lm8
    xs = [torch.randn(50, cfg.hidden, generator=torch.Generator().manual_seed(i)).to(gpu)
          for i in range(3)]
    lm.set_prefill_bits(8)
    want = [lm.prefill(x) for x in xs]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lm.prefill(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = lm.prefill(x)
    for i, bits in ((1, 32), (2, 8), (0, 32), (1, 8)):
        lm.set_prefill_bits(bits)
        eager = lm.prefill(xs[2])
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want[i])
        assert torch.equal(eager, want[2]) == (bits == 8)


def test_refusals(gpu, lm8):
    from larynx_amd import LxError
    lm = lm8[2]
    for bits in (4, 16, 0, -8):
        with pytest.raises(LxError):
            lm.set_prefill_bits(bits)


def test_together(gpu):
    """As a caller runs them: the stream's sum and norm, the head's projection, its scores."""
    announce("norm, projection and scores together")
    g = torch.Generator().manual_seed(4)
    rows, H, V = 70, 896, 6761
    x, add = torch.randn(rows, H, generator=g), torch.randn(rows, H, generator=g)
    w = 1 + 0.1 * torch.randn(H, generator=g)
    head = torch.randn(V, H, generator=g) * 0.1
    t = torch.randint(0, V, (rows,), generator=g).int()
    xd = x.to(gpu)
    hq = ops.q8_pack(head.to(gpu))
    y = ops.rms_norm_q8(xd, w.to(gpu), add=add.to(gpu))
    got = ops.token_logprobs(ops.linear_q8(y, hq), t.to(gpu), top=5)
    h = x + add
    assert torch.equal(xd.cpu(), h)
    eps = float(torch.tensor(1e-6))
    n = held(_norm(h.double(), w.double(), eps))[0]
    hw = held(head)[0]
    lp = torch.log_softmax(n @ hw.t(), 1)
    # logits off by the products' bound, and the scores by twice that and their own rounding
    S = (n.abs() @ hw.abs().t()).amax(1)
    tol = 2 * (H + 16) * 2.0 ** -23 * S + 230 * 2.0 ** -24 + 2.0 ** -19
    assert ((got.logp.cpu().double() - lp[torch.arange(rows), t.long()]).abs() <= tol).all()
    assert ((got.top_logp.cpu().double() - lp.topk(5, 1).values).abs() <= tol[:, None]).all()
