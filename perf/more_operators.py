"""The language model's prompt in eight bits, and its scoring, as measurable cases: the
residual's addition with an RMSNorm into 8-bit rows, projections of 8-bit rows on 8-bit weights,
and log probabilities of given tokens with entropy and top alternatives.

With `own` false run() computes them from elementary torch operations (any tree), with `own`
true through larynx_amd.ops.  Widths are the LM's own (Qwen2Config) or generic ones.

A matrix in 8 bits: blocks of 128 consecutive elements of a row (the last one short where the
row ends inside it) share 2^e, e the smallest integer >= -127 with max|v| <= 448 * 2^e; an
element is the e4m3 number nearest to v / 2^e (ties to the even code) and stands for that
number times 2^e.  The norm is formed in 64 bits, since a code next to a border decides a
whole step.
"""
import math

import torch

own = False

DEV = "cuda"
HIDDEN, INTER, HEADS, KV_HEADS, HD = 896, 4864, 14, 2, 64  # Qwen2Config
SPEECH_VOCAB, TEXT_VOCAB = 6761, 151936
SPEECH_TOKENS = 6561  # ids past the codebook are control tokens
BLOCK, TOP_CODE = 128, 448.0  # e4m3's largest number
EPS = float(torch.tensor(1e-6, dtype=torch.float32))
WIDE = 8192


def listed():
    return [
        # the input norm of one row: the smallest call
        dict(name="norm_1", kind="norm", rows=1, D=HIDDEN, add=True),
        # between two layers of a prompt with a long reference voice
        dict(name="norm_1531", kind="norm", rows=1531, D=HIDDEN, add=True),
        # a norm alone, at an odd width
        dict(name="norm_333_odd", kind="norm", rows=333, D=1001, add=False),
        # a wide layer's norm for a large batch: the most bytes
        dict(name="norm_8192_wide", kind="norm", rows=8192, D=WIDE, add=True),
        # the LM's fused q|k|v projection of one row (with bias): the smallest call
        dict(name="linear_qkv_1", kind="linear", M=1, N=HIDDEN + 2 * KV_HEADS * HD, K=HIDDEN,
             epi="bias"),
        # gate/up with SwiGLU, rows interleaved, over a prompt of 256
        dict(name="linear_gate_up_256", kind="linear", M=256, N=2 * INTER, K=HIDDEN, epi="swiglu"),
        # down into the residual stream, a prompt with a long reference voice
        dict(name="linear_down_1531", kind="linear", M=1531, N=HIDDEN, K=INTER, epi="resid"),
        # the speech head (an odd number of rows) over a short prompt
        dict(name="linear_head_177", kind="linear", M=177, N=SPEECH_VOCAB, K=HIDDEN, epi="none"),
        # a wide layer for a large batch: the most operations
        dict(name="linear_wide_4096", kind="linear", M=4096, N=WIDE, K=WIDE, epi="gelu"),
        # one decoded speech token with five alternatives: the smallest call
        dict(name="logprob_1", kind="logprob", rows=1, V=SPEECH_VOCAB, top=5),
        # scoring an utterance of 1531 tokens
        dict(name="logprob_1531", kind="logprob", rows=1531, V=SPEECH_VOCAB, top=0),
        # scoring 1000 positions over the text vocabulary with 20 alternatives: the most bytes
        dict(name="logprob_text_1000", kind="logprob", rows=1000, V=TEXT_VOCAB, top=20),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "logprob"])
    if kind == "norm":
        D = rng.choice([HIDDEN, _log_int(rng, 64, WIDE), _log_int(rng, 64, WIDE)])
        rows = _log_int(rng, 1, min(8192, 8192 * WIDE // D))
        return dict(kind=kind, rows=rows, D=D, add=rng.random() < 0.7)
    if kind == "linear":
        M = _log_int(rng, 1, 4096)
        K = rng.choice([HIDDEN, INTER, _log_int(rng, 64, WIDE), _log_int(rng, 64, WIDE)])
        N = _log_int(rng, 16, WIDE if rng.random() < 0.8 else min(TEXT_VOCAB, 134_000_000 // K))
        N = min(N, max(16, 2 ** 38 // (M * K)))
        epi = rng.choice(["none", "bias", "gelu", "resid", "swiglu"])
        if epi == "swiglu":
            N += N % 2
        return dict(kind=kind, M=M, N=N, K=K, epi=epi)
    V = rng.choice([SPEECH_VOCAB, _log_int(rng, 100, TEXT_VOCAB), TEXT_VOCAB])
    return dict(kind=kind, rows=_log_int(rng, 1, min(4096, 1000 * TEXT_VOCAB // V)), V=V,
                top=rng.choice([0, 1, rng.randint(2, 20), rng.randint(21, 64)]))


def work(case):
    if case["kind"] == "norm":
        n = case["rows"] * case["D"]
        scales = case["rows"] * -(-case["D"] // BLOCK)
        # rows in (and the sums out), codes out; the read-back: codes in, fp32 rows out
        return {"bytes": (12 if case["add"] else 4) * n + 2 * (n + scales) + 4 * n
                + 4 * case["D"], "flops": 8 * n}
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        cols = N // 2 if case["epi"] == "swiglu" else N
        b = (M + N) * (K + -(-K // BLOCK)) + 4 * M * cols
        if case["epi"] == "resid":
            b += 4 * M * N
        if case["epi"] == "bias":
            b += 4 * N
        return {"bytes": b, "flops": 2 * M * N * K}
    n, rows, top = case["rows"] * case["V"], case["rows"], case["top"]
    return {"bytes": 4 * n + rows * (4 + 8 + 8 * top), "flops": 5 * n}


# ---- inputs ---------------------------------------------------------------------------


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g).mul_(std)


def _norm_inputs(case, seed):
    """A residual stream with the few large channels that trained models have, the output of a
    layer to add to it, norm weights around one."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, D = case["rows"], case["D"]
    x = _randn(g, rows, D)
    x[:, ::97] *= 20.0
    add = _randn(g, rows, D, std=0.3) if case["add"] else None
    return x, add, _randn(g, D, std=0.2).add_(1.0)


def _linear_inputs(case, seed):
    """Weights at a trained layer's scale (std 1 / sqrt(K), a few large ones), activations of a
    normalised row, a residual stream."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    M, N, K = case["M"], case["N"], case["K"]
    W = _randn(g, N, K, std=K ** -0.5)
    W.view(-1)[:: 997].mul_(4.0)
    x = _randn(g, M, K)
    b = _randn(g, N, std=0.1) if case["epi"] == "bias" else None
    y = _randn(g, M, N) if case["epi"] == "resid" else None
    return W, x, b, y


def _logprob_inputs(case, seed):
    """Logits of a head (a few candidates far ahead), control tokens masked in every other row
    of speech logits; tokens mostly likely ones, some rows padding."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, V = case["rows"], case["V"]
    x = _randn(g, rows, V, std=2.0)
    ahead = torch.randint(0, V, (rows, 8), device=DEV, generator=g)
    x.scatter_add_(1, ahead, _randn(g, rows, 8, std=6.0).abs_())
    if V == SPEECH_VOCAB:
        x[::2, SPEECH_TOKENS:] = float("-inf")
    t = torch.where(torch.rand(rows, device=DEV, generator=g) < 0.7, ahead[:, 0],
                    torch.randint(0, V, (rows,), device=DEV, generator=g)).int()
    t[16::17] = -1
    return x, t


# ---- the plain forms ------------------------------------------------------------------


def _pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quant(v):
    """v (rows, K) -> e4m3 numbers (rows, K / 128 up, 128) and 2^e (.., 1), both in 64 bits."""
    v = torch.nn.functional.pad(v.double(), (0, -v.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))  # m in [1/2, 1)
    # 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-127)
    e = torch.where(m > 0, e, torch.full_like(e, -127))
    v = v * _pow2(-e)
    step = torch.frexp(v)[1].clamp(min=-5) - 4  # four significant bits, down to 2^-9
    return torch.round(v * _pow2(-step)) * _pow2(step), _pow2(e)


def _quant_codes(x):
    """The two as held: float8 codes and fp32 powers of two, in pieces of rows."""
    step = max(1, (1 << 26) // x.shape[1])
    parts = [_quant(x[r:r + step]) for r in range(0, x.shape[0], step)]
    return (torch.cat([q.to(torch.float8_e4m3fn) for q, _ in parts]),
            torch.cat([s.float() for _, s in parts]))


def _plain_norm(st):
    h = st["x"] + st["add"] if st["add"] is not None else st["x"]
    d = h.double()
    y = d / torch.sqrt(d.square().mean(1, keepdim=True) + EPS) * st["w"].double()
    q, s = _quant(y)
    y = (q * s).flatten(1)[:, :h.shape[1]].float()
    return (h, y) if st["add"] is not None else y


def _plain_linear(st):
    (qx, sx), (qw, sw) = st["xq"], st["wq"]
    acc = (qx.float() * sx).flatten(1) @ (qw.float() * sw).flatten(1).t()
    if st["epi"] == "bias":
        return acc + st["b"]
    if st["epi"] == "gelu":
        return 0.5 * acc * (1.0 + torch.tanh(0.7978845608028654 * (acc + 0.044715 * acc ** 3)))
    if st["epi"] == "resid":
        return st["y"] + acc
    if st["epi"] == "swiglu":
        g, u = acc[:, 0::2], acc[:, 1::2]
        return g / (1.0 + torch.exp(-g)) * u
    return acc


def _plain_logprob(st):
    x, t, top = st["x"], st["t"].long(), st["top"]
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    S = e.double().sum(1)
    ls = torch.log(S)
    given = d.gather(1, t.clamp(min=0)[:, None])[:, 0].double() - ls
    logp = torch.where(t >= 0, given, torch.zeros_like(given)).float()
    # a masked logit adds nothing
    T = torch.where(e > 0, e * d, torch.zeros_like(e)).double().sum(1)
    H = (ls - T / S).float()
    if not top:
        return logp, H
    # whole numbers that order as (value, lower index first); + 0.0 makes one of both zeros
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    key = order * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[1], device=x.device))
    ids = 2 ** 32 - 1 - (key.topk(top, 1).values & (2 ** 32 - 1))
    return logp, H, (d.gather(1, ids).double() - ls[:, None]).float(), ids.int()


# ---- the operators --------------------------------------------------------------------


def prepare(case, seed):
    st = dict(case)
    if own:
        from larynx_amd import ops
    if case["kind"] == "norm":
        st["x"], st["add"], st["w"] = _norm_inputs(case, seed)
        st["h"] = torch.empty_like(st["x"]) if case["add"] else None
    elif case["kind"] == "linear":
        W, x, st["b"], st["y"] = _linear_inputs(case, seed)
        pack = ops.q8_pack if own else _quant_codes
        st["wq"], st["xq"] = pack(W), pack(x)
        if own:
            kinds = {"none": None, "bias": None, "gelu": ops.LX_EPI_GELU_TANH,
                     "resid": ops.LX_EPI_RESID, "swiglu": ops.LX_EPI_SWIGLU_PAIRED}
            kind = kinds[case["epi"]]
            st["epilogue"] = None if kind is None else ops.Epilogue(kind=kind)
    else:
        st["x"], st["t"] = _logprob_inputs(case, seed)
    return st


def run(st):
    kind = st["kind"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "logprob": _plain_logprob}[kind](st)
    from larynx_amd import ops
    if kind == "norm":
        # the sum goes beside the stream, so that every pass adds to the same rows
        y = ops.rms_norm_q8(st["x"], st["w"], EPS, add=st["add"], sum_out=st["h"])
        y = ops.q8_unpack(y)
        return (st["h"], y) if st["add"] is not None else y
    if kind == "linear":
        return ops.linear_q8(st["xq"], st["wq"], st["b"], epilogue=st["epilogue"], resid=st["y"])
    got = ops.token_logprobs(st["x"], st["t"], top=st["top"])
    return (got.logp, got.entropy, got.top_logp, got.top_ids) if st["top"] else \
        (got.logp, got.entropy)


# ---- the definitions in 64 bits -------------------------------------------------------


def _e4m3_numbers():
    """All numbers >= 0 by their codes 0 .. 126: seven thirds of 2^-9 below 2^-6, then eight
    steps an octave."""
    low = [i * 2.0 ** -9 for i in range(8)]
    return torch.tensor(low + [(8 + i) * 2.0 ** (p - 10) for p in range(1, 16) for i in range(8)]
                        [:119], device=DEV, dtype=torch.float64)


def _exact_held(v):
    """What 8 bits hold of v (rows, K) in 64 bits."""
    table = _e4m3_numbers()
    borders = (table[:-1] + table[1:]) / 2
    powers = torch.tensor([2.0 ** i for i in range(-160, 160)], device=DEV, dtype=torch.float64)
    out = torch.empty_like(v)
    for k in range(0, v.shape[1], BLOCK):
        b = v[:, k:k + BLOCK]
        top = b.abs().max(1, keepdim=True).values
        # the first power not below top / 448 (a power of two times 448 is exact), from 2^-127
        s = powers[torch.searchsorted(TOP_CODE * powers, top).clamp(min=160 - 127)]
        a = (b.abs() / s).contiguous()
        i = torch.searchsorted(borders, a)  # borders before a
        tie = (i < len(borders)) & (borders[i.clamp(max=len(borders) - 1)] == a)
        i = torch.where(tie & (i % 2 == 1), i + 1, i)
        out[:, k:k + BLOCK] = torch.sign(b) * table[i] * s
    return out


def exact(case, seed):
    if case["kind"] == "norm":
        x, add, w = _norm_inputs(case, seed)
        h = x if add is None else (x.double() + add.double()).float()
        y = torch.empty(h.shape, dtype=torch.float64, device=DEV)
        for r in range(0, h.shape[0], 1024):
            d = h[r:r + 1024].double()
            power = torch.linalg.vector_norm(d, dim=1, keepdim=True) ** 2 / d.shape[1]
            y[r:r + 1024] = _exact_held(d * ((power + EPS) ** -0.5) * w.double())
        return y if add is None else (x.double() + add.double(), y)
    if case["kind"] == "linear":
        W, x, b, y = _linear_inputs(case, seed)
        acc = _exact_held(x.double()) @ _exact_held(W.double()).t()
        if case["epi"] == "bias":
            acc += b.double()
        elif case["epi"] == "gelu":
            acc = acc / (1.0 + torch.exp(-1.5957691216057308 * (acc + 0.044715 * acc * acc * acc)))
        elif case["epi"] == "resid":
            acc += y.double()
        elif case["epi"] == "swiglu":
            acc = acc[:, 0::2] * torch.sigmoid(acc[:, 0::2]) * acc[:, 1::2]
        return acc
    x, t = _logprob_inputs(case, seed)
    out = []
    for r in range(0, x.shape[0], 128):
        lp = torch.log_softmax(x[r:r + 128].double(), 1)
        tr = t[r:r + 128].long()
        given = torch.where(tr < 0, torch.zeros_like(lp[:, 0]),
                            lp[torch.arange(len(tr), device=DEV), tr.clamp(min=0)])
        H = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
        got = [given, H]
        if case["top"]:
            v, i = torch.sort(x[r:r + 128], dim=1, descending=True, stable=True)
            i = i[:, :case["top"]]
            got += [lp.gather(1, i), i.int()]
        out.append(got)
    return tuple(torch.cat([o[j] for o in out]) for j in range(len(out[0])))
