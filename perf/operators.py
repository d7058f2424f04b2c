"""The four-bit operators of the language model, as measurable cases: projections of few rows
on 4-bit weights with group scales, the append to a cache held in 4 bits with its read-back,
and attention over that cache.

With `own` false run() computes them from elementary torch operations (any tree), with `own`
true through larynx_amd.ops.  Widths are the LM's own (Qwen2Config) or generic ones.

A 4-bit weight: groups of G consecutive inputs of a row share a bf16 scale s = bf16(v / -8),
v the group's value of largest magnitude (the first of equals); q = clamp(rint(w / s) + 8, 0,
15) stands for s * (q - 8).  A cached key or value: the 64 channels of a group share z, the
largest bf16 not above their minimum, and s, the smallest bf16 not below (max - z) / 15; q =
clamp(rint((x - z) / s), 0, 15) stands for z + s * q.  Quotients are formed in 64 bits, since
a code next to a border decides a whole step.
"""
import math

import torch

own = False

DEV = "cuda"
HIDDEN, INTER, HEADS, KV_HEADS, HD = 896, 4864, 14, 2, 64  # Qwen2Config
SPEECH_VOCAB, TEXT_VOCAB = 6761, 151936
CACHE_GROUP = 64


def listed():
    return [
        # the LM's fused q|k|v projection of one decoded token (with bias): the smallest call
        dict(name="linear_qkv_1", kind="linear", M=1, N=HIDDEN + 2 * KV_HEADS * HD, K=HIDDEN,
             group=64, epi="bias"),
        # its gate/up projection with SwiGLU, rows interleaved
        dict(name="linear_gate_up_1", kind="linear", M=1, N=2 * INTER, K=HIDDEN, group=64,
             epi="swiglu"),
        # its down projection into the residual stream, four utterances decoded side by side
        dict(name="linear_down_4", kind="linear", M=4, N=HIDDEN, K=INTER, group=64, epi="resid"),
        # the speech head (an odd number of rows), three candidates
        dict(name="linear_head_3", kind="linear", M=3, N=SPEECH_VOCAB, K=HIDDEN, group=32,
             epi="none"),
        # the text table as an output head for a batch of 16: the most weight bytes
        dict(name="linear_vocab_16", kind="linear", M=16, N=TEXT_VOCAB, K=HIDDEN, group=64,
             epi="none"),
        # a wide layer for a batch of 64: the most rows
        dict(name="linear_wide_64", kind="linear", M=64, N=8192, K=8192, group=128, epi="gelu"),
        # one decoded token into the cache
        dict(name="append_1", kind="append", B=1, T=1, kv=KV_HEADS, hd=HD, pos=2047),
        # a prompt with a long reference voice into the cache
        dict(name="append_prompt", kind="append", B=1, T=1531, kv=KV_HEADS, hd=HD, pos=0),
        # one decoded token late in a long utterance
        dict(name="attend_1_2001", kind="attend", B=1, Tq=1, heads=HEADS, kv=KV_HEADS, hd=HD,
             ctx=2001),
        # 48 utterances of all lengths (an idle slot among them) decoded side by side
        dict(name="attend_48_4000", kind="attend", B=48, Tq=1, heads=HEADS, kv=KV_HEADS, hd=HD,
             ctx=4000),
        # wide heads over long contexts: the most cache bytes
        dict(name="attend_2_65536", kind="attend", B=2, Tq=1, heads=32, kv=8, hd=128, ctx=65536),
        # a chunk of a prompt over what is cached of it
        dict(name="attend_chunk_177", kind="attend", B=1, Tq=177, heads=HEADS, kv=KV_HEADS, hd=HD,
             ctx=1708),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "append", "attend", "attend"])
    if kind == "linear":
        K = 4 * _log_int(rng, 16, 2048)
        N = _log_int(rng, 16, min(TEXT_VOCAB, 67_000_000 // K))
        epi = rng.choice(["none", "bias", "gelu", "resid", "swiglu"])
        if epi == "swiglu":
            N += N % 2
        return dict(kind=kind, M=_log_int(rng, 1, 64), N=N, K=K,
                    group=rng.choice([32, 64, 128]), epi=epi)
    heads, kv, hd = rng.choice([(HEADS, KV_HEADS, HD), (HEADS, KV_HEADS, HD), (16, 16, 64),
                                (32, 8, 128), (8, 1, 128)])
    if kind == "append":
        T = _log_int(rng, 1, 1531)
        return dict(kind=kind, B=_log_int(rng, 1, max(1, 1531 * 128 // (T * kv * hd))), T=T, kv=kv,
                    hd=hd, pos=rng.randint(0, 4096 - T))
    Tq = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 256)])
    # caches up to the long case's bytes, products up to the chunk's
    ctx = _log_int(rng, max(1, Tq), 65536)
    most = min(2 * 65536 * 8 * 128 // (ctx * kv * hd),
               2 * 65536 * 32 * 128 // (ctx * Tq * heads * hd))
    while most < 1:
        ctx = max(Tq, ctx // 2)
        Tq = min(Tq, ctx)
        most = min(2 * 65536 * 8 * 128 // (ctx * kv * hd),
                   2 * 65536 * 32 * 128 // (ctx * Tq * heads * hd))
    return dict(kind=kind, B=_log_int(rng, 1, min(64, most)), Tq=Tq, heads=heads, kv=kv, hd=hd,
                ctx=ctx)


def _lens(case):
    """Cached rows of each sequence: all lengths up to ctx, one slot idle in a batch of 8 on."""
    B, ctx = case["B"], case["ctx"]
    lens = [max(1, -(-ctx * (i + 1) // B)) for i in range(B)]
    if B >= 8:
        lens[B // 2] = 0
    return lens


def work(case):
    if case["kind"] == "linear":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        cols = N // 2 if case["epi"] == "swiglu" else N
        b = N * K // 2 + 2 * N * -(-K // G) + 4 * M * K + 4 * M * cols
        if case["epi"] == "resid":
            b += 4 * M * N
        if case["epi"] == "bias":
            b += 4 * N
        return {"bytes": b, "flops": 2 * M * N * K}
    width = case["kv"] * case["hd"]
    row = width // 2 + 4 * (width // CACHE_GROUP)  # one row's keys, or values, in 4 bits
    if case["kind"] == "append":
        rows = case["B"] * case["T"]
        # fp32 rows in, codes out; the read-back: codes in, fp32 rows out
        return {"bytes": 2 * rows * (2 * 4 * width + 2 * row), "flops": 2 * rows * width * 6}
    keys, n, Tq = sum(_lens(case)), case["heads"] * case["hd"], case["Tq"]
    seen = sum(sum(max(0, l - Tq + t + 1) for t in range(Tq)) for l in _lens(case))
    return {"bytes": 2 * keys * row + 2 * 4 * case["B"] * Tq * n, "flops": 4 * seen * n}


# ---- inputs ---------------------------------------------------------------------------


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g).mul_(std)


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


def _kv(g, B, T, kv, hd):
    """Keys with the large fixed offsets of some channels that rotary models show, and values."""
    off = _randn(g, 1, 1, kv, hd)
    off[..., ::16] *= 8.0
    k = _randn(g, B, T, kv, hd).add_(off)
    v = _randn(g, B, T, kv, hd)
    return k, v


def _cache_inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    B, kv, hd = case["B"], case["kv"], case["hd"]
    if case["kind"] == "append":
        k, v = _kv(g, B, case["T"], kv, hd)
        pos = torch.full((B,), case["pos"], dtype=torch.int32, device=DEV)
        return k, v, pos
    # scores of standard deviation about 2 around each row's own mean
    q = _randn(g, B, case["Tq"], case["heads"] * hd, std=2.0)
    lens = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
    k, v = _kv(g, B, case["ctx"], kv, hd)
    return q, k, v, lens


# ---- the plain forms ------------------------------------------------------------------


def _bf16_not_above(x):
    """Largest bf16 <= x (fp32)."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where((x < 0) & (cut != bits), cut + 65536, cut).view(torch.float32)


def _bf16_not_below(r):
    """Smallest bf16 >= r >= 0 (64 bits)."""
    f = r.float()
    bits = f.view(torch.int32) + (f.double() < r).int()
    return ((bits + 65535) & -65536).view(torch.float32)


def _quant_cache(x):
    """x (..., hd) -> codes uint8 (..., hd / 64, 64), z and s (..., hd / 64, 1)."""
    x = x.unflatten(-1, (-1, CACHE_GROUP))
    z = _bf16_not_above(x.amin(-1, keepdim=True))
    d = x.amax(-1, keepdim=True).double() - z.double()
    s = _bf16_not_below(d / torch.full_like(d, 15.0))
    q = torch.round((x.double() - z.double()) / s.double()).clamp_(0, 15)
    return torch.where(s > 0, q, torch.zeros_like(q)).to(torch.uint8), z, s


def _quant_cache_rows(x, step=4096):
    """_quant_cache of (B, T, kv, hd) in pieces of T (the 64-bit intermediates are large)."""
    parts = [_quant_cache(x[:, t:t + step]) for t in range(0, x.shape[1], step)]
    return tuple(torch.cat([p[i] for p in parts], 1) for i in range(3))


def _dequant_cache(c):
    q, z, s = c
    return (z + s * q.float()).flatten(-2)


def _quant_weight(W, G):
    """Codes uint8 (N, K / G up, G) and scales fp32 (N, K / G up, 1)."""
    N, K = W.shape
    w = torch.nn.functional.pad(W, (0, -K % G)).view(N, -1, G)
    at = w.abs().argmax(-1, keepdim=True)  # the first of equals
    s = (w.gather(-1, at) * -0.125).bfloat16().float()
    q = torch.empty(w.shape, dtype=torch.uint8, device=w.device)
    for n in range(0, N, 16384):
        r = torch.round(w[n:n + 16384].double() / s[n:n + 16384].double()).add_(8).clamp_(0, 15)
        q[n:n + 16384] = torch.where(s[n:n + 16384] != 0, r, torch.full_like(r, 8.0)).to(torch.uint8)
    return q, s


def _plain_linear(st):
    q, s = st["w"]
    W = (s * (q.float() - 8.0)).flatten(1)[:, :st["x"].shape[1]]
    acc = st["x"] @ W.t()
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


def _plain_attend(q, k, v, lens, heads):
    """q (B, Tq, heads * hd), k / v (B, ctx, kv, hd)."""
    B, Tq = q.shape[:2]
    ctx, kv, hd = k.shape[1:]
    rep = heads // kv
    qg = q.view(B, Tq, kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(B, kv, Tq * rep, hd)
    kt = k.permute(0, 2, 3, 1).contiguous()
    s = (qg @ kt).mul_(hd ** -0.5)
    last = lens.long()[:, None] - Tq + torch.arange(Tq, device=q.device)  # (B, Tq)
    seen = torch.arange(ctx, device=q.device) <= last.repeat_interleave(rep, 1)[..., None]
    s.masked_fill_(~seen[:, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > float("-inf"), m, torch.zeros_like(m)))
    l = p.sum(-1, keepdim=True)
    o = (p @ v.transpose(1, 2).contiguous()) / torch.where(l > 0, l, torch.ones_like(l))
    return o.view(B, kv, Tq, rep, hd).permute(0, 2, 1, 3, 4).reshape(B, Tq, heads * hd)


# ---- the operators --------------------------------------------------------------------


def prepare(case, seed):
    st = dict(case)
    if own:
        from larynx_amd import ops
    if case["kind"] == "linear":
        W, st["x"], st["b"], st["y"] = _linear_inputs(case, seed)
        st["w"] = ops.q4_pack(W, case["group"]) if own else _quant_weight(W, case["group"])
        if own:
            kinds = {"none": None, "bias": None, "gelu": ops.LX_EPI_GELU_TANH,
                     "resid": ops.LX_EPI_RESID, "swiglu": ops.LX_EPI_SWIGLU_PAIRED}
            kind = kinds[case["epi"]]
            st["epilogue"] = None if kind is None else ops.Epilogue(kind=kind)
        return st
    if case["kind"] == "append":
        k, v, st["pos"] = _cache_inputs(case, seed)
        st["k"], st["v"] = k.flatten(2), v.flatten(2)
        if own:
            st["cache"] = ops.kv4_cache(case["B"], case["kv"], 4096, case["hd"])
        return st
    st["q"], k, v, st["lens"] = _cache_inputs(case, seed)
    if own:
        st["cache"] = ops.kv4_cache(case["B"], case["kv"], case["ctx"], case["hd"])
        zero = torch.zeros(case["B"], dtype=torch.int32, device=DEV)
        ops.kv4_append(st["cache"], k.flatten(2), v.flatten(2), zero)
    else:
        st["k"], st["v"] = _quant_cache_rows(k), _quant_cache_rows(v)
    return st


def run(st):
    kind = st["kind"]
    if not own:
        if kind == "linear":
            return _plain_linear(st)
        if kind == "append":
            shape = st["k"].shape
            return tuple(_dequant_cache(_quant_cache(x.unflatten(2, (st["kv"], -1)))).reshape(shape)
                         for x in (st["k"], st["v"]))
        return _plain_attend(st["q"], _dequant_cache(st["k"]), _dequant_cache(st["v"]), st["lens"],
                             st["heads"])
    from larynx_amd import ops
    if kind == "linear":
        # a residual epilogue adds into the stream it is given: every pass adds to a copy
        out = st["y"].clone() if st["epi"] == "resid" else None
        return ops.linear_q4(st["x"], st["w"], st["b"], epilogue=st["epilogue"], out=out)
    if kind == "append":
        ops.kv4_append(st["cache"], st["k"], st["v"], st["pos"])
        return ops.kv4_read(st["cache"], st["pos"], st["T"])
    return ops.attention_kv4(st["q"], st["cache"], st["lens"], st["heads"], max_len=st["ctx"])


# ---- the definitions in 64 bits -------------------------------------------------------


def _eight_bits(x, to):
    """x (64 bits) with 8 significant bits, the whole number of them taken by `to`."""
    m, e = torch.frexp(x)
    power = ((e.long() + (1023 - 8)) << 52).view(torch.float64)  # 2^(e - 8), no pow rounding
    return to(m * 256.0) * power


def _exact_cache(x):
    """What the cache holds of x (..., hd), hd a multiple of 64."""
    x = x.double().reshape(*x.shape[:-1], -1, CACHE_GROUP)
    z = _eight_bits(x.min(-1, keepdim=True).values, torch.floor)
    s = _eight_bits((x.max(-1, keepdim=True).values - z) / torch.tensor(15.0, device=x.device,
                                                                        dtype=torch.float64),
                    torch.ceil)
    steps = torch.where(s > 0, ((x - z) / s).round(), torch.zeros_like(x))
    return (z + steps.clamp(0, 15) * s).flatten(-2)


def _exact_weight(W, G):
    out = torch.zeros_like(W, dtype=torch.float64)
    for k in range(0, W.shape[1], G):
        w = W[:, k:k + G].double()
        top = w.abs().max(1, keepdim=True)
        s = _eight_bits(-torch.gather(w, 1, top.indices) / 8.0, torch.round)
        steps = torch.where(s != 0, (w / s).round(), torch.zeros_like(w))
        out[:, k:k + G] = steps.clamp(-8, 7) * s
    return out


def exact(case, seed):
    if case["kind"] == "linear":
        W, x, b, y = _linear_inputs(case, seed)
        acc = x.double() @ _exact_weight(W, case["group"]).t()
        if case["epi"] == "bias":
            acc += b.double()
        elif case["epi"] == "gelu":
            acc = acc / (1.0 + torch.exp(-1.5957691216057308 * (acc + 0.044715 * acc * acc * acc)))
        elif case["epi"] == "resid":
            acc += y.double()
        elif case["epi"] == "swiglu":
            acc = acc[:, 0::2] * torch.sigmoid(acc[:, 0::2]) * acc[:, 1::2]
        return acc
    if case["kind"] == "append":
        k, v, _ = _cache_inputs(case, seed)
        return _exact_cache(k).flatten(2), _exact_cache(v).flatten(2)
    q, k, v, _ = _cache_inputs(case, seed)
    B, Tq, hd, rep = case["B"], case["Tq"], case["hd"], case["heads"] // case["kv"]
    out = torch.zeros(B, Tq, case["heads"], hd, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(case)):
        for g in range(case["kv"] if n else 0):
            kg, vg = _exact_cache(k[b, :n, g]), _exact_cache(v[b, :n, g])
            qs = q[b].double().view(Tq, case["heads"], hd)[:, g * rep:(g + 1) * rep]
            s = (qs.reshape(-1, hd) @ kg.t()).view(Tq, rep, n) / math.sqrt(hd)
            ahead = torch.arange(n, device=DEV) - (n - Tq + torch.arange(Tq, device=DEV))[:, None]
            s = s.masked_fill((ahead > 0)[:, None], -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # a row that sees no key is zero
            out[b, :, g * rep:(g + 1) * rep] = (p.reshape(-1, n) @ vg).view(Tq, rep, hd)
    return out.flatten(2)
