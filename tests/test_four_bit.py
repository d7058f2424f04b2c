"""The four-bit entry points without a GPU: sizes, and what they refuse before any work."""
import ctypes as C

import pytest
import torch

from larynx_amd import ops
from larynx_amd._lib import (LX_EPI_GATED_RESID, LX_EPI_ROPE_PARTIAL,
                             LX_EPI_SWIGLU_PAIRED, LX_ERR_ARG, Epilogue, Kv4, lib)

P = 4096  # stands for a device address: nothing below may reach the device
O = 1 << 40  # another, for outputs


def test_sizes():
    # codes: tiles of 16 rows x 128 inputs at 1 KB; 16 bf16 scales per tile and group
    assert lib.lx_q4_bytes(1152, 896, 64) == 72 * 7 * (1024 + 2 * 32)
    assert lib.lx_q4_bytes(17, 132, 32) == 2 * 2 * (1024 + 4 * 32)
    assert lib.lx_q4_bytes(1, 4, 128) == 1024 + 32
    for bad in [(0, 4, 64), (1, 0, 64), (1, 6, 64), (1, 4, 16), (1, 4, 0), (-1, 4, 64),
                (2 ** 31 - 1, 2 ** 31 - 4, 64), (2 ** 28, 128, 64), (16, 2 ** 31 - 4, 64)]:
        assert lib.lx_q4_bytes(*bad) == 0, bad
    # records of 32 rows: 2304 bytes per 64 channels
    assert lib.lx_kv4_bytes(1, 2, 64, 4096) == 2 * 128 * 2304
    assert lib.lx_kv4_bytes(3, 1, 128, 33) == 3 * 2 * 2 * 2304
    assert lib.lx_kv4_bytes(64, 32, 128, 1 << 22) == 64 * 32 * (1 << 17) * 4608  # past 32 bits
    for bad in [(0, 1, 64, 1), (1, 0, 64, 1), (1, 1, 32, 1), (1, 1, 96, 1), (1, 1, 64, 0),
                (1, 1, 64, -5), (1, 1, 64, 2 ** 31 - 1), (1, 1, 64, 2 ** 31 - 128),
                (65536, 4, 64, 1), (4, 32768, 64, 1)]:
        assert lib.lx_kv4_bytes(*bad) == 0, bad


def test_pack_refusals():
    for args in [(None, P, 16, 64, 64), (P, None, 16, 64, 64), (P, P, 0, 64, 64),
                 (P, P, 16, 62, 64), (P, P, 16, 64, 48), (P + 4, P, 16, 64, 64),
                 (P, P + 8, 16, 64, 64)]:
        assert lib.lx_q4_pack_f32(*args, None) == LX_ERR_ARG, args
    for args in [(None, P, 16, 64, 64), (P, None, 16, 64, 64), (P, P, 16, 64, 63),
                 (P + 4, P, 16, 64, 64)]:
        assert lib.lx_q4_unpack_f32(*args, None) == LX_ERR_ARG, args


def _linear(x=P, ldx=64, w=P, group=64, bias=None, y=O, ldy=32, M=1, N=32, K=64, kind=None,
            ws=None, n=0):
    epi = None if kind is None else C.byref(Epilogue(kind=kind))
    return lib.lx_linear_q4_f32(x, ldx, w, group, bias, y, ldy, M, N, K, epi, ws, n, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(y=None), dict(M=0), dict(M=65), dict(M=-1), dict(N=0),
    dict(K=62, ldx=64), dict(ldx=60), dict(ldx=66), dict(ldy=31), dict(group=16), dict(x=P + 4),
    dict(w=P + 8), dict(y=O + 2), dict(bias=P + 1), dict(kind=LX_EPI_GATED_RESID),
    dict(kind=LX_EPI_ROPE_PARTIAL), dict(kind=9), dict(kind=-1),
    dict(kind=LX_EPI_SWIGLU_PAIRED, N=31), dict(kind=LX_EPI_SWIGLU_PAIRED, ldy=15),
])
def test_linear_refusals(kw):
    assert _linear(**kw) == LX_ERR_ARG
    assert b"linear_q4" in lib.lx_last_error()


def test_linear_workspace():
    # up to 4 rows, and K up to 1024, take none
    for M, N, K in [(1, 896, 4864), (4, 151936, 8192), (8, 896, 896), (64, 9728, 1024)]:
        assert lib.lx_linear_q4_ws_floats(M, N, K) == 0
    for bad in [(0, 896, 896), (65, 896, 896), (17, 0, 896), (17, 896, 6)]:
        assert lib.lx_linear_q4_ws_floats(*bad) == 0
    need = lib.lx_linear_q4_ws_floats(64, 1000, 8192)
    assert need and need % (64 * 1008) == 0
    assert lib.lx_linear_q4_ws_floats(1, 151936, 896) == 0
    K = 2 ** 26  # more splits than a launch has rows of workgroups
    assert _linear(M=5, N=16, K=K, ldx=K, ldy=16, ws=P, n=2 ** 40) == LX_ERR_ARG
    for ws, n in [(None, need), (P, need - 1), (P + 4, need)]:
        assert _linear(M=64, N=1000, K=8192, ldx=8192, ldy=1000, ws=ws, n=n) == LX_ERR_ARG
        assert b"workspace" in lib.lx_last_error()


def _cache(data=P, batch=2, heads=2, hd=64, rows=100):
    return C.byref(Kv4(data, batch, heads, hd, rows))


@pytest.mark.parametrize("cache", [
    dict(data=None), dict(data=P + 8), dict(batch=0), dict(heads=0), dict(hd=80), dict(rows=0)])
def test_bad_caches(cache):
    c = _cache(**cache)
    assert lib.lx_kv4_append_f32(c, P, 128, P, 128, 1, P, None) == LX_ERR_ARG
    assert lib.lx_kv4_read_f32(c, P, P, 1, P, None) == LX_ERR_ARG
    assert lib.lx_attention_kv4_f32(P, 256, c, P, O, 256, 1, 4, 0.125, 1, 0, None, 0,
                                    None) == LX_ERR_ARG
    assert lib.lx_attention_kv4_ws_floats(c, 1, 4, 0) == 0
    assert lib.lx_attention_kv4_ws_floats(None, 1, 4, 0) == 0


def test_cache_call_refusals():
    c = _cache()
    for args in [(None, 128, P, 128, 1, P), (P, 128, None, 128, 1, P), (P, 128, P, 128, 1, None),
                 (P, 127, P, 128, 1, P), (P, 128, P, 64, 1, P), (P, 128, P, 128, 0, P),
                 (P, 128, P, 128, -3, P)]:
        assert lib.lx_kv4_append_f32(c, *args, None) == LX_ERR_ARG, args
    for args in [(None, P, 1, P), (P, None, 1, P), (P, P, 0, P), (P, P, 1, None)]:
        assert lib.lx_kv4_read_f32(c, *args, None) == LX_ERR_ARG, args
    ok = dict(q=P, ldq=256, cache=c, lens=P, o=O, ldo=256, Tq=1, heads=4)
    for kw in [dict(q=None), dict(lens=None), dict(o=None), dict(ldq=252), dict(ldq=258),
               dict(ldo=252), dict(ldo=257), dict(Tq=0), dict(heads=3), dict(heads=0),
               dict(q=P + 4), dict(o=O + 8), dict(Tq=2 ** 31 - 1)]:
        a = {**ok, **kw}
        assert lib.lx_attention_kv4_f32(a["q"], a["ldq"], a["cache"], a["lens"], a["o"], a["ldo"],
                                        a["Tq"], a["heads"], 0.125, 1, 0, None, 0,
                                        None) == LX_ERR_ARG, kw
    # few workgroups over many rows: the keys are split, which takes a workspace
    big = _cache(batch=1, rows=4096)
    need = lib.lx_attention_kv4_ws_floats(big, 1, 4, 0)
    assert need > 0
    for ws, n in [(None, need), (P, need - 1), (P + 8, need)]:
        assert lib.lx_attention_kv4_f32(P, 256, big, P, O, 256, 1, 4, 0.125, 1, 0, ws, n,
                                        None) == LX_ERR_ARG
        assert b"workspace" in lib.lx_last_error()


@pytest.mark.parametrize("y,ldy,shared", [
    (0, 4096, True), (2044, 4096, True), (2048, 4096, False), (2048, 4000, True),
    (4064, 4096, False), (4068, 4096, True), (4096, 4096, True), (-32, 4096, False),
    (-28, 4096, True), (-4096, 4096, True), (15 * 4096 + 2048, 96, False),
    (15 * 4096 + 2044, 96, True), (-(15 * 4096 + 32), 4096, False), (-15 * 4096, 4096, True)])
def test_outputs_over_inputs_are_refused(y, ldy, shared):
    """16 rows of 2048 inputs, 4096 apart; 32 outputs y floats on.  The others are refused for the
    workspace they need."""
    x = 1 << 30
    rc = _linear(x=x, ldx=4096, y=x + 4 * y, ldy=ldy, M=16, N=32, K=2048)
    assert rc == LX_ERR_ARG
    assert (b"overlaps" if shared else b"workspace") in lib.lx_last_error()


@pytest.mark.parametrize("o,ldo,shared", [
    (0, 512, True), (256, 512, False), (252, 512, True), (512, 512, True), (1024, 256, False),
    (764, 512, True), (-256, 512, False), (-252, 512, True), (128, 256, True)])
def test_attention_outputs_over_queries_are_refused(o, ldo, shared):
    """2 sequences of a row of 256, 512 apart, over caches that take splits."""
    q, c = 1 << 30, _cache(batch=2, rows=4096)
    assert lib.lx_attention_kv4_f32(q, 512, c, P, q + 4 * o, ldo, 1, 4, 0.125, 1, 0, None, 0,
                                    None) == LX_ERR_ARG
    assert (b"overlaps" if shared else b"workspace") in lib.lx_last_error()


def test_python_refuses_host_tensors():
    x = torch.zeros(1, 64)
    with pytest.raises(ValueError):
        ops.q4_pack(x)
    w = ops.Q4Weight(torch.zeros(1024 + 64, dtype=torch.uint8), 16, 64, 64)
    with pytest.raises(ValueError):
        ops.linear_q4(x, w)
    with pytest.raises(ValueError):
        ops.q4_unpack(w)
    with pytest.raises(ValueError):
        ops.kv4_cache(1, 2, 16, head_dim=80)
    cache = ops.Kv4Cache(torch.zeros(4608, dtype=torch.uint8), 1, 2, 64, 16)
    kv, n = torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv4_append(cache, kv, kv, n)
    with pytest.raises(ValueError):
        ops.kv4_read(cache, n, 1)
    with pytest.raises(ValueError):
        ops.attention_kv4(torch.zeros(1, 1, 128), cache, n, 2)


@pytest.mark.parametrize("shape,want,strides,ok", [
    ((3, 64), (3, 64), None, 64), ((3, 64), (3, 64), (80, 1), 80), ((1, 64), (1, 64), (7, 1), 64),
    ((3, 64), (3, 60), None, None), ((3, 64), (2, 64), None, None), ((3, 64), (3, 64), (1, 3), None),
    ((2, 3, 64), (2, 3, 64), None, 64), ((2, 3, 64), (2, 3, 64), (240, 80, 1), 80),
    ((2, 3, 64), (2, 3, 64), (250, 80, 1), None), ((2, 1, 64), (2, 1, 64), (96, 5, 1), 96),
    ((1, 3, 64), (1, 3, 64), (7, 64, 1), 64), ((1, 1, 64), (1, 1, 64), (7, 7, 1), 64),
    ((2, 3, 64), (6, 64), None, None)])
def test_row_strides(shape, want, strides, ok):
    t = torch.zeros(shape) if strides is None else torch.zeros(1000).as_strided(shape, strides)
    if ok is None:
        with pytest.raises(ValueError):
            ops._rows(t, "t", want)
    else:
        assert ops._rows(t, "t", want) == ok


def test_types_and_containers():
    with pytest.raises(ValueError):
        ops._rows(torch.zeros(2, 64, dtype=torch.float16), "t", (2, 64))
    cache = ops.Kv4Cache(torch.zeros(2 * 4608, dtype=torch.uint8), 2, 2, 64, 16)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32),
                torch.zeros(4, dtype=torch.int32)[::2], torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            cache._check(bad, "n")
    with pytest.raises(ValueError):
        ops.Kv4Cache(torch.zeros(4608, dtype=torch.uint8), 2, 2, 64, 16)
    with pytest.raises(ValueError):
        ops.Kv4Cache(torch.zeros(4608 // 4), 1, 2, 64, 16)
    with pytest.raises(ValueError):
        ops.Q4Weight(torch.zeros(2111, dtype=torch.uint8), 16, 64, 64)
    with pytest.raises(ValueError):
        ops.Q4Weight(torch.zeros(0, dtype=torch.uint8), 16, 62, 64)


def test_struct_layout_matches_header():
    from test_abi import _c_layout
    fields = [f[0] for f in Kv4._fields_]
    got = _c_layout("lx_kv4", fields)
    assert got[0] == C.sizeof(Kv4)
    assert got[1:] == [getattr(Kv4, f).offset for f in fields]


def test_decode_bits_refuse_a_null_model():
    assert lib.lx_qwen2_set_decode_bits(None, 4, 64) == LX_ERR_ARG
