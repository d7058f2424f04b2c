"""The 8-bit and scoring entry points without a GPU: sizes, and what they refuse before any work."""
import copy
import ctypes as C
import pickle

import pytest
import torch

from larynx_amd import ops
from larynx_amd._lib import (LX_EPI_GATED_RESID, LX_EPI_GELU_TANH, LX_EPI_RESID,
                             LX_EPI_ROPE_PARTIAL, LX_EPI_SWIGLU_PAIRED, LX_ERR_ARG, Epilogue, Q8,
                             lib)
from q8_reference import E4M3, held

P = 4096  # stands for a device address: nothing below may reach the device
O = 1 << 40  # another, for outputs


def test_reference_is_the_format():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(E4M3, codes)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 300, generator=g, dtype=torch.float64).float()
    v, s = held(x)
    for b in range(3):
        blk = x[:, 128 * b:128 * b + 128]
        top = blk.abs().amax(1)
        assert (top <= 448 * s[:, b]).all() and (top > 224 * s[:, b]).all()
        want = (blk.double() / s[:, b:b + 1]).float().to(torch.float8_e4m3fn).double()
        assert torch.equal(v[:, 128 * b:128 * b + 128], want * s[:, b:b + 1])


def test_sizes():
    # tiles of 16 rows x 128 elements at 2 KB, and 16 bytes of scales each
    assert lib.lx_q8_bytes(1152, 896) == 72 * 7 * 2064
    assert lib.lx_q8_bytes(1, 1) == 2064
    assert lib.lx_q8_bytes(17, 129) == 2 * 2 * 2064
    assert lib.lx_q8_bytes(151936, 8192) == 9496 * 64 * 2064
    assert lib.lx_q8_bytes(1 << 22, 8192) == (1 << 18) * 64 * 2064  # past 32 bits
    for bad in [(0, 1), (1, 0), (-1, 5), (5, -1), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1)]:
        assert lib.lx_q8_bytes(*bad) == 0, bad


def _q(data=P, rows=8, K=256):
    return C.byref(Q8(data, rows, K))


BAD = [dict(data=None), dict(data=P + 8), dict(rows=0), dict(rows=-1), dict(K=0), dict(K=-5),
       dict(rows=2 ** 31 - 1), dict(K=2 ** 31 - 1)]


@pytest.mark.parametrize("kw", BAD)
def test_bad_matrices(kw):
    bad = _q(**kw)
    ld = 2 ** 32
    assert lib.lx_q8_pack_f32(O, ld, bad, None) == LX_ERR_ARG
    assert b"q8_pack" in lib.lx_last_error()
    assert lib.lx_q8_unpack_f32(bad, O, ld, None) == LX_ERR_ARG
    assert b"q8_unpack" in lib.lx_last_error()
    assert lib.lx_rmsnorm_q8_f32(O, ld, None, 0, None, 0, O, 1e-6, bad, None) == LX_ERR_ARG
    assert b"rmsnorm_q8" in lib.lx_last_error()
    for x, w in [(bad, _q()), (_q(), bad)]:
        assert lib.lx_linear_q8_f32(x, w, None, None, None, 0, O, ld, None) == LX_ERR_ARG
        assert b"linear_q8" in lib.lx_last_error()


def test_null_matrices():
    assert lib.lx_q8_pack_f32(O, 256, None, None) == LX_ERR_ARG
    assert lib.lx_q8_unpack_f32(None, O, 256, None) == LX_ERR_ARG
    assert lib.lx_rmsnorm_q8_f32(O, 256, None, 0, None, 0, O, 1e-6, None, None) == LX_ERR_ARG
    assert lib.lx_linear_q8_f32(None, _q(), None, None, None, 0, O, 8, None) == LX_ERR_ARG
    assert lib.lx_linear_q8_f32(_q(), None, None, None, None, 0, O, 8, None) == LX_ERR_ARG


def test_pack_refusals():
    for x, ld in [(None, 256), (O, 255), (O + 2, 256), (O, -1)]:
        assert lib.lx_q8_pack_f32(x, ld, _q(), None) == LX_ERR_ARG
        assert lib.lx_q8_unpack_f32(_q(), x, ld, None) == LX_ERR_ARG
    huge = _q(rows=2 ** 30, K=256)  # more lanes than a launch has
    assert lib.lx_q8_pack_f32(O, 256, huge, None) == LX_ERR_ARG
    assert lib.lx_q8_unpack_f32(huge, O, 256, None) == LX_ERR_ARG


NORM = dict(x=O, ldx=256, add=None, lda=0, sum=None, lds=0, w=P, q=None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(ldx=255), dict(x=O + 1), dict(w=P + 2),
    dict(add=O, lda=256), dict(sum=O, lds=256),  # one without the other
    dict(add=2 * O, lda=255, sum=3 * O, lds=256), dict(add=2 * O, lda=256, sum=3 * O, lds=255),
    dict(add=2 * O + 1, lda=256, sum=3 * O, lds=256),
    # sum over part of x or of add, or over x at another stride
    dict(add=2 * O, lda=256, sum=O + 4, lds=256), dict(add=2 * O, lda=256, sum=2 * O + 8, lds=256),
    dict(add=2 * O, lda=256, sum=O, lds=260),
])
def test_norm_refusals(kw):
    a = {**NORM, **kw}
    assert lib.lx_rmsnorm_q8_f32(a["x"], a["ldx"], a["add"], a["lda"], a["sum"], a["lds"], a["w"],
                                 1e-6, _q(), None) == LX_ERR_ARG
    assert b"rmsnorm_q8" in lib.lx_last_error()


@pytest.mark.parametrize("rows,K", [(2 ** 23, 2049), (2 ** 23, 10 ** 5), (2 ** 25, 896)])
def test_norm_too_many_rows(rows, K):
    assert lib.lx_rmsnorm_q8_f32(O, K, None, 0, None, 0, P, 1e-6, _q(rows=rows, K=K),
                                 None) == LX_ERR_ARG
    assert b"too many" in lib.lx_last_error()


def _linear(x=None, w=None, bias=None, kind=None, resid=None, ldr=0, y=O, ldy=32):
    epi = None if kind is None else C.byref(Epilogue(kind=kind))
    return lib.lx_linear_q8_f32(x or _q(), w or _q(rows=32), bias, epi, resid, ldr, y, ldy, None)


@pytest.mark.parametrize("kw", [
    dict(y=None), dict(ldy=31), dict(y=O + 2), dict(bias=P + 1), dict(w=_q(rows=32, K=255)),
    dict(kind=LX_EPI_GATED_RESID), dict(kind=LX_EPI_ROPE_PARTIAL), dict(kind=9), dict(kind=-1),
    dict(kind=LX_EPI_SWIGLU_PAIRED, w=_q(rows=31)), dict(kind=LX_EPI_SWIGLU_PAIRED, ldy=15),
    dict(resid=P, ldr=32), dict(resid=P, ldr=32, kind=LX_EPI_GELU_TANH),
    dict(resid=P, ldr=31, kind=LX_EPI_RESID), dict(resid=P + 1, ldr=32, kind=LX_EPI_RESID),
    dict(resid=O + 4, ldr=32, kind=LX_EPI_RESID), dict(resid=O, ldr=36, kind=LX_EPI_RESID),
])
def test_linear_refusals(kw):
    assert _linear(**kw) == LX_ERR_ARG
    assert b"linear_q8" in lib.lx_last_error()


def test_linear_too_many_outputs():
    big = _q(rows=2 ** 31 - 16)
    assert _linear(x=big, w=big, ldy=2 ** 31) == LX_ERR_ARG


SCORE = dict(x=O, ld=1000, rows=4, V=1000, tokens=P, logp=P, ent=P, top=3, tl=P, ti=P, ws=None, n=0)


def _score(**kw):
    a = {**SCORE, **kw}
    return lib.lx_token_logprobs_f32(a["x"], a["ld"], a["rows"], a["V"], a["tokens"], a["logp"],
                                     a["ent"], a["top"], a["tl"], a["ti"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(rows=0), dict(rows=-1), dict(V=0), dict(V=2 ** 24 + 1, ld=2 ** 25),
    dict(top=-1), dict(top=65), dict(V=2, top=3), dict(ld=999), dict(tokens=None), dict(logp=None),
    dict(tl=None), dict(ti=None), dict(tokens=None, logp=None, ent=None, top=0), dict(x=O + 2),
    dict(tokens=P + 1), dict(logp=P + 2), dict(ent=P + 2), dict(tl=P + 2), dict(ti=P + 1),
    dict(rows=2 ** 24, V=10 ** 6, ld=10 ** 6),
])
def test_score_refusals(kw):
    assert _score(**kw) == LX_ERR_ARG
    assert b"token_logprobs" in lib.lx_last_error()


def test_score_workspace():
    assert lib.lx_token_logprobs_ws_floats(1531, 6761, 64) == 0
    assert lib.lx_token_logprobs_ws_floats(5, 8192, 1) == 0
    for bad in [(0, 9000, 1), (1, 0, 1), (1, 9000, 65), (1, 9000, -1), (1, 2 ** 24 + 1, 0)]:
        assert lib.lx_token_logprobs_ws_floats(*bad) == 0
    need = lib.lx_token_logprobs_ws_floats(4, 20000, 3)
    assert need > 0
    for ws, n in [(None, need), (P, need - 1), (P + 8, need)]:
        assert _score(V=20000, ld=20000, ws=ws, n=n) == LX_ERR_ARG
        assert b"workspace" in lib.lx_last_error()


A, Q8_BYTES = 1 << 41, 4128  # an 8-bit matrix (8, 256)


@pytest.mark.parametrize("where", ["first", "last", "before"])
def test_outputs_over_inputs(where):
    """fp32 rows (8, 256) of stride 300 with elements in an 8-bit matrix's memory, one of the two
    written."""
    def rows(cols):
        return {"first": A, "last": A + Q8_BYTES - 4, "before": A - 4 * (7 * 300 + cols) + 4}[where]

    at = rows(256)
    q, other = _q(data=A), _q(data=1 << 50)
    far = 1 << 51
    calls = {
        "pack": lambda: lib.lx_q8_pack_f32(at, 300, q, None),
        "unpack": lambda: lib.lx_q8_unpack_f32(q, at, 300, None),
        "x": lambda: lib.lx_rmsnorm_q8_f32(at, 300, None, 0, None, 0, P, 1e-6, q, None),
        "x of a sum": lambda: lib.lx_rmsnorm_q8_f32(at, 300, far, 256, 2 * far, 256, P, 1e-6, q,
                                                    None),
        "add": lambda: lib.lx_rmsnorm_q8_f32(far, 256, at, 300, 2 * far, 256, P, 1e-6, q, None),
        "sum": lambda: lib.lx_rmsnorm_q8_f32(far, 256, 2 * far, 256, at, 300, P, 1e-6, q, None),
        "sum in place": lambda: lib.lx_rmsnorm_q8_f32(at, 300, far, 256, at, 300, P, 1e-6, q, None),
        "y over x": lambda: lib.lx_linear_q8_f32(q, _q(data=1 << 50, rows=256), None, None, None, 0,
                                                 at, 300, None),
        "y over w": lambda: lib.lx_linear_q8_f32(other, q, None, None, None, 0, rows(8), 300, None),
    }
    for name, call in calls.items():
        assert call() == LX_ERR_ARG, name
        assert b"overlap" in lib.lx_last_error(), (name, lib.lx_last_error())


def test_outputs_over_vectors():
    """The norm's weight under its sum or its codes, a bias under y."""
    far = 1 << 51
    for w, s in [(far + 4 * 255, far), (far - 4 * 255, far), (far + 4 * (7 * 256 + 255), far)]:
        assert lib.lx_rmsnorm_q8_f32(2 * far, 256, 3 * far, 256, s, 256, w, 1e-6, _q(data=A),
                                     None) == LX_ERR_ARG
        assert b"overlap" in lib.lx_last_error()
    for w in (A, A + Q8_BYTES - 4, A - 4 * 255):
        assert lib.lx_rmsnorm_q8_f32(2 * far, 256, None, 0, None, 0, w, 1e-6, _q(data=A),
                                     None) == LX_ERR_ARG
        assert b"overlap" in lib.lx_last_error()
    for b in (O, O - 4 * 31, O + 4 * (7 * 32 + 31)):
        assert _linear(bias=b) == LX_ERR_ARG
        assert b"overlap" in lib.lx_last_error()


@pytest.mark.parametrize("at", [O, O + 4 * (3 * 1100 + 999), O - 4])
def test_scores_over_logits(at):
    """Outputs with an element in the first or last of the rows of logits, workspaces too."""
    for kw in [dict(logp=at), dict(ent=at), dict(tl=at), dict(ti=at),
               dict(tokens=None, logp=None, ent=at, top=0)]:
        assert _score(ld=1100, **kw) == LX_ERR_ARG, kw
        assert b"overlaps the logits" in lib.lx_last_error(), kw
    need = lib.lx_token_logprobs_ws_floats(4, 20000, 3)
    for ws in (O, O - 4 * need + 16, O + 4 * (3 * 20100 + 19996)):
        assert _score(V=20000, ld=20100, ws=ws, n=need) == LX_ERR_ARG, ws
        assert b"overlaps the logits" in lib.lx_last_error()


def test_ops_refuse_host_tensors():
    x, w = torch.zeros(4, 256), torch.ones(256)
    with pytest.raises(ValueError, match="current device"):
        ops.q8_pack(x)
    with pytest.raises(ValueError, match="current device"):
        ops.rms_norm_q8(x, w)
    with pytest.raises(ValueError, match="current device"):
        ops.token_logprobs(x)
    q = ops.Q8Matrix(torch.zeros(lib.lx_q8_bytes(4, 256), dtype=torch.uint8), 4, 256)
    with pytest.raises(ValueError, match="current device"):
        ops.q8_unpack(q)
    with pytest.raises(ValueError, match="current device"):
        ops.linear_q8(q, q)


def test_matrix_of_other_bytes():
    n = lib.lx_q8_bytes(4, 256)
    for data in [torch.zeros(n - 1, dtype=torch.uint8), torch.zeros(n, dtype=torch.int8),
                 torch.zeros(2 * n, dtype=torch.uint8)[::2]]:
        with pytest.raises(ValueError, match="8-bit"):
            ops.Q8Matrix(data, 4, 256)
    with pytest.raises(ValueError, match="8-bit"):
        ops.Q8Matrix(torch.zeros(n, dtype=torch.uint8), 0, 256)


def test_matrix_copies():
    """A copy names its own bytes, not those of the matrix that it was made from; what a matrix says
    of itself does not change under it."""
    n = lib.lx_q8_bytes(4, 256)
    q = ops.Q8Matrix(torch.arange(n).to(torch.uint8), 4, 256)
    for c in [copy.deepcopy(q), pickle.loads(pickle.dumps(q)), copy.copy(q)]:
        assert (c.rows, c.K) == (4, 256) and torch.equal(c.data, q.data)
        assert Q8.from_buffer_copy(c._ref).data == c.data.data_ptr()
    assert copy.deepcopy(q).data.data_ptr() != q.data.data_ptr()
    for name, value in [("data", torch.zeros(n, dtype=torch.uint8)), ("rows", 3), ("K", 128)]:
        with pytest.raises(AttributeError):
            setattr(q, name, value)


@pytest.mark.parametrize("x", [torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4),
                               torch.zeros(8, 4).t(), torch.zeros(2, 4, 8)])
def test_ops_refuse_other_layouts(x):
    for call in [ops.q8_pack, ops.token_logprobs, lambda t: ops.rms_norm_q8(t, torch.ones(8))]:
        with pytest.raises(ValueError):
            call(x)


def test_struct_layout():
    from test_abi import _c_layout
    fields = [f[0] for f in Q8._fields_]
    got = _c_layout("lx_q8", fields)
    assert got[0] == C.sizeof(Q8) and got[1:] == [getattr(Q8, f).offset for f in fields]
