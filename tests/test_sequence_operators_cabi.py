"""What the C entries of the packed, single-token and log-probability calls refuse before they touch a GPU (the pointers here are
never read), the sizes of their workspaces, and what the Python functions say to tensors that are not on one."""
import ctypes
import importlib

import pytest
import torch

P = [ctypes.c_void_p(4096 * (i + 1)) for i in range(12)]
ODD = ctypes.c_void_p(4096 + 8)
ARG, UNSUPPORTED, SCRATCH = -1, -2, -4


@pytest.fixture(scope="module")
def so(pkg):
    import __graft_entry__ as entry
    import os
    if not os.path.exists(pkg.calls.SO_PATH):
        entry.build()
    return pkg.lib.load()


def fwd(so, q=P[0], k=P[1], v=P[2], offsets=P[3], out=P[4], lse=P[5], ws=P[6], nbytes=1 << 40, total=100, n=2, H=4, Hkv=2, d=64, sq=256, skv=128, so_=256, scale=0.1):
    return so.b200attn_fwd_bf16_ragged(q, k, v, offsets, out, lse, ws, nbytes, total, n, H, Hkv, d, sq, skv, so_, scale, None)


def bwd(so, q=P[0], k=P[1], v=P[2], out=P[3], dout=P[4], lse=P[5], offsets=P[6], dq=P[7], dk=P[8], dv=P[9], ws=P[10], nbytes=1 << 40, total=100, n=2, H=4, Hkv=2,
        d=64, sq=256, skv=128, so_=256, sdo=256, sdq=256, sdkv=128, scale=0.1):
    return so.b200attn_bwd_bf16_ragged(q, k, v, out, dout, lse, offsets, dq, dk, dv, ws, nbytes, total, n, H, Hkv, d, sq, skv, so_, sdo, sdq, sdkv, scale, None)


def dec(so, q=P[0], k=P[1], v=P[2], lengths=P[3], out=P[4], lse=P[5], ws=P[6], nbytes=1 << 40, B=2, T=100, H=4, Hkv=2, d=64, sq=256, k3=(12800, 128, 64),
        v3=(12800, 128, 64), scale=0.1):
    return so.b200attn_decode_bf16(q, k, v, lengths, out, lse, ws, nbytes, B, T, H, Hkv, d, sq, *k3, *v3, scale, None)


PACKED = [(dict(total=-1), ARG), (dict(n=-1), ARG), (dict(H=0), ARG), (dict(Hkv=0), ARG), (dict(Hkv=3), ARG), (dict(d=32), UNSUPPORTED), (dict(d=96), UNSUPPORTED),
          (dict(total=(1 << 30) + 1), UNSUPPORTED), (dict(H=65536 * 2, Hkv=1), UNSUPPORTED), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG),
          (dict(scale=float("inf")), ARG), (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(offsets=None), ARG), (dict(out=None), ARG), (dict(lse=None), ARG),
          (dict(ws=None), ARG), (dict(q=ODD), ARG), (dict(k=ODD), ARG), (dict(v=ODD), ARG), (dict(out=ODD), ARG), (dict(ws=ODD), ARG), (dict(sq=255), ARG), (dict(sq=260), ARG),
          (dict(sq=0), ARG), (dict(skv=120), ARG), (dict(skv=-128), ARG), (dict(so_=252), ARG), (dict(sq=1 << 40), ARG), (dict(nbytes=15), SCRATCH), (dict(nbytes=-1), SCRATCH)]


@pytest.mark.parametrize("change,code", PACKED, ids=lambda x: str(x))
def test_packed_attention_refuses(so, change, code):
    assert fwd(so, **change) == code
    assert b"ragged" in so.b200attn_last_error()
    assert bwd(so, **change) == code


@pytest.mark.parametrize("change", [dict(dq=None), dict(dk=ODD), dict(dv=None), dict(dout=None), dict(dout=ODD), dict(sdo=248), dict(sdq=255), dict(sdkv=64)], ids=str)
def test_packed_backward_refuses(so, change):
    assert bwd(so, **change) == ARG


def test_packed_attention_of_nothing(so):
    for f in (fwd, bwd):
        assert f(so, total=0, q=None, k=None, v=None, out=None, ws=None) == 0
        assert f(so, n=0, offsets=None) == 0


DECODE = [(dict(B=-1), ARG), (dict(T=-1), ARG), (dict(H=0), ARG), (dict(Hkv=3), ARG), (dict(d=80), UNSUPPORTED), (dict(B=65536), UNSUPPORTED), (dict(scale=0.0), ARG),
          (dict(scale=float("nan")), ARG), (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(lengths=None), ARG), (dict(out=None), ARG), (dict(lse=None), ARG),
          (dict(q=ODD), ARG), (dict(k=ODD), ARG), (dict(out=ODD), ARG), (dict(sq=-8), ARG), (dict(sq=4), ARG), (dict(k3=(12800, 130, 64)), ARG), (dict(v3=(12800, 128, -64)), ARG),
          (dict(T=1 << 20, nbytes=64), SCRATCH), (dict(T=1 << 20, ws=None), SCRATCH)]


@pytest.mark.parametrize("change,code", DECODE, ids=lambda x: str(x))
def test_single_token_attention_refuses(so, change, code):
    assert dec(so, **change) == code
    assert b"b200attn_decode_bf16" in so.b200attn_last_error()


def test_single_token_attention_of_nothing(so):
    assert dec(so, B=0, q=None, lengths=None, out=None) == 0


def test_workspace_sizes(so):
    size = so.b200attn_ragged_workspace_bytes
    assert size(-1, 1, 1, 1, 64, 0) == size(1, 1, 3, 2, 64, 0) == 0
    # the list holds one item per 128 rows and one more per sequence; 16 bytes each
    assert size(128 * 50, 7, 4, 2, 64, 0) >= 57 * 16
    # the backward: FP32 sums of dQ, two statistics, and for d = 64 two rows of 32 bytes
    rows = 1000 * 8
    assert size(1000, 3, 8, 8, 128, 1) >= rows * (128 * 4 + 8)
    assert size(1000, 3, 8, 8, 64, 1) >= rows * (64 * 4 + 8 + 64)
    # few key heads: partial dK and dV of up to every head of a group
    assert size(1000, 3, 8, 1, 128, 1) >= rows * (128 * 4 + 8) + 2 * 8 * 1000 * 128 * 4
    assert size(100000, 3, 8, 1, 128, 1) < 100000 * 8 * (128 * 4 + 8) * 1.1 + 2 * 100000 * 128 * 4
    assert so.b200attn_decode_workspace_bytes(64, 1024, 32, 8, 128) == 0  # few parts: they join inside a cluster
    assert so.b200attn_decode_workspace_bytes(1, 1 << 17, 32, 8, 128) > 32 * 8 * 130 * 4
    assert so.b200attn_decode_workspace_bytes(1, 1 << 17, 32, 7, 128) == 0


LP = dict(x=P[0], dtype=0, stride=50, t=P[1], rows=4, V=50, tau=1.0, lp=P[2], e=P[3], s=P[4], top=3, tl=P[5], tt=P[6])
LPG = dict(x=P[0], dtype=0, stride=50, t=P[1], e=P[2], s=P[3], g=P[4], ge=P[5], rows=4, V=50, tau=1.0, d=P[6], ds=50)


def logprobs(so, **change):
    a = LP | change
    return so.b200loss_token_logprobs(a["x"], a["dtype"], a["stride"], a["t"], a["rows"], a["V"], a["tau"], a["lp"], a["e"], a["s"], a["top"], a["tl"], a["tt"], None)


def logprobs_backward(so, **change):
    a = LPG | change
    return so.b200loss_token_logprobs_backward(a["x"], a["dtype"], a["stride"], a["t"], a["e"], a["s"], a["g"], a["ge"], a["rows"], a["V"], a["tau"], a["d"], a["ds"], None)


def test_token_logprobs_refuse(pkg):
    so = importlib.import_module(pkg.__name__ + ".loss_ops").load()
    both = [dict(dtype=2), dict(dtype=-1), dict(rows=-1), dict(V=0), dict(V=-5), dict(stride=49), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")), dict(tau=float("inf")),
            dict(tau=1e-7), dict(x=None), dict(t=None), dict(e=None), dict(s=None), dict(x=ctypes.c_void_p(4097)), dict(x=ctypes.c_void_p(4098))]
    for change in both + [dict(lp=None), dict(top=-1), dict(top=33), dict(top=20, V=19), dict(tl=None), dict(tt=None), dict(rows=1 << 30)]:
        assert logprobs(so, **change) == -1, change
        assert b"token_logprobs" in so.b200loss_last_error()
    for change in both + [dict(g=None), dict(d=None), dict(ds=49), dict(rows=1 << 30), dict(d=ctypes.c_void_p(4097))]:
        assert logprobs_backward(so, **change) == -1, change
    assert logprobs(so, rows=0, x=None, t=None) == 0 and logprobs_backward(so, rows=0, x=None, d=None) == 0


def test_tensors_that_are_not_on_a_gpu(pkg):
    ops, lo = pkg.ops, importlib.import_module(pkg.__name__ + ".loss_ops")
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(pkg.lib.B200AttnError):
        ops.attention_forward_bf16_ragged(q, q, q, n, 0.1)
    with pytest.raises(pkg.lib.B200AttnError):
        ops.attention_backward_bf16_ragged(q, q, q, q, q, q, n, 0.1)
    with pytest.raises(pkg.lib.B200AttnError):
        ops.attention_decode_bf16(q, q, q, n, 0.1)
    with pytest.raises(pkg.lib.B200AttnError):
        ops.attention_decode_bf16(None, q, q, n, 0.1)
    with pytest.raises(ValueError):
        lo.token_logprobs_forward(torch.zeros(2, 5), n)
    with pytest.raises(ValueError):
        lo.token_logprobs_backward(torch.zeros(2, 5), n, lo.TokenLogprobs(n, n, n, None, None, 1.0), n)
