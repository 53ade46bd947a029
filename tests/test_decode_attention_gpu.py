"""Attention of one new token per sequence over a cache, against a 64-bit restatement."""
import math

import pytest
import torch

from ragged_oracle import LSE_TOL, SECOND, U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def oracle(q, k, v, lengths, scale):
    """(out, lse, bound of out): P is rounded once before P V, and the output once; parts are joined in FP32."""
    B, H, d = q.shape
    out, tol = torch.zeros(B, H, d, dtype=torch.float64, device=DEV), torch.zeros(B, H, d, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=DEV)
    G = H // k.shape[2]
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        K, V = (t[b, :n].double().repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))  # (H, n, d)
        s = (K @ q[b].double()[:, :, None])[..., 0] * scale
        lse[b] = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[b][:, None])[:, None]
        out[b] = (p @ V)[:, 0]
        tol[b] = U * ((p @ V.abs())[:, 0] + out[b].abs())
    return out, lse, tol * SECOND + 1e-5


def check(got, want):
    out, lse, tol = want
    assert bool(((got[0].double() - out).abs() <= tol).all()), float(((got[0].double() - out).abs() - tol).max())
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got[1]), empty)
    assert bool(((got[1].double() - lse)[~empty].abs() <= LSE_TOL).all())


def make(B, T, H, Hkv, d, seed=0, heads_first=False):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(torch.bfloat16)
    if heads_first:
        return rnd(B, H, d), rnd(B, Hkv, T, d).transpose(1, 2), rnd(B, Hkv, T, d).transpose(1, 2)
    return rnd(B, H, d), rnd(B, T, Hkv, d), rnd(B, T, Hkv, d)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (8, 2), (7, 1), (16, 1), (20, 1), (33, 1), (24, 2)])
@pytest.mark.parametrize("T,lengths", [(1, [1, 0]), (16, [16, 3]), (100, [100, 17, 0, 1]), (700, [700, 129]), (5000, [4999, 1, 300])])
def test_against_the_oracle(pkg, T, lengths, H, Hkv, d):
    q, k, v = make(len(lengths), T, H, Hkv, d, seed=T + H)
    scale = 1.0 / math.sqrt(d)
    for b, n in enumerate(lengths):  # what lies behind a length is never read
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    check(pkg.ops.attention_decode_bf16(q, k, v, ints(lengths), scale), oracle(q, k, v, lengths, scale))


@pytest.mark.parametrize("heads_first", [False, True])
def test_layouts_and_strides(pkg, heads_first):
    B, T, H, Hkv, d = 3, 333, 6, 2, 64
    lengths = [333, 200, 64]
    q, k, v = make(B, T, H, Hkv, d, seed=1, heads_first=heads_first)
    v = v.clone(memory_format=torch.contiguous_format)  # another order than k
    wide = torch.zeros(B, (H + 4) * d, dtype=torch.bfloat16, device=DEV)
    wide[:, : H * d] = q.view(B, -1)
    check(pkg.ops.attention_decode_bf16(wide[:, : H * d].view(B, H, d), k[:, :], v, ints(lengths), 0.125), oracle(q, k, v, lengths, 0.125))
    check(pkg.ops.attention_decode_bf16(q, k[:, :300], v[:, :300], ints([300, 200, 64]), 0.125), oracle(q, k, v, [300, 200, 64], 0.125))


def test_cache_shared_by_all_sequences(pkg):
    q, k, v = make(3, 500, 4, 2, 128, seed=2)
    k1, v1 = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    check(pkg.ops.attention_decode_bf16(q, k1, v1, ints([500, 77, 300]), 0.1), oracle(q, k1, v1, [500, 77, 300], 0.1))


def test_empty_caches_and_no_sequences(pkg):
    q, k, v = make(2, 0, 4, 2, 64)
    out, lse = pkg.ops.attention_decode_bf16(q, k, v, ints([0, 5]), 0.1)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    q, k, v = make(0, 10, 4, 2, 64)
    out, lse = pkg.ops.attention_decode_bf16(q, k, v, ints([]), 0.1)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_lengths_are_clipped_and_results_repeat(pkg):
    q, k, v = make(2, 3000, 8, 2, 64, seed=3)
    a = pkg.ops.attention_decode_bf16(q, k, v, ints([3000, 0]), 0.125)
    for wild in ([1 << 30, -7], [3001, 0]):
        b = pkg.ops.attention_decode_bf16(q, k, v, ints(wild), 0.125)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_large_scores(pkg):
    q, k, v = make(2, 900, 4, 2, 64, seed=4)
    q, k = q * 16, k * 16
    out, lse, tol = oracle(q, k, v, [900, 500], 0.125)
    got = pkg.ops.attention_decode_bf16(q, k, v, ints([900, 500]), 0.125)
    # scores of thousands in FP32: an error of 2^-21 of sum |q||k| is an absolute error of lse and a relative one of P
    err = 2.0 ** -21 * 0.125 * float((q.abs().double().amax((0, 1)) * k.abs().double().amax((0, 1, 2))).sum())
    assert bool(((got[0].double() - out).abs() <= tol + 2 * err * 6).all())
    assert bool(((got[1].double() - lse).abs() <= err).all())


def test_offsets_beyond_32_bits(pkg):
    """A cache of more than 2^31 elements: the last sequence lies behind them."""
    B, T, Hkv, d = 3, 131072, 48, 128
    k = torch.zeros(B, T, Hkv, d, dtype=torch.bfloat16, device=DEV)
    assert k.numel() > 2 ** 31
    q, k2, v2 = make(1, T, Hkv, Hkv, d, seed=5)
    k[2] = k2[0]
    q3 = q.expand(3, -1, -1).contiguous()
    got = pkg.ops.attention_decode_bf16(q3, k, k, ints([4, 0, T]), 0.088)
    want = oracle(q, k2, k2, [T], 0.088)
    check((got[0][2:], got[1][2:]), want)


def test_captured_and_on_two_streams(pkg):
    pkg.ops.reserve(1, 128, 64)
    graphs = []
    for seed, (B, T, H, Hkv, d) in enumerate([(2, 2000, 8, 2, 128), (1, 5000, 4, 4, 64)]):
        q, k, v = make(B, T, H, Hkv, d, seed=30 + seed)
        n, stream = ints([T] * B), torch.cuda.Stream()
        with torch.cuda.stream(stream):
            pkg.ops.attention_decode_bf16(q, k, v, n, 0.1)
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                got = pkg.ops.attention_decode_bf16(q, k, v, n, 0.1)
        graphs.append((g, stream, q, k, v, n, got))
    for length in (1, 1999, 130):
        for g, stream, q, k, v, n, got in graphs:
            n.fill_(length)
            q.neg_()
        torch.cuda.synchronize()
        for g, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for g, stream, q, k, v, n, got in graphs:
            check(got, oracle(q, k, v, [length] * q.shape[0], 0.1))


def test_refusals(pkg):
    ops, Err = pkg.ops, pkg.lib.B200AttnError
    q, k, v = make(2, 64, 4, 2, 64)
    n = ints([64, 3])
    for a in [(q.float(), k, v, n), (q[:1], k, v, n), (q, k[:, :, :, :32], v, n), (q[:, :3], k, v, n), (q, k, v[:, :50], n), (q, k.float(), v, n), (q, k, v, n.long()),
              (q, k, v, n[:1]), (q, k, v, n.cpu()), (q.cpu(), k, v, n), (q, k.transpose(2, 3).contiguous().transpose(2, 3), v, n),
              (q, torch.empty(2, 64, 2, 68, dtype=torch.bfloat16, device=DEV)[..., :64], v, n)]:
        with pytest.raises(Err):
            ops.attention_decode_bf16(*a, 0.1)
    with pytest.raises(Err):
        ops.attention_decode_bf16(q, k, v, n, 0.0)
    with pytest.raises(Err):
        ops.attention_decode_bf16(q, k, v, n, 0.1, out=torch.empty(2, 4, 32, dtype=torch.bfloat16, device=DEV))
    x = torch.zeros(2, 4, 96, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(Err) as e:
        ops.attention_decode_bf16(x, x[:, :, None].contiguous().view(2, 4, 1, 96), x.view(2, 4, 1, 96), n, 0.1)
    assert e.value.code == pkg.lib.ERR_UNSUPPORTED
