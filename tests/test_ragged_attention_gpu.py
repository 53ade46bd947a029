"""Attention over packed sequences of different lengths with grouped heads (forward, backward) against the 64-bit oracle."""
import math

import pytest
import torch

from ragged_oracle import assert_close, attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("out", "lse", "dq", "dk", "dv")


def make(lengths, H, Hkv, d, behind=0, seed=0, fused=True):
    """Inputs for sum(lengths) + behind rows; with `fused` q, k, v are parts of one buffer."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(lengths) + behind
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(torch.bfloat16)
    if fused:
        buf = rnd(n, (H + 2 * Hkv) * d)
        q, k, v = (x.view(n, x.shape[1] // d, d) for x in buf.split([H * d, Hkv * d, Hkv * d], 1))
    else:
        q, k, v = rnd(n, H, d), rnd(n, Hkv, d), rnd(n, Hkv, d)
    ends = [0]
    for x in lengths:
        ends.append(ends[-1] + x)
    return q, k, v, rnd(n, H, d), torch.tensor(ends, dtype=torch.int32, device=DEV)


def run(ops, q, k, v, dout, offsets, scale, **given):
    out, lse = ops.attention_forward_bf16_ragged(q, k, v, offsets, scale, out=given.get("out"), lse=given.get("lse"))
    dq, dk, dv = ops.attention_backward_bf16_ragged(q, k, v, out, dout, lse, offsets, scale, dq=given.get("dq"), dk=given.get("dk"), dv=given.get("dv"))
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


LENGTHS = [[1], [5], [128], [129], [1, 1, 1], [0, 5, 0, 130, 0], [127, 128, 129], [300, 1, 64, 257], [513, 385], [17] * 9, [1500, 3]]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2), (6, 1), (21, 3)])
def test_forward_and_backward(pkg, lengths, H, Hkv, d):
    q, k, v, dout, offsets = make(lengths, H, Hkv, d, seed=len(lengths) * 7 + H)
    scale = 1.0 / math.sqrt(d)
    got = run(pkg.ops, q, k, v, dout, offsets, scale)
    pkg.ops.check_device_fault()
    assert_close(got, *attention(q, k, v, lengths, scale, dout), NAMES)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [0.02, 0.7])
def test_scales_and_large_scores(pkg, d, scale):
    lengths = [200, 77]
    q, k, v, dout, offsets = make(lengths, 2, 1, d, seed=3, fused=False)
    q, k = q * 4, k * 4  # scores of some hundreds: one key takes the whole row
    got = run(pkg.ops, q, k, v, dout, offsets, scale)
    val, tol = attention(q, k, v, lengths, scale, dout)
    # FP32 scores s carry an error of some 2^-21 of sum |q||k| scale, which P has as a relative error
    s_err = 2.0 ** -21 * float((q.abs().float().amax(0) * k.abs().float().amax()).sum(-1).amax()) * scale
    tol = {n: t + s_err * (1 + val[n].abs()) * (1 if n in ("out", "lse") else 40) for n, t in tol.items()}
    assert_close(got, val, tol, NAMES)


@pytest.mark.parametrize("d", [64, 128])
def test_many_short_sequences(pkg, d):
    lengths = [i % 4 for i in range(2600)] + [140]
    q, k, v, dout, offsets = make(lengths, 2, 1, d, seed=4)
    got = run(pkg.ops, q, k, v, dout, offsets, 0.1)
    assert_close(got, *attention(q, k, v, lengths, 0.1, dout), NAMES)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_no_sequence(pkg, d, bad):
    """Rows behind the last sequence hold what is not a number, are not read and not written."""
    lengths, H, Hkv, behind = [200, 70], 4, 2, 61
    q, k, v, dout, offsets = make(lengths, H, Hkv, d, behind=behind, seed=5)
    n = sum(lengths)
    for t in (q, k, v, dout):
        t[n:] = bad
    given = {name: torch.full((n + behind, heads, d), 7.0, dtype=torch.bfloat16, device=DEV) for name, heads in (("out", H), ("dq", H), ("dk", Hkv), ("dv", Hkv))}
    given["lse"] = torch.full((H, n + behind), 7.0, device=DEV)
    got = run(pkg.ops, q, k, v, dout, offsets, 0.125, **given)
    for name in NAMES:
        rows = got[name][:, n:] if name == "lse" else got[name][n:]
        assert bool((rows == 7.0).all()), name
    got = {name: got[name][:, :n] if name == "lse" else got[name][:n] for name in NAMES}
    assert_close(got, *attention(q, k, v, lengths, 0.125, dout), NAMES)
    fresh = run(pkg.ops, q, k, v, dout, offsets, 0.125)
    assert all(bool((fresh[name][n:] == 0).all()) for name in ("out", "dq", "dk", "dv")) and bool((fresh["lse"][:, n:] == 0).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_spoilt_sequence_spoils_no_other(pkg, d, bad):
    lengths = [90, 150, 200]
    q, k, v, dout, offsets = make(lengths, 4, 2, d, seed=6, fused=False)
    clean = run(pkg.ops, q, k, v, dout, offsets, 0.125)
    for t in (q, k, v, dout):
        t[90:240] = bad
    got = run(pkg.ops, q, k, v, dout, offsets, 0.125)
    for name in NAMES:
        for rows in (slice(0, 90), slice(240, 440)):
            a, b = (clean[name][:, rows], got[name][:, rows]) if name == "lse" else (clean[name][rows], got[name][rows])
            assert torch.equal(a, b), name  # at most two tiles meet in a dQ row: their sum has no order


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,H,Hkv", [([100 + 7 * i for i in range(20)], 6, 2), ([40, 900], 32, 8), ([700, 650, 500], 18, 2)], ids=["twenty", "two", "three"])
def test_other_grid_sizes(pkg, lengths, H, Hkv, d):
    """Grids between one and two CTAs per SM of short and of long sequences, and larger ones."""
    q, k, v, dout, offsets = make(lengths, H, Hkv, d, seed=14)
    got = run(pkg.ops, q, k, v, dout, offsets, 0.1)
    assert_close(got, *attention(q, k, v, lengths, 0.1, dout), NAMES)


@pytest.mark.parametrize("d", [64, 128])
def test_equal_lengths_agree_with_the_dense_path(pkg, d):
    """Bit by bit where both take the forward variant with two CTAs per SM: from 297 tiles and heads on."""
    B, H, T = 80, 2, 256
    q, k, v, dout, offsets = make([T] * B, H, H, d, seed=7, fused=False)
    got = run(pkg.ops, q, k, v, dout, offsets, 0.125)
    slab = lambda t: t.view(B, T, H, d).transpose(1, 2).contiguous()
    out, lse = pkg.ops.attention_forward_bf16(slab(q), slab(k), slab(v), 0.125)
    dq, dk, dv = pkg.ops.attention_backward_bf16(slab(q), slab(k), slab(v), out, slab(dout), lse, 0.125)
    assert torch.equal(slab(got["out"]), out)
    assert torch.equal(got["lse"].view(H, B, T).transpose(0, 1), lse)
    assert torch.equal(slab(got["dk"]), dk) and torch.equal(slab(got["dv"]), dv) and torch.equal(slab(got["dq"]), dq)


def test_gradients_against_differences(pkg):
    """The gradients are those of the forward's own outputs: a central difference of sum(out * dout) along a direction."""
    lengths, d, scale = [40, 150], 64, 0.125
    q, k, v, dout, offsets = make(lengths, 4, 2, d, seed=8, fused=False)
    got = run(pkg.ops, q, k, v, dout, offsets, scale)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        step = torch.randn(t.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9)).double() / 64
        f = lambda x: attention(*(x if other is t else other for other in (q, k, v)), lengths, scale)[0]["out"]
        want = float(((f(t.double() + step) - f(t.double() - step)) / 2 * dout.double()).sum())
        is_ = float((got[name].double() * step).sum())
        # the difference's third-order term and the gradient's roundings (random signs over thousands of elements)
        size = float((got[name].double() * step).norm())
        assert abs(want - is_) <= 0.02 * abs(want) + 8 * 2.0 ** -7 * size, (name, want, is_)


@pytest.mark.parametrize("d", [64, 128])
def test_written_parts_of_fused_buffers(pkg, d):
    """dq, dk, dv as parts of one buffer, out with padded rows."""
    lengths, H, Hkv = [130, 60], 4, 2
    q, k, v, dout, offsets = make(lengths, H, Hkv, d, seed=10)
    n = sum(lengths)
    wide = torch.full((n, (H + 2 * Hkv) * d + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    dq, dk, dv = (wide[:, a:b].view(n, -1, d) for a, b in ((0, H * d), (H * d, (H + Hkv) * d), ((H + Hkv) * d, (H + 2 * Hkv) * d)))
    out = torch.full((n, H * d + 16), 3.0, dtype=torch.bfloat16, device=DEV)
    got = run(pkg.ops, q, k, v, dout, offsets, 0.125, out=out[:, : H * d].view(n, H, d), dq=dq, dk=dk, dv=dv)
    assert_close(got, *attention(q, k, v, lengths, 0.125, dout), NAMES)
    assert bool((wide[:, -8:] == 3.0).all()) and bool((out[:, H * d :] == 3.0).all())


@pytest.mark.parametrize("d", [64, 128])
def test_captured_replayed_and_on_another_stream(pkg, d):
    """Two graphs of different shapes, replayed at the same time on two streams, with new lengths and values in place."""
    ops, scale = pkg.ops, 0.125
    first = [([100, 60, 30], 4, 2), ([257, 5], 2, 2)]
    graphs = []
    ops.reserve(1, 128, d)
    for i, (lengths, H, Hkv) in enumerate(first):
        q, k, v, dout, offsets = make(lengths, H, Hkv, d, seed=11 + i, fused=False)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            run(ops, q, k, v, dout, offsets, scale)
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                got = run(ops, q, k, v, dout, offsets, scale)
        graphs.append((g, stream, (q, k, v, dout, offsets), got, H, Hkv))
    for lengths in ([100, 60, 30], [1, 188, 1]):
        news = []
        for j, (g, stream, tensors, got, H, Hkv) in enumerate(graphs):
            n = tensors[0].shape[0]
            parts = lengths if j == 0 else [n - 9, 9]
            q, k, v, dout, offsets = make(parts, H, Hkv, d, seed=20 + j + lengths[0], fused=False)
            with torch.no_grad():
                for to, t in zip(tensors, (q, k, v, dout, offsets)):
                    to.copy_(t)
            news.append((parts, q, k, v, dout))
        torch.cuda.synchronize()
        for g, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for (parts, q, k, v, dout), (_, _, _, got, _, _) in zip(news, graphs):
            assert_close(got, *attention(q, k, v, parts, scale, dout), NAMES)
    ops.check_device_fault()


def test_empty(pkg):
    ops = pkg.ops
    q, k, v, dout, offsets = make([], 2, 1, 64)
    got = run(ops, q, k, v, dout, offsets, 0.125)
    assert got["out"].shape == (0, 2, 64) and got["dk"].shape == (0, 1, 64)
    q, k, v, dout, offsets = make([0, 0], 2, 1, 64, behind=5)
    got = run(ops, q, k, v, dout, offsets, 0.125)
    assert all(bool((got[n] == 0).all()) for n in NAMES)


def test_offsets_outside_the_rows_are_clipped(pkg):
    lengths = [100, 56]
    q, k, v, dout, offsets = make(lengths, 2, 1, 64, seed=13)
    want = run(pkg.ops, q, k, v, dout, offsets, 0.125)
    for wild in ([-5, 100, 1 << 30], [0, 100, 2147483647]):
        got = run(pkg.ops, q, k, v, dout, torch.tensor(wild, dtype=torch.int32, device=DEV), 0.125)
        assert all(torch.equal(want[n], got[n]) for n in NAMES)


def test_refusals(pkg):
    ops, Err = pkg.ops, pkg.lib.B200AttnError
    q, k, v, dout, offsets = make([100], 4, 2, 64, fused=False)
    out, lse = ops.attention_forward_bf16_ragged(q, k, v, offsets, 0.125)
    bad = [
        dict(q=q.float()), dict(q=q[:, :3]), dict(k=k[:50]), dict(k=k[:, :, :32]), dict(v=v[:, :1]), dict(offsets=offsets.long()), dict(offsets=offsets.cpu()),
        dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), dict(q=q.cpu()), dict(offsets=offsets[:0]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
        dict(v=torch.empty(100, 4 * 64, dtype=torch.bfloat16, device=DEV)[:, :128].view(100, 2, 64)),
        dict(q=torch.empty(100, 4 * 64 + 4, dtype=torch.bfloat16, device=DEV)[:, :256].view(100, 4, 64)),
        dict(q=torch.empty(100 * 256 + 8, dtype=torch.bfloat16, device=DEV)[4:-4].view(100, 4, 64)), dict(q=q[:1].expand(100, 4, 64)),
    ]
    for change in bad:
        a = dict(q=q, k=k, v=v, offsets=offsets, scale=0.125) | change
        with pytest.raises(Err):
            ops.attention_forward_bf16_ragged(a["q"], a["k"], a["v"], a["offsets"], a["scale"])
        with pytest.raises(Err):
            ops.attention_backward_bf16_ragged(a["q"], a["k"], a["v"], out, dout, lse, a["offsets"], a["scale"])
    with pytest.raises(Err):
        ops.attention_forward_bf16_ragged(q, k, v, offsets, 0.125, out=out[:50])
    with pytest.raises(Err):
        ops.attention_backward_bf16_ragged(q, k, v, out, dout, lse[:, :50].contiguous(), offsets, 0.125)
    small = torch.randn(64, 2, 32, device=DEV).to(torch.bfloat16)
    with pytest.raises(Err) as e:
        ops.attention_forward_bf16_ragged(small, small, small, offsets, 0.1)
    assert e.value.code == pkg.lib.ERR_UNSUPPORTED
