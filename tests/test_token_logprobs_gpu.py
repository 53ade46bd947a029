"""Log-probabilities of given tokens, entropy, top alternatives and their gradient against a 64-bit restatement."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = math.inf


@pytest.fixture(scope="module")
def lo(pkg):
    return importlib.import_module(pkg.__name__ + ".loss_ops")


def make(rows, V, dtype, seed=0, std=3.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(rows, V, generator=gen, device=DEV) * std).to(dtype)
    t = torch.randint(0, V, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    t[::5] = -1
    return x, t, torch.randn(rows, generator=gen, device=DEV), torch.randn(rows, generator=gen, device=DEV) * 0.1


def oracle(x, t, tau, top=0, g=None, ge=None):
    y = x.double() / tau
    empty = (x == -INF).all(-1)
    logp = torch.log_softmax(y, -1)
    logp[empty] = -INF
    p = logp.exp()
    plogp = torch.where(p == 0, 0.0, p * logp)
    r = {"entropy": -plogp.sum(-1), "logp": logp, "p": p}
    given = (t >= 0) & (t < x.shape[-1])
    at = torch.where(given, t, 0).long()
    r["logprobs"] = torch.where(given, logp.gather(-1, at[:, None])[:, 0], 0.0)
    if top:
        order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
        r["top_tokens"], r["top_logprobs"] = order.int(), logp.gather(-1, order)
    if g is not None:
        ge = torch.zeros_like(g) if ge is None else ge
        g1 = torch.where(given, g, 0.0).double()[:, None]
        onehot = torch.zeros_like(p).scatter_(-1, at[:, None], given.double()[:, None])
        inner = torch.where(p == 0, 0.0, p * (logp + r["entropy"][:, None]))
        d = (g1 * (onehot - p) - ge.double()[:, None] * inner) / tau
        dead = empty | ((g1[:, 0] == 0) & (ge == 0))
        d[dead] = 0
        # p is known to some 2e-5 (an argument of up to 60 in FP32, sums of thousands of terms); the type's rounding once; and
        # g / tau, which the target's element is where p is small, is g times a rounded 1 / tau, rounded: two half steps of FP32
        half = torch.finfo(x.dtype).eps / 2
        tol = half * d.abs() * 1.01 + 2 * 2.0 ** -24 * onehot * g1.abs() / tau + 2e-5 * torch.where(p == 0, 0.0, p * (g1.abs() + ge.double().abs()[:, None] * (logp.abs() + r["entropy"][:, None]))) / tau
        r["dlogits"], r["tol"] = d, torch.where(dead[:, None], 0.0, tol) + (1e-30 if x.dtype == torch.float32 else 1e-38)
    return r


def near(got, want, slack=0.0):
    """FP32: a logarithm of a sum (some 3e-5) and a difference of logits."""
    same = (got.double() == want) | (torch.isnan(got) & torch.isnan(want))
    off = (got.double() - want).abs() - 3e-5 - slack - 2.0 ** -21 * want.abs()
    assert bool((same | (off <= 0)).all()), float(off[~same].max())


def check(lo, x, t, tau=1.0, top=0, g=None, ge=None, **kw):
    r = lo.token_logprobs_forward(x, t, temperature=tau, top=top)
    want = oracle(x, t, tau, top, g, ge)
    near(r.logprobs, want["logprobs"])
    near(r.entropy, want["entropy"], 1e-4)  # sum of p ln p: |ln p| of some ten times 1e-5
    if top:
        assert torch.equal(r.top_tokens, want["top_tokens"])
        near(r.top_logprobs, want["top_logprobs"])
    else:
        assert r.top_logprobs is None and r.top_tokens is None
    if g is not None:
        d = lo.token_logprobs_backward(x, t, r, g, ge, **kw)
        assert d.dtype == x.dtype and d.shape == x.shape
        off = (d.double() - want["dlogits"]).abs() - want["tol"]
        assert bool((off <= 0).all()), float(off.max())
    return r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 65, 300, 1000, 1024, 1025, 2049, 5003, 14001, 20011, 50257, 131072])
@pytest.mark.parametrize("rows,tau", [(1, 1.0), (9, 0.7), (300, 1.5)])
def test_forward_and_backward(lo, V, rows, dtype, tau):
    x, t, g, ge = make(rows, V, dtype, seed=V + rows)
    check(lo, x, t, tau, min(20, V), g, ge)
    check(lo, x, t, tau, 0, g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(800, 20011), (3000, 2500), (400, 70001), (6001, 1100), (6001, 4001), (800, 6007)])
def test_many_rows(lo, rows, V, dtype):
    x, t, g, ge = make(rows, V, dtype, seed=V)
    check(lo, x, t, 1.0, 32, g, ge)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [7, 300, 1500, 8000, 40000])
@pytest.mark.parametrize("top", [1, 7, 32])
def test_equal_logits_go_by_the_lower_index(lo, V, top, dtype):
    top = min(top, V)
    x, t, g, ge = make(12, V, dtype, seed=V, std=0.0)             # all equal
    x[1::4] = torch.randint(0, 3, x[1::4].shape, device=DEV).to(dtype)  # three values
    x[2::4, ::2] = -0.0                                              # -0 and +0 are equal
    x[3::4] = (torch.arange(V, device=DEV) % 2048 == 5).to(dtype)       # large ones at one distance: all with one thread
    check(lo, x, t, 1.0, top, g, ge)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [33, 700, 3001, 14001, 50257])
def test_tokens_that_are_not_allowed(lo, V, dtype):
    x, t, g, ge = make(10, V, dtype, seed=V)
    x[0] = -INF                     # none allowed
    x[1] = -INF
    x[1, V // 2] = 3.0              # one allowed
    x[2] = -INF
    x[2, :: V // 5 + 1] = x[5, :: V // 5 + 1]  # a few, fewer than alternatives
    x[3, 1::2] = -INF
    x[4] = torch.finfo(dtype).min   # the type's lowest value everywhere: all equal
    x[6] = torch.finfo(dtype).min
    x[6, 3] = 1.0
    t[:8] = torch.tensor([0, V // 2, 1, 2, 3, -1, 3, 0], device=DEV)
    r = check(lo, x, t, 1.0, 12, g, ge)
    assert r.entropy[0] == 0 and r.entropy[1] == 0 and r.logprobs[0] == -INF and r.logprobs[1] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [33, 3001])
@pytest.mark.parametrize("tau,weight", [(1e-6, 1.0), (1e-3, 1.0), (1.0, 1e12), (1e6, 1.0)])
def test_masked_tokens_at_the_ends_of_the_temperature(lo, V, dtype, tau, weight):
    """A masked logit's gradient is 0 however large the factors beside its probability are."""
    x, t, g, ge = make(10, V, dtype, seed=V, std=3.0 * tau)
    x[1::3, 1::2] = -INF
    x[2::3, ::2] = torch.finfo(dtype).min
    t[1::3], t[2::3] = 2, 1
    check(lo, x, t, tau, 3, g, ge * weight)


@pytest.mark.parametrize("V", [50, 900, 4000, 60000])
@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_spoilt_rows(lo, V, bad):
    x, t, g, ge = make(6, V, torch.float32, seed=2)
    t[:] = 1
    clean = lo.token_logprobs_forward(x, t, top=3)
    x[2, V - 2] = bad
    x[4] = bad
    t[4] = -1
    g[4], ge[4] = 5.0, 0.0
    r = lo.token_logprobs_forward(x, t, top=3)
    d = lo.token_logprobs_backward(x, t, r, g, ge)
    assert bool(r.logprobs[2].isnan()) and bool(r.entropy[2].isnan()) and bool(d[2].isnan().any())
    assert r.logprobs[4] == 0 and bool((d[4] == 0).all())  # padding: no gradient, whatever the row holds
    assert r.top_tokens[2, 0] == V - 2 and r.top_tokens[4].tolist() == [0, 1, 2]
    rest = [0, 1, 3, 5]
    assert torch.equal(r.logprobs[rest], clean.logprobs[rest]) and torch.equal(r.top_tokens[rest], clean.top_tokens[rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,pad,shift", [(1200, 80, 0), (1201, 6, 1), (5003, 0, 3), (100, 28, 1)])
def test_strided_and_unaligned_rows(lo, V, pad, shift, dtype):
    """Rows of a wider buffer that start anywhere; the gradient into such rows, in place and at another alignment."""
    x, t, g, ge = make(21, V, dtype, seed=V)
    buf = torch.full((21 * (V + pad) + 8 + shift,), float("nan"), dtype=dtype, device=DEV)
    view = buf[shift : shift + 21 * (V + pad)].view(21, V + pad)[:, :V]
    view.copy_(x)
    check(lo, view, t, 1.0, 5, g, ge)
    for off in (shift, shift + 1, 0):
        out = torch.full((21 * (V + pad) + 8 + shift,), 9.0, dtype=dtype, device=DEV)
        d = out[off : off + 21 * (V + pad)].view(21, V + pad)[:, :V]
        check(lo, view, t, 1.0, 0, g, ge, dlogits=d)
        d.fill_(9.0)
        assert bool((out == 9.0).all())  # nothing beside the rows was written
    r = lo.token_logprobs_forward(view, t)
    want = lo.token_logprobs_backward(view, t, r, g, ge)
    got = lo.token_logprobs_backward(view, t, r, g, ge, dlogits=view)
    assert got is view and torch.equal(view, want)
    if pad:
        assert bool(buf[shift : shift + 21 * (V + pad)].view(21, V + pad)[:, V:].isnan().all())


def test_leading_dimensions(lo):
    x, t, g, ge = make(24, 300, torch.float32, seed=3)
    flat = lo.token_logprobs_forward(x, t, top=4)
    r = lo.token_logprobs_forward(x.view(2, 3, 4, 300), t.view(2, 3, 4), top=4)
    assert r.logprobs.shape == r.entropy.shape == (2, 3, 4) and r.stats.shape == (2, 3, 4, 2) and r.top_tokens.shape == (2, 3, 4, 4)
    assert torch.equal(r.logprobs.view(-1), flat.logprobs) and torch.equal(r.top_tokens.view(-1, 4), flat.top_tokens)
    d = lo.token_logprobs_backward(x.view(2, 3, 4, 300), t.view(2, 3, 4), r, g.view(2, 3, 4))
    assert d.shape == (2, 3, 4, 300)
    one = lo.token_logprobs_forward(x[0], t[0])
    assert one.logprobs.shape == () and one.logprobs == flat.logprobs[0]
    none = lo.token_logprobs_forward(x[:0], t[:0], top=2)
    assert none.top_tokens.shape == (0, 2) and lo.token_logprobs_backward(x[:0], t[:0], none, g[:0]).shape == (0, 300)


def test_matches_the_cross_entropy(lo):
    """-mean log-probability is the framework's loss, and its gradient the loss's."""
    x, t, *_ = make(64, 5003, torch.float32, seed=4)
    t.abs_()
    dl, loss = lo.cross_entropy_forward_backward(x.view(1, 64, -1), t.view(1, 64))
    r = lo.token_logprobs_forward(x, t)
    assert abs(float(loss) + float(r.logprobs.mean())) < 1e-4
    d = lo.token_logprobs_backward(x, t, r, torch.full((64,), -1 / 64, device=DEV))
    assert float((d - dl[0]).abs().max()) < 1e-6


def test_gradient_against_differences(lo):
    x, t, g, ge = make(6, 1300, torch.float32, seed=5)
    x[1, 7] = x[1].max() + 4
    r = lo.token_logprobs_forward(x, t, temperature=0.8)
    d = lo.token_logprobs_backward(x, t, r, g, ge).double()
    step = torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).double() * 1e-4

    def f(y):
        o = oracle(y, t, 0.8)
        return o["logprobs"] * g + o["entropy"] * ge

    want = (f(x.double() + step) - f(x.double() - step)) / 2
    got = (d * step).sum(-1)
    assert bool(((want - got).abs() <= 1e-3 * step.norm(dim=-1) * d.norm(dim=-1) + 1e-9).all())


@pytest.mark.parametrize("rows,V", [(3, 50257), (200, 3000), (50, 100), (40, 700)])
def test_captured_and_replayed(lo, rows, V):
    x, t, g, ge = make(rows, V, torch.bfloat16, seed=7)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        lo.token_logprobs_forward(x, t, top=5)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r = lo.token_logprobs_forward(x, t, top=5)
            d = lo.token_logprobs_backward(x, t, r, g, ge)
    for seed in (8, 9):
        for to, new in zip((x, t, g, ge), make(rows, V, torch.bfloat16, seed=seed)):
            to.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = oracle(x, t, 1.0, 5, g, ge)
        near(r.logprobs, want["logprobs"])
        assert torch.equal(r.top_tokens, want["top_tokens"])
        assert bool(((d.double() - want["dlogits"]).abs() <= want["tol"]).all())


def test_refusals(lo):
    x, t, g, ge = make(8, 50, torch.float32)
    r = lo.token_logprobs_forward(x, t)
    for a in [(x.half(), t), (x.cpu(), t), (x, t.long()), (x, t[:3]), (x, t.cpu()), (x.t(), t), (x[:, ::2], t), (x[:, :0], t), (x[:1].expand(8, 50), t)]:
        with pytest.raises(ValueError):
            lo.token_logprobs_forward(*a)
    for top in (-1, 33, 51):
        with pytest.raises(ValueError):
            lo.token_logprobs_forward(x, t, top=top)
    for tau in (0.0, -1.0, float("nan"), INF, 1e-7, 1e7):
        with pytest.raises(lo.B200LossError):
            lo.token_logprobs_forward(x, t, temperature=tau)
    for kw in [dict(grad_logprobs=g[:3]), dict(grad_logprobs=g.double()), dict(grad_entropy=ge[:3]), dict(dlogits=x.bfloat16()), dict(dlogits=torch.empty_like(x)[:, :40]),
               dict(dlogits=x.t()), dict(dlogits=torch.empty(1, 50, device=DEV).expand(8, 50))]:
        with pytest.raises(ValueError):
            lo.token_logprobs_backward(x, t, r, **({"grad_logprobs": g, "grad_entropy": ge} | kw))
