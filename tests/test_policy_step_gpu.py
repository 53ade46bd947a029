"""The operators as they are used together: sampling over a cache, scoring the samples, and a training step on them packed."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


class Model:
    """One attention layer between an embedding and a head, grouped heads, BF16 weights."""

    def __init__(self, V=500, C=128, H=4, Hkv=2, d=64, seed=0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rnd = lambda *s, std: (torch.randn(*s, generator=gen, device=DEV) * std).to(BF)
        self.H, self.Hkv, self.d, self.scale = H, Hkv, d, 1 / math.sqrt(d)
        self.emb, self.wqkv = rnd(V, C, std=1.0), rnd(C, (H + 2 * Hkv) * d, std=C ** -0.5)
        self.wo, self.head = rnd(H * d, C, std=(H * d) ** -0.5), rnd(C, V, std=2 * C ** -0.5)

    def qkv(self, x):
        n = x.shape[0]
        parts = (x @ self.wqkv).split([self.H * self.d, self.Hkv * self.d, self.Hkv * self.d], 1)
        return [t.view(n, -1, self.d) for t in parts]


def sample(pkg, lo, m, prompts, steps, gen):
    """Tokens of every sequence (prompt and samples), and the log-probabilities the sampler gave the sampled ones."""
    B, longest = len(prompts), max(map(len, prompts)) + steps
    k = torch.zeros(B, longest, m.Hkv, m.d, dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    texts, chosen = [list(p) for p in prompts], [[] for _ in prompts]
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for i in range(max(map(len, prompts)) - 1 + steps):
        fed = [b for b in range(B) if i < len(texts[b]) and len(texts[b]) < len(prompts[b]) + steps]
        if not fed:
            break
        tokens = torch.tensor([texts[b][i] if i < len(texts[b]) else 0 for b in range(B)], device=DEV)
        x = m.emb[tokens]
        q, kn, vn = m.qkv(x)
        for b in fed:
            k[b, i], v[b, i] = kn[b], vn[b]
            lengths[b] = i + 1
        out, _ = pkg.ops.attention_decode_bf16(q, k, v, lengths, m.scale)
        logits = (x + out.view(B, -1) @ m.wo) @ m.head
        picks = torch.multinomial(torch.softmax(logits.float(), -1), 1, generator=gen)[:, 0].int()
        lp = lo.token_logprobs_forward(logits, picks).logprobs
        for b in fed:
            if i == len(texts[b]) - 1:
                texts[b].append(int(picks[b]))
                chosen[b].append(float(lp[b]))
    return texts, chosen


def packed_step(pkg, lo, m, texts, weights, beta, rows=None):
    """Logits of the packed texts, the loss's parts, and the gradients of all weights: loss = -sum w logp(next token) - beta sum H."""
    tokens = torch.tensor(sum(texts, []), device=DEV)
    ends = [0]
    for t in texts:
        ends.append(ends[-1] + len(t))
    offsets = torch.tensor(ends, dtype=torch.int32, device=DEV)
    targets = torch.tensor(sum((t[1:] + [-1] for t in texts), []), dtype=torch.int32, device=DEV)
    x = m.emb[tokens]
    q, k, v = m.qkv(x)
    out, lse = pkg.ops.attention_forward_bf16_ragged(q, k, v, offsets, m.scale)
    y = x + out.view(len(tokens), -1) @ m.wo
    logits = y @ m.head
    r = lo.token_logprobs_forward(logits, targets, top=3)
    seen = (targets >= 0).float()
    dl = lo.token_logprobs_backward(logits, targets, r, -weights * seen, -beta * seen)
    dy = dl @ m.head.T
    dout = (dy @ m.wo.T).view_as(out)
    dqkv = torch.empty(len(tokens), (m.H + 2 * m.Hkv) * m.d, dtype=BF, device=DEV)
    dq, dk, dv = (t.view(len(tokens), -1, m.d) for t in dqkv.split([m.H * m.d, m.Hkv * m.d, m.Hkv * m.d], 1))
    pkg.ops.attention_backward_bf16_ragged(q, k, v, out, dout, lse, offsets, m.scale, dq=dq, dk=dk, dv=dv)
    dx = (dy + dqkv @ m.wqkv.T).float()
    grads = {"head": y.T @ dl, "wo": out.view(len(tokens), -1).T @ dy, "wqkv": x.T @ dqkv, "emb": torch.zeros_like(m.emb, dtype=torch.float32).index_add_(0, tokens, dx)}
    return logits, r, grads, seen


def reference_grads(m, texts, weights, beta):
    """The same loss in 64 bits, by autograd, one text after the other."""
    W = {n: getattr(m, n).double().requires_grad_() for n in ("emb", "wqkv", "wo", "head")}
    loss, at = 0.0, 0
    for t in texts:
        n = len(t)
        x = W["emb"][torch.tensor(t, device=DEV)]
        q, k, v = (p.view(n, -1, m.d).transpose(0, 1) for p in (x @ W["wqkv"]).split([m.H * m.d, m.Hkv * m.d, m.Hkv * m.d], 1))
        k, v = (p.repeat_interleave(m.H // m.Hkv, 0) for p in (k, v))
        s = (q @ k.transpose(1, 2) * m.scale).masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), -math.inf)
        o = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, -1)
        logp = torch.log_softmax((x + o @ W["wo"]) @ W["head"], -1)[:-1]
        w = weights[at : at + n - 1].double()
        loss = loss - (w * logp.gather(1, torch.tensor(t[1:], device=DEV)[:, None])[:, 0]).sum() + beta * (logp.exp() * logp).sum()
        at += n
    loss.backward()
    return {n: p.grad for n, p in W.items()}


def test_sample_score_and_train(pkg):
    lo = importlib.import_module(pkg.__name__ + ".loss_ops")
    m, gen = Model(), torch.Generator(device=DEV).manual_seed(1)
    prompts = [[5, 9, 2], list(range(40)), [7], list(range(100, 240))]
    texts, chosen = sample(pkg, lo, m, prompts, 20, gen)
    assert [len(t) for t in texts] == [len(p) + 20 for p in prompts]
    n = sum(map(len, texts))
    weights = torch.randn(n, generator=gen, device=DEV)
    logits, r, grads, seen = packed_step(pkg, lo, m, texts, weights, 0.01)
    pkg.ops.check_device_fault()
    # the packed pass gives the sampled tokens the log-probabilities that the sampler saw: the same products in BF16, of which
    # only the attention output is rounded after another order of sums (half a step of 2^-8 of values around 1, twice, then a
    # product with a head of norm 2 over 128 channels, and logits of some units rounded to 2^-8 on both sides)
    at = 0
    for t, p, c in zip(texts, prompts, chosen):
        got = r.logprobs[at + len(p) - 1 : at + len(t) - 1]
        assert float((got - torch.tensor(c, device=DEV)).abs().max()) < 0.15
        at += len(t)
    assert bool((r.logprobs[seen == 0] == 0).all())
    # the best alternative is the arg max, and no given token is above it
    assert torch.equal(r.top_tokens[:, 0].long(), logits.float().argmax(-1))
    assert bool((r.logprobs <= r.top_logprobs[:, 0] + 1e-6)[seen == 1].all())
    want = reference_grads(m, texts, weights, 0.01)
    for name, g in want.items():
        # every product of the chain rounds its operands and its result to BF16 (2^-8 each, five products deep, at random signs)
        off = float((grads[name].double() - g).norm() / g.norm())
        assert off < 0.03, (name, off)


def test_two_steps_on_two_streams(pkg):
    """Steps that run at the same time (their workspaces are their own) give what they give alone."""
    lo = importlib.import_module(pkg.__name__ + ".loss_ops")
    work = []
    for seed in (0, 1):
        m, gen = Model(seed=seed), torch.Generator(device=DEV).manual_seed(seed)
        texts = [[int(x) for x in torch.randint(0, 500, (n,), generator=gen, device=DEV)] for n in (300, 20, 129)]
        weights = torch.randn(449, generator=gen, device=DEV)
        work.append((m, texts, weights, packed_step(pkg, lo, m, texts, weights, 0.0)))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in work], [None, None]
    for _ in range(3):
        for i, (m, texts, weights, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                results[i] = packed_step(pkg, lo, m, texts, weights, 0.0)
        torch.cuda.synchronize()
        for (_, _, _, alone), again in zip(work, results):
            assert torch.equal(alone[0], again[0]) and torch.equal(alone[1].logprobs, again[1].logprobs)
            for name in ("head", "wo"):
                assert torch.equal(alone[2][name], again[2][name])
            for name in ("wqkv", "emb"):  # dQ is summed in no fixed order, in FP32, then rounded to BF16
                assert float((alone[2][name].float() - again[2][name].float()).norm()) <= 2 ** -8 * float(alone[2][name].float().norm())
