"""The operators for sequences of different lengths, as cases that can be timed and compared: causal attention with
grouped heads over packed sequences (a prompt pass, and a training pass with its gradients), its form for one new token
of every sequence over a cache of keys and values, and the log-probabilities of given tokens with entropy, top
alternatives and gradient.

`run` computes them in their plain form, elementary torch operations in 32 bits rounded once at the end, or, where `own` is
true, through the calls a user makes of the framework. `exact` computes them in 64 bits, written apart from the plain form."""
import importlib
import math
import random

import torch

own = False

LOW = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # three short dialogue turns in one small batch: launches and latencies are all there is
        {"name": "train_tiny", "kind": "train", "seqs": 3, "shortest": 17, "longest": 101, "mix": 1, "heads": 4, "kv_heads": 2, "dim": 64},
        # documents of 64 to 1024 tokens packed into one batch, the head layout of GPT-2 small
        {"name": "train_documents_d64", "kind": "train", "seqs": 32, "shortest": 64, "longest": 1024, "mix": 2, "heads": 12, "kv_heads": 12, "dim": 64},
        # fine-tuning on long texts, four query heads to a key head
        {"name": "train_grouped_d128", "kind": "train", "seqs": 9, "shortest": 333, "longest": 4095, "mix": 3, "heads": 32, "kv_heads": 8, "dim": 128},
        # two long prompts and some short ones before sampling: forward only
        {"name": "prompt_long_d128", "kind": "prompt", "seqs": 5, "shortest": 1500, "longest": 16384, "mix": 4, "heads": 16, "kv_heads": 4, "dim": 128},
        # sampling from a small model: few sequences, short caches
        {"name": "token_small_d64", "kind": "token", "batch": 4, "shortest": 100, "capacity": 1024, "mix": 5, "heads": 12, "kv_heads": 12, "dim": 64},
        # sampling for a large batch, caches filled to different lengths
        {"name": "token_batch_d128", "kind": "token", "batch": 64, "shortest": 300, "capacity": 4096, "mix": 6, "heads": 32, "kv_heads": 8, "dim": 128},
        # one very long context: the keys have to be split to fill the card
        {"name": "token_long_d128", "kind": "token", "batch": 1, "shortest": 100001, "capacity": 131072, "mix": 7, "heads": 32, "kv_heads": 8, "dim": 128},
        # scoring the last tokens of a few sequences, GPT-2's vocabulary, with alternatives
        {"name": "score_few", "kind": "score", "rows": 7, "vocab": 50257, "dtype": "bf16", "top": 8, "temperature": 1.0},
        # scoring whole sequences of a large vocabulary
        {"name": "score_rows_bf16", "kind": "score", "rows": 4096, "vocab": 131072, "dtype": "bf16", "top": 20, "temperature": 0.7},
        # training on log-probabilities and entropy, FP32 logits of GPT-2's vocabulary
        {"name": "policy_rows_fp32", "kind": "policy", "rows": 8192, "vocab": 50257, "dtype": "fp32", "temperature": 1.0},
        # the same on BF16 logits and a padded vocabulary
        {"name": "policy_rows_bf16", "kind": "policy", "rows": 6001, "vocab": 50304, "dtype": "bf16", "temperature": 1.3},
        # a model over characters: short rows, many of them
        {"name": "policy_characters", "kind": "policy", "rows": 16384, "vocab": 65, "dtype": "fp32", "temperature": 1.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["train", "train", "prompt", "token", "token", "score", "policy"])
    if kind in ("train", "prompt"):
        kv = rng.choice([1, 2, 4, 8, 12])
        group = rng.choice([1, 2, 3, 4, 8])
        while kv * group > 32:
            group = 1 if group == 2 else max(1, group // 2)
        longest = _spread(rng, 40, 4000 if kind == "train" else 9000)
        return {"kind": kind, "seqs": max(1, min(_spread(rng, 1, 64), 24000 // longest)), "shortest": max(1, longest // rng.randint(2, 40)), "longest": longest,
                "mix": rng.randrange(1 << 20), "heads": kv * group, "kv_heads": kv, "dim": rng.choice([64, 128])}
    if kind == "token":
        kv = rng.choice([1, 2, 4, 8])
        capacity = _spread(rng, 200, 60000)
        return {"kind": kind, "batch": max(1, min(_spread(rng, 1, 128), 500000 // (capacity * kv))), "shortest": max(1, capacity // rng.randint(1, 50)), "capacity": capacity,
                "mix": rng.randrange(1 << 20), "heads": kv * rng.choice([1, 2, 4, 5, 8]), "kv_heads": kv, "dim": rng.choice([64, 128])}
    vocab = _spread(rng, 50, 131072)
    case = {"kind": kind, "rows": max(1, min(_spread(rng, 1, 16384), 300000000 // vocab)), "vocab": vocab, "dtype": rng.choice(["bf16", "fp32"])}
    if kind == "score":
        case["top"] = rng.randint(1, 20)
    case["temperature"] = rng.choice([1.0, 0.6, 1.4])
    return case


def _lengths(case):
    """The sequences' lengths: spread evenly over the logarithm between the shortest and the longest, the longest among them."""
    rng = random.Random(case["mix"])
    if case["kind"] == "token":
        return [_spread(rng, case["shortest"], case["capacity"]) for _ in range(case["batch"])]
    lengths = [_spread(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    lengths[rng.randrange(len(lengths))] = case["longest"]
    return lengths


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * std).to(dtype)

    state = {"case": dict(case)}
    if case["kind"] in ("train", "prompt"):
        lengths = _lengths(case)
        total, H, K, d = sum(lengths), case["heads"], case["kv_heads"], case["dim"]
        # one fused projection output (queries, keys, values of all heads) that the three tensors are views of
        qkv = normal(total, (H + 2 * K) * d)
        state["q"] = qkv[:, : H * d].view(total, H, d)
        state["k"] = qkv[:, H * d : (H + K) * d].view(total, K, d)
        state["v"] = qkv[:, (H + K) * d :].view(total, K, d)
        ends = [0]
        for n in lengths:
            ends.append(ends[-1] + n)
        state["ends"] = ends
        state["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
        state["out"] = torch.empty(total, H, d, dtype=torch.bfloat16, device=dev)
        state["lse"] = torch.empty(H, total, dtype=torch.float32, device=dev)
        if case["kind"] == "train":
            state["dout"] = normal(total, H, d)
            state["grads"] = [torch.empty(total, h, d, dtype=torch.bfloat16, device=dev) for h in (H, K, K)]
    elif case["kind"] == "token":
        B, T, H, K, d = case["batch"], case["capacity"], case["heads"], case["kv_heads"], case["dim"]
        state["q"] = normal(B, H, d)
        state["k"], state["v"] = normal(B, T, K, d), normal(B, T, K, d)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    else:
        R, V = case["rows"], case["vocab"]
        # logits of a model that has learnt something: the given token stands out in most rows; a few rows are padding
        logits = torch.randn(R, V, generator=gen, device=dev, dtype=torch.float32).mul_(2.5)
        targets = torch.randint(0, V, (R,), generator=gen, device=dev, dtype=torch.int32)
        logits.scatter_add_(1, targets.long()[:, None], torch.rand(R, 1, generator=gen, device=dev) * 14.0)
        padding = torch.rand(R, generator=gen, device=dev) < 0.05
        state["logits"] = logits.to(LOW[case["dtype"]])
        state["targets"] = torch.where(padding, torch.full_like(targets, -1), targets)
        if case["kind"] == "policy":
            state["grad_logprobs"] = torch.where(padding, 0.0, torch.randn(R, generator=gen, device=dev))
            state["grad_entropy"] = torch.full((R,), 0.01, device=dev)
    return state


def run(state):
    case = state["case"]
    if own:
        return _own_run(state)
    if case["kind"] in ("train", "prompt"):
        return _plain_packed(state)
    if case["kind"] == "token":
        return _plain_token(state)
    return _plain_logprobs(state)


# ---------------------------------------------------------------- the framework's calls
def _package():
    return importlib.import_module("__graft_entry__").load_package()


def _own_run(s):
    case = s["case"]
    pkg = _package()
    if case["kind"] in ("train", "prompt"):
        scale = 1.0 / math.sqrt(case["dim"])
        out, lse = pkg.ops.attention_forward_bf16_ragged(s["q"], s["k"], s["v"], s["offsets"], scale, out=s["out"], lse=s["lse"])
        if case["kind"] == "prompt":
            return {"out": out, "lse": lse}
        dq, dk, dv = pkg.ops.attention_backward_bf16_ragged(s["q"], s["k"], s["v"], out, s["dout"], lse, s["offsets"], scale,
                                                            dq=s["grads"][0], dk=s["grads"][1], dv=s["grads"][2])
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if case["kind"] == "token":
        out, lse = pkg.ops.attention_decode_bf16(s["q"], s["k"], s["v"], s["lengths"], 1.0 / math.sqrt(case["dim"]))
        return {"out": out, "lse": lse}
    loss_ops = importlib.import_module(pkg.__name__ + ".loss_ops")
    r = loss_ops.token_logprobs_forward(s["logits"], s["targets"], temperature=case["temperature"], top=case.get("top", 0))
    if case["kind"] == "score":
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_tokens": r.top_tokens}
    dlogits = loss_ops.token_logprobs_backward(s["logits"], s["targets"], r, s["grad_logprobs"], s["grad_entropy"])
    return {"logprobs": r.logprobs, "entropy": r.entropy, "dlogits": dlogits}


# ---------------------------------------------------------------- the plain forms, 32 bits
def _plain_packed(s):
    case, low = s["case"], torch.bfloat16
    H, K, d = case["heads"], case["kv_heads"], case["dim"]
    G, scale = H // K, 1.0 / math.sqrt(d)
    train = case["kind"] == "train"
    parts = []
    for a, b in zip(s["ends"], s["ends"][1:]):  # sequences differ in length: one after the other, all their heads at once
        n = b - a
        q = s["q"][a:b].float().view(n, K, G, d).permute(1, 2, 0, 3)  # (K, G, n, d)
        k = s["k"][a:b].float().permute(1, 0, 2)[:, None]             # (K, 1, n, d)
        v = s["v"][a:b].float().permute(1, 0, 2)[:, None]
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
        p = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(hidden, float("-inf"))
        m = p.amax(-1, keepdim=True)
        p = p.sub_(m).exp_()
        l = p.sum(-1, keepdim=True)
        p = p.div_(l)
        o = p @ v
        part = [o.permute(2, 0, 1, 3).reshape(n, H, d).to(low), (m + l.log()).view(H, n)]
        if train:
            do = s["dout"][a:b].float().view(n, K, G, d).permute(1, 2, 0, 3)
            dv = (p.transpose(-1, -2) @ do).sum(1)
            ds = (do @ v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            dq = ds @ k
            dk = (ds.transpose(-1, -2) @ q).sum(1)
            part += [dq.permute(2, 0, 1, 3).reshape(n, H, d).to(low), dk.permute(1, 0, 2).to(low), dv.permute(1, 0, 2).to(low)]
        parts.append(part)
    cols = list(zip(*parts))
    r = {"out": torch.cat(cols[0]), "lse": torch.cat(cols[1], 1)}
    if train:
        r.update(dq=torch.cat(cols[2]), dk=torch.cat(cols[3]), dv=torch.cat(cols[4]))
    return r


def _plain_token(s):
    case = s["case"]
    B, T, H, K, d = case["batch"], case["capacity"], case["heads"], case["kv_heads"], case["dim"]
    q = s["q"].float().view(B, K, H // K, d)
    k, v = s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)  # (B, K, T, d)
    behind = torch.arange(T, device=q.device)[None] >= s["lengths"][:, None]
    x = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).masked_fill_(behind[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    p = (x - m).exp_()
    l = p.sum(-1, keepdim=True)
    return {"out": ((p @ v) / l).view(B, H, d).to(torch.bfloat16), "lse": (m + l.log()).view(B, H)}


def _plain_logprobs(s):
    case = s["case"]
    raw = s["logits"].float()
    x = raw / case["temperature"]
    x = x - x.amax(-1, keepdim=True)
    logp = x - x.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    entropy = -(p * logp).sum(-1)
    t = s["targets"].long()
    given = t >= 0
    logprobs = torch.where(given, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    if case["kind"] == "score":
        # the largest logits, equal ones by the lowest index: one ordered whole number for each (value, index)
        bits = (raw + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 20) + torch.arange(case["vocab"] - 1, -1, -1, device=raw.device)
        top = case["vocab"] - 1 - (order.topk(case["top"], -1).values & ((1 << 20) - 1))
        return {"logprobs": logprobs, "entropy": entropy, "top_logprobs": logp.gather(1, top), "top_tokens": top.int()}
    glp = torch.where(given, s["grad_logprobs"], 0.0)[:, None]
    d = p * (-glp - s["grad_entropy"][:, None] * (logp + entropy[:, None]))
    d.scatter_add_(1, t.clamp(min=0)[:, None], glp)
    return {"logprobs": logprobs, "entropy": entropy, "dlogits": (d / case["temperature"]).to(s["logits"].dtype)}


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] in ("train", "prompt"):
        H, K, d = case["heads"], case["kv_heads"], case["dim"]
        total = s["ends"][-1]
        dev = s["q"].device
        r = {"out": torch.empty(total, H, d, dtype=f64, device=dev), "lse": torch.empty(H, total, dtype=f64, device=dev)}
        if case["kind"] == "train":
            r.update({"dq": torch.empty(total, H, d, dtype=f64, device=dev), "dk": torch.zeros(total, K, d, dtype=f64, device=dev),
                      "dv": torch.zeros(total, K, d, dtype=f64, device=dev)})
        for a, b in zip(s["ends"], s["ends"][1:]):
            i = torch.arange(b - a, device=dev)
            visible = i[None, :] <= i[:, None]
            for h in range(H):
                g = h // (H // K)
                q, k, v = s["q"][a:b, h].to(f64), s["k"][a:b, g].to(f64), s["v"][a:b, g].to(f64)
                scores = torch.where(visible, q @ k.T / math.sqrt(d), -math.inf)
                lse = torch.logsumexp(scores, 1)
                p = torch.exp(scores - lse[:, None])
                del scores
                r["lse"][h, a:b] = lse
                r["out"][a:b, h] = p @ v
                if case["kind"] == "train":
                    do = s["dout"][a:b, h].to(f64)
                    dp = do @ v.T
                    r["dv"][a:b, g] += p.T @ do
                    ds = p * (dp - torch.sum(p * dp, 1, keepdim=True)) / math.sqrt(d)
                    r["dq"][a:b, h] = ds @ k
                    r["dk"][a:b, g] += ds.T @ q
        return r
    if case["kind"] == "token":
        H, K = case["heads"], case["kv_heads"]
        outs, lses = [], []
        for b, n in enumerate(_lengths(case)):
            k = s["k"][b, :n].to(f64).repeat_interleave(H // K, 1)
            v = s["v"][b, :n].to(f64).repeat_interleave(H // K, 1)
            scores = torch.einsum("hd,nhd->hn", s["q"][b].to(f64), k) / math.sqrt(case["dim"])
            outs.append(torch.einsum("hn,nhd->hd", torch.softmax(scores, 1), v))
            lses.append(torch.logsumexp(scores, 1))
        return {"out": torch.stack(outs), "lse": torch.stack(lses)}
    R, V, tau = case["rows"], case["vocab"], case["temperature"]
    parts = []
    step = max(1, (1 << 28) // V)
    for a in range(0, R, step):
        y = s["logits"][a : a + step].to(f64) / tau
        logp = torch.log_softmax(y, 1)
        p = torch.exp(logp)
        entropy = -(p * logp).sum(1)
        t = s["targets"][a : a + step].long()
        row = torch.arange(len(t), device=t.device)
        logprobs = torch.where(t >= 0, logp[row, t.clamp(min=0)], 0.0)
        if case["kind"] == "score":
            order = torch.sort(y, dim=1, descending=True, stable=True).indices[:, : case["top"]]
            parts.append((logprobs, entropy, torch.gather(logp, 1, order), order.int()))
        else:
            onehot = torch.zeros_like(p)
            onehot[row, t.clamp(min=0)] = (t >= 0).to(f64)
            g1, g2 = s["grad_logprobs"][a : a + step].to(f64)[:, None], s["grad_entropy"][a : a + step].to(f64)[:, None]
            g1 = torch.where(t[:, None] >= 0, g1, 0.0)
            parts.append((logprobs, entropy, ((onehot - p) * g1 - p * (logp + entropy[:, None]) * g2) / tau))
        del y, logp, p
    cols = [torch.cat(c) for c in zip(*parts)]
    return dict(zip(("logprobs", "entropy", "top_logprobs", "top_tokens") if case["kind"] == "score" else ("logprobs", "entropy", "dlogits"), cols))


def work(case):
    if case["kind"] in ("train", "prompt"):
        lengths, H, K, d = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
        total, pairs = sum(lengths), sum(n * (n + 1) // 2 for n in lengths)
        moved = total * d * 2 * (H + 2 * K) + total * d * 2 * H + total * H * 4  # q, k, v in; out, lse
        if case["kind"] == "train":
            moved += total * d * 2 * H + total * d * 2 * (H + 2 * K)             # dout in; dq, dk, dv
        return {"bytes": moved, "flops": (14 if case["kind"] == "train" else 4) * pairs * H * d}
    if case["kind"] == "token":
        keys, B, H, K, d = sum(_lengths(case)), case["batch"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": keys * K * d * 2 * 2 + B * H * d * 4 + B * H * 4, "flops": 4 * keys * H * d}
    n = case["rows"] * case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "score":
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    return {"bytes": 2 * n * size + case["rows"] * 20, "flops": 14 * n}
