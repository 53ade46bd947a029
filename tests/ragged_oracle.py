"""64-bit restatement of attention over packed sequences with grouped heads, forward and backward, together with elementwise
bounds on what BF16 operands may differ by: u = 2^-8 is half a step of BF16 relative to the value, and every rounding the
kernels make (P before P V and P^T dO, dS before dS K and dS^T Q, every BF16 output) counts once."""
import math

import torch

U = torch.finfo(torch.bfloat16).eps / 2
LSE_TOL = 2e-5   # FP32 accumulation of up to 128 products of BF16 values (|sum| of some ten) and one logarithm
SECOND = 1.02    # products of two roundings and the FP32 arithmetic between them


def attention(q, k, v, lengths, scale, dout=None):
    """q (n, H, d), k / v (n, Hkv, d), dout (n, H, d) of any float type, n >= sum(lengths). Returns (values, bounds), dicts of
    float64 tensors (out, lse and, with dout, dq, dk, dv) over the first sum(lengths) rows."""
    f = torch.float64
    H, Hkv = q.shape[1], k.shape[1]
    n, d, dev = sum(lengths), q.shape[2], q.device
    val = {"out": torch.zeros(n, H, d, dtype=f, device=dev), "lse": torch.zeros(H, n, dtype=f, device=dev)}
    tol = {"out": torch.zeros_like(val["out"]), "lse": torch.full_like(val["lse"], LSE_TOL)}
    if dout is not None:
        for name, heads in (("dq", H), ("dk", Hkv), ("dv", Hkv)):
            val[name] = torch.zeros(n, heads, d, dtype=f, device=dev)
            tol[name] = torch.zeros(n, heads, d, dtype=f, device=dev)
    a = 0
    for length in lengths:
        b = a + length
        seen = torch.ones(length, length, dtype=torch.bool, device=dev).tril()
        for h in range(H if length else 0):
            g = h // (H // Hkv)
            Q, K, V = q[a:b, h].to(f), k[a:b, g].to(f), v[a:b, g].to(f)
            s = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            o = p @ V
            o_err = U * (p @ V.abs() + o.abs())
            val["out"][a:b, h], val["lse"][h, a:b], tol["out"][a:b, h] = o, lse, o_err
            if dout is None:
                continue
            dO = dout[a:b, h].to(f)
            D = (dO * o).sum(1, keepdim=True)
            dp = dO @ V.T
            ds = p * (dp - D) * scale
            # P rounded, their product rounded, and D from the rounded output
            ds_err = 2 * U * ds.abs() + p * scale * (dO.abs() * o_err).sum(1, keepdim=True)
            val["dv"][a:b, g] += p.T @ dO
            tol["dv"][a:b, g] += U * (p.T @ dO.abs())
            val["dq"][a:b, h] = ds @ K
            tol["dq"][a:b, h] = ds_err @ K.abs()
            val["dk"][a:b, g] += ds.T @ Q
            tol["dk"][a:b, g] += ds_err.T @ Q.abs()
        a = b
    for name in ("dq", "dk", "dv"):
        if dout is not None:
            tol[name] += U * val[name].abs()
    # FP32 arithmetic (sums of up to some thousand terms, exponentials good to some 2^-21), relative to the same sums
    return val, {name: t if name == "lse" else t * SECOND + 1e-5 for name, t in tol.items()}


def assert_close(got, val, tol, names):
    for name in names:
        g = got[name].to(torch.float64)
        off = (g - val[name]).abs() - tol[name]
        assert bool((off <= 0).all()), f"{name}: {int((~(off <= 0)).sum())} of {off.numel()} outside, worst by {float(off.max()):.3g}"
