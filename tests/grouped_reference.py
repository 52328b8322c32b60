"""Attention with grouped heads in 64 bits, with bounds of what rounding may do to it.

The bounds follow the arithmetic that the kernels document. With u half a step of
the inputs' type (0 for float32 operands, which are not rounded) and w = 2^-24:

* a score is a float32 sum of D products, then one scaling and one subtraction: off
  by at most ``(D + 8) w`` times the sum of the products' magnitudes, and its
  exponential relatively by as much, with the sum it is divided by twice that: ``es``;
* the probabilities are rounded to the inputs' type for the product with V, and divided
  by the sum of the rounded ones: ``|do| <= u sum p |v| + u |o|`` from both, plus the
  result's own rounding ``u |o|`` and the float32 sum's ``K w sum p |v|``;
* a result of float16 is a multiple of 2^-24 where it is small: off by half of that;
* exponentials below float32's smallest normal, 2^-126, come out as zero: with what the tests here multiply
  them by, sums below 2^26, that is 2^-100 at the most;
* dS = P (dP - delta): dP is a float32 sum of Dv products, delta one with the output as
  it was returned; dS is rounded for its product, the product's sum once more.
"""

from __future__ import annotations

import math

import torch

W = 2.0 ** -24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def operand_step(dtype) -> float:
    """What rounding an operand costs: float32 ones are not rounded."""
    return 0.0 if dtype == torch.float32 else half_step(dtype)


class Head:
    """One query head of one sequence: rows q [M, D] against k [N, D], v [N, Dv] and the
    keys each row sees [M, N]; ``dout`` [M, Dv] for the gradients."""

    def __init__(self, q, k, v, seen, scale, dtype, dout=None):
        q, k, v = q.double(), k.double(), v.double()
        u, uo, n = operand_step(dtype), half_step(dtype), k.shape[0]
        d, dv = q.shape[1], v.shape[1]
        scores = torch.where(seen, scale * (q @ k.mT), -math.inf)
        size = torch.where(seen, abs(scale) * (q.abs() @ k.abs().mT), 0.0)
        es = 2 * (d + 8) * W * size.amax(-1, keepdim=True) + 8 * W
        p = torch.nan_to_num(torch.softmax(scores, -1))  # rows that see nothing: zeros
        self.out = p @ v
        weight = p @ v.abs()
        self.out_tol = u * weight + (u + uo) * self.out.abs() + (2 * es + (n + 16) * W) * weight
        if dout is None:
            return
        dout = dout.double()
        dp = dout @ v.mT
        delta = (dout * self.out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        ddelta = (dout.abs() * self.out_tol).sum(-1, keepdim=True) + (dv + 8) * W * (dout * self.out).abs().sum(-1, keepdim=True)
        ds_tol = p * (ddelta + (dv + 8) * W * (dout.abs() @ v.abs().mT)) + ds.abs() * (u + 2 * es + 8 * W)
        if dtype == torch.float16:  # bits below those of the sequence's largest dS
            top = 2 * dout.norm(dim=-1).amax() * v.norm(dim=-1).amax()
            ds_tol = ds_tol + seen * 2.0 ** -37 * top
        s, m = abs(scale), q.shape[0]
        self.dq, self.dk, self.dv = scale * ds @ k, scale * ds.mT @ q, p.mT @ dout
        self.dq_tol = s * (ds_tol + (n + 8) * W * ds.abs()) @ k.abs() + uo * self.dq.abs()
        self.dk_tol = s * (ds_tol + (m + 64) * W * ds.abs()).mT @ q.abs()
        lost = 2.0 ** -38 if dtype == torch.float16 else 0.0
        self.dv_tol = (p * (u + 2 * es + (m + 64) * W) + seen * lost).mT @ dout.abs()


def packed(q, k, v, offsets, causal, scale=None, valid_len=None, dout=None):
    """``{name: (value, bound)}`` in 64 bits: out, and with ``dout`` dq, dk, dv."""
    t, h, d = q.shape
    hk, dv = k.shape[1], v.shape[2]
    g, scale = h // hk, d ** -0.5 if scale is None else scale
    f64 = dict(dtype=torch.float64, device=q.device)
    names = ("out",) if dout is None else ("out", "dq", "dk", "dv")
    shapes = {"out": (t, h, dv), "dq": (t, h, d), "dk": (t, hk, d), "dv": (t, hk, dv)}
    res = {n: (torch.zeros(shapes[n], **f64), torch.zeros(shapes[n], **f64)) for n in names}
    for n, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        if valid_len is not None:
            b = a + min(b - a, max(0, valid_len[n]))
        if b <= a:
            continue
        i = torch.arange(b - a, device=q.device)
        seen = i[None, :] <= i[:, None] if causal else torch.ones(b - a, b - a, dtype=torch.bool, device=q.device)
        for head in range(h):
            kv = head // g
            one = Head(q[a:b, head], k[a:b, kv], v[a:b, kv], seen, scale, q.dtype, None if dout is None else dout[a:b, head])
            for name in names:
                at = head if name in ("out", "dq") else kv
                res[name][0][a:b, at] += getattr(one, name)
                res[name][1][a:b, at] += getattr(one, name + "_tol")
    for name in names:
        if name in ("dk", "dv"):
            res[name][1].add_(half_step(q.dtype) * res[name][0].abs())
    return res


def lineage(parents, context):
    """Which drafts each one sees, a list of them or None for one that is not there."""
    lines = []
    for i, p in enumerate(parents):
        if context + i < 0 or not -1 <= p < i:
            lines.append(None)
        elif p == -1:
            lines.append([i])
        else:
            lines.append(None if lines[p] is None else lines[p] + [i])
    return lines


def tree(q, k, v, lengths, parents=None, scale=None):
    """``(value, bound)`` of the drafts' attention, [B, H, T, Dv] in 64 bits."""
    b_all, h, t, d = q.shape
    hk, c, dv = k.shape[1], k.shape[2], v.shape[3]
    g, scale = h // hk, d ** -0.5 if scale is None else scale
    f64 = dict(dtype=torch.float64, device=q.device)
    out, tol = torch.zeros(b_all, h, t, dv, **f64), torch.zeros(b_all, h, t, dv, **f64)
    for b in range(b_all):
        n = min(max(0, lengths[b]), c)
        lines = lineage(range(-1, t - 1) if parents is None else parents[b], n - t)
        if parents is None:  # tokens at a negative position begin nothing
            lines = [None if n - t + i < 0 else [j for j in range(i + 1) if n - t + j >= 0] for i in range(t)]
        live = [i for i in range(t) if lines[i] is not None]
        if not live:
            continue
        seen = torch.zeros(len(live), n, dtype=torch.bool)
        seen[:, :max(0, n - t)] = True
        for at, i in enumerate(live):
            seen[at, [n - t + j for j in lines[i]]] = True
        used = seen.any(0).to(q.device)
        seen = seen.to(q.device)[:, used]
        for head in range(h):
            kv = head // g
            one = Head(q[b, head, live], k[b, kv, :n][used], v[b, kv, :n][used], seen, scale, q.dtype)
            out[b, head, live], tol[b, head, live] = one.out, one.out_tol
    return out, tol


def check(name, got, value, bound, norm=None):
    """Every element within its bound, and all of them together within ``norm`` of the value's 2-norm."""
    err = (got.double() - value).abs()
    bound = bound + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -100)
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all(), f"{name}: not finite"
    assert worst <= 0, f"{name}: {worst} past its bound, largest error {err.max().item()}"
    if norm is not None and value.norm() > 0:
        assert err.norm() <= norm * value.norm(), f"{name}: {(err.norm() / value.norm()).item()} of the 2-norm, allowed {norm}"
