"""Differential attention in float64 with bounds for what the kernels may be off by.

The kernels round, with ``u`` half a step of the element type: the
probabilities before their product with v, the mixed probabilities and dS
before theirs with dO, K and Q, and every result. Everything
else is float32: a sum of n products is off by at most n 2^-24 times the sum of
their magnitudes, an exponential by a few 2^-24 of itself plus its argument's
error. ``attention`` returns each result with the bound these add up to, element
by element.
"""

from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _visible(i0, rows, keys, causal):
    if not causal:
        return torch.ones(rows, keys, dtype=torch.bool)
    return torch.arange(keys)[None, :] <= (torch.arange(rows) + i0)[:, None]


def attention(q, k, v, lam, *, causal, scale=None, lengths=None, cached=False, dout=None):
    """``{name: (value, bound)}`` for out and, with ``dout``, dq, dk, dv, dlam (float64, on the CPU)."""
    u = half_step(q.dtype)
    q, k, v, lam = (t.detach().cpu().double() for t in (q, k, v, lam))
    dout = None if dout is None else dout.detach().cpu().double()
    b_all, h2, sq, d = q.shape
    _, hk, sk, dv = v.shape
    h = h2 // 2
    group = h // hk
    scale = d ** -0.5 if scale is None else scale
    lam = lam.reshape(-1).expand(h) if lam.numel() == 1 else lam
    lens = [sk] * b_all if lengths is None else [max(0, min(sk, n)) for n in lengths.cpu().tolist()]
    shapes = {"out": (b_all, h, sq, dv), "dq": q.shape, "dk": k.shape, "dv": v.shape, "dlam": (h,)}
    res = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64)) for n, s in shapes.items()}
    for b in range(b_all):
        n = lens[b]
        first = n - sq if cached else 0
        i0 = max(0, -first)                      # rows before it stand at negative positions
        i1 = sq if cached else min(sq, n)
        if i1 <= i0:
            continue
        for head in range(h):
            kv, lm = head // group, float(lam[head])
            seen = _visible(first + i0, i1 - i0, n, causal or cached)
            P, dP_rel = [], []
            for m in range(2):
                qm, km = q[b, 2 * head + m, i0:i1], k[b, 2 * kv + m, :n]
                s = (qm @ km.T) * scale
                mag = (qm.abs() @ km.abs().T) * abs(scale)
                s = s.masked_fill(~seen, -math.inf)
                P.append(torch.softmax(s, -1))
                # A score's error: its sum's, the product with scale log2 e, the subtraction; the row's own sum likewise.
                err = ((d + 4) * F32 * mag + 4 * F32 * (s.masked_fill(~seen, 0).abs() + 16)).masked_fill(~seen, 0)
                dP_rel.append(err + err.max(-1, keepdim=True).values + (n + 8) * F32)
            V = v[b, kv, :n]
            o = [p @ V for p in P]
            mag_o = [p @ V.abs() for p in P]
            err_o = [u * mag_o[m] + (P[m] * dP_rel[m]) @ V.abs() + (n + 8) * F32 * mag_o[m] for m in range(2)]
            out = o[0] - lm * o[1]
            out_err = err_o[0] + abs(lm) * err_o[1]
            out_err = out_err + (u + 4 * F32) * (out.abs() + out_err)
            res["out"][0][b, head, i0:i1] = out
            res["out"][1][b, head, i0:i1] = out_err
            if dout is None:
                continue
            do = dout[b, head, i0:i1]
            mixed = P[0] - lm * P[1]
            mixed_err = P[0] * dP_rel[0] + abs(lm) * P[1] * dP_rel[1] + 4 * F32 * (P[0] + abs(lm) * P[1])
            mixed_err = mixed_err + u * (mixed.abs() + mixed_err)
            rows = i1 - i0
            _add(res["dv"], (b, kv, slice(0, n)), mixed.T @ do,
                 mixed_err.T @ do.abs() + (rows + 8) * F32 * (mixed.abs().T @ do.abs()))
            dp = do @ V.T
            dp_mag = do.abs() @ V.abs().T
            dp_err = (dv + 4) * F32 * dp_mag
            # Saved in float32: each map's output.
            saved = [err_o[m] + 4 * F32 * o[m].abs() for m in range(2)]
            kept = [o[m].abs() for m in range(2)]
            for m in range(2):
                c = 1.0 if m == 0 else -lm
                delta = (do * o[m]).sum(-1, keepdim=True)
                delta_err = (do.abs() * (saved[m] + (dv + 4) * F32 * (kept[m] + saved[m]))).sum(-1, keepdim=True)
                t = dp - delta
                t_err = dp_err + delta_err + 4 * F32 * (dp_mag + delta.abs())
                ds = c * P[m] * t
                ds_err = abs(c) * P[m] * (dP_rel[m] * t.abs() + t_err + dP_rel[m] * t_err) + 4 * F32 * ds.abs()
                ds_err = ds_err + u * (ds.abs() + ds_err)
                km, qm = k[b, 2 * kv + m, :n], q[b, 2 * head + m, i0:i1]
                acc = (n + 8) * F32 * (ds.abs() @ km.abs())
                _add(res["dq"], (b, 2 * head + m, slice(i0, i1)), scale * (ds @ km),
                     abs(scale) * (ds_err @ km.abs() + acc))
                acc = (rows + 8) * F32 * (ds.abs().T @ qm.abs())
                _add(res["dk"], (b, 2 * kv + m, slice(0, n)), scale * (ds.T @ qm),
                     abs(scale) * (ds_err.T @ qm.abs() + acc))
                if m == 1:
                    # delta_1 back from dP: no rounding to the element type is left in it, only
                    # (1 - sum of P_1) times delta_1's error, which dP_rel covers.
                    err = (P[1] * (dP_rel[1] * (t.abs() + delta_err) + dp_err + 4 * F32 * dp_mag)).sum()
                    err = err + ((n + 8) * F32 * (P[1] * t.abs()).sum()) + (delta_err * dP_rel[1].max()).sum()
                    res["dlam"][0][head] -= delta.sum()
                    res["dlam"][1][head] += err + 8 * F32 * delta.abs().sum()
    for name in ("dq", "dk", "dv"):
        value, bound = res[name]
        bound += (u + 4 * F32) * (value.abs() + bound)
    return res


def _add(pair, at, value, bound):
    pair[0][at] += value
    pair[1][at] += bound


def assert_within(got, want, name, floor=0.0):
    """Every element within its bound (``floor``: half a step of the smallest subnormal, say)."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, f"{name}: shape {tuple(got.shape)}, expected {tuple(value.shape)}"
    off = (got - value).abs()
    bad = ~(off <= bound + floor)
    if bool(bad.any()):
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} beyond their bound, first {at}: "
                             f"got {float(got[at])}, want {float(value[at])}, bound {float(bound[at])}")
