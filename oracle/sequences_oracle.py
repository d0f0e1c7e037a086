"""Rotary positions and attention over packed sequences from their definitions in 64 bits, with bounds on how far a kernel
that sums in fp32 and rounds its results (and, in 16-bit types, P and dS before their products) may be off.
TEST INFRASTRUCTURE ONLY.

Units: u = ``finfo.eps / 2`` of the storage type, what one rounding does to a value; e = 2^-23, one addition in fp32 that cuts
off instead of rounding (as matrix instructions may), for which a sum of n terms is off by n e times the sum of magnitudes.
"""
import math

import torch

from .inputs_oracle import check, rounding  # noqa: F401  (check: for the tests)

E = 2.0 ** -23


def rotary(x, positions, frequencies, layout, amplitude=1.0, inverse=False):
    """(value, bound); x [..., N, H, D], positions of the axes before the heads."""
    n = frequencies.shape[0]
    X = x.double()
    turns = positions.double()[..., None, None] * (frequencies.double() / (2 * math.pi))
    angle = positions.double()[..., None, None] * frequencies.double() * (-1 if inverse else 1)
    cos, sin = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude
    part = X[..., :2 * n]
    a, b = (part[..., :n], part[..., n:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    join = lambda u, w: torch.cat([u, w], -1) if layout == "half" else torch.stack([u, w], -1).flatten(-2)  # noqa: E731
    y = torch.cat([join(a * cos - b * sin, a * sin + b * cos), X[..., 2 * n:]], -1)
    # the fraction of a turn: 1 / 2 pi, its product with the frequency and that with the position are rounded in 64 bits, and
    # so is the angle here, 2^-53 of the turns each, 2^-51 in all; doubled and rounded to fp32 (2^-24 of at most 1, pi
    # times that of a radian); sincospi within two units in the last place; three roundings of products and the sum
    off = abs(amplitude) * (turns.abs() * 2.0 ** -51 * 2 * math.pi + math.pi * 2.0 ** -24 + 2.0 ** -22 + 4 * 2.0 ** -24)
    err = (a.abs() + b.abs()) * off
    bound = torch.cat([join(err, err), torch.zeros_like(X[..., 2 * n:])], -1)
    return y, rounding(x.dtype, y) * (y != X).double() + bound


def attention(q, k, v, spans, causal, scale=None, d=None):
    """[(value, bound)] of o, and with d of dq, dk, dv.  spans: (first query, queries, first key, keys) of each sequence."""
    t, H, Hk, D = q.dtype, q.shape[1], k.shape[1], q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    G = H // Hk
    small = t != torch.float32
    u = torch.finfo(t).eps / 2 if small else 0.0
    # P and dS below the smallest normal fp16: half of the smallest step.  In the forward P is not yet divided by its row's sum,
    # of which a kernel makes sure that it is at least 2^-4.
    least = 2.0 ** -25 if t == torch.float16 else 0.0
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)  # noqa: E731
    out, eout = zeros(q), zeros(q)
    grads = [[zeros(x), zeros(x)] for x in (q, k, v)]
    for i0, nq, j0, nk in spans:
        if nq == 0 or nk == 0:
            continue
        hid = torch.zeros(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            hid = torch.arange(nk, device=q.device) > torch.arange(nk - nq, nk, device=q.device)[:, None]
        some = (~hid).any(-1, keepdim=True)
        for h in range(H):
            Q, K, V = q[i0:i0 + nq, h].double(), k[j0:j0 + nk, h // G].double(), v[j0:j0 + nk, h // G].double()
            s = (Q @ K.t()) * scale
            s = s.masked_fill(hid, -math.inf)
            p = torch.softmax(torch.where(some, s, 0.0), -1) * some
            p = p.masked_fill(hid, 0.0)
            mag = (Q.abs() @ K.abs().t()) * abs(scale)
            # an exponent: the score's sum of D terms, then three roundings of numbers up to the largest score or log-sum-exp;
            # the exponential itself 2^-21
            top = mag.masked_fill(hid, 0.0).amax(-1, keepdim=True) + math.log(nk + 1)
            ep = (D * E * mag).masked_fill(hid, 0.0).amax(-1, keepdim=True) + 8 * 2.0 ** -24 * top + 2.0 ** -21
            ep = 2 * ep + nk * E  # (of its own and of the row's sum)
            o = p @ V
            # P rounded, its sum of either the rounded or the unrounded values; the product's sum
            ebig = p @ V.abs()
            eo = (2 * u + 2 * ep + nk * E) * ebig + 16 * least * (V.abs().sum(0) + nk * ebig)
            out[i0:i0 + nq, h] = o
            eout[i0:i0 + nq, h] = eo + rounding(t, o.abs() + eo)
            if d is None:
                continue
            dO = d[i0:i0 + nq, h].double()
            dp = dO @ V.t()
            delta = (dO * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            edp = D * E * (dO.abs() @ V.abs().t())
            edelta = (dO.abs() * (eout[i0:i0 + nq, h] + D * E * o.abs())).sum(-1, keepdim=True)
            eds = p * (edp + edelta + 2.0 ** -23 * (dp.abs() + delta.abs())) * (1 + ep) + ds.abs() * (ep + u) + u * p * (edp + edelta) + least * (~hid)
            rows, keys = slice(i0, i0 + nq), slice(j0, j0 + nk)
            grads[0][0][rows, h] += scale * (ds @ K)
            grads[0][1][rows, h] += abs(scale) * (eds @ K.abs() + nk * E * (ds.abs() @ K.abs()))
            grads[1][0][keys, h // G] += scale * (ds.t() @ Q)
            grads[1][1][keys, h // G] += abs(scale) * (eds.t() @ Q.abs() + G * nq * E * (ds.abs().t() @ Q.abs()))
            grads[2][0][keys, h // G] += p.t() @ dO
            grads[2][1][keys, h // G] += (p * (ep + u) + least * (~hid)).t() @ dO.abs() + G * nq * E * (p.t() @ dO.abs())
    res = [(out, eout)]
    if d is not None:
        res += [(g, e + rounding(t, g.abs() + e)) for g, e in grads]
    return res
