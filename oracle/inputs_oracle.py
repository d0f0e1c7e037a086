"""The operators that make the attention's inputs, from their definitions in 64 bits, with bounds on how far a kernel
that works in fp32 and rounds its results once may be off.  TEST INFRASTRUCTURE ONLY.

A rounding to a type is off by at most half a step, ``finfo.eps / 2`` relative to the value (``rounding``).  Sums of n values
in fp32 are off by at most ``depth`` of those times the sum of magnitudes, ``depth`` the longest chain of additions.
"""
import torch

UNIT32 = 2.0 ** -24


def rounding(dtype, value):
    """Half a step of the type at the value.  Below ``finfo.tiny`` the steps no longer shrink (fp16: 2^-24 from 2^-14 down), so
    half a step there is what it is at ``tiny``: eps / 2 * tiny."""
    info = torch.finfo(dtype)
    return info.eps / 2 * value.abs().clamp_min(info.tiny)


def row_depth(C):
    """Roundings on the way of a value through a sum over a row: up to 1/128 of it one after another, a tree of the rest."""
    return 16 + C / 128


def rows_depth(N):
    """The same for a sum over N rows: up to 1/128 of them in turn, then the partial sums of at most 1 200 shares eight at a time."""
    return 64 + N / 128 + 150


def normalise(x, eps):
    mean = x.mean(-1, keepdim=True)
    r = (x - mean).square().mean(-1, keepdim=True).add(eps).rsqrt()
    return (x - mean) * r, r


def normalised_error(x, r):
    """Bound on the error of (x - mean) r in fp32, as (absolute, relative) parts: the mean is off by depth units of the
    largest value, which r carries over; and so is the spread that r is made of."""
    k = row_depth(x.shape[-1]) * UNIT32
    return 2 * k * (1 + x.abs().amax(-1, keepdim=True) * r)


def layer_norm(x, w, b, eps, dy=None):
    """[(value, bound)] of y, and with dy of dx, dw, db (None for a weight that is not there).  x, dy: [N, C] in storage types."""
    t, N, C = x.dtype, x.shape[0], x.shape[1]
    X = x.double()
    W = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    Bv = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    h, r = normalise(X, eps)
    eh = normalised_error(X, r)
    y = h * W + Bv
    res = [(y, rounding(t, y) + eh * W.abs() * (1 + h.abs()) + 4 * UNIT32 * (y.abs() + Bv.abs()))]
    if dy is None:
        return res
    D = dy.double()
    g = D * W
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    most = g.abs().amax(-1, keepdim=True) if C else g
    res.append((dx, rounding(t, dx) + 4 * r * most * (eh + row_depth(C) * UNIT32) * (1 + h.abs()) ** 2))
    depth = rows_depth(N) * UNIT32
    dw, db = (D * h).sum(0), D.sum(0)
    res.append(None if w is None else (dw, rounding(w.dtype, dw) + ((eh * (1 + h.abs()) + depth * h.abs()) * D.abs()).sum(0)))
    res.append(None if b is None else (db, rounding(b.dtype, db) + depth * D.abs().sum(0)))
    return res


def bucket(rel, scheme, n, max_distance):
    """The row of the table for a key ``rel`` ahead of its query, in whole numbers."""
    if scheme == "clip":
        return min(max(-rel, -max_distance), max_distance) + max_distance
    side = n if scheme == "log_causal" else n // 2
    a = max(-rel, 0) if scheme == "log_causal" else abs(rel)
    exact = side // 2
    m = side - exact
    f = a
    if a >= exact:
        f = exact
        while f + 1 < side and a ** m * exact ** (f + 1 - exact) >= max_distance ** (f + 1 - exact) * exact ** m:
            f += 1
    return f + (side if scheme == "log" and rel > 0 else 0)


def bucket_rows(q, k, scheme, n, max_distance):
    """[B, Rq, Rk] rows of the table; differences that 64 bits might not hold are taken in Python's whole numbers."""
    M = max_distance + 1
    of = torch.tensor([bucket(r, scheme, n, max_distance) for r in range(-M, M + 1)])
    if max((abs(v) for row in q + k for v in row), default=0) < 2 ** 61:
        rel = torch.tensor(k).unsqueeze(1) - torch.tensor(q).unsqueeze(2)
        return of[rel.clamp(-M, M) + M]
    rel = [[[min(max(kj - qi, -M), M) + M for kj in ks] for qi in qs] for qs, ks in zip(q, k)]
    return of[torch.tensor(rel, dtype=torch.long).reshape(len(q), len(q[0]), len(k[0]))]


def relative_bias(table, rows, base, out_dtype, d=None):
    """(out, [(dtable, bound)]): out to the bit (one addition in fp32, one rounding)."""
    v = table.float()[rows].permute(0, 3, 1, 2).unsqueeze(1)
    if base is not None:
        v = v + base.float()
    out = v.to(out_dtype)
    if d is None:
        return out, None
    H = table.shape[1]
    D = d.expand(d.shape).double().squeeze(1).permute(0, 2, 3, 1).reshape(-1, H)
    idx = rows.reshape(-1)
    zeros = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
    s, m = zeros.clone().index_add_(0, idx, D), zeros.clone().index_add_(0, idx, D.abs())
    # a lane adds up to 32 rows of 8 values of a strip, item after item; then 4 x 32 lanes, then the blocks
    return out, (s, rounding(table.dtype, s) + (600 + idx.numel() / 65536) * UNIT32 * m)


def pair_projection(z, W, g, b, eps, d=None):
    """[(value, bound)] of out, and with d of dz, dW, dg, db.  z: [B, I, J, C], d: [B, 1, H, I, J].  For 16-bit types a
    kernel may split an fp32 factor into two bf16 pieces (off by 2^-16) and leave out the product of the low pieces (2^-16)."""
    t, C, dev = z.dtype, z.shape[-1], z.device
    split = 3 * 2.0 ** -16 if t != torch.float32 else 8 * UNIT32
    Z, Wd = z.double(), W.double()
    G = torch.ones(C, dtype=torch.float64, device=dev) if g is None else g.double()
    Bv = torch.zeros(C, dtype=torch.float64, device=dev) if b is None else b.double()
    h, r = normalise(Z, eps)
    eh = normalised_error(Z, r)
    y = h * G + Bv
    mm = lambda a, w: torch.einsum("bijc,hc->bhij", a, w).unsqueeze(1)  # noqa: E731
    out = mm(y, Wd)
    mag = mm((h.abs() * (split + 2 * row_depth(C) * UNIT32) + eh * (1 + h.abs())) * G.abs() + Bv.abs() * row_depth(C) * UNIT32, Wd.abs())
    res = [(out, rounding(t, out) + mag)]
    if d is None:
        return res
    D = d.double().squeeze(1)
    dy = torch.einsum("bhij,hc->bijc", D, Wd)
    u = dy * G
    dz = r * (u - u.mean(-1, keepdim=True) - h * (u * h).mean(-1, keepdim=True))
    um = torch.einsum("bhij,hc->bijc", D.abs(), Wd.abs()) * G.abs()
    most = um.amax(-1, keepdim=True)
    res.append((dz, rounding(t, dz) + 4 * r * most * (split + eh + row_depth(C) * UNIT32) * (1 + h.abs()) ** 2))
    N = Z[..., 0].numel()
    depth = rows_depth(N) * UNIT32
    # the sums that the weights' gradients are made of, and their bounds
    M, s = torch.einsum("bhij,bijc->hc", D, h), D.sum((0, 2, 3))
    eM = torch.einsum("bhij,bijc->hc", D.abs(), h.abs() * (split + depth) + eh * (1 + h.abs()))
    es = depth * D.abs().sum((0, 2, 3))
    dW = M * G + s[:, None] * Bv
    res.append((dW, rounding(W.dtype, dW) + 2 * (eM * G.abs() + es[:, None] * Bv.abs()) + 4 * UNIT32 * ((M * G).abs() + (s[:, None] * Bv).abs())))
    dg, db = (Wd * M).sum(0), (Wd * s[:, None]).sum(0)
    more = (4 + W.shape[0]) * UNIT32
    res.append(None if g is None else (dg, rounding(g.dtype, dg) + (Wd.abs() * (eM + more * M.abs())).sum(0)))
    res.append(None if b is None else (db, rounding(b.dtype, db) + (Wd.abs() * (es + more * s.abs())[:, None]).sum(0)))
    return res


def check(name, got, want):
    """Every value within its bound.  One that lies above the largest number of the result's type (or may, within its bound)
    rounds to infinity of its sign."""
    if want is None:
        return
    value, bound = want
    got = got.detach()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.double() - value).abs()
    over = (value.abs() + bound > torch.finfo(got.dtype).max) & torch.isinf(got) & (torch.sign(got) == torch.sign(value))
    bad = ~(off <= bound) & ~over
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values are off by up to {float((off / bound.clamp_min(1e-300))[bad].max()):.3g} times what they may be"
