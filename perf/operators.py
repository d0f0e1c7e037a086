"""The operators around the attention as cases that can be timed one by one: layer norm, the learned
relative position bias, and the projection of the pair representation to a pair bias.

A case is one call of one operator, forward only (inference) or forward and backward (training).  Where
``own`` is false, ``run`` computes the operators in their plain form, elementary operations in 32 bits
(long sums in 64); where it is true, ``run`` calls the package.  Sizes are those of the package's workloads
(MSA [1,128,384] and [2,512,768], crops of 384 residues), their channel counts (pair 128, MSA 256), generic
ones, and odd ones: a protein has any number of residues.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def _norm(name, train, B, S, R, C, dtype, weights="fp32", affine=True, layout="dense"):
    """``layout``: "dense" rows; "turned" ([B,R,S,C] seen as [B,S,R,C], as column-wise attention normalises an
    MSA); "sliced" (the first C of 2 C columns of a fused projection)."""
    c = dict(op="norm", train=train, B=B, S=S, R=R, C=C, dtype=dtype, weights=weights, affine=affine, layout=layout)
    return c if name is None else dict(c, name=name)


def _relative(name, train, B, H, Rq, Rk, scheme, n, M, table, out, base=False):
    """``scheme``: "clip" (n = 2 M + 1 buckets), "log" or "log_causal" (n buckets up to distance M); ``base``: the
    bias is added to a pair bias that is there."""
    c = dict(op="relative", train=train, B=B, H=H, Rq=Rq, Rk=Rk, scheme=scheme, n=n, M=M, table=table, out=out, base=base)
    return c if name is None else dict(c, name=name)


def _projection(name, train, B, R, C, H, dtype, weights="fp32", affine=True, turned=False):
    """``turned``: pair[b,j,i] is read for (i,j), as attention around ending nodes does."""
    c = dict(op="projection", train=train, B=B, R=R, C=C, H=H, dtype=dtype, weights=weights, affine=affine, turned=turned)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a single short sequence in inference: launch and host time are all there is
        _norm("norm short, inference", False, 1, 1, 32, 256, "bf16"),
        # the MSA of a training crop before row attention: mixed precision, fp32 weights
        _norm("norm msa, training", True, 1, 128, 384, 256, "bf16"),
        # column-wise attention over the MSA of a large crop: the rows lie transposed; the largest
        _norm("norm large turned, training", True, 2, 512, 768, 256, "bf16", weights="bf16", layout="turned"),
        # a wide and odd number of channels in half precision
        _norm("norm odd wide, training", True, 1, 1, 1499, 1111, "fp16", weights="fp16"),
        # one query against a long row of keys, as in decoding: latency
        _relative("relative one query, inference", False, 1, 32, 1, 2048, "log_causal", 32, 128, "fp32", "bf16"),
        # residue offsets clipped at 32, one bias for a training crop
        _relative("relative crop, training", True, 1, 8, 384, 384, "clip", 65, 32, "fp32", "fp32"),
        # long sequences, logarithmic buckets
        _relative("relative long, training", True, 2, 16, 2048, 2048, "log", 32, 128, "bf16", "bf16"),
        # added to the pair bias of a protein of odd length, in single precision
        _relative("relative added odd, training", True, 1, 4, 437, 437, "clip", 65, 32, "fp32", "fp32", base=True),
        # pair bias of MSA row attention in a training crop
        _projection("projection crop, training", True, 1, 384, 128, 8, "bf16"),
        # a whole protein of odd length, triangle attention around ending nodes
        _projection("projection odd turned, inference", False, 1, 437, 128, 4, "fp16", weights="fp16", turned=True),
        # large crops
        _projection("projection large, training", True, 2, 768, 128, 8, "bf16", weights="bf16"),
        # a small template stack in single precision
        _projection("projection fp32, training", True, 1, 100, 64, 4, "fp32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "relative", "projection"])
    train = rng.random() < 0.65
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    weights = rng.choice(["fp32", dtype])
    if op == "norm":
        C = rng.choice([32, 64, 128, 256, 384, 512, 1024, 2048, 4096, 8192]) if rng.random() < 0.6 else _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, max(1, (1 << 26) // C))
        S = _log_int(rng, 1, min(rows, 512))
        return _norm(None, train, 1, S, max(1, rows // S), C, dtype, weights, rng.random() < 0.8,
                     rng.choice(["dense", "dense", "turned", "sliced"]))
    if op == "relative":
        scheme = rng.choice(["clip", "log", "log_causal"])
        M = _log_int(rng, 8, 300) if scheme == "clip" else rng.choice([64, 128, 200, 1000])
        n = 2 * M + 1 if scheme == "clip" else rng.choice([16, 32, 64])
        B, H = rng.choice([1, 1, 2]), rng.choice([1, 4, 8, 12, 16, 32])
        Rk = _log_int(rng, 1, 2048)
        Rq = 1 if rng.random() < 0.2 else Rk
        return _relative(None, train, B, H if B * H <= 32 else 16, Rq, Rk, scheme, n, M, weights, dtype, rng.random() < 0.3)
    C, H = rng.choice([32, 64, 100, 128, 128, 192, 256]), rng.choice([1, 4, 8, 8, 12, 16])
    R = _log_int(rng, 1, 768 if C * H <= 1024 else 512)
    return _projection(None, train, 1, R, C, H, dtype, weights, rng.random() < 0.8, rng.random() < 0.3)


def _log_edges(n, M, scheme):
    """E, and the distances from which on the buckets E + 1, E + 2, ... apply: the k-th is the smallest whole d with
    (d / E) ** m >= (M / E) ** k, in whole numbers; powers in 64 bits say where to look."""
    half = n // 2 if scheme == "log" else n
    E = half // 2
    m = half - E
    near = [int(E * (M / E) ** (k / m)) for k in range(1, m)]
    return E, [next(d for d in range(max(E, a - 1), a + 3) if d ** m * E ** k >= M ** k * E ** m) for k, a in enumerate(near, 1)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    train = case["train"]

    def normal(shape, std, dtype, mean=0.0):
        return torch.empty(shape, dtype=torch.float32, device=dev).normal_(mean, std, generator=g).to(DTYPES[dtype])

    st = dict(case=case)
    if case["op"] == "norm":
        B, S, R, C = (case[k] for k in "BSRC")
        # a residual stream: channels have their own offsets
        shape = (B, R, S, C) if case["layout"] == "turned" else (B, S, R, 2 * C if case["layout"] == "sliced" else C)
        offsets = torch.empty(shape[-1], device=dev).normal_(0.0, 0.5, generator=g)
        x = (torch.empty(shape, device=dev).normal_(0.0, 1.5, generator=g) + offsets).to(DTYPES[case["dtype"]])
        st["x"] = x.transpose(1, 2) if case["layout"] == "turned" else x[..., :C]
        st["w"] = normal((C,), 0.2, case["weights"], 1.0) if case["affine"] else None
        st["b"] = normal((C,), 0.2, case["weights"]) if case["affine"] else None
        if train:
            st["d"] = normal((B, S, R, C), 1.0, case["dtype"])
        leaves = ("x", "w", "b")
    elif case["op"] == "relative":
        B, H, Rq, Rk, n, M = (case[k] for k in ("B", "H", "Rq", "Rk", "n", "M"))
        # residue numbers: mostly consecutive, with gaps where a structure is not resolved and a jump between chains
        step = 1 + (torch.rand((B, Rk), generator=g, device=dev) < 0.02) * torch.randint(1, 40, (B, Rk), generator=g, device=dev)
        st["keys"] = torch.cumsum(step, 1)
        st["queries"] = st["keys"][:, Rk - Rq:].contiguous()
        st["table"] = normal((n, H), 0.5, case["table"])
        st["base"] = normal((B, 1, H, Rq, Rk), 1.0, case["out"]) if case["base"] else None
        if case["scheme"] != "clip":
            st["exact_up_to"], edges = _log_edges(n, M, case["scheme"])
            st["edges"] = torch.tensor(edges, dtype=torch.int64, device=dev)
        if train:
            st["d"] = normal((B, 1, H, Rq, Rk), 1.0, case["out"])
        leaves = ("table", "base")
    else:
        B, R, C, H = (case[k] for k in "BRCH")
        offsets = torch.empty(C, device=dev).normal_(0.0, 0.5, generator=g)
        z = (torch.empty((B, R, R, C), device=dev).normal_(0.0, 2.0, generator=g) + offsets).to(DTYPES[case["dtype"]])
        st["z"] = z.transpose(1, 2) if case["turned"] else z
        st["weight"] = normal((H, C), C ** -0.5, case["weights"])
        st["w"] = normal((C,), 0.2, case["weights"], 1.0) if case["affine"] else None
        st["b"] = normal((C,), 0.2, case["weights"]) if case["affine"] else None
        if train:
            st["d"] = normal((B, 1, H, R, R), 1.0, case["dtype"])
        leaves = ("z", "weight", "w", "b")
    if train:
        st["leaves"] = [st[k].requires_grad_() for k in leaves if st[k] is not None]
    return st


def _call(st):
    """The package's call of a case."""
    import evoformer_triton_b200 as evo
    case = st["case"]
    if case["op"] == "norm":
        return evo.layer_norm(st["x"], st["w"], st["b"], eps=EPS)
    if case["op"] == "relative":
        return evo.relative_position_bias(st["table"], st["queries"], st["keys"], max_distance=case["M"], buckets=case["scheme"],
                                          pair_bias=st["base"], dtype=DTYPES[case["out"]])
    return evo.pair_bias_projection(st["z"], st["weight"], st["w"], st["b"], eps=EPS)


def _normalised(x):
    x = x.float()
    centred = x - x.mean(-1, keepdim=True)
    r = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return centred * r, r


def _d_normalised(d, h, r):
    """The gradient of the rows from that of the normalised rows h."""
    return r * (d - d.mean(-1, keepdim=True) - h * (d * h).mean(-1, keepdim=True))


def _sum_rows(t):
    return t.reshape(-1, t.shape[-1]).sum(0, dtype=torch.float64)


def _plain_norm(st):
    x, w, b = st["x"].detach(), st["w"], st["b"]
    h, r = _normalised(x)
    y = (h if w is None else h * w.detach().float() + b.detach().float()).to(x.dtype)
    if not st["case"]["train"]:
        return [y]
    d = st["d"].float()
    dx = _d_normalised(d if w is None else d * w.detach().float(), h, r).to(x.dtype)
    return [y, dx] if w is None else [y, dx, _sum_rows(d * h).to(w.dtype), _sum_rows(d).to(b.dtype)]


def _rows(st):
    """The row of the table for every query and key, [B, Rq, Rk]."""
    case = st["case"]
    M = case["M"]
    ahead = st["keys"][:, None, :] - st["queries"][:, :, None]
    if case["scheme"] == "clip":
        return (-ahead).clamp(-M, M) + M
    E = st["exact_up_to"]
    a = ahead.abs() if case["scheme"] == "log" else (-ahead).clamp(min=0)
    f = torch.where(a < E, a, E + torch.bucketize(a, st["edges"], right=True))
    return f + (ahead > 0) * (case["n"] // 2) if case["scheme"] == "log" else f


def _plain_relative(st):
    case, table, base = st["case"], st["table"].detach(), st["base"]
    rows = _rows(st)
    bias = table.float()[rows].permute(0, 3, 1, 2).unsqueeze(1)
    out = (bias if base is None else bias + base.detach().float()).to(DTYPES[case["out"]])
    if not case["train"]:
        return [out]
    d = st["d"].squeeze(1).permute(0, 2, 3, 1).reshape(-1, case["H"])
    sums = torch.zeros(table.shape, dtype=torch.float64, device=d.device).index_add_(0, rows.reshape(-1), d.double())
    return [out, sums.to(table.dtype)] + ([] if base is None else [st["d"].to(base.dtype)])


def _plain_projection(st):
    z, W, w, b = (None if st[k] is None else st[k].detach() for k in ("z", "weight", "w", "b"))
    h, r = _normalised(z)
    y = h if w is None else h * w.float() + b.float()
    out = torch.matmul(y, W.float().t()).permute(0, 3, 1, 2).unsqueeze(1).to(z.dtype)
    if not st["case"]["train"]:
        return [out]
    d = st["d"].squeeze(1).permute(0, 2, 3, 1).float()
    dy = torch.matmul(d, W.float())
    dz = _d_normalised(dy if w is None else dy * w.float(), h, r).to(z.dtype)
    H, C = W.shape
    dW = torch.matmul(d.reshape(-1, H).double().t(), y.reshape(-1, C).double()).to(W.dtype)
    return [out, dz, dW] if w is None else [out, dz, dW, _sum_rows(dy * h).to(w.dtype), _sum_rows(dy).to(b.dtype)]


def run(state):
    if own:
        if not state["case"]["train"]:
            with torch.no_grad():
                return [_call(state)]
        out = _call(state)
        return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["d"])]
    with torch.no_grad():
        return {"norm": _plain_norm, "relative": _plain_relative, "projection": _plain_projection}[state["case"]["op"]](state)


def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiating them; buckets from whole numbers, distance by distance."""
    st = prepare(case, seed)
    leaves = {k: v.detach().double().requires_grad_(case["train"]) for k, v in st.items()
              if k in ("x", "w", "b", "table", "base", "z", "weight") and v is not None}
    rest = {k: st[k] for k in ("d", "queries", "keys") if k in st}
    wanted = [k for k in ("x", "table", "base", "z", "weight", "w", "b") if k in leaves]
    del st

    def norm(v):
        var, mean = torch.var_mean(v, dim=-1, unbiased=False, keepdim=True)
        v = (v - mean) / torch.sqrt(var + EPS)
        return v * leaves["w"] + leaves["b"] if "w" in leaves else v

    if case["op"] == "norm":
        out = norm(leaves["x"])
    elif case["op"] == "projection":
        out = torch.einsum("bijc,hc->bhij", norm(leaves["z"]), leaves["weight"]).unsqueeze(1)
    else:
        n, M, scheme = case["n"], case["M"], case["scheme"]

        def bucket(rel):  # rel: key minus query
            if scheme == "clip":
                return min(max(-rel, -M), M) + M
            half = n // 2 if scheme == "log" else n
            a = abs(rel) if scheme == "log" else max(-rel, 0)
            E = half // 2
            m = half - E
            if a < E:
                f = a
            else:
                k = 0
                while k + 1 < m and a ** m * E ** (k + 1) >= M ** (k + 1) * E ** m:
                    k += 1
                f = E + k
            return f + (half if scheme == "log" and rel > 0 else 0)

        of = torch.tensor([bucket(r) for r in range(-M - 1, M + 2)], device="cuda")
        rel = rest["keys"].unsqueeze(1) - rest["queries"].unsqueeze(2)
        rows = of[rel.clamp(-M - 1, M + 1) + M + 1]
        out = torch.stack([leaves["table"][:, h][rows] for h in range(case["H"])], 1).unsqueeze(1)
        if "base" in leaves:
            out = out + leaves["base"]
    if not case["train"]:
        return [out.detach()]
    return [out.detach(), *torch.autograd.grad(out, [leaves[k] for k in wanted], rest["d"].double())]


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    train = case["train"]
    if case["op"] == "norm":
        N, C = case["B"] * case["S"] * case["R"], case["C"]
        weights = 2 * C * size[case["weights"]] if case["affine"] else 0
        # x in, y out; with a gradient dy in and dx out (x is read once), weights in and their gradients out
        return {"bytes": N * C * size[case["dtype"]] * (4 if train else 2) + weights * (2 if train else 1),
                "flops": float(N * C * (23 if train else 8))}
    if case["op"] == "relative":
        B, H, Rq, Rk = (case[k] for k in ("B", "H", "Rq", "Rk"))
        scores = B * H * Rq * Rk * size[case["out"]]
        table = case["n"] * H * size[case["table"]]
        # the bias out, the one it is added to in; with a gradient d(bias) in, which is the other addend's as it is
        tensors = 1 + case["base"] + train
        return {"bytes": scores * tensors + table * (2 if train else 1) + 8 * B * (Rq + Rk), "flops": float(B * H * Rq * Rk * (2 if train else 1))}
    B, R, C, H = (case[k] for k in "BRCH")
    N, es = B * R * R, size[case["dtype"]]
    weights = (H * C + (2 * C if case["affine"] else 0)) * size[case["weights"]]
    # the pair representation in, the bias out; with a gradient d(bias) in and d(pair) out
    return {"bytes": N * es * (C + H) * (2 if train else 1) + weights * (2 if train else 1),
            "flops": 2.0 * N * C * H * (3 if train else 1) + float(N * C * (18 if train else 6))}
