"""The operators of packed sequences as cases that can be timed one by one: rotary positions, and attention over
packed sequences of different lengths with grouped heads.

A case is one call of one operator, forward only (inference) or forward and backward (training).  Where ``own``
is false, ``run`` computes the operators in their plain form, elementary operations in 32 bits (angles in 64);
where it is true, ``run`` calls the package.  Sizes are generic: proteins and crops have any number of residues,
several of them lie one behind another without padding, and a model that writes sequences asks for one token
at a time against the keys of those before.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotary(name, train, lengths, H, Hk, D, dtype, rotary, layout="half", start=0, factor=1.0, fused=False):
    """``lengths``: those of the packed sequences; ``rotary``: rotated values of the D of a head; ``start``: position of
    each sequence's first token; ``factor``: frequencies of the slow pairs are divided by it; ``fused``: q and k are
    slices of one projection."""
    c = dict(op="rotary", train=train, lengths=lengths, H=H, Hk=Hk, D=D, dtype=dtype, rotary=rotary, layout=layout, start=start,
             factor=factor, fused=fused)
    return c if name is None else dict(c, name=name)


def _attention(name, train, queries, keys, H, Hk, D, dtype, causal=True, slots=0):
    """``queries`` and ``keys``: lengths of the sequences (keys "": the same); ``slots``: the keys of each sequence lie at
    the start of a slot of that many in a cache; 0: packed."""
    c = dict(op="attention", train=train, queries=queries, keys=keys, H=H, Hk=Hk, D=D, dtype=dtype, causal=causal, slots=slots)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one new token each of a few sequences: launch and host time are all there is
        _rotary("rotary tokens, inference", False, "1 1 1 1 1 1 1 1", 32, 8, 128, "bf16", 128, start=1777),
        # packed sequences in training, q and k as they come from one projection; the largest
        _rotary("rotary packed, training", True, "5120 4099 3001 2500 1024 640", 32, 8, 128, "bf16", 128, fused=True),
        # neighbouring pairs of a part of the head, far positions, stretched for a longer context than trained on
        _rotary("rotary odd part far, training", True, "1499 37 2048 1 911", 12, 2, 96, "fp16", 64, "interleaved", start=1000003, factor=8.0),
        # a small encoder in single precision
        _rotary("rotary fp32, training", True, "437 384 300 129", 8, 8, 64, "fp32", 64),
        # a single new token of a short sequence: latency
        _attention("attention one token, inference", False, "1", "130", 32, 8, 128, "bf16"),
        # a batch of sequences, a new token each, against a cache with room to grow
        _attention("attention tokens, inference", False, " ".join(["1"] * 32),
                   "8000 411 5203 1 2777 6100 7391 129 4096 3500 977 7000 64 5555 2222 1800 7777 650 3333 4800 256 6666 1111 7123 2500 33 5900 4444 1025 8191 3800 512",
                   32, 8, 128, "bf16", slots=8192),
        # one long prompt; the largest
        _attention("attention long prompt, inference", False, "16384", "", 16, 4, 128, "bf16"),
        # pieces of prompts against the keys that are there already
        _attention("attention pieces, inference", False, "512 512 300 77", "4096 2500 300 6001", 16, 8, 64, "fp16"),
        # packed sequences in training
        _attention("attention packed, training", True, "2900 1700 1500 1024 600 300 168", "", 16, 4, 128, "bf16"),
        # many short proteins, every residue sees all of its own protein
        _attention("attention short both ways, training", True,
                   "53 211 97 130 64 1 180 240 33 77 256 128 119 201 15 90 143 222 68 31 250 104 177 84 199 46 161 127 129 8 235 112",
                   "", 8, 8, 64, "bf16", causal=False),
        # odd lengths, a head dimension between the usual ones, six heads a group
        _attention("attention odd, training", True, "1499 37 1 640 911", "", 12, 2, 96, "fp16"),
        # a small model in single precision
        _attention("attention fp32, training", True, "437 300 129", "", 4, 4, 64, "fp32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, n, lo, hi, total):
    out = []
    for _ in range(n):
        m = _log_int(rng, lo, hi)
        if out and sum(out) + m > total:
            break
        out.append(min(m, total))
    return out


def _text(lengths):
    return " ".join(map(str, lengths))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    Hk = rng.choice([1, 2, 4, 8])
    H = Hk * rng.choice([1, 2, 3, 4, 6])
    if rng.random() < 0.35:
        D = rng.choice([32, 64, 80, 96, 128, 128, 192])
        n = _log_int(rng, 1, 32)
        rotary = rng.choice([D, D, D // 2, D // 4 * 2])
        return _rotary(None, rng.random() < 0.6, _text(_lengths(rng, n, 1, 4096, 16384)), H, Hk, D, dtype, rotary,
                       rng.choice(["half", "interleaved"]), rng.choice([0, 0, 100, 40000, 5000001]), rng.choice([1.0, 1.0, 4.0, 16.0]), rng.random() < 0.5)
    D = rng.choice([32, 64, 64, 80, 96, 128, 128])
    causal = rng.random() < 0.75
    kind = rng.choice(["train", "train", "prompt", "tokens"])
    if kind == "train":
        lengths = _lengths(rng, _log_int(rng, 1, 32), 1, 3000, 2048 if dtype == "fp32" else 8192)
        return _attention(None, True, _text(lengths), "", H, Hk, D, dtype, causal)
    if kind == "prompt":
        queries = _lengths(rng, _log_int(rng, 1, 8), 16, 6000, 1024 if dtype == "fp32" else 8192)
        keys = [m + (_log_int(rng, 1, 2048) if rng.random() < 0.5 else 0) for m in queries]
        return _attention(None, False, _text(queries), _text(keys), H, Hk, D, dtype, causal)
    keys = _lengths(rng, _log_int(rng, 1, 32), 1, 8000, 1 << 18)
    if dtype == "fp32":
        keys = [min(m, 1000) for m in keys]
    queries = [min(m, 1 if rng.random() < 0.8 else rng.randint(2, 4)) for m in keys]
    return _attention(None, False, _text(queries), _text(keys), H, Hk, D, dtype, causal, 8192 if rng.random() < 0.5 else 0)


def _split(text):
    return [int(w) for w in text.split()]


def _sums(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# Frequencies of the pairs, radians a position: base ** (-2 i / rotary), the slow ones of them (less than one turn in
# ORIGINAL positions) divided by ``factor``, the fast ones (more than four) as they are, with a line between.
BASE, ORIGINAL, SLOW, FAST = 10000.0, 2048, 1.0, 4.0


def _frequencies(rotary, factor):
    f = BASE ** (torch.arange(0, rotary, 2, dtype=torch.float64) / -rotary)
    keep = ((ORIGINAL * f / (2 * math.pi) - SLOW) / (FAST - SLOW)).clamp(0, 1)
    return f / factor * (1 - keep) + f * keep


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt, H, Hk, D, train = DTYPES[case["dtype"]], case["H"], case["Hk"], case["D"], case["train"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=torch.float32, device=dev).normal_(0.0, std, generator=g).to(dt)

    st = dict(case=case)
    if case["op"] == "rotary":
        n = _split(case["lengths"])
        T = sum(n)
        if case["fused"]:  # the columns of q, k and v of one projection
            x = normal(T, H + 2 * Hk, D)
            st["q"], st["k"] = x[:, :H], x[:, H:H + Hk]
        else:
            st["q"], st["k"] = normal(T, H, D), normal(T, Hk, D)
        st["positions"] = torch.cat([torch.arange(m) for m in n]).to(dev) + case["start"]
        st["frequencies"] = _frequencies(case["rotary"], case["factor"]).to(dev)
        if train:
            st["d"] = [normal(T, H, D), normal(T, Hk, D)]
            st["leaves"] = [st[k].requires_grad_() for k in ("q", "k")]
        return st
    nq, nk = _split(case["queries"]), _split(case["keys"] or case["queries"])
    st["nq"], st["nk"] = nq, nk
    # projections of normalised rows, some of them with more to say than others
    st["q"] = normal(sum(nq), H, D, std=1.2)
    if case["slots"]:
        rows, st["starts"] = case["slots"] * len(nk), [case["slots"] * b for b in range(len(nk))]
        st["key_offsets"] = torch.tensor([[a, a + n] for a, n in zip(st["starts"], nk)], dtype=torch.int32, device=dev)
    else:
        rows, st["starts"] = sum(nk), _sums(nk)[:-1]
        st["key_offsets"] = torch.tensor(_sums(nk), dtype=torch.int32, device=dev) if case["keys"] else None
    st["k"], st["v"] = normal(rows, Hk, D, std=1.2), normal(rows, Hk, D)
    st["offsets"] = torch.tensor(_sums(nq), dtype=torch.int32, device=dev)
    if train:
        st["d"] = normal(sum(nq), H, D)
        st["leaves"] = [st[k].requires_grad_() for k in ("q", "k", "v")]
    return st


def _call(st):
    """The package's call of a case."""
    import evoformer_triton_b200 as evo
    case = st["case"]
    if case["op"] == "rotary":
        return list(evo.rotary_embedding(st["q"], st["k"], st["positions"], st["frequencies"], layout=case["layout"]))
    return [evo.packed_attention(st["q"], st["k"], st["v"], st["offsets"], st["key_offsets"], causal=case["causal"])]


def _turn(x, cos, sin, layout):
    """The first 2 n values of every head turned, n pairs by the angles of [T, 1, n]."""
    n = cos.shape[-1]
    x = x.detach().float()
    part = x[..., :2 * n]
    a, b = (part[..., :n], part[..., n:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rotary(st):
    angle = (st["positions"].double()[:, None] * st["frequencies"])[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    layout, dt = st["case"]["layout"], st["q"].dtype
    out = [_turn(st[k], cos, sin, layout).to(dt) for k in ("q", "k")]
    if st["case"]["train"]:
        out += [_turn(d, cos, -sin, layout).to(dt) for d in st["d"]]
    return out


def _plain_attention(st):
    case = st["case"]
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    H, Hk, D, train = case["H"], case["Hk"], case["D"], case["train"]
    G, scale = H // Hk, D ** -0.5
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if train else []
    for nq, nk, i0, j0 in zip(st["nq"], st["nk"], _sums(st["nq"]), st["starts"]):
        hidden = None
        if case["causal"]:
            hidden = torch.arange(nk, device=q.device) > torch.arange(nk - nq, nk, device=q.device)[:, None]
        for h in range(Hk):
            heads = slice(h * G, (h + 1) * G)
            qh = q[i0:i0 + nq, heads].float().transpose(0, 1)  # [G, nq, D]
            kh, vh = k[j0:j0 + nk, h].float(), v[j0:j0 + nk, h].float()
            s = torch.matmul(qh * scale, kh.t())
            if hidden is not None:
                s.masked_fill_(hidden, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()  # (a row without a key: all zeros)
            p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
            o = torch.matmul(p, vh)
            out[i0:i0 + nq, heads] = o.transpose(0, 1).to(q.dtype)
            if not train:
                continue
            d = st["d"][i0:i0 + nq, heads].float().transpose(0, 1)
            grads[2][j0:j0 + nk, h] = torch.matmul(p.transpose(1, 2), d).sum(0).to(q.dtype)
            ds = torch.matmul(d, vh.t()).sub_((d * o).sum(-1, keepdim=True)).mul_(p)
            grads[0][i0:i0 + nq, heads] = (torch.matmul(ds, kh) * scale).transpose(0, 1).to(q.dtype)
            grads[1][j0:j0 + nk, h] = (torch.matmul(ds.transpose(1, 2), qh).sum(0) * scale).to(q.dtype)
    return [out, *grads]


def run(state):
    if own:
        if not state["case"]["train"]:
            with torch.no_grad():
                return _call(state)
        out = _call(state)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, state["leaves"], state["d"])]
    with torch.no_grad():
        return {"rotary": _plain_rotary, "attention": _plain_attention}[state["case"]["op"]](state)


def exact(case, seed):
    """The definitions in 64 bits: a rotation as a product of complex numbers, attention row block by row block with its
    gradients by differentiating it."""
    st = prepare(case, seed)
    if case["op"] == "rotary":
        n, half = case["rotary"] // 2, case["layout"] == "half"
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), st["positions"].double()[:, None, None] * st["frequencies"])

        def rotated(x, by):
            x = x.detach().double()
            pairs = x[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2) if half else x[..., :2 * n].unflatten(-1, (n, 2))
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
            return torch.cat([(y.transpose(-1, -2) if half else y).flatten(-2), x[..., 2 * n:]], -1)

        out = [rotated(st[k], turn) for k in ("q", "k")]
        return out + [rotated(d, turn.conj()) for d in st["d"]] if case["train"] else out

    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    train, G = case["train"], case["H"] // case["Hk"]
    out, grads = torch.zeros_like(q), [torch.zeros_like(t) for t in (q, k, v)] if train else []
    for b, (nq, nk) in enumerate(zip(st["nq"], st["nk"])):
        i0, j0 = sum(st["nq"][:b]), st["starts"][b]
        for h in range(case["H"]):
            kh, vh = (t[j0:j0 + nk, h // G].clone().requires_grad_(train) for t in (k, v))
            for r in range(0, nq, 4096):
                rows = slice(i0 + r, i0 + min(r + 4096, nq))
                qh = q[rows, h].clone().requires_grad_(train)
                w = qh @ kh.t() / math.sqrt(case["D"])
                if case["causal"]:
                    last = torch.arange(r, r + len(qh), device="cuda") + nk - nq
                    seen = torch.arange(nk, device="cuda")[None, :] <= last[:, None]
                    some = (last >= 0)[:, None]
                    w = torch.softmax(torch.where(seen, w, torch.where(some, -math.inf, 0.0)), -1) * some
                else:
                    w = torch.softmax(w, -1)
                o = w @ vh
                out[rows, h] = o.detach()
                if train:
                    for t, d in zip((grads[0][rows, h], grads[1][j0:j0 + nk, h // G], grads[2][j0:j0 + nk, h // G]),
                                    torch.autograd.grad(o, (qh, kh, vh), st["d"][rows, h].double())):
                        t += d
    return [out, *grads]


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    train, H, Hk, D = case["train"], case["H"], case["Hk"], case["D"]
    if case["op"] == "rotary":
        T = sum(_split(case["lengths"]))
        # q and k in and out, and as much again for their gradients; the positions and frequencies
        return {"bytes": T * (H + Hk) * D * size * (4 if train else 2) + 8 * T + 4 * case["rotary"],
                "flops": float(T * (H + Hk) * case["rotary"] * 3 * (2 if train else 1))}
    nq, nk = _split(case["queries"]), _split(case["keys"] or case["queries"])
    pairs = 0  # (query, key) that see one another
    for n, m in zip(nq, nk):
        hid = min(n, m)
        pairs += n * m if not case["causal"] else hid * (hid + 1) // 2 + hid * (m - hid)
    q, kv = sum(nq) * H * D * size, sum(nk) * Hk * D * size
    # q, k, v in, o out; with a gradient d(o) in and d(q), d(k), d(v) out
    return {"bytes": 2 * q + 2 * kv + (2 * q + 2 * kv if train else 0),
            "flops": 2.0 * pairs * H * D * (7 if train else 2)}
