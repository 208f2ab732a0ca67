"""Measured cases of the token-sorting and the 4-bit (MXFP4) expert operators.

Four operators, each in the forms a program calls:

* ``dispatch``  - the (token, slot) pairs of a router's choice sorted by expert,
  and the tokens' rows copied into that order;
* ``combine``   - the experts' rows back at their tokens, weighted and summed;
  ``train`` adds the gradients of this and of the dispatch;
* ``quantize``  - bf16/f16/f32 into MXFP4 (with the rounded values, as training
  with 4-bit forward values keeps them);
* ``product``   - MXFP4 x MXFP4, one matrix or an expert stack over sorted rows;
  ``down`` first quantises silu(gate) * up, as the second expert product takes it.

Sizes: hidden 7168, expert width 2048, 256 experts of which a token takes 8,
the batch sizes 1, 64, 4096 and the width 3584 are this repository's own
configurations; the rest are generic.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
# the magnitudes of the eight positive e2m1 codes
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of four requests: a handful of rows, latency counts
        dict(name="dispatch decode", op="dispatch", tokens=4, top_k=8, experts=256, hidden=7168,
             dtype="bf16", held=1.0),
        # a prefill chunk of the same layer: 470 MB of sorted rows
        dict(name="dispatch prefill", op="dispatch", tokens=4096, top_k=8, experts=256,
             hidden=7168, dtype="bf16", held=1.0),
        # a rank that holds half of the experts (the other slots have no expert here), a width
        # whose rows are not 16-byte aligned
        dict(name="dispatch odd f32", op="dispatch", tokens=1021, top_k=6, experts=61,
             hidden=1030, dtype="f32", held=0.5),
        # the way back of a decode batch
        dict(name="combine decode", op="combine", tokens=64, top_k=8, experts=256, hidden=7168,
             dtype="bf16", held=1.0),
        # a training step's combine with all gradients, at the prefill chunk's size
        dict(name="train bf16", op="train", tokens=4096, top_k=8, experts=256, hidden=7168,
             dtype="bf16", held=1.0),
        # the same on a small fp32 model with odd sizes and slots without an expert
        dict(name="train odd f32", op="train", tokens=333, top_k=6, experts=61, hidden=1030,
             dtype="f32", held=0.8),
        # a decode batch's activations before a 4-bit product
        dict(name="quantize decode", op="quantize", rows=64, width=7168, dtype="bf16"),
        # a checkpoint's fp32 expert matrices converted on the GPU: eight of 2048 x 7168
        dict(name="quantize weights f32", op="quantize", rows=16384, width=7168, dtype="f32"),
        # the second half of the experts of a prefill chunk: SwiGLU, quantised, down product
        dict(name="down prefill", op="down", tokens=1024, top_k=8, experts=32, width=2048,
             out=3584, out_dtype="bf16", by_token=False, skew=0.25),
        # a batch of odd size through one matrix (a shared expert), fp32 results
        dict(name="product dense odd", op="product", tokens=77, top_k=1, experts=0, width=7168,
             out=2040, out_dtype="f32", by_token=False, skew=0.0),
        # one token through its eight experts: the weights' bytes are the cost
        dict(name="product one token", op="product", tokens=1, top_k=8, experts=256, width=7168,
             out=2048, out_dtype="bf16", by_token=True, skew=0.0),
        # a prefill chunk through the 32 experts one rank of eight holds, unevenly chosen
        dict(name="product prefill", op="product", tokens=2048, top_k=8, experts=32, width=7168,
             out=2048, out_dtype="bf16", by_token=True, skew=0.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "train", "quantize", "down", "product", "product"])
    if op in ("dispatch", "combine", "train"):
        experts = _log(rng, 8, 384)
        top_k = rng.randint(1, min(8, experts - 1))
        hidden = _log(rng, 64, 7168)
        # no more than the prefill chunk moves, in any type
        tokens = min(_log(rng, 1, 8192), 4096 * 8 * 7168 // (2 * top_k * hidden))
        return dict(op=op, tokens=max(1, tokens), top_k=top_k, experts=experts, hidden=hidden,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    held=rng.choice([1.0, 1.0, 0.5, 0.125]))
    if op == "quantize":
        width = 32 * _log(rng, 1, 224)
        rows = min(_log(rng, 1, 16384), 16384 * 7168 // width)
        return dict(op=op, rows=rows, width=width,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    experts = rng.choice([0, _log(rng, 4, 64), _log(rng, 32, 256)])
    if op == "down":
        experts = max(experts, 8)
    top_k = rng.randint(1, min(8, experts - 1)) if experts else 1
    width = 32 * _log(rng, 8, 224)
    out = _log(rng, 64, 3584)
    tokens = _log(rng, 1, 2048)
    # no more stored weights than 256 experts of 2048 x 3584, nor more work than the largest
    if experts * width * out > 256 * 2048 * 3584:
        experts = max(top_k + 1, 256 * 2048 * 3584 // (width * out))
    return dict(op=op, tokens=tokens, top_k=top_k, experts=experts, width=width, out=out,
                out_dtype="bf16" if op == "down" else rng.choice(["bf16", "bf16", "f32"]),
                by_token=op == "product" and experts > 0 and rng.random() < 0.5,
                skew=rng.choice([0.0, 0.25, 1.0]))


# ------------------------------------------------------------------ inputs

def _choose(gen, tokens, top_k, experts, skew=0.0):
    """A router's choice: top_k different experts a token, uniform or with the popularity of
    rank ** (-1.1 * skew)."""
    score = -torch.log(-torch.log(torch.rand((tokens, experts), generator=gen, device="cuda")
                                  .clamp_(1e-9, 1 - 1e-6)))
    if skew:
        score -= 1.1 * skew * torch.log(torch.arange(1, experts + 1, device="cuda").float())
    return score.topk(top_k, dim=1).indices.to(torch.int32)


def _sorted(ids, experts):
    """order [P], inverse [T, k], offsets [E + 1] of the pairs sorted by expert, stable."""
    flat = ids.reshape(-1).long()
    valid = (flat >= 0) & (flat < experts)
    key = torch.where(valid, flat, experts)
    order = torch.argsort(key, stable=True)
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=order.device)
    kept = valid.sum()
    inverse = torch.where(valid, row, -1)
    order = torch.where(torch.arange(order.numel(), device=order.device) < kept, order, -1)
    bound = torch.arange(experts + 1, device=ids.device)
    offsets = torch.searchsorted(key.sort().values, bound)
    return order.int(), inverse.reshape(ids.shape).int(), offsets.int()


def _codes(gen, rows, width, experts=0):
    """MXFP4 values of unit variance over sqrt(width): random codes, exponents of three octaves."""
    lead = (experts, rows) if experts else (rows,)
    packed = torch.randint(-2 ** 31, 2 ** 31, lead + (width // 8,), generator=gen, device="cuda",
                           dtype=torch.int64).to(torch.int32)
    mid = int(round(127 - math.log2(2.9 * math.sqrt(width))))
    scales = torch.randint(mid - 1, mid + 2, lead + (width // 32,), generator=gen, device="cuda",
                           dtype=torch.int32).to(torch.uint8)
    return packed, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    randn = lambda shape, dt: torch.randn(shape, generator=gen, device="cuda").to(DTYPES[dt])  # noqa: E731
    if c["op"] in ("dispatch", "combine", "train"):
        T, k, E, H = c["tokens"], c["top_k"], c["experts"], c["hidden"]
        ids = _choose(gen, T, k, E)
        if c["held"] < 1.0:  # an expert-parallel rank: slots of experts held elsewhere are -1
            ids = torch.where(torch.rand(ids.shape, generator=gen, device="cuda") < c["held"],
                              ids, -1)
        s["ids"] = ids
        if c["op"] == "dispatch":
            s["x"] = randn((T, H), c["dtype"])
        else:
            s["plan"] = _sorted(ids, E)
            s["ys"] = randn((T * k, H), c["dtype"])
            w = torch.rand((T, k), generator=gen, device="cuda") + 0.05
            s["weights"] = w / w.sum(1, keepdim=True)
        if c["op"] == "train":
            s["dout"] = randn((T, H), c["dtype"])
            s["dxs"] = randn((T * k, H), c["dtype"])
    elif c["op"] == "quantize":
        x = torch.randn((c["rows"], c["width"]), generator=gen, device="cuda")
        # rows of different size, as activations and weights have
        x *= torch.exp(torch.randn((c["rows"], 1), generator=gen, device="cuda"))
        s["x"] = x.to(DTYPES[c["dtype"]])
    else:
        T, k, E = c["tokens"], c["top_k"], c["experts"]
        s["w"] = _codes(gen, c["out"], c["width"], E)
        if c["op"] == "down":  # the first product's result: gate and up side by side
            s["x"] = randn((T * k, 2 * c["width"]), "bf16")
        else:
            s["a"] = _codes(gen, T if (c["by_token"] or not E) else T * k, c["width"])
        if E:
            s["ids"] = _choose(gen, T, k, E, c["skew"])
            s["plan"] = _sorted(s["ids"], E)
            off = s["plan"][2].tolist()
            s["most"] = max(b - a for a, b in zip(off, off[1:]))  # rows of the busiest expert
    return s


# -------------------------------------------------------------- plain form

def _values(packed, scales):
    """The numbers that codes and exponents stand for, fp32."""
    dev = packed.device
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=dev)
    shift = torch.arange(0, 32, 4, device=dev, dtype=torch.int32)
    code = (packed.unsqueeze(-1) >> shift) & 15
    v = lut.index_select(0, code.reshape(-1)).reshape(scales.shape + (32,))
    e = scales.to(torch.int32)
    two = torch.where(e == 0, 0x00400000, e << 23).view(torch.float32)
    return (v * two.unsqueeze(-1)).reshape(packed.shape[:-1] + (packed.shape[-1] * 8,))


def _round(x):
    """(values, packed, scales) of fp32 x: exponent floor(log2(largest)) - 2 per 32 elements, codes
    rounded to nearest even, saturating."""
    b = x.reshape(x.shape[0], -1, 32)
    most = b.abs().amax(-1)
    e = ((most.view(torch.int32) >> 23) - 2).clamp(0, 254)
    down = torch.where(e == 254, 0x00400000, (254 - e) << 23).view(torch.float32)
    up = torch.where(e == 0, 0x00400000, e << 23).view(torch.float32)
    m = (b * down.unsqueeze(-1)).abs()
    code = (m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (
        m > 5)
    lut = torch.tensor(E2M1, device=x.device)
    mag = lut.index_select(0, code.reshape(-1)).reshape(b.shape) * up.unsqueeze(-1)
    neg = torch.signbit(b)
    values = torch.where(neg, -mag, mag).reshape(x.shape)
    nibble = (code + 8 * neg.int()).reshape(x.shape[0], -1, 8)
    shift = torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    packed = (nibble.int() << shift).sum(-1, dtype=torch.int32)
    return values, packed, e.to(torch.uint8)


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "dispatch":
        order, inverse, offsets = _sorted(s["ids"], c["experts"])
        token = torch.div(order.long(), c["top_k"], rounding_mode="floor").clamp(min=0)
        xs = s["x"].float().index_select(0, token) * (order >= 0).unsqueeze(1)
        return {"order": order, "inverse": inverse, "offsets": offsets, "xs": xs.to(s["x"].dtype)}
    if op in ("combine", "train"):
        order, inverse, _ = s["plan"]
        held = inverse >= 0
        row = inverse.long().clamp(min=0)
        w = s["weights"] * held
        ys = s["ys"].float()
        out = (ys[row] * w.unsqueeze(-1)).sum(1).to(s["ys"].dtype)
        if op == "combine":
            return {"out": out}
        dout = s["dout"].float()
        pair = order.long().clamp(min=0)
        token = torch.div(pair, c["top_k"], rounding_mode="floor")
        kept = (order >= 0).unsqueeze(1)
        dys = dout[token] * w.reshape(-1)[pair].unsqueeze(1) * kept
        dw = (dout.unsqueeze(1) * ys[row]).sum(-1) * held
        dx = (s["dxs"].float()[row] * held.unsqueeze(-1)).sum(1)
        return {"out": out, "dys": dys.to(s["ys"].dtype), "dw": dw, "dx": dx.to(s["dxs"].dtype)}
    if op == "quantize":
        values, packed, scales = _round(s["x"].float())
        return {"values": values.to(s["x"].dtype), "packed": packed, "scales": scales}
    if op == "down":
        gate, up = s["x"].float().chunk(2, dim=1)
        a, _, _ = _round(gate / (1.0 + torch.exp(-gate)) * up)
    else:
        a = _values(*s["a"])
    dt = DTYPES[c["out_dtype"]]
    packed, scales = s["w"]
    if not c["experts"]:
        return (a @ _values(packed, scales).t()).to(dt)
    order, _, offsets = s["plan"]
    rows = order.numel()
    if c["by_token"]:
        a = a[torch.div(order.long(), c["top_k"], rounding_mode="floor")]
    # the experts that have rows, each one's rows padded to the busiest expert's: one batched
    # product
    hit = torch.nonzero(offsets[1:] > offsets[:-1]).squeeze(1)
    at = offsets[hit].long().unsqueeze(1) + torch.arange(s["most"], device=a.device)
    inside = at < offsets[hit + 1].long().unsqueeze(1)
    w = _values(packed[hit], scales[hit])
    each = torch.bmm(a[at.clamp(max=rows - 1)], w.transpose(1, 2))
    out = torch.empty((rows, c["out"]), dtype=dt, device=a.device)
    out[at[inside]] = each[inside].to(dt)
    return out


# ---------------------------------------------------------- the framework's

def _moe():
    import sys
    if "minirun-app_b200" not in sys.path:
        sys.path.insert(1, "minirun-app_b200")
    import minirun_moe
    return minirun_moe


def _handles(s):
    """The objects a program keeps beside its tensors: weights and sorted tokens."""
    M = s["M"] = _moe()
    c = s["case"]
    if "plan" in s:
        s["sorted"] = M.SortedTokens(*s["plan"], c["experts"])
    if "w" in s:
        s["weight"] = M.MXFP4Weights(*s["w"])
    if "a" in s:
        s["act"] = M.MXFP4Weights(*s["a"])
    return M


def _own(s):
    M = s.get("M") or _handles(s)
    c = s["case"]
    op = c["op"]
    if op == "dispatch":
        p = M.moe_sort(s["ids"], c["experts"])
        xs = M.moe_dispatch(s["x"], p)
        return {"order": p.order, "inverse": p.inverse, "offsets": p.offsets, "xs": xs}
    if op == "combine":
        return {"out": M.moe_combine(s["ys"], s["weights"], s["sorted"])}
    if op == "train":
        p = s["sorted"]
        out = M.moe_combine(s["ys"], s["weights"], p)
        dys, dw = M.moe_combine_backward(s["dout"], s["ys"], s["weights"], p)
        dx = M.moe_dispatch_backward(s["dxs"], p)
        return {"out": out, "dys": dys, "dw": dw, "dx": dx}
    if op == "quantize":
        q, values = M.mxfp4_quantize(s["x"], values=True)
        return {"values": values, "packed": q.packed, "scales": q.scales}
    dt = DTYPES[c["out_dtype"]]
    if op == "down":
        h = M.mxfp4_quantize_swiglu(s["x"])
        return M.mxfp4_grouped_mm(h, s["weight"], s["sorted"], out_dtype=dt)
    if not c["experts"]:
        return M.mxfp4_scaled_mm(s["act"], s["weight"], out_dtype=dt)
    return M.mxfp4_grouped_mm(s["act"], s["weight"], s["sorted"], by_token=c["by_token"],
                              out_dtype=dt)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c = case
    op = c["op"]
    if op in ("dispatch", "combine", "train"):
        T, P, H, b = c["tokens"], c["tokens"] * c["top_k"], c["hidden"], SIZE[c["dtype"]]
        held = P * c["held"]
        if op == "dispatch":
            # ids in; order, inverse, offsets out; rows in once and out sorted
            return {"bytes": 12 * P + 4 * c["experts"] + (T + P) * H * b, "flops": 0}
        forward = 8 * P + (held + T) * H * b
        if op == "combine":
            return {"bytes": forward, "flops": 2 * held * H}
        # ys, dout and dxs in once; out, dys, dw and dx out
        return {"bytes": 12 * P + (2 * held + P + 3 * T) * H * b, "flops": 6 * held * H}
    if op == "quantize":
        n, b = c["rows"] * c["width"], SIZE[c["dtype"]]
        return {"bytes": n * (2 * b + 17 / 32), "flops": 3 * n}
    P = c["tokens"] * c["top_k"]
    E = c["experts"]
    mats = E * (1 - (1 - c["top_k"] / E) ** c["tokens"]) if E else 1
    rows = c["tokens"] if c["by_token"] or not E else P
    fp4 = 17 / 32  # bytes of an element with its share of the exponent
    act = rows * c["width"] * (4 if op == "down" else fp4)  # down: gate and up in bf16
    return {"bytes": mats * c["out"] * c["width"] * fp4 + act +
            P * c["out"] * SIZE[c["out_dtype"]], "flops": 2 * P * c["width"] * c["out"]}


# ------------------------------------------------------------- in 64 bits

def _e2m1_64(packed, scales):
    byte = packed.contiguous().view(torch.uint8)
    code = torch.stack((byte % 16, byte // 16), dim=-1).flatten(-2).long()
    sign = 1.0 - 2.0 * (code // 8).double()
    ex, man = (code % 8) // 2, (code % 2).double()
    mag = torch.where(ex == 0, man * 0.5, (1 + man / 2) * torch.exp2((ex - 1).double()))
    scale = torch.ldexp(torch.ones((), dtype=torch.float64, device=packed.device),
                        scales.int() - 127)
    return sign * mag * scale.repeat_interleave(32, dim=-1)


def _round_64(x):
    """x, fp64 [rows, n], at the nearest MXFP4 number of its block."""
    b = x.reshape(-1, 32)
    _, top = torch.frexp(b.abs().amax(1))  # largest = m * 2**top, 0.5 <= m < 1
    e = (top.long() - 1 - 2).clamp(-127, 127)
    e = torch.where(b.abs().amax(1) == 0, torch.full_like(e, -127), e).unsqueeze(1)
    u = torch.ldexp(b, -e).abs().clamp(max=6.0)
    # spacing of the grid at u: 1/2 below 2, 1 below 4, 2 above
    step = torch.where(u < 2, 0.5, torch.where(u < 4, 1.0, 2.0)).double()
    return (torch.ldexp(torch.round(u / step) * step, e) * torch.sign(b)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "dispatch":
        ids = s["ids"].reshape(-1).tolist()
        E = case["experts"]
        order = [p for _, p in sorted((e, p) for p, e in enumerate(ids) if 0 <= e < E)]
        xs = torch.zeros((len(ids), case["hidden"]), dtype=torch.float64, device="cuda")
        if order:
            xs[:len(order)] = s["x"].double()[torch.tensor(order, device="cuda") //
                                              case["top_k"]]
        return {"order": None, "inverse": None, "offsets": None, "xs": xs}
    if op in ("combine", "train"):
        T, k = case["tokens"], case["top_k"]
        inv = s["plan"][1].long()
        H = case["hidden"]
        out = torch.zeros((T, H), dtype=torch.float64, device="cuda")
        dx, dw = torch.zeros_like(out), torch.zeros((T, k), dtype=torch.float64, device="cuda")
        dys = torch.zeros((T * k, H), dtype=torch.float64, device="cuda") if op == "train" else None
        for j in range(k):
            t = torch.nonzero(inv[:, j] >= 0).reshape(-1)
            r = inv[t, j]
            w = s["weights"][t, j].double().unsqueeze(1)
            y = s["ys"][r].double()
            out[t] += w * y
            if op == "train":
                g = s["dout"][t].double()
                dys[r] = w * g
                dw[t, j] = torch.einsum("th,th->t", g, y)
                dx[t] += s["dxs"][r].double()
        return {"out": out} if op == "combine" else {"out": out, "dys": dys, "dw": dw, "dx": dx}
    if op == "quantize":
        return {"values": _round_64(s["x"].double()), "packed": None, "scales": None}
    # products: one expert after another
    if op == "down":
        n = case["width"]
        x = s["x"].double()
        a = _round_64(x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:])
    else:
        a = _e2m1_64(*s["a"])
    packed, scales = s["w"]
    if not case["experts"]:
        return a @ _e2m1_64(packed, scales).T
    order, _, offsets = s["plan"]
    out = torch.zeros((order.numel(), case["out"]), dtype=torch.float64, device="cuda")
    off = offsets.tolist()
    for e in range(case["experts"]):
        if off[e] < off[e + 1]:
            r = torch.arange(off[e], off[e + 1], device="cuda")
            rows = a[order[r].long() // case["top_k"]] if case["by_token"] else a[r]
            out[r] = rows @ _e2m1_64(packed[e], scales[e]).T
    return out
