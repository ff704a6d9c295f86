"""Measured cases of the 4-bit (MXFP4) operators and of sampling.

Four operators: quantising a matrix to microscaled 4-bit floating point and reading it back ("quantise"), the product of dense rows with such a
matrix ("product"), the product of sparse histories with one ("scores"), and drawing items from scores ("sample").  With ``own`` false ``run``
computes them with elementary torch operations; with ``own`` true it calls recpack_amd.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32
_contexts = {}


def listed():
    return [
        # one block of user profiles at half precision, odd in both directions: the smallest call, latency
        {"name": "quantise profiles", "op": "quantise", "rows": 97, "cols": 1999, "type": "bf16", "transpose": False},
        # the item-item matrix of a 20 000 item catalogue, as it leaves an EASE fit, for products along its columns
        {"name": "quantise model", "op": "quantise", "rows": 20000, "cols": 20000, "type": "f32", "transpose": True},
        # one dense profile against a 20 000 item model: the weights' bytes bound it
        {"name": "product one profile", "op": "product", "m": 1, "n": 20000, "k": 20000, "type": "bf16"},
        # a small batch of f32 profiles against a small catalogue of odd size
        {"name": "product f32 batch", "op": "product", "m": 97, "n": 1999, "k": 2003, "type": "f32"},
        # a full batch of half precision profiles: 4-bit weights, 16-bit activations
        {"name": "product f16 batch", "op": "product", "m": 2048, "n": 20000, "k": 20000, "type": "f16"},
        # the same with the profiles quantised too: the matrix pipe's 4-bit rate
        {"name": "product 4-bit", "op": "product", "m": 4096, "n": 20000, "k": 20000, "type": "mxfp4"},
        # one user of a 100 000 item catalogue asks
        {"name": "scores one user", "op": "scores", "users": 1, "items": 100000, "history": 50, "type": "f32", "valued": False, "exclude": True},
        # a request batch with decayed interaction weights, small catalogue
        {"name": "scores weighted", "op": "scores", "users": 251, "items": 20000, "history": 100, "type": "bf16", "valued": True, "exclude": False},
        # a chunk of an offline pass over all users of a 50 000 item catalogue
        {"name": "scores batch", "op": "scores", "users": 1024, "items": 50000, "history": 50, "type": "f32", "valued": False, "exclude": True},
        # one user, one item drawn from the whole catalogue's nucleus
        {"name": "sample one row", "op": "sample", "rows": 1, "width": 100000, "draws": 1, "top_k": 0, "type": "f32", "lists": False},
        # slates of 20 from the best 200 of half precision score rows
        {"name": "sample slates", "op": "sample", "rows": 512, "width": 50000, "draws": 20, "top_k": 200, "type": "bf16", "lists": False},
        # slates from top-200 lists of predict, ragged
        {"name": "sample lists", "op": "sample", "rows": 8192, "width": 200, "draws": 10, "top_k": 200, "type": "f32", "lists": True},
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, v | 1 if rng.random() < 0.5 else v))

    op = rng.choice(["quantise", "product", "scores", "sample"])
    if op == "quantise":
        rows = size(1, 20000)
        return {"op": op, "rows": rows, "cols": size(1, 20000), "type": rng.choice(["f32", "f16", "bf16"]), "transpose": rng.random() < 0.5}
    if op == "product":
        kind = rng.choice(["f32", "f16", "bf16", "mxfp4"])
        return {"op": op, "m": size(1, 2048), "n": size(100, 16000), "k": size(32, 16000), "type": kind}
    if op == "scores":
        items, history = size(500, 50000), size(1, 100)
        users = size(1, max(1, min(1024, 2_500_000_000 // (items * history))))  # no more than the largest listed batch
        return {"op": op, "users": users, "items": items, "history": history, "type": rng.choice(["f32", "f16", "bf16"]),
                "valued": rng.random() < 0.5, "exclude": rng.random() < 0.5}
    lists = rng.random() < 0.3
    if lists:
        width = size(10, 1000)
        return {"op": op, "rows": size(1, 8192), "width": width, "draws": size(1, min(20, width)), "top_k": 0, "type": "f32", "lists": True}
    top_k = rng.choice([0, 0, 50, 200, 1000])
    return {"op": op, "rows": size(1, 512), "width": size(1000, 100000), "draws": 1 if top_k == 0 else size(1, 20), "top_k": top_k,
            "type": rng.choice(["f32", "f16", "bf16"]), "lists": False}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------

def _similarities(rows, cols, g):
    """What the rows of an item-item model look like: mostly small, a heavy tail, rows of different size."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x = x * x.abs() * 0.01
    return x * torch.rand(rows, 1, device="cuda", generator=g).add_(0.05)


def _packed(rows, cols, g):
    """A quantised matrix in hand: codes and scale bytes, padding zero.  Scales within a factor of 256, as a model's rows have them."""
    nb = -(-cols // BLOCK)
    codes = torch.randint(0, 256, (rows, nb * BLOCK // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.randint(112, 121, (rows, nb), device="cuda", generator=g, dtype=torch.uint8)
    if cols % 2:
        codes[:, cols // 2] &= 0x0F
    codes[:, (cols + 1) // 2:] = 0
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "quantise":
        s["x"] = _similarities(case["rows"], case["cols"], g).to(DTYPES[case["type"]])
    elif case["op"] == "product":
        a = torch.randn(case["m"], case["k"], device="cuda", generator=g)
        s["a"] = a.to(DTYPES.get(case["type"], torch.float32))
        s["codes"], s["scales"] = _packed(case["n"], case["k"], g)
    elif case["op"] == "scores":
        users, items = case["users"], case["items"]
        # lengths spread around the mean, an empty history now and then; popular items are in many histories
        lengths = (torch.rand(users, device="cuda", generator=g) * 2 * case["history"]).round().long().clamp(max=items)
        if users == 1:
            lengths.fill_(min(case["history"], items))
        indptr = torch.zeros(users + 1, dtype=torch.int32, device="cuda")
        indptr[1:] = lengths.cumsum(0)
        nnz = int(indptr[-1])
        user = torch.repeat_interleave(torch.arange(users, device="cuda"), lengths)
        item = (torch.rand(nnz, device="cuda", generator=g, dtype=torch.float64).pow(3) * items).long().clamp(max=items - 1)
        s["indices"] = torch.sort(user * items + item).values.remainder(items).int()
        s["indptr"] = indptr
        s["weights"] = torch.rand(nnz, device="cuda", generator=g) if case["valued"] else None
        s["codes"], s["scales"] = _packed(items, items, g)
    else:
        rows, width = case["rows"], case["width"]
        x = torch.randn(rows, width, device="cuda", generator=g).mul_(2.0)
        if not case["lists"]:  # some items cannot be recommended
            x.masked_fill_(torch.rand(rows, width, device="cuda", generator=g) < 0.05, -math.inf)
        s["scores"] = x.to(DTYPES[case["type"]])
        s["u"] = torch.rand(rows, case["draws"], device="cuda", generator=g)
        s["temperature"] = torch.rand(rows, device="cuda", generator=g).add_(0.5)
        s["top_p"] = torch.rand(rows, device="cuda", generator=g).mul_(0.3).add_(0.7)
        s["min_p"] = torch.rand(rows, device="cuda", generator=g).mul_(0.002)
        if case["lists"]:
            s["lengths"] = torch.randint(0, width + 1, (rows,), device="cuda", generator=g, dtype=torch.int32)
            s["ids"] = torch.randint(0, 100000, (rows, width), device="cuda", generator=g, dtype=torch.int32)
        else:
            s["lengths"] = s["ids"] = None
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------------------------

def _power(e):
    """2^e for whole -126 <= e <= 127, exact."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _round_4bit(x):
    """A float32 matrix rounded to MXFP4 along its rows: the values that the codes stand for."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 125)  # floor(log2(top)) - 2
    a = v * _power(-e)
    step = 0.5 + 0.5 * (a.abs() >= 2) + (a.abs() >= 4)
    q = (torch.round(a / step) * step).clamp(-6, 6)
    half = torch.div(e, 2, rounding_mode="floor")  # 2^-127 is no normal number: in two steps
    out = q * _power(half) * _power(e - half)
    out = torch.where(torch.isfinite(top), out, math.nan)
    return out.view(rows, -1)[:, :cols]


def _unpack(codes, scales, cols):
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1)
    v = torch.index_select(lut, 0, c.view(-1).int()).view(codes.shape[0], -1, BLOCK)
    return (v * _power(scales.int() - 127).unsqueeze(-1)).view(codes.shape[0], -1)[:, :cols]


def _plain_quantise(s):
    x = s["x"].float()
    return _round_4bit(x.t().contiguous() if s["transpose"] else x)


def _plain_product(s):
    a = s["a"].float()
    if s["type"] == "mxfp4":
        a = _round_4bit(a)
    return (a @ _unpack(s["codes"], s["scales"], s["k"]).t()).to(s["a"].dtype)


def _plain_scores(s):
    users, items = s["users"], s["items"]
    at = s["indices"].long()
    rows = _unpack(s["codes"].index_select(0, at), s["scales"].index_select(0, at), items)
    if s["weights"] is not None:
        rows = rows * s["weights"].unsqueeze(1)
    user = torch.repeat_interleave(torch.arange(users, device="cuda"), s["indptr"].diff().long())
    out = torch.zeros(users, items, device="cuda").index_add_(0, user, rows)
    if s["exclude"]:
        out[user, at] = -math.inf
    return out.to(DTYPES[s["type"]])


def _plain_sample(s):
    x = s["scores"].float()
    rows, width = x.shape
    ok = torch.isfinite(x)
    if s["lengths"] is not None:
        ok &= torch.arange(width, device="cuda") < s["lengths"].unsqueeze(1)
    x, order = torch.sort(x.masked_fill(~ok, -math.inf), dim=1, descending=True, stable=True)
    if s["top_k"]:
        x, order = x[:, :s["top_k"]], order[:, :s["top_k"]]
    # 64 bits from here: cumulative sums next to a border decide whole numbers
    z = (x.double() - x[:, :1].double().nan_to_num(neginf=0.0)) / s["temperature"].double().unsqueeze(1)
    mass = torch.exp(z)
    before = mass.cumsum(1) - mass
    total = mass.sum(1, keepdim=True)
    top_p, min_p = s["top_p"].double().unsqueeze(1), s["min_p"].double().unsqueeze(1)
    keep = ((before < top_p * total) | (top_p >= 1)) & (mass >= min_p) & torch.isfinite(x)
    z = z.masked_fill(~keep, -math.inf)
    picked, probs = [], []
    for d in range(s["draws"]):  # without replacement: each draw is from what the ones before it left
        best = z.amax(1, keepdim=True)
        p = torch.exp(z - best.nan_to_num(neginf=0.0))
        c = p.cumsum(1)
        at = (c <= s["u"][:, d:d + 1].double() * c[:, -1:]).sum(1, keepdim=True).clamp(max=p.shape[1] - 1)
        some = torch.isfinite(best)
        probs.append((p.gather(1, at) / c[:, -1:]).nan_to_num(nan=0.0).float())
        item = order.gather(1, at)
        item = item if s["ids"] is None else s["ids"].gather(1, item).long()
        picked.append(item.masked_fill(~some, -1).int())
        z = z.scatter(1, at, -math.inf)
    picked = torch.cat(picked, 1)
    return picked, torch.cat(probs, 1), (picked >= 0).sum(1).int()


# ---- the framework's calls -----------------------------------------------------------------------------------------------------------

def _context():
    from recpack_amd import get_context

    return get_context(torch.cuda.current_device())


def _own_quantise(s):
    from recpack_amd import ops

    ctx = _context()
    return ops.mxfp4_dequantize(ctx, ops.mxfp4_quantize(ctx, s["x"], transpose=s["transpose"]))


def _own_product(s):
    from recpack_amd import ops

    ctx = _context()
    a = ops.mxfp4_quantize(ctx, s["a"]) if s["type"] == "mxfp4" else s["a"]
    return ops.mxfp4_gemm_nt(ctx, a, ops.MXFP4(s["codes"], s["scales"], s["k"]), dtype=s["a"].dtype)


def _own_scores(s):
    from recpack_amd import ops

    return ops.mxfp4_scores(_context(), s["indptr"], s["indices"], ops.MXFP4(s["codes"], s["scales"], s["items"]), weights=s["weights"],
                            exclude_history=s["exclude"], dtype=DTYPES[s["type"]])


def _own_sample(s):
    from recpack_amd import ops

    return ops.sample(_context(), s["scores"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                      lengths=s["lengths"], ids=s["ids"])


def run(state):
    plain = {"quantise": _plain_quantise, "product": _plain_product, "scores": _plain_scores, "sample": _plain_sample}
    ours = {"quantise": _own_quantise, "product": _own_product, "scores": _own_scores, "sample": _own_sample}
    return (ours if own else plain)[state["op"]](state)


def work(case):
    packed = 0.5 + 1.0 / BLOCK
    if case["op"] == "quantise":  # written as codes, and read back as float32
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["type"]] + 2 * packed + 4), "flops": 2 * n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        size = SIZE.get(case["type"], 4)
        return {"bytes": m * k * size + n * k * packed + m * n * size, "flops": 2 * m * n * k}
    if case["op"] == "scores":
        u, n, h = case["users"], case["items"], case["history"]
        # the expected number of different rows when item = items * uniform^3: each is read once
        q = (np.arange(n + 1) / n) ** (1.0 / 3.0)
        rows = float(np.sum(1.0 - np.exp(u * h * np.log1p(-np.minimum(np.diff(q), 1 - 1e-12)))))
        return {"bytes": rows * n * packed + u * n * SIZE[case["type"]] + u * h * (8 if case["valued"] else 4), "flops": 2 * u * h * n}
    r, w, d = case["rows"], case["width"], case["draws"]
    return {"bytes": r * w * (SIZE[case["type"]] + (4 if case["lists"] else 0)) + r * d * 12, "flops": 8 * r * w}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------

def _values64(codes, scales, cols):
    """What codes and scale bytes stand for, from the format: sign, two exponent bits, one mantissa bit, block scale 2^(byte - 127)."""
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    for side, c in enumerate((codes & 0x0F, codes >> 4)):
        e, m = ((c >> 1) & 3).double(), (c & 1).double()
        size = torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)
        out[:, side::2] = torch.where(c >= 8, -size, size)
    out *= torch.repeat_interleave(torch.exp2(scales.double() - 127), BLOCK, dim=1)
    return out[:, :cols]


def _rounded64(x):
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = (torch.where(torch.exp2(e + 1) <= top, e + 1, e) - 2).clamp(-127, 125)
    a = v / torch.exp2(e)
    size = torch.zeros_like(a)
    # half way between two values goes to the one with the even mantissa
    for border, jump, up in ((.25, .5, 0), (.75, .5, 1), (1.25, .5, 0), (1.75, .5, 1), (2.5, 1., 0), (3.5, 1., 1), (5., 2., 0)):
        size += jump * ((a.abs() >= border) if up else (a.abs() > border))
    return (torch.copysign(size, a) * torch.exp2(e)).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        return _rounded64(s["x"].t().contiguous() if case["transpose"] else s["x"])
    if case["op"] == "product":
        a = _rounded64(s["a"]) if case["type"] == "mxfp4" else s["a"].double()
        return torch.matmul(a, _values64(s["codes"], s["scales"], case["k"]).t())
    if case["op"] == "scores":
        out = torch.zeros(case["users"], case["items"], dtype=torch.float64, device="cuda")
        ends = s["indptr"].tolist()
        for u in range(case["users"]):
            at = s["indices"][ends[u]:ends[u + 1]].long()
            if at.numel():
                v = _values64(s["codes"][at], s["scales"][at], case["items"])
                out[u] = v.sum(0) if s["weights"] is None else (v * s["weights"][ends[u]:ends[u + 1], None].double()).sum(0)
                if case["exclude"]:
                    out[u, at] = -math.inf
        return out
    scores, us = s["scores"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    temperature, top_p, min_p = (s[k].double().cpu().numpy() for k in ("temperature", "top_p", "min_p"))
    lengths = None if s["lengths"] is None else s["lengths"].cpu().numpy()
    ids = None if s["ids"] is None else s["ids"].cpu().numpy()
    items, probs = np.full(us.shape, -1, np.int32), np.zeros(us.shape)
    for r in range(case["rows"]):
        x = scores[r] if lengths is None else scores[r, :lengths[r]]
        there = np.flatnonzero(np.isfinite(x))
        if not there.size:
            continue
        there = there[np.argsort(-x[there], kind="stable")][:case["top_k"] or None]
        logit = (x[there] - x[there[0]]) / temperature[r]
        p = np.exp(logit)
        n = len(p) if top_p[r] >= 1 else 1 + int(np.searchsorted(np.cumsum(p), top_p[r] * p.sum()))
        n = min(n, int((p >= min_p[r]).sum()))
        there, logit = there[:n], logit[:n]
        for d in range(min(case["draws"], n)):
            p = np.exp(logit - logit[0])
            c = np.cumsum(p)
            k = min(int(np.searchsorted(c, us[r, d] * c[-1], side="right")), len(p) - 1)
            items[r, d] = there[k] if ids is None else ids[r, there[k]]
            probs[r, d] = p[k] / c[-1]
            there, logit = np.delete(there, k), np.delete(logit, k)
    return torch.from_numpy(items), torch.from_numpy(probs), torch.from_numpy((items >= 0).sum(1).astype(np.int32))
