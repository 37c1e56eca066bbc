"""Operators of the low-precision training path, each as a plain form in elementary torch operations and as a
call of the framework: the root-mean-square norm that adds the residual (and may hand over 8-bit codes), the
product of 8-bit operands with a scale for each block of 128, the linear layer built from it (forward and both
gradients), and an AdamW step over many tensors with moments in 32 or 8 bits.

Definitions that both forms share:

  norm      h = x + residual, rounded to the stream's type (h is an output, and the norm is of what is stored);
            y = h * rsqrt(mean(h^2) + eps) * w.  As 8-bit codes: with t = h * w and a = max |t| over a group of
            128 columns (at least 2^-96), codes = e4m3(t * (448 (1 / a))) and scale = a (1 / 448) * rsqrt(mean(h^2)
            + eps), so the codes do not depend on the row's statistic.
  quantise  a = max(max |x| over the block, 2^-96), scale = a (1 / 448), codes = e4m3(x * (448 (1 / a))), each
            step rounded to 32 bits; blocks of 1 x 128 (activations, gradients) or 128 x 128 (weights).
  product   out[m, n] = sum_k a[m, k] * sa[m, k // 128] * b[n, k] * sb[., k // 128] (+ bias[n]).
  AdamW     m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
            p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps).
            8-bit moments: blocks of 256 elements; m and sqrt(v) as e4m3 of u * (448 (1 / a)), a = max |u| over the
            block (at least 2^-96), with scale a (1 / 448); the code of sqrt(v) is at least 2^-9, the type's
            smallest value, where v > 0.
"""
import math
import random

import torch

own = False

F8 = torch.float8_e4m3fn
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
TINY = 2.0 ** -96
SHARE = 1.0 / 448.0  # of a block's largest value: the scale, at which that value gets the type's largest code
EPS = 1e-6
LR, B1, B2, ADAM_EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 1e-2

# The parameters of the 3-layer GraphSAGE (100 -> 256 -> 256 -> 47) that the framework trains: per layer two
# weights and a bias, and two vectors for each norm between the layers.
SAGE = [(256, 100), (256, 100), (256,), (256,), (256,), (256, 256), (256, 256), (256,), (256,), (256,), (47, 256),
        (47, 256), (47,)]


def listed():
    return [
        # one token of a served model: a call's fixed costs
        {"name": "norm one token fp8", "kind": "norm", "rows": 1, "f": 4096, "dtype": "bf16", "residual": True, "out": "fp8"},
        # training, wide hidden rows, a width that is no multiple of 128: output, stream and all gradients
        {"name": "norm train wide odd", "kind": "norm_train", "rows": 8191, "f": 5000, "dtype": "bf16", "residual": True},
        # one of four parts of the 2.45 M-node graph at the hidden width, handed to an 8-bit product
        {"name": "norm part fp8", "kind": "norm", "rows": 612500, "f": 256, "dtype": "bf16", "residual": True, "out": "fp8"},
        # a few tokens against a square weight: the weight's bytes count
        {"name": "product few tokens", "kind": "product", "m": 8, "n": 4096, "k": 4096, "b": "block", "out": "bf16", "bias": False},
        # the first layer's transform of one of four parts (100 features: less than one block)
        {"name": "product part K=100", "kind": "product", "m": 612500, "n": 256, "k": 100, "b": "block", "out": "bf16", "bias": True},
        # a large dense product, bound by the tensor cores
        {"name": "product square", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "b": "block", "out": "bf16", "bias": False},
        # the weight gradient of a hidden layer: a long sum into a small matrix, row scales on both sides
        {"name": "product weight gradient", "kind": "product", "m": 256, "n": 256, "k": 612500, "b": "row", "out": "fp32", "bias": False},
        # the output layer of the small configurations, forward and backward, 32-bit tensors around it
        {"name": "linear train small odd", "kind": "linear", "m": 5003, "k": 100, "n": 47, "dtype": "fp32", "bias": True},
        # a feed-forward layer, forward and backward
        {"name": "linear train large", "kind": "linear", "m": 16384, "k": 2048, "n": 8192, "dtype": "bf16", "bias": False},
        # the framework's own small model: many small tensors, latency
        {"name": "adamw model 32", "kind": "adamw", "sizes": "sage", "total": 0, "dtype": "fp32", "bits": 32},
        # a learnable embedding of the 2.45 M nodes beside the model
        {"name": "adamw embedding 8", "kind": "adamw", "sizes": "sage", "total": 245000000, "dtype": "fp32", "bits": 8},
        # a ragged mixture of many 16-bit tensors with 32-bit moments
        {"name": "adamw ragged bf16 32", "kind": "adamw", "sizes": "ragged", "total": 90000001, "dtype": "bf16", "bits": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "product", "product", "linear", "adamw"])
    if kind in ("norm", "norm_train"):
        f = _log(rng, 40, 8192)
        rows = _log(rng, 1, max(2, min(1000000, 150000000 // f)))
        c = {"kind": kind, "rows": rows, "f": f, "dtype": rng.choice(["fp32", "bf16", "fp16"]), "residual": rng.random() < 0.7}
        if kind == "norm":
            c["out"] = rng.choice(["fp8", "same"])
        return c
    if kind == "product":
        if rng.random() < 0.3:  # long sums into small matrices
            m, n, k = _log(rng, 16, 512), _log(rng, 16, 512), _log(rng, 4000, 600000)
            return {"kind": kind, "m": m, "n": n, "k": k, "b": "row", "out": "fp32", "bias": False}
        n, k = _log(rng, 16, 8192), _log(rng, 32, 8192)
        m = _log(rng, 1, max(2, min(600000, 2 ** 38 // (n * k), 150000000 // max(n, k))))
        return {"kind": kind, "m": m, "n": n, "k": k, "b": rng.choice(["block", "block", "row"]),
                "out": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5}
    if kind == "linear":
        n, k = _log(rng, 16, 4096), _log(rng, 16, 4096)
        m = _log(rng, 16, max(32, min(200000, 2 ** 36 // (n * k), 60000000 // max(n, k))))
        return {"kind": kind, "m": m, "k": k, "n": n, "dtype": rng.choice(["fp32", "bf16", "fp16"]), "bias": rng.random() < 0.5}
    return {"kind": kind, "sizes": rng.choice(["sage", "ragged"]), "total": _log(rng, 1000, 100000000),
            "dtype": rng.choice(["fp32", "fp32", "bf16"]), "bits": rng.choice([32, 8])}


# ---------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, rows, f, dtype):
    """Rows of unequal size with a few large columns, as hidden activations have them."""
    x = torch.randn(rows, f, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.exp(0.5 * torch.randn(1, f, device="cuda", generator=g))
    return x.to(dtype)


def _groups(x, width):
    """(rows, cols) -> (rows, groups, width), the last group filled up with zeros."""
    short = -x.size(1) % width
    if short:
        x = torch.nn.functional.pad(x, (0, short))
    return x.view(x.size(0), -1, width)


def _spread(scales, block, rows, cols):
    """The scale of each element: scales (rows or row blocks, column groups) -> (rows, cols)."""
    if block:
        scales = scales.repeat_interleave(128, 0)[:rows]
    return scales.repeat_interleave(128, 1)[:, :cols]


def _factor(a):
    return torch.reciprocal(a) * 448.0


def _quantise(x, block):
    """codes (as 32-bit values of the 8-bit type) and scales of x (rows, cols): the definition, in 32 bits."""
    x = x.float()
    a = _groups(x.abs(), 128).amax(2)
    if block:
        a = _groups(a.t(), 128).amax(2).t()
    a = a.clamp_min(TINY)
    return (x * _spread(_factor(a), block, *x.shape)).to(F8), a * SHARE


def _operand(x, block):
    """Codes whose rows start on 16 bytes, and scales that lie column by column: as quantize_fp8 lays them."""
    codes, scales = _quantise(x, block)
    rows, cols = codes.shape
    wide = torch.zeros(rows, -(-cols // 16) * 16, device="cuda", dtype=torch.uint8)
    wide[:, :cols] = codes.view(torch.uint8)
    return wide.view(F8)[:, :cols], scales.t().contiguous().t()


def _shapes(case):
    """The tensors of an optimiser case: the model's, and beside them one embedding or a ragged lot."""
    shapes = list(SAGE) if case["sizes"] == "sage" else []
    left = case["total"]
    if case["sizes"] == "sage":
        return shapes + ([(left,)] if left else [])
    i = 0
    while left > 0:  # from small vectors to matrices that hold a tenth of the whole
        n = min(left, max(1, (1, 7, 64, 1001, 4096, 65537, left // 10)[i % 7]))
        if len(shapes) >= 60:
            n = left
        shapes.append((n,))
        left -= n
        i += 1
    return shapes


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind in ("norm", "norm_train"):
        dt = DT[case["dtype"]]
        rows, f = case["rows"], case["f"]
        s["x"] = _activations(g, rows, f, dt)
        s["residual"] = _activations(g, rows, f, dt) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(f, device="cuda", generator=g)).to(dt)
        if kind == "norm_train":
            s["gy"] = torch.randn(rows, f, device="cuda", generator=g).to(dt)
            s["gh"] = torch.randn(rows, f, device="cuda", generator=g).to(dt) if case["residual"] else None
            for k in ("x", "residual", "w"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    elif kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["sa"] = _operand(_activations(g, m, k, torch.float32), False)
        w = torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)
        s["b"], s["sb"] = _operand(w, case["b"] == "block")
        s["bias"] = torch.randn(n, device="cuda", generator=g) if case["bias"] else None
    elif kind == "linear":
        dt = DT[case["dtype"]]
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _activations(g, m, k, dt).requires_grad_(True)
        s["w"] = (torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)).to(dt).requires_grad_(True)
        s["bias"] = (0.1 * torch.randn(n, device="cuda", generator=g)).to(dt).requires_grad_(True) if case["bias"] else None
        s["gy"] = torch.randn(m, n, device="cuda", generator=g).to(dt)
    else:
        dt = DT[case["dtype"]]
        # tensors that lie one behind the other in a buffer for each kind, each on a boundary of 64 elements
        shapes = _shapes(case)
        sizes = [math.prod(shape) for shape in shapes]
        places = [0]
        for n in sizes:
            places.append(places[-1] + -(-n // 64) * 64)
        eight = case["bits"] == 8
        flat = {"p": torch.zeros(places[-1], device="cuda", dtype=dt), "g": torch.zeros(places[-1], device="cuda", dtype=dt),
                "m": torch.zeros(places[-1], device="cuda", dtype=F8 if eight else torch.float32),
                "v": torch.zeros(places[-1], device="cuda", dtype=F8 if eight else torch.float32)}
        s["flat"] = flat
        for k, t in flat.items():
            s[k] = [t[at:at + n].view(shape) for at, n, shape in zip(places, sizes, shapes)]
        blocks = [-(-n // 256) for n in sizes]
        s["scales"] = []
        if eight:
            flat["scales"] = torch.zeros(sum(blocks), 2, device="cuda")
            s["scales"] = list(flat["scales"].split(blocks))
        for i, shape in enumerate(shapes):
            size = math.exp(random.Random(seed * 1000 + i).gauss(0, 1))  # gradients differ in size from tensor to tensor
            s["p"][i].copy_(0.05 * torch.randn(shape, device="cuda", generator=g))
            s["g"][i].copy_(1e-3 * size * torch.randn(shape, device="cuda", generator=g))
            m = 3e-4 * size * torch.randn(shape, device="cuda", generator=g)
            v = (1e-3 * size * torch.randn(shape, device="cuda", generator=g)).square_()
            if eight:
                m, v, scales = _pack(m, v)
                s["scales"][i].copy_(scales)
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)
        s["step"] = 100
    return s


# ---------------------------------------------------------------------------------------------- plain forms

def _norm_plain(x, residual, w):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    return h, hf, rstd


def _norm_run(s, fp8):
    x, residual, w = s["x"], s["residual"], s["w"]
    h, hf, rstd = _norm_plain(x, residual, w)
    extra = [] if residual is None else [h]
    if not fp8:
        return [(hf * rstd * w.float()).to(x.dtype)] + extra
    t = hf * w.float()
    a = _groups(t.abs(), 128).amax(2).clamp_min(TINY)
    codes = (t * _spread(_factor(a), False, *t.shape)).to(F8)
    return [codes, (a * SHARE) * rstd] + extra


def _norm_train_run(s):
    with torch.no_grad():
        x, residual, w, gy = s["x"], s["residual"], s["w"], s["gy"].float()
        h, hf, rstd = _norm_plain(x, residual, w)
        hat = hf * rstd
        y = (hat * w.float()).to(x.dtype)
        wg = gy * w.float()
        gx = rstd * (wg - hat * (wg * hat).mean(1, keepdim=True))
        if s["gh"] is not None:
            gx = gx + s["gh"].float()
        gw = (gy * hat).sum(0).to(w.dtype)
        gx = gx.to(x.dtype)
        return [y, gx, gw] + ([] if residual is None else [h, gx.clone()])


def _product_plain(a, sa, b, sb, block):
    a = a.float() * _spread(sa, False, *a.shape)
    b = b.float() * _spread(sb, block, *b.shape)
    return a @ b.t()


def _product_run(s):
    c = s["case"]
    out = _product_plain(s["a"], s["sa"], s["b"], s["sb"], c["b"] == "block")
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(DT[c["out"]])


def _linear_run(s):
    with torch.no_grad():
        x, w, gy = s["x"], s["w"], s["gy"]
        xq, wq, gq = _quantise(x, False), _quantise(w, True), _quantise(gy, False)
        y = _product_plain(*xq, *wq, True)
        if s["bias"] is not None:
            y = y + s["bias"].float()
        wt = _quantise(w.t(), True)
        gx = _product_plain(*gq, *wt, True)
        gw = _product_plain(*_quantise(gy.t(), False), *_quantise(x.t(), False), False)
        out = [y.to(x.dtype), gx.to(x.dtype), gw.to(w.dtype)]
        if s["bias"] is not None:
            out.append(gy.float().sum(0).to(x.dtype))
        return out


def _blocks(t, size=256):
    t = t.reshape(-1)
    short = -t.numel() % size
    return (torch.nn.functional.pad(t, (0, short)) if short else t).view(-1, size)


def _pack(m, v):
    """32-bit moments -> codes of m, codes of sqrt(v), scales (blocks, 2)."""
    shape, n = m.shape, m.numel()
    mb, rb = _blocks(m), _blocks(torch.sqrt(v))
    am = mb.abs().amax(1, keepdim=True).clamp_min(TINY)
    ar = rb.amax(1, keepdim=True).clamp_min(TINY)
    mc = (mb * (_factor(am))).to(F8).view(-1)[:n].view(shape)
    rc = rb * (_factor(ar))
    rc = torch.where(rb > 0, rc.clamp_min(2.0 ** -9), rc).to(F8).view(-1)[:n].view(shape)
    return mc, rc, torch.cat([am * SHARE, ar * SHARE], 1)


def _unpack(mc, rc, scales):
    n = mc.numel()
    m = (_blocks(mc.float()) * scales[:, :1]).view(-1)[:n].view(mc.shape)
    r = (_blocks(rc.float()) * scales[:, 1:]).view(-1)[:n].view(mc.shape)
    return m, r * r


def _adamw_plain(s):
    s["step"] += 1
    c1, c2 = 1.0 - B1 ** s["step"], 1.0 - B2 ** s["step"]
    for i, (p, g) in enumerate(zip(s["p"], s["g"])):
        g = g.float()
        if s["scales"]:
            m, v = _unpack(s["m"][i], s["v"][i], s["scales"][i])
        else:
            m, v = s["m"][i], s["v"][i]
        m = m * B1 + g * (1.0 - B1)
        v = v * B2 + (g * g) * (1.0 - B2)
        new = p.float() * (1.0 - LR * WD) - (LR / c1) * m / (torch.sqrt(v) / math.sqrt(c2) + ADAM_EPS)
        p.copy_(new)
        if s["scales"]:
            mc, rc, scales = _pack(m, v)
            s["m"][i].copy_(mc)
            s["v"][i].copy_(rc)
            s["scales"][i].copy_(scales)
        else:
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)


def _updated(s):
    """The buffers that hold every parameter and moment."""
    return {k: t for k, t in s["flat"].items() if k != "g"}


# ---------------------------------------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        if kind == "norm":
            return _norm_run(s, c["out"] == "fp8")
        if kind == "norm_train":
            return _norm_train_run(s)
        if kind == "product":
            return _product_run(s)
        if kind == "linear":
            return _linear_run(s)
        _adamw_plain(s)
        return _updated(s)
    from gnn_benchmark_b200 import dense, norm, optim

    if kind == "norm":
        call = norm.rms_norm_fp8 if c["out"] == "fp8" else norm.rms_norm
        r = call(s["x"], s["w"], residual=s["residual"], eps=EPS)
        return list(r) if isinstance(r, tuple) else [r]
    if kind == "norm_train":
        leaves = [t for t in (s["x"], s["w"], s["residual"]) if t is not None]
        r = norm.rms_norm(s["x"], s["w"], residual=s["residual"], eps=EPS)
        if s["residual"] is None:
            gx, gw = torch.autograd.grad(r, leaves, s["gy"])
            return [r, gx, gw]
        gx, gw, gr = torch.autograd.grad(r, leaves, (s["gy"], s["gh"]))
        return [r[0], gx, gw, r[1], gr]
    if kind == "product":
        return dense.matmul_fp8(s["a"], s["sa"], s["b"], s["sb"], bias=s["bias"], out_dtype=DT[c["out"]])
    if kind == "linear":
        y = dense.linear_fp8(s["x"], s["w"], s["bias"])
        leaves = [t for t in (s["x"], s["w"], s["bias"]) if t is not None]
        return [y] + list(torch.autograd.grad(y, leaves, s["gy"]))
    s["step"] += 1
    optim.adamw_step(s["p"], s["g"], s["m"], s["v"], step=s["step"], lr=LR, betas=(B1, B2), eps=ADAM_EPS,
                     weight_decay=WD, scales=s["scales"] or None)
    return _updated(s)


# ---------------------------------------------------------------------------------------------- cost and truth

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, e = case["rows"] * case["f"], SIZE[case["dtype"]]
        back = 1 if case["out"] == "fp8" else e
        b = n * (e + back + (2 * e if case["residual"] else 0)) + case["f"] * e
        if case["out"] == "fp8":
            b += 4 * case["rows"] * -(-case["f"] // 128)
        return {"bytes": b, "flops": 6 * n}
    if kind == "norm_train":
        # forward: x (and residual) in, y (and h) out; backward: h and the gradients of the outputs in, the stream's out
        n, e = case["rows"] * case["f"], SIZE[case["dtype"]]
        return {"bytes": n * e * (8 if case["residual"] else 5) + 2 * case["f"] * e, "flops": 16 * n}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // 128)
        b = (m + n) * k + m * n * SIZE[case["out"]] + 4 * kb * (m + (n if case["b"] == "row" else -(-n // 128)))
        return {"bytes": b + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "linear":
        m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
        return {"bytes": e * (2 * m * k + 2 * n * k + 2 * m * n), "flops": 6 * m * n * k}
    n = sum(math.prod(shape) for shape in _shapes(case))
    e = SIZE[case["dtype"]]
    return {"bytes": n * (3 * e + (4 if case["bits"] == 8 else 16)) + (-(-n // 256) * 16 if case["bits"] == 8 else 0), "flops": 14 * n}


def _exact_product(a, sa, b, sb, block):
    """Block by block of the sum, in 64 bits."""
    out = torch.zeros(a.size(0), b.size(0), device="cuda", dtype=torch.float64)
    for j in range(sa.size(1)):
        at = slice(128 * j, 128 * (j + 1))
        col = sb[:, j].double()
        if block:
            col = col[torch.arange(b.size(0), device="cuda") // 128]
        part = a[:, at].double() @ b[:, at].double().t()
        out += part * sa[:, j].double()[:, None] * col[None, :]
    return out


def _exact_codes(x, block):
    """The definition's codes and scales: a rounding in 32 bits is part of what the format is."""
    x = x.float().contiguous()
    rows, cols = x.shape
    high = 128 if block else 1
    top = torch.zeros(-(-rows // high), -(-cols // 128), device="cuda")
    codes = torch.empty(rows, cols, device="cuda", dtype=F8)
    for j in range(top.size(1)):
        part = x[:, 128 * j:128 * (j + 1)]
        a = part.abs().max(1).values
        if block:
            full = torch.zeros(top.size(0) * 128, device="cuda")
            full[:rows] = a
            a = full.view(-1, 128).max(1).values
        a = torch.maximum(a, torch.tensor(TINY, device="cuda"))
        top[:, j] = a
        factor = torch.ones_like(a) / a * 448.0
        if block:
            factor = factor[torch.arange(rows, device="cuda") // 128]
        codes[:, 128 * j:128 * (j + 1)] = (part * factor[:, None]).to(F8)
    return codes, top * torch.tensor(1.0 / 448.0, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind in ("norm", "norm_train"):
            x, w = s["x"], s["w"].double()
            h = x if s["residual"] is None else (x.double() + s["residual"].double()).to(x.dtype)
            hd = h.double()
            rms = torch.sqrt(torch.linalg.vector_norm(hd, dim=1, keepdim=True) ** 2 / hd.size(1) + EPS)
            stream = [] if s["residual"] is None else [h.double()]
            if kind == "norm" and case["out"] == "fp8":
                t = hd * w
                codes, scales = torch.empty_like(t), []
                for j in range(-(-t.size(1) // 128)):
                    part = t[:, 128 * j:128 * (j + 1)]
                    a = part.abs().max(1, keepdim=True).values.clamp_min(TINY)
                    codes[:, 128 * j:128 * (j + 1)] = (part / a * 448.0).to(F8).double()
                    scales.append(a / 448.0 / rms)
                return [codes, torch.cat(scales, 1)] + stream
            if kind == "norm":
                return [hd / rms * w] + stream
            gy = s["gy"].double()
            # d/dh of h_i w_i / rms: the second term is through rms, d rms / dh_i = h_i / (F rms)
            gx = gy * w / rms - hd * ((gy * w * hd).sum(1, keepdim=True) / (hd.size(1) * rms ** 3))
            if s["gh"] is not None:
                gx = gx + s["gh"].double()
            out = [hd / rms * w, gx, (gy * hd / rms).sum(0)]
            return out + ([] if s["residual"] is None else stream + [gx.clone()])
        if kind == "product":
            out = _exact_product(s["a"], s["sa"], s["b"], s["sb"], case["b"] == "block")
            return out if s["bias"] is None else out + s["bias"].double()
        if kind == "linear":
            x, w, gy = s["x"], s["w"], s["gy"]
            y = _exact_product(*_exact_codes(x, False), *_exact_codes(w, True), True)
            if s["bias"] is not None:
                y = y + s["bias"].double()
            gx = _exact_product(*_exact_codes(gy, False), *_exact_codes(w.t(), True), True)
            gw = _exact_product(*_exact_codes(gy.t(), False), *_exact_codes(x.t(), False), False)
            return [y, gx, gw] + ([] if s["bias"] is None else [gy.double().sum(0)])
        t = s["step"] + 1
        out = {k: torch.zeros(v.shape, device="cuda", dtype=torch.float64) for k, v in s["flat"].items() if k != "g"}
        place, block = 0, 0
        for i, p in enumerate(s["p"]):
            n = p.numel()
            g, m, v = (s[k][i].reshape(-1).double() for k in ("g", "m", "v"))
            if s["scales"]:
                scales = s["scales"][i].double().repeat_interleave(256, 0)[:n]
                m, v = m * scales[:, 0], (v * scales[:, 1]) ** 2
            m = B1 * m + (1.0 - B1) * g
            v = B2 * v + (1.0 - B2) * g * g
            step = m / (1.0 - B1 ** t) / (torch.sqrt(v / (1.0 - B2 ** t)) + ADAM_EPS)
            out["p"][place:place + n] = p.reshape(-1).double() * (1.0 - LR * WD) - LR * step
            if s["scales"]:
                count = -(-n // 256)
                for k, (name, u) in enumerate((("m", m), ("v", torch.sqrt(v)))):
                    full = torch.zeros(count * 256, device="cuda", dtype=torch.float64)
                    full[:n] = u
                    a = full.view(count, 256).abs().max(1).values.clamp_min(TINY)
                    out["scales"][block:block + count, k] = a / 448.0
                    code = (full.view(count, 256) / a[:, None] * 448.0).view(-1)[:n]
                    if name == "v":
                        code = torch.where(u > 0, code.clamp_min(2.0 ** -9), code)
                    out[name][place:place + n] = code.to(F8).double()
                block += count
            else:
                out["m"][place:place + n], out["v"][place:place + n] = m, v
            place += -(-n // 64) * 64
        return out
