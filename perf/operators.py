"""What the 8-bit and ragged linear operators are timed on, and their plain forms.

Four operators that a program calls one after the other: a root-mean-square norm with the residual's
addition (rows in 16 or 32 bits, or 8-bit rows with a scale for each 128 columns), the quantisation of
activations and weights, the 8-bit matrix product with a scale for each block of 128, and the product of
rows that are sorted by group (a camera stream, an expert) with one weight for each group.

`listed()` are named cases, `draw()` gives more of the same ranges; `prepare` makes the inputs of one, `run`
is one call (the plain torch form, or the package's kernels where `own` is true), `exact` the same in 64 bits.
"""
import importlib
import math

import numpy as np
import torch

own = False

PACKAGE = "a-lightweight-unsupervised-feature-extractor-_amd"
BLOCK = 128          # columns that share a scale
TOP = 448.0          # the largest e4m3 value
LEAST = 2.0 ** -117  # the least amax a scale is made for: below it the block's scale is LEAST / 448
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_size = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one frame of one stream: 256 detections' 512-channel means, normalised for the 8-bit head
        {"name": "norm8 frame", "op": "norm8", "rows": 256, "cols": 512, "dtype": "bf16", "residual": True},
        # every pixel row of 8 x 256 ROIs of 10 x 10, the width of the encoder, with the residual
        {"name": "norm pixels", "op": "norm", "rows": 204800, "cols": 512, "dtype": "bf16", "residual": True},
        # a training step's norm over the pixel rows of 7 x 7 ROIs, and its gradients
        {"name": "norm grad", "op": "norm_grad", "rows": 100352, "cols": 512, "dtype": "bf16", "residual": False},
        # the transition's 1024-wide input rows, quantised before its product
        {"name": "quant rows", "op": "quant", "rows": 204800, "cols": 1024, "dtype": "bf16", "block": 1},
        # an odd-sized weight in 32 bits, quantised once when a model is loaded
        {"name": "quant weight", "op": "quant", "rows": 5003, "cols": 1111, "dtype": "f32", "block": 128},
        # 16 detections through one wide layer: the weight's bytes are what counts
        {"name": "mm8 few rows", "op": "mm8", "m": 16, "n": 4096, "k": 4096, "out": "bf16", "block": 128, "bias": True},
        # a step's 8 x 256 embeddings against a gallery of 50000, each row with its own scale
        {"name": "mm8 gallery", "op": "mm8", "m": 2048, "n": 50000, "k": 128, "out": "f32", "block": 1, "bias": False},
        # a large layer: many rows, many columns
        {"name": "mm8 large", "op": "mm8", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "block": 128, "bias": False},
        # 8 streams' ragged detections, each through its own stream's 512-wide layer, in 8 bits
        {"name": "group8 streams", "op": "group8", "groups": 8, "rows": 1500, "n": 512, "k": 512, "out": "bf16", "block": 128},
        # the pixel rows of many ragged groups, in 8 bits
        {"name": "group8 many", "op": "group8", "groups": 64, "rows": 65536, "n": 2048, "k": 1024, "out": "bf16", "block": 128},
        # one or two rows for each of 64 groups, in 16 bits: the weights' bytes are what counts
        {"name": "group16 single", "op": "group16", "groups": 64, "rows": 80, "n": 1024, "k": 1024, "dtype": "bf16"},
        # a training step of a ragged layer: the product and both gradients
        {"name": "group16 grad", "op": "group16_grad", "groups": 16, "rows": 16384, "n": 2048, "k": 2048, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, v, step=16):
    """v, or the multiple of `step` below it, or an odd number near it."""
    return max(1, rng.choice((v, v // step * step or step, v // step * step or step, v | 1)))


def draw(rng):
    op = rng.choice(("norm", "norm8", "norm_grad", "quant", "mm8", "mm8", "mm8", "group8", "group8", "group16",
                     "group16_grad"))
    if op in ("norm", "norm8", "norm_grad", "quant"):
        cols = _odd(rng, _log(rng, 16, 8192))
        rows = _log(rng, 1, min(204800, 100_000_000 // cols))
        c = {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(("bf16", "bf16", "f16", "f32"))}
        if op == "quant":
            c["block"] = rng.choice((1, BLOCK))
        else:
            c["residual"] = rng.random() < 0.5
        return c
    if op == "mm8":
        k = _odd(rng, _log(rng, 32, 8192))
        n = _odd(rng, _log(rng, 32, 50000))
        m = _odd(rng, min(_log(rng, 1, 16384), 100_000_000 // n, 500_000_000_000 // (n * k) or 1))
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(("bf16", "bf16", "f16", "f32")),
                "block": rng.choice((1, BLOCK, BLOCK)), "bias": rng.random() < 0.5}
    g = _log(rng, 1, 64)
    k = _odd(rng, _log(rng, 64, 2048))
    n = _odd(rng, _log(rng, 64, 2048))
    rows = _log(rng, 1, 32768 if op != "group16_grad" else 16384)
    c = {"op": op, "groups": g, "rows": rows, "n": n, "k": k}
    if op == "group8":
        c.update(out=rng.choice(("bf16", "f16", "f32")), block=rng.choice((1, BLOCK)))
    else:
        c["dtype"] = rng.choice(("bf16", "f16"))
    return c


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op = case["op"]
    if op in ("norm", "norm8", "norm_grad", "quant"):
        r, c, e = case["rows"], case["cols"], _size[case["dtype"]]
        n = r * c
        if op == "quant":
            return {"bytes": n * (e + 1) + 4 * _blocks(c) * (r if case["block"] == 1 else _blocks(r)), "flops": 3 * n}
        res = case["residual"]
        if op == "norm":
            return {"bytes": n * e * (4 if res else 2) + c * e, "flops": 4 * n}
        if op == "norm8":
            return {"bytes": n * (e * (3 if res else 1) + 1) + 4 * r * _blocks(c) + c * e, "flops": 7 * n}
        # x, (residual), dy in; y, (h), dx, dw out: one gradient serves the input and the residual
        return {"bytes": n * e * (6 if res else 4) + 2 * c * e, "flops": 14 * n}
    if op == "mm8":
        m, n, k = case["m"], case["n"], case["k"]
        scales = m + (n if case["block"] == 1 else _blocks(n))
        return {"bytes": (m + n) * k + 4 * scales * _blocks(k) + m * n * _size[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    g, r, n, k = case["groups"], case["rows"], case["n"], case["k"]
    used = min(g, r)  # at most so many weights have rows
    if op == "group8":
        scales = r + used * (n if case["block"] == 1 else _blocks(n))
        return {"bytes": (r + used * n) * k + 4 * scales * _blocks(k) + r * n * _size[case["out"]], "flops": 2 * r * n * k}
    if op == "group16":
        return {"bytes": 2 * (r * k + used * n * k + r * n), "flops": 2 * r * n * k}
    # x, w, dy in; y, dx, dw (of every group) out
    return {"bytes": 2 * (2 * r * k + 2 * r * n + (used + g) * n * k), "flops": 6 * r * n * k}


# ------------------------------------------------------------------------------------------ inputs
def _quantised(v, block):
    """(e4m3 codes, f32 scales) of v [.., rows, cols], as quantize_fp8 lays them out: rows padded to 16 bytes, scales
    with the rows next to each other."""
    rows, cols = v.shape[-2:]
    kb, rb = _blocks(cols), (rows if block == 1 else _blocks(rows))
    step = 1 if block == 1 else BLOCK
    full = torch.zeros(v.shape[:-2] + (rb * step, kb * BLOCK), device=v.device)
    full[..., :rows, :cols] = v
    t = full.view(v.shape[:-2] + (rb, step, kb, BLOCK))
    scale = t.abs().amax((-3, -1)).clamp_min(LEAST) / TOP
    codes = (t / scale[..., :, None, :, None]).to(torch.float8_e4m3fn).view(full.shape)
    ld = -(-cols // 16) * 16
    return codes[..., :rows, :ld].contiguous()[..., :cols], scale.transpose(-1, -2).contiguous().transpose(-1, -2)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, device=dev, generator=gen).to(dtype)

    s = {"case": case}
    if op in ("norm", "norm8", "norm_grad", "quant"):
        r, c, dt = case["rows"], case["cols"], TYPES[case["dtype"]]
        # rows of different sizes, as features of different detections have
        size = torch.exp(torch.randn((r, 1), device=dev, generator=gen))
        s["x"] = (normal(r, c) * size).to(dt)
        if op == "quant":
            return s
        s["weight"] = (1 + 0.2 * normal(c)).to(dt)
        s["residual"] = normal(r, c, dtype=dt) if case["residual"] else None
        if op == "norm_grad":
            s["dy"] = normal(r, c, dtype=dt)
            s["dh"] = normal(r, c, dtype=dt) if case["residual"] else None
            for k in ("x", "weight", "residual"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s
    if op == "mm8":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["x_scale"] = _quantised(normal(m, k), 1)
        s["w"], s["w_scale"] = _quantised(normal(n, k) / math.sqrt(k), case["block"])
        s["bias"] = normal(n) if case["bias"] else None
        return s
    g, r, n, k = case["groups"], case["rows"], case["n"], case["k"]
    # ragged: some groups have many rows, some none
    rs = np.random.RandomState(seed % (1 << 31))
    counts = rs.multinomial(r, rs.dirichlet(np.full(g, 1.0)))
    s["sizes"] = [int(v) for v in counts]
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device=dev)
    x, w = normal(r, k), normal(g, n, k) / math.sqrt(k)
    if op == "group8":
        s["x"], s["x_scale"] = _quantised(x, 1)
        s["w"], s["w_scale"] = _quantised(w, case["block"])
        return s
    dt = TYPES[case["dtype"]]
    s["x"], s["w"] = x.to(dt), w.to(dt)
    if op == "group16_grad":
        s["dy"] = normal(r, n, dtype=dt)
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _plain_scales(v, block):
    """The scales [rows or row blocks, column blocks] of v, and each value's scale."""
    rows, cols = v.shape
    kb = _blocks(cols)
    full = torch.nn.functional.pad(v, (0, kb * BLOCK - cols)).view(rows, kb, BLOCK)
    top = full.abs().amax(2)
    if block != 1:
        rb = _blocks(rows)
        top = torch.nn.functional.pad(top, (0, 0, 0, rb * BLOCK - rows)).view(rb, BLOCK, kb).amax(1)
    top = top.clamp_min(LEAST)
    each = top.repeat_interleave(BLOCK, 1)[:, :cols]
    return top / TOP, each if block == 1 else each.repeat_interleave(BLOCK, 0)[:rows]


def _plain_quant(v, block):
    scale, top = _plain_scales(v, block)
    return (v * (TOP / top)).to(torch.float8_e4m3fn), scale


def _plain_norm(x, weight, residual):
    h = x.float() if residual is None else x.float() + residual.float()
    r = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    return h, r, h * r * weight.float()


def _widened(q, scale, block):
    """The values that 8-bit codes [rows, cols] stand for."""
    each = scale.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    if block != 1:
        each = each.repeat_interleave(BLOCK, 0)[:q.shape[0]]
    return q.float() * each


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quant":
        return _plain_quant(s["x"].float(), case["block"])
    if op in ("norm", "norm8", "norm_grad"):
        x, w, res = (t if t is None else t.detach() for t in (s["x"], s["weight"], s["residual"]))
        h, r, y = _plain_norm(x, w, res)
        more = () if res is None else (h.to(x.dtype),)
        if op == "norm":
            return (y.to(x.dtype),) + more
        if op == "norm8":
            return _plain_quant(y, 1) + more
        dy = s["dy"].float()
        dn, n = dy * w.float(), h * r
        dx = r * (dn - n * (dn * n).mean(1, keepdim=True))
        if res is not None:
            dx = dx + s["dh"].float()
        dx = dx.to(x.dtype)
        dw = (dy * n).sum(0).to(w.dtype)
        return (y.to(x.dtype),) + more + (dx, dw) + (() if res is None else (dx,))
    if op == "mm8":
        y = _widened(s["x"], s["x_scale"], 1) @ _widened(s["w"], s["w_scale"], case["block"]).t()
        if s["bias"] is not None:
            y += s["bias"]
        return y.to(TYPES[case["out"]])
    g, n, k, at = case["groups"], case["n"], case["k"], 0
    x = s["x"].detach()
    y = torch.empty((case["rows"], n), device=x.device, dtype=TYPES[case["out"]] if op == "group8" else x.dtype)
    if op == "group16_grad":
        dx, dw = torch.empty_like(x), torch.zeros((g, n, k), device=x.device, dtype=x.dtype)
    for i, size in enumerate(s["sizes"]):
        if size == 0:
            continue
        rows = slice(at, at + size)
        at += size
        if op == "group8":
            xs, ws = _widened(x[rows], s["x_scale"][rows], 1), _widened(s["w"][i], s["w_scale"][i], case["block"])
        else:
            xs, ws = x[rows].float(), s["w"].detach()[i].float()
        y[rows] = (xs @ ws.t()).to(y.dtype)
        if op == "group16_grad":
            dy = s["dy"][rows].float()
            dx[rows] = (dy @ ws).to(dx.dtype)
            dw[i] = (dy.t() @ xs).to(dw.dtype)
    return (y, dx, dw) if op == "group16_grad" else y


# -------------------------------------------------------------------------------- the package's calls
def _kernels(s):
    trk = getattr(_kernels, "package", None)  # a program imports it once, not at every call
    if trk is None:
        trk = _kernels.package = importlib.import_module(PACKAGE)
    case = s["case"]
    op = case["op"]
    if op == "quant":
        return trk.quantize_fp8(s["x"], block_rows=case["block"])
    if op == "norm":
        y = trk.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return y if s["residual"] is not None else (y,)
    if op == "norm8":
        return trk.rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    if op == "norm_grad":
        out = trk.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        if s["residual"] is None:
            return (out,) + torch.autograd.grad(out, (s["x"], s["weight"]), s["dy"])
        return out + torch.autograd.grad(out, (s["x"], s["weight"], s["residual"]), (s["dy"], s["dh"]))
    if op == "mm8":
        return trk.matmul_fp8(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], out_dtype=TYPES[case["out"]])
    if op == "group8":
        return trk.matmul_grouped(s["x"], s["w"], s["counts"], x_scale=s["x_scale"], w_scale=s["w_scale"],
                                  out_dtype=TYPES[case["out"]])
    y = trk.matmul_grouped(s["x"], s["w"], s["counts"])
    if op == "group16":
        return y
    return (y,) + torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])


def run(state):
    if own:
        return _kernels(state)
    return _plain(state)


# --------------------------------------------------------------------------------------- in 64 bits
def _round_e4m3(v):
    """v in 64 bits, rounded to the nearest e4m3 value (ties to even)."""
    exponent = torch.frexp(v)[1].double() - 1  # frexp's mantissa is in [1/2, 1)
    step = torch.exp2(exponent.clamp_min(-6) - 3)
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _exact_quant(v, block):
    rows, cols = v.shape
    rb = rows if block == 1 else _blocks(rows)
    scale = torch.empty((rb, _blocks(cols)), device=v.device, dtype=torch.float64)
    codes = torch.empty_like(v)
    for j in range(_blocks(cols)):
        part = v[:, j * BLOCK:(j + 1) * BLOCK]
        top = part.abs().amax(1)
        if block != 1:
            top = torch.stack([t.max() for t in top.split(BLOCK)])
        scale[:, j] = top.clamp_min(LEAST) / TOP
        each = scale[:, j] if block == 1 else scale[:, j].repeat_interleave(BLOCK)[:rows]
        codes[:, j * BLOCK:(j + 1) * BLOCK] = _round_e4m3(part / each[:, None])
    return codes, scale


def _exact_values(q, scale, block):
    v = q.to(torch.float64)
    for j in range(scale.shape[1]):
        each = scale[:, j].double()
        if block != 1:
            each = each.repeat_interleave(BLOCK)[:v.shape[0]]
        v[:, j * BLOCK:(j + 1) * BLOCK] *= each[:, None]
    return v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "quant":
            return _exact_quant(s["x"].double(), case["block"])
        if op in ("norm", "norm8", "norm_grad"):
            h, w = s["x"].double(), s["weight"].double()
            more = ()
            if s["residual"] is not None:
                h = h + s["residual"].double()
                more = (h,)
            root = torch.sqrt(h.square().sum(1, keepdim=True) / case["cols"] + EPS)
            y = h / root * w
            if op == "norm":
                return (y,) + more
            if op == "norm8":
                return _exact_quant(y, 1) + more
            g = s["dy"].double() * w
            dx = g / root - h * (g * h).sum(1, keepdim=True) / (case["cols"] * root ** 3)
            dw = (s["dy"].double() * h / root).sum(0)
            if s["residual"] is None:
                return (y, dx, dw)
            dx = dx + s["dh"].double()
            return (y, h, dx, dw, dx)
        if op == "mm8":
            y = torch.mm(_exact_values(s["x"], s["x_scale"], 1), _exact_values(s["w"], s["w_scale"], case["block"]).t())
            return y if s["bias"] is None else y + s["bias"].double()
        y = torch.zeros((case["rows"], case["n"]), device=s["x"].device, dtype=torch.float64)
        ends = np.cumsum(s["sizes"])
        if op == "group8":
            for i, end in enumerate(ends):
                a = end - s["sizes"][i]
                if end > a:
                    y[a:end] = torch.mm(_exact_values(s["x"][a:end], s["x_scale"][a:end], 1),
                                        _exact_values(s["w"][i], s["w_scale"][i], case["block"]).t())
            return y
        x, w = s["x"].double(), s["w"]
        dx, dw = torch.zeros_like(x), torch.zeros(w.shape, device=w.device, dtype=torch.float64)
        for i, end in enumerate(ends):
            a = end - s["sizes"][i]
            if end > a:
                y[a:end] = torch.mm(x[a:end], w[i].double().t())
                if op == "group16_grad":
                    dx[a:end] = torch.mm(s["dy"][a:end].double(), w[i].double())
                    dw[i] = torch.mm(s["dy"][a:end].double().t(), x[a:end])
        return (y, dx, dw) if op == "group16_grad" else y
