"""Block-scaled 8-bit products and Muon updates: the cases they are measured on, their plain forms and their exact results.

cast      values to 8-bit floating point and back, with a power-of-two scale for each block of 128 along the rows (or
          for each 128 x 128 block), optionally with the transposed copy that a weight gradient reads
serve     the product of freshly cast activations with weights held in 8 bits (y = x w^T)
matmul    the product of two 8-bit operands, optionally added to what the output holds (weight gradients)
linear    a linear layer's training step: casts, y = x w^T, dx = dy w, dw = dy^T x
ortho     Newton-Schulz orthogonalisation of one matrix
muon      the Muon update (momentum, orthogonalisation, decay, step) of a list of weights
"""
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_NS = (3.4445, -4.7750, 2.0315)  # the quintic of the Muon optimiser (K. Jordan, 2024)
_STEPS = 5
_MUON = {"lr": 0.02, "momentum": 0.95, "decay": 0.01, "rms": 0.2}

# the dense conv weights of the YOLOv8n detection head with 80 classes, as matrices [oc, ic * k * k]
_HEAD = ("64x576,64x576,64x64,64x1152,64x576,64x64,64x2304,64x576,64x64,"
         "80x576,80x720,80x80,80x1152,80x720,80x80,80x2304,80x720,80x80")


def listed():
    return [
        # one row handed to an 8-bit product: launch latency only
        {"name": "cast_1x4096", "kind": "cast", "rows": 1, "cols": 4096, "type": "bf16", "fmt": "e4m3", "block": 1,
         "both": False},
        # a layer's activations, in both orientations for the backward pass
        {"name": "cast_8192x4096_both", "kind": "cast", "rows": 8192, "cols": 4096, "type": "bf16", "fmt": "e4m3",
         "block": 1, "both": True},
        # one token through an 8-bit layer: bound by reading the weights
        {"name": "serve_1x4096x4096", "kind": "serve", "m": 1, "n": 4096, "k": 4096, "type": "bf16"},
        # a small ragged batch, contraction length no multiple of the block
        {"name": "serve_37x5120x2000", "kind": "serve", "m": 37, "n": 5120, "k": 2000, "type": "f16"},
        # a full training-size product
        {"name": "matmul_8192", "kind": "matmul", "m": 8192, "n": 8192, "k": 8192, "a": "e4m3", "b": "e4m3",
         "wblock": 128, "out": "bf16", "add": False},
        # a weight gradient over 16k tokens, e5m2 gradients, added to the buffer of earlier micro-batches
        {"name": "wgrad_4096x1000x16384", "kind": "matmul", "m": 4096, "n": 1000, "k": 16384, "a": "e5m2", "b": "e4m3",
         "wblock": 1, "out": "f32", "add": True},
        # forward and backward of one layer with every cast
        {"name": "linear_4096", "kind": "linear", "t": 4096, "n": 4096, "k": 4096},
        # one conv weight of the detection head
        {"name": "ortho_64x576", "kind": "ortho", "rows": 64, "cols": 576, "in": "f32", "out": "bf16"},
        # tall and ragged, full single precision
        {"name": "ortho_1000x333_f32", "kind": "ortho", "rows": 1000, "cols": 333, "in": "f32", "out": "f32"},
        # a large square weight
        {"name": "ortho_4096", "kind": "ortho", "rows": 4096, "cols": 4096, "in": "bf16", "out": "bf16"},
        # every dense conv weight of the detection head in one call
        {"name": "muon_head", "kind": "muon", "shapes": _HEAD},
        # the four matrices of a wider block in one call, one of them ragged
        {"name": "muon_block", "kind": "muon", "shapes": "1024x1024,4096x1024,1024x4096,1000x2049"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["cast", "serve", "matmul", "linear", "ortho", "muon"])
    if kind == "cast":
        return {"kind": kind, "rows": _spread(rng, 1, 8192), "cols": _spread(rng, 1, 4096),
                "type": rng.choice(["f32", "bf16", "f16"]), "fmt": rng.choice(["e4m3", "e5m2"]),
                "block": rng.choice([1, 128]), "both": rng.random() < 0.5}
    if kind == "serve":
        return {"kind": kind, "m": _spread(rng, 1, 256), "n": _spread(rng, 16, 8192), "k": _spread(rng, 16, 8192),
                "type": rng.choice(["bf16", "f16"])}
    if kind == "matmul":
        add = rng.random() < 0.5
        return {"kind": kind, "m": _spread(rng, 16, 8192), "n": _spread(rng, 16, 8192), "k": _spread(rng, 16, 8192),
                "a": rng.choice(["e4m3", "e5m2"]), "b": rng.choice(["e4m3", "e5m2"]), "wblock": rng.choice([1, 128]),
                "out": "f32" if add else rng.choice(["f32", "bf16", "f16"]), "add": add}
    if kind == "linear":
        return {"kind": kind, "t": _spread(rng, 16, 4096), "n": _spread(rng, 16, 4096), "k": _spread(rng, 16, 4096)}
    if kind == "ortho":
        return {"kind": kind, "rows": _spread(rng, 2, 4096), "cols": _spread(rng, 2, 4096),
                "in": rng.choice(["f32", "bf16"]), "out": rng.choice(["f32", "bf16"])}
    shapes = ["%dx%d" % (_spread(rng, 2, 1024), _spread(rng, 2, 4096)) for _ in range(rng.randint(1, 24))]
    return {"kind": kind, "shapes": ",".join(shapes)}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ------------------------------------------------------------------ inputs

def _activations(g, rows, cols, dtype):
    """Rows whose channels differ in scale, a few of them by much."""
    scale = torch.exp(0.7 * torch.randn(1, cols, generator=g, device="cuda"))
    scale = torch.where(torch.rand(1, cols, generator=g, device="cuda") < 0.01, 20 * scale, scale)
    return (torch.randn(rows, cols, generator=g, device="cuda") * scale).to(dtype)


def _gradients(g, rows, cols, dtype):
    """Small values whose rows differ in scale."""
    scale = 1e-4 * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    return (torch.randn(rows, cols, generator=g, device="cuda") * scale).to(dtype)


def _update(g, rows, cols):
    """A gradient with a few strong directions over a floor of noise."""
    k = min(16, rows, cols)
    s = 0.7 ** torch.arange(k, device="cuda", dtype=torch.float32)
    strong = (torch.randn(rows, k, generator=g, device="cuda") * s) @ torch.randn(k, cols, generator=g, device="cuda")
    return 1e-3 * (strong + 0.5 * torch.randn(rows, cols, generator=g, device="cuda"))


def _held(x, fmt, block):
    """What a program keeps of an operand in 8 bits: bytes [rows, round_up(cols, 16)] and scale bytes
    [ceil(rows / block), round_up(ceil(cols / 128), 4)], exponent + 127."""
    rows, cols = x.shape
    q, e = _cast(x, fmt, block)
    held = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.uint8, device=x.device)
    held[:, :cols] = q.view(torch.uint8)
    scale = torch.full((e.shape[0], (e.shape[1] + 3) // 4 * 4), 127, dtype=torch.uint8, device=x.device)
    scale[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return held, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "cast":
        s["x"] = _activations(g, case["rows"], case["cols"], _TORCH[case["type"]])
    elif kind == "serve":
        s["x"] = _activations(g, case["m"], case["k"], _TORCH[case["type"]])
        w = torch.randn(case["n"], case["k"], generator=g, device="cuda") / math.sqrt(case["k"])
        s["w"], s["w_scale"] = _held(w, "e4m3", 128)
    elif kind == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        make = _gradients if case["a"] == "e5m2" else _activations
        s["a"], s["a_scale"] = _held(make(g, m, k, torch.float32), case["a"], 1)
        s["b"], s["b_scale"] = _held(_activations(g, n, k, torch.float32), case["b"], case["wblock"])
        if case["add"]:
            s["c"] = torch.randn(m, n, generator=g, device="cuda") * 1e-2
    elif kind == "linear":
        t, n, k = case["t"], case["n"], case["k"]
        s["x"] = _activations(g, t, k, torch.bfloat16)
        s["w"] = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        s["dy"] = _gradients(g, t, n, torch.bfloat16)
    elif kind == "ortho":
        s["u"] = _update(g, case["rows"], case["cols"]).to(_TORCH[case["in"]])
    else:
        s["grad"] = [_update(g, r, c) for r, c in _shapes(case)]
        s["momentum"] = [x + 2 * _update(g, *x.shape) for x in s["grad"]]
        s["weight"] = [torch.randn(r, c, generator=g, device="cuda") / math.sqrt(c) for r, c in _shapes(case)]
    return s


# ------------------------------------------------------------------ plain forms

def _power(e):
    """2^e exactly, -126 <= e <= 127 (exp2 may be an ulp off, which decides ties)."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _cast(x, fmt, block):
    """(8-bit values, exponents [ceil(rows / block), ceil(cols / 128)])."""
    x = x.float()
    rows, cols = x.shape
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    size = torch.nn.functional.pad(size, (0, -cols % 128, 0, -rows % block))
    amax = size.view(size.shape[0] // block, block, size.shape[1] // 128, 128).amax((1, 3))
    m, ex = torch.frexp(amax)  # 448 and 57344 are 0.875 times a power of two
    e = ex - (9 if fmt == "e4m3" else 16) + (m > 0.875)
    e = torch.where(amax > 0, e.clamp(min=-126), torch.zeros_like(e))
    return (x * _power(-e).repeat_interleave(block, 0).repeat_interleave(128, 1)[:rows, :cols]).to(_FP8[fmt]), e


def _values(q, e, block):
    rows, cols = q.shape
    return q.float() * _power(e).repeat_interleave(block, 0).repeat_interleave(128, 1)[:rows, :cols]


def _rounded(x, fmt, block):
    return _values(*_cast(x, fmt, block), block)


def _unheld(held, scale, fmt, block, cols):
    return _values(held.view(_FP8[fmt])[:, :cols], scale[:, :(cols + 127) // 128].int() - 127, block)


def _orthogonal(u):
    x = u.float()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    norm = torch.linalg.vector_norm(x, dtype=torch.float64)
    x = torch.where(norm > 0, x / norm.clamp(min=1e-300), torch.zeros((), device=x.device)).float()
    a, b, c = _NS
    for _ in range(_STEPS):
        p = x @ x.t()
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.t() if tall else x


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "cast":
        t = _TORCH[case["type"]]
        out = [_rounded(s["x"], case["fmt"], case["block"]).to(t)]
        if case["both"]:
            out.append(_rounded(s["x"].t(), case["fmt"], case["block"]).to(t))
        return out
    if kind == "serve":
        return (_rounded(s["x"], "e4m3", 1) @ _unheld(s["w"], s["w_scale"], "e4m3", 128, case["k"]).t()).to(s["x"].dtype)
    if kind == "matmul":
        c = (_unheld(s["a"], s["a_scale"], case["a"], 1, case["k"])
             @ _unheld(s["b"], s["b_scale"], case["b"], case["wblock"], case["k"]).t())
        if case["add"]:
            s["c"] += c
            return s["c"]
        return c.to(_TORCH[case["out"]])
    if kind == "linear":
        x, w, dy = s["x"], _rounded(s["w"], "e4m3", 128), s["dy"]
        y = _rounded(x, "e4m3", 1) @ w.t()
        dx = _rounded(dy, "e5m2", 1) @ w
        dw = _rounded(dy.t(), "e5m2", 1) @ _rounded(x.t(), "e4m3", 1).t()
        return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw}
    if kind == "ortho":
        return _orthogonal(s["u"]).to(_TORCH[case["out"]])
    for w, m, g in zip(s["weight"], s["momentum"], s["grad"]):
        m.mul_(_MUON["momentum"]).add_(g)
        o = _orthogonal(g + _MUON["momentum"] * m)
        w.mul_(1 - _MUON["lr"] * _MUON["decay"]).sub_(_MUON["lr"] * _MUON["rms"] * math.sqrt(max(w.shape)) * o)
    return {"weight": s["weight"], "momentum": s["momentum"]}


# ------------------------------------------------------------------ the framework's calls

def _empty(rows, cols, dtype):
    return torch.empty(rows, cols, dtype=dtype, device="cuda")


def _own_cast(sy, x, fmt, block, both, stream):
    rows, cols = x.shape
    q = _empty(rows, sy.fp8_pitch(cols), torch.uint8)
    sc = _empty(-(-rows // block), sy.fp8_scale_pitch(cols), torch.uint8)
    qt = sct = None
    if both:
        qt = _empty(cols, sy.fp8_pitch(rows), torch.uint8)
        sct = _empty(-(-cols // block), sy.fp8_scale_pitch(rows), torch.uint8)
    sy.quantize_fp8_device(x.data_ptr(), _own_type(sy, x.dtype), cols, rows, cols, _own_fmt(sy, fmt), block, q.data_ptr(),
                           sc.data_ptr(), qt.data_ptr() if both else 0, sct.data_ptr() if both else 0, stream=stream)
    return q, sc, qt, sct


def _own_type(sy, dtype):
    return {torch.float32: sy.SY_TYPE_F32, torch.bfloat16: sy.SY_TYPE_BF16, torch.float16: sy.SY_TYPE_F16}[dtype]


def _own_fmt(sy, fmt):
    return sy.SY_FP8_E4M3 if fmt == "e4m3" else sy.SY_FP8_E5M2


def _own_matmul(sy, a, a_scale, a_fmt, b, b_scale, b_fmt, b_block, m, n, k, out, add, stream):
    sy.matmul_fp8_device(a.data_ptr(), a_scale.data_ptr(), _own_fmt(sy, a_fmt), 1, b.data_ptr(), b_scale.data_ptr(),
                         _own_fmt(sy, b_fmt), b_block, m, n, k, out.data_ptr(), _own_type(sy, out.dtype), n, add,
                         stream=stream)
    return out


def _own(s):
    import simdyolo_b200 as sy
    case, kind = s["case"], s["case"]["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "cast":
        x, fmt, block = s["x"], case["fmt"], case["block"]
        rows, cols = x.shape
        q, sc, qt, sct = _own_cast(sy, x, fmt, block, case["both"], stream)
        out = [torch.empty_like(x)]
        sy.dequantize_fp8_device(q.data_ptr(), sc.data_ptr(), rows, cols, _own_fmt(sy, fmt), block, out[0].data_ptr(),
                                 _own_type(sy, x.dtype), cols, stream=stream)
        if case["both"]:
            out.append(_empty(cols, rows, x.dtype))
            sy.dequantize_fp8_device(qt.data_ptr(), sct.data_ptr(), cols, rows, _own_fmt(sy, fmt), block,
                                     out[1].data_ptr(), _own_type(sy, x.dtype), rows, stream=stream)
        return out
    if kind == "serve":
        m, n, k = case["m"], case["n"], case["k"]
        q, sc, _, _ = _own_cast(sy, s["x"], "e4m3", 1, False, stream)
        return _own_matmul(sy, q, sc, "e4m3", s["w"], s["w_scale"], "e4m3", 128, m, n, k,
                           _empty(m, n, s["x"].dtype), False, stream)
    if kind == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        out = s["c"] if case["add"] else _empty(m, n, _TORCH[case["out"]])
        return _own_matmul(sy, s["a"], s["a_scale"], case["a"], s["b"], s["b_scale"], case["b"], case["wblock"], m, n,
                           k, out, case["add"], stream)
    if kind == "linear":
        t, n, k = case["t"], case["n"], case["k"]
        x, xs, xt, xts = _own_cast(sy, s["x"], "e4m3", 1, True, stream)
        w, ws, wt, wts = _own_cast(sy, s["w"], "e4m3", 128, True, stream)
        d, ds, dt, dts = _own_cast(sy, s["dy"], "e5m2", 1, True, stream)
        y = _own_matmul(sy, x, xs, "e4m3", w, ws, "e4m3", 128, t, n, k, _empty(t, n, s["x"].dtype), False, stream)
        dx = _own_matmul(sy, d, ds, "e5m2", wt, wts, "e4m3", 128, t, k, n, _empty(t, k, s["x"].dtype), False, stream)
        dw = _own_matmul(sy, dt, dts, "e5m2", xt, xts, "e4m3", 1, n, k, t, _empty(n, k, torch.float32), False, stream)
        return {"y": y, "dx": dx, "dw": dw}
    if kind == "ortho":
        rows, cols = case["rows"], case["cols"]
        out = _empty(rows, cols, _TORCH[case["out"]])
        if "work" not in s:
            need = sy.orthogonalize_workspace(rows, cols, _own_type(sy, out.dtype))
            s["work"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        sy.orthogonalize_device(s["u"].data_ptr(), _own_type(sy, s["u"].dtype), cols, rows, cols, _STEPS, out.data_ptr(),
                                _own_type(sy, out.dtype), cols, s["work"].data_ptr(), s["work"].numel(), stream=stream)
        return out
    if "list" not in s:
        s["list"] = sy.muon_tensors([(w.data_ptr(), m.data_ptr(), g.data_ptr(), *w.shape)
                                     for w, m, g in zip(s["weight"], s["momentum"], s["grad"])])
        s["options"] = sy.muon_options(lr=_MUON["lr"], momentum=_MUON["momentum"], weight_decay=_MUON["decay"],
                                       rms=_MUON["rms"], nesterov=True, steps=_STEPS)
        s["work"] = torch.empty(sy.muon_workspace(s["list"], s["options"]), dtype=torch.uint8, device="cuda")
    sy.muon_update_device(s["list"], s["options"], s["work"].data_ptr(), s["work"].numel(), stream=stream)
    return {"weight": s["weight"], "momentum": s["momentum"]}


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------ work and exact results

def work(case):
    kind = case["kind"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if kind == "cast":
        n = case["rows"] * case["cols"] * size[case["type"]]
        return {"bytes": n * (3 if case["both"] else 2), "flops": 0}
    if kind in ("serve", "matmul"):
        m, n, k = case["m"], case["n"], case["k"]
        moved = 2 * m * k + n * k + 2 * m * n
        if kind == "matmul":
            moved = m * k + n * k + m * n * size[case["out"]] * (2 if case["add"] else 1)
        return {"bytes": moved + (m + n) * k / 128, "flops": 2 * m * n * k}
    if kind == "linear":
        t, n, k = case["t"], case["n"], case["k"]
        return {"bytes": 2 * (t * k + t * n) * 2 + 2 * 4 * n * k, "flops": 6 * t * n * k}
    pairs = [(case["rows"], case["cols"])] if kind == "ortho" else _shapes(case)
    flops = sum(_STEPS * (3 * min(p) ** 2 * max(p) + min(p) ** 3) for p in pairs)  # symmetric products once
    per = size[case["in"]] + size[case["out"]] if kind == "ortho" else 20
    return {"bytes": per * sum(r * c for r, c in pairs), "flops": flops}


def _two(e):
    return ((e + 1023).long() << 52).view(torch.float64)


def _exact_values(x, fmt, block):
    """The cast in 64 bits: the block's exponent from its largest finite size, values rounded to the format's step."""
    x = x.double()
    rows, cols = x.shape
    bits, low, most = (3, -6, 448.0) if fmt == "e4m3" else (2, -14, 57344.0)
    padded = torch.zeros(-(-rows // block) * block, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    padded[:rows, :cols] = x
    tiles = padded.unflatten(0, (-1, block)).unflatten(2, (-1, 128))
    peak = tiles.abs().nan_to_num(0.0, 0.0, 0.0).amax(dim=(1, 3), keepdim=True)
    e = torch.ceil(torch.log2(peak / most))
    e = e + (peak > most * _two(e)).double() - (peak <= most * _two(e - 1)).double()
    e = torch.where(peak > 0, e.clamp(min=-126), torch.zeros_like(e))
    v = tiles * _two(-e)
    step = _two(torch.frexp(v.abs().clamp(min=2.0 ** low)).exponent - 1 - bits)
    return (torch.round(v / step) * step * _two(e)).flatten(2, 3).flatten(0, 1)[:rows, :cols]


def _exact_held(held, scale, fmt, block, cols):
    e = scale[:, :-(-cols // 128)].double() - 127
    each = _two(e)[torch.arange(held.shape[0], device=held.device) // block][:, torch.arange(cols, device=held.device) // 128]
    return held[:, :cols].contiguous().view(_FP8[fmt]).double() * each


def _exact_orthogonal(u):
    x = u.double()
    if x.shape[0] > x.shape[1]:
        return _exact_orthogonal(u.t()).t()
    total = (x * x).sum().sqrt()
    x = x / total if total > 0 else x
    a, b, c = _NS
    one = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(_STEPS):
        p = x.mm(x.t())
        x = (a * one + p.mm(b * one + c * p)).mm(x)
    return x


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "cast":
        out = [_exact_values(s["x"], case["fmt"], case["block"])]
        return out + [_exact_values(s["x"].t(), case["fmt"], case["block"])] if case["both"] else out
    if kind == "serve":
        return _exact_values(s["x"], "e4m3", 1).mm(_exact_held(s["w"], s["w_scale"], "e4m3", 128, case["k"]).t())
    if kind == "matmul":
        c = _exact_held(s["a"], s["a_scale"], case["a"], 1, case["k"]).mm(
            _exact_held(s["b"], s["b_scale"], case["b"], case["wblock"], case["k"]).t())
        return c + s["c"].double() if case["add"] else c
    if kind == "linear":
        w = _exact_values(s["w"], "e4m3", 128)
        return {"y": _exact_values(s["x"], "e4m3", 1).mm(w.t()), "dx": _exact_values(s["dy"], "e5m2", 1).mm(w),
                "dw": _exact_values(s["dy"].t(), "e5m2", 1).mm(_exact_values(s["x"].t(), "e4m3", 1).t())}
    if kind == "ortho":
        return _exact_orthogonal(s["u"])
    out = {"weight": [], "momentum": []}
    for w, m, g in zip(s["weight"], s["momentum"], s["grad"]):
        v = _MUON["momentum"] * m.double() + g.double()
        o = _exact_orthogonal(g.double() + _MUON["momentum"] * v)
        rate = _MUON["lr"] * _MUON["rms"] * max(w.shape) ** 0.5
        out["weight"].append(w.double() * (1 - _MUON["lr"] * _MUON["decay"]) - rate * o)
        out["momentum"].append(v)
    return out
