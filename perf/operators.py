"""Measured cases of the 8-bit training and serving operators.

Four operators, those of one training step of a RACE block held in 8 bits and
of its use for single tokens:

  norm      root-mean-square norm with the residual's addition; its result as
            it is (training, with gradients) or in 8 bits with one scale for
            each 128 columns (serving)
  product   matrix product of 8-bit rows (a scale for each 128 columns) with an
            8-bit weight (a scale for each 128 x 128 block)
  linear    a training pass of a linear layer held in 8 bits: both operands
            quantised, y = x W^T, dx = dy W and dW = dy^T x
  adamw     one AdamW step over every parameter of a model, with states in 32
            or in 8 bits

``own`` false: elementary torch operations in 32 bits, rounded once at the end.
``own`` true: the framework's entry points.
"""
import math

import torch

own = False

BLOCK = 128            # columns (or elements) that share one scale
TOP = 448.0            # largest value of the 8-bit format (4 exponent, 3 mantissa bits)
TINY = 2.0 ** -126     # smallest scale
EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP0, SEED = 1e-3, 0.9, 0.95, 1e-8, 0.1, 10, 1234
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # one decoded token of a 768-wide causal decoder: latency alone
        {"name": "norm_token", "op": "norm", "rows": 1, "width": 768, "dtype": "bf16", "mode": "8bit"},
        # the 65536-token prompt of the same decoder
        {"name": "norm_prompt", "op": "norm", "rows": 65536, "width": 768, "dtype": "bf16", "mode": "8bit"},
        # odd row count and a width that no vector divides, full precision, with gradients
        {"name": "norm_train_odd", "op": "norm", "rows": 4099, "width": 1001, "dtype": "f32", "mode": "train"},
        # one training batch of the 384-wide image encoder: 256 sequences of 785 tokens
        {"name": "norm_train_vit", "op": "norm", "rows": 200960, "width": 384, "dtype": "bf16", "mode": "train"},
        # query, key and value projections of one decoded token
        {"name": "product_token", "op": "product", "rows": 1, "outs": 2304, "inner": 768},
        # a batch of 16 tokens against a wide layer: the weight's bytes count
        {"name": "product_batch_wide", "op": "product", "rows": 16, "outs": 8192, "inner": 8192},
        # one 785-token sequence, sizes that no tile divides
        {"name": "product_ragged", "op": "product", "rows": 785, "outs": 1160, "inner": 776},
        # a long prompt through a wide layer: arithmetic alone
        {"name": "product_prompt", "op": "product", "rows": 16384, "outs": 8192, "inner": 4096},
        # a short ragged batch through a small layer, forward and backward
        {"name": "linear_train_ragged", "op": "linear", "rows": 1001, "outs": 1048, "inner": 520, "dtype": "bf16"},
        # query, key and value projections of the 768-wide decoder over 65536 tokens
        {"name": "linear_train_decoder", "op": "linear", "rows": 65536, "outs": 2304, "inner": 768, "dtype": "bf16"},
        # every tensor of the 12-layer, 384-wide encoder, states in 32 bits
        {"name": "adamw_vit", "op": "adamw", "layers": 12, "width": 384, "vocab": 1000, "dtype": "f32", "bits": 32},
        # a 1024-wide decoder with its embedding, states in 8 bits
        {"name": "adamw_decoder_8bit", "op": "adamw", "layers": 12, "width": 1024, "vocab": 32000, "dtype": "bf16", "bits": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "product", "linear", "adamw"])
    if op == "norm":
        width = _log(rng, 64, 8192)
        rows = _log(rng, 1, max(1, min(200960, 70_000_000 // width)))
        return {"op": op, "rows": rows, "width": width, "dtype": rng.choice(["bf16", "f32"]), "mode": rng.choice(["8bit", "train"])}
    if op == "product":
        outs, inner = _log(rng, 64, 8192), _log(rng, 64, 8192)
        return {"op": op, "rows": _log(rng, 1, min(16384, 2 ** 39 // (outs * inner))), "outs": outs, "inner": inner}
    if op == "linear":
        outs, inner = _log(rng, 64, 4096), _log(rng, 64, 4096)
        return {"op": op, "rows": _log(rng, 1, min(65536, 10 ** 11 // (outs * inner))), "outs": outs, "inner": inner, "dtype": rng.choice(["bf16", "f32"])}
    c = {"op": op, "layers": rng.randint(1, 12), "width": _log(rng, 33, 1024), "vocab": _log(rng, 10, 32000),
         "dtype": rng.choice(["bf16", "f32"]), "bits": rng.choice([8, 32])}
    while work(c)["bytes"] > 1.8e9 and c["layers"] > 1:
        c["layers"] -= 1
    return c


# ------------------------------------------------------------------ inputs


def _shapes(case):
    """The parameters of a pre-norm decoder: per layer four square projections,
    two feed-forward matrices and two norm weights, then the embedding."""
    w = case["width"]
    layer = [(w,), (w, w), (w, w), (w, w), (w, w), (w,), (4 * w, w), (w, 4 * w)]
    return layer * case["layers"] + [(case["vocab"], w)]


def _offsets(shapes):
    """Where each tensor starts in the flat buffers: on a multiple of BLOCK."""
    at, total = [], 0
    for s in shapes:
        at.append(total)
        total += -(-math.prod(s) // BLOCK) * BLOCK
    return at, total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    op = case["op"]
    if op == "norm":
        dt = DTYPES[case["dtype"]]
        s = (case["rows"], case["width"])
        # residual streams have a few columns far larger than the rest
        wide = 1.0 + 15.0 * (torch.rand(case["width"], generator=g, device="cuda") < 0.01)
        st = {"case": case, "x": normal(*s).to(dt), "residual": (normal(*s) * wide).to(dt), "weight": 1.0 + 0.2 * normal(case["width"])}
        if case["mode"] == "train":
            st |= {"dy": (0.01 * normal(*s)).to(dt), "dh": (0.01 * normal(*s)).to(dt)}
        return st
    if op == "product":
        m, n, k = case["rows"], case["outs"], case["inner"]
        a, sa = _quantize_rows(normal(m, k) * normal(m, 1).abs().add(0.1))
        b, sb = _quantize_square(0.02 * normal(n, k))
        return {"case": case, "a": _pitched(a), "sa": sa.t().contiguous().t(), "b": _pitched(b), "sb": sb}
    if op == "linear":
        dt = DTYPES[case["dtype"]]
        m, n, k = case["rows"], case["outs"], case["inner"]
        return {"case": case, "x": normal(m, k).to(dt), "w": 0.02 * normal(n, k), "dy": (normal(m, n) * 1e-3 * normal(m, 1).exp()).to(dt)}
    shapes = _shapes(case)
    at, total = _offsets(shapes)
    dt = DTYPES[case["dtype"]]
    p, grad = torch.zeros(total, dtype=dt, device="cuda"), torch.zeros(total, dtype=dt, device="cuda")
    m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    live = []
    for s, a in zip(shapes, at):
        n = math.prod(s)
        live.append((a, n))
        scale = torch.rand(1, generator=g, device="cuda") * 1e-3 + 1e-5
        p[a:a + n] = (0.02 * normal(n)).to(dt)
        size = (0.5 * normal(n)).exp() * scale      # each weight's own gradient size
        grad[a:a + n] = (size * normal(n)).to(dt)
        m[a:a + n] = 0.3 * size * normal(n)
        v[a:a + n] = size * size * (0.6 + 0.8 * torch.rand(n, generator=g, device="cuda"))
    st = {"case": case, "p": p, "grad": grad, "step": STEP0}
    if case["bits"] == 8:
        st["m"], st["ms"] = _quantize_flat(m)
        st["v"], st["vs"] = _quantize_flat(v.sqrt())
    else:
        st["m"], st["v"] = m, v
    if own:   # the optimizer that a training program keeps, at step STEP0
        from race_attention_b200.optim import AdamW
        params = []
        for s, (a, n) in zip(shapes, live):
            q = torch.nn.Parameter(p[a:a + n].view(s))
            q.grad = grad[a:a + n].view(s)
            params.append(q)
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
        opt.set_state(step=STEP0, exp_avg=st["m"], exp_avg_sq=st["v"], exp_avg_scale=st.get("ms"), exp_avg_sq_scale=st.get("vs"))
        st["opt"] = opt
    return st


def _pitched(codes):
    """Rows that start on 16-byte boundaries."""
    r, k = codes.shape
    out = torch.zeros((r, -(-k // 16) * 16), dtype=torch.uint8, device=codes.device)
    out[:, :k] = codes.view(torch.uint8)
    return out.view(F8)[:, :k]


# ------------------------------------------------------------------ one pass


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_norm(st):
    from race_attention_b200.fp8 import rms_norm
    if st["case"]["mode"] == "8bit":
        y, h = rms_norm(st["x"], st["weight"], residual=st["residual"], eps=EPS, quantize=True)
        return {"codes": y.codes, "scales": y.scales, "h": h}
    x, r, w = (st[n].detach().requires_grad_(True) for n in ("x", "residual", "weight"))
    y, h = rms_norm(x, w, residual=r, eps=EPS)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (st["dy"], st["dh"]))
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dr": dr, "dw": dw}


def _own_product(st):
    from race_attention_b200.fp8 import BlockFp8, fp8_matmul
    return fp8_matmul(BlockFp8(st["a"], st["sa"]), BlockFp8(st["b"], st["sb"]), out_dtype=torch.bfloat16)


def _own_linear(st):
    from race_attention_b200.fp8 import fp8_linear
    x, w = st["x"].detach().requires_grad_(True), st["w"].detach().requires_grad_(True)
    y = fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), st["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def _own_adamw(st):
    opt = st["opt"]
    opt.step()
    out = {"p": st["p"], "m": opt.exp_avg, "v": opt.exp_avg_sq}
    if st["case"]["bits"] == 8:
        out |= {"ms": opt.exp_avg_scale, "vs": opt.exp_avg_sq_scale}
    return out


_own = {"norm": _own_norm, "product": _own_product, "linear": _own_linear, "adamw": _own_adamw}


def _pad(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def _up(n):
    return -(-n // BLOCK) * BLOCK


def _codes(x, scale):
    return (x * (1.0 / scale)).clamp(-TOP, TOP).to(F8)


def _quantize_rows(x):
    """[R, K] -> codes, scales [R, ceil(K / 128)]."""
    r, k = x.shape
    b = _pad(x.float(), r, _up(k)).view(r, -1, BLOCK)
    s = (b.abs().amax(2) / TOP).clamp_min(TINY)
    return _codes(b, s[:, :, None]).view(r, -1)[:, :k], s


def _quantize_square(w):
    n, k = w.shape
    b = _pad(w.float(), _up(n), _up(k)).view(_up(n) // BLOCK, BLOCK, _up(k) // BLOCK, BLOCK)
    s = (b.abs().amax((1, 3)) / TOP).clamp_min(TINY)
    return _codes(b, s[:, None, :, None]).view(_up(n), _up(k))[:n, :k], s


def _quantize_flat(x):
    b = x.view(-1, BLOCK)
    s = (b.abs().amax(1) / TOP).clamp_min(TINY)
    return _codes(b, s[:, None]).view(-1), s


def _values_rows(codes, s):
    return codes.float() * s.repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _values_square(codes, s):
    return codes.float() * s.repeat_interleave(BLOCK, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _plain_norm(st):
    x, w = st["x"], st["weight"]
    h = x.float() + st["residual"].float()
    r = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = h * r * w
    if st["case"]["mode"] == "8bit":
        codes, s = _quantize_rows(y)
        return {"codes": codes, "scales": s, "h": h.to(x.dtype)}
    held = h.to(x.dtype).float()     # what a training program keeps for the backward pass
    dy = st["dy"].float()
    g = dy * w
    dx = st["dh"].float() + r * (g - held * (r * r) * (g * held).mean(1, keepdim=True))
    dw = (dy * held * r).sum(0)
    return {"y": y.to(x.dtype), "h": h.to(x.dtype), "dx": dx.to(x.dtype), "dr": dx.to(x.dtype), "dw": dw}


def _plain_product(st):
    return (_values_rows(st["a"], st["sa"]) @ _values_square(st["b"], st["sb"]).t()).to(torch.bfloat16)


def _plain_linear(st):
    x, w, dy = st["x"], st["w"], st["dy"]
    wv = _values_square(*_quantize_square(w))
    y = _values_rows(*_quantize_rows(x)) @ wv.t()
    dx = _values_rows(*_quantize_rows(dy)) @ wv
    # the weight's gradient sums over tokens, so both operands are quantised along them
    dw = _values_rows(*_quantize_rows(dy.t())) @ _values_rows(*_quantize_rows(x.t())).t()
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw}


def _noise(n, step, salt):
    """32 bits for each element, from its index, the seed and the step."""
    i = torch.arange(n, device="cuda")
    h = ((i ^ ((SEED + 0x9E3779B1 * step + salt) & 0xFFFFFFFF)) & 0xFFFFFFFF) * 0x9E3779B1 & 0xFFFFFFFF
    h = (h ^ (h >> 15)) * 0x6A09E667 & 0xFFFFFFFF
    return h ^ (h >> 16)


def _round_up_or_down(y, r16):
    """y >= 0, at most 448, to the 8-bit format: up with the probability of the part cut off."""
    low = (y < 2.0 ** -6).float() * 2.0 ** -6
    bits = (y + low).view(torch.int32) + (r16.int() << 4)
    return (bits & ~0xFFFFF).view(torch.float32) - low


def _hold(x, r16, least):
    b = x.view(-1, BLOCK)
    s = (b.abs().amax(1) / TOP).clamp_min(TINY)
    y = (b.abs() * (1.0 / s)[:, None]).clamp_max(TOP).view(-1)
    c = _round_up_or_down(y, r16)
    if least:   # a second moment above zero is never held as zero
        c = torch.where((y > 0) & (c == 0), torch.full_like(c, 2.0 ** -9), c)
    return (c * x.sign()).to(F8), s


def _plain_adamw(st):
    case, p, g = st["case"], st["p"], st["grad"].float()
    st["step"] += 1
    t = st["step"]
    if case["bits"] == 8:
        m = st["m"].float() * st["ms"].repeat_interleave(BLOCK)
        v = (st["v"].float() * st["vs"].repeat_interleave(BLOCK)).square()
    else:
        m, v = st["m"], st["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    q = p.float() * (1 - LR * DECAY)
    root = v.sqrt()
    q = q - (LR / (1 - BETA1 ** t)) * m / (root * (1 / math.sqrt(1 - BETA2 ** t)) + ADAM_EPS)
    if p.dtype == torch.bfloat16:      # up or down with the probability of the part cut off
        r = _noise(p.numel(), t, 1) & 0xFFFF
        q = ((q.view(torch.int32) + r.int()) & ~0xFFFF).view(torch.float32)
    p.copy_(q)
    if case["bits"] == 8:
        r = _noise(p.numel(), t, 0)
        st["m"], st["ms"] = _hold(m, r & 0xFFFF, False)
        st["v"], st["vs"] = _hold(root, r >> 16, True)
        return {"p": p, "m": st["m"], "v": st["v"], "ms": st["ms"], "vs": st["vs"]}
    st["m"], st["v"] = m, v
    return {"p": p, "m": m, "v": v}


_plain = {"norm": _plain_norm, "product": _plain_product, "linear": _plain_linear, "adamw": _plain_adamw}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "norm":
        e, n = (2 if case["dtype"] == "bf16" else 4), case["rows"] * case["width"]
        if case["mode"] == "8bit":
            return {"bytes": n * (3 * e + 1) + 4 * case["rows"] * -(-case["width"] // BLOCK) + 4 * case["width"], "flops": 6 * n}
        # forward: x, residual, y, h; backward: dy, dh, h, dx (one tensor for both branches)
        return {"bytes": 8 * e * n + 8 * case["width"], "flops": 16 * n}
    if op == "product":
        m, n, k = case["rows"], case["outs"], case["inner"]
        return {"bytes": (m + n) * k + 4 * (m * -(-k // BLOCK)) + 4 * (-(-n // BLOCK) * -(-k // BLOCK)) + 2 * m * n, "flops": 2 * m * n * k}
    if op == "linear":
        e, m, n, k = (2 if case["dtype"] == "bf16" else 4), case["rows"], case["outs"], case["inner"]
        return {"bytes": e * (m * k + m * n) + 4 * n * k + e * (m * n + m * k) + 4 * n * k, "flops": 6 * m * n * k}
    n = sum(math.prod(s) for s in _shapes(case))
    e = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": n * (3 * e + (16 if case["bits"] == 32 else 4)) + (0 if case["bits"] == 32 else 16 * n // BLOCK), "flops": 14 * n}


# ------------------------------------------------------------------ the definition in 64 bits


def _grid(y):
    """Spacing of the 8-bit format at |y| (float64)."""
    e = torch.frexp(y.abs().clamp_min(2.0 ** -12))[1] - 1
    return torch.exp2((e.clamp_min(-6) - 3).double())


def _exact_codes(y):
    d = _grid(y)
    return (torch.round(y / d) * d).clamp(-TOP, TOP)


def _exact_blocks(x, dim):
    """(codes, scales spread over x) with 128 consecutive elements of `dim` to a scale."""
    n = x.shape[dim]
    pad = x.new_zeros([(-n) % BLOCK if d == dim else s for d, s in enumerate(x.shape)])
    parts = torch.cat((x, pad), dim).unflatten(dim, (-1, BLOCK))
    s = (parts.abs().amax(dim + 1, keepdim=True) / TOP).clamp_min(TINY)
    wide = s.expand_as(parts).flatten(dim, dim + 1).narrow(dim, 0, n)
    return _exact_codes(x / wide), s.squeeze(dim + 1), wide


def _exact_square(w):
    n, k = w.shape
    i, j = torch.arange(n, device=w.device) // BLOCK, torch.arange(k, device=w.device) // BLOCK
    cell = i[:, None] * (int(j[-1]) + 1) + j
    top = torch.zeros(int(cell[-1, -1]) + 1, dtype=w.dtype, device=w.device)
    top.scatter_reduce_(0, cell.flatten(), w.abs().flatten(), "amax")
    s = (top / TOP).clamp_min(TINY)[cell]
    return _exact_codes(w / s) * s


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, res, w = (st[n].double() for n in ("x", "residual", "weight"))
        h = x + res
        rms = torch.sqrt((h * h).sum(1) / case["width"] + EPS)
        y = torch.einsum("rc,r,c->rc", h, 1 / rms, w)
        if case["mode"] == "8bit":
            codes, s, _ = _exact_blocks(y, 1)
            return {"codes": codes, "scales": s, "h": h}
        held = h.to(st["x"].dtype).double()
        g = torch.einsum("rc,c->rc", st["dy"].double(), w)
        dot = torch.einsum("rc,rc->r", g, held) / (case["width"] * rms ** 3)
        dx = st["dh"].double() + g / rms[:, None] - held * dot[:, None]
        dw = torch.einsum("rc,rc,r->c", st["dy"].double(), held, 1 / rms)
        return {"y": y, "h": h, "dx": dx, "dr": dx, "dw": dw}
    if op == "product":
        k, n = case["inner"], case["outs"]
        j = torch.arange(k, device="cuda") // BLOCK
        i = torch.arange(n, device="cuda") // BLOCK
        a = st["a"].double() * st["sa"].double()[:, j]
        b = st["b"].double() * st["sb"].double()[i][:, j]
        return torch.einsum("mk,nk->mn", a, b)
    if op == "linear":
        x, w, dy = (st[n].double() for n in ("x", "w", "dy"))
        val = lambda t, dim: (lambda c, s, wide: c * wide)(*_exact_blocks(t, dim))  # noqa: E731
        wv = _exact_square(w)
        return {"y": torch.einsum("mk,nk->mn", val(x, 1), wv), "dx": torch.einsum("mn,nk->mk", val(dy, 1), wv),
                "dw": torch.einsum("mn,mk->nk", val(dy, 0), val(x, 0))}
    t = STEP0 + 1
    g, p = st["grad"].double(), st["p"].double()
    if case["bits"] == 8:
        m = (st["m"].double().view(-1, BLOCK) * st["ms"].double()[:, None]).flatten()
        v = (st["v"].double().view(-1, BLOCK) * st["vs"].double()[:, None]).flatten() ** 2
    else:
        m, v = st["m"].double(), st["v"].double()
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    if case["dtype"] == "bf16":
        # rounded up or down: the part cut off, in 65536ths, and a 16-bit number
        d = torch.exp2((torch.frexp(p)[1] - 8).double())
        r = (_noise(p.numel(), t, 1) & 0xFFFF).double() / 65536
        p = torch.sign(p) * torch.floor(p.abs() / d + r) * d
    if case["bits"] == 32:
        return {"p": p, "m": m, "v": v}
    r = _noise(p.numel(), t, 0)
    held = []
    for x, n in ((m, r & 0xFFFF), (torch.sqrt(v), r >> 16)):
        s = (x.abs().view(-1, BLOCK).amax(1) / TOP).clamp_min(TINY)
        y = x.abs() / s.repeat_interleave(BLOCK)
        d = _grid(y)
        held.append((torch.sign(x) * torch.floor(y / d + n.double() / 65536).mul(d).clamp_max(TOP), s))
    (cm, sm), (cv, sv) = held
    cv = torch.where((v > 0) & (cv == 0), torch.full_like(cv, 2.0 ** -9), cv)
    return {"p": p, "m": cm, "v": cv, "ms": sm, "vs": sv}
