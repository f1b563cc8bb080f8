"""Operators of 8-bit transformer blocks: their cases, inputs, plain forms and exact values.

Kinds of case
  rope    rotary positions on queries and keys: adjacent-pair and half layouts, the whole head or
          its front part, one or two position axes, frequencies scaled for long contexts
  norm    the new residual stream and the next block's normalised input in one pass:
          r = residual_scale * x + gate * post(y),  h = norm(r)
  linear  product in 8-bit integers: rows of x scaled by their largest magnitude,
          y = act((q_x . q_w) * s_x * s_w + bias)
  block   the three as a block's entry uses them: norm with an 8-bit result, the QKV product on
          it, and the rotation of its queries and keys

``own`` False runs the plain forms (elementary torch operations in 32 bits, angles in 64),
True the operators of mast3r_runtime_b200.ops.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEVICE = "cuda:0"


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of one sequence far into a long context, shared key heads
        dict(name="rope one token", kind="rope", batch=1, tokens=1, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, axes=1, scaling="by_parts", factor=8.0, far=100000, dtype="bf16", packed=False),
        # a ragged prompt, adjacent pairs, the front half of the head, full precision
        dict(name="rope ragged part", kind="rope", batch=3, tokens=1237, heads=12, kv_heads=4, dim=96, rot=48,
             interleaved=True, axes=1, scaling="linear", factor=4.0, far=9000, dtype="fp32", packed=False),
        # both views of 64 image pairs, 24 x 32 patches, straight from the packed QKV projection
        dict(name="rope image batch", kind="rope", batch=128, tokens=768, heads=16, kv_heads=16, dim=64, rot=64,
             interleaved=False, axes=2, scaling="none", factor=1.0, far=0, dtype="fp16", packed=True),
        # one token: the launch and the row's own latency
        dict(name="norm one token", kind="norm", rows=1, dim=4096, norm="rms", post="rms", gates=0, bias=False,
             stream="bf16", branch="bf16", out="bf16", residual_scale=1.0),
        # an odd width and a ragged row count; a gate for each of 7 images
        dict(name="norm ragged gates", kind="norm", rows=7 * 577, dim=1001, norm="layer", post="layer", gates=7,
             bias=True, stream="fp32", branch="fp16", out="fp16", residual_scale=0.7),
        # the encoder's stream of 64 image pairs with a gate for each channel
        dict(name="norm image batch", kind="norm", rows=98304, dim=1024, norm="layer", post="none", gates=1,
             bias=True, stream="fp32", branch="bf16", out="bf16", residual_scale=1.0),
        # one token through an MLP input projection: the weights' bytes
        dict(name="linear one token", kind="linear", rows=1, k=1024, n=4096, act="gelu", bias=True, x="bf16",
             out="bf16"),
        # a handful of tokens decoded together
        dict(name="linear 24 tokens", kind="linear", rows=24, k=4096, n=4096, act="none", bias=False, x="bf16",
             out="bf16"),
        # one small image: 24 x 24 patches and one more token, a width that is no multiple of 16
        dict(name="linear ragged", kind="linear", rows=577, k=1000, n=1153, act="relu", bias=True, x="fp32",
             out="fp32"),
        # the encoder's MLP input projection on 64 image pairs
        dict(name="linear image batch", kind="linear", rows=98304, k=1024, n=4096, act="gelu", bias=True, x="fp16",
             out="fp16"),
        # the entry of an encoder block: one pair, and 32 pairs
        dict(name="block one pair", kind="block", seqs=2, grid_h=24, grid_w=32, dim=1024, norm="layer",
             stream="fp32", branch="fp16"),
        dict(name="block 32 pairs", kind="block", seqs=64, grid_h=24, grid_w=32, dim=1024, norm="layer",
             stream="fp32", branch="fp16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["rope", "norm", "linear", "block"])
    if kind == "rope":
        dim = rng.choice([32, 48, 64, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
        rot -= rot % 4
        kv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        heads = kv * rng.choice([1, 1, 2, 4, 8])
        most = 128 * 768 * 2 * 16 * 64 // ((heads + kv) * dim)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        total = log_int(1, most // (2 if dtype == "fp32" else 1))
        batch = min(total, log_int(1, 64))
        axes = rng.choice([1, 1, 1, 2])
        scaling = rng.choice(["none", "linear", "ntk", "by_parts"]) if axes == 1 else "none"
        return dict(kind=kind, batch=batch, tokens=max(1, total // batch), heads=heads, kv_heads=kv, dim=dim, rot=rot,
                    interleaved=rng.random() < 0.5, axes=axes, scaling=scaling,
                    factor=round(rng.uniform(1.5, 32.0), 2) if scaling != "none" else 1.0,
                    far=0 if axes == 2 else log_int(1, 1000000), dtype=dtype, packed=rng.random() < 0.5)
    if kind == "norm":
        dim = log_int(32, 8192)
        dim -= rng.choice([0, dim % 8, dim % 8, dim % 64 if dim >= 64 else 0])
        stream = rng.choice(["fp32", "bf16", "fp16"])
        most = 98304 * 1024 // dim
        gates = rng.choice([0, 1, rng.randint(2, 16)])
        rows = log_int(1, most)
        if gates > 1:
            rows = max(1, rows // gates) * gates
            if rows > most:
                gates = 1
                rows = most
        return dict(kind=kind, rows=rows, dim=dim, norm=rng.choice(["layer", "rms"]),
                    post=rng.choice(["none", "layer", "rms"]), gates=gates, bias=rng.random() < 0.5, stream=stream,
                    branch=rng.choice(["bf16", "fp16"]), out=rng.choice(["bf16", "fp16"]),
                    residual_scale=rng.choice([1.0, round(rng.uniform(0.3, 1.2), 3)]))
    if kind == "linear":
        while True:
            k, n = log_int(64, 16384), log_int(64, 16384)
            k -= rng.choice([0, k % 16, k % 64])
            n -= rng.choice([0, n % 8, n % 64])
            rows = log_int(1, 98304)
            if rows * k * n <= 98304 * 1024 * 4096 and rows * (k + n) <= 98304 * 5120:
                break
        return dict(kind=kind, rows=rows, k=k, n=n, act=rng.choice(["none", "gelu", "relu"]), bias=rng.random() < 0.5,
                    x=rng.choice(["bf16", "fp16", "fp32"]), out=rng.choice(["bf16", "fp16", "bf16", "fp32"]))
    dim = 64 * rng.choice([6, 8, 12, 14, 16])
    gh, gw = rng.randint(1, 36), rng.randint(1, 36)
    seqs = log_int(1, max(1, 64 * 768 * 1024 * 1024 // (gh * gw * dim * dim)))
    return dict(kind=kind, seqs=min(seqs, 2048), grid_h=gh, grid_w=gw, dim=dim, norm=rng.choice(["layer", "rms"]),
                stream=rng.choice(["fp32", "bf16"]), branch=rng.choice(["bf16", "fp16"]))


# ----------------------------------------------------------------------------- inputs
def frequencies(rot, base, scaling, factor, axes):
    """Radians a position of each pair in 64 bits, and the amplitude of the rotated values."""
    per_axis = rot // 2 // axes
    i = torch.arange(per_axis, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk":  # the base grows so that the slowest pair slows down by `factor`
        base = base * factor ** (rot / (rot - 2)) if rot > 2 else base
    f = base ** (-i / per_axis)
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":  # slow pairs are interpolated, fast ones kept, a ramp between 1 and 32 turns
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f.repeat(axes).to(DEVICE), amplitude


def grid_positions(h, w):
    y = torch.arange(h, device=DEVICE).view(h, 1).expand(h, w).reshape(-1)
    x = torch.arange(w, device=DEVICE).view(1, w).expand(h, w).reshape(-1)
    return torch.stack([y, x])


def quantized_weight(g, n, k):
    """Weights in 8 bits with a scale for each output channel, rows laid out on 16-byte boundaries."""
    w = torch.randn(n, k, generator=g, device=DEVICE).clamp_(-2, 2) * (0.5 / math.sqrt(k))
    scale = w.abs().amax(1) / 127
    q = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device=DEVICE)[:, :k]
    q.copy_((w / scale[:, None]).round())
    return q, scale


def affine(g, dim, bias):
    w = 1 + 0.1 * torch.randn(dim, generator=g, device=DEVICE)
    return w, 0.1 * torch.randn(dim, generator=g, device=DEVICE) if bias else None


def activations(g, rows, dim, dtype):
    """Values as a stream holds them: a few channels much larger than the rest."""
    loud = torch.exp(0.5 * torch.randn(dim, generator=g, device=DEVICE))
    return (torch.randn(rows, dim, generator=g, device=DEVICE) * loud).to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    c = dict(case)
    kind = c["kind"]
    s = {"case": c}
    if kind == "rope":
        b, t, h, kv, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        dt = DTYPES[c["dtype"]]
        if c["packed"]:  # views of one projection's output
            qkv = torch.randn(b, t, h + 2 * kv, d, generator=g, device=DEVICE).to(dt)
            s["q"], s["k"] = qkv[:, :, :h], qkv[:, :, h:h + kv]
        else:
            s["q"] = torch.randn(b, t, h, d, generator=g, device=DEVICE).to(dt)
            s["k"] = torch.randn(b, t, kv, d, generator=g, device=DEVICE).to(dt)
        s["inv_freq"], s["amplitude"] = frequencies(c["rot"], 100.0 if c["axes"] == 2 else 10000.0, c["scaling"],
                                                    c["factor"], c["axes"])
        if c["axes"] == 2:
            w = math.isqrt(t)
            s["positions"] = grid_positions(-(-t // w), w)[:, :t].contiguous()
        else:  # every sequence at a place of its own
            first = torch.randint(0, c["far"] + 1, (b, 1), generator=g, device=DEVICE)
            s["positions"] = first + torch.arange(t, device=DEVICE)
    elif kind == "norm":
        r, d = c["rows"], c["dim"]
        s["x"] = activations(g, r, d, c["stream"])
        s["y"] = activations(g, r, d, c["branch"])
        s["weight"], s["bias"] = affine(g, d, c["bias"])
        s["post_weight"], s["post_bias"] = affine(g, d, c["bias"]) if c["post"] != "none" else (None, None)
        s["gate"] = None
        if c["gates"] == 1:
            s["gate"] = 0.2 * torch.randn(d, generator=g, device=DEVICE)
        elif c["gates"] > 1:
            s["gate"] = 0.2 * torch.randn(c["gates"], d, generator=g, device=DEVICE)
    elif kind == "linear":
        s["x"] = activations(g, c["rows"], c["k"], c["x"])
        if c["rows"] >= 64:
            s["x"][-3:] = 0  # rows of padding behind the last image
        s["wq"], s["ws"] = quantized_weight(g, c["n"], c["k"])
        s["bias"] = 0.1 * torch.randn(c["n"], generator=g, device=DEVICE) if c["bias"] else None
    else:
        d, rows = c["dim"], c["seqs"] * c["grid_h"] * c["grid_w"]
        s["x"] = activations(g, rows, d, c["stream"])
        s["y"] = activations(g, rows, d, c["branch"])
        s["gate"] = 0.2 * torch.randn(d, generator=g, device=DEVICE)
        s["weight"], s["bias"] = affine(g, d, c["norm"] == "layer")
        s["wq"], s["ws"] = quantized_weight(g, 3 * d, d)
        s["qkv_bias"] = 0.1 * torch.randn(3 * d, generator=g, device=DEVICE)
        s["inv_freq"], s["amplitude"] = frequencies(64, 100.0, "none", 1.0, 2)
        s["positions"] = grid_positions(c["grid_h"], c["grid_w"])
    return s


# ----------------------------------------------------------------------------- plain forms
def plain_rope(x, positions, inv_freq, amplitude, interleaved, axes, dtype):
    """x [batch, tokens, heads, dim]; positions [tokens], [batch, tokens] or [2, tokens] with two axes."""
    half = inv_freq.numel()
    if axes == 2:  # the first half of the pairs turns with the row, the second with the column
        p = positions.double().repeat_interleave(half // 2, 0).t()[None]
    else:
        p = positions.double().reshape(-1, positions.shape[-1], 1)
    angle = (p * inv_freq).unsqueeze(2)
    c, s = (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()
    out = x.float().clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2].float(), x[..., 1:2 * half:2].float()
        out[..., 0:2 * half:2] = a * c - b * s
        out[..., 1:2 * half:2] = a * s + b * c
    else:
        a, b = x[..., :half].float(), x[..., half:2 * half].float()
        out[..., :half] = a * c - b * s
        out[..., half:2 * half] = a * s + b * c
    return out.to(dtype)


def plain_norm(t, kind, weight, bias):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * weight
    return t if bias is None else t + bias


def plain_quantize(x):
    """Nearest of 255 levels and the level's size for each row; in 64 bits, where a value halfway
    between two levels is met exactly."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    return torch.where(a > 0, x * 127 / a, 0).round().float(), (a / 127).float()


def plain_linear(q, s, wq, ws, bias, act, dtype):
    y = (q @ wq.float().t()) * s * ws
    if bias is not None:
        y = y + bias
    if act == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif act == "relu":
        y = y.clamp_min(0)
    return y.to(dtype)


def plain_residual(s, post="none", residual_scale=1.0):
    y = s["y"].float()
    if post != "none":
        y = plain_norm(y, post, s["post_weight"], s["post_bias"])
    g = s["gate"]
    if g is not None:
        y = (y.view(g.shape[0], -1, y.shape[-1]) * g[:, None]).view(y.shape) if g.dim() == 2 else y * g
    return residual_scale * s["x"].float() + y


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        from mast3r_runtime_b200 import ops

        if kind == "rope":
            return ops.rope(s["q"], s["k"], s["positions"], s["inv_freq"], amplitude=s["amplitude"],
                            interleaved=c["interleaved"], axes=c["axes"])
        if kind == "norm":
            return ops.residual_norm(s["x"], s["y"], s["weight"], s["bias"], norm=c["norm"],
                                     post_norm=None if c["post"] == "none" else c["post"],
                                     post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                                     residual_scale=c["residual_scale"], out_dtype=DTYPES[c["out"]])
        if kind == "linear":
            return ops.int8_linear(s["x"], s["wq"], s["ws"], s["bias"], act=c["act"], out_dtype=DTYPES[c["out"]])
        x, q, scale = ops.residual_norm(s["x"], s["y"], s["weight"], s["bias"], norm=c["norm"], gate=s["gate"],
                                        out_dtype=torch.int8)
        qkv = ops.int8_linear(q, s["wq"], s["ws"], s["qkv_bias"], x_scale=scale, out_dtype=DTYPES[c["branch"]])
        qkv = qkv.view(c["seqs"], c["grid_h"] * c["grid_w"], 3, c["dim"] // 64, 64)
        return x, *ops.rope(qkv[:, :, 0], qkv[:, :, 1], s["positions"], s["inv_freq"], axes=2), qkv[:, :, 2]
    if kind == "rope":
        how = (s["positions"], s["inv_freq"], s["amplitude"], c["interleaved"], c["axes"], DTYPES[c["dtype"]])
        return plain_rope(s["q"], *how), plain_rope(s["k"], *how)
    if kind == "norm":
        r = plain_residual(s, c["post"], c["residual_scale"])
        return r.to(DTYPES[c["stream"]]), plain_norm(r, c["norm"], s["weight"], s["bias"]).to(DTYPES[c["out"]])
    if kind == "linear":
        return plain_linear(*plain_quantize(s["x"]), s["wq"], s["ws"], s["bias"], c["act"], DTYPES[c["out"]])
    dt = DTYPES[c["branch"]]
    r = plain_residual(s)
    h = plain_norm(r, c["norm"], s["weight"], s["bias"])
    qkv = plain_linear(*plain_quantize(h), s["wq"], s["ws"], s["qkv_bias"], "none", dt)
    qkv = qkv.view(c["seqs"], c["grid_h"] * c["grid_w"], 3, c["dim"] // 64, 64)
    how = (s["positions"], s["inv_freq"], 1.0, False, 2, dt)
    return r.to(DTYPES[c["stream"]]), plain_rope(qkv[:, :, 0], *how), plain_rope(qkv[:, :, 1], *how), qkv[:, :, 2]


# ----------------------------------------------------------------------------- work
def work(case):
    c, kind = case, case["kind"]
    if kind == "rope":
        tokens = c["batch"] * c["tokens"]
        values = tokens * (c["heads"] + c["kv_heads"]) * c["dim"]
        places = 2 * c["tokens"] if c["axes"] == 2 else tokens
        return {"bytes": 2 * values * SIZES[c["dtype"]] + 8 * places + 4 * c["rot"],
                "flops": 3 * tokens * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if kind == "norm":
        n = c["rows"] * c["dim"]
        vectors = 1 + c["gates"] + c["bias"] + (c["post"] != "none") * (1 + c["bias"])
        return {"bytes": n * (2 * SIZES[c["stream"]] + SIZES[c["branch"]] + SIZES[c["out"]]) + 4 * vectors * c["dim"],
                "flops": n * (10 if c["post"] == "none" else 17)}
    if kind == "linear":
        m, k, n = c["rows"], c["k"], c["n"]
        return {"bytes": m * k * SIZES[c["x"]] + n * k + 4 * n * (1 + c["bias"]) + m * n * SIZES[c["out"]],
                "flops": 2 * m * n * k}
    d, rows = c["dim"], c["seqs"] * c["grid_h"] * c["grid_w"]
    bytes_ = rows * d * (2 * SIZES[c["stream"]] + 4 * SIZES[c["branch"]]) + 3 * d * d + 4 * (6 + 3) * d
    return {"bytes": bytes_, "flops": 2 * rows * d * 3 * d + 14 * rows * d + 6 * rows * d}


# ----------------------------------------------------------------------------- exact values
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    c, kind = s["case"], s["case"]["kind"]

    def wide(v):
        return None if v is None else v.double()

    def turned(x, interleaved, axes):
        # each pair of values is one complex number, multiplied by amplitude * exp(i * angle)
        n = s["inv_freq"].numel()
        place = s["positions"].double()
        if axes == 2:
            angle = torch.cat([place[0, :, None] * s["inv_freq"][:n // 2], place[1, :, None] * s["inv_freq"][n // 2:]], 1)
            angle = angle[None]
        else:
            angle = place.unsqueeze(-1) * s["inv_freq"]
        turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, :, None]
        x = x.double()
        front, tail = x[..., :2 * n], x[..., 2 * n:]
        if interleaved:
            z = torch.view_as_complex(front.reshape(*front.shape[:-1], n, 2).contiguous()) * turn
            front = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(front[..., :n], front[..., n:]) * turn
            front = torch.cat([z.real, z.imag], -1)
        return torch.cat([front, tail], -1)

    def normed(t, how, weight, bias):
        if how == "layer":
            t = (t - t.mean(-1, keepdim=True)) / (t.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt()
        else:
            t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        t = t * wide(weight)
        return t + wide(bias) if bias is not None else t

    def stream(post, alpha):
        y = wide(s["y"])
        if post != "none":
            y = normed(y, post, s["post_weight"], s["post_bias"])
        if s["gate"] is not None:
            g = wide(s["gate"]).reshape(-1, y.shape[-1])
            y = y * g.repeat_interleave(y.shape[0] // g.shape[0], 0)
        return alpha * wide(s["x"]) + y

    def product(x, bias, act):
        largest = x.abs().max(-1, keepdim=True).values
        levels = (127 * x).div(largest).nan_to_num(0).round()  # a row of zeros is 0 / 0
        y = torch.mm(levels, wide(s["wq"]).t()) * (largest / 127) * wide(s["ws"])
        if bias is not None:
            y += wide(bias)
        if act == "gelu":  # x * sigmoid(2 u) is x / 2 * (1 + tanh(u))
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return torch.relu(y) if act == "relu" else y

    if kind == "rope":
        return turned(s["q"], c["interleaved"], c["axes"]), turned(s["k"], c["interleaved"], c["axes"])
    if kind == "norm":
        r = stream(c["post"], c["residual_scale"])
        return r, normed(r, c["norm"], s["weight"], s["bias"])
    if kind == "linear":
        return product(wide(s["x"]), s["bias"], c["act"])
    r = stream("none", 1.0)
    qkv = product(normed(r, c["norm"], s["weight"], s["bias"]), s["qkv_bias"], "none")
    qkv = qkv.view(c["seqs"], c["grid_h"] * c["grid_w"], 3, c["dim"] // 64, 64)
    return r, turned(qkv[:, :, 0], False, 2), turned(qkv[:, :, 1], False, 2), qkv[:, :, 2]
