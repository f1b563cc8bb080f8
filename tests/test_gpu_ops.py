"""GPU tests of the operators on device tensors (mast3r_runtime_b200.ops) against plain
implementations in 64 bits, at the sizes, layouts and values where they can go wrong.

Tolerances count roundings: `half(dtype)` is half a step of the result's type relative to the
value, U = 2^-24 one 32-bit rounding.  8-bit values and integer sums are compared exactly."""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from mast3r_runtime_b200 import ops as o

    return o


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def close(got, want, tol):
    """|got - want| <= tol everywhere (tol: a tensor of want's shape)."""
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3e}"


# ----------------------------------------------------------------------------- quantize_rows
def levels(x):
    """Exact levels and scales: 127 x and (2 n + 1) a are exact in 64 bits, and a quotient of two
    32-bit values that is no tie is further from it than a 64-bit rounding."""
    a = x.double().abs().amax(-1, keepdim=True)
    q = torch.where(a > 0, 127 * x.double() / a, 0).round()
    return q.to(torch.int8), (a / 127).float().squeeze(-1)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 127), (5, 256), (3, 513), (130, 1000), (67, 1024), (9, 1025),
                                       (300, 4096), (2, 8200), (3, 16384), (1, 16383), (700, 768), (2000, 1000),
                                       (9, 641), (5, 2345), (3, 5003)])
def test_quantize_rows(ops, dtype, rows, cols):
    x = rnd(rows, cols, seed=rows + cols, dtype=DT[dtype])
    q, s = ops.quantize_rows(x)
    wq, wsc = levels(x)
    assert torch.equal(q, wq)
    assert torch.equal(s, wsc)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


def test_quantize_ties_and_tiny_magnitudes(ops):
    # 127 x / a is exactly n + 1/2 for every value (a = 127 * 2^e), and its neighbours
    a = 127.0
    v = torch.arange(-126.5, 127, 1.0)
    near = torch.cat([v, torch.nextafter(v, torch.tensor(1e9)), torch.nextafter(v, torch.tensor(-1e9))])
    x = torch.cat([near, torch.tensor([a])]).repeat(4, 1)
    x *= torch.tensor([1.0, 2.0 ** -120, 2.0 ** 100, 2.0 ** -60])[:, None]
    x = torch.cat([x, torch.zeros(2, x.shape[1])])
    x[5, 3] = 2.0 ** -149  # the smallest magnitude there is
    x = x.cuda()
    q, s = ops.quantize_rows(x)
    wq, _ = levels(x)
    assert torch.equal(q, wq)
    assert int(q[4].abs().max()) == 0 and float(s[4]) == 0 and int(q[5, 3]) == 127


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_quantize_every_16_bit_value(ops, dtype):
    """Every finite value of the type up to a row's largest one, for largest ones with many ties
    (127 and 1 times powers of two), few, and at both ends of the type's range."""
    t = DT[dtype]
    bits = torch.arange(0, 2 ** 15, dtype=torch.int32).to(torch.int16).view(t)
    bits = bits[torch.isfinite(bits)]
    fi = torch.finfo(t)
    for a in (1.0, 127.0, 254.0, 3.0, 1.9, 0.01, fi.max, fi.tiny, fi.smallest_normal / 2 ** 5, 2.0 ** 15 * 1.25):
        a = torch.tensor(a).to(t)
        v = bits[(bits <= a) & (bits >= a.float() / 4096)]
        v = torch.cat([v, -v, a[None]])
        x = torch.zeros(-(-v.numel() // 4000), 4001, dtype=t)
        x[:, 0] = a  # the largest one in every row
        for i in range(x.shape[0]):
            part = v[i * 4000:(i + 1) * 4000]
            x[i, 1:1 + part.numel()] = part
        x = x.cuda()
        q, s = ops.quantize_rows(x)
        assert torch.equal(q, levels(x)[0]), float(a)


def test_quantize_non_finite_rows_and_strides(ops):
    base = rnd(6, 40, 96, seed=3, dtype=torch.bfloat16)
    x = base[:, ::2, 8:83]  # rows evenly spaced within a block of 20, not across blocks
    with pytest.raises(ValueError):
        ops.quantize_rows(base[:, 1:39:2, :].transpose(0, 1))
    x = base.view(240, 96)[::3, 5:80]
    q, s = ops.quantize_rows(x)
    wq, wsc = levels(x)
    assert torch.equal(q, wq) and torch.equal(s, wsc)
    y = rnd(4, 33, seed=4)
    y[0, 7] = math.inf
    y[1, 32] = math.nan
    y[2, 0] = -math.inf
    y[2, 1] = math.nan
    q, s = ops.quantize_rows(y)
    assert int(q[:3].abs().max()) == 0
    assert math.isinf(s[0]) and math.isnan(s[1]) and math.isnan(s[2])
    assert torch.equal(q[3], levels(y[3:])[0][0])
    w = torch.ones(5, 48, dtype=torch.int8, device="cuda")[:, :33]
    out = ops.int8_linear(y, w, torch.ones(5, device="cuda"), act="relu")
    assert torch.isnan(out[:3]).all() and torch.isfinite(out[3]).all()


# ----------------------------------------------------------------------------- int8_linear
def ints(rows, k, seed, extreme=False):
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.int8)
    q[:, :k] = 127 if extreme else torch.randint(-127, 128, (rows, k), generator=g, dtype=torch.int8)
    q[:, k:] = 99  # the padding must not count
    return q.cuda()[:, :k]


def act64(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y.clamp_min(0) if act == "relu" else y


def linear64(q, s, w, ws, bias, act, out_dtype):
    """(value, tolerance): the sum is exact; then one rounding to 32 bits, two scale products, the
    bias, the activation and the result's type."""
    p = (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()
    y = p + (bias.double() if bias is not None else 0)
    tol = 4 * U * p.abs() + U * y.abs()
    if act == "gelu":
        # the derivative of the activation is at most 1.13; its tanh: 2^-11 relative for 16-bit
        # results, 4 roundings of the argument and the tanh for 32-bit ones
        t = 2.0 ** -11 + 8 * U if out_dtype is not torch.float32 else 16 * U
        tol = 1.13 * tol + 0.5 * y.abs() * t + 4 * U * y.abs()
    z = act64(y, act)
    # 2^-25: half a step of fp16's smallest values
    return z, tol + half(out_dtype) * (z.abs() + tol) + 2.0 ** -25


SHAPES = [(1, 1, 1), (1, 5, 16), (1, 4096, 1024), (2, 130, 257), (3, 1153, 1000), (7, 64, 4096), (8, 1000, 33),
          (9, 300, 512), (16, 4096, 640), (17, 129, 2048), (24, 2048, 4096), (33, 520, 128), (64, 1000, 999),
          (65, 96, 384), (128, 1152, 384), (129, 257, 129), (577, 1153, 1000), (1536, 2304, 768), (2500, 4100, 1040),
          (20000, 1040, 768), (19500, 1501, 1000), (26001, 600, 70), (220, 360, 11869), (452, 961, 2880), (1000, 130, 16384),
          (43, 316, 80), (129, 128, 4096)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", ["fp32", "bf16"])
def test_int8_linear_exact_sums(ops, m, n, k, out):
    q, w = ints(m, k, m + n), ints(n, k, n + k)
    s, ws = rnd(m, seed=5).abs() + 0.1, rnd(n, seed=6).abs() * 1e-4
    y = ops.int8_linear(q, w, ws, x_scale=s, out_dtype=DT[out])
    want, tol = linear64(q, s, w, ws, None, "none", DT[out])
    close(y, want, tol)


@pytest.mark.parametrize("m", [1, 4, 12, 40, 200, 700])
@pytest.mark.parametrize("x", DT)
@pytest.mark.parametrize("out,act,bias", [("fp16", "gelu", True), ("fp32", "gelu", True), ("bf16", "relu", False)])
def test_int8_linear_quantises_its_rows(ops, m, x, out, act, bias):
    k, n = 520, 333
    xs = rnd(m, k, seed=m, dtype=DT[x])
    if m > 1:
        xs[-1] = 0  # a row of padding
    w, ws = ints(n, k, 2), rnd(n, seed=6).abs() * 2e-4
    b = rnd(n, seed=8) if bias else None
    y = ops.int8_linear(xs, w, ws, b, act=act, out_dtype=DT[out])
    q, s = levels(xs)
    want, tol = linear64(q, s, w, ws, b, act, DT[out])
    close(y, want, tol)


@pytest.mark.parametrize("m,n,k", [(1, 40, 16384), (5, 130, 131071), (200, 130, 131071), (200, 130, 131056)])
@pytest.mark.parametrize("least", [False, True])
def test_int8_linear_largest_sums(ops, m, n, k, least):
    q, w = ints(m, k, 0, extreme=True), ints(n, k, 0, extreme=True)  # sums of 127^2 k, up to 2.1e9
    top = 128.0 if least else 127.0
    if least:
        q.fill_(-128), w.fill_(-128)
    one = torch.ones(max(m, n), device="cuda")
    y = ops.int8_linear(q, w, one[:n], x_scale=one[:m], out_dtype=torch.float32)
    assert (y.double() - top ** 2 * k).abs().max() <= U * top ** 2 * k


def test_int8_linear_layouts(ops):
    """Leading dimensions, strided rows of x, outputs that TMA cannot store, unaligned vectors."""
    k, n = 256, 77
    w = ints(n, k, 1)
    ws = (rnd(n + 1, seed=2).abs() * 1e-3)[1:]
    b = rnd(n + 1, seed=3)[1:]
    base = rnd(4, 50, 2 * k, seed=4, dtype=torch.float16)
    x = base[:, :, k - 3:2 * k - 3]
    for m in (x, x[:1, :3], x[2, 7]):
        y = ops.int8_linear(m, w, ws, b, act="none", out_dtype=torch.float32)
        flat = m.reshape(-1, k)
        q, s = levels(flat)
        want, tol = linear64(q, s, w, ws, b, "none", torch.float32)
        assert y.shape == (*m.shape[:-1], n)
        close(y.reshape(-1, n), want, tol)
    assert ops.int8_linear(x[:, :0], w, ws).shape == (4, 0, n)


# ----------------------------------------------------------------------------- residual_norm
def norm64(t, kind, w, b, eps=1e-6):
    """(value, error of 32-bit statistics): sums of at most 32 values a thread and 10 joins."""
    mean = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[..., :1])
    d = t - mean
    r = 1 / (d.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    w = torch.ones_like(t[0]) if w is None else w.double()
    v = d * r * w
    err = 64 * U * (v.abs() + t.abs().mean(-1, keepdim=True) * r * w.abs())
    if b is not None:
        v = v + b.double()
    return v, err + U * v.abs(), r * w.abs()


def residual64(x, y, gate, alpha, post, pw, pb):
    r = alpha * x.double()
    tol = 2 * U * r.abs()
    if y is not None:
        t = y.double()
        et = torch.zeros_like(t)
        if post:
            t, et, _ = norm64(t, post, pw, pb)
        g = torch.ones(1, t.shape[-1], dtype=torch.float64, device=t.device) if gate is None else gate.double()
        g = g.reshape(-1, t.shape[-1])
        g = g.repeat_interleave(t.shape[0] // g.shape[0], 0) if g.shape[0] > 1 else g
        tol = tol + (g * et).abs() + 2 * U * (g * t).abs()
        r = r + g * t
    return r, tol + U * r.abs()


def check_residual(ops, x, y, w, b, norm, out, **kw):
    xf, yf = x.reshape(-1, x.shape[-1]), None if y is None else y.reshape(-1, x.shape[-1])
    want_r, er = residual64(xf, yf, kw.get("gate"), np.float32(kw.get("residual_scale", 1.0)).item(),
                            kw.get("post_norm"), kw.get("post_weight"), kw.get("post_bias"))
    r, h = ops.residual_norm(x, y, w, b, norm=norm, out_dtype=out, **kw)
    # 2^-25: half a step of fp16's smallest values
    close(r.reshape(want_r.shape), want_r, er + half(x.dtype) * (want_r.abs() + er) + 2.0 ** -25)
    want_h, eh, slope = norm64(want_r, norm, w, b)
    # an error e of r moves h by slope e, and through the statistics by at most twice slope max(e) more
    eh = eh + slope * (er + 2 * (1 + want_h.abs().amax(-1, keepdim=True)) * er.amax(-1, keepdim=True))
    close(h.reshape(want_r.shape), want_h, eh + half(h.dtype) * (want_h.abs() + eh) + 2.0 ** -25)
    return r, h


@pytest.mark.parametrize("rows,cols", [(1, 1), (9, 8), (1003, 32), (70, 31), (41, 64), (77, 100), (35, 128), (3, 33),
                                       (4, 256), (7, 384), (130, 1000), (65, 1001), (64, 1024),
                                       (5, 1032), (301, 4096), (2, 4096), (3, 8191), (2, 16384), (7, 641), (9, 1155),
                                       (4, 1501), (5, 2345), (6, 3333), (3, 5003), (2, 9001), (5000, 552), (800, 768)])
@pytest.mark.parametrize("norm,post", [("layer", None), ("rms", "rms"), ("layer", "layer")])
def test_residual_norm(ops, rows, cols, norm, post):
    seed = rows * 7 + cols
    names = list(DT)
    xd, yd, od = names[seed % 3], names[(seed + 1) % 3], names[(seed // 3) % 3]
    x, y = rnd(rows, cols, seed=seed, dtype=DT[xd], scale=3), rnd(rows, cols, seed=seed + 1, dtype=DT[yd])
    w, b = 1 + 0.1 * rnd(cols, seed=1), 0.1 * rnd(cols, seed=2)
    kw = dict(post_norm=post, post_weight=0.5 + rnd(cols, seed=3).abs(), post_bias=rnd(cols, seed=4)) if post else {}
    check_residual(ops, x, y, w, b if norm == "layer" else None, norm, DT[od], gate=rnd(cols, seed=5),
                   residual_scale=0.75, **kw)


@pytest.mark.parametrize("per,groups", [(1, 6), (3, 2), (6, 1), (7, 1), (2 ** 32 - 1, 1), (2 ** 32, 1), (2 ** 33 + 2, 1)])
def test_rows_of_a_gate_through_the_c_abi(ops, per, groups):
    """Groups longer than the rows, past 32 bits too, are one group."""
    from test_ops_args import RESIDUAL

    from mast3r_runtime_b200 import _lib

    rows, cols = 6, 40
    x, y, gate = rnd(rows, cols, seed=1), rnd(rows, cols, seed=2), rnd(groups, cols, seed=3)
    r, h = torch.empty_like(x), torch.empty_like(x)
    lib = _lib.load()
    args = RESIDUAL.pack(0, 2, 2, 2, 1, 0, 1e-6, 1.0, rows, cols, cols, cols, cols, cols, per, cols, x.data_ptr(),
                         y.data_ptr(), gate.data_ptr(), 0, 0, 0, 0, r.data_ptr(), h.data_ptr(), 0,
                         torch.cuda.current_stream().cuda_stream)
    assert lib.m3r_residual_norm(args) == 0, lib.m3r_global_error()
    r2, h2 = ops.residual_norm(x, y, None, gate=gate)
    assert torch.equal(r, r2) and torch.equal(h, h2)
    rows_gate = gate.double().repeat_interleave(rows // groups, 0)
    assert (r.double() - (x.double() + rows_gate * y.double())).abs().max() <= 2 * U * (1 + 25)


@pytest.mark.parametrize("rows,cols,stream,branch", [(2400, 1536, "fp32", "bf16"), (1300, 4096, "bf16", "fp16"),
                                                     (300, 16384, "fp32", "fp32"), (640, 8192, "fp16", "fp16"),
                                                     (5000, 1024, "fp32", "bf16"), (4801, 776, "fp32", "fp32"),
                                                     (1300, 1000, "bf16", "bf16")])
def test_residual_norm_many_long_rows(ops, rows, cols, stream, branch):
    """More rows than blocks fit the device: each block works through several, some copied ahead."""
    x, y = rnd(rows, cols, seed=1, dtype=DT[stream]), rnd(rows, cols, seed=2, dtype=DT[branch])
    w, b = 1 + 0.1 * rnd(cols, seed=1), 0.1 * rnd(cols, seed=2)
    r, h = check_residual(ops, x, y, w, b, "layer", DT[branch], gate=rnd(cols, seed=5), post_norm="rms")
    x2 = x.clone()
    r2, h2 = ops.residual_norm(x2, y, w, b, norm="layer", out_dtype=DT[branch], gate=rnd(cols, seed=5), post_norm="rms",
                               inplace=True)
    assert r2 is x2 and torch.equal(r2, r) and torch.equal(h2, h)
    q, s = ops.quantize_rows(x)
    wq, wsc = levels(x)
    assert torch.equal(q, wq) and torch.equal(s, wsc)
    _, h3 = ops.residual_norm(x, None, w, None, norm="rms", out_dtype=torch.float32)
    _, q3, s3 = ops.residual_norm(x, None, w, None, norm="rms", out_dtype=torch.int8)
    assert torch.equal(q3, levels(h3)[0]) and torch.equal(s3, levels(h3)[1])


@pytest.mark.parametrize("stream", DT)
@pytest.mark.parametrize("branch", DT)
def test_residual_norm_types_and_gates(ops, stream, branch):
    x, y = rnd(6, 50, 200, seed=1, dtype=DT[stream]), rnd(6, 50, 200, seed=2, dtype=DT[branch])
    w = 1 + 0.1 * rnd(200, seed=1)
    check_residual(ops, x, y, w, None, "rms", DT[branch], gate=rnd(6, 200, seed=5))
    check_residual(ops, x, None, w, None, "rms", DT[stream], residual_scale=2.0)
    check_residual(ops, x, y, None, None, "layer", torch.float32)
    # strided rows, unaligned starts, in place
    wide = rnd(40, 777, seed=9, dtype=DT[stream])
    view = wide[::2, 5:405]
    keep = wide.clone()
    y2 = rnd(20, 400, seed=3, dtype=DT[branch])
    r, h = ops.residual_norm(view.clone(), y2, None)
    r2, h2 = ops.residual_norm(view, y2, None, inplace=True)
    # rows off the 16-byte grid are summed in another order: both results lie within norm64's
    # bound of the exact one, so within twice that of each other
    want, eh, slope = norm64(residual64(r0 := keep[::2, 5:405], y2, None, 1.0, None, None, None)[0], "layer", None, None)
    er = 2 * U * (r0.double().abs() + y2.double().abs())
    eh = eh + slope * (er + 2 * (1 + want.abs().amax(-1, keepdim=True)) * er.amax(-1, keepdim=True))
    assert r2 is view and torch.equal(r2, r)
    close(h2, h.double(), 2 * (eh + half(h.dtype) * (want.abs() + eh) + 2.0 ** -25))
    keep[::2, 5:405] = r
    assert torch.equal(wide, keep)  # nothing beside the rows was written


@pytest.mark.parametrize("cols", [24, 64, 65, 120, 768, 769, 1000, 1001, 3333, 4096])
def test_residual_norm_in_8_bits(ops, cols):
    x, y = rnd(33, cols, seed=1), rnd(33, cols, seed=2, dtype=torch.bfloat16)
    x[5] = 0
    y[5] = 0
    w, b = 1 + 0.1 * rnd(cols, seed=1), None
    r, h = ops.residual_norm(x, y, w, b, out_dtype=torch.float32)
    r2, q, s = ops.residual_norm(x, y, w, b, out_dtype=torch.int8)
    wq, wsc = levels(h)  # the same kernel's 32-bit result, quantised exactly
    assert torch.equal(r, r2) and torch.equal(q, wq) and torch.equal(s, wsc)
    assert float(s[5]) == 0 and int(q[5].abs().max()) == 0
    assert q.stride(0) % 16 == 0


# ----------------------------------------------------------------------------- rope
def rope64(x, pos, f, amplitude, interleaved, axes):
    """(value, tolerance) for x [batch, tokens, heads, dim], pos [axes, batch or 1, tokens]."""
    n = f.numel()
    p = pos.double()
    a = p[0][..., None] * f
    if axes == 2:
        a = torch.cat([p[0][..., None] * f[:n // 2], p[1][..., None] * f[n // 2:]], -1)
    a = a.unsqueeze(2)
    c, s = amplitude * a.cos(), amplitude * a.sin()
    out = x.double().clone()
    tol = torch.zeros_like(out)
    i = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    j = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    u, v = x[..., i].double(), x[..., j].double()
    out[..., i], out[..., j] = u * c - v * s, u * s + v * c
    # the fraction of a turn in 32 bits (pi U of the angle, as half a turn is pi), 2 steps of sine
    # and cosine, and 4 roundings of products and sum
    e = amplitude * (u.abs() + v.abs()) * (math.pi + 4 + 4) * U
    tol[..., i] = tol[..., j] = e + half(x.dtype) * e
    tol[..., :2 * n] += half(x.dtype) * out[..., :2 * n].abs() + (2.0 ** -25 if x.dtype is torch.float16 else 0)
    return out, tol


@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (96, 48), (80, 20), (50, 36), (33, 32), (256, 192), (4, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DT)
def test_rope(ops, dim, rot, interleaved, dtype):
    f, amp = ops.rope_frequencies(rot, scaling="by_parts", factor=4.0)
    for b, t, h, kv in ((1, 1, 3, 1), (2, 37, 4, 2), (3, 211, 1, 5)):
        q, k = rnd(b, t, h, dim, seed=1, dtype=DT[dtype]), rnd(b, t, kv, dim, seed=2, dtype=DT[dtype])
        pos = torch.randint(-1000, 1000000, (b, t), generator=torch.Generator().manual_seed(t)).cuda()
        oq, ok = ops.rope(q, k, pos, f, amplitude=amp, interleaved=interleaved)
        for x, o in ((q, oq), (k, ok)):
            want, tol = rope64(x, pos[None], f, amp, interleaved, 1)
            close(o, want, tol)
            assert torch.equal(o[..., rot:], x[..., rot:])


def test_rope_far_positions_and_shared_ones(ops):
    f, _ = ops.rope_frequencies(64, scaling="linear", factor=2.0)
    x = rnd(3, 16, 2, 64, seed=1)
    far = 2 ** 31 - 17
    pos = torch.arange(16, dtype=torch.int32).cuda() + (far - 15)
    o, none = ops.rope(x, None, pos, f)
    assert none is None
    want, tol = rope64(x, pos[None, None], f, 1.0, False, 1)
    # 2^31 turns of 2^-53 relative: 2^-22 / 2 pi of the angle on each side of the comparison
    tol = tol + (x.abs().amax(-1, keepdim=True) * 2.0 * 2 ** -22).double()
    close(o, want, tol)
    o3, _ = ops.rope(x[1], None, pos, f)
    assert torch.equal(o3, o[1])
    assert ops.rope(x[:, :0], None, pos[:0], f)[0].shape == (3, 0, 2, 64)


def test_rope_two_axes_match_the_models_rotation(ops):
    """The image tokens' rotation of the model's oracle (rope2d.py:133-146)."""
    from oracle import model

    f, _ = ops.rope_frequencies(64, base=100.0, axes=2)
    h, w, heads = 5, 7, 3
    y, x = torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij")
    pos = torch.stack([y.reshape(-1), x.reshape(-1)]).cuda()
    t = rnd(2, h * w, heads, 64, seed=3)
    o, _ = ops.rope(t, None, pos, f, axes=2)
    want, tol = rope64(t, pos[:, None], f, 1.0, False, 2)
    close(o, want, tol)
    cos, sin = model.rope_tables(model.positions(h, w), 64)
    r = model.rope(t.cpu().numpy().astype(np.float64).transpose(0, 2, 1, 3), cos, sin)
    # the oracle's angles (up to 7: a power, a reciprocal and a product in 32 bits, 6 roundings),
    # sines and cosines (2) are 32-bit values, and each result has two of them
    slack = (7 * 6 + 2) * U * 2 * float(t.abs().max())
    np.testing.assert_allclose(o.cpu().numpy().transpose(0, 2, 1, 3), r, rtol=0, atol=float(tol.max()) + slack)


def test_rope_views_planes_and_in_place(ops):
    f, _ = ops.rope_frequencies(64)
    b, t, h = 2, 45, 4
    qkv = rnd(b, t, 3, h, 64, seed=5, dtype=torch.bfloat16)
    keep = qkv.clone()
    pos = torch.arange(t, device="cuda")
    q, k, v = qkv.unbind(2)
    oq, ok = ops.rope(q, k, pos, f)
    want, tol = rope64(q, pos[None, None], f, 1.0, False, 1)
    close(oq, want, tol)
    planes = [torch.zeros(b, h, t, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.rope(q, k, pos, f, out=[p.transpose(1, 2) for p in planes])
    assert torch.equal(planes[0].transpose(1, 2), oq) and torch.equal(planes[1].transpose(1, 2), ok)
    assert torch.equal(qkv, keep)
    iq, ik = ops.rope(q, k, pos, f, inplace=True)
    assert iq is q and torch.equal(q, oq) and torch.equal(ik, ok) and torch.equal(v, keep[:, :, 2])


# ----------------------------------------------------------------------------- streams, graphs, chains
def block_entry(ops, s):
    x, h, sc = ops.residual_norm(s["x"], s["y"], s["w"], s["b"], gate=s["gate"], out_dtype=torch.int8)
    qkv = ops.int8_linear(h, s["wq"], s["ws"], s["bias"], x_scale=sc, out_dtype=torch.float16)
    q, k, v = qkv.view(2, -1, 3, 4, 64).unbind(2)
    q, k = ops.rope(q, k, s["pos"], s["f"], axes=2)
    return x, q, k, v


def block_state(ops, seed, grid=(6, 8)):
    d, t = 256, grid[0] * grid[1]
    wq, ws = ops.quantize_weight(rnd(3 * d, d, seed=seed, scale=d ** -0.5))
    yy, xx = torch.meshgrid(torch.arange(grid[0]), torch.arange(grid[1]), indexing="ij")
    return dict(x=rnd(2 * t, d, seed=seed), y=rnd(2 * t, d, seed=seed + 1, dtype=torch.float16),
                w=1 + 0.1 * rnd(d, seed=2), b=rnd(d, seed=3), gate=rnd(d, seed=4), wq=wq, ws=ws,
                bias=rnd(3 * d, seed=5), pos=torch.stack([yy.reshape(-1), xx.reshape(-1)]).cuda(),
                f=ops.rope_frequencies(64, base=100.0, axes=2)[0])


@pytest.mark.parametrize("grid", [(1, 1), (6, 8), (24, 32)])
def test_block_entry_chain(ops, grid):
    s = block_state(ops, 11, grid)
    x, q, k, v = block_entry(ops, s)
    r, er = residual64(s["x"], s["y"], s["gate"], 1.0, None, None, None)
    close(x, r, er + half(x.dtype) * r.abs())
    # from the operator's own 8-bit rows on, the rest is checked exactly as each operator is
    _, hq, hs = ops.residual_norm(s["x"], s["y"], s["w"], s["b"], gate=s["gate"], out_dtype=torch.int8)
    want, tol = linear64(hq, hs, s["wq"], s["ws"], s["bias"], "none", torch.float16)
    shape = (2, -1, 3, 4, 64)
    close(v, want.view(shape)[:, :, 2], tol.view(shape)[:, :, 2])
    for i, o in ((0, q), (1, k)):
        t, e = want.view(shape)[:, :, i], tol.view(shape)[:, :, i]
        turned, et = rope64(t.half(), s["pos"][:, None], s["f"], 1.0, False, 2)
        # both halves of a pair carry the product's error and the one of t.half()
        slack = e + half(torch.float16) * t.abs() + 2.0 ** -25
        slack = slack + slack.roll(32, -1)
        close(o, turned, et + slack * (1 + half(torch.float16)))


def test_streams_and_graphs(ops):
    a, b = block_state(ops, 21), block_state(ops, 31)
    want_a, want_b = block_entry(ops, a), block_entry(ops, b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):  # two chains at once, each with its own workspace
        with torch.cuda.stream(s1):
            ga = block_entry(ops, a)
        with torch.cuda.stream(s2):
            gb = block_entry(ops, b)
        got.append((ga, gb))
    torch.cuda.synchronize()
    for ga, gb in got:
        assert all(torch.equal(i, j) for i, j in zip(ga, want_a)) and all(torch.equal(i, j) for i, j in zip(gb, want_b))
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block_entry(ops, s)
        graphs.append((g, out))
    for s, seed in ((a, 41), (b, 51)):
        s["x"].copy_(rnd(*s["x"].shape, seed=seed))
    want_a, want_b = block_entry(ops, a), block_entry(ops, b)
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(i, j) for i, j in zip(graphs[0][1], want_a))
    assert all(torch.equal(i, j) for i, j in zip(graphs[1][1], want_b))
    ops.status(0)


def test_same_inputs_give_the_same_bits(ops):
    s = block_state(ops, 61)
    first = block_entry(ops, s)
    for _ in range(5):
        assert all(torch.equal(i, j) for i, j in zip(first, block_entry(ops, s)))


def test_captured_behind_copies_fills_and_joined_streams(ops):
    """The kernels ahead of an operator may be no kernels (a copy, a fill) or several (a join)."""
    rows, k, n = 50, 512, 200
    src, x, y = rnd(rows, k, seed=1), torch.empty(rows, k, device="cuda"), torch.empty(rows, k, device="cuda")
    w, ws = ops.quantize_weight(rnd(n, k, seed=2))
    g1 = 1 + 0.1 * rnd(k, seed=3)
    pos = torch.arange(rows, device="cuda")
    freq = ops.rope_frequencies(100)[0]
    side = torch.cuda.Stream()

    def run():
        now = torch.cuda.current_stream()
        x.copy_(src)
        q0, _ = ops.quantize_rows(x)            # behind a copy
        y.zero_()
        r0, h0 = ops.residual_norm(x, y, g1)    # behind a fill
        side.wait_stream(now)
        with torch.cuda.stream(side):
            y.copy_(src)
            p0 = ops.int8_linear(h0, w, ws)
        z = x * 2
        now.wait_stream(side)
        r1, h1 = ops.residual_norm(z, y, g1)    # behind two kernels
        p1 = ops.int8_linear(h1, w, ws)
        t, _ = ops.rope(p1.view(rows, 2, 100), None, pos, freq)
        return q0, r0, h0, p0, r1, h1, p1, t

    want = [v.clone() for v in run()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for seed in (1, 7):
        src.copy_(rnd(rows, k, seed=seed))
        if seed != 1:
            want = [v.clone() for v in run()]
        x.fill_(9), y.fill_(9)
        for _ in range(3):
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows", [1, 3, 24, 100, 600, 20000])
def test_linear_captured_with_its_quantisation(ops, rows):
    """The product starts while the quantisation still runs; captured, replayed on new inputs and
    mixed with calls outside the graph, the results stay those of one call at a time."""
    k, n = 1000, 520
    x = rnd(rows, k, seed=rows, dtype=torch.bfloat16)
    wq, ws = ops.quantize_weight(rnd(n, k, seed=2, scale=k ** -0.5))
    b = rnd(n, seed=3)
    ops.int8_linear(x, wq, ws, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        first = ops.int8_linear(x, wq, ws, b, act="gelu")
        second = ops.int8_linear(x * 0.5, wq, ws, b)
    for seed in (7, 8):
        x.copy_(rnd(rows, k, seed=seed, dtype=torch.bfloat16))
        g.replay()
        mixed = ops.int8_linear(x, wq, ws, b, act="gelu")
        torch.cuda.synchronize()
        want = ops.int8_linear(x, wq, ws, b, act="gelu")
        half_x = ops.int8_linear(x * 0.5, wq, ws, b)
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(mixed, want) and torch.equal(second, half_x)
        q, s = levels(x)
        ref, tol = linear64(q, s, wq, ws, b, "gelu", torch.bfloat16)
        close(want, ref, tol)


def test_calls_start_behind_what_they_read(ops):
    """An operator may be launched before the kernel ahead of it has finished: inputs, weights and scales
    written just before it, by torch or by another operator, on one stream or joined from another,
    eagerly and in a graph, are the ones it reads; and what it writes over has been read."""
    n, k, m = 512, 1024, 2048
    big = rnd(4096, 4096, seed=1)
    side = torch.cuda.Stream()
    xs = [rnd(m, k, seed=10 + i, dtype=torch.bfloat16) for i in range(3)]
    wt = [rnd(n, k, seed=20 + i, scale=k ** -0.5) for i in range(3)]
    f, _ = ops.rope_frequencies(64)
    pos = torch.arange(m, device="cuda")
    x, w = torch.empty_like(xs[0]), torch.empty_like(wt[0])

    def chain(ops, i, rows):
        big @ big  # keeps the device busy, so that launches queue up
        x.copy_(xs[i])
        w.copy_(wt[i])
        wq, ws = ops.quantize_weight(w)  # read by the next call
        y = ops.int8_linear(x[:rows], wq, ws)
        q, s = ops.quantize_rows(x)
        wq2, ws2 = ops.quantize_weight(w * 2)
        z = ops.int8_linear(q[:rows], wq2, ws2, x_scale=s[:rows], out_dtype=torch.bfloat16)
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            t = z * 3
            r, h = ops.residual_norm(t, y, None)
        main.wait_stream(side)
        o, _ = ops.rope(h.view(rows, -1, 64), None, pos[:rows], f)
        r2, h2 = ops.residual_norm(o.view(rows, n), z, None, inplace=True)
        y.zero_()
        return y, z, r, h, o, h2

    def alone(fn):
        """fn with the device idle before and after."""
        def call(*a, **kw):
            torch.cuda.synchronize()
            r = fn(*a, **kw)
            torch.cuda.synchronize()
            return r

        return call

    slow = SimpleNamespace(**{name: alone(getattr(ops, name)) for name in ops.__all__})
    for rows in (1, 4, 20, 200, m):
        want = [[v.clone() for v in chain(slow, i, rows)] for i in range(3)]
        for _ in range(3):
            got = [chain(ops, i, rows) for i in range(3)]
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert all(torch.equal(u, v) for u, v in zip(a, b))
        graphs = []
        for i in range(3):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = chain(ops, i, rows)
            graphs.append((g, out))
        for _ in range(2):
            for g, _ in graphs:
                g.replay()
        torch.cuda.synchronize()
        for (_, a), b in zip(graphs, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing has to be set up before a capture."""
    import subprocess
    import sys

    from conftest import ROOT

    code = (
        "import torch\n"
        "from mast3r_runtime_b200 import ops\n"
        "x = torch.randn(300, 256, device='cuda').half(); w = torch.randn(128, 256, device='cuda')\n"
        "f, _ = ops.rope_frequencies(64); pos = torch.arange(300, device='cuda')\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    wq, ws = ops.quantize_weight(w)\n"
        "    r, h = ops.residual_norm(x, x, None)\n"
        "    y = ops.int8_linear(h, wq, ws)\n"
        "    q, _ = ops.rope(y.view(300, 2, 64), None, pos, f)\n"
        "    z = ops.int8_linear(x[:1], wq, ws); t = ops.int8_linear(x[:20], wq, ws)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "r2, h2 = ops.residual_norm(x, x, None)\n"
        "y2 = ops.int8_linear(h2, *ops.quantize_weight(w))\n"
        "assert torch.equal(y, y2) and torch.equal(q, ops.rope(y2.view(300, 2, 64), None, pos, f)[0])\n"
        "assert torch.equal(z, ops.int8_linear(x[:1], wq, ws)) and torch.equal(t, ops.int8_linear(x[:20], wq, ws))\n"
        "print('fine')\n")
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "fine" in out.stdout, out.stderr[-2000:]


def test_threads(ops):
    """Calls from several threads at once, each on its own stream."""
    import threading

    states = [block_state(ops, 100 + i) for i in range(4)]
    want = [block_entry(ops, s) for s in states]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = block_entry(ops, states[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_another_device_than_the_current_one(ops):
    s = {k: v.to("cuda:1") if torch.is_tensor(v) else v for k, v in block_state(ops, 71).items()}
    want = block_entry(ops, block_state(ops, 71))
    got = block_entry(ops, s)
    assert torch.cuda.current_device() == 0
    for a, b in zip(got, want):
        assert a.device.index == 1 and torch.equal(a.cpu(), b.cpu())
    with pytest.raises(ValueError, match="different devices"):
        ops.residual_norm(s["x"], want[0].half(), None)


def test_more_than_2_to_the_31_elements(ops):
    """Offsets past 32 bits: the last rows and tokens of tensors of over 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    tokens, heads = 1_100_000, 16
    x = torch.zeros(tokens, heads, 128, dtype=torch.bfloat16, device="cuda")
    x[-2:] = rnd(2, heads, 128, seed=1, dtype=torch.bfloat16)
    pos = torch.arange(tokens, device="cuda")
    f, _ = ops.rope_frequencies(128)
    o, _ = ops.rope(x, None, pos, f)
    want, tol = rope64(x[None, -2:], pos[None, None, -2:], f, 1.0, False, 1)
    close(o[None, -2:], want, tol)
    planes = torch.zeros(heads, tokens, 128, dtype=torch.bfloat16, device="cuda")
    ops.rope(x, None, pos, f, out=(planes.transpose(0, 1), None))
    assert torch.equal(planes[:, -2:].transpose(0, 1), o[-2:])
    del planes, o
    rows = x.view(-1, 2048)
    r, h = ops.residual_norm(rows, rows, None, norm="rms")
    r2, h2 = ops.residual_norm(rows[-2:].clone(), rows[-2:].clone(), None, norm="rms")
    # two rows are a block each, many are copied ahead: the sums' order is the same
    assert torch.equal(r[-2:], r2)
    close(h[-2:], h2.double(), 2 * half(h.dtype) * h2.double().abs() + 1e-6)
    del r, h, x, rows
    q = torch.ones(600_000, 64, dtype=torch.int8, device="cuda")
    w = ints(4096, 64, 3)
    y = ops.int8_linear(q, w, torch.ones(4096, device="cuda"), x_scale=torch.ones(600_000, device="cuda"))
    assert torch.equal(y[-1].float(), w.float().sum(1).bfloat16().float()) and torch.equal(y[-1], y[0])


def test_refusals_on_the_device(ops):
    x = rnd(4, 32, seed=1)
    wq, ws = ops.quantize_weight(rnd(8, 32, seed=2))
    f, _ = ops.rope_frequencies(32)
    q, pos = x.view(4, 1, 32), torch.arange(4, device="cuda")
    for call, text in (
            (lambda: ops.quantize_rows(x.double()), "bfloat16, float16 or float32"),
            (lambda: ops.quantize_rows(x.t()), "contiguous"),
            (lambda: ops.quantize_rows(x[0, 0]), "dimension"),
            (lambda: ops.int8_linear(x, wq.float(), ws), "int8"),
            (lambda: ops.int8_linear(x[:, :16], wq, ws), "weight must be"),
            (lambda: ops.int8_linear(x, wq, ws[:4]), "weight_scale"),
            (lambda: ops.int8_linear(x, wq, ws, ws.half()), "bias"),
            (lambda: ops.int8_linear(x, wq, ws, act="tanh"), "activation"),
            (lambda: ops.int8_linear(x, wq, ws, out_dtype=torch.float64), "out_dtype"),
            (lambda: ops.int8_linear(x, wq, ws, x_scale=ws), "x_scale"),
            (lambda: ops.int8_linear(x.to(torch.int8), wq, ws), "x_scale"),
            (lambda: ops.int8_linear(rnd(4, 24).to(torch.int8)[:, 4:], wq[:, :20], ws, x_scale=ws[:4]), "16-byte"),
            (lambda: ops.int8_linear(x[:, 1:], wq[:, 1:], ws), "16-byte"),
            (lambda: ops.int8_linear(x, wq.cpu(), ws), "CUDA|device"),
            (lambda: ops.residual_norm(x, x[:2], None), "shape"),
            (lambda: ops.residual_norm(x, x, ws), "weight"),
            (lambda: ops.residual_norm(x, x, None, norm="batch"), "norm"),
            (lambda: ops.residual_norm(x, None, None, post_norm="rms"), "without y"),
            (lambda: ops.residual_norm(x, x, None, gate=x[:3]), "gate"),
            (lambda: ops.residual_norm(x, x, None, eps=float("nan")), "eps"),
            (lambda: ops.residual_norm(x[:1].expand(4, 32), x, None), "overlap"),
            (lambda: ops.rope(q, None, pos.float(), f), "positions"),
            (lambda: ops.rope(q, None, pos[:3], f), "positions"),
            (lambda: ops.rope(q, q.half(), pos, f), "type"),
            (lambda: ops.rope(q, q[:2], pos, f), "k must be"),
            (lambda: ops.rope(q, None, pos, ops.rope_frequencies(64)[0]), "frequencies"),
            (lambda: ops.rope(q, None, pos, f, inplace=True, out=(q, None)), "exclude"),
            (lambda: ops.rope(q, None, pos, f, out=(q.half(), None)), "match"),
            (lambda: ops.rope(q[:, :, :1].expand(4, 1, 32), None, pos, f), "contiguous"),
            (lambda: ops.rope(q.expand(4, 3, 32), None, pos, f, inplace=True), "share memory"),
            (lambda: ops.residual_norm(x.clone().requires_grad_(), x, None), "gradient")):
        with pytest.raises(ValueError, match=text):
            call()
    with torch.no_grad():
        ops.residual_norm(x.clone().requires_grad_(), x, None)
    with torch.inference_mode():
        y = x + 1
        ops.residual_norm(y, x, None, inplace=True)
    with pytest.raises(ValueError, match="inference"):
        ops.residual_norm(y, x, None, inplace=True)
    # an in-place call counts as a change of the tensor
    z = x.clone()
    v = z._version
    ops.residual_norm(z, x, None, inplace=True)
    assert z._version == v + 1
    ops.status(0)
