"""Operators of 8-bit transformer blocks on device tensors (C ABI: include/m3r_cuda.h).

    from mast3r_runtime_b200 import ops

    x, h, s = ops.residual_norm(x, y, weight, bias, gate=gate, out_dtype=torch.int8)
    qkv = ops.int8_linear(h, w, w_scale, w_bias, x_scale=s, out_dtype=torch.bfloat16)
    q, k, v = qkv.view(batch, tokens, 3, heads, dim).unbind(2)
    q, k = ops.rope(q, k, positions, inv_freq)

Tensors are torch CUDA tensors (this module is the only one of the package that imports
torch).  A call runs on its tensors' device and on that device's current torch stream, queues
its work without waiting, and can be captured into a CUDA graph; its results and workspace
come from torch's allocator.  All tensors of a call are on one device, and the last dimension
of the large ones is contiguous (other strides are free).  Bad arguments raise ValueError
before anything is launched, device errors RuntimeError.  The operators have no gradients: the
package runs models, it does not train them, and a call with a tensor that requires grad
outside torch.no_grad() is refused.
"""

from __future__ import annotations

import math
from functools import lru_cache
from struct import Struct

import torch

from . import _lib

__all__ = ["quantize_rows", "quantize_weight", "int8_linear", "residual_norm", "rope", "rope_frequencies", "status"]

_FLOAT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_ACT = {"none": 0, "gelu": 1, "relu": 2}
_NORM = {"layer": 1, "rms": 2}

# the argument structs of include/m3r_cuda.h, native layout
_QUANTIZE = Struct("@2i4q4P")
_LINEAR = Struct("@4i6q7Pq1P")
_RESIDUAL = Struct("@6i2f8q" "11P")
_ROPE = Struct("@5if7q2P" "2P7q" "2P7q" "P")

_stream = torch._C._cuda_getCurrentRawStream  # current_stream(device).cuda_stream without the objects


def _fail(text: str):
    raise ValueError(text)


def _check_device(op: str, t: torch.Tensor, *others) -> int:
    if not t.is_cuda:
        _fail(f"{op}: tensors must be on a CUDA device")
    dev = t.get_device()
    for o in others:
        if o is not None and o.get_device() != dev:
            _fail(f"{op}: tensors are on different devices")
    if torch.is_grad_enabled() and (t.requires_grad or any(o is not None and o.requires_grad for o in others)):
        _fail(f"{op}: no gradient is computed (use torch.no_grad() or detach the tensors)")
    return dev


def _rows(op: str, name: str, t: torch.Tensor):
    """(rows, cols, row stride) of a tensor [..., cols] whose rows are evenly spaced."""
    d = t.dim()
    if d == 2:
        rows, cols = t.shape
        ld, sc = t.stride()
    elif d == 0:
        _fail(f"{op}: {name} must have at least one dimension")
    else:
        shape, stride = t.shape, t.stride()
        cols, sc = shape[-1], stride[-1]
        rows, ld = 1, cols
        step = None
        for n, s in zip(shape[-2::-1], stride[-2::-1]):
            if n != 1:
                if step is None:
                    ld = s
                elif s != step and t.numel():
                    _fail(f"{op}: the rows of {name} are not evenly spaced (make it contiguous)")
                step = s * n
            rows *= n
    if sc != 1 and cols != 1:
        _fail(f"{op}: the last dimension of {name} must be contiguous")
    if ld < cols:
        if rows > 1:
            _fail(f"{op}: the rows of {name} overlap")
        ld = cols
    return rows, cols, ld


def _vector(op: str, name: str, t, n: int) -> int:
    """Address of an fp32 vector of n values (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != n:
        _fail(f"{op}: {name} must be a float32 tensor of shape [{n}], got {t.dtype} {list(t.shape)}")
    if n > 1 and t.stride(0) != 1:
        _fail(f"{op}: {name} must be contiguous")
    return t.data_ptr()


def _float_type(op: str, name: str, dtype) -> int:
    code = _FLOAT.get(dtype)
    if code is None:
        _fail(f"{op}: {name} must be bfloat16, float16 or float32, got {dtype}")
    return code


def _int8_rows(rows: int, cols: int, shape, device) -> torch.Tensor:
    """An int8 tensor [..., cols] with rows on 16-byte boundaries."""
    ld = -(-cols // 16) * 16
    q = torch.empty((rows, ld), dtype=torch.int8, device=device)
    if ld != cols:
        q = q[:, :cols]
    return q if len(shape) == 2 else q.unflatten(0, shape[:-1]) if len(shape) > 2 else q[0]


@lru_cache(maxsize=4096)
def _workspace_bytes(x_dtype: int, rows: int, n: int, k: int) -> int:
    b = _lib.load().m3r_int8_linear_workspace(x_dtype, rows, n, k)
    if b < 0:
        _lib.check(int(b))
    return b


def quantize_rows(x: torch.Tensor):
    """Rows of x [..., cols] in 8 bits: (q int8 [..., cols], scale float32 [...]).

    With a = max |row|, q is the integer nearest to 127 x / a (ties to even) and scale = a / 127,
    so that q * scale is x to half a step.  A row of zeros has scale 0.  A row with an infinity
    or a NaN holds zeros with an infinite or NaN scale: products with it are NaN.  q's rows lie
    on 16-byte boundaries, as int8_linear needs them.  cols is at most 16,384."""
    op = "quantize_rows"
    dev = _check_device(op, x)
    dt = _float_type(op, "x", x.dtype)
    rows, cols, ld = _rows(op, "x", x)
    q = _int8_rows(rows, cols, x.shape, x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _, _, ldq = _rows(op, "q", q)
    _lib.check(_lib.load().m3r_quantize_rows(_QUANTIZE.pack(
        dev, dt, rows, cols, ld, max(ldq, -(-cols // 16) * 16), x.data_ptr(), q.data_ptr(), scale.data_ptr(),
        _stream(dev))))
    return q, scale


def quantize_weight(w: torch.Tensor):
    """Weights [n, k] in 8 bits with a scale for each output channel, laid out for int8_linear:
    (q int8 [n, k] with 16-byte aligned rows, scale float32 [n])."""
    if w.dim() != 2:
        _fail(f"quantize_weight: weights must be [n, k], got {list(w.shape)}")
    return quantize_rows(w)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None, *,
                act: str = "none", out_dtype: torch.dtype | None = None, x_scale: torch.Tensor | None = None):
    """act((x . weight^T) + bias) in 8-bit integers: [..., k] x [n, k] -> [..., n].

    x in 16 or 32 bits is quantised row by row as quantize_rows does (k at most 16,384); x in int8
    comes with x_scale [...] (float32) and rows on 16-byte boundaries, as quantize_rows and
    residual_norm return them (k at most 131,072).  weight is int8 [n, k] with rows on 16-byte
    boundaries and weight_scale float32 [n], as quantize_weight returns them; bias float32 [n].
    The sum over k is exact; scales, bias and activation ("none", "gelu" in its tanh form, "relu")
    are applied in 32 bits and rounded once to out_dtype (default: x's type, bfloat16 for int8)."""
    op = "int8_linear"
    dev = _check_device(op, x, weight, weight_scale, bias, x_scale)
    rows, k, ldx = _rows(op, "x", x)
    if weight.dtype is not torch.int8 or weight.dim() != 2 or weight.shape[1] != k:
        _fail(f"{op}: weight must be int8 [n, {k}], got {weight.dtype} {list(weight.shape)}")
    n = weight.shape[0]
    if n < 1 or k < 1:
        _fail(f"{op}: empty weight {list(weight.shape)}")
    ldw, sw = weight.stride()
    if sw != 1 and k != 1:
        _fail(f"{op}: the rows of weight must be contiguous")
    if n == 1 and ldw < k:
        ldw = -(-k // 16) * 16
    if x.dtype is torch.int8:
        xt = _lib.DTYPE_I8
        if x_scale is None or x_scale.dtype is not torch.float32 or x_scale.shape != x.shape[:-1] or \
                not x_scale.is_contiguous():
            _fail(f"{op}: int8 rows need x_scale, a contiguous float32 tensor of shape {list(x.shape[:-1])}")
        if rows == 1:
            ldx = -(-k // 16) * 16
        ps = x_scale.data_ptr()
        out_dtype = out_dtype or torch.bfloat16
    else:
        xt = _float_type(op, "x", x.dtype)
        if x_scale is not None:
            _fail(f"{op}: x_scale belongs to int8 rows")
        ps = 0
        out_dtype = out_dtype or x.dtype
    ot = _float_type(op, "out_dtype", out_dtype)
    if act not in _ACT:
        _fail(f"{op}: unknown activation {act!r} (none, gelu or relu)")
    out = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=x.device)
    if rows == 0:
        return out
    need = _workspace_bytes(xt, rows, n, k)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device).data_ptr() if need else 0
    _lib.check(_lib.load().m3r_int8_linear(_LINEAR.pack(
        dev, xt, ot, _ACT[act], rows, n, k, ldx, ldw, n, x.data_ptr(), ps, weight.data_ptr(),
        _vector(op, "weight_scale", weight_scale, n), _vector(op, "bias", bias, n), out.data_ptr(), ws, need,
        _stream(dev))))
    return out


def residual_norm(x: torch.Tensor, y: torch.Tensor | None, weight: torch.Tensor | None,
                  bias: torch.Tensor | None = None, *, norm: str = "layer", post_norm: str | None = None,
                  post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, residual_scale: float = 1.0, eps: float = 1e-6,
                  out_dtype: torch.dtype | None = None, inplace: bool = False):
    """The norms before and after a block with its gate and residual scale, in one pass:

        t = y                                  or norm(y) * post_weight + post_bias with post_norm
        r = residual_scale * x + gate * t      the new residual stream, in x's type
        h = norm(r) * weight + bias            the next block's input, from the unrounded r

    x is the stream [..., cols], y the block's output of the same shape (or None: r is then
    residual_scale * x).  Norms are "layer" or "rms"; their weights and biases are float32 [cols] or
    None (1 and 0).  gate is float32 [cols], or [groups, cols] with the rows of x in that many equal
    groups in order (one gate for each image), or None (1).  cols is at most 16,384.

    Returns (r, h), h in out_dtype (default: y's type, else x's); with out_dtype torch.int8
    (r, q, scale) as quantize_rows makes them of h.  inplace writes r over x."""
    op = "residual_norm"
    dev = _check_device(op, x, y, weight, bias, post_weight, post_bias, gate)
    xt = _float_type(op, "x", x.dtype)
    rows, cols, ldx = _rows(op, "x", x)
    yt = py = ldy = 0
    if y is not None:
        yt = _float_type(op, "y", y.dtype)
        if y.shape != x.shape:
            _fail(f"{op}: x and y differ in shape: {list(x.shape)} and {list(y.shape)}")
        _, _, ldy = _rows(op, "y", y)
        py = y.data_ptr()
    nk = _NORM.get(norm) or _fail(f"{op}: unknown norm {norm!r} (layer or rms)")
    pk = 0 if post_norm is None else _NORM.get(post_norm) or _fail(f"{op}: unknown post norm {post_norm!r}")
    pg = per_gate = ld_gate = 0
    if gate is not None:
        if gate.dim() == 2:
            groups = gate.shape[0]
            if gate.dtype is not torch.float32 or gate.shape[1] != cols or groups < 1 or rows % groups or \
                    (cols > 1 and gate.stride(1) != 1) or (groups > 1 and gate.stride(0) < cols):
                _fail(f"{op}: gate must be float32 [groups, {cols}] with groups dividing {rows} rows, "
                      f"got {gate.dtype} {list(gate.shape)}")
            per_gate, ld_gate, pg = rows // groups, max(gate.stride(0), cols), gate.data_ptr()
        else:
            pg = _vector(op, "gate", gate, cols)
    out_dtype = out_dtype or (x if y is None else y).dtype
    r = x if inplace else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ldr = ldx if inplace else cols
    scale = None
    if out_dtype is torch.int8:
        ot = _lib.DTYPE_I8
        out = _int8_rows(rows, cols, x.shape, x.device)
        ldo = -(-cols // 16) * 16
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    else:
        ot = _float_type(op, "out_dtype", out_dtype)
        out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
        ldo = cols
    _lib.check(_lib.load().m3r_residual_norm(_RESIDUAL.pack(
        dev, xt, yt, ot, nk, pk, eps, residual_scale, rows, cols, ldx, ldy, ldr, ldo, per_gate, ld_gate,
        x.data_ptr(), py, pg, _vector(op, "post_weight", post_weight, cols), _vector(op, "post_bias", post_bias, cols),
        _vector(op, "weight", weight, cols), _vector(op, "bias", bias, cols), r.data_ptr(), out.data_ptr(),
        0 if scale is None else scale.data_ptr(), _stream(dev))))
    return (r, out) if scale is None else (r, out, scale)


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                     original_length: int = 4096, slow: float = 1.0, fast: float = 32.0, axes: int = 1, device="cuda"):
    """(inv_freq float64 [rot_dim / 2], amplitude) for rope: base^(-2 i / rot_dim) radians a position,
    scaled for contexts `factor` times longer than the model was trained on:

    "linear"    every frequency divided by factor
    "ntk"       base * factor^(rot_dim / (rot_dim - 2)): the slowest pair is divided by factor, the
                fastest kept
    "by_parts"  pairs that make fewer than `slow` turns in original_length positions are divided by
                factor, those with more than `fast` kept, a linear ramp between; the rotated values
                grow by amplitude = 0.1 ln(factor) + 1 (Peng et al. 2023)

    With axes = 2 each axis has the frequencies of a head part of rot_dim / 2."""
    if rot_dim < 2 * axes or rot_dim % (2 * axes) or axes not in (1, 2):
        _fail(f"rope_frequencies: rot_dim {rot_dim} must be a positive multiple of {2 * axes}")
    if not (factor >= 1.0 and math.isfinite(factor)) or not base > 0:
        _fail("rope_frequencies: factor must be at least 1 and base positive")
    part = rot_dim // axes
    if scaling == "ntk":
        base = base * factor ** (part / (part - 2)) if part > 2 else base
    f = base ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
    amplitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":
        keep = ((original_length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in ("none", "ntk"):
        _fail(f"rope_frequencies: unknown scaling {scaling!r} (none, linear, ntk or by_parts)")
    return f.repeat(axes).to(device), amplitude


def _rope_tensor(op: str, name: str, x: torch.Tensor, out: torch.Tensor, ref: torch.Tensor):
    """The fields of an m3r_rope_tensor for [tokens, heads, dim] or [batch, tokens, heads, dim]."""
    d = x.dim()
    if d not in (3, 4) or d != ref.dim() or x.shape[:-2] != ref.shape[:-2] or x.shape[-1] != ref.shape[-1]:
        _fail(f"{op}: {name} must be [tokens, heads, dim] or [batch, tokens, heads, dim], got {list(x.shape)}")
    if x.dtype is not ref.dtype:
        _fail(f"{op}: q and k differ in type")
    s, o = x.stride(), out.stride()
    if s[-1] != 1 or o[-1] != 1:
        _fail(f"{op}: the last dimension of {name} must be contiguous")
    if d == 3:
        return x.data_ptr(), out.data_ptr(), x.shape[1], 0, s[0], s[1], 0, o[0], o[1]
    return x.data_ptr(), out.data_ptr(), x.shape[2], s[0], s[1], s[2], o[0], o[1], o[2]


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
         amplitude: float = 1.0, interleaved: bool = False, axes: int = 1, inplace: bool = False, out=None):
    """Rotary positions on queries and keys [tokens, heads, dim] or [batch, tokens, heads, dim]
    (k may have other heads, or be None): pair i of a head's first 2 * len(inv_freq) values is
    turned by position * inv_freq[i] and scaled by amplitude; the values behind are copied.

    Pairs are (i, i + n), or (2 i, 2 i + 1) when interleaved.  positions are int32 or int64, [tokens]
    or [batch, tokens]; with axes = 2 ([2, tokens] or [2, batch, tokens]) the first half of the pairs
    turns with positions[0], the second with positions[1], as image tokens do with their row and
    column.  inv_freq is float64 (rope_frequencies); angles are reduced in 64 bits.

    Strides are free apart from the last dimension's (views of a packed projection).  Returns
    (q, k) turned: new tensors, q and k themselves with inplace, or the given out = (q_out, k_out)
    of the same shapes and type (of any strides: head-major planes for an attention kernel)."""
    op = "rope"
    n = inv_freq.shape[0] if inv_freq.dim() == 1 else 0
    if inv_freq.dtype is not torch.float64 or n < 1 or (n > 1 and inv_freq.stride(0) != 1):
        _fail(f"{op}: inv_freq must be a contiguous float64 vector")
    dev = _check_device(op, q, k, positions, inv_freq)
    dt = _float_type(op, "q", q.dtype)
    if inplace:
        if out is not None:
            _fail(f"{op}: inplace and out exclude each other")
        oq, ok = q, k
    elif out is not None:
        oq, ok = out
        for a, b in ((q, oq), (k, ok)):
            if (a is None) != (b is None) or (a is not None and (
                    a.shape != b.shape or a.dtype is not b.dtype or b.get_device() != dev)):
                _fail(f"{op}: out must match q and k in shape, type and device")
    else:
        oq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ok = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    tq = _rope_tensor(op, "q", q, oq, q)
    tk = (0,) * 9 if k is None else _rope_tensor(op, "k", k, ok, q)
    batch, tokens, dim = (q.shape[0] if q.dim() == 4 else 1), q.shape[-3], q.shape[-1]
    pd, ps, pst = positions.dim(), positions.shape, positions.stride()
    if axes not in (1, 2):
        _fail(f"{op}: axes must be 1 or 2")
    lead = axes - 1
    if positions.dtype is torch.int64:
        bits = 64
    elif positions.dtype is torch.int32:
        bits = 32
    else:
        _fail(f"{op}: positions must be int32 or int64, got {positions.dtype}")
    if pd not in (lead + 1, lead + 2) or (lead and ps[0] != 2) or ps[-1] != tokens or \
            (pd == lead + 2 and ps[lead] not in (1, batch)):
        _fail(f"{op}: positions {list(ps)} do not fit {axes} axes, batch {batch} and {tokens} tokens")
    pos_axis = pst[0] if lead else 0
    pos_batch = pst[lead] if pd == lead + 2 and ps[lead] > 1 else 0
    _lib.check(_lib.load().m3r_rope(_ROPE.pack(
        dev, dt, interleaved, axes, bits, amplitude, batch, tokens, dim, n, pos_axis, pos_batch, pst[-1],
        positions.data_ptr(), inv_freq.data_ptr(), *tq, *tk, _stream(dev))))
    return oq, ok


def status(device: int = 0) -> None:
    """Waits for the device's current stream and raises RuntimeError when a device-side wait of an
    operator ran out since the last call (the results of the calls since are undefined)."""
    _lib.check(_lib.load().m3r_operator_status(int(device), _stream(int(device))))
