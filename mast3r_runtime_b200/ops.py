"""Operators of 8-bit transformer blocks on device tensors (C ABI: include/m3r_cuda.h).

    from mast3r_runtime_b200 import ops

    x, h, s = ops.residual_norm(x, y, weight, bias, gate=gate, out_dtype=torch.int8)
    qkv = ops.int8_linear(h, w, w_scale, w_bias, x_scale=s, out_dtype=torch.bfloat16)
    q, k, v = qkv.view(batch, tokens, 3, heads, dim).unbind(2)
    q, k = ops.rope(q, k, positions, inv_freq)

Tensors are torch CUDA tensors (this module is the only one of the package that needs torch; its
compiled side is binding/torch_ops.cpp).  A call runs on its tensors' device and on that device's
current torch stream, queues its work without waiting, and can be captured into a CUDA graph; its
results and workspace come from torch's allocator.  All tensors of a call are on one device, and the
last dimension of the large ones is contiguous; rope takes any other strides, the row operators rows
that are evenly spaced.  Bad arguments raise ValueError before anything is launched, device errors
RuntimeError, and a wait on the device that ran out is reported by status().  The calls are plain
functions: torch.compile breaks its graph at each.  The operators have no
gradients: the package runs models, it does not train them, and a call with a tensor that requires
grad outside torch.no_grad(), or with one that carries a forward-mode tangent, is refused.
"""

from __future__ import annotations

import math

import torch

from . import _lib

try:
    from . import _torch_ops as _native
except ImportError as e:  # never a silent fallback
    raise ImportError(f"the operators' torch binding does not load ({e}): "
                      "run `python -m mast3r_runtime_b200.build`") from e

__all__ = ["quantize_rows", "quantize_weight", "int8_linear", "residual_norm", "rope", "rope_frequencies", "status"]


def quantize_rows(x: torch.Tensor):
    """Rows of x [..., cols] in 8 bits: (q int8 [..., cols], scale float32 [...]).

    With a = max |row|, q is the integer nearest to 127 x / a (ties to even) and scale = a / 127,
    so that q * scale is x to half a step.  A row of zeros has scale 0.  A row with an infinity
    or a NaN holds zeros with an infinite or NaN scale: products with it are NaN.  Rows below 1.5e-36
    have a subnormal scale, with fewer bits.  q's rows lie on 16-byte boundaries, as int8_linear
    needs them.  cols is at most 16,384."""
    return _native.quantize_rows(x)


def quantize_weight(w: torch.Tensor):
    """Weights [n, k] in 8 bits with a scale for each output channel, laid out for int8_linear:
    (q int8 [n, k] with 16-byte aligned rows, scale float32 [n])."""
    if w.dim() != 2:
        raise ValueError(f"quantize_weight: weights must be [n, k], got {list(w.shape)}")
    return _native.quantize_rows(w)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None, *,
                act: str = "none", out_dtype: torch.dtype | None = None, x_scale: torch.Tensor | None = None):
    """act((x . weight^T) + bias) in 8-bit integers: [..., k] x [n, k] -> [..., n].

    x in 16 or 32 bits is quantised row by row as quantize_rows does (k at most 16,384); x in int8
    comes with x_scale [...] (float32) and rows on 16-byte boundaries, as quantize_rows and
    residual_norm return them (k at most 131,071).  weight is int8 [n, k] with rows on 16-byte
    boundaries and weight_scale float32 [n], as quantize_weight returns them; bias float32 [n].
    The sum over k is exact; scales (the row's first: rows above 3.4e38 / (127 k) may give infinities),
    bias and activation ("none", "gelu" in its tanh form, "relu") are applied in 32 bits and rounded once
    to out_dtype (default: x's type, bfloat16 for int8)."""
    return _native.int8_linear(x, weight, weight_scale, bias, act, out_dtype, x_scale)


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
    (r, q, scale) as quantize_rows makes them of h.  inplace writes r over x: y may be x itself then,
    and nothing else may share memory with it."""
    return _native.residual_norm(x, y, weight, bias, norm, post_norm, post_weight, post_bias, gate, residual_scale,
                                 eps, out_dtype, inplace)


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
    if axes not in (1, 2) or rot_dim < 2 * axes or rot_dim % (2 * axes):
        raise ValueError(f"rope_frequencies: rot_dim {rot_dim} must be a positive multiple of 2 for each of 1 or 2 axes")
    if not (factor >= 1.0 and math.isfinite(factor)) or not base > 0 or not fast > slow:
        raise ValueError("rope_frequencies: factor must be at least 1, base positive and fast above slow")
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
        raise ValueError(f"rope_frequencies: unknown scaling {scaling!r} (none, linear, ntk or by_parts)")
    return f.repeat(axes).to(device), amplitude


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
         amplitude: float = 1.0, interleaved: bool = False, axes: int = 1, inplace: bool = False, out=None):
    """Rotary positions on queries and keys [tokens, heads, dim] or [batch, tokens, heads, dim]
    (k may have other heads, or be None): pair i of a head's first 2 * len(inv_freq) values is
    turned by position * inv_freq[i] and scaled by amplitude; the values behind are copied.

    Pairs are (i, i + n), or (2 i, 2 i + 1) when interleaved.  positions are int32 or int64, [tokens]
    or [batch, tokens]; with axes = 2 ([2, tokens] or [2, batch, tokens]) the first half of the pairs
    turns with positions[0], the second with positions[1], as image tokens do with their row and
    column.  inv_freq is float64 (rope_frequencies); angles are reduced in 64 bits, their sines and
    cosines taken in 32.

    Strides are free apart from the last dimension's (views of a packed projection).  Returns
    (q, k) turned: new tensors, q and k themselves with inplace, or the given out = (q_out, k_out)
    of the same shapes and type (of any strides: head-major planes for an attention kernel).  A result
    may be its own input (the same view), and shares memory with nothing else of the call."""
    oq, ok = out if out is not None else (None, None)
    return _native.rope(q, k, positions, inv_freq, amplitude, interleaved, axes, inplace, oq, ok)


def status(device: int = 0) -> None:
    """Waits for the device's current stream and raises RuntimeError when a device-side wait of an
    operator ran out since the last call (the results of the calls since are undefined)."""
    _lib.check(_lib.load().m3r_operator_status(int(device), torch.cuda.current_stream(int(device)).cuda_stream))
