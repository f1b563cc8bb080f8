"""GPU tests of the operators at the edges of their ranges: results far below the values they are
made from, columns and rows that are not finite, heads and head counts past a block's share, errors
of one call that must not show in the next, waits that run out.

Tolerances count roundings as test_gpu_ops.py does: U = 2^-24 is one 32-bit rounding, half(dtype)
half a step of the result's type."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_ops import DT, U, close, half, ops, residual64, rnd, rope64  # noqa: E402,F401


# ----------------------------------------------------------------------------- GELU
def gelu64(v):
    """v * sigmoid(2 u), u = sqrt(2 / pi) (v + 0.044715 v^3), which loses nothing where 1 + tanh(u)
    does, and the bound of its 32-bit form: the argument 2 u has 8 roundings (constants among them),
    the exponential 2^-22, reciprocal and products 16 U; v itself one, which the value's slope
    enlarges."""
    u2 = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    y = v * torch.sigmoid(u2)
    slope = 1 + v.abs() * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * v * v)
    return y, y.abs() * (8 * U * u2.abs() + 16 * U + 2 * U * slope)


def gelu_inputs(m, n):
    """8-bit rows and weights whose sums are one product each: column j of row i holds q_i * 127 * ws_j,
    from -12 to 12."""
    q = torch.zeros(m, 16, dtype=torch.int8)
    q[:, 0] = (torch.arange(m) * 37 % 255 - 127).to(torch.int8) if m > 4 else torch.tensor([-127, -64, -31, 90])[:m]
    w = torch.zeros(n, 16, dtype=torch.int8)
    w[:, 0] = 127
    ws = (torch.arange(n) + 1) * (12 / 127 / 127 / n)
    return q.cuda(), w.cuda(), ws.float().cuda()


# the one-launch kernel, the one that splits k, tiles of one CTA and of a pair
GELU_SHAPES = [(1, 40), (4, 200), (24, 200), (255, 300), (3000, 130), (20000, 1024)]


@pytest.mark.parametrize("m,n", GELU_SHAPES)
@pytest.mark.parametrize("out", DT)
def test_gelu_of_negative_values_keeps_its_digits(ops, m, n, out):  # noqa: F811
    """Each result is right to its own size, down to the ones far below the values they come from."""
    q, w, ws = gelu_inputs(m, n)
    y = ops.int8_linear(q, w, ws, x_scale=torch.ones(m, device="cuda"), act="gelu", out_dtype=DT[out])
    v = q[:, :1].double() * 127 * ws.double()
    want, tol = gelu64(v)
    # half a step of fp16's smallest values; results below 2^-120 may be zero
    least = 2.0 ** -25 if out == "fp16" else 2.0 ** -120
    close(y, want, tol + half(DT[out]) * (want.abs() + tol) + least)


@pytest.mark.parametrize("m,n", GELU_SHAPES)
@pytest.mark.parametrize("out", DT)
def test_gelu_columns_that_are_not_finite_stay_alone(ops, m, n, out):  # noqa: F811
    q, w, ws = gelu_inputs(m, n)
    one = torch.ones(m, device="cuda")
    y = ops.int8_linear(q, w, ws, x_scale=one, act="gelu", out_dtype=DT[out])
    ws[5], ws[18] = math.nan, math.inf
    z = ops.int8_linear(q, w, ws, x_scale=one, act="gelu", out_dtype=DT[out])
    keep = [j for j in range(n) if j not in (5, 18)]
    assert torch.equal(z[:, keep], y[:, keep])
    assert torch.isnan(z[:, 5]).all()
    up = q[:, 0] > 0
    assert torch.isposinf(z[up, 18]).all() and torch.isnan(z[~up, 18]).all()


# ----------------------------------------------------------------------------- errors
@pytest.mark.skipif("torch.cuda.device_count() >= 8")
def test_an_error_of_one_call_does_not_show_in_the_next(ops):  # noqa: F811
    """A device that does not exist fails that call alone."""
    from test_ops_args import QUANTIZE, RESIDUAL

    from mast3r_runtime_b200 import _lib

    lib = _lib.load()
    x, gate = rnd(6, 41, seed=1), rnd(41, seed=2)
    r, h = torch.empty_like(x), torch.empty_like(x)
    q, s = torch.empty(6, 48, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    none = torch.cuda.device_count()  # the first that does not exist
    args = RESIDUAL.pack(0, 2, 2, 2, 1, 0, 1e-6, 1.0, 6, 41, 41, 41, 41, 41, 0, 0, x.data_ptr(), x.data_ptr(),
                         gate.data_ptr(), 0, 0, 0, 0, r.data_ptr(), h.data_ptr(), 0, stream)
    bad = QUANTIZE.pack(none, 2, 6, 41, 41, 48, x.data_ptr(), q.data_ptr(), s.data_ptr(), 0)
    for _ in range(2):
        assert lib.m3r_quantize_rows(bad) == -3 and lib.m3r_global_error()
        assert lib.m3r_residual_norm(args) == 0, lib.m3r_global_error()
        want = residual64(x, x, gate, 1.0, None, None, None)
        close(r, *want)
    # nor does the engine's next launch see it
    from test_gpu_failure import _attention_ok

    assert lib.m3r_quantize_rows(bad) == -3 and _attention_ok(lib)
    # an error that another entry point left behind stays its own too
    d = torch.zeros(300, 24, device="cuda")
    nn = torch.empty(300, dtype=torch.int32, device="cuda")
    for _ in range(2):
        assert lib.m3r_match_nn_static(none, d.data_ptr(), d.data_ptr(), 300, 300, 24, nn.data_ptr(), nn.data_ptr(), 0,
                                       0) == -3
        assert _attention_ok(lib)
        assert lib.m3r_residual_norm(args) == 0, lib.m3r_global_error()


@pytest.mark.parametrize("which", [0, 1])
def test_a_wait_that_ran_out_is_reported_once(ops, which):  # noqa: F811
    """The product's kernels and the row kernels each record it; the next calls are sound."""
    from mast3r_runtime_b200 import _lib

    lib = _lib.load()
    ops.status(0)
    side = torch.cuda.Stream()
    for stream, limit in ((torch.cuda.current_stream(), 1_000_000), (side, 3_000_000)):
        assert lib.m3r_operator_wait_selftest(0, which, limit, stream.cuda_stream) == 0, lib.m3r_global_error()
        with torch.cuda.stream(stream):
            with pytest.raises(RuntimeError, match="timed out"):
                ops.status(0)
            ops.status(0)
            q, w, ws = gelu_inputs(200, 40)
            y = ops.int8_linear(q, w, ws, x_scale=torch.ones(200, device="cuda"), out_dtype=torch.float32)
            v = q[:, :1].double() * 127 * ws.double()
            close(y, v, 4 * U * v.abs())
            x = rnd(3000, 1024, seed=3)
            r, _ = ops.residual_norm(x, x, None)
            assert torch.equal(r, x + x)
            ops.status(0)


def test_wait_selftest_refusals(ops):  # noqa: F811
    from mast3r_runtime_b200 import _lib

    lib = _lib.load()
    for args in ((0, 2, 1000), (0, -1, 1000), (0, 0, 0), (0, 0, 20_000_000_000), (-1, 0, 1000)):
        assert lib.m3r_operator_wait_selftest(*args, None) == -1


# ----------------------------------------------------------------------------- rope
@pytest.mark.parametrize("dim,rot,dtype", [(4096, 4096, "fp32"), (4096, 2400, "bf16"), (1400, 1400, "fp32"),
                                           (1030, 1026, "fp16")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_heads_longer_than_a_block(ops, dim, rot, dtype, interleaved):  # noqa: F811
    """Heads with more accesses than a block has threads."""
    f, amp = ops.rope_frequencies(rot)
    for t, h, kv in ((1, 1, 1), (5, 3, 1)):
        q, k = rnd(1, t, h, dim, seed=1, dtype=DT[dtype]), rnd(1, t, kv, dim, seed=2, dtype=DT[dtype])
        pos = torch.arange(t, device="cuda") * 117 + 3
        for x, o in zip((q, k), ops.rope(q, k, pos, f, interleaved=interleaved)):
            want, tol = rope64(x, pos[None, None], f, 1.0, interleaved, 1)
            close(o, want, tol)


@pytest.mark.parametrize("tokens", [1, 700])
@pytest.mark.parametrize("heads,kv", [(300, 100), (257, 1), (1, 600), (512, 512)])
def test_rope_more_heads_than_a_block_takes(ops, tokens, heads, kv):  # noqa: F811
    f, _ = ops.rope_frequencies(16)
    q, k = rnd(1, tokens, heads, 24, seed=1), rnd(1, tokens, kv, 24, seed=2)
    pos = torch.arange(tokens, device="cuda") - 5
    for x, o in zip((q, k), ops.rope(q, k, pos, f)):
        want, tol = rope64(x, pos[None, None], f, 1.0, False, 1)
        close(o, want, tol)


# ----------------------------------------------------------------------------- residual_norm
@pytest.mark.parametrize("rows,cols", [(9, 24), (9, 1024), (9, 1001), (3000, 1024), (9, 5003), (700, 4096)])
@pytest.mark.parametrize("norm,post", [("layer", None), ("rms", "layer")])
def test_residual_norm_rows_that_are_not_finite_stay_alone(ops, rows, cols, norm, post):  # noqa: F811
    x, y = rnd(rows, cols, seed=1), rnd(rows, cols, seed=2, dtype=torch.bfloat16)
    w = 1 + 0.1 * rnd(cols, seed=3)
    kw = dict(norm=norm, post_norm=post)
    r, h = ops.residual_norm(x, y, w, out_dtype=torch.float32, **kw)
    x2, y2 = x.clone(), y.clone()
    x2[1, 3], x2[4, cols - 1], y2[6, 0], y2[8, cols // 2] = math.inf, math.nan, -math.inf, math.nan
    bad = [1, 4, 6, 8]
    good = [i for i in range(rows) if i not in bad]
    r2, h2 = ops.residual_norm(x2, y2, w, out_dtype=torch.float32, **kw)
    r3, q, s = ops.residual_norm(x2, y2, w, out_dtype=torch.int8, **kw)
    assert torch.equal(r2[good], r[good]) and torch.equal(h2[good], h[good])
    assert torch.equal(r3[good], r[good]) and torch.isfinite(s[good]).all()
    # an infinity or a NaN makes the layer norm's whole row NaN; in an RMS norm an infinite sum of
    # squares makes the finite values 0
    if norm == "layer":
        assert torch.isnan(h2[bad]).all()
    else:
        assert not torch.isfinite(h2[bad]).all(-1).any()
    assert int(q[bad].abs().max()) == 0 and not torch.isfinite(s[bad]).any()
    if post is None:
        assert torch.equal(r2[1, :3], r[1, :3]) and torch.isposinf(r2[1, 3]) and torch.isnan(r2[8, cols // 2])
