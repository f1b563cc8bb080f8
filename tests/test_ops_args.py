"""CPU tests of the operators' boundary: the packed argument structs have the C layout, and bad
arguments are refused before any device work, by the Python functions and by the C ABI."""

from __future__ import annotations

import subprocess
import textwrap
from struct import Struct, calcsize

import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")


# the argument structs of include/m3r_cuda.h, native layout
QUANTIZE = Struct("@2i4q4P")
LINEAR = Struct("@4i6q7PqP")
RESIDUAL = Struct("@6i2f8q11P")
ROPE = Struct("@5if7q2P" "2P7q" "2P7q" "P")


def test_argument_structs_match_c(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text(textwrap.dedent("""
        #include <stddef.h>
        #include <stdio.h>
        #include "m3r_cuda.h"
        #define P(x) printf("%zu\\n", (size_t)(x))
        int main(void) {
          P(sizeof(m3r_quantize_args)); P(offsetof(m3r_quantize_args, scale));
          P(sizeof(m3r_int8_linear_args)); P(offsetof(m3r_int8_linear_args, workspace_bytes));
          P(sizeof(m3r_residual_norm_args)); P(offsetof(m3r_residual_norm_args, x));
          P(sizeof(m3r_rope_args)); P(offsetof(m3r_rope_args, t));
          return 0;
        }
    """))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    c = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert c == [QUANTIZE.size, calcsize("@2i4q2P"), LINEAR.size, calcsize("@4i6q7P"),
                 RESIDUAL.size, calcsize("@6i2f8q"), ROPE.size, calcsize("@5if7q2P")]


def refused(fn, args, text):
    from mast3r_runtime_b200 import _lib

    lib = _lib.load()
    assert getattr(lib, fn)(args) == -1, text
    assert text in lib.m3r_global_error().decode()


def test_c_refusals():
    """Addresses are never dereferenced: every check comes before the first CUDA call."""

    def quantize(dev=0, dt=0, rows=2, cols=8, ldx=8, ldq=16, x=16, q=16, s=16):
        return QUANTIZE.pack(dev, dt, rows, cols, ldx, ldq, x, q, s, 0)

    for bad, text in ((dict(dt=3), "must be"), (dict(rows=-1), "rows out of range"), (dict(cols=0), "row length"),
                      (dict(cols=16385, ldx=16385, ldq=16400), "row length"), (dict(ldx=7), "stride"),
                      (dict(ldq=7), "stride"), (dict(x=0), "null"), (dict(x=17), "misaligned"),
                      (dict(rows=2 ** 31), "rows out of range"), (dict(s=18), "misaligned")):
        refused("m3r_quantize_rows", quantize(**bad), text)
    refused("m3r_quantize_rows", None, "null")

    def linear(xt=1, ot=1, act=0, m=400, n=32, k=64, ldx=64, ldw=64, ldo=32, x=256, xs=0, w=256, ws=256, b=0, o=256,
               work=256, size=1 << 20):
        return LINEAR.pack(0, xt, ot, act, m, n, k, ldx, ldw, ldo, x, xs, w, ws, b, o, work, size, 0)

    for bad, text in ((dict(xt=4), "x must be"), (dict(ot=3), "output must be"), (dict(act=3), "activation"),
                      (dict(m=-1), "rows out of range"), (dict(n=0), "n out of range"), (dict(k=0), "k out of range"),
                      (dict(k=16385, ldx=16400, ldw=16400), "k out of range"), (dict(ldw=72), "16-byte aligned"),
                      (dict(w=264), "16-byte aligned"), (dict(xs=256), "x_scale"), (dict(xt=3), "x_scale"),
                      (dict(xt=3, xs=256, ldx=72), "16-byte aligned"), (dict(xt=3, xs=256, x=8), "16-byte aligned"),
                      (dict(work=0), "workspace"), (dict(size=64), "workspace"), (dict(work=320), "workspace"),
                      (dict(ldo=31), "stride"), (dict(ws=0), "null"), (dict(o=0), "null"), (dict(o=257), "misaligned"),
                      (dict(b=257), "misaligned"), (dict(xt=3, xs=256, k=131072, ldx=131072, ldw=131072), "k out")):
        refused("m3r_int8_linear", linear(**bad), text)

    def norm(xt=2, yt=0, ot=0, kind=1, post=0, eps=1e-6, alpha=1.0, rows=4, cols=8, ldx=8, ldy=8, ldr=8, ldo=8, per=0,
             ldg=0, x=16, y=16, g=0, pw=0, pb=0, w=16, b=16, r=32, o=16, s=0):
        return RESIDUAL.pack(0, xt, yt, ot, kind, post, eps, alpha, rows, cols, ldx, ldy, ldr, ldo, per, ldg, x, y,
                                  g, pw, pb, w, b, r, o, s, 0)

    for bad, text in ((dict(xt=3), "x must be"), (dict(yt=3), "y must be"), (dict(ot=4), "output must be"),
                      (dict(kind=0), "unknown norm"), (dict(post=3), "post norm"), (dict(eps=-1.0), "eps"),
                      (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(y=0, g=16), "without y"),
                      (dict(pw=16), "post weights"), (dict(o=0), "null"), (dict(ot=3), "out_scale"),
                      (dict(s=16), "out_scale"), (dict(r=16, ldr=9), "same row stride"), (dict(ldy=4), "stride"),
                      (dict(g=16, per=2, ldg=4), "stride"), (dict(g=16, per=-1), "negative"), (dict(w=2), "misaligned"),
                      (dict(cols=16385), "row length")):
        refused("m3r_residual_norm", norm(**bad), text)

    def rope(dt=0, axes=1, bits=64, b=1, t=4, d=64, n=32, pos=16, f=16, x=16, o=16, h=2, xt=128, ot=128):
        return ROPE.pack(0, dt, 0, axes, bits, 1.0, b, t, d, n, 0, 0, 1, pos, f, x, o, h, 0, xt, 64, 0, ot, 64,
                              *(0,) * 9, 0)

    for bad, text in ((dict(dt=3), "values must be"), (dict(axes=3), "axes"), (dict(bits=16), "positions"),
                      (dict(d=1), "head size"), (dict(n=33), "more frequencies"), (dict(n=0), "more frequencies"),
                      (dict(axes=2, n=31), "even number"), (dict(b=-1), "batch"), (dict(pos=0), "null"),
                      (dict(pos=12), "misaligned"), (dict(x=0), "null"), (dict(h=0), "no tensor"),
                      (dict(h=-1), "heads"), (dict(ot=256), "same strides"), (dict(x=17), "misaligned")):
        refused("m3r_rope", rope(**bad), text)


def test_workspace_sizes():
    from mast3r_runtime_b200 import _lib

    f = _lib.load().m3r_int8_linear_workspace
    assert f(3, 100, 64, 64) == 0 and f(0, 0, 64, 64) == 0
    assert f(1, 1000, 64, 1001) >= 1000 * 1008 + 4000
    for bad in ((4, 1, 1, 1), (0, -1, 1, 1), (0, 1, 0, 1), (0, 1, 1, 0), (0, 1, 1, 131072)):
        assert f(*bad) == -1


def test_python_refusals():
    """Tensors on the CPU and wrong shapes or types raise ValueError."""
    from mast3r_runtime_b200 import ops

    x = torch.zeros(4, 32)
    w, ws = torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_linear(x, w, ws)
    with pytest.raises(ValueError, match="CUDA"):
        ops.residual_norm(x, x, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope(x.view(4, 1, 32), None, torch.arange(4), torch.ones(16, dtype=torch.float64))
    with pytest.raises(ValueError, match="inv_freq"):
        ops.rope(x.view(4, 1, 32), None, torch.arange(4), torch.ones(16))
    with pytest.raises(ValueError, match="n, k"):
        ops.quantize_weight(torch.zeros(3))


def test_rope_frequencies():
    from mast3r_runtime_b200 import ops

    f, a = ops.rope_frequencies(8, base=10000.0, device="cpu")
    assert a == 1.0 and f.dtype == torch.float64
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    g, _ = ops.rope_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    torch.testing.assert_close(g, f / 4)
    g, _ = ops.rope_frequencies(8, scaling="ntk", factor=4.0, device="cpu")
    torch.testing.assert_close(g[[0, -1]], torch.tensor([1.0, 0.001 / 4], dtype=torch.float64))
    g, a = ops.rope_frequencies(128, scaling="by_parts", factor=8.0, device="cpu")
    f, _ = ops.rope_frequencies(128, device="cpu")
    assert g[0] == f[0] and g[-1] == f[-1] / 8 and a > 1 and bool((g <= f).all()) and bool((g >= f / 8).all())
    g, _ = ops.rope_frequencies(64, base=100.0, axes=2, device="cpu")
    assert g.numel() == 32 and torch.equal(g[:16], g[16:]) and abs(float(g[1]) - 100 ** (-1 / 16)) < 1e-12
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=6, axes=2), dict(rot_dim=8, scaling="x"),
                dict(rot_dim=8, factor=0.5), dict(rot_dim=8, base=0.0), dict(rot_dim=8, axes=3)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**bad, device="cpu")


def test_column_walk_near_the_largest_n(tmp_path):
    """The few-row product accepts n up to 2^31 - 257: no warp leaves the columns, and each column is
    one warp's."""
    src = tmp_path / "walk.cpp"
    src.write_text(textwrap.dedent("""
        #include <stdint.h>
        #include <stdio.h>
        #include <initializer_list>
        #include "column_walk.h"
        // the last column that the warp starting at `at` reaches, or -1 when a group lies outside
        static long long last(uint32_t at, uint32_t step, uint32_t n) {
          m3r::ColumnWalk w{at, step, n};
          long long groups = 0, end = 0;
          for (; w.live(); w.next()) {
            for (uint32_t i = 0; i < 4; ++i)
              if (w.column(i) >= n || (long long)w.column(i) < end) return -1;
            end = w.column(3);
            if (++groups > (long long)n / step + 1) return -1;
          }
          return groups == (n - at + step - 1LL) / step ? end : -1;
        }
        int main() {
          const uint32_t step = 148 * 2 * 8 * 4;
          const uint32_t ns[] = {2147483391u, 2147483391u - 9471u, 2147474176u, 2147483390u, 9473u, 5u};
          for (uint32_t n : ns)
            for (uint32_t at : {0u, 4u, step / 2, step - 8, step - 4})
              if (at < n) {
                const long long e = last(at, step, n);
                if (e < 0 || e >= n || e + step < n) return printf("n %u from %u: %lld\\n", n, at, e), 1;
              }
          return 0;
        }
    """))
    exe = tmp_path / "walk"
    csrc = ROOT / "mast3r_runtime_b200" / "csrc"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(csrc), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout


@pytest.mark.parametrize("n_freq", [2 ** 62, 2 ** 62 + 16, 2 ** 63 - 1, 2 ** 32 + 16, 33])
def test_rope_frequency_counts_that_do_not_fit_32_bits(n_freq):
    refused("m3r_rope", ROPE.pack(0, 0, 0, 1, 64, 1.0, 1, 4, 64, n_freq, 0, 0, 1, 16, 16, 16, 16, 2, 0, 128, 64, 0, 128,
                                  64, *(0,) * 9, 0), "more frequencies")


def qkv(batch=2, tokens=5, heads=3, dim=8):
    return torch.zeros(batch, tokens, 3, heads, dim).unbind(2)


def rope_args(q, dim=8):
    return torch.arange(q.shape[-3]), torch.ones(dim // 2, dtype=torch.float64)


SHARED = "share memory|shares memory"


def test_rope_results_that_share_memory_are_refused():
    """A result may be its own input, and nothing else that the call reads or writes."""
    from mast3r_runtime_b200 import ops

    q, k, v = qkv()
    flat = torch.zeros(4000)
    freq = torch.ones(4, dtype=torch.float64)
    pos = torch.arange(5)
    strided = flat.as_strided((2, 5, 3, 8), (120, 20, 8, 1))  # a token's heads reach into the next token
    for kw in (dict(q=q, k=q, inplace=True), dict(q=q, k=q[:, :, 1:], inplace=True),
               dict(q=flat[:240].view(2, 5, 3, 8), k=flat[4:244].view(2, 5, 3, 8), inplace=True),
               dict(q=strided, k=None, inplace=True), dict(q=q, k=None, out=(strided, None)),
               dict(q=q, k=k, out=(v, v)), dict(q=q, k=k, out=(k, q)), dict(q=q, k=k, out=(k, v)),
               dict(q=q, k=k, out=(v, q)), dict(q=q, k=None, out=(q.as_strided(q.shape, (24, 48, 8, 1), 200), None)),
               dict(q=flat[:240].view(2, 5, 3, 8), k=None, out=(flat[8:248].view(2, 5, 3, 8), None)),
               dict(q=q.expand(2, 5, 3, 8), k=None, out=(flat[:24].expand(2, 5, 24).view(2, 5, 3, 8), None))):
        with pytest.raises(ValueError, match=SHARED):
            ops.rope(positions=pos, inv_freq=freq, **kw)
    whole = torch.zeros(2, 5, 3, 8)
    for data in (torch.zeros(60, dtype=torch.int64), torch.zeros(60, dtype=torch.float64)):
        as_float = data.view(torch.float32)
        with pytest.raises(ValueError, match=SHARED):
            ops.rope(as_float[:120].view(5, 3, 8), None, data[:5] if data.dtype is torch.int64 else pos,
                     data[:4] if data.dtype is torch.float64 else freq, inplace=True)
    # views that lie between one another without sharing an element get as far as the device
    planes = torch.zeros(2, 3, 5, 8)
    for kw in (dict(q=q, k=k, inplace=True), dict(q=q, k=k, out=(q, k)), dict(q=q, k=k, out=(v, k)),
               dict(q=q, k=None, out=(v, None)), dict(q=q, k=k, out=(planes.transpose(1, 2), whole)),
               dict(q=q[:, :, :1], k=q[:, :, 1:], inplace=True), dict(q=q[:1], k=q[1:], inplace=True),
               dict(q=q[..., :8:1], k=None, out=(planes.transpose(1, 2), None)), dict(q=q, k=q)):
        with pytest.raises(ValueError, match="CUDA"):
            ops.rope(positions=pos, inv_freq=freq, **kw)


def test_interleaved_views_against_every_offset():
    """The test of shared memory against a list of addresses, at every offset between two views."""
    from mast3r_runtime_b200 import ops

    flat = torch.zeros(4096)
    freq = torch.ones(2, dtype=torch.float64)

    def cells(t):
        at = torch.tensor([t.storage_offset()])
        for n, s in zip(t.shape, t.stride()):
            at = (at[:, None] + torch.arange(n) * s).reshape(-1)
        return at.tolist()

    seen = {True: 0, False: 0}
    for shape, a, b in (((2, 3, 2, 4), (60, 20, 8, 1), (60, 20, 8, 1)), ((2, 3, 2, 4), (60, 20, 8, 1), (40, 8, 20, 1)),
                        ((3, 2, 2, 4), (7, 24, 60, 1), (7, 24, 60, 1)), ((2, 3, 2, 4), (4, 16, 8, 1), (48, 8, 4, 1)),
                        ((1, 4, 3, 4), (0, 12, 4, 1), (0, 5, 24, 1)), ((2, 2, 2, 4), (64, 16, 32, 1), (64, 16, 32, 1)),
                        ((2, 2, 2, 4), (64, 16, 32, 1), (32, 64, 16, 1))):
        for off in range(0, 130):
            x, y = flat.as_strided(shape, a, 70), flat.as_strided(shape, b, off)
            twice = any(len(set(cells(t))) != len(cells(t)) for t in (x, y))
            same = off == 70 and a == b
            shared = twice or bool(set(cells(x)) & set(cells(y)))
            with pytest.raises(ValueError, match=SHARED if shared else "CUDA"):
                ops.rope(x, y, torch.arange(shape[1]), freq, inplace=True)
            if not same:
                with pytest.raises(ValueError, match=SHARED if shared else "CUDA"):
                    ops.rope(x, None, torch.arange(shape[1]), freq, out=(y, None))
            seen[shared] += 1
    assert min(seen.values()) > 40  # both answers are well covered


def test_residual_norm_in_place_over_its_inputs_is_refused():
    from mast3r_runtime_b200 import ops

    flat = torch.zeros(400)
    x = flat[40:360].view(10, 32)
    for kw in (dict(y=flat[8:328].view(10, 32)), dict(y=x.flip(0), weight=x[3]), dict(y=x, gate=x[9]),
               dict(y=None, bias=flat[30:62]), dict(y=x, post_norm="rms", post_weight=x[0]),
               dict(y=x, post_norm="rms", post_bias=flat[350:382]), dict(y=x.new_zeros(10, 32), gate=x[:2])):
        with pytest.raises(ValueError, match=SHARED):
            ops.residual_norm(x, kw.pop("y"), kw.pop("weight", None), inplace=True, **kw)
    wide = torch.zeros(10, 96)
    for kw in (dict(x=x, y=x), dict(x=x, y=None, weight=flat[:32]), dict(x=wide[:, :32], y=wide[:, 32:64]),
               dict(x=wide[:, 8:40], y=wide[:, 40:72], weight=wide[0, 72:].repeat(2)[:32])):
        with pytest.raises(ValueError, match="CUDA"):
            ops.residual_norm(kw.pop("x"), kw.pop("y"), kw.pop("weight", None), inplace=True, **kw)


def test_tangents_are_refused():
    """A forward-mode derivative would be dropped; without forward mode the value alone is used."""
    import torch.autograd.forward_ad as fwd

    from mast3r_runtime_b200 import ops

    x, w, ws = torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    q, pos, f = x.view(4, 1, 32), torch.arange(4), torch.ones(16, dtype=torch.float64)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        for call in (lambda: ops.quantize_rows(dual(x)), lambda: ops.int8_linear(dual(x), w, ws),
                     lambda: ops.int8_linear(x, w, ws, dual(ws)), lambda: ops.residual_norm(x, dual(x), None),
                     lambda: ops.residual_norm(x, x, None, gate=dual(x[0])), lambda: ops.rope(dual(q), None, pos, f),
                     lambda: ops.rope(q, q.clone(), pos, dual(f)), lambda: ops.quantize_weight(dual(x))):
            with pytest.raises(ValueError, match="gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
                call()
            with torch.inference_mode(), pytest.raises(ValueError, match="CUDA"):
                call()
        with pytest.raises(ValueError, match="CUDA"):
            ops.quantize_rows(x)


def test_tensors_whose_memory_is_not_their_values_are_refused():
    """The imaginary part of a conjugate is its memory with the sign still to change; a tensor of
    symbolic zeros has no memory."""
    from mast3r_runtime_b200 import ops

    lazy = torch.zeros(4, 32, dtype=torch.complex64).conj().imag
    assert lazy.is_neg()
    zero = torch._efficientzerotensor(4, 32)
    x, w, ws = torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    pos, f = torch.arange(4), torch.ones(16, dtype=torch.float64)
    for t in (lazy, zero):
        for call in (lambda: ops.quantize_rows(t), lambda: ops.int8_linear(t, w, ws),
                     lambda: ops.residual_norm(x, t, None), lambda: ops.residual_norm(t, None, None, inplace=True),
                     lambda: ops.residual_norm(x, x, t[0]), lambda: ops.rope(t.view(4, 1, 32), None, pos, f)):
            with pytest.raises(ValueError, match="values in memory"):
                call()
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_rows(lazy.resolve_neg())


@pytest.mark.parametrize("flag", [torch.zeros(2), "meta"])
def test_flags_without_a_truth_value_are_refused(flag):
    from mast3r_runtime_b200 import ops

    if flag == "meta":
        flag = torch.zeros((), device="meta")
    x = torch.zeros(4, 1, 32)
    with pytest.raises(ValueError, match="true or false"):
        ops.residual_norm(x[:, 0], x[:, 0], None, inplace=flag)
    for kw in (dict(inplace=flag), dict(interleaved=flag)):
        with pytest.raises(ValueError, match="true or false"):
            ops.rope(x, None, torch.arange(4), torch.ones(16, dtype=torch.float64), **kw)


@pytest.mark.parametrize("device", [-1, 16, 2 ** 31 - 1])
def test_device_numbers_out_of_range_are_bad_arguments(device):
    refused("m3r_quantize_rows", QUANTIZE.pack(device, 0, 2, 8, 8, 16, 16, 16, 16, 0), "device")
    refused("m3r_int8_linear", LINEAR.pack(device, 3, 1, 0, 4, 32, 64, 64, 64, 32, 256, 256, 256, 256, 0, 256, 0, 0, 0),
            "device")
    refused("m3r_residual_norm", RESIDUAL.pack(device, 2, 0, 0, 1, 0, 1e-6, 1.0, 4, 8, 8, 8, 8, 8, 0, 0, 16, 16, 0, 0, 0,
                                               16, 16, 32, 16, 0, 0), "device")
    refused("m3r_rope", ROPE.pack(device, 0, 0, 1, 64, 1.0, 1, 4, 64, 32, 0, 0, 1, 16, 16, 16, 16, 2, 0, 128, 64, 0, 128,
                                  64, *(0,) * 9, 0), "device")
    from mast3r_runtime_b200 import _lib

    assert _lib.load().m3r_operator_status(device, None) == -1


def test_the_same_view_by_other_strides_of_single_dimensions():
    """Strides of dimensions of size 1 are of no meaning."""
    from mast3r_runtime_b200 import ops

    flat = torch.zeros(2, 24)
    q = flat[:1].view(1, 1, 3, 8)
    freq = torch.ones(4, dtype=torch.float64)
    for strides in ((1, 24, 8, 1), (0, 0, 8, 1), (77, 5, 8, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            ops.rope(q, None, torch.zeros(1, dtype=torch.int64), freq, out=(q.as_strided(q.shape, strides), None))
    with pytest.raises(ValueError, match="CUDA"):
        ops.residual_norm(flat[:1], flat[:1].as_strided((1, 24), (3, 1)), None, inplace=True)
    with pytest.raises(ValueError, match=SHARED):
        ops.rope(q, None, torch.zeros(1, dtype=torch.int64), freq, out=(q.as_strided(q.shape, (0, 0, 8, 1), 1), None))
