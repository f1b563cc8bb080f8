// torch side of the operators (mast3r_runtime_b200/ops.py): checks the tensors of a call,
// allocates its results and workspace from torch's allocator and calls the C ABI of
// include/m3r_cuda.h on the tensors' device and that device's current stream.  It is compiled
// because a call of a small operator is bound by the host: the same checks, allocations and
// packing in Python took 10 to 16 us, of which the launch itself is under 4.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/m3r_cuda.h"

namespace {

using at::Tensor;

struct ArgError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

[[noreturn]] void fail(const char* op, const std::string& text) { throw ArgError(std::string(op) + ": " + text); }

std::string shape_text(const Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

// A Python argument as a tensor; `none` allows None (an undefined tensor).
Tensor tensor_arg(const char* op, const char* name, PyObject* o, bool none = false) {
    if (THPVariable_Check(o)) {
        const Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided) fail(op, std::string(name) + " must be a dense tensor");
        if (t.is_neg() || t._is_zerotensor())
            fail(op, std::string(name) + " does not hold its values in memory (use resolve_neg() or clone())");
        return t;
    }
    if (none && o == Py_None) return Tensor();
    fail(op, std::string(name) + " must be a tensor" + (none ? " or None" : ""));
}

// The device of a call's tensors.  No gradient is computed, in either mode of differentiation.
int64_t device_of(const char* op, std::initializer_list<const Tensor*> all) {
    int64_t dev = -1;
    const bool grad = c10::GradMode::is_enabled();
    const bool tangent = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor* t : all) {
        if (!t->defined()) continue;
        if (grad && t->requires_grad()) fail(op, "no gradient is computed (use torch.no_grad() or detach the tensors)");
        if (tangent && t->_fw_grad(0).defined())
            fail(op, "no forward-mode gradient is computed (pass the primal: torch.autograd.forward_ad.unpack_dual)");
    }
    for (const Tensor* t : all) {
        if (!t->defined()) continue;
        if (!t->is_cuda()) fail(op, "tensors must be on a CUDA device");
        if (dev < 0) dev = t->get_device();
        if (t->get_device() != dev) fail(op, "tensors are on different devices");
    }
    return dev;
}

// One term of a sum of whole multiples of steps (bytes): step * x with lo <= x <= hi.
struct Term {
    int64_t step, lo, hi;
};

int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0

// Whether the terms can add up to `target`; `moved`: so that an x other than the last term's is not zero.
// Terms come by falling step, so that with the steps of ordinary layouts (each beyond what the smaller
// ones reach together) two or three values of an x are tried; sums that take more than `budget` trials
// count as possible.
bool adds_up(const Term* t, size_t n, int64_t target, bool moved, int& budget) {
    if (n == 0) return target == 0 && moved;
    if (--budget < 0) return true;
    int64_t lo = 0, hi = 0;  // of the terms behind this one
    for (size_t i = 1; i < n; ++i) {
        lo += t[i].step * t[i].lo;
        hi += t[i].step * t[i].hi;
    }
    const int64_t first = std::max(t->lo, -floor_div(hi - target, t->step));
    const int64_t last = std::min(t->hi, floor_div(target - lo, t->step));
    for (int64_t x = first; x <= last; ++x)
        if (adds_up(t + 1, n - 1, target - t->step * x, moved || (x != 0 && n > 1), budget)) return true;
    return false;
}

constexpr int kOverlapTrials = 20000;

bool by_step(const Term& a, const Term& b) { return a.step > b.step; }

// Whether two of a tensor's elements share memory.
bool overlaps_itself(const Tensor& t) {
    if (t.numel() <= 1 || t.is_non_overlapping_and_dense()) return false;
    const int64_t size = static_cast<int64_t>(t.element_size());
    c10::SmallVector<Term, 8> terms;
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) == 1) continue;
        if (t.stride(i) == 0) return true;
        terms.push_back({t.stride(i) * size, 1 - t.size(i), t.size(i) - 1});
    }
    std::sort(terms.begin(), terms.end(), by_step);
    terms.push_back({1, 1 - size, size - 1});
    int budget = kOverlapTrials;
    return adds_up(terms.data(), terms.size(), 0, false, budget);
}

struct Extent {
    int64_t begin, end;  // bytes
    explicit Extent(const Tensor& t) : begin(reinterpret_cast<int64_t>(t.const_data_ptr())), end(begin) {
        for (int64_t i = 0; i < t.dim(); ++i) end += (t.size(i) - 1) * t.stride(i) * static_cast<int64_t>(t.element_size());
        end += static_cast<int64_t>(t.element_size());
    }
};

// Whether an element of `a` shares memory with one of `b`.  Views of one projection lie between one
// another without that.
bool overlaps(const Tensor& a, const Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    const Extent ea(a), eb(b);
    if (ea.end <= eb.begin || eb.end <= ea.begin) return false;
    c10::SmallVector<Term, 16> terms;
    // a's address less b's: a step that both have is one term
    auto add = [&](int64_t step, int64_t lo, int64_t hi) {
        if (step == 0) return;
        for (Term& t : terms)
            if (t.step == step) {
                t.lo += lo;
                t.hi += hi;
                return;
            }
        terms.push_back({step, lo, hi});
    };
    const int64_t sa = static_cast<int64_t>(a.element_size()), sb = static_cast<int64_t>(b.element_size());
    for (int64_t i = 0; i < a.dim(); ++i) add(a.stride(i) * sa, 0, a.size(i) - 1);
    for (int64_t i = 0; i < b.dim(); ++i) add(b.stride(i) * sb, 1 - b.size(i), 0);
    add(1, 1 - sb, sa - 1);
    std::sort(terms.begin(), terms.end(), by_step);
    int budget = kOverlapTrials;
    return adds_up(terms.data(), terms.size(), eb.begin - ea.begin, true, budget);
}

bool same_view(const Tensor& a, const Tensor& b) {
    if (a.const_data_ptr() != b.const_data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

// A tensor that a call writes over: its version counts, and no element is there twice.
void check_written(const char* op, const char* name, const Tensor& t) {
    if (t.is_inference() && !c10::InferenceMode::is_enabled())
        fail(op, std::string(name) + " is an inference tensor and can be written in inference mode only");
    if (overlaps_itself(t)) fail(op, std::string(name) + " has elements that share memory");
}

// What else the call reads or writes; `own`, which each element of the written tensor is made from, may be
// the tensor itself.
void check_apart(const char* op, const char* name, const Tensor& t, const Tensor& own,
                 std::initializer_list<std::pair<const char*, const Tensor*>> others) {
    if (own.defined() && !same_view(t, own) && overlaps(t, own))
        fail(op, std::string(name) + " shares memory with its input and is not the same view");
    for (const auto& o : others)
        if (o.second->defined() && overlaps(t, *o.second))
            fail(op, std::string(name) + " shares memory with " + o.first);
}

int float_code(const char* op, const char* name, at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return M3R_DTYPE_BF16;
        case at::kHalf: return M3R_DTYPE_F16;
        case at::kFloat: return M3R_DTYPE_F32;
        default: fail(op, std::string(name) + " must be bfloat16, float16 or float32, got " + c10::toString(t));
    }
}

// dtype argument: a torch.dtype, or None for `def`
at::ScalarType dtype_arg(const char* op, PyObject* o, at::ScalarType def) {
    if (o == Py_None) return def;
    if (!THPDtype_Check(o)) fail(op, "out_dtype must be a torch.dtype");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

double number_arg(const char* op, const char* name, PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        fail(op, std::string(name) + " must be a number");
    }
    return v;
}

bool bool_arg(const char* op, const char* name, PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        fail(op, std::string(name) + " must be true or false");
    }
    return v == 1;
}

// One of the names in `names` (its index), or `none` for None where that is allowed.
int name_arg(const char* op, const char* what, PyObject* o, std::initializer_list<const char*> names, int none = -1) {
    if (o == Py_None && none >= 0) return none;
    if (PyUnicode_Check(o)) {
        int i = 0;
        for (const char* n : names) {
            if (*n && PyUnicode_CompareWithASCIIString(o, n) == 0) return i;
            ++i;
        }
    }
    std::string text = std::string("unknown ") + what + " (";
    bool first = true;
    for (const char* n : names) {
        if (!*n) continue;
        text += std::string(first ? "" : ", ") + n;
        first = false;
    }
    fail(op, text + ")");
}

struct Rows {
    int64_t rows, cols, ld;
};

// A tensor [..., cols] whose rows are evenly spaced.
Rows rows_of(const char* op, const char* name, const Tensor& t) {
    const int64_t d = t.dim();
    if (d == 0) fail(op, std::string(name) + " must have at least one dimension");
    const auto size = t.sizes(), stride = t.strides();
    Rows r{1, size[d - 1], size[d - 1]};
    int64_t step = -1;  // what the next outer dimension's stride has to be
    for (int64_t i = d - 2; i >= 0; --i) {
        if (size[i] != 1) {
            if (step < 0)
                r.ld = stride[i];
            else if (stride[i] != step && t.numel() > 0)
                fail(op, "the rows of " + std::string(name) + " are not evenly spaced (make it contiguous)");
            step = stride[i] * size[i];
        }
        r.rows *= size[i];
    }
    if (r.cols > 1 && stride[d - 1] != 1) fail(op, "the last dimension of " + std::string(name) + " must be contiguous");
    if (r.ld < r.cols) {
        if (r.rows > 1) fail(op, "the rows of " + std::string(name) + " overlap");
        r.ld = r.cols;
    }
    return r;
}

// Address of a float32 vector of n values (null when undefined).
const float* vector_of(const char* op, const char* name, const Tensor& t, int64_t n) {
    if (!t.defined()) return nullptr;
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != n)
        fail(op, std::string(name) + " must be a float32 tensor of shape [" + std::to_string(n) + "], got " +
                     c10::toString(t.scalar_type()) + " " + shape_text(t));
    if (n > 1 && t.stride(0) != 1) fail(op, std::string(name) + " must be contiguous");
    return t.const_data_ptr<float>();
}

int64_t pad16(int64_t k) { return (k + 15) / 16 * 16; }

Tensor empty(at::IntArrayRef shape, at::ScalarType t, int64_t dev) {
    return at::detail::empty_cuda(shape, t, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt);
}

// An int8 tensor of `like`'s shape with rows on 16-byte boundaries.
Tensor empty_int8_rows(const Tensor& like, const Rows& r, int64_t dev) {
    const int64_t ld = pad16(r.cols);
    if (ld == r.cols) return empty(like.sizes(), at::kChar, dev);
    Tensor q = empty({r.rows, ld}, at::kChar, dev);
    c10::DimVector stride(like.dim(), 1);
    int64_t step = ld;
    for (int64_t i = like.dim() - 2; i >= 0; --i) {
        stride[i] = step;
        step *= like.size(i);
    }
    return q.as_strided(like.sizes(), stride);
}

Tensor empty_row_scales(const Tensor& like, int64_t dev) { return empty(like.sizes().slice(0, like.dim() - 1), at::kFloat, dev); }

void* stream_of(int64_t dev) {
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

// Calls an entry point without the interpreter lock and maps its status.
template <class Args>
void call(int (*fn)(const Args*), const Args& args) {
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = fn(&args);
    Py_END_ALLOW_THREADS;
    if (rc == M3R_OK) return;
    const std::string text = m3r_global_error();
    if (rc == M3R_ERR_ARG) throw ArgError(text);
    throw std::runtime_error(text + " (" + std::to_string(rc) + ")");
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

PyObject* tuple(std::initializer_list<PyObject*> items) {
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
    Py_ssize_t i = 0;
    for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
    return t;
}

PyObject* same(PyObject* o) {
    Py_INCREF(o);
    return o;
}

// ----------------------------------------------------------------------------- operators
// (x)
PyObject* quantize_rows(PyObject* const* a) {
    const char* op = "quantize_rows";
    const Tensor x = tensor_arg(op, "x", a[0]);
    const int64_t dev = device_of(op, {&x});
    m3r_quantize_args p = {};
    p.device = static_cast<int>(dev);
    p.dtype = float_code(op, "x", x.scalar_type());
    const Rows r = rows_of(op, "x", x);
    const Tensor q = empty_int8_rows(x, r, dev);
    const Tensor scale = empty_row_scales(x, dev);
    p.rows = r.rows;
    p.cols = r.cols;
    p.ldx = r.ld;
    p.ldq = pad16(r.cols);
    p.x = x.const_data_ptr();
    p.q = static_cast<int8_t*>(q.mutable_data_ptr());
    p.scale = static_cast<float*>(scale.mutable_data_ptr());
    p.stream = stream_of(dev);
    call(m3r_quantize_rows, p);
    return tuple({wrap(q), wrap(scale)});
}

// (x, weight, weight_scale, bias, act, out_dtype, x_scale)
PyObject* int8_linear(PyObject* const* a) {
    const char* op = "int8_linear";
    const Tensor x = tensor_arg(op, "x", a[0]), w = tensor_arg(op, "weight", a[1]),
                 ws = tensor_arg(op, "weight_scale", a[2]), bias = tensor_arg(op, "bias", a[3], true),
                 xs = tensor_arg(op, "x_scale", a[6], true);
    const int64_t dev = device_of(op, {&x, &w, &ws, &bias, &xs});
    const Rows r = rows_of(op, "x", x);
    if (w.scalar_type() != at::kChar || w.dim() != 2 || w.size(1) != r.cols || w.size(0) < 1 || r.cols < 1)
        fail(op, "weight must be int8 [n, " + std::to_string(r.cols) + "], got " + c10::toString(w.scalar_type()) +
                     " " + shape_text(w));
    m3r_int8_linear_args p = {};
    p.device = static_cast<int>(dev);
    p.rows = r.rows;
    p.k = r.cols;
    p.n = w.size(0);
    p.ldx = r.ld;
    if (p.k > 1 && w.stride(1) != 1) fail(op, "the rows of weight must be contiguous");
    p.ldw = p.n > 1 ? w.stride(0) : pad16(p.k);
    at::ScalarType def = x.scalar_type();
    if (def == at::kChar) {
        if (!xs.defined() || xs.scalar_type() != at::kFloat || xs.sizes() != x.sizes().slice(0, x.dim() - 1) ||
            !xs.is_contiguous())
            fail(op, "int8 rows need x_scale, a contiguous float32 tensor with a value for each row");
        p.x_dtype = M3R_DTYPE_I8;
        p.x_scale = static_cast<const float*>(xs.const_data_ptr());
        if (p.rows == 1) p.ldx = pad16(p.k);
        def = at::kBFloat16;
    } else {
        p.x_dtype = float_code(op, "x", def);
        if (xs.defined()) fail(op, "x_scale belongs to int8 rows");
    }
    const at::ScalarType out_type = dtype_arg(op, a[5], def);
    p.out_dtype = float_code(op, "out_dtype", out_type);
    p.act = name_arg(op, "activation", a[4], {"none", "gelu", "relu"});
    p.w_scale = vector_of(op, "weight_scale", ws, p.n);
    p.bias = vector_of(op, "bias", bias, p.n);
    c10::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = p.n;
    const Tensor out = empty(shape, out_type, dev);
    Tensor work;
    const int64_t need = m3r_int8_linear_workspace(p.x_dtype, p.rows, p.n, p.k);
    if (need < 0) throw ArgError(m3r_global_error());
    if (need > 0) {
        work = empty({need}, at::kByte, dev);
        p.workspace = work.mutable_data_ptr();
        p.workspace_bytes = need;
    }
    p.ldo = p.n;
    p.x = x.const_data_ptr();
    p.w = static_cast<const int8_t*>(w.const_data_ptr());
    p.out = out.mutable_data_ptr();
    p.stream = stream_of(dev);
    call(m3r_int8_linear, p);
    return wrap(out);
}

// (x, y, weight, bias, norm, post_norm, post_weight, post_bias, gate, residual_scale, eps, out_dtype, inplace)
PyObject* residual_norm(PyObject* const* a) {
    const char* op = "residual_norm";
    const Tensor x = tensor_arg(op, "x", a[0]), y = tensor_arg(op, "y", a[1], true),
                 w = tensor_arg(op, "weight", a[2], true), b = tensor_arg(op, "bias", a[3], true),
                 pw = tensor_arg(op, "post_weight", a[6], true), pb = tensor_arg(op, "post_bias", a[7], true),
                 gate = tensor_arg(op, "gate", a[8], true);
    const bool inplace = bool_arg(op, "inplace", a[12]);
    if (inplace) {
        check_written(op, "x", x);
        check_apart(op, "x", x, y, {{"weight", &w}, {"bias", &b}, {"post_weight", &pw}, {"post_bias", &pb}, {"gate", &gate}});
    }
    const int64_t dev = device_of(op, {&x, &y, &w, &b, &pw, &pb, &gate});
    const Rows r = rows_of(op, "x", x);
    m3r_residual_norm_args p = {};
    p.device = static_cast<int>(dev);
    p.x_dtype = float_code(op, "x", x.scalar_type());
    p.rows = r.rows;
    p.cols = r.cols;
    p.ldx = r.ld;
    if (y.defined()) {
        p.y_dtype = float_code(op, "y", y.scalar_type());
        if (y.sizes() != x.sizes()) fail(op, "x and y differ in shape: " + shape_text(x) + " and " + shape_text(y));
        p.ldy = rows_of(op, "y", y).ld;
        p.y = y.const_data_ptr();
    }
    p.norm = name_arg(op, "norm", a[4], {"", "layer", "rms"});
    p.post_norm = name_arg(op, "post norm", a[5], {"", "layer", "rms"}, 0);
    if (gate.defined()) {
        if (gate.dim() == 2) {
            const int64_t groups = gate.size(0);
            if (gate.scalar_type() != at::kFloat || gate.size(1) != r.cols || groups < 1 || r.rows % groups ||
                (r.cols > 1 && gate.stride(1) != 1) || (groups > 1 && gate.stride(0) < r.cols))
                fail(op, "gate must be float32 [groups, " + std::to_string(r.cols) + "] with groups dividing " +
                             std::to_string(r.rows) + " rows, got " + c10::toString(gate.scalar_type()) + " " +
                             shape_text(gate));
            p.rows_per_gate = r.rows / groups;
            p.ld_gate = groups > 1 ? gate.stride(0) : r.cols;
            p.gate = static_cast<const float*>(gate.const_data_ptr());
        } else {
            p.gate = vector_of(op, "gate", gate, r.cols);
        }
    }
    p.post_weight = vector_of(op, "post_weight", pw, r.cols);
    p.post_bias = vector_of(op, "post_bias", pb, r.cols);
    p.weight = vector_of(op, "weight", w, r.cols);
    p.bias = vector_of(op, "bias", b, r.cols);
    p.residual_scale = static_cast<float>(number_arg(op, "residual_scale", a[9]));
    p.eps = static_cast<float>(number_arg(op, "eps", a[10]));
    const at::ScalarType out_type = dtype_arg(op, a[11], (y.defined() ? y : x).scalar_type());
    const Tensor res = inplace ? x : empty(x.sizes(), x.scalar_type(), dev);
    p.ldr = inplace ? r.ld : r.cols;
    Tensor out, scale;
    if (out_type == at::kChar) {
        p.out_dtype = M3R_DTYPE_I8;
        out = empty_int8_rows(x, r, dev);
        scale = empty_row_scales(x, dev);
        p.ldo = pad16(r.cols);
        p.out_scale = static_cast<float*>(scale.mutable_data_ptr());
    } else {
        p.out_dtype = float_code(op, "out_dtype", out_type);
        out = empty(x.sizes(), out_type, dev);
        p.ldo = r.cols;
    }
    p.x = x.const_data_ptr();
    p.r = res.mutable_data_ptr();
    p.out = out.mutable_data_ptr();
    p.stream = stream_of(dev);
    call(m3r_residual_norm, p);
    if (inplace) res.unsafeGetTensorImpl()->bump_version();  // a graph that saved x notices
    PyObject* first = inplace ? same(a[0]) : wrap(res);
    return scale.defined() ? tuple({first, wrap(out), wrap(scale)}) : tuple({first, wrap(out)});
}

void rope_tensor(const char* op, const char* name, const Tensor& x, const Tensor& out, const Tensor& ref,
                 m3r_rope_tensor& t) {
    const int64_t d = x.dim();
    if ((d != 3 && d != 4) || d != ref.dim() || x.size(d - 1) != ref.size(d - 1) ||
        x.sizes().slice(0, d - 2) != ref.sizes().slice(0, d - 2))
        fail(op, std::string(name) + " must be [tokens, heads, dim] or [batch, tokens, heads, dim] as q is, got " +
                     shape_text(x));
    if (x.scalar_type() != ref.scalar_type()) fail(op, "q and k differ in type");
    const auto s = x.strides(), o = out.strides();
    if (s[d - 1] != 1 || o[d - 1] != 1) fail(op, "the last dimension of " + std::string(name) + " must be contiguous");
    t.x = x.const_data_ptr();
    t.out = out.mutable_data_ptr();
    t.heads = x.size(d - 2);
    t.x_batch = d == 4 ? s[0] : 0;
    t.x_token = s[d - 3];
    t.x_head = s[d - 2];
    t.out_batch = d == 4 ? o[0] : 0;
    t.out_token = o[d - 3];
    t.out_head = o[d - 2];
}

// (q, k, positions, inv_freq, amplitude, interleaved, axes, inplace, q_out, k_out)
PyObject* rope(PyObject* const* a) {
    const char* op = "rope";
    const Tensor q = tensor_arg(op, "q", a[0]), k = tensor_arg(op, "k", a[1], true),
                 pos = tensor_arg(op, "positions", a[2]), f = tensor_arg(op, "inv_freq", a[3]),
                 oq0 = tensor_arg(op, "out", a[8], true), ok0 = tensor_arg(op, "out", a[9], true);
    if (f.scalar_type() != at::kDouble || f.dim() != 1 || f.size(0) < 1 || (f.size(0) > 1 && f.stride(0) != 1))
        fail(op, "inv_freq must be a contiguous float64 vector");
    const bool inplace = bool_arg(op, "inplace", a[7]), interleaved = bool_arg(op, "interleaved", a[5]);
    Tensor oq, ok;
    if (inplace) {
        if (oq0.defined() || ok0.defined()) fail(op, "inplace and out exclude each other");
        oq = q;
        ok = k;
    } else if (oq0.defined() || ok0.defined()) {
        oq = oq0;
        ok = ok0;
        if (!oq.defined() || oq.sizes() != q.sizes() || oq.scalar_type() != q.scalar_type() ||
            ok.defined() != k.defined() ||
            (k.defined() && (ok.sizes() != k.sizes() || ok.scalar_type() != k.scalar_type())))
            fail(op, "out must match q and k in shape and type");
    }
    if (oq.defined()) {
        check_written(op, "q's result", oq);
        if (ok.defined()) {
            check_written(op, "k's result", ok);
            check_apart(op, "k's result", ok, k, {{"q's result", &oq}, {"q", &q}, {"positions", &pos}, {"inv_freq", &f}});
        }
        check_apart(op, "q's result", oq, q, {{"k", &k}, {"positions", &pos}, {"inv_freq", &f}});
    }
    const int64_t dev = device_of(op, {&q, &k, &pos, &f, &oq0, &ok0});
    m3r_rope_args p = {};
    p.device = static_cast<int>(dev);
    p.dtype = float_code(op, "q", q.scalar_type());
    if (!oq.defined()) {
        oq = empty(q.sizes(), q.scalar_type(), dev);
        if (k.defined()) ok = empty(k.sizes(), k.scalar_type(), dev);
    }
    rope_tensor(op, "q", q, oq, q, p.t[0]);
    if (k.defined()) rope_tensor(op, "k", k, ok, q, p.t[1]);
    const int64_t d = q.dim();
    p.batch = d == 4 ? q.size(0) : 1;
    p.tokens = q.size(d - 3);
    p.dim = q.size(d - 1);
    p.n_freq = f.size(0);
    p.amplitude = static_cast<float>(number_arg(op, "amplitude", a[4]));
    p.interleaved = interleaved;
    const double axes = number_arg(op, "axes", a[6]);
    if (axes != 1 && axes != 2) fail(op, "axes must be 1 or 2");
    p.axes = static_cast<int>(axes);
    p.pos_bits = pos.scalar_type() == at::kLong ? 64 : pos.scalar_type() == at::kInt ? 32 : 0;
    if (p.pos_bits == 0) fail(op, "positions must be int32 or int64");
    const int64_t lead = p.axes - 1, pd = pos.dim();
    if ((pd != lead + 1 && pd != lead + 2) || (lead && pos.size(0) != 2) || pos.size(pd - 1) != p.tokens ||
        (pd == lead + 2 && pos.size(lead) != 1 && pos.size(lead) != p.batch))
        fail(op, "positions " + shape_text(pos) + " do not fit " + std::to_string(p.axes) + " axes, batch " +
                     std::to_string(p.batch) + " and " + std::to_string(p.tokens) + " tokens");
    p.pos_axis = lead ? pos.stride(0) : 0;
    p.pos_batch = pd == lead + 2 && pos.size(lead) > 1 ? pos.stride(lead) : 0;
    p.pos_token = pos.stride(pd - 1);
    p.positions = pos.const_data_ptr();
    p.inv_freq = static_cast<const double*>(f.const_data_ptr());
    p.stream = stream_of(dev);
    call(m3r_rope, p);
    if (inplace || oq0.defined()) {  // a graph that saved them notices
        oq.unsafeGetTensorImpl()->bump_version();
        if (ok.defined()) ok.unsafeGetTensorImpl()->bump_version();
    }
    PyObject* rq = inplace ? same(a[0]) : oq0.defined() ? same(a[8]) : wrap(oq);
    PyObject* rk = !k.defined() ? same(Py_None) : inplace ? same(a[1]) : ok0.defined() ? same(a[9]) : wrap(ok);
    return tuple({rq, rk});
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const ArgError& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ENTRY(quantize_rows, 1), ENTRY(int8_linear, 7), ENTRY(residual_norm, 13), ENTRY(rope, 10),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&kModule); }
