// C ABI of the operators on device buffers (include/m3r_cuda.h): argument checks, device
// selection and exception -> status code mapping.  Every check comes before the first call
// into the CUDA runtime.
#include <limits>
#include <string>

#include "../../include/m3r_cuda.h"
#include "ops.h"
#include "tmap.h"

namespace m3r {
void set_global_error(const std::string& msg);  // api.cpp: the text m3r_global_error() returns
}

namespace {

constexpr int64_t kMaxExtent = int64_t(1) << 40;  // row strides: past any device's memory

template <class F>
int guarded(F&& fn) {
    try {
        fn();
        m3r::set_global_error("");
        return M3R_OK;
    } catch (const m3r::Error& x) {
        m3r::set_global_error(x.what());
        return x.code;
    } catch (const std::bad_alloc&) {
        m3r::set_global_error("host allocation failed");
        return M3R_ERR_NOMEM;
    } catch (const std::exception& x) {
        m3r::set_global_error(x.what());
        return M3R_ERR_CUDA;
    }
}

// The call's device for the scope; leaves the runtime alone when it is current already.
struct OpDevice {
    int prev = 0;
    bool set;
    explicit OpDevice(int dev) {
        M3R_CUDA(cudaGetDevice(&prev));
        set = prev != dev;
        if (set) M3R_CUDA(cudaSetDevice(dev));
    }
    ~OpDevice() {
        if (set) cudaSetDevice(prev);
    }
};

void check_device(const char* op, int dev) {
    M3R_REQUIRE(dev >= 0 && dev < M3R_MAX_DEVICES, std::string(op) + ": bad device");
}

bool is_float(int dt) { return dt == M3R_DTYPE_BF16 || dt == M3R_DTYPE_F16 || dt == M3R_DTYPE_F32; }

// `p` is aligned to its elements
bool elem_aligned(const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) % m3r::op_size(dt) == 0; }
bool f32_aligned(const float* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

void check_rows(const char* op, int64_t rows, int64_t cols) {
    const std::string s(op);
    M3R_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) - 256, s + ": rows out of range");
    M3R_REQUIRE(cols >= 1 && cols <= m3r::kRowMaxCols,
                s + ": row length out of range (1 to " + std::to_string(m3r::kRowMaxCols) + ")");
}

void check_ld(const char* what, int64_t ld, int64_t cols) {
    M3R_REQUIRE(ld >= cols && ld < kMaxExtent, std::string(what) + ": row stride shorter than a row or out of range");
}

m3r::RowNormParams quantize_params(const m3r_quantize_args& a) {
    check_rows("quantize_rows", a.rows, a.cols);
    M3R_REQUIRE(is_float(a.dtype), "quantize_rows: x must be bf16, fp16 or fp32");
    check_ld("quantize_rows: x", a.ldx, a.cols);
    check_ld("quantize_rows: q", a.ldq, a.cols);
    M3R_REQUIRE(a.rows == 0 || (a.x && a.q && a.scale), "quantize_rows: null buffer");
    M3R_REQUIRE(elem_aligned(a.x, a.dtype) && f32_aligned(a.scale), "quantize_rows: misaligned buffer");
    m3r::RowNormParams p = {};
    p.rows = a.rows;
    p.cols = static_cast<int>(a.cols);
    p.x_dt = a.dtype;
    p.out_dt = m3r::OP_I8;
    p.alpha = 1.0f;
    p.ldx = a.ldx;
    p.ldo = a.ldq;
    p.x = a.x;
    p.out = a.q;
    p.out_scale = a.scale;
    return p;
}

}  // namespace

extern "C" {

int m3r_quantize_rows(const m3r_quantize_args* args) {
    return guarded([&] {
        M3R_REQUIRE(args != nullptr, "quantize_rows: null arguments");
        check_device("quantize_rows", args->device);
        const m3r::RowNormParams p = quantize_params(*args);
        OpDevice g(args->device);
        m3r::row_norm(static_cast<cudaStream_t>(args->stream), p);
    });
}

int64_t m3r_int8_linear_workspace(int x_dtype, int64_t rows, int64_t n, int64_t k) {
    int64_t bytes = 0;
    const int rc = guarded([&] {
        M3R_REQUIRE(is_float(x_dtype) || x_dtype == M3R_DTYPE_I8, "int8_linear_workspace: unknown type of x");
        M3R_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) - 256 && n >= 1 && n < (int64_t(1) << 31) - 256 && k >= 1 &&
                        k <= m3r::kInt8MaxK,
                    "int8_linear_workspace: sizes out of range");
        bytes = static_cast<int64_t>(
            m3r::int8_linear_workspace(x_dtype, rows, static_cast<int>(n), static_cast<int>(k)));
    });
    return rc == M3R_OK ? bytes : rc;
}

int m3r_int8_linear(const m3r_int8_linear_args* args) {
    return guarded([&] {
        M3R_REQUIRE(args != nullptr, "int8_linear: null arguments");
        check_device("int8_linear", args->device);
        const m3r_int8_linear_args& a = *args;
        M3R_REQUIRE(is_float(a.x_dtype) || a.x_dtype == M3R_DTYPE_I8, "int8_linear: x must be bf16, fp16, fp32 or int8");
        M3R_REQUIRE(is_float(a.out_dtype), "int8_linear: the output must be bf16, fp16 or fp32");
        M3R_REQUIRE(a.act >= M3R_ACT_NONE && a.act <= M3R_ACT_RELU, "int8_linear: unknown activation");
        M3R_REQUIRE(a.rows >= 0 && a.rows < (int64_t(1) << 31) - 256, "int8_linear: rows out of range");
        M3R_REQUIRE(a.n >= 1 && a.n < (int64_t(1) << 31) - 256, "int8_linear: n out of range");
        const bool int8_x = a.x_dtype == M3R_DTYPE_I8;
        M3R_REQUIRE(a.k >= 1 && a.k <= (int8_x ? m3r::kInt8MaxK : m3r::kRowMaxCols),
                    "int8_linear: k out of range (1 to 131071 for 8-bit rows, to 16384 for rows to quantise)");
        check_ld("int8_linear: x", a.ldx, a.k);
        check_ld("int8_linear: w", a.ldw, a.k);
        check_ld("int8_linear: out", a.ldo, a.n);
        M3R_REQUIRE(a.w && a.w_scale && (a.rows == 0 || (a.x && a.out)), "int8_linear: null buffer");
        M3R_REQUIRE(int8_x == (a.x_scale != nullptr) || a.rows == 0,
                    "int8_linear: x_scale belongs to 8-bit rows, and to them only");
        M3R_REQUIRE(reinterpret_cast<uintptr_t>(a.w) % 16 == 0 && a.ldw % 16 == 0,
                    "int8_linear: the weights' rows must be 16-byte aligned (pad k to a multiple of 16)");
        M3R_REQUIRE(!int8_x || (reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx % 16 == 0),
                    "int8_linear: 8-bit rows of x must be 16-byte aligned (pad k to a multiple of 16)");
        M3R_REQUIRE(elem_aligned(a.x, a.x_dtype) && elem_aligned(a.out, a.out_dtype) && f32_aligned(a.x_scale) &&
                        f32_aligned(a.w_scale) && f32_aligned(a.bias),
                    "int8_linear: misaligned buffer");
        const int64_t need = static_cast<int64_t>(
            m3r::int8_linear_workspace(a.x_dtype, a.rows, static_cast<int>(a.n), static_cast<int>(a.k)));
        M3R_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need),
                    "int8_linear: the workspace is smaller than m3r_int8_linear_workspace says (" +
                        std::to_string(need) + " bytes)");
        M3R_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(a.workspace) % 256 == 0,
                    "int8_linear: the workspace must be 256-byte aligned");
        m3r::Int8LinearParams p = {};
        p.x_dt = a.x_dtype;
        p.out_dt = a.out_dtype;
        p.act = a.act;
        p.rows = a.rows;
        p.n = static_cast<int>(a.n);
        p.k = static_cast<int>(a.k);
        p.ldx = a.ldx;
        p.ldw = a.ldw;
        p.ldo = a.ldo;
        p.x = a.x;
        p.x_scale = a.x_scale;
        p.w = a.w;
        p.w_scale = a.w_scale;
        p.bias = a.bias;
        p.out = a.out;
        p.workspace = a.workspace;
        OpDevice g(a.device);
        m3r::int8_linear(static_cast<cudaStream_t>(a.stream), p);
    });
}

int m3r_residual_norm(const m3r_residual_norm_args* args) {
    return guarded([&] {
        M3R_REQUIRE(args != nullptr, "residual_norm: null arguments");
        check_device("residual_norm", args->device);
        const m3r_residual_norm_args& a = *args;
        check_rows("residual_norm", a.rows, a.cols);
        M3R_REQUIRE(is_float(a.x_dtype), "residual_norm: x must be bf16, fp16 or fp32");
        M3R_REQUIRE(a.y == nullptr || is_float(a.y_dtype), "residual_norm: y must be bf16, fp16 or fp32");
        M3R_REQUIRE(is_float(a.out_dtype) || a.out_dtype == M3R_DTYPE_I8,
                    "residual_norm: the output must be bf16, fp16, fp32 or int8");
        M3R_REQUIRE(a.norm == M3R_NORM_LAYER || a.norm == M3R_NORM_RMS, "residual_norm: unknown norm");
        M3R_REQUIRE(a.post_norm >= M3R_NORM_NONE && a.post_norm <= M3R_NORM_RMS, "residual_norm: unknown post norm");
        M3R_REQUIRE(a.eps >= 0.0f && a.eps <= std::numeric_limits<float>::max(),
                    "residual_norm: eps must be finite and not negative");
        M3R_REQUIRE(a.y != nullptr || (a.gate == nullptr && a.post_norm == M3R_NORM_NONE),
                    "residual_norm: a gate or a post norm without y");
        M3R_REQUIRE(a.post_norm != M3R_NORM_NONE || (a.post_weight == nullptr && a.post_bias == nullptr),
                    "residual_norm: post weights without a post norm");
        M3R_REQUIRE(a.rows == 0 || (a.x && a.out), "residual_norm: null buffer");
        M3R_REQUIRE((a.out_dtype == M3R_DTYPE_I8) == (a.out_scale != nullptr) || a.rows == 0,
                    "residual_norm: out_scale belongs to an 8-bit result, and to it only");
        check_ld("residual_norm: x", a.ldx, a.cols);
        if (a.y) check_ld("residual_norm: y", a.ldy, a.cols);
        if (a.r) check_ld("residual_norm: r", a.ldr, a.cols);
        check_ld("residual_norm: out", a.ldo, a.cols);
        M3R_REQUIRE(a.r != a.x || a.ldr == a.ldx || a.x == nullptr, "residual_norm: r over x needs the same row stride");
        if (a.gate) {
            M3R_REQUIRE(a.rows_per_gate >= 0, "residual_norm: rows_per_gate is negative");
            if (a.rows_per_gate > 0) check_ld("residual_norm: gate", a.ld_gate, a.cols);
        }
        M3R_REQUIRE(elem_aligned(a.x, a.x_dtype) && (!a.y || elem_aligned(a.y, a.y_dtype)) &&
                        elem_aligned(a.r, a.x_dtype) && elem_aligned(a.out, a.out_dtype) && f32_aligned(a.gate) &&
                        f32_aligned(a.post_weight) && f32_aligned(a.post_bias) && f32_aligned(a.weight) &&
                        f32_aligned(a.bias) && f32_aligned(a.out_scale),
                    "residual_norm: misaligned buffer");
        m3r::RowNormParams p = {};
        p.rows = a.rows;
        p.cols = static_cast<int>(a.cols);
        p.x_dt = a.x_dtype;
        p.y_dt = a.y_dtype;
        p.out_dt = a.out_dtype;
        p.norm = a.norm;
        p.post = a.post_norm;
        p.eps = a.eps;
        p.alpha = a.residual_scale;
        p.ldx = a.ldx;
        p.ldy = a.ldy;
        p.ldr = a.ldr;
        p.ldo = a.ldo;
        // the kernel divides in 32 bits; rows are fewer, so that a larger group is one group
        constexpr int64_t kOneGroup = std::numeric_limits<uint32_t>::max();
        p.rows_per_gate = a.rows_per_gate > 0 && a.rows_per_gate < kOneGroup ? a.rows_per_gate : kOneGroup;
        p.ld_gate = a.rows_per_gate > 0 ? a.ld_gate : 0;
        p.x = a.x;
        p.y = a.y;
        p.gate = a.gate;
        p.pw = a.post_weight;
        p.pb = a.post_bias;
        p.w = a.weight;
        p.b = a.bias;
        p.r = a.r;
        p.out = a.out;
        p.out_scale = a.out_scale;
        OpDevice g(a.device);
        m3r::row_norm(static_cast<cudaStream_t>(a.stream), p);
    });
}

int m3r_rope(const m3r_rope_args* args) {
    return guarded([&] {
        M3R_REQUIRE(args != nullptr, "rope: null arguments");
        check_device("rope", args->device);
        const m3r_rope_args& a = *args;
        M3R_REQUIRE(is_float(a.dtype), "rope: values must be bf16, fp16 or fp32");
        M3R_REQUIRE(a.axes == 1 || a.axes == 2, "rope: axes must be 1 or 2");
        M3R_REQUIRE(a.pos_bits == 32 || a.pos_bits == 64, "rope: positions must be 32- or 64-bit integers");
        M3R_REQUIRE(a.dim >= 2 && a.dim <= 4096, "rope: head size out of range (2 to 4096)");
        M3R_REQUIRE(a.n_freq >= 1 && a.n_freq <= a.dim / 2, "rope: more frequencies than pairs of the head");
        M3R_REQUIRE(a.axes == 1 || a.n_freq % 2 == 0, "rope: two axes need an even number of frequencies");
        M3R_REQUIRE(a.batch >= 0 && a.tokens >= 0 && a.batch < (int64_t(1) << 31) && a.tokens < (int64_t(1) << 31) &&
                        a.batch * a.tokens < (int64_t(1) << 31) - 64,
                    "rope: batch or tokens out of range");
        M3R_REQUIRE(a.batch * a.tokens == 0 || (a.positions && a.inv_freq), "rope: null positions or frequencies");
        M3R_REQUIRE(reinterpret_cast<uintptr_t>(a.positions) % (a.pos_bits / 8) == 0 &&
                        reinterpret_cast<uintptr_t>(a.inv_freq) % 8 == 0,
                    "rope: misaligned positions or frequencies");
        m3r::RopeParams p = {};
        int64_t heads = 0;
        for (int i = 0; i < 2; ++i) {
            const m3r_rope_tensor& t = a.t[i];
            M3R_REQUIRE(t.heads >= 0 && t.heads <= 65536, "rope: heads out of range");
            heads += t.heads;
            if (t.heads == 0) continue;
            M3R_REQUIRE(a.batch * a.tokens == 0 || (t.x && t.out), "rope: null tensor");
            M3R_REQUIRE(elem_aligned(t.x, a.dtype) && elem_aligned(t.out, a.dtype), "rope: misaligned tensor");
            M3R_REQUIRE(a.batch * a.tokens == 0 || t.x != t.out ||
                                        ((a.batch == 1 || t.x_batch == t.out_batch) &&
                                         (a.tokens == 1 || t.x_token == t.out_token) &&
                                         (t.heads == 1 || t.x_head == t.out_head)),
                        "rope: a tensor turned in place needs the same strides");
            p.t[i].x = t.x;
            p.t[i].out = t.out;
            p.t[i].heads = static_cast<int>(t.heads);
            p.t[i].xb = a.batch == 1 ? 0 : t.x_batch;
            p.t[i].xt = a.tokens == 1 ? 0 : t.x_token;
            p.t[i].xh = t.heads == 1 ? 0 : t.x_head;
            p.t[i].ob = a.batch == 1 ? 0 : t.out_batch;
            p.t[i].ot = a.tokens == 1 ? 0 : t.out_token;
            p.t[i].oh = t.heads == 1 ? 0 : t.out_head;
        }
        M3R_REQUIRE(heads > 0, "rope: no tensor");
        p.dt = a.dtype;
        p.interleaved = a.interleaved != 0;
        p.axes = a.axes;
        p.n_freq = static_cast<int>(a.n_freq);
        p.dim = static_cast<int>(a.dim);
        p.pos64 = a.pos_bits == 64;
        p.amplitude = a.amplitude;
        p.batch = a.batch;
        p.tokens = a.tokens;
        p.inv_freq = a.inv_freq;
        p.pos = a.positions;
        p.pos_axis = a.pos_axis;
        p.pos_b = a.pos_batch;
        p.pos_t = a.pos_token;
        OpDevice g(a.device);
        m3r::rope(static_cast<cudaStream_t>(a.stream), p);
    });
}

int m3r_operator_status(int device, void* stream) {
    return guarded([&] {
        check_device("operator_status", device);
        OpDevice g(device);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        int first = 0;
        for (int* at : {m3r::int8_linear_status(), m3r::row_norm_status()}) {
            int code = 0;
            M3R_CUDA(cudaMemcpyAsync(&code, at, sizeof(code), cudaMemcpyDeviceToHost, s));
            M3R_CUDA(cudaStreamSynchronize(s));
            if (code == 0) continue;
            M3R_CUDA(cudaMemsetAsync(at, 0, sizeof(code), s));  // the code alone, and before this returns
            M3R_CUDA(cudaStreamSynchronize(s));
            if (first == 0) first = code;
        }
        if (first) throw m3r::Error(m3r::kErrTimeout, "device wait timed out (code " + std::to_string(first) + ")");
    });
}

int m3r_operator_wait_selftest(int device, int which, unsigned long long limit_ns, void* stream) {
    return guarded([&] {
        check_device("operator_wait_selftest", device);
        M3R_REQUIRE(which == 0 || which == 1, "operator_wait_selftest: unknown group of kernels");
        M3R_REQUIRE(limit_ns > 0 && limit_ns <= 10000000000ull, "operator_wait_selftest: limit must be in (0, 10 s]");
        OpDevice g(device);
        m3r::run_out_wait(static_cast<cudaStream_t>(stream), which == 0 ? m3r::int8_linear_status() : m3r::row_norm_status(),
                          limit_ns);
    });
}

}  // extern "C"
