// Host interface of the operators on caller-owned device buffers (row_norm.cu, rope.cu,
// int8_linear.cu).  Argument checks are in ops_api.cpp; these launchers take checked
// arguments, run on the current device and only queue work on the stream.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace m3r {

// Element types of operator buffers (M3R_DTYPE_* of the C ABI).
enum OpDt : int { OP_BF16 = 0, OP_F16 = 1, OP_F32 = 2, OP_I8 = 3 };
enum NormKind : int { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };

inline int op_size(int dt) { return dt == OP_F32 ? 4 : dt == OP_I8 ? 1 : 2; }

constexpr int kRowMaxCols = 16384;  // longest row the row kernels hold in registers
constexpr int64_t kInt8MaxK = 131071;  // sums of two 8-bit values, -128 among them, stay below 2^31

// One pass over rows of `cols` values:  r = alpha x + gate * post(y),  h = norm(r) w + b.
struct RowNormParams {
    long long rows;
    int cols;
    int x_dt, y_dt, out_dt;
    int norm, post;
    float eps, alpha;
    long long ldx, ldy, ldr, ldo, ld_gate;  // elements
    long long rows_per_gate;
    const void* x;
    const void* y;      // may be null
    const float* gate;  // may be null
    const float* pw;    // post-norm weight / bias, may be null
    const float* pb;
    const float* w;     // norm weight / bias, may be null
    const float* b;
    void* r;            // may be null: the stream is not written
    void* out;
    float* out_scale;   // rows of an 8-bit result
};
void row_norm(cudaStream_t s, const RowNormParams& p);
// Device address of the code that the first wait of a row kernel to run out on the current device leaves
// (0: none).
int* row_norm_status();

// Rotary positions on up to two tensors [batch, tokens, heads, dim].
struct RopeTensor {
    const void* x;
    void* out;
    int heads;
    long long xb, xt, xh;  // element strides of batch, token, head
    long long ob, ot, oh;
};
struct RopeParams {
    int dt, interleaved, axes, n_freq, dim, pos64;
    float amplitude;
    long long batch, tokens;
    RopeTensor t[2];  // t[1].heads may be 0
    const double* inv_freq;
    const void* pos;
    long long pos_axis, pos_b, pos_t;  // element strides
};
void rope(cudaStream_t s, const RopeParams& p);

// Product in 8-bit integers (int8_linear.cu).
struct Int8LinearParams {
    int x_dt, out_dt, act;
    long long rows;
    int n, k;
    long long ldx, ldw, ldo;  // elements
    const void* x;
    const float* x_scale;  // x_dt == OP_I8
    const int8_t* w;
    const float* w_scale;
    const float* bias;  // may be null
    void* out;
    void* workspace;
};
size_t int8_linear_workspace(int x_dt, long long rows, int n, int k);
void int8_linear(cudaStream_t s, const Int8LinearParams& p);
// The same for the product's kernels.
int* int8_linear_status();

// selftest.cu: queues one warp that waits `limit_ns` for a signal that nothing sends and leaves the code of
// that at `status`, where it is 0.
void run_out_wait(cudaStream_t s, int* status, unsigned long long limit_ns);

}  // namespace m3r
