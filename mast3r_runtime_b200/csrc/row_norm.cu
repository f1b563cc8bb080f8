// Row operators in one pass over a row held in registers:
//
//   t = y,  or post-normalised  N(y) * pw + pb
//   r = alpha * x + gate * t                 (the new residual stream)
//   h = N(r) * w + b                         (the next block's input)
//
// with N the layer norm (v - mean) / sqrt(var + eps) or the RMS norm v / sqrt(mean(v^2) + eps),
// or no norm.  h leaves in 16 or 32 bits, or in 8 bits with a scale for the row:
// a = max |h|, q = the integer nearest to 127 h / a (ties to even), scale = a / 127.
//
// The work is bound by HBM: x, y in, r, h out, each once.  A row of at most 1,024 values
// belongs to one warp or a part of one (statistics by shuffles, no block barrier), a longer one to one
// block; x and y are loaded before the first reduction so that a warp keeps its whole
// row's bytes in flight.  All statistics are 32-bit, the variance in two passes over the
// registers.
#include "common.cuh"
#include "launch.h"
#include "ops.h"
#include "quantize.cuh"
#include "tmap.h"

namespace m3r {

namespace {

// First wait of a row kernel that ran out on this device (see mbar_wait).
__device__ DevStatus g_status;

__device__ __forceinline__ uint32_t op_bytes(int dt) { return dt == OP_F32 ? 4u : 2u; }

// The N = 8 * NCH values of a thread.  VEC: chunk c holds elements (tid + c * G) * 8 .. + 8
// of the row (one 16-byte access of a 16-bit type); else value i is element tid + i * G, with G
// (GT, the block's threads) known to the compiler, so that an access is one instruction.
template <bool VEC, int NCH, int GT>
struct RowSlice {
    int tid, D, rem;  // rem: elements from tid on
    int Gv;
    __device__ __forceinline__ RowSlice(int tid_, int G_, int D_) : tid(tid_), D(D_), rem(D_ - tid_), Gv(G_) {}
    __device__ __forceinline__ int G() const { return VEC ? Gv : GT; }
    __device__ __forceinline__ int chunk(int c) const { return (tid + c * G()) * 8; }
    __device__ __forceinline__ bool has(int i) const { return VEC ? chunk(i >> 3) < D : rem > i * GT; }

    template <class T>
    __device__ __forceinline__ void load(const T* p, float (&v)[8 * NCH]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                if (chunk(c) < D) {
                    if constexpr (sizeof(T) == 4) {
                        const float4* q = reinterpret_cast<const float4*>(p + chunk(c));
                        const float4 a = q[0], b = q[1];
                        v[8 * c] = a.x, v[8 * c + 1] = a.y, v[8 * c + 2] = a.z, v[8 * c + 3] = a.w;
                        v[8 * c + 4] = b.x, v[8 * c + 5] = b.y, v[8 * c + 6] = b.z, v[8 * c + 7] = b.w;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4*>(p + chunk(c));
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 f = Elem<T>::unpack(w[j]);
                            v[8 * c + 2 * j] = f.x;
                            v[8 * c + 2 * j + 1] = f.y;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[8 * c + j] = 0.0f;
                }
            }
        } else {
            p += tid;
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i) v[i] = has(i) ? to_f(p[i * GT]) : 0.0f;
        }
    }
    // Values 8 c .. 8 c + 8 of a float vector as long as the row (any of its values behind its end), or
    // `none` where there is no vector.
    __device__ __forceinline__ void vector8(const float* p, int c, float none, float (&o)[8]) const {
        if (p == nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = none;
        } else if constexpr (VEC) {
            const float4* q = reinterpret_cast<const float4*>(p + min(chunk(c), D - 8));
            const float4 a = q[0], b = q[1];
            o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w;
            o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
        } else {
            p += tid;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = has(8 * c + j) ? __ldg(p + (8 * c + j) * GT) : 0.0f;
        }
    }
    // v summed over the thread's part of the row: values behind the row's end may be anything
    __device__ __forceinline__ float part_sum(const float (&v)[8 * NCH]) const {
        float t = 0.0f;
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                uint64_t u = pair(v[8 * c], v[8 * c + 1]);
#pragma unroll
                for (int j = 2; j < 8; j += 2) u = add2(u, pair(v[8 * c + j], v[8 * c + j + 1]));
                const float2 f = unpair(u);
                t += chunk(c) < D ? f.x + f.y : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i) t += has(i) ? v[i] : 0.0f;
        }
        return t;
    }
    __device__ __forceinline__ float part_square_sum(const float (&v)[8 * NCH]) const {
        float t = 0.0f;
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                uint64_t u = pair(v[8 * c], v[8 * c + 1]);
                u = mul2(u, u);
#pragma unroll
                for (int j = 2; j < 8; j += 2) {
                    const uint64_t w = pair(v[8 * c + j], v[8 * c + j + 1]);
                    u = fma2(w, w, u);
                }
                const float2 f = unpair(u);
                t += chunk(c) < D ? f.x + f.y : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i) t += has(i) ? v[i] * v[i] : 0.0f;
        }
        return t;
    }
    __device__ __forceinline__ float part_max(const float (&v)[8 * NCH]) const {
        float t = 0.0f;
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                float u = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) u = max_abs(u, v[8 * c + j]);
                t = max_abs(t, chunk(c) < D ? u : 0.0f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i) t = max_abs(t, has(i) ? v[i] : 0.0f);
        }
        return t;
    }
    __device__ __forceinline__ void load_dt(int dt, const void* base, long long off, float (&v)[8 * NCH]) const {
        if (dt == OP_F32)
            load(static_cast<const float*>(base) + off, v);
        else if (dt == OP_F16)
            load(static_cast<const __half*>(base) + off, v);
        else
            load(static_cast<const __nv_bfloat16*>(base) + off, v);
    }
    template <class T>
    __device__ __forceinline__ void store(T* p, const float (&v)[8 * NCH]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                if (chunk(c) >= D) continue;
                if constexpr (sizeof(T) == 4) {
                    float4* q = reinterpret_cast<float4*>(p + chunk(c));
                    q[0] = make_float4(v[8 * c], v[8 * c + 1], v[8 * c + 2], v[8 * c + 3]);
                    q[1] = make_float4(v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]);
                } else {
                    uint4 u;
                    u.x = Elem<T>::pack(v[8 * c], v[8 * c + 1]);
                    u.y = Elem<T>::pack(v[8 * c + 2], v[8 * c + 3]);
                    u.z = Elem<T>::pack(v[8 * c + 4], v[8 * c + 5]);
                    u.w = Elem<T>::pack(v[8 * c + 6], v[8 * c + 7]);
                    *reinterpret_cast<uint4*>(p + chunk(c)) = u;
                }
            }
        } else {
            p += tid;
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i)
                if (has(i)) {
                    if constexpr (sizeof(T) == 4)
                        p[i * GT] = v[i];
                    else
                        p[i * GT] = Elem<T>::from(v[i]);
                }
        }
    }
    __device__ __forceinline__ void store_dt(int dt, void* base, long long off, const float (&v)[8 * NCH]) const {
        if (dt == OP_F32)
            store(static_cast<float*>(base) + off, v);
        else if (dt == OP_F16)
            store(static_cast<__half*>(base) + off, v);
        else
            store(static_cast<__nv_bfloat16*>(base) + off, v);
    }
};

// Sum / maximum over the LANES threads of a row in a warp (shuffles), or, with LANES = 0, over a
// block: a warp's shuffles, then one word of each warp.  `buf` alternates between two halves so
// that one barrier a reduction is enough.
template <int LANES>
struct RowReduce {
    float* buf;  // [2][32]
    int flip;
    unsigned mask;  // the row's lanes: rows of a warp may end in different rounds
    __device__ __forceinline__ explicit RowReduce(float* b) : buf(b), flip(0), mask(0xffffffffu) {
        if constexpr (LANES > 0 && LANES < 32) mask = ((1u << LANES) - 1u) << (threadIdx.x % 32 / LANES * LANES);
    }
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int o = LANES ? LANES / 2 : 16; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
        if constexpr (LANES == 0) {
            float* at = buf + 32 * flip;
            flip ^= 1;
            if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
            __syncthreads();
            const int warps = blockDim.x >> 5;
            v = static_cast<int>(threadIdx.x & 31) < warps ? at[threadIdx.x & 31] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        }
        return v;
    }
    __device__ __forceinline__ uint32_t max(uint32_t v) {
        if constexpr (LANES > 0 && LANES < 32) {
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) v = ::max(v, __shfl_xor_sync(mask, v, o));
            return v;
        }
        v = __reduce_max_sync(0xffffffffu, v);
        if constexpr (LANES == 0) {
            uint32_t* at = reinterpret_cast<uint32_t*>(buf + 32 * flip);
            flip ^= 1;
            if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
            __syncthreads();
            const int warps = blockDim.x >> 5;
            v = __reduce_max_sync(0xffffffffu, static_cast<int>(threadIdx.x & 31) < warps ? at[threadIdx.x & 31] : 0u);
        }
        return v;
    }
};

template <int N>
__device__ __forceinline__ void set(float (&v)[N], int i, uint64_t two) {
    const float2 f = unpair(two);
    v[i] = f.x, v[i + 1] = f.y;
}

template <bool VEC, int NCH, int LANES, int GT>
__device__ __forceinline__ void normalise(const RowSlice<VEC, NCH, GT>& s, RowReduce<LANES>& red, float (&v)[8 * NCH],
                                          int kind, float eps, const float* w, const float* b) {
    constexpr int N = 8 * NCH;
    const float inv_d = 1.0f / static_cast<float>(s.D);
    if (kind == NORM_LAYER) {
        const float mean = red.sum(s.part_sum(v)) * inv_d;
#pragma unroll
        for (int i = 0; i < N; i += 2) set(v, i, add2(pair(v[i], v[i + 1]), pair(-mean, -mean)));
    }
    const float rstd = rsqrtf(red.sum(s.part_square_sum(v)) * inv_d + eps);
    // the weight and bias vectors are read chunk by chunk: every row reads them from L1
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        float g[8], a[8];
        s.vector8(w, c, 1.0f, g);
        s.vector8(b, c, 0.0f, a);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const int i = 8 * c + j;
            set(v, i, fma2(mul2(pair(v[i], v[i + 1]), pair(rstd, rstd)), pair(g[j], g[j + 1]), pair(a[j], a[j + 1])));
        }
    }
}

template <bool EXACT16, bool VEC, int NCH, int LANES, int GT>
__device__ __forceinline__ void store_int8(const RowSlice<VEC, NCH, GT>& s, RowReduce<LANES>& red, const float (&v)[8 * NCH],
                                           int8_t* q, float* scale) {
    const uint32_t top = red.max(__float_as_uint(s.part_max(v)) & 0x7FFFFFFFu);
    const bool live = live_magnitude(top);
    const Quantizer z(__uint_as_float(top));
    if (s.tid == 0) *scale = z.a / 127.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        if (VEC && s.chunk(c) >= s.D) continue;
        const uint2 u = live ? quantize8<EXACT16>(v + 8 * c, z) : make_uint2(0, 0);
        if constexpr (VEC) {
            *reinterpret_cast<uint2*>(q + s.chunk(c)) = u;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (s.has(8 * c + j)) q[s.tid + (8 * c + j) * GT] = static_cast<int8_t>((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
        }
    }
}

// What a kernel does: the whole operator, or only x quantised to 8 bits, in fewer registers (more
// rows in flight: an SM needs about 40 KB of loads under way).
enum RowMode : int { ROW_FULL = 0, ROW_QUANTIZE_F32 = 1, ROW_QUANTIZE_16 = 2 };

// One row: load_x and load_y bring the thread's values, `loaded` is called once every thread of the
// row has its values (after a reduction's barrier).
template <int MODE, bool VEC, int NCH, int LANES, int GT, class LoadX, class LoadY, class Loaded>
__device__ __forceinline__ void row_body(const RowNormParams& p, const RowSlice<VEC, NCH, GT>& s, RowReduce<LANES>& red,
                                         long long row, LoadX&& load_x, LoadY&& load_y, Loaded&& loaded) {
    constexpr int N = 8 * NCH;
    float v[N];
    load_x(v);
    if constexpr (MODE != ROW_FULL) {
        store_int8<MODE == ROW_QUANTIZE_16>(s, red, v, static_cast<int8_t*>(p.out) + row * p.ldo, p.out_scale + row);
        loaded();
    } else {
        if (p.y != nullptr) {
            float t[N];
            load_y(t);
            if (p.post != NORM_NONE) normalise(s, red, t, p.post, p.eps, p.pw, p.pb);
            if (p.gate != nullptr) {
                const float* g = p.gate;
                if (p.ld_gate != 0)
                    g += static_cast<long long>(static_cast<uint32_t>(row) / static_cast<uint32_t>(p.rows_per_gate)) * p.ld_gate;
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    float gv[8];
                    s.vector8(g, c, 1.0f, gv);
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const int i = 8 * c + j;
                        set(v, i, fma2(pair(gv[j], gv[j + 1]), pair(t[i], t[i + 1]),
                                       mul2(pair(v[i], v[i + 1]), pair(p.alpha, p.alpha))));
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i += 2)
                    set(v, i, fma2(pair(v[i], v[i + 1]), pair(p.alpha, p.alpha), pair(t[i], t[i + 1])));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= p.alpha;
        }
        if (p.r != nullptr) s.store_dt(p.x_dt, p.r, row * p.ldr, v);
        if (p.norm != NORM_NONE) normalise(s, red, v, p.norm, p.eps, p.w, p.b);
        if (p.out_dt == OP_I8) {
            store_int8<false>(s, red, v, static_cast<int8_t*>(p.out) + row * p.ldo, p.out_scale + row);
            loaded();
        } else {
            loaded();
            s.store_dt(p.out_dt, p.out, row * p.ldo, v);
        }
    }
}

// At least this many blocks an SM: a warp's row in 64 to 96 registers; a block's 16-bit row to quantise in 32,
// so that all of an SM's threads load (24,576 rows of 4,096: 59 us, 72 with 43 registers).
constexpr int row_blocks(bool vec, int nch, int lanes, int mode) {
    return lanes && nch >= 3 && mode == ROW_FULL ? 9 - nch : vec && lanes == 0 && mode == ROW_QUANTIZE_16 ? 2 : 0;
}

// LANES threads of a warp to a row (a few rows to a warp when it is short), or 0: a block.
template <bool VEC, int NCH, int LANES, int MODE, int GT>
__global__ void __launch_bounds__(LANES ? 128 : VEC ? 1024 : GT, row_blocks(VEC, NCH, LANES, MODE))
    row_norm_kernel(const __grid_constant__ RowNormParams p) {
    if constexpr (VEC || MODE != ROW_FULL) grid_dependency_wait();
    if constexpr (MODE != ROW_FULL) grid_dependency_start();  // the product that follows may set itself up
    __shared__ float red_buf[64];
    RowReduce<LANES> red(red_buf);
    const int tid = LANES ? static_cast<int>(threadIdx.x % (LANES ? LANES : 1)) : static_cast<int>(threadIdx.x);
    const RowSlice<VEC, NCH, GT> s(tid, LANES ? LANES : VEC ? static_cast<int>(blockDim.x) : GT, p.cols);
    const int per = LANES ? static_cast<int>(blockDim.x) / (LANES ? LANES : 1) : 1;
    const long long first = static_cast<long long>(blockIdx.x) * per + (LANES ? threadIdx.x / (LANES ? LANES : 1) : 0);
    for (long long row = first; row < p.rows; row += static_cast<long long>(gridDim.x) * per)
        row_body<MODE>(
            p, s, red, row, [&](auto& v) { s.load_dt(p.x_dt, p.x, row * p.ldx, v); },
            [&](auto& t) { s.load_dt(p.y_dt, p.y, row * p.ldy, t); }, [] {});
}

// Many long rows: a block keeps its next rows of x and y on their way into shared memory with bulk
// copies, so that the loads do not wait for the reductions of the row before and take no registers
// (24,576 rows of 4,096, bf16: 133 us against 191; quantising alone gains nothing, 71 against 59).
constexpr int kStreamStages = 4;

__global__ void __launch_bounds__(1024) row_stream_kernel(const __grid_constant__ RowNormParams p, int stages) {
    extern __shared__ __align__(128) uint8_t ring[];  // [stages][x row, y row]
    __shared__ float red_buf[64];
    __shared__ uint64_t full[kStreamStages];
    __shared__ volatile int abort_flag;
    RowReduce<0> red(red_buf);
    const RowSlice<true, 2, 0> s(static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), p.cols);
    const uint32_t xb = p.cols * op_bytes(p.x_dt), yb = p.y != nullptr ? p.cols * op_bytes(p.y_dt) : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
        abort_flag = 0;
        fence_barrier_init();
    }
    __syncthreads();
    auto fetch = [&](long long row, int stage) {  // thread 0
        uint8_t* at = ring + stage * (xb + yb);
        mbar_arrive_expect_tx(&full[stage], xb + yb);
        bulk_load(at, static_cast<const uint8_t*>(p.x) + row * p.ldx * op_bytes(p.x_dt), xb, &full[stage]);
        if (yb) bulk_load(at + xb, static_cast<const uint8_t*>(p.y) + row * p.ldy * op_bytes(p.y_dt), yb, &full[stage]);
    };
    long long ahead = blockIdx.x;  // the next row to fetch
    if (threadIdx.x == 0)
        for (int i = 0; i < stages && ahead < p.rows; ++i, ahead += gridDim.x) fetch(ahead, i);
    uint32_t it = 0;
    bool ok = true;
    for (long long row = blockIdx.x; row < p.rows && ok; row += gridDim.x, ++it) {
        const int stage = it % stages;
        ok = mbar_wait(&full[stage], (it / stages) & 1, &abort_flag, kDevTimeoutProducer, &g_status.code);
        if (!ok) break;
        const uint8_t* at = ring + stage * (xb + yb);
        row_body<ROW_FULL>(
            p, s, red, row, [&](auto& v) { s.load_dt(p.x_dt, at, 0, v); }, [&](auto& t) { s.load_dt(p.y_dt, at + xb, 0, t); },
            [&] {
                if (threadIdx.x == 0 && ahead < p.rows) {
                    fetch(ahead, stage);
                    ahead += gridDim.x;
                }
            });
    }
    if (!ok && threadIdx.x == 0) {  // wait (bounded) for copies that may still be in flight
        volatile int dummy = 0;
        for (int i = 1; i < stages; ++i)
            mbar_wait(&full[(it + i) % stages], ((it + i) / stages) & 1, &dummy, kDevTimeoutProducer, &g_status.code);
    }
}

bool is_quantize(const RowNormParams& p) {
    return p.y == nullptr && p.r == nullptr && p.norm == NORM_NONE && p.out_dt == OP_I8 && p.alpha == 1.0f;
}

template <bool VEC, int NCH, int LANES, int GT = LANES>
void launch(cudaStream_t s, const RowNormParams& p, int threads) {
    const long long per = LANES ? threads / (LANES ? LANES : 1) : 1;
    long long grid = (p.rows + per - 1) / per;
    if (grid > 148 * 64) grid = 148 * 64;
    const LaunchConfig c(static_cast<unsigned>(grid), threads, 0, s);
    if (!is_quantize(p)) {
        if constexpr (VEC) {
            M3R_CUDA(cudaLaunchKernelEx(&c.cfg, row_norm_kernel<VEC, NCH, LANES, ROW_FULL, GT>, p));
        } else {
            // an ordinary launch: it reads the weight vectors as constants (__ldg), which may come from the
            // kernel before (40,001 rows of 129: 21 us against 27 with plain loads)
            const LaunchConfig plain(static_cast<unsigned>(grid), threads, 0, s, 0, false);
            M3R_CUDA(cudaLaunchKernelEx(&plain.cfg, row_norm_kernel<VEC, NCH, LANES, ROW_FULL, GT>, p));
        }
        return;
    }
    auto kern = p.x_dt == OP_F32 ? row_norm_kernel<VEC, NCH, LANES, ROW_QUANTIZE_F32, GT>
                                 : row_norm_kernel<VEC, NCH, LANES, ROW_QUANTIZE_16, GT>;
    M3R_CUDA(cudaLaunchKernelEx(&c.cfg, kern, p));
}

// All of an SM's registers (64 a thread) in as many blocks as that makes, and shared memory but for
// some that is left to L1, where the weight and gate vectors of every row come from (us with 225, 180 and
// 140 KB of rings, 16-bit branch and result, one norm: 24,576 rows of 4,096, bf16 138, 133, 133, with two
// norms and a gate 200, 186, 186; 50,000 of 2,048 137, 133, 146; 9,216 of 1,024 19.3, 17.5, 17.1.  Long 32-bit
// rows would rather have two rows of ring than L1: 24,576 of 4,096 197, 207, 207; 12,288 of 8,192 191, 234, 234).
// False where a block's share does not hold a row.
bool launch_stream(cudaStream_t s, const RowNormParams& p, int threads) {
    constexpr int kMost = 180 * 1024;
    const int per_sm = 1024 / threads;
    const int row = p.cols * (op_size(p.x_dt) + (p.y != nullptr ? op_size(p.y_dt) : 0));
    const int room = kMost / per_sm - 2048;
    const int stages = room / row < kStreamStages ? room / row : kStreamStages;
    if (stages < 1) return false;
    static unsigned done = 0;
    allow_smem(row_stream_kernel, kMost, done);
    const LaunchConfig c(static_cast<unsigned>(148 * per_sm), threads, stages * row, s, 0, false);
    M3R_CUDA(cudaLaunchKernelEx(&c.cfg, row_stream_kernel, p, stages));
    return true;
}

bool aligned(const void* p, long long ld, int dt, int bytes) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld * op_size(dt)) % bytes == 0);
}

// Rows to threads.  Short rows share a warp, 8 values a lane.  With many rows, a warp each up to
// 1,024 values (98,304 rows of 1,024, 32-bit stream: 188 us, against 209 with a block each; of 768: 141
// against 158); with few, a block each, so that a row's chain of loads and reductions is short: 8 values a
// thread while an SM holds all its rows at once (592 rows of 1,024, bf16 stream and two norms: 3.2 us, 3.8
// with 16 values), 16 above, where twice the rows are under way (2,304 rows: 7.1 and 6.1; 6,144: 18.2 and
// 17.5, 18.0 with a warp each; 32-bit stream, one norm: 6.9 and 6.6, 17.4, 17.8 and 19.3).  Of 768: 2,304
// rows 6.1 with a block each, 4.8 with a warp, 4,608 9.9 and 9.2; 32-bit 5.8 and 5.1, 10.5 and 11.9.
// More rows than that again are copied ahead (9,216 of 1,024, bf16: 23.7 and 22.7).
// Of 264 to 512, one norm: 1,200 rows of 512 2.9 with a block each and 3.1 with a warp, 2,400 3.8 and 3.6,
// 50,000 51.8 and 50.0; 32-bit 2,400 4.0 and 4.3, 50,000 53.0 and 51.7, of 320 44.2 and 40.5; quantised only, 600
// rows 1.9 and 1.8, 2,300 3.1 and 2.2 (the one rule for both costs these 0.9 us), 9,216 10.2 and 4.1.
// Quantised only: 300 rows of 1,024 1.7 us with a block each against 1.8, 1,000 2.6 against 1.9, 32-bit
// 2.65 against 2.7; 2,300 of 768 3.3 against 2.9.
void dispatch_vec(cudaStream_t s, const RowNormParams& p) {
    if (p.cols <= 32) return launch<true, 1, 4>(s, p, 128);
    if (p.cols <= 64) return launch<true, 1, 8>(s, p, 128);
    if (p.cols <= 128) return launch<true, 1, 16>(s, p, 128);
    if (p.cols <= 256) return launch<true, 1, 32>(s, p, 128);
    const bool quantize = is_quantize(p);
    const int few = p.x_dt == OP_F32 ? (quantize ? 12 : 32) : quantize ? 4 : 12;  // rows an SM
    if (p.cols <= 512 && p.rows > 148 * 16) return launch<true, 2, 32>(s, p, 128);
    if (p.cols <= 768 && p.rows > 148 * few) return launch<true, 3, 32>(s, p, 128);
    if (p.cols <= 1024 && p.rows > 148 * (quantize ? few : 96)) return launch<true, 4, 32>(s, p, 128);
    auto threads = [&](int nch) { return ((p.cols + 8 * nch - 1) / (8 * nch) + 31) / 32 * 32; };
    if (p.cols <= 1024 ? p.rows <= 148 * 8 || p.cols <= 768 || quantize : p.cols <= 8192 && p.rows <= 148 * 2)
        return launch<true, 1, 0>(s, p, threads(1));
    const int blocks = 148 * (1024 / threads(2));  // at 64 registers
    if (p.rows >= 2LL * blocks && !quantize && launch_stream(s, p, threads(2))) return;
    launch<true, 2, 0>(s, p, threads(2));
}

// Element accesses (odd widths, rows off the 16-byte grid): 8 or 16 values a thread, neighbouring
// threads at neighbouring elements.  Threads without a value cost as much as the others, so the blocks
// come in steps of a quarter to a half (24,576 rows of 513: 56 us in 128 threads, 44 in 96;
// 5,000 of 5,003: 115 us with 8 values in 704 threads, which an SM holds once, 79 with 16 in 320; 9,000 of
// 2,005, bf16 stream: 67 and 52; 4,039 of 1,001 with 16 values: 18.4 against 16.5).  They stay far from their
// bytes' time (in us, that time behind the stroke): an access of 2 bytes a thread, and no rows copied ahead.
// Norms, 16-bit branch and result: 24,576 of 513, bf16 42 / 15, 9,000 of 2,005 49 / 22, 40,001 of 129, 32-bit
// 19 / 9.5, 9,000 of 3,333 80 / 55; quantised only, bf16: 24,576 of 513 16 / 5.8, 98,304 of 1,001 86 / 45.
template <int NCH, int GT>
void launch_elements(cudaStream_t s, const RowNormParams& p) {
    launch<false, NCH, 0, GT>(s, p, GT);
}

void dispatch_elements(cudaStream_t s, const RowNormParams& p) {
    if (p.cols <= 32) return launch<false, 1, 4>(s, p, 128);
    if (p.cols <= 64) return launch<false, 1, 8>(s, p, 128);
    if (p.cols <= 128) return launch<false, 1, 16>(s, p, 128);
    if (p.cols <= 256) return launch<false, 1, 32>(s, p, 128);
    if (p.cols <= 8 * 64) return launch_elements<1, 64>(s, p);
    if (p.cols <= 8 * 96) return launch_elements<1, 96>(s, p);
    if (p.cols <= 8 * 128) return launch_elements<1, 128>(s, p);
    if (p.cols <= 8 * 160) return launch_elements<1, 160>(s, p);
    if (p.cols <= 16 * 96) return launch_elements<2, 96>(s, p);
    if (p.cols <= 16 * 128) return launch_elements<2, 128>(s, p);
    if (p.cols <= 16 * 160) return launch_elements<2, 160>(s, p);
    if (p.cols <= 16 * 256) return launch_elements<2, 256>(s, p);
    if (p.cols <= 16 * 320) return launch_elements<2, 320>(s, p);
    if (p.cols <= 16 * 512) return launch_elements<2, 512>(s, p);
    launch_elements<2, 1024>(s, p);
}

}  // namespace

int* row_norm_status() {
    void* at = nullptr;
    M3R_CUDA(cudaGetSymbolAddress(&at, g_status));
    return &static_cast<DevStatus*>(at)->code;
}

void row_norm(cudaStream_t s, const RowNormParams& p) {
    if (p.rows == 0) return;
    // 16-byte accesses (8 of 8-bit results) need whole chunks of 8 values and aligned rows
    const bool vec = p.cols % 8 == 0 && aligned(p.x, p.ldx, p.x_dt, 16) && aligned(p.y, p.ldy, p.y_dt, 16) &&
                     aligned(p.r, p.ldr, p.x_dt, 16) && aligned(p.out, p.ldo, p.out_dt, p.out_dt == OP_I8 ? 8 : 16) &&
                     aligned(p.gate, p.ld_gate, OP_F32, 16) && aligned(p.pw, 0, OP_F32, 16) &&
                     aligned(p.pb, 0, OP_F32, 16) && aligned(p.w, 0, OP_F32, 16) && aligned(p.b, 0, OP_F32, 16);
    if (vec)
        dispatch_vec(s, p);
    else
        dispatch_elements(s, p);
}

}  // namespace m3r
