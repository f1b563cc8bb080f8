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
// belongs to one warp (statistics by shuffles, no block barrier), a longer one to one
// block; x and y are loaded before the first reduction so that a warp keeps its whole
// row's bytes in flight.  All statistics are 32-bit, the variance in two passes over the
// registers.
#include "common.cuh"
#include "ops.h"
#include "tmap.h"

namespace m3r {

namespace {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

// The N = 8 * NCH values of a thread.  VEC: chunk c holds elements (tid + c * G) * 8 .. + 8
// of the row (one 16-byte access of a 16-bit type); else value i is element tid + i * G.
template <bool VEC, int NCH>
struct RowSlice {
    int tid, G, D;
    __device__ __forceinline__ int chunk(int c) const { return (tid + c * G) * 8; }
    __device__ __forceinline__ int elem(int i) const { return VEC ? chunk(i >> 3) + (i & 7) : tid + i * G; }
    __device__ __forceinline__ bool has(int i) const { return (VEC ? chunk(i >> 3) : elem(i)) < D; }

    template <class T>
    __device__ __forceinline__ void load(const T* p, float (&v)[8 * NCH], float fill) const {
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
                    for (int j = 0; j < 8; ++j) v[8 * c + j] = fill;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i) v[i] = elem(i) < D ? to_f(p[elem(i)]) : fill;
        }
    }
    __device__ __forceinline__ void load_dt(int dt, const void* base, long long off, float (&v)[8 * NCH]) const {
        if (dt == OP_F32)
            load(static_cast<const float*>(base) + off, v, 0.0f);
        else if (dt == OP_F16)
            load(static_cast<const __half*>(base) + off, v, 0.0f);
        else
            load(static_cast<const __nv_bfloat16*>(base) + off, v, 0.0f);
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
#pragma unroll
            for (int i = 0; i < 8 * NCH; ++i)
                if (elem(i) < D) {
                    if constexpr (sizeof(T) == 4)
                        p[elem(i)] = v[i];
                    else
                        p[elem(i)] = Elem<T>::from(v[i]);
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

// Sum / maximum over the threads of a row: a warp's shuffles, then one word of each warp.
// `buf` alternates between two halves so that one barrier a reduction is enough.
template <bool WARP>
struct RowReduce {
    float* buf;  // [2][32]
    int flip;
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if constexpr (!WARP) {
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
        v = __reduce_max_sync(0xffffffffu, v);
        if constexpr (!WARP) {
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

template <bool VEC, int NCH, bool WARP>
__device__ __forceinline__ void normalise(const RowSlice<VEC, NCH>& s, RowReduce<WARP>& red, float (&v)[8 * NCH],
                                          int kind, float eps, const float* w, const float* b) {
    constexpr int N = 8 * NCH;
    const float inv_d = 1.0f / static_cast<float>(s.D);
    float mean = 0.0f;
    if (kind == NORM_LAYER) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) t += v[i];
        mean = red.sum(t) * inv_d;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = s.has(i) ? v[i] - mean : 0.0f;
        q += v[i] * v[i];
    }
    const float rstd = rsqrtf(red.sum(q) * inv_d + eps);
    // the weight and bias vectors are read chunk by chunk: every row reads them from L1
    if constexpr (VEC) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (s.chunk(c) >= s.D) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float* u = v + 8 * c + 4 * h;
                const float4 g = w ? __ldg(reinterpret_cast<const float4*>(w + s.chunk(c)) + h) : make_float4(1, 1, 1, 1);
                const float4 a = b ? __ldg(reinterpret_cast<const float4*>(b + s.chunk(c)) + h) : make_float4(0, 0, 0, 0);
                u[0] = u[0] * rstd * g.x + a.x;
                u[1] = u[1] * rstd * g.y + a.y;
                u[2] = u[2] * rstd * g.z + a.z;
                u[3] = u[3] * rstd * g.w + a.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (s.has(i)) v[i] = v[i] * rstd * (w ? __ldg(w + s.elem(i)) : 1.0f) + (b ? __ldg(b + s.elem(i)) : 0.0f);
    }
}

// The integer nearest to 127 v / a, ties to even, decided by the two exact products 254 v and
// (2 m + 1) a on either side of a half.
__device__ __noinline__ int quantize_exact(float v, float p, float a) {
    const float lo = floorf(p);
    const double d = 254.0 * static_cast<double>(v) - (2.0 * static_cast<double>(lo) + 1.0) * static_cast<double>(a);
    const int l = static_cast<int>(lo);
    return d > 0.0 ? l + 1 : d < 0.0 ? l : (l & 1) ? l + 1 : l;
}

// Eight values in 8 bits.  p = v * inv lies within 2e-5 of 127 v / a (two roundings of a value up
// to 127), so that its nearest integer is the right one unless p is that near to a half: one test
// for the eight, taken for about one value in 10^5, sends them to quantize_exact.  Adding 1.5 * 2^23
// rounds p to the integer that then stands in the sum's low byte.
__device__ __forceinline__ uint2 quantize8(const float* v, float pre, float inv, float a) {
    constexpr float kMagic = 12582912.0f;
    float t[8], off = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float p = v[j] * inv;
        t[j] = p + kMagic;
        off = fmaxf(off, fabsf(p - (t[j] - kMagic)));
    }
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(t[j]);
    if (off > 0.49997f || pre != 1.0f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = v[j] * pre * inv;
            b[j] = fabsf(p - rintf(p)) > 0.49997f ? quantize_exact(v[j], p, a) : static_cast<int>(rintf(p));
        }
    }
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// The larger magnitude; NaN when either is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <bool VEC, int NCH, bool WARP>
__device__ __forceinline__ void store_int8(const RowSlice<VEC, NCH>& s, RowReduce<WARP>& red, const float (&v)[8 * NCH],
                                           int8_t* q, float* scale) {
    constexpr int N = 8 * NCH;
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (s.has(i)) m = max_abs(m, v[i]);
    // magnitudes compare as integers, and NaN above infinity above every number
    const uint32_t top = red.max(__float_as_uint(m) & 0x7FFFFFFFu);
    const float a = __uint_as_float(top);
    // rows without a finite, non-zero magnitude hold zeros: a zero scale gives zeros, an
    // infinite or NaN one gives NaN in every product
    const bool live = top != 0 && top < 0x7F800000u;
    // 127 / a overflows for magnitudes near the smallest: those rows are scaled up first
    const float pre = a < 1e-20f ? 0x1p100f : 1.0f;
    const float inv = 127.0f / (a * pre);
    if (s.tid == 0) *scale = a / 127.0f;
    if constexpr (VEC) {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if (s.chunk(c) < s.D)
                *reinterpret_cast<uint2*>(q + s.chunk(c)) = live ? quantize8(v + 8 * c, pre, inv, a) : make_uint2(0, 0);
    } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint2 u = live ? quantize8(v + 8 * c, pre, inv, a) : make_uint2(0, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (s.has(8 * c + j)) q[s.elem(8 * c + j)] = static_cast<int8_t>((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
        }
    }
}

// FULL: the whole operator; else only x quantised to 8 bits, in fewer registers (more rows in
// flight: an SM needs about 40 KB of loads under way).
template <bool VEC, int NCH, bool WARP, bool FULL>
__global__ void __launch_bounds__(WARP ? 128 : 1024) row_norm_kernel(const __grid_constant__ RowNormParams p) {
    constexpr int N = 8 * NCH;
    __shared__ float red_buf[64];
    RowReduce<WARP> red{red_buf, 0};
    RowSlice<VEC, NCH> s;
    s.D = p.cols;
    s.G = WARP ? 32 : static_cast<int>(blockDim.x);
    s.tid = WARP ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
    const long long per = WARP ? blockDim.x >> 5 : 1;
    for (long long row = blockIdx.x * per + (WARP ? threadIdx.x >> 5 : 0); row < p.rows; row += gridDim.x * per) {
        float v[N];
        s.load_dt(p.x_dt, p.x, row * p.ldx, v);
        if constexpr (!FULL) {
            store_int8<VEC, NCH, WARP>(s, red, v, static_cast<int8_t*>(p.out) + row * p.ldo, p.out_scale + row);
            continue;
        }
        if (p.y != nullptr) {
            float t[N];
            s.load_dt(p.y_dt, p.y, row * p.ldy, t);
            if (p.post != NORM_NONE) normalise<VEC, NCH, WARP>(s, red, t, p.post, p.eps, p.pw, p.pb);
            if (p.gate != nullptr) {
                const float* g = p.gate + (row / p.rows_per_gate) * p.ld_gate;
                float gv[N];
                s.load(g, gv, 0.0f);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = p.alpha * v[i] + gv[i] * t[i];
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = p.alpha * v[i] + t[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= p.alpha;
        }
        if (p.r != nullptr) s.store_dt(p.x_dt, p.r, row * p.ldr, v);
        if (p.norm != NORM_NONE) normalise<VEC, NCH, WARP>(s, red, v, p.norm, p.eps, p.w, p.b);
        if (p.out_dt == OP_I8)
            store_int8<VEC, NCH, WARP>(s, red, v, static_cast<int8_t*>(p.out) + row * p.ldo, p.out_scale + row);
        else
            s.store_dt(p.out_dt, p.out, row * p.ldo, v);
    }
}

template <bool VEC, int NCH, bool WARP>
void launch(cudaStream_t s, const RowNormParams& p, int threads) {
    const long long per = WARP ? threads / 32 : 1;
    long long grid = (p.rows + per - 1) / per;
    if (grid > 148 * 64) grid = 148 * 64;
    const bool full = p.y != nullptr || p.r != nullptr || p.norm != NORM_NONE || p.out_dt != OP_I8 || p.alpha != 1.0f;
    if (full)
        row_norm_kernel<VEC, NCH, WARP, true><<<static_cast<int>(grid), threads, 0, s>>>(p);
    else
        row_norm_kernel<VEC, NCH, WARP, false><<<static_cast<int>(grid), threads, 0, s>>>(p);
    M3R_CUDA(cudaGetLastError());
}

bool aligned(const void* p, long long ld, int dt, int bytes) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld * op_size(dt)) % bytes == 0);
}

template <bool VEC>
void dispatch(cudaStream_t s, const RowNormParams& p) {
    if (p.cols <= 256) return launch<VEC, 1, true>(s, p, 128);
    if (p.cols <= 512) return launch<VEC, 2, true>(s, p, 128);
    if (p.cols <= 1024) return launch<VEC, 4, true>(s, p, 128);
    auto threads = [&](int nch) { return ((p.cols + 8 * nch - 1) / (8 * nch) + 31) / 32 * 32; };
    if (p.cols <= 8192 && p.rows < 2 * 148) return launch<VEC, 1, false>(s, p, threads(1));
    launch<VEC, 2, false>(s, p, threads(2));
}

}  // namespace

void row_norm(cudaStream_t s, const RowNormParams& p) {
    if (p.rows == 0) return;
    // 16-byte accesses (8 of 8-bit results) need whole chunks of 8 values and aligned rows
    const bool vec = p.cols % 8 == 0 && aligned(p.x, p.ldx, p.x_dt, 16) && aligned(p.y, p.ldy, p.y_dt, 16) &&
                     aligned(p.r, p.ldr, p.x_dt, 16) && aligned(p.out, p.ldo, p.out_dt, p.out_dt == OP_I8 ? 8 : 16) &&
                     aligned(p.gate, p.ld_gate, OP_F32, 16) && aligned(p.pw, 0, OP_F32, 16) &&
                     aligned(p.pb, 0, OP_F32, 16) && aligned(p.w, 0, OP_F32, 16) && aligned(p.b, 0, OP_F32, 16);
    if (vec)
        dispatch<true>(s, p);
    else
        dispatch<false>(s, p);
}

}  // namespace m3r
