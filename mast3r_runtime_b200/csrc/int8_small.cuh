// The 8-bit product for few rows of x, where the weights' bytes are the work.
//
// int8_gemv_kernel (up to 4 rows): one launch for everything.  Every block quantises the rows
// itself, into shared memory, while its first weights travel; a warp takes 4 output channels at a
// time, its lanes 16 bytes of k each, and adds up four products an instruction.
//
// int8_skinny_kernel (few rows, or few tiles and a long k): the roles of the operands are exchanged --
// 128 output channels are the rows of the tensor-core tile, up to NT tokens its columns -- so that with
// few tokens a stage of the pipeline is mostly weights.  A cluster of up to 8 CTAs splits k; each leaves its sums in
// shared memory, and every CTA adds and finishes some of the tokens from all of them (integer
// sums: the order does not matter).
#pragma once

#include "column_walk.h"
#include "common.cuh"
#include "gemm.cuh"
#include "ops.h"
#include "quantize.cuh"

namespace m3r {

namespace {

// y = act(acc * xs * ws + bias), one value
__device__ __forceinline__ float finish1(int acc, float xs, float ws, float bias, int act) {
    const float v = fmaf(static_cast<float>(acc) * xs, ws, bias);
    if (act == ACT_GELU) {
        // x / 2 (1 + tanh u) as x / (1 + exp(-2 u)), which loses no digits where the tanh nears -1
        const float u = v * fmaf(v * v, 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
        return v * rcp_approx(1.0f + ex2_approx(-2.885390081777927f * u));
    }
    if (act == ACT_RELU) return v < 0.0f ? 0.0f : v;  // keeps NaN
    return v;
}

__device__ __forceinline__ void store1(void* out, int dt, long long at, float v) {
    if (dt == OP_F32)
        static_cast<float*>(out)[at] = v;
    else if (dt == OP_F16)
        static_cast<__half*>(out)[at] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
}

struct GemvParams {
    int M, N, K, kpad;  // kpad: K rounded up to 16
    int x_dt, out_dt, act, x_vec;
    long long ldx, ldw, ldo;
    const void* x;
    const float* x_scale;
    const int8_t* w;
    const float* ws;
    const float* bias;
    void* out;
};

constexpr int kGemvThreads = 256;
constexpr int kGemvCols = 4;

// Eight values of a row from element e on (zero behind its end).
template <class T>
__device__ __forceinline__ void gemv_load8(const T* row, int e, int K, bool vec, float (&v)[8]) {
    if (vec && e + 8 <= K) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(row + e);
            const float4 b = reinterpret_cast<const float4*>(row + e)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(row + e);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = Elem<T>::unpack(w[j]);
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = e + j < K ? to_f(row[e + j]) : 0.0f;
    }
}

// Rows of x quantised into shared memory (zero behind their end), their scales into `scale`.
template <class T, int MR>
__device__ __forceinline__ void gemv_quantise(const GemvParams& p, uint8_t* sx, float* scale, uint32_t (*part)[MR]) {
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(p.x);
    uint32_t top[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        float big = 0.0f;
        if (m < p.M)
            for (int e = tid * 8; e < p.K; e += kGemvThreads * 8) {
                float v[8];
                gemv_load8(x + m * p.ldx, e, p.K, p.x_vec, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) big = max_abs(big, v[j]);
            }
        top[m] = __reduce_max_sync(0xffffffffu, __float_as_uint(big) & 0x7FFFFFFFu);
        if ((tid & 31) == 0) part[tid >> 5][m] = top[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        uint32_t t = 0;
#pragma unroll
        for (int w = 0; w < kGemvThreads / 32; ++w) t = max(t, part[w][m]);
        const bool live = live_magnitude(t);
        const Quantizer z(__uint_as_float(t));
        if (tid == m) scale[m] = z.a / 127.0f;
        for (int e = tid * 8; e < p.kpad; e += kGemvThreads * 8) {
            uint2 q = make_uint2(0, 0);
            if (m < p.M && live) {
                float v[8];
                gemv_load8(x + m * p.ldx, e, p.K, p.x_vec, v);
                q = quantize8<sizeof(T) == 2>(v, z);
            }
            *reinterpret_cast<uint2*>(sx + m * p.kpad + e) = q;
        }
    }
}

template <int MR>
__global__ void __launch_bounds__(kGemvThreads) int8_gemv_kernel(const __grid_constant__ GemvParams p) {
    extern __shared__ __align__(16) uint8_t sx[];  // [MR][kpad]
    __shared__ float scale[MR];
    __shared__ uint32_t part[kGemvThreads / 32][MR];
    const int tid = threadIdx.x, lane = tid & 31;
    const int chunks = p.K / 16, tail = p.K % 16;  // whole 16 bytes of k, and what is left
    const uint32_t warps = gridDim.x * (kGemvThreads / 32);
    ColumnWalk cols{(blockIdx.x * (kGemvThreads / 32) + (tid >> 5)) * kGemvCols, warps * kGemvCols,
                    static_cast<uint32_t>(p.N)};

    // two steps of 16 bytes a lane for each channel; channels past the end read the last one
    uint4 w[kGemvCols][2];
    auto channel = [&](int i) { return p.w + static_cast<long long>(cols.column(i)) * p.ldw; };
    auto load = [&](int c) {
#pragma unroll
        for (int i = 0; i < kGemvCols; ++i) {
            const uint4* row = reinterpret_cast<const uint4*>(channel(i));
#pragma unroll
            for (int s = 0; s < 2; ++s) w[i][s] = c + 32 * s < chunks ? row[c + 32 * s] : make_uint4(0, 0, 0, 0);
        }
    };
    grid_dependency_wait();
    if (cols.live()) load(lane);
    if (p.x_dt == OP_I8) {
        for (int m = 0; m < MR; ++m) {
            const int8_t* row = static_cast<const int8_t*>(p.x) + m * p.ldx;
            for (int c = tid; c < chunks; c += kGemvThreads)
                reinterpret_cast<uint4*>(sx + m * p.kpad)[c] =
                    m < p.M ? reinterpret_cast<const uint4*>(row)[c] : make_uint4(0, 0, 0, 0);
            if (tid < tail) sx[m * p.kpad + chunks * 16 + tid] = m < p.M ? static_cast<uint8_t>(row[chunks * 16 + tid]) : 0;
        }
        if (tid < MR) scale[tid] = tid < p.M ? p.x_scale[tid] : 0.0f;
    } else if (p.x_dt == OP_F32) {
        gemv_quantise<float, MR>(p, sx, scale, part);
    } else if (p.x_dt == OP_F16) {
        gemv_quantise<__half, MR>(p, sx, scale, part);
    } else {
        gemv_quantise<__nv_bfloat16, MR>(p, sx, scale, part);
    }
    __syncthreads();

    while (cols.live()) {
        int acc[kGemvCols][MR] = {};
        const int8_t* last[kGemvCols];
        if (tail) {
#pragma unroll
            for (int i = 0; i < kGemvCols; ++i) last[i] = channel(i) + chunks * 16;
        }
        const uint32_t first = cols.at;
        for (int c = lane; c - lane < chunks; c += 64) {
            uint4 a[kGemvCols][2];
#pragma unroll
            for (int i = 0; i < kGemvCols; ++i) a[i][0] = w[i][0], a[i][1] = w[i][1];
            // the next weights travel while these are multiplied
            if (c - lane + 64 < chunks) {
                load(c + 64);
            } else {
                cols.next();
                if (cols.live()) load(lane);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (c + 32 * s < chunks) {
#pragma unroll
                    for (int m = 0; m < MR; ++m) {
                        const int4 v = *reinterpret_cast<const int4*>(sx + m * p.kpad + (c + 32 * s) * 16);
#pragma unroll
                        for (int i = 0; i < kGemvCols; ++i) {
                            acc[i][m] = __dp4a(static_cast<int>(a[i][s].x), v.x, acc[i][m]);
                            acc[i][m] = __dp4a(static_cast<int>(a[i][s].y), v.y, acc[i][m]);
                            acc[i][m] = __dp4a(static_cast<int>(a[i][s].z), v.z, acc[i][m]);
                            acc[i][m] = __dp4a(static_cast<int>(a[i][s].w), v.w, acc[i][m]);
                        }
                    }
                }
            }
        }
        if (chunks == 0) cols.next();
        if (lane < tail) {
#pragma unroll
            for (int i = 0; i < kGemvCols; ++i)
#pragma unroll
                for (int m = 0; m < MR; ++m)
                    acc[i][m] += static_cast<int>(last[i][lane]) *
                                 static_cast<int>(static_cast<int8_t>(sx[m * p.kpad + chunks * 16 + lane]));
        }
        int mine = 0;  // lane i * MR + m finishes channel i of row m
#pragma unroll
        for (int i = 0; i < kGemvCols; ++i)
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const int sum = __reduce_add_sync(0xffffffffu, acc[i][m]);
                if (lane == i * MR + m) mine = sum;
            }
        const uint32_t n = first + lane / MR;
        const int m = lane % MR;
        if (lane < kGemvCols * MR && n < cols.n && m < p.M) {
            const float b = p.bias ? p.bias[n] : 0.0f;
            store1(p.out, p.out_dt, m * p.ldo + n, finish1(mine, scale[m], p.ws[n], b, p.act));
        }
    }
}

// ------------------------------------------------------------------------- skinny
struct SkinnyParams {
    int M, N, tiles_n;
    int num_kb, split;  // k-blocks of 128 bytes, shared by `split` CTAs of a cluster
    const float* xs;
    const float* ws;
    const float* bias;
    int act, out_dt, out_vec;  // out_vec: 4 values of a row are an aligned access
    int early_w;               // the kernel before is the quantisation of this call
    void* out;
    long long ldo;
};

constexpr int kSkinnyThreads = 128;

template <int NT>
struct SkinnyCfg {
    static constexpr int W_BYTES = 128 * 128;
    static constexpr int X_BYTES = NT * 128;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
    // two CTAs an SM: about 100 KB each, and room for the 128 x NT sums in the same place
    static constexpr int STAGES = 98304 / STAGE_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
    static constexpr int TMEM_COLS = NT < 32 ? 32 : NT;
    static_assert(NT * 128 * 4 <= STAGES * STAGE_BYTES, "the sums fit the stages' memory");
    static_assert(X_BYTES % 1024 == 0, "operand tiles must be whole swizzle atoms");
};

__device__ __forceinline__ int4 ld_cluster_int4(uint32_t caddr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(caddr)
                 : "memory");
    return v;
}

template <int NT>
__global__ void __launch_bounds__(kSkinnyThreads)
    int8_skinny_kernel(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX,
                       const __grid_constant__ SkinnyParams p) {
    using C = SkinnyCfg<NT>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sW = smem;
    uint8_t* sX = smem + STAGES * C::W_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* done = full + 2 * STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + 2 * STAGES + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* err = &g_status.code;

    const int tid = threadIdx.x, warp = tid >> 5;
    const int split = p.split;
    const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int tile = blockIdx.x / split;
    const int m0 = tile / p.tiles_n * NT;  // the tile's tokens and channels
    const int n0 = tile % p.tiles_n * 128;
    const int tokens = min(NT, p.M - m0);
    const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * rank / split);
    const int kb1 = static_cast<int>(static_cast<long long>(p.num_kb) * (rank + 1) / split);

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&mapW);
        prefetch_tmap(&mapX);
    }
    if (warp == 1) tmem_alloc(tmem_slot, C::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (tid == 0) {
        // ------------------------------------------------ TMA producer
        // the first weights travel while this call's quantisation still runs: it has waited for all that
        // came before
        if (!p.early_w) grid_dependency_wait();
        const int early = min(STAGES, kb1 - kb0);
        for (int s = 0; s < early; ++s) {
            mbar_arrive_expect_tx(&full[s], C::STAGE_BYTES);
            tma_load_2d(sW + s * C::W_BYTES, &mapW, &full[s], (kb0 + s) * 128, n0);
        }
        grid_dependency_wait();
        for (int s = 0; s < early; ++s) tma_load_2d(sX + s * C::X_BYTES, &mapX, &full[s], (kb0 + s) * 128, m0);
        bool ok = true;
        int it = early;
        for (int kb = kb0 + early; kb < kb1; ++kb, ++it) {
            const int s = it % STAGES;
            if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, kDevTimeoutProducer, err)) {
                ok = false;
                break;
            }
            mbar_arrive_expect_tx(&full[s], C::STAGE_BYTES);
            tma_load_2d(sW + s * C::W_BYTES, &mapW, &full[s], kb * 128, n0);
            tma_load_2d(sX + s * C::X_BYTES, &mapX, &full[s], kb * 128, m0);
        }
        if (!ok) {  // drain: wait (bounded) for loads that may still be in flight
            volatile int dummy = 0;
            for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j)
                mbar_wait(&full[j % STAGES], (j / STAGES) & 1, &dummy, kDevTimeoutProducer, err);
        }
    } else if (tid == 32) {
        // ------------------------------------------------ MMA issuer
        constexpr uint32_t idesc = idesc_i8kind(128, NT);
        int it = 0;
        grid_dependency_wait();  // the limit of the waits below counts from here
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % STAGES;
            if (!mbar_wait(&full[s], (it / STAGES) & 1, abort_flag, kDevTimeoutMma, err)) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
                mma_i8_ss(tmem, umma_desc_sw128(smem_u32(sW + s * C::W_BYTES) + k * 32, 16, 1024),
                          umma_desc_sw128(smem_u32(sX + s * C::X_BYTES) + k * 32, 16, 1024), idesc,
                          it > 0 || k > 0 ? 1u : 0u);
            mma_commit(&empty[s]);
        }
        mma_commit(done);
    }
    __syncwarp();
    // ------------------------------------------------ sums to shared memory: part[token][channel]
    grid_dependency_wait();
    const int lane = tid & 31;
    float ws[4], bias[4];  // of the 4 channels that this thread finishes
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int n = n0 + 4 * lane + c;
        ws[c] = n < p.N ? p.ws[n] : 0.0f;
        bias[c] = n < p.N && p.bias ? p.bias[n] : 0.0f;
    }
    {
        volatile int dummy = 0;
        mbar_wait(done, 0, &dummy, kDevTimeoutEpilogue, err);
    }
    tc_fence_after();
    __syncthreads();  // every load has landed and been multiplied: the stages' memory is free
    int* part = reinterpret_cast<int*>(smem);
#pragma unroll 1
    for (int c = 0; c < NT; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * 128 + tid] = static_cast<int>(r[i]);
    }
    tc_fence_before();
    if (split > 1)
        cluster_sync();
    else
        __syncthreads();
    // ------------------------------------------------ tokens rank, rank + split, ... of all sums
    uint32_t peer[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
        peer[r] = cluster_addr(smem_u32(part + 4 * lane), static_cast<uint32_t>(r < split ? r : 0));
    constexpr int U = 2;  // tokens of a warp at once
    for (int t0 = rank + split * warp; t0 < tokens; t0 += 4 * U * split) {
        int4 v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int t = t0 + u * 4 * split;
                v[u][r] = r < split && t < tokens ? ld_cluster_int4(peer[r] + t * 512) : make_int4(0, 0, 0, 0);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t0 + u * 4 * split;
            if (t >= tokens) continue;
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < 8; ++r) sum[0] += v[u][r].x, sum[1] += v[u][r].y, sum[2] += v[u][r].z, sum[3] += v[u][r].w;
            const float xs = p.xs[m0 + t];
            float y[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = finish1(sum[c], xs, ws[c], bias[c], p.act);
            const long long at = (m0 + t) * p.ldo + n0 + 4 * lane;
            if (p.out_vec && n0 + 4 * lane + 4 <= p.N) {
                if (p.out_dt == OP_F32)
                    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
                else if (p.out_dt == OP_F16)
                    *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) =
                        make_uint2(Elem<__half>::pack(y[0], y[1]), Elem<__half>::pack(y[2], y[3]));
                else
                    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
                        make_uint2(Elem<__nv_bfloat16>::pack(y[0], y[1]), Elem<__nv_bfloat16>::pack(y[2], y[3]));
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n0 + 4 * lane + c < p.N) store1(p.out, p.out_dt, at + c, y[c]);
            }
        }
    }
    if (split > 1)
        cluster_sync();  // no CTA leaves while another reads its sums
    else
        __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

}  // namespace

}  // namespace m3r
