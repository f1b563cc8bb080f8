// Product in 8-bit integers with a scale for each row of x and each row of W:
//
//   y[i, n] = act( (sum_k q[i, k] w[n, k]) * s[i] * t[n] + bias[n] )
//
// x arrives as 8-bit rows with scales, or in 16 / 32 bits and is quantised row by row first
// (row_norm.cu).  Sums are exact in 32-bit integers (k <= 131,072 keeps 127^2 k below 2^31).
//
// Persistent tcgen05 kernel (kind::i8, twice the 16-bit rate): 320 threads -- warps 0-7
// epilogue, warp 8 TMA producer, warp 9 TMEM allocator and MMA issuer -- on tiles of
// 128 x BN (one CTA) or 256 x BN (a CTA pair, cta_group::2), k in blocks of 128 bytes (one
// swizzle atom a row), accumulators double-buffered in TMEM so that the epilogue of a tile
// overlaps the main loop of the next.
#include <mutex>

#include "common.cuh"
#include "gemm.cuh"
#include "ops.h"
#include "tmap.h"

namespace m3r {

namespace {

// First wait of any operator kernel that ran out on this device (see mbar_wait).
__device__ DevStatus g_status;

struct Int8Params {
    int M, N, num_kb, tiles_m, tiles_n;  // tiles_m: blocks of 128 CG rows
    const float* xs;
    const float* ws;
    const float* bias;
    int act, out_dt, c_tma;
    void* out;
    long long ldo;
};

template <int BN, int CG>
struct I8Cfg {
    static constexpr int B_ROWS = BN / CG;
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = B_ROWS * 128;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int EPI_STAGE_BYTES = kGemmEpiWarps * 4096;
    static constexpr int FIXED_BYTES = 1024 + EPI_STAGE_BYTES + 256;
    static constexpr int FIT = (227 * 1024 - FIXED_BYTES) / STAGE_BYTES;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int ACC_COLS = BN;
    static constexpr int TMEM_COLS = 2 * ACC_COLS;  // a power of two
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + FIXED_BYTES;
};

// Row blocks are walked in groups of 8 down the rows first, so that the CTAs at work share
// few row blocks of x and of W and both stay in L2 whatever their sizes.
__device__ __forceinline__ void tile_at(const Int8Params& p, int t, int& m, int& n) {
    constexpr int G = 8;
    const int group = t / (G * p.tiles_n);
    const int r = t - group * G * p.tiles_n;
    const int gm = min(G, p.tiles_m - group * G);
    n = r / gm;
    m = group * G + (r - n * gm);
}

// scale and bias of 32 columns: v = acc * xs * ws + bias, then the activation
__device__ __forceinline__ void finish32(const Int8Params& p, float (&v)[32], const uint32_t (&acc)[32], float xs,
                                         int col0) {
    const bool vec = col0 + 32 <= p.N && (reinterpret_cast<uintptr_t>(p.ws) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
    if (vec) {
        const float4* w4 = reinterpret_cast<const float4*>(p.ws + col0);
        const float4* b4 = reinterpret_cast<const float4*>(p.bias + col0);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float4 w = __ldg(w4 + q);
            const float4 b = p.bias ? __ldg(b4 + q) : make_float4(0, 0, 0, 0);
            v[4 * q] = static_cast<float>(static_cast<int>(acc[4 * q])) * xs * w.x + b.x;
            v[4 * q + 1] = static_cast<float>(static_cast<int>(acc[4 * q + 1])) * xs * w.y + b.y;
            v[4 * q + 2] = static_cast<float>(static_cast<int>(acc[4 * q + 2])) * xs * w.z + b.z;
            v[4 * q + 3] = static_cast<float>(static_cast<int>(acc[4 * q + 3])) * xs * w.w + b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const bool in = col0 + i < p.N;
            v[i] = static_cast<float>(static_cast<int>(acc[i])) * xs * (in ? __ldg(p.ws + col0 + i) : 0.0f) +
                   (in && p.bias ? __ldg(p.bias + col0 + i) : 0.0f);
        }
    }
    if (p.act == ACT_GELU) {
        if (p.out_dt == OP_F32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = gelu_tanh(v[i]);
        } else {
            // tanh.approx: relative error 2^-11 of the tanh, below the 16-bit result's rounding
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = gelu_fast(v[i]);
        }
    } else if (p.act == ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // keeps NaN
    }
}

// One tile's rows of this thread (tile row r), column group grp: units of 128 output bytes
// a row (32 fp32 or 64 16-bit columns), staged in shared memory and stored by TMA, or by
// row-contiguous thread stores where the output's layout does not allow TMA.
template <int BN>
__device__ __forceinline__ void i8_epilogue(const Int8Params& p, const CUtensorMap* map_out, uint32_t tacc,
                                            long long row0, int r, int grp, int n0, const RowStage& st) {
    const long long grow = row0 + r;
    const bool valid = grow < p.M;
    const bool wok = grow - st.lane < p.M;  // the warp's first row exists
    const float xs = valid ? __ldg(p.xs + grow) : 0.0f;
    const int unit = p.out_dt == OP_F32 ? 32 : 64;
#pragma unroll 1
    for (int c0 = grp * unit; c0 < BN; c0 += 2 * unit) {
        const int col0 = n0 + c0;
        if (col0 >= p.N) break;  // warp-uniform
        uint4 o[8];
        {
            uint32_t raw[32];
            float v[32];
            tmem_ld32(tacc + c0, raw);
            tmem_wait_ld();
            finish32(p, v, raw, xs, col0);
            if (p.out_dt == OP_F32) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    o[q] = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                                      __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
            } else {
                float hi[32];
                tmem_ld32(tacc + c0 + 32, raw);
                tmem_wait_ld();
                finish32(p, hi, raw, xs, col0 + 32);
                if (p.out_dt == OP_F16)
                    pack16x64<__half>(o, v, hi);
                else
                    pack16x64<__nv_bfloat16>(o, v, hi);
            }
        }
        if (p.c_tma && st.lane == 0) bulk_wait_read_all();
        __syncwarp();  // the previous unit's reads of the stage (threads or TMA) are done
        st.put_own(o);
        if (p.c_tma) {
            fence_proxy_async_smem();
            __syncwarp();
            if (st.lane == 0 && wok) {
                tma_store_2d(map_out, st.buf, col0, static_cast<int>(grow));
                bulk_commit();
            }
        } else {
            __syncwarp();
            const int esz = p.out_dt == OP_F32 ? 4 : 2;
            const int bytes = (col0 + unit <= p.N ? unit : p.N - col0) * esz;
            char* dst = valid ? static_cast<char*>(p.out) + (grow * p.ldo + col0) * esz : nullptr;
            const int c = st.lane & 7;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = i * 4 + (st.lane >> 3);
                char* d = reinterpret_cast<char*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
                const uint4 u = *st.at(row, c);
                if (d == nullptr) continue;
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
                if (esz == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c * 16 + 4 * e < bytes) *reinterpret_cast<uint32_t*>(d + c * 16 + 4 * e) = w[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c * 16 + 2 * e < bytes)
                            *reinterpret_cast<uint16_t*>(d + c * 16 + 2 * e) =
                                static_cast<uint16_t>(w[e >> 1] >> ((e & 1) * 16));
                }
            }
        }
    }
}

// CG = 2: launched as clusters of 2 CTAs; the even CTA's thread issues the M = 256 MMAs.  A
// wait that runs out raises the abort flag of both CTAs; neither leaves before the other.
template <int BN, int CG>
__global__ void __launch_bounds__(kGemmThreads, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                     const __grid_constant__ CUtensorMap mapC, const __grid_constant__ Int8Params p) {
    using C = I8Cfg<BN, CG>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * C::A_BYTES;
    uint8_t* epi_stage = smem + STAGES * C::STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(epi_stage + C::EPI_STAGE_BYTES);
    uint64_t* full = bars;
    uint64_t* empty = bars + STAGES;
    uint64_t* tfull = bars + 2 * STAGES;
    uint64_t* tempty = bars + 2 * STAGES + 2;
    uint64_t* mma_done = bars + 2 * STAGES + 4;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* err = &g_status.code;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = CG == 2 ? static_cast<int>(cluster_rank()) : 0;
    const bool leader = rank == 0;
    const int unit = blockIdx.x / CG;
    const int num_units = gridDim.x / CG;
    const int num_tiles = p.tiles_m * p.tiles_n;

    if (warp == kGemmTmaWarp && lane == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], CG * kGemmEpiWarps);
        }
        mbar_init(mma_done, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&mapA);
        prefetch_tmap(&mapB);
    }
    if (warp == kGemmMmaWarp) {
        if (CG == 2)
            tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
        else
            tmem_alloc(tmem_slot, C::TMEM_COLS);
    }
    tc_fence_before();
    if (CG == 2)
        cluster_sync();
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t full_c = CG == 2 ? cluster_addr(smem_u32(full), 0) : smem_u32(full);
    const uint32_t tempty_c = CG == 2 ? cluster_addr(smem_u32(tempty), 0) : smem_u32(tempty);
    const uint32_t peer_abort_c =
        CG == 2 ? cluster_addr(smem_u32(const_cast<int*>(abort_flag)), static_cast<uint32_t>(rank ^ 1)) : 0u;
    auto abort_pair = [&]() {
        *abort_flag = 1;
        if (CG == 2) st_cluster_u32(peer_abort_c, 1u);
    };

    if (warp == kGemmTmaWarp) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += num_units) {
                int m, n;
                tile_at(p, t, m, n);
                const int arow = (m * CG + rank) * 128;
                const int brow = n * BN + rank * C::B_ROWS;
                for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, kDevTimeoutProducer, err)) {
                        ok = false;
                        abort_pair();
                        break;
                    }
                    if (leader) mbar_arrive_expect_tx(&full[s], CG * C::STAGE_BYTES);
                    uint8_t* a_dst = sA + s * C::A_BYTES;
                    uint8_t* b_dst = sB + s * C::B_BYTES;
                    if (CG == 2) {
                        tma_load_2d_pair(a_dst, &mapA, full_c + s * 8, kb * 128, arow);
                        tma_load_2d_pair(b_dst, &mapB, full_c + s * 8, kb * 128, brow);
                    } else {
                        tma_load_2d(a_dst, &mapA, &full[s], kb * 128, arow);
                        tma_load_2d(b_dst, &mapB, &full[s], kb * 128, brow);
                    }
                }
            }
            if (!ok) {
                if (CG == 1) {
                    // drain: wait (bounded) for loads that may still be in flight
                    const uint32_t first = it > STAGES ? it - STAGES : 0;
                    for (uint32_t j = first; j < it; ++j) {
                        volatile int dummy = 0;
                        mbar_wait(&full[j % STAGES], (j / STAGES) & 1, &dummy, kDevTimeoutProducer, err);
                    }
                } else {
                    // this CTA's loads signal the even CTA's barriers: give loads in flight
                    // 1 ms (TMA loads take microseconds) before the CTA may leave
                    const unsigned long long t0 = global_timer_ns();
                    while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
                }
            }
        }
    } else if (warp == kGemmMmaWarp) {
        if (lane == 0 && leader) {
            constexpr uint32_t idesc = idesc_i8kind(128 * CG, BN);
            uint32_t it = 0, tcount = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += num_units, ++tcount) {
                const uint32_t buf = tcount & 1;
                if (!mbar_wait(&tempty[buf], ((tcount >> 1) & 1) ^ 1, abort_flag, kDevTimeoutMma, err)) {
                    ok = false;
                    abort_pair();
                    break;
                }
                tc_fence_after();
                const uint32_t dacc = tmem_base + buf * C::ACC_COLS;
                for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&full[s], (it / STAGES) & 1, abort_flag, kDevTimeoutMma, err)) {
                        ok = false;
                        abort_pair();
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(sA + s * C::A_BYTES);
                    const uint32_t b_addr = smem_u32(sB + s * C::B_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint64_t ad = umma_desc_sw128(a_addr + k * 32, 16, 1024);
                        const uint64_t bd = umma_desc_sw128(b_addr + k * 32, 16, 1024);
                        const uint32_t acc = (kb > 0 || k > 0) ? 1u : 0u;
                        if (CG == 2)
                            mma_i8_ss_pair(dacc, ad, bd, idesc, acc);
                        else
                            mma_i8_ss(dacc, ad, bd, idesc, acc);
                    }
                    if (CG == 2)
                        mma_commit_pair_both(&empty[s]);
                    else
                        mma_commit(&empty[s]);
                }
                if (ok) {
                    if (CG == 2)
                        mma_commit_pair_both(&tfull[buf]);
                    else
                        mma_commit(&tfull[buf]);
                }
            }
            // all issued MMAs complete before either CTA may release TMEM or leave
            if (CG == 2)
                mma_commit_pair_local(mma_done);
            else
                mma_commit(mma_done);
            volatile int dummy = 0;
            mbar_wait(mma_done, 0, &dummy, kDevTimeoutMma, err);
        }
    } else {
        const int quarter = warp & 3;
        const int grp = warp >> 2;
        const RowStage st{epi_stage + warp * 4096, lane};
        uint32_t tcount = 0;
        for (int t = unit; t < num_tiles; t += num_units, ++tcount) {
            const uint32_t buf = tcount & 1;
            int m, n;
            tile_at(p, t, m, n);
            if (!mbar_wait(&tfull[buf], (tcount >> 1) & 1, abort_flag, kDevTimeoutEpilogue, err)) {
                abort_pair();
                break;
            }
            tc_fence_after();
            const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * C::ACC_COLS;
            i8_epilogue<BN>(p, &mapC, tacc, static_cast<long long>(m * CG + rank) * 128, quarter * 32 + lane, grp,
                            n * BN, st);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2)
                    mbar_arrive_cluster(tempty_c + buf * 8);
                else
                    mbar_arrive(&tempty[buf]);
            }
        }
        if (lane == 0) bulk_wait_all();  // TMA stores of this warp complete before the CTA ends
    }
    __syncwarp();
    if (CG == 2)
        cluster_sync();
    else
        __syncthreads();
    if (warp == kGemmMmaWarp) {
        tc_fence_after();
        if (CG == 2)
            tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
        else
            tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

int sm_count(int dev) {
    static int n[16] = {};
    if (dev < 0 || dev >= 16) dev = 0;
    if (n[dev] == 0) M3R_CUDA(cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev));
    return n[dev];
}

template <int BN, int CG>
void launch(cudaStream_t s, const Int8LinearParams& q, const int8_t* xq, long long ldq, const float* xs) {
    using C = I8Cfg<BN, CG>;
    auto kern = int8_gemm_kernel<BN, CG>;
    int dev = 0;
    M3R_CUDA(cudaGetDevice(&dev));
    {
        static std::mutex mu;
        static unsigned done = 0;  // devices whose limit is raised
        std::lock_guard<std::mutex> lock(mu);
        if (dev >= 32 || !(done >> dev & 1)) {
            M3R_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
            if (dev < 32) done |= 1u << dev;
        }
    }
    Int8Params p;
    p.M = static_cast<int>(q.rows);
    p.N = q.n;
    p.num_kb = cdiv(q.k, 128);
    p.tiles_m = cdiv(q.rows, 128 * CG);
    p.tiles_n = cdiv(q.n, BN);
    p.xs = xs;
    p.ws = q.w_scale;
    p.bias = q.bias;
    p.act = q.act;
    p.out_dt = q.out_dt;
    p.out = q.out;
    p.ldo = q.ldo;
    const CUtensorMap ma = tmap_2d_u8(xq, q.rows, q.k, ldq, 128);
    const CUtensorMap mb = tmap_2d_u8(q.w, q.n, q.k, q.ldw, C::B_ROWS);
    CUtensorMap mc = ma;
    p.c_tma = reinterpret_cast<uintptr_t>(q.out) % 16 == 0 && q.ldo * op_size(q.out_dt) % 16 == 0;
    if (p.c_tma)
        mc = q.out_dt == OP_F32 ? tmap_2d_f32(q.out, q.rows, q.n, q.ldo, 32)
                                : tmap_2d(q.out_dt, q.out, q.rows, q.n, q.ldo, 32);
    const int units = p.tiles_m * p.tiles_n;
    const int max_units = sm_count(dev) / CG;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CG * (units < max_units ? units : max_units));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    M3R_CUDA(cudaLaunchKernelEx(&cfg, kern, ma, mb, mc, p));
}

long long padded_k(int k) { return (static_cast<long long>(k) + 15) / 16 * 16; }
size_t round256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace

// 8-bit rows of x, then their scales.
size_t int8_linear_workspace(int x_dt, long long rows, int n, int k) {
    (void)n;
    if (x_dt == OP_I8 || rows == 0) return 0;
    return round256(static_cast<size_t>(rows) * padded_k(k)) + round256(static_cast<size_t>(rows) * 4);
}

void int8_linear(cudaStream_t s, const Int8LinearParams& p) {
    if (p.rows == 0) return;
    const int8_t* xq = static_cast<const int8_t*>(p.x);
    long long ldq = p.ldx;
    const float* xs = p.x_scale;
    if (p.x_dt != OP_I8) {
        int8_t* q = static_cast<int8_t*>(p.workspace);
        float* sc = reinterpret_cast<float*>(q + round256(static_cast<size_t>(p.rows) * padded_k(p.k)));
        RowNormParams r = {};
        r.rows = p.rows;
        r.cols = p.k;
        r.x_dt = p.x_dt;
        r.out_dt = OP_I8;
        r.alpha = 1.0f;
        r.ldx = p.ldx;
        r.ldo = padded_k(p.k);
        r.x = p.x;
        r.out = q;
        r.out_scale = sc;
        row_norm(s, r);
        xq = q;
        ldq = padded_k(p.k);
        xs = sc;
    }
    int dev = 0;
    M3R_CUDA(cudaGetDevice(&dev));
    const int sms = sm_count(dev);
    // the largest tile that gives every SM one
    if (static_cast<long long>(cdiv(p.rows, 256)) * cdiv(p.n, 256) * 2 >= sms)
        launch<256, 2>(s, p, xq, ldq, xs);
    else if (static_cast<long long>(cdiv(p.rows, 128)) * cdiv(p.n, 128) >= sms)
        launch<128, 1>(s, p, xq, ldq, xs);
    else
        launch<64, 1>(s, p, xq, ldq, xs);
}

int int8_linear_status(cudaStream_t s) {
    DevStatus st;
    M3R_CUDA(cudaStreamSynchronize(s));
    M3R_CUDA(cudaMemcpyFromSymbol(&st, g_status, sizeof(st)));
    if (st.code != 0) {
        const DevStatus zero = {};
        M3R_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(zero)));
    }
    return st.code;
}

}  // namespace m3r
