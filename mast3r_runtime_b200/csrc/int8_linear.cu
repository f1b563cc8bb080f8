// Product in 8-bit integers with a scale for each row of x and each row of W:
//
//   y[i, n] = act( (sum_k q[i, k] w[n, k]) * s[i] * t[n] + bias[n] )
//
// x arrives as 8-bit rows with scales, or in 16 / 32 bits and is quantised row by row first
// (row_norm.cu).  Sums are exact in 32-bit integers (k <= 131,071 keeps 128^2 k below 2^31).
//
// Persistent tcgen05 kernel (kind::i8, twice the 16-bit rate): 320 threads -- warps 0-7
// epilogue, warp 8 TMA producer, warp 9 TMEM allocator and MMA issuer -- on tiles of
// 128 x BN (one CTA) or 256 x BN (a CTA pair, cta_group::2), k in blocks of 128 bytes (one
// swizzle atom a row), accumulators double-buffered in TMEM so that the epilogue of a tile
// overlaps the main loop of the next.
//
// Bound: at long k the tensor cores (8,192^3: 346 us, 3.18 PFLOP/s, 0.97 of twice the measured bf16
// rate); at short k the 12 TB/s or so at which all SMs together exchange tiles with L2 -- a k-block of
// a 256 x 256 tile brings 64 KB for 0.27 us of multiplication, and the results go out the same way
// (98,304 x 4,096 x 1,024: 330 us with a bf16 result, 2.5 PFLOP/s; 270 us without any results).
// Keeping the rows' whole k resident saves two fifths of that traffic, but leaves shared memory for
// three stages of W only: 394 us.
#include "common.cuh"
#include "gemm.cuh"
#include "launch.h"
#include "ops.h"
#include "tmap.h"

namespace m3r {

namespace {

// First wait of any operator kernel that ran out on this device (see mbar_wait).
__device__ DevStatus g_status;

}  // namespace

}  // namespace m3r

#include "int8_small.cuh"

namespace m3r {

namespace {

constexpr int kEpiWarps = 8;
constexpr int kEpiGroups = kEpiWarps / 4;         // warps that share a TMEM lane quarter
constexpr int kWarpCols = 256 / kEpiGroups;       // most columns of a tile that one warp handles
constexpr int kTmaWarp = kEpiWarps;
constexpr int kMmaWarp = kEpiWarps + 1;
constexpr int kThreads = (kEpiWarps + 2) * 32;

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
    // each epilogue warp: 4 KB of result rows, and the scale and bias of its columns
    static constexpr int EPI_STAGE_BYTES = kEpiWarps * 4096;
    static constexpr int COLS_BYTES = kEpiWarps * kWarpCols * 8;
    static constexpr int FIXED_BYTES = 1024 + EPI_STAGE_BYTES + COLS_BYTES + 256;
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

// -2 log2(e) sqrt(2 / pi), and that times 0.044715: with t = x (kGelu0 + kGelu1 x^2), the GELU's tanh form
// x / 2 (1 + tanh u) is x / (1 + 2^t), to a few 32-bit roundings of the result.  For 16-bit results too:
// 1 + tanh.approx(u) cancels where the tanh nears -1 (its error of 2^-11 is a fifth of the result at x = -3)
// and saves an eighth of the time at most (fp16 result from 8-bit rows: 24,576 x 4,096 x 1,024 95 us against
// 106, 1,536 x 4,096 x 1,024 13.7 against 15.5, 64 x 4,096 x 1,024 6.2 against 6.5).
constexpr float kGelu0 = -2.885390081777927f * 0.7978845608028654f;
constexpr float kGelu1 = -2.885390081777927f * 0.7978845608028654f * 0.044715f;

// Two neighbouring columns of a row: acc * xs * ws + bias, then the activation.
template <int ACT>
__device__ __forceinline__ uint64_t finish2(uint32_t a0, uint32_t a1, float xs, const ulonglong2& col) {
    uint64_t v = fma2(mul2(pair(static_cast<int>(a0), static_cast<int>(a1)), pair(xs, xs)), col.x, col.y);
    if constexpr (ACT == ACT_GELU) {
        const float2 t = unpair(mul2(v, fma2(mul2(v, v), pair(kGelu1, kGelu1), pair(kGelu0, kGelu0))));
        const float2 d = unpair(add2(pair(ex2_approx(t.x), ex2_approx(t.y)), pair(1.0f, 1.0f)));
        v = mul2(v, pair(rcp_approx(d.x), rcp_approx(d.y)));
    } else if constexpr (ACT == ACT_RELU) {
        const float2 x = unpair(v);
        v = pair(x.x < 0.0f ? 0.0f : x.x, x.y < 0.0f ? 0.0f : x.y);  // keeps NaN
    }
    return v;
}

// Four 8 x 8 blocks of 16-bit values in fragment order to shared memory: lane l gives the address of
// row l % 8 of block l / 8.
__device__ __forceinline__ void store_blocks(const void* row, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(a),
                 "r"(b), "r"(c), "r"(d)
                 : "memory");
}

template <int OUT>
struct OutType {
    using T = __half;
};
template <>
struct OutType<OP_BF16> {
    using T = __nv_bfloat16;
};

// One tile's 32 rows of a warp (from global row `row0`), column group grp: units of 128 output
// bytes a row (32 fp32 or 64 16-bit columns), staged in shared memory and stored by TMA, or by
// row-contiguous thread stores where the output's layout does not allow TMA.  The sums come from
// TMEM as fragments -- a thread has 2 columns of every 8, of 4 rows -- so that a column's scale and
// bias go to the 4 threads that need them: with a whole row a thread, broadcasting every column's
// 8 bytes to 32 threads took more shared-memory time than all else.  cols: (scale 2, bias 2) of the
// warp's column pairs; xs: the scales of the thread's rows 8 i + lane / 4.  `release` hands the
// accumulator back once the last of it is in registers.
template <int BN, int OUT, int ACT, class Release>
__device__ __forceinline__ void i8_epilogue(const Int8Params& p, const CUtensorMap* map_out, uint32_t tacc,
                                            long long row0, int grp, int n0, const RowStage& st,
                                            const ulonglong2* cols, const float (&xs)[4], Release&& release) {
    constexpr int unit = OUT == OP_F32 ? 32 : 64;
    constexpr int esz = OUT == OP_F32 ? 4 : 2;
    const int lane = st.lane;
    const int end = min(BN, p.N - n0);
    if (grp * unit >= end) release();
    cols += lane & 3;
#pragma unroll 1
    for (int c0 = grp * unit; c0 < end; c0 += kEpiGroups * unit, cols += unit / 2) {
        const int col0 = n0 + c0;
        uint32_t lo[unit / 2], hi[unit / 2];  // rows 0-15 and 16-31
        if constexpr (OUT == OP_F32) {
            tmem_ld_frag4(tacc + c0, lo);
            tmem_ld_frag4(tacc + (16u << 16) + c0, hi);
        } else {
            tmem_ld_frag8(tacc + c0, lo);
            tmem_ld_frag8(tacc + (16u << 16) + c0, hi);
        }
        if (p.c_tma && lane == 0) bulk_wait_read_all();
        tmem_wait_ld();
        if (c0 + kEpiGroups * unit >= end) release();
        __syncwarp();  // the previous unit's reads of the stage (threads or TMA) are done
        if constexpr (OUT == OP_F32) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const ulonglong2 c = cols[4 * g];
                const uint64_t v[4] = {finish2<ACT>(lo[4 * g], lo[4 * g + 1], xs[0], c),
                                       finish2<ACT>(lo[4 * g + 2], lo[4 * g + 3], xs[1], c),
                                       finish2<ACT>(hi[4 * g], hi[4 * g + 1], xs[2], c),
                                       finish2<ACT>(hi[4 * g + 2], hi[4 * g + 3], xs[3], c)};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    reinterpret_cast<uint64_t*>(st.at(8 * i + (lane >> 2), 2 * g + ((lane & 3) >> 1)))[lane & 1] = v[i];
            }
        } else {
#pragma unroll
            for (int g = 0; g < 8; g += 2) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const ulonglong2 c = cols[4 * (g + e)];
                    const uint32_t* l = lo + 4 * (g + e);
                    const uint32_t* h = hi + 4 * (g + e);
                    const float2 v[4] = {unpair(finish2<ACT>(l[0], l[1], xs[0], c)),
                                         unpair(finish2<ACT>(l[2], l[3], xs[1], c)),
                                         unpair(finish2<ACT>(h[0], h[1], xs[2], c)),
                                         unpair(finish2<ACT>(h[2], h[3], xs[3], c))};
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[4 * e + i] = Elem<typename OutType<OUT>::T>::pack(v[i].x, v[i].y);
                }
                // blocks: rows 0-7 and 8-15 (then 16-23 and 24-31) of column groups g and g + 1
                const int row = (lane & 7) + (lane & 8), chunk = g + (lane >> 4);
                store_blocks(st.at(row, chunk), w[0], w[1], w[4], w[5]);
                store_blocks(st.at(row + 16, chunk), w[2], w[3], w[6], w[7]);
            }
        }
        if (p.c_tma) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M) {
                tma_store_2d(map_out, st.buf, col0, static_cast<int>(row0));
                bulk_commit();
            }
        } else {
            __syncwarp();
            // element accesses, a row's 128 bytes by 32 lanes: any alignment, whole sectors
            const int bytes = (col0 + unit <= p.N ? unit : p.N - col0) * esz;
            const int rows = static_cast<int>(min(32LL, p.M - row0));
            char* d = static_cast<char*>(p.out) + (row0 * p.ldo + col0) * esz + lane * 4;
#pragma unroll 4
            for (int row = 0; row < rows; ++row, d += p.ldo * esz) {
                const uint32_t u = reinterpret_cast<const uint32_t*>(st.at(row, lane >> 2))[lane & 3];
                if (lane * 4 >= bytes) continue;
                if constexpr (esz == 4) {
                    *reinterpret_cast<uint32_t*>(d) = u;
                } else {
                    *reinterpret_cast<uint16_t*>(d) = static_cast<uint16_t>(u);
                    if (lane * 4 + 2 < bytes) *reinterpret_cast<uint16_t*>(d + 2) = static_cast<uint16_t>(u >> 16);
                }
            }
        }
    }
}

// CG = 2: launched as clusters of 2 CTAs; the even CTA's thread issues the M = 256 MMAs.  A
// wait that runs out raises the abort flag of both CTAs; neither leaves before the other.
template <int BN, int CG>
__global__ void __launch_bounds__(kThreads, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                     const __grid_constant__ CUtensorMap mapC, const __grid_constant__ Int8Params p) {
    using C = I8Cfg<BN, CG>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * C::A_BYTES;
    uint8_t* epi_stage = smem + STAGES * C::STAGE_BYTES;
    uint8_t* epi_cols = epi_stage + C::EPI_STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(epi_cols + C::COLS_BYTES);
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

    if (warp == kTmaWarp && lane == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], CG * kEpiWarps);
        }
        mbar_init(mma_done, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&mapA);
        prefetch_tmap(&mapB);
    }
    if (warp == kMmaWarp) {
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
    grid_dependency_wait();
    const uint32_t full_c = CG == 2 ? cluster_addr(smem_u32(full), 0) : smem_u32(full);
    const uint32_t tempty_c = CG == 2 ? cluster_addr(smem_u32(tempty), 0) : smem_u32(tempty);
    const uint32_t peer_abort_c =
        CG == 2 ? cluster_addr(smem_u32(const_cast<int*>(abort_flag)), static_cast<uint32_t>(rank ^ 1)) : 0u;
    auto abort_pair = [&]() {
        *abort_flag = 1;
        if (CG == 2) st_cluster_u32(peer_abort_c, 1u);
    };

    if (warp == kTmaWarp) {
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
    } else if (warp == kMmaWarp) {
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
        float4* const cols = reinterpret_cast<float4*>(epi_cols + warp * kWarpCols * 8);  // (scale 2, bias 2)
        uint32_t tcount = 0;
        for (int t = unit; t < num_tiles; t += num_units, ++tcount) {
            const uint32_t buf = tcount & 1;
            int m, n;
            tile_at(p, t, m, n);
            const long long row0 = static_cast<long long>(m * CG + rank) * 128 + quarter * 32;  // of the warp
            // the scales and biases of the tile, before its sums are there: lane l brings columns
            // 2 l and 2 l + 1 of each 64 that the warp handles, unit by unit
            __syncwarp();  // the previous tile's reads are done
#pragma unroll
            for (int j = 2 * lane; j < kWarpCols; j += 64) {
                const int c = n * BN + (p.out_dt == OP_F32 ? (grp + (j >> 5) * kEpiGroups) * 32 + (j & 31)
                                                           : (grp + (j >> 6) * kEpiGroups) * 64 + (j & 63));
                float4 q = make_float4(0, 0, 0, 0);
                if (c < p.N) {
                    q.x = p.ws[c];
                    if (p.bias) q.z = p.bias[c];
                }
                if (c + 1 < p.N) {
                    q.y = p.ws[c + 1];
                    if (p.bias) q.w = p.bias[c + 1];
                }
                cols[j >> 1] = q;
            }
            __syncwarp();
            float xs[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long r = row0 + 8 * i + (lane >> 2);
                xs[i] = r < p.M ? p.xs[r] : 0.0f;
            }
            if (!mbar_wait(&tfull[buf], (tcount >> 1) & 1, abort_flag, kDevTimeoutEpilogue, err)) {
                abort_pair();
                break;
            }
            tc_fence_after();
            const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * C::ACC_COLS;
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2)
                        mbar_arrive_cluster(tempty_c + buf * 8);
                    else
                        mbar_arrive(&tempty[buf]);
                }
            };
            // one copy of the epilogue for each result type and activation
            auto by_act = [&](auto out) {
                constexpr int OUT = decltype(out)::value;
                const ulonglong2* cl = reinterpret_cast<const ulonglong2*>(cols);
                if (p.act == ACT_GELU)
                    i8_epilogue<BN, OUT, ACT_GELU>(p, &mapC, tacc, row0, grp, n * BN, st, cl, xs, release);
                else if (p.act == ACT_RELU)
                    i8_epilogue<BN, OUT, ACT_RELU>(p, &mapC, tacc, row0, grp, n * BN, st, cl, xs, release);
                else
                    i8_epilogue<BN, OUT, ACT_NONE>(p, &mapC, tacc, row0, grp, n * BN, st, cl, xs, release);
            };
            if (p.out_dt == OP_F32)
                by_act(std::integral_constant<int, OP_F32>());
            else if (p.out_dt == OP_F16)
                by_act(std::integral_constant<int, OP_F16>());
            else
                by_act(std::integral_constant<int, OP_BF16>());
        }
        if (lane == 0) bulk_wait_all();  // TMA stores of this warp complete before the CTA ends
    }
    __syncwarp();
    if (CG == 2)
        cluster_sync();
    else
        __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        if (CG == 2)
            tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
        else
            tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

int sm_count() {
    int dev = 0, n = 0;
    M3R_CUDA(cudaGetDevice(&dev));
    M3R_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    return n;
}

template <int BN, int CG>
void launch(cudaStream_t s, const Int8LinearParams& q, const int8_t* xq, long long ldq, const float* xs, int sms) {
    using C = I8Cfg<BN, CG>;
    auto kern = int8_gemm_kernel<BN, CG>;
    static unsigned done = 0;
    allow_smem(kern, C::SMEM_BYTES, done);
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
    const int max_units = sms / CG;
    const LaunchConfig c(CG * (units < max_units ? units : max_units), kThreads, C::SMEM_BYTES, s, CG);
    M3R_CUDA(cudaLaunchKernelEx(&c.cfg, kern, ma, mb, mc, p));
}

template <int NT>
void launch_skinny(cudaStream_t s, const Int8LinearParams& q, const int8_t* xq, long long ldq, const float* xs,
                   int split) {
    using C = SkinnyCfg<NT>;
    auto kern = int8_skinny_kernel<NT>;
    static unsigned done = 0;
    allow_smem(kern, C::SMEM_BYTES, done);
    SkinnyParams p;
    p.M = static_cast<int>(q.rows);
    p.N = q.n;
    p.tiles_n = cdiv(q.n, 128);
    p.num_kb = cdiv(q.k, 128);
    p.split = split;
    p.xs = xs;
    p.ws = q.w_scale;
    p.bias = q.bias;
    p.act = q.act;
    p.out_dt = q.out_dt;
    p.out = q.out;
    p.ldo = q.ldo;
    p.out_vec = q.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(q.out) % (4 * op_size(q.out_dt)) == 0;
    const CUtensorMap mw = tmap_2d_u8(q.w, q.n, q.k, q.ldw, 128);
    const CUtensorMap mx = tmap_2d_u8(xq, q.rows, q.k, ldq, NT);
    p.early_w = q.x_dt != OP_I8;
    const int tiles = p.tiles_n * cdiv(q.rows, NT);
    const LaunchConfig c(static_cast<unsigned>(tiles) * split, kSkinnyThreads, C::SMEM_BYTES, s, split);
    M3R_CUDA(cudaLaunchKernelEx(&c.cfg, kern, mw, mx, p));
}

long long padded_k(int k) { return (static_cast<long long>(k) + 15) / 16 * 16; }
size_t round256(size_t b) { return (b + 255) / 256 * 256; }

// Time of a tile shape, from what the shapes measured alone: a start (with the last epilogue), and for
// every round of tiles over the SMs its k-blocks, each as long as the larger of the tile's own rate and
// the 12 TB/s at which all SMs together read L2, or its epilogue.  (us: 1,536 x 1,024 x 1,024 8.7, 6.6
// and 8.9 with tiles of 256 x 256, 128 x 128 and 128 x 64; 1,536 x 3,072 x 1,024 9.2, 9.8, 14.6; 300 x
// 4,096 x 4,096 16.1, 14.2, 23.4; 200 x 1,024 x 1,024 8.4, 6.3, 6.0.)
double tile_us(int bn, int cg, long long rows, int n, int k, int sms) {
    const double start = bn == 256 ? 6.3 : bn == 128 ? 4.2 : 4.0;
    const double block = bn == 256 ? 0.298 : bn == 128 ? 0.303 : 0.25;
    const double epilogue = bn == 256 ? 3.9 : bn == 128 ? 2.2 : 1.4;
    const long long tiles = static_cast<long long>(cdiv(rows, 128 * cg)) * cdiv(n, bn);
    const long long units = sms / cg;
    const long long rounds = (tiles + units - 1) / units;
    const double busy = static_cast<double>(tiles < units ? tiles : units) * cg;
    const double fabric = busy * (128 + bn / cg) * 128 / 12e6;  // us a k-block at 12 TB/s
    const double round = cdiv(k, 128) * (block > fabric ? block : fabric);
    return start + round + (rounds - 1) * (round > epilogue ? round : epilogue);
}

// The same for the kernel that splits k over clusters of `split` CTAs, with the split that takes least: its
// start, the k-blocks of an SM, the tokens that a CTA joins, 8 at a time, and 3 us for every two CTAs more
// than the two that an SM holds.  (us, 8-bit rows: 24 x 4,096 x 4,096 7.5, 64 x 1,024 x 4,096 6.9,
// 100 x 1,153 x 1,000 7.1, 128 x 4,096 x 4,096 12.3, 300 x 1,024 x 4,096 10.9 against 12.9 in tiles of 64
// columns, 1,024 x 256 x 8,192 12.0 against 22.3, 300 x 4,096 x 4,096 29 against 13.5.)
double skinny_us(long long rows, int n, int k, int sms, int& nt, int& split) {
    nt = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const double start = nt <= 32 ? 3.8 : 4.8;
    const double block = nt == 16 ? 0.25 : nt == 32 ? 0.27 : nt == 64 ? 0.45 : 0.6;
    const long long tiles = static_cast<long long>(cdiv(rows, nt)) * cdiv(n, 128);
    const int num_kb = cdiv(k, 128), tokens = rows < nt ? static_cast<int>(rows) : nt;
    double best = 0;
    split = 0;
    for (int sp = 1; sp <= 8 && sp <= num_kb; sp *= 2) {
        const long long rounds = (tiles * sp + sms - 1) / sms;
        const double us = start + (rounds - 1) / 2 * 3.0 + static_cast<double>(rounds) * cdiv(num_kb, sp) * block +
                          0.8 * cdiv(tokens, 8 * sp);
        if (split == 0 || us < best) {
            best = us;
            split = sp;
        }
    }
    return best;
}

// One or two rows that fit the default shared memory of a block, and up to 4 short ones, take the
// one-launch kernel (device time with n = 4,096: 4 rows of 1,024 5.3 us against 6.3 in the other, 4 of
// 4,096 8.8 against 7.9; 8 of 1,024 9.2 against 5.6).
bool use_gemv(long long rows, int k) { return rows <= 2 ? rows * padded_k(k) <= 40960 : rows <= 4 && k <= 2048; }

template <int MR>
void launch_gemv(cudaStream_t s, const Int8LinearParams& q, int sms) {
    GemvParams p;
    p.M = static_cast<int>(q.rows);
    p.N = q.n;
    p.K = q.k;
    p.kpad = static_cast<int>(padded_k(q.k));
    p.x_dt = q.x_dt;
    p.out_dt = q.out_dt;
    p.act = q.act;
    p.x_vec = reinterpret_cast<uintptr_t>(q.x) % 16 == 0 && q.ldx * op_size(q.x_dt) % 16 == 0;
    p.ldx = q.ldx;
    p.ldw = q.ldw;
    p.ldo = q.ldo;
    p.x = q.x;
    p.x_scale = q.x_scale;
    p.w = q.w;
    p.ws = q.w_scale;
    p.bias = q.bias;
    p.out = q.out;
    const int blocks = cdiv(q.n, kGemvCols * (kGemvThreads / 32));
    const int most = 2 * sms;
    const LaunchConfig c(blocks < most ? blocks : most, kGemvThreads, MR * p.kpad, s);
    M3R_CUDA(cudaLaunchKernelEx(&c.cfg, int8_gemv_kernel<MR>, p));
}

}  // namespace

// 8-bit rows of x, then their scales.
size_t int8_linear_workspace(int x_dt, long long rows, int n, int k) {
    (void)n;
    if (x_dt == OP_I8 || rows == 0 || use_gemv(rows, k)) return 0;
    return round256(static_cast<size_t>(rows) * padded_k(k)) + round256(static_cast<size_t>(rows) * 4);
}

void int8_linear(cudaStream_t s, const Int8LinearParams& p) {
    if (p.rows == 0) return;
    const int sms = sm_count();
    if (use_gemv(p.rows, p.k)) {
        if (p.rows == 1) return launch_gemv<1>(s, p, sms);
        if (p.rows == 2) return launch_gemv<2>(s, p, sms);
        return launch_gemv<4>(s, p, sms);
    }
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
    const double big = tile_us(256, 2, p.rows, p.n, p.k, sms), mid = tile_us(128, 1, p.rows, p.n, p.k, sms),
                 low = tile_us(64, 1, p.rows, p.n, p.k, sms);
    int nt = 0, split = 0;
    if (p.rows <= 1024) {
        const double few = skinny_us(p.rows, p.n, p.k, sms, nt, split);
        if (few > big || few > mid || few > low) nt = 0;
    }
    if (nt == 16)
        launch_skinny<16>(s, p, xq, ldq, xs, split);
    else if (nt == 32)
        launch_skinny<32>(s, p, xq, ldq, xs, split);
    else if (nt == 64)
        launch_skinny<64>(s, p, xq, ldq, xs, split);
    else if (nt == 128)
        launch_skinny<128>(s, p, xq, ldq, xs, split);
    else if (big <= mid && big <= low)
        launch<256, 2>(s, p, xq, ldq, xs, sms);
    else if (mid <= low)
        launch<128, 1>(s, p, xq, ldq, xs, sms);
    else
        launch<64, 1>(s, p, xq, ldq, xs, sms);
}

int* int8_linear_status() {
    void* at = nullptr;
    M3R_CUDA(cudaGetSymbolAddress(&at, g_status));
    return &static_cast<DevStatus*>(at)->code;
}

}  // namespace m3r
