// Rotary positions: pair i of a head's front part is turned by angle = position * inv_freq[i],
//
//   (u, v) -> amplitude * (u cos - v sin, u sin + v cos)
//
// with the pair (u, v) at (i, i + n_freq) in the half layout and at (2 i, 2 i + 1) in the
// adjacent-pair layout; values behind the front part are copied.  With two position axes the
// first half of the pairs turns with axis 0, the second with axis 1 (the image tokens of
// backends/python/rope2d.py:133-146).
//
// The work is bound by HBM (each value in and out once).  A block takes a few tokens: it
// computes their sines and cosines once, in shared memory, while the first values are on
// their way, and applies them to a range of heads with 16-byte accesses.  Few registers and
// many resident blocks hide the latency (2 or 4 accesses of a thread under way at once: 140
// and 194 us instead of 130).  Angles are reduced in 64 bits -- position * (inv_freq / 2 pi)
// minus its nearest integer -- so that a far position keeps its fraction of a turn: in 32
// bits position 1e6 would leave it with 2^-5 of a radian.  The fraction itself, its sine and
// cosine and their product with the amplitude are 32-bit values: the error of 32-bit results is
// 3.1e-8 to 5.7e-8 of them (root mean square, head sizes of 32 to 256), a quarter more on
// average than with these in 64 bits (3.0e-8 to 4.2e-8).
#include <algorithm>

#include "common.cuh"
#include "launch.h"
#include "ops.h"
#include "tmap.h"

namespace m3r {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 2048;  // sines and cosines of a block: 16 KB
constexpr int kMaxTokens = 64;    // tokens of a block
constexpr int kBlocksPerSm = 6;

constexpr int kMaxHeads = 256;    // heads of a block

struct RopeGrid {
    int tokens_per_block, heads_per_block, head_blocks;
    int rot_chunks, tail_chunks;
    int cols;  // threads along a head's chunks; kThreads / cols heads at a time
};

// VE values of T, at 2 to 16 bytes an access.
template <class T, int VE>
struct alignas(sizeof(T) * VE) Pack {
    T v[VE];
};

template <class T>
__device__ __forceinline__ float get_f(T x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same<T, __half>::value)
        return __half2float(x);
    else
        return __bfloat162float(x);
}
template <class T>
__device__ __forceinline__ T put_f(float x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else
        return Elem<T>::from(x);
}

// A thread turns one chunk of a head -- VE pairs in the half layout (two accesses), VE / 2 in the
// adjacent one (one; a single pair for VE = 1) -- and copies every `rot_chunks`-th chunk of the tail, so
// that all lanes do the same.
template <class T, int VE, bool ADJ>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) rope_kernel(const __grid_constant__ RopeParams p,
                                                                     const __grid_constant__ RopeGrid g) {
    using V = Pack<T, VE>;
    constexpr int PAIRS = ADJ ? (VE > 1 ? VE / 2 : 1) : VE;  // pairs a chunk
    constexpr bool TWO = !ADJ || VE == 1;                    // a pair is split over two accesses
    __shared__ float2 turn[kMaxAngles];                      // [token][frequency]: amplitude * (cos, sin)
    __shared__ double place[kMaxTokens][2];                  // the token's position on each axis
    __shared__ long long base[kMaxTokens][4];                // its offsets in the inputs and outputs of both tensors
    __shared__ const T* from[kMaxHeads];                     // where the block's heads start
    __shared__ T* to[kMaxHeads];
    const int all = static_cast<int>(p.batch * p.tokens);
    const int tok0 = static_cast<int>(blockIdx.x / g.head_blocks) * g.tokens_per_block;
    const int head0 = static_cast<int>(blockIdx.x % g.head_blocks) * g.heads_per_block;
    const int heads = min(g.heads_per_block, p.t[0].heads + p.t[1].heads - head0);
    const int split = p.t[0].heads - head0;  // the block's heads from here on are the second tensor's
    const int ntok = min(g.tokens_per_block, all - tok0);
    const int tid = threadIdx.x;
    grid_dependency_wait();
    if (tid < 2 * ntok) {
        const int tk = tid >> 1, axis = tid & 1;
        const int b = (tok0 + tk) / static_cast<int>(p.tokens), t = tok0 + tk - b * static_cast<int>(p.tokens);
        base[tk][axis] = b * p.t[axis].xb + t * p.t[axis].xt;
        base[tk][2 + axis] = b * p.t[axis].ob + t * p.t[axis].ot;
        if (axis < p.axes) {
            const long long at = axis * p.pos_axis + b * p.pos_b + t * p.pos_t;
            place[tk][axis] = p.pos64 ? static_cast<double>(static_cast<const long long*>(p.pos)[at])
                                      : static_cast<double>(static_cast<const int*>(p.pos)[at]);
        }
    }
    for (int h = tid; h < heads; h += kThreads) {
        const RopeTensor& x = p.t[h >= split];
        const long long at = h >= split ? h - split : h + head0;
        from[h] = static_cast<const T*>(x.x) + at * x.xh;
        to[h] = static_cast<T*>(x.out) + at * x.oh;
    }
    __syncthreads();
    const int rows = kThreads / g.cols;
    const int first = tid / g.cols;
    const int step_t = rows / heads, step_h = rows - step_t * heads;
    const int pairs = first < rows ? ntok * heads : 0;
    int c = tid % g.cols, j = first, tk = first / heads, h = first - tk * heads;
    const T* src;
    V lo, hi;
    auto load = [&]() {
        src = from[h] + base[tk][h >= split];
        const T* at = src + (ADJ && VE == 1 ? 2 * c : c * VE);
        lo = *reinterpret_cast<const V*>(at);
        if (TWO) hi = *reinterpret_cast<const V*>(at + (ADJ ? 1 : p.n_freq));
    };
    bool live = j < pairs;
    if (live) load();  // travels while the sines are computed
    for (int i = tid; i < ntok * p.n_freq; i += kThreads) {
        const int k = i / p.n_freq, f = i - k * p.n_freq;
        const double turns = place[k][p.axes == 2 && f >= p.n_freq / 2] * (p.inv_freq[f] * 0.15915494309189535);  // 1 / (2 pi)
        float sn, cs;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cs);
        turn[i] = make_float2(cs * p.amplitude, sn * p.amplitude);
    }
    __syncthreads();
    while (live) {
        T* dst = to[h] + base[tk][2 + (h >= split)];
        // behind the front part
        for (int e = c; e < g.tail_chunks; e += g.rot_chunks) {
            const int at = 2 * p.n_freq + e * VE;
            *reinterpret_cast<V*>(dst + at) = *reinterpret_cast<const V*>(src + at);
        }
        const float2* w = turn + tk * p.n_freq + c * PAIRS;
        if constexpr (TWO) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float a = get_f(lo.v[i]), b = get_f(hi.v[i]);
                const float2 r = w[i];
                lo.v[i] = put_f<T>(a * r.x - b * r.y);
                hi.v[i] = put_f<T>(a * r.y + b * r.x);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) {
                const float a = get_f(lo.v[2 * i]), b = get_f(lo.v[2 * i + 1]);
                const float2 r = w[i];
                lo.v[2 * i] = put_f<T>(a * r.x - b * r.y);
                lo.v[2 * i + 1] = put_f<T>(a * r.y + b * r.x);
            }
        }
        dst += ADJ && VE == 1 ? 2 * c : c * VE;
        *reinterpret_cast<V*>(dst) = lo;
        if (TWO) *reinterpret_cast<V*>(dst + (ADJ ? 1 : p.n_freq)) = hi;
        j += rows;
        tk += step_t;
        h += step_h;
        if (h >= heads) {
            h -= heads;
            ++tk;
        }
        if (j >= pairs) {  // the next chunk, of heads with more chunks than a block has threads
            c += g.cols;
            j = first;
            tk = first / heads;
            h = first - tk * heads;
            live = c < g.rot_chunks;
        }
        if (live) load();
    }
}

template <class T, int VE, bool ADJ>
void launch(cudaStream_t s, const RopeParams& p) {
    constexpr int PAIRS = ADJ ? (VE > 1 ? VE / 2 : 1) : VE;
    const long long all = p.batch * p.tokens;
    const int heads = p.t[0].heads + p.t[1].heads;
    RopeGrid g;
    g.rot_chunks = p.n_freq / PAIRS;
    // turned in place, the tail is where it belongs
    const bool in_place = (p.t[0].heads == 0 || p.t[0].x == p.t[0].out) && (p.t[1].heads == 0 || p.t[1].x == p.t[1].out);
    g.tail_chunks = in_place ? 0 : (p.dim - 2 * p.n_freq) / VE;
    g.cols = g.rot_chunks < kThreads ? g.rot_chunks : kThreads;
    // Tokens a block: a block costs its accesses a thread and some for its start (98,304 tokens of 32
    // heads of 64, with 2, 4, 8 and 16 accesses: 148, 135, 130, 134 us); while there are few blocks, the
    // last round of them over the SMs counts whole.  With few tokens the heads are split over blocks, and
    // each computes its tokens' sines.
    const int rows = kThreads / g.cols;
    const long long slots = 148LL * kBlocksPerSm;
    const int most = static_cast<int>(std::min<long long>({kMaxTokens, kMaxAngles / p.n_freq, all}));
    g.tokens_per_block = 1;
    double best = 0;
    for (int t = 1; t <= most; ++t) {
        const long long blocks = (all + t - 1) / t;
        const double rounds = blocks >= 4 * slots ? static_cast<double>(blocks) / slots + 0.5 : (blocks + slots - 1) / slots;
        const double cost = rounds * ((t * heads + rows - 1) / rows + 0.4);
        if (t == 1 || cost < best) {
            best = cost;
            g.tokens_per_block = t;
        }
    }
    const long long token_blocks = (all + g.tokens_per_block - 1) / g.tokens_per_block;
    g.heads_per_block = heads;
    if (g.tokens_per_block == 1 && token_blocks < slots) {
        const long long split = slots / token_blocks < heads ? slots / token_blocks : heads;
        g.heads_per_block = static_cast<int>((heads + split - 1) / split);
        // at least one access for every thread
        if (g.heads_per_block < rows) g.heads_per_block = rows < heads ? rows : heads;
    }
    if (g.heads_per_block > kMaxHeads) g.heads_per_block = kMaxHeads;
    g.head_blocks = (heads + g.heads_per_block - 1) / g.heads_per_block;
    const long long grid = token_blocks * g.head_blocks;
    M3R_REQUIRE(grid <= 0x7FFFFFFFLL, "rope: too many tokens for one call");
    const LaunchConfig c(static_cast<unsigned>(grid), kThreads, 0, s);
    M3R_CUDA(cudaLaunchKernelEx(&c.cfg, rope_kernel<T, VE, ADJ>, p, g));
}

// Largest vector that the layout, the alignment and every stride allow.
template <class T>
int pick_ve(const RopeParams& p) {
    int ve = 16 / static_cast<int>(sizeof(T));
    for (; ve > 1; ve /= 2) {
        bool ok = (p.interleaved ? 2 * p.n_freq : p.n_freq) % ve == 0 && (p.dim - 2 * p.n_freq) % ve == 0;
        for (const RopeTensor& t : p.t) {
            if (t.heads == 0) continue;
            const uintptr_t bytes = sizeof(T) * ve;
            ok = ok && reinterpret_cast<uintptr_t>(t.x) % bytes == 0 && reinterpret_cast<uintptr_t>(t.out) % bytes == 0;
            for (long long st : {t.xb, t.xt, t.xh, t.ob, t.ot, t.oh}) ok = ok && st % ve == 0;
        }
        if (ok) break;
    }
    return ve;
}

template <class T, int VE>
void by_layout(cudaStream_t s, const RopeParams& p) {
    p.interleaved ? launch<T, VE, true>(s, p) : launch<T, VE, false>(s, p);
}

template <class T>
void by_vector(cudaStream_t s, const RopeParams& p) {
    const int ve = pick_ve<T>(p);
    if constexpr (sizeof(T) == 2)
        if (ve == 8) return by_layout<T, 8>(s, p);
    if (ve == 4) return by_layout<T, 4>(s, p);
    if (ve == 2) return by_layout<T, 2>(s, p);
    by_layout<T, 1>(s, p);
}

}  // namespace

void rope(cudaStream_t s, const RopeParams& p) {
    if (p.batch * p.tokens == 0) return;
    if (p.dt == OP_F32)
        by_vector<float>(s, p);
    else if (p.dt == OP_F16)
        by_vector<__half>(s, p);
    else
        by_vector<__nv_bfloat16>(s, p);
}

}  // namespace m3r
