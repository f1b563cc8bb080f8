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
// computes their sines and cosines once, in shared memory, and applies them to a range of
// heads with 16-byte accesses.  Angles are reduced in 64 bits -- position * (inv_freq / 2 pi)
// minus its nearest integer -- so that a far position keeps its fraction of a turn: in 32
// bits position 1e6 would leave it with 2^-5 of a radian.
#include "common.cuh"
#include "ops.h"
#include "tmap.h"

namespace m3r {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 2048;  // sines and cosines of a block: 16 KB

struct RopeGrid {
    int tokens_per_block, heads_per_block, head_blocks, head_chunks;
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

// Head chunks of one (token, head): the half layout has n_freq / VE chunks of VE pairs (two
// accesses each), the adjacent one 2 n_freq / VE of VE / 2 pairs; then the chunks of the tail.
// VE = 1 of the adjacent layout takes a pair a chunk.
template <class T, int VE, bool ADJ>
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeParams p,
                                                        const __grid_constant__ RopeGrid g) {
    __shared__ float2 turn[kMaxAngles];  // [token][frequency]: amplitude * (cos, sin)
    const long long all = p.batch * p.tokens;
    const long long tok0 = static_cast<long long>(blockIdx.x / g.head_blocks) * g.tokens_per_block;
    const int head0 = static_cast<int>(blockIdx.x % g.head_blocks) * g.heads_per_block;
    const int heads_all = p.t[0].heads + p.t[1].heads;
    const int heads = min(g.heads_per_block, heads_all - head0);
    const int ntok = static_cast<int>(min(static_cast<long long>(g.tokens_per_block), all - tok0));
    for (int i = threadIdx.x; i < ntok * p.n_freq; i += kThreads) {
        const int tk = i / p.n_freq, f = i - tk * p.n_freq;
        const long long tok = tok0 + tk, b = tok / p.tokens, t = tok - b * p.tokens;
        const int axis = p.axes == 2 && f >= p.n_freq / 2;
        const long long at = axis * p.pos_axis + b * p.pos_b + t * p.pos_t;
        const double pos = p.pos64 ? static_cast<double>(static_cast<const long long*>(p.pos)[at])
                                   : static_cast<double>(static_cast<const int*>(p.pos)[at]);
        const double turns = pos * (p.inv_freq[f] * 0.15915494309189535);  // 1 / (2 pi)
        float s, c;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
        turn[i] = make_float2(c * p.amplitude, s * p.amplitude);
    }
    __syncthreads();
    constexpr int PAIRS = ADJ ? (VE > 1 ? VE / 2 : 1) : VE;  // pairs a chunk
    const int rot_chunks = p.n_freq / PAIRS;
    const int per_tok = heads * g.head_chunks;
    for (int i = threadIdx.x; i < ntok * per_tok; i += kThreads) {
        const int tk = i / per_tok;
        const int rem = i - tk * per_tok;
        const int hh = rem / g.head_chunks, c = rem - hh * g.head_chunks;
        const long long tok = tok0 + tk, b = tok / p.tokens, t = tok - b * p.tokens;
        int h = head0 + hh;
        const RopeTensor& x = h < p.t[0].heads ? p.t[0] : p.t[1];
        if (h >= p.t[0].heads) h -= p.t[0].heads;
        const T* src = static_cast<const T*>(x.x) + b * x.xb + t * x.xt + h * x.xh;
        T* dst = static_cast<T*>(x.out) + b * x.ob + t * x.ot + h * x.oh;
        using V = Pack<T, VE>;
        if (c >= rot_chunks) {  // behind the front part
            const int e = 2 * p.n_freq + (c - rot_chunks) * VE;
            *reinterpret_cast<V*>(dst + e) = *reinterpret_cast<const V*>(src + e);
            continue;
        }
        const float2* w = turn + tk * p.n_freq + c * PAIRS;
        if constexpr (!ADJ) {
            V lo = *reinterpret_cast<const V*>(src + c * VE);
            V hi = *reinterpret_cast<const V*>(src + p.n_freq + c * VE);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float u = get_f(lo.v[j]), v = get_f(hi.v[j]);
                const float2 a = w[j];
                lo.v[j] = put_f<T>(u * a.x - v * a.y);
                hi.v[j] = put_f<T>(u * a.y + v * a.x);
            }
            *reinterpret_cast<V*>(dst + c * VE) = lo;
            *reinterpret_cast<V*>(dst + p.n_freq + c * VE) = hi;
        } else if constexpr (VE > 1) {
            V q = *reinterpret_cast<const V*>(src + c * VE);
#pragma unroll
            for (int j = 0; j < VE / 2; ++j) {
                const float u = get_f(q.v[2 * j]), v = get_f(q.v[2 * j + 1]);
                const float2 a = w[j];
                q.v[2 * j] = put_f<T>(u * a.x - v * a.y);
                q.v[2 * j + 1] = put_f<T>(u * a.y + v * a.x);
            }
            *reinterpret_cast<V*>(dst + c * VE) = q;
        } else {
            const float u = get_f(src[2 * c]), v = get_f(src[2 * c + 1]);
            const float2 a = w[0];
            dst[2 * c] = put_f<T>(u * a.x - v * a.y);
            dst[2 * c + 1] = put_f<T>(u * a.y + v * a.x);
        }
    }
}

template <class T, int VE, bool ADJ>
void launch(cudaStream_t s, const RopeParams& p) {
    constexpr int PAIRS = ADJ ? (VE > 1 ? VE / 2 : 1) : VE;
    const long long all = p.batch * p.tokens;
    const int heads = p.t[0].heads + p.t[1].heads;
    RopeGrid g;
    g.head_chunks = p.n_freq / PAIRS + (p.dim - 2 * p.n_freq) / VE;
    // tokens a block: enough for every thread to have a sine, heads split over blocks while
    // there are few tokens (each block then recomputes its tokens' sines)
    g.tokens_per_block = kMaxAngles / p.n_freq;
    if (g.tokens_per_block > 8) g.tokens_per_block = 8;
    while (g.tokens_per_block > 1 && all / g.tokens_per_block < 2 * 148) g.tokens_per_block /= 2;
    const long long token_blocks = (all + g.tokens_per_block - 1) / g.tokens_per_block;
    g.heads_per_block = heads;
    const long long want = 2 * 148;
    if (token_blocks < want) {
        long long split = want / token_blocks;
        if (split > heads) split = heads;
        g.heads_per_block = static_cast<int>((heads + split - 1) / split);
        // at least one chunk for every thread
        const int least = (kThreads + g.tokens_per_block * g.head_chunks - 1) / (g.tokens_per_block * g.head_chunks);
        if (g.heads_per_block < least) g.heads_per_block = least < heads ? least : heads;
    }
    g.head_blocks = (heads + g.heads_per_block - 1) / g.heads_per_block;
    const long long grid = token_blocks * g.head_blocks;
    M3R_REQUIRE(grid <= 0x7FFFFFFFLL, "rope: too many tokens for one call");
    rope_kernel<T, VE, ADJ><<<static_cast<unsigned>(grid), kThreads, 0, s>>>(p, g);
    M3R_CUDA(cudaGetLastError());
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
