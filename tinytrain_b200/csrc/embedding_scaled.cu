// Scaled embedding lookup and its gradient by sorted tokens.
//
//   out[i,:] = scale * W[t_i,:]            (t_i = -1: a zero row)
//   dW[v,:] (+)= scale * sum_{i: t_i = v} dout[i,:]
// The gradient sorts the positions by token, so every row of dW is written
// once, by one summation in a fixed order: no floating-point atomics.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "ttk_common.cuh"
#include "ttk_internal.h"

namespace ttk {
namespace embs {

template <int VEC>
struct Vec;
template <>
struct Vec<1> {
    using T = float;
};
template <>
struct Vec<4> {
    using T = float4;
};
template <class T>
__device__ __forceinline__ T zero();
template <>
__device__ __forceinline__ float zero<float>() { return 0.0f; }
template <>
__device__ __forceinline__ float4 zero<float4>() { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float times(float a, float s) { return a * s; }
__device__ __forceinline__ float4 times(float4 a, float s) {
    return make_float4(a.x * s, a.y * s, a.z * s, a.w * s);
}
__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ float4 plus(float4 a, float4 b) {
    return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// Rows in pieces of 128 VEC-wide words (VEC = 4 where every row is 16-byte
// aligned, else 1), one piece per warp: four independent loads per lane.
template <int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const float* __restrict__ W,
                                                     const int64_t* __restrict__ idx,
                                                     float* __restrict__ out, int64_t N, int64_t D,
                                                     int64_t V, float scale, int64_t pieces) {
    using T = typename Vec<VEC>::T;
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int64_t i = item / pieces, words = D / VEC, w0 = (item - i * pieces) * 128 + lane;
    if (i >= N)
        return;
    const int64_t t = idx[i];
    const bool live = t >= 0 && t < V;
    if (!live && t != -1 && w0 == 0)
        report(kErrBadIndex);
    const T* src = reinterpret_cast<const T*>(W + (live ? t : 0) * D);
    T* dst = reinterpret_cast<T*>(out + i * D);
    T v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v[j] = live && w0 + 32 * j < words ? __ldg(src + w0 + 32 * j) : zero<T>();
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (w0 + 32 * j < words)
            __stcs(dst + w0 + 32 * j, live ? times(v[j], scale) : v[j]);
}

// ---------------------------------------------------------------- sorting --
// Stable radix sort of (token, position) by one cluster of 8 blocks, 8 bits
// a pass. Each warp owns a contiguous run of the keys: it counts its digits,
// the counts are scanned over the warps of the block and over the blocks
// (through distributed shared memory), and the warp then writes its keys in
// order. Tokens outside [0, V) become V and end up last.
// The sort occupies 8 SMs; when dW is written (not added to), the launch's
// other clusters meanwhile zero the rows of tokens that do not occur. Each of
// their blocks owns a range of rows and marks the tokens of that range in a
// bitmap of its own by reading all the ids (from L2), so it waits for nobody.
constexpr int SORT_CTAS = 8;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int RADIX = 256;
constexpr int64_t ROWS_A_ROUND = RADIX * SORT_WARPS * 32;  // rows one bitmap covers

// Rows [v0, v1) of dW that no id names are set to zero. VEC as above.
template <int VEC>
__device__ void zero_absent(const int64_t* __restrict__ idx, int64_t N, int64_t v0, int64_t v1,
                            float* __restrict__ dW, int64_t D, uint32_t* __restrict__ bits) {
    using T = typename Vec<VEC>::T;
    const int64_t words = D / VEC;
    for (int64_t a = v0; a < v1; a += ROWS_A_ROUND) {
        const int64_t e = min(v1, a + ROWS_A_ROUND);
        __syncthreads();
        for (int64_t i = threadIdx.x; i < (e - a + 31) / 32; i += SORT_THREADS)
            bits[i] = 0;
        __syncthreads();
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < N; i += SORT_THREADS) {
            const int64_t t = idx[i];
            if (t >= a && t < e)
                atomicOr(bits + ((t - a) >> 5), 1u << ((t - a) & 31));
        }
        __syncthreads();
        const int lane = threadIdx.x & 31;
        for (int64_t v = a + (threadIdx.x >> 5); v < e; v += SORT_WARPS)
            if (!((bits[(v - a) >> 5] >> ((v - a) & 31)) & 1u)) {
                T* row = reinterpret_cast<T*>(dW + v * D);
#pragma unroll 4
                for (int64_t c = lane; c < words; c += 32)
                    row[c] = zero<T>();
            }
    }
}

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(smem_in_cta(p, rank)) : "memory");
    return v;
}

template <int VEC>
__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
    sort_kernel(const int64_t* __restrict__ idx, int64_t N, int64_t V, int passes,
                uint64_t* __restrict__ bufa, uint64_t* __restrict__ bufb, float* __restrict__ dW,
                int64_t D) {
    __shared__ uint32_t hist[SORT_WARPS][RADIX];
    __shared__ uint32_t total[RADIX];
    __shared__ uint32_t wsum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (blockIdx.x >= SORT_CTAS) {  // whole clusters
        const int64_t nz = gridDim.x - SORT_CTAS, z = blockIdx.x - SORT_CTAS;
        zero_absent<VEC>(idx, N, V * z / nz, V * (z + 1) / nz, dW, D, &hist[0][0]);
        return;
    }
    const uint32_t rank = cluster_ctarank();
    const int64_t nwarps = SORT_CTAS * SORT_WARPS;
    const int64_t per = ((N + nwarps - 1) / nwarps + 31) / 32 * 32;
    const int64_t lo = (static_cast<int64_t>(rank) * SORT_WARPS + warp) * per;
    const int64_t hi = min(N, lo + per);
    auto load = [&](int pass, int64_t i) -> uint64_t {
        if (pass == 0) {
            const int64_t t = idx[i];
            const bool live = t >= 0 && t < V;
            if (!live && t != -1)
                report(kErrBadIndex);
            return (static_cast<uint64_t>(live ? t : V) << 32) | static_cast<uint64_t>(i);
        }
        return __ldcg(reinterpret_cast<const unsigned long long*>((pass & 1) ? bufa : bufb) + i);
    };
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = 32 + 8 * pass;
        for (int i = lane; i < RADIX; i += 32)
            hist[warp][i] = 0;
        __syncwarp();
        for (int64_t i = lo + lane; i - lane < hi; i += 32) {
            const bool ok = i < hi;
            const uint32_t d = ok ? static_cast<uint32_t>(load(pass, i) >> shift) & 255u : 256u;
            const uint32_t same = __match_any_sync(~0u, d);
            if (ok && (same & ((1u << lane) - 1)) == 0)
                hist[warp][d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        uint32_t run = 0;
        if (tid < RADIX) {
            uint32_t n[SORT_WARPS];
#pragma unroll
            for (int w = 0; w < SORT_WARPS; ++w)
                n[w] = hist[w][tid];
#pragma unroll
            for (int w = 0; w < SORT_WARPS; ++w) {
                hist[w][tid] = run;
                run += n[w];
            }
            total[tid] = run;
        }
        cluster_sync();
        uint32_t before = 0, all = 0, scan = 0;
        if (tid < RADIX) {
#pragma unroll
            for (uint32_t c = 0; c < SORT_CTAS; ++c) {
                const uint32_t v = ld_cluster(&total[tid], c);
                before += c < rank ? v : 0u;
                all += v;
            }
            scan = all;  // inclusive scan over the digits
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(~0u, scan, o);
                scan += lane >= o ? v : 0u;
            }
            if (lane == 31)
                wsum[warp] = scan;
        }
        __syncthreads();
        if (tid < RADIX) {
            uint32_t base = scan - all + before;
            for (int w = 0; w < warp; ++w)
                base += wsum[w];
            for (int w = 0; w < SORT_WARPS; ++w)
                hist[w][tid] += base;
        }
        __syncthreads();
        uint64_t* dst = (pass & 1) ? bufb : bufa;
        for (int64_t i = lo + lane; i - lane < hi; i += 32) {
            const bool ok = i < hi;
            const uint64_t key = ok ? load(pass, i) : 0;
            const uint32_t d = ok ? static_cast<uint32_t>(key >> shift) & 255u : 256u;
            const uint32_t same = __match_any_sync(~0u, d);
            const uint32_t below = __popc(same & ((1u << lane) - 1));
            if (ok)
                dst[hist[warp][d] + below] = key;
            __syncwarp();
            if (ok && below == 0)
                hist[warp][d] += __popc(same);
            __syncwarp();
        }
        __threadfence();
        cluster_sync();
    }
}

// ---------------------------------------------------------------- summing --
// The sorted positions are cut into chunks of L. A block sums one chunk, each
// thread one word of the row, and writes dW where a token's run ends. A run
// that crosses chunks leaves partial sums in part[chunk][0] (the chunk's
// first run, when it began earlier) and part[chunk][1] (its last run, when it
// began here and goes on); join_kernel adds those. So frequent tokens are
// spread over many blocks, and the order of every sum depends on N, D and the
// ids alone.
constexpr int MAX_L = 64;
constexpr int DEPTH = 8;  // rows in flight per thread

__device__ __forceinline__ uint32_t key_token(uint64_t k) { return static_cast<uint32_t>(k >> 32); }

template <int VEC>
__global__ void __launch_bounds__(256)
    chunk_kernel(const uint64_t* __restrict__ keys, int64_t N, int L, const float* __restrict__ dout,
                 float* __restrict__ dW, int accumulate, int64_t D, int64_t V, float scale,
                 float* __restrict__ part) {
    using T = typename Vec<VEC>::T;
    __shared__ uint64_t s_key[MAX_L + 2];  // the chunk's keys, its neighbours on both sides
    const int64_t first = static_cast<int64_t>(blockIdx.x) * L;
    const int n = static_cast<int>(min(static_cast<int64_t>(L), N - first));
    const uint64_t none = ~0ull;
    for (int i = threadIdx.x; i < n + 2; i += blockDim.x) {
        const int64_t p = first + i - 1;
        s_key[i] = p >= 0 && p < N ? keys[p] : none;
    }
    __syncthreads();
    const int64_t words = D / VEC;
    const int64_t c = static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x;
    if (c >= words)
        return;
    const uint64_t* key = s_key + 1;
    T* slots = reinterpret_cast<T*>(part) + static_cast<int64_t>(blockIdx.x) * 2 * words + c;
    T acc = zero<T>();
    int start = 0;  // of the current run
    for (int q0 = 0; q0 < n; q0 += DEPTH) {
        T v[DEPTH];
#pragma unroll
        for (int j = 0; j < DEPTH; ++j)
            v[j] = q0 + j < n && key_token(key[q0 + j]) < V
                       ? __ldcs(reinterpret_cast<const T*>(dout) +
                                static_cast<int64_t>(static_cast<uint32_t>(key[q0 + j])) * words + c)
                       : zero<T>();
#pragma unroll
        for (int j = 0; j < DEPTH; ++j) {
            const int q = q0 + j;
            if (q >= n)
                break;
            const uint32_t t = key_token(key[q]);
            if (t >= V)  // padding: nothing follows
                return;
            acc = plus(acc, v[j]);
            const bool more = key_token(key[q + 1]) == t;
            if (more && q + 1 < n)
                continue;
            const bool earlier = start == 0 && key_token(key[-1]) == t;
            if (earlier || more) {
                slots[earlier ? 0 : words] = acc;
            } else {
                T* d = reinterpret_cast<T*>(dW) + static_cast<int64_t>(t) * words + c;
                const T r = times(acc, scale);
                *d = accumulate ? plus(*d, r) : r;
            }
            acc = zero<T>();
            start = q + 1;
        }
    }
}

// One block per chunk and 32 words of the row: where a run begins in this
// chunk and goes on, its partial sums, eight interleaved sequences of chunks
// added in order.
constexpr int JOIN_WAYS = 8;
template <int VEC>
__global__ void __launch_bounds__(32 * JOIN_WAYS)
    join_kernel(const uint64_t* __restrict__ keys, int64_t N, int L, float* __restrict__ dW,
                int accumulate, int64_t D, int64_t V, float scale, const float* __restrict__ part) {
    using T = typename Vec<VEC>::T;
    __shared__ T s_part[JOIN_WAYS][32];
    const int lane = threadIdx.x & 31, way = threadIdx.x >> 5;
    const int64_t chunk = blockIdx.x, last = (chunk + 1) * L - 1;
    if (last + 1 >= N)
        return;
    const uint32_t t = key_token(keys[last]);
    if (t >= V || key_token(keys[last + 1]) != t ||
        (key_token(keys[chunk * L]) == t && chunk && key_token(keys[chunk * L - 1]) == t))
        return;
    const int64_t words = D / VEC, c = static_cast<int64_t>(blockIdx.y) * 32 + lane;
    const T* p = reinterpret_cast<const T*>(part) + c;
    T acc = zero<T>();
    if (c < words) {
        if (way == 0)
            acc = p[(2 * chunk + 1) * words];
        // chunk k's first run is this token's while position k L is
#pragma unroll 4
        for (int64_t k = chunk + 1 + way; k * L < N && key_token(keys[k * L]) == t; k += JOIN_WAYS)
            acc = plus(acc, p[2 * k * words]);
    }
    s_part[way][lane] = acc;
    __syncthreads();
    if (way == 0 && c < words) {
        for (int i = 1; i < JOIN_WAYS; ++i)
            acc = plus(acc, s_part[i][lane]);
        T* d = reinterpret_cast<T*>(dW) + static_cast<int64_t>(t) * words + c;
        const T r = times(acc, scale);
        *d = accumulate ? plus(*d, r) : r;
    }
}

struct Plan {
    int vec, threads, tiles, L;
    int64_t words, chunks;
    size_t keys;  // bytes of one key buffer
};

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

// Chunks as long as still give every SM a few blocks: a longer chunk leaves
// fewer partial rows to write and read again (each up to 2 D of L D words).
Plan plan(int64_t N, int64_t D, bool aligned) {
    Plan p;
    p.vec = aligned && D % 4 == 0 ? 4 : 1;
    p.words = D / p.vec;
    p.threads = static_cast<int>(std::min<int64_t>(256, (p.words + 31) / 32 * 32));
    p.tiles = static_cast<int>((p.words + p.threads - 1) / p.threads);
    p.L = MAX_L;
    while (p.L > 8 && (N + p.L - 1) / p.L * p.tiles < 148 * 6)
        p.L /= 2;
    p.chunks = (N + p.L - 1) / p.L;
    p.keys = align16(static_cast<size_t>(N) * 8);
    return p;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int VEC>
int backward(const float* dout, const int64_t* idx, float* dW, int accumulate, int64_t N, int64_t D,
             int64_t V, float scale, char* ws, const Plan& p, cudaStream_t st) {
    uint64_t* bufa = reinterpret_cast<uint64_t*>(ws);
    uint64_t* bufb = reinterpret_cast<uint64_t*>(ws + p.keys);
    float* part = reinterpret_cast<float*>(ws + 2 * p.keys);
    int passes = 1;
    while (passes < 4 && (V >> (8 * passes)))
        ++passes;
    // blocks that zero: at least 64 KB each, all clusters resident at once
    const int64_t zero_ctas =
        accumulate ? 0 : std::min<int64_t>(16, (V * D / (16384 * SORT_CTAS)) + 1) * SORT_CTAS;
    sort_kernel<VEC><<<static_cast<int>(SORT_CTAS + zero_ctas), SORT_THREADS, 0, st>>>(
        idx, N, V, passes, bufa, bufb, dW, D);
    int rc = check_launch("embedding_scaled_bwd sort");
    if (rc)
        return rc;
    const uint64_t* keys = (passes & 1) ? bufa : bufb;
    chunk_kernel<VEC><<<dim3(static_cast<unsigned>(p.chunks), static_cast<unsigned>(p.tiles)),
                        p.threads, 0, st>>>(keys, N, p.L, dout, dW, accumulate, D, V, scale, part);
    rc = check_launch("embedding_scaled_bwd sums");
    if (rc)
        return rc;
    join_kernel<VEC><<<dim3(static_cast<unsigned>(p.chunks),
                            static_cast<unsigned>((p.words + 31) / 32)),
                       32 * JOIN_WAYS, 0, st>>>(keys, N, p.L, dW, accumulate, D, V, scale, part);
    return check_launch("embedding_scaled_bwd join");
}

}  // namespace embs
}  // namespace ttk

using namespace ttk;
using namespace ttk::embs;

extern "C" {

int ttk_embedding_scaled_fwd(const float* W, const int64_t* idx, float* out, int64_t N, int64_t D,
                             int64_t V, float scale, void* stream) {
    if (N < 0 || D <= 0 || V <= 0 || (N && (!W || !idx || !out)))
        return set_error(TTK_ERR_ARG, "embedding_scaled_fwd: bad arguments");
    if (!N)
        return TTK_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = D % 4 == 0 && aligned16(W) && aligned16(out);
    const int64_t pieces = ((vec ? D / 4 : D) + 127) / 128, blocks = (N * pieces + 7) / 8;
    if (blocks > INT32_MAX)
        return set_error(TTK_ERR_ARG, "embedding_scaled_fwd: N * D too large");
    if (vec)
        lookup_kernel<4><<<static_cast<int>(blocks), 256, 0, st>>>(W, idx, out, N, D, V, scale, pieces);
    else
        lookup_kernel<1><<<static_cast<int>(blocks), 256, 0, st>>>(W, idx, out, N, D, V, scale, pieces);
    return check_launch("embedding_scaled_fwd");
}

size_t ttk_embedding_scaled_bwd_workspace_size(int64_t N, int64_t D, int64_t V) {
    if (N <= 0 || D <= 0 || V <= 0)
        return 16;
    // the scalar form's plan can have shorter chunks than the vector form's
    const Plan p = plan(N, D, true), q = plan(N, D, false);
    return 2 * p.keys + static_cast<size_t>(std::max(p.chunks, q.chunks)) * 2 * D * sizeof(float);
}

int ttk_embedding_scaled_bwd(const float* dout, const int64_t* idx, float* dW, int accumulate,
                             int64_t N, int64_t D, int64_t V, float scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
    if (N < 0 || D <= 0 || V <= 0 || !dW || (N && (!dout || !idx)))
        return set_error(TTK_ERR_ARG, "embedding_scaled_bwd: bad arguments");
    if (N > INT32_MAX || V >= INT32_MAX)
        return set_error(TTK_ERR_ARG, "embedding_scaled_bwd: N or V too large");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!N)
        return accumulate ? TTK_OK
                          : check_cuda(cudaMemsetAsync(dW, 0, static_cast<size_t>(V) * D * 4, st),
                                       "embedding_scaled_bwd: zero");
    if (!workspace || workspace_bytes < ttk_embedding_scaled_bwd_workspace_size(N, D, V) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15))
        return set_error(TTK_ERR_ARG,
                         "embedding_scaled_bwd: workspace too small or not 16-byte aligned");
    const Plan p = plan(N, D, aligned16(dout) && aligned16(dW));
    if (p.tiles > 65535 || (p.words + 31) / 32 > 65535)
        return set_error(TTK_ERR_ARG, "embedding_scaled_bwd: D too large");
    char* ws = static_cast<char*>(workspace);
    return p.vec == 4
               ? backward<4>(dout, idx, dW, accumulate, N, D, V, scale, ws, p, st)
               : backward<1>(dout, idx, dW, accumulate, N, D, V, scale, ws, p, st);
}

}  // extern "C"
