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

// One warp per row.
__global__ void __launch_bounds__(256) lookup_kernel(const float* __restrict__ W,
                                                     const int64_t* __restrict__ idx,
                                                     float* __restrict__ out, int64_t N, int64_t D,
                                                     int64_t V, float scale) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < N; i += warps) {
        const int64_t t = idx[i];
        const bool live = t >= 0 && t < V;
        if (!live && t != -1 && lane == 0)
            report(kErrBadIndex);
        for (int64_t c = lane; c < D; c += 32)
            out[i * D + c] = live ? scale * W[t * D + c] : 0.0f;
    }
}

// ---------------------------------------------------------------- sorting --
// Stable radix sort of (token, position) by one cluster of 8 blocks, 8 bits
// a pass. Each warp owns a contiguous run of the keys: it counts its digits,
// the counts are scanned over the warps of the block and over the blocks
// (through distributed shared memory), and the warp then writes its keys in
// order. Tokens outside [0, V) become V and end up last.
constexpr int SORT_CTAS = 8;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int RADIX = 256;

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(smem_in_cta(p, rank)) : "memory");
    return v;
}

__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
    sort_kernel(const int64_t* __restrict__ idx, int64_t N, int64_t V, int passes,
                uint64_t* __restrict__ bufa, uint64_t* __restrict__ bufb,
                uint32_t* __restrict__ seen) {
    __shared__ uint32_t hist[SORT_WARPS][RADIX];
    __shared__ uint32_t total[RADIX];
    __shared__ uint32_t wsum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = cluster_ctarank();
    const int64_t nwarps = SORT_CTAS * SORT_WARPS;
    const int64_t per = ((N + nwarps - 1) / nwarps + 31) / 32 * 32;
    const int64_t lo = (static_cast<int64_t>(rank) * SORT_WARPS + warp) * per;
    const int64_t hi = min(N, lo + per);
    // bitmap of the tokens that occur
    for (int64_t i = static_cast<int64_t>(rank) * SORT_THREADS + tid; i < (V + 31) / 32;
         i += SORT_CTAS * SORT_THREADS)
        seen[i] = 0;
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
            for (int w = 0; w < SORT_WARPS; ++w) {
                const uint32_t v = hist[w][tid];
                hist[w][tid] = run;
                run += v;
            }
            total[tid] = run;
        }
        cluster_sync();
        uint32_t before = 0, all = 0, scan = 0;
        if (tid < RADIX) {
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
            if (pass == 0 && ok) {
                const uint32_t t = static_cast<uint32_t>(key >> 32), bit = 1u << (t & 31);
                if (t < V && !(__ldcg(seen + (t >> 5)) & bit))
                    atomicOr(seen + (t >> 5), bit);
            }
        }
        __threadfence();
        cluster_sync();
    }
}

// One warp per sorted position; the warp at the start of a token's run sums it.
__global__ void __launch_bounds__(256) sum_kernel(const uint64_t* __restrict__ keys, int64_t N,
                                                  const float* __restrict__ dout,
                                                  float* __restrict__ dW, int accumulate, int64_t D,
                                                  int64_t V, float scale) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); p < N; p += warps) {
        const int64_t t = static_cast<int64_t>(keys[p] >> 32);
        if (t >= V || (p && static_cast<int64_t>(keys[p - 1] >> 32) == t))
            continue;
        int64_t end = p + 1;
        while (end < N && static_cast<int64_t>(keys[end] >> 32) == t)
            ++end;
        for (int64_t c = lane; c < D; c += 32) {
            float s = 0.0f;
            for (int64_t q = p; q < end; ++q)
                s += dout[static_cast<int64_t>(keys[q] & 0xffffffffu) * D + c];
            s *= scale;
            dW[t * D + c] = accumulate ? dW[t * D + c] + s : s;
        }
    }
}

// Rows without a token.
__global__ void __launch_bounds__(256) zero_kernel(const uint32_t* __restrict__ seen,
                                                   float* __restrict__ dW, int64_t D, int64_t V) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); v < V; v += warps)
        if (!((seen[v >> 5] >> (v & 31)) & 1u))
            for (int64_t c = lane; c < D; c += 32)
                dW[v * D + c] = 0.0f;
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

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
    lookup_kernel<<<grid_for(N, 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(W, idx, out, N, D,
                                                                                 V, scale);
    return check_launch("embedding_scaled_fwd");
}

size_t ttk_embedding_scaled_bwd_workspace_size(int64_t N, int64_t D, int64_t V) {
    (void)D;
    if (N <= 0 || V <= 0)
        return 16;
    return 2 * align16(static_cast<size_t>(N) * 8) + align16(static_cast<size_t>((V + 31) / 32) * 4);
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
    char* ws = static_cast<char*>(workspace);
    const size_t kb = align16(static_cast<size_t>(N) * 8);
    uint64_t* bufa = reinterpret_cast<uint64_t*>(ws);
    uint64_t* bufb = reinterpret_cast<uint64_t*>(ws + kb);
    uint32_t* seen = reinterpret_cast<uint32_t*>(ws + 2 * kb);
    int passes = 1;
    while (passes < 4 && (V >> (8 * passes)))
        ++passes;
    sort_kernel<<<SORT_CTAS, SORT_THREADS, 0, st>>>(idx, N, V, passes, bufa, bufb, seen);
    int rc = check_launch("embedding_scaled_bwd sort");
    if (rc)
        return rc;
    const uint64_t* keys = (passes & 1) ? bufa : bufb;
    sum_kernel<<<grid_for(N, 8), 256, 0, st>>>(keys, N, dout, dW, accumulate, D, V, scale);
    rc = check_launch("embedding_scaled_bwd sum");
    if (rc || accumulate)
        return rc;
    zero_kernel<<<grid_for(V, 8), 256, 0, st>>>(seen, dW, D, V);
    return check_launch("embedding_scaled_bwd zero");
}

}  // extern "C"
