// Scaled embedding lookup and its gradient by sorted tokens.
//
//   out[i,:] = scale * W[t_i,:]            (t_i = -1: a zero row)
//   dW[v,:] (+)= scale * sum_{i: t_i = v} dout[i,:]
// The gradient sorts the positions by token, so every row of dW is written
// once, by one summation in a fixed order: no floating-point atomics.
//
// Both are bound by HBM. Lookup, 32768 x 2048 of 32000 rows: 57 us, 6.1 TB/s of
// the rows read and written. Gradient of the same with an eighth of padding, dW
// written: 99 us, 5.0 TB/s of dout read and dW written (kernel by kernel the sort
// beside the zeroing of the rows without a token 43, the sums 49, the runs that cross
// chunks 13); added to dW, without padding 118 us.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "pdl.cuh"
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
    grid_wait();
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
// (token, position) pairs in ascending order, tokens outside [0, V) as V, so
// last. Two ways:
//   rank_kernel, up to 4096 positions: every pair is packed into 32 bits, and
//     a pair's place is the number of smaller ones, counted by one warp over
//     all of them in shared memory. No step waits for another (a gradient of
//     2000 x 768 of 32000 rows: 25.4 us against 28.5 by the other, 4096 x 768:
//     30.1 against 30.9, 8192 x 768: 41 against 34).
//   radix_kernel: a stable radix sort by one cluster of 8 blocks, 8 bits a
//     pass. Each warp owns a contiguous run of the pairs: it counts its digits,
//     the counts are scanned over the warps of the block and over the blocks
//     (through distributed shared memory), and the warp writes its pairs in
//     order (24 us for 32768 positions by itself). Up to 65536 positions the
//     pairs stay in the cluster's shared memory between the passes (LOCAL):
//     through global memory the passes would wait behind the zeroing blocks'
//     writes.
// Neither needs the whole machine; when dW is written (not added to), the
// launch's other blocks meanwhile zero the rows of tokens that do not occur.
// Each owns some of the rows and marks their tokens in a bitmap of its own by
// reading all the ids (from L2), so it waits for nobody.
constexpr int SORT_CTAS = 8;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int RADIX = 256;
constexpr int64_t LOCAL_MAX = 65536;  // 2 x 64 KB of pairs a block
constexpr uint32_t BITMAP_WORDS = RADIX * SORT_WARPS;
constexpr int RANK_BITS = 12;
constexpr int64_t RANK_MAX = 1 << RANK_BITS;
constexpr int RANK_THREADS = 256;
constexpr int RANK_KEYS = 4;  // places a warp counts at once

// The rows of dW that no id names are set to zero, in groups of 32: groups z,
// z + nz, z + 2 nz, ... here (frequent tokens have low ids in most vocabularies,
// so ranges of rows would be uneven). VEC as above.
template <int VEC>
__device__ void zero_absent(const int64_t* __restrict__ idx, int64_t N, int64_t V, uint32_t z,
                            uint32_t nz, float* __restrict__ dW, int64_t D,
                            uint32_t* __restrict__ bits) {
    using T = typename Vec<VEC>::T;
    const int64_t words = D / VEC;
    const uint32_t groups = static_cast<uint32_t>((V + 31) / 32);
    const uint32_t mine = z < groups ? (groups - z + nz - 1) / nz : 0;
    const uint32_t inv = 0xffffffffu / nz;
    for (uint32_t a = 0; a < mine; a += BITMAP_WORDS) {
        const uint32_t n = min(mine - a, BITMAP_WORDS);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
            bits[i] = 0;
        __syncthreads();
        for (int64_t i0 = threadIdx.x; i0 < N; i0 += 8 * static_cast<int64_t>(blockDim.x)) {
            int64_t t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                t[j] = i0 + j * static_cast<int64_t>(blockDim.x) < N ? idx[i0 + j * blockDim.x] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // group / nz, by the reciprocal's lower bound
                const uint32_t g = static_cast<uint32_t>(t[j]) >> 5;
                uint32_t q = __umulhi(g, inv), rest = g - q * nz;
                if (rest >= nz)
                    rest -= nz, ++q;
                const uint32_t bit = 1u << (t[j] & 31);
                // frequent tokens are marked once: atomics on one word queue up
                if (t[j] >= 0 && t[j] < V && rest == z && q - a < n &&
                    !(*const_cast<volatile uint32_t*>(bits + (q - a)) & bit))
                    atomicOr(bits + (q - a), bit);
            }
        }
        __syncthreads();
        const int lane = threadIdx.x & 31;
        for (uint32_t r = threadIdx.x >> 5; r < 32 * n; r += blockDim.x >> 5) {
            const int64_t v = (static_cast<int64_t>(a + (r >> 5)) * nz + z) * 32 + (r & 31);
            if (v < V && !((bits[r >> 5] >> (r & 31)) & 1u)) {
                T* row = reinterpret_cast<T*>(dW + v * D);
#pragma unroll 4
                for (int64_t c = lane; c < words; c += 32)
                    row[c] = zero<T>();
            }
        }
    }
}

template <int VEC>
__global__ void __launch_bounds__(RANK_THREADS)
    rank_kernel(const int64_t* __restrict__ idx, int N, int64_t V, int sorters,
                uint64_t* __restrict__ keys, uint32_t* __restrict__ count, float* __restrict__ dW,
                int64_t D) {
    // the pairs, or a zeroing block's bitmap
    __shared__ __align__(16) uint32_t pairs[RANK_MAX > BITMAP_WORDS ? RANK_MAX : BITMAP_WORDS];
    grid_wait();
    if (static_cast<int>(blockIdx.x) >= sorters) {
        const uint32_t nz = gridDim.x - sorters, z = blockIdx.x - sorters;
        zero_absent<VEC>(idx, N, V, z, nz, dW, D, pairs);
        return;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *count = 0;
    for (int i = threadIdx.x; i < (N + 3) / 4 * 4; i += RANK_THREADS) {
        uint32_t p = ~0u;  // no pair: greater than all of them
        if (i < N) {
            const int64_t t = idx[i];
            const bool live = t >= 0 && t < V;
            if (!live && t != -1 && blockIdx.x == 0)
                report(kErrBadIndex);
            p = static_cast<uint32_t>(live ? t : V) << RANK_BITS | static_cast<uint32_t>(i);
        }
        pairs[i] = p;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int i0 = (blockIdx.x * (RANK_THREADS / 32) + (threadIdx.x >> 5)) * RANK_KEYS; i0 < N;
         i0 += sorters * (RANK_THREADS / 32) * RANK_KEYS) {
        uint32_t mine[RANK_KEYS];
        int below[RANK_KEYS];
#pragma unroll
        for (int k = 0; k < RANK_KEYS; ++k) {
            mine[k] = pairs[min(i0 + k, N - 1)];
            below[k] = 0;
        }
#pragma unroll 4
        for (int j = lane; j < (N + 3) / 4; j += 32) {
            const uint4 v = reinterpret_cast<const uint4*>(pairs)[j];
#pragma unroll
            for (int k = 0; k < RANK_KEYS; ++k)
                below[k] += (v.x < mine[k]) + (v.y < mine[k]) + (v.z < mine[k]) + (v.w < mine[k]);
        }
#pragma unroll
        for (int k = 0; k < RANK_KEYS; ++k) {
            const int place = __reduce_add_sync(~0u, below[k]);
            if (lane == k && i0 + k < N)
                keys[place] = static_cast<uint64_t>(mine[k] >> RANK_BITS) << 32 |
                              (mine[k] & (RANK_MAX - 1));
        }
    }
}

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(smem_in_cta(p, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void st_cluster(uint64_t* p, uint32_t rank, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(smem_in_cta(p, rank)), "l"(v) : "memory");
}

template <int VEC, bool LOCAL>
__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
    radix_kernel(const int64_t* __restrict__ idx, int64_t N, int64_t V, int passes,
                 uint64_t* __restrict__ bufa, uint64_t* __restrict__ bufb,
                 uint32_t* __restrict__ count, float* __restrict__ dW, int64_t D) {
    extern __shared__ __align__(16) uint64_t pairs[];  // LOCAL: [2][pairs of a block]
    __shared__ uint32_t hist[SORT_WARPS][RADIX];
    __shared__ uint32_t total[RADIX];
    __shared__ uint32_t wsum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_wait();
    if (blockIdx.x >= SORT_CTAS) {  // whole clusters
        const uint32_t nz = gridDim.x - SORT_CTAS, z = blockIdx.x - SORT_CTAS;
        zero_absent<VEC>(idx, N, V, z, nz, dW, D, &hist[0][0]);
        return;
    }
    const uint32_t rank = cluster_ctarank();
    if (rank == 0 && tid == 0)
        *count = 0;
    const int64_t nwarps = SORT_CTAS * SORT_WARPS;
    const int64_t per = ((N + nwarps - 1) / nwarps + 31) / 32 * 32;
    const int64_t lo = (static_cast<int64_t>(rank) * SORT_WARPS + warp) * per;
    const int64_t hi = min(N, lo + per);
    const int64_t block = per * SORT_WARPS, mine = rank * block;  // this block's pairs
    auto first = [&](int64_t i) -> uint64_t {
        const int64_t t = idx[i];
        const bool live = t >= 0 && t < V;
        if (!live && t != -1)
            report(kErrBadIndex);
        return (static_cast<uint64_t>(live ? t : V) << 32) | static_cast<uint64_t>(i);
    };
    if (LOCAL) {  // pass 0 reads the second half, as every even pass
#pragma unroll 4
        for (int64_t i = lo + lane; i < hi; i += 32)
            pairs[block + i - mine] = first(i);
        __syncwarp();
    }
    auto load = [&](int pass, int64_t i) -> uint64_t {
        if (LOCAL)
            return pairs[((pass & 1) ? 0 : block) + i - mine];
        if (pass == 0)
            return first(i);
        return __ldcg(reinterpret_cast<const unsigned long long*>((pass & 1) ? bufa : bufb) + i);
    };
    auto store = [&](int pass, uint32_t place, uint64_t key) {
        if (LOCAL && pass + 1 < passes) {
            const uint32_t to = place / static_cast<uint32_t>(block);
            st_cluster(pairs + ((pass & 1) ? block : 0) + (place - to * block), to, key);
        } else {
            ((pass & 1) ? bufb : bufa)[place] = key;
        }
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
#pragma unroll
            for (int w = 0; w < SORT_WARPS; ++w)
                hist[w][tid] += base;
        }
        __syncthreads();
        for (int64_t i = lo + lane; i - lane < hi; i += 32) {
            const bool ok = i < hi;
            const uint64_t key = ok ? load(pass, i) : 0;
            const uint32_t d = ok ? static_cast<uint32_t>(key >> shift) & 255u : 256u;
            const uint32_t same = __match_any_sync(~0u, d);
            const uint32_t below = __popc(same & ((1u << lane) - 1));
            if (ok)
                store(pass, hist[warp][d] + below, key);
            __syncwarp();
            if (ok && below == 0)
                hist[warp][d] += __popc(same);
            __syncwarp();
        }
        if (!LOCAL)
            __threadfence();
        cluster_sync();
    }
}

// ---------------------------------------------------------------- summing --
// The sorted positions are cut into chunks of L. A block sums one chunk, each
// thread one word of the row, and writes dW where a token's run ends. A run
// that crosses chunks leaves partial sums in part[chunk][0] (the chunk's
// first run, when it began earlier) and part[chunk][1] (its last run, when it
// began here and goes on), and the chunk where it began goes on the list that
// join_kernel adds up. So frequent tokens are spread over many blocks, and the
// order of every sum depends on N, D and the ids alone (that of the list does
// not matter).
constexpr int MAX_L = 64;
constexpr int DEPTH = 8;  // rows in flight per thread

__device__ __forceinline__ uint32_t key_token(uint64_t k) { return static_cast<uint32_t>(k >> 32); }

template <int VEC>
__global__ void __launch_bounds__(256)
    chunk_kernel(const uint64_t* __restrict__ keys, int64_t N, int L, const float* __restrict__ dout,
                 float* __restrict__ dW, int accumulate, int64_t D, int64_t V, float scale,
                 float* __restrict__ part, uint32_t* __restrict__ count,
                 uint2* __restrict__ list) {
    using T = typename Vec<VEC>::T;
    __shared__ uint64_t s_key[MAX_L + 2];  // the chunk's keys, its neighbours on both sides
    const int64_t first = static_cast<int64_t>(blockIdx.x) * L;
    const int n = static_cast<int>(min(static_cast<int64_t>(L), N - first));
    const uint64_t none = ~0ull;
    grid_wait();
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
                if (!earlier && c == 0)
                    list[atomicAdd(count, 1u)] = make_uint2(blockIdx.x, t);
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

// Runs that cross chunks: a block takes one listed (chunk, token) and 256 words
// of the row at a time, and adds the partial sums in two interleaved sequences
// of chunks, then those two.
constexpr int JOIN_WORDS = 256;
constexpr int JOIN_THREADS = 2 * JOIN_WORDS;
template <int VEC>
__global__ void __launch_bounds__(JOIN_THREADS)
    join_kernel(const uint64_t* __restrict__ keys, int64_t N, int L, float* __restrict__ dW,
                int accumulate, int64_t D, float scale, const float* __restrict__ part,
                const uint32_t* __restrict__ count, const uint2* __restrict__ list) {
    using T = typename Vec<VEC>::T;
    __shared__ T s_part[JOIN_WORDS];
    const int at = threadIdx.x % JOIN_WORDS, way = threadIdx.x / JOIN_WORDS;
    const int64_t words = D / VEC, tiles = (words + JOIN_WORDS - 1) / JOIN_WORDS;
    grid_wait();
    const int64_t items = static_cast<int64_t>(*count) * tiles;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint2 run = list[item / tiles];
        const int64_t chunk = run.x, c = item % tiles * JOIN_WORDS + at;
        const T* p = reinterpret_cast<const T*>(part) + c;
        T* d = reinterpret_cast<T*>(dW) + static_cast<int64_t>(run.y) * words + c;
        // on their way while the run's length is found: its first two partial
        // sums (there are two at least) and the row to add to
        T acc = zero<T>(), old = zero<T>();
        if (c < words) {
            acc = p[(2 * (chunk + way) + (way ? 0 : 1)) * words];
            if (accumulate && way == 0)
                old = *d;
        }
        int64_t more = 0;  // chunks whose first run is this token's
        int found;
        do {
            const int64_t k = (chunk + 1 + more + threadIdx.x) * L;
            found = __syncthreads_count(k < N && key_token(keys[k]) == run.y);
            more += found;
        } while (found == JOIN_THREADS);
        if (c < words)
#pragma unroll 8
            for (int64_t k = chunk + 2 + way; k <= chunk + more; k += 2)
                acc = plus(acc, p[2 * k * words]);
        if (way)
            s_part[at] = acc;
        __syncthreads();
        if (way == 0 && c < words)
            *d = plus(times(plus(acc, s_part[at]), scale), old);
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

// Clusters of the radix kernel that are resident at once, the sort's among them
// (more of them would leave some for a second round: 32768 x 2048 took 120 us
// with 16 clusters and 103 us with 14).
template <int VEC>
int resident_clusters() {
    static std::atomic<int> known[16];  // by device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 16)
        dev = 0;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n)
        return n;
    constexpr int smem = 128 * 1024;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(SORT_CTAS);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SORT_CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(radix_kernel<VEC, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, radix_kernel<VEC, true>, &cfg) != cudaSuccess || n < 2) {
        cudaGetLastError();
        n = 2;
    }
    known[dev].store(n, std::memory_order_relaxed);
    return n;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workspace: two key buffers, the list's count, the list, the partial rows.
size_t workspace_bytes(const Plan& p, int64_t D) {
    return 2 * p.keys + 16 + align16(static_cast<size_t>(p.chunks) * 8) +
           static_cast<size_t>(p.chunks) * 2 * D * sizeof(float);
}

template <int VEC>
int backward(const float* dout, const int64_t* idx, float* dW, int accumulate, int64_t N, int64_t D,
             int64_t V, float scale, char* ws, const Plan& p, cudaStream_t st) {
    uint64_t* bufa = reinterpret_cast<uint64_t*>(ws);
    uint64_t* bufb = reinterpret_cast<uint64_t*>(ws + p.keys);
    uint32_t* count = reinterpret_cast<uint32_t*>(ws + 2 * p.keys);
    uint2* list = reinterpret_cast<uint2*>(count + 4);
    float* part = reinterpret_cast<float*>(ws + 2 * p.keys + 16 +
                                           align16(static_cast<size_t>(p.chunks) * 8));
    const uint64_t* keys = bufa;
    int rc;
    if (N <= RANK_MAX && V < (1ll << (32 - RANK_BITS)) - 1) {
        const int per = RANK_THREADS / 32 * RANK_KEYS;
        const int sorters = static_cast<int>(std::min<int64_t>((N + per - 1) / per, 128));
        // 32 KB of rows a zeroing block, several blocks an SM
        const int64_t zeros = accumulate ? 0 : std::min<int64_t>(148 * 5, V * D / 8192 + 1);
        rc = launch_pdl("embedding_scaled_bwd rank", rank_kernel<VEC>,
                        dim3(static_cast<unsigned>(sorters + zeros)), RANK_THREADS, 0, st, idx,
                        static_cast<int>(N), V, sorters, bufa, count, dW, D);
    } else {
        int passes = 1;
        while (passes < 4 && (V >> (8 * passes)))
            ++passes;
        // 64 KB of rows a zeroing block at least
        const int64_t zeros = accumulate ? 0
                                         : std::min<int64_t>(resident_clusters<VEC>() - 1,
                                                             V * D / (16384 * SORT_CTAS) + 1) *
                                               SORT_CTAS;
        const dim3 grid(static_cast<unsigned>(SORT_CTAS + zeros));
        if (N <= LOCAL_MAX) {
            const int64_t per = ((N + SORT_CTAS * SORT_WARPS - 1) / (SORT_CTAS * SORT_WARPS) + 31) / 32 * 32;
            const size_t smem = static_cast<size_t>(per) * SORT_WARPS * 2 * sizeof(uint64_t);
            const cudaError_t e = cudaFuncSetAttribute(
                radix_kernel<VEC, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
            if (e != cudaSuccess)
                return check_cuda(e, "embedding_scaled_bwd sort");
            rc = launch_pdl("embedding_scaled_bwd sort", radix_kernel<VEC, true>, grid,
                            SORT_THREADS, smem, st, idx, N, V, passes, bufa, bufb, count, dW, D);
        } else {
            rc = launch_pdl("embedding_scaled_bwd sort", radix_kernel<VEC, false>, grid,
                            SORT_THREADS, 0, st, idx, N, V, passes, bufa, bufb, count, dW, D);
        }
        keys = (passes & 1) ? bufa : bufb;
    }
    if (!rc)
        rc = launch_pdl("embedding_scaled_bwd sums", chunk_kernel<VEC>,
                        dim3(static_cast<unsigned>(p.chunks), static_cast<unsigned>(p.tiles)),
                        p.threads, 0, st, keys, N, p.L, dout, dW, accumulate, D, V, scale, part,
                        count, list);
    const int64_t items = p.chunks * ((p.words + JOIN_WORDS - 1) / JOIN_WORDS);  // at most
    if (!rc)
        rc = launch_pdl("embedding_scaled_bwd join", join_kernel<VEC>,
                        dim3(static_cast<unsigned>(std::min<int64_t>(items, 148 * 4))), JOIN_THREADS,
                        0, st, keys, N, p.L, dW, accumulate, D, scale,
                        static_cast<const float*>(part), static_cast<const uint32_t*>(count),
                        static_cast<const uint2*>(list));
    return rc;
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
    return launch_pdl("embedding_scaled_fwd", vec ? lookup_kernel<4> : lookup_kernel<1>,
                      dim3(static_cast<unsigned>(blocks)), 256, 0, st, W, idx, out, N, D, V, scale,
                      pieces);
}

size_t ttk_embedding_scaled_bwd_workspace_size(int64_t N, int64_t D, int64_t V) {
    if (N <= 0 || D <= 0 || V <= 0)
        return 16;
    // for either form: the scalar one has as many tiles of the columns or more, so its
    // chunks are as long or longer, and there are no more of them
    return workspace_bytes(plan(N, D, true), D);
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
    if (p.tiles > 65535)
        return set_error(TTK_ERR_ARG, "embedding_scaled_bwd: D too large");
    char* ws = static_cast<char*>(workspace);
    return p.vec == 4
               ? backward<4>(dout, idx, dW, accumulate, N, D, V, scale, ws, p, st)
               : backward<1>(dout, idx, dW, accumulate, N, D, V, scale, ws, p, st);
}

}  // extern "C"
