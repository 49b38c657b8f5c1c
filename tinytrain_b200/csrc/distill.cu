// Distillation loss on a teacher's top logits, with its gradient.
//
// Per row, with x the student's logits over C classes, (id_k, z_k) the
// teacher's list and T the temperature:
//   p = softmax(z / T) over the list,  q_T = softmax(x / T),  q_1 = softmax(x)
//   KD = sum_k p_k (log p_k - log q_T[id_k]),   CE = -log q_1[target]
//   L  = grad_scale * sum_rows w (alpha T^2 KD + (1 - alpha) CE)
//   dx = grad_scale * w (alpha T (q_T - P) + (1 - alpha)(q_1 - onehot))
// where P spreads p over the classes.
//
// Bound by HBM: the logits are read once and the gradient written once, 8
// bytes per logit. A cluster of CTAs shares a row and each thread keeps its
// part, up to 32 logits, in registers between the two: 64 registers a thread,
// so an SM holds 128 KB of rows, and with several clusters resident the reads
// of some rows overlap the exponentials and writes of others. A row of more
// than 8 x 16384 logits goes through the registers in tiles, and its gradient
// pass reads it again (from L2). The CTAs' maxima and sums meet in
// distributed shared memory. Warp 0 of each CTA works out the teacher's list
// while the row is on its way; the listed classes of a CTA's part are written
// once more at the end, with the teacher's and the label's terms.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "pdl.cuh"
#include "ttk_common.cuh"
#include "ttk_internal.h"

namespace ttk {
namespace distill {

constexpr int MAX_THREADS = 512;
constexpr int WORDS = 8;     // float4 words of a row per thread
constexpr int MAX_CTAS = 8;  // of a cluster (the portable limit)
constexpr int MAX_K = 1024;  // entries of one teacher list
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const float* logits;
    int64_t ld;
    const int32_t* ids;
    const void* top;
    int top_type;
    int64_t K;
    const int64_t* targets;
    const float* row_weight;
    int64_t N, C;
    float alpha, temperature, grad_scale;
    double* terms;  // [N][2]: w * KD, w * CE of each row
    float* dlogits;
    int64_t ldd;
};

__device__ __forceinline__ float load_top(const void* p, int type, int64_t i) {
    if (type == TTK_F32)
        return static_cast<const float*>(p)[i];
    if (type == TTK_BF16)
        return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

// exp((x - m) * c / log2 e) for c = log2 e / T. The difference is taken
// first: it is exact near the maximum, where the terms that count are.
__device__ __forceinline__ float exp_from(float x, float m, float c) {
    return exp2_approx((x - m) * c);
}

// (maximum, sum at temperature 1, sum at T) of part of a row.
struct Stat {
    float m, s1, sT;
};

// The statistics held by the lanes of a warp, as one, in every lane.
__device__ __forceinline__ Stat warp_merge(const Stat& a, float cT) {
    Stat r;
    r.m = warp_max(a.m);
    const float z = r.m == -INFINITY ? 0.0f : r.m;
    r.s1 = warp_sum(a.s1 * exp_from(a.m, z, LOG2E));
    r.sT = warp_sum(a.sT * exp_from(a.m, z, cT));
    return r;
}

__device__ __forceinline__ Stat load_stat(const Stat* p, uint32_t rank) {
    const uint32_t addr = smem_in_cta(p, rank);
    Stat r;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.m) : "r"(addr) : "memory");
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.s1) : "r"(addr + 4) : "memory");
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.sT) : "r"(addr + 8) : "memory");
    return r;
}

__device__ __forceinline__ void store_cluster(double* p, uint32_t rank, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(smem_in_cta(p, rank)), "d"(v) : "memory");
}

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// TWO: both temperatures' sums are needed; otherwise T alone (T = 1, or no
// labels). The row is cut into 16-byte words from the boundary at or before
// its start: `off` floats of the first word belong to the row before.
template <bool TWO>
__global__ void __launch_bounds__(MAX_THREADS, 2) row_kernel(const Args a, const int ctas) {
    extern __shared__ float dyn[];
    __shared__ Stat s_warp[MAX_THREADS / 32];
    __shared__ Stat s_cta;
    __shared__ float s_flags[2];         // list has entries, label in range
    __shared__ double s_kd[MAX_CTAS];    // in the cluster's first CTA
    __shared__ double s_ce[MAX_CTAS];
    const int C = static_cast<int>(a.C), K = static_cast<int>(a.K), pad = (K + 4) / 4 * 4;
    int* const s_id = reinterpret_cast<int*>(dyn);  // [K + 1]: -1 where not in this CTA's part
    float* const s_p = dyn + pad;                   // probability; gradient of the label
    float* const s_a = dyn + 2 * pad;               // log p
    float* const s_x = dyn + 3 * pad;               // the student's logit
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, T = blockDim.x;
    const uint32_t rank = cluster_ctarank();
    const float cT = LOG2E / a.temperature, invT = 1.0f / a.temperature;
    grid_wait();
    for (int64_t row = blockIdx.x / ctas; row < a.N; row += gridDim.x / ctas) {
        const float* const xr = a.logits + row * a.ld;
        float* const dr = a.dlogits ? a.dlogits + row * a.ldd : nullptr;
        const float w = a.row_weight ? a.row_weight[row] : 1.0f;
        const int off = static_cast<int>((reinterpret_cast<uintptr_t>(xr) & 15) >> 2);
        const int words = (off + C + 3) / 4, part = (words + ctas - 1) / ctas;
        const int w0 = static_cast<int>(rank) * part, w1 = min(words, w0 + part);
        // gradient words are aligned as the logits' are
        const bool same = ((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(dr)) & 15) == 0;
        auto store = [&](int wd, const float (&g)[4]) {
            const int c = 4 * wd - off;
            if (same && c >= 0 && c + 4 <= C) {
                *reinterpret_cast<float4*>(dr + c) = make_float4(g[0], g[1], g[2], g[3]);
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (c + u >= 0 && c + u < C)
                        dr[c + u] = g[u];
            }
        };
        const float zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (w == 0.0f) {  // masked row: its logits are not looked at
            if (dr)
                for (int wd = w0 + tid; wd < w1; wd += T)
                    store(wd, zeros);
            if (rank == 0 && tid == 0)
                a.terms[2 * row] = a.terms[2 * row + 1] = 0.0;
            continue;
        }
        // The row's part, tile by tile; the last tile stays in x.
        const int per = T * WORDS, tiles = (part + per - 1) / per;
        float x[4 * WORDS];
        auto load = [&](int tile) {
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                const int wd = w0 + tile * per + j * T + tid, c = 4 * wd - off;
                float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (wd < w1) {
                    if (c >= 0 && c + 4 <= C) {
                        v = *reinterpret_cast<const float4*>(xr + c);
                    } else {
                        if (c >= 0)
                            v.x = xr[c];
                        if (c + 1 >= 0 && c + 1 < C)
                            v.y = xr[c + 1];
                        if (c + 2 >= 0 && c + 2 < C)
                            v.z = xr[c + 2];
                        if (c + 3 < C)
                            v.w = xr[c + 3];
                    }
                }
                x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
            }
        };
        load(0);
        if (warp == 0) {
            // The teacher's list. NaN counts as present: it has to reach the
            // row's result.
            float zmax = -INFINITY;
            for (int k = lane; k < K; k += 32) {
                const int id = a.ids[row * a.K + k];
                const bool ok = id >= 0 && id < C;
                if (!ok && id != -1 && rank == 0)
                    report(kErrBadIndex);
                const float z = ok ? load_top(a.top, a.top_type, row * a.K + k) * invT : -INFINITY;
                const int wd = ok ? (id + off) >> 2 : -1;
                const bool here = wd >= w0 && wd < w1;
                s_id[k] = here ? id : -1;
                s_a[k] = z;
                s_x[k] = here ? xr[id] : 0.0f;
                zmax = fmaxf(zmax, z != z ? INFINITY : z);
            }
            zmax = warp_max(zmax);
            const bool has = zmax > -INFINITY;
            float sz = 0.0f;
            if (has)
                for (int k = lane; k < K; k += 32)
                    sz += expf(s_a[k] - zmax);
            sz = warp_sum(sz);
            const float logz = logf(sz), invz = 1.0f / sz;
            for (int k = lane; k < K; k += 32) {
                s_p[k] = has ? expf(s_a[k] - zmax) * invz : 0.0f;
                s_a[k] = has ? (s_a[k] - zmax) - logz : 0.0f;
            }
            if (lane == 0) {
                const int64_t t = a.targets ? a.targets[row] : -1;
                const bool ok = t >= 0 && t < C;
                if (!ok && t != -1 && rank == 0)
                    report(kErrBadIndex);
                const int wd = ok ? (static_cast<int>(t) + off) >> 2 : -1;
                const bool here = wd >= w0 && wd < w1;
                s_id[K] = here ? static_cast<int>(t) : -1;
                s_x[K] = here ? xr[t] : 0.0f;
                s_flags[0] = has ? 1.0f : 0.0f;
                s_flags[1] = ok ? 1.0f : 0.0f;
            }
            __syncwarp();
        }
        // Statistics: the warp's maximum first, so that the sums need no
        // rescaling but between tiles.
        Stat st{-INFINITY, 0.0f, 0.0f};
        for (int tile = 0;;) {
            float m = x[0];
#pragma unroll
            for (int i = 1; i + 1 < 4 * WORDS; i += 2)
                m = max3(m, x[i], x[i + 1]);
            m = warp_max(fmaxf(m, x[4 * WORDS - 1]));
            m = fmaxf(st.m, m);
            const float z = m == -INFINITY ? 0.0f : m;  // -inf - -inf would be NaN
            if (tile) {
                st.s1 *= exp_from(st.m, z, LOG2E);
                st.sT *= exp_from(st.m, z, cT);
            }
#pragma unroll
            for (int i = 0; i < 4 * WORDS; ++i) {
                if constexpr (TWO)
                    st.s1 += exp_from(x[i], z, LOG2E);
                st.sT += exp_from(x[i], z, cT);
            }
            st.m = m;
            if (++tile >= tiles)
                break;
            load(tile);
        }
        if constexpr (!TWO)
            st.s1 = st.sT;
        st.s1 = warp_sum(st.s1);
        st.sT = warp_sum(st.sT);
        if (lane == 0)
            s_warp[warp] = st;
        __syncthreads();
        const Stat none{-INFINITY, 0.0f, 0.0f};
        st = warp_merge(lane < (T >> 5) ? s_warp[lane] : none, cT);
        if (ctas > 1) {
            if (tid == 0)
                s_cta = st;
            cluster_arrive();
            cluster_wait();
            st = warp_merge(lane < ctas ? load_stat(&s_cta, lane) : none, cT);
        }
        const bool has = s_flags[0] != 0.0f, t_ok = s_flags[1] != 0.0f;
        const float m = st.m, logT = logf(st.sT);
        const float gs = a.grad_scale * w;
        const float gT = has ? gs * a.alpha * a.temperature : 0.0f;
        const float g1 = t_ok ? gs * (1.0f - a.alpha) : 0.0f;
        if (warp == 0) {  // this CTA's share of the loss, to the cluster's first CTA
            double kd = 0.0;
            for (int k = lane; k < K; k += 32)
                if (s_id[k] >= 0 && s_p[k] != 0.0f)
                    kd += static_cast<double>(s_p[k] * (s_a[k] - ((s_x[k] - m) * invT - logT)));
            kd = warp_sum_d(kd);
            if (lane == 0) {
                const double ce = s_id[K] >= 0 ? static_cast<double>(logf(st.s1) + (m - s_x[K])) : 0.0;
                if (ctas > 1) {
                    store_cluster(s_kd + rank, 0, kd);
                    store_cluster(s_ce + rank, 0, ce);
                } else {
                    a.terms[2 * row] = w * kd;
                    a.terms[2 * row + 1] = w * ce;
                }
            }
            __syncwarp();
        }
        if (ctas > 1)
            cluster_arrive();
        const float k1 = t_ok ? g1 / st.s1 : 0.0f, kT = has ? gT / st.sT : 0.0f;
        const bool use1 = TWO && k1 != 0.0f, useT = !TWO || kT != 0.0f;
        const float kk = TWO ? kT : (t_ok ? k1 : 0.0f) + kT;  // one temperature: one term
        auto base = [&](float v) {
            float g = useT ? kk * exp_from(v, m, cT) : 0.0f;
            if (use1)
                g += k1 * exp_from(v, m, LOG2E);
            return g;
        };
        if (dr) {
            for (int tile = tiles - 1;;) {
#pragma unroll
                for (int j = 0; j < WORDS; ++j) {
                    const int wd = w0 + tile * per + j * T + tid;
                    float g[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (has || t_ok)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            g[u] = base(x[4 * j + u]);
                    if (wd < w1)
                        store(wd, g);
                }
                if (--tile < 0)
                    break;
                load(tile);
            }
            __syncthreads();
            // The listed classes: the first entry of a class carries all of
            // its entries, in list order, then the label.
            for (int k = tid; k <= K; k += T) {
                const int id = s_id[k];
                if (id < 0)
                    continue;
                bool first = true;
                float sum = 0.0f;
                for (int j = 0; j < K; ++j)
                    if (s_id[j] == id) {
                        first = first && j >= k;
                        sum += s_p[j];
                    }
                if (first)
                    dr[id] = base(s_x[k]) - (gT * sum + (s_id[K] == id ? g1 : 0.0f));
            }
        }
        if (ctas > 1) {
            cluster_wait();
            if (rank == 0 && tid == 0) {
                double kd = 0.0, ce = 0.0;
                for (int i = 0; i < ctas; ++i)
                    kd += s_kd[i], ce += s_ce[i];
                a.terms[2 * row] = w * kd;
                a.terms[2 * row + 1] = w * ce;
            }
        }
        if (row + gridDim.x / ctas < a.N) {  // shared memory is free for the next row
            __syncthreads();
            if (ctas > 1) {
                cluster_arrive();
                cluster_wait();
            }
        }
    }
}

// loss = grad_scale * {alpha T^2 KD + (1 - alpha) CE, KD, CE} summed over the
// rows' terms in a fixed order.
__global__ void __launch_bounds__(1024) distill_sum_kernel(const double* __restrict__ terms,
                                                           int64_t N, float alpha, float temperature,
                                                           float grad_scale,
                                                           float* __restrict__ loss) {
    __shared__ double red[2][32];
    double kd = 0.0, ce = 0.0;
    grid_wait();
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < N; i += blockDim.x) {
        const double2 t = reinterpret_cast<const double2*>(terms)[i];
        kd += t.x;
        ce += t.y;
    }
    kd = warp_sum_d(kd);
    ce = warp_sum_d(ce);
    if ((threadIdx.x & 31) == 0) {
        red[0][threadIdx.x >> 5] = kd;
        red[1][threadIdx.x >> 5] = ce;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        kd = ce = 0.0;
        for (int i = 0; i < 32; ++i)
            kd += red[0][i], ce += red[1][i];
        kd *= grad_scale;
        ce *= grad_scale;
        const double a = alpha, t = temperature;
        loss[0] = static_cast<float>((a > 0.0 ? a * t * t * kd : 0.0) +
                                     (a < 1.0 ? (1.0 - a) * ce : 0.0));
        loss[1] = static_cast<float>(kd);
        loss[2] = static_cast<float>(ce);
    }
}

// As few CTAs to a row as hold it in registers; more, of at least 2048 logits
// each, while the rows do not fill the machine.
template <bool TWO>
int launch_rows(const Args& a, cudaStream_t st) {
    const int64_t words = (a.C + 6) / 4, cap = static_cast<int64_t>(MAX_THREADS) * WORDS;
    int ctas = static_cast<int>(std::min<int64_t>(MAX_CTAS, (words + cap - 1) / cap));
    while (ctas * 2 <= MAX_CTAS && a.N * ctas * 2 <= 148 * 8 && words / (ctas * 2) >= 512)
        ctas *= 2;
    const int64_t part = (words + ctas - 1) / ctas;
    const int threads = static_cast<int>(
        std::min<int64_t>(MAX_THREADS, ((part + WORDS - 1) / WORDS + 31) / 32 * 32));
    const int64_t rows = std::min<int64_t>(a.N, (1 << 30) / ctas);
    const size_t smem = static_cast<size_t>((a.K + 4) / 4 * 4) * 4 * sizeof(float);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, row_kernel<TWO>, a, ctas);
    const int rc = check_launch("distill_loss");
    return rc ? rc : check_cuda(e, "distill_loss");
}

}  // namespace distill
}  // namespace ttk

using namespace ttk;
using namespace ttk::distill;

extern "C" {

size_t ttk_distill_loss_workspace_size(int64_t N) {
    return static_cast<size_t>(std::max<int64_t>(N, 0)) * 2 * sizeof(double);
}

int ttk_distill_loss(const float* logits, int64_t ld, const int32_t* teacher_ids,
                     const void* teacher_logits, int teacher_type, int64_t K,
                     const int64_t* targets, const float* row_weight, int64_t N, int64_t C,
                     float alpha, float temperature, float grad_scale, float* loss, float* dlogits,
                     int64_t ldd, void* workspace, size_t workspace_bytes, void* stream) {
    if (N < 0 || C <= 0 || C > (1 << 30) || K < 0 || !loss || (N && !logits))
        return set_error(TTK_ERR_ARG, "distill_loss: bad arguments");
    if (ld < C || (dlogits && ldd < C))
        return set_error(TTK_ERR_ARG, "distill_loss: a row stride is shorter than the row");
    if (K > MAX_K)
        return set_error(TTK_ERR_ARG, "distill_loss: at most 1024 teacher entries per row");
    if (N && K && (!teacher_ids || !teacher_logits))
        return set_error(TTK_ERR_ARG, "distill_loss: null teacher list");
    if (teacher_type != TTK_F32 && teacher_type != TTK_BF16 && teacher_type != TTK_F16)
        return set_error(TTK_ERR_ARG, "distill_loss: unknown teacher type");
    if (!(alpha >= 0.0f && alpha <= 1.0f))
        return set_error(TTK_ERR_ARG, "distill_loss: alpha must be in [0, 1]");
    if (!(temperature >= FLT_MIN) || std::isinf(temperature))
        return set_error(TTK_ERR_ARG, "distill_loss: temperature must be positive and finite");
    if (dlogits == logits && dlogits && ldd != ld)
        return set_error(TTK_ERR_ARG, "distill_loss: in place needs equal row strides");
    if (N && (!workspace || workspace_bytes < ttk_distill_loss_workspace_size(N)))
        return set_error(TTK_ERR_ARG, "distill_loss: workspace too small");
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return set_error(TTK_ERR_ARG, "distill_loss: workspace must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* terms = static_cast<double*>(workspace);
    if (N) {
        const Args a{logits, ld, teacher_ids, teacher_logits, teacher_type, K, targets, row_weight,
                     N, C, alpha, temperature, grad_scale, terms, dlogits, ldd};
        const bool two = temperature != 1.0f && targets;
        const int rc = two ? launch_rows<true>(a, st) : launch_rows<false>(a, st);
        if (rc)
            return rc;
    }
    return launch_pdl("distill_loss sum", distill_sum_kernel, dim3(1), 1024, 0, st,
                      static_cast<const double*>(terms), N, alpha, temperature, grad_scale, loss);
}

}  // extern "C"
