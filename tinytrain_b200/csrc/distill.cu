// Distillation loss on a teacher's top logits, with its gradient.
//
// Per row, with x the student's logits over C classes, (id_k, z_k) the
// teacher's list and T the temperature:
//   p = softmax(z / T) over the list,  q_T = softmax(x / T),  q_1 = softmax(x)
//   KD = sum_k p_k (log p_k - log q_T[id_k]),   CE = -log q_1[target]
//   L  = grad_scale * sum_rows w (alpha T^2 KD + (1 - alpha) CE)
//   dx = grad_scale * w (alpha T (q_T - P) + (1 - alpha)(q_1 - onehot))
// where P spreads p over the classes. One block per row: a first pass keeps a
// running maximum and the running sums of exp(x - m) and exp((x - m) / T); a
// second writes the gradient without the teacher's and the label's terms; the
// few listed classes are then written once more with them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "ttk_common.cuh"
#include "ttk_internal.h"

namespace ttk {
namespace distill {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
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

// Running (maximum, sum at temperature 1, sum at T) of part of a row.
struct Stat {
    float m, s1, sT;
};

__device__ __forceinline__ void push(Stat& a, float x, float cT) {
    if (x > a.m) {
        if (a.m > -INFINITY) {
            a.s1 *= exp_from(a.m, x, LOG2E);
            a.sT *= exp_from(a.m, x, cT);
        }
        a.m = x;
    }
    // -inf adds nothing (and -inf - -inf would be NaN); NaN reaches the sums
    if (!(x == -INFINITY)) {
        a.s1 += exp_from(x, a.m, LOG2E);
        a.sT += exp_from(x, a.m, cT);
    }
}

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float cT) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float z = r.m == -INFINITY ? 0.0f : r.m;
    r.s1 = a.s1 * exp_from(a.m, z, LOG2E) + b.s1 * exp_from(b.m, z, LOG2E);
    r.sT = a.sT * exp_from(a.m, z, cT) + b.sT * exp_from(b.m, z, cT);
    return r;
}

__device__ float block_max(float v, float* red) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & (WARPS - 1)];
    return warp_max(v);
}

__device__ double block_sum(double v, double* red) {
    v = warp_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < WARPS; ++i)
        s += red[i];
    return s;
}

__global__ void __launch_bounds__(THREADS) distill_row_kernel(const Args a) {
    __shared__ Stat s_stat[WARPS];
    __shared__ float s_red[WARPS];
    __shared__ double s_redd[WARPS];
    __shared__ int s_id[MAX_K + 1];
    __shared__ float s_coef[MAX_K + 1];  // teacher's and label's gradient per entry
    const int tid = threadIdx.x;
    const float cT = LOG2E / a.temperature, invT = 1.0f / a.temperature;
    const int K = static_cast<int>(a.K);
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
        const float w = a.row_weight ? a.row_weight[row] : 1.0f;
        float* dr = a.dlogits ? a.dlogits + row * a.ldd : nullptr;
        // The teacher's list and the label. NaN counts as present: it has to
        // reach the row's result.
        __syncthreads();  // s_id, s_coef: the previous row is done with them
        float zmax = -INFINITY;
        for (int k = tid; k < K; k += THREADS) {
            const int id = a.ids[row * a.K + k];
            const bool ok = id >= 0 && id < a.C;
            if (!ok && id != -1)
                report(kErrBadIndex);
            const float z = ok ? load_top(a.top, a.top_type, row * a.K + k) * invT : -INFINITY;
            s_id[k] = ok ? id : -1;
            s_coef[k] = z;
            zmax = fmaxf(zmax, z != z ? INFINITY : z);
        }
        zmax = block_max(zmax, s_red);
        const bool has = zmax > -INFINITY;
        const int64_t t = a.targets ? a.targets[row] : -1;
        const bool t_ok = t >= 0 && t < a.C;
        if (tid == 0 && !t_ok && t != -1)
            report(kErrBadIndex);
        if (w == 0.0f || (!has && !t_ok)) {  // nothing to learn from: the row is not read
            if (dr)
                for (int64_t c = tid; c < a.C; c += THREADS)
                    dr[c] = 0.0f;
            if (tid == 0)
                a.terms[2 * row] = a.terms[2 * row + 1] = 0.0;
            continue;
        }
        const float* xr = a.logits + row * a.ld;
        Stat st{-INFINITY, 0.0f, 0.0f};
        for (int64_t c = tid; c < a.C; c += THREADS)
            push(st, xr[c], cT);
        for (int o = 16; o > 0; o >>= 1) {
            Stat b{__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s1, o),
                   __shfl_xor_sync(~0u, st.sT, o)};
            st = merge(st, b, cT);
        }
        __syncthreads();
        if ((tid & 31) == 0)
            s_stat[tid >> 5] = st;
        __syncthreads();
        st = s_stat[0];
        for (int i = 1; i < WARPS; ++i)
            st = merge(st, s_stat[i], cT);
        const float m = st.m, log1 = logf(st.s1), logT = logf(st.sT);

        // Teacher probabilities, KD, gradient coefficients.
        double sz = 0.0;
        if (has)
            for (int k = tid; k < K; k += THREADS)
                if (s_id[k] >= 0)
                    sz += expf(s_coef[k] - zmax);
        sz = block_sum(sz, s_redd);
        const float logz = logf(static_cast<float>(sz)), invz = static_cast<float>(1.0 / sz);
        const float gs = a.grad_scale * w;
        const float gT = gs * a.alpha * a.temperature;
        double kd = 0.0;
        if (has)
            for (int k = tid; k < K; k += THREADS) {
                float p = 0.0f;
                if (s_id[k] >= 0) {
                    const float z = s_coef[k] - zmax;
                    p = expf(z) * invz;
                    if (p != 0.0f)
                        kd += static_cast<double>(p * ((z - logz) - ((xr[s_id[k]] - m) * invT - logT)));
                }
                s_coef[k] = gT * p;
            }
        else
            for (int k = tid; k < K; k += THREADS)
                s_coef[k] = 0.0f;
        kd = block_sum(kd, s_redd);
        const float g1 = t_ok ? gs * (1.0f - a.alpha) : 0.0f;
        if (tid == 0) {
            s_id[K] = t_ok ? static_cast<int>(t) : -1;
            s_coef[K] = g1;
            a.terms[2 * row] = w * kd;
            a.terms[2 * row + 1] = t_ok ? static_cast<double>(w) * (log1 + (m - xr[t])) : 0.0;
        }
        if (!dr)
            continue;
        // Gradient without the listed terms; entries of the list are read
        // before the row is overwritten (dlogits may be logits).
        const float k1 = t_ok ? g1 / st.s1 : 0.0f, kT = has ? gT / st.sT : 0.0f;
        auto base = [&](float x) {
            return kT * exp_from(x, m, cT) + k1 * exp_from(x, m, LOG2E);
        };
        __syncthreads();
        constexpr int PER = (MAX_K + 1 + THREADS - 1) / THREADS;
        float fix[PER];
        bool write[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int k = i * THREADS + tid;
            fix[i] = 0.0f;
            write[i] = false;
            if (k <= K && s_id[k] >= 0) {
                // the first entry of a class carries all of its entries, in list order
                bool first = true;
                for (int j = 0; j < k; ++j)
                    first = first && s_id[j] != s_id[k];
                float sum = 0.0f;
                if (first)
                    for (int j = k; j <= K; ++j)
                        sum += s_id[j] == s_id[k] ? s_coef[j] : 0.0f;
                if (first)
                    fix[i] = base(xr[s_id[k]]) - sum;
                write[i] = first;
            }
        }
        __syncthreads();
        for (int64_t c = tid; c < a.C; c += THREADS)
            dr[c] = base(xr[c]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int k = i * THREADS + tid;
            if (write[i])
                dr[s_id[k]] = fix[i];
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
    for (int64_t i = threadIdx.x; i < N; i += blockDim.x) {
        kd += terms[2 * i];
        ce += terms[2 * i + 1];
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
    if (N < 0 || C <= 0 || C > INT32_MAX || K < 0 || !loss || (N && !logits))
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
    if (reinterpret_cast<uintptr_t>(workspace) & 7)
        return set_error(TTK_ERR_ARG, "distill_loss: workspace must be 8-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* terms = static_cast<double*>(workspace);
    if (N) {
        const Args a{logits, ld, teacher_ids, teacher_logits, teacher_type, K, targets, row_weight,
                     N, C, alpha, temperature, grad_scale, terms, dlogits, ldd};
        distill_row_kernel<<<grid_for(N, 1, 148 * 4), THREADS, 0, st>>>(a);
        const int rc = check_launch("distill_row_kernel");
        if (rc)
            return rc;
    }
    distill_sum_kernel<<<1, 1024, 0, st>>>(terms, N, alpha, temperature, grad_scale, loss);
    return check_launch("distill_sum_kernel");
}

}  // extern "C"
