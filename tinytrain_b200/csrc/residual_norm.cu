// Residual norm: the RMSNorm after a block, its gate, the residual scale, the
// residual add and the RMSNorm before the next block as one operator.
//
//   r1 = (mean(b^2) + eps)^-1/2,  h = a x + g (b r1 w1)
//   r2 = (mean(h^2) + eps)^-1/2,  y = h r2 w2
// Backward, with dh the gradient that reaches h past the norm and dy the one
// of y:
//   e = dy w2,  H = dh + r2 e - h r2^3/D sum(e h),  dx = a H
//   f = H g w1, db = r1 f - b r1^3/D sum(f b)
//   dw1 = sum_rows H g b r1,  dw2 = sum_rows dy h r2,  dg = H b r1 w1 summed
//   to g's shape
// sum(f b) needs H, which needs sum(e h); with c = g w1 b,
//   sum(f b) = sum((dh + r2 e) c) - r2^3/D sum(e h) sum(h c),
// so one round of row sums gives both.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "ttk_common.cuh"
#include "ttk_internal.h"

namespace ttk {
namespace resnorm {

struct Gate {
    const float* p;
    int kind;
    __device__ __forceinline__ float at(int64_t row, int64_t c, int64_t D) const {
        switch (kind) {
            case TTK_GATE_SCALAR: return p[0];
            case TTK_GATE_COLUMN: return p[c];
            case TTK_GATE_ROW: return p[row];
            case TTK_GATE_FULL: return p[row * D + c];
            default: return 1.0f;
        }
    }
};

// One warp per row, the row read once for each pass over it.
__global__ void __launch_bounds__(256) fwd_kernel(const float* __restrict__ x,
                                                  const float* __restrict__ b,
                                                  const float* __restrict__ w1, const Gate g,
                                                  const float* __restrict__ w2,
                                                  float* __restrict__ h, float* __restrict__ y,
                                                  float* __restrict__ rstd1,
                                                  float* __restrict__ rstd2,
                                                  __nv_bfloat16* __restrict__ split, int64_t R,
                                                  int64_t D, float alpha, float eps) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < R;
         row += warps) {
        const float* xr = x + row * D;
        const float* br = b + row * D;
        float* hr = h + row * D;
        float ss = 0.0f;
        for (int64_t c = lane; c < D; c += 32)
            ss += br[c] * br[c];
        const float r1 = 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(D) + eps);
        ss = 0.0f;
        for (int64_t c = lane; c < D; c += 32) {
            const float v = alpha * xr[c] + g.at(row, c, D) * (br[c] * r1 * w1[c]);
            hr[c] = v;
            ss += v * v;
        }
        const float r2 = 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(D) + eps);
        if (lane == 0) {
            rstd1[row] = r1;
            if (w2)
                rstd2[row] = r2;
        }
        if (w2)
            for (int64_t c = lane; c < D; c += 32) {
                const float v = hr[c] * r2 * w2[c];
                y[row * D + c] = v;
                if (split) {
                    __nv_bfloat16 hi, lo;
                    split_bf16(v, hi, lo);
                    split[row * D + c] = hi;
                    split[(R + row) * D + c] = lo;
                }
            }
    }
}

struct Bwd {
    const float *dh, *dy, *h, *b, *w1;
    Gate g;
    const float *w2, *r1, *r2;
    float *dx, *db, *dgate;
    float *part1, *part2;  // [blocks][D]: sums of H g b r1 (H b r1, gate per column), dy h r2
    double* partg;         // [blocks]: scalar gate
    int acc;
    int64_t R, D;
    float alpha;
};

// One block per row, each thread a fixed set of columns; a block's rows are
// summed into its partial rows.
__global__ void __launch_bounds__(256) bwd_kernel(const Bwd a) {
    extern __shared__ float sums[];  // [2][D]
    __shared__ float red[3][8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t D = a.D;
    for (int64_t c = tid; c < 2 * D; c += blockDim.x)
        sums[c] = 0.0f;
    const bool per_row = a.g.kind == TTK_GATE_SCALAR || a.g.kind == TTK_GATE_ROW;
    double gsum = 0.0;
    for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
        const int64_t o = row * D;
        const float r1 = a.r1[row], r2 = a.dy ? a.r2[row] : 0.0f;
        const float grow = per_row ? a.g.at(row, 0, D) : 1.0f;
        float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = tid; c < D; c += blockDim.x) {
            const float e = a.dy ? a.dy[o + c] * a.w2[c] : 0.0f;
            const float hv = a.dy ? a.h[o + c] : 0.0f;
            const float cc = (per_row ? 1.0f : a.g.at(row, c, D)) * a.w1[c] * a.b[o + c];
            s0 += e * hv;
            s1 += ((a.dh ? a.dh[o + c] : 0.0f) + r2 * e) * cc;
            s2 += hv * cc;
        }
        s0 = warp_sum(s0), s1 = warp_sum(s1), s2 = warp_sum(s2);
        __syncthreads();
        if (lane == 0)
            red[0][warp] = s0, red[1][warp] = s1, red[2][warp] = s2;
        __syncthreads();
        s0 = s1 = s2 = 0.0f;
        for (int i = 0; i < 8; ++i)
            s0 += red[0][i], s1 += red[1][i], s2 += red[2][i];
        const float k2 = r2 * r2 * r2 / static_cast<float>(D) * s0;
        const float dot = s1 - k2 * s2;  // sum(f b), without a row's own gate
        const float k1 = r1 * r1 * r1 / static_cast<float>(D) * dot * grow;
        for (int64_t c = tid; c < D; c += blockDim.x) {
            const float dyv = a.dy ? a.dy[o + c] : 0.0f, hv = a.dy ? a.h[o + c] : 0.0f;
            const float bv = a.b[o + c];
            const float H = (a.dh ? a.dh[o + c] : 0.0f) + (a.dy ? r2 * (dyv * a.w2[c]) - hv * k2 : 0.0f);
            const float gv = per_row ? grow : a.g.at(row, c, D);
            const float hb = H * bv * r1;
            const float db = r1 * (H * gv * a.w1[c]) - bv * k1;
            const float dx = a.alpha * H;
            a.dx[o + c] = (a.acc & TTK_ACC_DX) ? a.dx[o + c] + dx : dx;
            a.db[o + c] = (a.acc & TTK_ACC_DB) ? a.db[o + c] + db : db;
            sums[c] += a.g.kind == TTK_GATE_COLUMN ? hb : hb * gv;
            sums[D + c] += dyv * hv * r2;
            if (a.g.kind == TTK_GATE_FULL && a.dgate) {
                const float dg = hb * a.w1[c];
                a.dgate[o + c] = (a.acc & TTK_ACC_DGATE) ? a.dgate[o + c] + dg : dg;
            }
        }
        if (tid == 0 && a.g.kind == TTK_GATE_ROW && a.dgate)
            a.dgate[row] = (a.acc & TTK_ACC_DGATE) ? a.dgate[row] + r1 * dot : r1 * dot;
        gsum += static_cast<double>(r1 * dot);
    }
    __syncthreads();
    for (int64_t c = tid; c < D; c += blockDim.x) {
        a.part1[blockIdx.x * D + c] = sums[c];
        a.part2[blockIdx.x * D + c] = sums[D + c];
    }
    if (tid == 0)
        a.partg[blockIdx.x] = gsum;
}

// Column sums of the partial rows, in row order, into the weights' and the
// gate's gradients.
__global__ void __launch_bounds__(256) finish_kernel(const Bwd a, int64_t nb, float* dw1,
                                                     float* dw2) {
    const int64_t c = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const bool accw = a.acc & TTK_ACC_DW, accg = a.acc & TTK_ACC_DGATE;
    if (c < a.D) {
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t i = 0; i < nb; ++i) {
            s1 += a.part1[i * a.D + c];
            s2 += a.part2[i * a.D + c];
        }
        if (a.g.kind == TTK_GATE_COLUMN) {
            if (a.dgate)
                a.dgate[c] = (accg ? a.dgate[c] : 0.0f) + s1 * a.w1[c];
            s1 *= a.g.p[c];
        }
        if (dw1)
            dw1[c] = (accw ? dw1[c] : 0.0f) + s1;
        if (dw2)
            dw2[c] = (accw ? dw2[c] : 0.0f) + s2;
    }
    if (c == 0 && a.g.kind == TTK_GATE_SCALAR && a.dgate) {
        double s = 0.0;
        for (int64_t i = 0; i < nb; ++i)
            s += a.partg[i];
        a.dgate[0] = (accg ? a.dgate[0] : 0.0f) + static_cast<float>(s);
    }
}

int64_t bwd_blocks(int64_t R) { return std::min<int64_t>(std::max<int64_t>(R, 1), 296); }

}  // namespace resnorm
}  // namespace ttk

using namespace ttk;
using namespace ttk::resnorm;

static int check_gate(const float* gate, int kind, const char* msg) {
    if (kind < TTK_GATE_NONE || kind > TTK_GATE_FULL || (kind != TTK_GATE_NONE && !gate))
        return set_error(TTK_ERR_ARG, msg);
    return TTK_OK;
}

extern "C" {

int ttk_residual_norm_fwd(const float* x, const float* b, const float* w_post, const float* gate,
                          int gate_kind, const float* w_next, float* h, float* y, float* rstd_post,
                          float* rstd_next, void* y_split, int64_t R, int64_t D,
                          float residual_scale, float eps, void* stream) {
    if (R < 0 || D <= 0 || (R && (!x || !b || !w_post || !h || !rstd_post)))
        return set_error(TTK_ERR_ARG, "residual_norm_fwd: bad arguments");
    if (R && w_next && (!y || !rstd_next))
        return set_error(TTK_ERR_ARG, "residual_norm_fwd: w_next needs y and rstd_next");
    if (R)
        if (int rc = check_gate(gate, gate_kind, "residual_norm_fwd: bad gate"))
            return rc;
    if (y_split) {
        if (!w_next || D % 32 || (reinterpret_cast<uintptr_t>(y_split) & 15))
            return set_error(TTK_ERR_ARG, "residual_norm_fwd: planes need w_next, D a multiple of "
                                          "32 and 16-byte alignment");
        if (ttk_gemm_get_precision() != 0)
            return set_error(TTK_ERR_ARG,
                             "residual_norm_fwd: planes exist for the bf16x3 precision");
    }
    if (!R)
        return TTK_OK;
    fwd_kernel<<<grid_for(R, 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        x, b, w_post, Gate{gate, gate_kind}, w_next, h, y, rstd_post, rstd_next,
        static_cast<__nv_bfloat16*>(y_split), R, D, residual_scale, eps);
    return check_launch("residual_norm_fwd");
}

size_t ttk_residual_norm_bwd_workspace_size(int64_t R, int64_t D) {
    const int64_t nb = bwd_blocks(R);
    return static_cast<size_t>(nb) * (8 + 8 * static_cast<size_t>(D));
}

int ttk_residual_norm_bwd(const float* dh, const float* dy, const float* h, const float* b,
                          const float* w_post, const float* gate, int gate_kind,
                          const float* w_next, const float* rstd_post, const float* rstd_next,
                          float* dx, float* db, float* dw_post, float* dw_next, float* dgate,
                          int accumulate, int64_t R, int64_t D, float residual_scale,
                          void* workspace, size_t workspace_bytes, void* stream) {
    if (R < 0 || D <= 0 || (R && (!b || !w_post || !rstd_post || !dx || !db)))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: bad arguments");
    if (R && !dh && !dy)
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: neither dh nor dy");
    if (R && dy && (!h || !w_next || !rstd_next))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: dy needs h, w_next and rstd_next");
    if (R)
        if (int rc = check_gate(gate, gate_kind, "residual_norm_bwd: bad gate"))
            return rc;
    if (accumulate & ~(TTK_ACC_DX | TTK_ACC_DB | TTK_ACC_DW | TTK_ACC_DGATE))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: unknown accumulate bits");
    if (!workspace || workspace_bytes < ttk_residual_norm_bwd_workspace_size(R, D) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: workspace too small or not 16-byte aligned");
    const size_t smem = static_cast<size_t>(D) * 8;
    if (smem > 200 * 1024)
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: D too large");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t nb = R ? bwd_blocks(R) : 0;
    double* pg = static_cast<double*>(workspace);
    float* p1 = reinterpret_cast<float*>(pg + bwd_blocks(R));
    const Bwd a{dh, dy, h, b, w_post, Gate{gate, gate_kind}, w_next, rstd_post, rstd_next, dx, db,
                dgate, p1, p1 + nb * D, pg, accumulate, R, D, residual_scale};
    if (R) {
        if (smem > 48 * 1024)
            cudaFuncSetAttribute(bwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(smem));
        bwd_kernel<<<static_cast<int>(nb), 256, smem, st>>>(a);
        const int rc = check_launch("residual_norm_bwd");
        if (rc)
            return rc;
    }
    finish_kernel<<<static_cast<int>((D + 255) / 256), 256, 0, st>>>(a, nb, dw_post, dw_next);
    return check_launch("residual_norm_bwd sums");
}

}  // extern "C"
