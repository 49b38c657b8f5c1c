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
//
// Both directions are bound by HBM: 16 bytes per element forward (x, b in;
// h, y out), 24 backward (dh, dy, h, b in; dx, db out), 4 or 8 more with a
// gate per element. A row is spread over TPR threads that keep it in
// registers from its one read to its writes, and the next row's loads are
// issued before this row's sums, so a thread always has a row in flight.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "ttk_common.cuh"
#include "ttk_internal.h"

namespace ttk {
namespace resnorm {

struct Gate {
    const float* p;
    int kind;
    // The factor a whole row shares (1 where the gate is per column or element).
    __device__ __forceinline__ float of_row(int64_t row) const {
        return kind == TTK_GATE_SCALAR ? p[0] : kind == TTK_GATE_ROW ? p[row] : 1.0f;
    }
    __device__ __forceinline__ float at(int64_t row, int64_t c, int64_t D) const {
        return kind == TTK_GATE_COLUMN ? p[c] : kind == TTK_GATE_FULL ? p[row * D + c] : of_row(row);
    }
};

struct Fwd {
    const float *x, *b, *w1;
    Gate g;
    const float* w2;
    float *h, *y, *r1, *r2;
    __nv_bfloat16* split;
    int64_t R, D;
    float alpha, eps;
};

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

// One thread's share of a row: NV words of VEC consecutive floats (VEC = 4
// needs D % 4 == 0 and aligned tensors), word j at (j * TPR + t) * VEC.
template <int VEC, int NV>
struct Cols {
    static constexpr int E = VEC * NV;
    int64_t c[NV];
    bool in[NV];
    __device__ __forceinline__ Cols(int t, int tpr, int64_t D) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            c[j] = (static_cast<int64_t>(j) * tpr + t) * VEC;
            in[j] = c[j] < D;
        }
    }
    __device__ __forceinline__ void load(float (&v)[E], const float* row, bool ok) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if constexpr (VEC == 4) {
                const float4 q = ok && in[j] ? *reinterpret_cast<const float4*>(row + c[j])
                                             : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
            } else {
                v[j] = ok && in[j] ? row[c[j]] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void store(float* row, const float (&v)[E]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                if constexpr (VEC == 4)
                    *reinterpret_cast<float4*>(row + c[j]) =
                        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                else
                    row[c[j]] = v[j];
            }
    }
    __device__ __forceinline__ void add_store(float* row, const float (&v)[E], bool add) const {
        if (!add)
            return store(row, v);
        float o[E];
        load(o, row, true);
#pragma unroll
        for (int i = 0; i < E; ++i)
            o[i] += v[i];
        store(row, o);
    }
    // hi and lo planes of v, `plane` elements apart
    __device__ __forceinline__ void store_split(__nv_bfloat16* row, int64_t plane,
                                                const float (&v)[E]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                __nv_bfloat16 hi[VEC], lo[VEC];
#pragma unroll
                for (int u = 0; u < VEC; ++u)
                    split_bf16(v[VEC * j + u], hi[u], lo[u]);
                if constexpr (VEC == 4) {
                    *reinterpret_cast<uint2*>(row + c[j]) = *reinterpret_cast<const uint2*>(hi);
                    *reinterpret_cast<uint2*>(row + plane + c[j]) =
                        *reinterpret_cast<const uint2*>(lo);
                } else {
                    row[c[j]] = hi[0];
                    row[plane + c[j]] = lo[0];
                }
            }
    }
};

// Sums of N values over the threads of a row. A row of one warp needs no
// barrier; otherwise the warps meet in red, which the caller alternates
// between two halves so that one barrier per sum is enough.
constexpr int MAX_WARPS = 32;
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int tpr, bool one_warp) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] += __shfl_xor_sync(~0u, v[i], o);
    if (one_warp)
        return;
    const int warp = threadIdx.x >> 5, w0 = threadIdx.x / tpr * (tpr >> 5), nw = tpr >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i)
            red[i * MAX_WARPS + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = 0.0f;
        for (int w = 0; w < nw; ++w)
            s += red[i * MAX_WARPS + w0 + w];
        v[i] = s;
    }
}

template <int VEC, int NV, bool FULL>
__global__ void __launch_bounds__(512) fwd_rows_kernel(const Fwd a, int tpr) {
    constexpr int E = VEC * NV;
    __shared__ float red[2][MAX_WARPS];
    const int slot = threadIdx.x / tpr, slots = blockDim.x / tpr;
    const bool one_warp = tpr == 32;
    const int64_t D = a.D;
    const Cols<VEC, NV> cols(threadIdx.x - slot * tpr, tpr, D);
    const float inv = 1.0f / static_cast<float>(D);
    float w1[E], w2[E];  // w1 with a gate per column folded in
    cols.load(w1, a.w1, true);
    cols.load(w2, a.w2, a.w2 != nullptr);
    if (a.g.kind == TTK_GATE_COLUMN) {
        float g[E];
        cols.load(g, a.g.p, true);
#pragma unroll
        for (int i = 0; i < E; ++i)
            w1[i] *= g[i];
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * slots;
    float x[E], b[E], g[FULL ? E : 1];
    auto fetch = [&](int64_t row, float (&xv)[E], float (&bv)[E], float (&gv)[FULL ? E : 1]) {
        const bool ok = row < a.R;
        cols.load(bv, a.b + row * D, ok);
        cols.load(xv, a.x + row * D, ok);
        if constexpr (FULL)
            cols.load(gv, a.g.p + row * D, ok);
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * slots + slot;
    fetch(row, x, b, g);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * slots; base < a.R;
         base += step, row += step) {
        const bool ok = row < a.R;
        float nx[E], nb[E], ng[FULL ? E : 1];
        fetch(row + step, nx, nb, ng);
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < E; ++i)
            s[0] += b[i] * b[i];
        row_sum(s, red[0], tpr, one_warp);
        const float r1 = 1.0f / sqrtf(s[0] * inv + a.eps);
        const float k = ok ? r1 * a.g.of_row(row) : 0.0f;
        float h[E];
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float u = b[i] * k * w1[i];
            if constexpr (FULL)
                u *= g[i];
            h[i] = a.alpha * x[i] + u;
            s[0] += h[i] * h[i];
        }
        row_sum(s, red[1], tpr, one_warp);
        const float r2 = 1.0f / sqrtf(s[0] * inv + a.eps);
        if (ok) {
            cols.store(a.h + row * D, h);
            if (threadIdx.x == slot * tpr) {
                a.r1[row] = r1;
                if (a.w2)
                    a.r2[row] = r2;
            }
            if (a.w2) {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    h[i] *= r2 * w2[i];
                cols.store(a.y + row * D, h);
                if (a.split)
                    cols.store_split(a.split + row * D, a.R * D, h);
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i)
            x[i] = nx[i], b[i] = nb[i];
        if constexpr (FULL)
#pragma unroll
            for (int i = 0; i < E; ++i)
                g[i] = ng[i];
    }
}

template <int VEC, int NV, bool FULL>
__global__ void __launch_bounds__(512) bwd_rows_kernel(const Bwd a, int tpr) {
    constexpr int E = VEC * NV;
    extern __shared__ float sums[];  // [slots - 1][2][D]: the other slots' column sums
    __shared__ float red[2][3 * MAX_WARPS];
    __shared__ double s_g[MAX_WARPS];
    const int slot = threadIdx.x / tpr, slots = blockDim.x / tpr;
    const bool one_warp = tpr == 32, lead = threadIdx.x == slot * tpr;
    const int64_t D = a.D;
    const Cols<VEC, NV> cols(threadIdx.x - slot * tpr, tpr, D);
    const float inv = 1.0f / static_cast<float>(D);
    const bool column = a.g.kind == TTK_GATE_COLUMN, need_dy = a.dy != nullptr;
    float w1[E], w2[E];  // w1 with a gate per column folded in
    cols.load(w1, a.w1, true);
    cols.load(w2, a.w2, need_dy);
    if (column) {
        float g[E];
        cols.load(g, a.g.p, true);
#pragma unroll
        for (int i = 0; i < E; ++i)
            w1[i] *= g[i];
    }
    float s1[E], s2[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
        s1[i] = s2[i] = 0.0f;
    double gsum = 0.0;
    struct Row {
        float dh[E], dy[E], h[E], b[E], g[FULL ? E : 1];
        float r1, r2, gr;
    };
    auto fetch = [&](int64_t row, Row& v) {
        const bool ok = row < a.R;
        cols.load(v.dy, a.dy + row * D, ok && need_dy);
        cols.load(v.h, a.h + row * D, ok && need_dy);
        cols.load(v.dh, a.dh + row * D, ok && a.dh);
        cols.load(v.b, a.b + row * D, ok);
        if constexpr (FULL)
            cols.load(v.g, a.g.p + row * D, ok);
        v.r1 = ok ? a.r1[row] : 0.0f;
        v.r2 = ok && need_dy ? a.r2[row] : 0.0f;
        v.gr = ok ? a.g.of_row(row) : 0.0f;
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * slots;
    int64_t row = static_cast<int64_t>(blockIdx.x) * slots + slot;
    int parity = 0;
    Row v;
    fetch(row, v);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * slots; base < a.R;
         base += step, row += step, parity ^= 1) {
        const bool ok = row < a.R;
        Row n;
        fetch(row + step, n);
        float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float e = v.dy[i] * w2[i];
            float c = w1[i] * v.b[i];
            if constexpr (FULL)
                c *= v.g[i];
            s[0] += e * v.h[i];
            s[1] += (v.dh[i] + v.r2 * e) * c;
            s[2] += v.h[i] * c;
        }
        row_sum(s, red[parity], tpr, one_warp);
        const float k2 = v.r2 * v.r2 * v.r2 * inv * s[0];
        const float dot = s[1] - k2 * s[2];  // sum(f b) without a gate of the whole row
        const float k1 = v.r1 * v.r1 * v.r1 * inv * dot * v.gr, r1g = v.r1 * v.gr;
        if (ok) {
            float dx[E], db[E];
            [[maybe_unused]] float dg[FULL ? E : 1];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float H = v.dh[i] + v.r2 * (v.dy[i] * w2[i]) - v.h[i] * k2;
                float f = H * w1[i], hb = H * v.b[i] * r1g;
                if constexpr (FULL) {
                    dg[i] = hb * w1[i];
                    f *= v.g[i];
                    hb *= v.g[i];
                }
                dx[i] = a.alpha * H;
                db[i] = r1g * f - v.b[i] * k1;
                s1[i] += hb;
                s2[i] += v.dy[i] * v.h[i] * v.r2;
            }
            cols.add_store(a.dx + row * D, dx, a.acc & TTK_ACC_DX);
            cols.add_store(a.db + row * D, db, a.acc & TTK_ACC_DB);
            if constexpr (FULL)
                if (a.dgate)
                    cols.add_store(a.dgate + row * D, dg, a.acc & TTK_ACC_DGATE);
            if (lead) {
                const float d = v.r1 * dot;
                if (a.g.kind == TTK_GATE_ROW && a.dgate)
                    a.dgate[row] = (a.acc & TTK_ACC_DGATE) ? a.dgate[row] + d : d;
                gsum += static_cast<double>(d);
            }
        }
        v = n;
    }
    // the block's rows, slot by slot
    if (slots > 1) {
        if (slot) {
            cols.store(sums + (2 * slot - 2) * D, s1);
            cols.store(sums + (2 * slot - 1) * D, s2);
        }
        __syncthreads();
        if (slot == 0)
            for (int q = 1; q < slots; ++q) {
                float o[E];
                cols.load(o, sums + (2 * q - 2) * D, true);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    s1[i] += o[i];
                cols.load(o, sums + (2 * q - 1) * D, true);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    s2[i] += o[i];
            }
    }
    if (slot == 0) {
        cols.store(a.part1 + blockIdx.x * D, s1);
        cols.store(a.part2 + blockIdx.x * D, s2);
    }
    if (a.g.kind == TTK_GATE_SCALAR) {
        if (lead)
            s_g[slot] = gsum;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int q = 1; q < slots; ++q)
                gsum += s_g[q];
            a.partg[blockIdx.x] = gsum;
        }
    }
}

// Rows too wide for the registers of a block (D > 8192): one block per row,
// each row read once per pass over it.
constexpr int WIDE_THREADS = 512;

__global__ void __launch_bounds__(WIDE_THREADS) fwd_wide_kernel(const Fwd a) {
    __shared__ float red[2][MAX_WARPS];
    const int64_t D = a.D;
    for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
        const int64_t o = row * D;
        float s[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS)
            s[0] += a.b[o + c] * a.b[o + c];
        row_sum(s, red[0], WIDE_THREADS, false);
        const float r1 = 1.0f / sqrtf(s[0] / static_cast<float>(D) + a.eps);
        s[0] = 0.0f;
        for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS) {
            const float h = a.alpha * a.x[o + c] + a.g.at(row, c, D) * (a.b[o + c] * r1 * a.w1[c]);
            a.h[o + c] = h;
            s[0] += h * h;
        }
        row_sum(s, red[1], WIDE_THREADS, false);
        const float r2 = 1.0f / sqrtf(s[0] / static_cast<float>(D) + a.eps);
        if (threadIdx.x == 0) {
            a.r1[row] = r1;
            if (a.w2)
                a.r2[row] = r2;
        }
        if (a.w2)
            for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS) {
                const float y = a.h[o + c] * (r2 * a.w2[c]);  // this thread's own h
                a.y[o + c] = y;
                if (a.split) {
                    __nv_bfloat16 hi, lo;
                    split_bf16(y, hi, lo);
                    a.split[o + c] = hi;
                    a.split[a.R * D + o + c] = lo;
                }
            }
    }
}

// The column sums stay in the block's own partial rows (each thread reads and
// writes its own columns only).
__global__ void __launch_bounds__(WIDE_THREADS) bwd_wide_kernel(const Bwd a) {
    __shared__ float red[2][3 * MAX_WARPS];
    const int64_t D = a.D;
    float* p1 = a.part1 + blockIdx.x * D;
    float* p2 = a.part2 + blockIdx.x * D;
    const bool per_row = a.g.kind == TTK_GATE_SCALAR || a.g.kind == TTK_GATE_ROW;
    double gsum = 0.0;
    int parity = 0;
    for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x, parity ^= 1) {
        const int64_t o = row * D;
        const float r1 = a.r1[row], r2 = a.dy ? a.r2[row] : 0.0f, gr = a.g.of_row(row);
        float s[3] = {0.0f, 0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS) {
            const float e = a.dy ? a.dy[o + c] * a.w2[c] : 0.0f, h = a.dy ? a.h[o + c] : 0.0f;
            const float k = (per_row ? 1.0f : a.g.at(row, c, D)) * a.w1[c] * a.b[o + c];
            s[0] += e * h;
            s[1] += ((a.dh ? a.dh[o + c] : 0.0f) + r2 * e) * k;
            s[2] += h * k;
        }
        row_sum(s, red[parity], WIDE_THREADS, false);
        const float k2 = r2 * r2 * r2 / static_cast<float>(D) * s[0];
        const float dot = s[1] - k2 * s[2];
        const float k1 = r1 * r1 * r1 / static_cast<float>(D) * dot * gr;
        const bool first = row == blockIdx.x;
        for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS) {
            const float dy = a.dy ? a.dy[o + c] : 0.0f, h = a.dy ? a.h[o + c] : 0.0f;
            const float b = a.b[o + c], g = a.g.at(row, c, D);
            const float H =
                (a.dh ? a.dh[o + c] : 0.0f) + (a.dy ? r2 * (dy * a.w2[c]) - h * k2 : 0.0f);
            const float hb = H * b * r1;
            const float dx = a.alpha * H, db = r1 * (H * g * a.w1[c]) - b * k1;
            a.dx[o + c] = (a.acc & TTK_ACC_DX) ? a.dx[o + c] + dx : dx;
            a.db[o + c] = (a.acc & TTK_ACC_DB) ? a.db[o + c] + db : db;
            p1[c] = (first ? 0.0f : p1[c]) + (a.g.kind == TTK_GATE_COLUMN ? hb : hb * g);
            p2[c] = (first ? 0.0f : p2[c]) + dy * h * r2;
            if (a.g.kind == TTK_GATE_FULL && a.dgate) {
                const float dg = hb * a.w1[c];
                a.dgate[o + c] = (a.acc & TTK_ACC_DGATE) ? a.dgate[o + c] + dg : dg;
            }
        }
        if (threadIdx.x == 0 && a.g.kind == TTK_GATE_ROW && a.dgate)
            a.dgate[row] = (a.acc & TTK_ACC_DGATE) ? a.dgate[row] + r1 * dot : r1 * dot;
        gsum += static_cast<double>(r1 * dot);
    }
    if (threadIdx.x == 0)
        a.partg[blockIdx.x] = gsum;
}

// Column sums of the nb partial rows into the weights' and the gate's
// gradients: 32 columns a block, warp w adds rows w, w + 16, ... and the
// warps' sums are added in order.
constexpr int FIN_WARPS = 16;
__global__ void __launch_bounds__(32 * FIN_WARPS) finish_kernel(const Bwd a, int64_t nb, float* dw1,
                                                                float* dw2) {
    __shared__ float red[2][FIN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool accw = a.acc & TTK_ACC_DW, accg = a.acc & TTK_ACC_DGATE;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s1 = 0.0f, s2 = 0.0f;
    if (c < a.D) {
#pragma unroll 4
        for (int64_t i = warp; i < nb; i += FIN_WARPS) {
            s1 += a.part1[i * a.D + c];
            s2 += a.part2[i * a.D + c];
        }
    }
    red[0][warp][lane] = s1;
    red[1][warp][lane] = s2;
    __syncthreads();
    if (warp == 0 && c < a.D) {
        s1 = s2 = 0.0f;
#pragma unroll
        for (int w = 0; w < FIN_WARPS; ++w)
            s1 += red[0][w][lane], s2 += red[1][w][lane];
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
    if (blockIdx.x == 0 && warp == 1 && a.g.kind == TTK_GATE_SCALAR && a.dgate) {
        double s = 0.0;
        for (int64_t i = lane; i < nb; i += 32)
            s += a.partg[i];
        s = warp_sum_d(s);
        if (lane == 0)
            a.dgate[0] = (accg ? a.dgate[0] : 0.0f) + static_cast<float>(s);
    }
}

// ----------------------------------------------------------------- launch --

// Threads of a row for `per` words (of 4 floats, or single floats) each.
int row_threads(int64_t D, int vec, int per) {
    const int64_t words = (D + vec - 1) / vec;
    return static_cast<int>(((words + per - 1) / per + 31) / 32 * 32);
}

bool aligned16(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (reinterpret_cast<uintptr_t>(p) & 15)
            return false;
    return true;
}

// Blocks of `kernel` that are resident at once on the current device.
template <class Kernel>
int64_t resident(Kernel kernel, int threads, size_t smem) {
    int dev = 0, sms = 0, per = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        sms = 148;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem) != cudaSuccess ||
        per <= 0) {
        cudaGetLastError();
        per = 1;
    }
    return static_cast<int64_t>(sms) * per;
}

constexpr int64_t MAX_ROW = 8192;     // widest row kept in registers
constexpr int64_t MAX_BLOCKS = 2048;  // partial rows of the backward

template <int VEC, int NV, bool FULL>
int run_fwd(const Fwd& a, cudaStream_t st) {
    const int tpr = row_threads(a.D, VEC, NV), slots = std::max(1, 256 / tpr);
    const int threads = tpr * slots;
    const int64_t blocks = std::min((a.R + slots - 1) / slots,
                                    resident(fwd_rows_kernel<VEC, NV, FULL>, threads, 0));
    fwd_rows_kernel<VEC, NV, FULL><<<static_cast<int>(blocks), threads, 0, st>>>(a, tpr);
    return check_launch("residual_norm_fwd");
}

template <int VEC, int NV, bool FULL>
int run_bwd(const Bwd& a, int64_t* nb, cudaStream_t st) {
    const int tpr = row_threads(a.D, VEC, NV), slots = std::max(1, 256 / tpr);
    const int threads = tpr * slots;
    const size_t smem = static_cast<size_t>(slots - 1) * 2 * a.D * sizeof(float);
    if (*nb == 0) {  // ask for the blocks alone
        *nb = std::min({(a.R + slots - 1) / slots, MAX_BLOCKS,
                        resident(bwd_rows_kernel<VEC, NV, FULL>, threads, smem)});
        return TTK_OK;
    }
    bwd_rows_kernel<VEC, NV, FULL><<<static_cast<int>(*nb), threads, smem, st>>>(a, tpr);
    return check_launch("residual_norm_bwd");
}

int dispatch_fwd(const Fwd& a, bool vec, cudaStream_t st) {
    const bool full = a.g.kind == TTK_GATE_FULL;
    if (vec) {
        if (a.D <= 4096)
            return full ? run_fwd<4, 2, true>(a, st) : run_fwd<4, 2, false>(a, st);
        return full ? run_fwd<4, 4, true>(a, st) : run_fwd<4, 4, false>(a, st);
    }
    if (a.D <= 4096)
        return full ? run_fwd<1, 8, true>(a, st) : run_fwd<1, 8, false>(a, st);
    return full ? run_fwd<1, 16, true>(a, st) : run_fwd<1, 16, false>(a, st);
}

int dispatch_bwd(const Bwd& a, bool vec, int64_t* nb, cudaStream_t st) {
    if (a.D > MAX_ROW) {
        if (*nb == 0) {
            *nb = std::min<int64_t>(a.R, 296);
            return TTK_OK;
        }
        bwd_wide_kernel<<<static_cast<int>(*nb), WIDE_THREADS, 0, st>>>(a);
        return check_launch("residual_norm_bwd");
    }
    const bool full = a.g.kind == TTK_GATE_FULL;
    if (vec) {
        if (a.D <= 4096)
            return full ? run_bwd<4, 2, true>(a, nb, st) : run_bwd<4, 2, false>(a, nb, st);
        return full ? run_bwd<4, 4, true>(a, nb, st) : run_bwd<4, 4, false>(a, nb, st);
    }
    if (a.D <= 4096)
        return full ? run_bwd<1, 8, true>(a, nb, st) : run_bwd<1, 8, false>(a, nb, st);
    return full ? run_bwd<1, 16, true>(a, nb, st) : run_bwd<1, 16, false>(a, nb, st);
}

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
        if (!w_next || D % 32 || !aligned16({y_split}))
            return set_error(TTK_ERR_ARG, "residual_norm_fwd: planes need w_next, D a multiple of "
                                          "32 and 16-byte alignment");
        if (ttk_gemm_get_precision() != 0)
            return set_error(TTK_ERR_ARG,
                             "residual_norm_fwd: planes exist for the bf16x3 precision");
    }
    if (!R)
        return TTK_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    bool vec = D % 4 == 0 && aligned16({x, b, w_post, w_next, h, y});
    if (gate_kind == TTK_GATE_COLUMN || gate_kind == TTK_GATE_FULL)
        vec = vec && aligned16({gate});
    const Fwd a{x, b, w_post, Gate{gate, gate_kind}, w_next, h, y, rstd_post, rstd_next,
                static_cast<__nv_bfloat16*>(y_split), R, D, residual_scale, eps};
    if (D > MAX_ROW) {
        fwd_wide_kernel<<<grid_for(R, 1, 148 * 4), WIDE_THREADS, 0, st>>>(a);
        return check_launch("residual_norm_fwd");
    }
    return dispatch_fwd(a, vec, st);
}

// Partial rows for any kernel the backward may choose, and one double each.
size_t ttk_residual_norm_bwd_workspace_size(int64_t R, int64_t D) {
    const int64_t nb = std::min<int64_t>(std::max<int64_t>(R, 1), MAX_BLOCKS);
    return static_cast<size_t>(nb) * (8 + 8 * static_cast<size_t>(std::max<int64_t>(D, 0))) + 16;
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
        !aligned16({workspace}))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: workspace too small or not 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Bwd a{dh, dy, h, b, w_post, Gate{gate, gate_kind}, w_next, rstd_post, rstd_next, dx, db, dgate,
          nullptr, nullptr, nullptr, accumulate, R, D, residual_scale};
    int64_t nb = 0;
    if (R) {
        bool vec = D % 4 == 0 && aligned16({dh, dy, b, w_post, dx, db}) &&
                   (!dy || aligned16({h, w_next}));
        if (gate_kind == TTK_GATE_COLUMN)
            vec = vec && aligned16({gate});
        if (gate_kind == TTK_GATE_FULL)
            vec = vec && aligned16({gate, dgate});
        int rc = dispatch_bwd(a, vec, &nb, st);
        if (rc)
            return rc;
        a.part1 = static_cast<float*>(workspace);  // rows first: they are stored as float4
        a.part2 = a.part1 + nb * D;
        a.partg = reinterpret_cast<double*>(a.part2 + nb * D);  // 2 nb D floats: 8-byte aligned
        rc = dispatch_bwd(a, vec, &nb, st);
        if (rc)
            return rc;
    }
    finish_kernel<<<static_cast<int>((D + 31) / 32), 32 * FIN_WARPS, 0, st>>>(a, nb, dw_post,
                                                                              dw_next);
    return check_launch("residual_norm_bwd sums");
}

}  // extern "C"
