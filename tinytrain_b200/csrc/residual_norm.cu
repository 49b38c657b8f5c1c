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
//   sum(f b) = sum((dh + r2 e) c) - r2^2/D sum(e h) sum(h r2 c),
// so one round of row sums gives both. A third power of r is taken one factor at a
// time with the sum it belongs to: by itself it leaves fp32 where a row's values are
// past 1e13 or below 1e-13.
//
// Both directions are bound by HBM: 16 bytes per element forward (x, b in;
// h, y out), 24 backward (dh, dy, h, b in; dx, db out), 4 or 8 more with a
// gate per element. A row belongs to TPR threads (a slot of the block) that
// keep it in registers from its one read to its writes. The rows come through
// shared memory: one thread of the slot copies the slot's next rows with bulk
// copies, as many ahead as the memory holds, so the reads go on while the
// slot adds up, waits at its barrier and writes. (With plain loads a row ahead
// in registers instead: 225 and 339 us forward and backward where this took 176
// and 258, in calls one after the other.)
// Measured in a CUDA graph, on inputs that are not in L2: 32768 x 2048, gate per
// column, forward 197 us, 5.4 TB/s (half of it writes), backward 236 us, 6.8 TB/s (a
// third writes; a copy 6.55); backward of 3001 x 1111 with a gate per element 31 us,
// 3.4 TB/s: 7 rows a slot, of which the first load and the last store stand alone
// (30010 rows: 175 us, 6.1 TB/s).
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "pdl.cuh"
#include "row_span.h"
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

// One thread's share of a row: NV words of four floats, word j at 16-byte word
// j * TPR + t of the row. Rows of a width that is no multiple of four (ODD) begin
// `off` floats into their first word; the words that a row shares with its
// neighbours belong to it in part. A slot's rows are chosen to have one `off`,
// so that a thread's columns stay the same.
template <int NV, bool ODD>
struct Cols {
    static constexpr int E = 4 * NV;
    int w[NV];  // word of the row
    int c[NV];  // its first column (negative in the first word of an odd row)
    bool in[NV], full[NV], edge;
    int D;
    __device__ __forceinline__ Cols(int t, int tpr, int64_t width, int off)
        : edge(false), D(static_cast<int>(width)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            w[j] = j * tpr + t;
            c[j] = 4 * w[j] - (ODD ? off : 0);
            in[j] = c[j] < D;
            full[j] = ODD ? c[j] >= 0 && c[j] + 4 <= D : in[j];
            edge |= in[j] && !full[j];
        }
    }
    // Zeros in place of what the thread's words hold of the neighbouring rows:
    // one branch for all tensors, which only the two warps at a row's ends take.
    template <class... V>
    __device__ __forceinline__ void mask(V&... v) const {
        if (ODD && edge)
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int col = c[i / 4] + i % 4;
                const bool mine = col >= 0 && col < D;
                ((v[i] = mine ? v[i] : 0.0f), ...);
            }
    }
    // columns of p, whose alignment is the row's (ALIGNED) or any
    template <bool ALIGNED>
    __device__ __forceinline__ void load(float (&v)[E], const float* p, bool ok) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
            if (ok && full[j] && (ALIGNED || !ODD))
                q = *reinterpret_cast<const float4*>(p + c[j]);
            v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
            if (ODD && ok && in[j] && !(ALIGNED && full[j]))
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (c[j] + u >= 0 && c[j] + u < D)
                        v[4 * j + u] = p[c[j] + u];
        }
    }
    template <bool ALIGNED>
    __device__ __forceinline__ void store(float* p, const float (&v)[E]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (full[j] && (ALIGNED || !ODD))
                *reinterpret_cast<float4*>(p + c[j]) =
                    make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            if (ODD && in[j] && !(ALIGNED && full[j]))
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (c[j] + u >= 0 && c[j] + u < D)
                        p[c[j] + u] = v[4 * j + u];
        }
    }
    __device__ __forceinline__ void add_store(float* row, const float (&v)[E], bool add) const {
        if (!add)
            return store<true>(row, v);
        float o[E];
        load<true>(o, row, true);
#pragma unroll
        for (int i = 0; i < E; ++i)
            o[i] += v[i];
        store<true>(row, o);
    }
    // hi and lo planes of v, `plane` elements apart (widths of whole words)
    __device__ __forceinline__ void store_split(__nv_bfloat16* row, int64_t plane,
                                                const float (&v)[E]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in[j]) {
                __nv_bfloat16 hi[4], lo[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    split_bf16(v[4 * j + u], hi[u], lo[u]);
                *reinterpret_cast<uint2*>(row + c[j]) = *reinterpret_cast<const uint2*>(hi);
                *reinterpret_cast<uint2*>(row + plane + c[j]) = *reinterpret_cast<const uint2*>(lo);
            }
    }
};

// Sums of N values over the threads of a row, and whether `ok` holds in all of
// them. A row of one warp needs no barrier; otherwise the warps meet in red,
// which the caller alternates between two halves so that one barrier per sum
// is enough. Every thread of the slot gets here: its waits are bounded.
constexpr int MAX_WARPS = 16;
template <int N>
__device__ __forceinline__ bool row_sum(float (&v)[N], float* red, int slot, int tpr, bool ok) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] += __shfl_xor_sync(~0u, v[i], o);
    if (tpr == 32) {
        const bool all = __all_sync(~0u, ok);
        __syncwarp();  // the vote orders no memory: reads of a stage end before its next copy
        return all;
    }
    const int warp = threadIdx.x >> 5, w0 = slot * (tpr >> 5), nw = tpr >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i)
            red[i * MAX_WARPS + warp] = v[i];
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(static_cast<uint32_t>(ok)), "r"(1 + slot), "r"(tpr)
        : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = 0.0f;
        for (int w = 0; w < nw; ++w)
            s += red[i * MAX_WARPS + w0 + w];
        v[i] = s;
    }
    return all != 0;
}

constexpr int MAX_STAGES = 4;
constexpr int MAX_SLOTS = 8;

// The slot's stages of NT rows (one per tensor; a null tensor is skipped and
// reads as zeros), `pitch` floats each. A bulk copy moves a row's words whole,
// with what they hold of its neighbours, which Cols::mask takes out again; a word
// that the tensor's end cuts short is copied by floats (row_tail).
template <int NV, bool ODD, int NT>
struct Feed {
    static constexpr int E = 4 * NV;
    const float* t[NT];
    float* buf;  // [stages][NT][pitch]
    uint64_t* bar;
    int64_t first_cut, D;
    int off, pitch;

    __device__ __forceinline__ void issue(int stage, int64_t row) const {
        uint32_t bytes = static_cast<uint32_t>(D) * 4u;
        if (ODD) {
            const int end = static_cast<int>(off + D), tail = row_tail(row, first_cut, end);
            bytes = static_cast<uint32_t>((end - tail + 3) / 4) * 16u;
            if (tail)
                for (int i = 0; i < NT; ++i)
                    for (int k = end - tail; k < end; ++k)
                        if (t[i] && k >= off)
                            buf[(stage * NT + i) * pitch + k] = t[i][row * D - off + k];
        }
        uint32_t total = 0;
#pragma unroll
        for (int i = 0; i < NT; ++i)
            total += t[i] ? bytes : 0u;
        mbar_arrive_expect_tx(bar + stage, total);
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (t[i] && bytes)
                bulk_load(buf + (stage * NT + i) * pitch, t[i] + row * D - (ODD ? off : 0), bytes,
                          bar + stage);
    }
    __device__ __forceinline__ void read(float (&v)[E], int i, int stage,
                                         const Cols<NV, ODD>& cols) const {
        const float4* b = reinterpret_cast<const float4*>(buf + (stage * NT + i) * pitch);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const float4 q = t[i] && cols.in[j] ? b[cols.w[j]] : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
        }
    }
};

template <int NV, bool ODD, bool FULL>
__global__ void __launch_bounds__(512) fwd_rows_kernel(const Fwd a, int tpr, int pitch, int stages) {
    constexpr int E = 4 * NV, NT = FULL ? 3 : 2;
    extern __shared__ __align__(16) float smem[];
    __shared__ float red[2][MAX_WARPS];
    __shared__ __align__(8) uint64_t bars[MAX_SLOTS * MAX_STAGES];
    const int slot = threadIdx.x / tpr, slots = blockDim.x / tpr;
    const bool lead = threadIdx.x == slot * tpr;
    const int64_t D = a.D;
    const int64_t step = static_cast<int64_t>(gridDim.x) * slots;
    int64_t row = static_cast<int64_t>(blockIdx.x) * slots + slot;
    const int off = ODD ? static_cast<int>((row * D) & 3) : 0;
    const Cols<NV, ODD> cols(threadIdx.x - slot * tpr, tpr, D, off);
    Feed<NV, ODD, NT> feed;
    feed.t[0] = a.b, feed.t[1] = a.x;
    if constexpr (FULL)
        feed.t[2] = a.g.p;
    feed.buf = smem + static_cast<int64_t>(slot) * stages * NT * pitch;
    feed.bar = bars + slot * MAX_STAGES;
    feed.first_cut = first_cut_row(a.R, D);
    feed.D = D, feed.off = off, feed.pitch = pitch;
    if (lead) {
        for (int s = 0; s < stages; ++s)
            mbar_init(feed.bar + s, 1);
        fence_barrier_init();
    }
    __syncthreads();
    grid_wait();
    if (lead)
        for (int s = 0; s < stages && row + s * step < a.R; ++s)
            feed.issue(s, row + s * step);
    const float inv = 1.0f / static_cast<float>(D);
    float w1[E], w2[E];  // w1 with a gate per column folded in
    cols.template load<false>(w1, a.w1, true);
    cols.template load<false>(w2, a.w2, a.w2 != nullptr);
    if (a.g.kind == TTK_GATE_COLUMN) {
        float g[E];
        cols.template load<false>(g, a.g.p, true);
#pragma unroll
        for (int i = 0; i < E; ++i)
            w1[i] *= g[i];
    }
    int stage = 0;
    uint32_t phase = 0;
    for (; row < a.R; row += step) {
        const float gr = a.g.of_row(row);
        bool ok = mbar_wait(feed.bar + stage, phase, 90);
        float x[E], b[E], g[FULL ? E : 1];
        feed.read(b, 0, stage, cols);
        feed.read(x, 1, stage, cols);
        if constexpr (FULL)
            feed.read(g, 2, stage, cols);
        if constexpr (FULL)
            cols.mask(b, x, g);
        else
            cols.mask(b, x);
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < E; ++i)
            s[0] += b[i] * b[i];
        ok = row_sum(s, red[0], slot, tpr, ok);
        if (!ok) {
            // a copy did not arrive: the slot stops once its copies have ended
            if (lead)
                for (int64_t i = 0; i < stages && row + i * step < a.R; ++i) {
                    mbar_wait(feed.bar + stage, phase, 91);
                    if (++stage == stages)
                        stage = 0, phase ^= 1;
                }
            break;
        }
        if (lead && row + stages * step < a.R) {  // every thread has read the stage
            fence_async_smem();
            feed.issue(stage, row + stages * step);
        }
        if (++stage == stages)
            stage = 0, phase ^= 1;
        const float r1 = 1.0f / sqrtf(s[0] * inv + a.eps);
        const float k = r1 * gr;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float u = b[i] * k * w1[i];
            if constexpr (FULL)
                u *= g[i];
            x[i] = a.alpha * x[i] + u;  // h
            s[0] += x[i] * x[i];
        }
        cols.template store<true>(a.h + row * D, x);
        row_sum(s, red[1], slot, tpr, true);
        const float r2 = 1.0f / sqrtf(s[0] * inv + a.eps);
        if (lead) {
            a.r1[row] = r1;
            if (a.w2)
                a.r2[row] = r2;
        }
        if (a.w2) {
#pragma unroll
            for (int i = 0; i < E; ++i)
                x[i] *= r2 * w2[i];
            cols.template store<true>(a.y + row * D, x);
            if (a.split)
                cols.store_split(a.split + row * D, a.R * D, x);
        }
    }
}

// Rows whose terms a thread adds up in registers before they go to the sums in
// shared memory (its own, so without a barrier): chains of FOLD rows and of their
// sums instead of one chain. The weights' gradients of 32768 x 2048, 110 rows a
// slot, are then within 1.5e-7 of the 64-bit sums instead of 2.3e-7, at the
// same time (236 to 237 us). Slots of up to 2 FOLD rows keep one chain.
constexpr int FOLD = 16;

// folded: whether shared memory has room for those sums after the stages.
template <int NV, bool ODD, bool FULL>
__global__ void __launch_bounds__(512)
    bwd_rows_kernel(const Bwd a, int tpr, int pitch, int stages, bool folded) {
    constexpr int E = 4 * NV, NT = FULL ? 5 : 4;
    extern __shared__ __align__(16) float smem[];
    __shared__ float red[2][3 * MAX_WARPS];
    __shared__ double s_g[MAX_SLOTS];
    __shared__ __align__(8) uint64_t bars[MAX_SLOTS * MAX_STAGES];
    const int slot = threadIdx.x / tpr, slots = blockDim.x / tpr;
    const bool lead = threadIdx.x == slot * tpr;
    const int64_t D = a.D;
    const int64_t step = static_cast<int64_t>(gridDim.x) * slots;
    int64_t row = static_cast<int64_t>(blockIdx.x) * slots + slot;
    const int off = ODD ? static_cast<int>((row * D) & 3) : 0;
    const Cols<NV, ODD> cols(threadIdx.x - slot * tpr, tpr, D, off);
    const bool need_dy = a.dy != nullptr;
    Feed<NV, ODD, NT> feed;
    feed.t[0] = a.dy, feed.t[1] = need_dy ? a.h : nullptr, feed.t[2] = a.dh, feed.t[3] = a.b;
    if constexpr (FULL)
        feed.t[4] = a.g.p;
    feed.buf = smem + static_cast<int64_t>(slot) * stages * NT * pitch;
    feed.bar = bars + slot * MAX_STAGES;
    feed.first_cut = first_cut_row(a.R, D);
    feed.D = D, feed.off = off, feed.pitch = pitch;
    if (lead) {
        for (int s = 0; s < stages; ++s)
            mbar_init(feed.bar + s, 1);
        fence_barrier_init();
    }
    if (folded)
        for (int j = 0; j < 2 * NV; ++j)
            reinterpret_cast<float4*>(smem + slots * stages * NT * pitch)[j * blockDim.x + threadIdx.x] =
                make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    grid_wait();
    if (lead)
        for (int s = 0; s < stages && row + s * step < a.R; ++s)
            feed.issue(s, row + s * step);
    const float inv = 1.0f / static_cast<float>(D);
    float w1[E], w2[E];  // w1 with a gate per column folded in
    cols.template load<false>(w1, a.w1, true);
    cols.template load<false>(w2, a.w2, need_dy);
    if (a.g.kind == TTK_GATE_COLUMN) {
        float g[E];
        cols.template load<false>(g, a.g.p, true);
#pragma unroll
        for (int i = 0; i < E; ++i)
            w1[i] *= g[i];
    }
    float s1[E], s2[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
        s1[i] = s2[i] = 0.0f;
    double gsum = 0.0;
    int stage = 0, parity = 0;
    uint32_t phase = 0;
    while (row < a.R) {
        const int64_t until = folded ? min(a.R, row + FOLD * step) : a.R;
        for (; row < until; row += step, parity ^= 1) {
            const float r1 = a.r1[row], r2 = need_dy ? a.r2[row] : 0.0f, gr = a.g.of_row(row);
            bool ok = mbar_wait(feed.bar + stage, phase, 92);
            float dy[E], h[E], dh[E], b[E], g[FULL ? E : 1];
            feed.read(dy, 0, stage, cols);
            feed.read(h, 1, stage, cols);
            feed.read(dh, 2, stage, cols);
            feed.read(b, 3, stage, cols);
            if constexpr (FULL)
                feed.read(g, 4, stage, cols);
            if constexpr (FULL)
                cols.mask(dy, h, dh, b, g);
            else
                cols.mask(dy, h, dh, b);
            float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float e = dy[i] * w2[i];
                float c = w1[i] * b[i];
                if constexpr (FULL)
                    c *= g[i];
                s[0] += e * h[i];
                s[1] += (dh[i] + r2 * e) * c;
                s[2] += (h[i] * r2) * c;
            }
            ok = row_sum(s, red[parity], slot, tpr, ok);
            if (!ok) {
                // a copy did not arrive: the slot stops once its copies have ended
                if (lead)
                    for (int64_t i = 0; i < stages && row + i * step < a.R; ++i) {
                        mbar_wait(feed.bar + stage, phase, 93);
                        if (++stage == stages)
                            stage = 0, phase ^= 1;
                    }
                row = a.R;
                break;
            }
            if (lead && row + stages * step < a.R) {  // every thread has read the stage
                fence_async_smem();
                feed.issue(stage, row + stages * step);
            }
            if (++stage == stages)
                stage = 0, phase ^= 1;
            const float m2 = r2 * (r2 * (inv * s[0])), k2 = r2 * m2;
            const float dot = s[1] - m2 * s[2];  // sum(f b) without a gate of the whole row
            const float k1 = r1 * (r1 * (r1 * (inv * dot))) * gr, r1g = r1 * gr;
            float dx[E], db[E];
            [[maybe_unused]] float dg[FULL ? E : 1];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float H = dh[i] + r2 * (dy[i] * w2[i]) - h[i] * k2;
                float f = H * w1[i], hb = H * b[i] * r1g;
                if constexpr (FULL) {
                    dg[i] = hb * w1[i];
                    f *= g[i];
                    hb *= g[i];
                }
                dx[i] = a.alpha * H;
                db[i] = r1g * f - b[i] * k1;
                s1[i] += hb;
                s2[i] += dy[i] * h[i] * r2;
            }
            cols.add_store(a.dx + row * D, dx, a.acc & TTK_ACC_DX);
            cols.add_store(a.db + row * D, db, a.acc & TTK_ACC_DB);
            if constexpr (FULL)
                if (a.dgate)
                    cols.add_store(a.dgate + row * D, dg, a.acc & TTK_ACC_DGATE);
            if (lead) {
                const float d = r1 * dot;
                if (a.g.kind == TTK_GATE_ROW && a.dgate)
                    a.dgate[row] = (a.acc & TTK_ACC_DGATE) ? a.dgate[row] + d : d;
                gsum += static_cast<double>(d);
            }
        }
        if (folded) {
            float4* q = reinterpret_cast<float4*>(smem + slots * stages * NT * pitch) + threadIdx.x;
#pragma unroll
            for (int j = 0; j < 2 * NV; ++j, q += blockDim.x) {
                float* v = j < NV ? s1 + 4 * j : s2 + 4 * (j - NV);
                const float4 o = *q;
                v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
                if (row < a.R) {
                    *q = make_float4(v[0], v[1], v[2], v[3]);
                    v[0] = v[1] = v[2] = v[3] = 0.0f;
                }
            }
        }
    }
    // the block's rows, slot by slot, through the stages' memory
    if (slots > 1) {
        __syncthreads();
        if (slot) {
            cols.template store<false>(smem + (2 * slot - 2) * D, s1);
            cols.template store<false>(smem + (2 * slot - 1) * D, s2);
        }
        if (lead)
            s_g[slot] = gsum;
        __syncthreads();
        if (slot == 0)
            for (int q = 1; q < slots; ++q) {
                float o[E];
                cols.template load<false>(o, smem + (2 * q - 2) * D, true);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    s1[i] += o[i];
                cols.template load<false>(o, smem + (2 * q - 1) * D, true);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    s2[i] += o[i];
                if (lead)
                    gsum += s_g[q];
            }
    }
    if (slot == 0) {
        cols.template store<false>(a.part1 + blockIdx.x * D, s1);
        cols.template store<false>(a.part2 + blockIdx.x * D, s2);
        if (lead)
            a.partg[blockIdx.x] = gsum;
    }
}

// Rows too wide for the registers of a block (more than 2048 words), or tensors
// that do not start on a 16-byte boundary: one block per row, each row read once
// per pass over it.
constexpr int WIDE_THREADS = 512;

__global__ void __launch_bounds__(WIDE_THREADS) fwd_wide_kernel(const Fwd a) {
    __shared__ float red[2][MAX_WARPS];
    grid_wait();
    const int64_t D = a.D;
    for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
        const int64_t o = row * D;
        float s[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS)
            s[0] += a.b[o + c] * a.b[o + c];
        row_sum(s, red[0], 0, WIDE_THREADS, true);
        const float r1 = 1.0f / sqrtf(s[0] / static_cast<float>(D) + a.eps);
        s[0] = 0.0f;
        for (int64_t c = threadIdx.x; c < D; c += WIDE_THREADS) {
            const float h = a.alpha * a.x[o + c] + a.g.at(row, c, D) * (a.b[o + c] * r1 * a.w1[c]);
            a.h[o + c] = h;
            s[0] += h * h;
        }
        row_sum(s, red[1], 0, WIDE_THREADS, true);
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
    grid_wait();
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
            s[2] += (h * r2) * k;
        }
        row_sum(s, red[parity], 0, WIDE_THREADS, true);
        const float inv = 1.0f / static_cast<float>(D);
        const float m2 = r2 * (r2 * (inv * s[0])), k2 = r2 * m2;
        const float dot = s[1] - m2 * s[2];
        const float k1 = r1 * (r1 * (r1 * (inv * dot))) * gr;
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
// gradients: 32 columns a block, warp w adds rows w, w + 32, ... and the
// warps' sums are added in order. Bound by latency; 8, 16 or 32 columns with 256
// to 1024 threads, and a tree instead of the last loop, took the same within 1 us.
constexpr int FIN_WARPS = 32;
__global__ void __launch_bounds__(32 * FIN_WARPS) finish_kernel(const Bwd a, int64_t nb, float* dw1,
                                                                float* dw2) {
    __shared__ float red[2][FIN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool accw = a.acc & TTK_ACC_DW, accg = a.acc & TTK_ACC_DGATE;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s1 = 0.0f, s2 = 0.0f;
    grid_wait();
    if (c < a.D) {
#pragma unroll 8
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

// 16-byte words that a row may touch.
int64_t row_words(int64_t D) { return D % 4 ? (D + 6) / 4 : D / 4; }

bool aligned16(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (reinterpret_cast<uintptr_t>(p) & 15)
            return false;
    return true;
}

// The partial sums' places in the workspace, rows first (stored as float4).
void partials(Bwd& a, int64_t nb, void* ws) {
    a.part1 = static_cast<float*>(ws);
    a.part2 = a.part1 + nb * a.D;
    a.partg = reinterpret_cast<double*>(a.part2 + nb * a.D);  // after 2 nb D floats
}

constexpr int64_t MAX_WORDS = 2048;   // widest row kept in registers, in words
constexpr int64_t MAX_BLOCKS = 2048;  // partial rows of the backward
constexpr int SMEM_SM = 228 * 1024;    // shared memory of an SM
constexpr int SMEM_BLOCK = 1792;       // of a block beside its dynamic part (1 KB reserved, static)
constexpr int SMEM_MAX = 226 * 1024;   // dynamic part of one block

// Launch shape of a rows kernel: slots of TPR threads, whole rows each, up to
// 256 threads a block; as many blocks as the registers let an SM hold, and
// the shared memory left to each of them spent on stages.
struct Shape {
    int tpr, slots, threads, pitch, stages;
    bool folded;
    size_t smem;
    int64_t blocks;  // resident at once, or fewer
};

template <auto kernel>
Shape shape_of(int64_t R, int64_t D, int nv, int tensors, bool sums) {
    Shape s;
    s.tpr = static_cast<int>(((row_words(D) + nv - 1) / nv + 31) / 32 * 32);
    s.slots = std::max(1, std::min(MAX_SLOTS, 256 / s.tpr));
    s.threads = s.tpr * s.slots;
    s.pitch = static_cast<int>(row_words(D) * 4);
    // {SMs, blocks per SM} by device and block size, asked for once
    constexpr int kDevs = 16;
    static std::atomic<int> cache[kDevs][17];
    int dev = 0, sms = 0, per = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= kDevs)
        dev = 0;
    std::atomic<int>& c = cache[dev][s.threads / 32];
    const int known = c.load(std::memory_order_relaxed);
    if (known) {
        sms = known >> 8, per = known & 255;
    } else {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            sms = 148;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, s.threads, 0) !=
                cudaSuccess ||
            per <= 0)
            per = 1;
        cudaGetLastError();
        c.store(sms << 8 | per, std::memory_order_relaxed);
    }
    const size_t stage = static_cast<size_t>(s.slots) * tensors * s.pitch * sizeof(float);
    const int64_t rows = (R + static_cast<int64_t>(sms) * per * s.slots - 1) /
                         (static_cast<int64_t>(sms) * per * s.slots);  // per slot
    // where a slot has many rows, room for their sums
    const int64_t folds = static_cast<int64_t>(s.threads) * 2 * nv * 16;
    s.folded = sums && rows > 2 * FOLD;
    const int64_t room = (std::min(SMEM_SM / per - SMEM_BLOCK, SMEM_MAX) - (s.folded ? folds : 0)) /
                         static_cast<int64_t>(stage);
    s.stages = static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>({room, rows, static_cast<int64_t>(MAX_STAGES)})));
    s.smem = stage * s.stages + (s.folded ? folds : 0);
    while (per > 1 && per * (s.smem + SMEM_BLOCK) > SMEM_SM)
        --per;
    s.blocks = std::min({(R + s.slots - 1) / s.slots, MAX_BLOCKS, static_cast<int64_t>(sms) * per});
    // odd widths: the rows of a slot are whole words apart
    const int64_t apart = D % 4 == 0 ? 1 : D % 2 == 0 ? 2 : 4;
    while (s.blocks * s.slots < R && s.blocks * s.slots % apart)
        --s.blocks;
    return s;
}

template <int NV, bool ODD, bool FULL>
int run_fwd(const Fwd& a, cudaStream_t st) {
    const Shape s = shape_of<fwd_rows_kernel<NV, ODD, FULL>>(a.R, a.D, NV, FULL ? 3 : 2, false);
    return launch_pdl("residual_norm_fwd", fwd_rows_kernel<NV, ODD, FULL>,
                      dim3(static_cast<unsigned>(s.blocks)), s.threads, s.smem, st, a, s.tpr, s.pitch,
                      s.stages);
}

template <int NV, bool ODD, bool FULL>
int run_bwd(Bwd& a, int64_t* nb, void* ws, cudaStream_t st) {
    const Shape s = shape_of<bwd_rows_kernel<NV, ODD, FULL>>(a.R, a.D, NV, FULL ? 5 : 4, true);
    *nb = s.blocks;
    partials(a, *nb, ws);
    return launch_pdl("residual_norm_bwd", bwd_rows_kernel<NV, ODD, FULL>,
                      dim3(static_cast<unsigned>(*nb)), s.threads, s.smem, st, a, s.tpr, s.pitch,
                      s.stages, s.folded);
}

// `aligned`: every tensor of the rows starts on a 16-byte boundary.
int dispatch_fwd(const Fwd& a, bool aligned, cudaStream_t st) {
    const int64_t words = row_words(a.D);
    if (!aligned || words > MAX_WORDS)
        return launch_pdl("residual_norm_fwd", fwd_wide_kernel,
                          dim3(static_cast<unsigned>(grid_for(a.R, 1, 148 * 4))), WIDE_THREADS, 0,
                          st, a);
    const bool full = a.g.kind == TTK_GATE_FULL, odd = a.D % 4;
    if (words <= MAX_WORDS / 2) {
        if (odd)
            return full ? run_fwd<2, true, true>(a, st) : run_fwd<2, true, false>(a, st);
        return full ? run_fwd<2, false, true>(a, st) : run_fwd<2, false, false>(a, st);
    }
    if (odd)
        return full ? run_fwd<4, true, true>(a, st) : run_fwd<4, true, false>(a, st);
    return full ? run_fwd<4, false, true>(a, st) : run_fwd<4, false, false>(a, st);
}

int dispatch_bwd(Bwd& a, bool aligned, int64_t* nb, void* ws, cudaStream_t st) {
    const int64_t words = row_words(a.D);
    if (!aligned || words > MAX_WORDS) {
        *nb = std::min<int64_t>(a.R, 296);
        partials(a, *nb, ws);
        return launch_pdl("residual_norm_bwd", bwd_wide_kernel, dim3(static_cast<unsigned>(*nb)),
                          WIDE_THREADS, 0, st, a);
    }
    const bool full = a.g.kind == TTK_GATE_FULL, odd = a.D % 4;
    if (words <= MAX_WORDS / 2) {
        if (odd)
            return full ? run_bwd<2, true, true>(a, nb, ws, st) : run_bwd<2, true, false>(a, nb, ws, st);
        return full ? run_bwd<2, false, true>(a, nb, ws, st) : run_bwd<2, false, false>(a, nb, ws, st);
    }
    if (odd)
        return full ? run_bwd<4, true, true>(a, nb, ws, st) : run_bwd<4, true, false>(a, nb, ws, st);
    return full ? run_bwd<4, false, true>(a, nb, ws, st) : run_bwd<4, false, false>(a, nb, ws, st);
}

}  // namespace resnorm
}  // namespace ttk

using namespace ttk;
using namespace ttk::resnorm;

// Without rows a gate per row or element has no values, and may be null.
static int check_gate(const float* gate, int kind, int64_t R, const char* msg) {
    const bool values = kind == TTK_GATE_SCALAR || kind == TTK_GATE_COLUMN ||
                        (R && kind != TTK_GATE_NONE);
    if (kind < TTK_GATE_NONE || kind > TTK_GATE_FULL || (values && !gate))
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
    if (int rc = check_gate(gate, gate_kind, R, "residual_norm_fwd: bad gate"))
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
    bool aligned = aligned16({x, b, w_post, w_next, h, y});
    if (gate_kind == TTK_GATE_COLUMN || gate_kind == TTK_GATE_FULL)
        aligned = aligned && aligned16({gate});
    const Fwd a{x, b, w_post, Gate{gate, gate_kind}, w_next, h, y, rstd_post, rstd_next,
                static_cast<__nv_bfloat16*>(y_split), R, D, residual_scale, eps};
    return dispatch_fwd(a, aligned, st);
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
    if (int rc = check_gate(gate, gate_kind, R, "residual_norm_bwd: bad gate"))
        return rc;
    if (accumulate & ~(TTK_ACC_DX | TTK_ACC_DB | TTK_ACC_DW | TTK_ACC_DGATE))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: unknown accumulate bits");
    if (!workspace || workspace_bytes < ttk_residual_norm_bwd_workspace_size(R, D) ||
        !aligned16({workspace}))
        return set_error(TTK_ERR_ARG, "residual_norm_bwd: workspace too small or not 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!R) {  // sums of nothing: zeros, or what is there
        auto zero = [&](float* p, int64_t n, int bit) {
            return !p || !n || (accumulate & bit)
                       ? TTK_OK
                       : check_cuda(cudaMemsetAsync(p, 0, static_cast<size_t>(n) * 4, st),
                                    "residual_norm_bwd: zero");
        };
        const int64_t ng = gate_kind == TTK_GATE_SCALAR ? 1 : gate_kind == TTK_GATE_COLUMN ? D : 0;
        int rc = zero(dw_post, D, TTK_ACC_DW);
        if (!rc)
            rc = zero(dw_next, D, TTK_ACC_DW);
        return rc ? rc : zero(dgate, ng, TTK_ACC_DGATE);
    }
    Bwd a{dh, dy, h, b, w_post, Gate{gate, gate_kind}, w_next, rstd_post, rstd_next, dx, db, dgate,
          nullptr, nullptr, nullptr, accumulate, R, D, residual_scale};
    int64_t nb = 0;
    bool aligned = aligned16({dh, dy, b, w_post, dx, db}) && (!dy || aligned16({h, w_next}));
    if (gate_kind == TTK_GATE_COLUMN)
        aligned = aligned && aligned16({gate});
    if (gate_kind == TTK_GATE_FULL)
        aligned = aligned && aligned16({gate, dgate});
    if (int rc = dispatch_bwd(a, aligned, &nb, workspace, st))
        return rc;
    return launch_pdl("residual_norm_bwd sums", finish_kernel,
                      dim3(static_cast<unsigned>((D + 31) / 32)), 32 * FIN_WARPS, 0, st, a, nb,
                      dw_post, dw_next);
}

}  // extern "C"
