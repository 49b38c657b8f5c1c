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
// bytes per logit; next come the exponentials (two temperatures, for the sums
// and again for the gradient: four a logit). So a CTA takes whole rows, and
// its warps have roles:
//   - a producer thread copies the rows, chunk by chunk, into a ring in shared
//     memory, as far ahead as the ring holds (bulk copies);
//   - the compute warps run over a row's chunks twice: a running maximum and
//     the sums, then the gradient without the teacher's and the label's terms.
//     A chunk's place is free for the next row's chunk once its gradient is
//     written, so the copies never pause. Of a row longer than the ring the
//     last chunks stay there and the first in registers; the others are copied
//     again (from L2);
//   - a teacher warp works out the next row's list meanwhile, and writes the
//     listed classes once more after the row, with all their terms.
// Narrow rows run with fewer compute warps and more CTAs to an SM.
// Measured in a CUDA graph, on inputs that are not in L2: 8192 x 32000 at
// temperature 2 with lists of 64, loss and gradient, 385 us, 5.4 TB/s (386 at
// temperature 1, with half the exponentials: they are hidden); 1237 x 49999 with
// lists of 50, rows at any alignment, 107 us, 4.6 TB/s (a CTA has 4.2 rows, so the
// last round leaves most of them idle); loss alone, 4096 x 32000, 98 us, 5.3 TB/s,
// 128 x 32000 10.3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "pdl.cuh"
#include "ttk_common.cuh"
#include "ttk_internal.h"

namespace ttk {
namespace distill {

constexpr int MAX_PLACES = 16;
constexpr int SMEM_SM = 228 * 1024;    // an SM's shared memory
constexpr int SMEM_CTA = 2048;         // of a CTA beside its dynamic part (1 KB reserved, static)
constexpr int SMEM_MAX = 225 * 1024;   // dynamic part of one CTA
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

// Up to AHEAD entries of a lane, 32 apart, of a row's list from k0 on (no class past
// K) and the row's label, as they are in memory: nothing waits for the loads until
// they are used, so a row's are started while the row before is worked on.
constexpr int AHEAD = 4;
struct Entries {
    int id[AHEAD];
    uint32_t z[AHEAD];
    int64_t label;
    __device__ __forceinline__ void load(const Args& a, int64_t row, int k0) {
        const int K = row < a.N ? static_cast<int>(a.K) : 0, lane = threadIdx.x & 31;
        const int64_t at = row * a.K + k0 + lane;
        label = k0 == 0 && row < a.N && a.targets ? a.targets[row] : -1;
        const bool wide = a.top_type == TTK_F32;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            id[i] = -1, z[i] = 0;
            if (k0 + 32 * i < K && k0 + 32 * i + lane < K) {
                id[i] = a.ids[at + 32 * i];
                z[i] = wide ? static_cast<const uint32_t*>(a.top)[at + 32 * i]
                            : static_cast<const uint16_t*>(a.top)[at + 32 * i];
            }
        }
    }
    __device__ __forceinline__ float logit(int i, int type) const {
        return type == TTK_F32    ? __uint_as_float(z[i])
               : type == TTK_BF16 ? __uint_as_float(z[i] << 16)
                                  : __half2float(__ushort_as_half(static_cast<uint16_t>(z[i])));
    }
};

// exp((x - m) / T) as a power of two, c = log2 e / T. The difference is taken
// first: it is exact near the maximum, where the terms that count are, and
// right for rows at the type's lowest value, where x c would overflow.
__device__ __forceinline__ float pow_from(float x, float m, float c) {
    return exp2_approx((x - m) * c);
}
// Where to count from: the maximum, or 0 without one (-inf - -inf is NaN).
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.0f : m; }
constexpr float LN2 = 0.6931471805599453f;

// (maximum, sum at temperature 1, sum at T) of part of a row.
struct Stat {
    float m, s1, sT;
};

// The statistics held by the lanes of a warp, as one, in every lane.
__device__ __forceinline__ Stat warp_merge(const Stat& a, float cT) {
    Stat r;
    r.m = warp_max(a.m);
    const float z = origin(r.m);
    r.s1 = warp_sum(a.s1 * pow_from(a.m, z, LOG2E));
    r.sT = warp_sum(a.sT * pow_from(a.m, z, cT));
    return r;
}

// How a launch cuts its rows.
struct Cut {
    int chunk;   // words of a place
    int places;  // of the ring
    int hash;    // places of the teacher's hash table (a power of two)
};

// One row as words of 16 bytes: `words` of them start at `base`, and the `head`
// classes before and the rest after them, at most three each, are edges.
struct Row {
    const float* x;
    int head, words, chunks, keep;  // keep: last chunks that stay for the gradient
    __device__ __forceinline__ Row(const Args& a, int64_t row) : chunks(0), keep(0) {
        x = a.logits + row * a.ld;
        const int C = static_cast<int>(a.C);
        head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) >> 2, C);
        words = (C - head) >> 2;
    }
    __device__ __forceinline__ Row(const Args& a, const Cut& cut, int64_t row) : Row(a, row) {
        chunks = (words + cut.chunk - 1) / cut.chunk;
        keep = a.dlogits ? min(chunks, cut.places) : 0;
    }
    // chunks that did not stay, the first aside
    __device__ __forceinline__ int again(const Args& a) const {
        return a.dlogits ? max(chunks - keep - 1, 0) : 0;
    }
};

__device__ __forceinline__ float weight_of(const Args& a, int64_t row) {
    return a.row_weight && row < a.N ? a.row_weight[row] : 1.0f;
}

// What the compute warps hand to the teacher warp after a row's sums.
struct RowSums {
    float m, log1, logT, k1, kk;
    int kind;
};

// The gradient of a class without the listed terms: kind 0 none, 1 one
// temperature, 2 both.
__device__ __forceinline__ float base_grad(const RowSums& r, float x, float cT) {
    return r.kind == 0   ? 0.0f
           : r.kind == 1 ? r.kk * pow_from(x, r.m, cT)
                         : fmaf(r.k1, pow_from(x, r.m, LOG2E), r.kk * pow_from(x, r.m, cT));
}

// A teacher list in shared memory (two of them, for rows in turn).
struct List {
    int *id, *to;        // class, -1 for none; class from its first entry, else -1
    float *p, *a, *x;    // probability, log p, the student's logit
    float* sum;          // probability of all entries of the class (first entry)
    __device__ __forceinline__ List(float* at, int pad) {
        id = reinterpret_cast<int*>(at), to = id + pad;
        p = at + 2 * pad, a = p + pad, x = a + pad, sum = x + pad;
    }
};
constexpr int LIST_ARRAYS = 6;

struct Flags {
    int has, t;    // entries; the label's class or -1
    float x_t;     // its logit
    float w;       // the row's weight
    bool t_listed;
};

// Whether a class is in the list more than once. Up to 32 entries are compared
// lane with lane. More go through a table, in rounds: every entry that is
// still open puts its number into the table at its class's hash and reads what
// stands there: its own number or that of another entry of its class settle it,
// and that of another class leaves it open. Entries of one class share a place in
// every round, so none is missed; a place settles at least the entry that it
// holds, so the rounds end. The same in every lane.
__device__ __forceinline__ bool listed_twice(const List& l, int K, int* table, int size) {
    const int lane = threadIdx.x & 31;
    if (K <= 32) {
        const int id = lane < K && l.id[lane] >= 0 ? l.id[lane] : -1 - lane;
        return __any_sync(~0u, __match_any_sync(~0u, id) != 1u << lane);
    }
    uint32_t open = 0;  // bit i: entry 32 i + lane
#pragma unroll 4
    for (int k = lane; k < K; k += 32)
        if (l.id[k] >= 0)
            open |= 1u << (k >> 5);
    bool twice = false;
    for (uint32_t factor = 2654435761u; __any_sync(~0u, open != 0 && !twice); factor *= 0x9e3779b1u) {
        auto place = [&](int k) { return (static_cast<uint32_t>(l.id[k]) * factor >> 16) & (size - 1); };
#pragma unroll 4
        for (int k = lane; k < K; k += 32)
            if (open >> (k >> 5) & 1u)
                table[place(k)] = k;
        __syncwarp();
#pragma unroll 4
        for (int k = lane; k < K; k += 32)
            if (open >> (k >> 5) & 1u) {
                const int other = table[place(k)];
                if (l.id[other] == l.id[k]) {
                    twice = twice || other != k;
                    open &= ~(1u << (k >> 5));
                }
            }
        __syncwarp();
    }
    return __any_sync(~0u, twice);
}

// The teacher warp's work before a row's sums are known. `first` holds the row's
// first entries and, with NEXT, gets those of the row `next`; the student's logits of the
// first entries are waited for last.
template <bool NEXT>
__device__ __forceinline__ void teacher_prepare(const Args& a, const Cut& cut, int64_t row, int64_t next, float w,
                                const List& l, int* __restrict__ hash, Flags* flags,
                                Entries& first) {
    const int lane = threadIdx.x & 31, K = static_cast<int>(a.K), C = static_cast<int>(a.C);
    const float invT = 1.0f / a.temperature;
    const float* x = a.logits + row * a.ld;
    const int64_t label = first.label;
    float zmax = -INFINITY, x_first[AHEAD];
    auto take = [&](const Entries& e, int k0, float (&xs)[AHEAD]) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = k0 + 32 * i + lane;
            xs[i] = 0.0f;
            if (k0 + 32 * i < K) {
                int id = e.id[i];
                if (static_cast<unsigned>(id) >= static_cast<unsigned>(C)) {
                    if (id != -1)
                        report(kErrBadIndex);
                    id = -1;
                }
                if (id >= 0)
                    xs[i] = x[id];
                const float v = id >= 0 ? e.logit(i, a.top_type) : -INFINITY;
                if (k < K) {
                    l.id[k] = l.to[k] = id;
                    l.a[k] = v;
                }
                // NaN counts as present: it has to reach the row's result
                zmax = fmaxf(zmax, v != v ? INFINITY : v);
            }
        }
    };
    take(first, 0, x_first);
    for (int k0 = 32 * AHEAD; k0 < K; k0 += 32 * AHEAD) {
        float xs[AHEAD];
        first.load(a, row, k0);
        take(first, k0, xs);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (k0 + 32 * i + lane < K)
                l.x[k0 + 32 * i + lane] = xs[i];
    }
    const int t = label >= 0 && label < C ? static_cast<int>(label) : -1;
    if (t < 0 && label != -1 && lane == 0)
        report(kErrBadIndex);
    const float x_t = t >= 0 ? x[t] : 0.0f;
    if constexpr (NEXT)
        first.load(a, next, 0);
    zmax = warp_max(zmax);
    const bool has = zmax > -INFINITY;
    __syncwarp();
    float sz = 0.0f;
    bool on_t = false;
#pragma unroll 4
    for (int k = lane; k < K; k += 32) {
        // the difference first, as for the student's logits: z / T may overflow, and
        // its rounding grows with z (a division by T instead of the product: 202
        // instead of 185 us at 4096 x 16000 with lists of 250)
        const float d = has ? (l.a[k] - zmax) * invT : 0.0f, e = has ? expf(d) : 0.0f;
        l.a[k] = d;
        l.p[k] = e;
        sz += e;
        on_t = on_t || (t >= 0 && l.id[k] == t);
    }
    const bool twice = listed_twice(l, K, hash, cut.hash);
    sz = warp_sum(sz);
    const float logz = logf(sz), invz = 1.0f / sz;
#pragma unroll 4
    for (int k = lane; k < K; k += 32) {
        l.p[k] = l.sum[k] = has ? l.p[k] * invz : 0.0f;
        l.a[k] = has ? l.a[k] - logz : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (32 * i < K && 32 * i + lane < K)
            l.x[32 * i + lane] = x_first[i];
    __syncwarp();
    if (twice)
        // the first entry of a class carries all of its entries, in list order
        for (int k = lane; k < K; k += 32) {
            const int id = l.id[k];
            if (id < 0)
                continue;
            bool first = true;
            float sum = 0.0f;
            for (int j = 0; j < K; ++j)
                if (l.id[j] == id) {
                    first = first && j >= k;
                    sum += l.p[j];
                }
            l.sum[k] = sum;
            l.to[k] = first ? id : -1;
        }
    on_t = __any_sync(~0u, on_t);
    if (lane == 0)
        *flags = Flags{has, t, x_t, w, on_t};
    __syncwarp();
}

// The teacher warp's work after a row: its loss terms, and the gradient of the
// listed classes and of the label.
__device__ void teacher_finish(const Args& a, int64_t row, const List& l, const Flags& f,
                               const RowSums& r, float cT, bool write) {
    const int lane = threadIdx.x & 31, K = static_cast<int>(a.K);
    const float w = f.w, gs = a.grad_scale * w;
    const float gT = f.has ? gs * a.alpha * a.temperature : 0.0f;
    const float g1 = f.t >= 0 ? gs * (1.0f - a.alpha) : 0.0f, invT = 1.0f / a.temperature;
    float* dr = a.dlogits + row * a.ldd;
    float kd = 0.0f;
    for (int k = lane; k < K; k += 32) {
        if (l.id[k] >= 0 && l.p[k] != 0.0f)
            kd += l.p[k] * (l.a[k] - ((l.x[k] - r.m) * invT - LN2 * r.logT));
        if (a.dlogits && write && l.to[k] >= 0)
            dr[l.to[k]] =
                base_grad(r, l.x[k], cT) - (gT * l.sum[k] + (l.to[k] == f.t ? g1 : 0.0f));
    }
    kd = warp_sum(kd);
    if (lane == 0) {
        // not times log2 e and back: a label at the type's lowest value would overflow
        const float ce = f.t >= 0 ? LN2 * r.log1 - (f.x_t - r.m) : 0.0f;
        if (a.dlogits && write && f.t >= 0 && !f.t_listed)
            dr[f.t] = base_grad(r, f.x_t, cT) - g1;
        a.terms[2 * row] = r.kind ? static_cast<double>(w) * kd : 0.0;
        a.terms[2 * row + 1] = r.kind ? static_cast<double>(w) * ce : 0.0;
    }
}

// Adds G words to a thread's sums. They are relative to a reference st.m that is
// raised, and the sums with it, only when a value passes it by 2^16 or more: any
// reference that keeps the terms in range serves as well as the maximum.
template <bool TWO, int G>
__device__ __forceinline__ void push(Stat& st, const float4 (&v)[G], float slack, float cT) {
    float top = fmaxf(max3(v[0].x, v[0].y, v[0].z), v[0].w);
#pragma unroll
    for (int j = 1; j < G; ++j)
        top = max3(max3(top, v[j].x, v[j].y), v[j].z, v[j].w);
    if (!(top <= st.m + slack) && top > st.m) {
        if (st.m > -INFINITY) {
            st.s1 *= pow_from(st.m, top, LOG2E);
            st.sT *= pow_from(st.m, top, cT);
        }
        st.m = top;
    }
    const float z = origin(st.m);
#pragma unroll
    for (int j = 0; j < G; ++j) {
        if constexpr (TWO)
            st.s1 += (pow_from(v[j].x, z, LOG2E) + pow_from(v[j].y, z, LOG2E)) +
                     (pow_from(v[j].z, z, LOG2E) + pow_from(v[j].w, z, LOG2E));
        st.sT += (pow_from(v[j].x, z, cT) + pow_from(v[j].y, z, cT)) +
                 (pow_from(v[j].z, z, cT) + pow_from(v[j].w, z, cT));
    }
}
__device__ __forceinline__ float slack_of(float cT) { return 16.0f / fmaxf(cT, LOG2E); }

// A thread's sums before its first word: its edge class, or nothing (-inf).
__device__ __forceinline__ Stat first_stat(float x, float cT) {
    const float e = pow_from(x, origin(x), cT);  // 1; 0 of -inf; NaN
    return Stat{fmaxf(x, -INFINITY), e, e};
}

// What follows from a row's sums.
template <bool TWO>
__device__ __forceinline__ RowSums row_sums(const Args& a, const Stat& st, float w, bool has,
                                            bool t_ok) {
    const float gs = a.grad_scale * w;
    const float k1 = t_ok ? gs * (1.0f - a.alpha) / st.s1 : 0.0f;
    const float kT = has ? gs * a.alpha * a.temperature / st.sT : 0.0f;
    return RowSums{st.m, log2f(st.s1), log2f(st.sT), k1, TWO ? kT : k1 + kT,
                   !has && !t_ok ? 0 : !TWO || k1 == 0.0f ? 1 : 2};
}

// The gradient of one word, without the listed terms (base_grad). ALIGNED: the
// gradient's words are aligned as the logits' are.
template <int KIND, bool ALIGNED>
__device__ __forceinline__ void put(float* out, const float4& v, const RowSums& r, float cT) {
    const float e[4] = {v.x, v.y, v.z, v.w};
    float g[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        g[u] = KIND == 0   ? 0.0f
               : KIND == 1 ? r.kk * pow_from(e[u], r.m, cT)
                           : fmaf(r.k1, pow_from(e[u], r.m, LOG2E), r.kk * pow_from(e[u], r.m, cT));
    if (ALIGNED)
        *reinterpret_cast<float4*>(out) = make_float4(g[0], g[1], g[2], g[3]);
    else
        out[0] = g[0], out[1] = g[1], out[2] = g[2], out[3] = g[3];
}

// f(kind, aligned) with both as constants of the type.
template <class F>
__device__ __forceinline__ void by_kind(int kind, bool aligned, const F& f) {
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    if (kind == 0)
        f(I0{}, std::false_type{});
    else if (kind == 1 && aligned)
        f(I1{}, std::true_type{});
    else if (kind == 1)
        f(I1{}, std::false_type{});
    else if (aligned)
        f(I2{}, std::true_type{});
    else
        f(I2{}, std::false_type{});
}

// TWO: both temperatures' sums are needed; otherwise T alone (T = 1, or no
// labels). Waits are bounded: a thread whose wait ran out (`ok` false) waits no
// more and writes nothing, but passes every barrier, so the CTA ends.
template <bool TWO, int WARPS, int GROUP, int CTAS>
__global__ void __launch_bounds__(32 * (WARPS + 2), CTAS)
    row_kernel(const Args a, const Cut cut) {
    extern __shared__ __align__(16) float dyn[];
    __shared__ __align__(8) uint64_t full[MAX_PLACES], empty[MAX_PLACES];
    __shared__ __align__(8) uint64_t listed[2], stored[2];
    __shared__ Stat s_warp[2][WARPS];
    __shared__ RowSums s_sums[2];
    __shared__ Flags s_flags[2];
    constexpr int THREADS = 32 * WARPS;  // compute threads
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int pad = static_cast<int>(a.K + 3) / 4 * 4;
    float4* const ring = reinterpret_cast<float4*>(dyn);
    float* const lists = dyn + 4 * cut.places * cut.chunk;
    int* const hash = reinterpret_cast<int*>(lists + 2 * LIST_ARRAYS * pad);
    const float cT = LOG2E / a.temperature;
    if (tid == 0) {
        for (int i = 0; i < cut.places; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(listed + i, 1);
            mbar_init(stored + i, WARPS);
        }
        fence_barrier_init();
    }
    __syncthreads();
    grid_wait();
    bool ok = true;
    if (warp == WARPS) {
        // ---------------------------------------------------------- producer
        if (lane == 0) {
            int place = 0;
            uint32_t phase = 0, in_use = 0, last = 0;  // bits per place
            float w_next = weight_of(a, blockIdx.x);
            for (int64_t row = blockIdx.x; row < a.N && ok; row += gridDim.x) {
                const float w = w_next;
                w_next = weight_of(a, row + gridDim.x);
                if (w == 0.0f)
                    continue;
                const Row r(a, cut, row);
                const int copies = r.chunks + r.again(a);
                const float4* src = reinterpret_cast<const float4*>(r.x + r.head);
                for (int q = 0; q < copies; ++q) {
                    const int w0 = (q < r.chunks ? q : q - r.chunks + 1) * cut.chunk;
                    const uint32_t bytes = static_cast<uint32_t>(min(cut.chunk, r.words - w0)) * 16u;
                    ok = mbar_wait(empty + place, phase ^ 1u, 100);
                    if (!ok)
                        break;
                    fence_async_smem();
                    mbar_arrive_expect_tx(full + place, bytes);
                    bulk_load(ring + place * cut.chunk, src + w0, bytes, full + place);
                    in_use |= 1u << place;
                    last = (last & ~(1u << place)) | phase << place;
                    if (++place == cut.places)
                        place = 0, phase ^= 1u;
                }
            }
            // every copy has landed before the CTA ends
            for (int i = 0; i < cut.places; ++i)
                if (in_use >> i & 1u)
                    mbar_wait(full + i, last >> i & 1u, 101);
        }
    } else if (warp == WARPS + 1) {
        // ----------------------------------------------------------- teacher
        int64_t before = -1;  // the row before, not finished yet
        int n = 0;
        float w_next = weight_of(a, blockIdx.x);
        Entries ahead;
        ahead.load(a, blockIdx.x, 0);
        for (int64_t row = blockIdx.x;; row += gridDim.x) {
            const bool more = row < a.N;
            const float w = w_next;
            w_next = weight_of(a, row + gridDim.x);
            const bool work = more && w != 0.0f;
            if (work) {
                const int b = n & 1;
                teacher_prepare<true>(a, cut, row, row + gridDim.x, w,
                                List(lists + b * LIST_ARRAYS * pad, pad), hash, s_flags + b, ahead);
                if (lane == 0)
                    mbar_arrive(listed + b);
            } else if (more) {
                ahead.load(a, row + gridDim.x, 0);
                if (lane == 0)
                    a.terms[2 * row] = a.terms[2 * row + 1] = 0.0;
            }
            if ((work || !more) && before >= 0) {
                const int m = n - 1, b = m & 1;
                ok = ok && mbar_wait(stored + b, m >> 1 & 1, 102);
                ok = __all_sync(~0u, ok);
                teacher_finish(a, before, List(lists + b * LIST_ARRAYS * pad, pad), s_flags[b],
                               s_sums[b], cT, ok);
                __syncwarp();
            }
            if (!more)
                break;
            if (work)
                before = row, ++n;
        }
    } else {
        // ----------------------------------------------------------- compute
        int place = 0, n = 0;
        uint32_t phase = 0;
        const float slack = slack_of(cT);
        // This thread's edge class of a row (threads 0..2 before the words, 3..5
        // after them) and the row's weight, read a row ahead.
        auto edge_of = [&](const Row& r) {
            const int e = tid < 3 ? (tid < r.head ? tid : -1) : r.head + 4 * r.words + tid - 3;
            return tid < 6 && e < static_cast<int>(a.C) ? e : -1;
        };
        float w_next = 1.0f, x_next = -INFINITY;
        auto look = [&](int64_t row) {
            if (row >= a.N)
                return;
            w_next = weight_of(a, row);
            const Row r(a, cut, row);
            const int e = edge_of(r);
            x_next = e >= 0 ? r.x[e] : -INFINITY;
        };
        look(blockIdx.x);
        for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
            const Row r(a, cut, row);
            const float w = w_next, x_edge = x_next;
            float* const dr = a.dlogits + row * a.ldd;
            const bool same = ((reinterpret_cast<uintptr_t>(r.x) ^ reinterpret_cast<uintptr_t>(dr)) & 15) == 0;
            const int edge = edge_of(r);
            look(row + gridDim.x);
            if (w == 0.0f) {
                if (a.dlogits && ok) {
                    for (int i = tid; i < 4 * r.words; i += THREADS)
                        dr[r.head + i] = 0.0f;
                    if (edge >= 0)
                        dr[edge] = 0.0f;
                }
                continue;
            }
            const int b = n & 1;
            Stat st = first_stat(x_edge, cT);
            float4 held[GROUP];  // the first chunk
            int at = place;
            uint32_t ph = phase;
            for (int c = 0; c < r.chunks; ++c) {
                ok = ok && mbar_wait(full + at, ph, 103);
                const float4* buf = ring + at * cut.chunk;
                const int words = min(cut.chunk, r.words - c * cut.chunk);
                float4 v[GROUP];
                if (words == GROUP * THREADS) {
#pragma unroll
                    for (int j = 0; j < GROUP; ++j)
                        v[j] = buf[tid + j * THREADS];
                    push<TWO>(st, v, slack, cT);
                } else {
#pragma unroll
                    for (int j = 0; j < GROUP; ++j)
                        v[j] = tid + j * THREADS < words
                                   ? buf[tid + j * THREADS]
                                   : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    push<TWO>(st, v, slack, cT);
                }
                if (c == 0)
#pragma unroll
                    for (int j = 0; j < GROUP; ++j)
                        held[j] = v[j];
                if (c < r.chunks - r.keep) {
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(empty + at);
                }
                if (++at == cut.places)
                    at = 0, ph ^= 1u;
            }
            if constexpr (!TWO)
                st.s1 = st.sT;
            st = warp_merge(st, cT);
            if (lane == 0)
                s_warp[b][warp] = st;
            // two buffers: the next row's write comes after its own barrier
            asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
            const Stat none{-INFINITY, 0.0f, 0.0f};
            st = warp_merge(lane < WARPS ? s_warp[b][lane] : none, cT);
            ok = ok && mbar_wait(listed + b, n >> 1 & 1, 104);
            const RowSums sums = row_sums<TWO>(a, st, w, s_flags[b].has, s_flags[b].t >= 0);
            if (tid == 0)
                s_sums[b] = sums;
            if (a.dlogits) {
                // the first chunk, those that stayed, then the others again
                at = place + (r.chunks - r.keep) % cut.places;
                ph = phase ^ ((r.chunks - r.keep) / cut.places & 1);
                if (at >= cut.places)
                    at -= cut.places, ph ^= 1u;
                by_kind(sums.kind, same, [&](auto kind, auto aligned) {
                    constexpr int KIND = decltype(kind)::value;
                    constexpr bool ALIGNED = decltype(aligned)::value;
                    if (r.chunks > r.keep && ok) {
                        float* out = dr + r.head + 4 * tid;
#pragma unroll
                        for (int j = 0; j < GROUP; ++j)
                            if (tid + j * THREADS < cut.chunk)
                                put<KIND, ALIGNED>(out + 4 * j * THREADS, held[j], sums, cT);
                    }
                    for (int q = r.chunks - r.keep; q < r.chunks + r.again(a); ++q) {
                        const int w0 = (q < r.chunks ? q : q - r.chunks + 1) * cut.chunk;
                        if (q >= r.chunks)
                            ok = ok && mbar_wait(full + at, ph, 105);
                        const float4* buf = ring + at * cut.chunk + tid;
                        const int words = ok ? min(cut.chunk, r.words - w0) : 0;
                        float* out = dr + r.head + 4 * (w0 + tid);
                        if (words == GROUP * THREADS) {
#pragma unroll
                            for (int j = 0; j < GROUP; ++j)
                                put<KIND, ALIGNED>(out + 4 * j * THREADS, buf[j * THREADS], sums, cT);
                        } else {
#pragma unroll
                            for (int j = 0; j < GROUP; ++j)
                                if (tid + j * THREADS < words)
                                    put<KIND, ALIGNED>(out + 4 * j * THREADS, buf[j * THREADS], sums,
                                                       cT);
                        }
                        __syncwarp();
                        if (lane == 0)
                            mbar_arrive(empty + at);
                        if (++at == cut.places)
                            at = 0, ph ^= 1u;
                    }
                });
                if (edge >= 0 && ok)
                    dr[edge] = base_grad(sums, x_edge, cT);
            }
            place = at, phase = ph;
            __syncwarp();
            if (lane == 0)
                mbar_arrive(stored + b);
            ++n;
        }
    }
}

// Many narrow rows: a warp takes a row, with all of the above in turn, and reads
// it twice (the second time from L2). A row then costs a warp its latencies
// only, and 32 warps of an SM hide those.
constexpr int NARROW_WARPS = 4;  // of a CTA
constexpr int NARROW_GROUP = 4;
template <bool TWO>
__global__ void __launch_bounds__(32 * NARROW_WARPS, 8) narrow_kernel(const Args a, const Cut cut) {
    extern __shared__ __align__(16) float dyn[];
    __shared__ Flags s_flags[NARROW_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pad = static_cast<int>(a.K + 3) / 4 * 4;
    float* const mine = dyn + warp * (LIST_ARRAYS * pad + cut.hash);
    const List l(mine, pad);
    const float cT = LOG2E / a.temperature, slack = slack_of(cT);
    grid_wait();
    const int64_t step = static_cast<int64_t>(gridDim.x) * NARROW_WARPS;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * NARROW_WARPS + warp; row < a.N; row += step) {
        const Row r(a, row);
        const int C = static_cast<int>(a.C);
        float* const dr = a.dlogits + row * a.ldd;
        const float w = weight_of(a, row);
        if (w == 0.0f) {
            if (a.dlogits)
                for (int i = lane; i < C; i += 32)
                    dr[i] = 0.0f;
            if (lane == 0)
                a.terms[2 * row] = a.terms[2 * row + 1] = 0.0;
            continue;
        }
        const int e = lane < 3 ? (lane < r.head ? lane : -1) : r.head + 4 * r.words + lane - 3;
        const int edge = lane < 6 && e < C ? e : -1;
        const float x_edge = edge >= 0 ? r.x[edge] : -INFINITY;
        Entries first;
        first.load(a, row, 0);
        teacher_prepare<false>(a, cut, row, 0, w, l,
                               reinterpret_cast<int*>(mine + LIST_ARRAYS * pad), s_flags + warp, first);
        const Flags f = s_flags[warp];
        Stat st = first_stat(x_edge, cT);
        const float4* x4 = reinterpret_cast<const float4*>(r.x + r.head);
        for (int i = lane; i < r.words; i += 32 * NARROW_GROUP) {
            float4 v[NARROW_GROUP];
#pragma unroll
            for (int j = 0; j < NARROW_GROUP; ++j)
                v[j] = i + 32 * j < r.words
                           ? x4[i + 32 * j]
                           : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            push<TWO>(st, v, slack, cT);
        }
        if constexpr (!TWO)
            st.s1 = st.sT;
        st = warp_merge(st, cT);
        const RowSums sums = row_sums<TWO>(a, st, w, f.has, f.t >= 0);
        if (a.dlogits) {
            const bool same = ((reinterpret_cast<uintptr_t>(r.x) ^ reinterpret_cast<uintptr_t>(dr)) & 15) == 0;
            float* out = dr + r.head;
            if (sums.kind == 0) {
                for (int i = lane; i < 4 * r.words; i += 32)
                    out[i] = 0.0f;
            } else {
                // one loop for both kinds and alignments: this kernel's time goes
                // by its instructions, those that miss the cache among them
#pragma unroll 2
                for (int i = lane; i < r.words; i += 32) {
                    const float4 v = x4[i];
                    const float e[4] = {v.x, v.y, v.z, v.w};
                    float g[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        g[u] = sums.kk * pow_from(e[u], sums.m, cT);
                    if (sums.kind == 2)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            g[u] = fmaf(sums.k1, pow_from(e[u], sums.m, LOG2E), g[u]);
                    float* d = out + 4 * i;
                    if (same)
                        *reinterpret_cast<float4*>(d) = make_float4(g[0], g[1], g[2], g[3]);
                    else
                        d[0] = g[0], d[1] = g[1], d[2] = g[2], d[3] = g[3];
                }
            }
            if (edge >= 0)
                dr[edge] = base_grad(sums, x_edge, cT);
        }
        __syncwarp();
        teacher_finish(a, row, l, f, sums, cT, true);
        __syncwarp();
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

// Rows of up to this many classes go to narrow_kernel, if there are enough of
// them (at 16384 rows, temperature 2, list of 16: 1500 classes 60 us against 128
// by row_kernel, 3200 classes 118 against 145, 4000 classes 160 against 147;
// 300 rows of 1000 classes 40 against 26).
constexpr int64_t NARROW_MAX = 3584;
constexpr int64_t NARROW_ROWS = 148 * 8;

// How many CTAs share an SM: more of them hide the barriers between a row's two
// passes, fewer hold more of a row. As many as leave a row within 1.4 of their
// rings (8192 rows, temperature 2: 10000 classes 154 us with 8 against 163 with
// 4; 16000 classes 215 with 4 against 257 with 2; 20000 classes 269 against 262).
// Without a gradient nothing has to stay, and 4 were best (4096 x 32000: 104 us
// against 126 with 2). Compute warps and words per thread were swept for each.
template <bool TWO, int WARPS, int GROUP, int CTAS>
int launch(const Args& a, Cut cut, int64_t list_bytes, cudaStream_t st) {
    static std::atomic<int> known[16];      // SMs by device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 16)
        dev = 0;
    int sms = known[dev].load(std::memory_order_relaxed);
    if (!sms) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            sms = 148;
        const cudaError_t e = cudaFuncSetAttribute(
            row_kernel<TWO, WARPS, GROUP, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
        if (e != cudaSuccess)
            return check_cuda(e, "distill_loss");
        known[dev].store(sms, std::memory_order_relaxed);
    }
    const int64_t words = (a.C + 3) / 4, room = SMEM_SM / CTAS - SMEM_CTA - list_bytes;
    // a chunk gives every thread GROUP words; narrow rows have four chunks still
    cut.chunk = static_cast<int>(std::min<int64_t>(
        32 * WARPS * GROUP, std::max<int64_t>(32, ((words + 3) / 4 + 31) / 32 * 32)));
    cut.places = static_cast<int>(
        std::min<int64_t>(MAX_PLACES, std::max<int64_t>(2, room / (16 * cut.chunk))));
    const size_t smem = static_cast<size_t>(cut.places) * cut.chunk * 16 + list_bytes;
    const int64_t blocks = std::min<int64_t>(a.N, static_cast<int64_t>(sms) * CTAS);
    return launch_pdl("distill_loss", row_kernel<TWO, WARPS, GROUP, CTAS>, dim3(static_cast<unsigned>(blocks)),
                      32 * (WARPS + 2), smem, st, a, cut);
}

template <bool TWO>
int launch_rows(const Args& a, cudaStream_t st) {
    const int64_t words = (a.C + 3) / 4, pad = (a.K + 3) / 4 * 4;
    Cut cut;
    cut.hash = 32;
    while (cut.hash < 2 * a.K)
        cut.hash *= 2;
    const int64_t list_bytes = (2 * LIST_ARRAYS * pad + cut.hash) * 4;
    if (a.C <= NARROW_MAX && a.N >= NARROW_ROWS) {
        cut.chunk = 1, cut.places = 1;
        const size_t smem = static_cast<size_t>(NARROW_WARPS) * (LIST_ARRAYS * pad + cut.hash) * 4;
        if (smem > 48 * 1024) {
            const cudaError_t e = cudaFuncSetAttribute(
                narrow_kernel<TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
            if (e != cudaSuccess)
                return check_cuda(e, "distill_loss");
        }
        const int64_t blocks = std::min<int64_t>((a.N + NARROW_WARPS - 1) / NARROW_WARPS, 148 * 8);
        return launch_pdl("distill_loss", narrow_kernel<TWO>, dim3(static_cast<unsigned>(blocks)),
                          32 * NARROW_WARPS, smem, st, a, cut);
    }
    auto fits = [&](int ctas) {
        return words * 16 * 10 / 14 <= SMEM_SM / ctas - SMEM_CTA - list_bytes;
    };
    // Few rows, one to a CTA: the threads of a CTA hold the time down, not the
    // CTAs of an SM. Measured with 8 warps / as the rules below choose: 128 rows
    // of 32000 without a gradient 8.7 / 11.3 us, of 8192 with one 8.9 / 11.5 us,
    // 296 of 32000 10.2 / 12.4 us; 592 of 32000 16.1 / 14.4 us.
    if (a.N <= 2 * 148)
        return launch<TWO, 8, 4, 2>(a, cut, list_bytes, st);
    if (fits(8))
        return launch<TWO, 2, 4, 8>(a, cut, list_bytes, st);
    if (fits(4) || !a.dlogits)
        return launch<TWO, 4, 6, 4>(a, cut, list_bytes, st);
    return launch<TWO, 8, 4, 2>(a, cut, list_bytes, st);
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
