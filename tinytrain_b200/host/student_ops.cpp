// Scaled embedding, residual norm and distillation loss as graph nodes (the
// operators of a distilled student; no counterparts in the reference). Each
// backward accumulates into the inputs' gradients like the other ops' do, and
// writes instead where a gradient is still logically zero.
#include <algorithm>
#include <memory>
#include <stdexcept>

#include "internal.h"
#include "tinytrain/ops.h"
#include "ttk.h"

namespace tt {

using namespace detail;

namespace {

float* out_ptr(Tensor& t) { return t.impl()->data->device_for_overwrite(); }

// Where a kernel writes the gradient of `p`: the gradient itself, or scratch
// that deliver() adds to it afterwards (a tensor that is an input twice) or
// drops (one that needs no gradient).
struct GradDst {
    ImplPtr p;
    bool direct = false, overwrite = true;
    std::unique_ptr<Scratch> scratch;
    float* ptr = nullptr;

    GradDst(const ImplPtr& impl, bool twice) : p(impl) {
        if (p->requires_grad && !twice) {
            direct = true;
            ptr = grad_target(p, overwrite);
        } else {
            scratch.reset(new Scratch(static_cast<size_t>(p->numel) * 4));
            ptr = scratch->as<float>();
        }
    }
    void deliver() {
        if (!direct && p->requires_grad)
            check(ttk_axpy(1.0f, ptr, grad_rmw(p), p->numel, stream()), "grad axpy");
    }
};

}  // namespace

Tensor embedding_scaled(const Tensor& weight, const DeviceIds& idx, float scale) {
    if (weight.ndim() != 2)
        throw std::invalid_argument("embedding: weight must be 2D");
    const int64_t V = weight.dim(0), D = weight.dim(1), N = idx.size();
    if (N <= 0)
        throw std::invalid_argument("Tensor: dims must be positive");
    Tensor out = make_out({N, D}, weight.requires_grad());
    check(ttk_embedding_scaled_fwd(dread(weight.impl()), idx.data(), out_ptr(out), N, D, V, scale,
                                   stream()),
          "embedding_scaled");
    if (out.requires_grad()) {
        auto wo = weight.impl();
        Tensor::Impl* oo = out.impl().get();  // own node: raw, no cycle
        oo->prev = {wo};
        oo->backward_fn = [wo, oo, idx, N, D, V, scale]() {
            const float* g = grad_in(oo);
            if (!g || !wo->requires_grad)
                return;
            const size_t ws = ttk_embedding_scaled_bwd_workspace_size(N, D, V);
            Scratch w(ws);
            bool ow = false;
            float* d = grad_target(wo, ow);
            check(ttk_embedding_scaled_bwd(g, idx.data(), d, ow ? 0 : 1, N, D, V, scale, w.ptr, ws,
                                           stream()),
                  "embedding_scaled bwd");
        };
    }
    return out;
}

ResidualNorm residual_norm(const Tensor& x, const Tensor& block, const Tensor& w_post,
                           const Tensor& w_next, const Tensor& gate, float residual_scale,
                           float eps) {
    if (x.shape() != block.shape())
        throw std::invalid_argument("residual_norm: x and block must be alike");
    const int64_t D = x.dim(x.ndim() - 1), R = x.numel() / D;
    auto width = [&](const Tensor& w) { return w.ndim() == 1 && w.dim(0) == D; };
    if (!width(w_post) || !width(w_next))
        throw std::invalid_argument("residual_norm: weights must be [D]");
    const ImplPtr go = gate.impl();
    int kind = TTK_GATE_NONE;
    if (go) {
        const auto& s = gate.shape();
        if (s.size() == 1 && s[0] == 1)
            kind = TTK_GATE_SCALAR;
        else if (width(gate))
            kind = TTK_GATE_COLUMN;
        else if (s.size() == 2 && s[0] == R && s[1] == 1)
            kind = TTK_GATE_ROW;
        else if (gate.shape() == x.shape())
            kind = TTK_GATE_FULL;
        else
            throw std::invalid_argument("residual_norm: gate must be [1], [D], [R,1] or like x");
    }
    const bool rg = x.requires_grad() || block.requires_grad() || w_post.requires_grad() ||
                    w_next.requires_grad() || (go && go->requires_grad);
    ResidualNorm out{make_out(x.shape(), rg), make_out(x.shape(), rg)};
    auto r1 = std::make_shared<Buffer>(R), r2 = std::make_shared<Buffer>(R);
    // y large enough to feed tensor-core GEMMs gets its bf16x3 operand planes
    // from the same kernel, cached on its buffer as linear() looks them up.
    void* planes = nullptr;
    float* y = out_ptr(out.y);
    Buffer& yb = *out.y.impl()->data;
    if (D % 32 == 0 && R * D >= (1 << 20) && ttk_gemm_get_precision() == 0) {
        const size_t bytes = ttk_gemm_split_bytes(1, R, D);
        if (yb.split_bytes < bytes) {
            ttk_free(yb.split_dev, stream());
            yb.split_dev = nullptr;
            yb.split_bytes = 0;
            check(ttk_malloc(&yb.split_dev, bytes, stream()), "residual_norm planes");
            yb.split_bytes = bytes;
        }
        planes = yb.split_dev;
    }
    check(ttk_residual_norm_fwd(dread(x.impl()), dread(block.impl()), dread(w_post.impl()),
                                go ? dread(go) : nullptr, kind, dread(w_next.impl()),
                                out_ptr(out.h), y, r1->device_for_overwrite(),
                                r2->device_for_overwrite(), planes, R, D, residual_scale, eps,
                                stream()),
          "residual_norm");
    if (planes) {
        const int64_t key[7] = {0, 1, R, D, D, 0, 0};
        yb.split_version = yb.version;
        std::copy(key, key + 7, yb.split_key);
    }
    if (!rg)
        return out;
    // y hangs on h in the graph, so its node runs first: it only leaves its
    // gradient for h's node, which takes both through one kernel.
    auto dy = std::make_shared<std::shared_ptr<Buffer>>();
    Tensor::Impl* yo = out.y.impl().get();  // own nodes: raw, no cycle
    yo->prev = {out.h.impl()};
    yo->backward_fn = [yo, dy]() { *dy = yo->grad; };
    auto xo = x.impl(), bo = block.impl(), wp = w_post.impl(), wn = w_next.impl();
    Tensor::Impl* ho = out.h.impl().get();
    ho->prev = {xo, bo, wp, wn};
    if (go)
        ho->prev.push_back(go);
    ho->backward_fn = [xo, bo, wp, wn, go, kind, ho, dy, r1, r2, R, D, residual_scale]() {
        const std::shared_ptr<Buffer> gy = std::move(*dy);
        dy->reset();
        const float* dh = grad_in(ho);
        if (!dh && !gy)
            return;
        GradDst dx(xo, false), db(bo, bo == xo);
        std::unique_ptr<GradDst> dg;
        if (go && go->requires_grad)
            dg.reset(new GradDst(go, go == xo || go == bo || go == wp || go == wn));
        int acc = TTK_ACC_DW;
        acc |= dx.overwrite ? 0 : TTK_ACC_DX;
        acc |= db.overwrite ? 0 : TTK_ACC_DB;
        acc |= dg && !dg->overwrite ? TTK_ACC_DGATE : 0;
        const size_t ws = ttk_residual_norm_bwd_workspace_size(R, D);
        Scratch w(ws);
        check(ttk_residual_norm_bwd(dh, gy ? gy->device() : nullptr, dread(ho), dread(bo),
                                    dread(wp), go ? dread(go) : nullptr, kind, dread(wn),
                                    r1->device(), r2->device(), dx.ptr, db.ptr,
                                    wp->requires_grad ? grad_rmw(wp) : nullptr,
                                    wn->requires_grad && gy ? grad_rmw(wn) : nullptr,
                                    dg ? dg->ptr : nullptr, acc, R, D, residual_scale, w.ptr, ws,
                                    stream()),
              "residual_norm bwd");
        db.deliver();
        if (dg)
            dg->deliver();
    };
    return out;
}

TeacherTop::TeacherTop(const std::vector<int32_t>& ids_, const std::vector<float>& logits_,
                       int64_t k_)
    : k(k_) {
    if (k <= 0 || ids_.size() != logits_.size() || ids_.empty() ||
        static_cast<int64_t>(ids_.size()) % k)
        throw std::invalid_argument("TeacherTop: ids and logits must be [N, k] alike");
    n = static_cast<int64_t>(ids_.size()) / k;
    const size_t bytes = ids_.size() * 4;
    auto s = std::make_shared<Scratch>(2 * bytes);
    char* at = s->as<char>();
    check(ttk_memcpy_h2d(at, ids_.data(), bytes, stream()), "teacher upload");
    check(ttk_memcpy_h2d(at + bytes, logits_.data(), bytes, stream()), "teacher upload");
    ids = reinterpret_cast<const int32_t*>(at);
    logits = at + bytes;
    buf = std::shared_ptr<void>(s, s->ptr);
}

TeacherTop TeacherTop::borrow(const int32_t* ids, const void* logits, int type, int64_t n,
                              int64_t k) {
    TeacherTop t;
    t.ids = ids;
    t.logits = logits;
    t.type = type;
    t.n = n;
    t.k = k;
    return t;
}

Tensor distill_loss(const Tensor& logits, const TeacherTop& teacher, const DeviceIds& targets,
                    float alpha, float temperature, Tensor* parts) {
    if (logits.ndim() != 2)
        throw std::invalid_argument("distill_loss: logits must be 2D");
    const int64_t N = logits.dim(0), C = logits.dim(1);
    if (teacher.n != N)
        throw std::invalid_argument("distill_loss: teacher rows mismatch");
    if (targets.size() != 0 && targets.size() != N)
        throw std::invalid_argument("distill_loss: targets size mismatch");
    if (!(alpha >= 0.0f && alpha <= 1.0f) || !(temperature > 0.0f))
        throw std::invalid_argument("distill_loss: alpha in [0, 1] and temperature > 0 expected");
    Tensor out = make_out({1}, logits.requires_grad());
    Tensor all = make_out({3}, false);
    // The gradient for d(loss) = 1 comes with the loss (the rows are read once)
    // and is kept for the backward.
    auto lo = logits.impl();
    auto compute = [lo, teacher, targets, N, C, alpha, temperature](float* loss3, float* dlogits) {
        const size_t ws = ttk_distill_loss_workspace_size(N);
        Scratch w(ws);
        check(ttk_distill_loss(dread(lo), C, teacher.ids, teacher.logits, teacher.type, teacher.k,
                               targets.size() ? targets.data() : nullptr, nullptr, N, C, alpha,
                               temperature, 1.0f / static_cast<float>(N), loss3, dlogits, C, w.ptr,
                               ws, stream()),
              "distill_loss");
    };
    std::shared_ptr<Buffer> dlog;
    if (logits.requires_grad())
        dlog = std::make_shared<Buffer>(N * C);
    compute(out_ptr(all), dlog ? dlog->device_for_overwrite() : nullptr);
    check(ttk_memcpy_d2d(out_ptr(out), dread(all.impl()), 4, stream()), "distill_loss");
    if (parts)
        *parts = all;
    if (out.requires_grad()) {
        Tensor::Impl* oo = out.impl().get();  // own node: raw, no cycle
        oo->prev = {lo};
        oo->backward_fn = [lo, oo, dlog, compute]() mutable {
            deliver_loss_grad(oo, lo, dlog, [&](float* d) {
                Scratch loss3(3 * sizeof(float));
                compute(loss3.as<float>(), d);
            });
        };
    }
    return out;
}

}  // namespace tt
