// tt::embedding_scaled, tt::residual_norm and tt::distill_loss against the same
// values composed of the library's other ops, forward and backward, with the
// uses a graph can make of them: both outputs of residual_norm read or only one,
// one tensor given twice, inputs that need no gradient, a second backward that
// adds to the leaves. Each pair agrees within 5e-6 of the largest magnitude:
// both sides round each value some tens of times by 2^-24. A scalar gate's
// gradient is compared with sums in 64 bits. Prints "ok" and exits 0 on success.
#include <cmath>
#include <cstdio>
#include <string>
#include <vector>

#include "tinytrain/ops.h"
#include "tinytrain/tensor.h"

using tt::Tensor;

namespace {

int bad = 0;

void same(const std::string& what, const float* a, const float* b, int64_t n, double tol = 5e-6) {
    double num = 0, den = 1e-30;
    for (int64_t i = 0; i < n; ++i) {
        num = std::fmax(num, std::fabs(double(a[i]) - b[i]));
        den = std::fmax(den, std::fabs(double(b[i])));
    }
    if (!(num <= tol * den)) {
        std::printf("%s: %g\n", what.c_str(), num / den);
        ++bad;
    }
}

const float* vals(const Tensor& t) { return t.data(); }

Tensor leaf(const std::vector<int64_t>& shape, uint64_t seed, bool rg = true) {
    Tensor t = tt::randn(shape, seed);
    t.set_requires_grad(rg);
    return t;
}

// The gradient of a scalar gate in 64 bits: a sum over every element whose terms
// cancel, so that the composed ops' own 32-bit sum is no reference for it.
double scalar_gate_grad(const float* x, const float* b, const float* w1, const float* w2, double g,
                        const float* A, const float* B, int64_t R, int64_t D, double s, double eps,
                        int mode) {
    double total = 0.0;
    std::vector<double> u(static_cast<size_t>(D)), h(u), e(u);
    for (int64_t r = 0; r < R; ++r, x += D, b += D, A += D, B += D) {
        double bb = 0.0, hh = 0.0, eh = 0.0;
        for (int64_t c = 0; c < D; ++c)
            bb += double(b[c]) * b[c];
        const double r1 = 1.0 / std::sqrt(bb / double(D) + eps);
        for (int64_t c = 0; c < D; ++c) {
            u[c] = b[c] * r1 * w1[c];
            h[c] = s * x[c] + g * u[c];
            hh += h[c] * h[c];
        }
        const double r2 = 1.0 / std::sqrt(hh / double(D) + eps);
        for (int64_t c = 0; c < D; ++c) {
            e[c] = mode == 1 ? 0.0 : double(B[c]) * w2[c];
            eh += e[c] * h[c];
        }
        for (int64_t c = 0; c < D; ++c)
            total += u[c] * ((mode == 2 ? 0.0 : A[c]) + r2 * e[c] - h[c] * r2 * r2 * r2 / double(D) * eh);
    }
    return total;
}

// mode: which outputs reach the loss: 0 both, 1 h, 2 y. share: x is the block.
void norm_case(int64_t R, int64_t D, int gate_kind, int mode, bool share, bool x_grad) {
    const std::string name = "norm R" + std::to_string(R) + " D" + std::to_string(D) + " gate" +
                             std::to_string(gate_kind) + " mode" + std::to_string(mode) +
                             (share ? " shared" : "") + (x_grad ? "" : " frozen");
    const float s = 0.75f, eps = 1e-5f;
    std::vector<std::vector<float>> grads[2];
    std::vector<std::vector<float>> outs[2];
    for (int own = 0; own < 2; ++own) {
        Tensor x = leaf({R, D}, 1, x_grad), b = share ? x : leaf({R, D}, 2), w1 = leaf({D}, 3),
               w2 = leaf({D}, 4), A = tt::randn({R, D}, 5), B = tt::randn({R, D}, 6), g;
        if (gate_kind == 1)
            g = leaf({1}, 7);
        else if (gate_kind == 2)
            g = leaf({D}, 7);
        else if (gate_kind == 3)
            g = leaf({R, 1}, 7);
        else if (gate_kind == 4)
            g = leaf({R, D}, 7);
        for (int pass = 0; pass < 2; ++pass) {  // the second adds to the gradients
            Tensor h, y;
            if (own) {
                auto out = tt::residual_norm(x, b, w1, w2, g, s, eps);
                h = out.h, y = out.y;
            } else {
                Tensor u = tt::rmsnorm(b, w1, eps);
                if (gate_kind)
                    u = tt::mul(u, g);
                h = tt::add(tt::mul(x, tt::full({1}, s)), u);
                y = tt::rmsnorm(h, w2, eps);
            }
            Tensor loss = mode == 1   ? tt::sum_all(tt::mul(h, A))
                          : mode == 2 ? tt::sum_all(tt::mul(y, B))
                                      : tt::add(tt::sum_all(tt::mul(h, A)),
                                                tt::sum_all(tt::mul(y, B)));
            loss.backward();
            if (pass == 0) {
                outs[own].push_back({vals(h), vals(h) + R * D});
                outs[own].push_back({vals(y), vals(y) + R * D});
            }
        }
        for (Tensor* t : {&x, &b, &w1, &w2, &g})
            if (t->impl() && t->has_grad())
                grads[own].push_back({t->grad_data(), t->grad_data() + t->numel()});
        if (gate_kind == 1 && !own)  // two passes
            grads[own].back()[0] = static_cast<float>(
                2.0 * scalar_gate_grad(vals(x), vals(b), vals(w1), vals(w2), vals(g)[0], vals(A),
                                       vals(B), R, D, s, eps, mode));
    }
    for (size_t i = 0; i < outs[0].size(); ++i)
        same(name + " out" + std::to_string(i), outs[1][i].data(), outs[0][i].data(), R * D);
    // without y's gradient the composed form has none for w_next either
    if (grads[0].size() != grads[1].size()) {
        std::printf("%s: %zu gradients, %zu expected\n", name.c_str(), grads[1].size(),
                    grads[0].size());
        ++bad;
        return;
    }
    for (size_t i = 0; i < grads[0].size(); ++i)
        same(name + " grad" + std::to_string(i), grads[1][i].data(), grads[0][i].data(),
             static_cast<int64_t>(grads[0][i].size()));
}

void embedding_case(int64_t N, int64_t D, int64_t V) {
    std::vector<int64_t> ids(static_cast<size_t>(N));
    for (int64_t i = 0; i < N; ++i)
        ids[static_cast<size_t>(i)] = (i * i * 7 + i) % V;
    std::vector<float> g[2], o[2];
    for (int own = 0; own < 2; ++own) {
        Tensor W = leaf({V, D}, 1), G = tt::randn({N, D}, 2);
        tt::DeviceIds dev(ids);
        for (int pass = 0; pass < 2; ++pass) {
            Tensor e = own ? tt::embedding_scaled(W, dev, 8.0f)
                           : tt::mul(tt::embedding(W, dev), tt::full({1}, 8.0f));
            tt::sum_all(tt::mul(e, G)).backward();
            if (pass == 0)
                o[own].assign(vals(e), vals(e) + N * D);
        }
        g[own].assign(W.grad_data(), W.grad_data() + V * D);
    }
    same("embedding", o[1].data(), o[0].data(), N * D);
    same("embedding grad", g[1].data(), g[0].data(), V * D);
}

void distill_case(int64_t N, int64_t C) {
    // alpha 0: the labels' cross-entropy
    std::vector<int64_t> t(static_cast<size_t>(N));
    for (int64_t i = 0; i < N; ++i)
        t[static_cast<size_t>(i)] = (3 * i + 1) % C;
    // alpha 1, temperature 1, a list of every class: sum p (log p - log q)
    Tensor z = tt::randn({N, C}, 9);
    std::vector<int32_t> ids;
    for (int64_t i = 0; i < N; ++i)
        for (int64_t c = 0; c < C; ++c)
            ids.push_back(static_cast<int32_t>((c + i) % C));
    std::vector<float> top(ids.size());
    for (size_t i = 0; i < ids.size(); ++i)
        top[i] = vals(z)[static_cast<int64_t>(i) / C * C + ids[i]];
    tt::TeacherTop teacher(ids, top, C);
    for (int kd = 0; kd < 2; ++kd) {
        std::vector<float> g[2];
        float loss[2];
        for (int own = 0; own < 2; ++own) {
            Tensor x = leaf({N, C}, 8), l;
            Tensor s = tt::mul(x, tt::full({1}, 2.0f));  // an inner node
            if (own) {
                Tensor parts;
                l = tt::distill_loss(s, teacher, tt::DeviceIds(t), kd ? 1.0f : 0.0f, 1.0f, &parts);
                if (vals(parts)[0] != vals(l)[0] || vals(parts)[1 + (1 - kd)] != vals(l)[0])
                    std::printf("parts\n"), ++bad;
            } else if (kd) {
                Tensor p = tt::softmax(z, -1);
                Tensor d = tt::sub(tt::log_softmax(z, -1), tt::log_softmax(s, -1));
                l = tt::mul(tt::sum_all(tt::mul(p, d)), tt::full({1}, 1.0f / static_cast<float>(N)));
            } else {
                l = tt::cross_entropy(s, t);
            }
            loss[own] = vals(l)[0];
            tt::mul(l, tt::full({1}, 3.0f)).backward();
            l.backward();
            g[own].assign(x.grad_data(), x.grad_data() + N * C);
        }
        same("distill loss", &loss[1], &loss[0], 1);
        same("distill grad", g[1].data(), g[0].data(), N * C);
    }
}

template <class F>
void refused(const char* what, F f) {
    try {
        f();
    } catch (const std::invalid_argument&) {
        return;
    }
    std::printf("%s: not refused\n", what);
    ++bad;
}

}  // namespace

int main() {
    for (int gate = 0; gate < 5; ++gate)
        for (int mode = 0; mode < 3; ++mode) {
            norm_case(37, 96, gate, mode, false, true);
            norm_case(5, 33, gate, mode, true, true);
            norm_case(9, 64, gate, mode, false, false);
        }
    norm_case(4096, 256, 2, 0, false, true);  // with GEMM operand planes of y
    embedding_case(500, 48, 31);
    embedding_case(3000, 256, 2000);
    distill_case(23, 300);
    // the planes of y feed a projection as a split of y does
    {
        Tensor x = leaf({4096, 256}, 1), b = leaf({4096, 256}, 2), w1 = leaf({256}, 3),
               w2 = leaf({256}, 4), P = leaf({512, 256}, 5);
        Tensor y = tt::residual_norm(x, b, w1, w2).y;
        std::vector<float> copy(vals(y), vals(y) + y.numel());
        Tensor y2({4096, 256});
        y2.copy_from_host(copy.data());
        Tensor p = tt::linear(tt::residual_norm(x, b, w1, w2).y, P), q = tt::linear(y2, P);
        same("planes", vals(p), vals(q), p.numel(), 0.0);
    }
    Tensor a({4, 8}), w({8}), v({7});
    refused("shapes", [&] { tt::residual_norm(a, Tensor({4, 7}), w, w); });
    refused("weights", [&] { tt::residual_norm(a, a, v, w); });
    refused("gate", [&] { tt::residual_norm(a, a, w, w, Tensor({3})); });
    refused("teacher", [&] { tt::TeacherTop({1, 2, 3}, {1.f, 2.f, 3.f}, 2); });
    refused("rows", [&] {
        tt::distill_loss(a, tt::TeacherTop({1, 2}, {1.f, 2.f}, 1), tt::DeviceIds(), 1.0f, 1.0f);
    });
    refused("targets", [&] {
        tt::distill_loss(a, tt::TeacherTop({1, 2, 3, 4}, {1.f, 2.f, 3.f, 4.f}, 1),
                         tt::DeviceIds(std::vector<int64_t>{1}), 1.0f, 1.0f);
    });
    tt::synchronize();
    if (bad) {
        std::printf("%d checks failed\n", bad);
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
