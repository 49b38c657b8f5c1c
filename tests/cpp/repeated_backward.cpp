// Losses that keep their gradient from the forward pass (tt::distill_loss,
// tt::cross_entropy), run backward several times over one graph. Each pass has to
// add the same gradient, whatever became of the buffers that earlier passes
// filled: the leaf zeroed, scaled or added to, the logits a leaf, a view of one, or
// a sum whose terms share a buffer. The first pass is the reference: n passes
// leave n times its gradient, within the roundings of the additions. Arguments: the losses to check ("distill",
// "cross_entropy"). Prints "ok" and exits 0 on success.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "tinytrain/ops.h"
#include "tinytrain/tensor.h"

using tt::Tensor;

namespace {

constexpr int64_t N = 24, C = 300, K = 5;
int bad = 0;

using Vec = std::vector<float>;

Vec grad(const Tensor& t) { return Vec(t.grad_data(), t.grad_data() + t.numel()); }

void expect(const std::string& what, const Vec& got, const Vec& one, int times) {
    double worst = 0.0;
    for (size_t i = 0; i < got.size(); ++i) {
        const double want = double(one[i]) * times, err = std::fabs(got[i] - want);
        worst = std::fmax(worst, std::isnan(got[i]) ? INFINITY : err / (std::fabs(want) + 1e-30));
    }
    // A pass adds two terms at most, each addition rounded by 2^-24 of what stands
    // there (at most twice the result); `one` itself is rounded once.
    if (!(worst <= 4 * times * std::ldexp(1.0, -24))) {
        std::printf("%s: off by %g\n", what.c_str(), worst);
        ++bad;
    }
}

Tensor loss_of(const std::string& loss, const Tensor& logits) {
    std::vector<int64_t> t;
    std::vector<int32_t> ids;
    Vec top;
    for (int64_t i = 0; i < N; ++i) {
        t.push_back((7 * i + 3) % C);
        for (int64_t k = 0; k < K; ++k) {
            ids.push_back(static_cast<int32_t>((5 * i + 31 * k) % C));
            top.push_back(0.25f * static_cast<float>(k));
        }
    }
    if (loss == "cross_entropy")
        return tt::cross_entropy(logits, tt::DeviceIds(t));
    return tt::distill_loss(logits, tt::TeacherTop(ids, top, K), tt::DeviceIds(t), 0.5f, 2.0f);
}

// form: how the logits hang on the leaf
Tensor logits_of(int form, const Tensor& x) {
    switch (form) {
        case 0:
            return x;
        case 1:
            return tt::reshape(x, {N, C});
        case 2:
            return tt::add(x, tt::silu(x));
        case 3:
            return tt::reshape(tt::sub(x, tt::mul(x, tt::full({1}, 0.5f))), {N, C});
        default:
            return tt::mul(x, tt::full({1}, 2.0f));
    }
}

void run(const std::string& loss, int form) {
    const std::string name = loss + " form " + std::to_string(form);
    Tensor x = tt::randn(form == 1 || form == 3 ? std::vector<int64_t>{N * C}
                                                : std::vector<int64_t>{N, C}, 5);
    x.set_requires_grad(true);
    Tensor l = loss_of(loss, logits_of(form, x));
    l.backward();
    const Vec one = grad(x);
    double size = 0.0;
    for (float g : one)
        size += std::fabs(double(g));
    if (!(size > 0.0))
        std::printf("%s: no gradient\n", name.c_str()), ++bad;
    l.backward();
    expect(name + ", second pass added", grad(x), one, 2);
    l.backward();
    expect(name + ", third pass added", grad(x), one, 3);
    x.zero_grad();
    l.backward();
    expect(name + ", after zero_grad", grad(x), one, 1);
    tt::clip_grad_norm({&x}, 1e-4f);
    x.zero_grad();
    l.backward();
    expect(name + ", after clipping and zero_grad", grad(x), one, 1);
    l.backward();
    expect(name + ", added after that", grad(x), one, 2);
    // a second loss on the same logits
    Tensor y = tt::randn({N, C}, 5);
    y.set_requires_grad(true);
    Tensor s = logits_of(form == 1 || form == 3 ? 0 : form, y);
    Tensor a = loss_of(loss, s), b = tt::add(a, tt::sum_all(s));
    b.backward();
    const Vec both = grad(y);
    y.zero_grad();
    b.backward();
    expect(name + ", two uses of the logits", grad(y), both, 1);
    // scaled, then as it is
    tt::mul(a, tt::full({1}, 2.0f)).backward();
    y.zero_grad();
    a.backward();
    const Vec plain = grad(y);
    y.zero_grad();
    a.backward();
    expect(name + ", after a scaled pass", grad(y), plain, 1);
}

}  // namespace

int main(int argc, char** argv) {
    for (int i = 1; i < argc; ++i)
        for (int form = 0; form < 5; ++form)
            run(argv[i], form);
    tt::synchronize();
    if (bad || argc < 2) {
        std::printf("%d checks failed\n", bad);
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
