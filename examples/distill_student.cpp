// Distilling a small student from a teacher's stored top logits.
//
// The teacher is a GPTModel; for each batch its top K logits per position are
// kept, as a data pipeline would store them on disk. The student is a narrower
// decoder whose sub-layers are normalized before and after: a scaled embedding,
// then per block attention and feed-forward, each followed by one residual_norm
// (the norm after it, a learned gate per channel, the depth-scaled residual and
// the norm before the next sub-layer in one kernel), and the embedding table as
// its head. It trains on the distillation loss with AdamW.
//
//   python -m tinytrain_b200.build
//   g++ -std=c++20 -O2 -Iinclude -o distill_student examples/distill_student.cpp
//       -Ltinytrain_b200/lib -ltinytrain -lttk -Wl,-rpath,$PWD/tinytrain_b200/lib
//   ./distill_student [steps]
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <numeric>
#include <vector>

#include "tinytrain/model.h"
#include "tinytrain/ops.h"
#include "tinytrain/optim.h"

using tt::Tensor;

namespace {

constexpr int64_t VOCAB = 512, DIM = 128, HEADS = 4, LAYERS = 2, FFN = 256, SEQ = 64, BATCH = 8;
constexpr int64_t TOP = 32;

struct Student {
    struct Block {
        tt::Linear wq{DIM, DIM, 11}, wk{DIM, DIM, 12}, wv{DIM, DIM, 13}, wo{DIM, DIM, 14},
            wgate{DIM, FFN, 15}, wup{DIM, FFN, 16}, wdown{FFN, DIM, 17};
        // after the sub-layer: norm and gate; before the next one: norm
        tt::RMSNorm post_attn{DIM, 1e-5f}, pre_ffn{DIM, 1e-5f}, post_ffn{DIM, 1e-5f},
            pre_next{DIM, 1e-5f};
        Tensor gate_attn{{DIM}, 1.0f, true}, gate_ffn{{DIM}, 1.0f, true};
        explicit Block(uint64_t seed)
            : wq(DIM, DIM, seed), wk(DIM, DIM, seed + 1), wv(DIM, DIM, seed + 2),
              wo(DIM, DIM, seed + 3), wgate(DIM, FFN, seed + 4), wup(DIM, FFN, seed + 5),
              wdown(FFN, DIM, seed + 6) {}
    };
    tt::Embedding embed{VOCAB, DIM, 1};
    tt::RMSNorm first{DIM, 1e-5f};
    std::vector<Block> blocks;
    Tensor cos, sin;

    Student() {
        for (int64_t l = 0; l < LAYERS; ++l)
            blocks.emplace_back(100 + 10 * static_cast<uint64_t>(l));
        const int64_t half = DIM / HEADS / 2;
        std::vector<float> c, s;
        for (int64_t t = 0; t < SEQ; ++t)
            for (int64_t i = 0; i < half; ++i) {
                const float a = static_cast<float>(t) /
                                std::pow(10000.0f, static_cast<float>(i) / static_cast<float>(half));
                c.push_back(std::cos(a));
                s.push_back(std::sin(a));
            }
        cos = Tensor({SEQ, half});
        sin = Tensor({SEQ, half});
        cos.copy_from_host(c.data());
        sin.copy_from_host(s.data());
    }

    std::vector<Tensor*> parameters() {
        std::vector<Tensor*> p{&embed.weight, &first.weight};
        for (Block& b : blocks)
            for (Tensor* t : {&b.wq.weight, &b.wk.weight, &b.wv.weight, &b.wo.weight,
                              &b.post_attn.weight, &b.gate_attn, &b.pre_ffn.weight,
                              &b.wgate.weight, &b.wup.weight, &b.wdown.weight, &b.post_ffn.weight,
                              &b.gate_ffn, &b.pre_next.weight})
                p.push_back(t);
        return p;
    }

    Tensor forward(const tt::DeviceIds& ids) {
        const int64_t R = BATCH * SEQ, hd = DIM / HEADS;
        const float scale = 1.0f / std::sqrt(2.0f * LAYERS);  // of the residual
        Tensor h = tt::embedding_scaled(embed.weight, ids, std::sqrt(static_cast<float>(DIM)));
        Tensor y = tt::rmsnorm(h, first.weight, first.eps);
        for (Block& b : blocks) {
            auto heads = [&](tt::Linear& w) {
                return tt::reshape(tt::linear(y, w.weight), {BATCH, SEQ, HEADS, hd});
            };
            Tensor a = tt::causal_attention(heads(b.wq), heads(b.wk), heads(b.wv), cos, sin);
            a = tt::linear(tt::reshape(a, {R, DIM}), b.wo.weight);
            auto n = tt::residual_norm(h, a, b.post_attn.weight, b.pre_ffn.weight, b.gate_attn,
                                       1.0f - scale, 1e-5f);
            Tensor f = tt::ffn_swiglu(n.y, b.wgate.weight, b.wup.weight, b.wdown.weight);
            n = tt::residual_norm(n.h, f, b.post_ffn.weight, b.pre_next.weight, b.gate_ffn,
                                  1.0f - scale, 1e-5f);
            h = n.h, y = n.y;
        }
        return tt::linear(y, embed.weight);  // the table is the head too
    }
};

// The K largest logits of each row.
tt::TeacherTop top_of(const Tensor& logits, int64_t k) {
    const int64_t N = logits.dim(0), C = logits.dim(1);
    const float* x = logits.data();
    std::vector<int32_t> ids, order(static_cast<size_t>(C));
    std::vector<float> top;
    for (int64_t i = 0; i < N; ++i, x += C) {
        std::iota(order.begin(), order.end(), 0);
        std::partial_sort(order.begin(), order.begin() + k, order.end(),
                          [&](int32_t a, int32_t b) { return x[a] > x[b]; });
        for (int64_t j = 0; j < k; ++j) {
            ids.push_back(order[static_cast<size_t>(j)]);
            top.push_back(x[order[static_cast<size_t>(j)]]);
        }
    }
    return tt::TeacherTop(ids, top, k);
}

}  // namespace

int main(int argc, char** argv) {
    const int steps = argc > 1 ? std::atoi(argv[1]) : 40;
    tt::GPTConfig tc;
    tc.vocab_size = VOCAB, tc.dim = 256, tc.n_layers = 2, tc.n_heads = 8, tc.n_kv_heads = 8;
    tc.ffn_dim = 512, tc.max_seq_len = SEQ;
    tt::GPTModel teacher(tc, 7);

    // One batch of ids with padded ends; the label is the next id.
    std::vector<int64_t> ids, labels, shown;
    uint64_t r = 12345;
    for (int64_t i = 0; i < BATCH * SEQ; ++i) {
        r = r * 6364136223846793005ull + 1442695040888963407ull;
        ids.push_back(static_cast<int64_t>((r >> 33) % VOCAB));
    }
    for (int64_t i = 0; i < BATCH * SEQ; ++i) {
        const bool pad = i % SEQ >= SEQ - 8;
        shown.push_back(pad ? -1 : ids[static_cast<size_t>(i)]);
        labels.push_back(i % SEQ + 1 >= SEQ - 8 ? -1 : ids[static_cast<size_t>(i + 1)]);
    }
    const tt::TeacherTop top = top_of(teacher.forward(ids, BATCH, SEQ), TOP);
    const tt::DeviceIds dev(shown), targets(labels);

    Student student;
    tt::AdamW opt(student.parameters(), 3e-3f, 0.9f, 0.95f, 1e-8f, 0.0f);
    opt.set_clip_norm(1.0f);
    float first = 0.0f, last = 0.0f;
    for (int step = 0; step < steps; ++step) {
        opt.zero_grad();
        Tensor parts;
        Tensor loss = tt::distill_loss(student.forward(dev), top, targets, 0.8f, 2.0f, &parts);
        loss.backward();
        opt.step();
        const Tensor& p = parts;
        last = p.data()[0];
        if (step == 0)
            first = last;
        if (step % 10 == 0 || step == steps - 1)
            std::printf("step %3d  loss %.4f  teacher KL %.4f  cross-entropy %.4f\n", step,
                        static_cast<double>(p.data()[0]), static_cast<double>(p.data()[1]),
                        static_cast<double>(p.data()[2]));
    }
    tt::synchronize();
    return std::isfinite(last) && (steps < 2 || last < first) ? 0 : 1;
}
