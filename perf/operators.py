"""Measured cases of the operators a distilled student trains with: the scaled
embedding and its gradient, the residual norm (norm after a block, gate,
residual scale, norm before the next block) forward and backward, and the
distillation loss on a teacher's top logits with its gradient.

Widths, vocabulary and token counts are those of the 13M, 110M and 1B training
configurations (dim 256, 768, 2048; vocabulary 32000; 16 x 128, 64 x 1024 and
16 x 2048 tokens per micro-batch), one sequence of 128 tokens for the smallest
calls, and odd sizes between them.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
GATES = ("none", "scalar", "column", "row", "full")


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One sequence of the 13M model looked up: launch latency.
        dict(name="embed_lookup_128x256", op="embed_fwd", N=128, D=256, V=32000, pad=False),
        # One micro-batch of the 1B model (16 x 2048 tokens).
        dict(name="embed_lookup_32768x2048", op="embed_fwd", N=32768, D=2048, V=32000, pad=False),
        # The 13M model's step of 16 x 128 tokens: a gradient of 32000 rows, most without a token.
        dict(name="embed_grad_2048x256", op="embed_bwd", N=2048, D=256, V=32000, pad=False),
        # A 1B micro-batch with padded sequence ends: frequent ids repeat thousands of times.
        dict(name="embed_grad_32768x2048", op="embed_bwd", N=32768, D=2048, V=32000, pad=True),
        # One sequence of the 13M model through one block boundary: latency.
        dict(name="norm_fwd_128x256", op="norm_fwd", R=128, D=256, gate="none", alpha=1.0),
        # A 1B micro-batch, a learned gate per channel and a depth-scaled residual.
        dict(name="norm_fwd_32768x2048", op="norm_fwd", R=32768, D=2048, gate="column", alpha=0.75),
        # The 13M step's backward through a block boundary, one learned gate value.
        dict(name="norm_bwd_2048x256", op="norm_bwd", R=2048, D=256, gate="scalar", alpha=1.0),
        # A 1B micro-batch backward, gate per channel: three column sums.
        dict(name="norm_bwd_32768x2048", op="norm_bwd", R=32768, D=2048, gate="column", alpha=0.75),
        # Odd width and rows, a gate computed per element (its gradient is a full tensor).
        dict(name="norm_bwd_3001x1111", op="norm_bwd", R=3001, D=1111, gate="full", alpha=0.5),
        # Held-out loss of one sequence: no gradient.
        dict(name="distill_eval_128x32000", op="distill", N=128, C=32000, K=16, tau=1.0, alpha=1.0,
             teacher="float32", ragged=False, grad=False),
        # A training micro-batch: half the loss from the teacher at temperature 2, half from labels.
        dict(name="distill_train_8192x32000", op="distill", N=8192, C=32000, K=64, tau=2.0, alpha=0.5,
             teacher="bfloat16", ragged=False, grad=True),
        # Odd vocabulary, lists cut short, rows without a label or masked out of the loss.
        dict(name="distill_train_1237x49999", op="distill", N=1237, C=49999, K=50, tau=1.5, alpha=0.9,
             teacher="float16", ragged=True, grad=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_bwd", "norm_fwd", "norm_bwd", "distill", "distill"])
    if op == "distill":
        C = _spread(rng, 500, 60000)
        N = _spread(rng, 1, max(2, min(16384, 8192 * 32000 // C)))
        return dict(op=op, N=N, C=C, K=min(C, _spread(rng, 1, 256)), tau=rng.choice([1.0, 1.5, 2.0, 4.0]),
                    alpha=rng.choice([1.0, 0.9, 0.5]), teacher=rng.choice(["float32", "bfloat16", "float16"]),
                    ragged=rng.random() < 0.5, grad=rng.random() < 0.75)
    D = _spread(rng, 64, 2048)
    if rng.random() < 0.5:
        D = max(64, D // 64 * 64)
    n = _spread(rng, 1, 32768)
    if op.startswith("embed"):
        return dict(op=op, N=n, D=D, V=_spread(rng, 1000, 32000), pad=rng.random() < 0.5)
    return dict(op=op, R=n, D=D, gate=rng.choice(GATES), alpha=rng.choice([1.0, 0.75, 0.5]))


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tokens(N, V, pad, g):
    """Token ids with the frequencies of text: the id of rank r about as often
    as 1 / (r + 2.7); with `pad`, the last eighth of each 512 positions is -1.
    Looked up in sums made on the host: a parallel prefix sum on the device rounds
    differently from run to run, and some ids with it."""
    freq = np.cumsum(1.0 / (np.arange(V) + 2.7))
    u = torch.rand(N, device=g.device, dtype=torch.float64, generator=g)
    ids = torch.searchsorted(torch.from_numpy(freq / freq[-1]).to(g.device), u, right=True)
    ids = ids.clamp(max=V - 1)
    if pad:
        pos = torch.arange(N, device=g.device) % 512
        ids = torch.where(pos >= 448, torch.full_like(ids, -1), ids)
    return ids.contiguous()


def _gate(kind, R, D, g):
    shape = {"none": None, "scalar": (1,), "column": (D,), "row": (R, 1), "full": (R, D)}[kind]
    return None if shape is None else torch.rand(shape, device="cuda", generator=g) * 1.5 + 0.1


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    if op == "embed_fwd":
        N, D, V = case["N"], case["D"], case["V"]
        return dict(op=op, W=randn(V, D) * 0.02, ids=_tokens(N, V, case["pad"], g), scale=math.sqrt(D))
    if op == "embed_bwd":
        N, D, V = case["N"], case["D"], case["V"]
        return dict(op=op, dout=randn(N, D) * 1e-3, ids=_tokens(N, V, case["pad"], g), V=V, scale=math.sqrt(D))
    if op in ("norm_fwd", "norm_bwd"):
        R, D = case["R"], case["D"]
        s = dict(op=op, x=randn(R, D) * 2.0, b=randn(R, D) * 0.5, w_post=1 + 0.2 * randn(D),
                 w_next=1 + 0.2 * randn(D), gate=_gate(case["gate"], R, D, g), alpha=case["alpha"])
        if op == "norm_bwd":
            r1 = (s["b"].square().mean(1) + EPS).rsqrt()
            u = s["b"] * r1[:, None] * s["w_post"]
            h = s.pop("x") * s["alpha"] + (u if s["gate"] is None else u * s["gate"])
            s |= dict(h=h, r1=r1, r2=(h.square().mean(1) + EPS).rsqrt(), dh=randn(R, D) * 1e-2,
                      dy=randn(R, D) * 1e-2)
        return s
    N, C, K = case["N"], case["C"], case["K"]
    base = randn(N, C) * 2.0
    logits = base + randn(N, C) * 0.7
    base += randn(N, C) * 0.7
    top, ids = base.topk(K, dim=1)
    del base
    labels = ids[torch.arange(N, device="cuda"), torch.randint(0, K, (N,), device="cuda", generator=g)]
    ids = ids.to(torch.int32)
    weight = None
    if case["ragged"]:
        # lists of 1..K entries (the rest -1), a tenth of the rows without a
        # label, a tenth masked out, one row in 37 without a teacher list
        n = torch.randint(1, K + 1, (N, 1), device="cuda", generator=g)
        rows = torch.arange(N, device="cuda")
        n[rows % 37 == 5] = 0
        ids = torch.where(torch.arange(K, device="cuda") < n, ids, torch.full_like(ids, -1))
        labels = torch.where(torch.rand(N, device="cuda", generator=g) < 0.1, torch.full_like(labels, -1), labels)
        weight = (torch.rand(N, device="cuda", generator=g) >= 0.1).float()
    return dict(op=op, logits=logits, ids=ids.contiguous(), top=top.to(getattr(torch, case["teacher"])).contiguous(),
                labels=labels.contiguous(), weight=weight, alpha=case["alpha"], tau=case["tau"], grad=case["grad"])


# --------------------------------------------------------------- one pass --
def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "embed_fwd":
        live = s["ids"] >= 0
        return torch.where(live[:, None], s["W"][s["ids"].clamp(min=0)] * s["scale"], 0.0)
    if op == "embed_bwd":
        live = s["ids"] >= 0
        rows = torch.where(live[:, None], s["dout"] * s["scale"], 0.0)
        dW = torch.zeros((s["V"], rows.shape[1]), device="cuda")
        return dW.index_add_(0, s["ids"].clamp(min=0), rows)
    if op == "norm_fwd":
        b = s["b"]
        r1 = 1.0 / torch.sqrt((b * b).mean(1, keepdim=True) + EPS)
        u = b * r1 * s["w_post"]
        h = s["alpha"] * s["x"] + (u if s["gate"] is None else s["gate"] * u)
        r2 = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        return h, h * r2 * s["w_next"]
    if op == "norm_bwd":
        return _plain_norm_bwd(s)
    return _plain_distill(s)


def _plain_norm_bwd(s):
    h, b, w1, w2, gate = s["h"], s["b"], s["w_post"], s["w_next"], s["gate"]
    D = h.shape[1]
    r1, r2 = s["r1"][:, None], s["r2"][:, None]
    e = s["dy"] * w2
    dH = s["dh"] + r2 * e - h * (r2 ** 3 * (e * h).sum(1, keepdim=True) / D)
    n = dH if gate is None else dH * gate
    f = n * w1
    db = r1 * f - b * (r1 ** 3 * (f * b).sum(1, keepdim=True) / D)
    out = [s["alpha"] * dH, db, (n * b * r1).sum(0), (s["dy"] * h * r2).sum(0)]
    if gate is not None:
        dg = dH * (b * r1 * w1)
        if gate.numel() == 1:
            dg = dg.sum().reshape(1)
        elif gate.dim() == 1:
            dg = dg.sum(0)
        elif gate.shape[1] == 1 and D > 1:
            dg = dg.sum(1, keepdim=True)
        out.append(dg)
    return out


def _plain_distill(s):
    x, ids, t, tau, alpha = s["logits"], s["ids"].long(), s["labels"], s["tau"], s["alpha"]
    N = x.shape[0]
    w = torch.ones(N, device="cuda") if s["weight"] is None else s["weight"]
    w = w / N
    listed_ = ids >= 0
    z = torch.where(listed_, s["top"].float() / tau, -math.inf)
    top = z.max(1, keepdim=True).values
    has = (top > -math.inf).float()
    ez = torch.where(listed_ & (has > 0), torch.exp(z - top), 0.0)
    sz = ez.sum(1, keepdim=True)
    p = torch.where(has > 0, ez / sz, 0.0)
    m = x.max(1, keepdim=True).values
    eT = torch.exp((x - m) / tau)
    sT = eT.sum(1, keepdim=True)
    e1 = torch.exp(x - m)
    s1 = e1.sum(1, keepdim=True)
    xk = x.gather(1, ids.clamp(min=0))
    kd = torch.where(p > 0, p * (z - top - torch.log(sz) - (xk - m) / tau + torch.log(sT)), 0.0).sum(1)
    labelled = (t >= 0).float()
    ce = labelled * (torch.log(s1) + m - x.gather(1, t.clamp(min=0)[:, None])).squeeze(1)
    kd, ce = (w * kd).sum(), (w * ce).sum()
    loss = torch.stack([alpha * tau * tau * kd + (1 - alpha) * ce, kd, ce])
    if not s["grad"]:
        return loss, None
    a, c = (w * alpha * tau)[:, None], (w * (1 - alpha) * labelled)[:, None]
    d = a * has * (eT / sT) + c * (e1 / s1)
    d.scatter_add_(1, ids.clamp(min=0), -a * p)
    d.scatter_add_(1, t.clamp(min=0)[:, None], -c)
    return loss, d


def _run_own(s):
    from tinytrain_b200 import kernels as K
    op = s["op"]
    if op == "embed_fwd":
        return K.embedding_scaled_fwd(s["W"], s["ids"], s["scale"])
    if op == "embed_bwd":
        return K.embedding_scaled_bwd(s["dout"], s["ids"], s["V"], s["scale"])
    if op == "norm_fwd":
        h, y, _, _ = K.residual_norm_fwd(s["x"], s["b"], s["w_post"], s["w_next"], gate=s["gate"],
                                         residual_scale=s["alpha"], eps=EPS)
        return h, y
    if op == "norm_bwd":
        out = K.residual_norm_bwd(s["dh"], s["dy"], s["h"], s["b"], s["w_post"], s["w_next"], s["r1"],
                                  s["r2"], gate=s["gate"], residual_scale=s["alpha"])
        return [o for o in out if o is not None]
    return K.distill_loss(s["logits"], s["ids"], s["top"], targets=s["labels"], alpha=s["alpha"],
                          temperature=s["tau"], row_weight=s["weight"], want_grad=s["grad"])


# --------------------------------------------------------------- the work --
def work(case):
    op = case["op"]
    if op.startswith("embed"):
        N, D, V = case["N"], case["D"], case["V"]
        live = N // 512 * 448 + min(N % 512, 448) if case["pad"] else N  # positions with a token
        if op == "embed_bwd":  # the rows of padding need not be read
            return {"bytes": 4 * live * D + 4 * V * D + 8 * N, "flops": 2 * live * D}
        r = np.arange(V) + 2.7
        seen = 1.0 - np.exp(live * np.log1p(-(1.0 / r) / (1.0 / r).sum()))  # expected distinct rows
        return {"bytes": 4 * N * D + 4 * D * float(seen.sum()) + 8 * N, "flops": live * D}
    if op.startswith("norm"):
        n = case["R"] * case["D"]
        full = 4 * n if case["gate"] == "full" else 0
        if op == "norm_fwd":
            return {"bytes": 16 * n + full, "flops": 11 * n}
        return {"bytes": 24 * n + 2 * full, "flops": 28 * n}
    n, k = case["N"] * case["C"], case["N"] * case["K"]
    size = 4 + (4 if case["teacher"] == "float32" else 2)
    two = case["tau"] != 1.0 and case["alpha"] != 1.0
    return {"bytes": (8 if case["grad"] else 4) * n + k * size, "flops": (4 if two else 2) * (3 if case["grad"] else 2) * n}


# ---------------------------------------------------------------- 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    op = s["op"]
    if op == "embed_fwd":
        out = torch.zeros((case["N"], case["D"]), dtype=torch.float64, device="cuda")
        live = torch.nonzero(s["ids"] >= 0).squeeze(1)
        out[live] = s["W"].index_select(0, s["ids"][live]) * s["scale"]
        return out
    if op == "embed_bwd":
        # rows in the order of their ids: differences of a running sum at the ends of each id
        live = torch.nonzero(s["ids"] >= 0).squeeze(1)
        order = live[torch.argsort(s["ids"][live], stable=True)]
        total = torch.zeros((order.numel() + 1, case["D"]), dtype=torch.float64, device="cuda")
        total[1:] = torch.cumsum(s["dout"][order], 0)
        end = torch.cumsum(torch.bincount(s["ids"][live], minlength=s["V"]), 0)
        begin = torch.cat([end.new_zeros(1), end[:-1]])
        return (total[end] - total[begin]) * s["scale"]
    if op.startswith("norm"):
        return _exact_norm(s)
    return _exact_distill(case, s)


def _exact_norm(s):
    b, gate = s["b"], s["gate"]
    g = torch.ones((1, 1), dtype=torch.float64, device="cuda") if gate is None else gate
    if s["op"] == "norm_fwd":
        u = b / (b.pow(2).sum(1, keepdim=True) / b.shape[1] + EPS).sqrt() * s["w_post"]
        h = s["x"] * s["alpha"] + u * g
        return h, h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * s["w_next"]
    # with hat = v * rstd: the gradient through v * rstd is rstd * (d - hat * mean(d * hat))
    hat2, hat1 = s["h"] * s["r2"][:, None], b * s["r1"][:, None]
    d2 = s["dy"] * s["w_next"]
    dH = s["dh"] + s["r2"][:, None] * (d2 - hat2 * (d2 * hat2).mean(1, keepdim=True))
    d1 = dH * g * s["w_post"]
    out = [dH * s["alpha"], s["r1"][:, None] * (d1 - hat1 * (d1 * hat1).mean(1, keepdim=True)),
           torch.einsum("rd,rd->d", dH * g, hat1), torch.einsum("rd,rd->d", s["dy"], hat2)]
    if gate is not None:
        full = dH * hat1 * s["w_post"]
        out.append(full.sum_to_size(gate.shape) if gate.dim() == 2 or gate.numel() != 1 else full.sum().reshape(1))
    return out


def _exact_distill(case, s):
    x, N, tau, alpha = s["logits"], case["N"], s["tau"], s["alpha"]
    w = torch.full((N,), 1.0 / N, dtype=torch.float64, device="cuda")
    if s["weight"] is not None:
        w = w * s["weight"]
    kd_sum = ce_sum = 0.0
    d = torch.zeros_like(x) if s["grad"] else None
    for r0 in range(0, N, 1024):
        r = slice(r0, min(N, r0 + 1024))
        lq, l1 = torch.log_softmax(x[r] / tau, 1), torch.log_softmax(x[r], 1)
        # teacher probabilities laid out over the vocabulary
        dense = torch.full_like(lq, -math.inf)
        row, col = torch.nonzero(s["ids"][r] >= 0, as_tuple=True)
        dense[row, s["ids"][r][row, col].long()] = s["top"][r][row, col] / tau
        P = torch.nan_to_num(torch.softmax(dense, 1), nan=0.0)
        has = P.sum(1, keepdim=True)
        ent = torch.xlogy(P, P).sum(1)
        kd_sum = kd_sum + (w[r] * (ent - (P * lq).sum(1))).sum()
        onehot = torch.zeros_like(lq)
        lab = torch.nonzero(s["labels"][r] >= 0).squeeze(1)
        onehot[lab, s["labels"][r][lab]] = 1.0
        ce_sum = ce_sum - (w[r] * (onehot * l1).sum(1)).sum()
        if d is not None:
            d[r] = w[r][:, None] * (alpha * tau * (has * lq.exp() - P)
                                    + (1 - alpha) * (onehot.sum(1, keepdim=True) * l1.exp() - onehot))
    return torch.stack([alpha * tau * tau * kd_sum + (1 - alpha) * ce_sum, kd_sum, ce_sum]), d
