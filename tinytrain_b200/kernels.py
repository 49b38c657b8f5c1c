"""Thin torch-tensor front end over the ttk C ABI (include/ttk.h).

torch provides device memory and the current stream; every computation is a
ttk_* call into libttk.so. Used by the parity tests and the benchmark to drive
single kernels; the training path itself runs in the C++ tt:: library.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _ttk
from ._ttk import call


def _s():
    """The current stream's handle (torch.cuda.current_stream().cuda_stream, without the
    Stream object: 0.2 instead of 3.2 us)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _p(t):
    return None if t is None else t.data_ptr()


def _chk(t, name, dtype=torch.float32, shape=None):
    if not (t.is_cuda and t.dtype == dtype and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous {str(dtype).split('.')[-1]} CUDA tensor")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")


def _chk_all(names, shape, *tensors):
    """_chk(t, name, shape=shape) of every tensor that is not None, cheaply: small calls are
    bound by the host."""
    for t in tensors:
        if t is not None and (t.shape != shape or t.dtype != torch.float32 or
                              not t.is_contiguous() or not t.is_cuda):
            for name, u in zip(names, tensors):
                if u is t:
                    _chk(t, name, shape=shape)


@functools.lru_cache(maxsize=1024)
def _ws_size(fn, *sizes):
    """Workspace size functions whose result depends on the sizes alone."""
    return max(call(fn, *sizes), 16)


def workspace(nbytes: int, device=None) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device or "cuda")


def gemm(A, B, transA=False, transB=False, C_out=None, alpha=1.0, beta=0.0):
    """op(A) @ op(B) (+ beta*C) for 2-D or 3-D (batched) row-major tensors."""
    batched = A.dim() == 3
    if not batched:
        A, B = A.unsqueeze(0), B.unsqueeze(0)
    bt = A.shape[0]
    M, K = (A.shape[2], A.shape[1]) if transA else (A.shape[1], A.shape[2])
    N = B.shape[1] if transB else B.shape[2]
    if C_out is None:
        C_out = torch.empty((bt, M, N), dtype=torch.float32, device=A.device)
        beta = 0.0
    elif not batched:
        C_out = C_out.unsqueeze(0)
    ws_n = call("ttk_gemm_workspace_size", int(transA), int(transB), bt, M, N, K)
    ws = workspace(ws_n, A.device)
    call("ttk_gemm", int(transA), int(transB), bt, M, N, K, alpha, _p(A), A.shape[2],
         A.shape[1] * A.shape[2], _p(B), B.shape[2], B.shape[1] * B.shape[2], beta, _p(C_out),
         N, M * N, _p(ws), ws.numel(), _s())
    return C_out if batched else C_out[0]


def linear_fwd(X, W):
    """Y = X @ W^T (nn.cpp:23-26)."""
    return gemm(X, W, transB=True)


def linear_bwd(X, W, dY):
    """dX = dY @ W, dW = dY^T @ X (ops.cpp:672-694 through the transpose)."""
    return gemm(dY, W), gemm(dY, X, transA=True)


def rmsnorm_fwd(x, w, eps):
    R, D = x.shape
    y = torch.empty_like(x)
    rstd = torch.empty(R, dtype=torch.float32, device=x.device)
    call("ttk_rmsnorm_fwd", _p(x), _p(w), _p(y), _p(rstd), R, D, eps, _s())
    return y, rstd


def rmsnorm_fwd_split(x, w, eps):
    """(y, rstd, planes): the forward plus y's bf16x3 GEMM operand planes."""
    R, D = x.shape
    y = torch.empty_like(x)
    rstd = torch.empty(R, dtype=torch.float32, device=x.device)
    planes = workspace(call("ttk_gemm_split_bytes", 1, R, D), x.device)
    call("ttk_rmsnorm_fwd_split", _p(x), _p(w), _p(y), _p(rstd), R, D, eps, _p(planes), _s())
    return y, rstd, planes


def gemm_split(x):
    """bf16x3 operand planes of a 2-D fp32 tensor (ttk_gemm_split)."""
    R, D = x.shape
    planes = workspace(call("ttk_gemm_split_bytes", 1, R, D), x.device)
    call("ttk_gemm_split", _p(x), R, D, D, 0, 1, _p(planes), _s())
    return planes


def rmsnorm_bwd(x, w, rstd, dy, dx=None, dw=None, accumulate=False):
    R, D = x.shape
    if dx is None:
        dx = torch.empty_like(x)
    if dw is None:
        dw = torch.zeros_like(w)
    ws_n = call("ttk_rmsnorm_bwd_workspace_size", R, D)
    ws = workspace(ws_n, x.device)
    call("ttk_rmsnorm_bwd", _p(x), _p(w), _p(rstd), _p(dy), _p(dx), int(accumulate), _p(dw), R, D,
         _p(ws), ws.numel(), _s())
    return dx, dw


def swiglu_fwd(a, b):
    y = torch.empty_like(a)
    call("ttk_swiglu_fwd", _p(a), _p(b), _p(y), a.numel(), _s())
    return y


def swiglu_bwd(a, b, dy, da=None, db=None, accumulate=False):
    da = torch.empty_like(a) if da is None else da
    db = torch.empty_like(b) if db is None else db
    call("ttk_swiglu_bwd", _p(a), _p(b), _p(dy), _p(da), _p(db), int(accumulate), a.numel(), _s())
    return da, db


def cross_entropy(logits, targets, want_grad=True, dlogits=None):
    """Mean CE loss (ops.cpp:928-930) and d(loss)/d(logits) for d(loss) = 1."""
    N, Cn = logits.shape
    acc = torch.zeros(1, dtype=torch.float64, device=logits.device)
    if want_grad and dlogits is None:
        dlogits = torch.empty_like(logits)
    call("ttk_cross_entropy", _p(logits), _p(targets), N, Cn, _p(acc),
         _p(dlogits) if want_grad else None, 1.0 / N, _s())
    loss = torch.empty(1, dtype=torch.float32, device=logits.device)
    call("ttk_loss_finalize", _p(acc), 1.0 / N, _p(loss), _s())
    return loss, dlogits


def embedding_fwd(W, idx):
    V, D = W.shape
    N = idx.numel()
    out = torch.empty((N, D), dtype=torch.float32, device=W.device)
    call("ttk_embedding_fwd", _p(W), _p(idx), _p(out), N, D, V, _s())
    return out


def embedding_bwd(dout, idx, dW):
    V, D = dW.shape
    N = idx.numel()
    ws = workspace(call("ttk_embedding_bwd_workspace_size", N), dW.device)
    call("ttk_embedding_bwd", _p(dout), _p(idx), _p(dW), N, D, V, _p(ws), ws.numel(), _s())
    return dW


def embedding_scaled_fwd(W, idx, scale=1.0):
    """scale * W[idx] ([N, D]); idx -1 gives a zero row."""
    _chk(W, "W")
    _chk(idx, "idx", torch.int64)
    V, D = W.shape
    N = idx.numel()
    out = W.new_empty((N, D))
    call("ttk_embedding_scaled_fwd", W.data_ptr(), idx.data_ptr(), out.data_ptr(), N, D, V, scale,
         _s())
    return out


def embedding_scaled_bwd(dout, idx, V, scale=1.0, dW=None, accumulate=False):
    """Gradient of embedding_scaled_fwd for W [V, D], by sorted tokens: written
    into dW (zero rows for tokens that do not occur) or, with accumulate,
    added to it."""
    _chk(dout, "dout")
    _chk(idx, "idx", torch.int64)
    N, D = dout.shape
    if idx.numel() != N:
        raise ValueError(f"idx: expected {N} ids, got {idx.numel()}")
    if dW is not None:
        _chk(dW, "dW", shape=(V, D))
    else:
        dW = dout.new_zeros((V, D)) if accumulate else dout.new_empty((V, D))
    n = _ws_size("ttk_embedding_scaled_bwd_workspace_size", N, D, V)
    ws = dout.new_empty(n, dtype=torch.uint8)
    call("ttk_embedding_scaled_bwd", dout.data_ptr(), idx.data_ptr(), dW.data_ptr(),
         int(accumulate), N, D, V, scale, ws.data_ptr(), n, _s())
    return dW


def _gate_kind(gate, R, D):
    """TTK_GATE_* of a gate tensor: None, [1], [D], [R, 1] or [R, D]."""
    if gate is None:
        return 0
    _chk(gate, "gate")
    shape = tuple(gate.shape)
    if shape == (1,):
        return 1
    if shape == (D,):
        return 2
    if shape == (R, 1):
        return 3
    if shape == (R, D):
        return 4
    raise ValueError(f"gate: expected [1], [{D}], [{R}, 1] or [{R}, {D}], got {list(shape)}")


def residual_norm_fwd(x, b, w_post, w_next=None, gate=None, residual_scale=1.0, eps=1e-5,
                      planes=False):
    """(h, y, rstd_post, rstd_next): h = residual_scale * x + gate * rmsnorm(b, w_post),
    y = rmsnorm(h, w_next). Without w_next y and rstd_next are None. gate: None, [1], [D],
    [R, 1] or [R, D]. With planes also the bf16x3 GEMM operand planes of y."""
    R, D = x.shape
    _chk_all(("x", "b"), (R, D), x, b)
    _chk_all(("w_post", "w_next"), (D,), w_post, w_next)
    kind = _gate_kind(gate, R, D)
    h, r1 = torch.empty_like(x), x.new_empty(R)
    y, r2 = (None, None) if w_next is None else (torch.empty_like(x), x.new_empty(R))
    split = workspace(call("ttk_gemm_split_bytes", 1, R, D), x.device) if planes else None
    call("ttk_residual_norm_fwd", x.data_ptr(), b.data_ptr(), w_post.data_ptr(), _p(gate), kind,
         _p(w_next), h.data_ptr(), _p(y), r1.data_ptr(), _p(r2), _p(split), R, D, residual_scale,
         eps, _s())
    return (h, y, r1, r2, split) if planes else (h, y, r1, r2)


def residual_norm_bwd(dh, dy, h, b, w_post, w_next, rstd_post, rstd_next, gate=None,
                      residual_scale=1.0, dx=None, db=None, dw_post=None, dw_next=None,
                      dgate=None):
    """(dx, db, dw_post, dw_next, dgate) of residual_norm_fwd; dh or dy may be None (no gradient
    there). Output tensors that are given are added to; dgate is None without a gate (and refused
    if given), dw_next without dy (and left as it is if given: nothing is added)."""
    R, D = b.shape
    _chk_all(("dh", "dy", "h", "b", "dx", "db"), (R, D), dh, dy, h, b, dx, db)
    _chk_all(("w_post", "w_next", "dw_post", "dw_next"), (D,), w_post, w_next, dw_post, dw_next)
    _chk_all(("rstd_post", "rstd_next"), (R,), rstd_post, rstd_next)
    kind = _gate_kind(gate, R, D)
    acc = 0
    if dx is None:
        dx = torch.empty_like(b)
    else:
        acc |= 1
    if db is None:
        db = torch.empty_like(b)
    else:
        acc |= 2
    if dw_post is None and dw_next is None:
        dw_post = torch.empty_like(w_post)
        dw_next = None if dy is None else torch.empty_like(w_post)
    else:  # one flag covers both weights' gradients
        acc |= 4
        dw_post = torch.zeros_like(w_post) if dw_post is None else dw_post
        if dw_next is None and dy is not None:
            dw_next = torch.zeros_like(w_post)
    if gate is None:
        if dgate is not None:
            raise ValueError("dgate: there is no gate")
    elif dgate is None:
        dgate = torch.empty_like(gate)
    else:
        _chk(dgate, "dgate", shape=gate.shape)
        acc |= 8
    n = _ws_size("ttk_residual_norm_bwd_workspace_size", R, D)
    ws = b.new_empty(n, dtype=torch.uint8)
    call("ttk_residual_norm_bwd", _p(dh), _p(dy), _p(h), b.data_ptr(), w_post.data_ptr(), _p(gate),
         kind, _p(w_next), rstd_post.data_ptr(), _p(rstd_next), dx.data_ptr(), db.data_ptr(),
         dw_post.data_ptr(), None if dy is None else dw_next.data_ptr(), _p(dgate), acc, R, D,
         residual_scale, ws.data_ptr(), n, _s())
    return dx, db, dw_post, dw_next, dgate


_TEACHER_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def distill_loss(logits, teacher_ids, teacher_logits, targets=None, alpha=1.0, temperature=1.0,
                 row_weight=None, grad_scale=None, want_grad=True, dlogits=None):
    """(loss, dlogits): loss [3] = {alpha T^2 kd + (1 - alpha) ce, kd, ce}, sums over the rows
    times grad_scale (default 1 / N), kd against the teacher's top lists (ids [N, K] int32 with -1
    for no entry, logits [N, K] fp32, bf16 or fp16) and ce against targets (int64, -1 for none).
    logits [N, C] and dlogits may be views of wider rows (stride(1) = 1); dlogits may be logits."""
    N, C = logits.shape
    K = teacher_ids.shape[1]
    for t, name in ((logits, "logits"), (dlogits, "dlogits")):
        if t is not None and not (t.is_cuda and t.dtype == torch.float32 and
                                  tuple(t.shape) == (N, C) and (t.stride(1) == 1 or C == 1) and
                                  (t.stride(0) >= C or N <= 1)):
            raise ValueError(f"{name}: expected float32 CUDA rows [{N}, {C}] of unit stride")
    if teacher_logits.dtype not in _TEACHER_TYPES:
        raise ValueError("teacher_logits: expected float32, bfloat16 or float16")
    _chk(teacher_ids, "teacher_ids", torch.int32, (N, K))
    _chk(teacher_logits, "teacher_logits", teacher_logits.dtype, (N, K))
    if targets is not None:
        _chk(targets, "targets", torch.int64, (N,))
    if row_weight is not None:
        _chk(row_weight, "row_weight", shape=(N,))
    if want_grad and dlogits is None:
        dlogits = logits.new_empty((N, C))
    loss = logits.new_empty(3)
    n = _ws_size("ttk_distill_loss_workspace_size", N)
    ws = logits.new_empty(n, dtype=torch.uint8)
    call("ttk_distill_loss", logits.data_ptr(), max(logits.stride(0), C), teacher_ids.data_ptr(),
         teacher_logits.data_ptr(), _TEACHER_TYPES[teacher_logits.dtype], K, _p(targets),
         _p(row_weight), N, C, alpha, temperature, 1.0 / max(N, 1) if grad_scale is None else
         grad_scale, loss.data_ptr(), dlogits.data_ptr() if want_grad else None,
         max(dlogits.stride(0), C) if want_grad else 0, ws.data_ptr(), n, _s())
    return loss, dlogits if want_grad else None


def rope_fwd(x, cos, sin):
    B, T, H, D = x.shape
    y = torch.empty_like(x)
    call("ttk_rope_fwd", _p(x), _p(cos), _p(sin), _p(y), B, T, H, D, _s())
    return y


def rope_bwd(dy, cos, sin, dx=None, accumulate=False):
    B, T, H, D = dy.shape
    dx = torch.empty_like(dy) if dx is None else dx
    call("ttk_rope_bwd", _p(dy), _p(cos), _p(sin), _p(dx), int(accumulate), B, T, H, D, _s())
    return dx


def softmax_fwd(x, log=False):
    R, Cn = x.shape
    y = torch.empty_like(x)
    call("ttk_softmax_fwd", _p(x), _p(y), R, Cn, int(log), _s())
    return y


def softmax_bwd(y, dy, log=False, dx=None, accumulate=False):
    R, Cn = y.shape
    dx = torch.empty_like(y) if dx is None else dx
    call("ttk_softmax_bwd", _p(y), _p(dy), _p(dx), int(accumulate), R, Cn, int(log), _s())
    return dx


def rope_tables(T, hd, theta, device):
    """model.cpp:43-53 in float32 (computed on the host, as the model does)."""
    import numpy as np
    i = np.arange(hd // 2, dtype=np.float32)
    inv = np.float32(1) / np.power(np.float32(theta), (np.float32(2) * i) / np.float32(hd),
                                   dtype=np.float32)
    ang = np.arange(T, dtype=np.float32)[:, None] * inv[None, :]
    return (torch.from_numpy(np.cos(ang).astype(np.float32)).to(device),
            torch.from_numpy(np.sin(ang).astype(np.float32)).to(device))


def attention_fwd(q, k, v, cos, sin, scale=None, keep_ws=False):
    """(o, lse); with keep_ws also the workspace (q, k, v planes) for attention_bwd(fwd_ws=)."""
    B, T, H, hd = q.shape
    scale = float(hd) ** -0.5 if scale is None else scale
    o = torch.empty_like(q)
    lse = torch.empty((B, H, T), dtype=torch.float32, device=q.device)
    ws = workspace(call("ttk_attention_fwd_workspace_size", B, T, H, hd), q.device)
    call("ttk_attention_fwd", _p(q), _p(k), _p(v), _p(cos), _p(sin), _p(o), _p(lse), B, T, H, hd,
         scale, _p(ws), ws.numel(), _s())
    return (o, lse, ws) if keep_ws else (o, lse)


def attention_fwd_split(q, k, v, cos, sin, scale=None):
    """(o, lse, planes): the forward plus o's bf16x3 operand planes ([B*T, H*hd])."""
    B, T, H, hd = q.shape
    scale = float(hd) ** -0.5 if scale is None else scale
    o = torch.empty_like(q)
    lse = torch.empty((B, H, T), dtype=torch.float32, device=q.device)
    ws = workspace(call("ttk_attention_fwd_workspace_size", B, T, H, hd), q.device)
    planes = workspace(call("ttk_gemm_split_bytes", 1, B * T, H * hd), q.device)
    call("ttk_attention_fwd_split", _p(q), _p(k), _p(v), _p(cos), _p(sin), _p(o), _p(lse),
         _p(planes), B, T, H, hd, scale, _p(ws), ws.numel(), _s())
    return o, lse, planes


def attention_bwd(q, k, v, cos, sin, o, lse, do, scale=None, out=None, accumulate=False,
                  fwd_ws=None):
    """dq, dk, dv; with `out` = (dq, dk, dv) writes (or, with accumulate, adds) into them.
    fwd_ws: the forward's workspace (attention_fwd(keep_ws=True)), whose q, k, v planes are
    reused."""
    B, T, H, hd = q.shape
    scale = float(hd) ** -0.5 if scale is None else scale
    dq, dk, dv = out if out is not None else (torch.empty_like(q), torch.empty_like(k),
                                               torch.empty_like(v))
    if fwd_ws is not None and fwd_ws.numel() > 0:
        ws = workspace(call("ttk_attention_bwd_ex_workspace_size", B, T, H, hd), q.device)
        call("ttk_attention_bwd_ex", _p(q), _p(k), _p(v), _p(cos), _p(sin), _p(o), _p(lse),
             _p(do), _p(dq), _p(dk), _p(dv), int(accumulate), B, T, H, hd, scale, _p(fwd_ws),
             _p(ws), ws.numel(), _s())
        return dq, dk, dv
    ws = workspace(call("ttk_attention_bwd_workspace_size", B, T, H, hd), q.device)
    call("ttk_attention_bwd", _p(q), _p(k), _p(v), _p(cos), _p(sin), _p(o), _p(lse), _p(do),
         _p(dq), _p(dk), _p(dv), int(accumulate), B, T, H, hd, scale, _p(ws), ws.numel(), _s())
    return dq, dk, dv


def attention_bwd_split(q, k, v, cos, sin, o, lse, do, scale=None, out=None, accumulate=False,
                        fwd_ws=None):
    """(dq, dk, dv, planes): the backward plus the bf16x3 operand planes of dq,
    dk, dv, each as [B*T, H*hd] rows."""
    B, T, H, hd = q.shape
    scale = float(hd) ** -0.5 if scale is None else scale
    dq, dk, dv = out if out is not None else (torch.empty_like(q), torch.empty_like(k),
                                               torch.empty_like(v))
    reuse = fwd_ws is not None and fwd_ws.numel() > 0
    ws = workspace(call("ttk_attention_bwd_ex_workspace_size" if reuse else
                        "ttk_attention_bwd_workspace_size", B, T, H, hd), q.device)
    pb = call("ttk_gemm_split_bytes", 1, B * T, H * hd)
    planes = [workspace(pb, q.device) for _ in range(3)]
    call("ttk_attention_bwd_split", _p(q), _p(k), _p(v), _p(cos), _p(sin), _p(o), _p(lse),
         _p(do), _p(dq), _p(dk), _p(dv), int(accumulate), B, T, H, hd, scale,
         _p(fwd_ws) if reuse else None, _p(ws), ws.numel(), *(_p(x) for x in planes), _s())
    return dq, dk, dv, planes


def sumsq(tensors):
    acc = torch.zeros(1, dtype=torch.float64, device=tensors[0].device)
    ptrs = _ttk.ptr_array([t.data_ptr() for t in tensors])
    sizes = _ttk.i64_array([t.numel() for t in tensors])
    call("ttk_sumsq_multi", ptrs, sizes, len(tensors), _p(acc), _s())
    return acc


def adamw(params, grads, ms, vs, lr, b1, b2, eps, wd, step, sumsq_acc=None, max_norm=0.0,
          grad_scale=1.0):
    n = len(params)
    call("ttk_adamw_multi", _ttk.ptr_array([p.data_ptr() for p in params]),
         _ttk.ptr_array([g.data_ptr() for g in grads]), _ttk.ptr_array([m.data_ptr() for m in ms]),
         _ttk.ptr_array([v.data_ptr() for v in vs]), _ttk.i64_array([p.numel() for p in params]),
         n, lr, b1, b2, eps, wd, step, _p(sumsq_acc), max_norm, grad_scale, _s())
