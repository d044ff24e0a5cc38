"""Thin torch-tensor front end over the C ABI (libbrk.so) for tests and benchmarks.

torch is used for device memory and streams only; every operator below is one or more calls
into the hand-written CUDA kernels.  Nothing here computes on the host or through torch ops,
and a missing library or a non-CUDA tensor raises.
"""
import torch

from . import brk

_DT = {torch.float32: brk.F32, torch.float16: brk.F16}


def _dt(t):
    if t.dtype not in _DT:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return _DT[t.dtype]


def _chk(*ts):
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("blackriver_b200 operators run on CUDA tensors only (no CPU path)")
        if not t.is_contiguous():
            raise RuntimeError("tensors must be contiguous")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def layernorm(x, gamma, beta, eps=1e-5, out=None):
    _chk(x, gamma, beta, out)
    h = x.shape[-1]
    rows = x.numel() // h
    y = torch.empty_like(x) if out is None else out
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    var = torch.empty(rows, dtype=torch.float32, device=x.device)
    brk.call("brk_layernorm_fwd", _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), _ptr(mean), _ptr(var), rows, h, eps,
             _dt(x), stream())
    return y, mean, var


def layernorm_backward(dy, gamma, beta, var, y, eps=1e-5, dgamma=None, dbeta=None, dx=None, accumulate=False,
                       workspace=None, residual=None):
    _chk(dy, gamma, beta, var, y, dgamma, dbeta, dx, workspace, residual)
    h = dy.shape[-1]
    rows = dy.numel() // h
    dgamma = torch.empty_like(gamma) if dgamma is None else dgamma
    dbeta = torch.empty_like(beta) if dbeta is None else dbeta
    dx = torch.empty_like(dy) if dx is None else dx
    need = brk.lib().brk_layernorm_bwd_workspace_bytes(rows, h)
    if workspace is None:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dy.device)
    if residual is None:
        brk.call("brk_layernorm_bwd", _ptr(dy), _ptr(gamma), _ptr(beta), _ptr(var), _ptr(y), _ptr(dgamma), _ptr(dbeta),
                 _ptr(dx), rows, h, eps, _ptr(workspace), workspace.numel() * workspace.element_size(), int(accumulate),
                 _dt(dy), stream())
    else:
        brk.call("brk_layernorm_bwd_residual", _ptr(dy), _ptr(gamma), _ptr(beta), _ptr(var), _ptr(y), _ptr(residual), _ptr(dgamma),
                 _ptr(dbeta), _ptr(dx), rows, h, eps, _ptr(workspace), workspace.numel() * workspace.element_size(),
                 int(accumulate), _dt(dy), stream())
    return dgamma, dbeta, dx


def gelu(x, out=None):
    _chk(x, out)
    y = torch.empty_like(x) if out is None else out
    brk.call("brk_gelu_fwd", _ptr(x), _ptr(y), x.numel(), _dt(x), stream())
    return y


def gelu_backward(dy, x, out=None):
    _chk(dy, x, out)
    dx = torch.empty_like(x) if out is None else out
    brk.call("brk_gelu_bwd", _ptr(dy), _ptr(x), _ptr(dx), x.numel(), _dt(x), stream())
    return dx


def logsoftmax_nll(logits, target, row_loss=None, row_lse=None):
    _chk(logits, target, row_loss, row_lse)
    rows, vocab = logits.shape
    row_loss = torch.empty(rows, dtype=torch.float32, device=logits.device) if row_loss is None else row_loss
    brk.call("brk_logsoftmax_nll_fwd", _ptr(logits), _ptr(target), _ptr(row_loss), _ptr(row_lse), rows, vocab,
             _dt(logits), stream())
    return row_loss


def logsoftmax_nll_backward(logits, target, grad_scale, row_loss=None, dlogits=None):
    _chk(logits, target, row_loss, dlogits)
    rows, vocab = logits.shape
    row_loss = torch.empty(rows, dtype=torch.float32, device=logits.device) if row_loss is None else row_loss
    dlogits = torch.empty_like(logits) if dlogits is None else dlogits
    brk.call("brk_logsoftmax_nll_fwd_bwd", _ptr(logits), _ptr(target), _ptr(row_loss), _ptr(dlogits), rows, vocab,
             float(grad_scale), _dt(logits), stream())
    return row_loss, dlogits


def sum_f32(x, out=None):
    _chk(x, out)
    out = torch.empty(1, dtype=torch.float32, device=x.device) if out is None else out
    brk.call("brk_sum_f32", _ptr(x), _ptr(out), x.numel(), stream())
    return out


def loss_targets(ids, mask):
    _chk(ids, mask)
    b, t = ids.shape
    target = torch.empty_like(ids)
    count = torch.empty(1, dtype=torch.int32, device=ids.device)
    brk.call("brk_loss_targets", _ptr(ids), _ptr(mask), _ptr(target), _ptr(count), b, t, stream())
    return target, count


def add(a, b, out=None):
    _chk(a, b, out)
    c = torch.empty_like(a) if out is None else out
    brk.call("brk_add_bcast", _ptr(a), _ptr(b), _ptr(c), brk.dims4(a.shape), brk.dims4(b.shape), _dt(a), stream())
    return c


def fill(x, value):
    _chk(x)
    brk.call("brk_fill", _ptr(x), float(value), x.numel(), _dt(x), stream())
    return x


def cast(x, dtype):
    _chk(x)
    y = torch.empty(x.shape, dtype=dtype, device=x.device)
    brk.call("brk_cast", _ptr(x), _dt(x), _ptr(y), _DT[dtype], x.numel(), stream())
    return y


def transpose_0213(x, out=None):
    _chk(x, out)
    a, b, c, d = x.shape
    y = torch.empty((a, c, b, d), dtype=x.dtype, device=x.device) if out is None else out
    brk.call("brk_transpose_0213", _ptr(x), _ptr(y), a, b, c, d, _dt(x), stream())
    return y


def colsum(x, out=None, accumulate=False):
    _chk(x, out)
    rows, cols = x.shape
    out = torch.empty(cols, dtype=x.dtype, device=x.device) if out is None else out
    brk.call("brk_colsum", _ptr(x), _ptr(out), rows, cols, int(accumulate), _dt(x), stream())
    return out


def softmax(x, out=None):
    _chk(x, out)
    cols = x.shape[-1]
    y = torch.empty_like(x) if out is None else out
    brk.call("brk_softmax_fwd", _ptr(x), _ptr(y), x.numel() // cols, cols, _dt(x), stream())
    return y


def softmax_backward(dy, out, dx=None):
    _chk(dy, out, dx)
    cols = dy.shape[-1]
    dx = torch.empty_like(dy) if dx is None else dx
    brk.call("brk_softmax_bwd", _ptr(dy), _ptr(out), _ptr(dx), dy.numel() // cols, cols, _dt(dy), stream())
    return dx


def embedding_gather(table, ids):
    _chk(table, ids)
    vocab, h = table.shape
    out = torch.empty(tuple(ids.shape) + (h,), dtype=table.dtype, device=table.device)
    brk.call("brk_embedding_gather", _ptr(table), _ptr(ids), _ptr(out), ids.numel(), h, vocab, _dt(table), stream())
    return out


def alibi(heads, tokens, device="cuda"):
    import ctypes as C
    sl = (C.c_double * heads)()
    brk.lib().brk_alibi_slopes(heads, sl)
    slopes = torch.tensor(list(sl), dtype=torch.float64, device=device)
    out = torch.empty((1, heads, 1, tokens), dtype=torch.float32, device=device)
    brk.call("brk_alibi_build", _ptr(slopes), _ptr(out), heads, tokens, stream())
    return out


def xmask(mask):
    _chk(mask)
    b, t = mask.shape
    out = torch.empty((b, 1, t, t), dtype=torch.float32, device=mask.device)
    brk.call("brk_xmask_build", _ptr(mask), _ptr(out), b, t, stream())
    return out


def gemm(a, b, c, m, n, k, trans_a, trans_b, lda, ldb, ldc, batch=1, sa=0, sb=0, sc=0, alpha=1.0, beta=0.0, bias=None):
    _chk(a, b, c, bias)
    brk.call("brk_gemm", _ptr(a), _ptr(b), _ptr(c), m, n, k, int(trans_a), int(trans_b), lda, ldb, ldc, batch, sa, sb, sc,
             float(alpha), float(beta), _ptr(bias), _dt(a), stream())
    return c


def gemm_f16(a, b, c, m, n, k, trans_a, trans_b, lda, ldb, ldc, bias=None, residual=None, ldr=0, gelu_out=None, ldg=0,
             accumulate=False):
    """fp16 tensor-core GEMM (tcgen05/TMEM); raises if the layout is not supported."""
    _chk(a, b, c, bias, residual, gelu_out)
    brk.call("brk_gemm_f16", _ptr(a), _ptr(b), _ptr(c), m, n, k, int(trans_a), int(trans_b), lda, ldb, ldc, _ptr(bias),
             _ptr(residual), ldr, _ptr(gelu_out), ldg, int(accumulate), stream())
    return c


# --- packed documents ---
def _chk_all(expect, **named):
    """Each tensor (None passes): contiguous, on the current device, of its dtype and shape in `expect`."""
    for name, t in named.items():
        if t is None:
            continue
        _chk(t)
        _chk_device(t)
        dtype, shape = expect[name]
        if t.dtype != dtype or tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _chk_device(t):
    if t.device.index != torch.cuda.current_device():
        raise RuntimeError("tensors must live on the current device, whose stream the kernels are queued on")


def doc_plan(mask, prompt=None, ids=None):
    """Spans of packed documents: mask [batch, tokens] int32 numbers the documents (0 or less = padding), prompt marks
    the tokens of prompts.  Returns int32 spans [batch, tokens, 4] for doc_attn; with ids also the loss targets and their
    count: (spans, target, count)."""
    if mask.dim() != 2:
        raise ValueError("mask must be [batch, tokens]")
    like = (torch.int32, mask.shape)
    _chk_all({"mask": like, "prompt": like, "ids": like}, mask=mask, prompt=prompt, ids=ids)
    b, t = mask.shape
    spans = torch.empty((b, t, 4), dtype=torch.int32, device=mask.device)
    target = count = None
    if ids is not None:
        target = torch.empty_like(ids)
        count = torch.empty(1, dtype=torch.int32, device=ids.device)
    brk.call("brk_doc_plan", _ptr(mask), _ptr(prompt), _ptr(ids), b, t, _ptr(spans), _ptr(target), _ptr(count), stream())
    return spans if ids is None else (spans, target, count)


def _heads_view(name, t, batch, tokens, heads, dim):
    """Row stride of a [batch, tokens, heads, head_dim] fp16 tensor whose heads lie side by side in a token's row."""
    if not t.is_cuda:
        raise RuntimeError("blackriver_b200 operators run on CUDA tensors only (no CPU path)")
    _chk_device(t)
    if t.dtype != torch.float16:
        raise TypeError(f"unsupported dtype {t.dtype}")
    if t.dim() != 4 or t.shape[0] != batch or t.shape[1] != tokens or t.shape[3] != dim or (heads is not None and t.shape[2] != heads):
        raise ValueError(f"{name} must be [{batch}, {tokens}, {heads or 'heads'}, {dim}], got {tuple(t.shape)}")
    ld = t.stride(1) if tokens > 1 else t.stride(0) if batch > 1 else t.shape[2] * dim
    if t.numel() and ((dim > 1 and t.stride(3) != 1) or (t.shape[2] > 1 and t.stride(2) != dim) or (batch > 1 and t.stride(0) != tokens * ld)):
        raise ValueError(f"{name}: heads must lie side by side and tokens at one stride")
    return ld


def _doc_args(q, k, v, spans, slopes):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q, k and v must be [batch, tokens, heads, head_dim]")
    b, t, h, d = q.shape
    hk = k.shape[2]
    ld_q, ld_kv = _heads_view("q", q, b, t, h, d), _heads_view("k", k, b, t, hk, d)
    if _heads_view("v", v, b, t, hk, d) != ld_kv:
        raise ValueError("k and v must have the same row stride")
    _chk_all({"spans": (torch.int32, (b, t, 4)), "slopes": (torch.float32, (h,))}, spans=spans, slopes=slopes)
    return b, t, h, hk, d, ld_q, ld_kv


def doc_attn(q, k, v, spans, slopes=None, cap=0.0, out=None, lse=None):
    """Attention over packed documents: q [batch, tokens, heads, head_dim], k and v [batch, tokens, kv_heads, head_dim]
    fp16 (views of a fused projection are read in place), spans from doc_plan.  slopes [heads]: bias -slope * distance;
    cap: scores capped by cap * tanh(score / cap).  Returns (out, lse [batch, heads, tokens])."""
    b, t, h, hk, d, ld_q, ld_kv = _doc_args(q, k, v, spans, slopes)
    out = torch.empty((b, t, h, d), dtype=q.dtype, device=q.device) if out is None else out
    lse = torch.empty((b, h, t), dtype=torch.float32, device=q.device) if lse is None else lse
    ld_out = _heads_view("out", out, b, t, h, d)
    _chk_all({"lse": (torch.float32, (b, h, t))}, lse=lse)
    brk.call("brk_doc_attn_fwd", _ptr(q), _ptr(k), _ptr(v), ld_q, ld_kv, _ptr(out), ld_out, _ptr(lse), _ptr(spans), _ptr(slopes), float(cap),
             b, t, h, hk, d, stream())
    return out, lse


def doc_attn_backward(d_out, q, k, v, out, lse, spans, slopes=None, cap=0.0, dq=None, dk=None, dv=None, workspace=None):
    """Gradients (dq, dk, dv) of doc_attn; without dq, dk and dv they are views of one fused [batch, tokens, heads + 2 kv_heads,
    head_dim] buffer, as the projection's backward wants them."""
    b, t, h, hk, d, ld_q, ld_kv = _doc_args(q, k, v, spans, slopes)
    ld_out = _heads_view("out", out, b, t, h, d)
    if _heads_view("d_out", d_out, b, t, h, d) != ld_out:
        raise ValueError("out and d_out must have the same row stride")
    _chk_all({"lse": (torch.float32, (b, h, t))}, lse=lse)
    if dq is None and dk is None and dv is None:
        fused = torch.empty((b, t, h + 2 * hk, d), dtype=q.dtype, device=q.device)
        dq, dk, dv = fused[:, :, :h], fused[:, :, h:h + hk], fused[:, :, h + hk:]
    elif dq is None or dk is None or dv is None:
        raise ValueError("give all of dq, dk and dv, or none")
    ld_dq, ld_dkv = _heads_view("dq", dq, b, t, h, d), _heads_view("dk", dk, b, t, hk, d)
    if _heads_view("dv", dv, b, t, hk, d) != ld_dkv:
        raise ValueError("dk and dv must have the same row stride")
    if workspace is None:
        workspace = torch.empty(max(brk.lib().brk_doc_attn_bwd_workspace_bytes(b, t, h), 16), dtype=torch.uint8, device=q.device)
    _chk(workspace)
    _chk_device(workspace)
    brk.call("brk_doc_attn_bwd", _ptr(q), _ptr(k), _ptr(v), ld_q, ld_kv, _ptr(out), _ptr(d_out), ld_out, _ptr(lse), _ptr(dq), ld_dq, _ptr(dk),
             _ptr(dv), ld_dkv, _ptr(spans), _ptr(slopes), float(cap), b, t, h, hk, d, _ptr(workspace), workspace.numel() * workspace.element_size(), stream())
    return dq, dk, dv


# --- activations kept in 8 bits ---
ACT8_BLOCK = 128        # columns that share a scale


def _act8_shapes(rows, cols):
    return {"q": (torch.int8, (rows, cols)), "scale": (torch.float32, (rows, -(-cols // ACT8_BLOCK)))}


def _act8_new(rows, cols, device):
    return (torch.empty((rows, cols), dtype=torch.int8, device=device),
            torch.empty((rows, -(-cols // ACT8_BLOCK)), dtype=torch.float32, device=device))


def _rows_cols(t):
    if t.dim() < 1 or t.shape[-1] == 0:
        raise ValueError("activations need at least one column")
    return t.numel() // t.shape[-1], t.shape[-1]


def act8_pack(x):
    """x [..., cols] -> (q int8 [rows, cols], scale fp32 [rows, ceil(cols / 128)])."""
    _chk(x)
    _chk_device(x)
    rows, cols = _rows_cols(x)
    q, scale = _act8_new(rows, cols, x.device)
    brk.call("brk_act8_pack", _ptr(x), _ptr(q), _ptr(scale), rows, cols, _dt(x), stream())
    return q, scale


def act8_unpack(q, scale, dtype=torch.float16, out=None):
    """The kept values, [rows, cols] of `dtype` (or into out)."""
    rows, cols = _rows_cols(q)
    _chk_all(_act8_shapes(rows, cols), q=q, scale=scale)
    out = torch.empty((rows, cols), dtype=dtype, device=q.device) if out is None else out
    _chk_all({"out": (out.dtype, q.shape)}, out=out)
    brk.call("brk_act8_unpack", _ptr(q), _ptr(scale), _ptr(out), rows, cols, _dt(out), stream())
    return out


def gelu_act8(x, out=None):
    """gelu(x) and x kept in 8 bits: (y, q, scale)."""
    _chk(x, out)
    _chk_device(x)
    rows, cols = _rows_cols(x)
    y = torch.empty_like(x) if out is None else out
    _chk_all({"out": (x.dtype, x.shape)}, out=y)
    q, scale = _act8_new(rows, cols, x.device)
    brk.call("brk_gelu_fwd_act8", _ptr(x), _ptr(y), _ptr(q), _ptr(scale), rows, cols, _dt(x), stream())
    return y, q, scale


def gelu_backward_act8(dy, q, scale, out=None, recompute=False):
    """dy * gelu'(kept x); with recompute also gelu(kept x) again: dx, or (dx, y)."""
    _chk(dy, out)
    _chk_device(dy)
    rows, cols = _rows_cols(dy)
    _chk_all(_act8_shapes(rows, cols), q=q, scale=scale)
    dx = torch.empty_like(dy) if out is None else out
    _chk_all({"out": (dy.dtype, dy.shape)}, out=dx)
    y = torch.empty_like(dy) if recompute else None
    brk.call("brk_gelu_bwd_act8", _ptr(dy), _ptr(q), _ptr(scale), _ptr(dx), _ptr(y), rows, cols, _dt(dy), stream())
    return (dx, y) if recompute else dx


def layernorm_act8(x, gamma, beta, eps=1e-5, out=None):
    """LayerNorm that keeps the normalised rows in 8 bits: (y, q, scale, var)."""
    _chk(x, out)
    _chk_device(x)
    rows, cols = _rows_cols(x)
    vec = (x.dtype, (cols,))
    _chk_all({"gamma": vec, "beta": vec}, gamma=gamma, beta=beta)
    y = torch.empty_like(x) if out is None else out
    _chk_all({"out": (x.dtype, x.shape)}, out=y)
    q, scale = _act8_new(rows, cols, x.device)
    var = torch.empty(rows, dtype=torch.float32, device=x.device)
    brk.call("brk_layernorm_fwd_act8", _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), _ptr(q), _ptr(scale), _ptr(var), rows, cols, eps, _dt(x), stream())
    return y, q, scale, var


def layernorm_backward_act8(dy, gamma, var, q, scale, beta=None, residual=None, dgamma=None, dbeta=None, dx=None, accumulate=False, workspace=None):
    """LayerNorm backward from the kept rows: (dgamma, dbeta, dx), and with beta the forward's output again as a fourth."""
    _chk(dy)
    _chk_device(dy)
    rows, cols = _rows_cols(dy)
    if accumulate and (dgamma is None or dbeta is None):
        raise ValueError("accumulate needs dgamma and dbeta")
    vec, full = (dy.dtype, (cols,)), (dy.dtype, dy.shape)
    dgamma = torch.empty(cols, dtype=dy.dtype, device=dy.device) if dgamma is None else dgamma
    dbeta = torch.empty(cols, dtype=dy.dtype, device=dy.device) if dbeta is None else dbeta
    dx = torch.empty_like(dy) if dx is None else dx
    y = torch.empty_like(dy) if beta is not None else None
    _chk_all({"gamma": vec, "beta": vec, "dgamma": vec, "dbeta": vec, "var": (torch.float32, (rows,)), "residual": full, "dx": full, **_act8_shapes(rows, cols)},
             gamma=gamma, beta=beta, dgamma=dgamma, dbeta=dbeta, var=var, residual=residual, dx=dx, q=q, scale=scale)
    need = brk.lib().brk_layernorm_bwd_act8_workspace_bytes(rows, cols)
    if workspace is None:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dy.device)
    _chk(workspace)
    _chk_device(workspace)
    brk.call("brk_layernorm_bwd_act8", _ptr(dy), _ptr(gamma), _ptr(beta), _ptr(var), _ptr(q), _ptr(scale), _ptr(residual), _ptr(dgamma), _ptr(dbeta), _ptr(dx),
             _ptr(y), rows, cols, _ptr(workspace), workspace.numel() * workspace.element_size(), int(accumulate), _dt(dy), stream())
    return (dgamma, dbeta, dx) if y is None else (dgamma, dbeta, dx, y)


# --- operator-level compositions with the reference's semantics (blackriver/cuda_tensor.cpp) ---
def linear(x, w, bias, out=None):
    """op_linear (:147-193): y[n,o] = sum_i x[n,i] w[o,i] + b[o]."""
    o, i = w.shape
    n = x.numel() // i
    y = torch.empty(tuple(x.shape[:-1]) + (o,), dtype=x.dtype, device=x.device) if out is None else out
    return gemm(x, w, y, n, o, i, False, True, i, i, o, bias=bias)


def linear_backward(dy, x, w, x_g=None, w_g=None, b_g=None):
    """op_linear_backward (:731-812): b_g, then W_g = dy^T x, then x_g = dy W (x_g may alias x)."""
    o, i = w.shape
    n = x.numel() // i
    b_g = torch.empty(o, dtype=w.dtype, device=w.device) if b_g is None else b_g
    w_g = torch.empty_like(w) if w_g is None else w_g
    x_g = torch.empty_like(x) if x_g is None else x_g
    colsum(dy.view(n, o), out=b_g)
    gemm(dy, x, w_g, o, i, n, True, False, o, i, i)
    gemm(dy, w, x_g, n, i, o, False, False, o, i, i)
    return x_g, w_g, b_g


def qk(q, k, out=None):
    """op_qk (:278-330): S = Q K^T / sqrt(d), per (batch, head)."""
    b, h, t, d = q.shape
    s = torch.empty((b, h, t, t), dtype=q.dtype, device=q.device) if out is None else out
    return gemm(q, k, s, t, t, d, False, True, d, d, t, batch=b * h, sa=t * d, sb=t * d, sc=t * t, alpha=d ** -0.5)


def attn(p, v, out=None):
    """op_attn (:359-398): O = P V."""
    b, h, t, d = v.shape
    o = torch.empty_like(v) if out is None else out
    return gemm(p, v, o, t, d, t, False, False, t, d, d, batch=b * h, sa=t * t, sb=t * d, sc=t * d)


def softmax_attn_backward(dout, p, v, ds=None, dv=None):
    """op_softmax_attn_backward (:921-1002): dV = P^T dO; dS = softmax_bwd(P, dO V^T); ds may be p."""
    b, h, t, d = v.shape
    dv = torch.empty_like(v) if dv is None else dv
    ds = torch.empty_like(p) if ds is None else ds
    gemm(p, dout, dv, t, d, t, True, False, t, d, d, batch=b * h, sa=t * t, sb=t * d, sc=t * d)
    dp = torch.empty_like(p)
    gemm(dout, v, dp, t, t, d, False, True, d, d, t, batch=b * h, sa=t * d, sb=t * d, sc=t * t)
    softmax_backward(dp, p, dx=ds)
    return ds, dv


def qk_backward(ds, q, k, dq=None, dk=None):
    """op_qk_backward (:1005-1063): dQ = dS K / sqrt(d); dK = dS^T Q / sqrt(d)."""
    b, h, t, d = q.shape
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    sc = d ** -0.5
    gemm(ds, k, dq, t, d, t, False, False, t, d, d, batch=b * h, sa=t * t, sb=t * d, sc=t * d, alpha=sc)
    gemm(ds, q, dk, t, d, t, True, False, t, d, d, batch=b * h, sa=t * t, sb=t * d, sc=t * d, alpha=sc)
    return dq, dk
