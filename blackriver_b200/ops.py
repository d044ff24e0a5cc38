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
    # the raw handle without a Stream object around it, which takes 3 us to make
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


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
# These calls are short enough for their front end to be seen: one look at each tensor, and words only where one is refused.
def _device(t):
    """The current device, which `t` has to be on: the kernels are queued on its current stream."""
    if not t.is_cuda:
        raise RuntimeError("blackriver_b200 operators run on CUDA tensors only (no CPU path)")
    device = torch._C._cuda_getDevice()
    if t.get_device() != device:
        raise RuntimeError("tensors must live on the current device, whose stream the kernels are queued on")
    return device


def _refuse(name, t, dtype, shape, device):
    if not t.is_cuda:
        raise RuntimeError("blackriver_b200 operators run on CUDA tensors only (no CPU path)")
    if t.get_device() != device:
        raise RuntimeError(f"{name} must live on the current device, whose stream the kernels are queued on")
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    raise RuntimeError("tensors must be contiguous")


def _take(name, t, dtype, shape, device):
    """Address of a contiguous tensor of that type and shape on that device; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        _refuse(name, t, dtype, shape, device)
    return t.data_ptr()


_stream = torch._C._cuda_getCurrentRawStream


def _workspace(like, given, need, device):
    """(address, bytes, tensor) of the workspace given, or of a new one."""
    if given is None:
        given = torch.empty(max(need, 16), dtype=torch.uint8, device=like.device)
        return given.data_ptr(), max(need, 16), given
    return _take("workspace", given, given.dtype, given.shape, device), given.numel() * given.element_size(), given


def _result(name, t, like, device):
    """(tensor, address) of an output of the type and shape of `like`: the one given, or a new one."""
    if t is None:
        t = torch.empty_like(like)
        return t, t.data_ptr()
    return t, _take(name, t, like.dtype, like.shape, device)


def doc_plan(mask, prompt=None, ids=None):
    """Spans of packed documents: mask [batch, tokens] int32 numbers the documents (0 or less = padding), prompt marks
    the tokens of prompts.  Returns int32 spans [batch, tokens, 4] for doc_attn; with ids also the loss targets and their
    count: (spans, target, count)."""
    device = _device(mask)
    shape = mask.shape
    if len(shape) != 2:
        raise ValueError("mask must be [batch, tokens]")
    b, t = shape
    a_mask, a_prompt, a_ids = (_take(n, x, torch.int32, shape, device) for n, x in (("mask", mask), ("prompt", prompt), ("ids", ids)))
    spans = mask.new_empty((b, t, 4))
    if ids is None:
        brk.call("brk_doc_plan", a_mask, a_prompt, 0, b, t, spans.data_ptr(), 0, 0, _stream(device))
        return spans
    target = torch.empty_like(ids)
    count = ids.new_empty((1,))
    brk.call("brk_doc_plan", a_mask, a_prompt, a_ids, b, t, spans.data_ptr(), target.data_ptr(), count.data_ptr(), _stream(device))
    return spans, target, count


def _heads(name, t, b, n, h, d, device):
    """(address, row stride) of a [batch, tokens, heads, head_dim] fp16 tensor whose heads lie side by side in a token's row."""
    if t.get_device() != device:
        _refuse(name, t, t.dtype, t.shape, device)
    if t.dtype is not torch.float16:
        raise TypeError(f"unsupported dtype {t.dtype}")
    if t.shape != (b, n, h, d):
        raise ValueError(f"{name} must be [{b}, {n}, {h}, {d}], got {tuple(t.shape)}")
    s = t.stride()
    ld = s[1] if n > 1 else s[0] if b > 1 else h * d
    if b * n and ((d > 1 and s[3] != 1) or (h > 1 and s[2] != d) or (b > 1 and s[0] != n * ld)):
        raise ValueError(f"{name}: heads must lie side by side and tokens at one stride")
    return t.data_ptr(), ld


def _doc_args(q, k, v, spans, slopes):
    device = _device(q)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q, k and v must be [batch, tokens, heads, head_dim]")
    b, n, h, d = q.shape
    hk = k.shape[2]
    a_q, ld_q = _heads("q", q, b, n, h, d, device)
    a_k, ld_kv = _heads("k", k, b, n, hk, d, device)
    a_v, ld_v = _heads("v", v, b, n, hk, d, device)
    if ld_v != ld_kv:
        raise ValueError("k and v must have the same row stride")
    return device, b, n, h, hk, d, a_q, a_k, a_v, ld_q, ld_kv, _take("spans", spans, torch.int32, (b, n, 4), device), _take("slopes", slopes, torch.float32, (h,), device)


def doc_attn(q, k, v, spans, slopes=None, cap=0.0, out=None, lse=None):
    """Attention over packed documents: q [batch, tokens, heads, head_dim], k and v [batch, tokens, kv_heads, head_dim]
    fp16 (views of a fused projection are read in place), spans from doc_plan.  slopes [heads]: bias -slope * distance;
    cap: scores capped by cap * tanh(score / cap).  Returns (out, lse [batch, heads, tokens])."""
    device, b, n, h, hk, d, a_q, a_k, a_v, ld_q, ld_kv, a_spans, a_slopes = _doc_args(q, k, v, spans, slopes)
    if out is None:
        out = q.new_empty((b, n, h, d))
        a_out, ld_out = out.data_ptr(), h * d
    else:
        a_out, ld_out = _heads("out", out, b, n, h, d, device)
    if lse is None:
        lse = torch.empty(b, h, n, dtype=torch.float32, device=q.device)
        a_lse = lse.data_ptr()
    else:
        a_lse = _take("lse", lse, torch.float32, (b, h, n), device)
    brk.call("brk_doc_attn_fwd", a_q, a_k, a_v, ld_q, ld_kv, a_out, ld_out, a_lse, a_spans, a_slopes, cap, b, n, h, hk, d, _stream(device))
    return out, lse


def doc_attn_backward(d_out, q, k, v, out, lse, spans, slopes=None, cap=0.0, dq=None, dk=None, dv=None, workspace=None):
    """Gradients (dq, dk, dv) of doc_attn; without dq, dk and dv they are views of one fused [batch, tokens, heads + 2 kv_heads,
    head_dim] buffer, as the projection's backward wants them."""
    device, b, n, h, hk, d, a_q, a_k, a_v, ld_q, ld_kv, a_spans, a_slopes = _doc_args(q, k, v, spans, slopes)
    a_out, ld_out = _heads("out", out, b, n, h, d, device)
    a_do, ld_do = _heads("d_out", d_out, b, n, h, d, device)
    if ld_do != ld_out:
        raise ValueError("out and d_out must have the same row stride")
    a_lse = _take("lse", lse, torch.float32, (b, h, n), device)
    if dq is None and dk is None and dv is None:
        fused = q.new_empty((b, n, h + 2 * hk, d))
        dq, dk, dv = fused.split_with_sizes((h, hk, hk), 2)
        a_dq, ld_dq = fused.data_ptr(), (h + 2 * hk) * d
        a_dk, a_dv, ld_dkv = a_dq + 2 * h * d, a_dq + 2 * (h + hk) * d, ld_dq
    elif dq is None or dk is None or dv is None:
        raise ValueError("give all of dq, dk and dv, or none")
    else:
        a_dq, ld_dq = _heads("dq", dq, b, n, h, d, device)
        a_dk, ld_dkv = _heads("dk", dk, b, n, hk, d, device)
        a_dv, ld_dv = _heads("dv", dv, b, n, hk, d, device)
        if ld_dv != ld_dkv:
            raise ValueError("dk and dv must have the same row stride")
    a_ws, ws_bytes, workspace = _workspace(q, workspace, brk.lib().brk_doc_attn_bwd_workspace_bytes(b, n, h), device)
    brk.call("brk_doc_attn_bwd", a_q, a_k, a_v, ld_q, ld_kv, a_out, a_do, ld_out, a_lse, a_dq, ld_dq, a_dk, a_dv, ld_dkv, a_spans, a_slopes, cap, b, n, h, hk, d,
             a_ws, ws_bytes, _stream(device))
    return dq, dk, dv


# --- activations kept in 8 bits ---
ACT8_BLOCK = 128        # columns that share a scale


def _act8_like(t):
    """(device, rows, cols, address) of an activation tensor [..., cols]."""
    device = _device(t)
    shape = t.shape
    if not shape or shape[-1] == 0:
        raise ValueError("activations need at least one column")
    if not t.is_contiguous():
        raise RuntimeError("tensors must be contiguous")
    return device, t.numel() // shape[-1], shape[-1], t.data_ptr()


def _act8_new(t, rows, cols):
    q = torch.empty_like(t, dtype=torch.int8) if t.dim() == 2 else t.new_empty((rows, cols), dtype=torch.int8)
    return q, torch.empty(rows, -(-cols // ACT8_BLOCK), dtype=torch.float32, device=t.device)


def _act8_take(q, scale, rows, cols, device):
    return _take("q", q, torch.int8, (rows, cols), device), _take("scale", scale, torch.float32, (rows, -(-cols // ACT8_BLOCK)), device)


def act8_pack(x):
    """x [..., cols] -> (q int8 [rows, cols], scale fp32 [rows, ceil(cols / 128)])."""
    device, rows, cols, a_x = _act8_like(x)
    q, scale = _act8_new(x, rows, cols)
    brk.call("brk_act8_pack", a_x, q.data_ptr(), scale.data_ptr(), rows, cols, _dt(x), _stream(device))
    return q, scale


def act8_unpack(q, scale, dtype=torch.float16, out=None):
    """The kept values, [rows, cols] of `dtype` (or into out)."""
    device, rows, cols, _ = _act8_like(q)
    a_q, a_scale = _act8_take(q, scale, rows, cols, device)
    if out is None:
        out = torch.empty_like(q, dtype=dtype)
        a_out = out.data_ptr()
    else:
        a_out = _take("out", out, out.dtype, q.shape, device)
    brk.call("brk_act8_unpack", a_q, a_scale, a_out, rows, cols, _dt(out), _stream(device))
    return out


def gelu_act8(x, out=None):
    """gelu(x) and x kept in 8 bits: (y, q, scale)."""
    device, rows, cols, a_x = _act8_like(x)
    y, a_y = _result("out", out, x, device)
    q, scale = _act8_new(x, rows, cols)
    brk.call("brk_gelu_fwd_act8", a_x, a_y, q.data_ptr(), scale.data_ptr(), rows, cols, _dt(x), _stream(device))
    return y, q, scale


def gelu_backward_act8(dy, q, scale, out=None, recompute=False):
    """dy * gelu'(kept x); with recompute also gelu(kept x) again: dx, or (dx, y)."""
    device, rows, cols, a_dy = _act8_like(dy)
    a_q, a_scale = _act8_take(q, scale, rows, cols, device)
    dx, a_dx = _result("out", out, dy, device)
    y, a_y = _result("y", None, dy, device) if recompute else (None, 0)
    brk.call("brk_gelu_bwd_act8", a_dy, a_q, a_scale, a_dx, a_y, rows, cols, _dt(dy), _stream(device))
    return (dx, y) if recompute else dx


def layernorm_act8(x, gamma, beta, eps=1e-5, out=None):
    """LayerNorm that keeps the normalised rows in 8 bits: (y, q, scale, var)."""
    device, rows, cols, a_x = _act8_like(x)
    a_gamma, a_beta = _take("gamma", gamma, x.dtype, (cols,), device), _take("beta", beta, x.dtype, (cols,), device)
    y, a_y = _result("out", out, x, device)
    q, scale = _act8_new(x, rows, cols)
    var = torch.empty(rows, dtype=torch.float32, device=x.device)
    brk.call("brk_layernorm_fwd_act8", a_x, a_gamma, a_beta, a_y, q.data_ptr(), scale.data_ptr(), var.data_ptr(), rows, cols, eps, _dt(x), _stream(device))
    return y, q, scale, var


def layernorm_backward_act8(dy, gamma, var, q, scale, beta=None, residual=None, dgamma=None, dbeta=None, dx=None, accumulate=False, workspace=None):
    """LayerNorm backward from the kept rows: (dgamma, dbeta, dx), and with beta the forward's output again as a fourth."""
    device, rows, cols, a_dy = _act8_like(dy)
    if accumulate and (dgamma is None or dbeta is None):
        raise ValueError("accumulate needs dgamma and dbeta")
    dtype, vec = dy.dtype, (cols,)
    a_q, a_scale = _act8_take(q, scale, rows, cols, device)
    a_gamma, a_beta = _take("gamma", gamma, dtype, vec, device), _take("beta", beta, dtype, vec, device)
    a_var, a_residual = _take("var", var, torch.float32, (rows,), device), _take("residual", residual, dtype, dy.shape, device)
    dgamma, a_dgamma = _result("dgamma", dgamma, gamma, device)
    dbeta, a_dbeta = _result("dbeta", dbeta, gamma, device)
    dx, a_dx = _result("dx", dx, dy, device)
    y, a_y = _result("y", None, dy, device) if beta is not None else (None, 0)
    a_ws, ws_bytes, workspace = _workspace(dy, workspace, brk.lib().brk_layernorm_bwd_act8_workspace_bytes(rows, cols), device)
    brk.call("brk_layernorm_bwd_act8", a_dy, a_gamma, a_beta, a_var, a_q, a_scale, a_residual, a_dgamma, a_dbeta, a_dx, a_y, rows, cols, a_ws, ws_bytes,
             int(accumulate), _dt(dy), _stream(device))
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
