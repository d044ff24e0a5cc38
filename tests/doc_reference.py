"""Plain 64-bit forms of the packed-document operators, and how far fp16 tensor-core kernels may be from them."""
import math

import torch

HALF = 2.0 ** -11          # half a step of fp16, relative
TINY = 2.0 ** -25          # half a step of fp16 below its normal range


def plan(mask, prompt=None, ids=None):
    """Spans, targets and count by walking the tokens of each row (lists of ints)."""
    spans, targets, count = [], [], 0
    for b, row in enumerate(mask):
        row = [max(m, 0) for m in row]
        n, out, tg = len(row), [], []
        t = 0
        while t < n:
            e = t
            while e < n and row[e] == row[t]:
                e += 1
            pe = t
            if prompt is not None:
                while pe < e and prompt[b][pe]:
                    pe += 1
            for i in range(t, e):
                out.append((t, t, t, t) if row[t] == 0 else (t, max(i + 1, pe), t if i < pe else i, e))
                if ids is not None:
                    has = row[t] > 0 and i + 1 < e and not (prompt is not None and prompt[b][i + 1])
                    tg.append(ids[b][i + 1] if has else -100)
                    count += has
            t = e
        spans.append(out)
        targets.append(tg)
    return spans, targets, count


def visible(spans):
    """[batch, query, key] from spans [batch, tokens, 4]."""
    at = torch.arange(spans.shape[1])
    return (at >= spans[..., 0:1]) & (at < spans[..., 1:2])


def attention(q, k, v, spans, slopes=None, cap=0.0, d_out=None):
    """Values and elementwise error bounds, {name: (value, bound)}, of one call on CPU tensors [batch, tokens, heads, d].
    Bounds count the kernel's roundings: fp16 P and dS as operands (HALF each), results rounded to fp16 (HALF), delta from
    the rounded output, and 2^-14 relative for fp32 scores, exponentials and sums (score error below 2^-16 at these sizes)."""
    B, T, H, D = q.shape
    g = H // k.shape[2]
    f = lambda x: x.double().transpose(1, 2)  # noqa: E731
    q, k, v = f(q), f(k).repeat_interleave(g, 1), f(v).repeat_interleave(g, 1)
    vis = visible(spans)[:, None].expand(B, H, T, T)
    zero = lambda x: torch.where(vis, x, 0.0)  # noqa: E731
    x = q @ k.transpose(2, 3) / math.sqrt(D)
    dt = torch.ones_like(x)
    if cap:
        t = torch.tanh(x / cap)
        x, dt = cap * t, 1 - t * t
    if slopes is not None:
        at = torch.arange(T)
        x = x - slopes.double()[:, None, None] * (at[:, None] - at[None]).abs()
    x = torch.where(vis, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(x - top)
    l = p.sum(-1, keepdim=True)
    lse = torch.where(l > 0, top + torch.log(torch.where(l > 0, l, 1.0)), 0.0)[..., 0]
    p = p / torch.where(l > 0, l, 1.0)
    soft = 2.0 ** -14
    out = p @ v
    spread = p @ v.abs()
    e_out = HALF * 1.1 * (spread + out.abs()) + soft * spread + TINY * (1 + v.abs().amax())
    b = lambda y: y.transpose(1, 2)  # noqa: E731
    r = {"out": (b(out), b(e_out)), "lse": (lse, torch.full_like(lse, 1e-4))}
    if d_out is None:
        return r
    do = f(d_out)
    dp = do @ v.transpose(2, 3)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta) * dt
    e_p = p * (HALF * 1.1 + soft) + torch.where(vis, TINY, 0.0)
    e_delta = (do.abs() * e_out).sum(-1, keepdim=True) + 2.0 ** -20 * (do * out).abs().sum(-1, keepdim=True)
    e_ds = ds.abs() * (HALF * 1.1 + soft) + p * (e_delta + 2.0 ** -18 * (do.abs() @ v.abs().transpose(2, 3))) + p * soft * (dp.abs() + delta.abs()) + torch.where(vis, TINY, 0.0)
    s = 1 / math.sqrt(D)
    ds, e_p, e_ds = zero(ds), zero(e_p), zero(e_ds)
    group = lambda y: y.reshape(B, H // g, g, T, D).sum(2)  # noqa: E731
    dq, dk, dv = ds @ k * s, group(ds.transpose(2, 3) @ q) * s, group(p.transpose(2, 3) @ do)
    e_dq = e_ds @ k.abs() * s + HALF * 1.1 * dq.abs() + TINY
    e_dk = group(e_ds.transpose(2, 3) @ q.abs()) * s + HALF * 1.1 * dk.abs() + TINY
    e_dv = group(e_p.transpose(2, 3) @ do.abs()) + HALF * 1.1 * dv.abs() + TINY
    r |= {"dq": (b(dq), b(e_dq)), "dk": (b(dk), b(e_dk)), "dv": (b(dv), b(e_dv))}
    return r


def assert_close(got, value, bound, name):
    got = got.double().cpu()
    assert got.shape == value.shape, name
    off = (got - value).abs()
    worst = (off / bound).nan_to_num(nan=float("inf"), posinf=float("inf"))
    assert (off <= bound).all(), f"{name}: {worst.max():.3g} times the bound at {tuple(torch.nonzero(worst == worst.max())[0].tolist())}"
