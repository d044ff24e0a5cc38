"""What the packed-document and 8-bit entry points refuse, without a GPU: nothing is launched, nothing is read."""
import pytest
import torch

from blackriver_b200 import brk, ops

A = 256            # a plausible aligned address; the checks come before any access


def test_plan():
    f = lambda *a: brk.raw("brk_doc_plan", *a, 0)  # noqa: E731
    assert f(0, 0, 0, 1, 4, A, 0, 0) == brk.INPUT_ERROR
    assert f(A, 0, 0, 1, 4, 0, 0, 0) == brk.OUTPUT_ERROR
    assert f(A, 0, 0, 1, 4, A, A, 0) == brk.INPUT_ERROR           # targets need ids
    assert f(A, 0, A, 1, 4, A, 0, A) == brk.OUTPUT_ERROR          # a count needs targets
    assert f(A, 0, 0, -1, 4, A, 0, 0) == brk.ATTR_ERROR
    assert f(A, 0, 0, 1 << 16, 1 << 15, A, 0, 0) == brk.ATTR_ERROR
    assert f(A, 0, 0, 1, 4, A + 4, 0, 0) == brk.ATTR_ERROR
    assert f(A, 0, 0, 0, 4, A, 0, 0) == brk.OK


def fwd(q=A, k=A, v=A, ld_q=128, ld_kv=128, out=A, ld_out=128, lse=0, spans=A, slopes=0, cap=0.0, batch=1, tokens=4, heads=2, kv=2, d=64):
    return brk.raw("brk_doc_attn_fwd", q, k, v, ld_q, ld_kv, out, ld_out, lse, spans, slopes, cap, batch, tokens, heads, kv, d, 0)


def bwd(q=A, out=A, d_out=A, lse=A, dq=A, ld_dq=128, dk=A, dv=A, ld_dkv=128, ws=A, ws_bytes=1 << 20, ld_out=128, batch=1, tokens=4, heads=2, kv=2, d=64, cap=0.0):
    return brk.raw("brk_doc_attn_bwd", q, A, A, 128, 128, out, d_out, ld_out, lse, dq, ld_dq, dk, dv, ld_dkv, A, 0, cap, batch, tokens, heads, kv, d, ws,
                   ws_bytes, 0)


def test_attention():
    for name in ("q", "k", "v", "spans"):
        assert fwd(**{name: 0}) == brk.INPUT_ERROR
        assert fwd(**{name: A + 8}) == brk.ATTR_ERROR
    assert fwd(out=0) == brk.OUTPUT_ERROR
    bad = [dict(d=96), dict(d=0), dict(heads=0), dict(kv=0), dict(heads=3), dict(batch=-1), dict(tokens=-1), dict(ld_q=120), dict(ld_q=129), dict(ld_kv=64),
           dict(ld_out=127), dict(out=A + 2), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(tokens=(1 << 22) + 1),
           dict(batch=1 << 15, tokens=1 << 16), dict(heads=8192, kv=8192, ld_q=1 << 20, ld_kv=1 << 20, ld_out=1 << 20)]
    for b in bad:
        assert fwd(**b) == brk.ATTR_ERROR, b
    assert fwd(batch=0) == brk.OK and fwd(tokens=0) == brk.OK


def test_attention_backward():
    for name in ("q", "out", "d_out", "lse"):
        assert bwd(**{name: 0}) == brk.INPUT_ERROR
    for name in ("dq", "dk", "dv"):
        assert bwd(**{name: 0}) == brk.OUTPUT_ERROR
        assert bwd(**{name: A + 8}) == brk.ATTR_ERROR
    for b in (dict(ld_dq=64), dict(ld_dkv=132), dict(ws=0), dict(ws_bytes=31), dict(d_out=A + 8), dict(ld_out=136 + 1), dict(d=32), dict(cap=-2.0)):
        assert bwd(**b) == brk.ATTR_ERROR, b
    assert bwd(tokens=0, ws=0) == brk.OK
    assert brk.lib().brk_doc_attn_bwd_workspace_bytes(1, 4, 2) == 32
    assert brk.lib().brk_doc_attn_bwd_workspace_bytes(0, 4, 2) == 0


@pytest.mark.parametrize("dtype", [2, -1, 7])
def test_act8_dtype(dtype):
    assert brk.raw("brk_act8_pack", A, A, A, 1, 8, dtype, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_act8_unpack", A, A, A, 1, 8, dtype, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_gelu_fwd_act8", A, A, A, A, 1, 8, dtype, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_gelu_bwd_act8", A, A, A, A, 0, 1, 8, dtype, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_layernorm_fwd_act8", A, A, A, A, A, A, A, 1, 8, 1e-5, dtype, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_layernorm_bwd_act8", A, A, A, A, A, A, 0, A, A, A, 0, 1, 8, A, 1 << 20, 0, dtype, 0) == brk.ATTR_ERROR


def test_act8():
    for rows, cols in ((-1, 8), (1, 0), (1, -8), (1 << 31, 8), (1, (1 << 24) + 1)):
        assert brk.raw("brk_act8_pack", A, A, A, rows, cols, brk.F16, 0) == brk.ATTR_ERROR
        assert brk.raw("brk_act8_unpack", A, A, A, rows, cols, brk.F16, 0) == brk.ATTR_ERROR
        assert brk.raw("brk_layernorm_fwd_act8", A, A, A, A, A, A, A, rows, cols, 1e-5, brk.F16, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_act8_pack", 0, A, A, 1, 8, brk.F16, 0) == brk.INPUT_ERROR
    assert brk.raw("brk_act8_pack", A, 0, A, 1, 8, brk.F16, 0) == brk.OUTPUT_ERROR
    assert brk.raw("brk_act8_pack", A, A, A, 0, 8, brk.F16, 0) == brk.OK
    assert brk.raw("brk_act8_unpack", A, 0, A, 1, 8, brk.F16, 0) == brk.INPUT_ERROR
    assert brk.raw("brk_gelu_fwd_act8", A, 0, A, A, 1, 8, brk.F32, 0) == brk.OUTPUT_ERROR
    assert brk.raw("brk_gelu_bwd_act8", 0, A, A, A, 0, 1, 8, brk.F32, 0) == brk.INPUT_ERROR
    assert brk.raw("brk_layernorm_fwd_act8", A, A, A, A, A, A, 0, 1, 8, 1e-5, brk.F32, 0) == brk.OUTPUT_ERROR
    assert brk.raw("brk_layernorm_fwd_act8", A, A, A, A, A, A, A, 1, 8, -1.0, brk.F32, 0) == brk.ATTR_ERROR
    need = brk.lib().brk_layernorm_bwd_act8_workspace_bytes(4, 8)
    assert need == 4 * 2 * 8 * 4
    assert brk.raw("brk_layernorm_bwd_act8", A, A, 0, A, A, A, 0, A, A, A, A, 4, 8, A, need, 0, brk.F32, 0) == brk.INPUT_ERROR      # y needs beta
    assert brk.raw("brk_layernorm_bwd_act8", A, A, 0, A, A, A, 0, A, A, A, 0, 4, 8, A, need - 1, 0, brk.F32, 0) == brk.ATTR_ERROR
    assert brk.raw("brk_layernorm_bwd_act8", A, A, 0, A, A, A, 0, A, A, A, 0, 4, 8, 0, need, 0, brk.F32, 0) == brk.ATTR_ERROR


def test_front_end_takes_cuda_tensors_only():
    x = torch.zeros(2, 128)
    for call in (lambda: ops.act8_pack(x), lambda: ops.gelu_act8(x), lambda: ops.layernorm_act8(x, x[0], x[0]),
                 lambda: ops.doc_plan(torch.zeros(1, 4, dtype=torch.int32)),
                 lambda: ops.doc_attn(*[torch.zeros(1, 4, 2, 64).half()] * 3, torch.zeros(1, 4, 4, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_caps_outside_the_range_and_too_many_tiles():
    for cap in (1e-7, 1e-30, 10001.0, -0.5, float("-inf")):
        assert fwd(cap=cap) == brk.ATTR_ERROR and bwd(cap=cap) == brk.ATTR_ERROR
    assert fwd(batch=1 << 21, tokens=256, heads=1024, kv=1024, ld_q=1 << 16, ld_kv=1 << 16, ld_out=1 << 16) == brk.ATTR_ERROR
