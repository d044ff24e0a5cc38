"""Decoder layers on packed documents through the words machine: plan, LayerNorm, attention and GELU with 8-bit activations,
forward and backward, against the same layers in 64 bits.

Bounds are relative Frobenius norms, derived as follows.  Forward: a layer rounds to fp16 at most ten times between its input
and its output (LayerNorm, QKV, probabilities, attention, dense, LayerNorm, 4H, GELU, 4H->H and the sum), each by at most
2^-11 of what it rounds: 10 * 2^-11 = 4.9e-3 a layer.  Backward: a kept value is off by a uniform error of half a step, rms
top / 127 / sqrt(12); the largest of 128 normal values stays below 4.5 sigma, so 1.03e-2 of the row's sigma.  It enters a weight
gradient once through the operand that is rebuilt from it (1.03e-2), and once through gelu', whose slope is at most 0.8
where its rms is 0.58, at inputs of sigma 0.5 (0.71e-2); ten roundings to fp16 add 0.49e-2.  Together 2.2e-2 a layer."""
import numpy as np
import pytest
import torch

from doc_reference import plan, visible

pytestmark = pytest.mark.gpu
FORWARD, BACKWARD = 10 * 2.0 ** -11, 2.2e-2


@pytest.fixture(scope="module")
def host():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    from blackriver_b200 import host as _host
    try:
        _host.context_boot(0, None, 256 << 20)
        _host.collective_boot_local(0, 1)
        owned = True
    except _host.HostError:
        owned = False          # another test module of this process booted it already
    yield _host
    if owned:
        _host.context_shutdown()


def parameters(rng, hidden):
    r16 = lambda a: a.astype(np.float16).astype(np.float64)  # noqa: E731
    p = {}
    for name in ("input_layernorm", "post_attention_layernorm"):
        p[name + ".weight"] = r16(1 + 0.1 * rng.standard_normal(hidden))
        p[name + ".bias"] = r16(0.1 * rng.standard_normal(hidden))
    for name, o, i in (("query_key_value", 3, 1), ("dense", 1, 1), ("dense_h_to_4h", 4, 1), ("dense_4h_to_h", 1, 4)):
        p[name + ".weight"] = r16(0.5 / np.sqrt(i * hidden) * rng.standard_normal((o * hidden, i * hidden)))
        p[name + ".bias"] = r16(0.02 * rng.standard_normal(o * hidden))
    return {k: torch.tensor(v, requires_grad=True) for k, v in p.items()}


def layer(x, p, seen, slopes, heads, cap):
    B, T, H = x.shape
    norm = lambda v, name: torch.nn.functional.layer_norm(v, (H,), p[name + ".weight"], p[name + ".bias"], 1e-5)  # noqa: E731
    linear = lambda v, name: v @ p[name + ".weight"].T + p[name + ".bias"]  # noqa: E731
    q, k, v = (t.reshape(B, T, heads, -1).transpose(1, 2) for t in linear(norm(x, "input_layernorm"), "query_key_value").split(H, -1))
    s = q @ k.transpose(2, 3) / np.sqrt(H // heads)
    if cap:
        s = cap * torch.tanh(s / cap)
    at = torch.arange(T)
    s = s - slopes[:, None, None] * (at[:, None] - at[None]).abs()
    s = s.masked_fill(~seen[:, None], -1e30)
    a = (torch.softmax(s, -1) * seen[:, None]) @ v
    x = x + linear(a.transpose(1, 2).reshape(B, T, H), "dense")
    u = linear(norm(x, "post_attention_layernorm"), "dense_h_to_4h")
    return x + linear(0.5 * u * (1 + torch.tanh(0.79788456 * u * (1 + 0.044715 * u * u))), "dense_4h_to_h")


def off(got, want):
    want = np.asarray(want, np.float64)
    return float(np.linalg.norm(np.asarray(got, np.float64) - want) / np.linalg.norm(want))


@pytest.mark.parametrize("n_layers,batch,tokens,hidden,heads,cap,lengths", [
    (1, 2, 150, 256, 4, 0.0, [[60, -7, 83], [150]]),
    (2, 3, 77, 256, 2, 2.0, [[1, 76], [-77], [30, 2, 40]]),
])
def test_layers_forward_and_backward(host, n_layers, batch, tokens, hidden, heads, cap, lengths):
    from blackriver_b200 import words
    rng = np.random.default_rng(n_layers)
    mask, prompt = np.zeros((batch, tokens), np.int32), np.zeros((batch, tokens), np.int32)
    for b, row in enumerate(lengths):
        at = 0
        for number, n in enumerate(row):
            if n > 0:
                mask[b, at:at + n] = number + 1
                prompt[b, at:at + n // 3] = 1
            at += abs(n)
    ids = rng.integers(0, 999, (batch, tokens)).astype(np.int32)
    spans, target, _ = plan(mask.tolist(), prompt.tolist(), ids.tolist())
    params = [parameters(rng, hidden) for _ in range(n_layers)]
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float64)
    r16 = lambda a: a.astype(np.float16).astype(np.float64)  # noqa: E731
    x = torch.tensor(r16(rng.standard_normal((batch, tokens, hidden))), requires_grad=True)
    dy = r16(rng.standard_normal((batch, tokens, hidden)))
    seen = visible(torch.tensor(spans))
    y = x
    for p in params:
        y = layer(y, p, seen, slopes, heads, cap)
    y.backward(torch.tensor(dy))

    env = host.Env(n_layers + 1)
    try:
        env.execute(words.init_words(hidden=hidden, heads=heads, vocab=64, dtype="half", max_tokens=batch * tokens))
        env.execute(words.packed_words(n_layers, batch, tokens, hidden, heads, cap))
        env.execute("create_packed")
        for name, value in (("mask", mask), ("prompt", prompt), ("ids", ids), ("packed_in", x.detach().numpy())):
            env.write(name, value)
        for i, p in enumerate(params):
            env.execute(f"{i + 1} #")
            for name, value in p.items():
                env.write(name, value.detach().numpy())
        env.execute("0 # packed_plan packed_forward op.sync")
        assert np.array_equal(env.read("spans"), np.array(spans)) and np.array_equal(env.read("target"), np.array(target))
        assert off(env.read("packed_out"), y.detach()) <= FORWARD * n_layers
        env.write("packed_out_g", dy)
        env.execute("packed_backward op.sync")
        assert off(env.read("packed_in_g"), x.grad) <= BACKWARD * n_layers
        for i, p in enumerate(params):
            env.execute(f"{i + 1} #")
            for name, value in p.items():
                assert off(env.read(name + "_g"), value.grad) <= BACKWARD * n_layers, (i, name)
        # nothing is left of one run in the next (split products of the GEMMs may add up in another order: ten roundings again)
        first = {name: env.read(name + "_g") for name in params[-1]}
        env.execute("0 #")
        env.write("packed_in", x.detach().numpy())
        env.execute("packed_plan packed_forward op.sync")
        env.write("packed_out_g", dy)
        env.execute(f"packed_backward op.sync {n_layers} #")
        for name, value in first.items():
            assert off(env.read(name + "_g"), value) <= FORWARD * n_layers, name
        env.execute("op.kernel_status \"status\" !")
    finally:
        env.close()
    from blackriver_b200 import brk
    assert brk.lib().brk_doc_attn_status() == 0 and brk.lib().brk_flash_attn_status() == 0 and brk.lib().brk_gemm_f16_status() == 0


def test_words_keep_and_return_activations(host):
    rng = np.random.default_rng(5)
    for dtype, step in (("half", 2.0 ** -11), ("float", 2.0 ** -24)):
        x = rng.standard_normal((7, 200)).astype(np.float16 if dtype == "half" else np.float32)
        env = host.Env(1)
        try:
            for name, shape, kind in (("x", "7 200 2", dtype), ("y", "7 200 2", dtype), ("kept", "350 1", "int"), ("steps", "7 2 2", "float")):
                env.execute(f'{shape} "cuda" "{kind}" op.create "{name}" !')
            env.write("x", x)
            env.execute('"x" @ "kept" @ "steps" @ op.act8_pack "y" @ "kept" @ "steps" @ op.act8_unpack op.sync')
            steps = env.read("steps").astype(np.float64)
            q = env.read("kept").view(np.int8).reshape(7, 200).astype(np.float64)
            value = q * np.repeat(steps, 128, 1)[:, :200]
            assert np.all(np.abs(env.read("y") - value) <= np.abs(value) * (step + 2.0 ** -24))
            assert np.all(np.abs(value - x) <= np.repeat(steps, 128, 1)[:, :200] * (0.5 + 127 * 2.0 ** -22))
        finally:
            env.close()
