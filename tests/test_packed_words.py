"""The packed-document script on a machine without a GPU: it parses, and tensors on the host are refused, not misread."""

import pytest

from blackriver_b200 import host, words


def test_script_parses_and_names_every_word():
    env = host.Env(3)
    try:
        env.execute(words.init_words(hidden=128, heads=2, vocab=64, dtype="half"))
        env.execute(words.packed_words(2, 2, 16, 128, 2))
    finally:
        env.close()
    text = words.packed_words(2, 2, 16, 128, 2, cap=30.0)
    for word in ("op.doc_plan", "op.doc_attn", "op.doc_attn_backward", "op.layernorm_act8", "op.layernorm_act8_backward_residual", "op.gelu_act8",
                 "op.gelu_act8_backward"):
        assert f"{word}\n" in text
    assert " 2 2 1 30.0 op.doc_attn\n" in text


@pytest.mark.parametrize("script", [
    '"i" @ "i" @ "i" @ "s" @ "i" @ op.doc_plan', '"x" @ "s" @ "x" @ "f" @ 2 2 1 0 op.doc_attn',
    '"x" @ "x" @ "x" @ "f" @ "s" @ "x" @ 2 2 1 0 op.doc_attn_backward', '"x" @ "i" @ "f" @ op.act8_pack', '"x" @ "i" @ "f" @ op.act8_unpack',
    '"x" @ "x" @ "i" @ "f" @ op.gelu_act8', '"x" @ "i" @ "f" @ "x" @ "x" @ op.gelu_act8_backward',
    '"x" @ "f" @ "x" @ "x" @ "x" @ "i" @ "f" @ 0.00001 op.layernorm_act8',
    '"x" @ "x" @ "x" @ "f" @ "i" @ "f" @ "x" @ "x" @ "x" @ "x" @ op.layernorm_act8_backward',
    '"x" @ "x" @ "x" @ "f" @ "i" @ "f" @ "x" @ "x" @ "x" @ "x" @ "x" @ op.layernorm_act8_backward_residual',
])
def test_tensors_on_the_host_are_refused(script):
    env = host.Env(1)
    try:
        for name, shape, kind in (("x", "2 4 256 3", "half"), ("f", "64 1", "float"), ("i", "2 4 2", "int"), ("s", "2 4 4 3", "int")):
            env.execute(f'{shape} "cpu" "{kind}" op.create "{name}" !')
        with pytest.raises(host.HostError, match="returned -1"):
            env.execute(script)
    finally:
        env.close()
