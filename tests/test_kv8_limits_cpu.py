"""Calls of the 8-bit paged cache and of filtered sampling that are refused before they reach a kernel."""
import pytest
import torch

from trl_b200.ops import functional as F


@pytest.mark.parametrize("change, message", [
    (dict(slots=torch.zeros(3, dtype=torch.int32), lens=torch.zeros(4, dtype=torch.int32)), "seq_lens"),
    (dict(slots=torch.zeros(3, dtype=torch.int32), delta=torch.zeros(4, dtype=torch.int32)), "pos_delta"),
    (dict(delta=torch.zeros(2, dtype=torch.int32)), "pos_delta"), (dict(delta=torch.zeros(5, dtype=torch.int64)), "pos_delta"),
    (dict(qkv=torch.zeros(3, 512), bias=torch.zeros(512)), "bias"), (dict(qkv=torch.zeros(3, 512), bias=torch.zeros(256, dtype=torch.bfloat16)), "bias"),
    (dict(q_norm=torch.ones(64)), "q_norm"), (dict(k_norm=torch.ones(32, dtype=torch.bfloat16)), "k_norm"),
    (dict(k_norm=torch.ones(128, dtype=torch.bfloat16)[::2]), "k_norm"), (dict(table=torch.zeros(2, 1, dtype=torch.int32)), "block table")])
def test_rope_append_refuses_what_it_would_read_wrongly(change, message):
    from trl_b200.ops import cuda as K

    a = dict(qkv=torch.zeros(3, 512, dtype=torch.bfloat16), bias=None, q_norm=None, k_norm=None, lens=torch.zeros(5, dtype=torch.int32),
             slots=None, table=torch.zeros(5, 1, dtype=torch.int32), delta=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        K.kv8_rope_append(a["qkv"], a["bias"], a["q_norm"], a["k_norm"], 1e-6, a["lens"], a["slots"], a["table"],
                          torch.zeros(3, 4, 64, dtype=torch.bfloat16), *F.kv8_alloc(4, 2, 16, 64), 4, 1e4, pos_delta=a["delta"])


def test_attention_refuses_more_steps_than_it_can_count():
    """4096 sequences with room for 8.4 million tokens each have 2^31 steps of 16."""
    from trl_b200.ops import cuda as K

    B = 4096
    table = torch.empty(B, 65536, dtype=torch.int32)
    with pytest.raises(ValueError, match="2\\^31 steps"):
        K.kv8_decode_attn(torch.zeros(B, 1, 64, dtype=torch.bfloat16), *F.kv8_alloc(2, 1, 128, 64), table,
                          torch.full((B,), -1, dtype=torch.int32), 1.0)


@pytest.mark.parametrize("kv8", [False, True])
def test_only_prompts_into_an_8_bit_cache_need_starts(kv8):
    from types import SimpleNamespace

    from trl_b200.rollout.engine import _PrefillKV

    hook = _PrefillKV(SimpleNamespace(kv8=kv8), None, None, torch.tensor([2, 0], dtype=torch.int32))
    assert (hook.starts.tolist() == [0, 0]) if kv8 else hook.starts is None
