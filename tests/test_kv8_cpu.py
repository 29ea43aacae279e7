"""8-bit paged cache and filtered sampling on the CPU: definitions, and calls that are refused."""
import math

import pytest
import torch

from kv8_util import attention64, check_sample, filled_cache, table_of
from trl_b200.ops import functional as F


def test_scale_is_the_smallest_power_of_two():
    from trl_b200.oracle.ops import kv8_scale

    a = torch.tensor([0.0, 448.0, 448.0001, 447.9, 1.75, 1.7500001, 3.5, 2.0**-126, 3.3e38, 1e-40])
    e = torch.log2(kv8_scale(a)).int().tolist()
    assert e == [-100, 0, 1, 0, -8, -7, -7, -100, 120, -100]


def test_append_in_one_piece_and_token_by_token_stand_for_near_values():
    """Every entry is within e4m3's half step (2^-4 of the value, 2^-10 of a scale below the normal numbers), twice where a
    page's scale grew behind it."""
    g = torch.Generator().manual_seed(0)
    heads, page, dim, n = 2, 16, 64, 53
    k, v = (torch.randn(n, heads, dim, generator=g) * torch.linspace(0.1, 9, n)[:, None, None] for _ in range(2))
    table = table_of(1, 4, 9, g, "cpu")
    for pieces in ([n], [1] * n, [5, 11, 1, 30, 6]):
        cache = F.kv8_alloc(9, heads, page, dim)
        at = 0
        for m in pieces:
            F.kv8_append(k[at:at + m], v[at:at + m], *cache, table, torch.tensor([at], dtype=torch.int32),
                         cu_seqlens=torch.tensor([0, m], dtype=torch.int32))
            at += m
        for x, codes, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
            blocks = table[0].long()
            held = (codes[blocks].float() * scale[blocks][:, :, None, None]).transpose(0, 1).reshape(heads, -1, dim)[:, :n]
            top = scale[blocks].repeat_interleave(page, 0).t()[:, :n, None]
            want = x.transpose(0, 1)
            rounds = 1 if len(pieces) == 1 else 4  # a page's scale can grow a few times, each time rounding small values again
            assert ((held - want).abs() <= 2.0**-4 * want.abs() + rounds * 2.0**-10 * top).all()


def test_append_keeps_what_it_does_not_own():
    g = torch.Generator().manual_seed(1)
    cache, table = filled_cache([40, 40], 2, 16, 64, "cpu")
    was = [t.clone() for t in cache]
    k = torch.randn(3, 2, 64, generator=g)
    F.kv8_append(k, k, *cache, table, torch.tensor([-1, 18], dtype=torch.int32), cu_seqlens=torch.tensor([0, 0, 3], dtype=torch.int32))
    page = int(table[1, 1])
    for a, b in zip(cache, was):
        same = (a.float() == b.float()).flatten(1).all(1)
        assert same[torch.arange(len(same)) != page].all() and (a.dim() == 2 or not same[page])
    assert (cache[0][page, :, 5:].float() == was[0][page, :, 5:].float()).all()  # rows behind the last token
    assert (cache[2][page] >= was[2][page]).all()  # a page keeps its larger scale


def test_infinities_and_nan_are_held_as_nan():
    cache = F.kv8_alloc(1, 1, 16, 64)
    k = torch.ones(1, 1, 64)
    k[0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    F.kv8_append(k, k, *cache, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    held = cache[0][0, 0, 0].float() * cache[2]
    assert held[0, :3].isnan().all() and (held[0, 3:] == 1).all()


@pytest.mark.parametrize("window", [None, 7])
def test_attention_matches_its_definition(window):
    lens = [1, 16, 17, 0, 45]
    cache, table = filled_cache(lens, 2, 16, 64, "cpu")
    q = torch.randn(5, 6, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    out = F.kv8_decode_attn(q, *cache, table, torch.tensor([n - 1 for n in lens], dtype=torch.int32), 0.125, window=window)
    want, tol = attention64(q, cache, table, lens, 0.125, window)
    assert ((out.double() - want).abs() <= tol).all()
    assert (out[3] == 0).all()


def test_sampling_filters():
    """Probabilities 0.4, 0.3, 0.2, 0.1: the filters keep what they should, draws have the right frequencies."""
    p = torch.tensor([0.1, 0.4, 0.2, 0.3])
    logits = p.log()[None].repeat(4000, 1)
    rng = torch.randint(-2**31, 2**31 - 1, (4000,), generator=torch.Generator().manual_seed(0)).to(torch.int32)
    for kw, kept in (({"top_k": 2}, [1, 3]), ({"top_p": 0.69}, [1, 3]), ({"top_p": 0.71}, [1, 2, 3]), ({"min_p": 0.49}, [1, 2, 3]),
                     ({"top_k": 3, "top_p": 0.7}, [1, 3]), ({}, [0, 1, 2, 3]), ({"top_p": 0.0}, [1]), ({"temperature": 0.0}, [1])):
        tok, logp = F.sample_filtered(logits, rng, **kw)
        want = p[kept] / p[kept].sum() if kw != {"temperature": 0.0} else torch.ones(1)
        freq = torch.bincount(tok.long(), minlength=4).float() / 4000
        # five standard deviations of a share of 4000 draws
        assert ((freq[kept] - want).abs() <= 5 * (want * (1 - want) / 4000).sqrt() + 1e-9).all() and freq[kept].sum() == 1, kw
        if kw != {"temperature": 0.0}:
            assert torch.allclose(logp, want.log()[torch.tensor([kept.index(int(t)) for t in tok])], atol=1e-5)
            check_sample(logits[:50], rng[:50], tok[:50], logp[:50], **kw)


def test_sampling_ties_and_rows_without_tokens():
    inf = math.inf
    logits = torch.tensor([[1.0, 2, 2, 0], [-inf, -inf, -inf, -inf], [math.nan, 1, -inf, math.nan], [0, inf, 3, 0]])
    rng = torch.arange(4, dtype=torch.int32)
    tok, logp = F.sample_filtered(logits, rng, temperature=0.0)
    assert tok.tolist() == [1, 0, 1, 1]
    assert logp[1] == -inf and abs(float(logp[0]) + math.log(2)) < 1e-6 and logp[2] == 0 and logp[3] == 0
    tok, _ = F.sample_filtered(logits, rng, top_p=0.01)
    assert tok.tolist() == [1, 0, 1, 1]


def _cuda_args():
    cache = F.kv8_alloc(4, 2, 16, 64)
    return dict(k=torch.zeros(3, 2, 64), q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), cache=list(cache),
                table=torch.zeros(3, 1, dtype=torch.int32), lens=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("change, message", [
    (dict(k=torch.zeros(3, 2, 32)), "has to be"), (dict(k=torch.zeros(3, 2, 64, dtype=torch.int32)), "bf16, fp16 or fp32"),
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "int32"), (dict(lens=torch.zeros(2, dtype=torch.int32)), "one new token"),
    (dict(table=torch.zeros(2, 1, dtype=torch.int32)), "block table"), (dict(table=torch.zeros(3, dtype=torch.int32)), "rows, blocks"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "cu_seqlens"), (dict(slots=torch.zeros(2, dtype=torch.int32)), "slots"),
    (dict(max_new=0), "max_new")])
def test_append_refuses(change, message):
    from trl_b200.ops import cuda as K

    a = {**_cuda_args(), **change}
    with pytest.raises(ValueError, match=message):
        K.kv8_append(a["k"], a["k"], *a["cache"], a["table"], a["lens"], cu_seqlens=a.get("cu_seqlens"), slots=a.get("slots"),
                     max_new=a.get("max_new"))


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), "multiple of 2 heads"), (dict(q=torch.zeros(3, 4, 64)), "bf16 or fp16"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "q has to be"), (dict(lens=torch.zeros(2, dtype=torch.int32)), "lengths"),
    (dict(window=0), "window"), (dict(out=torch.zeros(3, 4, 64)), "out has to be"),
    (dict(slots=torch.zeros(2, dtype=torch.int32)), "slots"), (dict(q=torch.zeros(4097, 4, 64, dtype=torch.bfloat16)), "4096")])
def test_attention_refuses(change, message):
    from trl_b200.ops import cuda as K

    a = {**_cuda_args(), **change}
    with pytest.raises(ValueError, match=message):
        K.kv8_decode_attn(a["q"], *a["cache"], a["table"], a["lens"], 1.0, slots=a.get("slots"), window=a.get("window"), out=a.get("out"))


@pytest.mark.parametrize("which, value", [
    (0, torch.zeros(4, 2, 16, 64)), (0, torch.zeros(4, 2, 24, 64).to(torch.float8_e4m3fn)), (2, torch.ones(4, 3)),
    (3, torch.ones(4, 2, dtype=torch.float64)), (1, torch.zeros(4, 16, 2, 64).to(torch.float8_e4m3fn).transpose(1, 2))])
def test_caches_that_are_refused(which, value):
    from trl_b200.ops import cuda as K

    a = _cuda_args()
    a["cache"][which] = value
    with pytest.raises(ValueError):
        K.kv8_append(a["k"], a["k"], *a["cache"], a["table"], a["lens"])


def test_alloc_refuses():
    for page, dim in ((24, 64), (8, 64), (16, 80)):
        with pytest.raises(ValueError):
            F.kv8_alloc(4, 2, page, dim)


@pytest.mark.parametrize("kw, message", [
    (dict(logits=torch.zeros(3, dtype=torch.float32)), "vocabulary"), (dict(logits=torch.zeros(3, 5, dtype=torch.float64)), "bf16, fp16 or fp32"),
    (dict(rng=torch.zeros(2, dtype=torch.int32)), "rng"), (dict(rng=torch.zeros(3)), "rng"), (dict(top_p=torch.ones(2)), "top_p"),
    (dict(out_tok=torch.zeros(3, dtype=torch.int64)), "out_tok"), (dict(step_ptr=torch.zeros(1, dtype=torch.int64)), "step_ptr"), (dict(logits=torch.zeros(3, 0)), "vocabulary")])
def test_sampling_refuses(kw, message):
    from trl_b200.ops import cuda as K

    a = {"logits": torch.zeros(3, 5), "rng": torch.zeros(3, dtype=torch.int32), **kw}
    with pytest.raises(ValueError, match=message):
        K.sample_filtered(a.pop("logits"), a.pop("rng"), **a)


def test_an_engine_refuses_what_the_8_bit_cache_does_not_cover():
    from trl_b200.generation.generation import RolloutGeneration
    from trl_b200.rollout.engine import RolloutEngine
    from trl_b200.rollout.layered_engine import LayeredRolloutEngine
    from trl_b200.testing import make_tiny_model

    model = make_tiny_model("tiny-qwen2", head_dim=64)
    with pytest.raises(ValueError, match="kv_cache_dtype='int4'"):
        RolloutEngine(model, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="needs a GPU"):
        RolloutGeneration(model, kv_cache_dtype="fp8")
    eng = RolloutEngine.__new__(RolloutEngine)
    eng.model, eng.cfg, eng.tp, eng.kv8 = model, model.config, 1, True
    assert eng._check_model(128, None) == 64 and eng._check_model(128, 16) == 16 and not eng.attn_tc
    with pytest.raises(ValueError, match="16, 32, 64 or 128"):
        eng._check_model(128, 48)
    eng.tp = 2
    with pytest.raises(NotImplementedError, match="tensor parallel"):
        eng._check_model(128, None)
    eng = LayeredRolloutEngine.__new__(LayeredRolloutEngine)
    eng.model, eng.cfg, eng.tp, eng.kv8 = model, model.config, 1, True
    with pytest.raises(NotImplementedError, match="8-bit cache"):
        eng._check_model(128, None)


def test_a_trainer_on_the_cpu_refuses_an_8_bit_cache(tmp_path):
    from types import SimpleNamespace

    from trl_b200.trainer.grpo_config import GRPOConfig
    from trl_b200.trainer.online_base import OnlineTrainer

    args = GRPOConfig(output_dir=str(tmp_path), rollout_kv_cache_dtype="fp8", use_cpu=True)
    with pytest.raises(ValueError, match="rollout_kv_cache_dtype needs a GPU"):
        OnlineTrainer._get_rollout(SimpleNamespace(args=args, model=None, _rollout=None))


@pytest.mark.parametrize("change, message", [
    (dict(qkv=torch.zeros(3, 8 * 64 + 1, dtype=torch.bfloat16)), "dense rows"), (dict(bias=torch.zeros(512, dtype=torch.bfloat16)), "bias"),
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "seq_lens"), (dict(lens=torch.zeros(2, dtype=torch.int32)), "3 rows"),
    (dict(q_out=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), "q_out"), (dict(slots=torch.zeros(2, dtype=torch.int32)), "slots")])
def test_rope_append_refuses(change, message):
    from trl_b200.ops import cuda as K

    a = {**_cuda_args(), "qkv": torch.zeros(3, 8 * 64, dtype=torch.bfloat16), "q_out": torch.zeros(3, 4, 64, dtype=torch.bfloat16), **change}
    with pytest.raises(ValueError, match=message):
        K.kv8_rope_append(a["qkv"], a.get("bias"), None, None, 1e-6, a["lens"], a.get("slots"), a["table"], a["q_out"], *a["cache"], 4, 1e4)
