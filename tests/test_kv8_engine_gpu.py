"""The rollout engine on an 8-bit cache, and with its filters and draw in one kernel (B200)."""
import math

import pytest
import torch

from kv8_util import attention64

pytestmark = pytest.mark.gpu


def _model(dim=128, heads=2, kv_heads=1, name="tiny-qwen2"):
    from trl_b200.testing import make_tiny_model

    return make_tiny_model(name, dtype=torch.bfloat16, device="cuda", hidden_size=256, num_attention_heads=heads,
                           num_key_value_heads=kv_heads, head_dim=dim, intermediate_size=512)


def _watch(monkeypatch):
    """Every call that the engine makes is held against its definition; returns the counts."""
    from trl_b200.ops import cuda as K
    from trl_b200.oracle import ops as R

    seen = {"append": 0, "step": 0, "attend": 0}
    append, step, attend = K.kv8_append, K.kv8_rope_append, K.kv8_decode_attn

    def cpu(xs):
        return [x.cpu().clone() for x in xs]

    def same(got, want):
        for a, b in zip(got, want):
            if a.dtype == torch.float8_e4m3fn:
                a, b = a.view(torch.uint8), b.view(torch.uint8)
            assert torch.equal(a.cpu(), b)

    def my_append(k, v, *cache, cu_seqlens, slots, max_new):
        cache, (table, starts) = cache[:4], cache[4:]
        want = cpu(cache)
        append(k, v, *cache, table, starts, cu_seqlens=cu_seqlens, slots=slots, max_new=max_new)
        R.kv8_append(k.cpu(), v.cpu(), *want, table.cpu(), starts.cpu(), cu_seqlens.cpu(), slots.cpu())
        same(cache, want)
        seen["append"] += 1

    def my_step(qkv, bias, q_norm, k_norm, eps, lens, slot_ids, table, q_out, *cache, pos_delta=None):
        (cache, (Hq, theta)) = cache[:4], cache[4:]
        want, rows = cpu(cache), qkv.clone()
        step(qkv, bias, q_norm, k_norm, eps, lens, slot_ids, table, q_out, *cache, Hq, theta, pos_delta=pos_delta)
        # the rows that it writes are those of the 16-bit cache's kernel, in the same place of pages of 16
        B, heads, page, dim = lens.numel(), cache[0].shape[1], cache[0].shape[2], cache[0].shape[3]
        k16, v16 = (torch.zeros(B, 16, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q16, own = torch.empty_like(q_out), torch.arange(B, dtype=torch.int32, device="cuda")[:, None].expand(B, table.shape[1] * page // 16).contiguous()
        if rows.dtype == torch.float32:
            K.rope_kv_write_f32(rows, bias, q_norm, k_norm, eps, lens, None, own, 16, q16, k16, v16, Hq, heads, dim, theta, pos_delta=pos_delta)
        else:
            K.rope_kv_write(rows, lens, None, own, 16, q16, k16, v16, Hq, heads, dim, theta, pos_delta=pos_delta)
        live = lens >= 0
        # a bf16 step: sine and cosine of the two differ by far less than half of one, which can still fall on its border
        if bool(live.any()):
            assert torch.allclose(q_out[live].float(), q16[live].float(), rtol=2.0**-7, atol=2.0**-7 * float(q16[live].abs().max()))
        at = lens.clamp(min=0).long()
        for i in live.nonzero().flatten().tolist():
            page_id, row = int(table[i, at[i] // page]), int(at[i]) % page
            for codes, scale, new in ((cache[0], cache[2], k16), (cache[1], cache[3], v16)):
                got = codes[page_id, :, row].float() * scale[page_id][:, None]
                x = new[i, int(at[i]) % 16].float()
                # half a step of e4m3, of its smallest numbers 2^-10 of the scale, and the bf16 step of above
                tol = (2.0**-4 + 2.0**-7) * x.abs() + 2.0**-10 * scale[page_id][:, None] + 2.0**-7 * x.abs().amax()
                assert bool(((got - x).abs() <= tol).all())
        # and what is not the new row's page stays
        mine = {int(table[i, at[i] // page]) for i in live.nonzero().flatten().tolist()}
        rest = [p for p in range(cache[0].shape[0]) if p not in mine]
        for a, b in zip(cache, want):
            a, b = (x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x for x in (a.cpu(), b))
            assert torch.equal(a[rest], b[rest])
        seen["step"] += 1

    def my_attend(q, *cache, out):
        cache, (table, lens, scale) = cache[:4], cache[4:]
        attend(q, *cache, table, lens, scale, out=out)
        want, tol = attention64(q.cpu(), cpu(cache), table.cpu(), (lens + 1).tolist(), scale)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
        seen["attend"] += 1

    monkeypatch.setattr(K, "kv8_append", my_append)
    monkeypatch.setattr(K, "kv8_rope_append", my_step)
    monkeypatch.setattr(K, "kv8_decode_attn", my_attend)
    return seen


@pytest.mark.parametrize("gemm", ["own", "cublas"])
@pytest.mark.parametrize("dim, heads, kv_heads, name, page", [(128, 2, 1, "tiny-qwen2", None), (64, 4, 2, "tiny-qwen3", 16)])
def test_every_call_of_an_engine_is_right(monkeypatch, gemm, dim, heads, kv_heads, name, page):
    from trl_b200.rollout.engine import RolloutEngine
    from trl_b200.rollout.sampling import SamplingParams

    monkeypatch.setenv("TRL_B200_DECODE_GEMM", gemm)
    model = _model(dim, heads, kv_heads, name)
    eng = RolloutEngine(model, max_num_seqs=3, max_model_len=192, block_size=page, poll_every=4, use_cuda_graph=False, kv_cache_dtype="fp8")
    assert eng.k_cache[0].dtype == torch.float8_e4m3fn
    seen = _watch(monkeypatch)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(5, 1000, (n,), generator=g).tolist() for n in (1, 70, 63)]
    outs = eng.generate(prompts, SamplingParams(n=2, max_tokens=6, temperature=0.9, top_p=0.9, top_k=40, seed=3))
    assert len(outs) == 6 and all(len(o.token_ids) == 6 and len(o.logprobs) == 6 for o in outs)
    assert all(math.isfinite(x) and x <= 1e-5 for o in outs for x in o.logprobs)
    layers = eng.cfg.num_hidden_layers
    assert seen["append"] >= layers and seen["step"] == seen["attend"] >= 5 * layers
    assert eng.sched.num_free_blocks == eng.num_blocks


def test_a_captured_step_gives_the_tokens_of_the_launched_one():
    from trl_b200.rollout.engine import RolloutEngine
    from trl_b200.rollout.sampling import SamplingParams

    model = _model()
    prompts = [list(range(10, 10 + n)) for n in (7, 64, 90)]
    sp = SamplingParams(n=4, max_tokens=20, temperature=1.0, top_p=0.95, eos_token_id=2, seed=5)

    def run(graph):
        eng = RolloutEngine(model, max_num_seqs=5, max_model_len=128, poll_every=4, use_cuda_graph=graph, kv_cache_dtype="fp8")
        first = [(o.token_ids, o.logprobs) for o in eng.generate(prompts, sp)]
        again = [(o.token_ids, o.logprobs) for o in eng.generate(prompts, sp)]  # on pages that held other sequences
        assert first == again
        return first
    assert run(True) == run(False)


def test_greedy_tokens_are_mostly_those_of_a_16_bit_cache():
    """Not a bound on errors, which the calls' own tests give: that pages, slots and scales belong together."""
    from trl_b200.rollout.engine import RolloutEngine
    from trl_b200.rollout.sampling import SamplingParams

    model = _model()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(5, 1000, (n,), generator=g).tolist() for n in (5, 70, 16, 130)]
    sp = SamplingParams(n=2, max_tokens=12, greedy=True)
    outs = [RolloutEngine(model, max_num_seqs=4, max_model_len=192, poll_every=4, kv_cache_dtype=t).generate(prompts, sp) for t in ("fp8", "auto")]
    assert sum(a.token_ids[:3] == b.token_ids[:3] for a, b in zip(*outs)) >= 6


def _old_path(z, sp, seed, step):
    from trl_b200.ops import cuda as K
    from trl_b200.rollout.sampling import filter_top_k_top_p

    tok, logp = torch.empty(z.shape[0], dtype=torch.int32, device="cuda"), torch.empty(z.shape[0], device="cuda")
    y = filter_top_k_top_p(z.float() / max(sp.temperature, 1e-6), sp.top_k, sp.top_p).contiguous()
    K.sample_tokens(y, 1.0, sp.min_p, None, None, seed, step, False, tok, logp)
    return y, tok, logp


@pytest.mark.parametrize("vocab, dtype", [(997, torch.float32), (50257, torch.bfloat16), (151936, torch.bfloat16), (300001, torch.bfloat16)])
@pytest.mark.parametrize("kw", [dict(top_k=50), dict(top_p=0.9), dict(top_p=0.999, temperature=1.7), dict(top_k=1000, top_p=0.8, min_p=0.01, temperature=0.7)])
def test_a_seed_draws_what_filter_and_sampler_draw(vocab, dtype, kw):
    """Without random words a row's draw is that of the sampler for unfiltered rows behind the filters in plain operations.

    -log(u) by the fast logarithm is off by up to 2^-21.4 where u is near 1, and each of the two programs may round z - log(e)
    once more: a token with e = -log(u) may win if its key, off by (2^-21 + 2^-22 e) / e + 2^-21 (|z| + 32), reaches the largest."""
    from trl_b200.ops import cuda as K
    from trl_b200.oracle.ops import _hash_u32
    from trl_b200.rollout.sampling import SamplingParams

    sp = SamplingParams(**kw)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    z = (torch.randn(24, vocab, generator=g, device="cuda") * 2).to(dtype)
    step, seed = torch.tensor([11], dtype=torch.int32, device="cuda"), 0x1234567
    tok, logp = torch.empty(24, dtype=torch.int32, device="cuda"), torch.empty(24, device="cuda")
    K.sample_filtered(z, temperature=sp.temperature, top_k=sp.top_k or 0, top_p=sp.top_p, min_p=sp.min_p or 0.0, seed=seed,
                      step_ptr=step, out_tok=tok, out_logp=logp)
    y, want, want_logp = _old_path(z, sp, seed, step)
    y = y.cpu().double()
    if sp.min_p:
        y = torch.where(y >= y.amax(-1, keepdim=True) + math.log(sp.min_p), y, -math.inf)
    row = torch.arange(24)
    word = seed ^ _hash_u32((11 * 0x9E3779B9 + row) & 0xFFFFFFFF)
    col = torch.arange(vocab)
    h = _hash_u32((_hash_u32(word[:, None] ^ _hash_u32((col * 0x85EBCA6B + 0x165667B1) & 0xFFFFFFFF)) + col) & 0xFFFFFFFF)
    u = (((h >> 8).double() + 0.5) / 2**24).clamp(max=1 - 2.0**-25)
    e = -torch.log(u)
    key = y - torch.log(e)
    slack = (2.0**-21 + 2.0**-22 * e) / e + 2.0**-21 * (y.abs().clamp(max=1e4) + 32)
    for i in range(24):
        t = int(tok[i])
        assert y[i, t] > -math.inf, i
        best = int((key[i] - slack[i]).argmax())
        assert float(key[i, t] + slack[i, t]) >= float(key[i, best] - slack[i, best]), i
        if int((key[i] + slack[i] >= (key[i] - slack[i]).max()).sum()) == 1:
            assert t == int(want[i]), i
        if t == int(want[i]):
            # both sum exponentials in 32 bits, one of them by the fast exponential and in any order
            assert abs(float(logp[i] - want_logp[i])) <= 2.0**-16 + 2.0**-22 * abs(float(want_logp[i])), i
