"""What takes an 8-bit cache by an option: trainers, the server's engine and the generation front end (B200)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = dict(hidden_size=256, num_attention_heads=2, num_key_value_heads=1, head_dim=128, intermediate_size=512, num_hidden_layers=2)


def _model():
    from trl_b200.testing import make_tiny_model

    return make_tiny_model("tiny-qwen2", dtype=torch.bfloat16, device="cuda", seed=0, **SHAPE)


def _holds_8_bits(engine):
    return engine.kv8 and all(t.dtype == torch.float8_e4m3fn for t in (*engine.k_cache, *engine.v_cache))


def test_a_policy_trains_on_rollouts_from_an_8_bit_cache(tmp_path, tiny_tokenizer):
    """It runs, with finite losses and gradients.  (Top-k keeps 5 % of this model's mass, so the importance weights of 8 tokens are
    about 0.05^8: that every weight moves by a bf16 step is not to be expected.)"""
    from trl_b200 import GRPOConfig, GRPOTrainer
    from trl_b200.ops import cuda as K
    from trl_b200.testing import make_dataset

    model = _model()
    args = GRPOConfig(output_dir=str(tmp_path), per_device_train_batch_size=4, max_steps=2, logging_steps=1, learning_rate=5e-3,
                      save_strategy="no", report_to="none", bf16=True, num_generations=4, max_completion_length=8, use_vllm=True,
                      vllm_mode="colocate", top_p=0.95, top_k=50, rollout_kv_cache_dtype="fp8")
    tr = GRPOTrainer(model, lambda completions, **kw: [0.1 * len(c) + 0.01 * (hash(c) % 7) for c in completions], args,
                     train_dataset=make_dataset("standard_prompt_only", 16), processing_class=tiny_tokenizer)
    tr.train()
    assert _holds_8_bits(tr._rollout)
    steps = [h for h in tr.state.log_history if "loss" in h]
    assert len(steps) == 2 and all(math.isfinite(h["loss"]) and math.isfinite(h["grad_norm"]) and h["grad_norm"] > 0 for h in steps)
    K.check_status()


def test_server_and_generation_serve_from_an_8_bit_cache(tmp_path):
    from trl_b200.generation.generation import RolloutGeneration
    from trl_b200.rollout.sampling import SamplingParams
    from trl_b200.scripts.rollout_serve import EngineHolder, ServeArguments

    model = _model()
    model.save_pretrained(str(tmp_path))
    holder = EngineHolder(ServeArguments(model=str(tmp_path), max_num_seqs=4, max_model_len=128, kv_cache_dtype="fp8"))
    front = RolloutGeneration(model, max_num_seqs=4, max_model_len=128, kv_cache_dtype="fp8")
    assert _holds_8_bits(holder.engine) and _holds_8_bits(front.engine)
    prompts = [list(range(5, 5 + n)) for n in (3, 40, 64, 65, 17)]  # more requests than slots
    sp = SamplingParams(n=2, max_tokens=9, temperature=0.8, top_p=0.9, seed=4)
    outs = holder.generate(prompts, sp)
    _, ids, logps, _ = front.generate(prompts, sp)
    assert len(outs) == 10 and all(len(o.token_ids) == 9 for o in outs)
    assert ids == [o.token_ids for o in outs]  # the same weights, the same seed
    assert all(math.isfinite(x) and x <= 1e-5 for o in outs for x in o.logprobs)
