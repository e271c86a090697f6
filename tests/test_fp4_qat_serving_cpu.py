"""A policy trained with ``fp4_qat`` and its rollout engine with ``fp4_weights``: the same products, projection by projection."""
import pytest
import torch

from gcore_b200.models.config import ModelConfig
from gcore_b200.trainer.grpo_trainer import GrpoTrainer
from test_grpo_cpu import make_cfg, reward_has_small_token

PROMPTS = [[5, 6, 7, 8, 9], [10, 11, 12], [13, 14, 15, 16], [20, 21]]


def trainer(dtype="float32", acts="bf16", qat=True, **policy):
    cfg = make_cfg()
    cfg.policy.fp4_qat = qat
    for k, v in policy.items():
        setattr(cfg.policy, k, v)
    ie = cfg.sampler.infer_engine_configs[0]
    ie.fp4_weights, ie.fp4_activations = True, acts
    mcfg = ModelConfig(arch="qwen2", num_layers=2, hidden_size=256, num_attention_heads=4, num_kv_heads=2, ffn_hidden_size=352,
                       vocab_size=512, dtype=dtype)
    torch.manual_seed(0)
    return GrpoTrainer(cfg, model_cfg=mcfg, reward_fn=reward_has_small_token).setup()


def gaps(tr):
    """Largest difference of a projection's output between the engine and the trainer, over its largest value."""
    worst = 0.0
    for layer, lw in zip(tr.policy.model.decoder.layers, tr.engine.w.layers):
        for mod, name in ((layer.self_attention.linear_qkv, "qkv_w"), (layer.self_attention.linear_proj, "o_w"),
                          (layer.mlp.linear_fc1, "fc1_w"), (layer.mlp.linear_fc2, "fc2_w")):
            x = torch.randn(7, mod.in_local, generator=torch.Generator().manual_seed(3)).to(mod.weight)
            with torch.no_grad():
                want, got = mod(x), tr.engine._lin(x, lw, name, mod.bias)
            assert (mod.precision == "fp4_qat") == (name in lw.fp4)
            worst = max(worst, float((got.double() - want.double()).abs().max() / want.double().abs().max()))
    return worst


@pytest.mark.parametrize("dtype,tol", [("float32", 2 ** -18), ("bfloat16", 2 ** -6)])
@pytest.mark.parametrize("share", [True, False])
def test_the_engine_serves_the_products_that_the_policy_trains(dtype, tol, share):
    """Both are products of the same two matrices: in 32 bits the straight-through weight, w + (q - w), is off by 2^-23 and the sums
    of 352 products are the same; in bf16 either side is rounded once, 2^-8, and the largest value is at most twice a value's."""
    tr = trainer(dtype, share_rollout_weights=share)
    assert set(tr.engine.w.layers[0].fp4) == {"qkv_w", "o_w", "fc1_w"}   # 352 columns are not whole blocks of 128
    assert gaps(tr) < tol
    before = tr.engine.w.layers[0].fp4["fc1_w"].codes.clone()
    m = tr.step(PROMPTS)
    assert m["policy/grad_norm"] > 0 and gaps(tr) < tol
    assert not torch.equal(before, tr.engine.w.layers[0].fp4["fc1_w"].codes)


def test_log_probs_of_rollout_and_policy_agree():
    tr = trainer()
    tr.step(PROMPTS)
    for s in tr.last_samples:
        P, S = s["prompt_length"], s["sequence_length"]
        assert torch.allclose(s["logprobs"][P - 1:S - 1], s["rollout_log_probs"][P - 1:S - 1], atol=2e-3)


def test_a_policy_without_quantisation_is_served_in_4_bits_wherever_groups_are_whole():
    tr = trainer(qat=False, acts="fp8")
    assert set(tr.engine.w.layers[0].fp4) == {"qkv_w", "o_w", "fc1_w", "fc2_w"}
    assert tr.step(PROMPTS)["policy/grad_norm"] > 0


def test_adapters_and_block_fp8_are_refused_before_anything_is_built():
    with pytest.raises(ValueError, match="not in both"):
        trainer(qat=False, fp8=True)
    cfg = make_cfg()
    cfg.sampler.infer_engine_configs[0].fp4_weights = cfg.sampler.infer_engine_configs[0].fp8_weights = True
    with pytest.raises(ValueError, match="not in both"):
        GrpoTrainer(cfg, model_cfg=ModelConfig(num_layers=1, hidden_size=128, num_attention_heads=2, num_kv_heads=2, ffn_hidden_size=128,
                                               vocab_size=512, dtype="float32"), reward_fn=reward_has_small_token).setup()
    cfg.policy.lora.rank = 8
    for qat in (False, True):
        with pytest.raises(ValueError, match="LoRA"):
            trainer(qat=qat, lora=cfg.policy.lora)


def test_engines_that_are_not_served_in_4_bits_say_so():
    from types import SimpleNamespace
    from gcore_b200.entry import lm_infer, train_lm_distill
    from gcore_b200.rollout.disaggregated import SamplerServer
    from gcore_b200.trainer.disagg_trainer import DisaggGrpoTrainer
    cfg = make_cfg()
    cfg.sampler.infer_engine_configs[0].fp4_weights = True
    never = SimpleNamespace(cfg=cfg)   # whatever else they touch is missing
    for call in (lambda: SamplerServer(cfg, None, None), lambda: DisaggGrpoTrainer.setup(never),
                 lambda: train_lm_distill.off_policy_loop(never, [], 1, None), lambda: lm_infer.serve_checkpoint(cfg, {})):
        with pytest.raises(NotImplementedError, match="fp4_weights"):
            call()


@pytest.mark.parametrize("policy", [dict(), dict(share_rollout_weights=False),
                                    dict(share_rollout_weights=False, release_rollout_weights=True)])
@pytest.mark.parametrize("mode", ["fp4", "fp8"])
def test_a_hand_over_quantises_once(policy, mode, monkeypatch):
    if mode == "fp4":
        tr = trainer(**policy)
    else:
        tr = trainer_fp8(**policy)
    name = f"quantize_weights_{mode}"
    calls, quantise = [], getattr(tr.engine, name)
    monkeypatch.setattr(tr.engine, name, lambda *a, **k: calls.append(a) or quantise(*a, **k))
    tr.step(PROMPTS)
    assert len(calls) == 1
    lw = tr.engine.w.layers[0] if tr.engine.w is not None else None
    assert lw is None or (lw.fp4 if mode == "fp4" else lw.fp8)


def trainer_fp8(**policy):
    cfg = make_cfg()
    for k, v in policy.items():
        setattr(cfg.policy, k, v)
    cfg.sampler.infer_engine_configs[0].fp8_weights = True
    mcfg = ModelConfig(arch="qwen2", num_layers=2, hidden_size=256, num_attention_heads=4, num_kv_heads=2, ffn_hidden_size=352,
                       vocab_size=512, dtype="float32")
    return GrpoTrainer(cfg, model_cfg=mcfg, reward_fn=reward_has_small_token).setup()
