"""The rollout engine with 4-bit projections: what it serves, and what it refuses (PyTorch definitions)."""
import pytest
import torch

from gcore_b200.configs.base import ConfigError
from gcore_b200.configs.config import InferEngineConfig
from gcore_b200.models.config import ModelConfig
from gcore_b200.models.gpt import GPTModel
from gcore_b200.ops.quant import Fp4Weight
from gcore_b200.rollout.engine import InferEngine, RolloutWeights, SamplingParams

CFG = dict(num_layers=2, hidden_size=256, num_attention_heads=4, num_kv_heads=2, ffn_hidden_size=352, vocab_size=512, dtype="float32")
NAMES = ("qkv_w", "o_w", "fc1_w", "fc2_w")


def build():
    cfg = ModelConfig(**CFG)
    model = GPTModel(cfg, tp_size=1)
    model.reset_parameters(4)
    return cfg, model


def engine(cfg, model):
    e = InferEngine(cfg, RolloutWeights.from_model(model, clone=True), num_kv_blocks=64, kv_block_size=4, max_model_len=48,
                    use_cuda_graph=False)
    e.wake_up(("kv_cache",))
    return e


def generate(e):
    return e.generate([[5, 9, 33, 70, 2], [100, 101, 102]], SamplingParams(max_new_tokens=6, greedy=True))


def test_4_bit_serving_is_the_model_with_4_bit_values():
    cfg, model = build()
    served, plain = engine(cfg, model), engine(cfg, model)
    served.quantize_weights_fp4()
    assert set(served.w.layers[0].fp4) == set(NAMES) and served.w.layers[0].fp8 is None
    for lw in plain.w.layers:   # the values a model trained with fp4_qat multiplies with
        for name in NAMES:
            setattr(lw, name, Fp4Weight.of(getattr(lw, name).bfloat16()).values(torch.float32))
    for a, b in zip(generate(served), generate(plain)):
        assert a.out_tokens == b.out_tokens
        assert max(abs(x - y) for x, y in zip(a.out_logprobs, b.out_logprobs)) < 1e-4


def test_4_bit_serving_with_8_bit_activations_stays_near_and_follows_the_weights():
    cfg, model = build()
    e, ref = engine(cfg, model), engine(cfg, model)
    e.quantize_weights_fp4("fp8")
    ref.quantize_weights_fp4("bf16")
    h = torch.randn(3, 256)
    lw = e.w.layers[0]
    q, res = e._norm_for(h, lw.ln1, None, lw, "qkv_w")
    assert isinstance(q, tuple) and q[0].dtype == torch.float8_e4m3fn and q[1].dtype == torch.float8_e8m0fnu and res is h
    a, _ = e._mlp(lw, q, reduce=False)
    b, _ = ref._mlp(ref.w.layers[0], ref._norm_for(h, lw.ln1, None, ref.w.layers[0], "fc1_w")[0], reduce=False)
    assert (a - b).norm() / b.norm() < 0.1          # three e4m3 roundings of a sixteenth at most, mostly independent
    generate(e)
    old = e.w.layers[0].fp4["fc1_w"].codes.clone()
    for lw in e.w.layers:
        lw.fc1_w.mul_(-1)
    e.update_weights()
    new = e.w.layers[0].fp4["fc1_w"].codes
    assert e.fp4_activations == "fp8" and not torch.equal(new, old)
    e.quantize_weights_fp8()                        # the other mode takes over
    assert e.fp4_activations is None and e.w.layers[0].fp4 is None and e.w.layers[0].fp8
    e.quantize_weights_fp4()
    assert not e.fp8_enabled and e.w.layers[0].fp8 is None


def test_refusals():
    cfg, model = build()
    with pytest.raises(ValueError, match="activations"):
        engine(cfg, model).quantize_weights_fp4("int8")
    with pytest.raises(ConfigError, match="fp4_activations"):
        InferEngineConfig(fp4_activations="int8")
    with pytest.raises(ConfigError, match="not in both"):
        InferEngineConfig(fp4_weights=True, fp8_weights=True)
