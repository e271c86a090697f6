"""A policy trained with ``fp4_qat`` and its rollout engine with ``fp4_weights`` on the GPU: the same products, native kernels on
both sides."""
import pytest

from gcore_b200.ops import _lib
from test_fp4_qat_serving_cpu import PROMPTS, gaps, trainer

pytestmark = pytest.mark.gpu


def test_the_engine_serves_the_products_that_the_policy_trains():
    tr = trainer("bfloat16")
    assert tr.policy.device.type == "cuda" and set(tr.engine.w.layers[0].fp4) == {"qkv_w", "o_w", "fc1_w"}
    assert gaps(tr) < 2 ** -6   # either side is rounded once, 2^-8, and sums of 352 products are far more exact
    for _ in range(2):
        assert tr.step(PROMPTS)["policy/grad_norm"] > 0
    assert gaps(tr) < 2 ** -6
    s = tr.last_samples[0]
    P, S = s["prompt_length"], s["sequence_length"]
    gap = (s["logprobs"][P - 1:S - 1].cpu() - s["rollout_log_probs"][P - 1:S - 1].cpu()).abs().max()
    assert gap < 0.06   # the bound between the engine and the trainer's forward in bf16
    _lib.check_device_errors()
