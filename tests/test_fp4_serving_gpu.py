"""The rollout engine with quantised projections on the GPU: norms and activations that end in e4m3 inside captured decode steps, and
4-bit weights against the model that holds their values."""
import pytest
import torch

from gcore_b200.models.config import ModelConfig
from gcore_b200.models.gpt import GPTModel
from gcore_b200.ops import quant
from gcore_b200.rollout.engine import InferEngine, RolloutWeights, SamplingParams

pytestmark = pytest.mark.gpu

NAMES = ("qkv_w", "o_w", "fc1_w", "fc2_w")
CFG = dict(arch="qwen2", num_layers=2, hidden_size=512, num_attention_heads=4, num_kv_heads=2, head_dim=128, ffn_hidden_size=1024,
           vocab_size=2048, qkv_bias=True, dtype="bfloat16")


def build(**kw):
    cfg = ModelConfig(**{**CFG, **kw})
    torch.manual_seed(0)
    return cfg, GPTModel(cfg, recompute="none", device=torch.device("cuda")).eval()


def engine(cfg, model, graph=True):
    return InferEngine(cfg, RolloutWeights.from_model(model, clone=True), max_running_requests=8, max_model_len=64, kv_block_size=16,
                       sync_interval=4, use_cuda_graph=graph, device=torch.device("cuda"))


def generate(e, n_new=10):
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(3, 2048, (n,), generator=g).tolist() for n in (5, 9, 14, 7, 11)]
    reqs = e.generate(prompts, SamplingParams(max_new_tokens=n_new, temperature=1.0, seed=7), n=2)
    return [r.out_tokens for r in reqs], [r.out_logprobs for r in reqs]


def test_block_fp8_serving_gives_the_same_bits_as_the_unfused_chain(monkeypatch):
    cfg, model = build()
    a, b = engine(cfg, model), engine(cfg, model)
    a.quantize_weights_fp8()
    b.quantize_weights_fp8()
    fused = generate(a)
    assert a.stats["graph_replays"] > 0
    monkeypatch.setattr(InferEngine, "_input_scales", lambda self, h, lw, name: None)
    assert generate(b) == fused


def test_4_bit_serving_is_the_model_with_4_bit_values():
    """16-bit activations: the same products as a bf16 model with the weights' values, up to the order of a sum."""
    cfg, model = build()
    served, plain = engine(cfg, model), engine(cfg, model)
    served.quantize_weights_fp4()
    for lw in plain.w.layers:
        for name in NAMES:
            setattr(lw, name, quant.Fp4Weight.of(getattr(lw, name)).values().clone())
    (ta, la), (tb, lb) = generate(served), generate(plain)
    assert served.stats["graph_replays"] > 0
    same = 0
    for x, y, p, q in zip(ta, tb, la, lb):
        for i, (t, u) in enumerate(zip(x, y)):
            assert abs(p[i] - q[i]) < 0.06   # the bound between the engine and the trainer's forward in bf16
            if t != u:
                break
            same += 1
    assert same > 50   # of 100: a token differs only where two draws are within the noise of bf16


def test_4_bit_serving_with_8_bit_activations_runs_captured_and_as_launches():
    cfg, model = build()
    a, b = engine(cfg, model), engine(cfg, model, graph=False)
    for e in (a, b):
        e.quantize_weights_fp4("fp8")
    x, y = generate(a), generate(b)
    assert a.stats["graph_replays"] > 0 and x == y
    # and the norm, product, activation, product of one layer against 64 bits
    lw, h = a.w.layers[0], torch.randn(6, 512, device="cuda").bfloat16()
    with torch.no_grad():
        (q, s), _ = a._norm_for(h, lw.ln2, None, lw, "fc1_w")
        got, _ = a._mlp(lw, (q, s), reduce=False)
    w1, w2 = (lw.fp4[n].values(torch.float32).double() for n in ("fc1_w", "fc2_w"))
    g, u = ((q.double().unflatten(-1, (-1, 32)) * s.double()[..., None]).flatten(-2) @ w1.t()).chunk(2, -1)
    act = g * torch.sigmoid(g) * u
    # one bf16 rounding of gate and up and one e4m3 rounding of their product lie between: at most 2^-8 (1 + |gate|) + 2^-8 and
    # 2^-4 relative, and a group's smallest values 2^-10 of its scale, at most 2^-18 of its largest value twice
    tol = act.abs() * (2 ** -4 + 2 ** -8 * (2 + g.abs())) * 1.1 + act.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(
        -1, -1, 32).flatten(-2) * 2 ** -17
    want = act @ w2.t()
    assert ((got.double() - want).abs() <= tol @ w2.abs().t() + 2 ** -8 * want.abs() + 1e-6).all()


def test_widths_without_whole_tiles_are_served_too():
    """Contraction lengths of whole groups of 32 that are not whole tiles of 128."""
    cfg, model = build(hidden_size=416, num_attention_heads=4, num_kv_heads=2, head_dim=64, ffn_hidden_size=352)
    e = engine(cfg, model)
    for acts in ("bf16", "fp8"):
        e.quantize_weights_fp4(acts)
        assert set(e.w.layers[0].fp4) == set(NAMES)
        toks, lps = generate(e, 4)
        assert all(len(t) == 4 for t in toks) and all(torch.isfinite(torch.tensor(v)).all() for v in lps)
