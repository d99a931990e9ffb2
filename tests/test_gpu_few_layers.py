"""few_tokens in the layers a model uses: QoSMoELayer (config.few_tokens) and patch(few_tokens=).

Whole fp32 models, whose small calls then run as one kernel, keep their logits within 1e-4 (max|d| /
max|ref|), the tolerance of the layers' other path; calls above the limit are bit-equal to it."""
import pytest
import torch

from hf_models import QWEN_PLUGIN, SWITCH_PLUGIN, qwen_model, switch_model, token_batch
from oracle import oracle as O
from dsca_moe_b200 import QoSMoEConfig, QoSMoELayer, RequestStateTable, get_qosmoe_layers, patch, replace_qosmoe_layer

pytestmark = pytest.mark.gpu
pytest.importorskip("transformers")

F32_TOL = 1e-4


class Calls:
    """Counts an engine's one-kernel calls."""

    def __init__(self, engine):
        self.n, self.call = 0, engine.forward_few
        engine.forward_few = self

    def __call__(self, x):
        self.n += 1
        return self.call(x)


@pytest.mark.parametrize("few", [0, 32])
@torch.no_grad()
def test_switch_model(cuda, few):
    model = switch_model(seed=3).to(cuda)
    ids = token_batch(model.config.vocab_size, 4, 64, seed=4).to(cuda)
    dec = token_batch(model.config.vocab_size, 4, 5, seed=5).to(cuda)
    ref = model(input_ids=ids, decoder_input_ids=dec).logits
    cfg = QoSMoEConfig(rank=0, world_size=1, expert_cache_size=1 << 10, few_tokens=few)
    replace_qosmoe_layer(model, config=cfg, **SWITCH_PLUGIN)
    layers = get_qosmoe_layers(model)
    ctx = RequestStateTable(cfg).build_context({"attention_mask": torch.ones(4, 64, dtype=torch.long)})
    calls = []
    for layer in layers:
        layer.set_runtime_context(ctx)
        calls.append(Calls(layer.engine))
    got = model(input_ids=ids, decoder_input_ids=dec).logits
    torch.cuda.synchronize()
    for layer in layers:
        layer.engine.check()
    # the encoder's 256 tokens take the other path, the decoder's 20 the one kernel
    assert sum(c.n for c in calls) == (len(layers) // 2 if few else 0)
    assert O.max_rel_err(got.cpu().numpy(), ref.cpu().numpy()) < F32_TOL


@torch.no_grad()
def test_qwen_model_patched(cuda):
    model = qwen_model(seed=7, layers=3).to(cuda)
    ids = token_batch(model.config.vocab_size, 2, 16, seed=8).to(cuda)
    ref = model(input_ids=ids).logits
    assert patch(model, 0, 1, few_tokens=32) == 3
    engines = [m.engine for m in model.modules() if hasattr(m, "engine")]
    calls = [Calls(e) for e in engines]
    got = model(input_ids=ids).logits
    torch.cuda.synchronize()
    assert [c.n for c in calls] == [1, 1, 1]
    assert O.max_rel_err(got.cpu().numpy(), ref.cpu().numpy()) < F32_TOL
    for e in engines:
        e.check()
    ids = token_batch(model.config.vocab_size, 3, 11, seed=9).to(cuda)  # 33 tokens
    big = model(input_ids=ids).logits
    for e in engines:
        e.few_tokens = 0
    assert torch.equal(model(input_ids=ids).logits, big)
    assert [c.n for c in calls] == [1, 1, 1]


@pytest.mark.parametrize("T", [1, 32, 33])
def test_layer_statistics(cuda, T):
    """The statistics of a layer are the same whichever path runs it."""
    g = torch.Generator().manual_seed(11)
    E, d, F = 6, 64, 96
    sds = [{"wi.weight": torch.randn(F, d, generator=g) * 0.1, "wo.weight": torch.randn(d, F, generator=g) * 0.1}
           for _ in range(E)]
    router, x = torch.randn(E, d, generator=g), torch.randn(1, T, d, generator=g).to(cuda)
    res = []
    for few in (0, 32):
        cfg = QoSMoEConfig(rank=0, world_size=1, experts=sds, router_weights=router, d_model=d, num_experts=E,
                           expert_cache_size=E, collect_stats=True, few_tokens=few)
        layer = QoSMoELayer(cfg)
        layer.set_runtime_context(RequestStateTable(cfg).build_context(
            {"attention_mask": torch.ones(1, T, dtype=torch.long)}))
        y, (logits, idx) = layer(x)
        layer.engine.check()
        st = layer.get_statistics()
        assert len(st) == 1 and sum(st[0]["expert distribution"]) == T
        res.append((y, logits, idx, st[0]["expert distribution"], st[0]["total number of tokens sent"]))
    (y0, l0, i0, f0, s0), (y1, l1, i1, f1, s1) = res
    assert y0.shape == y1.shape == (1, T, d) and l0.shape == l1.shape and i0.shape == i1.shape
    assert torch.equal(i0, i1) and list(f0) == list(f1) and s0 == s1
    assert O.max_rel_err(y1.cpu().numpy(), y0.cpu().numpy()) < F32_TOL
