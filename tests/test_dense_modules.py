"""GatedFFN and what models put on it, without a GPU: the cases that run the old module's layers, and the refusals."""
import copy

import pytest
import torch
import torch.nn as nn


class Gated(nn.Module):
    def __init__(self, dropout=None, names=("gate_proj", "up_proj", "down_proj"), d=8, inter=16):
        super().__init__()
        for n, s in zip(names, ((d, inter), (d, inter), (inter, d))):
            setattr(self, n, nn.Linear(*s, bias=False))
        self.names, self.act_fn = names, nn.SiLU()
        if dropout is not None:
            self.dropout = dropout

    def forward(self, x):
        g, u, o = (getattr(self, n) for n in self.names)
        h = self.act_fn(g(x)) * u(x)
        return o(self.dropout(h) if hasattr(self, "dropout") else h)


class Adapter(nn.Module):
    """A low-rank addition that shows its base's weight, as adapters do."""

    def __init__(self, base):
        super().__init__()
        self.base, self.a, self.b = base, nn.Linear(base.in_features, 2, bias=False), nn.Linear(2, base.out_features, bias=False)

    @property
    def weight(self):
        return self.base.weight

    def forward(self, x):
        return self.base(x) + self.b(self.a(x))


def _t5(dropout=0.3, act="gated-gelu"):
    from transformers import T5Config
    from transformers.models.t5.modeling_t5 import T5DenseGatedActDense

    return T5DenseGatedActDense(T5Config(d_model=8, d_ff=16, dropout_rate=dropout, feed_forward_proj=act))


def test_t5_block_in_training_mode():
    """T5's gated MLP keeps its dropout: the same numbers and gradients from the same seed."""
    from dsca_moe_b200 import GatedFFN

    torch.manual_seed(1)
    old = _t5().train()
    new = GatedFFN(copy.deepcopy(old))
    assert new.training and new.act == "gelu" and new.state_dict().keys() == old.state_dict().keys()
    x = torch.randn(64, 8)
    outs = []
    for m in (old, new):
        torch.manual_seed(7)
        y = m(x)
        y.square().sum().backward()
        outs.append([y.detach()] + [p.grad for p in m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert (outs[0][0] - old.eval()(x)).abs().max() > 1e-3  # the dropout was on
    assert not GatedFFN(_t5().eval()).training
    assert not new.eval().dropout.training


def test_t5_block_with_wo_in_fp32():
    from dsca_moe_b200 import GatedFFN

    old = _t5().eval().to(torch.bfloat16)
    old.wo.to(torch.float32)
    x = torch.randn(5, 8, dtype=torch.bfloat16)
    y = GatedFFN(old)(x)
    assert y.dtype == torch.float32 and torch.equal(y, old(x))


@pytest.mark.parametrize("layer", ["gate_proj", "up_proj", "down_proj"])
def test_adapters_and_hooks(layer):
    """One that is there is refused; one put on afterwards has its effect, and its gradient."""
    from dsca_moe_b200 import GatedFFN

    old = Gated()
    setattr(old, layer, Adapter(getattr(old, layer)))
    with pytest.raises(ValueError, match="adapters"):
        GatedFFN(old)
    new = GatedFFN(Gated())
    setattr(new, layer, Adapter(getattr(new, layer)))
    ref = Gated()
    for n in ref.names:
        setattr(ref, n, getattr(new, n))
    x = torch.randn(3, 8)
    y = new(x)
    assert torch.equal(y, ref(x))
    y.sum().backward()
    assert getattr(new, layer).b.weight.grad.abs().sum() > 0

    class Other(nn.Linear):
        pass

    old = Gated()
    setattr(old, layer, Other(*reversed(getattr(old, layer).weight.shape), bias=False))
    with pytest.raises(ValueError, match="adapters"):
        GatedFFN(old)
    for put in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"):
        old, calls = Gated(), []
        getattr(getattr(old, layer), put)(lambda *a: calls.append(1))
        with pytest.raises(ValueError, match="hooks"):
            GatedFFN(old)
        new = GatedFFN(Gated())
        getattr(getattr(new, layer), put)(lambda *a: calls.append(1))
        new(torch.randn(3, 8, requires_grad=True)).sum().backward()
        assert calls == [1]
    old = Gated()
    getattr(old, layer).forward = lambda t: t
    with pytest.raises(ValueError, match="hooks"):
        GatedFFN(old)
    old = Gated()
    old.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="hooks"):
        GatedFFN(old)


def test_other_parts_are_refused():
    from dsca_moe_b200 import GatedFFN

    old = Gated()
    old.norm = nn.LayerNorm(16)
    with pytest.raises(ValueError, match="norm"):
        GatedFFN(old)
    with pytest.raises(ValueError, match="dropout"):
        GatedFFN(Gated(dropout=nn.AlphaDropout(0.1)))


def test_plain_layers_take_the_block():
    """Nothing hangs on the layers: the call goes to gated_ffn, which takes tensors on a GPU alone."""
    from dsca_moe_b200 import GatedFFN

    for m in (GatedFFN(Gated()), GatedFFN(Gated(dropout=nn.Dropout(0.0))), GatedFFN(Gated(dropout=nn.Dropout(0.5)).eval()),
              GatedFFN(_t5().eval())):
        with pytest.raises(ValueError, match="GPU"):
            m(torch.randn(2, 8))


def test_int8_scales_stay_fp32(monkeypatch):
    """A model that changes its type leaves the 8-bit weights what they were."""
    import dsca_moe_b200.dense as D

    def quantize(w):  # (the kernel's, on the host)
        s = w.abs().amax(1) / 127
        return torch.round(w / s[:, None]).to(torch.int8), s

    monkeypatch.setattr(D, "_quantize", quantize)
    model = nn.Sequential(nn.Linear(8, 8), D.GatedFFN(Gated(), int8=True))
    was = {k: v.clone() for k, v in model[1].state_dict().items()}
    assert len(was) == 6
    for change in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.bfloat16)):
        change(model)
        now = model[1].state_dict()
        assert now.keys() == was.keys() and all(now[k].dtype == was[k].dtype and torch.equal(now[k], was[k]) for k in was)
    assert model[0].weight.dtype == torch.bfloat16
    model.to("meta")
    assert all(b.device.type == "meta" and b.dtype == was[n].dtype for n, b in model[1].named_buffers())


def test_a_refused_layer_leaves_the_model_as_it_was():
    from dsca_moe_b200 import GatedFFN, replace_dense_ffn

    class Layer(nn.Module):
        def __init__(self):
            super().__init__()
            self.mlp = Gated()

    model = nn.Sequential(Layer(), Layer())
    model[1].mlp.act_fn = nn.GELU()
    with pytest.raises(ValueError, match="not offered"):
        replace_dense_ffn(model, "Layer", "Gated")
    assert type(model[0].mlp) is Gated
    model[1].mlp.act_fn = nn.ReLU()
    assert replace_dense_ffn(model, "Layer", "Gated") == 2
    assert [type(m.mlp) for m in model] == [GatedFFN, GatedFFN] and model[1].mlp.act == "relu"
