"""fused_layers=True runs the modules that the model has: hooked, wrapped, replaced or parametrised ones too."""

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


class Adapter(nn.Module):
    """A linear layer with a low-rank addition, as fine-tuning puts in its place."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.a, self.b = nn.Linear(base.in_features, 4, bias=False), nn.Linear(4, base.out_features, bias=False)

    def forward(self, x):
        return self.base(x) + self.b(self.a(x))


def _lm(dev, **kw):
    from wayfinder_attention_b200 import TransformerLM

    torch.manual_seed(9)
    return TransformerLM(70, d_model=64, n_layers=2, n_heads=2, d_ff=128, max_seq_len=40, dropout=0.0,
                         attention_type="dense_flash", fused_layers=True, **kw).to(dev)


def _both(lm, ids):
    """Logits on the fused operators and on PyTorch's layers, of the same modules."""
    fused = lm(ids)["logits"]
    _set(lm, False)
    plain = lm(ids)["logits"]
    _set(lm, True)
    return fused, plain


def _set(lm, on):
    lm.fused_layers = on
    for b in lm.blocks:
        b.fused_layers = b.attn.fused_linear = on


def _ids(dev):
    return torch.randint(1, 70, (2, 40), device=dev, generator=torch.Generator(device=dev).manual_seed(1))


PLACES = ["blocks.0.ff.0", "blocks.1.ff.3", "blocks.0.attn.q_proj", "blocks.1.attn.out_proj", "lm_head"]


@pytest.mark.parametrize("place", PLACES)
def test_adapters(place, cuda_device):
    lm = _lm(cuda_device)
    parent, _, name = place.rpartition(".")
    owner = lm.get_submodule(parent)
    ids = _ids(cuda_device)
    with torch.no_grad():
        before = lm(ids)["logits"]
        setattr(owner, name, Adapter(lm.get_submodule(place)).to(cuda_device))
        fused, plain = _both(lm, ids)
    assert (fused - plain).abs().max() <= 2e-4 and (fused - before).abs().max() > 1e-2


@pytest.mark.parametrize("place", PLACES + ["blocks.0.ln1", "blocks.1.ln2", "ln_f", "blocks.0.ff.1", "blocks.0.ff.4",
                                            "blocks.1.ff", "blocks.1.attn"])
def test_hooks(place, cuda_device):
    """A hook sees the module's output, as without the fused layers, and may replace it."""
    lm = _lm(cuda_device)
    ids = _ids(cuda_device)
    seen = []
    module = lm.get_submodule(place)
    handle = module.register_forward_hook(lambda m, i, o: seen.append(o.detach().clone()))
    with torch.no_grad():
        fused, plain = _both(lm, ids)
    assert len(seen) == 2 and (seen[0] - seen[1]).abs().max() <= 2e-4 and (fused - plain).abs().max() <= 2e-4
    handle.remove()
    module.register_forward_hook(lambda m, i, o: o * 0.5)
    with torch.no_grad():
        halved, plain = _both(lm, ids)
    assert (halved - plain).abs().max() <= 2e-4 and (halved - fused).abs().max() > 1e-2


def test_pre_hooks_and_backward_hooks(cuda_device):
    lm = _lm(cuda_device)
    ids, calls = _ids(cuda_device), []
    lm.blocks[0].ff[0].register_forward_pre_hook(lambda m, i: (i[0] * 2,))
    lm.blocks[1].ff[3].register_full_backward_hook(lambda m, gi, go: calls.append(1))
    fused, plain = _both(lm, ids)
    assert (fused - plain).abs().max() <= 2e-4
    fused.sum().backward()
    assert calls


def test_parametrised_and_replaced(cuda_device):
    lm = _lm(cuda_device)
    ids = _ids(cuda_device)
    nn.utils.parametrizations.weight_norm(lm.blocks[0].ff[0])
    lm.blocks[0].ff[1] = nn.Tanh()
    lm.blocks[1].ff[1] = nn.GELU(approximate="tanh")
    lm.blocks[1].ln1 = nn.RMSNorm(64).to(cuda_device)
    lm.blocks[1].ff.append(nn.Tanh())
    with torch.no_grad():
        fused, plain = _both(lm, ids)
    assert (fused - plain).abs().max() <= 2e-4


def test_dropout_of_its_own_mode(cuda_device):
    """A dropout that was put in training mode by itself acts, whatever the block's mode."""
    from wayfinder_attention_b200 import TransformerLM

    torch.manual_seed(5)
    lm = TransformerLM(70, d_model=64, n_layers=1, n_heads=2, d_ff=128, max_seq_len=40, dropout=0.5,
                       attention_type="dense_flash", fused_layers=True).to(cuda_device).eval()
    lm.blocks[0].ff[4].train()
    with torch.no_grad():
        ids = _ids(cuda_device)
        assert not torch.equal(lm(ids)["logits"], lm(ids)["logits"])
