"""A block on the fused layers adds its residual whatever attention module it was given."""

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


class IgnoresKeywords(nn.Module):
    """An attention that takes any keyword and knows of none."""

    def __init__(self, d):
        super().__init__()
        self.proj = nn.Linear(d, d)

    def forward(self, x, attn_mask=None, **kwargs):
        return self.proj(x)


class TakesNoKeywords(IgnoresKeywords):
    def forward(self, x, attn_mask=None):
        return self.proj(x)


def _modules(d):
    from wayfinder_attention_b200 import DenseSDPAAttention, KeyVectorSparseAttention, RouterMLP, RoutingSparseAttention

    class Overrides(DenseSDPAAttention):
        """Inherits the fused projections, not the residual."""

        def forward(self, x, **kwargs):
            return super().forward(x)

    return {
        "ignores keywords": IgnoresKeywords(d),
        "takes no keywords": TakesNoKeywords(d),
        "routing": RoutingSparseAttention(d, 2, RouterMLP(d, routing_dim=16), top_k=16, dropout=0.0),
        "key vectors": KeyVectorSparseAttention(d, 2, top_k=16, dropout=0.0),
        "dense": DenseSDPAAttention(d, 2, 0.0),
        "overrides": Overrides(d, 2, 0.0),
    }


@pytest.mark.parametrize("which", ["ignores keywords", "takes no keywords", "routing", "key vectors", "dense", "overrides"])
def test_residual_is_added(which, cuda_device):
    from wayfinder_attention_b200 import TransformerBlock

    torch.manual_seed(7)
    d = 64
    attn = _modules(d)[which]
    plain = TransformerBlock(d, 2, 128, 0.0, attn).to(cuda_device).eval()
    x = torch.randn(2, 48, d, device=cuda_device)
    with torch.no_grad():
        want = plain(x)
        fused = TransformerBlock(d, 2, 128, 0.0, attn, fused_layers=True).to(cuda_device).eval()
        fused.load_state_dict(plain.state_dict())
        got = fused(x)
    # fp32 through one block of values of size 4: 2^-14; retrieval may swap keys that tie to the last bits
    off = (got - want).abs().amax(-1) > 2.0 ** -12
    assert off.sum() <= (2 if which in ("routing", "key vectors") else 0)


def test_attention_replaced_later(cuda_device):
    from wayfinder_attention_b200 import TransformerLM

    torch.manual_seed(8)
    lm = TransformerLM(50, d_model=64, n_layers=1, n_heads=2, d_ff=128, max_seq_len=32, dropout=0.0,
                       attention_type="dense_flash", fused_layers=True)
    lm.blocks[0].attn = IgnoresKeywords(64)
    lm = lm.to(cuda_device).eval()
    ids = torch.randint(1, 50, (2, 32), device=cuda_device)
    with torch.no_grad():
        got = lm(ids)["logits"]
        lm.fused_layers = lm.blocks[0].fused_layers = False
        assert (got - lm(ids)["logits"]).abs().max() <= 1e-4
