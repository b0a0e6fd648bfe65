"""TransformerLM(fused_layers=True) under autocast: fp32 weights, 16-bit products, as PyTorch's layers run there."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("attention_type", ["dense_flash", "learned_address", "key_vector"])
def test_autocast(attention_type, dtype, cuda_device):
    from wayfinder_attention_b200 import TransformerLM

    args = dict(d_model=128, n_layers=2, n_heads=2, d_ff=256, max_seq_len=128, dropout=0.0,
                attention_type=attention_type, routing_top_k=32)
    torch.manual_seed(3)
    plain = TransformerLM(96, **args).to(cuda_device)
    fused = TransformerLM(96, fused_layers=True, **args).to(cuda_device)
    fused.load_state_dict(plain.state_dict())
    ids = torch.randint(1, 96, (2, 128), device=cuda_device)
    exact = plain(ids)["logits"].detach()
    with torch.autocast("cuda", dtype=dtype):
        a, b = plain(ids)["logits"], fused(ids)["logits"]
        assert a.dtype == b.dtype == dtype
        r = fused.score(ids)
    # both are the fp32 model with 16-bit roundings: as far from it as each other (the usual spread of
    # two such runs is well below a factor of 1.5)
    near, far = (b.float() - exact).norm(), (a.float() - exact).norm()
    assert near <= 1.5 * far
    (-r.logprob.mean()).backward()
    for n, p in fused.named_parameters():
        if ".address." not in n:
            assert p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all(), n


def test_operators_keep_their_types(cuda_device):
    """The operators themselves take what they are given: autocast is the modules'."""
    from wayfinder_attention_b200 import fused_linear, layer_norm

    x, w = torch.randn(4, 32, device=cuda_device), torch.randn(8, 32, device=cuda_device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert fused_linear(x, w).dtype == torch.float32 and layer_norm(x.bfloat16()).dtype == torch.bfloat16
