"""TransformerLM(fused_ends=True): a hook on the model itself and a subclass's forward see every scoring."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(cls, dev, fused_ends):
    torch.manual_seed(3)
    return cls(96, d_model=64, n_layers=1, n_heads=1, d_ff=128, max_seq_len=64, dropout=0.0, attention_type="dense_flash",
               fused_ends=fused_ends).to(dev)


def test_hooks_and_subclasses(cuda_device):
    from wayfinder_attention_b200 import TransformerLM

    class Cooler(TransformerLM):
        def forward(self, input_ids, attn_mask=None):
            return {"logits": super().forward(input_ids, attn_mask)["logits"] * 2.0}

    class Plain(TransformerLM):
        pass

    g = torch.Generator(device=cuda_device).manual_seed(4)
    ids = torch.randint(1, 96, (2, 40), device=cuda_device, generator=g)
    with torch.no_grad():
        for cls in (TransformerLM, Cooler, Plain):
            want, got = _model(cls, cuda_device, False).loss(ids), _model(cls, cuda_device, True).loss(ids)
            assert abs(want - got) <= 1e-5 * want, cls
        for hook in (lambda m, args, out: {"logits": out["logits"] * 2.0}, lambda m, args, out: None):
            want, got = (_model(TransformerLM, cuda_device, ends) for ends in (False, True))
            for lm in (want, got):
                lm.register_forward_hook(hook)
            assert abs(want.loss(ids) - got.loss(ids)) <= 1e-5 * want.loss(ids)
        seen = []
        lm = _model(TransformerLM, cuda_device, True)
        handle = lm.register_forward_pre_hook(lambda m, args: seen.append(1))
        lm.loss(ids)
        lm.score(ids)
        assert len(seen) == 2
        handle.remove()
        lm.loss(ids)
        assert len(seen) == 2
