"""TransformerLM on the fused layers: the same model as on PyTorch's, forward, scored and trained."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _pair(attention_type, dev, dtype=torch.float32, **kw):
    from wayfinder_attention_b200 import TransformerLM

    args = dict(d_model=128, n_layers=2, n_heads=2, d_ff=256, max_seq_len=256, dropout=0.0,
                attention_type=attention_type, routing_top_k=64, **kw)
    torch.manual_seed(3)
    plain = TransformerLM(96, **args).to(dev, dtype)
    fused = TransformerLM(96, fused_layers=True, **args).to(dev, dtype)
    fused.load_state_dict(plain.state_dict())
    return plain, fused


def _ids(dev, B=2, T=200, vocab=96):
    g = torch.Generator(device=dev).manual_seed(4)
    return torch.randint(1, vocab, (B, T), device=dev, generator=g)


def test_default_layers_are_unchanged(cuda_device):
    plain, _ = _pair("dense_flash", cuda_device)
    ids = _ids(cuda_device)
    x = plain.token_emb(ids) + plain.pos_emb(torch.arange(200, device=cuda_device))
    for b in plain.blocks:
        x = x + b.attn(b.ln1(x))
        x = x + b.ff(b.ln2(x))
    with torch.no_grad():
        assert torch.equal(plain(ids)["logits"], plain.lm_head(plain.ln_f(x)))


@pytest.mark.parametrize("attention_type", ["dense_flash", "learned_address", "key_vector"])
def test_fused_layers_match_pytorch_layers(attention_type, cuda_device):
    """fp32: logits of size about 10 agree to fp32 rounding through two blocks (2^-12 of it)."""
    plain, fused = _pair(attention_type, cuda_device)
    ids = _ids(cuda_device)
    with torch.no_grad():
        a, b = plain(ids)["logits"], fused(ids)["logits"]
    # retrieval may swap keys whose scores tie to the last bits: a row or two at most
    off = (a - b).abs().amax(-1) > 2.0 ** -12 * a.abs().max()
    assert off.sum() <= (0 if attention_type == "dense_flash" else 2)


def test_score_and_gradients_match_pytorch(cuda_device):
    plain, fused = _pair("dense_flash", cuda_device)
    ids = _ids(cuda_device)
    ids[1, 150:] = 0  # padding
    r = fused.score(ids, top_n=4)
    logits = plain(ids)["logits"]
    logp = F.log_softmax(logits[:, :-1], -1)
    nll = F.cross_entropy(logits[:, :-1].reshape(-1, 96), ids[:, 1:].reshape(-1), ignore_index=0, reduction="sum")
    want = logp.gather(-1, ids[:, 1:, None])[..., 0]
    kept = ids[:, 1:] != 0
    assert r.logprob.shape == (2, 199) and r.top_tokens.shape == (2, 199, 4)
    assert (r.logprob - want)[kept].abs().max() <= 1e-3 and not r.logprob[~kept].any()
    assert (r.entropy - torch.special.entr(logp.exp()).sum(-1)).abs().max() <= 1e-3
    assert (r.top_logprobs - logp.topk(4, -1).values).abs().max() <= 1e-3
    (-r.logprob.sum()).backward()
    nll.backward()
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        if name.endswith("k_proj.bias"):
            # a softmax does not see what all its scores share: this gradient is 0 but for rounding
            assert max(p.grad.norm(), q.grad.norm()) <= 1e-4 * fused.blocks[0].attn.q_proj.bias.grad.norm()
            continue
        # fp32 through two blocks and 350 tokens, the relative error of sums of that length
        assert (p.grad - q.grad).norm() <= 1e-3 * p.grad.norm() + 1e-6, name


def test_training_learns(cuda_device):
    """bf16, learned addresses: a few steps of SGD on one batch lower its loss, with every operator's gradient in it."""
    from wayfinder_attention_b200 import check_status

    _, lm = _pair("learned_address", cuda_device, torch.bfloat16)
    ids = _ids(cuda_device)
    losses = []
    for _ in range(8):
        lm.zero_grad(set_to_none=True)
        loss = -lm.score(ids).logprob.mean()
        loss.backward()
        # addresses pick keys and carry no gradient
        assert all(p.grad is not None and torch.isfinite(p.grad).all()
                   for n, p in lm.named_parameters() if ".address." not in n)
        with torch.no_grad():
            for p in lm.parameters():
                if p.grad is not None:
                    p -= 0.1 * p.grad / p.grad.float().norm().clamp_min(1e-6).to(p.dtype)
        losses.append(loss.item())
    check_status()
    assert losses[-1] < losses[0] - 0.2, losses


def test_dropout_comes_between_the_fused_layers(cuda_device):
    from wayfinder_attention_b200 import TransformerLM

    torch.manual_seed(5)
    lm = TransformerLM(96, d_model=64, n_layers=1, n_heads=2, d_ff=128, max_seq_len=64, dropout=0.5,
                       attention_type="dense_flash", fused_layers=True).to(cuda_device)
    ids = _ids(cuda_device, T=64)
    a, b = lm(ids)["logits"], lm(ids)["logits"]
    assert not torch.equal(a, b)
    lm.eval()
    with torch.no_grad():
        assert torch.equal(lm(ids)["logits"], lm(ids)["logits"])


def test_one_token_and_captured_graph(cuda_device):
    """A single position runs; a captured scoring pass equals its eager calls on new inputs."""
    from wayfinder_attention_b200 import CapturedForward

    _, fused = _pair("learned_address", cuda_device, torch.bfloat16,
                     retrieval_config={"use_fused_sparse": True, "method": "fused_causal"})
    fused.eval()
    with torch.no_grad():
        assert torch.isfinite(fused(_ids(cuda_device, B=3, T=1))["logits"]).all()
        ids = _ids(cuda_device)
        cap = CapturedForward(lambda i: tuple(fused.score(i, top_n=3)), ids)
        new = torch.flip(ids, (1,))
        got = [t.clone() for t in cap(new)]
        want = fused.score(new, top_n=3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
