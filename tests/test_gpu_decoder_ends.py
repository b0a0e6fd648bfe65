"""TransformerLM on the operators of its two ends: the same model, its loss and the tied weight's gradient, without logits."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _pair(dev, dtype=torch.float32, vocab=96, attention_type="dense_flash", **kw):
    """The model as it is by default, and with fused ends (and what else is asked for)."""
    from wayfinder_attention_b200 import TransformerLM

    args = dict(d_model=128, n_layers=2, n_heads=2, d_ff=256, max_seq_len=256, dropout=0.0,
                attention_type=attention_type, routing_top_k=64)
    torch.manual_seed(3)
    plain = TransformerLM(vocab, **args).to(dev, dtype)
    ends = TransformerLM(vocab, fused_ends=True, **args, **kw).to(dev, dtype)
    ends.load_state_dict(plain.state_dict())
    return plain, ends


def _ids(dev, B=2, T=200, vocab=96):
    g = torch.Generator(device=dev).manual_seed(4)
    ids = torch.randint(1, vocab, (B, T), device=dev, generator=g)
    ids[1, 150:] = 0  # padding
    return ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_forward_is_the_same(dtype, cuda_device):
    """The embedding is the same sum with the same rounding, and nothing else of the forward changes."""
    plain, ends = _pair(cuda_device, dtype)
    ids = _ids(cuda_device)
    with torch.no_grad():
        assert torch.equal(plain(ids)["logits"], ends(ids)["logits"])


@pytest.mark.parametrize("fused_layers", [False, True])
def test_loss_and_gradients_match_pytorch(fused_layers, cuda_device):
    plain, ends = _pair(cuda_device, fused_layers=fused_layers)
    ids = _ids(cuda_device)
    logits = plain(ids)["logits"]
    want = F.cross_entropy(logits[:, :-1].reshape(-1, 96), ids[:, 1:].reshape(-1), ignore_index=0)
    got = ends.loss(ids)
    assert got.dtype == torch.float32 and abs(got - want) <= 1e-5 * want
    assert abs(plain.loss(ids) - want) <= 1e-5 * want  # the default's loss too
    r = ends.score(ids)
    assert r.logprob.shape == (2, 199) and r.top_tokens.shape == (2, 199, 0) and not r.logprob[ids[:, 1:] == 0].any()
    four = ends.score(ids, top_n=4)  # alternatives need the logits
    assert four.top_tokens.shape == (2, 199, 4) and (four.logprob - r.logprob).abs().max() <= 1e-4
    got.backward()
    want.backward()
    for (name, p), q in zip(plain.named_parameters(), ends.parameters()):
        if name.endswith("k_proj.bias"):  # 0 but for rounding: a softmax does not see what all its scores share
            continue
        # fp32 through two blocks and 350 tokens, the relative error of sums of that length
        assert (p.grad - q.grad).norm() <= 1e-3 * p.grad.norm() + 1e-6, name


def test_a_batch_of_nothing_but_padding(cuda_device):
    _, ends = _pair(cuda_device)
    loss = ends.loss(torch.zeros(2, 20, dtype=torch.int64, device=cuda_device))
    loss.backward()
    assert loss == 0 and not any(p.grad.any() for p in ends.parameters() if p.grad is not None)


def test_training_step_of_all_operators(cuda_device):
    """bf16, learned addresses, a padded batch: every parameter but the addresses has a finite gradient.

    Behind the last attention it has the same bits twice; the gradients of retrieved keys and values, with
    all below them, are sums in an order that differs from pass to pass, with fused ends as without.
    """
    from wayfinder_attention_b200 import check_status

    _, ends = _pair(cuda_device, torch.bfloat16, vocab=1003, attention_type="learned_address", fused_layers=True)
    ids = _ids(cuda_device, vocab=1003)
    runs = []
    for _ in range(2):
        ends.zero_grad(set_to_none=True)
        ends.loss(ids).backward()
        runs.append({n: p.grad.clone() for n, p in ends.named_parameters() if p.grad is not None})
    check_status()
    assert all(".address." in n or (n in runs[0] and torch.isfinite(runs[0][n]).all()) for n, _ in ends.named_parameters())
    behind = [n for n in runs[0] if n.startswith(("ln_f.", "blocks.1.ff.", "blocks.1.ln2.", "blocks.1.attn.out_proj."))]
    assert len(behind) == 10 and all(torch.equal(runs[0][n], runs[1][n]) for n in behind)
    # tokens that do not occur, as input or as output, still get the head's gradient; positions behind the batch none
    assert runs[0]["token_emb.weight"].any(1).all() and not runs[0]["pos_emb.weight"][200:].any()


def test_captured_scoring_and_autocast(cuda_device):
    from wayfinder_attention_b200 import CapturedForward

    _, ends = _pair(cuda_device, torch.bfloat16, fused_layers=True)
    ids = _ids(cuda_device)
    with torch.no_grad():
        cap = CapturedForward(lambda i: tuple(ends.score(i))[:2], ids)
        new = torch.flip(ids, (1,))
        got = [t.clone() for t in cap(new)]
        want = ends.score(new)[:2]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    plain, ends = _pair(cuda_device, fused_layers=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = plain.loss(ids), ends.loss(ids)
    # bf16 rounds the logits of the one and not of the other
    assert abs(a - b) <= 2.0 ** -8 * a
    b.backward()
    assert ends.token_emb.weight.grad.dtype == torch.float32 and torch.isfinite(ends.token_emb.weight.grad).all()


def test_modules_that_are_not_what_they_stand_for_are_called(cuda_device):
    _, ends = _pair(cuda_device)
    ids = _ids(cuda_device)
    seen = []
    handles = [m.register_forward_hook(lambda *a, name=n: seen.append(name))
               for n, m in (("token", ends.token_emb), ("position", ends.pos_emb), ("head", ends.lm_head))]
    ends.loss(ids)
    assert sorted(seen) == ["head", "position", "token"]
    for h in handles:
        h.remove()
    ends.loss(ids)
    assert len(seen) == 3
    plain, ends = _pair(cuda_device)
    for lm in (plain, ends):
        lm.token_emb.padding_idx = 0  # its row takes no gradient from the embedding, only from the head
        lm.loss(ids).backward()
    assert (plain.token_emb.weight.grad[0] - ends.token_emb.weight.grad[0]).norm() <= 1e-3 * plain.token_emb.weight.grad[0].norm()


def test_no_logits_in_memory(cuda_device):
    """16384 tokens over 60001: 3.9 GB of fp32 logits; the pass stays below 1.2 GB, of which 512 MB are its piece of them."""
    from wayfinder_attention_b200 import linear_token_logprobs

    x = torch.randn(16384, 64, device=cuda_device).bfloat16().requires_grad_()
    w = torch.randn(60001, 64, device=cuda_device).bfloat16().requires_grad_()
    t = torch.randint(0, 60001, (16384,), device=cuda_device)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    linear_token_logprobs(x, w, t).logprob.mean().backward()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1.2e9
    assert torch.isfinite(x.grad).all() and torch.isfinite(w.grad).all()


@pytest.mark.parametrize("which", ["embedding", "head"])
def test_a_captured_backward_beside_a_live_graph(which, cuda_device):
    """Refused while a graph of the same leaf, made on the default stream, lives; captured and replayed once that is gone."""
    from wayfinder_attention_b200 import linear_token_logprobs, token_embedding

    w = torch.randn(300, 64, device=cuda_device).requires_grad_()
    x, tokens = torch.randn(70, 64, device=cuda_device), torch.randint(0, 300, (70,), device=cuda_device)

    def loss():
        if which == "embedding":
            return (token_embedding(tokens, w) * x).sum()
        return linear_token_logprobs(x, w, tokens).logprob.sum()

    def step():
        w.grad = None
        loss().backward()

    step()
    want = w.grad.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    alive = loss()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    got = w.grad
    got.zero_()
    graph.replay()
    assert torch.equal(got, want)
    step()  # and eager passes go on
    assert torch.equal(w.grad, want)
