"""token_logprobs where several blocks share a row and meet in the first one's shared memory.

The blocks of a row may start at different times when the GPU is busy; what they send must
not depend on it.  Bounds: logprob and entropy are sums of V terms in fp32.
"""

import pytest
import torch

from dense_utils import within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [5000, 9001, 20000, 131072])  # 2, 4 and 8 blocks a row
@pytest.mark.parametrize("rows", [1, 7, 18])
@pytest.mark.parametrize("top_n", [0, 20])
def test_blocks_of_a_row_on_a_busy_gpu(V, rows, top_n, cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(V + rows)
    x = torch.randn(rows, V, device=cuda_device, generator=g) * 2.5
    tokens = torch.randint(0, V, (rows,), device=cuda_device, generator=g)
    logp = torch.log_softmax(x.double(), -1)
    want = logp.gather(-1, tokens[:, None])[:, 0]
    entropy = torch.special.entr(logp.exp()).sum(-1)
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :top_n]
    busy, side = torch.randn(3000, 3000, device=cuda_device), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy * 0.5 + busy.T
    runs = [token_logprobs(x, tokens, top_n=top_n) for _ in range(30)]
    torch.cuda.synchronize()
    for r in runs:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
    # exponentials to 2^-19 each, sums of V terms, and the rounding of values of size |x| + log V
    off = 2.0 ** -19 * (1 + x.double().abs().amax(-1) + torch.log(torch.tensor(float(V))))
    within(runs[0].logprob, want, off, "logprob")
    within(runs[0].entropy, entropy, off, "entropy")
    assert torch.equal(runs[0].top_tokens, order)
