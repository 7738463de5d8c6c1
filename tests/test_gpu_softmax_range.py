"""GPU: logits of -inf without a bias in the vocabulary softmax."""
import pytest
import torch

from .test_gpu_vocab_softmax import BF16, F32, Exact, check_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [3, 40, 600])
@pytest.mark.parametrize("beside", [False, True])
def test_logits_of_minus_infinity_without_a_bias(n, dtype, beside):
    """Sums of products of -2 10^38: they pass float32's range, and their ids are out, the last ones or every tenth.  With them alone nothing is left."""
    from sage_amd import vocab_softmax as vs
    V, D, gone = 640, 40, 64
    g = torch.Generator().manual_seed(n)
    x = torch.full((n, D), 1e19, dtype=torch.float64)
    w = torch.randn(V, D, generator=g, dtype=torch.float64) * 1e-20
    out = torch.arange(V) % 10 == 4 if beside else torch.arange(V) >= V - gone
    w[out] = -2e19
    x, w, keep = x.to(dtype).cuda(), w.to(dtype).cuda(), torch.nonzero(~out).view(-1).cuda()
    t = (torch.arange(n) % len(keep)).cuda()
    for k in (0, 5):
        f = vs.token_logprobs(x, w, keep[t], alternatives=k)
        e = Exact(x, w[keep], None, t, k)
        if k:
            e.alt_ids = keep[e.alt_ids]
        check_forward(f, e, k)
    f = vs.token_logprobs(x, w[out.cuda()], t % gone, alternatives=2)
    assert torch.isneginf(f.lse).all() and (f.entropy == 0).all() and torch.isneginf(f.logprob).all() and (f.alt_ids == -1).all()
