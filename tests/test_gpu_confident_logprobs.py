"""GPU: log probabilities of targets that are predicted well.  log p_t = log(1 - rest), rest the sum of the other ids' probabilities; as a
logit less lse it would have the error of either.  Tolerance where p_t is above 0.55: rest is off by the others' logits and by
lse's, relative (Exact's tolerance of a probability), the logarithm's slope is 1 / p_t < 2, two roundings (u = 2^-24)."""
import pytest
import torch

from .softmax_tight import Tight
from .test_gpu_confident_targets import confident
from .test_gpu_vocab_softmax import BF16, F32, U, check_forward, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(1, 40, 50), (11, 300, 7), (44, 600, 50), (130, 4097, 300), (400, 2000, 128), (44, 60000, 50), (530, 1000, 64), (600, 5000, 100),
                                   (560, 2000, 200), (700, 30000, 300), (520, 1500, 512), (514, 700, 30)])
def test_log_probabilities_near_one(n, V, D, dtype):
    from sage_amd import vocab_softmax as vs
    for bias, k in ((False, 0), (True, 0), (True, 6)):
        x, w, b, t = confident(n, V, D, dtype, bias, seed=k)
        if n > 20:
            t[n // 2], t[n // 3] = -1, V - 1
        e = Tight(x, w, b, t, k)
        f = vs.token_logprobs(x, w, t, bias=b, alternatives=k)
        check_forward(f, e, k)
        rows = torch.nonzero(e.has).view(-1)
        others = e.p.clone()
        others[rows, t[rows]] = 0.0
        rest = others.sum(1)
        near = e.has & (rest < 0.45)
        assert n < 20 or int(near.sum()) > n // 2
        want = torch.log1p(-rest)
        tol = 2 * rest * (e.tol_p - 2 * U * e.finite.abs()).amax(1) + 2 * U * want.abs() + 1e-37
        close(f.logprob[near], want[near], tol[near], f"logprob {bias} {k}")
