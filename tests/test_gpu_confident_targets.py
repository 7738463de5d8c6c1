"""GPU: the gradient of tokens that are predicted well.  Their coefficient g (1 - p_t) is small; formed as the difference of g and a rounded
g p_t nothing is left of it.  Tolerances: softmax_tight.py."""
import math

import pytest
import torch

from .softmax_tight import Tight
from .test_gpu_vocab_softmax import BF16, F32, close, make

pytestmark = pytest.mark.gpu
LEFT = [0.5, 0.1, 0.03, 1e-2, 3e-3, 1e-3, 1e-4, 1e-5, 1e-7, 0.9, 0.999]        # 1 - p_t


def confident(n, V, D, dtype, bias, seed=0):
    """Each token's target row points along its x, as far as 1 - p_t asks for."""
    g = torch.Generator().manual_seed(seed + n * 31 + V * 17 + D)
    x = (torch.randn(n, D, generator=g) / math.sqrt(D)).to(dtype).double()
    w = torch.randn(V, D, generator=g).to(dtype).double()
    b = -torch.log(torch.randperm(V, generator=g).double() + 1.5).float().double() if bias else torch.zeros(V, dtype=torch.float64)
    t = torch.randperm(V, generator=g)[:n]
    w[t] *= 0.01
    left = torch.tensor([LEFT[i % len(LEFT)] for i in range(n)], dtype=torch.float64)
    for _ in range(2):                           # (the other targets' rows weigh in)
        s = x @ w.t() + b
        s[torch.arange(n), t] = -math.inf
        want = torch.logsumexp(s, 1) + torch.log1p(-left) - torch.log(left) - b[t]
        w[t] = (x * (want / (x * x).sum(1))[:, None]).to(dtype).double()
    return x.to(dtype).cuda(), w.to(dtype).cuda(), b.float().cuda() if bias else None, t.cuda()


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(1, 40, 50), (44, 600, 50), (130, 4097, 300), (33, 1000, 64), (77, 2000, 128), (40, 700, 200), (64, 1500, 512), (600, 5000, 100)])
def test_gradient_of_confident_tokens(n, V, D, dtype, entropy):
    from sage_amd import vocab_softmax as vs
    for bias in (False, True):
        x, w, b, t = confident(n, V, D, dtype, bias)
        e = Tight(x, w, b, t)
        left = 1 - e.p[torch.arange(n), t]
        assert n < 40 or float(left.min()) < 1e-4 < 0.5 < float(left.max())
        gl = -torch.linspace(0.5, 1.5, n).cuda() / n
        gh = torch.linspace(-1, 1, n).cuda() * 0.1 / n if entropy else None
        f = vs.token_logprobs(x, w, t, bias=b)
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gh)
        (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, gh, dtype)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw")
        if bias:
            close(db, wb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_target_of_many_confident_tokens(dtype):
    """The sum over tokens at one id; tokens without a target and tokens far from theirs between them."""
    from sage_amd import vocab_softmax as vs
    n, V, D = 300, 900, 50
    x, w, _, t = confident(n, V, D, dtype, False, seed=1)
    same = torch.arange(n, device="cuda") % 3 != 0
    x[same] = x[6].clone()
    t = torch.where(same, t[6], t)
    t[::7] = -1
    t[::11] = 5
    e = Tight(x, w, None, t)
    gl = torch.full((n,), -1.0 / n, device="cuda")
    f = vs.token_logprobs(x, w, t)
    dx, dw, _ = vs.token_logprobs_backward(x, w, t, f, gl)
    (wx, tx), (ww, tw), _ = e.gradient(gl, None, dtype)
    close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_certain_and_impossible_targets(dtype):
    """p_t that rounds to 1 and to 0, and a target that the bias takes out beside tokens that are certain."""
    from sage_amd import vocab_softmax as vs
    n, V, D = 40, 300, 32
    g = torch.Generator().manual_seed(3)
    x = torch.randn(n, D, generator=g).to(dtype).cuda()
    w = (torch.randn(V, D, generator=g) * 0.1).to(dtype).cuda()
    t = torch.arange(n, device="cuda") * 7
    w[t[:20]] = (x[:20].double() * 4).to(dtype)              # logits of about 128 over the rest
    w[t[20:30]] = (x[20:30].double() * -4).to(dtype)
    b = torch.zeros(V, device="cuda")
    b[t[30:35]] = float("-inf")
    e = Tight(x, w, b, t)
    gl = torch.linspace(-1, -0.5, n).cuda()
    f = vs.token_logprobs(x, w, t, bias=b)
    dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b)
    (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, None, dtype)
    close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


@pytest.mark.parametrize("n,V,D", [(300, 5000, 50), (64, 1000, 128), (128, 3000, 200), (257, 9000, 300), (100, 700, 512)])
def test_unlikely_targets_of_bf16_are_not_rounded_twice(n, V, D):
    """Tokens with targets of their own that are unlikely: a row of dw is g (1 - p_t) x, to half a step of its type (2^-8), and the other tokens' share, of which
    each weight is rounded once (2^-8).  Of the target's own weight no more than 2^-16 may be lost beside that."""
    from sage_amd import vocab_softmax as vs
    x, w, _, _ = make(n, V, D, BF16, seed=21, scale=0.3)
    t = torch.randperm(V, generator=torch.Generator().manual_seed(n))[:n].cuda()
    e = Tight(x, w, None, t)
    gl = -torch.linspace(0.5, 1.5, n).cuda() / n
    f = vs.token_logprobs(x, w, t)
    _, dw, _ = vs.token_logprobs_backward(x, w, t, f, gl)
    (_, _), (want, _), _ = e.gradient(gl, None, BF16)
    G = e.G.clone()
    own = G[torch.arange(n), t].abs()
    G[torch.arange(n), t] = 0.0
    others = G.abs().t().contiguous() @ e.x.abs()
    inner = torch.zeros_like(want)
    inner[t] = (own * (2.0 ** -16 + e.tol_p.amax(1)))[:, None] * e.x.abs()
    inner = inner + others * (2.0 ** -8 + e.tol_p.max()) + 64 * 2.0 ** -24 * (others + want.abs())
    close(dw, want, inner + 2.0 ** -8 * (want.abs() + inner) + 1e-37, "dw")
