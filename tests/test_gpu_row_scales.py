"""GPU: float32 rows of very different sizes beside each other where the rows are packed (more than 512 tokens, and in every gradient).
A row's result is its own, whatever its neighbours hold.  Tolerances: softmax_tight.py; ids whose logit is far below every
other are left out of the definition, so that its tolerances are those of the ids that count."""
import pytest
import torch

from .softmax_tight import Tight
from .test_gpu_vocab_softmax import BF16, F32, U, close, make

pytestmark = pytest.mark.gpu


def rows_agree(f, e, rows, k):
    close(f.lse[rows], e.lse[rows], e.tol_lse[rows], "lse")
    close(f.entropy[rows], e.H[rows], e.tol_H[rows], "entropy")
    close(f.logprob[rows], e.logprob[rows], (e.tol_lse + U * e.logprob.abs())[rows], "logprob")
    if k:
        assert torch.equal(f.alt_ids.long()[rows], e.alt_ids[rows])
        lp = e.alt_logprobs[rows]
        close(f.alt_logprobs[rows], lp, e.tol_lse[rows, None] + U * lp.abs(), "alternatives")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e4, 1e7, 1e9, 1e12, 1e30, float("inf")])
def test_a_large_token_beside_others(size, dtype):
    """One token in 32 is `size` times the others (inf: the type's largest value throughout, as a padded position may hold), and has no target."""
    from sage_amd import vocab_softmax as vs
    n, V, D, k = 640, 900, 50, 10
    x, w, b, t = make(n, V, D, dtype, "prior", seed=11)
    large = torch.arange(n, device="cuda") % 32 == 5
    t = torch.where(large, -1, t)
    clean = x.clone()
    x[large] = (x[large].double() * size).to(dtype) if size < 1e31 else torch.finfo(dtype).max
    e = Tight(clean, w, b, t, k)
    f = vs.token_logprobs(x, w, t, bias=b, alternatives=k)
    rows_agree(f, e, ~large, k)
    alone = vs.token_logprobs(clean, w, t, bias=b, alternatives=k)
    for a, c in zip(f, alone):
        assert torch.equal(a[~large], c[~large])             # bit for bit


@pytest.mark.parametrize("small, large", [(1e-6, 1e4), (1e-6, 1e5), (1.0, 1e8)])
def test_alternatives_of_small_tokens(small, large):
    from sage_amd import vocab_softmax as vs
    n, V, D, k = 576, 4000, 50, 5
    x, w, _, t = make(n, V, D, F32, seed=12)
    x *= small
    x[::32] *= large / small
    e = Tight(x, w, None, t, k)
    rows_agree(vs.token_logprobs(x, w, t, alternatives=k), e, torch.ones(n, dtype=torch.bool, device="cuda"), k)


@pytest.mark.parametrize("n", [40, 600])
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e20, -1e30])
def test_ids_that_their_weights_take_out(n, low):
    """The last element of x is 1, that of the weights an id's bias: `low` for one id in 8."""
    from sage_amd import vocab_softmax as vs
    V, D, k = 800, 50, 6
    x, w, _, _ = make(n, V, D, F32, seed=13)
    g = torch.Generator().manual_seed(2)
    x[:, -1] = 1.0
    out = torch.arange(V, device="cuda") % 8 == 3
    keep = torch.nonzero(~out).view(-1)
    t = torch.randint(-1, len(keep), (n,), generator=g).cuda()
    w[:, -1] = torch.where(out, low, 0.25)
    ids = torch.where(t >= 0, keep[t.clamp(min=0)], -1)
    e = Tight(x, w[keep], None, t, k)
    f = vs.token_logprobs(x, w, ids, alternatives=k)
    e.alt_ids = keep[e.alt_ids]
    rows_agree(f, e, torch.ones(n, dtype=torch.bool, device="cuda"), k)
    gl, gh = torch.linspace(-1, 1, n).cuda() / n, torch.linspace(0.5, -0.5, n).cuda() / n
    for h in (None, gh):
        dx, dw, _ = vs.token_logprobs_backward(x, w, ids, f, gl, grad_entropy=h)
        (wx, tx), (ww, tw), _ = e.gradient(gl, h, F32)
        close(dx, wx, tx, "dx"), close(dw[keep], ww, tw, "dw")
        assert (dw[out] == 0).all()


@pytest.mark.parametrize("n, V, D", [(640, 300, 50), (96, 1100, 300), (200, 700, 200), (64, 400, 512), (70, 300, 100)])
@pytest.mark.parametrize("size", [300.0, 1e5, 1e9])
def test_gradient_of_tokens_of_different_sizes(n, V, D, size):
    """A token `size` times the others, with a gradient as much smaller: it weighs as much in dw as the others, and they keep their bits.
    (It lies where the weights are 0: its logits are the bias, exactly.)"""
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(n, V, D, F32, "prior", seed=14)
    large, tail = torch.arange(n, device="cuda") % 32 == 9, D // 5
    x[large, :-tail] = 0.0
    x[large] *= size
    w[:, -tail:] = 0.0
    w[::16] = 0.0                                            # ids that no step has reached yet
    gl = torch.linspace(-1, 1.01, n).cuda()
    gl[large] /= size
    gh = gl.flip(0) * 0.2
    gh[large] = gl[large] * 0.1
    e = Tight(x, w, b, t)
    f = vs.token_logprobs(x, w, t, bias=b)
    for h in (None, gh):
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=h)
        (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, h, F32)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


@pytest.mark.parametrize("n, V, D", [(640, 600, 50), (96, 1100, 300), (200, 700, 200), (64, 400, 512)])
def test_weights_of_a_first_step(n, V, D):
    """Rows that a few steps have reached beside rows that hold what is left of their probability, 10^5 times smaller, and beside zeros."""
    from sage_amd import vocab_softmax as vs
    x, w, _, t = make(n, V, D, F32, seed=15)
    g = torch.Generator().manual_seed(5)
    size = torch.tensor([1.0, 1e-5, 0.0, 3e-6])[torch.randint(0, 4, (V,), generator=g)].cuda()
    w *= size[:, None]
    e = Tight(x, w, None, t, 8)
    f = vs.token_logprobs(x, w, t)
    gl = torch.full((n,), 1.0, device="cuda")
    for h in (None, gl * 0.1):
        dx, dw, _ = vs.token_logprobs_backward(x, w, t, f, gl, grad_entropy=h)
        (wx, tx), (ww, tw), _ = e.gradient(gl, h, F32)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw")
