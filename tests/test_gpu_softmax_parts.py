"""GPU: the gradient's results asked for one by one are those of the call for all of them, bit for bit, at every width's kernels; with
tokens that have a target and no gradient of it, targets and no entropy gradient, neither, and rows of different sizes."""
import pytest
import torch

from .softmax_tight import Tight
from .test_gpu_vocab_softmax import BF16, F32, close, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(70, 900, 50), (129, 2000, 100), (64, 3000, 200), (100, 1111, 300), (65, 700, 512), (33, 70001, 320)])
def test_results_one_by_one(n, V, D, dtype, entropy):
    from sage_amd import vocab_softmax as vs
    from sage_amd.parallel import get_engine
    eng, kind = get_engine(), 0 if dtype == F32 else 1
    x, w, b, t = make(n, V, D, dtype, "mask", seed=31)
    t = torch.where(torch.isneginf(b[t.clamp(min=0)]), -1, t)
    x[3::16] *= 2000.0
    x[3::16, 5:] = 0.0
    w[:, :5] *= 1e-4
    w[7::64] *= 1e-4
    t[: n // 4] = torch.nonzero(torch.isfinite(b)).view(-1)[3]           # one target of many
    gl = torch.linspace(-1, 1, n).cuda()
    gl[1::5] = 0.0
    gh = torch.linspace(0.5, -0.4, n).cuda() if entropy else None
    if entropy:
        gh[2::7] = 0.0
    f = vs.token_logprobs(x, w, t, bias=b)
    want = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gh)
    for got, (ref, tol), what in zip(want, Tight(x, w, b, t).gradient(gl, gh, dtype), ("dx", "dw", "db")):
        close(got, ref, tol, what)
    need = eng.token_logprobs_backward_workspace(kind, n, V, D)
    ws = torch.full((need // 4 + 64,), float("nan"), device="cuda")
    at = lambda q: 0 if q is None else q.data_ptr()
    for parts in ((1, 0, 0), (0, 1, 0), (0, 1, 1), (1, 1, 0)):
        out = [torch.full_like(r, 7.0) if on else None for r, on in zip(want, parts)]
        ws.fill_(float("nan"))
        eng.token_logprobs_backward_device(kind, n, V, D, at(x), D, at(w), D, at(b), at(t), at(f.lse), at(f.entropy), at(gl), at(gh),
                                           at(out[0]), D, at(out[1]), D, at(out[2]), at(ws), need, torch.cuda.current_stream().cuda_stream)
        for got, ref in zip(out, want):
            assert got is None or torch.equal(got, ref), parts
    assert torch.isnan(ws[(need + 3) // 4:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_entropy_gradient_beside_targets_without_one(dtype):
    """grad_logprob is None, the targets are given nevertheless: they have no part."""
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(90, 1000, 64, dtype, "prior", seed=32)
    gh = torch.linspace(-1, 1, 90).cuda()
    f = vs.token_logprobs(x, w, t, bias=b)
    e = Tight(x, w, b, torch.full_like(t, -1))
    for targets in (t, None):
        got = vs.token_logprobs_backward(x, w, targets, f, None, bias=b, grad_entropy=gh)
        for value, (ref, tol), what in zip(got, e.gradient(None, gh, dtype), ("dx", "dw", "db")):
            close(value, ref, tol, what)
