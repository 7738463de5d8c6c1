"""GPU: the vocabulary softmax where its kernels change: enough tokens for the weights to be packed first, vocabularies whose
gradient one range of tokens forms (stored without partial sums), row strides of the results, workspaces full of NaN.
Definition and tolerances are those of test_gpu_vocab_softmax.py."""

import pytest
import torch

from .test_gpu_vocab_softmax import BF16, F32, U, Exact, check_forward, close, exact_norm, grads_of, make

pytestmark = pytest.mark.gpu
WIDTHS = [1, 7, 8, 31, 50, 64, 65, 128, 129, 200, 256, 257, 300, 320, 321, 511, 512]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", WIDTHS)
def test_packed_weights(D, dtype):
    from sage_amd import vocab_softmax as vs
    for n, V, bias, k in ((513, 700, "none", 0), (600, 257, "mask", 32), (520, 1300, "prior", 5)):
        x, w, b, t = make(n, V, D, dtype, bias, seed=k)
        check_forward(vs.token_logprobs(x, w, t, bias=b, alternatives=k), Exact(x, w, b, t, k), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [17, 33, 48, 49, 64, 96, 97, 192, 321, 512])
def test_as_many_tokens_as_read_the_weights_as_they_lie(n, dtype):
    from sage_amd import vocab_softmax as vs
    for V, D, k in ((33, 50, 3), (9000, 50, 3), (1200, 300, 9), (5000, 511, 2)):
        x, w, b, t = make(n, V, D, dtype, "prior", seed=k)
        check_forward(vs.token_logprobs(x, w, t, bias=b, alternatives=k), Exact(x, w, b, t, k), k)


@pytest.mark.parametrize("low", [float("-inf"), -1e30])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_masks_and_empty_rows(dtype, low):
    from sage_amd import vocab_softmax as vs
    for V in (1, 70, 500):
        x, w, _, _ = make(530, V, 40, dtype)
        t = torch.arange(530, device="cuda") % V
        for m in (torch.ones(V, dtype=torch.bool), torch.arange(V) != V - 1, torch.arange(V) < min(V - 1, 64)):
            b = torch.where(m, low, 0.5).float().cuda()
            e = Exact(x, w, b, t, 5)
            f = vs.token_logprobs(x, w, t, bias=b, alternatives=5)
            check_forward(f, e, 5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_ties_and_bad_rows(dtype):
    from sage_amd import vocab_softmax as vs
    x, w, _, t = make(540, 3000, 24, dtype)
    w[1000:2000] = w[:1000]
    x[3] = x[539] = 0
    clean = vs.token_logprobs(x, w, t, alternatives=32)
    check_forward(clean, Exact(x, w, None, t, 32), 32)
    bad = x.clone()
    bad[7, 3], bad[500, 20] = float("nan"), float("inf")
    f = vs.token_logprobs(bad, w, t, alternatives=32)
    rows = torch.ones(540, dtype=torch.bool, device="cuda")
    rows[[7, 500]] = False
    for a, c in zip(f, clean):
        assert torch.equal(a[rows], c[rows])
    assert torch.isnan(f.lse[~rows]).all() and (f.alt_ids[~rows] == -1).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(70, 70001, 50), (33, 40003, 100), (129, 40003, 200), (5, 40003, 300), (64, 33001, 511), (1, 100000, 7)])
def test_gradient_of_a_long_vocabulary(n, V, D, dtype):
    from sage_amd import vocab_softmax as vs
    for bias, entropy in (("none", False), ("mask", True)):
        x, w, b, t = make(n, V, D, dtype, bias, seed=3)
        t[: n // 2] = V - 1                          # one target many times
        gl = torch.linspace(-1, 0.5, n).cuda()
        gh = torch.linspace(0.3, -0.2, n).cuda() if entropy else None
        f = vs.token_logprobs(x, w, t, bias=b)
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gh)
        (wx, tx), (ww, tw), (wb, tb) = Exact(x, w, b, t).gradient(gl, gh, dtype)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw")
        if db is not None:
            close(db, wb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(40, 900, 33), (40, 70001, 33), (530, 257, 130)])
def test_results_between_other_data(n, V, D, dtype):
    """The C-ABI with row strides of its own, some results left out, and a workspace that holds NaN."""
    from sage_amd import vocab_softmax as vs
    from sage_amd.parallel import get_engine
    eng, kind = get_engine(), 0 if dtype == F32 else 1
    x, w, b, t = make(n, V, D, dtype, "prior", seed=1)
    gl = torch.linspace(-1, 1, n).cuda()
    f = vs.token_logprobs(x, w, t, bias=b)
    want = vs.token_logprobs_backward(x, w, t, f, gl, bias=b)
    st = torch.cuda.current_stream().cuda_stream
    need = eng.token_logprobs_backward_workspace(kind, n, V, D)
    for parts in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 1, 1)):
        ws = torch.full((need // 4 + 64,), float("nan"), device="cuda")
        dx, dw = torch.full((n + 2, D + 5), 7.0, dtype=dtype, device="cuda"), torch.full((V + 2, D + 3), 7.0, dtype=dtype, device="cuda")
        db = torch.full((V + 2,), 7.0, device="cuda")
        eng.token_logprobs_backward_device(kind, n, V, D, x.data_ptr(), D, w.data_ptr(), D, b.data_ptr(), t.data_ptr(), f.lse.data_ptr(), f.entropy.data_ptr(),
                                           gl.data_ptr(), 0, dx[1:, 1:].data_ptr() if parts[0] else 0, D + 5, dw[1:, 1:].data_ptr() if parts[1] else 0, D + 3,
                                           db[1:].data_ptr() if parts[2] else 0, ws.data_ptr(), need, st)
        for got, ref, on in ((dx, want[0], parts[0]), (dw, want[1], parts[1])):
            keep = torch.full_like(got, 7.0)
            if on:
                keep[1:-1, 1:D + 1] = ref
            assert torch.equal(got, keep)
        assert torch.equal(db, torch.cat([db[:1] * 0 + 7, want[2], db[:1] * 0 + 7]) if parts[2] else torch.full_like(db, 7.0))
        assert torch.isnan(ws[(need + 3) // 4:]).all()
    # the forward call, with neither logprob nor entropy, and with alternatives
    for k in (0, 4):
        need = eng.token_logprobs_workspace(kind, n, V, D, k)
        ws = torch.full((need // 4 + 64,), float("nan"), device="cuda")
        lse, ids, lp = torch.full((n + 1,), 7.0, device="cuda"), torch.full((n * k + 1,), 7, dtype=torch.int32, device="cuda"), torch.full((n * k + 1,), 7.0, device="cuda")
        eng.token_logprobs_device(kind, n, V, D, x.data_ptr(), D, w.data_ptr(), D, b.data_ptr(), 0, k, 0, 0, lse.data_ptr(), ids.data_ptr(), lp.data_ptr(),
                                  ws.data_ptr(), need, st)
        ref = vs.token_logprobs(x, w, bias=b, alternatives=k)
        assert torch.equal(lse[:-1], ref.lse) and lse[-1] == 7 and ids[-1] == 7 and lp[-1] == 7
        if k:
            assert torch.equal(ids[:-1].view(n, k), ref.alt_ids) and torch.equal(lp[:-1].view(n, k), ref.alt_logprobs)
        assert torch.isnan(ws[(need + 3) // 4:]).all()


def test_the_two_calls_at_once():
    """Two streams, each with its own tensors and workspace."""
    from sage_amd import vocab_softmax as vs
    sides = [torch.cuda.Stream() for _ in range(2)]
    args = [make(600, 9000, 50, F32, "prior", seed=s) for s in range(2)]
    gl = torch.ones(600, device="cuda")

    def run(x, w, b, t):
        f = vs.token_logprobs(x, w, t, bias=b, alternatives=3)
        return (*f, *vs.token_logprobs_backward(x, w, t, f, gl, bias=b))
    want = [run(*a) for a in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                got[i].append(run(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, c) for result in got[i] for a, c in zip(result, want[i]))


@pytest.mark.parametrize("sizes", [[0], [0, 0], [1] * 128, [1] * 129, [256] * 128, [257] * 128, [32768], [32767, 1], [32767, 2], [1 << 22], [(1 << 22) + 1],
                                   [8191, 8192, 8193, 1 << 23]])
def test_clip_where_the_kernels_change(sizes):
    from sage_amd import vocab_softmax as vs
    for kinds in ([F32] * len(sizes), [BF16, F32] * len(sizes)):
        grads = grads_of(sizes, kinds)
        before, want = [t.clone() for t in grads], exact_norm(grads)
        limit = want * 0.3
        assert abs(float(vs.clip_grad_norm(grads, limit)) - want) <= 2.0 ** -23 * want
        for t, o in zip(before, grads):
            d = t.double() * (limit / want if want else 1.0)
            close(o, d, d.abs() * (torch.finfo(t.dtype).eps / 2 + 3 * 2.0 ** -24) + 1e-37, "clipped")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(3, 700, 50), (40, 20000, 50), (3, 700, 511), (530, 900, 50), (530, 900, 300), (530, 900, 512)])
def test_what_masked_rows_hold_does_not_matter(n, V, D, dtype):
    """The weights of masked ids: NaN, infinities and the type's largest values; targets among them."""
    from sage_amd import vocab_softmax as vs
    for low in (float("-inf"), -1e30):
        x, w, _, t = make(n, V, D, dtype, seed=4)
        g = torch.Generator().manual_seed(8)
        gone = torch.rand(V, generator=g) < 0.3
        gone[32:96] = True
        b = torch.where(gone, low, 0.25).float().cuda()
        clean, dirty = w.clone(), w.clone()
        clean[gone.cuda()] = 0
        for i, v in enumerate((float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).max)):
            dirty[torch.nonzero(gone).view(-1)[i::4].cuda()] = v
        ref = vs.token_logprobs(x, clean, t, bias=b, alternatives=6)
        e = Exact(x, clean, b, t, 6)
        check_forward(ref, e, 6)
        got = vs.token_logprobs(x, dirty, t, bias=b, alternatives=6)
        for a, c in zip(got, ref):
            assert torch.equal(a, c)
        t2 = torch.where(gone.cuda()[t.clamp(min=0)], -1, t)          # (the gradient of a masked target asks for its row)
        gl = torch.linspace(-1, 1, n).cuda()
        for a, c in zip(vs.token_logprobs_backward(x, dirty, t2, got, gl, bias=b, grad_entropy=gl), vs.token_logprobs_backward(x, clean, t2, ref, gl, bias=b, grad_entropy=gl)):
            assert torch.isfinite(a).all() and torch.equal(a, c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [50, 300])
def test_what_idle_tokens_hold_does_not_matter(D, dtype):
    """A padded batch: the rows without a target hold NaN, infinities and large values."""
    from sage_amd import vocab_softmax as vs
    n, V = 200, 1500
    x, w, b, t = make(n, V, D, dtype, "prior", seed=2)
    idle = torch.arange(n, device="cuda") % 3 == 1
    t[:] = torch.where(idle, -1, t.clamp(min=0))
    dirty = x.clone()
    for i, v in enumerate((float("nan"), float("inf"), torch.finfo(dtype).max)):
        dirty[torch.nonzero(idle).view(-1)[i::3]] = v
    clean = x.clone()
    clean[idle] = 0
    gl = torch.linspace(-1, 1, n).cuda() + 0.003
    gh = torch.where(idle, 0.0, gl)
    f, ref = vs.token_logprobs(dirty, w, t, bias=b), vs.token_logprobs(clean, w, t, bias=b)
    assert torch.equal(f.logprob, ref.logprob) and torch.equal(f.lse[~idle], ref.lse[~idle])
    for h in (None, gh):
        got, want = (vs.token_logprobs_backward(x, w, t, r, gl, bias=b, grad_entropy=h) for x, r in ((dirty, f), (clean, ref)))
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        assert (got[0][idle] == 0).all()
        (wx, tx), (ww, tw), (wb, tb) = Exact(clean, w, b, t).gradient(gl, h, dtype)
        close(got[0], wx, tx, "dx"), close(got[1], ww, tw, "dw"), close(got[2], wb, tb, "db")


def test_logits_far_from_zero():
    """Beyond float16, in which the largest logits of a chunk are kept; and so far that all of them look alike there."""
    from sage_amd import vocab_softmax as vs
    for n in (5, 530):
        x, w, _, t = make(n, 4000, 50, F32, seed=6)
        for shift in (300.0, -5000.0, 2e5, -2e5, 3e6):
            b = torch.full((4000,), shift, device="cuda")
            b[::5] = float("-inf")
            e = Exact(x, w, b, t, 7)
            f = vs.token_logprobs(x, w, t, bias=b, alternatives=7)
            check_forward(f, e, 7)
            b[7:] = float("-inf")                    # six ids are left
            check_forward(vs.token_logprobs(x, w, t, bias=b, alternatives=7), Exact(x, w, b, t, 7), 7)


@pytest.mark.parametrize("n,D,dtype", [(3, 512, BF16), (530, 300, BF16), (2, 512, F32), (40, 7, F32)])
def test_the_largest_vocabulary(n, D, dtype):
    from sage_amd import vocab_softmax as vs
    V = 1 << 20
    x, w, b, t = make(n, V, D, dtype, "mask", seed=9)
    t[0] = V - 1
    b[V - 1] = 0.0
    w[V - 1] = x[0] / x[0].float().norm() * 8            # the last id is the first row's most likely one, or nearly so
    f = vs.token_logprobs(x, w, t, bias=b, alternatives=12)
    check_forward(f, Exact(x, w, b, t, 12), 12)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_of_the_largest_vocabulary(dtype):
    from sage_amd import vocab_softmax as vs
    n, V, D = 20, 1 << 20, 65
    x, w, b, t = make(n, V, D, dtype, "prior", seed=9)
    t[0] = V - 1
    gl = torch.linspace(-1, 1, n).cuda()
    f = vs.token_logprobs(x, w, t, bias=b)
    dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b)
    (wx, tx), (ww, tw), (wb, tb) = Exact(x, w, b, t).gradient(gl, None, dtype)
    close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


def test_the_most_tokens():
    from sage_amd import vocab_softmax as vs
    n = 1 << 22
    x, w, _, t = make(n, 3, 2, F32, seed=1)
    e = Exact(x, w, None, t, 2)
    f = vs.token_logprobs(x, w, t, alternatives=2)
    close(f.lse, e.lse, e.tol_lse, "lse"), close(f.logprob, e.logprob, e.tol_lse + U * e.logprob.abs(), "logprob")
    assert torch.equal(f.alt_ids.long(), e.alt_ids)
    gl = torch.full((n,), 1.0 / n, device="cuda")
    dx, dw, _ = vs.token_logprobs_backward(x, w, t, f, gl)
    (wx, tx), (ww, tw), _ = e.gradient(gl, None, F32)
    close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw")
    with pytest.raises(ValueError, match="2\\^22"):
        vs.token_logprobs(torch.zeros(n + 1, 2, device="cuda"), w)
