"""GPU: the vocabulary softmax, its gradient and gradient clipping (sage_amd.vocab_softmax, include/sage_hip.h) against
plain float64 implementations.

Tolerances, with u = 2^-24 (half a float32 step) and D, V, n the lengths summed over:
  a logit          2 (D + 8) u B, B = max_v sum_d |x_d w_vd| + |b_v|: D products summed in any order, twice that because the
                   order and the rounding inside a matrix instruction are its own
  a sum of N terms of any sign, relative to the sum of their sizes: 8 sqrt(N) u (N independent roundings of at most u; 8
                   standard deviations), and 16 u for the exponential, its argument and the final logarithm
  lse              the logit's + the sum's over V + 4 u |lse|
  p                the logit's and lse's together, and u times the exponent's size, relative
  entropy          the derivative of H by the logits is p (log p + H): (1 + H) times twice lse's tolerance
  gradients        |G|'s error as an [n, V] matrix, taken through |w| or |x|, plus the sum's, plus half a step of the result's type;
                   bf16 inputs round G to bf16 before the second product: 2^-8 |G| more.
                   float32 products (where the weights are packed first, and in all gradients) take an element as two float16 of a value
                   scaled by a power of two, so that the largest of its 32 rows, m, lies in [2^12, 2^13): an element is off by
                   at most 2^-25 of that scale (half a step of the smallest float16), 2^-25 / 2^12 m = 2^-37 m, beside its
                   relative 2^-22; a weight likewise by 2^-25 of a scale in which the largest weight of its column times m
                   has come to at least 2^12: 2^-37 of the largest |G| m, times an element that may be m.  Each of the
                   N terms of a sum is thus off by at most 2^-36 of the largest |G| times the largest element, absolutely:
                   N 2^-36 max|G| max|w| more (it shows only where a sum is one term with an element 10^-7 of m)"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def make(n, V, D, dtype, bias="none", seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + V * 17 + D)
    x = torch.randn(n, D, generator=g).to(dtype).cuda()
    w = (torch.randn(V, D, generator=g) * (scale / math.sqrt(D))).to(dtype).cuda()
    b = None
    if bias == "prior":
        b = -torch.log(torch.randperm(V, generator=g).float() + 1.5).cuda()
    elif bias == "mask":
        b = torch.where(torch.rand(V, generator=g) < 0.4, float("-inf"), 0.3).float().cuda()
    t = torch.randint(-1, V, (n,), generator=g).cuda()
    return x, w, b, t


class Exact:
    """The operator's definition in float64, and the tolerances above."""

    def __init__(self, x, w, b, t, k=0):
        self.x, self.w, self.t = x.double(), w.double(), t
        n, V = x.shape[0], w.shape[0]
        D = x.shape[1]
        bias = torch.zeros(V, dtype=torch.float64, device=x.device) if b is None else torch.where(b <= -1e30, float("-inf"), b.double())
        self.s = self.x @ self.w.t().contiguous() + bias
        self.lse = torch.logsumexp(self.s, 1)
        self.logp = self.s - self.lse[:, None]
        self.empty = torch.isneginf(self.lse)
        self.p = torch.where(torch.isneginf(self.s), 0.0, torch.exp(self.logp))
        self.finite = torch.where(self.p > 0, self.logp, 0.0)
        self.H = -(self.p * self.finite).sum(1)
        self.has = t >= 0
        got = self.logp.gather(1, t.clamp(min=0)[:, None])[:, 0]
        self.logprob = torch.where(self.has, torch.where(self.empty, float("-inf"), got), 0.0)
        size = (self.x.abs() @ self.w.abs().t().contiguous() + torch.where(torch.isinf(bias), 0.0, bias.abs())).amax(1) if V else 0
        logit = 2 * (D + 8) * U * size
        lse = torch.where(self.empty, 0.0, self.lse)
        self.tol_lse = logit + (8 * math.sqrt(V) + 16) * U + 4 * U * lse.abs()
        self.tol_p = (logit + self.tol_lse + 8 * U)[:, None] + 2 * U * self.finite.abs()
        self.tol_H = (1 + self.H) * 2 * self.tol_lse
        if k:
            m = min(k, V)
            order = torch.sort(self.s, dim=1, descending=True, stable=True)
            gone = torch.isneginf(order.values[:, :m])
            ids = torch.where(gone, -1, order.indices[:, :m])
            lp = torch.where(gone, float("-inf"), order.values[:, :m] - lse[:, None])
            self.alt_ids = torch.cat([ids, torch.full((n, k - m), -1, device=x.device, dtype=ids.dtype)], 1)
            self.alt_logprobs = torch.cat([lp, torch.full((n, k - m), float("-inf"), device=x.device, dtype=lp.dtype)], 1)

    def gradient(self, g, h, dtype):
        """-> ((dx, tolerance), (dw, tolerance), (db, tolerance))"""
        n, V = self.s.shape
        g = torch.zeros(n, dtype=torch.float64, device=self.s.device) if g is None else torch.where(self.has, g.double(), 0.0)
        hd = torch.zeros_like(g) if h is None else torch.where(self.empty, 0.0, h.double())
        coefficient = g[:, None] + hd[:, None] * (self.finite + self.H[:, None])
        G = -self.p * coefficient
        err = self.p * (self.tol_p * (g.abs()[:, None] + hd.abs()[:, None] * (self.finite.abs() + self.H[:, None])) +
                        hd.abs()[:, None] * (self.tol_lse + self.tol_H)[:, None] + 4 * U * coefficient.abs())
        if self.has.any():
            rows = torch.nonzero(self.has).view(-1)
            G[rows, self.t[rows]] += g[rows]
            err[rows, self.t[rows]] += 2 * U * g[rows].abs()
        half = 0.0 if dtype == F32 else 2.0 ** -8
        mass = self.p * (g.abs()[:, None] + hd.abs()[:, None] * (self.finite.abs() + self.H[:, None]))
        if self.has.any():
            mass[rows, self.t[rows]] += g[rows].abs()
        err = err + half * mass
        step = torch.finfo(dtype).eps / 2

        def through(a, size, other, length):
            value = a @ other
            m = mass if a is G else mass.t().contiguous()
            tol = size @ other.abs() + (8 * math.sqrt(length) + 16) * U * m @ other.abs()
            if dtype == F32:
                tol = tol + length * 2.0 ** -36 * m.amax(1, keepdim=True) * other.abs().max()
            return value, tol + step * value.abs() * (1 + step) + step * tol + 1e-37
        Gt, et = G.t().contiguous(), err.t().contiguous()
        ones = torch.ones(n, 1, dtype=torch.float64, device=G.device)
        # (the bias's gradient is float32 and sums G before it is rounded to bf16)
        err32 = (err - half * mass).t().contiguous()
        db = Gt @ ones
        tdb = err32 @ ones + (8 * math.sqrt(n) + 16) * U * (mass.t().contiguous() @ ones) + 2 * U * db.abs() + 1e-37
        return through(G, err, self.w, V), through(Gt, et, self.x, n), (db[:, 0], tdb[:, 0])


def close(got, want, tol, what):
    got = got.double()
    same = (got == want) | ((got - want).abs() <= tol)
    bad = torch.nonzero(~same)
    assert not len(bad), f"{what}: {len(bad)} of {got.numel()} off, first at {bad[0].tolist()}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}, tolerance {tol[tuple(bad[0])]}"


def check_forward(f, e, k=0):
    close(f.lse, e.lse, e.tol_lse, "lse")
    close(f.entropy, torch.where(e.empty, 0.0, e.H), e.tol_H, "entropy")
    close(f.logprob, e.logprob, e.tol_lse + U * torch.where(torch.isinf(e.logprob), 0.0, e.logprob).abs(), "logprob")
    if k:
        assert torch.equal(f.alt_ids.long(), e.alt_ids)
        lp = torch.where(torch.isinf(e.alt_logprobs), 0.0, e.alt_logprobs)
        close(f.alt_logprobs, e.alt_logprobs, e.tol_lse[:, None] + U * lp.abs(), "alternatives")


SHAPES = [(1, 1, 1), (1, 2, 3), (2, 63, 50), (15, 64, 64), (17, 65, 65), (33, 127, 31), (65, 129, 128), (5, 1000, 129), (129, 1200, 50),
          (300, 4097, 200), (64, 640, 256), (31, 333, 257), (40, 2049, 300), (16, 511, 320), (130, 257, 321), (7, 5000, 511), (257, 770, 512)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", SHAPES)
def test_logprobs(n, V, D, dtype):
    from sage_amd import vocab_softmax as vs
    for bias, k in (("none", 0), ("prior", 1), ("mask", 10), ("none", 32)):
        x, w, b, t = make(n, V, D, dtype, bias, seed=k)
        check_forward(vs.token_logprobs(x, w, t, bias=b, alternatives=k), Exact(x, w, b, t, k), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", SHAPES)
def test_gradient(n, V, D, dtype):
    from sage_amd import vocab_softmax as vs
    for bias, entropy in (("none", False), ("prior", True), ("mask", True)):
        x, w, b, t = make(n, V, D, dtype, bias, seed=5)
        g = torch.Generator().manual_seed(V)
        gl = torch.randn(n, generator=g).cuda() / n
        gh = (torch.randn(n, generator=g).cuda() / n) if entropy else None
        f = vs.token_logprobs(x, w, t, bias=b)
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gh)
        e = Exact(x, w, b, t)
        (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, gh, dtype)
        assert dx.dtype == dtype and dw.dtype == dtype and (db is None) == (b is None)
        close(dx, wx, tx, f"dx {bias}")
        close(dw, ww, tw, f"dw {bias}")
        if db is not None:
            close(db, wb, tb, "db")


@pytest.mark.parametrize("n,V,D,dtype", [(1, 262144, 50, F32), (3, 131073, 300, BF16), (700, 70001, 50, F32), (513, 33000, 100, BF16)])
def test_long_vocabulary(n, V, D, dtype):
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(n, V, D, dtype, "prior")
    e = Exact(x, w, b, t, 10)
    check_forward(vs.token_logprobs(x, w, t, bias=b, alternatives=10), e, 10)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [3, 4, 7, 8, 50, 64, 65, 129, 200, 257, 300, 385, 511, 512])
def test_one_to_seventeen_tokens(D, dtype):
    """The kernel that reads the weights as they lie takes up to sixteen tokens, 1, 2, 4 or 8 at a time."""
    from sage_amd import vocab_softmax as vs
    for n in (1, 2, 3, 4, 5, 8, 9, 13, 16, 17):
        x, w, b, t = make(n, 300, D, dtype, ("none", "prior", "mask")[n % 3])
        check_forward(vs.token_logprobs(x, w, t, bias=b, alternatives=n), Exact(x, w, b, t, n), n)


def test_many_rows_cross_a_pass():
    """More rows than one pass of the forward kernels takes."""
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(16384 + 77, 300, 20, F32, "prior")
    e = Exact(x, w, b, t, 3)
    f = vs.token_logprobs(x, w, t, bias=b, alternatives=3)
    check_forward(f, e, 3)
    g = torch.full((x.shape[0],), -1.0 / x.shape[0], device="cuda")
    dx, dw, db = vs.token_logprobs_backward(x, w, t, f, g, bias=b)
    (wx, tx), (ww, tw), (wb, tb) = e.gradient(g, None, F32)
    close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


def test_gradient_against_differences():
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(6, 41, 9, F32, "prior", seed=3)
    gl, gh = torch.linspace(-1, 1, 6).cuda(), torch.linspace(0.5, -0.5, 6).cuda()
    f = vs.token_logprobs(x, w, t, bias=b)
    got = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gh)

    def loss(x, w, b):
        s = x @ w.t() + b
        logp = torch.log_softmax(s, 1)
        lp = torch.where(t >= 0, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
        return (gl.double() * lp - gh.double() * (logp.exp() * logp).sum(1)).sum()
    args = [x.double(), w.double(), b.double()]
    tol = [m for _, m in Exact(x, w, b, t).gradient(gl, gh, F32)]
    for i, (grad, m) in enumerate(zip(got, tol)):
        for at in ((0, 0), (3, 5), (5, 8), (2, 1)) if i < 2 else ((0,), (17,), (40,)):
            step = torch.zeros_like(args[i])
            step[at] = 1e-4
            up, down = [a + step if j == i else a for j, a in enumerate(args)], [a - step if j == i else a for j, a in enumerate(args)]
            slope = float(loss(*up) - loss(*down)) / 2e-4
            # (the third derivative times step^2 / 6: logits of size 10, x and w of size 3 -> below 1e3 * 1e-8 / 6)
            assert abs(float(grad[at]) - slope) <= float(m[at]) + 2e-6, (i, at, float(grad[at]), slope)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(dtype):
    """Rows inside wider ones, starting at any element; x and weight views of one tensor."""
    from sage_amd import vocab_softmax as vs
    g = torch.Generator().manual_seed(9)
    big = (torch.randn(900, 131, generator=g) * 0.3).to(dtype).cuda()
    for lo, D in ((0, 50), (1, 64), (3, 128), (7, 33)):
        x, w = big[3:200:2, lo:lo + D], big[201:, lo:lo + D]
        b = torch.linspace(-1, 1, 2 * w.shape[0]).cuda()[::2]
        t = torch.arange(x.shape[0], device="cuda").int() * 3
        f = vs.token_logprobs(x, w, t, bias=b, alternatives=4)
        e = Exact(x, w, b, t.long(), 4)
        check_forward(f, e, 4)
        gl = torch.randn(x.shape[0], generator=g).cuda()
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b)
        (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, None, dtype)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e30])
def test_masks_and_empty_rows(dtype, low):
    """Ids masked out by -inf or by the type's lowest value: all of them, all but one, whole chunks, the first and the last."""
    from sage_amd import vocab_softmax as vs
    for V in (1, 70, 500):
        x, w, _, _ = make(20, V, 40, dtype)
        t = torch.arange(20, device="cuda") % V
        masks = [torch.ones(V, dtype=torch.bool)]
        for keep in (0, V - 1, V // 2):
            masks.append(torch.ones(V, dtype=torch.bool))
            masks[-1][keep] = False
        masks.append(torch.arange(V) < min(V - 1, 64))
        for m in masks:
            b = torch.where(m, low, 0.5).float().cuda()
            e = Exact(x, w, b, t, 5)
            f = vs.token_logprobs(x, w, t, bias=b, alternatives=5)
            check_forward(f, e, 5)
            if bool(m.all()):
                assert torch.isneginf(f.lse).all() and (f.entropy == 0).all() and (f.alt_ids == -1).all() and torch.isneginf(f.logprob).all()
            gl, gh = torch.full((20,), 0.1).cuda(), torch.full((20,), -0.2).cuda()
            dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gh)
            (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, gh, dtype)
            close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_go_to_the_lowest_id(dtype):
    from sage_amd import vocab_softmax as vs
    x, w, _, t = make(12, 3000, 24, dtype)
    w[1000:2000] = w[:1000]                      # every logit of the first thousand twice, some three times
    w[2500:2600] = w[100:200]
    w[2999] = w[2998] = w[0]
    x[3] = 0                                     # all logits equal
    x[4] = 0
    e = Exact(x, w, None, t, 32)
    f = vs.token_logprobs(x, w, t, alternatives=32)
    assert torch.equal(f.alt_ids.long()[3:5], torch.arange(32, device="cuda").expand(2, 32))
    check_forward(f, e, 32)
    # float64 sums of one row's two copies are the same number, so the stable order of the definition is the lower id


def test_large_and_small_logits():
    """Rows that are nearly one-hot, nearly uniform, and far from zero."""
    from sage_amd import vocab_softmax as vs
    x, w, _, t = make(40, 2000, 50, F32)
    x *= torch.logspace(-6, 2, 40, device="cuda")[:, None]
    b = torch.full((2000,), 700.0, device="cuda")
    t = (x @ w.t()).argmax(1)
    for bias in (None, b, -b):
        e = Exact(x, w, bias, t, 2)
        f = vs.token_logprobs(x, w, t, bias=bias, alternatives=2)
        check_forward(f, e, 2)
        assert (f.logprob <= 0).all() and (f.entropy >= 0).all()
        gl = torch.full((40,), -1.0, device="cuda")
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=bias)
        (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, None, F32)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw")


def test_rows_of_very_different_sizes():
    """float32 rows share a power of two by 32: sizes from 1e-6 to 1e2 side by side, in x and in the weights."""
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(200, 900, 50, F32, "prior")
    x *= torch.logspace(-6, 2, 200, device="cuda")[torch.randperm(200, generator=torch.Generator().manual_seed(1)).cuda(), None]
    w *= torch.logspace(-5, 0.5, 900, device="cuda")[torch.randperm(900, generator=torch.Generator().manual_seed(2)).cuda(), None]
    gl, gh = torch.logspace(-9, 0, 200).cuda(), -torch.logspace(0, -9, 200).cuda()
    e = Exact(x, w, b, t, 5)
    f = vs.token_logprobs(x, w, t, bias=b, alternatives=5)
    check_forward(f, e, 5)
    for h in (None, gh):
        dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=h)
        (wx, tx), (ww, tw), (wb, tb) = e.gradient(gl, h, F32)
        close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


def test_not_a_number_stays_in_its_row():
    from sage_amd import vocab_softmax as vs
    for bias in ("none", "mask"):
        x, w, b, _ = make(40, 300, 50, F32, bias)
        t = torch.zeros(40, dtype=torch.int64, device="cuda")
        if b is not None:
            b[0] = 0.0
        clean = vs.token_logprobs(x, w, t, bias=b, alternatives=3)
        bad = x.clone()
        bad[7, 3], bad[30, 49] = float("nan"), float("inf")
        t2 = t.clone()
        t2[11] = 300                             # past the vocabulary
        f = vs.token_logprobs(bad, w, t2, bias=b, alternatives=3)
        rows = torch.ones(40, dtype=torch.bool, device="cuda")
        rows[[7, 30]] = False
        for name in ("lse", "entropy", "alt_ids", "alt_logprobs"):
            assert torch.equal(getattr(f, name)[rows], getattr(clean, name)[rows]), name
        assert torch.isnan(f.lse[~rows]).all() and torch.isnan(f.entropy[~rows]).all() and (f.alt_ids[~rows] == -1).all()
        assert torch.isnan(f.logprob[[7, 11, 30]]).all() and int(torch.isnan(f.logprob).sum()) == 3
        gl = torch.ones(40, device="cuda")
        dx, dw, _ = vs.token_logprobs_backward(bad, w, t2, f, gl, bias=b)
        assert torch.isnan(dx[[7, 11, 30]]).all() and torch.isfinite(dx[rows & (torch.arange(40, device="cuda") != 11)]).all()
        assert torch.isnan(dw).any()


def test_no_tokens_and_no_targets():
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(9, 100, 30, BF16, "prior")
    none = vs.token_logprobs(x[:0], w, t[:0], bias=b, alternatives=3)
    assert none.logprob.shape == (0,) and none.alt_ids.shape == (0, 3)
    dx, dw, db = vs.token_logprobs_backward(x[:0], w, t[:0], none, none.logprob, bias=b)
    assert dx.shape == (0, 30) and (dw == 0).all() and (db == 0).all() and dw.shape == (100, 30)
    f = vs.token_logprobs(x, w, bias=b)
    assert f.logprob is None and f.alt_ids is None
    e = Exact(x, w, b, torch.full_like(t, -1))
    close(f.lse, e.lse, e.tol_lse, "lse")
    gh = torch.linspace(-1, 1, 9).cuda()
    dx, dw, db = vs.token_logprobs_backward(x, w, None, f, None, bias=b, grad_entropy=gh)
    (wx, tx), (ww, tw), (wb, tb) = e.gradient(None, gh, BF16)
    close(dx, wx, tx, "dx"), close(dw, ww, tw, "dw"), close(db, wb, tb, "db")


def test_same_bits_every_time():
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(333, 5003, 50, BF16, "prior")
    gl = torch.randn(333, generator=torch.Generator().manual_seed(1)).cuda()
    first = None
    for _ in range(3):
        f = vs.token_logprobs(x, w, t, bias=b, alternatives=7)
        now = (*f, *vs.token_logprobs_backward(x, w, t, f, gl, bias=b, grad_entropy=gl))
        if first is not None:
            assert all(torch.equal(a, c) for a, c in zip(first, now))
        first = now


# ---- clipping -------------------------------------------------------------------------------------------------------
def grads_of(sizes, kinds, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(k).cuda() for n, k in zip(sizes, kinds)]


def exact_norm(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


@pytest.mark.parametrize("sizes", [[1], [7], [0, 5, 0], [32768], [32769, 3], [100003, 1, 17, 65536, 40000], [3 + 7 * i for i in range(300)],
                                   [262144 * 50, 262144 * 50]])
@pytest.mark.parametrize("kind", ["f32", "bf16", "mixed"])
def test_clip(sizes, kind):
    """The norm: 2 u; a scaled value: the factor's and the product's rounding (3 u) and half a step of its type."""
    from sage_amd import vocab_softmax as vs
    kinds = [F32 if kind == "f32" or (kind == "mixed" and i % 2) else BF16 for i in range(len(sizes))]
    grads = grads_of(sizes, kinds)
    before = [t.clone() for t in grads]
    want = exact_norm(grads)
    for limit in (want * 0.3, want * 1.001):
        out = [torch.full_like(t, 7.0) for t in grads]
        got = vs.clip_grad_norm(grads, limit, out=out)
        assert abs(float(got) - want) <= 2 * U * want
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        c = limit / want if want > limit else 1.0
        for t, o in zip(grads, out):
            close(o, t.double() * c, (t.double() * c).abs() * (torch.finfo(t.dtype).eps / 2 + 3 * U) + 1e-37, "clipped")
            if c == 1.0:
                assert torch.equal(o, t)
    norm = vs.clip_grad_norm(grads, want * 0.3)              # in place
    assert abs(float(norm) - want) <= 2 * U * want
    for t, o in zip(before, grads):
        close(o, t.double() * 0.3, (t.double() * 0.3).abs() * (torch.finfo(t.dtype).eps / 2 + 3 * U) + 1e-37, "clipped in place")


def test_clip_views_at_any_element():
    from sage_amd import vocab_softmax as vs
    for kind in (F32, BF16):
        flat = grads_of([5000], [kind])[0]
        cuts = [0, 1, 4, 11, 500, 1777, 4999]
        parts = [flat[a:b] for a, b in zip(cuts[:-1], cuts[1:])]
        keep, want = flat.clone(), exact_norm(parts)
        assert abs(float(vs.clip_grad_norm(parts, 1.0)) - want) <= 2 * U * want
        close(flat[:4999], keep[:4999].double() / want, (keep[:4999].double() / want).abs() * (torch.finfo(kind).eps / 2 + 3 * U) + 1e-37, "views")
        assert torch.equal(flat[4999:], keep[4999:])         # what lies behind the last tensor is left alone


def test_clip_extremes():
    from sage_amd import vocab_softmax as vs
    big = [torch.full((1000,), 3e30, device="cuda"), torch.full((9,), -2e-30, device="cuda")]
    want = 3e30 * math.sqrt(1000)
    assert abs(float(vs.clip_grad_norm(big, 1.0)) / want - 1) < 1e-6
    small = [torch.full((64,), 1e-30, device="cuda")]
    assert abs(float(vs.clip_grad_norm(small, 1.0)) / 8e-30 - 1) < 1e-6 and (small[0] == torch.tensor(1e-30)).all()
    for value in (float("inf"), float("nan")):
        bad = [torch.ones(100, device="cuda"), torch.ones(5, device="cuda")]
        bad[1][2] = value
        norm = float(vs.clip_grad_norm(bad, 0.5))
        assert not math.isfinite(norm) and (bad[0] == 1).all() and bad[1][0] == 1
    zero = [torch.zeros(10, device="cuda")]
    assert float(vs.clip_grad_norm(zero, 0.0)) == 0.0 and (zero[0] == 0).all()


# ---- together, streams, graphs, refusals ----------------------------------------------------------------------------------
def _step(vs, x, w, b, t, gl):
    f = vs.token_logprobs(x, w, t, bias=b, alternatives=5)
    dx, dw, db = vs.token_logprobs_backward(x, w, t, f, gl, bias=b)
    norm = vs.clip_grad_norm([dx, dw, db], 0.01)
    return (*f, dx, dw, db, norm)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_step_on_another_stream_and_in_a_graph(dtype):
    from sage_amd import vocab_softmax as vs
    x, w, b, t = make(200, 3000, 50, dtype, "prior")
    gl = torch.full((200,), -1 / 200.0, device="cuda")
    want = _step(vs, x, w, b, t, gl)
    e = Exact(x, w, b, t, 5)
    (wx, tx), (ww, tw), _ = e.gradient(gl, None, dtype)
    total = math.sqrt(float(want[5].double().square().sum() + want[6].double().square().sum() + want[7].double().square().sum()))
    assert total <= 0.01 * 1.01
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(vs, x, w, b, t, gl)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs = []
    for _ in range(2):                           # two graphs of the same inputs, replayed in turn and at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = _step(vs, x, w, b, t, gl)
        graphs.append((graph, held))
    for turn in range(3):
        x.copy_(make(200, 3000, 50, dtype, "prior", seed=turn)[0])
        for graph, held in graphs:
            for v in held:
                v.zero_()
            graph.replay()
        want = _step(vs, x, w, b, t, gl)
        torch.cuda.synchronize()
        for graph, held in graphs:
            assert all(torch.equal(a, c) for a, c in zip(held, want)), turn
    side2 = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0][0].replay()
    with torch.cuda.stream(side2):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    for graph, held in graphs:
        assert all(torch.equal(a, c) for a, c in zip(held, want))


def test_refusals():
    from sage_amd import vocab_softmax as vs
    from sage_amd.parallel import get_engine
    x, w, b, t = make(4, 100, 30, F32, "prior")
    with pytest.raises(ValueError, match="32 alternatives"):
        vs.token_logprobs(x, w, t, alternatives=33)
    with pytest.raises(ValueError, match="dimension above 512"):
        vs.token_logprobs(torch.zeros(2, 513, device="cuda"), torch.zeros(9, 513, device="cuda"))
    with pytest.raises(ValueError, match="vocab"):
        vs.token_logprobs(x, w[:0], None)
    with pytest.raises(ValueError, match="2\\^20"):
        vs.token_logprobs(x[:, :1], torch.zeros((1 << 20) + 1, 1, device="cuda"))
    with pytest.raises(ValueError, match="type, device and row length"):
        vs.token_logprobs(x, w.bfloat16(), t)
    with pytest.raises(ValueError, match="bias"):
        vs.token_logprobs(x, w, t, bias=b.double())
    with pytest.raises(ValueError, match="targets"):
        vs.token_logprobs(x, w, t[:3])
    with pytest.raises(ValueError, match="next to each other"):
        vs.token_logprobs(torch.zeros(30, 4, device="cuda").t(), w, t)
    with pytest.raises(ValueError, match="overlap"):
        vs.token_logprobs(x[0].expand(4, 30), w, t)
    f = vs.token_logprobs(x, w, t, bias=b)
    with pytest.raises(ValueError, match="grad_logprob"):
        vs.token_logprobs_backward(x, w, t, f, None)
    with pytest.raises(ValueError, match="max_norm"):
        vs.clip_grad_norm([x], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        vs.clip_grad_norm([x], float("nan"))
    with pytest.raises(ValueError, match="overlap"):
        vs.clip_grad_norm([x, x], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        vs.clip_grad_norm([w.view(-1)[:50], w.view(-1)[50:60]], 1.0, out=[w.view(-1)[40:90], torch.zeros(10, device="cuda")])
    # the C-ABI's own checks
    eng = get_engine()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    lse = torch.empty(4, device="cuda")
    need = eng.token_logprobs_workspace(0, 4, 100, 30)
    call = lambda **o: eng.token_logprobs_device(*{**dict(dtype=0, n=4, vocab=100, dim=30, x=x.data_ptr(), ldx=30, w=w.data_ptr(), ldw=30, b=0, t=0, k=0,
                                                        lp=0, H=0, lse=lse.data_ptr(), ids=0, alt=0, ws=ws.data_ptr(), nb=need, st=0), **o}.values())
    torch.cuda.synchronize()
    call()
    torch.cuda.synchronize()
    for bad, words in ((dict(dtype=2), "dtype"), (dict(n=-1), "n >= 0"), (dict(x=0), "d_x is null"), (dict(ldw=29), "rows overlap"), (dict(lse=0), "d_lse"),
                       (dict(nb=need - 1), "workspace"), (dict(ws=ws.data_ptr() + 8), "aligned"), (dict(lp=lse.data_ptr()), "d_targets"),
                       (dict(k=3), "d_alt_ids"), (dict(x=x.data_ptr() + 1), "aligned")):
        with pytest.raises(ValueError, match=words):
            call(**bad)
