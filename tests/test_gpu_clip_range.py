"""GPU: clip_grad_norm at the ends of float32's range: norms beyond it and factors below it."""
import math

import pytest
import torch

from .test_gpu_vocab_softmax import BF16, F32, U, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1000, 50_000])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("limit", [1.0, 1e-8, 1e30, 1e-38])
def test_clipping_by_a_very_small_factor(n, dtype, limit):
    """max_norm / N down to 10^-79: the factor is not a float32, the results are.  Each is off by the factor's and the product's rounding (3 u) and half a
    step of its type, and where it is small by twice half a step of the smallest float32 (2^-150) or bf16 (2^-134)."""
    from sage_amd import vocab_softmax as vs
    g = torch.Generator().manual_seed(n)
    grads = [(torch.rand(n, generator=g) * 2e38 + 1e38).to(dtype).cuda(), torch.full((3,), -3e38, dtype=dtype).cuda()]
    before = [t.clone() for t in grads]
    want = math.sqrt(sum(float((t.double() / 1e38).square().sum()) for t in grads)) * 1e38
    norm = float(vs.clip_grad_norm(grads, limit))
    assert norm == math.inf                                  # beyond float32, and the gradients are clipped by what it is
    for t, o in zip(before, grads):
        d = t.double() * (limit / want)
        close(o, d, d.abs() * (torch.finfo(dtype).eps / 2 + 3 * U) + (2.0 ** -149 if dtype == F32 else 2.0 ** -133), "clipped")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_infinite_gradient_beside_large_ones_clips_nothing(dtype):
    from sage_amd import vocab_softmax as vs
    for bad in (math.inf, math.nan):
        grads = [torch.full((500,), 3e38, dtype=dtype).cuda(), torch.tensor([1.0, bad], dtype=dtype).cuda()]
        before = [t.clone() for t in grads]
        assert not math.isfinite(float(vs.clip_grad_norm(grads, 1.0)))
        assert torch.equal(grads[0], before[0]) and float(grads[1][0]) == 1.0
