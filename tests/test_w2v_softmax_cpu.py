"""CPU: what the softmax operators refuse before any engine is asked for, and the pairs that the softmax word2vec back end trains on."""
from collections import Counter

import pytest
import torch

from sage_amd import embeddings, vocab_softmax as vs, w2v_softmax as w2v
from sage_amd.w2v_params import Word2VecParams


def _x(n=3, d=4, dtype=torch.float32):
    return torch.zeros((n, d), dtype=dtype)


@pytest.mark.parametrize("x, weight", [
    (_x(), _x()),                                                   # not on a GPU
    (_x(dtype=torch.float16), _x(dtype=torch.float16)),             # neither type
    (_x(dtype=torch.float64), _x()),
    (torch.zeros(4), _x()), (torch.zeros((2, 2, 2)), _x()),         # not matrices
    (None, _x()), ([[1.0, 2.0]], _x()),
])
def test_refused_inputs(x, weight):
    with pytest.raises(ValueError):
        vs.token_logprobs(x, weight, None)
    f = vs.TokenLogprobs(None, torch.zeros(3), torch.zeros(3), None, None)
    with pytest.raises(ValueError):
        vs.token_logprobs_backward(x, weight, torch.zeros(3, dtype=torch.int64), f, torch.zeros(3))


@pytest.mark.parametrize("grads, out", [
    ([], None), (iter(()), None),
    ([torch.zeros(4)], None),                                       # not on a GPU
    ([None], None), ([torch.zeros(4), 1.0], None),                  # not tensors
    ([torch.zeros(4, dtype=torch.float16)], None),
    ([torch.zeros(4)], []), ([torch.zeros(4)], [torch.zeros(4), torch.zeros(4)]),
])
def test_refused_gradients(grads, out):
    with pytest.raises(ValueError):
        vs.clip_grad_norm(grads, 1.0, out=out)


def test_backend_choice(monkeypatch):
    for name in ("softmax", " Softmax ", "hip", "gensim"):
        monkeypatch.setenv("SAGE_W2V_BACKEND", name)
        assert embeddings._backend() == name.strip().lower()
    monkeypatch.setenv("SAGE_W2V_BACKEND", "other")
    assert embeddings._backend() in ("hip", "gensim")


def test_only_skip_gram():
    with pytest.raises(ValueError, match="skip-gram"):
        w2v.train(None, [], Word2VecParams(sg=0), 1, 0.0, 1e-4)


@pytest.mark.parametrize("counts, window", [([], 3), ([1], 3), ([0, 0], 2), ([2], 1), ([5, 0, 1, 7, 3], 4), ([3, 3], 50), ([40, 1, 17], 5)])
def test_pairs_are_those_of_the_plain_loop(counts, window):
    n = sum(counts)
    ids = torch.randint(0, 9, (n,), generator=torch.Generator().manual_seed(3))
    lines = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts, dtype=torch.int64))
    inputs, targets = w2v.skip_gram_pairs(ids, lines, window, None, torch.Generator().manual_seed(5))
    reach = torch.randint(1, window + 1, ids.shape, generator=torch.Generator().manual_seed(5))
    want = Counter()
    for p in range(n):
        for q in range(max(0, p - int(reach[p])), min(n, p + int(reach[p]) + 1)):
            if q != p and lines[p] == lines[q]:
                want[(int(ids[q]), int(ids[p]))] += 1
    assert Counter(zip(inputs.tolist(), targets.tolist())) == want


def test_pairs_leave_out_what_is_not_kept():
    ids = torch.tensor([0, 1, 2, 1, 0, 2])
    lines = torch.zeros(6, dtype=torch.int64)
    keep = torch.tensor([1.5, 0.0, 1.0])                            # always, never, always
    inputs, targets = w2v.skip_gram_pairs(ids, lines, 1, keep, torch.Generator().manual_seed(1))
    assert Counter(zip(inputs.tolist(), targets.tolist())) == Counter({(0, 2): 3, (2, 0): 3})      # 0 2 0 2 are left
    assert len(w2v.skip_gram_pairs(ids, lines, 1, torch.zeros(3), torch.Generator().manual_seed(1))[0]) == 0


@pytest.mark.parametrize("counts, tokens", [([3, 4, 5], 7), ([3, 4, 5], 100), ([9, 1, 1, 9], 2), ([0, 0, 0], 1), ([0, 5, 0], 4), ([1] * 10, 3)])
def test_blocks_hold_whole_lines(counts, tokens):
    blocks = list(w2v.blocks_of_lines(torch.tensor(counts, dtype=torch.int64), tokens))
    assert [b for lo, hi, _, _ in blocks for b in range(lo, hi)] == list(range(len(counts)))
    for lo, hi, first, last in blocks:
        assert (first, last) == (sum(counts[:lo]), sum(counts[:hi])) and (last - first <= tokens or hi == lo + 1)
