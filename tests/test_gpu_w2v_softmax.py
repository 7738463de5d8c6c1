"""GPU: the softmax word2vec back end.  One step (rows gathered, token_logprobs, token_logprobs_backward, clip_grad_norm, both
updates) against the formulas in float64; the back end through get_embeddings and through a whole build_vocab run.

The tolerance of the step, with u = 2^-24.  A float32 element goes into the products as two float16 parts, off by at most
2^-22 of it; the product of the two small parts is left out: 3 * 4u of each |x||w|, and the 3 D sums add 3 D u: a logit is off
by at most (12 + 3 D) u S, S the largest sum of |x||w|.  The sum of exponentials has the same error at most, hence a
probability twice that relative to itself, and 64 u for the exponentials and their sums in parts of 32 and more.  The second
product adds (24 + 3 T) u of its |G||.| for T terms, and adding rows of equal inputs one u a row.  The clipping factor is off
by no more than the gradients' errors over their norm; each update rounds four times."""
import math

import numpy as np
import pytest
import torch

from sage_amd.w2v_params import Word2VecParams

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("size, clips", [(0.05, False), (0.5, True)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n, vocab, dim", [(1, 3, 1), (300, 701, 50), (129, 1200, 33)])
def test_one_step(n, vocab, dim, masked, size, clips):
    from sage_amd.w2v_softmax import SoftmaxSkipGram
    g = torch.Generator().manual_seed(n + vocab)
    ids = torch.arange(0, vocab, 2) if masked else None
    model = SoftmaxSkipGram(vocab, dim, ids.cuda() if masked else None)
    w_in, w_out = (torch.randn((vocab, dim), generator=g) * size for _ in range(2))
    model.w_in, model.w_out = w_in.cuda(), w_out.cuda()
    pick = ids if masked else torch.arange(vocab)
    inputs, targets = (pick[torch.randint(0, len(pick), (n,), generator=g)] for _ in range(2))
    inputs[n // 2:] = inputs[0]                                     # one input many times
    found = model.step(inputs.cuda(), targets.cuda(), 0.025)

    w_in, w_out = w_in.double(), w_out.double()
    x = w_in[inputs]
    z = x @ w_out.T
    if masked:
        off = torch.ones(vocab, dtype=torch.bool)
        off[ids] = False
        z[:, off] = -math.inf
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    G = torch.nn.functional.one_hot(targets, vocab).double() - p
    d_in, d_out = torch.zeros_like(w_in).index_add_(0, inputs, G @ w_out), G.T @ x
    norm, most = math.sqrt(float((d_in ** 2).sum() + (d_out ** 2).sum())), math.sqrt(n)
    if n > 1:
        assert (norm > 1.5 * most) if clips else (norm < most / 1.5)
    f = min(1.0, most / norm) if norm else 1.0

    logit = (12 + 3 * dim) * U * float((x.abs() @ w_out.abs().T).max())
    q = 2 * logit + 64 * U
    e_dx = q * (p @ w_out.abs()) + (24 + 3 * vocab) * U * (G.abs() @ w_out.abs())
    e_in = torch.zeros_like(w_in).index_add_(0, inputs, e_dx + n * U * (G.abs() @ w_out.abs()))
    e_out = q * (p.T @ x.abs()) + (24 + 3 * n) * U * (G.abs().T @ x.abs())
    e_f = math.sqrt(float((e_in ** 2).sum() + (e_out ** 2).sum())) / max(norm, 1e-30) + 2 * U if f < 1 else 0.0
    for got, w, d, e in ((model.w_in, w_in, d_in, e_in), (model.w_out, w_out, d_out, e_out)):
        want = w + 0.025 * f * d
        bound = 0.025 * f * (e + d.abs() * e_f) + 4 * U * (w.abs() + 0.025 * f * d.abs())
        assert ((got.cpu().double() - want).abs() <= bound).all()
    if masked:
        assert torch.equal(model.w_out.cpu()[off].double(), w_out[off])
    want = logp[torch.arange(n), targets]
    assert ((found.logprob.cpu().double() - want).abs() <= q + 8 * U * (want.abs() + z[z > -math.inf].abs().max())).all()


def _topics():
    words = [f"{w} ".encode() for w in ("apple", "pear", "plum", "grape", "bolt", "screw", "nail", "drill")]
    vocab = [bytes([i]) for i in range(256)] + words + [b"zebra "]
    rs = np.random.RandomState(2)
    lines = ["".join(words[j + i % 2 * 4].decode() for j in rs.randint(0, 4, 12)) for i in range(200)]
    return vocab, lines


def test_get_embeddings_softmax_backend(tmp_path, monkeypatch):
    import sage_amd
    from sage_amd import SaGeTokenizer, w2v_softmax
    from sage_amd.embeddings import get_embeddings
    from sage_amd.parallel import run_sage_parallel
    monkeypatch.setenv("SAGE_W2V_BACKEND", "softmax")
    sage_amd.setSageFolder(tmp_path)
    vocab, lines = _topics()
    model = SaGeTokenizer(vocab, 16)
    params = Word2VecParams(D=20, window_size=5, min_count=1)
    emb = get_embeddings(len(vocab), tmp_path, lines, model, 2, params)
    assert emb.shape == (len(vocab), 20) and emb.dtype == np.float64 and np.isfinite(emb).all()
    half = 0.5 / 20
    assert np.abs(emb[264]).max() <= half and not np.array_equal(emb[264], emb[264].astype(np.float32))     # never seen: a draw
    assert np.array_equal(emb[256:264], emb[256:264].astype(np.float32))                                    # float32 vectors widened
    assert np.abs(emb[256:264]).max() > half                                                                # and moved
    assert np.array_equal(get_embeddings(len(vocab), tmp_path, lines, model, 2, params), emb)               # loaded
    losses = run_sage_parallel(emb, lines, model, 2)[2]
    assert all(np.isfinite(v) for v in losses.values())

    # a batch smaller than the pairs, min_count, no subsampling; then what is most likely next to a token
    trained, occurs = w2v_softmax.train(model, lines + ["q"], Word2VecParams(D=20, min_count=2), 2, 0.0, 1e-4, batch=500)
    ids = sorted(np.nonzero(occurs >= 2)[0].tolist())
    assert occurs[ord("q")] == 1 and ord("q") not in ids and set(range(256, 264)) <= set(ids) and len(ids) < 32
    alt, logp = (t.cpu() for t in trained.predict(torch.tensor(ids).cuda(), 32))
    z = trained.w_in.cpu().double()[ids] @ trained.w_out.cpu().double()[ids].T
    want = torch.log_softmax(z, 1).sort(dim=1, descending=True).values
    size = float((trained.w_in.cpu().double()[ids].abs() @ trained.w_out.cpu().double()[ids].abs().T).max())
    assert ((logp[:, :len(ids)].double() - want).abs() <= 2 * (12 + 3 * 20) * U * size + 64 * U).all()
    assert (alt[:, len(ids):] == -1).all() and (logp[:, len(ids):] == -math.inf).all()
    assert all(sorted(row[:len(ids)]) == ids for row in alt.tolist())


def test_nothing_to_train_on(monkeypatch):
    from sage_amd import SaGeTokenizer
    from sage_amd.embeddings import train_embeddings
    monkeypatch.setenv("SAGE_W2V_BACKEND", "softmax")
    vocab, lines = _topics()
    model = SaGeTokenizer(vocab, 16)
    for corpus, params in (([], Word2VecParams()), ([""], Word2VecParams()), (["a"], Word2VecParams()), (lines, Word2VecParams(min_count=10 ** 6))):
        emb = train_embeddings(model, corpus, 1, params)
        assert emb.shape == (len(vocab), 50) and np.abs(emb).max() <= 0.01


def test_build_vocab_with_the_softmax_backend(tmp_path, monkeypatch):
    import sage_amd
    from sage_amd import synth
    monkeypatch.setenv("SAGE_W2V_BACKEND", "softmax")
    sage_amd.setSageFolder(tmp_path)
    corpus, off = synth.make_corpus(300, seed=21, n_types=1200, mean_log_words=2.6)
    vocab = synth.make_vocab(corpus, off, 1200, 16, sample_bytes=200_000)
    (tmp_path / "initial.vocab").write_text("".join(v.hex() + "\n" for v in vocab))
    (tmp_path / "corpus.txt").write_bytes(corpus.tobytes())
    builder = sage_amd.SaGeVocabBuilder([1200, 1000, 800, 600], [1200, 800], max_len=16, workers_number=2, random_seed=692653)
    builder.build_vocab("softmax", str(tmp_path / "corpus.txt"), str(tmp_path / "initial.vocab"), str(tmp_path / "partial.txt"), 300)
    emb = np.load(tmp_path / "results" / "softmax" / "embeddings" / "embeddings_1200.npy")
    assert emb.shape == (1200, 50) and np.isfinite(emb).all()
    assert (tmp_path / "results" / "softmax" / "sage_vocabs" / "sage_vocab_600.vocab").exists()
