"""Skip-gram word2vec with the softmax over the whole vocabulary: the objective that the reference's negative sampling
(embeddings.py:68-75) stands in for, affordable where no [pairs][vocabulary] matrix has to be stored
(sage_amd/vocab_softmax.py).  Windows, subsampling, learning rate and initial values are those of word2vec."""
from __future__ import annotations

import logging
import math
from typing import List, Optional, Tuple

import numpy as np
import torch

from . import vocab_softmax
from .w2v_params import Word2VecParams

BATCH = 8192               # pairs of one step
BLOCK_TOKENS = 1 << 20     # tokens whose pairs are formed, and shuffled, at a time


class SoftmaxSkipGram:
    """Input vectors and output vectors (float32 [vocab, dim] each) of log p(target | input) = log softmax(w_in[input] w_out^T),
    on one GPU.  `ids`: the ids that are trained; the others have no share in the softmax."""

    def __init__(self, vocab: int, dim: int, ids: Optional[torch.Tensor] = None, device: Optional[torch.device] = None, seed: int = 1):
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.rng = torch.Generator(self.device).manual_seed(seed)
        self.w_in = (torch.rand((vocab, dim), generator=self.rng, device=self.device) - 0.5) / dim
        self.w_out = torch.zeros((vocab, dim), device=self.device)
        self.bias = None
        if ids is not None:
            self.bias = torch.full((vocab,), -math.inf, device=self.device)
            self.bias[ids] = 0.0

    def gradients(self, inputs: torch.Tensor, targets: torch.Tensor
                  ) -> Tuple[torch.Tensor, torch.Tensor, vocab_softmax.TokenLogprobs]:
        """Of the sum of log p(targets | inputs): (for w_in, for w_out, what the forward pass found)."""
        x = self.w_in[inputs]
        found = vocab_softmax.token_logprobs(x, self.w_out, targets, bias=self.bias)
        dx, dw, _ = vocab_softmax.token_logprobs_backward(x, self.w_out, targets, found, torch.ones_like(found.logprob), bias=self.bias)
        return torch.zeros_like(self.w_in).index_add_(0, inputs, dx), dw, found

    def step(self, inputs: torch.Tensor, targets: torch.Tensor, alpha: float) -> vocab_softmax.TokenLogprobs:
        """One step up the sum over the pairs.  word2vec makes these steps pair by pair, so that each sees what the one
        before has done; made together they may overshoot where many pairs agree, so their norm is held to that of as many
        independent steps of norm 1."""
        d_in, d_out, found = self.gradients(inputs, targets)
        vocab_softmax.clip_grad_norm([d_in, d_out], math.sqrt(max(len(inputs), 1)))
        self.w_in.add_(d_in, alpha=alpha)
        self.w_out.add_(d_out, alpha=alpha)
        return found

    def predict(self, inputs: torch.Tensor, topn: int = 10) -> Tuple[torch.Tensor, torch.Tensor]:
        """The `topn` (at most 32) most likely neighbours of each input id and their log probabilities, [len(inputs), topn];
        -1 and -inf behind the last trained id."""
        found = vocab_softmax.token_logprobs(self.w_in[inputs], self.w_out, bias=self.bias, alternatives=topn)
        return found.alt_ids, found.alt_logprobs


def skip_gram_pairs(ids: torch.Tensor, lines: torch.Tensor, window: int, keep: Optional[torch.Tensor], rng: torch.Generator
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(inputs, targets) of the tokens `ids` (int64) of the lines `lines` (their numbers, token by token), shuffled: every target
    with its neighbours of the same line, up to a distance drawn from 1 to `window`.  `keep` [vocab]: the probability that a
    token of this id takes part at all."""
    if keep is not None:
        stay = torch.rand(ids.shape, generator=rng, device=ids.device) < keep[ids]
        ids, lines = ids[stay], lines[stay]
    reach = torch.randint(1, window + 1, ids.shape, generator=rng, device=ids.device)
    inputs, targets = [], []
    for d in range(1, min(window, len(ids) - 1) + 1):
        together = lines[:-d] == lines[d:]
        right, left = together & (reach[:-d] >= d), together & (reach[d:] >= d)
        inputs += [ids[d:][right], ids[:-d][left]]
        targets += [ids[:-d][right], ids[d:][left]]
    if not inputs:
        return ids[:0], ids[:0]
    order = torch.randperm(sum(map(len, inputs)), generator=rng, device=ids.device)
    return torch.cat(inputs)[order], torch.cat(targets)[order]


def tokenized(sage_model, corpus, device, lines_per_call: int = 20_000) -> Tuple[torch.Tensor, torch.Tensor]:
    """The corpus as ids (int32, on the device) and the number of tokens of each line (int64, on the host)."""
    ids: List[torch.Tensor] = []
    counts: List[np.ndarray] = []
    for lo in range(0, len(corpus), lines_per_call):
        got, _, _, n = sage_model.tokenize_lines(corpus[lo:lo + lines_per_call])
        ids.append(torch.from_numpy(np.array(got, dtype=np.int32)).to(device))
        counts.append(np.asarray(n, dtype=np.int64))
    if not ids:
        return torch.empty(0, dtype=torch.int32, device=device), torch.empty(0, dtype=torch.int64)
    return torch.cat(ids), torch.from_numpy(np.concatenate(counts))


def blocks_of_lines(counts: torch.Tensor, tokens: int):
    """(first line, line behind the last, first token, token behind the last) of runs of whole lines of at most `tokens` tokens
    (a longer line is a run of its own)."""
    ends = np.concatenate([[0], np.cumsum(counts.numpy())])
    lo = 0
    while lo < len(counts):
        hi = max(lo + 1, int(np.searchsorted(ends, ends[lo] + tokens, side="right")) - 1)
        yield lo, hi, int(ends[lo]), int(ends[hi])
        lo = hi


def train(sage_model, corpus, params: Word2VecParams, epochs: int, sample: float, min_alpha: float, seed: int = 1, batch: int = BATCH
          ) -> Tuple[SoftmaxSkipGram, np.ndarray]:
    """-> (the model, how often each id occurs in the corpus); ids that occur fewer than `params.min_count` times are left out."""
    if not params.sg:
        raise ValueError("the softmax word2vec back end implements skip-gram (sg=1), the reference's setting")
    device = torch.device("cuda", torch.cuda.current_device())
    vocab = sage_model.id_space()
    ids, counts = tokenized(sage_model, corpus, device)
    occurs = torch.bincount(ids, minlength=vocab)
    trained = occurs >= max(params.min_count, 1)
    model = SoftmaxSkipGram(vocab, params.D, torch.nonzero(trained).flatten(), device, seed)
    total = int(occurs[trained].sum())
    keep = None
    if sample > 0 and total:
        often = occurs.clamp(min=1).double() / (sample * total)
        keep = torch.where(trained, (often.sqrt() + 1) / often, 0.0).float()      # word2vec's subsampling of frequent tokens
    elif total:
        keep = trained.float()
    blocks = list(blocks_of_lines(counts, BLOCK_TOKENS)) if total else []
    for epoch in range(epochs):
        said, pairs = torch.zeros(2, dtype=torch.float64, device=device), 0
        for lo, hi, first, last in blocks:
            lines = torch.repeat_interleave(torch.arange(hi - lo), counts[lo:hi]).to(device)
            inputs, targets = skip_gram_pairs(ids[first:last].long(), lines, params.window_size, keep, model.rng)
            for at in range(0, len(inputs), batch):
                done = (epoch + (first + (last - first) * at / len(inputs)) / len(ids)) / epochs
                found = model.step(inputs[at:at + batch], targets[at:at + batch], max(min_alpha, params.ALPHA - (params.ALPHA - min_alpha) * done))
                said += torch.stack((found.logprob.sum(dtype=torch.float64), found.entropy.sum(dtype=torch.float64)))
            pairs += len(inputs)
        if pairs:
            loss, entropy = (said / pairs).tolist()
            logging.info(f"epoch {epoch + 1} of {epochs}: {pairs} pairs, {-loss:.4f} nats per pair, entropy {entropy:.4f}")
    if blocks:
        common = torch.topk(occurs, min(5, int(trained.sum()))).indices
        names = sage_model.inv_str_vocab
        for token, near in zip(common.tolist(), model.predict(common, 5)[0].tolist()):
            logging.info(f"most likely next to {names[token]!r}: {' '.join(names[i] for i in near if i >= 0)}")
    return model, occurs.cpu().numpy()
