"""The softmax over a whole vocabulary on torch tensors: log probabilities of given tokens with their entropy and the most
likely alternatives, the gradient of both, and the clipping of gradients by their global norm (C-ABI: include/sage_hip.h).

The reference trains its embeddings with negative samples in place of this softmax (embeddings.py:68-75) and scores with
log-sigmoids of row products (utils.py:125-138); here the sum over the vocabulary itself is taken, without storing a
[tokens][vocabulary] matrix.  All calls are enqueued on the current stream of the tensors' device and return at once, may
be captured into a graph (once a first call has made the device's engine), and take their workspace from torch's allocator."""
from __future__ import annotations

from array import array
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from .parallel import get_engine

_TYPES = {torch.float32: 0, torch.bfloat16: 1}


class TokenLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]         # float32 [n]: of the given targets; 0 where a target is negative
    entropy: torch.Tensor                   # float32 [n], in nats
    lse: torch.Tensor                       # float32 [n]: log of the sum of exponentials
    alt_ids: Optional[torch.Tensor]         # int32 [n, alternatives], most likely first; -1 where fewer ids are left
    alt_logprobs: Optional[torch.Tensor]    # float32 [n, alternatives]


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-dimensional tensor")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU")
    if t.numel() and t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the elements of a row must lie next to each other")
    if t.shape[0] > 1 and t.numel() and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows overlap (stride {t.stride(0)}, {t.shape[1]} elements)")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[1] != like.shape[1]):
        raise ValueError(f"{name} must have the type, device and row length of x")
    return t


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _vector(name: str, t: Optional[torch.Tensor], n: int, dtype, device) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (n,) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a tensor of {n} {dtype} on {device}")
    return t.contiguous()


def _targets(t: Optional[torch.Tensor], n: int, device) -> Optional[torch.Tensor]:
    if isinstance(t, torch.Tensor) and t.dtype == torch.int32:
        t = t.long()
    return _vector("targets", t, n, torch.int64, device)


def _stream(device) -> int:
    return torch.cuda.current_stream(device.index).cuda_stream


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def _not_recorded(**tensors) -> None:
    for name, t in tensors.items():
        if torch.is_grad_enabled() and isinstance(t, torch.Tensor) and t.requires_grad:
            raise ValueError(f"{name} requires a gradient, which autograd cannot find through this call: make it under torch.no_grad() and take "
                             "the gradient from token_logprobs_backward")


def token_logprobs(x: torch.Tensor, weight: torch.Tensor, targets: Optional[torch.Tensor] = None, *, bias: Optional[torch.Tensor] = None,
                   alternatives: int = 0) -> TokenLogprobs:
    """log p(targets[n] | x[n]) with p = softmax(x weight^T + bias), the entropy of p, and its `alternatives` largest ids.

    x [n, D] and weight [V, D] are both float32 or both bfloat16 with any row stride; bias float32 [V] (-inf masks an id);
    targets int64 or int32 [n] (negative: none; such a row of x may hold anything in the gradient).  What rows of masked ids hold
    does not matter.  D <= 512, V <= 2^20, at most 32 alternatives (ties: the lower id).  The results carry no gradient for
    autograd (token_logprobs_backward has it): tensors that require one are refused unless under torch.no_grad()."""
    _not_recorded(x=x, weight=weight, bias=bias)
    _rows("x", x)
    _rows("weight", weight, x)
    (n, dim), vocab, dev = x.shape, weight.shape[0], x.device
    bias = _vector("bias", bias, vocab, torch.float32, dev)
    targets = _targets(targets, n, dev)
    engine, kind = get_engine(dev.index), _TYPES[x.dtype]
    need = engine.token_logprobs_workspace(kind, n, vocab, dim, int(alternatives))
    logprob, entropy, lse = torch.empty((3, n), dtype=torch.float32, device=dev).unbind(0)
    if targets is None:
        logprob = None
    alt = (None, None)
    if alternatives:
        alt = (torch.empty((n, alternatives), dtype=torch.int32, device=dev), torch.empty((n, alternatives), dtype=torch.float32, device=dev))
    ws = _workspace(need, dev)
    engine.token_logprobs_device(kind, n, vocab, dim, x.data_ptr(), _stride(x), weight.data_ptr(), _stride(weight), _address(bias),
                                 _address(targets), int(alternatives), _address(logprob), entropy.data_ptr(), lse.data_ptr(),
                                 _address(alt[0]), _address(alt[1]), ws.data_ptr(), ws.numel(), _stream(dev))
    return TokenLogprobs(logprob, entropy, lse, *alt)


def token_logprobs_backward(x: torch.Tensor, weight: torch.Tensor, targets: Optional[torch.Tensor], forward: TokenLogprobs,
                            grad_logprob: Optional[torch.Tensor], *, bias: Optional[torch.Tensor] = None,
                            grad_entropy: Optional[torch.Tensor] = None
                            ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(dx, dweight, dbias) for the gradients of logprob and entropy (float32 [n], either may be None) of
    `forward = token_logprobs(x, weight, targets, bias=bias)`.  dx and dweight have the inputs' type; dbias is float32, None
    without a bias."""
    _rows("x", x)
    _rows("weight", weight, x)
    (n, dim), vocab, dev = x.shape, weight.shape[0], x.device
    bias = _vector("bias", bias, vocab, torch.float32, dev)
    targets = _targets(targets, n, dev)
    lse = _vector("forward.lse", forward.lse, n, torch.float32, dev)
    entropy = _vector("forward.entropy", forward.entropy, n, torch.float32, dev)
    grad_logprob = _vector("grad_logprob", grad_logprob, n, torch.float32, dev)
    grad_entropy = _vector("grad_entropy", grad_entropy, n, torch.float32, dev)
    if grad_logprob is None and grad_entropy is None:
        raise ValueError("need grad_logprob or grad_entropy")
    if grad_logprob is not None and targets is None:
        raise ValueError("grad_logprob needs targets")
    engine, kind = get_engine(dev.index), _TYPES[x.dtype]
    need = engine.token_logprobs_backward_workspace(kind, n, vocab, dim)
    dx = torch.empty((n, dim), dtype=x.dtype, device=dev)
    dw = torch.empty((vocab, dim), dtype=x.dtype, device=dev)
    db = torch.empty(vocab, dtype=torch.float32, device=dev) if bias is not None else None
    ws = _workspace(need, dev)
    engine.token_logprobs_backward_device(kind, n, vocab, dim, x.data_ptr(), _stride(x), weight.data_ptr(), _stride(weight),
                                          _address(bias), _address(targets), lse.data_ptr(), entropy.data_ptr(), _address(grad_logprob),
                                          _address(grad_entropy), dx.data_ptr(), dim, dw.data_ptr(), dim, _address(db), ws.data_ptr(),
                                          ws.numel(), _stream(dev))
    return dx, dw, db


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, *, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales `grads` (float32 and bfloat16 tensors, contiguous, all on one GPU) so that their global 2-norm is at most
    `max_norm`: in place, or into `out` (tensors of the same sizes and types).  Returns the norm before clipping, a float32
    scalar on the GPU.  An infinity or a NaN among the gradients makes the norm infinite or NaN and leaves them unchanged; finite
    gradients whose norm passes float32's range are clipped too (the norm returned is then infinite)."""
    grads = list(grads)
    out = grads if out is None else list(out)
    if not grads:
        raise ValueError("need at least one gradient")
    if len(out) != len(grads):
        raise ValueError(f"{len(grads)} gradients, but {len(out)} tensors for the result")
    if not all(isinstance(t, torch.Tensor) for t in (*grads, *out)):
        raise ValueError("gradients and results must be tensors")
    dev = grads[0].device
    for g, o in zip(grads, out):
        if g.dtype not in _TYPES or not g.is_cuda or g.device != dev or not g.is_contiguous():
            raise ValueError("gradients must be contiguous float32 or bfloat16 tensors on one GPU")
        if o is not g and (o.dtype != g.dtype or o.device != dev or o.numel() != g.numel() or not o.is_contiguous()):
            raise ValueError("results must be contiguous tensors of the gradients' sizes, types and device")
    engine = get_engine(dev.index)
    addresses = array("Q", [g.data_ptr() for g in grads])
    results = addresses if out is grads else array("Q", [o.data_ptr() for o in out])
    sizes = array("q", [g.numel() for g in grads])
    types = array("i", [_TYPES[g.dtype] for g in grads])
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _workspace(engine.clip_grad_norm_workspace(sizes), dev)
    engine.clip_grad_norm_device(addresses, results, sizes, types, max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                 _stream(dev))
    return norm
