"""CPU: tensors whose gradient autograd is to find.  The results of token_logprobs carry none (its gradient is a call of its own), so the call refuses them
where autograd would record it, before it looks for a GPU."""
import pytest
import torch

from sage_amd import vocab_softmax as vs


@pytest.mark.parametrize("which", [0, 1, 2])
def test_what_autograd_would_record_is_refused(which):
    args = [torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(5)]
    args[which].requires_grad_()
    call = lambda: vs.token_logprobs(args[0], args[1], torch.zeros(3, dtype=torch.int64), bias=args[2])
    with pytest.raises(ValueError, match="autograd"):
        call()
    with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):      # nothing is recorded there: the next check speaks
        call()
    args[which] = args[which].detach()
    with pytest.raises(ValueError, match="on a GPU"):
        call()
