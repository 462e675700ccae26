"""CPU tests of what the binding of the gradient norms and clipping reads, and
in which order."""

import pytest
import torch

import ilqr_native as nat


class _Own(Exception):
    pass


class _Number:
    """A batch dimension whose reading runs the caller's code."""

    def __init__(self, seen):
        self.seen = seen

    def __index__(self):
        self.seen.append(1)
        return 0


def test_batch_dims_are_read_before_the_tensors():
    """What reads them may change the caller's list of tensors, or the tensors
    (here those are refused, having no GPU: after the dimensions were read)."""
    seen = []
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.clip_grad_elements([torch.zeros(3)] * 2, 1.0, batch_dims=[_Number(seen), _Number(seen)])
    assert len(seen) == 2

    class Fails:
        def __index__(self):
            raise _Own
    with pytest.raises(_Own):
        nat.clip_grad_elements([torch.zeros(3)], 1.0, batch_dims=[Fails()])
    grads = [torch.zeros(3)]

    class Clears:
        def __index__(self):
            grads.clear()
            return 0
    with pytest.raises(RuntimeError, match="1 to 8"):
        nat.clip_grad_elements(grads, 1.0, batch_dims=[Clears()])
    with pytest.raises(OverflowError):
        nat.clip_grad_elements([torch.zeros(3)], 1.0, batch_dims=2**70)
