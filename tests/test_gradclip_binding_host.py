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


def test_batch_dims_of_every_kind():
    """Read (then the tensors are refused, having no GPU), or refused as what they are."""
    import numpy as np
    x = [torch.zeros(3, 4), torch.zeros(3)]
    for dims in (0, np.int64(0), np.int32(0), np.uint8(0), True, _Number([]), [0, 0], (0, np.int64(0)), np.zeros(2, int),
                 torch.zeros(2, dtype=torch.long), range(2), iter([0, 0]), {0: 1, 1: 2}):
        with pytest.raises(RuntimeError, match="CUDA"):
            nat.clip_grad_elements(x, 1.0, batch_dims=dims)
    for dims in (1.0, np.float64(0.0), None, "01", [0.0, 0.0], np.zeros(2), torch.tensor(0.5)):
        with pytest.raises(TypeError):
            nat.clip_grad_elements(x, 1.0, batch_dims=dims)
