"""The clipping of a policy's parameters against torch's, in the calls that
torch takes beside the plain one."""

import math

import pytest
import torch

import policy_mpc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_gradients_with_history_are_clipped_as_torch_clips_them():
    """A backward with create_graph=True, as a gradient penalty's. torch's sum of
    1000 squares in 32 bits takes under 32 roundings of 2^-24 to a value, its root
    half of what they make; ours, the factors and products a few: under 2^-18."""
    for p in (2.0, math.inf):
        pair = []
        for clip in (torch.nn.utils.clip_grad_norm_, policy_mpc.clip_grad_norm_):
            w = torch.randn(1000, generator=torch.Generator().manual_seed(1)).to(DEV).requires_grad_(True)
            (w.pow(3).sum()).backward(create_graph=True)
            version = w.grad._version
            n = clip([w], 0.5, norm_type=p)
            assert w.grad.requires_grad and w.grad._version > version and not n.requires_grad
            pair.append((w.grad.detach(), float(n)))
            w.grad = None
        assert abs(pair[0][1] - pair[1][1]) <= 2.0**-18 * pair[0][1]
        assert torch.allclose(pair[0][0], pair[1][0], rtol=2.0**-18, atol=0.0)


def test_norm_type_as_text():
    w = torch.zeros(3, device=DEV, requires_grad=True)
    w.grad = torch.tensor([3.0, 0.0, -4.0], device=DEV)
    assert float(policy_mpc.clip_grad_norm_([w], 2.0, norm_type="inf", error_if_nonfinite=True)) == 4.0
    assert torch.allclose(w.grad, torch.tensor([1.5, 0.0, -2.0], device=DEV), rtol=1e-6)
    with pytest.raises(ValueError, match="norm_type"):
        policy_mpc.clip_grad_norm_([w], 1.0, norm_type="1")
