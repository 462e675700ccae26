"""CPU tests of the clipping of a policy's parameters, with plain stand-ins for
the two native calls that it makes."""

import inspect
import math

import pytest
import torch

import policy_mpc


class _Plain:
    """The native calls in plain form, and what they were given."""

    def __init__(self):
        self.calls = []

    def grad_norm_total(self, grads, norm_type=2.0):
        assert not torch.is_grad_enabled() and isinstance(norm_type, float)
        self.calls.append(("total", list(grads)))
        flat = torch.cat([g.detach().reshape(-1).double() for g in grads])
        return flat.square().sum() if norm_type == 2.0 else flat.abs().max()

    def clip_grad_norm(self, grads, max_norm, norm_type=2.0, eps=1e-6, total=None, out=None):
        assert not torch.is_grad_enabled() and isinstance(norm_type, float) and out is grads
        if total is None:
            total = self.grad_norm_total(grads, norm_type)
            self.calls.pop()
        self.calls.append(("clip", list(grads)))
        norm = total.sqrt() if norm_type == 2.0 else total
        for g in out:
            g.mul_((max_norm / (norm + eps)).clamp(max=1.0).to(g.dtype))
        return out, norm.float()


@pytest.fixture
def plain(monkeypatch):
    p = _Plain()
    monkeypatch.setattr(policy_mpc._nat, "grad_norm_total", p.grad_norm_total)
    monkeypatch.setattr(policy_mpc._nat, "clip_grad_norm", p.clip_grad_norm)
    return p


def _net():
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.Linear(4, 9), torch.nn.Tanh(), torch.nn.Linear(9, 2))
    net(torch.randn(7, 4)).square().sum().backward()
    return net


def test_arguments_are_torchs():
    ours = inspect.signature(policy_mpc.clip_grad_norm_).parameters
    theirs = inspect.signature(torch.nn.utils.clip_grad_norm_).parameters
    assert list(ours) == [p for p in theirs if p != "foreach"]
    assert all(ours[p].default == theirs[p].default for p in ours)


def test_gradients_with_history_are_clipped(plain):
    """Those of a backward with create_graph=True (a gradient penalty's)."""
    w = torch.randn(5, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    (w.pow(3).sum()).backward(create_graph=True)
    assert w.grad.requires_grad
    before, version = w.grad.detach().clone(), w.grad._version
    n = policy_mpc.clip_grad_norm_([w], 0.5)
    assert torch.is_grad_enabled() and not n.requires_grad and w.grad._version > version
    assert torch.allclose(w.grad.detach(), before * 0.5 / (before.norm() + 1e-6))


def test_norm_types_that_torch_takes(plain):
    for given, want in (("inf", math.inf), (math.inf, math.inf), ("2", 2.0), (2, 2.0), (torch.tensor(2.0), 2.0)):
        a, b = _net(), _net()
        bound = 0.3 * float(torch.nn.utils.get_total_norm([q.grad for q in a.parameters()], want))
        na = torch.nn.utils.clip_grad_norm_(a.parameters(), bound, norm_type=given)
        nb = policy_mpc.clip_grad_norm_(b.parameters(), bound, norm_type=given)
        assert math.isclose(float(na), float(nb), rel_tol=2.0**-18)
        for u, v in zip(a.parameters(), b.parameters()):
            assert torch.allclose(u.grad, v.grad, rtol=2.0**-18, atol=0.0)
    with pytest.raises(ValueError):
        policy_mpc.clip_grad_norm_(_net().parameters(), 1.0, norm_type="two")
