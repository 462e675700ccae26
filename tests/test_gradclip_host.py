"""CPU tests of the gradient norms and clipping: the C ABI's checks of its
arguments (nothing is launched on a refused call) and the binding's."""

import ctypes
import math
from array import array

import pytest
import torch

import ilqr_native as nat

A = 0x10000  # stands for a device address


def _arr(code, *v):
    return array(code, v)


def _at(a):
    return a.buffer_info()[0] if isinstance(a, array) else a


def _norm(grads=(A, 2 * A), numel=(5, 7), dtypes=(0, 2), n=2, kind=0, norm=A, norms=None, total=None, ws=A,
          ws_bytes=1 << 30):
    g, s, t = _arr("Q", *grads), _arr("q", *numel), _arr("i", *dtypes)
    return nat.lib().ilqr_b200_grad_norm(_at(g), _at(s), _at(t), n, kind, norm, norms, total, ws, ws_bytes, None)


def _clip(grads=(A, 2 * A), out=(3 * A, 4 * A), numel=(5, 7), dtypes=(0, 0), n=2, kind=0, max_norm=1.0, eps=1e-6,
          total=None, ws=A, ws_bytes=1 << 30):
    g, o, s, t = _arr("Q", *grads), _arr("Q", *out), _arr("q", *numel), _arr("i", *dtypes)
    return nat.lib().ilqr_b200_grad_clip(_at(g), _at(o), _at(s), _at(t), n, kind, max_norm, eps, total, None, ws,
                                         ws_bytes, None)


def _elements(grads=(A,), out=(2 * A,), dtypes=(0,), layout=((1, 10, 0, 10, 0, 10),), B=4, max_norm=1.0, eps=1e-6,
              n=None):
    g, o, t = _arr("Q", *grads), _arr("Q", *out), _arr("i", *dtypes)
    lay = _arr("q", *[v for row in layout for v in row])
    return nat.lib().ilqr_b200_grad_clip_elements(_at(g), _at(o), _at(t), _at(lay), len(grads) if n is None else n, B,
                                                  max_norm, eps, 0, None, None)


def test_workspace_size():
    n = ctypes.c_size_t()
    f = nat.lib().ilqr_b200_grad_workspace_size
    sizes = []
    for k in (0, 1, 60, 61, 1000, 1001, 5000):
        assert f(k, ctypes.byref(n)) == 0 and n.value % 8 == 0
        sizes.append(n.value)
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert f(-1, ctypes.byref(n)) == 1 and f(3, None) == 1


def test_norm_refusals():
    assert _norm(n=-1) == 1
    assert _norm(kind=2) == 1
    assert _norm(dtypes=(0, 3)) == 1 and _norm(dtypes=(-1, 0)) == 1
    assert _norm(numel=(5, -1)) == 1
    assert _norm(numel=(5, (1 << 40) + 1)) == 1
    assert _norm(numel=(1 << 40, 1 << 40)) == 1
    assert _norm(grads=(A, 0)) == 1
    assert _norm(grads=(A + 2, A), dtypes=(0, 0)) == 2      # a float at an odd half
    assert _norm(grads=(A, A + 1), dtypes=(0, 2)) == 2
    assert _norm(norm=None) == 1                              # nothing to write
    assert _norm(ws=None) == 3 and _norm(ws_bytes=8) == 3
    assert _norm(ws=A + 4) == 2


def test_clip_refusals():
    assert _clip(kind=5) == 1
    assert _clip(out=(A, 0)) == 1
    for bad in (-1.0, math.nan):
        assert _clip(max_norm=bad) == 1 and _clip(eps=bad) == 1
    assert _clip(eps=math.inf) == 1
    assert _clip(total=A + 4) == 2
    assert _clip(out=(A + 2, 4 * A)) == 2
    assert _clip(ws=None) == 3
    # an output that another tensor of the call shares
    assert _clip(out=(3 * A, 3 * A)) == 7
    assert _clip(grads=(A, A), out=(A, A)) == 7                # the same tensor twice, in place
    assert _clip(out=(A + 4, 4 * A)) == 7                      # its own input, shifted
    assert _clip(out=(2 * A, 4 * A)) == 7                      # the other's input
    assert _clip(out=(3 * A, 3 * A + 16), numel=(5, 7)) == 7   # 20 bytes, then 4 of them again
    assert _clip(grads=(A, 2 * A), out=(A, 3 * A), numel=((2 * A - A) // 4 + 1, 7)) == 7
    # far from its own output, and within a long one of another tensor, in either order
    assert _clip(grads=(A, 5 * A + 400), out=(5 * A, 9 * A), numel=(1000, 7)) == 7
    assert _clip(grads=(5 * A + 400, A), out=(9 * A, 5 * A), numel=(7, 1000)) == 7
    assert _clip(grads=(A, 5 * A + 3996), out=(5 * A, 9 * A), numel=(1000, 7)) == 7


def test_elements_refusals():
    assert _elements(n=0) == 1 and _elements(grads=(A,) * 9, out=(A,) * 9, dtypes=(0,) * 9,
                                             layout=((1, 1, 0, 1, 0, 1),) * 9) == 1
    assert _elements(B=-1) == 1 and _elements(B=1 << 31) == 1
    assert _elements(B=0) == 0
    assert _elements(dtypes=(3,)) == 1
    assert _elements(max_norm=-1.0) == 1 and _elements(max_norm=math.nan) == 1 and _elements(eps=math.inf) == 1
    assert _elements(grads=(0,)) == 1 and _elements(out=(0,)) == 1
    assert _elements(layout=((-1, 10, 0, 10, 0, 10),)) == 1
    assert _elements(layout=((2, (1 << 30) + 1, 0, 10, 0, 10),)) == 1
    assert _elements(layout=((1, 10, 0, 1 << 60, 0, 10),)) == 1    # no byte offset wraps
    assert _elements(layout=((1, 10, 0, -10, 0, 10),)) == 1
    assert _elements(grads=(A + 2,)) == 2 and _elements(out=(2 * A + 1,)) == 2
    assert _elements(layout=((1, 10, 0, 10, 0, 9),)) == 7           # output slices share a value
    assert _elements(layout=((1, 10, 0, 10, 0, 0),)) == 7           # every element into one slice
    assert _elements(layout=((3, 10, 40, 10, 39, 10),)) == 7        # segments into one another
    assert _elements(out=(A + 40,)) == 7                            # its own input, one element on
    two = dict(dtypes=(0, 0), B=4)
    assert _elements(grads=(A, 2 * A), out=(3 * A, 3 * A + 4), layout=((1, 10, 0, 30, 0, 30),) * 2, **two) == 7
    assert _elements(grads=(A, A), out=(A, A), layout=((1, 10, 0, 10, 0, 10),) * 2, **two) == 7


def test_binding_refusals_without_gpu():
    x = torch.zeros(3)
    with pytest.raises(TypeError):
        nat.grad_norm(x)
    with pytest.raises(TypeError):
        nat.grad_norm([3])
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.grad_norm([x])
    with pytest.raises(RuntimeError, match="empty"):
        nat.grad_norm([])
    with pytest.raises(RuntimeError, match="empty"):
        nat.clip_grad_norm(iter([]), 1.0)
    with pytest.raises(RuntimeError, match="1 to 8"):
        nat.clip_grad_elements([], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        nat.grad_norm([x], norm_type=1.0)
    with pytest.raises(ValueError, match="max_norm"):
        nat.clip_grad_norm([x], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        nat.clip_grad_norm([x], math.nan)
    with pytest.raises(ValueError, match="eps"):
        nat.clip_grad_norm([x], 1.0, eps=-1e-6)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.clip_grad_norm([x], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.clip_grad_elements([x], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        nat.clip_grad_elements([x], math.nan)
    with pytest.raises(TypeError):
        nat.clip_grad_norm([x], "one")
    with pytest.raises(TypeError):
        nat.clip_grad_norm([x], 1.0, out=x)
    with pytest.raises(TypeError):
        nat.clip_grad_elements([x], 1.0, batch_dims=1.5)
    with pytest.raises(TypeError):
        nat.grad_norm(3)

    def fails():
        yield x
        raise KeyError("the caller's own")
    for call in (lambda: nat.grad_norm(fails()), lambda: nat.clip_grad_norm([x], 1.0, out=fails()),
                 lambda: nat.clip_grad_elements([x], 1.0, batch_dims=(1 // 0 for _ in range(1)))):
        with pytest.raises((KeyError, ZeroDivisionError)):
            call()


# ---- the paths' host logic ---------------------------------------------------

def test_operator_options_without_gpu():
    import mpc_compat
    m = mpc_compat.FastMPC(10, 4, 3)
    assert m.grad_clip is None and m.grad_norms is None
    m = mpc_compat.FastMPC(10, 4, 3, max_grad_norm=0.5)
    assert m.grad_clip.mode == "element" and m.grad_clip.max_norm == 0.5 and m.grad_norms is None
    m = mpc_compat.FastMPC(13, 4, 3, zero_nonfinite_grad=True)
    assert m.grad_clip.max_norm == math.inf and m.grad_clip.zero_nonfinite
    for bad in (dict(max_grad_norm=-1.0), dict(max_grad_norm=math.nan), dict(max_grad_norm=1.0, grad_clip="row"),
                dict(max_grad_norm=1.0, grad_clip="batch", zero_nonfinite_grad=True)):
        with pytest.raises(ValueError):
            mpc_compat.FastMPC(10, 4, 3, **bad)


def _plain(nat_module):
    """Plain CPU stands-in for the two calls that the sharded clipping makes."""
    def total(grads, norm_type=2.0):
        flat = torch.cat([g.reshape(-1).double() for g in grads])
        if norm_type == 2.0:
            return flat.square().sum()
        return flat.abs().max() if flat.numel() else torch.zeros((), dtype=torch.float64)

    def clip(grads, max_norm, norm_type=2.0, total=None, out=None):
        norm = total.sqrt() if norm_type == 2.0 else total
        for g, o in zip(grads, out):
            o.copy_(g * (max_norm / (norm + 1e-6)).clamp(max=1.0))
        return out, norm.float()
    nat_module.grad_norm_total, nat_module.clip_grad_norm = total, clip


def _worker(rank, world, port, q):
    import os
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path[:0] = [root, os.path.join(root, "ca-ac-mpc_b200")]
    import torch.distributed as dist
    import ilqr_native
    import ilqr_shard as sh
    _plain(ilqr_native)
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        said = []
        for B, p, bad in ((7, 2.0, None), (7, math.inf, None), (1, 2.0, None), (7, math.inf, 6), (7, 2.0, 6)):
            x0, c = _whole(B, bad)
            lo, hi = sh.shard_bounds(B, rank, world)
            g = {"x0": x0[lo:hi].clone(), "c": c[lo:hi].clone()}
            n = sh.clip_gradients(g, 0.5, norm_type=p)
            full = sh.gather_gradients(g, B, keys=("x0", "c"))
            said.append((float(n), full["x0"].numpy(), full["c"].numpy()))
        q.put((rank, said))
    finally:
        dist.destroy_process_group()


def _whole(B, bad):
    gen = torch.Generator().manual_seed(B)
    x0, c = torch.randn(B, 10, generator=gen), torch.randn(B, 4, 14, generator=gen)
    if bad is not None:
        c[bad, 1, 2] = math.nan
    return x0, c


def test_sharded_clipping_over_two_ranks():
    """Each rank scales by the norm of the whole batch; an empty shard takes
    part, and a NaN on one rank reaches the other whatever the norm."""
    import socket

    import numpy as np
    import torch.multiprocessing as mp
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=300) for _ in procs)
    for p in procs:
        p.join(timeout=120)
        assert p.exitcode == 0
    for k, (B, p, bad) in enumerate(((7, 2.0, None), (7, math.inf, None), (1, 2.0, None), (7, math.inf, 6),
                                     (7, 2.0, 6))):
        x0, c = _whole(B, bad)
        flat = torch.cat([x0.reshape(-1), c.reshape(-1)]).double()
        norm = float(flat.square().sum().sqrt()) if p == 2.0 else float(flat.abs().max())
        for rank in range(2):
            n, gx, gc = got[rank][k]
            if bad is not None:
                assert math.isnan(n) and np.isnan(gx).all() and np.isnan(gc).all()
                continue
            assert abs(n - norm) <= 2.0**-23 * norm
            scale = min(1.0, 0.5 / (norm + 1e-6))
            assert np.allclose(gx, x0.numpy() * scale, rtol=1e-6) and np.allclose(gc, c.numpy() * scale, rtol=1e-6)
