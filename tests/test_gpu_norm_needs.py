"""The norms' backward forms the gradients that are asked for and no other."""
import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    assert torch.cuda.is_available()
    dev = torch.device("cuda:0")
    rows = lambda: torch.randn(70, 40, device=dev)
    vector = lambda: torch.rand(40, device=dev) + 0.5
    return dict(torch=torch, ops=ops, dev=dev, args=[rows(), rows(), rows(), vector(), vector(), vector()], dy=rows(), dh=rows())


def test_every_choice(env):
    torch, ops = env["torch"], env["ops"]
    x, z, gate, post, res, pre = env["args"]
    _, _, stats = ops.norm_residual(*env["args"], want_stats=True)
    back = lambda **kw: ops.norm_residual_bwd(x, env["dy"], env["dh"], stats, z, gate, post, res, pre, **kw)
    every = back()
    for need in itertools.product([True, False], repeat=6):
        for on, got, want in zip(need, back(need=need), every):
            assert (got is not None) == on and (not on or torch.equal(got, want)), need


@pytest.mark.parametrize("leaves", [(0,), (1,), (2,), (3,), (4,), (5,), (0, 1), (3, 4, 5), (0, 1, 2)])
def test_frozen_operands_on_the_tape(env, leaves):
    torch, ops = env["torch"], env["ops"]
    _, _, stats = ops.norm_residual(*env["args"], want_stats=True)
    x, rest = env["args"][0], env["args"][1:]
    want = ops.norm_residual_bwd(x, env["dy"], env["dh"], stats, *rest)
    args = [t.clone().requires_grad_(i in leaves) for i, t in enumerate(env["args"])]
    for turn in range(2):                                    # the first call loads the code
        for t in args:
            t.grad = None
        y, h = ops.norm_residual_autograd(*args)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        torch.autograd.backward([y, h], [env["dy"], env["dh"]])
        grown = torch.cuda.max_memory_allocated() - before
    for i, (t, w) in enumerate(zip(args, want)):
        assert (t.grad is not None) == (i in leaves)
        if i in leaves:
            assert torch.equal(t.grad, w)
    if max(leaves) < 3:
        # rows only: their gradients (copied once by the tape at most), no workspace of the column sums
        size = x.numel() * 4 + 512
        assert grown <= 2 * len(leaves) * size
    if min(leaves) >= 3:
        # weights only: no gradient as large as the rows beside the column sums' workspace
        p = ops._norm_struct(*env["args"], "rms", 1e-6)
        import ctypes as C
        from gcn_amd import _lib
        room = _lib.load().gcnx_norm_residual_backward_workspace_bytes(C.byref(p))
        assert grown <= room + 512 + 2 * 3 * 1024
