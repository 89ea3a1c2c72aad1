"""Attention's gradients, one at a time, over matrices without rows or without columns."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 0), (0, 4), (4, 0), (4, 3)])
def test_one_gradient_at_a_time(shape):
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    dev = torch.device("cuda:0")
    none = np.zeros(0, np.int32)
    a = Csr.from_coo(none, none, np.zeros(0), shape, dev)
    for which in range(3):
        leaves = [torch.ones(n, h, 8, device=dev).requires_grad_(i == which) for i, (n, h) in enumerate(((shape[0], 2), (shape[1], 1), (shape[1], 1)))]
        out = ops.attention_autograd(a, *leaves)
        out.backward(torch.ones_like(out))
        assert leaves[which].grad.shape == leaves[which].shape and not leaves[which].grad.any()
