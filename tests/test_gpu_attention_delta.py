"""16-bit gradients of rows whose values are nearly alike, against bounds that the
rounding of the output does not enter."""
import pytest

import attention_delta
from attention_oracle import assert_within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", attention_delta.CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_delta_of_the_probabilities(case):
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    dev = torch.device("cuda:0")
    row, col, shape, operands = attention_delta.make(*case)
    a = Csr.from_coo(row, col, [1.0] * len(row), shape, dev)
    q, k, v, g = [t.to(dev) for t in operands]
    out, stats = ops.attention(a, q, k, v, want_stats=True)
    dq, dk, dv = ops.attention_bwd(a, q, k, v, out, stats, g)
    o = attention_delta.oracle(row, col, shape, operands, out.double().cpu().numpy())
    assert_within(out.float().cpu().numpy(), o.out, o.out_bound, "out")
    assert_within(dq.float().cpu().numpy(), o.dq, o.dq_bound, "dq")
    assert_within(dk.float().cpu().numpy(), o.dk, o.dk_bound, "dk")
    # lengths unknown: pieces instead of workgroups
    a._max_row = 0
    a.transpose()._max_row = 0
    again = ops.attention_bwd(a, q, k, v, out, stats, g)
    assert_within(again[0].float().cpu().numpy(), o.dq, o.dq_bound, "dq")
    assert_within(again[1].float().cpu().numpy(), o.dk, o.dk_bound, "dk")
