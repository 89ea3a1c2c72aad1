"""The bounds of tests/test_gpu_attention_delta.py are narrow enough to tell delta from
the probabilities from delta from the rounded output: the latter, planted in the
oracle, is out of them in every case."""
import numpy as np
import pytest

import attention_delta


@pytest.mark.parametrize("case", attention_delta.CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_delta_of_the_rounded_output_is_out_of_bounds(case):
    row, col, shape, operands = attention_delta.make(*case)
    o = attention_delta.oracle(row, col, shape, operands)
    edges = np.bincount(row, minlength=shape[0])
    # one edge: ds is zero whatever delta; beyond 1000 the fp32 sums' own bounds reach fp16's rounding
    told = (edges >= 2) & ((edges <= 1000) | (case[0] == "bfloat16"))
    over = (np.abs(o.wrong_dq - o.dq) / o.dq_bound).max(axis=(1, 2))
    assert (over[told] > 1.5).all(), over
    assert (np.abs(o.wrong_dk - o.dk) / o.dk_bound).max() > 2
