"""Infinities in edges that count, at heads of every shape: a logit of -inf is a
probability of zero, and what that edge's other elements hold changes nothing."""
import numpy as np
import pytest

from attention_oracle import U

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]
DIMS = [1, 2, 3, 4, 5, 7, 8, 9, 12, 15, 16, 20, 31, 65, 100, 255, 256]


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    assert torch.cuda.is_available()
    return dict(torch=torch, ops=ops, Csr=Csr, dev=torch.device("cuda:0"))


def _operands(env, dtype, dim, seed, rows, cols):
    torch = env["torch"]
    rng = np.random.RandomState(seed)
    make = lambda n: torch.from_numpy(rng.standard_normal((n, 2, dim)).astype(np.float32)).to(env["dev"]).to(getattr(torch, dtype))
    return make(rows), make(cols), make(cols), make(rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("use_values", [False, True])
def test_key_of_infinity(env, dtype, dim, use_values):
    """Column 3's key is infinite in one element and the queries are positive there,
    so that its logit is -inf in every row: the rows are those without the edge."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    rng = np.random.RandomState(dim)
    row = np.concatenate([rng.randint(0, 9, 60), np.arange(9), np.full(300, 9), [9]]).astype(np.int32)     # row 9: several pieces
    col = np.concatenate([rng.choice([0, 1, 2, 4, 5, 6], 60), np.full(9, 3), rng.choice([0, 1, 2, 4, 5, 6], 300), [3]]).astype(np.int32)
    a = env["Csr"].from_coo(row, col, np.zeros(len(row)), (10, 7), dev)
    without = env["Csr"].from_coo(row[col != 3], col[col != 3], np.zeros(int((col != 3).sum())), (10, 7), dev)
    for at in sorted({0, dim // 2, dim - 1}):
        q, k, v, g = _operands(env, dtype, dim, at + 1, 10, 7)
        q[:, :, at] = q[:, :, at].abs() + 1
        k[3, :, at] = float("-inf")
        out, stats = ops.attention(a, q, k, v, use_values=use_values, want_stats=True)
        want, want_stats = ops.attention(without, q, k, v, use_values=use_values, want_stats=True)
        assert torch.isfinite(out).all() and torch.isfinite(stats).all()
        # the same sums in another order: a rounding of each result, and fp32 sums of up to 301
        # terms (their absolute values add up to less than 1 + |out|)
        tol = 2 * torch.finfo(q.dtype).eps
        assert torch.allclose(out.float(), want.float(), rtol=tol, atol=400 * U + tol)
        # dk and dv of that column are sums of products with zeros; dq meets 0 * inf in that
        # element, as its formula does, and nowhere else
        dq, dk, dv = ops.attention_bwd(a, q, k, v, out, stats, g, use_values=use_values)
        assert torch.isfinite(dk).all() and torch.isfinite(dv).all() and not dk[3].any() and not dv[3].any()
        # (terms p |<g, v> - delta| |k| scale of a row: less than 20)
        other = [i for i in range(dim) if i != at]
        want = ops.attention_bwd(without, q, k, v, want, want_stats, g, use_values=use_values)[0][:, :, other].float()
        assert torch.allclose(dq[:, :, other].float(), want, rtol=tol, atol=(400 * U + tol) * 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_gradient_of_infinity(env, dtype, dim):
    """A gradient that is infinite in one element of one row: dv of that row's columns
    is infinite there and unchanged in every other element, other rows and columns are
    as without it."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    row, col = np.array([0, 0, 1, 1, 2], np.int32), np.array([0, 1, 1, 2, 2], np.int32)
    a = env["Csr"].from_coo(row, col, np.zeros(5), (3, 3), dev)
    q, k, v, g = _operands(env, dtype, dim, dim, 3, 3)
    out, stats = ops.attention(a, q, k, v, want_stats=True)
    want = ops.attention_bwd(a, q, k, v, out, stats, g)
    for at in sorted({0, dim - 1}):
        g2 = g.clone()
        g2[0, :, at] = float("inf")                  # row 0 only
        got = ops.attention_bwd(a, q, k, v, out, stats, g2)
        assert torch.equal(got[0][1:], want[0][1:])
        assert torch.equal(got[1][2], want[1][2]) and torch.equal(got[2][2], want[2][2])
        # dv of row 0's columns: infinite in that element, finite and unchanged in every other
        other = [i for i in range(dim) if i != at]
        assert torch.isinf(got[2][:2, :, at]).all() and torch.equal(got[2][:, :, other], want[2][:, :, other])
