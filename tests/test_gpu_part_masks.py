"""Edge masks on matrices that hold a part of their tuple's entries: the mask is in the
order of the whole tuple, for the products and for the attention, forward and
backward.  A mask of any other length is refused on the host."""
import numpy as np
import pytest

from attention_oracle import AttentionOracle, U, assert_within

pytestmark = pytest.mark.gpu

SHAPE = (60, 45)


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    assert torch.cuda.is_available()
    dev = torch.device("cuda:0")
    rng = np.random.RandomState(3)
    row, col = rng.randint(0, SHAPE[0], 1500).astype(np.int32), rng.randint(0, SHAPE[1], 1500).astype(np.int32)
    row[:400] = 7                                            # a row of several pieces
    stay = ~np.isin(row, [4, 20])                            # rows without an entry
    row, col = row[stay], col[stay]
    values = rng.standard_normal(len(row)).astype(np.float32)
    mask = (rng.rand(len(row)) < 0.6).astype(np.uint8)
    flag = (rng.rand(SHAPE[1]) < 0.5).astype(np.uint8)
    flag[-1] = 1
    return dict(torch=torch, ops=ops, dev=dev, rng=rng, row=row, col=col, values=values, mask=mask, flag=flag,
                a=Csr.from_coo(row, col, values, SHAPE, dev), mask_dev=torch.from_numpy(mask).to(dev))


def _parts(env):
    """(name, matrix, rows kept, tuple entries in it, whether it is transposed)"""
    a, torch = env["a"], env["torch"]
    kept = env["flag"][env["col"]] != 0
    sub = a.filter_columns(torch.from_numpy(env["flag"]).to(env["dev"]))
    whole = np.arange(SHAPE[0])
    yield "filtered", sub, whole, kept
    packed, rows = sub.compact_rows()
    yield "filtered, without empty rows", packed, rows.cpu().numpy(), kept
    few = np.setdiff1d(whole, [4])
    yield "one empty row left out", a.keep_rows(torch.from_numpy(few)), few, np.ones(len(env["row"]), bool)
    yield "filtered twice", sub.filter_columns(torch.ones(SHAPE[1], dtype=torch.uint8, device=env["dev"])), whole, kept


def test_only_the_tuple_s_length_is_taken(env):
    torch, ops = env["torch"], env["ops"]
    for name, m, rows, kept in _parts(env):
        assert m.input_nnz == len(env["row"]) and m.transpose().input_nnz == m.input_nnz, name
        q = torch.ones(m.n_rows, 1, 8, device=env["dev"])
        k = torch.ones(m.n_cols, 1, 8, device=env["dev"])
        for n in {m.nnz, m.input_nnz - 1, m.input_nnz + 1} - {m.input_nnz}:
            short = torch.ones(n, dtype=torch.uint8, device=env["dev"])
            with pytest.raises(ValueError):
                ops.attention(m, q, k, k, mask=short)
            with pytest.raises(ValueError):
                ops.spmm(m, k.view(-1, 8), mask=short)
        with pytest.raises(ValueError):
            ops.spmm(m, k.view(-1, 8), mask=torch.ones(2 * m.input_nnz, dtype=torch.uint8, device=env["dev"])[::2])


@pytest.mark.parametrize("use_values", [False, True])
def test_attention(env, use_values):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    rng = np.random.RandomState(5)
    for name, m, rows, kept in _parts(env):
        place = np.full(SHAPE[0], -1)
        place[rows] = np.arange(len(rows))
        make = lambda n: rng.standard_normal((n, 2, 8)).astype(np.float32)
        q, k, v, g = make(len(rows)), make(SHAPE[1]), make(SHAPE[1]), make(len(rows))
        o = AttentionOracle(place[env["row"]], env["col"], (len(rows), SHAPE[1]), *[x.astype(np.float64) for x in (q, k, v)],
                            float(np.float32(8 ** -0.5)), env["values"] if use_values else None, (env["mask"] != 0) & kept).backward(g.astype(np.float64))
        q, k, v, g = [torch.from_numpy(x).to(dev) for x in (q, k, v, g)]
        how = dict(use_values=use_values, mask=env["mask_dev"])
        out, stats = ops.attention(m, q, k, v, want_stats=True, **how)
        for what, got in zip(("out", "dq", "dk", "dv"), (out,) + ops.attention_bwd(m, q, k, v, out, stats, g, **how)):
            assert_within(got.cpu().numpy(), getattr(o, what), getattr(o, what + "_bound"), (name, what))


def test_product(env):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    rng = np.random.RandomState(6)
    for name, m, rows, kept in _parts(env):
        dense = np.zeros(SHAPE)
        on = (env["mask"] != 0) & kept
        np.add.at(dense, (env["row"][on], env["col"][on]), env["values"][on].astype(np.float64))
        size = np.zeros(SHAPE)
        np.add.at(size, (env["row"][on], env["col"][on]), np.abs(env["values"][on].astype(np.float64)))
        for t, d, s in ((m, dense[rows], size[rows]), (m.transpose(), dense[rows].T, size[rows].T)):
            b = rng.standard_normal((t.n_cols, 16)).astype(np.float32)
            got = ops.spmm(t, torch.from_numpy(b).to(dev), mask=env["mask_dev"])
            # one rounding a product and a sum, at most 400 of them
            assert_within(got.cpu().numpy(), d @ b, 402 * U * (s @ np.abs(b)) + 1e-37, name)


def test_mask_in_the_order_of_a_transpose_s_source(env):
    """A matrix without an index of its own (mask in the order of its nonzeros) and its
    transpose, whose index counts the same entries: forward and backward of both."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    b = env["a"].transpose(cache=False)
    assert b.input_index is None
    counts = (b.row_ptr[1:] - b.row_ptr[:-1]).cpu()
    row = torch.repeat_interleave(torch.arange(b.n_rows), counts).numpy()
    col = b.col_idx.cpu().numpy()
    rng = np.random.RandomState(8)
    mask = (rng.rand(b.nnz) < 0.7).astype(np.uint8)
    t = b.transpose()
    assert t.transpose() is b and t.input_nnz == b.nnz
    for m, r, c in ((t, col, row), (b, row, col)):
        make = lambda n: rng.standard_normal((n, 2, 8)).astype(np.float32)
        q, k, v, g = make(m.n_rows), make(m.n_cols), make(m.n_cols), make(m.n_rows)
        o = AttentionOracle(r, c, m.shape, *[x.astype(np.float64) for x in (q, k, v)], float(np.float32(8 ** -0.5)), None, mask).backward(g.astype(np.float64))
        leaves = [torch.from_numpy(x).to(dev).requires_grad_(True) for x in (q, k, v)]
        out = ops.attention_autograd(m, *leaves, mask=torch.from_numpy(mask).to(dev))
        out.backward(torch.from_numpy(g).to(dev))
        for what, got in zip(("out", "dq", "dk", "dv"), [out.detach()] + [x.grad for x in leaves]):
            assert_within(got.cpu().numpy(), getattr(o, what), getattr(o, what + "_bound"), what)
