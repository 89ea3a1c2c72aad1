"""A tensor that a backward pass needs and that one of the framework's kernels writes in
between: the backward pass refuses, as it does for torch's own in-place operations."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    assert torch.cuda.is_available()
    dev = torch.device("cuda:0")
    rng = np.random.RandomState(1)
    row, col = rng.randint(0, 20, 100).astype(np.int32), rng.randint(0, 20, 100).astype(np.int32)
    a = Csr.from_coo(row, col, rng.standard_normal(100).astype(np.float32), (20, 20), dev)
    return dict(torch=torch, ops=ops, dev=dev, a=a)


def _leaves(env, n=3, shape=(20, 1, 8)):
    return [env["torch"].randn(shape, device=env["dev"]).requires_grad_(True) for _ in range(n)]


def _refuses(env, out):
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_mask_drawn_again(env):
    torch, ops = env["torch"], env["ops"]
    q, k, v = _leaves(env)
    mask = ops.bernoulli_mask(env["a"].nnz, 0.5, 1, 0, env["dev"])
    out = ops.attention_autograd(env["a"], q, k, v, mask=mask)
    ops.bernoulli_mask(env["a"].nnz, 0.5, 2, 0, env["dev"], out=mask)
    _refuses(env, out)
    out = ops.attention_autograd(env["a"], q, k, v, mask=mask)          # nothing written: as ever
    ops.bernoulli_mask(env["a"].nnz, 0.5, 3, 0, env["dev"])
    out.sum().backward()
    assert torch.isfinite(q.grad).all()


def test_weights_stepped(env):
    torch, ops = env["torch"], env["ops"]
    for step in ("adamw", "adam"):
        for which in range(3):
            leaves = _leaves(env)
            out = ops.attention_autograd(env["a"], *leaves)
            w = leaves[which]
            with torch.no_grad():
                if step == "adamw":
                    ops.adamw_step([w], [torch.ones_like(w)], ops.adamw_state([w]), 0.1, 1)
                else:
                    ops.adam_step(w, torch.ones_like(w), torch.zeros_like(w), torch.zeros_like(w), 0.1, 1)
            _refuses(env, out)
    x, weight = torch.randn(20, 8, device=env["dev"]).requires_grad_(True), torch.ones(8, device=env["dev"]).requires_grad_(True)
    _, h = ops.norm_residual_autograd(x, pre_weight=weight)
    with torch.no_grad():
        ops.adamw_step([weight], [torch.ones_like(weight)], ops.adamw_state([weight]), 0.1, 1)
    _refuses(env, h)
    # a weight without a gradient is not written
    w = _leaves(env)
    out = ops.attention_autograd(env["a"], *w)
    with torch.no_grad():
        ops.adamw_step(w[:2], [None, None], ops.adamw_state(w[:2]), 0.1, 1)
    out.sum().backward()
    assert torch.isfinite(w[0].grad).all()


def test_every_result_tensor_counts_its_write(env):
    """The version counter of what the caller passes to be written moves; what is only
    read keeps its own."""
    torch, ops, dev, a = env["torch"], env["ops"], env["dev"], env["a"]
    new = lambda *s: torch.ones(s, device=dev)
    ids = torch.arange(20, dtype=torch.int32, device=dev)
    mask = torch.ones(160, dtype=torch.uint8, device=dev)
    b, w, out = new(20, 8), new(8, 8), new(20, 8)
    bits = torch.zeros(20, 1, dtype=torch.int32, device=dev)
    heads = new(20, 1, 8)
    calls = [
        lambda o: ops.spmm(a, b, out=o), lambda o: ops.gemm(b, w, out=o), lambda o: ops.dropout_rows_philox(b, ids, 0.5, 1, 0, out=o),
        lambda o: ops.dropout_dense(b, mask, 2.0, out=o), lambda o: ops.relu_dropout_bwd(b, b, out=o), lambda o: ops.gather_rows(b, ids, o),
        lambda o: ops.scatter_rows(b, ids, o), lambda o: ops.dropout_philox(b, 0.5, 1, 0, out=o),
        lambda o: ops.relu_dropout_bwd_philox(b, b, 0.5, 1, 0, out=o),
        lambda o: ops.masked_softmax_xent(b, b, mask[:20], grad_out=o),
        lambda o: ops.attention(a, heads, heads, heads, out=o.view(20, 1, 8)),
    ]
    for i, call in enumerate(calls):
        before = out._version, b._version
        call(out)
        assert out._version > before[0] and b._version == before[1], i
    before = bits._version, mask._version
    ops.pack_sign_bits(b, out=bits)
    ops.bernoulli_mask(160, 0.5, 1, 0, dev, out=mask)
    assert bits._version > before[0] and mask._version > before[1]
    before = mask._version
    ops.dropout_philox(b, 0.5, 1, 0, mask_out=mask)
    assert mask._version > before


def test_values_written_between_the_passes(env):
    torch, ops = env["torch"], env["ops"]
    from gcn_amd.sparse import Csr
    a = Csr(20, 20, env["a"].row_ptr, env["a"].col_idx, env["a"].val.clone())
    leaves = _leaves(env)
    out = ops.attention_autograd(a, *leaves, use_values=True)
    a.val.mul_(2.0)
    _refuses(env, out)
    out = ops.attention_autograd(a, *leaves)                             # values not in use: no matter
    a.val.mul_(2.0)
    out.sum().backward()
    assert torch.isfinite(leaves[0].grad).all()


@pytest.mark.parametrize("start", ["matrix", "transpose"])
def test_transpose_follows_the_values(env, start):
    """Values written in place after the transpose was built, on either of the two."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    from gcn_amd.sparse import Csr

    def copy(m):
        return Csr(m.n_rows, m.n_cols, m.row_ptr, m.col_idx, m.val.clone())

    a = copy(env["a"])
    if start == "transpose":
        a = a.transpose()
    q, k, v, g = [torch.randn(20, 2, 8, device=dev) for _ in range(4)]
    b = torch.randn(20, 8, device=dev)

    def gradients(m):
        out, stats = ops.attention(m, q, k, v, use_values=True, want_stats=True)
        x = b.clone().requires_grad_(True)
        ops.spmm_autograd(m, x).sum().backward()
        return (out,) + ops.attention_bwd(m, q, k, v, out, stats, g, use_values=True) + (x.grad,)

    first = gradients(a)
    other = a.transpose()
    for turn in range(3):
        if turn < 2:
            a.val.add_(torch.randn_like(a.val))
        else:
            other = a.transpose()                      # the transpose's: neither matrix is written over, both get a new one
            other.val.add_(1.0)
            kept = other.val.clone()
        want, got = gradients(copy(a)), gradients(a)
        for x, y in zip(want, got):
            assert torch.equal(x, y)
        assert torch.equal(a.transpose().val, copy(a).transpose().val)
        if turn < 2:
            assert not torch.equal(got[2], first[2])
        if turn < 2 and start == "matrix":
            assert a.transpose() is other              # same arrays: recorded launches read the values in force
    assert a.transpose() is a.transpose() and a.transpose() is not other and torch.equal(other.val, kept)
    for x, y in zip(gradients(copy(other)), gradients(other)):
        assert torch.equal(x, y)


def test_values_written_before_a_capture(env):
    """Under a capture the transpose cannot be made again: refused, unless its values
    are not read."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    from gcn_amd.sparse import Csr
    a = Csr(20, 20, env["a"].row_ptr, env["a"].col_idx, env["a"].val.clone())
    q, k, v, g = [torch.randn(20, 2, 8, device=dev) for _ in range(4)]
    how = dict(use_values=True)
    out, stats = ops.attention(a, q, k, v, want_stats=True, **how)
    ops.attention_bwd(a, q, k, v, out, stats, g, **how)
    want = ops.attention_bwd(a, q, k, v, *ops.attention(a, q, k, v, want_stats=True), g)
    a.val.mul_(0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, stats = ops.attention(a, q, k, v, want_stats=True, **how)
        with pytest.raises(RuntimeError, match="before the stream capture"):
            ops.attention_bwd(a, q, k, v, out, stats, g, **how)
        got = ops.attention_bwd(a, q, k, v, *ops.attention(a, q, k, v, want_stats=True), g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_matrix_made_in_inference_mode(env):
    """Its values have no version counter and cannot be saved: they are trusted."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    from gcn_amd.sparse import Csr
    rng = np.random.RandomState(2)
    with torch.inference_mode():
        a = Csr.from_coo(rng.randint(0, 20, 100), rng.randint(0, 20, 100), rng.standard_normal(100), (20, 20), dev)
        q = torch.randn(20, 1, 8, device=dev)
        ops.attention(a, q, q, q, use_values=True, out=torch.empty_like(q))
    leaves = _leaves(env)
    ops.attention_autograd(a, *leaves, use_values=True).sum().backward()
    assert all(torch.isfinite(t.grad).all() for t in leaves) and a.transpose() is a.transpose()
