"""Graph attention (forward and backward) against the 64-bit oracle on the host:
types, head layouts, odd sizes, strides, masks, empty and long rows, captures and
streams."""
import numpy as np
import pytest

from attention_oracle import AttentionOracle, assert_within

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    assert torch.cuda.is_available()
    return dict(torch=torch, ops=ops, Csr=Csr, dev=torch.device("cuda:0"))


def _pattern(rng, n_rows, n_cols, nnz, long_rows=(), empty=()):
    """Unsorted coordinates, duplicates included; ``long_rows``: (row, edges)."""
    row, col = rng.randint(0, n_rows, nnz), rng.randint(0, n_cols, nnz)
    for r, n in long_rows:
        row, col = np.concatenate([row[row != r], np.full(n, r)]), np.concatenate([col[row != r], rng.randint(0, n_cols, n)])
    stay = ~np.isin(row, np.asarray(empty, dtype=np.int64))
    return row[stay].astype(np.int32), col[stay].astype(np.int32)


class Case(object):
    def __init__(self, env, row, col, shape, heads, kv, dim, dtype="float32", values=None, mask=None, seed=0, layout="plain", scale=None):
        torch = self.torch = env["torch"]
        self.env, self.shape = env, shape
        rng = np.random.RandomState(seed + 7)
        self.dtype = getattr(torch, dtype)
        self.a = env["Csr"].from_coo(row, col, np.ones(len(row)) if values is None else values, shape, env["dev"])
        self.row, self.col, self.values, self.mask = row, col, values, mask
        self.scale = scale if scale is not None else dim ** -0.5
        make = lambda n, h: torch.from_numpy(rng.standard_normal((n, h, dim)).astype(np.float32)).to(env["dev"]).to(self.dtype)
        q, k, v, g = make(shape[0], heads), make(shape[1], kv), make(shape[1], kv), make(shape[0], heads)
        if layout == "fused":            # q | k | v slices of one tensor (square patterns, equal head counts)
            every = torch.stack([q, k, v], 1)
            q, k, v = every[:, 0], every[:, 1], every[:, 2]
        elif layout == "heads first":
            q, k, v, g = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g)]
        elif layout == "offset":         # rows that are not 16-byte aligned
            def shifted(t):
                flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
                return flat.copy_(t)
            q, k, v, g = [shifted(t) for t in (q, k, v, g)]
        elif layout == "broadcast":      # one query and one gradient for all rows
            q, g = q[:1].expand(shape[0], -1, -1), g[:1].expand(shape[0], -1, -1)
        self.q, self.k, self.v, self.g = q, k, v, g
        self.how = {"scale": scale, "use_values": values is not None,
                    "mask": torch.from_numpy(mask).to(env["dev"]) if mask is not None else None}

    def oracle(self):
        wide = lambda t: t.detach().double().cpu().numpy()
        shift = np.asarray(self.values, np.float32) if self.values is not None else None
        info = self.torch.finfo(self.dtype)
        return AttentionOracle(self.row, self.col, self.shape, wide(self.q), wide(self.k), wide(self.v), float(np.float32(self.scale)),
                               shift, self.mask, info.eps / 2, info.tiny).backward(wide(self.g))

    def run(self):
        ops = self.env["ops"]
        out, stats = ops.attention(self.a, self.q, self.k, self.v, want_stats=True, **self.how)
        return (out,) + ops.attention_bwd(self.a, self.q, self.k, self.v, out, stats, self.g, **self.how)

    def check(self):
        o = self.oracle()
        got = self.run()
        for name, t in zip(("out", "dq", "dk", "dv"), got):
            assert t.dtype == self.dtype
            assert_within(t.float().cpu().numpy(), getattr(o, name), getattr(o, name + "_bound"), name)
        return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 1), (1, 1, 4), (8, 8, 8), (4, 4, 16), (3, 3, 5), (6, 2, 24), (8, 1, 32), (5, 5, 64),
                                          (2, 1, 65), (1, 1, 128), (3, 1, 200), (2, 2, 255), (2, 2, 256), (20, 20, 8), (70, 35, 3)])
def test_head_layouts(env, dtype, heads, kv, dim):
    rng = np.random.RandomState(dim)
    row, col = _pattern(rng, 61, 47, 400, long_rows=[(5, 130), (60, 1)], empty=[0, 17])
    Case(env, row, col, (61, 47), heads, kv, dim, dtype, seed=heads).check()


@pytest.mark.parametrize("n_rows,n_cols,nnz", [(1, 1, 1), (1, 1, 5), (1, 300, 0), (1, 2000, 1500), (300, 1, 290), (5, 7, 0), (513, 2, 900), (2000, 1500, 9000)])
def test_pattern_shapes(env, n_rows, n_cols, nnz):
    rng = np.random.RandomState(nnz + n_rows)
    row, col = _pattern(rng, n_rows, n_cols, nnz)
    for dtype in TYPES:
        Case(env, row, col, (n_rows, n_cols), 4, 2, 16, dtype, seed=nnz).check()


@pytest.mark.parametrize("edges", [255, 256, 257, 258, 510, 511, 512, 513, 514, 1023, 1024, 1025, 2300])
@pytest.mark.parametrize("before", [0, 1, 511, 512, 700, 1024])
def test_long_rows(env, edges, before):
    """A row cut at multiples of 512 in the order of the nonzeros, and the column of
    the same length in the transpose, at every place relative to the cuts."""
    rng = np.random.RandomState(edges * 3 + before)
    row = np.concatenate([rng.randint(0, 3, before), np.full(edges, 3), rng.randint(4, 9, 40)]).astype(np.int32)
    col = rng.randint(0, 50, len(row)).astype(np.int32)
    for r, c in ((row, col), (col, row)):
        shape = (9, 50) if r is row else (50, 9)
        Case(env, r, c, shape, 2, 1, 12, "float32", seed=edges).check()
        Case(env, r, c, shape, 2, 2, 16, "bfloat16", seed=edges).check()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_many_pieces(env, dtype):
    """More pieces than the lanes that join them take in one go, one row and several."""
    rng = np.random.RandomState(71)
    for n_rows in (1, 3):
        row = rng.randint(0, n_rows, 60000).astype(np.int32)
        col = rng.randint(0, 700, 60000).astype(np.int32)
        Case(env, row, col, (n_rows, 700), 2, 1, 12, dtype, seed=3).check()
        Case(env, col, row, (700, n_rows), 4, 2, 3, dtype, seed=4).check()


@pytest.mark.parametrize("edges", [65536, 65537, 140000, 300000, 530000])
def test_one_row_of_every_piece_length(env, edges):
    """The fewer rows share the edges, the longer the pieces: 64 to 512 edges of one row."""
    rng = np.random.RandomState(edges)
    row = np.zeros(edges, np.int32)
    col = rng.randint(0, 900, edges).astype(np.int32)
    Case(env, row, col, (1, 900), 2, 1, 8, "float32", seed=1).check()
    Case(env, col, row, (900, 1), 1, 1, 16, "bfloat16", seed=2).check()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_few_and_of_many_pieces_side_by_side(env, dtype):
    """Rows that a wavefront joins, rows that a workgroup joins and rows in one piece,
    in the reach of the same workgroup."""
    rng = np.random.RandomState(73)
    edges = rng.choice([0, 1, 63, 64, 65, 100, 130, 600, 959, 960, 1025, 2100], 90)
    row = np.repeat(np.arange(90), edges).astype(np.int32)
    col = rng.randint(0, 333, len(row)).astype(np.int32)
    Case(env, row, col, (90, 333), 8, 2, 16, dtype, seed=5).check()
    Case(env, col, row, (333, 90), 3, 3, 40, dtype, seed=6).check()


@pytest.mark.parametrize("heads,kv,dim", [(5, 5, 8), (3, 1, 20), (11, 11, 65), (1, 1, 2)])
def test_long_rows_with_idle_lanes(env, heads, kv, dim):
    """Head counts that leave lanes of a wavefront idle, rows in pieces (the last piece
    at the end of the workspace) and rows of a workgroup."""
    rng = np.random.RandomState(dim)
    for long in (300, 900):
        row = np.concatenate([rng.randint(0, 4, 50), np.full(long, 4)]).astype(np.int32)
        col = rng.randint(0, 30, len(row)).astype(np.int32)
        for dtype in TYPES:
            Case(env, row, col, (5, 30), heads, kv, dim, dtype, seed=1).check()
            Case(env, col, row, (30, 5), heads, kv, dim, dtype, seed=2).check()


def test_offsets_past_32_bits(env):
    """Operands of more than 4 GiB, their last rows in use: as columns, then as rows."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    n, dim = (1 << 22) + 7, 256
    rng = np.random.RandomState(5)
    far = np.concatenate([[0, 1, n - 1, n - 2, n // 2], rng.randint(0, n, 20)]).astype(np.int32)
    near = rng.randint(0, 3, len(far)).astype(np.int32)
    small = Case(env, near, np.arange(len(far), dtype=np.int32), (3, len(far)), 1, 1, dim, "float32")
    want = small.check()
    at = torch.from_numpy(far.astype(np.int64)).to(dev)
    first = {int(f): i for i, f in reversed(list(enumerate(far)))}                      # a node drawn twice is one row
    same = torch.tensor([first[int(f)] for f in far], device=dev)
    big = lambda t: torch.zeros((n, 1, dim), device=dev).index_copy_(0, at, t[same])
    a = env["Csr"].from_coo(near, far, np.ones(len(far)), (3, n), dev)
    k, v = big(small.k), big(small.v)
    twin = Case(env, near, same.cpu().numpy().astype(np.int32), (3, len(far)), 1, 1, dim, "float32")
    want = twin.run()
    out, stats = ops.attention(a, small.q, k, v, want_stats=True)
    got = (out,) + ops.attention_bwd(a, small.q, k, v, out, stats, small.g)
    # the same sums, but where duplicates order an edge otherwise
    close = lambda x, y: torch.allclose(x, y, rtol=1e-4, atol=1e-4)
    assert close(got[0], want[0]) and close(got[1], want[1])
    for g, w in zip(got[2:], want[2:]):
        assert close(g[at], w[same])
        assert float(g.abs().sum()) == pytest.approx(float(w.abs().sum()), rel=1e-4)     # every other row is zero
    del k, v, got, out
    # the far nodes as rows
    a = env["Csr"].from_coo(far, near, np.ones(len(far)), (n, 3), dev)
    twin = Case(env, same.cpu().numpy().astype(np.int32), near, (len(far), 3), 1, 1, dim, "float32")
    want = twin.run()
    q, g = big(twin.q), big(twin.g)
    out, stats = ops.attention(a, q, twin.k, twin.v, want_stats=True)
    got = (out,) + ops.attention_bwd(a, q, twin.k, twin.v, out, stats, g)
    for x, w in zip(got[:2], want[:2]):
        assert close(x[at], w[same])
    for x, w in zip(got[2:], want[2:]):
        assert close(x, w)


def test_no_columns_and_no_rows(env):
    torch, ops = env["torch"], env["ops"]
    none = np.zeros(0, np.int32)
    for shape in ((4, 0), (0, 4), (0, 0)):
        a = env["Csr"].from_coo(none, none, np.zeros(0), shape, env["dev"])
        q, k = torch.ones(shape[0], 2, 8, device=env["dev"]), torch.ones(shape[1], 1, 8, device=env["dev"])
        out, stats = ops.attention(a, q, k, k, want_stats=True)
        assert out.shape == q.shape and not out.any()
        dq, dk, dv = ops.attention_bwd(a, q, k, k, out, stats, q)
        assert not dq.any() and not dk.any() and not dv.any() and dk.shape == k.shape


def test_row_length_hint_changes_nothing(env):
    rng = np.random.RandomState(2)
    row, col = _pattern(rng, 400, 300, 3000)              # no row is long; the hint says so, 0 = unknown does not
    c = Case(env, row, col, (400, 300), 4, 4, 16)
    known = c.run()
    c.a._max_row = 0
    c.a.transpose()._max_row = 0
    for x, y in zip(known, c.run()):
        assert c.torch.equal(x, y)


@pytest.mark.parametrize("layout", ["fused", "heads first", "offset", "broadcast"])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides(env, layout, dtype):
    rng = np.random.RandomState(11)
    row, col = _pattern(rng, 90, 90, 700, empty=[3])
    Case(env, row, col, (90, 90), 4, 4, 16, dtype, layout=layout).check()


@pytest.mark.parametrize("dtype", TYPES)
def test_mask_in_tuple_order(env, dtype):
    rng = np.random.RandomState(21)
    row, col = _pattern(rng, 120, 80, 1500, long_rows=[(9, 800)])
    mask = (rng.rand(len(row)) < 0.5).astype(np.uint8)
    mask[row == 4] = 0                                      # rows with nothing left, a column with nothing left
    mask[row == 119] = 0
    mask[col == 7] = 0
    c = Case(env, row, col, (120, 80), 4, 2, 16, dtype, mask=mask)
    got = c.check()
    assert not got[0][4].any() and not got[1][119].any() and not got[2][7].any() and not got[3][7].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_shift_logits(env, dtype):
    rng = np.random.RandomState(22)
    row, col = _pattern(rng, 100, 100, 900)
    values = rng.standard_normal(len(row)).astype(np.float32)
    values[rng.rand(len(row)) < 0.2] = -np.inf
    values[row == 5] = -np.inf                              # a row with nothing left
    lowest = row == 6
    values[lowest] = np.finfo(np.float32).min               # a row of lowest values: they are alike, the logits vanish beside them
    c = Case(env, row, col, (100, 100), 2, 2, 8, dtype, values=values)
    got = c.check()
    assert not got[0][5].any()
    n = lowest.sum()
    mean = c.v.float()[c.torch.from_numpy(col[lowest].astype(np.int64)).to(env["dev"])].mean(0)
    assert n > 1 and c.torch.allclose(got[0][6].float(), mean, rtol=float(c.torch.finfo(c.dtype).eps), atol=float(c.torch.finfo(c.dtype).eps))


def test_large_logits(env):
    """Logits of thousands: the probabilities of the backward are those of the forward."""
    rng = np.random.RandomState(23)
    row, col = _pattern(rng, 64, 64, 900)
    Case(env, row, col, (64, 64), 2, 2, 32, scale=300.0).check()


@pytest.mark.parametrize("how", ["mask", "values"])
def test_what_is_masked_is_not_read(env, how):
    torch = env["torch"]
    rng = np.random.RandomState(31)
    row, col = _pattern(rng, 50, 40, 600)
    off = (col % 5 == 0)
    if how == "mask":
        c = Case(env, row, col, (50, 40), 2, 2, 16, mask=(~off).astype(np.uint8))
    else:
        c = Case(env, row, col, (50, 40), 2, 2, 16, values=np.where(off, -np.inf, 0.25).astype(np.float32))
    clean = c.run()
    c.k[::5] = float("nan")
    c.v[::5] = float("inf")
    dirty = c.run()
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    live = torch.arange(40, device=env["dev"]) % 5 != 0
    for x, y in zip(clean[2:], dirty[2:]):
        assert torch.equal(x[live], y[live])
    # a row whose every edge is off: its NaN query reaches nobody
    c2 = Case(env, row, col, (50, 40), 2, 2, 16, mask=(row != 8).astype(np.uint8))
    before = c2.run()
    c2.q[8] = float("nan")
    c2.g[8] = float("inf")
    after = c2.run()
    assert torch.equal(before[2], after[2]) and torch.equal(before[3], after[3]) and torch.equal(before[0], after[0])


def test_nan_in_an_edge_that_counts_reaches_its_row(env):
    torch = env["torch"]
    row, col = np.array([0, 0, 1, 1], np.int32), np.array([0, 1, 1, 2], np.int32)
    c = Case(env, row, col, (2, 3), 1, 1, 8)
    c.k[0] = float("nan")
    out = c.run()[0]
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_gradients_against_differences(env):
    """<gradient, direction> against central differences of the 64-bit forward."""
    rng = np.random.RandomState(41)
    row, col = _pattern(rng, 30, 25, 200, empty=[2])
    c = Case(env, row, col, (30, 25), 4, 2, 6)
    _, dq, dk, dv = c.run()
    wide = lambda t: t.double().cpu().numpy()
    g = wide(c.g)

    def loss(q, k, v):
        return (AttentionOracle(row, col, (30, 25), q, k, v, c.scale).out * g).sum()

    base = [wide(t) for t in (c.q, c.k, c.v)]
    h = 1e-5
    for i, grad in enumerate((dq, dk, dv)):
        step = rng.standard_normal(base[i].shape)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * step, base[i] - h * step
        slope = (loss(*up) - loss(*down)) / (2 * h)
        terms = np.abs(wide(grad) * step).sum()
        # truncation h^2 and rounding 2^-52 / h of the differences; fp32 sums of the kernel
        assert abs(slope - (wide(grad) * step).sum()) <= terms * (1e-8 + 200 * 2.0 ** -24)


def test_autograd(env):
    torch, ops = env["torch"], env["ops"]
    rng = np.random.RandomState(42)
    row, col = _pattern(rng, 40, 40, 300)
    c = Case(env, row, col, (40, 40), 4, 2, 8)
    want = c.run()
    leaves = [t.clone().requires_grad_(True) for t in (c.q, c.k, c.v)]
    out = ops.attention_autograd(c.a, *leaves)
    assert torch.equal(out.detach(), want[0])
    out.backward(c.g)
    for t, w in zip(leaves, want[1:]):
        assert torch.equal(t.grad, w)
    # a broadcast query and a gradient of one value: torch sums the broadcast rows
    one = c.q[:1].clone().requires_grad_(True)
    ops.attention_autograd(c.a, one.expand(40, -1, -1), c.k, c.v).sum().backward()
    assert one.grad.shape == (1, 4, 8) and torch.isfinite(one.grad).all()
    # a mask changed between the two passes is noticed
    mask = torch.ones(c.a.nnz, dtype=torch.uint8, device=env["dev"])
    out = ops.attention_autograd(c.a, leaves[0], c.k, c.v, mask=mask)
    mask[0] = 0
    with pytest.raises(RuntimeError):
        out.backward(c.g)
    # only what is asked for
    out, stats = ops.attention(c.a, c.q, c.k, c.v, want_stats=True)
    dq, dk, dv = ops.attention_bwd(c.a, c.q, c.k, c.v, out, stats, c.g, need_kv=False)
    assert torch.equal(dq, want[1]) and dk is None and dv is None
    dq, dk, dv = ops.attention_bwd(c.a, c.q, c.k, c.v, out, stats, c.g, need_q=False)
    assert dq is None and torch.equal(dk, want[2]) and torch.equal(dv, want[3])


def test_same_bits_every_time_and_into_out(env):
    torch, ops = env["torch"], env["ops"]
    rng = np.random.RandomState(43)
    row, col = _pattern(rng, 300, 200, 6000, long_rows=[(7, 1500)])
    c = Case(env, row, col, (300, 200), 4, 4, 32, "bfloat16")
    first = c.run()
    for x, y in zip(first, c.run()):
        assert torch.equal(x, y)
    room = torch.full((302, 4, 40), 7.0, dtype=torch.bfloat16, device=env["dev"])
    ops.attention(c.a, c.q, c.k, c.v, out=room[1:301, :, :32])
    assert torch.equal(room[1:301, :, :32], first[0])
    assert bool((room[0] == 7).all()) and bool((room[301] == 7).all()) and bool((room[:, :, 32:] == 7).all())


def test_captured_and_replayed(env):
    """Two graphs, replayed in turn with eager work between, new inputs each time."""
    torch, ops = env["torch"], env["ops"]
    rng = np.random.RandomState(44)
    cases = []
    for seed in (1, 2):
        row, col = _pattern(rng, 200, 150, 4000, long_rows=[(7, 900)])
        c = Case(env, row, col, (200, 150), 4, 2, 16, seed=seed)
        c.run()                                             # builds the transpose, looks the longest rows up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.got = c.run()
        cases.append((c, graph))
    for turn in range(4):
        for c, graph in cases:
            c.q.copy_(torch.randn_like(c.q))
            graph.replay()
            eager = c.run()
            torch.cuda.synchronize()
            for x, y in zip(c.got, eager):
                assert torch.equal(x, y)


def test_two_streams_at_once(env):
    torch = env["torch"]
    rng = np.random.RandomState(45)
    streams, cases = [torch.cuda.Stream() for _ in range(2)], []
    for seed in (1, 2):
        row, col = _pattern(rng, 500, 400, 20000, long_rows=[(7, 5000)])
        c = Case(env, row, col, (500, 400), 4, 4, 32, seed=seed)
        cases.append((c, c.run()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, _want) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.run())
    torch.cuda.synchronize()
    for i, (_c, want) in enumerate(cases):
        for g in got[i]:
            for x, y in zip(g, want):
                assert torch.equal(x, y)


def test_refusals(env):
    torch, ops = env["torch"], env["ops"]
    c = Case(env, np.array([0, 1], np.int32), np.array([0, 1], np.int32), (2, 2), 2, 2, 8)
    with pytest.raises(TypeError):
        ops.attention(c.a, c.q.double(), c.k.double(), c.v.double())
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q, c.k.half(), c.v)
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q[:1], c.k, c.v)
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q, c.k[..., :4], c.v)
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q.transpose(1, 2).contiguous().transpose(1, 2), c.k, c.v)
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q, c.k[:, :1], c.v)
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q[:, :1], c.k, c.v)
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q, c.k, c.v, mask=torch.ones(1, dtype=torch.uint8, device=env["dev"]))
    with pytest.raises(ValueError):
        ops.attention(c.a, c.q, c.k, c.v, out=torch.empty(1, 2, 8, device=env["dev"]).expand(2, 2, 8))
    with pytest.raises(ValueError):
        wide = torch.zeros(2, 1, 257, device=env["dev"])
        ops.attention(c.a, wide, wide, wide)
    with pytest.raises(RuntimeError):
        ops.attention(c.a, c.q.cpu(), c.k, c.v)
    out, stats = ops.attention(c.a, c.q, c.k, c.v, want_stats=True)
    with pytest.raises(ValueError):
        ops.attention_bwd(c.a, c.q, c.k, c.v, out, stats[:1], c.g)
