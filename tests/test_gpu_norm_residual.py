"""Norms fused with a block's gate and residual scale against the 64-bit formulas on
the host, with error bounds derived from the kernel's arithmetic."""
import itertools

import numpy as np
import pytest

from attention_oracle import U, assert_within

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]
# A sum over a row: 8 terms a lane, 6 exchanges, up to 16 wavefronts; the division and
# the square root that follow it: one rounding each.
ROW = 36 * U


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    assert torch.cuda.is_available()
    return dict(torch=torch, ops=ops, dev=torch.device("cuda:0"))


def mean(a):
    return a.mean(1, keepdims=True)


def norm(v, e_v, layer, eps):
    """(unit, inv, bound of unit's error) of rows v known up to e_v."""
    mu = mean(v) if layer else np.zeros((len(v), 1))
    c = v - mu
    inv = 1 / np.sqrt(mean(c * c) + eps)
    unit = c * inv
    e_c = e_v + (mean(e_v) + ROW * mean(np.abs(v)) if layer else 0) + U * (np.abs(v) + np.abs(mu)) * layer
    # the mean square moves with the elements' errors along the row, and by its own sum's
    e_inv = ROW + inv * mean(np.abs(unit) * e_c) + mean((inv * e_c) ** 2)
    return unit, inv, inv * e_c + np.abs(unit) * (e_inv + 2 * U)


class Oracle(object):
    def __init__(self, x, z, gate, post, res, pre, layer, eps, half, tiny):
        self.__dict__.update(locals())
        one = np.ones(x.shape[1])
        self.u_e = np.zeros_like(x)
        if z is not None:
            self.z_unit, self.z_inv, e = norm(z, np.zeros_like(z), layer, eps) if post is not None else (z, None, np.zeros_like(z))
            self.e_z = e
            self.post1 = post if post is not None else one
            self.u = self.z_unit * self.post1
            self.e_u = np.abs(self.post1) * e + U * np.abs(self.u)
            self.res1 = res if res is not None else one
            if gate is None:
                self.sig, self.e_sig = np.ones_like(x), np.zeros_like(x)
            else:
                self.sig = 1 / (1 + np.exp(-gate))
                # the exponent's product, 2 ulp of the exponential and 1 of the reciprocal
                self.e_sig = self.sig * ((1 - self.sig) * (2 * np.abs(gate) + 4) + 4) * U
            f = self.res1 * self.sig
            self.y = x + f * self.u
            self.e_y = np.abs(f) * self.e_u + np.abs(self.res1 * self.u) * self.e_sig + 3 * U * np.abs(f * self.u) + U * np.abs(self.y)
        else:
            self.y, self.e_y = x, np.zeros_like(x)
        if pre is not None:
            self.y_unit, self.y_inv, self.e_yu = norm(self.y, self.e_y, layer, eps)
            self.h = self.y_unit * pre
            self.e_h = np.abs(pre) * self.e_yu + U * np.abs(self.h)

    def rounded(self, value, error):
        return error * (1 + self.half) + self.half * np.maximum(np.abs(value), self.tiny) + 1e-37

    def through(self, d, e_d, unit, e_unit, inv):
        """Backward through a norm: the gradient of the row and its error."""
        along = mean(d * unit)
        m = mean(d) if self.layer else 0 * along
        out = (d - m - unit * along) * inv
        size = np.abs(d) + np.abs(m) + np.abs(unit * along)
        e_along = mean(np.abs(unit) * e_d + np.abs(d) * e_unit) + ROW * mean(np.abs(d * unit))
        e_m = (mean(e_d) + ROW * mean(np.abs(d))) if self.layer else 0
        e = e_d + e_m + np.abs(unit) * e_along + e_unit * np.abs(along) + 4 * U * size
        # the inverse is the forward's, whose error moved the unit row alike
        return out, inv * e + np.abs(out) * (ROW + inv * mean(np.abs(unit) * (e_unit / inv)))

    def backward(self, dy, dh):
        g = np.zeros_like(self.x) if dy is None else dy
        e_g = np.zeros_like(g)
        n = len(g)
        cols = lambda terms, errors: (terms.sum(0), errors.sum(0) + (n + 40) * U * np.abs(terms).sum(0) + 1e-37)
        self.grads = {}
        if dh is not None:
            self.grads["dpre"] = cols(dh * self.y_unit, np.abs(dh) * (self.e_yu + 2 * U * np.abs(self.y_unit)))
            t = dh * self.pre
            back, e = self.through(t, U * np.abs(t), self.y_unit, self.e_yu + 2 * U * np.abs(self.y_unit), self.y_inv)
            g = g + back
            e_g = e + U * np.abs(g)
        self.grads["dx"] = g, self.rounded(g, e_g)
        if self.z is None:
            return self
        gs = g * self.sig
        e_gs = self.sig * e_g + np.abs(g) * self.e_sig + U * np.abs(gs)
        if self.res is not None:
            self.grads["dres"] = cols(gs * self.u, np.abs(self.u) * e_gs + np.abs(gs) * self.e_u + U * np.abs(gs * self.u))
        d = gs * self.res1
        e_d = np.abs(self.res1) * e_gs + U * np.abs(d)
        if self.gate is not None:
            dg = d * self.u * (1 - self.sig)
            e = (e_d * np.abs(self.u) + np.abs(d) * self.e_u) * (1 - self.sig) + np.abs(d * self.u) * (self.e_sig + U) + 3 * U * np.abs(dg)
            self.grads["dgate"] = dg, self.rounded(dg, e)
        if self.post is not None:
            self.grads["dpost"] = cols(d * self.z_unit, np.abs(self.z_unit) * e_d + np.abs(d) * (self.e_z + 2 * U * np.abs(self.z_unit)))
            d, e_d = self.through(d * self.post, np.abs(self.post) * e_d + U * np.abs(d * self.post), self.z_unit,
                                  self.e_z + 2 * U * np.abs(self.z_unit), self.z_inv)
        self.grads["dz"] = d, self.rounded(d, e_d)
        return self


class Case(object):
    def __init__(self, env, n, dim, dtype="float32", kind="rms", z=True, gate=True, post=True, res=True, pre=True, seed=0, eps=1e-6,
                 offset=0.0, layout="plain"):
        torch, dev = env["torch"], env["dev"]
        self.env, self.dtype, self.kind, self.eps = env, getattr(torch, dtype), kind, eps
        rng = np.random.RandomState(seed + n + dim)
        def rows(on, off=0.0):
            if not on:
                return None
            t = torch.from_numpy((rng.standard_normal((n, dim)) + off).astype(np.float32)).to(dev).to(self.dtype)
            if layout == "strided":
                room = torch.full((n, dim + 5), float("nan"), dtype=self.dtype, device=dev)
                room[:, 2:dim + 2] = t
                t = room[:, 2:dim + 2]
            return t
        vector = lambda on: torch.from_numpy((rng.rand(dim) + 0.5).astype(np.float32)).to(dev) if on else None
        self.x = rows(True, offset)
        self.ops = {"z": rows(z, offset), "gate": rows(z and gate), "post_weight": vector(z and post), "res_scale": vector(z and res),
                    "pre_weight": vector(pre)}
        self.dy, self.dh = rows(True), rows(pre)

    def run(self):
        ops = self.env["ops"]
        y, h, stats = ops.norm_residual(self.x, kind=self.kind, eps=self.eps, want_stats=True, **self.ops)
        return y, h, ops.norm_residual_bwd(self.x, self.dy, self.dh, stats, kind=self.kind, eps=self.eps, **self.ops)

    def oracle(self):
        wide = lambda t: None if t is None else t.double().cpu().numpy()
        o, info = self.ops, self.env["torch"].finfo(self.dtype)
        return Oracle(wide(self.x), wide(o["z"]), wide(o["gate"]), wide(o["post_weight"]), wide(o["res_scale"]), wide(o["pre_weight"]),
                      self.kind == "layer", float(np.float32(self.eps)), info.eps / 2, info.tiny).backward(wide(self.dy), wide(self.dh))

    def check(self):
        o = self.oracle()
        y, h, grads = self.run()
        num = lambda t: t.double().cpu().numpy()
        if self.ops["z"] is None:
            assert y is self.x
        else:
            assert_within(num(y), o.y, o.rounded(o.y, o.e_y), "y")
        if self.ops["pre_weight"] is None:
            assert h is None
        else:
            assert_within(num(h), o.h, o.rounded(o.h, o.e_h), "h")
        for name, t in zip(("dx", "dz", "dgate", "dpost", "dres", "dpre"), grads):
            assert (t is not None) == (name in o.grads), name
            if t is not None:
                assert_within(num(t), o.grads[name][0], o.grads[name][1], name)
        return y, h, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 7, 8, 9, 16, 31, 64, 100, 255, 256, 257, 500, 513, 1024, 1433, 2049, 4095, 4096])
def test_widths(env, dtype, kind, dim):
    Case(env, 19, dim, dtype, kind).check()


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 5001])
def test_row_counts(env, n):
    for dtype in TYPES:
        Case(env, n, 24, dtype, "layer").check()
        Case(env, n, 260, dtype, "rms").check()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("z,gate,post,res,pre", [c for c in itertools.product([True, False], repeat=5) if c[0] and (c[0] or c[4])]
                         + [(False, False, False, False, True)])
def test_every_part_may_be_absent(env, kind, z, gate, post, res, pre):
    Case(env, 50, 40, "bfloat16", kind, z, gate, post, res, pre).check()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows(env, dtype):
    Case(env, 33, 70, dtype, "layer", layout="strided").check()
    Case(env, 33, 64, dtype, "rms", layout="strided").check()


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_far_from_zero_and_rows_of_one_value(env, kind):
    """Rows around 100 (the mean is taken off before squaring), and rows whose variance
    is zero: eps alone divides."""
    Case(env, 40, 96, "float32", kind, offset=100.0).check()
    c = Case(env, 6, 32, "float32", kind, eps=1e-5)
    for t in (c.x, c.ops["z"]):
        t[2] = 0.0
        t[3] = 2.0
    c.check()


def test_extreme_gates(env):
    torch = env["torch"]
    c = Case(env, 4, 16, "float32")
    c.ops["gate"][0] = 1e4
    c.ops["gate"][1] = -1e4
    c.ops["gate"][2] = float("inf")
    c.ops["gate"][3] = -float("inf")
    y, h, grads = c.run()
    assert torch.equal(y[1], c.x[1]) and torch.equal(y[3], c.x[3])
    assert all(bool(torch.isfinite(t).all()) for t in (y, h) + grads)
    assert not grads[2].any() and not grads[1][1].any()


def test_missing_gradients_and_no_rows(env):
    torch, ops = env["torch"], env["ops"]
    c = Case(env, 20, 24)
    y, h, stats = ops.norm_residual(c.x, want_stats=True, **c.ops)
    zeros = torch.zeros_like(c.x)
    for dy, dh in ((None, c.dh), (c.dy, None)):
        got = ops.norm_residual_bwd(c.x, dy, dh, stats, **c.ops)
        want = ops.norm_residual_bwd(c.x, zeros if dy is None else dy, zeros if dh is None else dh, stats, **c.ops)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    none = Case(env, 0, 24)
    y, h, grads = none.run()
    assert y.shape == h.shape == (0, 24) and all(not t.any() for t in grads)


def test_autograd_and_differences(env):
    torch, ops = env["torch"], env["ops"]
    c = Case(env, 12, 10, kind="layer")
    y, h, want = c.run()
    names = ("z", "gate", "post_weight", "res_scale", "pre_weight")
    leaves = [c.x.clone().requires_grad_(True)] + [c.ops[n].clone().requires_grad_(True) for n in names]
    y2, h2 = ops.norm_residual_autograd(*leaves, kind="layer")
    assert torch.equal(y2.detach(), y) and torch.equal(h2.detach(), h)
    torch.autograd.backward([y2, h2], [c.dy, c.dh])
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    # against central differences of the formulas in 64 bits
    wide = [t.double().cpu().numpy() for t in [c.x] + [c.ops[n] for n in names]]
    dy, dh = c.dy.double().cpu().numpy(), c.dh.double().cpu().numpy()
    rng = np.random.RandomState(3)

    def loss(v):
        o = Oracle(*v, True, 1e-6, U, 0.0)
        return (o.y * dy).sum() + (o.h * dh).sum()

    for i, g in enumerate(want):
        step = rng.standard_normal(wide[i].shape)
        at = lambda s: [v + s * step if j == i else v for j, v in enumerate(wide)]
        slope = (loss(at(1e-6)) - loss(at(-1e-6))) / 2e-6
        terms = g.double().cpu().numpy() * step
        # truncation 1e-12 times third derivatives, cancellation 2^-52 / 1e-6; fp32 sums
        assert abs(slope - terms.sum()) <= 1e-6 * max(1.0, np.abs(terms).sum()) + 500 * U * np.abs(terms).sum()
    # the norm alone, and only one output used
    x = c.x.clone().requires_grad_(True)
    y3, h3 = ops.norm_residual_autograd(x, pre_weight=c.ops["pre_weight"])
    h3.sum().backward()
    assert torch.isfinite(x.grad).all() and torch.equal(y3, x)


def test_same_bits_captured_and_on_two_streams(env):
    torch = env["torch"]
    cases = [Case(env, 3000, 200, "bfloat16", seed=1), Case(env, 500, 2000, "float32", "layer", seed=2)]
    flat = lambda r: [t for t in (r[0], r[1]) + r[2]]
    first = [flat(c.run()) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(flat(c.run()))
        torch.cuda.synchronize()
        for g, f in zip(got, first):
            assert all(torch.equal(a, b) for a, b in zip(g, f))
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = flat(c.run())
        graphs.append((graph, out))
    for turn in range(3):
        for c, (graph, out) in zip(cases, graphs):
            c.x.copy_(torch.randn_like(c.x))
            graph.replay()
            eager = flat(c.run())
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(env):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    x = torch.zeros(4, 8, device=dev)
    w = torch.ones(8, device=dev)
    for bad in (dict(z=x.half()), dict(z=x[:2]), dict(z=x, gate=x[:, :4]), dict(z=x, post_weight=w[:4]), dict(z=x, post_weight=w.half()),
                dict(gate=x), dict(post_weight=w), dict(), dict(z=x, kind="batch"), dict(z=x.t().contiguous().t()[:, :8])):
        with pytest.raises(ValueError):
            ops.norm_residual(x, **bad)
    with pytest.raises(TypeError):
        ops.norm_residual(x.double(), pre_weight=w)
    with pytest.raises(ValueError):
        ops.norm_residual(torch.zeros(2, 4097, device=dev), pre_weight=torch.ones(4097, device=dev))
    with pytest.raises(RuntimeError):
        ops.norm_residual(x.cpu(), pre_weight=w)
    y, h, stats = ops.norm_residual(x, z=x, want_stats=True)
    with pytest.raises(ValueError):
        ops.norm_residual_bwd(x, x, x, stats, z=x)
    with pytest.raises(ValueError):
        ops.norm_residual_bwd(x, x, None, stats[:2], z=x)
