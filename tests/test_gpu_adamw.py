"""The many-tensor AdamW step against the formulas: 64 bits for the weights, the
fp32 operations one by one for the 8-bit state (bit for bit)."""
import numpy as np
import pytest

from attention_oracle import U

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]
BLOCK = 256


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    assert torch.cuda.is_available()
    return dict(torch=torch, ops=ops, dev=torch.device("cuda:0"))


def philox_words(quads, t, seed):
    """Philox4x32-10 of the counters (quads, t) under the 64-bit key: [len, 4] words."""
    quads = np.asarray(quads, np.uint64)
    m = np.uint64(0xffffffff)
    c = [quads & m, quads >> np.uint64(32), np.full_like(quads, t & 0xffffffff), np.full_like(quads, t >> 32)]
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return np.stack(c, 1).astype(np.uint32)


def scale_of(x):
    top = np.abs(x.reshape(-1, BLOCK)).max(1)
    f, e = np.frexp(top)
    e = np.maximum(np.where(top == 0, 0, e + (f > 0.875)) - 9, -100)
    return np.ldexp(np.float32(1), e).astype(np.float32)


def to_grid(x, scale, u, positive):
    x = (x.reshape(-1, BLOCK) / scale[:, None]).reshape(-1)
    size = np.abs(x)
    _, e = np.frexp(np.maximum(size, np.float32(2.0 ** -6)))
    step = np.ldexp(np.float32(1), e - 4).astype(np.float32)
    size = np.minimum(np.floor(size / step + u) * step, np.float32(448))
    if positive:
        size = np.where(x > 0, np.maximum(size, np.float32(2.0 ** -9)), size)
    return np.copysign(size, x).astype(np.float32)


class Host(object):
    """fp32 arithmetic operation by operation, state laid out as AdamWState."""

    def __init__(self, sizes, bits, seed):
        self.offsets, total = [], 0
        for n in sizes:
            self.offsets.append(total)
            total += -(-n // BLOCK) * BLOCK
        self.sizes, self.bits, self.seed = sizes, bits, seed
        self.m, self.v = np.zeros(total, np.float32), np.zeros(total, np.float32)    # 8 bits: m and sqrt(v) as the codes stand for
        self.ms = self.vs = np.ones(total // BLOCK, np.float32)

    def step(self, ws, gs, lr, t, b1, b2, eps, decay):
        f = np.float32
        w, g = np.zeros_like(self.m), np.zeros_like(self.m)
        live = np.zeros(len(self.m), bool)
        for i, (at, n) in enumerate(zip(self.offsets, self.sizes)):
            if gs[i] is not None:
                w[at:at + n], g[at:at + n] = ws[i].reshape(-1), gs[i].reshape(-1)
                live[at:at + -(-n // BLOCK) * BLOCK] = True
        v = self.v if self.bits == 32 else self.v * self.v
        m = self.m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * g) * f(1 - b2)
        root = np.sqrt(v)
        # the weights in 64 bits from the fp32 moments
        m64, v64 = m.astype(np.float64), v.astype(np.float64)
        new = w * (1 - lr * decay) - lr / (1 - b1 ** t) * m64 / (np.sqrt(v64) / np.sqrt(1 - b2 ** t) + eps)
        self.size = np.abs(w) + np.abs(new - w)
        if self.bits == 32:
            self.m, self.v = np.where(live, m, self.m), np.where(live, v, self.v)
        else:
            words = philox_words(np.arange(len(m) // 4), t, self.seed).reshape(-1)
            ms, vs = scale_of(m), scale_of(root)
            mq = to_grid(m, ms, (words & 0xffff).astype(f) * f(2.0 ** -16), False)
            vq = to_grid(root, vs, (words >> 16).astype(f) * f(2.0 ** -16), True)
            rows = live.reshape(-1, BLOCK)[:, 0]
            self.ms, self.vs = np.where(rows, ms, self.ms), np.where(rows, vs, self.vs)
            self.mc, self.vc = mq, vq
            self.m = np.where(live, mq * np.repeat(ms, BLOCK), self.m)
            self.v = np.where(live, vq * np.repeat(vs, BLOCK), self.v)
        return [new[at:at + n] if gs[i] is not None else ws[i].reshape(-1) for i, (at, n) in enumerate(zip(self.offsets, self.sizes))], \
            [self.size[at:at + n] for at, n in zip(self.offsets, self.sizes)]


def _held(state):
    """m and v (sqrt(v) in 8 bits) as the state's codes stand for them."""
    m, v = state.exp_avg.float(), state.exp_avg_sq.float()
    if state.bits == 8:
        m, v = m * state.exp_avg_scale.repeat_interleave(BLOCK), v * state.exp_avg_sq_scale.repeat_interleave(BLOCK)
    return m.cpu().numpy(), v.cpu().numpy()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad", [("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"), ("bfloat16", "bfloat16"),
                                        ("bfloat16", "float32"), ("float16", "float16"), ("float16", "float32"), ("float16", "bfloat16")])
@pytest.mark.parametrize("sizes", [[1], [3, 256, 257], [1433 * 16, 16 * 7], [5, 0, 1023, 1024, 4097, 70000] + list(range(1, 90))])
def test_steps(env, bits, param, grad, sizes):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    rng = np.random.RandomState(len(sizes) + bits)
    dt = getattr(torch, param)
    params = [torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dev).to(dt) for n in sizes]
    state = ops.adamw_state(params, bits=bits, seed=77)
    host = Host(sizes, bits, 77)
    half = torch.finfo(dt).eps / 2
    for t in range(1, 5):
        grads = [torch.from_numpy((rng.standard_normal(n) * 10.0 ** rng.uniform(-6, 2)).astype(np.float32)).to(dev).to(getattr(torch, grad))
                 for n in sizes]
        if t == 3 and len(sizes) > 1:
            grads[1] = None                          # stays, its state too
        before = [p.float().cpu().numpy() for p in params]
        decay = 0.1 if t != 2 else [0.01 * (i % 3) for i in range(len(sizes))]
        flat = np.zeros_like(host.m)
        for i, at in enumerate(host.offsets):
            flat[at:at + sizes[i]] = decay if t != 2 else decay[i]
        want, size = host.step(before, [g.float().cpu().numpy() if g is not None else None for g in grads], 0.01, t, 0.9, 0.99, 1e-8, flat)
        ops.adamw_step(params, grads, state, 0.01, t, 0.9, 0.99, 1e-8, decay)
        m, v = _held(state)
        assert np.array_equal(m, host.m) and np.array_equal(v, host.v)
        if bits == 8:
            assert np.array_equal(state.exp_avg_scale.cpu().numpy(), host.ms) and np.array_equal(state.exp_avg_sq_scale.cpu().numpy(), host.vs)
        for p, w, s in zip(params, want, size):
            got = p.double().cpu().numpy()
            # one rounding each: keep, the product with it, the root's product, eps, the
            # reciprocal (2), its product, the step and its product, the difference
            bound = 12 * U * s + half * np.maximum(np.abs(w), torch.finfo(dt).tiny) * (1 + 1e-6) + 1e-37
            assert np.all(np.abs(got - w) <= bound), (t, np.max(np.abs(got - w) / bound))
    if bits == 32:
        m, v = state.moments(0)
        assert torch.equal(m, state.exp_avg[:sizes[0]])


def test_large_tensors_take_several_tiles(env):
    """Enough elements for four tiles a wavefront, at every place of a tensor's end."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    rng = np.random.RandomState(5)
    for bits in (32, 8):
        sizes = [9000001, 1021, 5000 * 1024 // 3]
        params = [torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dev) for n in sizes]
        grads = [torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dev) for n in sizes]
        state, host = ops.adamw_state(params, bits=bits, seed=9), Host(sizes, bits, 9)
        want, size = host.step([p.cpu().numpy() for p in params], [g.cpu().numpy() for g in grads], 0.01, 1, 0.9, 0.999, 1e-8, 0.1)
        ops.adamw_step(params, grads, state, 0.01, 1, weight_decay=0.1)
        m, v = _held(state)
        assert np.array_equal(m, host.m) and np.array_equal(v, host.v)
        for p, w, s in zip(params, want, size):
            assert np.all(np.abs(p.double().cpu().numpy() - w) <= 13 * U * s)


def test_unaligned_tensors_and_neighbours(env):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    rng = np.random.RandomState(6)
    room = torch.from_numpy(rng.standard_normal(4000).astype(np.float32)).to(dev)
    before = room.clone()
    params = [room[1:1000], room[1003:1004], room[1005:3333]]
    grads = [torch.from_numpy(rng.standard_normal(p.numel() + 3).astype(np.float32)).to(dev).to(torch.bfloat16)[3:] for p in params]
    for bits in (32, 8):
        state = ops.adamw_state(params, bits=bits)
        ops.adamw_step(params, grads, state, 0.01, 1)
        aligned = [before[1:1000].clone(), before[1003:1004].clone(), before[1005:3333].clone()]
        ops.adamw_step(aligned, [g.clone() for g in grads], ops.adamw_state(aligned, bits=bits), 0.01, 1)
        for p, a in zip(params, aligned):
            assert torch.equal(p, a)
        touched = torch.zeros(4000, dtype=torch.bool, device=dev)
        for lo, hi in ((1, 1000), (1003, 1004), (1005, 3333)):
            touched[lo:hi] = True
        assert torch.equal(room[~touched], before[~touched])
        room.copy_(before)


def test_rounding_by_chance_keeps_the_mean(env):
    """One block per draw: the mean of what the codes stand for is the value."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    draws = 4096
    g = np.linspace(0.013, 1.0, BLOCK).astype(np.float32)
    grad = torch.from_numpy(np.tile(g, draws)).to(dev)
    params = [torch.zeros(draws * BLOCK, device=dev)]
    state = ops.adamw_state(params, bits=8, seed=3)
    ops.adamw_step(params, [grad], state, 0.0, 1)
    m, root = _held(state)
    for got, value in ((m, g * 0.1), (root, np.sqrt(g.astype(np.float64) ** 2 * 1e-3))):
        got = got.reshape(draws, BLOCK).astype(np.float64)
        step = np.maximum(np.abs(got).max(0) - np.abs(got).min(0), 1e-12)          # two neighbours of the grid
        # a mean of `draws` values that differ by a step at most: 6 standard deviations of half a step; 2^-17 of a step from u's 16 bits
        assert np.all(np.abs(got.mean(0) - value) <= step * (6 * 0.5 / np.sqrt(draws) + 2.0 ** -16))


def test_not_finite_elements_stay_alone(env):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    for bits in (32, 8):
        params = [torch.ones(600, device=dev)]
        grad = torch.full((600,), 0.5, device=dev)
        grad[7], grad[300] = float("nan"), float("inf")
        state = ops.adamw_state(params, bits=bits)
        ops.adamw_step(params, [grad], state, 0.01, 1)
        m, v = state.moments(0)
        bad = torch.zeros(600, dtype=torch.bool, device=dev)
        bad[7] = bad[300] = True
        assert torch.isfinite(params[0][~bad]).all() and torch.isfinite(m[~bad]).all() and torch.isfinite(v[~bad]).all()
        assert not torch.isfinite(m[bad]).any() and not torch.isfinite(v[bad]).any()
        assert float((m[~bad] - 0.05).abs().max()) <= 0.05 / 8


def test_device_counter_and_capture(env):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    for bits in (32, 8):
        start = [torch.randn(5000, device=dev), torch.randn(77, device=dev)]
        grads = [torch.randn(5000, device=dev), torch.randn(77, device=dev)]
        a, b = [p.clone() for p in start], [p.clone() for p in start]
        sa, sb = ops.adamw_state(a, bits=bits, seed=5), ops.adamw_state(b, bits=bits, seed=5)
        counter = ops.device_counter(dev, 0)
        graph = torch.cuda.CUDAGraph()
        ops.adamw_step(b, grads, sb, 1e-2, 1)             # loads the code before the capture
        for p, s in zip(b, start):
            p.copy_(s)
        sb.exp_avg.view(torch.uint8).zero_()
        sb.exp_avg_sq.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.counter_add(counter, 1)
            ops.adamw_step(b, grads, sb, 1e-2, counter)
        for t in range(1, 5):
            for g in grads:
                g.copy_(torch.randn_like(g))
            graph.replay()
            ops.adamw_step(a, grads, sa, 1e-2, t)
            torch.cuda.synchronize()
            for x, y in zip(a, b):
                # the two terms of the step come from the host's and the device's pow
                assert torch.allclose(x, y, rtol=0, atol=float(4 * U * (x.abs().max() + 1)))
            assert torch.equal(sa.exp_avg.view(torch.uint8), sb.exp_avg.view(torch.uint8))
            assert torch.equal(sa.exp_avg_sq.view(torch.uint8), sb.exp_avg_sq.view(torch.uint8))


def test_optimizer_in_a_session(env):
    """tf.train.AdamWOptimizer on a two-variable loss, eager and recorded, against
    the formulas; weight-decay terms of the loss are gradients."""
    import gcn_amd.tfcompat as tf
    torch = env["torch"]
    for bits in (32, 8):
        results = []
        for graph in (False, True):
            tf.reset_default_graph()
            tf.set_random_seed(1)
            a = tf.Variable(np.full((4, 8), 0.5, np.float32), name="a")
            b = tf.Variable(np.full((8, 3), -0.25, np.float32), name="b")
            loss = tf.Node(lambda run, x, y: (x @ y).square().sum(), (a, b)) + 0.1 * tf.nn.l2_loss(a)
            opt = tf.train.AdamWOptimizer(learning_rate=0.05, weight_decay=0.02, state_bits=bits)
            op = opt.minimize(loss)
            sess = tf.Session(config={"hip_graph": graph})
            sess.run(tf.global_variables_initializer())
            for _ in range(6):
                sess.run([op, loss])
            results.append((a.numpy(), b.numpy()))
        for x, y in zip(*results):
            assert np.allclose(x, y, rtol=0, atol=1e-6)
        w = {"a": np.full((4, 8), 0.5), "b": np.full((8, 3), -0.25)}
        mom = {k: [np.zeros_like(v), np.zeros_like(v)] for k, v in w.items()}
        for t in range(1, 7):
            p = w["a"] @ w["b"]
            grads = {"a": 2 * p @ w["b"].T + 0.1 * w["a"], "b": 2 * w["a"].T @ p}
            for k in w:
                m, v = mom[k]
                m[:] = 0.9 * m + 0.1 * grads[k]
                v[:] = 0.999 * v + 0.001 * grads[k] ** 2
                w[k] = w[k] * (1 - 0.05 * 0.02) - 0.05 / (1 - 0.9 ** t) * m / (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
        # 8 bits: a moment is a step of 1/8 off at most, a weight by that share of five steps of 0.05
        tol = 1e-4 if bits == 32 else 5 * 0.05 * 0.3
        assert np.abs(results[0][0] - w["a"]).max() <= tol and np.abs(results[0][1] - w["b"]).max() <= tol


def test_refusals(env):
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    a, b = torch.zeros(8, device=dev), torch.zeros(9, device=dev)
    with pytest.raises(ValueError):
        ops.adamw_state([])
    with pytest.raises(ValueError):
        ops.adamw_state([a], bits=4)
    with pytest.raises(ValueError):
        ops.adamw_state([a, b.half()])
    with pytest.raises(TypeError):
        ops.adamw_state([a.double()])
    with pytest.raises(RuntimeError):
        ops.adamw_state([a.cpu()])
    st = ops.adamw_state([a, b])
    for params, grads in (([a], [a]), ([a, b], [a]), ([b, a], [b, a]), ([a, b], [a, b.half()]), ([a, b], [a, torch.zeros(18, device=dev)[::2]])):
        with pytest.raises(ValueError):
            ops.adamw_step(params, grads, st, 0.1, 1)
    with pytest.raises(TypeError):
        ops.adamw_step([a, b], [a.double(), b.double()], st, 0.1, 1)
    with pytest.raises(ValueError):
        ops.adamw_step([a, a.view(8)], [a, a], ops.adamw_state([a, a]), 0.1, 1)
    flat = torch.zeros(17, device=dev)
    with pytest.raises(ValueError):
        ops.adamw_step([flat[8:16], flat[:9]], [a, b], st, 0.1, 1)
    ops.adamw_step([flat[9:], flat[:9]], [a, b], st, 0.1, 1)                    # side by side
    with pytest.raises(ValueError):
        ops.adamw_step([a, b], [a, b], st, 0.1, torch.zeros(1, device=dev))
    from gcn_amd._lib import GcnxError
    with pytest.raises(GcnxError):
        ops.adamw_step([a, b], [a, b], st, 0.1, 0)
    with pytest.raises(GcnxError):
        ops.adamw_step([a, b], [a, b], st, 0.1, 1, beta1=1.0)
    assert ops.adamw_step([a, b], [None, None], st, 0.1, 1) == [a, b]
