"""tf.train.AdamWOptimizer over variables that come, go and are loaded while others
train: every variable's moments are its own."""
import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import gcn_amd.tfcompat as tf
    assert torch.cuda.is_available()
    return dict(torch=torch, tf=tf, dev=torch.device("cuda:0"))


def _variables(env, *shapes):
    tf = env["tf"]
    rng = np.random.RandomState(len(shapes))
    out = [tf.Variable(rng.standard_normal(s).astype(np.float32), name="w%d" % i) for i, s in enumerate(shapes)]
    for v in out:
        v.initialize()
    return out


def _grads(env, variables, seed):
    torch = env["torch"]
    rng = np.random.RandomState(seed)
    return [torch.from_numpy(rng.standard_normal(v.static_shape).astype(np.float32)).to(env["dev"]) for v in variables]


def _moments(opt, v):
    return [x.clone() for x in opt.moments(v)]


@pytest.mark.parametrize("bits", [32, 8])
def test_loading_one_variable_leaves_the_others(env, bits):
    torch, tf = env["torch"], env["tf"]
    tf.reset_default_graph()
    a, b, c = _variables(env, (40, 30), (17,), (5, 100))
    opt = tf.train.AdamWOptimizer(0.01, state_bits=bits)
    for t in range(5):
        opt.apply([a, b, c], _grads(env, [a, b, c], t))
    before = [_moments(opt, v) for v in (a, c)]
    b.load(np.ones(17, np.float32))
    opt.apply([a, b, c], [None, None, None])             # nothing to do but to notice
    for was, v in zip(before, (a, c)):
        for x, y in zip(was, opt.moments(v)):
            assert torch.equal(x, y) and x.any()
    assert not any(x.any() for x in opt.moments(b))
    # the loaded one starts over, at the count that has been reached
    g = _grads(env, [b], 9)[0]
    opt.apply([a, b, c], [None, g, None])
    m, v = opt.moments(b)
    if bits == 32:
        assert torch.allclose(m, 0.1 * g, rtol=1e-6, atol=0) and torch.allclose(v, 0.001 * g * g, rtol=1e-4, atol=0)
    for was, x in zip(before, (a, c)):
        assert all(torch.equal(p, q) for p, q in zip(was, opt.moments(x)))


@pytest.mark.parametrize("bits", [32, 8])
def test_variables_that_come_later(env, bits):
    """A second model initialised in the middle changes not a bit of the first one's
    training, and trains itself; neither do steps with a part of the variables."""
    torch, tf = env["torch"], env["tf"]
    results = []
    for second in (False, True):
        tf.reset_default_graph()
        a, b = _variables(env, (64, 33), (9, 9))
        opt = tf.train.AdamWOptimizer(0.01, state_bits=bits, seed=4)
        late = []
        for t in range(8):
            if second and t == 3:
                late = _variables(env, (20,), (300, 2), (7,))
            if second and t == 6:
                late += _variables(env, (11,))
            if second and t == 5:                        # lists by turns
                opt.apply([b], _grads(env, [a, b], t)[1:])
                opt.step -= 1
                opt._step_dev -= 1
                opt.apply([a] + late, _grads(env, [a, b], t)[:1] + _grads(env, late, t))
            else:
                opt.apply([a, b] + late, _grads(env, [a, b], t) + _grads(env, late, t))
        results.append([a.tensor.detach().clone(), b.tensor.detach().clone()] + _moments(opt, a) + _moments(opt, b))
        if second:
            for v in late:
                assert all(x.any() for x in opt.moments(v)) and not np.array_equal(v.numpy(), v._init_value)
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_state_of_variables_that_are_gone_is_freed(env):
    torch, tf = env["torch"], env["tf"]
    tf.reset_default_graph()
    opt = tf.train.AdamWOptimizer(0.01)
    keep = _variables(env, (8,))
    sizes = []
    for t in range(6):
        big = _variables(env, (1 << 20,))
        opt.apply(keep + big, _grads(env, keep + big, t))
        del big
        tf.reset_default_graph()
        gc.collect()
        torch.cuda.synchronize()
        sizes.append(torch.cuda.memory_allocated())
    assert max(sizes[1:]) <= sizes[0] + (1 << 16) and all(x.any() for x in opt.moments(keep[0]))


def test_the_same_variable_twice(env):
    tf = env["tf"]
    tf.reset_default_graph()
    a, = _variables(env, (8,))
    with pytest.raises(ValueError):
        tf.train.AdamWOptimizer(0.01).apply([a, a], _grads(env, [a, a], 0))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_load_in_a_session(env, graph, bits):
    """A weight loaded between runs of a session, eager and recorded: the formulas in
    64 bits, the loaded variable's moments from zero."""
    tf = env["tf"]
    tf.reset_default_graph()
    a = tf.Variable(np.full((4, 8), 0.5, np.float32), name="a")
    b = tf.Variable(np.full((8, 3), -0.25, np.float32), name="b")
    loss = tf.Node(lambda run, x, y: (x @ y).square().sum(), (a, b))
    op = tf.train.AdamWOptimizer(learning_rate=0.05, weight_decay=0.02, state_bits=bits).minimize(loss)
    sess = tf.Session(config={"hip_graph": graph})
    sess.run(tf.global_variables_initializer())
    w = {"a": np.full((4, 8), 0.5), "b": np.full((8, 3), -0.25)}
    mom = {k: [np.zeros_like(v), np.zeros_like(v)] for k, v in w.items()}
    for t in range(1, 13):
        if t == 7:
            a.load(np.full((4, 8), 0.4, np.float32))
            w["a"][:] = np.float32(0.4)
            mom["a"][0][:] = mom["a"][1][:] = 0
        sess.run([op, loss])
        p = w["a"] @ w["b"]
        grads = {"a": 2 * p @ w["b"].T, "b": 2 * w["a"].T @ p}
        for k in w:
            m, v = mom[k]
            m[:] = 0.9 * m + 0.1 * grads[k]
            v[:] = 0.999 * v + 0.001 * grads[k] ** 2
            w[k] = w[k] * (1 - 0.05 * 0.02) - 0.05 / (1 - 0.9 ** t) * m / (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
        # fp32 sums of 8 products, a moment's roundings: far below a thousandth of a step of 0.05
        assert np.abs(a.numpy() - w["a"]).max() <= 1e-4 and np.abs(b.numpy() - w["b"]).max() <= 1e-4, t
        if bits == 8:      # what is held is rounded by chance: the next step goes on from there
            w = {"a": a.numpy().astype(np.float64), "b": b.numpy().astype(np.float64)}
            opt = op.optimizer
            mom = {k: [x.double().cpu().numpy().reshape(w[k].shape) for x in opt.moments(var)] for k, var in (("a", a), ("b", b))}
    assert sess.graph_replays == (12 - 2 if graph else 0)       # the first runs before and after the load are eager
    sess.close()


def test_first_step_under_a_capture_is_refused(env):
    """A recording that zeroed moments or set the count would do so at every replay."""
    torch, tf = env["torch"], env["tf"]
    tf.reset_default_graph()
    a, = _variables(env, (1000,))
    g = _grads(env, [a], 0)
    opt = tf.train.AdamWOptimizer(0.01)
    torch.cuda.synchronize()

    def record():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.apply([a], g)
        return graph

    with pytest.raises(RuntimeError, match="run a step before the capture"):
        record()
    opt.apply([a], g)
    a.load(np.zeros(1000, np.float32))
    with pytest.raises(RuntimeError, match="run a step before the capture"):
        record()
    opt.apply([a], g)
    with pytest.raises(ValueError):
        opt.moments(_variables(env, (3,))[0])
    twin, = _variables(env, (1000,))
    twin.load(a.numpy())
    m, v = _moments(opt, a)
    graph = record()
    other = tf.train.AdamWOptimizer(0.01)
    other.apply([twin], [None])
    other._groups[0].state.exp_avg[:1000], other._groups[0].state.exp_avg_sq[:1000] = m, v
    other._step_dev.copy_(opt._step_dev)
    for _ in range(3):
        graph.replay()
        other.apply([twin], g)
        torch.cuda.synchronize()
        assert torch.equal(a.tensor, twin.tensor)
        assert all(torch.equal(x, y) for x, y in zip(opt.moments(a), other.moments(twin)))


def test_no_memory_for_another_optimizer_s_moments(env):
    """A step with 8-bit state holds the weights and 2 + 1/32 bytes an element."""
    torch, tf = env["torch"], env["tf"]
    tf.reset_default_graph()
    gc.collect()
    n = 1 << 22
    small, = _variables(env, (256,))
    tf.train.AdamWOptimizer(0.01, state_bits=8).apply([small], _grads(env, [small], 0))      # loads the code
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    big, = _variables(env, (n,))
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 4 * n + 4096
    opt = tf.train.AdamWOptimizer(0.01, state_bits=8)
    opt.apply([big], [torch.ones(n, device=env["dev"])])
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 4 * n + 2 * n + n // 32 + 8192
    # the plain optimizer's are there when it asks, and start over with the variable
    adam = tf.train.AdamOptimizer(0.01)
    adam.apply([small], _grads(env, [small], 1))
    assert small.adam_m.any() and small.adam_v.any() and small.adam_m is small.adam_m
    small.load(np.zeros(256, np.float32))
    assert small.adam_m.shape == (256,) and not small.adam_m.any() and not small.adam_v.any()
    # recorded as a first step they would be zeroed by every replay
    fresh, = _variables(env, (16,))
    g = _grads(env, [fresh], 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the stream capture"):
        with torch.cuda.graph(graph):
            adam.apply([fresh], g)


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_moments_stay_where_they_are(env, bits):
    """One variable of a recorded step is gone and another has come: the recording goes
    on over the memory that it knows, bit for bit as without all that."""
    torch, tf = env["torch"], env["tf"]
    tf.reset_default_graph()
    pairs = []
    for _ in range(2):
        both = _variables(env, (1000,), (700,))
        opt = tf.train.AdamWOptimizer(0.01, state_bits=bits)
        opt.apply(both, _grads(env, both, 0))
        pairs.append((opt, both))
    (opt, both), (other, twins) = pairs
    grads = _grads(env, both, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.apply(both, grads)
    a, state = both[0], opt._groups[0].state
    for turn in range(5):
        graph.replay()
        other.apply(twins, grads)
        if turn == 1:
            del pairs, both
            tf.reset_default_graph()
            gc.collect()
            late = _variables(env, (900,))
            opt.apply(late, _grads(env, late, 3))
            opt._step_dev -= 1
            assert opt._groups[0].state is state and len(opt._groups) == 2
        torch.cuda.synchronize()
        assert torch.equal(a.tensor, twins[0].tensor)
        assert all(torch.equal(x, y) for x, y in zip(opt.moments(a), other.moments(twins[0])))
