"""The operators together as they are used: a network of attention blocks on a graph
(projections, attention over the neighbours, gated residual norms, masked loss) trained
with the many-tensor AdamW step, against the same network in 64 bits on the host."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

N, F, D, HEADS, KV, CLASSES, BLOCKS = 300, 20, 32, 4, 2, 5, 2
HD = D // HEADS


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    from gcn_amd.sparse import Csr
    assert torch.cuda.is_available()
    dev = torch.device("cuda:0")
    rng = np.random.RandomState(0)
    row, col = rng.randint(0, N, 2500), rng.randint(0, N, 2500)
    row[:700] = 3                                            # a node with many neighbours
    keep = row != 11                                         # a node with none
    row, col = row[keep].astype(np.int32), col[keep].astype(np.int32)
    values = (0.5 * rng.standard_normal(len(row))).astype(np.float32)
    a = Csr.from_coo(row, col, values, (N, N), dev)
    t = lambda *s: torch.from_numpy((rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)).to(dev)
    params = {"in": t(F, D), "out": t(D, CLASSES), "first": torch.ones(D, device=dev)}
    for b in range(BLOCKS):
        params.update({"q%d" % b: t(D, D), "k%d" % b: t(D, KV * HD), "v%d" % b: t(D, KV * HD), "o%d" % b: t(D, D), "g%d" % b: t(D, D),
                       "post%d" % b: torch.ones(D, device=dev), "res%d" % b: torch.full((D,), 0.5, device=dev),
                       "pre%d" % b: torch.ones(D, device=dev)})
    labels = np.eye(CLASSES, dtype=np.float32)[rng.randint(0, CLASSES, N)]
    mask = (rng.rand(N) < 0.4).astype(np.uint8)
    return dict(torch=torch, ops=ops, dev=dev, a=a, row=row, col=col, values=values, x=t(N, F) * 3, params=params,
                labels=torch.from_numpy(labels).to(dev), mask=torch.from_numpy(mask).to(dev), edge=rng)


def _forward(env, params, edge_mask):
    ops = env["ops"]
    y = ops.gemm_autograd(env["x"], params["in"])
    y, h = ops.norm_residual_autograd(y, pre_weight=params["first"])
    for b in range(BLOCKS):
        heads = lambda name, n: ops.gemm_autograd(h, params[name + str(b)]).view(N, n, HD)
        out = ops.attention_autograd(env["a"], heads("q", HEADS), heads("k", KV), heads("v", KV), use_values=True, mask=edge_mask)
        z = ops.gemm_autograd(out.reshape(N, D), params["o%d" % b])
        gate = ops.gemm_autograd(h, params["g%d" % b])
        y, h = ops.norm_residual_autograd(y, z, gate, params["post%d" % b], params["res%d" % b], params["pre%d" % b],
                                          kind="rms" if b else "layer")
    return ops.masked_softmax_xent_autograd(ops.gemm_autograd(h, params["out"]), env["labels"], env["mask"])[0]


def _host(env, params, edge_mask):
    torch = env["torch"]
    row, col = torch.from_numpy(env["row"].astype(np.int64)), torch.from_numpy(env["col"].astype(np.int64))
    on = torch.from_numpy(edge_mask != 0)
    row, col, shift = row[on], col[on], torch.from_numpy(env["values"]).double()[on]

    def norm(t, w, layer):
        if layer:
            t = t - t.mean(1, keepdim=True)
        return t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6) * w

    y = env["x"].double().cpu() @ params["in"]
    h = norm(y, params["first"], False)
    for b in range(BLOCKS):
        q, k, v = [(h @ params[c + str(b)]).view(N, -1, HD) for c in "qkv"]
        k, v = [t.repeat_interleave(HEADS // KV, 1) for t in (k, v)]
        s = (q[row] * k[col]).sum(2) * HD ** -0.5 + shift[:, None]
        w = torch.exp(s - s.detach().max())
        total = torch.zeros(N, HEADS, dtype=torch.double).index_add(0, row, w)
        out = torch.zeros(N, HEADS, HD, dtype=torch.double).index_add(0, row, w[:, :, None] * v[col]) / total.clamp(min=1e-300)[:, :, None]
        z = norm(out.reshape(N, D) @ params["o%d" % b], params["post%d" % b], b == 0)
        y = y + params["res%d" % b] * torch.sigmoid(h @ params["g%d" % b]) * z
        h = norm(y, params["pre%d" % b], b == 0)
    logits = h @ params["out"]
    m = env["mask"].double().cpu()
    loss = -(env["labels"].double().cpu() * torch.log_softmax(logits, 1)).sum(1)
    return (loss * m / m.mean()).mean()


def _edge_mask(seed, n):
    return (np.random.RandomState(seed).rand(n) < 0.85).astype(np.uint8)


def test_training_steps_match_64_bits(env):
    torch, ops = env["torch"], env["ops"]
    names = sorted(env["params"])
    params = {k: env["params"][k].clone().requires_grad_(True) for k in names}
    host = {k: env["params"][k].double().cpu().requires_grad_(True) for k in names}
    leaves = [params[k] for k in names]
    state = ops.adamw_state(leaves)
    moments = {k: [torch.zeros_like(host[k]), torch.zeros_like(host[k])] for k in names}
    for t in range(1, 4):
        em = _edge_mask(t, len(env["row"]))
        loss = _forward(env, params, torch.from_numpy(em).to(env["dev"]))
        grads = torch.autograd.grad(loss, leaves)
        want_loss = _host(env, host, em)
        want = torch.autograd.grad(want_loss, [host[k] for k in names])
        # some forty operations in a row, forward and backward, each within about a
        # hundred roundings of 2^-24 of its largest terms
        tol = 40 * 100 * 2.0 ** -24
        assert abs(float(loss) - float(want_loss)) <= tol * abs(float(want_loss))
        for k, g, w in zip(names, grads, want):
            off = float((g.double().cpu() - w).norm() / w.norm())
            assert off <= tol, (t, k, off)
        with torch.no_grad():
            ops.adamw_step(leaves, [g.contiguous() for g in grads], state, 1e-3, t, weight_decay=0.01)
            # the host's step from the gradients that the device had: an update is as
            # ill-conditioned as its gradient is small
            for i, k in enumerate(names):
                g = grads[i].double().cpu()
                m, v = moments[k]
                m.mul_(0.9).add_(g, alpha=0.1)
                v.mul_(0.999).addcmul_(g, g, value=0.001)
                new = host[k] * (1 - 1e-3 * 0.01) - 1e-3 / (1 - 0.9 ** t) * m / (torch.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
                assert float((params[k].double().cpu() - new).abs().max()) <= 20 * 2.0 ** -24 * (float(host[k].abs().max()) + 1e-2)
                host[k].copy_(params[k].double().cpu())


def test_training_step_captured(env):
    """The whole step (mask drawn, forward, backward, update in 8-bit state) in a HIP
    graph, replayed with eager work between: the weights of the eager loop, bit for bit."""
    torch, ops, dev = env["torch"], env["ops"], env["dev"]
    names, n_edges = sorted(env["params"]), len(env["row"])

    def step(params, state, counter):
        leaves = [params[k] for k in names]
        ops.counter_add(counter, 1)
        mask = ops.bernoulli_mask(n_edges, 0.85, 99, 0, dev, step=counter, step_stride=2 ** 20)
        loss = _forward(env, params, mask)
        grads = torch.autograd.grad(loss, leaves)
        with torch.no_grad():
            ops.adamw_step(leaves, [g.contiguous() for g in grads], state, 1e-3, counter, weight_decay=0.01)
        return loss.detach()

    def fresh():
        params = {k: env["params"][k].clone().requires_grad_(True) for k in names}
        return params, ops.adamw_state([params[k] for k in names], bits=8, seed=4), ops.device_counter(dev, 0)

    eager = fresh()
    losses = [step(*eager) for _ in range(4)]
    side = torch.cuda.Stream()
    warm = fresh()
    with torch.cuda.stream(side):
        step(*warm)
    torch.cuda.synchronize()
    recorded = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(*recorded)
    for t in range(4):
        graph.replay()
        again = float(loss)
        _ = ops.gemm(env["x"], env["params"]["in"])          # eager work between replays
        torch.cuda.synchronize()
        assert again == float(losses[t])
    for k in names:
        assert torch.equal(recorded[0][k], eager[0][k]), k
    assert torch.equal(recorded[1].exp_avg.view(torch.uint8), eager[1].exp_avg.view(torch.uint8))
