"""The AdamW step of tensors so large that it streams past the caches, and of 16-bit
tensors with several tiles a wavefront: the same bits as the same elements stepped in
small calls, which the formulas are tested on."""
import pytest

pytestmark = pytest.mark.gpu

# A step streams from 8.4 M elements and 256 MiB on: weights, gradients and state, 16 to
# 6 bytes an element.
LARGE = {("float32", "float32", 32): 20_000_001, ("float32", "bfloat16", 32): 22_000_003, ("bfloat16", "bfloat16", 32): 24_000_001,
         ("float16", "float32", 32): 22_000_001, ("float32", "float32", 8): 30_000_001, ("float32", "bfloat16", 8): 36_000_002,
         ("bfloat16", "bfloat16", 8): 48_000_003, ("float16", "float32", 8): 36_000_001}


@pytest.fixture(scope="module")
def env():
    import torch
    from gcn_amd import ops
    assert torch.cuda.is_available()
    return dict(torch=torch, ops=ops, dev=torch.device("cuda:0"))


def _part(ops, state, at, n):
    """A state of one tensor that is a part of another's only tensor: the same buffers,
    so the same places and random words."""
    part = object.__new__(ops.AdamWState)
    part.__dict__.update(state.__dict__)
    part.sizes, part.offsets = [n], [at]
    part._table = state._table[:1].copy()
    part._table["state"], part._table["n"] = at, n
    return part


def _same(torch, ops, dev, sizes, param, grad, bits, shift, steps=2):
    """Steps of all tensors at once against the same in calls of 2^20 elements."""
    torch.manual_seed(sum(sizes) % 1000)
    pt, gt = getattr(torch, param), getattr(torch, grad)
    bytes_each = torch.finfo(pt).bits // 8 + torch.finfo(gt).bits // 8 + (2 if bits == 8 else 8)

    def tensors(dtype):
        # `shift` elements off the allocation's alignment
        return [torch.randn(n + shift, device=dev).to(dtype)[shift:] for n in sizes]

    params = tensors(pt)
    twins = [torch.empty(p.numel() + shift, dtype=pt, device=dev)[shift:].copy_(p) for p in params]
    state, twin_state = ops.adamw_state(params, bits, seed=11), ops.adamw_state(twins, bits, seed=11)
    for t in range(1, steps + 1):
        grads = [g * 10.0 ** (1 - t) for g in tensors(gt)]
        ops.adamw_step(params, grads, state, 1e-2, t, weight_decay=0.1)
        for i, (w, g) in enumerate(zip(twins, grads)):
            for at in range(0, w.numel(), 1 << 20):
                n = min(1 << 20, w.numel() - at)
                ops.adamw_step([w[at:at + n]], [g[at:at + n]], _part(ops, twin_state, state.offsets[i] + at, n), 1e-2, t, weight_decay=0.1)
    for x, y in zip(params, twins):
        assert torch.equal(x, y) and torch.isfinite(x).all()
    raw = lambda x: x.view(torch.uint8)
    assert torch.equal(raw(state.exp_avg), raw(twin_state.exp_avg)) and torch.equal(raw(state.exp_avg_sq), raw(twin_state.exp_avg_sq))
    if bits == 8:
        assert torch.equal(state.exp_avg_scale, twin_state.exp_avg_scale) and torch.equal(state.exp_avg_sq_scale, twin_state.exp_avg_sq_scale)
    return sum(sizes) * bytes_each


@pytest.mark.parametrize("param,grad,bits", sorted(LARGE))
@pytest.mark.parametrize("shift", [0, 1])
def test_streamed(env, param, grad, bits, shift):
    n = LARGE[param, grad, bits]
    sizes = [n - 5_000_000, 1021, 5_000_000 - 1021 - 255, 255]       # ends inside a tile, a group of four tiles, one lane's four
    held = _same(env["torch"], env["ops"], env["dev"], sizes, param, grad, bits, shift)
    assert held > 256 << 20


@pytest.mark.parametrize("param,grad", [("bfloat16", "bfloat16"), ("float16", "float32"), ("float32", "float16"), ("bfloat16", "float16")])
@pytest.mark.parametrize("bits", [32, 8])
def test_several_tiles_a_wavefront_in_16_bits(env, param, grad, bits):
    held = _same(env["torch"], env["ops"], env["dev"], [9_000_003, 1021, 5], param, grad, bits, 1)
    assert held <= 256 << 20
