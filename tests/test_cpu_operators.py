"""Refusals of the attention, norm and AdamW entry points that need no GPU: bad
descriptors come back as status codes from the C ABI before anything is launched,
CPU tensors as RuntimeError from the Python ops."""
import ctypes as C

import pytest

PTR = 0x1000          # never followed: every call here is refused


@pytest.fixture(scope="module")
def lib():
    from gcn_amd import _lib
    return _lib.load()


def _csr(n_rows=4, n_cols=5, nnz=6):
    from gcn_amd import _lib
    return _lib.CsrStruct(n_rows, n_cols, nnz, PTR, PTR, PTR, 0, None)


def _attention(a, **kw):
    from gcn_amd import _lib
    f = dict(use_values=0, dtype=_lib.F32, edge_mask=None, mask_index=None, max_row_nnz=0, n_heads=4, n_kv_heads=2, head_dim=8, scale=1.0,
             q=PTR, q_row=32, q_head=8, k=PTR, k_row=16, k_head=8, v=PTR, v_row=16, v_head=8)
    f.update(kw)
    p = _lib.AttentionStruct(a=C.addressof(a), **f)
    p.matrix = a                     # kept alive
    return p


def test_attention_descriptors(lib):
    from gcn_amd import _lib
    a = _csr()
    fwd = lambda p, out=PTR, ws=None, n=0, chunk=None: lib.gcnx_attention_forward(C.byref(p), chunk, out, 32, 8, None, ws, n, None)
    for bad, code in ((dict(dtype=7), _lib.ERR_UNSUPPORTED), (dict(head_dim=0), _lib.ERR_UNSUPPORTED), (dict(head_dim=257), _lib.ERR_UNSUPPORTED),
                      (dict(n_heads=3), _lib.ERR_INVALID_ARG), (dict(n_kv_heads=0), _lib.ERR_INVALID_ARG), (dict(q=None), _lib.ERR_INVALID_ARG),
                      (dict(k=None), _lib.ERR_INVALID_ARG), (dict(q_row=-1), _lib.ERR_INVALID_ARG), (dict(v_head=1 << 30), _lib.ERR_INVALID_ARG)):
        assert fwd(_attention(a, **bad)) == code, bad
    assert fwd(_attention(a), out=None) == _lib.ERR_INVALID_ARG
    assert lib.gcnx_attention_forward(None, None, PTR, 32, 8, None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert fwd(_attention(_csr(n_rows=-1))) == _lib.ERR_INVALID_ARG
    assert fwd(_attention(_csr(n_cols=0))) == _lib.ERR_INVALID_ARG            # nonzeros in an empty matrix
    noval = _csr()
    noval.val = None
    assert fwd(_attention(noval, use_values=1)) == _lib.ERR_INVALID_ARG
    assert lib.gcnx_attention_forward(C.byref(_attention(a)), PTR, PTR, 32, 8, PTR + 4, None, 0, None) == _lib.ERR_INVALID_ARG
    assert fwd(_attention(a), ws=PTR + 8) == _lib.ERR_INVALID_ARG
    # nothing to do is no error, and needs no pointer
    assert fwd(_attention(_csr(0, 5, 0), q=None), out=None) == _lib.OK
    # more workgroups than a launch has: refused on the host
    assert fwd(_attention(_csr((1 << 31) - 2, 5, 6), n_heads=64, n_kv_heads=64, head_dim=256)) == _lib.ERR_UNSUPPORTED
    # long rows need a workspace unless the longest row is known to be short
    big = _csr(10, 10, 5000)
    need = lib.gcnx_attention_workspace_bytes(C.byref(_attention(big)))
    assert need > 0 and lib.gcnx_attention_workspace_bytes(C.byref(_attention(big, max_row_nnz=512))) == 0
    assert fwd(_attention(big)) == _lib.ERR_WORKSPACE
    assert fwd(_attention(big), ws=PTR, n=need - 1, chunk=PTR) == _lib.ERR_WORKSPACE
    assert fwd(_attention(big), ws=PTR, n=need) == _lib.ERR_INVALID_ARG        # no chunk table
    assert fwd(_attention(big, max_row_nnz=200)) == _lib.ERR_INVALID_ARG       # needed without pieces too
    assert b"attention" in lib.gcnx_last_error()


def test_attention_backward_descriptors(lib):
    from gcn_amd import _lib
    a, at = _csr(), _csr(5, 4, 6)

    def bwd(p, t=at, out=PTR, stats=PTR, dout=PTR, dq=PTR, dk=PTR, dv=PTR, ws=PTR, n=1 << 40, midx=None):
        return lib.gcnx_attention_backward(C.byref(p), PTR, C.byref(t), PTR, midx, 0, out, 32, 8, stats, dout, 32, 8, dq, dk, dv, ws, n, None)

    p = _attention(a)
    assert bwd(p, t=_csr(4, 5, 6)) == _lib.ERR_INVALID_ARG                     # not the transpose
    assert bwd(p, stats=None) == _lib.ERR_INVALID_ARG
    assert bwd(p, dout=None) == _lib.ERR_INVALID_ARG
    assert bwd(p, dk=None) == _lib.ERR_INVALID_ARG                             # dv without dk
    assert bwd(p, dq=None, dk=None, dv=None) == _lib.ERR_INVALID_ARG
    assert bwd(_attention(a, edge_mask=PTR)) == _lib.ERR_INVALID_ARG           # no index of the mask in the transpose
    assert bwd(p, ws=None, n=0) == _lib.ERR_WORKSPACE
    assert lib.gcnx_attention_backward_workspace_bytes(C.byref(p), 0) >= 4 * 4 * 16


def _norm(**kw):
    from gcn_amd import _lib
    f = dict(n=3, dim=8, dtype=_lib.F32, layer=0, eps=1e-6, x=PTR, x_ld=8, z=PTR, z_ld=8, gate=PTR, gate_ld=8, post_weight=PTR, res_scale=PTR,
             pre_weight=PTR)
    f.update(kw)
    return _lib.NormResidualStruct(**f)


def test_norm_descriptors(lib):
    from gcn_amd import _lib
    fwd = lambda p, y=PTR, h=PTR, ld=8, stats=None: lib.gcnx_norm_residual_forward(C.byref(p), y, ld, h, ld, stats, None)
    for bad, code in ((dict(dtype=3), _lib.ERR_UNSUPPORTED), (dict(dim=0), _lib.ERR_UNSUPPORTED), (dict(dim=4097), _lib.ERR_UNSUPPORTED),
                      (dict(n=-1), _lib.ERR_INVALID_ARG), (dict(x=None), _lib.ERR_INVALID_ARG), (dict(z=None), _lib.ERR_INVALID_ARG),
                      (dict(z=None, gate=None, post_weight=None, res_scale=None, pre_weight=None), _lib.ERR_INVALID_ARG),
                      (dict(x_ld=-8), _lib.ERR_INVALID_ARG)):
        assert fwd(_norm(**bad)) == code, bad
    assert fwd(_norm(), y=None) == _lib.ERR_INVALID_ARG
    assert fwd(_norm(), h=None) == _lib.ERR_INVALID_ARG
    assert fwd(_norm(), ld=7) == _lib.ERR_INVALID_ARG
    assert fwd(_norm(), stats=PTR + 4) == _lib.ERR_INVALID_ARG
    assert fwd(_norm(n=0, x=None)) == _lib.OK
    bwd = lambda p, dh=PTR, stats=PTR, dgate=PTR, dpre=PTR, ws=PTR, n=1 << 40: lib.gcnx_norm_residual_backward(
        C.byref(p), PTR, 8, dh, 8, stats, PTR, PTR, dgate, PTR, PTR, dpre, ws, n, None)
    assert bwd(_norm(gate=None)) == _lib.ERR_INVALID_ARG                       # a gradient of what is not there
    assert bwd(_norm(), dh=None) == _lib.ERR_INVALID_ARG
    assert bwd(_norm(pre_weight=None), dpre=None) == _lib.ERR_INVALID_ARG
    assert bwd(_norm(), stats=None) == _lib.ERR_INVALID_ARG
    assert bwd(_norm(), n=16) == _lib.ERR_WORKSPACE


def test_adamw_descriptors(lib):
    from gcn_amd import _lib

    def step(n_tensors=1, tensor=None, **kw):
        f = dict(w_dtype=_lib.F32, g_dtype=_lib.F32, state_bits=32, exp_avg=PTR, exp_avg_sq=PTR, exp_avg_scale=None, exp_avg_sq_scale=None,
                 lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8, t=1, t_dev=None, seed=0)
        f.update(kw)
        t = dict(w=PTR, grad=PTR, n=5, state=0, weight_decay=0.0)
        t.update(tensor or {})
        table = (_lib.AdamWTensorStruct * 1)(_lib.AdamWTensorStruct(**t))
        return lib.gcnx_adamw_step(C.byref(_lib.AdamWStruct(**f)), n_tensors, table, None, 0, None)

    for bad, code in ((dict(w_dtype=9), _lib.ERR_UNSUPPORTED), (dict(g_dtype=-1), _lib.ERR_UNSUPPORTED), (dict(state_bits=16), _lib.ERR_UNSUPPORTED),
                      (dict(t=0), _lib.ERR_INVALID_ARG), (dict(beta1=1.0), _lib.ERR_INVALID_ARG), (dict(beta2=-0.1), _lib.ERR_INVALID_ARG),
                      (dict(eps=-1.0), _lib.ERR_INVALID_ARG), (dict(exp_avg=None), _lib.ERR_INVALID_ARG), (dict(exp_avg_sq=PTR + 4), _lib.ERR_INVALID_ARG),
                      (dict(state_bits=8), _lib.ERR_INVALID_ARG), (dict(t_dev=PTR), _lib.ERR_WORKSPACE)):
        assert step(**bad) == code, bad
    for bad in (dict(w=None), dict(grad=None), dict(n=-1), dict(state=100), dict(state=-256)):
        assert step(tensor=bad) == _lib.ERR_INVALID_ARG, bad
    assert step(tensor=dict(n=1 << 40)) == _lib.ERR_UNSUPPORTED
    assert step(n_tensors=-1) == _lib.ERR_INVALID_ARG
    assert step(n_tensors=0) == _lib.OK
    assert step(tensor=dict(n=0, w=None, grad=None)) == _lib.OK


def test_structs_have_the_header_s_layout(tmp_path):
    """Offsets of every field of the ctypes mirrors against the C compiler's."""
    import os
    import subprocess
    from gcn_amd import _lib
    root = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
    pairs = (("gcnx_attention", _lib.AttentionStruct), ("gcnx_norm_residual", _lib.NormResidualStruct),
             ("gcnx_adamw_tensor", _lib.AdamWTensorStruct), ("gcnx_adamw", _lib.AdamWStruct))
    lines = []
    for name, mirror in pairs:
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f[0], name, f[0]) for f in mirror._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include "gcnx.h"\nint main(void) { %s return 0; }\n' % "\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)])
    want = {}
    for name, mirror in pairs:
        want[name] = C.sizeof(mirror)
        want.update(("%s.%s" % (name, f[0]), getattr(mirror, f[0]).offset) for f in mirror._fields_)
    got = dict(line.rsplit(" ", 1) for line in subprocess.check_output([str(exe)], text=True).splitlines())
    assert {k: int(v) for k, v in got.items()} == want
    assert _lib.ADAMW_BLOCK == 256 and _lib.ADAMW_WORKSPACE_BYTES == 256


def test_ops_refuse_cpu_tensors():
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from gcn_amd import ops
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError):
        ops.norm_residual(x, pre_weight=torch.ones(8))
    with pytest.raises(RuntimeError):
        ops.adamw_state([x])

    class Pattern(object):
        n_rows = n_cols = 2

    with pytest.raises(RuntimeError):
        ops.attention(Pattern(), x.view(2, 1, 8), x.view(2, 1, 8), x.view(2, 1, 8))


def test_a_mask_s_index_on_one_side_is_enough(lib):
    """Either the matrix or its transpose may hold the nonzeros in the mask's order (the
    call goes on to the next check, the workspace); both cannot."""
    from gcn_amd import _lib
    a, at = _csr(), _csr(5, 4, 6)

    def bwd(midx, t_midx):
        p = _attention(a, edge_mask=PTR, mask_index=midx)
        return lib.gcnx_attention_backward(C.byref(p), PTR, C.byref(at), PTR, t_midx, 0, PTR, 32, 8, PTR, PTR, 32, 8, PTR, PTR, PTR, None, 0, None)

    assert bwd(None, None) == _lib.ERR_INVALID_ARG
    assert bwd(PTR, None) == bwd(None, PTR) == bwd(PTR, PTR) == _lib.ERR_WORKSPACE


def test_gradients_of_no_rows_and_of_no_columns(lib):
    """Empty gradients have no address: nothing to do is no error."""
    from gcn_amd import _lib

    def bwd(rows, cols, **kw):
        a, at = _csr(rows, cols, 0), _csr(cols, rows, 0)
        f = dict(out=PTR, stats=PTR, dout=PTR, dq=None, dk=None, dv=None)
        f.update(kw)
        return lib.gcnx_attention_backward(C.byref(_attention(a)), PTR, C.byref(at), PTR, None, 0, f["out"], 32, 8, f["stats"], f["dout"],
                                           32, 8, f["dq"], f["dk"], f["dv"], PTR, 1 << 40, None)

    for shape in ((0, 0), (0, 5), (4, 0)):
        assert bwd(*shape) == _lib.OK, shape
    assert bwd(4, 5) == _lib.ERR_INVALID_ARG                       # there are some: asked for none of them
    assert bwd(4, 0, dk=PTR) == _lib.ERR_INVALID_ARG               # dk without dv
