"""Python entry points of the HIP kernels + their autograd glue.

torch is used for tensor ownership, streams and the autograd tape; every
product, reduction, loss and update below runs in ``libgcnhip.so`` through
ctypes.  What the drop-in layer path (``gcn_amd/layers.py``) leaves to torch's
own element-wise kernels, all of them off the measured path: the concatenation
of the per-support weights of a Chebyshev layer (``torch.cat``, once per step),
a layer's optional bias add, a relu that cannot be fused into the product that
feeds it (``torch.relu``), the ``x.repeat`` of the featureless multi-support
case and the ``part(k) - b2`` of the opt-in Clenshaw recurrence.  The large-graph
engine (``gcn_amd/engine.py``) uses none of them.
All functions raise on CPU tensors -- there is no fallback path.
"""
import contextlib
import ctypes as C

import numpy as np
import torch

from . import _lib
from .sparse import Csr, WORKSPACE, _ptr, _stream


def _check_dense(t, name):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise RuntimeError("%s must be a CUDA (ROCm) tensor; gcn_amd has no CPU path" % name)
    if t.dtype != torch.float32:
        raise TypeError("%s must be float32, got %s" % (name, t.dtype))
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError("%s must be a row-major 2-D tensor" % name)


def _written(*tensors):
    """Counts a kernel's write to tensors that the caller holds, as torch counts its own
    in-place operations: a backward pass that saved one of them refuses to run on what
    is there now."""
    torch.autograd.graph.increment_version(tensors)


# ------------------------------------------------------------------------ SpMM
def spmm(a, b, out=None, alpha=1.0, beta=0.0, mask=None, mask_scale=1.0, relu=False, b2=None,
         dropout=None, sign_bits=None, dropout_rows=None):
    """``out = act(alpha * A' @ b + beta * out)`` with ``A`` a :class:`Csr`.
    ``mask`` (uint8, in the order of the tuple ``A`` was built from) applies
    sparse dropout to the values on the fly.  Replaces ``dot(x, y, sparse=True)``
    (reference gcn/layers.py:30-33) and ``sparse_dropout`` (:21-27).
    With ``b2`` the dense operand is the row-wise concatenation ``[b; b2]``
    without being assembled (local rows + halo rows of a partitioned run).
    ``dropout=(keep, seed, offset, ld, col0)`` applies dropout to the output in
    the epilogue (element (r, c) has Philox index offset + r*ld + col0 + c).
    ``sign_bits`` (int32 [n_rows, width / 32]) also receives the sign pattern of
    the stored output, the layout :func:`pack_sign_bits` writes
    (:func:`spmm_supports_sign_bits`).  ``dropout_rows`` (int32 [n_rows]): output
    row r draws the dropout mask of row ``dropout_rows[r]`` instead of r -- for a
    matrix that holds a subset of the rows of A_hat next to each other
    (gcnx_spmm_csr_rows_f32)."""
    lib = _lib.load()
    _check_dense(b, "b")
    rows_b2 = 0
    if b2 is not None:
        _check_dense(b2, "b2")
        if b2.shape[1] != b.shape[1] or b2.device != b.device:
            raise ValueError("b and b2 differ in width or device")
        rows_b2 = b2.shape[0]
    if b.shape[0] + rows_b2 != a.n_cols:
        raise ValueError("shape mismatch: A is %s, operand has %d rows" % (a.shape, b.shape[0] + rows_b2))
    if b.device != a.device:
        raise ValueError("A and b live on different devices")
    width = b.shape[1]
    if out is None:
        if beta != 0.0:
            raise ValueError("beta != 0 needs an existing out")
        out = torch.empty((a.n_rows, width), dtype=torch.float32, device=b.device)
    else:
        _check_dense(out, "out")
        if tuple(out.shape) != (a.n_rows, width):
            raise ValueError("out has shape %s, expected %s" % (tuple(out.shape), (a.n_rows, width)))
        _written(out)
    midx = None
    if mask is not None:
        a.check_mask(mask)
        midx = a.input_index
    drop = None
    if dropout is not None and dropout[0] < 1.0:
        keep, seed, offset, ld, col0 = dropout
        drop = C.byref(_lib.DropoutStruct(float(keep), int(seed) & (2 ** 64 - 1), int(offset), int(ld),
                                          int(col0)))
    if dropout_rows is not None and drop is None:
        dropout_rows = None
    if dropout_rows is not None:
        dr = dropout_rows
        if mask is not None or dr.dtype != torch.int32 or dr.dim() != 1 or dr.numel() != a.n_rows or \
                not dr.is_contiguous() or dr.device != a.device:
            raise ValueError("dropout_rows: contiguous int32 [n_rows] on A's device, no value mask")
    if sign_bits is not None:
        sb = sign_bits
        if mask is not None or sb.dtype != torch.int32 or sb.dim() != 2 or sb.shape[0] != a.n_rows or \
                sb.shape[1] * 32 < width or sb.stride(1) != 1 or sb.device != a.device or \
                not spmm_supports_sign_bits(width):
            raise ValueError("sign_bits: int32 [n_rows, width / 32] on A's device, width % 32 == 0, no mask")
        _written(sb)
        if dropout_rows is None:
            with torch.cuda.device(a.device):
                need = lib.gcnx_spmm_workspace_bytes(a.struct_ref(), width)
                ws = WORKSPACE.get(need, a.device)
                _lib.check(lib.gcnx_spmm_csr_signs_f32(
                    a.struct_ref(), _ptr(a.chunk_row), _ptr(b), b.stride(0),
                    _ptr(b2 if rows_b2 else None), b2.stride(0) if rows_b2 else 0, b.shape[0],
                    _ptr(out), out.stride(0), width, float(alpha), float(beta), 1 if relu else 0, drop,
                    _ptr(sb), sb.stride(0), _ptr(ws), ws.numel(), _stream()))
            return out
    if dropout_rows is not None:
        with torch.cuda.device(a.device):
            need = lib.gcnx_spmm_workspace_bytes(a.struct_ref(), width)
            ws = WORKSPACE.get(need, a.device)
            _lib.check(lib.gcnx_spmm_csr_rows_f32(
                a.struct_ref(), _ptr(a.chunk_row), _ptr(b), b.stride(0),
                _ptr(b2 if rows_b2 else None), b2.stride(0) if rows_b2 else 0, b.shape[0],
                _ptr(out), out.stride(0), width, float(alpha), float(beta), 1 if relu else 0, drop,
                _ptr(dropout_rows), _ptr(sign_bits), sign_bits.stride(0) if sign_bits is not None else 0,
                _ptr(ws), ws.numel(), _stream()))
        return out
    with torch.cuda.device(a.device):
        need = lib.gcnx_spmm_workspace_bytes(a.struct_ref(), width)
        ws = WORKSPACE.get(need, a.device)
        _lib.check(lib.gcnx_spmm_csr_split_f32(
            a.struct_ref(), _ptr(a.chunk_row), _ptr(b), b.stride(0),
            _ptr(b2 if rows_b2 else None), b2.stride(0) if rows_b2 else 0, b.shape[0],
            _ptr(out), out.stride(0), width, float(alpha), float(beta), _ptr(mask), _ptr(midx),
            float(mask_scale), 1 if relu else 0, drop, _ptr(ws), ws.numel(), _stream()))
    return out


def spmm_supports_sign_bits(width):
    """Whether ``spmm(..., sign_bits=...)`` is served for this operand width."""
    return bool(_lib.load().gcnx_spmm_signs_supported(int(width)))


def spmm_supports_factored(width, inner):
    """Whether ``spmm_factored`` is served for this operand width / inner size."""
    return bool(_lib.load().gcnx_spmm_factored_supported(int(width), int(inner)))


def spmm_factored(a, d, w, gate_bits, gate_scale=1.0, trans_w=False, out=None, d2=None, gate_bits2=None):
    """``out = A @ G`` with ``G = where(bit, gate_scale * (D @ op(W)), 0)`` formed
    on the fly (never stored).  ``d`` [n_local_cols, inner] and ``gate_bits``
    (int32 [n_local_cols, width/32]) cover the first columns of ``a``; ``d2`` /
    ``gate_bits2`` the remaining ones (halo rows).  ``w`` is [inner, width], or
    [width, inner] with ``trans_w``."""
    lib = _lib.load()
    _check_dense(d, "d")
    _check_dense(w, "w")
    inner = d.shape[1]
    width = w.shape[0] if trans_w else w.shape[1]
    if (w.shape[1] if trans_w else w.shape[0]) != inner:
        raise ValueError("inner dimensions differ: d %s, w %s" % (tuple(d.shape), tuple(w.shape)))
    if gate_bits.dtype != torch.int32 or gate_bits.shape[0] != d.shape[0] or gate_bits.shape[1] * 32 < width:
        raise ValueError("gate_bits must be int32 [rows of d, ceil(width / 32)]")
    split = d.shape[0]
    if d2 is not None and d2.shape[0] > 0:
        _check_dense(d2, "d2")
        if gate_bits2 is None or gate_bits2.dtype != torch.int32 or gate_bits2.shape[0] != d2.shape[0] or \
                gate_bits2.shape[1] * 32 < width or d2.shape[1] != inner:
            raise ValueError("d2 / gate_bits2 do not match d / gate_bits")
        n_cols = split + d2.shape[0]
    else:
        d2, gate_bits2, n_cols = None, None, split
    if n_cols != a.n_cols:
        raise ValueError("operand rows (%d) != matrix columns (%d)" % (n_cols, a.n_cols))
    if out is None:
        out = torch.empty((a.n_rows, width), dtype=torch.float32, device=d.device)
    elif tuple(out.shape) != (a.n_rows, width) or out.stride(1) != 1:
        raise ValueError("out has shape %s, expected %s" % (tuple(out.shape), (a.n_rows, width)))
    else:
        _written(out)
    with torch.cuda.device(d.device):
        need = lib.gcnx_spmm_workspace_bytes(a.struct_ref(), width)
        ws = WORKSPACE.get(need, d.device)
        _lib.check(lib.gcnx_spmm_csr_factored_f32(
            a.struct_ref(), _ptr(a.chunk_row), _ptr(d), d.stride(0), _ptr(gate_bits), gate_bits.stride(0),
            _ptr(d2), d2.stride(0) if d2 is not None else 0, _ptr(gate_bits2),
            gate_bits2.stride(0) if gate_bits2 is not None else 0, split, _ptr(w), w.stride(0), int(trans_w),
            inner, float(gate_scale), _ptr(out), out.stride(0), width, _ptr(ws), ws.numel(), _stream()))
    return out


class _SpmmFn(torch.autograd.Function):
    """y = act(A' @ b).  Gradient w.r.t. b only: the sparse operands of the
    reference are placeholders, no gradient reaches their values
    (reference gcn/models.py:58)."""

    @staticmethod
    def forward(ctx, b, a, mask, mask_scale, relu):
        y = spmm(a, b, mask=mask, mask_scale=mask_scale, relu=relu)
        ctx.a = a
        ctx.mask = mask
        ctx.mask_scale = mask_scale
        ctx.relu = relu
        if relu:
            ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        dy = dy.contiguous()
        if ctx.relu:
            (y,) = ctx.saved_tensors
            dy = relu_dropout_bwd(y, dy)
        db = spmm(ctx.a.transpose(), dy, mask=ctx.mask, mask_scale=ctx.mask_scale)
        return db, None, None, None, None


def spmm_autograd(a, b, mask=None, mask_scale=1.0, relu=False):
    return _SpmmFn.apply(b, a, mask, mask_scale, relu)


class _SpmmAddFn(torch.autograd.Function):
    """y = act(alpha * A @ b + c) in one launch (c is copied into the output and
    accumulated onto).  Gradients: d b = alpha * A^T dy', d c = dy', with dy' the
    relu-gated dy."""

    @staticmethod
    def forward(ctx, b, c, a, alpha, relu):
        y = c.clone(memory_format=torch.contiguous_format)
        spmm(a, b, out=y, alpha=alpha, beta=1.0, relu=relu)
        ctx.a = a
        ctx.alpha = alpha
        ctx.relu = relu
        if relu:
            ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        dy = dy.contiguous()
        if ctx.relu:
            (y,) = ctx.saved_tensors
            dy = relu_dropout_bwd(y, dy)
        db = spmm(ctx.a.transpose(), dy, alpha=ctx.alpha) if ctx.needs_input_grad[0] else None
        return db, (dy if ctx.needs_input_grad[1] else None), None, None, None


def spmm_add_autograd(a, b, c, alpha=1.0, relu=False):
    return _SpmmAddFn.apply(b.contiguous(), c, a, float(alpha), relu)


# ------------------------------------------------------------------------ GEMM
def gemm(a, b, trans_a=False, trans_b=False, out=None, alpha=1.0, beta=0.0, relu=False, gate=None,
         gate_scale=1.0, a_dropout=None, a_dropout_rows=None, gate_bits=None, dropout=None, sign_bits=None):
    """``out = act(alpha * op(a) @ op(b) + beta * out)``, fp32.  Replaces
    ``dot(x, y, sparse=False)`` (reference gcn/layers.py:35).  With ``gate``
    (same shape as out) the epilogue is ``gate > 0 ? out * gate_scale : 0``: the
    backward of relu + dropout fused into the product that feeds it.
    ``a_dropout=(keep, seed, offset)`` applies dropout to ``a`` (as stored,
    row-major with its own row length) while it is read, so dropout(a) is never
    written (MFMA shapes only); with ``a_dropout_rows`` (int32, one per stored row
    of ``a``) row i draws the mask of row ``a_dropout_rows[i]`` (``a`` holds a
    gathered subset of the rows the mask is defined on; with a transposed ``a``
    only where :func:`gemm_supports_a_dropout_rows_t` says so).  ``gate_bits`` (uint32 /
    int32 [M, ceil(N/32)]) is the gate as one bit per element
    (:func:`pack_sign_bits`).  ``dropout=(keep, seed, offset, ld, col0)`` applies
    dropout to the output behind the activation, as in :func:`spmm`; with it,
    ``sign_bits`` (int32 [M, N/32]) receives the sign pattern of the stored
    output (fused epilogue only)."""
    lib = _lib.load()
    _check_dense(a, "a")
    _check_dense(b, "b")
    if sign_bits is not None and (dropout is None or dropout[0] >= 1.0):
        raise ValueError("sign_bits needs the fused output dropout (dropout with keep < 1)")
    M, K = (a.shape[1], a.shape[0]) if trans_a else (a.shape[0], a.shape[1])
    Kb, N = (b.shape[1], b.shape[0]) if trans_b else (b.shape[0], b.shape[1])
    if K != Kb:
        raise ValueError("inner dimensions differ: %d vs %d" % (K, Kb))
    if out is None:
        if beta != 0.0:
            raise ValueError("beta != 0 needs an existing out")
        out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    else:
        _check_dense(out, "out")
        if tuple(out.shape) != (M, N):
            raise ValueError("out has shape %s, expected %s" % (tuple(out.shape), (M, N)))
        _written(out)
    with torch.cuda.device(a.device):
        need = lib.gcnx_gemm_workspace_bytes(int(trans_a), int(trans_b), M, N, K)
        ws = WORKSPACE.get(need, a.device)
        if dropout is not None and dropout[0] < 1.0:
            if gate is not None or gate_bits is not None or (a_dropout is not None and a_dropout[0] < 1.0) \
                    or beta != 0.0:
                raise ValueError("output dropout excludes gate, gate_bits, a_dropout and beta")
            keep, seed, offset, ld, col0 = dropout
            fused = bool(lib.gcnx_gemm_relu_dropout_supported(int(trans_a), int(trans_b), M, N, K)) and \
                out.stride(0) % 4 == 0 and out.data_ptr() % 16 == 0 and a.stride(0) % 4 == 0 and \
                a.data_ptr() % 16 == 0 and (trans_b or N <= 32 or (b.stride(0) % 4 == 0 and b.data_ptr() % 16 == 0)) \
                and int(offset) % 4 == 0 and int(ld) % 4 == 0 and int(col0) % 4 == 0
            if sign_bits is not None:
                # sign words of the stored output straight from the fused epilogue
                if not fused or N % 32 or sign_bits.dtype != torch.int32 or tuple(sign_bits.shape) != (M, N // 32) \
                        or sign_bits.stride(1) != 1:
                    raise ValueError("sign_bits: int32 [M, N / 32], fused output dropout only (see "
                                     "gemm_supports_output_dropout), N % 32 == 0")
                _written(sign_bits)
                d = _lib.DropoutStruct(float(keep), int(seed) & (2 ** 64 - 1), int(offset), int(ld), int(col0))
                _lib.check(lib.gcnx_gemm_relu_dropout_signs_f32(
                    int(trans_a), int(trans_b), M, N, K, _ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(out),
                    out.stride(0), float(alpha), float(beta), 1 if relu else 0, C.byref(d), _ptr(sign_bits),
                    sign_bits.stride(0), _ptr(ws), ws.numel(), _stream()))
            elif fused:
                d = _lib.DropoutStruct(float(keep), int(seed) & (2 ** 64 - 1), int(offset), int(ld), int(col0))
                _lib.check(lib.gcnx_gemm_relu_dropout_f32(int(trans_a), int(trans_b), M, N, K, _ptr(a), a.stride(0),
                                                          _ptr(b), b.stride(0), _ptr(out), out.stride(0),
                                                          float(alpha), float(beta), 1 if relu else 0, C.byref(d),
                                                          _ptr(ws), ws.numel(), _stream()))
            else:
                # shapes outside the tall MFMA kernel: the product, then the same mask in place
                if int(ld) != N or int(col0) != 0 or not out.is_contiguous():
                    raise ValueError("unfused output dropout needs ld == N, col0 == 0 and a contiguous out")
                _lib.check(lib.gcnx_gemm_f32(int(trans_a), int(trans_b), M, N, K, _ptr(a), a.stride(0),
                                             _ptr(b), b.stride(0), _ptr(out), out.stride(0), float(alpha),
                                             0.0, 1 if relu else 0, _ptr(ws), ws.numel(), _stream()))
                dropout_philox(out.view(-1), keep, seed, offset, out=out.view(-1))
        elif a_dropout is not None and a_dropout[0] < 1.0:
            if gate is not None or relu or not a.is_contiguous():
                raise ValueError("a_dropout excludes gate / relu and needs a contiguous a")
            if gate_bits is not None:
                raise ValueError("a_dropout excludes gate_bits")
            keep, seed, offset = a_dropout
            d = _lib.DropoutStruct(float(keep), int(seed) & (2 ** 64 - 1), int(offset), a.shape[1], 0)
            if a_dropout_rows is not None:
                r = a_dropout_rows
                if r.dtype != torch.int32 or r.numel() != a.shape[0] or not r.is_contiguous() or r.device != a.device:
                    raise ValueError("a_dropout_rows: one contiguous int32 per stored row of a")
                if trans_a:
                    if trans_b:
                        raise ValueError("a_dropout_rows with a transposed a needs a plain b")
                    _lib.check(lib.gcnx_gemm_dropout_at_rows_f32(M, N, K, _ptr(a), a.stride(0), C.byref(d), _ptr(r),
                                                                 _ptr(b), b.stride(0), _ptr(out), out.stride(0),
                                                                 float(alpha), float(beta), _ptr(ws), ws.numel(),
                                                                 _stream()))
                else:
                    _lib.check(lib.gcnx_gemm_dropout_a_rows_f32(int(trans_b), M, N, K, _ptr(a), a.stride(0),
                                                                C.byref(d), _ptr(r), _ptr(b), b.stride(0),
                                                                _ptr(out), out.stride(0), float(alpha),
                                                                float(beta), _ptr(ws), ws.numel(), _stream()))
            else:
                _lib.check(lib.gcnx_gemm_dropout_a_f32(int(trans_a), int(trans_b), M, N, K, _ptr(a),
                                                       a.stride(0), C.byref(d), _ptr(b), b.stride(0),
                                                       _ptr(out), out.stride(0), float(alpha), float(beta),
                                                       _ptr(ws), ws.numel(), _stream()))
        elif gate_bits is not None:
            gb = gate_bits
            if gate is not None or relu:
                raise ValueError("gate_bits excludes gate / relu")
            if gb.dtype not in (torch.int32, torch.uint32) or gb.dim() != 2 or gb.shape[0] != M or \
                    gb.shape[1] * 32 < N or gb.stride(1) != 1 or gb.device != a.device:
                raise ValueError("gate_bits must be a 32-bit integer tensor [M, ceil(N/32)]")
            _lib.check(lib.gcnx_gemm_bitgated_f32(int(trans_a), int(trans_b), M, N, K, _ptr(a),
                                                  a.stride(0), _ptr(b), b.stride(0), _ptr(out),
                                                  out.stride(0), float(alpha), float(beta), _ptr(gb),
                                                  gb.stride(0), float(gate_scale), _ptr(ws),
                                                  ws.numel(), _stream()))
        elif gate is not None:
            _check_dense(gate, "gate")
            if tuple(gate.shape) != (M, N) or relu:
                raise ValueError("gate must have the shape of out and excludes relu")
            _lib.check(lib.gcnx_gemm_gated_f32(int(trans_a), int(trans_b), M, N, K, _ptr(a),
                                               a.stride(0), _ptr(b), b.stride(0), _ptr(out),
                                               out.stride(0), float(alpha), float(beta), _ptr(gate),
                                               gate.stride(0), float(gate_scale), _ptr(ws),
                                               ws.numel(), _stream()))
        else:
            _lib.check(lib.gcnx_gemm_f32(int(trans_a), int(trans_b), M, N, K, _ptr(a), a.stride(0),
                                         _ptr(b), b.stride(0), _ptr(out), out.stride(0), float(alpha),
                                         float(beta), 1 if relu else 0, _ptr(ws), ws.numel(), _stream()))
    return out


def dense_arith(mode=None):
    """Arithmetic of the large dense products on this thread: 0 = exactly split
    operands on the bf16 matrix pipe (fp32 accuracy, default), 1 = fp32-input MFMA
    chains only.  Returns the previous mode; ``None`` only reads."""
    return int(_lib.load().gcnx_dense_arith(-1 if mode is None else int(mode)))


def dropout_rows_philox(x, row_ids, keep, seed, offset, out=None):
    """Dropout of gathered rows: row i of ``x`` draws the mask of row
    ``row_ids[i]`` of the [*, W] matrix the mask is defined on (element index
    ``offset + row_ids[i] * W + c``)."""
    lib = _lib.load()
    _check_dense(x, "x")
    if row_ids.dtype != torch.int32 or row_ids.numel() != x.shape[0] or not row_ids.is_contiguous() or \
            row_ids.device != x.device:
        raise ValueError("row_ids: one contiguous int32 per row of x")
    if out is None:
        out = torch.empty_like(x)
    else:
        _check_dense(out, "out")
        if out.shape != x.shape:
            raise ValueError("out must have the shape of x")
        _written(out)
    with torch.cuda.device(x.device):
        _lib.check(lib.gcnx_dropout_rows_philox_f32(x.shape[0], x.shape[1], _ptr(x), x.stride(0), _ptr(row_ids),
                                                    float(keep), int(seed) & (2 ** 64 - 1), int(offset),
                                                    _ptr(out), out.stride(0), _stream()))
    return out


def pack_sign_bits(x, rows=None, out=None):
    """int32 [n, ceil(W/32)]: bit (c % 32) of word (i, c // 32) is set iff
    ``x[rows[i] if rows is not None else i, c] > 0``."""
    lib = _lib.load()
    _check_dense(x, "x")
    n = int(rows.numel()) if rows is not None else x.shape[0]
    width = x.shape[1]
    words = (width + 31) // 32
    if rows is not None and (rows.dtype != torch.int32 or not rows.is_contiguous() or rows.device != x.device):
        raise ValueError("rows must be a contiguous int32 tensor on the device of x")
    if out is None:
        out = torch.empty((n, words), dtype=torch.int32, device=x.device)
    elif out.dtype != torch.int32 or tuple(out.shape) != (n, words) or out.stride(1) != 1:
        raise ValueError("out must be int32 [n, ceil(W/32)]")
    else:
        _written(out)
    with torch.cuda.device(x.device):
        _lib.check(lib.gcnx_pack_sign_bits_f32(n, _ptr(rows) if rows is not None else None, _ptr(x),
                                               x.stride(0), width, _ptr(out), out.stride(0), _stream()))
    return out


def gemm_supports_output_dropout(trans_a, M, N, K):
    """Whether ``gemm(..., dropout=...)`` is fused into the product's epilogue
    for this shape (otherwise the mask is applied by a second kernel)."""
    return bool(_lib.load().gcnx_gemm_relu_dropout_supported(int(trans_a), 0, int(M), int(N), int(K)))


def gemm_supports_a_dropout(trans_a, M, N, K):
    """Whether ``gemm(..., a_dropout=...)`` is served for this shape."""
    return bool(_lib.load().gcnx_gemm_dropout_a_supported(int(trans_a), 0, int(M), int(N), int(K)))


class _GemmFn(torch.autograd.Function):
    """y = act(a @ b) with both gradients.  The arithmetic mode of the large
    products (:func:`dense_arith`) is a per-thread setting of the library and
    torch runs backward on a thread of its own, so the mode the forward product
    ran under is kept with the node and put in force around the backward
    products: forward and backward of one product use the same arithmetic."""

    @staticmethod
    def forward(ctx, a, b, relu):
        ctx.arith = dense_arith()
        y = gemm(a, b, relu=relu)
        ctx.relu = relu
        if relu:
            ctx.save_for_backward(a, b, y)
        else:
            ctx.save_for_backward(a, b)
        return y

    @staticmethod
    def backward(ctx, dy):
        dy = dy.contiguous()
        if ctx.relu:
            a, b, y = ctx.saved_tensors
            dy = relu_dropout_bwd(y, dy)
        else:
            a, b = ctx.saved_tensors
        before = dense_arith(ctx.arith)
        try:
            da = gemm(dy, b, trans_b=True) if ctx.needs_input_grad[0] else None
            db = gemm(a, dy, trans_a=True) if ctx.needs_input_grad[1] else None
        finally:
            dense_arith(before)
        return da, db, None


def gemm_supports_a_dropout_rows_t(M, N, K):
    """Whether ``gemm(a, b, trans_a=True, a_dropout=..., a_dropout_rows=...)`` is
    served for an [M, N] output summed over K stored rows."""
    return bool(_lib.load().gcnx_gemm_dropout_at_rows_supported(int(M), int(N), int(K)))


def gemm_autograd(a, b, relu=False):
    return _GemmFn.apply(a, b, relu)


# ------------------------------------------------------------------- attention
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _check_heads(t, name, rows, heads, dim, dtype, device):
    """The strides of ``t`` as [rows, heads, dim] with contiguous head vectors."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError("%s must be a CUDA (ROCm) tensor; gcn_amd has no CPU path" % name)
    stride = t.stride()
    if t.shape == (rows, heads, dim) and t.dtype == dtype and t.device == device and (stride[2] == 1 or dim == 1 or not t.numel()):
        return stride
    if t.dtype != dtype or t.device != device:
        raise ValueError("%s differs from q in dtype or device" % name)
    raise ValueError("%s must be [%d, %d, %d] with contiguous head vectors, got %s with strides %s" %
                     (name, rows, heads, dim, tuple(t.shape), stride))


def _attention_struct(a, q, k, v, scale, use_values, mask):
    """The descriptor of a call; its tensors are checked."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise RuntimeError("q must be a CUDA (ROCm) tensor; gcn_amd has no CPU path")
    dtype, dev = q.dtype, q.device
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError("q must be float32, bfloat16 or float16, got %s" % (dtype,))
    if q.dim() != 3 or not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("q and k must be [rows, heads, head_dim]")
    _, heads, dim = q.shape
    kv = k.shape[1]
    qs = _check_heads(q, "q", a.n_rows, heads, dim, dtype, dev)
    ks = _check_heads(k, "k", a.n_cols, kv, dim, dtype, dev)
    vs = _check_heads(v, "v", a.n_cols, kv, dim, dtype, dev)
    if dev != a.device:
        raise ValueError("the matrix and q live on different devices")
    if kv < 1 or heads < 1 or heads % kv:
        raise ValueError("%d query heads cannot share %d key heads" % (heads, kv))
    if not 1 <= dim <= 256:
        raise ValueError("head_dim must be 1..256, got %d" % dim)
    mask_ptr = index_ptr = None
    if mask is not None:
        a.check_mask(mask)
        mask_ptr = mask.data_ptr()
        if a.input_index is not None:
            index_ptr = a.input_index.data_ptr()
    return _lib.AttentionStruct(
        a.struct_address, 1 if use_values else 0, code, mask_ptr, index_ptr, a.max_row_nnz(), heads, kv, dim,
        dim ** -0.5 if scale is None else scale, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
        vs[1])


_HERE = contextlib.nullcontext()


def _on(device):
    """Makes ``device`` current for the launches of a ``with`` block."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _stream_of(device):
    """The current stream of ``device`` as the C ABI takes it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _at(t):
    """Address of a tensor or None."""
    return None if t is None else t.data_ptr()


def _like(t):
    """An uninitialised contiguous tensor of t's shape and type (the cheapest call for it)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _scratch(nbytes, device):
    # from torch's allocator, which orders the memory by stream and owns it in a
    # capture: two streams, or two recorded graphs, never share it
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def attention(a, q, k, v, scale=None, use_values=False, mask=None, out=None, want_stats=False):
    """Softmax attention of every row of ``a`` (a :class:`Csr`) over its columns:
    ``out[i, h] = sum_j softmax_j(scale * <q[i, h], k[j, h']> + a[i, j]) * v[j, h']``
    with the matrix values as logit shifts only if ``use_values``; query head ``h``
    reads key head ``h' = h // (heads / kv_heads)``.  ``q`` [n_rows, heads, head_dim],
    ``k`` and ``v`` [n_cols, kv_heads, head_dim], float32, bfloat16 or float16, any
    strides below 2^30 between head vectors; ``scale`` defaults to ``head_dim ** -0.5``.
    ``mask`` (uint8, in the order of the tuple ``a`` was built from, ``a.input_nnz``
    bytes) takes the edges with 0 out of the softmax, as a value of -inf does; a row
    with no edge left gives zeros.  ``out`` (default: a new tensor) must not share memory with
    ``q``, ``k`` or ``v``.  With ``want_stats`` returns ``(out, stats)``, what
    :func:`attention_bwd` needs.  The longest row of ``a`` is looked up at its first
    use (a host synchronisation; skipped under a stream capture, where it is taken as
    unknown: the same result but for the order of sums).  The attention-weighted
    sibling of :func:`spmm`
    (reference gcn/layers.py:219 sums the neighbours with fixed weights)."""
    lib = _lib.load()
    p = _attention_struct(a, q, k, v, scale, use_values, mask)
    dev = q.device
    fresh = out is None
    if fresh:
        out = _like(q)
        os = out.stride()
    else:
        os = _check_heads(out, "out", a.n_rows, q.shape[1], q.shape[2], q.dtype, dev)
        if any(s == 0 and n > 1 for s, n in zip(os, out.shape)):
            raise ValueError("out must be [n_rows, heads, head_dim] of distinct elements")
    stats = torch.empty((a.n_rows, q.shape[1], 2), dtype=torch.float32, device=dev) if want_stats else None
    with _on(dev):
        need = lib.gcnx_attention_workspace_bytes(C.byref(p))
        ws = _scratch(need, dev)
        _lib.check(lib.gcnx_attention_forward(C.byref(p), a.chunk_row.data_ptr(), out.data_ptr(), os[0], os[1], _at(stats), _at(ws),
                                              need, _stream_of(dev)))
    if not fresh:
        _written(out)
    return (out, stats) if want_stats else out


def attention_bwd(a, q, k, v, out, stats, d_out, scale=None, use_values=False, mask=None, need_q=True, need_kv=True):
    """``(dq, dk, dv)`` of :func:`attention` for the gradient ``d_out`` of its output,
    from its ``out`` and ``stats`` (the probabilities are formed again, edge by
    edge).  The gradients of shared key heads are summed over the query heads that
    share them.  ``need_q`` / ``need_kv`` False leaves those gradients out (None).
    Uses the transpose of ``a``, built at its first use: before a stream capture."""
    lib = _lib.load()
    p = _attention_struct(a, q, k, v, scale, use_values, mask)
    dev = q.device
    n_rows, heads, dim = q.shape
    os = _check_heads(out, "out", n_rows, heads, dim, q.dtype, dev)
    gs = _check_heads(d_out, "d_out", n_rows, heads, dim, q.dtype, dev)
    if stats.dtype != torch.float32 or stats.shape != (n_rows, heads, 2) or not stats.is_contiguous() or \
            stats.device != dev:
        raise ValueError("stats must be what attention(..., want_stats=True) returned")
    if not need_q and not need_kv:
        return None, None, None
    if a._t is None and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("attention_bwd under a stream capture: build a.transpose() before it")
    at = a.transpose() if use_values or a._t is None else a._t        # its values may be old ones where they are not read
    longest = at.max_row_nnz()
    dq = _like(q) if need_q else None
    dk = dv = None
    if need_kv:
        dk, dv = _like(k), _like(v)
    with _on(dev):
        need = lib.gcnx_attention_backward_workspace_bytes(C.byref(p), longest)
        ws = _scratch(need, dev)
        _lib.check(lib.gcnx_attention_backward(
            C.byref(p), a.chunk_row.data_ptr(), at.struct_ref(), at.chunk_row.data_ptr(),
            _at(at.input_index) if mask is not None else None, longest, out.data_ptr(), os[0], os[1], stats.data_ptr(),
            d_out.data_ptr(), gs[0], gs[1], _at(dq), _at(dk), _at(dv), _at(ws), need, _stream_of(dev)))
    return dq, dk, dv


class _AttentionFn(torch.autograd.Function):
    """Gradients w.r.t. q, k, v; none reaches the matrix values or the mask."""

    @staticmethod
    def forward(ctx, q, k, v, a, scale, use_values, mask):
        out, stats = attention(a, q, k, v, scale, use_values, mask, want_stats=True)
        ctx.save_for_backward(q, k, v, out, stats, mask, a.val if use_values and not a.val.is_inference() else None)
        ctx.how = (a, scale, use_values)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, out, stats, mask, _values = ctx.saved_tensors       # the values: refused here if written since
        a, scale, use_values = ctx.how
        if d_out.stride(2) != 1 and d_out.shape[2] > 1:
            d_out = d_out.contiguous()
        dq, dk, dv = attention_bwd(a, q, k, v, out, stats, d_out, scale, use_values, mask, ctx.needs_input_grad[0],
                                   ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return dq, dk if ctx.needs_input_grad[1] else None, dv if ctx.needs_input_grad[2] else None, None, None, None, None


def attention_autograd(a, q, k, v, scale=None, use_values=False, mask=None):
    """:func:`attention` on the autograd tape."""
    return _AttentionFn.apply(q, k, v, a, scale, use_values, mask)


# ----------------------------------------------------------------------- norms
def _check_rows(t, name, like=None):
    """The leading dimension of row-major [n, dim]."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError("%s must be a CUDA (ROCm) tensor; gcn_amd has no CPU path" % name)
    if t.dtype not in _DTYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1 and t.numel()):
        raise ValueError("%s must be a row-major 2-D tensor" % name)
    if like is not None and (shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError("%s differs from x in shape, dtype or device" % name)
    return stride[0]


def _check_weight(w, name, x):
    if w is None:
        return None
    if w.dtype != torch.float32 or w.dim() != 1 or w.numel() != x.shape[1] or not w.is_contiguous() or w.device != x.device:
        raise ValueError("%s must be contiguous float32 [%d] on x's device" % (name, x.shape[1]))
    return w.data_ptr()


def _norm_struct(x, z, gate, post_weight, res_scale, pre_weight, kind, eps):
    x_ld = _check_rows(x, "x")
    n, dim = x.shape
    if kind not in ("rms", "layer"):
        raise ValueError("kind must be 'rms' or 'layer', got %r" % (kind,))
    if not 1 <= dim <= 4096:
        raise ValueError("rows of 1..4096 elements, got %d" % dim)
    z_ld = gate_ld = 0
    if z is not None:
        z_ld = _check_rows(z, "z", x)
    elif gate is not None or post_weight is not None or res_scale is not None:
        raise ValueError("gate, post_weight and res_scale belong to z")
    elif pre_weight is None:
        raise ValueError("neither z nor pre_weight: nothing to do")
    if gate is not None:
        gate_ld = _check_rows(gate, "gate", x)
    return _lib.NormResidualStruct(n, dim, _DTYPES[x.dtype], 1 if kind == "layer" else 0, eps, x.data_ptr(), x_ld, _at(z), z_ld,
                                   _at(gate), gate_ld, _check_weight(post_weight, "post_weight", x),
                                   _check_weight(res_scale, "res_scale", x), _check_weight(pre_weight, "pre_weight", x))


def norm_residual(x, z=None, gate=None, post_weight=None, res_scale=None, pre_weight=None, kind="rms", eps=1e-6,
                  want_stats=False):
    """``(y, h, stats)``: the end of one block of a deep network and the norm in front
    of the next, row by row in one pass:
    ``y = x + res_scale * sigmoid(gate) * (norm(z) * post_weight)``,
    ``h = norm(y) * pre_weight``.  ``x`` (the residual stream), ``z`` (the block's
    output) and ``gate`` (logits) are row-major [n, dim], dim up to 4096, one of
    float32, bfloat16 and float16; the weights float32 [dim].  What is None is left
    out: no ``gate`` or ``res_scale`` multiplies by one, no ``post_weight`` takes ``z``
    as it is, no ``pre_weight`` gives no ``h`` (None), no ``z`` gives ``y = x`` (``x``
    itself) and ``h = norm(x) * pre_weight``.  ``norm`` divides by the root mean square
    (``kind="rms"``) or takes the mean off first (``"layer"``).  ``stats`` (None unless
    ``want_stats``) is what :func:`norm_residual_bwd` needs."""
    lib = _lib.load()
    p = _norm_struct(x, z, gate, post_weight, res_scale, pre_weight, kind, eps)
    dev, shape = x.device, x.shape
    y = _like(x) if z is not None else x
    h = _like(x) if pre_weight is not None else None
    stats = torch.empty((shape[0], 4), dtype=torch.float32, device=dev) if want_stats else None
    if shape[0]:
        with _on(dev):
            _lib.check(lib.gcnx_norm_residual_forward(C.byref(p), y.data_ptr(), y.stride(0), _at(h), shape[1], _at(stats),
                                                      _stream_of(dev)))
    return y, h, stats


def norm_residual_bwd(x, dy, dh, stats, z=None, gate=None, post_weight=None, res_scale=None, pre_weight=None, kind="rms",
                      eps=1e-6, need=(True,) * 6):
    """``(dx, dz, dgate, dpost, dres, dpre)`` of :func:`norm_residual` for the gradients
    ``dy`` and ``dh`` of its outputs (None: zero); None where there is no such operand
    and where ``need`` (one flag a gradient) is False.
    The row gradients have the type of ``x``, those of the weights are float32, summed
    over the rows in a fixed order."""
    lib = _lib.load()
    p = _norm_struct(x, z, gate, post_weight, res_scale, pre_weight, kind, eps)
    dy_ld = _check_rows(dy, "dy", x) if dy is not None else 0
    dh_ld = _check_rows(dh, "dh", x) if dh is not None else 0
    if dh is not None and pre_weight is None:
        raise ValueError("dh without pre_weight")
    n, dim = x.shape
    dev = x.device
    if stats.dtype != torch.float32 or stats.shape != (n, 4) or not stats.is_contiguous() or stats.device != dev:
        raise ValueError("stats must be what norm_residual(..., want_stats=True) returned")
    dx = _like(x) if need[0] else None
    dz = _like(x) if z is not None and need[1] else None
    dgate = _like(x) if gate is not None and need[2] else None
    made = [None, None, None]
    wanted = [i for i, w in enumerate((post_weight, res_scale, pre_weight)) if w is not None and need[3 + i]]
    summed = [i for i in wanted if n and (i < 2 or dh is not None)]
    if wanted:
        # one buffer for the (small) gradients of the weights; sums over nothing are zero
        buf = (torch.empty if len(summed) == len(wanted) else torch.zeros)((len(wanted), dim), dtype=torch.float32, device=dev)
        for row, i in zip(buf.unbind(0), wanted):
            made[i] = row
    if n and (dx is not None or dz is not None or dgate is not None or summed):
        with _on(dev):
            room = lib.gcnx_norm_residual_backward_workspace_bytes(C.byref(p)) if summed else 0
            ws = _scratch(room, dev)
            _lib.check(lib.gcnx_norm_residual_backward(
                C.byref(p), _at(dy), dy_ld, _at(dh), dh_ld, stats.data_ptr(), _at(dx), _at(dz), _at(dgate), _at(made[0]),
                _at(made[1]), _at(made[2]) if dh is not None else None, _at(ws), room, _stream_of(dev)))
    return (dx, dz, dgate) + tuple(made)


class _NormResidualFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, gate, post_weight, res_scale, pre_weight, kind, eps):
        y, h, stats = norm_residual(x, z, gate, post_weight, res_scale, pre_weight, kind, eps, want_stats=True)
        ctx.save_for_backward(x, z, gate, post_weight, res_scale, pre_weight, stats)
        ctx.how = (kind, eps)
        ctx.set_materialize_grads(False)
        return y if z is not None else x.view_as(x), h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        x, z, gate, post_weight, res_scale, pre_weight, stats = ctx.saved_tensors
        rows = lambda t: t if t is None or t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()
        return norm_residual_bwd(x, rows(dy), rows(dh), stats, z, gate, post_weight, res_scale, pre_weight, *ctx.how,
                                 need=ctx.needs_input_grad[:6]) + (None, None)


def norm_residual_autograd(x, z=None, gate=None, post_weight=None, res_scale=None, pre_weight=None, kind="rms", eps=1e-6):
    """``(y, h)`` of :func:`norm_residual` on the autograd tape."""
    return _NormResidualFn.apply(x, z, gate, post_weight, res_scale, pre_weight, kind, eps)


# ------------------------------------------------------------- loss / accuracy
def masked_softmax_xent(logits, labels, mask, want_grad=True, mask_total=0.0, grad_out=None):
    """Returns ``(loss_acc, grad)``: ``loss_acc`` is a 2-element device tensor
    ``[loss, accuracy]`` (reference gcn/metrics.py:4-20), ``grad`` = dloss/dlogits
    or None."""
    lib = _lib.load()
    _check_dense(logits, "logits")
    _check_dense(labels, "labels")
    n, c = logits.shape
    if tuple(labels.shape) != (n, c):
        raise ValueError("labels shape %s != logits shape %s" % (tuple(labels.shape), (n, c)))
    if mask.dtype != torch.uint8 or mask.numel() != n or mask.device != logits.device:
        raise ValueError("mask must be uint8 [n] on the logits' device")
    out = torch.empty(2, dtype=torch.float32, device=logits.device)
    grad = (grad_out if grad_out is not None else torch.empty_like(logits)) if want_grad else None
    with torch.cuda.device(logits.device):
        need = lib.gcnx_xent_workspace_bytes(n)
        ws = WORKSPACE.get(need, logits.device)
        _lib.check(lib.gcnx_masked_softmax_xent_f32(
            n, c, _ptr(logits), logits.stride(0), _ptr(labels), labels.stride(0), _ptr(mask),
            float(mask_total), _ptr(out), _ptr(grad), grad.stride(0) if grad is not None else 0,
            _ptr(ws), ws.numel(), _stream()))
    if want_grad and grad_out is not None:
        _written(grad_out)
    return out, grad


class _XentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, mask):
        # a mask uploaded by the session carries its count of set entries, which
        # saves the counting pass (two launches) on every step
        out, grad = masked_softmax_xent(logits.contiguous(), labels, mask, want_grad=True,
                                        mask_total=float(getattr(mask, "mask_total", 0.0)))
        ctx.save_for_backward(grad)
        loss, acc = out[0], out[1]
        ctx.mark_non_differentiable(acc)
        return loss, acc

    @staticmethod
    def backward(ctx, dloss, _dacc):
        (grad,) = ctx.saved_tensors
        return grad * dloss, None, None


def masked_softmax_xent_autograd(logits, labels, mask):
    """``(loss, accuracy)`` as 0-dim tensors; ``loss`` is differentiable."""
    return _XentFn.apply(logits, labels, mask)


# ------------------------------------------------------------------ elementwise
def device_counter(device, value=0):
    """A 64-bit step counter in device memory (int64 tensor of one element),
    advanced with :func:`counter_add` on the stream."""
    dev = torch.device(device)
    if dev.type != "cuda":
        raise RuntimeError("device_counter needs a CUDA (ROCm) device")
    return torch.full((1,), int(value), dtype=torch.int64, device=dev)


def counter_add(counter, inc=1):
    lib = _lib.load()
    if counter.device.type != "cuda" or counter.dtype != torch.int64 or counter.numel() != 1:
        raise ValueError("counter must be a one-element int64 CUDA tensor")
    with torch.cuda.device(counter.device):
        _lib.check(lib.gcnx_counter_add_u64(_ptr(counter), int(inc), _stream()))
    _written(counter)
    return counter


def bernoulli_mask(n, keep, seed, offset, device, out=None, step=None, step_stride=0):
    """uint8 mask, byte k = 1 with probability ``keep``, a pure function of
    (seed, offset + k) (Philox4x32-10).  With ``step`` (a device counter) the
    offset is advanced by ``step * step_stride`` when the kernel runs, so a launch
    recorded in a HIP graph draws a new mask on every replay."""
    lib = _lib.load()
    dev = torch.device(device)
    if dev.type != "cuda":
        raise RuntimeError("bernoulli_mask needs a CUDA (ROCm) device")
    if out is not None:
        if out.dtype != torch.uint8 or out.numel() != int(n) or not out.is_contiguous():
            raise ValueError("out must be a contiguous uint8 tensor of n elements")
        mask = out
    else:
        mask = torch.empty(int(n), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        if step is not None:
            if step.device.type != "cuda" or step.dtype != torch.int64 or step.numel() != 1:
                raise ValueError("step must be a one-element int64 CUDA tensor")
            _lib.check(lib.gcnx_bernoulli_mask_dev_u8(int(n), float(keep), int(seed) & (2 ** 64 - 1),
                                                      int(offset), _ptr(step), int(step_stride),
                                                      _ptr(mask), _stream()))
        else:
            _lib.check(lib.gcnx_bernoulli_mask_u8(int(n), float(keep), int(seed) & (2 ** 64 - 1),
                                                  int(offset), _ptr(mask), _stream()))
    if out is not None:
        _written(out)
    return mask


def dropout_dense(x, mask, scale, out=None):
    lib = _lib.load()
    if x.device.type != "cuda" or x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32 CUDA tensor")
    if mask.dtype != torch.uint8 or mask.numel() != x.numel():
        raise ValueError("mask must be uint8 with one byte per element")
    if out is None:
        out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.check(lib.gcnx_dropout_dense_f32(x.numel(), _ptr(x), _ptr(mask), float(scale),
                                              _ptr(out), _stream()))
    _written(out)
    return out


def relu_dropout_bwd(y, dy, mask=None, scale=1.0, out=None):
    """``dx = (y > 0 ? dy : 0)`` optionally times the dropout mask and scale."""
    lib = _lib.load()
    if y.device.type != "cuda" or not y.is_contiguous() or not dy.is_contiguous():
        raise ValueError("y and dy must be contiguous CUDA tensors")
    if y.numel() != dy.numel() or (mask is not None and mask.numel() != y.numel()):
        raise ValueError("y, dy and mask differ in size")
    dx = out if out is not None else torch.empty_like(dy)
    if dx.numel() != dy.numel() or not dx.is_contiguous():
        raise ValueError("out must be contiguous and as large as dy")
    with torch.cuda.device(y.device):
        _lib.check(lib.gcnx_relu_dropout_bwd_f32(y.numel(), _ptr(y), _ptr(dy), _ptr(mask),
                                                 float(scale), _ptr(dx), _stream()))
    if out is not None:
        _written(out)
    return dx


def gather_rows(src, idx, out):
    """``out[j, :] = src[idx[j], :]`` (``idx`` int32 on the device)."""
    lib = _lib.load()
    _check_dense(src, "src")
    _check_dense(out, "out")
    if idx.dtype != torch.int32 or idx.device != src.device or not idx.is_contiguous():
        raise ValueError("idx must be a contiguous int32 tensor on src's device")
    if out.shape[0] != idx.numel() or out.shape[1] != src.shape[1]:
        raise ValueError("out must be [len(idx), width]")
    with torch.cuda.device(src.device):
        _lib.check(lib.gcnx_gather_rows_f32(idx.numel(), _ptr(idx), _ptr(src), src.stride(0),
                                            src.shape[1], _ptr(out), out.stride(0), _stream()))
    _written(out)
    return out


def scatter_rows(src, idx, out):
    """``out[idx[j], :] = src[j, :]`` for distinct ``idx`` (int32 on the device);
    the other rows of ``out`` keep their contents."""
    lib = _lib.load()
    _check_dense(src, "src")
    _check_dense(out, "out")
    if idx.dtype != torch.int32 or idx.device != src.device or not idx.is_contiguous():
        raise ValueError("idx must be a contiguous int32 tensor on src's device")
    if src.shape[0] != idx.numel() or out.shape[1] != src.shape[1]:
        raise ValueError("src must be [len(idx), width of out]")
    with torch.cuda.device(src.device):
        _lib.check(lib.gcnx_scatter_rows_f32(idx.numel(), _ptr(idx), _ptr(src), src.stride(0),
                                             src.shape[1], _ptr(out), out.stride(0), _stream()))
    _written(out)
    return out


def csr_filter_columns(a, col_keep):
    """The sub-matrix of ``a`` (a Csr) with the nonzeros of the flagged columns only
    (Csr.filter_columns): for products whose operand is exactly zero in the other rows."""
    return a.filter_columns(col_keep)


def csr_compact_rows(a):
    """``(sub, rows)``: ``a`` without its empty rows and the int32 ids of the rows kept
    (Csr.compact_rows)."""
    return a.compact_rows()


def csr_keep_rows(a, rows):
    """``a`` restricted to the rows ``rows`` (ascending ids; every row left out must be
    empty), stored next to each other (Csr.keep_rows)."""
    return a.keep_rows(rows)


def csr_transpose(a):
    """A fresh exact transpose of ``a`` (Csr.transpose without the cache): set-up of
    derived matrices."""
    return a.transpose(cache=False)


def philox_uniform(shape, lo, hi, seed, offset, device):
    """fp32 tensor of U(lo, hi) values, element i a pure function of
    (seed, offset + i) (synthetic benchmark inputs)."""
    lib = _lib.load()
    dev = torch.device(device)
    if dev.type != "cuda":
        raise RuntimeError("philox_uniform needs a CUDA (ROCm) device")
    out = torch.empty(shape, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.gcnx_philox_uniform_f32(out.numel(), float(lo), float(hi),
                                               int(seed) & (2 ** 64 - 1), int(offset), _ptr(out),
                                               _stream()))
    return out


def dropout_philox(x, keep, seed, offset, out=None, mask_out=None):
    """``out = kept ? x / keep : 0`` with the Bernoulli(keep) mask regenerated
    from Philox (seed, offset + i): same bits as :func:`bernoulli_mask`."""
    lib = _lib.load()
    if x.device.type != "cuda" or x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32 CUDA tensor")
    if out is None:
        out = torch.empty_like(x)
    if out.numel() != x.numel() or not out.is_contiguous():
        raise ValueError("out must be contiguous and as large as x")
    with torch.cuda.device(x.device):
        _lib.check(lib.gcnx_dropout_philox_f32(x.numel(), _ptr(x), float(keep),
                                               int(seed) & (2 ** 64 - 1), int(offset), _ptr(out),
                                               _ptr(mask_out), _stream()))
    _written(out) if mask_out is None else _written(out, mask_out)
    return out


def relu_dropout_bwd_philox(y, dy, keep, seed, offset, out=None):
    """``dx = (y > 0 and kept) ? dy / keep : 0`` with the mask of
    :func:`dropout_philox` regenerated."""
    lib = _lib.load()
    if y.device.type != "cuda" or not y.is_contiguous() or not dy.is_contiguous() or y.numel() != dy.numel():
        raise ValueError("y and dy must be contiguous CUDA tensors of one size")
    dx = out if out is not None else torch.empty_like(dy)
    with torch.cuda.device(y.device):
        _lib.check(lib.gcnx_relu_dropout_bwd_philox_f32(y.numel(), _ptr(y), _ptr(dy), float(keep),
                                                        int(seed) & (2 ** 64 - 1), int(offset),
                                                        _ptr(dx), _stream()))
    if out is not None:
        _written(out)
    return dx


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mask, scale):
        ctx.mask = mask
        ctx.scale = scale
        return dropout_dense(x.contiguous(), mask, scale)

    @staticmethod
    def backward(ctx, dy):
        return dropout_dense(dy.contiguous(), ctx.mask, ctx.scale), None, None


def dropout_dense_autograd(x, mask, scale):
    return _DropoutFn.apply(x, mask, scale)


def adam_step(w, grad, m, v, lr, t, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0):
    """In-place TF-style Adam (reference gcn/models.py:142); ``t`` counts from 1
    and is either a Python int or a device counter (read when the kernel runs)."""
    lib = _lib.load()
    for name, x in (("w", w), ("grad", grad), ("m", m), ("v", v)):
        if x.device.type != "cuda" or x.dtype != torch.float32 or not x.is_contiguous():
            raise ValueError("%s must be a contiguous float32 CUDA tensor" % name)
    with torch.cuda.device(w.device):
        if isinstance(t, torch.Tensor):
            if t.device.type != "cuda" or t.dtype != torch.int64 or t.numel() != 1:
                raise ValueError("t must be an int or a one-element int64 CUDA tensor")
            _lib.check(lib.gcnx_adam_step_dev_f32(w.numel(), _ptr(w), _ptr(grad), _ptr(m), _ptr(v),
                                                  float(lr), float(beta1), float(beta2), float(eps),
                                                  float(weight_decay), _ptr(t), _stream()))
        else:
            _lib.check(lib.gcnx_adam_step_f32(w.numel(), _ptr(w), _ptr(grad), _ptr(m), _ptr(v),
                                              float(lr), float(beta1), float(beta2), float(eps),
                                              float(weight_decay), int(t), _stream()))
    _written(w, m, v)
    return w


class AdamWState(object):
    """The moments of :func:`adamw_step` for a list of tensors (:func:`adamw_state`),
    all in two flat buffers: tensor i's are the elements from ``offsets[i]`` on, every
    offset a multiple of 256.  ``bits`` 32: ``exp_avg`` and ``exp_avg_sq`` float32.  8:
    float8_e4m3fn codes, ``exp_avg`` of m and ``exp_avg_sq`` of sqrt(v), each to be
    multiplied by its block of 256's power of two in ``exp_avg_scale`` /
    ``exp_avg_sq_scale``; ``seed`` keys the random rounding."""

    def __init__(self, params, bits, seed):
        self.bits, self.seed = bits, int(seed) & (2 ** 64 - 1)
        self.sizes = [p.numel() for p in params]
        self.dtype, self.device = params[0].dtype, params[0].device
        self.offsets, total = [], 0
        for n in self.sizes:
            self.offsets.append(total)
            total += -(-n // _lib.ADAMW_BLOCK) * _lib.ADAMW_BLOCK
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=self.device)
        if bits == 32:
            self.exp_avg, self.exp_avg_sq = zeros(total, torch.float32), zeros(total, torch.float32)
            self.exp_avg_scale = self.exp_avg_sq_scale = None
        else:
            self.exp_avg, self.exp_avg_sq = [zeros(total, torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
            self.exp_avg_scale, self.exp_avg_sq_scale = [torch.ones_like(zeros(total // _lib.ADAMW_BLOCK, torch.float32))
                                                         for _ in range(2)]
        self._table = np.zeros(len(self.sizes), dtype=[("w", "u8"), ("grad", "u8"), ("n", "i8"), ("state", "i8"), ("decay", "f8")])
        self._table["state"], self._table["n"] = self.offsets, self.sizes

    def _parts(self, i):
        """Tensor i's part of every buffer (8-bit codes as bytes)."""
        at, end = self.offsets[i], self.offsets[i] - (-self.sizes[i] // _lib.ADAMW_BLOCK) * _lib.ADAMW_BLOCK
        codes = [t.view(torch.uint8) if self.bits == 8 else t for t in (self.exp_avg, self.exp_avg_sq)]
        scales = [self.exp_avg_scale, self.exp_avg_sq_scale] if self.bits == 8 else []
        return [t[at:end] for t in codes] + [t[at // _lib.ADAMW_BLOCK:end // _lib.ADAMW_BLOCK] for t in scales]

    def reset(self, i):
        """Zeroes the moments of tensor i."""
        for part, value in zip(self._parts(i), (0, 0, 1, 1)):
            part.fill_(value)

    def take(self, i, other, j):
        """Copies the moments of tensor j of another state of the same ``bits`` to tensor i."""
        if other.bits != self.bits or other.sizes[j] != self.sizes[i]:
            raise ValueError("states or tensors differ")
        for to, part in zip(self._parts(i), other._parts(j)):
            to.copy_(part)

    def moments(self, i):
        """``(m, v)`` of tensor i as flat float32 tensors."""
        at, n = self.offsets[i], self.sizes[i]
        m, v = self.exp_avg[at:at + n].float(), self.exp_avg_sq[at:at + n].float()
        if self.bits == 8:
            block = torch.arange(at, at + n, device=self.device) // _lib.ADAMW_BLOCK
            m, v = m * self.exp_avg_scale[block], (v * self.exp_avg_sq_scale[block]) ** 2
        return m, v


def adamw_state(params, bits=32, seed=0):
    """A zero :class:`AdamWState` for a list of contiguous tensors of one dtype
    (float32, bfloat16 or float16) on one device; ``bits`` 32 or 8."""
    params = list(params)
    if not params:
        raise ValueError("no tensors")
    if bits not in (32, 8):
        raise ValueError("bits must be 32 or 8, got %r" % (bits,))
    for p in params:
        if not isinstance(p, torch.Tensor) or p.device.type != "cuda":
            raise RuntimeError("params must be CUDA (ROCm) tensors; gcn_amd has no CPU path")
        if p.dtype not in _DTYPES:
            raise TypeError("params must be float32, bfloat16 or float16, got %s" % (p.dtype,))
        if p.dtype != params[0].dtype or p.device != params[0].device:
            raise ValueError("params differ in dtype or device")
    return AdamWState(params, bits, seed)


_numel_of, _index_of, _dense, _address_of = torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _uniform(tensors, dtype, index, sizes):
    """Whether all are contiguous tensors of one type on GPU ``index``, of these sizes
    (attribute by attribute: half the time of a loop over the tensors)."""
    n = len(sizes)
    return [t.dtype for t in tensors].count(dtype) == n and list(map(_index_of, tensors)).count(index) == n and \
        list(map(_numel_of, tensors)) == sizes and all(map(_dense, tensors))


def _overlap(addresses, sizes, itemsize):
    """Whether one of the tensors, taken in this order, begins before the end of an earlier one."""
    end = 0
    for at, n in zip(addresses, sizes):
        if n:
            if at < end:
                return True
            end = at + n * itemsize
    return False


def adamw_step(params, grads, state, lr, t, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01):
    """One in-place AdamW update of every tensor of ``params`` in one launch (one per 64
    tensors): ``m = beta1 m + (1 - beta1) g``, ``v = beta2 v + (1 - beta2) g^2``,
    ``w = w (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)``.
    ``state`` is the list's :func:`adamw_state`; ``grads`` (one dtype: float32, bfloat16
    or float16) has one contiguous tensor a param, or None: that param and its state
    stay as they are.  No two tensors may share memory.  ``t`` counts from 1 and is
    either a Python int or a device counter (read when the kernels run, and at least 1
    by then); ``weight_decay`` is a number or one a param.  The decoupled many-tensor
    sibling of :func:`adam_step`."""
    lib = _lib.load()
    count = len(state.sizes)
    params, grads = list(params), list(grads)
    if len(params) != count or len(grads) != count:
        raise ValueError("%d params and %d grads for a state of %d tensors" % (len(params), len(grads), count))
    dtype, dev, table, sizes = state.dtype, state.device, state._table, state.sizes

    if not _uniform(params, dtype, dev.index, sizes):
        raise ValueError("params must be the contiguous tensors the state was made for")
    live, decay = params, weight_decay
    if type(None) in map(type, grads):
        wanted = [i for i, g in enumerate(grads) if g is not None]
        live, grads, sizes = [[x[i] for i in wanted] for x in (params, grads, sizes)]
        table, decay = table[wanted], np.broadcast_to(np.asarray(decay, dtype=np.float64), count)[wanted]
    if not any(sizes):
        return params
    g_dtype = grads[0].dtype
    if g_dtype not in _DTYPES:
        raise TypeError("grads must be float32, bfloat16 or float16, got %s" % (g_dtype,))
    if not _uniform(grads, g_dtype, dev.index, sizes):
        raise ValueError("grads must be contiguous, of one dtype, on the params' device and of their sizes")
    w_ptr, g_ptr = list(map(_address_of, live)), list(map(_address_of, grads))
    if _overlap(w_ptr, sizes, dtype.itemsize) and _overlap(*zip(*sorted(zip(w_ptr, sizes))), dtype.itemsize):
        raise ValueError("params share memory")
    if isinstance(t, torch.Tensor):
        if t.device != dev or t.dtype != torch.int64 or t.numel() != 1:
            raise ValueError("t must be an int or a one-element int64 tensor on the params' device")
        t_ptr, t_host = t.data_ptr(), 0
    else:
        t_ptr, t_host = None, int(t)
    table = table.copy()
    table["w"], table["grad"], table["decay"] = w_ptr, g_ptr, decay
    p = _lib.AdamWStruct(_DTYPES[dtype], _DTYPES[g_dtype], state.bits, state.exp_avg.data_ptr(), state.exp_avg_sq.data_ptr(),
                         _at(state.exp_avg_scale), _at(state.exp_avg_sq_scale), lr, beta1, beta2, eps, t_host, t_ptr, state.seed)
    with _on(dev):
        need = _lib.ADAMW_WORKSPACE_BYTES if t_ptr else 0
        ws = _scratch(need, dev)
        _lib.check(lib.gcnx_adamw_step(C.byref(p), len(table), table.ctypes.data, _at(ws), need, _stream_of(dev)))
    _written(*live)
    return params


def l2_loss(w, scale=1.0, add=None):
    """One-element tensor ``(add or 0) + scale * sum(w ** 2) / 2`` (reference
    gcn/models.py:148-149: ``weight_decay * tf.nn.l2_loss(var)`` added into the
    loss).  No gradient is recorded: the decay gradient ``scale * w`` is applied
    inside :func:`adam_step` (``weight_decay``)."""
    lib = _lib.load()
    w = w.detach()
    if w.device.type != "cuda" or w.dtype != torch.float32 or not w.is_contiguous():
        raise ValueError("w must be a contiguous float32 CUDA tensor")
    if add is not None:
        add = add.detach()
        if add.device != w.device or add.dtype != torch.float32 or add.numel() != 1:
            raise ValueError("add must be a one-element float32 tensor on w's device")
    out = torch.empty(1, dtype=torch.float32, device=w.device)
    with torch.cuda.device(w.device):
        _lib.check(lib.gcnx_l2_loss_f32(w.numel(), _ptr(w), float(scale), _ptr(add), _ptr(out), _stream()))
    return out


def profile_spmm_events(start, stop):
    """Development / benchmark hook: the next SpMM calls of this thread record
    ``start`` right before and ``stop`` right after their main kernel on the
    launch stream (pass ``None, None`` to switch it off).  The arguments are
    ``torch.cuda.Event(enable_timing=True)`` objects that have been recorded at
    least once (so that their HIP handles exist)."""
    lib = _lib.load()
    a = C.c_void_p(start.cuda_event) if start is not None else C.c_void_p(0)
    b = C.c_void_p(stop.cuda_event) if stop is not None else C.c_void_p(0)
    lib.gcnx_profile_spmm_events(a, b)


__all__ = ["Csr", "spmm", "spmm_factored", "spmm_supports_factored", "spmm_autograd", "gemm", "gemm_supports_a_dropout", "gemm_autograd", "masked_softmax_xent",
           "masked_softmax_xent_autograd", "bernoulli_mask", "dropout_dense",
           "dropout_dense_autograd", "relu_dropout_bwd", "dropout_philox", "relu_dropout_bwd_philox", "philox_uniform", "gather_rows", "adam_step",
           "attention", "attention_bwd", "attention_autograd", "norm_residual", "norm_residual_bwd", "norm_residual_autograd",
           "AdamWState", "adamw_state", "adamw_step"]
