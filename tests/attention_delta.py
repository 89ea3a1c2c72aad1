"""The 16-bit backward of the graph attention with bounds that know how delta is formed:
from the probabilities in fp32, not from the output as it was rounded."""
import numpy as np

from attention_oracle import U, AttentionOracle


class DeltaOracle(AttentionOracle):
    """``rounded``: the output in the operands' type, what the kernel starts from:

        d0 = <dout, rounded>      rest = sum_j p (<dout, v_j> - d0)      delta = d0 + rest
        dq = scale (sum_j p (<dout, v_j> - d0) k_j - rest sum_j p k_j)

    With probabilities off by e_p (relative) whose sum is then off by as much:
    delta is off by e_p (sum p |<dout, v>| + |d0|), the products' own errors, and a
    rounding a term of rest.  The rounding of the output itself drops out."""

    def backward(self, d_out, rounded):
        dim = d_out.shape[2]
        ge, ke, qe, ve = d_out[self.row], self.k[self.col], self.q[self.row], self.v[self.col]
        deg, e_row, e_p = self.deg, self.e_p, self.e_p[self.row]
        dp = (ge * ve).sum(2)
        e_dp = (dim + 1) * U * (np.abs(ge) * np.abs(ve)).sum(2)
        delta = (d_out * self.out).sum(2)
        d0 = (d_out * rounded).sum(2)
        rest = delta - d0
        off = np.abs(dp - d0[self.row])
        rows = lambda x: self._rows(x[:, :, None])[:, :, 0]
        e_delta = e_row * (rows(self.p * np.abs(dp)) + np.abs(d0)) + rows(self.p * e_dp) + (deg + 6) * U * rows(self.p * off) + 2 * U * np.abs(delta)
        ds = self.p * (dp - delta[self.row])
        e_ds = self.p * (e_dp + e_delta[self.row] + U * (np.abs(dp) + np.abs(delta[self.row]))) + np.abs(ds) * (e_p + 4 * U)
        x, at = self.scale, np.bincount(self.col, minlength=self.n_cols)[:, None, None]
        half = lambda value, bound: bound * (1 + self.half) + self.half * np.maximum(np.abs(value), self.tiny) + 1e-37
        self.dq = x * self._rows(ds[:, :, None] * ke)
        terms = self.p * (off + np.abs(rest)[self.row])
        self.dq_bound = half(self.dq, x * (self._rows(e_ds[:, :, None] * np.abs(ke)) + (deg[:, :, None] + 8) * U * self._rows(terms[:, :, None] * np.abs(ke))))
        self.dk = x * self._cols(ds[:, :, None] * qe)
        self.dk_bound = half(self.dk, x * (self._cols(e_ds[:, :, None] * np.abs(qe)) +
                                           (at * self.group + 8) * U * self._cols(np.abs(ds)[:, :, None] * np.abs(qe))))
        # the same gradients with delta from the rounded output
        wrong = self.p * (dp - d0[self.row])
        self.wrong_dq, self.wrong_dk = x * self._rows(wrong[:, :, None] * ke), x * self._cols(wrong[:, :, None] * qe)
        return self


CASES = [(dtype, lengths, heads, kv, dim) for dtype in ("bfloat16", "float16")
         for lengths, heads, kv, dim in (([1, 2, 40, 64, 64], 2, 2, 16),            # rows of one wavefront
                                         ([100, 300, 500, 65], 4, 2, 16),           # rows of a workgroup
                                         ([900, 30, 1500, 700], 2, 1, 32),          # rows in pieces, joined by a wavefront
                                         ([1100, 10, 1300], 2, 1, 12),              # and by a workgroup
                                         ([400, 900], 3, 3, 5))]                    # heads shorter than a piece


def make(dtype, lengths, heads, kv, dim):
    """Rows whose values are nearly alike: v is 1 and 0 to 3 steps of its type, keys are
    around 1, so that <dout, v_j> - delta is far smaller than <dout, v_j>."""
    import torch
    rng = np.random.RandomState(len(lengths) + dim)
    row = np.repeat(np.arange(len(lengths)), lengths).astype(np.int32)
    cols = 97
    col = rng.randint(0, cols, len(row)).astype(np.int32)
    t = getattr(torch, dtype)
    cast = lambda a: torch.from_numpy(a.astype(np.float32)).to(t)
    step = torch.finfo(t).eps
    q = cast(rng.standard_normal((len(lengths), heads, dim)))
    k = cast(1.0 + 0.25 * rng.standard_normal((cols, kv, dim)))
    v = cast(1.0 + step * rng.randint(0, 4, (cols, kv, dim)))
    g = cast(rng.standard_normal((len(lengths), heads, dim)))
    return row, col, (len(lengths), cols), (q, k, v, g)


def oracle(row, col, shape, operands, rounded=None):
    import torch
    q, k, v, g = [t.double().cpu().numpy() for t in operands]
    info = torch.finfo(operands[0].dtype)
    o = DeltaOracle(row, col, shape, q, k, v, float(np.float32(q.shape[2] ** -0.5)), None, None, info.eps / 2, info.tiny)
    if rounded is None:
        rounded = torch.from_numpy(o.out).to(operands[0].dtype).double().numpy()
    return o.backward(g, rounded)
