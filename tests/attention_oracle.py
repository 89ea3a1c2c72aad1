"""Graph attention and its gradients in 64 bits on the host, edge by edge, with the
error bounds the kernels are held to."""
import numpy as np

U = 2.0 ** -24            # half a step of fp32


class AttentionOracle(object):
    """``row`` / ``col`` [nnz], ``shift`` and ``on`` [nnz] (or None) in one order;
    q [n_rows, H, D], k, v [n_cols, G, D] float64; ``half`` is half a step of the
    operands' type relative to the value (torch.finfo(t).eps / 2), ``tiny`` its
    smallest normal value."""

    def __init__(self, row, col, shape, q, k, v, scale, shift=None, on=None, half=U, tiny=0.0):
        self.row, self.col = np.asarray(row, np.int64), np.asarray(col, np.int64)
        keep = np.ones(len(self.row), bool) if on is None else np.asarray(on) != 0
        shift = np.zeros(len(self.row)) if shift is None else np.asarray(shift, np.float64)
        keep &= shift != -np.inf
        self.row, self.col, shift = self.row[keep], self.col[keep], shift[keep]
        self.n_rows, self.n_cols = shape
        self.q, self.scale, self.half = q, scale, half
        # Below the smallest normal value `tiny` the steps stay those at tiny: half a
        # step is half * tiny there, not half * |x| (fp16: 2^-11 * 2^-14 = 2^-25).
        self.tiny = tiny
        heads, dim = q.shape[1:]
        group = heads // k.shape[1]
        self.k, self.v = np.repeat(k, group, axis=1), np.repeat(v, group, axis=1)
        self.group = group
        qe, ke = q[self.row], self.k[self.col]
        self.s = scale * (qe * ke).sum(2) + shift[:, None]
        size = scale * (np.abs(qe) * np.abs(ke)).sum(2)
        top = np.full((self.n_rows, heads), -np.inf)
        np.maximum.at(top, self.row, self.s)
        top[top == -np.inf] = 0.0
        gap = top[self.row] - self.s
        w = np.exp(-gap)
        total = self._rows(w)
        self.p = w / total[self.row]
        deg = np.bincount(self.row, minlength=self.n_rows)[:, None]
        # a logit: dim products and sums, the scale, the shift; an exponent: the
        # difference, times log2(e), 2 ulp of the exponential
        self.e_s = ((dim + 2) * size + np.abs(self.s) + np.abs(shift)[:, None]) * U
        worst = np.zeros((self.n_rows, heads))
        np.maximum.at(worst, self.row, self.e_s + gap * 2 * U * (w > 1e-30))
        # relative error of a probability: its own logit's and the sum's, rescaling
        # by joined maxima included (two roundings a joined term)
        self.e_p = 2 * worst + (3 * deg + 16) * U
        ve = self.v[self.col]
        self.out = self._rows(self.p[:, :, None] * ve)
        mag = self._rows(self.p[:, :, None] * np.abs(ve))
        self.out_bound = mag * (self.e_p + (deg + 4) * U)[:, :, None] + half * np.maximum(np.abs(self.out), tiny) + 1e-37
        self.deg = deg

    def _rows(self, x):
        y = np.zeros((self.n_rows,) + x.shape[1:])
        np.add.at(y, self.row, x)
        return y

    def _cols(self, x):
        y = np.zeros((self.n_cols,) + x.shape[1:])
        np.add.at(y, self.col, x)
        return y.reshape(self.n_cols, -1, self.group, x.shape[2]).sum(2)

    def backward(self, d_out):
        """Sets dq, dk, dv and their bounds."""
        dim = d_out.shape[2]
        ge, ke, qe, ve = d_out[self.row], self.k[self.col], self.q[self.row], self.v[self.col]
        delta = (d_out * self.out).sum(2)
        dp = (ge * ve).sum(2)
        ds = self.p * (dp - delta[self.row])
        # delta is formed from the stored output, which is half a step off
        e_delta = (np.abs(d_out) * (self.out_bound + dim * U * np.abs(self.out))).sum(2)
        e_dp = (dim + 1) * U * (np.abs(ge) * np.abs(ve)).sum(2)
        e_p = self.e_p[self.row]
        e_ds = self.p * (e_dp + e_delta[self.row] + U * (np.abs(dp) + np.abs(delta[self.row]))) + np.abs(ds) * (e_p + 4 * U)
        at, group = np.bincount(self.col, minlength=self.n_cols)[:, None, None], self.group
        def bound(summed, terms, errors, count):
            return summed(errors) + (count * self.group + 4) * U * summed(terms)
        x = self.scale
        self.dq = x * self._rows(ds[:, :, None] * ke)
        self.dq_bound = x * bound(self._rows, np.abs(ds)[:, :, None] * np.abs(ke), e_ds[:, :, None] * np.abs(ke), self.deg[:, :, None])
        self.dk = x * self._cols(ds[:, :, None] * qe)
        self.dk_bound = x * bound(self._cols, np.abs(ds)[:, :, None] * np.abs(qe), e_ds[:, :, None] * np.abs(qe), at)
        self.dv = self._cols(self.p[:, :, None] * ge)
        self.dv_bound = bound(self._cols, self.p[:, :, None] * np.abs(ge), (self.p * (e_p + 2 * U))[:, :, None] * np.abs(ge), at)
        for name in ("dq", "dk", "dv"):
            b = getattr(self, name + "_bound")
            setattr(self, name + "_bound", b * (1 + self.half) + self.half * np.maximum(np.abs(getattr(self, name)), self.tiny) + 1e-37)
        return self


def assert_within(got, want, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        ratio = np.where(np.isfinite(got), np.abs(got - want) / bound, np.inf)
        i = np.unravel_index(np.argmax(np.where(bad, ratio, -1)), got.shape)
        raise AssertionError("%s: %d of %d off; worst at %s: got %r want %r bound %r" %
                             (what, int(bad.sum()), bad.size, i, got[i], want[i], bound[i]))
