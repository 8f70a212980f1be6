"""Large calls of the head's loss against the formulas in 64 bits: every row's nll, sampled rows of dx, sampled
columns of dw and db.  The logits pass through in blocks of rows; nothing of their size is kept."""
import numpy as np

from head_model import HALF, PAIR, Loss, widen


class Samples:
    """Of a test_gpu_head.Case: what nll, dx[rows], dw[:, cols] and db[cols] have to be, and the bounds of
    head_model.Loss for them."""

    def __init__(self, c, rows, cols, grad_type=None):
        self.rows, self.cols = np.asarray(rows), np.asarray(cols)
        gt = c.gt if grad_type is None else grad_type
        x, w = widen(c.x[:, :c.d]), widen(c.w)
        target = c.target.astype(np.int64)
        live = (target >= 0) & (target < c.vocab)
        x = np.where(live[:, None], x, 0.0)
        b = np.zeros(c.vocab) if c.b is None else c.b.astype(np.float64)
        aw, ab = np.abs(w), np.abs(b)
        self.nll, self.tol_nll = np.zeros(c.rows), np.zeros(c.rows)
        off, delta = np.zeros((c.rows, self.cols.size)), np.zeros((c.rows, self.cols.size))
        chain = 64 + 10 + 16 + c.vocab / 4096
        block = max(1, (1 << 26) // c.vocab)
        for a in range(0, c.rows, block):
            s = slice(a, min(a + block, c.rows))
            z = x[s] @ w + b
            top = z.max(1, keepdims=True)
            mag = (np.abs(x[s]) @ aw + ab).max(1, keepdims=True)
            at, r = np.where(live[s], target[s], 0), np.arange(z.shape[0])
            zt, zc = z[r, at], z[:, self.cols]
            z -= top
            lse = top + np.log(np.exp(z, out=z).sum(1, keepdims=True))
            eps_z = (c.d + 2) * 2.0 ** -23 * mag
            eps_p = 2 * eps_z + (3 * mag + 4 + chain) * 2.0 ** -23
            self.nll[s] = np.where(live[s], lse[:, 0] - zt, 0.0)
            self.tol_nll[s] = (eps_z + eps_p)[:, 0] + 2.0 ** -22 * np.abs(self.nll[s])
            p = np.exp(zc - lse)
            hit = (target[s][:, None] == self.cols[None, :]) & live[s][:, None]
            delta[s] = np.where(live[s][:, None], p - hit, 0.0) * c.scale
            off[s] = np.where(live[s][:, None], p * abs(c.scale) * eps_p, 0.0)
        self.live = live
        off += PAIR[gt] * np.abs(delta)
        off = np.where(live[:, None], off, 0.0) + (2.0 ** -133 if gt else 2.0 ** -140)
        old_dw = widen(c.dw0[:, self.cols]) if gt else c.dw0[:, self.cols].astype(np.float64)
        old_db = widen(c.db0[self.cols]) if gt else c.db0[self.cols].astype(np.float64)
        self.dw, self.db = x.T @ delta + old_dw, delta.sum(0) + old_db
        ad, ax, half = np.abs(delta), np.abs(x), HALF[gt]
        sums = (2 * c.rows + 8) * 2.0 ** -23
        self.tol_dw = ax.T @ off + sums * (ax.T @ ad) + 2 * half * np.abs(self.dw) + half * np.abs(old_dw)
        self.tol_db = off.sum(0) + sums * ad.sum(0) + 2 * half * np.abs(self.db) + half * np.abs(old_db)
        # rows are independent of each other: those of dx are a smaller call's
        part = Loss(widen(c.x[self.rows, :c.d]), w, c.b, target[self.rows], c.scale)
        self.dx, self.tol_dx = part.dx, part.tolerances(gt)[0]


def edges(n, every, rng, some):
    """Places of [0, n): both ends, either side of each multiple of `every`, and `some` drawn ones."""
    near = [k + e for k in range(0, n + 1, every) for e in (-1, 0) if 0 <= k + e < n]
    return np.unique(np.concatenate([[0, n - 1], near, rng.integers(0, n, some)]))
