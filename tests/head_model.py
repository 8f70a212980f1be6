"""The head's loss in numpy in 64 bits, from the formulas in include/anni_adam.h, and how far float
sums and the stated roundings may leave a result from it."""
import numpy as np

HALF = {0: 2.0 ** -24, 1: 2.0 ** -8}        # half a step of the result's type, relative
PAIR = {0: 2.0 ** -16, 1: 2.0 ** -8}        # of delta: two bf16 numbers, or one


def widen(u16):
    return (u16.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def bf16(x):
    """Round to nearest even, as uint16 bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


class Loss:
    """x [rows, d] and w [d, vocab] as float64 of bf16 numbers; bias float32 or None; old = (dw, db) before."""

    def __init__(self, x, w, bias, target, scale, old_dw=None, old_db=None):
        rows, vocab = x.shape[0], w.shape[1]
        self.live = (target >= 0) & (target < vocab)
        x = np.where(self.live[:, None], x, 0.0)        # whatever a row without a target holds
        b = np.zeros(vocab) if bias is None else bias.astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            z = x @ w + b
            top = z.max(1, keepdims=True)
            lse = top + np.log(np.exp(z - top).sum(1, keepdims=True))
            at = np.where(self.live, target, 0)
            r = np.arange(rows)
            self.nll = np.where(self.live, lse[:, 0] - z[r, at], 0.0)
            p = np.exp(z - lse)
        hit = np.zeros_like(p)
        hit[r[self.live], at[self.live]] = 1.0
        delta = np.where(self.live[:, None], p - hit, 0.0) * scale
        self.dx = delta @ w.T
        self.dw = x.T @ delta + (0.0 if old_dw is None else old_dw)
        self.db = delta.sum(0) + (0.0 if old_db is None else old_db)
        # how far off: a float sum of k terms, in any order and with its products exact, is within
        # k 2^-23 of the sum of their magnitudes (2^-24 each, twice that for sums inside an instruction)
        d = x.shape[1]
        ax, aw, ab = np.abs(x), np.abs(w), np.where(np.isfinite(b), np.abs(b), 0.0)
        self.mag = (ax @ aw + ab).max(1, keepdims=True)
        self.eps_z = (d + 2) * 2.0 ** -23 * self.mag
        # an exponential of an argument of at most 2 mag: the product with log2(e), the instruction itself,
        # and its sum over the vocabulary (64 in a lane, 10 folds, one fold in sixteen per tile)
        chain = 64 + 10 + 16 + vocab / 4096
        self.eps_p = 2 * self.eps_z + (3 * self.mag + 4 + chain) * 2.0 ** -23
        self.tol_nll = (self.eps_z + self.eps_p)[:, 0] + 2.0 ** -22 * np.abs(np.where(np.isfinite(self.nll), self.nll, 0.0))
        self.p, self.delta, self.scale, self.ax, self.aw = p, delta, scale, ax, aw
        self.old_dw, self.old_db = old_dw, old_db

    def tolerances(self, grad_type):
        rows, vocab = self.p.shape
        off = np.abs(self.p) * abs(self.scale) * self.eps_p + PAIR[grad_type] * np.abs(self.delta)
        off = np.where(self.live[:, None], off, 0.0) + (2.0 ** -133 if grad_type else 2.0 ** -140)
        ad = np.abs(self.delta)
        half = HALF[grad_type]
        dx = off @ self.aw.T + (2 * vocab + 8) * 2.0 ** -23 * (ad @ self.aw.T) + half * np.abs(self.dx)
        dw = self.ax.T @ off + (2 * rows + 8) * 2.0 ** -23 * (self.ax.T @ ad) + 2 * half * np.abs(self.dw)
        db = off.sum(0) + (2 * rows + 8) * 2.0 ** -23 * ad.sum(0) + 2 * half * np.abs(self.db)
        if self.old_dw is not None:
            dw = dw + half * np.abs(self.old_dw)
            db = db + half * np.abs(self.old_db)
        return dx, dw, db
