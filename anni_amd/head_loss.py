"""The head's loss (anni_head_loss of include/anni_adam.h) with its work area: softmax cross entropy
of x w + b over the vocabulary and its gradients, on device addresses; nothing here computes it."""
import ctypes as C

from . import lib as _l
from .lm_adam import DeviceBuffer


class HeadLoss:
    """Calls of one size: rows tokens, width d, vocab places.  grad=False: the loss alone, for evaluation.
    keep: the logits stay in the work area between the two passes; None: if that takes at most KEEP_MOST bytes."""

    KEEP_MOST = 2 << 30

    def __init__(self, rows, d, vocab, grad_type=_l.F32, grad=True, keep=None):
        self.L = _l.require_gpu()
        self.rows, self.d, self.vocab, self.grad_type, self.grad = rows, d, vocab, grad_type, grad
        sizes = rows, d, vocab, grad_type if grad else -1
        need = self.L.anni_head_loss_work_bytes(*sizes)
        most = self.L.anni_head_loss_work_bytes_keep(*sizes)
        if not need:
            raise ValueError("anni_head_loss refuses rows=%d d=%d vocab=%d grad_type=%d" % (rows, d, vocab, grad_type))
        if keep is None:
            keep = most - need <= self.KEEP_MOST
        self.work = DeviceBuffer(most if keep else need)
        self.job = _l.HeadJob()
        self.job.rows, self.job.d, self.job.vocab, self.job.grad_type = rows, d, vocab, grad_type
        self.job.d_work, self.job.work_bytes = self.work.ptr, self.work.nbytes

    def _fill(self, x, target, nll, scale, dx, ld_x, ld_dx):
        j = self.job
        j.d_x, j.d_target, j.d_nll, j.scale, j.d_dx = x, target, nll, scale, dx
        j.ld_x, j.ld_dx = ld_x or self.d, ld_dx or self.d
        return j

    def _done(self, rc):
        if rc != 0:
            raise RuntimeError("the head's loss was refused or failed: %s"
                               % self.L.gpu_debug_last_error().decode())

    def run(self, x, w, bias, target, nll, scale=1.0, dx=None, dw=None, db=None, ld_x=None, ld_dx=None):
        """Device addresses: x, w bf16, bias float or None, target int32, nll float; dx is written, dw and db are added to."""
        if not self.grad and (dx or dw or db):
            raise ValueError("made for the loss alone")
        j = self._fill(x, target, nll, scale, dx, ld_x, ld_dx)
        j.d_w, j.d_bias, j.d_dw, j.d_db = w, bias, dw, db
        self._done(self.L.anni_head_loss(C.byref(j)))

    def run_on(self, opt, w_tensor, b_tensor, x, target, nll, scale=1.0, dx=None, ld_x=None, ld_dx=None):
        """The same on an LmAdam's head: weights from its twins, gradients into its gradient flat (grad=False: none);
        dx in that flat's type."""
        if not self.grad and dx:
            raise ValueError("made for the loss alone")
        j = self._fill(x, target, nll, scale, dx, ld_x, ld_dx)
        self._done(self.L.anni_adam_head_loss(opt.h, w_tensor, -1 if b_tensor is None else b_tensor, C.byref(j),
                                              int(self.grad)))

    def free(self):
        self.work.free()
        self.job.d_work, self.job.work_bytes = None, 0
