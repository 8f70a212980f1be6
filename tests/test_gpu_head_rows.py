"""Rows without a target in the gradients of the head's loss, when w or the bias is not finite: 0 times infinity
is NaN, but such a row's dx is 0 and nothing of it reaches dw and db."""
import numpy as np
import pytest

from head_model import Loss, widen
from test_gpu_head import BF16, F32, Case, value

pytestmark = pytest.mark.gpu


# rows, d, vocab: dx in slices; in one slot; rows that a tile of any shape is not full of
@pytest.mark.parametrize("grad_type", [F32, BF16])
@pytest.mark.parametrize("bits", [0xFF80, 0x7F80, 0x7FC0])
@pytest.mark.parametrize("rows,d,vocab", [(40, 70, 300), (257, 200, 2051), (1, 9, 20)])
def test_dx_is_zero_whatever_w_holds(gpu, rows, d, vocab, bits, grad_type):
    """One line of w, one element of it, is -inf, inf or NaN.  A live row's dx is what the formula says: NaN at that
    line of w (0 times infinity, or a NaN), everywhere if the logit itself is not a number's."""
    c = Case(rows, d, vocab, grad_type, pad=0.0, model=False)
    line, place = d - 1, vocab - 3
    c.x[:, line] = 0x3F80                           # 1: the place's logit has w's sign
    c.w[line, place] = bits
    c.target[c.target == place] = 0
    dead = np.arange(rows) % 3 == 1 if rows > 1 else np.ones(1, bool)
    c.target[dead] = np.resize([-1, vocab, -2 ** 31], dead.sum())
    c.x[dead] = np.resize(np.array([0x7FC0, 0xFF80, 0x3F80], np.uint16), (dead.sum(), c.ld_x))
    c.place()
    c.run(c.plan())
    nll, dx, dw, db = c.outputs()
    assert not dx[dead].any() and not nll[dead].any()           # the bits of +0
    if rows == 1:
        assert (value(dw) == value(c.dw0)).all() and (value(db) == value(c.db0)).all()
        return
    got = value(dx)[~dead]
    if bits != 0xFF80:
        assert np.isnan(got).all() and np.isnan(nll[~dead]).all()
        return
    # probability 0 at that place: the rest is the loss of the vocabulary without it
    keep = np.arange(vocab) != place
    w = widen(c.w)
    w[line, place] = 0.0
    at = c.target.astype(np.int64)
    at = np.where(dead, -1, at - (at > place))
    L = Loss(widen(c.x), w[:, keep], c.b[keep], at, c.scale, value(c.dw0)[:, keep], value(c.db0)[keep])
    assert (np.abs(nll - L.nll) <= L.tol_nll)[~dead].all()
    assert np.isnan(got[:, line]).all()
    tol_dx, tol_dw, tol_db = L.tolerances(grad_type)
    # the place's own delta is 0 and adds the smallest number of delta's type to the bound
    ok = np.arange(d) != line
    assert (np.abs(got - L.dx[~dead])[:, ok] <= tol_dx[~dead][:, ok] + 2.0 ** -100).all()
    assert (np.abs(value(dw)[:, keep] - L.dw) <= tol_dw).all() and (np.abs(value(db)[keep] - L.db) <= tol_db).all()
    assert (value(dw)[:, place] == value(c.dw0)[:, place]).all() and value(db)[place] == value(c.db0)[place]


@pytest.mark.parametrize("grad_type", [F32, BF16])
def test_a_bias_that_is_infinite(gpu, grad_type):
    """Every live row has no distribution then; the others still take no part."""
    c = Case(70, 72, 520, grad_type, model=False)
    c.b[7] = np.inf
    live = (c.target >= 0) & (c.target < 520)
    c.place()
    c.run(c.plan())
    nll, dx, _dw, _db = c.outputs()
    assert not dx[~live].any() and not nll[~live].any()
    assert np.isnan(value(dx)[live]).all() and np.isnan(nll[live]).all()
