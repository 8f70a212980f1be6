"""Every kernel that a call of the head's loss can be made of, against the 64-bit model: the three shapes of the
logits' tiles with and without kept logits, of dx, and the two of dw with one or more slices, over one piece of the
vocabulary and several, each with float and bf16 gradients.  test_head_plan.py holds that the list covers them."""
import numpy as np
import pytest

from head_samples import Samples, edges
from test_gpu_head import BF16, F32, Case, value

pytestmark = pytest.mark.gpu

# rows, d, vocab, gradient type, padding; those whose logits do not always stay run with both work areas
GRADIENTS = [(rows, d, vocab, ty, pad) for rows, d, vocab, pad in [
    (254, 64, 256, 0.0),            # small tiles, dx and dw in slices
    (777, 331, 10007, 0.55),        # middle tiles, lines that are not aligned
    (300, 130, 20003, 0.2),         # middle tiles, the logits computed again
    (70, 499, 32701, 0.2),          # middle tiles, dw in large ones whose lines end inside them
    (1020, 499, 32704, 0.2),        # large tiles everywhere
    (1020, 257, 16381, 0.1),        # large tiles, lines that are not aligned
    (2040, 257, 16381, 0.1),        # the same with w copied
    (2040, 130, 16381, 0.1),        # large tiles, the logits computed again, middle dx
    (4000, 700, 250, 0.2),          # a vocabulary so short that dx is not cut
    (96, 1536, 100000, 0.1),        # few tokens of a wide head
] for ty in (F32, BF16)] + [
    (8300, 24, 30000, F32, 0.3),    # several pieces of the vocabulary: dw in slices in each
    (16500, 24, 30000, BF16, 0.3),
    (2100, 499, 60001, F32, 0.3),   # and dw in large tiles, the logits kept or computed again
    (4097, 499, 66000, BF16, 0.3),
] + [(rows, d, vocab, ty, 0.2) for rows, d, vocab in [      # each axis at its end
    (1 << 22, 1, 2), (5, 8, 1 << 22), (3, 1 << 16, 40), (262149, 24, 130)] for ty in (F32, BF16)]
LOSSES = [(254, 64, 256, True), (777, 331, 10007, True), (517, 712, 50257, False), (1020, 257, 16381, False),
          (2040, 257, 16381, True), (1020, 512, 32768, False)]


def some(c, seed):
    """Rows and columns on either side of the tiles' edges (as many as a quick model allows) and drawn ones."""
    rng = np.random.default_rng(seed)
    rows = edges(c.rows, 256, rng, 12)
    cols = edges(c.vocab, 256, rng, 24)
    if rows.size * c.vocab > 4 << 20:
        rows = np.unique(np.concatenate([rows[:4], rows[-4:], rng.choice(rows, 24)]))
    return rows, cols if cols.size <= 320 else np.unique(np.concatenate([cols[:16], cols[-16:], rng.choice(cols, 256)]))


# The bound of an element takes every rounding at its worst and the same sign.  Together they are many and of both
# signs, and their norm is that of random walks.  Float: a logit here is below 9 and so are its partial sums,
# sqrt(1536) of them round by 2^-23 of that each: 2^-14.6; the sum over a vocabulary of 10^5 adds
# sqrt(10^5) 2^-24 = 2^-15.7, the pair 2^-17, the exponential 20 * 2^-23: together below 2^-13, a 16th of what
# delta without its low half would leave.  bf16: half a step of delta and half a step of the result.
SHARE = {F32: 2.0 ** -13, BF16: 2.0 ** -7}


def near(name, got, want, tol, share=np.inf):
    err = np.abs(got - want)
    assert (err <= tol).all(), (name, float(np.max(err / tol)))
    assert np.linalg.norm(err) <= share * np.linalg.norm(want), (name, np.linalg.norm(err) / np.linalg.norm(want))


@pytest.mark.parametrize("rows,d,vocab,grad_type,pad", GRADIENTS)
def test_gradients_of_every_shape(gpu, rows, d, vocab, grad_type, pad):
    from anni_amd.head_loss import HeadLoss
    c = Case(rows, d, vocab, grad_type, pad=pad, model=False)
    at = some(c, rows)
    want = Samples(c, *at)
    least = gpu.anni_head_loss_work_bytes(rows, d, vocab, grad_type)
    most = gpu.anni_head_loss_work_bytes_keep(rows, d, vocab, grad_type)
    first = None
    for keep in [False, True] if most > least else [True]:
        c.place()
        plan = HeadLoss(rows, d, vocab, grad_type, keep=keep)
        plan.work.upload(np.full(min(plan.work.nbytes, 1 << 28), 0xFF, np.uint8))
        c.run(plan)
        out = c.outputs()
        nll, dx, dw, db = out
        near("nll", nll.astype(np.float64), want.nll, want.tol_nll)
        assert (nll[~want.live] == 0).all() and (value(dx)[~want.live] == 0).all()
        near("dx", value(dx[at[0]]), want.dx, want.tol_dx, SHARE[grad_type])
        near("dw", value(dw[:, at[1]]), want.dw, want.tol_dw, SHARE[grad_type])
        near("db", value(db[at[1]]), want.db, want.tol_db, SHARE[grad_type])
        if first:
            assert [a.tobytes() for a in out] == first
        first = [a.tobytes() for a in out]
        plan.free()
        for b in (c.dx_, c.dww, c.dbias, c.dt, c.dnll, c.ddx, c.ddw, c.ddb):
            b.buf.free()


@pytest.mark.parametrize("rows,d,vocab,bias", LOSSES)
def test_losses_of_every_shape(gpu, rows, d, vocab, bias):
    c = Case(rows, d, vocab, F32, bias=bias, pad=0.3, model=False)
    want = Samples(c, [0], [0])
    c.place()
    plan = c.plan(False)
    c.run(plan, grad=False)
    nll = c.dnll.get()
    near("nll", nll.astype(np.float64), want.nll, want.tol_nll)
    assert (nll[~want.live] == 0).all()
    c.run(plan, grad=False)
    assert c.dnll.get().tobytes() == nll.tobytes()
    plan.free()
