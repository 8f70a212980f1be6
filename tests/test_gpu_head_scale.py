"""The scale of the head's gradients: whatever it is, it is one factor of float sums, not a rounding that all tokens share."""
import numpy as np
import pytest

from head_model import widen
from test_gpu_head import BF16, F32, Case, value

pytestmark = pytest.mark.gpu


def half_steps(x):
    """Half a step of bf16 at each float64 number."""
    m, e = np.frexp(x)
    return np.where(x == 0, 2.0 ** -134, np.ldexp(1.0, e - 9))


# the middle of two bf16 numbers, a third, a power of two, a mean over tokens, loss scales, nothing
@pytest.mark.parametrize("scale", [(1 + 2.0 ** -8) / 64, 1 / 3.0, 2.0 ** -7, 1 / 96.0, 65536.0, -1.7, 0.0])
@pytest.mark.parametrize("rows,d,vocab", [(96, 72, 5000), (300, 200, 20003)])
def test_bf16_gradients_are_the_formulas_rounded(gpu, rows, d, vocab, scale):
    """A fresh head: every probability is about 1 / vocab, so delta is -scale at the target and next to nothing elsewhere.
    Its own rounding costs at most p of the target's 1 - p (p < 4 / vocab: the logits' deviation is 0.3) and half a step,
    2^-8, of what the other places give together, sqrt(rows / vocab) of the norm.  The rest is the result's
    rounding: an error within half a step, 1 / sqrt(3) of it in the mean square if it is spread evenly and 0.63
    where every result is a number of eight bits times 1 + 2^-8."""
    c = Case(rows, d, vocab, BF16, size=0.2, pad=0.2, bias=False, model=False)
    c.scale = scale
    c.dw0[:], c.db0[:] = 0, 0
    c.model()
    c.place()
    c.run(c.plan())
    _n, dx, dw, db = c.outputs()
    w = c.want
    for name, got, want in (("dx", dx, w.dx), ("dw", dw, w.dw), ("db", db, w.db)):
        err = np.linalg.norm(value(got) - want)
        bound = (1.0 if name == "db" else 0.75) * np.linalg.norm(half_steps(want))      # (db's errors are all alike)
        small = (4.0 / vocab + 2.0 ** -8 * np.sqrt((1 + rows) / vocab)) * np.linalg.norm(want)
        assert err <= bound + small, (name, err / np.linalg.norm(want), bound / np.linalg.norm(want))


@pytest.mark.parametrize("grad_type", [F32, BF16])
def test_a_power_of_two_scales_the_bits(gpu, grad_type):
    """The same gradients times 2^k, exactly: scale enters once."""
    outs = []
    for k in (0, -12, 9):
        c = Case(130, 200, 2051, grad_type, model=False)
        c.scale = 2.0 ** k
        c.dw0[:], c.db0[:] = 0, 0
        c.place()
        c.run(c.plan())
        outs.append([value(a) * 2.0 ** -k for a in c.outputs()[1:]])
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            # what a smaller scale pushes below the smallest normal number keeps fewer bits
            normal = np.abs(a) > 2.0 ** -110
            assert (a[normal] == b[normal]).all()
