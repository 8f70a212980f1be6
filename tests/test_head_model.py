"""The oracle of the head's loss against differences, and what its entry points refuse (no device needed)."""
import ctypes as C

import numpy as np
import pytest

from head_model import Loss, bf16, widen


def small(seed, rows=5, d=4, vocab=7):
    rng = np.random.default_rng(seed)
    x, w = widen(bf16(rng.standard_normal((rows, d)))), widen(bf16(rng.standard_normal((d, vocab))))
    b = rng.standard_normal(vocab).astype(np.float32)
    target = rng.integers(0, vocab, rows).astype(np.int32)
    target[1], target[3] = -1, vocab
    return x, w, b, target


@pytest.mark.parametrize("seed", [0, 1])
def test_gradients_of_the_model_against_differences(seed):
    x, w, b, target = small(seed)
    scale, h = 0.37, 1e-6
    L = Loss(x, w, b, target, scale)

    def total(x, w, b):
        return Loss(x, w, b.astype(np.float64), target, scale).nll.sum() * scale

    for arr, grad, put in ((x, L.dx, 0), (w, L.dw, 1), (b.astype(np.float64), L.db, 2)):
        for at in np.ndindex(arr.shape):
            up, down = arr.copy(), arr.copy()
            up[at] += h
            down[at] -= h
            args = [x, w, b.astype(np.float64)]
            hi, lo = list(args), list(args)
            hi[put], lo[put] = up, down
            # the difference's own error: h^2 times a third derivative of order 10, and 2^-53 * 20 / h
            assert abs((total(*hi) - total(*lo)) / (2 * h) - grad[at]) < 1e-8


def test_rows_without_a_target_take_no_part():
    x, w, b, target = small(2)
    a = Loss(x, w, b, target, 1.0)
    x[1], x[3] = np.nan, np.inf
    c = Loss(x, w, b, target, 1.0)
    assert (a.nll == c.nll).all() and (a.dw == c.dw).all() and (a.dx[[1, 3]] == 0).all() and a.nll[1] == a.nll[3] == 0


def test_work_area_sizes_and_refusals():
    from anni_amd import lib
    L = lib.load()
    f = L.anni_head_loss_work_bytes
    loss, bf, f32 = (f(4096, 1536, 100000, t) for t in (-1, lib.BF16, lib.F32))
    assert 0 < loss < bf <= f32
    assert f32 < 4096 * 100000 * 4          # less than the logits it avoids
    g = L.anni_head_loss_work_bytes_keep
    assert g(4096, 1536, 100000, lib.BF16) >= bf + 4096 * 100000 * 4 and g(4096, 1536, 100000, -1) == loss
    assert g(96, 1536, 100000, lib.BF16) == f(96, 1536, 100000, lib.BF16) and g(0, 8, 8, lib.F32) == 0
    assert f(1, 1, 1, -1) > 0 and f(1 << 22, 64, 256, lib.BF16) > 0
    for rows, d, vocab, ty in ((0, 8, 8, -1), (-1, 8, 8, -1), (8, 0, 8, -1), (8, 8, 0, -1), (8, 8, 8, -2),
                               (8, 8, 8, lib.FP8_E4M3), (8, 8, 8, lib.Q8), ((1 << 22) + 1, 8, 8, -1),
                               (8, (1 << 16) + 1, 8, -1), (8, 8, (1 << 22) + 1, -1),
                               ((1 << 20) + 1, 8, 1 << 18, -1)):
        assert f(rows, d, vocab, ty) == 0


def test_bad_jobs_are_refused():
    """Every refusal comes from the host's checks: nothing is launched with or without a device."""
    from anni_amd import lib
    L = lib.load()
    base = dict(rows=8, d=16, vocab=32, d_x=4096, ld_x=16, d_w=4096, d_target=4096, d_nll=4096, scale=1.0,
                d_work=4096, work_bytes=L.anni_head_loss_work_bytes(8, 16, 32, lib.F32))
    bad = [dict(d_x=None), dict(d_w=None), dict(d_target=None), dict(d_nll=None), dict(d_work=None),
           dict(rows=0), dict(d=0), dict(vocab=0), dict(rows=-3), dict(ld_x=15), dict(d_x=4097), dict(d_w=4097),
           dict(d_target=4098), dict(d_nll=4097), dict(d_bias=4098), dict(d_work=4096 + 128),
           dict(work_bytes=L.anni_head_loss_work_bytes(8, 16, 32, -1) - 1),
           dict(d_dx=4096, ld_dx=15), dict(d_dx=4098, ld_dx=16), dict(d_dw=4098), dict(d_db=4098),
           dict(d_dw=4097, grad_type=lib.BF16), dict(d_dw=4096, grad_type=lib.FP8_E4M3),
           dict(d_dw=4096, grad_type=lib.Q8), dict(d_dw=4096, grad_type=-1),
           dict(d_dw=4096, work_bytes=base["work_bytes"] - 1)]
    for change in bad:
        j = lib.HeadJob()
        for k, v in dict(base, **change).items():
            setattr(j, k, v)
        assert L.anni_head_loss(C.byref(j)) == -1, change
    assert L.anni_head_loss(None) == -1
    assert L.anni_adam_head_loss(None, 0, 1, C.byref(lib.HeadJob()), 0) == -1
