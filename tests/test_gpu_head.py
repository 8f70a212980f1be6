"""The head's loss and its gradients on the GPU against the 64-bit model (head_model.py): sizes around
every tile edge, strides and alignments, rows without targets, accumulation, pieces, streams, graphs."""
import ctypes as C

import numpy as np
import pytest

from head_model import Loss, bf16, widen
from helpers import same_bits
from test_gpu_graph import hip_runtime, ok

pytestmark = pytest.mark.gpu

F32, BF16, FP8 = 0, 1, 2
NP = {F32: np.float32, BF16: np.uint16}
GUARD = 64                  # bytes of a pattern on either side of every output


def store(a, grad_type):
    return np.ascontiguousarray(a, np.float32) if grad_type == F32 else bf16(a)


def value(a):
    return a.astype(np.float64) if a.dtype == np.float32 else widen(a)


class Buf:
    """Device memory with guard bytes around it; `skew` elements off its natural alignment."""

    def __init__(self, arr, skew=0):
        from anni_amd.lm_adam import DeviceBuffer
        arr = np.ascontiguousarray(arr)
        self.dt, self.shape, self.nbytes = arr.dtype, arr.shape, arr.nbytes
        self.at = GUARD + skew * arr.itemsize
        self.buf = DeviceBuffer(arr.nbytes + 2 * GUARD + 64)
        whole = np.full(self.buf.nbytes, 0xA5, np.uint8)
        whole[self.at:self.at + arr.nbytes] = np.frombuffer(arr.tobytes(), np.uint8)
        self.buf.upload(whole)
        self.ptr = self.buf.ptr + self.at

    def get(self):
        whole = self.buf.download(np.uint8, self.buf.nbytes)
        assert (whole[:self.at] == 0xA5).all() and (whole[self.at + self.nbytes:] == 0xA5).all(), "written outside"
        return np.frombuffer(whole[self.at:self.at + self.nbytes].tobytes(), self.dt).reshape(self.shape)


class Case:
    def __init__(self, rows, d, vocab, grad_type, seed=0, bias=True, pad=0.2, ld_x=None, ld_dx=None, skew=0,
                 size=1.0, model=True):
        rng = np.random.default_rng(seed + rows * 7 + d * 3 + vocab)
        self.rows, self.d, self.vocab, self.gt = rows, d, vocab, grad_type
        self.ld_x, self.ld_dx, self.skew = ld_x or d, ld_dx or d, skew
        self.x = bf16(rng.standard_normal((rows, self.ld_x)))
        self.w = bf16(rng.standard_normal((d, vocab)) * 1.5 * size / np.sqrt(d))
        self.b = rng.standard_normal(vocab).astype(np.float32) if bias else None
        self.target = rng.integers(0, vocab, rows).astype(np.int32)
        lost = rng.random(rows) < pad
        self.target[lost] = rng.choice([-1, -100, vocab, 2 ** 31 - 1, -2 ** 31], lost.sum())
        self.x[lost] = rng.choice(np.array([0x7FC0, 0x7F80, 0xFF80, 0x3F80], np.uint16), (lost.sum(), self.ld_x))
        self.scale = 0.75 / rows
        self.dw0 = store(rng.standard_normal((d, vocab)) * 1e-2 / rows, grad_type)
        self.db0 = store(rng.standard_normal(vocab) * 1e-2 / rows, grad_type)
        if model:
            self.model()

    def model(self):
        x = widen(self.x[:, :self.d])
        self.want = Loss(x, widen(self.w), self.b, self.target.astype(np.int64), self.scale, value(self.dw0),
                         value(self.db0))

    def place(self):
        k = self.skew
        self.dx_, self.dwx, self.dww = Buf(self.x, k), None, Buf(self.w, k)
        self.dbias = Buf(self.b, k) if self.b is not None else None
        self.dt, self.dnll = Buf(self.target, k), Buf(np.full(self.rows, 7e7, np.float32), k)
        self.ddx = Buf(np.full((self.rows, self.ld_dx), 0x4242, NP[self.gt]), k)
        self.ddw, self.ddb = Buf(self.dw0, k), Buf(self.db0, k)

    def run(self, plan, grad=True, parts=("dx", "dw", "db")):
        kw = dict(scale=self.scale, ld_x=self.ld_x, ld_dx=self.ld_dx)
        if grad:
            kw.update({k: v.ptr for k, v in (("dx", self.ddx), ("dw", self.ddw), ("db", self.ddb)) if k in parts})
        plan.run(self.dx_.ptr, self.dww.ptr, self.dbias.ptr if self.dbias else None, self.dt.ptr, self.dnll.ptr, **kw)

    def plan(self, grad=True):
        from anni_amd.head_loss import HeadLoss
        return HeadLoss(self.rows, self.d, self.vocab, self.gt, grad)

    def outputs(self):
        return self.dnll.get(), self.ddx.get(), self.ddw.get(), self.ddb.get()

    def check_nll(self):
        nll = self.dnll.get().astype(np.float64)
        w = self.want
        assert (np.abs(nll - w.nll) <= w.tol_nll).all(), float(np.max(np.abs(nll - w.nll) / w.tol_nll))
        assert (nll[~w.live] == 0).all()

    def check(self):
        self.check_nll()
        w = self.want
        _n, dx, dw, db = self.outputs()
        if self.ld_dx > self.d:
            assert (dx[:, self.d:] == np.full(1, 0x4242, NP[self.gt])[0]).all()      # the gap stays
        dx = dx[:, :self.d]
        assert (value(dx)[~w.live] == 0).all()
        # besides the bound on each element: the errors are many and of both signs, so their norm is no
        # more than half a step's share of the result's (the pair's and the sums' share for float)
        share = {F32: 2.0 ** -16, BF16: 2.0 ** -8}[self.gt]
        for name, got, want, tol in zip(("dx", "dw", "db"), (dx, dw, db), (w.dx, w.dw, w.db),
                                        w.tolerances(self.gt)):
            err = np.abs(value(got) - want)
            assert (err <= tol).all(), (name, float(np.max(err / tol)))
            assert np.linalg.norm(err) <= share * np.linalg.norm(want) + np.linalg.norm(w.eps_p) * 2 ** -6 * \
                np.linalg.norm(want), (name, float(np.linalg.norm(err) / np.linalg.norm(want)))


SIZES = [(1, 1, 1), (1, 64, 2), (2, 7, 130), (3, 65, 255), (63, 64, 256), (64, 130, 257), (65, 33, 512),
         (128, 64, 1003), (129, 331, 300), (256, 256, 256), (257, 128, 777), (300, 257, 1000)]


@pytest.mark.parametrize("grad_type", [F32, BF16])
@pytest.mark.parametrize("rows,d,vocab", SIZES)
def test_loss_and_gradients(gpu, rows, d, vocab, grad_type):
    c = Case(rows, d, vocab, grad_type, bias=(rows + d) % 3 != 0)
    c.place()
    plan = c.plan()
    c.run(plan)
    c.check()
    # once more: nll and dx the same bits, dw and db from what they are now
    nll, dx, c.dw0, c.db0 = c.outputs()
    c.model()
    c.run(plan)
    c.check()
    assert same_bits(nll, c.dnll.get()) and same_bits(dx, c.ddx.get())


@pytest.mark.parametrize("grad_type", [F32, BF16])
@pytest.mark.parametrize("rows,d,vocab", [(2500, 64, 256), (1030, 130, 131), (3000, 300, 70)])
def test_many_tokens_and_a_small_vocabulary(gpu, rows, d, vocab, grad_type):
    """dw has too few tiles for the chip: the tokens are cut into slices whose sums are added in order."""
    c = Case(rows, d, vocab, grad_type)
    c.place()
    plan = c.plan()
    c.run(plan)
    c.check()
    full = c.outputs()
    for parts in (("dw",), ("db",)):
        c.place()
        c.run(plan, parts=parts)
        for name, got, a, b in zip(("dw", "db"), c.outputs()[2:], full[2:], (c.dw0, c.db0)):
            assert same_bits(got, a if name in parts else b), name


@pytest.mark.parametrize("grad_type", [F32, BF16])
@pytest.mark.parametrize("rows,d,vocab,pad", [(150, 500, 403, 0.2), (1030, 270, 801, 0.0), (700, 520, 1001, 0.5)])
def test_odd_vocabularies_whose_weights_are_copied(gpu, rows, d, vocab, pad, grad_type):
    """Sizes at which the lines of w are laid out anew (the work area grows by d lines against an even vocabulary)."""
    even = gpu.anni_head_loss_work_bytes(rows, d, (vocab + 7) // 8 * 8, grad_type)
    assert gpu.anni_head_loss_work_bytes(rows, d, vocab, grad_type) >= even + d * vocab * 2
    c = Case(rows, d, vocab, grad_type, pad=pad, skew=1)
    c.place()
    plan = c.plan()
    plan.work.upload(np.full(plan.work.nbytes, 0xFF, np.uint8))
    c.run(plan)
    c.check()


@pytest.mark.parametrize("rows,d,vocab", SIZES)
def test_the_loss_alone_has_the_same_bits(gpu, rows, d, vocab):
    c = Case(rows, d, vocab, F32)
    c.place()
    c.run(c.plan())
    with_grad = c.dnll.get()
    c.place()
    c.run(c.plan(False), grad=False)
    c.check_nll()
    assert same_bits(with_grad, c.dnll.get())
    assert same_bits(c.ddw.get(), c.dw0) and same_bits(c.ddb.get(), c.db0)


@pytest.mark.parametrize("skew", [1, 2, 4, 8])
@pytest.mark.parametrize("grad_type", [F32, BF16])
def test_strides_and_alignment(gpu, grad_type, skew):
    c = Case(70, 72, 520, grad_type, ld_x=83, ld_dx=77, skew=skew)
    c.place()
    c.run(c.plan())
    c.check()


@pytest.mark.parametrize("parts", [("dx",), ("dw",), ("db",), ("dx", "db"), ("dw", "db")])
def test_some_of_the_gradients(gpu, parts):
    c = Case(70, 72, 520, BF16)
    c.place()
    c.run(c.plan())
    full = c.outputs()
    c.place()
    before = c.outputs()
    c.run(c.plan(), parts=parts)
    for name, got, a, b in zip(("nll", "dx", "dw", "db"), c.outputs(), full, before):
        assert same_bits(got, a if name == "nll" or name in parts else b), name


def test_no_row_has_a_target(gpu):
    c = Case(70, 72, 520, F32, pad=2.0)
    c.place()
    c.run(c.plan())
    nll, dx, dw, db = c.outputs()
    assert not nll.any() and not dx.any() and same_bits(dw, c.dw0) and same_bits(db, c.db0)


def test_masked_vocabulary(gpu):
    """Bias of -inf and of the lowest float: no probability, no gradient; a masked target has an infinite loss."""
    c = Case(66, 64, 700, F32, pad=0.0, model=False)
    c.b[::3] = -np.inf
    c.b[1::3] = np.finfo(np.float32).min
    c.target = (c.target // 3 * 3 + 2).astype(np.int32) % 699
    c.target[c.target % 3 != 2] = 2
    c.target[5] = 3                       # -inf
    c.model()
    assert np.isinf(c.want.nll[5]) and np.isfinite(np.delete(c.want.nll, 5)).all()
    c.place()
    c.run(c.plan())
    nll = c.dnll.get()
    assert np.isposinf(nll[5])
    keep = np.arange(66) != 5
    assert (np.abs(nll - c.want.nll)[keep] <= c.want.tol_nll[keep]).all()
    _n, dx, dw, db = c.outputs()
    for got, want, tol in zip((dx, dw, db), (c.want.dx, c.want.dw, c.want.db), c.want.tolerances(F32)):
        assert (np.abs(got - want) <= tol).all()
    untouched = (np.arange(700) % 3 != 2) & (np.arange(700) != 3)
    assert same_bits(dw[:, untouched].copy(), c.dw0[:, untouched].copy())


def test_values_that_are_not_finite_reach_what_they_belong_to(gpu):
    """A NaN in a live row: that row's loss and gradients, and dw and db (they sum over it); no other row's loss."""
    c = Case(70, 72, 520, F32, pad=0.0, model=False)
    c.x[9, 3] = 0x7FC0
    c.place()
    c.run(c.plan())
    nll, dx, dw, db = c.outputs()
    assert np.isnan(nll[9]) and np.isfinite(np.delete(nll, 9)).all()
    assert np.isnan(dx[9]).all() and np.isfinite(np.delete(dx, 9, 0)).all()
    assert np.isnan(dw).all() and np.isnan(db).all()


def test_weights_that_are_not_finite(gpu):
    """A column of -inf in the last lines of w (next to what pads the contracted axis): probability 0 or
    1 by the sign of x, as the formula has it."""
    c = Case(40, 70, 300, F32, pad=0.0, model=False)
    c.x[:, 69] = np.where(np.arange(40) % 2, 0x3F80, 0x4000)        # 1 and 2
    c.w[69, 17] = 0xFF80
    c.target[c.target == 17] = 18
    c.model()
    c.place()
    c.run(c.plan(False), grad=False)
    c.check_nll()
    assert np.isfinite(c.dnll.get()).all()


def test_extreme_logits(gpu):
    """Logits of thousands: the maximum is subtracted before any exponential."""
    c = Case(33, 64, 600, F32, size=300.0)
    assert np.abs(c.want.mag).max() > 1000          # an exponential overflows at 89
    c.place()
    c.run(c.plan())
    assert np.isfinite(c.dnll.get()).all()
    c.check_nll()


@pytest.mark.parametrize("rows,d,vocab,grad_type", [(2100, 24, 60001, F32), (4097, 24, 65000, BF16)])
def test_several_pieces_of_the_vocabulary(gpu, rows, d, vocab, grad_type):
    """Large enough that delta does not fit its part of the work area at once."""
    piece = 2.0 ** 29 / (((rows + 255) // 256 * 256) * (4 if grad_type == F32 else 2))
    assert vocab > piece
    c = Case(rows, d, vocab, grad_type, pad=0.3)
    c.place()
    c.run(c.plan())
    c.check()


@pytest.mark.parametrize("rows,d,vocab,grad_type", [(2100, 200, 60001, F32), (4097, 200, 65000, BF16),
                                                    (300, 200, 350100, F32), (300, 200, 350100, BF16)])
def test_logits_kept_or_computed_again_are_the_same_bits(gpu, rows, d, vocab, grad_type):
    """More than 512 MiB of logits: the least work area has no room for them.  (300 tokens: middle tiles.)"""
    from anni_amd.head_loss import HeadLoss
    least = gpu.anni_head_loss_work_bytes(rows, d, vocab, grad_type)
    most = gpu.anni_head_loss_work_bytes_keep(rows, d, vocab, grad_type)
    assert most - least >= rows * vocab * 4
    got = []
    for keep, size in ((False, least), (True, most)):
        c = Case(rows, d, vocab, grad_type, pad=0.3, model=False)
        c.place()
        plan = HeadLoss(rows, d, vocab, grad_type, keep=keep)
        assert plan.work.nbytes == size
        plan.work.upload(np.full(min(size, 1 << 30), 0xFF, np.uint8))
        c.run(plan)
        got.append([a.tobytes() for a in c.outputs()])
        plan.free()
    assert got[0] == got[1]


def test_more_logits_than_32_bits_count(gpu):
    """36000 x 60160 = 2.17e9 logits, kept and computed again: the same bits; some rows against 64 bits
    (with bf16 gradients: the bounds of one rounding of delta and of dx, as everywhere)."""
    from anni_amd.head_loss import HeadLoss
    rows, d, vocab = 36000, 200, 60160
    some = np.array([0, 1, 17999, 35712, 35713, 35999])
    got = []
    for keep in (True, False):
        c = Case(rows, d, vocab, BF16, pad=0.1, model=False)
        c.place()
        plan = HeadLoss(rows, d, vocab, BF16, keep=keep)
        c.run(plan)
        got.append(c.outputs())
        plan.free()
        assert all((a == b).all() for a, b in zip(got[0], got[-1]))
        for b in (c.dx_, c.dww, c.dbias, c.dt, c.dnll, c.ddx, c.ddw, c.ddb):
            b.buf.free()
    w = Loss(widen(c.x[some]), widen(c.w), c.b, c.target[some].astype(np.int64), c.scale)
    nll, dx = got[0][0][some].astype(np.float64), value(got[0][1][some])
    assert w.live.sum() > 1
    assert (np.abs(nll - w.nll) <= w.tol_nll).all()
    assert (np.abs(dx - w.dx) <= w.tolerances(BF16)[0]).all()


def test_dx_in_the_place_of_x(gpu):
    c = Case(130, 72, 520, BF16)
    c.place()
    c.ddx = c.dx_
    c.run(c.plan())
    c.check()


def test_a_freed_plan_is_refused(gpu):
    c = Case(8, 16, 40, F32, model=False)
    c.place()
    plan = c.plan()
    c.run(plan)
    plan.free()
    with pytest.raises(RuntimeError):
        c.run(plan)


def test_work_area_contents_do_not_matter(gpu):
    c = Case(70, 72, 520, F32)
    c.place()
    plan = c.plan()
    plan.work.upload(np.full(plan.work.nbytes, 0xFF, np.uint8))
    c.run(plan)
    c.check()


def test_two_calls_on_two_streams(gpu):
    hip = hip_runtime()
    cases = [Case(200, 72, 5000, F32, seed=1), Case(90, 130, 3001, BF16, seed=2)]
    streams = [C.c_void_p(), C.c_void_p()]
    plans = [c.plan() for c in cases]
    for c, s in zip(cases, streams):
        c.place()
        ok(hip.hipStreamCreate(C.byref(s)), "hipStreamCreate")
    try:
        for c, s, p in zip(cases, streams, plans):
            gpu.anni_gpu_set_stream(s)
            c.run(p)
        for s in streams:
            ok(hip.hipStreamSynchronize(s), "hipStreamSynchronize")
        gpu.anni_gpu_set_stream(None)
        for c in cases:
            c.check()
    finally:
        gpu.gpu_device_sync()
        gpu.anni_gpu_set_stream(None)
        for s in streams:
            hip.hipStreamDestroy(s)


def test_replays_from_a_captured_graph(gpu):
    hip = hip_runtime()
    c = Case(150, 72, 1500, F32)
    c.place()
    plan = c.plan()
    c.run(plan)
    want = c.outputs()
    stream = C.c_void_p()
    ok(hip.hipStreamCreate(C.byref(stream)), "hipStreamCreate")
    gpu.anni_gpu_set_stream(stream)
    try:
        graph, gexec = C.c_void_p(), C.c_void_p()
        gpu.anni_gpu_flush()
        ok(hip.hipStreamBeginCapture(stream, 2), "hipStreamBeginCapture")
        c.run(plan)
        ok(hip.hipStreamEndCapture(stream, C.byref(graph)), "hipStreamEndCapture")
        hip.hipGraphInstantiate.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
        ok(hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0), "hipGraphInstantiate")
        for _k in range(4):
            c.ddw.buf.upload(c.dw0, c.ddw.at)
            c.ddb.buf.upload(c.db0, c.ddb.at)
            plan.work.upload(np.full(plan.work.nbytes, 0x7F, np.uint8))
            ok(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
            ok(hip.hipStreamSynchronize(stream), "hipStreamSynchronize")
            for a, b in zip(want, c.outputs()):
                assert same_bits(a, b)
        ok(hip.hipGraphExecDestroy(gexec), "hipGraphExecDestroy")
        ok(hip.hipGraphDestroy(graph), "hipGraphDestroy")
    finally:
        gpu.gpu_device_sync()
        gpu.anni_gpu_set_stream(None)
        hip.hipStreamDestroy(stream)


@pytest.mark.parametrize("grad_type,moment_type", [(F32, F32), (BF16, 3), (F32, 3)])
def test_a_training_step_of_the_head(gpu, oracle, grad_type, moment_type):
    """Two microbatches' losses into an arena's gradient flat, then the step; the next loss reads the new twins."""
    from anni_amd.head_loss import HeadLoss
    from anni_amd.lm_adam import LmAdam
    rows, d, vocab = 90, 72, 1003
    tensors = [("w_head", d * vocab, 3), ("b_head", vocab, 0), ("rest", 5001, 3)]
    opt = LmAdam(tensors, grad_type=grad_type, moment_type=moment_type, beta2=0.95, weight_decay=0.1)
    rng = np.random.default_rng(5)
    p = (rng.standard_normal(opt.n) * 0.1).astype(np.float32)
    opt.upload("param", p)
    opt.seed_twins()
    plan, ev = HeadLoss(rows, d, vocab, grad_type), HeadLoss(rows, d, vocab, grad_type, grad=False)
    nll = Buf(np.zeros(rows, np.float32))
    batches = []
    for k in range(2):
        c = Case(rows, d, vocab, grad_type, seed=k)
        batches.append((c, Buf(c.x), Buf(c.target), Buf(np.zeros((rows, d), NP[grad_type]))))
    dw0 = np.zeros((d, vocab), NP[grad_type])
    db0 = np.zeros(vocab, NP[grad_type])
    for c, x, t, dx in batches:
        plan.run_on(opt, 0, 1, x.ptr, t.ptr, nll.ptr, c.scale, dx=dx.ptr)
        c.w, c.b, c.dw0, c.db0 = bf16(p[:d * vocab]).reshape(d, vocab), p[d * vocab:d * vocab + vocab], dw0, db0
        c.model()
        g = opt.download("grad")
        dw0, db0 = g[:d * vocab].reshape(d, vocab), g[d * vocab:d * vocab + vocab]
        assert not g[d * vocab + vocab:].any()
        c.dnll, c.ddx = nll, dx
        c.ddw = c.ddb = None
        c.check_nll()
        tol = c.want.tolerances(grad_type)
        for got, want, t_ in zip((dx.get(), dw0, db0), (c.want.dx, c.want.dw, c.want.db), tol):
            assert (np.abs(value(got) - want) <= t_).all()
    assert opt.step_scaled(1e-3) == 0
    assert not opt.download("grad").any()
    q = opt.download("param")
    c, x, t, _dx = batches[0]
    ev.run_on(opt, 0, 1, x.ptr, t.ptr, nll.ptr)
    c.w, c.b = bf16(q[:d * vocab]).reshape(d, vocab), q[d * vocab:d * vocab + vocab]
    c.model()
    c.check_nll()
    opt.free()


def test_refusals_on_an_arena(gpu):
    from anni_amd import lib
    from anni_amd.head_loss import HeadLoss
    from anni_amd.lm_adam import LmAdam
    d, vocab, rows = 16, 40, 8
    x, t, nll = Buf(np.zeros((rows, d), np.uint16)), Buf(np.zeros(rows, np.int32)), Buf(np.zeros(rows, np.float32))
    plan = HeadLoss(rows, d, vocab, F32)

    def tries(w, b, grad=True, width=d, **kw):
        opt = LmAdam([(d * vocab, 3), (vocab, 0), (77, 0)], **kw)
        plan.grad = grad
        plan.d = plan.job.d = width
        try:
            plan.run_on(opt, w, b, x.ptr, t.ptr, nll.ptr)
        finally:
            opt.free()

    tries(0, 1)
    tries(0, None)
    tries(0, 1, grad=False, grad_type=FP8)
    for args, kw in (((0, 2), {}), ((0, 3), {}), ((-1, 1), {}), ((3, 1), {}), ((2, None), {}),
                     ((0, 1), dict(grad_type=FP8)), ((0, 1), dict(twins=False)), ((0, 1), dict(grad_slots=0)),
                     ((0, 1), dict(width=15)), ((0, 0), {}), ((1, None), dict(width=8)), ((1, None), dict(width=40))):
        with pytest.raises(RuntimeError):
            tries(*args, **kw)
    with pytest.raises(ValueError):
        HeadLoss(rows, d, vocab, FP8)
    with pytest.raises(ValueError):
        HeadLoss(rows, d, vocab, F32, grad=False).run(x.ptr, x.ptr, None, t.ptr, nll.ptr, dx=x.ptr)
    with pytest.raises(ValueError):
        HeadLoss(rows, d, vocab, F32, grad=False).run_on(None, 0, 1, x.ptr, t.ptr, nll.ptr, dx=x.ptr)
    assert lib.load().anni_head_loss_work_bytes(rows, d, vocab, F32) == plan.work.nbytes
