"""The arena with 8-bit moments (ANNI_Q8): every step against the C oracle on the decoded moments
and the numpy model of the storage (q8_model.py): codes and exponents bit for bit, p to a last place
in at most a few elements (its step is within 2^-43, see near())."""
import ctypes as C
import tempfile

import numpy as np
import pytest

import q8_model as q8
from helpers import same_bits
from test_gpu_graph import hip_runtime, ok

pytestmark = pytest.mark.gpu

F32, BF16, FP8, Q8 = 0, 1, 2, 3
LISTS = {
    "one": [(1, 3)],
    "three": [(3, 1)],
    "block": [(256, 3)],
    "block+1": [(257, 3)],
    "tile": [(4096, 3)],
    "ragged": [(5000, 3), (3, 0), (0, 3), (4096 * 3, 3), (1, 1), (8191, 2), (255, 3), (40001, 3), (1023, 0)],
    "many": [(70, 3), (1, 0)] * 120 + [(4096 * 3, 3), (9, 2)],     # more tensors than helpers are started for
    "tails": [(70, 0)] * 40 + [(4096 * 2 + 5, 3)],
}


def new_arena(tensors, grad_type=F32, **kw):
    from anni_amd.lm_adam import LmAdam
    kw = dict(dict(beta2=0.95, weight_decay=0.1, grad_clip=1.0, skip_nonfinite=True), **kw)
    return LmAdam(tensors, grad_type=grad_type, moment_type=Q8, **kw), kw


def near(got, want):
    """The step on p is within 2^-43 of the host loop's, |step| <= lr (m and v of one history bound it by
    a few lr) and p moves by less than 2^3 times itself here: the float it rounds to can be the
    neighbour, when the exact value lies within 2^-43 |step| of the middle of two.  That is one
    element in 2^43 ulp(p) / |step| > 2^17 for the smallest p of these tests and 10^8 for ordinary ones:
    of the up to 70000 here at most three are let pass."""
    same = got.view(np.uint32) == want.view(np.uint32)
    return np.count_nonzero(~same) <= 3 and (np.abs(got.astype(np.float64) - want)
                                             <= np.spacing(np.abs(want)))[~same].all()


class Model:
    """Oracle + storage model of one arena."""

    def __init__(self, oracle, opt, tensors, grad_type, kw, p, scales=None):
        self.opt, self.oracle, self.n, self.gt = opt, oracle, opt.n, grad_type
        self.tensors, self.P = tensors, p.copy()
        self.M = np.zeros(self.n, np.float32)
        self.V = np.zeros(self.n, np.float32)
        scales = np.ones(len(tensors), np.float32) if scales is None else scales
        segs = [(opt.offsets[i], t[0], t[1] & 1, float(scales[i])) for i, t in enumerate(tensors)]
        kw = {k: v for k, v in kw.items() if k != "grad_slots"}
        self.O = oracle.Oracle(self.n, tensors=segs, grad_type=grad_type, **kw)

    def step(self, g, lr, t_before=None, grad_scale=1.0):
        st = self.opt.sync_stats()
        if t_before is not None:
            self.O.o.t = t_before
        self.O.step(self.P, g.copy(), self.M, self.V, lr, grad_scale=grad_scale, sumsq_override=st.last_sumsq)
        assert st.last_clipped == self.O.o.last_clipped and st.last_skipped == self.O.o.last_skipped
        t = self.O.o.t
        if not st.last_skipped:
            rm, rv = q8.dither(self.n, t)
            self.cm, self.bm = q8.encode_m(self.M, rm)
            self.cv, self.bv = q8.encode_v(self.V, rv)
            self.M, self.V = q8.decode_m(self.cm, self.bm), q8.decode_v(self.cv, self.bv)

    def check(self):
        o = self.opt
        got = o.download("param")
        assert near(got, self.P)
        self.P = got                        # the next step starts from the same p
        assert (o.download("m_exp") == self.bm).all() and (o.download("v_exp") == self.bv).all()
        assert (o.download("m") == self.cm).all() and (o.download("v") == self.cv).all()
        assert not o.download("grad").any()
        if o.o.d_param_bf16:
            tw = o.download("twin")
            for i, t in enumerate(self.tensors):
                a = o.offsets[i]
                want = self.oracle.bf16_rne(self.P[a:a + t[0]]) if t[1] & 2 else np.zeros(t[0], np.uint16)
                assert (tw[a:a + t[0]] == want).all()


def gradients(oracle, rng, tensors, grad_type, size):
    """A gradient in storage form whose tensors differ in magnitude, and per-tensor scales (fp8)."""
    n = sum(t[0] for t in tensors)
    g = rng.standard_normal(n)
    at = 0
    for k, t in enumerate(tensors):
        g[at:at + t[0]] *= 10.0 ** (k % 5 - 2)
        at += t[0]
    g = (g * (size / max(np.sqrt((g * g).sum()), 1e-30))).astype(np.float32)
    scales = np.ones(len(tensors), np.float32)
    if grad_type == BF16:
        return oracle.bf16_rne(g), scales
    if grad_type == FP8:
        q, at = np.zeros(n, np.uint8), 0
        for k, t in enumerate(tensors):
            if t[0]:
                q[at:at + t[0]], scales[k] = oracle.fp8_quantize(g[at:at + t[0]])
            at += t[0]
        return q, scales
    return g, scales


@pytest.mark.parametrize("which", sorted(LISTS))
@pytest.mark.parametrize("grad_type", [F32, BF16, FP8])
def test_steps_equal_the_oracle_and_the_storage_model(gpu, oracle, which, grad_type):
    tensors = LISTS[which]
    opt, kw = new_arena(tensors, grad_type)
    rng = np.random.default_rng(len(which) + grad_type)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    model = None
    for k in range(5):
        g, scales = gradients(oracle, rng, tensors, grad_type, 2.0 if k % 2 else 0.3)
        opt.upload("grad", g)
        if grad_type == FP8:
            opt.upload("gscale", scales)
        if model is None:
            model = Model(oracle, opt, tensors, grad_type, kw, p, scales)
        if grad_type == FP8:
            model.O.set_gscales(scales)
        assert opt.step_scaled(1e-3 * (k + 1), 0.5) == 0
        model.step(g, 1e-3 * (k + 1), grad_scale=0.5)
        model.check()
    opt.free()


def test_external_gradients_that_are_not_aligned(gpu, oracle):
    from anni_amd.lm_adam import DeviceBuffer
    tensors = LISTS["ragged"]
    opt, kw = new_arena(tensors, F32, grad_slots=0)
    buf = DeviceBuffer(4 * opt.n + 64)
    opt.bind_grad(buf.ptr + 4)
    rng = np.random.default_rng(3)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    model = Model(oracle, opt, tensors, F32, kw, p)
    for _k in range(2):
        g, _s = gradients(oracle, rng, tensors, F32, 0.5)
        buf.upload(g, 4)
        opt.step_scaled(1e-3)
        model.step(g, 1e-3)
        model.check()
    opt.free()


def test_extremes_of_the_state(gpu, oracle):
    """Huge, tiny, subnormal and vanishing moments; blocks of zeros; signs of zeros."""
    tensors = [(256 * 40 + 17, 3)]
    opt, kw = new_arena(tensors, F32, grad_clip=0.0)
    n = opt.n
    rng = np.random.default_rng(4)
    p = (rng.standard_normal(n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    model = Model(oracle, opt, tensors, F32, kw, p)
    for k in range(4):
        size = np.repeat(10.0 ** np.linspace(-44, 18, 41), 256)[:n]
        g = (rng.standard_normal(n) * size * 10.0 ** rng.uniform(-6, 0, n)).astype(np.float32)
        g[256 * 3:256 * 4] = 0.0
        g[256 * 5:256 * 5 + 9] = -0.0
        g[256 * 7 + 1:256 * 8] = 0.0
        opt.upload("grad", g)
        opt.step_scaled(1e-3)
        model.step(g, 1e-3)
        model.check()
    opt.free()


def test_without_skip_a_gradient_that_is_not_finite_poisons_its_block(gpu, oracle):
    tensors = [(256 * 20, 3)]
    opt, kw = new_arena(tensors, F32, grad_clip=0.0, skip_nonfinite=False)
    rng = np.random.default_rng(5)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    g = (rng.standard_normal(opt.n) * 1e-3).astype(np.float32)
    g[256 * 2 + 5] = np.nan
    g[256 * 4 + 5] = np.inf
    g[256 * 6 + 5] = 1e25           # only v overflows
    opt.upload("grad", g)
    opt.step_scaled(1e-3)
    bm, bv = opt.download("m_exp"), opt.download("v_exp")
    assert (np.flatnonzero(bm == 255) == [2, 4]).all() and (np.flatnonzero(bv == 255) == [2, 4, 6]).all()
    after = opt.download("param")
    assert np.flatnonzero(np.isnan(after)).tolist() == [256 * 2 + 5, 256 * 4 + 5]   # as the host loop leaves it
    pairs = opt.export_mv()
    assert np.isnan(pairs[512:768]).all() and np.isnan(pairs[256 * 6:256 * 7, 1]).all()
    assert np.isfinite(pairs[256 * 6:256 * 7, 0]).all() and np.isfinite(pairs[768:1024]).all()
    opt.upload("grad", np.zeros(opt.n, np.float32))
    opt.step_scaled(1e-3)
    after = opt.download("param").reshape(-1, 256)
    assert np.isnan(after[[2, 4, 6]]).all() and np.isfinite(np.delete(after, [2, 4, 6], 0)).all()
    opt.free()


def test_without_eps_a_place_without_gradients_is_the_host_loops_nan(gpu, oracle):
    tensors = [(4096 * 2 + 300, 3)]
    opt, kw = new_arena(tensors, F32, eps=0.0, grad_clip=0.0)
    rng = np.random.default_rng(16)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    g = (rng.standard_normal(opt.n) * 1e-3).astype(np.float32)
    g[[5, 4100, 8400]] = 0.0
    opt.upload("grad", g)
    opt.step_scaled(1e-3)
    assert np.flatnonzero(np.isnan(opt.download("param"))).tolist() == [5, 4100, 8400]
    opt.free()


def test_an_endless_eps_moves_nothing(gpu, oracle):
    opt, kw = new_arena([(4096 * 2 + 300, 0)], F32, eps=np.inf, grad_clip=0.0)
    rng = np.random.default_rng(17)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    opt.upload("grad", (rng.standard_normal(opt.n) * 1e-3).astype(np.float32))
    opt.step_scaled(1e-3)
    assert (opt.download("param") == p).all()
    opt.free()


@pytest.mark.parametrize("grad_type", [F32, BF16, FP8])
def test_switches_change_no_bit(gpu, oracle, monkeypatch, grad_type):
    """Tiles to a workgroup, the walk's direction, cache hints: 300 tiles, three steps each."""
    tensors = [(4096 * 290, 3), (7, 0), (4096 * 10 + 77, 2)]
    rng = np.random.default_rng(18)
    n = sum(t[0] for t in tensors)
    p = (rng.standard_normal(n) * 0.02).astype(np.float32)
    data = [gradients(oracle, rng, tensors, grad_type, 1e-3) for _ in range(3)]
    want = None
    try:
        for env in ({}, dict(ANNI_NT="0"), dict(ANNI_REVERSE="0", ANNI_KEEP_MB="0"), dict(ANNI_TILES_PER_WG="3"),
                    dict(ANNI_TILES_PER_WG="0", ANNI_BLOCKS_PER_CU="1"), dict(ANNI_PIPE="0"), dict(ANNI_PIPE="2")):
            with monkeypatch.context() as m:
                for k, v in env.items():
                    m.setenv(k, v)
                gpu.anni_gpu_reload_switches()
                opt, _kw = new_arena(tensors, grad_type, grad_clip=0.0)
                opt.upload("param", p)
                for g, scales in data:
                    opt.upload("grad", g)
                    if grad_type == FP8:
                        opt.upload("gscale", scales)
                    opt.step_scaled(1e-3)
                got = [opt.download(k).tobytes() for k in ("param", "m", "v", "m_exp", "v_exp", "twin")]
                opt.free()
            want = want or got
            assert got == want, env
    finally:
        gpu.anni_gpu_reload_switches()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_skipped_step_leaves_codes_and_exponents(gpu, oracle, bad):
    tensors = LISTS["ragged"]
    opt, kw = new_arena(tensors, F32)
    rng = np.random.default_rng(6)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    model = Model(oracle, opt, tensors, F32, kw, p)
    for k in range(3):
        g, _s = gradients(oracle, rng, tensors, F32, 0.5)
        if k == 1:
            g[5003] = bad
        opt.upload("grad", g)
        opt.step_scaled(1e-3)
        model.step(g, 1e-3)
        model.check()               # after the skipped step: the codes of the one before
    opt.free()


def some_state(opt, rng):
    opt.upload("param", (rng.standard_normal(opt.n) * 0.02).astype(np.float32))
    for _k in range(2):
        opt.upload("grad", (rng.standard_normal(opt.n) * 1e-3 * np.exp(rng.standard_normal(opt.n) * 3))
                   .astype(np.float32))
        opt.step_scaled(1e-3)
    return [opt.download(k) for k in ("m", "v", "m_exp", "v_exp")]


def decoded(state):
    cm, cv, bm, bv = state
    return q8.decode_m(cm, bm), q8.decode_v(cv, bv)


@pytest.mark.parametrize("n", [1, 255, 256 * 9, 256 * 9 + 3, (1 << 21) + 777])
def test_a_state_exported_and_imported_is_the_same(gpu, n):
    opt, _kw = new_arena([(n, 3)])
    rng = np.random.default_rng(7)
    before = some_state(opt, rng)
    m, v = decoded(before)
    pairs = opt.export_mv()
    assert same_bits(pairs[:, 0].copy(), m) and same_bits(pairs[:, 1].copy(), v)
    with tempfile.TemporaryFile() as f:
        opt.write_state(f.fileno(), 3, 4)
        f.seek(0)
        other, _kw = new_arena([(n, 3)])
        assert other.read_state(f.fileno()) == (3, 4) and other.t == opt.t
    again = decoded([other.download(k) for k in ("m", "v", "m_exp", "v_exp")])
    assert same_bits(again[0], m) and same_bits(again[1], v)
    # and both go on alike: a state is its values
    g = (rng.standard_normal(n) * 1e-3).astype(np.float32)
    other.upload("param", opt.download("param"))
    for o in (opt, other):
        o.upload("grad", g)
        o.step_scaled(1e-3)
    for k in ("param", "m", "v", "m_exp", "v_exp"):
        assert same_bits(opt.download(k), other.download(k))
    opt.free()
    other.free()


@pytest.mark.parametrize("first,count", [(0, 1), (255, 2), (256, 256), (100, 700), (1000, 1559)])
def test_partial_import(gpu, first, count):
    n = 2559
    opt, _kw = new_arena([(n, 3)])
    rng = np.random.default_rng(8)
    m, v = decoded(some_state(opt, rng))
    new = np.stack([rng.standard_normal(count) * 1e-4, rng.standard_normal(count) ** 2 * 1e-6], 1).astype(np.float32)
    new[0, 1] = -1.0                     # v has no sign
    opt.import_mv(new, first)
    m[first:first + count] = new[:, 0]
    v[first:first + count] = np.maximum(new[:, 1], 0)
    # every touched block: encoded to nearest under its new exponent; the others as they were
    touched = np.zeros(n, bool)
    touched[first // 256 * 256:((first + count - 1) // 256 + 1) * 256] = True
    wm, wv = q8.decode_m(*q8.encode_m(m)), q8.decode_v(*q8.encode_v(v))
    wm[~touched], wv[~touched] = m[~touched], v[~touched]
    got = opt.export_mv()
    assert same_bits(got[:, 0].copy(), wm) and same_bits(got[:, 1].copy(), wv)
    opt.free()


@pytest.mark.parametrize("moment_type", [F32, BF16, Q8])
@pytest.mark.parametrize("out_type", [F32, BF16])
def test_moments_read_on_the_device(gpu, oracle, moment_type, out_type):
    from anni_amd.lm_adam import DeviceBuffer, LmAdam
    n = 70003
    opt = LmAdam([(n, 3)], moment_type=moment_type, beta2=0.95)
    rng = np.random.default_rng(9)
    opt.upload("param", np.zeros(n, np.float32))
    opt.upload("grad", (rng.standard_normal(n) * np.exp(rng.standard_normal(n) * 3)).astype(np.float32))
    opt.step_scaled(1e-3)
    pairs = opt.export_mv()
    dt, size = (np.float32, 4) if out_type == F32 else (np.uint16, 2)
    a, b = DeviceBuffer(size * n + 64), DeviceBuffer(size * n + 64)
    for first, count, skew in ((0, n, 0), (0, n - 8, 1), (8, 4096, 0), (7, 999, 0), (n - 1, 1, 3), (256, 8, 8)):
        for buf in (a, b):
            buf.upload(np.full(size * n + 64, 0xA5, np.uint8))
        opt.read_moments(a.ptr + skew * size, b.ptr + skew * size, first, count, out_type)
        for buf, col in ((a, 0), (b, 1)):
            want = pairs[first:first + count, col].copy()
            want = want if out_type == F32 else oracle.bf16_rne(want)
            assert same_bits(buf.download(dt, count, skew * size), want)
            rest = buf.download(np.uint8, size * n + 64)
            assert (rest[:skew * size] == 0xA5).all() and (rest[(skew + count) * size:] == 0xA5).all()
    opt.read_moments(None, b.ptr, 0, 5, out_type)           # one of the two
    opt.free()


def test_refusals(gpu):
    from anni_amd import lib
    from anni_amd.lm_adam import DeviceBuffer, LmAdam
    with pytest.raises(RuntimeError):
        LmAdam([(100, 3)], grad_type=Q8)                     # a storage of moments only
    with pytest.raises(RuntimeError):
        LmAdam([(100, 3)], moment_type=FP8)
    with pytest.raises(RuntimeError):
        LmAdam([(100, 3)], moment_type=4)
    opt, _kw = new_arena([(100, 3)])
    buf = DeviceBuffer(1024)
    L = lib.load()
    bad = [(0, 101, BF16, buf.ptr, None), (-1, 1, BF16, buf.ptr, None), (0, -1, BF16, buf.ptr, None),
           (101, 0, BF16, buf.ptr, None), (1 << 62, 1 << 62, BF16, buf.ptr, None), (0, 100, Q8, buf.ptr, None),
           (0, 100, FP8, buf.ptr, None), (0, 100, BF16, None, None), (0, 100, F32, buf.ptr + 2, None),
           (0, 100, BF16, buf.ptr, buf.ptr + 1)]
    for first, count, ty, a, b in bad:
        assert L.anni_adam_read_moments(opt.h, first, count, ty, a, b) == -1
    assert L.anni_adam_read_moments(None, 0, 1, BF16, buf.ptr, None) == -1
    assert L.anni_adam_read_moments(opt.h, 100, 0, BF16, buf.ptr, None) == 0
    opt.free()


def test_offloaded_moments_keep_their_exponents(gpu):
    tensors = LISTS["ragged"]
    rng = np.random.default_rng(10)
    p = (rng.standard_normal(sum(t[0] for t in tensors)) * 0.02).astype(np.float32)
    gs = [(rng.standard_normal(p.size) * 1e-3).astype(np.float32) for _k in range(3)]
    out = []
    for on in (0, 1):
        opt, _kw = new_arena(tensors)
        opt.upload("param", p)
        if on:
            assert gpu.anni_adam_set_offload(opt.h, 1) == 0
        for g in gs:
            opt.upload("grad", g)
            opt.step_scaled(1e-3)
        pairs = opt.export_mv()
        assert gpu.anni_adam_set_offload(opt.h, 0) == 0
        out.append([opt.download(k) for k in ("param", "m", "v", "m_exp", "v_exp")] + [pairs])
        opt.free()
    for a, b in zip(*out):
        assert same_bits(a, b)


def test_derived_outputs_follow(gpu, oracle):
    tensors = [(5000, 3 | 4), (3, 0), (4096 * 3, 3 | 4), (8191, 1), (40000, 3)]
    opt, kw = new_arena(tensors)
    rng = np.random.default_rng(11)
    p = (rng.standard_normal(opt.n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    opt.enable_derived([(2, 4096, 0, 4096)], 4096 * 3)
    opt.seed_twins()
    model = Model(oracle, opt, tensors, F32, kw, p)
    for _k in range(2):
        g, _s = gradients(oracle, rng, tensors, F32, 2.0)
        opt.upload("grad", g)
        opt.step_scaled(1e-3)
        model.step(g, 1e-3)
        for i in (0, 2):
            a, k = opt.offsets[i], tensors[i][0]
            q, s = oracle.fp8_quantize(model.P[a:a + k])
            assert (opt.download("fp8twin", k, a) == q).all() and opt.download("wscale")[i] == s
        a = opt.offsets[2]
        assert (opt.download("pack") == oracle.bf16_rne(model.P[a:a + 4096 * 3])).all()
        assert (opt.download("m") == model.cm).all() and (opt.download("v") == model.cv).all()
    opt.free()


def test_step_and_read_replay_from_a_graph(gpu, oracle):
    from anni_amd.lm_adam import DeviceBuffer
    hip = hip_runtime()
    tensors = LISTS["ragged"]
    opt, kw = new_arena(tensors)
    n = opt.n
    rng = np.random.default_rng(12)
    p = (rng.standard_normal(n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    model = Model(oracle, opt, tensors, F32, kw, p)
    mo, vo = DeviceBuffer(4 * n), DeviceBuffer(4 * n)

    def new_grad(k):
        g, _s = gradients(oracle, rng, tensors, F32, 2.0 if k % 2 else 0.4)
        opt.upload("grad", g)
        return g

    stream = C.c_void_p()
    ok(hip.hipStreamCreate(C.byref(stream)), "hipStreamCreate")
    gpu.anni_gpu_set_stream(stream)
    try:
        g = new_grad(0)
        opt.step_scaled(1e-3)
        model.step(g, 1e-3, 0)
        model.check()
        g = new_grad(1)
        graph, gexec = C.c_void_p(), C.c_void_p()
        ok(hip.hipStreamBeginCapture(stream, 2), "hipStreamBeginCapture")
        rc = opt.step_scaled(2e-3)
        opt.read_moments(mo.ptr, vo.ptr, out_type=F32)
        ok(hip.hipStreamEndCapture(stream, C.byref(graph)), "hipStreamEndCapture")
        assert rc == 0 and graph.value
        hip.hipGraphInstantiate.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
        ok(hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0), "hipGraphInstantiate")
        for k in range(1, 5):
            g = g if k == 1 else new_grad(k)
            ok(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
            ok(hip.hipStreamSynchronize(stream), "hipStreamSynchronize")
            model.step(g, 2e-3, 1)                  # the recorded step carries its own t, and with it its dither
            model.check()
            assert same_bits(mo.download(np.float32, n), model.M) and same_bits(vo.download(np.float32, n), model.V)
        ok(hip.hipGraphExecDestroy(gexec), "hipGraphExecDestroy")
        ok(hip.hipGraphDestroy(graph), "hipGraphDestroy")
    finally:
        gpu.gpu_device_sync()
        gpu.anni_gpu_set_stream(None)
        hip.hipStreamDestroy(stream)
        opt.free()


def test_memory_is_a_quarter_of_the_float_moments(gpu):
    from anni_amd.lm_adam import LmAdam
    n = 1 << 20
    q, _kw = new_arena([(n, 3)])
    f = LmAdam([(n, 3)], beta2=0.95)
    assert f.resident_bytes - q.resident_bytes == 2 * (4 * n - n - n // 256)
    q.free()
    f.free()
