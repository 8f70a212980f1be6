"""8-bit moments: how p may differ from the host loop, element by element, and flats whose offsets pass 32 bits."""
import numpy as np
import pytest

import q8_model as q8
from helpers import same_bits

pytestmark = pytest.mark.gpu

F32, Q8 = 0, 3
B1, B2, EPS = 0.9, 0.95, 1e-8


class Host:
    """The host loop on a window [first, ...) of the flat (whole blocks), moments kept as the storage keeps them."""

    def __init__(self, p, first=0):
        assert first % q8.BLOCK == 0
        self.p, self.first, self.t = p.copy(), first, 0
        self.m, self.v = np.zeros(p.size, np.float32), np.zeros(p.size, np.float32)

    def step(self, g, lr, decay=None):
        """p after the step in double, before its rounding, and the step itself."""
        self.t += 1
        x = g.astype(np.float64)
        m = (B1 * self.m.astype(np.float64) + (1.0 - B1) * x).astype(np.float32)
        v = (B2 * self.v.astype(np.float64) + ((1.0 - B2) * x) * x).astype(np.float32)
        step = (lr * (m.astype(np.float64) / (1.0 - B1 ** self.t))) / (
            np.sqrt(v.astype(np.float64) / (1.0 - B2 ** self.t)) + EPS)
        exact = self.p.astype(np.float64) - step
        self.p = exact.astype(np.float32)
        rm, rv = q8.dither(g.size, self.t, self.first)
        self.cm, self.bm = q8.encode_m(m, rm)
        self.cv, self.bv = q8.encode_v(v, rv)
        self.m, self.v = q8.decode_m(self.cm, self.bm), q8.decode_v(self.cv, self.bv)
        return exact, step


def check_p(got, want, exact, step):
    """The step is within 2^-43 of the host loop's, and subtracting it in double rounds by 2^-53 of p on either side: p
    is the float nearest to a double that near the host loop's.  How many elements get another float than the host
    loop's is a matter of chance: a share of twice the bound over the distance of two floats."""
    off = 2.0 ** -43 * np.abs(step) + 2.0 ** -52 * np.abs(exact)
    ulp = np.spacing(np.maximum(np.abs(got), np.abs(want))).astype(np.float64)
    far = np.flatnonzero(np.abs(got.astype(np.float64) - exact) > off + ulp / 2)
    assert far.size == 0, (far[:5], got[far[:5]], exact[far[:5]])
    count = np.count_nonzero(got.view(np.uint32) != want.view(np.uint32))
    expected = float(np.minimum(2 * off / ulp, 1.0).sum())
    # five deviations of that count beyond it, and one
    assert count <= expected + 5 * np.sqrt(expected) + 1, (count, expected)
    return count


@pytest.mark.parametrize("skew", [0, 4])
def test_p_is_the_host_loops_or_next_to_it(gpu, skew):
    """4 M elements on the vector path, and element by element (a gradient flat that is not aligned)."""
    from anni_amd.lm_adam import DeviceBuffer, LmAdam
    n = (1 << 22) + 300
    opt = LmAdam([(n, 0)], moment_type=Q8, grad_slots=0, beta1=B1, beta2=B2, eps=EPS)
    buf = DeviceBuffer(4 * n + 64)
    opt.bind_grad(buf.ptr + skew)
    rng = np.random.default_rng(21)
    p = (rng.standard_normal(n) * 0.02).astype(np.float32)
    opt.upload("param", p)
    host = Host(p)
    for _k in range(3):
        g = (rng.standard_normal(n) * 1e-3 * np.exp(rng.standard_normal(n))).astype(np.float32)
        buf.upload(g, skew)
        opt.step_scaled(1e-3)
        exact, step = host.step(g, 1e-3)
        got = opt.download("param")
        print("elements with another float:", check_p(got, host.p, exact, step))
        assert same_bits(opt.download("m"), host.cm) and same_bits(opt.download("v"), host.cv)
        assert same_bits(opt.download("m_exp"), host.bm) and same_bits(opt.download("v_exp"), host.bv)
        host.p = got
    opt.free()


def test_a_flat_beyond_32_bits(gpu):
    """2^31 + 13065 elements: steps, read-out, export and import around the start, element 2^31 and the end;
    zeros everywhere else, which stay zeros."""
    from anni_amd.lm_adam import DeviceBuffer, LmAdam
    from anni_amd import lib
    half = 1 << 31
    n = half + 4096 * 3 + 777
    opt = LmAdam([(half - 5000, 0), (5100, 0), (n - half - 100, 0)], moment_type=Q8, twins=False,
                 layout=lib.LAYOUT_COMPACT, beta1=B1, beta2=B2, eps=EPS)
    assert opt.n == n
    rng = np.random.default_rng(22)
    spans = [(0, 8192), (half - 8192, 14336), (half + 8192, n - half - 8192)]
    hosts = []
    for first, count in spans:
        p = (rng.standard_normal(count) * 0.02).astype(np.float32)
        opt.upload("param", p, first)
        hosts.append(Host(p, first))
    blocks = opt.blocks

    def codes(which, first, count):
        return opt.download(which, count, first)

    for k in range(2):
        gs = [(rng.standard_normal(c) * 1e-3).astype(np.float32) for _f, c in spans]
        for (first, _c), g in zip(spans, gs):
            opt.upload("grad", g, first)
        opt.step_scaled(1e-3)
        for (first, count), g, h in zip(spans, gs, hosts):
            exact, step = h.step(g, 1e-3)
            got = opt.download("param", count, first)
            check_p(got, h.p, exact, step)
            h.p = got
            assert same_bits(codes("m", first, count), h.cm) and same_bits(codes("v", first, count), h.cv)
            b, nb = first // q8.BLOCK, (count + q8.BLOCK - 1) // q8.BLOCK
            assert same_bits(codes("m_exp", b, nb), h.bm) and same_bits(codes("v_exp", b, nb), h.bv)
            assert not opt.download("grad", count, first).any()
    quiet = half - 8192 - 65536
    assert not codes("m", quiet, 65536).any() and not opt.download("param", 65536, quiet).any()
    mo, vo = DeviceBuffer(4 * 30000), DeviceBuffer(4 * 30000)
    for first, count in ((half - 8192, 14336), (half - 3, 5001), (n - 4001, 4001)):
        opt.read_moments(mo.ptr, vo.ptr, first, count, F32)
        h = hosts[1] if first < half else hosts[2]
        a = first - h.first
        m, v = h.m[a:a + count], h.v[a:a + count]
        assert same_bits(mo.download(np.float32, count), m) and same_bits(vo.download(np.float32, count), v)
        pairs = opt.export_mv(first, count)
        assert same_bits(pairs[:, 0].copy(), m) and same_bits(pairs[:, 1].copy(), v)
    # whole blocks on either side of 2^31 imported anew
    new = np.stack([rng.standard_normal(512) * 1e-4, rng.standard_normal(512) ** 2 * 1e-6], 1).astype(np.float32)
    opt.import_mv(new, half - 256)
    want_m, want_v = q8.encode_m(new[:, 0].copy()), q8.encode_v(new[:, 1].copy())
    assert same_bits(codes("m", half - 256, 512), want_m[0]) and same_bits(codes("v", half - 256, 512), want_v[0])
    b = half // q8.BLOCK - 1
    assert same_bits(codes("m_exp", b, 2), want_m[1]) and same_bits(codes("v_exp", b, 2), want_v[1])
    assert same_bits(codes("m", half - 512, 256), hosts[1].cm[8192 - 512:8192 - 256]) and b + 2 < blocks
    opt.free()
