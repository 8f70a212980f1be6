"""The 8-bit moment formats by themselves: what the step's parity tests hold the GPU to."""
import numpy as np
import pytest

import q8_model as q8


def test_tables_are_the_formats_of_the_header():
    assert q8.TABLE_M.size == 128 and q8.TABLE_V.size == 256
    for table, fields in ((q8.TABLE_M, 16), (q8.TABLE_V, 32)):
        for code, value in enumerate(table):
            f, r = divmod(code, 8)
            e = f - (fields - 1)
            want = (1 + r / 8) * 2.0 ** e if f else r / 8 * 2.0 ** (1 - (fields - 1))
            assert value == want
    # m's codes are OCP E4M3 with 448 = 1.75 * 2^8 at the top of the block
    assert q8.TABLE_M[0x7E] * 2.0 ** 8 == 448.0 and q8.TABLE_M[1] * 2.0 ** 8 == 2.0 ** -9


@pytest.mark.parametrize("top", [1.0, 1.75, np.float32(1.7500001), 1.9999999, 3e-39, 1e-45, 0.0, 1e30])
def test_no_block_overflows_its_codes(top):
    x = np.zeros(300, np.float32)
    x[7] = top
    x[8] = -top
    x[299] = top / 3
    for enc, table in ((q8.encode_m, q8.TABLE_M), (q8.encode_v, q8.TABLE_V)):
        for rnd in (np.zeros(300), np.full(300, 65535.0), None):
            code, _b = enc(x if enc is q8.encode_m else np.abs(x), rnd)
            assert ((code & (127 if table is q8.TABLE_M else 255)) <= table.size - 2).all()


def test_values_on_the_grid_come_back():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal(5000) * np.exp(rng.standard_normal(5000) * 3)).astype(np.float32)
    rm, rv = q8.dither(5000, 9)
    for enc, dec, y, r in ((q8.encode_m, q8.decode_m, x, rm), (q8.encode_v, q8.decode_v, x * x, rv)):
        first = dec(*enc(y, r))
        again = dec(*enc(first))                    # an import of what was exported
        assert (first == again).all()
        dith = dec(*enc(first, r))                  # and a step that changes nothing
        assert (first == dith).all()


def test_rounding_is_within_a_step_and_unbiased():
    rng = np.random.default_rng(2)
    x = np.abs(rng.standard_normal(256)).astype(np.float32) + 0.01
    total = np.zeros(256)
    steps = 4000
    for t in range(1, steps + 1):
        _rm, rv = q8.dither(256, t)
        y = q8.decode_v(*q8.encode_v(x, rv)).astype(np.float64)
        assert (np.abs(y - x) <= x / 8).all()       # eight steps to the binade
        total += y
    # a two-valued variable a step of x / 8 apart has a deviation of at most x / 16; five of the mean's
    assert (np.abs(total / steps - x) <= 5 * x / 16 / np.sqrt(steps)).all()


def test_a_slow_average_moves_where_rounding_to_nearest_would_not():
    """v = 0.999 v + 0.001 g^2 from 4 towards 1: a step of it is below half a code."""
    dith = np.full(256, 4.0, np.float32)
    near = dith.copy()
    for t in range(1, 4001):
        _rm, rv = q8.dither(256, t)
        dith = q8.decode_v(*q8.encode_v((0.999 * dith + 0.001).astype(np.float32), rv))
        near = q8.decode_v(*q8.encode_v((0.999 * near + 0.001).astype(np.float32)))
    want = 1.0 + 3.0 * 0.999 ** 4000
    assert (near == 4.0).all()
    # the average's stationary deviation: a step of 1/8 of the value each time, weighed over ~1/0.002 steps,
    # below 0.125 / 2 * sqrt(1 / 0.002) * value = 1.4; the mean of 256 of them within five of its own
    assert abs(float(dith.mean()) - want) < 5 * 1.4 / 16


def test_positive_second_moments_never_vanish():
    v = np.full(256, 1e-30, np.float32)
    v[0] = 1.0
    code, _b = q8.encode_v(v, np.zeros(256))
    assert (code[1:] == 1).all()
    assert (q8.encode_v(np.zeros(256, np.float32), np.full(256, 65535.0))[0] == 0).all()


def test_dither_is_uniform_over_places_and_steps():
    for rows in (np.stack(q8.dither(1 << 16, 77)),
                 np.stack([np.array([q8.dither(1, t, 12345)[k][0] for t in range(1, 4097)]) for k in (0, 1)])):
        for r in rows:
            count = np.histogram(r, 16, (0, 65536))[0]
            want = r.size / 16
            assert (np.abs(count - want) < 5 * np.sqrt(want)).all()
