"""The 4-bit block and its layout, on the CPU: what the definition promises of every
block, and that a granule holds each code and scale in a place of its own."""
import numpy as np
import pytest

from tests import q4_ref


@pytest.mark.parametrize("D", [64, 128, 256])
def test_places_fill_a_granule(D):
    k, v, ks, vs = q4_ref.granule_places(D)
    halves = np.concatenate([(x[..., 0] * 2 + x[..., 1] // 4).ravel() for x in (k, v)])
    assert sorted(halves) == list(range(32 * D))  # 16 D bytes of codes
    scales = np.concatenate([ks.ravel(), vs.ravel()])
    assert sorted(np.concatenate([scales, scales + 1])) == list(range(16 * D, 18 * D))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_pack_and_unpack(D):
    rng = np.random.default_rng(D)
    k, v = rng.standard_normal((2, 3, 32, 2, D)).astype(np.float32)
    (kc, kd), (vc, vd) = q4_ref.quantize(k), q4_ref.quantize(v)
    kv, kds, vv, vds = q4_ref.unpack(q4_ref.pack(kc, kd, vc, vd))
    assert np.array_equal(kv, q4_ref.values(kc, kd)) and np.array_equal(vv, q4_ref.values(vc, vd))
    assert np.array_equal(kds, kd) and np.array_equal(vds, vd)


def test_values_are_exact_in_f16_and_near():
    rng = np.random.default_rng(1)
    for size in (1e-6, 1e-3, 1.0, 300.0, 6e4):
        x = (rng.standard_normal((400, 64)) * size).clip(-65000, 65000).astype(np.float32)
        code, d = q4_ref.quantize(x)
        y = q4_ref.values(code, d)
        assert np.array_equal(y, y.astype(np.float16).astype(np.float64))
        # d has 8 significant bits (or is a subnormal): from its unrounded value it is off
        # by 2^-8 of it or half the least f16; a value is half a step off, one at the end
        # of the range (8 steps) a whole one and 8 times d's own rounding
        step = np.abs(d.astype(np.float64)).repeat(32, -1).reshape(x.shape)
        slack = 8 * np.maximum(step * 2.0 ** -8, 2.0 ** -25)
        assert (np.abs(y - x) <= step * (1 + 2.0 ** -6) + slack).all()
        inside = (x.astype(np.float64) / np.where(step == 0, 1, step * np.sign(d.astype(np.float64)).repeat(32, -1).reshape(x.shape)) < 7.49) & (step > 0)
        assert (np.abs(y - x)[inside] <= (step * (0.5 + 2.0 ** -6) + slack)[inside]).all()


def test_special_blocks():
    x = np.zeros((6, 32), np.float32)
    x[1, 3], x[1, 4] = 2.0, -2.0           # a tie: the negative one counts
    x[2, 0] = 1e30                         # saturates
    x[3, 7] = -np.inf
    x[4, 9] = np.nan
    x[5, 1] = 2.0 ** -24                   # under f16: zeros
    code, d = q4_ref.quantize(x)
    y = q4_ref.values(code, d)
    assert d[0, 0] == 0 and (y[0] == 0).all()
    assert d[1, 0] == 0.25 and code[1, 4] == 0 and y[1, 4] == -2.0 and y[1, 3] == 1.75
    assert d[2, 0] == -8160 and y[2, 0] == 65280
    assert d[3, 0] == 8160 and y[3, 7] == -65280
    assert np.isnan(d[4, 0])
    assert d[5, 0] == 0 and (y[5] == 0).all()
