"""The 64-bit restatements of the long-context operators on inputs whose
answers are known by hand, and the host-side frequency table."""
import numpy as np
import pytest

import longctx_ref as ref


def test_nearest_codes():
    assert ref.nearest(np.array([0.5, 1.5, 2.5, -0.5, 200.0, -np.inf, np.nan]), "int8").tolist() == [0, 2, 2, 0, 127, -127, 0]
    # three fraction bits: 17 lies between 16 and 18, 19 between 18 and 20; the least step is 2^-9
    got = ref.nearest(np.array([17.0, 19.0, 460.0, 2.0 ** -10, 3 * 2.0 ** -10, np.nan]), "e4m3")
    assert got.tolist() == [16.0, 20.0, 448.0, 0.0, 2.0 ** -8, 0.0]


def test_power_scale():
    assert ref.power_scale(127.0, "int8") == 1.0
    assert ref.power_scale(127.5, "int8") == 2.0
    assert ref.power_scale(448.0, "e4m3") == 1.0
    assert ref.power_scale(0.0, "e4m3") == 2.0 ** -126


def test_append_raises_scale_of_a_started_block():
    z = np.zeros((1, 1, 16, 16))
    c = ref.Cache(z, z, np.zeros((1, 1)), np.zeros((1, 1)), "int8")
    one = np.full((1, 1, 16), 1.0)
    c.append((one, one), [0, 1], [1], [[0]])
    assert c.scale[0][0, 0] == 2.0 ** -6 and c.codes[0][0, 0, 0, 0] == 64
    c.append((one * 100, one), [0, 1], [2], [[0]])
    assert c.scale[0][0, 0] == 1.0 and c.codes[0][0, 0, :2, 0].tolist() == [1.0, 100.0]
    assert c.scale[1][0, 0] == 2.0 ** -6


def test_evict_keeps_the_heaviest_and_the_last():
    k = np.arange(32, dtype=np.float64).reshape(2, 1, 16, 1).repeat(16, 3)
    c = ref.Cache(k, k, np.array([[1.0], [4.0]]), np.ones((2, 1)), "int8")
    w = np.zeros((1, 1, 32))
    w[0, 0, [3, 20, 25]] = [1.0, 1.0, 1.0]
    lens, keep, left = c.evict([[0, 1]], [30], w, 4, 2)
    assert lens == [4] and keep[0][0].tolist() == [3, 20, 28, 29]  # 25 ties with 3 and 20 and comes last
    assert c.scale[0][0, 0] == 4.0 and c.codes[0][0, 0, :4, 0].tolist() == [1.0, 20.0, 28.0, 29.0]  # 3 / 4 to 1
    assert left[0, 0, :5].tolist() == [1.0, 1.0, 0.0, 0.0, 0.0]


def test_attention_of_equal_scores_is_the_mean():
    k = np.zeros((1, 1, 16, 16))
    v = np.arange(16.0).reshape(1, 1, 16, 1).repeat(16, 3)
    c = ref.Cache(k, v, np.ones((1, 1)), np.full((1, 1), 0.5), "int8")
    out, lse, sums, _, _ = ref.attention(c, np.ones((1, 1, 16)), [0, 1], [5], [[0]], 1.0)
    assert np.allclose(out, 1.0) and np.allclose(lse, np.log(5.0)) and np.allclose(sums[0], 0.2)
    out, lse, _, _, _ = ref.attention(c, np.ones((1, 1, 16)), [0, 1], [5], [[0]], 1.0, window=2)
    assert np.allclose(out, 1.75)


def test_logits_steps():
    y = ref.logits(np.array([2.0, -2.0, 1.0, 0.0]), [0, 1, 1, 7], 1, 2.0, 0.5, 0.25, [(2, 1.0), (2, 0.5)], np.array([1, 1, 1, 0], bool))
    assert y.tolist() == [1.0, -4.0 - 1.0 - 0.25, 2.5, -np.inf]


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("base", 8.0), ("parts", 16.0)])
@pytest.mark.parametrize("rot", [4, 64, 128, 256])
def test_frequency_table(pkg, scaling, factor, rot):
    got = pkg.rope_frequencies(rot, 10000.0, scaling, factor, 4096, 1.0, 32.0)
    want = ref.frequencies(rot, 10000.0, scaling, factor, 4096, 1.0, 32.0)
    # double powers and products: a few units of 2^-53, and half a unit of 2^-64
    turns = want / (2 * np.pi)
    assert np.all(np.abs(got.astype(np.float64) * 2.0 ** -64 - turns) <= 1e-14 * turns + 2.0 ** -65)


@pytest.mark.parametrize("bad", [dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(rot_dim=8, base=1.0),
                                 dict(rot_dim=8, scaling="linear", factor=0.5), dict(rot_dim=8, scaling="other"),
                                 dict(rot_dim=8, scaling="parts", low=2.0, high=2.0), dict(rot_dim=2, scaling="base", factor=2.0),
                                 dict(rot_dim=8, base=float("nan"))])
def test_frequency_table_refuses(pkg, bad):
    with pytest.raises(pkg.I4DError):
        pkg.rope_frequencies(**bad)
