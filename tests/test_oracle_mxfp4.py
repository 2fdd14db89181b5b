"""The MXFP4 oracle against brute force and closed forms: nearest codes, ties,
scales, and a page layout in which every code and scale has a place of its own."""
import numpy as np
import pytest

from oracle import mxfp4 as M


def test_codes_are_the_nearest_of_all_sixteen():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((64, 64)) * np.exp2(rng.integers(-20, 20, (64, 1)))
    codes, scales = M.quantise(x)
    got = M.values(codes, scales)
    unit = np.repeat(np.exp2(scales.astype(float) - 127), 32, -1)
    every = np.concatenate([M.E2M1, -M.E2M1])
    best = np.abs(x[..., None] - every * unit[..., None]).min(-1)
    assert np.array_equal(np.abs(x - got), best)
    # the largest value of a group lies in [4, 8) units
    top = np.abs(x).reshape(64, 2, 32).max(-1) / np.exp2(scales.astype(float) - 127)
    assert (top >= 4).all() and (top < 8).all()


def test_ties_go_to_the_even_code_and_large_values_to_six():
    row = np.zeros((1, 32))
    row[0, :9] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -5.0]
    codes, scales = M.quantise(row)
    assert scales[0, 0] == 127  # floor(log2 7.9) - 2 = 0
    assert M.values(codes, scales)[0, :9].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -4]


def test_scales_of_zero_tiny_and_infinite_groups():
    x = np.zeros((5, 32))
    x[1, 3] = 2.0 ** -126       # 2^-128 would be the scale: the smallest there is, 2^-127
    x[2, 0] = np.inf
    x[3, 31] = np.nan
    x[4, 5] = 3.0e38            # floor(log2) = 127
    codes, scales = M.quantise(x)
    assert scales[:, 0].tolist() == [0, 0, 255, 255, 252]
    v = M.values(codes, scales)
    assert (v[0] == 0).all() and v[1, 3] == 2.0 ** -126 and np.isnan(v[2:4]).all()
    assert v[4, 5] == 6 * 2.0 ** 125


@pytest.mark.parametrize("heads,dim", [(1, 64), (2, 64), (3, 128), (2, 128)])
def test_every_code_and_scale_of_a_block_has_its_own_place(heads, dim):
    slots = np.arange(48)
    for is_value in (False, True):
        at = M.code_at(slots, heads, dim, is_value)
        # two dims a byte, and the bytes are all there are
        assert np.array_equal(np.sort(at.ravel())[::2], np.arange(3 * M.half_bytes(heads, dim)))
        assert np.array_equal(at[..., 0::2], at[..., 1::2])
    assert np.array_equal(np.sort(M.scale_at(slots, heads, dim).ravel()), np.arange(3 * M.half_bytes(heads, dim) // 16))


def test_rows_come_back_as_they_were_put():
    rng = np.random.default_rng(2)
    heads, dim, blocks = 2, 128, 5
    x = rng.standard_normal((30, heads, dim))
    codes, sc = M.quantise(x)
    slots = rng.permutation(blocks * 16)[:30]
    for is_value in (False, True):
        pool = rng.integers(0, 256, blocks * M.half_bytes(heads, dim)).astype(np.uint8)
        scales = rng.integers(0, 256, len(pool) // 16).astype(np.uint8)
        M.put(pool, scales, slots, codes, sc, is_value)
        assert np.array_equal(M.get(pool, scales, slots, heads, dim, is_value), M.values(codes, sc))


def test_attention_of_equal_scores_is_the_mean_and_of_one_token_its_value():
    rng = np.random.default_rng(5)
    heads, dim, blocks = 2, 64, 3
    pools = [rng.integers(0, 256, blocks * M.half_bytes(heads, dim) // d).astype(np.uint8) for d in (1, 1, 16, 16)]
    for s in pools[2:]:
        s[:] = rng.integers(120, 130, len(s))
    q = np.zeros((2, 4, dim))
    out, spread, size, reach = M.decode(q, pools, [[2, 0], [1, 1]], [20, 1], heads)
    v = M.get(pools[1], pools[3], np.r_[32:48, 0:4], heads, dim, True)
    np.testing.assert_allclose(out[0], np.repeat(v.mean(0), 2, 0), rtol=1e-12, atol=1e-12)
    one = M.get(pools[1], pools[3], [16], heads, dim, True)[0]
    np.testing.assert_array_equal(out[1], np.repeat(one, 2, 0))
    assert (spread[1] == 0).all() and (reach == 0).all() and np.array_equal(size[1], np.abs(out[1]))
