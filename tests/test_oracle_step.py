"""The step oracle against the host manager's rule and by hand."""
import numpy as np

from oracle import step as S


def test_one_new_token_a_request_by_hand():
    # request 0: 17 cached tokens in pages 3, 8; request 1: none cached, page 5
    table, lens, first, slots, pos = S.tables([3, 8, 5], [0, 2, 3], [17, 0], None, 16, 3, 4)
    assert table.tolist() == [[3, 8, -1], [5, -1, -1]] and lens.tolist() == [18, 1]
    assert first.tolist() == [0, 1, 2] and slots.tolist() == [8 * 16 + 1, 5 * 16, -1, -1] and pos.tolist() == [17, 0, -1, -1]


def test_slots_of_a_chunk_follow_its_pages():
    table, lens, first, slots, pos = S.tables([6, 2, 9], [0, 3], [14], [20], 16, 3, 20)
    assert slots.tolist() == [6 * 16 + 14, 6 * 16 + 15] + [2 * 16 + i for i in range(16)] + [9 * 16, 9 * 16 + 1]
    assert np.array_equal(pos, np.arange(14, 34)) and lens.tolist() == [34]


def test_rotation_turns_pairs_as_complex_numbers_and_keeps_lengths():
    rng = np.random.default_rng(3)
    x, angle = rng.standard_normal((3, 64)), rng.standard_normal(16)
    line = np.concatenate([np.cos(angle), np.sin(angle)])
    for pairs in (False, True):
        y, _ = S.norm_rope(x, None, 0.0, line, 32, pairs)
        lo, hi = (slice(0, 32, 2), slice(1, 32, 2)) if pairs else (slice(0, 16), slice(16, 32))
        want = (x[:, lo] + 1j * x[:, hi]) * np.exp(1j * angle)
        np.testing.assert_allclose(y[:, lo] + 1j * y[:, hi], want, rtol=1e-12)
        assert np.array_equal(y[:, 32:], x[:, 32:])


def test_norm_leaves_a_mean_square_of_one():
    x = np.random.default_rng(4).standard_normal((2, 128)) * 50
    y, size = S.norm_rope(x, np.ones(128), 0.0, np.zeros(0), 0, False)
    np.testing.assert_allclose((y * y).mean(-1), 1.0, rtol=1e-12)
    assert np.array_equal(size, np.abs(y))
