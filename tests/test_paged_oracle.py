"""The serving operators' oracle (oracle/paged_oracle.py) against closed forms on the CPU; planted
mistakes in it are seen."""
import numpy as np

from oracle import afa_oracle as O
from oracle import paged_oracle as P


def test_pool_keeps_every_page_once():
    rng = np.random.default_rng(0)
    pool = P.Pool(40, 4, 6, 60)
    for _ in range(50):
        cached, new = rng.integers(0, 30, 6), rng.integers(0, 8, 6)
        out = pool.step(cached, new, 40, 8, 64)
        pages = sorted(p for t in pool.tables for p in t) + sorted(pool.free)
        assert sorted(pages) == list(range(40))
        slots = out[0][out[0] >= 0]
        assert len(set(slots)) == len(slots)
        for r in range(6):
            if out[5][r] == P.OK:
                assert len(pool.tables[r]) == -(-int(cached[r] + new[r]) // 4)


def test_statuses():
    pool = P.Pool(4, 2, 6, 8)
    out = pool.step([0, -1, 3, 0, 9, 0], [1, 1, 2, 9, 1, 1], 20, 4, 0)
    assert list(out[5]) == [P.OK, P.NEGATIVE, P.OK, P.TOO_MANY, P.TOO_LONG, P.NO_PAGES]
    assert list(out[3]) == [0, 1, 2, 4, 13, 14, 15]
    out = P.Pool(4, 2, 2, 8).step([0, 0], [3, 2], 4, 4, 0)
    assert list(out[5]) == [P.OK, P.PAST_END] and list(out[3]) == [0, 3, 4] and list(out[0]) == [0, 1, 2, -1]


def test_tree_masks():
    parents = np.array([-1, 0, 0, 2, 7, 1])  # node 4's parent is no earlier token: none
    _, pos, _, _, sees, _ = P.Pool(9, 4, 1, 32).step([5], [6], 6, 6, 64, parents)
    rows = [list(np.flatnonzero(r)) for r in sees]
    assert rows == [[0], [0, 1], [0, 2], [0, 2, 3], [4], [0, 1, 5]]
    assert list(pos) == [5, 6, 6, 7, 5, 7]
    words = P.mask_words(np.eye(64, dtype=bool))
    assert words[0, 0] == 1 and words[63, 0] == np.iinfo(np.int64).min


def test_rotation_is_the_oracles_for_one_axis():
    rng = np.random.default_rng(1)
    c, s = O.cayley_tables(16, 32)
    x = rng.standard_normal((2, 3, 32, 16))
    at = np.broadcast_to(np.arange(32)[None, :, None], (2, 32, 1))
    y = P.rotate_axes(x, c, s, at, (8,))
    x0, x1 = x[..., 0::2], x[..., 1::2]
    ref = np.stack((c * x0 - s * x1, s * x0 + c * x1), -1).reshape(x.shape)
    assert np.abs(y - ref).max() <= 1e-14
    assert np.abs(P.rotate_axes(y, c, s, at, (8,), back=True) - x).max() <= 1e-13
    # a planted mistake: the second section by the other axis.  Its first pair, k = 4, has
    # w = 1 / (1 + 4 (sqrt(10000) - 1) / 7)^2 = 3.0e-4: 31 positions turn it by 62 w = 0.0187 more, which
    # moves a pair of length >= 1 (the longest of the six rows at either end) by more than 0.01
    two = np.concatenate((at, at[:, ::-1]), -1)
    assert np.abs(P.rotate_axes(x, c, s, two, (4, 4)) - y).max() > 0.01


def test_attention_row_is_the_oracles():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((3, 40, 24))
    ref, den = O.afa_forward(q, k, v, 0.5, True, return_denominator=True)
    for i in (0, 1, 39):
        out, d, size, _ = P.attention_row(q[i], k[:i + 1], v[:i + 1], 0.5)
        assert np.abs(out - ref[i]).max() <= 1e-13 and abs(d - den[i, 0]) <= 1e-12 * d
        assert (np.abs(out) <= size + 1e-15).all()
    assert np.abs(P.attention_row(q[5], k[:5], v[:5], 0.5)[0] - ref[5]).max() > 1e-3  # its own key left out
