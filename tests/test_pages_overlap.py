"""k and v pages that share places through their strides are refused by the calls that write them, and those side by side in one
array are not: the check against sets of addresses, without a GPU."""
import ctypes
import itertools
import os
import random

import pytest

from algebraic_intelligence_amd import _lib
from tests.test_paged import DUMMY, _plan

ESZ = {_lib.AFA_BF16: 2, _lib.AFA_F32: 4, _lib.AFA_F64: 8}


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from algebraic_intelligence_amd import build
        build.build()
    return _lib.lib()


def _evict(lib, dt, shape, k, v, strides):
    """What evict_from_cache's call says; with a workspace that is too small, which is looked at last."""
    pages, K, page, D = shape
    c = (ctypes.c_int64 * 6)(*strides)
    return lib.afa_paged_evict(dt, pages, page, 1, 1, K, D, DUMMY, DUMMY, k, v, c, DUMMY, 1, 0, 0, DUMMY, page, DUMMY, DUMMY, DUMMY, 16,
                               None)


def _bytes(base, shape, strides, esz):
    at = {0}
    for n, st in zip(shape, strides):
        at = {a + i * st for a in at for i in range(n)}
    return {base + a * esz + b for a in at for b in range(esz)}


def _layout(rng, shape, gaps):
    """Strides of a random order of the axes but the last, with gaps between rows, and how many elements they span."""
    strides, span = [0, 0, 0, 1], shape[3] + (rng.randint(0, 4) if gaps else 0)
    for axis in rng.sample(range(3), 3):
        strides[axis] = span
        span = span * shape[axis] + (rng.randint(0, 3) if gaps else 0)
    return strides, span


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("alike", [True, False])
def test_shared_places_by_brute_force(lib, seed, alike):
    rng = random.Random(seed)
    seen = set()
    for _ in range(150):
        dt = rng.choice(list(ESZ))
        shape = [rng.randint(1, 4) for _ in range(3)] + [rng.randint(1, 6)]
        ks, span = _layout(rng, shape, rng.random() < 0.7)
        if rng.random() < 0.5:  # room beside each row, head or slot, for another's
            at = rng.choice([st for st in ks if st > 1] or [span])
            ks = [st * 2 if st >= at else st for st in ks]
        vs = ks if alike else _layout(rng, shape, True)[0]
        k = 1 << 20
        v = k + ESZ[dt] * rng.randint(-2 * span, 2 * span) + (rng.choice([0, 0, 1]) if ESZ[dt] > 2 else 0)
        want = not _bytes(k, shape, ks, ESZ[dt]).isdisjoint(_bytes(v, shape, vs, ESZ[dt]))
        rc = _evict(lib, dt, shape, k, v, ks[:3] + vs[:3])
        assert rc == (_lib.ERR_OVERLAP if want else _lib.ERR_WORKSPACE), (shape, ks, vs, v - k, want)
        seen.add(want)
    assert seen == {True, False}


@pytest.mark.parametrize("order", list(itertools.permutations(range(4))))
def test_large_pages_side_by_side(lib, order):
    """A large pool whose k and v lie side by side in any place of one array's order, apart by it; and one element nearer."""
    shape, esz = (20000, 8, 64, 128), 2
    sizes = {0: 20000, 1: 8, 2: 64, 3: 2}  # pages, heads, slots, k and v
    strides, span = {}, 128
    for axis in order:
        strides[axis], span = span, span * sizes[axis]
    s = [strides[0], strides[1], strides[2]] * 2
    k = 1 << 30
    assert _evict(lib, _lib.AFA_BF16, shape, k, k + esz * strides[3], s) == _lib.ERR_WORKSPACE
    assert _evict(lib, _lib.AFA_BF16, shape, k + esz * strides[3], k, s) == _lib.ERR_WORKSPACE
    for off in (-1, 1):
        assert _evict(lib, _lib.AFA_BF16, shape, k, k + esz * (strides[3] + off), s) == (
            _lib.ERR_OVERLAP if off < 0 or strides[3] < span // 2 else _lib.ERR_WORKSPACE)


def test_large_pages_in_two_orders(lib):
    """k by heads and then slots, v by slots and then heads, in the halves of each page of one array."""
    shape, half = (20000, 8, 64, 128), 8 * 64 * 128
    s = [2 * half, 64 * 128, 128, 2 * half, 128, 8 * 128]
    k = 1 << 30
    assert _evict(lib, _lib.AFA_BF16, shape, k, k + 2 * half, s) == _lib.ERR_WORKSPACE
    for off in (-1, 1, -half, half, 15000 * 2 * half - 1, -15000 * 2 * half + 1):
        assert _evict(lib, _lib.AFA_BF16, shape, k, k + 2 * (half + off), s) == _lib.ERR_OVERLAP


def test_strides_of_any_size(lib):
    """Numbers that no array has: an answer, and no overflow."""
    for s in (2 ** 62, -2 ** 63, 2 ** 46, 2 ** 45, 0, -1):
        for v in (DUMMY, 1 << 40, (1 << 63) + 8):
            assert _evict(lib, _lib.AFA_F64, (7, 3, 16, 8), DUMMY, v, [s, s, s, s, s, s]) in (_lib.ERR_OVERLAP, _lib.ERR_WORKSPACE)
            assert _evict(lib, _lib.AFA_F64, (7, 3, 16, 8), DUMMY, v, [s, 1, 8, 3, s, s]) in (_lib.ERR_OVERLAP, _lib.ERR_WORKSPACE)


def test_cache_write_refuses_shared_places(lib):
    p = _plan()
    s = (ctypes.c_int64 * 6)(*[16 * 4 * 64, 64, 4 * 64] * 2)  # (pages, slots, k and v, heads, dim)
    for off in (0, 64, -64, 32, 16 * 4 * 64):
        v = (1 << 20) + 2 * off
        assert lib.afa_paged_append(ctypes.byref(p), DUMMY, DUMMY, DUMMY, None, DUMMY, 1 << 20, v, s, None, None, 0, None, 1, None,
                                    None) == _lib.ERR_OVERLAP
        assert lib.afa_paged_append_norm(ctypes.byref(p), DUMMY, DUMMY, DUMMY, None, DUMMY, 1 << 20, v, s, DUMMY, DUMMY, 1e-6, None, None,
                                         0, None, 1, None, None) == _lib.ERR_OVERLAP


def test_status_of_shared_places(lib):
    assert "overlap" in lib.afa_status_string(_lib.ERR_OVERLAP).decode()
    with pytest.raises(ValueError, match="overlap"):
        _lib.check(_lib.ERR_OVERLAP, "evict_from_cache")
