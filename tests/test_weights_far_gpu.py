"""Accumulated attention weights of scores far from 0 on the GPU, with and without the matrix cores."""
import ctypes

import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from algebraic_intelligence_amd import _lib
from tests.test_paged_gpu import BF16, F32, F64, _Cache

pytestmark = pytest.mark.gpu


def _weights(x, den, flags):
    w = x.pool.new_weights()
    rc = _lib.lib().afa_paged_weights(x.plan._ref, x.q.data_ptr(), None, x.kp.data_ptr(), None, None, den.data_ptr(), w.data_ptr(),
                                      x.pool.max_len, flags, None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    return w


def _keys(x, own):
    """Keys own(r, c + n) for every request, in the pages too."""
    for r, (c, n) in enumerate(x.lens):
        x.k[r] = torch.tensor(own(r, c + n), device="cuda").to(x.dt)
        at = torch.arange(c + n, device="cuda")
        pg = torch.tensor(x.tables[r], device="cuda", dtype=torch.int64)[at // 16]
        x.kp[pg, :, at % 16] = x.k[r]


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F32, 64), (F32, 40), (BF16, 40), (F64, 64)])
def test_weights_of_a_score_of_minus_infinity(dt, D):
    """A key whose score passes the type of the sums, below: the attention lets it weigh the least there is, and so do the accumulated
    weights, in both kernels; the other keys' are as without it."""
    x = _Cache(dt, [(40, 2), (9, 1)], 4, 2, D, 16, max_tree=0, parents=False, seed=1)
    x.q = x.q.abs() + 0.25
    far = 1e300 if dt == F64 else 1e38
    x.q[:, :, 0] = far
    rng = np.random.default_rng(0)

    def own(r, n, low=-far):
        k = rng.standard_normal((n, 2, D))
        k[..., 0] = 0.0
        if r == 0:
            k[7, :, 0] = low
        return k

    _keys(x, own)
    _, den = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, 0.5, return_denominator=True)
    assert torch.isfinite(den).all()
    got = [_weights(x, den, flags) for flags in (0, _lib.FLAG_GENERIC)]
    least = 2.0 ** -1022 if dt == F64 else 2.0 ** -126
    for w in got:
        assert torch.isfinite(w).all() and (w[0, 7] >= 0).all() and float(w[0, 7]) <= 8 * 2 * least / 0.5, w[0, 7]
        assert (w[0, :7] > 0).all() and (w[0, 8:42] > 0).all()
    lens, kept = A.evict_from_cache(x.kp, x.vp, x.pool, got[1], torch.tensor([42, 10], dtype=torch.int32, device="cuda"), 41)
    assert lens.tolist() == [41, 10] and torch.equal(kept[0, :41], torch.cat((got[1][0, :7], got[1][0, 8:42])))
