"""Accumulated attention weights of scores far from 0 on the GPU, with and without the matrix cores."""
import ctypes

import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from algebraic_intelligence_amd import _lib
from oracle import paged_oracle as P
from tests.test_paged_gpu import BF16, F16, F32, F64, U, _Cache, _f64

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


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("flags", [0, _lib.FLAG_GENERIC])
def test_weights_of_rows_with_large_denominators(dt, D, flags):
    """Denominators up to fp32's end: a row gives its largest key 1, whatever the denominator, and others their shares.

    Scores are exact but for their scaling (16 u of a weight), the denominator is off by (121 + keys) u and 2.2e-4 on 16-bit inputs, as a
    weight is; the inverse of a denominator above 2^126 is a subnormal number with 22 bits or more: 2^-22.  Two keys of one score
    have half each."""
    x = _Cache(dt, [(37, 2), (70, 3), (0, 5)], 4, 2, D, 16, max_tree=0, parents=False, seed=D)
    T = x.q.shape[0]
    score = np.array([3000, 14000, 25000, 27600, 28500, 29500, 30500, 31500, 32500, 32700])[:T, None]
    unit = 4 if dt == F16 else 64
    first = np.floor(score * np.sqrt(D) / 64 / unit) * unit
    if dt == BF16:  # 8 bits
        first = torch.tensor(first).bfloat16().double().numpy()
        first = np.where(first * 64 / np.sqrt(D) > 32700, first - 64, first)
    q = np.zeros((T, 4, D))
    q[..., 0] = first
    x.q = torch.tensor(q, device="cuda").to(dt)

    def own(r, n):
        k = np.zeros((n, 2, D))
        k[0, :, 0] = 64.0
        k[min(2, n - 1):3, 1, 0] = 64.0  # the second head has two such keys in a request
        return k

    _keys(x, own)
    # the largest denominators are twice a weight in the second head: those that pass fp32 are left out below
    _, den = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, 0.5, return_denominator=True)
    w = _f64(_weights(x, den, flags))
    for r, (c, n) in enumerate(x.lens):
        want = np.zeros(c + n)
        k = _f64(x.k[r])
        for i in range(n):
            t = x.starts[r] + i
            for h in range(4):
                if not torch.isfinite(den[t, h]):
                    continue
                weight = np.where(np.arange(c + n) <= c + i, P.rho8(k[:, h // 2] @ _f64(x.q[t, h]) / np.sqrt(D)), 0)
                want += weight / (weight.sum() + 0.5)
        e = 2 * ((121 + c + n) * U + (2.2e-4 if dt != F32 else 0)) + 2.0 ** -22 + (4 * n + 4) * U
        assert (np.abs(w[r, :c + n] - want) <= e * want + 4 * n * 2.0 ** -126).all(), (r, w[r, :4], want[:4])
    assert (_f64(den) > 2.0 ** 126).any()
