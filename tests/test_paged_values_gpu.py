"""The serving operators' values where keys, values and weights are far from ordinary: scores that only other
rows see, weights below every 16-bit number, cached infinities.

Bounds count roundings as tests/test_paged_gpu.py does.
"""
import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from tests.test_paged_gpu import BF16, F16, F32, F64, U, _Cache, _close, _f64, _half, _tiny

pytestmark = pytest.mark.gpu


def _set_keys(x, page, change):
    """Every key that x's requests hold becomes change(key rows), in the pages and in x.k."""
    for r, (c, n) in enumerate(x.lens):
        at = torch.arange(c + n, device="cuda")
        pg = torch.tensor(x.tables[r], device="cuda", dtype=torch.int64)[at // page]
        x.k[r] = change(x.k[r]).to(x.dt)
        x.kp[pg, :, at % page] = x.k[r]


def _run(x, **kw):
    return A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, return_denominator=True, **kw)


# rows of a segment that the plan makes of (H, K, new): 16, 32, 64, 128
ROWS = [(2, 2, 11), (4, 2, 13), (4, 2, 30), (8, 2, 30)]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("H,K,n", ROWS)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32)])
def test_weights_do_not_depend_on_hidden_keys(dt, H, K, n, D, page):
    """A row's weights and their sum, bit for bit, whatever lies behind the last key and in the drafted keys
    that it does not see: the visible scores are about -4, those of the hidden keys far below -8."""
    x = _Cache(dt, [(20, n), (0, n // 2), (45, 1)], H, K, D, page, seed=D + n)
    # mean |a||b| of normal numbers is 2 / pi, so the scores have mean -4
    x.q = (x.q.abs() * (4 / (np.sqrt(D) * 2 / np.pi))).to(dt)
    _set_keys(x, page, lambda k: -k.abs())
    first = _run(x)
    # behind the last key of each request
    for r, (c, m) in enumerate(x.lens):
        if (c + m) % page:
            x.kp[x.tables[r][-1], :, (c + m) % page:] = -90.0
    for got, want in zip(_run(x), first):
        assert torch.equal(got, want)
    # a drafted key of the first request, for the rows that do not see it
    place = 20 + n // 2
    x.kp[x.tables[0][place // page], :, place % page] = -90.0
    hidden = torch.tensor(~x.sees[:, n // 2], device="cuda")
    hidden[n:] = True
    assert 0 < hidden[:n].sum() < n
    for got, want in zip(_run(x), first):
        assert torch.equal(got[hidden], want[hidden])
