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


@pytest.mark.parametrize("dt,score", [(t, s) for t in (BF16, F16, F32) for s in (90, 300, 1000, 3000)]
                         + [(F16, 15000), (F32, 15000)])
@pytest.mark.parametrize("H,K,n", ROWS)
def test_weights_far_below_one(dt, score, H, K, n):
    """Every score is the same far negative one and there is no sink: the result is the mean of the visible
    values.  The scores are exact (a^2 of 16 bits, 64 of them), so that a row's weights are equal and what
    they lose to their planes is common to all: each product's planes h^2, for fp16 planes 2^-25 of a row's
    largest weight, and N sums.  Each of the at most 2 N + 2 products, sums and scalings that falls below the smallest
    normal number, 2^-126, is off by half a subnormal step, 2^-150, of the N w that it is divided by."""
    a = {90: 3.375, 300: 6.125, 1000: 11.1875, 3000: 19.375, 15000: 43.25}[score]
    x = _Cache(dt, [(150, n), (33, n), (0, 2)], H, K, 64, 16, seed=n)
    x.q = torch.full_like(x.q, a)
    _set_keys(x, 16, lambda k: torch.full_like(k, -a))
    out, den = _run(x, sink_omega=0.0)
    w = (np.sqrt(1 + (8 * a * a) ** 2) + 8 * a * a) ** -8.0
    for r, (c, m) in enumerate(x.lens):
        v = _f64(x.v[r])
        for i in range(m):
            t = x.starts[r] + i
            see = np.concatenate((np.ones(c, bool), x.sees[t, :m]))
            N = int(see.sum())
            e = 105 * U + (0 if dt == F32 else 2.2e-4)
            _close(den[t], np.full(H, N * w), np.full(H, (e + N * U) * N * w), (r, i))
            mean, size = (np.repeat(y[see].mean(0), H // K, 0) for y in (v, np.abs(v)))
            e = 2 * N * U + (0 if dt == F32 else _half(dt) ** 2) + (N * 2.0 ** -25 if dt == F16 else 0)
            small = (2 * N + 2) * 2.0 ** -150 / (N * w)
            _close(out[t], mean, e * size + (_half(dt) + 2 * U) * np.abs(mean) + small + _tiny(dt), (r, i))


@pytest.mark.parametrize("scale", [45.0, 150.0])
def test_fp16_negative_scores(scale):
    """Random scores of about -230 and -770, no sink."""
    x = _Cache(F16, [(150, 3), (40, 20)], 2, 2, 64, 16, seed=4)
    x.q = ((x.q.abs() + 0.25) * scale).to(F16)
    _set_keys(x, 16, lambda k: -k.abs())
    x.check(sink=0.0)


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,n", ROWS)
@pytest.mark.parametrize("cached,D", [(40, 64), (700, 64), (60, 128), (60, 48)])
def test_cached_values_that_are_not_finite(dt, H, K, n, cached, D):
    """An infinity or NaN among the cached values is the result, in its feature, of every row of its request;
    infinities of both signs are NaN; nothing else changes."""
    x = _Cache(dt, [(cached, n), (33, n), (70, 1)], H, K, D, 16, seed=cached + n)
    first, den = _run(x)

    def put(key, feature, value):
        x.vp[x.tables[0][key // 16], :, key % 16, feature] = float(value)

    put(3, 5, "inf")
    put(9, 1, "-inf")
    put(11, 2, "nan")
    put(2, D - 1, "inf")
    put(cached - 1, D - 1, "-inf")
    put(cached + 1, 5, "-inf")  # drafted: NaN with the cached one in the rows that see it
    want = first.clone()
    want[:n, :, 5], want[:n, :, 1], want[:n, :, 2], want[:n, :, D - 1] = (float(s) for s in ("inf", "-inf", "nan", "nan"))
    sees = torch.tensor(x.sees[:n, 1], device="cuda")
    assert 0 < sees.sum() < n
    want[:n, :, 5][sees] = float("nan")
    out, same = _run(x)
    assert torch.equal(same, den)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(out), nan)
    assert torch.equal(out[~nan], want[~nan])


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,n", ROWS)
@pytest.mark.parametrize("D,page", [(64, 16), (40, 5)])
def test_scores_far_below_zero(dt, H, K, n, D, page):
    """A key whose score's eighth power, and whose square, no longer fit weighs nothing, as one of score -26250 or
    -33200 does (2^-125 or less beside weights of about 1): the same results bit for bit.  Its infinity is
    seen all the same.  A score of -infinity is the last of them; one of infinity or NaN makes its rows NaN."""
    x = _Cache(dt, [(40, n), (0, 3)], H, K, D, page, seed=n)
    x.q[..., 0] = 300.0
    _set_keys(x, page, lambda k: torch.cat((torch.zeros_like(k[..., :1]), k[..., 1:]), -1))
    where, slot = x.tables[0][7 // page], 7 % page
    at = x.kp[where, :, slot]
    at.zero_()
    at[:, 0] = -700.0
    x.vp[where, :, slot, 1] = 1.0
    want = _run(x)
    assert all(torch.isfinite(t).all() for t in want)
    for k in (-1200.0, -1e6, -3e30, float("-inf")):
        at[:, 0] = k
        for got, ref in zip(_run(x), want):
            assert torch.equal(got, ref), k
        x.vp[where, :, slot, 1] = float("inf")
        out, _ = _run(x)
        assert (out[:n, :, 1] == float("inf")).all()
        out[:n, :, 1] = want[0][:n, :, 1]
        assert torch.equal(out, want[0])
        x.vp[where, :, slot, 1] = 1.0
    for k in (float("inf"), float("nan")):
        at[:, 0] = k
        out, den = _run(x)
        assert torch.isnan(out[:n]).all() and not torch.isfinite(den[:n]).any()
        assert torch.equal(out[n:], want[0][n:])
