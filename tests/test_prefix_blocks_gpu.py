"""Attention behind a shared prefix with more blocks of rows a key head than the device holds workgroups of it, so that several of
them begin in one workgroup's stretch.  Against float64 in some of the heads, within the bounds of tests/test_prefix_gpu.py."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from tests.test_paged_gpu import BF16, F16, F32, U, _close, _f64, _half, _tiny, _weight_error
from tests.test_prefix_gpu import _Shared

pytestmark = pytest.mark.gpu


def _check_heads(x, heads, sink=0.5):
    out, den = x.call(sink, return_denominator=True)
    q, pk, pv = _f64(x.q[:, heads]), _f64(x.pk), _f64(x.pv)
    got, wants, bounds = _f64(out[:, heads]), np.zeros(q.shape), np.zeros(q.shape)
    wden, bden = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for r, (c, n) in enumerate(x.lens):
        for u, h in enumerate(heads):
            kh = h * x.K // x.H
            k, v = (np.concatenate((p[kh], _f64(own[r][:, kh]))) for p, own in ((pk, x.k), (pv, x.v)))
            for i in range(n):
                t, seen = x.starts[r] + i, pk.shape[1] + c + i + 1
                want, d, size, S = P.attention_row(q[t, u], k[:seen], v[:seen], sink)
                e = _weight_error(x.dt, x.D, S, seen)
                wants[t, u], wden[t, u], bden[t, u] = want, d, 2 * e * d
                bounds[t, u] = (2 * e + x.plane()) * size + (_half(x.dt) + 4 * U) * np.abs(want) + _tiny(x.dt)
    off = (np.abs(got - wants) > bounds).any((1, 2))
    assert not off.any(), ("rows", np.flatnonzero(off)[:8], int(off.sum()), "of", len(off))
    _close(den[:, heads], wden, bden, "denominator")
    return out


def _blocks(K, G, rows):
    """Requests of up to 130 new tokens, `rows` rows a key head in all, or up to G - 1 more."""
    left, lens = -(-rows // G), []
    while left:
        lens.append((len(lens) % 3, min(left, 130)))
        left -= lens[-1][1]
    return lens


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("share,G,D,L,per,more", [
    (2, 1, 32, 33, 1, -1), (2, 1, 32, 33, 1, 0), (2, 1, 32, 33, 1, 1), (2, 1, 32, 33, 2, 1), (2, 1, 64, 1, 3, 5), (2, 1, 128, 700, 2, 1),
    (8, 4, 48, 100, 2, 70), (4, 2, 96, 321, 2, -1), (1, 1, 64, 250, 3, 0), (2, 1, 256, 65, 2, 1),
])
def test_prefix_of_more_blocks_than_workgroups(dt, share, G, D, L, per, more):
    """`share` workgroups a key head, and per times as many blocks of 128 rows of it, or one row fewer or more; values that are
    not finite; the same bits each time."""
    K = 2 * torch.cuda.get_device_properties(0).multi_processor_count // share
    lens = _blocks(K, G, 128 * share * per + more)
    x = _Shared(dt, lens, K * G, K, D, 16, L, seed=D + L, max_tree=0, parents=False)
    out = _check_heads(x, [0, K * G // 2, K * G - 1])
    assert torch.equal(x.call(), out)
    x.pv[0, L - 1, 3], x.pv[0, 0, D - 1] = float("inf"), float("nan")
    got = x.call()
    assert (got[:, :G, 3] == float("inf")).all() and torch.isnan(got[:, :G, D - 1]).all()
    same = torch.ones_like(got, dtype=torch.bool)
    same[:, :G, 3] = same[:, :G, D - 1] = False
    assert torch.equal(got[same], out[same])
