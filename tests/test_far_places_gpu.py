"""The cache's operators where pages, and keys of a prefix, lie more than 2^32 bytes into their arrays; bounds of the operators' own
tests."""
import pytest
import torch

import algebraic_intelligence_amd as A
from oracle import cache_oracle as C
from tests.test_eviction_gpu import _check, _den
from tests.test_norm_gpu import _forward
from tests.test_paged_gpu import BF16, F16, F32, _Cache, _close, _f64, _i32
from tests.test_prefix_gpu import _Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F32, 40)])
def test_far_pages(dt, D):
    """Weights, the cache write with norms, and an eviction, with and without the matrix cores."""
    lens = [(70, 5), (300, 1), (0, 40)]
    x = _Cache(dt, lens, 8, 4, D, 16, seed=1, far=(1 << 32) // (16 * 4 * D * dt.itemsize) + 5)
    _check(x, _den(x))
    rows = lambda p: [torch.stack([p[x.tables[r][j // 16], :, j % 16] for j in range(c + n)])  # noqa: E731
                      for r, (c, n) in enumerate(lens)]
    T = x.q.shape[0]
    q, k, v = (torch.randn(T, h, D, device="cuda").to(dt) for h in (8, 4, 4))
    scale = torch.linspace(0.5, 2, D, device="cuda")
    A.append_to_cache(q, k, v, x.kp, x.vp, x.plan, norms=(scale, scale))
    want, bound = _forward(_f64(k)[None], _f64(scale), 1e-6, None, None, None, None, dt)
    new = [torch.cat([own[c:] for (c, _), own in zip(lens, rows(p))]) for p in (x.kp, x.vp)]
    _close(new[0][None], want, bound, "k")
    assert torch.equal(new[1], v)
    before, w = [rows(x.kp), rows(x.vp)], torch.rand(3, x.pool.max_len, device="cuda")
    got, _ = A.evict_from_cache(x.kp, x.vp, x.pool, w, _i32([c + n for c, n in lens]), 30, first=2, recent=4)
    assert got.tolist() == [30] * 3
    for p, was in zip((x.kp, x.vp), before):
        for r, own in enumerate(rows(p)):
            assert torch.equal(own[:30], was[r][C.kept(w[r].cpu().numpy(), sum(lens[r]), 30, 2, 4)])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("new", [3, 80])
def test_far_keys_of_a_prefix(dt, new):
    """Keys 2^22 elements apart, few and many rows."""
    L, D, apart = 1100, 64, 1 << 22
    x = _Shared(dt, [(9, new), (0, 1)], 2, 2, D, 16, L, seed=3, max_tree=0, parents=False)
    room = torch.empty(L * apart, dtype=dt, device="cuda")
    pk, pv = (room.as_strided((2, L, D), (D, apart, 1), at) for at in (0, 2 * D))
    x.pk, x.pv = pk.copy_(x.pk), pv.copy_(x.pv)
    assert (x.pv[0, -1].data_ptr() - x.pv.data_ptr()) > 1 << 32
    x.check()
