"""Attention of requests that share a prefix on the GPU, against float64 rows over the prefix and the request's own tokens.
Tolerances as derived in tests/test_paged_gpu.py: the prefix's keys are keys like the others.  With more than 64 rows a key head
(tokens times heads of a group) bf16 and fp16 weights enter the prefix's product in one plane of the type instead of two, off by
half a step h of it each: h more in the numerator, nothing in the row sums, which are of the weights in fp32."""
import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from oracle import paged_oracle as P
from tests.test_paged_gpu import (BF16, F16, F32, F64, LENS, U, _Cache, _close, _f64, _half, _i32, _tables, _tiny,
                                  _weight_error)

pytestmark = pytest.mark.gpu


class _Shared(_Cache):
    """A step whose requests see L keys and values before their own."""

    def __init__(self, dt, lens, H, K, D, page, L, layout="khld", pscale=1.0, **kw):
        super().__init__(dt, lens, H, K, D, page, **kw)
        rng = np.random.default_rng(L + D)
        self.pk, self.pv = (torch.tensor(rng.standard_normal((K, L, D)) * s, device="cuda").to(dt) for s in (pscale, 1.0))
        if layout == "lkhd":  # tokens before heads, as projections leave them, k and v side by side
            both = torch.stack((self.pk, self.pv)).permute(2, 0, 1, 3).contiguous()
            self.pk, self.pv = both[:, 0].transpose(0, 1), both[:, 1].transpose(0, 1)
        if layout == "gap":
            wide = torch.full((2, K, L + 3, D + 3), float("nan"), device="cuda", dtype=dt)
            wide[:, :, :L, 1:D + 1] = torch.stack((self.pk, self.pv))
            self.pk, self.pv = wide[0, :, :L, 1:D + 1], wide[1, :, :L, 1:D + 1]

    def call(self, sink=0.5, **kw):
        return A.paged_prefix_afa(self.q, self.pk, self.pv, self.kp, self.vp, self.plan, sink, **kw)

    def want(self, sink, sees=None):
        sees = self.sees if sees is None else sees
        T = self.q.shape[0]
        out, size = np.zeros((T, self.H, self.D)), np.zeros((T, self.H, self.D))
        den, e = np.zeros((T, self.H)), np.zeros((T, self.H))
        q, pk, pv = _f64(self.q), _f64(self.pk), _f64(self.pv)
        for r, (c, n) in enumerate(self.lens):
            k, v = _f64(self.k[r]), _f64(self.v[r])
            for i in range(n):
                t = self.starts[r] + i
                drafted = np.arange(n) <= i if n > sees.shape[1] else sees[t, :n]
                see = np.concatenate((np.ones(c, bool), drafted))
                for h in range(self.H):
                    kh = h * self.K // self.H
                    keys, values = np.concatenate((pk[kh], k[see, kh])), np.concatenate((pv[kh], v[see, kh]))
                    out[t, h], den[t, h], size[t, h], S = P.attention_row(q[t, h], keys, values, sink)
                    e[t, h] = _weight_error(self.dt, self.D, S, len(keys))
        return out, den, size, e

    def plane(self):
        """What one plane of the weights adds to the error of the numerator."""
        return _half(self.dt) if self.dt in (BF16, F16) and self.q.shape[0] * self.H // self.K > 64 else 0

    def check(self, sink=0.5, masks=None, sees=None, what="", **kw):
        out, den = self.call(sink, masks=masks, return_denominator=True, **kw)
        want, wden, size, e = self.want(sink, sees)
        u = 0 if self.dt == F64 else U
        bound = (2 * e[..., None] + self.plane()) * size + _half(self.dt) * np.abs(want) + 4 * u * np.abs(want) + _tiny(self.dt)
        live = sum(n for _, n in self.lens)
        _close(out[:live], want[:live], np.where(np.isnan(bound), 0, bound)[:live], what)
        _close(den[:live], wden[:live], (2 * e * wden)[:live], (what, "denominator"))
        return out, den


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,D,page,L,layout", [
    (4, 2, 64, 16, 1, "khld"), (2, 2, 128, 64, 31, "lkhd"), (6, 6, 48, 32, 333, "khld"), (8, 1, 96, 8, 64, "lkhd"),
    (3, 3, 32, 128, 100, "khld"), (4, 1, 256, 16, 77, "lkhd"), (6, 2, 40, 3, 50, "khld"), (16, 1, 64, 32, 129, "gap"),
    (2, 1, 80, 1, 5, "lkhd"), (1, 1, 7, 5, 300, "khld"), (12, 4, 128, 16, 65, "khld"),
])
def test_prefix(dt, H, K, D, page, L, layout):
    """Requests of every kind behind short and long prefixes: no cached tokens, no new ones, trees; rows behind the last 0."""
    x = _Shared(dt, LENS, H, K, D, page, L, layout, seed=D + page, tail=3)
    out, den = x.check(what=(H, K, D, page, L))
    assert (out[-3:] == 0).all() and (den[-3:] == 0).all()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,n,L,G,D", [(1, 1, 700, 1, 64), (3, 2, 1025, 1, 64), (17, 1, 513, 2, 128), (40, 1, 400, 4, 64),
                                       (70, 2, 321, 4, 128), (5, 33, 257, 1, 48), (150, 3, 161, 1, 32), (9, 2, 290, 4, 256)])
def test_prefix_rows(dt, R, n, L, G, D):
    """From one row a key head to several blocks of rows, each over prefixes that end inside a tile."""
    _Shared(dt, [(r % 5, n) for r in range(R)], 2 * G, 2, D, 16, L, seed=R, max_tree=0, parents=False).check(what=(R, n, L))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("scale,pscale", [(3.0, 1.0), (0.05, 1.0), (4.0, 2.0), (1.0, 0.0)])
def test_prefix_scores(dt, scale, pscale):
    """Scores from near 0 to beyond 30 of both signs, larger in the prefix or in the request's own tokens."""
    _Shared(dt, [(200, 4), (33, 9), (0, 3)], 4, 2, 64, 32, 250, seed=3, scale=scale, pscale=pscale).check(what=scale)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 48])
@pytest.mark.parametrize("scale,pscale,how", [(3.0, 1.0, None), (0.05, 1.0, None), (4.0, 2.0, None), (1.0, 0.0, None), (1.0, 8.0, None),
                                              (1.0, 6.0, "rising"), (1.0, 6.0, "falling"), (1.0, 1.0, "negative"),
                                              (6.0, 6.0, "negative")])
def test_prefix_scores_of_many_rows(dt, D, scale, pscale, how):
    """Scores near 0 and beyond 100 of both signs over more than 64 rows a key head; larger and smaller ones from tile to tile; a
    prefix that points away from all queries.  In fp16 a weight far below its row's largest is off by up to 2^-25 of that: 300
    of them by 9e-6, within the error of the weights (_weight_error)."""
    x = _Shared(dt, [(20, 40), (0, 33), (3, 9)], 4, 2, D, 16, 300, seed=6, scale=scale, pscale=pscale)
    if how in ("rising", "falling"):
        steps = torch.linspace(0.02, 1, 300, device="cuda")[None, :, None]
        x.pk = (x.pk.float() * (steps if how == "rising" else steps.flip(1))).to(dt)
    if how == "negative":
        x.q, x.pk = (x.q.abs() + 0.25).to(dt), -x.pk.abs()
    x.check(what=(D, scale, pscale, how))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_prefix_negative_scores(dt):
    """A prefix that all points away from the queries: weights far below 1, no sink."""
    x = _Shared(dt, [(0, 3), (0, 20)], 2, 2, 64, 16, 150, seed=4)
    x.q = (x.q.abs() + 0.25).to(dt)
    x.pk = -x.pk.abs()
    for r, (c, n) in enumerate(x.lens):
        at = torch.arange(c + n, device="cuda")
        pg = torch.tensor(x.tables[r], device="cuda", dtype=torch.int64)[at // 16]
        x.k[r] = (-x.k[r].abs()).to(dt)
        x.kp[pg, :, at % 16] = x.k[r]
    x.check(sink=0.0)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_prefix_is_what_pages_would_give(dt):
    """The same tokens as every request's first cached ones: paged_tree_afa's result, within both bounds."""
    L, page, K, D, lens = 96, 32, 2, 64, [(40, 3), (0, 1), (7, 5)]
    x = _Shared(dt, lens, 4, K, D, page, L, seed=7)
    out, den = x.check()
    y = _Cache(dt, [(c + L, n) for c, n in lens], 4, K, D, page, seed=7)
    y.q, y.plan.masks[:] = x.q, x.plan.masks
    for r, (c, n) in enumerate(lens):
        at = torch.arange(L + c + n, device="cuda")
        pg = torch.tensor(y.tables[r], device="cuda", dtype=torch.int64)[at // page]
        for pages_, own, first in ((y.kp, x.k[r], x.pk), (y.vp, x.v[r], x.pv)):
            pages_[pg, :, at % page] = torch.cat((first.transpose(0, 1), own))
    other, oden = A.paged_tree_afa(y.q, y.kp, y.vp, y.plan, 0.5, return_denominator=True)
    want, wden, size, e = x.want(0.5)
    _close(other, want, 2 * e[..., None] * size + 2 * _half(dt) * np.abs(want) + _tiny(dt), "pages")
    _close(oden, wden, 2 * e * wden, "pages")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_prefix_of_hidden_drafts(dt):
    """Masks that leave a row nothing of its own: the prefix alone; requests that are not served: 0; rows behind the last: as they were."""
    x = _Shared(dt, [(0, 4), (0, 2)], 4, 2, 64, 16, 70, seed=2, tail=2)
    none = torch.zeros_like(x.plan.masks)
    out, den = x.check(masks=none, sees=np.zeros_like(x.sees))
    assert (out[-2:] == 0).all() and (den[-2:] == 0).all()
    kept = torch.full_like(x.q, 9.0)
    x.call(masks=none, out=kept)
    assert torch.equal(kept[:-2], out[:-2]) and (kept[-2:] == 9).all()
    A.build_block_tables(x.plan, _i32([0, 10 ** 6]), _i32([4, 2]))
    got, den = x.call(0.25, return_denominator=True)
    assert (got[4:6] == 0).all() and (den[4:6] == 0.25).all() and (got[:4] != 0).any()
    A.build_block_tables(x.plan, _i32([0, 0]), _i32([0, 0]))
    got, den = x.call(0.25, return_denominator=True)
    assert (got == 0).all() and (den == 0).all()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("new", [9, 30, 130])
def test_prefix_values_that_are_not_finite(dt, new):
    """An infinity or a NaN in a prefix value is every row's result in that feature; NaN in a key is the row's.  Few and many
    rows a key head, in one block and in several."""
    x = _Shared(dt, [(50, 3), (0, new), (1, 1)], 4, 2, 64, 16, 200, seed=2)
    plain = x.call()
    x.pv[0, 17, 5], x.pv[1, 199, 63], x.pv[0, 3, 40] = float("inf"), float("-inf"), float("nan")
    got = x.call()
    assert (got[:, :2, 5] == float("inf")).all() and (got[:, 2:, 63] == float("-inf")).all() and torch.isnan(got[:, :2, 40]).all()
    same = torch.ones_like(got, dtype=torch.bool)
    same[:, :2, 5], same[:, 2:, 63], same[:, :2, 40] = False, False, False
    assert torch.equal(got[same], plain[same])
    # and where requests see a value of the other sign in their own tokens too
    x.vp.copy_(torch.where(torch.isnan(x.vp), x.vp, torch.full_like(x.vp, float("-inf"))))
    assert torch.isnan(x.call()[:, :2, 5]).all()
    x.pk[1, 100, 1] = float("nan")
    got = x.call()
    assert torch.isnan(got[:, 2:]).all()


def test_prefix_repeats_and_streams():
    """The same bits on every call, on another stream, and from two plans at once on two streams."""
    x = _Shared(BF16, [(100 + 7 * r, 1 + r % 3) for r in range(60)], 8, 2, 128, 16, 2999, seed=1, max_tree=0, parents=False)
    y = _Shared(BF16, [(30 + 5 * r, 2) for r in range(30)], 8, 2, 128, 16, 1777, seed=2, max_tree=0, parents=False)
    wx, wy = x.call(), y.call()
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for s, z in zip(sides, (x, y)):
            with torch.cuda.stream(s):
                got.append(z.call())
        torch.cuda.synchronize()
        assert torch.equal(got[0], wx) and torch.equal(got[1], wy)


def test_prefix_captured():
    """A step in a graph, replayed with other lengths, queries and prefixes, eager steps in between."""
    x = _Shared(BF16, [(100 + 7 * r, 1 + r % 3) for r in range(20)], 8, 2, 64, 16, 1000, seed=1, max_tree=0, parents=False, tail=9)
    cached, new = _i32([c for c, _ in x.lens]), _i32([n for _, n in x.lens])
    x.kp.nan_to_num_(0.5), x.vp.nan_to_num_(0.25)
    step = lambda: (A.build_block_tables(x.plan, cached, new), x.call(return_denominator=True))[1]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(5):
        x.q.normal_(), x.pk.normal_(), x.pv.normal_()
        cached.copy_(_i32([(c + 3 * i) % 200 for c, _ in x.lens]))
        new.copy_(_i32([(n + i) % 3 for _, n in x.lens]))
        graph.replay()
        a = [t.clone() for t in got]
        b = step()
        torch.cuda.synchronize()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_prefix_refusals():
    x = _Shared(BF16, [(5, 2)], 4, 2, 64, 16, 20)
    k, v = x.pk, x.pv
    call = lambda pk, pv, **kw: A.paged_prefix_afa(x.q, pk, pv, x.kp, x.vp, x.plan, **kw)  # noqa: E731
    for pk, pv in ((k[0], v), (k[:1], v), (k, v[:, :5]), (k[..., :32], v), (k[:, :0], v[:, :0]), (k.transpose(0, 2), v)):
        with pytest.raises(ValueError):
            call(pk, pv)
    with pytest.raises(ValueError, match="contiguous head"):
        call(k.transpose(1, 2).contiguous().transpose(1, 2), v)
    with pytest.raises(TypeError):
        call(k.half(), v)
    with pytest.raises(RuntimeError, match="GPU"):
        call(k.cpu(), v)
    with pytest.raises(RuntimeError, match="gradient"):
        call(k, v.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="overlap"):
        call(k, v, out=k.view(-1)[:x.q.numel()].view_as(x.q))
    with pytest.raises(ValueError, match="sink"):
        call(k, v, sink_omega=-1.0)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D,L", [(128, 20000), (32, 9001), (96, 7000)])
def test_prefix_of_many_rows_in_many_parts(dt, D, L):
    """One block of rows, whose keys all workgroups share, and a few of them: more parts than are added up at once; values that are
    not finite in some of the parts; the same bits each time."""
    for R in (70, 150):
        x = _Shared(dt, [(r % 3, 1) for r in range(R)], 1, 1, D, 16, L, seed=R, max_tree=0, parents=False)
        out, den = x.check(what=(D, L, R))
        assert torch.equal(x.call(), out)
        x.pv[0, L // 2, 3], x.pv[0, L - 1, D - 1] = float("inf"), float("nan")
        got = x.call()
        assert (got[:R, 0, 3] == float("inf")).all() and torch.isnan(got[:R, 0, D - 1]).all()
        same = torch.ones_like(got, dtype=torch.bool)
        same[..., 3] = same[..., D - 1] = False
        assert torch.equal(got[same], out[same])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R", [3, 60])
def test_prefix_beside_rows_of_nan(dt, R):
    """Rows of NaN, and those of requests that are not served, whatever they hold: their own results alone."""
    x = _Shared(dt, [(r % 5, 2) for r in range(R)], 4, 2, 64, 16, 500, seed=R, max_tree=0, parents=False)
    out, den = x.check()
    x.q[2, 1] = float("nan")
    cached = _i32([10 ** 6 if r == 0 else r % 5 for r in range(R)])
    A.build_block_tables(x.plan, cached, _i32([2] * R))
    x.q[0] = float("nan")
    got = x.call()
    assert (got[:2] == 0).all() and torch.isnan(got[2, 1]).all()
    same = torch.ones_like(got, dtype=torch.bool)
    same[:2], same[2, 1] = False, False
    assert torch.equal(got[same], out[same])


@pytest.mark.parametrize("dt", [BF16, F32, F64])
def test_prefix_in_the_librarys_own_workspace(dt):
    """The C call without a workspace: the same bits; and without the matrix cores, within the bounds."""
    import ctypes

    from algebraic_intelligence_amd import _lib
    x = _Shared(dt, [(5, 2), (40, 3)], 4, 2, 64, 16, 300, seed=3)
    want, _ = x.check()
    for flags in (_lib.FLAG_ZERO_TAIL, _lib.FLAG_ZERO_TAIL | _lib.FLAG_GENERIC):
        out = torch.empty_like(x.q)
        rc = _lib.lib().afa_paged_prefix_fwd(x.plan._ref, x.q.data_ptr(), None, x.pk.data_ptr(), x.pv.data_ptr(), 300, None,
                                             x.kp.data_ptr(), x.vp.data_ptr(), None, None, out.data_ptr(), None, 0.5, flags, None, 0,
                                             ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        if flags == _lib.FLAG_ZERO_TAIL or dt == F64:
            assert torch.equal(out, want)
        ref, _, size, e = x.want(0.5)
        _close(out, ref, 2 * e[..., None] * size + (_half(dt) + 4 * U) * np.abs(ref) + _tiny(dt), flags)
