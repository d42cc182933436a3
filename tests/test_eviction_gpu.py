"""Accumulated attention weights and eviction on the GPU.

Weights, against float64: a score is off by (D + 4) u S (S = max_j sum_d |q_d k_jd| / sqrt(D)), a weight by 8 of these and 105 u
(tests/test_paged_gpu.py), 2.2e-4 more on bf16 and fp16 inputs; a division and the sum over n rows add (n + 4) u.  All terms
are positive, so the sum is off by that of itself; adding it to what was there rounds once.  Eviction copies: exact."""
import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from oracle import cache_oracle as C
from oracle import paged_oracle as P
from tests.test_paged_gpu import BF16, F16, F32, F64, LENS, U, _Cache, _close, _f64, _i32, _pages, _tables

pytestmark = pytest.mark.gpu


def _given(x, den, sees=None):
    """What each token of every request is given, and the bound on it, in float64."""
    sees = x.sees if sees is None else sees
    out, bound = np.zeros((len(x.lens), x.pool.max_len)), np.zeros((len(x.lens), x.pool.max_len))
    q, den = _f64(x.q), _f64(den)
    for r, (c, n) in enumerate(x.lens):
        k = _f64(x.k[r])
        for i in range(n):
            t = x.starts[r] + i
            drafted = np.arange(n) <= i if n > sees.shape[1] else sees[t, :n]
            see = np.concatenate((np.ones(c, bool), drafted))
            for h in range(x.H):
                kh = k[:, h * x.K // x.H]
                w = np.where(see, P.rho8(kh @ q[t, h] / np.sqrt(x.D)), 0) / den[t, h] if den[t, h] else np.zeros(c + n)
                S = float(np.max(np.abs(kh) @ np.abs(q[t, h]))) / np.sqrt(x.D)
                e = (8 * (x.D + 4) * S + 105 + n * x.H + 4) * U + (2.2e-4 if x.dt in (BF16, F16) else 0)
                out[r, :c + n] += w
                bound[r, :c + n] += e * w
    return out, bound


def _check(x, den, masks=None, sees=None, what=""):
    before = torch.rand((len(x.lens), x.pool.max_len), device="cuda")
    w = before.clone()
    got = A.accumulate_cache_weights(x.q, x.kp, den, x.plan, w, masks=masks)
    assert got is w
    given, bound = _given(x, den, sees)
    want = _f64(before)
    for r, (c, n) in enumerate(x.lens):
        if n:
            want[r, c:c + n] = 0
    want += given
    _close(w, want, bound + 2 * U * want + 2.0 ** -149, what)
    # places of no token, and requests without rows, keep their bits
    for r, (c, n) in enumerate(x.lens):
        assert torch.equal(w[r, c + n if n else 0:], before[r, c + n if n else 0:])
    return w


def _den(x, **kw):
    return A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, 0.5, return_denominator=True, **kw)[1]


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,D,page", [
    (4, 2, 64, 16), (2, 2, 128, 64), (6, 6, 48, 32), (8, 1, 96, 8), (3, 3, 32, 128), (4, 1, 256, 16), (6, 2, 40, 3), (16, 1, 64, 32),
    (2, 1, 80, 1), (1, 1, 7, 5), (12, 4, 128, 16),
])
def test_weights(dt, H, K, D, page):
    x = _Cache(dt, LENS, H, K, D, page, seed=D + page, tail=3)
    _check(x, _den(x), what=(H, K, D, page))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("new,max_tree,parents,G", [(70, 64, True, 1), (64, 64, True, 2), (129, 192, True, 1), (100, 0, False, 4),
                                                    (33, 64, False, 8), (200, 64, False, 1), (257, 0, False, 1)])
def test_weights_of_long_drafts(dt, new, max_tree, parents, G):
    """Trees of more words than one, prompts longer than a tree, several blocks of rows and of keys."""
    x = _Cache(dt, [(45, new), (0, new // 2), (300, 1)], 2 * G, 2, 64, 32, max_tree, seed=new, parents=parents)
    _check(x, _den(x), what=(new, G))


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 48), (BF16, 256)])
@pytest.mark.parametrize("lens,G", [([(5, 200), (0, 150), (33, 190), (64, 170)], 1), ([(0, 64)] * 3, 1),
                                    ([(70, 130), (0, 0), (64, 129), (3, 140), (66, 131)], 2), ([(0, 300)], 3),
                                    ([(10, 130), (0, 0), (900, 1), (3, 140)], 4), ([(5, 300), (0, 220), (33, 290), (9, 0), (64, 270)], 4),
                                    ([(40, 600)], 2)])
def test_weights_of_prompts_alike(dt, D, lens, G):
    """Prompts of about one length, some with a request without tokens among them, and of other lengths."""
    x = _Cache(dt, lens, 2 * G, 2, D, 16, max_tree=0, seed=D + G, parents=False, tail=1)
    _check(x, _den(x), what=(lens, G))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("scale", [0.05, 3.0, 8.0])
def test_weights_of_far_scores(dt, scale):
    x = _Cache(dt, [(200, 4), (33, 9), (0, 3)], 4, 2, 64, 32, seed=3, scale=scale)
    _check(x, _den(x), what=scale)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_weights_sum_to_the_rows(dt):
    """Without a sink a row's weights sum to 1 over its tokens: each request's sum to its rows times heads."""
    x = _Cache(dt, [(100, 3), (0, 5), (31, 1), (640, 2)], 4, 2, 64, 16, seed=5)
    den = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, 0.0, return_denominator=True)[1]
    w = A.accumulate_cache_weights(x.q, x.kp, den, x.plan, x.pool.new_weights())
    rows = np.array([4.0 * n for _, n in x.lens])
    # both calls' weights: each off by its own bound
    e = 2 * ((8 * 68 * 10 + 105 + 700) * U + (2.2e-4 if dt != F32 else 0)) + 1e-5
    np.testing.assert_allclose(w.double().sum(1).cpu().numpy(), rows, rtol=e)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_weights_edges(dt):
    """Masks that hide every drafted token, rows whose denominator is 0, keys that are not finite where nobody sees them, pages of no
    pool, requests that are not served."""
    x = _Cache(dt, [(40, 4), (0, 2), (9, 1)], 4, 2, 64, 16, seed=2, tail=2)
    none = torch.zeros_like(x.plan.masks)
    _check(x, _den(x, masks=none), masks=none, sees=np.zeros_like(x.sees))
    den = _den(x)
    den[0] = 0
    _check(x, den)
    # a key of NaN that one token sees: its own weight alone
    before, clean = x.pool.new_weights(), x.pool.new_weights()
    A.accumulate_cache_weights(x.q, x.kp, _den(x), x.plan, clean)
    den = _den(x)
    x.kp[x.tables[1][0], :, 1] = float("nan")
    A.accumulate_cache_weights(x.q, x.kp, den, x.plan, before, masks=none)
    assert torch.equal(before[1, :2], torch.zeros(2, device="cuda"))
    x.plan.pool.block_tables[0, 1] = 10 ** 6
    w = torch.full_like(clean, 3.0)
    A.accumulate_cache_weights(x.q, x.kp, den, x.plan, w)
    assert (w[0, 16:32] == 3).all() and torch.equal(w[0, :16] - 3, (clean[0, :16] + 3) - 3) and torch.isnan(w[1, 1])
    A.build_block_tables(x.plan, _i32([10 ** 6, 0, 9]), _i32([4, 0, 1]))
    w = torch.full_like(clean, 3.0)
    A.accumulate_cache_weights(x.q, x.kp, den, x.plan, w)
    assert (w[:2] == 3).all() and (w[2, 10:] == 3).all()


@pytest.mark.parametrize("dt", [BF16, F32])
def test_weights_of_many_requests(dt):
    """More requests than a workgroup counts at a time, most of them short, some without new tokens."""
    lens = [(r % 7, (r % 3 != 0) * 1) for r in range(2500)]
    lens[1200] = (150, 2)
    x = _Cache(dt, lens, 2, 1, 32, 8, seed=1, max_tree=0, parents=False)
    _check(x, _den(x))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_weights_over_other_strides(dt):
    """Pages as (pages, slots, heads, dim) in memory, q inside a wider buffer, weights in wider rows; and without the matrix cores or a
    workspace, through the C call."""
    import ctypes

    from algebraic_intelligence_amd import _lib
    x = _Cache(dt, [(100, 3), (0, 20), (300, 1)], 4, 2, 64, 16, seed=5)
    den = _den(x)
    want = A.accumulate_cache_weights(x.q, x.kp, den, x.plan, x.pool.new_weights())
    q = torch.zeros(x.q.shape[0], 8, 64, device="cuda", dtype=dt)
    q[:, 2:6] = x.q
    pages = x.kp.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(3, x.pool.max_len + 5, device="cuda")
    got = A.accumulate_cache_weights(q[:, 2:6], pages, den, x.plan, wide[:, :x.pool.max_len])
    assert torch.equal(got, want) and (wide[:, x.pool.max_len:] == 0).all()
    for flags in (0, _lib.FLAG_GENERIC):
        w = x.pool.new_weights()
        rc = _lib.lib().afa_paged_weights(x.plan._ref, x.q.data_ptr(), None, x.kp.data_ptr(), None, None, den.data_ptr(), w.data_ptr(),
                                          x.pool.max_len, flags, None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0 and (flags or torch.equal(w, want))
        given, bound = _given(x, den)
        _close(w, given, bound + 2 * U * given, flags)


def test_weights_repeat_on_streams_and_in_graphs():
    x = _Cache(BF16, [(100 + 70 * r, 1 + r % 3) for r in range(30)], 8, 2, 128, 16, seed=1, max_tree=0, parents=False)
    den = _den(x)
    want = A.accumulate_cache_weights(x.q, x.kp, den, x.plan, x.pool.new_weights())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = A.accumulate_cache_weights(x.q, x.kp, den, x.plan, x.pool.new_weights())
    side.synchronize()
    assert torch.equal(got, want)
    w = x.pool.new_weights()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.accumulate_cache_weights(x.q, x.kp, den, x.plan, w)
    for _ in range(4):
        x.q.normal_()
        w.zero_()
        graph.replay()
        want = A.accumulate_cache_weights(x.q, x.kp, den, x.plan, x.pool.new_weights())
        torch.cuda.synchronize()
        assert torch.equal(w, want)


# ------------------------------------------------------------------------------------- eviction
class _Held:
    """Requests that hold pages in random order, every place with a value of its own."""

    def __init__(self, dt, lens, K, D, page, seed=0, layout="plain", slack=1):
        rng = np.random.default_rng(seed)
        R, need = len(lens), [-(-c // page) for c in lens]
        self.lens, self.page, pages = lens, page, sum(need) + 2
        self.pool = A.PagePool(pages, page, R, max(max(lens), 1) + slack * page)
        order = rng.permutation(pages)
        self.tables = []
        for r, n in enumerate(need):
            self.tables.append(order[:n])
            self.pool.block_tables[r, :n] = _i32(order[:n])
            order = order[n:]
        self.pool.held.copy_(_i32(need))
        shape = (pages, K, page, D)
        if layout == "side":  # (pages, slots, k and v, heads, dim) in memory
            both = torch.tensor(rng.standard_normal((pages, page, 2, K, D)), device="cuda").to(dt)
            self.kp, self.vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
        elif layout == "gap":
            wide = torch.tensor(rng.standard_normal((2, pages, K, page, D + 3)), device="cuda").to(dt)
            self.kp, self.vp = wide[0, ..., 1:D + 1], wide[1, ..., 1:D + 1]
        else:
            self.kp, self.vp = (torch.tensor(rng.standard_normal(shape), device="cuda").to(dt) for _ in range(2))
        w = np.exp(2 * rng.standard_normal((R, self.pool.max_len))).astype(np.float32)
        w[rng.random(w.shape) < 0.2] = 0.0  # ties
        self.w = torch.tensor(w, device="cuda")

    def check(self, budget, first=0, recent=0, lens=None):
        lens = self.lens if lens is None else lens
        weights, want = self.w.cpu().numpy(), [t.clone() for t in (self.kp, self.vp)]
        left, out = np.zeros_like(weights), []
        for r, c in enumerate(lens):
            c = min(max(c, 0), len(self.tables[r]) * self.page)
            places = C.kept(weights[r], c, budget, first, recent)
            assert len(places) == min(c, budget)
            out.append(len(places))
            left[r, :len(places)] = weights[r, places]
            table = torch.tensor(np.asarray(self.tables[r], np.int64), device="cuda")
            frm, to = (torch.tensor(p, dtype=torch.int64, device="cuda") for p in (places, range(len(places))))
            for pages in want:
                pages[table[to // self.page], :, to % self.page] = pages[table[frm // self.page], :, frm % self.page]
        before = self.w.clone()
        got, kept = A.evict_from_cache(self.kp, self.vp, self.pool, self.w, _i32(lens), budget, first=first, recent=recent)
        assert got.tolist() == out and got.dtype == torch.int32
        np.testing.assert_array_equal(kept.cpu().numpy().view(np.uint32), left.view(np.uint32))
        for a, b in zip((self.kp, self.vp), want):
            assert torch.equal(a, b)
        assert torch.equal(self.w.view(torch.int32), before.view(torch.int32))


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("K,D,page,layout", [(2, 64, 16, "plain"), (1, 128, 64, "side"), (6, 48, 8, "plain"), (3, 7, 5, "plain"),
                                             (2, 40, 1, "gap"), (1, 2, 3, "side"), (4, 6, 16, "plain"), (1, 1, 4, "plain")])
def test_evict(dt, K, D, page, layout):
    """Requests longer than the budget, as long, shorter, and empty; rows of every alignment."""
    x = _Held(dt, [300, 40, 41, 39, 0, 1, 1500, 64, 1024, 1025], K, D, page, seed=D, layout=layout)
    x.check(40, 3, 10)


@pytest.mark.parametrize("budget,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (100, 100, 0), (100, 0, 100), (100, 37, 63),
                                                 (100, 0, 0), (1023, 4, 100), (2000, 1, 1), (2999, 0, 7), (10 ** 7, 5, 5)])
def test_evict_budgets(budget, first, recent):
    _Held(BF16, [3000, 2001, 999, 100, 101], 2, 32, 16, seed=budget % 1000).check(budget, first, recent)


@pytest.mark.parametrize("what", ["equal", "zero", "signs", "odd", "bits", "rising", "falling"])
def test_evict_weights(what):
    """Equal weights keep the lower places; -0 is 0; infinities and NaN have their order; weights that differ in their last bit."""
    x = _Held(F16, [2500, 700, 65], 1, 16, 32, seed=3)
    n = x.w.shape[1]
    rng = np.random.default_rng(0)
    at = torch.arange(n, device="cuda", dtype=torch.float32)
    if what == "equal":
        x.w.fill_(0.75)
    if what == "zero":
        x.w = torch.where(torch.tensor(rng.random(x.w.shape) < 0.5, device="cuda"), 0.0, -0.0).float()
    if what == "signs":
        x.w = torch.randn_like(x.w)
    if what == "odd":
        x.w = torch.tensor(rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, 1, -1, 1e-45, 3e38], np.float32), x.w.shape),
                           device="cuda")
    if what == "bits":
        x.w = (0x3f800000 + torch.randint(0, 300, x.w.shape, device="cuda", dtype=torch.int32)).view(torch.float32)
    if what == "rising":
        x.w = (at + 1).expand_as(x.w).contiguous()
    if what == "falling":
        x.w = (n - at).expand_as(x.w).contiguous()
    for budget, first, recent in ((64, 0, 0), (600, 5, 50), (7, 2, 3)):
        x.check(budget, first, recent)


@pytest.mark.parametrize("dt,K,D,page,layout", [(F32, 2, 256, 16, "plain"), (F64, 1, 512, 64, "side"), (BF16, 3, 1000, 5, "plain"),
                                                (F16, 1, 1024, 32, "gap"), (F64, 2, 3, 7, "gap")])
def test_evict_rows_in_many_chunks(dt, K, D, page, layout):
    """Rows so long that a request's are moved by many workgroups, whose places are each other's sources: tokens that stay
    spread evenly, at the end, at the front, and at random."""
    x = _Held(dt, [4000, 3999, 1500, 2100], K, D, page, seed=D, layout=layout)
    n = x.w.shape[1]
    at = torch.arange(n, device="cuda")
    for weights in ((at % 2).float(), (at >= 1000).float(), (at % 64 < 32).float(), torch.rand(n, device="cuda")):
        x.w = weights.expand_as(x.w).contiguous()
        x.check(1000, 1, 3)
    x.check(1999)


@pytest.mark.parametrize("budget,first,recent,weights", [(9000, 10, 500, "plain"), (9000, 0, 0, "equal"), (1, 0, 0, "plain"),
                                                         (20000, 12000, 8000, "plain"), (16385, 9000, 1, "odd"), (33000, 3, 8192, "zero"),
                                                         (8192, 0, 8192, "plain"), (24576, 0, 17, "bits")])
def test_evict_long(budget, first, recent, weights):
    """Caches of several workgroups a request, beside short ones and lengths on both sides of a workgroup's tokens."""
    x = _Held(BF16, [40000, 24576, 8192, 8193, 100, 0, 16384, 16385, 36000], 1, 16, 64, seed=budget % 100)
    rng = np.random.default_rng(1)
    if weights == "equal":
        x.w.fill_(0.75)
    if weights == "zero":
        x.w = torch.where(torch.tensor(rng.random(x.w.shape) < 0.9, device="cuda"), 0.0, x.w)
    if weights == "odd":
        x.w = torch.tensor(rng.choice(np.array([np.nan, np.inf, -np.inf, 1, -1, 1e-45, 3e38], np.float32), x.w.shape), device="cuda")
    if weights == "bits":
        x.w = (0x3f800000 + torch.randint(0, 3000, x.w.shape, device="cuda", dtype=torch.int32)).view(torch.float32)
    x.check(budget, first, recent)


def test_evict_odd_lengths():
    """Lengths below 0 and past what a request's pages hold; weights in a wider buffer; a page of no pool is let be."""
    x = _Held(BF16, [100, 33, 64, 20], 2, 64, 16, seed=1, slack=4)
    x.check(30, 2, 5, lens=[-5, 10 ** 9, 2 ** 31 - 1, -2 ** 31])
    wide = torch.randn(4, x.pool.max_len + 9, device="cuda")
    x.w = wide[:, 3:x.pool.max_len + 3]
    x.check(12, 0, 0)
    x = _Held(BF16, [100, 33], 2, 64, 16, seed=1)
    x.pool.block_tables[0, 2] = 10 ** 6
    k = x.kp.clone()
    lens, _ = A.evict_from_cache(x.kp, x.vp, x.pool, x.w, _i32([100, 33]), 50)
    assert lens.tolist() == [50, 33]
    lost = torch.tensor(np.asarray(x.tables[0][2:3], np.int64), device="cuda")
    assert torch.equal(x.kp[lost], k[lost])


@pytest.mark.parametrize("slack", [1, 2000])
def test_evict_captured_and_on_a_stream(slack):
    """One workgroup a request, and several where max_len is long."""
    x = _Held(BF16, [3000, 200, 1500], 2, 64, 16, seed=1, slack=slack)
    k0, v0 = x.kp.clone(), x.vp.clone()
    lens = _i32(x.lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A.evict_from_cache(x.kp, x.vp, x.pool, x.w, lens, 128, first=4, recent=16)
    for i in range(4):
        x.w.copy_(torch.rand_like(x.w))
        lens.copy_(_i32([3000 - 500 * i, 200 - 30 * i, 100 + i]))
        x.kp.copy_(k0), x.vp.copy_(v0)
        graph.replay()
        a = [t.clone() for t in (*got, x.kp, x.vp)]
        x.kp.copy_(k0), x.vp.copy_(v0)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            b = [*A.evict_from_cache(x.kp, x.vp, x.pool, x.w, lens, 128, first=4, recent=16), x.kp, x.vp]
        side.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_evict_in_the_librarys_own_workspace():
    from algebraic_intelligence_amd import _lib
    x = _Held(BF16, [300, 20, 100], 2, 64, 16, seed=1)
    k, v, lens = x.kp.clone(), x.vp.clone(), _i32(x.lens)
    want = A.evict_from_cache(k, v, x.pool, x.w, lens, 64, first=2, recent=8)
    got, left, p = torch.empty_like(lens), torch.empty_like(x.w), x.pool
    rc = _lib.lib().afa_paged_evict(_lib.AFA_BF16, p.num_pages, p.page_size, 3, p.block_tables.shape[1], 2, 64, p.block_tables.data_ptr(),
                                    p.held.data_ptr(), x.kp.data_ptr(), x.vp.data_ptr(), None, lens.data_ptr(), 64, 2, 8, x.w.data_ptr(),
                                    x.w.shape[1], left.data_ptr(), got.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(got, want[0]) and torch.equal(left, want[1])
    assert torch.equal(x.kp, k) and torch.equal(x.vp, v)


def test_evict_twice_and_at_once():
    """Two pools on two streams at a time; a layer cut back, filled on and cut back again."""
    xs = [_Held(F32, [3000, 2000, 2500], 2, 256, 16, seed=s) for s in (1, 2)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    kept = [(x.kp.clone(), x.vp.clone()) for x in xs]
    for round_ in range(3):
        got = []
        for x, s, (k, v) in zip(xs, sides, kept):
            x.kp.copy_(k), x.vp.copy_(v)
        torch.cuda.synchronize()
        for x, s in zip(xs, sides):
            with torch.cuda.stream(s):
                got.append(A.evict_from_cache(x.kp, x.vp, x.pool, x.w, _i32(x.lens), 700, first=3, recent=60))
        torch.cuda.synchronize()
        for x, (k, v), (lens, left) in zip(xs, kept, got):
            again_k, again_v = k.clone(), v.clone()
            a, b = A.evict_from_cache(again_k, again_v, x.pool, x.w, _i32(x.lens), 700, first=3, recent=60)
            assert torch.equal(a, lens) and torch.equal(b, left) and torch.equal(again_k, x.kp) and torch.equal(again_v, x.vp)
    x = xs[0]
    x.w = torch.rand_like(x.w)
    x.check(900, 5, 5)
    x.w = torch.rand_like(x.w)
    x.check(300, 5, 5, lens=[900, 900, 900])


def test_refusals():
    x = _Cache(BF16, [(5, 2)], 4, 2, 64, 16)
    w, den = x.pool.new_weights(), torch.ones(2, 4, device="cuda")
    acc = lambda q=x.q, k=x.kp, d=den, w=w, **kw: A.accumulate_cache_weights(q, k, d, x.plan, w, **kw)  # noqa: E731
    for kw in (dict(q=x.q[:1]), dict(k=x.kp[:1]), dict(d=den[:1]), dict(w=w[:, :5]), dict(w=torch.zeros(1, 2 * w.shape[1], device="cuda")[:, ::2]),
               dict(masks=torch.zeros(1, 1, device="cuda"))):
        with pytest.raises(ValueError):
            acc(**kw)
    for kw in (dict(q=x.q.float()), dict(d=den.double()), dict(w=w.double()), dict(k=x.kp.half())):
        with pytest.raises(TypeError):
            acc(**kw)
    with pytest.raises(RuntimeError, match="gradient"):
        acc(d=den.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="GPU"):
        acc(w=w.cpu())
    y = _Held(BF16, [50], 2, 64, 16)
    lens = _i32([50])
    ev = lambda k=y.kp, v=y.vp, w=y.w, lens=lens, budget=20, **kw: A.evict_from_cache(k, v, y.pool, w, lens, budget, **kw)  # noqa: E731
    near = torch.zeros(y.kp.numel() + 64, device="cuda", dtype=BF16)
    near = near[:-64].view(y.kp.shape), near[64:].view(y.kp.shape)
    for kw in (dict(k=y.kp[:1]), dict(v=y.vp[:, :1]), dict(v=y.kp), dict(w=y.w[:, :2]), dict(lens=_i32([1, 2])), dict(budget=0),
               dict(budget=-1), dict(budget=1.5), dict(first=21), dict(first=10, recent=11), dict(recent=-1),
               dict(k=y.kp.transpose(2, 3).contiguous().transpose(2, 3)), dict(v=y.kp[:1].expand_as(y.kp)),
               dict(k=near[0], v=near[1])):
        with pytest.raises(ValueError):
            ev(**kw)
    with pytest.raises(TypeError):
        ev(lens=lens.long())
    with pytest.raises(TypeError):
        ev(k=y.kp.int(), v=y.vp.int())
    with pytest.raises(RuntimeError, match="GPU"):
        ev(k=y.kp.cpu(), v=y.vp.cpu())
    with pytest.raises(RuntimeError, match="gradient"):
        ev(k=y.kp.clone().requires_grad_(True))


@pytest.mark.parametrize("dt", [BF16, F32])
def test_a_served_batch(dt):
    """Requests that share a prompt, with normalised heads, decoded token by token: appended, attended behind the prefix, their
    weights followed, and cut back whenever they pass the budget.  A float64 cache that keeps the tokens' rows as lists
    goes along; each step's output is checked against it, within the bounds of tests/test_prefix_gpu.py."""
    from tests.test_prefix_gpu import _half, _tiny, _weight_error
    R, H, K, D, L, page, budget = 3, 4, 2, 64, 45, 16, 24
    rng = np.random.default_rng(0)
    pool = A.PagePool(12, page, R, 64)
    plan = A.DraftPlan(pool, 8, heads=H, kv_heads=K, head_dim=D, dtype=dt, max_new=4, max_tree=0)
    kp, vp = _pages(pool, K, D, dt)
    tab = _tables(200, D)
    qs, ks = (torch.tensor(1 + 0.2 * rng.standard_normal(D), device="cuda").float() for _ in range(2))
    pk, pv = (torch.tensor(rng.standard_normal((K, L, D)), device="cuda").to(dt) for _ in range(2))
    weights, cached, seen = pool.new_weights(), _i32([0] * R), np.zeros(R, int)
    rows = [[] for _ in range(R)]
    evicted = 0
    for step in range(30):
        new = np.array([1 + (step + r) % 2 for r in range(R)])
        A.build_block_tables(plan, cached, _i32(new))
        assert (plan.status == 0).all()
        T = int(new.sum())
        q, k, v = (torch.tensor(rng.standard_normal((8, n, D)), device="cuda").to(dt) for n in (H, K, K))
        at = np.concatenate([L + seen[r] + np.arange(new[r]) for r in range(R)] + [np.zeros(8 - T, int)])
        q = A.append_to_cache(q, k, v, kp, vp, plan, tab, positions=_i32(at), norms=(qs, ks))
        out, den = A.paged_prefix_afa(q, pk, pv, kp, vp, plan, return_denominator=True)
        A.accumulate_cache_weights(q, kp, den, plan, weights)
        slots = plan.slots.long()
        starts = np.concatenate([[0], np.cumsum(new)])
        for r in range(R):
            at_r = slots[starts[r]:starts[r + 1]]
            rows[r] += list(zip(_f64(kp[at_r // page, :, at_r % page]), _f64(vp[at_r // page, :, at_r % page])))
            for i in range(new[r]):
                t, m = starts[r] + i, len(rows[r]) - new[r] + i + 1
                for h in range(H):
                    kh = h * K // H
                    keys = np.concatenate([_f64(pk)[kh], [a[kh] for a, _ in rows[r][:m]]])
                    values = np.concatenate([_f64(pv)[kh], [b[kh] for _, b in rows[r][:m]]])
                    want, wden, size, S = P.attention_row(_f64(q)[t, h], keys, values, 0.5)
                    e = _weight_error(dt, D, S, len(keys))
                    _close(out[t, h], want, 2 * e * size + (_half(dt) + 4 * U) * np.abs(want) + _tiny(dt), (step, r, h))
                    _close(den[t, h], np.asarray(wden), np.asarray(2 * e * wden), "denominator")
        seen += new
        cached = _i32([len(x) for x in rows])
        if step % 7 == 6:
            before = weights.cpu().numpy()
            cached, weights = A.evict_from_cache(kp, vp, pool, weights, cached, budget, first=2, recent=6)
            for r in range(R):
                keep = C.kept(before[r], len(rows[r]), budget, 2, 6)
                evicted += len(rows[r]) - len(keep)
                rows[r] = [rows[r][j] for j in keep]
            assert cached.tolist() == [len(x) for x in rows]
    assert evicted > 20
