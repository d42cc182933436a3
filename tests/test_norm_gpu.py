"""Norms of q and k with their rotation on the GPU, in training and in the cache write, against
oracle/cache_oracle.py (float64).

Tolerances, derived from the arithmetic and not from runs.  u = 2^-24 (fp64: 2^-53), h half a step of the result's type
relative to it, D the head dimension.  The mean of D squares is off by (D + 3) u of itself, so that the inverse
root r is by half of that and 3 u for its own steps, and a scaled element by e = ((D + 3) / 2 + 6) u (two products and the
scale's rounding to fp32).  The rotation adds 3 u of |c x0| + |s x1|, each already off by e: a result is within
(e + 3 u) (|c x0| + |s x1|) + h |y|.  In the backward, back is off by 2 u Bk, Bk = |c g0| + |s g1|.  With S = |w| Bk and
M = mean(S |xh|), dx = r (h - xh mean(h xh)) is off by at most (2.5 D + 30) u r (S + |xh| M) + h |dx|: the second
term has r, xh and the mean's r, e each, D u for its sum and a few roundings.  A scale's gradient sums N
rows: (N + D / 2 + 15) u sum Bk |xh|.
"""
import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from oracle import cache_oracle as C
from oracle import paged_oracle as P
from tests.test_paged_gpu import BF16, F16, F32, F64, _close, _f64, _half, _i32, _pages, _plan, _tables, _tiny

pytestmark = pytest.mark.gpu


def _u(dt):
    return 2.0 ** -53 if dt == F64 else 2.0 ** -24


def _size(x, c, s, at, sections, back=False):
    """|c x0| + |s x1| and |s x0| + |c x1| of every pair."""
    if c is None:
        return np.abs(x)
    with np.errstate(invalid="ignore"):
        even = P.rotate_axes(np.abs(x), np.abs(c), -np.abs(s), at, sections)
        odd = P.rotate_axes(np.abs(x), np.abs(c), np.abs(s), at, sections)
    even[..., 1::2] = odd[..., 1::2]
    return even


def _forward(x, w, eps, c, s, at, sections, dt):
    D, u = x.shape[-1], _u(dt)
    y = C.norm_rotate(x, w, eps, c, s, at, sections)
    size = _size(C.norm_rotate(x, w, eps, None, None, None, None), c, s, at, sections)
    return y, ((D + 3) / 2 + 9) * u * size + _half(dt) * np.abs(y) * (1 + D * u) + _tiny(dt)


def _backward(x, w, eps, g, c, s, at, sections, dt):
    D, u = x.shape[-1], _u(dt)
    dx, dw = C.norm_rotate_gradient(x, w, eps, g, c, s, at, sections)
    r = 1 / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    Bk = _size(g, c, s, at, sections, True)
    S, xh = np.abs(w) * Bk, np.abs(x) * r
    M = np.mean(S * xh, -1, keepdims=True)
    N = x.size // D
    return ((dx, (2.5 * D + 30) * u * r * (S + xh * M) + _half(dt) * np.abs(dx) * (1 + D * u) + _tiny(dt)),
            (dw, (N + D / 2 + 15) * u * np.sum(Bk * xh, axis=(0, 1, 2)) + 1e-40))


def _calc(dt):
    return F64 if dt == F64 else F32


def _layouts(arrays, layout, D, dt):
    if layout == "blhd":
        return [a.transpose(1, 2).contiguous().transpose(1, 2) for a in arrays]
    if layout == "gap":  # rows inside a wider buffer, at an odd element
        wide = [torch.zeros((*a.shape[:3], D + 5), dtype=dt, device="cuda") for a in arrays]
        return [w[..., 1:D + 1].copy_(a) for w, a in zip(wide, arrays)]
    return arrays


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("B,H,K,L,D,sections,long,layout,scale_dt", [
    (2, 4, 2, 19, 64, (8, 12, 12), True, "blhd", F32), (1, 1, 1, 1, 2, (1,), False, "bhld", F32),
    (3, 6, 6, 33, 48, (10, 14), True, "bhld", BF16), (1, 5, 3, 7, 10, (2, 1, 1, 1), False, "blhd", F32),
    (2, 3, 1, 65, 128, (16, 24, 24), False, "bhld", F16), (1, 2, 2, 40, 96, (20, 0, 11), True, "blhd", F64),
    (2, 2, 1, 5, 36, (3, 4), True, "gap", F32), (1, 9, 4, 130, 64, (32,), True, "shared", F32),
    (1, 3, 2, 6, 256, (128,), False, "blhd", F32), (2, 1, 5, 9, 512, (256,), False, "bhld", F32),
    (1, 2, 1, 3, 1000, None, False, "bhld", F32), (1, 3, 2, 11, 7, "none", False, "blhd", F32),
    (5, 2, 2, 1, 64, "rows", False, "bhld", F32), (2, 2, 3, 9, 8, (2, 2), True, "blhd", F32), (2, 3, 2, 300, 80, "rows", False, "blhd", F32),
])
def test_norm_rotation_and_gradients(dt, B, H, K, L, D, sections, long, layout, scale_dt):
    """Chunked and ragged rows, shared positions, a row's index for a position, no rotation at all."""
    rng = np.random.default_rng(B * 100 + D)
    rows, eps = 307, 1e-6
    tab = pos = at = c = s = None
    cuts = sections if isinstance(sections, tuple) else None
    if sections != "none":
        tab = _tables(rows, D, _calc(dt))
        c, s = _f64(tab[0]), _f64(tab[1])
        at = rng.integers(0, rows, (B, L, len(cuts) if cuts else 1))
        if layout == "shared":
            at[:] = at[:1]
        if sections == "rows":
            at[:] = np.arange(L)[None, :, None]
        else:
            pos = torch.tensor(at[0] if layout == "shared" else at, dtype=torch.int64 if long else torch.int32, device="cuda")
    oracle_cuts = cuts or (D // 2,)
    arrays = [torch.tensor(rng.standard_normal((B, n, L, D)) * rng.uniform(0.1, 5, (B, n, L, 1)), device="cuda").to(dt)
              for n in (H, K, H, K)]
    q, k, gq, gk = _layouts(arrays, layout, D, dt)
    qs, ks = (torch.tensor(1 + 0.3 * rng.standard_normal(D), device="cuda").to(scale_dt) for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (q, k, qs, ks)]
    y, z = A.apply_ago_norm_rotations(q, k, qs, ks, tab, pos, cuts, eps=eps)
    dq, dk, dqs, dks = torch.autograd.grad((y, z), leaves, (gq, gk))
    for x, w, g, out, dx, dw, name in ((q, qs, gq, y, dq, dqs, "q"), (k, ks, gk, z, dk, dks, "k")):
        w64 = _f64(w.detach().to(_calc(dt)))
        assert out.shape == x.shape and out.dtype == dt and dx.dtype == dt and dw.dtype == scale_dt
        _close(out, *_forward(_f64(x), w64, eps, c, s, at, oracle_cuts, dt), name)
        (wx, bx), (ww, bw) = _backward(_f64(x), w64, eps, _f64(g), c, s, at, oracle_cuts, dt)
        _close(dx, wx, bx, ("d" + name, layout))
        _close(dw, ww, bw + _half(scale_dt) * np.abs(ww), "d" + name + "_scale")
    # q alone, the same bits; one gradient of the two
    assert torch.equal(A.apply_ago_norm_rotations(q, None, qs, None, tab, pos, cuts, eps=eps), y)
    y, z = A.apply_ago_norm_rotations(q.detach(), k, qs.detach(), ks, tab, pos, cuts, eps=eps)
    assert not y.requires_grad and z.requires_grad
    again = torch.autograd.grad(z, (k, ks), gk)
    assert torch.equal(again[0], dk)
    _close(again[1], *(lambda p: (p[0], p[1] + _half(scale_dt) * np.abs(p[0])))(_backward(
        _f64(k), _f64(ks.detach().to(_calc(dt))), eps, _f64(gk), c, s, at, oracle_cuts, dt)[1]), "dk_scale alone")


def test_norm_by_differences():
    rng = np.random.default_rng(5)
    q, k = (torch.tensor(rng.standard_normal((2, n, 5, 12)), device="cuda", requires_grad=True) for n in (2, 1))
    qs, ks = (torch.tensor(1 + rng.standard_normal(12) / 4, device="cuda", requires_grad=True) for _ in range(2))
    tab, pos = _tables(9, 12, F64), torch.tensor(rng.integers(0, 9, (5, 2)), device="cuda")
    f = lambda q, k, qs, ks: A.apply_ago_norm_rotations(q, k, qs, ks, tab, pos, (2, 3), eps=1e-3)  # noqa: E731
    assert torch.autograd.gradcheck(f, (q, k, qs, ks))


def test_norm_sums_many_rows_the_same_way_each_time():
    """Scale gradients over more rows than workgroups: within their bound and the same bits each time."""
    B, H, K, L, D = 3, 8, 2, 1111, 64
    rng = np.random.default_rng(1)
    q, k, gq, gk = (torch.tensor(rng.standard_normal((B, n, L, D)), device="cuda").to(BF16) for n in (H, K, H, K))
    qs, ks = (torch.tensor(1 + 0.3 * rng.standard_normal(D), device="cuda").float() for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (q, k, qs, ks)]
    tab = _tables(L, D)
    got = [torch.autograd.grad(A.apply_ago_norm_rotations(*leaves, tab), leaves, (gq, gk)) for _ in range(3)]
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    at = np.broadcast_to(np.arange(L)[None, :, None], (B, L, 1))
    for x, w, g, dx, dw in ((q, qs, gq, got[0][0], got[0][2]), (k, ks, gk, got[0][1], got[0][3])):
        (wx, bx), (ww, bw) = _backward(_f64(x), _f64(w), 1e-6, _f64(g), _f64(tab[0]), _f64(tab[1]), at, (D // 2,), BF16)
        _close(dx, wx, bx, "dx")
        _close(dw, ww, bw, "dw")


@pytest.mark.parametrize("dt,B,H,K,L,D,layout", [(BF16, 5, 6, 3, 7001, 64, "blhd"), (F32, 1, 5, 2, 9501, 128, "bhld"),
                                                 (F16, 3, 7, 2, 2901, 48, "blhd"), (BF16, 2, 5, 5, 3601, 96, "bhld")])
def test_norm_of_many_rows(dt, B, H, K, L, D, layout):
    """Groups of heads with a ragged last one, and results larger than the caches."""
    rng = np.random.default_rng(L)
    q, k, gq, gk = _layouts([torch.tensor(rng.standard_normal((B, n, L, D), dtype=np.float32), device="cuda").to(dt)
                             for n in (H, K, H, K)], layout, D, dt)
    qs, ks = (torch.tensor(1 + 0.3 * rng.standard_normal(D), device="cuda").float() for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (q, k, qs, ks)]
    tab = _tables(L, D)
    y = A.apply_ago_norm_rotations(*leaves, tab)
    dx, dw = (g[2 * i:2 * i + 2] for g in [torch.autograd.grad(y, leaves, (gq, gk))] for i in range(2))
    c, s, at = _f64(tab[0]), _f64(tab[1]), np.broadcast_to(np.arange(L)[None, :, None], (B, L, 1))
    for i, (x, w, g) in enumerate(((q, qs, gq), (k, ks, gk))):
        _close(y[i], *_forward(_f64(x), _f64(w), 1e-6, c, s, at, (D // 2,), dt), i)
        (wx, bx), (ww, bw) = _backward(_f64(x), _f64(w), 1e-6, _f64(g), c, s, at, (D // 2,), dt)
        _close(dx[i], wx, bx, ("dx", i))
        _close(dw[i], ww, bw, ("dw", i))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_norm_edges(dt):
    """Rows of zeros with and without eps, infinities and NaN, positions outside the tables, empty tensors, expanded cotangents."""
    D = 16
    x = torch.randn(1, 2, 6, D, device="cuda").to(dt)
    x[0, 0, 0] = 0
    x[0, 0, 1, 3] = float("inf")
    x[0, 0, 2, 4] = float("nan")
    w = torch.ones(D, device="cuda")
    tab = _tables(6, D)
    pos = torch.tensor([[0], [1], [2], [3], [-1], [6]], device="cuda")
    y = A.apply_ago_norm_rotations(x, None, w, None, tab, pos)
    nan = torch.isnan(y)
    assert (y[0, 0, 0] == 0).all() and nan[0, 0, 2].all() and nan[0, :, 4:].all() and not nan[0, 1, :4].any()
    assert not nan[0, 0, 0].any() and not nan[0, 0, 3].any()
    assert nan[0, 0, 1, 2:4].all() and (y[0, 0, 1, 4:] == 0).all()  # infinity times 0, the others times 0
    # the same mathematics in torch, in fp32: no eps, a row of zeros is NaN
    z = A.apply_ago_norm_rotations(x, None, w, None, eps=0.0)
    assert torch.isnan(z[0, 0, 0]).all() and not torch.isnan(z[0, 1]).any()
    for shape in ((0, 2, 4, D), (1, 2, 0, D), (1, 0, 4, D)):
        e, ws = torch.zeros(shape, device="cuda", dtype=dt, requires_grad=True), w.clone().requires_grad_(True)
        out = A.apply_ago_norm_rotations(e, None, ws, None, tab)
        assert out.shape == shape and out.dtype == dt
        d, dw = torch.autograd.grad(out.sum(), (e, ws))
        assert d.shape == shape and (dw == 0).all()
    both = A.apply_ago_norm_rotations(x[:, 1:], x[:, :0], w, w, tab, pos[:, :1].clamp(0, 5))
    assert both[1].shape == (1, 0, 6, D)
    assert torch.equal(both[0], A.apply_ago_norm_rotations(x[:, 1:], None, w, None, tab, pos.clamp(0, 5)))
    xs = x[:, 1:, :4].clone().requires_grad_(True)
    a = torch.autograd.grad(A.apply_ago_norm_rotations(xs, None, w, None, tab).sum(), xs)[0]
    b = torch.autograd.grad(A.apply_ago_norm_rotations(xs, None, w, None, tab), xs, torch.ones_like(xs))[0]
    assert torch.equal(a, b)


def test_norm_on_a_stream_and_captured():
    """Forward and backward in one graph on a side stream, replayed with other activations and cotangents."""
    tab = _tables(200, 64)
    new = lambda: [torch.randn(2, n, 77, 64, device="cuda", dtype=BF16) for n in (6, 2)]  # noqa: E731
    scales = [1 + torch.randn(64, device="cuda") / 4 for _ in range(2)]
    x, g, pos = new(), new(), torch.randint(0, 200, (2, 77, 1), device="cuda")

    def run(x, w):
        leaves = [t.requires_grad_(True) for t in (*x, *w)]
        y = A.apply_ago_norm_rotations(*leaves, tab, pos)
        return [t.detach() for t in y], torch.autograd.grad(y, leaves, g)

    clones = lambda: ([t.clone() for t in x], [t.detach().clone() for t in scales])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*clones())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = run([t.view_as(t) for t in x], [t.view_as(t) for t in scales])
    for _ in range(4):
        for t, n in zip(x + g, new() + new()):
            t.copy_(n)
        pos.random_(0, 200)
        graph.replay()
        ey, ed = run(*clones())
        torch.cuda.synchronize()
        for got, want in zip([*y, *d], [*ey, *ed]):
            assert torch.equal(got, want)


# ---------------------------------------------------------------------------------- cache write
@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,D,page,axes,layout", [
    (4, 2, 64, 16, 1, "fused"), (2, 2, 128, 64, 3, "plain"), (6, 6, 48, 8, 2, "fused"), (3, 1, 10, 3, 1, "plain"),
    (4, 4, 32, 1, 4, "pages"), (8, 1, 96, 32, 0, "fused"), (2, 1, 7, 5, 0, "plain"), (1, 1, 256, 16, 1, "gap"),
])
def test_append_with_norms(dt, H, K, D, page, axes, layout):
    """Rows of every status, as the cache write without norms: served tokens, a request without pages, rows behind the last
    request; v goes in as it is, and places of no token stay as they were."""
    rng = np.random.default_rng(D + page)
    cached, new = np.array([3, 0, 17, 2, 900]), np.array([5, 1, 9, 0, 2])
    T = 22
    pool, oracle = A.PagePool(40, page, 5, 60), P.Pool(40, page, 5, 60)
    plan = _plan(pool, T, 9, 64, H, K, D, dt)
    parents = np.array([rng.integers(-1, 2) for _ in range(T)])
    A.build_block_tables(plan, _i32(cached), _i32(new), _i32(parents))
    slots, positions, *_ = oracle.step(cached, new, T, 9, 64, parents)
    flat = torch.tensor(rng.standard_normal((T, H + 2 * K, D)), device="cuda").to(dt)
    q, k, v = flat[:, :H], flat[:, H:H + K], flat[:, H + K:]
    if layout != "fused":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if layout == "gap":
        wide = torch.zeros((T, H, D + 3), dtype=dt, device="cuda")
        q = wide[..., 1:D + 1].copy_(q)
    kp, vp = _pages(pool, K, D, dt, 7.0)
    if layout == "pages":  # (pages, slots, heads, dim) in memory, keys and values side by side
        both = torch.full((40, page, 2, K, D), 7.0, dtype=dt, device="cuda")
        kp, vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    qs, ks = (torch.tensor(1 + 0.3 * rng.standard_normal(D), device="cuda").to(_calc(dt)) for _ in range(2))
    rows, kw, rotary, c, s, at, sections = 64, {}, None, None, None, positions[:, None], None
    if axes:
        rotary = _tables(rows, D, _calc(dt))
        c, s = _f64(rotary[0]), _f64(rotary[1])
        sections = {1: (D // 2,), 2: (4, D // 2 - 4), 3: (16, 24, 24), 4: (4, 4, 4, 3)}[axes]
        if axes > 1:
            at = np.concatenate((at, rng.integers(0, rows, (T, axes - 1))), 1)
            kw = {"positions": _i32(at), "sections": sections}
    out = A.append_to_cache(q, k, v, kp, vp, plan, rotary, norms=(qs, ks), eps=1e-5, **kw)
    f = lambda x, w: _forward(_f64(x).transpose(1, 0, 2)[None], _f64(w), 1e-5, c, s, at[None], sections, dt)  # noqa: E731
    y, bound = f(q, qs)
    _close(out.transpose(0, 1)[None], y, bound, "q")
    yk, bk = f(k, ks)
    want_k, bound_k, want_v = np.full((40, K, page, D), 7.0), np.zeros((40, K, page, D)), np.full((40, K, page, D), 7.0)
    for t, slot in enumerate(slots):
        if slot >= 0:
            want_k[slot // page, :, slot % page], bound_k[slot // page, :, slot % page] = yk[0, :, t], bk[0, :, t]
            want_v[slot // page, :, slot % page] = _f64(v)[t]
    _close(kp, want_k, bound_k, "k")
    assert (_f64(vp) == want_v).all()


def test_append_with_norms_is_the_training_call():
    """Many tokens, the same bits as apply_ago_norm_rotations gives: serving meets what training made."""
    T, H, K, D = 700, 8, 2, 128
    pool = A.PagePool(100, 16, 2, 800)
    plan = _plan(pool, T, T, 0, H, K, D, BF16)
    A.build_block_tables(plan, _i32([3, 0]), _i32([400, 300]))
    q, k, v = (torch.randn(T, n, D, device="cuda", dtype=BF16) for n in (H, K, K))
    qs, ks = (1 + torch.randn(D, device="cuda") / 4 for _ in range(2))
    kp, vp = _pages(pool, K, D, BF16)
    tab = _tables(800, D)
    out = A.append_to_cache(q, k, v, kp, vp, plan, tab, norms=(qs, ks))
    y, z = A.apply_ago_norm_rotations(q.transpose(0, 1)[None], k.transpose(0, 1)[None], qs, ks, tab, plan.positions[None, :, None])
    assert torch.equal(out, y[0].transpose(0, 1))
    slots = plan.slots.long()
    assert torch.equal(kp[slots // 16, :, slots % 16], z[0].transpose(0, 1))
    assert torch.equal(vp[slots // 16, :, slots % 16], v)


def test_append_with_norms_of_many_tokens_is_the_training_call():
    """Groups of heads, the same bits as apply_ago_norm_rotations gives: serving meets what training made."""
    T, H, K, D = 3300, 6, 2, 128
    pool = A.PagePool(220, 16, 2, 2100)
    plan = _plan(pool, T, T, 0, H, K, D, BF16)
    A.build_block_tables(plan, _i32([3, 0]), _i32([2000, 1300]))
    q, k, v = (torch.randn(T, n, D, device="cuda", dtype=BF16) for n in (H, K, K))
    qs, ks = (1 + torch.randn(D, device="cuda") / 4 for _ in range(2))
    kp, vp = _pages(pool, K, D, BF16)
    tab = _tables(2100, D)
    out = A.append_to_cache(q, k, v, kp, vp, plan, tab, norms=(qs, ks))
    y, z = A.apply_ago_norm_rotations(q.transpose(0, 1)[None], k.transpose(0, 1)[None], qs, ks, tab, plan.positions[None, :, None])
    assert torch.equal(out, y[0].transpose(0, 1))
    slots = plan.slots.long()
    assert torch.equal(kp[slots // 16, :, slots % 16], z[0].transpose(0, 1))
    assert torch.equal(vp[slots // 16, :, slots % 16], v)


def test_norm_refusals():
    q, w = torch.zeros(1, 2, 3, 64, device="cuda", dtype=BF16), torch.ones(64, device="cuda")
    tab = _tables(20, 64)
    for args in ((q[0], None, w, None), (q, q[:, :, :2], w, w), (q, None, w, w), (q, q, w, None), (q, None, w[:32], None)):
        with pytest.raises(ValueError):
            A.apply_ago_norm_rotations(*args, tab)
    with pytest.raises(TypeError):
        A.apply_ago_norm_rotations(q, q.float(), w, w, tab)
    with pytest.raises(TypeError, match="q_scale"):
        A.apply_ago_norm_rotations(q, None, w.long(), None, tab)
    with pytest.raises(RuntimeError, match="GPU"):
        A.apply_ago_norm_rotations(q, None, w.cpu(), None, tab)
    with pytest.raises(RuntimeError, match="GPU"):
        A.apply_ago_norm_rotations(q.cpu(), None, w, None, tab)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            A.apply_ago_norm_rotations(q, None, w, None, tab, eps=eps)
    with pytest.raises(ValueError, match="rotary"):
        A.apply_ago_norm_rotations(q, None, w, None, None, torch.zeros(3, 1, device="cuda", dtype=torch.int64))
    with pytest.raises(ValueError, match="even"):
        A.apply_ago_norm_rotations(q[..., :7], None, w[:7], None, tab)
    with pytest.raises(ValueError, match="positions"):
        A.apply_ago_norm_rotations(q, None, w, None, tab, torch.zeros(4, 1, device="cuda", dtype=torch.int64))
    leaf = q.clone().requires_grad_(True)
    d, = torch.autograd.grad(A.apply_ago_norm_rotations(leaf, None, w, None, tab).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.float().sum(), leaf)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q.float(), torch.ones_like(q.float()))
        with pytest.raises((RuntimeError, NotImplementedError)):
            A.apply_ago_norm_rotations(dual, None, w, None, tab)
    pool = A.PagePool(8, 16, 2, 64)
    plan = _plan(pool, 10, heads=4, kv_heads=2)
    q, k = torch.zeros(10, 4, 64, device="cuda", dtype=BF16), torch.zeros(10, 2, 64, device="cuda", dtype=BF16)
    kp, vp = _pages(pool, 2, 64, BF16)
    with pytest.raises(TypeError, match="norms"):
        A.append_to_cache(q, k, k, kp, vp, plan, tab, norms=w)
    with pytest.raises(ValueError, match="k_scale"):
        A.append_to_cache(q, k, k, kp, vp, plan, tab, norms=(w, w[:2]))
    with pytest.raises(ValueError, match="eps"):
        A.append_to_cache(q, k, k, kp, vp, plan, tab, norms=(w, w), eps=-1)
    with pytest.raises(RuntimeError, match="gradient"):
        A.append_to_cache(q, k, k, kp, vp, plan, tab, norms=(w.clone().requires_grad_(True), w))


def test_norm_changed_positions_are_noticed():
    """Positions changed between the two passes are an error, not another gradient."""
    q, w = torch.randn(1, 2, 3, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda")
    pos = torch.zeros(3, 1, device="cuda", dtype=torch.int64)
    y = A.apply_ago_norm_rotations(q, None, w, None, _tables(20, 64), pos)
    pos += 1
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_norm_in_the_librarys_own_workspace():
    """The C call without a workspace: the same bits."""
    from algebraic_intelligence_amd import _lib
    B, H, L, D = 2, 4, 50, 64
    q, g = (torch.randn(B, H, L, D, device="cuda", dtype=BF16) for _ in range(2))
    w = 1 + torch.randn(D, device="cuda") / 4
    leaf, scale = q.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = torch.autograd.grad(A.apply_ago_norm_rotations(leaf, None, scale, None), (leaf, scale), g)
    dq, dw = torch.empty_like(q), torch.empty_like(w)
    rc = _lib.lib().ago_norm_rotate_axes_bwd(_lib.AFA_BF16, B, H, 0, L, D, q.data_ptr(), None, g.data_ptr(), None, dq.data_ptr(), None,
                                             None, w.data_ptr(), None, dw.data_ptr(), None, 1e-6, None, None, 0, None, 4, 0, 1, None,
                                             None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(dq, want[0]) and torch.equal(dw, want[1])
