"""The serving operators on the GPU against oracle/paged_oracle.py (float64, token by token): plans over
long random lives of a pool, positions of several axes with their gradients, the cache write, the
attention of drafted trees over pages whose unused places hold NaN, and whole steps, captured too.

Tolerances, derived from the arithmetic and not from runs.  u = 2^-24 is half a step of fp32, h(t) half a
step of the result's type relative to it, and a smallest result may be off by half a smallest
subnormal.  A rotated element is two products and a sum in fp32 and one rounding: off by at most
2 u (|c x0| + |s x1|) + h(t) |y|.  A score is D products summed in fp32 and a scaling: off by
(D + 4) u S, S = max_j sum_d |q_d k_jd| / sqrt(D).  rho(s)^8 turns an error ds of s into a relative one
of 8 ds; its own evaluation has at most 6 roundings or hardware approximations of 1 ulp (2 u) in
rho, multiplied by 8 by the squarings, which add 7 u, and 2 u for a reciprocal: 105 u.  The branch-free
form, taken for scores above -8 only, is off by at most 16 * 8^2 * 2.1e-7 = 2.2e-4 on bf16 and fp16
inputs.  Weights enter the product with v in two planes of the type, off by h(t)^2 each, and fp16 ones
scaled so that a row's largest is at least 1, those below the subnormals by 2^-25 of it.  Sums over
N keys add N u.  So out is off by at most e A + h(t) |out| and the denominator by e of itself,
A = sum_j w_j |v_j| / den, with e the sum of these.
"""
import ctypes

import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from oracle import afa_oracle as O
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
U = 2.0 ** -24


def _f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _half(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def _weight_error(dt, D, S, n):
    if dt == F64:
        return (8 * (D + 4) * S + 200 + n) * 2.0 ** -53
    e = (8 * (D + 4) * S + 105 + n) * U
    if dt != F32:
        e += 2.2e-4 + _half(dt) ** 2
    return e + (n * 2.0 ** -25 if dt == F16 else 0)


# --------------------------------------------------------------------------------------- plans
def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _plan(pool, T, max_new=None, max_tree=64, heads=2, kv_heads=1, head_dim=64, dtype=BF16):
    return A.DraftPlan(pool, T, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, max_new=max_new,
                       max_tree=max_tree)


def _same_plan(plan, want, max_tree):
    slots, positions, requests, starts, sees, status = want
    np.testing.assert_array_equal(plan.status.cpu().numpy(), status)
    np.testing.assert_array_equal(plan.starts.cpu().numpy(), starts)
    np.testing.assert_array_equal(plan.requests.cpu().numpy(), requests)
    np.testing.assert_array_equal(plan.slots.cpu().numpy(), slots)
    np.testing.assert_array_equal(plan.positions.cpu().numpy(), positions)
    if max_tree:
        np.testing.assert_array_equal(plan.masks.cpu().numpy(), P.mask_words(sees))


def _same_pool(pool, oracle):
    width = pool.block_tables.shape[1]
    table = np.array([t + [-1] * (width - len(t)) for t in oracle.tables])
    np.testing.assert_array_equal(pool.block_tables.cpu().numpy(), table)
    np.testing.assert_array_equal(pool.held.cpu().numpy(), [len(t) for t in oracle.tables])
    head, count = pool.ring_state.tolist()
    ring = pool.ring.cpu().numpy()
    assert count == len(oracle.free)
    np.testing.assert_array_equal(ring[(head + np.arange(count)) % len(ring)], oracle.free)


@pytest.mark.parametrize("pages,page,R,max_len,T,max_new,max_tree,tree", [
    (64, 16, 5, 300, 90, 40, 64, True), (30, 1, 3, 40, 30, 20, 64, True), (200, 3, 40, 50, 300, 12, 0, False),
    (4000, 8, 1500, 60, 5000, 9, 128, True), (2500, 4, 1024, 30, 2000, 4, 64, False),
    (300, 64, 2, 12000, 9000, 5000, 256, True), (400, 512, 40, 100000, 150000, 100000, 64, True), (1, 7, 1, 7, 7, 7, 64, True), (60, 32, 33, 100, 64, 64, 192, True),
])
def test_plans_over_a_pools_life(pages, page, R, max_len, T, max_new, max_tree, tree):
    """Random steps, among them ones that no request, some or all can be served in: lengths and
    counts past every limit, negative ones, empty requests, trees with wrong parents."""
    rng = np.random.default_rng(pages + R)
    pool, oracle = A.PagePool(pages, page, R, max_len), P.Pool(pages, page, R, max_len)
    plan = _plan(pool, T, max_new, max_tree)
    for step in range(8):
        most = max(1, min(max_new, 2 * T // R, 5000))
        cached, new = rng.integers(0, max_len, R), rng.integers(0, most + 1, R)
        if step % 2:
            cached = np.minimum(cached, 2 * pages * page // R // (step + 1))
        if step in (2, 5):
            odd = rng.integers(0, R, max(1, R // 8))
            cached[odd] = rng.choice([-1, 0, max_len, 2 ** 31 - 1], len(odd))
            new[odd] = rng.choice([-3, 0, max_new, max_new + 1, 2 ** 31 - 1 if step == 5 else 1], len(odd))
        if step == 6:
            cached[:], new[:] = 0, 0
        parents = rng.integers(-2, max(2, most), T) if tree and step != 3 else None
        A.build_block_tables(plan, _i32(cached), _i32(new), None if parents is None else _i32(parents))
        want = oracle.step(cached, new, T, max_new, max_tree, parents)
        _same_plan(plan, want, max_tree)
        _same_pool(pool, oracle)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 128, 200, 255, 256])
def test_tree_shapes(n):
    """Chains, stars, combs and random trees of every size of a mask's words."""
    rng = np.random.default_rng(n)
    chain = np.arange(n) - 1
    comb = np.where(np.arange(n) % 2 == 1, chain, np.maximum(chain - 1, -1))
    shapes = [chain, np.full(n, -1), np.minimum(chain, 0), comb, np.array([rng.integers(-1, i) if i else -1 for i in range(n)])]
    T = n * len(shapes)
    pool, oracle = A.PagePool(200, 16, len(shapes), 400), P.Pool(200, 16, len(shapes), 400)
    plan = _plan(pool, T, n, 256)
    cached, new, parents = np.arange(len(shapes)) * 7, np.full(len(shapes), n), np.concatenate(shapes)
    A.build_block_tables(plan, _i32(cached), _i32(new), _i32(parents))
    _same_plan(plan, oracle.step(cached, new, T, n, 256, parents), 256)


def test_build_refusals():
    pool = A.PagePool(8, 16, 2, 64)
    plan = _plan(pool, 10)
    two, tokens = _i32([0, 0]), _i32([0] * 10)
    with pytest.raises(TypeError, match="int32"):
        A.build_block_tables(plan, two.long(), two)
    with pytest.raises(ValueError, match="shape"):
        A.build_block_tables(plan, two, tokens)
    with pytest.raises(ValueError, match="parents"):
        A.build_block_tables(plan, two, two, two)
    with pytest.raises(RuntimeError, match="GPU"):
        A.build_block_tables(plan, two.cpu(), two)
    with pytest.raises(ValueError, match="max_tree"):
        A.build_block_tables(_plan(pool, 10, max_tree=0), two, two, tokens)


# ------------------------------------------------------------------------------------ rotations
def _tables(rows, D, dtype=F32):
    r = A.build_cayley_rotary_matrix(D, rows, dtype=dtype)
    return r.c, r.s


def _rotation_bound(x, c, s, at, sections, dt, back=False):
    y = P.rotate_axes(x, c, s, at, sections, back)
    size = P.rotate_axes(np.abs(x), np.abs(c), -np.abs(s), at, sections)
    size[..., 1::2] = P.rotate_axes(np.abs(x), np.abs(c), np.abs(s), at, sections)[..., 1::2]
    u = 2.0 ** -53 if dt == F64 else U
    return y, 2 * u * np.abs(size) + (0 if dt in (F32, F64) else _half(dt)) * np.abs(y) * (1 + 4 * u) + _tiny(dt)


def _close(got, want, bound, what):
    got = _f64(got)
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), what
    off = np.abs(got - want)[~nan] - bound[~nan]
    assert off.size == 0 or off.max() <= 0, (what, float(off.max()))


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("B,H,K,L,D,sections,long,layout", [
    (2, 4, 2, 19, 64, (8, 12, 12), True, "blhd"), (1, 1, 1, 1, 2, (1,), False, "bhld"),
    (3, 6, 6, 33, 48, (10, 14), True, "bhld"), (1, 5, 3, 7, 10, (2, 1, 1, 1), False, "blhd"),
    (2, 3, 1, 65, 128, (16, 24, 24), False, "bhld"), (1, 2, 2, 40, 96, (20, 0, 11), True, "blhd"),
    (2, 2, 1, 5, 36, (3, 4), True, "gap"), (1, 9, 4, 130, 64, (32,), True, "shared"),
])
def test_axis_rotation_and_gradient(dt, B, H, K, L, D, sections, long, layout):
    rng = np.random.default_rng(B * 100 + D)
    rows = 37
    tab = _tables(rows, D, F64 if dt == F64 else F32)
    c, s = _f64(tab[0]), _f64(tab[1])
    at = rng.integers(0, rows, (B, L, len(sections)))
    if layout == "shared":
        at[:] = at[:1]
    pos = torch.tensor(at[0] if layout == "shared" else at, dtype=torch.int64 if long else torch.int32, device="cuda")
    arrays = [torch.tensor(rng.standard_normal((B, n, L, D)), device="cuda").to(dt) for n in (H, K, H, K)]
    if layout == "blhd":
        arrays = [a.transpose(1, 2).contiguous().transpose(1, 2) for a in arrays]
    if layout == "gap":  # rows inside a wider buffer, at an odd element
        wide = [torch.zeros((*a.shape[:3], D + 5), dtype=dt, device="cuda") for a in arrays]
        arrays = [w[..., 1:D + 1].copy_(a) for w, a in zip(wide, arrays)]
    q, k, gq, gk = arrays
    q.requires_grad_(True)
    k.requires_grad_(True)
    yq, yk = A.apply_ago_axis_rotations(q, k, tab, pos, sections)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for got, x, back in ((yq, q, False), (yk, k, False), (dq, gq, True), (dk, gk, True)):
        assert got.shape == x.shape and got.dtype == dt
        _close(got, *_rotation_bound(_f64(x), c, s, at, sections, dt, back), (layout, back))
    # q alone, and one gradient of the two
    assert torch.equal(A.apply_ago_axis_rotations(q, None, tab, pos, sections), yq)
    yq, yk = A.apply_ago_axis_rotations(q.detach(), k, tab, pos, sections)
    assert not yq.requires_grad and torch.equal(torch.autograd.grad(yk, k, gk)[0], dk)


def test_axis_rotation_by_differences():
    rng = np.random.default_rng(5)
    q, k = (torch.tensor(rng.standard_normal((2, n, 5, 12)), device="cuda", requires_grad=True) for n in (2, 1))
    tab, pos = _tables(9, 12, F64), torch.tensor(rng.integers(0, 9, (5, 2)), device="cuda")
    f = lambda q, k: A.apply_ago_axis_rotations(q, k, tab, pos, (2, 3))  # noqa: E731
    assert torch.autograd.gradcheck(f, (q, k))
    assert torch.autograd.gradgradcheck(f, (q, k))


def test_axis_rotation_of_one_axis_is_the_rotation():
    """Positions 0, 1, ... of one axis: the values of apply_ago_rotations in fp32, bit for bit."""
    q, k = torch.randn(2, 2, 3, 50, 64, device="cuda")
    rot = A.build_cayley_rotary_matrix(64, 50)
    want = A.apply_ago_rotations(q, k, rot, seq_axis=2)
    got = A.apply_ago_axis_rotations(q, k, rot, torch.arange(50, device="cuda")[:, None])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_axis_rotation_edges():
    """Positions outside the tables give NaN in their pairs only, pairs behind the sections keep
    every value, NaN and infinities included; empty tensors; tables of another type."""
    q = torch.randn(1, 2, 4, 16, device="cuda")
    q[..., 8:] = float("inf")
    q[0, 0, 0, 9] = float("nan")
    tab = _tables(6, 16)
    pos = torch.tensor([[0, 5], [-1, 2], [3, 6], [2 ** 31 + 1, -2 ** 40]], device="cuda")
    y = A.apply_ago_axis_rotations(q, None, tab, pos, (2, 2))
    assert torch.equal(y[..., 8:].nan_to_num(7.0), q[..., 8:].nan_to_num(7.0))
    nan = torch.isnan(y[0, 0, :, :8]).cpu().numpy()
    want = np.zeros((4, 8), bool)
    want[1, :4], want[2, 4:], want[3] = True, True, True
    np.testing.assert_array_equal(nan, want)
    for shape in ((0, 2, 4, 16), (1, 2, 0, 16), (1, 0, 4, 16)):
        e = torch.zeros(shape, device="cuda")
        at = torch.zeros(shape[2], 2, dtype=torch.int64, device="cuda")
        assert A.apply_ago_axis_rotations(e, None, tab, at, (2, 2)).shape == shape
    both = A.apply_ago_axis_rotations(q, q[:, :0], tab, pos, (2, 2))
    assert both[1].shape == (1, 0, 4, 16) and torch.equal(both[0].nan_to_num(7.0), y.nan_to_num(7.0))
    low = tuple(t.bfloat16() for t in tab)
    z = A.apply_ago_axis_rotations(q, None, low, pos, (2, 2))
    assert torch.equal(z.nan_to_num(7.0), A.apply_ago_axis_rotations(q, None, tuple(t.float() for t in low), pos, (2, 2)).nan_to_num(7.0))


def test_axis_rotation_on_a_stream():
    q = torch.randn(4, 8, 500, 64, device="cuda", dtype=BF16)
    tab, pos = _tables(40, 64), torch.randint(0, 40, (4, 500, 3), device="cuda")
    want = A.apply_ago_axis_rotations(q, None, tab, pos, (8, 12, 12))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = A.apply_ago_axis_rotations(q, None, tab, pos, (8, 12, 12))
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_axis_rotation_and_gradient():
    """Forward and backward in one graph, replayed with other activations, positions and cotangents;
    the eager calls use leaves of their own, so that no eager graph of the captured ones lives."""
    tab, cuts = _tables(40, 64), (8, 12, 12)
    new = lambda: [torch.randn(2, n, 77, 64, device="cuda", dtype=BF16) for n in (6, 2)]  # noqa: E731
    x, g, pos = new(), new(), torch.randint(0, 40, (2, 77, 3), device="cuda")

    def run(x):
        leaves = [t.requires_grad_(True) for t in x]
        y = A.apply_ago_axis_rotations(*leaves, tab, pos, cuts)
        return [t.detach() for t in y], torch.autograd.grad(y, leaves, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run([t.clone() for t in x])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = run([t.view_as(t) for t in x])
    for _ in range(5):
        for t, n in zip(x + g, new() + new()):
            t.copy_(n)
        pos.random_(0, 40)
        graph.replay()
        ey, ed = run([t.clone() for t in x])
        torch.cuda.synchronize()
        for got, want in zip([*y, *d], [*ey, *ed]):
            assert torch.equal(got, want)


# ---------------------------------------------------------------------------------- cache write
def _pages(pool, K, D, dt, fill=0.0):
    return tuple(torch.full_like(t, fill) for t in pool.new_pages(K, D, dt))


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,D,page,axes,layout", [
    (4, 2, 64, 16, 1, "fused"), (2, 2, 128, 64, 3, "plain"), (6, 6, 48, 8, 2, "fused"), (3, 1, 10, 3, 1, "plain"),
    (4, 4, 32, 1, 4, "pages"), (8, 1, 96, 32, 0, "fused"), (2, 1, 7, 5, 0, "plain"), (1, 1, 256, 16, 1, "gap"),
])
def test_append(dt, H, K, D, page, axes, layout):
    """Rows of every status: served tokens, a request without pages, rows behind the last request."""
    rng = np.random.default_rng(D + page)
    cached, new = np.array([3, 0, 17, 2, 900]), np.array([5, 1, 9, 0, 2])
    T = 22
    pool, oracle = A.PagePool(40, page, 5, 60), P.Pool(40, page, 5, 60)
    plan = _plan(pool, T, 9, 64, H, K, D, dt)
    parents = np.array([rng.integers(-1, 2) for _ in range(T)])
    A.build_block_tables(plan, _i32(cached), _i32(new), _i32(parents))
    slots, positions, *_ = oracle.step(cached, new, T, 9, 64, parents)
    assert (slots[-7:] == -1).all() and (slots[:15] >= 0).all()
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
    rows, kw, rotary = 64, {}, None
    sections = {0: None, 1: (D // 2,), 2: (4, D // 2 - 4), 3: (16, 24, 24), 4: (4, 4, 4, 3)}[axes]
    if axes:
        rotary = _tables(rows, D, F64 if dt == F64 else F32)
        at = positions[:, None]
        if axes > 1:
            at = np.concatenate((at, rng.integers(0, rows, (T, axes - 1))), 1)
            kw = {"positions": _i32(at), "sections": sections}
    out = A.append_to_cache(q, k, v, kp, vp, plan, rotary, **kw)
    turn = (lambda x: _rotation_bound(_f64(x).transpose(1, 0, 2)[None], _f64(rotary[0]), _f64(rotary[1]), at[None], sections,
                                      dt)) if axes else (lambda x: (_f64(x).transpose(1, 0, 2)[None], np.zeros((1, x.shape[1], T, D))))
    y, bound = turn(q)
    _close(out.transpose(0, 1)[None], y, bound, "q")
    (yk, bk), (yv, bv) = turn(k), (_f64(v).transpose(1, 0, 2)[None], None)
    want_k, bound_k, want_v = np.full((40, K, page, D), 7.0), np.zeros((40, K, page, D)), np.full((40, K, page, D), 7.0)
    for t, slot in enumerate(slots):
        if slot >= 0:
            want_k[slot // page, :, slot % page], bound_k[slot // page, :, slot % page] = yk[0, :, t], bk[0, :, t]
            want_v[slot // page, :, slot % page] = yv[0, :, t]
    _close(kp, want_k, bound_k, "k")
    assert (_f64(vp) == want_v).all()


def test_append_refusals():
    pool = A.PagePool(8, 16, 2, 64)
    plan = _plan(pool, 10, heads=4, kv_heads=2)
    q, k = torch.zeros(10, 4, 64, device="cuda", dtype=BF16), torch.zeros(10, 2, 64, device="cuda", dtype=BF16)
    kp, vp = _pages(pool, 2, 64, BF16)
    tab = _tables(20, 64)
    for args in ((q[:9], k, k, kp, vp), (q, q, k, kp, vp), (q, k, k[..., :32], kp, vp), (q, k, k, kp[:4], vp),
                 (q, k, k, kp, vp.transpose(2, 3))):
        with pytest.raises(ValueError):
            A.append_to_cache(*args, plan, tab)
    with pytest.raises(TypeError):
        A.append_to_cache(q.float(), k, k, kp, vp, plan, tab)
    with pytest.raises(TypeError):
        A.append_to_cache(q, k, k, kp.half(), vp, plan, tab)
    with pytest.raises(RuntimeError, match="GPU"):
        A.append_to_cache(q.cpu(), k, k, kp, vp, plan, tab)
    with pytest.raises(ValueError, match="rotary"):
        A.append_to_cache(q, k, k, kp, vp, plan, None, positions=_i32([0] * 10))
    with pytest.raises(ValueError, match="sections"):
        A.append_to_cache(q, k, k, kp, vp, plan, tab, positions=_i32([[0, 0]] * 10))
    with pytest.raises(TypeError, match="int32"):
        A.append_to_cache(q, k, k, kp, vp, plan, tab, positions=torch.zeros(10, dtype=torch.int64, device="cuda"))


# ------------------------------------------------------------------------------------ attention
class _Cache:
    """A step over random keys and values: every place of the pages that holds none is NaN."""

    def __init__(self, dt, lens, H, K, D, page, max_tree=64, seed=0, scale=1.0, tail=0, parents=True, max_new=None, far=0):
        rng = np.random.default_rng(seed)
        self.dt, self.H, self.K, self.D = dt, H, K, D
        self.lens, R = lens, len(lens)
        T = sum(n for _, n in lens) + tail
        longest = max(c + n for c, n in lens)
        pages = sum(-(-(c + n) // page) for c, n in lens) + 3
        self.pool = A.PagePool(pages + far, page, R, longest + page)
        order = rng.permutation(pages) + far
        if far == 0:
            self.pool.ring.copy_(_i32(order))
        else:
            self.pool.ring[:pages].copy_(_i32(order))
            self.pool.ring_state.copy_(_i32([0, pages]))
        self.plan = _plan(self.pool, T, max_new or max(1, max(n for _, n in lens)), max_tree, H, K, D, dt)
        tree = None
        if parents and max_tree:
            tree = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for _, n in lens]
                                  + [np.full(tail, -1)]).astype(np.int32)
            tree = np.concatenate((tree, np.full(T - len(tree), -1))).astype(np.int32)
        A.build_block_tables(self.plan, _i32([c for c, _ in lens]), _i32([n for _, n in lens]),
                             None if tree is None else _i32(tree))
        oracle = P.Pool(pages + far, page, R, longest + page)
        oracle.free = list(order)
        *_, starts, sees, status = oracle.step([c for c, _ in lens], [n for _, n in lens], T, T, max_tree, tree)
        assert (status == 0).all()
        self.starts, self.sees, self.tables = starts, sees, oracle.tables
        self.kp, self.vp = _pages(self.pool, K, D, dt, float("nan"))
        self.q = (torch.tensor(rng.standard_normal((T, H, D)), device="cuda") * scale).to(dt)
        self.k, self.v = [], []
        for r, (c, n) in enumerate(lens):
            at = torch.arange(c + n, device="cuda")
            pg = torch.tensor(oracle.tables[r], device="cuda", dtype=torch.int64)[at // page]
            for pages_, rows in ((self.kp, self.k), (self.vp, self.v)):
                x = torch.tensor(rng.standard_normal((c + n, K, D)), device="cuda").to(dt)
                pages_[pg, :, at % page] = x
                rows.append(x)

    def want(self, sink, sees=None):
        """(out, denominators, A, e) of every row; rows behind the last request 0."""
        sees = self.sees if sees is None else sees
        T = self.q.shape[0]
        out, size = np.zeros((T, self.H, self.D)), np.zeros((T, self.H, self.D))
        den, e = np.zeros((T, self.H)), np.zeros((T, self.H))
        q = _f64(self.q)
        for r, (c, n) in enumerate(self.lens):
            k, v = _f64(self.k[r]), _f64(self.v[r])
            for i in range(n):
                t = self.starts[r] + i
                drafted = np.arange(n) <= i if n > sees.shape[1] else sees[t, :n]
                see = np.concatenate((np.ones(c, bool), drafted))
                for h in range(self.H):
                    kh = h * self.K // self.H
                    out[t, h], den[t, h], size[t, h], S = P.attention_row(q[t, h], k[see, kh], v[see, kh], sink)
                    e[t, h] = _weight_error(self.dt, self.D, S, int(see.sum()))
        return out, den, size, e

    def check(self, sink=0.5, masks=None, sees=None, what=""):
        out, den = A.paged_tree_afa(self.q, self.kp, self.vp, self.plan, sink, masks=masks, return_denominator=True)
        want, wden, size, e = self.want(sink, sees)
        u = 0 if self.dt == F64 else U
        bound = 2 * e[..., None] * size + _half(self.dt) * np.abs(want) + 4 * u * np.abs(want) + _tiny(self.dt)
        _close(out, want, np.where(np.isnan(bound), 0, bound), what)
        _close(den, wden, 2 * e * wden, (what, "denominator"))
        return out


# (cached, new) of each request: single tokens, lengths on both sides of a tile and of a page, no cached
# tokens, no new ones, longer ones
LENS = [(0, 1), (1, 1), (31, 1), (32, 1), (33, 5), (0, 7), (63, 2), (64, 0), (15, 17), (130, 3), (300, 12), (0, 0), (7, 9)]


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("H,K,D,page", [
    (4, 2, 64, 16), (2, 2, 128, 64), (6, 6, 48, 32), (8, 1, 96, 8), (3, 3, 32, 128), (4, 1, 256, 16), (6, 2, 40, 3), (16, 1, 64, 32),
    (2, 1, 80, 1), (1, 1, 7, 5), (12, 4, 128, 16),
])
def test_attention(dt, H, K, D, page):
    _Cache(dt, LENS, H, K, D, page, seed=D + page, tail=3).check(what=(H, K, D, page))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D,scale", [(64, 3.0), (128, 0.05), (64, 8.0)])
def test_attention_scores(dt, D, scale):
    """Scores from near 0 to beyond 30 of both signs: fp16 weights that no fp16 number holds."""
    _Cache(dt, [(200, 4), (33, 9), (0, 3)], 4, 2, D, 32, seed=3, scale=scale).check(what=scale)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_attention_negative_scores(dt):
    """Keys that all point away from the query: weights far below 1, no sink."""
    x = _Cache(dt, [(150, 3), (40, 20)], 2, 2, 64, 16, seed=4)
    x.q = (x.q.abs() + 0.25).to(dt)
    for r, (c, n) in enumerate(x.lens):
        at = torch.arange(c + n, device="cuda")
        pg = torch.tensor(x.tables[r], device="cuda", dtype=torch.int64)[at // 16]
        x.k[r] = (-x.k[r].abs()).to(dt)
        x.kp[pg, :, at % 16] = x.k[r]
    x.check(sink=0.0)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("new,max_tree,parents,G", [(70, 64, True, 1), (64, 64, True, 2), (129, 192, True, 1), (256, 256, True, 1),
                                                    (100, 0, False, 4), (33, 64, False, 8), (200, 64, False, 1)])
def test_attention_long_drafts(dt, new, max_tree, parents, G):
    """Trees of more words than one, prompts longer than a tree, several row blocks."""
    _Cache(dt, [(45, new), (0, new // 2), (300, 1)], 2 * G, 2, 64, 32, max_tree, seed=new, parents=parents).check()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_attention_long_cache(dt):
    """Thousands of cached keys, split over workgroups, beside short ones; one more key than a split."""
    for lens in ([(5000, 3), (17, 2), (2048, 1)], [(4097, 9)], [(128, 1)], [(129, 1)], [(3999, 4), (0, 4)]):
        _Cache(dt, lens, 4, 2, 64, 64, seed=lens[0][0]).check(what=lens)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("sink", [0.0, 0.5])
def test_attention_given_masks(dt, sink):
    """Masks of the caller's: rows that see nothing are 0 with or without a sink, bits past the
    request's tokens count for nothing, and no cached token is hidden by them."""
    x = _Cache(dt, [(0, 40), (0, 5), (37, 20)], 4, 2, 64, 16, seed=8)
    rng = np.random.default_rng(9)
    sees = rng.random(x.sees.shape) < 0.3
    sees[[0, 3, 41, 44]] = False
    masks = torch.tensor(P.mask_words(sees), device="cuda")
    out = x.check(sink, masks, sees)
    assert (out[0] == 0).all() and (out[44] == 0).all()


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("D,page", [(64, 32), (128, 16), (48, 64), (256, 32)])
def test_attention_masked_places(dt, D, page):
    """Infinities and NaN in drafted keys and values reach the rows that see them and no others."""
    x = _Cache(dt, [(20, 30), (0, 12)], 4, 2, D, page, seed=11)
    first = x.check()
    at = torch.tensor(x.tables[0], device="cuda", dtype=torch.int64)
    for j, (which, value) in {3: (x.vp, "inf"), 9: (x.vp, "nan"), 14: (x.kp, "nan"), 21: (x.vp, "-inf")}.items():
        which[at[(20 + j) // page], :, (20 + j) % page, D // 2] = float(value)
    out = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan)
    hit = x.sees[:, [3, 9, 14, 21]]
    hit[30:] = False
    hit = torch.tensor(hit, device="cuda")
    assert torch.equal(out[~hit.any(1)], first[~hit.any(1)])
    bad = ~torch.isfinite(out)
    assert bad[hit[:, 2]].all()
    only_v = hit.any(1) & ~hit[:, 2]
    assert bad[only_v][..., D // 2].all() and not bad[only_v][..., :D // 2].any() and not bad[only_v][..., D // 2 + 1:].any()
    up = hit[:, 0] & ~hit[:, 1:].any(1)
    assert (out[up][..., D // 2] == float("inf")).all() and up.any()


def test_attention_leaves_the_rows_behind():
    x = _Cache(BF16, [(40, 3), (5, 2)], 4, 2, 64, 16, seed=12, tail=6)
    whole = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan)
    assert (whole[5:] == 0).all()
    out = torch.full_like(x.q, 3.0)
    got, den = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, out=out, return_denominator=True)
    assert got is out and torch.equal(out[:5], whole[:5]) and (out[5:] == 3.0).all() and (den[5:] == 0).all()
    q = torch.empty(11, 4, 192, dtype=BF16, device="cuda")[..., 64:128].copy_(x.q)
    assert torch.equal(A.paged_tree_afa(q, x.kp, x.vp, x.plan), whole)
    q = torch.empty(11, 4, 67, dtype=BF16, device="cuda")[..., 1:65].copy_(x.q)  # rows of no alignment
    off = (A.paged_tree_afa(q, x.kp, x.vp, x.plan).float() - whole.float()).abs()
    assert (off <= 2.0 ** -7 * whole.float().abs() + 1e-3).all()


def test_attention_unserved_requests_and_bad_pages():
    """Requests without pages or too long have rows of 0; page ids outside the pool hold no keys."""
    pool = A.PagePool(4, 16, 4, 64)
    plan = _plan(pool, 8, 4, 64, 2, 1, 64, BF16)
    A.build_block_tables(plan, _i32([20, 60, 3, 0]), _i32([2, 1, 3, 2]))
    assert plan.status.tolist() == [0, 1, 1, 1]
    kp, vp = _pages(pool, 1, 64, BF16, 1.0)
    q = torch.ones(8, 2, 64, device="cuda", dtype=BF16)
    out, den = A.paged_tree_afa(q, kp, vp, plan, return_denominator=True)
    assert (out[2:] == 0).all() and (den[2:] == torch.tensor([0.5] * 6, device="cuda")[:, None]).all()
    assert (out[:2] > 0.9).all()
    plan.pool.block_tables[0, 0] = 99
    few, part = A.paged_tree_afa(q, kp, vp, plan, return_denominator=True)
    # 16 of the 21 and 22 keys that the two rows see are gone: s = 8, equal weights
    w = P.rho8(np.float64(8.0))
    np.testing.assert_allclose(part[:2].cpu().numpy(), [[5 * w + 0.5] * 2, [6 * w + 0.5] * 2], rtol=1e-4)


def test_attention_across_2_31_elements():
    """Pages whose elements lie beyond 2^31 in both arrays."""
    page, K, D = 64, 2, 128
    x = _Cache(BF16, [(150, 3), (33, 2)], 4, K, D, page, seed=13, far=(1 << 31) // (page * K * D) + 5)
    assert x.kp.numel() > 1 << 31
    x.check()


def test_attention_refusals():
    x = _Cache(BF16, [(40, 3)], 4, 2, 64, 16)
    call = lambda q=x.q, k=x.kp, v=x.vp, p=x.plan, **kw: A.paged_tree_afa(q, k, v, p, **kw)  # noqa: E731
    for bad in (-0.5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="sink_omega"):
            call(sink_omega=bad)
    with pytest.raises(ValueError):
        call(q=x.q[:2])
    with pytest.raises(TypeError):
        call(q=x.q.half())
    with pytest.raises(ValueError):
        call(k=x.kp[:1])
    with pytest.raises(RuntimeError, match="GPU"):
        call(v=x.vp.cpu())
    with pytest.raises(ValueError, match="masks"):
        call(masks=x.plan.masks.int())
    with pytest.raises(ValueError, match="masks"):
        call(masks=x.plan.masks[:2])
    with pytest.raises(ValueError, match="out"):
        call(out=torch.empty_like(x.q, dtype=F32))
    with pytest.raises(ValueError, match="out"):
        call(out=x.q)
    both = torch.zeros((x.q.shape[0] + 1, *x.q.shape[1:]), device="cuda", dtype=x.q.dtype)
    with pytest.raises(ValueError, match="overlap"):
        call(q=both[1:], out=both[:-1])
    with pytest.raises(ValueError, match="max_tree"):
        p = _plan(x.pool, 3, max_tree=0, heads=4, kv_heads=2)
        A.paged_tree_afa(x.q, x.kp, x.vp, p, masks=x.plan.masks)


def test_attention_of_a_fresh_plan():
    """A plan that no step has filled: every row is behind the last request's."""
    pool = A.PagePool(4, 16, 2, 32)
    plan = _plan(pool, 5)
    kp, vp = _pages(pool, 1, 64, BF16, float("nan"))
    assert (A.paged_tree_afa(torch.ones(5, 2, 64, device="cuda", dtype=BF16), kp, vp, plan) == 0).all()


# ------------------------------------------------------------------------------------ whole steps
def _dense_rows(q, k, v, rotary):
    """algebraic_flash_attention of one sequence (L, H, D) / (L, K, D), rotated inside the call."""
    G = q.shape[1] // k.shape[1]
    q, k, v = q.transpose(0, 1)[None], k.repeat_interleave(G, 1).transpose(0, 1)[None], v.repeat_interleave(G, 1).transpose(0, 1)[None]
    return A.algebraic_flash_attention(q, k, v, causal=True, rotary_params=rotary)[0].transpose(0, 1)


@pytest.mark.parametrize("dt,H,K,D,page", [(F32, 4, 2, 64, 16), (BF16, 4, 4, 128, 32), (F16, 6, 2, 48, 8), (F64, 2, 1, 20, 5)])
def test_decoding_with_drafts_is_causal_attention(dt, H, K, D, page):
    """Three sequences decoded through a prompt, drafted trees of which a path is accepted, and single
    tokens: the rows on the accepted path are those of causal attention over the whole sequence.

    Both sides round rotated q and k and the result to the type: an element of q or k off by half a step of the
    type moves a score by at most 2 h(t) S and a weight by 16 h(t) S."""
    rng = np.random.default_rng(D)
    R, L = 3, 90
    rot = A.build_cayley_rotary_matrix(D, 128, dtype=F64 if dt == F64 else F32)
    seq = [tuple((torch.tensor(rng.standard_normal((L, n, D)), device="cuda") * 0.5).to(dt) for n in (H, K, K)) for _ in range(R)]
    dense = [_dense_rows(*s, rot) for s in seq]
    pool = A.PagePool(100, page, R, L + 20)
    kp, vp = _pages(pool, K, D, dt, float("nan"))
    done = np.array([0, 0, 0])
    steps = [(40, 0), (17, 0), (1, 0), (1, 6), (3, 9), (1, 0), (5, 2), (1, 30)]  # accepted tokens, other nodes
    for accept, others in steps:
        new = np.array([accept + others, accept, accept + others])
        T = int(new.sum()) + 2
        plan = _plan(pool, T, int(new.max()), 64, H, K, D, dt)
        rows = [torch.randn(T, n, D, device="cuda").to(dt) for n in (H, K, K)]
        parents, path, at = np.full(T, -1), [], 0
        for r in range(R):
            n = int(new[r])
            on = np.sort(rng.choice(n, accept, replace=False))
            for i in range(n):
                before = [j for j in on if j < i]
                parents[at + i] = (before[-1] if before else -1) if i in on else (rng.integers(-1, i) if i else -1)
            for x, whole in zip(rows, seq[r]):
                x[at + torch.tensor(on, device="cuda")] = whole[done[r]:done[r] + accept]
            path.append(at + on)
            at += n
        A.build_block_tables(plan, _i32(done), _i32(new), _i32(parents) if others else None)
        assert (plan.status == 0).all()
        q = A.append_to_cache(*rows, kp, vp, plan, rot)
        out = A.paged_tree_afa(q, kp, vp, plan)
        for r in range(R):
            want = dense[r][done[r]:done[r] + accept].double()
            S = 0.25 * 3.0 * np.sqrt(D)  # |q . k| / sqrt(D) of normal vectors of scale 1/2, beyond 3 sigma per feature
            tol = (16 * _half(dt) * S + 4 * _half(dt)) if dt != F64 else 1e-12
            size = seq[r][2].double().abs().max()
            assert (out[path[r]].double() - want).abs().max() <= tol * size, (accept, others, r)
        # the accepted path is stored again where the next step expects it
        keep = _plan(pool, R * accept, accept, 0, H, K, D, dt)
        A.build_block_tables(keep, _i32(done), _i32([accept] * R))
        chosen = torch.tensor(np.concatenate(path), device="cuda")
        A.append_to_cache(*(x[chosen].contiguous() for x in rows), kp, vp, keep, rot)
        done += accept
    A.build_block_tables(keep, _i32([0] * R), _i32([0] * R))
    assert pool.held.tolist() == [0] * R and pool.ring_state[1].item() == pool.num_pages


def _step(x, cached, new, parents, qkv, rot, kp, vp, plan):
    A.build_block_tables(plan, cached, new, parents)
    q = A.append_to_cache(*qkv, kp, vp, plan, rot)
    return A.paged_tree_afa(q, kp, vp, plan, return_denominator=True)


def test_captured_steps():
    """Two steps of one pool captured into graphs that share a memory pool, replayed in turn with other
    lengths, parents and activations, with eager steps between: every replay equals the eager step."""
    H, K, D, T, R = 4, 2, 64, 24, 5
    rng = np.random.default_rng(20)
    rot = A.build_cayley_rotary_matrix(D, 4096)
    mine, theirs = A.PagePool(200, 16, R, 2000), A.PagePool(200, 16, R, 2000)
    kp, vp = _pages(mine, K, D, BF16, 0.0)
    ek, ev = kp.clone(), vp.clone()
    lens, fresh, parents = _i32([0] * R), _i32([1] * R), _i32([-1] * T)
    qkv = [torch.zeros(T, n, D, device="cuda", dtype=BF16) for n in (H, K, K)]
    plans = [_plan(mine, T, 12, 64, H, K, D), _plan(mine, T, 12, 64, H, K, D)]
    eager = _plan(theirs, T, 12, 64, H, K, D)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(None, lens, fresh, parents, qkv, rot, kp, vp, plans[0])
    torch.cuda.current_stream().wait_stream(side)
    _step(None, lens, fresh, parents, qkv, rot, ek, ev, eager)
    graphs, outs = [], []
    for plan in plans:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(_step(None, lens, fresh, parents, qkv, rot, kp, vp, plan))
        graphs.append(g)
    for turn in range(10):
        new = rng.integers(0, 5, R)
        lens.copy_(_i32(rng.integers(0, 600 if turn % 3 else 1500, R) // (1 if turn % 4 else 8)))
        fresh.copy_(_i32(new))
        parents.copy_(_i32(rng.integers(-1, 4, T)))
        for x in qkv:
            x.copy_(torch.randn(x.shape, device="cuda"))
        which = turn % 2
        graphs[which].replay()
        want = _step(None, lens, fresh, parents, qkv, rot, ek, ev, eager)
        torch.cuda.synchronize()
        total = int(new.sum())
        assert torch.equal(plans[which].slots, eager.slots) and torch.equal(mine.held, theirs.held)
        assert torch.equal(kp, ek) and torch.equal(vp, ev)
        for got, ref in zip(outs[which], want):
            assert torch.equal(got[:total], ref[:total]), turn


def test_steps_on_two_streams():
    """Two caches stepped at the same time on streams of their own."""
    xs = [_Cache(BF16, [(700, 6), (90, 2)], 4, 2, 64, 32, seed=s) for s in (30, 31)]
    want = [A.paged_tree_afa(x.q, x.kp, x.vp, x.plan) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                got[i].append(A.paged_tree_afa(x.q, x.kp, x.vp, x.plan))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_results_repeat():
    x = _Cache(F16, [(3000, 6), (90, 2), (1500, 1)], 4, 2, 64, 32, seed=40)
    first = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan)
    for _ in range(5):
        assert torch.equal(A.paged_tree_afa(x.q, x.kp, x.vp, x.plan), first)
