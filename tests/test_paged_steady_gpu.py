"""The serving operators at the sizes at which they spend their time: attention whose workgroups run through tens of
key tiles, several requests and more pages than they hold entries of, in every instance of the kernel; pages of
other stride orders; rotations and cache writes of several heads a thread, and past the caches; a decoded
sequence row by row.

Bounds count roundings as tests/test_paged_gpu.py does.
"""
import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from oracle import paged_oracle as P
from tests.test_paged_gpu import (BF16, F16, F32, F64, U, _Cache, _close, _f64, _half, _i32, _plan, _rotation_bound, _tables, _tiny,
                                  _weight_error)

pytestmark = pytest.mark.gpu

LEAD, SHORTEST, TILE = 4, 4, 32  # units of the plan's line: a segment's start, a workgroup's least, keys of a unit


def _units(lens, group, bytes_, kv_heads):
    """(rows of a segment, units of a workgroup, units of a key head) as the plan shares the work."""
    most = max(n for _, n in lens) * group
    rows = 16
    while rows < most and rows < (128 if bytes_ <= 256 else 64):
        rows *= 2
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    slots = max(1, (1 if bytes_ >= 512 else 2) * cus // kv_heads)
    total = sum(-(-n * group // rows) * (LEAD + -(-(c + n) // TILE)) for c, n in lens if n)
    return rows, max(total // slots + 1, SHORTEST), total


class _Steady:
    """A step of drafted trees over many key heads: every place of the pages that holds no key is NaN."""

    def __init__(self, dt, lens, H, K, D, page, max_tree=64, seed=0):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        T = sum(n for _, n in lens)
        self.dt, self.lens, self.H, self.K, self.D = dt, lens, H, K, D
        need = [-(-(c + n) // page) for c, n in lens]
        self.pool = A.PagePool(sum(need), page, len(lens), max(c + n for c, n in lens))
        order = rng.permutation(sum(need))
        self.pool.ring.copy_(_i32(order))
        self.plan = _plan(self.pool, T, max(n for _, n in lens), max_tree, H, K, D, dt)
        parents = None
        if max_tree:
            parents = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for _, n in lens])
        A.build_block_tables(self.plan, _i32([c for c, _ in lens]), _i32([n for _, n in lens]),
                             None if parents is None else _i32(parents))
        assert (self.plan.status == 0).all()
        new = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dt)  # noqa: E731
        self.kp, self.vp = (new(sum(need), K, page, D) for _ in range(2))
        self.q = new(T, H, D)
        self.sees, self.tables, at = [], [], 0
        for r, (c, n) in enumerate(lens):
            self.tables.append(order[at:at + need[r]])
            at += need[r]
            if (c + n) % page:
                for pages in (self.kp, self.vp):
                    pages[int(self.tables[r][-1]), :, (c + n) % page:] = float("nan")
            see = np.ones((n, c + n), bool)
            first = sum(m for _, m in lens[:r])
            for i in range(n):
                see[i, c:] = False
                j = i
                while j >= 0:
                    see[i, c + j] = True
                    j = j - 1 if parents is None else int(parents[first + j])
            self.sees.append(see)

    def run(self, kp=None, vp=None):
        return A.paged_tree_afa(self.q, self.kp if kp is None else kp, self.vp if vp is None else vp, self.plan,
                                return_denominator=True)

    def check(self, kv_heads):
        """Every row of the query heads of some key heads against 64 bits."""
        out, den = self.run()
        assert torch.isfinite(out).all() and torch.isfinite(den).all()
        G, row = self.H // self.K, 0
        for r, (c, n) in enumerate(self.lens):
            pages = torch.tensor(self.tables[r], device="cuda")
            for hk in kv_heads:
                k, v = (p[pages, hk].reshape(-1, self.D)[:c + n] for p in (self.kp, self.vp))
                k, v = _f64(k), _f64(v)
                q = _f64(self.q[row:row + n, hk * G:(hk + 1) * G])
                s = (q @ k.T) / np.sqrt(self.D)
                w = P.rho8(s) * self.sees[r][:, None, :]
                wden = w.sum(-1) + 0.5
                S = ((np.abs(q) @ np.abs(k).T) / np.sqrt(self.D) * self.sees[r][:, None, :]).max(-1)
                N = self.sees[r].sum(-1)[:, None]
                e = np.vectorize(lambda S, N: _weight_error(self.dt, self.D, S, N))(S, N)
                want, size = w @ v / wden[..., None], w @ np.abs(v) / wden[..., None]
                bound = 2 * e[..., None] * size + (_half(self.dt) + 4 * U) * np.abs(want) + _tiny(self.dt)
                what = (r, hk)
                _close(out[row:row + n, hk * G:(hk + 1) * G], want, bound, what)
                _close(den[row:row + n, hk * G:(hk + 1) * G], wden, 2 * e * wden, what)
            row += n
        return out


LONG = [(3000, 13), (1700, 9), (40, 13)] + [(90 + 17 * i, 5 + i % 4) for i in range(8)]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 48, 64, 96, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 4, 8])
def test_long_stretches(dt, D, group):
    """Every instance of the matrix-core kernel, its workgroups over a dozen and more tiles of several requests."""
    K = 64
    bytes_ = D * dt.itemsize
    rows, stretch, total = _units(LONG, group, bytes_, K)
    assert rows == min(16 * group, 128 if bytes_ <= 256 else 64)
    slots = total / stretch
    assert stretch >= 24 and slots > 3
    x = _Steady(dt, LONG, K * group, K, D, 16, seed=D + group)
    first = x.check([0, 37, 63])
    assert torch.equal(x.run()[0], first)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("group,page", [(1, 8), (1, 64), (2, 8), (2, 64), (4, 8), (4, 64), (8, 8), (8, 32)])
def test_more_pages_than_a_wave_holds(dt, group, page):
    """A workgroup (a wave's own part of it up to 32 rows) over more than 64 pages of 8 tokens, with few slots a head."""
    K = 256 if group <= 2 else 64
    lens = [(5000, 13), (700, 2), (2100, 7), (0, 1)]
    rows, stretch, _ = _units(lens, group, 64 * dt.itemsize, K)
    waves = {16: 4, 32: 4 if dt != F32 else 2}.get(rows, 1)
    assert stretch // waves * TILE > 64 * 8
    x = _Steady(dt, lens, K * group, K, 64, page, seed=page + group)
    first = x.check([1, K // 2, K - 1])
    assert torch.equal(x.run()[0], first)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("group", [1, 8])
def test_prompts_over_long_stretches(dt, group):
    """Chains longer than a tree: each row block ends at its own last key."""
    lens = [(0, 700), (900, 300), (33, 1), (0, 129)]
    _, stretch, _ = _units(lens, group, 64 * dt.itemsize, 64)
    assert stretch >= 24
    x = _Steady(dt, lens, 64 * group, 64, 64, 32, seed=group)
    # without parents each token follows the one before it, in the short requests too
    A.build_block_tables(x.plan, _i32([c for c, _ in lens]), _i32([n for _, n in lens]))
    x.sees = [np.tril(np.ones((n, c + n), bool), c) for c, n in lens]
    x.check([0, 63])


@pytest.mark.parametrize("dt", [F16])
@pytest.mark.parametrize("group", [1, 2, 4, 8])
def test_growing_fp16_weights(dt, group):
    """Later keys weigh ever more, so that sums of many tiles are scaled down again and again."""
    K = 64
    x = _Steady(dt, LONG, K * group, K, 64, 16, seed=50 + group)
    x.q = x.q.abs()
    for r, (c, n) in enumerate(LONG):
        grow = torch.linspace(0.02, 6.0, c + n, device="cuda")
        at = torch.arange(c + n, device="cuda")
        pages = torch.tensor(x.tables[r], device="cuda")[at // 16]
        x.kp[pages, :, at % 16] = (x.kp[pages, :, at % 16].abs() * grow[:, None, None]).to(dt)
    x.check([0, 41])


@pytest.mark.parametrize("dt", [BF16, F16, F32, F64])
@pytest.mark.parametrize("D,page,group", [(64, 16, 2), (128, 32, 8), (48, 8, 1), (64, 64, 4), (40, 5, 2)])
@pytest.mark.parametrize("layout", ["slots first", "heads first", "side by side", "padded", "one of them"])
def test_attention_over_other_page_strides(dt, D, page, group, layout):
    """Pages of any stride order hold the same keys: the same results bit for bit."""
    K = 3
    x = _Cache(dt, [(200, 7), (33, 13), (0, 5), (70, 1)], K * group, K, D, page, seed=D + page)
    want = A.paged_tree_afa(x.q, x.kp, x.vp, x.plan, return_denominator=True)
    n = x.kp.shape[0]
    new = lambda *shape: torch.full(shape, float("nan"), dtype=dt, device="cuda")  # noqa: E731
    if layout == "slots first":
        kp, vp = (new(n, page, K, D).transpose(1, 2) for _ in range(2))
    elif layout == "heads first":
        kp, vp = (new(K, n, page, D).transpose(0, 1) for _ in range(2))
    elif layout == "side by side":
        both = new(n, page, 2, K, D)
        kp, vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    elif layout == "padded":
        kp, vp = new(n, K, page, D + 8)[..., :D], new(n, K + 1, page + 2, D + 16)[:, 1:, 2:, 8:D + 8]
    else:
        kp, vp = x.kp, new(n, page, K, D).transpose(1, 2)
    kp.copy_(x.kp)
    vp.copy_(x.vp)
    assert not (kp.is_contiguous() and vp.is_contiguous())
    for got, ref in zip(A.paged_tree_afa(x.q, kp, vp, x.plan, return_denominator=True), want):
        assert torch.equal(got, ref)


# ------------------------------------------------------------------------ rotations and cache writes
@pytest.mark.parametrize("dt,B,H,K,L,D,sections", [
    (BF16, 1, 5, 2, 5003, 128, (16, 24, 24)), (F16, 2, 9, 1, 6571, 128, (40, 20)), (F32, 3, 5, 2, 3137, 128, (16, 24, 24)),
    (BF16, 1, 12, 0, 11001, 48, (24,)), (F32, 1, 3, 3, 12289, 64, (8, 12, 12)), (BF16, 3, 7, 4, 8191, 64, (1, 2, 3, 4)),
])
@pytest.mark.parametrize("layout", ["blhd", "bhld"])
def test_rotation_of_many_tokens(dt, B, H, K, L, D, sections, layout):
    """Several heads a thread, their number no multiple of four: the whole call's results are those of short
    stretches of it, bit for bit, and a sample of tokens is checked against 64 bits."""
    assert B * L * (H + K) * D * dt.itemsize // 16 >= 1 << 19
    rng = np.random.default_rng(L)
    tab = _tables(300, D)
    pos = torch.tensor(rng.integers(0, 300, (B, L, len(sections))), device="cuda")

    def new(n):
        x = torch.randn(B, L, n, D, device="cuda").to(dt).transpose(1, 2)
        return x if layout == "blhd" else x.contiguous()

    q, k = new(H), new(K) if K else None
    got = A.apply_ago_axis_rotations(q, k, tab, pos, sections)
    got = got if K else (got,)
    step = 499
    for l0 in range(0, L, step):
        part = slice(l0, min(l0 + step, L))
        want = A.apply_ago_axis_rotations(q[:, :, part], None if k is None else k[:, :, part], tab, pos[:, part], sections)
        for y, ref in zip(got, want if K else (want,)):
            assert torch.equal(y[:, :, part], ref), l0
    some = np.unique(np.concatenate(([0, 1, L - 2, L - 1], rng.integers(0, L, 40))))
    for y, x in zip(got, (q, k)):
        _close(y[:, :, some], *_rotation_bound(_f64(x[:, :, some]), _f64(tab[0]), _f64(tab[1]), pos.cpu().numpy()[:, some],
                                               sections, dt), layout)


@pytest.mark.parametrize("dt,H,K,D,page,tokens", [(BF16, 6, 2, 128, 64, 3301), (F32, 5, 1, 64, 16, 4703), (F16, 3, 3, 48, 32, 9803)])
def test_append_of_many_tokens(dt, H, K, D, page, tokens):
    """Several heads a thread: q and k as the rotation alone gives them, every other place as it was."""
    assert tokens * (H + 2 * K) * D * dt.itemsize // 16 >= 1 << 19
    lens = [(77, tokens - 1500), (0, 1499), (5, 1)]
    pool = A.PagePool(sum(-(-(c + n) // page) for c, n in lens) + 2, page, 3, tokens + 100)
    plan = _plan(pool, tokens + 9, tokens, 0, H, K, D, dt)
    A.build_block_tables(plan, _i32([c for c, _ in lens]), _i32([n for _, n in lens]))
    assert (plan.status == 0).all()
    T = tokens + 9
    flat = torch.randn(T, H + 2 * K, D, device="cuda").to(dt)
    q, k, v = flat[:, :H], flat[:, H:H + K], flat[:, H + K:]
    kp, vp = (torch.full_like(p, 7.0) for p in pool.new_pages(K, D, dt))
    want_k, want_v = kp.clone(), vp.clone()
    tab = _tables(tokens + 100, D)
    out = A.append_to_cache(q, k, v, kp, vp, plan, tab)
    turn = lambda x: A.apply_ago_axis_rotations(x.transpose(0, 1)[None], None, tab, plan.positions[:, None])[0].transpose(0, 1)  # noqa: E731
    assert torch.equal(out, turn(q))
    slots = plan.slots[:tokens].long()
    assert (slots >= 0).all() and (plan.slots[tokens:] == -1).all()
    want_k[slots // page, :, slots % page] = turn(k)[:tokens]
    want_v[slots // page, :, slots % page] = v[:tokens]
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


# ------------------------------------------------------------------------------------ whole steps
@pytest.mark.parametrize("dt,H,K,D,page", [(F32, 4, 2, 64, 16), (BF16, 4, 4, 128, 32), (F16, 6, 2, 48, 8), (BF16, 8, 1, 64, 64)])
def test_decoded_rows_are_the_sequences(dt, H, K, D, page):
    """Three sequences decoded through a prompt, drafted trees of which a path is accepted, and single
    tokens.  The rows on the accepted path against 64-bit attention over the sequence's own keys, rotated
    and rounded apart from the cache: each within its own bound, which is far below the row."""
    rng = np.random.default_rng(D)
    R, L, G = 3, 90, H // K
    rot = A.build_cayley_rotary_matrix(D, 128)
    at = torch.arange(L, device="cuda")[:, None]
    seq, turned = [], []
    for _ in range(R):
        q, k, v = (torch.tensor(rng.standard_normal((L, n, D)), device="cuda").to(dt) for n in (H, K, K))
        seq.append((q, k, v))
        yq, yk = A.apply_ago_axis_rotations(q.transpose(0, 1)[None], k.transpose(0, 1)[None], rot, at)
        turned.append((yq[0].transpose(0, 1), _f64(yk[0]), _f64(v.transpose(0, 1))))
    pool = A.PagePool(100, page, R, L + 20)
    kp, vp = (torch.full_like(p, float("nan")) for p in pool.new_pages(K, D, dt))
    done = np.zeros(R, int)
    for accept, others in [(40, 0), (17, 0), (1, 0), (1, 6), (3, 9), (1, 0), (5, 2), (1, 30)]:
        new = np.array([accept + others, accept, accept + others])
        T = int(new.sum()) + 2
        plan = _plan(pool, T, int(new.max()), 64, H, K, D, dt)
        rows = [torch.randn(T, n, D, device="cuda").to(dt) for n in (H, K, K)]
        parents, path, first = np.full(T, -1), [], 0
        for r in range(R):
            n = int(new[r])
            on = np.sort(rng.choice(n, accept, replace=False))
            for i in range(n):
                before = [j for j in on if j < i]
                parents[first + i] = (before[-1] if before else -1) if i in on else (rng.integers(-1, i) if i else -1)
            for x, whole in zip(rows, seq[r]):
                x[first + torch.tensor(on, device="cuda")] = whole[done[r]:done[r] + accept]
            path.append(first + on)
            first += n
        A.build_block_tables(plan, _i32(done), _i32(new), _i32(parents) if others else None)
        assert (plan.status == 0).all()
        q = A.append_to_cache(*rows, kp, vp, plan, rot)
        out = A.paged_tree_afa(q, kp, vp, plan)
        for r in range(R):
            yq, yk, yv = turned[r]
            assert torch.equal(q[path[r]], yq[done[r]:done[r] + accept])
            for i, row in enumerate(path[r]):
                j = done[r] + i
                for h in range(H):
                    ref, _, size, S = P.attention_row(_f64(yq[j, h]), yk[h // G, :j + 1], yv[h // G, :j + 1], 0.5)
                    e = _weight_error(dt, D, S, j + 1)
                    bound = 2 * e * size + (_half(dt) + 4 * U) * np.abs(ref) + _tiny(dt)
                    assert np.linalg.norm(bound) <= np.linalg.norm(ref) / 8
                    _close(out[row, h], ref, bound, (accept, others, r, i, h))
        # the accepted path is stored again where the next step expects it
        keep = _plan(pool, R * accept, accept, 0, H, K, D, dt)
        A.build_block_tables(keep, _i32(done), _i32([accept] * R))
        chosen = torch.tensor(np.concatenate(path), device="cuda")
        A.append_to_cache(*(x[chosen].contiguous() for x in rows), kp, vp, keep, rot)
        done += accept
