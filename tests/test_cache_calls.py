"""Normalised heads, the shared prefix, accumulated weights and eviction without a GPU: refusals of the Python layer and of
the C ABI, all before any device work, and the oracle they are tested against."""
import ctypes
import math
import os

import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from algebraic_intelligence_amd import _lib, attention
from oracle import cache_oracle as C
from tests.test_paged import DUMMY, POINTERS, SIZES, _plan, _StubPlan


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from algebraic_intelligence_amd import build
        build.build()
    return _lib.lib()


# ---------------------------------------------------------------------------------------- C ABI
def _append(lib, p=None, q=DUMMY, k=DUMMY, v=DUMMY, out=DUMMY, kp=DUMMY, vp=DUMMY, qs=DUMMY, ks=DUMMY, eps=1e-6, rc=DUMMY, rs=DUMMY,
            n=9, pos=None, axes=1):
    return lib.afa_paged_append_norm(ctypes.byref(p or _plan()), q, k, v, None, out, kp, vp, None, qs, ks, eps, rc, rs, n, pos, axes,
                                     None, None)


def _prefix(lib, p=None, q=DUMMY, k=DUMMY, v=DUMMY, n=10, kp=DUMMY, vp=DUMMY, masks=None, out=DUMMY, sink=0.5, ws=None, size=0):
    return lib.afa_paged_prefix_fwd(ctypes.byref(p or _plan()), q, None, k, v, n, None, kp, vp, None, masks, out, None, sink, 0, ws,
                                    size, None)


def _weights(lib, p=None, q=DUMMY, kp=DUMMY, masks=None, den=DUMMY, w=DUMMY, row=64, ws=None, size=0):
    return lib.afa_paged_weights(ctypes.byref(p or _plan()), q, None, kp, None, masks, den, w, row, 0, ws, size, None)


@pytest.mark.parametrize("kw,code", SIZES + POINTERS + [(dict(schedule=DUMMY + 4), _lib.ERR_ALIGN)])
def test_the_plan_is_checked_by_every_call(lib, kw, code):
    p = _plan(**kw)
    assert _append(lib, p) == code and _prefix(lib, p) == code and _weights(lib, p) == code
    if (kw, code) in SIZES:
        assert lib.afa_paged_prefix_workspace_size(ctypes.byref(p), 10) == 0


def test_no_plan(lib):
    assert lib.afa_paged_append_norm(None, *[DUMMY] * 3, None, *[DUMMY] * 3, None, DUMMY, DUMMY, 1e-6, None, None, 0, None, 1, None,
                                     None) == _lib.ERR_NULL
    assert lib.afa_paged_prefix_fwd(None, DUMMY, None, DUMMY, DUMMY, 1, None, DUMMY, DUMMY, None, None, DUMMY, None, 0.5, 0, None, 0,
                                    None) == _lib.ERR_NULL
    assert lib.afa_paged_weights(None, DUMMY, None, DUMMY, None, None, DUMMY, DUMMY, 1, 0, None, 0, None) == _lib.ERR_NULL
    assert lib.afa_paged_prefix_workspace_size(None, 1) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ERR_NULL), (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL), (dict(out=None), _lib.ERR_NULL),
    (dict(out=None, rc=None, rs=None), _lib.ERR_NULL), (dict(kp=None), _lib.ERR_NULL), (dict(vp=None), _lib.ERR_NULL),
    (dict(qs=None), _lib.ERR_NULL), (dict(ks=None), _lib.ERR_NULL), (dict(eps=-1.0), _lib.ERR_EPS),
    (dict(eps=math.nan), _lib.ERR_EPS), (dict(eps=math.inf), _lib.ERR_EPS), (dict(rs=None), _lib.ERR_ROTARY),
    (dict(n=0), _lib.ERR_ROTARY), (dict(p=_plan(head_dim=63)), _lib.ERR_ROTARY), (dict(axes=2), _lib.ERR_NULL),
])
def test_append_norm_arguments(lib, kw, code):
    assert _append(lib, **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ERR_NULL), (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL), (dict(kp=None), _lib.ERR_NULL),
    (dict(vp=None), _lib.ERR_NULL), (dict(out=None), _lib.ERR_NULL), (dict(n=0), _lib.ERR_SHAPE), (dict(n=-1), _lib.ERR_SHAPE),
    (dict(n=(1 << 29) + 1), _lib.ERR_SHAPE), (dict(sink=-1.0), _lib.ERR_SINK), (dict(sink=math.nan), _lib.ERR_SINK),
    (dict(p=_plan(max_tree=0), masks=DUMMY), _lib.ERR_UNSUPPORTED), (dict(ws=DUMMY, size=16), _lib.ERR_WORKSPACE),
    (dict(ws=DUMMY + 4, size=1 << 40), _lib.ERR_ALIGN), (dict(p=_plan(max_tokens=1 << 26, heads=1, kv_heads=1)), _lib.ERR_SHAPE),
])
def test_prefix_arguments(lib, kw, code):
    assert _prefix(lib, **kw) == code


def test_prefix_workspace_grows_with_the_rows(lib):
    size = lambda **kw: lib.afa_paged_prefix_workspace_size(ctypes.byref(_plan(**kw)), 100)  # noqa: E731
    assert 0 < size() < size(max_tokens=512) and size(dtype=_lib.AFA_F64) == 0
    assert lib.afa_paged_prefix_workspace_size(ctypes.byref(_plan()), 0) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ERR_NULL), (dict(kp=None), _lib.ERR_NULL), (dict(den=None), _lib.ERR_NULL), (dict(w=None), _lib.ERR_NULL),
    (dict(row=63), _lib.ERR_SHAPE), (dict(row=-64), _lib.ERR_SHAPE), (dict(p=_plan(max_tree=0), masks=DUMMY), _lib.ERR_UNSUPPORTED),
    (dict(ws=DUMMY, size=16), _lib.ERR_WORKSPACE), (dict(ws=DUMMY + 4, size=1 << 40), _lib.ERR_ALIGN),
])
def test_weights_arguments(lib, kw, code):
    assert _weights(lib, **kw) == code


def _evict(lib, dt=_lib.AFA_BF16, pages=8, page=16, R=2, width=4, K=2, D=64, table=DUMMY, held=DUMMY, kp=DUMMY, vp=DUMMY, cached=DUMMY,
           budget=20, first=0, recent=0, w=DUMMY, row=64, left=DUMMY, lens=DUMMY, ws=None, size=0):
    return lib.afa_paged_evict(dt, pages, page, R, width, K, D, table, held, kp, vp, None, cached, budget, first, recent, w, row, left,
                               lens, ws, size, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=4), _lib.ERR_DTYPE), (dict(pages=0), _lib.ERR_SHAPE), (dict(page=0), _lib.ERR_SHAPE), (dict(R=0), _lib.ERR_SHAPE),
    (dict(width=0), _lib.ERR_SHAPE), (dict(K=0), _lib.ERR_SHAPE), (dict(D=0), _lib.ERR_HEAD_DIM), (dict(D=1025), _lib.ERR_HEAD_DIM),
    (dict(pages=1 << 28), _lib.ERR_SHAPE), (dict(R=1 << 22, K=1 << 10), _lib.ERR_SHAPE),
    *[(dict([(n, None)]), _lib.ERR_NULL) for n in ("table", "held", "kp", "vp", "cached", "w", "left", "lens")],
    (dict(budget=0), _lib.ERR_SHAPE), (dict(budget=65), _lib.ERR_SHAPE), (dict(first=-1), _lib.ERR_SHAPE),
    (dict(recent=-1), _lib.ERR_SHAPE), (dict(first=21), _lib.ERR_SHAPE), (dict(first=10, recent=11), _lib.ERR_SHAPE),
    (dict(first=20, recent=2 ** 62), _lib.ERR_SHAPE), (dict(row=63), _lib.ERR_SHAPE), (dict(ws=DUMMY, size=16), _lib.ERR_WORKSPACE),
    (dict(ws=DUMMY + 8, size=1 << 40), _lib.ERR_ALIGN),
])
def test_evict_arguments(lib, kw, code):
    assert _evict(lib, **kw) == code


def test_evict_workspace(lib):
    size = lib.afa_paged_evict_workspace_size
    assert size(2, 64, 20, 2, 64) >= 2 * 20 * 4
    for bad in ((0, 64, 20, 2, 64), (2, 0, 1, 2, 64), (2, 64, 0, 2, 64), (2, 64, 65, 2, 64), (2, 64, 20, 0, 64), (2, 64, 20, 2, 1025)):
        assert size(*bad) == 0


_NORM = dict(dt=_lib.AFA_BF16, B=1, H=2, K=2, L=4, D=8, q=DUMMY, k=DUMMY, gq=DUMMY, gk=DUMMY, yq=DUMMY, yk=DUMMY, qs=DUMMY, ks=DUMMY,
             dqs=DUMMY, dks=DUMMY, eps=1e-6, rc=DUMMY, rs=DUMMY, n=9, pos=DUMMY, esz=8, pos_b=0, axes=2, sections=(2, 2), ws=None, size=0)


def _norm(lib, backward, **kw):
    c = {**_NORM, **kw}
    cuts = None if c["sections"] is None else (ctypes.c_int32 * len(c["sections"]))(*c["sections"])
    sizes = c["dt"], c["B"], c["H"], c["K"], c["L"], c["D"], c["q"], c["k"]
    turn = c["eps"], c["rc"], c["rs"], c["n"], c["pos"], c["esz"], c["pos_b"], c["axes"], cuts
    if backward:
        return lib.ago_norm_rotate_axes_bwd(*sizes, c["gq"], c["gk"], c["yq"], c["yk"], None, c["qs"], c["ks"], c["dqs"], c["dks"], *turn,
                                            c["ws"], c["size"], None)
    return lib.ago_norm_rotate_axes(*sizes, c["yq"], c["yk"], None, c["qs"], c["ks"], *turn, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=9), _lib.ERR_DTYPE), (dict(B=0), _lib.ERR_SHAPE), (dict(H=0), _lib.ERR_SHAPE), (dict(K=-1), _lib.ERR_SHAPE),
    (dict(L=0), _lib.ERR_SHAPE), (dict(D=0), _lib.ERR_SHAPE), (dict(D=(1 << 24) + 2), _lib.ERR_SHAPE), (dict(q=None), _lib.ERR_NULL),
    (dict(k=None), _lib.ERR_NULL), (dict(yq=None), _lib.ERR_NULL), (dict(yk=None), _lib.ERR_NULL), (dict(qs=None), _lib.ERR_NULL),
    (dict(ks=None), _lib.ERR_NULL), (dict(eps=-1.0), _lib.ERR_EPS), (dict(eps=math.nan), _lib.ERR_EPS), (dict(rc=None), _lib.ERR_ROTARY),
    (dict(rs=None), _lib.ERR_ROTARY), (dict(pos=None), _lib.ERR_NULL), (dict(pos=None, axes=1, sections=None, pos_b=4), _lib.ERR_NULL),
    (dict(esz=2), _lib.ERR_UNSUPPORTED), (dict(n=0), _lib.ERR_ROTARY), (dict(D=7), _lib.ERR_ROTARY),
    (dict(sections=(3, 2)), _lib.ERR_ROTARY), (dict(sections=None), _lib.ERR_NULL), (dict(axes=0), _lib.ERR_ROTARY),
    (dict(B=1 << 40, L=1 << 40), _lib.ERR_SHAPE), (dict(H=1 << 40), _lib.ERR_SHAPE),
])
def test_norm_arguments(lib, kw, code):
    assert _norm(lib, False, **kw) == code and _norm(lib, True, **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(gq=None), _lib.ERR_NULL), (dict(gk=None), _lib.ERR_NULL), (dict(dqs=None), _lib.ERR_NULL), (dict(dks=None), _lib.ERR_NULL),
    (dict(ws=DUMMY, size=16), _lib.ERR_WORKSPACE), (dict(ws=DUMMY + 4, size=1 << 40), _lib.ERR_ALIGN),
])
def test_norm_backward_arguments(lib, kw, code):
    assert _norm(lib, True, **kw) == code


def test_norm_backward_workspace(lib):
    size = lib.ago_norm_rotate_axes_bwd_workspace_size
    assert size(_lib.AFA_BF16, 64) > 0 and size(_lib.AFA_F64, 64) == 2 * size(_lib.AFA_F32, 64)
    assert size(9, 64) == 0 and size(_lib.AFA_F32, 0) == 0


# ------------------------------------------------------------------------------ the Python layer
def test_norm_refusals_without_a_gpu():
    q, k, w = torch.zeros(2, 4, 6, 8), torch.zeros(2, 2, 6, 8), torch.ones(8)
    tables = (torch.ones(10, 4), torch.zeros(10, 4))
    call = lambda q=q, k=k, qs=w, ks=w, t=tables, **kw: A.apply_ago_norm_rotations(q, k, qs, ks, t, **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="GPU"):
        call()
    for bad in (k[0], k[:1], k[:, :, :5], k[..., :4], None):
        with pytest.raises(ValueError):
            call(k=bad)
    with pytest.raises(TypeError, match="dtype"):
        call(k=k.double())
    with pytest.raises(TypeError):
        call(q=q.int())


def _stub_norm(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(attention, "_norm_launch", lambda q, k, *rest: (torch.zeros(q.shape), None if k is None else
                                                                        torch.zeros(k.shape)))


def test_norm_checks(monkeypatch):
    _stub_norm(monkeypatch)
    q, w = torch.ones(2, 4, 6, 8), torch.ones(8)
    tables, at = (torch.ones(10, 4), torch.zeros(10, 4)), torch.zeros(6, 2, dtype=torch.int64)
    call = lambda q=q, qs=w, t=tables, p=at, s=(2, 2), **kw: A.apply_ago_norm_rotations(q, None, qs, None, t, p, s, **kw)  # noqa: E731
    assert call().shape == q.shape and call(qs=w.double()).shape == q.shape and call(p=None, s=None).shape == q.shape
    assert A.apply_ago_norm_rotations(q[..., :7], None, w[:7], None).shape == (2, 4, 6, 7)
    for bad in (w[:4], torch.ones(8, 1), torch.ones(1)):
        with pytest.raises(ValueError, match="q_scale"):
            call(qs=bad)
    for bad in (w.int(), [1.0] * 8, None):
        with pytest.raises(TypeError, match="q_scale"):
            call(qs=bad)
    for bad in (-1e-9, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            call(eps=bad)
    for bad in ((2,), (3, 2), (-1, 2), None):
        with pytest.raises(ValueError, match="sections"):
            call(s=bad)
    with pytest.raises(ValueError, match="rotary_params"):
        call(t=None)
    with pytest.raises(ValueError, match="even"):
        A.apply_ago_norm_rotations(q[..., :7], None, w[:7], None, tables)
    with pytest.raises(ValueError, match="at least one feature"):
        A.apply_ago_norm_rotations(q[..., :0], None, w[:0], None)
    with pytest.raises(TypeError, match="int32 or int64"):
        call(p=at.float())


def test_norm_refuses_tangents(monkeypatch):
    """A dual q, k or scale is refused, also where no gradient is recorded, and never comes back without its tangent."""
    from torch.autograd import forward_ad

    _stub_norm(monkeypatch)
    q, k, w = torch.ones(2, 4, 6, 8), torch.ones(2, 2, 6, 8), torch.ones(8)
    call = lambda q, k, qs, ks: A.apply_ago_norm_rotations(q, k, qs, ks, (torch.ones(10, 4), torch.zeros(10, 4)))  # noqa: E731
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(q), None, w, None), (dual(q), k, w, w), (q, dual(k), w, w), (q, k, dual(w), w), (q, k, w, dual(w))):
            with pytest.raises(NotImplementedError):
                call(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call(*args)
        assert call(q, k, w, w)[1].shape == k.shape


class _Pool:
    device, num_pages, page_size, max_requests, max_len = torch.device("cpu"), 3, 16, 2, 32
    block_tables = torch.zeros(2, 2, dtype=torch.int32)


class _Plan(_StubPlan):
    pool, kv_heads, _ws = _Pool(), 2, None


def test_serving_calls_refuse_gradients_and_tangents():
    from torch.autograd import forward_ad

    plan = _Plan()
    w8, lens = torch.ones(8), torch.zeros(2, dtype=torch.int32)

    def calls(t):
        return {"append_to_cache": lambda: A.append_to_cache(t["q"], t["k"], t["v"], t["k_pages"], t["v_pages"], plan,
                                                             norms=(t["q_scale"], t["k_scale"])),
                "paged_prefix_afa": lambda: A.paged_prefix_afa(t["q"], t["k_prefix"], t["v_prefix"], t["k_pages"], t["v_pages"], plan),
                "accumulate_cache_weights": lambda: A.accumulate_cache_weights(t["q"], t["k_pages"], t["den"], plan, t["weights"]),
                "evict_from_cache": lambda: A.evict_from_cache(t["k_pages"], t["v_pages"], plan.pool, t["weights"], lens, 4)}

    uses = {"append_to_cache": ("q", "k", "v", "k_pages", "v_pages", "q_scale", "k_scale"),
            "paged_prefix_afa": ("q", "k_prefix", "v_prefix", "k_pages", "v_pages"),
            "accumulate_cache_weights": ("q", "k_pages", "den", "weights"), "evict_from_cache": ("k_pages", "v_pages", "weights")}

    def tensors():
        return {**plan.tensors(), "q_scale": w8.clone(), "k_scale": w8.clone(), "k_prefix": torch.zeros(2, 5, 8),
                "v_prefix": torch.zeros(2, 5, 8), "den": torch.ones(6, 4), "weights": torch.zeros(2, 32)}

    for name, used in uses.items():
        for which in used:
            t = tensors()
            t[which].requires_grad_(True)
            with pytest.raises(RuntimeError, match="gradient"):
                calls(t)[name]()
            with forward_ad.dual_level(), torch.no_grad():
                t = tensors()
                t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
                with pytest.raises(NotImplementedError):
                    calls(t)[name]()


def test_prefix_checks():
    plan = _Plan()
    t = plan.tensors()
    k = torch.zeros(2, 5, 8)
    call = lambda k=k, v=k, **kw: A.paged_prefix_afa(t["q"], k, v, t["k_pages"], t["v_pages"], plan, **kw)  # noqa: E731
    for bad in (k[0], k[:1], k[:, :0], k[..., :4], torch.zeros(2, 8, 5)):
        with pytest.raises(ValueError, match="prefix"):
            call(k=bad, v=bad)
    with pytest.raises(ValueError, match="v_prefix"):
        call(v=k[:, :4])
    with pytest.raises(TypeError, match="k_prefix"):
        call(k=k.half())
    with pytest.raises(ValueError, match="contiguous head"):
        call(v=torch.zeros(2, 8, 5).transpose(1, 2))
    with pytest.raises(ValueError, match="sink_omega"):
        call(sink_omega=math.nan)


# ------------------------------------------------------------------------------------ the oracle
def test_kept_by_brute_force():
    """Every set of the right size that holds the sure ones: none weighs more, and of equal ones none comes earlier."""
    from itertools import combinations

    rng = np.random.default_rng(0)
    for n, budget, first, recent in ((7, 4, 1, 1), (6, 3, 0, 0), (8, 5, 2, 3), (5, 5, 1, 1), (6, 1, 0, 1)):
        w = rng.integers(0, 3, n).astype(float)
        got = C.kept(w, n, budget, first, recent)
        sure = {j for j in range(n) if j < first or j >= n - recent} if n > budget else set(range(n))
        assert sure <= set(got) and len(got) == min(n, budget) and got == sorted(got)
        best = max((sum(w[list(c)]), [-j for j in c]) for c in combinations(range(n), len(got)) if sure <= set(c))
        assert (sum(w[got]), [-j for j in got]) == best


def test_norm_gradient_by_differences():
    rng = np.random.default_rng(1)
    x, w, g = rng.standard_normal((1, 2, 3, 8)), 1 + rng.standard_normal(8) / 4, rng.standard_normal((1, 2, 3, 8))
    a = rng.uniform(0, 6, (9, 4))
    at = rng.integers(0, 9, (1, 3, 2))
    rot = np.cos(a), np.sin(a), at, (2, 1)
    f = lambda x, w: np.sum(C.norm_rotate(x, w, 1e-3, *rot) * g)  # noqa: E731
    dx, dw = C.norm_rotate_gradient(x, w, 1e-3, g, *rot)
    for arr, d in ((x, dx), (w, dw)):
        for i in rng.integers(0, arr.size, 10):
            e = np.zeros(arr.size)
            e[i] = 1e-6
            e = e.reshape(arr.shape)
            up, down = (f(x + s * e, w) if arr is x else f(x, w + s * e) for s in (1, -1))
            assert abs((up - down) / 2e-6 - d.reshape(-1)[i]) < 1e-6 * (1 + abs(d.reshape(-1)[i]))
