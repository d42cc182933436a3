"""Norms of rows near the ends of fp32's range on the GPU, against float64 (bounds of tests/test_norm_gpu.py)."""
import numpy as np
import pytest
import torch

import algebraic_intelligence_amd as A
from tests.test_norm_gpu import _backward, _forward
from tests.test_paged_gpu import BF16, F32, F64, _close, _f64, _i32, _pages, _plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [BF16, F32, F64])
@pytest.mark.parametrize("D", [8, 64, 128, 7, 600])
@pytest.mark.parametrize("eps,size", [(0.0, 1e-19), (0.0, 3e-20), (0.0, 2e-21), (1e-40, 1e-20), (1e-42, 1e-22), (1e-39, 0.0)])
def test_norm_of_small_rows(dt, D, eps, size):
    """Means of squares, with eps, below fp32's normal numbers: a square is off by up to half of its smallest one there, 2^-150, so the
    mean, with eps, by 2^-149 and the inverse root by half of what that is of it."""
    rng = np.random.default_rng(D)
    x = torch.tensor(rng.uniform(0.5, 2, (2, 3, 5, D)) * rng.choice([-1.0, 1.0], (2, 3, 5, D)) * size, device="cuda").to(dt)
    scale = torch.tensor(rng.uniform(0.5, 2, D), device="cuda").to(F64 if dt == F64 else F32)
    g = torch.tensor(rng.uniform(-1, 1, (2, 3, 5, D)) * size, device="cuda").to(dt)
    leaves = x.clone().requires_grad_(True), scale.clone().requires_grad_(True)
    y = A.apply_ago_norm_rotations(leaves[0], None, leaves[1], None, eps=eps)
    dx, dw = torch.autograd.grad(y, leaves, g)
    eps32 = eps if dt == F64 else float(np.float32(eps))
    mean = np.mean(_f64(x) ** 2, -1, keepdims=True) + eps32
    r = 0.0 if dt == F64 else (2.0 ** -149 + 2.0 ** -150) / mean / 2  # relative, of the inverse root
    assert np.max(r) < 0.05
    want, bound = _forward(_f64(x), _f64(scale), eps32, None, None, None, None, dt)
    _close(y, want, bound + 1.1 * r * np.abs(want), "y")
    (wx, bx), (ww, bw) = _backward(_f64(x), _f64(scale), eps32, _f64(g), None, None, None, None, dt)
    # r once in dx, and three times in its second term; a dot product of such g and x is as far down as the squares
    xh, root = np.abs(_f64(x)) / np.sqrt(mean), 1 / np.sqrt(mean)
    part = np.mean(np.abs(_f64(g) * _f64(scale)) * xh, -1, keepdims=True)
    low = 0.0 if dt == F64 else 2 * 2.0 ** -150
    more = 1.2 * r * root * (np.abs(_f64(g) * _f64(scale)) + 3 * xh * part) + 1.1 * root ** 2 * xh * low
    _close(dx, wx, bx + more, "dx")
    _close(dw, ww, bw + 1.1 * np.max(r) * np.sum(np.abs(_f64(g)) * xh, (0, 1, 2)), "dw")


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("D", [64, 40])
def test_small_rows_on_their_way_into_the_cache(dt, D):
    pool = A.PagePool(8, 16, 2, 64)
    plan = _plan(pool, 6, heads=4, kv_heads=2, head_dim=D, dtype=dt)
    A.build_block_tables(plan, _i32([0, 3]), _i32([2, 4]))
    rng = np.random.default_rng(0)
    q, k, v = (torch.tensor(rng.uniform(0.5, 2, (6, h, D)) * 1e-20, device="cuda").to(dt) for h in (4, 2, 2))
    one = torch.ones(D, device="cuda")
    kp, vp = _pages(pool, 2, D, dt)
    out = A.append_to_cache(q, k, v, kp, vp, plan, norms=(one, one), eps=0.0)
    for x, got in ((q, out), (k, torch.stack([kp[s // 16, :, s % 16] for s in plan.slots.tolist()]))):
        x = _f64(x)[None]
        want, bound = _forward(x, np.ones(D), 0.0, None, None, None, None, dt)
        r = (2.0 ** -149 + 2.0 ** -150) / np.mean(x ** 2, -1, keepdims=True) / 2
        _close(got[None], want, bound + 1.1 * r * np.abs(want), "cache")


@pytest.mark.parametrize("dt", [BF16, F32, F64])
@pytest.mark.parametrize("D", [64, 7, 600])
@pytest.mark.parametrize("size", [1e20, 1e37, 2e38])
def test_gradient_of_rows_past_the_range(dt, D, size):
    """Rows whose mean square passes fp32's range give 0, and so do their gradients, whose true values are |g| / |x|; they add nothing to a
    scale's gradient.  Infinities and NaN stay visible."""
    x = torch.full((1, 2, 3, D), size, device="cuda", dtype=dt)
    x[0, 0, 1] = 0.5
    g = torch.full_like(x, 8.0)
    scale = torch.linspace(0.5, 2, D, device="cuda", dtype=F64 if dt == F64 else F32)
    leaves = x.clone().requires_grad_(True), scale.requires_grad_(True)
    y = A.apply_ago_norm_rotations(leaves[0], None, leaves[1], None)
    dx, dw = torch.autograd.grad(y, leaves, g)
    if dt == F64:
        assert torch.isfinite(y).all() and torch.isfinite(dx).all() and torch.isfinite(dw).all()
        return
    rest = torch.ones(1, 2, 3, dtype=torch.bool, device="cuda")
    rest[0, 0, 1] = False
    assert (y[rest] == 0).all() and (dx[rest] == 0).all()
    alone = x[:, :1, 1:2].clone()
    (wx, bx), (ww, bw) = _backward(_f64(alone), _f64(scale), 1e-6, _f64(g[:, :1, 1:2]), None, None, None, None, dt)
    _close(dx[:, :1, 1:2], wx, bx, "the ordinary row")
    _close(dw, ww, bw, "its scale's gradient")
    x[0, 1, 2, 3] = float("inf")
    g[0, 1, 0, 2] = float("nan")
    leaves = x.clone().requires_grad_(True), scale.detach().requires_grad_(True)
    y = A.apply_ago_norm_rotations(leaves[0], None, leaves[1], None)
    dx, dw = torch.autograd.grad(y, leaves, g)
    assert torch.isnan(y[0, 1, 2, 3]) and torch.isnan(dx[0, 1, 2, 3]) and torch.isnan(dx[0, 1, 0, 2]) and torch.isnan(dw[2])
