"""A cache kept small: requests over a budget keep the tokens that attention gives most.

In every layer, ``accumulate_cache_weights`` adds to each cached token what the step's rows gave it, from the denominators that
``paged_tree_afa`` or ``paged_prefix_afa`` returned; once requests are longer than they may be, ``evict_from_cache`` cuts them
back to a budget, layer by layer: each layer keeps tokens of its own choice, and all the same number, so that one pool still
serves them all.  The reference trains only and has no counterpart.

After an eviction a token's place in the cache is no longer its position: ``append_to_cache`` then takes ``positions``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .paged import DraftPlan, PagePool, _expanded, _lengths, _no_gradient, _no_tangents, _refuse, _rows

__all__ = ["accumulate_cache_weights", "evict_from_cache"]


def _weights(pool, weights):
    """The row stride of accumulated weights."""
    if weights.dtype != torch.float32:
        raise TypeError(f"weights must be float32, got {weights.dtype}")
    shape = (pool.max_requests, pool.max_len)
    if weights.shape != shape:
        raise ValueError(f"weights must have shape {shape}, got {tuple(weights.shape)}")
    if weights.device != pool.device:
        _lib.require_device(weights)
        raise ValueError(f"weights must be on the pool's device {pool.device}, got {weights.device}")
    row, one = weights.stride()
    if (one != 1 and shape[1] > 1) or (row < shape[1] and shape[0] > 1):
        raise ValueError("weights need contiguous rows that do not overlap")
    return max(row, shape[1])


def accumulate_cache_weights(q: torch.Tensor, k_pages: torch.Tensor, denominator: torch.Tensor, plan: DraftPlan,
                             weights: torch.Tensor, *, masks: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Add to ``weights`` (max_requests, max_len), fp32, what the step's rows give each token of their request:
    weights[r, j] += sum over rows i that see token j, and heads, of rho(s_ij)^8 / denominator[i, head].

    q (max_tokens, heads, head_dim), ``k_pages`` and ``masks`` are those of the step's attention, and ``denominator``
    (max_tokens, heads) is what it returned, sink and shared prefix included.  The step's own tokens are set rather than
    added to, so that a place needs no clearing when it is taken again.  Requests without new tokens, and those that were not
    served, keep their weights.  A key whose score is -infinity weighs the least there is.  Tokens of a drafted tree that is not
    kept count as rows too: for the accepted ones alone, call it with the plan by which they are stored again.  The sums are formed
    in a fixed order.  Returns weights."""
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or denominator.requires_grad
                                    or weights.requires_grad):
        _no_gradient("accumulate_cache_weights")
    if forward_ad._current_level >= 0:
        _no_tangents("accumulate_cache_weights", q, k_pages, denominator, weights)
    q, sq = _rows(plan, "q", q, plan._q_shape)
    dev = plan.device
    if k_pages.dtype != plan.dtype or k_pages.shape != plan._page_shape or k_pages.device != dev:
        _refuse(plan, "k_pages", k_pages, plan._page_shape)
    page_strides = None
    if not k_pages.is_contiguous():
        at = k_pages.stride()
        if at[3] != 1 and plan.head_dim != 1:
            raise ValueError("k_pages needs a contiguous head dimension")
        page_strides = _lib.pack3(at[0], at[1], at[2])
    shape = (plan.max_tokens, plan.heads)
    if denominator.dtype != _lib.accum_dtype(plan.dtype):
        raise TypeError(f"denominator must be {_lib.accum_dtype(plan.dtype)}, got {denominator.dtype}")
    if denominator.shape != shape or denominator.device != dev:
        raise ValueError(f"denominator must have shape {shape} on {dev}, got {tuple(denominator.shape)} on {denominator.device}")
    denominator = denominator.contiguous()
    row = _weights(plan.pool, weights)
    if masks is not None:
        if plan.max_tree == 0:
            raise ValueError("masks need a plan with max_tree")
        if masks.dtype != torch.int64 or masks.shape != plan.masks.shape or masks.device != dev:
            raise ValueError(f"masks must be int64 of shape {tuple(plan.masks.shape)} on {dev}")
        masks = masks.contiguous()
    with _lib.on_device(dev):
        rc = _lib.lib().afa_paged_weights(
            plan._ref, q.data_ptr(), None if q.is_contiguous() else _lib.pack2(sq[0], sq[1]), k_pages.data_ptr(),
            page_strides, _lib.ptr(masks), denominator.data_ptr(), weights.data_ptr(), row, 0, _lib.ptr(plan._ws),
            plan._ws_bytes, _lib.stream_ptr(dev))
    _lib.check(rc, "afa_paged_weights")
    return weights


def evict_from_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, pool: PagePool, weights: torch.Tensor,
                     cached_lens: torch.Tensor, budget: int, *, first: int = 0,
                     recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cut requests of more than ``budget`` of their ``cached_lens`` (max_requests,) int32 tokens back to it, in one layer.

    Its ``first`` oldest tokens stay, its ``recent`` newest (first + recent at most budget), and of the others those of the
    largest ``weights`` (max_requests, max_len), the lower place among equal ones; NaN counts as the largest.  What stays keeps its
    order and moves to places 0 .. budget - 1 of the request's pages, in place in ``k_pages`` and ``v_pages`` (num_pages,
    kv_heads, page_size, head_dim); pages of k and v that share places are refused, as far as addresses and strides tell.  Places
    behind the budget keep their contents; pages go back to the pool with the next ``build_block_tables`` for the lengths that this
    returns.  A length is taken as at most what the request's pages hold.

    Returns (lens, weights): the lengths, (max_requests,) int32, and a new (max_requests, max_len) tensor of what the
    tokens that stay had, 0 behind them.  With the same budget every layer of a pool returns the same lengths."""
    if torch.is_grad_enabled() and (k_pages.requires_grad or v_pages.requires_grad or weights.requires_grad):
        _no_gradient("evict_from_cache")
    if forward_ad._current_level >= 0:
        _no_tangents("evict_from_cache", k_pages, v_pages, weights)
    dev = pool.device
    dt = _lib.dtype_code(k_pages.dtype)
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.ndim != 4 or t.shape[0] != pool.num_pages or t.shape[2] != pool.page_size or min(t.shape) < 1:
            raise ValueError(f"{name} must have shape ({pool.num_pages}, kv_heads, {pool.page_size}, head_dim), got "
                             f"{tuple(t.shape)}")
        if t.device != dev:
            _lib.require_device(t)
            raise ValueError(f"{name} must be on the pool's device {dev}, got {t.device}")
    if v_pages.dtype != k_pages.dtype or v_pages.shape != k_pages.shape:
        raise ValueError(f"k_pages and v_pages must be alike, got {tuple(k_pages.shape)} {k_pages.dtype} and "
                         f"{tuple(v_pages.shape)} {v_pages.dtype}")
    _, kv_heads, _, head_dim = k_pages.shape
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    page_strides = None
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        _expanded("k_pages", k_pages)
        _expanded("v_pages", v_pages)
        k, v = k_pages.stride(), v_pages.stride()
        if (k[3] != 1 or v[3] != 1) and head_dim != 1:
            raise ValueError("k_pages and v_pages need a contiguous head dimension")
        page_strides = _lib.pack6(k[0], k[1], k[2], v[0], v[1], v[2])
    elif abs(kp - vp) < k_pages.numel() * k_pages.element_size():
        raise ValueError("k_pages and v_pages must not overlap")
    if kp == vp:
        raise ValueError("k_pages and v_pages must not overlap")
    cached_lens = _lengths("cached_lens", cached_lens, dev, (pool.max_requests,))
    row = _weights(pool, weights)
    for name, n in (("budget", budget), ("first", first), ("recent", recent)):
        if int(n) != n or n < 0:
            raise ValueError(f"{name} must be a nonnegative integer, got {n}")
    if budget < 1 or first + recent > budget:
        raise ValueError(f"the budget ({budget}) must be positive and hold the first ({first}) and the recent ({recent}) tokens")
    budget = min(int(budget), pool.max_len)
    first = min(int(first), budget)
    recent = min(int(recent), budget - first)
    lens = torch.empty(pool.max_requests, dtype=torch.int32, device=dev)
    left = torch.empty((pool.max_requests, pool.max_len), dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        size = _lib.workspace_size("afa_paged_evict_workspace_size", dev, pool.max_requests, pool.max_len, budget,
                                   kv_heads, head_dim)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        rc = _lib.lib().afa_paged_evict(
            dt, pool.num_pages, pool.page_size, pool.max_requests, pool.block_tables.shape[1], kv_heads, head_dim,
            pool.block_tables.data_ptr(), pool.held.data_ptr(), kp, vp, page_strides, cached_lens.data_ptr(), budget, first,
            recent, weights.data_ptr(), row, left.data_ptr(), lens.data_ptr(), ws.data_ptr(), size, _lib.stream_ptr(dev))
    _lib.check(rc, "afa_paged_evict")
    return lens, left
