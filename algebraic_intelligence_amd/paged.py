"""Serving with AFA: drafted trees of tokens over a paged key/value cache.

A serving step is one ``build_block_tables`` for the whole model and, in every layer, one
``append_to_cache`` (q and k normalised and rotated, k and v stored) and one ``paged_tree_afa``, or one
``paged_prefix_afa`` where all requests share a prefix that no page holds.  Nothing in a step
needs the lengths on the host, so a step of fixed sizes can be captured into a HIP graph and replayed
with other lengths, parents and activations in the same tensors.  The reference trains only and has
no counterpart; the attention is its AFA (src/kernels/pallas_afa.py:104-151) over other keys.

``PagePool`` holds which pages belong to which request; ``DraftPlan`` the buffers of one step, the
attention's partial sums among them.  Calls that share a plan must be ordered on one stream (or by
events); steps that run at the same time need a plan each.  The pool is brought up to date by one
``build_block_tables`` at a time, and the calls of a plan read its block tables: a plan is good until
another one is built on its pool.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from .attention import _axis_sections, _axis_tables, _norm_eps, _norm_scale

__all__ = ["PagePool", "DraftPlan", "build_block_tables", "append_to_cache", "paged_tree_afa", "paged_prefix_afa"]


class _Plan(ctypes.Structure):
    """afa_paged_plan of include/afa.h."""

    _fields_ = ([(n, ctypes.c_int64) for n in ("num_pages", "page_size", "requests", "table_width", "max_tokens", "max_new",
                                               "max_tree", "heads", "kv_heads", "head_dim", "dtype")]
                + [(n, ctypes.c_void_p) for n in ("block_tables", "held", "ring", "ring_state", "slots", "positions",
                                                  "token_request", "starts", "status", "masks", "schedule")])


def _device(device) -> torch.device:
    if device is None:
        if not torch.cuda.is_available():
            raise RuntimeError("the paged cache lives on the GPU, and no HIP device is visible")
        return torch.device("cuda", torch.cuda.current_device())
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError(f"the AFA kernels run on the GPU: the paged cache needs a HIP device, got {device}")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


def _positive(**sizes):
    for name, n in sizes.items():
        if int(n) != n or n <= 0:
            raise ValueError(f"{name} must be a positive integer, got {n}")


class PagePool:
    """The pages of a cache and the requests that hold them.

    ``num_pages`` pages of ``page_size`` tokens serve up to ``max_requests`` requests of up to
    ``max_len`` tokens each.  One pool serves all layers of a model: a page has the same id in each
    layer's (num_pages, kv_heads, page_size, head_dim) k and v arrays (``new_pages``).

    ``block_tables`` (max_requests, pages of max_len) int32: request r's pages in order, -1 behind
    them; ``held`` (max_requests,) int32: how many; ``ring`` (num_pages,) int32 and ``ring_state``
    (2,) int32 = (head, count): the free pages, a queue that starts at ring[head].  All on the
    device and brought up to date in place by ``build_block_tables``.
    """

    def __init__(self, num_pages: int, page_size: int, max_requests: int, max_len: int, *, device=None):
        _positive(num_pages=num_pages, page_size=page_size, max_requests=max_requests, max_len=max_len)
        self.num_pages, self.page_size, self.max_requests = int(num_pages), int(page_size), int(max_requests)
        width = -(-int(max_len) // self.page_size)
        if self.num_pages * self.page_size >= 1 << 31 or width * self.page_size > 1 << 30:
            raise ValueError("a pool holds fewer than 2^31 tokens and a request at most 2^30")
        self.max_len = width * self.page_size
        self.device = _device(device)
        new = {"dtype": torch.int32, "device": self.device}
        self.block_tables = torch.full((self.max_requests, width), -1, **new)
        self.held = torch.zeros(self.max_requests, **new)
        self.ring = torch.arange(self.num_pages, **new)
        self.ring_state = torch.tensor([0, self.num_pages], **new)

    def new_weights(self) -> torch.Tensor:
        """The accumulated attention weights of one layer's cached tokens, (max_requests, max_len) in fp32, 0."""
        return torch.zeros((self.max_requests, self.max_len), dtype=torch.float32, device=self.device)

    def new_pages(self, kv_heads: int, head_dim: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
        """k and v pages of one layer, (num_pages, kv_heads, page_size, head_dim) each, not initialised."""
        _lib.dtype_code(dtype)
        shape = (self.num_pages, kv_heads, self.page_size, head_dim)
        return torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)


class DraftPlan:
    """The buffers of a serving step over ``pool`` for layers of ``heads`` query and ``kv_heads``
    key/value heads of ``head_dim`` features in ``dtype``.

    ``max_tokens`` rows hold the new tokens of all requests, packed in request order; one request has
    at most ``max_new`` of them (default: max_tokens).  ``max_tree`` (0, or a multiple of 64 up to 256)
    is the most nodes of a drafted tree; requests with more new tokens are prompts, whose tokens
    follow one another.

    After ``build_block_tables``: ``slots`` (max_tokens,) int32 page * page_size + offset of each token,
    -1 where it has none; ``positions`` (max_tokens,) int32 cached tokens + depth in the tree;
    ``requests`` (max_tokens,) int32, -1 behind the last request's tokens; ``starts`` (R + 1,) int32 the
    requests' first rows; ``status`` (R,) int32, 0 or why a request was not served (include/afa.h,
    AFA_PAGED_*: 1 too few free pages, 2 longer than max_len, 3 more than max_new, 4 past max_tokens, 5 a negative
    length); ``masks`` (max_tokens, max_tree / 64) int64, bit i of a row's words: the row sees
    drafted token i of its request (None without trees).
    """

    def __init__(self, pool: PagePool, max_tokens: int, *, heads: int, kv_heads: Optional[int] = None, head_dim: int,
                 dtype: torch.dtype, max_new: Optional[int] = None, max_tree: int = 64):
        kv_heads = heads if kv_heads is None else kv_heads
        max_new = max_tokens if max_new is None else max_new  # a request cannot have more than all
        _positive(max_tokens=max_tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, max_new=max_new)
        if heads % kv_heads != 0:
            raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
        max_new = min(max_new, max_tokens)
        if max_tree not in (0, 64, 128, 192, 256):
            raise ValueError(f"max_tree must be 0, 64, 128, 192 or 256, got {max_tree}")
        self.pool, self.dtype = pool, dtype
        self.max_tokens, self.heads, self.kv_heads, self.head_dim = int(max_tokens), int(heads), int(kv_heads), int(head_dim)
        self.max_tree = int(max_tree)
        dev = self.device = pool.device
        self._q_shape = (self.max_tokens, self.heads, self.head_dim)
        self._kv_shape = (self.max_tokens, self.kv_heads, self.head_dim)
        self._page_shape = (pool.num_pages, self.kv_heads, pool.page_size, self.head_dim)
        self._q_bytes = self.max_tokens * self.heads * self.head_dim * dtype.itemsize
        self._page_bytes = pool.num_pages * self.kv_heads * pool.page_size * self.head_dim * dtype.itemsize
        self._len_shape = (pool.max_requests,)
        c = self._c = _Plan(num_pages=pool.num_pages, page_size=pool.page_size, requests=pool.max_requests,
                            table_width=pool.block_tables.shape[1], max_tokens=max_tokens, max_new=max_new,
                            max_tree=max_tree, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=_lib.dtype_code(dtype))
        self._ref = ctypes.byref(c)
        with _lib.on_device(dev):
            schedule = _lib.lib().afa_paged_schedule_bytes(self._ref)
            if schedule == 0:
                raise ValueError("a plan of these sizes is not supported")
            self._ws_bytes = _lib.lib().afa_paged_workspace_size(self._ref)
        ints = {"dtype": torch.int32, "device": dev}
        self.slots = torch.full((self.max_tokens,), -1, **ints)
        self.positions = torch.zeros(self.max_tokens, **ints)
        self.requests = torch.full((self.max_tokens,), -1, **ints)
        self.starts = torch.zeros(pool.max_requests + 1, **ints)
        self.status = torch.zeros(pool.max_requests, **ints)
        self.masks = torch.zeros((self.max_tokens, max_tree // 64), dtype=torch.int64, device=dev) if max_tree else None
        # zeros: a plan without a step has no items
        self._schedule = torch.zeros(schedule // 4, **ints)
        # the attention's partial sums; calls that share a plan are ordered, so they share these too
        self._ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=dev) if self._ws_bytes else None
        for name, t in (("block_tables", pool.block_tables), ("held", pool.held), ("ring", pool.ring),
                        ("ring_state", pool.ring_state), ("slots", self.slots), ("positions", self.positions),
                        ("token_request", self.requests), ("starts", self.starts), ("status", self.status),
                        ("masks", self.masks), ("schedule", self._schedule)):
            setattr(c, name, _lib.ptr(t))

    @property
    def max_new(self) -> int:
        return self._c.max_new


def _lengths(name, t, dev, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != dev:
        _lib.require_device(t)
        raise ValueError(f"{name} must be on the plan's device {dev}, got {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def build_block_tables(plan: DraftPlan, cached_lens: torch.Tensor, new_lens: torch.Tensor,
                       parents: Optional[torch.Tensor] = None) -> DraftPlan:
    """Plan a step: ``cached_lens`` tokens of each request are in the cache and ``new_lens`` come
    now, (max_requests,) int32 each.  Every request is given exactly the pages of both; pages beyond
    them go back to the pool, where the next call finds them, so a length of 0 + 0 ends a request.  A
    request that cannot be served (``plan.status``) keeps what it held, and its tokens get no slots.

    ``parents`` (max_tokens,) int32: for each new token, the index among its request's new tokens of
    the one it follows, or -1 where it follows the cached ones (also taken for a value that is no earlier
    token).  Without it, and in requests of more than max_tree tokens, each token follows the one
    before it.  Returns the plan; nothing is read back to the host."""
    pool = plan.pool
    dev = pool.device
    cached_lens = _lengths("cached_lens", cached_lens, dev, plan._len_shape)
    new_lens = _lengths("new_lens", new_lens, dev, plan._len_shape)
    if parents is not None:
        if plan.max_tree == 0:
            raise ValueError("parents need a plan with max_tree")
        parents = _lengths("parents", parents, dev, (plan.max_tokens,))
    with _lib.on_device(dev):
        rc = _lib.lib().afa_paged_build(plan._ref, cached_lens.data_ptr(), new_lens.data_ptr(), _lib.ptr(parents),
                                        _lib.stream_ptr(dev))
    _lib.check(rc, "afa_paged_build")
    return plan


def _no_gradient(name):
    raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or with detached tensors")


def _no_tangents(name, *tensors):
    """Refuses tensors that carry a tangent, within a forward-mode level."""
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no derivative, and a tensor carries a tangent")


def _pages(plan, k_pages, v_pages):
    """Strides of the pages (page, head, slot of k, then of v), None where both are contiguous."""
    dt, shape, dev = plan.dtype, plan._page_shape, plan.device
    if k_pages.dtype != dt or k_pages.shape != shape or k_pages.device != dev:
        _refuse(plan, "k_pages", k_pages, shape)
    if v_pages.dtype != dt or v_pages.shape != shape or v_pages.device != dev:
        _refuse(plan, "v_pages", v_pages, shape)
    if k_pages.is_contiguous() and v_pages.is_contiguous():
        return None
    k, v = k_pages.stride(), v_pages.stride()
    if (k[3] != 1 or v[3] != 1) and plan.head_dim != 1:
        raise ValueError("k_pages and v_pages need a contiguous head dimension")
    return _lib.pack6(k[0], k[1], k[2], v[0], v[1], v[2])


def _rows(plan, name, t, shape):
    """t, of the plan's dtype and device and of shape (max_tokens, heads, head_dim), with a contiguous head dimension,
    and its strides."""
    if t.dtype != plan.dtype or t.shape != shape or t.device != plan.device:
        _refuse(plan, name, t, shape)
    at = t.stride()
    if at[2] != 1 and plan.head_dim != 1:
        t = t.contiguous()
        at = t.stride()
    return t, at


def _like_rows(q):
    """An empty contiguous tensor like q."""
    y = torch.empty_like(q)  # half the time of torch.empty
    return y if y.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)


def _meet(out, t, contiguous, out_bytes, bytes_):
    """Whether the address ranges of out, which is contiguous, and t meet."""
    a, b = out.data_ptr(), t.data_ptr()
    if not contiguous:
        bytes_ = t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))
    return a < b + bytes_ and b < a + out_bytes


def _expanded(name, t):
    if any(st == 0 and n > 1 for n, st in zip(t.shape, t.stride())):
        raise ValueError(f"{name} must not be an expanded tensor")


def _refuse(plan, name, t, shape):
    if t.dtype != plan.dtype:
        raise TypeError(f"{name} must be {plan.dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    _lib.require_device(t)
    raise ValueError(f"{name} must be on the plan's device {plan.device}, got {t.device}")


def append_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    plan: DraftPlan, rotary_params=None, *, positions: Optional[torch.Tensor] = None,
                    sections=None, norms=None, eps: float = 1e-6) -> torch.Tensor:
    """Rotate the step's q (max_tokens, heads, head_dim) and k (max_tokens, kv_heads, head_dim), store k and v
    at the tokens' slots of ``k_pages`` and ``v_pages``, and return the rotated q.

    ``norms``: (q_scale, k_scale), (head_dim,) each; q and k are normalised, scaled and then rotated as in
    ``apply_ago_norm_rotations``, with its ``eps``, in the same launch.

    ``rotary_params``: Cayley tables (positions, head_dim / 2), in fp32 (fp64 for fp64 inputs; others are
    cast); a position outside them gives NaN.  None: k is stored and q returned as they are.
    ``positions`` (max_tokens, A) int32 with ``sections`` gives positions of A axes as in
    ``apply_ago_axis_rotations``; (max_tokens,) or None, the plan's positions, is one axis.  Tokens
    without a slot are not stored.  The pages hold k and v in places of their own, apart from q, k and v: k_pages and v_pages
    that share places are refused, as far as addresses and strides tell.
    For inference: inputs that require a gradient are refused where gradients are recorded."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_pages.requires_grad
                                    or v_pages.requires_grad):
        _no_gradient("append_to_cache")
    if forward_ad._current_level >= 0:
        _no_tangents("append_to_cache", q, k, v, k_pages, v_pages)
    if norms is not None:
        eps = _norm_eps(eps)
        if not isinstance(norms, (tuple, list)) or len(norms) != 2:
            raise TypeError("norms must be a pair (q_scale, k_scale)")
        q_scale = _norm_scale("q_scale", norms[0], plan.head_dim, plan.dtype, plan.device)
        k_scale = _norm_scale("k_scale", norms[1], plan.head_dim, plan.dtype, plan.device)
        if torch.is_grad_enabled() and (q_scale.requires_grad or k_scale.requires_grad):
            _no_gradient("append_to_cache")
        if forward_ad._current_level >= 0:
            _no_tangents("append_to_cache", q_scale, k_scale)
    (q, sq), (k, sk), (v, sv) = (_rows(plan, "q", q, plan._q_shape), _rows(plan, "k", k, plan._kv_shape),
                                 _rows(plan, "v", v, plan._kv_shape))
    page_strides = _pages(plan, k_pages, v_pages)
    # two of a step's rows must not be written to one place, as far as addresses and strides tell
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if kp == vp or (page_strides is None and abs(kp - vp) < plan._page_bytes):
        raise ValueError("k_pages and v_pages must not overlap")
    if page_strides is not None:
        _expanded("k_pages", k_pages)
        _expanded("v_pages", v_pages)
    dev = plan.device
    c = s = None
    axes, cuts = 1, None
    q_out = q
    if rotary_params is not None:
        c, s = _axis_tables(rotary_params, plan.head_dim, plan.dtype, dev)
        if positions is not None:
            axes = 1 if positions.ndim == 1 else positions.shape[-1]
            shape = (plan.max_tokens,) if positions.ndim == 1 else (plan.max_tokens, axes)
            positions = _lengths("positions", positions, dev, shape)
        cuts = _axis_sections(sections, axes, plan.head_dim // 2)
        q_out = _like_rows(q)
    elif positions is not None or sections is not None:
        raise ValueError("positions and sections need rotary_params")
    strides = None
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        strides = _lib.pack6(sq[0], sq[1], sk[0], sk[1], sv[0], sv[1])
    if norms is not None:
        if c is None:
            q_out = _like_rows(q)
        with _lib.on_device(dev):
            rc = _lib.lib().afa_paged_append_norm(
                plan._ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, q_out.data_ptr(), kp, vp, page_strides,
                q_scale.data_ptr(), k_scale.data_ptr(), eps, _lib.ptr(c), _lib.ptr(s), 0 if c is None else c.shape[0],
                _lib.ptr(positions), axes, cuts, _lib.stream_ptr(dev))
        _lib.check(rc, "afa_paged_append_norm")
        return q_out
    with _lib.on_device(dev):
        rc = _lib.lib().afa_paged_append(
            plan._ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, None if c is None else q_out.data_ptr(),
            kp, vp, page_strides, _lib.ptr(c), _lib.ptr(s), 0 if c is None else c.shape[0],
            _lib.ptr(positions), axes, cuts, _lib.stream_ptr(dev))
    _lib.check(rc, "afa_paged_append")
    return q_out


def paged_tree_afa(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, plan: DraftPlan, sink_omega: float = 0.5,
                   *, masks: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   return_denominator: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """AFA of the step's tokens over the cache: row i of a request, q (max_tokens, heads, head_dim), sees its
    request's cached tokens and the drafted ones of its mask, which ``append_to_cache`` has stored.

    Returns out (max_tokens, heads, head_dim), or (out, d) with d = sum_j rho(s_ij)^8 + sink_omega of shape
    (max_tokens, heads) in fp32 (fp64 for fp64 inputs).  heads / kv_heads query heads share a key/value
    head.  ``masks`` replaces the plan's (max_tokens, max_tree / 64) int64 masks: they hide drafted tokens
    only, and none in requests of more than max_tree new tokens.  A row that sees no key is 0, and a key
    that a row does not see, whatever its page holds, does not touch it; an infinity or a NaN in a value
    that it sees is its result in that feature.  Rows behind the last request's are 0, or left as they
    were where ``out`` is given.  For inference: tensors that require a gradient are refused where gradients
    are recorded."""
    return _attend("paged_tree_afa", q, None, k_pages, v_pages, plan, sink_omega, masks, out, return_denominator)


def paged_prefix_afa(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k_pages: torch.Tensor,
                     v_pages: torch.Tensor, plan: DraftPlan, sink_omega: float = 0.5, *, masks: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None,
                     return_denominator: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``paged_tree_afa`` of requests that begin with the same tokens: every row sees the keys and values of
    ``k_prefix`` and ``v_prefix`` (kv_heads, prefix length, head_dim), of any strides with a contiguous head
    dimension, and then its request's cached and drafted tokens.

    The prefix is kept once and met once for all rows of the step, whatever the number of requests.  The pool's lengths count a
    request's own tokens, so that the positions of ``append_to_cache`` are the plan's plus the prefix's length:
    ``positions=plan.positions + k_prefix.shape[1]``.  The plan, q, masks, out and what is returned are as in
    ``paged_tree_afa``; rows of requests that were not served are 0.

    A plan of more than 64 rows a key head (max_tokens * heads / kv_heads) with bf16 or fp16 and head_dim up to 128 rounds the
    weights over the prefix to that type once, in all of its steps; others, and the weights of the requests' own keys, keep
    twice its digits.  In fp16 a weight far below a row's largest is off by up to 2^-29 of that: very many such keys, 2^18 and
    more, can be seen in the result."""
    return _attend("paged_prefix_afa", q, (k_prefix, v_prefix), k_pages, v_pages, plan, sink_omega, masks, out,
                   return_denominator)


def _prefix(plan, k_prefix, v_prefix):
    """The prefix's strides (head and key of k, then of v), None where both are contiguous, and its length."""
    if k_prefix.ndim != 3 or k_prefix.shape[1] < 1 or k_prefix.shape[1] > 1 << 29:
        raise ValueError(f"k_prefix must have shape ({plan.kv_heads}, length, {plan.head_dim}) with a length of 1 to 2^29, got "
                         f"{tuple(k_prefix.shape)}")
    shape = (plan.kv_heads, k_prefix.shape[1], plan.head_dim)
    for name, t in (("k_prefix", k_prefix), ("v_prefix", v_prefix)):
        if t.dtype != plan.dtype or t.shape != shape or t.device != plan.device:
            _refuse(plan, name, t, shape)
    if k_prefix.is_contiguous() and v_prefix.is_contiguous():
        return None, shape[1]
    k, v = k_prefix.stride(), v_prefix.stride()
    if (k[2] != 1 or v[2] != 1) and plan.head_dim != 1:
        raise ValueError("k_prefix and v_prefix need a contiguous head dimension")
    return _lib.pack4(k[0], k[1], v[0], v[1]), shape[1]


def _attend(name, q, prefix, k_pages, v_pages, plan, sink_omega, masks, out, return_denominator):
    if not 0.0 <= sink_omega < float("inf"):
        raise ValueError("sink_omega must be finite and nonnegative")
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad
                                    or (out is not None and out.requires_grad)
                                    or (prefix is not None and (prefix[0].requires_grad or prefix[1].requires_grad))):
        _no_gradient(name)
    if forward_ad._current_level >= 0:
        _no_tangents(name, q, k_pages, v_pages, *(prefix or ()))
    q, sq = _rows(plan, "q", q, plan._q_shape)
    page_strides = _pages(plan, k_pages, v_pages)
    if prefix is not None:
        prefix_strides, length = _prefix(plan, *prefix)
    dev = plan.device
    if masks is not None:
        if plan.max_tree == 0:
            raise ValueError("masks need a plan with max_tree")
        if masks.dtype != torch.int64 or masks.shape != plan.masks.shape or masks.device != dev:
            raise ValueError(f"masks must be int64 of shape {tuple(plan.masks.shape)} on {dev}")
        masks = masks.contiguous()
    strides = None if q.is_contiguous() else _lib.pack2(sq[0], sq[1])
    flags = 0
    if out is None:
        out = torch.empty_like(q) if strides is None else _like_rows(q)
        flags = _lib.FLAG_ZERO_TAIL
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous, of shape {tuple(q.shape)}, {q.dtype} on {dev}")
    elif (_meet(out, q, strides is None, plan._q_bytes, plan._q_bytes)
          or _meet(out, k_pages, page_strides is None, plan._q_bytes, plan._page_bytes)
          or _meet(out, v_pages, page_strides is None, plan._q_bytes, plan._page_bytes)):
        raise ValueError("out must not overlap q, k_pages or v_pages")
    elif prefix is not None and any(_meet(out, t, False, plan._q_bytes, 0) for t in prefix):
        raise ValueError("out must not overlap k_prefix or v_prefix")
    den = None
    if return_denominator:
        new = torch.empty if flags else torch.zeros
        den = new((plan.max_tokens, plan.heads), dtype=_lib.accum_dtype(q.dtype), device=dev)
    if prefix is not None:
        with _lib.on_device(dev):
            size = _lib.lib().afa_paged_prefix_workspace_size(plan._ref, length)
            ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
            rc = _lib.lib().afa_paged_prefix_fwd(
                plan._ref, q.data_ptr(), strides, prefix[0].data_ptr(), prefix[1].data_ptr(), length, prefix_strides,
                k_pages.data_ptr(), v_pages.data_ptr(), page_strides, _lib.ptr(masks), out.data_ptr(), _lib.ptr(den),
                sink_omega, flags, _lib.ptr(ws), size, _lib.stream_ptr(dev))
        _lib.check(rc, "afa_paged_prefix_fwd")
        return (out, den) if return_denominator else out
    with _lib.on_device(dev):
        rc = _lib.lib().afa_paged_fwd(
            plan._ref, q.data_ptr(), strides, k_pages.data_ptr(), v_pages.data_ptr(), page_strides, _lib.ptr(masks),
            out.data_ptr(), _lib.ptr(den), sink_omega, flags, _lib.ptr(plan._ws), plan._ws_bytes, _lib.stream_ptr(dev))
    _lib.check(rc, "afa_paged_fwd")
    return (out, den) if return_denominator else out
