"""More operators by which this framework's speed is followed: normalised heads, a prompt that a whole batch
shares, and a cache that is kept small.

One case is one call (a norm in training: the call and its gradients) of

  norm     ``apply_ago_norm_rotations``: q and k normalised head by head, scaled and rotated;
  append   ``append_to_cache`` with norms: the same of a step's new tokens, and k and v stored in their slots;
  prefix   ``paged_prefix_afa``: the new tokens' attention over a prefix that all requests share, and over
           their own cached and drafted tokens;
  weights  ``accumulate_cache_weights``: what each cached token was given by the step's rows, added up;
  evict    ``evict_from_cache``: requests over a budget keep their tokens of the largest weights.

``prepare`` makes what a serving or training program holds before the call: activations, scales, pages,
Cayley tables, the shared prefix's keys and values, accumulated weights, and the pool and plan that it keeps between
steps.  Pages and weights are brought up to date in place.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = torch.device("cuda")
_EPS = 1e-6
_OMEGA = 0.5


# -------------------------------------------------------------------------------------- cases
def _norm(mode, batch, heads, kv_heads, seq, head_dim, sections, dtype):
    return {"kind": "norm", "mode": mode, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq": seq,
            "head_dim": head_dim, "sections": sections, "dtype": dtype}


def _step(kind, requests, context, new, tree, heads, kv_heads, head_dim, page, dtype, spread=True, **more):
    """Cached lengths run from about context / 8 to context, and new ones from new / 2 to new, where they spread."""
    return {"kind": kind, "requests": requests, "context": context, "new": new, "tree": tree, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "spread": spread, **more}


def _evict(requests, context, budget, first, recent, kv_heads, head_dim, page, dtype):
    return {"kind": "evict", "requests": requests, "context": context, "new": 0, "tree": 0, "heads": kv_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "spread": True, "budget": budget,
            "first": first, "recent": recent}


def listed():
    return [
        # The new tokens of a small decoding step on their way into the cache: latency.
        {"name": "append_norm_step", **_step("append", 24, 4096, 1, 0, 12, 12, 64, 64, "bf16", sections="32")},
        # Storing the prompts of a batch, grouped heads.
        {"name": "append_norm_prompts", **_step("append", 8, 64, 2048, 0, 16, 4, 128, 32, "fp16", False, sections="64")},
        # Training the 125M model's layer on a batch of 4096-token sequences.
        {"name": "norm_train_4k", **_norm("train", 8, 12, 12, 4096, 64, "32", "bf16")},
        # A video clip in full precision (time, height, width), grouped heads, an odd length.
        {"name": "norm_train_video_f32", **_norm("train", 1, 16, 4, 8189, 128, "16,24,24", "fp32")},
        # A few requests that begin with one short instruction: the smallest call of a shared prefix.
        {"name": "prefix_token", **_step("prefix", 4, 200, 1, 0, 12, 12, 64, 64, "bf16", prefix=1000)},
        # A large batch of single tokens behind one long system prompt.
        {"name": "prefix_steps", **_step("prefix", 256, 512, 1, 0, 16, 4, 128, 64, "bf16", prefix=8192)},
        # Speculative decoding of many questions about one long document.
        {"name": "prefix_drafts", **_step("prefix", 32, 2048, 32, 64, 16, 4, 128, 64, "fp16", prefix=30001)},
        # The pilot model's heads (6 of 48) in full precision, ragged.
        {"name": "prefix_pilot_f32", **_step("prefix", 20, 301, 5, 0, 6, 6, 48, 32, "fp32", prefix=3001)},
        # Following the weights of a batch of single tokens over up to 8k.
        {"name": "weights_steps", **_step("weights", 64, 8192, 1, 0, 16, 4, 128, 64, "bf16")},
        # The weights that a batch of prompts leaves on its own tokens.
        {"name": "weights_prompts", **_step("weights", 8, 64, 2048, 0, 12, 12, 64, 32, "bf16", False)},
        # A batch of requests of up to 8k cut back to 2048 tokens each.
        {"name": "evict_batch", **_evict(64, 8192, 2048, 4, 512, 4, 128, 64, "bf16")},
        # Few long documents, of up to 128k, cut back to a quarter.
        {"name": "evict_long", **_evict(4, 131072, 32768, 64, 4096, 4, 128, 128, "fp16")},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "append", "prefix", "prefix", "prefix", "weights", "weights", "evict", "evict"])
    page = rng.choice([16, 32, 64, 128])
    D = rng.choice([48, 64, 96, 128])
    kv = rng.choice([2, 4, 6, 8, 12])
    group = rng.choice([1, 1, 2, 4])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    tree = 64 if rng.random() < 0.5 else 0
    cut = rng.choice([[4], [4], [1, 3], [1, 1, 2], [2, 1, 1]])
    sections = ",".join(str(D // 8 * c) for c in cut)
    if kind == "norm":
        tokens = max(1, _log_int(rng, 16, 32768) * 24 // (kv * (group + 1)) * 64 // D // (2 if dtype == "fp32" else 1))
        seq = min(tokens, _log_int(rng, 1, 8192))
        return _norm(rng.choice(["forward", "train", "train"]), max(1, tokens // seq), kv * group, kv, seq, D, sections, dtype)
    if kind == "append":
        new = _log_int(rng, 1, 1024)
        requests = max(1, min(64, _log_int(rng, 1, 8192) // new))
        return _step(kind, requests, _log_int(rng, 16, 2048), new, tree if new <= 64 else 0, kv * group, kv, D, page, dtype,
                     sections=sections)
    if kind == "evict":
        context = _log_int(rng, 64, 131072)
        requests = max(1, min(96, 4 * 131072 * 4 * 128 // (context * kv * D * (2 if dtype == "fp32" else 1)), _log_int(rng, 1, 96)))
        budget = max(1, int(context * rng.uniform(0.1, 0.9)))
        first, recent = rng.randint(0, min(64, budget // 2)), rng.randint(0, budget // 2)
        return _evict(requests, context, budget, first, recent, kv, D, page, dtype)
    if kind == "weights" and rng.random() < 0.4:
        new = _log_int(rng, 65, 2048)
        requests = max(1, min(16, _log_int(rng, 1, 16), 8 * 2048 * 2048 * 12 // (new * new * kv * group)))
        return _step(kind, requests, rng.randint(1, 256), new, 0, kv * group, kv, D, page, dtype)
    new = _log_int(rng, 1, 40)
    context = _log_int(rng, 16, 8192)
    # no more cached elements than 64 requests of up to 8k hold in 4 heads of 128
    most = 64 * 8192 * 4 * 128 // (context * kv * D)
    requests = max(1, min(256, most, _log_int(rng, 1, 256), 1024 // new))
    case = _step(kind, requests, context, new, tree, kv * group, kv, D, page, dtype)
    if kind == "prefix":
        # no more products than the many questions about one document need
        most = 32 * 32 * 30001 * 16 * 128 // (requests * new * kv * group * D * (4 if dtype == "fp32" else 1))
        case["prefix"] = max(1, min(most, _log_int(rng, 16, 65536)))
    return case


def _lens(case):
    """(cached, new) tokens of each request: the case's alone, whatever the seed."""
    rng = random.Random(case["requests"] * 7919 + case["context"])
    cached, new = [], []
    for _ in range(case["requests"]):
        cached.append(rng.randint(max(1, case["context"] // 8), case["context"]) if case["spread"] else case["context"])
        new.append(rng.randint((case["new"] + 1) // 2, case["new"]) if case["spread"] else case["new"])
    return cached, new


def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def work(case):
    esz = 4 if case["dtype"] == "fp32" else 2
    D, H, K = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "norm":
        # x in and y out; in training x and the cotangent in again and the gradient out
        per = case["batch"] * case["seq"] * (H + K) * D
        train = case["mode"] == "train"
        return {"bytes": (5 if train else 2) * per * esz, "flops": (18 if train else 7) * per}
    cached, new = _lens(case)
    T = sum(new)
    if case["kind"] == "append":
        return {"bytes": 2 * T * (H + 2 * K) * D * esz, "flops": 7 * T * (H + K) * D}
    if case["kind"] == "evict":
        kept = [min(c, case["budget"]) for c in cached]
        moved = sum(k for k, c in zip(kept, cached) if c > k)
        return {"bytes": 4 * moved * K * D * esz + 4 * (sum(cached) + sum(kept)), "flops": sum(cached)}
    keys = sum(c + n for c, n in zip(cached, new))
    pairs = sum(n * (c + (1 if case["tree"] else (n + 1) / 2)) for c, n in zip(cached, new))
    if case["kind"] == "weights":
        return {"bytes": keys * K * D * esz + T * H * (D * esz + 4) + 8 * keys, "flops": 2 * pairs * H * D}
    return {"bytes": (2 * (keys + case["prefix"]) * K + 2 * T * H) * D * esz,
            "flops": 4 * (pairs + T * case["prefix"]) * H * D}


# ------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed))


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device=_DEV).to(dtype)


def _scale(D, g):
    """A norm's learned scale, in the full precision that a program keeps it in."""
    return 1 + 0.2 * torch.randn(D, generator=g, device=_DEV)


def _rotary(rows, head_dim):
    """Cayley tables (c, s) in fp32: row m turns pair k by 2 m atan(w_k), w_k = 1 / (1 + alpha k)^2."""
    pairs = head_dim // 2
    alpha = (math.sqrt(10000.0) - 1.0) / max(pairs - 1, 1)
    k = torch.arange(pairs, dtype=torch.float64, device=_DEV)
    m = torch.arange(rows, dtype=torch.float64, device=_DEV)
    ang = 2.0 * m[:, None] * torch.atan(1.0 / (1.0 + alpha * k) ** 2)[None, :]
    return torch.cos(ang).float(), torch.sin(ang).float()


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _plan_step(case, seed):
    """A serving step: lengths, each request's pages in random order, and where its new tokens belong."""
    cached, new = _lens(case)
    rng = np.random.default_rng(seed)
    P, R = case["page"], case["requests"]
    width = -(-(case["context"] + case["new"]) // P) + 1
    need = [-(-(c + n) // P) for c, n in zip(cached, new)]
    pages = sum(need) + R
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((R, width), -1, np.int32)
    at = 0
    for r, h in enumerate(need):
        table[r, :h] = order[at:at + h]
        at += h
    starts = np.concatenate([[0], np.cumsum(new)])
    request = np.repeat(np.arange(R), new)
    index = np.arange(sum(new)) - starts[request]
    place = np.array(cached)[request] + index
    parents, masks, depth = None, None, index
    if case["tree"]:
        parents = np.concatenate([rng.integers(-1, np.arange(n)) for n in new]).astype(np.int32)
        masks = np.zeros((sum(new), case["tree"] // 64), np.uint64)
        for t, (r, i, p) in enumerate(zip(request, index, parents)):
            if p >= 0:
                masks[t] = masks[starts[r] + p]
            masks[t, i // 64] |= np.uint64(1) << np.uint64(i % 64)
        depth = np.array([sum(bin(int(w)).count("1") for w in row) - 1 for row in masks])
        masks = torch.from_numpy(masks.view(np.int64)).to(_DEV)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int64)).to(_DEV)  # noqa: E731
    step = {"cached_lens": _int32(cached), "new_lens": _int32(new), "tokens": sum(new), "pages": pages, "page": P,
            "width": width, "most_new": case["new"], "tree": case["tree"], "masks": masks, "held": _int32(need),
            "parents": None if parents is None else torch.from_numpy(parents).to(_DEV),
            "block_tables": torch.from_numpy(table).to(_DEV), "starts": to(starts), "request": to(request),
            "index": to(index), "place": to(place), "positions": to(np.array(cached)[request] + depth),
            "ring": torch.from_numpy(np.concatenate([order[at:], np.zeros(at, np.int32)])).to(_DEV),
            "ring_state": _int32([0, pages - at])}
    step["slots"] = step["block_tables"].long()[step["request"], step["place"] // P] * P + step["place"] % P
    return step


def _pool(case, step):
    """The framework's pool in the step's state."""
    import algebraic_intelligence_amd as A

    pool = A.PagePool(step["pages"], step["page"], case["requests"], step["width"] * step["page"])
    for name in ("block_tables", "held", "ring", "ring_state"):
        getattr(pool, name).copy_(step[name])
    return pool


def _plan(case, step):
    """A plan for the case's heads, made for the step."""
    import algebraic_intelligence_amd as A

    plan = A.DraftPlan(_pool(case, step), step["tokens"], heads=case["heads"], kv_heads=case["kv_heads"],
                       head_dim=case["head_dim"], dtype=_DTYPES[case["dtype"]], max_new=step["most_new"],
                       max_tree=case["tree"])
    return A.build_block_tables(plan, step["cached_lens"], step["new_lens"], step["parents"])


def prepare(case, seed):
    kind = case["kind"]
    g = _gen(seed)
    dt = _DTYPES[case["dtype"]]
    state = {"kind": kind}
    D, H, K = case["head_dim"], case["heads"], case["kv_heads"]
    if kind == "norm":
        B, L = case["batch"], case["seq"]
        state["sections"] = _sections(case)
        axes = len(state["sections"])
        rows = 4096
        state["rotary"] = _rotary(rows, D)
        # the activations as a model's projections leave them: (batch, tokens, heads, dim), seen as (B, H, L, D)
        for name, n in (("q", H), ("k", K)):
            state[name] = _randn((B, L, n, D), g, dt).transpose(1, 2)
            state["g" + name] = _randn((B, L, n, D), g, dt).transpose(1, 2)
            state[name + "_scale"] = _scale(D, g)
        # frames, rows and columns of patches at some offset, one token after the other
        side = 32
        t = torch.arange(L, device=_DEV)[None, :] + torch.randint(0, side * side, (B, 1), generator=g, device=_DEV)
        at = torch.randint(0, rows // 2, (B, 1), generator=g, device=_DEV)
        grid = (at + t // (side * side), t // side % side, t % side) if axes > 1 else ((at + t) % rows,)
        state["positions"] = torch.stack(grid[:axes], -1)
        state["train"] = case["mode"] == "train"
        if state["train"]:
            for name in ("q", "k", "q_scale", "k_scale"):
                state[name].requires_grad_(True)
        return state
    state["step"] = step = _plan_step(case, seed)
    if own and kind != "evict":
        state["plan"] = _plan(case, step)
    T = step["tokens"]
    page_shape = (step["pages"], K, step["page"], D)
    state["k_pages"], state["v_pages"] = _randn(page_shape, g, dt), _randn(page_shape, g, dt)
    if kind == "evict":
        if own:
            state["pool"] = _pool(case, step)
        # a few tokens hold most of the weight, and some none at all
        weights = torch.randn((case["requests"], step["width"] * step["page"]), generator=g, device=_DEV).mul_(2).exp_()
        state["weights"] = torch.where(weights < 0.05, torch.zeros_like(weights), weights)
        state["budget"], state["first"], state["recent"] = case["budget"], case["first"], case["recent"]
        return state
    if kind == "append":
        qkv = _randn((T, H + 2 * K, D), g, dt)
        state["q"], state["k"], state["v"] = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
        state["q_scale"], state["k_scale"] = _scale(D, g), _scale(D, g)
        state["sections"] = _sections(case)
        state["rotary"] = _rotary(max(4096, case["context"] + case["new"]), D)
        axes = len(state["sections"])
        state["positions"] = None
        if axes > 1:
            more = torch.randint(0, 64, (T, axes - 1), generator=g, device=_DEV, dtype=torch.int32)
            state["positions"] = torch.cat((step["positions"].int()[:, None], more), 1).contiguous()
        return state
    state["q"] = _randn((T, H, D), g, dt)
    if kind == "prefix":
        state["k_prefix"], state["v_prefix"] = _randn((K, case["prefix"], D), g, dt), _randn((K, case["prefix"], D), g, dt)
        return state
    # what the step's attention returned beside its output
    state["denominator"] = _own_weights(state).sum(-1).add_(_OMEGA)[step["request"], step["index"]]
    weights = torch.randn((case["requests"], step["width"] * step["page"]), generator=g, device=_DEV).exp_()
    at = torch.arange(weights.shape[1], device=_DEV)[None, :]
    state["weights"] = torch.where(at < step["cached_lens"][:, None], weights, torch.zeros_like(weights))
    return state


# ---------------------------------------------------------------------------------- plain forms
def _turned(x, positions, rotary, sections, back=False):
    """x (..., heads, D) in 32 bits turned by the rows positions (..., A) of the tables, pair p by its section's axis."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device=_DEV), torch.tensor(sections, device=_DEV),
                                   output_size=sum(sections))
    pairs = torch.arange(sum(sections), device=_DEV)
    row = positions.long()[..., axis]
    c, s = (t[row, pairs][..., None, :] for t in rotary)
    if back:
        s = -s
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack((c * x0 - s * x1, s * x0 + c * x1), -1).flatten(-2)


def _normed(x):
    """(x in 32 bits over its root mean square along the last axis, the root's inverse)."""
    x = x.float()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return x * r, r


def _norm_plain(x, scale, positions, rotary, sections):
    return _turned(_normed(x)[0] * scale, positions, rotary, sections).to(x.dtype)


def _norm_gradient_plain(x, scale, g, positions, rotary, sections):
    """(dx, dscale) of _norm_plain."""
    xh, r = _normed(x)
    back = _turned(g.float(), positions, rotary, sections, True)
    h = back * scale
    dx = r * (h - xh * (h * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), (back * xh).flatten(0, -2).sum(0)


def _octic(s):
    """rho(s)^8 with rho(s) = s + sqrt(1 + s^2); rho(-s) = 1 / rho(s)."""
    rho = s.abs() + torch.sqrt(1 + s * s)
    rho2 = rho * rho
    rho4 = rho2 * rho2
    rho8 = rho4 * rho4
    return torch.where(s < 0, 1 / rho8, rho8)


def _gathered(step, pages):
    """(R, K, length, D) of the requests' cached and new tokens in 32 bits, places past the end cleared."""
    P = step["page"]
    length = int(step["block_tables"].shape[1]) * P
    place = torch.arange(length, device=_DEV)
    live = place[None, :] < (step["cached_lens"] + step["new_lens"]).long()[:, None]
    page = step["block_tables"][:, place // P].clamp(min=0).long()
    rows = pages[page, :, (place % P).expand_as(page)].float()
    return torch.where(live[:, :, None, None], rows, torch.zeros((), device=_DEV)).transpose(1, 2).contiguous()


def _own_weights(state):
    """rho(s)^8 of every new token's rows with its request's keys, (R, most new, H, length); 0 where it sees none."""
    step, q = state["step"], state["q"]
    T, H, D = q.shape
    N, R = step["most_new"], step["cached_lens"].numel()
    k = _gathered(step, state["k_pages"])
    K, length = k.shape[1], k.shape[2]
    G = H // K
    rows = (step["starts"][:-1, None] + torch.arange(N, device=_DEV)[None, :]).clamp(max=T - 1)
    queries = q.float()[rows].view(R, N, K, G, D).permute(0, 2, 1, 3, 4).reshape(R, K, N * G, D)
    weight = _octic(queries @ k.transpose(2, 3).contiguous() / math.sqrt(D))
    place = torch.arange(length, device=_DEV)
    cached, new = step["cached_lens"].long(), step["new_lens"].long()
    drafted = place[None, :] - cached[:, None]  # index among the new tokens, (R, length)
    if step["masks"] is None:
        sees = drafted[:, None, :] <= torch.arange(N, device=_DEV)[None, :, None]
    else:
        at = drafted.clamp(0, step["tree"] - 1)[:, None, :].expand(R, N, length)
        sees = (torch.gather(step["masks"][rows], 2, at // 64) >> (at % 64)) & 1 > 0
        sees = sees | (drafted[:, None, :] < 0)
    sees = sees & (drafted < new[:, None])[:, None, :] & (torch.arange(N, device=_DEV)[None, :] < new[:, None])[:, :, None]
    weight = weight.view(R, K, N, G, length).permute(0, 2, 1, 3, 4).reshape(R, N, H, length)
    return torch.where(sees[:, :, None, :], weight, torch.zeros((), device=_DEV))


def _prefix_plain(state):
    step, q, k_prefix, v_prefix = (state[n] for n in ("step", "q", "k_prefix", "v_prefix"))
    T, H, D = q.shape
    K = k_prefix.shape[0]
    G, R, N = H // K, step["cached_lens"].numel(), step["most_new"]
    # the prefix against all rows of a key head at once
    rows = q.float().view(T, K, G, D).transpose(0, 1).reshape(K, T * G, D)
    shared = _octic(rows @ k_prefix.float().transpose(1, 2).contiguous() / math.sqrt(D))
    back = lambda x: x.view(K, T, G, -1).transpose(0, 1).reshape(T, H, -1)  # noqa: E731
    top, bottom = back(shared @ v_prefix.float()), back(shared.sum(-1, keepdim=True))
    weight = _own_weights(state)
    length = weight.shape[-1]
    v = _gathered(step, state["v_pages"])
    by_head = weight.view(R, N, K, G, length).permute(0, 2, 1, 3, 4).reshape(R, K, N * G, length)
    mine = (by_head @ v).view(R, K, N, G, D).permute(0, 2, 1, 3, 4).reshape(R, N, H, D)
    request, index = step["request"], step["index"]
    top = top + mine[request, index]
    bottom = bottom + weight.sum(-1, keepdim=True)[request, index] + _OMEGA
    return (top / bottom).to(q.dtype), bottom[..., 0]


def _weights_plain(state):
    step, weights = state["step"], state["weights"]
    R, N = step["cached_lens"].numel(), step["most_new"]
    share = torch.zeros((R, N, state["q"].shape[1], 1), device=_DEV)
    share[step["request"], step["index"]] = 1 / state["denominator"][..., None]
    given = (_own_weights(state) * share).sum((1, 2))
    place = torch.arange(given.shape[1], device=_DEV)[None, :]
    cached = step["cached_lens"].long()[:, None]
    live = place < cached + step["new_lens"].long()[:, None]
    weights.copy_(torch.where(live, torch.where(place < cached, weights, torch.zeros_like(weights)) + given, weights))
    return weights


def _evict_plain(state):
    step, weights, budget = state["step"], state["weights"], state["budget"]
    P, cached = step["page"], step["cached_lens"].long()[:, None]
    place = torch.arange(weights.shape[1], device=_DEV)[None, :]
    most = torch.full_like(weights, math.inf)
    sure = (place < state["first"]) | (place >= cached - state["recent"])
    rank = torch.where(place < cached, torch.where(sure, most, weights), -most)
    order = torch.sort(rank, dim=1, descending=True, stable=True)[1]
    kept = order[:, :min(budget, weights.shape[1])].sort(dim=1)[0]
    # requests within the budget keep all they have
    kept = torch.where(cached > budget, kept, place[:, :kept.shape[1]])
    lens = cached[:, 0].clamp(max=budget)
    to = place[:, :kept.shape[1]].expand_as(kept)
    moved = (to < lens[:, None]) & (kept != to)
    request, to, kept_flat = moved.nonzero()[:, 0], to[moved], kept[moved]
    table = step["block_tables"].long()
    for pages in (state["k_pages"], state["v_pages"]):
        pages[table[request, to // P], :, to % P] = pages[table[request, kept_flat // P], :, kept_flat % P]
    left = torch.zeros_like(weights)
    left[:, :kept.shape[1]] = torch.where(place[:, :kept.shape[1]] < lens[:, None], weights.gather(1, kept),
                                          torch.zeros((), device=_DEV))
    return lens.int(), left, state["k_pages"], state["v_pages"]


# ------------------------------------------------------------------------------------------ run
def run(state):
    kind = state["kind"]
    if own:
        import algebraic_intelligence_amd as A
    if kind == "norm":
        q, k, qs, ks, positions, rotary, sections = (state[n] for n in ("q", "k", "q_scale", "k_scale", "positions", "rotary",
                                                                         "sections"))
        if own:
            y, z = A.apply_ago_norm_rotations(q, k, qs, ks, rotary, positions, sections, eps=_EPS)
            if not state["train"]:
                return y, z
            return y.detach(), z.detach(), *torch.autograd.grad((y, z), (q, k, qs, ks), (state["gq"], state["gk"]))
        args = positions, rotary, sections
        flat = lambda x: x.detach().transpose(1, 2)  # noqa: E731
        out = tuple(_norm_plain(flat(x), w.detach(), *args).transpose(1, 2) for x, w in ((q, qs), (k, ks)))
        if not state["train"]:
            return out
        (dq, dqs), (dk, dks) = (_norm_gradient_plain(flat(x), w.detach(), flat(g), *args)
                                for x, w, g in ((q, qs, state["gq"]), (k, ks, state["gk"])))
        return *out, dq.transpose(1, 2), dk.transpose(1, 2), dqs, dks
    k_pages, v_pages = state["k_pages"], state["v_pages"]
    if kind == "append":
        q, k, v, qs, ks, rotary, sections = (state[n] for n in ("q", "k", "v", "q_scale", "k_scale", "rotary", "sections"))
        if own:
            y = A.append_to_cache(q, k, v, k_pages, v_pages, state["plan"], rotary, positions=state["positions"],
                                  sections=sections, norms=(qs, ks), eps=_EPS)
            return y, k_pages, v_pages
        slots, positions = state["step"]["slots"], state["positions"]
        positions = state["step"]["positions"][:, None] if positions is None else positions
        page, offset = slots // state["step"]["page"], slots % state["step"]["page"]
        k_pages[page, :, offset] = _norm_plain(k, ks, positions, rotary, sections)
        v_pages[page, :, offset] = v
        return _norm_plain(q, qs, positions, rotary, sections), k_pages, v_pages
    if kind == "prefix":
        if own:
            return A.paged_prefix_afa(state["q"], state["k_prefix"], state["v_prefix"], k_pages, v_pages, state["plan"],
                                      _OMEGA, return_denominator=True)
        return _prefix_plain(state)
    if kind == "weights":
        if own:
            return A.accumulate_cache_weights(state["q"], k_pages, state["denominator"], state["plan"], state["weights"])
        return _weights_plain(state)
    if own:
        lens, left = A.evict_from_cache(k_pages, v_pages, state["pool"], state["weights"], state["step"]["cached_lens"],
                                        state["budget"], first=state["first"], recent=state["recent"])
        return lens, left, k_pages, v_pages
    return _evict_plain(state)


# ---------------------------------------------------------------------------------------- exact
def _exact_turned(x, positions, rotary, sections, sign):
    """Pair by pair as complex numbers in 64 bits: (x0 + i x1)(c + i s)."""
    at = 0
    z = torch.view_as_complex(x.contiguous().view(*x.shape[:-1], -1, 2))
    turn = torch.ones(*positions.shape[:-1], z.shape[-1], dtype=torch.complex128, device=_DEV)
    for axis, n in enumerate(sections):
        row = positions[..., axis].long()
        turn[..., at:at + n] = torch.complex(rotary[0][row, at:at + n].double(), sign * rotary[1][row, at:at + n].double())
        at += n
    return torch.view_as_real(z * turn[..., None, :]).flatten(-2)


def _exact_norm(x, scale, g, args):
    """(y, dx, dscale) of rows x (..., heads, D): the norm's Jacobian applied to the cotangent, in 64 bits."""
    x, scale = x.detach().double(), scale.detach().double()
    size = (x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS) ** 0.5
    y = _exact_turned(x / size * scale, *args, 1)
    if g is None:
        return y, None, None
    back = _exact_turned(g.double(), *args, -1)
    dscale = (back * x / size).reshape(-1, x.shape[-1]).sum(0)
    dot = (back * scale * x).sum(-1, keepdim=True)
    return y, back * scale / size - x * dot / (x.shape[-1] * size ** 3), dscale


def _exact_octic(s):
    return torch.where(s < 0, (torch.sqrt(1 + s * s) - s) ** -8.0, (s + torch.sqrt(1 + s * s)) ** 8)


def _exact_requests(case, state):
    """For each request: its first row, its rows, its tokens' pages and places, and which keys a row sees."""
    step = state["step"]
    cached, new = _lens(case)
    parents = None if step["parents"] is None else step["parents"].cpu().tolist()
    first = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        held = step["block_tables"][r, :-(-(c + n) // step["page"])].long()
        rows = lambda p, held=held, m=c + n: p[held].transpose(0, 1).reshape(p.shape[1], -1, p.shape[3])[:, :m].double()  # noqa: E731
        if parents is None:
            sees = torch.ones(n, c + n, dtype=torch.bool, device=_DEV).tril(c)
        else:
            sees = torch.ones(n, c + n, dtype=torch.bool)
            sees[:, c:] = False
            for i in range(n):
                j = i
                while j >= 0:
                    sees[i, c + j] = True
                    j = parents[first + j]
            sees = sees.to(_DEV)
        yield r, first, n, c, rows, sees
        first += n


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "norm":
        args = state["positions"], state["rotary"], state["sections"]
        got = [_exact_norm(state[n].transpose(1, 2), state[n + "_scale"],
                           state["g" + n].transpose(1, 2) if state["train"] else None, args) for n in ("q", "k")]
        out = tuple(y.transpose(1, 2) for y, _, _ in got)
        return (*out, *(d.transpose(1, 2) for _, d, _ in got), *(d for _, _, d in got)) if state["train"] else out
    step = state["step"]
    if kind == "append":
        at = state["positions"] if state["positions"] is not None else step["positions"][:, None]
        args = at, state["rotary"], state["sections"]
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        for pages, rows in ((k_pages, _exact_norm(state["k"], state["k_scale"], None, args)[0]), (v_pages, state["v"].double())):
            by_token = pages.transpose(1, 2).reshape(-1, *rows.shape[1:])
            by_token[step["slots"]] = rows
            pages.copy_(by_token.view(pages.shape[0], step["page"], *rows.shape[1:]).transpose(1, 2))
        return _exact_norm(state["q"], state["q_scale"], None, args)[0], k_pages, v_pages
    if kind == "evict":
        cached, _ = _lens(case)
        weights = state["weights"].double()
        left = torch.zeros_like(weights)
        k_pages, v_pages = state["k_pages"], state["v_pages"]
        host = state["weights"].cpu().numpy()
        for r, c in enumerate(cached):
            m = min(c, case["budget"])
            if m < c:
                sure = [j for j in range(c) if j < case["first"] or j >= c - case["recent"]]
                rest = np.setdiff1d(np.arange(c), sure)
                rest = rest[np.lexsort((rest, -host[r, rest]))][:m - len(sure)]
                kept = torch.from_numpy(np.sort(np.concatenate([np.array(sure, np.int64), rest]))).to(_DEV)
            else:
                kept = torch.arange(c, device=_DEV)
            left[r, :m] = weights[r, kept]
            held = step["block_tables"][r, :-(-c // step["page"])].long()
            for pages in (k_pages, v_pages):
                rows = pages[held].transpose(1, 2).reshape(-1, K, D)
                rows[:m] = rows[kept]
                pages[held] = rows.view(held.numel(), step["page"], K, D).transpose(1, 2)
        return None, left, k_pages.double(), v_pages.double()
    cached, new = _lens(case)
    pairs = sum(n * (c + n) for c, n in zip(cached, new)) + sum(new) * case.get("prefix", 0)
    if pairs * H * D > 8e11 or case["requests"] * H > 8192:
        return None
    q = state["q"].double()
    G = H // K
    if kind == "weights":
        out = state["weights"].double()
        share = 1 / state["denominator"].double()
        for r, first, n, c, rows, sees in _exact_requests(case, state):
            k = rows(state["k_pages"])
            out[r, c:c + n] = 0
            for h in range(H):
                w = _exact_octic(q[first:first + n, h] @ k[h // G].t() / math.sqrt(D)) * sees
                out[r, :c + n] += share[first:first + n, h] @ w
        return out
    top, bottom = torch.empty_like(q), torch.full(q.shape[:2], _OMEGA, dtype=torch.float64, device=_DEV)
    for h in range(H):
        k, v = state["k_prefix"][h // G].double(), state["v_prefix"][h // G].double()
        w = _exact_octic(q[:, h] @ k.t() / math.sqrt(D))
        top[:, h] = w @ v
        bottom[:, h] += w.sum(-1)
    for r, first, n, c, rows, sees in _exact_requests(case, state):
        k, v = rows(state["k_pages"]), rows(state["v_pages"])
        for h in range(H):
            w = _exact_octic(q[first:first + n, h] @ k[h // G].t() / math.sqrt(D)) * sees
            top[first:first + n, h] += w @ v[h // G]
            bottom[first:first + n, h] += w.sum(-1)
    return top / bottom[..., None], bottom
