"""The serving operators by which this framework's speed is followed: drafted trees of tokens over a
paged key/value cache.

One case is one call (a rotation in training: the call and its gradients) of

  tables     ``build_block_tables``: request lengths and parents to pages, slots, positions and masks;
  rotate     ``apply_ago_axis_rotations``: q and k turned by positions of several axes;
  append     ``append_to_cache``: q and k of the new tokens rotated, k and v stored in their slots;
  attention  ``paged_tree_afa``: the new tokens' attention over the cache and their own tree.

``prepare`` makes what a serving or training program holds before the call: activations, pages,
lengths, Cayley tables, and the pool and plan that it keeps between steps.  The pool's pages are kept
up to date in place: a ``tables`` call for the same lengths again finds them as it left them, and
returns the same.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = torch.device("cuda")


# -------------------------------------------------------------------------------------- cases
def _tables(requests, context, new, tree, page, spread=True):
    """Lengths run from about context / 8 to context where they spread."""
    return {"kind": "tables", "requests": requests, "context": context, "new": new, "tree": tree, "page": page,
            "spread": spread}


def _rotate(mode, batch, heads, kv_heads, seq, head_dim, sections, dtype):
    return {"kind": "rotate", "mode": mode, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq": seq,
            "head_dim": head_dim, "sections": sections, "dtype": dtype}


def _append(requests, context, new, tree, heads, kv_heads, head_dim, page, sections, dtype):
    return {"kind": "append", "requests": requests, "context": context, "new": new, "tree": tree, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "sections": sections, "dtype": dtype,
            "spread": True}


def _attention(requests, context, new, tree, heads, kv_heads, head_dim, page, dtype, spread=True):
    return {"kind": "attention", "requests": requests, "context": context, "new": new, "tree": tree, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "spread": spread}


def listed():
    return [
        # The plan of a plain decoding step: one new token for each request of a small batch.
        {"name": "tables_step", **_tables(24, 4096, 1, 0, 64)},
        # The plan of a large batch that drafts trees, with pages shorter than any tile.
        {"name": "tables_trees", **_tables(512, 8192, 48, 64, 16)},
        # Rotating the new tokens of a decoding step, one time axis and two of an image.
        {"name": "rotate_step", **_rotate("forward", 48, 12, 12, 1, 64, "8,12,12", "bf16")},
        # Training the 125M model's layer on image patches (height, width after a time axis).
        {"name": "rotate_image_train", **_rotate("train", 8, 12, 12, 2048, 64, "8,12,12", "bf16")},
        # A video clip in full precision, grouped heads, a length that is no multiple of anything.
        {"name": "rotate_video_f32", **_rotate("train", 1, 16, 4, 8189, 128, "16,24,24", "fp32")},
        # Storing one step's drafted tokens: latency.
        {"name": "append_step", **_append(16, 2048, 8, 64, 16, 4, 128, 64, "64", "bf16")},
        # Storing the prompts of a batch: 16k tokens of 16 heads, three axes.
        {"name": "append_prompts", **_append(8, 64, 2048, 0, 16, 16, 64, 32, "8,12,12", "fp16")},
        # One request, one new token, a short context: the smallest call of a decoder.
        {"name": "attention_token", **_attention(1, 700, 1, 0, 12, 12, 64, 64, "bf16", False)},
        # Speculative decoding of a batch: trees of up to 32 nodes over contexts of up to 8k.
        {"name": "attention_trees", **_attention(32, 8192, 32, 64, 16, 4, 128, 64, "bf16")},
        # Long documents: few requests, contexts of 128k, short drafts, grouped heads.
        {"name": "attention_long", **_attention(4, 131072, 6, 64, 16, 4, 128, 128, "fp16")},
        # A large batch of single tokens, every head with its own keys.
        {"name": "attention_steps", **_attention(96, 4096, 1, 0, 16, 16, 64, 16, "bf16")},
        # The pilot model's heads (6 of 48) in full precision, ragged.
        {"name": "attention_pilot_f32", **_attention(40, 3001, 13, 64, 6, 6, 48, 32, "fp32")},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rotate", "append", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "tables":
        new = _log_int(rng, 1, 64)
        return _tables(_log_int(rng, 1, 512), _log_int(rng, 64, 8192), new, 64 if rng.random() < 0.6 else 0, page)
    D = rng.choice([48, 64, 96, 128])
    kv = rng.choice([2, 4, 6, 8, 12])
    group = rng.choice([1, 1, 2, 4])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    cut = rng.choice([[4], [1, 3], [1, 1, 2], [2, 1, 1]])
    sections = ",".join(str(D // 8 * c) for c in cut)
    if kind == "rotate":
        mode = rng.choice(["forward", "train"])
        tokens = max(1, _log_int(rng, 16, 16384) * 12 // (kv * group))
        seq = min(tokens, _log_int(rng, 1, 8192))
        return _rotate(mode, max(1, tokens // seq), kv * group, kv, seq, D, sections, dtype)
    if kind == "append":
        new = _log_int(rng, 1, 1024)
        requests = max(1, min(64, _log_int(rng, 1, 8192) // new))
        return _append(requests, _log_int(rng, 16, 2048), new, 64 if new <= 64 and rng.random() < 0.6 else 0,
                       kv * group, kv, D, page, sections, dtype)
    new = _log_int(rng, 1, 40)
    context = _log_int(rng, 64, 65536)
    # no more cached elements than the long documents hold
    most = 4 * 131072 * 4 * 128 // (context * kv * D)
    requests = max(1, min(96, most, _log_int(rng, 1, 128)))
    return _attention(requests, context, new, 64 if rng.random() < 0.6 else 0, kv * group, kv, D, page, dtype)


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
    if case["kind"] == "rotate":
        per = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        passes = 2 if case["mode"] == "train" else 1
        esz = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": passes * 2 * per * esz, "flops": passes * 3 * per}
    cached, new = _lens(case)
    T, R = sum(new), case["requests"]
    if case["kind"] == "tables":
        # lengths and pages held, in and out; per token its page, slot, position and request, parent and mask
        return {"bytes": 28 * R + 16 * T + (12 * T if case["tree"] else 0), "flops": 10 * T}
    esz = 4 if case["dtype"] == "fp32" else 2
    D, H, K = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        return {"bytes": 2 * T * (H + 2 * K) * D * esz, "flops": 3 * T * (H + K) * D}
    keys = sum(c + n for c, n in zip(cached, new))
    pairs = sum(n * (c + 1) for c, n in zip(cached, new))
    return {"bytes": (2 * keys * K + 2 * T * H) * D * esz, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed))


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device=_DEV).to(dtype)


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


def _step(case, seed):
    """A serving step: lengths, a random tree for each request (where the case has trees), and a pool
    in the middle of its life, whose pages lie in random order."""
    cached, new = _lens(case)
    rng = np.random.default_rng(seed)
    P, R = case["page"], case["requests"]
    width = -(-(case["context"] + case["new"]) // P) + 1
    need = [-(-(c + n) // P) for c, n in zip(cached, new)]
    # before the step some requests hold a page fewer than they need, some one too many
    held = [min(width, max(0, n + int(rng.integers(-1, 2)))) for n in need]
    pages = sum(need) + 2 * R
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((R, width), -1, np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    head = int(rng.integers(0, pages))
    ring = np.zeros(pages, np.int32)
    ring[(head + np.arange(pages - at)) % pages] = order[at:]
    parents = np.concatenate([rng.integers(-1, np.arange(n)) for n in new]).astype(np.int32) if case["tree"] else None
    return {"cached_lens": _int32(cached), "new_lens": _int32(new), "held": _int32(held),
            "block_tables": torch.from_numpy(table).to(_DEV), "ring": torch.from_numpy(ring).to(_DEV),
            "ring_state": _int32([head, pages - at]), "tokens": sum(new), "pages": pages, "page": P,
            "most_new": case["new"], "width": width,
            "tree": case["tree"], "parents": None if parents is None else torch.from_numpy(parents).to(_DEV)}


def _plan(case, step):
    """The framework's pool, in the step's state, and a plan for the case's heads."""
    import algebraic_intelligence_amd as A

    pool = A.PagePool(step["pages"], step["page"], case["requests"], step["width"] * step["page"])
    for name in ("block_tables", "held", "ring", "ring_state"):
        getattr(pool, name).copy_(step[name])
    dtype = _DTYPES[case.get("dtype", "bf16")]
    return A.DraftPlan(pool, step["tokens"], heads=case.get("heads", 12), kv_heads=case.get("kv_heads", 12),
                       head_dim=case.get("head_dim", 64), dtype=dtype, max_new=step["most_new"], max_tree=case["tree"])


def prepare(case, seed):
    kind = case["kind"]
    g = _gen(seed)
    dt = _DTYPES[case.get("dtype", "bf16")]
    state = {"kind": kind}
    if kind == "rotate":
        B, L, D = case["batch"], case["seq"], case["head_dim"]
        state["sections"] = _sections(case)
        axes = len(state["sections"])
        rows = 4096
        state["rotary"] = _rotary(rows, D)
        # the activations as a model's projections leave them: (batch, tokens, heads, dim), seen as (B, H, L, D)
        for name, H in (("q", case["heads"]), ("k", case["kv_heads"])):
            state[name] = _randn((B, L, H, D), g, dt).transpose(1, 2)
            state["g" + name] = _randn((B, L, H, D), g, dt).transpose(1, 2)
        # frames, rows and columns of patches at some offset, one token after the other
        side = 32
        t = torch.arange(L, device=_DEV)[None, :] + torch.randint(0, side * side, (B, 1), generator=g, device=_DEV)
        at = torch.randint(0, rows // 2, (B, 1), generator=g, device=_DEV)
        grid = (at + t // (side * side), t // side % side, t % side) if axes > 1 else ((at + t) % rows,)
        state["positions"] = torch.stack(grid[:axes], -1)
        state["train"] = case["mode"] == "train"
        if state["train"]:
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
        return state
    state["step"] = step = _step(case, seed)
    if own:
        state["plan"] = _plan(case, step)
    if kind == "tables":
        return state
    # the later operators find the step planned
    state["now"] = _tables_plain(step)
    if own:
        import algebraic_intelligence_amd as A

        A.build_block_tables(state["plan"], step["cached_lens"], step["new_lens"], step["parents"])
    T, H, K, D = step["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    page_shape = (step["pages"], K, step["page"], D)
    state["k_pages"], state["v_pages"] = _randn(page_shape, g, dt), _randn(page_shape, g, dt)
    if kind == "append":
        qkv = _randn((T, H + 2 * K, D), g, dt)
        state["q"], state["k"], state["v"] = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
        state["sections"] = _sections(case)
        state["rotary"] = _rotary(max(4096, case["context"] + case["new"]), D)
        axes = len(state["sections"])
        state["positions"] = None
        if axes > 1:
            more = torch.randint(0, 64, (T, axes - 1), generator=g, device=_DEV, dtype=torch.int32)
            state["positions"] = torch.cat((state["now"][1][:, None], more), 1).contiguous()
        return state
    state["q"] = _randn((T, H, D), g, dt)
    return state


# ---------------------------------------------------------------------------------- plain forms
def _tables_plain(step):
    """(slots, positions, requests, starts, masks, block_tables, held, ring, ring_state)."""
    cached, new, held = (step[n].long() for n in ("cached_lens", "new_lens", "held"))
    table, ring, P = step["block_tables"], step["ring"], step["page"]
    head, count = step["ring_state"].long()
    pages, T = ring.numel(), step["tokens"]
    need = (cached + new + P - 1) // P
    grow, shrink = (need - held).clamp(min=0), (held - need).clamp(min=0)
    column = torch.arange(table.shape[1], device=_DEV)[None, :]
    fresh = (column >= held[:, None]) & (column < need[:, None])
    back = (column >= need[:, None]) & (column < held[:, None])
    source = (head + (torch.cumsum(grow, 0) - grow)[:, None] + column - held[:, None]) % pages
    target = (head + count + (torch.cumsum(shrink, 0) - shrink)[:, None] + column - need[:, None]) % pages
    table_out = torch.where(fresh, ring[source], torch.where(back, torch.full_like(table, -1), table))
    ring_out = torch.cat((ring, ring[:1]))
    ring_out[torch.where(back, target, torch.full_like(target, pages))] = table
    taken, given = grow.sum(), shrink.sum()
    state_out = torch.stack(((head + taken) % pages, count - taken + given)).int()
    ends = torch.cumsum(new, 0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    token = torch.arange(T, device=_DEV)
    request = torch.searchsorted(ends, token, right=True)
    index = token - starts[request]
    place = cached[request] + index
    slots = table_out[request, place // P] * P + place % P
    if not step["tree"]:
        positions, masks = place, None
    else:
        # bits of each token and its ancestors, by doubling the distance to the ancestor that is looked at
        parents = step["parents"].long()
        up = torch.where(parents >= 0, starts[request] + parents, torch.full_like(parents, T))
        up = torch.cat((up, up.new_full((1,), T)))
        sees = torch.zeros((T + 1, step["tree"]), dtype=torch.bool, device=_DEV)
        sees[:T] = index[:, None] == torch.arange(step["tree"], device=_DEV)[None, :]
        for _ in range(step["tree"].bit_length()):
            sees, up = sees | sees[up], up[up]
        sees = sees[:T]
        positions = cached[request] + sees.sum(1) - 1
        bits = sees.view(T, -1, 64).long() << torch.arange(64, device=_DEV)
        masks = bits.sum(2)
    return [slots.int(), positions.int(), request.int(), starts.int(), masks, table_out, need.int(), ring_out[:-1],
            state_out]


def _turned(x, positions, rotary, sections, back=False):
    """x (..., heads, D) turned by the rows positions (..., A) of the tables, pair p by its section's axis."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device=_DEV), torch.tensor(sections, device=_DEV),
                                   output_size=sum(sections))
    pairs = torch.arange(sum(sections), device=_DEV)
    row = positions.long()[..., axis]
    c, s = (t[row, pairs][..., None, :] for t in rotary)
    if back:
        s = -s
    x0, x1 = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack((c * x0 - s * x1, s * x0 + c * x1), -1).flatten(-2).to(x.dtype)


def _octic(s):
    """rho(s)^8 with rho(s) = s + sqrt(1 + s^2); rho(-s) = 1 / rho(s)."""
    rho = s.abs() + torch.sqrt(1 + s * s)
    rho2 = rho * rho
    rho4 = rho2 * rho2
    rho8 = rho4 * rho4
    return torch.where(s < 0, 1 / rho8, rho8)


def _attention_plain(state, omega=0.5):
    step, q, now = state["step"], state["q"], state["now"]
    k_pages, v_pages = state["k_pages"], state["v_pages"]
    _, _, request, starts, masks, table, _, _, _ = now
    cached, new = step["cached_lens"].long(), step["new_lens"].long()
    T, H, D = q.shape
    K, P, R = k_pages.shape[1], step["page"], cached.numel()
    G, N = H // K, step["most_new"]
    length = table.shape[1] * P
    place = torch.arange(length, device=_DEV)
    live = place[None, :] < (cached + new)[:, None]
    page = table[:, place // P].clamp(min=0).long()
    offset = (place % P).expand_as(page)
    # (R, K, length, D), rows past the end cleared
    k, v = (torch.where(live[:, :, None, None], p[page, :, offset], torch.zeros((), dtype=p.dtype, device=_DEV))
            .float().transpose(1, 2).contiguous() for p in (k_pages, v_pages))
    rows = (starts[:-1, None].long() + torch.arange(N, device=_DEV)[None, :]).clamp(max=T - 1)
    queries = q.float()[rows].view(R, N, K, G, D).permute(0, 2, 1, 3, 4).reshape(R, K, N * G, D)
    weight = _octic(queries @ k.transpose(2, 3).contiguous() / math.sqrt(D))
    drafted = place[None, :] - cached[:, None]  # index among the new tokens, (R, length)
    if masks is None:
        sees = drafted[:, None, :] <= torch.arange(N, device=_DEV)[None, :, None]
    else:
        words = masks[rows]  # (R, N, W)
        at = drafted.clamp(0, step["tree"] - 1)[:, None, :].expand(R, N, length)
        sees = (torch.gather(words, 2, at // 64) >> (at % 64)) & 1 > 0
        sees = sees | (drafted[:, None, :] < 0)
    sees = sees & live[:, None, :]
    sees = sees[:, None, :, None, :].expand(R, K, N, G, length).reshape(R, K, N * G, length)
    weight = torch.where(sees, weight, torch.zeros((), device=_DEV))
    out = weight @ v / (weight.sum(-1, keepdim=True) + omega)
    out = out.view(R, K, N, G, D).permute(0, 2, 1, 3, 4).reshape(R, N, H, D)
    request = request.long()
    return out[request, torch.arange(T, device=_DEV) - starts.long()[request]].to(q.dtype)


# ------------------------------------------------------------------------------------------ run
def run(state):
    kind = state["kind"]
    if kind == "tables":
        step = state["step"]
        if own:
            import algebraic_intelligence_amd as A

            plan = A.build_block_tables(state["plan"], step["cached_lens"], step["new_lens"], step["parents"])
            pool = plan.pool
            return [plan.slots, plan.positions, plan.requests, plan.starts, plan.masks if step["tree"] else None,
                    pool.block_tables, pool.held, pool.ring, pool.ring_state]
        return _tables_plain(step)
    if kind == "rotate":
        q, k, positions, rotary, sections = (state[n] for n in ("q", "k", "positions", "rotary", "sections"))
        if own:
            import algebraic_intelligence_amd as A

            q_rot, k_rot = A.apply_ago_axis_rotations(q, k, rotary, positions, sections)
            if not state["train"]:
                return q_rot, k_rot
            return q_rot.detach(), k_rot.detach(), *torch.autograd.grad((q_rot, k_rot), (q, k), (state["gq"], state["gk"]))
        turn = lambda x, back: _turned(x.detach().transpose(1, 2), positions, rotary, sections, back).transpose(1, 2)  # noqa: E731
        out = turn(q, False), turn(k, False)
        return (*out, turn(state["gq"], True), turn(state["gk"], True)) if state["train"] else out
    if kind == "append":
        q, k, v, k_pages, v_pages, rotary, sections = (state[n] for n in ("q", "k", "v", "k_pages", "v_pages", "rotary",
                                                                           "sections"))
        if own:
            import algebraic_intelligence_amd as A

            q_rot = A.append_to_cache(q, k, v, k_pages, v_pages, state["plan"], rotary, positions=state["positions"],
                                      sections=sections)
            return q_rot, k_pages, v_pages
        slots, positions = state["now"][0].long(), state["positions"]
        positions = state["now"][1][:, None] if positions is None else positions
        page, offset = slots // state["step"]["page"], slots % state["step"]["page"]
        k_pages[page, :, offset] = _turned(k, positions, rotary, sections)
        v_pages[page, :, offset] = v
        return _turned(q, positions, rotary, sections), k_pages, v_pages
    if own:
        import algebraic_intelligence_amd as A

        return A.paged_tree_afa(state["q"], state["k_pages"], state["v_pages"], state["plan"], sink_omega=0.5)
    return _attention_plain(state)


# ---------------------------------------------------------------------------------------- exact
def _exact_turned(x, positions, rotary, sections, sign):
    """Pair by pair as complex numbers in 64 bits: (x0 + i x1)(c + i s)."""
    at = 0
    z = torch.view_as_complex(x.double().contiguous().view(*x.shape[:-1], -1, 2))
    turn = torch.ones(*positions.shape[:-1], z.shape[-1], dtype=torch.complex128, device=_DEV)
    for axis, n in enumerate(sections):
        row = positions[..., axis].long()
        turn[..., at:at + n] = torch.complex(rotary[0][row, at:at + n].double(), sign * rotary[1][row, at:at + n].double())
        at += n
    return torch.view_as_real(z * turn[..., None, :]).flatten(-2)


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    state = prepare(case, seed)
    if case["kind"] == "rotate":
        args = state["positions"], state["rotary"], state["sections"]
        names = [("q", 1), ("k", 1)] + ([("gq", -1), ("gk", -1)] if state["train"] else [])
        return tuple(_exact_turned(state[n].detach().transpose(1, 2), *args, sign).transpose(1, 2) for n, sign in names)
    step = state["step"]
    cached, new = _lens(case)
    slots, positions, _, _, _, table = state["now"][:6]
    P = step["page"]
    if case["kind"] == "append":
        at = state["positions"] if state["positions"] is not None else positions[:, None]
        args = at, state["rotary"], state["sections"], 1
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        k_rot = _exact_turned(state["k"], *args)
        flat = slots.long()
        for pages, rows in ((k_pages, k_rot), (v_pages, state["v"].double())):
            by_token = pages.transpose(1, 2).reshape(-1, *rows.shape[1:])
            by_token[flat] = rows
            pages.copy_(by_token.view(pages.shape[0], P, *rows.shape[1:]).transpose(1, 2))
        return _exact_turned(state["q"], *args), k_pages, v_pages
    if sum(c * n for c, n in zip(cached, new)) * case["heads"] * case["head_dim"] > 4e11:
        return None
    K, G = case["kv_heads"], case["heads"] // case["kv_heads"]
    parents = None if step["parents"] is None else step["parents"].cpu().tolist()
    outs, first = [], 0
    for r, (c, n) in enumerate(zip(cached, new)):
        held = table[r, :-(-(c + n) // P)].long()
        k, v = (p[held].transpose(0, 1).reshape(K, -1, p.shape[-1])[:, :c + n].double()
                for p in (state["k_pages"], state["v_pages"]))
        sees = torch.ones(n, c + n, dtype=torch.bool)
        for i in range(n):
            sees[i, c:] = False
            j = i
            while j >= 0:
                sees[i, c + j] = True
                j = j - 1 if parents is None else parents[first + j]
        sees = sees.to(_DEV)
        q = state["q"][first:first + n].double()
        out = torch.empty_like(q)
        for h in range(case["heads"]):
            s = q[:, h] @ k[h // G].t() / math.sqrt(q.shape[-1])
            w = (s + torch.sqrt(1 + s * s)) ** 8
            w = torch.where(s < 0, (torch.sqrt(1 + s * s) - s) ** -8.0, w) * sees
            out[:, h] = w @ v[h // G] / (w.sum(-1, keepdim=True) + 0.5)
        outs.append(out)
        first += n
    return torch.cat(outs)
