"""The serving operators' call surface without a GPU: refusals of the Python layer and of the C ABI, all
before any device work."""
import ctypes
import math
import os

import pytest
import torch

import algebraic_intelligence_amd as A
from algebraic_intelligence_amd import _lib, paged

DUMMY = 0x1000  # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from algebraic_intelligence_amd import build
        build.build()
    return _lib.lib()


def _plan(**kw):
    sizes = dict(num_pages=8, page_size=16, requests=2, table_width=4, max_tokens=16, max_new=8, max_tree=64, heads=4,
                 kv_heads=2, head_dim=64, dtype=_lib.AFA_BF16)
    pointers = {n: DUMMY for n, _ in paged._Plan._fields_ if n not in sizes}
    return paged._Plan(**{**sizes, **pointers, **kw})


SIZES = [
    (dict(dtype=4), _lib.ERR_DTYPE), (dict(dtype=-1), _lib.ERR_DTYPE), (dict(num_pages=0), _lib.ERR_SHAPE),
    (dict(page_size=0), _lib.ERR_SHAPE), (dict(requests=0), _lib.ERR_SHAPE), (dict(table_width=0), _lib.ERR_SHAPE),
    (dict(max_tokens=0), _lib.ERR_SHAPE), (dict(max_new=17), _lib.ERR_SHAPE), (dict(max_new=0), _lib.ERR_SHAPE),
    (dict(heads=5), _lib.ERR_SHAPE), (dict(heads=0), _lib.ERR_SHAPE), (dict(kv_heads=8), _lib.ERR_SHAPE),
    (dict(max_tree=63), _lib.ERR_SHAPE), (dict(max_tree=320), _lib.ERR_SHAPE), (dict(max_tree=-64), _lib.ERR_SHAPE),
    (dict(head_dim=0), _lib.ERR_HEAD_DIM), (dict(head_dim=1025), _lib.ERR_HEAD_DIM),
    (dict(num_pages=1 << 27), _lib.ERR_SHAPE), (dict(table_width=1 << 27), _lib.ERR_SHAPE),
    (dict(num_pages=1 << 62, page_size=1 << 62), _lib.ERR_SHAPE),
    (dict(max_tokens=1 << 26, heads=64, kv_heads=1), _lib.ERR_SHAPE),
]
POINTERS = [(dict([(n, None)]), _lib.ERR_NULL) for n in ("block_tables", "held", "ring", "ring_state", "slots", "positions",
                                                        "token_request", "starts", "status", "masks", "schedule")]


@pytest.mark.parametrize("kw,code", SIZES + POINTERS + [(dict(schedule=DUMMY + 4), _lib.ERR_ALIGN)])
def test_plan_is_checked_by_every_call(lib, kw, code):
    p = ctypes.byref(_plan(**kw))
    assert lib.afa_paged_build(p, DUMMY, DUMMY, None, None) == code
    assert lib.afa_paged_append(p, DUMMY, DUMMY, DUMMY, None, DUMMY, DUMMY, DUMMY, None, None, None, 0, None, 1, None,
                                None) == code
    assert lib.afa_paged_fwd(p, DUMMY, None, DUMMY, DUMMY, None, None, DUMMY, None, 0.5, 0, None, 0, None) == code
    if (kw, code) in SIZES:
        assert lib.afa_paged_schedule_bytes(p) == 0 and lib.afa_paged_workspace_size(p) == 0


def test_no_plan(lib):
    assert lib.afa_paged_build(None, DUMMY, DUMMY, None, None) == _lib.ERR_NULL
    assert lib.afa_paged_schedule_bytes(None) == 0 and lib.afa_paged_workspace_size(None) == 0


def test_build_arguments(lib):
    p = ctypes.byref(_plan())
    assert lib.afa_paged_build(p, None, DUMMY, None, None) == _lib.ERR_NULL
    assert lib.afa_paged_build(p, DUMMY, None, None, None) == _lib.ERR_NULL


def _append(lib, p=None, q=DUMMY, k=DUMMY, v=DUMMY, out=DUMMY, kp=DUMMY, vp=DUMMY, rc=DUMMY, rs=DUMMY, n=9, pos=None, axes=1,
            sections=None):
    sections = None if sections is None else (ctypes.c_int32 * len(sections))(*sections)
    return lib.afa_paged_append(ctypes.byref(p or _plan()), q, k, v, None, out, kp, vp, None, rc, rs, n, pos, axes, sections,
                                None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ERR_NULL), (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL),
    (dict(kp=None), _lib.ERR_NULL), (dict(vp=None), _lib.ERR_NULL), (dict(out=None), _lib.ERR_NULL),
    (dict(rs=None), _lib.ERR_ROTARY), (dict(n=0), _lib.ERR_ROTARY), (dict(p=_plan(head_dim=63)), _lib.ERR_ROTARY),
    (dict(axes=2), _lib.ERR_NULL), (dict(axes=2, pos=DUMMY), _lib.ERR_NULL), (dict(axes=0, pos=DUMMY), _lib.ERR_ROTARY),
    (dict(axes=5, pos=DUMMY, sections=[1] * 5), _lib.ERR_ROTARY),
    (dict(axes=2, pos=DUMMY, sections=[16, 17]), _lib.ERR_ROTARY),
    (dict(axes=2, pos=DUMMY, sections=[-1, 4]), _lib.ERR_ROTARY),
    (dict(axes=2, pos=DUMMY, sections=[2 ** 31 - 1, 2 ** 31 - 1]), _lib.ERR_ROTARY),
])
def test_append_arguments(lib, kw, code):
    assert _append(lib, **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ERR_NULL), (dict(kp=None), _lib.ERR_NULL), (dict(vp=None), _lib.ERR_NULL),
    (dict(out=None), _lib.ERR_NULL), (dict(sink=-1.0), _lib.ERR_SINK), (dict(sink=math.nan), _lib.ERR_SINK),
    (dict(sink=math.inf), _lib.ERR_SINK), (dict(p=_plan(max_tree=0), masks=DUMMY), _lib.ERR_UNSUPPORTED),
    (dict(p=_plan(max_tokens=1 << 26, heads=1, kv_heads=1)), _lib.ERR_SHAPE),
])
def test_fwd_arguments(lib, kw, code):
    call = dict(p=_plan(), q=DUMMY, kp=DUMMY, vp=DUMMY, masks=None, out=DUMMY, sink=0.5)
    call.update(kw)
    assert lib.afa_paged_fwd(ctypes.byref(call["p"]), call["q"], None, call["kp"], call["vp"], None, call["masks"],
                             call["out"], None, call["sink"], 0, None, 0, None) == code


def _axes(lib, dt=_lib.AFA_BF16, B=1, H=2, K=2, L=4, D=8, q=DUMMY, k=DUMMY, yq=DUMMY, yk=DUMMY, rc=DUMMY, rs=DUMMY, n=9,
          pos=DUMMY, esz=8, axes=2, sections=(2, 2)):
    cuts = None if sections is None else (ctypes.c_int32 * len(sections))(*sections)
    return lib.ago_rotate_axes(dt, B, H, K, L, D, q, k, yq, yk, None, rc, rs, n, pos, esz, 0, axes, cuts, 0, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=9), _lib.ERR_DTYPE), (dict(B=0), _lib.ERR_SHAPE), (dict(H=0), _lib.ERR_SHAPE), (dict(K=-1), _lib.ERR_SHAPE),
    (dict(L=0), _lib.ERR_SHAPE), (dict(D=0), _lib.ERR_SHAPE), (dict(q=None), _lib.ERR_NULL), (dict(k=None), _lib.ERR_NULL),
    (dict(yq=None), _lib.ERR_NULL), (dict(yk=None), _lib.ERR_NULL), (dict(rc=None), _lib.ERR_NULL),
    (dict(rs=None), _lib.ERR_NULL), (dict(pos=None), _lib.ERR_NULL), (dict(esz=2), _lib.ERR_UNSUPPORTED),
    (dict(n=0), _lib.ERR_ROTARY), (dict(D=7), _lib.ERR_ROTARY), (dict(sections=(3, 2)), _lib.ERR_ROTARY),
    (dict(sections=(-1, 2)), _lib.ERR_ROTARY), (dict(sections=None), _lib.ERR_NULL), (dict(axes=0), _lib.ERR_ROTARY),
    (dict(axes=5, sections=(0,) * 5), _lib.ERR_ROTARY), (dict(B=1 << 40, L=1 << 40), _lib.ERR_SHAPE),
    (dict(B=1 << 16, L=1 << 16), _lib.ERR_SHAPE),
])
def test_rotate_axes_arguments(lib, kw, code):
    assert _axes(lib, **kw) == code


# ------------------------------------------------------------------------------ the Python layer
def test_pool_and_plan_sizes():
    for bad in (0, -1, 1.5):
        with pytest.raises(ValueError, match="num_pages"):
            A.PagePool(bad, 16, 1, 16)
        with pytest.raises(ValueError, match="max_len"):
            A.PagePool(1, 16, 1, bad)
    with pytest.raises(ValueError, match="2\\^31"):
        A.PagePool(1 << 27, 16, 1, 16)
    with pytest.raises(RuntimeError, match="HIP device|GPU"):
        A.PagePool(4, 16, 1, 64, device="cpu")
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="HIP device"):
            A.PagePool(4, 16, 1, 64)

    class Pool:
        device = torch.device("cpu")

    new = dict(heads=4, kv_heads=2, head_dim=64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiple"):
        A.DraftPlan(Pool(), 8, **{**new, "kv_heads": 3})
    with pytest.raises(ValueError, match="max_new"):
        A.DraftPlan(Pool(), 8, max_new=0, **new)
    with pytest.raises(ValueError, match="max_tree"):
        A.DraftPlan(Pool(), 8, max_tree=32, **new)
    with pytest.raises(ValueError, match="max_tokens"):
        A.DraftPlan(Pool(), 0, **new)


def test_axis_rotation_refusals():
    q, k = torch.zeros(2, 4, 6, 8), torch.zeros(2, 2, 6, 8)
    tables = (torch.ones(10, 4), torch.zeros(10, 4))
    at = torch.zeros(6, 2, dtype=torch.int64)
    call = lambda q=q, k=k, t=tables, p=at, s=(2, 2): A.apply_ago_axis_rotations(q, k, t, p, s)  # noqa: E731
    with pytest.raises(RuntimeError, match="GPU"):
        call()
    for bad in (k[0], k[:1], k[:, :, :5], k[..., :4]):
        with pytest.raises(ValueError):
            call(k=bad)
    with pytest.raises(TypeError, match="dtype"):
        call(k=k.double())
    with pytest.raises(TypeError):
        call(q=q.int())
    with pytest.raises(ValueError, match="even"):
        call(q=q[..., :7], k=k[..., :7])
    with pytest.raises(TypeError, match="int32 or int64"):
        call(p=at.float())
    for bad in (at[:5], at[0], torch.zeros(3, 6, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="positions"):
            call(p=bad)
    for bad in ((2,), (3, 2), (-1, 2), (1.5, 1), None):
        with pytest.raises(ValueError, match="sections"):
            call(s=bad)
    with pytest.raises(ValueError, match="axes"):
        call(p=torch.zeros(6, 5, dtype=torch.int64), s=(1,) * 5)
    with pytest.raises(ValueError, match="axes"):
        call(p=torch.zeros(6, 0, dtype=torch.int64), s=())


def _stub_rotation(monkeypatch):
    """The rotation's checks and autograd on the CPU, with the launch left out."""
    from algebraic_intelligence_amd import attention

    monkeypatch.setattr(_lib, "require_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(attention, "_axes_launch", lambda q, k, *rest: (torch.zeros(q.shape), None if k is None else
                                                                        torch.zeros(k.shape)))


def test_axis_rotation_refuses_tangents(monkeypatch):
    """A dual q or k is refused, also where no gradient is recorded, and never comes back without its tangent."""
    from torch.autograd import forward_ad

    _stub_rotation(monkeypatch)
    q, k = torch.ones(2, 4, 6, 8), torch.ones(2, 2, 6, 8)
    tables, at = (torch.ones(10, 4), torch.zeros(10, 4)), torch.zeros(6, 2, dtype=torch.int64)
    call = lambda q, k: A.apply_ago_axis_rotations(q, k, tables, at, (2, 2))  # noqa: E731
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(q), None), (dual(q), k), (q, dual(k))):
            with pytest.raises(NotImplementedError):
                call(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call(*args)
        assert call(q, k)[1].shape == k.shape and call(q, None).shape == q.shape
    assert call(q, k)[0].shape == q.shape


class _StubPlan:
    """What the serving calls look at before any device work, on the CPU."""

    def __init__(self, dtype=torch.float32):
        self.dtype, self.device, self.head_dim, self.max_tree, self.max_tokens, self.heads = dtype, torch.device("cpu"), 8, 64, 6, 4
        self._q_shape, self._kv_shape, self._page_shape = (6, 4, 8), (6, 2, 8), (3, 2, 16, 8)
        self.masks = torch.zeros(6, 1, dtype=torch.int64)
        self._q_bytes, self._page_bytes = 6 * 4 * 8 * dtype.itemsize, 3 * 2 * 16 * 8 * dtype.itemsize

    def tensors(self):
        new = lambda shape: torch.zeros(shape, dtype=self.dtype)  # noqa: E731
        return {"q": new(self._q_shape), "k": new(self._kv_shape), "v": new(self._kv_shape), "k_pages": new(self._page_shape),
                "v_pages": new(self._page_shape)}


def _serve(plan, t, **kw):
    """(name, call) of the two serving calls on tensors t."""
    rotary = torch.ones(9, 4), torch.zeros(9, 4)
    return [("append_to_cache", lambda: A.append_to_cache(t["q"], t["k"], t["v"], t["k_pages"], t["v_pages"], plan, rotary)),
            ("paged_tree_afa", lambda: A.paged_tree_afa(t["q"], t["k_pages"], t["v_pages"], plan, **kw))]


def _reaches_the_device(call):
    """Every check of the call passes: it ends only where it asks for the GPU."""
    if not torch.cuda.is_available():
        with pytest.raises((RuntimeError, AttributeError, ctypes.ArgumentError, AssertionError)) as e:
            call()
        assert "gradient" not in str(e.value) and "overlap" not in str(e.value) and "tangent" not in str(e.value)


@pytest.mark.parametrize("name", ["q", "k", "v", "k_pages", "v_pages"])
def test_serving_refuses_what_needs_a_gradient(name):
    """No input loses a gradient or a tangent without a word; under no_grad the same tensors are taken."""
    from torch.autograd import forward_ad

    plan = _StubPlan()
    t = plan.tensors()
    plain = t[name]
    for what, call in _serve(plan, t):
        if name in ("k", "v") and what == "paged_tree_afa":
            continue
        t[name] = plain.clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match=f"{what} has no gradient"):
            call()
        with torch.no_grad():
            _reaches_the_device(call)
        with forward_ad.dual_level():
            t[name] = forward_ad.make_dual(plain, torch.ones_like(plain))
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                call()
            t[name] = plain
            _reaches_the_device(call)
    out = plain.clone().requires_grad_(True)
    if name == "q":
        with pytest.raises(RuntimeError, match="no gradient"):
            A.paged_tree_afa(plain, t["k_pages"], t["v_pages"], plan, out=out)


def test_serving_refuses_shared_places():
    """Pages that would be written twice, and results over what other workgroups still read."""
    plan = _StubPlan()
    t = plan.tensors()
    append = lambda: _serve(plan, t)[0][1]()  # noqa: E731
    attend = lambda out: _serve(plan, t, out=out)[1][1]  # noqa: E731
    for call in (append, attend(torch.zeros(6, 4, 8))):
        _reaches_the_device(call)
    n = t["k_pages"].numel()
    room = torch.zeros(2 * n)
    apart = room[n:].view(plan._page_shape)
    t["k_pages"] = room[:n].view(plan._page_shape)
    for bad in (t["k_pages"], room[8:n + 8].view(plan._page_shape), room[n - 8:2 * n - 8].view(plan._page_shape)):
        t["v_pages"] = bad
        with pytest.raises(ValueError, match="overlap"):
            append()
    t["v_pages"] = apart
    _reaches_the_device(append)
    t["v_pages"] = torch.zeros(3, 1, 16, 8).expand(3, 2, 16, 8)
    with pytest.raises(ValueError, match="expanded"):
        append()
    both = torch.zeros(3, 16, 2, 2, 8)  # keys and values side by side share no place
    t["k_pages"], t["v_pages"] = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    _reaches_the_device(append)
    t["v_pages"] = t["k_pages"]
    with pytest.raises(ValueError, match="overlap"):
        append()
    t["k_pages"], t["v_pages"] = room[:n].view(plan._page_shape), apart
    for at in (0, n - 1, 2 * n - 192):
        with pytest.raises(ValueError, match="overlap"):
            attend(room[at:at + 192].view(6, 4, 8))()
