"""Attention behind a shared prefix where scores are far from 0, against float64.

The scores are formed without a rounding: q and k hold small whole numbers times a power of two, and their products' sums stay
below 2^24.  Scaling one rounds twice, off by 2 u of it, which is at most 16 u of the weight (d ln rho^8 / ds = 8 / sqrt(1 + s^2)).
So a weight is off by (105 + 16) u, 2.2e-4 more on bf16 and fp16 inputs (tests/test_paged_gpu.py), and by what the planes of the
product and the sums over the keys add there."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from tests.test_paged_gpu import BF16, F16, F32, U, _half, _tiny, _weight_error
from tests.test_prefix_gpu import _Shared

pytestmark = pytest.mark.gpu


class _Exact(_Shared):
    """Requests of one token each, or prompts, without drafted trees, whose q and keys are set by `place`."""

    def __init__(self, dt, lens, H, K, D, L):
        super().__init__(dt, lens, H, K, D, 16, L, seed=D, max_tree=0, parents=False)

    def place(self, q, prefix, own):
        """q (T, H, D), prefix (K, L, D), and own(r, c + n): a request's keys, (c + n, K, D)."""
        to = lambda x: torch.tensor(x, device="cuda").to(self.dt)  # noqa: E731
        self.q, self.pk = to(q), to(prefix)
        for r, (c, n) in enumerate(self.lens):
            self.k[r] = to(own(r, c + n))
            at = torch.arange(c + n, device="cuda")
            pg = torch.tensor(self.tables[r], device="cuda", dtype=torch.int64)[at // 16]
            self.kp[pg, :, at % 16] = self.k[r]

    def compare(self, sink, what):
        out, den = (t.double().cpu().numpy() for t in self.call(sink, return_denominator=True))
        q, pk, pv = (t.double().cpu().numpy() for t in (self.q, self.pk, self.pv))
        for r, (c, n) in enumerate(self.lens):
            k, v = self.k[r].double().cpu().numpy(), self.v[r].double().cpu().numpy()
            for i in range(n):
                t, seen = self.starts[r] + i, c + i + 1
                for h in range(self.H):
                    kh = h * self.K // self.H
                    keys, values = np.concatenate((pk[kh], k[:seen, kh])), np.concatenate((pv[kh], v[:seen, kh]))
                    want, d, size, _ = P.attention_row(q[t, h], keys, values, sink)
                    e = _weight_error(self.dt, self.D, 0, len(keys)) + 16 * U
                    # a sum this far down is in fp32's subnormals, a step of 2^-149 of them for every key
                    low = 2 * len(keys) * 2.0 ** -149 / d
                    bound = (2 * e + self.plane()) * size + (_half(self.dt) + 4 * U) * np.abs(want) + _tiny(self.dt) + low
                    off = np.abs(out[t, h] - want) - bound
                    assert off.max() <= 0, (what, "row", t, h, out[t, h, :4], want[:4], float(off.max()))
                    assert abs(den[t, h] - d) <= 2 * e * d + 2 * len(keys) * 2.0 ** -149, (what, "denominator", t, h, den[t, h], d)


LENS = [(0, 30), (3, 45), (20, 25)]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("where", ["all", "first", "own"])
@pytest.mark.parametrize("few", [False, True])
def test_prefix_far_below(dt, D, where, few):
    """Scores from about -10 to -13000: of every key, without a sink; of the first two tiles of a prefix whose other keys are
    ordinary ones; of the prefix alone.  Rows of one size, and of many beside each other; few and many rows a key head."""
    rng = np.random.default_rng(D)
    x = _Exact(dt, [(0, 9), (5, 13)] if few else LENS, 4, 2, D, 300)
    T = x.q.shape[0]
    m = rng.integers(1, 4, (T, 4, D)).astype(np.float64)
    far = lambda n: -rng.integers(3, 6, (n, 2, D)).astype(np.float64)  # noqa: E731
    near = lambda n: np.where(np.arange(D) == 0, rng.choice([-1.0, 1.0], (n, 2, 1)), 0.0)  # noqa: E731
    prefix = far(300)
    if where == "first":
        prefix[64:] = near(236)
    sizes = [0.125, 0.5, 2, 8, 16, 24, 32, 48, 64, 96, 128]
    mixed = rng.choice(sizes, (T, 4, 1))
    for size in [*(sizes if dt == F16 else sizes[::3]), mixed]:
        x.place(m * size, prefix.transpose(1, 0, 2), lambda r, n: (far if where == "all" else near)(n))
        x.compare(0.0 if where == "all" else 0.5, (where, "mixed" if size is mixed else size))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("few", [False, True])
def test_prefix_far_above(dt, D, few):
    """One key of a score up to 30000, whose weight of up to 2^127 is a row's, beside ordinary ones; v is at most 1."""
    rng = np.random.default_rng(D)
    x = _Exact(dt, [(0, 9), (5, 13)] if few else LENS, 4, 2, D, 70)
    T = x.q.shape[0]
    x.pv.clamp_(-1, 1)
    prefix = np.zeros((2, 70, D))
    prefix[:, :, 0] = rng.choice([-1.0, 1.0], (2, 70))
    prefix[:, 40, 0] = 64.0
    q = np.zeros((T, 4, D))
    for score in (3000, 14000, 22000, 25000, 29000):
        # q's first feature in steps that bf16 holds
        q[..., 0] = np.floor(score * np.sqrt(D) / 64 / 32) * 32 if dt == BF16 else np.floor(score * np.sqrt(D) / 64)
        x.place(q, prefix, lambda r, n: np.where(np.arange(D) == 0, rng.choice([-1.0, 0.0], (n, 2, 1)), 0.0))
        x.compare(0.5, score)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 32), (F16, 48), (F16, 96), (F16, 128), (F32, 48)])
@pytest.mark.parametrize("few", [False, True])
def test_prefix_where_weights_end(dt, D, few):
    """Keys of one score beyond -27554, prefix and own, weigh 2^-126 each: without a sink a row is the mean of all values, however far
    the keys are.  The mean of N values is off by N u of their sizes and its own rounding."""
    x = _Exact(dt, [(0, 9), (5, 13)] if few else LENS, 4, 2, D, 90)
    T = x.q.shape[0]
    one = lambda n: np.broadcast_to(np.where(np.arange(D) == 0, -64.0, 0.0), (n, 2, D))  # noqa: E731
    for score in (29000, 1e5, 7e5) if dt == F16 else (29000, 1e5, 1e9, 1e17, 1e36):
        q = score * np.sqrt(D) / 64
        x.place(np.full((T, 4, D), min(q, 60000.0) if dt == F16 else q), one(90).transpose(1, 0, 2), lambda r, n: one(n))
        out, den = (t.double().cpu().numpy() for t in x.call(0.0, return_denominator=True))
        pv = x.pv.double().cpu().numpy()
        for r, (c, n) in enumerate(x.lens):
            v = x.v[r].double().cpu().numpy()
            for i in range(n):
                t, seen = x.starts[r] + i, c + i + 1
                for h in range(4):
                    values = np.concatenate((pv[h // 2], v[:seen, h // 2]))
                    want, size = values.mean(0), np.abs(values).mean(0)
                    bound = 2 * len(values) * U * size + (_half(dt) + 4 * U) * np.abs(want) + _tiny(dt)
                    assert (np.abs(out[t, h] - want) <= bound).all(), (score, t, h, out[t, h, :3], want[:3])
                    assert abs(den[t, h] / 2.0 ** -126 - len(values)) <= 2 * len(values) ** 2 * U, (score, den[t, h])


@pytest.mark.parametrize("L", [30001, 65536])
@pytest.mark.parametrize("D", [32, 128])
def test_prefix_of_one_key_above_very_many_in_fp16(D, L):
    """A first key of large weight and value 0, then keys of one weight and value 1, which so are all of a row's result: rows with
    from 2^-14 to 2^-26 of the first one's weight for each of them.

    A row's factor leaves its largest weight at 16 or above, so that fp16 holds the others to half a step of it, 2^-11, or to half of
    its smallest one: 2^-25 / 16 of the largest.  Equal weights of 11 bits add up without a rounding within the 16 keys of a
    product, whose result is added to the sum by one rounding or a cut, 2^-23: L / 16 of them.  The row sums add L / 32 of
    fp32 weights by u each, and those of a tile by 5 u."""
    K = 2 * torch.cuda.get_device_properties(0).multi_processor_count  # one workgroup has all of a head's prefix
    T = 96
    x = _Shared(F16, [(0, 1)] * T, K, K, D, 16, 16, seed=1, max_tree=0, parents=False)
    a = 1.0 + np.arange(T) / 64
    first, small = 5.0, np.exp2(-(14 + 12 * np.arange(T) / (T - 1)) / 8)  # (rho's eighth root of the shares)
    rho = first * a + np.sqrt(1 + (first * a) ** 2)
    s = (rho * small - 1 / (rho * small)) / 2  # rho(s) = rho * small
    q = np.zeros((T, 1, D))
    q[:, 0, 0], q[:, 0, 1] = a * np.sqrt(D), s * np.sqrt(D)
    x.q = torch.tensor(q, device="cuda").half().expand(T, K, D).contiguous()
    pk = torch.zeros(1, L, D, device="cuda", dtype=F16)
    pk[:, 0, 0], pk[:, 1:, 1] = first, 1.0
    pv = torch.ones(1, L, D, device="cuda", dtype=F16)
    pv[:, 0] = 0.0
    x.pk, x.pv = pk.expand(K, L, D), pv.expand(K, L, D)
    x.kp.zero_(), x.vp.zero_()  # a row's own key weighs 1, its value is 0
    out, den = x.call(0.5, return_denominator=True)
    assert torch.equal(out, out[:, :1].expand_as(out)) and torch.equal(den, den[:, :1].expand_as(den))
    q = x.q[:, 0].double().cpu().numpy()
    weigh = lambda score: P.rho8(score / np.sqrt(D))  # noqa: E731
    top, low = weigh(q[:, 0] * first), weigh(q[:, 1])
    wden = top + (L - 1) * low + 1.5
    want = (L - 1) * low / wden
    e = (121 + 16 + L / 32 + 5) * U + 2.2e-4
    got, gden = out[:, 0].double().cpu().numpy(), den[:, 0].double().cpu().numpy()
    bound = (2 * e + L / 16 * 2.0 ** -23 + 2.0 ** -11 + 2.0 ** -11) * want + (L - 1) * 2.0 ** -29 * np.maximum(top, low) / wden
    off = np.abs(got - want[:, None]) - bound[:, None]
    at = int(np.argmax(off.max(1)))
    assert off.max() <= 0, ("row", at, got[at, 0], want[at], bound[at], low[at] / top[at])
    assert (np.abs(gden - wden) <= e * wden).all()
