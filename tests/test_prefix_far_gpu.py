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
