"""Float64 / integer restatements of the norms of q and k, of the weights that tokens of a cache are given and of what a cache
keeps, as their definitions read.  Test infrastructure only."""
import numpy as np

from oracle import paged_oracle as P


def norm_rotate(x, scale, eps, c, s, positions, sections):
    """x (B, H, L, D) normalised over D, scaled and turned (no tables: not turned)."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * scale
    return y if c is None else P.rotate_axes(y, c, s, positions, sections)


def norm_rotate_gradient(x, scale, eps, g, c, s, positions, sections):
    """(dx, dscale) by the quotient rule on x / n, n = sqrt(mean(x^2) + eps)."""
    x, back = np.asarray(x, np.float64), np.asarray(g, np.float64)
    if c is not None:
        back = P.rotate_axes(back, c, s, positions, sections, True)
    n = np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    h = back * scale
    dx = h / n - x * np.sum(h * x, -1, keepdims=True) / (x.shape[-1] * n ** 3)
    return dx, np.sum(back * x / n, axis=tuple(range(x.ndim - 1)))


def kept(weights, cached, budget, first, recent):
    """Places of the tokens that a request keeps, in their order: by sorting, one token at a time."""
    if cached <= budget:
        return list(range(cached))
    sure = [j for j in range(cached) if j < first or j >= cached - recent]
    rest = [j for j in range(cached) if first <= j < cached - recent]
    # NaN counts as the largest; equal weights by their place
    rest.sort(key=lambda j: (0, 0.0, j) if np.isnan(weights[j]) else (1, -float(weights[j]), j))
    return sorted(sure + rest[:budget - len(sure)])
