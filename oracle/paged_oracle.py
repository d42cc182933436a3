"""Float64 / integer restatements of the paged-cache serving operators, request by request and token by
token, as their definitions read.  Test infrastructure only."""
import numpy as np

OK, NO_PAGES, TOO_LONG, TOO_MANY, PAST_END, NEGATIVE = range(6)


class Pool:
    """A pool's pages: tables as lists, the free pages as a queue."""

    def __init__(self, num_pages, page_size, requests, max_len):
        self.page_size, self.width = page_size, -(-max_len // page_size)
        self.tables = [[] for _ in range(requests)]
        self.free = list(range(num_pages))

    def step(self, cached, new, max_tokens, max_new, max_tree, parents=None):
        """(slots, positions, requests, starts, masks as rows of bools, status) of a step; the pool follows."""
        P, R = self.page_size, len(self.tables)
        status, starts, at = [], [0], 0
        grown = 0
        takes, gives = [], []
        for r in range(R):
            c, n = int(cached[r]), int(new[r])
            st = NEGATIVE if c < 0 or n < 0 else TOO_MANY if n > max_new else TOO_LONG if c + n > self.width * P else OK
            at += max(n, 0)
            if st == OK and n > 0 and at > max_tokens:
                st = PAST_END
            starts.append(min(at, max_tokens))
            held = len(self.tables[r])
            need = -(-(c + n) // P) if st == OK else held
            grown += max(need - held, 0)
            if need > held and grown > len(self.free):
                st, need = NO_PAGES, held
            status.append(st)
            takes.append(max(need - held, 0))
            gives.append(max(held - need, 0))
        taken, self.free = self.free[:sum(takes)], self.free[sum(takes):]
        for r in range(R):
            self.tables[r] += taken[:takes[r]]
            del taken[:takes[r]]
            if gives[r]:
                self.free += self.tables[r][-gives[r]:]
                del self.tables[r][-gives[r]:]
        slots, positions, requests, sees = [], [], [], []
        for r in range(R):
            n, c = starts[r + 1] - starts[r], int(cached[r])
            for i in range(n):
                row = [False] * max_tree
                if status[r] != OK:
                    slots.append(-1)
                    positions.append(0)
                else:
                    place = c + i
                    slots.append(self.tables[r][place // P] * P + place % P)
                    if n > max_tree:
                        positions.append(place)
                    else:
                        j, depth = i, -1
                        while j >= 0:
                            row[j] = True
                            depth += 1
                            up = j - 1 if parents is None else int(parents[starts[r] + j])
                            j = up if 0 <= up < j else -1
                        positions.append(c + depth)
                requests.append(r)
                sees.append(row)
        rest = max_tokens - len(slots)
        return (np.array(slots + [-1] * rest), np.array(positions + [0] * rest), np.array(requests + [-1] * rest),
                np.array(starts), np.array(sees + [[False] * max_tree] * rest).reshape(max_tokens, max_tree),
                np.array(status))


def mask_words(sees):
    """Rows of bools (T, 64 W) as int64 words (T, W)."""
    T, n = sees.shape
    bits = sees.reshape(T, n // 64, 64).astype(np.uint64) << np.arange(64, dtype=np.uint64)
    return np.bitwise_or.reduce(bits, axis=2).view(np.int64)


def rotate_axes(x, c, s, positions, sections, back=False):
    """x (B, H, L, D) by table rows positions (B, L, A), pair by pair; NaN outside the tables."""
    x = np.asarray(x, dtype=np.float64)
    y = x.copy()
    p = 0
    for a, n in enumerate(sections):
        for _ in range(n):
            m = positions[:, :, a]
            inside = (m >= 0) & (m < len(c))
            at = np.where(inside, m, 0)
            cm, sm = (np.where(inside, np.asarray(t, dtype=np.float64)[at, p], np.nan)[:, None, :] for t in (c, s))
            sm = -sm if back else sm
            y[..., 2 * p] = cm * x[..., 2 * p] - sm * x[..., 2 * p + 1]
            y[..., 2 * p + 1] = sm * x[..., 2 * p] + cm * x[..., 2 * p + 1]
            p += 1
    return y


def rho8(s):
    rho = np.abs(s) + np.sqrt(1.0 + s * s)
    return np.where(s < 0, 1.0 / rho, rho) ** 8


def attention_row(q, keys, values, sink):
    """One row over its visible keys: (out, denominator, sum_j w_j |v_j| / denominator, max_j |q||k_j|)."""
    D = q.shape[-1]
    if len(keys) == 0:
        return np.zeros(D), sink, np.zeros(D), 0.0
    w = rho8(keys @ q / np.sqrt(D))
    den = w.sum() + sink
    size = np.abs(keys) @ np.abs(q) / np.sqrt(D)
    with np.errstate(invalid="ignore"):
        return w @ values / den, den, w @ np.abs(values) / den, float(np.max(size))
