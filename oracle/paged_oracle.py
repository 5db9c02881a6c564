"""Plain restatements, in Python and 64 bits on the CPU, of the paged cache's bookkeeping, its attention, packed
sequences' attention and token log probabilities. They follow the definitions, not the kernels."""
from __future__ import annotations

import math

import torch


class Tables:
    """The bookkeeping of a paged cache, one request and one page at a time."""

    def __init__(self, n_streams: int, n_pages: int, page: int, max_len: int):
        self.page, self.max_len = page, max_len
        self.rows = [[] for _ in range(n_streams)]
        self.lens = [0] * n_streams
        self.free = list(range(n_pages - 1, -1, -1))

    def plan(self, streams, new, total):
        starts, slots, positions, seen, cu, short = [], [-1] * total, [0] * total, set(), [0], 0
        for s, m in zip(streams, new):
            first = s not in seen
            seen.add(s)
            ok = 0 <= s < len(self.rows) and first and m >= 0 and self.lens[s] + m <= self.max_len
            if ok:
                need = max(0, -(-(self.lens[s] + m) // self.page) - len(self.rows[s]))
                ok = need == 0 or short + need <= len(self.free)
                short += 0 if ok else need  # those behind stand behind it
            if ok:
                start = self.lens[s]
                self.rows[s] += [self.free.pop() for _ in range(need)]
                self.lens[s] += m
                for t in range(m):
                    at = cu[-1] + t
                    if at < total:
                        positions[at] = start + t
                        slots[at] = self.rows[s][(start + t) // self.page] * self.page + (start + t) % self.page
            starts.append(start if ok else -1)
            cu.append(min(cu[-1] + max(m, 0), total))
        return cu, starts, slots, positions

    def truncate(self, streams, lens):
        seen, back = set(), []
        for s, n in zip(streams, lens):
            first = s not in seen
            seen.add(s)
            if not (0 <= s < len(self.rows) and first and 0 <= n <= self.lens[s]):
                continue
            keep = -(-n // self.page)
            back += self.rows[s][keep:]
            self.rows[s], self.lens[s] = self.rows[s][:keep], n
        self.free += back[::-1]


def attention(q, k, v, limit, scale):
    """fp64 softmax(scale q k) v: q ``[n, H, D]``, k and v ``[L, Hk, D]``, query t sees the keys below ``limit[t]``; none: zeros.
    What a query does not see does not count, whatever it is. Also the largest sum of |q| |k| of a score."""
    n, H, D = q.shape
    Hk = k.shape[1]
    out, big = torch.zeros(n, H, D, dtype=torch.float64), 0.0
    q, k, v = q.double(), k.double(), v.double()
    for t in range(n):
        m = int(limit[t])
        if m <= 0:
            continue
        for h in range(H):
            kk, vv = k[:m, h // (H // Hk)], v[:m, h // (H // Hk)]
            out[t, h] = torch.softmax(kk @ q[t, h] * scale, 0) @ vv
            big = max(big, float((kk.abs() @ q[t, h].abs()).max()))
    return out, big


def logprobs(x, tokens, top, blocked=None):
    """fp64 log probabilities, entropies, and the alternatives' log probabilities and ids, row by row."""
    x = x.double()
    if blocked is not None:
        x = x.masked_fill(blocked[:, : x.shape[1]], -math.inf)
    lp, entropy, values, ids = [], [], [], []
    for row, t in zip(x, tokens.tolist()):
        V = row.numel()
        if bool((row.isnan() | (row == math.inf)).any()):
            lp.append(math.nan), entropy.append(math.nan), values.append([math.nan] * top), ids.append([-1] * top)
            continue
        m = float(row.max())
        if m == -math.inf:
            d, log_z, h = row, 0.0, 0.0
        else:
            d = row - m
            e = d.exp()
            log_z = math.log1p(float(e.sum()) - 1.0)
            h = log_z - float((e * d.masked_fill(e == 0, 0)).sum() / e.sum())
        lp.append(float(d[t]) - log_z if 0 <= t < V else math.nan)
        entropy.append(h)
        order = sorted((i for i in range(V) if row[i] > -math.inf), key=lambda i: (-float(row[i]), i))[:top]
        values.append([float(d[i]) - log_z for i in order] + [-math.inf] * (top - len(order)))
        ids.append(order + [-1] * (top - len(order)))
    f = lambda a: torch.tensor(a, dtype=torch.float64)
    return f(lp), f(entropy), f(values).view(len(lp), top), torch.tensor(ids, dtype=torch.int64).view(len(lp), top)
