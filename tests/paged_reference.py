"""64-bit statements of the paged batch operators (include/plamo_paged.h) and
the scenes their tests run on: page tables in a shuffled pool whose every
unused row holds NaN, so that a read past a length shows."""
import math

import numpy as np
import torch

ROWS, DIM = 64, 128


def pages_for(rows):
    return -(-rows // ROWS)


def plan_by_hand(held, added, tables, free, rows, base, head=0):
    """The plan one row after another (a step that fits)."""
    tables = [list(t) for t in tables]
    lengths, starts, slots, positions = [], [0], [], []
    for r, (h, n) in enumerate(zip(held, added)):
        for i in range(h, h + n):
            if i % ROWS == 0:
                tables[r][i // ROWS] = free[head]
                head += 1
            slots.append(tables[r][i // ROWS] * ROWS + i % ROWS)
            positions.append(base + i)
        lengths.append(h + n)
        starts.append(len(slots))
    new = len(slots)
    slots += [-1] * (rows - new)
    positions += [0] * (rows - new)
    return lengths, starts, slots, positions, [0, new, head, max(lengths, default=0)], tables


def rotate_store(qkv, q_norm, k_norm, table, positions, query_heads, kv_heads):
    """(queries, keys, values) of every row, in 64 bits."""
    x = qkv.double().cpu().reshape(qkv.shape[0], -1, DIM)
    turn = table.double().cpu()[positions.long().cpu()]
    cos, sin = turn[:, None, :DIM // 2], turn[:, None, DIM // 2:]

    def heads(part, weight):
        part = part / torch.sqrt((part ** 2).mean(-1, keepdim=True) + 1e-6) * (weight.double().cpu() + 1)
        a, b = part[..., :DIM // 2], part[..., DIM // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q, k, v = x.split([query_heads, kv_heads, kv_heads], 1)
    return heads(q, q_norm), heads(k, k_norm), v


class Scene:
    """A batch for attention: requests of (held, new) own rows behind `prefix`
    rows, in a pool of `dtype` with shuffled pages. The keys and values that
    exist are kept in 64 bits; every other row of the pool is NaN."""

    def __init__(self, requests, prefix, query_heads, kv_heads, dtype, seed=0, spare_rows=0, spread=1.5, pool_pages=None,
                 device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.requests, self.prefix = list(requests), prefix
        self.qh, self.kh, self.dtype = query_heads, kv_heads, dtype
        lengths = [h + n for h, n in self.requests]
        counts = [pages_for(n) for n in lengths]
        need = sum(counts) + pages_for(prefix)
        pages = pool_pages or need + 3
        order = torch.randperm(need + 3, generator=g) + (pages - need - 3)  # the pool's last pages
        self.prefix_pages = order[:pages_for(prefix)].int().to(device)
        rest = order[pages_for(prefix):].tolist()
        stride = max(counts, default=0) + 2
        tables = torch.full((len(lengths), stride), -7, dtype=torch.int32)  # -7: no page, never to be read
        self.pool = torch.empty(pages, 2, ROWS, kv_heads, DIM, dtype=dtype, device=device)
        self.pool[pages - need - 3:] = float("nan")

        def fill(ids, count):
            kv = [torch.randn(count, kv_heads, DIM, generator=g).to(dtype) for _ in range(2)]
            for i, page in enumerate(ids):
                n = min(ROWS, count - i * ROWS)
                for kind in (0, 1):
                    self.pool[page, kind, :n] = kv[kind][i * ROWS:i * ROWS + n].to(device)
            return [t.double() for t in kv]

        self.shared = fill(self.prefix_pages.tolist(), prefix)
        self.own = []
        for r, n in enumerate(lengths):
            ids, rest = rest[:counts[r]], rest[counts[r]:]
            tables[r, :counts[r]] = torch.tensor(ids, dtype=torch.int32)
            self.own.append(fill(ids, n))
        new = [n for _, n in self.requests]
        self.rows = sum(new) + spare_rows
        self.tables = tables.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=device)
        self.q = (torch.randn(self.rows, query_heads, DIM, generator=g) * spread).to(dtype).to(device)

    def expected(self, window=0, scale=DIM ** -0.5):
        """(result, tolerance) for every element.

        Tolerance, from the operator's roundings with A = sum p |v| / sum p:
        a BF16 result is rounded once (8 bits: 2^-8 |o|), and its softmax weights too,
        above and below the fraction line (2 * 2^-8 A). Scores err by at most
        E = scale * max_j sum |q k_j| * 2^-17 (32 chained adds that truncate,
        2^-23 each, and FP32 terms dropped below 2^-21), weights by e^E - 1,
        twice again; 2^-17 A covers the exponentials and the FP32 sums.
        """
        g = self.qh // self.kh
        out = torch.zeros(self.rows, self.qh, DIM, dtype=torch.float64)
        tol = torch.full_like(out, 1e-30)
        q = self.q.double().cpu()
        row = 0
        for r, (held, new) in enumerate(self.requests):
            k = torch.cat([self.shared[0], self.own[r][0]])
            v = torch.cat([self.shared[1], self.own[r][1]])
            for i in range(new):
                at = self.prefix + held + i
                lo = max(0, at + 1 - window) if window else 0
                kk, vv = k[lo:at + 1], v[lo:at + 1]
                for h in range(self.kh):
                    heads = slice(h * g, (h + 1) * g)
                    s = q[row, heads] @ kk[:, h].T * scale
                    p = torch.softmax(s, -1)
                    out[row, heads] = p @ vv[:, h]
                    a = p @ vv[:, h].abs()
                    e = (q[row, heads].abs() @ kk[:, h].abs().T).amax(-1, keepdim=True) * abs(scale) * 2.0 ** -17
                    t = a * (2 * torch.expm1(e) + 2.0 ** -17)
                    if self.dtype == torch.bfloat16:
                        t = t + 2.0 ** -8 * out[row, heads].abs() + 2 * 2.0 ** -8 * a
                    tol[row, heads] = t
                row += 1
        return out, tol


def check(got, want, tol, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs()
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"
