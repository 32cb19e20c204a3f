"""64-bit statements of the operators for draft trees and adapters
(include/plamo_paged.h), and the scenes their tests run on."""

import torch

from paged_reference import DIM, Scene, pages_for


def random_tree(rows, g, depth=None):
    """Parents of a tree of `rows` rows, each below an earlier one (of less than `depth` generations)."""
    parents, depths = [], []
    for i in range(rows):
        open_rows = [j for j in range(i) if depth is None or depths[j] < depth]
        p = open_rows[int(torch.randint(len(open_rows), (1,), generator=g))] if open_rows else -1
        parents.append(p)
        depths.append(0 if p < 0 else depths[p] + 1)
    return parents


def line_of(parents, i):
    """A row and those above it, the farthest first."""
    line = [i]
    while parents[line[0]] >= 0:
        line.insert(0, parents[line[0]])
    return line


def tree_by_hand(trees, held, words, base, rows):
    """(positions, masks as lists of unsigned words) of the batch, padding included."""
    positions, masks = [], []
    for parents, h in zip(trees, held):
        for i in range(len(parents)):
            line = line_of(parents, i)
            positions.append(base + h + len(line) - 1)
            masks.append([sum(1 << (j - 32 * w) for j in line if j // 32 == w) for w in range(words)])
    pad = rows - len(positions)
    return positions + [0] * pad, masks + [[0] * words] * pad


def signed(masks):
    return torch.tensor([[w - (w >> 31 << 32) for w in row] for row in masks], dtype=torch.int32)


class TreeScene(Scene):
    """A batch of draft trees for attention: `requests` are (held, parents)."""

    def __init__(self, requests, prefix, query_heads, kv_heads, dtype, seed=0, words=None, **more):
        super().__init__([(h, len(parents)) for h, parents in requests], prefix, query_heads, kv_heads, dtype, seed=seed, **more)
        self.trees = [list(parents) for _, parents in requests]
        most = max((len(t) for t in self.trees), default=0)
        self.words = words or max(1, -(-most // 32))
        _, masks = tree_by_hand(self.trees, [h for h, _ in requests], self.words, 0, self.rows)
        # what each row sees of its request's new rows
        self.sees = [[line_of(parents, i) for i in range(len(parents))] for parents in self.trees]
        self.masks = signed(masks).reshape(self.rows, self.words).to(self.q.device)

    def set_masks(self, sees):
        """Any masks: per request and row the new rows seen, in rising order."""
        self.sees = sees
        masks = [[sum(1 << (j - 32 * w) for j in row if j // 32 == w) for w in range(self.words)] for r in sees for row in r]
        masks += [[0] * self.words] * (self.rows - len(masks))
        self.masks = signed(masks).reshape(self.rows, self.words).to(self.q.device)

    def expected(self, window=0, scale=DIM ** -0.5):
        """(result, tolerance) for every element.

        Tolerance with A = sum p |v| / sum p: scores err by at most E = scale *
        max_j sum |q k_j| * 2^-17 (32 chained adds that truncate, 2^-23 each, and
        terms dropped below 2^-21), weights by e^E - 1, above and below the
        fraction line; 2^-15 A covers the weights' 16 bits in a BF16 value
        product, the exponentials and the FP32 sums; a BF16 result is rounded by
        2^-8 of itself at most.
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
                seen = list(range(self.prefix + held)) + [self.prefix + held + j for j in self.sees[r][i]]
                if window:
                    seen = seen[-window:]
                if seen:
                    kk, vv = k[seen], v[seen]
                    for h in range(self.kh):
                        heads = slice(h * g, (h + 1) * g)
                        s = q[row, heads] @ kk[:, h].T * scale
                        p = torch.softmax(s, -1)
                        out[row, heads] = p @ vv[:, h]
                        a = p @ vv[:, h].abs()
                        e = (q[row, heads].abs() @ kk[:, h].abs().T).amax(-1, keepdim=True) * abs(scale) * 2.0 ** -17
                        t = a * (2 * torch.expm1(e) + 2.0 ** -15)
                        if self.dtype == torch.bfloat16:
                            t = t + 2.0 ** -8 * out[row, heads].abs()
                        tol[row, heads] = t
                row += 1
        return out, tol


def accept_by_hand(trees, tokens, chosen, held, tables, free, head):
    """One request after another; lists in, lists out."""
    counts, kept, last, path, after, back = [], [], [], [], [], []
    row = 0
    for r, parents in enumerate(trees):
        n = len(parents)
        at, walked = (0 if n else -1), []
        while at >= 0:
            walked.append(at)
            below = [i for i in range(at + 1, n) if parents[i] == at and tokens[row + i] == chosen[row + at]]
            at = below[0] if below else -1
        counts.append(len(walked))
        kept.append(held[r] + len(walked))
        last.append(chosen[row + walked[-1]] if walked else -1)
        path += walked + [-1] * (n - len(walked))
        after += [chosen[row + i] for i in walked] + [-1] * (n - len(walked))
        back += tables[r][pages_for(kept[r]):pages_for(held[r] + n)]
        row += n
    free = list(free)
    free[head - len(back):head] = back
    return counts, kept, last, path, after, [0, sum(counts), head - len(back), max(kept, default=0)], free


def adapters_expected(x, base, a, b, ids, starts, scales):
    """(result, tolerance) of out = base + scale * B (A x).

    With S = sum |a x| of a rank: its products (exact: BF16 times BF16 terms) are added
    16 at a time to a chain of at most 3 columns / 128 steps, which truncate
    by 2^-22 of what is added up, and the warps' and splits' sums by 2^-24 each
    (8 + columns / 512); what the terms of an FP32 x leave out is below 2^-23. The same
    holds for B h, over 3 rank / 16 + 1 steps, its inputs off by the former; the
    product with the scale and the sum with base round by 2^-24 each, the result by
    half a step of its type.
    """
    out = base.double().cpu().clone()
    tol = torch.full_like(out, 1e-30)
    columns, rank = a.shape[2], a.shape[1]
    first = (3 * columns / 128 + 2) * 2.0 ** -22 + (8 + columns / 512) * 2.0 ** -24 + 2.0 ** -23
    second = (3 * rank / 16 + 2) * 2.0 ** -22
    for r, i in enumerate(ids):
        if i < 0:
            continue
        rows = slice(starts[r], starts[r + 1])
        aa, bb, xx = a[i].double().cpu(), b[i].double().cpu(), x[rows].double().cpu()
        s = scales[i].double().item() if scales is not None else 1.0
        h, size = xx @ aa.T, xx.abs() @ aa.abs().T
        delta = s * (h @ bb.T)
        out[rows] += delta
        spread = abs(s) * (size @ bb.abs().T)
        t = spread * first + abs(s) * (h.abs() @ bb.abs().T) * (second + 2.0 ** -23) + 2.0 ** -23 * (out[rows].abs() + delta.abs())
        if base.dtype == torch.bfloat16:
            t = t + 2.0 ** -8 * out[rows].abs()
        tol[rows] = t + 1e-30
    return out, tol


