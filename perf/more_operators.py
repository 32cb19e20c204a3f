"""Operators of a verification step with draft trees and per-request adapters: what is measured of them, and
their plain forms.

A server that verifies several drafted continuations of each request at once runs, beside the paged batch
operators that plan and store a step's rows:

  tree       once per step: positions and visibility masks of the drafted rows from their parents;
  attention  per layer: every drafted row over the prefix that all requests share, its request's held rows, and
             of the drafted ones itself and its ancestors;
  accept     once per step: the longest path of drafts that the model's choices confirm, its rows moved together
             in every layer's cache, pages that no row reaches any more back on the free list;
  adapters   beside a shared projection: out = base + scale * B (A x), with each request's own low-rank A and B.

Pages are laid out [2][64][kv heads][128]: 64 key rows, then 64 value rows. Heads have 128 dimensions, as in
every model profile of this repository.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64
DIM = 128
# hidden size, query heads, KV heads, MLP's inner size
PROFILES = {"0.8b": (1536, 16, 1, 6144), "2b": (2560, 24, 4, 10240), "8b": (4096, 32, 4, 16384),
            "31b": (5120, 64, 8, 25600)}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VOCABULARY = 100000
_backend = None


def _framework():
    """The framework's backend on this GPU, opened once as a program does."""
    global _backend
    if _backend is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(root, "plamo-3-translate.c_b200")
        spec = importlib.util.spec_from_file_location("plamo_b200", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        module = importlib.util.module_from_spec(spec)
        sys.modules["plamo_b200"] = module
        spec.loader.exec_module(module)
        _backend = module.Backend(device=0)
    return _backend


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # The eight requests that one GPU serves at a time, 16 drafts each: pure latency.
        {"name": "tree_8x16", "op": "tree", "requests": 8, "held_lo": 430, "held_hi": 455, "new_lo": 16, "new_hi": 16,
         "depth": 6, "base": 12},
        # A large server's trees of one to 64 rows.
        {"name": "tree_256x64", "op": "tree", "requests": 256, "held_lo": 0, "held_hi": 4000, "new_lo": 1, "new_hi": 64,
         "depth": 12, "base": 4097},
        # The walk and the move in the 24 layers of a small model, FP32 caches as the token loop keeps them.
        {"name": "accept_8x16_2b_fp32", "op": "accept", "model": "2b", "cache": "fp32", "layers": 24, "requests": 8,
         "held_lo": 30, "held_hi": 127, "new_lo": 16, "new_hi": 16, "depth": 6},
        # A large batch, eight layers: pages come back from most requests.
        {"name": "accept_256x64_8b_bf16", "op": "accept", "model": "8b", "cache": "bf16", "layers": 8, "requests": 256,
         "held_lo": 0, "held_hi": 190, "new_lo": 1, "new_hi": 64, "depth": 12},
        # One layer of eight requests' verification behind the 12-token template, FP32 cache.
        {"name": "verify_8x16_template_fp32", "op": "attention", "model": "8b", "cache": "fp32", "requests": 8,
         "prefix": 12, "held_lo": 430, "held_hi": 455, "new_lo": 16, "new_hi": 16, "depth": 6, "window": 0},
        # A sliding-window layer (2,049 rows visible) that the held rows outgrow, FP32 cache.
        {"name": "verify_12x24_window_fp32", "op": "attention", "model": "2b", "cache": "fp32", "requests": 12,
         "prefix": 455, "held_lo": 700, "held_hi": 2300, "new_lo": 24, "new_hi": 24, "depth": 8, "window": 2049},
        # A serving batch behind a long shared instruction, one row past whole pages.
        {"name": "verify_61x32_prefix_4097", "op": "attention", "model": "8b", "cache": "bf16", "requests": 61,
         "prefix": 4097, "held_lo": 100, "held_hi": 1000, "new_lo": 17, "new_hi": 32, "depth": 8, "window": 0},
        # One request alone over a long context with a wide tree: all work split along the keys.
        {"name": "verify_1x64_131072", "op": "attention", "model": "2b", "cache": "bf16", "requests": 1, "prefix": 0,
         "held_lo": 131008, "held_hi": 131008, "new_lo": 64, "new_hi": 64, "depth": 10, "window": 0},
        # The largest model's heads, trees of any size behind a long document: the compute-bound end.
        {"name": "verify_64x64_prefix_8192", "op": "attention", "model": "31b", "cache": "bf16", "requests": 64,
         "prefix": 8192, "held_lo": 1, "held_hi": 2000, "new_lo": 1, "new_hi": 64, "depth": 12, "window": 0},
        # A decode step's QKV projection, every request its own adapter: the adapters stream by.
        {"name": "adapters_8x1_8b_fp32", "op": "adapters", "model": "8b", "projection": "qkv", "type": "fp32",
         "requests": 8, "new_lo": 1, "new_hi": 1, "rank": 16, "adapters": 8, "none": 0},
        # A decode step of a larger batch, larger adapters, the largest model's QKV projection.
        {"name": "adapters_61x1_31b_bf16", "op": "adapters", "model": "31b", "projection": "qkv", "type": "bf16",
         "requests": 61, "new_lo": 1, "new_hi": 1, "rank": 64, "adapters": 61, "none": 0},
        # Ragged prompts over a few adapters, some requests without one.
        {"name": "adapters_16_prompts_8b_fp32", "op": "adapters", "model": "8b", "projection": "o", "type": "fp32",
         "requests": 16, "new_lo": 129, "new_hi": 1023, "rank": 32, "adapters": 4, "none": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "accept", "attention", "attention", "attention", "adapters", "adapters"])
    model = rng.choice(sorted(PROFILES))
    if op == "adapters":
        kind = rng.choice(["decode", "verify", "prompts"])
        projection = rng.choice(["qkv", "o", "gate_up", "down"])
        n_in, n_out = _widths(model, projection)
        requests = _log(rng, 1, {"decode": 128, "verify": 64, "prompts": 16}[kind])
        new = {"decode": 1, "verify": rng.randint(2, 64), "prompts": _log(rng, 65, 1023)}[kind]
        new = max(1, min(new, 70_000_000 // (requests * (n_in + 2 * n_out))))
        adapters = _log(rng, 1, 64)
        rank = 8 * _log(rng, 1, 16)
        while rank > 8 and min(adapters, requests) * rank * (n_in + n_out) > 120_000_000:
            rank -= 8
        return {"op": op, "model": model, "projection": projection, "type": rng.choice(["bf16", "fp32"]),
                "requests": requests, "new_lo": 1 if kind == "decode" else rng.randint(1, new), "new_hi": new, "rank": rank,
                "adapters": adapters, "none": rng.choice([0, 0, rng.randint(2, 5)])}
    new = _log(rng, 1, 256)
    depth = rng.randint(1, 24)
    if op == "tree":
        requests = _log(rng, 1, min(2048, 65536 // new))
        return {"op": op, "requests": requests, "held_lo": 0, "held_hi": _log(rng, 1, 100000), "new_lo": rng.randint(0, new),
                "new_hi": new, "depth": depth, "base": rng.choice([0, 12, _log(rng, 13, 20000)])}
    if op == "accept":
        requests = _log(rng, 1, min(256, 16384 // new))
        cache = rng.choice(["bf16", "fp32"])
        held = _log(rng, 1, 300)
        per_layer = requests * (1 + (held + new) / PAGE) * 2 * PAGE * PROFILES[model][2] * DIM * TYPES[cache].itemsize
        return {"op": op, "model": model, "cache": cache, "layers": max(1, min(rng.randint(1, 32), int(6e8 / per_layer))),
                "requests": requests, "held_lo": rng.randint(0, held), "held_hi": held, "new_lo": rng.randint(1, new),
                "new_hi": new, "depth": depth}
    cache = rng.choice(["bf16", "bf16", "fp32"])
    prefix = rng.choice([0, 12, _log(rng, 13, 16384), _log(rng, 13, 16384)])
    window = rng.choice([0, 0, 2049, _log(rng, 1, 4000)])
    if rng.random() < 0.2:  # one request over a long context
        held = _log(rng, 8192, 131008)
        return {"op": op, "model": rng.choice(["0.8b", "2b"]), "cache": cache, "requests": 1, "prefix": 0, "held_lo": held,
                "held_hi": held, "new_lo": min(new, 64 if cache == "bf16" else 16), "new_hi": min(new, 64 if cache == "bf16" else 16),
                "depth": depth, "window": rng.choice([0, 0, window])}
    requests, held = _log(rng, 1, 64), _log(rng, 1, 4000)
    if cache == "fp32":
        prefix, held, requests = min(prefix, 4096), min(held, 2300), min(requests, 12)
    budget = 3e11 if cache == "bf16" else 1.5e10  # multiply-adds' worth of work, scores and values
    while requests * new * PROFILES[model][1] * (prefix + held) * 2 * DIM > budget:
        if new > 16:
            new = max(16, new // 2)
        elif requests > 1:
            requests = max(1, requests // 2)
        else:
            prefix //= 2
    return {"op": op, "model": model, "cache": cache, "requests": requests, "prefix": prefix, "held_lo": rng.randint(0, held),
            "held_hi": held, "new_lo": rng.randint(1, new), "new_hi": new, "depth": depth, "window": window}


def _spread(lo, hi, count, step):
    """`count` whole numbers from lo to hi, spread evenly but out of order: the same for a case on every seed."""
    return (lo + np.floor((np.arange(count) * step + 0.5) % 1.0 * (hi - lo + 1))).astype(np.int64)


def _lengths(case):
    held = _spread(case.get("held_lo", 0), case.get("held_hi", 0), case["requests"], 0.6180339887498949)
    new = _spread(case["new_lo"], case["new_hi"], case["requests"], 0.7548776662466927)
    if new.sum() == 0:
        new[0] = 1
    return held, new


def _pages(rows):
    return (rows + PAGE - 1) // PAGE


def _words(case):
    return int(_pages(_lengths(case)[1].max() * 2))  # 32 rows to a word


def _widths(model, projection):
    """Input and output width of a projection."""
    hidden, qh, kh, inner = PROFILES[model]
    return {"qkv": (hidden, (qh + 2 * kh) * DIM), "o": (qh * DIM, hidden), "gate_up": (hidden, 2 * inner),
            "down": (inner, hidden)}[projection]


def _adapter_ids(case):
    """Each request's adapter; every `none`-th has none. Requests come ordered by adapter, as a server keeps them."""
    ids = np.sort(_spread(0, case["adapters"] - 1, case["requests"], 0.5698402909980532))
    if case["none"]:
        ids[case["none"] - 1::case["none"]] = -1
    return ids


def work(case):
    held, new = _lengths(case)
    rows, requests = int(new.sum()), case["requests"]
    if case["op"] == "tree":
        return {"bytes": 4 * (2 * requests + 1 + rows * (2 + _words(case))), "flops": rows}
    if case["op"] == "adapters":
        n_in, n_out = _widths(case["model"], case["projection"])
        ids, b, rank = _adapter_ids(case), TYPES[case["type"]].itemsize, case["rank"]
        used, active = len(set(ids[(ids >= 0) & (new > 0)].tolist())), int(new[ids >= 0].sum())
        return {"bytes": used * rank * (n_in + n_out) * 2 + active * n_in * b + 2 * rows * n_out * b + 8 * requests,
                "flops": 2 * active * rank * (n_in + n_out)}
    _, qh, kh, _ = PROFILES[case["model"]]
    b = TYPES[case["cache"]].itemsize
    if case["op"] == "accept":
        # On average half of the accepted rows lie off the first chain and are moved: about a fifth of the depth each.
        moved = int(np.minimum(new - 1, case["depth"]).sum()) // 5
        return {"bytes": 4 * (3 * rows + 5 * requests + 2 * rows) + case["layers"] * moved * 4 * kh * DIM * b, "flops": rows}
    prefix, window = case["prefix"], case["window"]
    pairs = seen = 0
    first = prefix  # the first prefix row that any query sees
    for h, n in zip(held.tolist(), new.tolist()):
        if not n:
            continue
        total = prefix + h + 1  # of every row at least: the prefix, the held rows, itself
        pairs += n * (min(total, window) if window else total)
        skipped = max(0, total - window) if window else 0
        seen += n + h - max(0, min(h, skipped - prefix))
        first = min(first, skipped)
    keys = seen + prefix - first
    return {"bytes": 2 * keys * kh * DIM * b + 2 * rows * qh * DIM * b + 4 * (3 * requests + keys // PAGE + rows * _words(case)),
            "flops": 4 * DIM * qh * pairs}


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _int32(values):
    return torch.as_tensor(np.ascontiguousarray(values, dtype=np.int32)).cuda()


def _tables(counts, order, columns):
    """Page tables: request r's counts[r] pages, taken from `order` one request after another; -1 where no page is."""
    at = np.arange(columns)[None, :]
    first = (np.cumsum(counts) - counts)[:, None]
    index = torch.as_tensor(np.where(at < counts[:, None], first + at, -1)).cuda()
    return torch.where(index >= 0, order[index.clamp(min=0)], -1).to(torch.int32).contiguous()


def _trees(case, seed):
    """(parents, depths) of every request's rows: the likeliest continuation first, a chain of up to `depth` rows
    behind row 0 (the last token, already certain), then alternatives hung below any earlier row."""
    rng = np.random.default_rng(int(seed))
    parents, depths = [], []
    for n in _lengths(case)[1].tolist():
        chain = min(n - 1, case["depth"])
        parent, depth = list(range(-1, min(n, chain + 1) - 1)), list(range(min(n, chain + 1)))
        open_rows = [i for i, d in enumerate(depth) if d < chain]  # rows that can have children
        for i in range(len(parent), n):
            at = open_rows[int(rng.integers(len(open_rows)))]
            parent.append(at)
            depth.append(depth[at] + 1)
            if depth[i] < chain:
                open_rows.append(i)
        parents.append(np.array(parent, dtype=np.int64))
        depths.append(np.array(depth, dtype=np.int64))
    return parents, depths


def _masks(parents, words):
    """Rows' bits and their ancestors', 32 to a word."""
    out = []
    for parent in parents:
        bits = np.zeros((len(parent), words * 32), dtype=bool)
        for i, p in enumerate(parent.tolist()):
            if p >= 0:
                bits[i] = bits[p]
            bits[i, i] = True
        out.append(np.packbits(bits, axis=1, bitorder="little").view("<i4").reshape(len(parent), words))
    return np.concatenate(out).astype(np.int32)


def _choices(parents, depths, case, seed):
    """Drafted tokens, and the token the model chooses after each: a path of drafts is confirmed, along the first
    chain for a while, then perhaps through alternatives."""
    rng = np.random.default_rng(int(seed) + 1)
    tokens, chosen = [], []
    for parent, depth in zip(parents, depths):
        n = len(parent)
        token, choice = rng.integers(0, VOCABULARY, n), rng.integers(0, VOCABULARY, n)
        if n:
            chain = min(n - 1, case["depth"])
            at = int(rng.integers(0, chain + 1))
            choice[:at] = token[1:at + 1]
            while True:
                below = [i for i in np.flatnonzero(parent == at).tolist() if i > chain]
                if not below or rng.random() < 0.25:
                    break
                child = below[int(rng.integers(len(below)))]
                choice[at] = token[child]
                at = child
        tokens.append(token)
        chosen.append(choice)
    return np.concatenate(tokens), np.concatenate(chosen)


def prepare(case, seed):
    g = _generator(seed)
    held, new = _lengths(case)
    rows, starts = int(new.sum()), np.concatenate([[0], np.cumsum(new)])
    if case["op"] == "adapters":
        n_in, n_out = _widths(case["model"], case["projection"])
        kind, rank, count = TYPES[case["type"]], case["rank"], case["adapters"]
        ids = _adapter_ids(case)

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, generator=g, device="cuda").mul_(scale)

        return {"case": case, "x": normal(rows, n_in).to(kind), "base": normal(rows, n_out).to(kind),
                "a": normal(count, rank, n_in, scale=n_in ** -0.5).to(torch.bfloat16),
                "b": normal(count, n_out, rank, scale=0.3).to(torch.bfloat16),
                "scales": torch.rand(count, generator=g, device="cuda").add_(0.5), "ids": _int32(ids), "starts": _int32(starts),
                "host_ids": ids.tolist(), "host_starts": starts.tolist()}
    parents, depths = _trees(case, seed)
    s = {"case": case, "parents": _int32(np.concatenate(parents)), "starts": _int32(starts), "lengths": _int32(held + new),
         "most_new": int(new.max())}
    if case["op"] == "tree":
        return s
    _, qh, kh, _ = PROFILES[case["model"]]
    cache = TYPES[case["cache"]]
    counts = _pages(held + new)
    own_pages, prefix = int(counts.sum()), case.get("prefix", 0)
    prefix_pages = _pages(prefix)
    pages = own_pages + prefix_pages + 2
    order = torch.randperm(pages, generator=g, device="cuda")
    s["tables"] = _tables(counts, order[prefix_pages:], int(counts.max()) + 1)
    if case["op"] == "accept":
        tokens, chosen = _choices(parents, depths, case, seed)
        spent = int((counts - _pages(held)).sum())  # pages that the step's plan took from the free list
        pools = [torch.randn(pages, 2, PAGE, kh, DIM, generator=g, device="cuda").to(cache) for _ in range(case["layers"])]
        free = torch.randperm(spent + 50, generator=g, device="cuda").to(torch.int32)
        return {**s, "tokens": _int32(tokens), "chosen": _int32(chosen), "pools": pools, "free": free,
                "summary": _int32([0, rows, spent, (held + new).max()])}
    pool = torch.randn(pages, 2, PAGE, kh, DIM, generator=g, device="cuda", dtype=torch.float32)
    # Heads come normalised and rotated: unit-size entries times the norm's weight, scores a few units wide.
    q = torch.randn(rows, qh, DIM, generator=g, device="cuda").mul_(1.5).to(cache)
    return {**s, "q": q, "pool": pool.to(cache), "masks": torch.as_tensor(_masks(parents, _words(case))).cuda(),
            "prefix_pages": order[:prefix_pages].to(torch.int32).contiguous(), "prefix": prefix, "window": case["window"],
            "most_rows": int((held + new).max())}


# ---- plain forms -----------------------------------------------------------

def _owners(s, rows):
    """Each row's request, and its place among the request's rows."""
    starts = s["starts"].long()
    at = torch.arange(rows, device=starts.device)
    owner = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    return owner, at - starts[owner]


def _tree_plain(s):
    parents, starts, lengths = s["parents"].long(), s["starts"].long(), s["lengths"].long()
    rows, words = parents.shape[0], _words(s["case"])
    owner, index = _owners(s, rows)
    held = lengths - (starts[1:] - starts[:-1])
    seen = torch.zeros(rows, words * 32, dtype=torch.bool, device=parents.device)
    at, depth = index.clone(), torch.zeros_like(index)
    for _ in range(s["case"]["depth"] + 1):  # one generation up at a time
        real = at >= 0
        seen[real.nonzero()[:, 0], at[real]] = True
        at = torch.where(real, parents[(starts[owner] + at.clamp(min=0))], -1)
        depth += at >= 0
    bits = torch.arange(32, device=parents.device)
    masks = (seen.view(rows, words, 32).long() << bits).sum(-1)
    masks = torch.where(masks >= 2 ** 31, masks - 2 ** 32, masks)
    return {"positions": (s["case"]["base"] + held[owner] + depth).int(), "masks": masks.int()}


def _accept_plain(s):
    parents, tokens, chosen = s["parents"].long(), s["tokens"].long(), s["chosen"].long()
    starts, lengths, tables = s["starts"].long(), s["lengths"].long(), s["tables"].long()
    rows, requests, most = parents.shape[0], lengths.shape[0], s["most_new"]
    owner, index = _owners(s, rows)
    added = starts[1:] - starts[:-1]

    def padded(values, fill):
        out = torch.full((requests, most), fill, dtype=torch.long, device=values.device)
        out[owner, index] = values
        return out

    parent, token, choice = padded(parents, -2), padded(tokens, -1), padded(chosen, -1)
    current, alive, counts = torch.zeros_like(added), added > 0, torch.zeros_like(added)
    path, taken = torch.full_like(parent, -1), torch.full_like(parent, -1)
    last = torch.full_like(added, -1)
    every = torch.arange(requests, device=parents.device)
    for step in range(min(most, s["case"]["depth"] + 1)):
        pick = choice[every, current]
        path[:, step] = torch.where(alive, current, -1)
        taken[:, step] = torch.where(alive, pick, -1)
        last = torch.where(alive, pick, last)
        counts += alive
        match = (parent == current[:, None]) & (token == pick[:, None])
        alive = alive & match.any(1)
        current = torch.where(alive, match.int().argmax(1), current)
    held = lengths - added
    now = held + counts
    # accepted rows to their places, in every layer
    k = torch.arange(most, device=parents.device)
    request, step = (k[None] < counts[:, None]).nonzero(as_tuple=True)
    source, target = held[request] + path[request, step], held[request] + step
    for pool in s["pools"]:
        kept = pool[tables[request, source // PAGE], :, source % PAGE]
        pool[tables[request, target // PAGE], :, target % PAGE] = kept
    # pages that no row reaches any more
    column = torch.arange(tables.shape[1], device=parents.device)[None]
    back = (column >= _pages(now)[:, None]) & (column < _pages(lengths)[:, None])
    ids = tables[back]
    free, head = s["free"], s["summary"][2].long()
    free[head - ids.shape[0] + torch.arange(ids.shape[0], device=parents.device)] = ids.int()
    summary = torch.stack([torch.zeros_like(head), counts.sum(), head - ids.shape[0], now.max()])
    return {"counts": counts.int(), "lengths": now.int(), "path": path[owner, index].int(), "tokens": taken[owner, index].int(),
            "last": last.int(), "summary": summary.int(), "free": free, "pools": s["pools"]}


def _attention_plain(s):
    q, pool, lengths, starts = s["q"].float(), s["pool"], s["lengths"].long(), s["starts"].long()
    rows, qh, _ = q.shape
    kh = pool.shape[3]
    group, requests, prefix, window = qh // kh, lengths.shape[0], s["prefix"], s["window"]
    most_new, most = s["most_new"], s["most_rows"]
    q = q.view(rows, kh, group, DIM) * DIM ** -0.5
    owner, index = _owners(s, rows)
    held = (lengths - (starts[1:] - starts[:-1]))[owner]
    bits = ((s["masks"].long()[:, :, None] >> torch.arange(32, device=q.device)) & 1).flatten(1).bool()
    depth = bits.sum(1) - 1
    position = held + depth  # behind the prefix

    # scores over the request's own rows, requests padded to the longest
    own_pages = pool[s["tables"][:, : _pages(most)].long().clamp(min=0)]
    k = own_pages[:, :, 0].float().reshape(requests, -1, kh, DIM)
    v = own_pages[:, :, 1].float().reshape(requests, -1, kh, DIM)
    padded = q.new_zeros(requests, most_new, kh, group, DIM)
    padded[owner, index] = q
    scores = torch.matmul(padded.permute(0, 2, 1, 3, 4).reshape(requests, kh, -1, DIM), k.permute(0, 2, 3, 1))
    scores = scores.view(requests, kh, most_new, group, -1).permute(0, 2, 1, 3, 4)[owner, index]
    keys = torch.arange(scores.shape[-1], device=q.device)[None]
    draft = (keys - held[:, None]).clamp(min=0, max=bits.shape[1] - 1)
    seen = torch.where(keys < held[:, None], True, bits.gather(1, draft) & (keys - held[:, None] < bits.shape[1]))
    if window:  # an ancestor stands at the position of its depth
        depth_of = torch.zeros(requests, bits.shape[1], dtype=torch.long, device=q.device)
        depth_of[owner, index] = depth
        place = torch.where(keys < held[:, None], keys, held[:, None] + depth_of[owner].gather(1, draft))
        seen &= place > position[:, None] - window
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)

    # and over the prefix, every query of the batch at once
    if prefix:
        shared = pool[s["prefix_pages"].long()]
        pk = shared[:, 0].float().reshape(-1, kh, DIM)[:prefix]
        pv = shared[:, 1].float().reshape(-1, kh, DIM)[:prefix]
        flat = q.permute(1, 0, 2, 3).reshape(kh, rows * group, DIM)
        before = torch.matmul(flat, pk.permute(1, 2, 0)).view(kh, rows, group, prefix)
        if window:
            hidden = torch.arange(prefix, device=q.device)[None] <= (position + prefix)[:, None] - window
            before = before.masked_fill(hidden[None, :, None], -math.inf)
        m = torch.maximum(m, before.amax(-1, keepdim=True).permute(1, 0, 2, 3))
    p = torch.exp(scores - m)
    total = p.sum(-1, keepdim=True)
    spread = p.new_zeros(requests, most_new, kh, group, p.shape[-1])
    spread[owner, index] = p
    out = torch.matmul(spread.permute(0, 2, 1, 3, 4).reshape(requests, kh, most_new * group, -1), v.transpose(1, 2))
    out = out.view(requests, kh, most_new, group, DIM).permute(0, 2, 1, 3, 4)[owner, index]
    if prefix:
        p = torch.exp(before - m.permute(1, 0, 2, 3))
        total = total + p.sum(-1, keepdim=True).permute(1, 0, 2, 3)
        out = out + torch.matmul(p.view(kh, rows * group, prefix), pv.transpose(0, 1)).view(kh, rows, group, DIM).permute(1, 0, 2, 3)
    return (out / total).reshape(rows, qh, DIM).to(s["pool"].dtype)


def _adapters_plain(s):
    out = s["base"].float()
    if out is s["base"]:
        out = out.clone()
    runs = []  # consecutive requests of one adapter: [adapter, first row, end]
    for r, a in enumerate(s["host_ids"]):
        lo, hi = s["host_starts"][r], s["host_starts"][r + 1]
        if runs and runs[-1][0] == a:
            runs[-1][2] = hi
        else:
            runs.append([a, lo, hi])
    for a, lo, hi in runs:
        if a >= 0 and hi > lo:
            inner = torch.matmul(s["x"][lo:hi].float(), s["a"][a].float().t())
            out[lo:hi] += s["scales"][a] * torch.matmul(inner, s["b"][a].float().t())
    return out.to(s["base"].dtype)


def run(state):
    op, s = state["case"]["op"], state
    if not own:
        return {"tree": _tree_plain, "accept": _accept_plain, "attention": _attention_plain, "adapters": _adapters_plain}[op](s)
    backend = _framework()
    if op == "tree":
        t = backend.paged_tree(s["parents"], s["starts"], s["lengths"], s["most_new"], base=s["case"]["base"])
        return {"positions": t.positions, "masks": t.masks}
    if op == "accept":
        a = backend.paged_accept(s["parents"], s["tokens"], s["chosen"], s["starts"], s["lengths"], s["tables"], s["free"],
                                 s["summary"])
        backend.paged_keep(s["pools"], a.path, s["starts"], s["lengths"], s["tables"])
        return {"counts": a.counts, "lengths": a.lengths, "path": a.path, "tokens": a.tokens, "last": a.last,
                "summary": a.summary, "free": s["free"], "pools": s["pools"]}
    if op == "attention":
        return backend.paged_attention(s["q"], s["pool"], s["starts"], s["lengths"], s["tables"],
                                       prefix_pages=s["prefix_pages"], prefix_rows=s["prefix"], window=s["window"],
                                       most_new=s["most_new"], masks=s["masks"])
    return backend.paged_adapters(s["x"], s["base"], s["a"], s["b"], s["ids"], s["starts"], scales=s["scales"])


# ---- the definitions in 64 bits ----------------------------------------------

def _exact_tree(s):
    parents, starts, lengths = s["parents"].tolist(), s["starts"].tolist(), s["lengths"].tolist()
    positions, masks = [], np.zeros((len(parents), _words(s["case"])), dtype=np.uint32)
    for r, length in enumerate(lengths):
        lo, hi = starts[r], starts[r + 1]
        for row in range(lo, hi):
            i, generations = row - lo, 0
            while i >= 0:
                masks[row, i // 32] |= np.uint32(1 << (i % 32))
                i = parents[lo + i]
                generations += 1
            positions.append(s["case"]["base"] + length - (hi - lo) + generations - 1)
    return {"positions": np.array(positions, np.int32), "masks": masks.view(np.int32)}


def _exact_accept(s):
    parents, tokens, chosen = s["parents"].tolist(), s["tokens"].tolist(), s["chosen"].tolist()
    starts, lengths, tables = s["starts"].tolist(), s["lengths"].tolist(), s["tables"].tolist()
    free, head = s["free"].tolist(), s["summary"].tolist()[2]
    path, taken = [-1] * len(parents), [-1] * len(parents)
    counts, last, back = [], [], []
    flat = [pool.permute(0, 2, 1, 3, 4).reshape(-1, 2, *pool.shape[3:]).clone() for pool in s["pools"]]
    sources, targets = [], []
    for r, length in enumerate(lengths):
        lo, hi = starts[r], starts[r + 1]
        held, at, steps = length - (hi - lo), 0 if hi > lo else -1, 0
        last.append(-1)
        while at >= 0:
            path[lo + steps], taken[lo + steps] = at, chosen[lo + at]
            last[r] = chosen[lo + at]
            if at != steps:
                sources.append(tables[r][(held + at) // PAGE] * PAGE + (held + at) % PAGE)
                targets.append(tables[r][(held + steps) // PAGE] * PAGE + (held + steps) % PAGE)
            steps += 1
            children = [i for i in range(hi - lo) if parents[lo + i] == at and tokens[lo + i] == chosen[lo + at]]
            at = children[0] if children else -1
        counts.append(steps)
        back += tables[r][_pages(held + steps):_pages(length)]
    free[head - len(back):head] = back
    now = [length - (starts[r + 1] - starts[r]) + counts[r] for r, length in enumerate(lengths)]
    pools = []
    for pool, f in zip(s["pools"], flat):
        f[targets] = f[sources]
        pools.append(f.view(pool.shape[0], PAGE, 2, *pool.shape[3:]).permute(0, 2, 1, 3, 4).contiguous())
    return {"counts": np.array(counts, np.int32), "lengths": np.array(now, np.int32), "path": np.array(path, np.int32),
            "tokens": np.array(taken, np.int32), "last": np.array(last, np.int32),
            "summary": np.array([0, sum(counts), head - len(back), max(now)], np.int32), "free": np.array(free, np.int32),
            "pools": pools}


def _exact_attention(s):
    pool, q = s["pool"], s["q"].double()
    kh, qh = pool.shape[3], q.shape[1]
    out = torch.zeros_like(q)

    def rows_of(pages, count, kind):
        return pool[pages.long(), kind].reshape(-1, kh, DIM)[:count].double()

    shared = [rows_of(s["prefix_pages"], s["prefix"], kind) for kind in (0, 1)]
    starts, lengths, parents = s["starts"].tolist(), s["lengths"].tolist(), s["parents"].tolist()
    for r, length in enumerate(lengths):
        pages = s["tables"][r, : _pages(length)]
        k, v = (torch.cat([shared[kind], rows_of(pages, length, kind)]) for kind in (0, 1))
        lo, n = starts[r], starts[r + 1] - starts[r]
        before = s["prefix"] + length - n
        seen = torch.zeros(n, before + n, dtype=torch.bool)
        for i in range(n):
            line = [i]  # itself and its ancestors, the nearest first
            while parents[lo + line[-1]] >= 0:
                line.append(parents[lo + line[-1]])
            line = [before + j for j in reversed(line)]
            window = s["window"] or before + n
            seen[i, max(0, before + len(line) - window):before] = True
            seen[i, line[-window:]] = True
        seen = seen.to(q.device)
        for first in range(0, n, 64):
            part = slice(lo + first, lo + min(n, first + 64))
            for h in range(kh):
                heads = slice(h * (qh // kh), (h + 1) * (qh // kh))
                score = torch.einsum("ngd,kd->ngk", q[part, heads], k[:, h]) / math.sqrt(DIM)
                weight = torch.softmax(score.masked_fill(~seen[first:first + 64, None], -math.inf), -1)
                out[part, heads] = torch.einsum("ngk,kd->ngd", weight, v[:, h])
    return out


def _exact_adapters(s):
    out = s["base"].double()
    for r, a in enumerate(s["ids"].tolist()):
        rows = slice(*s["starts"][r:r + 2].tolist())
        if a >= 0:
            inner = torch.einsum("nk,rk->nr", s["x"][rows].double(), s["a"][a].double())
            out[rows] += torch.einsum("nr,or->no", inner * s["scales"][a].double(), s["b"][a].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "attention": _exact_attention, "adapters": _exact_adapters}[case["op"]](s)
