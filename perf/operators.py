"""The paged-batch operators: what is measured of them, and their plain forms.

Three operators carry a step of a batch of requests whose keys and values live in pages of 64 rows and
which share a prompt prefix:

  plan       page tables and slot maps from the requests' lengths: which page each new row goes to, new
             pages taken from a free list, all on the GPU;
  store      between the QKV projection and attention: RMSNorm and RoPE of the query and key heads, keys
             and values into their slots, queries out;
  attention  every query over the prefix that all requests share (read once for all of them) and over its
             own request's rows, causal, with an optional sliding window.

Pages are laid out [2][64][kv heads][128]: 64 key rows, then 64 value rows. Heads have 128 dimensions, as in
every model profile of this repository (16/1, 24/4, 32/4 and 64/8 query/KV heads).
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
EPS = 1e-6
PROFILES = {"0.8b": (16, 1), "2b": (24, 4), "8b": (32, 4), "31b": (64, 8)}  # query heads, KV heads
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
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
        # A decode step of the eight requests that one GPU serves at a time: pure latency.
        {"name": "plan_decode_8", "op": "plan", "requests": 8, "held_lo": 430, "held_hi": 470, "new_lo": 1, "new_hi": 1,
         "spare_rows": 0},
        # A decode step of a large server: every request one row, lengths from nothing to 4,000.
        {"name": "plan_decode_4096", "op": "plan", "requests": 4096, "held_lo": 0, "held_hi": 4000, "new_lo": 1,
         "new_hi": 1, "spare_rows": 0},
        # Prompts arriving together, some requests idle, a row count fixed for graph capture with rows to spare.
        {"name": "plan_prompts_64", "op": "plan", "requests": 64, "held_lo": 0, "held_hi": 700, "new_lo": 0,
         "new_hi": 2047, "spare_rows": 100},
        # One layer of the eight-request decode step, FP32 cache as the token loop keeps it.
        {"name": "store_decode_8b_fp32", "op": "store", "model": "8b", "source": "fp32", "cache": "fp32", "rows": 8,
         "base": 12},
        # One layer of a prompt batch into a BF16 cache; an odd row count.
        {"name": "store_prompts_8b_bf16", "op": "store", "model": "8b", "source": "fp32", "cache": "bf16",
         "rows": 8191, "base": 455},
        # The eight-request decode step of a translation prompt behind the 12-token template, FP32 cache.
        {"name": "decode_8x450_fp32", "op": "attention", "model": "8b", "cache": "fp32", "requests": 8, "prefix": 12,
         "held_lo": 430, "held_hi": 455, "new_lo": 1, "new_hi": 1, "window": 0},
        # A serving batch behind a long shared instruction, one row past whole pages.
        {"name": "decode_61_prefix_4097", "op": "attention", "model": "8b", "cache": "bf16", "requests": 61,
         "prefix": 4097, "held_lo": 100, "held_hi": 1000, "new_lo": 1, "new_hi": 1, "window": 0},
        # A large batch behind a very long shared document, the largest model's heads.
        {"name": "decode_256_prefix_16384", "op": "attention", "model": "31b", "cache": "bf16", "requests": 256,
         "prefix": 16384, "held_lo": 1, "held_hi": 1000, "new_lo": 1, "new_hi": 1, "window": 0},
        # One request alone over a long context: nothing shared, all work split along the keys.
        {"name": "decode_1x131072", "op": "attention", "model": "2b", "cache": "bf16", "requests": 1, "prefix": 0,
         "held_lo": 131071, "held_hi": 131071, "new_lo": 1, "new_hi": 1, "window": 0},
        # Ragged prompts behind a shared instruction: the compute-bound end.
        {"name": "prompts_16_prefix_2048", "op": "attention", "model": "8b", "cache": "bf16", "requests": 16,
         "prefix": 2048, "held_lo": 0, "held_hi": 300, "new_lo": 129, "new_hi": 1023, "window": 0},
        # Verification blocks of 16 draft tokens in a sliding-window layer (2,049 rows visible), FP32 cache.
        {"name": "verify_12x16_window_fp32", "op": "attention", "model": "2b", "cache": "fp32", "requests": 12,
         "prefix": 455, "held_lo": 700, "held_hi": 2300, "new_lo": 16, "new_hi": 16, "window": 2049},
        # Translation prompts behind the template, FP32 cache.
        {"name": "prompts_6_template_fp32", "op": "attention", "model": "2b", "cache": "fp32", "requests": 6,
         "prefix": 12, "held_lo": 0, "held_hi": 0, "new_lo": 300, "new_hi": 455, "window": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "attention", "attention", "attention"])
    if op == "plan":
        requests = _log(rng, 1, 4096)
        most = 1 if rng.random() < 0.5 else max(1, min(2048, 65536 // requests))
        hi = _log(rng, 1, 4000)
        return {"op": op, "requests": requests, "held_lo": rng.randint(0, hi), "held_hi": hi,
                "new_lo": 1 if most == 1 else rng.randint(0, 2), "new_hi": max(2, _log(rng, 2, max(2, most))) if most > 1 else 1,
                "spare_rows": rng.choice([0, 0, rng.randint(1, 300)])}
    model = rng.choice(sorted(PROFILES))
    if op == "store":
        rows = _log(rng, 1, 8191)
        return {"op": op, "model": model if rows <= 4096 else "8b", "source": rng.choice(["fp32", "bf16"]),
                "cache": rng.choice(["fp32", "bf16"]), "rows": rows, "base": _log(rng, 1, 20000)}
    cache = rng.choice(["bf16", "bf16", "fp32"])
    kind = rng.choice(["decode", "decode", "verify", "prompts", "long"])
    prefix = rng.choice([0, 12, _log(rng, 13, 16384), _log(rng, 13, 16384)])
    window = rng.choice([0, 0, 2049, _log(rng, 1, 4000)])
    if kind == "long":
        held = _log(rng, 8192, 131071)
        return {"op": op, "model": rng.choice(["0.8b", "2b", "8b"]), "cache": cache, "requests": 1, "prefix": prefix,
                "held_lo": held, "held_hi": held, "new_lo": 1, "new_hi": 1, "window": rng.choice([0, 0, window])}
    if kind == "prompts":
        requests, new = _log(rng, 1, 16), _log(rng, 17, 1023)
        held, prefix = rng.choice([0, _log(rng, 1, 300)]), min(prefix, 2048)
        if cache == "fp32":
            model = rng.choice(["0.8b", "2b"])
            requests, prefix = min(requests, 6), min(prefix, 1000)
        return {"op": op, "model": model if model != "31b" or requests <= 8 else "8b", "cache": cache, "requests": requests,
                "prefix": prefix, "held_lo": 0, "held_hi": held, "new_lo": rng.randint(1, new), "new_hi": new,
                "window": window}
    requests = _log(rng, 1, 256 if kind == "decode" else 32)
    held = _log(rng, 1, min(8000, max(1, (1000 if cache == "bf16" else 500) * 256 // requests)))
    new = 1 if kind == "decode" else rng.randint(2, 16)
    if kind == "verify":
        held, prefix = min(held, 4000), min(prefix, 8192)
    if cache == "fp32":
        prefix = min(prefix, 4096)
    return {"op": op, "model": model, "cache": cache, "requests": requests, "prefix": prefix,
            "held_lo": rng.randint(0, held), "held_hi": held, "new_lo": 1 if kind == "decode" else rng.randint(1, new),
            "new_hi": new, "window": window}


def _spread(lo, hi, count, step):
    """`count` whole numbers from lo to hi, spread evenly but out of order: the same for a case on every seed."""
    return (lo + np.floor((np.arange(count) * step + 0.5) % 1.0 * (hi - lo + 1))).astype(np.int64)


def _lengths(case):
    held = _spread(case["held_lo"], case["held_hi"], case["requests"], 0.6180339887498949)
    new = _spread(case["new_lo"], case["new_hi"], case["requests"], 0.7548776662466927)
    if new.sum() == 0:
        new[0] = 1
    return held, new


def _pages(rows):
    return (rows + PAGE - 1) // PAGE


def work(case):
    if case["op"] == "plan":
        held, new = _lengths(case)
        r, rows = case["requests"], int(new.sum()) + case["spare_rows"]
        taken = int((_pages(held + new) - _pages(held)).sum())
        partial = int(((new > 0) & (held % PAGE > 0)).sum())
        # lengths in and out, starts, a slot and a position per row, page ids: taken ones read and written, started ones read
        return {"bytes": 4 * (3 * r + r + 1 + 2 * rows + 2 * taken + partial + 4), "flops": 4 * rows}
    qh, kh = PROFILES[case["model"]]
    if case["op"] == "store":
        rows, a = case["rows"], TYPES[case["source"]].itemsize
        b = TYPES[case["cache"]].itemsize
        width = (qh + 2 * kh) * DIM
        return {"bytes": rows * (width * (a + b) + DIM * 4 + 8) + 4 * DIM, "flops": rows * (qh + kh) * DIM * 9}
    held, new = _lengths(case)
    b = TYPES[case["cache"]].itemsize
    prefix, window = case["prefix"], case["window"]
    rows = int(new.sum())
    pairs = seen = 0
    first = prefix  # the first prefix row that any query sees
    for h, n in zip(held.tolist(), new.tolist()):
        at = prefix + h + np.arange(n, dtype=np.int64)
        low = np.maximum(0, at - window + 1) if window else np.zeros(n, np.int64)
        pairs += int((at - low + 1).sum())
        if n:
            seen += h + n - max(0, int(low[0]) - prefix)
            first = min(first, int(low[0]))
    keys = seen + prefix - first
    return {"bytes": 2 * keys * kh * DIM * b + 2 * rows * qh * DIM * b + 4 * (3 * case["requests"] + keys // PAGE),
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


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "plan":
        held, new = _lengths(case)
        have, want = _pages(held), _pages(held + new)
        total, need = int(have.sum()), int((want - have).sum())
        order = torch.randperm(total + need + 64, generator=g, device="cuda")
        return {"case": case, "held": _int32(held), "added": _int32(new),
                "tables": _tables(have, order, int(want.max()) + 1), "free": order[total:].to(torch.int32).contiguous(),
                "rows": int(new.sum()) + case["spare_rows"], "base": 12}
    qh, kh = PROFILES[case["model"]]
    cache = TYPES[case["cache"]]
    if case["op"] == "store":
        rows = case["rows"]
        qkv = torch.randn(rows, (qh + 2 * kh) * DIM, generator=g, device="cuda").mul_(1.7).to(TYPES[case["source"]])
        # Each request adds up to 200 rows behind the shared prefix, its pages anywhere in the pool.
        pages = _pages(rows) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(rows, device="cuda") + 5
        slots = (order[at // PAGE] * PAGE + at % PAGE).to(torch.int32)
        positions = (case["base"] + torch.arange(rows, device="cuda") % 200).to(torch.int32)
        half = DIM // 2
        angle = torch.arange(case["base"] + 200, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        table = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        norms = [torch.rand(DIM, generator=g, device="cuda").sub_(0.5).to(torch.bfloat16) for _ in range(2)]
        return {"case": case, "qkv": qkv, "slots": slots, "positions": positions, "table": table, "q_norm": norms[0],
                "k_norm": norms[1], "pool": torch.zeros(pages, 2, PAGE, kh, DIM, dtype=cache, device="cuda")}
    held, new = _lengths(case)
    lengths, prefix = held + new, case["prefix"]
    counts = _pages(lengths)
    own_pages, prefix_pages = int(counts.sum()), _pages(prefix)
    order = torch.randperm(own_pages + prefix_pages + 2, generator=g, device="cuda")
    pool = torch.randn(own_pages + prefix_pages + 2, 2, PAGE, kh, DIM, generator=g, device="cuda", dtype=torch.float32)
    # Heads come normalised and rotated: unit-size entries times the norm's weight, scores a few units wide.
    q = torch.randn(int(new.sum()), qh, DIM, generator=g, device="cuda").mul_(1.5).to(cache)
    return {"case": case, "q": q, "pool": pool.to(cache), "starts": _int32(np.concatenate([[0], np.cumsum(new)])),
            "lengths": _int32(lengths), "tables": _tables(counts, order[prefix_pages:], int(counts.max()) + 1),
            "prefix_pages": order[:prefix_pages].to(torch.int32).contiguous(), "prefix": prefix, "window": case["window"],
            "most_new": int(new.max()), "most_rows": int(lengths.max())}


# ---- plain forms -----------------------------------------------------------

def _plan_plain(s):
    held, added, tables, free, rows = s["held"].long(), s["added"].long(), s["tables"], s["free"].long(), s["rows"]
    lengths = held + added
    starts = torch.cat([held.new_zeros(1), added.cumsum(0)])
    have, want = (held + PAGE - 1) // PAGE, (lengths + PAGE - 1) // PAGE
    taken = want - have
    first = taken.cumsum(0) - taken
    at = torch.arange(rows, device=held.device)
    real = at < starts[-1]
    at = torch.minimum(at, starts[-1] - 1)
    owner = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    row = held[owner] + at - starts[owner]
    page = row // PAGE
    new = page >= have[owner]
    ids = torch.where(new, free[torch.where(new, first[owner] + page - have[owner], 0)], tables[owner, page].long())
    tables[owner, page] = ids.to(torch.int32)
    slots = torch.where(real, ids * PAGE + row % PAGE, -1)
    positions = torch.where(real, row + s["base"], 0)
    status = (taken.sum() > free.numel()).long() + 2 * (want.max() > tables.shape[1]).long() + 4 * (starts[-1] > rows).long()
    summary = torch.stack([status, starts[-1], taken.sum(), lengths.max()])
    return {"lengths": lengths.int(), "starts": starts.int(), "slots": slots.int(), "positions": positions.int(),
            "summary": summary.int(), "tables": tables}


def _norm_rotate(x, weight, cos, sin):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (weight.float() + 1.0)
    a, b = x[..., : DIM // 2], x[..., DIM // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _store_plain(s):
    pool, slots = s["pool"], s["slots"].long()
    kh = pool.shape[3]
    x = s["qkv"].float().view(s["qkv"].shape[0], -1, DIM)
    qh = x.shape[1] - 2 * kh
    at = s["table"][s["positions"].long()]
    cos, sin = at[:, None, : DIM // 2], at[:, None, DIM // 2:]
    q = _norm_rotate(x[:, :qh], s["q_norm"], cos, sin)
    k = _norm_rotate(x[:, qh:qh + kh], s["k_norm"], cos, sin)
    pool[slots // PAGE, 0, slots % PAGE] = k.to(pool.dtype)
    pool[slots // PAGE, 1, slots % PAGE] = x[:, qh + kh:].to(pool.dtype)
    return {"q": q.to(pool.dtype), "pool": pool}


def _attention_plain(s):
    q, pool, lengths, starts = s["q"].float(), s["pool"], s["lengths"].long(), s["starts"].long()
    rows, qh, _ = q.shape
    kh = pool.shape[3]
    group, requests, prefix, window = qh // kh, lengths.shape[0], s["prefix"], s["window"]
    most_new, most = s["most_new"], s["most_rows"]
    q = q.view(rows, kh, group, DIM) * DIM ** -0.5
    at = torch.arange(rows, device=q.device)
    owner = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    index = at - starts[owner]
    row = lengths[owner] - (starts[owner + 1] - starts[owner]) + index  # the query's place among its request's own rows

    # scores over the request's own rows, requests padded to the longest
    own_pages = pool[s["tables"][:, : _pages(most)].long().clamp(min=0)]
    k = own_pages[:, :, 0].float().reshape(requests, -1, kh, DIM)
    v = own_pages[:, :, 1].float().reshape(requests, -1, kh, DIM)
    padded = q.new_zeros(requests, most_new, kh, group, DIM)
    padded[owner, index] = q
    scores = torch.matmul(padded.permute(0, 2, 1, 3, 4).reshape(requests, kh, -1, DIM), k.permute(0, 2, 3, 1))
    scores = scores.view(requests, kh, most_new, group, -1).permute(0, 2, 1, 3, 4)[owner, index]
    keys = torch.arange(scores.shape[-1], device=q.device)
    seen = keys[None] <= row[:, None]
    if window:
        seen &= keys[None] > row[:, None] - window
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
            hidden = torch.arange(prefix, device=q.device)[None] <= (row + prefix)[:, None] - window
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


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plan_plain, "store": _store_plain, "attention": _attention_plain}[op](state)
    backend, s = _framework(), state
    if op == "plan":
        p = backend.paged_plan(s["held"], s["added"], s["tables"], s["free"], s["rows"], base=s["base"])
        return {"lengths": p.lengths, "starts": p.starts, "slots": p.slots, "positions": p.positions, "summary": p.summary,
                "tables": s["tables"]}
    if op == "store":
        q = backend.paged_store(s["qkv"], s["pool"], s["slots"], s["positions"], s["q_norm"], s["k_norm"], s["table"])
        return {"q": q, "pool": s["pool"]}
    return backend.paged_attention(s["q"], s["pool"], s["starts"], s["lengths"], s["tables"],
                                   prefix_pages=s["prefix_pages"], prefix_rows=s["prefix"], window=s["window"])


# ---- the definitions in 64 bits ----------------------------------------------

def _exact_plan(s):
    held, added = s["held"].cpu().numpy(), s["added"].cpu().numpy()
    tables, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy()
    slots, positions = np.full(s["rows"], -1, np.int32), np.zeros(s["rows"], np.int32)
    starts, taken, row = np.zeros(len(held) + 1, np.int32), 0, 0
    for r, (h, n) in enumerate(zip(held.tolist(), added.tolist())):
        for i in range(h, h + n):
            if i % PAGE == 0:
                tables[r, i // PAGE] = free[taken]
                taken += 1
            slots[row] = tables[r, i // PAGE] * PAGE + i % PAGE
            positions[row] = s["base"] + i
            row += 1
        starts[r + 1] = row
    return {"lengths": held + added, "starts": starts, "slots": slots, "positions": positions,
            "summary": np.array([0, row, taken, (held + added).max()], np.int32), "tables": tables}


def _exact_store(s):
    x = s["qkv"].double().unflatten(1, (-1, DIM))
    pool = s["pool"].double()
    kh = pool.shape[3]
    qh = x.shape[1] - 2 * kh
    rotated = x[:, :qh + kh].clone()
    angle = s["table"].double()[s["positions"].long()]
    turn = torch.complex(angle[:, : DIM // 2], angle[:, DIM // 2:])[:, None]
    for heads, weight in ((slice(0, qh), s["q_norm"]), (slice(qh, qh + kh), s["k_norm"])):
        h = rotated[:, heads]
        h = h / (h.pow(2).sum(-1, keepdim=True) / DIM + EPS).sqrt() * (1.0 + weight.double())
        z = torch.complex(h[..., : DIM // 2].contiguous(), h[..., DIM // 2:].contiguous()) * turn
        rotated[:, heads] = torch.cat([z.real, z.imag], -1)
    flat = pool.permute(1, 0, 2, 3, 4).reshape(2, -1, kh, DIM)
    flat[0, s["slots"].long()] = rotated[:, qh:]
    flat[1, s["slots"].long()] = x[:, qh + kh:]
    return {"q": rotated[:, :qh], "pool": flat.view(2, -1, PAGE, kh, DIM).permute(1, 0, 2, 3, 4)}


def _exact_attention(s):
    pool, q = s["pool"], s["q"].double()
    kh, qh = pool.shape[3], q.shape[1]
    out = torch.zeros_like(q)

    def rows_of(pages, count, kind):
        return pool[pages.long(), kind].reshape(-1, kh, DIM)[:count].double()

    shared = [rows_of(s["prefix_pages"], s["prefix"], kind) for kind in (0, 1)]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for r, length in enumerate(lengths):
        pages = s["tables"][r, : _pages(length)]
        k, v = (torch.cat([shared[kind], rows_of(pages, length, kind)]) for kind in (0, 1))
        n = starts[r + 1] - starts[r]
        for lo in range(0, n, 64):
            hi = min(n, lo + 64)
            place = s["prefix"] + length - n + torch.arange(lo, hi, device=q.device)[:, None]
            key = torch.arange(k.shape[0], device=q.device)[None]
            seen = (key <= place) & ((key > place - s["window"]) if s["window"] else True)
            for h in range(kh):
                heads = slice(h * (qh // kh), (h + 1) * (qh // kh))
                part = q[starts[r] + lo:starts[r] + hi, heads]
                score = torch.einsum("ngd,kd->ngk", part, k[:, h]) / math.sqrt(DIM)
                weight = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1)
                out[starts[r] + lo:starts[r] + hi, heads] = torch.einsum("ngk,kd->ngd", weight, v[:, h])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "store":
        q = _exact_store(s)
        return {"q": q["q"].reshape(case["rows"], -1, DIM), "pool": q["pool"]}
    return _exact_plan(s)
