"""Paged batch operators (include/plamo_paged.h) against 64-bit statements of
them: plan, store, attention, their refusals and status bits, streams, graphs
and a whole step."""
import ctypes

import numpy as np
import pytest
import torch

from conftest import load_package
from paged_reference import DIM, ROWS, Scene, check, pages_for, plan_by_hand, rotate_store

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def be():
    b = load_package().Backend(device=0)
    yield b
    b.close()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- plan ------------------------------------------------------------------

def plan_scene(requests, seed, extra=3):
    rng = np.random.default_rng(seed)
    held, added = [h for h, _ in requests], [n for _, n in requests]
    have = [pages_for(h) for h in held]
    want = [pages_for(h + n) for h, n in requests]
    ids = rng.permutation(sum(want) + extra).tolist()
    stride = max(want, default=0) + 1
    tables = []
    for n in have:
        tables.append(ids[:n] + [-1] * (stride - n))
        ids = ids[n:]
    return held, added, tables, ids


PLANS = {
    "one": [(0, 1)],
    "none_added": [(5, 0), (64, 0)],
    "edges": [(0, 0), (0, 64), (64, 1), (63, 1), (63, 2), (127, 1), (128, 128), (1, 200), (0, 65), (0, 0)],
    "decode": [(i * 37 % 300, 1) for i in range(2500)],
    "tiles": [(3, 1023), (0, 1), (70, 1), (0, 1024), (1, 2049), (64, 0), (5, 5000)],
    "ragged": [(i * 53 % 190, (i * i * 7) % 90) for i in range(700)],
}


@pytest.mark.parametrize("name", sorted(PLANS))
@pytest.mark.parametrize("spare", [0, 1, 1500])
def test_plan_places_every_row(be, name, spare):
    requests = PLANS[name]
    held, added, tables, free = plan_scene(requests, 3)
    rows = sum(added) + spare
    want = plan_by_hand(held, added, tables, free, rows, 455)
    t = ints(tables)
    got = be.paged_plan(ints(held), ints(added), t, ints(free), rows, base=455)
    for g, w in zip(got, want[:5]):
        assert g.tolist() == list(w)
    assert t.tolist() == want[5]


def test_plan_continues_an_earlier_plans_free_list(be):
    held, added, tables, free = plan_scene([(0, 100), (64, 1)], 4, extra=30)
    t, f = ints(tables), ints(free)
    first = be.paged_plan(ints(held), ints(added), t, f, 101)
    used = pages_for(100) + 1
    assert first.summary.tolist() == [0, 101, used, 100]
    held2, added2 = [100, 65], [64, 0]  # 28 of them fill the second page, the rest a third
    second = be.paged_plan(first.lengths, ints(added2), t, f, 64, after=first)
    want = plan_by_hand(held2, added2, [r[:] for r in t.tolist()], free, 64, 0, head=used)
    assert second.slots.tolist() == want[2]
    assert second.summary.tolist() == [0, 64, used + 1, 164]


@pytest.mark.parametrize("name,change,bit", [
    ("pages", lambda s: s.update(free=s["free"][:1]), 1),
    ("table", lambda s: s.update(tables=[t[:2] for t in s["tables"]]), 2),
    ("rows", lambda s: s.update(rows=s["rows"] - 1), 4),
    ("negative", lambda s: s.update(added=[-1] + s["added"][1:]), 8),
    ("negative held", lambda s: s.update(held=[-64] + s["held"][1:]), 8),
    ("past 2^31", lambda s: s.update(held=[2 ** 31 - 2] + s["held"][1:]), 8),
])
def test_plan_declines_a_step_as_a_whole(be, name, change, bit):
    held, added, tables, free = plan_scene([(10, 60), (0, 130), (64, 7)], 5)
    s = dict(held=held, added=added, tables=tables, free=free, rows=sum(added))
    change(s)
    t = ints(s["tables"])
    got = be.paged_plan(ints(s["held"]), ints(s["added"]), t, ints(s["free"]), s["rows"])
    assert got.summary[0].item() & bit
    assert got.summary.tolist()[1:3] == [0, 0]
    assert got.slots.tolist() == [-1] * s["rows"] and got.positions.tolist() == [0] * s["rows"]
    assert got.lengths.tolist() == s["held"] and got.starts.tolist() == [0] * 4
    assert t.tolist() == s["tables"]


def test_plan_of_no_requests_pads_every_row(be):
    got = be.paged_plan(ints([]), ints([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), ints([3]), 5)
    assert got.slots.tolist() == [-1] * 5 and got.summary.tolist() == [0, 0, 0, 0] and got.starts.tolist() == [0]


# ---- store -------------------------------------------------------------------

def rope_table(count):
    angle = np.arange(count)[:, None] * 10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))
    return torch.tensor(np.concatenate([np.cos(angle), np.sin(angle)], 1), dtype=torch.float32, device="cuda")


def store_tolerance(want, cache):
    """FP32: the norm's sum, root and quotient, two products and a sum, each
    rounded to 2^-24: 2^-20 of the pair's size. BF16 rounds that once more."""
    half = torch.cat([want[..., DIM // 2:], want[..., :DIM // 2]], -1)
    size = torch.sqrt(want ** 2 + half ** 2)
    return 2.0 ** -20 * size + (2.0 ** -8 * want.abs() if cache == BF16 else 0) + 1e-30


@pytest.mark.parametrize("source", [FP32, BF16])
@pytest.mark.parametrize("cache", [FP32, BF16])
@pytest.mark.parametrize("heads,rows,pad", [((16, 1), 1, 0), ((24, 4), 7, 4), ((64, 8), 65, 0), ((3, 3), 300, 12),
                                            ((32, 4), 517, 0)])
def test_store_matches_its_formula(be, source, cache, heads, rows, pad):
    qh, kh = heads
    g = torch.Generator().manual_seed(rows + qh)
    wide = (torch.randn(rows, (qh + 2 * kh) * DIM + pad, generator=g) * 1.7).to(source).cuda()
    qkv = wide[:, :(qh + 2 * kh) * DIM]
    pages = pages_for(rows) + 2
    slots = torch.randperm(pages * ROWS, generator=g)[:rows].int()
    slots[rows // 2] = -1
    positions = torch.randint(0, 5000, (rows,), generator=g).int()
    norms = [(torch.rand(DIM, generator=g) - 0.5).to(BF16).cuda() for _ in range(2)]
    table = rope_table(5000)
    pool = torch.full((pages, 2, ROWS, kh, DIM), 3.0, dtype=cache, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = be.paged_store(qkv, pool, slots.cuda(), positions.cuda(), *norms, table, status=status)
    assert status.item() == 0
    wq, wk, wv = rotate_store(qkv, *norms, table, positions, qh, kh)
    wq[rows // 2] = 0
    check(q, wq, store_tolerance(wq, cache), "queries")
    rest = torch.full((pages, 2, ROWS, kh, DIM), 3.0, dtype=torch.float64)
    tol = torch.full_like(rest, 1e-30)
    for r, s in enumerate(slots.tolist()):
        if s >= 0:
            rest[s // ROWS, 0, s % ROWS], rest[s // ROWS, 1, s % ROWS] = wk[r], wv[r]
            tol[s // ROWS, 0, s % ROWS] = store_tolerance(wk[r], cache)
            tol[s // ROWS, 1, s % ROWS] = store_tolerance(wv[r], cache)
    check(pool, rest, tol, "pool")


def test_store_leaves_out_what_lies_outside(be):
    qkv = torch.randn(4, 6 * DIM, device="cuda")
    norms = [torch.zeros(DIM, dtype=BF16, device="cuda")] * 2
    for slots, positions, bit in (([0, 2 * ROWS, 1, 2], [0, 1, 2, 3], 16), ([0, -2, 1, 2], [0, 1, 2, 3], 16),
                                  ([0, 5, 1, 2], [0, 10, 2, 3], 32), ([0, 5, 1, 2], [0, -1, 2, 3], 32)):
        pool = torch.zeros(2, 2, ROWS, 2, DIM, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        q = be.paged_store(qkv, pool, ints(slots), ints(positions), *norms, rope_table(10), status=status)
        assert status.item() == bit
        stored = pool.abs().amax((0, 1, 3, 4)).nonzero().flatten().tolist()
        assert stored == [0, 1, 2]
        assert (q[1] == 0).all() and (q[[0, 2, 3]].abs().amax((1, 2)) > 0).all()


# ---- attention -----------------------------------------------------------------

def attend(be, s, **more):
    return be.paged_attention(s.q, s.pool, s.starts, s.lengths, s.tables, prefix_pages=s.prefix_pages,
                              prefix_rows=s.prefix, **more)


BATCHES = {
    "first_token": [(0, 1)],
    "page_ends": [(62, 1), (63, 1), (64, 1), (127, 1), (128, 1)],
    "blocks": [(0, 2), (61, 5), (100, 16), (3, 0), (64, 3)],
    "prompts": [(0, 65), (10, 130), (64, 33)],
    "mixed": [(200, 1), (0, 150), (5, 1), (0, 0), (333, 7), (90, 40)],
}


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 1, 64, 130])
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_attention_matches_its_formula(be, name, prefix, dtype):
    s = Scene(BATCHES[name], prefix, 24, 4, dtype, seed=prefix)
    check(attend(be, s), *s.expected(), name)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (16, 1), (32, 4), (64, 8), (40, 1), (14, 2), (70, 1), (300, 1)])
def test_attention_head_layouts(be, heads, dtype):
    s = Scene([(70, 1), (0, 3), (20, 21)], 77, *heads, dtype, seed=heads[0])
    check(attend(be, s), *s.expected(), str(heads))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [1, 2, 64, 100, 129, 300, 10 ** 6])
def test_attention_windows(be, window, dtype):
    s = Scene([(0, 1), (250, 1), (90, 20), (0, 140), (64, 1)], 150, 8, 2, dtype, seed=window % 97)
    check(attend(be, s, window=window), *s.expected(window), f"window {window}")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix,held", [(2000, 1), (0, 5000), (1111, 3333)])
def test_attention_split_along_the_keys(be, prefix, held, dtype):
    s = Scene([(held, 1)], prefix, 12, 2, dtype, seed=held)
    check(attend(be, s), *s.expected(), "split")


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("heads", [(16, 2), (14, 2)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_of_a_batch_behind_a_long_prefix(be, dtype, heads, window):
    """Prefix work that takes tiles in BF16 though every request is short."""
    s = Scene([(i * 7 % 130, 1 if i % 10 else 2) for i in range(150)], 1500, *heads, dtype, seed=11)
    check(attend(be, s, window=window), *s.expected(window), "long prefix")
    s = Scene([(i * 7 % 130, 1) for i in range(150)], 1500, *heads, dtype, seed=12)
    check(attend(be, s, window=window), *s.expected(window), "long prefix, one row each")


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-20, 0.3])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_scales(be, dtype, scale):
    s = Scene([(0, 70), (90, 1)], 40, 8, 2, dtype, seed=13)
    check(attend(be, s, scale=scale), *s.expected(scale=scale), f"scale {scale}")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_many_requests(be, dtype):
    s = Scene([(i * 13 % 150, 0 if i % 11 == 3 else 1) for i in range(700)], 70, 4, 2, dtype, seed=2)
    check(attend(be, s), *s.expected(), "700 requests")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_sharp_scores(be, dtype):
    """Scores hundreds of units apart: all weight on a few rows."""
    s = Scene([(300, 1), (30, 40)], 100, 8, 2, dtype, seed=8, spread=40.0)
    check(attend(be, s), *s.expected(), "sharp")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_strided_rows_and_given_result(be, dtype):
    s = Scene([(70, 1), (0, 30)], 5, 8, 2, dtype, seed=6, spare_rows=3)
    want = s.expected()
    wide = torch.full((s.rows, 12, DIM), float("nan"), dtype=dtype, device="cuda")
    wide[:, 2:10] = s.q
    out = torch.full((s.rows, 9, DIM), 7.0, dtype=dtype, device="cuda")
    s.q = wide[:, 2:10]
    got = attend(be, s, out=out[:, :8])
    check(got, *want, "strided")
    assert (out[:, 8] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_padding_and_unheld_rows_are_zero(be, dtype):
    s = Scene([(40, 2), (0, 3)], 66, 8, 2, dtype, seed=1, spare_rows=4)
    want, tol = s.expected()
    s.lengths = ints([42, 1])  # the second request holds one of its three rows: the last
    s.requests, s.own[1] = [(40, 2), (0, 1)], [t[:1] for t in s.own[1]]
    q, s.q = s.q, s.q[[0, 1, 4, 5, 6, 7, 8]]
    rows, s.rows = s.rows, 7
    w, t = s.expected()
    want[2:5], tol[2:5] = 0, 1e-30
    want[4], tol[4] = w[2], t[2]
    s.q, s.rows = q, rows
    check(attend(be, s), want, tol, "unheld")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window", [0, 90])
def test_attention_rows_not_seen_never_matter(be, bad, window, dtype):
    """A key and a value that are not finite reach exactly the rows that see them."""
    s = Scene([(80, 40), (10, 1)], 30, 8, 2, dtype, seed=3)
    want, tol = s.expected(window)
    at = 100  # own row of the first request: new row 20
    page = s.tables[0, at // ROWS].item()
    s.pool[page, 1, at % ROWS, :, 5] = bad
    first = attend(be, s, window=window)
    seen = torch.zeros(s.rows, dtype=torch.bool)
    seen[20:40] = True  # from its own row on; the window reaches back past it
    assert not torch.isfinite(first.float().cpu()[seen][..., 5]).any()
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[seen, :, 5] = True
    check(torch.where(hit, torch.zeros((), dtype=torch.float64), first.double().cpu()), torch.where(hit, 0.0, want), tol, "value")
    s.pool[page, 0, at % ROWS] = float("nan")
    second = attend(be, s, window=window)
    check(second[~seen], want[~seen], tol[~seen], "key")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("requests", [[(0, 1), (5, 1)], [(0, 40), (70, 1)], [(0, 300)]])
def test_attention_of_keys_that_are_no_numbers(be, requests, dtype):
    """A row all of whose keys are NaN has no result; its neighbours have theirs."""
    s = Scene(requests, 0, 8, 2, dtype, seed=3)
    want, tol = s.expected()
    s.pool[s.tables[0, 0], 0, 0] = float("nan")  # the first request's first key: all its rows see it
    got = attend(be, s)
    n = requests[0][1]
    assert torch.isnan(got[:n]).all()
    check(got[n:], want[n:], tol[n:], "the others")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_values_fallen_out_of_the_window(be, dtype):
    s = Scene([(80, 40), (70, 1)], 100, 8, 2, dtype, seed=3)
    want, tol = s.expected(60)
    s.pool[s.prefix_pages.long(), 1] = float("nan")
    s.pool[s.prefix_pages.long()[-1:], 1, 20:36] = s.shared[1][84:].to(dtype).cuda()
    for r, held in ((0, 80), (1, 70)):
        for row in range(held + 1 - 60):  # seen by none of the request's new rows
            s.pool[s.tables[r, row // ROWS], 1, row % ROWS] = float("inf")
    check(attend(be, s, window=60), want, tol, "window")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_reports_pages_outside_the_pool(be, dtype):
    s = Scene([(100, 1), (200, 1)], 0, 8, 2, dtype, seed=9)
    want, tol = s.expected()
    for page in (-1, s.pool.shape[0], 2 ** 31 - 1):
        s.tables[0, 1] = page
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = attend(be, s, status=status)
        assert status.item() == 16
        check(got[1:], want[1:], tol[1:], "the other request")
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("new", [1, 50])
def test_attention_reports_counts_outside_their_arrays(be, dtype, new):
    """Lengths past the table, negative ones, and rows past the batch: a bit each, the other request as ever."""
    s = Scene([(100, new), (70, 1)], 30, 8, 2, dtype, seed=9)
    want, tol = s.expected()
    good = s.lengths.clone(), s.starts.clone()
    for lengths, starts, bit in (([2 ** 31 - 1, 71], None, 2), ([-5, 71], None, 8), (None, [-3, new, new + 1], 4)):
        s.lengths = good[0] if lengths is None else ints(lengths)
        s.starts = good[1] if starts is None else ints(starts)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = attend(be, s, status=status)
        assert status.item() & bit and not status.item() & 64
        check(got[new:], want[new:], tol[new:], "the other request")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_is_the_same_every_time(be, dtype):
    s = Scene([(i * 29 % 400, 1 + i % 3) for i in range(60)], 700, 16, 2, dtype, seed=4)
    first = attend(be, s)
    for _ in range(3):
        assert torch.equal(attend(be, s), first)


def test_attention_beyond_32_bit_offsets(be):
    """Pages past 2^32 elements of the pool."""
    pages = 40000  # x 131072 elements
    s = Scene([(130, 1), (0, 70)], 100, 16, 8, BF16, seed=7, pool_pages=pages)
    assert s.tables.max().item() * 2 * ROWS * 8 * DIM > 2 ** 32
    check(attend(be, s), *s.expected(), "far pages")
    qkv = torch.randn(3, 32 * DIM, device="cuda")
    norms = [torch.zeros(DIM, dtype=BF16, device="cuda")] * 2
    slots = [(pages - 1) * ROWS + 5, (pages - 2) * ROWS, 7]
    table = rope_table(4)
    be.paged_store(qkv, s.pool, ints(slots), ints([0, 1, 2]), *norms, table)
    _, k, v = rotate_store(qkv, *norms, table, ints([0, 1, 2]), 16, 8)
    for r, slot in enumerate(slots):
        check(s.pool[slot // ROWS, 0, slot % ROWS], k[r], store_tolerance(k[r], BF16))
        check(s.pool[slot // ROWS, 1, slot % ROWS], v[r], store_tolerance(v[r], BF16))


def test_attention_of_an_empty_batch(be):
    s = Scene([], 10, 8, 2, BF16, spare_rows=3)
    assert (attend(be, s) == 0).all()
    s = Scene([(5, 0)], 10, 8, 2, BF16)
    assert attend(be, s).shape == (0, 8, DIM)


# ---- together --------------------------------------------------------------------

def test_a_step_on_another_stream_and_in_a_graph(be):
    """plan, store and attention of a decode step captured once, replayed as
    the requests grow: each replay equals the calls made one by one."""
    qh, kh, prefix, requests = 8, 2, 70, 3
    g = torch.Generator().manual_seed(12)
    base = Scene([(0, 0)], prefix, qh, kh, BF16, seed=12, pool_pages=40)
    pool, table = base.pool, rope_table(prefix + 400)
    norms = [(torch.rand(DIM, generator=g) - 0.5).to(BF16).cuda() for _ in range(2)]
    qkv = torch.zeros(requests + 1, (qh + 2 * kh) * DIM, device="cuda")
    held, added = ints([0, 62, 120]), ints([1, 1, 1])
    tables = torch.full((requests, 5), -1, dtype=torch.int32, device="cuda")
    tables[1, 0], tables[2, 0], tables[2, 1] = 0, 1, 2
    pool[:3] = torch.randn(3, 2, ROWS, kh, DIM, generator=g).to(BF16).cuda()
    free = ints(list(range(3, 30)))
    start = pool.clone(), tables.clone()

    def step(held, pool, tables, after):
        plan = be.paged_plan(held, added, tables, free, requests + 1, base=prefix, after=after)
        q = be.paged_store(qkv, pool, plan.slots, plan.positions, *norms, table)
        return plan, be.paged_attention(q, pool, plan.starts, plan.lengths, tables, prefix_pages=base.prefix_pages,
                                        prefix_rows=prefix)

    inputs = [torch.randn(requests + 1, (qh + 2 * kh) * DIM, generator=g).cuda() for _ in range(5)]
    wants, h, after = [], held.clone(), None
    for x in inputs:
        qkv.copy_(x)
        after, out = step(h, pool, tables, after)
        wants.append(out.clone())
        h = after.lengths.clone()
    assert (wants[0][requests:] == 0).all() and torch.isfinite(wants[-1]).all()

    pool2, tables2 = start
    head = torch.zeros(4, dtype=torch.int32, device="cuda")
    side, kept = torch.cuda.Stream(), held.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        before = load_package().paged.Plan(None, None, None, None, head)
        graph.capture_begin()
        plan, out = step(kept, pool2, tables2, before)
        kept.copy_(plan.lengths)
        head.copy_(plan.summary)
        graph.capture_end()
        for x, want in zip(inputs, wants):
            qkv.copy_(x)
            graph.replay()
            assert torch.equal(out, want)
    torch.cuda.synchronize()
    assert kept.tolist() == [5, 67, 125] and torch.equal(tables2, tables)


@pytest.mark.parametrize("args,bound", [([], 2e-2), (["--fp32"], 2e-4)])
def test_example_serves_a_batch_as_each_request_alone(args, bound):
    """BF16: each layer's keys, values, queries and results are rounded to 2^-8,
    differently placed pages only regroup the sums, so a few roundings' worth
    (2 layers, 20 fed-back steps) may differ; FP32: the same of 2^-24, with the
    projections' 1e-6 and the feedback's growth on top."""
    import importlib.util
    import os
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("paged_batch", os.path.join(ROOT, "examples", "paged_batch.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.main(args) <= bound


# ---- refusals ----------------------------------------------------------------------

def test_attention_refuses_wrong_arguments(be):
    s = Scene([(5, 1)], 3, 8, 2, BF16)
    launches = be.lib.plamo_cuda_kernel_launches(be.ctx)

    def bad(**change):
        a = dict(q=s.q, pool=s.pool, starts=s.starts, lengths=s.lengths, tables=s.tables, prefix_pages=s.prefix_pages,
                 prefix_rows=3)
        a.update(change)
        with pytest.raises(ValueError):
            be.paged_attention(**a)

    bad(q=s.q.float())
    bad(q=s.q[:, :3])                      # 3 query heads over 2 KV heads
    bad(q=s.q.cpu())
    bad(pool=s.pool[:, :, :, :, :64])
    bad(pool=s.pool.half())
    bad(pool=s.pool.transpose(1, 2))
    bad(starts=s.starts.long())
    bad(starts=s.starts[:1])
    bad(tables=s.tables[:, ::2])
    bad(prefix_pages=None)
    bad(prefix_rows=65)                    # one page holds 64
    bad(prefix_rows=-1)
    bad(window=-1)
    bad(scale=float("nan"))
    bad(out=torch.empty(1, 7, DIM, dtype=BF16, device="cuda"))
    bad(status=torch.zeros(2, dtype=torch.int32, device="cuda"))
    shifted = torch.empty(8 * DIM + 1, dtype=BF16, device="cuda")[1:].view(1, 8, DIM)
    bad(q=shifted)                         # not on a 16-byte boundary
    assert be.lib.plamo_cuda_kernel_launches(be.ctx) == launches


def test_c_entries_decline(be):
    abi = load_package()._abi
    s = Scene([(5, 1)], 0, 8, 2, BF16)
    out = torch.empty_like(s.q)
    shape = abi.PagedAttentionArgs(rows=1, requests=1, table_stride=s.tables.shape[1], pages=s.pool.shape[0],
                                   query_heads=8, kv_heads=2, type=0)
    size = be.lib.plamo_paged_attention_workspace(be.ctx, ctypes.byref(shape))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    good = dict(q=s.q.data_ptr(), pool=s.pool.data_ptr(), out=out.data_ptr(), starts=s.starts.data_ptr(),
                lengths=s.lengths.data_ptr(), tables=s.tables.data_ptr(), workspace=ws.data_ptr(),
                workspace_bytes=size, rows=1, q_stride=8 * DIM, out_stride=8 * DIM, requests=1,
                table_stride=s.tables.shape[1], pages=s.pool.shape[0], query_heads=8, kv_heads=2, type=0, scale=0.1, stream=1)

    def call(**change):
        return be.lib.plamo_paged_attention(be.ctx, ctypes.byref(abi.PagedAttentionArgs(**{**good, **change})))

    assert call() == 1
    declines = be.info().declines
    changes = [dict(q=0), dict(pool=0), dict(out=0), dict(starts=0), dict(lengths=0), dict(tables=0), dict(workspace=0),
               dict(workspace=ws.data_ptr() + 16), dict(workspace_bytes=size - 1), dict(type=2), dict(kv_heads=0),
               dict(kv_heads=3), dict(pages=0), dict(q_stride=8), dict(out_stride=8 * DIM + 4), dict(scale=float("inf")),
               dict(prefix_rows=5), dict(rows=1 << 40), dict(prefix_rows=1 << 40)]
    for change in changes:
        assert call(**change) == 0, change
        assert be.info().note.decode().startswith("paged_attention: ")
    assert be.info().declines == declines + len(changes)
    assert be.lib.plamo_paged_attention(be.ctx, None) == 0 and be.lib.plamo_paged_attention(None, None) == 0
    assert be.lib.plamo_paged_attention_workspace(be.ctx, ctypes.byref(abi.PagedAttentionArgs())) == 0
    for name, args in (("plamo_paged_plan", abi.PagedPlanArgs()), ("plamo_paged_store", abi.PagedStoreArgs(rows=1))):
        assert getattr(be.lib, name)(be.ctx, ctypes.byref(args)) == 0
        assert getattr(be.lib, name)(be.ctx, None) == 0
    torch.cuda.synchronize()


def test_plan_and_store_refuse_wrong_arguments(be):
    i = ints([1, 2])
    t = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for a in ((i.long(), i, t, i, 3), (i, i[:1], t, i, 3), (i, i, t[:1], i, 3), (i, i, t.T, i, 3), (i, i, t, t, 3),
              (i, i, t, i, -1), (i.cpu(), i, t, i, 3)):
        with pytest.raises(ValueError):
            be.paged_plan(*a)
    with pytest.raises(ValueError):
        be.paged_plan(i, i, t, i, 3, base=-1)
    pool = torch.zeros(2, 2, ROWS, 2, DIM, device="cuda")
    qkv = torch.zeros(2, 6 * DIM, device="cuda")
    norm, table = torch.zeros(DIM, dtype=BF16, device="cuda"), rope_table(4)
    good = [qkv, pool, i, i, norm, norm, table]
    for at, value in ((0, qkv.half()), (0, qkv[:, :5 * DIM + 1]), (0, qkv[:, :4 * DIM]), (0, qkv.T), (1, pool[0]),
                      (1, pool.half()), (2, i[:1]), (3, i.long()), (4, norm.float()), (5, norm[:5]), (6, table[:, :64]),
                      (6, table.double())):
        with pytest.raises(ValueError):
            be.paged_store(*[value if n == at else a for n, a in enumerate(good)])
