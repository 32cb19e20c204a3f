"""Paged batch operators (include/plamo_paged.h) at the edges of what they take:
malformed device counts, counts near their types' ends, aliased buffers."""
import ctypes

import pytest
import torch

from conftest import load_package
from paged_reference import DIM, ROWS, Scene, check

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def be():
    b = load_package().Backend(device=0)
    yield b
    b.close()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def attend(be, s, **more):
    return be.paged_attention(s.q, s.pool, s.starts, s.lengths, s.tables, prefix_pages=s.prefix_pages,
                              prefix_rows=s.prefix, **more)


@pytest.mark.parametrize("rows,requests", [(65536, 65536), (65536, 131072), (70000, 70000)])
def test_overlapping_rows_past_2_31_stay_in_the_workspace(be, rows, requests):
    """Starts 0, rows, 0, rows, ...: the requests' row counts add up to 2^31 and
    2^32. Reported, and nothing is written beside the workspace or the result."""
    abi = load_package()._abi
    starts = torch.zeros(requests + 1, dtype=torch.int32, device="cuda")
    starts[1::2] = rows
    lengths, tables = torch.full((requests,), 5, dtype=torch.int32, device="cuda"), torch.zeros(requests, 1, dtype=torch.int32, device="cuda")
    q = torch.zeros(rows, 1, DIM, dtype=BF16, device="cuda")
    out = torch.full((rows + 2, 1, DIM), 7.0, dtype=BF16, device="cuda")
    pool = torch.zeros(1, 2, ROWS, 1, DIM, dtype=BF16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = abi.PagedAttentionArgs(q=q.data_ptr(), pool=pool.data_ptr(), out=out[1:].data_ptr(), starts=starts.data_ptr(),
                               lengths=lengths.data_ptr(), tables=tables.data_ptr(), status=status.data_ptr(), rows=rows,
                               q_stride=DIM, out_stride=DIM, requests=requests, table_stride=1, pages=1, query_heads=1,
                               kv_heads=1, type=0, scale=0.1, stream=1)
    size, guard = be.lib.plamo_paged_attention_workspace(be.ctx, ctypes.byref(a)), 1 << 24
    whole = torch.full((guard + size + guard,), 0x5a, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = whole.data_ptr() + guard, size
    torch.cuda.synchronize()
    assert be.lib.plamo_paged_attention(be.ctx, ctypes.byref(a)) == 1
    torch.cuda.synchronize()
    assert status.item() & 4 and not status.item() & 64
    assert (whole[:guard] == 0x5a).all() and (whole[guard + size:] == 0x5a).all()
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    s = Scene([(5, 1), (70, 40)], 0, 1, 1, BF16)  # the next call is as ever
    check(attend(be, s), *s.expected())


def test_counts_near_2_31_are_declined(be):
    """Shapes alone: nothing is enqueued."""
    abi = load_package()._abi

    def size(**change):
        shape = dict(rows=8, requests=4, table_stride=2, pages=8, query_heads=8, kv_heads=2, type=0)
        return be.lib.plamo_paged_attention_workspace(be.ctx, ctypes.byref(abi.PagedAttentionArgs(**{**shape, **change})))

    assert size() and size(requests=1 << 30) and size(rows=1 << 27)
    for change in (dict(requests=(1 << 30) + 1), dict(requests=2 ** 31 - 100), dict(rows=(1 << 27) + 1),
                   dict(rows=(1 << 30) + 1, query_heads=1, kv_heads=1), dict(requests=1 << 62), dict(rows=1 << 62)):
        assert size(**change) == 0, change
        assert "2^30" in be.info().note.decode()


def plan_args(abi, held, added, tables, free, rows, out):
    """A plan's record over int32 tensors; `out`: lengths, starts, slots, positions, summary."""
    return abi.PagedPlanArgs(
        held=held.data_ptr(), added=added.data_ptr(), tables=tables.data_ptr(), free_pages=free.data_ptr(), head=0,
        lengths=out[0].data_ptr(), starts=out[1].data_ptr(), slots=out[2].data_ptr(), positions=out[3].data_ptr(),
        summary=out[4].data_ptr(), requests=held.numel(), table_stride=tables.shape[1], free_count=free.numel(), rows=rows,
        base=7, stream=1)


@pytest.mark.parametrize("requests,new", [(5, 3), (64, 16), (64, 17), (2000, 1), (300, 2000)])
@pytest.mark.parametrize("short", [0, 1])
def test_plan_advances_its_lengths_in_place(be, requests, new, short):
    """lengths == held, below and above the 1,024 rows of one CTA, and where the step is declined."""
    abi = load_package()._abi
    held, added = ints([i * 37 % 200 for i in range(requests)]), ints([new] * requests)
    rows = requests * new - short  # one row too few: declined as a whole
    tables = torch.arange(requests * 40, dtype=torch.int32, device="cuda").view(requests, 40)
    free = torch.arange(100000, 200000, dtype=torch.int32, device="cuda")
    want_tables = tables.clone()
    want = be.paged_plan(held, added, want_tables, free, rows, base=7)
    out = [torch.full((n,), -9, dtype=torch.int32, device="cuda") for n in (requests, requests + 1, rows, rows, 4)]
    out[0] = held  # in place
    torch.cuda.synchronize()
    assert be.lib.plamo_paged_plan(be.ctx, ctypes.byref(plan_args(abi, held, added, tables, free, rows, out))) == 1
    for got, w in zip(out, want):
        assert torch.equal(got, w)
    assert torch.equal(tables, want_tables) and bool(want.summary[0]) == bool(short)


def test_plan_declines_buffers_that_overlap(be):
    abi = load_package()._abi
    requests, rows = 8, 3000
    buf = torch.zeros(20000, dtype=torch.int32, device="cuda")
    held, added, tables, free = buf[:8], buf[100:108], buf[200:600].view(8, 50), buf[1000:1100]
    out = [buf[2000:2008], buf[3000:3009], buf[4000:7000], buf[8000:11000], buf[12000:12004]]

    def call(**change):
        args = plan_args(abi, held, added, tables, free, rows, out)
        for name, value in change.items():
            setattr(args, name, value)
        return be.lib.plamo_paged_plan(be.ctx, ctypes.byref(args))

    launches = be.lib.plamo_cuda_kernel_launches(be.ctx)
    at = buf.data_ptr()
    for change in (dict(lengths=at + 4), dict(lengths=at + 4 * 100), dict(starts=at), dict(slots=at + 4 * 300),
                   dict(positions=at + 4 * 1099), dict(summary=at + 4 * 107), dict(held=at + 4 * 201), dict(head=at + 4 * 3004),
                   dict(slots=at + 4 * 7500), dict(tables=at + 4 * 990), dict(starts=at + 4 * 12003)):
        assert call(**change) == 0, change
        assert "overlap" in be.info().note.decode()
    assert be.lib.plamo_cuda_kernel_launches(be.ctx) == launches
    assert call() == 1
    torch.cuda.synchronize()


@pytest.mark.parametrize("bad", [-1, -64, 1 << 25, 2 ** 31 - 1])
@pytest.mark.parametrize("where", ["table", "free list"])
def test_rows_on_page_ids_that_are_none_are_reported(be, where, bad):
    """Not taken for padding: the store leaves them out and says so."""
    tables, free = ints([[0, -1, -1], [1, -1, -1]]), ints([2, 3, 4])
    if where == "table":
        tables[1, 0] = bad  # rows 70, 71 of the batch: held page of the second request
    else:
        free[1] = bad       # the second request's first new page: its rows from own row 64 on
    plan = be.paged_plan(ints([10, 62]), ints([70, 4]), tables, free, 80)
    lost = [70, 71] if where == "table" else [72, 73]
    slots = plan.slots.tolist()
    assert [i for i, s in enumerate(slots) if s == -2] == lost and slots[74:] == [-1] * 6
    assert all(s >= 0 for i, s in enumerate(slots[:74]) if i not in lost) and plan.summary.tolist()[:2] == [0, 74]
    pool = torch.zeros(5, 2, ROWS, 2, DIM, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    norm, table = torch.zeros(DIM, dtype=BF16, device="cuda"), torch.ones(100, DIM, device="cuda")
    q = be.paged_store(torch.randn(80, 6 * DIM, device="cuda"), pool, plan.slots, plan.positions, norm, norm, table, status=status)
    assert status.item() == 16 and (q[lost] == 0).all() and (q[74:] == 0).all()
    assert int((pool.abs().amax((1, 3, 4)) > 0).sum()) == 72


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 40])
@pytest.mark.parametrize("new", [1, 60])
def test_rows_before_the_first_start_are_zero_and_reported(be, new, prefix, dtype):
    s = Scene([(100, new), (70, 1)], prefix, 8, 2, dtype, seed=9)
    want, tol = s.expected()
    first = 3
    s.q = torch.cat([s.q.new_full((first, 8, DIM), 2.0), s.q])
    s.starts = s.starts + first
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(s.q, float("nan"))
    assert attend(be, s, out=out, status=status) is out
    assert status.item() == 4 and (out[:first] == 0).all()
    check(out[first:], want, tol, "the requests' rows")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 40])
@pytest.mark.parametrize("rows,starts", [(20, [0, 12, 5, 20]), (20, [0, 6, 0, 20]), (300, [0, 200, 100, 250]), (20, [9, 4, 2, 0])])
def test_starts_that_decrease_leave_zeros(be, rows, starts, prefix, dtype):
    s = Scene([(100, 1)] * 3, prefix, 8, 2, dtype, seed=9)
    s.q = torch.randn(rows, 8, DIM, device="cuda").to(dtype)
    s.starts = ints(starts)
    for _ in range(2):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full_like(s.q, float("nan"))
        attend(be, s, out=out, status=status)
        assert status.item() & 4 and not status.item() & 64
        assert (out == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 100])
@pytest.mark.parametrize("requests", [[(0, 1), (70, 1), (200, 1)], [(0, 3), (70, 2), (5, 4)], [(0, 90), (70, 40), (300, 1)]])
def test_rows_all_of_whose_scores_are_minus_infinity(be, requests, prefix, dtype):
    """They see keys, so theirs is 0 / 0, no result; one finite score is the whole result;
    rows that are not held stay zero."""
    s = Scene(requests, prefix, 8, 2, dtype, seed=5, spread=0.2)
    s.q[..., 0] = 1.0
    s.pool[s.prefix_pages.long(), 0, :, :, 0] = -float("inf")
    for r, (held, new) in enumerate(requests):
        for row in range(held + new):
            s.pool[s.tables[r, row // ROWS], 0, row % ROWS, :, 0] = -float("inf")
    # The last request's own row 2 (its new row, or one held) has an ordinary key.
    r, (held, new) = len(requests) - 1, requests[-1]
    s.pool[s.tables[r, 0], 0, 2, :, 0] = 0.5
    got = attend(be, s)
    first = int(s.starts[r])
    assert torch.isnan(got[:first]).all()
    value = s.own[r][1][2].repeat_interleave(4, 0)
    want = value.expand(new, 8, DIM).clone()
    check(got[first:], want, 2.0 ** -8 * want.abs() + 1e-30 if dtype == BF16 else 2.0 ** -20 * want.abs() + 1e-30, "one score")
    s.lengths = s.lengths.clone()
    s.lengths[0] = 0
    got = attend(be, s)
    assert (got[:requests[0][1]] == 0).all() and torch.isnan(got[requests[0][1]:first]).all()


def test_calls_without_a_status_word_report_to_the_backend(be):
    be.paged_status()
    s = Scene([(100, 1), (200, 1)], 0, 8, 2, BF16, seed=9)
    attend(be, s)
    assert be.paged_status() == 0
    s.tables[0, 1] = -1
    attend(be, s)
    s.lengths = ints([2 ** 31 - 1, 201])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(be, s)
        assert be.paged_status() == 16 | 2
        assert be.paged_status() == 0
    pool, norm = torch.zeros(1, 2, ROWS, 2, DIM, device="cuda"), torch.zeros(DIM, dtype=BF16, device="cuda")
    store = (torch.ones(2, 6 * DIM, device="cuda"), pool, ints([0, 1]), ints([0, 9]), norm, norm, torch.ones(5, DIM, device="cuda"))
    be.paged_store(*store)
    own = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert be.paged_status() == 32
    be.paged_store(*store, status=own)  # a word of its own: there only
    assert be.paged_status() == 0 and own.item() == 32


def test_example_of_many_steps_has_a_rotation_for_each():
    """FP32 and one layer: the bound of a step's roundings in the shorter run holds, whatever the steps."""
    import importlib.util
    import os
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("paged_batch", os.path.join(ROOT, "examples", "paged_batch.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.main(["--fp32", "--steps", "420", "--requests", "1", "--layers", "1", "--prefix", "3"]) <= 2e-4


def launches_of(be, call):
    before = be.lib.plamo_cuda_kernel_launches(be.ctx)
    result = call()
    return result, be.lib.plamo_cuda_kernel_launches(be.ctx) - before


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 12, 300])
@pytest.mark.parametrize("spare", [1, 7])
def test_spare_rows_of_a_decode_step_ask_for_no_other_kernels(be, spare, prefix, dtype):
    """(The prefix's units are numbered over spare rows too, so sums may be cut elsewhere.)"""
    s = Scene([(i * 53 % 400, 1) for i in range(61)], prefix, 32, 4, dtype, seed=31)
    s.tables = torch.nn.functional.pad(s.tables, (0, 64), value=-7)  # room for 4,096 rows more
    want, tol = s.expected()
    _, few = launches_of(be, lambda: attend(be, s))
    s.q = torch.cat([s.q, s.q[:1].expand(spare, -1, -1)])
    got, some = launches_of(be, lambda: attend(be, s, most_new=1))
    check(got[:61], want, tol, "requests' rows")
    assert (got[61:] == 0).all() and some == few


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_a_prompt_among_idle_slots_gets_tiles(be, dtype):
    s = Scene([(0, 0)] * 200 + [(30, 190)] + [(0, 0)] * 200, 300, 16, 2, dtype, seed=32)
    s.tables = torch.nn.functional.pad(s.tables, (0, 20), value=-7)
    alone = Scene([(30, 190)], 300, 16, 2, dtype, seed=32)
    alone.tables = torch.nn.functional.pad(alone.tables, (0, 20), value=-7)
    _, tiles = launches_of(be, lambda: attend(be, alone))
    got, count = launches_of(be, lambda: attend(be, s, most_new=190))
    assert count == tiles
    check(got, *s.expected(), "prompt among idle slots")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("most_new", [1, 2, 40, 150, 10 ** 9])
def test_results_do_not_depend_on_what_most_new_says(be, most_new, dtype):
    s = Scene([(200, 1), (0, 150), (5, 1), (0, 0), (333, 7), (90, 40)], 70, 24, 4, dtype, seed=33)
    check(attend(be, s, most_new=most_new), *s.expected(), f"most_new {most_new}")
    with pytest.raises(ValueError):
        attend(be, s, most_new=-1)


def test_few_pairs_read_a_long_prefix_in_the_row_kernel(be):
    """One request's prefix is read once there; many requests' in the tile kernel."""
    pool = torch.zeros(1200, 2, ROWS, 4, DIM, dtype=BF16, device="cuda")
    pages = torch.arange(1, 1025, dtype=torch.int32, device="cuda")

    def count(requests, rows):
        q = torch.ones(requests, 32, DIM, dtype=BF16, device="cuda")
        one = torch.ones(requests, dtype=torch.int32, device="cuda")
        starts = torch.arange(requests + 1, dtype=torch.int32, device="cuda")
        out, launches = launches_of(be, lambda: be.paged_attention(q, pool, starts, one, torch.zeros(requests, 1, dtype=torch.int32, device="cuda"),
                                                                   prefix_pages=pages, prefix_rows=rows))
        assert (out == 0).all()
        return launches

    assert count(1, 65536) == count(2, 65536) == count(16, 1000) == 2
    assert count(8, 65536) == count(61, 4096) == 3


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("requests,prefix", [([(300, 1), (40, 1)], 0), ([(300, 1), (40, 1)], 200), ([(0, 300), (60, 90)], 200),
                                             ([(20, 5), (200, 8)], 30)])
def test_infinite_values_that_are_seen_make_infinite_results(be, requests, prefix, sign, dtype):
    """No number would be a zero part of a weight times an infinity."""
    s = Scene(requests, prefix, 8, 2, dtype, seed=41)
    want, tol = s.expected()
    hit = torch.zeros_like(want, dtype=torch.bool)
    if prefix:
        s.pool[s.prefix_pages[0], 1, 3, :, 7] = sign * float("inf")
        hit[:, :, 7] = True
    first, (held, new) = 0, requests[0]
    s.pool[s.tables[0, 0], 1, 9, :, 100] = sign * float("inf")
    hit[first + max(0, 9 - held):first + new, :, 100] = True
    got = attend(be, s).double().cpu()
    assert (got[hit] == sign * float("inf")).all()
    check(torch.where(hit, 0.0, got), torch.where(hit, 0.0, want), tol, "the other dimensions")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_requests_that_hold_nothing_need_no_page_table(be, dtype):
    """Tables of no columns, and a rotation table of no positions, beside rows that are all padding."""
    tables, none = torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints([0, 0])
    plan = be.paged_plan(none, none, tables, ints([]), 3)
    assert plan.summary.tolist() == [0, 0, 0, 0] and plan.slots.tolist() == [-1] * 3
    assert be.paged_plan(none, ints([0, 1]), tables, ints([4]), 3).summary[0].item() == 2
    pool, norm = torch.ones(2, 2, ROWS, 2, DIM, dtype=dtype, device="cuda"), torch.zeros(DIM, dtype=BF16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    empty = torch.empty(0, DIM, device="cuda")
    q = be.paged_store(torch.ones(3, 6 * DIM, device="cuda"), pool, plan.slots, plan.positions, norm, norm, empty, status=status)
    assert (q == 0).all() and (pool == 1).all()
    for prefix in (0, 70):
        out = be.paged_attention(q, pool, plan.starts, plan.lengths, tables, prefix_pages=ints([0, 1]), prefix_rows=prefix, status=status)
        assert (out == 0).all()
    assert status.item() == 0
    be.paged_store(torch.ones(3, 6 * DIM, device="cuda"), pool, ints([5, -1, -1]), plan.positions, norm, norm, empty, status=status)
    assert status.item() == 32 and (pool == 1).all()
    be.paged_attention(q, pool, ints([0, 1, 3]), ints([1, 2]), tables, status=status)
    assert status.item() & 2
