"""Draft trees in a paged batch (include/plamo_paged.h) against 64-bit statements:
masks and positions, attention, the confirmed path, the moved rows, refusals
and status bits, streams, graphs and a whole step."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT, load_package
from paged_reference import DIM, ROWS, Scene, check, pages_for
from paged_tree_reference import TreeScene, accept_by_hand, random_tree, signed, tree_by_hand

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def be():
    b = load_package().Backend(device=0)
    yield b
    b.close()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(trees):
    out = [0]
    for t in trees:
        out.append(out[-1] + len(t))
    return out


def gen(seed):
    return torch.Generator().manual_seed(seed)


def some_trees(sizes, seed, depth=None):
    g = gen(seed)
    return [random_tree(n, g, depth) for n in sizes]


CHAIN = list(range(-1, 15))
STAR = [-1] + [0] * 31
TREES = {
    "one": [[-1]],
    "chain_star": [CHAIN, [], STAR],
    "two_roots": [[-1, -1, 0, 1, 2]],
    "sizes": some_trees([1, 31, 32, 33, 0, 64, 65], 1),
    "largest": some_trees([256, 0, 255, 129], 2),
    "long_chain": [list(range(-1, 255))],
    "many": some_trees([i * 7 % 40 for i in range(300)], 3, depth=5),
}


# ---- masks and positions -----------------------------------------------------

@pytest.mark.parametrize("spare", [0, 3, 1000])
@pytest.mark.parametrize("name", sorted(TREES))
def test_tree_masks_and_positions(be, name, spare):
    trees = TREES[name]
    held = [i * 53 % 500 for i in range(len(trees))]
    starts = starts_of(trees)
    rows = starts[-1] + spare
    status = ints([0])
    got = be.paged_tree(ints(sum(trees, []) + [9] * spare), ints(starts), ints([h + len(t) for h, t in zip(held, trees)]),
                        max(map(len, trees)), base=455, status=status)
    positions, masks = tree_by_hand(trees, held, got.masks.shape[1], 455, rows)
    assert got.positions.tolist() == positions
    assert torch.equal(got.masks.cpu(), signed(masks))
    assert status.item() == 0


@pytest.mark.parametrize("parents,at", [([-1, 1, 0], 1), ([-2, 0], 0), ([-1, 0, 7], 2), ([0, 0], 0), ([-1, -2 ** 31, 1], 1),
                                        ([-1, 2 ** 31 - 1], 1)])
def test_tree_reports_parents_out_of_range(be, parents, at):
    status = ints([0])
    got = be.paged_tree(ints(parents), ints([0, len(parents)]), ints([5 + len(parents)]), 3, status=status)
    mended = parents[:at] + [-1] + parents[at + 1:]
    positions, masks = tree_by_hand([mended], [5], 1, 0, len(parents))
    assert status.item() == 128
    assert got.positions.tolist() == positions and torch.equal(got.masks.cpu(), signed(masks))


def test_tree_reports_more_rows_than_bits(be):
    trees = [list(range(-1, 39)), [-1, 0]]
    status = ints([0])
    got = be.paged_tree(ints(sum(trees, [])), ints([0, 40, 42]), ints([45, 2]), 32, status=status)
    assert status.item() == 128
    _, masks = tree_by_hand([trees[0][:32]], [5], 1, 0, 32)
    assert torch.equal(got.masks[:32].cpu(), signed(masks))
    assert got.masks[32:].tolist() == [[0]] * 8 + [[1], [3]]


def test_tree_of_no_requests_pads_every_row(be):
    got = be.paged_tree(ints([3, 3]), ints([0]), ints([]), 1)
    assert got.positions.tolist() == [0, 0] and got.masks.tolist() == [[0], [0]]


# ---- attention -----------------------------------------------------------------

def attend(be, s, **more):
    return be.paged_attention(s.q, s.pool, s.starts, s.lengths, s.tables, prefix_pages=s.prefix_pages, prefix_rows=s.prefix,
                              masks=s.masks, **more)


def wide(s, columns=2100):
    """Page tables with room for so many rows that the tile kernels are asked for."""
    s.tables = torch.nn.functional.pad(s.tables, (0, columns), value=-7)
    return s


BATCHES = {
    "first_token": [(0, [-1])],
    "page_ends": [(62, [-1, 0, 0]), (63, [-1, 0, 1]), (64, [-1]), (125, [-1, 0, 0, 1]), (128, [-1, 0])],
    "trees": [(0, CHAIN), (100, STAR), (3, []), (60, some_trees([24], 4)[0])],
    "wide": [(200, some_trees([64], 5)[0]), (0, some_trees([130], 6)[0]), (333, [-1, 0, 0, 2, 2]), (1, some_trees([33], 7)[0])],
}


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 1, 130, 600])
@pytest.mark.parametrize("name", sorted(BATCHES))
def test_attention_matches_its_formula(be, name, prefix, dtype, tables):
    s = TreeScene(BATCHES[name], prefix, 24, 4, dtype, seed=prefix)
    status = ints([0])
    check(attend(be, wide(s) if tables == "long" else s, status=status), *s.expected(), name)
    assert status.item() == 0


@pytest.mark.parametrize("prefix", [77, 700])
@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (16, 1), (32, 4), (40, 1), (14, 2), (70, 1), (300, 1)])
def test_attention_head_layouts(be, heads, dtype, tables, prefix):
    s = TreeScene([(70, [-1]), (0, [-1, 0, 0]), (20, some_trees([21], 8)[0]), (130, CHAIN)], prefix, *heads, dtype, seed=heads[0])
    check(attend(be, wide(s) if tables == "long" else s), *s.expected(), str(heads))


@pytest.mark.parametrize("prefix", [150, 530])
@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 129, 300, 10 ** 6])
def test_attention_windows(be, window, dtype, tables, prefix):
    s = TreeScene([(0, [-1]), (250, CHAIN), (90, some_trees([40], 9)[0]), (0, list(range(-1, 70))), (64, [-1, 0, 0])], prefix, 8, 2,
                  dtype, seed=window % 97)
    check(attend(be, wide(s) if tables == "long" else s, window=window), *s.expected(window), f"window {window}")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix,held,rows", [(2000, 1, 5), (0, 5000, 64), (1111, 3333, 33), (0, 4000, 2)])
def test_attention_split_along_the_keys(be, prefix, held, rows, dtype):
    s = TreeScene([(held, some_trees([rows], rows)[0])], prefix, 12, 2, dtype, seed=held)
    check(attend(be, s, most_new=rows), *s.expected(), "split")


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_of_many_trees_behind_a_long_prefix(be, dtype, window):
    """Requests of one row beside trees of up to 40: short ones' own rows and others' tiles are joined with shared tiles."""
    trees = some_trees([(1, 2, 40, 17, 0, 33)[i % 6] for i in range(40)], 11)
    s = TreeScene([(i * 37 % 330, t) for i, t in enumerate(trees)], 1500, 16, 2, dtype, seed=11, spare_rows=7)
    want = s.expected(window)
    check(attend(be, s, window=window, most_new=40), *want, "long prefix")
    check(attend(be, wide(s), window=window), *want, "long prefix and tables")


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-20, 0.3])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_scales(be, dtype, scale):
    s = wide(TreeScene([(0, some_trees([70], 13)[0]), (90, [-1, 0])], 40, 8, 2, dtype, seed=13))
    check(attend(be, s, scale=scale), *s.expected(scale=scale), f"scale {scale}")


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_sharp_scores(be, dtype, tables):
    s = TreeScene([(300, [-1]), (30, some_trees([40], 14)[0])], 100, 8, 2, dtype, seed=8, spread=40.0)
    check(attend(be, wide(s) if tables == "long" else s), *s.expected(), "sharp")


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_strided_rows_and_given_result(be, dtype, tables):
    s = TreeScene([(70, [-1, 0, 0]), (0, some_trees([30], 15)[0])], 5, 8, 2, dtype, seed=6, spare_rows=3)
    want = s.expected()
    rows = torch.full((s.rows, 12, DIM), float("nan"), dtype=dtype, device="cuda")
    rows[:, 2:10] = s.q
    out = torch.full((s.rows, 9, DIM), 7.0, dtype=dtype, device="cuda")
    s.q = rows[:, 2:10]
    check(attend(be, wide(s) if tables == "long" else s, out=out[:, :8]), *want, "strided")
    assert (out[:, 8] == 7).all()


def any_masks(s, seed, share):
    """Masks of no tree: rows that see later ones, not themselves, nothing at all."""
    g = gen(seed)
    s.set_masks([[[j for j in range(n) if torch.rand(1, generator=g) < share and i % 4] for i in range(n)] for _, n in s.requests])
    return s


@pytest.mark.parametrize("window", [0, 3, 70])
@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix,held", [(0, 0), (0, 40), (90, 0), (600, 5)])
def test_attention_takes_any_masks(be, prefix, held, dtype, tables, window):
    """Every fourth row's mask is empty; with no prefix and no held rows it sees nothing and is zero."""
    s = any_masks(TreeScene([(held, CHAIN), (held, some_trees([70], 16)[0]), (held, [-1])], prefix, 8, 2, dtype, seed=prefix), 3, 0.3)
    check(attend(be, wide(s) if tables == "long" else s, window=window), *s.expected(window), "any masks")


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 66, 600])
def test_attention_bits_past_a_requests_rows_mean_nothing(be, prefix, dtype, tables):
    s = TreeScene([(40, CHAIN), (0, some_trees([9], 17)[0]), (61, [-1, 0])], prefix, 8, 2, dtype, seed=2, words=3)
    want = s.expected()
    row = 0
    for _, n in s.requests:
        bits = torch.full((3,), -1, dtype=torch.int32)
        for w in range(3):
            low = min(max(n - 32 * w, 0), 32)
            bits[w] = -1 << low if low < 32 else 0
        s.masks[row:row + n] |= bits.cuda()
        row += n
    check(attend(be, wide(s) if tables == "long" else s), *want, "bits past the rows")


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 66, 600])
def test_attention_padding_and_unheld_requests_are_zero(be, prefix, dtype, tables):
    s = TreeScene([(40, [-1, 0]), (0, CHAIN), (7, STAR)], prefix, 8, 2, dtype, seed=1, spare_rows=4)
    want, tol = s.expected()
    want[2:18], tol[2:18] = 0, 1e-30
    s.lengths[1] = 15  # holds one row fewer than it adds
    check(attend(be, wide(s) if tables == "long" else s), want, tol, "unheld")


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("prefix,window", [(30, 0), (30, 90), (600, 0)])
def test_attention_rows_not_seen_never_matter(be, bad, prefix, window, dtype, tables):
    """A drafted row's key and value that are not finite reach exactly the rows below it."""
    s = TreeScene([(80, some_trees([40], 18)[0]), (10, [-1, 0])], prefix, 8, 2, dtype, seed=3)
    if tables == "long":
        wide(s)
    want, tol = s.expected(window)
    j = 3
    at = 80 + j
    page = s.tables[0, at // ROWS].item()
    s.pool[page, 1, at % ROWS, :, 5] = bad
    first = attend(be, s, window=window)
    seen = torch.tensor([j in line for line in s.sees[0]] + [False, False])
    assert 1 < seen.sum() < 40
    assert not torch.isfinite(first.float().cpu()[seen][..., 5]).any()
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[seen, :, 5] = True
    check(torch.where(hit, torch.zeros((), dtype=torch.float64), first.double().cpu()), torch.where(hit, 0.0, want), tol, "value")
    s.pool[page, 0, at % ROWS] = float("nan")
    second = attend(be, s, window=window)
    check(second[~seen], want[~seen], tol[~seen], "key")
    assert torch.isnan(second.float().cpu()[seen]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tables", ["short", "long"])
def test_attention_scores_of_minus_infinity_have_no_result(be, dtype, tables):
    """Seeing scores of -infinity only is not seeing nothing."""
    s = TreeScene([(0, [-1, 0, 0]), (0, CHAIN)], 0, 8, 2, dtype, seed=3)
    want, tol = s.expected()
    s.q[0] = s.q[0].abs() + 1  # the root sees itself alone
    s.pool[s.tables[0, 0], 0, 0] = float("-inf")
    got = attend(be, wide(s) if tables == "long" else s)
    assert torch.isnan(got[0]).all()
    check(got[3:], want[3:], tol[3:], "the others")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [30, 600])
def test_attention_reports_what_lies_outside(be, dtype, prefix):
    s = wide(TreeScene([(100, CHAIN), (200, [-1, 0])], prefix, 8, 2, dtype, seed=9))
    want, tol = s.expected()
    page = s.tables[0, 1].item()
    for bad in (-1, s.pool.shape[0], 2 ** 31 - 1):
        s.tables[0, 1] = bad
        status = ints([0])
        got = attend(be, s, status=status)
        assert status.item() == 16 and torch.isfinite(got).all()
        check(got[16:], want[16:], tol[16:], "the other request")
    s.tables[0, 1] = page
    status = ints([0])
    s.words, s.masks = 1, s.masks[:, :1].contiguous()
    s.trees[0] = CHAIN
    attend(be, s, status=status)
    assert status.item() == 0
    many = wide(TreeScene([(3, some_trees([40], 1)[0]), (9, [-1])], prefix, 8, 2, dtype))
    want, tol = many.expected()
    many.masks = many.masks[:, :1].contiguous()
    got = attend(be, many, status=status)
    assert status.item() == 128
    check(got[40:], want[40:], tol[40:], "the other request")
    check(got[:32], want[:32], tol[:32], "rows that have bits")


@pytest.mark.parametrize("change", [lambda s: s.starts.copy_(ints([0, 30, 20, 42])), lambda s: s.starts.copy_(ints([0, 16, 48, 2 ** 30])),
                                    lambda s: s.starts.copy_(ints([-5, 16, 48, 50])), lambda s: s.lengths.copy_(ints([-1, 2 ** 31 - 1, 3]))])
@pytest.mark.parametrize("prefix", [0, 600])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_of_counts_outside_their_arrays_stays_in_bounds(be, dtype, prefix, change):
    s = wide(TreeScene([(40, CHAIN), (7, STAR), (100, [-1, 0])], prefix, 8, 2, dtype, seed=1))
    out = torch.full((s.rows + 2, 8, DIM), 7.0, dtype=dtype, device="cuda")
    change(s)
    status = ints([0])
    attend(be, s, out=out[1:-1], status=status)
    assert status.item() & ~64 and not status.item() & 64
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    s = wide(TreeScene([(40, CHAIN), (7, STAR), (100, [-1, 0])], prefix, 8, 2, dtype, seed=1))
    check(attend(be, s), *s.expected(), "the next call")


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_of_chains_is_the_plain_one(be, dtype, tables):
    """Masks of chains see what a causal batch sees."""
    s = TreeScene([(70, CHAIN), (5, [-1]), (130, list(range(-1, 60)))], 40, 16, 2, dtype, seed=5)
    if tables == "long":
        wide(s)
    want, tol = s.expected()
    check(attend(be, s), want, tol, "trees")
    plain = be.paged_attention(s.q, s.pool, s.starts, s.lengths, s.tables, prefix_pages=s.prefix_pages, prefix_rows=s.prefix)
    check(plain, want, tol, "plain")


@pytest.mark.parametrize("prefix", [12, 700])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_is_the_same_every_time_captured_and_on_another_stream(be, dtype, prefix):
    trees = some_trees([16, 40, 1, 33, 8], 21)
    s = wide(TreeScene([(i * 97 % 400, t) for i, t in enumerate(trees)], prefix, 16, 2, dtype, seed=4))
    first = attend(be, s)
    assert all(torch.equal(attend(be, s), first) for _ in range(3))
    stream, out = torch.cuda.Stream(), torch.zeros_like(first)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attend(be, s, out=out)
    stream.synchronize()
    assert torch.equal(out, first)
    graph, captured = torch.cuda.CUDAGraph(), torch.zeros_like(first)
    with torch.cuda.graph(graph):
        attend(be, s, out=captured)
    captured.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, first)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_on_two_streams_at_once(be, dtype):
    """Each call has a workspace of its own."""
    scenes = [wide(TreeScene([(i * 97 % 400, t) for i, t in enumerate(some_trees(sizes, 21))], prefix, 16, 2, dtype, seed=4))
              for sizes, prefix in (([16, 40, 1, 33, 8], 700), ([12, 30, 64], 12))]
    want = [attend(be, s) for s in scenes]
    streams, got = [torch.cuda.Stream() for _ in scenes], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(attend(be, scenes[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_pages_past_four_gigabytes(be, dtype, tables):
    """A pool whose used pages lie more than 2^32 bytes behind its start gives what a small one does."""
    s = TreeScene([(i * 131 % 300, t) for i, t in enumerate(some_trees([16, 40, 3], 2))], 200, 16, 8, dtype, seed=6)
    if tables == "long":
        wide(s)
    be.paged_status()
    small, used = attend(be, s), s.pool.shape[0]
    page_bytes = s.pool[0].numel() * s.pool.element_size()
    first = 2 ** 32 // page_bytes + 5
    large = torch.empty(first + used, *s.pool.shape[1:], dtype=dtype, device="cuda")
    large[first:] = s.pool
    s.pool = large
    s.tables = torch.where(s.tables >= 0, s.tables + first, s.tables)
    s.prefix_pages = s.prefix_pages + first
    assert torch.equal(attend(be, s), small)
    path = torch.full((s.q.shape[0],), -1, dtype=torch.int32, device="cuda")
    path[:3] = ints([0, 5, 9])
    before = large[first:].clone()
    be.paged_keep([large], path, s.starts, s.lengths, s.tables)
    be.paged_keep([before], path, s.starts, s.lengths, torch.where(s.tables >= 0, s.tables - first, s.tables))
    assert torch.equal(large[first:].view(torch.uint8), before.view(torch.uint8))  # (rows of no request hold NaN)
    assert be.paged_status() == 0


# ---- acceptance and the moved rows --------------------------------------------------

def accept_scene(sizes, seed, vocabulary=3, held=None, tables=None):
    """Trees with so few tokens that paths of all lengths and siblings with one token occur."""
    g = gen(seed)
    trees = [random_tree(n, g) for n in sizes]
    rows = sum(sizes)
    tokens = torch.randint(vocabulary, (rows,), generator=g).tolist()
    chosen = torch.randint(vocabulary, (rows,), generator=g).tolist()
    held = held or [int(x) for x in torch.randint(200, (len(sizes),), generator=g)]
    counts = [pages_for(h + n) for h, n in zip(held, sizes)]
    order = torch.randperm(sum(counts) + 9, generator=g).tolist()
    stride, tables = max(counts, default=0) + 1, []
    for n in counts:
        tables.append(order[:n] + [-7] * (stride - n))
        order = order[n:]
    head = sum(pages_for(h + n) - pages_for(h) for h, n in zip(held, sizes))
    free = [10 ** 6 + i for i in range(head + 5)]
    return trees, tokens, chosen, held, tables, free, head


ACCEPTS = {
    "one": [1],
    "none": [0, 0],
    "sizes": [16, 0, 1, 64, 33, 256, 2],
    "sixty_four": [(i * 11) % 50 for i in range(64)],
    "sixty_five": [(i * 13) % 70 for i in range(65)],
    "many": [(i * 7) % 20 for i in range(2500)],
}


def call_accept(be, s, spare=0):
    trees, tokens, chosen, held, tables, free, head = s
    f = ints(free)
    lengths = ints([h + len(t) for h, t in zip(held, trees)])
    got = be.paged_accept(ints(sum(trees, []) + [0] * spare), ints(tokens + [0] * spare), ints(chosen + [0] * spare),
                          ints(starts_of(trees)), lengths, ints(tables), f, ints([0, len(tokens), head, 0]))
    return got, f


@pytest.mark.parametrize("spare", [0, 70])
@pytest.mark.parametrize("name", sorted(ACCEPTS))
def test_accept_walks_each_tree(be, name, spare):
    s = accept_scene(ACCEPTS[name], len(name))
    counts, kept, last, path, after, summary, free = accept_by_hand(*s)
    got, f = call_accept(be, s, spare)
    assert got.counts.tolist() == counts and got.lengths.tolist() == kept and got.last.tolist() == last
    assert got.path.tolist() == path + [-1] * spare and got.tokens.tolist() == after + [-1] * spare
    assert got.summary.tolist() == summary
    assert f.tolist() == free


def test_accept_takes_the_first_of_siblings_and_no_later_root(be):
    trees = [[-1, 0, 0, 1, -1, 4]]
    s = (trees, [5, 8, 8, 9, 5, 9], [8, 9, 9, 1, 9, 1], [0], [[3, -7]], [3], 1)
    got, _ = call_accept(be, s)
    assert got.path.tolist() == [0, 1, 3, -1, -1, -1] and got.tokens.tolist() == [8, 9, 1, -1, -1, -1]
    assert got.last.tolist() == [1]


@pytest.mark.parametrize("requests", [3, 100])
def test_accept_reports_what_does_not_fit(be, requests):
    s = list(accept_scene([20] * requests, 3, vocabulary=10 ** 6, held=[60] * requests))  # one row each is kept, a page comes back
    counts, kept, *_ = accept_by_hand(*s)
    assert kept[0] == 61
    s[6] = requests - 1  # the list cannot have held them
    got, f = call_accept(be, s)
    assert got.summary.tolist() == [1, requests, requests - 1, 61] and f.tolist() == s[5]
    assert got.lengths.tolist() == kept
    s[6] = len(s[5]) + 1  # nor so many entries
    got, f = call_accept(be, s)
    assert got.summary[0].item() == 1 and f.tolist() == s[5]
    s = list(accept_scene([20] * requests, 3, vocabulary=10 ** 6, held=[60] * requests))
    s[4] = [t[:1] for t in s[4]]
    got, f = call_accept(be, s)
    assert got.summary[0].item() == 2 and f.tolist() == s[5]
    s = list(accept_scene([20] * requests, 3, vocabulary=10 ** 6, held=[60] * requests))
    s[3] = [-1] + s[3][1:]  # holds fewer rows than it adds
    got, _ = call_accept(be, s)
    assert got.summary[0].item() == 8 and got.counts[0].item() == 0 and got.lengths[0].item() == 19
    assert got.path[:20].tolist() == [-1] * 20


def test_accept_after_a_declined_plan_keeps_what_was_held(be):
    held, added = ints([10, 64]), ints([5, 3])
    tables, free = ints([[0, -1], [1, -1]]), ints([])  # no free page
    plan = be.paged_plan(held, added, tables, free, 8)
    assert plan.summary[0].item() == 1
    got = be.paged_accept(ints([-1] * 8), ints([0] * 8), ints([0] * 8), plan.starts, plan.lengths, tables, free, plan)
    assert got.counts.tolist() == [0, 0] and got.lengths.tolist() == [10, 64] and got.summary.tolist() == [1, 0, 0, 64]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,layers,name", [(1, 1, "sizes"), (3, 5, "sizes"), (8, 2, "sixty_five"), (2, 130, "one_large")])
def test_keep_moves_the_confirmed_rows(be, heads, layers, name, dtype):
    sizes = {**ACCEPTS, "one_large": [256, 40]}[name]
    s = accept_scene(sizes, 5, vocabulary=2)
    trees, _, _, held, tables, _, _ = s
    _, kept, _, path, *_ = accept_by_hand(*s)
    pages = max(max(t) for t in tables) + 2
    g = gen(6)
    pools = [torch.randn(pages, 2, ROWS, heads, DIM, generator=g).to(dtype).cuda() for _ in range(layers)]
    want = [p.clone() for p in pools]
    row, moved = 0, 0
    for r, t in enumerate(trees):
        for k in range(kept[r] - held[r]):
            src, dst = held[r] + path[row + k], held[r] + k
            for w, p in zip(want, pools):
                w[tables[r][dst // ROWS], :, dst % ROWS] = p[tables[r][src // ROWS], :, src % ROWS]
            moved += src != dst
        row += len(t)
    assert moved
    status = ints([0])
    be.paged_keep(pools if layers > 1 else pools[0], ints(path), ints(starts_of(trees)),
                  ints([h + len(t) for h, t in zip(held, trees)]), ints(tables), status=status)
    assert status.item() == 0
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_keep_leaves_out_pages_that_are_none_and_paths_that_fall(be):
    pool = torch.randn(3, 2, ROWS, 2, DIM, device="cuda")
    before = pool.clone()
    for bad in (-1, 3, 2 ** 31 - 1):
        status = ints([0])
        be.paged_keep(pool, ints([0, 2, 3, -1]), ints([0, 4]), ints([66]), ints([[0, bad]]), status=status)  # own rows 62 to 65
        assert status.item() == 16
        want = before.clone()
        assert torch.equal(pool, want)  # 64 -> 63 and 65 -> 64 both touch the page
    be.paged_keep(pool, ints([1, 3, 2, -1]), ints([0, 4]), ints([14]), ints([[2]]))
    want = before.clone()
    want[2, :, 10], want[2, :, 11] = before[2, :, 11], before[2, :, 13]
    assert torch.equal(pool, want)
    be.paged_keep(pool, ints([0, 200, 5]), ints([0, 3]), ints([13]), ints([[1]]))  # past the request's rows
    be.paged_keep(pool, ints([2, 3]), ints([0, 2]), ints([1]), ints([[1]]))  # not held
    assert torch.equal(pool, want)


def test_keep_is_only_reached_by_distinct_pools(be):
    pool = torch.zeros(2, 2, ROWS, 2, DIM, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        be.paged_keep([pool, pool], ints([0]), ints([0, 1]), ints([1]), ints([[0]]))
    be.paged_keep([], ints([0]), ints([0, 1]), ints([1]), ints([[0]]))


def test_a_verification_step_captured_and_replayed(be):
    """Plan, tree, store, attention, accept and keep in one graph; each replay equals the calls by hand, and
    the pages taken and given back balance."""
    trees = some_trees([20, 7, 33, 0, 12], 30)
    requests, rows, kh, qh = len(trees), sum(map(len, trees)) + 6, 2, 8
    g = gen(31)
    parents = ints(sum(trees, []) + [-1] * 6)
    qkv = torch.randn(rows, (qh + 2 * kh) * DIM, generator=g).cuda()
    norms = [torch.zeros(DIM, dtype=BF16, device="cuda")] * 2
    table = torch.randn(2000, DIM, generator=g).cuda()
    tokens, chosen = (torch.randint(2, (rows,), generator=g).int().cuda() for _ in range(2))
    pools = [torch.zeros(40, 2, ROWS, kh, DIM, device="cuda") for _ in range(2)]
    added = ints([len(t) for t in trees])
    free = torch.randperm(40, generator=g).int().cuda()
    held, tables, head = ints([0] * requests), torch.full((requests, 9), -1, dtype=torch.int32, device="cuda"), ints([0, 0, 0, 0])

    class Before:
        summary = head

    def step():
        plan = be.paged_plan(held, added, tables, free, rows, after=Before)
        t = be.paged_tree(parents, plan.starts, plan.lengths, 33)
        outs = []
        for pool in pools:
            q = be.paged_store(qkv, pool, plan.slots, t.positions, *norms, table)
            outs.append(be.paged_attention(q, pool, plan.starts, plan.lengths, tables, most_new=33, masks=t.masks))
        a = be.paged_accept(parents, tokens, chosen, plan.starts, plan.lengths, tables, free, plan)
        be.paged_keep(pools, a.path, plan.starts, plan.lengths, tables)
        held.copy_(a.lengths)
        head.copy_(a.summary)
        return outs + [a.path]

    def reset():
        held.zero_(), head.zero_(), tables.fill_(-1)
        free.copy_(order)
        for pool in pools:
            pool.zero_()

    order = free.clone()
    by_hand = []
    for _ in range(4):
        by_hand.append([t.clone() for t in step()] + [held.clone(), head.clone(), tables.clone()] + [p.clone() for p in pools])
    assert head[0].item() == 0 and head[2].item() == sum(pages_for(n) for n in held.tolist())
    used = [tables[r, i].item() for r, n in enumerate(held.tolist()) for i in range(pages_for(n))]
    assert len(set(used)) == len(used) and not set(used) & set(free[head[2].item():].tolist())
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    reset()
    for want in by_hand:
        graph.replay()
        for a, b in zip(outs + [held, head, tables] + pools, want):
            assert torch.equal(a, b)
    assert be.paged_status() == 0


def test_refusals(be):
    p, s, n = ints([-1, 0]), ints([0, 2]), ints([2])
    with pytest.raises(ValueError, match="256"):
        be.paged_tree(p, s, n, 257)
    with pytest.raises(ValueError, match="starts"):
        be.paged_tree(p, n, n, 2)
    with pytest.raises(ValueError, match="parents"):
        be.paged_tree(p.long(), s, n, 2)
    with pytest.raises(ValueError, match="out of range"):
        be.paged_tree(p, s, n, 2, base=-1)
    tables, free = ints([[0]]), ints([0])
    with pytest.raises(ValueError, match="chosen"):
        be.paged_accept(p, p, n, s, n, tables, free, ints([0, 0, 0, 0]))
    with pytest.raises(ValueError, match="after"):
        be.paged_accept(p, p, p, s, n, tables, free, free)
    with pytest.raises(ValueError, match="overlap"):
        be.paged_accept(p, p, p, s, n, tables, tables[0], ints([0, 0, 0, 0]))
    pool = torch.zeros(1, 2, ROWS, 1, DIM, device="cuda")
    with pytest.raises(ValueError, match="one shape"):
        be.paged_keep([pool, pool.bfloat16()], p, s, n, tables)
    q = torch.zeros(2, 1, DIM, device="cuda")
    for masks in (torch.zeros(2, 9, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, 0, dtype=torch.int32),
                  torch.zeros(2, 1)):
        with pytest.raises(ValueError, match="masks"):
            be.paged_attention(q, pool, s, n, tables, masks=masks.cuda())
    s2 = Scene([(3, 1)], 0, 8, 2, BF16)
    check(be.paged_attention(s2.q, s2.pool, s2.starts, s2.lengths, s2.tables), *s2.expected())


@pytest.mark.parametrize("args", [[], ["--bf16"], ["--requests", "70", "--steps", "6", "--prefix", "1100"]])
def test_example_decodes_with_drafts_as_row_by_row(args):
    """FP32 pools: rows in trees and alone differ by 1e-6 or so, the two likeliest tokens' scores by more. In BF16 a
    rounding may choose another token, and what follows is another text."""
    spec = importlib.util.spec_from_file_location("paged_trees", os.path.join(ROOT, "examples", "paged_trees.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    drafted, plain = module.main(args)
    for d, p in zip(drafted, plain, strict=True):
        assert len(d) <= len(p) and (d == p[:len(d)] or "--bf16" in args)
