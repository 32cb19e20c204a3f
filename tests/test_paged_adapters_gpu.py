"""Low-rank adapters of a batch's requests (include/plamo_paged.h) against a 64-bit
statement: types, ranks, ragged rows, strides, refusals, streams and graphs."""
import pytest
import torch

from conftest import load_package
from paged_reference import check
from paged_tree_reference import adapters_expected

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def be():
    b = load_package().Backend(device=0)
    yield b
    b.close()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, new, ids, columns, outputs, rank, x_type=FP32, kind=FP32, adapters=None, spare=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.ids, self.starts = list(ids), [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        rows, count = self.starts[-1] + spare, adapters or max(ids, default=0) + 1
        self.x = torch.randn(rows, columns, generator=g).to(x_type).cuda()
        self.base = torch.randn(rows, outputs, generator=g).to(kind).cuda()
        self.a = (torch.randn(count, rank, columns, generator=g) * columns ** -0.5).to(BF16).cuda()
        self.b = torch.randn(count, outputs, rank, generator=g).to(BF16).cuda()
        self.scales = (torch.rand(count, generator=g) + 0.5).cuda()

    def expected(self):
        return adapters_expected(self.x, self.base, self.a, self.b, self.ids, self.starts, self.scales)

    def run(self, be, **more):
        return be.paged_adapters(self.x, self.base, self.a, self.b, ints(self.ids), ints(self.starts),
                                 **{"scales": self.scales, **more})


LAYOUTS = {
    "one": ([1], [0]),
    "decode": ([1] * 21, [i // 4 % 5 for i in range(21)]),
    "each_its_own": ([1] * 19, list(range(19))),
    "none": ([1, 3, 0, 20, 1], [-1, 0, 1, -1, 2]),
    "trees": ([17, 1, 33, 0, 8, 24], [3, 3, 0, 1, 0, 2]),
    "prompts": ([129, 300, 1, 64, 511], [0, 0, 1, 2, 1]),
    "gaps": ([0, 17, 33, 0, 400, 15, 16], [0, -1, 1, 2, 2, -1, 0]),
    "more_gaps": ([0, 17, 33, 0, 500, 15, 16], [0, -1, 1, 2, 2, -1, 0]),
}


@pytest.mark.parametrize("x_type,kind", [(FP32, FP32), (BF16, BF16), (FP32, BF16), (BF16, FP32)])
@pytest.mark.parametrize("columns,outputs,rank", [(512, 384, 16), (1000, 136, 8), (64, 1048, 40), (2560, 8, 64), (8, 200, 256)])
@pytest.mark.parametrize("name", sorted(LAYOUTS))
def test_adapters_match_their_formula(be, name, columns, outputs, rank, x_type, kind):
    c = Case(*LAYOUTS[name], columns, outputs, rank, x_type, kind, seed=rank)
    status = ints([0])
    check(c.run(be, status=status, most_new=max(LAYOUTS[name][0])), *c.expected(), name)
    assert status.item() == 0


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 48, 72, 96, 128, 136, 200, 256])
@pytest.mark.parametrize("kind", [FP32, BF16])
@pytest.mark.parametrize("new", [[1, 2, 5], [70, 200, 3], [333, 690, 12]])
def test_adapters_of_every_rank(be, rank, kind, new):
    c = Case(new, [0, 1, 0], 776, 520, rank, kind, kind, seed=rank)
    check(c.run(be), *c.expected(), f"rank {rank}")


@pytest.mark.parametrize("columns,outputs", [(4096, 5120), (16384, 4096), (4096, 32768), (5120, 10240)])
@pytest.mark.parametrize("kind", [FP32, BF16])
@pytest.mark.parametrize("new", [[1] * 9, [250, 190]])
def test_adapters_of_the_models_projections(be, columns, outputs, kind, new):
    c = Case(new, [i % 3 for i in range(len(new))], columns, outputs, 16, kind, kind, seed=1)
    check(c.run(be), *c.expected(), "projection")


@pytest.mark.parametrize("kind", [FP32, BF16])
@pytest.mark.parametrize("new", [[1, 4, 3], [540, 4, 3]])
def test_adapters_strides_and_places(be, kind, new):
    """Strided rows, a result of its own, the result in place; padding keeps base's."""
    c = Case(new, [0, -1, 1], 264, 392, 16, kind, kind, spare=5, seed=2)
    want, tol = c.expected()
    rows = c.x.shape[0]
    x, base = torch.full((rows, 280), float("nan"), dtype=kind, device="cuda"), torch.full((rows, 400), 3.0, dtype=kind, device="cuda")
    x[:, 8:272], base[:, 8:] = c.x, c.base
    plain = c.run(be)
    check(plain, want, tol, "plain")
    for r in (slice(new[0], new[0] + 4), slice(sum(new), rows)):  # no adapter, and padding
        assert torch.equal(plain[r], c.base[r])
    c.x, c.base = x[:, 8:272], base[:, 8:]
    out = torch.full((rows + 2, 408), 7.0, dtype=kind, device="cuda")
    got = c.run(be, out=out[1:-1, 8:400])
    assert torch.equal(got, plain) and (out[:, :8] == 7).all() and (out[:, 400:] == 7).all()
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    in_place = c.run(be, out=c.base)
    assert torch.equal(in_place, plain) and (base[:, :8] == 3).all()


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 170, 400, 1]])
def test_adapters_of_others_never_matter(be, new):
    """Adapters and rows that hold no numbers reach their own requests only."""
    c = Case(new, [0, 1, 2, 0], 256, 136, 24, seed=3)
    want, tol = c.expected()
    c.a[1], c.b[1], c.scales[1] = float("nan"), float("inf"), float("nan")
    c.x[c.starts[2]:c.starts[3]] = float("inf")
    got = c.run(be)
    for r in (0, 3):
        rows = slice(c.starts[r], c.starts[r + 1])
        check(got[rows], want[rows], tol[rows], f"request {r}")
    assert not torch.isfinite(got[c.starts[1]:c.starts[3]]).any()


@pytest.mark.parametrize("new", [1, 500, 600])
@pytest.mark.parametrize("kind", [FP32, BF16])
def test_adapters_of_infinite_rows(be, kind, new):
    """One infinite entry times weights of one sign is infinite, not undefined."""
    c = Case([new], [0], 64, 16, 8, kind, kind, seed=4)
    c.a, c.b = c.a.abs() + 0.1, c.b.abs() + 0.1
    c.x[new // 2, 5] = float("inf")
    got = c.run(be).float()
    assert (got[new // 2] == float("inf")).all()
    assert torch.isfinite(got[:new // 2]).all() and torch.isfinite(got[new // 2 + 1:]).all()


def test_adapters_without_scales_requests_or_adapters(be):
    c = Case([2, 590], [1, 0], 64, 72, 16, seed=5)
    ones, c.scales = c.scales, None
    check(c.run(be), *c.expected(), "no scales")
    c.scales = ones
    empty = be.paged_adapters(c.x, c.base, c.a, c.b, ints([]), ints([0]))
    assert torch.equal(empty, c.base)
    none = be.paged_adapters(c.x, c.base, c.a[:0], c.b[:0], ints([-1, -1]), ints(c.starts))
    assert torch.equal(none, c.base)
    assert be.paged_adapters(c.x[:0], c.base[:0], c.a, c.b, ints([0]), ints([0, 0])).shape == (0, 72)
    assert be.paged_status() == 0


@pytest.mark.parametrize("new", [[2, 3, 1], [2, 500, 1]])
@pytest.mark.parametrize("bad", [2, -2, 2 ** 31 - 1, -2 ** 31])
def test_adapters_report_ids_that_are_none(be, bad, new):
    c = Case(new, [0, -1, 1], 64, 72, 16, adapters=2, seed=6)
    want, tol = c.expected()
    c.ids[1] = bad
    status = ints([0])
    check(c.run(be, status=status), want, tol, "bad id")
    assert status.item() == 256


@pytest.mark.parametrize("rows", [20, 200, 300])
@pytest.mark.parametrize("starts", [[0, 50, 20, 70], [-9, 10, 20, 10 ** 9], [5, 10, 20, 30], [2 ** 31 - 1, -2 ** 31, 7, 9]])
def test_adapters_of_starts_outside_the_batch_stay_in_bounds(be, starts, rows):
    c = Case([rows, 30, rows], [0, 1, 0], 64, 72, 16, seed=7)
    out = torch.full((2 * rows + 32, 72), 7.0, device="cuda")
    c.starts = starts
    c.run(be, out=out[1:-1])
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[-1] == 7).all()


@pytest.mark.parametrize("new", [[1, 1, 6], [229, 3, 200], [229, 3, 330]])
def test_adapters_are_the_same_every_time_captured_and_on_another_stream(be, new):
    c = Case(new, [0, 1, 0], 1024, 264, 32, seed=8)
    first = c.run(be)
    assert all(torch.equal(c.run(be), first) for _ in range(3))
    ids, starts = ints(c.ids), ints(c.starts)
    stream, out = torch.cuda.Stream(), torch.zeros_like(first)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        be.paged_adapters(c.x, c.base, c.a, c.b, ids, starts, scales=c.scales, out=out)
    stream.synchronize()
    assert torch.equal(out, first)
    graph, captured = torch.cuda.CUDAGraph(), torch.zeros_like(first)
    with torch.cuda.graph(graph):
        be.paged_adapters(c.x, c.base, c.a, c.b, ids, starts, scales=c.scales, out=captured)
    for _ in range(2):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, first)


def test_refusals(be):
    c = Case([2], [0], 64, 72, 16)
    good = dict(x=c.x, base=c.base, a=c.a, b=c.b, ids=ints([0]), starts=ints([0, 2]))

    def call(match, **change):
        with pytest.raises(ValueError, match=match):
            be.paged_adapters(**{**good, **change})

    call("rank", a=c.a[:, :15].contiguous(), b=c.b[:, :, :15].contiguous())
    call("rank", a=torch.zeros(1, 264, 64, dtype=BF16, device="cuda"), b=torch.zeros(1, 72, 264, dtype=BF16, device="cuda"))
    call("multiples of 8", x=c.x[:, :60].contiguous(), a=c.a[:, :, :60].contiguous())
    call("multiples of 8", base=c.base[:, :70].contiguous(), b=c.b[:, :70].contiguous())
    call("outputs|adapters", b=c.b[:, :64].contiguous())
    call("rows", base=c.base[:1])
    call("ids", ids=torch.zeros(1, device="cuda"))
    call("starts", starts=ints([0]))
    call("scales", scales=torch.ones(2, device="cuda"))
    call("BF16 or FP32", x=c.x.half())
    call("BF16", a=c.a.float())
    call("out", out=c.base.bfloat16())
    call("16-byte", x=torch.zeros(2, 66, device="cuda")[:, 1:65])
    wide = torch.zeros(3, 144, device="cuda")
    call("out may be base", base=wide[:2, :72], out=wide[:2, 8:80])
    call("out may be base", base=wide[:2, :72], out=wide[1:, :72])
    call("out may be base", x=wide[:2, 72:136], out=wide[:2, :80][:, 8:])
    be.paged_adapters(**{**good, "base": wide[:2, :72], "out": wide[:2, 72:]})  # beside one another


@pytest.mark.parametrize("rows,rank", [(20_000, 8), (700, 64), (2_000, 128), (60, 256)])
def test_long_sums_of_one_sign_lose_nothing(be, rows, rank):
    """All terms positive, so that what is cut off sums adds up. Chains of 12 MMAs at most, cut by up to 2^-23 of the
    sum each, then FP32 additions: 4,096 columns by no fewer than 64, or ranks by 32, and up to 64 partial sums,
    a rounding of 2^-24 each. (One chain over the columns would be off by some 4e-5.)"""
    g = torch.Generator(device="cuda").manual_seed(3)
    columns, outputs = 4096, 16
    be.paged_status()
    x = torch.rand(rows, columns, generator=g, device="cuda")
    a = torch.rand(1, rank, columns, generator=g, device="cuda").to(torch.bfloat16)
    b = torch.rand(1, outputs, rank, generator=g, device="cuda").to(torch.bfloat16)
    starts, ids = torch.tensor([0, rows], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    got = be.paged_adapters(x, torch.zeros(rows, outputs, device="cuda"), a, b, ids, starts)
    want = x.double() @ a[0].double().T @ b[0].double().T
    bound = 12 * 2 ** -23 + (64 + 64) * 2 ** -24 + 12 * 2 ** -23 + 8 * 2 ** -24
    assert ((got.double() - want).abs() / want).max().item() <= bound
    assert be.paged_status() == 0


@pytest.mark.parametrize("each", [1, 40, 50])
def test_starts_that_decrease_are_reported(be, each):
    """By the kernels of few rows and of many; rows before the fault are those of their request."""
    requests, rank = 12, 16
    rows = requests * each
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, 64, generator=g, device="cuda")
    a, b = (torch.randn(1, *shape, generator=g, device="cuda").to(torch.bfloat16) for shape in ((rank, 64), (24, rank)))
    ids = torch.zeros(requests, dtype=torch.int32, device="cuda")
    base = torch.zeros(rows, 24, device="cuda")
    good = [each * r for r in range(requests + 1)]
    be.paged_status()
    for wrong in (good[:3] + [good[3] - 2 * each] + good[4:], good[:-1] + [rows + 1]):
        be.paged_adapters(x, base, a, b, ids, torch.tensor(wrong, dtype=torch.int32, device="cuda"))
        assert be.paged_status() == 4
    be.paged_adapters(x, base, a, b, ids, torch.tensor(good, dtype=torch.int32, device="cuda"))
    assert be.paged_status() == 0


@pytest.mark.parametrize("new", [1, 60])
def test_calls_on_two_streams_at_once(be, new):
    """Each has a workspace of its own."""
    g = torch.Generator(device="cuda").manual_seed(9)
    requests, columns, outputs, rank = 24, 1024, 512, 32
    starts = torch.arange(requests + 1, dtype=torch.int32, device="cuda") * new
    ids = torch.arange(requests, dtype=torch.int32, device="cuda") % 3
    sides = []
    for _ in range(2):
        x, base = (torch.randn(requests * new, n, generator=g, device="cuda") for n in (columns, outputs))
        a, b = (torch.randn(3, *shape, generator=g, device="cuda").to(torch.bfloat16) for shape in ((rank, columns), (outputs, rank)))
        sides.append((x, base, a, b, ids, starts))
    want = [be.paged_adapters(*side) for side in sides]
    streams, got = [torch.cuda.Stream() for _ in sides], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(be.paged_adapters(*sides[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
