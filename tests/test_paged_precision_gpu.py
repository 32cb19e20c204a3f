"""What BF16 pools' attention loses against 64 bits beyond its results' own
rounding (include/plamo_paged.h): where a row's weight lies on few keys, a weight's
rounding shows in every dimension."""
import copy

import pytest
import torch

from conftest import load_package
from paged_reference import Scene

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def be():
    b = load_package().Backend(device=0)
    yield b
    b.close()


def beyond_rounding(be, s):
    """(relative L2 of the result, its bound).

    A result is y = o + d rounded to BF16, with |d| <= (2 (e^E - 1) + 2^-17) A
    from scores, exponentials and FP32 sums (Scene.expected), and 2^-15 A from
    the softmax weights, carried in two BF16 terms: the second is at most 2^-7 of
    the weight, its own rounding 2^-8 of that. The last rounding is not
    correlated with d, so the squares add; 2 % covers the chance correlation
    over the thousands of elements here.
    """
    wide, sizes = copy.copy(s), copy.copy(s)
    wide.dtype = sizes.dtype = torch.float32
    o, d = wide.expected()
    sizes.shared = [s.shared[0], s.shared[1].abs()]
    sizes.own = [[k, v.abs()] for k, v in s.own]
    a, _ = sizes.expected()
    rounding = o.to(BF16).double() - o
    got = be.paged_attention(s.q, s.pool, s.starts, s.lengths, s.tables, prefix_pages=s.prefix_pages, prefix_rows=s.prefix)
    bound = 1.02 * torch.sqrt(rounding.norm() ** 2 + (d + 2.0 ** -15 * a).norm() ** 2) / o.norm()
    return ((got.double().cpu() - o).norm() / o.norm()).item(), bound.item()


@pytest.mark.parametrize("requests,prefix,spread", [([(40, 200), (0, 130)], 300, 4.0), ([(40, 200), (0, 130)], 300, 2.0),
                                                    ([(0, 300)], 0, 1.0)])
def test_prompts_lose_only_their_results_rounding(be, requests, prefix, spread):
    off, bound = beyond_rounding(be, Scene(requests, prefix, 8, 2, BF16, seed=21, spread=spread))
    assert off <= bound, f"{off:.3e}, bound {bound:.3e}"


def test_a_shared_prefix_in_tiles_loses_only_the_results_rounding(be):
    s = Scene([(0, 1)] * 1200, 130, 16, 2, BF16, seed=22, spread=1.0)
    off, bound = beyond_rounding(be, s)
    assert off <= bound, f"{off:.3e}, bound {bound:.3e}"


@pytest.mark.parametrize("heads", [(8, 1), (16, 1)])
@pytest.mark.parametrize("prefix", [0, 7])
def test_decode_rows_lose_only_their_results_rounding(be, prefix, heads):
    s = Scene([(i * 7 % 30, 1) for i in range(150)], prefix, *heads, BF16, seed=23, spread=1.0)
    off, bound = beyond_rounding(be, s)
    assert off <= bound, f"{off:.3e}, bound {bound:.3e}"
