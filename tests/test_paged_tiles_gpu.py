"""The attention tests on batches whose page tables have room for so many rows
that requests of more than 32 (row, head) pairs go to the tile kernels, which
short tables keep in the row kernel."""
import pytest
import torch

import test_paged_edges_gpu as edges
import test_paged_gpu as base
from paged_reference import Scene
from test_paged_edges_gpu import (test_infinite_values_that_are_seen_make_infinite_results,  # noqa: F401
                                  test_rows_all_of_whose_scores_are_minus_infinity,
                                  test_rows_before_the_first_start_are_zero_and_reported, test_starts_that_decrease_leave_zeros)
from test_paged_gpu import (be, test_attention_head_layouts, test_attention_is_the_same_every_time,  # noqa: F401
                            test_attention_many_requests, test_attention_matches_its_formula,
                            test_attention_of_keys_that_are_no_numbers, test_attention_padding_and_unheld_rows_are_zero,
                            test_attention_reports_counts_outside_their_arrays, test_attention_reports_pages_outside_the_pool,
                            test_attention_rows_not_seen_never_matter, test_attention_scales, test_attention_sharp_scores,
                            test_attention_strided_rows_and_given_result, test_attention_values_fallen_out_of_the_window,
                            test_attention_windows)

pytestmark = pytest.mark.gpu

short_tables = base.attend


def attend(be, s, **more):
    tables, s.tables = s.tables, torch.nn.functional.pad(s.tables, (0, 2100), value=-7)
    try:
        return short_tables(be, s, **more)
    finally:
        s.tables = tables


@pytest.fixture(autouse=True)
def long_tables(monkeypatch):
    monkeypatch.setattr(base, "attend", attend)
    monkeypatch.setattr(edges, "attend", attend)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_tables_ask_for_the_tile_kernels(be, dtype):  # noqa: F811
    s = Scene([(70, 1), (0, 8)], 0, 8, 1, dtype)
    _, few = edges.launches_of(be, lambda: short_tables(be, s))
    _, more = edges.launches_of(be, lambda: attend(be, s))
    assert more == few + 1
