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
