"""The operators of draft trees and adapters without a GPU: record layouts, exports,
checks of torch arguments."""
import ctypes
import os
import subprocess
import types

import pytest
import torch

from conftest import ROOT, load_package
from test_paged_args import BF16, DIM, FP32, INT, NoCalls, On, ROWS


def test_records_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes records, checked by a C compiler."""
    abi = load_package()._abi
    lines = ['#include "plamo_paged.h"', "#include <stddef.h>"]
    for record, name in ((abi.PagedTreeArgs, "tree"), (abi.PagedTreeAttentionArgs, "tree_attention"), (abi.PagedAcceptArgs, "accept"),
                         (abi.PagedKeepArgs, "keep"), (abi.PagedAdaptersArgs, "adapters")):
        c = f"struct plamo_paged_{name}_args"
        lines.append(f'_Static_assert(sizeof({c}) == {ctypes.sizeof(record)}, "{name}");')
        for field, _ in record._fields_:
            lines.append(f'_Static_assert(offsetof({c}, {field}) == {getattr(record, field).offset}, "{name} {field}");')
    lines.append(f'_Static_assert(PLAMO_PAGED_TREE_ROWS == {abi.PAGED_TREE_ROWS}, "tree rows");')
    source = tmp_path / "records.c"
    source.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(source)],
                   check=True)


def test_entries_decline_without_a_context():
    lib, abi = load_package().load(), load_package()._abi
    for name, record in (("tree", abi.PagedTreeArgs), ("tree_attention", abi.PagedTreeAttentionArgs),
                         ("tree_attention_workspace", abi.PagedTreeAttentionArgs), ("accept", abi.PagedAcceptArgs),
                         ("keep", abi.PagedKeepArgs), ("adapters", abi.PagedAdaptersArgs),
                         ("adapters_workspace", abi.PagedAdaptersArgs)):
        assert getattr(lib, f"plamo_paged_{name}")(None, ctypes.byref(record())) == 0


@pytest.mark.parametrize("ours,theirs", [(0, 1), (1, 0), (3, 2)])
def test_tensors_of_another_gpu_are_refused(ours, theirs, monkeypatch):
    paged = load_package().paged
    monkeypatch.setattr(paged, "_stream", lambda torch, device: pytest.fail("a stream was asked for"))
    backend = types.SimpleNamespace(device=ours, lib=NoCalls(), ctx=None)

    def on(shape, dtype, index=theirs):
        return On(torch.zeros(shape, dtype=dtype), index)

    ids, starts, tables, summary = on(2, INT), on(3, INT), on((2, 3), INT), on(4, INT)
    pool = on((2, 2, ROWS, 2, DIM), BF16)
    calls = [lambda: paged.tree(backend, ids, starts, ids, 2),
             lambda: paged.accept(backend, ids, ids, ids, starts, ids, tables, ids, summary),
             lambda: paged.keep(backend, [pool], ids, starts, ids, tables),
             lambda: paged.adapters(backend, on((2, 8), FP32), on((2, 8), FP32), on((1, 8, 8), BF16), on((1, 8, 8), BF16), ids, starts)]
    for call in calls:
        with pytest.raises(ValueError, match=f"GPU,? {ours}"):
            call()
    # and the later arguments each
    here = lambda shape, dtype: on(shape, dtype, ours)  # noqa: E731
    mixed = [lambda: paged.tree(backend, here(2, INT), starts, here(2, INT), 2),
             lambda: paged.tree(backend, here(2, INT), here(3, INT), ids, 2),
             lambda: paged.accept(backend, here(2, INT), ids, here(2, INT), here(3, INT), here(2, INT), here((2, 3), INT), here(2, INT), here(4, INT)),
             lambda: paged.accept(backend, here(2, INT), here(2, INT), here(2, INT), here(3, INT), here(2, INT), here((2, 3), INT), here(2, INT), summary),
             lambda: paged.keep(backend, [here((2, 2, ROWS, 2, DIM), BF16), pool], here(2, INT), here(3, INT), here(2, INT), here((2, 3), INT)),
             lambda: paged.adapters(backend, here((2, 8), FP32), here((2, 8), FP32), here((1, 8, 8), BF16), on((1, 8, 8), BF16), here(2, INT), here(3, INT)),
             lambda: paged.adapters(backend, here((2, 8), FP32), here((2, 8), FP32), here((1, 8, 8), BF16), here((1, 8, 8), BF16), here(2, INT), here(3, INT),
                                    scales=on(1, FP32))]
    for call in mixed:
        with pytest.raises(ValueError, match=f"GPU,? {ours}"):
            call()
