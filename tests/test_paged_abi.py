"""The paged operators' C interface: exports, record layouts, constants."""
import ctypes
import os
import re
import subprocess

from conftest import ROOT, load_package


def header():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "plamo_paged.h")).read(), flags=re.S)


def test_library_exports_the_paged_operators():
    pkg = load_package()
    pkg.load()
    names = sorted(set(re.findall(r"\b(plamo_paged_\w+)\s*\(", header())))
    assert sorted(pkg._abi.PAGED_SIGNATURES) == names
    out = subprocess.run(["nm", "-D", "--defined-only", pkg.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = set(re.findall(r"\sT\s(plamo_\w+)", out))
    assert not [n for n in names if n not in exported]


def test_records_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes records, checked by a C compiler."""
    abi = load_package()._abi
    lines = ['#include "plamo_paged.h"', "#include <stddef.h>"]
    for record, name in ((abi.PagedPlanArgs, "plan"), (abi.PagedStoreArgs, "store"), (abi.PagedAttentionArgs, "attention")):
        c = f"struct plamo_paged_{name}_args"
        lines.append(f'_Static_assert(sizeof({c}) == {ctypes.sizeof(record)}, "{name}");')
        for field, _ in record._fields_:
            lines.append(f'_Static_assert(offsetof({c}, {field}) == {getattr(record, field).offset}, "{name} {field}");')
    for name, value in (("ROWS", abi.PAGED_ROWS), ("DIM", abi.PAGED_DIM), ("BF16", abi.PAGED_BF16), ("FP32", abi.PAGED_FP32)):
        lines.append(f'_Static_assert(PLAMO_PAGED_{name} == {value}, "{name}");')
    source = tmp_path / "records.c"
    source.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(source)],
                   check=True)


def test_entries_decline_without_a_context():
    lib = load_package().load()
    abi = load_package()._abi
    assert lib.plamo_paged_plan(None, ctypes.byref(abi.PagedPlanArgs())) == 0
    assert lib.plamo_paged_store(None, ctypes.byref(abi.PagedStoreArgs())) == 0
    assert lib.plamo_paged_attention(None, ctypes.byref(abi.PagedAttentionArgs())) == 0
    assert lib.plamo_paged_attention_workspace(None, ctypes.byref(abi.PagedAttentionArgs())) == 0
