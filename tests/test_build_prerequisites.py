"""The library is rebuilt when any file that its sources include has changed."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG_DIR, ROOT


def included():
    found, todo = set(), [os.path.join(PKG_DIR, "csrc", n) for n in os.listdir(os.path.join(PKG_DIR, "csrc"))]
    while todo:
        path = todo.pop()
        for name in re.findall(r'^#include "([^"]+)"', open(path).read(), flags=re.M):
            for folder in (os.path.dirname(path), os.path.join(ROOT, "include")):
                at = os.path.normpath(os.path.join(folder, name))
                if os.path.exists(at) and at not in found:
                    found.add(at)
                    todo.append(at)
    return sorted(found)


@pytest.mark.skipif(not shutil.which("make"), reason="needs make")
def test_a_changed_header_rebuilds_the_library():
    files = included()
    assert len(files) > 10
    lib = os.path.join(PKG_DIR, "lib", "libplamo_cuda.so")
    for path in files:
        # -o: everything else counts as old, so that only `path` (-W: as if changed now) can ask for a build.
        others = [x for f in files + [os.path.join(PKG_DIR, "csrc", n) for n in os.listdir(os.path.join(PKG_DIR, "csrc"))]
                  if f != path for x in ("-o", f)]
        run = subprocess.run(["make", "-n", "-C", PKG_DIR, lib, "-W", path, *others], capture_output=True, text=True, check=True)
        assert "-shared" in run.stdout, f"{os.path.relpath(path, ROOT)} is no prerequisite"
