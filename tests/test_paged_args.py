"""The paged operators' checks of torch arguments that need no GPU: tensors that
claim to be on one, and a library that must not be called."""
import types

import pytest
import torch

from conftest import load_package

ROWS, DIM = 64, 128
BF16, FP32, INT = torch.bfloat16, torch.float32, torch.int32


class On:
    """A CPU tensor that says that it is on GPU `index`."""

    def __init__(self, tensor, index):
        self.tensor, self.index = tensor, index

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.tensor, name)


class NoCalls:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.mark.parametrize("ours,theirs", [(0, 1), (1, 0), (3, 2)])
def test_tensors_of_another_gpu_are_refused(ours, theirs, monkeypatch):
    paged = load_package().paged
    monkeypatch.setattr(paged, "_stream", lambda torch, device: pytest.fail("a stream was asked for"))
    backend = types.SimpleNamespace(device=ours, lib=NoCalls(), ctx=None)

    def on(shape, dtype):
        return On(torch.zeros(shape, dtype=dtype), theirs)

    ids, tables = on(2, INT), on((2, 3), INT)
    pool, norm = on((2, 2, ROWS, 2, DIM), BF16), on(DIM, BF16)
    calls = [lambda: paged.plan(backend, ids, ids, tables, ids, 3),
             lambda: paged.store(backend, on((2, 6 * DIM), FP32), pool, ids, ids, norm, norm, on((4, DIM), FP32)),
             lambda: paged.attention(backend, on((2, 8, DIM), BF16), pool, on(3, INT), ids, tables)]
    for call in calls:
        with pytest.raises(ValueError, match=f"GPU, {ours}"):
            call()


def test_a_backend_knows_its_gpu(monkeypatch):
    pkg = load_package()
    lib = types.SimpleNamespace(plamo_cuda_open=lambda cfg, err, cap: 1, plamo_cuda_close=lambda ctx: None)
    monkeypatch.setattr(pkg._abi, "load", lambda: lib)
    assert pkg.Backend(device=3).device == 3
