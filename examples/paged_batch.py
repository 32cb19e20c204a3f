#!/usr/bin/env python3
"""Serving a batch behind a shared prefix: the attention blocks of a small
model, prompts and decode steps, on the paged operators.

    python examples/paged_batch.py [--requests 6] [--steps 20] [--layers 2] [--fp32]

Each layer projects the batch's rows (the library's BF16 projection), stores
queries, keys and values (paged_store), attends over the prefix that every
request shares and over its own rows (paged_attention), projects back and adds
the result to the rows. One plan (paged_plan) places a step's rows for all
layers: their pools have the same pages. Odd layers look back over a sliding
window, as the model's sliding layers do.

Weights and inputs are synthetic. At the end the same requests run alone, one
after another, each with the prefix among its own pages, and the two results
are compared.
"""
import argparse
import importlib.util
import os
import sys

import numpy as np
import torch

ROWS, DIM = 64, 128


def load_package():
    if "plamo_b200" in sys.modules:
        return sys.modules["plamo_b200"]
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "plamo-3-translate.c_b200")
    spec = importlib.util.spec_from_file_location("plamo_b200", os.path.join(root, "__init__.py"),
                                                  submodule_search_locations=[root])
    module = importlib.util.module_from_spec(spec)
    sys.modules["plamo_b200"] = module
    spec.loader.exec_module(module)
    return module


class Model:
    """Attention blocks with synthetic weights, and their pools."""

    def __init__(self, backend, layers, hidden, query_heads, kv_heads, window, cache, positions, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.backend, self.hidden, self.qh, self.kh, self.cache = backend, hidden, query_heads, kv_heads, cache
        width = (query_heads + 2 * kv_heads) * DIM

        def weight(*shape):
            return (torch.randn(*shape, generator=g) * 0.02).to(torch.bfloat16).cuda()

        self.layers = [dict(qkv=weight(width, hidden), out=weight(hidden, query_heads * DIM),
                            norms=[weight(DIM), weight(DIM)], window=window if i % 2 else 0) for i in range(layers)]
        half = DIM // 2
        angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(half) / half)
        self.table = torch.tensor(np.concatenate([np.cos(angle), np.sin(angle)], 1), dtype=torch.float32).cuda()

    def pools(self, pages):
        return [torch.zeros(pages, 2, ROWS, self.kh, DIM, dtype=self.cache, device="cuda") for _ in self.layers]

    def project(self, x, w):
        """x . w^T through the library: FP32 rows, BF16 weights."""
        y = torch.empty(x.shape[0], w.shape[0], device="cuda")
        torch.cuda.current_stream().synchronize()  # the projection runs on the backend's own stream
        rc = self.backend.lib.plamo_cuda_gemm_device(self.backend.ctx, x.data_ptr(), x.shape[1], w.data_ptr(), y.data_ptr(),
                                                     w.shape[0], x.shape[0], w.shape[0], x.shape[1])
        if rc != 1:
            raise RuntimeError(self.backend.info().note.decode())
        return y

    def step(self, x, pools, plan, tables, prefix_pages, prefix_rows, most_new):
        """The batch's rows [rows, hidden] through every layer, at most `most_new` of them one request's."""
        for layer, pool in zip(self.layers, pools):
            qkv = self.project(x, layer["qkv"])
            q = self.backend.paged_store(qkv, pool, plan.slots, plan.positions, *layer["norms"], self.table)
            a = self.backend.paged_attention(q, pool, plan.starts, plan.lengths, tables, prefix_pages=prefix_pages,
                                             prefix_rows=prefix_rows, window=layer["window"], most_new=most_new)
            x = x + self.project(a.float().reshape(x.shape[0], -1), layer["out"])
        return x


def serve(model, prefix, prompts, steps, shared):
    """Each request's prompt rows, then `steps` more rows fed from its last one.
    shared: the prefix once, before all; else ahead of each prompt."""
    requests = len(prompts)
    if not shared:
        prompts = [torch.cat([prefix, p]) for p in prompts]
    most = max(p.shape[0] for p in prompts) + steps
    per_request, prefix_count = -(-most // ROWS) + 1, -(-prefix.shape[0] // ROWS) if shared else 0
    pools = model.pools(prefix_count + requests * per_request)
    ints = dict(dtype=torch.int32, device="cuda")
    prefix_pages, prefix_rows = None, 0
    if shared:  # the prefix is a request of its own whose pages become the prefix's table
        table = torch.full((1, prefix_count), -1, **ints)
        plan = model.backend.paged_plan(torch.zeros(1, **ints), torch.full((1,), prefix.shape[0], **ints), table,
                                        torch.arange(prefix_count, **ints), prefix.shape[0])
        model.step(prefix, pools, plan, table, None, 0, prefix.shape[0])
        prefix_pages, prefix_rows = table[0].contiguous(), prefix.shape[0]
    free = prefix_count + torch.randperm(requests * per_request, generator=torch.Generator().manual_seed(1)).int().cuda()
    tables = torch.full((requests, per_request), -1, **ints)
    held = torch.zeros(requests, **ints)
    added = torch.tensor([p.shape[0] for p in prompts], **ints)
    x, plan, outputs = torch.cat(prompts), None, []
    for step in range(steps + 1):
        plan = model.backend.paged_plan(held, added, tables, free, x.shape[0], base=prefix_rows, after=plan)
        y = model.step(x, pools, plan, tables, prefix_pages, prefix_rows, 1 if step else max(p.shape[0] for p in prompts))
        last = (plan.starts[1:] - 1).long()
        outputs.append(y[last])
        x = torch.nn.functional.normalize(y[last], dim=1) * model.hidden ** 0.5  # the next row of each request
        held, added = plan.lengths, torch.ones(requests, **ints)
        if plan.summary[0].item():
            raise RuntimeError(f"plan declined: status {plan.summary[0].item()}")
    if status := model.backend.paged_status():
        raise RuntimeError(f"the layers' calls report status {status}")
    return torch.stack(outputs)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prefix", type=int, default=150)
    ap.add_argument("--fp32", action="store_true", help="FP32 pools (BF16 otherwise)")
    a = ap.parse_args(argv)
    backend = load_package().Backend(device=0)
    try:
        hidden = 512
        lengths = [5 + 31 * i % 90 for i in range(a.requests)]
        model = Model(backend, a.layers, hidden, 8, 2, 100, torch.float32 if a.fp32 else torch.bfloat16,
                      a.prefix + max(lengths) + a.steps)
        g = torch.Generator().manual_seed(2)
        prefix = torch.randn(a.prefix, hidden, generator=g).cuda()
        prompts = [torch.randn(n, hidden, generator=g).cuda() for n in lengths]
        together = serve(model, prefix, prompts, a.steps, shared=True)
        alone = torch.cat([serve(model, prefix, [p], a.steps, shared=False) for p in prompts], 1)
        off = ((together - alone).norm() / alone.norm()).item()
        print(f"{a.requests} requests behind {a.prefix} shared rows, {a.steps} steps: "
              f"relative difference from each request alone {off:.2g}")
        return off
    finally:
        backend.close()


if __name__ == "__main__":
    main()
