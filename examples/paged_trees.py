#!/usr/bin/env python3
"""Drafted tokens verified in trees, each request with its own adapter: greedy
decoding of a small model on the paged operators.

    python examples/paged_trees.py [--requests 6] [--steps 12] [--layers 2] [--bf16]

A drafter guesses from a token alone the two likeliest next ones, after each of
them two more, and after those one: a tree of 1 + 2 + 4 + 4 rows. One step of the model takes the last
token and its tree for every request: a plan (paged_plan), the rows' positions
and masks (paged_tree), in each layer the projections with the requests'
adapters added (paged_adapters), the rows stored (paged_store) and attention over the
prefix, the request's own rows and the row's ancestors (paged_attention with
masks). The path that the model's choices confirm (paged_accept) moves together in
every pool (paged_keep), and the next step goes on after it. Nothing is read on the host
before the end.

Weights and inputs are synthetic. At the end the same requests run row by row,
without drafts, and the tokens are compared.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from paged_batch import ROWS, Model, load_package  # noqa: E402

# Rows of a request's tree: the last token, two after it, two after each of these, one after each of those.
PARENTS = [-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6]
CHOICE = [0, 0, 1, 0, 1, 0, 1, 0, 0, 0, 0]  # which of the drafter's guesses after its parent
LEVELS = [(1, 3), (3, 7), (7, 11)]


class TokenModel(Model):
    """The attention blocks behind an embedding, with adapters on their projections and a head."""

    def __init__(self, backend, layers, hidden, query_heads, kv_heads, window, cache, positions, vocabulary, adapters, rank):
        super().__init__(backend, layers, hidden, query_heads, kv_heads, window, cache, positions)
        g = torch.Generator().manual_seed(7)

        def weight(*shape, scale):
            return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).cuda()

        self.embedding = torch.randn(vocabulary, hidden, generator=g).cuda() * 0.3
        self.head = weight(vocabulary, hidden, scale=hidden ** -0.5)
        for layer in self.layers:
            for name in ("qkv", "out"):
                outputs, columns = layer[name].shape
                layer[name + "_a"] = weight(adapters, rank, columns, scale=columns ** -0.5)
                layer[name + "_b"] = weight(adapters, outputs, rank, scale=0.1 * rank ** -0.5)

    def adapted(self, x, layer, name, ids, starts, most_new):
        y = self.project(x, layer[name])
        return self.backend.paged_adapters(x, y, layer[name + "_a"], layer[name + "_b"], ids, starts, out=y, most_new=most_new)

    def choices(self, tokens, positions, masks, pools, plan, tables, prefix_pages, prefix_rows, ids, most_new):
        """The token that the model chooses after each row; masks: None where every row sees those before it."""
        x = self.embedding[tokens.long()]
        for layer, pool in zip(self.layers, pools):
            qkv = self.adapted(x, layer, "qkv", ids, plan.starts, most_new)
            q = self.backend.paged_store(qkv, pool, plan.slots, positions, *layer["norms"], self.table)
            a = self.backend.paged_attention(q, pool, plan.starts, plan.lengths, tables, prefix_pages=prefix_pages,
                                             prefix_rows=prefix_rows, window=layer["window"], most_new=most_new, masks=masks)
            x = x + self.adapted(a.float().reshape(x.shape[0], -1), layer, "out", ids, plan.starts, most_new)
        return self.project(x, self.head).argmax(1).int()

    def guesses(self):
        """[vocabulary, 2]: the likeliest tokens after each, by its embedding alone."""
        return self.project(self.embedding, self.head).topk(2, 1).indices.int()


def serve(model, prefix, prompts, ids, steps, drafts):
    """`steps` steps after the prompts; each request's tokens. drafts: whether in trees."""
    requests, longest, backend = len(prompts), max(p.numel() for p in prompts), model.backend
    tree = PARENTS if drafts else [-1]
    most = longest + steps * len(LEVELS) + steps + len(tree)
    per_request, prefix_count = -(-most // ROWS) + 1, -(-prefix.numel() // ROWS)
    pools = model.pools(prefix_count + requests * per_request)
    ints = dict(dtype=torch.int32, device="cuda")
    # The prefix is a request of its own whose pages become the prefix's table.
    table = torch.full((1, prefix_count), -1, **ints)
    plan = backend.paged_plan(torch.zeros(1, **ints), torch.full((1,), prefix.numel(), **ints), table,
                              torch.arange(prefix_count, **ints), prefix.numel())
    model.choices(prefix, plan.positions, None, pools, plan, table, None, 0, torch.full((1,), -1, **ints), prefix.numel())
    shared = dict(prefix_pages=table[0].contiguous(), prefix_rows=prefix.numel(), ids=ids)
    free = prefix_count + torch.randperm(requests * per_request, generator=torch.Generator().manual_seed(1)).int().cuda()
    tables = torch.full((requests, per_request), -1, **ints)
    added = torch.tensor([p.numel() for p in prompts], **ints)
    plan = backend.paged_plan(torch.zeros(requests, **ints), added, tables, free, sum(p.numel() for p in prompts), base=prefix.numel())
    chosen = model.choices(torch.cat(prompts), plan.positions, None, pools, plan, tables, most_new=longest, **shared)
    last, held, before = chosen[(plan.starts[1:] - 1).long()], plan.lengths, plan
    summaries, out = [plan.summary], [(last[:, None], torch.ones(requests, **ints))]
    guesses = model.guesses()
    parents, added = torch.tensor(tree * requests, **ints), torch.full((requests,), len(tree), **ints)
    above, choice = torch.tensor(tree, device="cuda"), torch.tensor(CHOICE[:len(tree)], device="cuda")
    for _ in range(steps):
        tokens = torch.empty(requests, len(tree), **ints)
        tokens[:, 0] = last
        for begin, end in LEVELS if drafts else []:
            tokens[:, begin:end] = guesses[tokens[:, above[begin:end]].long(), choice[begin:end]]
        tokens = tokens.reshape(-1)
        plan = backend.paged_plan(held, added, tables, free, tokens.numel(), base=prefix.numel(), after=before)
        rows = backend.paged_tree(parents, plan.starts, plan.lengths, len(tree), base=prefix.numel())
        chosen = model.choices(tokens, rows.positions, rows.masks, pools, plan, tables, most_new=len(tree), **shared)
        before = backend.paged_accept(parents, tokens, chosen, plan.starts, plan.lengths, tables, free, plan)
        backend.paged_keep(pools, before.path, plan.starts, plan.lengths, tables)
        held, last = before.lengths, before.last
        summaries.append(before.summary)
        out.append((before.tokens.reshape(requests, -1), before.counts))
    if any(s[0].item() for s in summaries):
        raise RuntimeError(f"a step declined: status {[s[0].item() for s in summaries]}")
    if status := backend.paged_status():
        raise RuntimeError(f"the layers' calls report status {status}")
    out = [(tokens.tolist(), counts.tolist()) for tokens, counts in out]
    return [sum((tokens[r][:counts[r]] for tokens, counts in out), []) for r in range(requests)]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--steps", type=int, default=12)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prefix", type=int, default=150)
    ap.add_argument("--bf16", action="store_true", help="BF16 pools (FP32 otherwise)")
    a = ap.parse_args(argv)
    backend = load_package().Backend(device=0)
    try:
        vocabulary, lengths = 512, [5 + 31 * i % 90 for i in range(a.requests)]
        model = TokenModel(backend, a.layers, 512, 8, 2, 100, torch.bfloat16 if a.bf16 else torch.float32,
                           a.prefix + max(lengths) + a.steps * (1 + len(LEVELS)) + len(PARENTS), vocabulary, 4, 16)
        g = torch.Generator().manual_seed(2)
        prefix = torch.randint(vocabulary, (a.prefix,), generator=g).int().cuda()
        prompts = [torch.randint(vocabulary, (n,), generator=g).int().cuda() for n in lengths]
        ids = torch.tensor([i % 5 - 1 for i in range(a.requests)], dtype=torch.int32, device="cuda")  # every fifth has none
        drafted = serve(model, prefix, prompts, ids, a.steps, True)
        plain = serve(model, prefix, prompts, ids, max(map(len, drafted)) - 1, False)
        same = sum(d == p[:len(d)] for d, p in zip(drafted, plain))
        print(f"{a.requests} requests behind {a.prefix} shared rows, {a.steps} steps: {sum(map(len, drafted)) / a.requests / (a.steps + 1):.2f} "
              f"tokens a step; {same} of {a.requests} have the tokens of decoding row by row")
        return drafted, plain
    finally:
        backend.close()


if __name__ == "__main__":
    main()
