"""Operators of a paged batch step on torch tensors (include/plamo_paged.h).

Requests behind one shared prompt prefix keep their keys and values in a pool
of 64-row pages, [pages, 2, 64, kv_heads, 128] in BF16 or FP32. A step plans
its rows once (`plan`), then per layer stores the projection's rows (`store`)
and attends (`attention`). Calls are enqueued on torch's current stream and
return without waiting; tensors they allocate come from torch's allocator.
Wrong arguments raise ValueError. What only the GPU can see is reported as
PLAMO_PAGED_* bits, in the plan's summary or in a `status` tensor (one int32,
zeroed by the caller).
"""
import ctypes
from typing import NamedTuple

from . import _abi

ROWS, DIM = _abi.PAGED_ROWS, _abi.PAGED_DIM


class Plan(NamedTuple):
    """What a step's operators need of its rows (int32 tensors)."""
    lengths: object    # [requests] own rows after the step
    starts: object     # [requests + 1] first batch row of each request
    slots: object      # [rows] page * 64 + row in the page, -1 for padding
    positions: object  # [rows]
    summary: object    # [4] status bits, new rows, free-list entries used so far, longest length


def _torch():
    import torch
    return torch


def _stream(torch, device):
    return torch.cuda.current_stream(device).cuda_stream or 1  # 0 names the context's own stream there


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _ints(torch, t, shape, name):
    _need(t.dtype == torch.int32 and t.is_cuda and t.is_contiguous() and
          (shape is None or tuple(t.shape) == shape), f"{name}: a contiguous int32 tensor on the GPU"
          + (f" of shape {shape}" if shape else ""))


def _type(torch, t, name):
    if t.dtype == torch.bfloat16:
        return _abi.PAGED_BF16
    _need(t.dtype == torch.float32, f"{name}: BF16 or FP32")
    return _abi.PAGED_FP32


def _pool(torch, pool):
    _need(pool.dim() == 5 and tuple(pool.shape[1:3]) == (2, ROWS) and pool.shape[4] == DIM and pool.is_cuda and
          pool.is_contiguous(), f"pool: a contiguous [pages, 2, {ROWS}, kv_heads, {DIM}] tensor on the GPU")
    return _type(torch, pool, "pool"), pool.shape[0], pool.shape[3]


def _run(backend, call, args):
    rc = call(backend.ctx, ctypes.byref(args))
    if rc == 0:
        raise ValueError(backend.info().note.decode())
    if rc < 0:
        raise RuntimeError(backend.info().note.decode())


def _same_device(*tensors):
    first = tensors[0].device
    for t in tensors[1:]:
        _need(t is None or t.device == first, "all tensors must be on one GPU")
    return first


def plan(backend, held, added, tables, free_pages, rows, base=0, after=None):
    """Give this step's rows their pages and slots.

    held, added: [requests] own rows held before the step, and rows it adds;
    tables: [requests, pages per request] page ids, its new entries written in
    place; free_pages: ids of free pages, taken from the front (from where
    `after`, an earlier Plan over the same list, stopped); rows: batch rows, at
    least the sum of `added`; base: position of own row 0 (the prefix's rows).
    A step that cannot be taken as a whole sets bits in summary[0], and every
    slot is then -1, every other state as before.
    """
    torch = _torch()
    requests = held.shape[0]
    _ints(torch, held, (requests,), "held")
    _ints(torch, added, (requests,), "added")
    _need(tables.dim() == 2 and tables.shape[0] == requests, "tables: [requests, pages per request]")
    _ints(torch, tables, None, "tables")
    _need(free_pages.dim() == 1, "free_pages: one dimension")
    _ints(torch, free_pages, None, "free_pages")
    _need(rows >= 0, "rows: not negative")
    device = _same_device(held, added, tables, free_pages, None if after is None else after.summary)
    # One allocation, a 16-byte boundary for each part.
    sizes = [requests, requests + 1, rows, rows, 4]
    offsets, total = [], 0
    for n in sizes:
        offsets.append(total)
        total += -(-n // 4) * 4
    buffer = torch.empty(total, dtype=torch.int32, device=device)
    parts = [buffer[o:o + n] for o, n in zip(offsets, sizes)]
    at = buffer.data_ptr()
    p = [at + 4 * o for o in offsets]
    head = 0 if after is None else after.summary.data_ptr() + 8
    args = _abi.PagedPlanArgs(held.data_ptr(), added.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), head, p[0], p[1],
                              p[2], p[3], p[4], requests, tables.shape[1], free_pages.shape[0], rows, base,
                              _stream(torch, device))
    _run(backend, backend.lib.plamo_paged_plan, args)
    return Plan(*parts)


def store(backend, qkv, pool, slots, positions, q_norm, k_norm, table, status=None):
    """Between the QKV projection and attention: q and k heads are normalised
    (RMSNorm with `norm` + 1) and rotated, k and v written to their slots.

    qkv: [rows, (query_heads + 2 * kv_heads) * 128] BF16 or FP32 (rows may be
    strided); slots, positions: [rows] of the plan; q_norm, k_norm: [128] BF16;
    table: [positions, 128] FP32, cos | sin of each position. Returns the
    queries, [rows, query_heads, 128] of the pool's type.
    """
    torch = _torch()
    kind, pages, kv_heads = _pool(torch, pool)
    _need(qkv.dim() == 2 and qkv.shape[1] % DIM == 0 and qkv.is_cuda and (qkv.stride(1) == 1 or qkv.shape[0] == 0),
          f"qkv: [rows, heads * {DIM}] on the GPU, each row contiguous")
    rows, heads = qkv.shape[0], qkv.shape[1] // DIM
    query_heads = heads - 2 * kv_heads
    _need(query_heads > 0, "qkv: no query heads beside the pool's kv_heads")
    qkv_kind = _type(torch, qkv, "qkv")
    _ints(torch, slots, (rows,), "slots")
    _ints(torch, positions, (rows,), "positions")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        _need(t.dtype == torch.bfloat16 and tuple(t.shape) == (DIM,) and t.is_cuda and t.is_contiguous(),
              f"{name}: a contiguous BF16 [{DIM}] tensor on the GPU")
    _need(table.dtype == torch.float32 and table.dim() == 2 and table.shape[1] == DIM and table.is_cuda and
          table.is_contiguous(), f"table: a contiguous FP32 [positions, {DIM}] tensor on the GPU")
    if status is not None:
        _ints(torch, status, (1,), "status")
    device = _same_device(qkv, pool, slots, positions, q_norm, k_norm, table, status)
    q = torch.empty(rows, query_heads, DIM, dtype=pool.dtype, device=device)
    args = _abi.PagedStoreArgs(qkv.data_ptr(), pool.data_ptr(), q.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                               q_norm.data_ptr(), k_norm.data_ptr(), table.data_ptr(),
                               0 if status is None else status.data_ptr(), rows, max(qkv.stride(0), heads * DIM) if rows <= 1
                               else qkv.stride(0), query_heads * DIM, pages, table.shape[0], query_heads, kv_heads, qkv_kind,
                               kind, _stream(torch, device))
    _run(backend, backend.lib.plamo_paged_store, args)
    return q


def attention(backend, q, pool, starts, lengths, tables, prefix_pages=None, prefix_rows=0, window=0, scale=None, out=None,
              status=None):
    """Every query over the shared prefix and its own request's rows, causal.

    q: [rows, query_heads, 128] of the pool's type (rows may be strided);
    starts, lengths: of the plan; tables: [requests, pages per request];
    prefix_pages: the shared prefix's pages, prefix_rows rows of them used;
    window: rows a query sees, itself included (0: all before it); scale: of
    the scores, 1 / sqrt(128) unless given. Returns `out`, allocated if None.
    """
    torch = _torch()
    kind, pages, kv_heads = _pool(torch, pool)

    def rows_of(t, name):
        _need(t.dim() == 3 and t.shape[2] == DIM and t.is_cuda and t.dtype == pool.dtype and
              (t.shape[0] == 0 or (t.stride(2) == 1 and (t.shape[1] == 1 or t.stride(1) == DIM))),
              f"{name}: [rows, query_heads, {DIM}] of the pool's type on the GPU, each row contiguous")
        return t.stride(0) if t.shape[0] > 1 else t.shape[1] * DIM

    q_stride = rows_of(q, "q")
    rows, query_heads = q.shape[0], q.shape[1]
    requests = lengths.shape[0]
    _ints(torch, lengths, (requests,), "lengths")
    _ints(torch, starts, (requests + 1,), "starts")
    _need(tables.dim() == 2 and tables.shape[0] == requests, "tables: [requests, pages per request]")
    _ints(torch, tables, None, "tables")
    _need(prefix_rows >= 0 and window >= 0, "prefix_rows and window: not negative")
    if prefix_rows:
        _need(prefix_pages is not None and prefix_pages.dim() == 1 and prefix_pages.shape[0] * ROWS >= prefix_rows,
              "prefix_pages: one dimension, pages for prefix_rows rows")
        _ints(torch, prefix_pages, None, "prefix_pages")
    if status is not None:
        _ints(torch, status, (1,), "status")
    if out is None:
        out = torch.empty(rows, query_heads, DIM, dtype=pool.dtype, device=q.device)
    else:
        _need(out.shape == q.shape, "out: of q's shape")
    out_stride = rows_of(out, "out")
    device = _same_device(q, pool, out, starts, lengths, tables, prefix_pages, status)
    args = _abi.PagedAttentionArgs(q.data_ptr(), pool.data_ptr(), out.data_ptr(), starts.data_ptr(), lengths.data_ptr(),
                                   tables.data_ptr(), prefix_pages.data_ptr() if prefix_rows else 0, 0, 0,
                                   0 if status is None else status.data_ptr(), rows, q_stride, out_stride, requests,
                                   tables.shape[1], prefix_rows, pages, window, query_heads, kv_heads, kind,
                                   DIM ** -0.5 if scale is None else scale, _stream(torch, device))
    size = backend.lib.plamo_paged_attention_workspace(backend.ctx, ctypes.byref(args))
    if not size:
        raise ValueError(backend.info().note.decode())
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    _run(backend, backend.lib.plamo_paged_attention, args)
    return out
