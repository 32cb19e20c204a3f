"""Operators of a paged batch step on torch tensors (include/plamo_paged.h).

Requests behind one shared prompt prefix keep their keys and values in a pool
of 64-row pages, [pages, 2, 64, kv_heads, 128] in BF16 or FP32. A step plans
its rows once (`plan`), then per layer stores the projection's rows (`store`)
and attends (`attention`). Calls are enqueued on torch's current stream and
return without waiting; tensors they allocate come from torch's allocator.
Wrong arguments raise ValueError, tensors of another GPU than the backend's
among them. What only the GPU can see is reported as PLAMO_PAGED_* bits, in the
plan's summary and in a `status` tensor (one int32, zeroed by the caller), or
where a call is given none in a word of the backend's that `status()` reads.
"""
import ctypes
from typing import NamedTuple

from . import _abi

ROWS, DIM = _abi.PAGED_ROWS, _abi.PAGED_DIM


class Plan(NamedTuple):
    """What a step's operators need of its rows (int32 tensors)."""
    lengths: object    # [requests] own rows after the step
    starts: object     # [requests + 1] first batch row of each request
    slots: object      # [rows] page * 64 + row in the page, -1 for padding, -2 where the page id is none
    positions: object  # [rows]
    summary: object    # [4] status bits, new rows, free-list entries used so far, longest length


_t = None


def _torch():
    global _t
    if _t is None:
        import torch
        _t = torch
    return _t


def _stream(torch, device):
    """torch's current stream of device index `device`; 0 would name the context's own stream, 1 is the default one."""
    return torch._C._cuda_getCurrentRawStream(device) or 1


# The checks sit on the path of calls that take a few microseconds in all: plain
# comparisons, messages only when one fails.

def _ints(torch, t, count, device, name):
    if t.dtype != torch.int32 or t.get_device() != device or not t.is_contiguous() or (count >= 0 and t.numel() != count):
        raise ValueError(f"{name}: a contiguous int32 tensor on GPU {device}" + (f" with {count} entries" if count >= 0 else ""))


def _type(torch, t, name):
    if t.dtype == torch.bfloat16:
        return _abi.PAGED_BF16
    if t.dtype != torch.float32:
        raise ValueError(f"{name}: BF16 or FP32")
    return _abi.PAGED_FP32


def _pool(torch, pool, backend):
    """(type, pages, kv_heads, device index) of a pool."""
    if pool.dim() != 5 or not pool.is_contiguous() or pool.get_device() != backend.device:
        raise ValueError(f"pool: a contiguous [pages, 2, {ROWS}, kv_heads, {DIM}] tensor on the backend's GPU, {backend.device}")
    pages, two, rows, kv_heads, dim = pool.shape
    if two != 2 or rows != ROWS or dim != DIM:
        raise ValueError(f"pool: a contiguous [pages, 2, {ROWS}, kv_heads, {DIM}] tensor on the GPU")
    return _type(torch, pool, "pool"), pages, kv_heads, pool.get_device()


def _tables(torch, tables, requests, device):
    if tables.dim() != 2 or tables.shape[0] != requests:
        raise ValueError("tables: [requests, pages per request]")
    _ints(torch, tables, -1, device, "tables")
    return tables.shape[1]


def _status(torch, status, device):
    if status is None:
        return 0
    _ints(torch, status, 1, device, "status")
    return status.data_ptr()


def _run(backend, call, args):
    rc = call(backend.ctx, ctypes.byref(args))
    if rc == 0:
        raise ValueError(backend.info().note.decode())
    if rc < 0:
        raise RuntimeError(backend.info().note.decode())


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
    requests, device = held.numel(), held.get_device()
    if device != backend.device or rows < 0:
        raise ValueError(f"held: on the backend's GPU, {backend.device}; rows: not negative")
    _ints(torch, held, requests, device, "held")
    _ints(torch, added, requests, device, "added")
    _ints(torch, free_pages, -1, device, "free_pages")
    if free_pages.dim() != 1:
        raise ValueError("free_pages: one dimension")
    stride = _tables(torch, tables, requests, device)
    head = 0
    if after is not None:
        _ints(torch, after.summary, 4, device, "after.summary")
        head = after.summary.data_ptr() + 8
    buffer = held.new_empty(2 * requests + 2 * rows + 5)
    at = buffer.data_ptr()
    starts = at + 4 * requests
    slots = starts + 4 * requests + 4
    positions = slots + 4 * rows
    args = _abi.PagedPlanArgs(held.data_ptr(), added.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), head, at, starts,
                              slots, positions, positions + 4 * rows, requests, stride, free_pages.numel(), rows, base,
                              _stream(torch, device))
    _run(backend, backend.lib.plamo_paged_plan, args)
    return Plan(*buffer.unsafe_split_with_sizes((requests, requests + 1, rows, rows, 4)))  # (split takes 3 us more)


def store(backend, qkv, pool, slots, positions, q_norm, k_norm, table, status=None):
    """Between the QKV projection and attention: q and k heads are normalised
    (RMSNorm with `norm` + 1) and rotated, k and v written to their slots.

    qkv: [rows, (query_heads + 2 * kv_heads) * 128] BF16 or FP32 (rows may be
    strided); slots, positions: [rows] of the plan; q_norm, k_norm: [128] BF16;
    table: [positions, 128] FP32, cos | sin of each position. Returns the
    queries, [rows, query_heads, 128] of the pool's type.
    """
    torch = _torch()
    kind, pages, kv_heads, device = _pool(torch, pool, backend)
    if qkv.dim() != 2 or qkv.get_device() != device:
        raise ValueError(f"qkv: [rows, heads * {DIM}] on the pool's GPU")
    rows, width = qkv.shape
    row_stride, step = qkv.stride()
    query_heads = width // DIM - 2 * kv_heads
    if width % DIM or query_heads <= 0 or (step != 1 and rows):
        raise ValueError(f"qkv: contiguous rows of {DIM} * (query heads + 2 * {kv_heads}) entries")
    qkv_kind = _type(torch, qkv, "qkv")
    _ints(torch, slots, rows, device, "slots")
    _ints(torch, positions, rows, device, "positions")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t.dtype != torch.bfloat16 or t.numel() != DIM or t.get_device() != device or not t.is_contiguous():
            raise ValueError(f"{name}: a contiguous BF16 [{DIM}] tensor on the pool's GPU")
    if (table.dtype != torch.float32 or table.dim() != 2 or table.shape[1] != DIM or table.get_device() != device or
            not table.is_contiguous()):
        raise ValueError(f"table: a contiguous FP32 [positions, {DIM}] tensor on the pool's GPU")
    q = pool.new_empty((rows, query_heads, DIM))
    args = _abi.PagedStoreArgs(qkv.data_ptr(), pool.data_ptr(), q.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                               q_norm.data_ptr(), k_norm.data_ptr(), table.data_ptr(), _status(torch, status, device), rows,
                               row_stride if rows > 1 else width, query_heads * DIM, pages, table.shape[0], query_heads,
                               kv_heads, qkv_kind, kind, _stream(torch, device))
    _run(backend, backend.lib.plamo_paged_store, args)
    return q


def attention(backend, q, pool, starts, lengths, tables, prefix_pages=None, prefix_rows=0, window=0, scale=None, out=None,
              status=None, most_new=0):
    """Every query over the shared prefix and its own request's rows, causal.

    q: [rows, query_heads, 128] of the pool's type (rows may be strided);
    starts, lengths: of the plan; tables: [requests, pages per request];
    prefix_pages: the shared prefix's pages, prefix_rows rows of them used;
    window: rows a query sees, itself included (0: all before it); scale: of
    the scores, 1 / sqrt(128) unless given; most_new: rows of the request that
    adds most (1 in a decode step; 0: not known), which chooses the kernels where
    q has rows of padding or lengths idle slots. Returns `out`, allocated if None.
    """
    torch = _torch()
    kind, pages, kv_heads, device = _pool(torch, pool, backend)
    q_stride = _rows(torch, q, pool, device, "q")
    rows, query_heads, _ = q.shape
    requests = lengths.numel()
    _ints(torch, lengths, requests, device, "lengths")
    _ints(torch, starts, requests + 1, device, "starts")
    stride = _tables(torch, tables, requests, device)
    if prefix_rows < 0 or window < 0 or most_new < 0:
        raise ValueError("prefix_rows, window and most_new: not negative")
    prefix = 0
    if prefix_rows:
        if prefix_pages is None or prefix_pages.dim() != 1 or prefix_pages.numel() * ROWS < prefix_rows:
            raise ValueError("prefix_pages: one dimension, pages for prefix_rows rows")
        _ints(torch, prefix_pages, -1, device, "prefix_pages")
        prefix = prefix_pages.data_ptr()
    if out is None:
        out = pool.new_empty((rows, query_heads, DIM))
        out_stride = query_heads * DIM
    else:
        if out.shape != q.shape:
            raise ValueError("out: of q's shape")
        out_stride = _rows(torch, out, pool, device, "out")
    args = _abi.PagedAttentionArgs(q.data_ptr(), pool.data_ptr(), out.data_ptr(), starts.data_ptr(), lengths.data_ptr(),
                                   tables.data_ptr(), prefix, 0, 0, _status(torch, status, device), rows, q_stride, out_stride,
                                   requests, stride, prefix_rows, pages, window, query_heads, kv_heads, kind,
                                   DIM ** -0.5 if scale is None else scale, _stream(torch, device), most_new)
    size = backend.lib.plamo_paged_attention_workspace(backend.ctx, ctypes.byref(args))
    if not size:
        raise ValueError(backend.info().note.decode())
    workspace = pool.new_empty(size, dtype=torch.uint8)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), size
    _run(backend, backend.lib.plamo_paged_attention, args)
    return out


def status(backend):
    """PLAMO_PAGED_* bits set by stores and attention calls without a `status`
    tensor since last asked (they are then clear). Waits for torch's current
    stream; calls on others count once those have run them."""
    _torch().cuda.current_stream(backend.device).synchronize()
    return backend.lib.plamo_paged_status(backend.ctx)


def _rows(torch, t, pool, device, name):
    """Row stride of [rows, heads, 128] queries or results."""
    if t.dim() == 3 and t.dtype == pool.dtype and t.get_device() == device:
        rows, heads, dim = t.shape
        row, head, step = t.stride()
        if dim == DIM and (rows == 0 or (step == 1 and (heads == 1 or head == DIM))):
            return row if rows > 1 else heads * DIM
    raise ValueError(f"{name}: [rows, query_heads, {DIM}] of the pool's type and GPU, each row contiguous")
