"""One serving step over the paged KV cache, on device tensors.

For a host that runs its own projections and keeps the step on the GPU: page
tables and slot maps from the sequences' lengths (`build_page_tables`), RoPE
with the write to the cache (`rope_append`), attention of every sequence's new
tokens (`paged_attention_chunk`), and the next tokens (`sample_rows`).  The
definitions stand in include/tinybrain_cuda.h.

Tensors are torch tensors on one GPU, which need not be the current one; every
call runs on torch's current stream of that GPU, returns without waiting and
may be captured into a CUDA graph.  The cache is the framework's pool,
[pages][layers][K, V][kv heads][16][head dim] fp32.  Wrong arguments raise
ValueError before anything runs; bad pages and positions found on the device
are reported by `check_device`.

A step (row counts on the device; buffers of the largest step):

    build_page_tables(cached, new, free, table, offsets, total, seq, pos, slot, info)
    for layer in range(num_layers):
        ...                                             # q, k, v projections
        rope_append(q, k, v, pos, slot, rope, pool, q, layer=layer, num_rows=offsets[-1:])
        paged_attention_chunk(q, offsets, total, pool, table, out, layer=layer, max_new=.., max_len=..)
    token = sample_rows(logits, uniform, temperature=.., top_k=.., top_p=.., min_p=..)[0]
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import call

PAGE_TOKENS = 16
PAGES_OK, PAGES_BAD_LENGTH, PAGES_ROWS_EXCEEDED, PAGES_EXHAUSTED = range(4)

_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64
_stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _flat(t, name, dtype, device, n=None):
    """A contiguous 1-D tensor of `dtype` on `device`, of n values where n is given."""
    if not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == device and t.dim() == 1
            and (n is None or t.shape[0] == n) and (t.shape[0] <= 1 or t.stride(0) == 1)):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor [{'n' if n is None else n}] on {device}, got "
                         f"{_say(t)}")
    return t.data_ptr()


def _rows(t, name, device, rows=None, cols=None):
    """An fp32 tensor [rows, cols] whose rows are contiguous (any row stride of at least a row)."""
    if not (isinstance(t, torch.Tensor) and t.dtype == _F32 and t.device == device and t.dim() == 2
            and (rows is None or t.shape[0] == rows) and (cols is None or t.shape[1] == cols)
            and (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])):
        want = [("rows" if rows is None else rows), ("cols" if cols is None else cols)]
        raise ValueError(f"{name} must be a float32 tensor {want} with contiguous rows on {device}, got {_say(t)}")
    return t.data_ptr(), (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _say(t):
    if not isinstance(t, torch.Tensor):
        return type(t).__name__
    return f"{t.dtype} {list(t.shape)} strides {list(t.stride())} on {t.device}"


def _gpu(t, name):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{name} must be a CUDA tensor, got {_say(t)}")
    return t.device


def _pool(pool, device, layer):
    if not (isinstance(pool, torch.Tensor) and pool.dtype == _F32 and pool.device == device and pool.dim() == 6
            and pool.shape[2] == 2 and pool.shape[4] == PAGE_TOKENS and pool.is_contiguous() and pool.numel()):
        raise ValueError("kv pool must be a contiguous float32 tensor [pages, layers, 2, kv_heads, 16, head_dim] on "
                         f"{device}, got {_say(pool)}")
    _need(0 <= layer < pool.shape[1], f"layer {layer} is outside the pool's {pool.shape[1]} layers")
    return pool.shape[0], pool.shape[1], pool.shape[3], pool.shape[5]


def _table(table, device):
    if not (isinstance(table, torch.Tensor) and table.dtype == _I32 and table.device == device and table.dim() == 2
            and table.is_contiguous() and table.numel()):
        raise ValueError(f"page table must be a contiguous int32 tensor [sequences, pages] on {device}, got "
                         f"{_say(table)}")
    return table.shape


def build_page_tables(cached_lens, new_lens, free_pages, page_table, row_offsets, total_lens, row_seq, row_pos,
                      row_slot, info):
    """Page tables and slot maps of a step (tb_page_tables_build_dev).

    In: cached_lens, new_lens int32 [sequences]; free_pages int32 [n].  In and
    out: page_table int32 [sequences, pages].  Out: row_offsets [sequences + 1],
    total_lens [sequences], row_seq, row_pos [rows], row_slot int64 [rows], info
    int32 [4] = rows, pages taken (off free_pages' front), PAGES_* status, first
    bad sequence.  A step that does not fit has no rows and takes no page."""
    device = _gpu(page_table, "page_table")
    batch, stride = _table(page_table, device)
    rows = row_seq.shape[0] if isinstance(row_seq, torch.Tensor) and row_seq.dim() == 1 else None
    call("tb_page_tables_build_dev", _stream_of(device.index), _flat(cached_lens, "cached_lens", _I32, device, batch),
         _flat(new_lens, "new_lens", _I32, device, batch), batch, _flat(free_pages, "free_pages", _I32, device) or None,
         free_pages.shape[0], page_table.data_ptr(), stride, rows,
         _flat(row_offsets, "row_offsets", _I32, device, batch + 1),
         _flat(total_lens, "total_lens", _I32, device, batch), _flat(row_seq, "row_seq", _I32, device),
         _flat(row_pos, "row_pos", _I32, device, rows), _flat(row_slot, "row_slot", _I64, device, rows),
         _flat(info, "info", _I32, device, 4))
    return info


def rope_table(positions: int, head_dim: int, device) -> torch.Tensor:
    """The runner's (cos, sin) table [positions, head_dim / 2, 2] on `device` (tb_rope_table)."""
    host = torch.empty(positions, head_dim // 2, 2, dtype=_F32)
    call("tb_rope_table", positions, head_dim, C.c_void_p(host.data_ptr()))
    return host.to(device)


def rope_append(q, k, v, row_pos, row_slot, rope, pool, q_out=None, *, layer, num_rows=None):
    """RoPE on q and k; k and v to their cache slots; q to q_out (tb_rope_append_paged_dev).

    q [rows, heads * d], k and v [rows, kv_heads * d] with any row stride (the
    columns of a fused projection); q_out may be q.  num_rows: the step's row
    count on the device (row_offsets[-1:]), or None for all.  Returns q_out."""
    device = _gpu(pool, "kv pool")
    pages, layers, kv, d = _pool(pool, device, layer)
    qp, ld_q = _rows(q, "q", device)
    rows = q.shape[0]
    if q_out is None:
        q_out = torch.empty(rows, q.shape[1], dtype=_F32, device=device)
    _need(q.shape[1] % (kv * d) == 0 and q.shape[1], f"q has {q.shape[1]} columns for {kv} kv heads of {d}")
    kp, ld_k = _rows(k, "k", device, rows, kv * d)
    vp, ld_v = _rows(v, "v", device, rows, kv * d)
    op, ld_o = _rows(q_out, "q_out", device, rows, q.shape[1])
    if not (isinstance(rope, torch.Tensor) and rope.dtype == _F32 and rope.device == device and rope.dim() == 3
            and rope.shape[1] * 2 == d and rope.shape[2] == 2 and rope.is_contiguous() and rope.numel()):
        raise ValueError(f"rope must be a contiguous float32 tensor [positions, {d // 2}, 2] on {device}, got "
                         f"{_say(rope)}")
    if rows:
        call("tb_rope_append_paged_dev", _stream_of(device.index), qp, ld_q, kp, ld_k, vp, ld_v, rows,
             None if num_rows is None else _flat(num_rows, "num_rows", _I32, device, 1),
             _flat(row_pos, "row_pos", _I32, device)
             if row_pos.shape[0] >= rows else _short("row_pos", row_pos, rows),
             _flat(row_slot, "row_slot", _I64, device)
             if row_slot.shape[0] >= rows else _short("row_slot", row_slot, rows),
             rope.data_ptr(), rope.shape[0], layer, layers, q.shape[1] // d, kv, d, pool.data_ptr(), pages, op, ld_o)
    return q_out


def _short(name, t, rows):
    raise ValueError(f"{name} holds {t.shape[0]} of {rows} rows")


def paged_attention_chunk(q, row_offsets, total_lens, pool, page_table, out=None, *, layer, max_new, max_len,
                          workspace=None):
    """Attention of each sequence's new tokens over its pages (tb_paged_attention_chunk_dev).

    q, out [rows, heads * d]; row_offsets int32 [sequences + 1] and total_lens
    [sequences] as build_page_tables writes them; max_new and max_len bound a
    sequence's new tokens and length (they shape the launch; larger ones stay
    right).  workspace: a uint8 tensor of paged_attention_chunk_workspace bytes
    that no overlapping call uses; None takes one from torch's allocator for
    this call.  Returns out."""
    device = _gpu(pool, "kv pool")
    pages, layers, kv, d = _pool(pool, device, layer)
    batch, stride = _table(page_table, device)
    qp, ld_q = _rows(q, "q", device)
    rows, cols = q.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=_F32, device=device)
    op, ld_o = _rows(out, "out", device, rows, cols)
    _need(cols % (kv * d) == 0 and cols, f"q has {cols} columns for {kv} kv heads of {d}")
    offsets = _flat(row_offsets, "row_offsets", _I32, device, batch + 1)
    totals = _flat(total_lens, "total_lens", _I32, device, batch)
    _need(1 <= max_new < 1 << 31 and 1 <= max_len < 1 << 31, "max_new and max_len must be at least 1")
    if not rows:
        return out
    heads = cols // d
    if workspace is None:
        workspace = torch.empty(paged_attention_chunk_workspace(rows, batch, max_new, max_len, heads, kv, d),
                                dtype=torch.uint8, device=device)
    wp = _flat(workspace, "workspace", torch.uint8, device)
    call("tb_paged_attention_chunk_dev", _stream_of(device.index), qp, ld_q, rows, offsets, totals, batch,
         pool.data_ptr(), pages, page_table.data_ptr(), stride, max_new, max_len, layer, layers, heads, kv, d, op,
         ld_o, wp or None, workspace.shape[0])
    return out


def paged_attention_chunk_workspace(rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim) -> int:
    """Bytes of workspace that paged_attention_chunk needs for these bounds on the current GPU's model."""
    n = C.c_int64(0)
    call("tb_paged_attention_chunk_workspace", rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim,
         C.byref(n))
    return n.value


def sample_rows(logits, uniform, token=None, prob=None, entropy=None, *, temperature=None, top_k=None, top_p=None,
                min_p=None):
    """One token per row of logits [rows, vocab] from uniform [rows] in [0, 1) (tb_sample_rows_dev).

    temperature, top_p, min_p float32 and top_k int32 [rows], or None for off.
    Returns (token int32, prob, entropy); a row with nothing above -inf gives -1."""
    device = _gpu(logits, "logits")
    lp, ld = _rows(logits, "logits", device)
    rows, vocab = logits.shape
    _need(vocab >= 1, "logits have no columns")
    token = torch.empty(rows, dtype=_I32, device=device) if token is None else token
    prob = torch.empty(rows, dtype=_F32, device=device) if prob is None else prob
    entropy = torch.empty(rows, dtype=_F32, device=device) if entropy is None else entropy
    if rows:
        each = lambda t, name, dtype: None if t is None else _flat(t, name, dtype, device, rows)  # noqa: E731
        call("tb_sample_rows_dev", _stream_of(device.index), lp, ld, rows, vocab, each(temperature, "temperature", _F32),
             each(top_k, "top_k", _I32), each(top_p, "top_p", _F32), each(min_p, "min_p", _F32),
             _flat(uniform, "uniform", _F32, device, rows), _flat(token, "token", _I32, device, rows),
             _flat(prob, "prob", _F32, device, rows), _flat(entropy, "entropy", _F32, device, rows))
    return token, prob, entropy


def check_device(device=None):
    """Waits for torch's current stream and raises TinyBrainError for what the calls above recorded on the device
    (a page or position outside its table, a device-side wait that ran out); clears the record."""
    index = torch.device("cuda" if device is None else device).index
    with torch.cuda.device(torch.cuda.current_device() if index is None else index):
        call("tb_paged_attention_noalloc_status", torch.cuda.current_stream().cuda_stream, 1)
