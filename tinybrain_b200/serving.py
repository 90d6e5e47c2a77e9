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

A step (row counts on the device; buffers of the largest step).  The tokens are
sampled from each sequence's last row alone (of one without new tokens: some row):

    build_page_tables(cached, new, free, table, offsets, total, seq, pos, slot, info)
    last = (offsets[1:] - 1).clamp(min=0)
    for layer in range(num_layers):
        ...                                             # q, k, v projections
        rope_append(q, k, v, pos, slot, rope, pool, q, layer=layer, num_rows=offsets[-1:])
        paged_attention_chunk(q, offsets, total, pool, table, out, layer=layer, max_new=.., max_len=..)
    ...                                                 # logits of the rows `last`: [sequences, vocab]
    token = sample_rows(logits, uniform, temperature=.., top_k=.., top_p=.., min_p=..)[0]
"""
from __future__ import annotations

import ctypes as C
import functools

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


# The checks below run for every tensor of every call, a large part of a small
# call's cost: attributes that torch answers fastest, the messages only on failure.
def _flat(t, name, dtype, gpu, n=None):
    """The address of a contiguous 1-D tensor of `dtype` on GPU `gpu`, of n values where n is given."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == gpu and t.dim() == 1
            and (n is None or t.numel() == n) and t.is_contiguous()):
        return t.data_ptr()
    raise ValueError(f"{name} must be a contiguous {dtype} tensor [{'n' if n is None else n}] on cuda:{gpu}, got "
                     f"{_say(t)}")


def _rows(t, name, gpu, rows=None, cols=None):
    """Address and row stride of an fp32 tensor [rows, cols] whose rows are contiguous (any stride of at least a row)."""
    if isinstance(t, torch.Tensor) and t.dtype is _F32 and t.get_device() == gpu and t.dim() == 2:
        n, width = t.shape
        if (rows is None or n == rows) and (cols is None or width == cols):
            if t.is_contiguous():
                return t.data_ptr(), width
            step, inner = t.stride()
            if (inner == 1 or width <= 1) and (n <= 1 or step >= width):
                return t.data_ptr(), step if n > 1 else width
    want = [("rows" if rows is None else rows), ("cols" if cols is None else cols)]
    raise ValueError(f"{name} must be a float32 tensor {want} with contiguous rows on cuda:{gpu}, got {_say(t)}")


def _say(t):
    if not isinstance(t, torch.Tensor):
        return type(t).__name__
    return f"{t.dtype} {list(t.shape)} strides {list(t.stride())} on {t.device}"


def _gpu(t, name):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{name} must be a CUDA tensor, got {_say(t)}")
    return t.get_device()


def _pool(pool, layer):
    gpu = _gpu(pool, "kv pool")
    shape = pool.shape
    if not (pool.dtype is _F32 and len(shape) == 6 and shape[2] == 2 and shape[4] == PAGE_TOKENS
            and pool.is_contiguous() and pool.numel()):
        raise ValueError(f"kv pool must be a contiguous float32 tensor [pages, layers, 2, kv_heads, 16, head_dim], got "
                         f"{_say(pool)}")
    if not 0 <= layer < shape[1]:
        raise ValueError(f"layer {layer} is outside the pool's {shape[1]} layers")
    return gpu, shape[0], shape[1], shape[3], shape[5]


def _table(table, gpu):
    if not (isinstance(table, torch.Tensor) and table.dtype is _I32 and table.get_device() == gpu and table.dim() == 2
            and table.is_contiguous() and table.numel()):
        raise ValueError(f"page table must be a contiguous int32 tensor [sequences, pages] on cuda:{gpu}, got "
                         f"{_say(table)}")
    return table.shape


def _call(name, *args):
    status = getattr(_lib.load(), name)(*args)
    if status:
        _lib.check(status)


def build_page_tables(cached_lens, new_lens, free_pages, page_table, row_offsets, total_lens, row_seq, row_pos,
                      row_slot, info):
    """Page tables and slot maps of a step (tb_page_tables_build_dev).

    In: cached_lens, new_lens int32 [sequences]; free_pages int32 [n].  In and
    out: page_table int32 [sequences, pages].  Out: row_offsets [sequences + 1],
    total_lens [sequences], row_seq, row_pos [rows], row_slot int64 [rows], info
    int32 [4] = rows, pages taken (off free_pages' front), PAGES_* status, first
    bad sequence.  A step that does not fit has no rows and takes no page."""
    gpu = _gpu(page_table, "page_table")
    batch, stride = _table(page_table, gpu)
    rows = row_seq.numel() if isinstance(row_seq, torch.Tensor) else None
    free = _flat(free_pages, "free_pages", _I32, gpu)
    _call("tb_page_tables_build_dev", _stream_of(gpu), _flat(cached_lens, "cached_lens", _I32, gpu, batch),
          _flat(new_lens, "new_lens", _I32, gpu, batch), batch, free or None, free_pages.numel(), page_table.data_ptr(),
          stride, rows, _flat(row_offsets, "row_offsets", _I32, gpu, batch + 1),
          _flat(total_lens, "total_lens", _I32, gpu, batch), _flat(row_seq, "row_seq", _I32, gpu),
          _flat(row_pos, "row_pos", _I32, gpu, rows), _flat(row_slot, "row_slot", _I64, gpu, rows),
          _flat(info, "info", _I32, gpu, 4))
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
    gpu, pages, layers, kv, d = _pool(pool, layer)
    qp, ld_q = _rows(q, "q", gpu)
    rows, cols = q.shape
    if q_out is None:
        q_out = torch.empty(rows, cols, dtype=_F32, device=pool.device)
    _need(cols and cols % (kv * d) == 0, "q has no whole heads per kv head")
    kp, ld_k = _rows(k, "k", gpu, rows, kv * d)
    vp, ld_v = _rows(v, "v", gpu, rows, kv * d)
    op, ld_o = _rows(q_out, "q_out", gpu, rows, cols)
    if not (isinstance(rope, torch.Tensor) and rope.dtype is _F32 and rope.get_device() == gpu and rope.dim() == 3
            and rope.shape[1:] == (d // 2, 2) and d % 2 == 0 and rope.is_contiguous() and rope.numel()):
        raise ValueError(f"rope must be a contiguous float32 tensor [positions, {d // 2}, 2] on cuda:{gpu}, got "
                         f"{_say(rope)}")
    pos, slot = _flat(row_pos, "row_pos", _I32, gpu), _flat(row_slot, "row_slot", _I64, gpu)
    if row_pos.numel() < rows or row_slot.numel() < rows:
        raise ValueError(f"row_pos and row_slot hold {row_pos.numel()} and {row_slot.numel()} of {rows} rows")
    count = None if num_rows is None else _flat(num_rows, "num_rows", _I32, gpu, 1)
    if rows:
        _call("tb_rope_append_paged_dev", _stream_of(gpu), qp, ld_q, kp, ld_k, vp, ld_v, rows, count, pos, slot,
              rope.data_ptr(), rope.shape[0], layer, layers, cols // d, kv, d, pool.data_ptr(), pages, op, ld_o)
    return q_out


def paged_attention_chunk(q, row_offsets, total_lens, pool, page_table, out=None, *, layer, max_new, max_len,
                          workspace=None):
    """Attention of each sequence's new tokens over its pages (tb_paged_attention_chunk_dev).

    q, out [rows, heads * d]; row_offsets int32 [sequences + 1] and total_lens
    [sequences] as build_page_tables writes them; max_new and max_len bound a
    sequence's new tokens and length (they shape the launch; larger ones stay
    right).  workspace: a uint8 tensor of paged_attention_chunk_workspace bytes
    that no overlapping call uses; None takes one from torch's allocator for
    this call: up to 30 MB, and for long prompts as much more as one layer's K and V
    of sequences * max_len tokens, at most 1 GiB (a tight max_len keeps it small).
    The header states the accuracy.  Returns out."""
    gpu, pages, layers, kv, d = _pool(pool, layer)
    batch, stride = _table(page_table, gpu)
    qp, ld_q = _rows(q, "q", gpu)
    rows, cols = q.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=_F32, device=pool.device)
    op, ld_o = _rows(out, "out", gpu, rows, cols)
    _need(cols and cols % (kv * d) == 0, "q has no whole heads per kv head")
    offsets = _flat(row_offsets, "row_offsets", _I32, gpu, batch + 1)
    totals = _flat(total_lens, "total_lens", _I32, gpu, batch)
    _need(1 <= max_new < 1 << 31 and 1 <= max_len < 1 << 31, "max_new and max_len must be at least 1")
    if not rows:
        return out
    heads = cols // d
    if workspace is None:
        workspace = torch.empty(paged_attention_chunk_workspace(rows, batch, max_new, max_len, heads, kv, d),
                                dtype=torch.uint8, device=pool.device)
    work = _flat(workspace, "workspace", torch.uint8, gpu)
    _call("tb_paged_attention_chunk_dev", _stream_of(gpu), qp, ld_q, rows, offsets, totals, batch, pool.data_ptr(),
          pages, page_table.data_ptr(), stride, max_new, max_len, layer, layers, heads, kv, d, op, ld_o, work or None,
          workspace.numel())
    return out


@functools.lru_cache(maxsize=1024)
def paged_attention_chunk_workspace(rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim) -> int:
    """Bytes of workspace that paged_attention_chunk needs for these bounds."""
    n = C.c_int64(0)
    call("tb_paged_attention_chunk_workspace", rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim,
         C.byref(n))
    return n.value


def sample_rows(logits, uniform, token=None, prob=None, entropy=None, *, temperature=None, top_k=None, top_p=None,
                min_p=None):
    """One token per row of logits [rows, vocab] from uniform [rows] in [0, 1) (tb_sample_rows_dev).

    temperature, top_p, min_p float32 and top_k int32 [rows], or None for off.
    Returns (token int32, prob, entropy); a row with nothing above -inf gives -1."""
    gpu = _gpu(logits, "logits")
    lp, ld = _rows(logits, "logits", gpu)
    rows, vocab = logits.shape
    _need(vocab >= 1, "logits have no columns")
    if token is None:
        token = torch.empty(rows, dtype=_I32, device=logits.device)
    if prob is None:
        prob = torch.empty(rows, dtype=_F32, device=logits.device)
    if entropy is None:
        entropy = torch.empty(rows, dtype=_F32, device=logits.device)
    if rows:
        _call("tb_sample_rows_dev", _stream_of(gpu), lp, ld, rows, vocab,
              None if temperature is None else _flat(temperature, "temperature", _F32, gpu, rows),
              None if top_k is None else _flat(top_k, "top_k", _I32, gpu, rows),
              None if top_p is None else _flat(top_p, "top_p", _F32, gpu, rows),
              None if min_p is None else _flat(min_p, "min_p", _F32, gpu, rows),
              _flat(uniform, "uniform", _F32, gpu, rows), _flat(token, "token", _I32, gpu, rows),
              _flat(prob, "prob", _F32, gpu, rows), _flat(entropy, "entropy", _F32, gpu, rows))
    return token, prob, entropy


def check_device(device=None):
    """Waits for torch's current stream and raises TinyBrainError for what the calls above recorded on the device
    (a page or position outside its table, a device-side wait that ran out); clears the record."""
    index = torch.device("cuda" if device is None else device).index
    with torch.cuda.device(torch.cuda.current_device() if index is None else index):
        call("tb_paged_attention_noalloc_status", torch.cuda.current_stream().cuda_stream, 1)
