"""A 4-bit paged key/value cache: the part of a serving step between the
packed linear layers of :mod:`csed499ii_b200`.

* :func:`kv4_cache` -- one layer's cache tensor;
* :func:`kv4_schedule` -- block tables, slots and positions of a step, built on
  the GPU from the requests' lengths;
* :func:`kv4_append` / :func:`kv4_read` -- quantise keys and values into slots,
  and read slots back;
* :func:`kv4_attention` -- attention over the cache, for single tokens, a few
  tokens, prompts and steps that mix them.

The reference (hyeonu453/CSED499II) ends at the linear layers and has no
counterpart.  A page holds ``page_size`` tokens of every key/value head in
tiles of 16; each row of one token and head is 4-bit codes with a scale and an
offset (the row's minimum) in the model's type.  ``include/sm100_marlin.h`` has
the layout byte by byte.  Nothing here copies to the host or waits for the GPU.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ext, _stream_ptr

__all__ = ["kv4_cache", "kv4_schedule", "kv4_append", "kv4_read", "kv4_attention", "kv4_workspace",
           "KV4Step", "KV4_FATES"]

# what became of a request in kv4_schedule (SM100_MARLIN_KV4_* of the C header)
KV4_FATES = {"ok": 0, "no pages": 1, "table full": 2, "rows full": 3}

_DTYPES = {torch.half: 0, torch.bfloat16: 1}
_INT32 = torch.int32
# 16-bit elements of a tile -> channels of a head
_DIMS = {8 * 64 + 64: 64, 8 * 128 + 64: 128}


def _raise(name, err):
    raise RuntimeError(f"{name}: sm100_marlin error {err}: {_ext.describe(err)}")


def _entry(name):
    return getattr(_ext.load(), "sm100_marlin_" + name)


def _check_ints(name, t, dev, numel=None):
    if not t.is_cuda or t.get_device() != dev:
        raise RuntimeError(f"{name} must be a CUDA tensor on device {dev}")
    if t.dtype is not _INT32:
        raise RuntimeError(f"{name} must have dtype torch.int32, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise RuntimeError(f"{name} must have {numel} entries, got {t.numel()}")


def _check_tables(t, dev, batch):
    if not t.is_cuda or t.get_device() != dev:
        raise RuntimeError(f"block_tables must be a CUDA tensor on device {dev}")
    if t.dtype is not _INT32:
        raise RuntimeError(f"block_tables must have dtype torch.int32, got {t.dtype}")
    if t.dim() != 2 or t.size(0) != batch:
        raise RuntimeError(f"block_tables must have one row for each of the {batch} requests")
    if t.size(1) > 1 and t.stride(1) != 1:
        raise RuntimeError("block_tables must have contiguous rows")


def _cache_shape(cache):
    """(pages, kv_heads, page_size, head_dim, dtype code, device) of a cache tensor."""
    dtype = _DTYPES.get(cache.dtype)
    if dtype is None:
        raise RuntimeError(f"cache must be torch.half or torch.bfloat16, got {cache.dtype}")
    dev = cache.get_device()
    if dev < 0:
        raise RuntimeError("cache must be a CUDA tensor")
    shape = cache.shape
    dim = _DIMS.get(shape[-1]) if len(shape) == 4 else None
    if dim is None or not cache.is_contiguous():
        raise RuntimeError("cache must be a contiguous tensor as kv4_cache makes it, "
                           "(pages, kv_heads, page_size / 16, 8 * head_dim + 64)")
    return shape[0], shape[1], shape[2] * 16, dim, dtype, dev


def kv4_cache(pages, kv_heads, head_dim, page_size=64, dtype=torch.half, device="cuda"):
    """One layer's empty cache for ``pages`` pages of ``page_size`` tokens.

    A ``(pages, kv_heads, page_size / 16, 8 * head_dim + 64)`` tensor of the
    model's type that holds codes, scales and offsets (not values).
    @head_dim: 64 or 128
    @page_size: a multiple of 16
    @dtype: ``torch.half`` or ``torch.bfloat16``, that of the keys and queries
    """
    if head_dim not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    if page_size <= 0 or page_size % 16 != 0:
        raise ValueError("page_size must be a positive multiple of 16")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be torch.half or torch.bfloat16")
    if pages < 0 or kv_heads <= 0 or pages * page_size >= 2**31:
        raise ValueError("pages * page_size must be below 2**31 and kv_heads positive")
    return torch.zeros((pages, kv_heads, page_size // 16, 8 * head_dim + 64), dtype=dtype,
                       device=device)


class KV4Step(NamedTuple):
    """What :func:`kv4_schedule` returns; every field is an int32 tensor.

    ``starts``, ``slots``, ``positions`` and ``fate`` can share one allocation: who
    keeps one of them for long, or saves it, clones it."""

    lens: torch.Tensor        # (batch,) tokens in the cache after the step
    free_count: torch.Tensor  # (1,) free pages after the step
    starts: torch.Tensor      # (batch + 1,) first row of each request
    slots: torch.Tensor       # (rows,) page * page_size + place, or -1
    positions: torch.Tensor   # (rows,) position of the row's token in its request
    fate: torch.Tensor        # (batch,) KV4_FATES


def kv4_schedule(new_lens, lens, block_tables, free_pages, free_count, rows, page_size,
                 lens_out=None, free_count_out=None):
    """Block tables, slots and positions of one step, in one launch.

    Request ``b`` adds ``new_lens[b]`` tokens to the ``lens[b]`` that it has in
    the cache; a negative entry ends it, and its pages go back before any are
    handed out.  ``free_pages[:free_count]`` is a stack of free page ids, whose
    top goes out first, to the requests in order.  A request that cannot be
    served is refused whole: its ``fate`` says why, its length stays and its
    rows get slot -1; once the pages do not reach, later requests that need
    one are refused too.
    @new_lens, @lens: ``torch.int`` ``(batch,)``, at most 8192 requests
    @block_tables: ``torch.int`` ``(batch, width)``; new entries are written
    @free_pages: ``torch.int``; pages given back are written from ``free_count`` on
    @free_count: ``torch.int`` ``(1,)``
    @rows: rows of the step, padding included (slot -1, position 0 past the last request's)
    @lens_out, @free_count_out: tensors for the new lengths and count; they may
        lie in ``new_lens``, ``lens`` and ``free_count`` (a step that is replayed
        from a CUDA graph updates the last two in place)
    """
    fast = _ext._torch_fast if _ext._torch_fast_tried else _ext.torch_fast()
    if fast is not None:
        done = fast.kv4_schedule(new_lens, lens, block_tables, free_pages, free_count, rows, page_size,
                                 lens_out, free_count_out)
        if done is not None:
            if done[0]:
                _raise("kv4_schedule", done[0])
            return KV4Step(*done[1:])
    dev = new_lens.get_device()
    batch, tables_shape = new_lens.numel(), block_tables.shape
    # one combined test; the checks with their messages only run when it fails
    if not (dev >= 0 and new_lens.dtype is _INT32 and lens.dtype is _INT32 and lens.get_device() == dev
            and lens.numel() == batch <= 8192 and block_tables.dtype is _INT32
            and block_tables.get_device() == dev and len(tables_shape) == 2 and tables_shape[0] == batch
            and free_pages.dtype is _INT32 and free_pages.get_device() == dev
            and free_count.dtype is _INT32 and free_count.get_device() == dev and free_count.numel() == 1
            and new_lens.is_contiguous() and lens.is_contiguous() and block_tables.is_contiguous()
            and free_pages.is_contiguous() and 0 <= rows < 2**31 and 0 < page_size < 2**31
            and free_pages.numel() < 2**31 and tables_shape[1] < 2**31):
        if dev < 0:
            raise RuntimeError("new_lens must be a CUDA tensor")
        _check_ints("new_lens", new_lens, dev)
        _check_ints("lens", lens, dev, batch)
        _check_ints("free_pages", free_pages, dev)
        _check_ints("free_count", free_count, dev, 1)
        _check_tables(block_tables, dev, batch)
        if batch > 8192:
            raise RuntimeError("kv4_schedule takes at most 8192 requests")
        if not (0 <= rows < 2**31 and 0 < page_size < 2**31):
            raise RuntimeError("rows must not be negative, page_size must be positive, both below 2**31")
        if free_pages.numel() >= 2**31 or tables_shape[1] >= 2**31:
            raise RuntimeError("free_pages and the rows of block_tables must have less than 2**31 entries")
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    else:
        _check_ints("lens_out", lens_out, dev, batch)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    else:
        _check_ints("free_count_out", free_count_out, dev, 1)
    device = new_lens.device
    starts = torch.empty(batch + 1, dtype=_INT32, device=device)
    slots = torch.empty(rows, dtype=_INT32, device=device)
    positions = torch.empty(rows, dtype=_INT32, device=device)
    fate = torch.empty_like(lens)
    err = _entry("kv4_schedule")(
        new_lens.data_ptr(), lens.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
        tables_shape[1], batch, free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), rows,
        page_size, lens_out.data_ptr(), free_count_out.data_ptr(), starts.data_ptr(), slots.data_ptr(),
        positions.data_ptr(), fate.data_ptr(), dev, _stream_ptr(dev))
    if err:
        _raise("kv4_schedule", err)
    return KV4Step(lens_out, free_count_out, starts, slots, positions, fate)


def _check_rows(name, t, cache, heads, dim, dev):
    if not t.is_cuda or t.get_device() != dev:
        raise RuntimeError(f"{name} must be a CUDA tensor on device {dev}")
    if t.dtype is not cache.dtype:
        raise RuntimeError(f"{name} must have the cache's dtype {cache.dtype}, got {t.dtype}")
    if t.dim() != 3 or t.size(2) != dim or (heads is not None and t.size(1) != heads):
        raise RuntimeError(f"{name} must be (tokens, {'heads' if heads is None else heads}, {dim})")
    if t.stride(2) != 1:
        raise RuntimeError(f"{name} must have contiguous channels")


def kv4_append(k, v, cache, slots):
    """Quantise keys and values into ``cache`` at ``slots``.

    @k, @v: ``(tokens, kv_heads, head_dim)`` of the cache's type; tokens and
        heads may have any stride (slices of a fused projection's output)
    @slots: ``torch.int`` ``(tokens,)``, no slot twice; rows whose slot is
        outside the cache (-1) are skipped
    """
    fast = _ext._torch_fast if _ext._torch_fast_tried else _ext.torch_fast()
    if fast is not None:
        err = fast.kv4_append(k, v, cache, slots)
        if err == 0:
            return
        if err is not None:
            _raise("kv4_append", err)
    pages, heads, page_size, dim, dtype, dev = _cache_shape(cache)
    shape, k_at, v_at, kind = k.shape, k.stride(), v.stride(), cache.dtype
    tokens = shape[0] if shape else 0
    if not (k.dtype is kind and v.dtype is kind and k.get_device() == dev and v.get_device() == dev
            and shape == (tokens, heads, dim) == v.shape and k_at[2] == 1 and v_at[2] == 1
            and slots.dtype is _INT32 and slots.get_device() == dev and slots.numel() == tokens
            and slots.is_contiguous()):
        _check_rows("k", k, cache, heads, dim, dev)
        _check_rows("v", v, cache, heads, dim, dev)
        if v.size(0) != tokens:
            raise RuntimeError("k and v must have the same number of tokens")
        _check_ints("slots", slots, dev, tokens)
    err = _entry("kv4_append")(
        k.data_ptr(), k_at[0], k_at[1], v.data_ptr(), v_at[0], v_at[1], cache.data_ptr(), pages, heads,
        page_size, dim, dtype, slots.data_ptr(), tokens, dev, _stream_ptr(dev))
    if err:
        _raise("kv4_append", err)


def kv4_read(cache, slots):
    """Keys and values at ``slots``, each ``(tokens, kv_heads, head_dim)`` in the
    cache's type; zeros where a slot is outside the cache.  The two can share one
    allocation."""
    fast = _ext._torch_fast if _ext._torch_fast_tried else _ext.torch_fast()
    if fast is not None:
        done = fast.kv4_read(cache, slots)
        if done is not None:
            if done[0]:
                _raise("kv4_read", done[0])
            return done[1], done[2]
    pages, heads, page_size, dim, dtype, dev = _cache_shape(cache)
    _check_ints("slots", slots, dev)
    tokens = slots.numel()
    k = torch.empty((tokens, heads, dim), dtype=cache.dtype, device=cache.device)
    v = torch.empty_like(k)
    err = _entry("kv4_read")(cache.data_ptr(), pages, heads, page_size, dim, dtype, slots.data_ptr(),
                             tokens, k.data_ptr(), v.data_ptr(), dev, _stream_ptr(dev))
    if err:
        _raise("kv4_read", err)
    return k, v


_workspaces = {}


def kv4_workspace(device="cuda"):
    """A workspace for :func:`kv4_attention` calls that follow one another (its
    first 4096 bytes are zero, and left so by every call)."""
    device = torch.device(device)
    dev = device.index if device.index is not None else torch.cuda.current_device()
    space = torch.empty(max(_ext.load().sm100_marlin_kv4_workspace_bytes(dev), 4096) // 4, dtype=_INT32,
                        device=torch.device("cuda", dev))
    space[:1024].zero_()
    return space


def _capturing(dev):
    """Whether the current stream of ``dev`` is being captured into a graph."""
    if dev == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(dev):
        return torch.cuda.is_current_stream_capturing()


def _workspace(dev, stream):
    # A graph may be replayed beside the stream that it was captured on, and beside
    # other graphs: it gets its own, in its own memory.  (Stream 0 cannot be captured.)
    if stream and _capturing(dev):
        return kv4_workspace(torch.device("cuda", dev))
    found = _workspaces.get((dev, stream))
    if found is None:
        found = _workspaces[dev, stream] = kv4_workspace(torch.device("cuda", dev))
    return found


def _attention_error(err, dev):
    if err == _ext.ERR_SCRATCH:
        need = _ext.load().sm100_marlin_kv4_workspace_bytes(dev) // 4
        raise RuntimeError(f"workspace must be of size at least {need}.")
    _raise("kv4_attention", err)


def kv4_attention(q, cache, block_tables, lens, starts=None, max_new=None, window=0, scale=None,
                  out=None, workspace=None):
    """Attention of each request's last tokens over what it has in the cache.

    Request ``b``'s rows of ``q`` are ``starts[b]:starts[b + 1]``, the last of
    its ``lens[b]`` tokens (append them first); each sees the keys up to its
    own position and, with ``window``, only that many of them.  Rows that see
    nothing and rows of no request are zeros.  Sums are in 32 bits; the weights of
    the values have 11 bits, or 22 for ``torch.half`` with at most 64 rows of a
    request for a key/value head.
    @q: ``(rows, heads, head_dim)`` of the cache's type, ``heads`` a multiple of
        the cache's; rows and heads may have any stride
    @block_tables: ``torch.int`` ``(batch, width)``, @lens: ``torch.int`` ``(batch,)``
    @starts: ``torch.int`` ``(batch + 1,)``; None: one row for each request
    @max_new: no request has more rows than this (default: all of ``q``'s); it
        picks the kernels, so give it for steps of single or few tokens: they are
        slower without.  Rows of a request that has more can be NaN
    @scale: of the scores, default ``1 / sqrt(head_dim)``
    @out: ``(rows, heads, head_dim)``, contiguous
    @workspace: :func:`kv4_workspace`; None: one that the module keeps for the
        current stream, or in a capture one that is the graph's own.  Graphs
        that share a memory pool share it too: do not replay them at once
    """
    fast = _ext._torch_fast if _ext._torch_fast_tried else _ext.torch_fast()
    if fast is not None and out is None and cache.is_cuda:
        space = workspace
        if space is None:
            dev = cache.get_device()
            space = _workspace(dev, _stream_ptr(dev))
        done = fast.kv4_attention(q, cache, block_tables, lens, starts, max_new, window, scale, space)
        if done is not None:
            if done[0]:
                _attention_error(done[0], cache.get_device())
            return done[1]
    pages, heads, page_size, dim, dtype, dev = _cache_shape(cache)
    shape, at, tables_shape, batch = q.shape, q.stride(), block_tables.shape, lens.numel()
    if not (q.dtype is cache.dtype and q.get_device() == dev and len(shape) == 3 and shape[2] == dim
            and at[2] == 1 and lens.dtype is _INT32 and lens.get_device() == dev and lens.is_contiguous()
            and block_tables.dtype is _INT32 and block_tables.get_device() == dev
            and len(tables_shape) == 2 and tables_shape[0] == batch and block_tables.is_contiguous()
            and max(batch, shape[0], tables_shape[1]) < 2**31 - 1):
        _check_rows("q", q, cache, None, dim, dev)
        _check_ints("lens", lens, dev)
        _check_tables(block_tables, dev, batch)
        if max(batch, shape[0], tables_shape[1]) >= 2**31 - 1:
            raise RuntimeError("requests, rows of q and entries of a table must be less than 2**31 - 1")
    rows, q_heads = shape[0], shape[1]
    if q_heads == 0 or q_heads % heads != 0:
        raise RuntimeError(f"q must have a multiple of {heads} heads, got {q_heads}")
    if starts is None:
        if rows != batch:
            raise RuntimeError(f"without starts q must have one row for each of the {batch} requests")
        max_new, starts_at = 1, 0
    else:
        _check_ints("starts", starts, dev, batch + 1)
        max_new, starts_at = rows if max_new is None else max_new, starts.data_ptr()
    if not (0 <= window < 2**31 and 0 <= max_new < 2**31):
        raise ValueError("window and max_new must not be negative, and be below 2**31")
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    else:
        _check_rows("out", out, cache, q_heads, dim, dev)
        if out.size(0) != rows or not out.is_contiguous():
            raise RuntimeError("out must be contiguous and have q's shape")
    stream = _stream_ptr(dev)
    if workspace is None:
        workspace = _workspace(dev, stream)
    else:
        _check_ints("workspace", workspace, dev)
    err = _entry("kv4_attention")(
        q.data_ptr(), at[0], at[1], cache.data_ptr(), pages, heads, page_size, dim, dtype,
        block_tables.data_ptr(), block_tables.stride(0), tables_shape[1], lens.data_ptr(), starts_at,
        batch, rows, q_heads, max_new, window, dim**-0.5 if scale is None else scale, out.data_ptr(),
        workspace.data_ptr(), 4 * workspace.numel(), dev, stream)
    if err:
        _attention_error(err, dev)
    return out
