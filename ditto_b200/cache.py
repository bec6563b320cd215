"""Page operations of a paged key/value cache: reserving, copying, forking, freeing and compacting pages.

Argument marshalling over the C ABI, like `ops`, through which these operators are reached.  A cache is
  pools        tensors [pages, ...] that share one numbering of pages: the keys and the values of every layer
  block_table  [sequences, columns] int32, the pages of each sequence in order, -1 where it has none
  lengths      [sequences] int32, positions in use
  references   [pages] int32, how many entries of the table name a page: 0 for a free one
All of it is read and written on the device in stream order: the calls can be captured, and nothing waits for the host.  Free pages are
taken lowest first, so the same tables give the same tables.  What a call cannot do shows in device_status().
"""
import ctypes

import torch

from . import _lib
from . import masked as _masked
from . import ops as _ops


def _tables(block_table, lengths, references, page_size):
    _masked._check_table(block_table, lengths, None)
    _masked._check(references, "references", torch.int32, block_table.device, 1)
    if page_size is not None and page_size < 1:
        raise ValueError(f"page_size must be positive, got {page_size}")
    return _lib.TablesArgs(table=block_table.data_ptr(), lengths=lengths.data_ptr(), references=references.data_ptr(),
                           stride=max(block_table.stride(0), block_table.shape[1]), sequences=block_table.shape[0], cols=block_table.shape[1],
                           page=page_size or 0, pages=references.shape[0])


def _pools(pools, pages, device):
    """The pools' argument block, with the array of addresses that has to outlive the call."""
    if isinstance(pools, torch.Tensor):
        pools = (pools,)
    if not pools:
        raise ValueError("no pools")
    first = pools[0]
    for t in pools:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError("pools must be CUDA tensors (ditto_b200 has no CPU path)")
        if t.device != (device or first.device):
            raise ValueError(f"a pool is on {t.device}, expected {device or first.device}")
        if t.dim() < 2 or t.shape != first.shape or t.dtype != first.dtype or t.stride() != first.stride():
            raise ValueError("pools must be tensors [pages, ...] of one shape, type and stride")
        if pages is not None and t.shape[0] != pages:
            raise ValueError(f"a pool has {t.shape[0]} pages, references {pages}")
        if t.data_ptr() % 16:
            raise ValueError("pools must be aligned to 16 bytes")
    if first.shape[0] and not first[0].is_contiguous():
        raise ValueError("a page must be contiguous")
    page_bytes, stride = first[0].numel() * first.element_size() if first.shape[0] else 0, first.stride(0) * first.element_size()
    if first.shape[0] == 1:
        stride = page_bytes
    if page_bytes == 0 or page_bytes % 16 or stride % 16 or stride < page_bytes:
        raise ValueError(f"pages of {page_bytes} bytes, {stride} apart, are not supported (multiples of 16, not overlapping)")
    base = (ctypes.c_void_p * len(pools))(*(t.data_ptr() for t in pools))
    return _lib.PoolsArgs(base=ctypes.cast(base, ctypes.c_void_p), count=len(pools), pages=first.shape[0], page_bytes=page_bytes,
                          stride_bytes=stride), base


def _ids(t, name, device):
    _masked._check(t, name, torch.int32, device, 1)
    return t.shape[0]


def _call(name, device, *args):
    lib = _lib.load()
    with _ops._on_device(device):
        rc = getattr(lib, name)(*args, _ops._status_ptr(device), torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, name)
    _ops._enable_fast(device)
    _ops.launch_count += 1


def _scratch(tables, n, device):
    need = _lib.load().ditto_b200_cache_workspace_bytes(ctypes.byref(tables), n)
    buf, ptr = _masked._workspace(need, device)
    return buf, ptr, need


def cache_copy(pools, source, target):
    """Copies page source[i] to page target[i] in every pool (int32, on the device; a negative id: no copy).  No target may be another target
    or a source; ids out of range are passed over."""
    n = _ids(source, "source", None)
    if _ids(target, "target", source.device) != n:
        raise ValueError(f"{n} sources, {target.shape[0]} targets")
    args, _base = _pools(pools, None, source.device)
    if n:
        _call("ditto_b200_cache_copy", source.device, ctypes.byref(args), source.data_ptr(), target.data_ptr(), n)


def cache_reserve(block_table, lengths, references, counts, page_size):
    """lengths += counts, with the new pages that takes in the table and in references.  All or nothing: without enough free pages or columns
    nothing changes, and device_status() is STATUS_NO_PAGES."""
    t = _tables(block_table, lengths, references, page_size)
    if _ids(counts, "counts", block_table.device) != t.sequences:
        raise ValueError(f"counts must hold {t.sequences} values, got {counts.shape[0]}")
    if t.sequences == 0:
        return
    _not_empty(t)
    _buf, ptr, need = _scratch(t, 0, block_table.device)
    _call("ditto_b200_cache_reserve", block_table.device, ctypes.byref(t), counts.data_ptr(), ptr, need)


def _not_empty(t):
    if t.cols == 0 or t.pages == 0:
        raise ValueError("block_table has no columns, or references no pages")


def cache_fork(pools, block_table, lengths, references, parents, children, page_size):
    """Sequence children[i] becomes a copy of sequence parents[i] (int32, on the device): it shares the full pages and gets a copy of a last page
    that is not full, in the lowest free page.  Children are sequences without pages, all different, none a parent; a parent may have any
    number of them.  All or nothing as in cache_reserve."""
    if _ops._fast is not None and _ops._fast.cache_fork(pools, block_table, lengths, references, parents, children, page_size):
        _ops.launch_count += 1
        return
    t = _tables(block_table, lengths, references, page_size)
    device = block_table.device
    n = _ids(parents, "parents", device)
    if _ids(children, "children", device) != n:
        raise ValueError(f"{n} parents, {children.shape[0]} children")
    args, _base = _pools(pools, t.pages, device)
    if n == 0:
        return
    if n > t.sequences:
        raise ValueError(f"{n} children of {t.sequences} sequences cannot all be different")
    _not_empty(t)
    _buf, ptr, need = _scratch(t, n, device)
    _call("ditto_b200_cache_fork", device, ctypes.byref(args), ctypes.byref(t), parents.data_ptr(), children.data_ptr(), n, ptr, need)


def cache_free(block_table, lengths, references, sequences):
    """Gives back the pages of the sequences (int32, on the device): rows become -1, lengths 0.  A sequence that is named twice is freed once."""
    if _ops._fast is not None and _ops._fast.cache_free(block_table, lengths, references, sequences):
        _ops.launch_count += 1
        return
    t = _tables(block_table, lengths, references, None)
    n = _ids(sequences, "sequences", block_table.device)
    if n and t.sequences:
        _not_empty(t)
        _call("ditto_b200_cache_free", block_table.device, ctypes.byref(t), sequences.data_ptr(), n)


def cache_compact(pools, block_table, references, out_table=None, out_references=None):
    """Moves the live pages to the front of the pools and returns the table and the references that go with it (new tensors, or out_table and
    out_references, which may be the old ones).  With n live pages the k-th of those behind the first n goes to the k-th free place among
    them; the pages that are left keep their contents."""
    if _ops._fast is not None and out_table is None and out_references is None:
        r = _ops._fast.cache_compact(pools, block_table, references)
        if r is not None:
            _ops.launch_count += 1
            return r
    _masked._check_rows(block_table, None)
    device = block_table.device
    _masked._check(references, "references", torch.int32, device, 1)
    args, _base = _pools(pools, references.shape[0], device)
    if out_table is None:
        out_table = torch.empty(block_table.shape, dtype=torch.int32, device=device)
    else:
        _masked._check_rows(out_table, device, "out_table")
        if out_table.shape != block_table.shape:
            raise ValueError(f"out_table has shape {tuple(out_table.shape)}, expected {tuple(block_table.shape)}")
    if out_references is None:
        out_references = torch.empty(references.shape, dtype=torch.int32, device=device)
    else:
        _masked._check(out_references, "out_references", torch.int32, device, 1)
        if out_references.shape != references.shape:
            raise ValueError(f"out_references has shape {tuple(out_references.shape)}, expected {tuple(references.shape)}")
    sequences, cols = block_table.shape
    if sequences == 0 or cols == 0:
        raise ValueError("block_table is empty")
    t = _lib.TablesArgs(table=block_table.data_ptr(), lengths=None, references=references.data_ptr(), stride=max(block_table.stride(0), cols),
                        sequences=sequences, cols=cols, page=0, pages=references.shape[0])
    _buf, ptr, need = _scratch(t, 0, device)
    _call("ditto_b200_cache_compact", device, ctypes.byref(args), ctypes.byref(t), out_table.data_ptr(), max(out_table.stride(0), cols),
          out_references.data_ptr(), ptr, need)
    return out_table, out_references
