"""Attention with masks and modified scores, with gradients, and attention over a paged cache.

Argument marshalling over the C ABI, like `ops`, through which these operators are reached.
"""
import ctypes

import torch

from . import _lib
from . import ops as _ops


def _check(t, name, dtype, device, dims, strided=False):
    """A CUDA tensor on `device` of `dims` dimensions; strided: rows of the last dimension contiguous and 16-byte aligned, the other
    strides any."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (ditto_b200 has no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must be {dims}-D, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if not strided:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous (compact row-major)")
    elif t.numel():
        if t.stride(-1) != 1 and t.shape[-1] != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        if t.data_ptr() % 16 or any(n > 1 and (s <= 0 or s % 8) for n, s in zip(t.shape[:-1], t.stride()[:-1])):
            raise ValueError(f"{name}: 16-byte alignment is needed, of the data and of every stride (multiples of 8 elements, above 0): "
                             f"strides {t.stride()}; .contiguous() makes them so")


def _strides(t, kind):
    """Strides in elements of all but the last dimension; those of dimensions of one entry mean nothing and are made valid."""
    return kind(*(s if n > 1 else 8 for n, s in zip(t.shape[:-1], t.stride()[:-1])))


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _element(query, name="query"):
    if not isinstance(query, torch.Tensor) or not query.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (ditto_b200 has no CPU path)")
    if query.dtype not in _ops._DTYPE_CODE:
        raise TypeError(f"{name} dtype {query.dtype} not supported (float16 / bfloat16)")
    return query.dtype


def _check_heads(heads, kv_heads, d):
    if kv_heads == 0 or heads % kv_heads or heads // kv_heads > 128:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key heads (a multiple, at most 128 times as many)")
    if d % 8 or not 0 < d <= 128:
        raise ValueError(f"head dimension {d} not supported (multiples of 8 up to 128)")


def _check_rules(heads, batch, device, scale, cap, slopes, prefix, causal):
    if not scale > 0 or scale == float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if cap is not None and (not cap > 0 or cap == float("inf")):
        raise ValueError(f"cap must be positive and finite, or None, got {cap}")
    if slopes is not None:
        _check(slopes, "slopes", torch.float32, device, 1)
        if slopes.shape[0] != heads:
            raise ValueError(f"slopes must hold {heads} values, got {slopes.shape[0]}")
        if slopes.requires_grad:
            raise ValueError("slopes get no gradient: detach them")
    if prefix is not None:
        if not causal:
            raise ValueError("prefix needs causal=True: without it every query sees the prefix already")
        _check(prefix, "prefix", torch.int32, device, 1)
        if prefix.shape[0] != batch:
            raise ValueError(f"prefix must hold {batch} values, got {prefix.shape[0]}")


def _masked_args(query, key, value, out, lse, scale, causal, prefix, documents, slopes, cap):
    """Checks the operands of a call and returns its argument block (out and lse may be None: to be filled in)."""
    dtype = _element(query)
    device = query.device
    _check(query, "query", dtype, device, 4, strided=True)
    _check(key, "key", dtype, device, 4, strided=True)
    _check(value, "value", dtype, device, 4, strided=True)
    batch, M, heads, d = query.shape
    L, kv_heads = key.shape[1], key.shape[2]
    if tuple(key.shape) != (batch, L, kv_heads, d) or tuple(value.shape) != tuple(key.shape):
        raise ValueError(f"inconsistent shapes: {tuple(query.shape)}, {tuple(key.shape)}, {tuple(value.shape)}")
    _check_heads(heads, kv_heads, d)
    _check_rules(heads, batch, device, scale, cap, slopes, prefix, causal)
    if documents is not None:
        _check(documents, "documents", torch.int32, device, 2)
        if tuple(documents.shape) != (batch, L):
            raise ValueError(f"documents has shape {tuple(documents.shape)}, expected {(batch, L)}: one id a key position")
        if M > L:
            raise ValueError(f"documents: the queries are the last positions of the keys, {M} of {L} cannot be")
    if out is not None:
        _check(out, "out", dtype, device, 4, strided=True)
        if out.shape != query.shape:
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(query.shape)}")
    if lse is not None:
        _check(lse, "lse", torch.float32, device, 3)
        if tuple(lse.shape) != (batch, M, heads):
            raise ValueError(f"lse has shape {tuple(lse.shape)}, expected {(batch, M, heads)}")
    three = _lib.Strides3
    return _lib.MaskedArgs(
        q=_ptr(query), k=_ptr(key), v=_ptr(value), out=_ptr(out), lse=_ptr(lse), q_strides=_strides(query, three),
        k_strides=_strides(key, three), v_strides=_strides(value, three), out_strides=_strides(query if out is None else out, three),
        batch=batch, M=M, L=L, heads=heads, kv_heads=kv_heads, head_dim=d, dtype=_ops._DTYPE_CODE[dtype], causal=1 if causal else 0,
        scale=float(scale), cap=float(cap or 0.0), slopes=_ptr(slopes), prefix=_ptr(prefix), documents=_ptr(documents))


def _workspace(need, device):
    """(tensor, pointer) of `need` bytes from the caching allocator: in stream order, so every call and captured graph has its own."""
    if not need:
        return None, None
    buf = torch.empty(need, dtype=torch.uint8, device=device)
    return buf, buf.data_ptr()


def _forward(query, key, value, out, want_lse, scale, causal, prefix, documents, slopes, cap):
    args = _masked_args(query, key, value, out, None, scale, causal, prefix, documents, slopes, cap)
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        args.out, args.out_strides = out.data_ptr(), _strides(out, _lib.Strides3)
    lse = torch.empty(query.shape[:3], dtype=torch.float32, device=query.device) if want_lse else None
    if out.numel() == 0:
        return out, lse
    if key.shape[1] == 0:                  # nothing to see
        out.zero_()
        if want_lse:
            lse.fill_(float("-inf"))
        return out, lse
    args.lse = _ptr(lse)
    lib = _lib.load()
    with _ops._on_device(query.device):
        need = lib.ditto_b200_masked_workspace_bytes(ctypes.byref(args), 0)
        _buf, ws = _workspace(need, query.device)
        rc = lib.ditto_b200_masked_attention(ctypes.byref(args), ws, need, _ops._status_ptr(query.device),
                                             torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "ditto_b200_masked_attention")
    _ops._enable_fast(query.device)
    _ops.launch_count += 1
    return out, lse


def masked_attention(query, key, value, out=None, scale=1.0, causal=False, prefix=None, documents=None, slopes=None, cap=None,
                     return_lse=False):
    """Attention whose scores may be capped, biased by distance and masked.

    query [batch, M, heads, d]; key, value [batch, L, kv_heads, d], heads a multiple of kv_heads; rows of d contiguous, other
    strides multiples of 8 elements; float16 or bfloat16; d a multiple of 8 up to 128.  Query i stands at position i + L - M.

      s = scale * q . k;   cap: s = cap * tanh(s / cap);   slopes [heads] float32: s -= slopes[h] * |position - j|
      causal: key j is seen by positions from j on, and where prefix [batch] int32 is given by all if j < prefix[b]
      documents [batch, L] int32: only keys of the query's own document are seen; a negative id sees nothing and is not seen

    Returns out [batch, M, heads, d] = softmax over what is seen, times value (0 for a row that sees nothing), and with return_lse also the
    float32 log of the sum of exponentials [batch, M, heads] (-inf for such a row; it gets no gradient).  Gradients of query, key and value
    flow where autograd asks for them (`out` cannot be given then).
    Values that a row does not see have weight 0 and must be finite, padding included; keys that it does not see may be anything here, and must be
    finite where there are gradients.
    """
    if _ops._fast is not None:
        r = _ops._fast.masked(query, key, value, out, scale, causal, prefix, documents, slopes, cap, return_lse)
        if r is not None:
            _ops.launch_count += 1
            return r
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (query, key, value)):
        if out is not None:
            raise ValueError("out cannot be given where gradients are asked for")
        result, lse = _Masked.apply(query, key, value, scale, causal, prefix, documents, slopes, cap)
    else:
        result, lse = _forward(query, key, value, out, return_lse, scale, causal, prefix, documents, slopes, cap)
    return (result, lse) if return_lse else result


def masked_attention_backward(grad_out, query, key, value, out, lse, scale=1.0, causal=False, prefix=None, documents=None, slopes=None,
                              cap=None):
    """Gradients (of query, key, value) of masked_attention from the gradient of its result; out and lse are what it returned for these
    operands and rules.  Sums are taken in a fixed order: the same call gives the same bits."""
    if _ops._fast is not None:
        r = _ops._fast.masked_backward(grad_out, query, key, value, out, lse, scale, causal, prefix, documents, slopes, cap)
        if r is not None:
            _ops.launch_count += 1
            return r
    args = _masked_args(query, key, value, out, lse, scale, causal, prefix, documents, slopes, cap)
    _check(grad_out, "grad_out", query.dtype, query.device, 4, strided=True)
    if grad_out.shape != query.shape:
        raise ValueError(f"grad_out has shape {tuple(grad_out.shape)}, expected {tuple(query.shape)}")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key, value))
    if query.numel() == 0 or key.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    lib = _lib.load()
    with _ops._on_device(query.device):
        need = lib.ditto_b200_masked_workspace_bytes(ctypes.byref(args), 1)
        _buf, ws = _workspace(need, query.device)
        rc = lib.ditto_b200_masked_attention_backward(
            ctypes.byref(args), _ptr(grad_out), _strides(grad_out, _lib.Strides3), _ptr(dq), _ptr(dk), _ptr(dv), ws, need,
            _ops._status_ptr(query.device), torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "ditto_b200_masked_attention_backward")
    _ops._enable_fast(query.device)
    _ops.launch_count += 1
    return dq, dk, dv


class _Masked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, scale, causal, prefix, documents, slopes, cap):
        out, lse = _forward(query, key, value, None, True, scale, causal, prefix, documents, slopes, cap)
        ctx.save_for_backward(query, key, value, out, lse, prefix, documents, slopes)
        ctx.rules = (scale, causal, cap)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, _grad_lse):
        query, key, value, out, lse, prefix, documents, slopes = ctx.saved_tensors
        scale, causal, cap = ctx.rules
        try:
            _check(grad_out, "grad_out", query.dtype, query.device, 4, strided=True)
        except ValueError:                     # an expanded gradient, say that of a sum
            grad_out = grad_out.contiguous()
        grads = masked_attention_backward(grad_out, query, key, value, out, lse, scale, causal, prefix, documents, slopes, cap)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None, None, None)


def _check_cache(key_pages, value_pages, block_table, lengths, query_starts, dtype, device, tokens):
    _check(key_pages, "key_pages", dtype, device, 4, strided=True)
    _check(value_pages, "value_pages", dtype, device, 4, strided=True)
    if key_pages.shape != value_pages.shape:
        raise ValueError(f"inconsistent shapes: {tuple(key_pages.shape)}, {tuple(value_pages.shape)}")
    if key_pages.numel() == 0:
        raise ValueError("the cache has no pages")
    _check_table(block_table, lengths, device)
    batch = lengths.shape[0]
    if query_starts is not None:
        _check(query_starts, "query_starts", torch.int32, device, 1)
        if query_starts.shape[0] != batch + 1:
            raise ValueError(f"query_starts must hold {batch + 1} values, got {query_starts.shape[0]}")
    elif tokens != batch:
        raise ValueError(f"{tokens} tokens for {batch} sequences: query_starts says whose they are")


def _check_table(block_table, lengths, device):
    _check_rows(block_table, device)
    _check(lengths, "lengths", torch.int32, block_table.device, 1)
    if block_table.shape[0] != lengths.shape[0]:
        raise ValueError(f"block_table has {block_table.shape[0]} rows, lengths {lengths.shape[0]} values")


def _check_rows(block_table, device, name="block_table"):
    if not isinstance(block_table, torch.Tensor) or not block_table.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (ditto_b200 has no CPU path)")
    if block_table.dtype != torch.int32:
        raise TypeError(f"{name} has dtype {block_table.dtype}, expected torch.int32")
    if block_table.dim() != 2 or (block_table.numel() and block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError(f"{name} must be 2-D with contiguous rows")
    if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError(f"{name}: rows overlap")
    if device is not None and block_table.device != device:
        raise ValueError(f"{name} is on {block_table.device}, expected {device}")


def paged_attention(query, key_pages, value_pages, block_table, lengths, query_starts=None, out=None, scale=1.0, prefix=None, slopes=None,
                    cap=None):
    """Causal attention of new tokens over a paged cache that holds their keys and values already (cache_append writes them).

    query [tokens, heads, d]: tokens query_starts[b] to query_starts[b + 1] are the last ones of sequence b; without query_starts
    there is one token a sequence.  key_pages, value_pages [pages, page, kv_heads, d], page 16, 32, 64 or a multiple of 128;
    block_table [batch, columns] int32: position j of sequence b is slot j % page of page block_table[b, j // page]; lengths [batch]
    int32 counts a sequence's keys with those of its new tokens.  scale, prefix, slopes and cap as in masked_attention.

    Returns out [tokens, heads, d]; tokens in front of the first sequence or behind the last are left as they are.  Slots behind a
    sequence's end may hold anything.  A page id out of range reads as zeros and shows in device_status(); lengths are cut to what a row of
    the table reaches.  The contents of block_table, lengths and query_starts are read on the device only: a captured call follows them.
    """
    if _ops._fast is not None:
        r = _ops._fast.paged(query, key_pages, value_pages, block_table, lengths, query_starts, out, scale, prefix, slopes, cap)
        if r is not None:
            _ops.launch_count += 1
            return r
    dtype = _element(query)
    device = query.device
    _check(query, "query", dtype, device, 3, strided=True)
    tokens, heads, d = query.shape
    _check_cache(key_pages, value_pages, block_table, lengths, query_starts, dtype, device, tokens)
    pages, page, kv_heads, kd = key_pages.shape
    if kd != d:
        raise ValueError(f"inconsistent shapes: {tuple(query.shape)}, {tuple(key_pages.shape)}")
    if page not in (16, 32, 64) and page % 128:
        raise ValueError(f"pages of {page} positions are not supported (16, 32, 64 or a multiple of 128)")
    batch = lengths.shape[0]
    _check_heads(heads, kv_heads, d)
    _check_rules(heads, batch, device, scale, cap, slopes, prefix, True)
    if out is None:
        # (tokens that belong to no sequence stay as they are: zeros here)
        out = (torch.empty if query_starts is None else torch.zeros)(query.shape, dtype=dtype, device=device)
    else:
        _check(out, "out", dtype, device, 3, strided=True)
        if out.shape != query.shape:
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(query.shape)}")
    if out.numel() == 0 or batch == 0:
        return out
    if block_table.shape[1] == 0:              # no room for any key
        raise ValueError("block_table has no columns")
    two, three = _lib.Strides2, _lib.Strides3
    args = _lib.PagedArgs(
        q=_ptr(query), key_pages=_ptr(key_pages), value_pages=_ptr(value_pages), out=_ptr(out), q_strides=_strides(query, two),
        out_strides=_strides(out, two), key_strides=_strides(key_pages, three), value_strides=_strides(value_pages, three),
        table=_ptr(block_table), lengths=_ptr(lengths), starts=_ptr(query_starts), table_stride=max(block_table.stride(0), 1), tokens=tokens,
        batch=batch, pages=pages, page=page, table_cols=block_table.shape[1], heads=heads, kv_heads=kv_heads, head_dim=d,
        dtype=_ops._DTYPE_CODE[dtype], scale=float(scale), cap=float(cap or 0.0), slopes=_ptr(slopes), prefix=_ptr(prefix))
    lib = _lib.load()
    with _ops._on_device(device):
        need = lib.ditto_b200_paged_workspace_bytes(ctypes.byref(args))
        _buf, ws = _workspace(need, device)
        rc = lib.ditto_b200_paged_attention(ctypes.byref(args), ws, need, _ops._status_ptr(device), torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "ditto_b200_paged_attention")
    _ops._enable_fast(query.device)
    _ops.launch_count += 1
    return out


def cache_append(keys, values, key_pages, value_pages, block_table, lengths, query_starts=None):
    """Writes new tokens' keys and values [tokens, kv_heads, d] (float16 or bfloat16) to their places in the pages.

    Arguments as for paged_attention, which reads them from there: lengths counts the new tokens already.  Tokens whose place has no valid
    page are passed over, which shows in device_status()."""
    if _ops._fast is not None and _ops._fast.append(keys, values, key_pages, value_pages, block_table, lengths, query_starts):
        _ops.launch_count += 1
        return
    dtype = _element(keys, "keys")
    device = keys.device
    _check(keys, "keys", dtype, device, 3, strided=True)
    _check(values, "values", dtype, device, 3, strided=True)
    if keys.shape != values.shape:
        raise ValueError(f"inconsistent shapes: {tuple(keys.shape)}, {tuple(values.shape)}")
    tokens, kv_heads, d = keys.shape
    _check_cache(key_pages, value_pages, block_table, lengths, query_starts, dtype, device, tokens)
    pages, page, h, kd = key_pages.shape
    if (h, kd) != (kv_heads, d):
        raise ValueError(f"inconsistent shapes: {tuple(keys.shape)}, {tuple(key_pages.shape)}")
    if d % 8:
        raise ValueError(f"head dimension {d} not supported (multiples of 8)")
    if keys.numel() == 0 or lengths.shape[0] == 0:
        return
    if block_table.shape[1] == 0:
        raise ValueError("block_table has no columns")
    two, three = _lib.Strides2, _lib.Strides3
    args = _lib.AppendArgs(
        keys=_ptr(keys), values=_ptr(values), key_pages=_ptr(key_pages), value_pages=_ptr(value_pages), k_strides=_strides(keys, two),
        v_strides=_strides(values, two), key_strides=_strides(key_pages, three), value_strides=_strides(value_pages, three),
        table=_ptr(block_table), lengths=_ptr(lengths), starts=_ptr(query_starts), table_stride=max(block_table.stride(0), 1), tokens=tokens,
        batch=lengths.shape[0], pages=pages, page=page, table_cols=block_table.shape[1], kv_heads=kv_heads, head_dim=d)
    lib = _lib.load()
    with _ops._on_device(device):
        rc = lib.ditto_b200_cache_append(ctypes.byref(args), _ops._status_ptr(device), torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "ditto_b200_cache_append")
    _ops._enable_fast(keys.device)
    _ops.launch_count += 1
