"""Attention over an 8-bit paged cache, past the localized selection.

The converter says which physical slots of a rank's cache a query row selected;
the operators here keep that cache and attend to it:

``append_quantized``
    Store new tokens as e4m3 codes, one float32 scale for each page and head.
``attend_selected``
    Attention of each query row over its slots, as
    :func:`silkern_b200.localize_rowwise` and :func:`silkern_b200.topk_localize`
    emit them: padding (-1) anywhere, any order, counts optional.
``attend_window``
    Attention through the block table over a sliding window and a few first
    tokens that stay visible, or over the whole context; one query for each
    sequence or pieces of prompts.
``merge_partials``
    Each rank's output and log-sum-exp over its own tokens, joined.

The cache is a pair of ``torch.float8_e4m3fn`` tensors (num_blocks, block_size,
kv_heads, dim), dim 64 or 128, with scales float32 (num_blocks, kv_heads). A
latent cache is one such tensor with one head and dim 576, whose first 512
columns are the values too: pass ``None`` for its values and value scales. A
page's tokens are consecutive rank-local tokens, owned as the converter's
contract says (silkern/contract.py:8-36).

Every buffer is the caller's; nothing is allocated and nothing synchronises, so
calls can be captured in a CUDA graph. They run on the current stream of the
buffers' device. While ``torch.compile`` traces the caller, each routes through
its op of the same name (:mod:`silkern_b200.ops`). Each raises
:class:`LocalizationError` before launch on an unsupported binding or geometry.
What a call writes shares no memory with what it reads, nor with itself (as an
expanded tensor does), or the call is refused;
buffers that lie between one another's rows, as column slices of one tensor do,
share none (where their largest strides are equal: others are compared as whole
ranges of memory). They are for serving and have no backward pass: while gradients are recorded, a
buffer that requires grad is refused.

Attention expects what :func:`append_quantized` writes: finite codes (no NaN
code, 0x7f or 0xff, at a token that any query of the call sees) and scales that
are 0, NaN or in [2**-100, 2**100].
"""

from __future__ import annotations

import ctypes
import math

from silkern_b200 import _native, ops
from silkern_b200.contract import _validate_dcp_config
from silkern_b200.errors import LocalizationError
from silkern_b200.kernels import _check_status, _compiling, _is_int, _traced_op

#: Dimensions of a latent cache: keys, and the leading part that is the value.
LATENT_KEY_DIM = 576
LATENT_VALUE_DIM = 512
#: Status bits (OR-ed into ``status``) besides SILKERN_STATUS_BAD_REQUEST (1)
#: and STATUS_BAD_LENGTH (2): a slot or page outside the cache, left out; and a
#: wait inside an attention kernel that ran out of its bound, whose results are NaN.
STATUS_BAD_SLOT = 8
STATUS_WAIT_TIMEOUT = 16

_INT32_MAX = 2**31 - 1
_TYPES: dict = {}


def _type_code(torch, dtype):
    if not _TYPES:
        _TYPES.update({torch.bfloat16: 0, torch.float16: 1})
    code = _TYPES.get(dtype)
    if code is None:
        raise LocalizationError("queries, new tokens and outputs must be bfloat16 or float16")
    return code


def _refuse_gradients(torch, *tensors) -> None:
    """The operators have no backward pass; autograd would lose them silently."""
    if torch.is_grad_enabled():
        for t in tensors:
            if getattr(t, "requires_grad", False):
                raise LocalizationError(
                    "no gradient flows through the cache's operators: call them under torch.no_grad() or "
                    "torch.inference_mode(), or detach their buffers")


def _on_device(torch, required, optional, what: str) -> int:
    """The index of the device that the buffers are on: every required one, and
    the optional ones that are not None."""
    device = -1
    host = mixed = False
    tensor = torch.Tensor
    for tensors, may_lack in ((required, False), (optional, True)):
        for t in tensors:
            if t is None and may_lack:
                continue
            if not isinstance(t, tensor):
                raise LocalizationError(f"all {what} buffers must be torch tensors")
            index = t.get_device()
            if index != device or index < 0:
                if not t.is_cuda:
                    host = True
                elif device >= 0:
                    mixed = True
                else:
                    device = index
    if host:
        raise LocalizationError(f"all {what} buffers must be CUDA tensors")
    if mixed:
        raise LocalizationError(f"all {what} buffers must be on the same device")
    return device


def _launch(torch, device: int, what: str, entry, *args) -> None:
    """Call ``entry(*args, stream)`` on the current stream of ``device``."""
    if not ops.registered():
        ops.register()
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device == torch.cuda.current_device():
        code = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            code = entry(*args, stream)
    if code:
        _native.check(code, what)


def _check_ints(torch, tensors, names: str) -> None:
    int32 = torch.int32
    for t in tensors:
        if t is not None and (t.dtype is not int32 or not t.is_contiguous()):
            raise LocalizationError(f"{names} must be contiguous int32 tensors")


def _status_pointer(torch, status, device: int):
    return None if status is None else _check_status(torch, status, torch.device("cuda", device))


def _cache(torch, k_cache, v_cache, k_scale, v_scale) -> _native.Cache:
    """The checked ``silkern_cache_v1`` of a cache's tensors."""
    if (v_cache is None) != (v_scale is None):
        raise LocalizationError("v_cache and v_scale are both given or both None")
    shape = k_cache.shape
    if len(shape) != 4:
        raise LocalizationError("caches must be (num_blocks, block_size, kv_heads, dim)")
    blocks, block_size, kv_heads, dim = shape
    if blocks < 1 or block_size < 1 or kv_heads < 1:
        raise LocalizationError("cache dimensions must be positive")
    if block_size > 65536 or blocks * block_size > _INT32_MAX:
        raise LocalizationError("block_size is at most 65536 and num_blocks * block_size below 2**31")
    if v_cache is None:
        if kv_heads != 1 or dim != LATENT_KEY_DIM:
            raise LocalizationError(
                f"a cache without values is latent: one head and dim {LATENT_KEY_DIM}")
    elif dim not in (64, 128) or v_cache.shape != shape:
        raise LocalizationError("k_cache and v_cache must have the same shape, dim 64 or 128")
    scales = (blocks, kv_heads)
    numbers = []
    for cache, scale in ((k_cache, k_scale), (v_cache, v_scale)):
        if cache is None:
            numbers.append((None, None, 0, 0, 0))
            continue
        if cache.dtype is not torch.float8_e4m3fn:
            raise LocalizationError("caches must use float8_e4m3fn")
        if scale.dtype is not torch.float32 or scale.shape != scales or not scale.is_contiguous():
            raise LocalizationError("scales must be contiguous float32 (num_blocks, kv_heads)")
        sb, st, sh, sd = cache.stride()
        pointer = cache.data_ptr()
        if sd != 1 or (sb | st | sh | pointer) & 15:
            raise LocalizationError(
                "caches need unit column stride, other strides that are multiples of 16 and 16-byte alignment")
        numbers.append((pointer, scale.data_ptr(), sb, st, sh))
    (k, ks, kb, kt, kh), (v, vs, vb, vt, vh) = numbers
    return _native.Cache(k, v, ks, vs, blocks, block_size, kv_heads, dim,
                         LATENT_VALUE_DIM if v_cache is None else dim, kb, kt, kh, vb, vt, vh)


def _check_table(block_table) -> None:
    if block_table.ndim != 2 or block_table.shape[0] < 1 or block_table.shape[1] < 1:
        raise LocalizationError("block_table must be 2D and non-empty")


def _check_owner(block_size, dcp_size, dcp_rank, dcp_interleave) -> None:
    if not (type(dcp_size) is type(dcp_rank) is type(dcp_interleave) is int
            and 0 <= dcp_rank < dcp_size and dcp_interleave > 0):
        _validate_dcp_config(dcp_size, dcp_rank, dcp_interleave)
    if block_size % dcp_interleave:
        raise LocalizationError("the cache's block_size must be divisible by dcp_interleave")
    if dcp_size * dcp_interleave > _INT32_MAX:
        raise LocalizationError("dcp_size * dcp_interleave must be below 2**31")


def _check_scale(softmax_scale) -> None:
    try:
        finite = math.isfinite(softmax_scale)
    except (TypeError, ValueError, RuntimeError) as error:  # RuntimeError: a tensor of several elements
        raise LocalizationError("softmax_scale must be a finite number") from error
    if not finite:
        raise LocalizationError("softmax_scale must be finite")


def _check_queries(torch, q, cache, out, lse, softmax_scale):
    """Checks of an attention call's queries and results: (rows, heads, q's row
    and head stride, out's, type code)."""
    dtype = q.dtype
    code = _type_code(torch, dtype)
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.key_dim:
        raise LocalizationError("q must be (rows, heads, key_dim) with the cache's key_dim")
    rows, heads, _ = shape
    if rows < 1 or heads < 1 or heads > 65535 or heads % cache.kv_heads:
        raise LocalizationError("q needs at least one row, and heads in a positive multiple of the cache's heads")
    out_row, out_head, out_column = out.stride() if out.ndim == 3 else (0, 0, 0)
    if out.dtype is not dtype or out.shape != (rows, heads, cache.value_dim) or out_column != 1:
        raise LocalizationError(f"out must be (rows, heads, {cache.value_dim}) of q's type with unit column stride")
    if lse.dtype is not torch.float32 or lse.shape != (rows, heads) or not lse.is_contiguous():
        raise LocalizationError("lse must be contiguous float32 (rows, heads)")
    q_row, q_head, q_column = q.stride()
    if q_column != 1 or (q_row | q_head) & 7 or q.data_ptr() & 15:
        raise LocalizationError(
            "q needs unit column stride, other strides that are multiples of 8 and 16-byte alignment")
    _check_scale(softmax_scale)
    return rows, heads, q_row, q_head, out_row, out_head, code


def append_quantized(
    keys,
    values,
    k_cache,
    v_cache,
    k_scale,
    v_scale,
    cu_tokens,
    starts,
    req_ids,
    block_table,
    *,
    dcp_size: int = 1,
    dcp_rank: int = 0,
    dcp_interleave: int = 1,
    status=None,
) -> None:
    """Store the new tokens of each sequence in the 8-bit cache.

    ``keys`` is (tokens, kv_heads, key_dim) in bfloat16 or float16, ``values``
    (tokens, kv_heads, value_dim) of the same type, or ``None`` for a latent
    cache; both have unit column stride. Key and value cache may take turns in
    one buffer, page by page or row by row, but share no byte. Sequence ``b`` has the tokens
    ``cu_tokens[b]:cu_tokens[b + 1]`` (int32, one more element than sequences),
    at the positions from ``starts[b]`` on of the request ``req_ids[b]``. The
    positions of this rank go through ``block_table[req_ids[b]]`` into their
    pages; others are skipped.

    Scales are powers of two: with ``m`` the largest magnitude among the call's
    tokens in one page and head, the scale becomes the larger of what it was
    and the smallest power of two ``w`` with ``448 w >= m`` (within 2**-100 and
    2**100). A page whose first token is among the call's is new: its old scale
    does not count, so pages need no clearing before they are used again.
    Where the scale of a page grows, the codes that it holds are rescaled. An
    infinity or NaN among a page's new values makes the scale NaN, and so
    everything read from that page and head, until the page is new again.

    A page takes tokens from one sequence of a call at most: copy a page that
    several requests share before one of them appends to it. ``status`` gets 1
    for a request id outside the table, 2 for a sequence that starts below 0
    or ends past position 2**31 - 2, 8 for a token whose page is outside its table row or the cache; such
    tokens are not stored.
    """
    import torch

    _refuse_gradients(torch, keys, values, k_cache, v_cache, k_scale, v_scale)
    if _compiling(torch):
        return _traced_op(torch, "append_quantized")(
            keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids, block_table, dcp_size,
            dcp_rank, dcp_interleave, status)
    device = _on_device(torch, (keys, k_cache, k_scale, cu_tokens, starts, req_ids, block_table),
                        (values, v_cache, v_scale), "append")
    code = _type_code(torch, keys.dtype)
    _check_ints(torch, (cu_tokens, starts, req_ids, block_table), "cu_tokens, starts, req_ids and block_table")
    cache = _cache(torch, k_cache, v_cache, k_scale, v_scale)
    if (values is None) != (v_cache is None):
        raise LocalizationError("values are given exactly when the cache has values")
    tokens = keys.shape[0] if keys.ndim == 3 else 0
    wanted = (tokens, cache.kv_heads, cache.key_dim)
    places = []
    for new in (keys, values):
        if new is None:
            places += (None, 0, 0)
            continue
        row, head, column = new.stride() if new.ndim == 3 else (0, 0, 0)
        if new.dtype is not keys.dtype or new.shape != wanted or tokens < 1 or column != 1:
            raise LocalizationError(
                "keys and values must be (tokens, kv_heads, dim) of one type with unit column stride")
        places += (new.data_ptr(), row, head)
    sequences = starts.shape[0] if starts.ndim == 1 else 0
    if sequences < 1 or cu_tokens.shape != (sequences + 1,) or req_ids.shape != (sequences,):
        raise LocalizationError("starts and req_ids need one element per sequence, cu_tokens one more")
    _check_table(block_table)
    _check_owner(cache.block_size, dcp_size, dcp_rank, dcp_interleave)
    status_ptr = _status_pointer(torch, status, device)
    table_rows, table_width = block_table.shape
    _launch(torch, device, "append_quantized", _native.load().silkern_append_quantized_v1,
            ctypes.addressof(cache), *places, code, tokens, cu_tokens.data_ptr(), starts.data_ptr(),
            req_ids.data_ptr(), sequences, block_table.data_ptr(), table_rows, table_width, int(dcp_size),
            int(dcp_rank), int(dcp_interleave), status_ptr)


def attend_selected(
    q,
    slots,
    k_cache,
    v_cache,
    k_scale,
    v_scale,
    out,
    lse,
    *,
    softmax_scale: float,
    counts=None,
    status=None,
) -> None:
    """Attention of each query row over the cache slots selected for it.

    ``q`` is (rows, heads, key_dim) in bfloat16 or float16, its address and
    strides multiples of 16 bytes; ``out`` (rows, heads, value_dim) of the same
    type, ``lse`` float32 (rows, heads). Query head ``h`` reads cache head
    ``h // (heads // kv_heads)``. ``slots`` is int32 (rows, width) with unit
    column stride: what the converter writes. Negative slots are padding and
    may stand anywhere; with ``counts`` (int32, (rows,)) only the first
    ``counts[r]`` columns of row ``r`` are looked at, which is right for
    compacted rows. A slot that is listed twice counts twice.

    ``lse`` is the natural log of the sum of ``exp(softmax_scale * q . k)``, for
    :func:`merge_partials`. A row without a slot gets output 0 and lse -inf.
    ``status`` gets 2 for a count outside the row (clamped), 8 for a slot past
    the cache (left out) and 16 for a wait inside the kernel that ran out, whose
    results are NaN (it does not occur in a working launch).

    Keys are shared among the GPU's SMs by the number of rows and heads and by
    the width, not by the counts: where rows times cache heads exceed half the
    SMs, each row's keys of a head are read by one SM. Call few very long rows
    apart from many short ones.
    """
    import torch

    _refuse_gradients(torch, q, k_cache, v_cache, k_scale, v_scale, out, lse)
    if _compiling(torch):
        return _traced_op(torch, "attend_selected")(
            q, slots, k_cache, v_cache, k_scale, v_scale, out, lse, softmax_scale, counts, status)
    device = _on_device(torch, (q, slots, k_cache, k_scale, out, lse), (v_cache, v_scale, counts), "attention")
    _check_ints(torch, (counts,), "counts")
    cache = _cache(torch, k_cache, v_cache, k_scale, v_scale)
    rows, heads, q_row, q_head, out_row, out_head, code = _check_queries(torch, q, cache, out, lse, softmax_scale)
    if slots.dtype is not torch.int32 or slots.ndim != 2 or slots.shape[0] != rows or slots.shape[1] < 1:
        raise LocalizationError("slots must be int32 with one non-empty row for each row of q")
    slots_row, slots_column = slots.stride()
    width = slots.shape[1]
    if slots_column != 1 and width > 1:
        raise LocalizationError("slots must have unit column stride")
    if counts is not None and counts.shape != (rows,):
        raise LocalizationError("counts must contain one element per row")
    status_ptr = _status_pointer(torch, status, device)
    _launch(torch, device, "attend_selected", _native.load().silkern_attend_selected_v1,
            ctypes.addressof(cache), q.data_ptr(), q_row, q_head, code, rows, heads, slots.data_ptr(), slots_row,
            width, None if counts is None else counts.data_ptr(), out.data_ptr(), out_row, out_head,
            lse.data_ptr(), softmax_scale, status_ptr)


def attend_window(
    q,
    cu_tokens,
    lengths,
    req_ids,
    block_table,
    k_cache,
    v_cache,
    k_scale,
    v_scale,
    out,
    lse,
    *,
    softmax_scale: float,
    window: int = 0,
    sinks: int = 0,
    dcp_size: int = 1,
    dcp_rank: int = 0,
    dcp_interleave: int = 1,
    status=None,
) -> None:
    """Attention through the block table, over a window and the first tokens.

    Sequence ``b`` has the queries ``cu_tokens[b]:cu_tokens[b + 1]`` of ``q``
    (int32, one more element than sequences): the last tokens of the request
    ``req_ids[b]``, which is ``lengths[b]`` tokens long with them. The query at
    position ``t`` sees the positions ``max(0, t + 1 - window)`` to ``t`` and
    the first ``sinks`` positions up to ``t``; with ``window`` 0 it sees all up
    to ``t``. Of these it attends to the ones that this rank owns. Queries at
    one position of each sequence (decode) and pieces of prompts take the same
    call; rows of ``q`` at and past ``cu_tokens[-1]`` are left as they were in
    ``out`` and ``lse``.

    Layouts, types and results are those of :func:`attend_selected`. A query
    that sees none of this rank's tokens gets output 0 and lse -inf. ``status``
    gets 1 for a request id outside the table (its queries see nothing), 2 for
    a length below the number of queries (those at negative positions see
    nothing), 8 for a visible token whose page is outside the table row or the
    cache (left out) and 16 as in :func:`attend_selected`, whose sharing of the
    keys holds as well: one sequence of 131072 tokens takes 82 us alone, and 673
    among 15 of 1000, with 8 cache heads. Call long sequences apart.
    """
    import torch

    _refuse_gradients(torch, q, k_cache, v_cache, k_scale, v_scale, out, lse)
    if _compiling(torch):
        return _traced_op(torch, "attend_window")(
            q, cu_tokens, lengths, req_ids, block_table, k_cache, v_cache, k_scale, v_scale, out, lse,
            softmax_scale, window, sinks, dcp_size, dcp_rank, dcp_interleave, status)
    device = _on_device(torch, (q, cu_tokens, lengths, req_ids, block_table, k_cache, k_scale, out, lse),
                        (v_cache, v_scale), "attention")
    _check_ints(torch, (cu_tokens, lengths, req_ids, block_table), "cu_tokens, lengths, req_ids and block_table")
    cache = _cache(torch, k_cache, v_cache, k_scale, v_scale)
    rows, heads, q_row, q_head, out_row, out_head, code = _check_queries(torch, q, cache, out, lse, softmax_scale)
    sequences = lengths.shape[0] if lengths.ndim == 1 else 0
    if sequences < 1 or cu_tokens.shape != (sequences + 1,) or req_ids.shape != (sequences,):
        raise LocalizationError("lengths and req_ids need one element per sequence, cu_tokens one more")
    _check_table(block_table)
    _check_owner(cache.block_size, dcp_size, dcp_rank, dcp_interleave)
    if not _is_int(window) or not 0 <= window <= _INT32_MAX or not _is_int(sinks) or not 0 <= sinks <= _INT32_MAX:
        raise LocalizationError("window and sinks must be non-negative int32 integers")
    status_ptr = _status_pointer(torch, status, device)
    table_rows, table_width = block_table.shape
    _launch(torch, device, "attend_window", _native.load().silkern_attend_window_v1,
            ctypes.addressof(cache), q.data_ptr(), q_row, q_head, code, rows, heads, cu_tokens.data_ptr(),
            lengths.data_ptr(), req_ids.data_ptr(), sequences, block_table.data_ptr(), table_rows, table_width,
            int(window), int(sinks), int(dcp_size), int(dcp_rank), int(dcp_interleave), out.data_ptr(), out_row,
            out_head, lse.data_ptr(), softmax_scale, status_ptr)


def merge_partials(outs, lses, out, lse=None) -> None:
    """Join the ranks' partial attention results into the whole one.

    ``outs`` is (ranks, rows, heads, dim) in bfloat16 or float16 with unit
    column stride, ``lses`` contiguous float32 (ranks, rows, heads): each rank's
    :func:`attend_selected` or :func:`attend_window` over its own tokens.
    ``out`` (rows, heads, dim) becomes the average of the partial outputs
    weighted by ``exp(lses)``, ``lse`` (optional, float32 (rows, heads)) the log
    of the weights' sum. A partial result with lse -inf is not read; where every
    rank's is, out is 0 and lse -inf. The ranks are added in order.
    """
    import torch

    _refuse_gradients(torch, outs, lses, out, lse)
    if _compiling(torch):
        return _traced_op(torch, "merge_partials")(outs, lses, out, lse)
    device = _on_device(torch, (outs, lses, out), (lse,), "merge")
    dtype = outs.dtype
    code = _type_code(torch, dtype)
    if outs.ndim != 4 or outs.numel() < 1:
        raise LocalizationError("outs must be a non-empty (ranks, rows, heads, dim)")
    ranks, rows, heads, dim = outs.shape
    if out.dtype is not dtype or out.shape != (rows, heads, dim):
        raise LocalizationError("out must be (rows, heads, dim) of the type of outs")
    in_rank, in_row, in_head, in_column = outs.stride()
    out_row, out_head, out_column = out.stride()
    if dim > 1 and (in_column != 1 or out_column != 1):
        raise LocalizationError("outs and out must have unit column stride")
    if lses.dtype is not torch.float32 or lses.shape != (ranks, rows, heads) or not lses.is_contiguous():
        raise LocalizationError("lses must be contiguous float32 (ranks, rows, heads)")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (rows, heads) or not lse.is_contiguous()):
        raise LocalizationError("lse must be contiguous float32 (rows, heads)")
    _launch(torch, device, "merge_partials", _native.load().silkern_merge_partials_v1,
            outs.data_ptr(), in_rank, in_row, in_head, lses.data_ptr(), code, ranks, rows, heads, dim,
            out.data_ptr(), out_row, out_head, None if lse is None else lse.data_ptr())
