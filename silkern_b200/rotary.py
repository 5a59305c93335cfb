"""Queries and new keys, before the 8-bit cache stores and asks them.

``rotate_heads``
    The root-mean-square norm of each head's first columns and the rotation of
    some of its columns by position, for queries and keys in one launch. What
    :func:`silkern_b200.append_quantized` stores and the attention operators ask
    comes out of it.
``rotary_frequencies``
    The frequencies that it rotates by, scaled for long contexts or not.

Buffers, streams, errors and gradients are as in :mod:`silkern_b200.attention`,
but that an output may be its own input.
"""

from __future__ import annotations

import ctypes
import math

from silkern_b200 import _native, attention
from silkern_b200.errors import LocalizationError
from silkern_b200.kernels import _compiling, _is_int, _traced_op

#: Most columns of a head.
MOST_COLUMNS = 1024


def rotary_frequencies(
    columns: int,
    *,
    base: float = 10000.0,
    factor: float = 1.0,
    method: str = "none",
    original_length: int | None = None,
    slow: float = 1.0,
    fast: float = 32.0,
    device=None,
):
    """The frequencies of ``columns`` rotary columns, and the amplitude that goes with them.

    Frequency ``i`` of the ``columns // 2`` is ``base ** (-2 i / columns)`` radians
    for each position. ``method`` scales them for contexts ``factor`` times as
    long as those trained on: ``"positions"`` divides all by ``factor``; ``"base"``
    enlarges the base until the lowest frequency is divided by ``factor`` and the
    highest stays; ``"parts"`` divides those that turn fewer than ``slow`` times
    within ``original_length`` positions, keeps those that turn more than ``fast``
    times, and goes linearly in the number of turns from one to the other in between,
    with an amplitude of ``0.1 ln(factor) + 1`` ("YaRN: Efficient Context Window
    Extension of Large Language Models", sections 3.1 to 3.4). Programs that go
    linearly in the column's number between the two bounds get other
    frequencies in between: make those of a model that was trained so by its own
    rule, and pass them to :func:`rotate_heads`, which takes any. Returns
    (float32 tensor of ``columns // 2``, float).
    """
    import torch

    if not _is_int(columns) or columns < 2 or columns % 2:
        raise LocalizationError("rotary columns must be a positive even integer")
    base, factor = float(_number(base, "base")), float(_number(factor, "factor"))
    if base <= 0 or factor < 1:
        raise LocalizationError("base must be positive and factor at least 1")
    if method not in ("none", "positions", "base", "parts"):
        raise LocalizationError('method must be "none", "positions", "base" or "parts"')
    amplitude = 1.0
    if method == "base" and columns > 2:
        try:
            base = base * factor ** (columns / (columns - 2))
        except OverflowError:
            base = math.inf
        if base == math.inf:
            raise LocalizationError("factor is too large for this base")
    # The largest is the first, which is 1, or the last. (On the host: the tensors may be
    # of any default device, or traced.)
    last = (columns - 2) / columns * -math.log(base) - (math.log(factor) if method == "positions" else 0.0)
    if last > math.log(torch.finfo(torch.float32).max):
        raise LocalizationError("base is too small: its frequencies pass float32's range")
    step = torch.arange(0, columns, 2, dtype=torch.float64) / columns
    frequencies = base**-step
    if method == "positions":
        frequencies = frequencies / factor
    elif method == "parts":
        if not _is_int(original_length) or not 1 <= original_length <= 2**31 - 1:
            raise LocalizationError('"parts" needs an original_length, a positive int32 integer')
        try:
            ordered = 0 <= slow < fast
        except (TypeError, ValueError, RuntimeError) as error:
            raise LocalizationError("slow and fast must be numbers") from error
        if not ordered:
            raise LocalizationError('"parts" needs 0 <= slow < fast')
        turns = original_length * frequencies / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        frequencies = frequencies * (keep + (1 - keep) / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    return frequencies.to(torch.float32).to(device), amplitude


def _number(value, name: str) -> float:
    try:
        finite = math.isfinite(value)
    except (TypeError, ValueError, RuntimeError, OverflowError) as error:
        raise LocalizationError(f"{name} must be a finite number") from error
    if not finite:
        raise LocalizationError(f"{name} must be finite")
    return value


def _heads(torch, x, out, weight, dtype, dim, tokens, weight_type, name: str) -> _native.Heads:
    if x.ndim != 3 or x.dtype is not dtype or x.shape[0] != tokens or x.shape[2] != dim or x.shape[1] < 1:
        raise LocalizationError("q and k must be (tokens, heads, dim) of one type, with equal tokens and dim")
    if out.dtype is not dtype or out.shape != x.shape:
        raise LocalizationError(f"{name}_out must have the shape and type of {name}")
    in_token, in_head, in_column = x.stride()
    out_token, out_head, out_column = out.stride()
    if dim > 1 and (in_column != 1 or out_column != 1):
        raise LocalizationError("q, k and their outputs must have unit column stride")
    if x.shape[1] > 65535:
        raise LocalizationError("at most 65535 heads")
    columns = 0
    if weight is not None:
        if weight.ndim != 1 or not 1 <= weight.shape[0] <= dim or not weight.is_contiguous() or weight.dtype is not weight_type:
            raise LocalizationError(
                "weights must be contiguous, of 1 to dim elements, all of one type: float32 or that of q")
        columns = weight.shape[0]
    return _native.Heads(x.data_ptr(), out.data_ptr(), None if weight is None else weight.data_ptr(), in_token, in_head,
                         out_token, out_head, x.shape[1], columns)


def rotate_heads(
    q,
    k,
    positions,
    frequencies,
    q_out,
    k_out,
    *,
    q_weight=None,
    k_weight=None,
    eps: float = 1e-6,
    rotary_start: int = 0,
    interleaved: bool = False,
    amplitude: float = 1.0,
) -> None:
    """Norm and rotate queries and keys.

    ``q`` is (tokens, heads, dim) and ``k`` (tokens, kv_heads, dim) in bfloat16
    or float16 with unit column stride, dim up to 1024; ``k`` and ``k_out`` may be
    ``None``. With a weight, the first ``weight.shape[0]`` columns ``x`` of each
    head become ``x * weight / sqrt(mean(x**2) + eps)`` first. Then the columns
    from ``rotary_start`` on, twice as many as there are ``frequencies`` (float32,
    radians for each position), rotate by ``positions[token] * frequencies[i]``
    (int32, one for each token, of any sign): pair ``i`` is column ``i`` of them
    and the one ``len(frequencies)`` further, or columns ``2 i`` and ``2 i + 1``
    where ``interleaved``. ``amplitude`` multiplies the rotated columns; the others
    stay. Weights are float32 or of the type of ``q``.

    Everything between is float32 with one rounding at the end, and angles are
    worked out in 64 bits, so that far positions keep their precision. ``q_out``
    may be ``q`` itself and ``k_out`` ``k`` itself (the same places, element for
    element); otherwise outputs share no memory with any buffer of the call.
    Views of one fused projection will do: any strides for tokens and heads.
    """
    import torch

    attention._refuse_gradients(torch, q, k, q_out, k_out, q_weight, k_weight, frequencies)
    if _compiling(torch):
        return _traced_op(torch, "rotate_heads")(q, k, positions, frequencies, q_out, k_out, q_weight, k_weight, eps,
                                                 rotary_start, interleaved, amplitude)
    if (k is None) != (k_out is None):
        raise LocalizationError("k and k_out are both given or both None")
    if k is None and k_weight is not None:
        raise LocalizationError("a weight for keys needs keys")
    device = attention._on_device(torch, (q, positions, frequencies, q_out), (k, k_out, q_weight, k_weight), "rotation")
    dtype = q.dtype
    code = attention._type_code(torch, dtype)
    if q.ndim != 3 or q.shape[0] < 1 or not 1 <= q.shape[2] <= MOST_COLUMNS:
        raise LocalizationError(f"q must be (tokens, heads, dim), with a token at least and dim up to {MOST_COLUMNS}")
    tokens, _, dim = q.shape
    weight = q_weight if q_weight is not None else k_weight
    weight_type = dtype if weight is None else weight.dtype
    if weight_type is not dtype and weight_type is not torch.float32:
        raise LocalizationError("weights must be float32 or of the type of q")
    sets = [_heads(torch, q, q_out, q_weight, dtype, dim, tokens, weight_type, "q")]
    if k is not None:
        sets.append(_heads(torch, k, k_out, k_weight, dtype, dim, tokens, weight_type, "k"))
    if positions.dtype is not torch.int32 or positions.shape != (tokens,) or not positions.is_contiguous():
        raise LocalizationError("positions must be contiguous int32, one for each token")
    if frequencies.dtype is not torch.float32 or frequencies.ndim != 1 or not frequencies.is_contiguous():
        raise LocalizationError("frequencies must be contiguous one-dimensional float32")
    pairs = frequencies.shape[0]
    if not _is_int(rotary_start) or pairs < 1 or rotary_start < 0 or rotary_start + 2 * pairs > dim:
        raise LocalizationError("the rotary columns, two for each frequency from rotary_start on, must lie within dim")
    if not isinstance(interleaved, bool):
        raise LocalizationError("interleaved must be a bool")
    _number(amplitude, "amplitude")
    if _number(eps, "eps") < 0:
        raise LocalizationError("eps must not be negative")
    attention._launch(torch, device, "rotate_heads", _native.load().silkern_rotate_heads_v1, ctypes.addressof(sets[0]),
            ctypes.addressof(sets[1]) if k is not None else None, code, tokens, dim, positions.data_ptr(),
            frequencies.data_ptr(), pairs, int(rotary_start), int(interleaved), int(weight_type is torch.float32), amplitude, eps)
