"""``torch.library`` custom ops over the C ABI.

    torch.ops.silkern_b200.localize_rowwise(req_ids, block_table, tokens, out, counts,
                                            block_size, dcp_size, dcp_rank, dcp_interleave,
                                            compact_valid_to_front, num_warps, status)
    torch.ops.silkern_b200.localize_hierarchical(req_ids, block_table, tokens, out, counts,
                                                 mapped, local_positions, tile_counts, tile_offsets,
                                                 block_size, dcp_size, dcp_rank, dcp_interleave,
                                                 compact_valid_to_front, tile_size, num_warps, status)
    torch.ops.silkern_b200.append_quantized, .read_quantized, .rotate_heads, .attend_selected,
                           .attend_window, .attend_shared and .merge_partials,
                                            with the arguments of the launchers, all positional

Each op declares the buffers the kernel writes as mutated (``out``, ``counts``,
the tile workspace and ``status``; the hierarchical op's ``mapped`` and
``local_positions`` are only read for their shapes) and has a fake
implementation, so ``torch.compile`` traces a call as one opaque node, with no
graph break, where the ctypes call of the eager launchers would break the
graph. At run time an op does exactly what the eager launcher does: the
reference's checks, then one C ABI call on the current stream.

The public launchers in :mod:`silkern_b200.kernels`,
:mod:`silkern_b200.attention` and :mod:`silkern_b200.rotary` route through these ops
while ``torch.compile`` traces them and call the C ABI directly otherwise: a
trip through the dispatcher costs tens of microseconds of host time per call,
which an eager caller would pay for nothing.

:func:`register` is idempotent. It runs when :mod:`silkern_b200.kernels` is
imported after torch, and on the first eager launch otherwise; a program that
compiles a call before either should call it first.
"""

# No ``from __future__ import annotations``: torch.library reads the
# annotations below as types to build the op schemas.
from typing import Optional

_REGISTERED = False


def registered() -> bool:
    return _REGISTERED


def register() -> None:
    """Define the ``silkern_b200`` ops (once per process)."""
    global _REGISTERED
    if _REGISTERED:
        return
    import torch

    from silkern_b200 import attention, kernels, rotary

    @torch.library.custom_op("silkern_b200::localize_rowwise", mutates_args=("out", "counts", "status"))
    def localize_rowwise(
        req_ids: torch.Tensor,
        block_table: torch.Tensor,
        tokens: torch.Tensor,
        out: torch.Tensor,
        counts: torch.Tensor,
        block_size: int,
        dcp_size: int,
        dcp_rank: int,
        dcp_interleave: int,
        compact_valid_to_front: bool,
        num_warps: int,
        status: Optional[torch.Tensor],
    ) -> None:
        kernels._rowwise_eager(req_ids, block_table, tokens, out, counts, block_size=block_size,
                               dcp_size=dcp_size, dcp_rank=dcp_rank, dcp_interleave=dcp_interleave,
                               compact_valid_to_front=compact_valid_to_front, num_warps=num_warps,
                               status=status)

    @localize_rowwise.register_fake
    def _(req_ids, block_table, tokens, out, counts, block_size, dcp_size, dcp_rank, dcp_interleave,
          compact_valid_to_front, num_warps, status) -> None:
        return None

    @torch.library.custom_op(
        "silkern_b200::localize_hierarchical",
        mutates_args=("out", "counts", "tile_counts", "tile_offsets", "status"),
    )
    def localize_hierarchical(
        req_ids: torch.Tensor,
        block_table: torch.Tensor,
        tokens: torch.Tensor,
        out: torch.Tensor,
        counts: torch.Tensor,
        mapped: torch.Tensor,
        local_positions: torch.Tensor,
        tile_counts: torch.Tensor,
        tile_offsets: torch.Tensor,
        block_size: int,
        dcp_size: int,
        dcp_rank: int,
        dcp_interleave: int,
        compact_valid_to_front: bool,
        tile_size: int,
        num_warps: int,
        status: Optional[torch.Tensor],
    ) -> None:
        kernels._hierarchical_eager(req_ids, block_table, tokens, out, counts, mapped, local_positions,
                                    tile_counts, tile_offsets, block_size=block_size, dcp_size=dcp_size,
                                    dcp_rank=dcp_rank, dcp_interleave=dcp_interleave,
                                    compact_valid_to_front=compact_valid_to_front, tile_size=tile_size,
                                    num_warps=num_warps, status=status)

    @localize_hierarchical.register_fake
    def _(req_ids, block_table, tokens, out, counts, mapped, local_positions, tile_counts, tile_offsets,
          block_size, dcp_size, dcp_rank, dcp_interleave, compact_valid_to_front, tile_size, num_warps,
          status) -> None:
        return None

    # The cache's launchers take the eager path when they run outside a trace.
    @torch.library.custom_op(
        "silkern_b200::append_quantized", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale", "status")
    )
    def append_quantized(
        keys: torch.Tensor,
        values: Optional[torch.Tensor],
        k_cache: torch.Tensor,
        v_cache: Optional[torch.Tensor],
        k_scale: torch.Tensor,
        v_scale: Optional[torch.Tensor],
        cu_tokens: torch.Tensor,
        starts: torch.Tensor,
        req_ids: torch.Tensor,
        block_table: torch.Tensor,
        dcp_size: int,
        dcp_rank: int,
        dcp_interleave: int,
        status: Optional[torch.Tensor],
    ) -> None:
        attention.append_quantized(keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids,
                                   block_table, dcp_size=dcp_size, dcp_rank=dcp_rank,
                                   dcp_interleave=dcp_interleave, status=status)

    @append_quantized.register_fake
    def _(keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids, block_table, dcp_size,
          dcp_rank, dcp_interleave, status) -> None:
        return None

    @torch.library.custom_op("silkern_b200::read_quantized", mutates_args=("keys", "values", "status"))
    def read_quantized(
        keys: torch.Tensor,
        values: Optional[torch.Tensor],
        k_cache: torch.Tensor,
        v_cache: Optional[torch.Tensor],
        k_scale: torch.Tensor,
        v_scale: Optional[torch.Tensor],
        cu_tokens: torch.Tensor,
        starts: torch.Tensor,
        req_ids: torch.Tensor,
        block_table: torch.Tensor,
        dcp_size: int,
        dcp_rank: int,
        dcp_interleave: int,
        status: Optional[torch.Tensor],
    ) -> None:
        attention.read_quantized(keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids,
                                 block_table, dcp_size=dcp_size, dcp_rank=dcp_rank, dcp_interleave=dcp_interleave,
                                 status=status)

    @read_quantized.register_fake
    def _(keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids, block_table, dcp_size,
          dcp_rank, dcp_interleave, status) -> None:
        return None

    @torch.library.custom_op("silkern_b200::rotate_heads", mutates_args=("q_out", "k_out"))
    def rotate_heads(
        q: torch.Tensor,
        k: Optional[torch.Tensor],
        positions: torch.Tensor,
        frequencies: torch.Tensor,
        q_out: torch.Tensor,
        k_out: Optional[torch.Tensor],
        q_weight: Optional[torch.Tensor],
        k_weight: Optional[torch.Tensor],
        eps: float,
        rotary_start: int,
        interleaved: bool,
        amplitude: float,
    ) -> None:
        rotary.rotate_heads(q, k, positions, frequencies, q_out, k_out, q_weight=q_weight, k_weight=k_weight, eps=eps,
                            rotary_start=rotary_start, interleaved=interleaved, amplitude=amplitude)

    @rotate_heads.register_fake
    def _(q, k, positions, frequencies, q_out, k_out, q_weight, k_weight, eps, rotary_start, interleaved,
          amplitude) -> None:
        return None

    @torch.library.custom_op("silkern_b200::attend_selected", mutates_args=("out", "lse", "status"))
    def attend_selected(
        q: torch.Tensor,
        slots: torch.Tensor,
        k_cache: torch.Tensor,
        v_cache: Optional[torch.Tensor],
        k_scale: torch.Tensor,
        v_scale: Optional[torch.Tensor],
        out: torch.Tensor,
        lse: torch.Tensor,
        softmax_scale: float,
        counts: Optional[torch.Tensor],
        status: Optional[torch.Tensor],
    ) -> None:
        attention.attend_selected(q, slots, k_cache, v_cache, k_scale, v_scale, out, lse,
                                  softmax_scale=softmax_scale, counts=counts, status=status)

    @attend_selected.register_fake
    def _(q, slots, k_cache, v_cache, k_scale, v_scale, out, lse, softmax_scale, counts, status) -> None:
        return None

    @torch.library.custom_op("silkern_b200::attend_window", mutates_args=("out", "lse", "status"))
    def attend_window(
        q: torch.Tensor,
        cu_tokens: torch.Tensor,
        lengths: torch.Tensor,
        req_ids: torch.Tensor,
        block_table: torch.Tensor,
        k_cache: torch.Tensor,
        v_cache: Optional[torch.Tensor],
        k_scale: torch.Tensor,
        v_scale: Optional[torch.Tensor],
        out: torch.Tensor,
        lse: torch.Tensor,
        softmax_scale: float,
        window: int,
        sinks: int,
        dcp_size: int,
        dcp_rank: int,
        dcp_interleave: int,
        status: Optional[torch.Tensor],
    ) -> None:
        attention.attend_window(q, cu_tokens, lengths, req_ids, block_table, k_cache, v_cache, k_scale, v_scale,
                                out, lse, softmax_scale=softmax_scale, window=window, sinks=sinks,
                                dcp_size=dcp_size, dcp_rank=dcp_rank, dcp_interleave=dcp_interleave,
                                status=status)

    @attend_window.register_fake
    def _(q, cu_tokens, lengths, req_ids, block_table, k_cache, v_cache, k_scale, v_scale, out, lse, softmax_scale,
          window, sinks, dcp_size, dcp_rank, dcp_interleave, status) -> None:
        return None

    @torch.library.custom_op("silkern_b200::attend_shared", mutates_args=("out", "lse", "workspace", "status"))
    def attend_shared(
        q: torch.Tensor,
        cu_tokens: torch.Tensor,
        lengths: torch.Tensor,
        req_ids: torch.Tensor,
        cu_groups: torch.Tensor,
        prefixes: torch.Tensor,
        block_table: torch.Tensor,
        k_cache: torch.Tensor,
        v_cache: torch.Tensor,
        k_scale: torch.Tensor,
        v_scale: torch.Tensor,
        out: torch.Tensor,
        lse: torch.Tensor,
        workspace: torch.Tensor,
        softmax_scale: float,
        dcp_size: int,
        dcp_rank: int,
        dcp_interleave: int,
        status: Optional[torch.Tensor],
    ) -> None:
        attention.attend_shared(q, cu_tokens, lengths, req_ids, cu_groups, prefixes, block_table, k_cache, v_cache,
                                k_scale, v_scale, out, lse, workspace, softmax_scale=softmax_scale, dcp_size=dcp_size,
                                dcp_rank=dcp_rank, dcp_interleave=dcp_interleave, status=status)

    @attend_shared.register_fake
    def _(q, cu_tokens, lengths, req_ids, cu_groups, prefixes, block_table, k_cache, v_cache, k_scale, v_scale, out,
          lse, workspace, softmax_scale, dcp_size, dcp_rank, dcp_interleave, status) -> None:
        return None

    @torch.library.custom_op("silkern_b200::merge_partials", mutates_args=("out", "lse"))
    def merge_partials(
        outs: torch.Tensor, lses: torch.Tensor, out: torch.Tensor, lse: Optional[torch.Tensor]
    ) -> None:
        attention.merge_partials(outs, lses, out, lse)

    @merge_partials.register_fake
    def _(outs, lses, out, lse) -> None:
        return None

    _REGISTERED = True
