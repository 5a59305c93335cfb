"""The 8-bit cache's operators in 64 bits, row by row: the oracle of the CUDA kernels.

Test infrastructure only. Everything is computed by torch in float64 on the
tensors' own device, from the operators' definitions.
"""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def owned(position, dcp_size, dcp_rank, dcp_interleave):
    """(mask of this rank's positions, their rank-local tokens) of an int64 tensor."""
    run = position // dcp_interleave
    local = run // dcp_size * dcp_interleave + position % dcp_interleave
    return run % dcp_size == dcp_rank, local


def append(keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids, block_table, *,
           dcp_size=1, dcp_rank=0, dcp_interleave=1):
    """Copies of (k_cache, v_cache, k_scale, v_scale) with the new tokens in place."""
    results = []
    block_size = k_cache.shape[1]
    cu, first, req, table = (t.tolist() for t in (cu_tokens, starts, req_ids, block_table))
    for new, cache, scale in ((keys, k_cache, k_scale), (values, v_cache, v_scale)):
        if cache is None:
            results.append((None, None))
            continue
        cache, scale = cache.clone(), scale.clone()
        for b in range(len(first)):
            rows = torch.arange(cu[b], cu[b + 1], device=cache.device)
            mine, local = owned(rows - cu[b] + first[b], dcp_size, dcp_rank, dcp_interleave)
            rows, local = rows[mine], local[mine]
            for page in torch.unique(local // block_size).tolist():
                here = local // block_size == page
                block, offset = table[req[b]][page], local[here] % block_size
                for head in range(cache.shape[2]):
                    x = new[rows[here], head].double()
                    most = float(x.abs().max())
                    old = 0.0 if int(offset[0]) == 0 else float(scale[block, head])
                    if not math.isfinite(most) or math.isnan(old):
                        scale[block, head] = math.nan
                        cache[block, offset, head] = torch.zeros_like(x).to(cache.dtype)
                        continue
                    want = 0.0
                    if most > 0:
                        want = 2.0 ** min(max(math.ceil(math.log2(most / E4M3_MAX)), -100), 100)
                        if want < 2.0**100 and want * E4M3_MAX < most:  # log2 rounded
                            want *= 2
                        if want > 2.0**-100 and want / 2 * E4M3_MAX >= most:
                            want /= 2
                    use = max(old, want)
                    if use > old and int(offset[0]) != 0:
                        rest = torch.ones(block_size, dtype=torch.bool, device=cache.device)
                        rest[offset] = False
                        held = cache[block, rest, head].float().double() * (old / use)
                        cache[block, rest, head] = held.float().to(cache.dtype)
                    codes = (x / use if use > 0 else x * 0).clamp(-E4M3_MAX, E4M3_MAX)
                    cache[block, offset, head] = codes.float().to(cache.dtype)
                    scale[block, head] = use
        results.append((cache, scale))
    (k, ks), (v, vs) = results
    return k, v, ks, vs


def read(keys, values, k_cache, v_cache, k_scale, v_scale, cu_tokens, starts, req_ids, block_table, *,
         dcp_size=1, dcp_rank=0, dcp_interleave=1):
    """Float64 copies of (keys, values) with the stored tokens in place."""
    results = []
    block_size = k_cache.shape[1]
    cu, first, req = (t.tolist() for t in (cu_tokens, starts, req_ids))
    for new, cache, scale in ((keys, k_cache, k_scale), (values, v_cache, v_scale)):
        if cache is None:
            results.append(None)
            continue
        new = new.double().clone()
        for b in range(len(first)):
            if not 0 <= req[b] < block_table.shape[0] or first[b] < 0:
                continue
            rows = torch.arange(cu[b], cu[b + 1], device=cache.device)
            mine, local = owned(rows - cu[b] + first[b], dcp_size, dcp_rank, dcp_interleave)
            mine &= local // block_size < block_table.shape[1]
            rows, local = rows[mine], local[mine]
            block = block_table[req[b]].long()[local // block_size]
            good = (block >= 0) & (block < cache.shape[0])
            rows, local, block = rows[good], local[good], block[good]
            new[rows] = cache[block, local % block_size].float().double() * scale[block].double()[:, :, None]
        results.append(new)
    return tuple(results)


def attend_row(q, slot, k_cache, v_cache, k_scale, v_scale, softmax_scale):
    """One query row (heads, dim) over its int64 slots: (out, lse, spread, near).

    ``spread`` (heads, value_dim) is the weighted mean of the values'
    magnitudes: an error of relative size u in each weight moves ``out`` by at
    most ``u * spread``. ``near`` is the same with each weight replaced by the
    largest among its neighbours, up to 127 places away: an error of u times
    the largest weight of a weight's run of 128 moves ``out`` by at most
    ``u * near``."""
    heads, kv_heads = q.shape[0], k_cache.shape[2]
    value_dim = 512 if v_cache is None else v_cache.shape[3]
    if slot.numel() == 0:
        zero = torch.zeros((heads, value_dim), dtype=torch.float64, device=q.device)
        return zero, torch.full((heads,), -math.inf, dtype=torch.float64, device=q.device), zero, zero
    block, offset = slot // k_cache.shape[1], slot % k_cache.shape[1]
    k = k_cache[block, offset].float().double() * k_scale[block].double()[:, :, None]
    v = k[:, :, :value_dim] if v_cache is None else (
        v_cache[block, offset].float().double() * v_scale[block].double()[:, :, None])
    grouped = q.double().reshape(kv_heads, heads // kv_heads, -1)
    score = torch.einsum("hgd,nhd->hgn", grouped, k) * softmax_scale
    lse = torch.logsumexp(score, dim=-1)
    weight = torch.exp(score - lse[..., None])
    out = torch.einsum("hgn,nhd->hgd", weight, v)
    spread = torch.einsum("hgn,nhd->hgd", weight, v.abs())
    around = torch.nn.functional.max_pool1d(weight, 255, stride=1, padding=127)
    near = torch.einsum("hgn,nhd->hgd", around, v.abs())
    return out.reshape(heads, value_dim), lse.reshape(heads), spread.reshape(heads, value_dim), near.reshape(heads, value_dim)


def attend_selected(q, slots, k_cache, v_cache, k_scale, v_scale, *, softmax_scale, counts=None):
    total = k_cache.shape[0] * k_cache.shape[1]
    rows = []
    for r in range(q.shape[0]):
        s = slots[r].long()
        if counts is not None:
            s = s[: min(max(int(counts[r]), 0), slots.shape[1])]
        s = s[(s >= 0) & (s < total)]
        rows.append(attend_row(q[r], s, k_cache, v_cache, k_scale, v_scale, softmax_scale))
    return tuple(torch.stack(part) for part in zip(*rows))


def attend_window(q, cu_tokens, lengths, req_ids, block_table, k_cache, v_cache, k_scale, v_scale, *,
                  softmax_scale, window=0, sinks=0, dcp_size=1, dcp_rank=0, dcp_interleave=1):
    """(out, lse, spread, near) of the rows below cu_tokens[-1]."""
    rows = []
    block_size = k_cache.shape[1]
    cu, length, req = (t.tolist() for t in (cu_tokens, lengths, req_ids))
    for b in range(len(length)):
        for i in range(cu[b], cu[b + 1]):
            last = length[b] - (cu[b + 1] - i)
            position = torch.arange(max(last + 1, 0), device=q.device)
            if window:
                position = position[(position > last - window) | (position < sinks)]
            mine, local = owned(position, dcp_size, dcp_rank, dcp_interleave)
            local = local[mine]
            slot = torch.empty(0, dtype=torch.int64, device=q.device)
            if 0 <= req[b] < block_table.shape[0]:
                local = local[local // block_size < block_table.shape[1]]
                block = block_table[req[b]].long()[local // block_size]
                good = (block >= 0) & (block < k_cache.shape[0])
                slot = (block * block_size + local % block_size)[good]
            rows.append(attend_row(q[i], slot, k_cache, v_cache, k_scale, v_scale, softmax_scale))
    return tuple(torch.stack(part) for part in zip(*rows))


def attend_shared(q, cu_tokens, lengths, req_ids, cu_groups, prefixes, block_table, k_cache, v_cache, k_scale, v_scale, *,
                  softmax_scale, dcp_size=1, dcp_rank=0, dcp_interleave=1):
    """(out, lse, spread, peak) of the rows in [cu_tokens[0], cu_tokens[-1]). ``peak`` (rows, heads,
    value_dim) is a row's largest product of weight and value scale, times the sum of its codes' magnitudes."""
    rows = []
    block_size, heads, kv_heads = k_cache.shape[1], q.shape[1], k_cache.shape[2]
    cu, length, req, cut, prefix = (t.tolist() for t in (cu_tokens, lengths, req_ids, cu_groups, prefixes))
    for b in range(len(length)):
        group = next((g for g in range(len(prefix)) if cut[g] <= b < cut[g + 1]), None)
        for i in range(cu[b], cu[b + 1]):
            last = length[b] - (cu[b + 1] - i)
            position = torch.arange(max(last + 1, 0), device=q.device)
            slots = []
            for behind in (False, True):
                leader = req[b] if group is None or behind else req[cut[group]]
                inside = position < (0 if group is None else prefix[group])
                mine, local = owned(position, dcp_size, dcp_rank, dcp_interleave)
                local = local[mine & (~inside if behind else inside)]
                if 0 <= leader < block_table.shape[0]:
                    local = local[local // block_size < block_table.shape[1]]
                    block = block_table[leader].long()[local // block_size]
                    good = (block >= 0) & (block < k_cache.shape[0])
                    slots.append((block * block_size + local % block_size)[good])
            slot = torch.cat(slots) if slots else torch.empty(0, dtype=torch.int64, device=q.device)
            out, lse, spread, _ = attend_row(q[i], slot, k_cache, v_cache, k_scale, v_scale, softmax_scale)
            peak = torch.zeros_like(out)
            if slot.numel():
                block, offset = slot // block_size, slot % block_size
                k = k_cache[block, offset].float().double() * k_scale[block].double()[:, :, None]
                score = torch.einsum("hgd,nhd->hgn", q[i].double().reshape(kv_heads, heads // kv_heads, -1), k) * softmax_scale
                scaled = score + v_scale[block].double().T[:, None].log2() * math.log(2.0)
                most = torch.exp(scaled.amax(-1).reshape(heads) - lse)
                codes = v_cache[block, offset].float().double().abs().sum(0)
                peak = most[:, None] * codes.repeat_interleave(heads // kv_heads, 0)
            rows.append((out, lse, spread, peak))
    return tuple(torch.stack(part) for part in zip(*rows))


def merge(outs, lses):
    lse = torch.logsumexp(lses.double(), dim=0)
    weight = torch.where(lses > -math.inf, torch.exp(lses.double() - lse), 0.0)
    seen = torch.where((lses > -math.inf)[..., None], outs.double(), 0.0)
    return (weight[..., None] * seen).sum(0), lse, (weight[..., None] * seen.abs()).sum(0)
