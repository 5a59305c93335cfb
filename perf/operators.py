"""The attention operators over the 8-bit paged cache, as workloads: their plain forms in torch, the
framework's calls, and what each pass has to read, write and compute.

Four operators make one decode step's way past the localized selection:

* ``append``: new tokens go into the paged e4m3 cache, with one float32 scale for each page and head;
* ``selected``: attention over the rank-local slots that the converter emits;
* ``window``: attention over a sliding window and a few first tokens that stay visible, through the
  block table (a window of 0 is the whole context);
* ``merge``: the partial results of the context-parallel ranks become one.

A page is ``block`` consecutive rank-local tokens. Token ``t`` of a sequence belongs to rank
``(t / interleave) % dcp`` and is that rank's local token
``(t / (dcp * interleave)) * interleave + t % interleave``.
"""

import math

import numpy as np
import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One decode step writes one token of each of 64 sequences: the call that runs every layer, every step.
        {"name": "append_decode", "op": "append", "batch": 64, "tokens": 64, "past": 1000, "kv_heads": 8, "dim": 128,
         "latent": False, "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # Pieces of four prompts of unlike length into a latent cache (one head, keys of 512 + 64) shared by two ranks.
        {"name": "append_prompt_latent", "op": "append", "batch": 4, "tokens": 8192, "past": 333, "kv_heads": 1, "dim": 576,
         "latent": True, "block": 64, "dcp": 2, "interleave": 1, "type": "bf16"},
        # A single request in flight: only the latency counts.
        {"name": "selected_one_latent", "op": "selected", "batch": 1, "top_k": 2048, "heads": 128, "kv_heads": 1, "dim": 576,
         "latent": True, "block": 64, "dcp": 1, "interleave": 1, "min_len": 32768, "max_len": 32768, "type": "bf16"},
        # The mixed-length decode batch of the converter's headline workload: 256 x 2048 over four ranks.
        {"name": "selected_mixed_latent", "op": "selected", "batch": 256, "top_k": 2048, "heads": 128, "kv_heads": 1, "dim": 576,
         "latent": True, "block": 64, "dcp": 4, "interleave": 1, "min_len": 1024, "max_len": 65536, "type": "bf16"},
        # The 64 x 2048 decode batch over two ranks, heads in eight groups of eight.
        {"name": "selected_grouped", "op": "selected", "batch": 64, "top_k": 2048, "heads": 64, "kv_heads": 8, "dim": 128,
         "latent": False, "block": 64, "dcp": 2, "interleave": 1, "min_len": 32768, "max_len": 32768, "type": "bf16"},
        # The wide rows of the hierarchical converter, 32 x 16384 over eight ranks, with the 16 heads of one tensor-parallel shard.
        {"name": "selected_wide_latent", "op": "selected", "batch": 32, "top_k": 16384, "heads": 16, "kv_heads": 1, "dim": 576,
         "latent": True, "block": 64, "dcp": 8, "interleave": 1, "min_len": 131072, "max_len": 131072, "type": "fp16"},
        # Decode with a window and sinks, 128 sequences of unlike length.
        {"name": "window_decode", "op": "window", "batch": 128, "tokens": 128, "min_len": 100, "max_len": 32768, "window": 4096,
         "sinks": 4, "heads": 64, "kv_heads": 8, "dim": 128, "latent": False, "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # One long sequence, whole context: a single query row over 131072 tokens.
        {"name": "window_one_long", "op": "window", "batch": 1, "tokens": 1, "min_len": 131072, "max_len": 131072, "window": 0,
         "sinks": 0, "heads": 64, "kv_heads": 8, "dim": 128, "latent": False, "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # Pieces of three prompts (odd lengths) with a short window: many queries share their keys.
        {"name": "window_prompt", "op": "window", "batch": 3, "tokens": 4001, "min_len": 2000, "max_len": 5000, "window": 1024,
         "sinks": 4, "heads": 32, "kv_heads": 4, "dim": 64, "latent": False, "block": 32, "dcp": 1, "interleave": 1, "type": "fp16"},
        # Two ranks' partial results of one request.
        {"name": "merge_one", "op": "merge", "ranks": 2, "rows": 1, "heads": 128, "dim": 512, "type": "bf16"},
        # Eight ranks' partial results of the 128-row decode step.
        {"name": "merge_batch", "op": "merge", "ranks": 8, "rows": 128, "heads": 128, "dim": 512, "type": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "selected", "selected", "window", "window", "merge"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "merge":
        return {"op": op, "ranks": rng.randint(1, 8), "rows": _log_int(rng, 1, 128), "heads": rng.choice([1, 7, 16, 64, 128]),
                "dim": rng.choice([64, 128, 512]), "type": kind}
    latent = rng.random() < 0.5
    kv_heads = 1 if latent else rng.choice([1, 2, 3, 8])
    dim = 576 if latent else rng.choice([64, 128])
    dcp = rng.choice([1, 1, 2, 4, 8])
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "latent": latent, "dcp": dcp,
            "interleave": rng.choice([1, 1, 4, 16]), "type": kind}
    case["block"] = rng.choice([16, 32, 48, 64, 128])
    if op == "append":
        batch = _log_int(rng, 1, 128)
        most = 8192 if latent else 8192 // kv_heads
        case.update(batch=batch, tokens=batch if rng.random() < 0.5 else _log_int(rng, batch, max(batch, most)),
                    past=_log_int(rng, 1, 2000))
        return case
    case["heads"] = rng.choice([5, 16, 24, 64, 128]) if latent else kv_heads * rng.choice([1, 2, 5, 8, 16])
    if op == "selected":
        top_k = _log_int(rng, 17, 16384)
        high = _log_int(rng, max(64, top_k), 131072) if top_k < 131072 else top_k
        case.update(top_k=top_k, batch=_log_int(rng, 1, max(1, min(256, 400_000 // top_k, 16_000_000 // high))),
                    min_len=max(1, high // rng.choice([1, 3, 50])), max_len=high)
        return case
    case["sinks"] = rng.choice([0, 1, 4, 128])
    if rng.random() < 0.6:
        high = _log_int(rng, 1, 131072)
        window = 0 if rng.random() < 0.3 else _log_int(rng, 1, 8192)
        seen = min(high, window + case["sinks"]) if window else high
        batch = _log_int(rng, 1, max(1, min(256, 8_000_000 // high, 400_000 // seen)))
        case.update(batch=batch, tokens=batch, min_len=max(1, high // rng.choice([1, 3, 50])), max_len=high, window=window)
    else:
        case["sinks"] = min(case["sinks"], 4)
        batch = rng.randint(1, 5)
        each = _log_int(rng, 2, 600 if latent else 1200)
        high = each + _log_int(rng, 1, 3000)
        case.update(batch=batch, tokens=batch * each - rng.randint(0, batch - 1), min_len=high // 2 + each, max_len=high + each,
                    window=_log_int(rng, 1, 600 if latent else 1100))
    return case


# ------------------------------------------------------------------------------------- shapes of a case

def _value_dim(case):
    return 512 if case["latent"] else case["dim"]


def _lengths(case):
    """Whole lengths of the sequences: even steps from the shortest to the longest."""
    n = case["batch"]
    if case["op"] == "append":
        past = [1 + (case["past"] - 1) * (i + 1) // n for i in range(n)]
        return [p + q for p, q in zip(past, _new_tokens(case))]
    low, high = case["min_len"], case["max_len"]
    return [max(1, low + (high - low) * (i + 1) // n) for i in range(n)]


def _new_tokens(case):
    """How many of the call's tokens each sequence has: all alike, but for odd pieces moved from neighbour to neighbour."""
    n, total = case["batch"], case["tokens"]
    got = [total // n + (i < total % n) for i in range(n)]
    if total >= 8 * n:
        for i in range(0, n - 1, 2):
            move = got[i] // 3
            got[i], got[i + 1] = got[i] - move, got[i + 1] + move
    return got


def _seen(case, length):
    """Visible positions of the query at `length` - 1, over all ranks."""
    if not case["window"]:
        return length
    window = min(case["window"], length)
    return window + min(case["sinks"], length - window)


def work(case):
    op = case["op"]
    if op == "merge":
        n = case["rows"] * case["heads"]
        return {"bytes": n * (case["ranks"] + 1) * (2 * case["dim"] + 4), "flops": n * case["ranks"] * 2 * case["dim"]}
    dim, value = case["dim"], _value_dim(case)
    token = case["kv_heads"] * (dim if case["latent"] else dim + value)  # bytes of one token in the cache
    dcp, block = case["dcp"], case["block"]
    if op == "append":
        new, scales = case["tokens"] / dcp, 0
        for n in _new_tokens(case):
            scales += -(-n // (dcp * block)) * case["kv_heads"] * (1 if case["latent"] else 2)
        return {"bytes": new * token * (2 + 1) + 8 * scales + 12 * case["batch"], "flops": 2 * new * token}
    heads = case["heads"]
    if op == "selected":
        keys = sum(min(case["top_k"], n) for n in _lengths(case)) / dcp
        rows, index, pairs = case["batch"], 4 * keys, keys
    else:
        keys = pairs = index = 0
        for length, n in zip(_lengths(case), _new_tokens(case)):
            first = length - n + 1
            spread = length if not case["window"] else min(length, case["window"] + n - 1)
            keys += (spread + min(case["sinks"] if case["window"] else 0, length - spread)) / dcp
            index += 4 * (length / (dcp * block) if not case["window"] else spread / (dcp * block))
            pairs += sum(_seen(case, x) for x in range(first, length + 1)) / dcp
        rows = case["tokens"]
    return {"bytes": keys * token + index + rows * heads * (2 * (dim + value) + 4), "flops": 2 * pairs * heads * (dim + value)}


# --------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _cache(case, pages, g):
    """A filled paged cache: keys and values of about unit size, one scale for each page and head."""
    def part(dim):
        shape = (pages, case["block"], case["kv_heads"], dim)
        cache = torch.empty(shape, dtype=E4M3, device="cuda")
        flat = cache.view(-1)
        step = 1 << 28
        for at in range(0, flat.numel(), step):
            n = min(step, flat.numel() - at)
            x = torch.randn(n, generator=g, device="cuda", dtype=torch.float16).mul_(64).clamp_(-E4M3_MAX, E4M3_MAX)
            flat[at : at + n] = x.to(E4M3)
        scale = torch.randn((pages, case["kv_heads"]), generator=g, device="cuda").mul_(0.3).exp_().mul_(2.0**-6)
        return cache, scale
    k, ks = part(case["dim"])
    v, vs = (None, None) if case["latent"] else part(case["dim"])
    return k, v, ks, vs


def _localized(lengths, top_k, table, case, rank, g):
    """Rank-local slots of `top_k` random positions of each sequence, in random order, survivors first, and their counts."""
    batch, longest = len(lengths), int(max(lengths))
    longest = max(longest, top_k)
    length = torch.tensor(lengths, device="cuda")[:, None]
    score = torch.rand((batch, longest), generator=g, device="cuda")
    score = torch.where(torch.arange(longest, device="cuda") < length, score, -1.0)
    best, token = score.topk(top_k, dim=1)
    group = case["dcp"] * case["interleave"]
    kept = (best >= 0) & ((token // case["interleave"]) % case["dcp"] == rank)
    local = token // group * case["interleave"] + token % case["interleave"]
    slot = table.gather(1, (local // case["block"]).clamp(max=table.shape[1] - 1)).long() * case["block"] + local % case["block"]
    slot = torch.where(kept, slot, -1)
    order = torch.argsort((~kept).to(torch.int8), dim=1, stable=True)
    return slot.gather(1, order).to(torch.int32), kept.sum(1).to(torch.int32)


def prepare(case, seed):
    g, dtype = _generator(seed), TYPES[case["type"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "merge":
        ranks, rows, heads, dim = case["ranks"], case["rows"], case["heads"], case["dim"]
        s["outs"] = randn(ranks, rows, heads, dim)
        s["lses"] = torch.randn((ranks, rows, heads), generator=g, device="cuda") * 2 + 5
        if ranks > 1:  # some ranks own none of a row's selection
            none = torch.rand((ranks, rows, 1), generator=g, device="cuda") < 0.05
            s["outs"].masked_fill_(none[..., None], 0.0)
            s["lses"].masked_fill_(none, -math.inf)
        s["out"], s["lse"] = torch.empty_like(s["outs"][0]), torch.empty_like(s["lses"][0])
        return s
    lengths, dcp = _lengths(case), case["dcp"]
    s["rank"] = int(seed) % dcp
    batch, per_page = case["batch"], case["block"] * dcp
    width = max(1, -(-(max(lengths) + case["interleave"] * dcp) // per_page))
    table = torch.randperm(batch * width, generator=g, device="cuda").to(torch.int32).view(batch, width)
    s["table"], s["req"] = table, torch.randperm(batch, generator=g, device="cuda").to(torch.int32)
    order = torch.randperm(batch, generator=g, device="cuda").tolist()
    lengths = [lengths[i] for i in order]
    s["k"], s["v"], s["ks"], s["vs"] = _cache(case, batch * width, g)
    dim, value = case["dim"], _value_dim(case)
    s["softmax_scale"] = dim**-0.5
    if case["op"] == "append":
        new = [_new_tokens(case)[i] for i in order]
        s["starts"] = ints([n - m for n, m in zip(lengths, new)])
        s["cu"] = ints(np.concatenate([[0], np.cumsum(new)]))
        size = torch.randn((case["tokens"], 1, 1), generator=g, device="cuda").mul_(0.5).exp_()
        s["new_k"] = (randn(case["tokens"], case["kv_heads"], dim).float() * size).to(dtype)
        s["new_v"] = None if case["latent"] else (randn(case["tokens"], case["kv_heads"], value).float() * size).to(dtype)
        return s
    if case["op"] == "selected":
        rows = batch
        s["slots"], s["counts"] = _localized(lengths, case["top_k"], table[s["req"].long()], case, s["rank"], g)
    else:
        rows = case["tokens"]
        new = [_new_tokens(case)[i] for i in order]
        s["lengths"], s["cu"] = ints(lengths), ints(np.concatenate([[0], np.cumsum(new)]))
        # The most that any query sees: a launch-time number that a user's program knows as well.
        s["most"] = max(_seen(case, n) for n in lengths)
    s["q"] = randn(rows, case["heads"], dim)
    s["out"] = torch.empty((rows, case["heads"], value), dtype=dtype, device="cuda")
    s["lse"] = torch.empty((rows, case["heads"]), dtype=torch.float32, device="cuda")
    return s


# ---------------------------------------------------------------------------------------- plain forms

def _plain_append(s):
    case = s["case"]
    n, dcp, inter, block = case["tokens"], case["dcp"], case["interleave"], case["block"]
    t = torch.arange(n, device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    position = s["starts"].long()[seq] + t - s["cu"].long()[seq]
    kept = (position // inter) % dcp == s["rank"]
    local = position // (dcp * inter) * inter + position % inter
    page = s["table"].long()[s["req"].long()[seq], (local // block).clamp(max=s["table"].shape[1] - 1)][kept]
    offset = (local % block)[kept]
    result = []
    for cache, scale, new in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        if cache is None:
            continue
        x = new[kept].float()
        fresh = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
        fresh[page[offset == 0]] = True
        old = torch.where(fresh[:, None], 0.0, scale)
        most = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
        # The smallest power of two whose 448-fold reaches the largest value: 448 = 0.875 * 2^9.
        fraction, exponent = torch.frexp(most)
        power = (exponent - 9 + (fraction > 0.875)).clamp(-100, 100)
        want = torch.where(most > 0, torch.ldexp(torch.ones_like(most), power), 0.0)
        use = torch.maximum(old, want)
        grown = page[(use > old)[page].any(-1) & ~fresh[page]]
        ratio = torch.where(use > 0, old / use, 1.0)
        held = cache[grown].float() * ratio[grown][:, None, :, None]
        cache[grown] = held.to(E4M3)
        step = use[page][..., None]
        cache[page, offset] = torch.where(step > 0, x / step, 0.0).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        scale[page] = use[page]
        result += [cache, scale]
    return result


def _plain_softmax(s, q, slot, valid):
    """softmax(q k) v over the slots of each row where valid, and the log of the sum."""
    case = s["case"]
    rows, heads, kv, value = q.shape[0], case["heads"], case["kv_heads"], _value_dim(case)
    slot = torch.where(valid, slot, 0).long()
    page = slot // case["block"]
    hide = ~valid[..., None, None]
    k = (s["k"].flatten(0, 1)[slot].float() * s["ks"][page][..., None]).masked_fill_(hide, 0.0)
    if case["latent"]:
        v = k[..., :value]
    else:
        v = (s["v"].flatten(0, 1)[slot].float() * s["vs"][page][..., None]).masked_fill_(hide, 0.0)
    q = q.float().view(rows, kv, heads // kv, -1) * s["softmax_scale"]
    score = q @ k.permute(0, 2, 3, 1)
    score.masked_fill_(~valid[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v.transpose(1, 2)) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).view(rows, heads)
    return out.view(rows, heads, value).to(s["out"].dtype), lse


def _plain_window(s):
    case = s["case"]
    t = torch.arange(case["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    length = s["lengths"].long()[seq] - (s["cu"].long()[seq + 1] - 1 - t)  # positions up to the query's own
    low = torch.zeros_like(length) if not case["window"] else (length - case["window"]).clamp(min=0)
    first = low if not case["window"] else torch.minimum(low, torch.full_like(low, case["sinks"]))
    j = torch.arange(s["most"], device="cuda")[None, :]
    position = torch.where(j < first[:, None], j, j - first[:, None] + low[:, None])
    dcp, inter = case["dcp"], case["interleave"]
    valid = (position < length[:, None]) & ((position // inter) % dcp == s["rank"])
    local = position // (dcp * inter) * inter + position % inter
    row = s["table"].long()[s["req"].long()[seq]]
    slot = row.gather(1, (local // case["block"]).clamp(max=row.shape[1] - 1)) * case["block"] + local % case["block"]
    return _plain_softmax(s, s["q"], slot, valid)


def _plain_merge(s):
    top = s["lses"].amax(0)
    w = (s["lses"] - torch.where(top > -math.inf, top, 0.0)).exp_()
    total = w.sum(0)
    out = (w[..., None] * s["outs"].float()).sum(0) / torch.where(total > 0, total, 1.0)[..., None]
    return out.to(s["outs"].dtype), top + total.log()


def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["op"] == "append":
        return _plain_append(state)
    if case["op"] == "selected":
        return _plain_softmax(state, state["q"], state["slots"], state["slots"] >= 0)
    return _plain_window(state) if case["op"] == "window" else _plain_merge(state)


def _own(s):
    import silkern_b200 as silkern

    case = s["case"]
    if case["op"] == "merge":
        silkern.merge_partials(s["outs"], s["lses"], s["out"], s["lse"])
        return s["out"], s["lse"]
    dcp = {"dcp_size": case["dcp"], "dcp_rank": s["rank"], "dcp_interleave": case["interleave"]}
    if case["op"] == "append":
        silkern.append_quantized(s["new_k"], s["new_v"], s["k"], s["v"], s["ks"], s["vs"], s["cu"], s["starts"], s["req"], s["table"], **dcp)
        return [s["k"], s["ks"]] if case["latent"] else [s["k"], s["ks"], s["v"], s["vs"]]
    if case["op"] == "selected":
        silkern.attend_selected(s["q"], s["slots"], s["k"], s["v"], s["ks"], s["vs"], s["out"], s["lse"],
                                softmax_scale=s["softmax_scale"], counts=s["counts"])
    else:
        silkern.attend_window(s["q"], s["cu"], s["lengths"], s["req"], s["table"], s["k"], s["v"], s["ks"], s["vs"], s["out"], s["lse"],
                              softmax_scale=s["softmax_scale"], window=case["window"], sinks=case["sinks"], **dcp)
    return s["out"], s["lse"]


# ------------------------------------------------------------------- the definitions once more, in 64 bits

def _owned(case, rank, position):
    """(whether the rank holds the position, the rank-local token) of an array of positions."""
    run_of, within = np.divmod(position, case["interleave"])
    return run_of % case["dcp"] == rank, run_of // case["dcp"] * case["interleave"] + within


def _exact_append(case, s):
    cu, starts, req, table = (s[n].cpu().numpy() for n in ("cu", "starts", "req", "table"))
    result = []
    for cache, scale, new in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        if cache is None:
            continue
        held, sizes, x = cache.double(), scale.double(), new.double()
        for b in range(case["batch"]):
            position = np.arange(starts[b], starts[b] + cu[b + 1] - cu[b])
            kept, local = _owned(case, s["rank"], position)
            where, local = np.flatnonzero(kept) + cu[b], local[kept]
            for logical in np.unique(local // case["block"]):
                here = local // case["block"] == logical
                offset = torch.from_numpy(local[here] % case["block"]).cuda()
                rows = x[torch.from_numpy(where[here]).cuda()]
                page = int(table[req[b], logical])
                old = torch.zeros_like(sizes[page]) if local[here][0] % case["block"] == 0 else sizes[page].clone()
                most = rows.abs().amax((0, 2))
                want = torch.where(most > 0, torch.exp2(torch.ceil(torch.log2(most.clamp(min=1e-300) / E4M3_MAX)).clamp(-100, 100)), 0.0)
                use = torch.maximum(old, want)
                if bool((old > 0).any()) and bool((use > old).any()):
                    held[page] = (held[page] * (old / use.clamp(min=1e-300))[None, :, None]).float().to(E4M3).double()
                held[page, offset] = (rows / use.clamp(min=1e-300)[None, :, None]).float().to(E4M3).double()
                sizes[page] = use
        result += [held, sizes]
    return result


def _exact_row(case, s, query, slot, softmax_scale):
    """One query row (heads, dim) over its visible slots."""
    heads, kv, value = case["heads"], case["kv_heads"], _value_dim(case)
    if slot.numel() == 0:
        return torch.zeros((heads, value), dtype=torch.float64, device="cuda"), torch.full((heads,), -math.inf, dtype=torch.float64, device="cuda")
    page, offset = slot // case["block"], slot % case["block"]
    k = s["k"][page, offset].double() * s["ks"][page].double()[:, :, None]
    v = k[:, :, :value] if case["latent"] else s["v"][page, offset].double() * s["vs"][page].double()[:, :, None]
    of = torch.arange(heads, device="cuda") // (heads // kv)
    score = torch.einsum("hgd,nhd->hgn", query.double().view(kv, heads // kv, -1), k).reshape(heads, -1) * softmax_scale
    lse = torch.logsumexp(score, dim=1)
    weight = (score - lse[:, None]).exp().view(kv, heads // kv, -1)
    assert int(of[-1]) == kv - 1
    return torch.einsum("hgn,nhd->hgd", weight, v).reshape(heads, value), lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "merge":
        lse = torch.logsumexp(s["lses"].double(), dim=0)
        weight = torch.where(s["lses"] > -math.inf, (s["lses"].double() - lse).exp(), 0.0)
        return torch.einsum("rbh,rbhd->bhd", weight, s["outs"].double()), lse
    outs, lses = [], []
    if case["op"] == "selected":
        for row in range(case["batch"]):
            slot = s["slots"][row].long()
            o, m = _exact_row(case, s, s["q"][row], slot[slot >= 0], s["softmax_scale"])
            outs.append(o), lses.append(m)
        return torch.stack(outs), torch.stack(lses)
    if case["tokens"] > 3000 and case["tokens"] * case["window"] > 2**23:
        return None
    cu, lengths, req = (s[n].cpu().numpy() for n in ("cu", "lengths", "req"))
    for b in range(case["batch"]):
        table = s["table"][int(req[b])].long()
        for i in range(cu[b], cu[b + 1]):
            end = int(lengths[b]) - (int(cu[b + 1]) - i) + 1
            position = np.arange(end)
            if case["window"]:
                position = position[(position >= end - case["window"]) | (position < case["sinks"])]
            kept, local = _owned(case, s["rank"], position)
            local = torch.from_numpy(local[kept]).cuda()
            o, m = _exact_row(case, s, s["q"][i], table[local // case["block"]] * case["block"] + local % case["block"], s["softmax_scale"])
            outs.append(o), lses.append(m)
    return torch.stack(outs), torch.stack(lses)
