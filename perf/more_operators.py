"""What stands on either side of the 8-bit paged cache, as workloads: plain forms in torch, the framework's
calls, and what each pass has to read, write and compute.

Three operators of a serving step:

* ``rotate``: queries and new keys, before they are stored and asked: an optional root-mean-square norm of
  each head's first columns, then the rotation by position of some of its columns, in one pass;
* ``read``: a stretch of each sequence's cached tokens, back as 16-bit keys and values;
* ``shared``: attention of sequences in groups that have their first tokens in common: a group's prefix is
  stored once, in the pages of its first sequence, and read once for all of the group's queries.

Token ``t`` of a sequence belongs to rank ``(t / interleave) % dcp`` and is that rank's local token
``(t / (dcp * interleave)) * interleave + t % interleave``; a page is ``block`` consecutive local tokens.
"""

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One decode step of 64 sequences: the call that runs in every layer of every step, with normed heads.
        {"name": "rotate_decode", "op": "rotate", "tokens": 64, "heads": 64, "kv_heads": 8, "dim": 128, "start": 0, "rotary": 128,
         "q_norm": 128, "k_norm": 128, "interleaved": False, "base": 10000.0, "amplitude": 1.0, "far": 32768, "type": "bf16"},
        # A prompt's pieces at far positions, frequencies stretched for a long context.
        {"name": "rotate_prompt", "op": "rotate", "tokens": 8192, "heads": 64, "kv_heads": 8, "dim": 128, "start": 0, "rotary": 128,
         "q_norm": 128, "k_norm": 128, "interleaved": False, "base": 1000000.0, "amplitude": 1.2, "far": 131072, "type": "bf16"},
        # Latent heads of 512 + 64: the key's first part is normed, the last part rotated, in neighbouring pairs.
        {"name": "rotate_latent", "op": "rotate", "tokens": 1001, "heads": 128, "kv_heads": 1, "dim": 576, "start": 512, "rotary": 64,
         "q_norm": 0, "k_norm": 512, "interleaved": True, "base": 10000.0, "amplitude": 1.0, "far": 131072, "type": "bf16"},
        # Half of each small head rotates, without norms; an odd number of tokens.
        {"name": "rotate_part", "op": "rotate", "tokens": 4001, "heads": 32, "kv_heads": 4, "dim": 64, "start": 0, "rotary": 32,
         "q_norm": 0, "k_norm": 0, "interleaved": False, "base": 10000.0, "amplitude": 1.0, "far": 5000, "type": "fp16"},
        # One short stretch of one latent sequence: latency.
        {"name": "read_one_latent", "op": "read", "batch": 1, "tokens": 333, "past": 1000, "kv_heads": 1, "dim": 576, "latent": True,
         "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # The contexts of eight sequences of unlike length, for a prompt's next pieces.
        {"name": "read_grouped", "op": "read", "batch": 8, "tokens": 65536, "past": 100, "kv_heads": 8, "dim": 128, "latent": False,
         "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # A rank's half of four latent contexts.
        {"name": "read_latent_ranks", "op": "read", "batch": 4, "tokens": 32768, "past": 1, "kv_heads": 1, "dim": 576, "latent": True,
         "block": 64, "dcp": 2, "interleave": 16, "type": "fp16"},
        # Four requests behind a short common instruction: only the latency counts.
        {"name": "shared_small", "op": "shared", "batch": 4, "groups": 1, "each": 1, "prefix": 1000, "own_min": 3, "own_max": 100,
         "heads": 16, "kv_heads": 2, "dim": 64, "block": 32, "dcp": 1, "interleave": 1, "type": "fp16"},
        # A decode batch of 128 that answers questions about one document of 32768 tokens.
        {"name": "shared_decode", "op": "shared", "batch": 128, "groups": 1, "each": 1, "prefix": 32768, "own_min": 20, "own_max": 1000,
         "heads": 64, "kv_heads": 8, "dim": 128, "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # 256 sequences in five groups of unlike size, prefixes that end inside a page, over four ranks.
        {"name": "shared_groups", "op": "shared", "batch": 256, "groups": 5, "each": 1, "prefix": 16333, "own_min": 1, "own_max": 4000,
         "heads": 64, "kv_heads": 8, "dim": 128, "block": 64, "dcp": 4, "interleave": 1, "type": "bf16"},
        # Sixteen samples that continue one long context.
        {"name": "shared_long", "op": "shared", "batch": 16, "groups": 1, "each": 1, "prefix": 131072, "own_min": 1, "own_max": 300,
         "heads": 64, "kv_heads": 8, "dim": 128, "block": 64, "dcp": 1, "interleave": 1, "type": "bf16"},
        # Short pieces (five drafted tokens each) of 24 sequences in two groups.
        {"name": "shared_pieces", "op": "shared", "batch": 24, "groups": 2, "each": 5, "prefix": 4099, "own_min": 200, "own_max": 2000,
         "heads": 32, "kv_heads": 4, "dim": 64, "block": 48, "dcp": 1, "interleave": 1, "type": "fp16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "read", "shared", "shared", "shared"])
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "rotate":
        dim = rng.choice([64, 80, 128, 128, 192, 256, 576])
        heads, kv_heads = rng.choice([(5, 5), (16, 2), (32, 4), (64, 8), (128, 1)])
        rotary = 64 if dim == 576 else 2 * rng.choice([dim // 2, dim // 2, dim // 4, 8])
        start = 512 if dim == 576 else rng.choice([0, 0, dim - rotary])
        norm = rng.choice([0, dim, dim]) if dim != 576 else rng.choice([0, 512])
        most = max(1, 600_000_000 // (dim * (heads + kv_heads) * 8))
        case.update(tokens=_log_int(rng, 1, min(8192, most)), heads=heads, kv_heads=kv_heads, dim=dim, start=start, rotary=rotary,
                    q_norm=norm, k_norm=norm, interleaved=rng.random() < 0.4, base=rng.choice([10000.0, 500000.0]),
                    amplitude=rng.choice([1.0, 1.0, 1.3]), far=_log_int(rng, 10, 1_000_000))
        return case
    case.update(block=rng.choice([16, 32, 48, 64, 128]), dcp=rng.choice([1, 1, 1, 2, 4, 8]), interleave=rng.choice([1, 1, 4, 16]))
    if op == "read":
        latent = rng.random() < 0.5
        kv_heads = 1 if latent else rng.choice([1, 2, 3, 8])
        batch = _log_int(rng, 1, 64)
        case.update(batch=batch, tokens=_log_int(rng, batch, 65536), past=_log_int(rng, 1, 2000), kv_heads=kv_heads,
                    dim=576 if latent else rng.choice([64, 128]), latent=latent)
        return case
    kv_heads = rng.choice([1, 2, 3, 8])
    heads = kv_heads * rng.choice([1, 2, 5, 8, 16])
    each = rng.choice([1, 1, 1, 2, 5])
    batch = _log_int(rng, 1, 256 // each)
    most = max(64, min(131072, 280_000_000 // (batch * each * heads)))
    prefix = _log_int(rng, 1, most)
    own_max = each + _log_int(rng, 1, max(1, min(4000, 500_000 // (batch * each))))
    case.update(batch=batch, groups=rng.randint(1, min(batch, 6)), each=each, prefix=prefix, own_min=rng.choice([each, own_max]),
                own_max=own_max, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]))
    return case


# ------------------------------------------------------------------------------------- shapes of a case

def _pieces(case):
    """How many of a read's tokens each sequence has: alike, but for odd pieces moved from neighbour to neighbour."""
    n, total = case["batch"], case["tokens"]
    got = [total // n + (i < total % n) for i in range(n)]
    if total >= 8 * n:
        for i in range(0, n - 1, 2):
            move = got[i] // 3
            got[i], got[i + 1] = got[i] - move, got[i + 1] + move
    return got


def _starts(case):
    return [(case["past"] - 1) * (i + 1) // case["batch"] for i in range(case["batch"])]


def _groups(case):
    """(sequences, prefix length) of each group: the first the largest, with the longest prefix."""
    n, g = case["batch"], case["groups"]
    sizes = [1] * g
    for i in range(n - g):
        sizes[0 if i % 2 else i // 2 % g] += 1
    return [(size, max(1, case["prefix"] * (g - i) // g)) for i, size in enumerate(sizes)]


def _own_lengths(case):
    """Tokens of each sequence behind its prefix, its queries included."""
    low, high, n = max(case["own_min"], case["each"]), max(case["own_max"], case["each"]), case["batch"]
    return [low + (high - low) * ((7 * i + 3) % n + 1) // n for i in range(n)]


def work(case):
    op = case["op"]
    if op == "rotate":
        n = case["tokens"]
        pairs = n * (case["heads"] + case["kv_heads"]) * case["rotary"] // 2
        normed = n * (case["heads"] * case["q_norm"] + case["kv_heads"] * case["k_norm"])
        return {"bytes": 4 * n * (case["heads"] + case["kv_heads"]) * case["dim"] + 4 * n + 2 * case["rotary"] + 4 * (case["q_norm"] + case["k_norm"]),
                "flops": 6 * pairs + 4 * normed}
    dim, dcp, block = case["dim"], case["dcp"], case["block"]
    if op == "read":
        token = case["kv_heads"] * (dim if case["latent"] else 2 * dim)
        n = case["tokens"] / dcp
        pages = sum(-(-m // (dcp * block)) for m in _pieces(case))
        return {"bytes": n * token * 3 + pages * (4 + 4 * case["kv_heads"] * (1 if case["latent"] else 2)) + 12 * case["batch"], "flops": n * token}
    token = 2 * case["kv_heads"] * dim
    at, keys, pairs = 0, 0, 0
    own_lengths = _own_lengths(case)
    for size, prefix in _groups(case):
        keys += prefix / dcp
        for own_length in own_lengths[at : at + size]:
            keys += own_length / dcp
            pairs += sum(prefix + own_length - i for i in range(case["each"])) / dcp
        at += size
    rows = case["batch"] * case["each"]
    scales = keys / block * 4 * (1 + 2 * case["kv_heads"])
    return {"bytes": keys * token + scales + rows * case["heads"] * (4 * dim + 4), "flops": 4 * pairs * case["heads"] * dim}


# --------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums(counts):
    total = [0]
    for n in counts:
        total.append(total[-1] + n)
    return total


def _cache(case, pages, g):
    """A filled paged cache: keys and values of about unit size, one scale for each page and head."""
    def part(dim):
        cache = torch.empty((pages, case["block"], case["kv_heads"], dim), dtype=E4M3, device="cuda")
        flat = cache.view(-1)
        step = 1 << 28
        for at in range(0, flat.numel(), step):
            n = min(step, flat.numel() - at)
            x = torch.randn(n, generator=g, device="cuda", dtype=torch.float16).mul_(64).clamp_(-E4M3_MAX, E4M3_MAX)
            flat[at : at + n] = x.to(E4M3)
        return cache, torch.randn((pages, case["kv_heads"]), generator=g, device="cuda").mul_(0.3).exp_().mul_(2.0**-6)
    k, ks = part(case["dim"])
    v, vs = (None, None) if case.get("latent") else part(case["dim"])
    return k, v, ks, vs


def _local_pages(case, tokens):
    """Pages that any rank may need for the first `tokens` positions."""
    return max(1, -(-(tokens + case["interleave"] * case["dcp"]) // (case["block"] * case["dcp"])))


def prepare(case, seed):
    g, dtype = _generator(seed), TYPES[case["type"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    s = {"case": case}
    if case["op"] == "rotate":
        n, dim, rotary = case["tokens"], case["dim"], case["rotary"]
        s["q"], s["k"] = randn(n, case["heads"], dim), randn(n, case["kv_heads"], dim)
        # Consecutive positions of a few pieces, each from a place of its own.
        first = torch.randint(0, case["far"], (-(-n // 256),), generator=g, device="cuda")
        s["positions"] = (first.repeat_interleave(256)[:n] + torch.arange(n, device="cuda") % 256).to(torch.int32)
        s["frequencies"] = (case["base"] ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda()
        for name in ("q", "k"):
            columns = case[name + "_norm"]
            s[name + "_weight"] = 1 + 0.1 * torch.randn(columns, generator=g, device="cuda") if columns else None
            s[name + "_out"] = torch.empty_like(s[name])
        return s
    s["rank"] = int(seed) % case["dcp"]
    batch = case["batch"]
    s["req"] = torch.randperm(batch, generator=g, device="cuda").to(torch.int32)
    if case["op"] == "read":
        pieces, starts = _pieces(case), _starts(case)
        width = _local_pages(case, max(a + b for a, b in zip(starts, pieces)))
        s["table"] = torch.randperm(batch * width, generator=g, device="cuda").to(torch.int32).view(batch, width)
        s["k"], s["v"], s["ks"], s["vs"] = _cache(case, batch * width, g)
        s["cu"], s["starts"] = _ints(_sums(pieces)), _ints(starts)
        s["keys"] = torch.zeros((case["tokens"], case["kv_heads"], case["dim"]), dtype=dtype, device="cuda")
        s["values"] = None if case["latent"] else torch.zeros_like(s["keys"])
        return s
    groups, own_lengths, per_page = _groups(case), _own_lengths(case), case["block"] * case["dcp"]
    prefixes = [p for size, p in groups for _ in range(size)]
    lengths = [p + n for p, n in zip(prefixes, own_lengths)]
    width = _local_pages(case, max(lengths))
    # Whole pages of a prefix are its first sequence's; every other page is a sequence's own.
    source, at = [], 0
    for size, prefix in groups:
        for i in range(size):
            whole = prefix // per_page if i else 0
            source.append((at, whole, _local_pages(case, lengths[at + i])))
        at += size
    fresh = torch.randperm(sum(n - whole for _, whole, n in source), generator=g, device="cuda").to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    at, rows = 0, s["req"].tolist()
    for b, (leader, whole, n) in enumerate(source):
        table[rows[b], :whole] = table[rows[leader], :whole]
        table[rows[b], whole:n] = fresh[at : at + n - whole]
        at += n - whole
    s["table"] = table
    s["k"], s["v"], s["ks"], s["vs"] = _cache(case, fresh.numel(), g)
    tokens = batch * case["each"]
    s["cu"], s["lengths"] = _ints(_sums([case["each"]] * batch)), _ints(lengths)
    s["cu_groups"], s["prefixes"] = _ints(_sums([size for size, _ in groups])), _ints([p for _, p in groups])
    s["softmax_scale"] = case["dim"] ** -0.5
    s["q"] = randn(tokens, case["heads"], case["dim"])
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((tokens, case["heads"]), dtype=torch.float32, device="cuda")
    if own:
        import silkern_b200 as silkern

        s["workspace"] = torch.empty(silkern.shared_workspace_bytes(tokens, case["heads"], case["kv_heads"], case["dim"], batch, len(groups)),
                                     dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------------------- plain forms

def _plain_rotate(s):
    case = s["case"]
    start, half = case["start"], case["rotary"] // 2
    angle = s["positions"].double()[:, None] * s["frequencies"].double()
    cos, sin = ((f(angle) * case["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    results = []
    for name in ("q", "k"):
        x, weight = s[name].float(), s[name + "_weight"]
        if weight is not None:
            n = weight.numel()
            x[..., :n] *= (x[..., :n].square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
        r = x[..., start : start + 2 * half]
        a, b = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., :half], r[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        x[..., start : start + 2 * half] = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
        results.append(x.to(s[name].dtype))
    return results


def _slots(case, table, position, rank):
    """(whether the rank holds each position, its slot) through rows of the table."""
    dcp, inter, block = case["dcp"], case["interleave"], case["block"]
    local = position // (dcp * inter) * inter + position % inter
    page = table.gather(-1, (local // block).clamp(max=table.shape[-1] - 1)).long()
    return (position // inter) % dcp == rank, page * block + local % block


def _held(cache, scale, slot, block):
    return cache.flatten(0, 1)[slot].float() * scale[slot // block][..., None]


def _plain_read(s):
    case = s["case"]
    t = torch.arange(case["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    position = s["starts"].long()[seq] + t - s["cu"].long()[seq]
    kept, slot = _slots(case, s["table"][s["req"].long()[seq]].long(), position[:, None], s["rank"])
    kept, slot = kept[:, 0], slot[:, 0]
    result = []
    for out, cache, scale in ((s["keys"], s["k"], s["ks"]), (s["values"], s["v"], s["vs"])):
        if cache is not None:
            out[kept] = _held(cache, scale, slot[kept], case["block"]).to(out.dtype)
            result.append(out)
    return result


def _plain_shared(s):
    case = s["case"]
    block, kv, dim, each = case["block"], case["kv_heads"], case["dim"], case["each"]
    tokens, heads, _ = s["q"].shape
    per = heads // kv
    q = (s["q"].float() * s["softmax_scale"]).view(tokens, kv, per, dim)
    out, lse = torch.empty((tokens, kv, per, dim), device="cuda"), torch.empty((tokens, kv, per), device="cuda")
    most, at, own_lengths = max(_own_lengths(case)), 0, _own_lengths(case)
    for size, prefix in _groups(case):
        rows = slice(at * each, (at + size) * each)
        table = s["table"][s["req"][at : at + size].long()].long()
        kept, slot = _slots(case, table[0], torch.arange(prefix, device="cuda"), s["rank"])
        k, v = (_held(c, f, slot[kept], block) for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
        # Each sequence's own tokens, padded to the longest.
        j = torch.arange(most, device="cuda")[None, :]
        own_length = torch.tensor(own_lengths[at : at + size], device="cuda")[:, None]
        kept, slot = _slots(case, table, (prefix + j).expand(size, most), s["rank"])
        kept = kept & (j < own_length)
        slot = torch.where(kept, slot, 0)
        last = own_length - each + torch.arange(each, device="cuda")  # the last token that each query sees
        seen = kept[:, None] & (j[None] <= last[..., None])  # (size, each, most)
        for h in range(kv):
            x = q[rows, h].reshape(size, each * per, dim)
            before = x.flatten(0, 1) @ k[:, h].T
            ko, vo = (_held(c[:, :, h : h + 1], f[:, h : h + 1], slot, block)[:, :, 0].masked_fill_(~kept[..., None], 0.0)
                      for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            behind = (x @ ko.transpose(1, 2)).masked_fill_(~seen.repeat_interleave(per, 1), -math.inf)
            behind = behind.flatten(0, 1)
            top = behind.amax(-1, keepdim=True)
            if before.shape[1]:
                top = torch.maximum(top, before.amax(-1, keepdim=True))
            base = torch.where(top > -math.inf, top, 0.0)
            before, behind = (before - base).exp_(), (behind - base).exp_()
            total = before.sum(-1, keepdim=True) + behind.sum(-1, keepdim=True)
            y = before @ v[:, h] + (behind.view(size, each * per, most) @ vo).flatten(0, 1)
            out[rows, h] = (y / torch.where(total > 0, total, 1.0)).view(size * each, per, dim)
            lse[rows, h] = (top + total.log()).view(size * each, per)
        at += size
    return out.view(tokens, heads, dim).to(s["q"].dtype), lse.view(tokens, heads)


def run(state):
    if own:
        return _own(state)
    return {"rotate": _plain_rotate, "read": _plain_read, "shared": _plain_shared}[state["case"]["op"]](state)


def _own(s):
    import silkern_b200 as silkern

    case = s["case"]
    if case["op"] == "rotate":
        silkern.rotate_heads(s["q"], s["k"], s["positions"], s["frequencies"], s["q_out"], s["k_out"], q_weight=s["q_weight"],
                             k_weight=s["k_weight"], eps=EPS, rotary_start=case["start"], interleaved=case["interleaved"],
                             amplitude=case["amplitude"])
        return [s["q_out"], s["k_out"]]
    dcp = {"dcp_size": case["dcp"], "dcp_rank": s["rank"], "dcp_interleave": case["interleave"]}
    if case["op"] == "read":
        silkern.read_quantized(s["keys"], s["values"], s["k"], s["v"], s["ks"], s["vs"], s["cu"], s["starts"], s["req"], s["table"], **dcp)
        return [s["keys"]] if case["latent"] else [s["keys"], s["values"]]
    silkern.attend_shared(s["q"], s["cu"], s["lengths"], s["req"], s["cu_groups"], s["prefixes"], s["table"], s["k"], s["v"], s["ks"],
                          s["vs"], s["out"], s["lse"], s["workspace"], softmax_scale=s["softmax_scale"], **dcp)
    return s["out"], s["lse"]


# ------------------------------------------------------------------- the definitions once more, in 64 bits

def _exact_rotate(case, s):
    turn = torch.polar(torch.full((), case["amplitude"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["frequencies"].double()))[:, None]
    first = torch.arange(case["rotary"] // 2, device="cuda")
    first, second = (2 * first, 2 * first + 1) if case["interleaved"] else (first, first + case["rotary"] // 2)
    results = []
    for x, weight in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if weight is not None:
            n = weight.numel()
            size = torch.linalg.vector_norm(y[..., :n], dim=-1, keepdim=True)
            y = torch.cat((y[..., :n] / torch.sqrt(size**2 / n + EPS) * weight.double(), y[..., n:]), -1)
        z = torch.complex(y[..., case["start"] + first], y[..., case["start"] + second]) * turn
        y[..., case["start"] + first], y[..., case["start"] + second] = z.real, z.imag
        results.append(y)
    return results


def _exact_slots(case, s, row, begin, end):
    """Slots of the rank's positions in [begin, end), through one row of the table."""
    run_of = torch.arange(begin // case["interleave"], -(-end // case["interleave"]), device="cuda")
    run_of = run_of[run_of % case["dcp"] == s["rank"]]
    within = torch.arange(case["interleave"], device="cuda")
    position = (run_of[:, None] * case["interleave"] + within).flatten()
    local = (torch.div(run_of, case["dcp"], rounding_mode="floor")[:, None] * case["interleave"] + within).flatten()
    inside = (position >= begin) & (position < end)
    position, local = position[inside], local[inside]
    return position, s["table"][row].long()[local // case["block"]], local % case["block"]


def _exact_read(case, s):
    result = []
    cu, starts, req = s["cu"].tolist(), s["starts"].tolist(), s["req"].tolist()
    for out, cache, scale in ((s["keys"], s["k"], s["ks"]), (s["values"], s["v"], s["vs"])):
        if cache is None:
            continue
        whole = out.double()
        for b in range(case["batch"]):
            position, page, offset = _exact_slots(case, s, req[b], starts[b], starts[b] + cu[b + 1] - cu[b])
            whole[cu[b] - starts[b] + position] = cache[page, offset].double() * scale[page].double()[:, :, None]
        result.append(whole)
    return result


def _exact_shared(case, s):
    each, kv, dim = case["each"], case["kv_heads"], case["dim"]
    lengths, req, at = s["lengths"].tolist(), s["req"].tolist(), 0
    out, lse = s["q"].double(), s["lse"].double()
    for size, prefix in _groups(case):
        def held(row, begin, end):
            position, page, offset = _exact_slots(case, s, row, begin, end)
            k, v = (c[page, offset].double() * f[page].double()[:, :, None] for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            return position, k.transpose(0, 1), v.transpose(0, 1)  # (heads, tokens, dim)
        first = held(req[at], 0, prefix)
        for b in range(at, at + size):
            rows = slice(b * each, (b + 1) * each)
            x = s["q"][rows].double().view(each, kv, -1, dim).transpose(0, 1).reshape(kv, -1, dim)
            parts = [first, held(req[b], prefix, lengths[b])]
            score = torch.cat([x @ k.transpose(1, 2) for _, k, _ in parts], -1) * s["softmax_scale"]
            position = torch.cat([p for p, _, _ in parts])
            limit = lengths[b] - each + torch.arange(each, device="cuda").repeat_interleave(case["heads"] // kv)
            score = torch.where(position <= limit[:, None], score, -math.inf)
            if score.shape[-1] == 0:
                total = torch.full(score.shape[:-1], -math.inf, dtype=torch.float64, device="cuda")
            else:
                total = torch.logsumexp(score, -1)
            weight = torch.where(score > -math.inf, (score - total[..., None]).exp(), 0.0)
            cut = parts[0][0].numel()
            y = weight[..., :cut] @ parts[0][2] + weight[..., cut:] @ parts[1][2]
            out[rows] = y.view(kv, each, -1, dim).transpose(0, 1).reshape(each, -1, dim)
            lse[rows] = total.view(kv, each, -1).transpose(0, 1).reshape(each, -1)
        at += size
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "read": _exact_read, "shared": _exact_shared}[case["op"]](case, s)
