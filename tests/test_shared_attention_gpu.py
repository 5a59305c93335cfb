"""Attention behind shared prefixes, on the device, against 64-bit arithmetic."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import attention as oracle  # noqa: E402
from tests.attention_cases import HALF_STEP, assert_shared, make_cache  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)

TYPES = [torch.bfloat16, torch.float16]


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def sums(counts):
    return ints(*[sum(counts[:i]) for i in range(len(counts) + 1)])


def workspace_of(q, cache, sequences, groups):
    n = silkern.shared_workspace_bytes(q.shape[0], q.shape[1], cache[0].shape[2], q.shape[2], sequences, groups)
    return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN, wherever it is read as numbers


class Batch:
    """Sequences in groups, over a table whose rows name pages of their own."""

    def __init__(self, sizes, prefixes, own, each, *, heads=8, kv_heads=2, dim=128, block=16, dcp=1, dtype=torch.bfloat16, seed=0, alone=0):
        """``sizes`` and ``prefixes`` of the groups; ``own`` tokens behind the prefix and ``each`` queries of each
        sequence; the last ``alone`` sequences belong to no group."""
        n = len(own)
        g = torch.Generator().manual_seed(seed)
        before = [p for size, p in zip(sizes, prefixes) for _ in range(size)] + [0] * alone
        assert len(before) == n
        lengths = [max(b, 0) + o for b, o in zip(before, own)]
        width = max(1, -(-(max(lengths) + 16 * dcp) // (block * dcp)))
        self.cache = make_cache(n * width, block, kv_heads, dim, seed=seed)
        self.table = torch.randperm(n * width, generator=g).to(torch.int32).view(n, width).cuda()
        self.req = torch.randperm(n, generator=g).to(torch.int32).cuda()
        self.cu, self.lengths = sums(each), ints(*lengths)
        self.cu_groups, self.prefixes = sums(sizes), ints(*prefixes)
        self.q = randn(sum(each), heads, dim, dtype=dtype, seed=seed + 1)
        self.scale = dim**-0.5

    def args(self):
        return (self.q, self.cu, self.lengths, self.req, self.cu_groups, self.prefixes, self.table, *self.cache)

    def call(self, out=None, lse=None, work=None, **kw):
        rows, heads, dim = self.q.shape
        out = torch.full((rows, heads, dim), 7.0, dtype=self.q.dtype, device="cuda") if out is None else out
        lse = torch.full((rows, heads), 7.0, device="cuda") if lse is None else lse
        work = workspace_of(self.q, self.cache, self.lengths.numel(), self.prefixes.numel()) if work is None else work
        silkern.attend_shared(*self.args(), out, lse, work, softmax_scale=self.scale, **kw)
        return out, lse

    def check(self, **kw):
        out, lse = self.call(**kw)
        for name in ("status", "out", "lse", "work"):
            kw.pop(name, None)
        first, last = int(self.cu[0]), int(self.cu[-1])
        want = oracle.attend_shared(*self.args(), softmax_scale=self.scale, **kw)
        assert_shared(out[first:last], lse[first:last], want, self.q, self.cache[0], self.cache[2], self.scale)
        for rest in (slice(0, first), slice(last, None)):
            assert bool((out[rest] == 7).all()) and bool((lse[rest] == 7).all())
        return out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 5), (1, 16), (3, 17), (1, 64), (1, 130), (2, 300)])
@pytest.mark.parametrize("prefix", [1, 128, 333])
def test_head_layouts(dtype, dim, kv_heads, group, prefix) -> None:
    Batch([3], [prefix], [1, 40, 129], [1, 1, 1], heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, seed=group).check()


@pytest.mark.parametrize("dim,block", [(64, 32), (128, 64), (128, 17), (64, 1), (128, 256)])
@pytest.mark.parametrize("prefixes", [[0, 0], [-5, 1], [127, 129], [2, 700], [1500, 31]])
@pytest.mark.parametrize("each", [1, 3])
def test_prefixes_groups_and_pages(dim, block, prefixes, each) -> None:
    """Two groups and a sequence of its own, lengths from one token on, several queries to a sequence."""
    own = [each, each + 1, each + 127, each + 128, each + 300, each + 5, each + 60]
    Batch([4, 2], prefixes, own, [each] * 7, dim=dim, block=block, seed=block, alone=1).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dcp,il", [(2, 1), (4, 16), (8, 1), (3, 8)])
def test_ranks(dtype, dcp, il) -> None:
    b = Batch([1, 5], [77, 1000], [1, 2, 3, 100, 500, 20], [1, 1, 3, 1, 2, 1], block=16, dcp=dcp, dtype=dtype, seed=dcp)
    outs, lses = [], []
    for rank in range(dcp):
        out, lse = b.check(dcp_size=dcp, dcp_rank=rank, dcp_interleave=il)
        outs.append(out), lses.append(lse)
    joined, lse = torch.empty_like(outs[0]), torch.empty_like(lses[0])
    silkern.merge_partials(torch.stack(outs), torch.stack(lses), joined, lse)
    # The rounding of each rank's output to the type, and that of the joined one.
    all_tokens = Batch([1, 5], [77, 1000], [1, 2, 3, 100, 500, 20], [1, 1, 3, 1, 2, 1], block=16, dcp=dcp, dtype=dtype, seed=dcp)
    parts = [oracle.attend_shared(*all_tokens.args(), softmax_scale=b.scale, dcp_size=dcp, dcp_rank=r, dcp_interleave=il) for r in range(dcp)]
    want, want_lse, _ = oracle.merge(torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]))
    spread = sum(torch.exp(p[1] - want_lse)[..., None] * p[2] for p in parts)
    assert bool(((joined.double() - want).abs() <= 4 * HALF_STEP[dtype] * spread + 1e-6).all())
    assert float((lse.double() - want_lse).abs().max()) < 2.0**-15


@pytest.mark.parametrize("dim", [64, 128])
def test_many_sequences_and_long_prefixes(dim) -> None:
    n = 70
    own = [1 + 13 * i % 300 for i in range(n)]
    Batch([40, 0, 30], [5000, 99, 2049], own, [1] * n, dim=dim, block=64, heads=16, kv_heads=2, seed=dim).check()


def test_one_long_sequence_among_short_ones() -> None:
    own = [20000] + [5] * 20
    Batch([1], [3], own, [1] * 21, block=64, heads=8, kv_heads=1, seed=3, alone=20).check()


def test_prompt_pieces_and_prefixes_that_queries_stand_in() -> None:
    b = Batch([3], [200], [150, 260, 1], [150, 200, 1], heads=4, kv_heads=2, dim=64, seed=4)
    b.check()
    b.prefixes = ints(270)  # past positions of the first sequence's queries, whose own tokens they see through the first row
    b.check()
    b.prefixes = ints(100000)
    b.check()


def test_cut_tokens_lengths_and_empty_sequences() -> None:
    """Rows before the first and behind the last sequence; sequences without queries; lengths below the queries."""
    b = Batch([2, 3], [60, 130], [3, 4, 5, 6, 7], [1, 1, 1, 1, 1], seed=5)
    b.q = randn(14, 8, 128, dtype=torch.bfloat16, seed=6)
    b.cu = ints(2, 2, 5, 5, 9, 11)
    b.lengths = ints(70, 2, 140, 3, 0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = b.check(status=status)
    assert int(status) == 2
    assert bool((lse[2:3] == -math.inf).all()) and bool((out[9:11] == 0).all())


def test_bad_requests_and_pages_are_left_out_and_flagged() -> None:
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def check(change, want):
        b = Batch([3], [100], [30, 40, 50], [1, 1, 1], seed=7)
        change(b)
        status.zero_()
        b.check(status=status)
        assert int(status) == want

    check(lambda b: None, 0)
    check(lambda b: b.req.__setitem__(1, 3), 1)
    check(lambda b: b.req.__setitem__(0, -1), 1)  # the row of the prefix
    check(lambda b: b.table.__setitem__((int(b.req[0]), 2), b.cache[0].shape[0]), 8)
    check(lambda b: b.table.__setitem__((int(b.req[2]), 8), -1), 8)
    check(lambda b: b.table.__setitem__((int(b.req[2]), 0), -1), 0)  # a prefix's page that is not read
    check(lambda b: setattr(b, "table", b.table[:, :8].contiguous()), 8)


def test_what_nobody_sees_does_not_matter() -> None:
    """NaN codes and scales behind each sequence's end, in others' pages and in the unread pages of the prefix."""
    b = Batch([3], [100], [30, 40, 50], [1, 1, 1], seed=8)
    before = b.call()
    seen = torch.zeros(b.cache[0].shape[:2], dtype=torch.bool)
    table, req = b.table.cpu(), b.req.tolist()
    for i, length in enumerate(b.lengths.tolist()):
        for t in range(length):
            row = req[0] if t < 100 else req[i]
            seen[table[row, t // 16], t % 16] = True
    for codes, scale in ((b.cache[0], b.cache[2]), (b.cache[1], b.cache[3])):
        codes.view(torch.uint8)[~seen.cuda()] = 0x7F
        scale[~seen.any(1).cuda()] = math.nan
    after = b.call()
    assert all(torch.equal(x, y) for x, y in zip(before, after))


def test_nan_reaches_its_readers_only() -> None:
    for part in (2, 3):  # the scale of a page's keys, of its values
        b = Batch([2], [100], [30, 40], [1, 1], heads=6, kv_heads=2, seed=9)
        b.cache[part][int(b.table[int(b.req[1]), 7]), 1] = math.nan  # own tokens of the second
        out, lse = b.call()
        assert bool(out[0].isfinite().all()) and bool(out[1, :3].isfinite().all()) and bool(out[1, 3:].isnan().all())
        assert bool(lse[1, 3:].isnan().all()) == (part == 2)
    b = Batch([2], [100], [30, 40], [1, 1], heads=6, kv_heads=2, seed=9)
    b.q[1, 2, 5] = math.nan
    out, lse = b.call()
    assert bool(out[1, 2].isnan().all()) and bool(lse[1, 2].isnan())
    assert int(out.isnan().any(-1).sum()) == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_queries_of_every_size(dtype, dim) -> None:
    b = Batch([2], [300], [30, 40], [1, 1], heads=8, kv_heads=2, dim=dim, dtype=dtype, seed=10)
    size = torch.tensor([2.0**-14, 2.0**-7, 1.0, 2.0**3, 2.0**6, 0.0, 2.0**-3, 2.0], device="cuda")
    b.q = (b.q.float() * size[:, None]).to(dtype)
    b.q[0, 4, ::2] *= 2.0**-12  # large and small columns side by side
    b.scale = 0.02
    b.check()


@pytest.mark.parametrize("order", ["near", "rising", "falling", "random", "zero"])
def test_value_scales_of_every_size(order) -> None:
    b = Batch([2], [900], [200, 300], [1, 1], heads=8, kv_heads=2, seed=11)
    vs, ks = b.cache[3], b.cache[2]
    n = vs.shape[0]
    g = torch.Generator().manual_seed(12)
    step = {"near": torch.randint(-3, 4, (n,), generator=g), "rising": torch.arange(n) * 190 // n - 95,
            "falling": 95 - torch.arange(n) * 190 // n, "random": torch.randint(-60, 61, (n,), generator=g),
            "zero": torch.randint(-3, 4, (n,), generator=g)}[order]
    place = torch.argsort(b.table[int(b.req[0])].cpu())  # in the prefix's order, for its pages
    scales = torch.ldexp(torch.ones(n), step)
    row = b.table[int(b.req[0])].long().cpu()
    ordered = torch.ldexp(torch.ones(row.numel()), step[torch.linspace(0, n - 1, row.numel()).long()])
    scales[row] = ordered
    if order == "zero":
        scales[row[::3]] = 0.0
    assert place.numel() == row.numel()
    vs.copy_(scales[:, None].expand(n, 2))
    ks.fill_(2.0**-6)
    out, lse = b.call()
    want = oracle.attend_shared(*b.args(), softmax_scale=b.scale)
    assert_shared(out, lse, want, b.q, b.cache[0], b.cache[2], b.scale)


@pytest.mark.parametrize("flip", [False, True])
def test_one_large_weight_does_not_swallow_many_small_ones(flip) -> None:
    b = Batch([2], [130 * 64], [1, 1], [1, 1], heads=16, kv_heads=1, block=64, seed=13)
    k, v, ks, vs = b.cache
    ks.fill_(2.0**-6), vs.fill_(2.0**-6)
    b.q = torch.zeros_like(b.q)
    b.q[..., 127] = 1.0
    codes = k.float()
    codes[..., 127] = 0.0
    at = 130 * 64 - 1 if flip else 0
    codes[int(b.table[int(b.req[0]), at // 64]), at % 64, 0, 127] = 448.0
    k.copy_(codes.to(torch.float8_e4m3fn))
    b.scale = 9.3 / 7.0
    b.check()


def test_scores_that_rise_and_fall_from_run_to_run() -> None:
    """References that have to move at every tile, and scores far below them."""
    for falling in (False, True):
        b = Batch([2], [1500], [100, 120], [1, 1], heads=4, kv_heads=1, block=16, seed=14)
        ks = b.cache[2]
        row = b.table[int(b.req[0])].long()
        size = torch.linspace(2.0**-9, 2.0**-3, row.numel(), device="cuda")
        ks[row] = (size.flip(0) if falling else size)[:, None]
        b.check()


def test_strides_of_queries_outputs_and_caches() -> None:
    b = Batch([2, 1], [140, 20], [30, 40, 9], [1, 2, 1], heads=8, kv_heads=4, dim=64, block=17, seed=15)
    b.cache = make_cache(b.cache[0].shape[0], 17, 4, 64, seed=16, layout="htd")
    b.q = randn(4, 12, 88, dtype=torch.bfloat16, seed=17)[:, 2:10, 8:72]
    store = torch.full((4, 9, 67), 7.0, dtype=torch.bfloat16, device="cuda")
    b.check(out=store[:, 1:, 1:65])
    assert bool((store[:, 0] == 7).all()) and bool((store[:, :, 0] == 7).all()) and bool((store[..., 65:] == 7).all())
    wide = torch.full((8, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    b.check(out=wide.transpose(0, 1))


def test_equal_calls_give_equal_bits_and_agree_with_the_window() -> None:
    b = Batch([5, 6], [3000, 1000], [5, 300, 70, 1, 1, 128, 64, 33, 200, 150, 1000], [1] * 11, heads=32, kv_heads=4, block=64, seed=18)
    for g, (first, last) in enumerate(((0, 5), (5, 11))):  # every row names the shared pages, as a table of copies would
        whole = int(b.prefixes[g]) // 64
        for i in range(first + 1, last):
            b.table[int(b.req[i]), :whole] = b.table[int(b.req[first]), :whole]
    out, lse = b.check()
    for _ in range(3):
        again = b.call()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    b.prefixes = ints(*[int(p) // 64 * 64 for p in b.prefixes])
    out, lse = b.check()
    other, other_lse = torch.empty_like(out), torch.empty_like(lse)
    silkern.attend_window(b.q, b.cu, b.lengths, b.req, b.table, *b.cache, other, other_lse, softmax_scale=b.scale)
    want = oracle.attend_shared(*b.args(), softmax_scale=b.scale)
    # Each within its own bound of the same numbers: twice 2^-8 of the values' mean magnitude, and the outputs' steps.
    assert bool(((out.double() - other.double()).abs() <= 2.0**-6 * want[2]).all())
    assert float((lse - other_lse).abs().max()) < 2.0**-15


@pytest.mark.parametrize("kv_heads,group,dim", [(4, 8, 128), (1, 24, 64), (2, 4, 128)])
def test_ctas_with_items_of_both_sorts(kv_heads, group, dim) -> None:
    """Enough keys for whole runs of tiles in each CTA, behind prefixes of more and of less than 128 rows, so that CTAs go
    from items whose slots take turns to items whose slots go together and back."""
    sizes = [1, 90, 3, 40, 2, 130, 1]
    prefixes = [3000, 2500, 700, 1111, 4000, 900, 64]
    own = [1 + 331 * i % 1500 for i in range(sum(sizes) + 5)]
    Batch(sizes, prefixes, own, [1] * len(own), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, block=64, seed=30, alone=5).check()


@pytest.mark.parametrize("groups,alone", [(3, 1500), (1024, 3), (1025, 3), (1400, 700)])
def test_more_sequences_and_groups_than_a_plan_holds_at_once(groups, alone) -> None:
    sizes = [i % 2 for i in range(groups - 1)] + [2]
    prefixes = [i % 23 for i in range(groups)]
    own = [1 + i % 7 for i in range(sum(sizes) + alone)]
    Batch(sizes, prefixes, own, [(i + 1) % 3 and 1 for i in range(len(own))], heads=2, kv_heads=1, dim=64, seed=33, alone=alone).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_scales_that_are_not_positive(dtype, scale) -> None:
    b = Batch([3], [300], [30, 1, 150], [1, 2, 1], dtype=dtype, seed=31)
    b.scale = scale
    b.check()


def test_equal_requests_and_equal_pages() -> None:
    """Several sequences of one request, and a page that stands twice in a row."""
    b = Batch([3], [200], [30, 40, 50], [1, 1, 1], seed=32)
    b.req[1] = b.req[0]
    b.table[int(b.req[0]), 3] = b.table[int(b.req[0]), 2]
    b.check()


def test_graphs_streams_two_at_once_and_compiled_callers() -> None:
    b = Batch([3], [1000], [30, 40, 150], [1, 1, 2], heads=16, kv_heads=2, seed=19)
    c = Batch([2], [500], [10, 20], [1, 1], heads=16, kv_heads=2, seed=20)
    want_b, want_c = b.check(), c.check()
    torch.cuda.synchronize()
    got = [torch.zeros_like(t) for t in (*want_b, *want_c)]
    work = [workspace_of(x.q, x.cache, x.lengths.numel(), 1) for x in (b, c)]
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        b.call(got[0], got[1], work[0])
        b.call(got[0], got[1], work[0])  # two in a row share a workspace
    with torch.cuda.graph(graphs[1]):
        c.call(got[2], got[3], work[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, (*want_b, *want_c)))
    # new lengths and contents through the same graph
    b.lengths.add_(-5), b.q.mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    again = b.check()
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])

    @torch.compile(fullgraph=True)
    def step(q, out, lse, work):
        silkern.attend_shared(q, b.cu, b.lengths, b.req, b.cu_groups, b.prefixes, b.table, *b.cache, out, lse, work,
                              softmax_scale=b.scale)

    out, lse = torch.zeros_like(again[0]), torch.zeros_like(again[1])
    step(b.q, out, lse, work[0])
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_refusals_on_the_device() -> None:
    b = Batch([2], [100], [30, 40], [1, 1], seed=21)
    out, lse = b.check()
    work = workspace_of(b.q, b.cache, 2, 1)
    names = ("q", "cu_tokens", "lengths", "req_ids", "cu_groups", "prefixes", "block_table", "k_cache", "v_cache", "k_scale", "v_scale")
    good = dict(zip(names, b.args())) | dict(out=out, lse=lse, workspace=work, softmax_scale=0.1)
    silkern.attend_shared(**good)
    latent = make_cache(4, 16, 1, 576, latent=True)
    for bad in (dict(q=b.q[0]), dict(q=b.q.float()), dict(q=b.q[..., :64]), dict(out=out[:1]), dict(out=out.half()), dict(lse=lse.double()),
                dict(cu_tokens=ints(0, 1)), dict(lengths=ints(1, 2, 3)), dict(req_ids=ints(0)), dict(cu_groups=ints(0)),
                dict(prefixes=ints(1, 2)), dict(prefixes=ints(1).long()), dict(prefixes=ints()), dict(block_table=b.table[0]),
                dict(block_table=b.table.T), dict(workspace=work[:-1]), dict(workspace=work[::2]), dict(workspace=torch.empty(2, device="cuda")),
                dict(workspace=work.cpu()), dict(softmax_scale=math.inf), dict(softmax_scale="x"), dict(dcp_size=0), dict(dcp_rank=1),
                dict(dcp_interleave=3), dict(v_cache=None, v_scale=None), dict(out=b.q), dict(lse=lse[:, :1].expand(2, 8)),
                dict(status=torch.zeros(1, device="cuda")), dict(workspace=out)):
        with pytest.raises(silkern.LocalizationError):
            silkern.attend_shared(**{**good, **bad})
    with pytest.raises(silkern.LocalizationError):
        silkern.attend_shared(torch.zeros(2, 8, 576, dtype=torch.bfloat16, device="cuda"), *b.args()[1:7], *latent,
                              torch.empty(2, 8, 512, dtype=torch.bfloat16, device="cuda"), lse, work, softmax_scale=0.1)


def test_places_past_32_bits() -> None:
    """A cache whose last pages lie past 4 GiB."""
    blocks = (1 << 32) // (64 * 2 * 128) + 40
    k = torch.zeros((blocks, 64, 2, 128), dtype=torch.float8_e4m3fn, device="cuda")
    v = torch.zeros_like(k)
    b = Batch([2], [300], [30, 40], [1, 1], heads=8, kv_heads=2, block=64, seed=22)
    n = b.cache[0].shape[0]
    k[-n:], v[-n:] = b.cache[0], b.cache[1]
    ks, vs = torch.zeros((blocks, 2), device="cuda"), torch.zeros((blocks, 2), device="cuda")
    ks[-n:], vs[-n:] = b.cache[2], b.cache[3]
    want = b.check()
    b.table += blocks - n
    b.cache = (k, v, ks, vs)
    got = b.call()
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_a_step_from_projections_to_outputs() -> None:
    """rotate, append and attend, as one step of a server: against 64-bit arithmetic on what the cache then holds."""
    n, heads, kv_heads, dim, prefix = 6, 16, 2, 128, 200
    frequencies, amplitude = silkern.rotary_frequencies(dim, factor=4.0, method="parts", original_length=4096, device="cuda")
    width, blocks = 5, 40
    table = torch.randperm(blocks, generator=torch.Generator().manual_seed(23))[: n * width].to(torch.int32).view(n, width).cuda()
    cache = [torch.zeros((blocks, 64, kv_heads, dim), dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
    scales = [torch.zeros((blocks, kv_heads), device="cuda") for _ in range(2)]
    weight = torch.ones(dim, device="cuda")

    def put(x, values, positions, cu, starts, req):
        silkern.rotate_heads(x[:, :heads], x[:, heads:], positions, frequencies, x[:, :heads], x[:, heads:], q_weight=weight,
                             k_weight=weight, amplitude=amplitude)
        silkern.append_quantized(x[:, heads:], values, *cache, *scales, cu, starts, req, table)

    # The prefix by the first sequence, then one token of every sequence.
    x = randn(prefix, heads + kv_heads, dim, dtype=torch.bfloat16, seed=24)
    put(x, randn(prefix, kv_heads, dim, dtype=torch.bfloat16, seed=25), torch.arange(prefix, dtype=torch.int32).cuda(), ints(0, prefix),
        ints(0), ints(0))
    x = randn(n, heads + kv_heads, dim, dtype=torch.bfloat16, seed=26)
    order = ints(0, 1, 2, 3, 4, 5)
    put(x, randn(n, kv_heads, dim, dtype=torch.bfloat16, seed=27), torch.full((n,), prefix, dtype=torch.int32).cuda(),
        sums([1] * n), torch.full((n,), prefix, dtype=torch.int32).cuda(), order)
    args = (x[:, :heads], sums([1] * n), torch.full((n,), prefix + 1, dtype=torch.int32).cuda(), order, ints(0, n), ints(prefix), table,
            *cache, *scales)
    out, lse = torch.empty((n, heads, dim), dtype=torch.bfloat16, device="cuda"), torch.empty((n, heads), device="cuda")
    work = workspace_of(x[:, :heads], (cache[0],), n, 1)
    silkern.attend_shared(*args, out, lse, work, softmax_scale=dim**-0.5)
    want = oracle.attend_shared(*args, softmax_scale=dim**-0.5)
    assert_shared(out, lse, want, x[:, :heads], cache[0], scales[0], dim**-0.5)
    keys, values = torch.zeros((prefix, kv_heads, dim), dtype=torch.bfloat16, device="cuda"), torch.zeros((prefix, kv_heads, dim), dtype=torch.bfloat16, device="cuda")
    silkern.read_quantized(keys, values, *cache, *scales, ints(0, prefix), ints(0), ints(0), table)
    assert bool((keys != 0).any(-1).all()) and bool((values != 0).any(-1).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 64), (10, 2, 128)])
def test_prompts_of_many_blocks_behind_a_prefix(dtype, heads, kv_heads, dim) -> None:
    """Own segments of dozens of blocks, each over keys up to its last query's, beside short ones and behind a prefix."""
    each = [1500, 1, 700, 333]
    Batch([3], [777], [n + 20 * (n % 2) for n in each], each, heads=heads, kv_heads=kv_heads, dim=dim, block=64, dtype=dtype, seed=40,
          alone=1).check()


def test_value_scales_farther_apart_than_the_first_tiles_reach() -> None:
    """Pages of the prefix whose value scales rise, or fall, by more than 2^4 and 2^6 in steps: the second reference
    takes over in the middle, and the small ones' share of the outputs is theirs."""
    for falling in (False, True):
        b = Batch([2], [900], [200, 300], [1, 1], heads=8, kv_heads=2, seed=41)
        pages = b.table[int(b.req[0])].long()
        step = torch.arange(pages.numel(), device="cuda") // 8 * 3 - 10
        assert int(step[:57].max() - step[0]) > 10  # 57 pages of 16 hold the prefix; a tile is 8 of them
        b.cache[3][pages] = torch.ldexp(torch.ones(pages.numel(), device="cuda"), step.flip(0) if falling else step)[:, None]
        b.check()
