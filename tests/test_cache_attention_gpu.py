"""Attention over the 8-bit cache, on the device, against 64-bit arithmetic."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import attention as oracle  # noqa: E402
from tests.attention_cases import HALF_STEP, assert_attention, make_cache  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)

SHAPES = {"d64": (64, 64, False), "d128": (128, 128, False), "latent": (576, 512, True)}
TYPES = [torch.bfloat16, torch.float16]


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def results(rows, heads, value_dim, dtype):
    return (torch.full((rows, heads, value_dim), 7.0, dtype=dtype, device="cuda"),
            torch.full((rows, heads), 7.0, dtype=torch.float32, device="cuda"))


def selected(q, slots, cache, value_dim, **kw):
    out, lse = results(q.shape[0], q.shape[1], value_dim, q.dtype)
    silkern.attend_selected(q, slots, *cache, out, lse, **kw)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 5), (1, 16), (3, 17), (1, 33), (1, 64), (1, 130)])
@pytest.mark.parametrize("width", [1, 127, 129, 700])
def test_selected_head_layouts_and_widths(shape, dtype, kv_heads, group, width) -> None:
    dim, value_dim, latent = SHAPES[shape]
    if latent and kv_heads > 1:
        pytest.skip("a latent cache has one head")
    cache = make_cache(11, 48, kv_heads, dim, latent=latent, seed=width)
    rows = 3
    g = torch.Generator().manual_seed(width + group)
    slots = torch.randint(0, 11 * 48, (rows, width), generator=g, dtype=torch.int32)
    slots[torch.rand((rows, width), generator=g) < 0.2] = -1
    slots[1] = -1  # a row without a slot
    counts = torch.tensor([width, width, max(0, width - 5)], dtype=torch.int32).cuda()
    slots = slots.cuda()
    q = randn(rows, kv_heads * group, dim, dtype=dtype, seed=group)
    scale = dim**-0.5
    for use in (None, counts):
        out, lse = selected(q, slots, cache, value_dim, softmax_scale=scale, counts=use)
        want = oracle.attend_selected(q, slots, *cache, softmax_scale=scale, counts=use)
        assert_attention(out, lse, want, q, cache[0], cache[2], scale)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rows,width", [(1, 16384), (5, 4096), (40, 1000), (300, 257)])
def test_selected_long_rows_and_batches(shape, rows, width) -> None:
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(300, 64, 1, dim, latent=latent, seed=3)
    g = torch.Generator().manual_seed(rows)
    slots = torch.randint(0, 300 * 64, (rows, width), generator=g, dtype=torch.int32)
    counts = torch.randint(0, width + 1, (rows,), generator=g, dtype=torch.int32)
    counts[0] = width
    for r in range(rows):
        slots[r, counts[r]:] = -1
    slots, counts = slots.cuda(), counts.cuda()
    q = randn(rows, 16, dim, dtype=torch.bfloat16, seed=5) * 2
    out, lse = selected(q, slots, cache, value_dim, softmax_scale=dim**-0.5, counts=counts)
    want = oracle.attend_selected(q, slots, *cache, softmax_scale=dim**-0.5, counts=counts)
    assert_attention(out, lse, want, q, cache[0], cache[2], dim**-0.5)


@pytest.mark.parametrize("shape", ["d64", "d128"])
def test_selected_strides_and_layouts(shape) -> None:
    dim, value_dim, _ = SHAPES[shape]
    cache = make_cache(9, 17, 4, dim, seed=1, layout="htd")
    wide = torch.randint(-1, 9 * 17, (6, 400), generator=torch.Generator().manual_seed(2), dtype=torch.int32).cuda()
    slots = wide[::2, 5:305]
    q = randn(3, 12, dim + 24, dtype=torch.bfloat16, seed=3)[:, :8, 8 : 8 + dim]
    store = torch.full((3, 9, value_dim + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = store[:, 1:, 1 : 1 + value_dim], torch.empty((3, 8), device="cuda")
    silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=0.1)
    want = oracle.attend_selected(q, slots, *cache, softmax_scale=0.1)
    assert_attention(out, lse, want, q, cache[0], cache[2], 0.1)
    assert bool((store[:, 0] == 7).all()) and bool((store[:, :, 0] == 7).all()) and bool((store[..., 1 + value_dim:] == 7).all())


def test_selected_bad_slots_and_counts_are_left_out_and_flagged() -> None:
    cache = make_cache(4, 16, 2, 128, seed=4)
    slots = torch.randint(0, 64, (4, 150), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).cuda()
    q = randn(4, 4, 128, dtype=torch.bfloat16, seed=6)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = selected(q, slots, cache, 128, softmax_scale=0.09, status=status)
    assert status.item() == 0
    slots[1, 70] = 64
    slots[2, 3] = 2**31 - 1
    out, lse = selected(q, slots, cache, 128, softmax_scale=0.09, status=status)
    assert status.item() == 8
    assert_attention(out, lse, oracle.attend_selected(q, slots, *cache, softmax_scale=0.09), q, cache[0], cache[2], 0.09)
    status.zero_()
    counts = torch.tensor([-3, 151, 150, 0], dtype=torch.int32).cuda()
    slots.clamp_(max=63)
    out, lse = selected(q, slots, cache, 128, softmax_scale=0.09, counts=counts, status=status)
    assert status.item() == 2
    want = oracle.attend_selected(q, slots, *cache, softmax_scale=0.09, counts=counts)
    assert_attention(out, lse, want, q, cache[0], cache[2], 0.09)


@pytest.mark.parametrize("shape", SHAPES)
def test_what_is_not_selected_does_not_matter(shape) -> None:
    """NaN codes, NaN and infinite scales in pages and tokens that no slot names."""
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(8, 32, 1, dim, latent=latent, seed=7)
    g = torch.Generator().manual_seed(8)
    slots = torch.randint(0, 6 * 32, (2, 200), generator=g, dtype=torch.int32)
    slots = torch.where(slots % 32 < 30, slots, -1).cuda()
    q = randn(2, 16, dim, dtype=torch.bfloat16, seed=9)
    before = selected(q, slots, cache, value_dim, softmax_scale=0.05)
    for codes, scale in ((cache[0], cache[2]), (cache[1], cache[3])):
        if codes is not None:
            codes.view(torch.uint8)[:, 30:] = 0x7F
            codes.view(torch.uint8)[6:] = 0xFF
            scale[6], scale[7] = math.nan, math.inf
    after = selected(q, slots, cache, value_dim, softmax_scale=0.05)
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_a_scale_that_is_not_a_number_reaches_its_readers_only() -> None:
    cache = make_cache(4, 16, 2, 64, seed=10)
    slots = torch.arange(64, dtype=torch.int32).view(2, 32).cuda()
    q = randn(2, 6, 64, dtype=torch.float16, seed=11)
    cache[2][3, 1] = math.nan
    out, lse = selected(q, slots, cache, 64, softmax_scale=0.125)
    assert bool(out[0].isfinite().all()) and bool(out[1, :3].isfinite().all())
    assert bool(out[1, 3:].isnan().all()) and bool(lse[1, 3:].isnan().all())


@pytest.mark.parametrize("shape", SHAPES)
def test_one_large_weight_does_not_swallow_many_small_ones(shape) -> None:
    """A first token far above the rest, whose many weights still add up (an
    attention sink), in both orders."""
    dim, value_dim, latent = SHAPES[shape]
    blocks = 130
    cache = make_cache(blocks, 64, 1, dim, latent=latent, seed=12)
    k, v, ks, vs = cache
    ks.fill_(2.0**-6)
    if vs is not None:
        vs.fill_(2.0**-6)
    q = torch.zeros((2, 16, dim), dtype=torch.bfloat16, device="cuda")
    q[..., dim - 1] = 1.0
    codes = k.float()
    codes[..., dim - 1] = 0.0
    codes[0, 0, 0, dim - 1] = 448.0  # 7.0 in the last column, times the scale below: 9.3 nats above the rest
    k.copy_(codes.to(torch.float8_e4m3fn))
    order = torch.arange(blocks * 64, dtype=torch.int32).cuda()
    slots = torch.stack([order, order.flip(0)])
    scale = 9.3 / 7.0
    out, lse = selected(q, slots, cache, value_dim, softmax_scale=scale)
    want = oracle.attend_selected(q, slots, *cache, softmax_scale=scale)
    assert_attention(out, lse, want, q, k, ks, scale)


def test_scales_far_apart() -> None:
    """Pages whose value scales are 2**90 apart: the output follows the values
    that the weights leave, whichever page has them."""
    cache = make_cache(6, 32, 1, 128, seed=13)
    cache[3][:, 0] = torch.tensor([2.0**-45, 2.0**45, 1.0, 0.0, 2.0**-20, 2.0**-45]).cuda()
    q = randn(4, 8, 128, dtype=torch.bfloat16, seed=14)
    rows = [[0, 5], [0, 2], [1, 4], [3, 4]]
    slots = torch.stack([torch.cat([torch.arange(32 * p, 32 * p + 32) for p in r]) for r in rows]).to(torch.int32).cuda()
    out, lse = selected(q, slots, cache, 128, softmax_scale=0.09)
    assert_attention(out, lse, oracle.attend_selected(q, slots, *cache, softmax_scale=0.09), q, cache[0], cache[2], 0.09)


def window_case(lengths, new, *, dim, latent, kv_heads, heads, block_size, dcp, rank, interleave, dtype, seed, extra=0,
                layout="thd"):
    g = torch.Generator().manual_seed(seed)
    width = max(1, -(-(max(lengths) + dcp * interleave) // (dcp * block_size)))
    n = len(lengths)
    cache = make_cache(n * width, block_size, kv_heads, dim, latent=latent, seed=seed, layout=layout)
    table = torch.randperm(n * width, generator=g).to(torch.int32).view(n, width).cuda()
    req = torch.randperm(n, generator=g).to(torch.int32).cuda()
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    q = randn(sum(new) + extra, heads, dim, dtype=dtype, seed=seed + 1)
    return q, cu, torch.tensor(lengths, dtype=torch.int32).cuda(), req, table, cache, dict(
        dcp_size=dcp, dcp_rank=rank, dcp_interleave=interleave)


def check_window(q, cu, lengths, req, table, cache, value_dim, **kw):
    out, lse = results(q.shape[0], q.shape[1], value_dim, q.dtype)
    silkern.attend_window(q, cu, lengths, req, table, *cache, out, lse, **kw)
    torch.cuda.synchronize()
    kw.pop("status", None)
    n = int(cu[-1])
    want = oracle.attend_window(q, cu, lengths, req, table, *cache, **kw)
    assert_attention(out[:n], lse[:n], want, q, cache[0], cache[2], kw["softmax_scale"])
    assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all())
    return out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 4), (128, 0), (300, 129), (5000, 4)])
@pytest.mark.parametrize("dcp,rank,interleave,block_size", [(1, 0, 1, 64), (4, 3, 1, 17), (2, 0, 16, 48)])
def test_window_decode(shape, dtype, window, sinks, dcp, rank, interleave, block_size) -> None:
    dim, value_dim, latent = SHAPES[shape]
    lengths = [1, 2, 130, 513, 1900, 17, 128]
    case = window_case(lengths, [1] * 7, dim=dim, latent=latent, kv_heads=1 if latent else 2, heads=10, block_size=block_size,
                       dcp=dcp, rank=rank, interleave=interleave, dtype=dtype, seed=window + sinks)
    q, cu, lens, req, table, cache, own = case
    check_window(q, cu, lens, req, table, cache, value_dim, softmax_scale=dim**-0.5, window=window, sinks=sinks, **own)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads", [2, 6, 20, 64])
@pytest.mark.parametrize("window,sinks,dcp", [(0, 0, 1), (64, 3, 1), (129, 1, 2), (1, 130, 1)])
def test_window_prompt_pieces(shape, dtype, heads, window, sinks, dcp) -> None:
    dim, value_dim, latent = SHAPES[shape]
    lengths, new = [150, 7, 301, 40], [150, 0, 33, 1]
    case = window_case(lengths, new, dim=dim, latent=latent, kv_heads=1 if latent else 2, heads=heads, block_size=32,
                       dcp=dcp, rank=dcp - 1, interleave=1, dtype=dtype, seed=heads, extra=3)
    q, cu, lens, req, table, cache, own = case
    check_window(q, cu, lens, req, table, cache, value_dim, softmax_scale=dim**-0.5, window=window, sinks=sinks, **own)


@pytest.mark.parametrize("shape", SHAPES)
def test_window_one_long_sequence(shape) -> None:
    dim, value_dim, latent = SHAPES[shape]
    case = window_case([40001], [1], dim=dim, latent=latent, kv_heads=1, heads=8, block_size=64, dcp=1, rank=0,
                       interleave=1, dtype=torch.bfloat16, seed=5, layout="thd" if latent else "htd")
    q, cu, lens, req, table, cache, own = case
    check_window(q, cu, lens, req, table, cache, value_dim, softmax_scale=dim**-0.5, **own)


def test_window_many_short_sequences() -> None:
    lengths = [1 + (7 * i) % 300 for i in range(1500)]
    new = [min(lengths[i], (i * i) % 4) for i in range(1500)]
    q, cu, lens, req, table, cache, own = window_case(lengths, new, dim=64, latent=False, kv_heads=1, heads=3, block_size=16,
                                                      dcp=1, rank=0, interleave=1, dtype=torch.bfloat16, seed=2)
    check_window(q, cu, lens, req, table, cache, 64, softmax_scale=0.125, window=50, sinks=2, **own)


def test_window_bad_requests_lengths_and_pages_are_flagged() -> None:
    q, cu, lens, req, table, cache, own = window_case([100, 200, 64], [1, 1, 1], dim=128, latent=False, kv_heads=2, heads=8,
                                                      block_size=16, dcp=1, rank=0, interleave=1, dtype=torch.bfloat16, seed=3)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(softmax_scale=0.1, status=status, **own)
    check_window(q, cu, lens, req, table, cache, 128, **kw)
    assert status.item() == 0
    for request in (-1, 3, 2**31 - 1):
        status.zero_()
        bad = req.clone()
        bad[1] = request
        out, lse = check_window(q, cu, lens, bad, table, cache, 128, **kw)
        assert status.item() == 1 and bool((out[1] == 0).all())
    status.zero_()
    short = lens.clone()
    short[2] = 0
    out, _ = check_window(q, cu, short, req, table, cache, 128, **kw)
    assert status.item() == 2 and bool((out[2] == 0).all())
    for entry in (-1, table.numel(), 2**31 - 1):
        status.zero_()
        worse = table.clone()
        worse[req[0], 2] = entry
        check_window(q, cu, lens, req, worse, cache, 128, **kw)
        assert status.item() == 8
    status.zero_()
    longer = lens.clone()
    longer[1] = table.shape[1] * 16 + 40  # past the table row: the tokens there are left out
    check_window(q, cu, longer, req, table, cache, 128, **kw)
    assert status.item() == 8


def test_window_hidden_tokens_do_not_matter() -> None:
    """NaN codes before the window, past the length, and in pages not seen."""
    q, cu, lens, req, table, cache, own = window_case([300, 77], [1, 1], dim=64, latent=False, kv_heads=1, heads=4,
                                                      block_size=16, dcp=1, rank=0, interleave=1, dtype=torch.bfloat16, seed=4)
    kw = dict(softmax_scale=0.125, window=50, sinks=3, **own)
    before = check_window(q, cu, lens, req, table, cache, 64, **kw)
    seen = torch.zeros(cache[0].shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate([300, 77]):
        for p in list(range(3)) + list(range(n - 50, n)):
            seen[table[req[b], p // 16], p % 16] = True
    for codes in (cache[0], cache[1]):
        codes.view(torch.uint8)[~seen] = 0x7F
    out, lse = results(2, 4, 64, q.dtype)
    silkern.attend_window(q, cu, lens, req, table, *cache, out, lse, **kw)
    assert torch.equal(out, before[0]) and torch.equal(lse, before[1])


def test_captured_replayed_and_on_another_stream() -> None:
    cache = make_cache(64, 64, 1, 576, latent=True, seed=20)
    slots = torch.randint(0, 4096, (6, 900), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).cuda()
    q = randn(6, 40, 576, dtype=torch.bfloat16, seed=21)
    out, lse = results(6, 40, 512, q.dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=0.04)
    side.synchronize()
    want = out.clone(), lse.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=0.04)
    for _ in range(20):
        out.zero_(), lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    slots.copy_(slots.flip(1))
    slots[:, 400:] = -1
    graph.replay()
    torch.cuda.synchronize()
    assert_attention(out, lse, oracle.attend_selected(q, slots, *cache, softmax_scale=0.04), q, cache[0], cache[2], 0.04)


def test_calls_on_two_streams_at_once() -> None:
    """Kernels of unlike shapes that share the GPU give what they give alone."""
    small, latent = make_cache(200, 64, 4, 128, seed=30), make_cache(200, 64, 1, 576, latent=True, seed=31)
    g = torch.Generator().manual_seed(32)
    slots = torch.randint(0, 200 * 64, (90, 1024), dtype=torch.int32, generator=g).cuda()
    qs, ql = randn(90, 32, 128, dtype=torch.bfloat16, seed=33), randn(90, 64, 576, dtype=torch.bfloat16, seed=34)
    wants = (selected(qs, slots, small, 128, softmax_scale=0.09), selected(ql, slots, latent, 512, softmax_scale=0.04))
    outs = [results(90, 32, 128, torch.bfloat16), results(90, 64, 512, torch.bfloat16)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, q, cache, (out, lse), scale in zip(streams, (qs, ql), (small, latent), outs, (0.09, 0.04)):
            with torch.cuda.stream(stream):
                silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=scale)
    torch.cuda.synchronize()
    for got, want in zip(outs, wants):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------------ append

def same_cache(got, want):
    for a, b in zip(got, want):
        if a is None:
            assert b is None
        elif a.dtype == torch.float32:
            assert torch.equal(a.nan_to_num(-5.0), b.nan_to_num(-5.0))
        else:
            assert torch.equal(a.float().nan_to_num(-5.0), b.float().nan_to_num(-5.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("latent,kv_heads,dim", [(False, 3, 64), (False, 8, 128), (True, 1, 576)])
@pytest.mark.parametrize("dcp,rank,interleave,block_size", [(1, 0, 1, 64), (2, 1, 1, 16), (4, 2, 8, 8), (3, 0, 5, 15)])
def test_append_is_the_definition_bit_for_bit(dtype, latent, kv_heads, dim, dcp, rank, interleave, block_size) -> None:
    g = torch.Generator().manual_seed(dim + dcp)
    starts, new = [0, 5, 31, 64, 200, 3, 100], [70, 1, 0, 1, 300, 2, 130]
    n, width = len(new), 40
    cache = [t if t is None else t.clone() for t in make_cache(n * width, block_size, kv_heads, dim, latent=latent, seed=1)]
    before = [t if t is None else t.clone() for t in cache]
    table = torch.randperm(n * width, generator=g).to(torch.int32).view(n, width).cuda()
    req = torch.randperm(n, generator=g).to(torch.int32).cuda()
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    at = torch.tensor(starts, dtype=torch.int32).cuda()
    size = torch.exp(torch.randn((sum(new), 1, 1), generator=g) * 3)
    keys = (torch.randn((sum(new), kv_heads, dim), generator=g) * size).to(dtype).cuda()
    values = None if latent else (torch.randn((sum(new), kv_heads, dim), generator=g) * size).to(dtype).cuda()
    own = dict(dcp_size=dcp, dcp_rank=rank, dcp_interleave=interleave)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    silkern.append_quantized(keys, values, *cache, cu, at, req, table, status=status, **own)
    torch.cuda.synchronize()
    assert status.item() == 0
    same_cache(cache, oracle.append(keys, values, *before, cu, at, req, table, **own))


def test_append_token_by_token_is_append_at_once() -> None:
    """Powers of two: the order of growth leaves no trace in codes that stay
    normal, and here every token's codes do (largest over smallest magnitude
    below 2**13)."""
    x = (1 + torch.rand((50, 2, 64), generator=torch.Generator().manual_seed(3))) * torch.exp2(
        torch.arange(50) % 7 - 3.0)[:, None, None]
    x = x.to(torch.bfloat16).cuda()
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    whole = [t.clone() for t in make_cache(4, 16, 2, 64, seed=5)]
    single = [t.clone() for t in whole]
    silkern.append_quantized(x, x, *whole, ints(0, 50), ints(0), ints(0), table)
    for i in range(50):
        silkern.append_quantized(x[i : i + 1], x[i : i + 1], *single, ints(0, 1), ints(i), ints(0), table)
    torch.cuda.synchronize()
    for a, b in zip(whole, single):
        if a.dtype == torch.float32:
            assert torch.equal(a, b)
        else:
            a, b = (t[table[0].long()].reshape(64, 2, 64)[:50].float() for t in (a, b))
            assert torch.equal(a, b)


def test_append_odd_values() -> None:
    """Zeros, infinities, NaN, the type's largest and smallest magnitudes, and a
    page that is used again after each."""
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    table = ints(0, 1).view(1, 2)
    for value in (0.0, math.inf, -math.inf, math.nan, 3.3e38, 1e-38, 448.0, 449.0, -2.0**-40):
        cache = [t.clone() for t in make_cache(2, 8, 1, 64, seed=6)]
        x = torch.randn((6, 1, 64), generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).cuda()
        if value == 0.0:
            x.zero_()
        x[4, 0, 9] = value
        for start in (0, 5, 0):
            new = x if start != 5 else x[:2]
            before = [t.clone() for t in cache]
            cu = ints(0, new.shape[0])
            silkern.append_quantized(new, new, *cache, cu, ints(start), ints(0), table)
            torch.cuda.synchronize()
            same_cache(cache, oracle.append(new, new, *before, cu, ints(start), ints(0), table))
        if not math.isfinite(value):
            assert bool(cache[2][0].isnan().all())
    cache = [t.clone() for t in make_cache(2, 8, 1, 64, seed=6)]
    cache[2].fill_(math.nan)
    one = torch.ones((1, 1, 64), dtype=torch.float16, device="cuda")
    silkern.append_quantized(one, one, *cache, ints(0, 1), ints(3), ints(0), table)
    assert bool(cache[2][0].isnan().all())
    silkern.append_quantized(one, one, *cache, ints(0, 1), ints(0), ints(0), table)
    assert cache[2][0].item() == 2.0**-8


def test_append_leaves_the_rest_alone_and_flags_what_it_skips() -> None:
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.randn((12, 1, 64), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    table = ints(0, 1, 2, 3).view(2, 2)
    for starts, req, entry, bit in (((0, 0), (0, 2), None, 1), ((0, 0), (-1, 1), None, 1), ((-4, 0), (0, 1), None, 2),
                                    ((2**31 - 2, 0), (0, 1), None, 2), ((28, 0), (0, 1), None, 8), ((0, 0), (0, 1), -1, 8),
                                    ((0, 0), (0, 1), 4, 8)):
        cache = [t.clone() for t in make_cache(4, 16, 1, 64, seed=9)]
        before = [t.clone() for t in cache]
        use = table.clone()
        if entry is not None:
            use[0, 0] = entry
        status.zero_()
        silkern.append_quantized(x, x, *cache, ints(0, 6, 9), ints(*starts), ints(*req), use, status=status)
        torch.cuda.synchronize()
        assert status.item() == bit
        touched = {int(use[r, p // 16]) for b, r in enumerate(req) if 0 <= r < 2 and 0 <= starts[b] < 2**31 - 10
                   for p in range(starts[b], starts[b] + (6, 3)[b]) if p // 16 < 2}
        for page in range(4):
            for a, b in zip(cache, before):
                same = torch.equal(a[page].float(), b[page].float())
                if page not in touched:
                    assert same, (starts, req, entry, page)
                elif a.dtype == torch.float8_e4m3fn:  # a scale stays where it reaches the new tokens as well
                    assert not same, (starts, req, entry, page)


# ------------------------------------------------------------------------------------------------- merge

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ranks,rows,heads,dim", [(1, 1, 1, 1), (2, 3, 5, 64), (8, 17, 16, 512), (3, 2, 7, 33), (70, 2, 3, 128)])
def test_merge(dtype, ranks, rows, heads, dim) -> None:
    outs = randn(ranks, rows, heads, dim, dtype=dtype, seed=1)
    lses = (torch.randn((ranks, rows, heads), generator=torch.Generator().manual_seed(2)) * 20).cuda()
    if ranks > 1:
        lses[0, 0] = -math.inf
        outs[0, 0] = math.nan  # what an empty rank leaves is not read
    if rows > 1:
        lses[:, 1, 0] = -math.inf
    out, lse = results(rows, heads, dim, dtype)
    silkern.merge_partials(outs, lses, out, lse)
    want, want_lse, spread = oracle.merge(outs, lses)
    u = HALF_STEP[dtype]
    # half a step of the output, plus (ranks + 8) roundings of float32 in sum, exponential and quotient;
    # an exponent below 100 in size is itself 2**-17 off at most
    bound = u * want.abs() + ((ranks + 8) * 2.0**-23 + 2.0**-16) * spread + 2.0**-25
    assert bool(((out.double() - want).abs() <= bound).all())
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and bool((out[empty] == 0).all())
    assert bool(((lse.double() - want_lse)[~empty].abs() <= (ranks + 8) * 2.0**-23 + 2.0**-22 * want_lse[~empty].abs()).all())
    silkern.merge_partials(outs, lses, out)  # lse is optional


def test_merge_strides() -> None:
    outs = randn(3, 5, 12, 72, dtype=torch.bfloat16, seed=3).transpose(1, 2)[:, 1:, :, 3:68]
    lses = torch.randn((3, 11, 5), generator=torch.Generator().manual_seed(4)).cuda()
    store = torch.full((11, 6, 70), 7.0, dtype=torch.bfloat16, device="cuda")
    out = store[:, 1:, 2:67]
    silkern.merge_partials(outs, lses, out)
    want, _, spread = oracle.merge(outs, lses)
    assert bool(((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-16 * spread).all())
    assert bool((store[:, 0] == 7).all()) and bool((store[..., :2] == 7).all()) and bool((store[..., 67:] == 7).all())


# ------------------------------------------------------------------------------------------ the whole step

@pytest.mark.parametrize("latent", [False, True])
def test_a_decode_step_over_ranks_is_attention_over_the_whole_selection(latent) -> None:
    """Append a prompt and a token on every rank, select with the fused top-k,
    attend to the localized slots, merge: the result of one rank that has all,
    within the roundings of the partial outputs. Captured in one graph."""
    dim, value_dim = (576, 512) if latent else (128, 128)
    kv_heads, heads, block_size, dcp, batch, length, top_k = (1 if latent else 2), 16, 16, 4, 3, 500, 128
    g = torch.Generator().manual_seed(40)
    x = torch.randn((batch * length, kv_heads, dim), generator=g).to(torch.bfloat16).cuda()
    y = None if latent else torch.randn((batch * length, kv_heads, dim), generator=g).to(torch.bfloat16).cuda()
    cu = torch.arange(0, batch * length + 1, length, dtype=torch.int32).cuda()
    zero, req = torch.zeros(batch, dtype=torch.int32).cuda(), torch.arange(batch, dtype=torch.int32).cuda()
    logits = torch.randn((batch, length), generator=g).cuda()
    lens = torch.full((batch,), length, dtype=torch.int32).cuda()
    q = torch.randn((batch, heads, dim), generator=g).to(torch.bfloat16).cuda()
    scale = dim**-0.5

    def rank_state(size):
        width = -(-length // (size * block_size)) + 1
        cache = [t if t is None else t.clone() for t in make_cache(batch * width, block_size, kv_heads, dim, latent=latent, seed=size)]
        table = torch.randperm(batch * width, generator=g).to(torch.int32).view(batch, width).cuda()
        slots = torch.empty((batch, top_k), dtype=torch.int32, device="cuda")
        return cache, table, slots, torch.empty(batch, dtype=torch.int32, device="cuda")

    def step(state, size, rank, out, lse):
        cache, table, slots, counts = state
        own = dict(dcp_size=size, dcp_rank=rank)
        silkern.append_quantized(x, y, *cache, cu, zero, req, table, **own)
        silkern.topk_localize(logits, lens, req, table, slots, counts, block_size=block_size, **own)
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=scale, counts=counts if size > 1 else None)

    whole, whole_lse = results(batch, heads, value_dim, torch.bfloat16)
    alone = rank_state(1)
    step(alone, 1, 0, whole, whole_lse)
    outs = torch.empty((dcp, batch, heads, value_dim), dtype=torch.bfloat16, device="cuda")
    lses = torch.empty((dcp, batch, heads), device="cuda")
    out, lse = results(batch, heads, value_dim, torch.bfloat16)
    states = [rank_state(dcp) for _ in range(dcp)]

    def ranks():
        for r in range(dcp):
            step(states[r], dcp, r, outs[r], lses[r])
        silkern.merge_partials(outs, lses, out, lse)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ranks()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ranks()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    cache, _, slots, _ = alone
    want, want_lse, spread, near = oracle.attend_selected(q, slots, *cache, softmax_scale=scale)
    assert_attention(whole, whole_lse, (want, want_lse, spread, near), q, cache[0], cache[2], scale)
    # A rank's pages hold other tokens, so scales differ, and with them only codes that are subnormal in
    # one of the two (below 2**-6 of a code range that starts at 224): 2**-10 of a scale of at most 2**-5,
    # on both keys and values. Each partial output adds a rounding of its own.
    loose = 2.0**-10 * 2.0**-5 * (1 + float(q.double().abs().sum(-1).max()) * scale * 4)
    assert float(((out.double() - want).abs() - 3 * 2.0**-8 * spread).max()) <= loose
    assert float((lse.double() - want_lse).abs().max()) <= loose


# --------------------------------------------------------------------------------------- refusals, far places

def good_calls():
    """name -> (launcher, positional buffers by name, keywords) of calls that are right."""
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v, ks, vs = make_cache(4, 16, 2, 64, seed=50)
    q, out, lse = randn(3, 4, 64, dtype=torch.bfloat16, seed=51), *results(3, 4, 64, torch.bfloat16)
    cache = dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)
    table = ints(0, 1, 2, 3).view(2, 2)
    sequence = dict(cu_tokens=ints(0, 2, 3), lengths=ints(5, 9), req_ids=ints(0, 1), block_table=table)
    new = randn(3, 2, 64, dtype=torch.bfloat16, seed=52)
    return {
        "selected": (silkern.attend_selected, dict(q=q, slots=table.repeat(2, 1)[:3], **cache, out=out, lse=lse),
                     dict(softmax_scale=0.1)),
        "window": (silkern.attend_window, dict(q=q, **sequence, **cache, out=out, lse=lse), dict(softmax_scale=0.1)),
        "append": (silkern.append_quantized, dict(keys=new, values=new.clone(), **cache, cu_tokens=ints(0, 2, 3),
                                                  starts=ints(0, 4), req_ids=ints(0, 1), block_table=table), {}),
        "merge": (silkern.merge_partials, dict(outs=randn(2, 3, 4, 64, dtype=torch.bfloat16, seed=53),
                                               lses=torch.zeros((2, 3, 4), device="cuda"), out=out, lse=lse), {}),
    }


REFUSED = [
    ("selected window", "q", lambda t: t.float(), "bfloat16 or float16"),
    ("selected window", "q", lambda t: t[:, :3], "multiple of the cache's heads"),
    ("selected window", "q", lambda t: t[..., :32], "key_dim"),
    ("selected window", "q", lambda t: t[:0], "at least one row"),
    ("selected window", "q", lambda t: torch.cat([t, t], -1).view(3, 4, 64, 2)[..., 0], "unit column stride"),
    ("selected window", "q", lambda t: torch.cat([t, t], -1)[..., 1:65], "16-byte alignment"),
    ("selected window", "out", lambda t: t.half(), "of q's type"),
    ("selected window", "out", lambda t: t[:2], "out must be"),
    ("selected window", "lse", lambda t: t.double(), "float32"),
    ("selected window", "lse", lambda t: t.t().contiguous().t(), "contiguous"),
    ("selected window append", "k_cache", lambda t: t.view(torch.uint8), "float8_e4m3fn"),
    ("selected window append", "k_cache", lambda t: t[0], "num_blocks, block_size"),
    ("selected window append", "v_cache", lambda t: t[:2], "the same shape"),
    ("selected window append", "v_cache", lambda t: None, "both given or both None"),
    ("selected window append", "k_scale", lambda t: t.half(), "scales must be"),
    ("selected window append", "v_scale", lambda t: t.t().contiguous().t(), "scales must be"),
    ("selected", "slots", lambda t: t.long(), "slots must be int32"),
    ("selected", "slots", lambda t: t[:2], "slots must be int32"),
    ("selected", "slots", lambda t: t.t().contiguous().t(), "unit column stride"),
    ("window append", "cu_tokens", lambda t: t[:2], "cu_tokens one more"),
    ("window append", "req_ids", lambda t: t.long(), "contiguous int32"),
    ("window append", "block_table", lambda t: t[0], "2D"),
    ("window", "lengths", lambda t: t[:1], "one element per sequence"),
    ("append", "keys", lambda t: t[:, :1], "must be (tokens"),
    ("append", "values", lambda t: t.half(), "of one type"),
    ("append", "values", lambda t: None, "exactly when"),
    ("merge", "outs", lambda t: t[0], "ranks, rows, heads, dim"),
    ("merge", "lses", lambda t: t.half(), "lses must be"),
    ("merge", "out", lambda t: t.half(), "type of outs"),
    ("merge", "lse", lambda t: t[:2], "lse must be"),
    ("selected window append merge", "any", lambda t: t.cpu(), "CUDA tensors"),
]


@pytest.mark.parametrize("names,buffer,change,message", REFUSED, ids=[f"{r[1]}-{r[3][:12]}" for r in REFUSED])
def test_launchers_refuse(names, buffer, change, message) -> None:
    for name in names.split():
        call, buffers, kw = good_calls()[name]
        call(*buffers.values(), **kw)
        for which in list(buffers) if buffer == "any" else [buffer]:
            wrong = dict(buffers)
            wrong[which] = change(wrong[which])
            with pytest.raises(silkern.LocalizationError) as caught:
                call(*wrong.values(), **kw)
            assert message in str(caught.value), (name, which, str(caught.value))


@pytest.mark.parametrize("names,kw,message", [
    ("selected window", dict(softmax_scale=math.inf), "finite"), ("window", dict(window=-1), "window and sinks"),
    ("window", dict(sinks=2.0), "window and sinks"), ("window append", dict(dcp_size=0), "dcp"),
    ("window append", dict(dcp_rank=True), "integers"), ("window append", dict(dcp_interleave=3), "divisible"),
    ("selected window append", dict(status=torch.zeros(1)), "status"), ("selected", dict(counts=torch.zeros(2, dtype=torch.int32)), ""),
])
def test_launchers_refuse_numbers(names, kw, message) -> None:
    for name in names.split():
        call, buffers, more = good_calls()[name]
        with pytest.raises(silkern.LocalizationError) as caught:
            call(*buffers.values(), **{**more, **kw})
        assert message in str(caught.value)


def test_results_must_not_lie_in_inputs() -> None:
    call, b, kw = good_calls()["selected"]
    for which, other in (("out", b["q"]), ("lse", b["k_scale"].flatten().repeat(2)[:12].view(3, 4))):
        with pytest.raises(silkern.LocalizationError, match="overlaps"):
            wrong = {**b, which: other}
            if which == "lse":
                wrong["k_scale"] = other.view(-1)[:8].view(4, 2)
            call(*wrong.values(), **kw)


@pytest.mark.parametrize("shape", ["d128", "latent"])
def test_places_past_32_bits(shape) -> None:
    """Slots whose bytes lie more than 4 GB into the cache, and append to them."""
    dim, value_dim, latent = SHAPES[shape]
    heads = 1 if latent else 2
    blocks = 70_000 if latent else 300_000  # 5.2 and 2 x 4.9 GB
    block_size = 128 if latent else 64
    small = make_cache(6, block_size, heads, dim, latent=latent, seed=60)
    cache = [None if t is None else torch.zeros((blocks, *t.shape[1:]), dtype=t.dtype, device="cuda") for t in small]
    places = torch.tensor([0, blocks // 3, blocks // 2, blocks - 3, blocks - 2, blocks - 1]).cuda()
    for t, s in zip(cache, small):
        if t is not None:
            t.view(torch.uint8)[places] = s.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else s.view(torch.uint8)
    assert cache[0].numel() > 2**32
    g = torch.Generator().manual_seed(61)
    local = torch.randint(0, 6 * block_size, (3, 500), generator=g).cuda()
    slots = (places[local // block_size] * block_size + local % block_size).to(torch.int32)
    q = randn(3, 8, dim, dtype=torch.bfloat16, seed=62)
    out, lse = selected(q, slots, cache, value_dim, softmax_scale=dim**-0.5)
    near, near_lse = selected(q, local.to(torch.int32), small, value_dim, softmax_scale=dim**-0.5)
    assert torch.equal(out, near) and torch.equal(lse, near_lse)
    x = torch.randn((200, heads, dim), generator=g).to(torch.bfloat16).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (x, None if latent else x), (ints(0, 200), ints(0), ints(0))
    silkern.append_quantized(*args[0], *cache, *args[1], places[2:].to(torch.int32)[None])
    silkern.append_quantized(*args[0], *small, *args[1], ints(2, 3, 4, 5)[None])
    torch.cuda.synchronize()
    same_cache([None if t is None else t[places] for t in cache], small)


def test_grids_that_follow_one_another_see_what_was_written() -> None:
    """Append, localize, attend and merge back to back, on fresh values each
    time: each kernel starts before the one ahead ends, and reads its results."""
    g = torch.Generator().manual_seed(70)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = [t.clone() for t in make_cache(64, 16, 1, 128, seed=71)]
    table = torch.randperm(64, generator=g).to(torch.int32).view(2, 32).cuda()
    req, cu, starts = ints([0, 1]), ints([0, 400, 800]), ints([0, 0])
    q = randn(2, 16, 128, dtype=torch.bfloat16, seed=72)
    got = []
    for step in range(12):
        x = torch.randn((800, 1, 128), generator=g).to(torch.bfloat16).cuda()
        tokens = torch.stack([torch.randperm(400, generator=g)[:300] for _ in range(2)]).to(torch.int32).cuda()
        slots, counts = torch.empty_like(tokens), torch.empty(2, dtype=torch.int32, device="cuda")
        out, lse = results(2, 16, 128, torch.bfloat16)
        whole, whole_lse = results(2, 16, 128, torch.bfloat16)
        torch.cuda.synchronize()
        silkern.append_quantized(x, x, *cache, cu, starts, req, table)
        silkern.localize_rowwise(req, table, tokens, slots, counts, block_size=16, dcp_size=1, dcp_rank=0)
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=0.09)
        silkern.merge_partials(out[None], lse[None], whole, whole_lse)
        torch.cuda.synchronize()
        want = oracle.attend_selected(q, slots, *cache, softmax_scale=0.09)
        assert_attention(out, lse, want, q, cache[0], cache[2], 0.09)
        assert torch.equal(whole, out)
        got.append(out)
    assert not torch.equal(got[0], got[1])


@pytest.mark.parametrize("rows,heads", [(16, 16), (19, 16), (37, 16), (75, 16), (150, 16), (310, 16), (444, 64), (520, 64)])
@pytest.mark.parametrize("shape", ["d64", "latent"])
def test_batches_around_the_splitting_rules(shape, rows, heads) -> None:
    """Batches on both sides of where clusters, a CTA's pipelines and leftover
    items split the keys, with rows of every length among them."""
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(40, 64, 1, dim, latent=latent, seed=80)
    g = torch.Generator().manual_seed(rows)
    slots = torch.randint(0, 2560, (rows, 600), generator=g, dtype=torch.int32)
    counts = torch.randint(0, 601, (rows,), generator=g, dtype=torch.int32)
    counts[-5:] = torch.tensor([0, 600, 1, 128, 129])
    slots, counts = slots.cuda(), counts.cuda()
    q = randn(rows, heads, dim, dtype=torch.bfloat16, seed=81)
    out, lse = selected(q, slots, cache, value_dim, softmax_scale=dim**-0.5, counts=counts)
    want = oracle.attend_selected(q, slots, *cache, softmax_scale=dim**-0.5, counts=counts)
    assert_attention(out, lse, want, q, cache[0], cache[2], dim**-0.5)


def test_odd_queries() -> None:
    """Zero, tiny, huge and unlike heads of one CTA; a NaN or infinity in one
    head's query makes that head NaN and no other."""
    cache = make_cache(4, 64, 1, 128, seed=90)
    slots = torch.arange(200, dtype=torch.int32).view(1, 200).cuda()
    for dtype in TYPES:
        q = randn(1, 12, 128, dtype=dtype, seed=91)
        q[0, 1] = 0
        q[0, 2] *= 2.0**-20 if dtype == torch.float16 else 2.0**-60
        q[0, 3] *= 300.0
        q[0, 4, 5:] = 0
        q[0, 5] = 0
        q[0, 5, 7] = 2.0**-14
        out, lse = selected(q, slots, cache, 128, softmax_scale=0.09)
        want = oracle.attend_selected(q, slots, *cache, softmax_scale=0.09)
        for h in range(12):  # a bound of its own for each head
            assert_attention(out[:, h : h + 1], lse[:, h : h + 1].contiguous(), tuple(t[:, h : h + 1] for t in want),
                             q[:, h : h + 1], cache[0], cache[2], 0.09)
        q[0, 6, 9], q[0, 7, 3] = math.nan, math.inf
        after, after_lse = selected(q, slots, cache, 128, softmax_scale=0.09)
        odd = torch.zeros(12, dtype=torch.bool, device="cuda")
        odd[6:8] = True
        assert bool(after[0, odd].isnan().all()) and bool(after_lse[0, odd].isnan().all())
        assert torch.equal(after[0, ~odd], out[0, ~odd]) and torch.equal(after_lse[0, ~odd], lse[0, ~odd])


@pytest.mark.parametrize("latent", [False, True])
def test_compiled_step_in_a_graph_is_the_eager_step(latent) -> None:
    """append, both attentions and merge under torch.compile, captured and
    replayed: bit for bit what the launchers give when called one by one."""
    from silkern_b200 import ops

    ops.register()
    dim, value_dim, heads = (576, 512, 32) if latent else (128, 128, 16)
    kv_heads = 1 if latent else 4
    cache = [t if t is None else t.clone() for t in make_cache(12, 16, kv_heads, dim, latent=latent, seed=50)]
    other = [t if t is None else t.clone() for t in cache]
    table = torch.randperm(12, generator=torch.Generator().manual_seed(51)).to(torch.int32).view(3, 4).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    cu, starts, lengths, req = ints(0, 1, 2, 3), ints(20, 0, 47), ints(21, 1, 48), ints(1, 0, 2)
    slots = torch.randint(-1, 192, (3, 70), dtype=torch.int32, generator=torch.Generator().manual_seed(52)).cuda()
    q = randn(3, heads, dim, dtype=torch.bfloat16, seed=53)
    new = randn(3, kv_heads, dim, dtype=torch.bfloat16, seed=54)

    def step(cache, outs, lses, out, lse):
        silkern.append_quantized(new, None if latent else new, *cache, cu, starts, req, table)
        silkern.attend_selected(q, slots, *cache, outs[0], lses[0], softmax_scale=0.05)
        silkern.attend_window(q, cu, lengths, req, table, *cache, outs[1], lses[1], softmax_scale=0.05, window=30, sinks=2)
        silkern.merge_partials(outs, lses, out, lse)

    def buffers():
        return (torch.zeros((2, 3, heads, value_dim), dtype=torch.bfloat16, device="cuda"),
                torch.zeros((2, 3, heads), device="cuda"), *results(3, heads, value_dim, torch.bfloat16))

    want = buffers()
    step(cache, *want)
    torch.cuda.synchronize()
    got = buffers()
    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            compiled(other, *got)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        compiled(other, *got)
    for t in got:
        t.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    same_cache(other, cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads", [5, 30, 64])
@pytest.mark.parametrize("rows", [1, 2, 8, 11, 15, 21, 26, 33, 44])
def test_items_shared_by_clusters_of_any_size(shape, dtype, heads, rows) -> None:
    """As many rows as clusters of 16, 10, 9, 6, 5, 4 and 3 have room for, or a
    row more or less: ranks that are no power of two, more ranks than columns."""
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(90, 64, 1, dim, latent=latent, seed=rows)
    slots = torch.randint(-1, 90 * 64, (rows, 4229), dtype=torch.int32, generator=torch.Generator().manual_seed(rows)).cuda()
    q = randn(rows, heads, dim, dtype=dtype, seed=heads)
    out, lse = selected(q, slots, cache, value_dim, softmax_scale=dim**-0.5)
    want = oracle.attend_selected(q, slots, *cache, softmax_scale=dim**-0.5)
    assert_attention(out, lse, want, q, cache[0], cache[2], dim**-0.5)


# -------------------------------------------------------------------------------- buffers that lie between one another

@pytest.mark.parametrize("shape", SHAPES)
def test_results_between_the_rows_and_heads_of_the_queries(shape) -> None:
    """q and out as column slices of one buffer, by rows and by heads: no byte is both."""
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(9, 32, 1, dim, latent=latent, seed=100)
    slots = torch.randint(-1, 288, (5, 150), generator=torch.Generator().manual_seed(101), dtype=torch.int32).cuda()
    whole = randn(5, 4, dim, dtype=torch.bfloat16, seed=102)
    want = selected(whole, slots, cache, value_dim, softmax_scale=0.07)
    rows = torch.zeros((5, 4 * dim + 4 * value_dim + 8), dtype=torch.bfloat16, device="cuda")
    heads = torch.zeros((5, 4, dim + value_dim + 16), dtype=torch.bfloat16, device="cuda")
    for q, out in ((rows[:, : 4 * dim].unflatten(1, (4, dim)), rows[:, 4 * dim : -8].unflatten(1, (4, value_dim))),
                   (heads[..., :dim], heads[..., dim : dim + value_dim])):
        q.copy_(whole)
        lse = torch.empty((5, 4), device="cuda")
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=0.07)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(q, whole)
        with pytest.raises(silkern.LocalizationError, match="overlaps"):
            silkern.attend_selected(q, slots, *cache, q[..., :value_dim], lse, softmax_scale=0.07)


def test_merge_between_its_partial_results() -> None:
    """One buffer of (rows, ranks + 1, heads, dim) holds the partial outputs and their join."""
    outs = randn(3, 6, 4, 64, dtype=torch.float16, seed=103)
    lses = torch.randn((3, 6, 4), generator=torch.Generator().manual_seed(104)).cuda()
    want, want_lse = results(6, 4, 64, torch.float16)
    silkern.merge_partials(outs, lses, want, want_lse)
    held = torch.zeros((6, 4, 4, 64), dtype=torch.float16, device="cuda")
    held[:, :3] = outs.transpose(0, 1)
    silkern.merge_partials(held[:, :3].transpose(0, 1), lses, held[:, 3], want_lse)
    assert torch.equal(held[:, 3], want) and torch.equal(held[:, :3].transpose(0, 1), outs)
    with pytest.raises(silkern.LocalizationError, match="overlaps"):
        silkern.merge_partials(held[:, :3].transpose(0, 1), lses, held[:, 2], want_lse)


# ---------------------------------------------------------------------------------------- keys and values laid out apart

LAYOUTS = ["unlike", "heads_first_values", "pages", "rows", "heads", "spread_pages"]


def cache_in_layout(layout, blocks, block_size, kv_heads, dim, seed):
    """The same cache, as two contiguous tensors and in a layout of K and V that is given by name."""
    plain = make_cache(blocks, block_size, kv_heads, dim, seed=seed)
    byte = dict(dtype=torch.uint8, device="cuda")
    if layout == "unlike":  # keys token by token with room between, values head by head
        k = torch.full((blocks, block_size, kv_heads + 1, dim + 16), 0x7F, **byte)[:, :, 1:, 16:]
        v = torch.full((blocks, kv_heads, block_size, dim), 0x7F, **byte).permute(0, 2, 1, 3)
    elif layout == "heads_first_values":  # pages of values among one another
        k = torch.full((blocks, block_size, kv_heads, dim), 0x7F, **byte)
        v = torch.full((block_size, kv_heads, blocks, dim), 0x7F, **byte).permute(2, 0, 1, 3)
    elif layout == "pages":
        k, v = torch.full((blocks, 2, block_size, kv_heads, dim), 0x7F, **byte).unbind(1)
    elif layout == "rows":
        k, v = torch.full((blocks, block_size, 2, kv_heads, dim), 0x7F, **byte).unbind(2)
    elif layout == "heads":
        k, v = torch.full((blocks, block_size, kv_heads, 2, dim), 0x7F, **byte).unbind(3)
    else:  # a page of keys after every third page
        k = torch.full((3 * blocks, block_size, kv_heads, dim), 0x7F, **byte)[2::3]
        v = torch.full((blocks, block_size, kv_heads, dim), 0x7F, **byte)
    for view, codes in ((k, plain[0]), (v, plain[1])):
        view.copy_(codes.view(torch.uint8))
    return plain, (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), plain[2].clone(), plain[3].clone())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("kv_heads,dim", [(3, 64), (2, 128), (1, 128)])
def test_keys_and_values_in_layouts_of_their_own(kv_heads, dim, layout, dtype) -> None:
    """Attention and append see places, not layouts: bit for bit what two
    contiguous tensors give, which is held against 64 bits."""
    plain, apart = cache_in_layout(layout, 24, 16, kv_heads, dim, seed=110)
    g = torch.Generator().manual_seed(111)
    heads = 4 * kv_heads
    slots = torch.randint(-1, 24 * 16, (90, 500), generator=g, dtype=torch.int32).cuda()
    table = torch.randperm(24, generator=g).to(torch.int32).view(2, 12).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(90, heads, dim, dtype=dtype, seed=112)
    place = (ints(0, 50, 90), ints(192, 150), ints(1, 0), table)
    for rows in (1, 90):
        got = selected(q[:rows], slots[:rows], apart, dim, softmax_scale=0.1)
        want = selected(q[:rows], slots[:rows], plain, dim, softmax_scale=0.1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert_attention(*want, oracle.attend_selected(q[:rows], slots[:rows], *plain, softmax_scale=0.1), q[:rows], plain[0],
                         plain[2], 0.1)
    got, want = results(90, heads, dim, dtype), results(90, heads, dim, dtype)
    silkern.attend_window(q, *place, *apart, *got, softmax_scale=0.1, window=60, sinks=3)
    silkern.attend_window(q, *place, *plain, *want, softmax_scale=0.1, window=60, sinks=3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    new = [torch.randn((90, kv_heads, dim), generator=g).to(dtype).cuda() for _ in range(2)]
    order = (ints(0, 50, 90), ints(100, 3), ints(1, 0), table)
    same = oracle.append(*new, *plain, *order)
    silkern.append_quantized(*new, *apart, *order)
    torch.cuda.synchronize()
    same_cache(apart, same)


def test_first_calls_from_several_threads_at_once() -> None:
    """A fresh process, whose threads are the first to ask for launch
    permissions and cluster sizes, each on a stream of its own."""
    import subprocess
    import sys

    code = """
import threading, torch
import silkern_b200 as silkern
from tests.attention_cases import make_cache
torch.cuda.init()
jobs, start = [], threading.Barrier(6)
for i, (dim, heads, rows) in enumerate([(64, 8, 1), (128, 64, 1), (576, 16, 3), (64, 8, 200), (128, 8, 90), (576, 128, 40)]):
    latent = dim == 576
    cache = make_cache(40, 64, 1, dim, latent=latent, seed=i)
    q = torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda()
    slots = torch.randint(0, 2560, (rows, 2000), dtype=torch.int32, generator=torch.Generator().manual_seed(i)).cuda()
    outs = [torch.empty((rows, heads, 512 if latent else dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    jobs.append((q, slots, cache, outs, [torch.empty((rows, heads), device="cuda") for _ in range(2)]))
torch.cuda.synchronize()
errors = []
def run(q, slots, cache, outs, lses):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for _ in range(20):
                silkern.attend_selected(q, slots, *cache, outs[0], lses[0], softmax_scale=0.05)
            torch.cuda.current_stream().synchronize()
    except Exception as error:
        errors.append(error)
threads = [threading.Thread(target=run, args=job) for job in jobs]
for t in threads: t.start()
for t in threads: t.join()
assert not errors, errors
for q, slots, cache, outs, lses in jobs:
    silkern.attend_selected(q, slots, *cache, outs[1], lses[1], softmax_scale=0.05)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(lses[0], lses[1]) and bool(torch.isfinite(lses[0]).all())
print("threads agree")
"""
    proc = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and "threads agree" in proc.stdout, proc.stderr[-2000:]
