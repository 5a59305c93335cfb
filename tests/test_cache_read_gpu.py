"""Reading the 8-bit cache back, on the device."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import attention as oracle  # noqa: E402
from tests.attention_cases import HALF_STEP, make_cache  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)

TYPES = [torch.bfloat16, torch.float16]


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def assert_read(got, want):
    """A product rounded to float32 (2^-24) and to the type; fp16's smallest step is 2^-24."""
    if want is None:
        return
    u = HALF_STEP[got.dtype]
    error = (got.double() - want).abs()
    assert bool((error <= u * want.abs() * (1 + 2.0**-10) + (2.0**-25 if got.dtype == torch.float16 else 1e-45)).all())


def run(cache, keys, values, cu, starts, req, table, **kw):
    want = oracle.read(keys, values, *cache, cu, starts, req, table, **kw)
    silkern.read_quantized(keys, values, *cache, cu, starts, req, table, **kw)
    assert_read(keys, want[0])
    if values is not None:
        assert_read(values, want[1])


def buffers(tokens, heads, dim, latent, dtype):
    keys = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device="cuda")
    return keys, None if latent else torch.full_like(keys, -7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,latent", [(64, 1, False), (64, 3, False), (128, 8, False), (128, 5, False), (576, 1, True)])
@pytest.mark.parametrize("block", [1, 16, 17, 48, 64])
@pytest.mark.parametrize("dcp,il", [(1, 1), (2, 1), (3, 4), (8, 16)])
def test_layouts_pages_and_ranks(dtype, dim, heads, latent, block, dcp, il) -> None:
    if block % il:
        pytest.skip("a page holds whole runs")
    width = -(-400 // (block * dcp)) + 1
    cache = make_cache(3 * width, block, heads, dim, latent=latent, seed=block)
    table = torch.randperm(3 * width, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(3, width).cuda()
    lengths = [0, 1, 130, 0, 33, 200, 31, 32]
    cu = ints(*[sum(lengths[:i]) for i in range(len(lengths) + 1)])
    starts, req = ints(5, 399, 7, 0, 0, 190, 64, 100), ints(0, 1, 2, 0, 1, 0, 2, 1)
    for rank in {0, dcp - 1}:
        keys, values = buffers(sum(lengths) + 9, heads, dim, latent, dtype)
        run(cache, keys, values, cu, starts, req, table, dcp_size=dcp, dcp_rank=rank, dcp_interleave=il)
        assert bool((keys[-9:] == 7).all()) and (latent or bool((values[-9:] == -7).all()))


def test_many_sequences_of_one_token_and_long_ones() -> None:
    cache = make_cache(600, 16, 2, 128, seed=1)
    table = torch.randperm(600, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(4, 150).cuda()
    n = 1500
    g = torch.Generator().manual_seed(2)
    keys, values = buffers(n, 2, 128, False, torch.bfloat16)
    run(cache, keys, values, torch.arange(n + 1, dtype=torch.int32).cuda(), torch.randint(0, 2400, (n,), generator=g).to(torch.int32).cuda(),
        torch.randint(0, 4, (n,), generator=g).to(torch.int32).cuda(), table)
    keys, values = buffers(9600, 2, 128, False, torch.float16)
    run(cache, keys, values, ints(0, 2400, 4800, 7200, 9600), ints(0, 0, 0, 0), ints(3, 1, 0, 2), table)


def test_strides_and_unaligned_outputs() -> None:
    cache = make_cache(12, 16, 4, 64, seed=3, layout="htd")
    table = torch.arange(12, dtype=torch.int32).view(2, 6).cuda()
    store = torch.full((70, 2, 4, 67), 7.0, dtype=torch.bfloat16, device="cuda")
    keys, values = store[:, 0, :, 1:65], store[:, 1, :, 3:]
    run(cache, keys, values, ints(0, 40, 70), ints(3, 50), ints(1, 0), table)
    assert bool((store[:, 0, :, 0] == 7).all()) and bool((store[:, 0, :, 65:] == 7).all()) and bool((store[:, 1, :, :3] == 7).all())
    wide = torch.full((4, 75, 72), 7.0, dtype=torch.float16, device="cuda")
    run(cache, wide[:, 5:, 8:].transpose(0, 1), wide.clone()[:, 5:, 8:].transpose(0, 1), ints(0, 40, 70), ints(3, 50), ints(1, 0), table)
    assert bool((wide[:, :5] == 7).all()) and bool((wide[..., :8] == 7).all())


def test_bad_requests_lengths_and_pages_leave_rows_and_are_flagged() -> None:
    cache = make_cache(6, 16, 2, 64, seed=4)
    table = ints(0, 1, 2, 3, 4, 5).view(2, 3)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(starts, req, tab=table):
        keys, values = buffers(40, 2, 64, False, torch.bfloat16)
        status.zero_()
        want = oracle.read(keys, values, *cache, ints(0, 20, 40), starts, req, tab)
        silkern.read_quantized(keys, values, *cache, ints(0, 20, 40), starts, req, tab, status=status)
        assert_read(keys, want[0]), assert_read(values, want[1])
        return int(status)

    assert call(ints(0, 5), ints(0, 1)) == 0
    assert call(ints(0, 5), ints(0, 2)) == 1
    assert call(ints(0, 5), ints(-1, 1)) == 1
    assert call(ints(-1, 5), ints(0, 1)) == 2
    assert call(ints(0, 40), ints(0, 1)) == 8  # past the table row
    assert call(ints(0, 5), ints(0, 1), ints(0, 6, 2, 3, -1, 5).view(2, 3)) == 8
    keys, values = buffers(40, 2, 64, False, torch.bfloat16)
    status.zero_()
    silkern.read_quantized(keys, values, *cache, ints(0, 20, 40), ints(0, 2**31 - 10), ints(0, 1), table, status=status)
    assert int(status) == 2 and bool((keys[20:] == 7).all())


def test_scales_of_every_size_and_codes_that_are_not_numbers() -> None:
    k, v, ks, vs = make_cache(4, 16, 1, 64, seed=5)
    ks.copy_(torch.tensor([2.0**-100, 2.0**100, 0.0, math.nan]).view(4, 1))
    v.view(torch.uint8)[0, 3, 0, 7] = 0x7F
    keys, values = buffers(64, 1, 64, False, torch.bfloat16)
    silkern.read_quantized(keys, values, k, v, ks, vs, ints(0, 64), ints(0), ints(0), ints(0, 1, 2, 3).view(1, 4))
    want = oracle.read(*buffers(64, 1, 64, False, torch.bfloat16), k, v, ks, vs, ints(0, 64), ints(0), ints(0), ints(0, 1, 2, 3).view(1, 4))
    assert_read(keys[:48], want[0][:48])
    assert bool(keys[48:].isnan().all()) and bool((keys[32:48] == 0).all())
    assert bool(values[3, 0, 7].isnan()) and int(values.isnan().sum()) == 1


def test_what_append_stored_comes_back_exactly_where_codes_hold_it() -> None:
    """Numbers of 4 bits over powers of two, appended and read on two ranks: the same numbers."""
    g = torch.Generator().manual_seed(6)
    x = (torch.randint(8, 16, (100, 2, 128), generator=g) * torch.tensor([-1.0, 1.0])[torch.randint(0, 2, (100, 2, 128), generator=g)])
    keys = x.to(torch.bfloat16).cuda()
    values = (x.flip(0) / 64).to(torch.bfloat16).cuda()
    got_k, got_v = torch.zeros_like(keys), torch.zeros_like(values)
    table = ints(3, 0, 2, 1).view(1, 4)
    for rank in (0, 1):
        cache = [torch.zeros((4, 16, 2, 128), dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
        scales = [torch.zeros((4, 2), device="cuda") for _ in range(2)]
        own = dict(dcp_size=2, dcp_rank=rank, dcp_interleave=8)
        silkern.append_quantized(keys, values, *cache, *scales, ints(0, 100), ints(0), ints(0), table, **own)
        silkern.read_quantized(got_k, got_v, *cache, *scales, ints(0, 100), ints(0), ints(0), table, **own)
    assert torch.equal(got_k, keys) and torch.equal(got_v, values)


def test_graphs_and_compiled_callers() -> None:
    cache = make_cache(8, 16, 2, 64, seed=7)
    table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
    cu, starts, req = ints(0, 40, 70), ints(3, 20), ints(1, 0)
    want, got = buffers(70, 2, 64, False, torch.bfloat16), buffers(70, 2, 64, False, torch.bfloat16)
    silkern.read_quantized(*want, *cache, cu, starts, req, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        silkern.read_quantized(*got, *cache, cu, starts, req, table)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    @torch.compile(fullgraph=True)
    def step(keys, values):
        silkern.read_quantized(keys, values, *cache, cu, starts, req, table)

    got = buffers(70, 2, 64, False, torch.bfloat16)
    step(*got)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
