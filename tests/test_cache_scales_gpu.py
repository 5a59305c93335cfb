"""Scales of every size that the 8-bit cache may hold, on the device, against 64-bit arithmetic.

The softmax's sum does not know the values' scales, and the weights that meet
the values do: pages of zero values, of very small and very large ones, and of
both beside each other, with scores that rise and fall from tile to tile.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import attention as oracle  # noqa: E402
from tests.attention_cases import HALF_STEP, score_error  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)

PAGE = 128  # a tile of the kernel, so that a tile's values have one scale


def stepped_cache(dim, kv_heads, heights, scales, seed):
    """One page for each entry of ``heights``: keys whose column 0 is that many
    nats (for a query with 1 there), and values of the page's scale."""
    g = torch.Generator().manual_seed(seed)
    shape = (len(heights), PAGE, kv_heads, dim)
    k = (torch.randn(shape, generator=g) * 0.5).clamp(-2, 2)
    k[..., 0] = torch.tensor(heights, dtype=torch.float32)[:, None, None]
    v = (torch.randn(shape, generator=g) * 64).clamp(-448, 448)
    vs = torch.tensor(scales, dtype=torch.float32)[:, None].repeat(1, kv_heads)
    return (k.to(torch.float8_e4m3fn).cuda(), v.to(torch.float8_e4m3fn).cuda(), torch.ones_like(vs).cuda(), vs.cuda())


def queries(rows, heads, dim, dtype, seed):
    q = torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(seed)) * 0.3
    q[..., 0] = 1.0
    return q.to(dtype).cuda()


def assert_near(out, lse, want, q, cache, pages):
    """The bounds of ``assert_attention``, with what far scales add: u = log2(p)
    + log2(vscale) is below 256 in size, so that its rounding and that of log2(p)
    taken back out of it are 2**-17 each, three of them 2**-15 nats; and each page
    may move the references once, a factor that is 2**-22 off."""
    ref, ref_lse, spread, near = want
    ds = score_error(q, cache[0], cache[2], 1.0) + 2.0**-15 + pages * 2.0**-22
    assert bool(torch.isfinite(lse).all())
    assert float(((lse.double() - ref_lse).abs() - 2.0**-22 * ref_lse.abs()).max()) <= ds + 2.0**-20
    u = HALF_STEP[out.dtype]
    relative, floor = {torch.bfloat16: (2.0**-8 + 2.0**-11, 2.0**-15), torch.float16: (2.0**-12, 2.0**-18)}[out.dtype]
    subnormal = 2.0**-25 if out.dtype == torch.float16 else 1e-38
    bound = u * ref.abs() + (relative + 2 * ds) * spread + floor * near + subnormal
    fits = ref.abs() < torch.finfo(out.dtype).max / 2  # a float16 output may be past its type
    bad = ~((out.double() - ref).abs() <= bound) & fits
    assert not bool(bad.any()), f"{int(bad.sum())} outputs off"


FALLING, RISING = (44, 0, 30, 0, 20, 0), (0, 20, 0, 30, 0, 44)
FAR = 2.0**100
PATTERNS = {
    "zero": (0.0,), "floor": (1 / FAR,), "small": (2.0**-70,), "ceiling": (FAR,),
    "far_apart": (FAR, 1 / FAR), "far_apart_reversed": (1 / FAR, FAR), "apart_131": (2.0**40, 2.0**-95),
    "zero_beside_usual": (0.0, 2.0**-6, 0.0), "zero_beside_large": (2.0**40, 0.0), "zero_beside_floor": (1 / FAR, 0.0, 1 / FAR),
    "usual": (2.0**-6, 2.0**-24, 2.0**24),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heights", [FALLING, RISING, (0, 0, 0)], ids=["falling", "rising", "level"])
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("dim,rows,pages", [(64, 90, 6), (128, 90, 6), (128, 1, 70), (64, 3, 140)])
def test_sums_do_not_depend_on_the_values_scales(dim, rows, pages, pattern, heights, dtype) -> None:
    """Whole items (90 rows) and items shared by a cluster's ranks (1 and 3),
    and the joining with a rank whose values are usual ones."""
    scales = PATTERNS[pattern]
    cache = stepped_cache(dim, 2, [heights[i % len(heights)] for i in range(pages)],
                          [scales[i % len(scales)] for i in range(pages)], seed=dim + pages)
    q = queries(rows, 4, dim, dtype, seed=rows)
    slots = torch.arange(pages * PAGE, dtype=torch.int32).repeat(rows, 1).cuda()
    outs = torch.empty((2, rows, 4, dim), dtype=dtype, device="cuda")
    lses = torch.empty((2, rows, 4), device="cuda")
    silkern.attend_selected(q, slots, *cache, outs[0], lses[0], softmax_scale=1.0)
    want = oracle.attend_selected(q[:3], slots[:3], *cache, softmax_scale=1.0)
    assert_near(outs[0, :3], lses[0, :3], want, q, cache, pages)
    assert bool(torch.isfinite(lses[0]).all())
    usual = (*cache[:3], torch.full_like(cache[3], 2.0**-6))
    silkern.attend_selected(q, slots, *usual, outs[1], lses[1], softmax_scale=1.0)
    if dtype == torch.float16 and max(scales) > 1:
        return
    out, lse = torch.empty_like(outs[0]), torch.empty_like(lses[0])
    silkern.merge_partials(outs, lses, out, lse)
    joined, joined_lse, spread = oracle.merge(outs, lses)
    assert bool(((lse.double() - joined_lse).abs() <= 2.0**-20 + 2.0**-22 * joined_lse.abs()).all())
    assert bool(((out.double() - joined).abs() <= HALF_STEP[dtype] * joined.abs() + 2.0**-16 * spread + 2.0**-24).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4)])
@pytest.mark.parametrize("scale", [0.0, 2.0**-70, 2.0**-100])
@pytest.mark.parametrize("heights", [FALLING, RISING], ids=["falling", "rising"])
def test_pieces_of_prompts_over_zero_and_small_values(heights, scale, window, sinks, dtype) -> None:
    """Queries that share a CTA's keys see different ones of them."""
    cache = stepped_cache(64, 2, list(heights), [scale] * 6, seed=5)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    q = queries(67, 8, 64, dtype, seed=6)
    out, lse = torch.empty_like(q), torch.empty((67, 8), device="cuda")
    call = dict(softmax_scale=1.0, window=window, sinks=sinks)
    place = (ints(0, 40, 67), ints(700, 333), ints(1, 0), ints(*range(6), *range(6)).view(2, 6))
    silkern.attend_window(q, *place, *cache, out, lse, **call)
    assert_near(out, lse, oracle.attend_window(q, *place, *cache, **call), q, cache, 7)


def test_values_that_do_not_count_may_score_highest() -> None:
    """A sink over zeroed values: the usual page's outputs keep their own precision."""
    for dtype in (torch.bfloat16, torch.float16):
        cache = stepped_cache(128, 1, [20, 0, 0], [0.0, 2.0**-6, 2.0**-6], seed=8)
        q = queries(2, 8, 128, dtype, seed=9)
        slots = torch.arange(3 * PAGE, dtype=torch.int32).repeat(2, 1).cuda()
        out, lse = torch.empty_like(q), torch.empty((2, 8), device="cuda")
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=1.0)
        assert_near(out, lse, oracle.attend_selected(q, slots, *cache, softmax_scale=1.0), q, cache, 3)


def test_a_scale_that_is_not_a_number_beside_far_scales() -> None:
    """NaN reaches the heads and queries that see its page, and no other."""
    cache = stepped_cache(64, 2, [0, 30, 0, 44, 0], [1 / FAR, 0.0, 1.0, FAR, 2.0**-70], seed=10)
    cache[3][4, 1] = math.nan
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    q = queries(20, 4, 64, torch.bfloat16, seed=11)
    out, lse = torch.empty_like(q), torch.empty((20, 4), device="cuda")
    place = (ints(0, 20), ints(4 * PAGE + 10), ints(0), ints(*range(5)).view(1, 5))
    silkern.attend_window(q, *place, *cache, out, lse, softmax_scale=1.0)
    # query i is at position 502 + i: the page of position 512 on is seen from query 10 on, by heads 2 and 3
    odd = torch.zeros((20, 4), dtype=torch.bool, device="cuda")
    odd[10:, 2:] = True
    assert torch.equal(lse.isnan(), odd) and torch.equal(out.isnan().all(-1), odd) and torch.equal(out.isnan().any(-1), odd)
    want = oracle.attend_window(q, *place, *cache, softmax_scale=1.0)
    ds = score_error(q, cache[0], cache[2], 1.0) + 2.0**-14
    assert float(((lse.double() - want[1]).abs() - 2.0**-22 * want[1].abs())[~odd].max()) <= ds


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("rows,pages", [(80, 5), (1, 50)])
@pytest.mark.parametrize("scales", [(0.0,), (0.0, 2.0**-6), (2.0**-6, 0.0), (2.0**-70, 0.0, 2.0**-6), (2.0**-100, 2.0**-70)])
def test_latent_pages_of_zeros_and_small_keys(scales, rows, pages, heads, dtype) -> None:
    """A latent key's scale is its value's as well."""
    g = torch.Generator().manual_seed(12)
    k = (torch.randn((pages, PAGE, 1, 576), generator=g) * 64).clamp(-448, 448).to(torch.float8_e4m3fn).cuda()
    cache = (k, None, torch.tensor([scales[i % len(scales)] for i in range(pages)]).view(pages, 1).cuda(), None)
    q = queries(rows, heads, 576, dtype, seed=13) * 4
    slots = torch.arange(pages * PAGE, dtype=torch.int32).repeat(rows, 1).cuda()
    out, lse = torch.empty((rows, heads, 512), dtype=dtype, device="cuda"), torch.empty((rows, heads), device="cuda")
    silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=1.0)
    want = oracle.attend_selected(q[:3], slots[:3], *cache, softmax_scale=1.0)
    assert_near(out[:3], lse[:3], want, q, cache, pages)
