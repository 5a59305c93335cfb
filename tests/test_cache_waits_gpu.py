"""The bound on the waits inside the attention kernels: what a call that gives up leaves, and that
a long item alone does not make it give up."""

from __future__ import annotations

import contextlib

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from silkern_b200 import _native  # noqa: E402
from silkern_b200.attention import STATUS_WAIT_TIMEOUT  # noqa: E402
from tests.attention_cases import make_cache  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)

SHAPES = {"d64": (64, 64, False), "d128": (128, 128, False), "latent": (576, 512, True)}


@contextlib.contextmanager
def wait_bound(cycles):
    lib = _native.load()
    before = lib.silkern_attend_wait_bound_v1(cycles)
    try:
        yield
        torch.cuda.synchronize()
    finally:
        lib.silkern_attend_wait_bound_v1(before)


def test_the_bound_is_set_and_returned() -> None:
    lib = _native.load()
    before = lib.silkern_attend_wait_bound_v1(-1)
    assert before == 4_000_000_000
    assert lib.silkern_attend_wait_bound_v1(123) == before
    assert lib.silkern_attend_wait_bound_v1(2**32 + 1) == 123
    assert lib.silkern_attend_wait_bound_v1(before) == 123


def assert_right_or_nan(got, want):
    """Each (row, head) as it should be, or NaN throughout; how many are NaN."""
    out, lse = got
    odd = lse.isnan()
    assert torch.equal(out.isnan().any(-1), odd) and torch.equal(out.isnan().all(-1), odd)
    assert torch.equal(out[~odd], want[0][~odd]) and torch.equal(lse[~odd], want[1][~odd])
    return int(odd.sum())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("rows", [1, 9, 80, 200])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bound", [0, 1])
def test_a_selection_that_gives_up_leaves_nan(bound, shape, rows, heads, dtype) -> None:
    """Items of a pipeline, of a cluster and of two CTAs; the next call is right
    again. Bound 0 gives up at once; bound 1 where a wait lasts longer than the
    hardware suspends a thread, as the one for an item's end does in the middle
    of a whole item, and one for a tile, all that a cluster's ranks have, need not."""
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(64, 64, 1, dim, latent=latent, seed=1)
    g = torch.Generator().manual_seed(rows)
    slots = torch.randint(0, 4096, (rows, 20_000), generator=g, dtype=torch.int32).cuda()
    counts = torch.randint(10_000, 20_001, (rows,), generator=g, dtype=torch.int32).cuda()
    counts[rows // 2 + 1 :: 7] = 0
    q = torch.randn((rows, heads, dim), generator=g).to(dtype).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(**more):
        out = torch.full((rows, heads, value_dim), 7.0, dtype=dtype, device="cuda")
        lse = torch.full((rows, heads), 7.0, device="cuda")
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=dim**-0.5, counts=counts, **more)
        return out, lse

    want = call(status=status)
    assert status.item() == 0 and not bool(want[1].isnan().any())
    with wait_bound(bound):
        got, silent = call(status=status), call()
    odd = assert_right_or_nan(got, want)
    assert status.item() == (STATUS_WAIT_TIMEOUT if odd else 0)
    # 80 items go to 80 of a latent kernel's 148 pipelines, and else to the two pipelines of a CTA each
    if bound == 0 or rows == 200 or (latent and rows == 80):
        assert odd > 0 and assert_right_or_nan(silent, want) > 0
    again = call()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("shape", SHAPES)
def test_a_window_that_gives_up_leaves_other_rows_alone(shape) -> None:
    dim, value_dim, latent = SHAPES[shape]
    cache = make_cache(300, 64, 1, dim, latent=latent, seed=2)
    g = torch.Generator().manual_seed(3)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.randperm(300, generator=g).to(torch.int32).view(1, 300).cuda()
    place = (ints(0, 40, 41, 50), ints(19_000, 0, 9_000), ints(0, 0, 0), table)
    q = torch.randn((60, 16, dim), generator=g).to(torch.bfloat16).cuda()

    def call():
        out = torch.full((60, 16, value_dim), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((60, 16), 7.0, device="cuda")
        silkern.attend_window(q, *place, *cache, out, lse, softmax_scale=dim**-0.5)
        return out, lse

    want = call()
    with wait_bound(0):
        got = call()
    assert assert_right_or_nan(got, want) > 0
    assert bool((got[0][50:] == 7).all()) and bool((got[1][50:] == 7).all())


def test_an_item_may_last_longer_than_a_wait() -> None:
    """Half a millisecond for each tile, and items of several milliseconds: the
    wait for an item's end has its tiles' bound, not one's."""
    dim, rows = 576, 90
    cache = make_cache(512, 64, 1, dim, latent=True, seed=4)
    slots = torch.randint(0, 512 * 64, (1, 400_000), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    slots = slots.expand(rows, -1)
    q = torch.randn((rows, 16, dim), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    out, lse = torch.empty((rows, 16, 512), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, 16), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    cycles = 1_000_000
    with wait_bound(cycles):
        begin.record()
        silkern.attend_selected(q, slots, *cache, out, lse, softmax_scale=dim**-0.5, status=status)
        end.record()
    # at 2 GHz at most, an item that lasts the whole call exceeds the bound four times over
    assert begin.elapsed_time(end) * 2e6 > 4 * cycles
    assert status.item() == 0 and bool(torch.isfinite(lse).all())
