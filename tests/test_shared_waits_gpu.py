"""The waits inside the kernel of attend_shared: what a call that gives up leaves, and that a long
run of tiles alone does not make it give up; and arrays that descend."""

from __future__ import annotations

import contextlib
import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from silkern_b200 import _native  # noqa: E402
from silkern_b200.attention import STATUS_WAIT_TIMEOUT  # noqa: E402
from silkern_b200.topk import STATUS_BAD_LENGTH  # noqa: E402
from tests.attention_cases import make_cache  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)


@contextlib.contextmanager
def wait_bound(cycles):
    lib = _native.load()
    before = lib.silkern_attend_wait_bound_v1(cycles)
    try:
        yield
        torch.cuda.synchronize()
    finally:
        lib.silkern_attend_wait_bound_v1(before)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Call:
    def __init__(self, heads, kv_heads, dim, dtype, rows=40):
        g = torch.Generator().manual_seed(heads)
        self.cache = make_cache(400, 64, kv_heads, dim, seed=1)
        self.table = torch.randperm(400, generator=g).to(torch.int32).view(4, 100).cuda()
        self.cu, self.lengths, self.req = ints(1, 2, 12, 13, 37), ints(4000, 3500, 1, 6400), ints(0, 1, 2, 3)
        self.cu_groups, self.prefixes = ints(0, 2, 4), ints(3001, 1)
        self.q = torch.randn((rows, heads, dim), generator=g).to(dtype).cuda()
        self.status = ints(0)
        self.work = torch.empty(silkern.shared_workspace_bytes(rows, heads, kv_heads, dim, 4, 2), dtype=torch.uint8, device="cuda")

    def __call__(self, **more):
        rows, heads, dim = self.q.shape
        out = torch.full((rows, heads, dim), 7.0, dtype=self.q.dtype, device="cuda")
        lse = torch.full((rows, heads), 7.0, device="cuda")
        silkern.attend_shared(self.q, self.cu, self.lengths, self.req, self.cu_groups, self.prefixes, self.table, *self.cache,
                              out, lse, self.work, softmax_scale=dim**-0.5, **more)
        return out, lse


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 64, torch.bfloat16), (64, 1, 128, torch.float16), (8, 8, 128, torch.bfloat16)])
@pytest.mark.parametrize("bound", [0, 1])
def test_a_call_that_gives_up_leaves_nan(bound, heads, kv_heads, dim, dtype) -> None:
    """All of its rows are NaN, others are left alone, and the next call is right again."""
    call = Call(heads, kv_heads, dim, dtype)
    want = call(status=call.status)
    assert int(call.status) == 0 and bool(want[1].isfinite().all())
    with wait_bound(bound):
        got = call(status=call.status)
        silent = call()
    assert int(call.status) in ((STATUS_WAIT_TIMEOUT,) if bound == 0 else (0, STATUS_WAIT_TIMEOUT))
    for out, lse in (got, silent):
        gone = bool(lse[1].isnan().any())
        assert gone or bound == 1
        if gone:
            assert bool(out[1:37].isnan().all()) and bool(lse[1:37].isnan().all())
        else:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert all(bool((t[rest] == 7).all()) for t in (out, lse) for rest in (slice(0, 1), slice(37, None)))
    again = call()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_a_fragment_may_last_longer_than_a_wait() -> None:
    """A long sequence's end and more than the fragments known ahead in one CTA: its walk through
    them waits for all of the long one's tiles."""
    alone, keys = 20, 148 * 2500 * 128
    cache = make_cache(64, 64, 1, 128, seed=4)
    width = keys // 64 + 1
    table = torch.randint(0, 64, (2, width), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    q = torch.randn((1 + alone, 4, 128), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    out, lse = torch.empty_like(q), torch.empty((1 + alone, 4), device="cuda")
    work = torch.empty(silkern.shared_workspace_bytes(1 + alone, 4, 1, 128, 1 + alone, 1), dtype=torch.uint8, device="cuda")
    status = ints(0)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    cycles = 1_000_000
    with wait_bound(cycles):
        begin.record()
        silkern.attend_shared(q, torch.arange(2 + alone, dtype=torch.int32, device="cuda"), ints(keys, *[9] * alone), ints(0, *[1] * alone),
                              ints(0, 1), ints(0), table, *cache, out, lse, work, softmax_scale=128**-0.5, status=status)
        end.record()
    # at 2 GHz at most, a CTA that works throughout the call exceeds the bound twice over
    assert begin.elapsed_time(end) * 2e6 > 2 * cycles
    assert int(status) == 0 and bool(lse.isfinite().all()) and bool(out.isfinite().all())


@pytest.mark.parametrize("cu,groups", [
    ((0, 40, 0, 40, 3), (0, 2, 4)),
    ((5, 3, 12, 13, 37), (0, 2, 4)),
    ((1, 2, 12, 13, 37), (0, 4, 1)),
    ((1, 2, 12, 13, 37), (3, 0, 4)),
    ((-9, 400, -400, 400, 20), (4, -1, 9)),
])
def test_arrays_that_descend_are_flagged_and_nothing_is_seen(cu, groups) -> None:
    call = Call(8, 2, 128, torch.bfloat16)
    good = call()
    call.cu, call.cu_groups = ints(*cu), ints(*groups)
    guard = call.work.numel()
    whole = torch.full((guard + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    call.work = whole[:guard]
    out, lse = call(status=call.status)
    assert int(call.status) == STATUS_BAD_LENGTH
    assert bool((whole[guard:] == 0x5A).all())
    first, last = min(max(cu[0], 0), 40), min(max(cu[-1], 0), 40)
    assert bool((out[first:last] == 0).all()) and bool((lse[first:last] == -math.inf).all())
    assert all(bool((t[rest] == 7).all()) for t in (out, lse) for rest in (slice(0, first), slice(max(first, last), None)))
    call.cu, call.cu_groups = ints(1, 2, 12, 13, 37), ints(0, 2, 4)
    again = call()
    assert torch.equal(again[0], good[0]) and torch.equal(again[1], good[1])


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (64, 1, 128), (48, 1, 64)])
def test_waits_that_run_out_in_the_middle(heads, kv_heads, dim) -> None:
    """Bounds from a fraction of a tile's time to that of many tiles: warps give up at every point of the work, beside
    others that are through with theirs or still issue. A call is right, or NaN throughout with its status bit; the next
    one is right."""
    call = Call(heads, kv_heads, dim, torch.bfloat16)
    want = call(status=call.status)
    assert int(call.status) == 0 and bool(want[1].isfinite().all())
    for bound in [int(100 * 1.5**i) for i in range(16)]:
        call.status.zero_()
        with wait_bound(bound):
            out, lse = call(status=call.status)
        gone = int(call.status) != 0
        assert int(call.status) in (0, STATUS_WAIT_TIMEOUT)
        if gone:
            assert bool(out[1:37].isnan().all()) and bool(lse[1:37].isnan().all())
        else:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        again = call()
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
