"""Rotation of heads on the device, against 64-bit arithmetic."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import rotary as oracle  # noqa: E402
from tests.attention_cases import HALF_STEP  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("a CUDA device is required", allow_module_level=True)

TYPES = [torch.bfloat16, torch.float16]


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def assert_rotated(got, want):
    """Within half a step of the type, and the float32 arithmetic's errors: a sum of squares of at most 1024
    columns goes through at most 80 multiply-adds and 5 exchanges (each 2^-24 of the sum), halved by the root, a
    root of 2 units in the last place, and four products: 2^-18.5 + 2^-22 + 2^-22; cos and sin are off by the angle's
    rounding (2^-26 turns are 2^-23.3) and 2 units: 2^-22 of the pair's magnitudes. Together below 2^-17 of them. fp16's
    smallest step is 2^-24."""
    ref, size = want
    bound = HALF_STEP[got.dtype] * ref.abs() + 2.0**-17 * size + (2.0**-25 if got.dtype == torch.float16 else 1e-38)
    error = (got.double() - ref).abs()
    assert bool((error <= bound).all()), f"worst {float((error / bound).max()):.3g} bounds"


def check(q, k, positions, frequencies, q_weight=None, k_weight=None, inplace=False, **kw):
    want_q = oracle.rotate(q, positions, frequencies, weight=q_weight, **kw)
    want_k = None if k is None else oracle.rotate(k, positions, frequencies, weight=k_weight, **kw)
    q_out = q if inplace else torch.full_like(q, 7.0)
    k_out = k if inplace or k is None else torch.full_like(k, 7.0)
    silkern.rotate_heads(q, k, positions, frequencies, q_out, k_out, q_weight=q_weight, k_weight=k_weight, **kw)
    assert_rotated(q_out, want_q)
    if k is not None:
        assert_rotated(k_out, want_k)
    return q_out, k_out


def positions_of(tokens, seed, most=200000):
    p = torch.randint(0, most, (tokens,), generator=torch.Generator().manual_seed(seed))
    p[0] = 0
    return p.to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,start,pairs", [
    (64, 0, 32), (64, 0, 16), (64, 32, 16), (128, 0, 64), (128, 64, 32), (128, 8, 8), (80, 0, 40), (96, 16, 24), (192, 128, 32),
    (256, 0, 128), (576, 512, 32), (1024, 0, 512), (1024, 512, 8), (8, 0, 4), (16, 0, 8), (2, 0, 1), (7, 1, 2), (66, 3, 31),
    (100, 0, 50), (128, 0, 4), (128, 4, 64 - 4), (1023, 1, 511)])
@pytest.mark.parametrize("norms", [None, "whole", "part"])
def test_columns_and_layouts(dtype, interleaved, dim, start, pairs, norms) -> None:
    tokens, heads, kv_heads = 5, 6, 3
    q, k = randn(tokens, heads, dim, dtype=dtype, seed=dim), randn(tokens, kv_heads, dim, dtype=dtype, seed=dim + 1) * 3
    frequencies, amplitude = silkern.rotary_frequencies(2 * pairs, factor=8.0, method="parts", original_length=4096, device="cuda")
    n = {None: 0, "whole": dim, "part": max(1, dim * 2 // 3)}[norms]
    weights = {}
    if n:
        weights = dict(q_weight=1 + randn(n, dtype=torch.float32, seed=3) / 4, k_weight=1 + randn(max(1, n // 2), dtype=torch.float32, seed=4))
    check(q, k, positions_of(tokens, 5), frequencies, rotary_start=start, interleaved=interleaved, amplitude=amplitude, **weights)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(1, 1, None, 128), (1, 64, 8, 128), (64, 64, 8, 128), (333, 5, 5, 64),
                                                       (2000, 32, 4, 64), (3, 130, 1, 576), (700, 3, 2, 80)])
def test_tokens_and_heads(dtype, tokens, heads, kv_heads, dim) -> None:
    q = randn(tokens, heads, dim, dtype=dtype, seed=1)
    k = None if kv_heads is None else randn(tokens, kv_heads, dim, dtype=dtype, seed=2)
    frequencies, _ = silkern.rotary_frequencies(dim, device="cuda")
    weight = (1 + randn(dim, dtype=torch.float32, seed=3) / 4).to(dtype)
    check(q, k, positions_of(tokens, 4), frequencies, q_weight=weight, eps=1e-5)
    if k is not None:
        check(q, k, positions_of(tokens, 4), frequencies, k_weight=weight)


def test_far_and_negative_positions() -> None:
    p = torch.tensor([0, 1, -1, 131071, 1048575, -99999, 2**24 + 1, 2**27 + 3], dtype=torch.int32).cuda()
    q = randn(8, 4, 128, dtype=torch.float16, seed=1)
    frequencies, _ = silkern.rotary_frequencies(128, device="cuda")
    for interleaved in (False, True):
        check(q, None, p, frequencies, interleaved=interleaved)
    check(q, None, torch.full_like(p, 2**31 - 1), frequencies / 1024)
    check(q, None, torch.full_like(p, -(2**31)), frequencies / 1024)


@pytest.mark.parametrize("dim,column", [(128, 0), (128, 8), (64, 1), (72, 0)])
def test_views_of_one_projection_in_place(dim, column) -> None:
    """q, k and v side by side in one buffer: the others' columns stay."""
    heads, kv_heads, tokens = 8, 2, 37
    width = (heads + 2 * kv_heads) * dim + 24
    store = randn(tokens, width, dtype=torch.bfloat16, seed=dim)
    before = store.clone()
    q = store[:, column : column + heads * dim].view(tokens, heads, dim)
    k = store[:, column + heads * dim : column + (heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    frequencies, _ = silkern.rotary_frequencies(dim, device="cuda")
    weight = 1 + randn(dim, dtype=torch.float32, seed=5) / 4
    check(q, k, positions_of(tokens, 6), frequencies, q_weight=weight, k_weight=weight, inplace=True)
    end = column + (heads + kv_heads) * dim
    assert torch.equal(store[:, :column], before[:, :column]) and torch.equal(store[:, end:], before[:, end:])
    # heads outermost, in and out
    x = randn(heads, tokens, dim, dtype=torch.bfloat16, seed=7).transpose(0, 1)
    out = torch.full((heads, tokens + 1, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    silkern.rotate_heads(x, None, positions_of(tokens, 6), frequencies, out[:, 1:].transpose(0, 1), None)
    assert_rotated(out[:, 1:].transpose(0, 1), oracle.rotate(x, positions_of(tokens, 6), frequencies))
    assert bool((out[:, 0] == 7).all())


def test_zeros_infinities_and_nan_stay_in_their_head() -> None:
    q = randn(3, 4, 64, dtype=torch.bfloat16, seed=1)
    q[0, 0] = 0
    q[1, 1, 5] = float("nan")
    q[2, 2, 63] = float("inf")
    frequencies, _ = silkern.rotary_frequencies(64, device="cuda")
    weight = torch.ones(64, device="cuda")
    out = torch.empty_like(q)
    silkern.rotate_heads(q, None, positions_of(3, 2), frequencies, out, None, q_weight=weight)
    clean = torch.ones(3, 4, dtype=torch.bool)
    clean[1, 1] = clean[2, 2] = False
    want = oracle.rotate(q, positions_of(3, 2), frequencies, weight=weight)
    assert_rotated(out[clean], (want[0][clean], want[1][clean]))
    assert bool((out[0, 0] == 0).all()) and bool(out[1, 1].isnan().all())


def test_refusals_on_the_device() -> None:
    q, k = randn(3, 4, 64, dtype=torch.bfloat16, seed=1), randn(3, 2, 64, dtype=torch.bfloat16, seed=2)
    good = dict(q=q, k=k, positions=positions_of(3, 1), frequencies=torch.ones(16, device="cuda"), q_out=torch.empty_like(q),
                k_out=torch.empty_like(k))
    silkern.rotate_heads(**good)
    w = torch.ones(64, device="cuda")
    for bad in (dict(q=q[:2]), dict(q=q[0]), dict(k=k[..., :32]), dict(k=k.half()), dict(q_out=torch.empty_like(q).half()),
                dict(q_out=q[:, :2]), dict(positions=positions_of(4, 1)), dict(positions=positions_of(3, 1).long()),
                dict(frequencies=torch.ones(33, device="cuda")), dict(frequencies=torch.ones(0, device="cuda")),
                dict(frequencies=torch.ones(16, device="cuda").double()), dict(frequencies=torch.ones(32, device="cuda")[::2]),
                dict(rotary_start=33), dict(rotary_start=-1), dict(rotary_start=1.0), dict(interleaved=1), dict(amplitude=float("nan")),
                dict(amplitude="1"), dict(eps=-1.0), dict(eps=None), dict(q_weight=torch.ones(65, device="cuda")),
                dict(q_weight=w, k_weight=w.bfloat16()), dict(q_weight=w.half()), dict(q_weight=w[::2]), dict(q_out=q.flip(0).transpose(0, 1)),
                dict(q_out=k), dict(k_out=q[:, :2]), dict(q_out=q[:1].expand(3, 4, 64)), dict(positions=positions_of(3, 1).cpu()),
                dict(q=q.float()), dict(k=None), dict(q=None)):
        with pytest.raises(silkern.LocalizationError):
            silkern.rotate_heads(**{**good, **bad})
    shifted = torch.empty(q.numel() + 64, dtype=q.dtype, device="cuda")
    with pytest.raises(silkern.LocalizationError):
        silkern.rotate_heads(**{**good, "q": shifted[64:].view_as(q), "q_out": shifted[:-64].view_as(q)})


def test_graphs_streams_and_compiled_callers() -> None:
    q, k = randn(70, 8, 128, dtype=torch.bfloat16, seed=1), randn(70, 2, 128, dtype=torch.bfloat16, seed=2)
    frequencies, _ = silkern.rotary_frequencies(128, device="cuda")
    p = positions_of(70, 3)
    weight = torch.ones(128, device="cuda")
    want_q, want_k = torch.empty_like(q), torch.empty_like(k)

    def step(q, k, p, q_out, k_out):
        silkern.rotate_heads(q, k, p, frequencies, q_out, k_out, q_weight=weight, k_weight=weight)

    step(q, k, p, want_q, want_k)
    torch.cuda.synchronize()
    out_q, out_k = torch.zeros_like(q), torch.zeros_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, k, p, out_q, out_k)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out_q, want_q) and torch.equal(out_k, want_k)
    out_q.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, p, out_q, out_k)
    side.synchronize()
    assert torch.equal(out_q, want_q)
    out_q.zero_(), out_k.zero_()
    torch.compile(step, fullgraph=True)(q, k, p, out_q, out_k)
    assert torch.equal(out_q, want_q) and torch.equal(out_k, want_k)

    def inplace(q, k, p):
        silkern.rotate_heads(q, k, p, frequencies, q, k, q_weight=weight, k_weight=weight)

    a, b = q.clone(), k.clone()
    torch.compile(inplace, fullgraph=True)(a, b, p)
    assert torch.equal(a, want_q) and torch.equal(b, want_k)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads,norm", [(1, None, 576), (1, None, 512), (2, 1, 512), (1, None, 0)])
def test_several_tokens_a_cta_and_two_slots_a_lane(interleaved, heads, kv_heads, norm) -> None:
    """Few heads of 576 columns, of thousands of tokens: the keys of a long latent prompt alone."""
    tokens = 4003  # four to a CTA, three in the last
    q = randn(tokens, heads, 576, dtype=torch.bfloat16, seed=1)
    k = None if kv_heads is None else randn(tokens, kv_heads, 576, dtype=torch.bfloat16, seed=2)
    frequencies, _ = silkern.rotary_frequencies(64, device="cuda")
    weight = 1 + randn(norm, dtype=torch.float32, seed=3) / 4 if norm else None
    p = positions_of(tokens, 4)
    check(q, k, p, frequencies, q_weight=weight, rotary_start=512, interleaved=interleaved)
    if k is not None:
        check(q, k, p, frequencies, k_weight=weight, rotary_start=512, interleaved=interleaved)
    check(q, k, p, frequencies, q_weight=weight, rotary_start=512, interleaved=interleaved, inplace=True)


def test_views_of_one_projection_in_place_under_compile() -> None:
    """q and k as slices of one buffer, written in place by a compiled caller that goes on with both."""
    tokens, heads, kv_heads, dim = 37, 8, 2, 128
    x = randn(tokens, heads + 2 * kv_heads, dim, dtype=torch.bfloat16, seed=1)
    frequencies, _ = silkern.rotary_frequencies(dim, device="cuda")
    weight = torch.ones(dim, device="cuda")
    p = positions_of(tokens, 3)

    def step(x):
        q, k = x[:, :heads], x[:, heads : heads + kv_heads]
        silkern.rotate_heads(q, k, p, frequencies, q, k, q_weight=weight, k_weight=weight)
        return q * 2, k + 1, x[:, heads + kv_heads :].clone()

    want_x = x.clone()
    want = step(want_x)
    got = torch.compile(step, fullgraph=True)(x)
    assert torch.equal(x, want_x) and all(torch.equal(a, b) for a, b in zip(got, want))
