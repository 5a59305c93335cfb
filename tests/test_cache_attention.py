"""The 8-bit cache's entry points without a GPU: refusals before any launch, and the oracle itself.

The C ABI checks its arguments on the host before any CUDA call, so rejected
calls are made with addresses that are never dereferenced.
"""

from __future__ import annotations

import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import attention as oracle  # noqa: E402
from silkern_b200 import _native, ops  # noqa: E402
from silkern_b200.build import build  # noqa: E402
from tests.attention_cases import make_cache  # noqa: E402

K, V, KS, VS, Q, OUT, LSE, IDX, STEP = (0x100000000 * (i + 1) for i in range(9))


@pytest.fixture(scope="module")
def lib():
    build()
    return _native.load()


def cache(latent=False, **over):
    dim, heads = (576, 1) if latent else (128, 2)
    f = dict(k=K, v=None if latent else V, k_scale=KS, v_scale=None if latent else VS, num_blocks=8, block_size=16,
             kv_heads=heads, key_dim=dim, value_dim=512 if latent else dim, k_block=16 * heads * dim, k_token=heads * dim,
             k_head=dim, v_block=0 if latent else 16 * heads * dim, v_token=0 if latent else heads * dim,
             v_head=0 if latent else dim)
    f.update(over)
    return _native.Cache(*[f[name] for name, _ in _native.Cache._fields_])


def selected(lib, c, **over):
    a = dict(q=Q, q_row=256, q_head=128, type=0, rows=2, heads=2, slots=IDX, slots_row=32, width=32, counts=None, out=OUT,
             out_row=256, out_head=128, lse=LSE, scale=0.1)
    a.update(over)
    return lib.silkern_attend_selected_v1(ctypes.addressof(c), a["q"], a["q_row"], a["q_head"], a["type"], a["rows"],
                                          a["heads"], a["slots"], a["slots_row"], a["width"], a["counts"], a["out"],
                                          a["out_row"], a["out_head"], a["lse"], a["scale"], None, None)


def window(lib, c, **over):
    a = dict(q=Q, type=0, rows=2, heads=2, cu=IDX, lengths=IDX + STEP, req=IDX + 2 * STEP, seqs=2, table=IDX + 3 * STEP,
             table_rows=2, table_width=4, window=0, sinks=0, dcp=1, rank=0, il=1, out=OUT, lse=LSE, scale=0.1)
    a.update(over)
    return lib.silkern_attend_window_v1(ctypes.addressof(c), a["q"], 256, 128, a["type"], a["rows"], a["heads"], a["cu"],
                                        a["lengths"], a["req"], a["seqs"], a["table"], a["table_rows"], a["table_width"],
                                        a["window"], a["sinks"], a["dcp"], a["rank"], a["il"], a["out"], 256, 128, a["lse"],
                                        a["scale"], None, None)


def append(lib, c, **over):
    a = dict(keys=Q, values=OUT, type=0, tokens=3, cu=IDX, starts=IDX + STEP, req=IDX + 2 * STEP, seqs=1,
             table=IDX + 3 * STEP, table_rows=1, table_width=4, dcp=1, rank=0, il=1)
    a.update(over)
    return lib.silkern_append_quantized_v1(ctypes.addressof(c), a["keys"], 256, 128, a["values"], 256, 128, a["type"],
                                           a["tokens"], a["cu"], a["starts"], a["req"], a["seqs"], a["table"],
                                           a["table_rows"], a["table_width"], a["dcp"], a["rank"], a["il"], None, None)


def merge(lib, **over):
    a = dict(outs=Q, lses=IDX, type=0, ranks=2, rows=2, heads=2, dim=8, out=OUT, lse=LSE)
    a.update(over)
    return lib.silkern_merge_partials_v1(a["outs"], 32, 16, 8, a["lses"], a["type"], a["ranks"], a["rows"], a["heads"],
                                         a["dim"], a["out"], 16, 8, a["lse"], None)


CACHE_REFUSALS = [
    (dict(k=None), 1), (dict(k_scale=None), 1), (dict(v=None), 1), (dict(v_scale=None), 1), (dict(key_dim=96), 9),
    (dict(value_dim=64), 9), (dict(kv_heads=0), 9), (dict(num_blocks=0), 9), (dict(block_size=0), 4),
    (dict(block_size=65537), 4), (dict(num_blocks=2**31 // 16), 9), (dict(k_token=250), 9), (dict(v_head=-16), 9),
    (dict(k=K + 8), 9), (dict(v=V + 4), 9),
]


@pytest.mark.parametrize(("over", "code"), CACHE_REFUSALS)
def test_cache_refusals(lib, over, code) -> None:
    c = cache(**over)
    assert selected(lib, c) == code
    assert window(lib, c) == code
    assert append(lib, c) == code


def test_latent_cache_refusals(lib) -> None:
    for over in (dict(value_dim=576), dict(kv_heads=2), dict(v=V), dict(v_scale=VS)):
        assert selected(lib, cache(latent=True, **over)) == 9
    assert append(lib, cache(latent=True)) == 9  # values for a cache that has none


@pytest.mark.parametrize(("over", "code"), [
    (dict(q=None), 1), (dict(out=None), 1), (dict(lse=None), 1), (dict(slots=None), 1), (dict(type=2), 11),
    (dict(rows=0), 2), (dict(rows=2**31), 2), (dict(heads=0), 10), (dict(heads=3), 10), (dict(heads=65536), 10),
    (dict(q_row=260), 9), (dict(q_head=4), 9), (dict(q=Q + 2), 9), (dict(width=0), 2), (dict(width=2**31 - 1), 2),
    (dict(scale=math.inf), 12), (dict(scale=math.nan), 12), (dict(out=Q), 6), (dict(out=Q + 500), 6), (dict(lse=IDX), 6),
    (dict(out=K), 6), (dict(lse=VS), 6), (dict(lse=OUT + 1000), 6), (dict(counts=OUT), 6),
])
def test_attend_selected_refusals(lib, over, code) -> None:
    assert selected(lib, cache(), **over) == code


@pytest.mark.parametrize(("over", "code"), [
    (dict(cu=None), 1), (dict(lengths=None), 1), (dict(req=None), 1), (dict(table=None), 1), (dict(seqs=0), 2),
    (dict(seqs=2**26), 2), (dict(table_rows=0), 2), (dict(table_width=0), 2), (dict(window=-1), 12), (dict(sinks=-1), 12),
    (dict(window=2**31), 12), (dict(dcp=0), 3), (dict(rank=1), 3), (dict(il=0), 3), (dict(il=3), 4),
    (dict(dcp=2**30, il=16), 3), (dict(heads=5), 10), (dict(out=IDX), 6), (dict(lse=IDX + 3 * STEP + 16), 6),
])
def test_attend_window_refusals(lib, over, code) -> None:
    assert window(lib, cache(), **over) == code


@pytest.mark.parametrize(("over", "code"), [
    (dict(keys=None), 1), (dict(values=None), 1), (dict(cu=None), 1), (dict(starts=None), 1), (dict(req=None), 1),
    (dict(table=None), 1), (dict(type=7), 11), (dict(tokens=0), 2), (dict(seqs=0), 2), (dict(table_width=0), 2),
    (dict(dcp=2, rank=2), 3), (dict(il=5), 4), (dict(keys=K), 6), (dict(values=KS), 6), (dict(table=V + 64), 6),
    (dict(starts=VS), 6),
])
def test_append_refusals(lib, over, code) -> None:
    assert append(lib, cache(), **over) == code


@pytest.mark.parametrize(("over", "code"), [
    (dict(outs=None), 1), (dict(lses=None), 1), (dict(out=None), 1), (dict(type=-1), 11), (dict(ranks=0), 2),
    (dict(rows=0), 2), (dict(heads=0), 2), (dict(dim=0), 2), (dict(rows=2**40), 2), (dict(out=Q + 64), 6), (dict(lse=IDX), 6),
    (dict(lse=OUT), 6),
])
def test_merge_refusals(lib, over, code) -> None:
    assert merge(lib, **over) == code


def test_status_strings_of_the_new_codes(lib) -> None:
    for code in (9, 10, 11, 12):
        assert _native.status_string(code) != "unknown status"


def test_launchers_refuse_host_tensors() -> None:
    k, v, ks, vs = make_cache(2, 4, 1, 64, device="cpu")
    q = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(silkern.LocalizationError, match="must be CUDA tensors"):
        silkern.attend_selected(q, table, k, v, ks, vs, q.clone(), torch.zeros(1, 1), softmax_scale=1.0)
    with pytest.raises(silkern.LocalizationError, match="must be CUDA tensors"):
        silkern.attend_window(q, ints, ints[:1], ints[:1], table, k, v, ks, vs, q.clone(), torch.zeros(1, 1), softmax_scale=1.0)
    with pytest.raises(silkern.LocalizationError, match="must be CUDA tensors"):
        silkern.append_quantized(q, q, k, v, ks, vs, ints, ints[:1], ints[:1], table)
    with pytest.raises(silkern.LocalizationError, match="must be CUDA tensors"):
        silkern.merge_partials(q[None], torch.zeros(1, 1, 1), q.clone())
    with pytest.raises(silkern.LocalizationError, match="must be torch tensors"):
        silkern.merge_partials([1], torch.zeros(1, 1, 1), q.clone())


# ---------------------------------------------------------------------- the oracle

def test_oracle_attention_is_softmax_of_the_stored_values() -> None:
    k, v, ks, vs = make_cache(5, 8, 2, 64, seed=1, device="cpu")
    q = torch.randn((3, 6, 64), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    slots = torch.randint(-1, 40, (3, 20), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    out, lse, spread, near = oracle.attend_selected(q, slots, k, v, ks, vs, softmax_scale=0.2)
    for r in range(3):
        for h in range(6):
            s = [i for i in slots[r].tolist() if i >= 0]
            keys = torch.stack([k[i // 8, i % 8, h // 3].float().double() * ks[i // 8, h // 3].double() for i in s])
            values = torch.stack([v[i // 8, i % 8, h // 3].float().double() * vs[i // 8, h // 3].double() for i in s])
            w = torch.softmax(keys @ q[r, h].double() * 0.2, dim=0)
            assert torch.allclose(out[r, h], w @ values, rtol=1e-12, atol=1e-12)
            assert bool((spread[r, h] <= near[r, h] + 1e-12).all())


def test_oracle_window_of_ranks_merges_to_the_whole() -> None:
    g = torch.Generator().manual_seed(4)
    length, block_size, dcp = 61, 4, 2
    q = torch.randn((5, 2, 64), generator=g).to(torch.float16)
    x = torch.randn((length, 1, 64), generator=g).to(torch.bfloat16)
    cu, lens, req = (torch.tensor(t, dtype=torch.int32) for t in ([0, 5], [length], [0]))
    parts, sizes = [], (1, dcp)
    for size in sizes:
        outs = []
        for rank in range(size):
            width = -(-length // (size * block_size)) + 1
            empty = make_cache(width, block_size, 1, 64, seed=5, device="cpu")
            table = torch.randperm(width, generator=g).to(torch.int32)[None]
            own = dict(dcp_size=size, dcp_rank=rank)
            stored = oracle.append(x, x, *empty, torch.tensor([0, length]), torch.tensor([0]), req, table, **own)
            outs.append(oracle.attend_window(q, cu, lens, req, table, *stored, softmax_scale=0.1, window=20, sinks=3, **own))
        parts.append(oracle.merge(torch.stack([o[0] for o in outs]), torch.stack([o[1] for o in outs])))
    # the ranks' pages have other scales: powers of two, so all codes but subnormal ones agree
    assert torch.allclose(parts[0][0], parts[1][0], rtol=0, atol=2.0**-9)
    assert torch.allclose(parts[0][1], parts[1][1], rtol=0, atol=2.0**-9)


def test_oracle_append_scales_are_the_smallest_powers_of_two() -> None:
    for most in (448.0, 449.0, 1.0, 1.75, 1.7578125, 3e-38, 1e38):
        k, v, ks, vs = make_cache(1, 4, 1, 64, seed=6, device="cpu")
        x = torch.zeros((2, 1, 64), dtype=torch.bfloat16)
        x[1, 0, 7] = most
        most = float(x.max())
        one = torch.tensor([0], dtype=torch.int32)
        _, _, scale, _ = oracle.append(x, x, k, v, ks, vs, torch.tensor([0, 2]), one, one, one[None])
        s = float(scale[0, 0])
        assert math.frexp(s)[0] == 0.5 and 448 * s >= min(most, 448 * 2.0**100)
        assert s == 2.0**-100 or s / 2 * 448 < most


# ---------------------------------------------------------------------- further refusals, ops

def test_a_scale_that_overflows_in_base_two_is_refused(lib) -> None:
    """3e38 is a float32, 3e38 * log2(e) is not."""
    assert selected(lib, cache(), scale=3e38) == 12
    assert window(lib, cache(), scale=-3e38) == 12


def test_ops_mark_exactly_the_written_buffers() -> None:
    ops.register()
    written = {name: {a.name for a in getattr(torch.ops.silkern_b200, name).default._schema.arguments
                      if a.alias_info is not None and a.alias_info.is_write}
               for name in ("append_quantized", "attend_selected", "attend_window", "merge_partials")}
    assert written == {"append_quantized": {"k_cache", "v_cache", "k_scale", "v_scale", "status"},
                       "attend_selected": {"out", "lse", "status"}, "attend_window": {"out", "lse", "status"},
                       "merge_partials": {"out", "lse"}}


@pytest.mark.parametrize("latent", [False, True])
def test_launchers_trace_as_op_nodes_without_a_graph_break(latent) -> None:
    """One node for each of the four launchers, and fake implementations that
    launch nothing; the backend only inspects the graph."""
    ops.register()
    graphs = []

    def inspect(gm, example_inputs):
        graphs.append(gm)
        return lambda *args: None

    k, v, ks, vs = make_cache(2, 4, 1, 576 if latent else 64, latent=latent, device="cpu")
    dim, value_dim = (576, 512) if latent else (64, 64)
    q = torch.zeros((1, 2, dim), dtype=torch.bfloat16)
    new = torch.zeros((1, 1, dim), dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros((1, 1), dtype=torch.int32)
    outs, lses = torch.zeros((2, 1, 2, value_dim), dtype=torch.bfloat16), torch.zeros(2, 1, 2)
    out = torch.zeros((1, 2, value_dim), dtype=torch.bfloat16)

    def step(q, new, ints, one, table, outs, lses, out):
        silkern.append_quantized(new, None if latent else new, k, v, ks, vs, ints, one, one, table)
        silkern.attend_selected(q, table, k, v, ks, vs, outs[0], lses[0], softmax_scale=0.1, counts=one)
        silkern.attend_window(q, ints, one, one, table, k, v, ks, vs, outs[1], lses[1], softmax_scale=0.1, window=3)
        silkern.merge_partials(outs, lses, out)

    torch._dynamo.reset()
    torch.compile(step, backend=inspect, fullgraph=True)(q, new, ints, ints[:1].clone(), table, outs, lses, out)
    assert len(graphs) == 1
    targets = [str(node.target) for node in graphs[0].graph.nodes if node.op == "call_function"]
    for name in ("append_quantized", "attend_selected", "attend_window", "merge_partials"):
        assert sum(f"silkern_b200.{name}" in t for t in targets) == 1


def test_merge_refuses_columns_past_its_numbers(lib) -> None:
    """Columns are counted in 32 bits, up to 256 at a step: from 2**31 - 255 on
    the count would turn negative and never end."""
    for dim in (2**31 - 255, 2**31 - 1, 2**31):
        assert merge(lib, dim=dim) == 2
    assert merge(lib, dim=2**31 - 256, out=Q + 64) == 6  # a size that can be counted, found to overlap


# ---------------------------------------------------------------------- bindings that are not what a call needs

def host_calls():
    """name -> (launcher, buffers by name, keywords): right but for lying on the host, which is looked at
    after what these tests ask for."""
    k, v, ks, vs = make_cache(2, 4, 1, 64, device="cpu")
    cache = dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)
    q, out, lse = torch.zeros((1, 1, 64), dtype=torch.bfloat16), torch.zeros((1, 1, 64), dtype=torch.bfloat16), torch.zeros(1, 1)
    cu, one, table = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    return {
        "selected": (silkern.attend_selected, dict(q=q, slots=table, **cache, out=out, lse=lse), dict(softmax_scale=1.0)),
        "window": (silkern.attend_window, dict(q=q, cu_tokens=cu, lengths=one, req_ids=one, block_table=table, **cache,
                                               out=out, lse=lse), dict(softmax_scale=1.0)),
        "append": (silkern.append_quantized, dict(keys=q, values=q.clone(), **cache, cu_tokens=cu, starts=one, req_ids=one,
                                                  block_table=table), {}),
        "merge": (silkern.merge_partials, dict(outs=q[None], lses=lse[None], out=out, lse=lse.clone()), {}),
    }


OPTIONAL = {"v_cache", "v_scale", "values"}


@pytest.mark.parametrize("name", ["selected", "window", "append", "merge"])
def test_a_missing_buffer_is_refused(name) -> None:
    call, buffers, kw = host_calls()[name]
    for which in buffers:
        if which in OPTIONAL or (name, which) == ("merge", "lse"):
            continue
        for wrong in (None, 3, [1.0]):
            with pytest.raises(silkern.LocalizationError, match="must be torch tensors"):
                call(**{**buffers, which: wrong}, **kw)


GRADIENTS = [("selected", "q"), ("selected", "out"), ("selected", "lse"), ("selected", "k_scale"), ("window", "q"),
             ("window", "v_scale"), ("append", "keys"), ("append", "values"), ("append", "k_scale"), ("merge", "outs"),
             ("merge", "lses"), ("merge", "out")]


@pytest.mark.parametrize("name,which", GRADIENTS)
def test_a_call_that_autograd_records_is_refused(name, which) -> None:
    """There is no backward pass: a result without a graph would drop the gradients."""
    call, buffers, kw = host_calls()[name]
    buffers[which] = buffers[which].clone().requires_grad_()
    with pytest.raises(silkern.LocalizationError, match="no gradient"):
        call(**buffers, **kw)
    with torch.no_grad(), pytest.raises(silkern.LocalizationError, match="must be CUDA tensors"):
        call(**buffers, **kw)


def test_a_traced_call_that_autograd_records_is_refused() -> None:
    ops.register()
    call, buffers, kw = host_calls()["merge"]
    buffers["outs"] = buffers["outs"].clone().requires_grad_()
    torch._dynamo.reset()
    with pytest.raises(Exception, match="no gradient"):
        torch.compile(lambda b: call(**b), backend="eager", fullgraph=True)(buffers)


@pytest.mark.parametrize("scale", ["0.1", None, 0.1j, [0.1], torch.ones(2), math.inf, -math.inf, math.nan])
def test_a_softmax_scale_that_is_no_finite_number_is_refused(scale) -> None:
    from silkern_b200 import attention

    with pytest.raises(silkern.LocalizationError, match="finite"):
        attention._check_scale(scale)
    for good in (0.1, 2, torch.tensor(0.5)):
        attention._check_scale(good)


@pytest.mark.parametrize("offset", [0, 2 * 128, 2 * 255, 2 * 1023, -2 * 16, 2 * 1024 * 3 + 2 * 200])
def test_results_between_the_rows_of_their_inputs_may_not_reach_into_them(lib, offset) -> None:
    """Rows of 1024 elements: q has the first 256 of each, out would have 256 that meet them."""
    assert selected(lib, cache(), rows=4, q_row=1024, out_row=1024, out=Q + offset) == 6
    assert selected(lib, cache(), rows=4, q_row=1024, out_row=1040, out=Q + 2 * 256) == 6  # steps that differ
    assert selected(lib, cache(), rows=4, q_row=1024, out_row=1024, out=OUT, lse=OUT + 2 * 256) == 6


def test_append_refuses_keys_and_values_in_the_same_place(lib) -> None:
    """Keys and values are written by CTAs of their own: they may take turns in one buffer, not share it."""
    for v in (K, K + 16 * 256 * 3, K + 128, K - 16 * 256):
        assert append(lib, cache(v=v)) == 6
    halves = dict(k_block=2 * 16 * 256, v_block=2 * 16 * 256)  # (num_blocks, 2, block_size, kv_heads, dim)
    assert append(lib, cache(v=K + 16 * 256 - 16, **halves)) == 6


def test_outputs_that_overlap_themselves_are_refused(lib) -> None:
    """Expanded outputs, and strides that are less than what they step over."""
    for row, head in ((0, 128), (256, 0), (128, 128), (256, 64), (248, 128), (8, 8)):
        assert selected(lib, cache(), out_row=row, out_head=head) == 6
    for blocks, tokens, heads in ((0, 256, 128), (16 * 256, 0, 128), (16 * 256, 256, 0), (16 * 256, 128, 128), (256, 256, 128)):
        layout = dict(k_block=blocks, k_token=tokens, k_head=heads)
        assert append(lib, cache(**layout)) == 6
        assert append(lib, cache(**{name.replace("k_", "v_"): n for name, n in layout.items()})) == 6
    assert lib.silkern_merge_partials_v1(Q, 32, 16, 8, IDX, 0, 2, 2, 2, 8, OUT, 0, 8, LSE, None) == 6
    assert lib.silkern_merge_partials_v1(Q, 32, 16, 8, IDX, 0, 2, 2, 2, 8, OUT, 16, 4, LSE, None) == 6


def test_strides_past_the_row_numbers_are_refused(lib) -> None:
    """A row's number, in steps of what divides the strides, has to fit 31 bits: 16-byte steps reach 2**35 bytes."""
    far = dict(num_blocks=2, k_head=16 * 11, k_token=16 * 22, k_block=2**35)
    values = {name.replace("k_", "v_"): n for name, n in far.items()}
    results = dict(out=2**45, lse=2**46)  # behind the caches' bytes
    for c in (cache(**far), cache(**values)):
        assert selected(lib, c, **results) == 9
        assert window(lib, c, **results) == 9
    latent = cache(latent=True, num_blocks=2, k_token=592, k_block=2**35)
    assert selected(lib, latent, out_row=1024, out_head=512, **results) == 9


def test_strides_that_run_backwards_are_followed(lib) -> None:
    """From C, rows may lie from the last address to the first: an overlap with them is seen there."""
    assert selected(lib, cache(), rows=4, q_row=-256, out=Q - 2 * 256 * 3) == 6
    assert selected(lib, cache(), rows=4, out=Q + 2 * 256 * 3, out_row=-256) == 6
    assert selected(lib, cache(), rows=4, out=Q + 2 * 256 * 7 - 2, out_row=-256) == 6
    assert selected(lib, cache(), rows=4, slots=IDX, slots_row=-32, lse=IDX - 4 * 32 * 3) == 6
    assert lib.silkern_merge_partials_v1(Q, 32, 16, 8, IDX, 0, 2, 2, 2, 8, Q + 2 * 72, -16, 8, LSE, None) == 6
