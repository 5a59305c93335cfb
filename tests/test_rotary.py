"""Rotation of heads and reading of the 8-bit cache without a GPU: refusals, frequencies and the oracle."""

from __future__ import annotations

import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import silkern_b200 as silkern  # noqa: E402
from oracle import rotary as oracle  # noqa: E402
from silkern_b200 import _native, ops  # noqa: E402
from silkern_b200.build import build  # noqa: E402

Q, K, QO, KO, WQ, WK, POS, FREQ = (0x100000000 * (i + 1) for i in range(8))


@pytest.fixture(scope="module")
def lib():
    build()
    return _native.load()


def rotate(lib, with_k=True, **over):
    a = dict(q=Q, k=K, q_out=QO, k_out=KO, q_weight=WQ, k_weight=WK, heads=4, kv_heads=2, q_norm=64, k_norm=64, type=0, tokens=3,
             dim=64, positions=POS, frequencies=FREQ, pairs=16, start=0, interleaved=0, f32=1, amplitude=1.0, eps=1e-6,
             q_token=256, q_head=64, out_token=256, out_head=64)
    a.update(over)
    sets = [_native.Heads(a["q"], a["q_out"], a["q_weight"], a["q_token"], a["q_head"], a["out_token"], a["out_head"], a["heads"],
                          a["q_norm"]),
            _native.Heads(a["k"], a["k_out"], a["k_weight"], 128, 64, 128, 64, a["kv_heads"], a["k_norm"])]
    return lib.silkern_rotate_heads_v1(ctypes.addressof(sets[0]), ctypes.addressof(sets[1]) if with_k else None, a["type"],
                                       a["tokens"], a["dim"], a["positions"], a["frequencies"], a["pairs"], a["start"],
                                       a["interleaved"], a["f32"], a["amplitude"], a["eps"], None)


@pytest.mark.parametrize(("over", "code"), [
    (dict(q=None), 1), (dict(q_out=None), 1), (dict(k=None), 1), (dict(k_out=None), 1), (dict(positions=None), 1),
    (dict(frequencies=None), 1), (dict(q_weight=None), 1), (dict(k_weight=None), 1), (dict(type=2), 11), (dict(type=-1), 11),
    (dict(tokens=0), 2), (dict(tokens=2**31), 2), (dict(dim=0), 2), (dict(dim=1025), 2), (dict(heads=0), 10),
    (dict(kv_heads=65536), 10), (dict(pairs=0), 13), (dict(pairs=33), 13), (dict(start=-1), 13), (dict(start=33), 13),
    (dict(start=2**31 - 1), 13), (dict(q_norm=65), 13), (dict(k_norm=-1), 13), (dict(amplitude=math.inf), 13),
    (dict(amplitude=math.nan), 13), (dict(eps=-1e-6), 13), (dict(eps=math.nan), 13),
    (dict(q_out=Q + 2), 6), (dict(q_out=Q, out_token=512), 6), (dict(q_out=K), 6), (dict(k_out=Q + 128), 6), (dict(k_out=QO), 6),
    (dict(q_out=POS), 6), (dict(k_out=FREQ), 6), (dict(q_out=WQ), 6), (dict(k_out=WQ), 6), (dict(out_token=192), 6),
    (dict(out_head=0), 6),
])
def test_rotate_refusals(lib, over, code) -> None:
    assert rotate(lib, **over) == code


def test_rotate_refusals_without_keys(lib) -> None:
    assert rotate(lib, with_k=False, q=None) == 1
    assert rotate(lib, with_k=False, q_out=Q + 2) == 6
    assert _native.status_string(13) != "unknown status"


def tensors(**over):
    a = dict(q=torch.zeros(3, 4, 16, dtype=torch.bfloat16), k=torch.zeros(3, 2, 16, dtype=torch.bfloat16),
             positions=torch.zeros(3, dtype=torch.int32), frequencies=torch.ones(8))
    a.update(q_out=torch.empty_like(a["q"]), k_out=torch.empty_like(a["k"]))
    a.update(over)
    return a


def test_launchers_refuse_host_tensors_and_gradients() -> None:
    with pytest.raises(silkern.LocalizationError, match="CUDA"):
        silkern.rotate_heads(**tensors())
    with pytest.raises(silkern.LocalizationError, match="torch tensors"):
        silkern.rotate_heads(**tensors(q=[1]))
    with pytest.raises(silkern.LocalizationError, match="both given or both None"):
        silkern.rotate_heads(**tensors(k=None))
    with pytest.raises(silkern.LocalizationError, match="needs keys"):
        silkern.rotate_heads(**tensors(k=None, k_out=None), k_weight=torch.ones(4))
    for name in ("q", "k_out", "frequencies"):
        a = tensors()
        a[name].requires_grad_()
        with pytest.raises(silkern.LocalizationError, match="gradient"):
            silkern.rotate_heads(**a)
        with torch.no_grad(), pytest.raises(silkern.LocalizationError, match="CUDA"):
            silkern.rotate_heads(**a)


def test_the_new_ops_are_registered() -> None:
    ops.register()
    written = {"rotate_heads": {"q_out", "k_out"}, "read_quantized": {"keys", "values", "status"}}
    for name, mutated in written.items():
        schema = getattr(torch.ops.silkern_b200, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == mutated


@pytest.mark.parametrize("columns", [2, 8, 64, 128])
def test_frequencies_by_their_definitions(columns) -> None:
    plain, amplitude = silkern.rotary_frequencies(columns, base=500.0)
    want = torch.tensor([500.0 ** (-2 * i / columns) for i in range(columns // 2)], dtype=torch.float64)
    half = 2.0**-24
    assert plain.dtype == torch.float32 and amplitude == 1.0
    assert ((plain.double() - want).abs() <= half * want).all()
    stretched, amplitude = silkern.rotary_frequencies(columns, base=500.0, factor=4.0, method="positions")
    assert ((stretched.double() - want / 4).abs() <= half * want).all() and amplitude == 1.0
    stretched, _ = silkern.rotary_frequencies(columns, base=500.0, factor=4.0, method="base")
    assert float(stretched[0]) == 1.0
    if columns > 2:
        assert abs(float(stretched[-1]) / float(want[-1] / 4) - 1) < 2.0**-20
    stretched, amplitude = silkern.rotary_frequencies(columns, base=500.0, factor=4.0, method="parts", original_length=100,
                                                      slow=1.0, fast=8.0)
    assert amplitude == 0.1 * math.log(4.0) + 1
    for f, w in zip(stretched.double().tolist(), want.tolist()):
        turns = 100 * w / (2 * math.pi)
        keep = min(max((turns - 1.0) / 7.0, 0.0), 1.0)
        assert abs(f - w * (keep + (1 - keep) / 4)) <= 2 * half * w


@pytest.mark.parametrize("bad", [dict(columns=0), dict(columns=7), dict(columns=True), dict(base=0.0), dict(base=math.inf),
                                 dict(factor=0.5), dict(method="other"), dict(method="parts"),
                                 dict(method="parts", original_length=10, slow=3.0, fast=3.0)])
def test_frequency_refusals(bad) -> None:
    with pytest.raises(silkern.LocalizationError):
        silkern.rotary_frequencies(**{"columns": 8, "factor": 2.0, **bad})


def test_the_oracle_turns_pairs_and_keeps_lengths() -> None:
    x = torch.randn(5, 3, 20, dtype=torch.float64)
    f = torch.tensor([1.0, 0.1, 0.01])
    p = torch.tensor([0, 1, -7, 1000, 2**31 - 1])
    for interleaved in (False, True):
        y, _ = oracle.rotate(x, p, f, rotary_start=4, interleaved=interleaved)
        assert torch.equal(y[..., :4], x[..., :4]) and torch.equal(y[..., 10:], x[..., 10:])
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.allclose(y[0], x[0])
        back, _ = oracle.rotate(y, -p, f, rotary_start=4, interleaved=interleaved)
        assert torch.allclose(back, x, atol=1e-12)
    y, _ = oracle.rotate(x, p, f, weight=torch.ones(20), eps=0.0)
    assert torch.allclose(y.norm(dim=-1), torch.full((5, 3), math.sqrt(20.0), dtype=torch.float64))


READ = dict(keys=Q, values=K, type=0, tokens=3, cu=POS, starts=POS + 0x100000, req=POS + 0x200000, seqs=1, table=POS + 0x300000,
            table_rows=1, table_width=4, dcp=1, rank=0, il=1)
CACHE = dict(k=QO, v=KO, k_scale=WQ, v_scale=WK, num_blocks=8, block_size=16, kv_heads=2, key_dim=128, value_dim=128,
             k_block=4096, k_token=256, k_head=128, v_block=4096, v_token=256, v_head=128)


@pytest.mark.parametrize(("over", "code"), [
    (dict(keys=None), 1), (dict(values=None), 1), (dict(cu=None), 1), (dict(starts=None), 1), (dict(req=None), 1),
    (dict(table=None), 1), (dict(type=7), 11), (dict(tokens=0), 2), (dict(tokens=2**31), 2), (dict(seqs=0), 2),
    (dict(seqs=2**30), 2), (dict(table_rows=0), 2), (dict(table_width=0), 2), (dict(dcp=2, rank=2), 3), (dict(il=5), 4),
    (dict(keys=QO), 6), (dict(values=WQ), 6), (dict(keys=POS), 6), (dict(values=Q + 64), 6), (dict(values=KO + 4096), 6),
    (dict(row=128), 6),
])
def test_read_refusals(lib, over, code) -> None:
    a = {**READ, "row": 256, **over}
    c = _native.Cache(*[CACHE[name] for name, _ in _native.Cache._fields_])
    assert lib.silkern_read_quantized_v1(ctypes.addressof(c), a["keys"], a["row"], 128, a["values"], 256, 128, a["type"], a["tokens"],
                                         a["cu"], a["starts"], a["req"], a["seqs"], a["table"], a["table_rows"], a["table_width"],
                                         a["dcp"], a["rank"], a["il"], None, None) == code


def test_read_launcher_refuses_what_append_refuses() -> None:
    z = torch.zeros
    code = torch.float8_e4m3fn
    a = dict(keys=z(3, 2, 64, dtype=torch.bfloat16), values=z(3, 2, 64, dtype=torch.bfloat16),
             k_cache=z(4, 16, 2, 64).to(code), v_cache=z(4, 16, 2, 64).to(code), k_scale=z(4, 2), v_scale=z(4, 2),
             cu_tokens=z(2, dtype=torch.int32), starts=z(1, dtype=torch.int32), req_ids=z(1, dtype=torch.int32),
             block_table=z(1, 4, dtype=torch.int32))
    with pytest.raises(silkern.LocalizationError, match="read buffers must be CUDA"):
        silkern.read_quantized(**a)
    with pytest.raises(silkern.LocalizationError, match="torch tensors"):
        silkern.read_quantized(**{**a, "k_scale": None})
    a["keys"].requires_grad_()
    with pytest.raises(silkern.LocalizationError, match="gradient"):
        silkern.read_quantized(**a)


@pytest.mark.parametrize("bad", [
    dict(base="x"), dict(base=None), dict(base=1j), dict(base=10**400), dict(base=torch.tensor([1e4, 2.0])), dict(factor="2"),
    dict(factor=None), dict(factor=10**400), dict(base=1e300, factor=1e300, method="base"),
    dict(base=1e300, factor=1e12, method="base"), dict(base=1e-300),
    dict(method="parts", original_length=4096, slow=None), dict(method="parts", original_length=4096, slow="a"),
    dict(method="parts", original_length=4096, fast=None), dict(method="parts", original_length=4096, fast=math.nan),
    dict(method="parts", original_length=10**400),
    dict(method="parts", original_length=4096.0), dict(method=["parts"]), dict(method=None)])
def test_frequencies_of_no_numbers_are_refused(bad) -> None:
    """With a LocalizationError, and so are those that float32 does not hold."""
    with pytest.raises(silkern.LocalizationError):
        silkern.rotary_frequencies(**{"columns": 64, "factor": 2.0, **bad})


def test_frequencies_in_traced_callers_and_on_other_default_devices() -> None:
    """Nothing in the making of frequencies looks at a tensor's contents."""
    want, _ = silkern.rotary_frequencies(64, factor=4.0, method="parts", original_length=4096)

    @torch.compile(fullgraph=True, backend="eager")
    def scaled(x):
        f, amplitude = silkern.rotary_frequencies(64, factor=4.0, method="parts", original_length=4096)
        return x * f * amplitude

    assert torch.allclose(scaled(torch.ones(32)), want * (0.1 * math.log(4.0) + 1))
    with torch.device("meta"):
        f, _ = silkern.rotary_frequencies(64)
    assert f.device.type == "meta" and f.shape == (32,)
    for base in (1e-37, 1e-30):  # large, and within float32
        assert bool(silkern.rotary_frequencies(64, base=base)[0].isfinite().all())
