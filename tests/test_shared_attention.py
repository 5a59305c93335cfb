"""Attention behind shared prefixes without a GPU: refusals, the op, the workspace and the oracle."""

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

K, V, KS, VS, Q, OUT, LSE, IDX, WORK = (0x100000000 * (i + 1) for i in range(9))
STEP = 0x100000


@pytest.fixture(scope="module")
def lib():
    build()
    return _native.load()


def cache(**over):
    f = dict(k=K, v=V, k_scale=KS, v_scale=VS, num_blocks=8, block_size=16, kv_heads=2, key_dim=128, value_dim=128,
             k_block=4096, k_token=256, k_head=128, v_block=4096, v_token=256, v_head=128)
    f.update(over)
    return _native.Cache(*[f[name] for name, _ in _native.Cache._fields_])


def shared(lib, c, **over):
    a = dict(q=Q, q_row=512, q_head=128, type=0, rows=2, heads=4, cu=IDX, lengths=IDX + STEP, req=IDX + 2 * STEP, seqs=2,
             cu_groups=IDX + 3 * STEP, prefixes=IDX + 4 * STEP, groups=1, table=IDX + 5 * STEP, table_rows=2, table_width=4, dcp=1,
             rank=0, il=1, out=OUT, lse=LSE, scale=0.1, work=WORK)
    a["bytes"] = max(0, lib.silkern_shared_workspace_v1(2, 4, 2, 128, 2, 1))
    a.update(over)
    return lib.silkern_attend_shared_v1(ctypes.addressof(c), a["q"], a["q_row"], a["q_head"], a["type"], a["rows"], a["heads"],
                                        a["cu"], a["lengths"], a["req"], a["seqs"], a["cu_groups"], a["prefixes"], a["groups"],
                                        a["table"], a["table_rows"], a["table_width"], a["dcp"], a["rank"], a["il"], a["out"], 512,
                                        128, a["lse"], a["scale"], a["work"], a["bytes"], None, None)


@pytest.mark.parametrize(("over", "code"), [
    (dict(q=None), 1), (dict(out=None), 1), (dict(lse=None), 1), (dict(cu=None), 1), (dict(lengths=None), 1), (dict(req=None), 1),
    (dict(cu_groups=None), 1), (dict(prefixes=None), 1), (dict(table=None), 1), (dict(work=None), 1), (dict(type=2), 11),
    (dict(rows=0), 2), (dict(rows=2**31), 2), (dict(seqs=0), 2), (dict(seqs=2**30), 2), (dict(groups=0), 2), (dict(groups=2**30), 2),
    (dict(table_rows=0), 2), (dict(table_width=0), 2), (dict(heads=0), 10), (dict(heads=3), 10), (dict(heads=65536), 10),
    (dict(bytes=0), 8), (dict(q_row=260), 9), (dict(q_head=4), 9), (dict(q=Q + 2), 9), (dict(work=WORK + 8), 9),
    (dict(scale=math.inf), 12), (dict(scale=math.nan), 12), (dict(dcp=0), 3), (dict(rank=1), 3), (dict(il=3), 4),
    (dict(out=Q), 6), (dict(lse=IDX), 6), (dict(out=K), 6), (dict(lse=VS), 6), (dict(work=Q), 6), (dict(work=OUT), 6),
    (dict(work=IDX + 4 * STEP), 6), (dict(out=IDX + 3 * STEP), 6), (dict(work=V + 4096), 6),
])
def test_refusals(lib, over, code) -> None:
    assert shared(lib, cache(), **over) == code


def test_cache_refusals(lib) -> None:
    for over, code in ((dict(k=None), 1), (dict(v=None), 1), (dict(v_scale=None), 1), (dict(key_dim=96), 9), (dict(k_token=250), 9)):
        assert shared(lib, cache(**over)) == code
    latent = cache(v=None, v_scale=None, kv_heads=1, key_dim=576, value_dim=512, k_block=16 * 576, k_token=576, v_block=0, v_token=0,
                   v_head=0)
    assert shared(lib, latent) == 9


def test_workspace_sizes(lib) -> None:
    small = silkern.shared_workspace_bytes(1, 8, 1, 128, 1, 1)
    assert 0 < small <= silkern.shared_workspace_bytes(100, 64, 8, 128, 100, 3)
    for bad in ((0, 8, 1, 128, 1, 1), (1, 8, 3, 128, 1, 1), (1, 8, 1, 96, 1, 1), (1, 8, 1, 128, 0, 1), (1, 8, 1, 128, 1, 2**30),
                (1, 65536, 1, 128, 1, 1), (1.0, 8, 1, 128, 1, 1), (True, 8, 1, 128, 1, 1)):
        with pytest.raises(silkern.LocalizationError):
            silkern.shared_workspace_bytes(*bad)


def test_launcher_refuses_host_tensors_and_gradients() -> None:
    k, v, ks, vs = make_cache(4, 16, 2, 64, device="cpu")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    a = dict(q=q, cu_tokens=ints(0, 1, 2), lengths=ints(3, 4), req_ids=ints(0, 1), cu_groups=ints(0, 2), prefixes=ints(2),
             block_table=ints(0, 1).view(2, 1), k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, out=torch.empty_like(q),
             lse=torch.empty(2, 4), workspace=torch.empty(1024, dtype=torch.uint8), softmax_scale=0.1)
    with pytest.raises(silkern.LocalizationError, match="CUDA"):
        silkern.attend_shared(**a)
    with pytest.raises(silkern.LocalizationError, match="torch tensors"):
        silkern.attend_shared(**{**a, "workspace": None})
    with pytest.raises(silkern.LocalizationError, match="gradient"):
        silkern.attend_shared(**{**a, "q": q.clone().requires_grad_()})


def test_the_op_is_registered() -> None:
    ops.register()
    schema = torch.ops.silkern_b200.attend_shared.default._schema
    written = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    assert written == {"out", "lse", "workspace", "status"}


@pytest.mark.parametrize("prefix", [0, 5, 16, 33])
def test_the_oracle_with_copied_tables_is_the_window_oracle(prefix) -> None:
    """Where every sequence's own row names the shared pages too, nothing tells the two apart."""
    cache = make_cache(9, 8, 2, 64, device="cpu", seed=1)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table = ints(0, 1, 2, 3, 4, 5, 0, 1, 2, 3, 4, 6, 0, 1, 2, 3, 4, 7).view(3, 6)
    q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    cu, lengths, req = ints(0, 1, 3, 4), ints(40, 44, 37), ints(2, 0, 1)
    got = oracle.attend_shared(q, cu, lengths, req, ints(0, 3), ints(prefix), table, *cache, softmax_scale=0.1)
    want = oracle.attend_window(q, cu, lengths, req, table, *cache, softmax_scale=0.1)
    assert torch.allclose(got[0], want[0], atol=1e-12) and torch.allclose(got[1], want[1], atol=1e-12)


def test_more_segments_than_the_plan_counts_are_refused(lib) -> None:
    """A group and a sequence are a segment each; the plan walks them in rounds of 1024 with 32-bit numbers, the round's
    end included."""
    most = 2**30 - 1
    assert lib.silkern_shared_workspace_v1(1, 8, 1, 128, most, most) == -2
    assert lib.silkern_shared_workspace_v1(1, 8, 1, 128, most, 1) > 0
    assert lib.silkern_shared_workspace_v1(1, 8, 1, 128, 1, most) > 0
    assert shared(lib, cache(), seqs=most, groups=most, bytes=2**60) == 2
    with pytest.raises(silkern.LocalizationError):
        silkern.shared_workspace_bytes(1, 8, 1, 128, most, most)
