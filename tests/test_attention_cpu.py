"""Attention over token sequences: what the entry points refuse, before any launch (no GPU), and the oracle against itself."""
import ctypes
import math

import pytest
import torch

from aexrt_b200 import _native, ops
from tests import _attention as oracle

FAKE = ctypes.c_void_p(4096)  # never dereferenced: the checks come first


def _desc(**kw):
    d = _native.AexrtB200AttentionDesc()
    base = dict(struct_size=ctypes.sizeof(d), dtype=0, num_seqs=2, q_tokens=10, max_q=4, q_heads=8, kv_heads=2, head_dim=64,
                causal=1, scale=0.125, kv_tokens=16, page_size=16, table_columns=4, table_stride=4, q_token_stride=512,
                q_head_stride=64, out_token_stride=512, out_head_stride=64, k_token_stride=128, k_head_stride=64,
                k_page_stride=2048, v_token_stride=128, v_head_stride=64, v_page_stride=2048)
    base.update(kw)
    for key, value in base.items():
        setattr(d, key, value)
    return d


SHARED = [
    (dict(struct_size=8), "struct_size"),
    (dict(dtype=2), "dtype"),
    (dict(num_seqs=65536), "65535 sequences"),
    (dict(head_dim=0), "head_dim"),
    (dict(head_dim=60), "head_dim"),
    (dict(head_dim=136), "head_dim"),
    (dict(kv_heads=0), "q_heads"),
    (dict(q_heads=0), "q_heads"),
    (dict(q_heads=7), "q_heads"),
    (dict(q_heads=258, out_token_stride=258 * 64), "128 query heads"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"),
    (dict(q_tokens=(1 << 30) + 1), "2^30"),
    (dict(q_token_stride=513), "multiples of 8"),
    (dict(k_head_stride=4), "multiples of 8"),
    (dict(v_token_stride=1 << 39), "out of range"),
    (dict(out_head_stride=56), "overlap"),
    (dict(out_token_stride=504), "overlap"),
    (dict(out_token_stride=64, out_head_stride=64), "overlap"),
    (dict(out_token_stride=64, out_head_stride=632), "overlap"),
]


@pytest.mark.parametrize("kw,msg", SHARED)
def test_attention_descriptions_are_refused(kw, msg):
    lib = _native.load()
    d = _desc(**kw)
    assert lib.aexrt_b200_attention_packed(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None) == 0
    assert msg in _native.last_error()
    assert lib.aexrt_b200_attention_paged_workspace(ctypes.byref(d)) == 2 ** 64 - 1
    assert lib.aexrt_b200_attention_paged(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, 1 << 40,
                                          None) == 0
    assert msg in _native.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(page_size=0), "page_size"), (dict(page_size=4), "page_size"), (dict(page_size=24), "page_size"),
    (dict(page_size=2048), "page_size"), (dict(table_stride=3), "table_stride"), (dict(k_page_stride=12), "multiples of 8"),
    (dict(table_columns=(1 << 26) + 1, table_stride=1 << 27), "2^30 tokens"),
])
def test_paged_descriptions_are_refused(kw, msg):
    lib = _native.load()
    d = _desc(**kw)
    assert lib.aexrt_b200_attention_paged(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, 1 << 40,
                                          None) == 0
    assert msg in _native.last_error()


def test_null_and_misaligned_pointers_are_refused():
    lib = _native.load()
    d = ctypes.byref(_desc())
    odd = ctypes.c_void_p(4104)
    packed = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None]
    for i in (0, 1, 2, 3, 4, 5):
        args = list(packed)
        args[i] = None
        assert lib.aexrt_b200_attention_packed(d, *args) == 0 and "null" in _native.last_error()
    for i in (0, 1, 2, 5):
        args = list(packed)
        args[i] = odd
        assert lib.aexrt_b200_attention_packed(d, *args) == 0 and "aligned" in _native.last_error()
    paged = [FAKE] * 7 + [None, FAKE, 1 << 40, None]
    for i in range(7):
        args = list(paged)
        args[i] = None
        assert lib.aexrt_b200_attention_paged(d, *args) == 0 and "null" in _native.last_error()
    assert lib.aexrt_b200_attention_packed(None, *packed) == 0 and "null" in _native.last_error()
    assert lib.aexrt_b200_attention_status(None) == 0


def test_empty_calls_succeed_without_a_launch():
    lib = _native.load()
    for kw in (dict(q_tokens=0), dict(num_seqs=0)):
        assert lib.aexrt_b200_attention_packed(ctypes.byref(_desc(**kw)), None, None, None, None, None, None, None, None) == 1
        assert lib.aexrt_b200_attention_paged(ctypes.byref(_desc(**kw)), None, None, None, None, None, None, None, None, None,
                                              0, None) == 1


def _tables_args(**kw):
    a = dict(ctx=FAKE, new=FAKE, n=4, page=16, table=FAKE, columns=8, stride=8, free=FAKE, cap=10, state=FAKE, state_out=FAKE,
             cu=FAKE, kv=FAKE, slots=FAKE, slot_cap=32, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(n=16385), "requests"), (dict(page=0), "page_size"), (dict(page=12), "page_size"), (dict(page=2048), "page_size"),
    (dict(stride=7), "table_stride"), (dict(ctx=None), "null"), (dict(new=None), "null"), (dict(table=None), "null"),
    (dict(free=None), "null"), (dict(state=None), "null"), (dict(state_out=None), "null"), (dict(cu=None), "null"),
    (dict(kv=None), "null"), (dict(slots=None), "null"), (dict(slot_cap=(1 << 30) + 1), "2^30"),
])
def test_page_tables_refusals(kw, msg):
    assert _native.load().aexrt_b200_page_tables(*_tables_args(**kw)) == 0
    assert msg in _native.last_error()


def _append_args(**kw):
    a = dict(k=FAKE, v=FAKE, tokens=4, heads=2, dim=64, kts=128, khs=64, vts=128, vhs=64, slots=FAKE, kc=FAKE, vc=FAKE,
             pages=4, page=16, kps=2048, kcts=128, kchs=64, vps=2048, vcts=128, vchs=64, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dim=0), "head_dim"), (dict(dim=12), "head_dim"), (dict(heads=0), "kv_heads"), (dict(page=12), "page_size"),
    (dict(pages=1 << 27), "2^31"), (dict(kts=4), "multiples of 8"), (dict(vps=1 << 39), "out of range"),
    (dict(k=None), "null"), (dict(slots=None), "null"), (dict(vc=None), "null"), (dict(v=ctypes.c_void_p(4104)), "aligned"),
    (dict(kc=ctypes.c_void_p(4104)), "aligned"), (dict(tokens=(1 << 30) + 1), "2^30"),
])
def test_kv_append_refusals(kw, msg):
    assert _native.load().aexrt_b200_kv_append(*_append_args(**kw)) == 0
    assert msg in _native.last_error()
    assert _native.load().aexrt_b200_kv_append(*_append_args(tokens=0, k=None)) == 1


def test_tensor_wrappers_refuse_bad_shapes():
    h = torch.float16
    q, k = torch.zeros(4, 8, 64, dtype=h), torch.zeros(4, 2, 64, dtype=h)
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_packed(q, k, k, cu, cu)
    with pytest.raises(ValueError, match="3 dimensions"):
        ops.attention_packed(q[0], k, k, cu, cu)
    with pytest.raises(ValueError, match="contiguous"):
        ops.attention_packed(q.transpose(1, 2), k, k, cu, cu)
    with pytest.raises(ValueError, match="out must"):
        ops.attention_packed(q, k, k, cu, cu, out=q[:2])
    with pytest.raises(ValueError, match="lse"):
        ops.attention_packed(q, k, k, cu, cu, lse=torch.zeros(4, 8, dtype=torch.float64))
    with pytest.raises(ValueError, match="4 dimensions"):
        ops.attention_paged(q, k, k, cu[None], cu, cu, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.page_tables(cu, cu, torch.zeros(2, 3, dtype=torch.int32), cu, cu, 16, max_tokens=4)
    with pytest.raises(ValueError, match="max_q"):
        ops.attention_paged(q, torch.zeros(2, 16, 2, 64, dtype=h), torch.zeros(2, 16, 2, 64, dtype=h), cu[None], cu, cu[:1], -1)
    with pytest.raises(ValueError, match="max_tokens"):
        ops.page_tables(cu, cu, torch.zeros(2, 3, dtype=torch.int32), cu, cu, 16)
    with pytest.raises(ValueError, match="one type"):
        ops.kv_append(k, k, cu, torch.zeros(2, 16, 2, 64), torch.zeros(2, 16, 2, 64))
    with pytest.raises(ValueError, match="agree"):
        ops.kv_append(k, k, cu, torch.zeros(2, 16, 3, 64, dtype=h), torch.zeros(2, 16, 3, 64, dtype=h))


@pytest.mark.parametrize("lq,lk,causal", [(5, 5, True), (7, 3, True), (3, 9, True), (4, 6, False), (3, 0, True)])
def test_the_two_oracles_agree(lq, lk, causal):
    g = torch.Generator().manual_seed(lq * 10 + lk)
    q = torch.randn(lq, 4, 16, generator=g).to(torch.float16)
    k, v = (torch.randn(lk, 2, 16, generator=g).to(torch.float16) for _ in range(2))
    a, b = oracle.attend(q, k, v, 0.25, causal), oracle.attend_block(q, k, v, 0.25, causal)
    for x, y in zip(a[:2], b[:2]):
        assert torch.allclose(x, y, rtol=1e-12, atol=1e-15)
    assert bool((a[2] <= b[2] + 1e-15).all()) and torch.allclose(a[3], b[3], rtol=1e-12)
    if causal and lq > lk:
        assert bool((a[0][:lq - lk] == 0).all()) and bool(torch.isinf(a[1][:lq - lk]).all())


def test_oracle_row_ignores_what_it_does_not_see():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(6, 2, 8, generator=g).to(torch.float16) for _ in range(3))
    want = oracle.attend(q, k, v, 0.3, True)[0]
    k[4:], v[4:] = math.nan, math.inf
    got = oracle.attend(q, k, v, 0.3, True)[0]
    assert torch.equal(got[:4], want[:4]) and bool(torch.isnan(got[4:]).all())
