"""Arguments of the token-sequence wrappers that no call can take: refused with a ValueError before anything is launched (no GPU)."""
import ctypes

import pytest
import torch

from aexrt_b200 import _native, ops

H, I = torch.float16, torch.int32


def attention(**kw):
    a = dict(q=torch.zeros(4, 8, 64, dtype=H), k=torch.zeros(4, 2, 64, dtype=H), cu=torch.zeros(2, dtype=I), scale=None)
    a.update(kw)
    return ops.attention_packed(a["q"], a["k"], a["k"], a["cu"], a["cu"], scale=a["scale"])


def paged(**kw):
    a = dict(q=torch.zeros(4, 8, 64, dtype=H), kc=torch.zeros(2, 16, 2, 64, dtype=H), table=torch.zeros(1, 3, dtype=I),
             cu=torch.zeros(2, dtype=I), lens=torch.zeros(1, dtype=I), max_q=4, scale=None)
    a.update(kw)
    return ops.attention_paged(a["q"], a["kc"], a["kc"], a["table"], a["cu"], a["lens"], a["max_q"], scale=a["scale"],
                               workspace=torch.zeros(16, dtype=torch.uint8))


@pytest.mark.parametrize("call", [attention, paged])
def test_scales_and_sizes_that_fit_no_field(call):
    with pytest.raises(ValueError, match="out of range"):
        call(scale="wide")
    with pytest.raises(ValueError):  # heads of no elements: refused, not divided by
        call(q=torch.zeros(4, 8, 0, dtype=H), k=torch.zeros(4, 2, 0, dtype=H), kc=torch.zeros(2, 16, 2, 0, dtype=H))


def test_max_q_out_of_range():
    with pytest.raises(ValueError, match="out of range"):
        paged(max_q=1 << 32)
    for n, most in ((-1, 4), (1 << 32, 4), (1, 1 << 40)):
        with pytest.raises(ValueError, match="out of range"):
            ops.attention_paged_workspace(torch.zeros(4, 8, 64, dtype=H), torch.zeros(2, 16, 2, 64, dtype=H), n, most)


def test_vectors_without_a_dimension():
    scalar = torch.zeros((), dtype=I)
    with pytest.raises(ValueError, match="cu_q must have one dimension"):
        attention(cu=scalar)
    with pytest.raises(ValueError, match="kv_lens must have one dimension"):
        paged(lens=scalar)
    v, table = torch.zeros(2, dtype=I), torch.zeros(2, 3, dtype=I)
    for args, name in (((scalar, v, table, v, v), "ctx_lens"), ((v, v, table, scalar, v), "free_pages")):
        with pytest.raises(ValueError, match=f"{name} must have one dimension"):
            ops.page_tables(*args, 16, max_tokens=4)
    with pytest.raises(ValueError, match="slot_map must have one dimension"):
        ops.page_tables(v, v, table, v, v, 16, slot_map=scalar)


@pytest.mark.parametrize("page", [-16, (1 << 32) + 16])
def test_page_sizes_that_32_bits_would_cut(page):
    v = torch.zeros(2, dtype=I)
    with pytest.raises(ValueError, match="out of range"):
        ops.page_tables(v, v, torch.zeros(2, 3, dtype=I), v, v, page, max_tokens=4)


def test_append_of_more_rows_than_32_bits_count():
    n = (1 << 32) + 4
    k = torch.zeros(1, 2, 64, dtype=H).expand(n, 2, 64)
    cache = torch.zeros(2, 16, 2, 64, dtype=H)
    with pytest.raises(ValueError, match="out of range"):
        ops.kv_append(k, k, torch.zeros(4, dtype=I), cache, cache)


@pytest.mark.parametrize("scale,taken", [(1.01e38, False), (3.4e38, False), (1e38, True), (0.0, True), (1.401298464e-45, True)])
def test_scales_from_0_to_1e38(scale, taken):
    """Through the C entry points, on a description of no rows, which is taken without a launch."""
    d = _native.AexrtB200AttentionDesc(struct_size=ctypes.sizeof(_native.AexrtB200AttentionDesc), dtype=0, num_seqs=1, q_tokens=0,
                                       max_q=1, q_heads=2, kv_heads=1, head_dim=64, causal=1, scale=scale, kv_tokens=4, page_size=16,
                                       table_columns=1, table_stride=1, q_token_stride=128, q_head_stride=64, out_token_stride=128,
                                       out_head_stride=64, k_token_stride=64, k_head_stride=64, k_page_stride=1024,
                                       v_token_stride=64, v_head_stride=64, v_page_stride=1024)
    lib, at = _native.load(), ctypes.byref(d)
    for got in (lib.aexrt_b200_attention_packed(at, *[None] * 8), lib.aexrt_b200_attention_paged(at, *[None] * 9, 0, None)):
        assert got == int(taken)
        assert taken or "scale must be from 0 to 1e38" in _native.last_error()
    assert lib.aexrt_b200_attention_paged_workspace(at) == (0 if taken else 2 ** 64 - 1)
