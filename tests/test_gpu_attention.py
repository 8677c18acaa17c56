"""Attention over token sequences on the GPU against the definition in 64 bits: packed prompts, the paged cache with one, a
few and many new tokens, its tables and writes, and all of them as a serving step runs them."""
import ctypes
import math
import random

import pytest
import torch

from aexrt_b200 import _native, ops
from tests import _attention as oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def rand(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def expect(q, ks, vs, q_lens, scale, causal, block=True):
    """Oracle over sequences: ks, vs lists of [lk, hk, d]."""
    parts, a = [], 0
    f = oracle.attend_block if block else oracle.attend
    for lq, k, v in zip(q_lens, ks, vs):
        parts.append(f(q[a:a + lq], k, v, scale, causal))
        a += lq
    return [torch.cat(x) for x in zip(*parts)]


def split(t, lens):
    return list(torch.split(t[:sum(lens)], lens))


def no_status():
    assert ops.attention_status() == 0


# ---------------------------------------------------------------- packed prompts
PACKED = [
    # q lengths, k lengths (None: the same), q heads, kv heads, head size
    ([1], None, 1, 1, 8),
    ([1, 1, 1], None, 4, 4, 64),
    ([2], [1], 2, 1, 64),
    ([17, 0, 1, 64, 3], None, 8, 8, 64),
    ([127], None, 2, 2, 128),
    ([128], None, 2, 1, 128),
    ([129], None, 4, 1, 128),
    ([255, 256, 257], None, 2, 2, 64),
    ([300, 5, 0, 513], None, 8, 2, 128),
    ([40, 200], None, 6, 2, 80),
    ([33, 190], None, 5, 1, 104),
    ([100], None, 7, 1, 40),
    ([70, 300], None, 3, 3, 16),
    ([50, 129], None, 9, 3, 24),
    ([64, 130], [0, 300], 4, 2, 128),
    ([130, 7, 400], [5, 600, 129], 4, 1, 64),
    ([20], None, 128, 1, 64),
    ([37], None, 100, 1, 72),
    ([1025], None, 2, 2, 96),
    ([700, 900], None, 4, 4, 56),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed_matches_the_definition(case, causal, dtype):
    q_lens, k_lens, hq, hk, d = PACKED[case]
    k_lens = k_lens or q_lens
    g = generator(case)
    q = rand(g, sum(q_lens), hq, d, dtype=dtype, std=2.0)
    k, v = rand(g, sum(k_lens), hk, d, dtype=dtype), rand(g, sum(k_lens), hk, d, dtype=dtype)
    scale = d ** -0.5
    out, lse = ops.attention_packed(q, k, v, ints(oracle.sums(q_lens)), ints(oracle.sums(k_lens)), causal=causal,
                                    return_lse=True)
    no_status()
    want = expect(q, split(k, k_lens), split(v, k_lens), q_lens, scale, causal)
    oracle.check(out, lse, *want)


@pytest.mark.parametrize("seed", range(12))
def test_packed_random_shapes(seed):
    rng = random.Random(seed)
    hk = rng.choice([1, 2, 3, 4])
    grp = rng.choice([1, 2, 3, 4, 6, 8, 16])
    d = 8 * rng.randint(1, 16)
    n = rng.randint(1, 9)
    q_lens = [rng.choice([0, 1, 2, 31, 128, rng.randint(1, 700)]) for _ in range(n)]
    k_lens = q_lens if rng.random() < 0.5 else [rng.choice([0, 1, 128, 256, rng.randint(1, 900)]) for _ in range(n)]
    dtype, causal = rng.choice([F16, BF16]), rng.random() < 0.6
    g = generator(1000 + seed)
    q = rand(g, sum(q_lens), hk * grp, d, dtype=dtype, std=rng.choice([0.1, 1.0, 8.0]))
    k, v = rand(g, sum(k_lens), hk, d, dtype=dtype), rand(g, sum(k_lens), hk, d, dtype=dtype)
    scale = rng.choice([d ** -0.5, 0.0, 1.0])
    out, lse = ops.attention_packed(q, k, v, ints(oracle.sums(q_lens)), ints(oracle.sums(k_lens)), causal=causal,
                                    scale=scale, return_lse=True)
    no_status()
    oracle.check(out, lse, *expect(q, split(k, k_lens), split(v, k_lens), q_lens, scale, causal))


def test_packed_reads_strided_slices_and_writes_strided_rows():
    """q, k and v as slices of one projection, out as columns of a wider buffer, heads before tokens."""
    g = generator(5)
    lens, hq, hk, d = [200, 91], 8, 2, 64
    t = sum(lens)
    qkv = rand(g, t, (hq + 2 * hk) * d + 8, dtype=BF16)
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    v = qkv[:, (hq + hk) * d:(hq + 2 * hk) * d].unflatten(1, (hk, d))
    cu = ints(oracle.sums(lens))
    want = expect(q, split(k, lens), split(v, lens), lens, d ** -0.5, True)
    wide = torch.full((t, hq, d + 24), 7.0, dtype=BF16, device="cuda")
    out, lse = ops.attention_packed(q, k, v, cu, cu, out=wide[:, :, 8:8 + d], return_lse=True)
    oracle.check(out, lse, *want)
    assert bool((wide[:, :, :8] == 7).all()) and bool((wide[:, :, 8 + d:] == 7).all())
    heads_first = torch.empty(hq, t, d, dtype=BF16, device="cuda")
    out = ops.attention_packed(q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1),
                               v, cu, cu, out=heads_first.transpose(0, 1))
    oracle.check(out, None, *want)


def test_packed_leaves_rows_behind_the_last_sequence():
    g = generator(6)
    q, k, v = (rand(g, 300, 4, 64, dtype=F16) for _ in range(3))
    out = torch.full_like(q, 3.0)
    lse = torch.full((300, 4), 5.0, device="cuda")
    ops.attention_packed(q, k, v, ints([0, 100, 170]), ints([0, 100, 170]), out=out, lse=lse)
    assert bool((out[170:] == 3).all()) and bool((lse[170:] == 5).all())
    # rows before the first sequence too
    out.fill_(3.0)
    ops.attention_packed(q, k, v, ints([40, 100, 170]), ints([0, 100, 170]), out=out)
    assert bool((out[:40] == 3).all()) and bool((out[170:] == 3).all())
    oracle.check(out[40:170], None, *expect(q[40:], [k[:100], k[100:170]], [v[:100], v[100:170]], [60, 70], 0.125, True))


@pytest.mark.parametrize("cu_q,cu_k", [([0, 50, 1000], [0, 50, 1000]), ([0, 90, 40], [0, 90, 40]), ([-5, 20, 100], [-9, 20, 100]),
                                       ([0, 100], [2 ** 31 - 1, -2 ** 31])])
def test_packed_offsets_outside_the_tensors_are_cut(cu_q, cu_k):
    """Whatever the offsets say, rows outside the tensors are neither read nor written."""
    g = generator(7)
    q, k, v = (rand(g, 100, 2, 64, dtype=F16) for _ in range(3))
    out = ops.attention_packed(q, k, v, ints(cu_q), ints(cu_k))
    no_status()
    cut = [min(max(x, 0), 100) for x in cu_q]
    cutk = [min(max(x, 0), 100) for x in cu_k]
    for s in range(len(cut) - 1):
        lq, lk = cut[s + 1] - cut[s], max(0, cutk[s + 1] - cutk[s])
        if lq > 0:
            want = oracle.attend_block(q[cut[s]:cut[s + 1]], k[cutk[s]:cutk[s] + lk], v[cutk[s]:cutk[s] + lk], 0.125, True)
            oracle.check(out[cut[s]:cut[s + 1]], None, *want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_packed_masked_values_reach_nothing(bad, dtype):
    """A neighbour sequence full of NaN or infinities, and such keys in a row's own future."""
    g = generator(8)
    lens, d = [150, 77, 300], 64
    q, k, v = (rand(g, sum(lens), 4, d, dtype=dtype) for _ in range(3))
    cu = ints(oracle.sums(lens))
    clean = ops.attention_packed(q, k, v, cu, cu)
    k[150:227], v[150:227] = bad, bad
    out = ops.attention_packed(q, k, v, cu, cu)
    assert torch.equal(out[:150], clean[:150]) and torch.equal(out[227:], clean[227:])
    # the last keys of the third sequence: rows before them see nothing of it
    k, v = (rand(g, sum(lens), 4, d, dtype=dtype) for _ in range(2))
    clean = ops.attention_packed(q, k, v, cu, cu)
    first = 227 + 290
    v[first, 1, 3] = bad
    v[first + 2, 1, 3] = -bad
    v[first + 4, 2] = bad
    out, lse = ops.attention_packed(q, k, v, cu, cu, return_lse=True)
    assert torch.equal(out[:first], clean[:first])
    oracle.check(out, lse, *expect(q, split(k, lens), split(v, lens), lens, d ** -0.5, True, block=False))
    k[first + 1, 0] = bad
    out = ops.attention_packed(q, k, v, cu, cu)
    assert torch.equal(out[:first], clean[:first])
    assert bool(torch.isnan(out[first + 1:, 0]).all()) or bad == -math.inf or bad == math.inf


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_packed_visible_non_finite_values_come_through(bad):
    g = generator(9)
    q, k, v = (rand(g, 400, 2, 64, dtype=BF16) for _ in range(3))
    v[3, 0, 5] = bad
    cu = ints([0, 400])
    for causal in (True, False):
        out, lse = ops.attention_packed(q, k, v, cu, cu, causal=causal, return_lse=True)
        want = expect(q, [k], [v], [400], 0.125, causal, block=False)
        oracle.check(out, lse, *want)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_non_finite_score_makes_its_rows_nan(bad, dtype):
    """A visible key with NaN, or whose score overflows to +inf, wherever in a tile it lies; other rows are left alone."""
    g = generator(32)
    n, d = 300, 64
    q = rand(g, n, 1, d, dtype=dtype).abs() + 0.1  # every score with an infinite key is +inf
    k, v = (rand(g, n, 1, d, dtype=dtype) for _ in range(2))
    cu, page = ints([0, n]), 16
    clean = ops.attention_packed(q, k, v, cu, cu)
    table = torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None]
    for key in list(range(0, n, 7)) + [0, 31, 32, 127, 128, n - 1]:
        kk = k.clone()
        kk[key] = bad
        out, lse = ops.attention_packed(q, kk, v, cu, cu, return_lse=True)
        assert torch.equal(out[:key], clean[:key])
        assert bool(torch.isnan(out[key:]).all()) and bool(torch.isnan(lse[key:]).all())
        kc, vc = (torch.zeros(table.shape[1], page, 1, d, dtype=dtype, device="cuda") for _ in range(2))
        ops.kv_append(kk, v, torch.arange(n, dtype=torch.int32, device="cuda"), kc, vc)
        out = ops.attention_paged(q[-3:], kc, vc, table, ints([0, 3]), ints([n]), 3)
        assert bool(torch.isnan(out[-1]).all()) and (key > n - 3 or bool(torch.isnan(out).all()))


def test_packed_large_and_rising_scores():
    """Scores that grow along the keys, so that the running maximum keeps moving, and scores far below it."""
    for dtype in (F16, BF16):
        n, d = 900, 64
        g = generator(10)
        q = torch.full((n, 2, d), 1.0, dtype=dtype, device="cuda")
        ramp = torch.linspace(-60, 60, n, device="cuda")[:, None, None].expand(n, 2, d) / d
        k = (ramp + 0.02 * torch.randn(n, 2, d, generator=g, device="cuda")).to(dtype)
        k[:, 1] = k[:, 1].flip(0)
        v = rand(g, n, 2, d, dtype=dtype)
        cu = ints([0, n])
        for causal in (True, False):
            out, lse = ops.attention_packed(q, k, v, cu, cu, causal=causal, scale=2.0, return_lse=True)
            oracle.check(out, lse, *expect(q, [k], [v], [n], 2.0, causal))


@pytest.mark.parametrize("dtype,size", [(F16, 60000.0), (BF16, 1e18), (F16, 300.0)])
def test_scores_of_any_finite_size(dtype, size):
    """Equal huge scores give the mean, and one that is larger still takes all: packed, one token and a chunk over a cache."""
    n, d, page = 300, 64, 16
    g = generator(37)
    q = torch.full((n, 2, d), size, dtype=dtype, device="cuda")
    k = torch.full((n, 2, d), size, dtype=dtype, device="cuda")
    k[40:, 1] = -k[40:, 1]
    v = rand(g, n, 2, d, dtype=dtype)
    cu = ints([0, n])
    u = oracle.half_step(dtype)
    kc, vc = (torch.zeros(-(-n // page), page, 2, d, dtype=dtype, device="cuda") for _ in range(2))
    ops.kv_append(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), kc, vc)
    table = torch.arange(kc.shape[0], dtype=torch.int32, device="cuda")[None]
    mean = v.double().cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None, None]
    mean[40:, 1] = mean[39, 1]  # head 1: the keys from 40 on score far below
    # probabilities are 1 before normalising, so exact in 16 bits: the output's rounding and fp32 sums of n terms
    tol = u * mean.abs() + n * 2.0 ** -22 * v.double().abs().max() + 2.0 ** -25
    for out, rows in ((ops.attention_packed(q, k, v, cu, cu), slice(0, n)),
                      (ops.attention_paged(q[-1:], kc, vc, table, ints([0, 1]), ints([n]), 1), slice(n - 1, n)),
                      (ops.attention_paged(q[-80:], kc, vc, table, ints([0, 80]), ints([n]), 80), slice(n - 80, n))):
        assert bool(((out.double() - mean[rows]).abs() <= tol[rows]).all())


def test_packed_large_values_keep_their_range():
    """fp16's largest values: the weighted sum stays within them."""
    g = generator(11)
    q, k = (rand(g, 260, 2, 64, dtype=F16) for _ in range(2))
    v = torch.full((260, 2, 64), 65504.0, dtype=F16, device="cuda")
    cu = ints([0, 260])
    out = ops.attention_packed(q, k, v, cu, cu)
    assert bool(torch.isfinite(out).all())
    oracle.check(out, None, *expect(q, [k], [v], [260], 0.125, True))


def test_packed_many_short_sequences():
    rng = random.Random(3)
    lens = [rng.choice([0, 1, 1, 2, 5, 9, 40]) for _ in range(500)]
    g = generator(12)
    q, k, v = (rand(g, sum(lens) + 3, 2, 32, dtype=F16) for _ in range(3))
    cu = ints(oracle.sums(lens))
    out, lse = ops.attention_packed(q, k, v, cu, cu, return_lse=True)
    no_status()
    want = expect(q, split(k, lens), split(v, lens), lens, 32 ** -0.5, True)
    oracle.check(out[:sum(lens)], lse[:sum(lens)], *want)


@pytest.mark.parametrize("n", [100, 128, 129, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_every_item_is_taken_once(n, causal):
    """Many sequences of very different lengths: the order of the work (by keys, or by sequence when there are many) leaves
    nothing out; rows nobody writes would keep the sentinel."""
    rng = random.Random(n)
    q_lens = [rng.choice([0, 1, 3, 130, 257, rng.randint(1, 500)]) for _ in range(n)]
    k_lens = [rng.choice([x, x, 0, rng.randint(0, 700)]) for x in q_lens]
    g = generator(n)
    q = rand(g, sum(q_lens), 4, 64, dtype=BF16)
    k, v = (rand(g, sum(k_lens), 2, 64, dtype=BF16) for _ in range(2))
    out = torch.full_like(q, 1000.0)
    out, lse = ops.attention_packed(q, k, v, ints(oracle.sums(q_lens)), ints(oracle.sums(k_lens)), causal=causal, out=out,
                                    return_lse=True)
    no_status()
    oracle.check(out, lse, *expect(q, split(k, k_lens), split(v, k_lens), q_lens, 0.125, causal))


def test_packed_long_sequence():
    g = generator(13)
    lens = [8200, 3, 1500]
    q = rand(g, sum(lens), 2, 128, dtype=BF16, std=2.0)
    k, v = (rand(g, sum(lens), 1, 128, dtype=BF16) for _ in range(2))
    cu = ints(oracle.sums(lens))
    out, lse = ops.attention_packed(q, k, v, cu, cu, return_lse=True)
    no_status()
    oracle.check(out, lse, *expect(q, split(k, lens), split(v, lens), lens, 128 ** -0.5, True))


# ---------------------------------------------------------------- the paged cache
def cache_of(gen, kv_lens, page, hk, d, dtype, spare=3, layout="tokens", poison=None):
    """A cache that holds kv_lens keys in shuffled pages: (k_cache, v_cache, table, ks, vs)."""
    need = [-(-n // page) for n in kv_lens]
    total = sum(need) + spare
    shape = (total, page, hk, d) if layout == "tokens" else (total, hk, page, d)
    kc, vc = (rand(gen, *shape, dtype=dtype) for _ in range(2))
    if layout != "tokens":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(len(kv_lens))).tolist()
    table = torch.full((len(kv_lens), max(need, default=0) + 2), 10 ** 9, dtype=torch.int32)
    at, used = 0, torch.zeros(total, page, dtype=torch.bool)
    for i, n in enumerate(need):
        ids = order[at:at + n]
        at += n
        table[i, :n] = torch.tensor(ids, dtype=torch.int32)
        for c, p in enumerate(ids):
            used[p, :max(0, min(page, kv_lens[i] - c * page))] = True
    if poison is not None:
        free = ~used.cuda()
        kc[free], vc[free] = poison, poison
    table = table.cuda()
    ks, vs = [], []
    for i, n in enumerate(kv_lens):
        ids = table[i, :need[i]].long()
        ks.append(kc[ids].flatten(0, 1)[:n])
        vs.append(vc[ids].flatten(0, 1)[:n])
    return kc, vc, table, ks, vs


PAGED = [
    # new tokens, kv lengths, q heads, kv heads, head size, page size
    ([1], [1], 1, 1, 8, 8),
    ([1], [1000], 32, 8, 128, 16),
    ([1, 1, 1, 1], [0, 1, 16, 17], 8, 2, 64, 16),
    ([1] * 5, [700, 3, 64, 65, 2049], 8, 1, 128, 32),
    ([1] * 3, [333, 127, 129], 4, 4, 96, 64),
    ([1, 1], [5000, 40], 16, 1, 128, 16),
    ([1], [900], 64, 2, 64, 128),
    ([1, 1], [800, 90], 7, 1, 72, 16),
    ([1, 0, 1], [130, 5, 260], 40, 8, 128, 256),
    ([5, 5, 5], [5, 700, 133], 4, 4, 96, 32),
    ([3, 0, 2, 1], [1000, 4, 2, 66], 8, 2, 64, 16),
    ([8, 2], [8, 515], 16, 2, 128, 16),
    ([4], [600], 12, 4, 40, 8),
    ([9, 16], [300, 16], 4, 4, 128, 64),
    ([64, 30], [64, 1000], 8, 2, 128, 16),
    ([200, 1], [900, 900], 8, 2, 64, 32),
    ([257], [2000], 2, 2, 128, 128),
    ([130, 70], [100, 70], 4, 1, 88, 16),
    ([300, 20], [1300, 20], 12, 4, 128, 1024),
    ([17], [40], 3, 1, 120, 8),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged_matches_the_definition(case, causal, dtype):
    new, kv, hq, hk, d, page = PAGED[case]
    g = generator(50 + case)
    layout = "tokens" if case % 2 == 0 else "heads"
    kc, vc, table, ks, vs = cache_of(g, kv, page, hk, d, dtype, layout=layout, poison=math.nan if case % 3 else math.inf)
    q = rand(g, sum(new), hq, d, dtype=dtype, std=2.0)
    out, lse = ops.attention_paged(q, kc, vc, table, ints(oracle.sums(new)), ints(kv), max(new), causal=causal, return_lse=True)
    no_status()
    oracle.check(out, lse, *expect(q, ks, vs, new, d ** -0.5, causal))


@pytest.mark.parametrize("seed", range(14))
def test_paged_random_shapes(seed):
    rng = random.Random(100 + seed)
    hk, grp, d = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16, 20]), 8 * rng.randint(1, 16)
    n = rng.randint(1, 20)
    most = rng.choice([1, 1, 3, 8, 40, 150])
    new = [rng.randint(0, most) for _ in range(n)]
    kv = [x + rng.choice([0, 0, 1, 63, 64, rng.randint(0, 900), rng.randint(0, 4000)]) for x in new]
    page, dtype, causal = rng.choice([8, 16, 32, 64, 128, 512]), rng.choice([F16, BF16]), rng.random() < 0.7
    g = generator(2000 + seed)
    kc, vc, table, ks, vs = cache_of(g, kv, page, hk, d, dtype, layout=rng.choice(["tokens", "heads"]), poison=math.nan)
    q = rand(g, sum(new) + 2, hk * grp, d, dtype=dtype, std=rng.choice([0.3, 3.0]))
    out = torch.full_like(q, 9.0)
    out, lse = ops.attention_paged(q, kc, vc, table, ints(oracle.sums(new)), ints(kv), most, causal=causal, out=out,
                                   return_lse=True)
    no_status()
    t = sum(new)
    assert bool((out[t:] == 9).all())
    oracle.check(out[:t], lse[:t], *expect(q, ks, vs, new, d ** -0.5, causal))


@pytest.mark.parametrize("new", [1, 3, 70])
def test_paged_long_context(new):
    g = generator(14)
    kv = [33000, 11, 9000]
    kc, vc, table, ks, vs = cache_of(g, kv, 16, 2, 128, BF16)
    q = rand(g, 3 * new, 8, 128, dtype=BF16, std=2.0)
    out, lse = ops.attention_paged(q, kc, vc, table, ints([0, new, 2 * new, 3 * new]), ints(kv), new, return_lse=True)
    no_status()
    oracle.check(out, lse, *expect(q, ks, vs, [new] * 3, 128 ** -0.5, True))


@pytest.mark.parametrize("new", [1, 80])
def test_paged_cache_offsets_beyond_32_bits(new):
    """Pages whose element offsets exceed 2^32: a small cache at the end of a wide buffer."""
    page, hk, d, pages = 16, 1, 64, 6
    buffer = torch.empty((1 << 30) + (1 << 27), dtype=torch.int64, device="cuda")  # 9 GB
    flat = buffer.view(BF16)
    stride = (flat.numel() - page * hk * d) // (pages - 1) // 8 * 8
    assert stride * (pages - 1) > 2 ** 32
    kc = torch.as_strided(flat, (pages, page, hk, d), (stride, hk * d, d, 1))
    vc = torch.as_strided(flat[page * hk * d:], (pages, page, hk, d), (stride - 8 * page * hk * d, hk * d, d, 1))
    g = generator(15)
    for p in range(pages):
        kc[p] = rand(g, page, hk, d, dtype=BF16)
        vc[p] = rand(g, page, hk, d, dtype=BF16)
    ids = [5, 0, 4, 3, 1]
    n = 75 if new == 1 else 80
    table = ints([ids])
    k, v = (c[torch.tensor(ids, device="cuda")].flatten(0, 1)[:n] for c in (kc, vc))
    q = rand(g, new, 4, d, dtype=BF16)
    out = ops.attention_paged(q, kc, vc, table, ints([0, new]), ints([n]), new)
    no_status()
    oracle.check(out, None, *expect(q, [k], [v], [new], d ** -0.5, True))
    # and the write to such a page
    row = rand(g, 2, hk, d, dtype=BF16)
    ops.kv_append(row, -row, ints([5 * page + 3, 4 * page + 15]), kc, vc)
    assert torch.equal(kc[5, 3], row[0]) and torch.equal(vc[4, 15], -row[1])


@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_paged_masked_values_reach_nothing(new, bad):
    """Non-finite keys among the new tokens reach only the rows that see them."""
    g = generator(16)
    kv, d = [300, 128 + new], 64
    kc, vc, table, ks, vs = cache_of(g, kv, 16, 2, d, BF16)
    q = rand(g, 2 * new, 4, d, dtype=BF16)
    cu = ints([0, new, 2 * new])
    clean = ops.attention_paged(q, kc, vc, table, cu, ints(kv), new)
    pages, rows = table[:, :], kv
    last = [(int(pages[i, (n - 1) // 16]), (n - 1) % 16) for i, n in enumerate(rows)]
    for i, (p, r) in enumerate(last):
        vc[p, r, i] = bad
        vs[i][-1, i] = bad
    out, lse = ops.attention_paged(q, kc, vc, table, cu, ints(kv), new, return_lse=True)
    assert torch.equal(out[:new - 1], clean[:new - 1]) and torch.equal(out[new:2 * new - 1], clean[new:2 * new - 1])
    oracle.check(out, lse, *expect(q, ks, vs, [new] * 2, d ** -0.5, True, block=False))


@pytest.mark.parametrize("new", [1, 100])
def test_paged_bad_table_entries_read_as_zeros(new):
    """Entries outside the cache: rows of zeros and the status bit, no access outside."""
    g = generator(17)
    kc, vc, table, ks, vs = cache_of(g, [100], 16, 2, 64, F16)
    q = rand(g, new, 4, 64, dtype=F16)
    for bad in (-1, 2 ** 31 - 1, -2 ** 31, kc.shape[0]):
        table[0, 2] = bad
        ks[0][32:48], vs[0][32:48] = 0, 0
        out, lse = ops.attention_paged(q, kc, vc, table, ints([0, new]), ints([100]), new, return_lse=True)
        assert ops.attention_status() == ops.ATTENTION_BAD_PAGE
        oracle.check(out, lse, *expect(q, ks, vs, [new], 0.125, True))
    no_status()


def test_paged_lengths_beyond_the_table_are_cut():
    g = generator(18)
    kc, vc, table, ks, vs = cache_of(g, [64, 64], 16, 2, 64, F16)
    table = table[:, :4].contiguous()
    q = rand(g, 2, 4, 64, dtype=F16)
    out = ops.attention_paged(q, kc, vc, table, ints([0, 1, 2]), ints([2 ** 31 - 1, -7]), 1)
    no_status()
    oracle.check(out[:1], None, *expect(q, ks[:1], vs[:1], [1], 0.125, True))
    assert bool((out[1] == 0).all())


def test_paged_tokens_beyond_max_q_are_left_out():
    g = generator(19)
    kc, vc, table, ks, vs = cache_of(g, [64, 64], 16, 2, 64, F16)
    q = rand(g, 9, 4, 64, dtype=F16)
    out = torch.full_like(q, 4.0)
    ops.attention_paged(q, kc, vc, table, ints([0, 6, 9]), ints([64, 64]), 3, out=out)
    want = expect(q, ks, vs, [6, 3], 0.125, True)
    oracle.check(out[:3], None, *[w[:3] for w in want])
    oracle.check(out[6:], None, *[w[6:] for w in want])
    assert bool((out[3:6] == 4).all())


def test_paged_refuses_a_small_workspace():
    g = generator(20)
    kc, vc, table, _, _ = cache_of(g, [64], 16, 2, 64, F16)
    q = rand(g, 1, 4, 64, dtype=F16)
    ws = ops.attention_paged_workspace(q, kc, 1, 1)
    if ws.numel():
        with pytest.raises(_native.AexrtError, match="workspace"):
            ops.attention_paged(q, kc, vc, table, ints([0, 1]), ints([64]), 1, workspace=ws[:-16])


@pytest.mark.parametrize("new", [1, 5, 200])
def test_paged_repeats_bit_for_bit(new):
    g = generator(21)
    kc, vc, table, _, _ = cache_of(g, [3000 + new, 70 + new, 511 + new], 16, 4, 128, BF16)
    q = rand(g, 3 * new, 16, 128, dtype=BF16, std=2.0)
    args = (q, kc, vc, table, ints([0, new, 2 * new, 3 * new]), ints([3000 + new, 70 + new, 511 + new]), new)
    first = ops.attention_paged(*args, return_lse=True)
    for _ in range(5):
        again = ops.attention_paged(*args, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---------------------------------------------------------------- tables and writes
def run_tables(ctx, new, columns, page, free, top, capacity, seed=0, in_place=False, stride=None):
    rng = random.Random(seed)
    table = [[rng.randrange(1000, 2000) if c < min(columns, -(-max(0, x) // page)) else 77 for c in range(columns)] for x in ctx]
    want = oracle.tables(ctx, new, table, free, top, page, capacity)
    base = torch.full((len(ctx), stride or columns), 55, dtype=torch.int32, device="cuda")
    base[:, :columns] = ints(table).reshape(len(ctx), columns)
    t = base[:, :columns]
    c, a, f, st = ints(ctx), ints(new), ints(free), ints([top, 123])
    kw = dict(kv_lens=c, free_state_out=st) if in_place else {}
    cu, kv, slots, state = ops.page_tables(c, a, t, f, st, page, max_tokens=capacity, **kw)
    got = [x.tolist() for x in (cu, kv, t, slots, state)]
    for name, x, y in zip(("cu_q", "kv_lens", "table", "slot_map", "state"), got, want):
        assert x == list(y), name
    if stride:
        assert bool((base[:, columns:] == 55).all())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", [
    ([0], [1], 4, 16, 10, 8), ([5, 0, 16, 31, 32], [1, 0, 1, 1, 1], 4, 16, 10, 8), ([100, 7], [300, 0], 30, 8, 100, 400),
    ([0] * 40, [3] * 40, 2, 1, 200, 120), ([64] * 3, [65, 1, 200], 3, 64, 100, 300), ([10, 20, 30], [50, 60, 70], 20, 16, 3, 200),
    ([10, 20], [50, 60], 20, 16, 0, 40), ([-4, 8], [-3, 9], 4, 16, 10, 20), ([], [], 4, 16, 10, 5), ([0, 0], [0, 0], 4, 16, 10, 0),
    ([1000], [5000], 1, 1024, 3, 6100),
])
def test_tables_match(case, in_place):
    ctx, new, columns, page, free, capacity = case
    run_tables(ctx, new, columns, page, list(range(500, 500 + free)), free, capacity, in_place=in_place)
    run_tables(ctx, new, columns, page, list(range(500, 500 + free)), free, capacity, in_place=in_place, stride=columns + 3)


@pytest.mark.parametrize("seed", range(8))
def test_tables_random(seed):
    rng = random.Random(seed)
    n = rng.choice([1, 3, 31, 32, 33, 1023, 1024, 1025, 2500])
    page = rng.choice([1, 8, 16, 64])
    ctx = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 300)]) for _ in range(n)]
    new = [rng.choice([0, 1, 1, page, rng.randint(0, 40)]) for _ in range(n)]
    columns = rng.choice([3, 20, 400])
    free = [rng.randrange(5000) for _ in range(rng.choice([0, 10, 20000]))]
    top = rng.choice([len(free), max(0, len(free) - 5), len(free) + 9, -3])
    run_tables(ctx, new, columns, page, free, top, rng.choice([sum(new), sum(new) + 13, max(0, sum(new) - 7)]), seed)


def test_tables_most_requests():
    rng = random.Random(4)
    n = 16384
    ctx, new = [rng.randint(0, 40) for _ in range(n)], [rng.randint(0, 2) for _ in range(n)]
    run_tables(ctx, new, 6, 8, list(range(20000)), 20000, sum(new))


def test_tables_lengths_near_the_limit():
    """Sums are cut below 2^31 instead of wrapping."""
    big = 2 ** 31 - 1
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    cu, kv, slots, state = ops.page_tables(ints([5, big, 0]), ints([big, big, big]), table, ints([1, 2, 3, 4, 5, 6, 7]), ints([7, 0]),
                                           16, max_tokens=40)
    assert cu.tolist() == [0, big - 5, big - 5, big]
    assert kv.tolist()[0] == big and kv.tolist()[1] == big
    # of the 7 free pages, 1 goes to the first request's second column and 2 to the third request
    assert state.tolist() == [7 - 3, 0] and table.tolist() == [[-1, 7], [-1, -1], [6, 5]]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,hk,d,page,layout", [(1, 1, 8, 8, "tokens"), (7, 2, 64, 16, "heads"), (300, 3, 72, 16, "tokens"),
                                                    (1000, 8, 128, 1, "tokens"), (129, 5, 40, 1024, "heads")])
def test_append_writes_its_rows_and_no_others(tokens, hk, d, page, layout, dtype):
    g = generator(tokens)
    pages = -(-tokens // page) + 3
    shape = (pages, page, hk, d) if layout == "tokens" else (pages, hk, page, d)
    kc, vc = (rand(g, *shape, dtype=dtype) for _ in range(2))
    if layout == "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
    if tokens > 5:
        slots[1], slots[3], slots[4] = -1, pages * page, 2 ** 31 - 1
    wide = rand(g, tokens, 2 * hk * d + 8, dtype=dtype)
    k, v = wide[:, :hk * d].unflatten(1, (hk, d)), wide[:, hk * d:2 * hk * d].unflatten(1, (hk, d))
    want_k, want_v = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = k[t], v[t]
    ops.kv_append(k, v, slots, kc, vc)
    assert torch.equal(kc.view(torch.int16), want_k.view(torch.int16)) and torch.equal(vc.view(torch.int16), want_v.view(torch.int16))


# ---------------------------------------------------------------- together
def serve(steps, hq, hk, d, page, dtype, capture):
    """Requests fed in chunks through tables, append and paged attention; every step against packed attention's oracle."""
    n = len(steps[0])
    g = generator(77)
    pages, columns, most = 400, 64, max(sum(s) for s in steps) + 5
    wide = max(max(s) for s in steps)
    kc, vc = (torch.full((pages, page, hk, d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((n, columns), -1, dtype=torch.int32, device="cuda")
    free, state = torch.randperm(pages, generator=g, device="cuda").to(torch.int32), ints([pages, 0])
    lens, new = ints([0] * n), ints([0] * n)
    q = torch.zeros(most, hq, d, dtype=dtype, device="cuda")
    k, v = (torch.zeros(most, hk, d, dtype=dtype, device="cuda") for _ in range(2))
    cu, slots, out = ints([0] * (n + 1)), ints([0] * most), torch.zeros_like(q)
    ws = ops.attention_paged_workspace(q, kc, n, wide)

    def step():
        ops.page_tables(lens, new, table, free, state, page, cu_q=cu, kv_lens=lens, slot_map=slots, free_state_out=state)
        ops.kv_append(k, v, slots, kc, vc)
        ops.attention_paged(q, kc, vc, table, cu, lens, wide, out=out, workspace=ws)

    graph = None
    if capture:
        step()  # a step of no tokens, before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    ks, vs = [torch.zeros(0, hk, d, dtype=dtype, device="cuda") for _ in range(n)], [torch.zeros(0, hk, d, dtype=dtype,
                                                                                                   device="cuda") for _ in range(n)]
    for s in steps:
        t = sum(s)
        new.copy_(ints(s))
        for x in (q, k, v):
            x[:t] = rand(g, t, *x.shape[1:], dtype=dtype)
            x[t:] = math.nan
        out.fill_(6.0)
        graph.replay() if capture else step()
        a = 0
        for i, c in enumerate(s):
            ks[i], vs[i] = torch.cat([ks[i], k[a:a + c]]), torch.cat([vs[i], v[a:a + c]])
            a += c
        assert state.tolist()[1] == 0
        assert lens.tolist() == [x.shape[0] for x in ks]
        oracle.check(out[:t], None, *expect(q, ks, vs, s, d ** -0.5, True))
        assert bool((out[t:] == 6).all())
    no_status()
    assert state.tolist()[0] == pages - sum(-(-x.shape[0] // page) for x in ks)


STEPS = [[100, 0, 37, 1], [1, 300, 1, 1], [1, 1, 1, 0], [64, 1, 130, 2], [1, 1, 1, 1], [0, 0, 0, 0], [1, 1, 0, 1]]


@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("hq,hk,d,page,dtype", [(8, 2, 128, 16, BF16), (4, 4, 64, 32, F16), (6, 1, 80, 8, BF16)])
def test_serving_steps(hq, hk, d, page, dtype, capture):
    serve(STEPS, hq, hk, d, page, dtype, capture)


@pytest.mark.parametrize("capture", [False, True])
def test_serving_single_tokens(capture):
    serve([[1, 1, 1]] + [[1, 0, 1], [1, 1, 1]] * 20, 8, 2, 64, 8, F16, capture)


def test_a_prompt_in_chunks_equals_the_prompt_at_once():
    """Both ways through the kernels, against one oracle's bound."""
    g = generator(30)
    n, hq, hk, d, page = 700, 8, 2, 128, 16
    q = rand(g, n, hq, d, dtype=BF16, std=2.0)
    k, v = (rand(g, n, hk, d, dtype=BF16) for _ in range(2))
    cu = ints([0, n])
    want = expect(q, [k], [v], [n], d ** -0.5, True)
    oracle.check(ops.attention_packed(q, k, v, cu, cu), None, *want)
    kc, vc = (torch.zeros(-(-n // page), page, hk, d, dtype=BF16, device="cuda") for _ in range(2))
    ops.kv_append(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), kc, vc)
    table = torch.arange(kc.shape[0], dtype=torch.int32, device="cuda")[None]
    for sizes in ([n], [256, 256, 188], [1] * 5 + [128, 3, n - 136]):
        at, parts = 0, []
        for c in sizes:
            at += c
            parts.append(ops.attention_paged(q[at - c:at], kc, vc, table, ints([0, c]), ints([at]), c))
        oracle.check(torch.cat(parts), None, *want)


def test_on_another_stream_and_side_by_side():
    g = generator(31)
    sets = []
    for i in range(3):
        kv = [900 + 40 * i, 60]
        kc, vc, table, ks, vs = cache_of(g, kv, 16, 2, 128, BF16)
        q = rand(g, 2, 8, 128, dtype=BF16)
        sets.append((q, kc, vc, table, ints([0, 1, 2]), ints(kv), expect(q, ks, vs, [1, 1], 128 ** -0.5, True)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [None] * len(sets)
    for _ in range(20):
        for i, (st, x) in enumerate(zip(streams, sets)):
            if i % 2:
                with torch.cuda.stream(st):
                    outs[i] = ops.attention_paged(*x[:6], 1, return_lse=True)
            else:
                outs[i] = ops.attention_paged(*x[:6], 1, return_lse=True, stream=st, out=x[0].new_empty(x[0].shape),
                                              workspace=ops.attention_paged_workspace(x[0], x[1], 2, 1))
                st.synchronize()
    torch.cuda.synchronize()
    for o, x in zip(outs, sets):
        oracle.check(o[0], o[1], *x[6])


@pytest.mark.parametrize("new", [1, 90])
def test_workspaces_allocated_for_another_stream_are_kept_until_it_is_done(new):
    """Calls on a side stream that allocate their own workspaces, with other work on the current stream that would reuse
    their memory at once."""
    g = generator(33)
    kv = [6000, 4000 + new]
    kc, vc, table, ks, vs = cache_of(g, kv, 16, 2, 128, BF16)
    q = rand(g, 2 * new, 8, 128, dtype=BF16)
    cu, lens = ints([0, new, 2 * new]), ints(kv)
    want = expect(q, ks, vs, [new] * 2, 128 ** -0.5, True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [torch.empty_like(q) for _ in range(8)]
    for o in outs:
        ops.attention_paged(q, kc, vc, table, cu, lens, new, out=o, stream=side)
        size = ops.attention_paged_workspace(q, kc, 2, new).numel()
        torch.full((max(1, size // 4),), math.nan, device="cuda")
    torch.cuda.synchronize()
    for o in outs:
        oracle.check(o, None, *want)


def test_two_captured_graphs_share_a_workspace_in_turn():
    g = generator(34)
    sets, graphs = [], []
    for kv in ([5000, 70], [33, 2100]):
        kc, vc, table, ks, vs = cache_of(g, kv, 16, 2, 64, F16)
        q = rand(g, 2, 8, 64, dtype=F16)
        sets.append([q, kc, vc, table, ints([0, 1, 2]), ints(kv), expect(q, ks, vs, [1, 1], 0.125, True), torch.empty_like(q)])
    ws = ops.attention_paged_workspace(sets[0][0], sets[0][1], 2, 1)
    for x in sets:
        ops.attention_paged(*x[:6], 1, out=x[7], workspace=ws)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.attention_paged(*x[:6], 1, out=x[7], workspace=ws)
    for _ in range(3):
        for gr, x in zip(graphs, sets):
            x[7].fill_(5.0)
            ws.random_()
            gr.replay()
            oracle.check(x[7], None, *x[6])


def test_broadcast_heads():
    """k and v of one head expanded over several (stride 0): the result of a real copy, or a refusal."""
    g = generator(35)
    q = rand(g, 70, 4, 64, dtype=F16)
    k, v = (rand(g, 70, 1, 64, dtype=F16) for _ in range(2))
    cu = ints([0, 70])
    want = ops.attention_packed(q, k.expand(70, 4, 64).contiguous(), v.expand(70, 4, 64).contiguous(), cu, cu)
    try:
        out = ops.attention_packed(q, k.expand(70, 4, 64), v.expand(70, 4, 64), cu, cu)
    except _native.AexrtError:
        return
    assert torch.equal(out, want)


@pytest.mark.parametrize("ctx,new,heads", [([30000], 70, (8, 2)), ([20000, 300, 9000], 65, (4, 4)), ([50, 12000, 700, 0, 3000], 33, (8, 2)),
                                           ([9000], 300, (4, 1)), ([15000] * 3, 80, (2, 1)), ([700], 65, (4, 4))])
def test_paged_split_over_long_contexts(ctx, new, heads):
    """Few items over long and ragged contexts: the key ranges of an item go to several blocks."""
    g = generator(36)
    hq, hk = heads
    kv = [c + new for c in ctx]
    kc, vc, table, ks, vs = cache_of(g, kv, 16, hk, 128, BF16, poison=math.nan)
    q = rand(g, new * len(ctx), hq, 128, dtype=BF16, std=2.0)
    cu = ints(oracle.sums([new] * len(ctx)))
    for causal in (True, False):
        out, lse = ops.attention_paged(q, kc, vc, table, cu, ints(kv), new, causal=causal, return_lse=True)
        no_status()
        oracle.check(out, lse, *expect(q, ks, vs, [new] * len(ctx), 128 ** -0.5, causal))


def test_with_programmatic_launches():
    """The library's programmatic launch flag: kernels that follow one another still see each other's writes."""
    lib = _native.load()
    assert lib.aexrt_b200_set_launch_flags(_native.LAUNCH_PROGRAMMATIC)
    try:
        serve(STEPS, 8, 2, 128, 16, BF16, True)
        serve(STEPS, 8, 2, 64, 16, F16, False)
    finally:
        lib.aexrt_b200_set_launch_flags(0)
