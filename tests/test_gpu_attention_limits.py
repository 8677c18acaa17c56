"""Attention over token sequences at the borders of what its entry points accept: extreme scales and values, non-finite values that
meet, empty caches, sums near 2^31, other streams, long items."""
import math

import pytest
import torch

from aexrt_b200 import _native, ops
from tests import _attention as oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def paged_of(k, v, page=16):
    """One sequence's keys and values in a cache of their own: (k_cache, v_cache, block table)."""
    n, pages = k.shape[0], -(-k.shape[0] // page)
    kc, vc = (torch.zeros(pages, page, *k.shape[1:], dtype=k.dtype, device="cuda") for _ in range(2))
    kc.flatten(0, 1)[:n], vc.flatten(0, 1)[:n] = k, v
    return kc, vc, torch.arange(pages, dtype=torch.int32, device="cuda")[None]


def every_way(q, k, v, scale, causal, news):
    """The same attention through every kernel: yields (name, out, lse, rows) for the packed call over q and for the last `new` rows
    of q over a cache, for each of `news`."""
    n, cu = k.shape[0], ints([0, q.shape[0]])
    yield ("packed", *ops.attention_packed(q, k, v, cu, ints([0, n]), causal=causal, scale=scale, return_lse=True),
           slice(0, q.shape[0]))
    kc, vc, table = paged_of(k, v)
    for new in news:
        yield (f"paged {new}", *ops.attention_paged(q[-new:], kc, vc, table, ints([0, new]), ints([n]), new, causal=causal, scale=scale,
                                                    return_lse=True), slice(q.shape[0] - new, q.shape[0]))
    assert ops.attention_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,lens", [(1, [0, 0]), (1, [40, 0]), (5, [5, 300]), (90, [0, 90]), (70, [3000, 70])])
def test_an_empty_cache_reads_as_zeros(new, lens, dtype):
    """A cache of no pages: rows without keys give 0 and -inf, keys of table entries are zeros, and q's memory is no cache."""
    g = generator(20)
    hq, hk, d, page = 8, 2, 128, 16
    q = rand(g, 2 * new, hq, d, dtype=dtype)
    kc, vc = (torch.empty(0, page, hk, d, dtype=dtype, device="cuda") for _ in range(2))
    columns = -(-max(lens) // page)
    table = torch.zeros(2, columns, dtype=torch.int32, device="cuda")
    out, lse = ops.attention_paged(q, kc, vc, table, ints([0, new, 2 * new]), ints(lens), new, return_lse=True)
    assert ops.attention_status() == (ops.ATTENTION_BAD_PAGE if columns else 0)
    assert bool((out == 0).all())
    i = torch.arange(new, device="cuda")
    seen = torch.cat([(i + 1 + n - new).clamp(0, n) for n in lens])
    want = torch.log(seen.double())[:, None].expand(-1, hq)  # equal scores of 0
    empty = torch.isinf(want)
    assert torch.equal(lse[empty].double(), want[empty])
    assert bool(((lse - want)[~empty].abs() <= seen.max() * 2.0 ** -23 + 2.0 ** -20).all())


@pytest.mark.parametrize("capacity", [40, 200000])
def test_tables_of_nearly_2_31_new_pages(capacity):
    """Pages of one token and an empty stack: the last pages are written, none beyond them."""
    columns, top = 2 ** 30, 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 12 * 2 ** 30:
        pytest.skip("needs 12 GB")
    base = torch.full((2 * columns + 2,), 7, dtype=torch.int32, device="cuda")
    table = base[1:-1].view(2, columns)
    free = ints([5, 6, 9])
    cu, kv, slots, state = ops.page_tables(ints([0, 0]), ints([columns, columns]), table, free, ints([3, 0]), 1, max_tokens=capacity)
    assert cu.tolist() == [0, columns, top] and state.tolist() == [0, top - 3]
    assert table[0, :4].tolist() == [9, 6, 5, -1] and slots[:4].tolist() == [9, 6, 5, -1]
    assert int((base == -1).sum()) == top - 3 and int((slots == -1).sum()) == capacity - 3
    assert base[[0, -1, -2]].tolist() == [7, 7, 7]  # the sums end at 2^31 - 1: the last column is not taken


def test_tables_of_most_requests_in_place():
    """The largest shared memory in one cluster of blocks."""
    n = 16384
    g = torch.Generator().manual_seed(21)
    ctx, new = (torch.randint(0, high, (n,), generator=g).tolist() for high in (40, 3))
    table = [[1000 + c for c in range(6)] for _ in range(n)]
    want = oracle.tables(ctx, new, table, list(range(20000)), 20000, 8, sum(new))
    lens, t, state = ints(ctx), ints(table), ints([20000, 0])
    cu, kv, slots, state_out = ops.page_tables(lens, ints(new), t, ints(list(range(20000))), state, 8, max_tokens=sum(new), kv_lens=lens,
                                               free_state_out=state)
    for got, exp in zip((cu, kv, t, slots, state_out), want):
        assert got.tolist() == [list(x) if isinstance(x, (list, tuple)) else x for x in exp]


def test_sums_over_many_keys_keep_their_small_terms():
    """One value of 65504 and many of about 2^-10 with equal probabilities.  A tensor-core sum cuts each product to 2^-25 of what is
    summed so far, so that the small ones vanish beside the large one unless the keys are summed in stretches.  The bound: 2^14
    products a stretch, each cut by 2^-25 of the sum at most, 2^10 sums of 16 cut by 2^-23, some hundred stretches added in fp32, and
    the output's rounding.  Probabilities are 1, so they and their sum are exact."""
    d, small, page = 64, 0.99 * 2.0 ** -10, 1024

    def check(out, lse, n, what):
        v = torch.full((1,), small, dtype=F16, device="cuda").double()
        want = (65504 + (n - 1) * v) / n
        over = (out.double() - want).abs() / (want * (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -16 + 2.0 ** -11))
        assert bool((over <= 1).all()), f"{what}: {float(over.max()):.3g} of the bound"
        assert bool(((lse - math.log(n)).abs() <= 2.0 ** -19).all()), what

    n = 2 ** 18
    for rows in (1, 200):
        q = torch.zeros(rows, 1, d, dtype=F16, device="cuda")
        k = torch.zeros(n, 1, d, dtype=F16, device="cuda")
        v = torch.full((n, 1, d), small, dtype=F16, device="cuda")
        v[5] = 65504
        check(*ops.attention_packed(q, k, v, ints([0, rows]), ints([0, n]), causal=False, return_lse=True), n, ("packed", rows))
    # a cache of two pages, the second one repeated; as many sequences as there are blocks, so that no item is split
    kc = torch.zeros(2, page, 1, d, dtype=F16, device="cuda")
    vc = torch.full((2, page, 1, d), small, dtype=F16, device="cuda")
    vc[0, 5] = 65504
    for seqs, n, rows in ((300, 2 ** 20, 1), (300, 2 ** 20, 40), (300, 2 ** 17, 80)):
        table = torch.ones(seqs, n // page, dtype=torch.int32, device="cuda")
        table[:, 0] = 0
        q = torch.zeros(seqs * rows, 1, d, dtype=F16, device="cuda")
        cu = ints([i * rows for i in range(seqs + 1)])
        check(*ops.attention_paged(q, kc, vc, table, cu, ints([n] * seqs), rows, causal=False, return_lse=True), n, ("paged", rows))
    assert ops.attention_status() == 0


@pytest.mark.parametrize("extra", [0, 37])
def test_an_item_of_more_than_a_hundred_million_keys(extra):
    """One row over so many keys that its one block works for longer than any wait's limit.  Equal scores: probabilities of 1, whose sums
    are exact below 2^27 (steps of 8 for sums of 16), so the outputs are shares of n, rounded once."""
    n, tail, d = 2 ** 27 - 4096 + extra, 2 ** 22, 8
    q = torch.ones(1, 1, d, dtype=F16, device="cuda")
    k = torch.zeros(n, 1, d, dtype=F16, device="cuda")
    v = torch.zeros(n, 1, d, dtype=F16, device="cuda")
    v[:, :, 0] = 1
    v[-tail:, :, 1] = 1
    v[:tail, :, 2] = 1
    out, lse = ops.attention_packed(q, k, v, ints([0, 1]), ints([0, n]), causal=False, return_lse=True)
    assert ops.attention_status() == 0
    want = torch.tensor([1.0, tail / n, tail / n] + [0.0] * 5, dtype=torch.float64, device="cuda")
    assert bool(((out[0, 0].double() - want).abs() <= want * (2.0 ** -11 + 2.0 ** -22)).all())
    assert abs(float(lse[0, 0]) - math.log(n)) <= 2.0 ** -19  # one step of fp32 at 18.7


def busy(*shapes):
    """Work queued on the current stream that will write NaN (or -1) into memory which is free for the next tensors of these shapes."""
    tensors = [torch.zeros(s, dtype=t, device="cuda") for s, t in shapes]
    torch.cuda._sleep(200_000_000)  # a tenth of a second
    for t in tensors:
        t.fill_(math.nan if t.dtype.is_floating_point else -1)


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("new", [1, 90])
def test_tensors_made_for_another_stream_are_not_in_use_here(new, handle):
    """Calls on a side stream that make their outputs and workspaces, while the current stream still has work queued on memory
    that it has freed."""
    g = generator(22)
    q, n = rand(g, new, 8, 128, dtype=BF16, std=2.0), 6000
    k, v = (rand(g, n, 2, 128, dtype=BF16) for _ in range(2))
    kc, vc, table = paged_of(k, v)
    cu, lens, cu_k = ints([0, new]), ints([n]), ints([0, n])
    want = oracle.attend_block(q, k, v, 128 ** -0.5, True)
    size = ops.attention_paged_workspace(q, kc, 1, new).numel()
    side = torch.cuda.Stream()
    stream = side.cuda_stream if handle else side
    torch.cuda.synchronize()
    shapes = ((q.shape, BF16), (q.shape[:2], torch.float32), ((size,), torch.uint8))
    busy(*shapes)
    got = [ops.attention_paged(q, kc, vc, table, cu, lens, new, return_lse=True, stream=stream)]
    busy(*shapes)
    got.append(ops.attention_packed(q, k, v, cu, cu_k, return_lse=True, stream=stream))
    torch.cuda.synchronize()
    for out, lse in got:
        oracle.check(out, lse, *want)
    made, allocate = [], ops.attention_paged_workspace

    def spy(*args):
        made.append((torch.cuda.current_stream().cuda_stream, allocate(*args)))
        return made[-1][1]

    ops.attention_paged_workspace = spy  # the workspace is taken where it is used
    try:
        ops.attention_paged(q, kc, vc, table, cu, lens, new, stream=stream)
    finally:
        ops.attention_paged_workspace = allocate
    assert [s for s, _ in made] == [side.cuda_stream]
    assert torch.cuda.current_stream() == torch.cuda.default_stream()


def test_tables_made_for_another_stream_are_not_in_use_here():
    n = 300
    ctx, new, table = ints([20] * n), ints([1] * n), torch.full((n, 4), 9, dtype=torch.int32, device="cuda")
    free, state = ints(list(range(50))), ints([50, 0])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    i32 = torch.int32
    busy(((n + 1,), i32), ((n,), i32), ((n,), i32), ((2,), i32))
    cu, kv, slots, state = ops.page_tables(ctx, new, table, free, state, 16, max_tokens=n, stream=side)
    torch.cuda.synchronize()
    assert cu.tolist() == list(range(n + 1)) and kv.tolist() == [21] * n
    assert slots.tolist() == [9 * 16 + 4] * n and state.tolist() == [50, 0]


@pytest.mark.parametrize("new", [1, 100])
def test_status_covers_calls_on_side_streams(new):
    """A bad table entry met by a call that is still to run when the status is asked for."""
    g = generator(23)
    q = rand(g, new, 2, 64, dtype=F16)
    kc, vc, table = paged_of(*(rand(g, 200, 2, 64, dtype=F16) for _ in range(2)))
    table[0, 3] = -1
    cu, lens = ints([0, new]), ints([200])
    ws = ops.attention_paged_workspace(q, kc, 1, new)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert ops.attention_status() == 0
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        ops.attention_paged(q, kc, vc, table, cu, lens, new, workspace=ws)
    assert ops.attention_status() == ops.ATTENTION_BAD_PAGE
    assert ops.attention_status() == 0


def test_status_is_read_by_one_of_many_readers():
    from concurrent.futures import ThreadPoolExecutor

    g = generator(24)
    q = rand(g, 1, 2, 64, dtype=F16)
    kc, vc, table = paged_of(*(rand(g, 40, 2, 64, dtype=F16) for _ in range(2)))
    table[0, 1] = kc.shape[0]
    assert ops.attention_status() == 0
    with ThreadPoolExecutor(8) as pool:
        for _ in range(20):
            ops.attention_paged(q, kc, vc, table, ints([0, 1]), ints([40]), 1)
            got = list(pool.map(lambda _: ops.attention_status(), range(8)))
            assert sorted(got) == [0] * 7 + [ops.ATTENTION_BAD_PAGE]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("keys", [300, 20000])
@pytest.mark.parametrize("first,last", [(-math.inf, math.inf), (math.inf, -math.inf), (math.nan, math.inf), (math.inf, math.inf)])
def test_infinities_that_meet(first, last, keys, dtype):
    """An infinity of V that every row of a tile sees, and one near the end that only the last rows see: the rows that see both get
    what their sum is."""
    g = generator(4)
    q = rand(g, 80, 4, 64, dtype=dtype)
    k, v = (rand(g, keys, 2, 64, dtype=dtype) for _ in range(2))
    v[0, 0, 3] = v[1, 1, 40] = first
    v[-1, 0, 3] = v[-3, 1, 40] = last
    want = oracle.attend(q, k, v, 0.125, True)
    for name, out, lse, rows in every_way(q, k, v, 0.125, True, (1, 2, 15, 80)):
        oracle.check(out, lse, *[w[rows] for w in want], name)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_an_infinite_value_in_a_row_of_nan_scores(dtype):
    g = generator(5)
    q = rand(g, 80, 2, 64, dtype=dtype)
    k, v = (rand(g, 300, 2, 64, dtype=dtype) for _ in range(2))
    k[5, 0], v[-1, 0, 7] = math.nan, math.inf
    want = oracle.attend(q, k, v, 0.125, True)
    assert bool(torch.isnan(want[0][:, 0]).all())
    for name, out, lse, rows in every_way(q, k, v, 0.125, True, (1, 2, 80)):
        oracle.check(out, None, *[w[rows] for w in want], name)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("keys", [17, 33, 49, 65, 81, 700])
def test_a_nan_score_reaches_lse(keys, dtype):
    """The last key alone is NaN, wherever the computing warps' shares of a unit end."""
    g = generator(3)
    q = rand(g, 1, 4, 64, dtype=dtype)
    k, v = (rand(g, keys, 2, 64, dtype=dtype) for _ in range(2))
    k[-1, 1] = math.nan
    want = oracle.attend(q, k, v, 0.125, True)
    assert bool(torch.isnan(want[1][:, 2:]).all())
    for name, out, lse, rows in every_way(q, k, v, 0.125, True, (1,)):
        assert torch.equal(torch.isnan(out), torch.isnan(want[0])), name
        assert torch.equal(torch.isnan(lse), torch.isnan(want[1])), name


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -130, 2.0 ** -120, 2.0 ** -90])
def test_small_scales_of_large_scores(scale):
    """Scores near the end of fp32 under scales down to 0: the scaled scores are what counts."""
    g = generator(1)
    n, d = 300, 64
    q, k = ((torch.rand(n, 2, d, generator=g, device="cuda") + 0.5).mul(1e18).to(BF16) for _ in range(2))
    k = torch.where(torch.rand(n, 2, 1, generator=g, device="cuda") < 0.5, k, -k)  # scores of both signs, about 6e37
    v = rand(g, n, 2, d, dtype=BF16)
    want = oracle.attend_block(q, k, v, scale, True)
    for name, out, lse, rows in every_way(q, k, v, scale, True, (1, 5, 80)):
        oracle.check(out, lse, *[w[rows] for w in want], name)


def test_large_scales_of_small_scores():
    """The largest scale, over scores of 1e-35."""
    g = generator(2)
    n, d, scale = 300, 64, float(torch.tensor(1e38))  # as fp32 holds it
    q, k = ((torch.rand(n, 2, d, generator=g, device="cuda") + 1).mul(1e-18).to(BF16) for _ in range(2))
    k = torch.where(torch.rand(n, 2, d, generator=g, device="cuda") < 0.5, k, -k)  # no product is subnormal
    v = rand(g, n, 2, d, dtype=BF16)
    want = oracle.attend_block(q, k, v, scale, True)
    for name, out, lse, rows in every_way(q, k, v, scale, True, (1, 5, 80)):
        oracle.check(out, lse, *[w[rows] for w in want], name)


@pytest.mark.parametrize("scale", [1.01e38, 3e38])
def test_scales_whose_exponents_pass_fp32_are_refused(scale):
    q = torch.zeros(1, 1, 8, dtype=BF16, device="cuda")
    with pytest.raises(_native.AexrtError, match="scale must be from 0 to 1e38"):
        ops.attention_packed(q, q, q, ints([0, 1]), ints([0, 1]), scale=scale)
    kc, vc, table = paged_of(q, q)
    with pytest.raises(_native.AexrtError, match="scale must be from 0 to 1e38"):
        ops.attention_paged(q, kc, vc, table, ints([0, 1]), ints([1]), 1, scale=scale)


def test_fp16_averages_of_its_largest_value_stay_finite():
    """Every value 65504: an average cannot pass it, whatever the probabilities' rounding adds up to.  Scores a over the second half of
    the keys, 0 over the first, so that the later probabilities are e^a as fp16 rounds it."""
    n, heads, d = 512, 16, 64
    rows = 40
    a = torch.linspace(0.1, 5.0, rows * heads, device="cuda").reshape(rows, heads)
    q = torch.zeros(rows, heads, d, dtype=F16, device="cuda")
    q[..., 0] = a.to(F16)
    k = torch.zeros(n, 1, d, dtype=F16, device="cuda")
    k[n // 2:, :, 0] = 1
    v = torch.full((n, 1, d), 65504.0, dtype=F16, device="cuda")
    v[:, :, d // 2:] = -65504.0
    want = oracle.attend_block(q, k, v, 1.0, False)
    for name, out, lse, at in every_way(q, k, v, 1.0, False, (1, 2, 4, 40)):
        assert bool(torch.isfinite(out).all()), name
        oracle.check(out, lse, *[w[at] for w in want], name)
    # many (sequence, head) pairs, so that a block keeps several units of each
    seqs = 400
    kc, vc, table = paged_of(k, v)
    a = torch.linspace(0.1, 5.0, seqs * heads, device="cuda").reshape(seqs, heads)
    q = torch.zeros(seqs, heads, d, dtype=F16, device="cuda")
    q[..., 0] = a.to(F16)
    out = ops.attention_paged(q, kc, vc, table.expand(seqs, -1).contiguous(), ints(list(range(seqs + 1))), ints([n] * seqs), 1, scale=1.0)
    assert bool(torch.isfinite(out).all())
    # infinite values stay what they are
    v[3, 0, 0], v[4, 0, d - 1] = math.inf, -math.inf
    for name, out, lse, at in every_way(q[:40], k, v, 1.0, False, (1, 40)):
        assert bool((out[..., 0] == math.inf).all()) and bool((out[..., d - 1] == -math.inf).all()), name
        assert bool(torch.isfinite(out[..., 1:d - 1]).all()), name


def test_fp16_keeps_the_mass_of_small_probabilities():
    """One key far above all others, which together count: each of their probabilities is 2^-25.6 of the largest.  The bound is the
    oracle's with its last term's step taken relative to probabilities of up to 2^7: n 2^-32 V."""
    def check(out, k, v, q, what):
        s = (q.double() @ k.double().T)
        p = torch.exp(s - s.max())
        p /= p.sum()
        want, size, n = p @ v.double(), p @ v.double().abs(), k.shape[0]
        u = oracle.half_step(F16)
        tol = size * (u + 2 * 2.0 ** -17 + n * 2.0 ** -22) + u * want.abs() + n * 2.0 ** -32 * v.double().abs().max() + 2.0 ** -25
        # scores: one product each, exact in fp32, so no term for them
        over = (out.double() - want).abs() / tol
        assert bool((over <= 1).all()), f"{what}: {float(over.max()):.3g} of the bound"

    d = 64
    for n, size in ((32768, 100.0), (2048, 60000.0)):
        k = torch.zeros(n, 1, d, dtype=F16, device="cuda")
        k[0, 0, 0] = 17.75
        v = torch.full((n, 1, d), size, dtype=F16, device="cuda")
        v[0] = 0
        for rows in (1, 100):
            q = torch.zeros(rows, 1, d, dtype=F16, device="cuda")
            q[..., 0] = 1
            for name, out, lse, at in every_way(q, k, v, 1.0, False, (rows,)):
                for r in range(out.shape[0]):
                    check(out[r, 0], k[:, 0], v[:, 0], q[at][r, 0], (name, n))
        seqs = 300  # one block has many units of a sequence
        kc, vc, table = paged_of(k, v)
        q = torch.zeros(seqs, 1, d, dtype=F16, device="cuda")
        q[..., 0] = 1
        out = ops.attention_paged(q, kc, vc, table.expand(seqs, -1).contiguous(), ints(list(range(seqs + 1))), ints([n] * seqs), 1, scale=1.0)
        for r in range(0, seqs, 7):
            check(out[r, 0], k[:, 0], v[:, 0], q[r, 0], ("rows", n))


def unit_weights(call, keys_of, lens, dim, unit=64):
    """Equal scores and values that are 1 in one column per unit of keys: every unit's weight is read from the outputs, dim units a
    call.  call(v_of) -> [(out row [heads, dim], lse row, seen keys, sequence)], v_of(s) the values of a sequence."""
    units = -(-max(lens) // unit)
    for w in range(0, units, dim):
        def values(s):
            n = lens[s]
            v = torch.zeros(n, keys_of, dim, device="cuda")
            at = torch.arange(n, device="cuda")
            col = at // unit - w
            on = (col >= 0) & (col < dim)
            v[at[on], :, col[on]] = 1
            return v

        for out, lse, seen, s in call(values):
            edges = torch.arange(w, w + dim, device="cuda") * unit
            count = (seen - edges).clamp(0, unit).double()
            want = count / max(seen, 1)
            # counts are exact sums of ones; the normaliser, its reciprocal and the product round in fp32, the output once
            tol = want * (oracle.half_step(out.dtype) + 2.0 ** -21) + 2.0 ** -25
            assert bool(((out.double() - want).abs() <= tol).all()), (s, seen, w)
            if seen:
                assert bool(((lse - math.log(seen)).abs() <= 2.0 ** -19).all()), (s, seen)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,new,hq,hk", [
    ([33000, 11, 9000, 64, 65, 63, 1], 1, 8, 2), ([33000, 11, 9000], 3, 4, 1), ([20000, 129], 9, 16, 4), ([33000, 700, 9000], 70, 4, 2),
    ([9000, 9001, 8999], 200, 4, 4), ([64 * i + i % 3 for i in range(1, 60)], 1, 2, 2), ([3000] * 40, 5, 6, 3)])
def test_every_unit_of_keys_counts_once(lens, new, hq, hk, dtype):
    """The borders between blocks' shares of the keys, in both paged kernels: no unit is lost and none is taken twice."""
    d, page = 128, 16
    new_of = [min(new, n) for n in lens]
    kc, vc = (torch.zeros(sum(-(-n // page) for n in lens), page, hk, d, dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((len(lens), -(-max(lens) // page)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        m = -(-n // page)
        table[i, :m] = torch.arange(at, at + m, dtype=torch.int32, device="cuda").flip(0)
        at += m
    q = torch.zeros(sum(new_of), hq, d, dtype=dtype, device="cuda")
    cu = oracle.sums(new_of)

    def call(values):
        for i, n in enumerate(lens):
            ids = table[i, :-(-n // page)].long()
            rows = torch.zeros(len(ids) * page, hk, d, device="cuda")
            rows[:n] = values(i)
            vc[ids] = rows.view(len(ids), page, hk, d).to(dtype)
        for causal in (True, False):
            out, lse = ops.attention_paged(q, kc, vc, table, ints(cu), ints(lens), max(new_of), causal=causal, return_lse=True)
            for i, n in enumerate(lens):
                for r in {0, new_of[i] - 1, new_of[i] // 2}:
                    yield out[cu[i] + r], lse[cu[i] + r], r + 1 + n - new_of[i] if causal else n, i

    unit_weights(call, hk, lens, d)
    assert ops.attention_status() == 0


@pytest.mark.parametrize("lens", [[9000, 300], [128 * i + i for i in range(1, 20)]])
def test_every_unit_of_a_prompt_counts_once(lens):
    hq, hk, d = 4, 2, 64
    cu = oracle.sums(lens)
    q, k = (torch.zeros(cu[-1], h, d, dtype=BF16, device="cuda") for h in (hq, hk))

    def call(values):
        v = torch.cat([values(i) for i in range(len(lens))]).to(BF16)
        for causal in (True, False):
            out, lse = ops.attention_packed(q, k, v, ints(cu), ints(cu), causal=causal, return_lse=True)
            for i, n in enumerate(lens):
                for r in {0, 1, 127, n // 2, n - 2, n - 1}:
                    yield out[cu[i] + r], lse[cu[i] + r], r + 1 if causal else n, i

    unit_weights(call, hk, lens, d)


def test_heads_and_tokens_of_stride_0():
    """Broadcast key/value heads, a broadcast key and broadcast queries: as copies of them."""
    g = generator(25)
    q = rand(g, 70, 4, 64, dtype=F16)
    k, v = (rand(g, 70, 1, 64, dtype=F16) for _ in range(2))
    one = rand(g, 1, 4, 64, dtype=F16)
    cu = ints([0, 70])
    for args in ((q, k.expand(70, 4, 64), v.expand(70, 4, 64)), (q, one.expand(70, 4, 64), one.expand(70, 4, 64)),
                 (one.expand(70, 4, 64), q, q), (q[:, :1].expand(70, 4, 64), q, q)):
        want = ops.attention_packed(*(t.contiguous() for t in args), cu, cu, return_lse=True)
        got = ops.attention_packed(*args, cu, cu, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    kc, vc, table = paged_of(k, v)
    for new in (1, 70):
        args = (q[-new:], kc.expand(-1, 16, 4, 64), vc.expand(-1, 16, 4, 64))
        rest = (table, ints([0, new]), ints([70]), new)
        assert torch.equal(ops.attention_paged(*args, *rest), ops.attention_paged(*(t.contiguous() for t in args), *rest))


@pytest.mark.parametrize("n", [128, 129, 200])
def test_many_sequences_of_many_rows_over_a_cache(n):
    """More sequences than the tensor-core kernel orders by length, some of them empty or without new tokens."""
    import random

    rng, g = random.Random(n), generator(26)
    new = [rng.choice([0, 1, 40, 65, 130]) for _ in range(n)]
    lens = [x + rng.choice([0, 1, 15, 300, 1100]) if rng.random() < 0.9 else 0 for x in new]
    hq, hk, d, page = 4, 2, 64, 32
    need = [-(-x // page) for x in lens]
    kc, vc = (rand(g, sum(need) + 1, page, hk, d, dtype=BF16) for _ in range(2))
    kc[-1], vc[-1] = math.nan, math.nan
    table = torch.full((n, max(need)), sum(need), dtype=torch.int32, device="cuda")
    at, parts, rows = 0, [], 0
    q = rand(g, sum(new), hq, d, dtype=BF16, std=2.0)
    for i, m in enumerate(need):
        ids = torch.arange(at, at + m, device="cuda")
        table[i, :m] = ids.int()
        at += m
        parts.append(oracle.attend_block(q[rows:rows + new[i]], kc[ids].flatten(0, 1)[:lens[i]], vc[ids].flatten(0, 1)[:lens[i]],
                                         0.125, True))
        rows += new[i]
    out = torch.full_like(q, 1000.0)
    out, lse = ops.attention_paged(q, kc, vc, table, ints(oracle.sums(new)), ints(lens), max(new), out=out, return_lse=True)
    assert ops.attention_status() == 0
    oracle.check(out, lse, *[torch.cat(x) for x in zip(*parts)])


def test_prompts_captured_and_replayed_with_other_lengths():
    g = generator(27)
    t, hq, hk, d, n = 900, 8, 2, 128, 6
    q, out = (torch.zeros(t, hq, d, dtype=BF16, device="cuda") for _ in range(2))
    k, v = (torch.zeros(t, hk, d, dtype=BF16, device="cuda") for _ in range(2))
    lse, cu = torch.zeros(t, hq, device="cuda"), ints([0] * (n + 1))
    ops.attention_packed(q, k, v, cu, cu, out=out, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_packed(q, k, v, cu, cu, out=out, lse=lse)
    for lens in ([900, 0, 0, 0, 0, 0], [1, 1, 1, 1, 1, 1], [130, 256, 0, 77, 300, 1], [0] * 6, [0, 0, 0, 0, 0, 641]):
        for x in (q, k, v):
            x.copy_(rand(g, *x.shape, dtype=BF16))
        cu.copy_(ints(oracle.sums(lens)))
        out.fill_(5.0)
        lse.fill_(7.0)
        graph.replay()
        s = sum(lens)
        parts = [oracle.attend_block(a, b, c, d ** -0.5, True) for a, b, c in zip(*(torch.split(x[:s], lens) for x in (q, k, v)))]
        oracle.check(out[:s], lse[:s], *[torch.cat(x) for x in zip(*parts)])
        assert bool((out[s:] == 5).all()) and bool((lse[s:] == 7).all())
    assert ops.attention_status() == 0


@pytest.mark.parametrize("new", [1, 7, 90, 400])
def test_outputs_in_place_of_the_queries(new):
    """out may be q."""
    g = generator(28)
    lens = [5000, new, 40 + new]
    q, kv = rand(g, 3 * new, 8, 128, dtype=BF16), [(rand(g, n, 2, 128, dtype=BF16), rand(g, n, 2, 128, dtype=BF16)) for n in lens]
    cu = ints([0, new, 2 * new, 3 * new])
    k, v = (torch.cat(x) for x in zip(*kv))
    want = ops.attention_packed(q, k, v, cu, ints(oracle.sums(lens)))
    here = q.clone()
    assert ops.attention_packed(here, k, v, cu, ints(oracle.sums(lens)), out=here) is here and torch.equal(here, want)
    caches = [paged_of(a, b) for a, b in kv]
    kc, vc = (torch.cat([c[i] for c in caches]) for i in (0, 1))
    table, at = torch.full((3, max(c[2].shape[1] for c in caches)), -1, dtype=torch.int32, device="cuda"), 0
    for i, c in enumerate(caches):
        table[i, :c[2].shape[1]] = c[2][0] + at
        at += c[2].shape[1]
    want = ops.attention_paged(q, kc, vc, table, cu, ints(lens), new)
    here = q.clone()
    ops.attention_paged(here, kc, vc, table, cu, ints(lens), new, out=here)
    assert torch.equal(here, want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [1, 4, 16, 32])
def test_few_rows_over_several_stretches(group, dtype):
    """Contexts longer than what a warp sums at a time, each inside one block's share: values and infinities of all stretches."""
    g = generator(29)
    n, d, seqs = 140001, 64, 300
    k, v = (rand(g, n, 1, d, dtype=dtype) for _ in range(2))
    v[70000, 0, 7], v[-1, 0, 5], v[-1, 0, 7] = -math.inf, math.inf, math.inf  # the last key: the second row's alone
    kc, vc, table = paged_of(k, v, 1024)
    q = rand(g, 2 * seqs, group, d, dtype=dtype)
    out, lse = ops.attention_paged(q, kc, vc, table.expand(seqs, -1).contiguous(), ints([2 * i for i in range(seqs + 1)]),
                                   ints([n] * seqs), 2, return_lse=True)
    assert ops.attention_status() == 0
    for s in (0, 148, seqs - 1):
        at = slice(2 * s, 2 * s + 2)
        oracle.check(out[at], lse[at], *oracle.attend(q[at], k, v, 0.125, True), f"sequence {s}")


def test_items_behind_one_of_a_hundred_million_keys():
    """The long item has one row, so that half of its block's softmax warps have nothing to do in it and wait for the next item's
    first scores as long as it lasts."""
    g = generator(30)
    n, d, short, rows = 2 ** 27 - 4096, 8, 320, 200
    k_lens, q_lens = [n] + [rows] * short, [1] + [rows] * short
    q = torch.zeros(1 + rows * short, 1, d, dtype=F16, device="cuda")
    k, v = (torch.zeros(n + rows * short, 1, d, dtype=F16, device="cuda") for _ in range(2))
    v[:n, :, 0] = 1
    for x, a in ((q, 1), (k, n), (v, n)):
        x[a:] = rand(g, rows * short, 1, d, dtype=F16)
    out, lse = ops.attention_packed(q, k, v, ints(oracle.sums(q_lens)), ints(oracle.sums(k_lens)), causal=False, return_lse=True)
    assert ops.attention_status() == 0
    assert out[0, 0].tolist() == [1.0] + [0.0] * 7 and abs(float(lse[0, 0]) - math.log(n)) <= 2.0 ** -19
    for i in (0, 146, 147, 148, 293, 294, 295, 319):  # of the first block's second item and around
        at, kat = slice(1 + rows * i, 1 + rows * (i + 1)), slice(n + rows * i, n + rows * (i + 1))
        oracle.check(out[at], lse[at], *oracle.attend_block(q[at], k[kat], v[kat], d ** -0.5, False), f"sequence {i}")


@pytest.mark.parametrize("new", [1, 70])
def test_most_sequences_and_many_heads(new):
    """65535 sequences in one call (the few-rows kernel, and the tensor-core one as if each could bring 70 rows), and 4096 heads."""
    g = generator(31)
    n, d, page = 65535, 8, 8
    q = rand(g, n, 1, d, dtype=F16)
    kc, vc = (rand(g, 50, page, 1, d, dtype=F16) for _ in range(2))
    table = torch.randint(0, 50, (n, 1), generator=g, device="cuda").int()
    lens = torch.randint(0, page + 1, (n,), generator=g, device="cuda").int()
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    out, lse = ops.attention_paged(q, kc, vc, table, cu, lens, new, scale=0.5, return_lse=True)
    k, v = (c[table[:, 0].long(), :, 0].double() for c in (kc, vc))
    s = 0.5 * (q.double() @ k.transpose(1, 2))[:, 0]
    s = s.masked_fill(torch.arange(page, device="cuda")[None] >= lens[:, None], -math.inf)
    top = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(lens > 0, top, 0.0)[:, None])
    want, size = (p[:, None] @ v)[:, 0], (p[:, None] @ v.abs())[:, 0]
    # as the oracle's bound: scores are sums of 8 products, off by 10 * 2^-23 of theirs at most
    e_s = (10 * 2.0 ** -23 * 0.5 * (q.double().abs() @ k.abs().transpose(1, 2))[:, 0]).amax(1, keepdim=True)
    u = oracle.half_step(F16)
    tol = size * (u + 2 * e_s + 2.0 ** -16 + 2.0 ** -19) + u * want.abs() + 2.0 ** -25
    assert bool(((out[:, 0].double() - want).abs() <= tol).all())
    empty = lens == 0
    assert bool((lse[empty] == -math.inf).all()) and bool(((lse[:, 0] - top).abs()[~empty] <= 2.0 ** -16).all())
    h = 4096
    q, k, v = (rand(g, 5, h, d, dtype=BF16) for _ in range(3))
    want = oracle.attend_block(q, k, v, 0.3, True)
    for name, out, lse, rows in every_way(q, k, v, 0.3, True, (1, 5)):
        oracle.check(out, lse, *[w[rows] for w in want], name)


def test_offsets_of_queries_and_outputs_beyond_32_bits():
    """Heads and tokens of q, k, v and out far apart in one wide buffer."""
    if torch.cuda.mem_get_info()[0] < 30 * 2 ** 30:
        pytest.skip("needs 30 GB")
    g = generator(32)
    flat = torch.empty(10 * 2 ** 30, dtype=BF16, device="cuda")
    hq, d, n = 2, 64, 3
    far = (2 ** 32 + 2 ** 20) // 8 * 8
    def wide(start, heads, across):  # [n, heads, d] with heads (or tokens) 2^32 elements apart
        strides = (d, far, 1) if across == "heads" else (far // 2, d, 1)
        t = torch.as_strided(flat, (n, heads, d), strides, start)
        t.copy_(rand(g, n, heads, d, dtype=BF16))
        return t
    for across in ("heads", "tokens"):
        q, k, v, out = (wide(4096 * i, hq, across) for i in range(4))
        want = oracle.attend_block(q.contiguous(), k.contiguous(), v.contiguous(), 0.125, True)
        cu = ints([0, n])
        ops.attention_packed(q, k, v, cu, cu, out=out)
        oracle.check(out.contiguous(), None, *want, across)
        kc, vc, table = paged_of(k.contiguous(), v.contiguous())
        for rows in (n, 1):
            out.zero_()
            ops.attention_paged(q[n - rows:], kc, vc, table, ints([0, rows]), cu[1:], 40 if rows == n else 1, out=out[n - rows:])
            oracle.check(out[n - rows:].contiguous(), None, *[w[n - rows:] for w in want], across)
    assert ops.attention_status() == 0


@pytest.mark.parametrize("n,rows", [(4, 2560), (20, 2560), (128, 2560), (60, 700)])
def test_offsets_that_go_back_stay_inside_the_workspace(n, rows):
    """Every second sequence has all query rows again: far more work than rows and sequences suggest.  Only the workspace's own
    bytes are written."""
    import random

    rng, g = random.Random(n), generator(33)
    q = rand(g, rows, 2, 64, dtype=F16)
    kc, vc = (rand(g, 40, 16, 1, 64, dtype=F16) for _ in range(2))
    lens = [rng.choice([100, 640, 9000, 30000]) for _ in range(n)]
    table = torch.randint(0, 40, (n, 1875), generator=g, device="cuda").int()
    size = ops.attention_paged_workspace(q, kc, n, rows).numel()
    assert size
    buffer = torch.full((size + 2 ** 24,), 0x5a, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 1000.0)
    ops.attention_paged(q, kc, vc, table, ints([i % 2 * rows for i in range(n + 1)]), ints(lens), rows, out=out,
                        workspace=buffer[:size])
    assert ops.attention_status() == 0
    assert bool((buffer[size:] == 0x5a).all())
    assert bool((out.abs() < 100).all())  # rows of several sequences hold one of theirs
