"""Workloads of the sequence-attention operators: packed prompts, the paged cache, its tables and its writes.

Each case is one call of one operator, as a serving step makes it.  ``own`` selects what ``run`` calls: the
plain forms below (elementary torch operations in fp32) or the framework's kernels.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- lengths
def _spread(total, n, mix, least=1):
    """n ragged lengths (each at least `least`) that add up to total."""
    rng = random.Random(mix)
    w = [math.exp(rng.gauss(0.0, 0.8)) for _ in range(n)]
    spare = total - least * n
    cut = [int(spare * x / sum(w)) for x in w]
    cut[rng.randrange(n)] += spare - sum(cut)
    return [least + c for c in cut]


def _lengths(case):
    """(query lengths, key lengths) of an attention case; (context, new) lengths of a tables case."""
    n, mix = case["seqs"], case["mix"]
    if case["op"] == "packed":
        q = _spread(case["tokens"], n, mix) if case["ragged"] else [case["tokens"] // n] * n
        k = q if not case["cross"] else _spread(case["cross"], n, mix + 1)
        return q, k
    if case["op"] == "paged":
        ctx = _spread(case["context"], n, mix, 0) if case["ragged"] else [case["context"] // n] * n
        return [case["new"]] * n, [c + case["new"] for c in ctx]
    ctx = _spread(case["context"], n, mix, 0)
    return ctx, (_spread(case["new"], n, mix + 1) if case["ragged"] else [case["new"] // n] * n)


def _pages(tokens, size):
    return (tokens + size - 1) // size


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a handful of short prompts arriving at an idle server: latency of the smallest prefill
        {"name": "prompt_short_fp16", "op": "packed", "dtype": "fp16", "seqs": 4, "tokens": 122, "ragged": True, "cross": 0,
         "q_heads": 8, "kv_heads": 8, "dim": 64, "causal": True, "mix": 1},
        # full attention over 40 x 40 feature maps, 4 heads: the detectors' attention block at four times the input side
        {"name": "map_full_fp16", "op": "packed", "dtype": "fp16", "seqs": 16, "tokens": 16 * 1600, "ragged": False, "cross": 0,
         "q_heads": 4, "kv_heads": 4, "dim": 64, "causal": False, "mix": 2},
        # an ordinary prefill batch: ragged prompts, grouped heads
        {"name": "prompt_ragged_bf16", "op": "packed", "dtype": "bf16", "seqs": 19, "tokens": 15001, "ragged": True, "cross": 0,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "mix": 3},
        # one long document
        {"name": "prompt_long_bf16", "op": "packed", "dtype": "bf16", "seqs": 1, "tokens": 16384, "ragged": True, "cross": 0,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "mix": 4},
        # one user, one token: latency of the smallest decode step
        {"name": "token_one_fp16", "op": "paged", "dtype": "fp16", "seqs": 1, "context": 1000, "ragged": True, "new": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "mix": 5},
        # a decode step of a full server: ragged contexts
        {"name": "token_batch_bf16", "op": "paged", "dtype": "bf16", "seqs": 64, "context": 262144, "ragged": True, "new": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "mix": 6},
        # five drafted tokens a request checked at once, no head sharing, a head size that is no power of two
        {"name": "draft_check_fp16", "op": "paged", "dtype": "fp16", "seqs": 32, "context": 70001, "ragged": True, "new": 5,
         "q_heads": 16, "kv_heads": 16, "dim": 96, "page": 32, "causal": True, "mix": 7},
        # a prompt taken in chunks: 1024 new tokens each over what is cached
        {"name": "chunk_long_bf16", "op": "paged", "dtype": "bf16", "seqs": 2, "context": 32768, "ragged": True, "new": 1024,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "mix": 8},
        # tables of a decode step: one token for each of 256 requests
        {"name": "tables_step", "op": "tables", "seqs": 256, "context": 500000, "ragged": False, "new": 256, "page": 16,
         "columns": 2048, "spare": 50, "mix": 9},
        # tables of a prefill step
        {"name": "tables_prompt", "op": "tables", "seqs": 64, "context": 20000, "ragged": True, "new": 65536, "page": 16,
         "columns": 2048, "spare": 50, "mix": 10},
        # a decode step's rows into the cache
        {"name": "append_step_fp16", "op": "append", "dtype": "fp16", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16,
         "pages": 512, "mix": 11},
        # a prefill step's rows into the cache
        {"name": "append_prompt_bf16", "op": "append", "dtype": "bf16", "tokens": 32768, "kv_heads": 8, "dim": 128, "page": 16,
         "pages": 4096, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "paged", "paged", "tables", "append"])
    mix = rng.randrange(1 << 30)
    kv = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if kv * group > 48:
        group = 1
    heads = {"dtype": rng.choice(["fp16", "bf16"]), "q_heads": kv * group, "kv_heads": kv,
             "dim": rng.choice([16, 32, 40, 64, 64, 80, 96, 104, 128, 128, 128])}
    if op == "packed":
        seqs = _log(rng, 1, 48)
        tokens = max(seqs, _log(rng, 16, 16000))
        cross = max(seqs, _log(rng, 16, 8000)) if rng.random() < 0.25 else 0
        return {"op": op, **heads, "seqs": seqs, "tokens": tokens, "ragged": True, "cross": cross,
                "causal": rng.random() < 0.7, "mix": mix}
    if op == "paged":
        new = rng.choice([1, 1, 1, 2, 3, 7, _log(rng, 8, 1500)])
        seqs = _log(rng, 1, 96 if new < 8 else 6)
        context = _log(rng, 64, min(200000, 250000000 // (kv * heads["dim"])) if new < 8 else 30000)
        return {"op": op, **heads, "seqs": seqs, "context": context, "ragged": True, "new": new,
                "page": rng.choice([16, 16, 32, 64, 128]), "causal": True, "mix": mix}
    if op == "tables":
        seqs = _log(rng, 1, 700)
        step = rng.random() < 0.5
        case = {"op": op, "seqs": seqs, "context": _log(rng, 16, 400000), "ragged": not step,
                "new": seqs if step else max(seqs, _log(rng, 64, 65536)), "page": rng.choice([16, 32, 64, 128]), "mix": mix}
        # at times a free stack that runs out, or a row that is too short for its request
        case["spare"] = rng.choice([50, 50, 50, -1, -20])
        widest = max(_pages(a + b, case["page"]) for a, b in zip(*_lengths(case)))
        case["columns"] = max(1, widest + rng.choice([0, 5, 100, -1]))
        return case
    tokens = _log(rng, 1, 32000)
    page = rng.choice([16, 16, 32, 64, 128])
    return {"op": op, "dtype": heads["dtype"], "tokens": tokens, "kv_heads": kv, "dim": heads["dim"], "page": page,
            "pages": _pages(tokens, page) + _log(rng, 1, 2000), "mix": mix}


# ---------------------------------------------------------------- inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    """What a serving loop holds before the call: activations, cache, tables, and the buffers that it keeps from step to step."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + case["mix"] % 1000003)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(DTYPES[case["dtype"]])

    st = {"case": case, "op": case["op"]}
    if case["op"] == "packed":
        q, k = _lengths(case)
        st.update(q_lens=q, k_lens=k, cu_q=_ints(_sums(q)), cu_k=_ints(_sums(k)), scale=case["dim"] ** -0.5)
        # scores of a trained head spread by a few units
        st["q"] = normal(sum(q), case["q_heads"], case["dim"], std=2.0)
        st["k"] = normal(sum(k), case["kv_heads"], case["dim"])
        st["v"] = normal(sum(k), case["kv_heads"], case["dim"])
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(st["q"].shape[:2], dtype=torch.float32, device="cuda")
    elif case["op"] == "paged":
        q, k = _lengths(case)
        page = case["page"]
        need = [_pages(x, page) for x in k]
        total = sum(need) + 7
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(k), max(need) + 3), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        st.update(q_lens=q, k_lens=k, cu_q=_ints(_sums(q)), kv_lens=_ints(k), table=table, scale=case["dim"] ** -0.5)
        st["q"] = normal(sum(q), case["q_heads"], case["dim"], std=2.0)
        st["k_cache"] = normal(total, page, case["kv_heads"], case["dim"])
        st["v_cache"] = normal(total, page, case["kv_heads"], case["dim"])
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(st["q"].shape[:2], dtype=torch.float32, device="cuda")
        if own:
            from aexrt_b200 import ops

            st["workspace"] = ops.attention_paged_workspace(st["q"], st["k_cache"], len(k), case["new"])
    elif case["op"] == "tables":
        ctx, new = _lengths(case)
        page, columns = case["page"], case["columns"]
        have = [_pages(c, page) for c in ctx]
        total = sum(have) + max(1, sum(_pages(c + n, page) for c, n in zip(ctx, new)) - sum(have) + case["spare"])
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(ctx), columns), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(have):
            n = min(n, columns)
            table[i, :n] = order[at:at + n]
            at += n
        free = order[at:].contiguous()
        st.update(ctx=_ints(ctx), new=_ints(new), table=table, free=free, state=_ints([free.numel(), 0]),
                  tokens=sum(new), next_state=_ints([0, 0]), cu_q=_ints([0] * (len(ctx) + 1)),
                  kv_lens=_ints([0] * len(ctx)), slots=_ints([0] * sum(new)))
    else:
        n, page = case["tokens"], case["page"]
        slots = case["pages"] * page
        st["slots"] = torch.randperm(slots, generator=gen, device="cuda")[:n].to(torch.int32)
        if n > 3:
            st["slots"][n // 2] = -1  # a padded row of the batch
        st["k"] = normal(n, case["kv_heads"], case["dim"])
        st["v"] = normal(n, case["kv_heads"], case["dim"])
        st["k_cache"] = normal(case["pages"], page, case["kv_heads"], case["dim"])
        st["v_cache"] = normal(case["pages"], page, case["kv_heads"], case["dim"])
    return st


# ---------------------------------------------------------------- plain forms
def _attend(q, k, v, scale, causal, out, lse):
    """softmax(q k^T scale) v of one sequence, a block of rows at a time, in fp32."""
    lq, hq, d = q.shape
    lk, hk = k.shape[0], k.shape[1]
    if lk == 0:
        out.zero_()
        lse.fill_(-math.inf)
        return
    g = hq // hk
    kt = k.float().permute(1, 2, 0).unsqueeze(1)  # [hk, 1, d, lk]
    vt = v.float().permute(1, 0, 2).unsqueeze(1)  # [hk, 1, lk, d]
    step = max(1, min(lq, (1 << 28) // (hq * lk)))
    for a in range(0, lq, step):
        b = min(lq, a + step)
        end = max(0, min(lk, b + lk - lq)) if causal else lk
        if end == 0:
            out[a:b] = 0
            lse[a:b] = -math.inf
            continue
        qf = q[a:b].float().reshape(b - a, hk, g, d).permute(1, 2, 0, 3)
        s = (qf @ kt[..., :end]) * scale
        if causal:
            seen = torch.arange(end, device=q.device)[None, :] <= torch.arange(a, b, device=q.device)[:, None] + (lk - lq)
            s = torch.where(seen, s, -math.inf)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        p = torch.exp(s - m)
        total = p.sum(-1, keepdim=True)
        o = (p @ vt[..., :end, :]) / torch.where(total == 0, 1.0, total)
        out[a:b] = o.permute(2, 0, 1, 3).reshape(b - a, hq, d).to(out.dtype)
        lse[a:b] = (m + torch.log(total))[..., 0].permute(2, 0, 1).reshape(b - a, hq)


def _plain_tables(st):
    case = st["case"]
    page, columns = case["page"], case["columns"]
    ctx, new = st["ctx"].long(), st["new"].long()
    kv = ctx + new
    cu = torch.zeros(len(ctx) + 1, dtype=torch.int64, device="cuda")
    cu[1:] = new.cumsum(0)
    have = ((ctx + page - 1) // page).clamp(max=columns)
    take = ((kv + page - 1) // page).clamp(max=columns) - have
    first = take.cumsum(0) - take
    top = st["state"][0].long()
    wanted = torch.arange(st["tokens"] + len(ctx), device="cuda")
    row = torch.searchsorted(take.cumsum(0), wanted, right=True)
    there = row < len(ctx)
    row = row.clamp(max=len(ctx) - 1)
    col = have[row] + wanted - first[row]
    ids = torch.where(wanted < top, st["free"].long()[(top - 1 - wanted).clamp(min=0)], -1)
    table = st["table"]
    table.view(-1)[(row * columns + col)[there]] = ids[there].int()
    token = torch.arange(st["tokens"], device="cuda")
    row = torch.searchsorted(cu[1:], token, right=True)
    pos = ctx[row] + token - cu[row]
    col = pos // page
    ids = table[row, col.clamp(max=columns - 1)].long()
    slots = torch.where((col < columns) & (ids >= 0), ids * page + pos % page, -1)
    asked = take.sum()
    state = torch.stack([(top - asked).clamp(min=0), (asked - top).clamp(min=0)])
    return cu.int(), kv.int(), table, slots.int(), state.int()


def run(st):
    case = st["case"]
    if own:
        from aexrt_b200 import ops

        if st["op"] == "packed":
            return ops.attention_packed(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], causal=case["causal"],
                                        scale=st["scale"], out=st["out"], lse=st["lse"])
        if st["op"] == "paged":
            return ops.attention_paged(st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu_q"], st["kv_lens"],
                                       case["new"], causal=case["causal"], scale=st["scale"], out=st["out"], lse=st["lse"],
                                       workspace=st["workspace"])
        if st["op"] == "tables":
            cu, kv, slots, state = ops.page_tables(st["ctx"], st["new"], st["table"], st["free"], st["state"], case["page"],
                                                   cu_q=st["cu_q"], kv_lens=st["kv_lens"], slot_map=st["slots"],
                                                   free_state_out=st["next_state"])
            return cu, kv, st["table"], slots, state
        ops.kv_append(st["k"], st["v"], st["slots"], st["k_cache"], st["v_cache"])
        return st["k_cache"], st["v_cache"]
    if st["op"] == "packed":
        a = b = 0
        for lq, lk in zip(st["q_lens"], st["k_lens"]):
            _attend(st["q"][a:a + lq], st["k"][b:b + lk], st["v"][b:b + lk], st["scale"], case["causal"],
                    st["out"][a:a + lq], st["lse"][a:a + lq])
            a += lq
            b += lk
        return st["out"], st["lse"]
    if st["op"] == "paged":
        a, page = 0, case["page"]
        for i, (lq, lk) in enumerate(zip(st["q_lens"], st["k_lens"])):
            ids = st["table"][i, :_pages(lk, page)].long()
            k, v = (st[c][ids].flatten(0, 1)[:lk] for c in ("k_cache", "v_cache"))
            _attend(st["q"][a:a + lq], k, v, st["scale"], case["causal"], st["out"][a:a + lq], st["lse"][a:a + lq])
            a += lq
        return st["out"], st["lse"]
    if st["op"] == "tables":
        return _plain_tables(st)
    slots = st["slots"].long()
    there = slots >= 0
    for rows, cache in (("k", "k_cache"), ("v", "v_cache")):
        st[cache].flatten(0, 1)[slots[there]] = st[rows][there]
    return st["k_cache"], st["v_cache"]


# ---------------------------------------------------------------- what a pass cannot do without
def _seen(lq, lk, causal):
    """(row, key) pairs that the mask leaves."""
    if not causal:
        return lq * lk
    empty = max(0, lq - lk)
    return sum((lk - lq + 1 + empty, lk)) * (lq - empty) // 2


def work(case):
    if case["op"] in ("packed", "paged"):
        q, k = _lengths(case)
        pairs = sum(_seen(a, b, case["causal"]) for a, b in zip(q, k))
        rows, keys = sum(q) * case["q_heads"], sum(k) * case["kv_heads"]
        extra = 4 * 2 * len(q)
        if case["op"] == "paged":
            extra += 4 * sum(_pages(x, case["page"]) for x in k)
        return {"bytes": 2 * case["dim"] * (2 * rows + 2 * keys) + 4 * rows + extra,
                "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    if case["op"] == "tables":
        ctx, new = _lengths(case)
        taken = sum(_pages(c + n, case["page"]) - _pages(c, case["page"]) for c, n in zip(ctx, new))
        # the pages that the new tokens go to, the free ids taken, the lengths, the slots
        return {"bytes": 8 * taken + 4 * len(ctx) + 16 * len(ctx) + 4 * sum(new) + 20, "flops": sum(new) + 4 * len(ctx)}
    row = 2 * case["kv_heads"] * case["dim"]
    return {"bytes": case["tokens"] * (4 * row + 4), "flops": 0}


# ---------------------------------------------------------------- values from the definitions, in 64 bits
def _exact_head(q, k, v, scale, shift):
    """One query head over its sequence: q [lq, d], k, v [lk, d] in fp64; row i sees keys 0 .. i + shift (all: None)."""
    lq, lk = q.shape[0], k.shape[0]
    o = torch.zeros(lq, v.shape[1], dtype=torch.float64, device=q.device)
    lse = torch.full((lq,), -math.inf, dtype=torch.float64, device=q.device)
    if lk == 0:
        return o, lse
    keys = torch.arange(lk, device=q.device)
    for a in range(0, lq, 4096):
        b = min(lq, a + 4096)
        s = torch.mm(q[a:b], k.t()).mul_(scale)
        if shift is not None:
            s.masked_fill_(keys[None, :] > torch.arange(a, b, device=q.device)[:, None] + shift, -math.inf)
        total = torch.logsumexp(s, 1)
        live = total > -math.inf
        w = torch.exp_(s.sub_(torch.where(live, total, 0.0)[:, None]))
        o[a:b] = torch.mm(w, v)
        lse[a:b] = total
    return o, lse


def _exact_tables(st):
    case = st["case"]
    page, columns = case["page"], case["columns"]
    ctx, new, free = st["ctx"].tolist(), st["new"].tolist(), st["free"].tolist()
    table = st["table"].tolist()
    top, missing = st["state"].tolist()[0], 0
    cu, kv, slots = [0], [], []
    for i, (c, n) in enumerate(zip(ctx, new)):
        cu.append(cu[-1] + n)
        kv.append(c + n)
        for col in range(min(_pages(c, page), columns), min(_pages(c + n, page), columns)):
            if top:
                top -= 1
                table[i][col] = free[top]
            else:
                missing += 1
        for p in range(c, c + n):
            held = table[i][p // page] if p // page < columns else -1
            slots.append(held * page + p % page if held >= 0 else -1)
    return tuple(_ints(x) for x in (cu, kv, table, slots, [top, missing]))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(st)
    if case["op"] == "append":
        caches = []
        for rows, cache in (("k", "k_cache"), ("v", "v_cache")):
            host = st[cache].cpu()
            at, new = st["slots"].tolist(), st[rows].cpu()
            for t, s in enumerate(at):
                if s >= 0:
                    host[s // case["page"], s % case["page"]] = new[t]
            caches.append(host)
        return tuple(caches)
    group = case["q_heads"] // case["kv_heads"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(st["lse"].shape, dtype=torch.float64, device="cuda")
    a = b = 0
    for i, (lq, lk) in enumerate(zip(st["q_lens"], st["k_lens"])):
        if case["op"] == "packed":
            k, v = st["k"][b:b + lk], st["v"][b:b + lk]
        else:
            at = torch.arange(lk, device="cuda")
            held = st["table"][i].long()[at // case["page"]]
            k, v = (st[c][held, at % case["page"]] for c in ("k_cache", "v_cache"))
        for h in range(case["q_heads"]):
            out[a:a + lq, h], lse[a:a + lq, h] = _exact_head(
                st["q"][a:a + lq, h].double(), k[:, h // group].double(), v[:, h // group].double(), st["scale"],
                lk - lq if case["causal"] else None)
        a += lq
        b += lk
    return out, lse
