"""Oracle of attention over token sequences: the definition in 64 bits, over the keys that a row sees and no others, with
the error bound that the kernels' arithmetic allows at each output."""
import math

import torch


def sums(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, scale, causal):
    """One sequence: q [lq, hq, d], k, v [lk, hk, d] -> (out, lse, bound of out, bound of lse), fp64 on q's device.

    The bound counts, with u half a step of the 16-bit type and A = sum_j p_j |v_j| (p normalised):
      u A          each probability rounded to 16 bits for the second product
      u |o|        the output's rounding
      2 e_s A      scores: d + 2 products and sums in fp32, each off by at most 2^-23 of the sum of |q||k| (accumulation may truncate),
                   in numerator and normaliser
      2 e_x A      exp: 2^-13 (bf16) or 2^-17 (fp16) relative
      n 2^-22 A    the sums over n keys in fp32, added in any order: both products' (|p v| and p)
      n 2^-25 V    fp16 only: probabilities below fp16's normal range, rounded to a step of 2^-24, V = max |v| (of the finite ones)
    """
    lq, hq, d = q.shape
    lk, hk, _ = k.shape
    u = half_step(q.dtype)
    e_x = 2.0 ** -13 if q.dtype == torch.bfloat16 else 2.0 ** -17
    out = torch.zeros(lq, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((lq, hq), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    g = hq // hk
    for i in range(lq):
        seen = min(lk, i + 1 + lk - lq) if causal else lk
        if seen <= 0:
            continue
        for h in range(hk):
            qi = q[i, h * g:(h + 1) * g].double()
            kk, vv = k[:seen, h].double(), v[:seen, h].double()
            s = scale * qi @ kk.T
            e_s = ((d + 2) * 2.0 ** -23 * scale * (qi.abs() @ kk.abs().T)).amax(1, keepdim=True)
            top = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - top)
            o, a = p @ vv, p @ vv.abs()
            out[i, h * g:(h + 1) * g] = o
            lse[i, h * g:(h + 1) * g] = top[:, 0]
            t = a * (u + 2 * e_s + 2 * e_x + seen * 2.0 ** -22) + u * o.abs()
            if q.dtype == torch.float16:
                t = t + seen * 2.0 ** -25 * vv[vv.isfinite()].abs().max() + 2.0 ** -25  # the output's own subnormal step
            tol[i, h * g:(h + 1) * g] = t + 1e-30
            tol_lse[i, h * g:(h + 1) * g] = (e_s[:, 0] + e_x + seen * 2.0 ** -23 + 2.0 ** -22 * (1 + top[:, 0].abs()))
    return out, lse, tol, tol_lse


def attend_block(q, k, v, scale, causal):
    """:func:`attend` over all rows at once, for finite inputs and longer sequences (rows in blocks)."""
    lq, hq, d = q.shape
    lk, hk, _ = k.shape
    u = half_step(q.dtype)
    e_x = 2.0 ** -13 if q.dtype == torch.bfloat16 else 2.0 ** -17
    out = torch.zeros(lq, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((lq, hq), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    if lk == 0:
        return out, lse, tol, tol_lse
    keys = torch.arange(lk, device=q.device)
    for h in range(hq):
        kk, vv = k[:, h // (hq // hk)].double(), v[:, h // (hq // hk)].double()
        for a in range(0, lq, 2048):
            b = min(lq, a + 2048)
            qq = q[a:b, h].double()
            rows = torch.arange(a, b, device=q.device)
            seen = (rows + 1 + lk - lq).clamp(0, lk) if causal else torch.full_like(rows, lk)
            mask = keys[None, :] >= seen[:, None]
            s = (scale * qq @ kk.T).masked_fill(mask, -math.inf)
            e_s = ((d + 2) * 2.0 ** -23 * scale * (qq.abs() @ kk.abs().T)).masked_fill(mask, 0).amax(1, keepdim=True)
            top = torch.logsumexp(s, 1, keepdim=True)
            live = top > -math.inf
            p = torch.exp(s - torch.where(live, top, 0.0))
            o, w = p @ vv, p @ vv.abs()
            n = seen[:, None].double()
            t = w * (u + 2 * e_s + 2 * e_x + n * 2.0 ** -22) + u * o.abs()
            if q.dtype == torch.float16:
                t = t + n * 2.0 ** -25 * vv.abs().max() + 2.0 ** -25
            out[a:b, h], lse[a:b, h] = o, top[:, 0]
            tol[a:b, h] = torch.where(live, t + 1e-30, 0.0)
            tol_lse[a:b, h] = torch.where(live, e_s + e_x + n * 2.0 ** -23 + 2.0 ** -22 * (1 + top.abs()), 0.0)[:, 0]
    return out, lse, tol, tol_lse


def check(got, got_lse, want, lse, tol, tol_lse, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN places differ"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    fin = torch.isfinite(want)
    over = ((got - want).abs() / (tol + 1e-300))[fin]
    bad = ((got - want).abs() > tol)[fin]
    assert not bad.any(), f"{what}: {int(bad.sum())} outputs off, worst {float(over.max()):.3g} of the bound"
    if got_lse is not None:
        got_lse = got_lse.double()
        same = torch.isinf(lse)
        assert torch.equal(got_lse[same], lse[same]), f"{what}: lse of empty rows"
        fin = torch.isfinite(lse)
        off = (got_lse - lse).abs()[fin]
        assert bool((off <= tol_lse[fin]).all()), f"{what}: lse off by {float(off.max()):.3g}"


def tables(ctx, new, table, free, state, page, capacity):
    """The tables of a step in plain Python: (cu_q, kv_lens, table, slot_map, state)."""
    columns = len(table[0]) if table else 0
    table = [list(r) for r in table]
    top, missing, cu, kv, slots = min(max(0, state), len(free)), 0, [0], [], []
    for i, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(0, c), max(0, n)
        cu.append(cu[-1] + n)
        kv.append(c + n)
        for col in range(min(-(-c // page), columns), min(-(-(c + n) // page), columns)):
            if top:
                top -= 1
                table[i][col] = free[top]
            else:
                missing += 1
                table[i][col] = -1
        for p in range(c, c + n):
            held = table[i][p // page] if p // page < columns else -1
            slots.append(held * page + p % page if held >= 0 else -1)
    slots = (slots + [-1] * capacity)[:capacity]
    return cu, kv, table, slots, [top, missing]
