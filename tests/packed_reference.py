"""Plain 64-bit forms of the packed operators, and the error their kernels may have."""
import numpy as np
import torch


def starts(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int32)


def attend(q, k, v, pos, window, sinks, live=None):
    """One sequence in float64: q [n, Hq, D] at positions pos, k and v [m, Hk, D], live [m] (linked keys).
    Returns (o, a, e): the outputs, sum_j p_j |v_j|, and the largest sum_d |q_d k_jd| / sqrt(D) of each row.
    Hidden keys take no part at all, whatever they hold."""
    n, Hq, D = q.shape
    m, Hk, _ = k.shape
    q, k, v = (x.double().cpu() for x in (q, k, v))
    o, a, e = (torch.zeros(n, Hq, D, dtype=torch.float64) for _ in range(3))
    j = torch.arange(m)
    for i in range(n):
        p0 = int(pos[i])
        see = (j <= p0) & ((j < sinks) | (j > p0 - window) if window > 0 else torch.ones(m, dtype=torch.bool))
        if live is not None:
            see &= live
        if not bool(see.any()):
            continue
        for h in range(Hk):
            G = Hq // Hk
            qi, kk, vv = q[i, h * G:(h + 1) * G], k[see, h], v[see, h]
            s = qi @ kk.t() / D ** 0.5
            p = torch.softmax(s, -1)
            o[i, h * G:(h + 1) * G] = p @ vv
            a[i, h * G:(h + 1) * G] = p @ vv.abs()
            e[i, h * G:(h + 1) * G] = ((qi.abs() @ kk.abs().t()) / D ** 0.5).amax(-1, keepdim=True)
    return o, a, e


def tolerance(o, a, e, keys, D, out_dtype, p_dtype, v_rounded, scores=0.0, v_scale=0.0):
    """What the kernels' roundings may add up to, element by element.

    * the output: half a step of its type;
    * the probabilities are rounded to p_dtype in numerator and row sum: each half a step, so 2 u a at most;
      those below 2^-21 of the largest (fp16 subnormals) are off by 2^-32 of it, keys of them;
    * v_scale (over INT4 pages, up to that): what is rounded is probability times scale, and only in the
      numerator, so u a less; but relative to the largest such product, at 2^7 or more: its subnormals are off by
      2^-25 each, times a code of up to 8, over a row sum of 2^7 / v_scale or more: 2^-29 v_scale for each key;
    * v_rounded: V itself is rounded once to fp16 (code * scale): half a step of a;
    * scores: D products summed in 32 bits, two fused scalings and the running maximum: D + 16 roundings of
      e at 2^-24, which move every weight by that much relative (natural exponent), numerator and sum: twice;
    * scores: what else moves a score, absolute (quantized_scores): twice a's share again;
    * exp2 itself: 2^-22 relative, twice; the sums over the keys: at most keys 32-bit additions each.
    """
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
    t = u[out_dtype] * o.abs() + 2 * u[p_dtype] * a + (2.0 ** -11 * a if v_rounded else 0)
    t = t + 2 * (D + 16) * 2.0 ** -24 * e * a + 2 * scores * a + (2 * 2.0 ** -22 + 2 * keys * 2.0 ** -24) * a
    t = t - (u[p_dtype] * a if v_scale else 0) + keys * 2.0 ** -29 * v_scale
    return t + 2.0 ** -24 + keys * 2.0 ** -32 * a  # (2^-24: half a step of fp16's subnormals)


def quantized_scores(q, scale, staged):
    """By how much scores over INT4 keys may be off beyond the sums' own roundings, for q [n, Hq, D] and scales up
    to ``scale``. Staged chunks sum exact codes, and their factors add three roundings to those counted for the
    sums. Others sum codes that stand 1032 (or 72) too high, so that a partial sum is up to (1032 + 7) sum_d |q_d|
    before the scale, with D + 16 roundings of it at 2^-24."""
    D = q.shape[2]
    biased = 1039.0 * (D + 16) * 2.0 ** -24 * scale / D ** 0.5 * q.double().cpu().abs().sum(-1, keepdim=True)
    return 0.0 if staged else biased


def check(got, want, tol, what=""):
    g = got.double().cpu()
    assert g.shape == want.shape
    bad = ~((g - want).abs() <= tol)
    if bad.any():
        r = torch.where(bad, (g - want).abs() / tol, torch.zeros_like(tol))
        i = int(r.nan_to_num(torch.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {np.unravel_index(i, g.shape)}: "
                             f"got {g.flatten()[i]}, want {want.flatten()[i]}, may differ by {tol.flatten()[i]}")


def check_prompt(out, q, k, v, lens, window, sinks, first=0, rows=None):
    """All rows, or those of a truth tensor ``rows`` (one per row of the sequences), against the 64-bit form."""
    a = first
    D = q.shape[2]
    for n in lens:
        o, w, e = attend(q[a:a + n], k[a:a + n], v[a:a + n], np.arange(n), window, sinks)
        r = slice(None) if rows is None else rows[a - first:a - first + n]
        tol = tolerance(o, w, e, n, D, out.dtype, out.dtype, False)
        check(out[a:a + n].cpu()[r], o[r], tol[r], f"rows {a}..{a + n - 1}")
        a += n


def advance(new, ctx, tables, ring, span, bs, rows):
    """One step's index tensors, request by request: (tables, ctx, span, cu, slots, positions, status)."""
    tables, ctx = tables.copy(), ctx.copy()
    B, M = tables.shape
    C = len(ring)
    head, count = int(span[0]) % C, min(max(int(span[1]), 0), C)
    status, cu = np.zeros(B, np.int32), np.zeros(B + 1, np.int32)
    slots, positions = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    pages = asked = taken = t = 0
    for b in range(B):
        c, n = int(ctx[b]), int(new[b])
        have = -(-c // bs)
        if n < 0 or c < 0 or c + n > M * bs:
            status[b], n = 1, 0
        elif n and c % bs and tables[b, have - 1] < 0:
            status[b], n = 2, 0
        need = -(-(c + n) // bs) - have if n else 0
        pages, asked = pages + need, asked + n
        if need and pages > count:
            status[b], n = 3, 0
        elif n and asked > rows:
            status[b], n = 4, 0
        for j in range(need if n else 0):
            tables[b, have + j] = ring[(head + taken) % C]
            taken += 1
        for i in range(c, c + n):
            positions[t], slots[t] = i, int(tables[b, i // bs]) * bs + i % bs
            t += 1
        ctx[b] = c + n
        cu[b + 1] = t
    return tables, ctx, np.array([(head + taken) % C, count - taken], np.int32), cu, slots, positions, status
