"""Plain 64-bit forms of the operators that keep a cache small, and the error their kernels may have."""
import numpy as np
import torch


def visible(pos, m, window, sinks, live=None):
    """[len(pos), m]: which of m keys the queries at positions pos see."""
    p, j = torch.as_tensor(np.asarray(pos), dtype=torch.int64)[:, None], torch.arange(m)[None]
    see = j <= p
    if window > 0:
        see = see & ((j < sinks) | (j > p - window))
    return see if live is None else see & live[None]


def softmax(s, see):
    """Softmax of s over its last dimension among the visible entries; zeros where there are none."""
    s = torch.where(see, s, -torch.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:-1] + (1,))
    w = torch.where(see, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, w / total, 0.0)


def weight_sums(q, k, pos, window, sinks, live=None):
    """One sequence in float64: q [n, Hq, D] at positions pos, k [m, Hk, D]. (the weights summed over rows and group
    [Hk, m], what the kernel's roundings may add up to there).

    * a score is D products and a few scalings in 32 bits: D + 16 roundings of e = sum_d |q_d k_jd| / sqrt(D); a
      weight's exponent holds one such score and the row's lse, which is off by as much, and their difference is
      rounded once, at most e + log2(m) + 1 in size: 2 (D + 24) 2^-24 e and 4 (log2(m) + 1) 2^-24 relative;
    * two exp2 and the row's sum, merged over tiles: 4 of 2^-22 and m additions;
    * the sum over rows and group: one rounding per row of what is there so far;
    * weights below 2^-126 are gone: rows of them."""
    n, Hq, D = q.shape
    m, Hk, _ = k.shape
    G = Hq // Hk
    q, k = q.double().cpu(), k.double().cpu()
    see = visible(pos, m, window, sinks, live)
    out, tol = torch.zeros(Hk, m, dtype=torch.float64), torch.zeros(Hk, m, dtype=torch.float64)
    for h in range(Hk):
        for g in range(G):
            s = (q[:, h * G + g] @ k[:, h].t()) / D ** 0.5
            e = torch.where(see, q[:, h * G + g].abs() @ k[:, h].abs().t() / D ** 0.5, 0.0).amax(-1, keepdim=True) \
                if m else s
            w = softmax(s, see)
            out[h] += w.sum(0)
            rel = 2 * (D + 24) * 2.0 ** -24 * e + (4 * (np.log2(max(m, 2)) + 1) + m + n * G) * 2.0 ** -24 + 2.0 ** -20
            tol[h] += (w * rel).sum(0) + n * 2.0 ** -126
    return out, tol


def int4_row_bytes(t, D):
    """Offsets in a (page, head) block of everything that belongs to token t's row, except the nibble order: K and V
    code bytes, K and V scale bytes (page layout: lane 8 p + c owns tokens p, p + 8 and dims [c D / 8, (c + 1) D / 8))."""
    d = np.arange(0, D, 2)
    lane, r = 8 * (t % 8) + d // (D // 8), d % (D // 8)
    k = lane * (D // 8) + t // 8 * (D // 16) + r // 2
    v = 8 * D + lane * (D // 8) + r // 4 * 4 + t // 8 * 2 + r % 4 // 2
    s = [16 * D + part * 32 * (D // 64) + 2 * (g * 16 + 2 * (t % 8) + t // 8) + i
         for part in (0, 1) for g in range(D // 64) for i in (0, 1)]
    return np.concatenate([k, v, s])


def compact(scores, pools, fmt, tables, ctx, keep, ring, span, nb, bs, K, sinks, recent):
    """compact_cache, request by request. pools: [k, v] fp16 [nb, bs, H, D], or [pages] u8 [nb, H, bytes]; all numpy and
    copied. Returns (tables, ctx, span, scores, kept, status, ring, pools)."""
    old = pools
    pools, tables_in, scores_in = [x.copy() for x in pools], tables, scores
    tables, ctx_out, ring, scores = tables.copy(), ctx.copy(), ring.copy(), scores.copy()
    N, H, L = scores.shape
    M, C = tables.shape[1], len(ring)
    head, count = int(span[0]) % C, min(max(int(span[1]), 0), C)
    kept, status = np.full((N, H, K), -1, np.int32), np.zeros(N, np.int32)
    listed = {}
    for b in range(N):
        bad = ctx[b] < 0 or ctx[b] > M * bs or ctx[b] > L or keep[b] > K
        status[b] = 1 if bad else 0
        if not bad:
            for i in range(-(-int(ctx[b]) // bs)):
                if 0 <= tables[b, i] < nb:
                    listed.setdefault(int(tables[b, i]), []).append(b)
    shared = {b for rows in listed.values() if len(rows) > 1 for b in rows}
    asked = asked_back = taken = back = 0
    for b in range(N):
        if status[b]:
            continue
        c = int(ctx[b])
        old_pages = [int(x) for x in tables_in[b, :-(-c // bs)]]
        alive = [j for j in range(c) if 0 <= old_pages[j // bs] < nb]
        if b in shared:
            status[b] = 4
            continue
        if keep[b] < 0 or len(alive) <= keep[b]:
            status[b] = 2
            continue
        n = int(keep[b])
        linked = [x for x in old_pages if 0 <= x < nb]
        need = -(-n // bs)
        asked, asked_back = asked + need, asked_back + len(linked)
        if asked > count or asked_back > C - count:
            status[b] = 3
            continue
        fresh = [int(ring[(head + taken + i) % C]) for i in range(need)]
        taken += need
        s = min(sinks, n)
        r = min(recent, n - s)
        safe = [j for j in alive if j < s or j >= c - r]
        others = [j for j in alive if s <= j < c - r]
        row = np.zeros((H, L), np.float32)
        for h in range(H):
            order = sorted(others, key=lambda j: (np.isnan(scores_in[b, h, j]), -np.nan_to_num(scores_in[b, h, j], nan=0.0, posinf=np.inf, neginf=-np.inf), j))
            got = sorted(safe + order[:n - len(safe)])
            kept[b, h, :n] = got
            row[h, :n] = scores_in[b, h, got]
            for i, j in enumerate(got):
                if not 0 <= fresh[i // bs] < nb:
                    continue
                if fmt == "fp16":
                    for x, y in zip(pools, old):
                        x[fresh[i // bs], i % bs, h] = y[old_pages[j // bs], j % bs, h]
                else:
                    D = 128 if pools[0].shape[2] == 2176 else 64
                    pools[0][fresh[i // bs], h, int4_row_bytes(i % bs, D)] = old[0][old_pages[j // bs], h, int4_row_bytes(j % bs, D)]
        for x in linked:
            ring[(head + count + back) % C] = x
            back += 1
        tables[b] = -1
        tables[b, :need] = fresh
        ctx_out[b] = n
        scores[b] = row
    return tables, ctx_out, np.array([(head + taken) % C, count - taken + back], np.int32), scores, kept, status, ring, pools


def latent(q, c, pos, rank, scale, window, sinks, live=None):
    """One sequence in float64: q [n, Hq, W] at positions pos, c [m, W]. (o [n, Hq, rank], sum_j p_j |c_j|, and the largest
    scale sum_d |q_d c_jd| of each row, as packed_reference.tolerance takes them.) Hidden tokens take no part at all."""
    n, Hq, W = q.shape
    m = c.shape[0]
    q, c = q.double().cpu(), c.double().cpu()
    see = visible(pos, m, window, sinks, live)
    c = torch.where(see.any(0)[:, None], c, 0.0) if m else c
    o, a, e = (torch.zeros(n, Hq, rank, dtype=torch.float64) for _ in range(3))
    for h in range(Hq):
        if not m:
            break
        w = torch.zeros(n, m, dtype=torch.float64)
        for i in range(n):
            j = see[i].nonzero()[:, 0]
            if j.numel():
                w[i, j] = torch.softmax(scale * (c[j] @ q[i, h]), 0)
                o[i, h], a[i, h] = w[i, j] @ c[j, :rank], w[i, j] @ c[j, :rank].abs()
                e[i, h] = (abs(scale) * (c[j].abs() @ q[i, h].abs())).max()
    return o, a, e


def latent_tolerance(o, a, e, keys, W, dtype):
    """packed_reference.tolerance with W products in a score; the kernel's merges of partial sums add one factor of an
    exp2 (2^-22) and one rounding each to numerator and denominator, of at most `keys` / 64 parts."""
    from packed_reference import tolerance
    return tolerance(o, a, e, keys, W, dtype, dtype, False) + 2 * (2.0 ** -22 + (keys / 64 + 1) * 2.0 ** -24) * a
