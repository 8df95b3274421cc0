"""Performance cases of a cache that is kept small: eviction by accumulated attention weight, and latent attention.

A case is one call that a serving program makes per layer:

* ``scores``: the attention weights that packed queries give the tokens of a paged cache (4-bit or fp16 keys,
  grouped heads), summed over the queries and the heads of a group and added to what earlier steps gave them;
* ``compact``: the tokens of least weight leave the cache: the others move to fresh pages of the free ring in their
  order, head by head, and the old pages go back to it;
* ``latent``: attention of packed queries over a paged cache that holds one vector per token for all heads
  (keys of its whole width, values its first ``rank`` elements): the absorbed form;
* ``expanded``: causal attention over whole packed prompts with keys of a per-head part and a rotary part shared by
  all heads: the form in which a latent model reads its prompts.

``own`` chooses between the framework's operators and their plain forms (elementary torch operations in 32 bits).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "memopt-transformer-runtime_amd")


def _memopt():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import memopt_C
    return memopt_C


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _scores(**kw):
    case = dict(kind="scores", layout="int4", seqs=1, ctx=4096, ragged=False, heads=32, kv_heads=8, dim=128, window=-1,
                sinks=0, chunk=1, chunks=0)
    case.update(kw)
    return case


def _compact(**kw):
    case = dict(kind="compact", layout="int4", seqs=1, ctx=4096, ragged=False, kv_heads=8, dim=128, keep=1024, sinks=4,
                recent=64)
    case.update(kw)
    return case


def _latent(**kw):
    case = dict(kind="latent", dtype="bf16", seqs=1, ctx=4096, ragged=False, heads=16, rank=512, rope=64, window=-1,
                sinks=0, chunk=1, chunks=0)
    case.update(kw)
    return case


def _expanded(**kw):
    case = dict(kind="expanded", dtype="bf16", seqs=1, longest=1024, shortest=0, heads=16, dim=128, rope=64, window=-1,
                sinks=0)
    case.update(kw)
    return case


def listed():
    return [
        # One user on a small model (8 query heads of 64 on 2 key heads), one token: the latency of one call.
        _scores(name="scores_one", ctx=1024, heads=8, kv_heads=2, dim=64),
        # A served batch's decode step that keeps count: 32 sequences of unequal length up to 8192.
        _scores(name="scores_batch", seqs=32, ctx=8192, ragged=True),
        # What the end of a prompt looks at: 4 prompts in the default (fp16) cache, the last 512 tokens of each.
        _scores(name="scores_chunk", layout="fp16", seqs=4, ctx=6000, ragged=True, chunk=512, chunks=4),
        # One short request of a small model is cut to a quarter: latency.
        _compact(name="compact_one", ctx=1024, kv_heads=2, dim=64, keep=256, recent=32),
        # A batch under memory pressure: 16 requests of up to 8192 tokens are cut to 2048 at most.
        _compact(name="compact_batch", seqs=16, ctx=8192, ragged=True, keep=2048),
        # One user's long context in the default (fp16) cache: 16384 tokens, half of them stay.
        _compact(name="compact_fp16", layout="fp16", ctx=16384, keep=8192, recent=256),
        # One user on a small latent model: latency.
        _latent(name="latent_one", dtype="fp16", ctx=1024, heads=8, rank=256, rope=32),
        # The ordinary decode step: 32 sequences of unequal length up to 8192, 16 heads.
        _latent(name="latent_batch", seqs=32, ctx=8192, ragged=True),
        # Many heads over one latent: 16 sequences, 128 heads, where products count as much as bytes.
        _latent(name="latent_heads", seqs=16, ctx=8192, ragged=True, heads=128),
        # Continuous batching: 12 sequences, 3 of them with the next 256 tokens of their prompts.
        _latent(name="latent_mixed", seqs=12, ctx=6000, ragged=True, chunk=256, chunks=3),
        # A batch of prompts as they arrive: 24 of 20 to 2500 tokens, packed.
        _expanded(name="expanded_packed", seqs=24, longest=2500, shortest=20),
        # Long documents: 3 prompts of up to 9000 tokens, 32 heads.
        _expanded(name="expanded_long", dtype="fp16", seqs=3, longest=9000, shortest=400, heads=32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scores", "scores", "compact", "compact", "latent", "latent", "latent", "expanded", "expanded"])
    window = rng.choice([-1, -1, -1, 512, 1024, 2048, 4096])
    sinks = rng.choice([0, 4, 16]) if window > 0 else 0
    many = rng.random() < 0.4
    if kind in ("scores", "compact"):
        heads, kv_heads, dim = rng.choice([(8, 2, 64), (12, 4, 64), (8, 8, 64), (20, 4, 64), (8, 1, 128), (32, 8, 128),
                                           (32, 8, 128), (40, 8, 128), (32, 4, 128)])
        layout = rng.choice(["int4", "int4", "fp16"])
        seqs = _log_int(rng, 1, 64)
        most = 4800 if many and kind == "scores" else 65536 if layout == "int4" else 16384
        ctx = _log_int(rng, 64, min(most, 2 ** 20 // (seqs * kv_heads)))
        ragged = rng.random() < 0.7
        if kind == "scores":
            return _scores(layout=layout, seqs=seqs, ctx=ctx, ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim,
                           window=window, sinks=sinks, chunk=_log_int(rng, 2, min(512, ctx // 3)) if many else 1,
                           chunks=rng.randint(1, min(seqs, 4)) if many else 0)
        keep = _log_int(rng, 16, ctx)
        return _compact(layout=layout, seqs=seqs, ctx=ctx, ragged=ragged, kv_heads=kv_heads, dim=dim, keep=keep,
                        sinks=rng.choice([0, 4, 4, 16]), recent=_log_int(rng, 1, max(1, keep // 2)))
    if kind == "latent":
        rank, rope = rng.choice([(512, 64), (512, 64), (256, 64), (256, 32), (128, 32), (512, 32), (128, 64)])
        heads = rng.choice([5, 8, 16, 16, 32, 64, 128])
        seqs = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 64, min(65536, 2 ** 21 // (seqs * heads), 2 ** 17 // heads if many else 65536))
        return _latent(dtype=rng.choice(["fp16", "bf16"]), seqs=seqs, ctx=ctx, ragged=rng.random() < 0.7, heads=heads,
                       rank=rank, rope=rope, window=window, sinks=sinks,
                       chunk=_log_int(rng, 2, min(256, ctx // 3)) if many else 1,
                       chunks=rng.randint(1, min(seqs, 3)) if many else 0)
    seqs = rng.choice([1, 1, 2, 5, 16, 60])
    longest = _log_int(rng, 16, int(9000 / math.sqrt(seqs)))
    return _expanded(dtype=rng.choice(["fp16", "bf16"]), seqs=seqs, longest=longest,
                     shortest=_log_int(rng, 1, longest) if seqs > 1 else 0, heads=rng.choice([5, 8, 16, 32]),
                     dim=rng.choice([64, 128, 128]), rope=rng.choice([32, 64, 64]), window=window, sinks=sinks)


# ---------------------------------------------------------------------------
# Inputs (from the seed alone)
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, g, dtype, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype).mul_(std)


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _lens(case):
    """(context lengths, query counts): contexts between a third of ctx and ctx; the first `chunks` sequences
    bring a chunk of queries, the others one."""
    n, ctx = case["seqs"], case["ctx"]
    lens = [ctx - (i * 977 + 13) % max(1, 2 * ctx // 3) if case["ragged"] and i else ctx for i in range(n)]
    return lens, [case["chunk"] if i < case.get("chunks", 0) else 1 for i in range(n)]


def _prompt_lens(case):
    """From the longest down to the shortest prompt, evenly in the logarithm, in a mixed order (no case has a
    multiple of 7 prompts)."""
    n, hi, lo = case["seqs"], case["longest"], case["shortest"]
    if n == 1:
        return [hi]
    return [int(round(hi * (lo / hi) ** ((i * 7 + 3) % n / (n - 1)))) for i in range(n)]


def _int4_groups(x):
    """Group-64 codes 0 .. 15 and fp16 scales of x [..., D]."""
    xf = x.float().unflatten(-1, (-1, 64))
    s = xf.abs().amax(-1, keepdim=True) / 7.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    codes = (xf / s).round_().add_(8.0).clamp_(0, 15).to(torch.uint8).flatten(-2)
    return codes, s.squeeze(-1).half()


def _pack(codes, part):
    """Page bytes [n, heads, 8 dim] of codes [n, heads, 16, dim] of part 0 (K) or 1 (V).

    Lane 8 p + c of a (page, head) block owns tokens p and p + 8 and the dims [c dim / 8, (c + 1) dim / 8): its K
    bytes are token p's and then token p + 8's, its V bytes two of each in turn (4 dims).
    """
    n, heads, _, dim = codes.shape
    byte = codes[..., 0::2] | (codes[..., 1::2] << 4)
    byte = byte.view(n, heads, 2, 8, 8, dim // 32, 2)                             # half, p, c, unit of 4 dims, byte
    byte = byte.permute(0, 1, 3, 4, 2, 5, 6) if part == 0 else byte.permute(0, 1, 3, 4, 5, 2, 6)
    return byte.reshape(n, heads, 8 * dim)


def _unpack(byte, part):
    """The codes [n, heads, 16, dim] of page bytes [n, heads, 8 dim]."""
    n, heads, b = byte.shape
    dim = b // 8
    code = torch.stack([byte & 15, byte >> 4], -1)
    if part == 0:
        code = code.view(n, heads, 8, 8, 2, dim // 32, 2, 2).permute(0, 1, 4, 2, 3, 5, 6, 7)
    else:
        code = code.view(n, heads, 8, 8, dim // 32, 2, 2, 2).permute(0, 1, 5, 2, 3, 4, 6, 7)
    return code.reshape(n, heads, 16, dim)


def _regions(blocks, part):
    """(codes [n, heads, 16, dim], scales [n, heads, 16, groups]) of INT4 blocks [n, heads, bytes]; scales lie by
    group, then p, then token half."""
    n, heads, size = blocks.shape
    groups = 1 if size == 16 * 64 + 64 else 2
    dim = 64 * groups
    codes = _unpack(blocks[:, :, part * 8 * dim:(part + 1) * 8 * dim].contiguous(), part)
    o = 16 * dim + part * 32 * groups
    scale = blocks[:, :, o:o + 32 * groups].contiguous().view(torch.float16)
    return codes, scale.view(n, heads, groups, 8, 2).permute(0, 1, 4, 3, 2).reshape(n, heads, 16, groups)


def _set_regions(blocks, part, codes, scales):
    n, heads, _, dim = codes.shape
    groups = dim // 64
    blocks[:, :, part * 8 * dim:(part + 1) * 8 * dim] = _pack(codes, part)
    sc = scales.reshape(n, heads, 2, 8, groups).permute(0, 1, 4, 3, 2).reshape(n, heads, 16 * groups).contiguous()
    o = 16 * dim + part * 32 * groups
    blocks[:, :, o:o + 32 * groups] = sc.view(torch.uint8)


def _int4_pages(pages, heads, dim, g):
    """A pool of INT4 pages [pages, heads, 16 dim + 64 (dim / 64)] of normal keys and values with 1 % of outliers:
    a (page, head) block holds K codes, V codes, K scales and V scales."""
    buf = torch.empty((pages, heads, 16 * dim + dim), dtype=torch.uint8, device=DEV)
    step = max(1, 2 ** 26 // (16 * heads * dim))
    for p0 in range(0, pages, step):
        n = min(step, pages - p0)
        for part in (0, 1):
            x = _normal((n, heads, 16, dim), g, torch.float16)
            x.mul_(torch.rand(x.shape, generator=g, device=DEV, dtype=torch.float16).lt_(0.01).mul_(7.0).add_(1.0))
            _set_regions(buf[p0:p0 + n], part, *_int4_groups(x))
    return buf


def _paged_inputs(case, seed):
    """What the cases over a paged cache share: lengths, tables of shuffled pages, and the generator."""
    g = _gen(seed)
    ctx, qn = _lens(case)
    per = (max(ctx) + 15) // 16
    bt = torch.randperm(case["seqs"] * per, generator=g, device=DEV).to(torch.int32).view(case["seqs"], per)
    return g, dict(case=case, ctx=ctx, qn=qn, bt=bt, cl=_i32(ctx), cu=_i32(_starts(qn)))


def _scores_inputs(case, seed):
    g, st = _paged_inputs(case, seed)
    Hk, D, nb = case["kv_heads"], case["dim"], st["bt"].numel()
    st["kc"] = _int4_pages(nb, Hk, D, g) if case["layout"] == "int4" else _normal((nb, 16, Hk, D), g, torch.float16)
    st["q"] = _normal((sum(st["qn"]), case["heads"], D), g, torch.float16)
    # what earlier steps gave, as much as about one of them
    st["scores"] = torch.rand((case["seqs"], Hk, max(st["ctx"])), generator=g, device=DEV)
    st["scores"].mul_(2 * case["heads"] / Hk * case["chunk"] / case["ctx"])
    return st


def _compact_inputs(case, seed):
    g = _gen(seed)
    n, Hk, D = case["seqs"], case["kv_heads"], case["dim"]
    ctx, _ = _lens(case)
    have, want = ([(c + 15) // 16 for c in x] for x in (ctx, [min(case["keep"], c) for c in ctx]))
    M = max(have) + 4
    nb = sum(have) + sum(want) + 5
    pages = torch.randperm(nb, generator=g, device=DEV).to(torch.int32).cpu().numpy()
    tables = np.full((n, M), -1, np.int32)
    at = 0
    for b in range(n):
        tables[b, :have[b]] = pages[at:at + have[b]]
        at += have[b]
    ring = np.full(nb, -1, np.int32)
    head = int(seed) * 7919 % nb
    ring[(head + np.arange(nb - at)) % nb] = pages[at:]
    st = dict(case=case, ctx=ctx, bt=_i32(tables), cl=_i32(ctx), ring=_i32(ring), span=_i32([head, nb - at]),
              keep=_i32([case["keep"]] * n))
    if case["layout"] == "int4":
        st["kc"] = st["vc"] = _int4_pages(nb, Hk, D, g)
    else:
        st["kc"], st["vc"] = (_normal((nb, 16, Hk, D), g, torch.float16) for _ in range(2))
    # Accumulated weights: a few tokens have most of them, some none at all (ties).
    w = torch.exp(2.0 * torch.randn((n, Hk, M * 16), generator=g, device=DEV))
    w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.1, 0.0, w)
    st["scores"] = torch.where(torch.arange(M * 16, device=DEV) < st["cl"][:, None, None], w, 0.0)
    return st


def _latent_inputs(case, seed):
    g, st = _paged_inputs(case, seed)
    width = case["rank"] + case["rope"]
    st["c"] = _normal((st["bt"].numel(), 16, width), g, _dtype(case))
    st["q"] = _normal((sum(st["qn"]), case["heads"], width), g, _dtype(case))
    # (the scale of a head's own width of 128 and the rotary part)
    st["scale"] = (128 + case["rope"]) ** -0.5
    return st


def _expanded_inputs(case, seed):
    g = _gen(seed)
    lens = _prompt_lens(case)
    T, H, D, P = sum(lens), case["heads"], case["dim"], case["rope"]
    # keys and values as the up-projection of the latents leaves them, side by side in each head
    kv = _normal((T, H, 2 * D), g, _dtype(case))
    return dict(case=case, lens=lens, q=_normal((T, H, D + P), g, _dtype(case)), k=kv[:, :, :D], v=kv[:, :, D:],
                kr=_normal((T, P), g, _dtype(case)), cu=_i32(_starts(lens)))


def prepare(case, seed):
    if case["kind"] == "scores":
        st = _scores_inputs(case, seed)
        if own:
            # (sums go to a buffer of their own here, so that every pass starts from the same ones)
            st["sums"] = torch.empty_like(st["scores"])
        return st
    if case["kind"] == "compact":
        st = _compact_inputs(case, seed)
        if own:
            st["out"] = _memopt().compact_cache_buffers(case["seqs"], case["kv_heads"], st["bt"].shape[1],
                                                        st["scores"].shape[2], case["keep"], st["bt"].device)
        return st
    return _latent_inputs(case, seed) if case["kind"] == "latent" else _expanded_inputs(case, seed)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return {"scores": _run_scores, "compact": _run_compact, "latent": _run_latent,
            "expanded": _run_expanded}[state["case"]["kind"]](state)


def _softmax_rows(s, hidden):
    """softmax of s over its last dimension without the hidden entries; zeros where all are hidden."""
    s = s.masked_fill(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _hidden(pos, keys, window, sinks):
    """[queries, keys]: key j is hidden from the query at position i unless j <= i and (j < sinks or j > i - window)."""
    i, j = pos[:, None], torch.arange(keys, device=DEV)[None]
    see = j <= i
    if window > 0:
        see = see & ((j < sinks) | (j > i - window))
    return ~see


def _run_scores(st):
    case = st["case"]
    if own:
        return _memopt().attention_scores(st["q"], st["kc"], st["bt"], st["cl"], st["cu"], max(st["qn"]),
                                          max(st["ctx"]), case["window"], num_sink_tokens=case["sinks"],
                                          scores=st["scores"], out=st["sums"])
    out = st["scores"].clone()
    Hk, D, G = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    a = 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["qn"])):
        pages = st["kc"][st["bt"][b, :(c + 15) // 16].long()]
        if case["layout"] == "int4":
            codes, scales = _regions(pages, 0)
            k = (codes.float() - 8.0).unflatten(-1, (-1, 64)) * scales.float().unsqueeze(-1)
            k = k.flatten(-2).permute(1, 3, 0, 2)                                  # [Hk, D, pages, 16]
        else:
            k = pages.float().permute(2, 3, 0, 1)
        k = k.reshape(Hk, D, -1)[:, :, :c].contiguous()
        for i0 in range(0, n, 128):
            i1 = min(n, i0 + 128)
            rows = st["q"][a + i0:a + i1].float().view(i1 - i0, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)
            s = torch.matmul(rows, k).view(Hk, G, i1 - i0, c) / math.sqrt(D)
            pos = torch.arange(c - n + i0, c - n + i1, device=DEV)
            out[b, :, :c] += _softmax_rows(s, _hidden(pos, c, case["window"], case["sinks"])).sum((1, 2))
        a += n
    return out


def _run_compact(st):
    case = st["case"]
    if own:
        r = _memopt().compact_cache(st["scores"], st["kc"], st["vc"], st["bt"], st["cl"], st["keep"], st["ring"],
                                    st["span"], num_sink_tokens=case["sinks"], num_recent_tokens=case["recent"],
                                    out=st["out"])
        return [r.block_tables, r.context_lens, r.free_span, r.scores, r.kept, r.status, st["ring"], st["kc"], st["vc"]]
    N, M = st["bt"].shape
    Hk, L, K, C = case["kv_heads"], st["scores"].shape[2], case["keep"], st["ring"].shape[0]
    head, count = st["span"][0].long(), st["span"][1].long()
    ctx, keep = st["cl"].long(), st["keep"].long()
    have, n = (ctx + 15) // 16, torch.minimum(keep, ctx)
    # who is compacted: those with more tokens than they may keep, while the free pages last
    asks = ctx > keep
    need = torch.where(asks, (n + 15) // 16, 0)
    short = asks & (torch.cumsum(need, 0) > count)
    moved = asks & ~short
    status = torch.where(short, 3, torch.where(moved, 0, 2))
    need = torch.where(moved, need, 0)
    back = torch.where(moved, have, 0)
    # which tokens: sinks, the last ones, then the largest scores (ties: the first)
    j = torch.arange(L, device=DEV)
    sink = torch.clamp(n, max=case["sinks"])
    recent = torch.minimum(n - sink, torch.full_like(n, case["recent"]))
    safe = (j < sink[:, None]) | ((j >= (ctx - recent)[:, None]) & (j < ctx[:, None]))
    key = st["scores"].masked_fill(safe[:, None], math.inf).masked_fill((j >= ctx[:, None])[:, None], -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order).contiguous())
    first = torch.sort(torch.where(rank < n[:, None, None], j.expand_as(rank), L), dim=-1).values[:, :, :K]
    i = torch.arange(K, device=DEV)
    live = (i < n[:, None])[:, None] & moved[:, None, None]
    kept = torch.where(live, first, -1)
    src = kept.clamp(min=0)
    scores = torch.zeros_like(st["scores"])
    scores[:, :, :K] = torch.where(live, st["scores"].gather(-1, src), 0.0)
    scores = torch.where(moved[:, None, None], scores, st["scores"])
    # pages
    col = torch.arange(M, device=DEV)[None]
    at = torch.cumsum(need, 0) - need
    fresh = st["ring"][(head + at[:, None] + col) % C]
    tables = torch.where(moved[:, None], torch.where(col < need[:, None], fresh, -1), st["bt"])
    where = torch.where(moved[:, None] & (col < have[:, None]),
                        (head + count + (torch.cumsum(back, 0) - back)[:, None] + col) % C, C)
    ring = torch.cat([st["ring"], st["ring"].new_zeros(1)]).scatter_(0, where.flatten(), st["bt"].flatten())[:C]
    st["ring"].copy_(ring)
    span = torch.stack([(head + need.sum()) % C, count - need.sum() + back.sum()])
    # rows
    Kp = (K + 15) // 16 * 16
    src = torch.nn.functional.pad(src, (0, Kp - K))
    live = torch.nn.functional.pad(live, (0, Kp - K))
    page = st["bt"].gather(1, (src // 16).flatten(1)).view_as(src).long()                       # [N, Hk, Kp]
    new = torch.where(col[:, :Kp // 16] < need[:, None], tables[:, :Kp // 16], st["kc"].shape[0]).long()
    for b in range(N):
        m = Kp // 16 if st["ctx"][b] > K else 0                # (the free pages suffice for all of them here)
        if m == 0:
            continue
        to = new[b, :m]                                                                         # fresh pages
        p, t, ok = (x[b, :, :16 * m] for x in (page, src % 16, live))
        h = torch.arange(Hk, device=DEV)[:, None]
        if case["layout"] == "fp16":
            for pool in (st["kc"], st["vc"]):
                rows = torch.where(ok[..., None], pool[p, t, h], pool[to].permute(2, 0, 1, 3).reshape(Hk, 16 * m, -1))
                pool[to] = rows.view(Hk, m, 16, -1).permute(1, 2, 0, 3)
        else:
            old = st["bt"][b, :int(st["ctx"][b] + 15) // 16].long()
            blocks, target = st["kc"][old], st["kc"][to]
            f = src[b, :, :16 * m].unsqueeze(-1)
            for part in (0, 1):
                got = []
                for x, y in zip(_regions(blocks, part), _regions(target, part)):
                    x, y = (z.permute(1, 0, 2, 3).flatten(1, 2) for z in (x, y))                # [Hk, tokens, .]
                    z = torch.where(ok[..., None], x.gather(1, f.expand(-1, -1, x.shape[-1])), y)
                    got.append(z.view(Hk, m, 16, -1).permute(1, 0, 2, 3))
                _set_regions(target, part, *got)
            st["kc"][to] = target
    i32 = torch.int32
    return [tables, torch.where(moved, n, ctx).to(i32), span.to(i32), scores, kept.to(i32), status.to(i32), st["ring"],
            st["kc"], st["vc"]]


def _run_latent(st):
    case = st["case"]
    if own:
        return _memopt().latent_attention(st["q"], st["c"], st["bt"], st["cl"], st["cu"], max(st["qn"]), max(st["ctx"]),
                                          st["scale"], case["rank"], case["window"], num_sink_tokens=case["sinks"])
    H, R = case["heads"], case["rank"]
    out = torch.empty((st["q"].shape[0], H, R), dtype=st["q"].dtype, device=DEV)
    a = 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["qn"])):
        x = st["c"][st["bt"][b, :(c + 15) // 16].long()].flatten(0, 1)[:c].float()
        xt = x.t().contiguous()
        for i0 in range(0, n, 64):
            i1 = min(n, i0 + 64)
            s = (st["q"][a + i0:a + i1].float().flatten(0, 1) @ xt).view(i1 - i0, H, c) * st["scale"]
            pos = torch.arange(c - n + i0, c - n + i1, device=DEV)
            p = _softmax_rows(s, _hidden(pos, c, case["window"], case["sinks"])[:, None])
            out[a + i0:a + i1] = (p.flatten(0, 1) @ x[:, :R]).view(i1 - i0, H, R).to(out.dtype)
        a += n
    return out


def _run_expanded(st):
    case = st["case"]
    if own:
        return _memopt().latent_prompt_attention(st["q"], st["k"], st["kr"], st["v"], st["cu"], case["window"],
                                                 num_sink_tokens=case["sinks"])
    H, D, P = case["heads"], case["dim"], case["rope"]
    out = torch.empty((st["q"].shape[0], H, D), dtype=st["q"].dtype, device=DEV)
    a = 0
    for n in st["lens"]:
        k = torch.cat([st["k"][a:a + n].float(), st["kr"][a:a + n].float()[:, None].expand(-1, H, -1)], -1)
        k = k.permute(1, 2, 0).contiguous()
        v = st["v"][a:a + n].float().permute(1, 0, 2).contiguous()
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            q = st["q"][a + i0:a + i1].float().permute(1, 0, 2)
            s = torch.matmul(q, k[:, :, :i1].contiguous()) / math.sqrt(D + P)
            p = _softmax_rows(s, _hidden(torch.arange(i0, i1, device=DEV), i1, case["window"], case["sinks"]))
            out[a + i0:a + i1] = torch.matmul(p, v[:, :i1].contiguous()).permute(1, 0, 2).to(out.dtype)
        a += n
    return out


# ---------------------------------------------------------------------------
# Least work
# ---------------------------------------------------------------------------

def _pairs(first, n, window, sinks):
    """Visible (query, key) pairs of queries at positions first .. first + n - 1."""
    pos = np.arange(first, first + n, dtype=np.float64)
    if window <= 0:
        return float((pos + 1).sum())
    behind = np.maximum(0, pos + 1 - window)
    return float((pos + 1 - behind + np.minimum(behind, sinks)).sum())


def work(case):
    if case["kind"] == "expanded":
        lens = _prompt_lens(case)
        H, D, P = case["heads"], case["dim"], case["rope"]
        pairs = sum(_pairs(0, n, case["window"], case["sinks"]) for n in lens)
        return {"bytes": 2 * sum(lens) * (H * (4 * D + P) + P), "flops": 2 * (2 * D + P) * H * pairs}
    ctx, qn = _lens(case)
    if case["kind"] == "compact":
        Hk, D, sinks = case["kv_heads"], case["dim"], case["sinks"]
        per_token = Hk * (4 * D if case["layout"] == "fp16" else D + 4 * (D // 64))
        L = (max((c + 15) // 16 for c in ctx) + 4) * 16
        bytes_ = 0
        for c in ctx:
            n = min(case["keep"], c)
            bytes_ += 4 * Hk * (c + L)                                  # scores, whole rows written
            if c > n:
                bytes_ += n * (2 * per_token + 4 * Hk) + 8 * ((n + 15) // 16 + (c + 15) // 16)
        return {"bytes": bytes_, "flops": 0}
    bytes_, pairs = 0, 0.0
    if case["kind"] == "scores":
        Hk, D, Hq = case["kv_heads"], case["dim"], case["heads"]
        per_token = Hk * (2 * D if case["layout"] == "fp16" else D // 2 + 2 * (D // 64))
        per_row, per_pair = 2 * Hq * D, 2 * D * Hq
        bytes_ += 8 * case["seqs"] * Hk * max(ctx)
    else:
        width = case["rank"] + case["rope"]
        per_token, per_row = 2 * width, 2 * case["heads"] * (width + case["rank"])
        per_pair = 2 * (width + case["rank"]) * case["heads"]
    for c, n in zip(ctx, qn):
        seen = c
        if case["window"] > 0:
            seen = min(c, n + case["window"] - 1)
            seen += min(case["sinks"], c - seen)
        bytes_ += seen * per_token + n * per_row + 4 * ((seen + 15) // 16)
        pairs += _pairs(c - n, n, case["window"], case["sinks"])
    return {"bytes": bytes_, "flops": per_pair * pairs}


# ---------------------------------------------------------------------------
# 64-bit results from the operators' definitions
# ---------------------------------------------------------------------------

def _weights(q, k, pos, scale, window, sinks):
    """float64 softmax weights [rows, keys] of queries q [rows, d] at positions pos [rows] over keys k [keys, d]."""
    j = torch.arange(k.shape[0], device=DEV)
    see = j[None] <= pos[:, None]
    if window > 0:
        see &= (j[None] < sinks) | (pos[:, None] - j[None] < window)
    s = torch.where(see, q @ k.t().contiguous() * scale, float("-inf"))
    w = torch.where(see, torch.exp(s - s.max(1, keepdim=True).values), 0.0)
    total = w.sum(1, keepdim=True)
    return torch.where(total > 0, w / total, 0.0)


def _exact_scores(case, seed):
    st = _scores_inputs(case, seed)
    D, G = case["dim"], case["heads"] // case["kv_heads"]
    if case["layout"] == "int4":
        token, dim = np.meshgrid(np.arange(16), np.arange(D), indexing="ij")
        lane = 8 * (token % 8) + dim // (D // 8)
        byte = lane * (D // 8) + token // 8 * (D // 16) + dim % (D // 8) // 2
        at = 16 * D + 2 * (dim // 64 * 16 + 2 * (token % 8) + token // 8)
        byte, at, low = (torch.from_numpy(x).to(DEV) for x in (byte, at, dim % 2 == 0))
    out, a = st["scores"].double(), 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["qn"])):
        pages = st["bt"][b, :(c + 15) // 16].long()
        for h in range(case["kv_heads"]):
            if case["layout"] == "int4":
                blk = st["kc"][pages, h]
                code = torch.where(low, blk[:, byte] & 15, blk[:, byte] >> 4).double() - 8
                scale = torch.stack([blk[:, at], blk[:, at + 1]], -1).contiguous().view(torch.float16)[..., 0]
                k = (code * scale.double()).reshape(-1, D)[:c]
            else:
                k = st["kc"][pages, :, h].reshape(-1, D)[:c].double()
            pos = torch.arange(c - n, c, device=DEV)
            for g in range(G):
                w = _weights(st["q"][a:a + n, h * G + g].double(), k, pos, D ** -0.5, case["window"], case["sinks"])
                out[b, h, :c] += w.sum(0)
        a += n
    return out


def _exact_compact(case, seed):
    st = _compact_inputs(case, seed)
    tables, ring, sc = (st[x].cpu().numpy().copy() for x in ("bt", "ring", "scores"))
    head, count = (int(x) for x in st["span"].cpu())
    N, Hk, L = sc.shape
    K, C, D = case["keep"], ring.size, case["dim"]
    kept, status, lens = np.full((N, Hk, K), -1, np.int32), np.zeros(N, np.int32), np.array(st["ctx"], np.int32)
    kc = st["kc"].clone()
    vc = kc if case["layout"] == "int4" else st["vc"].clone()
    asked = taken = back = 0
    if case["layout"] == "int4":
        # a row's bytes in its block: per dim the nibble's place, per group the scale's
        def place(t, d, part):
            lane, r = 8 * (t % 8) + d // (D // 8), d % (D // 8)
            if part == 0:
                return lane * (D // 8) + t // 8 * (D // 16) + r // 2
            return 8 * D + lane * (D // 8) + r // 4 * 4 + t // 8 * 2 + r % 4 // 2

        places = np.zeros((16, D + 4 * (D // 64)), np.int64)
        for t in range(16):
            x = [place(t, d, part) for part in (0, 1) for d in range(0, D, 2)]
            for part in (0, 1):
                for g in range(D // 64):
                    o = 16 * D + part * 32 * (D // 64) + 2 * (g * 16 + 2 * (t % 8) + t // 8)
                    x += [o, o + 1]
            places[t] = x
        places = torch.from_numpy(places).to(DEV)
    for b in range(N):
        c = int(lens[b])
        if c <= K:
            status[b] = 2
            continue
        need, old = -(-K // 16), tables[b, :-(-c // 16)].copy()
        asked += need
        if asked > count:
            status[b] = 3
            continue
        fresh = ring[(head + taken + np.arange(need)) % C].copy()
        taken += need
        sinks = min(case["sinks"], K)
        recent = min(case["recent"], K - sinks)
        free = np.arange(sinks, c - recent)
        row = np.zeros((Hk, L), np.float32)
        for h in range(Hk):
            best = free[np.argsort(-sc[b, h, free], kind="stable")[:K - sinks - recent]]
            kept[b, h] = np.sort(np.concatenate([np.arange(sinks), best, np.arange(c - recent, c)]))
            row[h, :K] = sc[b, h, kept[b, h]]
            src = torch.from_numpy(kept[b, h].astype(np.int64)).to(DEV)
            dst = torch.arange(K, device=DEV)
            p0, p1 = (torch.from_numpy(x.astype(np.int64)).to(DEV)[y // 16] for x, y in ((old, src), (fresh, dst)))
            if case["layout"] == "int4":
                kc[p1[:, None], h, places[dst % 16]] = st["kc"][p0[:, None], h, places[src % 16]]
            else:
                kc[p1, dst % 16, h] = st["kc"][p0, src % 16, h]
                vc[p1, dst % 16, h] = st["vc"][p0, src % 16, h]
        sc[b] = row
        ring[(head + count + back + np.arange(old.size)) % C] = old
        back += old.size
        tables[b] = -1
        tables[b, :need] = fresh
        lens[b] = K
    span = np.array([(head + taken) % C, count - taken + back], np.int32)
    return [torch.from_numpy(x) for x in (tables, lens, span, sc.astype(np.float64), kept, status, ring)] + [kc, vc]


def _exact_latent(case, seed):
    st = _latent_inputs(case, seed)
    H, R = case["heads"], case["rank"]
    out, a = [], 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["qn"])):
        x = st["c"][st["bt"][b, :(c + 15) // 16].long()].reshape(-1, st["c"].shape[2])[:c].double()
        seq = []
        for i in range(0, n, 16):
            m = min(16, n - i)
            pos = torch.arange(c - n + i, c - n + i + m, device=DEV).repeat_interleave(H)
            w = _weights(st["q"][a + i:a + i + m].double().reshape(m * H, -1), x, pos, st["scale"], case["window"],
                         case["sinks"])
            seq.append((w @ x[:, :R].contiguous()).view(m, H, R))
        out += seq
        a += n
    return torch.cat(out)


def _exact_expanded(case, seed):
    st = _expanded_inputs(case, seed)
    H, D, P = case["heads"], case["dim"], case["rope"]
    out, a = torch.zeros((st["q"].shape[0], H, D), dtype=torch.float64, device=DEV), 0
    for n in st["lens"]:
        for h in range(H):
            k = torch.cat([st["k"][a:a + n, h], st["kr"][a:a + n]], -1).double()
            v = st["v"][a:a + n, h].double()
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                w = _weights(st["q"][a + i:a + i + m, h].double(), k, torch.arange(i, i + m, device=DEV),
                             (D + P) ** -0.5, case["window"], case["sinks"])
                out[a + i:a + i + m, h] = w @ v
        a += n
    return out


def exact(case, seed):
    # (products of the full, unmasked score matrices; some 10 TFLOP are 20 seconds)
    if case["kind"] == "expanded":
        cost = sum(float(n) * n for n in _prompt_lens(case)) * case["heads"] * (case["dim"] * 2 + case["rope"]) * 2
    elif case["kind"] == "compact":
        cost = 0.0
    else:
        width = case["dim"] if case["kind"] == "scores" else 2 * case["rank"] + case["rope"]
        cost = sum(float(c) * n for c, n in zip(*_lens(case))) * case["heads"] * width * 2
    if cost > 8e12:
        return None
    return {"scores": _exact_scores, "compact": _exact_compact, "latent": _exact_latent,
            "expanded": _exact_expanded}[case["kind"]](case, seed)
