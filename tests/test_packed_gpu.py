"""packed_attention against its 64-bit form: grouped heads, query counts, contexts, masks, formats, plans, refusals."""
import numpy as np
import oracle as O
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import attend, check, quantized_scores, starts, tolerance

pytestmark = pytest.mark.gpu

FORMATS = ["int4", "fp16"]
FILL = 128 * 256  # rows of the whole batch over all key heads that give each compute unit a tile of 128


def staged_rows(T, Hq):
    """Rows (tokens times query heads per key head) from which a chunk attends from a staged copy."""
    return 512 if T * Hq >= 2 * FILL else 1024 if T * Hq >= FILL else 2 ** 31


class Case:
    """A paged cache of random keys and values and packed queries over it."""

    def __init__(self, fmt, ctx, qn, Hq, Hk, D, seed=0, bs=16, spare=0, M=None):
        rng = np.random.default_rng(seed)
        self.fmt, self.ctx, self.qn, self.D, self.bs = fmt, list(ctx), list(qn), D, bs
        B = len(ctx)
        per = [-(-c // bs) for c in ctx]
        self.M = M or max(1, max(per, default=1)) + spare
        nb = max(1, sum(per)) + 3
        perm = rng.permutation(nb).astype(np.int32)
        self.tables = np.full((B, self.M), -1, np.int32)
        at = 0
        for b in range(B):
            self.tables[b, :per[b]] = perm[at:at + per[b]]
            at += per[b]
        self.unused = perm[at:]
        shape = (nb, bs, Hk, D)
        self.k, self.v = (rng.standard_normal(shape).astype(np.float16) for _ in range(2))
        T = sum(qn)
        self.q = torch.from_numpy(rng.standard_normal((T, Hq, D)).astype(np.float16)).to(dev())
        self.cu = torch.from_numpy(starts(qn)).to(dev())
        self.load()

    def load(self):
        """Put the pools on the device (quantized, for INT4) and keep the values that they stand for."""
        if self.fmt == "int4":
            pages = O.to_int4_pages(self.k, self.v)
            self.kc = self.vc = torch.from_numpy(pages).to(dev())
            self.kval, self.vval = page_values(pages, self.D)
        else:
            self.kc, self.vc = (torch.from_numpy(x).to(dev()) for x in (self.k, self.v))
            self.kval, self.vval = (torch.from_numpy(x).double() for x in (self.k, self.v))
        self.bt = torch.from_numpy(self.tables).to(dev())
        self.cl = torch.from_numpy(np.array(self.ctx, np.int32)).to(dev())

    def args(self, most=None, window=-1):
        return (self.q, self.kc, self.vc, self.bt, self.cl, self.cu, max(self.qn, default=0) if most is None else most,
                max(1, self.M * self.bs), window)

    def check(self, out, window=-1, sinks=0, rows=None):
        """All rows, or those of a truth tensor ``rows``, against the 64-bit form."""
        a = 0
        for b, (c, n) in enumerate(zip(self.ctx, self.qn)):
            m = max(0, min(c, self.M * self.bs))
            pages = torch.from_numpy(self.tables[b, :-(-m // self.bs)]).long()
            live = (pages >= 0) & (pages < self.k.shape[0])
            k, v = (x[pages.clamp(0, self.k.shape[0] - 1)].flatten(0, 1)[:m] for x in (self.kval, self.vval))
            some = np.arange(n)
            if n > 150:  # the first and last rows, and some of those between
                some = np.unique(np.concatenate([np.arange(20), n - 1 - np.arange(20), np.random.default_rng(n).integers(0, n, 30)]))
            o, w, e = attend(self.q[a:a + n][some], k, v, (c - n) + some, window, sinks,
                             live.repeat_interleave(self.bs)[:m])
            scores, staged, v_scale = 0.0, False, 0.0
            if self.fmt == "int4":
                G = self.q.shape[1] // self.k.shape[2]
                staged = n * G >= staged_rows(*self.q.shape[:2])
                scores = quantized_scores(self.q[a:a + n][some], float(self.kval.abs().max()) / 7, staged)
                v_scale = 0.0 if staged else float(self.vval.abs().max()) / 7
            tol = tolerance(o, w, e, m, self.D, torch.float16, torch.float16, staged, scores, v_scale)
            r = slice(None) if rows is None else rows[a:a + n][some]
            check(out[a:a + n].cpu()[some][r], o[r], tol[r], f"sequence {b}")
            a += n


def page_values(pages, D):
    """(code - 8) * scale of a page buffer in float64: (K, V) [nb, 16, H, D]."""
    out = []
    parts = O.int4_pages_split(pages, D)
    for codes, scales in (parts[:2], parts[2:]):
        c = torch.from_numpy(O.unpack_codes(codes).reshape(*codes.shape[:3], D).astype(np.float64)) - 8
        s = torch.from_numpy(scales.astype(np.float64))
        out.append((c.unflatten(-1, (-1, 64)) * s[..., None]).flatten(-2))
    return out


HEADS = [(8, 2, 64), (4, 4, 64), (5, 1, 128), (32, 8, 128), (16, 1, 64), (20, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D", HEADS)
def test_decode(fmt, Hq, Hk, D):
    c = Case(fmt, [1, 15, 16, 17, 33, 100, 257, 64], [1] * 8, Hq, Hk, D, seed=Hq)
    c.check(memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 64), (10, 2, 128), (3, 3, 128), (16, 1, 64)])
@pytest.mark.parametrize("ctx,qn", [([50, 40, 300], [3, 0, 20]), ([128, 1, 90, 17], [128, 1, 33, 1]), ([5, 0, 7], [5, 0, 7]),
                                    ([2, 600], [4, 6]), ([40] * 70, [1, 0, 2, 3, 1] * 14), ([33], [17])], ids=str)
def test_mixed_query_counts(fmt, Hq, Hk, D, ctx, qn):
    """None, one or many queries per sequence; more queries than context (the first see nothing and give 0)."""
    c = Case(fmt, ctx, qn, Hq, Hk, D, seed=sum(qn) + D)
    c.check(memopt_C.packed_attention(*c.args()))
    c.check(memopt_C.packed_attention(*c.args(most=10 ** 6)))


@pytest.mark.parametrize("Hq,Hk,D,qn", [(8, 2, 64, [1, 40, 32, 1, 3, 33, 1]), (32, 8, 128, [33, 1, 32, 2, 200]),
                                        (12, 1, 128, [1, 11, 10, 1]), (64, 1, 64, [600, 2, 1, 3, 1]),
                                        (64, 1, 128, [1, 2, 600])])
def test_short_sequences_beside_long_ones_keep_what_a_weight_rounding_loses(Hq, Hk, D, qn):
    """Over pages, sequences of up to 128 rows (tokens times query heads per key head) hold their weights in two 16-bit
    operands, whatever else the batch brings. A window of one token makes each row its own value: it is off by the
    output's rounding, 2^-11, by the 2^-22 that two operands leave, and by a few roundings in 32 bits (less than 2^-20
    in all), or by half a step of fp16's subnormals. (A single operand is off by 2^-11 more.)"""
    c = Case("int4", [n + 40 + 3 * i for i, n in enumerate(qn)], qn, Hq, Hk, D, seed=D + len(qn))
    G = Hq // Hk
    out = memopt_C.packed_attention(*c.args(window=1)).double().cpu()
    c.check(out.half(), 1, 0)
    at = 0
    for b, (ctx, n) in enumerate(zip(c.ctx, c.qn)):
        pages = torch.from_numpy(c.tables[b, :-(-ctx // 16)]).long()
        v = c.vval[pages].flatten(0, 1)[ctx - n:ctx].repeat_interleave(G, 1)
        if n * G <= 128:
            off = (out[at:at + n] - v).abs()
            assert bool((off <= (2.0 ** -11 + 2.0 ** -20) * v.abs() + 2.0 ** -25).all()), (b, float((off / v.abs()).nan_to_num().max()))
        at += n


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 3), (100, 16), (100, 33), (5, 400), (2 ** 31 - 1, 2 ** 31 - 1),
                                          (0, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_windows_and_sinks(fmt, window, sinks, D):
    c = Case(fmt, [300, 90, 40], [1, 40, 7], 6, 2, D, seed=window % 100 + sinks % 7)
    out = memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks)
    c.check(out, window if 0 < window <= c.M * 16 else c.M * 16, sinks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D,ctx,qn", [(8, 2, 64, [3000], [1]), (8, 1, 128, [5000, 100, 2500], [1, 1, 1]),
                                            (20, 1, 128, [2100], [3]), (32, 8, 128, [1500], [1]),
                                            (4, 2, 64, [2500, 600], [40, 1]), (8, 2, 64, [6100], [1]),
                                            (8, 4, 64, [4000, 9000], [1, 2]), (32, 8, 128, [7000], [1]),
                                            (16, 1, 64, [6100], [1]), (10, 1, 128, [5300, 4700], [1, 1])])
def test_long_contexts_in_splits(fmt, Hq, Hk, D, ctx, qn):
    c = Case(fmt, ctx, qn, Hq, Hk, D, seed=7)
    plan = memopt_C.PreparedPackedAttention(*c.args())
    assert plan.workspace_bytes > 0
    for _ in range(3):  # (the workspace holds the call before)
        plan.out.fill_(float("nan"))
        c.check(plan())
    c.check(memopt_C.packed_attention(*c.args(window=700), num_sink_tokens=5), 700, 5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_unlinked_pages_and_entries_past_the_pool(fmt, D):
    c = Case(fmt, [200, 48, 130, 30], [1, 20, 3, 1], 8, 2, D, seed=3)
    c.tables[0, 3] = c.tables[0, 7] = c.tables[2, 8] = -1
    c.tables[1, 1] = 10 ** 6
    c.tables[2, 0] = -5
    c.tables[3, :] = -1  # nothing left: zeros
    c.load()
    out = memopt_C.packed_attention(*c.args())
    c.check(out)
    assert bool((out[-1] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D,ctx,qn", [(64, 1, 128, [200, 700, 65, 300], [192, 7, 65, 250]),
                                            (32, 2, 64, [640, 400, 333, 64], [640, 400, 63, 64]),
                                            (30, 10, 64, [1, 400, 350, 600], [1, 342, 341, 500]),
                                            (32, 8, 128, [900, 255, 256, 5], [897, 255, 256, 1]),
                                            (64, 1, 128, [600, 500, 8, 70], [600, 430, 8, 7])])
def test_long_chunks(fmt, Hq, Hk, D, ctx, qn):
    """Chunks on both sides of the length from which they attend from a staged copy, beside single tokens."""
    c = Case(fmt, ctx, qn, Hq, Hk, D, seed=Hq + qn[0])
    assert sum(qn) * Hq >= FILL
    plan = memopt_C.PreparedPackedAttention(*c.args())
    for _ in range(2):
        plan.out.fill_(float("nan"))
        c.check(plan())
    c.check(memopt_C.packed_attention(*c.args(window=90), num_sink_tokens=7), 90, 7)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (63, 64), (130, 65), (17, 200), (5, 2 ** 31 - 1),
                                          (2 ** 31 - 1, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_long_chunks_windows_and_sinks(fmt, window, sinks, D):
    c = Case(fmt, [640, 90, 250], [300, 4, 220], 64, 1, D, seed=window % 100 + sinks % 7)
    out = memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks)
    c.check(out, min(window, c.M * 16), sinks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_long_chunks_unlinked_pages(fmt, D):
    c = Case(fmt, [500, 320, 100, 257], [250, 100, 1, 257], 64, 1, D, seed=3)
    c.tables[0, 3] = c.tables[0, 20] = c.tables[0, 31] = -1
    c.tables[1, :5] = 10 ** 6
    c.tables[3, :] = -7  # nothing left: zeros
    c.load()
    out = memopt_C.packed_attention(*c.args())
    c.check(out)
    assert bool((out[-257:] == 0).all())
    c.check(memopt_C.packed_attention(*c.args(window=70), num_sink_tokens=60), 70, 60)


@pytest.mark.parametrize("bs", [32, 48, 64])
def test_long_chunks_fp16_page_sizes(bs):
    c = Case("fp16", [830, 297, 200], [730, 297, 1], 32, 2, 64, seed=bs, bs=bs)
    c.check(memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_chunks_outside_the_block_table(fmt):
    """More queries than context, and contexts past the table: the keys that the table holds."""
    c = Case(fmt, [64, 64, 20], [200, 200, 200], 64, 1, 64, seed=3, M=4)
    c.ctx = [70, 1000, -3]
    c.load()
    c.check(memopt_C.packed_attention(*c.args()[:7], 2000, -1), 2000, 0)
    c.ctx = [300, 150, 201]
    c.load()
    c.check(memopt_C.packed_attention(*c.args()[:7], 2000, 100), 100, 0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,ctx,M,window,sinks", [(1162, 4511, 55, 500, 0), (1162, 4511, 55, 500, 70), (1162, 2000, 55, 64, 0),
                                                  (1100, 1500, 55, 300, 200), (1100, 1300, 82, -1, 0),
                                                  (1100, 1300, 82, 100, 4)])
def test_long_chunks_of_one_query_head_per_key_head(fmt, D, n, ctx, M, window, sinks):
    """A tile of 128 rows spans 128 positions: its last wave can see nothing where its first one does, in particular
    behind the block table by more than the window (such rows give 0)."""
    c = Case(fmt, [min(ctx, 16 * M)], [n], 32, 32, D, seed=n, M=M)
    assert n * 32 >= FILL and n >= staged_rows(n, 32)
    c.ctx = [ctx]
    c.load()
    out = memopt_C.packed_attention(*c.args()[:7], 5000, window, num_sink_tokens=sinks)
    c.check(out, window, sinks)
    if window > 0 and sinks == 0:
        dark = torch.arange(ctx - n, ctx) - window + 1 >= 16 * M
        assert bool((out[dark.to(dev())] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_chunks_among_many_sequences(fmt):
    qn = [1 + 59 * (i % 5 == 1) for i in range(70)]
    c = Case(fmt, [100 + 3 * (i % 11) for i in range(70)], qn, 64, 2, 64, seed=9)
    c.check(memopt_C.packed_attention(*c.args()))
    qn = [1] * 290 + [120, 0, 140]
    c = Case(fmt, [2] * 290 + [120, 9, 333], qn, 64, 2, 64, seed=9)
    c.check(memopt_C.packed_attention(*c.args()))


def test_long_chunks_of_more_sequences_than_are_staged():
    """Block tables of 2^20 tokens leave room for copies of four sequences: only chunks that must be among four."""
    for qn in ([100] * 6, [100, 97, 300, 100, 1, 1]):
        c = Case("int4", [320, 100, 310, 100, 100, 101], qn, 64, 2, 64, seed=4, M=65536)
        c.check(memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(-1, 0), (70, 3)])
def test_long_chunks_odd_values_reach_only_the_rows_that_see_them(fmt, window, sinks):
    def case():
        return Case(fmt, [600, 70], [510, 10], 64, 1, 64, seed=11)

    good, lay = case(), memopt_C.int4_layout(64)
    W = window if window > 0 else good.M * 16
    pos = torch.arange(90, 600)
    for token, bad, where in [(160, float("nan"), "v"), (599, float("inf"), "v"), (95, float("nan"), "k"),
                              (64, float("nan"), "kv"), (0, float("nan"), "v"), (128, float("nan"), "v")]:
        c = case()
        page, row = c.tables[0, token // 16], token % 16
        for x in where:
            if fmt == "fp16":
                (c.kc if x == "k" else c.vc)[page, row, :, 33] = bad
            else:
                c.kc.view(torch.float16)[page, :, lay[x + "scales"] // 2 + 2 * (row % 8) + row // 8] = bad
        out = memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks)
        see = (token <= pos) & ((pos - token < window) | (token < sinks)) if window > 0 else token <= pos
        see = torch.cat([see, torch.zeros(10, dtype=torch.bool)])
        good.check(out, W, sinks, ~see)
        hit = out[see.to(dev())]
        if hit.numel():
            assert bool((~hit[..., 33].isfinite()).all()), (token, bad, where)
    # behind the context
    want = memopt_C.packed_attention(*good.args(window=window), num_sink_tokens=sinks)
    tail = good.tables[0, 600 // 16]
    if fmt == "fp16":
        good.kc[tail, 600 % 16:] = good.vc[tail, 600 % 16:] = float("nan")
    else:
        for x in ("kscales", "vscales"):
            for row in range(600 % 16, 16):
                good.kc.view(torch.float16)[tail, :, lay[x] // 2 + 2 * (row % 8) + row // 8] = float("nan")
    assert torch.equal(memopt_C.packed_attention(*good.args(window=window), num_sink_tokens=sinks), want)


@pytest.mark.parametrize("bs", [16, 32, 48, 64])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_page_sizes(bs, D):
    c = Case("fp16", [130, 40, 97], [2, 40, 1], 4, 2, D, seed=bs, bs=bs)
    c.check(memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("fmt", FORMATS)
def test_contexts_outside_the_block_table(fmt):
    """A context past the table's last page, or below zero, reads only what the table holds."""
    c = Case(fmt, [64, 64, 20], [1, 2, 1], 4, 2, 64, seed=3, M=4)
    c.ctx = [70, 1000, -3]
    c.load()
    a = memopt_C.packed_attention(*c.args()[:7], 2000, -1)
    c.check(a, 2000, 0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (40, 3)])
def test_odd_values_reach_only_the_rows_that_see_them(fmt, D, window, sinks):
    """inf and NaN in the cache: behind the context, in window gaps, in later positions of a chunk."""
    Hq, Hk, ctx, qn = 4, 2, [150, 70], [60, 1]

    def case(where=None, bad=None, token=0):
        c = Case(fmt, ctx, qn, Hq, Hk, D, seed=11)
        if where is not None:
            page, row = c.tables[0, token // 16], token % 16
            for x in (["k", "v"] if where == "kv" else [where]):
                if fmt == "fp16":
                    (c.kc if x == "k" else c.vc)[page, row, :, D // 2 + 1] = bad
                else:
                    lay = memopt_C.int4_layout(D)
                    scales = c.kc.view(torch.float16)[..., lay[x + "scales"] // 2:]
                    scales[page, :, 16 * ((D // 2 + 1) // 64) + 2 * (row % 8) + row // 8] = bad
        return c

    good = case()
    W = window if window > 0 else good.M * 16
    pos = torch.arange(90, 150)
    for token, bad, where in [(120, float("nan"), "v"), (149, float("inf"), "v"), (95, float("nan"), "k"),
                              (64, float("nan"), "kv"), (0, float("nan"), "v"), (101, float("nan"), "v")]:
        c = case(where, bad, token)
        out = memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks)
        see = (token <= pos) & ((pos - token < window) | (token < sinks)) if window > 0 else token <= pos
        see = torch.cat([see, torch.zeros(1, dtype=torch.bool)])
        good.check(out, W, sinks, ~see)
        hit = out[see.to(dev())]
        if hit.numel():
            assert bool((~hit[..., D // 2 + 1].isfinite()).all()), (token, bad, where)
    # behind the context, and in a page that no table names
    c = case()
    tail = c.tables[0, 150 // 16]
    if fmt == "fp16":
        for x in (c.kc, c.vc):
            x[tail, 150 % 16:] = float("nan")
            x[torch.from_numpy(c.unused).long()] = float("nan")
    else:
        lay = memopt_C.int4_layout(D)
        s = c.kc.view(torch.float16)[tail]
        for x in ("kscales", "vscales"):
            for row in range(150 % 16, 16):
                for grp in range(D // 64):
                    s[:, lay[x] // 2 + 16 * grp + 2 * (row % 8) + row // 8] = float("nan")
    good.check(memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks), W, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,qn", [(3000, 1), (3000, 5), (3000, 40), (420, 40), (20000, 1)])
def test_infinities_pass_the_merge(D, ctx, qn):
    """A column in which every row sees one inf of V is that inf, in whatever part of a split block it lies; the
    others are what they were."""
    c = Case("fp16", [ctx], [qn], 8, 2, D, seed=ctx)
    want = memopt_C.packed_attention(*c.args()).cpu()
    for token in (0, ctx // 3, ctx // 2, ctx - qn):
        for bad in (float("inf"), float("-inf")):
            page = int(c.tables[0, token // 16])
            keep = c.vc[page, token % 16, :, 5].clone()
            c.vc[page, token % 16, :, 5] = bad
            out = memopt_C.packed_attention(*c.args()).cpu()
            c.vc[page, token % 16, :, 5] = keep
            assert bool((out[..., 5] == bad).all()), (token, bad)
            out[..., 5] = want[..., 5]
            assert torch.equal(out, want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (200, 40)])
@pytest.mark.parametrize("qn", [1, 3, 40])
def test_odd_values_beside_an_unlinked_page(D, window, sinks, qn):
    """inf and NaN of V in the linked half of a 32-token step whose other page is gone, where every row sees it."""
    for token, gone in ((40, 3), (329, 21), (385, 25)):
        c = Case("fp16", [420], [qn], 8, 2, D, seed=token)
        c.tables[0, gone] = -1
        c.load()
        want = memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks)
        c.check(want, window, sinks)
        pos = torch.arange(420 - qn, 420)
        see = (token <= pos) & ((pos - token < window) | (token < sinks)) if window > 0 else token <= pos
        for bad in (float("inf"), float("nan"), float("-inf")):
            c.vc[c.tables[0, token // 16], token % 16, :, 5] = bad
            out = memopt_C.packed_attention(*c.args(window=window), num_sink_tokens=sinks).cpu()
            where = out[..., 5]
            assert bool((where[see].isnan() if bad != bad else where[see] == bad).all()), (token, bad)
            out[..., 5][see] = want.cpu()[..., 5][see]
            assert torch.equal(out, want.cpu())


@pytest.mark.parametrize("D", [64, 128])
def test_evicted_rows_and_extreme_scales(D):
    """Scale 0 (rows that eviction removed), the largest scales of the format, and tiny ones."""
    c = Case("int4", [100, 64], [1, 5], 4, 2, D, seed=5)
    c.v[:] *= np.float16(3000)
    c.k[3::4] *= np.float16(2.0 ** -10)
    c.load()
    pages = c.kc.cpu().numpy()
    lay = memopt_C.int4_layout(D)
    sc = pages[..., lay["kscales"]:].view(np.float16)
    sc[::2, :, 3::5] = 0
    c.kc = c.vc = torch.from_numpy(pages).to(dev())
    c.kval, c.vval = page_values(pages, D)
    c.check(memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("D", [64, 128])
def test_long_chunks_evicted_rows_and_extreme_scales(D):
    """Scales of 0 in one group or all, the largest beside the smallest: what the staged keys' factors hold."""
    c = Case("int4", [540, 64], [510, 5], 64, 1, D, seed=5)
    c.k[:] *= np.float16(0.25)
    c.k[::5, ..., D // 2:] *= np.float16(2.0 ** -12)
    c.k[1::5, ..., :D // 2] *= np.float16(2.0 ** -12)
    c.v[:] *= np.float16(3000)
    c.load()
    pages = c.kc.cpu().numpy()
    lay = memopt_C.int4_layout(D)
    sc = pages[..., lay["kscales"]:lay["kscales"] + 32 * (D // 64)].view(np.float16)
    sc[::2, :, 3::5] = 0
    sc[1::4, :, :4] = 0
    sc[2::4, :, -7:] = 0
    c.kc = c.vc = torch.from_numpy(pages).to(dev())
    c.kval, c.vval = page_values(pages, D)
    c.check(memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,qn", [(4, [1, 2]), (64, [520, 3])], ids=["decode", "long chunk"])
def test_pages_past_4_gib(fmt, Hq, qn):
    """Byte offsets past 32 bits: the same pages at the end of a pool of more than 4 GiB."""
    c = Case(fmt, [600, 77], qn, Hq, 1, 128, seed=6)
    want = memopt_C.packed_attention(*c.args())
    nb = c.kc.shape[0]
    first = 2 ** 32 // (2176 if fmt == "int4" else 4096) + 5
    pools = []
    for x in ([c.kc] if fmt == "int4" else [c.kc, c.vc]):
        pools.append(torch.empty((first + nb, *x.shape[1:]), dtype=x.dtype, device=dev()))
        pools[-1][first:] = x
    c.kc, c.vc = pools[0], pools[-1]
    c.bt = torch.where(c.bt >= 0, c.bt + first, c.bt)
    assert torch.equal(memopt_C.packed_attention(*c.args()), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_strides_padding_and_out(fmt):
    c = Case(fmt, [60, 200], [4, 30], 6, 2, 64, seed=2)
    want = memopt_C.packed_attention(*c.args())
    c.check(want)
    q = c.q
    c.q = torch.empty((34, 9, 128), dtype=q.dtype, device=dev())[:, ::3, :].repeat(1, 2, 1)[:, :, 64:].copy_(q)
    assert not c.q.is_contiguous() and torch.equal(memopt_C.packed_attention(*c.args()), want)
    c.q = torch.empty((34, 6, 65), dtype=q.dtype, device=dev())[..., 1:].copy_(q)
    assert torch.equal(memopt_C.packed_attention(*c.args()), want)
    buf = torch.full((34, 6, 128), 5.0, dtype=q.dtype, device=dev())
    memopt_C.packed_attention(*c.args(), out=buf[..., :64])
    assert torch.equal(buf[..., :64], want) and bool((buf[..., 64:] == 5).all())
    # rows of no sequence
    c.q = torch.full((50, 6, 64), float("nan"), dtype=q.dtype, device=dev())
    c.q[8:42] = q
    c.cu += 8
    out = torch.full((50, 6, 64), 3.0, dtype=q.dtype, device=dev())
    memopt_C.packed_attention(*c.args(), out=out)
    assert torch.equal(out[8:42], want) and bool((out[:8] == 3).all()) and bool((out[42:] == 3).all())
    c.cu = torch.tensor([-4, 38, 900], dtype=torch.int32, device=dev())  # clamped to 0 .. 50
    memopt_C.packed_attention(*c.args(most=50), out=out)
    empty = Case(fmt, [20, 20], [0, 0], 6, 2, 64)
    assert memopt_C.packed_attention(*empty.args()).shape == (0, 6, 64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_contiguous_queries_off_the_alignment_are_copied(fmt):
    c = Case(fmt, [60, 200], [4, 30], 6, 2, 64, seed=2)
    want = memopt_C.packed_attention(*c.args())
    flat = torch.empty(c.q.numel() + 8, dtype=c.q.dtype, device=dev())[4:4 + c.q.numel()]
    c.q = flat.view(c.q.shape).copy_(c.q)
    assert c.q.is_contiguous() and c.q.data_ptr() % 16 == 8
    assert torch.equal(memopt_C.packed_attention(*c.args()), want)
    with pytest.raises(RuntimeError, match="read in place"):
        memopt_C.PreparedPackedAttention(*c.args())


@pytest.mark.parametrize("fmt", FORMATS)
def test_pool_views_are_taken(fmt):
    """The live pool's views, written by write_cache."""
    g = torch.Generator(device=dev()).manual_seed(0)
    memopt_C.init_pool(12, 16, 2, 64, kv_format=fmt)
    k, v = (torch.randn((100, 2, 64), generator=g, device=dev(), dtype=torch.float16) for _ in range(2))
    memopt_C.write_cache(k, v, None, torch.arange(100, dtype=torch.int32, device=dev()) + 16)
    q = torch.randn((1, 8, 64), generator=g, device=dev(), dtype=torch.float16)
    bt = torch.arange(1, 8, dtype=torch.int32, device=dev())[None].contiguous()
    cl, cu = (torch.tensor(x, dtype=torch.int32, device=dev()) for x in ([100], [0, 1]))
    out = memopt_C.packed_attention(q, memopt_C.get_key_pool(), memopt_C.get_value_pool(), bt, cl, cu, 1, 112)
    if fmt == "int4":
        buf = memopt_C.get_int4_pages()
        assert torch.equal(memopt_C.packed_attention(q, buf, buf, bt, cl, cu, 1, 112), out)
        k, v = (x[1:].flatten(0, 1)[:100] for x in page_values(buf.cpu().numpy(), 64))
    o, w, e = attend(q, k, v, [99], -1, 0)
    scores = quantized_scores(q, float(k.abs().max()) / 7, False) if fmt == "int4" else 0.0
    v_scale = float(v.abs().max()) / 7 if fmt == "int4" else 0.0
    check(out, o, tolerance(o, w, e, 100, 64, torch.float16, torch.float16, False, scores, v_scale))


def test_same_heads_agree_with_the_paged_attention():
    """One query head per key head: the rectangular causal call and the packed one compute the same function."""
    for fmt in FORMATS:
        c = Case(fmt, [90, 90, 90], [5, 5, 5], 4, 4, 64, seed=1)
        a = memopt_C.packed_attention(*c.args(window=50), num_sink_tokens=2)
        b = memopt_C.dynamic_sparse_attention(c.q.view(3, 5, 4, 64), c.kc, c.vc, c.bt, c.cl, 96, 50, num_sink_tokens=2,
                                              causal=True)
        assert float((a - b.view(15, 4, 64)).abs().max()) <= 2e-3


def test_plans_on_two_streams_and_in_graphs():
    """Two captured plans replayed on two streams (each with its own workspace), lengths changed in between."""
    cases = [Case("int4", [2000, 900], [1, 1], 8, 2, 64, seed=s) for s in (1, 2)]
    plans = [memopt_C.PreparedPackedAttention(*c.args()) for c in cases]
    assert all(p.workspace_bytes for p in plans)
    for p in plans:
        p()
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for p in plans:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            p()
    for ctx in ([2000, 900], [1, 2000], [1999, 17]):
        for c, p in zip(cases, plans):
            c.ctx = [min(n, 16 * int((c.tables[b] >= 0).sum())) for b, n in enumerate(ctx)]
            c.cl.copy_(torch.tensor(c.ctx, dtype=torch.int32))
            p.out.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, p in zip(cases, plans):
            c.check(p.out)
            assert torch.equal(p.out, memopt_C.packed_attention(*c.args()))


@pytest.mark.parametrize("explicit", [True, False])
def test_first_call_of_a_plan_on_another_stream(explicit):
    """A plan made behind queued work of one stream is ready for a call on another, whatever its memory held."""
    c = Case("int4", [3000, 2500], [1, 1], 8, 2, 64, seed=31)
    want = memopt_C.packed_attention(*c.args())
    c.check(want)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    busy = torch.ones((4096, 4096), device=dev())
    size = memopt_C.PreparedPackedAttention(*c.args()).workspace_bytes
    for _ in range(5):
        dirty = torch.full((size,), 0xFF, dtype=torch.uint8, device=dev())  # (its memory is the next plan's)
        del dirty
        out = torch.zeros_like(c.q)
        other.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            busy = busy @ busy * 0
        plan = memopt_C.PreparedPackedAttention(*c.args(), out=out)
        if explicit:
            plan(other.cuda_stream)
        else:
            with torch.cuda.stream(other):
                plan()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_captured_long_chunks_follow_the_lengths_on_the_device(fmt):
    """One captured plan, replayed as chunks grow and shrink across the length from which they are staged; and eager
    calls of another shape in between."""
    c = Case(fmt, [700, 300, 90], [500, 20, 10], 64, 1, 64, seed=21, spare=2)
    plan = memopt_C.PreparedPackedAttention(*c.args(most=530))
    plan()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
    other = Case(fmt, [100, 40], [1, 1], 8, 2, 64, seed=2)
    for ctx, qn in [([700, 300, 90], [500, 20, 10]), ([530, 1, 90], [530, 0, 0]), ([8, 300, 90], [8, 250, 7]),
                    ([690, 299, 0], [265, 265, 0]), ([700, 300, 90], [500, 20, 10])]:
        c.ctx, c.qn = ctx, qn
        c.cl.copy_(torch.tensor(ctx, dtype=torch.int32))
        c.cu.copy_(torch.from_numpy(starts(qn)))
        for _ in range(2):
            plan.out.fill_(9.0)
            graph.replay()
            other.check(memopt_C.packed_attention(*other.args()))
            c.check(plan.out[:sum(qn)])
            assert bool((plan.out[sum(qn):] == 9).all())


def test_refusals():
    c = Case("fp16", [20], [2], 4, 2, 64)
    q, kc, vc, bt, cl, cu = c.args()[:6]

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            memopt_C.packed_attention(*args, 2, 32, -1, **kw)

    refused("CUDA", q.cpu(), kc, vc, bt, cl, cu)
    refused("key_cache must be a CUDA", q, kc.cpu(), vc, bt, cl, cu)
    refused("3-D", q[None], kc, vc, bt, cl, cu)
    refused("fp16", q.float(), kc, vc, bt, cl, cu)
    refused("fp16 or INT4", q, kc.float(), vc.float(), bt, cl, cu)
    refused("4-D", q, kc[0], vc[0], bt, cl, cu)
    refused("4-D", q, kc, vc[:1], bt, cl, cu)
    refused("contiguous", q, kc[:, :, ::2], vc[:, :, ::2], bt, cl, cu)
    refused("multiple of num_kv_heads", q[:, :3], kc, vc, bt, cl, cu)
    refused("context_lens", q, kc, vc, bt, cl.long(), cu)
    refused("context_lens", q, kc, vc, bt, cl.repeat(2), cu)
    refused("block_tables", q, kc, vc, bt.repeat(2, 1), cl, cu)
    refused("cu_seqlens", q, kc, vc, bt, cl, cu.long())
    refused("out must be", q, kc, vc, bt, cl, cu, out=torch.empty_like(q).float())
    refused("gradients", q.clone().requires_grad_(), kc, vc, bt, cl, cu)
    refused("16 tokens", q, kc[:, :8].contiguous(), vc[:, :8].contiguous(), bt, cl, cu)
    refused("head_dim must be", q[..., :32].contiguous(), kc[..., :32].contiguous(), vc[..., :32].contiguous(), bt, cl, cu)
    p = Case("int4", [20], [2], 4, 2, 64)
    refused("page buffer", q, p.kc[..., :100].contiguous(), p.kc[..., :100].contiguous(), bt, cl, cu)
    refused("both", q, p.kc, p.kc.clone(), bt, cl, cu)
    refused("page buffer", q, p.kc[:, :, None], p.kc[:, :, None], bt, cl, cu)
    with pytest.raises(RuntimeError, match="negative"):
        memopt_C.packed_attention(q, kc, vc, bt, cl, cu, -1, 32)
    with pytest.raises(RuntimeError, match="read in place"):
        memopt_C.PreparedPackedAttention(q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, bt, cl, cu, 2, 32)
