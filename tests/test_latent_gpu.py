"""latent_attention and write_latent against their 64-bit forms: widths, heads, row counts, masks, odd values, refusals."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C, same_bits
from packed_reference import check, starts
from small_cache_reference import latent, latent_tolerance

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
WIDTHS = [(512, 64), (256, 64), (128, 64), (512, 32), (256, 32), (128, 32)]


class Case:
    """A paged latent cache of random rows and packed queries over it."""

    def __init__(self, dtype, ctx, qn, Hq, rank=512, rope=64, seed=0, bs=16, spare=0, M=None, std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.qn, self.rank, self.bs, self.dtype = list(ctx), list(qn), rank, bs, dtype
        per = [-(-max(c, 0) // bs) for c in ctx]
        self.M = M or max(1, max(per, default=1)) + spare
        self.nb = max(1, sum(per)) + 3
        perm = torch.randperm(self.nb, generator=g).to(torch.int32).numpy()
        self.tables = np.full((len(ctx), self.M), -1, np.int32)
        at = 0
        for b in range(len(ctx)):
            k = min(per[b], self.M)
            self.tables[b, :k] = perm[at:at + k]
            at += per[b]
        self.c = torch.randn(self.nb, bs, rank + rope, generator=g).to(dtype).to(dev())
        self.q = (torch.randn(sum(qn), Hq, rank + rope, generator=g) * std).to(dtype).to(dev())
        self.scale = (128 + rope) ** -0.5
        self.cu = torch.from_numpy(starts(qn)).to(dev())
        self.load()

    def load(self):
        self.bt = torch.from_numpy(self.tables).to(dev())
        self.cl = torch.from_numpy(np.array(self.ctx, np.int32)).to(dev())

    def run(self, window=-1, sinks=0, most=None, longest=None, out=None):
        return memopt_C.latent_attention(self.q, self.c, self.bt, self.cl, self.cu, max(self.qn, default=0) if most is None else most,
                                         max(1, self.M * self.bs) if longest is None else longest, self.scale, self.rank,
                                         window, num_sink_tokens=sinks, out=out)

    def check(self, out, window=-1, sinks=0, rows=None, keys=None):
        """All rows, or those of a truth tensor ``rows``; of long chunks the first, the last and some between."""
        a = 0
        host = self.c.cpu()
        for b, (c, n) in enumerate(zip(self.ctx, self.qn)):
            m = max(0, min(c, self.M * self.bs if keys is None else keys))
            pages = torch.from_numpy(self.tables[b, :-(-m // self.bs)]).long()
            live = ((pages >= 0) & (pages < self.nb)).repeat_interleave(self.bs)[:m]
            x = host[pages.clamp(0, self.nb - 1)].flatten(0, 1)[:m]
            some = np.arange(n)
            if n > 60:
                some = np.unique(np.concatenate([np.arange(8), n - 1 - np.arange(8), np.random.default_rng(n).integers(0, n, 12)]))
            r = slice(None) if rows is None else rows[a:a + n][some]
            o, w, e = latent(self.q[a:a + n][some], x, (c - n) + some, self.rank, self.scale, window, sinks, live)
            tol = latent_tolerance(o, w, e, m, self.q.shape[2], self.dtype)
            check(out[a:a + n].cpu()[some][r], o[r], tol[r], f"sequence {b}")
            a += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank,rope", WIDTHS)
@pytest.mark.parametrize("Hq", [1, 5, 16, 40, 128])
def test_single_tokens(dtype, rank, rope, Hq):
    c = Case(dtype, [1, 15, 16, 17, 33, 64, 65, 100, 257], [1] * 9, Hq, rank, rope, seed=Hq)
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank,rope,Hq", [(512, 64, 16), (256, 32, 3), (128, 64, 64), (512, 32, 33)])
@pytest.mark.parametrize("ctx,qn", [([50, 40, 300], [3, 0, 20]), ([128, 1, 90, 17], [128, 1, 33, 1]), ([5, 0, 7], [5, 0, 7]),
                                    ([2, 600], [4, 6]), ([40] * 70, [1, 0, 2, 3, 1] * 14), ([33], [17]), ([0, 9], [1, 0])],
                         ids=str)
def test_mixed_query_counts(dtype, rank, rope, Hq, ctx, qn):
    """None, one or many queries per sequence; more queries than context (the first see nothing and give 0)."""
    c = Case(dtype, ctx, qn, Hq, rank, rope, seed=sum(qn) + Hq)
    c.check(c.run())
    c.check(c.run(most=10 ** 6))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 3), (64, 64), (100, 16), (100, 33), (5, 400),
                                          (2 ** 31 - 1, 2 ** 31 - 1), (0, 3)])
@pytest.mark.parametrize("rank,rope,Hq", [(512, 64, 16), (128, 32, 6)])
def test_windows_and_sinks(dtype, window, sinks, rank, rope, Hq):
    c = Case(dtype, [300, 90, 40], [1, 40, 7], Hq, rank, rope, seed=window % 100 + sinks % 7)
    c.check(c.run(window, sinks), window if 0 < window <= c.M * 16 else c.M * 16, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank,rope,Hq,ctx,qn", [(512, 64, 16, [3000], [1]), (512, 64, 128, [5000, 100, 2500], [1, 1, 1]),
                                                 (256, 64, 8, [2100], [3]), (128, 32, 5, [1500], [1]),
                                                 (512, 64, 16, [2500, 600], [40, 1]), (512, 32, 16, [6100], [1]),
                                                 (256, 32, 16, [700, 900, 64], [300, 1, 64])])
def test_long_contexts_in_parts(dtype, rank, rope, Hq, ctx, qn):
    c = Case(dtype, ctx, qn, Hq, rank, rope, seed=7)
    first = c.run()
    c.check(first)
    assert torch.equal(c.run(), first)  # (the split is fixed, and so is the order of sums)
    c.check(c.run(700, 5), 700, 5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_batches_of_more_sequences_than_workgroups(dtype):
    rng = np.random.default_rng(1)
    ctx = rng.integers(0, 90, 700).tolist()
    c = Case(dtype, ctx, [int(x > 0) for x in ctx], 4, 128, 32, seed=2)
    c.check(c.run())
    c = Case(dtype, [700] + [3] * 300 + [400], [1] * 302, 4, 512, 64, seed=2)
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.1, 4.0])
def test_scales(dtype, scale):
    """Weights that hardly differ, and rows whose weight is nearly all on one key late or early (the maximum moves)."""
    c = Case(dtype, [200, 333], [1, 9], 16, 256, 64, seed=1)
    c.scale = scale
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rising_scores(dtype):
    """Every tile raises the row's maximum by far: what was summed before it nearly vanishes."""
    c = Case(dtype, [1024, 500], [1, 4], 16, 512, 64, seed=1)
    up = torch.linspace(-3, 3, 1024, device=dev())
    for b in range(2):
        pages = c.bt[b, :-(-c.ctx[b] // 16)].long()
        x = c.c[pages].flatten(0, 1)
        x[:, 512:] = up[:x.shape[0], None].to(dtype)
        c.c[pages] = x.view(-1, 16, 576)
    c.q[:, :, 512:] = 3
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_unlinked_pages_and_entries_past_the_pool(dtype):
    c = Case(dtype, [200, 48, 130, 30], [1, 20, 3, 1], 8, 256, 64, seed=3)
    c.tables[0, 3] = c.tables[0, 7] = c.tables[2, 8] = -1
    c.tables[1, 1] = 10 ** 6
    c.tables[2, 0] = -5
    c.tables[3, :] = -1  # nothing left: zeros
    c.load()
    out = c.run()
    c.check(out)
    assert bool((out[-1] == 0).all())
    c.check(c.run(70, 20), 70, 20)


@pytest.mark.parametrize("qn", [[1, 2, 1], [30, 20, 25]])
def test_contexts_outside_the_block_table_and_past_max_seq_len(qn):
    c = Case(torch.bfloat16, [64, 64, 20], qn, 8, 256, 64, seed=3, M=4)
    c.ctx = [70, 1000, -3]
    c.load()
    c.check(c.run(longest=2000), 2000, 0)
    c.ctx = [64, 40, 20]
    c.load()
    c.check(c.run(longest=33), 33, 0, keys=33)


@pytest.mark.parametrize("bs", [16, 32, 48, 64])
def test_page_sizes(bs):
    c = Case(torch.float16, [130, 40, 97], [2, 40, 1], 4, 256, 64, seed=bs, bs=bs)
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(-1, 0), (70, 3)])
@pytest.mark.parametrize("rank,rope", [(512, 64), (128, 32)])
def test_odd_values_reach_only_the_rows_that_see_them(dtype, window, sinks, rank, rope):
    def case():
        return Case(dtype, [300, 70], [210, 10], 3, rank, rope, seed=11)

    good = case()
    W = window if window > 0 else good.M * 16
    pos = torch.arange(90, 300)
    for token, bad, col in [(160, float("nan"), 3), (299, float("inf"), rank - 1), (95, float("-inf"), 64), (0, float("nan"), 5),
                            (128, float("nan"), rank + 1), (64, float("inf"), 33)]:
        c = case()
        c.c[c.tables[0, token // 16], token % 16, col] = bad
        out = c.run(window, sinks)
        see = (token <= pos) & ((pos - token < window) | (token < sinks)) if window > 0 else token <= pos
        see = torch.cat([see, torch.zeros(10, dtype=torch.bool)])
        good.check(out, W, sinks, ~see)
        hit = out[see.to(dev())]
        if hit.numel() and (col >= rank or bad != bad):
            assert bool((~hit.isfinite()).all()), (token, bad, col)  # (a NaN score)
    # behind the context, and in pages of nobody
    want = good.run(window, sinks)
    good.c[good.tables[0, 300 // 16], 300 % 16:] = float("nan")
    free = np.setdiff1d(np.arange(good.nb), good.tables)
    good.c[free] = float("inf")
    assert torch.equal(good.run(window, sinks), want)


def test_infinite_values_of_weight():
    """An inf that a row sees with a finite score is its result there, in masked tiles as in whole ones."""
    c = Case(torch.float16, [200], [100], 2, 128, 32, seed=5)
    c.q[:, :, 7] = 0  # (column 7 takes no part in the scores: 0 inf would be NaN)
    c.q.zero_()
    c.c[c.tables[0, 150 // 16], 150 % 16, 7] = 65504
    c.check(c.run())


def _steep(dtype, ctx, qn, low, high=40.0):
    """A case whose scores the first rotary element alone sets: keys lie at the level `low`, from the last 64 on at
    `high`, which is (high - low) 64 scale log2(e), more than 250 powers of two at the defaults, above them."""
    c = Case(dtype, [ctx], [qn], 16, seed=4)
    c.q.zero_()
    c.q[:, :, 512] = 64
    pages = c.bt[0, :-(-ctx // 16)].long()
    x = c.c[pages].flatten(0, 1)
    x[:, 512:] = 0
    x[:, 512] = low
    x[64:128, 512] = high
    c.c[pages] = x.view(-1, 16, 576)
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qn", [1, 70])
@pytest.mark.parametrize("token", [10, 1500, 1800])
def test_a_nan_far_below_the_other_parts(dtype, qn, token):
    """A row that sees a NaN is NaN, however small the weights of the part of its keys in which the NaN lies."""
    c = _steep(dtype, 2000, qn, -40.0)
    good = c.run()
    c.check(good)
    c.c[c.tables[0, token // 16], token % 16, 3] = float("nan")
    assert bool(c.run().isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_part_of_nothing_but_nan(dtype):
    """Beside parts whose scores lie far above or below 0."""
    for low, high in ((0.0, 40.0), (-40.0, 40.0), (-80.0, -40.0)):
        c = _steep(dtype, 2000, 1, low, high)
        c.check(c.run())
        c.c[c.bt[0, 4 * 9:4 * 10].long()] = float("nan")  # (keys 576 to 639)
        assert bool(c.run().isnan().all()), (low, high)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx,qn", [(200, 100), (2000, 70), (2000, 1)])
@pytest.mark.parametrize("back", [2, 40, 64])
def test_infinite_elements_of_weight_zero(dtype, ctx, qn, back):
    """A key with an inf where the queries are negative has the score -inf: rows that see it have 0 inf = NaN or inf in
    that column, and everywhere else what the other keys give; the other rows nothing of it."""
    c = Case(dtype, [ctx], [qn], 4, 128, 32, seed=5)
    c.q[:, :, 7] = -1
    token = ctx - back
    c.c[c.tables[0, token // 16], token % 16, 7] = float("inf")
    out = c.run().cpu()
    pages = torch.from_numpy(c.tables[0, :-(-ctx // 16)]).long()
    x, live = c.c.cpu()[pages].flatten(0, 1)[:ctx], torch.ones(ctx, dtype=torch.bool)
    live[token] = False
    pos = ctx - qn + np.arange(qn)
    o, w, e = latent(c.q, x, pos, 128, c.scale, -1, 0, live)
    tol = latent_tolerance(o, w, e, ctx, 160, dtype)
    see = torch.from_numpy(pos >= token)
    other = torch.arange(128) != 7
    check(out[~see], o[~see], tol[~see], "rows before it")
    check(out[see][:, :, other], o[see][:, :, other], tol[see][:, :, other], "its rows' other columns")
    assert not bool(out[see][:, :, 7].isfinite().any())


@pytest.mark.parametrize("power", [126, 100, -96])
@pytest.mark.parametrize("ctx,qn", [([300, 70], [40, 1]), ([3000], [1])])
def test_latents_of_bfloat16s_range(power, ctx, qn):
    """Latents up to nearly the type's largest, all alike or of both signs, and small ones, where the rotary part alone
    sets the scores: their means are in its range, and scaling by a power of two, exact, changes nothing else."""
    c = Case(torch.bfloat16, ctx, qn, 16, 256, 64, seed=9)
    c.q[:, :, :256] = 0
    some = c.c[:, :, :256].clamp(-3.5, 3.5)
    for latents in (torch.full_like(some, 3.5), some):
        c.c[:, :, :256] = latents * 2.0 ** power
        out = c.run()
        assert bool(out.isfinite().all())
        c.c[:, :, :256] = latents
        c.check((out.double() * 2.0 ** -power).bfloat16())


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_that_are_not_finite_stay_in_their_rows(dtype):
    c = Case(dtype, [100, 80], [5, 1], 16, 256, 64, seed=5)
    want = c.run()
    c.q[2, 3, 0] = float("nan")
    out = c.run()
    assert bool(out[2, 3].isnan().all())
    out[2, 3] = want[2, 3]
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_outputs_and_rows_of_no_sequence(dtype):
    c = Case(dtype, [200, 90], [3, 41], 6, 128, 64, seed=8)
    want, plain, T = c.run(), c.q, 44
    wide = torch.zeros(T, 10, 192 + 8, dtype=dtype, device=dev())
    wide[:, 2:8, 8:] = plain
    c.q = wide[:, 2:8, 8:]
    assert torch.equal(c.run(), want)
    c.q = plain.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(c.run(), want)
    odd = torch.zeros(T * 6 * 192 + 3, dtype=dtype, device=dev())[3:].view(T, 6, 192)
    odd.copy_(plain)
    c.q = odd
    assert torch.equal(c.run(), want)
    c.q = plain
    out = torch.full((T, 6, 2, 128), 7.0, dtype=dtype, device=dev())
    assert torch.equal(c.run(out=out[:, :, 1]), want) and bool((out[:, :, 0] == 7).all())
    c.cu = torch.tensor([2, 3, 30], dtype=torch.int32, device=dev())  # rows 0, 1 and 30 .. belong to nobody
    out = torch.full((T, 6, 128), 7.0, dtype=dtype, device=dev())
    c.run(out=out, most=41)
    assert bool((out[:2] == 7).all()) and bool((out[30:] == 7).all()) and not bool((out[2:30] == 7).any())
    c.cu = torch.tensor([-5, 10 ** 6, 50], dtype=torch.int32, device=dev())  # clamped
    c.run(out=out)


def test_cache_past_4_gib():
    nb = 2 ** 32 // (16 * 576 * 2) + 40
    big = torch.zeros(nb, 16, 576, dtype=torch.bfloat16, device=dev())
    c = Case(torch.bfloat16, [500], [2], 16, seed=2)
    want = c.run()
    at = torch.arange(nb - c.M, nb, device=dev())
    big[at] = c.c[c.bt[0].long()]
    c.c, c.bt = big, at.to(torch.int32)[None]
    assert torch.equal(c.run(), want)


def test_captured_calls_and_other_streams():
    c = Case(torch.bfloat16, [500, 70, 33], [1, 20, 2], 16, seed=6)
    out = torch.zeros(23, 16, 512, dtype=torch.bfloat16, device=dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(out=out)
    for ctx in ([500, 70, 33], [20, 60, 2], [499, 20, 30]):
        c.ctx = ctx
        c.cl.copy_(torch.tensor(ctx, dtype=torch.int32))
        c.q.copy_(torch.randn(c.q.shape))
        g.replay()
        want = c.run()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        c.check(out)
    want, got = c.run(), []
    for _ in range(8):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(c.run())
        got.append(c.run())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("given,meant", [([-5, 3, 2 ** 31 - 1], [0, 3, 9]), ([2, 1, 5], [1, 1, 5]), ([9, -1, 9], [0, 0, 9]),
                                         ([-2 ** 31, -1, 4], [0, 0, 4])])
def test_starts_out_of_range_or_order(given, meant):
    """Starts are held within the rows, and a sequence that would end before it begins has none."""
    c = Case(torch.float16, [400, 90], [3, 6], 5, 128, 32, seed=2)
    for most in (9, 2):
        outs = []
        for cu in (given, meant):
            c.cu = torch.tensor(cu, dtype=torch.int32, device=dev())
            outs.append(c.run(most=most, out=torch.full((9, 5, 128), 7.0, dtype=c.dtype, device=dev())))
        first = [c.cu[0].item(), c.cu[1].item()]
        rows = [r for b, a in enumerate(first) for r in range(a, min(a + most, c.cu[b + 1].item()))]
        assert torch.equal(outs[0][rows], outs[1][rows])
        rest = [r for r in range(9) if r not in rows]
        assert torch.equal(outs[0][rest], torch.full_like(outs[0][rest], 7.0))


def test_empty_calls():
    c = Case(torch.float16, [20, 30], [1, 1], 4, 128, 32)
    assert c.run(most=0).shape == (2, 4, 128)
    q = c.q
    c.q = q[:0]
    assert c.run().shape == (0, 4, 128)
    c.q, c.cu, c.bt, c.cl = q, c.cu[:1], c.bt[:0], c.cl[:0]
    assert c.run(most=1).shape == (2, 4, 128)
    c = Case(torch.float16, [20, 30], [1, 1], 4, 128, 32)
    assert bool((c.run(longest=0) == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,P", [(512, 64), (128, 32), (40, 8), (64, 0)])
def test_write_latent(dtype, R, P):
    g = torch.Generator().manual_seed(R)
    cache = torch.randn(9, 16, R + P, generator=g).to(dtype).to(dev())
    want = cache.clone()
    x = torch.randn(50, R + P + 8, generator=g).to(dtype).to(dev())
    slots = torch.randperm(144, generator=g)[:50].to(torch.int32)
    slots[[3, 20, 33]] = torch.tensor([-1, 144, 2 ** 31 - 1], dtype=torch.int32)
    ok = (slots >= 0) & (slots < 144)
    want.view(144, -1)[slots[ok].long().to(dev())] = x[ok.to(dev()), :R + P]
    memopt_C.write_latent(x[:, :R], x[:, R:R + P], slots.to(dev()), cache)  # views of one projection
    same_bits(cache.view(torch.int16), want.view(torch.int16).cpu().numpy())
    memopt_C.write_latent(x[:, 1:R + 1], x[:, 1:P + 1], slots.to(dev()), cache)  # off the alignment
    assert torch.equal(cache.view(144, -1)[slots[0].item()], torch.cat([x[0, 1:R + 1], x[0, 1:P + 1]]))
    memopt_C.write_latent(x[:0, :R], x[:0, R:R + P], slots[:0].to(dev()), cache)


def test_many_tokens_written():
    cache = torch.zeros(3000, 32, 576, dtype=torch.bfloat16, device=dev())
    x = torch.randn(90000, 576, device=dev()).bfloat16()
    slots = torch.randperm(96000, device=dev())[:90000].to(torch.int32)
    memopt_C.write_latent(x[:, :512], x[:, 512:], slots, cache)
    assert torch.equal(cache.view(-1, 576)[slots.long()], x)


def test_refusals():
    c = Case(torch.float16, [90, 40], [1, 1], 4, 128, 32)

    def call(out=None, **kw):
        a = {**dict(q=c.q, c=c.c, bt=c.bt, cl=c.cl, cu=c.cu, most=1, longest=96, rank=128), **kw}
        return memopt_C.latent_attention(a["q"], a["c"], a["bt"], a["cl"], a["cu"], a["most"], a["longest"], 0.1, a["rank"], out=out)

    o = torch.zeros(2, 4, 128, dtype=torch.float16, device=dev())
    for text, kw in [("query must be a CUDA", dict(q=c.q.cpu())), ("3-D", dict(q=c.q[0])), ("fp16 or bf16", dict(q=c.q.float())),
                     ("query's dtype", dict(c=c.c.bfloat16())), ("CUDA tensor", dict(c=c.c.cpu())), ("contiguous", dict(c=c.c[:, ::2])),
                     ("contiguous", dict(c=c.c[:, :, :96].contiguous())), ("rank", dict(rank=160)), ("rank", dict(rank=0)),
                     ("rank must be 128", dict(rank=64)), ("rope_dim", dict(q=c.q[:, :, :136], c=c.c[:, :, :136].contiguous())),
                     ("multiple of 16", dict(c=c.c[:, :8].contiguous())), ("no heads", dict(q=c.q[:, :0])),
                     ("cu_seqlens", dict(cu=c.cu.long())), ("context_lens", dict(cl=c.cl[:1])), ("block_tables", dict(bt=c.bt[:1])),
                     ("negative", dict(most=-1)), ("negative", dict(longest=-1)), ("out must be", dict(out=o[:, :, :64])),
                     ("out must be", dict(out=o.bfloat16())), ("overlap", dict(out=o[:, :1].expand(2, 4, 128))),
                     ("CUDA tensor", dict(out=o.cpu()))]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    with pytest.raises(RuntimeError, match="no gradients"):
        call(q=c.q.clone().requires_grad_())
    x, s = torch.zeros(5, 160, dtype=torch.float16, device=dev()), torch.zeros(5, dtype=torch.int32, device=dev())
    for text, args in [("latents must be a CUDA", (x[:, :128].cpu(), x[:, 128:], s, c.c)), ("2-D", (x[:4, :128], x[:, 128:], s, c.c)),
                       ("fp16 or bf16", (x[:, :128].float(), x[:, 128:], s, c.c)), ("dtype", (x[:, :128], x[:, 128:].bfloat16(), s, c.c)),
                       ("contiguous", (x[:, :120], x[:, 128:], s, c.c)), ("slot_mapping", (x[:, :128], x[:, 128:], s.long(), c.c)),
                       ("multiples of 8", (x[:, :124], x[:, 124:], s, c.c)), ("CUDA tensor", (x[:, :128], x[:, 128:], s, c.c.cpu()))]:
        with pytest.raises(RuntimeError, match=text):
            memopt_C.write_latent(*args)
