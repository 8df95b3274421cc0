"""attention_scores against its 64-bit form: heads, row counts, masks, formats, in place, odd values, refusals."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import check
from small_cache_reference import weight_sums
from test_packed_gpu import Case

pytestmark = pytest.mark.gpu

FORMATS = ["int4", "fp16"]


def run(c, window=-1, sinks=0, most=None, longest=None, **kw):
    q, kc, _, bt, cl, cu = c.args()[:6]
    return memopt_C.attention_scores(q, kc, bt, cl, cu, max(c.qn, default=0) if most is None else most,
                                     max(1, c.M * c.bs) if longest is None else longest, window, num_sink_tokens=sinks, **kw)


def check_scores(c, out, window=-1, sinks=0, before=None, keys=None):
    """Every entry of out [B, Hk, L] against the 64-bit form; `keys`: tokens that are looked at."""
    a, L = 0, out.shape[2]
    for b, (ctx, n) in enumerate(zip(c.ctx, c.qn)):
        m = max(0, min(ctx, c.M * c.bs if keys is None else keys))
        pages = torch.from_numpy(c.tables[b, :-(-m // c.bs)]).long()
        live = ((pages >= 0) & (pages < c.k.shape[0])).repeat_interleave(c.bs)[:m]
        k = c.kval[pages.clamp(0, c.k.shape[0] - 1)].flatten(0, 1)[:m]
        w, tol = weight_sums(c.q[a:a + n], k, ctx - n + np.arange(n), window, sinks, live)
        a += n
        w, tol = (torch.nn.functional.pad(x, (0, max(0, L - m)))[:, :L] for x in (w, tol))
        old = torch.zeros_like(w) if before is None else before[b].double().cpu()
        want = old + w
        check(out[b], want, tol + 2.0 ** -23 * want.abs(), f"sequence {b}")


HEADS = [(8, 2, 64), (4, 4, 64), (5, 1, 128), (32, 8, 128), (16, 1, 64), (20, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D", HEADS)
def test_single_tokens(fmt, Hq, Hk, D):
    c = Case(fmt, [1, 15, 16, 17, 33, 100, 257, 64], [1] * 8, Hq, Hk, D, seed=Hq)
    check_scores(c, run(c))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 64), (10, 2, 128), (3, 3, 128), (16, 1, 64)])
@pytest.mark.parametrize("ctx,qn", [([50, 40, 300], [3, 0, 20]), ([128, 1, 90, 17], [128, 1, 33, 1]), ([5, 0, 7], [5, 0, 7]),
                                    ([2, 600], [4, 6]), ([40] * 70, [1, 0, 2, 3, 1] * 14), ([33], [17]), ([0, 9], [1, 0])],
                         ids=str)
def test_mixed_query_counts(fmt, Hq, Hk, D, ctx, qn):
    """None, one or many queries per sequence; more queries than context (the first see nothing and add nothing)."""
    c = Case(fmt, ctx, qn, Hq, Hk, D, seed=sum(qn) + D)
    check_scores(c, run(c))
    check_scores(c, run(c, most=10 ** 6))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 3), (100, 16), (100, 33), (5, 400), (2 ** 31 - 1, 2 ** 31 - 1),
                                          (0, 3)])
@pytest.mark.parametrize("D,qn", [(64, [1, 40, 7]), (128, [1, 40, 7]), (128, [1, 2, 3])])
def test_windows_and_sinks(fmt, window, sinks, D, qn):
    c = Case(fmt, [700, 90, 400], qn, 6, 2, D, seed=window % 100 + sinks % 7)
    check_scores(c, run(c, window, sinks), window if 0 < window <= c.M * 16 else c.M * 16, sinks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D,ctx,qn", [(8, 2, 64, [3000], [1]), (8, 1, 128, [5000, 100, 2500], [1, 1, 1]),
                                            (32, 8, 128, [1500], [1]), (4, 2, 64, [2500, 600], [40, 1]),
                                            (16, 1, 64, [6100], [1]), (8, 2, 128, [1300, 900], [200, 130]),
                                            (64, 1, 64, [600], [300])])
def test_long_contexts(fmt, Hq, Hk, D, ctx, qn):
    c = Case(fmt, ctx, qn, Hq, Hk, D, seed=7)
    first = run(c)
    check_scores(c, first)
    assert torch.equal(run(c), first)  # (one order of sums)
    check_scores(c, run(c, 700, 5), 700, 5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qn", [[1, 1, 1, 1], [1, 20, 3, 1]])
@pytest.mark.parametrize("D", [64, 128])
def test_unlinked_pages_and_entries_past_the_pool(fmt, qn, D):
    c = Case(fmt, [200, 48, 130, 30], qn, 8, 2, D, seed=3)
    c.tables[0, 3] = c.tables[0, 7] = c.tables[2, 8] = -1
    c.tables[1, 1] = 10 ** 6
    c.tables[2, 0] = -5
    c.tables[3, :] = -1  # nothing left
    c.load()
    out = run(c)
    check_scores(c, out)
    assert bool((out[3] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qn", [[1, 2, 1], [1, 60, 9]])
def test_adding_to_scores(fmt, qn):
    """In place, into another tensor, into fewer and into more positions than the contexts have."""
    c = Case(fmt, [300, 77, 16], qn, 8, 2, 64, seed=5)
    for L in (c.M * 16, 100, 1000):
        before = torch.rand(3, 2, L, device=dev())
        out = run(c, scores=before)
        check_scores(c, out, before=before)
        other = torch.full_like(before, float("nan"))
        assert run(c, scores=before, out=other) is other and torch.equal(other, out)
        twice = before.clone()
        assert run(c, scores=twice, out=twice) is twice and torch.equal(twice, out)
    sums = run(c)
    parts = run(c, out=torch.full((3, 2, 50), float("nan"), device=dev()))
    assert sums.shape == (3, 2, c.M * 16) and torch.equal(parts, sums[:, :, :50])
    assert torch.allclose(sums.sum(-1).cpu(), torch.tensor(qn).float()[:, None].expand(3, 2) * 4, rtol=1e-4)


@pytest.mark.parametrize("qn", [[1, 1], [20, 1]])
def test_no_rows_leaves_scores(qn):
    c = Case("int4", [90, 40], qn, 8, 2, 64)
    before = torch.rand(2, 2, 96, device=dev())
    q, kc, _, bt, cl, cu = c.args()[:6]
    for args in ((q[:0], kc, bt, cl, torch.zeros_like(cu), 5, 96), (q, kc, bt, cl, cu, 0, 96), (q, kc, bt, cl, cu, 5, 0)):
        assert torch.equal(memopt_C.attention_scores(*args, scores=before), before)
    assert memopt_C.attention_scores(q, kc, bt, cl, cu, 1, 0).shape == (2, 2, 0)
    none = memopt_C.attention_scores(q[:0], kc, bt[:0], cl[:0], cu[:1], 1, 96)
    assert none.shape == (0, 2, 96)


@pytest.mark.parametrize("most", [1, 30])
@pytest.mark.parametrize("given,meant", [([-5, 3, 2 ** 31 - 1], [0, 3, 30]), ([2, 1, 5], [1, 1, 5]), ([30, -1, 9], [0, 0, 9])])
def test_starts_out_of_range_or_order(given, meant, most):
    """Starts are held within the rows, and a sequence that would end before it begins has none."""
    c = Case("int4", [400, 90], [3, 27], 8, 2, 64, seed=2)
    outs = []
    for cu in (given, meant):
        c.cu = torch.tensor(cu, dtype=torch.int32, device=dev())
        outs.append(run(c, most=most))
    assert torch.equal(*outs)
    if meant[1] == meant[0]:
        assert not outs[0][0].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qn", [[1, 2, 1], [30, 20, 25]])
def test_contexts_outside_the_block_table_and_past_max_seq_len(fmt, qn):
    c = Case(fmt, [64, 64, 20], qn, 4, 2, 64, seed=3, M=4)
    c.ctx = [70, 1000, -3]
    c.load()
    check_scores(c, run(c, longest=2000), 2000, 0)
    c.ctx = [64, 40, 20]
    c.load()
    check_scores(c, run(c, longest=33, scores=torch.zeros(3, 2, 64, device=dev())), 33, 0, keys=33)


@pytest.mark.parametrize("bs", [16, 32, 48, 64])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_page_sizes(bs, D):
    c = Case("fp16", [630, 40, 97], [2, 40, 1], 4, 2, D, seed=bs, bs=bs)
    check_scores(c, run(c))
    c.qn = [1, 1, 1]
    c.cu = torch.arange(4, dtype=torch.int32, device=dev())
    check_scores(c, run(c))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qn", [[1, 1], [70, 33]])
def test_hidden_odd_keys_change_nothing(fmt, qn):
    """inf and NaN behind the context, outside the window and in pages of nobody."""
    c = Case(fmt, [330, 50], qn, 8, 2, 64, seed=4)
    want = run(c, 100, 4)
    lay = memopt_C.int4_layout(64)
    hidden = [(0, t) for t in range(4, 330 - qn[0] - 99)] + [(1, t) for t in (50, 55, 63)] + [(0, t) for t in range(330, 336)]
    for i, (b, t) in enumerate(hidden):
        bad = [float("nan"), float("inf"), -float("inf")][i % 3]
        page, row = int(c.tables[b, t // 16]), t % 16
        if fmt == "fp16":
            c.kc[page, row, :, 5] = bad
        else:
            c.kc.view(torch.float16)[page, :, lay["kscales"] // 2 + 2 * (row % 8) + row // 8] = bad
    assert torch.equal(run(c, 100, 4), want)
    # a NaN in sight: its rows' weights are NaN, other sequences keep theirs
    page = int(c.tables[0, 300 // 16])
    if fmt == "fp16":
        c.kc[page, 300 % 16, 0, 5] = float("nan")
    else:
        c.kc.view(torch.float16)[page, 0, lay["kscales"] // 2 + 2 * (300 % 8) + 300 % 16 // 8] = float("nan")
    out = run(c, 100, 4)
    assert torch.equal(out[1], want[1]) and torch.equal(out[0, 1], want[0, 1])
    assert bool(out[0, 0, 240:329 - qn[0]].isnan().all())


@pytest.mark.parametrize("ctx,qn", [(257, 1), (65, 1), (257, 20), (321, 20), (3, 1)])
def test_a_nan_alone_in_its_tile(ctx, qn):
    """The last key is NaN: the one row that sees it (with nothing else of its tile, or nothing at all but it) adds NaN to
    every key it sees, and so to all of its sequence."""
    c = Case("fp16", [ctx, 40], [qn, 1], 4, 2, 64, seed=4)
    c.kc[int(c.tables[0, (ctx - 1) // 16]), (ctx - 1) % 16, 0, 3] = float("nan")
    out = run(c)
    assert bool(out[0, 0, :ctx].isnan().all()) and not bool(out[0, 1].isnan().any()) and not bool(out[1].isnan().any())
    out = run(c, window=1)
    assert bool(out[0, 0, ctx - 1].isnan()) and int(out[0, 0].isnan().sum()) == 1


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qn", [[1, 3], [30, 41]])
def test_strided_and_far_query_rows(fmt, qn):
    c = Case(fmt, [200, 90], qn, 6, 2, 64, seed=8)
    want = run(c)
    plain = c.q
    T = sum(qn)
    wide = torch.zeros(T, 10, 64, dtype=torch.float16, device=dev())
    wide[:, 2:8] = plain
    c.q = wide[:, 2:8]
    assert torch.equal(run(c), want)
    c.q = plain.transpose(0, 1).contiguous().transpose(0, 1)  # head by head
    assert torch.equal(run(c), want)
    odd = torch.zeros(T * 6 * 64 + 3, dtype=torch.float16, device=dev())[3:].view(T, 6, 64)  # off the alignment
    odd.copy_(plain)
    c.q = odd
    assert torch.equal(run(c), want)
    far = torch.zeros(6 * 2 ** 27 + 64, dtype=torch.float16, device=dev()).as_strided((T, 6, 64), (64, 2 ** 27, 1))
    far.copy_(plain)
    c.q = far
    assert torch.equal(run(c), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 64), (16, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (90, 20)])
def test_rows_shared_by_workgroups(fmt, Hq, Hk, D, window, sinks):
    """256 rows and more per key head and few key tiles: parts of the rows are added up; adding in place, and to more
    and fewer positions than there are tiles for."""
    c = Case(fmt, [700, 513, 90, 0], [700, 300, 1, 0], Hq, Hk, D, seed=Hq + D)
    check_scores(c, run(c, window, sinks), window, sinks)
    for L in (100, 1500):
        before = torch.rand(4, Hk, L, device=dev())
        out = run(c, window, sinks, scores=before)
        check_scores(c, out, window, sinks, before=before)
        assert torch.equal(run(c, window, sinks, scores=before), out)
        assert torch.equal(run(c, window, sinks, scores=before, out=before), out)


def test_keys_past_4_gib():
    """Pages behind 4 GiB of the pool."""
    nb = 2 ** 32 // (16 * 1 * 128 * 2) + 40
    kc = torch.zeros(nb, 16, 1, 128, dtype=torch.float16, device=dev())
    c = Case("fp16", [200], [1], 4, 1, 128, seed=2)
    want = run(c)
    at = torch.arange(nb - c.M, nb, device=dev())
    kc[at] = c.kc[c.bt[0].long()]
    out = memopt_C.attention_scores(c.q, kc, at.to(torch.int32)[None], c.cl, c.cu, 1, c.M * 16)
    assert torch.equal(out, want)


@pytest.mark.parametrize("qn", [0, 1])
def test_batches_whose_weights_are_kept_in_groups(qn):
    """600 requests of up to 4096 tokens and 16 rows per key head: 1.26 GB of weights, more than are kept at a time."""
    rng = np.random.default_rng(3)
    ctx = rng.integers(1, 60, 600).tolist()
    ctx[3], ctx[500], ctx[599] = 1000, 700, 4096
    n = [qn or int(b % 3 == 0) for b in range(600)]
    c = Case("int4", ctx, n, 128, 8, 64, seed=5)
    assert c.M == 256
    before = torch.rand(600, 8, 4096, device=dev())
    out = run(c, scores=before)
    q, kc, _, bt, cl, cu = c.args()[:6]
    for a, z in ((0, 200), (200, 600)):  # (each half's weights are kept at once)
        first, last = sum(n[:a]), sum(n[:z])
        part = memopt_C.attention_scores(q[first:last], kc, bt[a:z], cl[a:z], cu[a:z + 1] - first, 1, 4096, scores=before[a:z])
        assert torch.equal(out[a:z], part)
    for b in (3, 499, 500, 599):
        first, m = sum(n[:b]), ctx[b]
        k = c.kval[torch.from_numpy(c.tables[b, :-(-m // 16)]).long()].flatten(0, 1)[:m]
        w, tol = weight_sums(c.q[first:first + n[b]], k, m - n[b] + np.arange(n[b]), -1, 0)
        want = before[b].double().cpu()
        want[:, :m] += w
        tol = torch.nn.functional.pad(tol, (0, 4096 - m))
        check(out[b], want, tol + 2.0 ** -23 * want.abs(), f"sequence {b}")
    assert run(c, scores=before, out=before) is before and torch.equal(before, out)


def test_pool_view_is_the_page_buffer():
    memopt_C.init_pool(20, 16, 2, 64, kv_format="int4")
    x = torch.randn(100, 2, 64, device=dev()).half()
    memopt_C.write_cache(x, x, None, torch.arange(100, dtype=torch.int32, device=dev()))
    q = torch.randn(1, 8, 64, device=dev()).half()
    bt = torch.arange(7, dtype=torch.int32, device=dev())[None]
    cl, cu = (torch.tensor(v, dtype=torch.int32, device=dev()) for v in ([100], [0, 1]))
    a = memopt_C.attention_scores(q, memopt_C.get_key_pool(), bt, cl, cu, 1, 112)
    b = memopt_C.attention_scores(q, memopt_C.get_int4_pages(), bt, cl, cu, 1, 112)
    assert torch.equal(a, b) and abs(float(a.sum()) - 8) < 1e-4


@pytest.mark.parametrize("qn", [[1, 1, 1], [40, 1, 33]])
def test_captured_calls_and_other_streams(qn):
    """Replays follow the tensors' contents; calls on two streams at once have workspaces of their own."""
    c = Case("int4", [500, 70, 33], qn, 8, 2, 64, seed=6)
    acc = torch.zeros(3, 2, c.M * 16, device=dev())
    one = run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(c, scores=acc)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(c, scores=acc, out=acc)
    assert bool((acc == 0).all())
    want = torch.zeros_like(acc)
    for i in range(3):
        g.replay()
        want = run(c, scores=want)
        torch.cuda.synchronize()
        assert torch.equal(acc, want)
        c.q.copy_(torch.randn_like(c.q))
    c.q.copy_(torch.from_numpy(np.random.default_rng(1).standard_normal(tuple(c.q.shape)).astype(np.float16)))
    one, got = run(c), []
    for _ in range(8):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(run(c))
        got.append(run(c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, one) for x in got)


def test_refusals():
    c = Case("fp16", [90, 40], [1, 1], 8, 2, 64)
    q, kc, _, bt, cl, cu = c.args()[:6]
    good = dict(q=q, kc=kc, bt=bt, cl=cl, cu=cu, most=1, longest=96)

    def call(scores=None, out=None, **kw):
        a = {**good, **kw}
        return memopt_C.attention_scores(a["q"], a["kc"], a["bt"], a["cl"], a["cu"], a["most"], a["longest"], scores=scores,
                                         out=out)

    f32 = torch.zeros(2, 2, 96, device=dev())
    for text, kw in [("query must be a CUDA", dict(q=q.cpu())), ("query must be fp16", dict(q=q.float())),
                     ("query must be fp16", dict(q=q[0])), ("CUDA tensor", dict(kc=kc.cpu())),
                     ("key_cache must be fp16", dict(kc=kc.float())), ("contiguous", dict(kc=kc[:, ::2])),
                     ("contiguous", dict(kc=kc[..., :32].contiguous())), ("multiple of num_kv_heads", dict(q=q[:, :7])),
                     ("cu_seqlens", dict(cu=cu.long())), ("context_lens", dict(cl=cl[:1])), ("block_tables", dict(bt=bt[:1])),
                     ("block_tables", dict(bt=bt[0])), ("negative", dict(most=-1)), ("negative", dict(longest=-1)),
                     ("scores must be", dict(scores=f32[:1])), ("scores must be", dict(scores=f32.double())),
                     ("scores must be", dict(scores=torch.zeros(2, 2, 192, device=dev())[:, :, ::2])),
                     ("out must be", dict(scores=f32, out=f32[:, :, :50])), ("out must be", dict(out=f32.half())),
                     ("CUDA tensor", dict(out=f32.cpu())), ("INT4", dict(kc=kc.view(torch.uint8))),
                     ("16 tokens", dict(kc=kc.view(-1, 8, 2, 64)))]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    with pytest.raises(RuntimeError, match="no gradients"):
        call(q=q.clone().requires_grad_())
    with torch.no_grad():
        call(q=q.clone().requires_grad_())
