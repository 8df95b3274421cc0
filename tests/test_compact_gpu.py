"""compact_cache against its definition, bit for bit: which tokens stay, where they go, the ring, refused requests."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C, same_bits
from small_cache_reference import compact

pytestmark = pytest.mark.gpu

FORMATS = ["int4", "fp16"]


class Cache:
    """A pool of random bytes (no NaN among fp16 rows matters: rows are moved as bits), tables, a ring and scores."""

    def __init__(self, fmt, ctx, Hk, D, seed=0, bs=16, spare_pages=40, M=None, L=None, scores="few ties"):
        rng = np.random.default_rng(seed)
        self.fmt, self.bs, self.Hk, self.D = fmt, bs, Hk, D
        self.ctx = np.array(ctx, np.int32)
        per = [-(-max(c, 0) // bs) for c in ctx]
        N, self.M = len(ctx), M or max(per, default=1) + 1
        self.nb = sum(per) + spare_pages
        pages = rng.permutation(self.nb).astype(np.int32)
        self.tables = np.full((N, self.M), -1, np.int32)
        at = 0
        for b in range(N):
            k = min(per[b], self.M)
            self.tables[b, :k] = pages[at:at + k]
            at += per[b]
        self.head = int(rng.integers(0, self.nb))
        self.ring = np.full(self.nb, -7, np.int32)
        free = pages[at:]
        self.ring[(self.head + np.arange(len(free))) % self.nb] = free
        self.span = np.array([self.head, len(free)], np.int32)
        if fmt == "int4":
            self.pools = [rng.integers(0, 256, (self.nb, Hk, 17 * D), dtype=np.uint8)]
        else:
            self.pools = [rng.integers(0, 2 ** 16, (self.nb, bs, Hk, D), dtype=np.uint16).view(np.float16) for _ in range(2)]
        self.L = L or self.M * bs
        x = rng.standard_normal((N, Hk, self.L))
        self.scores = (np.round(x * 3) if scores == "ties" else x).astype(np.float32)

    def run(self, keep, sinks, recent, K=None, out=None):
        K = max(1, max(keep, default=1)) if K is None else K
        t = [torch.from_numpy(x.copy()).to(dev()) for x in self.pools]
        ring, span = (torch.from_numpy(x.copy()).to(dev()) for x in (self.ring, self.span))
        r = memopt_C.compact_cache(*(torch.from_numpy(x).to(dev()) for x in (self.scores,)), t[0], t[-1],
                                   *(torch.from_numpy(x).to(dev()) for x in (self.tables, self.ctx, np.array(keep, np.int32))),
                                   ring, span, num_sink_tokens=sinks, num_recent_tokens=recent,
                                   **(dict(max_keep=K) if out is None else dict(out=out)))
        want = compact(self.scores, self.pools, self.fmt, self.tables, self.ctx, np.array(keep, np.int32), self.ring,
                       self.span, self.nb, self.bs, K, sinks, recent)
        for got, w in zip((r.status, r.context_lens, r.free_span, r.block_tables, r.kept, r.scores, ring), (
                want[5], want[1], want[2], want[0], want[4], want[3], want[6])):
            same_bits(got, w)
        for got, w in zip(t, want[7]):
            same_bits(got, w)
        assert span.cpu().tolist() == self.span.tolist()
        return r, want


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hk,D", [(2, 64), (1, 128), (8, 128), (5, 64)])
@pytest.mark.parametrize("scores", ["ties", "few ties"])
def test_requests_of_many_lengths(fmt, Hk, D, scores):
    c = Cache(fmt, [1, 15, 16, 17, 33, 100, 257, 64, 0], Hk, D, seed=Hk + D, scores=scores)
    for keep, sinks, recent in [([0, 1, 15, 16, 32, 40, 33, 64, 0], 4, 8), ([5] * 9, 0, 0), ([17] * 9, 4, 100),
                                ([3] * 9, 100, 1), ([50, -1, 3, -5, 12, 99, 256, 63, 7], 1, 1)]:
        c.run(keep, sinks, recent)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ctx,keep", [([5000, 1024, 3001], [1000, 1023, 2999]), ([9000], [8999]), ([20000], [77]),
                                      ([1025, 1023], [1024, 1])])
def test_long_contexts(fmt, ctx, keep):
    c = Cache(fmt, ctx, 2, 64, seed=ctx[0], spare_pages=800, scores="ties")
    c.run(keep, 4, 64)
    c.run(keep, 0, 0)


def test_a_context_of_100000_tokens():
    c = Cache("int4", [100003], 1, 64, seed=1, spare_pages=2000)
    x = np.abs(c.scores)
    c.scores = np.where(x < 0.3, np.float32(0), x)
    order = np.lexsort((np.arange(4, 99503), -c.scores[0, 0, 4:99503]))[:30000 - 504] + 4
    want = np.sort(np.concatenate([np.arange(4), order, np.arange(99503, 100003)]))
    pages = torch.from_numpy(c.pools[0]).to(dev())
    r = memopt_C.compact_cache(torch.from_numpy(c.scores).to(dev()), pages, pages,
                               *(torch.from_numpy(x).to(dev()) for x in (c.tables, c.ctx, np.array([30000], np.int32), c.ring,
                                                                         c.span)), num_recent_tokens=500, max_keep=30000)
    assert r.status.tolist() == [0]
    assert np.array_equal(r.kept[0, 0].cpu().numpy(), want)
    assert np.array_equal(r.scores[0, 0, :30000].cpu().numpy(), c.scores[0, 0, want])


@pytest.mark.parametrize("fmt", FORMATS)
def test_scores_of_every_kind(fmt):
    """inf, NaN of both signs, -0 beside 0, subnormals, negatives; all alike."""
    c = Cache(fmt, [300, 290, 310], 2, 64, seed=3)
    special = np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-40, -1e-40, 3.4e38, -3.4e38], np.float32)
    c.scores[0] = special[np.random.default_rng(1).integers(0, 10, c.scores[0].shape)]
    c.scores[1] = np.float32(0.25)
    c.scores[2, 0] = np.nan
    c.scores[2, 1] = -np.inf
    for keep in (1, 40, 150, 280):
        c.run([keep] * 3, 4, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_unlinked_pages_leave(fmt, D):
    """Tokens of pages that are not linked are not there: not among the sinks, the last ones or the best."""
    c = Cache(fmt, [200, 150, 90, 64], 2, D, seed=5)
    c.tables[0, [0, 5, 12]] = [-1, -9, c.nb]
    c.tables[1, 9] = -1
    c.tables[3, :] = -1
    for keep in ([100, 60, 89, 1], [152, 150, 10, 0], [151, 134, 90, 64], [3, 2, 1, 0]):
        c.run(keep, 8, 20)


@pytest.mark.parametrize("bs", [16, 32, 48])
def test_fp16_page_sizes(bs):
    c = Cache("fp16", [200, 97, 48], 2, 64, seed=bs, bs=bs)
    c.run([70, 96, 47], 4, 10)
    c.run([32, 33, 16], 0, 0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_that_do_not_last(fmt):
    """Requests are served in order while what all of them so far ask for lasts; the ring's room counts as well."""
    c = Cache(fmt, [100, 200, 90, 300], 2, 64, seed=6, spare_pages=9)
    r, _ = c.run([60, 96, 40, 16], 4, 4)  # 4 + 6 (no) + 3 + 1 pages
    assert r.status.tolist() == [0, 3, 3, 3]
    r, _ = c.run([60, -1, 40, 16], 4, 4)
    assert r.status.tolist() == [0, 2, 0, 0]
    c.span[1] = 0
    assert c.run([60, 96, 40, 0], 4, 4)[0].status.tolist() == [3, 3, 3, 3]
    c = Cache(fmt, [100, 100], 2, 64, seed=6, spare_pages=30)
    c.ring = c.ring[:37].copy()  # (a ring smaller than the pool: room for one request's 7 pages)
    c.ring[:] = np.setdiff1d(np.arange(c.nb), c.tables)[:1]
    free = np.setdiff1d(np.arange(c.nb), c.tables).astype(np.int32)
    c.span = np.array([3, len(free)], np.int32)
    c.ring[(3 + np.arange(len(free))) % 37] = free
    assert c.run([20, 20], 4, 4)[0].status.tolist() == [0, 3]


@pytest.mark.parametrize("fmt", FORMATS)
def test_rings_wrap_and_spans_out_of_range(fmt):
    for head in (-3, 0, 40, 10 ** 9):
        c = Cache(fmt, [100, 80], 2, 64, seed=8, spare_pages=30)
        free = c.ring[(c.head + np.arange(30)) % c.nb].copy()
        c.ring[:] = -7
        c.ring[(head + np.arange(30)) % c.nb] = free
        c.span[0] = head
        c.run([50, 33], 4, 4)
    c.span[1] = 10 ** 9  # (no more than the ring holds: nothing can come back)
    assert c.run([50, 33], 4, 4)[0].status.tolist() == [3, 3]
    c.span[1] = -5
    assert c.run([50, 33], 4, 4)[0].status.tolist() == [3, 3]


def test_ring_entries_that_are_no_pages():
    c = Cache("int4", [100, 80], 2, 64, seed=8, spare_pages=30)
    c.ring[(c.head + 1) % c.nb] = -1
    c.ring[(c.head + 2) % c.nb] = c.nb + 5
    c.run([50, 33], 4, 4)


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_listed_twice(fmt):
    """In one request or in two: neither is compacted, whatever the other asks for."""
    c = Cache(fmt, [100, 200, 90, 300, 50], 2, 64, seed=6)
    c.tables[0, 3] = c.tables[1, 7]
    c.tables[3, 2] = c.tables[3, 9]
    assert c.run([60, 96, 40, 16, 20], 4, 4)[0].status.tolist() == [4, 4, 0, 4, 0]
    assert c.run([60, -1, 40, 16, 20], 4, 4)[0].status.tolist() == [4, 4, 0, 4, 0]
    c.tables[1, 7] = -1
    c.tables[0, 6] = c.tables[2, 5]  # the last, partial pages
    assert c.run([60, 96, 40, 16, 20], 4, 4)[0].status.tolist() == [4, 0, 4, 4, 0]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("why", ["keep", "scores"])
@pytest.mark.parametrize("refused", [0, 1])
def test_pages_shared_with_a_refused_request(fmt, why, refused):
    """A request whose `keep` or length the call does not take still holds its pages: who shares one keeps it too."""
    ctx = [100, 100, 90]
    ctx[refused] = 200
    c = Cache(fmt, ctx, 2, 64, seed=6, L=250 if why == "keep" else 150)
    other = 1 - refused
    lost = int(c.tables[other, 3])
    c.tables[other, 3] = c.tables[refused, 7]
    keep = [40, 40, 40]
    if why == "keep":
        keep[refused] = 60
    t = [torch.from_numpy(x.copy()).to(dev()) for x in c.pools]
    ring, span, tables = (torch.from_numpy(x.copy()).to(dev()) for x in (c.ring, c.span, c.tables))
    scores, lens = torch.from_numpy(c.scores).to(dev()), torch.from_numpy(c.ctx).to(dev())
    r = memopt_C.compact_cache(scores, t[0], t[-1], tables, lens, torch.tensor(keep, dtype=torch.int32, device=dev()), ring,
                               span, num_recent_tokens=4, max_keep=50)
    status = [4, 4, 0]
    status[refused] = 1
    assert r.status.tolist() == status
    assert torch.equal(r.block_tables[:2], tables[:2]) and torch.equal(r.scores[:2], scores[:2])
    assert r.context_lens.tolist() == ctx[:2] + [40] and bool((r.kept[:2] == -1).all())
    head, count = r.free_span.tolist()
    free = ring[(head + torch.arange(count, device=dev())) % c.nb].tolist()
    held = set(r.block_tables[r.block_tables >= 0].tolist())
    assert not held & set(free) and held | set(free) | {lost} == set(range(c.nb)) and len(set(free)) == count


@pytest.mark.parametrize("fmt", FORMATS)
def test_invalid_requests(fmt):
    c = Cache(fmt, [100, 200, 90, 60], 2, 64, seed=6, M=14, L=150)
    c.ctx[2] = -4
    r, _ = c.run([60, 96, 40, 59], 4, 4, K=59)
    assert r.status.tolist() == [1, 1, 1, 0]
    c.ctx[:] = [10 ** 9, 2 ** 31 - 1, -2 ** 31, 60]
    assert c.run([60, 96, 40, 59], 4, 4, K=100)[0].status.tolist() == [1, 1, 1, 0]


def test_many_requests():
    rng = np.random.default_rng(4)
    ctx = rng.integers(0, 60, 1500).tolist()
    c = Cache("int4", ctx, 1, 64, seed=1, spare_pages=900)
    c.run(rng.integers(-2, 30, 1500).tolist(), 2, 4)
    c = Cache("int4", [3] * 4096, 1, 64, seed=1, spare_pages=3000)
    c.run([1] * 4096, 1, 0)


def test_kept_buffers_and_empty_calls():
    c = Cache("int4", [100, 80], 2, 64, seed=2)
    out = memopt_C.compact_cache_buffers(2, 2, c.M, c.L, 64, dev())
    for t in (getattr(out, n) for n in out.FIELDS):
        t.fill_(77)
    for keep in ([50, 33], [64, -1], [0, 0]):
        r, _ = c.run(keep, 4, 4, K=64, out=out)
        assert r is out
    with pytest.raises(AttributeError):
        out.kept = out.kept
    none = Cache("int4", [], 2, 64, M=3, L=48)
    r, _ = none.run([], 4, 4, K=5)
    assert r.kept.shape == (0, 2, 5) and r.free_span.tolist() == none.span.tolist()
    none = Cache("fp16", [0, 0], 2, 64)
    none.run([0, 0], 4, 4, K=0)


def test_captured_calls_and_other_streams():
    c = Cache("int4", [700, 90, 333], 2, 64, seed=9)
    args = [torch.from_numpy(x).to(dev()) for x in (c.scores, c.pools[0])]
    args += [args[1]] + [torch.from_numpy(x).to(dev()) for x in (c.tables, c.ctx, np.array([100, 50, 64], np.int32), c.ring,
                                                                  c.span)]
    out = memopt_C.compact_cache_buffers(3, 2, c.M, c.L, 128, dev())
    start = args[1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        memopt_C.compact_cache(*args, out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        memopt_C.compact_cache(*args, out=out)
    for i in range(3):
        args[0].copy_(torch.randn_like(args[0]))
        args[1].copy_(start)
        g.replay()
        got = [x.clone() for x in (out.kept, out.scores, out.block_tables, out.context_lens, out.free_span, args[1])]
        args[1].copy_(start)
        r = memopt_C.compact_cache(*args, max_keep=128)
        torch.cuda.synchronize()
        for x, y in zip(got, (r.kept, r.scores, r.block_tables, r.context_lens, r.free_span, args[1])):
            assert torch.equal(x, y)


def test_attention_over_a_compacted_cache_is_attention_over_what_stayed():
    """Dropping the tokens of weight zero changes nothing: scores say which, keys far below the others."""
    rng = np.random.default_rng(0)
    ctx, Hk, D = 200, 2, 64
    memopt_C.init_pool(40, 16, Hk, D, kv_format="int4")
    k = rng.standard_normal((ctx, Hk, D)).astype(np.float16)
    dead = rng.permutation(np.arange(4, 190))[:100]
    k[dead] = np.float16(-30)  # queries are positive
    kt, vt = (torch.from_numpy(x).to(dev()) for x in (k, rng.standard_normal((ctx, Hk, D)).astype(np.float16)))
    memopt_C.write_cache(kt, vt, None, torch.arange(ctx, dtype=torch.int32, device=dev()))
    q = torch.rand(1, 4, D, device=dev()).half() + 1
    bt = torch.full((1, 20), -1, dtype=torch.int32, device=dev())
    bt[0, :13] = torch.arange(13)
    cl, cu = (torch.tensor(x, dtype=torch.int32, device=dev()) for x in ([ctx], [0, 1]))
    kc, vc = memopt_C.get_pool_tensors()
    before = memopt_C.packed_attention(q, kc, vc, bt, cl, cu, 1, 320)
    scores = memopt_C.attention_scores(q, kc, bt, cl, cu, 1, 320)
    assert bool((scores[:, :, torch.from_numpy(dead).to(dev())] == 0).all())
    ring = torch.arange(40, dtype=torch.int32, device=dev())
    span = torch.tensor([13, 27], dtype=torch.int32, device=dev())
    keep = torch.tensor([100], dtype=torch.int32, device=dev())
    r = memopt_C.compact_cache(scores, kc, vc, bt, cl, keep, ring, span, num_recent_tokens=10, max_keep=100)
    assert r.status.tolist() == [0] and r.context_lens.tolist() == [100]
    assert not np.intersect1d(r.kept.cpu().numpy(), dead).size
    after = memopt_C.packed_attention(q, kc, vc, r.block_tables, r.context_lens, cu, 1, 320)
    # the same weights summed in another order; one rounding of the output
    assert torch.allclose(after.float(), before.float(), rtol=2 ** -9, atol=1e-4)
    again = memopt_C.attention_scores(q, kc, r.block_tables, r.context_lens, cu, 1, 320)
    assert torch.allclose(again[:, :, :100], r.scores[:, :, :100], rtol=1e-4, atol=1e-7)


def test_refusals():
    c = Cache("fp16", [90, 40], 2, 64)
    base = [torch.from_numpy(x).to(dev()) for x in (c.scores, c.pools[0], c.pools[1], c.tables, c.ctx,
                                                    np.array([50, 20], np.int32), c.ring, c.span)]
    names = ["scores", "kc", "vc", "bt", "cl", "keep", "ring", "span"]

    def call(**kw):
        a = dict(zip(names, base))
        opts = {k: kw.pop(k) for k in ("max_keep", "out") if k in kw} or dict(max_keep=64)
        a.update(kw)
        return memopt_C.compact_cache(*(a[n] for n in names), **opts)

    s, kc, vc, bt, cl, keep, ring, span = base
    out = memopt_C.compact_cache_buffers(2, 2, c.M, c.L, 64, dev())
    for text, kw in [("scores must be a CUDA", dict(scores=s.cpu())), ("f32", dict(scores=s.double())),
                     ("f32", dict(scores=s[:, :, ::2])), ("CUDA tensor", dict(kc=kc.cpu())), ("context_lens", dict(cl=cl.long())),
                     ("context_lens", dict(cl=cl[:1])), ("keep", dict(keep=keep[:1])), ("block_tables", dict(bt=bt[:1])),
                     ("free_pages", dict(ring=ring.long())), ("free_pages", dict(ring=ring[::2])), ("free_span", dict(span=ring)),
                     ("fp16 or INT4", dict(kc=kc.float())), ("contiguous", dict(kc=kc[:, :, :1], vc=vc[:, :, :1])),
                     ("contiguous", dict(vc=vc[:4])), ("INT4", dict(kc=kc.view(torch.uint8))),
                     ("not an INT4", dict(kc=kc.view(torch.uint8).view(c.nb, 2, -1), vc=vc.view(torch.uint8).view(c.nb, 2, -1))),
                     ("max_keep or out", dict(max_keep=None)), ("max_keep or out", dict(max_keep=-1)),
                     ("differs", dict(max_keep=63, out=out)), ("other sizes", dict(out=out, bt=bt[:, :-1].contiguous())),
                     ("more of them kept", dict(max_keep=c.L + 1)),
                     ("16 tokens", dict(kc=kc.view(-1, 8, 2, 64), vc=vc.view(-1, 8, 2, 64))),
                     ("head_dim", dict(kc=kc.view(-1, 32, 2, 32), vc=vc.view(-1, 32, 2, 32))),
                     ("must not overlap", dict(out=memopt_C.CompactStep(bt, out.context_lens, out.free_span, out.scores,
                                                                        out.kept, out.status))),
                     ("must not overlap", dict(out=memopt_C.CompactStep(out.block_tables, cl, out.free_span, out.scores,
                                                                        out.kept, out.status))),
                     ("must not overlap", dict(out=memopt_C.CompactStep(out.block_tables, out.context_lens, out.free_span, s,
                                                                        out.kept, out.status)))]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    with pytest.raises(RuntimeError, match="kept"):
        memopt_C.CompactStep(out.block_tables, out.context_lens, out.free_span, out.scores, out.kept[:1], out.status)
    with pytest.raises(RuntimeError, match="CUDA"):
        memopt_C.CompactStep(out.block_tables.cpu(), out.context_lens, out.free_span, out.scores, out.kept, out.status)
    call(out=memopt_C.CompactStep(out.block_tables, out.context_lens, span, out.scores, out.kept, out.status))


def test_refusals_of_page_buffers_name_the_call():
    """A page buffer that is not contiguous, or two of them, given to any operator over INT4 pages."""
    c = Cache("int4", [90, 40], 2, 64)
    wide = torch.zeros(c.nb, 2, 17 * 64 + 8, dtype=torch.uint8, device=dev())
    pages = wide[:, :, :17 * 64].contiguous()
    s, bt, cl, ring, span = (torch.from_numpy(x).to(dev()) for x in (c.scores, c.tables, c.ctx, c.ring, c.span))
    keep, cu = (torch.tensor(x, dtype=torch.int32, device=dev()) for x in ([50, 20], [0, 1, 2]))
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=dev())
    calls = {"compact_cache": lambda k, v: memopt_C.compact_cache(s, k, v, bt, cl, keep, ring, span, max_keep=60),
             "packed_attention": lambda k, v: memopt_C.packed_attention(q, k, v, bt, cl, cu, 1, 96),
             "attention_scores": lambda k, v: memopt_C.attention_scores(q, k, bt, cl, cu, 1, 96),
             "dynamic_sparse_attention": lambda k, v: memopt_C.dynamic_sparse_attention(
                 q[:, None, :2].contiguous(), k, v, bt, cl, 96, -1)}
    for name, call in calls.items():
        with pytest.raises(RuntimeError, match=f"^{name}: INT4 page buffer must be contiguous"):
            call(wide[:, :, :17 * 64], wide[:, :, :17 * 64])
        if name != "attention_scores":
            with pytest.raises(RuntimeError, match=f"^{name}: pass the INT4 page buffer as both"):
                call(pages, pages.clone())
