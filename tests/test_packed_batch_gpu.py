"""The packed operators together, as a serving loop uses them: PackedBatch over prompts, chunks, decode steps, refusals,
releases and a captured step; grouped heads through PolicyForward and autochunk_prefill. Against 64-bit forms that
keep every request's rows on the host."""
import numpy as np
import oracle as O
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import attend, check, quantized_scores, tolerance

pytestmark = pytest.mark.gpu

FORMATS = ["int4", "fp16"]


def R():
    import memopt_runtime
    return memopt_runtime


def cached(rows, fmt):
    """What the cache holds of rows [n, H, D]: (values in 64 bits, the largest scale)."""
    if fmt == "fp16":
        return torch.from_numpy(rows).double(), 0.0
    n, H, D = rows.shape
    pool = np.zeros((-(-n // 16), 16, H, D), np.float16)
    pool.reshape(-1, H, D)[:n] = rows
    codes, scales = O.int4_pages_split(O.to_int4_pages(pool, pool), D)[:2]
    c = torch.from_numpy(O.unpack_codes(codes).reshape(*codes.shape[:3], D).astype(np.float64)) - 8
    s = torch.from_numpy(scales.astype(np.float64))
    v = (c.unflatten(-1, (-1, 64)) * s[..., None]).flatten(-2)
    return v.flatten(0, 1)[:n], float(s[:n].max()) if n else 0.0


def compare(got, q, k, v, first, fmt, window, sinks, what):
    """Rows `got` for queries q at positions first .. over the host rows k, v (fp16 arrays [n, H, D])."""
    D = q.shape[2]
    kk, ks = cached(k, fmt)
    vv, vs = cached(v, fmt)
    o, a, e = attend(q, kk, vv, first + np.arange(len(q)), window, sinks)
    scores = quantized_scores(q, ks, False) if fmt == "int4" else 0.0
    check(got.cpu(), o, tolerance(o, a, e, len(k), D, torch.float16, torch.float16, False, scores, vs), what)


class Host:
    """The requests' rows, kept on the host."""

    def __init__(self, n, Hk, D):
        self.k = [np.zeros((0, Hk, D), np.float16) for _ in range(n)]
        self.v = [np.zeros((0, Hk, D), np.float16) for _ in range(n)]

    def extend(self, r, k, v):
        self.k[r], self.v[r] = (np.concatenate([a, b.cpu().numpy()]) for a, b in ((self.k[r], k), (self.v[r], v)))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Hq,Hk,D,window,sinks", [(8, 2, 64, -1, 0), (4, 1, 128, 50, 3)])
def test_serving_loop(fmt, Hq, Hk, D, window, sinks):
    n, rows = 6, 240
    rng = torch.Generator().manual_seed(D)
    batch = R().PackedBatch(40, Hk, D, n, 400, rows, kv_format=fmt, window_size=window, num_sink_tokens=sinks)
    assert memopt_C.free_blocks_count() == 0
    host = Host(n, Hk, D)

    def step(want, prompts=False, status=None):
        new = torch.tensor([want.get(r, 0) for r in range(n)], dtype=torch.int32, device=dev())
        s = batch.advance(new)
        q, k, v = (torch.randn((rows, h, D), generator=rng).half().to(dev()) for h in (Hq, Hk, Hk))
        cu, got = s.cu_seqlens.tolist(), s.status.tolist()
        assert got == [(status or {}).get(r, 0) for r in range(n)]
        for t in (q, k, v):
            t[cu[-1]:] = float("nan")  # rows of no request
        out = torch.full((rows, Hq, D), 7.0, dtype=torch.float16, device=dev())
        assert batch.attend(q, k, v, prompts=prompts, out=out) is out
        assert bool((out[cu[-1]:] == 7).all())
        for r in range(n):
            a, b, first = cu[r], cu[r + 1], len(host.k[r])
            assert b - a == (0 if got[r] else want.get(r, 0))
            if a == b:
                continue
            assert s.positions[a:b].tolist() == list(range(first, first + b - a))
            host.extend(r, k[a:b], v[a:b])
            compare(out[a:b], q[a:b], host.k[r], host.v[r], first, "fp16" if prompts else fmt, window, sinks,
                    f"request {r}")
        assert s.context_lens.tolist() == [len(x) for x in host.k]

    step({0: 40, 2: 1, 5: 100}, prompts=True)
    step({0: 1, 1: 70, 2: 1, 5: 1})                       # decode steps beside a chunk
    for _ in range(3):
        step({0: 1, 1: 1, 2: 1, 5: 1})
    step({0: 1, 1: 90, 3: 16, 4: 2})
    free = int(batch.state.free_span[1])
    # request 2: past max_tokens. Request 5: 104 + 256 tokens are 16 pages more, all that were free, and request 3
    # (16 + 1 tokens) took one of them.
    assert free == 16
    step({0: 1, 2: 500, 3: 1, 5: 256}, status={2: 1, 5: 3})
    # 15 pages are free: request 1 (163 + 200 tokens) takes 12, request 4 (2 + 41) needs 2, but rows 201 .. 241 of 240.
    step({1: 200, 4: 41}, status={4: 4})
    batch.release([0, 5, 0])
    for r in (0, 5):
        host.k[r], host.v[r] = host.k[r][:0], host.v[r][:0]
    step({0: 33, 2: 1, 5: 17})
    step({0: 1, 1: 1, 2: 1, 3: 1, 4: 1, 5: 1})
    batch.release(range(n))
    assert batch.state.free_span[1] == 40 and sorted(batch.free_pages.tolist()) == list(range(40))
    assert bool((batch.tables == -1).all())


def test_pages_that_do_not_last():
    batch = R().PackedBatch(4, 1, 64, 3, 64, 64)
    new = torch.tensor([30, 30, 1], dtype=torch.int32, device=dev())
    assert batch.advance(new).status.tolist() == [0, 0, 3]
    batch.release([1])
    assert batch.advance(torch.tensor([1, 0, 30], dtype=torch.int32, device=dev())).status.tolist() == [0, 0, 0]
    with pytest.raises(RuntimeError, match="no such request"):
        batch.release([3])


def ring(batch):
    """The free pages, front first."""
    head, count = batch.state.free_span.tolist()
    pages = batch.free_pages.tolist()
    return [pages[(head + i) % len(pages)] for i in range(count)]


class Evicting:
    """Requests of 90 and 40 tokens over 12 pages, and scores that evict tokens 16 .. 47 of the first in every head."""

    def __init__(self, fmt):
        self.fmt, self.rng = fmt, torch.Generator().manual_seed(8)
        self.batch = R().PackedBatch(12, 2, 64, 3, 112, 96 + 44, kv_format=fmt)
        self.host = Host(3, 2, 64)
        self.live = [np.ones(112, bool) for _ in range(3)]
        self.step({0: 90, 1: 40})
        self.scores = torch.arange(90, 0, -1, dtype=torch.float32, device=dev()).repeat(1, 2, 1)
        self.scores[:, :, 16:48] -= 200
        self.ratio = 0.64  # ceil(57.6) = 58 of 90 stay

    def step(self, want):
        b = self.batch
        s = b.advance(torch.tensor([want.get(r, 0) for r in range(3)], dtype=torch.int32, device=dev()))
        assert s.status.tolist() == [0, 0, 0]
        q, k, v = (torch.randn((b.num_rows, h, 64), generator=self.rng).half().to(dev()) for h in (8, 2, 2))
        out, cu = b.attend(q, k, v), s.cu_seqlens.tolist()
        for r in want:
            x, y, first = cu[r], cu[r + 1], len(self.host.k[r])
            self.host.extend(r, k[x:y], v[x:y])
            n = len(self.host.k[r])
            (kk, ks), (vv, vs) = cached(self.host.k[r], self.fmt), cached(self.host.v[r], self.fmt)
            o, a, e = attend(q[x:y], kk, vv, np.arange(first, n), -1, 0, torch.from_numpy(self.live[r][:n]))
            scores = quantized_scores(q[x:y], ks, False) if self.fmt == "int4" else 0.0
            check(out[x:y], o, tolerance(o, a, e, n, 64, torch.float16, torch.float16, False, scores, vs), f"request {r}")


@pytest.mark.parametrize("fmt", FORMATS)
def test_release_of_a_request_with_evicted_pages(fmt):
    """The holes that eviction leaves in a block table are no pages to give back."""
    e = Evicting(fmt)
    held = [p for p in e.batch.tables[0].tolist() if p >= 0]
    votes = torch.zeros(12, dtype=torch.int32, device=dev())
    memopt_C.evict_tokens(e.scores, e.batch.tables[:1], votes, e.ratio, 0)
    assert e.batch.tables[0].tolist() == [held[0], -1, -1, *held[3:], -1]
    before = ring(e.batch)
    e.batch.release([0])
    assert ring(e.batch) == before + [held[0], *held[3:]]
    e.host.k[0], e.host.v[0] = e.host.k[0][:0], e.host.v[0][:0]
    e.step({2: 112, 1: 1})  # all seven pages
    assert ring(e.batch) == [] and int(e.batch.tables[2].min()) >= 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_evict_release_and_admit_again(fmt):
    """Pages that PackedBatch.evict frees are in the ring once, and serve other requests."""
    e = Evicting(fmt)
    held = e.batch.tables[0].tolist()
    before = ring(e.batch)
    assert e.batch.evict([0], e.scores, e.ratio) == sorted(held[1:3])
    assert ring(e.batch) == before + sorted(held[1:3])
    assert e.batch.tables[0].tolist() == [held[0], -1, -1, *held[3:]]
    e.live[0][16:48] = False
    e.step({0: 7, 1: 1})    # (request 0 goes on: 97 tokens, one page more)
    e.step({2: 60, 0: 1})   # the ring's last two, and the two that were freed
    assert sorted(ring(e.batch)) == [] and set(held[1:3]) <= set(e.batch.tables[2].tolist())
    e.batch.release([0])
    e.host.k[0], e.host.v[0] = e.host.k[0][:0], e.host.v[0][:0]
    e.live[0][:] = True
    e.step({0: 70, 1: 1, 2: 1})
    e.batch.release([0, 1, 2])
    assert sorted(ring(e.batch)) == list(range(12))


def test_evict_refusals():
    e = Evicting("int4")
    for match, requests, scores in [("no such request", [3], e.scores), ("twice", [0, 0], e.scores.repeat(2, 1, 1)),
                                    ("scores", [0, 1], e.scores), ("scores", [1], e.scores), ("scores", [2], e.scores),
                                    ("scores", [0], e.scores[0])]:
        with pytest.raises(RuntimeError, match=match):
            e.batch.evict(requests, scores, 0.5)
    assert e.batch.evict([], e.scores[:0], 0.5) == []
    assert len(ring(e.batch)) == 3


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("planned", [True, False])
def test_captured_step(fmt, planned):
    """advance_batch, write_cache and a plan (or the eager call) in one graph, replayed as the requests grow across
    pages."""
    n, Hq, Hk, D = 5, 8, 2, 64
    batch = R().PackedBatch(60, Hk, D, n, 160, n, kv_format=fmt)
    host = Host(n, Hk, D)
    rng = torch.Generator().manual_seed(1)
    q, k, v = (torch.empty((n, h, D), dtype=torch.float16, device=dev()) for h in (Hq, Hk, Hk))
    new = torch.zeros(n, dtype=torch.int32, device=dev())
    out = torch.empty_like(q)
    plan = batch.attend_plan(q, max_new=2, out=out)

    def work():
        batch.advance(new)
        if planned:
            memopt_C.write_cache(k, v, None, batch.state.slots, validate_slots=False)
            assert plan() is out
        else:
            batch.attend(q, k, v, max_new=2, out=out)

    work()  # (nothing new: no rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for i in range(40):
        want = [1] * n if i % 7 else [1, 0, 2, 0, 1]
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=rng))
        new.copy_(torch.tensor(want, dtype=torch.int32))
        if i == 5:
            work()  # an eager step between replays
        else:
            graph.replay()
        cu = batch.state.cu_seqlens.tolist()
        assert cu == np.concatenate([[0], np.cumsum(want)]).tolist()
        for r in range(n):
            a, b, first = cu[r], cu[r + 1], len(host.k[r])
            host.extend(r, k[a:b], v[a:b])
            if b > a and i % 6 == 0:
                compare(out[a:b], q[a:b], host.k[r], host.v[r], first, fmt, -1, 0, f"replay {i} request {r}")
    assert batch.state.context_lens.tolist() == [len(x) for x in host.k]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(-1, 0), (40, 4)])
def test_grouped_heads_through_the_runtime(fmt, window, sinks):
    """autochunk_prefill, then PolicyForward steps of one and three tokens, with four query heads per cache head."""
    Hq, Hk, D, S = 8, 2, 64, 150
    rng = torch.Generator().manual_seed(3)

    def rand(*shape):
        return torch.randn(shape, generator=rng).half().to(dev())

    cache = R().PagedKVCache(40, Hk, D, kv_format=fmt)
    host = Host(2, Hk, D)
    for s in (0, 1):
        cache.add_sequence(s)
        q, k, v = rand(S, Hq, D), rand(S, Hk, D), rand(S, Hk, D)
        out = R().autochunk_prefill(cache, s, q, k, v, window, sinks, chunk_tokens=64)
        host.extend(s, k, v)
        for a in range(0, S, 64):
            b = min(S, a + 64)
            compare(out[a:b], q[a:b], host.k[s][:b], host.v[s][:b], a, fmt, window, sinks, f"chunk at {a}")
    forward = R().PolicyForward(cache, type("P", (), {"retain_ratio": 1.0, "use_int4": fmt == "int4"}), window, sinks)
    for T in (1, 3, 1):
        q, k, v = rand(2, T, Hq, D), rand(2, T, Hk, D), rand(2, T, Hk, D)
        out = forward.step([0, 1], q, k, v)
        assert out.shape == q.shape
        for s in (0, 1):
            first = len(host.k[s])
            host.extend(s, k[s], v[s])
            compare(out[s], q[s], host.k[s], host.v[s], first, fmt, window, sinks, f"sequence {s}")
    with pytest.raises(RuntimeError, match="multiple"):
        forward.attend([0, 1], rand(2, 1, 3, D))


@pytest.mark.parametrize("fmt", FORMATS)
def test_grouped_prefill_stays_within_its_budget(fmt):
    """Memory that a chunk call takes beside the prompt's own tensors, and its queries and outputs, fit the budget."""
    Hq, Hk, D, S, budget = 32, 8, 128, 512, 20 << 20
    cache = R().PagedKVCache(S // 16 + 2, Hk, D, kv_format=fmt)
    cache.add_sequence(0)
    q, k, v = (torch.randn((S, h, D), device=dev()).half() for h in (Hq, Hk, Hk))
    chunk = R().chunk_tokens_for_budget(budget, S, Hq, D, num_kv_heads=Hk, kv_format=fmt)
    assert chunk < S
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = R().autochunk_prefill(cache, 0, q, k, v, budget_bytes=budget)
    taken = torch.cuda.max_memory_allocated() - before - out.numel() * 2
    assert taken + 4 * chunk * Hq * D <= budget + 65536  # (the index tensors)
    first = S - 40
    compare(out[first:], q[first:], k.cpu().numpy(), v.cpu().numpy(), first, fmt, -1, 0, "the last rows")


@pytest.mark.parametrize("fmt", FORMATS)
def test_attend_before_the_first_advance(fmt):
    """No request has rows yet: nothing is written, whatever the step's memory held."""
    dirty = [torch.ones(n, dtype=torch.int32, device=dev()) for n in (3, 2, 4, 8, 8, 3) * 4]
    del dirty
    batch = R().PackedBatch(4, 1, 64, 3, 32, 8, kv_format=fmt)
    assert batch.state.cu_seqlens.tolist() == [0] * 4 and batch.state.context_lens.tolist() == [0] * 3
    assert batch.state.slots.tolist() == [-1] * 8 and batch.state.positions.tolist() == [-1] * 8
    pages = [x.clone() for x in (memopt_C.get_key_pool(), memopt_C.get_value_pool())]
    q = torch.randn((8, 4, 64), device=dev()).half()
    out = torch.full_like(q, 7.0)
    for prompts in (False, True):
        batch.attend(q, q[:, :1], q[:, 1:2], prompts=prompts, out=out)
    assert bool((out == 7).all())
    assert all(torch.equal(a, b) for a, b in zip(pages, (memopt_C.get_key_pool(), memopt_C.get_value_pool())))


def test_refusals():
    for match, kw in [("2\\^31", dict(num_blocks=2 ** 28)), ("2\\^31", dict(num_blocks=0)), ("4096", dict(num_requests=4097)),
                      ("4096", dict(num_requests=0)), ("positive", dict(max_tokens=0)), ("positive", dict(num_rows=0)),
                      ("head_dim", dict(head_dim=32)), ("head_dim", dict(block_size=8)),
                      ("head_dim", dict(block_size=32, kv_format="int4"))]:
        args = dict(num_blocks=4, num_kv_heads=1, head_dim=64, num_requests=2, max_tokens=32, num_rows=8)
        with pytest.raises(RuntimeError, match=match):
            R().PackedBatch(**{**args, **kw})
    batch = R().PackedBatch(4, 1, 64, 2, 32, 8)
    q = torch.zeros((4, 1, 64), dtype=torch.float16, device=dev())
    with pytest.raises(RuntimeError, match="num_rows=8"):
        batch.attend(q, q, q)
