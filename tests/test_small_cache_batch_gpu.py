"""The operators that keep a cache small, together, as a serving loop uses them: PackedBatch with weights and compaction,
LatentBatch over prompts, chunks and decode steps."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import check
from small_cache_reference import latent, latent_tolerance, weight_sums
from test_packed_batch_gpu import cached, compare

pytestmark = pytest.mark.gpu


def R():
    import memopt_runtime
    return memopt_runtime


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=dev())


class Text:
    """One request's cached rows per head, on the host, with the weights that they got."""

    def __init__(self, Hk, D):
        self.k = np.zeros((0, Hk, D), np.float16)
        self.v = np.zeros((0, Hk, D), np.float16)
        self.w, self.tol = torch.zeros(Hk, 0, dtype=torch.float64), torch.zeros(Hk, 0, dtype=torch.float64)
        self.length = 0  # of the text

    def extend(self, k, v):
        n, Hk = len(k), self.k.shape[1]
        self.k, self.v = (np.concatenate([a, b.cpu().numpy()]) for a, b in ((self.k, k), (self.v, v)))
        z = torch.zeros(Hk, n, dtype=torch.float64)
        self.w, self.tol = torch.cat([self.w, z], 1), torch.cat([self.tol, z], 1)
        self.length += n

    def add(self, w, tol):
        self.w = self.w + w
        self.tol = self.tol + tol + 2.0 ** -23 * self.w

    def keep(self, kept):
        """kept [Hk, n]: the positions that stay, per head."""
        self.k, self.v = (np.stack([x[kept[h], h] for h in range(len(kept))], 1) for x in (self.k, self.v))
        self.w, self.tol = (torch.stack([x[h, kept[h]] for h in range(len(kept))]) for x in (self.w, self.tol))


@pytest.mark.parametrize("fmt", ["int4", "fp16"])
@pytest.mark.parametrize("Hq,Hk,D,window,sinks", [(8, 2, 64, -1, 0), (4, 1, 128, 60, 3)])
def test_a_loop_that_counts_and_compacts(fmt, Hq, Hk, D, window, sinks):
    n, rows = 4, 200
    batch = R().PackedBatch(60, Hk, D, n, 320, rows, kv_format=fmt, window_size=window, num_sink_tokens=sinks,
                            track_weights=True)
    g = torch.Generator().manual_seed(D)
    texts = [Text(Hk, D) for _ in range(n)]

    def step(new):
        q, k, v = (torch.randn(rows, h, D, generator=g).half().to(dev()) for h in (Hq, Hk, Hk))
        st = batch.advance(ints(*new))
        assert st.status.tolist() == [0] * n
        out = batch.attend(q, k, v, max_new=max(new))
        assert batch.accumulate(q, max_new=max(new)) is batch.weights
        at, where = 0, []
        for r, m in enumerate(new):
            t = texts[r]
            first, start = len(t.k), t.length
            t.extend(k[at:at + m], v[at:at + m])
            pos = first + np.arange(m)
            where += list(range(start, start + m))
            if m:
                compare(out[at:at + m], q[at:at + m], t.k, t.v, first, fmt, window, sinks, f"request {r}")
                t.add(*weight_sums(q[at:at + m], cached(t.k, fmt)[0], pos, window, sinks))
            check(batch.weights[r, :, :len(t.k)], t.w, t.tol, f"weights of {r}")
            assert bool((batch.weights[r, :, len(t.k):] == 0).all())
            at += m
        assert batch.token_positions().tolist() == where + [-1] * (rows - at)
        return st

    step([60, 40, 0, 90])
    step([1, 1, 30, 1])
    before = [batch.state.context_lens.tolist(), batch.tables.clone(), batch.weights.clone()]
    w = batch.weights.cpu()
    done = batch.compact([3, 0, 2], 32, num_sink_tokens=2, num_recent_tokens=8)
    assert done == [3, 0] and batch.state.context_lens.tolist() == [32, before[0][1], 30, 32]
    assert batch.removed.tolist() == [before[0][0] - 32, 0, 0, before[0][3] - 32]
    assert torch.equal(batch.tables[1:3], before[1][1:3]) and torch.equal(batch.weights[1:3], before[2][1:3])
    for r in (0, 3):
        c, kept = before[0][r], []
        for h in range(Hk):
            mid = np.argsort(-w[r, h, 2:c - 8].numpy(), kind="stable")[:22] + 2
            kept.append(np.sort(np.concatenate([np.arange(2), mid, np.arange(c - 8, c)])))
        texts[r].keep(kept)
    # no page is lost and none is there twice
    live = torch.cat([batch.tables[batch.tables >= 0],
                      batch.free_pages[(batch.state.free_span[0] + torch.arange(int(batch.state.free_span[1]), device=dev())) % 60]])
    assert sorted(live.tolist()) == list(range(60))
    for new in ([1, 1, 1, 1], [40, 0, 1, 7], [1, 1, 1, 1]):
        step(new)
    batch.release([0])
    assert bool((batch.weights[0] == 0).all()) and batch.removed.tolist()[0] == 0
    texts[0] = Text(Hk, D)
    step([17, 1, 0, 1])


def test_compaction_where_pages_are_short():
    """Six requests fill the pool but for three pages: they are compacted two by two, as pages come back."""
    batch = R().PackedBatch(63, 1, 64, 6, 160, 1000, track_weights=True)
    x = torch.randn(1000, 1, 64, device=dev()).half()
    q = torch.randn(1000, 2, 64, device=dev()).half()
    batch.advance(ints(*[160] * 6))
    batch.attend(q, x, x, max_new=160)
    batch.accumulate(q, max_new=160)
    assert batch.state.free_span.tolist()[1] == 3
    assert batch.compact([5, 1, 0, 2, 3, 4], 20) == [5, 1, 0, 2, 3, 4]  # 2 pages each
    assert batch.state.context_lens.tolist() == [20] * 6 and batch.state.free_span.tolist()[1] == 63 - 12
    assert len(set(batch.tables[batch.tables >= 0].tolist())) == 12
    full = R().PackedBatch(10, 1, 64, 1, 160, 160, track_weights=True)
    full.advance(ints(160))
    full.attend(q[:160], x[:160], x[:160])
    assert full.compact([0], 20) == [] and full.state.context_lens.tolist() == [160]  # not one page to move to
    assert full.compact([0], 0) == [0] and full.state.free_span.tolist()[1] == 10


def test_positions_outlast_a_compaction():
    """Where the step's rows stand in their texts does not change when tokens before them leave, and neither do the next
    rows' places; rows of a released request stand nowhere."""
    batch = R().PackedBatch(60, 1, 64, 3, 320, 200, track_weights=True)
    q, k = (torch.randn(200, h, 64, device=dev()).half() for h in (2, 1))
    for new in ([101, 20, 7], [1, 3, 0], [2, 1, 4]):
        batch.advance(ints(*new))
        batch.attend(q, k, k, max_new=max(new))
        batch.accumulate(q, max_new=max(new))
        rows = sum(new)
        want = batch.token_positions()
        assert bool((want[rows:] == -1).all()) and bool((want[:rows] >= 0).all())
        first = [int(n) for n in batch.state.context_lens + batch.removed]
        assert want[:rows].tolist() == [p for f, m in zip(first, new) for p in range(f - m, f)]
        batch.compact([0, 2], 5 if new[0] == 1 else 64, num_recent_tokens=1)
        assert torch.equal(batch.token_positions(), want)
    assert batch.removed.tolist()[0] > 0
    batch.release([0])
    assert batch.token_positions()[:rows].tolist() == [-1] * new[0] + want[new[0]:rows].tolist()


def test_a_full_pool_is_tried_once(monkeypatch):
    """All requests of a call keep the same number of tokens: where the first finds no room, none does."""
    batch = R().PackedBatch(40, 1, 64, 4, 160, 640, track_weights=True)
    batch.advance(ints(160, 160, 160, 160))
    assert batch.state.status.tolist() == [0] * 4
    calls, one = [], memopt_C.compact_cache
    monkeypatch.setattr("memopt_C.compact_cache", lambda *a, **kw: calls.append(1) or one(*a, **kw))
    assert batch.compact([2, 0, 1, 3], 20) == [] and len(calls) == 1
    assert batch.state.context_lens.tolist() == [160] * 4 and batch.state.free_span.tolist()[1] == 0
    batch.release([1])
    calls.clear()
    assert batch.compact([2, 0, 3], 20) == [2, 0, 3] and len(calls) == 1


@pytest.mark.parametrize("name", ["list", "generator", "empty"])
def test_released_requests_start_without_weights(name):
    batch = R().PackedBatch(40, 1, 64, 2, 160, 100, track_weights=True)
    x = torch.randn(100, 1, 64, device=dev()).half()
    batch.advance(ints(60, 40))
    batch.attend(x, x, x, max_new=60)
    batch.accumulate(x, max_new=60)
    batch.compact([0], 30)
    before = batch.weights.clone()
    batch.release({"list": [0, 0], "generator": (r for r in [0]), "empty": []}[name])
    gone = name != "empty"
    assert batch.removed.tolist() == [0 if gone else 30, 0]
    assert bool((batch.weights[0] == 0).all()) == gone and torch.equal(batch.weights[1], before[1])
    assert batch.state.context_lens.tolist() == [0 if gone else 30, 40]


def test_refusals():
    batch = R().PackedBatch(10, 1, 64, 2, 160, 20)
    q = torch.zeros(20, 1, 64, dtype=torch.float16, device=dev())
    for call in (lambda: batch.accumulate(q), lambda: batch.compact([0], 4)):
        with pytest.raises(RuntimeError, match="track_weights"):
            call()
    batch = R().PackedBatch(10, 1, 64, 2, 160, 20, track_weights=True)
    for text, call in [("num_rows", lambda: batch.accumulate(q[:3])), ("twice", lambda: batch.compact([0, 0], 4)),
                       ("no such", lambda: batch.compact([2], 4)), ("negative", lambda: batch.compact([0], -1))]:
        with pytest.raises(RuntimeError, match=text):
            call()
    assert batch.compact([], 4) == [] and batch.compact([0, 1], 4) == []
    L = R().LatentBatch
    for text, args in [("the pool must hold", (0, 128, 32, 1, 10, 10)), ("4096", (4, 128, 32, 0, 10, 10)), ("positive", (4, 128, 32, 1, 0, 10)),
                       ("rank must be", (4, 100, 32, 1, 10, 10)), ("rope_dim", (4, 128, 48, 1, 10, 10))]:
        with pytest.raises(RuntimeError, match=text):
            L(*args)
    with pytest.raises(RuntimeError, match="dtype"):
        L(4, 128, 32, 1, 10, 10, dtype=torch.float32)
    lat = L(4, 128, 32, 1, 10, 10)
    with pytest.raises(RuntimeError, match="num_rows"):
        lat.attend(torch.zeros(3, 2, 160, dtype=torch.bfloat16, device=dev()), None, None, 1.0)
    with pytest.raises(RuntimeError, match="no such"):
        lat.release([1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank,rope,H,window,sinks,bs", [(512, 64, 16, -1, 0, 16), (128, 32, 5, 50, 3, 32)])
def test_a_latent_loop(dtype, rank, rope, H, window, sinks, bs):
    n, rows = 5, 180
    batch = R().LatentBatch(60, rank, rope, n, 256, rows, block_size=bs, dtype=dtype, window_size=window, num_sink_tokens=sinks)
    g = torch.Generator().manual_seed(rank)
    scale = (64 + rope) ** -0.5
    held = [torch.zeros(0, rank + rope, dtype=dtype) for _ in range(n)]

    def rand(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(dev())

    def step(new, prompts=False):
        st = batch.advance(ints(*new))
        assert st.status.tolist() == [0] * n
        down = rand(rows, rank + rope)  # one projection gives both parts
        c, kr = down[:, :rank], down[:, rank:]
        if prompts:
            q, k, v = rand(rows, H, 64 + rope), rand(rows, H, 64), rand(rows, H, 64)
            out = batch.attend_prompts(q, k, c, kr, v)
            want = memopt_C.latent_prompt_attention(q, k, kr, v, st.cu_seqlens, window, num_sink_tokens=sinks)
            assert torch.equal(out[:sum(new)], want[:sum(new)])
        else:
            q = rand(rows, H, rank + rope)
            out = batch.attend(q, c, kr, scale, max_new=max(new))
        at = 0
        for r, m in enumerate(new):
            first = len(held[r])
            held[r] = torch.cat([held[r], down[at:at + m].cpu()])
            if m and not prompts:
                some = np.arange(m) if m <= 40 else np.unique(np.r_[0:15, m - 15:m])
                o, a, e = latent(q[at:at + m][some], held[r], first + some, rank, scale, window, sinks)
                check(out[at:at + m][some], o, latent_tolerance(o, a, e, len(held[r]), rank + rope, dtype), f"request {r}")
            at += m

    step([60, 33, 0, 5, 80], prompts=True)
    step([1, 1, 40, 1, 1])
    step([1, 0, 1, 100, 1])
    batch.release([3, 0])
    held[0] = held[3] = torch.zeros(0, rank + rope, dtype=dtype)
    assert batch.state.context_lens.tolist()[0] == 0
    step([70, 1, 1, 20, 1])
    step([1, 1, 1, 1, 1])


def test_a_captured_step_that_counts():
    batch = R().PackedBatch(40, 2, 64, 3, 200, 3, track_weights=True)
    q, k, v = (torch.randn(3, h, 64, device=dev()).half() for h in (8, 2, 2))
    one, out = ints(1, 1, 1), torch.zeros(3, 8, 64, dtype=torch.float16, device=dev())

    def step():
        batch.advance(one)
        batch.attend(q, k, v, max_new=1, out=out)
        batch.accumulate(q, max_new=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(20):
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert batch.state.context_lens.tolist() == [2 + i] * 3
    # every step gave each sequence and key head four rows' weight
    assert torch.allclose(batch.weights.sum(-1), torch.full((3, 2), 84.0, device=dev()), rtol=1e-5)
