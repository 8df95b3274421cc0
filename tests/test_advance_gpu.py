"""advance_batch against a request-by-request form: placements, refusals in order, rings, in-place steps, graphs."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import advance

pytestmark = pytest.mark.gpu


def state(rng, B, M, bs, most_ctx, spare):
    ctx = rng.integers(0, most_ctx + 1, B).astype(np.int32)
    have = -(-ctx // bs)
    C = int(have.sum()) + spare + 3
    pages = rng.permutation(C).astype(np.int32)
    tables = np.full((B, M), -1, np.int32)
    at = 0
    for b in range(B):
        tables[b, :have[b]] = pages[at:at + have[b]]
        at += have[b]
    ring = np.full(C, -7, np.int32)
    head = int(rng.integers(0, C))
    ring[(head + np.arange(spare)) % C] = pages[at:at + spare]
    return ctx, tables, ring, np.array([head, spare], np.int32)


def run(new, ctx, tables, ring, span, bs, rows):
    d = [torch.from_numpy(np.ascontiguousarray(x)).to(dev()) for x in (new, ctx, tables, ring, span)]
    r = memopt_C.advance_batch(*d, bs, rows)
    assert torch.equal(d[1].cpu(), torch.from_numpy(ctx)) and torch.equal(d[4].cpu(), torch.from_numpy(span))
    return (d[2], r.context_lens, r.free_span, r.cu_seqlens, r.slots, r.positions, r.status)


def same(got, want):
    for name, g, w in zip(("tables", "ctx", "span", "cu", "slots", "positions", "status"), got, want):
        assert np.array_equal(g.cpu().numpy(), w), name


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 255, 256, 257, 1024, 1025, 2500, 4096])
@pytest.mark.parametrize("bs", [16, 32, 1])
def test_decode_steps(B, bs):
    rng = np.random.default_rng(B)
    ctx, tables, ring, span = state(rng, B, 40, bs, 39 * bs, B)
    new = (rng.random(B) < 0.9).astype(np.int32)
    same(run(new, ctx, tables, ring, span, bs, B), advance(new, ctx, tables, ring, span, bs, B))


@pytest.mark.parametrize("B,most", [(1, 5000), (7, 40), (60, 700), (300, 200), (1100, 33)])
@pytest.mark.parametrize("pressure", ["none", "pages", "rows", "both"])
def test_mixed_counts_and_pressure(B, most, pressure):
    rng = np.random.default_rng(B + most)
    bs, M = 16, (most + 600) // 16
    new = (rng.integers(0, most + 1, B) * (rng.random(B) < 0.8)).astype(np.int32)
    spare = int((new // bs + 1).sum())
    ctx, tables, ring, span = state(rng, B, M, bs, 500, spare // 2 if pressure in ("pages", "both") else spare)
    rows = int(new.sum()) // (2 if pressure in ("rows", "both") else 1) + (5 if pressure == "none" else 0)
    want = advance(new, ctx, tables, ring, span, bs, rows)
    same(run(new, ctx, tables, ring, span, bs, rows), want)
    if B > 1 and pressure == "pages":
        assert (want[6] == 3).any() and (want[6][new > 0] == 0).any()
    if B > 1 and pressure == "rows":
        assert (want[6] == 4).any()


def test_every_status():
    bs, M = 16, 4
    ctx = np.array([10, 64, 60, -1, 5, 20, 16, 0, 30, 3], np.int32)
    new = np.array([3, 1, 5, 2, -4, 1, 1, 20, 1, 100], np.int32)
    tables = np.arange(40, dtype=np.int32).reshape(10, 4)
    tables[5, 1] = -1
    ring = np.arange(100, 120, dtype=np.int32)
    for count, rows in [(20, 40), (1, 40), (0, 40), (20, 4), (20, 0), (-3, 40), (10 ** 9, 40)]:
        for head in (0, 19, 45, -1):
            span = np.array([head, count], np.int32)
            same(run(new, ctx, tables, ring, span, bs, rows), advance(new, ctx, tables, ring, span, bs, rows))
    assert sorted(set(advance(new, ctx, tables, ring, np.array([0, 1], np.int32), bs, 4)[6])) == [0, 1, 2, 3, 4]


def test_sums_that_pass_32_bits():
    """What 1200 requests ask for adds up past 2^32 rows; only those before the sum passes the rows are served."""
    new = np.tile(np.array([1, 2 ** 24, 2 ** 24 - 5, 0], np.int32), 300)
    ctx, tables = np.zeros(1200, np.int32), np.full((1200, 8), -1, np.int32)
    ring, span = np.arange(64, dtype=np.int32), np.array([3, 64], np.int32)
    for bs in (2 ** 21, 2 ** 27):
        got = run(new, ctx, tables, ring, span, bs, 100)
        same(got, advance(new, ctx, tables, ring, span, bs, 100))


def test_slots_past_32_bits_are_skipped():
    """A page whose slots do not fit int32 gives slot -1 (which the writers skip), never a wrapped one."""
    ring, span = np.array([2 ** 27 + 1, 2 ** 27 - 1], np.int32), np.array([0, 2], np.int32)
    got = run(np.array([16, 16], np.int32), np.zeros(2, np.int32), np.full((2, 1), -1, np.int32), ring, span, 16, 32)
    slots = got[4].cpu().numpy()
    assert (slots[:16] == -1).all() and (slots[16:] == (2 ** 27 - 1) * 16 + np.arange(16)).all()


def test_in_place_steps_in_a_graph():
    """Ten decode steps replayed from one captured call, advanced in place, against the plain form."""
    rng = np.random.default_rng(1)
    B, bs, M = 33, 16, 20
    ctx, tables, ring, span = state(rng, B, M, bs, 100, 40)
    new = np.ones(B, np.int32)
    dn, dc, dt, dr, ds = (torch.from_numpy(x).to(dev()) for x in (new, ctx, tables, ring, span))
    buf = memopt_C.advance_batch_buffers(B, B + 4, dev())
    buf = buf.replace(context_lens=dc, free_span=ds)
    memopt_C.advance_batch(dn, dc, dt, dr, ds, bs, out=buf)
    for d, x in ((dc, ctx), (dt, tables), (ds, span)):
        d.copy_(torch.from_numpy(x))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        memopt_C.advance_batch(dn, dc, dt, dr, ds, bs, out=buf)
    for step in range(10):
        new = rng.integers(0, 3, B).astype(np.int32) if step % 3 == 2 else np.ones(B, np.int32)
        dn.copy_(torch.from_numpy(new))
        graph.replay()
        torch.cuda.synchronize()
        want = advance(new, ctx, tables, ring, span, bs, B + 4)
        same((dt, buf.context_lens, buf.free_span, buf.cu_seqlens, buf.slots, buf.positions, buf.status), want)
        tables, ctx, span = want[:3]


def test_rows_of_their_own_launch():
    rng = np.random.default_rng(2)
    new = np.array([9000, 0, 1, 4000, 17], np.int32)
    ctx, tables, ring, span = state(rng, 5, 700, 16, 300, 900)
    for rows in (8192, 8193, 14000):
        same(run(new, ctx, tables, ring, span, 16, rows), advance(new, ctx, tables, ring, span, 16, rows))


def test_refusals():
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev())  # noqa: E731
    ok = [z(3), z(3), z(3, 4), z(9), z(2)]

    def refused(match, args, *rest, **kw):
        with pytest.raises(RuntimeError, match=match):
            memopt_C.advance_batch(*args, *rest, **kw)

    refused("num_rows or out", ok, 16)
    refused("CUDA", [ok[0].cpu()] + ok[1:], 16, 4)
    refused("CUDA", ok[:3] + [ok[3].cpu(), ok[4]], 16, 4)
    refused("int32", [ok[0].long()] + ok[1:], 16, 4)
    refused("context_lens", [ok[0], z(4)] + ok[2:], 16, 4)
    refused("block_tables", ok[:2] + [z(4, 4)] + ok[3:], 16, 4)
    refused("block_tables", ok[:2] + [z(3, 8)[:, ::2]] + ok[3:], 16, 4)
    refused("free_span", ok[:4] + [z(3)], 16, 4)
    refused("sizes must be positive", ok, 0, 4)
    refused("sizes must be positive", [z(0), z(0), z(0, 4), z(9), z(2)], 16, 4)
    refused("sizes must be positive", [z(3), z(3), z(3, 4), z(0), z(2)], 16, 4)
    refused("4096 requests", [z(4097), z(4097), z(4097, 4), z(9), z(2)], 16, 4)
    refused("2\\^31", ok, 2 ** 30, 4)
    refused("differs", ok, 16, 4, out=memopt_C.advance_batch_buffers(3, 5, dev()))
    refused("another device or number", ok, 16, out=memopt_C.advance_batch_buffers(4, 5, dev()))
    for field, t, match in [("status", z(2), "status"), ("slots", z(6), "positions"), ("slots", z(5).cpu(), "CUDA"),
                            ("positions", z(10)[::2], "positions"), ("context_lens", z(3).long(), "context_lens")]:
        with pytest.raises(RuntimeError, match=match):
            memopt_C.advance_batch_buffers(3, 5, dev()).replace(**{field: t})
    with pytest.raises(TypeError):
        memopt_C.advance_batch_buffers(3, 5, dev()).replace(rows=z(5))


def test_a_step_s_tensors_are_exchanged_by_replace_alone():
    """The addresses are taken when the step is made, so a field that could be assigned would not be written to."""
    step = memopt_C.advance_batch_buffers(3, 8, dev())
    for name in memopt_C.BatchStep.FIELDS + ("device",):
        with pytest.raises(AttributeError):
            setattr(step, name, getattr(step, name))
    slots = torch.full((8,), 7, dtype=torch.int32, device=dev())
    other = step.replace(slots=slots)
    assert other.slots is slots and step.slots is not slots and other.cu_seqlens is step.cu_seqlens
    i32 = dict(dtype=torch.int32, device=dev())
    memopt_C.advance_batch(torch.tensor([2, 0, 1], **i32), torch.zeros(3, **i32), torch.full((3, 2), -1, **i32),
                           torch.arange(4, **i32), torch.tensor([0, 4], **i32), 16, out=other)
    assert slots.tolist() == [0, 1, 16, -1, -1, -1, -1, -1]
