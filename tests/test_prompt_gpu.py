"""prompt_attention against its 64-bit form: lengths, head layouts, types, strides, masks, streams, graphs, refusals."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import check_prompt, starts

pytestmark = pytest.mark.gpu


def make(T, Hq, Hk, D, dtype, seed, fused=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, Hq + 2 * Hk, D), generator=g).to(dtype).to(dev())
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
    return (q, k, v) if fused else tuple(t.contiguous() for t in (q, k, v))


def cu_of(lens, first=0):
    return torch.from_numpy(starts(lens, first)).to(dev())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [32], [33, 64, 65], [127, 128, 129, 0, 5], [0, 257, 0], [300, 1, 190]],
                         ids=str)
def test_lengths(dtype, D, lens):
    q, k, v = make(sum(lens), 4, 2, D, dtype, sum(lens) + D)
    check_prompt(memopt_C.prompt_attention(q, k, v, cu_of(lens)), q, k, v, lens, -1, 0)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (3, 1), (8, 8), (12, 4), (16, 8), (20, 4), (16, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts(Hq, Hk, D):
    lens = [70, 20, 131]
    q, k, v = make(sum(lens), Hq, Hk, D, torch.float16, Hq + Hk, fused=True)
    check_prompt(memopt_C.prompt_attention(q, k, v, cu_of(lens)), q, k, v, lens, -1, 0)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (63, 4), (64, 64), (65, 70), (100, 16), (200, 5),
                                          (1000, 3), (5, 1000), (-1, 4), (0, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_windows_and_sinks(window, sinks, D):
    lens = [333, 40, 150]
    q, k, v = make(sum(lens), 2, 1, D, torch.float16, 5)
    out = memopt_C.prompt_attention(q, k, v, cu_of(lens), window, num_sink_tokens=sinks)
    check_prompt(out, q, k, v, lens, window, sinks)


@pytest.mark.parametrize("count,most", [(70, 9), (300, 4), (257, 40)])
def test_many_sequences(count, most):
    lens = np.random.default_rng(count).integers(0, most, count).tolist()
    q, k, v = make(sum(lens), 2, 1, 64, torch.bfloat16, count)
    check_prompt(memopt_C.prompt_attention(q, k, v, cu_of(lens)), q, k, v, lens, -1, 0)


@pytest.mark.parametrize("D", [64, 128])
def test_long_rows_of_large_scores(D):
    """Scores far apart (the running maximum rises again and again) on a few thousand keys."""
    lens = [1500]
    q, k, v = make(1500, 1, 1, D, torch.float16, 3)
    k = (k * torch.linspace(0.1, 6.0, 1500, device=dev())[:, None, None]).half()
    check_prompt(memopt_C.prompt_attention(q, k, v, cu_of(lens)), q, k, v, lens, -1, 0)


def test_strides_that_are_read_in_place_and_others():
    lens = [90, 45]
    T = sum(lens)
    q, k, v = make(T, 4, 2, 64, torch.float16, 9)
    want = memopt_C.prompt_attention(q, k, v, cu_of(lens))
    check_prompt(want, q, k, v, lens, -1, 0)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]  # [H, T, D] in memory
    odd = [torch.empty((T, t.shape[1], 65), dtype=t.dtype, device=dev())[..., :64].copy_(t) for t in (q, k, v)]
    every_other = [torch.empty((T, t.shape[1], 128), dtype=t.dtype, device=dev())[..., ::2].copy_(t) for t in (q, k, v)]
    wide = [torch.empty((T, 3 * t.shape[1], 96), dtype=t.dtype, device=dev())[:, ::3, 8:72].copy_(t) for t in (q, k, v)]
    for ins in (heads_first, odd, every_other, wide):
        assert torch.equal(memopt_C.prompt_attention(*ins, cu_of(lens)), want)
    one = k[:, :1].expand(T, 2, 64)  # one key head seen as two: head stride 0
    assert torch.equal(memopt_C.prompt_attention(q, one, v, cu_of(lens)),
                       memopt_C.prompt_attention(q, one.contiguous(), v, cu_of(lens)))
    same = k[:1].expand(T, 2, 64)  # one token seen as all: token stride 0
    assert torch.equal(memopt_C.prompt_attention(q, same, v, cu_of(lens)),
                       memopt_C.prompt_attention(q, same.contiguous(), v, cu_of(lens)))
    buf = torch.full((T, 4, 128), 7.0, dtype=torch.float16, device=dev())
    assert memopt_C.prompt_attention(q, k, v, cu_of(lens), out=buf[..., 64:]).data_ptr() == buf[..., 64:].data_ptr()
    assert torch.equal(buf[..., 64:], want) and bool((buf[..., :64] == 7).all())


def shifted(t):
    """A contiguous tensor with t's values at an address that no 16 divide."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)[4:4 + t.numel()]
    assert flat.data_ptr() % 16 == 8
    return flat.view(t.shape).copy_(t)


def test_contiguous_inputs_off_the_alignment_are_copied():
    lens = [90, 45]
    q, k, v = make(135, 4, 2, 64, torch.float16, 9)
    want = memopt_C.prompt_attention(q, k, v, cu_of(lens))
    for i in range(3):
        ins = [shifted(t) if i == j else t for j, t in enumerate((q, k, v))]
        assert torch.equal(memopt_C.prompt_attention(*ins, cu_of(lens)), want)
    assert torch.equal(memopt_C.prompt_attention(*(shifted(t) for t in (q, k, v)), cu_of(lens)), want)


def test_token_strides_past_the_kernels_range():
    """Rows 2^23 elements apart and more (a position of a [tokens, positions, heads, head_dim] buffer)."""
    lens = [2, 1]
    q, k, v = make(3, 4, 2, 64, torch.float16, 9)
    want = memopt_C.prompt_attention(q, k, v, cu_of(lens))
    for stride in (2 ** 23 - 8, 2 ** 23, 2 ** 23 + 8):
        far = [torch.empty(3 * stride, dtype=t.dtype, device=dev()).as_strided(t.shape, (stride, 64, 1)).copy_(t)
               for t in (q, k, v)]
        assert torch.equal(memopt_C.prompt_attention(*far, cu_of(lens)), want)


def test_outputs_whose_rows_overlap_are_refused():
    """Every (token, head) row has a place of its own in ``out``, in whichever order tokens and heads lie."""
    lens = [9, 11]
    q, k, v = make(20, 4, 2, 64, torch.float16, 9)
    want = memopt_C.prompt_attention(q, k, v, cu_of(lens))
    for strides in ((256, 64), (64, 1280), (512, 128), (72, 1440), (320, 80), (64, 1288), (256, 64 * 20 * 4)):
        out = torch.empty(2 ** 15, dtype=q.dtype, device=dev()).as_strided(q.shape, (*strides, 1))
        assert torch.equal(memopt_C.prompt_attention(q, k, v, cu_of(lens), out=out), want)
    for strides in ((64, 64), (64, 128), (128, 64), (248, 64), (64, 1272), (192, 128), (64, 0)):
        out = torch.empty(2 ** 15, dtype=q.dtype, device=dev()).as_strided(q.shape, (*strides, 1))
        with pytest.raises(RuntimeError, match="overlap"):
            memopt_C.prompt_attention(q, k, v, cu_of(lens), out=out)
    one = torch.empty(2 ** 12, dtype=q.dtype, device=dev())
    for shape, strides in (((1, 4, 64), (64, 64)), ((20, 1, 64), (64, 8)), ((1, 1, 64), (64, 0))):
        t, h, _ = shape
        n = [t]
        a, b, c = q[:t, :h].contiguous(), k[:t, :1].contiguous(), v[:t, :1].contiguous()
        out = one.as_strided(shape, (*strides, 1))
        assert torch.equal(memopt_C.prompt_attention(a, b, c, cu_of(n), out=out),
                           memopt_C.prompt_attention(a, b, c, cu_of(n)))


def test_rows_of_no_sequence_stay_as_they_are():
    """Padding before, between (none can be) and behind the sequences is neither read nor written."""
    lens, first, T = [40, 100], 7, 160
    q, k, v = make(T, 2, 1, 64, torch.float16, 4)
    for t in (q, k, v):
        t[:first] = float("nan")
        t[first + 140:] = float("nan")
    out = torch.full_like(q, 3.0)
    memopt_C.prompt_attention(q, k, v, cu_of(lens, first), out=out)
    check_prompt(out, q, k, v, lens, -1, 0, first)
    assert bool((out[:first] == 3).all()) and bool((out[first + 140:] == 3).all())
    memopt_C.prompt_attention(q, k, v, cu_of([0, 0]), out=out)  # nothing at all
    assert memopt_C.prompt_attention(q, k, v, cu_of([])).shape == q.shape
    assert memopt_C.prompt_attention(q[:0], k[:0], v[:0], cu_of([0])).shape == (0, 2, 64)


def test_starts_outside_the_rows_are_clamped():
    q, k, v = make(50, 2, 1, 64, torch.float16, 4)
    cu = torch.tensor([-5, 30, 1000], dtype=torch.int32, device=dev())
    check_prompt(memopt_C.prompt_attention(q, k, v, cu), q, k, v, [30, 20], -1, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (40, 3)])
def test_odd_values_reach_only_the_rows_that_see_them(dtype, D, window, sinks):
    """NaN and inf in a key or value: rows that do not see that token are those of the values without it."""
    n = 200
    q, k, v = make(n, 2, 1, D, dtype, 8)
    i = torch.arange(n)
    for token, bad, where in [(150, float("nan"), "v"), (150, float("inf"), "v"), (64, float("-inf"), "v"),
                              (31, float("nan"), "k"), (127, float("nan"), "kv"), (0, float("nan"), "v")]:
        k2, v2 = k.clone(), v.clone()
        if "k" in where:
            k2[token] = bad
        if "v" in where:
            v2[token, :, D // 2 + 1] = bad
        out = memopt_C.prompt_attention(q, k2, v2, cu_of([n]), window, num_sink_tokens=sinks)
        see = (token <= i) & ((i - token < window) | (token < sinks)) if window > 0 else token <= i
        check_prompt(out, q, k, v, [n], window, sinks, rows=~see)
        hit = out[see.to(dev())].float().cpu()
        if "k" in where:
            assert bool(hit.isnan().all())
        else:
            col = hit[..., D // 2 + 1]
            assert bool((col.isnan() if bad != bad else col == bad).all()), (token, bad)
            rest = torch.cat([hit[..., :D // 2 + 1], hit[..., D // 2 + 2:]], -1)
            assert bool(rest.isfinite().all())


def test_queries_that_are_not_finite_stay_in_their_rows():
    n = 140
    q, k, v = make(n, 2, 1, 64, torch.float16, 8)
    q2 = q.clone()
    q2[70] = float("nan")
    out = memopt_C.prompt_attention(q2, k, v, cu_of([n]))
    assert bool(out[70].isnan().all())
    check_prompt(out, q, k, v, [n], -1, 0, rows=torch.arange(n) != 70)


def test_side_stream_and_two_at_once():
    lens = [700, 300]
    a, b = make(1000, 4, 2, 64, torch.float16, 1), make(1000, 4, 2, 64, torch.float16, 2)
    cu = cu_of(lens)
    want = [memopt_C.prompt_attention(*x, cu) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append([memopt_C.prompt_attention(*x, cu) for _ in range(5)])
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


def test_captured_calls_follow_the_lengths_on_the_device():
    q, k, v = make(256, 4, 2, 64, torch.float16, 6)
    cu = cu_of([200, 56])
    out = torch.zeros_like(q)
    memopt_C.prompt_attention(q, k, v, cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        memopt_C.prompt_attention(q, k, v, cu, out=out)
    for lens in ([200, 56], [1, 255], [0, 256], [130, 100]):
        cu.copy_(cu_of(lens))
        q.normal_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(q)
        memopt_C.prompt_attention(q, k, v, cu, out=eager)
        assert torch.equal(out, eager)
        check_prompt(out, q, k, v, lens, -1, 0)


def test_refusals():
    q, k, v = make(20, 4, 2, 64, torch.float16, 0)
    cu = cu_of([20])

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            memopt_C.prompt_attention(*args, **kw)

    refused("CUDA", q.cpu(), k, v, cu)
    refused("keys must be a CUDA", q, k.cpu(), v, cu)
    refused("3-D", q[0], k, v, cu)
    refused("fp16 or bf16", q.float(), k.float(), v.float(), cu)
    refused("dtype", q, k.bfloat16(), v, cu)
    refused("kv heads", q, k[:19], v, cu)
    refused("kv heads", q, k, v[:, :1], cu)
    refused("multiple of num_kv_heads", q[:, :3], k, v, cu)
    refused("int32", q, k, v, cu.long())
    refused("1-D", q, k, v, cu[None])
    refused("head_dim must be", q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), cu)
    refused("out must be", q, k, v, cu, out=torch.empty_like(q).bfloat16())
    refused("out must have", q, k, v, cu, out=torch.empty((20, 4, 65), dtype=q.dtype, device=dev())[..., 1:])
    refused("overlap", q, k, v, cu, out=torch.empty((20, 1, 64), dtype=q.dtype, device=dev()).expand(20, 4, 64))
    refused("out must be a CUDA", q, k, v, cu, out=q.cpu())
    refused("gradients", q.requires_grad_(), k, v, cu)
    with torch.no_grad():
        memopt_C.prompt_attention(q, k, v, cu)
