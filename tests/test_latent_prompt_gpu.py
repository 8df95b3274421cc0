"""latent_prompt_attention against its 64-bit form: widths, lengths, masks, strides, odd values, refusals; and against the
absorbed form over a cache of the same latents."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev, memopt_C
from packed_reference import attend, check, starts, tolerance

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
WIDTHS = [(128, 64), (128, 32), (64, 64), (64, 32)]


def make(T, H, D, P, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    shapes = ((T, H, D + P), (T, H, D), (T, P), (T, H, D))
    return [torch.randn(s, generator=g).to(dtype).to(dev()) for s in shapes]


def cu_of(lens, first=0):
    return torch.from_numpy(starts(lens, first)).to(dev())


def check_expanded(out, q, k, r, v, lens, window=-1, sinks=0, first=0, rows=None, scale=None):
    """All rows (of long prompts the first, the last and some between), or those of a truth tensor ``rows``."""
    H, D = k.shape[1:]
    W = q.shape[2]
    scale = W ** -0.5 if scale is None else scale
    a = first
    for n in lens:
        some = np.arange(n) if n <= 320 else np.unique(np.concatenate(
            [np.arange(10), n - 1 - np.arange(10), np.random.default_rng(n).integers(0, n, 30)]))
        keep = torch.ones(len(some), dtype=torch.bool) if rows is None else rows[a - first:a - first + n][some]
        kk = torch.cat([k[a:a + n].double(), r[a:a + n].double()[:, None].expand(-1, H, -1)], -1)
        o, w, e = attend(q[a:a + n][some].double() * (scale * W ** 0.5), kk, torch.nn.functional.pad(v[a:a + n].double(), (0, W - D)),
                         some, window, sinks)
        o, w, e = o[..., :D], w[..., :D], e[..., :D]
        tol = tolerance(o, w, e, n, W, out.dtype, out.dtype, False)
        check(out[a:a + n].cpu()[some][keep], o[keep], tol[keep], f"rows {a}..{a + n - 1}")
        a += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,P", WIDTHS)
@pytest.mark.parametrize("lens", [[1], [63, 64, 65], [127, 1, 0, 128, 2], [129, 300], [257]], ids=str)
def test_lengths(dtype, D, P, lens):
    x = make(sum(lens), 3, D, P, dtype, len(lens) + D)
    check_expanded(memopt_C.latent_prompt_attention(*x, cu_of(lens)), *x, lens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,P", WIDTHS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (63, 4), (64, 64), (65, 70), (200, 5), (1000, 3), (5, 1000),
                                          (-1, 4), (0, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_windows_and_sinks(dtype, D, P, window, sinks):
    lens = [300, 70, 129]
    x = make(sum(lens), 2, D, P, dtype, 3)
    out = memopt_C.latent_prompt_attention(*x, cu_of(lens), window, num_sink_tokens=sinks)
    check_expanded(out, *x, lens, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,P,H", [(128, 64, 16), (64, 32, 5)])
def test_long_prompts_and_many(dtype, D, P, H):
    for lens in ([2100], [40] * 70 + [900], [3] * 300):
        x = make(sum(lens), H, D, P, dtype, 5)
        check_expanded(memopt_C.latent_prompt_attention(*x, cu_of(lens)), *x, lens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0])
def test_scales(dtype, scale):
    x = make(200, 2, 64, 64, dtype, 1)
    out = memopt_C.latent_prompt_attention(*x, cu_of([200]), scale=scale)
    check_expanded(out, *x, [200], scale=scale)


def test_rising_scores():
    q, k, r, v = make(700, 2, 128, 64, torch.bfloat16, 1)
    r.copy_(torch.linspace(-3, 3, 700, device=dev())[:, None].expand(-1, 64))
    q[:, :, 128:] = 3
    check_expanded(memopt_C.latent_prompt_attention(q, k, r, v, cu_of([700])), q, k, r, v, [700])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Views of the up-projection, of a projection with the rotary keys behind the latents, head by head, off the
    alignment, and tokens 2^23 elements apart."""
    T, H, D, P = 150, 4, 128, 64
    q, k, r, v = make(T, H, D, P, dtype, 4)
    cu = cu_of([100, 50])
    want = memopt_C.latent_prompt_attention(q, k, r, v, cu)
    kv = torch.cat([k, v], -1)
    down = torch.cat([torch.zeros(T, 512, dtype=dtype, device=dev()), r], -1)
    assert torch.equal(memopt_C.latent_prompt_attention(q, kv[:, :, :D], down[:, 512:], kv[:, :, D:], cu), want)
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(memopt_C.latent_prompt_attention(turned[0], turned[1], r, turned[2], cu), want)
    odd = [torch.zeros(x.numel() + 3, dtype=dtype, device=dev())[3:].view(x.shape).copy_(x) for x in (q, k, r, v)]
    assert torch.equal(memopt_C.latent_prompt_attention(*odd, cu), want)
    far = torch.zeros(T * 2 ** 23, dtype=dtype, device=dev()).view(T, -1)
    far[:, :P] = r
    assert torch.equal(memopt_C.latent_prompt_attention(q, k, far[:, :P], v, cu), want)
    out = torch.full((T, H, 2, D), 7.0, dtype=dtype, device=dev())
    assert torch.equal(memopt_C.latent_prompt_attention(q, k, r, v, cu, out=out[:, :, 1]), want)
    assert bool((out[:, :, 0] == 7).all())


def test_rows_of_no_sequence_and_clamped_starts():
    x = make(60, 2, 64, 32, torch.float16, 4)
    out = torch.full((60, 2, 64), 7.0, dtype=torch.float16, device=dev())
    memopt_C.latent_prompt_attention(*x, cu_of([20, 15], 5), out=out)
    check_expanded(out, *x, [20, 15], first=5)
    assert bool((out[:5] == 7).all()) and bool((out[40:] == 7).all())
    cu = torch.tensor([-5, 30, 1000], dtype=torch.int32, device=dev())
    check_expanded(memopt_C.latent_prompt_attention(*x, cu), *x, [30, 30])
    assert memopt_C.latent_prompt_attention(*x, cu_of([])).shape == (60, 2, 64)
    assert memopt_C.latent_prompt_attention(*(t[:0] for t in x), cu_of([0])).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,P", [(128, 64), (64, 32)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (40, 3)])
def test_odd_values_reach_only_the_rows_that_see_them(dtype, D, P, window, sinks):
    n = 200
    q, k, r, v = make(n, 2, D, P, dtype, 8)
    i = torch.arange(n)
    for token, bad, where in [(150, float("nan"), "v"), (150, float("inf"), "v"), (64, float("-inf"), "v"),
                              (31, float("nan"), "k"), (127, float("nan"), "r"), (0, float("nan"), "v"), (128, float("nan"), "r")]:
        k2, r2, v2 = k.clone(), r.clone(), v.clone()
        if where == "k":
            k2[token] = bad
        if where == "r":
            r2[token, 3] = bad
        if where == "v":
            v2[token, :, D // 2 + 1] = bad
        out = memopt_C.latent_prompt_attention(q, k2, r2, v2, cu_of([n]), window, num_sink_tokens=sinks)
        see = (token <= i) & ((i - token < window) | (token < sinks)) if window > 0 else token <= i
        check_expanded(out, q, k, r, v, [n], window, sinks, rows=~see)
        hit = out[see.to(dev())].float().cpu()
        if where != "v":
            assert bool(hit.isnan().all())
        else:
            col = hit[..., D // 2 + 1]
            assert bool((col.isnan() if bad != bad else col == bad).all()), (token, bad)
            assert bool(torch.cat([hit[..., :D // 2 + 1], hit[..., D // 2 + 2:]], -1).isfinite().all())
    q2 = q.clone()
    q2[70, 1, D + 2] = float("nan")
    out = memopt_C.latent_prompt_attention(q2, k, r, v, cu_of([n]))
    assert bool(out[70, 1].isnan().all()) and bool(out[70, 0].isfinite().all())
    check_expanded(out, q, k, r, v, [n], rows=i != 70)


def test_captured_calls_and_other_streams():
    x = make(256, 4, 64, 64, torch.bfloat16, 6)
    cu = cu_of([200, 56])
    out = torch.zeros(256, 4, 64, dtype=torch.bfloat16, device=dev())
    memopt_C.latent_prompt_attention(*x, cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        memopt_C.latent_prompt_attention(*x, cu, out=out)
    for lens in ([200, 56], [1, 255], [0, 256], [130, 100]):
        cu.copy_(cu_of(lens))
        x[0].normal_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(out)
        memopt_C.latent_prompt_attention(*x, cu, out=eager)
        assert torch.equal(out, eager)
        check_expanded(out, *x, lens)
    y = make(256, 4, 64, 64, torch.bfloat16, 7)
    want = [memopt_C.latent_prompt_attention(*t, cu) for t in (x, y)]
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s, t in zip(streams, (x, y)):
        with torch.cuda.stream(s):
            got.append([memopt_C.latent_prompt_attention(*t, cu) for _ in range(5)])
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o[:230], w[:230]) for o in outs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_both_forms_of_one_layer_agree(dtype):
    """A small latent layer: prompts in the expanded form, and the same rows in the absorbed form over the cache that
    write_latent filled. What differs are the roundings to 16 bits on either way: keys, values and queries on theirs."""
    g = torch.Generator().manual_seed(3)
    H, D, R, P, lens = 4, 128, 256, 64, [90, 37]
    T = sum(lens)
    c, kr = (torch.randn(T, n, generator=g).to(dtype).to(dev()) for n in (R, P))
    wk, wv = (torch.randn(H, D, R, generator=g).to(dev()) / R ** 0.5 for _ in range(2))
    q = torch.randn(T, H, D + P, generator=g).to(dtype).to(dev())
    k, v = (torch.matmul(c.float()[None], w.transpose(1, 2).contiguous()).transpose(0, 1).to(dtype) for w in (wk, wv))
    cu = cu_of(lens)
    a = memopt_C.latent_prompt_attention(q, k, kr, v, cu).float()
    cache = torch.zeros(20, 16, R + P, dtype=dtype, device=dev())
    tables = torch.tensor([[3, 1, 4, 15, 9, 2], [6, 5, 8, -1, -1, -1]], dtype=torch.int32, device=dev())
    slots = torch.cat([tables[b, torch.arange(n, device=dev()) // 16] * 16 + torch.arange(n, device=dev()) % 16
                       for b, n in enumerate(lens)]).to(torch.int32)
    memopt_C.write_latent(c, kr, slots, cache)
    qa = torch.matmul(q[:, :, :D].float().transpose(0, 1).contiguous(), wk).transpose(0, 1).to(dtype)
    o = memopt_C.latent_attention(torch.cat([qa, q[:, :, D:]], -1), cache, tables,
                                  torch.tensor(lens, dtype=torch.int32, device=dev()), cu, max(lens), 96, (D + P) ** -0.5, R)
    b = torch.matmul(o.float().transpose(0, 1).contiguous(), wv.transpose(1, 2).contiguous()).transpose(0, 1)
    u = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -8
    # scores differ by roundings of keys and queries, 2 u of some 10 at most, and so weights; outputs by a few more
    assert float((a - b).norm() / a.norm()) < 30 * u


def test_refusals():
    q, k, r, v = make(20, 4, 64, 32, torch.float16, 0)
    cu = cu_of([20])

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            memopt_C.latent_prompt_attention(*args, **kw)

    refused("CUDA", q.cpu(), k, r, v, cu)
    refused("rope_keys must be a CUDA", q, k, r.cpu(), v, cu)
    refused("3-D", q[0], k, r, v, cu)
    refused("2-D", q, k, r[:, None], v, cu)
    refused("fp16 or bf16", q.float(), k.float(), r.float(), v.float(), cu)
    refused("dtype", q, k, r.bfloat16(), v, cu)
    refused("keys and values must be", q, k[:19], r, v, cu)
    refused("keys and values must be", q, k[:, :2], r, v, cu)
    refused("keys and values must be", q, k, r[:, :16], v, cu)
    refused("keys and values must be", q, k, r, v[..., :32], cu)
    refused("head_dim must be", q[..., :48], k[..., :32], r[:, :16], v[..., :32], cu)
    refused("rope_dim 32 or 64", q[..., :80], k, r[:, :16], v, cu)
    refused("int32", q, k, r, v, cu.long())
    refused("1-D", q, k, r, v, cu[None])
    refused("out must be", q, k, r, v, cu, out=torch.empty_like(q))
    refused("out must be", q, k, r, v, cu, out=torch.empty_like(k).bfloat16())
    refused("overlap", q, k, r, v, cu, out=torch.empty((20, 1, 64), dtype=q.dtype, device=dev()).expand(20, 4, 64))
    refused("gradients", q, k, r.clone().requires_grad_(), v, cu)
    with torch.no_grad():
        memopt_C.latent_prompt_attention(q, k, r.clone().requires_grad_(), v, cu)


@pytest.mark.parametrize("power", [126, 100, -96])
@pytest.mark.parametrize("lens", [[300, 70], [1500]], ids=str)
def test_values_of_bfloat16s_range(power, lens):
    """Values up to nearly the type's largest, all alike or of both signs, and small ones: their means are in its range,
    and scaling by a power of two, exact, changes nothing else."""
    q, k, r, v = make(sum(lens), 2, 128, 64, torch.bfloat16, 9)
    for values in (torch.full_like(v, 3.5), v.clamp(-3.5, 3.5)):
        out = memopt_C.latent_prompt_attention(q, k, r, values * 2.0 ** power, cu_of(lens))
        assert bool(out.isfinite().all())
        check_expanded((out.double() * 2.0 ** -power).bfloat16(), q, k, r, values, lens)
