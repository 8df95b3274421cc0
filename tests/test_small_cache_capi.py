"""CPU tests of the C entries of weights, compaction and latent attention: what they refuse before anything is launched,
and the workspace they ask for. Pointers here are never dereferenced."""
import ctypes

import pytest

OK, INVALID, UNSUPPORTED = 0, 1, 4
P = 256  # an aligned address


@pytest.fixture(scope="module")
def C():
    import memopt_C
    memopt_C._lib.memopt_last_error.restype = ctypes.c_char_p
    return memopt_C


def refused(C, rc, code, text):
    assert (rc, text in C._lib.memopt_last_error().decode()) == (code, True), (rc, C._lib.memopt_last_error())


SCORES = dict(query=P, scores=P, out=P, tokens=8, batch=8, num_heads=8, num_kv_heads=2, head_dim=64, q_ts=512, q_hs=64,
              kv_format=1, key_cache=P, block_size=16, num_kv_blocks=100, block_tables=P, max_blocks=20, context_lens=P,
              query_starts=P, max_query_len=1, max_seq_len=320, window=-1, sinks=0, scores_len=320, workspace=P,
              workspace_bytes=1 << 40)
COMPACT = dict(scores=P, scores_out=2 * P, kept=P, kv_format=1, key_cache=P, value_cache=0, num_kv_blocks=100, block_tables=P,
               context_lens=P, keep=P, block_tables_out=2 * P, context_lens_out=2 * P, status=P, free_pages=P, free_span=P,
               free_span_out=P, num_requests=4, num_kv_heads=2, head_dim=64, max_blocks=20, block_size=16, num_free_pages=100,
               scores_len=320, max_keep=64, sinks=4, recent=0, workspace=P, workspace_bytes=1 << 40)
LATENT = dict(query=P, cache=P, out=P, dtype=0, tokens=8, batch=8, num_heads=16, rank=512, rope_dim=64, q_ts=9216, q_hs=576,
              o_ts=8192, o_hs=512, block_size=16, num_kv_blocks=100, block_tables=P, max_blocks=20, context_lens=P,
              query_starts=P, max_query_len=1, max_seq_len=320, window=-1, sinks=0, scale=0.1, workspace=P,
              workspace_bytes=1 << 40)
EXPANDED = dict(query=P, key=P, rope_key=P, value=P, out=P, dtype=0, tokens=32, batch=2, num_heads=4, head_dim=128, rope_dim=64,
                q_ts=768, q_hs=192, k_ts=512, k_hs=128, r_ts=64, v_ts=512, v_hs=128, o_ts=512, o_hs=128, query_starts=P,
                window=-1, sinks=0, scale=0.1)


def call(C, what, base, size=False, **kw):
    assert set(kw) <= set(base), kw
    struct, ws, fn = {"scores": (C._SCORES, C._c_scores_ws, C._c_scores), "compact": (C._COMPACT, C._c_compact_ws, C._c_compact),
                      "latent": (C._LATENT, C._c_latent_ws, C._c_latent),
                      "expanded": (C._LATENT_PROMPT, None, C._c_latent_prompt)}[what]
    d = struct.pack(*{**base, **kw}.values()) + (b"\0" * 4 if what == "expanded" else b"")
    if size:
        need = ctypes.c_int64(-1)
        assert ws(d, ctypes.byref(need)) == OK
        return need.value
    return fn(d, None)


@pytest.mark.parametrize("text,code,change", [
    ("negative", INVALID, dict(tokens=-1)), ("negative", INVALID, dict(batch=-1)), ("negative", INVALID, dict(max_query_len=-1)),
    ("negative", INVALID, dict(scores_len=-1)), ("multiple of num_kv_heads", INVALID, dict(num_heads=7)),
    ("multiple of num_kv_heads", INVALID, dict(num_kv_heads=0)), ("fp16 pool or INT4", UNSUPPORTED, dict(kv_format=2)),
    ("head_dim", UNSUPPORTED, dict(head_dim=80)), ("empty cache", INVALID, dict(num_kv_blocks=0)),
    ("empty cache", INVALID, dict(max_blocks=0)), ("empty cache", INVALID, dict(block_size=0)),
    ("16 tokens", UNSUPPORTED, dict(block_size=32)), ("16 tokens", UNSUPPORTED, dict(kv_format=0, block_size=24)),
    ("2^30", UNSUPPORTED, dict(max_blocks=2 ** 27)), ("2^30", UNSUPPORTED, dict(scores_len=2 ** 30 + 1)),
    ("too many", UNSUPPORTED, dict(tokens=2 ** 28)), ("too many", UNSUPPORTED, dict(batch=65536)),
    ("too many", UNSUPPORTED, dict(max_blocks=2 ** 26, max_seq_len=2 ** 30)),
    ("too far apart", UNSUPPORTED, dict(q_ts=2 ** 25)), ("too far apart", UNSUPPORTED, dict(q_hs=2 ** 28)),
    ("too far apart", UNSUPPORTED, dict(q_ts=-512)), ("aligned", INVALID, dict(query=P + 8)), ("aligned", INVALID, dict(q_hs=68)),
    ("aligned", INVALID, dict(key_cache=P + 4)), ("aligned", INVALID, dict(workspace=P + 8)), ("null", INVALID, dict(query=0)),
    ("null", INVALID, dict(out=0)), ("null", INVALID, dict(key_cache=0)), ("null", INVALID, dict(block_tables=0)),
    ("null", INVALID, dict(context_lens=0)), ("null", INVALID, dict(query_starts=0)),
    ("workspace needs", INVALID, dict(workspace=0)), ("workspace needs", INVALID, dict(workspace_bytes=100)),
])
def test_scores_refusals(C, text, code, change):
    refused(C, call(C, "scores", SCORES, **change), code, text)


def test_scores_empty_calls_and_workspace(C):
    for change in (dict(batch=0), dict(scores_len=0)):
        assert call(C, "scores", SCORES, query=0, out=0, workspace=0, workspace_bytes=0, **change) == OK
    assert call(C, "scores", SCORES, size=True, tokens=0) == call(C, "scores", SCORES, size=True, max_query_len=0) == 0
    assert call(C, "scores", SCORES, size=True, max_seq_len=0) == 0
    refused(C, C._c_scores(None, None), INVALID, "null")
    # single tokens: 4 rows of 512 (two tiles of 256) weights, and a maximum and a sum per 64 keys, for 8 x 2 units
    assert call(C, "scores", SCORES, size=True) == 8 * 2 * 4 * (512 * 4 + 8 * 8)
    # chunks (32 rows): the same per tile of 256 keys and row, and the rows' lse
    assert call(C, "scores", SCORES, size=True, max_query_len=8) == 2 * 8 * 4 * (2 * 8) + 2 * 8 * 4 * 4
    # a batch padded to many rows, each request with one: by requests, not by rows
    assert call(C, "scores", SCORES, size=True, tokens=4096) == call(C, "scores", SCORES, size=True)


def test_scores_that_overlap_out_in_part(C):
    size = 4 * 8 * 2 * 320
    for d in (4 - size, -256, 4, size - 4):
        refused(C, call(C, "scores", SCORES, scores=2 ** 20 + d, out=2 ** 20), INVALID, "overlap")


@pytest.mark.parametrize("tokens,heads", [(2 ** 26, 8), (2 ** 25, 32), (2 ** 24 + 3, 64), (2 ** 27, 4)])
def test_scores_workspace_of_very_many_rows(C, tokens, heads):
    """Sizes that pass 32 bits on the way: a maximum and a sum per row and key tile, and the rows' lse."""
    need = call(C, "scores", SCORES, size=True, tokens=tokens, num_heads=heads, num_kv_heads=heads, batch=1, max_query_len=tokens,
                q_ts=64 * heads, max_seq_len=256)
    sums = 4 * 8 * heads * 256  # (of eight workgroups that may share a tile's rows)
    assert need == 8 * heads * tokens + (4 * heads * tokens + 255) // 256 * 256 + sums


@pytest.mark.parametrize("batch,heads,kv_heads,tokens", [(64, 128, 8, 65536), (1024, 32, 8, 8192), (4096, 32, 8, 8192),
                                                         (8, 16, 1, 2 ** 20), (4096, 16, 2, 4096)])
def test_scores_workspace_of_large_batches_of_single_tokens(C, batch, heads, kv_heads, tokens):
    """The rows' weights are kept for some sequences at a time: 1 GiB of them, and their maxima and sums, at most."""
    size = dict(tokens=batch, batch=batch, num_heads=heads, num_kv_heads=kv_heads, q_ts=64 * heads, max_blocks=tokens // 16,
                max_seq_len=tokens, scores_len=tokens)
    all_of_them = 4 * batch * heads * tokens
    need = call(C, "scores", SCORES, size=True, **size)
    assert min(all_of_them, 2 ** 30) * 0.9 < need < 2 ** 30 * (1 + 8 * 4 / (4 * 256)) + 512
    one = 4 * heads * 2 ** 28  # (a sequence past the limit by itself: its own weights)
    size.update(max_blocks=2 ** 24, max_seq_len=2 ** 28, scores_len=2 ** 28, batch=1)
    assert one <= call(C, "scores", SCORES, size=True, **size) < one * 1.04


@pytest.mark.parametrize("text,code,change", [
    ("negative", INVALID, dict(num_requests=-1)), ("negative", INVALID, dict(scores_len=-1)), ("negative", INVALID, dict(max_keep=-1)),
    ("empty cache", INVALID, dict(num_kv_heads=0)), ("empty cache", INVALID, dict(num_kv_blocks=0)),
    ("empty cache", INVALID, dict(max_blocks=0)), ("empty cache", INVALID, dict(num_free_pages=0)),
    ("4096", UNSUPPORTED, dict(num_requests=4097)), ("fp16 pool or INT4", UNSUPPORTED, dict(kv_format=2)),
    ("head_dim", UNSUPPORTED, dict(head_dim=96)), ("16 tokens", UNSUPPORTED, dict(block_size=32)),
    ("2^30", UNSUPPORTED, dict(max_blocks=2 ** 27)), ("more of them kept", UNSUPPORTED, dict(max_keep=321)),
    ("2^30", UNSUPPORTED, dict(num_kv_blocks=2 ** 31)), ("2^30", UNSUPPORTED, dict(num_requests=4096, max_blocks=2 ** 20)),
    ("too many", UNSUPPORTED, dict(num_requests=4096, max_keep=2 ** 18, scores_len=2 ** 18, max_blocks=2 ** 14)),
    ("null", INVALID, dict(scores=0)), ("null", INVALID, dict(scores_out=0)), ("null", INVALID, dict(kept=0)),
    ("null", INVALID, dict(key_cache=0)), ("null", INVALID, dict(kv_format=0)), ("null", INVALID, dict(block_tables=0)),
    ("null", INVALID, dict(context_lens=0)), ("null", INVALID, dict(keep=0)), ("null", INVALID, dict(block_tables_out=0)),
    ("null", INVALID, dict(context_lens_out=0)), ("null", INVALID, dict(status=0)), ("null", INVALID, dict(free_pages=0)),
    ("null", INVALID, dict(free_span=0)), ("null", INVALID, dict(free_span_out=0)),
    ("must not overlap", INVALID, dict(scores_out=P)), ("must not overlap", INVALID, dict(block_tables_out=P)),
    ("must not overlap", INVALID, dict(context_lens_out=P)), ("aligned", INVALID, dict(key_cache=P + 8)),
    ("aligned", INVALID, dict(workspace=P + 4)), ("workspace needs", INVALID, dict(workspace=0)),
    ("workspace needs", INVALID, dict(workspace_bytes=100)),
])
def test_compact_refusals(C, text, code, change):
    refused(C, call(C, "compact", COMPACT, **change), code, text)


def test_compact_results_that_overlap(C):
    """Results share no byte with an input, their last and first among them, nor with each other."""
    need = call(C, "compact", COMPACT, size=True)
    size = dict(scores=4 * 2 * 320 * 4, scores_out=4 * 2 * 320 * 4, kept=4 * 2 * 64 * 4, block_tables=4 * 20 * 4, context_lens=16,
                keep=16, block_tables_out=4 * 20 * 4, context_lens_out=16, status=16, free_pages=400, free_span=8, free_span_out=8,
                workspace=need)
    at = {name: (i + 1) << 20 for i, name in enumerate(size)}
    results = ("scores_out", "kept", "block_tables_out", "context_lens_out", "status", "free_span_out")
    for fmt, caches in ((1, dict(key_cache=100 * 2 * 17 * 64)), (0, dict(key_cache=100 * 16 * 2 * 64 * 2, value_cache=100 * 16 * 2 * 64 * 2))):
        place = {**COMPACT, **at, **{n: (100 + i) << 20 for i, n in enumerate(caches)}, "kv_format": fmt}
        sizes = {**size, **caches}
        for r in results:
            for x in sizes:
                if x == r or x == "workspace":
                    continue
                for where in (place[x] + sizes[x] - 4, place[x] - sizes[r] + 4):
                    refused(C, call(C, "compact", {**place, r: where}), INVALID, "must not overlap")


def test_compact_workspace(C):
    refused(C, C._c_compact(None, None), INVALID, "null")
    assert call(C, "compact", COMPACT, size=True, num_requests=0) == 0
    assert call(C, "compact", COMPACT, size=True) == (4 * (5 * 4 + 4 + 100) + 255) // 256 * 256


@pytest.mark.parametrize("text,code,change", [
    ("dtype", INVALID, dict(dtype=2)), ("negative", INVALID, dict(tokens=-1)), ("negative", INVALID, dict(batch=-1)),
    ("negative", INVALID, dict(max_query_len=-1)), ("no heads", INVALID, dict(num_heads=0)), ("no heads", INVALID, dict(num_kv_blocks=0)),
    ("no heads", INVALID, dict(max_blocks=0)), ("rank must be", UNSUPPORTED, dict(rank=384)),
    ("rope_dim", UNSUPPORTED, dict(rope_dim=16)), ("multiple of 16", UNSUPPORTED, dict(block_size=24)),
    ("2^30", UNSUPPORTED, dict(max_blocks=2 ** 27)), ("aligned", INVALID, dict(query=P + 8)), ("aligned", INVALID, dict(q_ts=9220)),
    ("aligned", INVALID, dict(o_hs=516)), ("aligned", INVALID, dict(cache=P + 2)), ("aligned", INVALID, dict(workspace=P + 8)),
    ("too many", UNSUPPORTED, dict(tokens=2 ** 27)), ("too many", UNSUPPORTED, dict(tokens=2 ** 16, num_heads=256)),
    ("null", INVALID, dict(query=0)), ("null", INVALID, dict(cache=0)), ("null", INVALID, dict(out=0)),
    ("null", INVALID, dict(block_tables=0)), ("null", INVALID, dict(context_lens=0)), ("null", INVALID, dict(query_starts=0)),
    ("workspace needs", INVALID, dict(workspace=0)), ("workspace needs", INVALID, dict(workspace_bytes=100)),
])
def test_latent_refusals(C, text, code, change):
    refused(C, call(C, "latent", LATENT, **change), code, text)


def test_latent_empty_calls_and_workspace(C):
    for change in (dict(tokens=0), dict(batch=0), dict(max_query_len=0)):
        assert call(C, "latent", LATENT, query=0, workspace=0, workspace_bytes=0, **change) == OK
        assert call(C, "latent", LATENT, size=True, **change) == 0
    refused(C, C._c_latent(None, None), INVALID, "null")
    # two parts of 32 rows for each workgroup: (8 x 16 / 32 + 8) tiles of rows x 5 of keys, 60, and of workgroups the next
    # multiple of 8 (XCDs)
    assert call(C, "latent", LATENT, size=True) == 64 * 2 * 32 * (512 + 2) * 4
    assert call(C, "latent", LATENT, size=True, max_seq_len=2 ** 20, max_blocks=65536) == 256 * 2 * 32 * (512 + 2) * 4


@pytest.mark.parametrize("text,code,change", [
    ("dtype", INVALID, dict(dtype=2)), ("negative", INVALID, dict(tokens=-1)), ("no heads", INVALID, dict(num_heads=0)),
    ("head_dim", UNSUPPORTED, dict(head_dim=96)), ("rope_dim", UNSUPPORTED, dict(rope_dim=128)), ("null", INVALID, dict(query=0)),
    ("null", INVALID, dict(key=0)), ("null", INVALID, dict(rope_key=0)), ("null", INVALID, dict(value=0)), ("null", INVALID, dict(out=0)),
    ("null", INVALID, dict(query_starts=0)), ("aligned", INVALID, dict(query=P + 8)), ("aligned", INVALID, dict(r_ts=68)),
    ("aligned", INVALID, dict(v_hs=4)), ("strides", UNSUPPORTED, dict(k_ts=64)), ("strides", UNSUPPORTED, dict(r_ts=32)),
    ("strides", UNSUPPORTED, dict(v_ts=1 << 23)), ("too many", UNSUPPORTED, dict(tokens=2 ** 29)),
    ("too many", UNSUPPORTED, dict(tokens=2 ** 20, batch=2 ** 20, num_heads=32)),
])
def test_latent_prompt_refusals(C, text, code, change):
    refused(C, call(C, "expanded", EXPANDED, **change), code, text)


def test_latent_prompt_empty_calls(C):
    refused(C, C._c_latent_prompt(None, None), INVALID, "null")
    assert call(C, "expanded", EXPANDED, tokens=0, query=0) == OK and call(C, "expanded", EXPANDED, batch=0, query_starts=0) == OK


def test_write_latent_refusals(C):
    def write(l=P, ls=512, r=P, rs=64, T=4, R=512, Q=64, slots=P, cache=P, n=100):
        return C._c_write_latent(l, ls, r, rs, T, R, Q, slots, cache, n, None)

    refused(C, write(T=-1), INVALID, "negative")
    refused(C, write(n=-1), INVALID, "negative")
    for kw in (dict(R=0), dict(R=12), dict(Q=-8), dict(Q=4), dict(R=1 << 20)):
        refused(C, write(**kw), UNSUPPORTED, "multiples of 8")
    for kw in (dict(l=None), dict(r=None), dict(slots=None), dict(cache=None)):
        refused(C, write(**kw), INVALID, "null")
    for kw in (dict(l=P + 8), dict(r=P + 2), dict(cache=P + 4), dict(ls=516), dict(rs=4)):
        refused(C, write(**kw), INVALID, "aligned")
    refused(C, write(T=2 ** 30), UNSUPPORTED, "too many")
    assert write(T=0, l=None) == OK
