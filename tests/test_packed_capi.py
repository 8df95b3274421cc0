"""CPU tests of the packed operators' C entries: what they refuse before anything is launched, and the workspace they
ask for. Pointers here are never dereferenced."""
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


def prompt(C, **kw):
    d = C.PromptDesc(P, P, P, P, 0, 32, 2, 4, 2, 64, 256, 64, 128, 64, 128, 64, 256, 64, P, -1, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return C._c_prompt(ctypes.byref(d), None)


@pytest.mark.parametrize("text,code,change", [
    ("dtype", INVALID, dict(dtype=2)), ("negative", INVALID, dict(tokens=-1)), ("negative", INVALID, dict(batch=-1)),
    ("multiple of num_kv_heads", INVALID, dict(num_heads=5)), ("multiple of num_kv_heads", INVALID, dict(num_heads=0)),
    ("multiple of num_kv_heads", INVALID, dict(num_kv_heads=0)),
    ("head_dim", UNSUPPORTED, dict(head_dim=96)), ("null", INVALID, dict(query=None)), ("null", INVALID, dict(key=None)),
    ("null", INVALID, dict(value=None)), ("null", INVALID, dict(out=None)), ("null", INVALID, dict(query_starts=None)),
    ("aligned", INVALID, dict(query=P + 8)), ("aligned", INVALID, dict(k_token_stride=132)),
    ("aligned", INVALID, dict(v_head_stride=4)), ("aligned", INVALID, dict(o_token_stride=258)),
    ("strides", UNSUPPORTED, dict(k_token_stride=32)), ("strides", UNSUPPORTED, dict(v_token_stride=1 << 23)),
    ("too many", UNSUPPORTED, dict(tokens=2 ** 29)),
])
def test_prompt_refusals(C, text, code, change):
    refused(C, prompt(C, **change), code, text)


def test_prompt_launches_of_too_many_threads(C):
    """Tiles are counted as if every sequence but the empty ones left one part full: 2^24 tiles of 256 threads are more
    than a launch holds."""
    refused(C, prompt(C, tokens=2 ** 20, batch=2 ** 20, num_heads=32, num_kv_heads=32), UNSUPPORTED, "too many")
    refused(C, prompt(C, tokens=2 ** 19, batch=2 ** 20, num_heads=32, num_kv_heads=32), UNSUPPORTED, "too many")


def test_prompt_null_and_empty(C):
    refused(C, C._c_prompt(None, None), INVALID, "null")
    assert prompt(C, tokens=0) == OK and prompt(C, batch=0, query_starts=None) == OK


def test_prompt_bytes_are_the_descriptor(C):
    """The bytes that memopt_C packs are those of the ctypes mirror."""
    args = (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, -1, 21)
    assert C._PROMPT.pack(*args) == bytes(C.PromptDesc(*args))
    assert [C._count32(n) for n in (-2 ** 40, -1, 0, 7, 2 ** 40)] == [-1, -1, 0, 7, 2 ** 31 - 1]


def packed(C, call=True, **kw):
    d = C.PackedDesc(P, P, 8, 8, 8, 2, 64, 512, 64, 512, 64, 1, P, None, 16, 100, P, 20, P, P, 1, 320, -1, 0, P, 1 << 40)
    for k, v in kw.items():
        setattr(d, k, v)
    need, zeroed = ctypes.c_int64(-1), ctypes.c_int64(-1)
    rc = C._c_packed_ws(ctypes.byref(d), ctypes.byref(need), ctypes.byref(zeroed))
    return (C._c_packed(ctypes.byref(d), None) if call else rc), need.value, zeroed.value


@pytest.mark.parametrize("text,code,change", [
    ("negative", INVALID, dict(tokens=-1)), ("negative", INVALID, dict(batch=-2)),
    ("negative", INVALID, dict(max_query_len=-1)), ("multiple of num_kv_heads", INVALID, dict(num_heads=7)),
    ("fp16 pool or INT4", UNSUPPORTED, dict(kv_format=2)), ("head_dim", UNSUPPORTED, dict(head_dim=80)),
    ("empty cache", INVALID, dict(num_kv_blocks=0)), ("empty cache", INVALID, dict(max_blocks_per_seq=0)),
    ("empty cache", INVALID, dict(block_size=0)), ("16 tokens", UNSUPPORTED, dict(block_size=32)),
    ("16 tokens", UNSUPPORTED, dict(kv_format=0, block_size=24)), ("aligned", INVALID, dict(query=P + 2)),
    ("aligned", INVALID, dict(o_head_stride=68)), ("aligned", INVALID, dict(workspace=P + 8)),
    ("aligned", INVALID, dict(key_cache=P + 4)), ("null", INVALID, dict(query=None)), ("null", INVALID, dict(out=None)),
    ("null", INVALID, dict(kv_format=0, value_cache=None)), ("null", INVALID, dict(block_tables=None)),
    ("null", INVALID, dict(context_lens=None)), ("null", INVALID, dict(query_starts=None)),
    ("workspace needs", INVALID, dict(workspace=None)), ("workspace needs", INVALID, dict(workspace_bytes=100)),
    ("32 bits", UNSUPPORTED, dict(max_blocks_per_seq=2 ** 27)), ("too many", UNSUPPORTED, dict(tokens=2 ** 28)),
    ("too many", UNSUPPORTED, dict(batch=4000, tokens=4000, max_blocks_per_seq=2 ** 26)),
])
def test_packed_refusals(C, text, code, change):
    refused(C, packed(C, **change)[0], code, text)


def test_packed_empty_calls_need_nothing(C):
    for change in (dict(tokens=0), dict(batch=0), dict(max_query_len=0)):
        assert packed(C, workspace=None, workspace_bytes=0, query=None, **change) == (OK, 0, 0)
    refused(C, C._c_packed(None, None), INVALID, "null")


def test_packed_workspace(C):
    """Counters of every block; two partial blocks of each workgroup; staged copies where long chunks can fill the GPU
    (256 CUs), of at most 2 GiB."""
    def size(**kw):
        rc, need, zeroed = packed(C, call=False, **kw)
        assert rc == OK and 0 < zeroed <= need and zeroed % 256 == 0
        return need, zeroed

    need, zeroed = size()
    assert zeroed == 256  # 8 sequences x 2 key heads x 4 bytes, rounded up
    partials = 256 * 2 * 2 * 8 * (64 + 2) * 4  # kMaxParts workgroups, two blocks of 8 rows each, 2 key heads
    assert need - zeroed == partials
    # 32 rows (8 tokens x 4 heads) per sequence: blocks of 32 rows; 16 rows: of 16
    assert size(max_query_len=8, tokens=64)[0] - size(max_query_len=8, tokens=64)[1] == 4 * partials
    assert size(max_query_len=4, tokens=32)[0] - size(max_query_len=4, tokens=32)[1] == 2 * partials
    # chunks of 512 rows (128 tokens), 8 query heads: staged from 128 x 256 / 8 tokens on
    chunks = dict(max_query_len=512, max_seq_len=4096, max_blocks_per_seq=256)
    small, full = size(tokens=4095, **chunks)[0], size(tokens=4096, **chunks)[0]
    token = 2 * 64 * 2 * 2  # K and V of two heads
    extra = 8 * 4096 * (token + 2 * 8) + 8 * 4096 // 16  # eight sequences: values, factors, links
    assert 0 <= full - small - extra <= 3 * 256
    # a window bounds the copies
    assert size(tokens=4096, window_size=256, **chunks)[0] < small + 8 * (256 + 512 + 256) * (token + 32)
    # contexts of 2^20 tokens: four sequences' copies fit
    long = dict(max_query_len=512, max_seq_len=1 << 20, max_blocks_per_seq=65536)
    assert 4 * 2 ** 20 * token == 2 ** 31 <= size(tokens=4096, **long)[0] < 2 ** 31 + 2 ** 27
    assert size(tokens=4096, kv_format=0, **long)[0] < size(tokens=4096, **long)[0]  # (no factors)


@pytest.mark.parametrize("text,code,at,value", [
    ("positive", INVALID, 11, 0), ("4096", UNSUPPORTED, 11, 4097), ("positive", INVALID, 12, 0),
    ("positive", INVALID, 13, 0), ("positive", INVALID, 14, 0), ("positive", INVALID, 15, -1),
    ("2^31", UNSUPPORTED, 12, 2 ** 27),
] + [("null", INVALID, i, 0) for i in range(11)])
def test_advance_refusals(C, text, code, at, value):
    args = [P] * 11 + [4, 8, 32, 16, 4]
    args[at] = value
    refused(C, C._c_advance(C._ADVANCE.pack(*args), None), code, text)
    refused(C, C._c_advance(None, None), INVALID, "null")
