"""What the paged 4-bit cache and the block tables refuse, and what they launch, followed without a GPU (the library's own
objects on a HIP runtime in host memory that notes kernels instead of running them)."""
import ctypes as C

import numpy as np
import pytest

from test_host_runtime import host  # noqa: F401  (the fixture)

EINVAL, EUNSUPPORTED = 1, 4


def p(a):
    return C.c_void_p(a.ctypes.data)


def i32(*v):
    return np.array(v, np.int32)


def new_cache(host, blocks=8, bs=16, heads=2, hd=64):
    return host.new("pg_paged_kv4_create", host.ctx, blocks, bs, heads, hd)


def status(host, name, *args):
    return getattr(host.lib, name)(*args)


@pytest.mark.parametrize("args", [(0, 16, 2, 64), (8, 15, 2, 64), (8, 8, 2, 64), (8, 512, 2, 64), (8, 48, 2, 64), (8, 16, 0, 64), (8, 16, 65536, 64),
                                  (8, 16, 2, 0), (8, 16, 2, 257), (1 << 27, 16, 1, 64), (1 << 32, 16, 1, 64)])
def test_create_refuses(host, args):
    h = C.c_void_p(1)
    assert status(host, "pg_paged_kv4_create", host.ctx, *args, C.byref(h)) == EINVAL
    assert not h.value


def test_create_reports_memory_and_capture(host):
    before = host.lib.pghost_used()
    host.lib.pghost_limit(before + (1 << 20))
    h = C.c_void_p()
    assert status(host, "pg_paged_kv4_create", host.ctx, 1000, 64, 8, 128, C.byref(h)) == 3
    host.lib.pghost_limit(C.c_size_t(-1).value)
    assert host.lib.pghost_used() == before                              # nothing is left behind
    host.lib.pghost_begin_capture(host.stream())
    assert status(host, "pg_paged_kv4_create", host.ctx, 8, 16, 2, 64, C.byref(h)) == 2
    assert host.lib.pghost_end_capture(host.stream()) and host.lib.pghost_recorded() == 0
    c = new_cache(host, 4, 32, 3, 80)
    got = [C.c_size_t() for _ in range(5)]
    host.ok("pg_paged_kv4_info", c, *[C.byref(x) for x in got])
    assert [x.value for x in got] == [4, 32, 3, 80, 4 * 3 * (32 * (128 + 8) + 2 * 128 + 16)]
    host.lib.pg_paged_kv4_free(host.ctx, c)


def extend_args(host, **k):
    a = dict(lens=i32(3, 0), new=i32(2, 5), batch=2, bs=16, free=i32(0, 1, 2, 3), count=i32(4), blocks=4, table=np.full((2, 4), -1, np.int32), width=4,
             lens_out=i32(0, 0), count_out=i32(0), starts=i32(0, 0, 0), granted=i32(0, 0), slots=np.zeros(7, np.int32), tokens=7)
    a.update(k)
    v = [x if isinstance(x, int) else p(x) if x is not None else None for x in
         (a[n] for n in ("lens", "new", "batch", "bs", "free", "count", "blocks", "table", "width", "lens_out", "count_out", "starts", "granted", "slots", "tokens"))]
    return [host.ctx, *v], a


@pytest.mark.parametrize("wrong", [dict(bs=24), dict(bs=0), dict(width=0), dict(lens=None), dict(count=None), dict(slots=None), dict(starts=None), dict(batch=1 << 24),
                                   dict(tokens=1 << 31), dict(count=i32(5)), dict(count=i32(-1)), dict(lens=i32(-1, 0)), dict(new=i32(2, -5)), dict(tokens=6),
                                   dict(free=i32(0, 1, 2, 4)), dict(free=i32(0, 1, -1, 3)), dict(width=1 << 28)])
def test_extend_refuses(host, wrong):
    args, keep = extend_args(host, **wrong)
    host.lib.pghost_clear_launches()
    assert status(host, "pg_block_tables_extend", *args) == EINVAL, wrong
    assert host.lib.pghost_num_launches() == 0


def test_release_refuses(host):
    flags, lens, table, free, count = i32(1, 0), i32(3, 0), np.zeros((2, 4), np.int32), i32(0, 1, 2, 3), i32(2)
    good = [host.ctx, p(flags), p(lens), 2, 16, p(table), 4, p(free), p(count), 4]
    for at, v in ((1, None), (2, None), (4, 17), (5, None), (6, 0), (7, None), (8, None), (8, p(i32(5)))):
        args = list(good)
        args[at] = v
        assert status(host, "pg_block_tables_release", *args) == EINVAL


def test_append_and_read_refuse(host):
    c = new_cache(host)
    k = np.zeros((3, 2, 64), np.float32)
    out = np.zeros_like(k)
    for slots in (i32(0, 1, 128), i32(0, 1, -2), i32(5, 1, 5)):          # 8 blocks of 16; a slot named twice
        assert status(host, "pg_paged_kv4_append", host.ctx, c, p(k), p(k), 3, p(slots)) == EINVAL
    host.ok("pg_paged_kv4_append", host.ctx, c, p(k), p(k), 3, p(i32(-1, 4, -1)))  # rows left out may be many
    for slots in (i32(0, 1, 128), i32(0, -1, 2)):
        assert status(host, "pg_paged_kv4_read", host.ctx, c, p(slots), 3, p(out), p(out)) == EINVAL
    for args in ((None, p(k), 3, p(i32(0, 1, 2))), (p(k), None, 3, p(i32(0, 1, 2))), (p(k), p(k), 3, None)):
        assert status(host, "pg_paged_kv4_append", host.ctx, c, *args) == EINVAL
    assert status(host, "pg_paged_kv4_append", host.ctx, None, p(k), p(k), 3, p(i32(0, 1, 2))) == EINVAL
    host.ok("pg_paged_kv4_append", host.ctx, c, None, None, 0, None)      # nothing to do
    host.lib.pg_paged_kv4_free(host.ctx, c)


def step(host, c, **k):
    """Two requests of 20 and 5 tokens, 2 and 1 of them new, 4 query heads."""
    a = dict(q=np.zeros((3, 4, 64), np.float32), heads=4, starts=i32(0, 2, 3), lens=i32(20, 5), batch=2, tokens=3, table=np.array([[0, 1], [2, -1]], np.int32), width=2,
             scale=0.125, mask=1, window=0, sinks=0, cap=0.0, out=np.zeros((3, 4, 64), np.float32), top=2, first=1, recent=1,
             selected=np.array([[[0, 1]] * 2] * 2 + [[[0, -1]] * 2], np.int32))
    a.update(k)
    return {n: p(v) if isinstance(v, np.ndarray) else v for n, v in a.items()}, a


BAD_STEPS = [dict(heads=3), dict(heads=0), dict(batch=65536), dict(width=0), dict(q=None), dict(starts=None), dict(lens=None), dict(table=None),
             dict(starts=i32(1, 2, 3)), dict(starts=i32(0, 2, 4)), dict(starts=i32(0, 3, 2)), dict(starts=i32(0, -1, 3)), dict(lens=i32(33, 5)), dict(lens=i32(-1, 5)),
             dict(lens=i32(1, 5)), dict(table=np.array([[0, 8], [2, -1]], np.int32)), dict(table=np.array([[0, -1], [2, -1]], np.int32)),
             dict(table=np.array([[0, 1], [-7, -1]], np.int32))]


@pytest.mark.parametrize("wrong", BAD_STEPS + [dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("nan")), dict(mask=3), dict(mask=-1),
                                               dict(out=None)])
def test_attention_refuses(host, wrong):
    c = new_cache(host)
    a, keep = step(host, c, **wrong)
    host.lib.pghost_clear_launches()
    assert status(host, "pg_paged_kv4_attention", host.ctx, c, a["q"], a["heads"], a["starts"], a["lens"], a["batch"], a["tokens"], a["table"], a["width"], a["scale"], a["mask"],
                  a["window"], a["sinks"], a["cap"], a["out"]) == EINVAL, wrong
    assert host.lib.pghost_num_launches() == 0
    host.lib.pg_paged_kv4_free(host.ctx, c)


@pytest.mark.parametrize("wrong", [w for w in BAD_STEPS if not {"q", "heads"} & set(w) and not (w.get("starts") is not None and w["starts"].max() > 3)])
def test_summarise_refuses(host, wrong):
    c = new_cache(host)
    a, keep = step(host, c, **wrong)
    assert status(host, "pg_paged_kv4_summarise", host.ctx, c, a["starts"], a["lens"], a["batch"], a["table"], a["width"]) == EINVAL, wrong
    host.lib.pg_paged_kv4_free(host.ctx, c)


@pytest.mark.parametrize("wrong", BAD_STEPS + [dict(top=0), dict(top=1), dict(recent=0), dict(first=2), dict(first=1 << 63, recent=1), dict(selected=None)])
def test_select_refuses(host, wrong):
    c = new_cache(host)
    a, keep = step(host, c, **wrong)
    assert status(host, "pg_paged_kv4_select", host.ctx, c, a["q"], a["heads"], a["starts"], a["lens"], a["batch"], a["tokens"], a["table"], a["width"], a["top"], a["first"],
                  a["recent"], a["selected"]) == EINVAL, wrong
    host.lib.pg_paged_kv4_free(host.ctx, c)


@pytest.mark.parametrize("wrong", BAD_STEPS + [dict(selected=np.array([[[0, 0]] * 2] * 3, np.int32)), dict(selected=np.array([[[1, 0]] * 2] * 3, np.int32)),
                                               dict(selected=np.array([[[0, 2]] * 2] * 3, np.int32)), dict(selected=np.array([[[0, 1]] * 2] * 3, np.int32)),
                                               dict(selected=np.array([[[-2, 0]] * 2] * 3, np.int32)), dict(selected=np.array([[[-1, 0]] * 2] * 3, np.int32)[..., ::-1] - 1),
                                               dict(top=0), dict(selected=None), dict(scale=float("nan")), dict(cap=-1.0)])
def test_attention_selected_refuses(host, wrong):
    c = new_cache(host)
    a, keep = step(host, c, **wrong)
    assert status(host, "pg_paged_kv4_attention_selected", host.ctx, c, a["q"], a["heads"], a["starts"], a["lens"], a["batch"], a["tokens"], a["table"], a["width"],
                  a["selected"], a["top"], a["scale"], a["cap"], a["out"]) == EINVAL, wrong
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_device_forms_refuse_small_scratch_and_large_launches(host):
    c = new_cache(host, 4096, 64, 2, 128)
    buf = host.alloc(1 << 16)
    n = C.c_size_t()
    host.ok("pg_paged_kv4_attention_scratch", host.ctx, c, 8, 1, 1, 4096, C.byref(n))
    assert n.value > 0                                                    # one long request: its keys are divided
    args = lambda scratch, size: (host.ctx, c, buf, 1024, 128, 8, buf, buf, 1, 1, 1, buf, 4096, 0.1, 1, 0, 0, 0.0, scratch, size, buf)  # noqa: E731
    assert status(host, "pg_paged_kv4_attention_dev", *args(None, n.value)) == EINVAL
    assert status(host, "pg_paged_kv4_attention_dev", *args(buf, n.value - 1)) == EINVAL
    assert status(host, "pg_paged_kv4_attention_dev", *args(C.c_void_p(buf.value + 4), n.value)) == EINVAL
    host.ok("pg_paged_kv4_attention_dev", *args(buf, n.value))
    sel = lambda width: (host.ctx, c, buf, 1024, 128, 8, buf, buf, 1, 1, buf, width, 8, 1, 1, buf)  # noqa: E731
    host.ok("pg_paged_kv4_select_dev", *sel(36864))
    assert status(host, "pg_paged_kv4_select_dev", *sel(36865)) == EUNSUPPORTED
    assert status(host, "pg_paged_kv4_select_dev", host.ctx, c, buf, 1024, 128, 8, buf, buf, 1, 1 << 22, buf, 4096, 8, 1, 1, buf) == EUNSUPPORTED
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_scratch_does_not_depend_on_the_rows_there_are(host):
    """max_query is a bound: a step of fewer rows in all takes the scratch that was reported for the bound."""
    c = new_cache(host, 4096, 64, 2, 128)
    buf = host.alloc(1 << 16)
    for batch, most in ((100, 12), (100, 3), (1, 64), (30, 200)):
        n = C.c_size_t()
        host.ok("pg_paged_kv4_attention_scratch", host.ctx, c, 8, batch, most, 64, C.byref(n))
        for tokens in (1, 4, 8, 64):
            host.ok("pg_paged_kv4_attention_dev", host.ctx, c, buf, 1024, 128, 8, buf, buf, batch, tokens, most, buf, 64, 0.1, 1, 0, 0, 0.0, buf, n.value, buf)
    assert status(host, "pg_paged_kv4_attention_dev", host.ctx, c, buf, 1024, 128, 8, buf, buf, 1, 1, 1 << 31, buf, 64, 0.1, 1, 0, 0, 0.0, buf, 1 << 40, buf) == EINVAL
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_summaries_refuse_more_blocks_than_a_launch_takes(host):
    c = new_cache(host, 64, 16, 2, 64)
    buf = host.alloc(1 << 16)
    for tokens, want in (((1 << 28) - 64, 0), (1 << 28, EUNSUPPORTED), ((1 << 31) - 1, EUNSUPPORTED)):
        assert status(host, "pg_paged_kv4_summarise_dev", host.ctx, c, buf, buf, 1, tokens, buf, 64) == want, tokens
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_a_cache_stays_on_its_device(host):
    """One device here: the context's number (its first word) is changed for the calls."""
    c = new_cache(host, 64, 16, 2, 64)
    buf = host.alloc(1 << 16)
    calls = [("pg_paged_kv4_append_dev", (host.ctx, c, buf, buf, 128, 64, 4, buf)), ("pg_paged_kv4_read_dev", (host.ctx, c, buf, 4, buf, buf)),
             ("pg_paged_kv4_summarise_dev", (host.ctx, c, buf, buf, 4, 4, buf, 64)), ("pg_paged_kv4_read_summaries_dev", (host.ctx, c, buf, 4, buf, buf)),
             ("pg_paged_kv4_attention_dev", (host.ctx, c, buf, 512, 64, 8, buf, buf, 4, 4, 1, buf, 4, 0.1, 1, 0, 0, 0.0, buf, 0, buf)),
             ("pg_paged_kv4_select_dev", (host.ctx, c, buf, 512, 64, 8, buf, buf, 4, 4, buf, 64, 8, 1, 1, buf)),
             ("pg_paged_kv4_attention_selected_dev", (host.ctx, c, buf, 512, 64, 8, buf, buf, 4, 4, buf, 64, buf, 8, 0.1, 0.0, buf, 0, buf))]
    device = C.c_int.from_address(host.ctx.value)
    assert device.value == 0
    for name, args in calls:
        host.ok(name, *args)
        device.value = 1
        try:
            assert status(host, name, *args) == EINVAL, name
        finally:
            device.value = 0
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_a_step_is_captured_as_launches_alone(host):
    """Nothing of a step's device forms allocates, waits or copies."""
    c = new_cache(host, 4096, 64, 2, 128)
    buf = host.alloc(1 << 20)
    n = C.c_size_t()
    host.ok("pg_paged_kv4_attention_scratch", host.ctx, c, 8, 4, 1, 1024, C.byref(n))
    calls = [("pg_block_tables_extend_dev", (host.ctx, buf, buf, 4, 64, buf, buf, 4096, buf, 1024, buf, buf, buf, buf, buf, 4)),
             ("pg_block_tables_extend_dev", (host.ctx, buf, buf, 4, 64, buf, buf, 4096, buf, 1024, buf, buf, buf, buf, buf, 100000)),
             ("pg_block_tables_release_dev", (host.ctx, buf, buf, 4, 64, buf, 1024, buf, buf, 4096)),
             ("pg_paged_kv4_append_dev", (host.ctx, c, buf, buf, 256, 128, 4, buf)),
             ("pg_paged_kv4_summarise_dev", (host.ctx, c, buf, buf, 4, 4, buf, 1024)),
             ("pg_paged_kv4_read_dev", (host.ctx, c, buf, 4, buf, buf)),
             ("pg_paged_kv4_read_summaries_dev", (host.ctx, c, buf, 4, buf, buf)),
             ("pg_paged_kv4_attention_dev", (host.ctx, c, buf, 1024, 128, 8, buf, buf, 4, 4, 1, buf, 1024, 0.1, 1, 0, 0, 0.0, buf, n.value, buf)),
             ("pg_paged_kv4_select_dev", (host.ctx, c, buf, 1024, 128, 8, buf, buf, 4, 4, buf, 1024, 8, 1, 1, buf)),
             ("pg_paged_kv4_attention_selected_dev", (host.ctx, c, buf, 1024, 128, 8, buf, buf, 4, 4, buf, 1024, buf, 8, 0.1, 0.0, buf, 1 << 40, buf))]
    for name, args in calls:
        st, recorded, whole = host.captured(name, *args)
        assert st == 0 and whole and recorded in (1, 2) and host.lib.pghost_copied() == 0, name
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_mirror_refuses_shapes_before_the_library():
    """The NumPy mirror's own checks; no context is made."""
    from peregrine_amd import paged

    c = paged.PagedKV4Cache.__new__(paged.PagedKV4Cache)
    c.num_kv_heads, c.head_dim, c._h = 2, 64, None
    with pytest.raises(ValueError):
        c.append(np.zeros((3, 2, 32)), np.zeros((3, 2, 32)), i32(0, 1, 2))
    with pytest.raises(ValueError):
        c.append(np.zeros((3, 2, 64)), np.zeros((2, 2, 64)), i32(0, 1, 2))
    with pytest.raises(ValueError):
        c.attention(np.zeros((3, 3, 64)), i32(0, 3), i32(5), np.zeros((1, 2), np.int32), 0.1)
    with pytest.raises(ValueError):
        c.attention(np.zeros((3, 4, 64)), i32(0, 3), i32(5), np.zeros((2, 2), np.int32), 0.1)
    with pytest.raises(ValueError):
        c.attention(np.zeros((3, 4, 64)), i32(0, 3), i32(5), np.zeros((1, 2), np.int32), 0.1, paged.AttentionMask.causal(2))
    with pytest.raises(ValueError):
        c.attention_selected(np.zeros((3, 4, 64)), i32(0, 3), i32(5), np.zeros((1, 2), np.int32), np.zeros((3, 4, 2), np.int32), 0.1)
