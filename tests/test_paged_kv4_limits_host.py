"""Refusals of the block tables and the paged 4-bit cache at the ends of what they take, without a GPU (the library's own objects on a
HIP runtime in host memory that notes kernels instead of running them)."""
import ctypes as C

import numpy as np
import pytest

from test_host_runtime import host  # noqa: F401  (the fixture)
from test_paged_kv4_host import EINVAL, extend_args, i32, new_cache, p, status, step


def table(*rows):
    return np.array(rows, np.int32)


def taken(host, name, args):
    """The call comes as far as its kernel, which writes nothing here."""
    host.lib.pghost_clear_launches()
    assert status(host, name, *args) != EINVAL and host.lib.pghost_num_launches() > 0


# Two requests of 20 and 0 tokens in blocks of 16, four blocks in all, tables of four.
GOOD = dict(lens=i32(20, 0), table=table([2, 3, -1, -1], [-1] * 4), count=i32(2))


@pytest.mark.parametrize("wrong", [dict(lens=i32(65, 0)), dict(lens=i32(20, 65)), dict(lens=i32(2 ** 31 - 1, 0)), dict(table=table([2, 4, -1, -1], [-1] * 4)),
                                   dict(table=table([-1, 3, -1, -1], [-1] * 4)), dict(table=table([2, 1 << 28, -1, -1], [-1] * 4)), dict(lens=i32(33, 0)), dict(lens=i32(20, 1))])
def test_extend_refuses_lengths_behind_the_table_and_entries_that_are_no_block(host, wrong):
    args, keep = extend_args(host, **GOOD)
    taken(host, "pg_block_tables_extend", args)
    args, keep = extend_args(host, **{**GOOD, **wrong})
    host.lib.pghost_clear_launches()
    assert status(host, "pg_block_tables_extend", *args) == EINVAL, wrong
    assert host.lib.pghost_num_launches() == 0


def release_args(host, **k):
    a = dict(flags=i32(1, 0), lens=i32(20, 70), table=table([2, 3, -1, -1], [9, 9, 9, 9]), free=i32(0, 1, 2, 3), count=i32(2))
    a.update(k)
    return [host.ctx, p(a["flags"]), p(a["lens"]), 2, 16, p(a["table"]), 4, p(a["free"]), p(a["count"]), 4], a


@pytest.mark.parametrize("wrong", [dict(lens=i32(65, 0)), dict(lens=i32(-1, 0)), dict(table=table([2, 4, -1, -1], [9] * 4)), dict(table=table([2, -1, -1, -1], [9] * 4)),
                                   dict(count=i32(3)), dict(flags=i32(1, 1)), dict(flags=i32(1, 1), lens=i32(20, 16), table=table([2, 3, -1, -1], [2, -1, -1, -1]))])
def test_release_refuses_what_is_no_request_and_more_blocks_than_there_are(host, wrong):
    args, keep = release_args(host)                                       # (the request that stays is not looked at)
    taken(host, "pg_block_tables_release", args)
    args, keep = release_args(host, **wrong)
    host.lib.pghost_clear_launches()
    assert status(host, "pg_block_tables_release", *args) == EINVAL, wrong
    assert host.lib.pghost_num_launches() == 0


WRAPS = [(1 << 60) + 1, (1 << 60) + 8, 1 << 60, 1 << 63, 1 << 27]        # times 16 tokens a block: past 64 bits, or past 31


@pytest.mark.parametrize("many", WRAPS)
def test_tables_and_choices_whose_tokens_wrap_are_refused(host, many):
    c, buf, n = new_cache(host), host.alloc(1 << 12), C.c_size_t()
    dense = lambda width: (host.ctx, c, buf, 256, 64, 4, buf, buf, 2, 3, 2, buf, width, 0.125, 1, 0, 0, 0.0, buf, 1 << 14, buf)  # noqa: E731
    chosen = lambda width, top: (host.ctx, c, buf, 256, 64, 4, buf, buf, 2, 3, buf, width, buf, top, 0.125, 0.0, buf, 1 << 14, buf)  # noqa: E731
    select = lambda width: (host.ctx, c, buf, 256, 64, 4, buf, buf, 2, 3, buf, width, 2, 1, 1, buf)  # noqa: E731
    calls = [("pg_paged_kv4_attention_dev", dense, (2,)), ("pg_paged_kv4_attention_selected_dev", chosen, (2, 2)), ("pg_paged_kv4_select_dev", select, (2,)),
             ("pg_paged_kv4_summarise_dev", lambda width: (host.ctx, c, buf, buf, 2, 3, buf, width), (2,)),
             ("pg_paged_kv4_attention_scratch", lambda width: (host.ctx, c, 4, 2, 2, width, C.byref(n)), (2,)),
             ("pg_paged_kv4_selected_scratch", lambda top: (host.ctx, c, 4, 3, top, C.byref(n)), (2,))]
    for name, args, good in calls:
        host.ok(name, *args(*good))
        host.lib.pghost_clear_launches()
        for at in range(len(good)):
            assert status(host, name, *args(*good[:at], many, *good[at + 1:])) == EINVAL, name
        assert host.lib.pghost_num_launches() == 0
    a, keep = step(host, c, width=many, top=many)
    for name, args in (("pg_paged_kv4_attention", ("q", "heads", "starts", "lens", "batch", "tokens", "table", "width", "scale", "mask", "window", "sinks", "cap", "out")),
                       ("pg_paged_kv4_summarise", ("starts", "lens", "batch", "table", "width")),
                       ("pg_paged_kv4_select", ("q", "heads", "starts", "lens", "batch", "tokens", "table", "width", "top", "first", "recent", "selected"))):
        assert status(host, name, host.ctx, c, *(a[x] for x in args)) == EINVAL, name
    a["width"] = 2
    args = ("q", "heads", "starts", "lens", "batch", "tokens", "table", "width", "selected", "top", "scale", "cap", "out")
    assert status(host, "pg_paged_kv4_attention_selected", host.ctx, c, *(a[x] for x in args)) == EINVAL
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_tables_end_short_of_the_position_that_stands_for_none(host):
    """2^31 - 256 tokens: positions there and a tile behind them are still numbers of 32 bits."""
    most = (2 ** 31 - 256) // 16
    c, buf, n = new_cache(host), host.alloc(1 << 12), C.c_size_t()
    dense = lambda width: (host.ctx, c, buf, 256, 64, 4, buf, buf, 2, 3, 2, buf, width, 0.125, 1, 0, 0, 0.0, buf, 1 << 40, buf)  # noqa: E731
    chosen = lambda top: (host.ctx, c, buf, 256, 64, 4, buf, buf, 2, 3, buf, 8, buf, top, 0.125, 0.0, buf, 1 << 40, buf)  # noqa: E731
    for name, args in (("pg_paged_kv4_attention_dev", dense), ("pg_paged_kv4_attention_selected_dev", chosen),
                       ("pg_paged_kv4_attention_scratch", lambda width: (host.ctx, c, 4, 2, 2, width, C.byref(n))),
                       ("pg_paged_kv4_selected_scratch", lambda top: (host.ctx, c, 4, 3, top, C.byref(n)))):
        host.ok(name, *args(most))
        for more in (most + 1, (1 << 27) - 1):
            assert status(host, name, *args(more)) == EINVAL, name
    host.lib.pg_paged_kv4_free(host.ctx, c)


@pytest.mark.parametrize("row", [[-1, 0, 1], [0, -1, 1], [0, -1, 0], [-1, -1, 0], [1, -1, 0]])
def test_chosen_blocks_behind_a_gap_are_refused(host, row):
    c = new_cache(host)
    args = ("q", "heads", "starts", "lens", "batch", "tokens", "table", "width", "selected", "top", "scale", "cap", "out")
    for sel, want in (([0, 1, -1], None), ([0, -1, -1], None), ([-1, -1, -1], None), (row, EINVAL)):
        a, keep = step(host, c, selected=np.array([[sel] * 2] * 2 + [[[0, -1, -1]] * 2], np.int32), top=3)
        host.lib.pghost_clear_launches()
        st = status(host, "pg_paged_kv4_attention_selected", host.ctx, c, *(a[x] for x in args))
        assert (st == EINVAL) == (want == EINVAL) and (host.lib.pghost_num_launches() == 0) == (want == EINVAL), sel
    host.lib.pg_paged_kv4_free(host.ctx, c)


def test_mirror_refuses_numbers_that_32_bits_do_not_hold():
    """They would have become others: slot 2^32 + 3 slot 3.  No context is made."""
    from peregrine_amd import paged

    c = paged.PagedKV4Cache.__new__(paged.PagedKV4Cache)
    c.num_kv_heads, c.head_dim, c._h = 2, 64, None
    t = paged.BlockTables.__new__(paged.BlockTables)
    t.batch = 2
    k, q, ok_table = np.zeros((3, 2, 64)), np.zeros((3, 4, 64)), np.zeros((1, 2), np.int64)
    for bad in (2 ** 32 + 3, 2 ** 31, -2 ** 31 - 1, 0.5, float("nan")):
        for call in (lambda: c.append(k, k, [0, 1, bad]), lambda: c.read([bad]), lambda: t.extend([1, bad]), lambda: c.attention(q, [0, bad], [5], ok_table, 0.1),
                     lambda: c.attention(q, [0, 3], [bad], ok_table, 0.1), lambda: c.summarise([0, 3], [5], np.array([[0, bad]])),
                     lambda: c.attention_selected(q, [0, 3], [5], ok_table, np.full((3, 2, 1), bad), 0.1)):
            with pytest.raises(ValueError, match="32-bit"):
                call()
    assert (paged._ints([1.0, -1.0], "x") == [1, -1]).all() and paged._ints(np.zeros((2, 0)), "x").dtype == np.int32
