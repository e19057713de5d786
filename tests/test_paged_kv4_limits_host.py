"""Refusals of the block tables and the paged 4-bit cache at the ends of what they take, without a GPU (the library's own objects on a
HIP runtime in host memory that notes kernels instead of running them)."""
import numpy as np
import pytest

from test_host_runtime import host  # noqa: F401  (the fixture)
from test_paged_kv4_host import EINVAL, extend_args, i32, p, status


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
