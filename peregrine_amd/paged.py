"""A key/value cache that many requests share, held in 4 bits, with the block tables that say where each request's tokens
lie (no counterpart in the reference, whose caches belong to one sequence each).  Arrays in and out are NumPy's; a serving
loop that keeps its lengths and tables on the device calls the `_dev` forms of the C ABI instead."""
import ctypes as C

import numpy as np

from . import _ffi
from .context import default_context
from .llama import AttentionMask
from .quant import _ptr


def _ints(a, what):
    """`a` as 32-bit integers; numbers that are none are refused, not wrapped."""
    a = np.asarray(a)
    if a.dtype == np.int32:
        return np.ascontiguousarray(a)
    with np.errstate(invalid="ignore"):
        b = np.ascontiguousarray(a, np.int32)
    if not (b == a).all():
        raise ValueError(f"{what}: not 32-bit integers")
    return b


def _i32(a, n, what):
    a = _ints(a, what).reshape(-1)
    if a.size != n:
        raise ValueError(f"{what}: {a.size} values, not {n}")
    return a


class BlockTables:
    """Lengths and block tables of `batch` requests over a pool of `num_blocks` blocks of `block_size` tokens."""

    def __init__(self, batch, num_blocks, block_size, max_blocks, ctx=None):
        self.ctx = ctx or default_context()
        self.batch, self.num_blocks, self.block_size, self.max_blocks = int(batch), int(num_blocks), int(block_size), int(max_blocks)
        self.lens = np.zeros(self.batch, np.int32)
        self.table = np.full((self.batch, self.max_blocks), -1, np.int32)
        self.free_list = np.arange(self.num_blocks - 1, -1, -1, dtype=np.int32)   # block 0 is handed out first
        self.free_count = np.array([self.num_blocks], np.int32)

    def extend(self, new_lens, max_tokens=None):
        """Room for new_lens[b] more tokens of request b: (query_start [batch + 1], granted [batch], slots [max_tokens])."""
        new = _i32(new_lens, self.batch, "BlockTables.extend: new_lens")
        n = int(new.sum()) if max_tokens is None else int(max_tokens)
        starts, granted, slots = np.zeros(self.batch + 1, np.int32), np.zeros(self.batch, np.int32), np.zeros(n, np.int32)
        lens, count = np.zeros_like(self.lens), np.zeros_like(self.free_count)
        _ffi.check(_ffi.lib.pg_block_tables_extend(
            self.ctx.handle, _ptr(self.lens), _ptr(new), self.batch, self.block_size, _ptr(self.free_list), _ptr(self.free_count), self.num_blocks,
            _ptr(self.table), self.max_blocks, _ptr(lens), _ptr(count), _ptr(starts), _ptr(granted), _ptr(slots), n))
        self.lens, self.free_count = lens, count
        return starts, granted, slots

    def release(self, done):
        """The blocks of the requests with a true `done` back to the pool."""
        flags = _i32(np.asarray(done) != 0, self.batch, "BlockTables.release: done")
        _ffi.check(_ffi.lib.pg_block_tables_release(self.ctx.handle, _ptr(flags), _ptr(self.lens), self.batch, self.block_size, _ptr(self.table),
                                                    self.max_blocks, _ptr(self.free_list), _ptr(self.free_count), self.num_blocks))


class PagedKV4Cache:
    """`num_blocks` blocks of `block_size` tokens' keys and values, a row of 4-bit codes with one centre and step per
    token and head (include/peregrine_hip.h says how a row is rounded)."""

    def __init__(self, num_blocks, block_size, num_kv_heads, head_dim, ctx=None):
        self.ctx = ctx or default_context()
        self.num_blocks, self.block_size, self.num_kv_heads, self.head_dim = int(num_blocks), int(block_size), int(num_kv_heads), int(head_dim)
        self._h = C.c_void_p()
        _ffi.check(_ffi.lib.pg_paged_kv4_create(self.ctx.handle, self.num_blocks, self.block_size, self.num_kv_heads, self.head_dim, C.byref(self._h)))

    def _rows(self, a, what):
        a = np.ascontiguousarray(a, np.float32)
        if a.ndim != 3 or a.shape[1] % self.num_kv_heads or a.shape[2] != self.head_dim:
            raise ValueError(f"{what} is not [tokens, heads, {self.head_dim}] with a multiple of {self.num_kv_heads} heads")
        return a

    def _step(self, query_start, seq_lens, block_table):
        lens = _ints(seq_lens, "seq_lens").reshape(-1)
        table = _ints(block_table, "block_table")
        if table.ndim != 2 or table.shape[0] != lens.size:
            raise ValueError("block_table is not [batch, max_blocks]")
        return _i32(query_start, lens.size + 1, "query_start"), lens, table

    @property
    def nbytes(self):
        n = C.c_size_t()
        _ffi.check(_ffi.lib.pg_paged_kv4_info(self._h, None, None, None, None, C.byref(n)))
        return n.value

    def append(self, k, v, slots):
        """k, v [tokens, num_kv_heads, head_dim] into their slots (-1: left out)."""
        k, v = self._rows(k, "k"), self._rows(v, "v")
        if k.shape != v.shape or k.shape[1] != self.num_kv_heads:
            raise ValueError("PagedKV4Cache.append: k and v are not [tokens, num_kv_heads, head_dim]")
        slots = _i32(slots, k.shape[0], "slots")
        _ffi.check(_ffi.lib.pg_paged_kv4_append(self.ctx.handle, self._h, _ptr(k.reshape(-1)), _ptr(v.reshape(-1)), k.shape[0], _ptr(slots)))

    def read(self, slots):
        """(k, v) of the slots, [n, num_kv_heads, head_dim] each, as the values that the codes stand for."""
        slots = _ints(slots, "PagedKV4Cache.read: slots").reshape(-1)
        k, v = (np.zeros((slots.size, self.num_kv_heads, self.head_dim), np.float32) for _ in range(2))
        _ffi.check(_ffi.lib.pg_paged_kv4_read(self.ctx.handle, self._h, _ptr(slots), slots.size, _ptr(k.reshape(-1)), _ptr(v.reshape(-1))))
        return k, v

    def attention(self, q, query_start, seq_lens, block_table, scale, mask=None, logit_cap=None):
        """q [tokens, num_q_heads, head_dim] -> the same shape.  `mask`: AttentionMask.causal(0) (the default), .none() or
        .causal_sliding_window(0, window, sink_tokens); a row's position is its token's, so an offset other than 0 is refused."""
        mask = mask or AttentionMask.causal(0)
        if mask.offset:
            raise ValueError("PagedKV4Cache.attention: rows stand at the ends of their requests: the mask's offset is 0")
        q = self._rows(q, "q")
        starts, lens, table = self._step(query_start, seq_lens, block_table)
        out = np.zeros_like(q)
        _ffi.check(_ffi.lib.pg_paged_kv4_attention(self.ctx.handle, self._h, _ptr(q.reshape(-1)), q.shape[1], _ptr(starts), _ptr(lens), lens.size, q.shape[0],
                                                   _ptr(table.reshape(-1)), table.shape[1], float(scale), mask.kind, mask.window, mask.sink_tokens,
                                                   float(logit_cap or 0.0), _ptr(out.reshape(-1))))
        return out

    def summarise(self, query_start, seq_lens, block_table):
        """Brings the summaries of the blocks that a step's rows touched up to date (after its append)."""
        starts, lens, table = self._step(query_start, seq_lens, block_table)
        _ffi.check(_ffi.lib.pg_paged_kv4_summarise(self.ctx.handle, self._h, _ptr(starts), _ptr(lens), lens.size, _ptr(table.reshape(-1)), table.shape[1]))

    def select(self, q, query_start, seq_lens, block_table, top_k, first_blocks=1, recent_blocks=1):
        """The blocks to read for each row and key head: [tokens, num_kv_heads, top_k], ascending, -1 behind them."""
        q = self._rows(q, "q")
        starts, lens, table = self._step(query_start, seq_lens, block_table)
        out = np.full((q.shape[0], self.num_kv_heads, int(top_k)), -1, np.int32)
        _ffi.check(_ffi.lib.pg_paged_kv4_select(self.ctx.handle, self._h, _ptr(q.reshape(-1)), q.shape[1], _ptr(starts), _ptr(lens), lens.size, q.shape[0],
                                                _ptr(table.reshape(-1)), table.shape[1], int(top_k), int(first_blocks), int(recent_blocks), _ptr(out.reshape(-1))))
        return out

    def attention_selected(self, q, query_start, seq_lens, block_table, selected, scale, logit_cap=None):
        """Causal attention over the selected blocks alone."""
        q = self._rows(q, "q")
        starts, lens, table = self._step(query_start, seq_lens, block_table)
        sel = _ints(selected, "PagedKV4Cache.attention_selected: selected")
        if sel.ndim != 3 or sel.shape[:2] != (q.shape[0], self.num_kv_heads):
            raise ValueError("PagedKV4Cache.attention_selected: selected is not [tokens, num_kv_heads, top_k]")
        out = np.zeros_like(q)
        _ffi.check(_ffi.lib.pg_paged_kv4_attention_selected(self.ctx.handle, self._h, _ptr(q.reshape(-1)), q.shape[1], _ptr(starts), _ptr(lens), lens.size, q.shape[0],
                                                            _ptr(table.reshape(-1)), table.shape[1], _ptr(sel.reshape(-1)), sel.shape[2], float(scale),
                                                            float(logit_cap or 0.0), _ptr(out.reshape(-1))))
        return out

    def free(self):
        if self._h:
            _ffi.lib.pg_paged_kv4_free(self.ctx.handle, self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
