"""The paged 4-bit cache on the GPU against plain NumPy (tests/paged_ref.py): whole numbers and stored values bit for bit,
attention within a bound by arithmetic (paged_ref.attend says which) and, over all of a call's outputs, 2-norms within 3e-6:
sixteen roundings' worth of f32, which independent ones stay far under."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from devbuf import DevBuf

pytestmark = pytest.mark.gpu
F = np.float32


def lib():
    from peregrine_amd import _ffi
    return _ffi.lib


def ok(st):
    from peregrine_amd import _ffi
    _ffi.check(st)


def bits(a):
    return np.ascontiguousarray(a, F).view(np.uint32)


def same(got, want, what=""):
    """Bit for bit, NaNs as NaNs."""
    got, want = np.asarray(got), np.asarray(want)
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), what
    assert (bits(got)[~nan] == bits(want)[~nan]).all(), what


def ints(a):
    return np.ascontiguousarray(a, np.int32)


class World:
    """A cache, its reference, and requests with shuffled blocks.  Every slot that is not a request's token holds NaN rows."""

    def __init__(self, ctx, lens, heads, hd, bs, seed=0, spare=2, poison=True, loud=0.5, first_block=0):
        self.ctx, self.lens, self.heads, self.hd, self.bs = ctx, np.array(lens, np.int32), heads, hd, bs
        rng = self.rng = np.random.default_rng(seed)
        need = [-(-n // bs) for n in lens]
        self.nb = first_block + sum(need) + spare
        order = first_block + rng.permutation(self.nb - first_block)
        self.width = max(1, max(need)) + 1
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at: at + n]
            at += n
        from peregrine_amd import paged
        self.cache, self.ref = paged.PagedKV4Cache(self.nb, bs, heads, hd, ctx), R.Cache(self.nb if first_block == 0 else 1, bs, heads, hd)
        if first_block:
            self.ref = None
        if poison:
            every = np.arange(self.nb * bs, dtype=np.int32)
            x = np.full((every.size, heads, hd), np.nan, F)
            self.put(x, x, every)
        self.loud = (loud * rng.standard_normal((heads, hd))).astype(F)
        for b, n in enumerate(lens):
            if n:
                self.put(self.keys(n), rng.standard_normal((n, heads, hd)).astype(F), self.slots(b, np.arange(n)))

    def keys(self, n):
        return (self.rng.standard_normal((n, self.heads, self.hd)).astype(F) + self.loud).astype(F)

    def slots(self, b, pos):
        return R.slots_of(self.table[b], np.asarray(pos), self.bs).astype(np.int32)

    def put(self, k, v, slots):
        self.cache.append(k, v, slots)
        if self.ref:
            self.ref.append(k, v, slots)

    def q(self, rows, q_heads, std=1.5):
        return (std * self.rng.standard_normal((rows, q_heads, self.hd))).astype(F)

    def check(self, got, q, rows, scale, mask=1, window=0, sinks=0, cap=0.0, only=None, what=""):
        """got [tokens, q_heads, hd] of requests with `rows` rows each at their ends; only(t, head) -> the blocks read."""
        group, t, off, size = q.shape[1] // self.heads, 0, 0.0, 0.0
        for b, n in enumerate(rows):
            keys = np.arange(self.lens[b])
            at = self.slots(b, keys) if self.lens[b] else np.zeros(0, np.int64)
            k, v = self.ref.f64(0, at), self.ref.f64(1, at)
            for i in range(n):
                pos = self.lens[b] - n + i
                seen = np.ones(keys.size, bool) if mask == 0 else keys <= pos
                if mask == 2:
                    seen &= (pos - keys <= window) | (keys < sinks)
                for j in range(q.shape[1]):
                    h = j // group
                    s = seen if only is None else seen & np.isin(keys // self.bs, only(t, h))
                    want, bound = R.attend(q[t, j], k[:, h], v[:, h], scale, s, cap)
                    d = np.abs(got[t, j] - want)
                    assert (d <= bound).all(), f"{what}: request {b}, row {i}, head {j}: off by {d.max():.3g}, bound {bound.min():.3g}"
                    off += (d ** 2).sum()
                    size += (want ** 2).sum()
                t += 1
        assert size == 0 or (off / size) ** 0.5 < 3e-6, f"{what}: 2-norm off by {(off / size) ** 0.5:.3g}"


# ------------------------------------------------------------------------------------------------------ tables
def extend_ref(lens, new, bs, width, table, free, count, max_tokens):
    table, lens, out, granted, starts, slots, used, asked = table.copy(), lens.copy(), lens.copy(), [], [0], np.full(max_tokens, -1, np.int32), 0, 0
    for b, (n, a) in enumerate(zip(np.maximum(lens, 0), np.maximum(new, 0))):
        have = -(-int(n) // bs)
        fits = int(n) + int(a) <= width * bs
        need = -(-(int(n) + int(a)) // bs) - have if fits else 0
        yes = fits and (need == 0 or asked + need <= count)
        if yes:
            for j in range(need):
                table[b, have + j] = free[count - 1 - asked - j]
            used += need
            for i in range(a):
                if starts[-1] + i < max_tokens:
                    slots[starts[-1] + i] = table[b, (n + i) // bs] * bs + (n + i) % bs
        asked += need
        out[b] = n + a if yes else n
        granted.append(int(yes))
        starts.append(min(starts[-1] + int(a), max_tokens))
    return table, out, count - used, starts, granted, slots


@pytest.mark.parametrize("batch", [1, 5, 64, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("bs,most,new,short", [(16, 300, 1, False), (64, 500, 40, True), (128, 90, 2, True), (16, 200, 9, False)])
def test_extend_is_the_scan(ctx, batch, bs, most, new, short):
    rng = np.random.default_rng(batch * 7 + bs + new)
    lens, add = rng.integers(0, most, batch).astype(np.int32), rng.integers(0, new + 1, batch).astype(np.int32)
    width = max(1, -(-(most + new) // bs) - (1 if short else 0))         # a table some requests do not fit (of no blocks is refused)
    have = -(-lens // bs)
    lens = np.minimum(lens, width * bs).astype(np.int32)
    have = -(-lens // bs)
    need = int((-(-(lens + add) // bs) - have).clip(0).sum())
    nb = int(have.sum()) + need + 3
    ids = rng.permutation(nb).astype(np.int32)
    table = np.full((batch, width), -1, np.int32)
    at = 0
    for b in range(batch):
        table[b, :have[b]] = ids[at: at + have[b]]
        at += have[b]
    count = max(0, need // 2) if short else need + 3
    free = np.zeros(nb, np.int32)
    free[:count] = ids[at: at + count]
    tokens = int(add.sum()) + 3
    want = extend_ref(lens, add, bs, width, table, free, count, tokens)
    dev = [DevBuf(ctx, host=x) for x in (lens, add, free, ints([count]), table)]
    out = [DevBuf(ctx, host=np.full(n, 77, np.int32)) for n in (batch + 1, batch, tokens)]
    for _ in range(2):                                                    # the same inputs again: the same outputs
        lens_out, count_out = DevBuf(ctx, host=np.full(batch, 77, np.int32)), DevBuf(ctx, host=ints([77]))
        ok(lib().pg_block_tables_extend_dev(ctx.handle, dev[0].ptr, dev[1].ptr, batch, bs, dev[2].ptr, dev[3].ptr, nb, dev[4].ptr, width, lens_out.ptr, count_out.ptr,
                                            out[0].ptr, out[1].ptr, out[2].ptr, tokens))
        got = [dev[4].to_host(np.int32).reshape(batch, width), lens_out.to_host(np.int32), count_out.to_host(np.int32)[0], out[0].to_host(np.int32), out[1].to_host(np.int32),
               out[2].to_host(np.int32)]
        for g, w in zip(got, want):
            assert (np.asarray(g) == np.asarray(w)).all()


def test_extend_in_place_cuts_what_does_not_fit(ctx):
    """Lengths and count written over their inputs; negative lengths count as 0, a slot map that is too short is cut."""
    lens, add, free = ints([-4, 17, 3]), ints([2, -9, 20]), ints([5, 6, 7, 8])
    table = ints([[-1, -1], [3, 4], [2, -1]])
    for tokens in (30, 11, 1, 0):
        want = extend_ref(lens, add, 16, 2, table, free, 4, tokens)
        d = [DevBuf(ctx, host=x) for x in (lens, add, free, ints([4]), table, np.zeros(4, np.int32), np.zeros(3, np.int32), np.full(tokens + 2, 55, np.int32))]
        ok(lib().pg_block_tables_extend_dev(ctx.handle, d[0].ptr, d[1].ptr, 3, 16, d[2].ptr, d[3].ptr, 9, d[4].ptr, 2, d[0].ptr, d[3].ptr, d[5].ptr, d[6].ptr, d[7].ptr, tokens))
        got = [d[4].to_host(np.int32).reshape(3, 2), d[0].to_host(np.int32), d[3].to_host(np.int32)[0], d[5].to_host(np.int32), d[6].to_host(np.int32)]
        for g, w in zip(got, want):
            assert (np.asarray(g) == np.asarray(w)).all()
        slots = d[7].to_host(np.int32)
        assert (slots[:tokens] == want[5]).all() and (slots[tokens:] == 55).all()


@pytest.mark.parametrize("batch,most_new,in_place", [(30, 900, False), (30, 900, True), (700, 40, True), (4097, 6, False), (4097, 6, True), (2000, 12, False)])
def test_extend_over_many_rows(ctx, batch, most_new, in_place):
    """More rows than one workgroup maps to slots: by several, or by a second launch where lengths are written over their inputs."""
    rng = np.random.default_rng(batch + most_new)
    bs = 16
    lens, add = rng.integers(0, 200, batch).astype(np.int32), rng.integers(0, most_new + 1, batch).astype(np.int32)
    width = -(-(200 + most_new) // bs)
    have = -(-lens // bs)
    need = int((-(-(lens + add) // bs) - have).sum())
    nb = int(have.sum()) + need + 3
    ids = rng.permutation(nb).astype(np.int32)
    table = np.full((batch, width), -1, np.int32)
    for b, at in enumerate(np.cumsum(have) - have):
        table[b, :have[b]] = ids[at: at + have[b]]
    count = need - 20                                                     # the last requests get none
    free = np.zeros(nb, np.int32)
    free[:count] = ids[have.sum(): have.sum() + count]
    tokens = int(add.sum()) + 5
    assert tokens > 4096
    want = extend_ref(lens, add, bs, width, table, free, count, tokens)
    d = [DevBuf(ctx, host=x) for x in (lens, add, free, ints([count]), table, np.zeros(batch + 1, np.int32), np.zeros(batch, np.int32), np.full(tokens, 77, np.int32))]
    lens_out, count_out = (d[0], d[3]) if in_place else (DevBuf(ctx, host=np.full(batch, 77, np.int32)), DevBuf(ctx, host=ints([77])))
    ok(lib().pg_block_tables_extend_dev(ctx.handle, d[0].ptr, d[1].ptr, batch, bs, d[2].ptr, d[3].ptr, nb, d[4].ptr, width, lens_out.ptr, count_out.ptr, d[5].ptr, d[6].ptr,
                                        d[7].ptr, tokens))
    got = [d[4].to_host(np.int32).reshape(batch, width), lens_out.to_host(np.int32), count_out.to_host(np.int32)[0], d[5].to_host(np.int32), d[6].to_host(np.int32),
           d[7].to_host(np.int32)]
    for g, x in zip(got, want):
        assert (np.asarray(g) == np.asarray(x)).all()


@pytest.mark.parametrize("batch", [1, 70, 1100])
def test_release_gives_every_block_back_in_order(ctx, batch):
    rng = np.random.default_rng(batch)
    from peregrine_amd import paged
    t = paged.BlockTables(batch, batch * 6, 16, 5, ctx)
    t.extend(rng.integers(0, 80, batch))
    assert (t.lens >= 0).all()
    before = {b: list(t.table[b][t.table[b] >= 0]) for b in range(batch)}
    flags = rng.random(batch) < 0.6
    free0 = list(t.free_list[: t.free_count[0]])
    lens0 = t.lens.copy()
    t.release(flags)
    want = free0 + [e for b in range(batch) if flags[b] for e in before[b]]
    assert list(t.free_list[: t.free_count[0]]) == want
    assert (t.lens == np.where(flags, 0, lens0)).all() and (t.table[flags] == -1).all()
    t.release(np.ones(batch))
    assert sorted(t.free_list[: t.free_count[0]]) == list(range(batch * 6))


def test_release_skips_entries_that_are_no_block(ctx):
    d = [DevBuf(ctx, host=x) for x in (ints([1, 1]), ints([40, 500]), ints([[3, -1, 9], [4, 2, 1]]), np.zeros(5, np.int32), ints([1]))]
    ok(lib().pg_block_tables_release_dev(ctx.handle, d[0].ptr, d[1].ptr, 2, 16, d[2].ptr, 3, d[3].ptr, d[4].ptr, 5))
    assert d[4].to_host(np.int32)[0] == 5 and list(d[3].to_host(np.int32)) == [0, 3, 4, 2, 1]


# ------------------------------------------------------------------------------------------------------ append, read
@pytest.mark.parametrize("hd", [1, 7, 40, 64, 80, 100, 128, 130, 192, 256])
@pytest.mark.parametrize("heads,bs", [(1, 16), (3, 64), (8, 128)])
def test_append_stores_the_formula_bit_for_bit(ctx, hd, heads, bs):
    from peregrine_amd import paged
    rng = np.random.default_rng(hd * 10 + heads)
    n, nb = 150, 300 // bs + 2
    k, v = (rng.standard_normal((n, heads, hd)) * np.exp(rng.uniform(-12, 12, (n, heads, 1)))).astype(F), rng.standard_normal((n, heads, hd)).astype(F)
    v += rng.uniform(-50, 50, (n, heads, 1)).astype(F)                    # a centre far from 0
    k[0], k[1], k[2, 0, 0], k[3, -1, -1], k[4] = 0, 3.7, np.nan, -np.inf, 1e-39   # a row of zeros, a constant, none finite, denormals
    k[5, :, 0], k[6] = 3e38, -0.0
    if hd > 1:
        k[5, :, 1] = -3e38                                                # a spread beyond f32
    slots = rng.permutation(nb * bs)[:n].astype(np.int32)
    slots[10] = -1
    c, ref = paged.PagedKV4Cache(nb, bs, heads, hd, ctx), R.Cache(nb, bs, heads, hd)
    c.append(k, v, slots)
    ref.append(k, v, slots)
    every = np.arange(nb * bs)
    for side, got in enumerate(c.read(every)):
        same(got, ref.f32(side, every), f"side {side}")


@pytest.mark.parametrize("hd,shift", [(64, 0), (128, 1), (80, 0), (100, 2), (256, 3)])
def test_append_from_strided_rows(ctx, hd, shift):
    """Heads first as a cache has them, rows of a fused product, and rows that no vector load can take."""
    from peregrine_amd import paged
    rng = np.random.default_rng(hd)
    heads, n, bs, nb = 2, 21, 16, 4
    x = rng.standard_normal((2, heads, n, hd)).astype(F)
    slots = rng.permutation(nb * bs)[:n].astype(np.int32)
    ref = R.Cache(nb, bs, heads, hd)
    ref.append(x[0].transpose(1, 0, 2), x[1].transpose(1, 0, 2), slots)
    for token_stride, head_stride in ((hd, n * hd), (heads * hd * 3 + shift, hd), (heads * (hd + shift), hd + shift)):
        big = np.zeros((2, shift + n * max(token_stride, 1) + heads * head_stride + hd), F)
        for side in range(2):
            for h in range(heads):
                for t in range(n):
                    at = shift + t * token_stride + h * head_stride
                    big[side, at: at + hd] = x[side, h, t]
        c, k, v, s = paged.PagedKV4Cache(nb, bs, heads, hd, ctx), DevBuf(ctx, host=big[0]), DevBuf(ctx, host=big[1]), DevBuf(ctx, host=slots)
        ok(lib().pg_paged_kv4_append_dev(ctx.handle, c._h, C.c_void_p(k.ptr.value + 4 * shift), C.c_void_p(v.ptr.value + 4 * shift), token_stride, head_stride, n, s.ptr))
        for side, got in enumerate(c.read(slots)):
            same(got, ref.f32(side, slots))


def test_append_and_read_leave_out_slots_that_are_none(ctx):
    from peregrine_amd import paged
    heads, hd, bs, nb = 2, 64, 16, 2
    c, x = paged.PagedKV4Cache(nb, bs, heads, hd, ctx), np.ones((5, heads, hd), F)
    k, s = DevBuf(ctx, host=x), DevBuf(ctx, host=ints([-1, 32, 2 ** 31 - 1, -2 ** 31, 7]))
    ok(lib().pg_paged_kv4_append_dev(ctx.handle, c._h, k.ptr, k.ptr, heads * hd, hd, 5, s.ptr))
    every, _ = c.read(np.arange(nb * bs))
    assert (every[7] == 1).all() and (np.delete(every, 7, 0) == 0).all()
    o = DevBuf(ctx, host=np.full(x.size, 9, F)), DevBuf(ctx, host=np.full(x.size, 9, F))
    ok(lib().pg_paged_kv4_read_dev(ctx.handle, c._h, s.ptr, 5, o[0].ptr, o[1].ptr))
    for b in o:
        got = b.to_host(F).reshape(x.shape)
        assert (got[:4] == 0).all() and (got[4] == 1).all()


# ------------------------------------------------------------------------------------------------------ attention
MASKS = [dict(), dict(mask=0), dict(mask=2, window=0, sinks=0), dict(mask=2, window=20, sinks=3), dict(mask=2, window=100, sinks=70), dict(cap=5.0)]


@pytest.mark.parametrize("hd,heads,group,bs", [(64, 2, 7, 16), (128, 2, 4, 64), (256, 1, 8, 32), (80, 3, 1, 16), (128, 1, 16, 128), (40, 1, 17, 16), (128, 1, 40, 256), (200, 2, 2, 64), (1, 1, 3, 16)])
@pytest.mark.parametrize("rows", ["one", "few", "many"])
def test_attention_against_64_bits(ctx, hd, heads, group, bs, rows):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 0, 130, 257, 300] if rows != "many" else [1, 20, 0, 70, 131]
    w = World(ctx, lens, heads, hd, bs, seed=hd + group)
    n = [min(x, r) for x, r in zip(lens, {"one": [1] * 14, "few": [1, 2, 3, 4, 5, 0, 2, 3, 1, 4, 0, 5, 3, 2], "many": [1, 20, 0, 37, 131]}[rows])]
    q = w.q(sum(n), heads * group)
    starts = np.concatenate([[0], np.cumsum(n)])
    for m in MASKS if rows != "many" else MASKS[:1] + MASKS[3:]:
        from peregrine_amd import llama
        mask = llama.AttentionMask(m.get("mask", 1), 0, m.get("window", 0), m.get("sinks", 0))
        got = w.cache.attention(q, starts, w.lens, w.table, hd ** -0.5, mask, m.get("cap"))
        w.check(got, q, n, hd ** -0.5, what=str(m), **m)


@pytest.mark.parametrize("hd,group,lens,bs", [(128, 4, [4111, 900], 64), (64, 1, [5000], 16), (256, 2, [3001], 128)])
def test_attention_over_long_contexts(ctx, hd, group, lens, bs):
    """Keys divided between workgroups and joined; one request's queries far from the others'."""
    w = World(ctx, lens, 2, hd, bs, seed=5, poison=False)
    q = w.q(len(lens), 2 * group)
    for std in (0.05, 1.0, 8.0):                                          # flat, ordinary and peaked rows
        x = (q * F(std)).astype(F)
        got = w.cache.attention(x, np.arange(len(lens) + 1), w.lens, w.table, hd ** -0.5)
        w.check(got, x, [1] * len(lens), hd ** -0.5, what=f"std {std}")
        again = w.cache.attention(x, np.arange(len(lens) + 1), w.lens, w.table, hd ** -0.5)
        assert (bits(got) == bits(again)).all()


def test_one_key_among_many_and_values_of_very_different_sizes(ctx):
    """A key that takes nearly all of a row's weight, thousands with next to none; values from 1e-20 to 1e20."""
    hd, n = 128, 2000
    w = World(ctx, [n], 1, hd, 64, seed=9, poison=False)
    q = w.q(1, 2, std=1.0)
    k = (0.3 * w.rng.standard_normal((n, 1, hd))).astype(F)
    k[1234, 0] = q[0, 0] * F(1.4)
    v = (w.rng.standard_normal((n, 1, hd)) + 1).astype(F)
    w.put(k, v, w.slots(0, np.arange(n)))
    w.check(w.cache.attention(q, [0, 1], w.lens, w.table, hd ** -0.5), q, [1], hd ** -0.5, what="needle")
    v = (v * np.exp(np.linspace(-46, 46, n))[:, None, None]).astype(F)
    for order in (np.arange(n), np.arange(n)[::-1]):
        w.put(k, v[order], w.slots(0, np.arange(n)))
        w.check(w.cache.attention(q, [0, 1], w.lens, w.table, hd ** -0.5), q, [1], hd ** -0.5, what="values")


@pytest.mark.parametrize("hd,group,rows", [(64, 1, 1), (128, 4, 1), (128, 8, 1), (128, 16, 1), (64, 16, 1), (256, 4, 1), (256, 8, 1), (256, 16, 1), (64, 4, 20), (128, 4, 20), (256, 4, 20)])
def test_values_near_the_smallest(ctx, hd, group, rows):
    """Rows' steps at and just over the smallest there is (2^-120), zeros before and between them."""
    n = 150
    w = World(ctx, [n], 1, hd, 16, seed=hd + group + rows, poison=False)
    for top in (1e-35, 2e-34):
        v = (w.rng.standard_normal((n, 1, hd)) * np.exp(w.rng.uniform(-3, 0, (n, 1, 1))) * top / 3).astype(F)
        v[:70], v[100] = 0, 0
        w.put(w.keys(n), v, w.slots(0, np.arange(n)))
        q = w.q(rows, group)
        w.check(w.cache.attention(q, [0, rows], w.lens, w.table, hd ** -0.5), q, [rows], hd ** -0.5, what=f"values of {top}")


@pytest.mark.parametrize("batch,heads,group", [(140, 4, 4), (256, 3, 2), (257, 2, 8), (256, 3, 16), (65, 8, 20)])
def test_more_requests_than_run_at_once(ctx, batch, heads, group):
    """Requests are taken the longest first then; lengths that are equal, and none."""
    hd = 64
    lens = np.random.default_rng(batch + group).integers(0, 40, batch) * np.where(np.arange(batch) % 5 == 0, 4, 1)
    lens[-1], lens[batch // 2] = 0, 150
    w = World(ctx, [int(x) for x in lens], heads, hd, 16, seed=batch, poison=False)
    rows = [int(min(x, 1)) for x in lens]
    q = w.q(sum(rows), heads * group)
    w.check(w.cache.attention(q, np.concatenate([[0], np.cumsum(rows)]), w.lens, w.table, hd ** -0.5), q, rows, hd ** -0.5)


class Step:
    """Device arrays of a step, for the `_dev` forms."""

    def __init__(self, ctx, w, q, starts, lens=None, table=None, max_query=None):
        self.ctx, self.w, self.q = ctx, w, q
        lens, table = w.lens if lens is None else lens, w.table if table is None else table
        self.batch, self.tokens, self.width = len(lens), q.shape[0], table.shape[1]
        self.d = [DevBuf(ctx, host=x) for x in (ints(starts), ints(lens), ints(table), q)]
        self.max_query = max_query or int(max(1, np.diff(starts).max()))
        n = C.c_size_t()
        ok(lib().pg_paged_kv4_attention_scratch(ctx.handle, w.cache._h, q.shape[1], self.batch, self.max_query, self.width, C.byref(n)))
        self.scratch = DevBuf(ctx, max(16, n.value))
        self.size = n.value
        self.out = DevBuf(ctx, host=np.full(q.shape, 123.0, F))

    def attention(self, ctx=None, strides=None, mask=1, window=0, sinks=0, cap=0.0, q=None):
        starts, lens, table, qd = self.d
        st = strides or (self.q.shape[1] * self.q.shape[2], self.q.shape[2])
        ok(lib().pg_paged_kv4_attention_dev((ctx or self.ctx).handle, self.w.cache._h, q or qd.ptr, *st, self.q.shape[1], starts.ptr, lens.ptr, self.batch, self.tokens,
                                            self.max_query, table.ptr, self.width, self.w.hd ** -0.5, mask, window, sinks, cap, self.scratch.ptr, self.size, self.out.ptr))

    def result(self):
        return self.out.to_host(F).reshape(self.q.shape)


def test_rows_behind_the_last_are_left_and_strided_queries_read(ctx):
    w = World(ctx, [40, 7], 2, 64, 16, seed=3)
    n, heads, hd = [3, 2], 6, 64
    q = w.q(9, heads)                                                     # four rows more than the step has
    s = Step(ctx, w, q, [0, 3, 5])
    s.attention()
    got = s.result()
    w.check(got[:5], q[:5], n, hd ** -0.5)
    assert (got[5:] == 123).all()
    for shape, strides, at in (((heads, 9, hd), (hd, 9 * hd), lambda t, j: (j, t)), ((9, heads, hd + 3), (heads * (hd + 3), hd + 3), lambda t, j: (t, j))):
        x = np.full(shape, np.nan, F)
        for t in range(9):
            for j in range(heads):
                x[at(t, j)][:hd] = q[t, j]
        buf = DevBuf(ctx, host=x)
        s.out = DevBuf(ctx, host=np.full(q.shape, 123.0, F))
        s.attention(strides=strides, q=buf.ptr)
        assert (bits(s.result()) == bits(got)).all()


def test_rows_that_see_no_key_are_zero(ctx):
    """More rows than tokens (their positions are before the first), an empty request, and a request of no rows."""
    w = World(ctx, [2, 0, 5], 1, 64, 16, seed=4)
    q = w.q(8, 2)
    s = Step(ctx, w, q, [0, 4, 7, 8])
    for mask, window in ((1, 0), (2, 1), (0, 0)):
        s.attention(mask=mask, window=window)
        got = s.result()
        w2 = got.copy()
        if mask:
            assert (got[:2] == 0).all()
            w.check(w2[[2, 3, 7]], q[[2, 3, 7]], [2, 0, 1], 64 ** -0.5, mask=mask, window=window)
        assert (got[4:7] == 0).all()


def test_table_entries_that_are_no_block_are_left_out(ctx):
    w = World(ctx, [100], 2, 128, 16, seed=6, poison=False)
    q = w.q(1, 4)
    table = w.table.copy()
    table[0, 1], table[0, 3], table[0, 5] = -1, w.nb, 2 ** 31 - 1
    s = Step(ctx, w, q, [0, 1], table=table)
    s.attention()
    w.check(s.result(), q, [1], 128 ** -0.5, only=lambda t, h: [0, 2, 4, 6])
    s = Step(ctx, w, q, [0, 1], lens=ints([10 ** 9]))                     # a length behind the table is cut to it
    s.attention()
    s2 = Step(ctx, w, q, [0, 1], lens=ints([-5]))
    s2.attention()
    assert np.isfinite(s.result()).all() and (s2.result() == 0).all()


def test_values_that_are_not_finite_reach_the_rows_that_see_them_and_no_others(ctx):
    w = World(ctx, [70], 2, 64, 16, seed=7)
    q = w.q(6, 4)                                                         # rows at 64 .. 69
    bad = w.keys(1)
    bad[0, 1, 3] = np.inf                                                 # key head 1 alone
    w.put(bad, np.ones((1, 2, 64), F), w.slots(0, [67]))
    got = w.cache.attention(q, [0, 6], w.lens, w.table, 0.125)
    assert np.isnan(got[3:, 2:]).all() and np.isfinite(got[:3]).all() and np.isfinite(got[:, :2]).all()
    w.put(w.keys(1), np.full((1, 2, 64), np.nan, F), w.slots(0, [66]))
    w.put(w.keys(1), np.ones((1, 2, 64), F), w.slots(0, [67]))
    got = w.cache.attention(q, [0, 6], w.lens, w.table, 0.125)
    assert np.isnan(got[2:]).all() and np.isfinite(got[:2]).all()
    w.put(w.keys(1), np.ones((1, 2, 64), F), w.slots(0, [66]))
    x = q.copy()
    x[1, 2, 5], x[4, 0, 0] = np.nan, -np.inf
    got = w.cache.attention(x, [0, 6], w.lens, w.table, 0.125)
    want = np.zeros((6, 4), bool)
    want[1, 2] = want[4, 0] = True
    assert (np.isnan(got).all(-1) == want).all() and np.isfinite(got[~want]).all()
    x[:] = 0                                                              # all scores alike
    w.check(w.cache.attention(x, [0, 6], w.lens, w.table, 0.125), x, [6], 0.125)


def test_a_cache_of_more_than_four_gigabytes(ctx):
    """Blocks whose records begin behind 2^32 bytes, slots behind 2^22: the same bits as in a small cache."""
    heads, hd, bs, n = 8, 256, 256, 700
    far = (5 << 30) // (heads * bs * (hd + 8))
    a, b = (World(ctx, [n], heads, hd, bs, seed=11, poison=False, first_block=f) for f in (0, far))
    assert b.cache.nbytes > 5 << 30
    b.table = np.where(a.table >= 0, a.table + far, -1).astype(np.int32)
    rng = np.random.default_rng(1)
    k, v, q = rng.standard_normal((n, heads, hd)).astype(F), rng.standard_normal((n, heads, hd)).astype(F), rng.standard_normal((2, 2 * heads, hd)).astype(F)
    out = []
    for w in (a, b):
        w.cache.append(k, v, w.slots(0, np.arange(n)))
        w.cache.summarise([0, n], w.lens, w.table)
        sel = w.cache.select(q, [0, 2], w.lens, w.table, 2)
        out.append((w.cache.attention(q, [0, 2], w.lens, w.table, 0.06), sel, w.cache.attention_selected(q, [0, 2], w.lens, w.table, sel, 0.06), *w.cache.read(w.slots(0, np.arange(n)))))
        w.cache.free()
    for x, y in zip(*out):
        assert (x == y).all()


# ------------------------------------------------------------------------------------------------------ selection
@pytest.mark.parametrize("hd,heads,group,bs", [(64, 2, 3, 16), (128, 2, 4, 32), (256, 1, 8, 16), (80, 1, 20, 16), (40, 3, 1, 64)])
def test_summaries_and_selection_are_exact(ctx, hd, heads, group, bs):
    lens = [1, bs, bs + 1, 20 * bs - 3, 37 * bs + 5, 0, 9 * bs]
    w = World(ctx, lens, heads, hd, bs, seed=hd, spare=1)
    w.put(np.full((1, heads, hd), np.nan, F), np.ones((1, heads, hd), F), w.slots(4, [3 * bs + 1]))   # a block that is not to be missed
    w.put(np.zeros((bs, heads, hd), F), np.ones((bs, heads, hd), F), w.slots(6, np.arange(2 * bs, 3 * bs)))
    starts = np.concatenate([[0], np.cumsum(lens)])
    w.cache.summarise(starts, w.lens, w.table)
    for b, n in enumerate(lens):
        blocks = -(-n // bs)
        if not blocks:
            continue
        d = [DevBuf(ctx, host=x) for x in (w.table[b, :blocks], np.zeros((blocks, heads, hd), F), np.zeros((blocks, heads, hd), F))]
        ok(lib().pg_paged_kv4_read_summaries_dev(ctx.handle, w.cache._h, d[0].ptr, blocks, d[1].ptr, d[2].ptr))
        got = [x.to_host(F).reshape(blocks, heads, hd) for x in d[1:]]
        for j in range(blocks):
            lo, hi, s = R.summary(w.ref.f32(0, w.slots(b, np.arange(j * bs, min(n, j * bs + bs)))))
            with np.errstate(all="ignore"):
                for g, x in zip(got, (lo, hi)):
                    same(g[j], (x.astype(F) * s[:, None]).astype(F), f"request {b}, block {j}")
    rows = [1, 2, 3, 1, 5, 0, 2]
    q = w.q(sum(rows), heads * group)
    q[4, 0], q[5, 1 % (heads * group)] = 0, np.nan
    st = np.concatenate([[0], np.cumsum(rows)])
    for top, first, recent in ((4, 1, 1), (9, 0, 3), (2, 0, 1), (60, 2, 2), (3, 2, 1)):
        got = w.cache.select(q, st, w.lens, w.table, top, first, recent)
        t = 0
        for b, n in enumerate(rows):
            for i in range(n):
                w.ref.lens_now = lens[b]
                want = R.select(q[t].reshape(heads, group, hd), w.ref, w.table[b], lens[b] - n + i, top, first, recent)
                assert (got[t] == want).all(), f"top {top}: request {b}, row {i}"
                t += 1
        good = ~np.isnan(q).any((1, 2))
        out = w.cache.attention_selected(q, st, w.lens, w.table, got, hd ** -0.5)
        assert np.isnan(out[~good]).any(-1).sum() == (~good).sum()
        t = 0
        for b, n in enumerate(rows):                                      # (request 4's rows see a NaN key: its block is selected)
            if b != 4 and good[t: t + n].all() and n:
                one = World.__new__(World)
                one.__dict__.update(w.__dict__, lens=w.lens[b: b + 1], table=w.table[b: b + 1])
                one.check(out[t: t + n], q[t: t + n], [n], hd ** -0.5, only=lambda i, h: got[t + i, h])
            t += n


def test_equal_scores_take_the_earlier_blocks(ctx):
    bs, n = 16, 16 * 300
    w = World(ctx, [n], 1, 64, bs, seed=1, poison=False)
    row = w.keys(1)
    w.put(np.repeat(row, n, 0), np.ones((n, 1, 64), F), w.slots(0, np.arange(n)))
    w.cache.summarise([0, n], w.lens, w.table)
    q = w.q(1, 2)
    for top in (1, 2, 7, 64, 65, 255, 299):
        got = w.cache.select(q, [0, 1], w.lens, w.table, top, 0, 1)
        assert list(got[0, 0]) == list(range(top - 1)) + [299]


@pytest.mark.parametrize("hd,heads,group,bs,n,top", [(128, 2, 4, 64, 9000, 20), (64, 1, 2, 16, 20000, 100), (128, 1, 33, 16, 3000, 31)])
def test_selected_attention_over_long_contexts(ctx, hd, heads, group, bs, n, top):
    w = World(ctx, [n], heads, hd, bs, seed=2, poison=False)
    w.cache.summarise([0, n], w.lens, w.table)
    q = w.q(2, heads * group)
    sel = w.cache.select(q, [0, 2], w.lens, w.table, top, 1, 2)
    w.ref.lens_now = n
    for t in range(2):
        assert (sel[t] == R.select(q[t].reshape(heads, group, hd), w.ref, w.table[0], n - 2 + t, top, 1, 2)).all()
    got = w.cache.attention_selected(q, [0, 2], w.lens, w.table, sel, hd ** -0.5)
    w.check(got, q, [2], hd ** -0.5, only=lambda t, h: sel[t, h])
    full = w.cache.attention_selected(q, [0, 2], w.lens, w.table, np.tile(np.arange(-(-n // bs), dtype=np.int32), (2, heads, 1)), hd ** -0.5, 4.0)
    w.check(full, q, [2], hd ** -0.5, cap=4.0, what="all blocks")


@pytest.mark.parametrize("hd,heads,group,bs,rows,lens", [(64, 8, 1, 16, [150, 3, 0, 130], [420, 300, 40, 131]), (128, 4, 4, 16, [70, 1, 61], [500, 9, 61]), (80, 8, 3, 16, [40, 33], [90, 333]),
                                                       (256, 4, 8, 32, [66], [700]), (128, 8, 6, 16, [21, 0, 12], [220, 100, 500]), (64, 4, 2, 64, [200, 90], [2300, 91])])
def test_selection_for_prompts_is_exact(ctx, hd, heads, group, bs, rows, lens):
    """Enough rows a request that several of them share a workgroup; groups of rows across two requests' border."""
    w = World(ctx, lens, heads, hd, bs, seed=hd + group, spare=1)
    w.put(np.full((1, heads, hd), np.nan, F), np.ones((1, heads, hd), F), w.slots(0, [3 * bs + 1]))
    w.put(np.zeros((2 * bs, heads, hd), F), np.ones((2 * bs, heads, hd), F), w.slots(0, np.arange(bs, 3 * bs)))       # equal scores
    w.cache.summarise(np.concatenate([[0], np.cumsum(lens)]), w.lens, w.table)
    q = w.q(sum(rows), heads * group)
    q[5, 0], q[6] = np.nan, 0
    starts = np.concatenate([[0], np.cumsum(rows)])
    looked = sorted(set(w.rng.integers(0, sum(rows), 12)) | {0, 5, 6, 7, rows[0] - 1, min(rows[0], sum(rows) - 1), sum(rows) - 1})
    for top, first, recent in ((4, 1, 1), (9, 0, 3), (2, 0, 1), (3, 2, 1), (60, 2, 2)):
        got = w.cache.select(q, starts, w.lens, w.table, top, first, recent)
        for t in looked:
            b = int(np.searchsorted(starts, t, "right")) - 1
            w.ref.lens_now = lens[b]
            want = R.select(q[t].reshape(heads, group, hd), w.ref, w.table[b], lens[b] - rows[b] + t - starts[b], top, first, recent)
            assert (got[t] == want).all(), f"top {top}: row {t} of request {b}"


def test_selected_entries_that_break_the_rules_contribute_nothing(ctx):
    w = World(ctx, [100], 1, 64, 16, seed=8)
    q = w.q(1, 2)
    sel = ints([[[2, 2, 1, 4, -1, 6, 9, 2 ** 31 - 1]]])                    # again, not above, a gap, the own block, behind it
    n = C.c_size_t()
    ok(lib().pg_paged_kv4_selected_scratch(ctx.handle, w.cache._h, 2, 1, 8, C.byref(n)))
    d = [DevBuf(ctx, host=x) for x in (ints([0, 1]), w.lens, w.table, q, sel, np.zeros_like(q))]
    scratch = DevBuf(ctx, max(16, n.value))
    ok(lib().pg_paged_kv4_attention_selected_dev(ctx.handle, w.cache._h, d[3].ptr, 128, 64, 2, d[0].ptr, d[1].ptr, 1, 1, d[2].ptr, w.width, d[4].ptr, 8, 0.125, 0.0,
                                                 scratch.ptr, n.value, d[5].ptr))
    # an entry counts where it is above the one before it: 2, 4 (after 1), 6 (after -1)
    w.check(d[5].to_host(F).reshape(q.shape), q, [1], 0.125, only=lambda t, h: [2, 4, 6])


# ------------------------------------------------------------------------------------------------------ together
def test_a_server_runs_on_them(ctx):
    """Requests come, grow and go over a small pool: tables, append, summaries, attention and selection step by step against the
    reference that is told only what was granted."""
    from peregrine_amd import paged
    rng = np.random.default_rng(0)
    batch, nb, bs, width, heads, group, hd = 5, 14, 16, 12, 2, 3, 64   # a pool that does not hold every step
    t, c, ref = paged.BlockTables(batch, nb, bs, width, ctx), paged.PagedKV4Cache(nb, bs, heads, hd, ctx), R.Cache(nb, bs, heads, hd)
    refused = 0
    for step in range(14):
        new = np.where(t.lens == 0, rng.integers(0, 90, batch), rng.integers(0, 3, batch)).astype(np.int32)
        starts, granted, slots = t.extend(new, int(new.sum()) + 2)
        refused += int((granted == 0).sum())
        n = int(starts[-1])
        k, v, q = (rng.standard_normal((n + 2, h, hd)).astype(F) for h in (heads, heads, heads * group))
        c.append(k, v, slots)
        ref.append(k, v, slots)
        used = sorted(e for b in range(batch) for e in t.table[b, : -(-t.lens[b] // bs)])
        assert len(set(used)) == len(used) and len(used) + t.free_count[0] == nb
        rows = np.where(granted, new, 0)                                  # a request that got nothing is not run this step
        keep = np.concatenate([np.arange(starts[b], starts[b + 1]) for b in range(batch) if granted[b]] + [np.zeros(0, int)]).astype(int)
        st = np.concatenate([[0], np.cumsum(rows)])
        if not keep.size:
            t.release(t.lens > 0)
            continue
        c.summarise(st, t.lens, t.table)
        w = World.__new__(World)
        w.lens, w.heads, w.hd, w.bs, w.table, w.ref = t.lens, heads, hd, bs, t.table, ref
        w.check(c.attention(q[keep], st, t.lens, t.table, 0.125), q[keep], rows, 0.125, what=f"step {step}")
        sel = c.select(q[keep], st, t.lens, t.table, 3)
        w.check(c.attention_selected(q[keep], st, t.lens, t.table, sel, 0.125), q[keep], rows, 0.125, only=lambda i, h: sel[i, h], what=f"step {step}, selected")
        if step % 3 == 2:
            t.release(rng.random(batch) < 0.4)
    assert refused > 0


def test_a_step_replayed_from_a_graph(ctx):
    """A decoding step -- tables, append, summaries, attention, selection, attention over it -- captured once and replayed with other
    requests, eager work of the same kind in between: every replay is the eager step's bits."""
    from test_gpu_graph_replay import Hip
    from peregrine_amd import paged
    hip = Hip()
    batch, bs, heads, group, hd, nb, width, top = 6, 16, 2, 4, 128, 400, 64, 5
    rng = np.random.default_rng(2)
    c, ref_c = (paged.PagedKV4Cache(nb, bs, heads, hd, ctx) for _ in range(2))
    fill = rng.standard_normal((nb * bs, heads, hd)).astype(F)
    for x in (c, ref_c):
        x.append(fill, fill[::-1], np.arange(nb * bs))
    big = [rng.standard_normal((batch + 2, h, hd)).astype(F) for h in (heads, heads, heads * group)]
    ids = rng.permutation(nb).astype(np.int32)

    def make(cache):
        d = {n: DevBuf(ctx, host=x) for n, x in dict(lens=np.zeros(batch, np.int32), new=np.zeros(batch, np.int32), free=np.zeros(nb, np.int32), count=ints([0]),
                                                     table=np.zeros((batch, width), np.int32), lens2=np.zeros(batch, np.int32), count2=ints([0]), starts=np.zeros(batch + 1, np.int32),
                                                     granted=np.zeros(batch, np.int32), slots=np.zeros(batch + 2, np.int32), k=big[0], v=big[1], q=big[2],
                                                     sel=np.zeros((batch + 2, heads, top), np.int32), out=np.zeros_like(big[2]), out2=np.zeros_like(big[2])).items()}
        n1, n2 = C.c_size_t(), C.c_size_t()
        ok(lib().pg_paged_kv4_attention_scratch(ctx.handle, cache._h, heads * group, batch, 1, width, C.byref(n1)))
        ok(lib().pg_paged_kv4_selected_scratch(ctx.handle, cache._h, heads * group, batch + 2, top, C.byref(n2)))
        d["s1"], d["s2"] = DevBuf(ctx, max(16, n1.value)), DevBuf(ctx, max(16, n2.value))

        def step():
            L, h, p = lib(), ctx.handle, {n: x.ptr for n, x in d.items()}
            ok(L.pg_block_tables_extend_dev(h, p["lens"], p["new"], batch, bs, p["free"], p["count"], nb, p["table"], width, p["lens2"], p["count2"], p["starts"], p["granted"],
                                            p["slots"], batch + 2))
            ok(L.pg_paged_kv4_append_dev(h, cache._h, p["k"], p["v"], heads * hd, hd, batch + 2, p["slots"]))
            ok(L.pg_paged_kv4_summarise_dev(h, cache._h, p["starts"], p["lens2"], batch, batch + 2, p["table"], width))
            at = (heads * group * hd, hd, heads * group, p["starts"], p["lens2"], batch, batch + 2)
            ok(L.pg_paged_kv4_attention_dev(h, cache._h, p["q"], *at, 1, p["table"], width, 0.09, 1, 0, 0, 0.0, p["s1"], n1.value, p["out"]))
            ok(L.pg_paged_kv4_select_dev(h, cache._h, p["q"], *at, p["table"], width, top, 1, 1, p["sel"]))
            ok(L.pg_paged_kv4_attention_selected_dev(h, cache._h, p["q"], *at, p["table"], width, p["sel"], top, 0.09, 0.0, p["s2"], n2.value, p["out2"]))
        return d, step

    def put(d, seed):
        r = np.random.default_rng(seed)
        lens = r.integers(0, width * bs - 1, batch).astype(np.int32)
        need, at = -(-lens // bs), 0
        table = np.full((batch, width), -1, np.int32)
        for b in range(batch):
            table[b, :need[b]] = ids[at: at + need[b]]
            at += need[b]
        free = np.zeros(nb, np.int32)
        free[: nb - at] = ids[at:]
        new = r.integers(0, 2, batch).astype(np.int32)
        vals = dict(lens=lens, new=new, table=table, free=free, count=ints([nb - at]), k=r.standard_normal(big[0].shape).astype(F), v=r.standard_normal(big[1].shape).astype(F),
                    q=r.standard_normal(big[2].shape).astype(F), out=np.full(big[2].shape, 5, F), out2=np.full(big[2].shape, 6, F), sel=np.full((batch + 2, heads, top), -7, np.int32))
        for n, x in vals.items():
            ok(lib().pg_memcpy_h2d(ctx.handle, d[n].ptr, C.c_void_p(np.ascontiguousarray(x).ctypes.data), x.nbytes))

    def outputs(d):
        ctx.sync()
        return [d[n].to_host(np.uint32) for n in ("table", "lens2", "count2", "starts", "granted", "slots", "sel", "out", "out2")]

    (d, step), (e, eager) = make(c), make(ref_c)
    put(d, 100)
    step()
    put(e, 100)
    eager()
    ctx.sync()
    graph, ex = hip.capture(ctx.stream, step)
    try:
        for seed in range(5):
            put(e, seed)
            eager()
            want = outputs(e)
            put(d, seed)
            ctx.sync()
            hip.ok(hip.lib.hipGraphLaunch(ex, ctx.stream), "hipGraphLaunch")
            for a, b in zip(outputs(d), want):
                assert (a == b).all(), f"replay {seed}"
    finally:
        hip.lib.hipGraphExecDestroy(ex)
        hip.lib.hipGraphDestroy(graph)


def test_two_streams_read_one_cache_at_once(ctx):
    from peregrine_amd import Context
    w = World(ctx, [3000, 2500], 2, 128, 64, seed=12, poison=False)
    q = w.q(2, 8)
    with Context(0) as other:
        a, b = Step(ctx, w, q, [0, 1, 2]), Step(ctx, w, q, [0, 1, 2])
        a.attention()
        ctx.sync()
        want = a.result()
        for _ in range(20):
            a.attention()
            b.attention(ctx=other)
        ctx.sync()
        other.sync()
        assert (bits(a.result()) == bits(want)).all() and (bits(b.result()) == bits(want)).all()


def test_a_cache_may_outlive_the_work_of_its_context(ctx):
    """Freed on another context than the one it was made on."""
    from peregrine_amd import Context, paged
    c = paged.PagedKV4Cache(4, 16, 1, 64, ctx)
    x = np.ones((3, 1, 64), F)
    with Context(0) as other:
        c.append(x, x, [0, 1, 2])
        c.ctx = other
        c.append(2 * x, x, [3, 4, 5])
        k, _ = c.read([0, 3])
        assert (k[0] == 1).all() and (k[1] == 2).all()
        c.free()


@pytest.mark.parametrize("hd,heads,group,bs,lens,rows", [(128, 2, 4, 64, [700, 90], [300, 90]), (64, 1, 7, 16, [200, 33, 400], [200, 2, 101]), (256, 2, 1, 32, [500], [257]), (80, 1, 2, 128, [300], [130])])
def test_prompts_leave_out_what_is_no_block_and_read_nothing_behind(ctx, hd, heads, group, bs, lens, rows):
    """Pieces of prompts with every mask, with table entries that are no block in the middle of what they see; NaN rows behind
    the last token and in every block that is not theirs."""
    w = World(ctx, lens, heads, hd, bs, seed=hd + 1)
    q = w.q(sum(rows), heads * group)
    starts = np.concatenate([[0], np.cumsum(rows)])
    for m in (dict(), dict(mask=0), dict(mask=2, window=33, sinks=70), dict(mask=2, window=5, sinks=0), dict(cap=3.0)):
        s = Step(ctx, w, q, starts)
        s.attention(**m)
        w.check(s.result(), q, rows, hd ** -0.5, what=str(m), **m)
    table = w.table.copy()
    gone = [1, 2] if bs < 64 else [1]
    table[0, gone[0]], table[0, gone[-1]] = -1, w.nb + 3
    s = Step(ctx, w, q, starts, table=table)
    s.attention()
    got = s.result()
    one = World.__new__(World)
    one.__dict__.update(w.__dict__, lens=w.lens[:1], table=w.table[:1])
    one.check(got[: rows[0]], q[: rows[0]], rows[:1], hd ** -0.5, only=lambda t, h: [j for j in range(w.width) if j not in gone], what="no block")


@pytest.mark.parametrize("hd,heads,group", [(63, 2, 4), (125, 2, 4), (250, 1, 8), (64, 2, 8), (128, 1, 16), (256, 1, 4)])
def test_prompts_from_strided_queries_and_rows_before_the_first_token(ctx, hd, heads, group):
    """Queries that no vector load can take give the bits of packed ones; of a request with more rows than tokens the first see no
    key; rows beyond max_query, which is a bound on what is computed, and behind the last are left."""
    lens, rows, n = [90, 30], [80, 50], heads * group
    w = World(ctx, lens, heads, hd, 16, seed=hd)
    q = w.q(sum(rows) + 3, n)
    starts = [0, 80, 130]
    got = []
    for pad in (0, 1, 4):
        x = np.full((q.shape[0], n, hd + pad), np.nan, F)
        x[..., :hd] = q
        buf, s = DevBuf(ctx, host=x), Step(ctx, w, q, starts)
        s.attention(strides=(n * (hd + pad), hd + pad), q=buf.ptr)
        got.append(s.result())
    assert (bits(got[0]) == bits(got[1])).all() and (bits(got[0]) == bits(got[2])).all()
    seen = np.r_[0:80, 100:130]
    assert (got[0][80:100] == 0).all() and (got[0][130:] == 123).all()
    w.check(got[0][seen], q[seen], [80, 30], hd ** -0.5)
    s = Step(ctx, w, q, starts, max_query=60)
    s.attention()
    cut = s.result()
    assert (cut[60:80] == 123).all()
    w.check(cut[np.r_[100:130]], q[np.r_[100:130]], [0, 30], hd ** -0.5)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompts_replayed_from_a_graph(ctx, hd):
    """Pieces of prompts, and the choice of blocks for them, captured once; other queries and lengths at each replay."""
    from test_gpu_graph_replay import Hip
    hip, heads, group, bs, rows, top = Hip(), 2, 4, 16, [90, 170], 3
    w = World(ctx, [700, 400], heads, hd, bs, seed=hd, poison=False)
    w.cache.summarise([0, 700, 1100], w.lens, w.table)
    q = w.q(sum(rows), heads * group)
    s, e = (Step(ctx, w, q, [0, 90, 260]) for _ in range(2))
    sel = [DevBuf(ctx, host=np.zeros((sum(rows), heads, top), np.int32)) for _ in range(2)]

    def step(x, out):
        x.attention(mask=2, window=300, sinks=4)
        starts, lens, table, qd = x.d
        ok(lib().pg_paged_kv4_select_dev(ctx.handle, w.cache._h, qd.ptr, heads * group * hd, hd, heads * group, starts.ptr, lens.ptr, 2, sum(rows), table.ptr, x.width, top, 1, 1,
                                         out.ptr))

    step(s, sel[0])
    ctx.sync()
    graph, ex = hip.capture(ctx.stream, lambda: step(s, sel[0]))
    try:
        for i in range(4):
            lens, x = ints([700 - 100 * i, 400 - 70 * i]), w.q(sum(rows), heads * group)
            for y in (s, e):
                for b, a in ((y.d[1], lens), (y.d[3], x)):
                    ok(lib().pg_memcpy_h2d(ctx.handle, b.ptr, C.c_void_p(a.ctypes.data), a.nbytes))
            step(e, sel[1])
            ctx.sync()
            hip.ok(hip.lib.hipGraphLaunch(ex, ctx.stream), "hipGraphLaunch")
            ctx.sync()
            assert (bits(s.result()) == bits(e.result())).all() and (sel[0].to_host(np.int32) == sel[1].to_host(np.int32)).all(), f"replay {i}"
    finally:
        hip.lib.hipGraphExecDestroy(ex)
        hip.lib.hipGraphDestroy(graph)


def check_some(w, got, q, rows, scale, count, mask=1, window=0, sinks=0, cap=0.0, gone=()):
    """World.check on `count` rows and heads, the first and the last of each request among them; gone: (request, block) that are none."""
    starts, group, kv = np.concatenate([[0], np.cumsum(rows)]), q.shape[1] // w.heads, {}
    picks = [(int(t), int(j)) for t, j in zip(w.rng.integers(0, starts[-1], count), w.rng.integers(0, q.shape[1], count))]
    picks += [(int(t), 0) for b, n in enumerate(rows) if n for t in (starts[b], starts[b + 1] - 1)]
    off = size = 0.0
    for t, j in picks:
        b = int(np.searchsorted(starts, t, "right")) - 1
        if b not in kv:
            at = w.slots(b, np.arange(w.lens[b]))
            kv[b] = w.ref.f64(0, at), w.ref.f64(1, at)
        keys, pos = np.arange(w.lens[b]), w.lens[b] - rows[b] + t - starts[b]
        seen = np.ones(keys.size, bool) if mask == 0 else keys <= pos
        if mask == 2:
            seen &= (pos - keys <= window) | (keys < sinks)
        for x, block in gone:
            seen &= (x != b) | (keys // w.bs != block)
        want, bound = R.attend(q[t, j], kv[b][0][:, j // group], kv[b][1][:, j // group], scale, seen, cap)
        d = np.abs(got[t, j] - want)
        assert (d <= bound).all(), f"row {t}, head {j}: off by {d.max():.3g}, bound {bound.min():.3g}"
        off, size = off + (d ** 2).sum(), size + (want ** 2).sum()
    assert size == 0 or (off / size) ** 0.5 < 3e-6


def kernels_of(ctx, call):
    ctx.profile_begin()
    call()
    ctx.sync()
    return set(ctx.profile_end())


@pytest.mark.parametrize("hd,group,bs", [(40, 16, 16), (64, 12, 32), (100, 16, 16), (128, 16, 64), (200, 12, 16), (256, 16, 32)])
def test_prompts_of_many_requests(ctx, hd, group, bs):
    """Enough rows for the prompts' own kernels: every mask, requests of no rows and no tokens, blocks that are none, NaN in every
    slot that is not theirs and in a row that only some see."""
    heads, lens = 8, [90, 1, 0, 33, 64, 65, 17, 80, 48, 5, 77, 16, 31, 90, 2, 60, 70, 12, 88, 20]
    w = World(ctx, lens, heads, hd, bs, seed=hd)
    rows = [min(n, r) for n, r in zip(lens, [90, 1, 0, 20, 64, 30, 17, 79, 0, 5, 40, 16, 31, 1, 2, 60, 33, 12, 88, 20])]
    q = w.q(sum(rows), heads * group)
    starts = np.concatenate([[0], np.cumsum(rows)])
    own = "kv4_prompt_kernel" if hd > 128 else "kv4_prompt32_kernel"
    for m in (dict(), dict(mask=0), dict(mask=2, window=20, sinks=3), dict(mask=2, window=0, sinks=0), dict(cap=5.0)):
        s = Step(ctx, w, q, starts)
        assert own in kernels_of(ctx, lambda: s.attention(**m))
        check_some(w, s.result(), q, rows, hd ** -0.5, 250, **m)
    gone = [(0, 1), (4, 0), (15, 60 // bs if bs < 64 else 0)]
    table = w.table.copy()
    for i, (b, j) in enumerate(gone):
        table[b, j] = (-1, w.nb, 2 ** 31 - 1)[i]
    s = Step(ctx, w, q, starts, table=table)
    s.attention()
    got = s.result()
    check_some(w, got, q, rows, hd ** -0.5, 250, gone=gone)
    assert np.isfinite(got).all()
    w.put(w.keys(1), np.full((1, heads, hd), np.nan, F), w.slots(0, [50]))
    s = Step(ctx, w, q, starts)
    s.attention()
    nan = np.isnan(s.result()).all((1, 2))
    assert (nan == ((np.arange(len(q)) >= 50) & (np.arange(len(q)) < 90))).all() and np.isfinite(s.result()[~nan]).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_long_prompt_divided_between_workgroups(ctx, hd):
    heads, group, n, rows = 4, 4, 8100, 2048
    w = World(ctx, [n], heads, hd, 64, seed=hd, poison=False)
    q = w.q(rows, heads * group)
    own = "kv4_prompt_kernel" if hd > 128 else "kv4_prompt32_kernel"
    for m in (dict(), dict(cap=20.0)):
        s = Step(ctx, w, q, [0, rows])
        assert kernels_of(ctx, lambda: s.attention(**m)) == {own, "kv4_join_kernel"}
        check_some(w, s.result(), q, [rows], hd ** -0.5, 40, **m)


def test_cpp_host_mirror():
    """tests/cpp/paged_kv4.cpp over the C++ mirror's namespace paged; built by __graft_entry__.build()."""
    import os
    import subprocess
    binary = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "paged_kv4")
    r = subprocess.run([binary], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "OK: all checks passed" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
