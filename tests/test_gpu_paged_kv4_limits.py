"""The paged 4-bit cache and the block tables on the GPU at the ends of what they take: cut slot maps, entries that are no block,
rows whose sums are far apart."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from devbuf import DevBuf
from test_gpu_paged_kv4 import F, Step, World, bits, check_some, extend_ref, ints, kernels_of, lib, ok

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("batch,most_new,in_place", [(30, 900, False), (30, 900, True), (4097, 6, False), (4097, 6, True)])
def test_a_slot_map_that_is_too_short_keeps_the_first_rows(ctx, batch, most_new, in_place):
    """Over several workgroups and in a launch of its own, as over one: a request that the cut goes through keeps its first rows' slots."""
    rng = np.random.default_rng(batch + in_place)
    bs = 16
    lens, add = rng.integers(0, 200, batch).astype(np.int32), rng.integers(0, most_new + 1, batch).astype(np.int32)
    add[::7] -= 9                                                         # some are negative: they count as 0
    width = -(-(200 + most_new) // bs)
    have, more = -(-lens // bs), add.clip(0)
    need = int((-(-(lens + more) // bs) - have).sum())
    nb = int(have.sum()) + need
    ids = rng.permutation(nb).astype(np.int32)
    table = np.full((batch, width), -1, np.int32)
    for b, at in enumerate(np.cumsum(have) - have):
        table[b, :have[b]] = ids[at: at + have[b]]
    free = np.zeros(nb, np.int32)
    free[:need] = ids[have.sum():]
    ends = np.cumsum(more)
    middle = int(np.searchsorted(ends, 0.7 * ends[-1]))
    middle += int(np.argmax(more[middle:] > 1))                           # a request of two rows and more
    for tokens in (int(ends[middle]) - 1, int(ends[middle]), int(ends[middle]) - int(more[middle]) + 1):
        assert 4096 < tokens < ends[-1]
        want = extend_ref(lens, add, bs, width, table, free, need, tokens)
        d = [DevBuf(ctx, host=x) for x in (lens, add, free, ints([need]), table, np.zeros(batch + 1, np.int32), np.zeros(batch, np.int32), np.full(tokens + 2, 77, np.int32))]
        lens_out, count_out = (d[0], d[3]) if in_place else (DevBuf(ctx, host=np.full(batch, 77, np.int32)), DevBuf(ctx, host=ints([77])))
        ok(lib().pg_block_tables_extend_dev(ctx.handle, d[0].ptr, d[1].ptr, batch, bs, d[2].ptr, d[3].ptr, nb, d[4].ptr, width, lens_out.ptr, count_out.ptr, d[5].ptr, d[6].ptr,
                                            d[7].ptr, tokens))
        slots = d[7].to_host(np.int32)
        got = [d[4].to_host(np.int32).reshape(batch, width), lens_out.to_host(np.int32), count_out.to_host(np.int32)[0], d[5].to_host(np.int32), d[6].to_host(np.int32), slots[:-2]]
        for g, w in zip(got, want):
            assert (np.asarray(g) == np.asarray(w)).all()
        assert (slots[-2:] == 77).all()


# ------------------------------------------------------------------------------------------------------ entries that are no block
def test_slots_of_entries_that_are_no_block_are_none(ctx):
    """Old entries of a table and entries of the free list that name no block: -1 for their rows, and no slot of another block."""
    bs, nb, width = 16, 40, 700
    bad = ints([-1, nb, 1 << 27, 1 << 28, (1 << 28) + 3, 2 ** 31 - 1, -2 ** 31, -2 ** 31 + 5])
    for batch, tokens in ((8, 300), (8, 6000), (4097, 6000)):
        lens, add = np.full(batch, 2 * bs - 3, np.int32), np.full(batch, 1, np.int32)
        add[:8] = 5                                                       # three rows in the old block, two in a new one
        table = np.full((batch, width), 7, np.int32)
        table[:8, 1] = bad
        free, count = np.concatenate([bad, ints([1, 2])])[::-1].copy(), 10
        with np.errstate(over="ignore"):                                  # (the reference's slots of such entries, replaced below)
            want = extend_ref(lens, add, bs, width, table, free, count, tokens)
        slots = want[5].reshape(-1).astype(np.int64)
        for r in range(8):
            slots[5 * r: 5 * r + 3] = -1
            e = int(want[0][r, 2])
            slots[5 * r + 3: 5 * r + 5] = [16 * e, 16 * e + 1] if 0 <= e < nb else -1
        for in_place in (False, True):
            d = [DevBuf(ctx, host=x) for x in (lens, add, free, ints([count]), table, np.zeros(batch + 1, np.int32), np.zeros(batch, np.int32), np.full(tokens, 77, np.int32))]
            lens_out, count_out = (d[0], d[3]) if in_place else (DevBuf(ctx, host=lens), DevBuf(ctx, host=ints([0])))
            ok(lib().pg_block_tables_extend_dev(ctx.handle, d[0].ptr, d[1].ptr, batch, bs, d[2].ptr, d[3].ptr, nb, d[4].ptr, width, lens_out.ptr, count_out.ptr, d[5].ptr,
                                                d[6].ptr, d[7].ptr, tokens))
            assert (d[4].to_host(np.int32).reshape(batch, width) == want[0]).all()
            assert (d[7].to_host(np.int32) == slots).all(), (batch, tokens, in_place)


# ------------------------------------------------------------------------------------------------------ rows far apart
# hd, key heads, group, rows, tokens, kernels: every kernel of attention, its keys in one run and divided.
FEW, ROWS, P32, P256, JOIN = "kv4_few_kernel", "kv4_rows_kernel", "kv4_prompt32_kernel", "kv4_prompt_kernel", "kv4_join_kernel"
SHORT = [(64, 1, 4, 1, 600, {FEW}), (128, 2, 3, 1, 600, {FEW}), (256, 1, 4, 1, 450, {FEW}), (64, 1, 8, 1, 600, {FEW}), (100, 1, 4, 2, 600, {FEW}), (256, 1, 6, 1, 450, {FEW}),
         (64, 1, 16, 1, 600, {ROWS}), (128, 1, 4, 5, 600, {ROWS}), (256, 2, 16, 1, 450, {ROWS})]
LONG = [(128, 1, 4, 1, 5000, {FEW, JOIN}), (64, 2, 8, 1, 5000, {FEW, JOIN}), (256, 1, 3, 1, 3000, {FEW, JOIN}), (128, 1, 16, 1, 5000, {ROWS, JOIN}), (200, 1, 4, 5, 3000, {ROWS, JOIN})]
PROMPTS = [(64, 8, 16, 400, 600, {P32}), (100, 8, 16, 400, 600, {P32}), (128, 8, 16, 400, 600, {P32}), (250, 8, 16, 400, 600, {P256})]
DIVIDED = [(128, 4, 4, 2048, 8100, {P32, JOIN}), (256, 4, 4, 2048, 8100, {P256, JOIN})]


def one_request(ctx, hd, heads, group, rows, n, seed=0):
    w = World(ctx, [n], heads, hd, 16 if n < 1000 else 64, seed=hd + group + seed, poison=False)
    return w, w.q(rows, heads * group)


@pytest.mark.parametrize("hd,heads,group,rows,n,kernels", SHORT + LONG + PROMPTS[2:] + DIVIDED)
def test_what_is_not_finite_is_not_lost_beside_a_key_of_all_the_weight(ctx, hd, heads, group, rows, n, kernels):
    """A NaN key or value reaches every row that sees it, also where another key is so far above it that its weight is 0 in f32, in
    whichever of a row's tiles and runs the two lie."""
    w, q = one_request(ctx, hd, heads, group, rows, n)
    q[:] = 8
    zero, loud = np.zeros((1, heads, hd), F), np.full((1, heads, hd), 4, F)     # scores of 0 and of 32 sqrt(hd): 256 and more
    keys, values = np.zeros((n, heads, hd), F), w.rng.standard_normal((n, heads, hd)).astype(F)
    w.put(keys, values, w.slots(0, np.arange(n)))
    nan = np.full((1, heads, hd), np.nan, F)
    first = n - rows                                                      # the first row's own token
    s = Step(ctx, w, q, [0, rows])
    for at in (5, first):
        w.put(loud, values[[at]], w.slots(0, [at]))
        for p in [1, 130, first - 1, n - 1] if rows > 100 else [1, 70, 130, 200, 290, n // 2, n // 2 + 70, first - 1, n - 1]:
            if p == at:
                continue
            for k, v in ((zero, nan), (nan, values[[p]])):
                w.put(k, v, w.slots(0, [p]))
                assert kernels_of(ctx, s.attention) == kernels
                got = s.result()
                sees = first + np.arange(rows) >= p
                assert np.isnan(got[sees]).all(), f"loud at {at}, NaN at {p}: {np.isfinite(got[sees]).any(-1).sum()} rows lost it"
                assert np.isfinite(got[~sees]).all()
            w.put(zero, values[[p]], w.slots(0, [p]))
        w.put(zero, values[[at]], w.slots(0, [at]))


def test_what_is_not_finite_is_not_lost_in_selected_blocks(ctx):
    for hd, group, n in ((128, 4, 5000), (64, 16, 5000), (128, 8, 500)):
        w, q = one_request(ctx, hd, 1, group, 1, n)
        q[:] = 8
        keys, values = np.zeros((n, 1, hd), F), w.rng.standard_normal((n, 1, hd)).astype(F)
        keys[9] = 4
        w.put(keys, values, w.slots(0, np.arange(n)))
        sel = np.arange(-(-n // w.bs), dtype=np.int32)[None, None]
        assert np.isfinite(w.cache.attention_selected(q, [0, 1], w.lens, w.table, sel, hd ** -0.5)).all()
        for p in (0, 140, n // 2, n - 1):
            w.put(keys[[p]], np.full((1, 1, hd), np.nan, F), w.slots(0, [p]))
            assert np.isnan(w.cache.attention_selected(q, [0, 1], w.lens, w.table, sel, hd ** -0.5)).all(), p
            w.put(keys[[p]], values[[p]], w.slots(0, [p]))


def run(ctx, w, q, kernels, **m):
    s = Step(ctx, w, q, [0, len(q)])
    assert kernels_of(ctx, lambda: s.attention(**m)) == kernels
    return s.result()


def attend_by_weight(q, k, v, scale, seen):
    """R.attend's value, and a bound in which a value row counts by its weight: p d is two f16, 2^-21 of it and an end of at most
    2^-25 where the largest p d that the row has seen so far is scaled to 2^9 at least, so 2^-34 of that, times |n - 7.5| <= 7.5: with
    7.5 d at most 1.02 of the value row's largest, 2^-33 of the largest p |v| for each of N keys.  All else as there."""
    want, _ = R.attend(q, k, v, scale, seen)
    k, v, q = k[seen], v[seen], q.astype(np.float64)
    s = k @ q * scale
    size = np.abs(scale) * (np.abs(k) @ np.abs(q) + 2 * np.abs(k).max(1) * np.abs(q).sum())
    m = s.max()
    err = np.abs(scale) * np.abs(q).max() / (127 * 65536) * np.abs(k).sum(1) + 2.0 ** -24 * (8 * size + 2 * (np.abs(s) + abs(m)) / np.log(2)) + 2.0 ** -22
    p = np.exp(s - m)
    p /= p.sum()
    each = p * np.abs(v).max(1)
    return want, 2 * ((err + 2.0 ** -21 + (len(p) + 64) * 2.0 ** -24) * each).sum() + 2.0 ** -33 * len(p) * each.max()


def check_by_weight(w, got, q, rows, scale, count):
    at = w.slots(0, np.arange(w.lens[0]))
    k, v, group, first = w.ref.f64(0, at), w.ref.f64(1, at), q.shape[1] // w.heads, w.lens[0] - rows
    picks = [(t, j) for t in range(rows) for j in range(q.shape[1])]
    if len(picks) > count:
        picks = [picks[i] for i in w.rng.permutation(len(picks))[:count]] + [(0, 0), (rows - 1, q.shape[1] - 1)]
    off = size = 0.0
    for t, j in picks:
        h = j // group
        want, bound = attend_by_weight(q[t, j], k[:, h], v[:, h], scale, np.arange(w.lens[0]) <= first + t)
        d = np.abs(got[t, j] - want)
        assert (d <= bound).all(), f"row {t}, head {j}: off by {d.max():.3g}, bound {bound:.3g}"
        off, size = off + (d ** 2).sum(), size + (want ** 2).sum()
    assert (off / size) ** 0.5 < 3e-6, f"2-norm off by {(off / size) ** 0.5:.3g}"


@pytest.mark.parametrize("hd,heads,group,rows,n,kernels", SHORT + LONG[:4] + PROMPTS + DIVIDED)
def test_large_values_of_no_weight_take_no_bits(ctx, hd, heads, group, rows, n, kernels):
    """Values far larger than the others' on keys whose weight is next to none: alone, in every fourth tile, in all that come first."""
    w, q = one_request(ctx, hd, heads, group, rows, n, seed=1)
    q[:] = 1 + 0.1 * w.rng.standard_normal(q.shape)
    at = np.arange(n)
    for which, gap, ratio in ((at == 0, 60, 2.0 ** 20), (at < n // 4, 60, 2.0 ** 20), (at % 256 < 64, 90, 2.0 ** 60), (at == 300, 200, 2.0 ** 110)):
        k = (0.3 * w.rng.standard_normal((n, heads, hd))).astype(F)
        v = w.rng.standard_normal((n, heads, hd)).astype(F)
        k[which] -= F(gap / hd ** 0.5)
        v[which] *= F(ratio)
        w.put(k, v, w.slots(0, at))
        check_by_weight(w, run(ctx, w, q, kernels), q, rows, hd ** -0.5, 40)


@pytest.mark.parametrize("hd,heads,group,rows,n,kernels", SHORT + LONG + PROMPTS + DIVIDED[:1])
def test_large_constant_values_under_rising_scores(ctx, hd, heads, group, rows, n, kernels):
    """Value rows of one number, whose steps are 0, and scores that rise by 60 behind the first tiles: the sums of p z stay finite."""
    w, q = one_request(ctx, hd, heads, group, rows, n, seed=2)
    q[:] = 1
    k, v = np.zeros((n, heads, hd), F), np.full((n, heads, hd), 2.0 ** 85, F)
    k[min(300, n - rows):] = F(60 / hd ** 0.5)
    for sign in (1, -1):
        w.put(k, sign * v, w.slots(0, np.arange(n)))
        got = run(ctx, w, q, kernels)
        # p's error is common to the sums of p z and of p; each is of n + 64 roundings
        assert np.abs(got / (sign * 2.0 ** 85) - 1).max() <= 2 * (n + 64) * 2.0 ** -24


@pytest.mark.parametrize("hd,heads,group,rows,n,kernels", [SHORT[0], SHORT[1], SHORT[3], SHORT[6], SHORT[7], SHORT[8]] + PROMPTS)
def test_queries_of_the_largest_numbers(ctx, hd, heads, group, rows, n, kernels):
    """Rows whose largest is 2^127 and more, over keys near the smallest: ordinary scores, the same on every kernel."""
    w, q = one_request(ctx, hd, heads, group, rows, n, seed=3)
    q *= F(1e36)
    q[..., 3] = F(2e38) * np.where(np.arange(heads * group) % 2, 1, -1)
    k = (1.5e-37 * w.rng.standard_normal((n, heads, hd))).astype(F)
    w.put(k, w.rng.standard_normal((n, heads, hd)).astype(F), w.slots(0, np.arange(n)))
    check_some(w, run(ctx, w, q, kernels), q, [rows], hd ** -0.5, 60)


# ------------------------------------------------------------------------------------------------------ refused requests
def test_rows_of_a_refused_request_change_nothing_for_the_others(ctx):
    """What pg_block_tables_extend_dev refuses keeps its rows in the packed step: they are not stored, they get what rows at the end of
    the request's old tokens get (0 before its first), and the other requests' rows, blocks and summaries are as without them."""
    heads, group, hd, bs, top = 2, 4, 64, 16, 3
    w = World(ctx, [40, 70, 3, 90], heads, hd, bs, seed=2, spare=8)
    w.cache.summarise([0, 40, 110, 113, 203], w.lens, w.table)
    rows, n = [4, 12, 30, 2], 48                                          # the middle ones need a block, and there is none
    used = set(w.table[w.table >= 0])
    free = ints([b for b in range(w.nb) if b not in used] + [0] * len(used))
    new_table = np.concatenate([w.table, np.full((4, 2), -1, np.int32)], 1)
    d = [DevBuf(ctx, host=x) for x in (w.lens, ints(rows), free, ints([0]), new_table, np.zeros(4, np.int32), ints([0]), np.zeros(5, np.int32), np.zeros(4, np.int32),
                                       np.zeros(n, np.int32))]
    ok(lib().pg_block_tables_extend_dev(ctx.handle, d[0].ptr, d[1].ptr, 4, bs, d[2].ptr, d[3].ptr, w.nb, d[4].ptr, w.width + 2, d[5].ptr, d[6].ptr, d[7].ptr, d[8].ptr, d[9].ptr, n))
    lens, starts, granted, slots = (d[i].to_host(np.int32) for i in (5, 7, 8, 9))
    assert list(granted) == [1, 0, 0, 1] and list(lens) == [44, 70, 3, 92] and (slots[4:46] == -1).all() and (slots[:4] >= 0).all()
    k, v, q = w.keys(n), w.rng.standard_normal((n, heads, hd)).astype(F), w.q(n, heads * group)
    before = [x[slots_of] for x in w.cache.read(np.arange(w.nb * bs)) for slots_of in [w.slots(1, np.arange(70))]]
    w.put(k, v, slots)
    table = d[4].to_host(np.int32).reshape(4, -1)

    def step(starts, lens, table, q):
        """(outputs, chosen blocks, outputs over them, summaries of every block) of the step's `_dev` calls."""
        s, sel = Step(ctx, w, q, starts, lens=lens, table=table), DevBuf(ctx, host=np.full((len(q), heads, top), -9, np.int32))
        at, h, c = (heads * group * hd, hd, heads * group, s.d[0].ptr, s.d[1].ptr, s.batch, len(q)), ctx.handle, w.cache._h
        ok(lib().pg_paged_kv4_summarise_dev(h, c, s.d[0].ptr, s.d[1].ptr, s.batch, len(q), s.d[2].ptr, s.width))
        s.attention()
        out = s.result()
        ok(lib().pg_paged_kv4_select_dev(h, c, s.d[3].ptr, *at, s.d[2].ptr, s.width, top, 1, 1, sel.ptr))
        size = C.c_size_t()
        ok(lib().pg_paged_kv4_selected_scratch(h, c, heads * group, len(q), top, C.byref(size)))
        scratch, sums = DevBuf(ctx, max(16, size.value)), [DevBuf(ctx, host=np.zeros((w.nb, heads, hd), F)) for _ in range(2)]
        ok(lib().pg_paged_kv4_attention_selected_dev(h, c, s.d[3].ptr, *at, s.d[2].ptr, s.width, sel.ptr, top, hd ** -0.5, 0.0, scratch.ptr, size.value, s.out.ptr))
        every = DevBuf(ctx, host=np.arange(w.nb, dtype=np.int32))
        ok(lib().pg_paged_kv4_read_summaries_dev(h, c, every.ptr, w.nb, sums[0].ptr, sums[1].ptr))
        return out, sel.to_host(np.int32).reshape(len(q), heads, top), s.result(), [x.to_host(np.uint32) for x in sums]

    keep = np.r_[0:4, 46:48]
    alone = step([0, 4, 6], lens[[0, 3]], table[[0, 3]], q[keep])
    whole = step(starts, lens, table, q)
    for a, b in zip(alone[:3], whole[:3]):
        assert (np.asarray(a).view(np.uint32) == np.asarray(b)[keep].view(np.uint32)).all()
    assert all((a == b).all() for a, b in zip(alone[3], whole[3]))
    for a, b in zip(before, w.cache.read(w.slots(1, np.arange(70)))):
        assert (bits(a) == bits(b)).all()
    w.lens, w.table = lens, table
    old = World.__new__(World)
    old.__dict__.update(w.__dict__, lens=lens[1:2], table=table[1:2])
    for out in (whole[0], whole[2]):
        assert np.isfinite(out).all() and (out[16:43] == 0).all()         # 30 rows over 3 tokens: 27 are before the first
    old.check(whole[0][4:16], q[4:16], [12], hd ** -0.5)


# ------------------------------------------------------------------------------------------------------ prompts' own kernels
@pytest.mark.parametrize("hd", [40, 63, 64, 100, 125, 128, 200, 250, 256])
def test_own_kernels_of_prompts_take_strided_queries_and_leave_rows_behind(ctx, hd):
    """test_prompts_from_strided_queries_and_rows_before_the_first_token with rows enough for the prompts' own kernels."""
    heads, group, lens, rows = 8, 16, [500, 60], [420, 100]
    own, n = P256 if hd > 128 else P32, heads * group
    w = World(ctx, lens, heads, hd, 16, seed=hd)
    q = w.q(sum(rows) + 3, n)
    starts, got = [0, 420, 520], []
    for pad in (0, 1, 4):
        x = np.full((q.shape[0], n, hd + pad), np.nan, F)
        x[..., :hd] = q
        buf, s = DevBuf(ctx, host=x), Step(ctx, w, q, starts)
        assert kernels_of(ctx, lambda: s.attention(strides=(n * (hd + pad), hd + pad), q=buf.ptr)) == {own}
        got.append(s.result())
    assert (bits(got[0]) == bits(got[1])).all() and (bits(got[0]) == bits(got[2])).all()
    seen = np.r_[0:420, 460:520]
    assert (got[0][420:460] == 0).all() and (got[0][520:] == 123).all()
    check_some(w, got[0][seen], q[seen], [420, 60], hd ** -0.5, 100)
    s = Step(ctx, w, q, starts, max_query=390)
    assert kernels_of(ctx, s.attention) == {own}
    cut = s.result()
    assert (cut[390:420] == 123).all() and (bits(cut[:390]) == bits(got[0][:390])).all() and (bits(cut[420:]) == bits(got[0][420:])).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_own_kernels_of_prompts_near_the_smallest_values(ctx, hd):
    n, rows, heads, group = 500, 400, 8, 16
    w, q = one_request(ctx, hd, heads, group, rows, n)
    for top in (1e-35, 2e-34):
        v = (w.rng.standard_normal((n, heads, hd)) * np.exp(w.rng.uniform(-3, 0, (n, heads, 1))) * top / 3).astype(F)
        v[:70], v[100] = 0, 0
        w.put(w.keys(n), v, w.slots(0, np.arange(n)))
        check_some(w, run(ctx, w, q, {P256 if hd > 128 else P32}), q, [rows], hd ** -0.5, 60)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_own_kernels_of_prompts_replayed_from_a_graph(ctx, hd):
    """Captured once; other queries, lengths and tables at each replay, eager work of the same kind between."""
    from test_gpu_graph_replay import Hip
    hip, heads, group, rows = Hip(), 8, 16, [300, 120]
    w = World(ctx, [700, 400], heads, hd, 16, seed=hd, poison=False)
    q = w.q(sum(rows), heads * group)
    s, e = (Step(ctx, w, q, [0, 300, 420]) for _ in range(2))
    own, m = P256 if hd > 128 else P32, dict(mask=2, window=300, sinks=4)
    assert kernels_of(ctx, lambda: s.attention(**m)) == {own}
    ctx.sync()
    graph, ex = hip.capture(ctx.stream, lambda: s.attention(**m))
    try:
        for i in range(4):
            lens, x = ints([700 - 100 * i, 400 - 70 * i]), w.q(sum(rows), heads * group)
            table = w.table if i % 2 == 0 else np.where(w.table >= 0, w.rng.permutation(w.nb).astype(np.int32)[w.table], -1).astype(np.int32)
            for y in (s, e):
                for b, a in ((y.d[1], lens), (y.d[2], table), (y.d[3], x)):
                    ok(lib().pg_memcpy_h2d(ctx.handle, b.ptr, C.c_void_p(a.ctypes.data), a.nbytes))
            e.attention(**m)
            ctx.sync()
            hip.ok(hip.lib.hipGraphLaunch(ex, ctx.stream), "hipGraphLaunch")
            ctx.sync()
            assert (bits(s.result()) == bits(e.result())).all(), f"replay {i}"
            if i == 0:
                check_some(w, s.result(), x, rows, hd ** -0.5, 60, **m)
    finally:
        hip.lib.hipGraphExecDestroy(ex)
        hip.lib.hipGraphDestroy(graph)


@pytest.mark.parametrize("hd,heads,group,rows,n,kernels", [(128, 2, 4, 1, 5000, {FEW, JOIN}), (64, 2, 2, 3, 5000, {FEW, JOIN}), (256, 1, 7, 1, 5000, {FEW, JOIN}),
                                                           (128, 2, 4, 9, 5000, {ROWS, JOIN}), (64, 1, 16, 3, 5000, {ROWS, JOIN}), (256, 1, 4, 4, 5000, {ROWS, JOIN})] + DIVIDED)
def test_windows_with_sinks_over_divided_keys(ctx, hd, heads, group, rows, n, kernels):
    """Sinks and window cut by the borders of the runs, runs in which some rows or all see nothing."""
    w, q = one_request(ctx, hd, heads, group, rows, n, seed=4)
    for m in (dict(window=2000, sinks=4), dict(window=3000, sinks=700), dict(window=2000, sinks=700, cap=5.0), dict(window=3000, sinks=0)):
        check_some(w, run(ctx, w, q, kernels, mask=2, **m), q, [rows], hd ** -0.5, 24, mask=2, **m)


# ------------------------------------------------------------------------------------------------------ chosen blocks
@pytest.mark.parametrize("hd,group", [(64, 4), (128, 8), (64, 16), (256, 3), (256, 16)])
def test_chosen_entries_count_wherever_they_stand_in_the_list(ctx, hd, group):
    """Entries that contribute nothing ahead of ones that do, in contexts of fewer blocks than the list has entries."""
    w = World(ctx, [40, 40, 20, 300, 40], 1, hd, 16, seed=hd + group)
    lists = [[-1, 0, 1, 2, -1, -1], [7, -1, 0, -1, 1, 2], [-1, -1, -1, -1, 0, 1], [-1, 3, 5, -1, 8, 18], [5, -1, -1, -1, -1, 1]]
    blocks = [[0, 1, 2], [0, 1, 2], [0, 1], [3, 5, 8, 18], [1]]
    q, top = w.q(5, group), 70
    sel = np.full((5, 1, top), -1, np.int32)
    for t, x in enumerate(lists):
        sel[t, 0, :len(x) - 1], sel[t, 0, top - 1 - t] = x[:-1], x[-1]       # the last one far behind the others
    n = C.c_size_t()
    ok(lib().pg_paged_kv4_selected_scratch(ctx.handle, w.cache._h, group, 5, top, C.byref(n)))
    d = [DevBuf(ctx, host=x) for x in (np.arange(6, dtype=np.int32), w.lens, w.table, q, sel, np.zeros_like(q))]
    scratch = DevBuf(ctx, max(16, n.value))
    ok(lib().pg_paged_kv4_attention_selected_dev(ctx.handle, w.cache._h, d[3].ptr, group * hd, hd, group, d[0].ptr, d[1].ptr, 5, 5, d[2].ptr, w.width, d[4].ptr, top, hd ** -0.5,
                                                 0.0, scratch.ptr, n.value, d[5].ptr))
    w.check(d[5].to_host(F).reshape(q.shape), q, [1] * 5, hd ** -0.5, only=lambda t, h: blocks[t])


@pytest.mark.parametrize("batch", [40, 1030, 2050])
def test_release_of_more_blocks_than_there_are_fills_the_list_and_no_more(ctx, batch):
    """The same blocks in many tables: the first that fit go onto the list, in order, and nothing is written behind it."""
    nb, width = 50, 7
    table = np.arange(batch * width, dtype=np.int32).reshape(batch, width) % nb
    table[::3, 2] = -1
    lens, free = np.full(batch, 16 * width, np.int32), np.full(nb + 4, 77, np.int32)
    d = [DevBuf(ctx, host=x) for x in (np.ones(batch, np.int32), lens, table, free, ints([5]))]
    ok(lib().pg_block_tables_release_dev(ctx.handle, d[0].ptr, d[1].ptr, batch, 16, d[2].ptr, width, d[3].ptr, d[4].ptr, nb))
    got = d[3].to_host(np.int32)
    given = table.reshape(-1)[table.reshape(-1) >= 0][: nb - 5]
    assert (got[:5] == 77).all() and (got[5:nb] == given).all() and (got[nb:] == 77).all() and d[4].to_host(np.int32)[0] == nb
    assert (d[1].to_host(np.int32) == 0).all() and (d[2].to_host(np.int32) == -1).all()


def test_windows_of_more_than_two_to_the_thirty_tokens(ctx):
    """A context of that length, all but a few of its blocks none: a window that reaches its first tokens shows them."""
    hd, group, bs, far = 64, 4, 256, 1 << 30
    n = far + 300
    w = World(ctx, [600], 1, hd, bs, seed=1, poison=False)               # three blocks: the first, the second and the last of the context
    table = np.full((1, -(-n // bs)), -1, np.int32)
    table[0, :2], table[0, -1] = w.table[0, :2], w.table[0, 2]
    q = w.q(1, group)
    keys = np.concatenate([np.arange(2 * bs), np.arange(n // bs * bs, n)])    # positions that have a block
    at = R.slots_of(table[0], keys, bs)
    w.put(w.keys(len(at)), w.rng.standard_normal((len(at), 1, hd)).astype(F), at.astype(np.int32))
    k, v = w.ref.f64(0, at), w.ref.f64(1, at)
    for window in (far + 100, far + 299, far - 1, (1 << 31) - 1, 1 << 40):
        s = Step(ctx, w, q, [0, 1], lens=ints([n]), table=table)
        s.attention(mask=2, window=window)
        got = s.result()
        for j in range(group):
            want, bound = R.attend(q[0, j], k[:, 0], v[:, 0], hd ** -0.5, n - 1 - keys <= window)
            assert (np.abs(got[0, j] - want) <= bound).all(), window
