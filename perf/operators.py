"""A key/value cache that many requests share, held in 4 bits: the block tables that are made for a step's requests, the
append of a step's keys and values, attention that reads the 4-bit rows (single tokens, a few tokens, prompts), and
attention over the blocks that a cheap score selects for each query.

A row is one head of one token, for keys and for values.  It is kept as codes n of 0 .. 15 with a centre z and a step d, both
bfloat16: value = z + d * (n - 7.5).  Blocks hold `block` tokens; a request's block table names its blocks in order.

Every case is one pass of a server's step through one of these operators.  `own` False: the plain form, in elementary torch
operations; True: the framework's calls.
"""
import ctypes as C
import math

import torch

own = False

DEVICE = "cuda"
INT8_MOST = 127.0


# ------------------------------------------------------------------------------------------------------------ inputs
def _lens(n, most, ragged):
    """Lengths of n requests, the first `most`, the others spread over a quarter of it and up; all alike if not ragged."""
    if not ragged:
        return [most] * n
    return [most] + [max(1, int(most * (0.25 + 0.75 * ((b * 0.6180339887) % 1.0)))) for b in range(1, n)]


def _shape(case):
    """(lengths, new rows) of each request, on the host: lengths count the new rows."""
    lens = _lens(case["batch"], case["most"], case["ragged"])
    rows = [min(r, n) for r, n in zip(_lens(case["batch"], case["rows"], case["ragged"]), lens)]
    return lens, rows


def _width(case):
    return -(-case["most"] // case["block"])


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _tables(lens, block, g, spare=0):
    """Block tables over a shuffled pool: (table [batch, width], blocks in the pool); -1 behind a request's last block."""
    need = torch.tensor([-(-n // block) for n in lens])
    total, width = int(need.sum()) + spare, int(need.max())
    order = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)
    at = torch.arange(width)[None, :]
    first = (need.cumsum(0) - need)[:, None]
    index = torch.where(at < need[:, None], first + at, -1).to(DEVICE)
    return torch.where(index >= 0, order[index.clamp_min(0)], torch.full_like(order[:1], -1)).contiguous(), total


def _positions(lens, rows):
    """For packed rows: the request of each and its position (the rows stand at the ends of their requests)."""
    n = torch.tensor(rows, device=DEVICE)
    b = torch.repeat_interleave(torch.arange(len(rows), device=DEVICE), n)
    start = n.cumsum(0) - n
    pos = torch.arange(int(n.sum()), device=DEVICE) - start[b] + (torch.tensor(lens, device=DEVICE) - n)[b]
    return b, pos


def _slots(table, lens, rows, block):
    b, pos = _positions(lens, rows)
    return (table[b, pos // block].long() * block + pos % block).to(torch.int32)


def _starts(rows):
    return _ints([0] + list(torch.tensor(rows).cumsum(0)))


def _keys(n, heads, hd, g, loud):
    """Keys: N(0, 1) with a bias by channel, a few of them loud, as keys have them."""
    return torch.randn(n, heads, hd, generator=g, device=DEVICE) + loud


def _loud(heads, hd, g):
    bias = 0.5 * torch.randn(heads, hd, generator=g, device=DEVICE)
    bias[:, torch.randperm(hd, generator=g, device=DEVICE)[: max(1, hd // 32)]] *= 6.0
    return bias


# -------------------------------------------------------------------------------------------------- the rows in 4 bits
def _up_to_bf16(x):
    """Positive finite float32, rounded up to a bfloat16."""
    return ((x.contiguous().view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)


def _quantise(x):
    """x [..., hd] f32 -> (codes uint8, z, d): float32 operations, each rounded once."""
    lo, hi = x.amin(-1), x.amax(-1)
    z = (0.5 * lo + 0.5 * hi).to(torch.bfloat16).float()
    h = torch.maximum(hi - z, z - lo)
    d = torch.where(h == 0, torch.zeros_like(h), _up_to_bf16(h / 7.5).clamp_min(2.0 ** -120))
    r = torch.where(h == 0, torch.zeros_like(h), 1.0 / d)
    n = torch.round((x - z[..., None]) * r[..., None] + 7.5).clamp_(0, 15)
    return n.to(torch.uint8), z, d


def _values(n, z, d):
    return d[..., None] * (n.float() - 7.5) + z[..., None]


# ------------------------------------------------------------------------------------------- the framework's side (own)
def _ptr(t):
    return C.c_void_p(t.data_ptr())


class _Cache:
    """The framework's paged 4-bit cache and the context that its calls are made on."""

    def __init__(self, blocks, block, heads, hd):
        from peregrine_amd import _ffi, default_context

        self.lib, self.check, self.ctx = _ffi.lib, _ffi.check, default_context()
        self.h = C.c_void_p()
        self.call("pg_paged_kv4_create", blocks, block, heads, hd, C.byref(self.h))

    def call(self, name, *args):
        self.check(getattr(self.lib, name)(self.ctx.handle, *args))

    def append(self, k, v, slots):
        self.call("pg_paged_kv4_append_dev", self.h, _ptr(k), _ptr(v), k.stride(0), k.stride(1), k.shape[0], _ptr(slots))

    def scratch(self, name, *args):
        n = C.c_size_t()
        self.call(name, self.h, *args, C.byref(n))
        return torch.empty(max(256, n.value), dtype=torch.uint8, device=DEVICE)

    def __del__(self):
        if self.h:
            self.lib.pg_paged_kv4_free(self.ctx.handle, self.h)
            self.h = C.c_void_p()


# ------------------------------------------------------------------------------------------------------- block tables
class Tables:
    """A step's block tables and slot map: requests with `most` tokens at most get `rows` new ones at most each."""

    @staticmethod
    def draw(rng):
        block = rng.choice([16, 32, 64, 128])
        return {"batch": _log(rng, 1, 1500), "most": _log(rng, 40, 20000), "rows": _log(rng, 1, 200), "block": block, "ragged": True, "short": rng.random() < 0.3}

    @staticmethod
    def prepare(case, seed):
        g = _gen(seed)
        lens, rows = _shape(case)
        old = [n - r for n, r in zip(lens, rows)]
        block, width = case["block"], _width(case) + 1
        table, used = _tables([max(1, n) for n in old], block, g)
        table = torch.where(torch.arange(table.shape[1], device=DEVICE)[None, :] * block < _ints(old)[:, None], table, -1)
        full = torch.full((case["batch"], width), -1, dtype=torch.int32, device=DEVICE)
        full[:, : table.shape[1]] = table
        need = sum(-(-n // block) - -(-o // block) for n, o in zip(lens, old))
        free = max(1, need * 3 // 4) if case["short"] else need + 100  # "short": the pool does not hold what all requests ask for
        pool = used + free
        free_list = torch.zeros(pool, dtype=torch.int32, device=DEVICE)
        free_list[:free] = used + torch.randperm(free, generator=g, device=DEVICE).to(torch.int32)
        s = {"old": _ints(old), "new": _ints(rows), "table": full, "free_list": free_list, "free": _ints([free]), "block": block, "pool": pool,
             "tokens": sum(rows) + 7}  # the slot map of a step is a little longer than what the step needs
        if own:
            from peregrine_amd import _ffi, default_context

            s |= {"lib": _ffi.lib, "check": _ffi.check, "ctx": default_context()}
            s["out"] = [torch.zeros(n, dtype=torch.int32, device=DEVICE) for n in (case["batch"], 1, case["batch"] + 1, case["batch"], s["tokens"])]
        return s

    @staticmethod
    def run(s):
        if own:
            lens, free, starts, granted, slots = s["out"]
            batch, width = s["table"].shape
            s["check"](s["lib"].pg_block_tables_extend_dev(
                s["ctx"].handle, _ptr(s["old"]), _ptr(s["new"]), batch, s["block"], _ptr(s["free_list"]), _ptr(s["free"]), s["pool"],
                _ptr(s["table"]), width, _ptr(lens), _ptr(free), _ptr(starts), _ptr(granted), _ptr(slots), s["tokens"]))
            return {"table": s["table"], "lens": lens, "free": free, "starts": starts, "granted": granted, "slots": slots}
        old, new, table, block = s["old"].long(), s["new"].long(), s["table"], s["block"]
        batch, width = table.shape
        have = (old + block - 1) // block
        fits = old + new <= width * block
        need = torch.where(fits, (old + new + block - 1) // block - have, 0)
        upto = need.cumsum(0)
        granted = fits & ((need == 0) | (upto <= s["free"]))
        lens = torch.where(granted, old + new, old)
        taken = torch.where(granted, need, 0)
        at = torch.arange(width, device=table.device)[None, :] - have[:, None]
        inside = (at >= 0) & (at < taken[:, None])
        pick = s["free"].long() - 1 - ((upto - need)[:, None] + at)
        table = torch.where(inside, s["free_list"][pick.clamp(0, s["pool"] - 1)], table)
        starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
        row = torch.arange(s["tokens"], device=table.device)
        b = torch.searchsorted(starts, row, right=True) - 1
        behind = b >= batch
        b = b.clamp_max(batch - 1)
        pos = old[b] + row - starts[b]
        slots = torch.where(granted[b] & ~behind, table[b, (pos // block).clamp_max(width - 1)].long() * block + pos % block, -1)
        i = torch.int32
        return {"table": table, "lens": lens.to(i), "free": (s["free"] - torch.where(granted, need, 0).sum()).to(i), "starts": starts.to(i),
                "granted": granted.to(i), "slots": slots.to(i)}

    @staticmethod
    def work(case):
        lens, rows = _shape(case)
        block = case["block"]
        new = sum(-(-n // block) - -(-(n - r) // block) for n, r in zip(lens, rows))
        return {"bytes": 4.0 * (5 * case["batch"] + 2 * new + sum(rows) + 10), "flops": 0.0}

    @staticmethod
    def exact(case, seed):
        return None  # whole numbers


# -------------------------------------------------------------------------------------------------------------- append
class Append:
    """A step's keys and values into the cache: quantised, stored, the touched blocks' summaries brought up to date.  What
    is stored is returned as the values it stands for."""

    @staticmethod
    def draw(rng):
        rows = rng.choice([1, 1, rng.randint(2, 6), _log(rng, 16, 1500)])
        return {"batch": _log(rng, 1, max(1, 4000 // rows)), "most": rows + _log(rng, 1, 300), "rows": rows, "block": rng.choice([16, 32, 64, 128]), "ragged": True,
                "heads": rng.choice([1, 2, 4, 8]), "hd": rng.choice([40, 64, 80, 96, 128, 192, 256])}

    @staticmethod
    def prepare(case, seed):
        g = _gen(seed)
        lens, rows = _shape(case)
        heads, hd, block = case["heads"], case["hd"], case["block"]
        table, blocks = _tables(lens, block, g, spare=2)
        b, pos = _positions(lens, rows)
        last = (pos % block == block - 1) | (pos == _ints(lens)[b] - 1)
        touched = table[b, pos // block][last].contiguous()  # the blocks that hold new rows
        slots = _slots(table, lens, rows, block)
        loud = _loud(heads, hd, g)
        every = _slots(table, lens, lens, block)
        old_k, old_v = _keys(len(every), heads, hd, g, loud), torch.randn(len(every), heads, hd, generator=g, device=DEVICE)
        k, v = _keys(len(slots), heads, hd, g, loud), torch.randn(len(slots), heads, hd, generator=g, device=DEVICE)
        s = {"k": k, "v": v, "slots": slots, "table": table, "lens": _ints(lens), "starts": _starts(rows), "touched": touched, "block": block,
             "batch": len(lens)}
        if own:
            c = s["cache"] = _Cache(blocks, block, heads, hd)
            torch.cuda.synchronize()
            c.append(old_k, old_v, every)
            c.ctx.sync()
            s["out"] = [torch.empty_like(k), torch.empty_like(v)] + [torch.empty(len(touched), heads, hd, device=DEVICE) for _ in range(2)]
        else:
            s["n"], s["z"], s["d"] = (torch.zeros(blocks * block, 2, heads, *x, dtype=t, device=DEVICE) for x, t in (((hd,), torch.uint8), ((), torch.float32), ((), torch.float32)))
            s["n"][every.long()], s["z"][every.long()], s["d"][every.long()] = _quantise(torch.stack([old_k, old_v], 1))
            fill = torch.zeros(blocks, dtype=torch.long, device=DEVICE)  # tokens in each block
            need = torch.tensor([-(-n // block) for n in lens], device=DEVICE)
            at = torch.arange(table.shape[1], device=DEVICE)[None, :]
            fill[table.clamp_min(0).long()[at < need[:, None]]] = (s["lens"][:, None] - at * block).clamp(0, block)[at < need[:, None]].long()
            s["fill"] = fill
        return s

    @staticmethod
    def run(s):
        if own:
            c = s["cache"]
            k, v, lo, hi = s["out"]
            n = s["k"].shape[0]
            c.append(s["k"], s["v"], s["slots"])
            c.call("pg_paged_kv4_summarise_dev", c.h, _ptr(s["starts"]), _ptr(s["lens"]), s["batch"], n, _ptr(s["table"]), s["table"].shape[1])
            c.call("pg_paged_kv4_read_dev", c.h, _ptr(s["slots"]), n, _ptr(k), _ptr(v))
            c.call("pg_paged_kv4_read_summaries_dev", c.h, _ptr(s["touched"]), s["touched"].shape[0], _ptr(lo), _ptr(hi))
            return {"k": k, "v": v, "lo": lo, "hi": hi}
        at = s["slots"].long()
        s["n"][at], s["z"][at], s["d"][at] = _quantise(torch.stack([s["k"], s["v"]], 1))
        kv = _values(s["n"][at], s["z"][at], s["d"][at])
        rows = s["touched"].long()[:, None] * s["block"] + torch.arange(s["block"], device=at.device)
        keys = _values(s["n"][rows, 0], s["z"][rows, 0], s["d"][rows, 0])  # [touched, block, heads, hd]
        (lo, hi), scale = _summary(keys, torch.arange(s["block"], device=at.device) < s["fill"][s["touched"].long()][:, None])
        return {"k": kv[:, 0].contiguous(), "v": kv[:, 1].contiguous(), "lo": lo * scale, "hi": hi * scale}

    @staticmethod
    def work(case):
        lens, rows = _shape(case)
        heads, hd, block = case["heads"], case["hd"], case["block"]
        n = sum(rows)
        touched = sum(-(-n // block) - (n - r) // block for n, r in zip(lens, rows))
        return {"bytes": float(heads * (n * (8 * hd + hd + 8 + 8 * hd) + touched * (block * (hd // 2 + 4) + 2 * hd + 4 + 8 * hd)) + 4 * n), "flops": 12.0 * n * heads * hd}

    @staticmethod
    def exact(case, seed):
        return None  # a code next to the border of two is one or the other by float32 roundings, which the definition counts as its own


def _summary(keys, live):
    """keys [blocks, block, heads, hd], live [blocks, block] -> ((lo, hi) as whole numbers, scale), [blocks, heads, hd]."""
    lo = keys.masked_fill(~live[..., None, None], math.inf).amin(1)
    hi = keys.masked_fill(~live[..., None, None], -math.inf).amax(1)
    most = torch.maximum(lo.abs(), hi.abs()).amax(-1, keepdim=True)
    r = torch.where(most < 2.0 ** -100, torch.zeros_like(most), INT8_MOST / most)
    return (torch.round(lo * r), torch.round(hi * r)), most / INT8_MOST


def _plainly(kind, case, seed):
    """prepare() as it is for the plain form."""
    global own
    was, own = own, False
    try:
        return kind.prepare(case, seed)
    finally:
        own = was


# ----------------------------------------------------------------------------------------------------------- attention
def _filled(case, seed):
    """A cache with every request's rows, and a step's queries."""
    g = _gen(seed)
    lens, rows = _shape(case)
    heads, hd, block = case["heads"], case["hd"], case["block"]
    table, blocks = _tables(lens, block, g, spare=1)
    slots = _slots(table, lens, lens, block)
    total = len(slots)
    s = {"table": table, "lens": _ints(lens), "starts": _starts(rows), "block": block, "batch": len(lens), "scale": hd ** -0.5, "group": case["q_heads"] // heads, "rows": max(rows),
         "tokens": sum(rows), "heads": heads, "hd": hd, "most": max(lens)}
    loud = _loud(heads, hd, g)
    if own:
        c = s["cache"] = _Cache(blocks, block, heads, hd)
    else:
        s["n"] = torch.zeros(blocks * block, 2, heads, hd, dtype=torch.uint8, device=DEVICE)
        s["z"], s["d"] = (torch.zeros(blocks * block, 2, heads, device=DEVICE) for _ in range(2))
    piece = max(1, (1 << 27) // (heads * hd))
    for at in range(0, total, piece):
        to = slots[at: at + piece].contiguous()
        k, v = _keys(len(to), heads, hd, g, loud), torch.randn(len(to), heads, hd, generator=g, device=DEVICE)
        if own:
            torch.cuda.synchronize()
            c.append(k, v, to)
            c.ctx.sync()
        else:
            s["n"][to.long()], s["z"][to.long()], s["d"][to.long()] = _quantise(torch.stack([k, v], 1))
    s["q"] = 1.5 * torch.randn(s["tokens"], case["q_heads"], hd, generator=g, device=DEVICE)
    if own:
        s["out"] = torch.empty(s["tokens"], case["q_heads"], hd, device=DEVICE)
    return s


class Attention:
    """A step's queries against the whole of each request's rows: single tokens (rows 1), a few, or prompts."""

    @staticmethod
    def draw(rng):
        heads, group, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8, 16]), rng.choice([64, 80, 96, 128, 128, 256])
        rows = rng.choice([1, 1, 1, rng.randint(2, 5), _log(rng, 20, 1500)])
        most = rows + _log(rng, 1, 60000 if rows < 6 else 12000)
        batch = max(1, _log(rng, 1, max(1, min(96, (300000 if rows < 6 else 30000) // most))))
        window = rng.choice([0, 0, 0, 0, _log(rng, 8, 2000)])
        return {"batch": batch, "most": most, "rows": rows, "block": rng.choice([16, 32, 64, 128]), "ragged": True, "heads": heads, "q_heads": heads * group, "hd": hd,
                "window": window, "sinks": rng.choice([0, 4]) if window else 0, "cap": rng.choice([0.0, 0.0, 0.0, 30.0])}

    @staticmethod
    def prepare(case, seed):
        s = _filled(case, seed)
        s |= {"window": case["window"], "sinks": case["sinks"], "cap": case["cap"]}
        if own:
            s["scratch"] = s["cache"].scratch("pg_paged_kv4_attention_scratch", case["q_heads"], s["batch"], s["rows"], s["table"].shape[1])
        return s

    @staticmethod
    def run(s):
        if own:
            c, q = s["cache"], s["q"]
            c.call("pg_paged_kv4_attention_dev", c.h, _ptr(q), q.stride(0), q.stride(1), q.shape[1], _ptr(s["starts"]), _ptr(s["lens"]), s["batch"], s["tokens"], s["rows"],
                   _ptr(s["table"]), s["table"].shape[1], s["scale"], 2 if s["window"] else 1, s["window"], s["sinks"], s["cap"], _ptr(s["scratch"]), s["scratch"].numel(), _ptr(s["out"]))
            return s["out"]
        batch, heads, group, hd, rows, most, block = (s[k] for k in ("batch", "heads", "group", "hd", "rows", "most", "block"))
        at = torch.arange(most, device=DEVICE)
        slot = s["table"].clamp_min(0).long()[:, at // block] * block + at % block  # [batch, most]
        k, v = (_values(s["n"][slot, i], s["z"][slot, i], s["d"][slot, i]).permute(0, 2, 1, 3).contiguous() for i in (0, 1))  # [batch, heads, most, hd]
        row = torch.arange(rows, device=DEVICE)
        count = s["starts"].diff()
        index = (s["starts"][:-1, None] + row).clamp_max(s["tokens"] - 1).long()  # [batch, rows]
        q = s["q"][index].view(batch, rows, heads, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * rows, hd)
        x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(batch, heads, group, rows, most).mul_(s["scale"])
        if s["cap"]:
            x = s["cap"] * torch.tanh(x / s["cap"])
        far = (s["lens"] - count)[:, None, None] + row[:, None] - at  # [batch, rows, most]: how far the key is behind the query
        seen = (far >= 0) & (at < s["lens"][:, None, None])
        if s["window"]:
            seen &= (far <= s["window"]) | (at < s["sinks"])
        x = x.masked_fill_(~seen[:, None, None], -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
        total = x.sum(-1, keepdim=True)
        y = torch.matmul(x.view(batch, heads, group * rows, most), v).view(batch, heads, group, rows, hd) / total.clamp_min(1e-30)
        return y.permute(0, 3, 1, 2, 4)[row < count[:, None]].reshape(s["tokens"], heads * group, hd)

    @staticmethod
    def work(case):
        lens, rows = _shape(case)
        seen = read = 0
        for n, r in zip(lens, rows):
            w = case["window"] + 1 + case["sinks"] if case["window"] else n
            seen += sum(min(p + 1, w) for p in range(n - r, n))
            read += min(n, w + r - 1)
        hd = case["hd"]
        return {"bytes": float(read * case["heads"] * (hd + 8) + sum(rows) * case["q_heads"] * hd * 8), "flops": 4.0 * hd * seen * case["q_heads"]}

    @staticmethod
    def exact(case, seed):
        if Attention.work(case)["flops"] > 2e13:
            return None
        s = _plainly(Attention, case, seed)
        lens, rows = _shape(case)
        out = torch.zeros(s["tokens"], case["q_heads"], s["hd"], dtype=torch.float64, device=DEVICE)
        done = 0
        for b, (n, r) in enumerate(zip(lens, rows)):
            slot = _slots(s["table"][b: b + 1], [n], [n], s["block"]).long()
            pos = torch.arange(n - r, n, device=DEVICE)[:, None]
            key = torch.arange(n, device=DEVICE)[None, :]
            seen = key <= pos
            if case["window"]:
                seen = seen & ((pos - key <= case["window"]) | (key < case["sinks"]))
            for h in range(s["heads"]):
                kv = s["z"][slot, :, h, None].double() + s["d"][slot, :, h, None].double() * (s["n"][slot, :, h].double() - 7.5)  # [n, 2, hd]
                for j in range(h * s["group"], (h + 1) * s["group"]):
                    x = s["q"][done: done + r, j].double() @ kv[:, 0].T * s["scale"]
                    if case["cap"]:
                        x = case["cap"] * torch.tanh(x / case["cap"])
                    out[done: done + r, j] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ kv[:, 1]
            done += r
        return out


# ---------------------------------------------------------------------------------------------------- selected blocks
class Selected:
    """A step's queries against the blocks that score highest for each of them and each key head."""

    @staticmethod
    def draw(rng):
        heads, group, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 80, 128, 128, 256])
        rows = rng.choice([1, 1, 1, rng.randint(2, 5), _log(rng, 10, 200)])
        block = rng.choice([16, 32, 64])
        top = _log(rng, 4, 2048 // block)
        most = rows + _log(rng, 1, 60000 if rows < 6 else 8000)
        batch = max(1, _log(rng, 1, max(1, min(64, (200000 if rows < 6 else 8000) // most))))
        return {"batch": batch, "most": most, "rows": rows, "block": block, "ragged": True, "heads": heads, "q_heads": heads * group, "hd": hd, "top": top,
                "first": rng.choice([0, 1]), "recent": rng.choice([1, 2])}

    @staticmethod
    def prepare(case, seed):
        s = _filled(case, seed)
        s |= {k: case[k] for k in ("top", "first", "recent")}
        lens, rows = _shape(case)
        s["b"], s["pos"] = _positions(lens, rows)
        if own:
            c = s["cache"]
            c.call("pg_paged_kv4_summarise_dev", c.h, _ptr(_starts(lens)), _ptr(s["lens"]), s["batch"], sum(lens), _ptr(s["table"]), s["table"].shape[1])
            s["scratch"] = c.scratch("pg_paged_kv4_selected_scratch", case["q_heads"], s["tokens"], s["top"])
            s["selected"] = torch.empty(s["tokens"], s["heads"], s["top"], dtype=torch.int32, device=DEVICE)
            c.ctx.sync()
        else:
            blocks = s["n"].shape[0] // s["block"]
            fill = torch.zeros(blocks, dtype=torch.long, device=DEVICE)
            at = torch.arange(s["table"].shape[1], device=DEVICE)[None, :]
            live = at * s["block"] < s["lens"][:, None]
            fill[s["table"].long()[live]] = (s["lens"][:, None] - at * s["block"]).clamp(0, s["block"])[live].long()
            lo, hi = (torch.zeros(blocks, s["heads"], s["hd"], device=DEVICE) for _ in range(2))
            sb = torch.zeros(blocks, s["heads"], device=DEVICE)
            piece = max(1, (1 << 27) // (s["block"] * s["heads"] * s["hd"]))
            for i in range(0, blocks, piece):
                j = min(blocks, i + piece)
                rows_of = slice(i * s["block"], j * s["block"])
                keys = _values(s["n"][rows_of, 0], s["z"][rows_of, 0], s["d"][rows_of, 0]).view(j - i, s["block"], s["heads"], s["hd"])
                (lo[i:j], hi[i:j]), scale = _summary(keys, torch.arange(s["block"], device=DEVICE) < fill[i:j, None].clamp_min(1))
                sb[i:j] = scale[..., 0]
            s |= {"lo": lo, "hi": hi, "sb": sb}
        return s

    @staticmethod
    def run(s):
        if own:
            c, q = s["cache"], s["q"]
            c.call("pg_paged_kv4_select_dev", c.h, _ptr(q), q.stride(0), q.stride(1), q.shape[1], _ptr(s["starts"]), _ptr(s["lens"]), s["batch"], s["tokens"],
                   _ptr(s["table"]), s["table"].shape[1], s["top"], s["first"], s["recent"], _ptr(s["selected"]))
            c.call("pg_paged_kv4_attention_selected_dev", c.h, _ptr(q), q.stride(0), q.stride(1), q.shape[1], _ptr(s["starts"]), _ptr(s["lens"]), s["batch"], s["tokens"],
                   _ptr(s["table"]), s["table"].shape[1], _ptr(s["selected"]), s["top"], s["scale"], 0.0, _ptr(s["scratch"]), s["scratch"].numel(), _ptr(s["out"]))
            return {"selected": s["selected"], "out": s["out"]}
        heads, group, hd, block, top, tokens = (s[k] for k in ("heads", "group", "hd", "block", "top", "tokens"))
        q = s["q"].view(tokens, heads, group, hd)
        most = q.abs().amax(-1, keepdim=True)
        x = torch.round(q * torch.where(most < 2.0 ** -100, torch.zeros_like(most), INT8_MOST / most))
        sq = most[..., 0] / INT8_MOST
        table = s["table"][s["b"]].clamp_min(0).long()  # [tokens, width]
        width = table.shape[1]
        hi, lo = (s[k][table].permute(0, 2, 3, 1).contiguous() for k in ("hi", "lo"))  # [tokens, heads, hd, width]
        whole = torch.matmul(x.clamp_min(0), hi) + torch.matmul(x.clamp_max(0), lo)  # sums of whole numbers under 2^24: exact
        score = (whole * sq[..., None] * s["sb"][table].permute(0, 2, 1)[:, :, None]).amax(2)  # [tokens, heads, width]
        at = torch.arange(width, device=DEVICE)
        last = (s["pos"] // block)[:, None, None]
        score = torch.where((at < s["first"]) | (at > last - s["recent"]), math.inf, score)
        score = torch.where(at > last, -math.inf, score)
        order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]  # of equals the lowest first
        chosen = torch.where(order <= last, order, width).sort(-1).values
        if chosen.shape[-1] < top:
            chosen = torch.nn.functional.pad(chosen, (0, top - chosen.shape[-1]), value=width)
        live = chosen < width
        selected = torch.where(live, chosen, -1).to(torch.int32)
        key = (chosen * block)[..., None] + torch.arange(block, device=DEVICE)  # [tokens, heads, top, block]: positions
        seen = (live[..., None] & (key <= s["pos"][:, None, None, None])).view(tokens, heads, 1, top * block)
        rows = table[torch.arange(tokens, device=DEVICE)[:, None, None], chosen.clamp_max(width - 1)]
        slot = (rows * block)[..., None] + torch.arange(block, device=DEVICE)
        slot = slot.view(tokens, heads, top * block)
        head = torch.arange(heads, device=DEVICE)[None, :, None]
        k, v = (_values(s["n"][slot, i, head], s["z"][slot, i, head], s["d"][slot, i, head]) for i in (0, 1))  # [tokens, heads, keys, hd]
        y = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
        y = y.masked_fill(~seen, -math.inf)
        y = torch.exp(y - y.amax(-1, keepdim=True))
        y = torch.matmul(y, v) / y.sum(-1, keepdim=True)
        return {"selected": selected, "out": y.reshape(tokens, heads * group, hd)}

    @staticmethod
    def work(case):
        lens, rows = _shape(case)
        heads, hd, block = case["heads"], case["hd"], case["block"]
        summaries = sum(-(-n // block) for n in lens) * heads * (2 * hd + 4)
        keys = sum(min(p + 1, case["top"] * block) for n, r in zip(lens, rows) for p in range(n - r, n))
        once = sum(min(n, r * case["top"] * block) for n, r in zip(lens, rows))  # what all of a request's queries can have read
        scores = sum((p // block + 1) for n, r in zip(lens, rows) for p in range(n - r, n))
        return {"bytes": float(summaries + once * heads * (hd + 8) + sum(rows) * (case["q_heads"] * hd * 8 + 4 * heads * case["top"])),
                "flops": 4.0 * hd * case["q_heads"] * (keys + scores)}

    @staticmethod
    def exact(case, seed):
        s = _plainly(Selected, case, seed)
        if s["tokens"] * s["heads"] > 5000:
            return None
        out = torch.zeros(s["tokens"], case["q_heads"], s["hd"], dtype=torch.float64, device=DEVICE)
        for t in range(s["tokens"]):
            pos, line = int(s["pos"][t]), s["table"][s["b"][t]].long()
            last = pos // s["block"]
            mine = line[: last + 1]
            for h in range(s["heads"]):
                q = s["q"][t, h * s["group"]: (h + 1) * s["group"]].double()
                most = q.abs().amax(1, keepdim=True)
                # the score's own definition: 8-bit queries and summaries, sums of whole numbers, two float32 products
                x = torch.round((q.float() * (INT8_MOST / most.float())).double())
                sums = (x.clamp_min(0)[:, None] * s["hi"][mine, h].double() + x.clamp_max(0)[:, None] * s["lo"][mine, h].double()).sum(-1)
                score = (sums.float() * (most.float() / INT8_MOST) * s["sb"][mine, h]).amax(0).double()
                score[: s["first"]] = math.inf
                score[max(0, last + 1 - s["recent"]):] = math.inf
                chosen = torch.sort(torch.argsort(score, descending=True, stable=True)[: s["top"]]).values
                key = (chosen[:, None] * s["block"] + torch.arange(s["block"], device=DEVICE)).flatten()
                key = key[key <= pos]
                slot = line[key // s["block"]] * s["block"] + key % s["block"]
                kv = s["z"][slot, :, h, None].double() + s["d"][slot, :, h, None].double() * (s["n"][slot, :, h].double() - 7.5)
                out[t, h * s["group"]: (h + 1) * s["group"]] = torch.softmax(q @ kv[:, 0].T * s["scale"], -1) @ kv[:, 1]
        return {"selected": None, "out": out}


KINDS = {"tables": Tables, "append": Append, "attention": Attention, "selected": Selected}


def listed():
    llama = {"heads": 8, "q_heads": 32, "hd": 128, "block": 64}
    whole = {"window": 0, "sinks": 0, "cap": 0.0}
    return [
        # a decoding step of 256 requests: a new token each, a new block for some
        {"name": "tables_256_decoding", "kind": "tables", "batch": 256, "most": 8192, "rows": 1, "block": 64, "ragged": True, "short": False},
        # a step that admits prompts, with blocks of 16 tokens and a pool that does not hold all of them
        {"name": "tables_200_prompts_pool_short", "kind": "tables", "batch": 200, "most": 2500, "rows": 1777, "block": 16, "ragged": True, "short": True},
        # the same two steps' keys and values: 48 requests decoding, and prompts of up to 1000 tokens behind shared beginnings
        {"name": "append_48_decoding", "kind": "append", "batch": 48, "most": 300, "rows": 1, "block": 64, "ragged": True, "heads": 8, "hd": 128},
        {"name": "append_prompts_24x1000", "kind": "append", "batch": 24, "most": 1100, "rows": 1000, "block": 64, "ragged": True, "heads": 8, "hd": 128},
        # one user's first tokens, a small model: latency
        {"name": "decode_1_of_37", "kind": "attention", "batch": 1, "most": 37, "rows": 1, "block": 16, "ragged": False, "heads": 2, "q_heads": 14, "hd": 64, **whole},
        # a decoding batch of the benchmark's layer, ragged
        {"name": "decode_32_to_4000", "kind": "attention", "batch": 32, "most": 4000, "rows": 1, "ragged": True, **llama, **whole},
        # few long contexts, three draft tokens and the last one checked at once
        {"name": "verify_4_rows_2_of_131072", "kind": "attention", "batch": 2, "most": 131072, "rows": 4, "ragged": False, **llama, **whole},
        # a full server
        {"name": "decode_128_to_12000", "kind": "attention", "batch": 128, "most": 12000, "rows": 1, "ragged": True, **llama, **whole},
        # short ragged prompts with a sliding window, sinks and capped logits, heads of 256
        {"name": "prompts_6x700_window", "kind": "attention", "batch": 6, "most": 900, "rows": 700, "block": 32, "ragged": True, "heads": 4, "q_heads": 16, "hd": 256,
         "window": 255, "sinks": 4, "cap": 30.0},
        # a piece of a long prompt
        {"name": "prompt_piece_2048_at_16384", "kind": "attention", "batch": 1, "most": 16384, "rows": 2048, "ragged": False, **llama, **whole},
        # long contexts read in part: 64 blocks of 64 for each query and key head
        {"name": "selected_8_of_65536", "kind": "selected", "batch": 8, "most": 65536, "rows": 1, "ragged": True, "top": 64, "first": 1, "recent": 2, **llama},
        # a piece of a prompt read in part
        {"name": "selected_piece_300_at_8000", "kind": "selected", "batch": 1, "most": 8000, "rows": 300, "ragged": False, "block": 32, "heads": 8, "q_heads": 32, "hd": 128, "top": 48,
         "first": 1, "recent": 4},
    ]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["tables", "append", "attention", "attention", "selected"])
        c = {"kind": kind, **KINDS[kind].draw(rng)}
        if kind == "selected" and c["top"] < c["first"] + c["recent"]:
            continue
        if _cost(c) <= most:
            return c


def _cost(case):
    """Of the order of the time that a pass of the plain form takes."""
    w = work(case)
    return max(w["bytes"], w["flops"] / 20)


def prepare(case, seed):
    s = KINDS[case["kind"]].prepare(case, seed)
    s["kind"] = KINDS[case["kind"]]
    torch.cuda.synchronize()
    return s


def run(state):
    return state["kind"].run(state)


def work(case):
    return KINDS[case["kind"]].work(case)


def exact(case, seed):
    return KINDS[case["kind"]].exact(case, seed)
