"""The operators of the paged 8-bit key / value cache, as they are measured: block tables and slot maps built from request lengths
(`slots`), the append that quantises new keys and values into pages (`append`) and attention over those pages (`attention`).

A page holds `block` tokens of one kv head: keys [blocks, kv_heads, block, hd16], values [blocks, kv_heads, hd16, block] (a value's tokens
stand next to each other), hd16 = head_dim rounded up to 16, in float8_e4m3fn ("fp8") or int8, with one power-of-two scale for
each page and head: x = code * scale.  Pages come back as they are held, codes next to their scales: the codes are defined to the
bit (dividing by a power of two is exact, so every code is one rounding of the exact value).

The plain forms below are elementary torch operations over whole tensors, in 32 bits (64 where a rotated key is rounded to its code)."""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"fp8": 448.0, "int8": 127.0}                     # the largest code
EXP = {"fp8": (-15, 7), "int8": (-24, 9)}               # the scales' exponents: the smallest resolve fp16's own quantum, the largest code stays finite in fp16


# ---- cases --------------------------------------------------------------------------------------------------------------------------

def _slots(name, rows, block, past, new, ended=0, tail=0):
    """rows sequences that hold `past` tokens at most and bring `new` at most (uniform: all of them bring exactly that)."""
    return {"name": name, "op": "slots", "rows": rows, "block": block, "past": past, "new": new, "ended": ended, "tail": tail}


def _append(name, rows, new, past, kv_heads, hd, block, code, rope):
    return {"name": name, "op": "append", "rows": rows, "new": new, "past": past, "kv_heads": kv_heads, "hd": hd, "block": block, "code": code, "rope": rope}


def _attention(name, rows, new, past, heads, kv_heads, hd, block, code, rope, ragged):
    return {"name": name, "op": "attention", "rows": rows, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads, "hd": hd, "block": block,
            "code": code, "rope": rope, "ragged": ragged}


def listed():
    return [
        # one user's next token: nothing but latency
        _slots("slots: one row, one token", 1, 64, 2047, 1),
        # a serving step of 256 users of very different lengths, some of whom have just ended
        _slots("slots: step of 256 rows", 256, 64, 8000, 1, ended=9),
        # a queue of prompts of all lengths taken in at once, in a buffer longer than they are
        _slots("slots: 2048 prompts", 2048, 16, 200, 500, ended=31, tail=777),
        # the new token of 64 users into a 70B layer's cache
        _append("append: 64 rows, one token", 64, 1, 4000, 8, 128, 64, "fp8", True),
        # a 7B layer's full prompt
        _append("append: prompt of 2048", 1, 2048, 0, 32, 128, 64, "fp8", True),
        # prompts of ragged lengths continued from ragged lengths
        _append("append: ragged, int8", 40, 6000, 900, 8, 128, 32, "int8", False),
        # one user's next token at the end of a 7B context
        _attention("decode: one row, 7B", 1, 1, 2047, 32, 32, 128, 64, "fp8", True, False),
        # four drafted tokens each for five users of a 3B model (head_dim 100)
        _attention("decode: four drafts, hd 100", 5, 4, 700, 32, 32, 100, 16, "fp8", True, True),
        # a 70B layer's serving step with ragged lengths
        _attention("decode: 96 ragged rows, 70B", 96, 1, 16383, 64, 8, 128, 64, "int8", True, True),
        # long documents
        _attention("decode: 8 rows of 65536, 70B", 8, 1, 65535, 64, 8, 128, 64, "fp8", False, False),
        # a 7B layer's full prompt
        _attention("prompt of 2048, 7B", 1, 2048, 0, 32, 32, 128, 64, "fp8", True, False),
        # a piece of a long prompt next to short and single-token rows, 70B
        _attention("prompt pieces, 70B", 3, 1000, 12000, 64, 8, 128, 32, "int8", True, True),
    ]


def _log(rng, lo, hi):
    """a whole number of lo..hi, spread over the logarithm"""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["slots", "append", "attention", "attention"])
    block = rng.choice([16, 32, 64, 128])
    code = rng.choice(["fp8", "int8"])
    rope = rng.random() < 0.6
    if op == "slots":
        rows, new = _log(rng, 1, 2048), _log(rng, 1, 500) if rng.random() < 0.6 else 1
        return _slots("drawn", rows, block, _log(rng, 1, 8000), new, ended=rng.randint(0, rows // 8), tail=rng.choice([0, 1, 333]))
    hd = rng.choice([64, 80, 100, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 32])
    if op == "append":
        rows = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, 60000 * 8 // (rows * max(kv_heads, 8) * 2)))
        return _append("drawn", rows, new, _log(rng, 1, 4000), kv_heads, hd, block, code, rope)
    group = rng.choice([1, 1, 3, 4, 8, 16]) if kv_heads <= 8 else 1
    if rng.random() < 0.6:                                # tokens one at a time, or a few drafted ones
        rows, new = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 5])
        past = _log(rng, 1, max(1, 400000 * 8 * 128 // (rows * max(kv_heads, 8) * hd)))
    else:                                                 # prompts and pieces of prompts
        rows = _log(rng, 1, 4)
        new = _log(rng, 17, 2048 // rows)
        past = _log(rng, 1, max(1, 24_000_000 * 16 // (rows * new * kv_heads * group)))
        past = min(past, 20000)
    return _attention("drawn", rows, new, past, kv_heads * group, kv_heads, hd, block, code, rope, rng.random() < 0.7)


# ---- inputs -------------------------------------------------------------------------------------------------------------------------

def _lens(case, seed):
    """(past, new) of every row, on the host: what a scheduler has decided.  Ragged rows spread over the logarithm of their length; one
    has the full length, and from three rows on one brings nothing.  The lengths belong to the case, their order to the seed."""
    rows, past, new = case["rows"], case["past"], case["new"]
    if not case.get("ragged", True) or rows == 1:
        return [past] * rows, [new] * rows
    rng = random.Random(rows * 1000003 + past * 1009 + new)
    ps = [past] + [_log(rng, 1, past + 1) - 1 for _ in range(rows - 1)]
    ns = [new] + [_log(rng, 1, new) for _ in range(rows - 1)]
    if rows >= 3:
        ns[-1] = 0
    order = list(range(rows))
    random.Random(seed).shuffle(order)
    return [ps[b] for b in order], [ns[b] for b in order]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _power(e):
    """2 ** e, exact, in 32 bits"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(gen, shape, code):
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)
    return (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn) if code == "fp8" else (x * 30).round_().clamp_(-127, 127).to(torch.int8)


def _pool(gen, case, blocks):
    """Pages and scales as a cache in use holds them."""
    bs, kvh, hd16, code = case["block"], case["kv_heads"], (case["hd"] + 15) // 16 * 16, case["code"]
    kp, vp = _codes(gen, (blocks, kvh, bs, hd16), code), _codes(gen, (blocks, kvh, hd16, bs), code)
    kp[..., case["hd"]:] = 0
    vp[..., case["hd"]:, :] = 0
    lo = -8 if code == "fp8" else -6
    ks, vs = (_power(torch.randint(lo, lo + 3, (blocks, kvh), generator=gen, device=DEV)) for _ in range(2))
    return kp, vp, ks, vs


def _tables(case, ps, ns, gen, spare=3):
    """Block tables of rows whose blocks lie anywhere in the pool: (table, number of blocks in the pool)."""
    bs = case["block"]
    need = [(p + n + bs - 1) // bs for p, n in zip(ps, ns)]
    width, blocks = max(1, max(need)), sum(need) + spare
    order = torch.randperm(blocks, generator=gen, device=DEV)[:sum(need)].to(torch.int32)
    at = torch.arange(width, device=DEV)[None, :]
    need_d = torch.tensor(need, device=DEV)[:, None]
    first = torch.cumsum(need_d, 0) - need_d
    table = torch.where(at < need_d, order[(first + at).clamp_(max=max(0, sum(need) - 1))], torch.full((), -1, dtype=torch.int32, device=DEV))
    return table, blocks


def _angles(positions, hd):
    """sin / cos tables [positions, hd] as the model keeps them."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device=DEV).float() / hd))
    f = torch.arange(positions, device=DEV).float()[:, None] * inv[None, :]
    f = torch.cat((f, f), 1)
    return f.sin().half(), f.cos().half()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    ps, ns = _lens(case, seed)
    s = {"case": case}
    if case["op"] == "slots":
        bs, rows = case["block"], case["rows"]
        rng = random.Random(seed)
        gone = set(rng.sample(range(rows), case["ended"]))
        held = [(p + bs - 1) // bs + (rng.random() < 0.1) for p in ps]      # a few rows hold a block ahead
        cap = (max(ps) + case["new"] + bs) // bs + 1
        blocks = sum((p + n + bs - 1) // bs + 1 for p, n in zip(ps, ns)) + 5
        spare = blocks - sum(held)
        order = torch.randperm(blocks, generator=gen, device=DEV).to(torch.int32)
        at, held_d = torch.arange(cap, device=DEV)[None, :], torch.tensor(held, device=DEV)[:, None]
        first = torch.cumsum(held_d, 0) - held_d
        s["table"] = torch.where(at < held_d, order[(first + at).clamp_(max=blocks - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
        head = rng.randrange(blocks)
        s["ring"] = torch.full((blocks,), -1, dtype=torch.int32, device=DEV)
        s["ring"][(head + torch.arange(spare, device=DEV)) % blocks] = order[sum(held):]
        s["counters"] = _ints([head, spare, 0, 0])
        s["held"] = _ints(held)
        s["past"], s["new"] = _ints(ps), _ints([-1 if b in gone else n for b, n in enumerate(ns)])
        s["rows"] = sum(ns) + case["tail"]                # the buffer was made for the rows that have ended, too
        return s
    table, blocks = _tables(case, ps, ns, gen)
    s["table"], s["past"], s["new"] = table, _ints(ps), _ints(ns)
    starts = [sum(ns[:b]) for b in range(len(ns))]
    s["starts"] = _ints(starts + [sum(ns)])
    s["kp"], s["vp"], s["ks"], s["vs"] = _pool(gen, case, blocks)
    s["sin"], s["cos"] = _angles(max(p + n for p, n in zip(ps, ns)), case["hd"]) if case["rope"] else (None, None)
    t = sum(ns) + 2                                       # two rows behind the last sequence
    if case["op"] == "attention":
        s["q"] = torch.randn(t, case["heads"] * case["hd"], generator=gen, device=DEV, dtype=torch.float16)
        s["out"] = torch.zeros_like(s["q"])
        s["longest"] = max(p + n for p, n in zip(ps, ns))
        return s
    row = torch.repeat_interleave(torch.arange(len(ns), device=DEV), torch.tensor(ns, device=DEV))
    pos = s["past"].long()[row] + torch.arange(sum(ns), device=DEV) - s["starts"].long()[row]
    slot = s["table"].long()[row, pos // case["block"]] * case["block"] + pos % case["block"]
    behind = torch.full((2,), -1, device=DEV)
    s["slots"], s["positions"] = torch.cat((slot, behind)).to(torch.int32), torch.cat((pos, behind * 0)).to(torch.int32)
    channel = torch.exp(torch.randn(case["kv_heads"] * case["hd"], generator=gen, device=DEV))      # keys have a few strong channels
    s["k"] = (torch.randn(t, case["kv_heads"] * case["hd"], generator=gen, device=DEV) * channel).half()
    s["v"] = torch.randn(t, case["kv_heads"] * case["hd"], generator=gen, device=DEV).half()
    return s


# ---- the operators ------------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        from exllama_amd import cuda_ext
        c, s = state["case"], state
        if op == "slots":
            starts, slots, positions = cuda_ext.ext_paged_slots(s["past"], s["new"], s["held"], s["table"], s["ring"], s["counters"], c["block"],
                                                                s["rows"], max_new=c["new"])
            return {"starts": starts, "slots": slots, "positions": positions, "table": s["table"], "held": s["held"], "ring": s["ring"],
                    "counters": s["counters"]}
        if op == "append":
            cuda_ext.ext_paged_append(s["k"], s["v"], s["slots"], s["kp"], s["vp"], s["ks"], s["vs"], positions=s["positions"], sin=s["sin"], cos=s["cos"])
            return {"key_pages": s["kp"], "value_pages": s["vp"], "key_scales": s["ks"], "value_scales": s["vs"]}
        return cuda_ext.ext_paged_attention(s["q"], s["starts"], s["past"], s["new"], s["table"], s["kp"], s["vp"], s["ks"], s["vs"], c["heads"],
                                            max_new=c["new"], sin=s["sin"], cos=s["cos"], out=s["out"])
    return {"slots": _plain_slots, "append": _plain_append, "attention": _plain_attention}[op](state)


def _plain_slots(s):
    bs, table, ring, rows = s["case"]["block"], s["table"], s["ring"], s["rows"]
    blocks, (count, width) = ring.numel(), table.shape
    past, new, held = s["past"].long(), s["new"].long(), s["held"].long()
    head, avail = s["counters"][0].long(), s["counters"][1].long()
    take = new.clamp(0, s["case"]["new"])
    ends = torch.cumsum(take, 0).clamp(max=rows)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    take = starts[1:] - starts[:-1]
    end = (past + take).clamp(max=width * bs)
    gone = new < 0
    want = torch.where(gone, 0, (torch.div(end + bs - 1, bs, rounding_mode="floor") - held).clamp(min=0))
    base = torch.cumsum(want, 0) - want
    got = torch.minimum((avail - base).clamp(min=0), want)
    back = torch.where(gone, held, 0)
    tail = torch.cumsum(back, 0) - back + head + avail
    at = torch.arange(width, device=table.device)[None, :]
    fresh = (at >= held[:, None]) & (at < (held + got)[:, None])
    from_ring = ring[(head + base[:, None] + at - held[:, None]).remainder(blocks)]
    old = gone[:, None] & (at < held[:, None])
    ring_at = torch.where(old, (tail[:, None] + at).remainder(blocks), blocks)
    ring_new = torch.cat((ring, ring[:1]))
    ring_new.scatter_(0, ring_at.reshape(-1), torch.where(old, table, ring_new[ring_at]).reshape(-1))
    table.copy_(torch.where(old, -1, torch.where(fresh, from_ring, table)))
    ring.copy_(ring_new[:blocks])
    kept = torch.where(gone, 0, held + got)
    s["held"].copy_(kept)
    s["counters"].copy_(torch.stack((torch.remainder(head + got.sum(), blocks), avail - got.sum() + back.sum(), (want - got).sum(), avail * 0)))
    t = torch.arange(rows, device=table.device)
    row = torch.searchsorted(ends, t, right=True).clamp(max=count - 1)
    pos = past[row] + t - starts[row]
    inside = t < ends[-1]
    page = table[row, torch.div(pos, bs, rounding_mode="floor").clamp(max=width - 1)].long()
    there = inside & (pos < kept[row] * bs) & (page >= 0)
    return {"starts": starts.to(torch.int32), "slots": torch.where(there, page * bs + pos % bs, -1).to(torch.int32),
            "positions": torch.where(inside, pos, 0).to(torch.int32), "table": table, "held": s["held"], "ring": ring, "counters": s["counters"]}


def _rotated(x, sin, cos, positions):
    """x [tokens, heads, hd] rotated by halves, in x's type"""
    half = x.shape[-1] // 2
    si, co = sin[positions].to(x.dtype)[:, None, :], cos[positions].to(x.dtype)[:, None, :]
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat((lo * co[..., :half] - hi * si[..., :half], hi * co[..., half:] + lo * si[..., half:]), -1)


def _scale_for(amax, code):
    """the least power of two that brings amax to the codes' range"""
    f, e = torch.frexp(amax)
    tf, te = math.frexp(TOP[code])
    e = e - te + (f > tf).to(e.dtype)
    return _power(torch.where(amax > 0, e, EXP[code][0]).clamp(*EXP[code]))


def _encode(x, code):
    """codes' bits of x, which is already divided by its scale"""
    if code == "fp8":
        return x.clamp(-448, 448).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(x.isnan(), 0, x).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)


def _plain_append(s):
    c = s["case"]
    some = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot = s["slots"][some].long()
    page, off = torch.div(slot, c["block"], rounding_mode="floor"), slot % c["block"]
    first = torch.ones_like(page, dtype=torch.bool)
    first[1:] = page[1:] != page[:-1]
    k, v = (s[n][some].view(-1, c["kv_heads"], c["hd"]).double() for n in ("k", "v"))
    if s["sin"] is not None:
        k = _rotated(k, s["sin"], s["cos"], s["positions"][some].long())
    _plain_into_pages(c, k, page, off, first, s["kp"], s["ks"], True)
    _plain_into_pages(c, v, page, off, first, s["vp"], s["vs"], False)
    return {"key_pages": s["kp"], "value_pages": s["vp"], "key_scales": s["ks"], "value_scales": s["vs"]}


def _plain_into_pages(c, x, page, off, first, codes, scales, is_key):
    """x [tokens, kv_heads, hd] in 64 bits to place off of page, in place on codes and scales; `first`: the first token of a page"""
    code, bs = c["code"], c["block"]
    lead = torch.nonzero(first)[:, 0]
    pages, kept = page[lead], off[lead]                   # the pages that are written, and how many tokens of each stay
    heads = torch.arange(c["kv_heads"], device=page.device)
    cap = TOP[code] * 2.0 ** EXP[code][1]
    x = x.clamp(-cap, cap)
    amax = torch.zeros_like(scales, dtype=torch.float64).scatter_reduce_(0, page[:, None].expand(-1, c["kv_heads"]), torch.where(x.isnan(), 0, x.abs()).amax(-1), "amax")
    fresh = _scale_for(amax[pages], code)
    before = torch.where(kept[:, None] > 0, scales[pages], fresh)
    now = torch.maximum(fresh, before)
    bits = codes.view(torch.uint8)
    held = bits[pages].view(CODE[code]).float()
    moved = _encode(held * (before / now)[:, :, None, None], code)
    token = torch.arange(bs, device=page.device).view((1, 1, bs, 1) if is_key else (1, 1, 1, bs))
    bits[pages] = torch.where(token < kept[:, None, None, None], moved, bits[pages])
    scales[pages] = now
    hd16 = codes.shape[-1] if is_key else codes.shape[-2]
    new = _encode(torch.nn.functional.pad(_rounded(x / scales[page].double()[:, :, None], code), (0, hd16 - c["hd"])), code)
    if is_key:
        bits[page[:, None], heads[None, :], off[:, None]] = new
    else:
        bits[page[:, None], heads[None, :], :, off[:, None]] = new


def _rounded(x, code):
    """a code's value of every x, rounded from 64 bits at once (a cast over 32 bits would round twice)"""
    if code == "int8":
        return x.round()
    _, e = torch.frexp(x)
    step = _power((e - 1).clamp(min=-6) - 3).double()
    return (x / step).round() * step


def _plain_attention(s):
    c = s["case"]
    kvh, hd, bs, n_max, longest = c["kv_heads"], c["hd"], c["block"], c["new"], s["longest"]
    heads, group = c["heads"], c["heads"] // c["kv_heads"]
    q, past, new, starts = s["q"], s["past"].long(), s["new"].long(), s["starts"].long()
    rows, dev = past.numel(), q.device
    i = torch.arange(n_max, device=dev)
    at = (starts[:-1, None] + i[None, :]).clamp(max=q.shape[0] - 1)
    x = q[at.reshape(-1)].view(-1, heads, hd).float()
    if s["sin"] is not None:
        x = _rotated(x, s["sin"], s["cos"], (past[:, None] + i[None, :]).clamp(max=s["sin"].shape[0] - 1).reshape(-1))
    x = x.view(rows, n_max, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(rows, kvh, n_max * group, hd)
    width = (longest + bs - 1) // bs
    page = s["table"][:, :width].long()
    known = (page >= 0) & (page < s["ks"].shape[0])
    page = page.clamp(0, s["ks"].shape[0] - 1)
    k = s["kp"].view(torch.uint8)[page].view(CODE[c["code"]]).float()
    k = (k * s["ks"][page][..., None, None])[..., :hd].permute(0, 2, 4, 1, 3).reshape(rows, kvh, hd, width * bs)
    w = torch.matmul(x, k).div_(math.sqrt(hd)).view(rows, kvh, n_max, group, width * bs)
    del k
    j = torch.arange(width * bs, device=dev)
    seen = (j[None, None, :] <= (past[:, None] + i[None, :])[:, :, None]) & (j[None, None, :] < (past + new)[:, None, None])
    seen = (seen & known.repeat_interleave(bs, 1)[:, None, :])[:, None, :, None, :]
    w = w.masked_fill_(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    v = s["vp"].view(torch.uint8)[page].view(CODE[c["code"]]).float()
    v = (v * s["vs"][page][..., None, None])[..., :hd, :].permute(0, 2, 1, 4, 3).reshape(rows, kvh, width * bs, hd)
    tail = (j[None, :] < (past + new)[:, None]) & known.repeat_interleave(bs, 1)
    v = v.masked_fill_(~tail[:, None, :, None], 0.0)      # what lies behind a sequence may be anything
    o = torch.matmul(w.view(rows, kvh, n_max * group, width * bs), v).view(rows, kvh, n_max, group, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(total)).permute(0, 2, 1, 3, 4).reshape(rows, n_max, heads * hd)
    t = torch.arange(q.shape[0], device=dev)
    row = torch.searchsorted(starts[1:], t, right=True).clamp(max=rows - 1)
    inside = (t < starts[-1])[:, None]
    s["out"].copy_(torch.where(inside, o[row, (t - starts[row]).clamp(0, n_max - 1)].half(), s["out"]))
    return s["out"]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------

def work(case):
    ps, ns = _lens(case, 1)
    if case["op"] == "slots":
        rows, t = case["rows"], sum(ns)
        pages = sum((p + n + case["block"] - 1) // case["block"] - p // case["block"] for p, n in zip(ps, ns))
        return {"bytes": 4 * (4 * rows + 2 * (t + case["tail"]) + pages), "flops": 0}
    kvh, hd = case["kv_heads"], case["hd"]
    t = sum(ns)
    if case["op"] == "append":
        pages = sum((p + n + case["block"] - 1) // case["block"] - p // case["block"] for p, n in zip(ps, ns))
        angles = 4 * hd * min(t, max(p + n for p, n in zip(ps, ns))) if case["rope"] else 0
        return {"bytes": t * kvh * hd * 6 + pages * kvh * 8 + t * 8 + angles, "flops": t * kvh * hd * (6 if case["rope"] else 4)}
    keys = sum(p + n for p, n in zip(ps, ns) if n)
    seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(ps, ns))
    return {"bytes": keys * kvh * 2 * hd + 8 * keys // case["block"] * kvh + 4 * t * case["heads"] * hd, "flops": 4 * seen * case["heads"] * hd}


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------------------------

def exact(case, seed):
    def value(x, code):
        """e4m3's or int8's nearest value to each double, ties to even, in numpy"""
        x = np.clip(x, -TOP[code], TOP[code])
        if code == "int8":
            return np.rint(np.nan_to_num(x, nan=0.0))
        step = np.ldexp(1.0, np.maximum(np.frexp(x)[1] - 1, -6) - 3)
        return np.rint(x / step) * step

    def append(s, c):
        code, bs, kvh, hd = c["code"], c["block"], c["kv_heads"], c["hd"]
        slots, pos = s["slots"].cpu().numpy(), s["positions"].cpu().numpy()
        pages = {n: s[n].double().cpu().numpy() for n in ("kp", "vp")}
        scales = {n: s[n].cpu().numpy().astype(np.float64) for n in ("ks", "vs")}
        x = {"kp": s["k"].cpu().numpy().astype(np.float64).reshape(-1, kvh, hd), "vp": s["v"].cpu().numpy().astype(np.float64).reshape(-1, kvh, hd)}
        if s["sin"] is not None:
            sin, cos = (s[n].cpu().numpy().astype(np.float64)[pos][:, None] for n in ("sin", "cos"))
            turned = np.concatenate((-x["kp"][..., hd // 2:], x["kp"][..., :hd // 2]), -1)
            x["kp"] = x["kp"] * cos + turned * sin
        lo, hi = EXP[code]
        t = 0
        while t < len(slots):
            if slots[t] < 0:
                t += 1
                continue
            page, off, n = slots[t] // bs, slots[t] % bs, 1
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] // bs == page:
                n += 1
            for p, q in (("kp", "ks"), ("vp", "vs")):
                new = np.clip(x[p][t:t + n], -TOP[code] * 2.0 ** hi, TOP[code] * 2.0 ** hi)                  # [n, kvh, hd]
                amax = np.abs(new).max((0, 2))
                want = np.array([next(e for e in range(lo, hi + 1) if e == hi or a <= TOP[code] * 2.0 ** e) for a in amax])
                now = np.ldexp(1.0, want)
                body = pages[p][page] if p == "kp" else pages[p][page].transpose(0, 2, 1)                      # [kvh, bs, hd16], a view
                if off:
                    now = np.maximum(now, scales[q][page])
                    body[:, :off] = value(body[:, :off] * (scales[q][page] / now)[:, None, None], code)
                scales[q][page] = now
                body[:, off:off + n, :hd] = value(new / now[None, :, None], code).transpose(1, 0, 2)
                body[:, off:off + n, hd:] = 0
            t += n
        return {"key_pages": None if code == "int8" else pages["kp"], "value_pages": None if code == "int8" else pages["vp"], "key_scales": scales["ks"],
                "value_scales": scales["vs"]}

    def attention(s, c):
        heads, kvh, hd, bs = c["heads"], c["kv_heads"], c["hd"], c["block"]
        past, new, starts = s["past"].tolist(), s["new"].tolist(), s["starts"].tolist()
        out = s["out"].double()
        for b in range(len(past)):
            n, keys = new[b], past[b] + new[b]
            if n == 0:
                continue
            pages = s["table"][b, :(keys + bs - 1) // bs].long()
            q = s["q"][starts[b]:starts[b] + n].double().view(n, heads, hd)
            if s["sin"] is not None:
                turned = torch.cat((-q[..., hd // 2:], q[..., :hd // 2]), -1)
                q = q * s["cos"][past[b]:keys].double()[:, None] + turned * s["sin"][past[b]:keys].double()[:, None]
            hide = torch.arange(keys, device=DEV)[None, :] > past[b] + torch.arange(n, device=DEV)[:, None]
            for g in range(kvh):
                k = s["kp"].view(torch.uint8)[pages, g].view(CODE[c["code"]]).double() * s["ks"][pages, g].double()[:, None, None]
                v = s["vp"].view(torch.uint8)[pages, g].view(CODE[c["code"]]).double() * s["vs"][pages, g].double()[:, None, None]
                k = k.reshape(-1, k.shape[-1])[:keys, :hd]
                v = v.transpose(1, 2).reshape(-1, v.shape[1])[:keys, :hd]
                for h in range(g * heads // kvh, (g + 1) * heads // kvh):
                    w = torch.softmax((q[:, h] @ k.t() / math.sqrt(hd)).masked_fill(hide, -math.inf), -1)
                    out[starts[b]:starts[b] + n, h * hd:(h + 1) * hd] = w @ v
        return out

    if case["op"] == "slots":
        return None                                       # whole numbers: there is nothing to round
    if case["op"] == "append":
        return append(prepare(case, seed), case) if sum(_lens(case, seed)[1]) * case["kv_heads"] * case["hd"] <= 1 << 26 else None
    return attention(prepare(case, seed), case)
