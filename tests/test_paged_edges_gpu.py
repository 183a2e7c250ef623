"""The paged 8-bit cache where it can go wrong without a loose bound noticing: rotated queries beyond fp16's range, small weights in long rows, every key
counted once over all the cuts of a row, and what a rotated query keeps behind fp16's digits."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from test_paged_gpu import DEV, _angles, _attention_case, _dev, _numbers, _pool, _pool_dev, _runs, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext():
    from exllama_amd import cuda_ext
    return cuda_ext


def _attention(ext, host, dev, heads, rope=False, scale=0.0):
    """The call's result as numbers [rows, heads, hd]; NaN in rows that belong to no row of the batch."""
    out = torch.full((host["q"].shape[0], heads * host["q"].shape[2]), float("nan"), dtype=torch.float16, device=DEV)
    ext.ext_paged_attention(dev["q"], dev["starts"], dev["past"], dev["new"], dev["table"], *dev["pool"], heads, max_new=int(host["new"].max()), out=out,
                            scale=scale, **(dict(sin=dev["sin"], cos=dev["cos"]) if rope else {}))
    return out.cpu().double().numpy().reshape(host["q"].shape)


def _sharp(host, bits, rope=True, scale=None, **other):
    args = dict(host, **other)
    return P.attention(args["q"], args["starts"], args["past"], args["new"], args["table"], *args["pool"], int(args["new"].max()), scale=scale, sharp=bits,
                       **(dict(sin=args["sin"], cos=args["cos"]) if rope else {}))


def _rest(hd, heads, kvh, new):
    """The bits that a rotated query keeps: two fp16 numbers, but one where head_dim is over 128 and a row has more than 16 queries for a kv head."""
    return 11 if hd > 128 and new * heads // kvh > 16 else 22


def _set_q(host, dev, q):
    host["q"] = q.astype(np.float16)
    dev["q"] = torch.from_numpy(host["q"]).reshape(len(q), -1).to(DEV)


# ---- numbers at the ends of their ranges --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,heads,kvh,lens", [(128, 4, 2, [(70, 3), (5, 1)]), (128, 4, 1, [(200, 4)]), (256, 2, 2, [(40, 5)]), (256, 4, 2, [(0, 60)]),
                                               (100, 4, 2, [(30, 6)]), (64, 4, 2, [(90, 70)]), (128, 8, 2, [(600, 40), (3, 9)])])
def test_rotated_queries_beyond_fp16(ext, code, hd, heads, kvh, lens):
    """A rotated element is up to sqrt(2) times as large as fp16's largest number; its keys are small, so that the scores are ordinary ones."""
    rng = np.random.default_rng(hd + heads)
    host, dev = _attention_case(rng, code, hd, heads, kvh, 16, lens)
    q, half = host["q"].astype(np.float64), hd // 2
    for c in (0, 1, half - 1):
        some = rng.random(q.shape[:2]) < 0.5
        q[some, c], q[some, c + half] = 60000.0 * rng.choice([-1, 1], int(some.sum())), 61000.0 * rng.choice([-1, 1], int(some.sum()))
        small = rng.integers(-3, 4, host["pool"][0][..., 0].shape)
        for k in (c, c + half):
            host["pool"][0][..., k] = np.where(np.isnan(host["pool"][0][..., k]), np.nan, small * (2.0 ** -9 if code == "fp8" else 1.0))
    host["pool"][2] = np.ldexp(1.0, rng.integers(-9, -6, host["pool"][2].shape) - (5 if code == "int8" else 0))
    dev["pool"] = _pool_dev(host["pool"], code)
    _set_q(host, dev, q)
    turned = P.rotate(host["q"][:lens[0][1]].astype(np.float64), host["sin"], host["cos"], lens[0][0] + np.arange(lens[0][1]))
    want, bound = _sharp(host, _rest(hd, heads, kvh, int(host["new"].max())))
    got, some = _attention(ext, host, dev, heads, rope=True), ~np.isnan(bound)
    assert np.abs(turned).max() > 65520
    assert np.isfinite(got[some]).all()
    assert (np.abs(got - want)[some] <= bound[some]).all()


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("below", [17.5, 19.5, 22.5])
@pytest.mark.parametrize("new", [1, 40])
def test_many_small_weights_beside_a_large_one(ext, code, below, new):
    """One key, the row's first, with a score of 0, 65535 others `below` powers of two under it and with values of 1: together they are a tenth of the result, or
    a quarter, or a hundredth.  64 rows of 32 heads, all on the same pages, so that no wave and no workgroup begins in the middle of one."""
    hd, heads, keys, block, n = 64, 32, 65536, 128, 64
    blocks, kind = keys // block, {"fp8": torch.float8_e4m3fn, "int8": torch.int8}[code]
    kp = torch.zeros(blocks, heads, block, hd, dtype=torch.float32, device=DEV)
    kp[..., 0] = -16
    kp[0, :, 0, 0] = 0
    kp = kp.to(kind)
    vp = torch.ones(blocks, heads, hd, block, dtype=torch.float32, device=DEV)
    vp[0, :, :, 0] = 0
    vp = vp.to(kind)
    scales = torch.ones(blocks, heads, device=DEV)
    q = torch.zeros(n * new, heads, hd, dtype=torch.float16, device=DEV)
    q[..., 0] = below / 16                                    # (exact)
    past = np.full(n, keys - new)
    out = ext.ext_paged_attention(q.view(n * new, -1), _dev(np.arange(n + 1) * new), _dev(past), _dev(np.full(n, new)),
                                  _dev(np.tile(np.arange(blocks), (n, 1))), kp, vp, scales, scales, heads, max_new=new, scale=float(np.log(2)))
    others = (keys - new + np.arange(new)) * 2.0 ** -below
    want = np.tile(others / (1 + others), n)[:, None, None]
    # a weight's rounding, the same for all of them (2^-11), the result's (2^-11), the scores' (2^-20 each with log 2 in 32 bits), and the sums', at most 2^-24
    # each and all to one side: the denominator's of 1024 tiles (2^-14), the product's of 4096 steps of 16 keys (2^-12)
    tol = 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -18 + 2.0 ** -14 + 2.0 ** -12
    got = out.view(n * new, heads, hd).cpu().double().numpy()
    assert np.abs(got / want - 1).max() <= tol


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,heads,kvh,lens", [(128, 4, 2, [(130, 3), (5, 1)]), (64, 4, 2, [(90, 70)]), (256, 4, 2, [(700, 40)]), (128, 2, 2, [(2000, 1)])])
def test_scores_beyond_every_ordinary_size(ext, code, hd, heads, kvh, lens):
    """Scores of 2^29 and more, where neighbours in 32 bits lie 32 apart: the largest takes all the weight, and nothing overflows."""
    rng = np.random.default_rng(hd + heads)
    host, dev = _attention_case(rng, code, hd, heads, kvh, 16, lens)
    _set_q(host, dev, rng.choice([-1.0, 1.0], host["q"].shape) * rng.integers(20000, 60000, host["q"].shape))
    host["pool"][2][:] = 2.0 ** P.EXP[code][1]
    dev["pool"] = _pool_dev(host["pool"], code)
    want, _ = _sharp(host, 22, rope=False)
    got, some = _attention(ext, host, dev, heads), ~np.isnan(want)
    assert np.isfinite(got[some]).all()
    # one key takes all: its value to fp16 (2^-11) and by a quotient (2^-23) -- where the first two scores lie far apart for 32 bits
    top = np.full(want.shape[:2], np.inf)
    for b, (past, new) in enumerate(lens):
        for i in range(new):
            j = np.arange(past + i + 1)
            page = host["table"][b][j // 16]
            for h in range(heads):
                g = h * kvh // heads
                s = np.sort((host["pool"][0][page, g, j % 16, :hd] * host["pool"][2][page, g][:, None]) @ host["q"][host["starts"][b] + i, h].astype(np.float64))
                s *= hd ** -0.5
                # (a score's terms are summed in 32 bits: 2 hd roundings of 2^-24 of what they add up to, at most hd * 2^16 * 2^16 / sqrt(hd))
                top[host["starts"][b] + i, h] = (s[-1] - s[-2] if len(s) > 1 else np.inf) / (2 * hd * 2.0 ** -24 * hd ** 0.5 * 2.0 ** 32)
    sure = some & (top > 2)[..., None]
    assert sure.any() and (np.abs(got - want)[sure] <= 2.0 ** -10 * np.abs(want[sure]) + 2.0 ** -25).all()


# ---- every key, once ----------------------------------------------------------------------------------------------------------------------

# few queries: in one stretch, in several, several rows in one; single tokens and drafts; many: in one piece and in several, beside short rows
EVERY = [(128, 32, 32, 64, [(2047, 1)]), (128, 16, 2, 32, [(5000, 1), (100, 1), (2000, 1), (0, 1)]), (64, 4, 2, 16, [(777, 5), (63, 3), (64, 2), (0, 5)]),
         (256, 4, 2, 128, [(3000, 2), (1, 2)]), (128, 8, 1, 64, [(6000, 4)]), (100, 8, 8, 16, [(1300, 1), (62, 1), (63, 1), (64, 1)]),
         (128, 8, 8, 16, [(191 + 37 * i, 1) for i in range(60)]), (128, 4, 4, 64, [(9000, 1)]), (64, 64, 64, 32, [(3000, 1), (40, 0), (2999, 1)]),
         (128, 8, 1, 64, [(6000, 20)]), (128, 4, 4, 64, [(0, 700), (1500, 90)]), (256, 4, 2, 128, [(1000, 129), (50, 1)]), (64, 4, 4, 16, [(2300, 40), (7, 1)]),
         (128, 16, 2, 16, [(200, 300), (3, 260)]), (100, 4, 2, 32, [(4100, 33), (60, 257)])]


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("equal", [True, False])
@pytest.mark.parametrize("hd,heads,kvh,block,lens", EVERY)
def test_every_key_counts_once(ext, code, equal, hd, heads, kvh, block, lens):
    """A key's value is 1 in two columns, of its place in its tile of 64 and of its tile, and 0 elsewhere; its score is a whole power of two (0, or -12 .. 12 drawn
    for the key, so that the softmax's reference moves).  Every weight is then an fp16 number, a column is the sum of one class of keys over the
    sum of all, and a tile that is lost or taken twice anywhere changes its column by far more than the roundings."""
    rng = np.random.default_rng(hd + len(lens))
    host, dev = _attention_case(rng, code, hd, heads, kvh, block, lens)
    kc, vc, ks, vs = host["pool"]
    half = hd // 2
    power = {}
    for b, (past, new) in enumerate(lens):
        j = np.arange(past + new)
        page, off = host["table"][b][j // block], j % block
        power[b] = np.zeros(len(j)) if equal else np.clip(rng.integers(-6, 7, len(j) // 64 + 1)[j // 64] + rng.integers(-6, 7, len(j)), -12, 12)
        kc[page, :, off] = 0.0
        vc[page, :, :, off] = 0.0
        kc[page, :, off, 0] = power[b][:, None]
        vc[page, :, (j % 64) % half, off] = 64.0
        vc[page, :, half + (j // 64) % half, off] = 64.0
    ks[:] = 1.0
    vs[:] = 2.0 ** 7
    dev["pool"] = _pool_dev(host["pool"], code)
    q = np.zeros(host["q"].shape)
    q[..., 0] = 1.0
    _set_q(host, dev, q)
    got = _attention(ext, host, dev, heads, scale=float(np.log(2)))
    for b, (past, new) in enumerate(lens):
        if not new:
            continue
        j = np.arange(past + new)
        w = np.zeros((len(j), hd))
        w[j, (j % 64) % half] += 2.0 ** power[b]
        w[j, half + (j // 64) % half] += 2.0 ** power[b]
        want = 2.0 ** 13 * (np.cumsum(w, 0) / np.cumsum(2.0 ** power[b])[:, None])[past:]
        x = got[host["starts"][b]:host["starts"][b] + new]
        # the result's rounding (2^-11; 2^-25 below fp16's normal range), sums of positive numbers in 32 bits (a lane adds a quarter of the keys: at most
        # 2^-26 of the sum for each key, numerator and denominator) and exp2 (2^-21 for scores that log 2 in 32 bits makes 2^-20 off at most)
        tol = 2.0 ** -11 + len(j) * 2.0 ** -25 + 2.0 ** -18
        assert (np.abs(x - want[:, None]) <= tol * want[:, None] + 2.0 ** -25).all(), (b, past, new)


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,heads,kvh,block,lens,spread,bites", [
    (128, 4, 2, 16, [(60, 8), (5, 3)], 8, True), (128, 4, 2, 64, [(10, 40)], 8, True), (128, 4, 2, 64, [(100, 40)], 32, True), (64, 4, 2, 32, [(10, 40)], 8, True),
    (100, 4, 2, 16, [(10, 40)], 16, True), (100, 4, 4, 16, [(20, 6), (9, 1)], 16, True), (256, 2, 2, 64, [(10, 7)], 4, False), (256, 4, 2, 64, [(200, 40)], 2, False),
    (128, 8, 1, 64, [(6000, 20)], 2, False), (128, 4, 4, 64, [(9000, 1)], 2, False), (128, 16, 2, 32, [(5000, 1), (100, 1), (2000, 1)], 2, False)])
def test_a_rotated_query_keeps_what_fp16_leaves(ext, code, hd, heads, kvh, block, lens, spread, bites):
    """Against the bound of a kernel that holds a rotated query to 22 bits.  `bites`: the formula with the rotated query rounded to fp16 breaks that bound, so
    that a kernel which drops the rest fails."""
    spread *= 1 if code == "fp8" else 3                       # (int8 codes are a third as large)
    host, dev = _attention_case(np.random.default_rng(1), code, hd, heads, kvh, block, lens, spread=spread)
    want, bound = _sharp(host, _rest(hd, heads, kvh, int(host["new"].max())))
    some = ~np.isnan(bound)
    if bites:
        rounded = host["q"].astype(np.float64)
        for b, (past, new) in enumerate(lens):
            rows = slice(host["starts"][b], host["starts"][b] + new)
            rounded[rows] = P.rotate(rounded[rows], host["sin"], host["cos"], past + np.arange(new)).astype(np.float16)
        off, _ = _sharp(host, 22, rope=False, q=rounded)
        assert (np.abs(off - want)[some] > bound[some]).mean() > 0.005
    got = _attention(ext, host, dev, heads, rope=True)
    assert (np.abs(got - want)[some] <= bound[some]).all()


# ---- append: every number of rows that a workgroup can take ---------------------------------------------------------------------------------

@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,kvh,block,spec", [
    (64, 8, 16, [(0, 900), (-1, -5), (3, 700), (15, 2)] + [(9, 1)] * 70 + [(0, 300)]),                   # 16000 token rows * heads: 16 rows a workgroup
    (64, 8, 32, [(0, 2000), (-1, -3), (31, 1500)] + [(9, 1)] * 50 + [(5, 9), (1, 2)]),                   # 28600: 32 rows
    (100, 8, 16, [(0, 900), (-1, -5), (3, 700), (15, 2)] + [(9, 1)] * 70), (100, 4, 128, [(7, 5000), (-1, -70), (0, 1), (120, 60)]),
    (16, 32, 64, [(0, 700), (63, 1), (0, 64), (1, 63)] + [(60, 9)] * 9)])
def test_append_of_every_chunk(ext, code, hd, kvh, block, spec):
    rng = np.random.default_rng(hd + kvh)
    blocks = sum(-(-(o % block + n) // block) for o, n in spec if n > 0) + 2
    pool = _pool(rng, blocks, kvh, block, hd, code)
    dev = _pool_dev(pool, code)
    slots, pos = _runs(rng, blocks, block, spec)
    t = len(slots)
    x = (rng.normal(0, 1, (2, t, kvh, hd)) * np.exp(rng.normal(0, 1.5, (2, 1, kvh, hd)))).astype(np.float16)
    sin, cos = _angles(6000, hd)
    ext.ext_paged_append(*(torch.from_numpy(y).reshape(t, -1).to(DEV) for y in x), _dev(slots), *dev, positions=_dev(pos), sin=sin.to(DEV), cos=cos.to(DEV))
    P.append(x[0], x[1], slots, *pool, code, pos, sin.numpy(), cos.numpy())
    for name, got, want in zip(("keys", "values", "key scales", "value scales"), dev, pool):
        assert _same(_numbers(got), want), name


# ---- pools that run dry ---------------------------------------------------------------------------------------------------------------------

class _Dry:
    """Three rows on a pool of six pages of 16 that hold another sequence's leavings, NaN among them."""

    def __init__(self, rng):
        self.rng, self.hd, self.kvh, self.heads, self.block = rng, 64, 2, 4, 16
        codes = P.nearest(rng.normal(0, 100, (6, 2, 16, 64)), "fp8"), P.nearest(rng.normal(0, 100, (6, 2, 64, 16)), "fp8")
        for c in codes:
            c[rng.random(c.shape) < 0.3] = np.nan
        self.pool = [codes[0], codes[1], np.full((6, 2), 2.0 ** 7), np.full((6, 2), 2.0 ** 7)]
        self.dpool = _pool_dev(self.pool, "fp8")
        self.past, self.held, self.counters = np.zeros(3, np.int32), np.zeros(3, np.int32), np.array([0, 6, 0, 0], np.int32)
        self.table, self.ring = np.full((3, 5), -1, np.int32), rng.permutation(6).astype(np.int32)
        self.d = {k: _dev(getattr(self, k)) for k in ("past", "held", "table", "ring", "counters")}

    def step(self, ext, new, max_len=80, check=True):
        """One pass; returns (slots, the result) and, with `check`, holds both against the oracle."""
        rows = int(np.maximum(new, 0).sum())
        q, k, v = (self.rng.normal(0, 1, (rows, h, self.hd)).astype(np.float16) for h in (self.heads, self.kvh, self.kvh))
        dq, dk, dv = (torch.from_numpy(x).reshape(rows, x.shape[1] * self.hd).to(DEV) for x in (q, k, v))
        dnew, top = _dev(new), max(int(np.max(new)), 1)
        starts, slots, _ = ext.ext_paged_slots(self.d["past"], dnew, self.d["held"], self.d["table"], self.d["ring"], self.d["counters"], 16, rows, max_new=top,
                                               max_len=max_len)
        ext.ext_paged_append(dk, dv, slots, *self.dpool)
        fits = torch.minimum(dnew.clamp(min=0), (max_len - self.d["past"]).clamp(min=0))
        out = ext.ext_paged_attention(dq, starts, self.d["past"], fits, self.d["table"], *self.dpool, self.heads, max_new=top)
        got = out.cpu().double().numpy().reshape(rows, self.heads, self.hd)
        if check:
            s, want_slots, _ = P.slots(self.past, new, self.held, self.table, self.ring, self.counters, 16, max_len, top, rows)
            P.append(k, v, want_slots, *self.pool, "fp8")
            want, bound = P.attention(q, s, self.past, fits.cpu().numpy(), self.table, *self.pool, top)
            for name in ("held", "table", "ring", "counters"):
                assert np.array_equal(self.d[name].cpu().numpy(), getattr(self, name)), name
            assert np.array_equal(slots.cpu().numpy(), want_slots)
            some = ~np.isnan(bound)
            assert (np.abs(got - want)[some] <= bound[some]).all()
        assert np.isfinite(got).all()
        return slots.cpu().numpy(), got


def test_a_row_that_lost_tokens_reads_no_other_rows_pages(ext):
    """past_lens advanced by all of new_lens although the pool ran dry: when pages come free again, the row gets none of them, and every result is
    that of the keys it holds; set back to what it holds, it goes on."""
    dry = _Dry(np.random.default_rng(0))

    def blindly(new):
        dry.past += np.maximum(new, 0).astype(np.int32)
        dry.past[new < 0] = 0
        dry.d["past"].copy_(_dev(dry.past))

    for new in ([40, 30, 10], [1, 1, 1], [0, 5, 6], [1, 1, 1]):       # 3 + 2 + 1 pages: all; then row 1 and row 2 lose tokens
        dry.step(ext, np.array(new))
        blindly(np.array(new))
    assert dry.held.tolist() == [3, 2, 1] and dry.past.tolist() == [42, 37, 18]
    dry.step(ext, np.array([-1, 0, 0]))                               # three pages come free
    blindly(np.array([-1, 0, 0]))
    held = dry.held.copy()
    for new in ([0, 1, 1], [0, 0, 2], [20, 1, 3]):
        slots, _ = dry.step(ext, np.array(new))
        blindly(np.array(new))
        assert (slots[new[0]:] == -1).all() and dry.counters[2] > 0
    assert (dry.held[1:] == held[1:]).all()
    dry.past[:] = np.minimum(dry.past, dry.held * 16)                 # set back
    dry.d["past"].copy_(_dev(dry.past))
    dry.step(ext, np.array([0, 1, 0]))
    assert dry.held[1] == held[1] + 1


def test_lengths_that_advance_by_what_was_placed(ext):
    """The rule for a step on the device: past = min(past + new, held * block, max_len).  A row that is short of pages or at max_len (which cuts a page) stays
    where it is, and goes on when it can."""
    dry = _Dry(np.random.default_rng(1))
    for new in ([40, 30, 10], [9, 5, 1], [1, 5, 6], [1, 1, 1], [-1, 1, 1], [0, 9, 9], [0, 1, 9], [30, 9, 9], [1, 1, 1]):
        new = np.array(new)
        slots, _ = dry.step(ext, new, max_len=44)
        d = dry.d
        taken = _dev(new).clamp(min=0)
        d["past"].copy_(torch.minimum(torch.minimum(d["past"] + taken, d["held"] * 16), torch.full_like(taken, 44)))
        placed = np.array([(slots[s:s + n] >= 0).sum() for s, n in zip(np.cumsum(np.maximum(new, 0)) - np.maximum(new, 0), np.maximum(new, 0))])
        dry.past = np.where(new < 0, 0, dry.past + placed).astype(np.int32)
        assert d["past"].tolist() == dry.past.tolist()
    assert dry.past.max() == 44


@pytest.mark.parametrize("n,rows,stride", [(3, 40, 0), (64, 300, 0), (65, 300, 0), (300, 1000, 0), (512, 4096, 0), (513, 2000, 0), (300, 5000, 0), (2100, 9000, 0),
                                           (5000, 20000, 0), (300, 300 * 4, 4), (700, 700 * 4, 4)])
def test_slots_of_rows_that_lost_tokens(ext, n, rows, stride):
    """Lengths beyond the held blocks in a third of the rows, among ended, idle and ordinary ones: in one workgroup's wave, in all of its waves, and in the scan
    of its own launch, once around and twice."""
    for seed in range(3):
        rng = np.random.default_rng(seed)
        width, block, spare = 9, 16, 2 * n
        held = rng.integers(0, 7, n).astype(np.int32)
        past = np.maximum(held * block - rng.integers(0, block, n), 0)
        past = np.where(rng.random(n) < 0.3, held * block + rng.integers(1, 40, n), past)
        new = rng.integers(0, 5, n)
        new[rng.random(n) < 0.2] = 0
        new[rng.random(n) < 0.1] = -1
        blocks = int(held.sum()) + spare
        order = rng.permutation(blocks)
        table, at = np.full((n, width), -1, np.int32), 0
        for b in range(n):
            table[b, :held[b]] = order[at:at + held[b]]
            at += held[b]
        head = int(rng.integers(blocks))
        ring = np.full(blocks, -7, np.int32)
        ring[(head + np.arange(spare)) % blocks] = order[at:]
        counters = np.array([head, spare, 0, 0], np.int32)
        d = [_dev(x) for x in (past, new, held, table, ring, counters)]
        got = ext.ext_paged_slots(*d, block, rows, max_new=4, row_stride=stride)
        want = P.slots(past, new, held, table, ring, counters, block, width * block, 4, rows, stride)
        for name, x, y in zip(("starts", "slots", "positions", "held", "table", "ring", "counters"), (*got, *d[2:]), (*want, held, table, ring, counters)):
            assert np.array_equal(x.cpu().numpy(), y), (name, seed)
        assert n < 60 or counters[2] > 0


# ---- tensors at other addresses -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd", [128, 100])
def test_angles_that_begin_anywhere(ext, hd):
    """sin and cos tables at an odd element of a buffer: the same results to the bit."""
    rng = np.random.default_rng(hd)
    host, dev = _attention_case(rng, "fp8", hd, 4, 2, 16, [(70, 3), (5, 20)])
    x = [torch.from_numpy(rng.normal(0, 1, (23, 2 * hd)).astype(np.float16)).to(DEV) for _ in range(2)]
    slots = _dev(np.r_[np.arange(3) + 5, np.arange(20) + 32])
    results = []
    for at in (0, 1, 3):
        sin, cos = (torch.cat((t.new_zeros(at), t.flatten()))[at:].view(t.shape) for t in (dev["sin"], dev["cos"]))
        assert sin.data_ptr() % 16 == 2 * at
        pool = [p.clone() for p in dev["pool"]]
        ext.ext_paged_append(*x, slots, *pool, positions=_dev(np.r_[np.arange(3) + 70, np.arange(20) + 5]), sin=sin, cos=cos)
        out = ext.ext_paged_attention(dev["q"], dev["starts"], dev["past"], dev["new"], dev["table"], *dev["pool"], 4, max_new=20, sin=sin, cos=cos)
        one = ext.ext_paged_attention(dev["q"], dev["starts"], dev["past"], _dev([3, 1]), dev["table"], *dev["pool"], 4, max_new=3, sin=sin, cos=cos)
        results.append([out, one] + [p.view(torch.uint8) for p in pool])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
