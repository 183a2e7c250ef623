"""The paged 8-bit cache on the GPU against its 64-bit oracle: block tables and slot maps (equal), the append (equal to the bit) and attention
(within the bound that the oracle derives from fp16 roundings and fp32 sums), alone and together as a serving loop runs them."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

TYPE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ext():
    from exllama_amd import cuda_ext
    return cuda_ext


def _dev(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).to(DEV)


def _to_type(codes, code):
    """numbers -> pages on the device"""
    return torch.from_numpy(np.ascontiguousarray(codes)).float().to(TYPE[code]).to(DEV)


def _numbers(pages):
    return pages.cpu().float().double().numpy()


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def _angles(n, hd):
    f = np.arange(n)[:, None] / 10000.0 ** (np.arange(0, hd, 2) / hd)[None, :]
    f = np.concatenate((f, f), 1)
    return torch.from_numpy(np.sin(f)).half(), torch.from_numpy(np.cos(f)).half()


# ---- block tables and slot maps -------------------------------------------------------------------------------------------------------

def _slot_case(rng, n, width, block, max_past, max_new, spare, ended=0.1, hold=0.2):
    past = rng.integers(0, max_past + 1, n)
    new = rng.integers(0, max_new + 1, n)
    held = np.minimum(-(-past // block) + (rng.random(n) < hold), width)
    new[rng.random(n) < ended] = -1
    blocks = int(held.sum()) + spare
    order = rng.permutation(blocks)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for b in range(n):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    head = int(rng.integers(blocks))
    ring = np.full(blocks, -7, np.int32)
    ring[(head + np.arange(spare)) % blocks] = order[at:]
    return past, new, held.astype(np.int32), table, ring, np.array([head, spare, 0, 0], np.int32)


@pytest.mark.parametrize("n,width,block,past,new,spare,rows,stride", [
    (1, 1, 16, 0, 1, 1, 1, 0), (1, 40, 64, 2047, 1, 2, 1, 0), (3, 9, 16, 100, 40, 30, 200, 0), (65, 12, 32, 200, 100, 400, 5000, 0),
    (256, 130, 64, 8000, 1, 300, 256, 0), (1025, 7, 16, 60, 50, 3000, 40000, 0), (2100, 3, 128, 200, 1, 2000, 2000, 0),
    (7, 20, 16, 100, 30, 60, 7 * 30, 30), (1500, 5, 32, 100, 5, 1500, 1500 * 4, 4),
    (40, 10, 16, 100, 60, 3, 3000, 0),                        # the ring runs dry
    (40, 4, 16, 60, 60, 200, 3000, 0),                        # rows outgrow their table
    (30, 20, 16, 100, 60, 200, 333, 0), (9, 20, 16, 50, 60, 90, 100, 12)])   # token rows run out
def test_slots(ext, n, width, block, past, new, spare, rows, stride):
    for seed in range(3):
        rng = np.random.default_rng(seed)
        past_l, new_l, held, table, ring, counters = _slot_case(rng, n, width, block, min(past, width * block), new, spare, ended=0.0 if n == 1 else 0.1)
        max_len = width * block - int(rng.integers(0, block))
        max_new = max(1, new - int(rng.integers(0, 2)))
        d = {k: _dev(v) for k, v in (("past", past_l), ("new", new_l), ("held", held), ("table", table), ("ring", ring), ("counters", counters))}
        for again in range(2):                                # the second call finds the blocks there (or takes those that the first gave back)
            want = P.slots(past_l, new_l, held, table, ring, counters, block, max_len, max_new, rows, stride)
            got = ext.ext_paged_slots(d["past"], d["new"], d["held"], d["table"], d["ring"], d["counters"], block, rows, max_new=max_new,
                                      max_len=max_len, row_stride=stride)
            for name, x, y in (("starts", got[0], want[0]), ("slots", got[1], want[1]), ("positions", got[2], want[2]), ("held", d["held"], held),
                               ("table", d["table"], table), ("ring", d["ring"], ring), ("counters", d["counters"], counters)):
                assert np.array_equal(x.cpu().numpy(), y), (name, seed, again)


# ---- append ---------------------------------------------------------------------------------------------------------------------------

def _pool(rng, blocks, kvh, block, hd, code):
    hd16 = (hd + 15) // 16 * 16
    lo, hi = P.EXP[code]
    kc, vc = (P.nearest(rng.normal(0, P.TOP[code] / 3, s), code) for s in ((blocks, kvh, block, hd16), (blocks, kvh, hd16, block)))
    kc[..., hd:] = 0
    vc[..., hd:, :] = 0
    ks, vs = (np.ldexp(1.0, rng.integers(-9, -5, (blocks, kvh))) for _ in range(2))
    return [kc, vc, ks, vs]


def _pool_dev(pool, code):
    return [_to_type(pool[0], code), _to_type(pool[1], code), _dev(pool[2], torch.float32), _dev(pool[3], torch.float32)]


def _runs(rng, blocks, block, spec):
    """Slots of runs [(offset, tokens)], each from a page of its own on (over as many pages as it takes), with skipped rows between."""
    pages, slots, pos = list(rng.permutation(blocks)), [], []
    for off, n in spec:
        if n < 0:
            slots += [-1] * -n
            pos += [0] * -n
            continue
        page = None
        for i in range(n):
            if page is None or (off + i) % block == 0:
                page = pages.pop()
            slots.append(page * block + (off + i) % block)
            pos.append(off + i)
    return np.array(slots), np.array(pos)


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,kvh,block,spec,rope", [
    (128, 8, 64, [(0, 1)], True), (128, 2, 16, [(5, 1), (15, 1), (0, 1), (9, 1)], True), (64, 3, 32, [(0, 100), (-1, -3), (31, 2), (7, 70)], True),
    (100, 4, 16, [(3, 40), (0, 16), (0, 1)], True), (80, 1, 128, [(0, 128), (100, 60)], False), (256, 2, 64, [(60, 9), (0, 64), (-1, -1)], True),
    (4, 5, 16, [(0, 3), (15, 18)], True), (128, 32, 64, [(0, 200)], False), (20, 2, 128, [(64, 64), (127, 130)], True),
    (16, 3, 128, [(0, 128), (90, 50), (1, 1)], True), (48, 2, 32, [(2, 30), (0, 9), (31, 40)], True), (240, 1, 128, [(0, 128), (127, 9)], True),
    (96, 40, 64, [(0, 700), (-1, -40), (9, 8)], False)])
def test_append(ext, code, hd, kvh, block, spec, rope):
    rng = np.random.default_rng(hd + kvh)
    pool = _pool(rng, 16, kvh, block, hd, code)
    dev = _pool_dev(pool, code)
    slots, pos = _runs(rng, 16, block, spec)
    t = len(slots)
    x = (rng.normal(0, 1, (2, t, kvh, hd)) * np.exp(rng.normal(0, 1.5, (2, 1, kvh, hd)))).astype(np.float16)
    x[:, rng.random(t) < 0.2] *= 30                            # tokens that raise their page's scale
    sin, cos = _angles(800, hd)
    wide = torch.zeros(t, 2 * kvh * hd + 4, dtype=torch.float16, device=DEV)      # keys and values as two views of one projection's output
    k, v = wide[:, 4:4 + kvh * hd], wide[:, 4 + kvh * hd:]
    k.copy_(torch.from_numpy(x[0]).reshape(t, -1))
    v.copy_(torch.from_numpy(x[1]).reshape(t, -1))
    kw = dict(positions=_dev(pos), sin=sin.to(DEV), cos=cos.to(DEV)) if rope else {}
    for again in range(2):                                    # (the second time nothing may move: the scales already hold)
        ext.ext_paged_append(k, v, _dev(slots), *dev, **kw)
        P.append(x[0], x[1], slots, *pool, code, pos, *((sin.numpy(), cos.numpy()) if rope else (None, None)))
        for name, got, want in zip(("keys", "values", "key scales", "value scales"), dev, pool):
            assert _same(_numbers(got), want), (name, again)


@pytest.mark.parametrize("code", ["fp8", "int8"])
def test_append_of_values_at_the_borders(ext, code):
    """Zeros, subnormals, the largest finite numbers, infinities and NaN; and halfway points of every scale."""
    rng = np.random.default_rng(3)
    hd, block = 64, 16
    rows = [np.zeros(hd), np.full(hd, 2.0 ** -24), np.r_[65504.0, -65504.0, np.linspace(-60000, 60000, hd - 2)], np.r_[np.inf, -np.inf, np.ones(hd - 2)],
            np.r_[np.nan, np.linspace(-1, 1, hd - 1)], np.full(hd, np.nan), np.r_[448.0, np.arange(hd - 1) / 8 + 16], np.r_[449.0, np.arange(hd - 1) / 8 + 16],
            np.r_[127.0, np.arange(hd - 1) - 30.5], np.r_[127.5, np.arange(hd - 1) - 30.5], np.r_[2.0 ** -14, np.arange(hd - 1) * 2.0 ** -24]]
    x = np.stack([np.stack(rows), np.stack(rows[::-1])]).astype(np.float16)[:, :, None]
    t = len(rows)
    for slots in (np.arange(t) * block, np.arange(t) + 2 * block, np.arange(t)[::-1] * block + 7):       # a page each, one page, behind kept tokens
        pool = _pool(rng, t, 1, block, hd, code)
        dev = _pool_dev(pool, code)
        ext.ext_paged_append(_dev(x[0, :, 0], torch.float16), _dev(x[1, :, 0], torch.float16), _dev(slots), *dev)
        P.append(x[0], x[1], slots, *pool, code)
        for name, got, want in zip(("keys", "values", "key scales", "value scales"), dev, pool):
            assert _same(_numbers(got), want), name


def test_append_leaves_the_rest(ext):
    """Slots outside the pool, and every byte that belongs to no new token (behind the run, other pages), stay as they were."""
    rng = np.random.default_rng(4)
    pool = _pool(rng, 5, 2, 32, 64, "fp8")
    dev = _pool_dev(pool, "fp8")
    before = [x.clone() for x in dev]
    x = torch.randn(4, 128, dtype=torch.float16, device=DEV)
    ext.ext_paged_append(x, x, _dev([-1, 5 * 32, 2 ** 31 - 1, -2 ** 31]), *dev)
    for a, b in zip(before, dev):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    ext.ext_paged_append(x[:1], x[:1], _dev([2 * 32 + 9]), *dev)
    bits = [(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, dev)]
    (k0, k1), (v0, v1) = bits[:2]
    for a, b in ((k0, k1), (v0, v1)):
        assert torch.equal(a[[0, 1, 3, 4]], b[[0, 1, 3, 4]])
    assert torch.equal(k0[2, :, 10:], k1[2, :, 10:]) and torch.equal(v0[2, :, :, 10:], v1[2, :, :, 10:])


# ---- attention ------------------------------------------------------------------------------------------------------------------------

def _attention_case(rng, code, hd, heads, kvh, block, lens, tail=2, blocks_more=3, spread=1.0):
    """lens: [(past, new)]; returns (host, device) dicts."""
    n = len(lens)
    width = max(1, max(-(-(p + m) // block) for p, m in lens))
    need = [-(-(p + m) // block) for p, m in lens]
    blocks = sum(need) + blocks_more
    order = rng.permutation(blocks)
    table, at = np.full((n, width), -1, np.int32), 0
    for b in range(n):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    pool = _pool(rng, blocks, kvh, block, hd, code)
    # what lies behind the sequences may be anything: NaN codes, other rows' leavings
    for b, (p, m) in enumerate(lens):
        off = (p + m) % block
        if off:
            pool[0][table[b, need[b] - 1], :, off:] = np.nan if code == "fp8" else 127
            pool[1][table[b, need[b] - 1], :, :, off:] = np.nan if code == "fp8" else 127
    for page in order[at:]:
        pool[0][page] = pool[1][page] = np.nan if code == "fp8" else 127
    new = np.array([m for _, m in lens])
    starts = np.concatenate(([0], np.cumsum(new)))
    q = (rng.normal(0, spread, (int(starts[-1]) + tail, heads, hd))).astype(np.float16)
    sin, cos = _angles(max(p + m for p, m in lens) + 1, hd)
    host = dict(q=q, starts=starts, past=np.array([p for p, _ in lens]), new=new, table=table, pool=pool, sin=sin.numpy(), cos=cos.numpy(), width=width)
    dev = dict(q=torch.from_numpy(q).reshape(len(q), -1).to(DEV), starts=_dev(starts), past=_dev(host["past"]), new=_dev(new), table=_dev(table),
               pool=_pool_dev(pool, code), sin=sin.to(DEV), cos=cos.to(DEV))
    return host, dev


def _check_attention(ext, host, dev, heads, rope, max_new=None, q=None, scale=0.0, tag=""):
    rows = host["q"].shape[0]
    max_new = int(host["new"].max()) if max_new is None else max_new
    out = torch.full((rows, host["q"].shape[1] * host["q"].shape[2]), 7.5, dtype=torch.float16, device=DEV)
    kw = dict(sin=dev["sin"], cos=dev["cos"]) if rope else {}
    ext.ext_paged_attention(dev["q"] if q is None else q, dev["starts"], dev["past"], dev["new"], dev["table"], *dev["pool"], heads, max_new=max_new,
                            out=out, scale=scale, **kw)
    want, bound = P.attention(host["q"], host["starts"], host["past"], host["new"], host["table"], *host["pool"], max_new, scale=scale,
                              **(dict(sin=host["sin"], cos=host["cos"]) if rope else {}))
    got = out.cpu().double().numpy().reshape(want.shape)
    none = np.isnan(bound).all((1, 2))
    assert (got[none] == 7.5).all(), (tag, "rows of no sequence were written")
    assert np.isfinite(got[~none]).all(), (tag, "not finite")
    worst = float((np.abs(got - want)[~none] / np.maximum(bound[~none], 1e-30)).max()) if (~none).any() else 0.0
    assert worst <= 1.0, (tag, worst)
    return out


SHAPES = [(128, 32, 32), (128, 8, 1), (128, 64, 8), (64, 6, 2), (100, 4, 4), (80, 8, 8), (256, 4, 2), (128, 40, 1), (4, 2, 1), (128, 3, 1)]


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,heads,kvh", SHAPES)
def test_attention_of_single_tokens(ext, code, hd, heads, kvh):
    for seed, (block, lens) in enumerate([(16, [(0, 1)]), (64, [(63, 1), (64, 1), (0, 1), (500, 0), (130, 1)]), (32, [(31, 1), (5, 1), (300, 1)]),
                                          (128, [(255, 1), (256, 1), (1, 1)]), (16, [(1100, 1), (3, 1), (17, 1)])]):
        host, dev = _attention_case(np.random.default_rng(seed), code, hd, heads, kvh, block, lens)
        _check_attention(ext, host, dev, heads, rope=seed % 2 == 0, tag=(block, lens))


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,heads,kvh", SHAPES)
def test_attention_of_several_tokens(ext, code, hd, heads, kvh):
    for seed, (block, lens) in enumerate([(16, [(0, 4), (33, 2), (7, 0), (90, 4)]), (64, [(0, 37)]), (32, [(40, 70), (100, 1), (0, 33)]),
                                          (128, [(127, 3), (300, 17), (1, 140)])]):
        host, dev = _attention_case(np.random.default_rng(seed + 10), code, hd, heads, kvh, block, lens)
        _check_attention(ext, host, dev, heads, rope=seed % 2 == 1, tag=(block, lens))


@pytest.mark.parametrize("code,hd,heads,kvh,block,lens,rope", [
    ("fp8", 128, 8, 8, 64, [(0, 513)], True), ("int8", 128, 16, 2, 16, [(200, 300), (3, 260)], False), ("fp8", 64, 4, 4, 32, [(0, 700)], False),
    ("int8", 256, 4, 2, 128, [(1000, 129), (50, 1)], True), ("fp8", 128, 16, 2, 32, [(5000, 1), (100, 1), (2000, 1)], True),
    ("int8", 128, 4, 4, 64, [(9000, 1)], True), ("fp8", 128, 8, 1, 64, [(6000, 20)], True), ("fp8", 100, 4, 2, 16, [(4100, 9), (60, 257)], True)])
def test_attention_of_long_rows(ext, code, hd, heads, kvh, block, lens, rope):
    host, dev = _attention_case(np.random.default_rng(5), code, hd, heads, kvh, block, lens, spread=2.0)
    _check_attention(ext, host, dev, heads, rope)


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("lens", [[(200, 1), (40, 1), (33, 1)], [(200, 30), (40, 90), (64, 300)]])
def test_attention_with_pages_that_are_not_there(ext, code, lens):
    """Table entries outside the pool are not seen; a row without any page gives zeros."""
    for seed in range(3):
        rng = np.random.default_rng(seed)
        host, dev = _attention_case(rng, code, 128, 8, 2, 16, lens)
        table = host["table"]
        for bad in (-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1, len(host["pool"][0])):
            table[0, rng.integers(table.shape[1])] = bad
        table[1] = -1
        dev["table"] = _dev(table)
        out = _check_attention(ext, host, dev, 8, rope=seed == 0)
        assert (out[int(host["starts"][1]):int(host["starts"][2])] == 0).all()


def test_attention_of_strided_rows_scale_and_limits(ext):
    host, dev = _attention_case(np.random.default_rng(6), "fp8", 128, 8, 2, 32, [(50, 6), (0, 9), (70, 3)])
    wide = torch.zeros(host["q"].shape[0], 8 * 128 + 260, dtype=torch.float16, device=DEV)
    q = wide[:, 4:4 + 1024]
    q.copy_(dev["q"])
    _check_attention(ext, host, dev, 8, True, q=q)
    _check_attention(ext, host, dev, 8, True, scale=0.02)
    _check_attention(ext, host, dev, 8, False, max_new=5)     # the rows' tokens behind max_new are not computed
    dev["q"], host["q"] = dev["q"][:12].contiguous(), host["q"][:12]
    _check_attention(ext, host, dev, 8, False)                # token rows run out


def test_attention_of_padded_rows(ext):
    """starts a fixed distance apart: the padding between the rows stays as it was."""
    rng = np.random.default_rng(7)
    host, dev = _attention_case(rng, "int8", 64, 4, 4, 16, [(20, 5), (0, 9), (33, 1)])
    host["starts"] = np.array([0, 9, 18, 27])
    host["q"] = rng.normal(0, 1, (27, 4, 64)).astype(np.float16)
    dev["q"], dev["starts"] = torch.from_numpy(host["q"]).reshape(27, -1).to(DEV), _dev(host["starts"])
    _check_attention(ext, host, dev, 4, True)


def test_attention_of_lengths_beyond_the_table(ext):
    """past + new beyond the block table: what the table holds is seen."""
    host, dev = _attention_case(np.random.default_rng(8), "fp8", 128, 4, 4, 16, [(60, 4), (44, 20)])      # (full pages: nothing planted lies inside the lengths)
    host["past"] = np.array([70, 1000])
    dev["past"] = _dev(host["past"])
    _check_attention(ext, host, dev, 4, False)


def test_page_offsets_beyond_32_bits(ext):
    """A pool of over 4 GiB: the last pages are written and read where they are."""
    blocks, kvh, block, hd = 2200, 128, 128, 128              # 4.6 GB of keys, as many of values
    kp = torch.empty(blocks, kvh, block, hd, dtype=torch.int8, device=DEV)
    vp = torch.empty(blocks, kvh, hd, block, dtype=torch.int8, device=DEV)
    ks, vs = torch.zeros(blocks, kvh, device=DEV), torch.zeros(blocks, kvh, device=DEV)
    x = torch.randn(2, 3, kvh * hd, dtype=torch.float16, device=DEV)
    q = torch.randn(1, kvh * hd, dtype=torch.float16, device=DEV)
    page = blocks - 1
    ext.ext_paged_append(x[0], x[1], _dev(page * block + np.arange(3)), kp, vp, ks, vs)
    out = ext.ext_paged_attention(q, _dev([0, 1]), _dev([2]), _dev([1]), _dev([[page]]), kp, vp, ks, vs, kvh, max_new=1)
    small = [np.zeros((1, kvh, block, hd)), np.zeros((1, kvh, hd, block)), np.ones((1, kvh)), np.ones((1, kvh))]
    P.append(x[0].cpu().numpy().reshape(3, kvh, hd), x[1].cpu().numpy().reshape(3, kvh, hd), np.arange(3), *small, "int8")
    assert np.array_equal(_numbers(kp[page, :, :3]), small[0][0, :, :3]) and np.array_equal(_numbers(vp[page, :, :, :3]), small[1][0, :, :, :3])
    want, bound = P.attention(q.cpu().numpy().reshape(1, kvh, hd), np.array([0, 1]), np.array([2]), np.array([1]), np.array([[0]]), *small, 1)
    assert (np.abs(out.cpu().double().numpy().reshape(want.shape) - want) <= bound).all()


# ---- together -------------------------------------------------------------------------------------------------------------------------

class _Loop:
    """A few rows served together: prompts, single tokens, ends and new beginnings, the oracle beside every step."""

    def __init__(self, code, hd, heads, kvh, block, n, width, blocks, seed):
        self.rng = np.random.default_rng(seed)
        self.code, self.hd, self.heads, self.kvh, self.block, self.n = code, hd, heads, kvh, block, n
        hd16 = (hd + 15) // 16 * 16
        self.pool = [np.zeros((blocks, kvh, block, hd16)), np.zeros((blocks, kvh, hd16, block)), np.ones((blocks, kvh)), np.ones((blocks, kvh))]
        self.dpool = _pool_dev(self.pool, code)
        self.past, self.held = np.zeros(n, np.int32), np.zeros(n, np.int32)
        self.table, self.ring = np.full((n, width), -1, np.int32), self.rng.permutation(blocks).astype(np.int32)
        self.counters = np.array([0, blocks, 0, 0], np.int32)
        self.d = {k: _dev(getattr(self, k)) for k in ("past", "held", "table", "ring", "counters")}
        self.d["new"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        sin, cos = _angles(width * block, hd)
        self.sin, self.cos, self.dsin, self.dcos = sin.numpy(), cos.numpy(), sin.to(DEV), cos.to(DEV)

    def inputs(self, rows):
        return [self.rng.normal(0, 1, (rows, h, self.hd)).astype(np.float16) for h in (self.heads, self.kvh, self.kvh)]

    def launch(self, ext, dq, dk, dv, out, max_new):
        starts, slots, positions = ext.ext_paged_slots(self.d["past"], self.d["new"], self.d["held"], self.d["table"], self.d["ring"], self.d["counters"],
                                                       self.block, dq.shape[0], max_new=max_new)
        ext.ext_paged_append(dk, dv, slots, *self.dpool, positions=positions, sin=self.dsin, cos=self.dcos)
        ext.ext_paged_attention(dq, starts, self.d["past"], self.d["new"], self.d["table"], *self.dpool, self.heads, max_new=max_new, sin=self.dsin,
                                cos=self.dcos, out=out)
        self.d["past"].add_(self.d["new"].clamp(min=0))

    def expect(self, new, q, k, v, max_new):
        starts, slots, positions = P.slots(self.past, new, self.held, self.table, self.ring, self.counters, self.block, self.table.shape[1] * self.block,
                                           max_new, len(q))
        P.append(k, v, slots, *self.pool, self.code, positions, self.sin, self.cos)
        r = P.attention(q, starts, self.past, new, self.table, *self.pool, max_new, sin=self.sin, cos=self.cos)
        self.past += np.maximum(new, 0).astype(np.int32)
        return r

    def agree(self, out, want, bound, tag):
        for name in ("held", "table", "ring", "counters", "past"):
            assert np.array_equal(self.d[name].cpu().numpy(), getattr(self, name)), (tag, name)
        for name, got, x in zip(("keys", "values", "key scales", "value scales"), self.dpool, self.pool):
            assert _same(_numbers(got), x), (tag, name)
        got = out.cpu().double().numpy().reshape(want.shape)
        some = ~np.isnan(bound).all((1, 2))
        assert (np.abs(got - want)[some] <= bound[some]).all(), tag


@pytest.mark.parametrize("code,hd,heads,kvh,block", [("fp8", 128, 8, 2, 16), ("int8", 64, 4, 4, 32), ("int8", 100, 6, 2, 16)])
def test_a_serving_loop(ext, code, hd, heads, kvh, block):
    loop = _Loop(code, hd, heads, kvh, block, n=5, width=8, blocks=24, seed=9)
    news = [[20, 0, 3, 40, 1], [1, 0, 1, 1, 1], [1, 30, 1, -1, 1], [1, 1, 1, 17, 1], [3, 1, -1, 1, 9], [1, 1, 12, 1, 1]]
    for step, new in enumerate(news):
        new = np.array(new)
        rows, max_new = int(np.maximum(new, 0).sum()) + 1, int(new.max())
        q, k, v = loop.inputs(rows)
        loop.d["new"].copy_(_dev(new))
        out = torch.zeros(rows, heads * hd, dtype=torch.float16, device=DEV)
        loop.launch(ext, *(torch.from_numpy(x).reshape(rows, -1).to(DEV) for x in (q, k, v)), out, max_new)
        want, bound = loop.expect(new, q, k, v, max_new)
        loop.past[new < 0] = 0
        loop.d["past"][loop.d["new"] < 0] = 0
        loop.agree(out, want, bound, step)


def test_captured_steps_replay_while_lengths_grow(ext):
    """One step of single tokens captured once (slots, append, attention, the lengths' advance) and replayed over page ends, with eager work of
    the same process between the replays; a second graph over another loop shares nothing with it."""
    loops, graphs, bufs = [], [], []
    side = torch.cuda.Stream()
    for seed in (11, 12):
        loop = _Loop("fp8", 128, 8, 2, 16, n=3, width=6, blocks=20, seed=seed)
        loop.d["new"].fill_(1)
        x = [torch.zeros(3, h * 128, dtype=torch.float16, device=DEV) for h in (8, 2, 2)]
        out = torch.zeros(3, 8 * 128, dtype=torch.float16, device=DEV)
        state = {k: v.clone() for k, v in loop.d.items()}, [p.clone() for p in loop.dpool]
        with torch.cuda.stream(side):
            loop.launch(ext, *x, out, 1)                       # (the first call of a process loads the kernels)
        torch.cuda.synchronize()
        for k, v in state[0].items():
            loop.d[k].copy_(v)
        for p, v in zip(loop.dpool, state[1]):
            p.copy_(v)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loop.launch(ext, *x, out, 1)
        loops.append(loop); graphs.append(g); bufs.append((x, out))
    for step in range(20):
        for loop, g, (x, out) in zip(loops, graphs, bufs):
            host = loop.inputs(3)
            for d, h in zip(x, host):
                d.copy_(torch.from_numpy(h).reshape(3, -1))
            g.replay()
            torch.zeros(100000, device=DEV).add_(1).sum()
        torch.cuda.synchronize()
        for loop, (x, out) in zip(loops, bufs):
            host = [t.cpu().numpy().reshape(3, -1, 128) for t in x]
            want, bound = loop.expect(np.ones(3, np.int64), *host, 1)
            loop.agree(out, want, bound, step)


def test_calls_on_two_streams_do_not_meet(ext):
    """The same pages read by two streams at once, each with lengths of its own, many times: every result is the one-stream result."""
    host, dev = _attention_case(np.random.default_rng(13), "int8", 128, 16, 2, 16, [(900, 1), (1500, 1), (30, 1)])
    other = dict(dev, past=_dev(host["past"] // 2))
    call = lambda d: ext.ext_paged_attention(d["q"], d["starts"], d["past"], d["new"], d["table"], *d["pool"], 16, max_new=1)  # noqa: E731
    one, two = call(dev), call(other)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = ([], [])
    for _ in range(20):
        for s, d, g in zip(streams, (dev, other), got):
            with torch.cuda.stream(s):
                g.append(call(d))
    torch.cuda.synchronize()
    assert all(torch.equal(x, one) for x in got[0]) and all(torch.equal(x, two) for x in got[1])


# ---- calls that are allowed and rarely made ----------------------------------------------------------------------------------------------

def test_append_of_many_rows(ext):
    """Enough token rows that a workgroup looks at 32 of them: long runs, runs of one token, skipped rows."""
    rng = np.random.default_rng(20)
    hd, kvh, block, blocks = 16, 32, 128, 80
    pool = _pool(rng, blocks, kvh, block, hd, "fp8")
    dev = _pool_dev(pool, "fp8")
    slots, pos = _runs(rng, blocks, block, [(3, 1500), (0, 1), (-1, -33), (127, 1400), (64, 64), (5, 2), (0, 1200), (-1, -1)] + [(9, 1)] * 20)
    t = len(slots)
    assert t * kvh > 131072
    x = rng.normal(0, 1, (2, t, kvh, hd)).astype(np.float16)
    ext.ext_paged_append(*(torch.from_numpy(y).reshape(t, -1).to(DEV) for y in x), _dev(slots), *dev)
    P.append(x[0], x[1], slots, *pool, "fp8")
    for name, got, want in zip(("keys", "values", "key scales", "value scales"), dev, pool):
        assert _same(_numbers(got), want), name


@pytest.mark.parametrize("n,max_new", [(70, 1), (300, 1), (300, 3), (70, 60), (300, 40)])
def test_attention_of_many_rows(ext, n, max_new):
    """More rows than a wave, and than a workgroup, looks at once; most of them short, some without a token."""
    rng = np.random.default_rng(n + max_new)
    new = rng.integers(0, min(max_new, 4) + 1, n)
    new[rng.integers(n)] = max_new
    past = np.where(rng.random(n) < 0.05, 400, rng.integers(0, 40, n))
    host, dev = _attention_case(rng, "int8", 64, 2, 1, 16, [(int(p), int(m)) for p, m in zip(past, new)])
    _check_attention(ext, host, dev, 2, True)


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hd,lens", [(128, [(90, 3), (700, 1)]), (256, [(5, 1)]), (64, [(90, 70), (700, 200)]), (100, [(1200, 90)])])
def test_attention_under_the_largest_scales(ext, code, hd, lens):
    """The upper end of the scales' range: codes * scale up to 65024 and 57344, keys and values alike, a scale for each page and head."""
    rng = np.random.default_rng(hd)
    host, dev = _attention_case(rng, code, hd, 4, 2, 16, lens)
    for i in (2, 3):
        host["pool"][i] = np.ldexp(1.0, rng.integers(3, P.EXP[code][1] + 1, host["pool"][i].shape))
        dev["pool"][i] = _dev(host["pool"][i], torch.float32)
    host["q"] = (host["q"].astype(np.float64) * 2.0 ** -13).astype(np.float16)
    dev["q"] = torch.from_numpy(host["q"]).reshape(len(host["q"]), -1).to(DEV)
    _check_attention(ext, host, dev, 4, True)
    _check_attention(ext, host, dev, 4, False)


# hd, heads, kv heads, (past, new): few queries, in one stretch and in several; many, in one piece and in several
NAN_CASES = [(128, 4, 4, (70, 20)), (64, 8, 8, (1900, 30)), (256, 2, 2, (62, 14)), (100, 4, 2, (30, 16)), (128, 8, 1, (62, 4)), (128, 2, 2, (40, 200)),
             (64, 4, 1, (900, 100)), (256, 2, 1, (1500, 130)), (80, 2, 2, (0, 300))]


@pytest.mark.parametrize("what", ["value", "key", "query"])
@pytest.mark.parametrize("hd,heads,kvh,row", NAN_CASES)
def test_nan_stays_where_it_is_seen(ext, what, hd, heads, kvh, row):
    """A token whose value, key or query is NaN: the queries that see it (and its columns; all of its row) are NaN, no other is."""
    for block in (16, 64):
        host, dev = _attention_case(np.random.default_rng(hd + block), "fp8", hd, heads, kvh, block, [row, (33, 2)])
        past, new = row
        group, at, j = heads // kvh, past + new // 3, new // 3
        page, off = host["table"][0, at // block], at % block
        want, bound = P.attention(host["q"], host["starts"], host["past"], host["new"], host["table"], *host["pool"], int(host["new"].max()))
        nan = np.isnan(bound)
        expect = np.zeros_like(nan)
        if what == "value":
            cols = [0, 7 % hd, hd - 1]
            host["pool"][1][page, 0, cols, off] = np.nan
            for c in cols:
                expect[j:new, :group, c] = True
        elif what == "key":
            host["pool"][0][page, kvh - 1, off, 3] = np.nan
            expect[j:new, heads - group:] = True
        else:
            host["q"][j, 1, hd - 2] = np.nan
            dev["q"] = torch.from_numpy(host["q"]).reshape(len(host["q"]), -1).to(DEV)
            expect[j, 1] = True
        dev["pool"] = _pool_dev(host["pool"], "fp8")
        got = ext.ext_paged_attention(dev["q"], dev["starts"], dev["past"], dev["new"], dev["table"], *dev["pool"], heads,
                                      max_new=int(host["new"].max())).cpu().double().numpy().reshape(want.shape)
        assert np.array_equal(np.isnan(got), expect)
        ok = ~expect & ~nan
        assert (np.abs(got - want)[ok] <= bound[ok]).all()


def test_calls_without_rows(ext):
    pool = _pool_dev(_pool(np.random.default_rng(21), 3, 2, 16, 64, "int8"), "int8")
    before = [p.clone() for p in pool]
    x = torch.zeros(0, 128, dtype=torch.float16, device=DEV)
    none, one = torch.zeros(0, dtype=torch.int32, device=DEV), _dev([1])
    ext.ext_paged_append(x, x, none, *pool)
    ext.ext_paged_append(x, x, none, *pool, positions=none, sin=torch.zeros(4, 64, dtype=torch.float16, device=DEV),
                         cos=torch.zeros(4, 64, dtype=torch.float16, device=DEV))
    assert ext.ext_paged_attention(x, _dev([0, 0]), one, one, _dev([[0, 1]]), *pool, 2).shape == (0, 128)
    y = torch.zeros(3, 128, dtype=torch.float16, device=DEV)
    out = ext.ext_paged_attention(y, _dev([0, 0]), one, one, _dev([[0, 1]]), *pool, 2, max_new=0, out=torch.full_like(y, 3))
    assert (out == 3).all()
    held, table, ring, counters = _dev([0]), _dev([[-1, -1]]), _dev([0, 1, 2]), _dev([0, 3, 0, 0])
    starts, slots, positions = ext.ext_paged_slots(_dev([5]), _dev([0]), held, table, ring, counters, 16, 0)
    assert starts.tolist() == [0, 0] and slots.numel() == 0 and positions.numel() == 0
    assert held.tolist() == [1] and table.tolist() == [[0, -1]] and counters.tolist() == [1, 2, 0, 0]
    for a, b in zip(before, pool):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_all_rows_end_at_once(ext):
    """Every block goes back, in the rows' order, and is handed out again by the next call."""
    past, held, table = _dev([40, 0, 17]), _dev([3, 0, 2]), _dev([[4, 1, 0], [-1, -1, -1], [3, 2, -1]])
    ring, counters = _dev([-7] * 5), _dev([2, 0, 0, 0])
    _, slots, _ = ext.ext_paged_slots(past, _dev([-1, -1, -1]), held, table, ring, counters, 16, 4)
    assert held.tolist() == [0, 0, 0] and (table == -1).all() and (slots == -1).all()
    assert counters.tolist() == [2, 5, 0, 0] and ring.tolist() == [3, 2, 4, 1, 0]
    past.zero_()
    ext.ext_paged_slots(past, _dev([0, 33, 32]), held, table, ring, counters, 16, 65)
    assert table.tolist() == [[-1, -1, -1], [4, 1, 0], [3, 2, -1]] and counters.tolist() == [2, 0, 0, 0]


def test_padded_batch_through_all_three(ext):
    """Rows a fixed distance apart, from the slots on: the padding is neither stored nor computed."""
    rng, (n, stride, hd, heads, kvh, block, blocks) = np.random.default_rng(22), (4, 9, 64, 4, 2, 16, 30)
    past, held = np.zeros(n, np.int32), np.zeros(n, np.int32)
    table, ring, counters = np.full((n, 4), -1, np.int32), rng.permutation(blocks).astype(np.int32), np.array([7, blocks, 0, 0], np.int32)
    pool = [np.zeros((blocks, kvh, block, hd)), np.zeros((blocks, kvh, hd, block)), np.ones((blocks, kvh)), np.ones((blocks, kvh))]
    dpool = _pool_dev(pool, "fp8")
    d = [_dev(x) for x in (past, held, table, ring, counters)]
    for new in ([9, 3, 0, 20], [1, 1, 9, 1], [1, 9, 1, 1]):
        new = np.array(new)
        q, k, v = (rng.normal(0, 1, (n * stride, h, hd)).astype(np.float16) for h in (heads, kvh, kvh))
        dq, dk, dv = (torch.from_numpy(x).reshape(n * stride, -1).to(DEV) for x in (q, k, v))
        starts, slots, positions = P.slots(past, new, held, table, ring, counters, block, 64, stride, n * stride, stride)
        gstarts, gslots, gpos = ext.ext_paged_slots(d[0], _dev(new), d[1], d[2], d[3], d[4], block, n * stride, max_new=stride, row_stride=stride)
        assert gstarts.tolist() == starts.tolist() and gslots.tolist() == slots.tolist() and gpos.tolist() == positions.tolist()
        ext.ext_paged_append(dk, dv, gslots, *dpool)
        P.append(k, v, slots, *pool, "fp8")
        new = np.minimum(new, stride)
        out = torch.full((n * stride, heads * hd), 7.5, dtype=torch.float16, device=DEV)
        ext.ext_paged_attention(dq, gstarts, d[0], _dev(new), d[2], *dpool, heads, max_new=stride, out=out)
        want, bound = P.attention(q, starts, past, new, table, *pool, stride)
        got, none = out.cpu().double().numpy().reshape(want.shape), np.isnan(bound)
        assert (got[none] == 7.5).all() and (np.abs(got - want)[~none] <= bound[~none]).all()
        past += new.astype(np.int32)
        d[0].copy_(_dev(past))


def test_captured_prompt_pieces_replay(ext):
    """Attention of many queries captured once (rows cut into pieces, joined), replayed under other lengths, with eager work in between; a second
    graph captured beside it has a workspace of its own."""
    host, dev = _attention_case(np.random.default_rng(23), "fp8", 128, 8, 2, 64, [(1700, 120), (300, 60), (0, 90)])
    call = lambda past, new, out: ext.ext_paged_attention(dev["q"], dev["starts"], past, new, dev["table"], *dev["pool"], 8, max_new=120,  # noqa: E731
                                                          sin=dev["sin"], cos=dev["cos"], out=out)
    sets = [(host["past"], host["new"]), (host["past"] // 2, host["new"]), (host["past"], np.array([120, 0, 3])), (host["past"] * 0, np.array([1, 60, 90]))]
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        past, new, out = dev["past"].clone(), dev["new"].clone(), torch.zeros_like(dev["q"])
        with torch.cuda.stream(side):
            call(past, new, out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(past, new, out)
        graphs.append((g, past, new, out))
    for step in range(8):
        eager = []
        for u, (g, past, new, out) in enumerate(graphs):
            p, m = sets[(step + u) % 4]
            past.copy_(_dev(p)); new.copy_(_dev(m)); out.fill_(7.5)
            eager.append(call(_dev(p), _dev(m), torch.full_like(out, 7.5)))
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (g, past, new, out), want in zip(graphs, eager):
            assert torch.equal(out, want), step


def test_prompts_on_two_streams_do_not_meet(ext):
    host, dev = _attention_case(np.random.default_rng(24), "int8", 128, 4, 2, 32, [(1500, 100), (900, 150)])
    other = dict(dev, past=_dev(host["past"] // 3))
    call = lambda d: ext.ext_paged_attention(d["q"], d["starts"], d["past"], d["new"], d["table"], *d["pool"], 4, max_new=150)  # noqa: E731
    one, two = call(dev), call(other)
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), ([], [])
    for _ in range(10):
        for s, d, g in zip(streams, (dev, other), got):
            with torch.cuda.stream(s):
                g.append(call(d))
    torch.cuda.synchronize()
    assert all(torch.equal(x, one) for x in got[0]) and all(torch.equal(x, two) for x in got[1])


def test_out_must_not_overlap_q(ext):
    host, dev = _attention_case(np.random.default_rng(25), "fp8", 64, 2, 2, 16, [(20, 3)])
    args = (dev["starts"], dev["past"], dev["new"], dev["table"], *dev["pool"], 2)
    with pytest.raises(RuntimeError, match="overlaps"):
        ext.ext_paged_attention(dev["q"], *args, out=dev["q"])
    with pytest.raises(RuntimeError, match="overlaps"):
        ext.ext_paged_attention(dev["q"][:3], *args, out=dev["q"][2:5])
    both = torch.cat((dev["q"], dev["q"]))                     # next to each other is fine
    assert ext.ext_paged_attention(both[:5], *args, out=both[5:]).data_ptr() == both[5:].data_ptr()


def test_compiled_binding_and_ctypes_path_agree(ext):
    """The compiled binding against the ctypes methods that it replaces: the same results to the bit, the same refusals."""
    fast, slow = ext.FAST_BINDING, type(ext.exllama_ext)
    assert fast is not None and ext.paged_slots is fast.paged_slots and ext.paged_append is fast.paged_append and ext.paged_attention is fast.paged_attention
    results = []
    for pick in (lambda n: getattr(fast, n), lambda n: lambda *a, **k: getattr(slow, n)(ext.exllama_ext, *a, **k)):
        rng = np.random.default_rng(26)
        pool = _pool_dev(_pool(rng, 12, 2, 16, 64, "fp8"), "fp8")
        past, new, held, table = _dev([5, 30]), _dev([4, 9]), _dev([0, 0]), torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
        ring, counters = _dev(rng.permutation(12)), _dev([3, 12, 0, 0])
        sin, cos = (x.to(DEV) for x in _angles(64, 64))
        x = [torch.from_numpy(rng.normal(0, 1, (14, h * 64)).astype(np.float16)).to(DEV) for h in (4, 2, 2)]
        starts, slots, positions = pick("paged_slots")(past, new, held, table, ring, counters, 16, 14, max_len=60)
        pick("paged_append")(x[1], x[2], slots, *pool, positions, sin, cos)
        out = torch.full((14, 256), 7.5, dtype=torch.float16, device=DEV)
        assert pick("paged_attention")(x[0], starts, past, new, table, *pool, 4, 9, sin, cos, 0.1, out) is out
        fresh = pick("paged_attention")(x[0], starts, past, new, table, *pool, 4)
        results.append([starts, slots, positions, held, table, ring, counters, *[p.view(torch.uint8) for p in pool], out, fresh])
        for bad in (dict(out=out.float()), dict(out=out[:3]), dict(sin=sin), dict(sin=sin[:, :32], cos=cos[:, :32])):
            with pytest.raises(RuntimeError):
                pick("paged_attention")(x[0], starts, past, new, table, *pool, 4, **bad)
        with pytest.raises(RuntimeError):
            pick("paged_append")(x[1], x[2][:5], slots, *pool)
        with pytest.raises(RuntimeError):
            pick("paged_append")(x[1], x[2], slots[:5], *pool)
        with pytest.raises(RuntimeError):
            pick("paged_slots")(past, new[:1], held, table, ring, counters, 16, 14)
        with pytest.raises(RuntimeError):
            pick("paged_slots")(past, new, held, table[:1], ring, counters, 16, 14)
    assert all(torch.equal(a, b) for a, b in zip(*results))
