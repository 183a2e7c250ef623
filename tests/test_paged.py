"""The paged 8-bit cache on the CPU: its oracle against the formulas' own properties, and the refusals of the entry points (nothing is launched)."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P


def test_codes_are_the_nearest():
    for code in ("fp8", "int8"):
        if code == "fp8":
            every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
            every = np.unique(every[np.isfinite(every)])
        else:
            every = np.arange(-127.0, 128.0)
        assert np.array_equal(P.nearest(every, code), every)
        rng = np.random.default_rng(0)
        x = np.concatenate((rng.uniform(-500, 500, 4000), rng.normal(0, 0.01, 4000), (every[1:] + every[:-1]) / 2))
        got = P.nearest(x, code)
        best = np.abs(np.clip(x, every[0], every[-1])[:, None] - every[None]).min(1)
        assert np.isin(got, every).all() and np.array_equal(np.abs(np.clip(x, every[0], every[-1]) - got), best)
        if code == "fp8":                                     # ties to even: torch's own cast agrees on every value, the halfway points among them
            y = torch.from_numpy(x).float()                   # (rounded twice, so only where 32 bits hold x)
            same = y.double().numpy() == x
            assert np.array_equal(got[same], y.clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()[same])


def test_exponent_is_the_least():
    for code, (lo, hi) in P.EXP.items():
        for amax in (0.0, 2.0 ** -24, 1.0, 126.99, 127.0, 127.01, 448.0, 448.5, 57344.0, 65504.0):
            e = P.exponent(amax, code)
            assert lo <= e <= hi and (amax <= P.TOP[code] * 2.0 ** e or e == hi) and (e == lo or amax > P.TOP[code] * 2.0 ** (e - 1))


def test_growing_a_page_token_by_token_equals_one_append_when_the_first_token_is_the_largest():
    rng = np.random.default_rng(1)
    k, v = rng.normal(0, 1, (2, 16, 2, 16)).astype(np.float16)
    k[0], v[0] = 9.0, -7.0
    for code in ("fp8", "int8"):
        whole, steps = ([np.zeros((3, 2, 16, 16)), np.zeros((3, 2, 16, 16)), np.ones((3, 2)), np.ones((3, 2))] for _ in range(2))
        slot = 16 + np.arange(16)
        P.append(k, v, slot, *whole, code)
        for t in range(16):
            P.append(k[t:t + 1], v[t:t + 1], slot[t:t + 1], *steps, code)
        for a, b in zip(whole, steps):
            assert np.array_equal(a, b)


def test_slots_give_back_and_take():
    ring, counters = np.array([5, 6, 7, 0, 1, 2, 3, 4], np.int32), np.array([3, 5, 0, 0], np.int32)
    table, held = np.full((3, 4), -1, np.int32), np.array([2, 0, 1], np.int32)
    table[0, :2], table[2, 0] = [5, 6], 7
    past, new = np.array([20, 0, 15]), np.array([-1, 40, 3])
    starts, slots, positions = P.slots(past, new, held, table, ring, counters, 16, 64, 64, 50)
    assert starts.tolist() == [0, 0, 40, 43] and held.tolist() == [0, 3, 2]
    assert table.tolist() == [[-1] * 4, [0, 1, 2, -1], [7, 3, -1, -1]]
    assert counters.tolist() == [7, 3, 0, 0] and [int(ring[(7 + i) % 8]) for i in range(3)] == [4, 5, 6]
    assert slots[:40].tolist() == [16 * (i // 16) + i % 16 for i in range(40)] and slots[40:].tolist() == [127, 48, 49] + [-1] * 7
    assert positions[40:43].tolist() == [15, 16, 17]


@pytest.fixture(scope="module")
def ext():
    from exllama_amd import cuda_ext
    return cuda_ext


def test_refuses_cpu_tensors_and_wrong_types(ext):
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        ext.ext_paged_slots(i, i, i, torch.zeros(4, 2, dtype=torch.int32), i, i, 16, 4)
    with pytest.raises(RuntimeError, match="incorrect datatype"):
        ext.ext_paged_slots(i.long(), i, i, torch.zeros(4, 2, dtype=torch.int32), i, i, 16, 4)
    kp, vp, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 64, 16, dtype=torch.int8), torch.zeros(2, 1)
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        ext.ext_paged_append(x, x, i, kp, vp, s, s)
    with pytest.raises(RuntimeError, match="incorrect datatype"):
        ext.ext_paged_append(x, x, i, kp.float(), vp, s, s)
    with pytest.raises(RuntimeError, match="value_pages"):
        ext.ext_paged_append(x, x, i, kp, kp, s, s)
    with pytest.raises(RuntimeError, match="columns"):
        ext.ext_paged_append(torch.zeros(4, 100, dtype=torch.float16), x, i, kp, vp, s, s)
    with pytest.raises(RuntimeError, match="scales must be"):
        ext.ext_paged_append(x, x, i, kp, vp, s[:1], s)
    with pytest.raises(RuntimeError, match="HIP device"):
        ext.ext_paged_attention(x, i, i, i, torch.zeros(4, 2, dtype=torch.int32), kp, vp, s, s, 1)
    with pytest.raises(RuntimeError, match="num_heads"):
        ext.ext_paged_attention(x, i, i, i, torch.zeros(4, 2, dtype=torch.int32), kp, vp, s, s, 3)


def test_c_entries_refuse_before_they_launch(ext):
    """The C entries' own checks, called without a device: each returns a code and a message."""
    lib = ext._lib.load()
    p = C.c_void_p(4096)                                      # never read: every call below is refused first

    def slots(n=1, width=4, block=16, blocks=8, max_len=64, max_new=1, rows=1, stride=0, past=p):
        return lib.exl_paged_slots(past, p, p, p, p, p, n, width, block, blocks, max_len, max_new, rows, stride, p, p, p, p, None)

    def append(ks=64, vs=64, rows=1, code=0, blocks=8, kvh=1, block=16, hd=64, pos=None, sin=None, cos=None, angle_rows=0, k=p, pages=p):
        return lib.exl_paged_append(k, p, ks, vs, p, rows, pages, p, p, p, code, blocks, kvh, block, hd, pos, sin, cos, angle_rows, None)

    def attention(qs=64, n=1, rows=1, max_new=1, width=4, code=0, blocks=8, block=16, heads=1, kvh=1, hd=64, sin=None, cos=None, angle_rows=0, q=p, ws=0):
        return lib.exl_paged_attention(q, qs, p, p, p, n, rows, max_new, p, width, p, p, p, p, code, blocks, block, heads, kvh, hd, 0.0, sin, cos,
                                       angle_rows, p, None, ws, None)

    bad = [(slots, kw) for kw in ({"n": 0}, {"width": 0}, {"block": 24}, {"block": 256}, {"blocks": 0}, {"max_len": 65}, {"max_new": -1}, {"rows": -1},
                                  {"stride": -1}, {"past": None}, {"blocks": 2 ** 27 + 1}, {"max_len": -1})]
    bad += [(append, kw) for kw in ({"ks": 60}, {"vs": 66}, {"rows": -1}, {"code": 2}, {"blocks": 0}, {"kvh": 0}, {"block": 8}, {"hd": 66}, {"hd": 260},
                                    {"sin": p}, {"sin": p, "cos": p, "angle_rows": 4}, {"sin": p, "cos": p, "pos": p}, {"k": None},
                                    {"k": C.c_void_p(4100)}, {"pages": C.c_void_p(4104)})]
    bad += [(attention, kw) for kw in ({"qs": 62}, {"n": 0}, {"rows": -1}, {"max_new": -1}, {"width": 0}, {"code": 3}, {"blocks": 0}, {"block": 48},
                                       {"heads": 3, "kvh": 2, "qs": 192}, {"hd": 2}, {"hd": 288, "qs": 288}, {"sin": p}, {"sin": p, "cos": p}, {"q": None},
                                       {"width": 2 ** 28, "block": 16}, {"q": C.c_void_p(4100)})]
    for fn, kw in bad:
        assert fn(**kw) < 0, (fn.__name__, kw)
        msg = lib.exl_last_error().decode()
        assert msg.startswith("paged_" + fn.__name__), (fn.__name__, kw, msg)
    assert append(rows=0) == 0 and attention(rows=0) == 0 and attention(max_new=0) == 0


def test_c_attention_refuses_a_small_workspace_and_an_out_that_overlaps(ext):
    lib = ext._lib.load()
    p, far = C.c_void_p(4096), C.c_void_p(1 << 20)            # never read: every call below is refused first

    def attention(out, ws, ws_bytes, rows=40, n=2):
        return lib.exl_paged_attention(p, 64, p, p, p, n, rows, rows, p, 400, p, p, p, p, 0, 8, 16, 1, 1, 64, 0.0, None, None, 0, out, ws, ws_bytes, None)

    for rows in (1, 40):                                      # few queries, and many
        need = lib.exl_paged_attention_workspace(2, rows, rows, 1, 1, 64, 400, 16)
        assert need > 0
        for out, ws, ws_bytes, what in ((far, None, need, "workspace"), (far, p, need - 1, "workspace"), (far, C.c_void_p(4104), need, "workspace"),
                                        (p, p, need, "overlaps"), (C.c_void_p(4096 + 128 * rows - 2 * 4), p, need, "overlaps")):
            assert attention(out, ws, ws_bytes, rows) < 0
            assert what in lib.exl_last_error().decode(), (rows, what)
    assert lib.exl_paged_attention_workspace(0, 1, 1, 1, 1, 64, 4, 16) == 0 and lib.exl_paged_attention_workspace(1, 1, 1, 3, 2, 64, 4, 16) == 0


def test_c_entries_take_empty_tensors(ext):
    """No rows: nothing is launched, and the addresses of empty tensors (null) are fine."""
    lib = ext._lib.load()
    p = C.c_void_p(4096)
    assert lib.exl_paged_append(None, None, 64, 64, None, 0, p, p, p, p, 0, 8, 1, 16, 64, None, p, p, 4, None) == 0
    assert lib.exl_paged_attention(None, 64, p, p, p, 1, 0, 1, p, 4, p, p, p, p, 0, 8, 16, 1, 1, 64, 0.0, None, None, 0, None, None, 0, None) == 0


def test_kernels_fit_their_registers():
    """No paged kernel spills, and each fits the waves per SIMD that it is declared for (512 registers of a SIMD: 256 for two waves)."""
    import os
    import sys
    import tempfile

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "exllama_amd", "libexl_amd.so")
    if not os.path.exists(path):
        pytest.skip("libexl_amd.so not built")
    sys.path.insert(0, os.path.join(root, "scripts"))
    import isa_lint

    with tempfile.TemporaryDirectory() as d:
        res = {n: r for n, r in isa_lint.kernel_resources(path, d).items() if "paged_" in n}
    assert sum("paged_attn_few" in n for n in res) == 10 and sum("paged_attn_many" in n for n in res) == 20 and sum("paged_append" in n for n in res) == 20
    for n, r in res.items():
        assert r["scratch"] == 0, (n, r)
        total = r["vgpr"]                                      # (of both kinds)
        if "paged_attn_few" in n or "paged_attn_many" in n:
            one = "ELi256E" in n or "ILi0ELi128ELi2E" in n or "ILi1ELi128ELi2E" in n
            assert total <= (512 if one else 256), (n, r)
        elif "paged_attn_join" in n:
            assert total <= 128, (n, r)
        elif "paged_slots" in n:
            assert total <= 128, (n, r)                        # 1024 threads
