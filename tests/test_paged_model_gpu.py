"""ExLlama.forward over an ExLlamaPagedCache: against the fp16 cache holding the same codes' values, ragged rows against rows alone, pages given back
and taken again, and what is refused."""
import numpy as np
import pytest
import torch

from exllama_amd import synth
from oracle import paged_oracle as P
from parity import PATHS_TOL, _model_close

pytestmark = pytest.mark.gpu

# Two passes whose fp16 projections differ in the last place (2^-10 of a number, two paths) store a few codes that differ by one: a number lies that
# near to a border with a chance of 2 * 2^-10 / 2^-3 = 2^-6 (e4m3; int8: 127 / 1024 for a page's largest numbers, about 2^-5 on average) and then moves by
# 2^-3 of itself (1 / 32 of a typical one), which is 2^-3 * 2^-3 = 2^-6 of the numbers' norm.  Keys and values both: twice that, 3 %.
PAGED_TOL = 3e-2

TYPE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}


def _model(dims, max_seq_len=160, act_order=False, **config):
    from exllama_amd.model import ExLlama, ExLlamaConfig
    cfg = ExLlamaConfig(synth.config_dict(dims))
    cfg.max_seq_len = max_seq_len
    for k, v in config.items():
        setattr(cfg, k, v)
    return ExLlama(cfg, tensors=synth.make_checkpoint(dims, groupsize=64, act_order=act_order, seed=5, device="cpu", zeros="rand"))


def _ids(dims, rows, n, seed=0):
    return torch.randint(1, dims.vocab_size, (rows, n), generator=torch.Generator().manual_seed(seed)).to("cuda:0")


@pytest.mark.parametrize("code", ["fp8", "int8"])
@pytest.mark.parametrize("hidden,heads,kvh", [(512, 4, 4), (1024, 8, 2), (256, 4, 4)])
def test_one_layer_against_the_formulas(code, hidden, heads, kvh):
    """A model of one layer: keys and values depend on the tokens alone.  The pages after a prompt stand for the fp16 cache's keys and values within a
    code's rounding, and a further token's logits are those of the oracle's attention over the pages, put through the rest of the layer."""
    from exllama_amd.model import ExLlamaCache, ExLlamaPagedCache
    dims = synth.LlamaDims(hidden, 2 * hidden, 1, heads, num_key_value_heads=kvh, vocab_size=512)
    model = _model(dims)
    ids, hd = _ids(dims, 1, 70), dims.head_dim
    paged = ExLlamaPagedCache(model, block_size=32, dtype=TYPE[code])
    fp16 = ExLlamaCache(model)
    model.forward(ids, paged, preprocess_only=True)
    model.forward(ids, fp16, preprocess_only=True)
    table = paged._dev["cuda:0"]["table"].cpu().numpy()[0]
    numbers = lambda: [t.cpu().float().double().numpy() for t in paged.pages[0]]  # noqa: E731
    kc, vc, ks, vs = numbers()
    for t, page in enumerate(np.repeat(table[:3], 32)[:70]):
        i = t % 32
        for x, x16, s in ((kc[page, :, i, :hd] * ks[page][:, None], fp16.key_states[0][0, :, t], ks[page]),
                          (vc[page, :, :hd, i] * vs[page][:, None], fp16.value_states[0][0, :, t], vs[page])):
            x16 = x16.cpu().double().numpy()
            # a code's rounding: half a step of int8, 2^-4 of an e4m3 number (2^-10 of a scale below its normal range); the fp16 cache's own: three
            # roundings in its rotation and two paths' fp16 projections, each at most a unit in the last place of the largest (2^-10)
            step = s[:, None] / 2 if code == "int8" else np.maximum(np.abs(x16) * 2.0 ** -4, s[:, None] * 2.0 ** -10)
            assert (np.abs(x - x16) <= step * (1 + 2.0 ** -6) + 6 * np.abs(x16).max() * 2.0 ** -10).all(), t
    nxt = _ids(dims, 1, 1, seed=9)
    got = model.forward(nxt, paged).cpu()
    kc, vc, ks, vs = numbers()
    layer = model.layers[0]
    normed = layer.input_layernorm.forward(model.embed(nxt))
    q = layer.self_attn.q_proj.forward(normed).view(1, heads, hd).cpu().numpy()
    sin, cos = (t.view(-1, hd).cpu().numpy() for t in model.sincos["cuda:0"])
    want, _ = P.attention(q, np.array([0, 1]), np.array([70]), np.array([1]), table[None], kc, vc, ks, vs, 1, sin=sin, cos=cos)
    hidden_states = model.embed(nxt)
    layer.self_attn.o_proj.forward(torch.from_numpy(want).half().view(1, 1, -1).to("cuda:0"), None, out=hidden_states, accumulate=True)
    layer.mlp.forward_residual(layer.post_attention_layernorm.forward(hidden_states), hidden_states, None)
    _model_close(got[0], model.head(hidden_states).cpu()[0], PATHS_TOL, f"{code} {hidden}")
    model.free_unmanaged()


@pytest.mark.parametrize("code,block,act", [("fp8", 16, False), ("int8", 64, True)])
def test_ragged_rows_equal_rows_alone(code, block, act):
    """Right-padded rows of three lengths, then single tokens for some of them: each row's logits are those of the row by itself."""
    from exllama_amd.model import ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128_GQA
    model = _model(dims, act_order=act, max_input_len=90)                      # three rows of 50: two chunks
    ids = _ids(dims, 3, 50, seed=1)
    lens = [50, 7, 31]
    batch = ExLlamaPagedCache(model, batch_size=3, block_size=block, dtype=TYPE[code])
    alone = [ExLlamaPagedCache(model, block_size=block, dtype=TYPE[code]) for _ in lens]
    got = model.forward(ids, batch, row_lens=lens).cpu()
    assert batch.seq_lens == lens and batch.current_seq_len == 50
    for b, n in enumerate(lens):
        want = model.forward(ids[b:b + 1, :n], alone[b]).cpu()
        _model_close(got[b], want[0], PAGED_TOL, f"prompt row {b}")
    for step, take in enumerate(([1, 1, 1], [1, 0, 1], [0, 1, 1])):
        nxt = _ids(dims, 3, 1, seed=20 + step)
        got = model.forward(nxt, batch, row_lens=take).cpu()
        for b in range(3):
            if take[b]:
                want = model.forward(nxt[b:b + 1], alone[b]).cpu()
                _model_close(got[b], want[0], PAGED_TOL, f"step {step} row {b}")
    assert batch.seq_lens == [52, 9, 34]
    model.free_unmanaged()


def test_all_logits_and_rewinding():
    """last_id_only=False gives every position; set_seq_lens drops tokens, and what comes again gives the same logits."""
    from exllama_amd.model import ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128
    model = _model(dims)
    ids = _ids(dims, 2, 40, seed=2)
    cache = ExLlamaPagedCache(model, batch_size=2, block_size=32)
    every = model.forward(ids, cache, last_id_only=False).cpu()
    assert every.shape == (2, 40, dims.vocab_size)
    cache.set_seq_lens([32, 0])                                   # a page's end, and the beginning: the pages begin anew, with scales of their own tokens
    again = model.forward(ids[:, 32:], cache, last_id_only=False, row_lens=[8, 0]).cpu()
    _model_close(again[0], every[0, 32:], PAGED_TOL, "rewound")
    assert cache.seq_lens == [40, 0]
    cache.current_seq_len = 0
    _model_close(model.forward(ids, cache).cpu()[:, 0], every[:, -1], PAGED_TOL, "anew")
    model.free_unmanaged()


def test_pages_are_given_back_and_taken_again():
    """A pool that holds half of what the rows could reach: a row that has ended makes room for another, the device's bookkeeping and the host's agree."""
    from exllama_amd.model import ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128
    model = _model(dims)
    cache = ExLlamaPagedCache(model, batch_size=3, block_size=16, num_blocks=12, dtype=torch.int8)
    ids = _ids(dims, 3, 70, seed=3)
    model.forward(ids, cache, row_lens=[70, 50, 33], preprocess_only=True)     # 5 + 4 + 3 blocks: all of them
    with pytest.raises(RuntimeError, match="release rows"):
        model.forward(ids[:, :20], cache, row_lens=[20, 0, 0])
    assert cache.seq_lens == [70, 50, 33]                         # (nothing was done)
    cache.release(1)
    assert cache.seq_lens == [70, 0, 33]
    one = ExLlamaPagedCache(model, block_size=16, dtype=torch.int8)
    got = model.forward(ids[:, :40], cache, row_lens=[0, 40, 0]).cpu()
    _model_close(got[1], model.forward(ids[1:2, :40], one).cpu()[0], PAGED_TOL, "on pages of another row")
    d = cache._dev["cuda:0"]
    assert d["held"].tolist() == cache._held == [5, 3, 3] and d["counters"].tolist()[1] == cache._free == 1 and d["counters"].tolist()[2] == 0
    cache.zero()
    assert cache.seq_lens == [0, 0, 0] and cache._free == 12 and d["counters"].tolist()[1] == 12
    assert sorted(d["ring"].tolist()) == list(range(12)) and bool((d["table"] == -1).all())
    model.free_unmanaged()


def test_refusals():
    from exllama_amd.model import ExLlamaCache, ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128
    model = _model(dims)
    ids = _ids(dims, 2, 8)
    cache = ExLlamaPagedCache(model, batch_size=2, max_seq_len=64)
    for kw in ({"input_mask": torch.ones(2, 8, dtype=torch.bool)}, {"row_lens": [8]}, {"row_lens": [9, 1]}, {"row_lens": [-1, 1]}):
        with pytest.raises(RuntimeError):
            model.forward(ids, cache, **kw)
    with pytest.raises(RuntimeError, match="rows"):
        model.forward(ids[:1], cache)
    with pytest.raises(RuntimeError, match="exceeds the cache length"):
        model.forward(_ids(dims, 2, 65), cache)
    with pytest.raises(RuntimeError, match="row_lens needs"):
        model.forward(ids, ExLlamaCache(model, batch_size=2), row_lens=[8, 8])
    with pytest.raises(RuntimeError, match="fp16"):
        model.enable_decode_graph(cache)
    with pytest.raises(RuntimeError, match="longer"):
        ExLlamaPagedCache(model, max_seq_len=10 ** 6)
    with pytest.raises(RuntimeError, match="dtype"):
        ExLlamaPagedCache(model, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="none longer"):
        cache.set_seq_lens([1, 0])
    with pytest.raises(RuntimeError, match="no such row"):
        cache.release(2)
    assert cache.seq_lens == [0, 0]
    model.free_unmanaged()


def test_a_pass_in_chunks_is_refused_before_its_first_chunk():
    """max_input_len cuts the pass; what the pool or the rows cannot hold as a whole changes nothing."""
    from exllama_amd.model import ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128
    model = _model(dims, max_input_len=32)
    cache = ExLlamaPagedCache(model, batch_size=2, block_size=16, num_blocks=6, max_seq_len=100)
    ids = _ids(dims, 2, 120, seed=6)
    model.forward(ids[:, :10], cache, preprocess_only=True)
    state = {k: v.clone() for k, v in cache._dev["cuda:0"].items()}
    for n, match in ((80, "release rows"), (120, "exceeds the cache length")):
        with pytest.raises(RuntimeError, match=match):
            model.forward(ids[:, :n], cache)
        assert cache.seq_lens == [10, 10] and cache._held == [1, 1] and cache._free == 4
        assert all(torch.equal(v, state[k]) for k, v in cache._dev["cuda:0"].items())
    assert model.forward(ids[:, :38], cache).shape == (2, 1, dims.vocab_size) and cache.seq_lens == [48, 48] and cache._free == 0
    model.free_unmanaged()
