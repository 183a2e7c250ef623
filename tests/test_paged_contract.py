"""What the paged 8-bit cache promises at its borders, on the CPU: rows that lost tokens, sizes at the end of 32 bits, refusals with a message."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P


def test_a_row_that_lost_tokens_gets_no_block():
    """past_lens beyond the held blocks: no block and no slot, what is lacking counts; set back, or with nothing held and nothing new, the row is served."""
    def call(past, new, held):
        table, ring, counters = np.full((2, 6), -1, np.int32), np.arange(8, dtype=np.int32), np.array([2, 6, 0, 0], np.int32)
        table[0, :held] = [0, 1][:held]
        held = np.array([held, 0], np.int32)
        _, slots, _ = P.slots(np.array([past, 0]), np.array([new, 3]), held, table, ring, counters, 16, 96, 8, 8)
        return held.tolist(), slots.tolist(), int(counters[2])

    assert call(33, 2, 2) == ([2, 1], [-1, -1, 32, 33, 34, -1, -1, -1], 1)
    assert call(33, 0, 2) == ([2, 1], [32, 33, 34, -1, -1, -1, -1, -1], 1)
    assert call(1, 1, 0) == ([0, 1], [-1, 32, 33, 34, -1, -1, -1, -1], 1)
    assert call(32, 2, 2) == ([3, 1], [32, 33, 48, 49, 50, -1, -1, -1], 0)
    assert call(33, 0, 0) == ([3, 1], [80, 81, 82, -1, -1, -1, -1, -1], 0)


@pytest.fixture(scope="module")
def ext():
    from exllama_amd import cuda_ext
    return cuda_ext


def test_attention_refuses_tables_at_the_end_of_32_bits(ext):
    """A length is rounded up to a tile of 64 keys in 32 bits: tables of more than 2^31 - 65 tokens are refused, the largest below is not (it is refused for its
    workspace, the last check before a launch)."""
    lib = ext._lib.load()
    p, far = C.c_void_p(4096), C.c_void_p(1 << 20)            # never read: every call below is refused first

    def attention(width, block, rows):
        assert lib.exl_paged_attention(p, 64, p, p, p, 1, rows, rows, p, width, p, p, p, p, 0, 8, block, 1, 1, 64, 0.0, None, None, 0, far, None, 0, None) < 0
        return lib.exl_last_error().decode()

    for rows in (1, 40):
        for block in (16, 32, 64, 128):
            most = (2 ** 31 - 65) // block
            assert "workspace" in attention(most, block, rows)
            assert "block table" in attention(most + 1, block, rows), block


# ---- the model's side ---------------------------------------------------------------------------------------------------------------------

def _bare_cache(batch_size=1):
    from exllama_amd.model import ExLlamaPagedCache
    cache = object.__new__(ExLlamaPagedCache)                 # (no device here: what is asked of it below needs none of its tensors)
    cache.batch_size, cache.step = batch_size, {}
    return cache


@pytest.mark.parametrize("batch_size", [1, 8])
def test_the_decode_report_names_the_path_of_a_paged_cache(batch_size):
    import types

    from exllama_amd.model import ExLlama
    model = object.__new__(ExLlama)
    model._decoder, model.layers = None, []
    model.config = types.SimpleNamespace(tp=None, fused_attn=True, head_dim=128, hidden_size=4096, intermediate_size=11008,
                                         device_map=types.SimpleNamespace(layers=["cuda:0"]))
    report = model.decode_path_report(_bare_cache(batch_size))
    assert report["tier"] == "ops_general" and len(report["why_not_faster"]) == 1 and "ExLlamaPagedCache" in report["why_not_faster"][0]
    other = types.SimpleNamespace(batch_size=batch_size)      # any other cache is answered as before
    assert model.decode_path_report(other)["tier"] == ("ops_fused" if batch_size == 1 else "layer_call")


def test_what_a_paged_cache_cannot_do_it_refuses_with_a_message():
    cache = _bare_cache()
    for call in (cache.roll_left, cache.clone, lambda: cache.copy_states(cache, 0, 1, 0, 1, 0, 1, 0, 1)):
        with pytest.raises(RuntimeError, match="ExLlamaPagedCache"):
            call()


@pytest.mark.parametrize("kw,match", [({"block_size": 24}, "block_size"), ({"block_size": 256}, "block_size"), ({"num_blocks": 0}, "one block"),
                                      ({"num_blocks": -3}, "one block"), ({"batch_size": 0}, "one row"), ({"dtype": torch.float16}, "dtype")])
def test_a_paged_cache_that_cannot_work_is_refused_before_it_takes_memory(kw, match):
    import types

    from exllama_amd.model import ExLlamaPagedCache
    config = types.SimpleNamespace(tp=None, max_seq_len=64, head_dim=64, num_hidden_layers=1, num_key_value_heads=1,
                                   device_map=types.SimpleNamespace(layers=["meta"]))
    with pytest.raises(RuntimeError, match=match):
        ExLlamaPagedCache(types.SimpleNamespace(config=config), **kw)
