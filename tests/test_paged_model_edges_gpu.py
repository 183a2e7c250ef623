"""ExLlama over an ExLlamaPagedCache beyond its forward pass: what it reports and what it refuses."""
import pytest
import torch

from exllama_amd import synth
from test_paged_model_gpu import _ids, _model

pytestmark = pytest.mark.gpu


def test_single_token_passes_are_counted_and_no_prompt():
    from exllama_amd.model import ExLlamaCache, ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128
    model = _model(dims, max_input_len=32)
    cache, fp16 = ExLlamaPagedCache(model, batch_size=2, block_size=16), ExLlamaCache(model)
    model.reset_decode_path_counts()
    model.forward(_ids(dims, 2, 50), cache, preprocess_only=True)             # four chunks, none of them a single-token pass
    assert model.decode_path_report(cache)["forwards_by_tier"] == {}
    for _ in range(3):
        model.forward(_ids(dims, 2, 1), cache)
    report = model.decode_path_report(cache)
    assert report["forwards_by_tier"] == {"ops_general": 3} and report["last_forward_tier"] == report["tier"] == "ops_general"
    model.forward(_ids(dims, 1, 4), fp16, preprocess_only=True)
    model.forward(_ids(dims, 1, 1), fp16)
    assert model.decode_path_report(fp16)["last_forward_tier"] == model.decode_path_report(fp16)["tier"] == "ops_fused"
    model.free_unmanaged()


def test_layers_without_a_prepared_pass_are_refused():
    """forward_layers by itself (a link of a layer split runs it so) has no slots for the tokens: a message, and nothing is written."""
    from exllama_amd.model import ExLlamaPagedCache
    dims = synth.LLAMA_TINY_HD128
    model = _model(dims)
    cache = ExLlamaPagedCache(model, block_size=16)
    ids = _ids(dims, 1, 5)
    with pytest.raises(RuntimeError, match="ExLlama.forward"):
        model.forward_layers(model.embed(ids), cache)
    assert cache.seq_lens == [0] and not any(bool(p.view(torch.uint8).any()) for p in cache.pages[0][:2])
    model.forward(ids, cache, preprocess_only=True)
    with pytest.raises(RuntimeError, match="ExLlama.forward"):
        model.forward_layers(model.embed(ids), cache)
    assert cache.seq_lens == [5]
    model.free_unmanaged()
