"""Page bookkeeping of the key/value cache and the refusals of cached decoding, on the CPU."""

from __future__ import annotations

import pytest
import torch

from cs244c_llama_zero_b200.models import LlamaForCausalLM, ModelConfig, PagedKVCache


def _cfg(**kw):
    args = dict(name="t", vocab_size=97, max_seq_len=64, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=256)
    args.update(kw)
    return ModelConfig(**args)


def test_pages_are_handed_out_once_and_returned():
    cache = PagedKVCache(_cfg(), n_pages=6, page_size=16, dtype="int8", device="cpu")
    a, b = cache.add_sequence(), cache.add_sequence()
    step = cache.extend([a, b], [17, 3])
    assert step.kv_lens.tolist() == [17, 3] and step.q_starts.tolist() == [0, 17, 20] and step.max_q_len == 17
    assert step.positions.tolist() == list(range(17)) + [0, 1, 2]
    used = step.block_table[0, :2].tolist() + step.block_table[1, :1].tolist()
    assert len(set(used)) == 3 and cache.free_pages == 3
    step = cache.extend([b, a], [1, 1])
    assert step.q_starts is None and step.kv_lens.tolist() == [4, 18] and step.positions.tolist() == [3, 17]
    assert step.block_table[1, :2].tolist() == used[:2] and cache.free_pages == 3
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.extend([a, b], [1, 61])
    assert cache.length(a) == 18 and cache.length(b) == 4 and cache.free_pages == 3
    cache.release(a)
    assert cache.free_pages == 5 and cache.length(a) == 0
    again = cache.extend([a], [80])
    assert sorted(again.block_table[0].tolist()) == sorted(set(range(6)) - {used[2]})


def test_bad_arguments():
    cfg = _cfg()
    for kw, match in ((dict(dtype="fp4"), "cache dtype"), (dict(page_size=24), "page_size"), (dict(n_pages=0), "n_pages")):
        with pytest.raises(ValueError, match=match):
            PagedKVCache(cfg, **{**dict(n_pages=2, device="cpu"), **kw})
    cache = PagedKVCache.for_batch(cfg, 2, 20, page_size=16, device="cpu")
    assert cache.free_pages == 4 and cache.layers[0].k.shape == (4, 2, 16, 64) and cache.layers[0].k_scale is None
    for seqs, rows in (([0, 0], [1, 1]), ([0], [1, 2]), ([0], [-1])):
        with pytest.raises(ValueError, match="extend"):
            cache.extend(seqs, rows)


def test_cached_generation_needs_the_b200_backend():
    model = LlamaForCausalLM(_cfg()).eval()
    ids = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="b200 backend"):
        model.generate(ids, 2, kv_cache="bf16")
    with pytest.raises(ValueError, match="b200 backend"):
        model.generate(ids, 2, repetition_penalty=1.2)
    with pytest.raises(ValueError, match="b200 backend"):
        model.decode_weights()
    assert torch.equal(model.generate(ids, 0), ids) and torch.equal(model.generate(ids, -3), ids)
    assert model.generate(ids.int(), 2, temperature=0.0).dtype == torch.int64
