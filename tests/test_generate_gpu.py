"""Cached generation on the B200 backend against the eager model that recomputes every token."""

from __future__ import annotations

import pytest
import torch

from cs244c_llama_zero_b200.models import LlamaForCausalLM, ModelConfig, PagedKVCache

pytestmark = pytest.mark.gpu


def _models(hd, tied=True, max_seq_len=300):
    cfg = ModelConfig(name="gen", vocab_size=1000, max_seq_len=max_seq_len, dim=4 * hd, n_layers=3, n_heads=4,
                      n_kv_heads=2, ffn_dim=512, tie_word_embeddings=tied, initializer_range=0.08)
    torch.manual_seed(3)
    eager = LlamaForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    fast = LlamaForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    fast.load_state_dict(eager.state_dict())
    fast.set_backend("b200")
    oracle = LlamaForCausalLM(cfg).cuda().double().eval()
    oracle.load_state_dict({k: v.double() for k, v in eager.state_dict().items()})
    return cfg, eager, fast, oracle


@pytest.mark.parametrize("hd,tied", [(64, True), (128, False)])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3", "int8"])
def test_logits_of_prompts_chunks_and_single_tokens(hd, tied, dtype):
    """Prompts of odd lengths, cut into chunks, then single tokens: the logits after every step are as close
    to the 64-bit model as those of the eager bf16 model are (unquantised: 1.5 times its error; 8-bit caches
    add the rounding of K and V, a relative 2^-4 for e4m3 and 1/254 of a row's maximum for int8, which the
    factors leave room for)."""
    cfg, eager, fast, oracle = _models(hd, tied)
    ids = torch.randint(0, cfg.vocab_size, (2, 200), device="cuda")
    cache = PagedKVCache.for_batch(cfg, 2, 200, page_size=16, dtype=dtype)
    weights = fast.decode_weights()
    have = [0, 0]
    with torch.no_grad():
        for rows in ((70, 33), (61, 1), (1, 100), (1, 1), (1, 1), (3, 2)):
            new = torch.cat([ids[s, h:h + n] for s, (h, n) in enumerate(zip(have, rows))])
            got = fast.decode_step(new, cache, [0, 1], rows, weights)
            have = [h + n for h, n in zip(have, rows)]
            for s in range(2):
                want = oracle(ids[s:s + 1, :have[s]]).logits[0, -1]
                plain = eager(ids[s:s + 1, :have[s]]).logits[0, -1]
                err, base = (got[s].double() - want).norm(), (plain.double() - want).norm()
                factor = {"bf16": 1.5, "int8": 4.0, "e4m3": 12.0}[dtype]
                assert err <= factor * base + 1e-3 * want.norm(), (rows, s, float(err / want.norm()),
                                                                   float(base / want.norm()))


def test_generate_with_cache_equals_recomputation():
    """Greedy tokens with the cache are those of the same backend without it, where that one accepts the
    length (128), as long as the two best logits are further apart than both paths' rounding."""
    cfg, eager, fast, oracle = _models(64, max_seq_len=140)
    ids = torch.randint(0, cfg.vocab_size, (3, 128), device="cuda")
    with torch.no_grad():
        cached = fast.generate(ids, 12, temperature=0.0, kv_cache="bf16")
        assert torch.equal(cached[:, :128], ids)
        for n in range(128, 140):  # every pick is (nearly) the 64-bit model's best for the same prefix
            logits = oracle(cached[:, :n]).logits[:, -1]
            picked = logits.gather(1, cached[:, n:n + 1])[:, 0]
            spread = logits.std(dim=-1)
            assert (picked >= logits.amax(-1) - 0.05 * spread).all()


def test_generate_adjusts_logits():
    cfg, eager, fast, oracle = _models(64)
    ids = torch.randint(0, cfg.vocab_size, (2, 17), device="cuda")
    words = (cfg.vocab_size + 31) // 32
    allowed = torch.zeros(words, dtype=torch.int32, device="cuda")
    allowed[3] = -1  # tokens 96 .. 127
    out = fast.generate(ids, 20, temperature=0.0, kv_cache="int8", frequency_penalty=1e4, allowed_tokens=allowed)
    new = out[:, 17:]
    assert ((new >= 96) & (new < 128)).all()
    for row in new.tolist():
        assert len(set(row)) == len(row)  # nothing twice while there is something else
    bias = torch.zeros(cfg.vocab_size, device="cuda")
    bias[5] = 1e4
    assert (fast.generate(ids, 3, temperature=1.0, top_k=5, kv_cache="e4m3", logit_bias=bias)[:, 17:] == 5).all()


def test_refusals():
    cfg, eager, fast, oracle = _models(64)
    ids = torch.zeros(1, 290, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="do not fit"):
        fast.generate(ids, 12, kv_cache="bf16")
    assert fast.generate(ids, 11, temperature=0.0, kv_cache="bf16").shape == (1, 301)
    cache = PagedKVCache.for_batch(cfg, 1, 300)
    with pytest.raises(ValueError, match="at least one row"):
        fast.decode_step(ids[0, :0], cache, [0], [0])
    with pytest.raises(ValueError, match="max_seq_len"):
        fast.decode_step(torch.zeros(301, dtype=torch.int64, device="cuda"), cache, [0], [301])
