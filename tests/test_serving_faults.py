"""Calls of the serving operators that must be refused or must leave everything as it was, on the CPU."""

from __future__ import annotations

import pytest
import torch

from tests.serving_reference import Batch


@pytest.fixture(scope="module")
def F():
    from cs244c_llama_zero_b200 import ops

    if not ops.extension_available():
        pytest.skip("extension not built")
    from cs244c_llama_zero_b200.ops import functional

    return functional


def _moved(t: torch.Tensor, by: int) -> torch.Tensor:
    """The tensor's values in a contiguous view that starts ``by`` elements into its storage."""
    base = torch.zeros(t.numel() + by, dtype=t.dtype)
    view = base[by:].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("by", [1, 2, 3])
def test_scales_off_a_16_byte_boundary_are_refused(F, which, by):
    """The kernel for few rows copies scales 16 bytes at a time; every operator refuses them alike."""
    b = Batch([2, 1], [5, 17], 4, 2, 64, "int8", 16)
    pages = b.pages()
    bad = pages._replace(**{which: _moved(getattr(pages, which), by)})
    calls = [lambda p: F.paged_attention(b.q, p, b.table, b.lens, b.starts, b.max_q),
             lambda p: F.kv_cache_write(p, b.k, b.v, b.table, b.lens, b.starts),
             lambda p: F.kv_cache_read(p, b.table, b.lens, b.starts, total=3)]
    for call in calls:
        with pytest.raises(RuntimeError, match=which + " must be 16-byte aligned"):
            call(bad)
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):  # 16 bytes further on they pass
            call(pages._replace(**{which: _moved(getattr(pages, which), 4)}))


@pytest.mark.parametrize("scale", [1e-50, 1e-39, 0.0, -1.0, 1e31, float("inf"), float("nan")])
def test_scales_that_fp32_cannot_hold_are_refused(F, scale):
    """The kernels multiply in fp32: what is 0 or not normal there is refused, not passed on as 0."""
    b = Batch([2, 1], [5, 17], 4, 2, 64, "bf16", 16)
    with pytest.raises(RuntimeError, match="scale must be"):
        F.paged_attention(b.q, b.pages(), b.table, b.lens, b.starts, b.max_q, scale=scale)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.paged_attention(b.q, b.pages(), b.table, b.lens, b.starts, b.max_q, scale=2.0 ** -126)


# ------------------------------------------------------------------------------------------ decoding over a cache
def _model(**kw):
    """A model whose decode_step runs on the CPU up to the first kernel."""
    from cs244c_llama_zero_b200.models import LlamaForCausalLM, ModelConfig

    args = dict(name="t", vocab_size=97, max_seq_len=64, dim=256, n_layers=3, n_heads=4, n_kv_heads=2, ffn_dim=256)
    model = LlamaForCausalLM(ModelConfig(**{**args, **kw})).eval()
    model.backend = "b200"
    return model


def _cache(model, **kw):
    from cs244c_llama_zero_b200.models import PagedKVCache

    args = {**model.cfg.__dict__, **kw}
    return PagedKVCache.for_batch(type(model.cfg)(**args), 2, 40, page_size=16, device="cpu")


@pytest.mark.parametrize("change", [dict(n_layers=2), dict(n_layers=4), dict(n_kv_heads=1), dict(dim=512)])
def test_a_cache_of_another_model_is_refused(F, monkeypatch, change):
    """Fewer layers in the cache than in the model would leave the model's last ones out."""
    monkeypatch.setattr(F, "decode_block", lambda x, *a: x)
    model = _model()
    cache = _cache(model, **change)
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="decode_step: the cache"):
        model.decode_step(ids, cache, [0, 1], [2, 1], [None] * 3)
    assert cache.length(0) == 0 and cache.free_pages == 6


@pytest.mark.parametrize("count", [0, 2, 4])
def test_weights_of_other_layers_are_refused(F, monkeypatch, count):
    monkeypatch.setattr(F, "decode_block", lambda x, *a: x)
    model = _model()
    with pytest.raises(ValueError, match="decode_step: weights"):
        model.decode_step(torch.zeros(3, dtype=torch.int64), _cache(model), [0, 1], [2, 1], [None] * count)


def test_every_layer_runs_once(F, monkeypatch):
    seen = []
    monkeypatch.setattr(F, "decode_block", lambda x, w, cfg, pages, *a: seen.append((w, pages)) or x)
    model = _model()
    cache = _cache(model)
    logits = model.decode_step(torch.zeros(3, dtype=torch.int64), cache, [0, 1], [2, 1], list("abc"))
    assert logits.shape == (2, 97)
    assert [w for w, _ in seen] == list("abc") and all(p is q for (_, p), q in zip(seen, cache.layers))
    assert cache.length(0) == 2 and cache.length(1) == 1


def _state(cache):
    return cache.free_pages, list(cache._free), [list(p) for p in cache._pages], [cache.length(s) for s in range(2)]


@pytest.mark.parametrize("where", ["first", "last", "positions"])
def test_a_step_that_fails_leaves_the_cache_as_it_was(F, monkeypatch, where):
    """Whatever refuses a step, the tokens that it did not compute are not counted as cached."""
    model = _model()
    cache = _cache(model)
    monkeypatch.setattr(F, "decode_block", lambda x, *a: x)
    model.decode_step(torch.zeros(18, dtype=torch.int64), cache, [0, 1], [15, 3], [None] * 3)
    before = _state(cache)
    calls = []

    def block(x, *a):
        calls.append(1)
        if where == "first" or len(calls) == 3:
            raise RuntimeError("refused")
        return x

    monkeypatch.setattr(F, "decode_block", block)
    if where == "positions":
        def tables(*a):
            raise RuntimeError("refused")
        monkeypatch.setattr(F, "rope_tables_t", tables)
    with pytest.raises(RuntimeError, match="refused"):
        model.decode_step(torch.zeros(19, dtype=torch.int64), cache, [1, 0], [14, 5], [None] * 3)
    assert _state(cache) == before
    step = cache.extend([0, 1], [1, 1])  # and it goes on from there
    assert step.kv_lens.tolist() == [16, 4] and step.positions.tolist() == [15, 3]


@pytest.mark.parametrize("seq", [-1, -2, 2, 100])
def test_sequences_that_do_not_exist_are_refused(F, seq):
    """A negative number is not the sequence counted from the end: -1 and 1 would be one sequence twice."""
    model = _model()
    cache = _cache(model)
    cache.extend([0, 1], [17, 3])
    before = _state(cache)
    for call in (lambda: cache.length(seq), lambda: cache.release(seq), lambda: cache.extend([seq], [1]),
                 lambda: cache.extend([1, seq], [1, 1]), lambda: cache.retract([seq], [1]),
                 lambda: model.decode_step(torch.zeros(2, dtype=torch.int64), cache, [1, seq], [1, 1], [None] * 3)):
        with pytest.raises(IndexError, match="no sequence"):
            call()
    assert _state(cache) == before


@pytest.mark.parametrize("name", ["bias", "repetition_penalty", "frequency_penalty", "presence_penalty", "out"])
def test_logit_parts_that_want_a_gradient_are_refused(F, name):
    """There is no backward pass: none is dropped in silence, whichever tensor asks for it."""
    one = torch.ones(2)
    args = dict(logits=torch.zeros(2, 40), history=torch.zeros(2, 3, dtype=torch.int64),
                history_lens=torch.zeros(2, dtype=torch.int32), repetition_penalty=one, frequency_penalty=one,
                presence_penalty=one, bias=torch.zeros(40), out=torch.zeros(2, 40))
    args[name] = args[name].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        F.adjust_logits(**args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.adjust_logits(**args)


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "out"])
def test_pages_that_want_a_gradient_are_refused(F, name):
    b = Batch([2, 1], [5, 17], 4, 2, 64, "int8" if "scale" in name else "bf16", 16)
    pages, out = b.pages(), torch.zeros_like(b.q)
    if name == "out":
        out.requires_grad_()
    else:
        pages = pages._replace(**{name: getattr(pages, name).clone().requires_grad_()})
    calls = [lambda: F.paged_attention(b.q, pages, b.table, b.lens, b.starts, b.max_q, out=out)]
    if name != "out":
        calls += [lambda: F.kv_cache_write(pages, b.k, b.v, b.table, b.lens, b.starts),
                  lambda: F.kv_cache_read(pages, b.table, b.lens, b.starts, total=3)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()


def test_retract_takes_no_more_than_there_is(F):
    cache = _cache(_model())
    cache.extend([0, 1], [17, 3])
    before = _state(cache)
    for seqs, rows in (([0, 0], [9, 9]), ([1], [4]), ([0], [-1]), ([0, 1], [1])):
        with pytest.raises(ValueError, match="retract"):
            cache.retract(seqs, rows)
    assert _state(cache) == before
    cache.retract([0, 1], [2, 3])
    assert cache.length(0) == 15 and cache.length(1) == 0 and cache.free_pages == 5


# ------------------------------------------------------------------------------------------ generation without a cache
def _generate_by_concatenation(model, ids, count, temperature, top_k):
    """Generation by appending each token to a tensor of its own."""
    with torch.no_grad():
        for _ in range(count):
            last = model(ids[:, -model.cfg.max_seq_len:]).logits[:, -1]
            ids = torch.cat([ids, model._pick_next(last, temperature, top_k)], dim=1)
    return ids


@pytest.mark.parametrize("prompt", [1, 7, 16, 23])
@pytest.mark.parametrize("temperature,top_k", [(0.0, None), (1.0, None), (0.7, 5)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_generation_without_a_cache(prompt, temperature, top_k, dtype):
    """Several sequences, prompts shorter and longer than the window, and past its end."""
    from cs244c_llama_zero_b200.models import LlamaForCausalLM, ModelConfig

    torch.manual_seed(1)
    model = LlamaForCausalLM(ModelConfig(name="t", vocab_size=97, max_seq_len=16, dim=64, n_layers=2, n_heads=4,
                                         n_kv_heads=2, ffn_dim=64, initializer_range=0.2)).eval()
    ids = torch.randint(0, 97, (3, prompt), dtype=dtype)
    torch.manual_seed(2)
    want = _generate_by_concatenation(model, ids, 20, temperature, top_k)
    torch.manual_seed(2)
    got = model.generate(ids, 20, temperature=temperature, top_k=top_k)
    assert got.dtype == want.dtype and torch.equal(got, want)
