"""Refusals of the serving operators, on the CPU: every check on shapes and types comes before the device."""

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


def _batch(fmt="e4m3", **kw):
    args = dict(q_lens=[2, 1], kv_lens=[5, 17], heads=4, kv_heads=2, hd=64, fmt=fmt, page=16)
    args.update(kw)
    return Batch(**args)


def test_cpu_tensors_are_refused_last(F):
    b = _batch()
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.paged_attention(b.q, b.pages(), b.table, b.lens, b.starts, b.max_q)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.kv_cache_write(b.pages(), b.k, b.v, b.table, b.lens, b.starts)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.kv_cache_read(b.pages(), b.table, b.lens, b.starts, total=3)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        F.adjust_logits(torch.zeros(2, 10))


@pytest.mark.parametrize("change,match", [
    (dict(k=lambda p: p.k.half()), "one shape|same dtype"),
    (dict(k=lambda p: p.k.float(), v=lambda p: p.v.float()), "bfloat16, float8_e4m3fn or int8"),
    (dict(k_scale=lambda p: None), "need k_scale and v_scale"),
    (dict(k_scale=lambda p: p.k_scale.double()), "contiguous float32"),
    (dict(v_scale=lambda p: p.v_scale[:, :1]), "contiguous float32"),
    (dict(k=lambda p: p.k[:, :, :12].contiguous(), v=lambda p: p.v[:, :, :12].contiguous()), "page_size must be"),
    (dict(k=lambda p: p.k[:0], v=lambda p: p.v[:0], k_scale=lambda p: p.k_scale[:0], v_scale=lambda p: p.v_scale[:0]),
     "at least one page"),
    (dict(k=lambda p: p.k[..., :32].contiguous(), v=lambda p: p.v[..., :32].contiguous()), "head_dim must be 64 or 128"),
    (dict(v=lambda p: p.v.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
])
def test_bad_pages(F, change, match):
    b = _batch()
    pages = b.pages()
    pages = pages._replace(**{k: f(pages) for k, f in change.items()})
    with pytest.raises(RuntimeError, match=match):
        F.paged_attention(b.q, pages, b.table, b.lens, b.starts, b.max_q)
    with pytest.raises(RuntimeError, match=match):
        F.kv_cache_write(pages, b.k, b.v, b.table, b.lens, b.starts)


def test_bf16_pages_take_no_scales(F):
    b = _batch("bf16")
    pages = b.pages()._replace(k_scale=torch.zeros(b.n_pages, 2, 16), v_scale=torch.zeros(b.n_pages, 2, 16))
    with pytest.raises(RuntimeError, match="bf16 pages have none"):
        F.kv_cache_read(pages, b.table, b.lens, b.starts, total=3)


def test_bad_batches(F):
    b = _batch()
    p = b.pages()
    cases = [
        ((b.q, p, b.table.long(), b.lens, b.starts, 2), "block_table must be int32"),
        ((b.q, p, b.table, b.lens[:1], b.starts, 2), "kv_lens must be"),
        ((b.q, p, b.table, b.lens.long(), b.starts, 2), "kv_lens must be"),
        ((b.q, p, b.table, b.lens, b.starts[:2], 2), "q_starts must be"),
        ((b.q, p, b.table, b.lens), "one new token"),
        ((b.q, p, b.table, b.lens, b.starts, 0), "max_q_len"),
        ((b.q.float(), p, b.table, b.lens, b.starts, 2), "must be bfloat16"),
        ((b.q[:, :3], p, b.table, b.lens, b.starts, 2), "multiple of kv_heads"),
        ((b.q[..., :32], p, b.table, b.lens, b.starts, 2), "q must be"),
        ((b.q.transpose(1, 2).contiguous().transpose(1, 2), p, b.table, b.lens, b.starts, 2), "unit stride"),
    ]
    for args, match in cases:
        with pytest.raises(RuntimeError, match=match):
            F.paged_attention(*args)
    with pytest.raises(ValueError, match="max_q_len"):
        F.paged_attention(b.q, p, b.table, b.lens, b.starts)
    with pytest.raises(ValueError, match="total"):
        F.kv_cache_read(p, b.table, b.lens, b.starts)
    with pytest.raises(RuntimeError, match="share memory"):
        F.paged_attention(b.q, p, b.table, b.lens, b.starts, 2, out=b.q)
    with pytest.raises(RuntimeError, match="overlap"):
        F.paged_attention(b.q, p, b.table, b.lens, b.starts, 2, out=torch.zeros(999, dtype=torch.bfloat16).as_strided((3, 4, 64), (64, 64, 1)))
    with pytest.raises(RuntimeError, match="scale must be"):
        F.paged_attention(b.q, p, b.table, b.lens, b.starts, 2, scale=float("nan"))
    odd = torch.zeros(3, 4 * 64 + 4, dtype=torch.bfloat16)[:, :256].view(3, 4, 64)
    with pytest.raises(RuntimeError, match="positive multiples of 8"):
        F.paged_attention(odd, p, b.table, b.lens, b.starts, 2)
    with pytest.raises(RuntimeError, match="k must be"):
        F.kv_cache_write(p, b.k[:, :1], b.v, b.table, b.lens, b.starts)
    with pytest.raises(RuntimeError, match="bfloat16 or float32"):
        F.kv_cache_read(p, b.table, b.lens, b.starts, total=3, dtype=torch.float16)


def test_no_backward(F):
    b = _batch()
    with pytest.raises(RuntimeError, match="no backward"):
        F.paged_attention(b.q.float().requires_grad_().bfloat16(), b.pages(), b.table, b.lens, b.starts, 2)
    with pytest.raises(RuntimeError, match="no backward"):
        F.adjust_logits(torch.zeros(2, 8, requires_grad=True))


def test_bad_logits(F):
    x = torch.zeros(2, 40)
    hist, lens, one = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.ones(2)
    cases = [
        (dict(logits=x.double()), "bfloat16, float16 or float32"),
        (dict(logits=x.t()), "unit column stride"),
        (dict(logits=x, repetition_penalty=one), "need a history"),
        (dict(logits=x, history=hist), "go together"),
        (dict(logits=x, prompt_lens=lens), "needs a history"),
        (dict(logits=x, history=hist.int(), history_lens=lens, repetition_penalty=one), "history must be int64"),
        (dict(logits=x, history=hist, history_lens=lens, repetition_penalty=one.double()), "repetition_penalty"),
        (dict(logits=x, history=hist, history_lens=lens.long(), frequency_penalty=one), "history_lens"),
        (dict(logits=x, bias=torch.zeros(39)), "bias must be"),
        (dict(logits=x, bias=torch.zeros(40).half()), "bias must be"),
        (dict(logits=x, allowed=torch.zeros(1, dtype=torch.int32)), "bitmask"),
        (dict(logits=x, out=torch.zeros(2, 40).half()), "shape and dtype"),
        (dict(logits=torch.zeros(3, 40)[:2], out=torch.zeros(1, 40).expand(2, 40)), "overlap"),
    ]
    for kw, match in cases:
        with pytest.raises(RuntimeError, match=match):
            F.adjust_logits(**kw)
    wide = torch.zeros(2, 80)
    with pytest.raises(RuntimeError, match="share memory"):
        F.adjust_logits(wide[:, :40], out=wide[:, 20:60])


# ------------------------------------------------------------------------------------------ work division
@pytest.mark.parametrize("tile_tokens,unit_log2,grid", [(16, 6, 296), (2, 6, 5), (64, 7, 148), (42, 7, 7), (256, 7, 1),
                                                        (1, 6, 592)])
@pytest.mark.parametrize("seed", range(4))
def test_every_unit_is_done_once(F, tile_tokens, unit_log2, grid, seed):
    """The blocks' ranges cover all units of all items once, in order, and no block has more to do than its
    share (units, and two places for each item that begins in it) and one item's start."""
    from cs244c_llama_zero_b200 import ops

    from tests.serving_reference import ragged

    q, kv = ragged(seed, (1, 3, 40, 300)[seed], (1, 200, 90, 3)[seed], (5000, 700, 300, 900)[seed])
    q[-1] = max(q[-1], 1)
    kv[0] = 0  # rows that see nothing
    starts = torch.tensor([sum(q[:i]) for i in range(len(q) + 1)], dtype=torch.int32)
    lens = torch.tensor(kv, dtype=torch.int32)
    heads = 3
    parts = ops.load_extension().paged_schedule(starts, lens, 100_000, sum(q), max(q), heads, tile_tokens, unit_log2,
                                                grid)
    want = []
    for b, (n, t) in enumerate(zip(q, kv)):
        for h in range(heads):
            for rt in range(-(-n // tile_tokens)):
                visible = t - n + min(n, (rt + 1) * tile_tokens)
                want.append((b, h, rt, max(1, -(-visible // (1 << unit_log2)))))
    got, sizes = [], {}
    for block, b, h, rt, u0, u1, units in parts:
        sizes[block] = sizes.get(block, 0) + u1 - u0 + (2 if u0 == 0 else 0)
        assert 0 <= u0 < u1 <= units
        if u0 == 0:
            got.append([b, h, rt, 0])
        assert got[-1][:3] == [b, h, rt] and got[-1][3] == u0
        got[-1][3] = u1
    assert [tuple(g) for g in got] == want
    total = sum(w[3] + 2 for w in want)
    blocks = min(grid, total)
    assert list(sizes) == sorted(sizes) and max(sizes) < blocks
    assert max(sizes.values()) <= -(-total // blocks) + 2
    # at most two parts per block, its first and its last one
    for block in sizes:
        cut = [i for i, p in enumerate(q for q in parts if q[0] == block) if p[5] - p[4] != p[6]]
        assert set(cut) <= {0, sum(q[0] == block for q in parts) - 1}


def test_bad_sequences_get_no_units(F):
    from cs244c_llama_zero_b200 import ops

    starts = torch.tensor([0, 2, 1, 4, 9, 10], dtype=torch.int32)  # rows that run backwards, too many, too few
    lens = torch.tensor([64, 64, 65, 64, -1], dtype=torch.int32)  # 65: past the table
    parts = ops.load_extension().paged_schedule(starts, lens, 64, 10, 4, 1, 4, 6, 8)
    assert [p[1:] for p in parts] == [[0, 0, 0, 0, 1, 1]]
