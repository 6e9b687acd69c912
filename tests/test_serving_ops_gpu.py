"""The serving operators on the GPU against plain 64-bit forms: paged cache, attention over it, logits."""

from __future__ import annotations

import pytest
import torch

from tests.serving_reference import FORMATS, Batch, adjusted, quantise, ragged, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F():
    from cs244c_llama_zero_b200 import ops
    from cs244c_llama_zero_b200.ops import functional

    ops.load_extension().reset_device_errors()
    yield functional
    ops.check_device_errors()


@pytest.fixture
def errors():
    """For tests that provoke error records: the record is read and cleared."""
    from cs244c_llama_zero_b200 import ops

    ext = ops.load_extension()
    assert list(ext.read_device_errors())[0] == 0
    yield lambda: list(ext.read_device_errors())
    ext.reset_device_errors()


def _meta(b, starts=True):
    return b.table.cuda(), b.lens.cuda(), b.starts.cuda() if starts else None


def _check(got, want, tol):
    bad = (got.double().cpu() - want).abs() > tol
    bad |= ~torch.isfinite(got.cpu())
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}, "
                           f"worst {(((got.double().cpu() - want).abs() / tol).max()):.3f} of the bound")


def _attend(F, b, **kw):
    table, lens, starts = _meta(b)
    return F.paged_attention(b.q.cuda(), b.pages("cuda"), table, lens, starts, b.max_q, **kw)


HEADS = [(12, 4, 64), (18, 6, 64), (32, 8, 64), (16, 8, 128), (32, 8, 128)]


# ------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens(F, fmt, heads, page):
    """One new token per sequence, lengths around every tile and page edge, an empty sequence among them."""
    kv = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 2]
    b = Batch([1] * len(kv), kv, *heads, fmt, page, seed=1)
    table, lens, _ = _meta(b)
    got = F.paged_attention(b.q.cuda(), b.pages("cuda"), table, lens)
    want, mag, size = b.attention()
    _check(got, want, tolerance(want, mag, size, fmt != "bf16"))
    assert (got[1] == 0).all()


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads", [(4, 4, 64), (14, 2, 128), (16, 1, 128), (5, 1, 64), (24, 1, 64), (40, 1, 128)])
def test_group_sizes(F, fmt, heads):
    """Groups of 1, 5, 7, 16, 24 and 40 query heads, for one and for several new tokens."""
    for q, kv in (([1, 1, 1], [33, 200, 5]), ([3, 1, 2], [33, 200, 5]), ([9, 40, 1], [130, 41, 260])):
        b = Batch(q, kv, *heads, fmt, 32, seed=2)
        want, mag, size = b.attention()
        _check(_attend(F, b), want, tolerance(want, mag, size, fmt != "bf16"))


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_chunks(F, fmt, heads, page):
    """Chunks of odd lengths over earlier tokens; sequences without new tokens between them."""
    b = Batch([130, 0, 1, 65, 17, 300, 43], [130, 50, 1, 200, 144, 311, 170], *heads, fmt, page, seed=3)
    want, mag, size = b.attention()
    _check(_attend(F, b), want, tolerance(want, mag, size, fmt != "bf16"))


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("q_len", [1, 2, 4, 7, 16])
def test_few_tokens_long_cache(F, fmt, q_len):
    """Few rows over a long cache: the token axis is split over the SMs and joined."""
    b = Batch([q_len, q_len], [5000, 3001], 8, 2, 128, fmt, 64, seed=4, amplitude=2.0)
    want, mag, size = b.attention()
    _check(_attend(F, b), want, tolerance(want, mag, size, fmt != "bf16"))


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("hd", [64, 128])
def test_items_that_span_blocks(F, fmt, hd):
    """Items of many units, cut by the blocks' ranges, with one tile or two and ends inside a tile: what a
    stage held before, and what lies behind the sequence in its last page, must not show."""
    for q, kv in (([200], [1500]), ([1, 17, 200], [3000, 900, 1500]), ([40, 64, 8], [2047, 2049, 1111])):
        b = Batch(q, kv, 8, 2, hd, fmt, 16, seed=15)
        want, mag, size = b.attention()
        _check(_attend(F, b), want, tolerance(want, mag, size, fmt != "bf16"))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads", [(12, 3, 64), (8, 2, 128)])
def test_long_chunks_of_8_bit_pages(F, fmt, heads):
    """Enough rows that the codes are expanded once for all of a sequence's tiles; short and empty sequences,
    rows behind the last one and a wide block table in the same batch; scales of very different size."""
    b = Batch([520, 0, 3, 300, 5], [700, 90, 3, 300, 0], *heads, fmt, 16, seed=17, behind=3)
    for which in range(2):  # every seventh token 2^12 times larger or smaller than the others
        b.scales[which][:, :, ::7] *= 2.0 ** (12 if which else -12)
    want, mag, size = b.attention()
    wide = torch.cat([b.table, torch.full((5, 40), b.n_pages + 9, dtype=torch.int32)], 1).cuda()
    out = torch.full(b.q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    F.paged_attention(b.q.cuda(), b.pages("cuda"), wide, b.lens.cuda(), b.starts.cuda(), b.max_q, out=out)
    _check(out[:b.total], want, tolerance(want, mag, size, True))
    assert (out[b.total:] == 7).all() and (out[b.total - 5:b.total] == 0).all()
    again = F.paged_attention(b.q.cuda(), b.pages("cuda"), wide, b.lens.cuda(), b.starts.cuda(), b.max_q)
    assert torch.equal(again[:b.total], out[:b.total])


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_rows_before_the_first_token_are_zero(F, fmt):
    """More new tokens than cached ones: the first rows stand before the sequence and see nothing."""
    for q, kv in (([5, 3], [2, 0]), ([200, 150], [60, 0])):
        b = Batch(q, kv, 12, 4, 64, fmt, 16, seed=5)
        want, mag, size = b.attention()
        got = _attend(F, b)
        _check(got, want, tolerance(want, mag, size, fmt != "bf16"))
        assert (got[:q[0] - kv[0]] == 0).all() and (got[q[0]:] == 0).all()


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [70, 3, 129]])
def test_strided_rows_and_rows_behind(F, q_lens):
    """q inside a wider projection, out inside a wider tensor; rows behind the last sequence stay."""
    kv = [n + 90 for n in q_lens]
    b = Batch(q_lens, kv, 16, 8, 128, "int8", 32, seed=6, behind=4)
    fused = torch.full((b.q.shape[0], 40, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    fused[:, 8:24] = b.q.cuda()
    wide = torch.full((b.q.shape[0], 20, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 2:18, :128]
    table, lens, starts = _meta(b)
    got = F.paged_attention(fused[:, 8:24], b.pages("cuda"), table, lens, starts, b.max_q, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, mag, size = b.attention()
    _check(out[:b.total], want, tolerance(want, mag, size, True))
    assert (wide[b.total:] == 7).all() and (wide[:, :2] == 7).all() and (wide[:, 18:] == 7).all()
    assert (wide[:, :, 128:] == 7).all()


@pytest.mark.parametrize("q_len", [1, 150])
def test_scale_and_large_scores(F, q_len):
    """Scores of several hundred: the running maximum moves far, and an explicit scale."""
    b = Batch([q_len], [700], 12, 4, 64, "bf16", 16, seed=7, amplitude=30.0)
    want, mag, size = b.attention(scale=0.3)
    _check(_attend(F, b, scale=0.3), want, tolerance(want, mag, size, False))


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_ragged_draws(F, fmt):
    for seed in range(4):
        q, kv = ragged(seed, 9, (1, 6, 40, 150)[seed], (900, 300, 300, 500)[seed])
        q[0] = max(1, q[0])
        b = Batch(q, [max(n, 1) for n in kv], *HEADS[seed], fmt, (16, 32, 64, 128)[seed], seed=seed + 20)
        want, mag, size = b.attention()
        _check(_attend(F, b), want, tolerance(want, mag, size, fmt != "bf16"))


def test_empty_batches(F):
    b = Batch([0, 0], [5, 0], 4, 2, 64, "bf16", 16)
    assert _attend(F, b).shape == (0, 4, 64)
    none = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    table, lens, _ = _meta(b)
    assert F.paged_attention(none, b.pages("cuda"), table[:0], lens[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [40, 30, 20, 10]])
def test_bad_metadata_is_skipped_and_recorded(F, errors, q_lens):
    """A page that does not exist reads as nothing wrong elsewhere; a length past the table skips the sequence."""
    kv = [n + 50 for n in q_lens]
    b = Batch(q_lens, kv, 8, 2, 64, "bf16", 16, seed=8)
    want, mag, size = b.attention()
    tol = tolerance(want, mag, size, False)
    for what in ("page", "length", "negative"):
        table, lens, starts = _meta(b)
        if what == "page":
            table[1, 1] = b.n_pages + 100
        elif what == "length":
            lens[1] = table.shape[1] * 16 + 1
        else:
            lens[1] = -3
        out = torch.full(b.q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
        F.paged_attention(b.q.cuda(), b.pages("cuda"), table, lens, starts, b.max_q, out=out)
        assert errors()[0] == 6
        rows = torch.ones(b.total, dtype=torch.bool)
        rows[int(b.starts[1]):int(b.starts[2])] = False
        _check(out[rows.cuda()], want[rows], tol[rows])
        if what != "page":
            assert (out[~rows.cuda()] == 9).all()
        from cs244c_llama_zero_b200 import ops

        ops.load_extension().reset_device_errors()


def test_too_many_new_tokens_are_skipped_and_recorded(F, errors):
    b = Batch([3, 20, 2], [30, 40, 50], 8, 2, 64, "int8", 16, seed=9)
    table, lens, starts = _meta(b)
    out = torch.full(b.q.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    F.paged_attention(b.q.cuda(), b.pages("cuda"), table, lens, starts, 4, out=out)
    assert errors()[0] == 6
    assert (out[3:23] == 9).all() and (out[:3] != 9).any() and (out[23:] != 9).any()


@pytest.mark.parametrize("q_lens", [[1, 1], [60, 9]])
def test_attention_graph_and_streams(F, q_lens):
    """Captured and replayed with new lengths; two streams at once."""
    b = Batch(q_lens, [400, 300], 16, 8, 128, "e4m3", 64, seed=10)
    pages, q = b.pages("cuda"), b.q.cuda()
    table, lens, starts = _meta(b)
    want = F.paged_attention(q, pages, table, lens, starts, b.max_q)
    short = lens - 100
    want_short = F.paged_attention(q, pages, table, short, starts, b.max_q)
    torch.cuda.synchronize()
    live = lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.paged_attention(q, pages, table, live, starts, b.max_q)
    graph.replay()
    assert torch.equal(out, want)
    live.copy_(short)
    graph.replay()
    assert torch.equal(out, want_short)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for s, ln in zip(streams, (lens, short)):
            with torch.cuda.stream(s):
                results.append(F.paged_attention(q, pages, table, ln, starts, b.max_q))
    torch.cuda.synchronize()
    for i, r in enumerate(results):
        assert torch.equal(r, want if i % 2 == 0 else want_short)


def test_attention_repeats_bit_for_bit(F):
    b = Batch([1, 17, 200], [3000, 900, 1500], 32, 8, 128, "bf16", 16, seed=11)
    first = _attend(F, b)
    for _ in range(3):
        assert torch.equal(_attend(F, b), first)


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("q_lens", [[1, 1], [70, 150], [520, 9]])
def test_head_major_queries(F, fmt, q_lens):
    """q as [heads, tokens, head_dim] in memory: the token stride is the smaller one."""
    b = Batch(q_lens, [n + 20 for n in q_lens], 8, 2, 128, fmt, 32, seed=18)
    table, lens, starts = _meta(b)
    q = b.q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    got = F.paged_attention(q, b.pages("cuda"), table, lens, starts, b.max_q)
    assert torch.equal(got, _attend(F, b))


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
@pytest.mark.parametrize("q_len", [1, 12, 60, 600])
def test_poisoned_rows_show(F, fmt, q_len):
    """A key or value with a NaN or an infinity, written into the cache: the rows that see it are NaN, and
    other sequences are as before."""
    b = Batch([q_len, q_len], [q_len + 200, q_len + 130], 4, 1, 64, fmt, 16, seed=19)
    clean = _attend(F, b)
    for bad_k, bad_v in ((float("nan"), None), (None, float("nan")), (None, float("inf"))):
        pages = b.pages("cuda")
        k, v = torch.ones(1, 1, 64, dtype=torch.bfloat16), torch.ones(1, 1, 64, dtype=torch.bfloat16)
        if bad_k is not None:
            k[0, 0, 3] = bad_k
        if bad_v is not None:
            v[0, 0, 3] = bad_v
        at = torch.tensor([61], dtype=torch.int32).cuda()  # token 60 of sequence 0
        F.kv_cache_write(pages, k.cuda(), v.cuda(), b.table[:1].cuda(), at)
        out = F.paged_attention(b.q.cuda(), pages, *_meta(b), b.max_q)
        assert torch.equal(out[q_len:], clean[q_len:])
        if fmt == "bf16" and bad_v is not None:  # unquantised, only its column is lost
            assert not torch.isfinite(out[:q_len, :, 3]).any()
        else:
            assert torch.isnan(out[:q_len]).all()


@pytest.mark.parametrize("fmt,n_pages", [("bf16", 17000), ("int8", 34000)])
@pytest.mark.parametrize("q_len", [1, 200])
def test_pools_past_32_bit_offsets(F, fmt, n_pages, q_len):
    """Pools of more than 4 GB: the same pages at their end give the same result, and take writes there."""
    b = Batch([q_len], [q_len + 300], 8, 8, 128, fmt, 128, seed=20)
    small = b.pages("cuda")
    table, lens, starts = _meta(b)
    want = F.paged_attention(b.q.cuda(), small, table, lens, starts, b.max_q)
    big = [None if t is None else torch.empty((n_pages,) + tuple(t.shape[1:]), dtype=t.dtype, device="cuda")
           for t in small]
    for s, t in zip(small, big):
        if s is not None:
            t[-b.n_pages:].copy_(s)
    assert big[0].numel() * big[0].element_size() > 1 << 32
    pages = F.KVPages(*big)
    moved = table + (n_pages - b.n_pages)
    assert torch.equal(F.paged_attention(b.q.cuda(), pages, moved, lens, starts, b.max_q), want)
    F.kv_cache_write(pages, b.k.cuda(), b.v.cuda(), moved, lens, starts)
    F.kv_cache_write(small, b.k.cuda(), b.v.cuda(), table, lens, starts)
    for x, y in zip(F.kv_cache_read(pages, moved, lens, starts, total=q_len),
                    F.kv_cache_read(small, table, lens, starts, total=q_len)):
        assert torch.equal(x, y)


def test_first_call_inside_a_capture():
    """The process's first kernel may be one that a graph capture records."""
    import os
    import subprocess
    import sys

    code = """
import torch
from cs244c_llama_zero_b200.ops import functional as F
pages = F.KVPages(*[torch.ones(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)])
q = torch.ones(1, 4, 64, dtype=torch.bfloat16, device="cuda")
table = torch.tensor([[2, 1]], dtype=torch.int32).cuda()
lens = torch.tensor([20], dtype=torch.int32).cuda()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = F.paged_attention(q, pages, table, lens)
graph.replay()
torch.cuda.synchronize()
assert (out == 1).all()
print("captured")
"""
    root = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


# ------------------------------------------------------------------------------------------ cache
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 1, 128), (3, 3, 64)])
@pytest.mark.parametrize("page", [16, 128])
def test_write_and_read_back(F, fmt, heads, page):
    b = Batch([3, 0, 1, 40, 130], [20, 7, 1, 40, 141], *heads, fmt, page, seed=12, behind=3)
    pages = b.pages("cuda")
    before = [t.clone() for t in pages if t is not None]
    table, lens, starts = _meta(b)
    kv = heads[1]
    fused = torch.randn(b.q.shape[0], 3 * kv + 1, heads[2]).to(torch.bfloat16)
    fused[:, kv:2 * kv], fused[:, 2 * kv:3 * kv] = b.k, b.v
    fused = fused.cuda()
    F.kv_cache_write(pages, fused[:, kv:2 * kv], fused[:, 2 * kv:3 * kv], table, lens, starts)
    k, v = F.kv_cache_read(pages, table, lens, starts, total=b.total, dtype=torch.float32)
    for got, x in ((k, b.k[:b.total]), (v, b.v[:b.total])):
        if fmt == "bf16":
            assert torch.equal(got.cpu(), x.float())
        else:  # the codes exactly, the values to the rounding of scale and product (2^-24 each)
            codes, scale = quantise(x, fmt)
            want = codes * scale[..., None]
            assert ((got.double().cpu() - want).abs() <= 2.0 ** -22 * want.abs()).all()
    half = F.kv_cache_read(pages, table, lens, starts, total=b.total)
    assert torch.equal(half[0], k.to(torch.bfloat16)) and torch.equal(half[1], v.to(torch.bfloat16))
    # nothing else in the pools moved
    written = torch.zeros(b.n_pages, page, dtype=torch.bool)
    for s in range(len(b.q_lens)):
        for t in range(b.kv_lens[s] - b.q_lens[s], b.kv_lens[s]):
            written[b.table[s, t // page], t % page] = True
    for old, new in zip(before, [t for t in pages if t is not None]):
        keep = (~written)[:, None].expand(old.shape[:3])
        bytes_of = lambda t: t.cpu()[keep].contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(bytes_of(old), bytes_of(new))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_codes_at_ties_and_edges(F, fmt):
    """Every pair (x, max) of 8-bit significands, which holds all exact ties, and rows of tiny, huge,
    zero and non-finite values."""
    sig = torch.arange(128, 256, dtype=torch.float64)
    x = torch.zeros(128, 9, 1, 64, dtype=torch.float64)
    for i, s in enumerate((0, -1, -2, -3, -4, -5, -6, -7, -8)):
        x[:, i, 0, 0] = sig
        x[:, i, 0, 1:] = (sig[:63] if i % 2 else sig[65:]) * 2.0 ** s * (-1.0 if i % 3 == 0 else 1.0)
    x[:, :, 0, 1:] = torch.minimum(x[:, :, 0, 1:].abs(), x[:, :, 0, :1]) * x[:, :, 0, 1:].sign()
    x = x.view(-1, 1, 64)
    x = torch.cat([x, x[:40] * 2.0 ** -140, x[:40] * 2.0 ** 119, torch.zeros(3, 1, 64, dtype=torch.float64)])
    rows = x.to(torch.bfloat16)
    n = rows.shape[0]
    rows[-1, 0, 5] = float("inf")
    rows[-2, 0, 6] = float("nan")
    b = Batch([n], [n], 1, 1, 64, fmt, 16, seed=13)
    pages = b.pages("cuda")
    table, lens, starts = _meta(b)
    F.kv_cache_write(pages, rows.cuda(), rows.cuda(), table, lens, starts)
    k, _ = F.kv_cache_read(pages, table, lens, starts, total=n, dtype=torch.float32)
    assert torch.isnan(k[-2:]).all() and (k[-3] == 0).all()
    places = table[0].cpu().long()[torch.arange(n) // 16], torch.arange(n) % 16
    got = pages.k.view(torch.uint8).cpu()[places[0], 0, places[1]].view(FORMATS[fmt]).double()
    codes, scale = quantise(rows[:-2, 0], fmt)
    assert torch.equal(got[:-2], codes)
    stored = pages.k_scale.cpu()[places[0], 0, places[1]][:-2].double()
    assert ((stored - scale).abs() <= 2.0 ** -24 * scale + 2.0 ** -149).all()


def test_write_graph_and_bad_pages(F, errors):
    b = Batch([2, 3], [20, 33], 4, 2, 64, "e4m3", 16, seed=14)
    pages = b.pages("cuda")
    table, lens, starts = _meta(b)
    k, v = b.k.cuda(), b.v.cuda()
    F.kv_cache_write(pages, k, v, table, lens, starts)
    want = F.kv_cache_read(pages, table, lens, starts, total=5)
    k2 = torch.zeros_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.kv_cache_write(pages, k2, v, table, lens, starts)
        got = F.kv_cache_read(pages, table, lens, starts, total=5)
    graph.replay()
    assert (got[0] == 0).all() and torch.equal(got[1], want[1])
    k2.copy_(k)
    graph.replay()
    assert torch.equal(got[0], want[0])
    assert errors()[0] == 0
    table[1] = -5
    keep = [t.clone() for t in pages]
    F.kv_cache_write(pages, k, v, table, lens, starts)
    assert errors()[0] == 6
    for old, new in zip(keep, pages):
        assert torch.equal(old.view(torch.uint8), new.view(torch.uint8))
    lens[0] = 10_000
    out = F.kv_cache_read(pages, table, lens, starts, total=5)
    assert (out[0][2:] == 0).all()


# ------------------------------------------------------------------------------------------ logits
def _logit_case(batch, vocab, dtype, length, seed):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(batch, vocab, generator=gen) * 4).to(dtype)
    history = (torch.rand(batch, max(length, 1), generator=gen) ** 3 * vocab).long().clamp(max=vocab - 1)
    lens = torch.randint(0, length + 1, (batch,), generator=gen, dtype=torch.int32)
    lens[0] = length
    prompts = (lens * torch.rand(batch, generator=gen)).int()
    rep = 0.7 + torch.rand(batch, generator=gen)
    freq, pres = torch.randn(batch, generator=gen), torch.randn(batch, generator=gen)
    bias = torch.randn(vocab, generator=gen)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (batch, (vocab + 31) // 32), generator=gen).int()
    return logits, history, lens, prompts, rep, freq, pres, bias, allowed


def _logit_tol(want, logits, dtype, length):
    """One rounding to the type (half a step), fp32 before it: five operations on values up to the largest
    intermediate (here below |l| * 2 + |result| + 10 + 5 * length), half a step of 2^-24 each."""
    big = logits.double().abs() * 2 + want.abs().nan_to_num(posinf=0.0) + 10 + 5 * length
    return torch.finfo(dtype).eps / 2 * want.abs().nan_to_num(posinf=0.0) + 5 * 2.0 ** -24 * big * (1 + torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,vocab,length", [(1, 1, 3), (2, 31, 0), (3, 1000, 50), (2, 8191, 700), (2, 32000, 300),
                                                (1, 9999, 1), (2, 5000, 3000), (2, 600, 5000)])
def test_logits(F, dtype, batch, vocab, length):
    logits, history, lens, prompts, rep, freq, pres, bias, allowed = _logit_case(batch, vocab, dtype, length, vocab)
    cu = [t.cuda() for t in (logits, history, lens, prompts, rep, freq, pres, bias, allowed)]
    want = adjusted(logits, history, lens, prompts, rep, freq, pres, bias, allowed)
    got = F.adjust_logits(*cu)
    assert torch.equal(torch.isinf(got.cpu()), torch.isinf(want))
    fin = torch.isfinite(want)
    err = (got.double().cpu() - want).abs()
    tol = _logit_tol(want, logits, dtype, length)
    assert (err[fin] <= tol[fin]).all()
    assert F.adjust_logits(*cu, out=cu[0]).data_ptr() == cu[0].data_ptr()
    assert torch.equal(cu[0], got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_parts_and_strides(F, dtype):
    """Each part alone, rows at any alignment, one mask or bias for all rows or one for each."""
    logits, history, lens, prompts, rep, freq, pres, bias, allowed = _logit_case(3, 5003, dtype, 90, 5)
    bias2 = torch.randn(3, 5003)
    for off_in, off_out in ((0, 0), (1, 1), (3, 3), (1, 2), (0, 5)):
        wide = torch.zeros(3, 5100, dtype=dtype, device="cuda")
        src = wide[:, off_in:off_in + 5003]
        src.copy_(logits)
        target = torch.full((3, 5017), 5.0, dtype=dtype, device="cuda")
        for parts in (dict(repetition_penalty=rep), dict(frequency_penalty=freq, prompt_lens=prompts),
                      dict(presence_penalty=pres), dict(bias=bias2), dict(bias=bias), dict(allowed=allowed[0].contiguous()),
                      dict(allowed=allowed), dict()):
            hist = {} if set(parts) <= {"bias", "allowed"} else dict(history=history, history_lens=lens)
            kw = {k: v.cuda() for k, v in {**parts, **hist}.items()}
            out = F.adjust_logits(src, out=target[:, off_out:off_out + 5003], **kw)
            want = adjusted(logits, hist.get("history"), lens, parts.get("prompt_lens"), parts.get("repetition_penalty"),
                            parts.get("frequency_penalty"), parts.get("presence_penalty"), parts.get("bias"),
                            parts.get("allowed"))
            fin = torch.isfinite(want)
            assert torch.equal(torch.isinf(out.cpu()), ~fin)
            tol = _logit_tol(want, logits, dtype, 90)
            assert ((out.double().cpu() - want).abs()[fin] <= tol[fin]).all()
        assert (target[:, :off_out] == 5).all() and (target[:, off_out + 5003:] == 5).all()


def test_logits_special_values(F):
    """Masked rows, infinities and NaN: a masked NaN becomes -inf, an unmasked one stays."""
    x = torch.tensor([[float("nan"), float("-inf"), float("inf"), torch.finfo(torch.float32).min, 1.0]] * 2).cuda()
    allowed = torch.tensor([[0], [31]], dtype=torch.int32).cuda()
    hist = torch.tensor([[1, 2, 3, 0, 4]] * 2).cuda()
    lens = torch.full((2,), 5, dtype=torch.int32).cuda()
    out = F.adjust_logits(x, hist, lens, repetition_penalty=torch.full((2,), 2.0).cuda(), allowed=allowed)
    assert torch.isinf(out[0]).all() and (out[0] < 0).all()
    assert torch.isnan(out[1, 0]) and out[1, 1] == float("-inf") and out[1, 2] == float("inf")
    assert out[1, 3] == float("-inf") and out[1, 4] == 0.5


def test_logits_bad_ids_are_skipped_and_recorded(F, errors):
    x = torch.ones(2, 100).cuda()
    hist = torch.tensor([[5, 100, -1, 5], [7, 7, 7, 2 ** 40]]).cuda()
    lens = torch.tensor([3, 9], dtype=torch.int32).cuda()
    out = F.adjust_logits(x, hist, lens, frequency_penalty=torch.full((2,), 0.25).cuda())
    assert errors()[0] == 6
    want = torch.ones(2, 100)
    want[0, 5] = 0.75
    assert torch.equal(out.cpu(), want)


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt", list(FORMATS))
def test_a_conversation(F, fmt):
    """A prompt in two chunks, then single tokens, all written and attended over in one cache: each row
    equals plain attention over what the cache gives back."""
    H, KV, hd, page = 12, 4, 64, 16
    gen = torch.Generator().manual_seed(30)
    lengths = [(37, 21), (30, 45)] + [(1, 1)] * 4
    pool = Batch([0, 0], [80, 80], H, KV, hd, fmt, page, seed=31)
    pages, table = pool.pages("cuda"), pool.table.cuda()
    have = [0, 0]
    for step, new in enumerate(lengths):
        have = [h + n for h, n in zip(have, new)]
        starts = torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32).cuda()
        lens = torch.tensor(have, dtype=torch.int32).cuda()
        rows = new[0] + new[1]
        qkv = torch.randn(rows, H + 2 * KV, hd, generator=gen).to(torch.bfloat16).cuda()
        F.kv_cache_write(pages, qkv[:, H:H + KV], qkv[:, H + KV:], table, lens, starts)
        out = F.paged_attention(qkv[:, :H], pages, table, lens, starts, max(new))
        everything = torch.tensor([0, have[0], sum(have)], dtype=torch.int32).cuda()
        k, v = F.kv_cache_read(pages, table, lens, everything, total=sum(have), dtype=torch.float32)
        for s in range(2):
            lo, hi = int(everything[s]), int(everything[s + 1])
            q = qkv[int(starts[s]):int(starts[s + 1]), :H].double().cpu()
            ks = k[lo:hi].double().cpu().repeat_interleave(H // KV, 1)
            vs = v[lo:hi].double().cpu().repeat_interleave(H // KV, 1)
            sc = torch.einsum("ihd,jhd->hij", q, ks) * hd ** -0.5
            size = torch.einsum("ihd,jhd->hij", q.abs(), ks.abs()) * hd ** -0.5
            hidden = torch.arange(have[s])[None] > (torch.arange(new[s]) + have[s] - new[s])[:, None]
            p = torch.softmax(sc.masked_fill(hidden, float("-inf")), -1)
            want, mag = torch.einsum("hij,jhd->ihd", p, vs), torch.einsum("hij,jhd->ihd", p, vs.abs())
            size = size.masked_fill(hidden, 0.0).amax(-1).t()[..., None]
            _check(out[int(starts[s]):int(starts[s + 1])], want, tolerance(want, mag, size, fmt != "bf16"))
