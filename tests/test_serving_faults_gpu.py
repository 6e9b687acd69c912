"""Corners of the serving operators on the GPU, against their 64-bit definitions: rows and units of zeros, values of
extreme size, infinities and NaN in places that a row does not see, scratch memory that is not to be had."""

from __future__ import annotations

import pytest
import torch

from tests.serving_bounds import bound, norm_bound
from tests.serving_reference import FORMATS, Batch

pytestmark = pytest.mark.gpu

QUANTISED = ["e4m3", "int8"]
# (heads, kv heads, head size), new tokens: few rows, few rows split over the warps, a chunk whose codes are expanded
# in its tiles, one long enough that they are expanded once
FORMS = [((8, 2, 64), 3), ((8, 2, 64), 14), ((8, 2, 64), 60), ((8, 2, 64), 150),
         ((16, 8, 128), 4), ((16, 8, 128), 60), ((16, 8, 128), 150)]


@pytest.fixture(scope="module")
def F():
    from cs244c_llama_zero_b200 import ops
    from cs244c_llama_zero_b200.ops import functional

    ops.load_extension().reset_device_errors()
    yield functional
    ops.check_device_errors()


def _attend(F, b, **kw):
    return F.paged_attention(b.q.cuda(), b.pages("cuda"), b.table.cuda(), b.lens.cuda(), b.starts.cuda(), b.max_q, **kw)


def _attend_many(F, b, copies=24, pages=None, **kw):
    """The batch ``copies`` times over the same pages, so that a block's range holds several units of an item."""
    starts = torch.cat([b.starts[:1]] + [b.starts[1:] + i * b.total for i in range(copies)])
    pages = b.pages("cuda") if pages is None else pages
    out = F.paged_attention(b.q.repeat(copies, 1, 1).cuda(), pages, b.table.repeat(copies, 1).cuda(),
                            b.lens.repeat(copies).cuda(), starts.cuda(), b.max_q, **kw)
    return out.view(copies, *b.q.shape)


def _check(got, b, want=None, rows=slice(None), **kw):
    want, mag, size = b.attention(**kw) if want is None else want
    got = got[:b.total].double().cpu()
    far = ~((got - want).abs() <= bound(want, mag, size, b.fmt))
    far = far[rows]
    assert not far.any(), (f"{int(far.sum())} of {far.numel()} outside, first at {far.nonzero()[0].tolist()}: "
                           f"{got[rows][far][0]} for {want[rows][far][0]}")


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads,q_len", FORMS)
@pytest.mark.parametrize("k_size,scale", [(2.0 ** -14, None), (1.0, 1e-4), (2.0 ** -60, 1e-20)])
def test_zero_query_rows(F, fmt, heads, q_len, k_size, scale):
    """A row of zeros has equal scores: the mean of the visible V, however small K and the scale are."""
    b = Batch([q_len, 2], [q_len + 70, 40], *heads, fmt, 16, seed=40)
    b.q[::3] = 0
    b.q[1, :1] = 0
    if fmt == "bf16":
        b.pools[0] = (b.pools[0].float() * k_size).to(torch.bfloat16)
    else:
        b.scales[0] *= k_size
    want = b.attention(scale=scale)
    _check(_attend(F, b, scale=scale), b, want)
    for got in _attend_many(F, b, scale=scale):
        _check(got, b, want)


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads,q_len", FORMS)
@pytest.mark.parametrize("v_size", [1.0, 2.0 ** -8, 2.0 ** -18, 2.0 ** -60])
def test_units_whose_values_are_zero(F, fmt, heads, q_len, v_size):
    """The first 192 tokens have V = 0 (and, in sequence 1, all): they count in the sum of the weights only, whatever
    size the V behind them has, and also where their scores are the larger ones."""
    b = Batch([q_len, q_len], [q_len + 330, 300], *heads, fmt, 32, seed=41)
    for s, n in ((0, 192), (1, 300)):
        for t in range(n):
            at = b.table[s, t // 32], t % 32
            b.pools[1][at[0], :, at[1]] = 0
            if fmt != "bf16":
                b.scales[1][at[0], :, at[1]] = 0
    if fmt == "bf16":
        b.pools[1] = (b.pools[1].float() * v_size).to(torch.bfloat16)
    else:
        b.scales[1] *= v_size
    want = b.attention()
    _check(_attend(F, b), b, want)
    for got in _attend_many(F, b):
        _check(got, b, want)


@pytest.mark.parametrize("fmt", QUANTISED)
@pytest.mark.parametrize("heads,q_len", FORMS)
def test_scales_of_minus_zero(F, fmt, heads, q_len):
    """A row of zeros may have been stored with the scale -0."""
    b = Batch([q_len], [q_len + 200], *heads, fmt, 16, seed=51)
    for which in range(2):
        at = b.table[0, 2 + which], slice(None), 3
        b.pools[which][at], b.scales[which][at] = 0, -0.0
    _check(_attend(F, b), b)


@pytest.mark.parametrize("fmt", QUANTISED)
def test_many_values_of_zero(F, fmt):
    """Tens of thousands of zero V in one block's range, ahead of others, with scores that rise by less than makes
    the running maximum follow: the sum of their weights stays in range.  (The sequences share their pages.)"""
    page, n, batch = 128, 32768, 512
    pages = n // page
    code = torch.full((pages, 1, page, 64), 127, dtype=torch.int8)
    k = code.clone() if fmt == "int8" else code.float().to(torch.float8_e4m3fn)
    unit = float(k.float().max())
    k_scale = torch.full((pages, 1, page), 1.0 / unit)  # k = 1
    k_scale[0, 0, :64] = 1e-6  # the first scores are next to 0, the others 7.9 / log2(e)
    v = k.clone()
    v_scale = torch.zeros(pages, 1, page)
    v_scale[-1, 0, -32:] = 1.0 / unit  # the last 32 values are 1
    cache = F.KVPages(*[t.cuda() for t in (k, v, k_scale, v_scale)])
    q = torch.full((batch, 1, 64), 1.0, dtype=torch.bfloat16).cuda()
    table = torch.arange(pages, dtype=torch.int32).expand(batch, pages).contiguous().cuda()
    lens = torch.full((batch,), n, dtype=torch.int32).cuda()
    score = 7.9 * 0.6931471805599453
    out = F.paged_attention(q, cache, table, lens, scale=score / 64).double().cpu()
    low = torch.exp(torch.tensor(-score * (1 - 1e-6 * unit), dtype=torch.float64))
    want = 32 / (n - 64 + 64 * low)
    # the result's rounding, the weights' (fp16), and scores of 8 in fp32
    assert ((out - want).abs() <= want * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -16)).all(), (out.min(), out.max(), want)


@pytest.mark.parametrize("fmt", QUANTISED)
@pytest.mark.parametrize("heads,q_len", FORMS)
@pytest.mark.parametrize("exponent", [110, 121])
def test_values_of_huge_size(F, fmt, heads, q_len, exponent):
    """V up to 2^(exponent + 4): no factor on the way leaves its type's range."""
    b = Batch([q_len], [q_len + 200], *heads, fmt, 16, seed=42)
    b.scales[1] *= 2.0 ** exponent
    _check(_attend(F, b), b)


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads,q_len", FORMS + [((4, 4, 64), 130), ((4, 4, 128), 300), ((64, 1, 64), 5)])
@pytest.mark.parametrize("bad", ["k nan", "v nan", "v inf", "v -inf"])
def test_poisoned_tokens_in_masked_places(F, fmt, heads, q_len, bad):
    """A NaN or an infinity in a new token's key or value: the rows ahead of it do not see it and are what they are
    without it; the rows from it on are not finite (8-bit pages and keys: NaN throughout; V in bf16: in its column)."""
    b = Batch([q_len, q_len], [q_len + 75, q_len + 9], *heads, fmt, 16, seed=43)
    want = b.attention()
    kv, hd = heads[1], heads[2]
    new = q_len // 2  # the poisoned row of sequence 0
    pos = b.kv_lens[0] - q_len + new
    pages = b.pages("cuda")
    k, v = torch.ones(1, kv, hd), torch.ones(1, kv, hd)
    (k if bad[0] == "k" else v)[0, :, 5] = float(bad[2:])
    at = torch.tensor([pos + 1], dtype=torch.int32).cuda()
    F.kv_cache_write(pages, k.bfloat16().cuda(), v.bfloat16().cuda(), b.table[:1].cuda(), at)
    out = F.paged_attention(b.q.cuda(), pages, b.table.cuda(), b.lens.cuda(), b.starts.cuda(), b.max_q)
    outs = [out, *_attend_many(F, b, pages=pages)]
    for out in outs:
        _check(out, b, want, rows=slice(0, new))
        _check(out, b, want, rows=slice(q_len, 2 * q_len))
    if fmt != "bf16" or bad[0] == "k":
        assert all(torch.isnan(out[new:q_len]).all() for out in outs)
        return
    where = b.table[0, pos // 16], slice(None), pos % 16
    b.pools[0][where], b.pools[1][where] = 1.0, 1.0  # what was written, with something finite in the column
    others = torch.arange(hd) != 5
    cut = [t[new:q_len][..., others if t.shape[-1] == hd else slice(None)] for t in b.attention()]
    for out in outs:
        seen = out[new:q_len].double().cpu()
        assert not torch.isfinite(seen[..., 5]).any()
        assert ((seen[..., others] - cut[0]).abs() <= bound(*cut, fmt)).all()


@pytest.mark.parametrize("fmt", QUANTISED)
def test_scratch_memory_that_is_not_to_be_had(F, fmt):
    """Codes are expanded once into scratch memory sized by the block table's width; where the allocator has none left,
    the same call expands them in its tiles and gives the result all the same."""
    b = Batch([300], [420], 8, 2, 128, fmt, 128, seed=44)
    wide = torch.zeros(1, 3000, dtype=torch.int32)  # room for 384000 tokens: 393 MB of fp16 units
    wide[:, :b.table.shape[1]] = b.table
    args = (b.q.cuda(), b.pages("cuda"), wide.cuda(), b.lens.cuda(), b.starts.cuda(), b.max_q)
    roomy = F.paged_attention(*args)
    _check(roomy, b)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (100 << 20)) / total)
        out = F.paged_attention(*args)
        torch.cuda.synchronize()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    _check(out, b)


# ------------------------------------------------------------------------------------------ precision
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("heads,q_len", FORMS + [((12, 4, 64), 1), ((32, 8, 128), 1), ((12, 4, 64), 400), ((32, 8, 64), 90)])
def test_rounding_of_ordinary_activations(F, fmt, heads, q_len):
    """Element by element inside the bound of the form's own roundings, and as a whole near what they add up to."""
    b = Batch([q_len, 1, q_len], [q_len + 700, 333, q_len], *heads, fmt, 64, seed=45)
    want, mag, size = b.attention()
    got = _attend(F, b)
    _check(got, b, (want, mag, size))
    error = (got.double().cpu() - want).norm() / want.norm()
    assert error <= norm_bound(fmt), float(error)


@pytest.mark.parametrize("fmt", QUANTISED)
@pytest.mark.parametrize("heads,q_len", FORMS)
def test_scales_of_different_size_in_a_unit(F, fmt, heads, q_len):
    """Every seventh token's K 2^12 times smaller and V 2^12 times larger than the others'."""
    b = Batch([q_len, 3], [q_len + 400, 90], *heads, fmt, 16, seed=46)
    b.scales[0][:, :, ::7] *= 2.0 ** -12
    b.scales[1][:, :, ::7] *= 2.0 ** 12
    _check(_attend(F, b), b)


# ------------------------------------------------------------------------------------------ generation
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fmt", list(FORMATS))
def test_the_next_token_with_and_without_a_cache(hd, fmt):
    """The same backend with a cache and without one picks the same token wherever the 64-bit model's two best
    logits are further apart than what both paths' logits are off by."""
    from cs244c_llama_zero_b200.models import LlamaForCausalLM, ModelConfig, PagedKVCache

    cfg = ModelConfig(name="gen", vocab_size=1000, max_seq_len=140, dim=4 * hd, n_layers=3, n_heads=4, n_kv_heads=2,
                      ffn_dim=512, initializer_range=0.08)
    torch.manual_seed(3)
    model = LlamaForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    oracle = LlamaForCausalLM(cfg).cuda().double().eval()
    oracle.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    model.set_backend("b200")
    ids = torch.randint(0, cfg.vocab_size, (24, 128), device="cuda")
    with torch.no_grad():
        want = oracle(ids).logits[:, -1]
        plain = model(ids).logits[:, -1].double()
        cache = PagedKVCache.for_batch(cfg, 24, 128, dtype=fmt)
        cached = model.decode_step(ids.reshape(-1), cache, range(24), [128] * 24).double()
        off = torch.maximum((plain - want).abs().amax(-1), (cached - want).abs().amax(-1))
        best = want.topk(2, dim=-1).values
        clear = best[:, 0] - best[:, 1] > 2 * off  # either of the two logits may be off by that much
        assert clear.any()
        with_cache = model.generate(ids, 1, temperature=0.0, kv_cache=fmt)
        without = model.generate(ids, 1, temperature=0.0)
    assert torch.equal(with_cache[:, :128], ids) and torch.equal(without[:, :128], ids)
    assert torch.equal(with_cache[clear, 128], without[clear, 128])
    assert torch.equal(without[clear, 128], want.argmax(-1)[clear])


# ------------------------------------------------------------------------------------------ calls that the limits allow
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("group", [65, 100, 127, 128])
@pytest.mark.parametrize("hd", [64, 128])
def test_the_largest_groups(F, fmt, group, hd):
    """A tile holds one token's heads, and up to 63 rows of nothing."""
    for q, kv in (([1, 1], [200, 33]), ([3, 0, 1], [150, 20, 128])):
        b = Batch(q, kv, group, 1, hd, fmt, 16, seed=47)
        _check(_attend(F, b), b)


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("q_lens", [[1, 2], [5, 33]])
def test_thousands_of_sequences(F, fmt, q_lens):
    """Far more sequences than threads that divide the work among them."""
    b = Batch(q_lens, [40, 33], 8, 2, 64, fmt, 16, seed=48)
    want = b.attention()
    outs = _attend_many(F, b, copies=3000).double().cpu()
    assert ((outs - want[0]).abs() <= bound(*want, fmt)).all()


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("max_q_len", [1, 4, 8, 30, 1000, 2 ** 31 - 1])
def test_a_loose_bound_on_new_tokens(F, fmt, max_q_len):
    """max_q_len chooses the form; any bound that holds gives the same result."""
    b = Batch([1, 1, 1], [77, 300, 1], 8, 2, 128, fmt, 16, seed=49)
    out = F.paged_attention(b.q.cuda(), b.pages("cuda"), b.table.cuda(), b.lens.cuda(), b.starts.cuda(), max_q_len)
    _check(out, b)


def test_logits_captured_and_on_two_streams(F):
    """A captured call reads what its tensors hold at replay, in place too; two streams do not meet."""
    gen = torch.Generator().manual_seed(50)
    logits = torch.randn(3, 9001, generator=gen).cuda()
    history = torch.randint(0, 9001, (3, 3000), generator=gen).cuda()
    lens = torch.tensor([3000, 10, 0], dtype=torch.int32).cuda()
    rep = torch.full((3,), 1.3).cuda()
    want = F.adjust_logits(logits, history, lens, repetition_penalty=rep)
    short = torch.tensor([5, 2900, 1], dtype=torch.int32).cuda()
    want_short = F.adjust_logits(logits, history, short, repetition_penalty=rep)
    torch.cuda.synchronize()
    live, place = lens.clone(), logits.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.adjust_logits(logits, history, live, repetition_penalty=rep)
        F.adjust_logits(place, history, live, repetition_penalty=rep, out=place)
    graph.replay()
    assert torch.equal(out, want) and torch.equal(place, want)
    live.copy_(short)
    place.copy_(logits)
    graph.replay()
    assert torch.equal(out, want_short) and torch.equal(place, want_short)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for s, n in zip(streams, (lens, short)):
            with torch.cuda.stream(s):
                results.append(F.adjust_logits(logits, history, n, repetition_penalty=rep))
    torch.cuda.synchronize()
    for i, r in enumerate(results):
        assert torch.equal(r, want if i % 2 == 0 else want_short)
