"""Workloads of the serving operators: paged key/value cache, attention over it, logit adjustment.

Each case is one call (or one write / read-back pair) as a decoding loop makes it.  ``run`` computes it
with the framework's kernels when ``own`` is true, else with elementary torch operations in 32 bits.
Head layouts are those of the model presets (heads / kv heads / head size): 12/4/64, 18/6/64, 32/8/64,
16/8/128 and 32/8/128; vocabularies 32000 and 128256.

A cache layer is a pool of pages ``[n_pages, kv_heads, page_size, head_dim]`` in bf16, e4m3 or int8, the
latter two with one fp32 scale per token and head: ``scale = max|x| / M``, ``code = round(x * M / max|x|)``
with ``M`` = 448 (e4m3) or 127 (int8).  A sequence's pages are listed in its row of the block table.  The
last ``q_len`` of its ``kv_len`` cached tokens are the new ones; a new token sees itself and what is before.
"""

import math
import random

import torch

own = False

FORMATS = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}
HEADS = ((12, 4, 64), (18, 6, 64), (32, 8, 64), (16, 8, 128), (32, 8, 128))
LOGIT_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def _attention(name, batch, heads, q_len, ragged_q, kv_len, ragged_kv, fmt, page, shape_seed):
    h, kv, hd = heads
    return {"name": name, "op": "attention", "batch": batch, "heads": h, "kv_heads": kv, "head_dim": hd,
            "q_len": q_len, "ragged_q": ragged_q, "kv_len": kv_len, "ragged_kv": ragged_kv, "format": fmt,
            "page": page, "shape_seed": shape_seed}


def _cache(name, op, batch, heads, q_len, ragged_q, kv_len, fmt, page, shape_seed):
    case = _attention(name, batch, heads, q_len, ragged_q, kv_len, True, fmt, page, shape_seed)
    case["op"] = op
    return case


def _logits(name, batch, vocab, dtype, history, extras, shape_seed):
    return {"name": name, "op": "logits", "batch": batch, "vocab": vocab, "dtype": dtype, "history": history,
            "extras": extras, "shape_seed": shape_seed}


def listed():
    return [
        # one user, one token: latency
        _attention("decode_single_user", 1, (32, 8, 128), 1, False, 2048, False, "bf16", 64, 1),
        # a batch of small-model conversations of very different ages, unquantised
        _attention("decode_small_model_batch", 256, (12, 4, 64), 1, False, 2048, True, "bf16", 32, 2),
        # a serving batch over an e4m3 cache in small pages
        _attention("decode_ragged_e4m3", 61, (16, 8, 128), 1, False, 4096, True, "e4m3", 16, 3),
        # a few long documents in int8: the cache is read at memory speed
        _attention("decode_long_int8", 4, (32, 8, 128), 1, False, 131072, True, "int8", 128, 4),
        # a handful of proposed tokens per sequence checked in one pass
        _attention("verify_few_tokens", 8, (32, 8, 64), 16, True, 8192, True, "int8", 64, 5),
        # prompts of a mixed batch, most of them fresh, written as e4m3
        _attention("prompts_ragged_e4m3", 9, (12, 4, 64), 1500, True, 2200, True, "e4m3", 64, 6),
        # one chunk of a long prompt: bound by the tensor cores
        _attention("prompt_chunk_long", 1, (32, 8, 128), 2048, False, 16384, False, "bf16", 64, 7),
        # what one decode step appends
        _cache("append_step", "append", 64, (32, 8, 128), 1, False, 2048, "e4m3", 64, 8),
        # what a batch of prompts appends
        _cache("append_prompts", "append", 12, (16, 8, 128), 2731, True, 4096, "int8", 32, 9),
        # whole sequences read back, as for handing them to another engine
        _cache("read_sequences", "read", 24, (32, 8, 128), 4096, True, 4096, "e4m3", 64, 10),
        # one user, a short history, penalties only
        _logits("logits_single_user", 1, 32000, "bf16", 150, False, 11),
        # a serving batch with biases and grammar masks on a large vocabulary
        _logits("logits_batch_masked", 256, 128256, "fp32", 2048, True, 12),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread evenly over its logarithm."""
    return max(low, min(high, int(round(2.0 ** rng.uniform(math.log2(low), math.log2(high + 1)) - 0.5))))


_MAX_CODES = 4 * 131072 * 8  # cached (token, head) rows of the largest decode case
_MAX_PAIRS = 2048 * 15360 * 32  # (query, visible token, head) triples of the largest chunk case


def draw(rng):
    kind = rng.choice(("decode", "decode", "chunk", "chunk", "append", "read", "logits"))
    heads = rng.choice(HEADS)
    fmt = rng.choice(("bf16", "e4m3", "int8"))
    page = rng.choice((16, 32, 64, 128))
    seed = rng.randrange(1 << 30)
    if kind == "decode":
        batch = _spread(rng, 1, 256)
        kv_len = _spread(rng, 1, min(131072, _MAX_CODES // (batch * heads[1])))
        case = _attention("", batch, heads, 1, False, kv_len, rng.random() < 0.7, fmt, page, seed)
    elif kind == "chunk":
        batch = _spread(rng, 1, 16)
        q_len = _spread(rng, 2, 4096 // batch + 2)
        room = max(q_len, min(32768, _MAX_PAIRS // (batch * q_len * heads[0])))
        kv_len = _spread(rng, q_len, room)
        case = _attention("", batch, heads, q_len, rng.random() < 0.7, kv_len, rng.random() < 0.7, fmt, page, seed)
    elif kind == "append":
        batch = _spread(rng, 1, 128)
        q_len = 1 if rng.random() < 0.4 else _spread(rng, 1, 32768 // batch)
        case = _cache("", "append", batch, heads, q_len, q_len > 1 and rng.random() < 0.7,
                      q_len + _spread(rng, 1, 2048), fmt, page, seed)
    elif kind == "read":
        batch = _spread(rng, 1, 64)
        q_len = _spread(rng, 1, 65536 // batch)
        case = _cache("", "read", batch, heads, q_len, rng.random() < 0.7, q_len, fmt, page, seed)
    else:
        vocab = rng.choice((32000, 128256, rng.randrange(500, 130000)))
        case = _logits("", _spread(rng, 1, 200), vocab, rng.choice(sorted(LOGIT_TYPES)), _spread(rng, 1, 4096),
                       rng.random() < 0.6, seed)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------ shapes
def _lengths(case):
    """Per sequence: new tokens and cached tokens (the new ones among them).  From the case alone."""
    rng = random.Random(case["shape_seed"])
    q_lens, kv_lens = [], []
    for b in range(case["batch"]):
        q = _spread(rng, 1, case["q_len"]) if case["ragged_q"] and b > 0 else case["q_len"]
        kv = case["kv_len"]
        if case["ragged_kv"] and b > 0:
            kv = rng.randint(1, case["kv_len"])
        q_lens.append(q)
        kv_lens.append(max(kv, q))
    return q_lens, kv_lens


def _history_lengths(case):
    rng = random.Random(case["shape_seed"])
    lens = [case["history"] if b == 0 else rng.randint(0, case["history"]) for b in range(case["batch"])]
    return lens, [rng.randint(0, n) for n in lens]


def _pairs(q_lens, kv_lens):
    """(new token, visible token) pairs over the batch."""
    return sum(q * (kv - q) + q * (q + 1) // 2 for q, kv in zip(q_lens, kv_lens))


def work(case):
    if case["op"] == "logits":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["batch"] * case["vocab"]
        total = 2 * n * size + 8 * sum(_history_lengths(case)[0])
        if case["extras"]:
            total += n // 8 + 4 * case["vocab"]
        return {"bytes": total, "flops": 2 * n}
    q_lens, kv_lens = _lengths(case)
    hd, kvh = case["head_dim"], case["kv_heads"]
    row = 2 * hd if case["format"] == "bf16" else hd + 4  # one head of one token's K (or V) in the cache
    new = sum(q_lens)
    meta = 4 * sum((n + case["page"] - 1) // case["page"] for n in kv_lens) + 8 * case["batch"]
    if case["op"] == "append":  # read k and v, write them to the cache, read them back as fp32
        return {"bytes": 2 * new * kvh * (2 * hd + 2 * row + 4 * hd) + meta, "flops": 6 * new * kvh * hd}
    if case["op"] == "read":
        return {"bytes": 2 * new * kvh * (row + 2 * hd) + meta, "flops": 2 * new * kvh * hd}
    return {"bytes": 2 * sum(kv_lens) * kvh * row + 4 * new * case["heads"] * hd + meta,
            "flops": 4 * _pairs(q_lens, kv_lens) * case["heads"] * hd}


# ------------------------------------------------------------------------------------------ inputs
def _rows(gen, *shape):
    """Activations as projections produce them: channels of different strength, heads of different size."""
    strength = torch.empty(shape[-2:], device="cuda").log_normal_(0.0, 0.5, generator=gen)
    return (torch.randn(shape, device="cuda", generator=gen) * strength).to(torch.bfloat16)


def _quantise(x, fmt):
    """Codes and scales of rows ``[..., hd]`` in the cache's format."""
    if fmt == "bf16":
        return x, None
    x = x.float()
    top = x.abs().amax(dim=-1, keepdim=True)
    limit = torch.full_like(top, CODE_MAX[fmt])
    q = torch.where(top > 0, x * limit / top, torch.zeros_like(x))
    q = q.round().to(torch.int8) if fmt == "int8" else q.to(torch.float8_e4m3fn)
    return q, (top / limit).squeeze(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, gen)
    q_lens, kv_lens = _lengths(case)
    batch, kvh, hd, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    counts = [(n + page - 1) // page for n in kv_lens]
    n_pages = sum(counts) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(batch, max(counts), dtype=torch.int32)
    used = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[used:used + n]
        used += n
    pools, scales = [], []
    for _ in range(2):
        pool = torch.empty(n_pages, kvh, page, hd, dtype=FORMATS[case["format"]], device="cuda")
        scale = None if case["format"] == "bf16" else torch.empty(n_pages, kvh, page, device="cuda")
        step = max(1, (1 << 27) // (kvh * page * hd))
        for p in range(0, n_pages, step):
            rows = _rows(gen, min(step, n_pages - p), page, kvh, hd).transpose(1, 2)
            codes, s = _quantise(rows, case["format"])
            pool[p:p + step] = codes
            if scale is not None:
                scale[p:p + step] = s
        pools.append(pool)
        scales.append(scale)
    starts = [0]
    for q in q_lens:
        starts.append(starts[-1] + q)
    state = {"case": case, "q_lens": q_lens, "kv_lens": kv_lens, "k_pages": pools[0], "v_pages": pools[1],
             "k_scale": scales[0], "v_scale": scales[1], "table": table.cuda(),
             "lens": torch.tensor(kv_lens, dtype=torch.int32).cuda(),
             "starts": torch.tensor(starts, dtype=torch.int32).cuda() if max(q_lens) > 1 else None,
             "max_q": max(q_lens), "total": starts[-1]}
    if case["op"] == "attention":
        state["q"] = _rows(gen, starts[-1], case["heads"], hd)
    if case["op"] == "append":  # k and v are column blocks of the fused q | k | v projection
        fused = _rows(gen, starts[-1], case["heads"] + 2 * kvh, hd)
        state["k"] = fused[:, case["heads"]:case["heads"] + kvh]
        state["v"] = fused[:, case["heads"] + kvh:]
    return state


def _prepare_logits(case, gen):
    batch, vocab = case["batch"], case["vocab"]
    lens, prompts = _history_lengths(case)
    state = {"case": case}
    state["logits"] = (torch.randn(batch, vocab, device="cuda", generator=gen) * 3.0).to(LOGIT_TYPES[case["dtype"]])
    # few tokens are frequent, most are rare
    u = torch.rand(batch, max(1, case["history"]), device="cuda", generator=gen)
    state["history"] = (u ** 4 * vocab).long().clamp_(max=vocab - 1)
    state["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    state["prompts"] = torch.tensor(prompts, dtype=torch.int32).cuda()
    state["repetition"] = 1.0 + 0.3 * torch.rand(batch, device="cuda", generator=gen)
    state["frequency"] = 0.5 * torch.rand(batch, device="cuda", generator=gen)
    state["presence"] = 0.5 * torch.rand(batch, device="cuda", generator=gen)
    state["bias"] = state["allowed"] = None
    if case["extras"]:
        sparse = torch.rand(vocab, device="cuda", generator=gen) < 0.01
        state["bias"] = torch.randn(vocab, device="cuda", generator=gen) * sparse
        # a grammar leaves some rows a handful of tokens and others nearly all
        share = torch.where(torch.arange(batch, device="cuda") % 2 == 0, 0.95, 0.01)[:, None]
        words = (vocab + 31) // 32
        packed = torch.zeros(batch, words, dtype=torch.int64, device="cuda")
        for bit in range(32):
            packed |= (torch.rand(batch, words, device="cuda", generator=gen) < share).long() << bit
        state["allowed"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
    return state


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "attention":
        return _plain_attention(state)
    if op == "append":
        _plain_write(state)
        return _plain_read(state, torch.float32)
    if op == "read":
        return _plain_read(state, torch.bfloat16)
    return _plain_logits(state)


def _run_own(state, op):
    from cs244c_llama_zero_b200.ops import functional as F

    if op == "logits":
        return F.adjust_logits(state["logits"], state["history"], state["lens"], prompt_lens=state["prompts"],
                               repetition_penalty=state["repetition"], frequency_penalty=state["frequency"],
                               presence_penalty=state["presence"], bias=state["bias"], allowed=state["allowed"])
    pages = F.KVPages(state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"])
    if op == "attention":
        return F.paged_attention(state["q"], pages, state["table"], state["lens"], q_starts=state["starts"],
                                 max_q_len=state["max_q"])
    if op == "append":
        F.kv_cache_write(pages, state["k"], state["v"], state["table"], state["lens"], q_starts=state["starts"])
    dtype = torch.float32 if op == "append" else torch.bfloat16
    return F.kv_cache_read(pages, state["table"], state["lens"], q_starts=state["starts"], total=state["total"],
                           dtype=dtype)


def _sequence(state, b, which):
    """K (or V) of sequence ``b`` as fp32 ``[kv_heads, kv_len, hd]``."""
    case = state["case"]
    n = state["kv_lens"][b]
    ids = state["table"][b, :(n + case["page"] - 1) // case["page"]].long()
    x = state[which + "_pages"][ids].float()
    if state[which + "_scale"] is not None:
        x = x * state[which + "_scale"][ids].unsqueeze(-1)
    return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])[:, :n]


def _plain_attention(state):
    case = state["case"]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty_like(state["q"])
    row = 0
    for b, (qn, n) in enumerate(zip(state["q_lens"], state["kv_lens"])):
        q = state["q"][row:row + qn].float().view(qn, case["kv_heads"], group, case["head_dim"])
        q = q.permute(1, 2, 0, 3).reshape(case["kv_heads"], group * qn, case["head_dim"])
        k, v = _sequence(state, b, "k"), _sequence(state, b, "v")
        s = torch.matmul(q, k.transpose(1, 2)).mul_(case["head_dim"] ** -0.5)
        if qn > 1:
            pos = torch.arange(n - qn, n, device="cuda").repeat(group)
            s.masked_fill_(torch.arange(n, device="cuda")[None, :] > pos[:, None], float("-inf"))
        s -= s.amax(dim=-1, keepdim=True)
        s.exp_()
        o = torch.matmul(s, v) / s.sum(dim=-1, keepdim=True)
        o = o.view(case["kv_heads"], group, qn, case["head_dim"]).permute(2, 0, 1, 3)
        out[row:row + qn] = o.reshape(qn, case["heads"], case["head_dim"])
        row += qn
    return out


def _places(state):
    """Page and offset of every new token, in the order of the rows."""
    q = torch.tensor(state["q_lens"]).cuda()
    n = torch.tensor(state["kv_lens"]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(state["q_lens"]), device="cuda"), q)
    first = (torch.cumsum(q, 0) - q)[seq]
    pos = (n - q)[seq] + torch.arange(seq.numel(), device="cuda") - first
    page = state["case"]["page"]
    return state["table"][seq, pos // page].long(), pos % page


def _plain_write(state):
    ids, offs = _places(state)
    for which in ("k", "v"):
        codes, scale = _quantise(state[which], state["case"]["format"])
        state[which + "_pages"][ids, :, offs] = codes
        if scale is not None:
            state[which + "_scale"][ids, :, offs] = scale


def _plain_read(state, dtype):
    ids, offs = _places(state)
    out = []
    for which in ("k", "v"):
        x = state[which + "_pages"].view(torch.int8 if state[which + "_scale"] is not None else torch.bfloat16)
        x = x[ids, :, offs].view(state[which + "_pages"].dtype).float()
        if state[which + "_scale"] is not None:
            x = x * state[which + "_scale"][ids, :, offs].unsqueeze(-1)
        out.append(x.to(dtype))
    return tuple(out)


def _plain_logits(state):
    logits, history = state["logits"], state["history"]
    x = logits.float()
    where = torch.arange(history.shape[1], device="cuda")[None, :]
    inside = where < state["lens"][:, None]
    generated = inside & (where >= state["prompts"][:, None])
    seen = torch.zeros_like(x).scatter_add_(1, history, inside.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, history, generated.float())
    r = state["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - (state["frequency"][:, None] * count + state["presence"][:, None] * (count > 0))
    if state["bias"] is not None:
        x = x + state["bias"]
    if state["allowed"] is not None:
        bits = (state["allowed"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        bits = bits.reshape(x.shape[0], -1)[:, :x.shape[1]]
        x = x.masked_fill(bits == 0, float("-inf"))
    return x.to(logits.dtype)


# ------------------------------------------------------------------------------------------ definition
def exact(case, seed):
    """What ``run`` returns, computed in 64 bits from the definitions, one head or row at a time."""
    state = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(state)
    if case["op"] == "attention":
        return _exact_attention(state)
    kvh, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    out = []
    for which in ("k", "v"):
        if case["op"] == "append":  # the value that the nearest code stands for; the cache gives it back
            x = state[which].double()
            if case["format"] != "bf16":
                top, limit = x.abs().amax(-1, keepdim=True), CODE_MAX[case["format"]]
                ratio = torch.where(top > 0, x * limit / top, 0.0)  # one rounding: ties stay ties
                if case["format"] == "int8":
                    near = torch.round(ratio)
                else:  # e4m3: 4 significant bits, spacing 2^-9 below 2^-6
                    exponent = torch.floor(torch.log2(ratio.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
                    spacing = torch.exp2(exponent - 3.0)
                    near = torch.round(ratio / spacing) * spacing
                x = near * top / limit
            out.append(x)
            continue
        rows = []
        for b, (qn, n) in enumerate(zip(state["q_lens"], state["kv_lens"])):
            pos = torch.arange(n - qn, n)
            flat = (state["table"][b].cpu().long()[pos // page].cuda() * kvh * page)[:, None]
            flat = flat + torch.arange(kvh, device="cuda") * page + (pos % page).cuda()[:, None]
            x = state[which + "_pages"].view(torch.uint8).reshape(-1, hd * (2 if case["format"] == "bf16" else 1))
            x = x[flat.reshape(-1)].view(FORMATS[case["format"]]).double().view(qn, kvh, hd)
            if state[which + "_scale"] is not None:
                x = x * state[which + "_scale"].reshape(-1)[flat].double()[:, :, None]
            rows.append(x)
        out.append(torch.cat(rows))
    return tuple(out)


def _exact_attention(state):
    case = state["case"]
    kvh, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // kvh
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(state["kv_lens"]):
        qn = state["q_lens"][b]
        row = sum(state["q_lens"][:b])
        ids = state["table"][b, :-(-n // page)].long()
        visible = torch.ones(qn, n, dtype=torch.bool, device="cuda").tril(n - qn)
        for head in range(kvh):
            k = state["k_pages"][ids, head].double()
            v = state["v_pages"][ids, head].double()
            if state["k_scale"] is not None:
                k = k * state["k_scale"][ids, head].double()[:, :, None]
                v = v * state["v_scale"][ids, head].double()[:, :, None]
            k, v = k.view(-1, hd)[:n], v.view(-1, hd)[:n]
            for h in range(head * group, (head + 1) * group):
                s = state["q"][row:row + qn, h].double() @ k.T / hd ** 0.5
                p = torch.softmax(torch.where(visible, s, float("-inf")), dim=-1)
                out[row:row + qn, h] = p @ v
    return out


def _exact_logits(state):
    case = state["case"]
    vocab = case["vocab"]
    rows = []
    for b in range(case["batch"]):
        n, start = int(state["lens"][b]), int(state["prompts"][b])
        x = state["logits"][b].double()
        seen = torch.bincount(state["history"][b, :n], minlength=vocab) > 0
        count = torch.bincount(state["history"][b, start:n], minlength=vocab).double()
        r = state["repetition"][b].double()
        x = torch.where(seen & (x > 0), x / r, torch.where(seen, x * r, x))
        x = x - state["frequency"][b].double() * count - state["presence"][b].double() * (count > 0)
        if state["bias"] is not None:
            x = x + state["bias"].double()
            words = state["allowed"][b].long() & 0xFFFFFFFF
            token = torch.arange(vocab, device="cuda")
            x = torch.where((words[token // 32] >> (token % 32)) & 1 == 1, x, float("-inf"))
        rows.append(x)
    return torch.stack(rows)
