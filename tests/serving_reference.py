"""Plain 64-bit forms of the serving operators, and batches for their tests (CPU tensors)."""

from __future__ import annotations

import random
from typing import List, Optional, Sequence, Tuple

import torch

FORMATS = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}


def quantise(x: torch.Tensor, fmt: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes (as numbers) and scales of rows ``[..., hd]`` in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, x * CODE_MAX[fmt] / top, torch.zeros_like(x))
    codes = q.round() if fmt == "int8" else q.float().to(torch.float8_e4m3fn).double()
    return codes, (top / CODE_MAX[fmt]).squeeze(-1)


class Batch:
    """A paged pool with random contents, and sequences over it.  Everything behind a sequence's end, and
    every page that no sequence owns, holds NaN (8-bit formats: NaN scales)."""

    def __init__(self, q_lens: Sequence[int], kv_lens: Sequence[int], heads: int, kv_heads: int, hd: int, fmt: str,
                 page: int, seed: int = 0, behind: int = 0, amplitude: float = 1.0) -> None:
        gen = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        self.heads, self.kv_heads, self.hd, self.fmt, self.page = heads, kv_heads, hd, fmt, page
        counts = [-(-n // page) for n in kv_lens]
        self.n_pages = sum(counts) + 2
        order = torch.randperm(self.n_pages, generator=gen)
        self.table = torch.full((len(counts), max(counts + [1]) + 1), self.n_pages + 7, dtype=torch.int32)
        used = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[used:used + n].int()
            used += n
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32)
        self.lens = torch.tensor(list(kv_lens), dtype=torch.int32)
        self.total = starts[-1]
        self.max_q = max(list(q_lens) + [1])
        rows = self.total + behind
        strength = torch.empty(hd).log_normal_(0.0, 0.5, generator=gen)
        self.q = (torch.randn(rows, heads, hd, generator=gen) * amplitude).to(torch.bfloat16)
        self.k = (torch.randn(rows, kv_heads, hd, generator=gen) * strength).to(torch.bfloat16)
        self.v = (torch.randn(rows, kv_heads, hd, generator=gen) * strength).to(torch.bfloat16)
        self.pools, self.scales = [], []
        live = torch.zeros(self.n_pages, page, dtype=torch.bool)
        for b, n in enumerate(kv_lens):
            for t in range(n):
                live[self.table[b, t // page], t % page] = True
        self.live = live
        for _ in range(2):
            x = (torch.randn(self.n_pages, kv_heads, page, hd, generator=gen) * strength).to(torch.bfloat16)
            dead = ~live[:, None, :, None]
            if fmt == "bf16":
                self.pools.append(x.masked_fill(dead, float("nan")))
                self.scales.append(None)
            else:
                codes, scale = quantise(x, fmt)
                codes = codes.float().to(FORMATS[fmt])
                if fmt == "e4m3":  # dead places: the NaN code
                    codes = codes.view(torch.uint8).masked_fill(dead, 0x7F).view(torch.float8_e4m3fn)
                self.pools.append(codes)
                self.scales.append(scale.float().masked_fill(~live[:, None, :], float("nan")))

    def pages(self, device: str = "cpu"):
        from cs244c_llama_zero_b200.ops.functional import KVPages

        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return KVPages(move(self.pools[0]), move(self.pools[1]), move(self.scales[0]), move(self.scales[1]))

    def sequence(self, b: int, which: int) -> torch.Tensor:
        """K (0) or V (1) of sequence ``b``: float64 ``[kv_len, kv_heads, hd]``."""
        rows = []
        for t in range(self.kv_lens[b]):
            p, o = int(self.table[b, t // self.page]), t % self.page
            x = self.pools[which][p, :, o].double()
            if self.scales[which] is not None:
                x = x * self.scales[which][p, :, o].double()[:, None]
            rows.append(x)
        return torch.stack(rows) if rows else torch.zeros(0, self.kv_heads, self.hd, dtype=torch.float64)

    def attention(self, scale: Optional[float] = None):
        """Per row and head: the output, ``sum_j p_j |v_j|`` and the largest ``scale * sum_d |q_d k_d|``."""
        scale = self.hd ** -0.5 if scale is None else scale
        group = self.heads // self.kv_heads
        out = torch.zeros(self.total, self.heads, self.hd, dtype=torch.float64)
        mag = torch.zeros_like(out)
        size = torch.zeros(self.total, self.heads, 1, dtype=torch.float64)
        for b, (qn, n) in enumerate(zip(self.q_lens, self.kv_lens)):
            r0 = int(self.starts[b])
            k = self.sequence(b, 0).repeat_interleave(group, 1)
            v = self.sequence(b, 1).repeat_interleave(group, 1)
            q = self.q[r0:r0 + qn].double()
            s = torch.einsum("ihd,jhd->hij", q, k) * scale
            a = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * scale
            hidden = torch.arange(n)[None, :] > (torch.arange(qn) + n - qn)[:, None]
            p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)
            out[r0:r0 + qn] = torch.einsum("hij,jhd->ihd", p, v)
            mag[r0:r0 + qn] = torch.einsum("hij,jhd->ihd", p, v.abs())
            if n > 0:
                size[r0:r0 + qn] = a.masked_fill(hidden, 0.0).amax(-1).t()[..., None]
        return out, mag, size


def tolerance(out: torch.Tensor, mag: torch.Tensor, size: torch.Tensor, quantised: bool) -> torch.Tensor:
    """Rounding bound of the attention kernels, u = 2^-8 (half a step of bf16): the result is rounded once
    (u |o|), each probability once before it meets V (u sum p |v|).  8-bit caches may also be expanded to
    bf16 keys and values first: u sum p |v| again, and scores off by u * scale * sum |q k|, which moves a
    probability by that relative amount, and the normaliser likewise (2 u size sum p |v|).  The fp32 parts
    (scores, exponentials, sums) add a few 2^-22 per unit of score: 2^-20 (1 + size) sum p |v|."""
    u = 2.0 ** -8
    tol = u * out.abs() + (u + 2.0 ** -20 * (1 + size)) * mag
    if quantised:
        tol = tol + (u + 2 * u * size) * mag
    return tol * 1.02 + 1e-30  # second-order terms


def adjusted(logits, history, lens, prompts, rep, freq, pres, bias, allowed) -> torch.Tensor:
    out = logits.double()
    vocab = logits.shape[1]
    for b in range(logits.shape[0]):
        if history is not None:
            n = int(lens[b])
            start = 0 if prompts is None else int(prompts[b])
            hist: List[int] = [int(t) for t in history[b, :n]]
            for t in set(hist):
                l = out[b, t]
                if rep is not None:
                    l = l / float(rep[b]) if l > 0 else l * float(rep[b])
                count = hist[start:].count(t)
                if count:
                    l = l - (float(freq[b]) * count if freq is not None else 0.0)
                    l = l - (float(pres[b]) if pres is not None else 0.0)
                out[b, t] = l
        if bias is not None:
            out[b] += (bias if bias.dim() == 1 else bias[b]).double()
        if allowed is not None:
            mask = allowed if allowed.dim() == 1 else allowed[b]
            for t in range(vocab):
                if not (int(mask[t // 32]) >> (t % 32)) & 1:
                    out[b, t] = float("-inf")
    return out


def ragged(seed: int, batch: int, max_q: int, max_kv: int) -> Tuple[List[int], List[int]]:
    rng = random.Random(seed)
    q = [rng.randint(0, max_q) for _ in range(batch)]
    return q, [max(n, rng.randint(0, max_kv)) for n in q]
