"""Rounding bounds of the attention kernels over a paged cache, format by format.

Half steps, relative to the value: bf16 2^-8, fp16 2^-11, fp32 2^-24.  With p the probabilities, mag = sum p |v|
and size = the largest scale * sum_d |q_d k_d| that a row meets (``Batch.attention``):

* every form rounds the result once to bf16 (2^-8 |o|) and sums in fp32 (scores, exponentials and sums: a few
  2^-22 for each unit of score, 2^-20 (1 + size) mag);
* bf16 pages: each probability once to bf16 before it meets V (2^-8 mag);
* 8-bit pages, few rows: each weight once to fp16 (2^-11 mag); q, the codes and the powers of two are exact.
  q keeps its 8 bits down to 2^-17 of its row's maximum and is off by 2^-25 of that below;
* 8-bit pages, chunks: each weight once to fp16 (2^-11 mag), V twice (a token's factor, its product with the code:
  2 * 2^-11 mag), K twice (a score is off by 2 * 2^-11 size, which moves its probability and the normaliser by that
  relative amount: 2 * 2 * 2^-11 size mag).

The bounds are those of the wider 8-bit form, so that they hold whichever one a call takes.
"""

from __future__ import annotations

import torch

BF16, FP16 = 2.0 ** -8, 2.0 ** -11


def bound(out: torch.Tensor, mag: torch.Tensor, size: torch.Tensor, fmt: str) -> torch.Tensor:
    """For each element, how far the kernel's output may be from the 64-bit one."""
    tol = BF16 * out.abs() + 2.0 ** -20 * (1 + size) * mag
    tol = tol + (BF16 * mag if fmt == "bf16" else (3 * FP16 + 4 * FP16 * size) * mag)
    return tol * 1.02 + 2.0 ** -133  # second-order terms; a bf16 result below 2^-126 keeps 2^-133


def norm_bound(fmt: str) -> float:
    """For a whole output of ordinary activations: error norm over result norm.

    A rounding to nearest is off by its half step times a number spread evenly over [-1, 1]; the value it is relative
    to lies anywhere in its binade, whose mean square is 1.5 / ln 2 = 2.16 times the square of its lower end.  So a
    rounding adds u / sqrt(3) / sqrt(2.16) = 0.39 u to the relative norm: 0.0015 for the result, the same again for
    bf16 probabilities, 0.0002 for fp16 ones, 0.0003 for V.  A score that is off by 0.39 * 2^-11 of its size (up to 4
    for these activations) twice adds 0.0011.  In quadrature: bf16 0.0022, 8-bit 0.0019; with a fifth on top.  K and V
    rounded to bf16 instead of fp16 would give 0.0040 or more."""
    return 0.0027 if fmt == "bf16" else 0.0023
