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
