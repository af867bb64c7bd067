"""Scales of the text-transformer attentions at the ends of their range, and cache sizes at the end of theirs."""
import pytest
import torch

import mold_b200 as mb
from mold_b200 import _lib, ops
from tests.test_text_ops import INVALID, NOT_READY, cache, paged, read, varlen, write


def test_a_small_scale_does_not_become_the_default():
    """Below the smallest 32-bit number a scale would reach the library as 0, which stands for 1 / sqrt(D)."""
    for scale in (1e-50, 5e-324, 1e-46, 1e-40):
        assert _lib.F32(ops._scale(scale)).value > 0
    assert ops._scale(0.25) == 0.25 and ops._scale(None) == 0.0
    for scale in (0, -1e-50, float("nan")):
        with pytest.raises(ValueError, match="positive"):
            ops._scale(scale)


@pytest.mark.parametrize("call", [varlen, paged])
def test_a_scale_whose_product_with_log2_e_is_not_finite_is_refused(call):
    assert call(scale=2.4e38) == call(scale=3.0e38) == INVALID
    if not torch.cuda.is_available():
        assert call(scale=2.3e38) == NOT_READY


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-50, 1e-42, 1e-30])
def test_tiny_scales_weigh_all_keys_alike(cuda, scale):
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((40, h, 64), generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    out = mb.attention_varlen(q, k, v, cu, causal=False, scale=scale)
    mean, size = (x.double().mean(0).repeat_interleave(2, 0)[None] for x in (v, v.abs()))
    # the output's rounding to bf16, the weights' (1 is exact), and the 32-bit sums
    assert ((out.double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -16 * size).all()
    table, lens = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), cu[1:].contiguous()
    cache = mb.KVCache(3, 16, 2, 64)
    cache.write(k, v, table, lens, cu=cu)
    out = mb.attention_paged(q[:1], cache, table, lens, scale=scale)
    assert ((out.double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -16 * size).all()


@pytest.mark.parametrize("heads,page", [(3, 16), (7, 64), (1, 16), (5, 256)])
def test_every_cache_below_2_to_the_31_rows_is_taken(heads, page):
    most = ((1 << 31) - 1) // (heads * page)
    for call in (paged, write, read):
        kw = {"H": 2 * heads, "ldq": 256 * heads, "ldo": 256 * heads} if call is paged else dict(ldk=128 * heads,
                                                                                                 ldv=128 * heads)
        if not torch.cuda.is_available():
            assert call(cache=cache(n_pages=most, n_kv_heads=heads, page_size=page), **kw) == NOT_READY
        assert call(cache=cache(n_pages=most + 1, n_kv_heads=heads, page_size=page), **kw) == INVALID


def test_more_tiles_than_a_launch_has_blocks_are_refused():
    """As an argument out of range, not as a failure of the device."""
    big = dict(H=128, Hkv=128, D=64, ldq=128 * 64, ldk=128 * 64, ldv=128 * 64, ldo=128 * 64)
    assert varlen(n=(1 << 24) - 1, tq=1 << 20, **big) == INVALID
    if not torch.cuda.is_available():
        assert varlen(n=(1 << 24) - 1, **{**big, "H": 64, "Hkv": 64}) == NOT_READY
