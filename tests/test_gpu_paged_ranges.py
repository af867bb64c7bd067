"""One-token attention over 8-bit caches where scales and scores range widely: value scales over many powers of two, of
either sign and next to the smallest numbers, growing scores, queries with an outlying channel. Against a 64-bit
restatement over the numbers that the cache holds."""
import math

import pytest
import torch

import mold_b200 as mb
from tests import text_util as U

pytestmark = pytest.mark.gpu
TYPES = [torch.int8, torch.float8_e4m3fn]
SHAPES = [(8, 2, 128), (6, 2, 64), (24, 2, 128), (20, 1, 64)]  # up to 8 query heads a key head, and more


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rand(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


def close(got, ref, tol):
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {(off / tol).max():.2f}"


def attention64(q, k, v, dtype, scale=None):
    """q [H, D], k / v [n, H_kv, D] in f64 -> (out, tolerance) f64 [H, D], over all n keys. With A = sum_j w_j |v_j|:
      2^-8 |out| + 2^-134     the output's rounding to bf16, the smallest bf16 numbers included
      2^-11 A                 a weight's rounding to f16 in its normal range
      n 2^-36 max(max |v|, 2^-106)   below that range: half its last step, 2^-25, with 2^11 for a weight of 1 on the row of
                              the largest value scale, which counts as 2^-115 at least (codes are at most 448 < 2^9; the
                              n weights' sum is at least 1, the weight of the reference score): 448 * 2^-115 < 2^-106
      2^-11 A                 exponentials (2^-22) and f32 sums, in numerator and denominator
      2^-131                  joining the warps' parts: a factor of 2^-126 times an exponential is off by 2^-150 at most, on
                              at most 2^11 * 2^7 times the sum of weights
      (e^2d - 1) A            scores off by d: D additions in f32, one step each, D 2^-23 scale max_j sum |q k_j|; and the
                              query's form, u scale max |q| max_j sum |k_j|: int8 half a step of 1 / 32639 of the row's
                              largest magnitude, e4m3 half of f16's smallest step, 2^-25, of at most that magnitude
    """
    H, D = q.shape
    n, G = k.shape[0], H // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    k, v = (x.transpose(0, 1).repeat_interleave(G, 0) for x in (k, v))  # [H, n, D]
    q = q.double()[:, None]
    s = (q @ k.transpose(1, 2))[:, 0] * scale
    w = torch.softmax(s, -1)[:, None]
    out, a = (w @ v)[:, 0], (w @ v.abs())[:, 0]
    d = D * 2.0 ** -23 * scale * (q.abs() @ k.abs().transpose(1, 2)).amax((1, 2))
    u = 0.5 / 32639 if dtype == torch.int8 else 2.0 ** -25
    d = d + u * scale * q.abs().amax((1, 2)) * k.abs().sum(-1).amax(-1)
    tol = 2.0 ** -8 * out.abs() + 2.0 ** -134 + 2.0 ** -131 + (2.0 ** -10 + torch.expm1(2 * d)[:, None]) * a
    return out, tol + n * 2.0 ** -36 * max(float(v.abs().amax()), 2.0 ** -106)


def check(q, cache, pages, lengths, out, scale=None):
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = U.cached64(cache, pages, b, n)
        close(out[b], *attention64(q[b], k, v, cache.k.dtype, scale))


def tables(pages):
    """The pages' own narrow table (parts joined in a cluster where they are few) and a wide one (cut over all SMs)."""
    wide = torch.full((pages.table.shape[0], 400), -1, dtype=torch.int32, device="cuda")
    wide[:, :pages.table.shape[1]] = pages.table
    return pages.table, wide


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("order", ["ascending", "descending", "zeros_first", "shuffled"])
def test_value_scales_over_many_powers(cuda, dtype, H, Hkv, D, order):
    """Rows of V from 2^-20 to 2^10 along the length, on growing keys: the reference of the value scales moves by orders of
    magnitude, and differs between warps, blocks and parts."""
    lengths = [1000, 77, 0, 2500]
    pages = U.Pages(lengths, 16, seed=3)
    cache = mb.KVCache(pages.n_pages, 16, Hkv, D, dtype)
    T = sum(lengths)
    k, v = rand((T, Hkv, D), 1), rand((T, Hkv, D), 2)
    at = 0
    for n in lengths:
        if n:
            e = torch.linspace(-20, 10, n, device="cuda")
            if order == "descending":
                e = e.flip(0)
            elif order == "shuffled":
                e = e[torch.randperm(n, generator=torch.Generator().manual_seed(n)).cuda()]
            f = torch.exp2(e)
            if order == "zeros_first":
                f[:n // 3] = 0
            v[at:at + n] *= f[:, None, None].bfloat16()
            k[at:at + n] *= torch.linspace(0.1, 3.0, n, device="cuda")[:, None, None].bfloat16()
        at += n
    cache.write(k, v, pages.table, ints(lengths), cu=U.offsets(lengths))
    q = rand((len(lengths), H, D), 4)
    for table in tables(pages):
        for scale in (None, 2.0 ** -9):
            out = mb.attention_paged(q, cache, table, ints(lengths), scale=scale)
            check(q, cache, pages, lengths, out, scale)
    assert mb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16] + TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_growing_scores(cuda, dtype, H, Hkv, D):
    """Scores that keep growing along the length move the reference point again and again."""
    lengths = [1500, 300]
    pages = U.Pages(lengths, 32, seed=5)
    cache = mb.KVCache(pages.n_pages, 32, Hkv, D, dtype)
    k, v = rand((1800, Hkv, D), 11), rand((1800, Hkv, D), 12)
    k *= torch.cat([torch.linspace(0.2, 8.0, n, device="cuda") for n in lengths])[:, None, None].bfloat16()
    cache.write(k, v, pages.table, ints(lengths), cu=U.offsets(lengths))
    q = rand((2, H, D), 13, 1.5)
    for table in tables(pages):
        out = mb.attention_paged(q, cache, table, ints(lengths))
        if dtype != torch.bfloat16:
            check(q, cache, pages, lengths, out)
            continue
        for b, n in enumerate(lengths):
            kk, vv = U.cached64(cache, pages, b, n)
            keep = torch.ones((1, n), dtype=torch.bool, device="cuda")
            close(out[b:b + 1], *U.attention64(q[b:b + 1], kk, vv, keep))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_queries_with_an_outlying_channel(cuda, dtype, H, Hkv, D):
    """One channel of q far above the others, where the keys are small: the others' scores decide."""
    lengths = [200]
    pages = U.Pages(lengths, 64, seed=6)
    cache = mb.KVCache(pages.n_pages, 64, Hkv, D, dtype)
    k, v = rand((200, Hkv, D), 21), rand((200, Hkv, D), 22)
    k[:, :, 3] = 0
    cache.write(k, v, pages.table, ints(lengths), cu=U.offsets(lengths))
    q = rand((1, H, D), 23)
    q[:, :, 3] = 100.0
    check(q, cache, pages, lengths, mb.attention_paged(q, cache, pages.table, ints(lengths)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("scales", ["negative", "either", "2^-120", "2^-140", "small_and_zero", "keys"])
def test_finite_scales_of_another_writer(cuda, dtype, H, Hkv, D, scales):
    """Caches whose scales this library did not write: any finite number reads back as code times scale, and attention
    uses the same values."""
    lengths, page = [70, 900], 32
    pages = U.Pages(lengths, page, seed=7)
    g = torch.Generator(device="cuda").manual_seed(8)
    shape = (pages.n_pages, Hkv, page, D)
    k, v = (torch.randint(-127, 128, shape, generator=g, device="cuda") for _ in range(2))
    k, v = (x.to(torch.int8) if dtype == torch.int8 else x.float().to(dtype) for x in (k, v))
    ks, vs = (torch.rand(shape[:3], generator=g, device="cuda") + 0.5 for _ in range(2))
    ks /= 127 * math.sqrt(D) / 4
    sign = torch.randint(0, 2, shape[:3], generator=g, device="cuda") * 2.0 - 1
    power = torch.randint(-20, 1, shape[:3], generator=g, device="cuda").float()
    if scales == "keys":
        ks *= sign
    elif scales == "negative":
        vs *= -1
    elif scales == "either":
        vs *= sign
    elif scales == "small_and_zero":
        vs = vs * 2.0 ** -100 * torch.exp2(power) * (power < -3)
    else:
        vs = vs * 2.0 ** -100 * (2.0 ** -20 if scales == "2^-120" else 2.0 ** -40)
    cache = mb.KVCache.from_tensors(k, v, ks, vs)
    got = cache.read(pages.table, U.offsets(lengths), sum(lengths))
    q = rand((2, H, D), 9)
    for b, n in enumerate(lengths):
        at = sum(lengths[:b])
        for x, ref in zip(got, U.cached64(cache, pages, b, n)):
            assert torch.equal(x[at:at + n], ref.float().bfloat16())
    for table in tables(pages):
        check(q, cache, pages, lengths, mb.attention_paged(q, cache, table, ints(lengths)))
    assert mb.device_status() == 0
