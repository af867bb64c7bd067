"""Packed prompt attention and the paged key-value cache (write, read, one-token attention) against plain 64-bit
implementations, at the sizes, masks and layouts where they can go wrong. Tolerances: tests/text_util.py."""
import ctypes
import random

import pytest
import torch

import mold_b200 as mb
from mold_b200 import _lib
from tests import text_util as U

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.int8, torch.float8_e4m3fn]


def rand(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def close(got, ref, tol):
    assert torch.isfinite(got).all()
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got.double() - ref).abs() / tol).max():.2f}"


# ---------------------------------------------------------------- packed prompts

LENGTHS = {
    "ones": ([1], [1]),
    "tile_edges": ([63, 64, 65, 127, 128, 129], [63, 64, 65, 127, 128, 129]),
    "empty_and_short": ([0, 5, 0, 1, 3], [4, 0, 0, 1, 7]),
    "more_queries_than_keys": ([7, 130, 70], [3, 1, 64]),
    "past": ([1, 20, 64, 33], [1000, 129, 300, 33]),
    "long": ([777], [1301]),
    "many": ([(7 * i) % 31 for i in range(70)], [(7 * i) % 31 + (i % 3) * 40 for i in range(70)]),
}


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 128), (8, 2, 64), (28, 4, 128), (24, 1, 64), (5, 1, 128)])
def test_varlen(cuda, H, Hkv, D, lengths, causal):
    ms, ns = LENGTHS[lengths]
    q = rand((sum(ms), H, D), 1, 1.5)
    k, v = rand((sum(ns), Hkv, D), 2), rand((sum(ns), Hkv, D), 3)
    out = mb.attention_varlen(q, k, v, U.offsets(ms), U.offsets(ns), causal=causal)
    close(out, *U.varlen64(q, k, v, ms, ns, causal))
    assert mb.device_status() == 0


@pytest.mark.parametrize("G", [2, 3, 48, 100, 128])
def test_varlen_group_sizes(cuda, G):
    ms, ns = [3, 140], [9, 140]
    q, k, v = rand((143, G, 64), 4), rand((149, 1, 64), 5), rand((149, 1, 64), 6)
    out = mb.attention_varlen(q, k, v, U.offsets(ms), U.offsets(ns))
    close(out, *U.varlen64(q, k, v, ms, ns, True))


def test_varlen_growing_scores_rescale(cuda):
    """Scores that keep growing along the keys move every row's reference point again and again; a scale of one's own."""
    n, H, D = 500, 4, 128
    q = rand((n, H, D), 7)
    k = rand((n, 2, D), 8) * torch.linspace(0.2, 6.0, n, device="cuda")[:, None, None].bfloat16()
    v = rand((n, 2, D), 9)
    cu = U.offsets([n])
    for scale in (0.3, 2.0 ** -10):
        out = mb.attention_varlen(q, k, v, cu, scale=scale)
        close(out, *U.varlen64(q, k, v, [n], [n], True, scale))


def test_varlen_strided_views_and_rows_behind(cuda):
    """Views of one fused projection, odd strides that need a copy, and rows behind the last sequence left alone."""
    T, H, Hkv, D = 150, 6, 2, 64
    qkv = rand((T, H + 2 * Hkv, D), 10)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    ms = [40, 77]  # 33 rows belong to nobody
    out = torch.full((T, H + 1, D), 7.0, device="cuda", dtype=torch.bfloat16)
    got = mb.attention_varlen(q, k, v, U.offsets(ms), out=out[:, :H])
    ref, tol = U.varlen64(q, k, v, ms, ms, True)
    close(got[:117], ref, tol)
    assert (out[117:] == 7).all() and (out[:, H] == 7).all()
    odd = torch.empty(T * H * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(T, H, D).copy_(q)  # 2-byte aligned
    swapped = k.transpose(0, 1).contiguous().transpose(0, 1)  # heads outside tokens
    assert torch.equal(mb.attention_varlen(odd, swapped, v, U.offsets(ms))[:117], got[:117])
    with pytest.raises(ValueError, match="out"):
        mb.attention_varlen(q, k, v, U.offsets(ms), out=odd)


@pytest.mark.parametrize("pad,start", [(0, 8), (8, 0), (8, 8), (0, 16), (0, 0)])
def test_varlen_output_alignment(cuda, pad, start):
    """Rows of out that begin at odd multiples of 16 bytes, all of them or every other one."""
    T, H, Hkv, D = 77, 4, 2, 64
    q, k, v = rand((T, H, D), 12), rand((T, Hkv, D), 13), rand((T, Hkv, D), 14)
    flat = torch.full((T * (H * D + pad) + 32,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = flat[start:].as_strided((T, H, D), (H * D + pad, D, 1))
    want = mb.attention_varlen(q, k, v, ints([0, 30, T]))
    mb.attention_varlen(q, k, v, ints([0, 30, T]), out=out)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert (flat == 7).all()  # nothing beside the rows


@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 128), (16, 2, 64)])
def test_varlen_what_is_masked_does_not_reach_a_row(cuda, H, Hkv, D):
    """NaN and infinities in keys and values of later positions, other sequences and unowned rows."""
    ms = [90, 170, 30]
    q, k, v = rand((300, H, D), 11), rand((300, Hkv, D), 12), rand((300, Hkv, D), 13)
    cu = U.offsets(ms)
    ref, tol = U.varlen64(q, k, v, ms, ms, True)
    clean = mb.attention_varlen(q, k, v, cu)
    close(clean[:290], ref, tol)
    k2, v2 = k.clone(), v.clone()
    k2[290:], v2[290:] = float("nan"), float("inf")
    at = 90 + 100  # position 100 of the second sequence
    k2[at, 0, 3] = float("nan")
    v2[at, 0, 5] = float("inf")
    v2[at + 40, 0, 9] = float("nan")
    got = mb.attention_varlen(q, k2, v2, cu)
    free = torch.ones(300, dtype=torch.bool, device="cuda")
    free[at:260] = False
    free[290:] = False
    close(got[free], ref[free[:290]], tol[free[:290]])
    G = H // Hkv
    assert got[at:260, :G].isnan().all()  # a NaN key reaches every channel of its group's rows from its position on
    close(got[at:260, G:], ref[at:260, G:], tol[at:260, G:])
    # values alone: only their channels
    got = mb.attention_varlen(q, k, v2, cu)
    want = ref.clone()
    want[at:260, :G, 5] = float("inf")
    want[at + 40:260, :G, 9] = float("nan")
    odd = ~torch.isfinite(want)
    assert torch.equal(got[:290].double()[odd].nan_to_num(3.0), want[odd].nan_to_num(3.0))
    close(got[:290][~odd], ref[~odd], tol[~odd])
    # without a causal mask, the sequence's end is the only border
    got = mb.attention_varlen(q, k2, v2, cu, causal=False)
    full, ftol = U.varlen64(q, k, v, ms, ms, False)
    close(got[:90], full[:90], ftol[:90])
    close(got[260:290], full[260:], ftol[260:])
    # infinite scores: softmax of +inf is NaN, as is one of -inf alone; -inf beside others is weight 0
    k3 = k.clone()
    q3 = q.clone()
    q3[:, :, 0] = 1.0
    k3[89, :, 0] = float("inf")
    k3[90, :, 0] = float("-inf")
    got = mb.attention_varlen(q3, k3, v, cu)
    assert got[89].isnan().all() and torch.isfinite(got[:89]).all() and got[90].isnan().all()
    assert torch.isfinite(got[91:290]).all()


def test_varlen_repeats_captures_and_streams(cuda):
    ms = [33, 200, 5]
    q, k, v = rand((238, 8, 128), 14), rand((238, 2, 128), 15), rand((238, 2, 128), 16)
    cu = U.offsets(ms)
    a = mb.attention_varlen(q, k, v, cu)
    assert torch.equal(a, mb.attention_varlen(q, k, v, cu))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = mb.attention_varlen(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mb.attention_varlen(q, k, v, cu, out=out)
    for seed in (17, 18):
        q.copy_(rand(q.shape, seed))
        cu.copy_(U.offsets([100, 1, 137] if seed == 18 else ms))
        graph.replay()
        assert torch.equal(out, mb.attention_varlen(q, k, v, cu))


def test_varlen_offsets_past_32_bits(cuda):
    """Rows far apart: the last ones begin more than 2^31 elements from the first."""
    T, ld = 66000, 1 << 15
    big = torch.empty((T, ld), device="cuda", dtype=torch.bfloat16)
    q, k, v = (big[:, 64 * i:64 * i + 64].unsqueeze(1) for i in range(3))
    for i, x in enumerate((q, k, v)):
        x[T - 40:] = rand((40, 1, 64), 20 + i)
    out = big[:, 256:320].unsqueeze(1)
    mb.attention_varlen(q, k, v, ints([T - 40, T]), out=out)
    close(out[T - 40:], *U.varlen64(q[T - 40:], k[T - 40:], v[T - 40:], [40], [40], True))


# ---------------------------------------------------------------- cache

def make(dtype, lengths, page, Hkv, D, seed=0, width=None, extra=3):
    pages = U.Pages(lengths, page, seed=seed, width=width, extra=extra)
    return mb.KVCache(pages.n_pages, page, Hkv, D, dtype), pages


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,Hkv,D", [(16, 1, 128), (64, 3, 64), (256, 8, 128)])
def test_write_and_read_back(cuda, dtype, page, Hkv, D):
    """Two pieces of each prompt; codes and scales equal the definition's bit for bit, other rows stay as they were."""
    old, new = [0, 5, 100, 16, 33, 0], [1, 0, 70, 17, 300, 4]
    full = [a + b for a, b in zip(old, new)]
    cache, pages = make(dtype, full, page, Hkv, D)
    for t in cache._tensors:
        t.view(torch.uint8).fill_(1)
    before = [t.clone() for t in cache._tensors]
    rows = {}
    for piece, (n, lens) in enumerate(((old, old), (new, full))):
        kv = rand((sum(n) + 2, 2 * Hkv, D), 30 + piece)
        kv[:, :, 1] *= 20
        k, v = kv[:, :Hkv], kv[:, Hkv:]
        cache.write(k, v, pages.table, ints(lens), cu=U.offsets(n))
        at = 0
        for b, m in enumerate(n):
            rows.setdefault(b, []).append((k[at:at + m], v[at:at + m]))
            at += m
    touched = torch.zeros((pages.n_pages, page), dtype=torch.bool, device="cuda")
    for b, n in enumerate(full):
        want = [torch.cat([r[i] for r in rows[b]]) for i in (0, 1)]
        p, o = pages.rows(b, n)
        touched[p, o] = True
        for x, s, ref in zip((cache.k, cache.v), (cache.k_scale, cache.v_scale), want):
            if dtype == torch.bfloat16:
                assert torch.equal(x[p, :, o], ref)
                continue
            c, sc = U.encode(ref, dtype)
            assert torch.equal(s[p, :, o].cpu(), sc)
            got = x.view(torch.uint8)[p, :, o]
            got = got.view(torch.int8).double() if dtype == torch.int8 else U.e4m3_values().cuda()[got.long()]
            assert torch.equal(got.cpu(), c)
    for t, b4 in zip(cache._tensors, before):
        same = (t == b4) if t.dtype != torch.float8_e4m3fn else t.view(torch.uint8) == b4.view(torch.uint8)
        same = same.flatten(3).all(-1) if t.dim() == 4 else same
        assert same.transpose(1, 2)[~touched].all()
    # read back: the 32-bit product rounded once; rows behind the last sequence stay
    cu = U.offsets(full)
    k, v = (torch.full((sum(full) + 3, Hkv, D), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    cache.read(pages.table, cu, k=k, v=v)
    k2, v2 = cache.read(pages.table, cu)
    assert (k[sum(full):] == 7).all() and (v[sum(full):] == 7).all()
    assert torch.equal(k[:sum(full)], k2) and torch.equal(v[:sum(full)], v2)
    at = 0
    for b, n in enumerate(full):
        for got, ref in zip((k2, v2), U.cached64(cache, pages, b, n)):
            assert torch.equal(got[at:at + n], ref.float().bfloat16())
        at += n
    assert mb.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_write_odd_rows(cuda, dtype):
    """All-zero rows, rows of one value, the smallest and largest numbers, NaN and infinities."""
    D, vals = 64, [0.0, -0.0, 2.0 ** -126, 2.0 ** -101, 2.0 ** -100, 1e-20, 3.0, 3.3e38, -3.3e38]
    x = torch.zeros((len(vals) + 4, 1, D), device="cuda", dtype=torch.bfloat16)
    for i, s in enumerate(vals):
        x[i, 0, i % D] = s
        x[i, 0, 40] = s / 3
    n = len(vals)
    x[n], x[n + 1, 0, 5], x[n + 2, 0, 6], x[n + 3, 0, 7] = -1.7, float("nan"), float("inf"), float("-inf")
    x[n + 1:, 0, 20] = 1.0
    cache, pages = make(dtype, [n + 4], 16, 1, D)
    cache.write(x, -x, pages.table, ints([n + 4]), cu=U.offsets([n + 4]))
    k, v = cache.read(pages.table, U.offsets([n + 4]))
    assert k[n + 1:].isnan().all() and v[n + 1:].isnan().all()
    c, s = U.encode(x[:n + 1], dtype)
    want = (c * s[..., None].double()).float().bfloat16()
    assert torch.equal(k[:n + 1].cpu(), want) and torch.equal(v[:n + 1].cpu(), -want)
    assert (k[:4] == 0).all()


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("exponent", [-100, 0, 120])
def test_write_scales_and_ties(cuda, dtype, exponent):
    """Rows whose largest value has each of the 128 bf16 fractions, full of values that lie on or next to the border of
    two codes: scales, inverses and products are rounded as the definition says."""
    D, half = 128, 0.5 if dtype == torch.int8 else 2.0 ** -4
    top = torch.arange(128, 256).double() / 128
    grid = torch.arange(1, D).double() / D
    codes = torch.floor(grid * 126) + half if dtype == torch.int8 else U.e4m3_values()[torch.arange(1, D) % 119 + 8] * (1 + half)
    x = torch.cat([top[:, None], codes[None] * top[:, None] / U.TOP[dtype]], 1)
    x = (x * 2.0 ** exponent).bfloat16()[:, None].cuda()
    x[:, :, 1::2] *= -1
    cache, pages = make(dtype, [128], 32, 1, D)
    cache.write(x, x, pages.table, ints([128]), cu=U.offsets([128]))
    p, o = pages.rows(0, 128)
    c, s = U.encode(x, dtype)
    assert torch.equal(cache.k_scale[p, :, o].cpu(), s) and torch.equal(cache.v_scale[p, :, o].cpu(), s)
    got = cache.k.view(torch.uint8)[p, :, o]
    got = got.view(torch.int8).double() if dtype == torch.int8 else U.e4m3_values().cuda()[got.long()]
    assert torch.equal(got.cpu(), c)


def test_write_every_code(cuda):
    """All 256 e4m3 and 255 int8 codes come out of the kernels' decoding as their numbers."""
    t = U.e4m3_values()
    for dtype, values in ((torch.int8, torch.arange(-127, 128).double()), (torch.float8_e4m3fn, t[~t.isnan()])):
        D = 64
        rows = -(-values.numel() // (D - 1))
        x = torch.zeros((rows, D), dtype=torch.float64)
        x[:, 0] = U.TOP[dtype]
        for i, val in enumerate(values.tolist()):
            x[i // (D - 1), 1 + i % (D - 1)] = val
        x = x.bfloat16()[:, None].cuda()
        cache, pages = make(dtype, [1] * rows, 16, 1, D)  # the scale is 1
        cache.write(x, x, pages.table, ints([1] * rows))
        k, v = cache.read(pages.table, U.offsets([1] * rows))
        assert torch.equal(k, x) and torch.equal(v, x)
        # attention over a single position returns its value row
        assert torch.equal(mb.attention_paged(rand((rows, 1, D), 3), cache, pages.table, ints([1] * rows)), x)


def test_write_one_token_each(cuda):
    """The generation step's form, with sequences of a padded batch passed over."""
    lens = [1, 0, 17, 64, -3, 200]
    cache, pages = make(torch.bfloat16, [max(n, 0) for n in lens], 16, 2, 128)
    k, v = rand((6, 2, 128), 40), rand((6, 2, 128), 41)
    cache.write(k, v, pages.table, ints(lens))
    seen = 0
    for b, n in enumerate(lens):
        if n > 0:
            p, o = pages.rows(b, n)
            assert torch.equal(cache.k[p[-1], :, o[-1]], k[b]) and torch.equal(cache.v[p[-1], :, o[-1]], v[b])
            seen += 1
    assert int((cache.k != 0).any(-1).any(1).sum()) == seen
    assert mb.device_status() == 0


def test_write_before_position_zero_and_unowned_rows(cuda):
    """A length shorter than the rows of its sequence keeps the last ones; rows before the first and behind the last
    sequence belong to nobody; offsets that do not begin at 0."""
    cache, pages = make(torch.int8, [40, 40], 16, 2, 64)
    k, v = rand((70, 2, 64), 45), rand((70, 2, 64), 46)
    cache.write(k, v, pages.table, ints([10, 33]), cu=ints([3, 20, 60]))
    assert mb.device_status() == 0
    n = [10, 33]
    for b, first in ((0, 10), (1, 27)):  # sequence 0: rows 3 .. 19, the last ten; sequence 1: rows 20 .. 59, the last 33
        c, s = U.encode(k[first:first + n[b]], torch.int8)
        p, o = pages.rows(b, n[b])
        assert torch.equal(cache.k[p, :, o].cpu().double(), c) and torch.equal(cache.k_scale[p, :, o].cpu(), s)
    kk, vv = (torch.full((50, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    cache.read(pages.table, ints([2, 12, 45]), k=kk, v=vv)
    assert (kk[:2] == 7).all() and (kk[45:] == 7).all() and (vv[:2] == 7).all() and (vv[45:] == 7).all()
    whole = cache.read(pages.table, U.offsets([10, 33]))
    assert torch.equal(kk[2:45], whole[0]) and torch.equal(vv[2:45], whole[1])


def test_bad_pages_are_reported_and_not_touched(cuda):
    """Page numbers outside the cache, and positions behind the table: an error status, no access, the rest right."""
    cache, pages = make(torch.int8, [40, 40], 16, 2, 64)
    k, v = rand((80, 2, 64), 42), rand((80, 2, 64), 43)
    cu, lens = U.offsets([40, 40]), ints([40, 40])
    cache.write(k, v, pages.table, lens, cu=cu)
    ok = cache.read(pages.table, cu)
    before = cache.k.clone()
    bad = pages.table.clone()
    bad[0, 1], bad[1, 2] = pages.n_pages, -5
    assert mb.device_status() == 0
    cache.write(k, v, bad, lens, cu=cu)
    assert mb.device_status() == _lib.DEV_BAD_PAGE and torch.equal(cache.k, before)
    got = cache.read(bad, cu)
    assert mb.device_status() == _lib.DEV_BAD_PAGE
    for x, y in zip(got, ok):
        assert (x[16:32] == 0).all() and (x[72:] == 0).all()
        assert torch.equal(x[:16], y[:16]) and torch.equal(x[32:72], y[32:72])
    cache.write(k, v, pages.table[:, :2], lens, cu=cu)  # 40 positions, 32 in the table
    assert mb.device_status() == _lib.DEV_BAD_PAGE and torch.equal(cache.k, before)
    # attention leaves keys without a page out
    q = rand((2, 4, 64), 44)
    out = mb.attention_paged(q, cache, bad, lens)
    assert mb.device_status() == _lib.DEV_BAD_PAGE
    for b, left in ((0, list(range(16)) + list(range(32, 40))), (1, list(range(32)))):
        kk, vv = U.cached64(cache, pages, b, 40)
        keep = torch.ones((1, len(left)), dtype=torch.bool, device="cuda")
        ref, tol = U.attention64(q[b:b + 1], kk[left], vv[left], keep, half_weights=True)
        close(out[b:b + 1], ref, tol)


# ---------------------------------------------------------------- one token

def filled(dtype, lengths, page, Hkv, D, seed, width=None):
    cache, pages = make(dtype, lengths, page, Hkv, D, seed=seed, width=width)
    # rows that no sequence has: whatever would do most harm
    if dtype == torch.bfloat16:
        cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))
    else:
        cache.k.view(torch.uint8).fill_(0x7f), cache.v.view(torch.uint8).fill_(0x7f)
        cache.k_scale.fill_(float("nan")), cache.v_scale.fill_(float("nan"))
    kv = rand((sum(lengths), 2 * Hkv, D), seed + 1)
    kv[:, :Hkv, 2] *= 6
    cache.write(kv[:, :Hkv], kv[:, Hkv:], pages.table, ints(lengths), cu=U.offsets(lengths))
    return cache, pages


def check_paged(q, cache, pages, lengths, out, scale=None):
    for b, n in enumerate(lengths):
        k, v = U.cached64(cache, pages, b, n)
        ref, tol = U.attention64(q[b:b + 1], k, v, torch.ones((1, n), dtype=torch.bool, device="cuda"), scale,
                                 half_weights=cache.k.dtype != torch.bfloat16)
        close(out[b:b + 1], ref, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 64), (28, 4, 128), (8, 8, 128), (16, 1, 64), (24, 1, 128), (33, 1, 64),
                                     (64, 8, 64), (10, 2, 128)])
@pytest.mark.parametrize("page", [16, 128])
def test_paged(cuda, dtype, H, Hkv, D, page):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 2000]
    cache, pages = filled(dtype, lengths, page, Hkv, D, 50)
    q = rand((len(lengths), H, D), 52, 1.5)
    out = mb.attention_paged(q, cache, pages.table, ints(lengths))
    check_paged(q, cache, pages, lengths, out)
    assert torch.equal(out, mb.attention_paged(q, cache, pages.table, ints(lengths)))
    assert mb.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[1], [40], [30011], [70000, 3], [100] * 150 + [9000] + [0] * 149, [65] * 1000])
def test_paged_splits(cuda, dtype, lengths):
    """From one tile to far more than there are blocks, even and lopsided batches, more sequences than threads."""
    cache, pages = filled(dtype, lengths, 32, 2, 128, 60)
    q = rand((len(lengths), 10, 128), 61, 2.0)
    out = mb.attention_paged(q, cache, pages.table, ints(lengths))
    some = range(len(lengths)) if len(lengths) < 10 else random.Random(1).sample(range(len(lengths)), 20) + [150]
    for b in some:
        k, v = U.cached64(cache, pages, b, lengths[b])
        keep = torch.ones((1, lengths[b]), dtype=torch.bool, device="cuda")
        close(out[b:b + 1], *U.attention64(q[b:b + 1], k, v, keep, half_weights=dtype != torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 1, 128), (12, 4, 64), (40, 2, 128)])
def test_paged_short_and_long_tables(cuda, dtype, H, Hkv, D):
    """The same sequences under a table of few pages, whose parts meet in a cluster, and one of many, which is cut over
    all SMs; 1 to more tiles than a cluster has blocks, and none."""
    for lengths in ([700], [0, 1, 4000], [64, 65], [512, 513, 1100], [0]):
        cache, pages = filled(dtype, lengths, 16, Hkv, D, 150)
        q = rand((len(lengths), H, D), 151, 1.5)
        wide = torch.full((len(lengths), 300), -1, dtype=torch.int32, device="cuda")
        wide[:, :pages.table.shape[1]] = pages.table
        for table in (pages.table, wide):
            out = mb.attention_paged(q, cache, table, ints(lengths))
            check_paged(q, cache, pages, lengths, out)
            assert torch.equal(out, mb.attention_paged(q, cache, table, ints(lengths)))
    assert mb.device_status() == 0


def test_paged_layouts_scale_and_padding(cuda):
    """Strided q and out, a table wider than the pages, lengths behind the table cut to it, negative lengths, scales."""
    lengths = [100, 7, 48]
    cache, pages = filled(torch.int8, lengths, 16, 2, 64, 70, width=40)
    q = rand((3, 9, 64), 71)[:, :6]
    out = torch.full((3, 8, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    wide = torch.full((3, 50), 12345, dtype=torch.int32, device="cuda")
    wide[:, :40] = pages.table
    for scale in (None, 1.0, 2.0 ** -12):
        mb.attention_paged(q, cache, wide[:, :40], ints(lengths), scale=scale, out=out[:, :6])
        check_paged(q, cache, pages, lengths, out[:, :6], scale)
        assert (out[:, 6:] == 7).all()
    got = mb.attention_paged(q, cache, pages.table[:, :3].contiguous(), ints([100, 7, 1 << 30]))
    check_paged(q, cache, pages, [48, 7, 48], got)
    got = mb.attention_paged(q, cache, pages.table, ints([-1, 7, 0]))
    assert (got[0] == 0).all() and (got[2] == 0).all()
    assert mb.device_status() == 0
    with pytest.raises(ValueError, match="positive"):
        mb.attention_paged(q, cache, pages.table, ints(lengths), scale=-1.0)
    with pytest.raises(ValueError, match="kv_lens"):
        mb.attention_paged(q, cache, pages.table, ints([1, 2]))
    with pytest.raises(ValueError, match="table"):
        mb.attention_paged(q, cache, pages.table[:2], ints(lengths))
    with pytest.raises(ValueError, match="int32"):
        mb.attention_paged(q, cache, pages.table.long(), ints(lengths))
    with pytest.raises(mb.MoldError, match="multiple"):
        mb.attention_paged(q[:, :5], cache, pages.table, ints(lengths))


def test_paged_not_finite(cuda):
    """What is not finite in a cached key or value reaches its own sequence and group only."""
    lengths = [50, 300]
    cache, pages = filled(torch.bfloat16, lengths, 16, 2, 64, 80)
    q = rand((2, 8, 64), 81)
    q[:, :, 0] = 1.0
    clean = mb.attention_paged(q, cache, pages.table, ints(lengths))
    p, o = pages.rows(1, 300)
    cache.k[p[200], 1, o[200], 0] = float("inf")
    cache.v[p[10], 0, o[10], 5] = float("-inf")
    got = mb.attention_paged(q, cache, pages.table, ints(lengths))
    assert torch.equal(got[0], clean[0]) and got[1, 4:].isnan().all()
    assert (got[1, :4, 5] == float("-inf")).all()
    got[1, :4, 5] = clean[1, :4, 5]
    assert torch.equal(got[1, :4], clean[1, :4])
    cache.k[p[200], 1, o[200], 0] = float("-inf")  # weight 0
    cache.k[p[201], 1, o[201]] = float("nan")
    got = mb.attention_paged(q, cache, pages.table, ints(lengths))
    assert got[1, 4:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("width", [None, 300])
def test_paged_not_finite_8_bit(cuda, dtype, width):
    """A cached row that was NaN when it was written makes its group's output NaN, and nothing else; queries that are not
    finite make theirs."""
    cache, pages = filled(dtype, [70, 500], 16, 2, 128, 82, width=width)
    q = rand((2, 6, 128), 83)
    lens = ints([70, 500])
    clean = mb.attention_paged(q, cache, pages.table, lens)
    new = rand((2, 2, 128), 84)
    new[1, 1, 7] = float("nan")
    cache.write(new, rand((2, 2, 128), 85), pages.table, ints([0, 500]))
    got = mb.attention_paged(q, cache, pages.table, lens)
    assert torch.equal(got[0], clean[0]) and got[1, 3:].isnan().all() and torch.isfinite(got[1, :3]).all()
    q[0, 2, 5], q[0, 4, 6] = float("inf"), float("nan")
    got = mb.attention_paged(q, cache, pages.table, lens)
    assert got[0, 2].isnan().all() and got[0, 4].isnan().all()
    assert torch.equal(got[0, [0, 1, 3, 5]], clean[0, [0, 1, 3, 5]])


def test_paged_offsets_past_32_bits(cuda):
    """The last pages of a cache of more than 2^32 elements."""
    n_pages, Hkv, page, D = 4300, 32, 256, 128
    k = torch.empty((n_pages, Hkv, page, D), device="cuda", dtype=torch.int8)
    v, ks, vs = torch.empty_like(k), *(torch.empty((n_pages, Hkv, page), device="cuda") for _ in range(2))
    cache = mb.KVCache.from_tensors(k, v, ks, vs)
    pages = U.Pages([300], page, extra=0)
    pages.host = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32)
    pages.table = pages.host.cuda()
    kn, vn = rand((300, Hkv, D), 90), rand((300, Hkv, D), 91)
    cache.write(kn, vn, pages.table, ints([300]), cu=U.offsets([300]))
    got = cache.read(pages.table, U.offsets([300]), 300)
    for x, y in zip(got, (kn, vn)):
        c, s = U.encode(y, torch.int8)
        assert torch.equal(x.cpu(), (c * s[..., None].double()).float().bfloat16())
    q = rand((1, Hkv, D), 92)
    check_paged(q, cache, pages, [300], mb.attention_paged(q, cache, pages.table, ints([300])))


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", TYPES)
def test_generation_run(cuda, dtype):
    """Prompts in two pieces through the cache, then tokens one by one inside one captured graph: every output equals
    64-bit attention over the rows that the cache holds."""
    H, Hkv, D, page = 12, 3, 64, 16
    first, second, steps = [20, 3, 64], [30, 1, 100], 5
    total = [a + b + steps for a, b in zip(first, second)]
    cache, pages = make(dtype, total, page, Hkv, D)
    lens = [0, 0, 0]
    for piece, new in enumerate((first, second)):
        T = sum(new)
        qkv = rand((T, H + 2 * Hkv, D), 100 + piece)
        q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        lens = [a + b for a, b in zip(lens, new)]
        cache.write(k, v, pages.table, ints(lens), cu=U.offsets(new))
        kk, vv = cache.read(pages.table, U.offsets(lens), sum(lens))
        out = mb.attention_varlen(q, kk, vv, U.offsets(new), U.offsets(lens))
        close(out, *U.varlen64(q, kk, vv, new, lens, True))
    qkv = torch.empty((3, H + 2 * Hkv, D), device="cuda", dtype=torch.bfloat16)
    dev_lens, out = ints(lens), torch.empty((3, H, D), device="cuda", dtype=torch.bfloat16)

    def step():
        dev_lens.add_(1)
        cache.write(qkv[:, H:H + Hkv], qkv[:, H + Hkv:], pages.table, dev_lens)
        mb.attention_paged(qkv[:, :H], cache, pages.table, dev_lens, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        qkv.copy_(rand(qkv.shape, 110 + i))
        graph.replay()
        lens = [n + 1 for n in lens]
        check_paged(qkv[:, :H], cache, pages, lens, out)
        for b, n in enumerate(lens):
            k, v = U.cached64(cache, pages, b, n)
            for x, y in ((k, qkv[b, H:H + Hkv]), (v, qkv[b, H + Hkv:])):
                # the newest row is the one just written: half a code step of its largest magnitude (int8 1/254,
                # e4m3 2^-4 of the value) at most
                slack = {torch.bfloat16: 0.0, torch.int8: 1 / 253.0, torch.float8_e4m3fn: 2.0 ** -4}[dtype]
                assert ((x[-1] - y.double()).abs() <= slack * y.double().abs().amax(-1, keepdim=True)).all()
    assert mb.device_status() == 0


def test_two_graphs_do_not_share_a_workspace(cuda):
    """Two captured calls replayed at once on two streams give what each gives alone."""
    sets, graphs, outs, refs = [], [], [], []
    for i in range(2):
        lengths = [3000 + 500 * i, 40]
        cache, pages = filled(torch.bfloat16, lengths, 16, 2, 128, 120 + i)
        q, lens = rand((2, 8, 128), 130 + i), ints(lengths)
        refs.append(mb.attention_paged(q, cache, pages.table, lens))
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
        with torch.cuda.graph(g):
            mb.attention_paged(q, cache, pages.table, lens, out=out)
        sets.append((cache, pages, q, lens))
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, refs))


def test_small_workspace_refused(cuda):
    cache, pages = filled(torch.bfloat16, [20], 16, 1, 64, 140)
    q = rand((1, 2, 64), 141)
    ws = torch.empty(64, dtype=torch.uint8, device="cuda")
    rc = mb.lib().mb_attention_paged(q.data_ptr(), 128, ctypes.byref(cache._c), ints([20]).data_ptr(),
                                     pages.table.data_ptr(), pages.table.shape[1], pages.table.shape[1], 1, 2, 0.0,
                                     q.data_ptr(), 128, ws.data_ptr(), 64, None)
    assert rc == _lib.MB_ERR_INVALID and b"workspace" in mb.lib().mb_last_error()


@pytest.mark.parametrize("how", ["stream", "other_stream", "graph", "graph_copy", "graph_other_stream"])
def test_calls_wait_for_what_came_before(cuda, how):
    """Inputs that a slow kernel, a copy or another stream has only just made, eagerly and in captured graphs; and each call
    right behind the one whose results it takes."""
    H, Hkv, D, lengths = 6, 2, 128, [70, 33]
    cache, pages = make(torch.int8, lengths, 16, Hkv, D)
    lens, cu, T = ints(lengths), U.offsets(lengths), sum(lengths)
    src = [[rand(s, 150 + 10 * i + j) for j, s in enumerate(((T, H, D), (T, Hkv, D), (T, Hkv, D)))] for i in range(2)]
    now = [torch.empty_like(x) for x in src[0]]
    held = [torch.empty_like(x) for x in src[0]]
    kk, vv = torch.empty_like(src[0][1]), torch.empty_like(src[0][2])
    out, last = torch.empty_like(src[0][0]), torch.empty((2, H, D), device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()

    def make_inputs():
        torch.cuda._sleep(400000)  # clocks
        for x, y in zip(now, held):
            if how == "graph_copy":
                x.copy_(y)
            else:
                torch.add(y, 0.0, out=x)

    def calls():
        cache.write(now[1], now[2], pages.table, lens, cu=cu)
        cache.read(pages.table, cu, k=kk, v=vv)
        mb.attention_varlen(now[0], kk, vv, cu, out=out)
        mb.attention_paged(out[cu[1:].long() - 1] if graph is None else out[:2], cache, pages.table, lens, out=last)

    def run():
        if "other" in how:
            here = torch.cuda.current_stream()
            side.wait_stream(here)
            with torch.cuda.stream(side):
                make_inputs()
            here.wait_stream(side)
        else:
            make_inputs()
        calls()

    graph = torch.cuda.CUDAGraph() if "graph" in how else None
    refs = []
    for inputs in src:
        for x, y in zip(now, inputs):
            x.copy_(y)
        torch.cuda.synchronize()
        calls()
        torch.cuda.synchronize()
        refs.append([x.clone() for x in (kk, vv, out, last)])
    if graph is not None:
        with torch.cuda.graph(graph):
            run()
    for i in (0, 1, 1, 0, 1):
        for x, y in zip(held, src[i]):
            x.copy_(y)
        for x in (kk, vv, out, last):
            x.fill_(float("nan"))
        run() if graph is None else graph.replay()
        got = [x.clone() for x in (kk, vv, out, last)]
        assert all(torch.equal(x, y) for x, y in zip(got, refs[i]))
    assert mb.device_status() == 0
