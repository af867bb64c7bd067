"""Packed prompt attention over thousands of sequences: short, empty and padded ones, and the time that a tile's search
takes. A sequence's rows do not depend on the others of the batch, so calls over a few sequences each give the same bits."""
import random

import pytest
import torch

import mold_b200 as mb
from tests import text_util as U

pytestmark = pytest.mark.gpu


def rand(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").bfloat16()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def batch(kind):
    r = random.Random(7)
    if kind == "short":
        ms = [r.randint(0, 40) for _ in range(3000)]
    elif kind == "mostly_empty":
        ms = [0] * 1500 + [5, 0, 130] + [0] * 2000 + [1] + [0] * 700
    elif kind == "one_token":
        ms = [1] * 2049
    else:
        ms = [r.choice([0, 1, 300]) if i % 97 == 0 else 2 for i in range(1025)]
    # keys: as many, a few more (a prefix), or now and then none at all
    return ms, [r.choice([0, m, m, m + 3, m + 70]) if m else r.choice([0, 4]) for m in ms]


@pytest.mark.parametrize("kind", ["short", "mostly_empty", "one_token", "lopsided"])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (9, 3, 128), (2, 2, 64)])
def test_many_sequences(cuda, kind, H, Hkv, D):
    ms, ns = batch(kind)
    before, behind = 13, 900  # rows of nobody
    q = rand((before + sum(ms) + behind, H, D), 1)
    k, v = rand((sum(ns), Hkv, D), 2), rand((sum(ns), Hkv, D), 3)
    cu_q = U.offsets(ms) + before
    cu_k = U.offsets(ns)
    out = torch.full_like(q, 7.0)
    mb.attention_varlen(q, k, v, cu_q, cu_k, out=out)
    assert (out[:before] == 7).all() and (out[before + sum(ms):] == 7).all()
    few = torch.full_like(q, 7.0)
    for b in range(0, len(ms), 30):
        mb.attention_varlen(q, k, v, cu_q[b:b + 31].contiguous(), cu_k[b:b + 31].contiguous(), out=few)
    assert torch.equal(out, few)
    host = cu_q.tolist(), cu_k.tolist()
    full = [b for b, m in enumerate(ms) if m]
    for b in random.Random(8).sample(full, min(4, len(full))):
        rows, keys = slice(host[0][b], host[0][b + 1]), slice(host[1][b], host[1][b + 1])
        ref, tol = U.varlen64(q[rows], k[keys], v[keys], [ms[b]], [ns[b]], True)
        assert ((out[rows].double() - ref).abs() <= tol).all()
    assert mb.device_status() == 0


def test_padded_rows_and_sequences(cuda):
    """A batch of fixed size, as a captured graph holds it, of which little is in use."""
    H, Hkv, D, T = 4, 2, 128, 20000
    q, k, v = rand((T, H, D), 4), rand((T, Hkv, D), 5), rand((T, Hkv, D), 6)
    cu = ints([0, 100, 140] + [140] * 600)
    out = torch.full_like(q, 7.0)
    mb.attention_varlen(q, k, v, cu, out=out)
    ref, tol = U.varlen64(q[:140], k[:140], v[:140], [100, 40], [100, 40], True)
    assert ((out[:140].double() - ref).abs() <= tol).all() and (out[140:] == 7).all()
    assert mb.device_status() == 0


def test_offsets_that_do_not_ascend_touch_no_row_outside(cuda):
    """Offsets out of range or order: whatever the rows inside become, none outside the tensors is touched, and the call
    ends."""
    H, Hkv, D, T = 4, 2, 64, 300
    r = random.Random(9)
    flat = torch.full(((T + 200) * H * D,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = flat[100 * H * D:(100 + T) * H * D].view(T, H, D)
    q, k, v = rand((T, H, D), 10), rand((T, Hkv, D), 11), rand((T, Hkv, D), 12)
    for n in (5, 40, 1100):
        cu = ints([r.randint(-1000, 1000) for _ in range(n + 1)])
        mb.attention_varlen(q, k, v, cu, ints([r.randint(-1000, 1000) for _ in range(n + 1)]), out=out)
    assert mb.device_status() == 0
    assert (flat[:100 * H * D] == 7).all() and (flat[(100 + T) * H * D:] == 7).all()


def test_time_grows_with_the_number_of_sequences_alone(cuda):
    """16 times the sequences take 16 times as long, not 256: a tile is not found by going through all of them."""
    H, Hkv, D, m = 8, 8, 64, 4

    def time(n):
        q, k, v = rand((n * m, H, D), 13), rand((n * m, Hkv, D), 14), rand((n * m, Hkv, D), 15)
        cu = torch.arange(0, n * m + 1, m, dtype=torch.int32, device="cuda")
        best = 1e30
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            mb.attention_varlen(q, k, v, cu)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(32768) < 32 * time(2048)
