"""Refusals of the text-transformer entry points (packed attention, paged cache), none of which needs a GPU: the C ABI
rejects bad shapes, strides, alignments and types with the documented status before any device work, and the Python
front refuses tensors that do not fit together."""
import ctypes
import os
import re

import pytest
import torch

import mold_b200 as mb
from mold_b200 import _lib

P = 1 << 20  # an aligned address that no refused call may follow
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cache(**kw):
    f = dict(k=P, v=P, k_scale=None, v_scale=None, n_pages=4, page_size=16, n_kv_heads=2, head_dim=128,
             dtype=_lib.KV_BF16)
    f.update(kw)
    return ctypes.byref(_lib.KVCacheC(**f))


def varlen(**kw):
    f = dict(q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, tq=10, tk=10, H=4, Hkv=2, D=128, cu_q=P, cu_k=P, n=1, causal=1,
             scale=0.0, out=P, ldo=512, stream=None)
    f.update(kw)
    return mb.lib().mb_attention_varlen(*f.values())


def paged(**kw):
    f = dict(q=P, ldq=512, cache=cache(), lens=P, table=P, ldt=8, width=8, n=2, H=4, scale=0.0, out=P, ldo=512, ws=P,
             nbytes=1 << 30, stream=None)
    f.update(kw)
    return mb.lib().mb_attention_paged(*f.values())


def write(**kw):
    f = dict(cache=cache(), k=P, ldk=256, v=P, ldv=256, tokens=2, cu=None, lens=P, table=P, ldt=8, width=8, n=2,
             stream=None)
    f.update(kw)
    return mb.lib().mb_kv_write(*f.values())


def read(**kw):
    f = dict(cache=cache(), cu=P, table=P, ldt=8, width=8, n=2, tokens=5, k=P, ldk=256, v=P, ldv=256, stream=None)
    f.update(kw)
    return mb.lib().mb_kv_read(*f.values())


INVALID, UNSUPPORTED, NOT_READY = _lib.MB_ERR_INVALID, _lib.MB_ERR_UNSUPPORTED, _lib.MB_ERR_NOT_READY


@pytest.mark.parametrize("kw,status", [
    (dict(D=96), UNSUPPORTED), (dict(H=129, Hkv=1, ldq=129 * 128, ldo=129 * 128), UNSUPPORTED),
    (dict(H=5), INVALID), (dict(H=0), INVALID), (dict(Hkv=0), INVALID), (dict(tq=-1), INVALID),
    (dict(tk=1 << 30), INVALID), (dict(n=-1), INVALID), (dict(scale=-1.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(cu_q=None), INVALID),
    (dict(cu_k=None), INVALID), (dict(q=None), INVALID), (dict(q=P + 8), INVALID), (dict(ldq=511), INVALID),
    (dict(ldq=516), INVALID), (dict(ldk=128), INVALID), (dict(v=P + 2), INVALID), (dict(out=None), INVALID),
    (dict(ldo=500), INVALID), (dict(k=None), INVALID),
])
def test_varlen_refuses(kw, status):
    assert varlen(**kw) == status, mb.lib().mb_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(cache=None), INVALID), (dict(cache=cache(dtype=3)), UNSUPPORTED), (dict(cache=cache(head_dim=80)), UNSUPPORTED),
    (dict(cache=cache(page_size=24)), INVALID), (dict(cache=cache(page_size=8)), INVALID),
    (dict(cache=cache(page_size=512)), INVALID), (dict(cache=cache(n_pages=0)), INVALID),
    (dict(cache=cache(n_pages=1 << 31)), INVALID), (dict(cache=cache(n_kv_heads=0)), INVALID),
    (dict(cache=cache(k=None)), INVALID), (dict(cache=cache(v=P + 8)), INVALID),
    (dict(cache=cache(dtype=_lib.KV_I8)), INVALID),
    (dict(cache=cache(dtype=_lib.KV_E4M3, k_scale=P + 4, v_scale=P)), INVALID),
    (dict(n=-1), INVALID), (dict(width=-1), INVALID), (dict(ldt=7), INVALID), (dict(table=None), INVALID),
])
def test_cache_and_table_refused_by_all(kw, status):
    for call in (paged, write, read):
        assert call(**kw) == status, (call.__name__, mb.lib().mb_last_error())


@pytest.mark.parametrize("call,kw", [
    (paged, dict(H=5)), (paged, dict(H=0)), (paged, dict(scale=-0.5)), (paged, dict(lens=None)), (paged, dict(q=P + 4)),
    (paged, dict(ldq=256)), (paged, dict(ldo=513)), (paged, dict(out=None)),
    (write, dict(tokens=3)), (write, dict(tokens=-1)), (write, dict(lens=None)), (write, dict(k=P + 8)),
    (write, dict(ldv=128)), (write, dict(ldk=260)), (write, dict(v=None)),
    (read, dict(tokens=-1)), (read, dict(cu=None)), (read, dict(k=None)), (read, dict(ldk=250)), (read, dict(v=P + 8)),
])
def test_own_arguments_refused(call, kw):
    assert call(**kw) == INVALID, mb.lib().mb_last_error()


def test_nothing_to_do_succeeds_and_the_rest_needs_init():
    """Empty calls need no device; a whole call on a machine without one, or before mb_init, says so."""
    assert varlen(tq=0) == varlen(n=0) == paged(n=0) == write(tokens=0, n=0) == read(tokens=0) == _lib.MB_OK
    if not torch.cuda.is_available():
        assert varlen() == paged() == write() == read() == NOT_READY


def test_workspace_size():
    n = ctypes.c_size_t(0)
    f = mb.lib().mb_attention_paged_workspace
    assert f(4, 8, 2, 128, ctypes.byref(n)) == _lib.MB_OK and 0 < n.value < 1 << 28
    small = n.value
    assert f(4096, 8, 2, 128, ctypes.byref(n)) == _lib.MB_OK and n.value > small
    assert f(4, 8, 3, 128, ctypes.byref(n)) == INVALID and f(4, 8, 2, 100, ctypes.byref(n)) == UNSUPPORTED
    assert f(4, 8, 2, 128, None) == INVALID


def test_python_front_refuses_cpu_tensors_and_types():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        mb.attention_varlen(q, q, q, cu)
    with pytest.raises(TypeError, match="dtype"):
        mb.KVCache.from_tensors(q[None].half(), q[None].half())
    with pytest.raises(ValueError, match="scale"):
        mb.KVCache.from_tensors(q[None].to(torch.int8), q[None].to(torch.int8))
    with pytest.raises(ValueError, match="scale"):
        mb.KVCache.from_tensors(q[None], q[None], torch.zeros(1, 4, 2), torch.zeros(1, 4, 2))


def test_crate_cache_struct_matches_the_header():
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mold_b200.h")).read(), flags=re.S)
    ffi = open(os.path.join(ROOT, "crates", "mold-b200", "src", "ffi.rs")).read()
    c = re.findall(r"(\w+);", re.search(r"typedef struct \{([^{}]*?)\}\s*mb_kv_cache;", hdr, flags=re.S).group(1))
    rs = re.findall(r"pub (\w+):", re.search(r"pub struct MbKvCache \{(.*?)\n\}", ffi, flags=re.S).group(1))
    assert c == rs == [f[0] for f in _lib.KVCacheC._fields_]
