"""Torch-tensor front of the single-kernel C-ABI entry points.

Each function takes CUDA tensors, checks dtypes/contiguity, and passes raw
pointers plus the current torch stream to libmold_b200.so.
"""
import ctypes

import numpy as np
import torch

from ._lib import (STEP_CALLBACK, InpaintC, KVCacheC, KV_BF16, KV_E4M3, KV_I8, DT_BF16, DT_F32, EPI_GATE_RESIDUAL, EPI_GELU_TANH, EPI_NONE, GGML_BF16, GGML_F16, GGML_F32,
                   GGML_Q4_0, GGML_Q4_1, GGML_Q4_K, GGML_Q5_0, GGML_Q5_1, GGML_Q5_K, GGML_Q6_K, GGML_Q8_0, check, lib)

# (values, bytes) per GGUF block
_BLOCK = {GGML_F32: (1, 4), GGML_F16: (1, 2), GGML_BF16: (1, 2), GGML_Q8_0: (32, 34), GGML_Q4_K: (256, 144),
          GGML_Q4_0: (32, 18), GGML_Q4_1: (32, 20), GGML_Q5_0: (32, 22), GGML_Q5_1: (32, 24), GGML_Q5_K: (256, 176),
          GGML_Q6_K: (256, 210)}
_inited = set()


def init(device=0):
    """mb_init for `device` (idempotent); also makes it torch's current device."""
    torch.cuda.set_device(device)
    if device not in _inited:
        check(lib().mb_init(device))
        _inited.add(device)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _dt(t):
    if t.dtype == torch.float32:
        return DT_F32
    if t.dtype == torch.bfloat16:
        return DT_BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def row_bytes(ggml_type, n_cols):
    be, bb = _BLOCK[ggml_type]
    if n_cols % be:
        raise ValueError(f"n_cols {n_cols} not a multiple of block {be}")
    return n_cols // be * bb


class QTensor:
    """A GGUF tensor held as raw GGML bytes: rows = output features, blocks along cols
    (candle's QTensor)."""

    def __init__(self, ggml_type, shape, raw):
        self.ggml_type = int(ggml_type)
        self.shape = tuple(int(s) for s in shape)
        raw = np.ascontiguousarray(raw, dtype=np.uint8).reshape(-1)
        n_rows = int(np.prod(self.shape[:-1])) if len(self.shape) > 1 else 1
        if raw.size != n_rows * row_bytes(self.ggml_type, self.shape[-1]):
            raise ValueError("raw byte count does not match shape/type")
        self.raw = raw

    @property
    def n_rows(self):
        return int(np.prod(self.shape[:-1])) if len(self.shape) > 1 else 1

    @property
    def n_cols(self):
        return self.shape[-1]


class QMatMul:
    """Device copy of a quantized weight; forward(x) = x W^T (candle QMatMul)."""

    def __init__(self, handle, n_rows, n_cols, ggml_type, device):
        self._h = handle
        self.n_rows, self.n_cols, self.ggml_type, self.device = n_rows, n_cols, ggml_type, device

    @classmethod
    def from_weights(cls, qt: QTensor, device=0):
        init(device)
        h = ctypes.c_void_p()
        check(lib().mb_weight_create(qt.ggml_type, qt.n_rows, qt.n_cols, qt.raw.ctypes.data_as(ctypes.c_void_p),
                                     qt.raw.size, 0, ctypes.byref(h)))
        return cls(h, qt.n_rows, qt.n_cols, qt.ggml_type, device)

    @classmethod
    def from_device_bytes(cls, raw, ggml_type, n_rows, n_cols, device=0):
        """A weight from GGUF bytes already in device memory (a uint8 CUDA tensor, GGUF layout);
        the library takes its own copy."""
        init(device)
        h = ctypes.c_void_p()
        check(lib().mb_weight_create(int(ggml_type), n_rows, n_cols, ctypes.c_void_p(raw.data_ptr()), raw.numel(), 1,
                                     ctypes.byref(h)))
        return cls(h, n_rows, n_cols, int(ggml_type), device)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value and lib is not None:
            try:
                lib().mb_weight_destroy(h)
            except Exception:
                pass
            self._h = None

    @property
    def handle(self):
        return self._h

    def forward(self, x, bias=None, epilogue=EPI_NONE, gelu_from=0, gate=None, residual=None, out=None,
                out_dtype=None):
        """x [..., K] (bf16 or f32, CUDA) -> [..., N]. Epilogues as mb_qlinear."""
        return qlinear(self, x, bias=bias, epilogue=epilogue, gelu_from=gelu_from, gate=gate, residual=residual,
                       out=out, out_dtype=out_dtype)

    __call__ = forward

    def download(self):
        """The weight's bytes in GGUF layout (host uint8 [n_rows * row bytes])."""
        out = np.empty(self.n_rows * row_bytes(self.ggml_type, self.n_cols), dtype=np.uint8)
        check(lib().mb_weight_download(self._h, out.ctypes.data_as(ctypes.c_void_p), out.size))
        return out

    def lora_merge(self, A, B, scale, row_offset=0):
        """In place: rows [row_offset, row_offset + B.shape[0]) += scale * (B @ A), re-quantized to
        the weight's own type (mb_weight_lora_merge). A [rank, n_cols], B [rows, rank] (CUDA)."""
        A, B = _lora_operands(A, B)
        check(lib().mb_weight_lora_merge(self._h, int(row_offset), B.shape[0], _ptr(A), _ptr(B), A.shape[0],
                                         float(scale), _stream()))


def _lora_operands(A, B):
    A = A.contiguous().float()
    B = B.contiguous().float()
    if A.dim() != 2 or B.dim() != 2 or B.shape[1] != A.shape[0]:
        raise ValueError(f"LoRA shapes A {tuple(A.shape)} and B {tuple(B.shape)} do not chain")
    if not (A.is_cuda and B.is_cuda):
        raise ValueError("LoRA A and B must be CUDA tensors")
    return A, B


def qlinear(w: QMatMul, x, bias=None, epilogue=EPI_NONE, gelu_from=0, gate=None, residual=None, out=None,
            out_dtype=None):
    K, N = w.n_cols, w.n_rows
    if x.shape[-1] != K:
        raise ValueError(f"x has K={x.shape[-1]}, weight expects {K}")
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    if epilogue == EPI_GATE_RESIDUAL:
        out_dtype = torch.float32
    if out is None:
        out_dtype = out_dtype or x.dtype
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    y2 = out.reshape(-1, out.shape[-1])
    res = residual.reshape(-1, residual.shape[-1]) if residual is not None else None
    check(lib().mb_qlinear(w.handle, _ptr(x2), _dt(x2), M, x2.stride(0), _ptr(y2), _dt(y2), y2.stride(0),
                           _ptr(bias), epilogue, gelu_from, _ptr(gate), _ptr(res), res.stride(0) if res is not None else 0,
                           _stream()))
    return out.reshape(*x.shape[:-1], N) if out.dim() == 2 and x.dim() != 2 else out


def dequantize(w: QMatMul, dtype=torch.float32):
    out = torch.empty((w.n_rows, w.n_cols), dtype=dtype, device=f"cuda:{w.device}")
    check(lib().mb_dequant(w.handle, _ptr(out), _dt(out), _stream()))
    return out


def qgemv(w: QMatMul, x, apply_silu=False, bias=None):
    y = torch.empty(w.n_rows, dtype=torch.float32, device=x.device)
    check(lib().mb_qgemv(w.handle, _ptr(x.contiguous()), int(apply_silu), _ptr(bias), _ptr(y), _stream()))
    return y


def ln_modulate(x, shift, scale):
    M, C = x.shape
    y = torch.empty((M, C), dtype=torch.bfloat16, device=x.device)
    check(lib().mb_ln_modulate(_ptr(x), M, C, x.stride(0), _ptr(shift), _ptr(scale), _ptr(y), y.stride(0), _stream()))
    return y


def rope_table(ids, axes_dim=(16, 56, 56), theta=10000):
    L, n_axes = ids.shape
    pe = torch.empty((L, sum(axes_dim) // 2, 2, 2), dtype=torch.float32, device=ids.device)
    ax = (ctypes.c_int * len(axes_dim))(*axes_dim)
    check(lib().mb_rope_table(_ptr(ids.contiguous()), L, n_axes, ax, theta, _ptr(pe), _stream()))
    return pe


def qk_norm_rope(qkv, H, q_scale, k_scale, pe, row_offset=0, L_total=None, q=None, k=None, v=None, kv_pos=None):
    """kv_pos (int32 [L_total], optional): k / v of sequence row r go to row kv_pos[r]."""
    M = qkv.shape[0]
    L_total = L_total or M
    if q is None:
        q = torch.empty((H, L_total, 128), dtype=torch.bfloat16, device=qkv.device)
        k = torch.empty_like(q)
        v = torch.empty_like(q)
    if kv_pos is None:
        check(lib().mb_qk_norm_rope(_ptr(qkv), M, qkv.stride(0), H, _ptr(q_scale), _ptr(k_scale), _ptr(pe),
                                    row_offset, L_total, _ptr(q), _ptr(k), _ptr(v), _stream()))
    else:
        assert kv_pos.dtype == torch.int32 and kv_pos.numel() >= L_total
        check(lib().mb_qk_norm_rope_ex(_ptr(qkv), M, qkv.stride(0), H, _ptr(q_scale), _ptr(k_scale), _ptr(pe),
                                       row_offset, L_total, _ptr(q), _ptr(k), _ptr(v), _ptr(kv_pos), _stream()))
    return q, k, v


def key_order(txt_mask, l_img):
    """Key order for a masked joint sequence cat[txt, img]: kept text keys, image keys, masked
    text keys. Returns (kv_pos int32 [L], n_valid_keys) for qk_norm_rope / attention."""
    m = torch.as_tensor(txt_mask).to("cpu", torch.bool).reshape(-1)
    lt = m.numel()
    nv = int(m.sum())
    pos = torch.empty(lt + l_img, dtype=torch.int32)
    pos[:lt][m] = torch.arange(nv, dtype=torch.int32)
    pos[:lt][~m] = torch.arange(lt - nv, dtype=torch.int32) + nv + l_img
    pos[lt:] = torch.arange(l_img, dtype=torch.int32) + nv
    return pos, nv + l_img


def attention(q, k, v, n_valid_keys=None, out=None, split_row=None, out2=None):
    """q [H, Lq, 128], k/v [H, Lk, 128] bf16 -> out [Lq, H*128] bf16. With split_row, rows
    [split_row, Lq) go to out2 (same row stride) instead."""
    H, Lq, D = q.shape
    Lk = k.shape[1]
    if out is None:
        out = torch.empty((Lq if split_row is None else split_row, H * D), dtype=torch.bfloat16, device=q.device)
    if split_row is None:
        check(lib().mb_attention(_ptr(q), _ptr(k), _ptr(v), H, Lq, Lk, n_valid_keys or Lk, _ptr(out),
                                 out.stride(0), _stream()))
        return out
    if out2 is None:
        out2 = torch.empty((Lq - split_row, H * D), dtype=torch.bfloat16, device=q.device)
    assert out2.stride(0) == out.stride(0)
    check(lib().mb_attention_ex(_ptr(q), _ptr(k), _ptr(v), H, Lq, Lk, n_valid_keys or Lk, _ptr(out), out.stride(0),
                                split_row, _ptr(out2), _stream()))
    return out, out2


def rms_norm(x, w, eps=1e-6):
    """DynamicRmsNorm: x f32 [M, C] -> bf16 x / sqrt(mean(x^2) + eps) * w."""
    M, C = x.shape
    y = torch.empty((M, C), dtype=torch.bfloat16, device=x.device)
    check(lib().mb_rms_norm(_ptr(x), M, C, x.stride(0), _ptr(w), float(eps), _ptr(y), y.stride(0), _stream()))
    return y


def cfg_euler_step(img, cond, uncond, guidance, dt, channels=16, pp=4):
    """img += CFG(cond, uncond) * dt on packed latents [n_tok, channels * pp] (f32, in place)."""
    n_tok = img.shape[0]
    check(lib().mb_cfg_euler_step(_ptr(img), _ptr(cond), _ptr(uncond), n_tok, channels, pp, float(guidance),
                                  float(dt), _stream()))
    return img


def euler_step(img, pred, dt):
    check(lib().mb_euler_step(_ptr(img), _ptr(pred), img.numel(), float(dt), _stream()))
    return img


def device_status():
    s = ctypes.c_int(0)
    check(lib().mb_device_status(ctypes.byref(s)))
    return s.value


def gguf_inspect(path):
    """[(name, ggml_type, shape outermost-first)] of a GGUF file's tensors (no GPU needed)."""
    buf = ctypes.create_string_buffer(1 << 22)
    n = ctypes.c_int64(0)
    check(lib().mb_gguf_inspect(str(path).encode(), buf, len(buf), ctypes.byref(n)))
    out = []
    for line in buf.value.decode().split("\n"):
        if line:
            f = line.split("\t")
            out.append((f[0], int(f[1]), tuple(int(x) for x in f[2:])))
    return out


# ---------------------------------------------------------------- text transformers
# A generation step makes hundreds of these calls, so the checks are kept to a few attribute reads each.

def _ready(first, *others):
    """The one device of the tensors (None ones aside), initialised, as an index."""
    dev = first.get_device()  # -1 on the CPU
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on different devices ({first.device} and {t.device})")
    if dev not in _inited:
        if dev < 0:
            raise ValueError("tensors must be CUDA tensors")
        with torch.cuda.device(dev):
            check(lib().mb_init(dev))
        _inited.add(dev)
    return dev


def _launch(dev, fn, *args):
    """fn(*args, stream) on device `dev` and its current stream, whichever device is current."""
    st = torch._C._cuda_getCurrentRawStream(dev)
    if dev == torch._C._cuda_getDevice():
        status = fn(*args, st)
    else:
        with torch.cuda.device(dev):
            status = fn(*args, st)
    if status:
        check(status)


def _heads(x, name, copy=True):
    """(x, address, row stride, rows, heads, head size) of a bf16 [rows, heads, D] tensor whose rows are whole and
    16-byte aligned; a tensor laid out otherwise is copied, or with copy=False refused."""
    if x.dtype is not torch.bfloat16 or x.dim() != 3:
        raise ValueError(f"{name} must be bf16 [rows, heads, head_dim], got {x.dtype} {tuple(x.shape)}")
    rows, h, d = x.shape
    ptr = x.data_ptr()
    if ptr & 15 == 0:
        if x.is_contiguous():
            return x, ptr, h * d, rows, h, d
        s0, s1, s2 = x.stride()
        if s2 == 1 and (h == 1 or s1 == d) and (rows <= 1 or (s0 >= h * d and s0 & 7 == 0)):
            return x, ptr, (s0 if rows > 1 else h * d), rows, h, d
    if not copy:
        raise ValueError(f"{name} must have whole rows, 16-byte aligned (strides {x.stride()})")
    x = x.clone(memory_format=torch.contiguous_format)
    return x, x.data_ptr(), h * d, rows, h, d


def _ints(x, name, n=None):
    """(x's address, entries) of an int32 vector, of n entries where n is given."""
    if x.dtype is not torch.int32 or x.dim() != 1 or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector, got {x.dtype} {tuple(x.shape)}")
    m = x.shape[0]
    if n is not None and m != n:
        raise ValueError(f"{name} has {m} entries, expected {n}")
    return x.data_ptr(), m


def _table(table, n_seqs):
    """(table, address, row stride, pages a row) of an int32 page table of n_seqs rows."""
    if table.dtype is not torch.int32 or table.dim() != 2:
        raise ValueError(f"table must be int32 [sequences, pages], got {table.dtype} {tuple(table.shape)}")
    n, width = table.shape
    if n != n_seqs:
        raise ValueError(f"table has {n} rows for {n_seqs} sequences")
    ld = width
    if not table.is_contiguous():
        ld, s1 = table.stride()
        if n <= 1 or (width > 1 and s1 != 1) or ld < width:
            table, ld = table.contiguous(), width
    return table, table.data_ptr(), ld, width


def _scale(scale):
    if scale is None:
        return 0.0
    if not scale > 0:
        raise ValueError(f"scale must be positive, got {scale}")
    return max(float(scale), 2.0 ** -126)  # a smaller one may be 0 in 32 bits, which stands for the default


def attention_varlen(q, k, v, cu_q, cu_k=None, causal=True, scale=None, out=None):
    """Attention of packed prompts with grouped heads: q [Tq, H, D], k / v [Tk, H_kv, D] bf16 -> out [Tq, H, D].
    Sequence b has query rows [cu_q[b], cu_q[b+1]) and key rows [cu_k[b], cu_k[b+1]) (int32, on the device; cu_k
    defaults to cu_q); with `causal` its queries are its last positions. A row without keys is 0; rows of out behind
    the last sequence are not written."""
    cu_k = cu_q if cu_k is None else cu_k
    dev = _ready(q, k, v, cu_q, cu_k, out)
    q, q_ptr, ldq, tq, h, d = _heads(q, "q")
    k, k_ptr, ldk, tk, hk, dk = _heads(k, "k")
    v, v_ptr, ldv, tv, hv, dv = _heads(v, "v")
    if tk != tv or hk != hv or dk != d or dv != d:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    cq_ptr, n = _ints(cu_q, "cu_q")
    ck_ptr, _ = _ints(cu_k, "cu_k", n)
    if n < 1:
        raise ValueError("cu_q must have one entry more than there are sequences")
    out, o_ptr, ldo = _out(out, q)
    _launch(dev, lib().mb_attention_varlen, q_ptr, ldq, k_ptr, ldk, v_ptr, ldv, tq, tk, h, hk, d, cq_ptr, ck_ptr, n - 1,
            1 if causal else 0, _scale(scale), o_ptr, ldo)
    return out


def _out(out, q):
    """(out, address, row stride): the caller's tensor, or a new one, shaped like q."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        return out, out.data_ptr(), q.shape[1] * q.shape[2]
    if out.shape != q.shape:
        raise ValueError(f"out is {tuple(out.shape)}, q {tuple(q.shape)}")
    return _heads(out, "out", copy=False)[:3]


_KV_TYPES = {torch.bfloat16: KV_BF16, torch.int8: KV_I8, torch.float8_e4m3fn: KV_E4M3}


class KVCache:
    """Paged key-value cache of one attention layer: k, v [n_pages, n_kv_heads, page_size, head_dim] in bf16, or in
    int8 / float8_e4m3fn codes with an f32 scale a row (k_scale, v_scale [n_pages, n_kv_heads, page_size]).

    A sequence's position p is at offset p % page_size of page table[b, p // page_size]; the caller hands out pages.
    page_size is a power of two from 16 to 256, head_dim 64 or 128."""

    def __init__(self, n_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device=None):
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        scales = [None, None] if dtype == torch.bfloat16 else [torch.zeros(shape[:3], device=device) for _ in range(2)]
        self._hold(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   *scales)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None):
        """A cache over tensors that the caller has; they are used in place. Scales that this library did not write may be
        any finite numbers."""
        self = cls.__new__(cls)
        self._hold(k, v, k_scale, v_scale)
        return self

    def _hold(self, k, v, k_scale, v_scale):
        if k.dtype not in _KV_TYPES:
            raise TypeError(f"unsupported cache dtype {k.dtype}")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must both be [pages, heads, page, head_dim]")
        if (k.dtype == torch.bfloat16) != (k_scale is None) or (k_scale is None) != (v_scale is None):
            raise ValueError("an 8-bit cache has k_scale and v_scale, a bf16 cache has none")
        for s in (k_scale, v_scale):
            if s is not None and (s.dtype != torch.float32 or s.shape != k.shape[:3]):
                raise ValueError(f"scales must be float32 {tuple(k.shape[:3])}")
        self._tensors = [t for t in (k, v, k_scale, v_scale) if t is not None]
        if not all(t.is_contiguous() for t in self._tensors):
            raise ValueError("cache tensors must be contiguous")
        self.device_index = _ready(*self._tensors)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self._c = KVCacheC(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if k_scale is not None else None,
                           v_scale.data_ptr() if v_scale is not None else None, self.n_pages, self.page_size,
                           self.n_kv_heads, self.head_dim, _KV_TYPES[k.dtype])
        self._ref = ctypes.byref(self._c)
        self._workspaces = {}

    def _workspace_bytes(self, n_seqs, heads):
        """mb_attention_paged_workspace for n_seqs sequences of `heads` query heads (a function of these sizes)."""
        got = self._workspaces.get((n_seqs, heads))
        if got is None:
            nbytes = ctypes.c_size_t(0)
            with torch.cuda.device(self.device_index):
                check(lib().mb_attention_paged_workspace(n_seqs, heads, self.n_kv_heads, self.head_dim,
                                                         ctypes.byref(nbytes)))
            got = self._workspaces[n_seqs, heads] = nbytes.value
        return got

    def _rows(self, x, name, copy=True):
        x, ptr, ld, rows, h, d = _heads(x, name, copy)
        if h != self.n_kv_heads or d != self.head_dim:
            raise ValueError(f"{name} is {tuple(x.shape)}, the cache has {self.n_kv_heads} heads of {self.head_dim}")
        return x, ptr, ld, rows

    def write(self, k, v, table, kv_lens, cu=None):
        """Append rows k, v (bf16 [T, n_kv_heads, head_dim]): sequence b's rows [cu[b], cu[b+1]) become its last
        positions, kv_lens[b] (int32, the length after the call) at their end. Without cu, row b is sequence b's one
        new position. Rows that would come before position 0 are passed over (kv_lens[b] <= 0 in a padded batch)."""
        dev = _ready(self.k, k, v, table, kv_lens, cu)
        k, k_ptr, ldk, rows = self._rows(k, "k")
        v, v_ptr, ldv, v_rows = self._rows(v, "v")
        if rows != v_rows:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        lens_ptr, n = _ints(kv_lens, "kv_lens")
        cu_ptr = None if cu is None else _ints(cu, "cu", n + 1)[0]
        table, t_ptr, ldt, width = _table(table, n)
        _launch(dev, lib().mb_kv_write, self._ref, k_ptr, ldk, v_ptr, ldv, rows, cu_ptr, lens_ptr, t_ptr, ldt, width, n)

    def read(self, table, cu, n_tokens=None, k=None, v=None):
        """The first cu[b+1] - cu[b] positions of each sequence, packed: k, v bf16 [n_tokens, n_kv_heads, head_dim].
        n_tokens (default: cu's last entry, which waits for the device) or k and v give the size; rows behind the last
        sequence are not written."""
        dev = _ready(self.k, table, cu, k, v)
        cu_ptr, n = _ints(cu, "cu")
        n -= 1
        if n < 0:
            raise ValueError("cu must have one entry more than there are sequences")
        if (k is None) != (v is None):
            raise ValueError("give both k and v or neither")
        if k is None:
            rows = int(cu[-1]) if n_tokens is None else int(n_tokens)
            k = torch.empty((rows, self.n_kv_heads, self.head_dim), dtype=torch.bfloat16, device=self.k.device)
            v = torch.empty_like(k)
            k_ptr, v_ptr, ldk = k.data_ptr(), v.data_ptr(), self.n_kv_heads * self.head_dim
            ldv = ldk
        else:
            k, k_ptr, ldk, rows = self._rows(k, "k", copy=False)
            v, v_ptr, ldv, v_rows = self._rows(v, "v", copy=False)
            if rows != v_rows or (n_tokens is not None and n_tokens != rows):
                raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} and n_tokens {n_tokens} do not fit")
        table, t_ptr, ldt, width = _table(table, n)
        _launch(dev, lib().mb_kv_read, self._ref, cu_ptr, t_ptr, ldt, width, n, rows, k_ptr, ldk, v_ptr, ldv)
        return k, v


def attention_paged(q, cache: KVCache, table, kv_lens, scale=None, out=None):
    """Attention of one new token of each sequence over its cached positions 0 .. kv_lens[b] - 1: q [B, H, D] bf16 ->
    out [B, H, D]; a sequence without positions gives 0. Equal calls give equal bits."""
    dev = _ready(cache.k, q, table, kv_lens, out)
    q, q_ptr, ldq, n, h, d = _heads(q, "q")
    if d != cache.head_dim:
        raise ValueError(f"q has head_dim {d}, the cache {cache.head_dim}")
    lens_ptr, _ = _ints(kv_lens, "kv_lens", n)
    table, t_ptr, ldt, width = _table(table, n)
    out, o_ptr, ldo = _out(out, q)
    nbytes = cache._workspace_bytes(n, h)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)  # of this call alone: the stream's, or the graph's
    _launch(dev, lib().mb_attention_paged, q_ptr, ldq, cache._ref, lens_ptr, t_ptr, ldt, width, n, h, _scale(scale),
            o_ptr, ldo, ws.data_ptr(), nbytes)
    return out


def denoise_extras(inpaint, on_step):
    """ctypes arguments of the *_denoise_ex calls: (pointer to an mb_inpaint or None, callback,
    objects to keep alive while the steps run). inpaint = (mask, original, noise), f32 CUDA
    tensors shaped like the packed latent (1 = repaint, 0 = preserve); on_step(step, total) is
    called from a CUDA host-function thread once each step has finished on the device (keep it
    short, and synchronise the stream before relying on every call having happened)."""
    keep = []
    ip = None
    if inpaint is not None:
        ts = [a.contiguous().float() for a in inpaint]
        keep += ts
        ip = InpaintC(*[ctypes.c_void_p(a.data_ptr()) for a in ts])
        keep.append(ip)
    cb = STEP_CALLBACK(lambda user, step, total: on_step(step, total)) if on_step is not None else STEP_CALLBACK()
    keep.append(cb)
    return (ctypes.byref(ip) if ip is not None else None), cb, keep
