"""Plain 64-bit restatements of the text-transformer operators, for the tests."""
import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def offsets(lengths, device="cuda"):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def attention64(q, k, v, keep, scale=None, half_weights=False):
    """q [m, H, D], k / v [n, H_kv, D], keep [m, n] (bool) -> (out, tolerance), both f64 [m, H, D].

    Tolerance of the kernels' result against out, element by element, with A = sum_j w_j |v_j|:
      2^-8 |out|        the output's rounding to bf16
      2^-8 A            each weight's rounding to bf16 before the product with v
      2 d A, d = D 2^-23 max_j scale sum |q k_j|   the f32 accumulation of the scores (D additions, each off by at most
                        one step, in numerator and denominator)
      n 2^-36 max |v|   with half_weights (8-bit caches): the weights are f16 numbers, 2^11 standing for a weight of 1
                        on the row with the largest value scale. Below f16's 2^-14 they are off by up to half its last
                        step, 2^-25, which is 2^-36 of that row's largest value; the n weights' sum is at least 1, the
                        weight of the reference score. Above, 2^-11 of the weight is within the 2^-8 A, and so are the
                        query's digits: off by 2^-17 max |q| a channel, times sum |k| scale, far below 2^-9
      2^-11 A           exponentials (polynomial 7.5e-5 = 2^-13.7, MUFU 2^-22) in numerator and denominator, f32 sums
    """
    m, H, D = q.shape
    n, G = k.shape[0], H // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if n == 0 or m == 0:
        z = torch.zeros((m, H, D), dtype=torch.float64, device=q.device)
        return z, z.clone()
    q, k, v = q.double().transpose(0, 1), k.double().transpose(0, 1), v.double().transpose(0, 1)
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    s = q @ k.transpose(1, 2) * scale
    off = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~keep, 0.0).amax(-1, keepdim=True) * D * 2.0 ** -23
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    out, a = w @ v, w @ v.abs()
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -11 + 2 * off) * a
    if half_weights:
        tol = tol + n * 2.0 ** -36 * v.abs().amax()
    return out.transpose(0, 1), tol.transpose(0, 1)


def varlen64(q, k, v, ms, ns, causal, scale=None):
    outs, tols, a, c = [], [], 0, 0
    for m, n in zip(ms, ns):
        i = torch.arange(m, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        keep = (j <= i + n - m) if causal else torch.ones((m, n), dtype=torch.bool, device=q.device)
        o, t = attention64(q[a:a + m], k[c:c + n], v[c:c + n], keep, scale)
        outs.append(o)
        tols.append(t)
        a, c = a + m, c + n
    return torch.cat(outs), torch.cat(tols)


def e4m3_values():
    """The 256 codes' numbers, from the format's definition (NaN at 0x7f and 0xff)."""
    out = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        x = math.nan if c & 127 == 127 else (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        out.append(-x if c & 128 else x)
    return torch.tensor(out, dtype=torch.float64)


def encode(x, dtype):
    """(codes as f64 numbers, scales f32) of bf16 rows x [..., D]: scale, inverse and product are f32 by definition, the
    nearest code is searched among all of them (ties to the even code)."""
    f = x.float()
    top = f.abs().amax(-1, keepdim=True).cpu()
    t = torch.tensor(TOP[dtype], dtype=torch.float32)
    ok = top >= 2.0 ** -100
    inv = torch.where(ok, t / torch.where(ok, top, torch.ones_like(top)), torch.zeros_like(top))
    y = (f.cpu() * inv).double()
    if dtype == torch.int8:
        c = torch.round(y).clamp(-127, 127)  # ties to even
    else:
        grid = e4m3_values()[:127]  # 0 .. 448, ascending
        a = y.abs().clamp(max=448.0)
        hi = torch.searchsorted(grid, a.contiguous()).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        dl, dh = a - grid[lo], grid[hi] - a
        pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        c = grid[pick] * torch.where(y < 0, -1.0, 1.0)
    s = torch.where(ok, top / t, torch.zeros_like(top))
    return c, s[..., 0]


class Pages:
    """Page tables over a pool of n_pages, handed out in a shuffled order; entries behind a sequence's pages are -1."""

    def __init__(self, lengths, page, extra=3, width=None, seed=0, device="cuda"):
        need = [-(-n // page) for n in lengths]
        self.n_pages = sum(need) + extra
        order = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(need + [1]) if width is None else width
        t = torch.full((len(lengths), width), -1, dtype=torch.int32)
        for b, m in enumerate(need):
            t[b, :m] = torch.tensor([order.pop() for _ in range(m)], dtype=torch.int32)
        self.host, self.page = t, page
        self.table = t.to(device)

    def rows(self, b, n):
        """(page, offset) of positions 0 .. n - 1 of sequence b, as index tensors on the device."""
        p = torch.arange(n)
        return self.host[b][p // self.page].long().cuda(), (p % self.page).cuda()


def cached64(cache, pages, b, n):
    """Sequence b's first n cached rows of k and v as f64 [n, H_kv, D]."""
    page, at = pages.rows(b, n)
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if x.dtype == torch.bfloat16:
            out.append(x[page, :, at].double())
        else:
            c = x.view(torch.uint8)[page, :, at].view(torch.uint8).long()
            t = e4m3_values().cuda() if x.dtype == torch.float8_e4m3fn else (
                torch.arange(256, device="cuda") + 128).remainder(256).double() - 128
            out.append(t[c] * s[page, :, at].double()[..., None])
    return out
