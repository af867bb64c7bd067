// K12 / K13: the paged key-value cache of a text transformer, written (bf16, or 8-bit codes with
// one f32 scale for each row of head_dim values) and read back.
//
// A group of head_dim / 16 threads owns a (token, head) row of k and the same row of v, two times 16 bytes
// of bf16 a thread; the groups of a warp work on neighbouring tokens and search for the sequence together,
// while the rows are on their way. 11k rows of 8 x 128 written and 25k read, int8: 39.6 us, 216 MB in and out or
// 5.5 TB/s. Of these some 135 MB pass HBM (3.5 TB/s), the codes and part of the output stay in L2: no single
// unit is full (issue slots 60 to 65 %, ALU pipe 53 to 58 %), and two short launches start and end. Instructions
// count, hence packed f32 arithmetic and no integer conversions or divisions (55 us with them). More rows a
// thread or larger blocks lose (2 rows: 41.2, 4: 48 us; a generation step 6.1 and 9.6 against 4.8 us), and so do accesses of 32
// bytes (40.4 against 39.9).
#include <string>

#include "attn_util.cuh"
#include "common.cuh"
#include "internal.h"
#include "kv_cache.cuh"

namespace mb {
namespace kv {

constexpr int kThreads = 128;
constexpr int kHalves = 2;  // 16-byte pieces of a bf16 row that a thread holds, half a row apart

// The sequence whose rows hold t: the last b with cu[b] <= t, its rows [c0, c1), and its entry of `per_seq` (NULL: 0). All
// lanes of the warp with the same t; 32 entries a step, and the last step's loads serve for all of it, since each load
// that waits for another costs as much as the row's own. Whatever cu holds, b is in [0, n).
struct Span {
  int b;
  int64_t c0, c1;
  int value;
};
MB_DEV Span seq_of(const int32_t* cu, const int32_t* per_seq, int n, int64_t t) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 32) {
    const int step = (n + 31) >> 5, at = lane * step;
    const unsigned le = __ballot_sync(0xffffffffu, at < n && cu[lo + (at < n ? at : 0)] <= t);
    const int k = max(__popc(le), 1) - 1;  // le is a run of ones from bit 0
    lo += k * step;
    n = min(step, n - k * step);
  }
  const int edge = lane <= n ? cu[lo + lane] : 0;
  const int value = per_seq && lane < n ? per_seq[lo + lane] : 0;
  const int k = max(__popc(__ballot_sync(0xffffffffu, lane < n && edge <= t)), 1) - 1;
  Span s;
  s.b = lo + k;
  s.c0 = __shfl_sync(0xffffffffu, edge, k);
  s.c1 = __shfl_sync(0xffffffffu, edge, (k + 1) & 31);
  if (k == 31) s.c1 = cu[lo + 32];
  s.value = __shfl_sync(0xffffffffu, value, k);
  return s;
}

using attn::add2;
using attn::pk2;
using attn::up2;
MB_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
MB_DEV uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A block works on one head, its groups on neighbouring tokens: their rows and scales lie side by side in the cache, and
// neighbouring blocks read the other heads of the same tokens. Token of the warp's first group:
template <int SIDE>
MB_DEV int64_t first_token(int heads, int& h) {
  const uint32_t chunk = blockIdx.x / (uint32_t)heads;
  h = (int)(blockIdx.x - chunk * heads);
  return ((int64_t)chunk * (kThreads / 32) + (threadIdx.x >> 5)) * SIDE;
}
// On to the sequence that holds t, at or behind the present one.
MB_DEV void advance(Span& s, const int32_t* cu, const int32_t* per_seq, int n, int64_t t) {
  while (t >= s.c1 && s.b + 1 < n) {
    s.b++, s.c0 = s.c1, s.c1 = cu[s.b + 1];
    if (per_seq) s.value = per_seq[s.b];
  }
}

struct WriteParams {
  Cache c;
  const __nv_bfloat16 *k, *v;
  int64_t ldk, ldv, n_tokens;
  const int32_t *cu, *lens, *table;
  int64_t ld_table;
  int table_width, n_seqs;
  int* status;
};

// fl(T / m) and fl(m / T) for a positive bf16 number m (bits `top` of the f32) from 2^-100 on. Both are scaled by powers
// of two from m in [1, 2), where one correction by the remainder (Markstein's) rounds the quotient correctly; the tests
// compare all 128 fractions with division.
template <int CODES>
MB_DEV void scales_of(uint32_t top, float& s, float& r) {
  constexpr float T = CODES == MB_KV_I8 ? 127.f : 448.f, IT = 1.f / T;
  const uint32_t e = (top & 0x7f800000u) - 0x3f800000u;  // exponent, to be added to an f32's bits
  const float f = __uint_as_float(top - e);
  float q = f * IT;
  q = fmaf(fmaf(-q, T, f), IT, q);
  s = __uint_as_float(__float_as_uint(q) + e);
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(f));
  float z = T * y;
  z = fmaf(fmaf(-z, f, T), y, z);
  r = __uint_as_float(__float_as_uint(z) - e);
}

// A row's values of this thread as codes, and the row's scale.
template <int CODES, int GROUP>
MB_DEV void encode_row(const uint4 (&x)[kHalves], uint2 (&out)[kHalves], float& scale) {
  // largest magnitude: the bit patterns of non-negative bf16 numbers order like the numbers, NaN last
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kHalves; i++) {
    top = max_u16x2(top, max_u16x2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu));
    top = max_u16x2(top, max_u16x2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
  }
#pragma unroll
  for (int o = GROUP / 2; o; o >>= 1) top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
  top = max(top << 16, top & 0xffff0000u);
  float r;
  scales_of<CODES>(top, scale, r);
  if (top - 0x0d800000u >= 0x7f800000u - 0x0d800000u) {  // below 2^-100, or not finite: then any code reads back as NaN
    r = 0.f;
    scale = top < 0x0d800000u ? 0.f : __uint_as_float(0x7fc00000u);
  }
  const uint64_t r2 = pk2(r, r);
#pragma unroll
  for (int i = 0; i < kHalves; i++) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      uint64_t a = mul2(pk2(bf16_lo(w[2 * j]), bf16_hi(w[2 * j])), r2);
      uint64_t b = mul2(pk2(bf16_lo(w[2 * j + 1]), bf16_hi(w[2 * j + 1])), r2);
      float y0, y1, y2, y3;
      if (CODES == MB_KV_I8) {
        // |y| <= 127 (1 + 2^-23); adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the
        // low byte (the conversion instruction runs at a quarter of the rate). Scalar additions: a packed one after the
        // packed product came out as one fused operation, without the product's rounding, and took ties the wrong way.
        up2(a, y0, y1), up2(b, y2, y3);
        const uint32_t v0 = __float_as_uint(__fadd_rn(y0, 12582912.f)), v1 = __float_as_uint(__fadd_rn(y1, 12582912.f));
        const uint32_t v2 = __float_as_uint(__fadd_rn(y2, 12582912.f)), v3 = __float_as_uint(__fadd_rn(y3, 12582912.f));
        o[j] = __byte_perm(__byte_perm(v0, v1, 0x0040), __byte_perm(v2, v3, 0x0040), 0x5410);
      } else {
        uint16_t lo, hi;
        up2(a, y0, y1), up2(b, y2, y3);
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y1), "f"(y0));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y3), "f"(y2));
        o[j] = (uint32_t)lo | ((uint32_t)hi << 16);
      }
    }
    out[i] = make_uint2(o[0], o[1]);
  }
}

template <int CODES, int D>
__global__ void __launch_bounds__(kThreads) k_kv_write(const WriteParams p) {
  wait_before();
  constexpr int GROUP = D / 16, SIDE = 32 / GROUP;
  const int lane = threadIdx.x % GROUP;
  int h;
  const int64_t t0 = first_token<SIDE>(p.c.heads, h), t = t0 + (threadIdx.x & 31) / GROUP;
  if (t0 >= p.n_tokens) return;
  const bool here = t < p.n_tokens;
  uint4 kx[kHalves], vx[kHalves];
#pragma unroll
  for (int j = 0; j < kHalves; j++) {
    kx[j] = vx[j] = make_uint4(0, 0, 0, 0);
    if (here) {
      kx[j] = ld_stream((const uint4*)(p.k + t * p.ldk + h * D) + j * GROUP + lane);
      vx[j] = ld_stream((const uint4*)(p.v + t * p.ldv + h * D) + j * GROUP + lane);
    }
  }
  int64_t dst = -1, pos = -1;
  Span seq = {(int)t, 0, 0, 0};
  if (p.cu) {
    seq = seq_of(p.cu, p.lens, p.n_seqs, t0);
    if (here) {
      advance(seq, p.cu, p.lens, p.n_seqs, t);
      if (t >= seq.c0 && t < seq.c1) pos = seq.value - (seq.c1 - t);
    }
  } else if (here) {
    pos = (int64_t)p.lens[seq.b] - 1;
  }
  if (pos >= 0) dst = row_of(p.c, p.table + (int64_t)seq.b * p.ld_table, p.table_width, pos, h, p.status);
  if (CODES == MB_KV_BF16) {
    if (dst >= 0)
#pragma unroll
      for (int j = 0; j < kHalves; j++) {
        ((uint4*)p.c.k)[dst * (D / 8) + j * GROUP + lane] = kx[j];
        ((uint4*)p.c.v)[dst * (D / 8) + j * GROUP + lane] = vx[j];
      }
  } else {  // shuffles inside: every lane
    float ks, vs;
    uint2 kc[kHalves], vc[kHalves];
    encode_row<CODES, GROUP>(kx, kc, ks);
    encode_row<CODES, GROUP>(vx, vc, vs);
    if (dst >= 0) {
#pragma unroll
      for (int j = 0; j < kHalves; j++) {
        ((uint2*)p.c.k)[dst * (D / 8) + j * GROUP + lane] = kc[j];
        ((uint2*)p.c.v)[dst * (D / 8) + j * GROUP + lane] = vc[j];
      }
      if (lane == 0) p.c.k_scale[dst] = ks;
      if (lane == 1) p.c.v_scale[dst] = vs;
    }
  }
}

struct ReadParams {
  Cache c;
  const int32_t *cu, *table;
  int64_t ld_table;
  int table_width, n_seqs;
  int64_t n_tokens;
  __nv_bfloat16 *k, *v;
  int64_t ldk, ldv;
  int* status;
};

// Two numbers that codes 2 i and 2 i + 1 of a word stand for (before the scale), exactly.
template <int CODES>
MB_DEV uint64_t decode2(uint32_t w, int i) {
  if (CODES == MB_KV_I8) {
    // byte c + 128 in the last place of 2^23
    const uint32_t u = w ^ 0x80808080u;
    return add2(pk2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + 2 * i)),
                      __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7651 + 2 * i))),
                pk2(-8388736.f, -8388736.f));
  }
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (16 * i))));
  const float2 f = __half22float2(*(const __half2*)&h);
  return pk2(f.x, f.y);
}

template <int CODES>
struct Held {  // a thread's values of a row as the cache holds them
  uint4 x[kHalves];
  float s;
};
template <int CODES, int D>
MB_DEV void load_row(Held<CODES>& r, const void* base, const float* scales, int64_t src, int lane) {
  constexpr int GROUP = D / 16;
  r.s = 0.f;
#pragma unroll
  for (int j = 0; j < kHalves; j++) {
    r.x[j] = make_uint4(0, 0, 0, 0);
    if (src < 0) continue;
    if (CODES == MB_KV_BF16) {
      r.x[j] = ld_stream((const uint4*)base + src * (D / 8) + j * GROUP + lane);
    } else {
      const uint2 c = ld_stream((const uint2*)base + src * (D / 8) + j * GROUP + lane);
      r.x[j].x = c.x, r.x[j].y = c.y;
    }
  }
  if (CODES != MB_KV_BF16 && src >= 0) r.s = scales[src];
}
template <int CODES>
MB_DEV uint4 decode_row(const Held<CODES>& r, int j) {
  if (CODES == MB_KV_BF16) return r.x[j];
  const uint64_t s2 = pk2(r.s, r.s);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    // f32 product, then one rounding to bf16
    float a, b;
    up2(mul2(decode2<CODES>(i < 2 ? r.x[j].x : r.x[j].y, i & 1), s2), a, b);
    o[i] = pack_bf16x2(a, b);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int CODES, int D>
__global__ void __launch_bounds__(kThreads) k_kv_read(const ReadParams p) {
  wait_before();
  constexpr int GROUP = D / 16, SIDE = 32 / GROUP;
  const int lane = threadIdx.x % GROUP;
  int h;
  const int64_t t0 = first_token<SIDE>(p.c.heads, h), t = t0 + (threadIdx.x & 31) / GROUP;
  if (t0 >= p.n_tokens) return;
  Span seq = seq_of(p.cu, nullptr, p.n_seqs, t0);
  if (t >= p.n_tokens) return;
  advance(seq, p.cu, nullptr, p.n_seqs, t);
  if (t < seq.c0 || t >= seq.c1) return;  // nobody's row
  const int64_t src = row_of(p.c, p.table + (int64_t)seq.b * p.ld_table, p.table_width, t - seq.c0, h, p.status);
  Held<CODES> kx, vx;
  load_row<CODES, D>(kx, p.c.k, p.c.k_scale, src, lane);
  load_row<CODES, D>(vx, p.c.v, p.c.v_scale, src, lane);
#pragma unroll
  for (int j = 0; j < kHalves; j++) {
    *((uint4*)(p.k + t * p.ldk + h * D) + j * GROUP + lane) = decode_row<CODES>(kx, j);
    *((uint4*)(p.v + t * p.ldv + h * D) + j * GROUP + lane) = decode_row<CODES>(vx, j);
  }
}

// Blocks for the rows of n_tokens tokens
inline int64_t blocks_of(int64_t n_tokens, const mb_kv_cache* c) {
  const int64_t tokens = kThreads / (c->head_dim / 16);  // of a block
  return (n_tokens + tokens - 1) / tokens * c->n_kv_heads;
}

// f(codes, head_dim) with both as types
template <class F>
cudaError_t dispatch(const mb_kv_cache* c, F f) {
  using std::integral_constant;
  auto by_dim = [&](auto codes) {
    return c->head_dim == 64 ? f(codes, integral_constant<int, 64>()) : f(codes, integral_constant<int, 128>());
  };
  if (c->dtype == MB_KV_I8) return by_dim(integral_constant<int, MB_KV_I8>());
  if (c->dtype == MB_KV_E4M3) return by_dim(integral_constant<int, MB_KV_E4M3>());
  return by_dim(integral_constant<int, MB_KV_BF16>());
}

}  // namespace kv

mb_status check_kv_cache(const mb_kv_cache* c) {
  MB_CHECK(c, MB_ERR_INVALID, "cache is NULL");
  MB_CHECK(c->dtype == MB_KV_BF16 || c->dtype == MB_KV_I8 || c->dtype == MB_KV_E4M3, MB_ERR_UNSUPPORTED,
           "cache dtype must be MB_KV_BF16, MB_KV_I8 or MB_KV_E4M3");
  MB_CHECK(c->head_dim == 64 || c->head_dim == 128, MB_ERR_UNSUPPORTED, "cache head_dim must be 64 or 128");
  MB_CHECK(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0, MB_ERR_INVALID,
           "page_size must be a power of two from 16 to 256");
  MB_CHECK(c->n_kv_heads > 0 && c->n_kv_heads <= 65535 && c->n_pages > 0 && c->n_pages < (1LL << 31), MB_ERR_INVALID,
           "cache sizes must be positive, n_pages below 2^31 and n_kv_heads below 65536");
  MB_CHECK(c->n_pages <= ((1LL << 31) - 1) / ((int64_t)c->n_kv_heads * c->page_size), MB_ERR_INVALID,
           "n_pages * n_kv_heads * page_size must be below 2^31");
  MB_CHECK(c->k && c->v, MB_ERR_INVALID, "cache k or v is NULL");
  MB_CHECK(((uintptr_t)c->k & 15) == 0 && ((uintptr_t)c->v & 15) == 0, MB_ERR_INVALID,
           "cache k and v must be 16-byte aligned");
  if (c->dtype != MB_KV_BF16)
    MB_CHECK(c->k_scale && c->v_scale && ((uintptr_t)c->k_scale & 15) == 0 && ((uintptr_t)c->v_scale & 15) == 0,
             MB_ERR_INVALID, "an 8-bit cache needs 16-byte aligned k_scale and v_scale");
  return MB_OK;
}

mb_status check_kv_table(const int32_t* table, int64_t ld_table, int table_width, int n_seqs) {
  MB_CHECK(n_seqs >= 0 && n_seqs < (1 << 24), MB_ERR_INVALID, "n_seqs must be from 0 to 2^24 - 1");
  MB_CHECK(table_width >= 0 && ld_table >= table_width && table_width < (1 << 23), MB_ERR_INVALID,
           "table_width must be from 0 to 2^23 - 1 and ld_table >= table_width");
  MB_CHECK(table || n_seqs == 0 || table_width == 0, MB_ERR_INVALID, "table is NULL");
  return MB_OK;
}

kv::Cache device_cache(const mb_kv_cache* c) {
  kv::Cache d;
  d.k = c->k;
  d.v = c->v;
  d.k_scale = c->k_scale;
  d.v_scale = c->v_scale;
  d.n_pages = c->n_pages;
  d.heads = c->n_kv_heads;
  d.page_log2 = __builtin_ctz((unsigned)c->page_size);
  return d;
}

static bool rows_ok(const void* p, int64_t ld, int64_t width) {
  return p && ((uintptr_t)p & 15) == 0 && ld >= width && ld % 8 == 0;
}

}  // namespace mb

using namespace mb;

extern "C" {

mb_status mb_kv_write(const mb_kv_cache* cache, const void* k, int64_t ldk, const void* v, int64_t ldv,
                      int64_t n_tokens, const int32_t* cu, const int32_t* kv_lens, const int32_t* table,
                      int64_t ld_table, int table_width, int n_seqs, void* stream) {
  mb_status s = check_kv_cache(cache);
  if (s == MB_OK) s = check_kv_table(table, ld_table, table_width, n_seqs);
  if (s != MB_OK) return s;
  const int64_t width = (int64_t)cache->n_kv_heads * cache->head_dim;
  MB_CHECK(n_tokens >= 0 && n_tokens < (1LL << 31), MB_ERR_INVALID, "n_tokens must be from 0 to 2^31 - 1");
  MB_CHECK(cu || n_tokens == n_seqs, MB_ERR_INVALID, "without cu there is one token for each sequence");
  if (n_tokens == 0 || n_seqs == 0) return MB_OK;
  MB_CHECK(kv_lens, MB_ERR_INVALID, "kv_lens is NULL");
  MB_CHECK(rows_ok(k, ldk, width) && rows_ok(v, ldv, width), MB_ERR_INVALID,
           "k and v must be 16-byte aligned with row strides of at least a row, multiples of 8");
  const int64_t blocks = kv::blocks_of(n_tokens, cache);
  MB_CHECK(blocks < (1LL << 31), MB_ERR_INVALID, "too many rows for one launch");
  MB_CHECK(device_status_ready(), MB_ERR_NOT_READY, "call mb_init on this device first");
  const kv::WriteParams p = {device_cache(cache), (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, ldk, ldv, n_tokens,
                             cu, kv_lens, table, ld_table, table_width, n_seqs, device_status_ptr()};
  MB_CUDA(kv::dispatch(cache, [&](auto codes, auto dim) {
    return launch_close(kv::k_kv_write<decltype(codes)::value, decltype(dim)::value>, dim3((unsigned)blocks), kv::kThreads, 0,
                        (cudaStream_t)stream, 1, p);
  }));
  return MB_OK;
}

mb_status mb_kv_read(const mb_kv_cache* cache, const int32_t* cu, const int32_t* table, int64_t ld_table,
                     int table_width, int n_seqs, int64_t n_tokens, void* k, int64_t ldk, void* v, int64_t ldv,
                     void* stream) {
  mb_status s = check_kv_cache(cache);
  if (s == MB_OK) s = check_kv_table(table, ld_table, table_width, n_seqs);
  if (s != MB_OK) return s;
  const int64_t width = (int64_t)cache->n_kv_heads * cache->head_dim;
  MB_CHECK(n_tokens >= 0 && n_tokens < (1LL << 31), MB_ERR_INVALID, "n_tokens must be from 0 to 2^31 - 1");
  if (n_tokens == 0 || n_seqs == 0) return MB_OK;
  MB_CHECK(cu, MB_ERR_INVALID, "cu is NULL");
  MB_CHECK(rows_ok(k, ldk, width) && rows_ok(v, ldv, width), MB_ERR_INVALID,
           "k and v must be 16-byte aligned with row strides of at least a row, multiples of 8");
  const int64_t blocks = kv::blocks_of(n_tokens, cache);
  MB_CHECK(blocks < (1LL << 31), MB_ERR_INVALID, "too many rows for one launch");
  MB_CHECK(device_status_ready(), MB_ERR_NOT_READY, "call mb_init on this device first");
  const kv::ReadParams p = {device_cache(cache), cu, table, ld_table, table_width, n_seqs, n_tokens,
                            (__nv_bfloat16*)k, (__nv_bfloat16*)v, ldk, ldv, device_status_ptr()};
  MB_CUDA(kv::dispatch(cache, [&](auto codes, auto dim) {
    return launch_close(kv::k_kv_read<decltype(codes)::value, decltype(dim)::value>, dim3((unsigned)blocks), kv::kThreads, 0,
                        (cudaStream_t)stream, 1, p);
  }));
  return MB_OK;
}

}  // extern "C"
