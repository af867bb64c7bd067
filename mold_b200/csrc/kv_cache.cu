// K12 / K13: the paged key-value cache of a text transformer, written (bf16, or 8-bit codes with
// one f32 scale for each row of head_dim values) and read back.
//
// Both move each row once: a group of head_dim / 8 threads owns a (token, head) row of k and the
// same row of v, 16 bytes of bf16 a thread. Bound by HBM.
#include <mutex>
#include <string>

#include "common.cuh"
#include "internal.h"
#include "kv_cache.cuh"

namespace mb {
namespace kv {

// The sequence whose rows hold t: the last b with cu[b] <= t. Whatever cu holds, b is in [0, n).
MB_DEV int seq_of(const int32_t* cu, int n, int64_t t) {
  int lo = 0, hi = n;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid; else hi = mid;
  }
  return lo;
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

// A row's eight values of this thread as codes; scale: what the row's codes stand for times.
template <int CODES, int GROUP>
MB_DEV uint2 encode_row(const uint4& x, float& scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  // largest magnitude: the bit patterns of non-negative floats order like the floats, NaN last
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) top = max(top, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
#pragma unroll
  for (int o = GROUP / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  constexpr float T = CODES == MB_KV_I8 ? 127.f : 448.f;
  const bool finite = top < 0x7f800000u;
  const bool some = finite && top >= 0x0d800000u;  // 2^-100: below it the inverse would overflow
  const float m = __uint_as_float(top);
  scale = some ? __fdiv_rn(m, T) : finite ? 0.f : __uint_as_float(0x7fc00000u);
  const float r = some ? __fdiv_rn(T, m) : 0.f;
  uint32_t out[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      y[2 * j] = __fmul_rn(bf16_lo(w[2 * i + j]), r);
      y[2 * j + 1] = __fmul_rn(bf16_hi(w[2 * i + j]), r);
    }
    if (!finite) y[0] = y[1] = y[2] = y[3] = 0.f;  // NaN and infinity times 0
    if (CODES == MB_KV_I8) {
      // |y| <= 127 (1 + 2^-23) rounds to at most 127
      uint32_t b = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) b |= ((uint32_t)__float2int_rn(y[j]) & 255u) << (8 * j);
      out[i] = b;
    } else {
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
      out[i] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
  }
  return make_uint2(out[0], out[1]);
}

template <int CODES, int D>
__global__ void __launch_bounds__(256) k_kv_write(const WriteParams p) {
  constexpr int GROUP = D / 8;
  const int lane = threadIdx.x % GROUP;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / GROUP;
  const int heads = p.c.heads;
  const int64_t t = row / heads;
  const int h = (int)(row - t * heads);
  int64_t dst = -1;
  if (t < p.n_tokens) {
    int b = (int)t;
    int64_t pos = 0, first = 0;
    if (p.cu) {
      b = seq_of(p.cu, p.n_seqs, t);
      const int64_t c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1);
      first = (t >= c0 && t < c1) ? t - c1 : INT64_MIN / 2;
    } else {
      first = -1;
    }
    pos = (int64_t)__ldg(p.lens + b) + first;
    if (pos >= 0) dst = row_of(p.c, p.table + (int64_t)b * p.ld_table, p.table_width, pos, h, p.status);
  }
  // whole groups agree on dst; the shuffles below need every lane of the warp
  uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
  if (dst >= 0) {
    kx = ld_stream((const uint4*)(p.k + t * p.ldk + (int64_t)h * D) + lane);
    vx = ld_stream((const uint4*)(p.v + t * p.ldv + (int64_t)h * D) + lane);
  }
  if (CODES == MB_KV_BF16) {
    if (dst >= 0) {
      ((uint4*)p.c.k)[dst * GROUP + lane] = kx;
      ((uint4*)p.c.v)[dst * GROUP + lane] = vx;
    }
  } else {
    float ks, vs;
    const uint2 kc = encode_row<CODES, GROUP>(kx, ks), vc = encode_row<CODES, GROUP>(vx, vs);
    if (dst >= 0) {
      ((uint2*)p.c.k)[dst * GROUP + lane] = kc;
      ((uint2*)p.c.v)[dst * GROUP + lane] = vc;
      if (lane == 0) {
        p.c.k_scale[dst] = ks;
        p.c.v_scale[dst] = vs;
      }
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

template <int CODES, int D>
MB_DEV uint4 decode_row(const void* base, const float* scales, int64_t src, int lane) {
  constexpr int GROUP = D / 8;
  if (CODES == MB_KV_BF16) return ld_stream((const uint4*)base + src * GROUP + lane);
  const uint2 c = ld_stream((const uint2*)base + src * GROUP + lane);
  const float s = __ldg(scales + src);
  const uint32_t w[2] = {c.x, c.y};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    float y[4];
    decode4<CODES>(w[i], y);
    // f32 product, then one rounding to bf16
    o[2 * i] = pack_bf16x2(__fmul_rn(y[0], s), __fmul_rn(y[1], s));
    o[2 * i + 1] = pack_bf16x2(__fmul_rn(y[2], s), __fmul_rn(y[3], s));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int CODES, int D>
__global__ void __launch_bounds__(256) k_kv_read(const ReadParams p) {
  constexpr int GROUP = D / 8;
  const int lane = threadIdx.x % GROUP;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / GROUP;
  const int heads = p.c.heads;
  const int64_t t = row / heads;
  const int h = (int)(row - t * heads);
  if (t >= p.n_tokens) return;
  const int b = seq_of(p.cu, p.n_seqs, t);
  const int64_t c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1);
  if (t < c0 || t >= c1) return;
  const int64_t src = row_of(p.c, p.table + (int64_t)b * p.ld_table, p.table_width, t - c0, h, p.status);
  uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
  if (src >= 0) {
    kx = decode_row<CODES, D>(p.c.k, p.c.k_scale, src, lane);
    vx = decode_row<CODES, D>(p.c.v, p.c.v_scale, src, lane);
  }
  *((uint4*)(p.k + t * p.ldk + (int64_t)h * D) + lane) = kx;
  *((uint4*)(p.v + t * p.ldv + (int64_t)h * D) + lane) = vx;
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
  MB_CHECK(c->n_pages < (1LL << 31) / ((int64_t)c->n_kv_heads * c->page_size), MB_ERR_INVALID,
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
  const int64_t blocks = (n_tokens * cache->n_kv_heads * (cache->head_dim / 8) + 255) / 256;
  MB_CHECK(blocks < (1LL << 31), MB_ERR_INVALID, "too many rows for one launch");
  MB_CHECK(device_status_ready(), MB_ERR_NOT_READY, "call mb_init on this device first");
  const kv::WriteParams p = {device_cache(cache), (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, ldk, ldv, n_tokens,
                             cu, kv_lens, table, ld_table, table_width, n_seqs, device_status_ptr()};
  MB_CUDA(kv::dispatch(cache, [&](auto codes, auto dim) {
    kv::k_kv_write<decltype(codes)::value, decltype(dim)::value><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
    return cudaGetLastError();
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
  const int64_t blocks = (n_tokens * cache->n_kv_heads * (cache->head_dim / 8) + 255) / 256;
  MB_CHECK(blocks < (1LL << 31), MB_ERR_INVALID, "too many rows for one launch");
  MB_CHECK(device_status_ready(), MB_ERR_NOT_READY, "call mb_init on this device first");
  const kv::ReadParams p = {device_cache(cache), cu, table, ld_table, table_width, n_seqs, n_tokens,
                            (__nv_bfloat16*)k, (__nv_bfloat16*)v, ldk, ldv, device_status_ptr()};
  MB_CUDA(kv::dispatch(cache, [&](auto codes, auto dim) {
    kv::k_kv_read<decltype(codes)::value, decltype(dim)::value><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
    return cudaGetLastError();
  }));
  return MB_OK;
}

}  // extern "C"
