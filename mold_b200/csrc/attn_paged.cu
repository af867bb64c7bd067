// K14: attention of one new token of each sequence over a paged key-value cache (bf16, or 8-bit codes
// with a scale a row), split over the cached length and joined.
//
// Work is counted in tiles of kWarps * KEYS keys of one unit = (sequence, key head, up to 16 of the
// query heads that read it). The tiles of all units in a row are cut into equal runs, one for each
// block of a grid that fills the SMs, so blocks end together however far the lengths lie apart. A
// block's part of a unit that it does not hold whole goes to the workspace as (max, sum, unnormalised
// output); k_join adds a unit's parts in the order of the blocks.
//
// Keys and values go from memory straight into the operand registers of the warp matrix products
// (q k^T: m16n8k16 with the query heads as rows; p v: the same with the keys as depth). Which k index
// of a product stands for which channel is free as long as both operands agree, so every lane loads 16
// contiguous bytes of a row and no operand passes through shared memory; values of two keys are paired
// with a byte permute. 8-bit codes are integers or e4m3 numbers that bf16 holds exactly: the products
// run on the codes, the key's scale multiplies the score, the value's scale the weight, before the
// weight's one rounding to bf16. Scores, maximum, sum and output stay in f32.
#include <string>

#include "common.cuh"
#include "internal.h"
#include "kv_cache.cuh"

namespace mb {
namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;      // query rows of a unit
constexpr int kBlocksPerSm = 2;

struct Part {  // of a unit's work: its first block and how many blocks hold a piece (1: none is joined)
  int first, pieces;
};

struct Params {
  const __nv_bfloat16* q;
  int64_t ldq;
  kv::Cache c;
  const int32_t *lens, *table;
  int64_t ld_table;
  int table_width, n_seqs;
  int H, G, q_tiles, units_per_seq;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t ldo;
  Part* parts;       // [units]
  float *part_ml;    // [2 * blocks][2][kRows]
  float *part_o;     // [2 * blocks][kRows][D]
  int* status;
};

MB_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two codes as a bf16 pair, exactly. `x` holds them in the low (int8) or high (e4m3) byte of its halves; the other
// bytes may hold anything.
//   int8: the low seven bits under the exponent of 128 give 128 + (c mod 128); the sign bit makes 256 of the 128
//   that is taken off.
//   e4m3: exponent and mantissa bits moved to bf16's places give c * 2^-120, subnormal codes included.
template <int CODES>
MB_DEV uint32_t codes_bf16x2(uint32_t x) {
  __nv_bfloat162 r;
  if (CODES == MB_KV_I8) {
    const uint32_t a = (x & 0x007f007fu) | 0x43004300u, b = (x & 0x00800080u) | 0x43004300u;
    r = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  } else {
    const uint32_t a = ((x >> 4) & 0x07f007f0u) | (x & 0x80008000u), b = 0x7b807b80u;
    r = __hmul2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  }
  return *(uint32_t*)&r;
}
// Bytes i and j of w (8-bit codes of neighbouring channels), or byte i of two words, as a bf16 pair.
template <int CODES>
MB_DEV uint32_t pair_in_word(uint32_t w, int i, int j) {
  return codes_bf16x2<CODES>(CODES == MB_KV_I8 ? __byte_perm(w, 0, i | (j << 8)) : __byte_perm(w, 0, (i << 4) | (j << 12)));
}
template <int CODES>
MB_DEV uint32_t pair_of_words(uint32_t w0, uint32_t w1, int i) {
  return codes_bf16x2<CODES>(CODES == MB_KV_I8 ? __byte_perm(w0, w1, i | ((4 + i) << 8))
                                               : __byte_perm(w0, w1, (i << 4) | ((4 + i) << 12)));
}

// One warp's keys of a step, in operand registers. KEYS a multiple of 16; lane = 4 g + t.
//   k: lane (g, t) holds, of key 8 nt + g, the 16 bytes at t of every 64-byte piece of the row.
//   v: lane (g, t) holds, of keys 16 kg + {2t, 2t + 1, 2t + 8, 2t + 9}, the bytes at g of every eighth.
template <int CODES, int D, int KEYS>
struct Tile {
  static constexpr int EB = CODES == MB_KV_BF16 ? 2 : 1;
  static constexpr int KW = D * EB / 16;              // words of a key row a lane holds
  static constexpr int VB = D * EB / 8 < 16 ? 8 : 16;  // bytes of a value load
  static constexpr int VC = D * EB / 8 / VB;          // value loads of a row a lane makes
  static constexpr int VW = D * EB / 32;              // words of a value row a lane holds
  uint32_t k[KEYS / 8][KW];
  uint32_t v[KEYS / 16][4][VW];
  float2 ks[KEYS / 8], vs[KEYS / 8];

  // rows[i]: cache row of key 16 i of the step, -1 for none; left: keys of the step that exist
  MB_DEV void load_k(const kv::Cache& c, const int64_t (&rows)[KEYS / 16], int left, int g, int t) {
#pragma unroll
    for (int nt = 0; nt < KEYS / 8; nt++) {
      const int64_t row = rows[nt / 2] + (nt & 1) * 8 + g;
      const bool ok = rows[nt / 2] >= 0 && nt * 8 + g < left;
      const uint4* src = (const uint4*)((const uint8_t*)c.k + row * (D * EB)) + t;
#pragma unroll
      for (int i = 0; i < KW / 4; i++) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (ok) x = kv::ld_stream(src + 4 * i);
        k[nt][4 * i] = x.x, k[nt][4 * i + 1] = x.y, k[nt][4 * i + 2] = x.z, k[nt][4 * i + 3] = x.w;
      }
      if (CODES != MB_KV_BF16) {
        const int64_t r2 = rows[nt / 2] + (nt & 1) * 8 + 2 * t;
        ks[nt] = rows[nt / 2] >= 0 && nt * 8 + 2 * t < left ? *(const float2*)(c.k_scale + r2) : make_float2(0.f, 0.f);
      }
    }
  }
  MB_DEV void load_v(const kv::Cache& c, const int64_t (&rows)[KEYS / 16], int left, int g, int t) {
#pragma unroll
    for (int kg = 0; kg < KEYS / 16; kg++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int key = 2 * t + (j & 1) + (j >> 1) * 8;
        const bool ok = rows[kg] >= 0 && kg * 16 + key < left;
        const uint8_t* src = (const uint8_t*)c.v + (rows[kg] + key) * (D * EB) + g * VB;
#pragma unroll
        for (int i = 0; i < VC; i++) {
          if (VB == 16) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (ok) x = kv::ld_stream((const uint4*)(src + i * 128));
            v[kg][j][4 * i] = x.x, v[kg][j][4 * i + 1] = x.y;
            v[kg][j][4 * i + 2 < VW ? 4 * i + 2 : 0] = x.z, v[kg][j][4 * i + 3 < VW ? 4 * i + 3 : 0] = x.w;
          } else {
            uint2 x = make_uint2(0, 0);
            if (ok) x = kv::ld_stream((const uint2*)src);
            v[kg][j][0] = x.x, v[kg][j][1] = x.y;
          }
        }
      }
      if (CODES != MB_KV_BF16) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int key = kg * 16 + u * 8 + 2 * t;
          const float2 s = rows[kg] >= 0 && key < left ? *(const float2*)(c.v_scale + rows[kg] + u * 8 + 2 * t)
                                                       : make_float2(0.f, 0.f);
          vs[kg * 2 + u] = make_float2(s.x, key + 1 < left ? s.y : 0.f);
        }
      }
    }
  }
  // operand words (two 16-bit k pairs) of product step s of key row nt
  MB_DEV void k_operand(int nt, int s, uint32_t& b0, uint32_t& b1) const {
    if (CODES == MB_KV_BF16) {
      b0 = k[nt][2 * s], b1 = k[nt][2 * s + 1];
    } else {
      b0 = pair_in_word<CODES>(k[nt][s], 0, 1), b1 = pair_in_word<CODES>(k[nt][s], 2, 3);
    }
  }
  // operand words of output column tile n for the 16 keys of group kg
  MB_DEV void v_operand(int kg, int n, uint32_t& b0, uint32_t& b1) const {
    if (CODES == MB_KV_BF16) {
      const int w = n / 2, sel = n & 1 ? 0x7632 : 0x5410;
      b0 = __byte_perm(v[kg][0][w], v[kg][1][w], sel), b1 = __byte_perm(v[kg][2][w], v[kg][3][w], sel);
    } else {
      b0 = pair_of_words<CODES>(v[kg][0][n / 4], v[kg][1][n / 4], n & 3);
      b1 = pair_of_words<CODES>(v[kg][2][n / 4], v[kg][3][n / 4], n & 3);
    }
  }
  // channel of element (n, column c) of the output
  static MB_DEV int channel(int n, int c) {
    return CODES == MB_KV_BF16 ? (n / 8) * 64 + c * 8 + (n & 7) : c * (D / 8) + n;
  }
  // first channel of the four that lane t's query operand holds at product step s
  static MB_DEV int q_channel(int s, int t) {
    return CODES == MB_KV_BF16 ? (s / 2) * 32 + t * 8 + (s & 1) * 4 : (s / 4) * 64 + t * 16 + (s & 3) * 4;
  }
};

// Run of tiles of block c of n: [first, last)
MB_DEV int64_t run_start(int64_t total, int c, int n) { return total * c / n; }
// The block whose run holds tile t
MB_DEV int run_owner(int64_t total, int64_t t, int n) { return (int)(((t + 1) * n - 1) / total); }

template <int CODES, int D, bool WIDE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) k_attention_paged(const Params p) {
  constexpr int KEYS = CODES == MB_KV_BF16 ? 16 : 32;
  constexpr int kTileKeys = kWarps * KEYS;
  constexpr int ROWS = WIDE ? 16 : 8;
  constexpr int KS = D / 16;  // product steps over the channels
  using T = Tile<CODES, D, KEYS>;
  __shared__ float s_o[kWarps][ROWS][D];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  __shared__ int64_t s_sum[kWarps + 1];
  __shared__ int64_t s_at;  // tiles before the sequence
  __shared__ int s_seq;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t cap = (int64_t)p.table_width << p.c.page_log2;
  const int U = p.units_per_seq;
  auto length = [&](int b) -> int64_t {
    if (b >= p.n_seqs) return 0;
    const int64_t n = __ldg(p.lens + b);
    return n < 0 ? 0 : n < cap ? n : cap;
  };
  auto tiles_of = [&](int64_t len) { return (len + kTileKeys - 1) / kTileKeys; };
  // tiles of sequences base .. base + threadIdx.x together (block-wide), and of all kThreads
  auto scan = [&](int base, int64_t& all) {
    int64_t x = tiles_of(length(base + (int)threadIdx.x)) * U;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = x;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) x += s_sum[w];
      all += s_sum[w];
    }
    return x;
  };

  int64_t total = 0, all, incl = 0;
  for (int base = 0; base < p.n_seqs; base += kThreads) {
    incl = scan(base, all);
    total += all;
  }
  const int c = blockIdx.x;
  // sequences without positions: their rows are 0
  for (int b = c; b < p.n_seqs; b += gridDim.x)
    if (length(b) == 0)
      for (int i = threadIdx.x; i < p.H * D / 8; i += kThreads) *((uint4*)(p.out + b * p.ldo) + i) = make_uint4(0, 0, 0, 0);
  // every block of a run has a tile, so that the blocks between a unit's first and last hold pieces of it
  const int n_blocks = (int)(total < gridDim.x ? total : gridDim.x);
  if (c >= n_blocks) return;
  const int64_t t0 = run_start(total, c, n_blocks), t1 = run_start(total, c + 1, n_blocks);
  int64_t before = 0;
  for (int base = 0;; base += kThreads) {
    if (p.n_seqs > kThreads) incl = scan(base, all); else all = total;
    const int64_t own = tiles_of(length(base + (int)threadIdx.x)) * U;
    const int64_t end = before + incl;
    if (t0 < end && t0 >= end - own) s_seq = base + threadIdx.x, s_at = end - own;
    before += all;
    if (t0 < before) break;
  }
  __syncthreads();

  int b = s_seq;
  int64_t at = s_at, tile = t0;
  while (tile < t1) {
    int64_t len = length(b);
    int64_t nt = tiles_of(len);
    while (tile >= at + nt * U) {  // next sequence that has tiles
      if (b >= p.n_seqs) return;
      at += nt * U;
      len = length(++b);
      nt = tiles_of(len);
    }
    const int unit = (int)((tile - at) / nt);
    const int64_t unit_at = at + unit * nt;
    const int64_t last = min(t1, unit_at + nt);
    const int kt0 = (int)(tile - unit_at), kt1 = (int)(last - unit_at);
    const int hk = unit / p.q_tiles, qt = unit - hk * p.q_tiles;
    const int rows = min(kRows, p.G - qt * kRows);
    const int head0 = hk * p.G + qt * kRows;

    // query operand: rows g and g + 8, rows that do not exist 0
    uint32_t qa[KS][WIDE ? 4 : 2];
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const __nv_bfloat16* src = p.q + (int64_t)b * p.ldq + (int64_t)head0 * D + T::q_channel(s, t);
      uint2 x = make_uint2(0, 0);
      if (g < rows) x = *(const uint2*)(src + (int64_t)g * D);
      qa[s][0] = x.x, qa[s][1] = x.y;
      if (WIDE) {
        uint2 y = make_uint2(0, 0);
        if (g + 8 < rows) y = *(const uint2*)(src + (int64_t)(g + 8) * D);
        qa[s][WIDE ? 2 : 0] = y.x, qa[s][WIDE ? 3 : 1] = y.y;
        if (!WIDE) qa[s][0] = x.x, qa[s][1] = x.y;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int32_t* table = p.table + (int64_t)b * p.ld_table;

    for (int kt = kt0; kt < kt1; kt++) {
      const int64_t key0 = (int64_t)kt * kTileKeys + warp * KEYS;
      if (key0 >= len) break;
      const int left = (int)min(len - key0, (int64_t)KEYS);
      int64_t rows16[KEYS / 16];
#pragma unroll
      for (int i = 0; i < KEYS / 16; i++)
        rows16[i] = i * 16 < left ? kv::row_of(p.c, table, p.table_width, key0 + i * 16, hk, p.status) : -1;
      T x;
      x.load_k(p.c, rows16, left, g, t);
      x.load_v(p.c, rows16, left, g, t);
      float s[KEYS / 8][4];
#pragma unroll
      for (int nt8 = 0; nt8 < KEYS / 8; nt8++) {
        s[nt8][0] = s[nt8][1] = s[nt8][2] = s[nt8][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; i++) {
          uint32_t b0, b1;
          x.k_operand(nt8, i, b0, b1);
          mma16816(s[nt8], qa[i][0], WIDE ? qa[i][WIDE ? 2 : 0] : 0u, qa[i][1], WIDE ? qa[i][WIDE ? 3 : 1] : 0u, b0, b1);
        }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt8 = 0; nt8 < KEYS / 8; nt8++) {
        const float f0 = p.scale_log2 * (CODES == MB_KV_BF16 ? 1.f : x.ks[nt8].x);
        const float f1 = p.scale_log2 * (CODES == MB_KV_BF16 ? 1.f : x.ks[nt8].y);
        const bool in = rows16[nt8 / 2] >= 0;
        const bool k0 = in && nt8 * 8 + 2 * t < left, k1 = in && nt8 * 8 + 2 * t + 1 < left;
#pragma unroll
        for (int r = 0; r < (WIDE ? 2 : 1); r++) {
          s[nt8][2 * r] = k0 ? s[nt8][2 * r] * f0 : -INFINITY;
          s[nt8][2 * r + 1] = k1 ? s[nt8][2 * r + 1] * f1 : -INFINITY;
          mx[r] = fmaxf(mx[r], fmaxf(s[nt8][2 * r], s[nt8][2 * r + 1]));
        }
      }
      float ref[2], alpha[2];
#pragma unroll
      for (int r = 0; r < (WIDE ? 2 : 1); r++) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float mn = fmaxf(m[r], mx[r]);
        ref[r] = mn == -INFINITY ? 0.f : mn;  // nothing but -inf so far: weights 0
        alpha[r] = ex2_approx(m[r] - ref[r]);
        m[r] = mn;
        l[r] *= alpha[r];
      }
      if (!WIDE) ref[1] = 0.f, alpha[1] = 1.f;
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < D / 8; n++) {
          o[n][0] *= alpha[0], o[n][1] *= alpha[0];
          if (WIDE) o[n][2] *= alpha[1], o[n][3] *= alpha[1];
        }
      }
#pragma unroll
      for (int kg = 0; kg < KEYS / 16; kg++) {
        uint32_t a[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int nt8 = 2 * kg + u;
#pragma unroll
          for (int r = 0; r < (WIDE ? 2 : 1); r++) {
            const float p0 = ex2_approx(s[nt8][2 * r] - ref[r]), p1 = ex2_approx(s[nt8][2 * r + 1] - ref[r]);
            l[r] += p0 + p1;
            a[2 * u + r] = CODES == MB_KV_BF16 ? pack_bf16x2(p0, p1) : pack_bf16x2(p0 * x.vs[nt8].x, p1 * x.vs[nt8].y);
          }
        }
#pragma unroll
        for (int n = 0; n < D / 8; n++) {
          uint32_t b0, b1;
          x.v_operand(kg, n, b0, b1);
          mma16816(o[n], a[0], a[1], a[2], a[3], b0, b1);
        }
      }
    }

    // the warps' parts together
#pragma unroll
    for (int r = 0; r < (WIDE ? 2 : 1); r++) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) s_m[warp][g + 8 * r] = m[r], s_l[warp][g + 8 * r] = l[r];
#pragma unroll
      for (int n = 0; n < D / 8; n++) {
        s_o[warp][g + 8 * r][T::channel(n, 2 * t)] = o[n][2 * r];
        s_o[warp][g + 8 * r][T::channel(n, 2 * t + 1)] = o[n][2 * r + 1];
      }
    }
    __syncthreads();
    const bool whole = kt0 == 0 && kt1 == nt;
    const int64_t slot = 2 * c + (kt0 == 0 ? 1 : 0);
    constexpr int RP = kThreads / D;  // rows at a time
    for (int r = threadIdx.x / D; r < rows; r += RP) {
      const int d = threadIdx.x % D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; w++) top = fmaxf(top, s_m[w][r]);
      const float ref1 = top == -INFINITY ? 0.f : top;
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        const float f = ex2_approx(s_m[w][r] - ref1);
        acc += f * s_o[w][r][d];
        sum += f * s_l[w][r];
      }
      if (whole) {
        p.out[(int64_t)b * p.ldo + (int64_t)(head0 + r) * D + d] = __float2bfloat16_rn(acc / sum);
      } else {
        p.part_o[(slot * kRows + r) * D + d] = acc;
        if (d == 0) {
          p.part_ml[slot * 2 * kRows + r] = top;
          p.part_ml[slot * 2 * kRows + kRows + r] = sum;
        }
      }
    }
    if (kt0 == 0 && threadIdx.x == 0) {
      Part part;
      part.first = c;
      part.pieces = whole ? 1 : run_owner(total, unit_at + nt - 1, n_blocks) - c + 1;
      p.parts[(int64_t)b * U + unit] = part;
    }
    __syncthreads();
    tile = last;
  }
}

// Adds up the parts of each unit that several blocks hold. One block a unit and row.
template <int D>
__global__ void __launch_bounds__(D) k_join(const Params p) {
  const int u = blockIdx.x, r = blockIdx.y, d = threadIdx.x;
  const int b = u / p.units_per_seq, unit = u - b * p.units_per_seq;
  const int hk = unit / p.q_tiles, qt = unit - hk * p.q_tiles;
  if (r >= p.G - qt * kRows || __ldg(p.lens + b) <= 0 || p.table_width == 0) return;
  const Part part = p.parts[u];
  if (part.pieces <= 1) return;
  auto slot = [&](int i) { return (int64_t)2 * (part.first + i) + (i == 0 ? 1 : 0); };
  float top = -INFINITY;
  for (int i = 0; i < part.pieces; i++) top = fmaxf(top, p.part_ml[slot(i) * 2 * kRows + r]);
  const float ref = top == -INFINITY ? 0.f : top;
  float acc = 0.f, sum = 0.f;
  for (int i = 0; i < part.pieces; i++) {
    const int64_t s = slot(i);
    const float f = ex2_approx(p.part_ml[s * 2 * kRows + r] - ref);
    acc += f * p.part_o[(s * kRows + r) * D + d];
    sum += f * p.part_ml[s * 2 * kRows + kRows + r];
  }
  p.out[(int64_t)b * p.ldo + (int64_t)(hk * p.G + qt * kRows + r) * D + d] = __float2bfloat16_rn(acc / sum);
}

struct Layout {
  int64_t units, blocks;
  size_t ml, o, bytes;  // offsets of the parts' statistics and outputs
};
Layout layout(int n_seqs, int H, int H_kv, int D) {
  Layout a;
  a.units = (int64_t)n_seqs * H_kv * ((H / H_kv + kRows - 1) / kRows);
  a.blocks = (int64_t)num_sms() * kBlocksPerSm;
  a.ml = ((size_t)a.units * sizeof(Part) + 255) / 256 * 256;
  a.o = a.ml + (size_t)a.blocks * 2 * 2 * kRows * sizeof(float);
  a.bytes = a.o + (size_t)a.blocks * 2 * kRows * D * sizeof(float);
  return a;
}

template <int CODES, int D>
cudaError_t launch(const Params& p, int64_t blocks, int64_t units, cudaStream_t st) {
  if (p.G > 8)
    k_attention_paged<CODES, D, true><<<(unsigned)blocks, kThreads, 0, st>>>(p);
  else
    k_attention_paged<CODES, D, false><<<(unsigned)blocks, kThreads, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  k_join<D><<<dim3((unsigned)units, (unsigned)(p.G < kRows ? p.G : kRows)), D, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace paged
}  // namespace mb

using namespace mb;

static mb_status check_heads(int n_seqs, int H, int H_kv, int D) {
  MB_CHECK(D == 64 || D == 128, MB_ERR_UNSUPPORTED, "head size D must be 64 or 128");
  MB_CHECK(n_seqs >= 0 && n_seqs < (1 << 24), MB_ERR_INVALID, "n_seqs must be from 0 to 2^24 - 1");
  MB_CHECK(H > 0 && H_kv > 0 && H % H_kv == 0 && H <= 65535, MB_ERR_INVALID,
           "H must be a positive multiple of H_kv, at most 65535");
  MB_CHECK((int64_t)n_seqs * H < (1LL << 31), MB_ERR_INVALID, "n_seqs * H must be below 2^31");
  return MB_OK;
}

extern "C" {

mb_status mb_attention_paged_workspace(int n_seqs, int H, int H_kv, int D, size_t* bytes) {
  MB_CHECK(bytes, MB_ERR_INVALID, "bytes is NULL");
  const mb_status s = check_heads(n_seqs, H, H_kv, D);
  if (s != MB_OK) return s;
  *bytes = paged::layout(n_seqs, H, H_kv, D).bytes;
  return MB_OK;
}

mb_status mb_attention_paged(const void* q, int64_t ldq, const mb_kv_cache* cache, const int32_t* kv_lens,
                             const int32_t* table, int64_t ld_table, int table_width, int n_seqs, int H, float scale,
                             void* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
  mb_status s = check_kv_cache(cache);
  if (s == MB_OK) s = check_kv_table(table, ld_table, table_width, n_seqs);
  if (s == MB_OK) s = check_heads(n_seqs, H, cache->n_kv_heads, cache->head_dim);
  if (s != MB_OK) return s;
  MB_CHECK(scale >= 0.f && scale <= 3.0e38f, MB_ERR_INVALID, "scale must be positive and finite (0: 1 / sqrt(D))");
  if (n_seqs == 0) return MB_OK;
  const int D = cache->head_dim;
  MB_CHECK(kv_lens, MB_ERR_INVALID, "kv_lens is NULL");
  MB_CHECK(q && ((uintptr_t)q & 15) == 0 && ldq >= (int64_t)H * D && ldq % 8 == 0, MB_ERR_INVALID,
           "q must be 16-byte aligned with ldq >= H * D, a multiple of 8");
  MB_CHECK(out && ((uintptr_t)out & 15) == 0 && ldo >= (int64_t)H * D && ldo % 8 == 0, MB_ERR_INVALID,
           "out must be 16-byte aligned with ldo >= H * D, a multiple of 8");
  MB_CHECK(device_status_ready(), MB_ERR_NOT_READY, "call mb_init on this device first");
  const paged::Layout a = paged::layout(n_seqs, H, cache->n_kv_heads, D);
  MB_CHECK(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= a.bytes, MB_ERR_INVALID,
           "workspace must be 16-byte aligned and of mb_attention_paged_workspace bytes");
  paged::Params p;
  p.q = (const __nv_bfloat16*)q;
  p.ldq = ldq;
  p.c = device_cache(cache);
  p.lens = kv_lens;
  p.table = table;
  p.ld_table = ld_table;
  p.table_width = table_width;
  p.n_seqs = n_seqs;
  p.H = H;
  p.G = H / cache->n_kv_heads;
  p.q_tiles = (p.G + paged::kRows - 1) / paged::kRows;
  p.units_per_seq = cache->n_kv_heads * p.q_tiles;
  p.scale_log2 = (float)((scale > 0.f ? (double)scale : 1.0 / sqrt((double)D)) * 1.4426950408889634);
  p.out = (__nv_bfloat16*)out;
  p.ldo = ldo;
  p.parts = (paged::Part*)workspace;
  p.part_ml = (float*)((char*)workspace + a.ml);
  p.part_o = (float*)((char*)workspace + a.o);
  p.status = device_status_ptr();
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (D == 64)
    e = cache->dtype == MB_KV_BF16 ? paged::launch<MB_KV_BF16, 64>(p, a.blocks, a.units, st)
        : cache->dtype == MB_KV_I8 ? paged::launch<MB_KV_I8, 64>(p, a.blocks, a.units, st)
                                   : paged::launch<MB_KV_E4M3, 64>(p, a.blocks, a.units, st);
  else
    e = cache->dtype == MB_KV_BF16 ? paged::launch<MB_KV_BF16, 128>(p, a.blocks, a.units, st)
        : cache->dtype == MB_KV_I8 ? paged::launch<MB_KV_I8, 128>(p, a.blocks, a.units, st)
                                   : paged::launch<MB_KV_E4M3, 128>(p, a.blocks, a.units, st);
  MB_CUDA(e);
  return MB_OK;
}

}  // extern "C"
