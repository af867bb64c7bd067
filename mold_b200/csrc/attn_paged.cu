// K14: attention of one new token of each sequence over a paged key-value cache (bf16, or 8-bit codes
// with a scale a row), split over the cached length and joined.
//
// Work is counted in tiles of kTileKeys keys of one unit = (sequence, key head, up to 16 of the query
// heads that read it), and Shape::UNIT_COST for a unit's own expense. All units in a row are cut into
// runs of equal cost, one for each block of a grid that fills the SMs, so blocks end together however far
// the lengths lie apart. A block's part of a unit that it does not hold whole goes to the workspace as
// (max, sum, unnormalised output); k_join adds a unit's parts in the order of the blocks.
//
// One warp of a block walks the run and keeps a ring of tiles in flight: page numbers, one TMA box of 16 to
// 64 keys x 128 bytes after the other (keys, values; 128-byte swizzle), scales and the unit's queries, all
// landing on the stage's mbarrier. It runs ahead over the borders of units, so a batch of short
// sequences keeps memory as busy as a long one. Four warps take 16 keys of a tile each: scores and outputs
// as warp products (at one token a sequence there is too little arithmetic for more). Which depth index of
// the scores' product stands for which channel is free as long as both operands agree, so a lane reads 16
// contiguous bytes of a key row. Scores, maximum, sum and output stay in f32; over a bf16 cache the weights
// are rounded to bf16 for the product with the values (2^-8 of each; their sum takes them unrounded).
//
// Both products are formed transposed: keys (16) are the rows of K q^T and channels those of V^T p^T, with
// 8 query heads as columns, so that no row of a product is idle where few heads share a key head. A
// register transposition (movmatrix) takes the weights from one to the other.
//
// 8-bit caches: the products run on the codes, the key's scale multiplies the score, the value's scale
// the weight.
//   int8 scores need no conversion of codes: a query becomes s (256 h + l) with int8 digits h and l, off by
//   at most 1 / 65278 of its row's largest magnitude (half a step of 1 / 32639), and the integer sums are
//   exact. A row below 2^-100 counts as 0.
//   e4m3 scores: codes to f16, which holds every code, with the query row times a power of two in f16 (off
//   by at most 2^-25 of the row's largest magnitude). The 8-bit float product is no help here: it measured
//   as many instructions as the conversion.
//   Values become f16, and the weights are rounded to f16 as p * (value scale / largest magnitude of a value
//   scale so far) * 2^11, relative to 2^-11 down to 2^-25 of the largest and to 2^-36 of it below. Scales may
//   be any finite numbers, of either sign.
// Converting codes to bf16 instead kept the ALU pipe at 58 % and memory at 3.1 TB/s.
//
// Bound by HBM, or nearly: 64 sequences of 64 to 4096 keys, 32 / 8 heads of 128, bf16: 51.1 us, 5.2 TB/s; 2 of 100001 to 131072,
// int8: 88.9 us, 5.8 TB/s; 160 of 256 to 8192, 64 / 8 heads, e4m3: 152.9 us, 5.3 TB/s (at full clock 142.6; DRAM at 73 %, ALU pipe at
// 50 %). Medians, timed in turn with a plain sum over as many bytes, which takes 48.0, 94.5 and 141.4 us. More than 8 heads a key
// head over 8-bit caches are bound by the products' latency (16 heads of 128: 3.6 to 4.1 TB/s).
#include <math.h>

#include <string>

#include "common.cuh"
#include "internal.h"
#include "kv_cache.cuh"

namespace mb {
namespace paged {

constexpr int kWarps = 4;                   // that compute; one more loads
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kRows = 16;                   // query rows of a unit
constexpr int kMaxBlocksPerSm = 4;
constexpr int kTileKeys = 16 * kWarps;
constexpr int kCluster = 8;
constexpr float kSlack = 4.f;               // log2 of how far a weight may pass 1
constexpr float kWeightOne = 2048.f;        // f16 form of a weight of 1 with the largest value scale: 2^15 at most
constexpr float kLeastScale = 2.407412430484045e-35f;  // 2^-115: smaller value scales count as this, so that kWeightOne over
                                                       // the largest is finite (2^126 at most)

// Cost of a tile. A unit costs Shape::UNIT_COST besides its tiles (queries, joining the warps, output), more beside the
// smaller tiles of an 8-bit cache. Without it blocks with many short units end last: 64 sequences up to 4096, bf16, cost
// 0 / 3 / 6 / 12: 55.4 / 51.3 / 51.6 / 52.8 us; 160 up to 8192, e4m3, 8 / 12 / 16: 146 / 143 / 143 us; 512 of 30 to 600, int8,
// 8 / 16 / 24: 111 / 104 / 105 us; others lose past 16.
constexpr int kTileCost = 4;

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
  int box;  // 16-key groups of a tile that one copy brings: 1, 2 or 4, as a page holds them
  float scale_log2;
  __nv_bfloat16* out;
  int64_t ldo;
  Part* parts;       // [units]
  float *part_ml;    // [2 * blocks][2][kRows]
  float *part_o;     // [2 * blocks][kRows][D]
  int blocks;        // that the workspace has room for
  int* status;
};

MB_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
MB_DEV void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

MB_DEV void mma16816_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
MB_DEV void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrives once the thread's copies so far are there.
MB_DEV void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A float of another block of the cluster, at the place of p in this one.
MB_DEV float ld_cluster(const float* p, int rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(smem_in_cta(p, rank)) : "memory");
  return x;
}
// 32 channels of int8 codes; exact.
MB_DEV void mma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held as row g, columns 2t and 2t + 1 a lane.
MB_DEV uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// 16 keys x 32 channels of codes, transposed: r[2 i + j] holds, for channel 16 i + 8 j + g, keys 4t .. 4t + 3.
MB_DEV void ldmatrix_b8_x2_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// The four codes of a word as two f16 pairs, exactly. int8: byte c + 128 under the exponent of 1024 is 1152 + c.
template <int CODES>
MB_DEV void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (CODES == MB_KV_I8) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*(const __half2*)&a, off), y = __hsub2(*(const __half2*)&b, off);
    lo = *(const uint32_t*)&x, hi = *(const uint32_t*)&y;
  } else {
    asm("{\n .reg .b16 x, y;\n mov.b32 {x, y}, %2;\n cvt.rn.f16x2.e4m3x2 %0, x;\n cvt.rn.f16x2.e4m3x2 %1, y;\n}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// Four neighbouring channels of a query row (bf16 pairs x, y) as a word of high and one of low digits; `f` brings the
// row's largest magnitude to 32639.
MB_DEV void query_digits(uint2 x, float f, uint32_t& h, uint32_t& l) {
  const float q[4] = {bf16_lo(x.x) * f, bf16_hi(x.x) * f, bf16_lo(x.y) * f, bf16_hi(x.y) * f};
  h = l = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int v = __float2int_rn(q[i]), hi = (v + 128) >> 8;  // low digit in [-128, 127]
    h |= ((uint32_t)hi & 255u) << (8 * i);
    l |= ((uint32_t)v & 255u) << (8 * i);
  }
}
MB_DEV uint32_t scaled_f16x2(uint32_t x, float f) {
  const __half2 h = __floats2half2_rn(bf16_lo(x) * f, bf16_hi(x) * f);
  return *(const uint32_t*)&h;
}

// A tile's place in shared memory and how its rows are read. A row of 256 bytes lies in two planes of 128-byte
// lines; shorter rows share or fill a line. The swizzle moves 16-byte pieces inside a line by its number mod 8.
template <int CODES, int D, bool WIDE>
struct Shape {
  static constexpr int EB = CODES == MB_KV_BF16 ? 2 : 1;
  static constexpr int ROWB = D * EB;                             // bytes of a row
  static constexpr int PLANES = ROWB / 128 > 1 ? ROWB / 128 : 1;
  static constexpr int LINEB = ROWB < 128 ? ROWB : 128;           // bytes of a row in a line
  static constexpr int GROUPB = 16 * LINEB;                       // 16 keys in a plane
  static constexpr int PLANEB = kTileKeys * LINEB;
  static constexpr int KVB = PLANES * PLANEB;
  static constexpr int SCALEB = CODES == MB_KV_BF16 ? 0 : kTileKeys * 4;
  static constexpr int STAGEB = 2 * KVB + (2 * SCALEB + 1023) / 1024 * 1024;
  static constexpr int ROWS = WIDE ? 16 : 8;        // query rows that are kept
  static constexpr int QB = ROWS * D * 2;
  static constexpr int QSLOTS = WIDE ? 1 : 2;
  static constexpr int QW = D / 16;                 // four-channel groups of a row that a lane holds
  static constexpr int NR = WIDE ? 2 : 4;           // 16-channel output tiles that are merged at a time
  static constexpr int MERGE_PITCH = NR * 16 + 4;   // floats; rows 2t begin 8 banks apart
  static constexpr int MERGEB = kWarps * ROWS * MERGE_PITCH * 4;
  static constexpr int UNIT_COST = CODES == MB_KV_BF16 ? 3 : 12;
  // Blocks on an SM, as many as registers allow where there is little arithmetic in flight: 64 sequences of 8000, 8 key heads of
  // 64, int8: 114 us with 3, 108 with 4 (4 heads a key head); 168 with 2, 157 with 3 (16). Heads of 128 spill instead (16:
  // 148 us with 2, 193 with 3).
  static constexpr int BLOCKS = CODES == MB_KV_BF16 ? 2 : D == 64 ? (WIDE ? 3 : 4) : (WIDE ? 2 : 3);
  static constexpr int kBudget = (228 / BLOCKS - 2) * 1024;  // of a block: 1 KB is the system's, 1 KB for alignment
  static constexpr int kFixed = QSLOTS * QB + MERGEB + 2 * kWarps * kRows * 4 + 1024;  // and barriers, descriptors
  static constexpr int STAGES = (kBudget - kFixed) / STAGEB < 8 ? (kBudget - kFixed) / STAGEB : 8;
  static constexpr size_t kSmem = 1024 + (size_t)STAGES * STAGEB + kFixed;
  static_assert(STAGES >= 2, "ring too short");

  // cost of a unit of nt tiles; tiles of the unit at `at` that begin before x
  static MB_DEV int64_t unit_cost(int64_t nt) { return nt > 0 ? UNIT_COST + kTileCost * nt : 0; }
  static MB_DEV int tiles_before(int64_t at, int64_t nt, int64_t x) {
    const int64_t n = (x - at - UNIT_COST + kTileCost - 1) / kTileCost;
    return x <= at + UNIT_COST ? 0 : (int)(n < nt ? n : nt);
  }
  static MB_DEV uint32_t at(int key, int byte) {  // of a row's byte in K or V, swizzled
    const uint32_t off = (uint32_t)(key * LINEB + (byte & 127));
    return (uint32_t)(byte >> 7) * PLANEB + (off ^ ((off >> 3) & 0x70));
  }
  // first channel of group w of the four-channel groups that lane t holds of a row
  static MB_DEV int q_channel(int w, int t) {
    return CODES == MB_KV_BF16 ? (w / 4) * 64 + t * 16 + (w & 3) * 4 : t * (D / 4) + w * 4;
  }
  // The key of a warp's 16 that is row 8 u + j of the scores. Values of 8-bit types come as keys 4t .. 4t + 3 a lane,
  // so the weights have to as well.
  static MB_DEV int key_of(int u, int j) {
    return CODES == MB_KV_BF16 ? u * 8 + j : (j >> 1) * 4 + u * 2 + (j & 1);
  }
};

// What the loading warp says of a stage.
struct Desc {
  int left;         // keys of the tile that exist
  int groups;       // bit i: its 16 keys from 16 i on are there
  int q_slot;       // the unit's first tile in this run: where its queries are; else -1
  int last;         // the unit's last tile in this run
  int seq, unit;
  int slot;         // last: workspace slot for the part; -1: the unit is whole
  int end;          // the block's last tile
};

// Where block c of n begins in the row of units; a tile is done by the block in whose run its cost begins.
MB_DEV int64_t run_start(int64_t total, int c, int n) { return total * c / n; }
MB_DEV int run_owner(int64_t total, int64_t at, int n) { return (int)(((at + 1) * n - 1) / total); }

// CLUSTER: kCluster blocks share one unit, evenly, and join in their shared memory; no workspace, no second launch.
template <int CODES, int D, bool WIDE, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, Shape<CODES, D, WIDE>::BLOCKS)
    k_attention_paged(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const Params p) {
  using S = Shape<CODES, D, WIDE>;
  constexpr int QW = S::QW, STAGES = S::STAGES;
  constexpr int RR = WIDE ? 2 : 1;  // eights of query rows
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* part = (float*)smem;  // CLUSTER, once all tiles are done: [ROWS][D] outputs, [ROWS] maxima, [ROWS] sums
  uint8_t* s_q = smem + (size_t)STAGES * S::STAGEB;
  float* s_merge = (float*)(s_q + S::QSLOTS * S::QB);
  float* s_m = s_merge + S::MERGEB / 4;  // [kWarps][kRows]
  float* s_l = s_m + kWarps * kRows;
  uint64_t* full = (uint64_t*)(s_l + kWarps * kRows);  // [STAGES]
  uint64_t* empty = full + 8;                          // [STAGES]
  uint64_t* q_empty = empty + 8;                       // [S::QSLOTS]
  uint64_t* merge_bar = q_empty + S::QSLOTS;
  int64_t* s_sum = (int64_t*)(merge_bar + 1);          // [kWarps + 1]
  int64_t* s_at = s_sum + kWarps + 1;                  // tiles before the run's first sequence
  Desc* desc = (Desc*)(s_at + 1);                      // [STAGES]
  float* s_v = (float*)(desc + 8);                     // [kWarps]
  int* s_seq = (int*)(s_v + kWarps);
  volatile int* abort_flag = s_seq + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t cap = (int64_t)p.table_width << p.c.page_log2;
  const int U = p.units_per_seq;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&full[i], CODES == MB_KV_BF16 ? 1 : 33);  // and 32 lanes' copies of scales
      mbar_init(&empty[i], kWarps);
    }
    for (int i = 0; i < S::QSLOTS; i++) mbar_init(&q_empty[i], kWarps);
    mbar_init(merge_bar, kWarps);
    *abort_flag = 0;
    *s_seq = -1;
    fence_mbar_init();
  }
  wait_before();
  auto length = [&](int b) -> int64_t {
    if (b >= p.n_seqs) return 0;
    const int64_t n = p.lens[b];
    return n < 0 ? 0 : n < cap ? n : cap;
  };
  auto tiles_of = [&](int64_t len) { return (len + kTileKeys - 1) / kTileKeys; };
  // The run: from position x0 to x1 of a row of units of cost `total`, first unit (b, unit) at `at`.
  const int c = blockIdx.x;
  int b, unit, n_blocks = 1;
  int64_t len, nt, at = 0, x0, x1, total = 0;
  const int rank = CLUSTER ? (int)cluster_rank() : 0;
  if constexpr (CLUSTER) {
    const int u = c / kCluster;
    b = u / U, unit = u - b * U;
    len = length(b), nt = tiles_of(len);
    total = S::unit_cost(nt);
    const int64_t first = nt * rank / kCluster, end = nt * (rank + 1) / kCluster;
    x0 = S::UNIT_COST + kTileCost * first, x1 = first < end ? S::UNIT_COST + kTileCost * end : x0;
    __syncthreads();  // the barriers are initialised
  } else {
    // cost of sequences base .. base + threadIdx.x together (block-wide), and of all kThreads
    auto scan = [&](int base, int64_t& all) {
      int64_t x = S::unit_cost(tiles_of(length(base + (int)threadIdx.x))) * U;
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
      for (int w = 0; w <= kWarps; w++) {
        if (w < warp) x += s_sum[w];
        all += s_sum[w];
      }
      return x;
    };

    int64_t all, incl = 0;
    for (int base = 0; base < p.n_seqs; base += kThreads) {
      incl = scan(base, all);
      total += all;
    }
    // sequences without positions: their rows are 0
    for (int b = c; b < p.n_seqs; b += gridDim.x)
      if (length(b) == 0)
        for (int i = threadIdx.x; i < p.H * D / 8; i += kThreads) *((uint4*)(p.out + b * p.ldo) + i) = make_uint4(0, 0, 0, 0);
    // A run is a tile's cost at least, so that every block between a unit's first and last holds a piece of it.
    n_blocks = (int)(total / kTileCost < gridDim.x ? total / kTileCost : gridDim.x);
    if (c >= n_blocks) return;
    x0 = run_start(total, c, n_blocks), x1 = run_start(total, c + 1, n_blocks);
    int64_t before = 0;
    for (int base = 0; base < p.n_seqs; base += kThreads) {
      if (p.n_seqs > kThreads) incl = scan(base, all); else all = total;
      const int64_t own = S::unit_cost(tiles_of(length(base + (int)threadIdx.x))) * U;
      const int64_t end = before + incl;
      if (x0 < end && x0 >= end - own) *s_seq = base + threadIdx.x, *s_at = end - own;
      before += all;
      if (x0 < before) break;
    }
    __syncthreads();
    // the first unit of the run, and whether any tile begins in it
    b = *s_seq;
    if (b < 0) return;  // here and below: lengths that changed under the call
    len = length(b), nt = tiles_of(len), at = *s_at;
    if (nt == 0) return;
    unit = (int)((x0 - at) / S::unit_cost(nt));
    if (unit >= U) return;
    at += unit * S::unit_cost(nt);
    if (S::tiles_before(at, nt, x0) >= S::tiles_before(at, nt, x1) &&
        (at + S::unit_cost(nt) >= total || at + S::unit_cost(nt) + S::UNIT_COST >= x1))
      return;
  }

  if (warp == kWarps) {
    // ---------------------------------------------------------------- loads
    if (lane == 0) {
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
    }
    int n_seg = 0, it = 0;
    bool ok = true;
    while (ok && at + S::UNIT_COST < x1) {
      const int kt0 = S::tiles_before(at, nt, x0), kt1 = S::tiles_before(at, nt, x1);
      const int64_t next_at = at + S::unit_cost(nt);
      const bool end = next_at >= total || next_at + S::UNIT_COST >= x1;
      const int hk = unit / p.q_tiles, qt = unit - hk * p.q_tiles;
      const int rows = min(kRows, p.G - qt * kRows);
      const bool whole = kt0 == 0 && kt1 == nt;
      const int32_t* table = p.table + (int64_t)b * p.ld_table;
      if (!CLUSTER && kt0 == 0 && kt1 > 0 && lane == 0) {
        Part part;
        part.first = c;
        part.pieces = whole ? 1 : run_owner(total, at + S::UNIT_COST + kTileCost * (nt - 1), n_blocks) - c + 1;
        p.parts[(int64_t)b * U + unit] = part;
      }
      const int qs = n_seg % S::QSLOTS;
      int64_t row32 = -1;  // cache row of 16-key group lane of the next 32
      for (int kt = kt0; kt < kt1 && ok; kt++, it++) {
        const int64_t key0 = (int64_t)kt * kTileKeys;
        const int left = (int)min(len - key0, (int64_t)kTileKeys);
        const int ahead = (kt - kt0) % (32 / kWarps) * kWarps;  // this tile's first group among them
        if (ahead == 0) {
          const int64_t k32 = key0 + lane * 16;
          row32 = kt + lane / kWarps < kt1 && k32 < len ? kv::row_of(p.c, table, p.table_width, k32, hk, p.status) : -1;
        }
        const unsigned groups = (__ballot_sync(0xffffffffu, row32 >= 0) >> ahead) & ((1u << kWarps) - 1);
        const int s = it % STAGES;
        if (!(ok = mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, p.status, kDevTimeoutAttn))) break;
        if (kt == kt0 &&
            !(ok = mbar_wait(&q_empty[qs], ((n_seg / S::QSLOTS) & 1) ^ 1, abort_flag, p.status, kDevTimeoutAttn)))
          break;
        uint8_t* st = smem + (size_t)s * S::STAGEB;
        const uint32_t q_bytes = kt == kt0 ? (uint32_t)(rows * D * 2) : 0u;
        if (lane == 0) {
          Desc d;
          d.left = left;
          d.groups = (int)groups;
          d.q_slot = kt == kt0 ? qs : -1;
          d.last = kt == kt1 - 1;
          d.seq = b;
          d.unit = unit;
          d.slot = whole ? -1 : 2 * c + (kt0 == 0 ? 1 : 0);
          d.end = d.last && end;
          desc[s] = d;
          const unsigned firsts = p.box == 4 ? 1 : p.box == 2 ? 5 : 15;  // groups that begin a box
          mbar_expect_tx(&full[s], __popc(groups & firsts) * p.box * 2u * 16 * S::ROWB + q_bytes);
        }
        __syncwarp();
        // lane 8 i + j: copy j of the box that begins with group i (planes of K, planes of V); keys of a
        // page behind the sequence's end come along
        const int gi = lane >> 3, j = lane & 7;
        const int64_t grow = __shfl_sync(0xffffffffu, row32, ahead + gi);
        if (grow >= 0 && (gi & (p.box - 1)) == 0) {
          if (j < 2 * S::PLANES) {
            const int plane = j % S::PLANES;
            const bool is_v = j >= S::PLANES;
            uint8_t* dst = st + (is_v ? S::KVB : 0) + plane * S::PLANEB + gi * S::GROUPB;
            // rows shorter than a line lie two to a line of the map
            tma_load_2d(dst, is_v ? &tv : &tk, &full[s], plane * 128, (int)(grow * S::LINEB / 128));
          }
        }
        if (CODES != MB_KV_BF16) {
          // scales: 16 bytes a lane of K (0-15) or V. Bulk copies of 64 bytes took as long to issue as those of the rows.
          const int i = lane & 15;
          const int64_t from = __shfl_sync(0xffffffffu, row32, ahead + (i >> 2));
          if (from >= 0)
            cp_async16(st + 2 * S::KVB + (lane >> 4) * S::SCALEB + i * 16,
                       (lane >> 4 ? p.c.v_scale : p.c.k_scale) + from + (i & 3) * 4);
          cp_async_arrive(&full[s]);
        }
        if (lane == 31 && q_bytes)
          bulk_load(s_q + qs * S::QB, p.q + (int64_t)b * p.ldq + (int64_t)(hk * p.G + qt * kRows) * D, q_bytes, &full[s]);
      }
      n_seg += kt0 < kt1;
      at = next_at;
      if (++unit == U) {  // next sequence that has tiles
        unit = 0;
        do {
          len = length(++b);
          nt = tiles_of(len);
        } while (nt == 0 && b < p.n_seqs);
        if (b >= p.n_seqs) break;
      }
    }
    // the block's memory must outlive its copies, whatever the other warps do
    volatile int never = 0;
    for (int i = it < STAGES ? 0 : it - STAGES; i < it; i++)
      mbar_wait(&full[i % STAGES], (i / STAGES) & 1, &never, p.status, kDevTimeoutAttn);
  } else if (x0 < x1) {
    // ---------------------------------------------------------------- products
    // Query operand of row 8 r + g, by four-channel groups: two pairs (bf16; f16 for e4m3), or a high and a low digit word
    // (int8); and what brings the scores of rows 8 r + 2t and + 1 back to size, times log2(e).
    constexpr bool B16 = CODES == MB_KV_BF16, I8 = CODES == MB_KV_I8;
    uint32_t qa[RR][QW][2];
    float q_size[RR][2];
    // o: channels 16 i + g (0, 1) and + 8 (2, 3) of rows 8 r + 2t and + 1; m, l: of these rows
    float o[RR][D / 16][4], m[RR][2], l[RR][2];
    float v_ref = 0.f, v_inv = 0.f;  // 8-bit: largest magnitude of a value scale so far, and kWeightOne over it
    uint32_t merges = 0;
    for (int it = 0;; it++) {
      const int s = it % STAGES;
      if (!mbar_wait(&full[s], (it / STAGES) & 1, abort_flag, p.status, kDevTimeoutAttn)) break;
      const Desc d = desc[s];
      uint8_t* sk = smem + (size_t)s * S::STAGEB;
      uint8_t* sv = sk + S::KVB;
      if (d.q_slot >= 0) {
        const int rows = min(kRows, p.G - (d.unit % p.q_tiles) * kRows);
#pragma unroll
        for (int r = 0; r < RR; r++) {
          const bool have = g + 8 * r < rows;
          const uint8_t* src = s_q + d.q_slot * S::QB + (g + 8 * r) * D * 2;
          uint32_t top = 0;  // largest magnitude's bits: non-negative floats order like integers, NaN last
#pragma unroll
          for (int i = 0; i < QW; i++) {
            uint2 x = make_uint2(0, 0);
            if (have) x = *(const uint2*)(src + S::q_channel(i, t) * 2);
            qa[r][i][0] = x.x, qa[r][i][1] = x.y;
            if (!B16) {
              top = max(top, max((x.x << 16) & 0x7fff0000u, (x.y << 16) & 0x7fff0000u));
              top = max(top, max(x.x & 0x7fff0000u, x.y & 0x7fff0000u));
            }
          }
          float back = 1.f;
          if (!B16) {
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float f;
            if (I8) {
              // below 2^-100 the row counts as 0
              const bool some = top >= 0x0d800000u;
              f = some ? 32639.f / __uint_as_float(top) : 0.f;
              back = some ? __uint_as_float(top) / 32639.f : 0.f;
            } else {  // to [1, 2) by a power of two
              const int e = min(max((int)(top >> 23), 1), 253);
              f = __uint_as_float((uint32_t)(254 - e) << 23);
              back = __uint_as_float((uint32_t)e << 23);
            }
            if (top >= 0x7f800000u) f = 0.f, back = __uint_as_float(0x7fc00000u);  // NaN or infinity in the row
#pragma unroll
            for (int i = 0; i < QW; i++) {
              if (I8) {
                uint32_t h, w;
                query_digits(make_uint2(qa[r][i][0], qa[r][i][1]), f, h, w);
                qa[r][i][0] = h, qa[r][i][1] = w;
              } else {
                qa[r][i][0] = scaled_f16x2(qa[r][i][0], f), qa[r][i][1] = scaled_f16x2(qa[r][i][1], f);
              }
            }
          }
          back *= p.scale_log2;
          q_size[r][0] = __shfl_sync(0xffffffffu, back, 8 * t), q_size[r][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
          for (int i = 0; i < D / 16; i++) o[r][i][0] = o[r][i][1] = o[r][i][2] = o[r][i][3] = 0.f;
          m[r][0] = m[r][1] = -INFINITY, l[r][0] = l[r][1] = 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[d.q_slot]);
        v_ref = v_inv = 0.f;
      }
      const int key0 = warp * 16;
      if ((d.groups >> warp) & 1) {
        const int left = d.left - key0;  // of this warp's 16 keys; > 0
        // 8-bit values are read ahead of the scores, whose latency hides theirs; where 16 rows leave no registers for
        // them, when their turn comes
        uint32_t vw[B16 ? 1 : D / 32][4];
        auto load_v = [&](int i) {
          ldmatrix_b8_x2_trans(smem_u32(sv + S::at(key0 + (lane & 15), (2 * i + (lane >> 4)) * 16)), vw[B16 ? 0 : i]);
        };
        if (!B16 && !WIDE) {
#pragma unroll
          for (int i = 0; i < D / 32; i++) load_v(i);
        }
        // scores: sc[r][2 u + e] of key key_of(u, g) and row 8 r + 2t + e
        const int key_a = S::key_of(0, g), key_b = S::key_of(1, g);
        float sc[RR][4];
        int hi[RR][4], lo[RR][4];
#pragma unroll
        for (int r = 0; r < RR; r++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[r][e] = 0.f, hi[r][e] = lo[r][e] = 0;
        constexpr int LB = S::LINEB / 4;  // a lane's bytes of a row in a line
#pragma unroll
        for (int pl = 0; pl < S::PLANES; pl++) {
          uint32_t wa[LB / 4], wb[LB / 4];
#pragma unroll
          for (int i = 0; i < LB / 16; i++) {
            const uint4 x = *(const uint4*)(sk + S::at(key0 + key_a, pl * 128 + t * LB + i * 16));
            const uint4 y = *(const uint4*)(sk + S::at(key0 + key_b, pl * 128 + t * LB + i * 16));
            wa[4 * i] = x.x, wa[4 * i + 1] = x.y, wa[4 * i + 2] = x.z, wa[4 * i + 3] = x.w;
            wb[4 * i] = y.x, wb[4 * i + 1] = y.y, wb[4 * i + 2] = y.z, wb[4 * i + 3] = y.w;
          }
          if (CODES == MB_KV_E4M3) {
#pragma unroll
            for (int i = 0; i < LB / 4; i++) {
              uint32_t a[4];
              codes_f16<CODES>(wa[i], a[0], a[2]);
              codes_f16<CODES>(wb[i], a[1], a[3]);
#pragma unroll
              for (int r = 0; r < RR; r++) mma16816_f16(sc[r], a[0], a[1], a[2], a[3], qa[r][i][0], qa[r][i][1]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < LB / 8; i++)
#pragma unroll
              for (int r = 0; r < RR; r++) {
                if (B16) {
                  const uint32_t* q = qa[r][B16 ? pl * 4 + i : 0];
                  mma16816(sc[r], wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], q[0], q[1]);
                } else {
                  const int x = B16 ? 0 : 2 * i, y = B16 ? 0 : 2 * i + 1;
                  mma16832(hi[r], wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], qa[r][x][0], qa[r][y][0]);
                  mma16832(lo[r], wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], qa[r][x][1], qa[r][y][1]);
                }
              }
          }
        }
        // scales of the two keys; those of rows that do not exist may be anything
        const bool in_a = key_a < left, in_b = key_b < left;
        float ks_a = 1.f, ks_b = 1.f, vs_a = 1.f, vs_b = 1.f;
        if (!B16) {
          const float* scale = (const float*)(sk + 2 * S::KVB) + key0;
          ks_a = scale[key_a], ks_b = scale[key_b];
          vs_a = in_a ? scale[kTileKeys + key_a] : 0.f, vs_b = in_b ? scale[kTileKeys + key_b] : 0.f;
        }
        // The reference points move (and the output with them) only when a score passes its row's by more than 2^kSlack,
        // or a value scale's magnitude the largest so far.
        bool move = !B16 && fmaxf(fabsf(vs_a), fabsf(vs_b)) > v_ref;
#pragma unroll
        for (int r = 0; r < RR; r++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            if (I8) {  // below 2^30
              sc[r][e] = (float)(hi[r][e] * 256 + lo[r][e]);
              sc[r][2 + e] = (float)(hi[r][2 + e] * 256 + lo[r][2 + e]);
            }
            sc[r][e] = in_a ? sc[r][e] * (ks_a * q_size[r][e]) : -INFINITY;
            sc[r][2 + e] = in_b ? sc[r][2 + e] * (ks_b * q_size[r][e]) : -INFINITY;
            move |= fmaxf(sc[r][e], sc[r][2 + e]) > m[r][e] + kSlack;
          }
        if (__any_sync(0xffffffffu, move)) {
          float shrink = 1.f;
          if (!B16) {
            float vm = fmaxf(fabsf(vs_a), fabsf(vs_b));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, x));
            if (vm > v_ref) {  // the same in all lanes
              vm = fmaxf(vm, kLeastScale);
              shrink = v_ref / vm;
              v_ref = vm;
              v_inv = kWeightOne / vm;
            }
          }
#pragma unroll
          for (int r = 0; r < RR; r++) {
            float alpha[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float mx = fmaxf(sc[r][e], sc[r][2 + e]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
              const float mn = mx > m[r][e] + kSlack ? mx : m[r][e];
              alpha[e] = mn == -INFINITY ? 1.f : ex2_approx(m[r][e] - mn);
              m[r][e] = mn;
              l[r][e] *= alpha[e];
              alpha[e] *= shrink;
            }
#pragma unroll
            for (int i = 0; i < D / 16; i++)
              o[r][i][0] *= alpha[0], o[r][i][1] *= alpha[1], o[r][i][2] *= alpha[0], o[r][i][3] *= alpha[1];
          }
        }
        vs_a *= v_inv, vs_b *= v_inv;
        uint32_t w8[RR][2];  // weights as B operand: keys 8 u + 2t and + 1 of row 8 r + g
#pragma unroll
        for (int r = 0; r < RR; r++) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float ref = m[r][e] == -INFINITY ? 0.f : m[r][e];  // nothing but -inf so far: weights 0
            w[e] = ex2_approx(sc[r][e] - ref), w[2 + e] = ex2_approx(sc[r][2 + e] - ref);
            l[r][e] += w[e] + w[2 + e];
          }
          if (B16) {
            w8[r][0] = movmatrix(pack_bf16x2(w[0], w[1])), w8[r][1] = movmatrix(pack_bf16x2(w[2], w[3]));
          } else {
            const __half2 a = __floats2half2_rn(w[0] * vs_a, w[1] * vs_a), b = __floats2half2_rn(w[2] * vs_b, w[3] * vs_b);
            w8[r][0] = movmatrix(*(const uint32_t*)&a), w8[r][1] = movmatrix(*(const uint32_t*)&b);
          }
        }
        if (B16) {
          // values that do not exist may be NaN: zero their rows first (a tile's partial last group only)
          if (left < 16) {
            for (int i = lane; i < (16 - left) * (S::ROWB / 16); i += 32) {
              const int key = key0 + left + i / (S::ROWB / 16);
              *(uint4*)(sv + S::at(key, (i % (S::ROWB / 16)) * 16)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          // one instruction: channels 16 i and 16 i + 8 of keys 0-7, then of keys 8-15
          const int key = key0 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
          for (int i = 0; i < D / 16; i++) {
            uint32_t a0, a1, a2, a3;
            ldmatrix_x4_trans(smem_u32(sv + S::at(key, (2 * i + ((lane >> 3) & 1)) * 16)), a0, a1, a2, a3);
#pragma unroll
            for (int r = 0; r < RR; r++) mma16816(o[r][i], a0, a1, a2, a3, w8[r][0], w8[r][1]);
          }
        } else {
          // a weight of 0 silences codes of rows that do not exist, but for e4m3's NaN: those become 0
#pragma unroll
          for (int i = 0; i < D / 16; i += 2) {
            if (WIDE) load_v(i / 2);
#pragma unroll
            for (int j = 0; j < 2; j++) {
              uint32_t a[4];  // {channels g, g + 8} x {keys 4t, 4t + 1; 4t + 2, 4t + 3}
#pragma unroll
              for (int e = 0; e < 2; e++) {
                uint32_t x = vw[B16 ? 0 : i / 2][2 * j + e];
                if (CODES == MB_KV_E4M3 && left < 16)
                  x &= 4 * t >= left ? 0u : left - 4 * t >= 4 ? 0xffffffffu : (1u << (8 * (left - 4 * t))) - 1u;
                codes_f16<CODES>(x, a[e], a[2 + e]);
              }
#pragma unroll
              for (int r = 0; r < RR; r++) mma16816_f16(o[r][i + j], a[0], a[1], a[2], a[3], w8[r][0], w8[r][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (!d.last) continue;

      // the warps' parts together, NR column tiles at a time
      const int hk = d.unit / p.q_tiles, qt = d.unit - hk * p.q_tiles;
      const int rows = min(kRows, p.G - qt * kRows), head0 = hk * p.G + qt * kRows;
#pragma unroll
      for (int r = 0; r < RR; r++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], x);
          if (g == 0) s_m[warp * kRows + 8 * r + 2 * t + e] = m[r][e], s_l[warp * kRows + 8 * r + 2 * t + e] = l[r][e];
        }
      if (lane == 0) s_v[warp] = B16 ? 1.f : v_ref / kWeightOne;
      bool ok = true;
      auto meet = [&] {  // of the four warps
        __syncwarp();
        if (lane == 0) mbar_arrive(merge_bar);
        ok = ok && mbar_wait(merge_bar, merges & 1, abort_flag, p.status, kDevTimeoutAttn);
        merges++;
      };
#pragma unroll
      for (int i0 = 0; i0 < D / 16; i0 += S::NR) {
#pragma unroll
        for (int i = 0; i < S::NR; i++)
#pragma unroll
          for (int r = 0; r < RR; r++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              s_merge[(warp * S::ROWS + 8 * r + 2 * t + (e & 1)) * S::MERGE_PITCH + i * 16 + g + (e >> 1) * 8] = o[r][i0 + i][e];
        meet();
        if (!ok) break;
        for (int i = threadIdx.x; i < rows * S::NR * 16; i += 32 * kWarps) {
          const int r = i / (S::NR * 16), col = i % (S::NR * 16), ch = i0 * 16 + col;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWarps; w++) top = fmaxf(top, s_m[w * kRows + r]);
          const float ref1 = top == -INFINITY ? 0.f : top;
          float acc = 0.f, sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; w++) {
            const float f = ex2_approx(s_m[w * kRows + r] - ref1);
            acc += f * s_v[w] * s_merge[(w * S::ROWS + r) * S::MERGE_PITCH + col];
            sum += f * s_l[w * kRows + r];
          }
          if (CLUSTER) {
            part[r * D + ch] = acc;
            if (ch == 0) part[S::ROWS * D + r] = top, part[S::ROWS * D + S::ROWS + r] = sum;
          } else if (d.slot < 0) {
            p.out[(int64_t)d.seq * p.ldo + (int64_t)(head0 + r) * D + ch] = __float2bfloat16_rn(acc / sum);
          } else {
            p.part_o[((int64_t)d.slot * kRows + r) * D + ch] = acc;
            if (ch == 0) {
              p.part_ml[(int64_t)d.slot * 2 * kRows + r] = top;
              p.part_ml[(int64_t)d.slot * 2 * kRows + kRows + r] = sum;
            }
          }
        }
        meet();
        if (!ok) break;
      }
      if (!ok || d.end) break;
    }
  }

  if constexpr (CLUSTER) {
    // the unit's parts lie in its blocks' memory; each block joins every eighth row
    __syncwarp();
    cluster_sync();
    const int hk = unit / p.q_tiles, qt = unit - hk * p.q_tiles;
    const int rows = min(kRows, p.G - qt * kRows), head0 = hk * p.G + qt * kRows;
    auto has_tiles = [&](int k) { return nt * k / kCluster < nt * (k + 1) / kCluster; };
    for (int r = rank; r < rows; r += kCluster)
      for (int d = threadIdx.x; d < D; d += kThreads) {
        float top = -INFINITY, m[kCluster], acc = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < kCluster; k++) {
          m[k] = has_tiles(k) ? ld_cluster(part + S::ROWS * D + r, k) : -INFINITY;
          top = fmaxf(top, m[k]);
        }
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int k = 0; k < kCluster; k++)
          if (has_tiles(k)) {
            const float f = ex2_approx(m[k] - ref);
            acc += f * ld_cluster(part + r * D + d, k);
            sum += f * ld_cluster(part + S::ROWS * D + S::ROWS + r, k);
          }
        p.out[(int64_t)b * p.ldo + (int64_t)(head0 + r) * D + d] = __float2bfloat16_rn(nt > 0 ? acc / sum : 0.f);
      }
    __syncwarp();
    cluster_sync();  // no block's memory goes while another reads it
  }
}

// Adds up the parts of each unit that several blocks hold, in the blocks' order; one block for each unit and query row.
constexpr int kJoinWarps = 4;
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) k_join(const Params p) {
  __shared__ float4 s_acc[kJoinWarps][32];
  wait_before();
  const int u = blockIdx.x, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = u / p.units_per_seq, unit = u - b * p.units_per_seq;
  const int hk = unit / p.q_tiles, qt = unit - hk * p.q_tiles;
  if (r >= p.G - qt * kRows || p.table_width == 0) return;
  const int len = p.lens[b];
  const Part part = p.parts[u];
  if (len <= 0 || part.pieces <= 1) return;
  // left by another call where this one gave up a wait, or lengths changed under it
  if (part.first < 0 || part.pieces > p.blocks - part.first) return;
  auto slot = [&](int i) { return (int64_t)2 * (part.first + i) + (i == 0 ? 1 : 0); };
  // every warp the statistics of all parts, 32 at a time
  float top = -INFINITY;
  for (int i = lane; i < part.pieces; i += 32) top = fmaxf(top, p.part_ml[slot(i) * 2 * kRows + r]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int i0 = 0; i0 < part.pieces; i0 += 32) {
    const int n = min(32, part.pieces - i0);
    float f = 0.f;
    if (lane < n) {
      f = ex2_approx(p.part_ml[slot(i0 + lane) * 2 * kRows + r] - ref);
      sum += f * p.part_ml[slot(i0 + lane) * 2 * kRows + kRows + r];
    }
#pragma unroll 8
    for (int i = warp; i < n; i += kJoinWarps) {
      const float w = __shfl_sync(0xffffffffu, f, i);
      if (lane < D / 4) {
        const float4 x = *((const float4*)(p.part_o + (slot(i0 + i) * kRows + r) * D) + lane);
        acc.x += w * x.x, acc.y += w * x.y, acc.z += w * x.z, acc.w += w * x.w;
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  s_acc[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && lane < D / 4) {
#pragma unroll
    for (int w = 1; w < kJoinWarps; w++) {
      const float4 x = s_acc[w][lane];
      acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
    }
    uint2 y;
    y.x = pack_bf16x2(acc.x / sum, acc.y / sum);
    y.y = pack_bf16x2(acc.z / sum, acc.w / sum);
    *((uint2*)(p.out + (int64_t)b * p.ldo + (int64_t)(hk * p.G + qt * kRows + r) * D) + lane) = y;
  }
}

struct Layout {
  int64_t units, blocks;
  size_t ml, o, bytes;  // offsets of the parts' statistics and outputs
};
Layout layout(int n_seqs, int H, int H_kv, int D) {
  Layout a;
  a.units = (int64_t)n_seqs * H_kv * ((H / H_kv + kRows - 1) / kRows);
  a.blocks = (int64_t)num_sms() * kMaxBlocksPerSm;
  a.ml = ((size_t)a.units * sizeof(Part) + 255) / 256 * 256;
  a.o = a.ml + (size_t)a.blocks * 2 * 2 * kRows * sizeof(float);
  a.bytes = a.o + (size_t)a.blocks * 2 * kRows * D * sizeof(float);
  return a;
}

template <int CODES, int D, bool WIDE, bool CLUSTER>
cudaError_t launch_attention(const Params& p, int64_t units, cudaStream_t st) {
  using S = Shape<CODES, D, WIDE>;
  CUtensorMap tk, tv;
  // lines of 128 bytes: rows of 256 bytes as two columns of boxes, rows of 64 two to a line
  const uint64_t inner = S::ROWB < 128 ? 128 : S::ROWB;
  const uint64_t rows = ((uint64_t)p.c.n_pages * p.c.heads << p.c.page_log2) * S::ROWB / inner;
  for (int i = 0; i < 2; i++)
    if (!make_tmap_2d(i ? &tv : &tk, i ? p.c.v : p.c.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, inner, rows, inner, 128,
                      S::GROUPB / 128 * p.box, CU_TENSOR_MAP_SWIZZLE_128B))
      return cudaErrorInvalidValue;
  auto kernel = k_attention_paged<CODES, D, WIDE, CLUSTER>;
  static int attr_done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_done[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem);
    if (e != cudaSuccess) return e;
    attr_done[dev & 63] = 1;
  }
  return launch_close(kernel, dim3((unsigned)(CLUSTER ? units * kCluster : num_sms() * S::BLOCKS)), kThreads, S::kSmem, st,
                      CLUSTER ? kCluster : 1, tk, tv, p);
}

template <int CODES, int D, bool WIDE>
cudaError_t launch(const Params& p, int64_t units, cudaStream_t st) {
  using S = Shape<CODES, D, WIDE>;
  const int64_t keys = (int64_t)p.table_width << p.c.page_log2;  // at most, of a sequence
  // Few units of a few tiles a block: their parts meet inside a cluster instead of in a second launch. bf16, in a graph:
  // one sequence of 700, 28/4 heads, 7.1 us against 10.0; eight of 4000 13.6 against 16.3; one of 4000, 32/8 heads, 11.8
  // against 11.5, where 64 blocks leave SMs idle. More or longer ones want all SMs, and the even cut.
  if (keys > kTileKeys && keys <= 8 * kCluster * kTileKeys && units * kCluster <= (int64_t)num_sms() * S::BLOCKS)
    return launch_attention<CODES, D, WIDE, true>(p, units, st);
  cudaError_t e = launch_attention<CODES, D, WIDE, false>(p, units, st);
  // a unit that fits a tile is never split
  if (e != cudaSuccess || keys <= kTileKeys) return e;
  return launch_close(k_join<D>, dim3((unsigned)units, (unsigned)(p.G < kRows ? p.G : kRows)), 32 * kJoinWarps, 0, st, 1, p);
}

template <int CODES, int D>
cudaError_t launch(const Params& p, int64_t units, cudaStream_t st) {
  return p.G > 8 ? launch<CODES, D, true>(p, units, st) : launch<CODES, D, false>(p, units, st);
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
  MB_CHECK(scale >= 0.f && scale <= 2.3e38f, MB_ERR_INVALID, "scale must be positive, at most 2.3e38 (0: 1 / sqrt(D))");
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
  // 8-bit: with 16 keys a copy the loading warp was behind (64 sequences of 8000, heads of 64, 162 us against 116). bf16 has
  // twice the bytes in a copy, and would read keys behind the end for nothing (64 sequences of 64 to 4096: 50.7 against 52.1).
  p.box = cache->dtype == MB_KV_BF16 ? 1 : cache->page_size >= paged::kTileKeys ? 4 : cache->page_size / 16;
  p.scale_log2 = (float)((scale > 0.f ? (double)scale : 1.0 / sqrt((double)D)) * 1.4426950408889634);
  p.out = (__nv_bfloat16*)out;
  p.ldo = ldo;
  p.parts = (paged::Part*)workspace;
  p.part_ml = (float*)((char*)workspace + a.ml);
  p.part_o = (float*)((char*)workspace + a.o);
  p.blocks = (int)a.blocks;
  p.status = device_status_ptr();
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (D == 64)
    e = cache->dtype == MB_KV_BF16 ? paged::launch<MB_KV_BF16, 64>(p, a.units, st)
        : cache->dtype == MB_KV_I8 ? paged::launch<MB_KV_I8, 64>(p, a.units, st)
                                   : paged::launch<MB_KV_E4M3, 64>(p, a.units, st);
  else
    e = cache->dtype == MB_KV_BF16 ? paged::launch<MB_KV_BF16, 128>(p, a.units, st)
        : cache->dtype == MB_KV_I8 ? paged::launch<MB_KV_I8, 128>(p, a.units, st)
                                   : paged::launch<MB_KV_E4M3, 128>(p, a.units, st);
  MB_CUDA(e);
  return MB_OK;
}

}  // extern "C"
