// K11: attention of packed prompts, causal or not, grouped heads, on tcgen05 + TMEM (sm_100a).
//
// Two blocks on an SM, each working on one 128-row query tile at a time: while one waits for its first
// tiles or writes its output, the other computes (one block with two tiles, K4's layout, left the tensor
// pipe at 32 % on a ragged batch). A block takes over the work of blocks that have not started
// (clusterlaunchcontrol), so that it finds the next tile and loads it under the present one.
//   - A tile's rows are TQ = 128 / G tokens of all G query heads of one key head (row = token * G +
//     head), one TMA box of G heads x TQ tokens: the group shares each K / V block, and a causal tile
//     spans few tokens, so little of its diagonal blocks is masked work.
//   - A tile's sequence and place are found from cu_q by a scan, or in large batches by a search; a sequence's last
//     tiles (the longest under a causal mask) come first.
//   warp 0    next tile; TMA: the Q tile, then 64-key blocks of K and V into rings of their own.
//   warp 1    MMA issuer. S(g) = Q K_g^T goes to one half of the S columns while the softmax works on the
//             other: PV(g), then S(g + 2).
//   warp 2    guards V: a P V product adds 0 * v for every masked key of a block, so in the blocks that a
//             mask or the sequence's end crosses it zeroes rows of other sequences and values that are not
//             finite before the product reads them; rows that may see such a value add it at the end (a
//             slow path that ordinary data never takes).
//   warps 4-7 softmax, one thread a query row (= TMEM lane), as in K4 (attention.cu): 64 scores in
//             registers, P written back over S as bf16 (2^-8 of each weight: the products' type; the sum of
//             weights takes them unrounded), lazy rescale of O. Only blocks that cross a row's limit are masked.
// TMEM (256 columns a block): S [0, 128) in halves of 64, O [128, 128 + D).
//
// Bound by the softmax's chain on one thread a row (its exponentials alone take the tensor core's time)
// and, in long runs, by the board's power. One prompt of 8201 tokens, 32 / 8 heads of 128: 547 us, 1008 TFLOP/s
// (0.61 of the measured burst rate; at full clock 478 us); 24 prompts of 32 to 2048 tokens: 213 us (184). Heads of 64, one
// prompt of 8201: 401 us. Measured and not kept: two softmax
// groups on alternate blocks (568 against 542 us on the long prompt: 16 softmax warps slow the issuer),
// 128-key score products with two groups (607 us: one S buffer), K4's share of polynomial exponentials
// (618 against 556 us), the output by TMA (no stage is free under the next tile's loads), a tile's output after
// the next one's first softmax (220 against 209 us on the 24).
#include <math.h>

#include <string>

#include "attn_util.cuh"
#include "common.cuh"
#include "internal.h"

namespace mb {
namespace varlen {
using namespace attn;

constexpr int BKV = 64;
constexpr int kThreads = 256;
constexpr int kK = 2, kV = 3;  // ring lengths: a V block stays until its P V product, a softmax later
constexpr float kRescaleThreshold = 8.f;

struct Params {
  const int32_t *cu_q, *cu_k;
  int n_seqs;
  int64_t total_q, total_k;
  int Hkv, G, TQ, causal;
  unsigned blocks;
  float scale_log2;
  const __nv_bfloat16* v;
  int64_t ldv;
  __nv_bfloat16* out;
  int64_t ldo;
  bool wide_out;  // rows of out begin at multiples of 32 bytes
  int* status;
};

MB_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
MB_DEV float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 32 bytes of an output row. Each thread has a row of its own, so every piece is in another line: stores of 32 bytes (24
// prompts of 32 to 2048 tokens, 220 us with 16 bytes -> 209), or of 16 where rows begin at odd multiples of 16. Exchanging
// pieces between lanes for longer runs of a row gained no more.
MB_DEV void store_row(__nv_bfloat16* to, const uint32_t (&x)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]),
                 "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                 : "memory");
  } else {
    *(uint4*)to = make_uint4(x[0], x[1], x[2], x[3]);
    *(uint4*)(to + 8) = make_uint4(x[4], x[5], x[6], x[7]);
  }
}
MB_DEV bool finite_bf16(uint32_t bits) { return (bits & 0x7f80u) != 0x7f80u; }

// A tile, as warp 0 tells the others.
struct Work {
  int valid;             // 0: there is none left
  int hk;                // key head
  int q_start, k_start;  // first packed row of the sequence
  int m, n;              // queries, keys
  int tok0;              // first token of the tile
};
constexpr int kWorkReaders = 6;  // MMA issuer, guard and four softmax warps

// A tile is found in one of two ways. Up to kFewSeqs sequences, find_work adds up the tiles of the sequences before it. Each
// search passes over all of those, so the time would grow with the square of their number; from there on find_slot searches in
// steps of 32, over slots of which some are without a tile. 32 / 8 heads of 128, prompts of 16 to 64 tokens, sums / slots:
// 64 prompts 15.4 / 17.7 us, 128 29.2 / 28.2, 192 49.2 / 39.5, 256 72.8 / 51.8, 4096 by slots 813; 128 of 16 to 512 tokens
// 215 / 223.
constexpr int kFewSeqs = 128;
constexpr int kMostPassed = 64;  // slots without a tile, one after the other, until a block ends

// Sequence and tile of item `idx` (counting each sequence's tiles of `span` tokens); false behind the last. With offsets
// that overlap the sums may wrap; a tile outside its sequence is none.
MB_DEV bool find_work(const Params& p, int idx, int span, Work& w) {
  const int lane = threadIdx.x & 31;
  auto clampq = [&](int x) { return max(0, min(x, (int)p.total_q)); };
  auto clampk = [&](int x) { return max(0, min(x, (int)p.total_k)); };
#pragma unroll 1
  for (int base = 0; base < p.n_seqs; base += 32) {
    const int b = base + lane;
    int q0 = 0, m = 0, k0 = 0, n = 0;
    if (b < p.n_seqs) {
      q0 = clampq(p.cu_q[b]);
      m = max(0, clampq(p.cu_q[b + 1]) - q0);
      k0 = clampk(p.cu_k[b]);
      n = max(0, clampk(p.cu_k[b + 1]) - k0);
    }
    int x = (m + span - 1) / span;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, idx < x);
    if (hit) {
      const int src = __ffs(hit) - 1;
      w.q_start = __shfl_sync(0xffffffffu, q0, src);
      w.m = __shfl_sync(0xffffffffu, m, src);
      w.k_start = __shfl_sync(0xffffffffu, k0, src);
      w.n = __shfl_sync(0xffffffffu, n, src);
      const int last = __shfl_sync(0xffffffffu, x, src) - 1 - idx;  // last tile first
      w.tok0 = last * span;
      return last >= 0 && last <= (w.m - 1) / span && w.m > 0;
    }
    idx -= __shfl_sync(0xffffffffu, x, 31);
  }
  return false;
}

// Sequence and tile of slot `idx`; false for a slot without one. Sequence b has the slots from cu_q[b] / span + b on, in
// whole numbers: as many as it has tiles, or one more. Offsets that do not ascend may name any sequence; the tile lies
// inside it all the same.
MB_DEV bool find_slot(const Params& p, int idx, int span, Work& w) {
  const int lane = threadIdx.x & 31;
  auto clampq = [&](int x) { return max(0, min(x, (int)p.total_q)); };
  auto clampk = [&](int x) { return max(0, min(x, (int)p.total_k)); };
  int lo = 0, n = p.n_seqs;
#pragma unroll 1
  while (n > 32) {
    const int step = (n + 31) >> 5, at = lane * step, b = lo + (at < n ? at : 0);
    const unsigned le = __ballot_sync(0xffffffffu, at < n && clampq(p.cu_q[b]) / span + b <= idx);
    const int k = max(__popc(le), 1) - 1;  // le is a run of ones from bit 0
    lo += k * step;
    n = min(step, n - k * step);
  }
  const int b = lo + lane;
  int q0 = 0, m = 0, k0 = 0, nk = 0;
  if (lane < n) {
    q0 = clampq(p.cu_q[b]);
    m = max(0, clampq(p.cu_q[b + 1]) - q0);
    k0 = clampk(p.cu_k[b]);
    nk = max(0, clampk(p.cu_k[b + 1]) - k0);
  }
  const int first = q0 / span + b;
  const int src = max(__popc(__ballot_sync(0xffffffffu, lane < n && first <= idx)), 1) - 1;
  w.q_start = __shfl_sync(0xffffffffu, q0, src);
  w.m = __shfl_sync(0xffffffffu, m, src);
  w.k_start = __shfl_sync(0xffffffffu, k0, src);
  w.n = __shfl_sync(0xffffffffu, nk, src);
  const int last = (w.m + span - 1) / span - 1 - (idx - __shfl_sync(0xffffffffu, first, src));  // last tile first
  w.tok0 = last * span;
  return last >= 0 && last <= (w.m - 1) / span && w.m > 0;
}

// Asks for a block of this grid that has not started, to be cancelled: 16 bytes at `to`, counted by `bar`.
MB_DEV void take_block(void* to, uint64_t* bar) {
  fence_proxy_async_smem();  // the last answer has been read
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(to)),
               "r"(smem_u32(bar))
               : "memory");
}
// The cancelled block's index, whose work is the caller's now; -1: all have started.
MB_DEV int taken_block(const void* from) {
  uint32_t ok, x;
  asm volatile(
      "{\n .reg .pred p;\n .reg .b128 r;\n .reg .b32 y, z, w;\n ld.shared.b128 r, [%2];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, r;\n}\n"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(from))
      : "memory");
  return ok ? (int)x : -1;
}

template <int D>
struct Smem {
  static constexpr uint32_t kQ = 128 * D * 2, kQHalf = 128 * 128;        // the Q tile and one 64-channel atom column
  static constexpr uint32_t kBlock = BKV * D * 2, kHalf = BKV * 128;     // a K or V block
  static constexpr uint32_t kBars = kQ + (kK + kV) * kBlock;
  // two blocks on an SM, neither one (shared memory) nor three (TMEM)
  static constexpr size_t kBytes = kBars + 512 < 80 * 1024 ? 80 * 1024 : kBars + 512;
  static_assert(2 * (kBytes + 1024) <= 228 * 1024, "two blocks on an SM");
};

// MANY: more than kFewSeqs sequences
template <int D, bool MANY>
__global__ void __launch_bounds__(kThreads, 2)
    k_attention_varlen(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const Params p) {
  using S = Smem<D>;
  constexpr int CH = D / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = smem + S::kQ;
  uint8_t* sV = sK + kK * S::kBlock;
  uint64_t* bars = (uint64_t*)(smem + S::kBars);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;    // [kK]
  uint64_t* k_empty = bars + 4;   // [kK]
  uint64_t* v_full = bars + 6;    // [kV]
  uint64_t* v_ok = bars + 9;      // [kV]: guarded
  uint64_t* v_empty = bars + 12;  // [kV]
  uint64_t* s_full = bars + 15;   // [half]
  uint64_t* p_full = bars + 17;   // [half]
  uint64_t* o_full = bars + 19;
  uint64_t* pv_done = bars + 20;     // one completion per P V product
  uint64_t* work_full = bars + 21;   // [2]
  uint64_t* work_empty = bars + 23;  // [2]
  uint64_t* next_bar = bars + 25;
  uint8_t* next = (uint8_t*)(bars + 26);  // 16 bytes
  Work* work = (Work*)(bars + 28);        // [2]
  volatile int* odd_v = (volatile int*)(work + 2);  // [2]: a value that is not finite was zeroed for this tile
  uint32_t* tmem_slot = (uint32_t*)(work + 2) + 2;
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, TQ = p.TQ;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kK; i++) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kV; i++) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ok[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&work_full[i], 1);
      mbar_init(&work_empty[i], kWorkReaders);
    }
    mbar_init(o_full, 1);
    mbar_init(pv_done, 1);
    mbar_init(next_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  wait_before();  // ahead of the allocation: a block of the kernel before this one may need these columns to end
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.status, kDevTimeoutAttn); };
  // keys that the mask leaves token i of the sequence: the first keys_of(w, i)
  auto keys_of = [&](const Work& w, int i) { return p.causal ? max(0, min(i + 1 + w.n - w.m, w.n)) : w.n; };
  auto blocks_of = [&](const Work& w) { return (keys_of(w, min(w.tok0 + TQ, w.m) - 1) + BKV - 1) / BKV; };
  // Every role walks the same tiles. Rings and phases run on over them: block g of a tile is block kb + g of all.

  if (warp == 0) {
    int block = blockIdx.x, qn = 0, kb = 0, asked = 0;
    if (lane == 0) {
      tma_prefetch_desc(&tq);
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
    }
    bool ok = true;
    int nk = 0, nv = 0;  // blocks loaded, of all tiles
    int it = 0, passed = 0;
    for (int turn = 0; ok; turn++) {
      Work w;
      w.valid = 0;
      if (block >= 0) {
        const int item = block / p.Hkv;
        w.valid = MANY ? find_slot(p, item, TQ, w) : find_work(p, item, TQ, w);
        w.hk = block - item * p.Hkv;
      }
      // slots without a tile are passed over, but not so many that the other warps would give up waiting
      passed = w.valid ? 0 : passed + 1;
      const bool end = !w.valid && (!MANY || block < 0 || passed == kMostPassed);
      if (w.valid || end) {
        if (lane == 0) {
          if ((ok = wait(&work_empty[it & 1], ((it >> 1) & 1) ^ 1))) {
            work[it & 1] = w;
            mbar_arrive(&work_full[it & 1]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        it++;
      }
      if (!ok || end) break;
      const int n_kv = w.valid ? blocks_of(w) : 0;
      if (lane == 0 && n_kv > 0) {
        if ((ok = wait(q_empty, (qn & 1) ^ 1))) {
          mbar_expect_tx(q_full, (uint32_t)(CH * G * TQ * 128));
          for (int c = 0; c < CH; c++)
            tma_load_4d(sQ + c * S::kQHalf, &tq, q_full, 0, w.hk * G, w.q_start + w.tok0, c);
          qn++;
        }
        // V of block j - 1 after K of block j: the scores need their K first
        for (int j = 0; j <= n_kv && ok; j++) {
          if (j == n_kv - 1) {  // late, so that blocks with little left take what is left
            take_block(next, next_bar);
            asked++;
          }
          if (j < n_kv) {
            const int s = (kb + j) % kK;
            if (!(ok = wait(&k_empty[s], (((kb + j) / kK) & 1) ^ 1))) break;
            mbar_expect_tx(&k_full[s], S::kBlock);
            tma_load_4d(sK + s * S::kBlock, &tk, &k_full[s], 0, w.hk, w.k_start + j * BKV, 0);
            nk++;
          }
          if (j > 0) {
            const int s = (kb + j - 1) % kV;
            if (!(ok = wait(&v_empty[s], (((kb + j - 1) / kV) & 1) ^ 1))) break;
            mbar_expect_tx(&v_full[s], S::kBlock);
            tma_load_4d(sV + s * S::kBlock, &tv, &v_full[s], 0, w.hk, w.k_start + (j - 1) * BKV, 0);
            nv++;
          }
        }
      }
      kb += n_kv;
      if (lane == 0 && ok) {
        if (asked == turn) {  // no tile, or one without keys
          take_block(next, next_bar);
          asked++;
        }
        if ((ok = wait(next_bar, turn & 1))) block = taken_block(next);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      block = __shfl_sync(0xffffffffu, block, 0);
    }
    if (lane == 0) {
      // the block's memory must outlive its copies, whatever the other warps do
      volatile int never = 0;
      auto drain = [&](uint64_t* bar, int n) {
        if (n > 0) mbar_wait(bar, (n - 1) & 1, &never, p.status, kDevTimeoutAttn);
      };
      drain(next_bar, asked);
      drain(q_full, qn);
      for (int i = 0; i < kK; i++) drain(&k_full[i], (nk - i + kK - 1) / kK);
      for (int i = 0; i < kV; i++) drain(&v_full[i], (nv - i + kV - 1) / kV);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = idesc_bf16(128, BKV, false);
    constexpr uint32_t idesc_o = idesc_bf16(128, D, true);
    const uint32_t qa = smem_u32(sQ);
    int kb = 0, qn = 0;
    bool ok = true;
    for (int it = 0; ok; it++) {
      if (!(ok = wait(&work_full[it & 1], (it >> 1) & 1))) break;
      const Work w = work[it & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&work_empty[it & 1]);
      if (!w.valid) break;
      const int n_kv = blocks_of(w);
      if (n_kv == 0) continue;
      // S(g) = Q K_g^T into S half (kb + g) & 1
      auto issue_s = [&](int g) {
        const int b = kb + g, s = b % kK;
        if (!(ok = wait(&k_full[s], (b / kK) & 1))) return;
        tc_fence_after();
        const uint32_t ka = smem_u32(sK) + s * S::kBlock;
#pragma unroll
        for (int c = 0; c < CH; c++)
          umma_ss_x4_elect(tmem + (b & 1) * 64, sw128_desc(qa + c * S::kQHalf, 16, 1024),
                           sw128_desc(ka + c * S::kHalf, 16, 1024), idesc_s, c > 0);
        if (lane == 0) {
          umma_commit(&s_full[b & 1]);
          umma_commit(&k_empty[s]);
          if (g == n_kv - 1) umma_commit(q_empty);
        }
        __syncwarp();
      };
      if (!(ok = wait(q_full, qn & 1))) break;
      issue_s(0);
      if (ok && n_kv > 1) issue_s(1);
      for (int g = 0; g < n_kv && ok; g++) {
        const int b = kb + g, s = b % kV;
        if (!(ok = wait(&p_full[b & 1], (b >> 1) & 1))) break;
        if (!(ok = wait(&v_ok[s], (b / kV) & 1))) break;
        tc_fence_after();
        // O += P(g) V_g, P read from TMEM (bf16 pairs over the first 32 columns of its S half); V [keys, d] is MN-major:
        // 64-wide d chunks kHalf apart, 8-key groups 1024 B apart. The first P of a tile comes after its softmax warps
        // have read the last tile's O.
        umma_ts_x4_elect(tmem + 128, tmem + (b & 1) * 64, sw128_desc(smem_u32(sV) + s * S::kBlock, S::kHalf, 1024), idesc_o,
                         g > 0 ? 1u : 0u);
        if (lane == 0) {
          umma_commit(pv_done);
          umma_commit(&v_empty[s]);
          if (g == n_kv - 1) umma_commit(o_full);
        }
        __syncwarp();
        if (g + 2 < n_kv) issue_s(g + 2);
      }
      kb += n_kv;
      qn++;
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- V guard
    int kb = 0;
    bool ok = true;
    for (int it = 0; ok; it++) {
      if (!(ok = wait(&work_full[it & 1], (it >> 1) & 1))) break;
      const Work w = work[it & 1];
      if (!w.valid) break;
      if (lane == 0) odd_v[it & 1] = 0;
      __syncwarp();
      const int n_kv = blocks_of(w);
      // blocks from this one on hold keys that some row is not to see
      const int guard0 = keys_of(w, w.tok0) / BKV;
      for (int j = 0; j < n_kv; j++) {
        const int s = (kb + j) % kV;
        if (!(ok = wait(&v_full[s], ((kb + j) / kV) & 1))) break;
        if (j >= guard0) {
          uint8_t* v = sV + s * S::kBlock;
          // 16-byte pieces by address: a row is 128 bytes of each atom column, and the swizzle moves pieces
          // inside a row only
          const int rows = min(BKV, w.n - j * BKV);
          for (int i = rows * 8 + lane; i < BKV * 8; i += 32)
#pragma unroll
            for (int c = 0; c < CH; c++) *(uint4*)(v + c * S::kHalf + i * 16) = make_uint4(0, 0, 0, 0);
          if (p.causal) {
            __nv_bfloat162 acc = __float2bfloat162_rn(0.f);
            const __nv_bfloat162 zero = acc;
            for (int c = 0; c < CH; c++)
#pragma unroll 4
              for (int i = lane; i < rows * 8; i += 32) {
                const uint4 x = *(const uint4*)(v + c * S::kHalf + i * 16);
                acc = __hfma2(*(const __nv_bfloat162*)&x.x, zero, acc);  // NaN from what is not finite, and it stays
                acc = __hfma2(*(const __nv_bfloat162*)&x.y, zero, acc);
                acc = __hfma2(*(const __nv_bfloat162*)&x.z, zero, acc);
                acc = __hfma2(*(const __nv_bfloat162*)&x.w, zero, acc);
              }
            const uint32_t bits = *(const uint32_t*)&acc;
            if (!finite_bf16(bits) || !finite_bf16(bits >> 16)) {
              odd_v[it & 1] = 1;
              for (int c = 0; c < CH; c++)
                for (int i = lane; i < rows * 8; i += 32) {
                  uint32_t* x = (uint32_t*)(v + c * S::kHalf + i * 16);
                  for (int e = 0; e < 4; e++) {
                    uint32_t y = x[e];
                    if (!finite_bf16(y)) y &= 0xffff0000u;
                    if (!finite_bf16(y >> 16)) y &= 0x0000ffffu;
                    x[e] = y;
                  }
                }
            }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[s]);
      }
      kb += n_kv;
      __syncwarp();
      if (lane == 0) mbar_arrive(&work_empty[it & 1]);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax
    const int r = (warp - 4) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)((warp - 4) * 32) << 16;
    const uint32_t tO = tmem + 128 + lane_addr;
    const int row_tok = r / G, row_head = r % G;
    const float sc = p.scale_log2;
    int kb = 0, qn = 0;
    bool ok = true;
    for (int it = 0; ok; it++) {
      if (!(ok = wait(&work_full[it & 1], (it >> 1) & 1))) break;
      const Work w = work[it & 1];
      if (!w.valid) break;
      const int n_kv = blocks_of(w);
      const int all_see = keys_of(w, w.tok0);  // keys that every row sees
      const int tok = w.tok0 + row_tok;
      const bool mine = r < TQ * G && tok < w.m;  // this row is one of the sequence's
      const int keys = keys_of(w, min(tok, w.m - 1));
      float m_run = -INFINITY, l_run = 0.f;
      for (int g = 0; g < n_kv; g++) {
        const int b = kb + g;
        if (!(ok = wait(&s_full[b & 1], (b >> 1) & 1))) break;
        tc_fence_after();
        const uint32_t tSh = tmem + (b & 1) * 64 + lane_addr;
        uint32_t v[2][32];
        tmem_ld32(tSh, v[0]);
        tmem_ld32(tSh + 32, v[1]);
        tmem_wait_ld();
        const bool masked = (g + 1) * BKV > all_see;  // the same for the whole tile
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const int valid = keys - g * BKV - c * 32;
            const uint32_t bits = valid <= 0 ? 0u : valid >= 32 ? 0xffffffffu : (1u << valid) - 1u;
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (!((bits >> i) & 1)) v[c][i] = __float_as_uint(-INFINITY);
          }
        }
        float mc[4];  // four independent chains
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const uint32_t* x = &v[c >> 1][(c & 1) * 16];
          mc[c] = max_nan(__uint_as_float(x[0]), __uint_as_float(x[1]));
#pragma unroll
          for (int i = 2; i < 16; i += 2) mc[c] = max3_nan(mc[c], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        }
        const float m_new = max_nan(m_run, max3_nan(mc[0], mc[1], max_nan(mc[2], mc[3])) * sc);
        // lazy rescale: only rows whose max grew by more than 2^8 (or turned NaN) move their reference point
        const bool need = g == 0 || !(m_new <= m_run + kRescaleThreshold);
        const float alpha = (need && g > 0 && mine) ? ex2_approx(m_run - m_new) : 1.f;
        if (need) m_run = m_new;
        const float ref = m_run == -INFINITY ? 0.f : m_run;  // no key so far: weights 0
        const uint64_t sc2 = pk2(sc, sc), nm2 = pk2(-ref, -ref);
        uint64_t sum2 = pk2(0.f, 0.f);
        // All exponentials on the MUFU pipe: with K4's share of 6 in 32 as polynomials on the FMA pipe this kernel lost 10 %
        // (8201 tokens, 32/8 heads: 556 -> 618 us).
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const uint64_t x2 = fma2(pk2(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), sc2, nm2);
            float x0, x1;
            up2(x2, x0, x1);
            const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
            sum2 = add2(sum2, pk2(e0, e1));
            pk[i] = pack_bf16x2(e0, e1);
          }
          tmem_st16a(tSh + c * 16, pk);
        }
        float sa, sb;
        up2(sum2, sa, sb);
        if (g > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // O must hold P V of block g - 1 before it is rescaled
          if (!(ok = wait(pv_done, (b - 1) & 1))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; c++) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
        tmem_wait_st();
        l_run = l_run * alpha + (sa + sb);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b & 1]);
      }
      if (ok && n_kv > 0) ok = wait(o_full, qn & 1);
      if (!ok) break;
      kb += n_kv;
      qn += n_kv > 0;
      tc_fence_after();
      // a row without keys is 0; a maximum of NaN or +inf, or -inf over keys, makes softmax NaN
      const float inv = keys <= 0 ? 0.f : fabsf(m_run) < INFINITY ? 1.f / l_run : __uint_as_float(0x7fc00000u);
      __nv_bfloat16* orow = p.out + (int64_t)(w.q_start + tok) * p.ldo + (int64_t)(w.hk * G + row_head) * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; c++) {
        uint32_t o[32];
        if (n_kv > 0) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++) o[i] = 0u;
        }
        if (mine) {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            uint32_t y[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
              y[i] = pack_bf16x2(__uint_as_float(o[16 * u + 2 * i]), __uint_as_float(o[16 * u + 2 * i + 1]));
            store_row(orow + c * 32 + u * 16, y, p.wide_out);
          }
        }
      }
      if (odd_v[it & 1] && mine) {
        // values that are not finite and that the row sees; one by one, since this hardly ever runs
#pragma unroll 1
        for (int key = all_see / BKV * BKV; key < keys; key++) {
          const __nv_bfloat16* src = p.v + (int64_t)(w.k_start + key) * p.ldv + (int64_t)w.hk * D;
#pragma unroll 1
          for (int i = 0; i < D; i++) {
            const float y = __bfloat162float(src[i]);
            if (!(fabsf(y) < INFINITY)) orow[i] = __float2bfloat16_rn(__bfloat162float(orow[i]) + y);
          }
        }
      }
      tc_fence_before();  // O has been read: the next tile's first P, and the product after it, follow
      __syncwarp();
      if (lane == 0) mbar_arrive(&work_empty[it & 1]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <int D, bool MANY>
cudaError_t launch(const Params& p, const void* q, int64_t ldq, const void* k, int64_t ldk, int H, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  // {channel of an atom column, head, token, atom column}: the columns of a K or V block land behind each other in one
  // copy (four copies of 32 rows in their place: 3 %); those of Q, whose boxes may be less than 128 rows, in one each. A
  // sequence's end inside a box reads the next sequence's rows, which the masks leave out.
  auto map = [&](CUtensorMap* m, const void* x, int64_t heads, int64_t rows, int64_t ld, int box_heads, int box_rows,
                 int box_cols) {
    return make_tmap_4d(m, x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, {64, (uint64_t)heads, (uint64_t)(rows > 0 ? rows : 1), D / 64},
                        {D * 2, (uint64_t)ld * 2, 128}, {64, (uint32_t)box_heads, (uint32_t)box_rows, (uint32_t)box_cols},
                        CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (!map(&tq, q, H, p.total_q, ldq, p.G, p.TQ, 1) || !map(&tk, k, p.Hkv, p.total_k, ldk, 1, BKV, D / 64) ||
      !map(&tv, p.v, p.Hkv, p.total_k, p.ldv, 1, BKV, D / 64))
    return cudaErrorInvalidValue;
  static int attr_done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_done[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(k_attention_varlen<D, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Smem<D>::kBytes);
    if (e != cudaSuccess) return e;
    attr_done[dev & 63] = 1;
  }
  return launch_close(k_attention_varlen<D, MANY>, dim3(p.blocks), kThreads, Smem<D>::kBytes, st, 1, tq, tk, tv, p);
}

template <int D>
cudaError_t launch(const Params& p, const void* q, int64_t ldq, const void* k, int64_t ldk, int H, cudaStream_t st) {
  return p.n_seqs > kFewSeqs ? launch<D, true>(p, q, ldq, k, ldk, H, st) : launch<D, false>(p, q, ldq, k, ldk, H, st);
}

}  // namespace varlen
}  // namespace mb

using namespace mb;

extern "C" mb_status mb_attention_varlen(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                         int64_t ldv, int64_t total_q, int64_t total_k, int H, int H_kv, int D,
                                         const int32_t* cu_q, const int32_t* cu_k, int n_seqs, int causal, float scale,
                                         void* out, int64_t ldo, void* stream) {
  MB_CHECK(D == 64 || D == 128, MB_ERR_UNSUPPORTED, "head size D must be 64 or 128");
  MB_CHECK(H > 0 && H_kv > 0 && H % H_kv == 0 && H <= 65535, MB_ERR_INVALID,
           "H must be a positive multiple of H_kv, at most 65535");
  MB_CHECK(H / H_kv <= 128, MB_ERR_UNSUPPORTED, "at most 128 query heads may share a key head");
  MB_CHECK(total_q >= 0 && total_q < (1LL << 30) && total_k >= 0 && total_k < (1LL << 30), MB_ERR_INVALID,
           "total_q and total_k must be from 0 to 2^30 - 1");
  MB_CHECK(n_seqs >= 0 && n_seqs < (1 << 24), MB_ERR_INVALID, "n_seqs must be from 0 to 2^24 - 1");
  MB_CHECK(scale >= 0.f && scale <= 2.3e38f, MB_ERR_INVALID, "scale must be positive, at most 2.3e38 (0: 1 / sqrt(D))");
  if (total_q == 0 || n_seqs == 0) return MB_OK;
  MB_CHECK(cu_q && cu_k, MB_ERR_INVALID, "cu_q or cu_k is NULL");
  auto rows_ok = [](const void* x, int64_t ld, int64_t width) {
    return x && ((uintptr_t)x & 15) == 0 && ld >= width && ld % 8 == 0 && ld < (1LL << 38);
  };
  MB_CHECK(rows_ok(q, ldq, (int64_t)H * D) && rows_ok(out, ldo, (int64_t)H * D), MB_ERR_INVALID,
           "q and out must be 16-byte aligned with row strides of at least H * D, multiples of 8");
  MB_CHECK(total_k == 0 || (rows_ok(k, ldk, (int64_t)H_kv * D) && rows_ok(v, ldv, (int64_t)H_kv * D)), MB_ERR_INVALID,
           "k and v must be 16-byte aligned with row strides of at least H_kv * D, multiples of 8");
  const int64_t blocks = (total_q / (128 / (H / H_kv)) + n_seqs) * H_kv;  // each sequence rounds up once
  MB_CHECK(blocks < (1LL << 31), MB_ERR_INVALID, "too many tiles for one launch");
  MB_CHECK(device_status_ready(), MB_ERR_NOT_READY, "call mb_init on this device first");
  varlen::Params p;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.n_seqs = n_seqs;
  p.total_q = total_q;
  p.total_k = total_k;
  p.Hkv = H_kv;
  p.G = H / H_kv;
  p.TQ = 128 / p.G;
  p.blocks = (unsigned)blocks;
  p.causal = causal != 0;
  p.scale_log2 = (float)((scale > 0.f ? (double)scale : 1.0 / sqrt((double)D)) * 1.4426950408889634);
  p.v = (const __nv_bfloat16*)v;
  p.ldv = ldv;
  p.out = (__nv_bfloat16*)out;
  p.ldo = ldo;
  p.wide_out = ((uintptr_t)out & 31) == 0 && ldo % 16 == 0;
  p.status = device_status_ptr();
  if (total_k == 0) {  // no key anywhere: the maps need some memory to describe, and no block reads it
    k = q;
    ldk = p.ldv = ldq;
    p.v = (const __nv_bfloat16*)q;
  }
  MB_CUDA(D == 64 ? varlen::launch<64>(p, q, ldq, k, ldk, H, (cudaStream_t)stream)
                  : varlen::launch<128>(p, q, ldq, k, ldk, H, (cudaStream_t)stream));
  return MB_OK;
}
