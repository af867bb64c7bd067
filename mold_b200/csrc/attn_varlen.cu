// K11: attention of packed prompts, causal or not, grouped heads, on tcgen05 + TMEM (sm_100a).
//
// The structure is K4's (attention.cu): two 128-row query tiles a block, scores and output in TMEM, one
// softmax thread a row, two MMA issuers, 64-key sub-blocks. What differs:
//   - A tile's rows are TQ = 128 / G tokens of all G query heads of one key head (row = token * G +
//     head), one TMA box of G heads x TQ tokens: the group shares each K / V block, and a causal tile
//     spans few tokens, so little of its diagonal blocks is masked work.
//   - A block finds its sequence and tile from cu_q by a scan; a sequence's last tiles (the longest under
//     a causal mask) come first.
//   - Each tile stops at the last 64-key sub-block that its mask leaves; only sub-blocks that cross a
//     row's limit are masked.
//   - Warp 3 guards V: a P V product adds 0 * v for every masked key of a block, so in the blocks that a
//     mask or the sequence's end crosses it zeroes rows of other sequences and values that are not finite
//     before the product reads them; rows that may see such a value add it at the end (a slow path that
//     ordinary data never takes).
#include <math.h>

#include <string>

#include "attn_util.cuh"
#include "common.cuh"
#include "internal.h"

namespace mb {
namespace varlen {
using namespace attn;

constexpr int BKV = 128, NT = 2;
constexpr int kThreads = 384;
constexpr float kRescaleThreshold = 8.f;
constexpr int kPolyPerChunk = 6;  // exponentials of every 32 on the FMA pipe, as in K4

struct Params {
  const int32_t *cu_q, *cu_k;
  int n_seqs;
  int64_t total_q, total_k;
  int Hkv, G, TQ, causal;
  float scale_log2;
  const __nv_bfloat16* v;
  int64_t ldv;
  __nv_bfloat16* out;
  int64_t ldo;
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
MB_DEV bool finite_bf16(uint32_t bits) { return (bits & 0x7f80u) != 0x7f80u; }

// What a block works on. Computed by warp 0.
struct Work {
  int q_start, k_start;  // first packed row of the sequence
  int m, n;              // queries, keys
  int tok0;              // first token of tile 0
};

// Sequence and tile of item `idx` (counting each sequence's tiles of `span` tokens); false behind the last.
MB_DEV bool find_work(const Params& p, int64_t idx, int span, Work& w) {
  const int lane = threadIdx.x & 31;
  auto clampq = [&](int64_t x) { return (int)(x < 0 ? 0 : x < p.total_q ? x : p.total_q); };
  auto clampk = [&](int64_t x) { return (int)(x < 0 ? 0 : x < p.total_k ? x : p.total_k); };
  for (int base = 0; base < p.n_seqs; base += 32) {
    const int b = base + lane;
    int q0 = 0, m = 0;
    if (b < p.n_seqs) {
      q0 = clampq(__ldg(p.cu_q + b));
      m = max(0, clampq(__ldg(p.cu_q + b + 1)) - q0);
    }
    int64_t x = (m + span - 1) / span;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, idx < x);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t end = __shfl_sync(0xffffffffu, x, src);
      w.q_start = __shfl_sync(0xffffffffu, q0, src);
      w.m = __shfl_sync(0xffffffffu, m, src);
      const int k0 = clampk(__ldg(p.cu_k + base + src));
      w.k_start = k0;
      w.n = max(0, clampk(__ldg(p.cu_k + base + src + 1)) - k0);
      w.tok0 = (int)(end - 1 - idx) * span;  // last tile first
      return true;
    }
    idx -= __shfl_sync(0xffffffffu, x, 31);
  }
  return false;
}

template <int D>
struct Smem {
  static constexpr uint32_t kTile = 128 * D * 2;
  static constexpr uint32_t kHalf = 128 * 64 * 2;  // one 64-channel atom column of a tile
  static constexpr size_t kBytes = 1024 + 6 * (size_t)kTile + 512;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    k_attention_varlen(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const Params p) {
  constexpr uint32_t kTile = Smem<D>::kTile, kHalf = Smem<D>::kHalf;
  constexpr int CH = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;              // 2 tiles
  uint8_t* sK = smem + 2 * kTile;  // 2 stages
  uint8_t* sV = smem + 4 * kTile;  // 2 stages
  uint64_t* bars = (uint64_t*)(smem + 6 * kTile);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;    // [2] per stage
  uint64_t* v_full = bars + 3;    // [2]
  uint64_t* kv_empty = bars + 5;  // [2]
  uint64_t* s_full = bars + 7;    // [tile][half]
  uint64_t* p_full = bars + 11;   // [tile][half]
  uint64_t* o_full = bars + 15;   // [tile]
  uint64_t* pv_done = bars + 17;  // [tile]
  uint64_t* v_ok = bars + 19;     // [2] per stage: guarded blocks
  uint32_t* tmem_slot = (uint32_t*)(bars + 21);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* odd_v = (volatile int*)(tmem_slot + 2);  // a value that is not finite was zeroed
  int* found = (int*)(tmem_slot + 3);
  Work* work = (Work*)(tmem_slot + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G, TQ = p.TQ;
  const int64_t item = blockIdx.x / p.Hkv;
  const int hk = (int)(blockIdx.x - item * p.Hkv);

  if (warp == 0) {
    Work w;
    const bool ok = find_work(p, item, NT * TQ, w);
    if (lane == 0) {
      *found = ok;
      if (ok) *work = w;
      mbar_init(q_full, 1);
      for (int i = 0; i < 2; i++) {
        mbar_init(&k_full[i], 1);
        mbar_init(&v_full[i], 1);
        mbar_init(&v_ok[i], 1);
        mbar_init(&kv_empty[i], 3);  // one arrival per MMA issuer and one of the V guard
        mbar_init(&o_full[i], 1);
        mbar_init(&pv_done[i], 1);
      }
      for (int i = 0; i < 4; i++) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 4);
      }
      *abort_flag = 0;
      *odd_v = 0;
      fence_mbar_init();
    }
  }
  __syncthreads();
  if (!*found) return;
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Work w = *work;

  // keys that the mask leaves token i of the sequence: the first keys_of(i)
  auto keys_of = [&](int i) { return p.causal ? max(0, min(i + 1 + w.n - w.m, w.n)) : w.n; };
  // sub-blocks of tile t, and the keys that all of its rows see
  auto tile_subs = [&](int t) {
    const int first = w.tok0 + t * TQ;
    return first >= w.m ? 0 : (keys_of(min(first + TQ, w.m) - 1) + 63) / 64;
  };
  const int n_sub0 = tile_subs(0), n_sub1 = tile_subs(1);
  const int n_kv = (max(n_sub0, n_sub1) + 1) / 2;
  // blocks from this one on hold keys that some row is not to see
  const int guard0 = keys_of(w.tok0) / BKV;

  if (warp == 0) {
    if (lane == 0 && n_kv > 0) {
      tma_prefetch_desc(&tq);
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
      const int tiles = n_sub1 > 0 ? 2 : 1;  // tile 1 never has fewer keys than tile 0
      mbar_expect_tx(q_full, (uint32_t)(tiles * CH * G * TQ * 128));
      for (int t = 0; t < tiles; t++)
        for (int c = 0; c < CH; c++)
          tma_load_3d(sQ + t * kTile + c * kHalf, &tq, q_full, c * 64, hk * G, w.q_start + w.tok0 + t * TQ);
      for (int j = 0; j < n_kv; j++) {
        const int s = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        if (!(mbar_wait(&kv_empty[s], ph ^ 1, abort_flag, p.status, kDevTimeoutAttn))) break;
        mbar_expect_tx(&k_full[s], kTile);
        for (int c = 0; c < CH; c++)
          tma_load_3d(sK + s * kTile + c * kHalf, &tk, &k_full[s], c * 64, hk, w.k_start + j * BKV);
        mbar_expect_tx(&v_full[s], kTile);
        for (int c = 0; c < CH; c++)
          tma_load_3d(sV + s * kTile + c * kHalf, &tv, &v_full[s], c * 64, hk, w.k_start + j * BKV);
      }
    }
  } else if (warp == 1 || warp == 2) {
    const int t = warp - 1;
    constexpr uint32_t idesc_s = idesc_bf16(128, 64, false);
    constexpr uint32_t idesc_o = idesc_bf16(128, D, true);
    const uint32_t qa = smem_u32(sQ) + t * kTile;
    const int n_sub = t ? n_sub1 : n_sub0;
    bool ok = n_kv == 0 || mbar_wait(q_full, 0, abort_flag, p.status, kDevTimeoutAttn);
    // S_t(g) = Q_t K_g^T (64 keys) into S half g & 1
    auto issue_s = [&](int g) {
      const int hh = g & 1;
      const uint32_t ka = smem_u32(sK + ((g >> 1) & 1) * kTile) + hh * 8192;
#pragma unroll
      for (int kk = 0; kk < D / 16; kk++) {
        const uint32_t off = (kk >> 2) * kHalf + (kk & 3) * 32;
        umma_ss_elect(tmem + t * 128 + hh * 64, sw128_desc(qa + off, 16, 1024), sw128_desc(ka + off, 16, 1024),
                      idesc_s, kk > 0);
      }
      if (lane == 0) umma_commit(&s_full[t * 2 + hh]);
      __syncwarp();
    };
    // O_t += P_t(g) V_g; the block's stage is released with the tile's last sub-block of it
    auto issue_pv = [&](int g) {
      const int hh = g & 1;
      const uint32_t va = smem_u32(sV + ((g >> 1) & 1) * kTile);
#pragma unroll
      for (int kk = 0; kk < 4; kk++) {
        const uint64_t bdesc = sw128_desc(va + (hh * 4 + kk) * 16 * 128, kHalf, 1024);
        umma_ts_elect(tmem + 256 + t * 128, tmem + t * 128 + hh * 64 + kk * 8, bdesc, idesc_o,
                      (g > 0 || kk > 0) ? 1u : 0u);
      }
      if (lane == 0) {
        umma_commit(&pv_done[t]);
        if (hh == 1 || g == n_sub - 1) umma_commit(&kv_empty[(g >> 1) & 1]);
      }
      __syncwarp();
    };
    if (ok && n_sub > 0) {
      if ((ok = mbar_wait(&k_full[0], 0, abort_flag, p.status, kDevTimeoutAttn))) {
        tc_fence_after();
        issue_s(0);
        if (n_sub > 1) issue_s(1);
      }
    }
    for (int g = 0; g < n_sub && ok; g++) {
      const int hh = g & 1, j = g >> 1;
      if (hh == 0) {
        if (!(ok = j < guard0 ? mbar_wait(&v_full[j & 1], (j >> 1) & 1, abort_flag, p.status, kDevTimeoutAttn)
                              : mbar_wait(&v_ok[j & 1], ((j - guard0) >> 1) & 1, abort_flag, p.status,
                                          kDevTimeoutAttn)))
          break;
      }
      if (!(ok = (mbar_wait(&p_full[t * 2 + hh], j & 1, abort_flag, p.status, kDevTimeoutAttn)))) break;
      tc_fence_after();
      issue_pv(g);
      if (g + 2 < n_sub) {
        if (hh == 0 &&
            !(ok = (mbar_wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, abort_flag, p.status, kDevTimeoutAttn))))
          break;
        tc_fence_after();
        issue_s(g + 2);
      }
    }
    if (ok && n_sub > 0 && lane == 0) umma_commit(&o_full[t]);
    __syncwarp();
    // blocks that only the other tile reads: this issuer's arrival once each has been loaded
    for (int j = (n_sub + 1) / 2; j < n_kv && ok; j++) {
      ok = mbar_wait(&k_full[j & 1], (j >> 1) & 1, abort_flag, p.status, kDevTimeoutAttn);
      if (ok && lane == 0) mbar_arrive(&kv_empty[j & 1]);
      __syncwarp();
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- V guard
    // Takes part in every block, so that it never falls a phase of a barrier behind.
    for (int j = 0; j < n_kv; j++) {
      const int s = j & 1;
      if (!mbar_wait(&v_full[s], (j >> 1) & 1, abort_flag, p.status, kDevTimeoutAttn)) break;
      if (j < guard0) {
        if (lane == 0) mbar_arrive(&kv_empty[s]);
        __syncwarp();
        continue;
      }
      uint8_t* v = sV + s * kTile;
      // 16-byte pieces by address: a row is 128 bytes of each atom column, and the swizzle moves pieces
      // inside a row only
      const int rows = min(BKV, w.n - j * BKV);
      for (int i = rows * 8 + lane; i < BKV * 8; i += 32)
#pragma unroll
        for (int c = 0; c < CH; c++) *(uint4*)(v + c * kHalf + i * 16) = make_uint4(0, 0, 0, 0);
      if (p.causal) {
        __nv_bfloat162 acc = __float2bfloat162_rn(0.f);
        const __nv_bfloat162 zero = acc;
        for (int c = 0; c < CH; c++)
#pragma unroll 4
          for (int i = lane; i < rows * 8; i += 32) {
            const uint4 x = *(const uint4*)(v + c * kHalf + i * 16);
            acc = __hfma2(*(const __nv_bfloat162*)&x.x, zero, acc);  // NaN from what is not finite, and it stays
            acc = __hfma2(*(const __nv_bfloat162*)&x.y, zero, acc);
            acc = __hfma2(*(const __nv_bfloat162*)&x.z, zero, acc);
            acc = __hfma2(*(const __nv_bfloat162*)&x.w, zero, acc);
          }
        const uint32_t bits = *(const uint32_t*)&acc;
        if (!finite_bf16(bits) || !finite_bf16(bits >> 16)) {
          *odd_v = 1;
          for (int c = 0; c < CH; c++)
            for (int i = lane; i < rows * 8; i += 32) {
              uint32_t* x = (uint32_t*)(v + c * kHalf + i * 16);
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
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_ok[s]);
        mbar_arrive(&kv_empty[s]);
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- softmax
    // 4 warps per tile; thread = query row = TMEM lane.
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_addr, tO = tmem + 256 + t * 128 + lane_addr;
    const int first = w.tok0 + t * TQ;
    const int tok = first + r / G, head = hk * G + r % G;
    const bool mine = r < TQ * G && tok < w.m;  // this row is one of the sequence's
    const int keys = keys_of(min(tok, w.m - 1));
    const int all_see = keys_of(min(first, w.m - 1));
    const int n_sub = t ? n_sub1 : n_sub0;
    const float sc = p.scale_log2;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int g = 0; g < n_sub; g++) {
      const int hh = g & 1;
      if (!(ok = (mbar_wait(&s_full[t * 2 + hh], (g >> 1) & 1, abort_flag, p.status, kDevTimeoutAttn))))
        break;
      tc_fence_after();
      const uint32_t tSh = tS + hh * 64;
      uint32_t v[2][32];
      tmem_ld32(tSh, v[0]);
      tmem_ld32(tSh + 32, v[1]);
      tmem_wait_ld();
      const bool masked = (g + 1) * 64 > all_see;  // the same for the whole tile
      if (masked) {
        const int valid = keys - g * 64;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (c * 32 + i >= valid) v[c][i] = __float_as_uint(-INFINITY);
      }
      float mc[2];
#pragma unroll
      for (int c = 0; c < 2; c++) {
        mc[c] = max_nan(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]));
#pragma unroll
        for (int i = 2; i < 32; i += 2) mc[c] = max3_nan(mc[c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
      }
      const float m_new = max_nan(m_run, max_nan(mc[0], mc[1]) * sc);
      // lazy rescale: only rows whose max grew by more than 2^8 (or turned NaN) move their reference point
      const bool need = g == 0 || !(m_new <= m_run + kRescaleThreshold);
      const float alpha = (need && g > 0 && mine) ? ex2_approx(m_run - m_new) : 1.f;
      if (need) m_run = m_new;
      const float ref = m_run == -INFINITY ? 0.f : m_run;  // no key so far: weights 0
      const uint64_t sc2 = pk2(sc, sc), nm2 = pk2(-ref, -ref);
      uint64_t sum2 = pk2(0.f, 0.f);
      // In masked sub-blocks all exponentials are the exact-zero kind: the polynomial ends at 2^-126.
#pragma unroll
      for (int c = 0; c < 2; c++) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const uint64_t x2 = fma2(pk2(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), sc2, nm2);
          float e0, e1;
          if (2 * i < kPolyPerChunk && !masked) {
            exp2_poly3(x2, e0, e1);
          } else {
            float x0, x1;
            up2(x2, x0, x1);
            e0 = ex2_approx(x0);
            e1 = ex2_approx(x1);
          }
          sum2 = add2(sum2, pk2(e0, e1));
          pk[i] = pack_bf16x2(e0, e1);
        }
        tmem_st16a(tSh + c * 16, pk);
      }
      float sa, sb;
      up2(sum2, sa, sb);
      if (g > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // O_t must hold P V of sub-block g - 1 before it is rescaled
        if (!(ok = mbar_wait(&pv_done[t], (g - 1) & 1, abort_flag, p.status, kDevTimeoutAttn))) break;
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
      if (lane == 0) mbar_arrive(&p_full[t * 2 + hh]);
    }
    if (ok && n_sub > 0) ok = mbar_wait(&o_full[t], 0, abort_flag, p.status, kDevTimeoutAttn);
    if (ok) {
      tc_fence_after();
      // a row without keys is 0; a maximum of NaN or +inf, or -inf over keys, makes softmax NaN
      const float inv = keys <= 0 ? 0.f : fabsf(m_run) < INFINITY ? 1.f / l_run : __uint_as_float(0x7fc00000u);
      __nv_bfloat16* orow = p.out + (int64_t)(w.q_start + tok) * p.ldo + (int64_t)head * D;
      const bool odd = *odd_v;
#pragma unroll 1
      for (int c = 0; c < D / 32; c++) {
        uint32_t o[32];
        if (n_sub > 0) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; i++) o[i] = keys > 0 ? __float_as_uint(__uint_as_float(o[i]) * inv) : 0u;
        if (odd) {
#pragma unroll 1
          for (int key = guard0 * BKV; key < keys; key++) {
            const uint32_t* src =
                (const uint32_t*)(p.v + (int64_t)(w.k_start + key) * p.ldv + (int64_t)hk * D + c * 32);
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const uint32_t y = __ldg(src + i);
              if (!finite_bf16(y)) o[2 * i] = __float_as_uint(__uint_as_float(o[2 * i]) + bf16_lo(y));
              if (!finite_bf16(y >> 16)) o[2 * i + 1] = __float_as_uint(__uint_as_float(o[2 * i + 1]) + bf16_hi(y));
            }
          }
        }
        if (mine) {
#pragma unroll
          for (int u = 0; u < 4; u++) {
            uint4 w4;
            w4.x = pack_bf16x2(__uint_as_float(o[8 * u + 0]), __uint_as_float(o[8 * u + 1]));
            w4.y = pack_bf16x2(__uint_as_float(o[8 * u + 2]), __uint_as_float(o[8 * u + 3]));
            w4.z = pack_bf16x2(__uint_as_float(o[8 * u + 4]), __uint_as_float(o[8 * u + 5]));
            w4.w = pack_bf16x2(__uint_as_float(o[8 * u + 6]), __uint_as_float(o[8 * u + 7]));
            *(uint4*)(orow + c * 32 + u * 8) = w4;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
cudaError_t launch(const Params& p, const void* q, int64_t ldq, const void* k, int64_t ldk, int H, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  const uint64_t head = D * 2, keys = p.total_k > 0 ? (uint64_t)p.total_k : 1;
  // {channel, head, token}; a sequence's end inside a box reads the next sequence's rows, which the masks leave out
  if (!make_tmap_3d(&tq, q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, D, (uint64_t)H, (uint64_t)p.total_q, head,
                    (uint64_t)ldq * 2, 64, (uint32_t)p.G, (uint32_t)p.TQ, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_3d(&tk, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, D, (uint64_t)p.Hkv, keys, head,
                    (uint64_t)ldk * 2, 64, 1, BKV, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_3d(&tv, p.v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, D, (uint64_t)p.Hkv, keys, head,
                    (uint64_t)p.ldv * 2, 64, 1, BKV, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  static int attr_done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_done[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(k_attention_varlen<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Smem<D>::kBytes);
    if (e != cudaSuccess) return e;
    attr_done[dev & 63] = 1;
  }
  const int64_t blocks = (p.total_q / (NT * p.TQ) + p.n_seqs) * p.Hkv;  // each sequence rounds up once
  if (blocks >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  k_attention_varlen<D><<<(unsigned)blocks, kThreads, Smem<D>::kBytes, st>>>(tq, tk, tv, p);
  return cudaGetLastError();
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
  MB_CHECK(scale >= 0.f && scale <= 3.0e38f, MB_ERR_INVALID, "scale must be positive and finite (0: 1 / sqrt(D))");
  if (total_q == 0 || n_seqs == 0) return MB_OK;
  MB_CHECK(cu_q && cu_k, MB_ERR_INVALID, "cu_q or cu_k is NULL");
  auto rows_ok = [](const void* x, int64_t ld, int64_t width) {
    return x && ((uintptr_t)x & 15) == 0 && ld >= width && ld % 8 == 0 && ld < (1LL << 38);
  };
  MB_CHECK(rows_ok(q, ldq, (int64_t)H * D) && rows_ok(out, ldo, (int64_t)H * D), MB_ERR_INVALID,
           "q and out must be 16-byte aligned with row strides of at least H * D, multiples of 8");
  MB_CHECK(total_k == 0 || (rows_ok(k, ldk, (int64_t)H_kv * D) && rows_ok(v, ldv, (int64_t)H_kv * D)), MB_ERR_INVALID,
           "k and v must be 16-byte aligned with row strides of at least H_kv * D, multiples of 8");
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
  p.causal = causal != 0;
  p.scale_log2 = (float)((scale > 0.f ? (double)scale : 1.0 / sqrt((double)D)) * 1.4426950408889634);
  p.v = (const __nv_bfloat16*)v;
  p.ldv = ldv;
  p.out = (__nv_bfloat16*)out;
  p.ldo = ldo;
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
