// Gradients of cross attention for sm_100a (b200_cross_attn_bwd_bf16):
// tcgen05 + TMEM + TMA, on the layout of the forward kernel (attn_sm100.cuh).
// With P = exp(scale Q K^T - lse) and delta = rowsum(dO o O):
//   dV = P^T dO,  dS = P o (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q.
//
// attn_bwd_delta_kernel writes delta and lse (in the exp2 domain) of every
// query row, padded to whole tiles (+inf, 0: such rows get P = 0).
// attn_bwd_kernel is one grid of two kinds of CTA, one per SM:
//   dK/dV: one per 128-key tile, key/value head and batch entry, walking over
//          the 128-row query tiles of every query head of the group;
//   dQ:    one per 128-row query tile, head and batch entry, walking over the
//          key tiles of its batch entry.
// Both recompute S and dP, 4 + 3 products a tile pair where a single pass
// would need 5.  In exchange nothing is added across CTAs: the gradients of
// shared heads are sums in a fixed order, with no atomics and no fp32
// copy of dQ.  dK/dV CTAs come first in the grid (with grouped heads they are
// the longer ones), dQ CTAs fill their last wave.
//
// One body for both kinds.  X1, X2 are the CTA's own tiles, Y1, Y2 the
// streamed ones; rows of the products are X's rows (TMEM lanes), columns Y's:
//   dK/dV: X = K, V   Y = Q, dO   T1 = S^T, T2 = dP^T;  acc1 (dK) += dS^T Q, acc2 (dV) += P^T dO
//   dQ:    X = Q, dO  Y = K, V    T1 = S,   T2 = dP;    acc1 (dQ) += dS K
// P and dS go back to TMEM as bf16 (the A operand of the second products);
// every Y tile serves once as a K-major and once as an MN-major operand.
//
// 384 threads: warps 0..7 compute, two warpgroups of 64 columns each, one
// thread per row; warp 8 TMA producer, warp 9 MMA issuer and TMEM owner, warps
// 10, 11 zero the K rows past the last key in the last tile of a dQ CTA (they
// may hold NaN, and 0 x NaN would reach dQ).
// TMEM, 512 columns: a warpgroup puts P and dS over its own half of T1, so no
// warp waits for another.  dK/dV: T1 and T2 swap two regions from tile to
// tile, T1 of the next tile being computed while dS of this one is.  dQ: T1
// has two regions of its own, a tile ahead, T2 a third.
// Every wait is bounded, as in the forward kernel.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>

#include "attn_sm100.cuh"
#include "gemm_sm100.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

struct AttnBwdParams {
  int32_t q_len, kv_len, heads, kv_heads, group, batch;
  int32_t q_tiles, kv_tiles;
  int32_t dkv_ctas;        // CTAs [0, dkv_ctas) compute dK and dV, the others dQ
  const int32_t* kv_lens;  // [batch] or NULL
  float scale, scale_log2;
  // [batch * heads][q_tiles * 128], of attn_bwd_delta_kernel.
  float* lse2;
  float* delta;
  uint64_t timeout_ns;
  uint32_t* status;
};

struct AttnBwdMaps {
  CUtensorMap q, k, v, dout, dq, dk, dv;
};

struct AttnBwdDeltaParams {
  const __nv_bfloat16* o;
  int64_t o_batch, o_seq, o_head;
  const __nv_bfloat16* dout;
  int64_t d_batch, d_seq, d_head;
  const float* lse;  // [batch, heads, q_len]
  float* lse2;
  float* delta;
  int32_t q_len, heads, padded;  // padded = q_tiles * 128
  int32_t rows;                  // batch * heads
};

// One warp per query row, 8 bytes of O and dO a lane: bound by reading both once.
__global__ void __launch_bounds__(256) attn_bwd_delta_kernel(const __grid_constant__ AttnBwdDeltaParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = (int)(threadIdx.x & 31u);
  const int row = (int)blockIdx.x * 8 + ((int)threadIdx.x >> 5);
  const int bh = (int)blockIdx.y + 65535 * (int)blockIdx.z;
  const int head = bh % p.heads;
  const int64_t bat = bh / p.heads;
  if (row >= p.padded || bh >= p.rows) return;
  float sum = 0.0f, lse2 = INFINITY;
  if (row < p.q_len) {
    const uint2 a = *reinterpret_cast<const uint2*>(p.o + bat * p.o_batch + row * p.o_seq + head * p.o_head + 4 * lane);
    const uint2 b = *reinterpret_cast<const uint2*>(p.dout + bat * p.d_batch + row * p.d_seq + head * p.d_head + 4 * lane);
    auto dot = [&](uint32_t x, uint32_t y) {
      sum = fmaf(__uint_as_float(x << 16), __uint_as_float(y << 16), sum);
      sum = fmaf(__uint_as_float(x & 0xffff0000u), __uint_as_float(y & 0xffff0000u), sum);
    };
    dot(a.x, b.x);
    dot(a.y, b.y);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    lse2 = p.lse[(size_t)bh * p.q_len + row] * 1.4426950408889634f;
  }
  if (lane == 0) {
    p.lse2[(size_t)bh * p.padded + row] = lse2;
    p.delta[(size_t)bh * p.padded + row] = sum;
  }
}

template <bool kDQ>
struct AttnBwdPlan {
  static constexpr int kTileBytes = 128 * 128 * 2;
  // dQ keeps T1 a tile ahead and so holds K a tile longer.
  static constexpr int kY1Stages = kDQ ? 3 : 2;
  static constexpr int kY2Stages = 2;
  static constexpr int kOffX1 = 0, kOffX2 = kTileBytes;
  static constexpr int kOffY1 = 2 * kTileBytes;
  static constexpr int kOffY2 = kOffY1 + kY1Stages * kTileBytes;
  static constexpr int kOffVec = kOffY2 + kY2Stages * kTileBytes;  // dK/dV: lse2 and delta of a Y1 stage's rows
  static constexpr int kOffBar = kOffVec + (kDQ ? 0 : kY1Stages * 1024);
  static constexpr int kNumBars = 2 + 2 * kY1Stages + 2 * kY2Stages + 2 + 1 + 1 + 1 + 2 + 2;
  static constexpr int kOffTmemHolder = kOffBar + kNumBars * 8;
  static constexpr int kOffAbort = kOffTmemHolder + 4;
  static constexpr int kBytes = kOffAbort + 4;
  static constexpr int kAllocBytes = kBytes + 1024;
  static_assert(kAllocBytes <= 232448, "attention backward shared memory plan exceeds 227 KiB");
};
constexpr int kAttnBwdSmem = AttnBwdPlan<true>::kAllocBytes > AttnBwdPlan<false>::kAllocBytes
                                 ? AttnBwdPlan<true>::kAllocBytes
                                 : AttnBwdPlan<false>::kAllocBytes;

template <bool kDQ>
__device__ __forceinline__ void attn_bwd_body(const AttnBwdMaps& tm, const AttnBwdParams& p, int cta) {
  using Plan = AttnBwdPlan<kDQ>;
  constexpr int S1 = Plan::kY1Stages, S2 = Plan::kY2Stages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_u32);
  const uint32_t sX1 = base + Plan::kOffX1, sX2 = base + Plan::kOffX2;
  auto sY1 = [&](int i) { return base + (uint32_t)(Plan::kOffY1 + (i % S1) * Plan::kTileBytes); };
  auto sY2 = [&](int i) { return base + (uint32_t)(Plan::kOffY2 + (i % S2) * Plan::kTileBytes); };
  const uint32_t bar0 = base + Plan::kOffBar;
  const uint32_t x_full = bar0;
  const uint32_t y1_raw = bar0 + 8u;  // dQ: the last K tile has landed, its rows past the last key not yet zero
  auto y1_full = [&](int i) { return bar0 + 8u * (2 + i % S1); };
  auto y1_empty = [&](int i) { return bar0 + 8u * (2 + S1 + i % S1); };
  auto y2_full = [&](int i) { return bar0 + 8u * (2 + 2 * S1 + i % S2); };
  auto y2_empty = [&](int i) { return bar0 + 8u * (2 + 2 * S1 + S2 + i % S2); };
  auto y1_par = [](int i) { return (uint32_t)(i / S1) & 1u; };
  auto y2_par = [](int i) { return (uint32_t)(i / S2) & 1u; };
  constexpr int kB = 2 + 2 * S1 + 2 * S2;
  auto t1_full = [&](int i) { return bar0 + 8u * (kB + (i & 1)); };
  const uint32_t t2_full = bar0 + 8u * (kB + 2);
  const uint32_t t2_read = bar0 + 8u * (kB + 3);  // both warpgroups hold T2 in registers
  const uint32_t p_ready = bar0 + 8u * (kB + 4);
  auto ds_ready = [&](int i) { return bar0 + 8u * (kB + 5 + (i & 1)); };
  const uint32_t acc_full = bar0 + 8u * (kB + 7);
  const uint32_t drain = bar0 + 8u * (kB + 8);
  volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(base_ptr + Plan::kOffTmemHolder);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_ptr + Plan::kOffAbort);

  const int warp = (int)threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31u;
  // This CTA's tile: dK/dV: key tile of a key/value head; dQ: query tile of a head.
  const int own_tiles = kDQ ? p.q_tiles : p.kv_tiles;
  const int own_heads = kDQ ? p.heads : p.kv_heads;
  const int tile = cta % own_tiles;
  const int head = (cta / own_tiles) % own_heads;
  const int bat = (cta / own_tiles) / own_heads;

  if (warp == kAttnProducerWarp && lane == 0) {
    mbar_init(x_full, 1);
    mbar_init(y1_raw, 1);
    for (int s = 0; s < S1; ++s) {
      mbar_init(y1_full(s), 1);
      mbar_init(y1_empty(s), 1);
    }
    for (int s = 0; s < S2; ++s) {
      mbar_init(y2_full(s), 1);
      mbar_init(y2_empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(t1_full(s), 1);
      mbar_init(ds_ready(s), 8);
    }
    mbar_init(t2_full, 1);
    mbar_init(t2_read, 8);
    mbar_init(p_ready, 8);
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == kAttnMmaWarp) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_holder)), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_launch_dependents();
  pdl_wait();

  const int kv_len = attn_kv_len(p.kv_lens, bat, p.kv_len);
  const int kv_tiles = (kv_len + 127) / 128;
  // Streamed tiles: dK/dV: the query tiles of the group's heads, none for a
  // key tile past the last key; dQ: the key tiles.
  const int n = kDQ ? kv_tiles : (tile < kv_tiles ? p.group * p.q_tiles : 0);
  // dQ: rows of the last K tile past the last key, which TMA filled from memory.
  const bool clean = kDQ && kv_len < p.kv_len && kv_len % 128 != 0;
  // TMEM regions of T1 and T2 of tile i (see the head of the file).
  auto reg1 = [&](int i) { return tmem_base + (kDQ ? ((i & 1) ? 384u : 0u) : ((i & 1) ? 128u : 0u)); };
  auto reg2 = [&](int i) { return tmem_base + (kDQ ? 128u : ((i & 1) ? 0u : 128u)); };
  const uint32_t acc1 = tmem_base + 256u;
  const uint32_t acc2 = tmem_base + 384u;  // dK/dV only

  if (warp >= kAttnProducerWarp) {
    setmaxnreg_dec<kAttnRegsOther>();
    if (warp == kAttnProducerWarp) {
      // ---- TMA producer ------------------------------------------------------
      if (lane == 0 && n > 0) {
        const uint64_t pol_keep = l2_policy_evict_last();  // streamed tiles: read by many CTAs
        const uint64_t pol_once = l2_policy_evict_first();
        auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int h, int row, uint64_t pol) {
          for (int c = 0; c < 2; ++c) tma_load_4d(dst + (uint32_t)(c * 16384), map, bar, 64 * c, h, row, bat, pol);
        };
        mbar_arrive_expect_tx(x_full, 2 * Plan::kTileBytes);
        load(sX1, kDQ ? &tm.q : &tm.k, x_full, head, tile * 128, pol_once);
        load(sX2, kDQ ? &tm.dout : &tm.v, x_full, head, tile * 128, pol_once);
        int y1_issued = 0, y2_issued = 0;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
          const int y_head = kDQ ? head / p.group : head * p.group + i / p.q_tiles;
          const int y_row = (kDQ ? i : i % p.q_tiles) * 128;
          if (!mbar_wait(y1_empty(i), y1_par(i) ^ 1u, p.timeout_ns, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t y1_bar = clean && i == n - 1 ? y1_raw : y1_full(i);
          mbar_arrive_expect_tx(y1_bar, Plan::kTileBytes + (kDQ ? 0 : 1024));
          load(sY1(i), kDQ ? &tm.k : &tm.q, y1_bar, y_head, y_row, pol_keep);
          if constexpr (!kDQ) {
            const size_t at = ((size_t)bat * p.heads + y_head) * (size_t)(p.q_tiles * 128) + y_row;
            const uint32_t vec = base + (uint32_t)(Plan::kOffVec + (i % S1) * 1024);
            bulk_load(vec, p.lse2 + at, 512, y1_bar);
            bulk_load(vec + 512, p.delta + at, 512, y1_bar);
          }
          ++y1_issued;
          if (!mbar_wait(y2_empty(i), y2_par(i) ^ 1u, p.timeout_ns, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(y2_full(i), Plan::kTileBytes);
          load(sY2(i), kDQ ? &tm.v : &tm.dout, y2_full(i), y_head, y_row, pol_keep);
          ++y2_issued;
        }
        if (!ok) attn_raise(p, abort_flag, kDevTimeoutProducer);
        // Let the copies in flight land before the CTA can leave.
        bool drained = mbar_wait(x_full, 0u, p.timeout_ns, nullptr);
        for (int i = y1_issued - 1; drained && i >= 0 && i >= y1_issued - S1; --i) {
          drained = clean && i == n - 1 ? mbar_wait(y1_raw, 0u, p.timeout_ns, nullptr)
                                        : mbar_wait(y1_full(i), y1_par(i), p.timeout_ns, nullptr);
        }
        for (int i = y2_issued - 1; drained && i >= 0 && i >= y2_issued - S2; --i) {
          drained = mbar_wait(y2_full(i), y2_par(i), p.timeout_ns, nullptr);
        }
        if (!drained) attn_raise(p, abort_flag, kDevTimeoutDrain);
      }
      __syncwarp();
    } else if (warp == kAttnMmaWarp) {
      // ---- MMA issuer ----------------------------------------------------------
      if (lane == 0 && n > 0) {
        constexpr uint32_t idesc_t = idesc_bf16_f32(128, 128, false, false);  // X (K-major) x Y^T (K-major)
        constexpr uint32_t idesc_a = idesc_bf16_f32(128, 128, false, true);   // P or dS (TMEM) x Y (MN-major)
        auto kmajor = [](uint32_t t, int k) {
          return smem_desc_sw128(t + (uint32_t)((k >> 2) * 16384 + (k & 3) * 32), 16, 1024);
        };
        auto mnmajor = [](uint32_t t, int k) { return smem_desc_sw128(t + (uint32_t)(k * 2048), 16384, 1024); };
        auto product = [&](uint32_t d, uint32_t x, uint32_t y) {
#pragma unroll
          for (int k = 0; k < 8; ++k) umma_bf16(d, kmajor(x, k), kmajor(y, k), idesc_t, k > 0 ? 1u : 0u);
        };
        // A = 16-column slices of P (offset 0) or dS (offset 32) over both halves of T1.
        auto accumulate = [&](uint32_t d, uint32_t a, uint32_t y, bool first) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            umma_bf16_ts(d, a + (uint32_t)((k >> 2) * 64 + (k & 3) * 8), mnmajor(y, k), idesc_a, !first || k > 0 ? 1u : 0u);
          }
        };
        auto wait = [&](uint32_t bar, uint32_t par) {
          if (!mbar_wait(bar, par, p.timeout_ns, abort_flag)) return false;
          tc_fence_after();
          return true;
        };
        auto issue_t1 = [&](int i) {
          if (!wait(y1_full(i), y1_par(i))) return false;
          product(reg1(i), sX1, sY1(i));
          umma_commit(t1_full(i));
          return true;
        };
        auto issue_t2 = [&](int i) {
          if (!wait(y2_full(i), y2_par(i))) return false;
          product(reg2(i), sX2, sY2(i));
          umma_commit(t2_full);
          if (kDQ) umma_commit(y2_empty(i));  // its only use
          return true;
        };
        auto run = [&]() {
          if (!wait(x_full, 0u) || !issue_t1(0) || !issue_t2(0)) return false;
          if (kDQ && n > 1 && !issue_t1(1)) return false;
          for (int i = 0; i < n; ++i) {
            if constexpr (kDQ) {
              if (!wait(t2_read, (uint32_t)i & 1u)) return false;
              if (i + 1 < n && !issue_t2(i + 1)) return false;
              if (!wait(ds_ready(i), (uint32_t)(i >> 1) & 1u)) return false;
              accumulate(acc1, reg1(i) + 32u, sY1(i), i == 0);
              umma_commit(y1_empty(i));
              if (i + 2 < n && !issue_t1(i + 2)) return false;
            } else {
              if (!wait(p_ready, (uint32_t)i & 1u)) return false;
              accumulate(acc2, reg1(i), sY2(i), i == 0);
              umma_commit(y2_empty(i));
              if (!wait(t2_read, (uint32_t)i & 1u)) return false;
              if (i + 1 < n && !issue_t1(i + 1)) return false;
              if (!wait(ds_ready(i), (uint32_t)(i >> 1) & 1u)) return false;
              accumulate(acc1, reg1(i) + 32u, sY1(i), i == 0);
              umma_commit(y1_empty(i));
              if (i + 1 < n && !issue_t2(i + 1)) return false;
            }
          }
          umma_commit(acc_full);
          return true;
        };
        if (!run()) attn_raise(p, abort_flag, kDevTimeoutMma);
        umma_commit(drain);
        if (!mbar_wait(drain, 0u, p.timeout_ns, nullptr)) attn_raise(p, abort_flag, kDevTimeoutDrain);
      }
      __syncwarp();
    } else if (clean && n > 0) {
      // ---- warps 10, 11: zero the K rows past the last key ---------------------
      const bool got = mbar_wait(y1_raw, 0u, p.timeout_ns, abort_flag);
      if (__all_sync(0xffffffffu, got)) {
        const uint32_t t = sY1(n - 1);
        const int cells = (128 * n - kv_len) * 16;  // 16-byte cells, both 64-column atoms
        for (int c = (warp - kAttnMmaWarp - 1) * 32 + (int)lane; c < cells; c += 64) {
          const uint32_t dst = t + (uint32_t)(((c >> 3) & 1) * 16384 + (127 - (c >> 4)) * 128 + (c & 7) * 16);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0u) : "memory");
        }
        fence_proxy_async_smem();  // before the tensor cores read them
      } else if (lane == 0) {
        attn_raise(p, abort_flag, kDevTimeoutProducer);
      }
      named_bar_sync(1, 64);
      if (warp == kAttnMmaWarp + 1 && lane == 0) mbar_arrive(y1_full(n - 1));
      __syncwarp();
    }
  } else {
    setmaxnreg_inc<kAttnRegsSoftmax>();
    // ---- P and dS; warpgroup wg has columns 64 wg .. 64 wg + 63 -----------------
    const int wg = warp >> 2, qw = warp & 3;
    const int row = qw * 32 + (int)lane;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const uint32_t half = lane_off + (uint32_t)(wg * 64);
    float row_lse = 0.0f, row_delta = 0.0f;  // dQ: of this thread's query row
    if constexpr (kDQ) {
      const size_t at = ((size_t)bat * p.heads + head) * (size_t)(p.q_tiles * 128) + tile * 128 + row;
      row_lse = p.lse2[at];
      row_delta = p.delta[at];
    }
    // dK/dV: rows past the last key hold whatever memory holds: P = dS = 0.
    const bool partial = !kDQ && tile * 128 + 128 > kv_len;
    const bool row_ok = kDQ || tile * 128 + row < kv_len;
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t par) {
      const bool got = mbar_wait(bar, par, p.timeout_ns, abort_flag);
      ok = __all_sync(0xffffffffu, got);
      if (ok) tc_fence_after();
      return ok;
    };
    auto publish = [&](uint32_t bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int i = 0; i < n; ++i) {
      if (!wait(t1_full(i), (uint32_t)(i >> 1) & 1u)) break;
      float e[64];
      {
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(reg1(i) + half, r[0]);
        tmem_ld_32x32b_x32(reg1(i) + half + 32u, r[1]);
        tmem_ld_wait_regs(r[0]);
        tmem_ld_wait_regs(r[1]);
#pragma unroll
        for (int c = 0; c < 64; ++c) e[c] = __uint_as_float(r[c >> 5][c & 31]);
      }
      const float* vec = reinterpret_cast<const float*>(base_ptr + Plan::kOffVec + (i % S1) * 1024) + wg * 64;
      if constexpr (!kDQ) {
        // The vectors came with Y1: the wait makes them visible to this thread.
        if (!wait(y1_full(i), y1_par(i))) break;
      }
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        float4 l4 = make_float4(row_lse, row_lse, row_lse, row_lse);
        if constexpr (!kDQ) l4 = *reinterpret_cast<const float4*>(vec + c);
        const float2 sc = make_float2(p.scale_log2, p.scale_log2);
        const float2 a = __ffma2_rn(make_float2(e[c], e[c + 1]), sc, make_float2(-l4.x, -l4.y));
        const float2 b = __ffma2_rn(make_float2(e[c + 2], e[c + 3]), sc, make_float2(-l4.z, -l4.w));
        e[c] = fast_exp2(a.x);
        e[c + 1] = fast_exp2(a.y);
        e[c + 2] = fast_exp2(b.x);
        e[c + 3] = fast_exp2(b.y);
      }
      if (kDQ && i == n - 1 && n * 128 > kv_len) {
        const int lim = kv_len - i * 128 - wg * 64;
#pragma unroll
        for (int c = 0; c < 64; ++c) e[c] = c < lim ? e[c] : 0.0f;
      }
      if constexpr (!kDQ) {
        if (partial) {
#pragma unroll
          for (int c = 0; c < 64; ++c) e[c] = row_ok ? e[c] : 0.0f;
        }
        uint32_t pw[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) pw[c] = pack_bf16x2(e[2 * c], e[2 * c + 1]);
        tmem_st_32x32b_x32(reg1(i) + half, pw);
        tmem_st_wait();
        publish(p_ready);
      }
      if (!wait(t2_full, (uint32_t)i & 1u)) break;
      uint32_t dw[32];
      {
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(reg2(i) + half, r[0]);
        tmem_ld_32x32b_x32(reg2(i) + half + 32u, r[1]);
        tmem_ld_wait_regs(r[0]);
        tmem_ld_wait_regs(r[1]);
        publish(t2_read);
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          float4 d4 = make_float4(row_delta, row_delta, row_delta, row_delta);
          if constexpr (!kDQ) d4 = *reinterpret_cast<const float4*>(vec + 128 + c);
          const uint32_t* t = &r[c >> 5][c & 31];
          const float2 a = __fmul2_rn(make_float2(e[c], e[c + 1]),
                                      __fadd2_rn(make_float2(__uint_as_float(t[0]), __uint_as_float(t[1])), make_float2(-d4.x, -d4.y)));
          const float2 b = __fmul2_rn(make_float2(e[c + 2], e[c + 3]),
                                      __fadd2_rn(make_float2(__uint_as_float(t[2]), __uint_as_float(t[3])), make_float2(-d4.z, -d4.w)));
          dw[c >> 1] = pack_bf16x2(a.x, a.y);
          dw[(c >> 1) + 1] = pack_bf16x2(b.x, b.y);
        }
      }
      // 0 x (NaN - delta): masked places again, on the packed pairs.
      if (kDQ && i == n - 1 && n * 128 > kv_len) {
        const int lim = kv_len - i * 128 - wg * 64;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          dw[c] &= (2 * c < lim ? 0xffffu : 0u) | (2 * c + 1 < lim ? 0xffff0000u : 0u);
        }
      }
      if (partial) {
#pragma unroll
        for (int c = 0; c < 32; ++c) dw[c] = row_ok ? dw[c] : 0u;
      }
      tmem_st_32x32b_x32(reg1(i) + half + 32u, dw);
      tmem_st_wait();
      publish(ds_ready(i));
    }
    // ---- gradients out: acc -> bf16 -> TMA store through X1 / X2 ------------------
    // dQ: warpgroup wg stores columns 64 wg ..; dK/dV: warpgroup 0 dK, 1 dV.
    if (n > 0 && ok) wait(acc_full, 0u);
    if (ok) {
      const float f = kDQ || wg == 0 ? p.scale : 1.0f;
      const uint32_t acc = (kDQ || wg == 0 ? acc1 : acc2) + lane_off;
      const CUtensorMap* map = kDQ ? &tm.dq : (wg == 0 ? &tm.dk : &tm.dv);
#pragma unroll 1
      for (int h = 0; h < (kDQ ? 1 : 2); ++h) {
        const int col = kDQ ? wg * 64 : h * 64;
        const uint32_t stage = (wg == 0 ? sX1 : sX2) + (uint32_t)(h * 16384 + qw * 4096);
        uint32_t lo[32], hi[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(acc + (uint32_t)col, lo);
          tmem_ld_32x32b_x32(acc + (uint32_t)(col + 32), hi);
          tmem_ld_wait_regs(lo);
          tmem_ld_wait_regs(hi);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          lo[c] = n > 0 && row_ok ? __float_as_uint(__uint_as_float(lo[c]) * f) : 0u;
          hi[c] = n > 0 && row_ok ? __float_as_uint(__uint_as_float(hi[c]) * f) : 0u;
        }
        stage_row64(lo, hi, false, stage, 0u, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_4d(map, stage, col, head, tile * 128 + qw * 32, bat);
          bulk_commit_group();
        }
      }
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
    } else if (lane == 0) {
      attn_raise(p, abort_flag, kDevTimeoutEpilogue);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kAttnMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

__global__ void __launch_bounds__(kAttnThreads, 1)
    attn_bwd_kernel(const __grid_constant__ AttnBwdMaps tm, const __grid_constant__ AttnBwdParams p) {
#if B200_NO_SM100A_FEATURES
  if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, (uint32_t)kDevWrongArch);
#else
  const int cta = (int)blockIdx.x;
  if (cta < p.dkv_ctas) {
    attn_bwd_body<false>(tm, p, cta);
  } else {
    attn_bwd_body<true>(tm, p, cta - p.dkv_ctas);
  }
#endif  // B200_NO_SM100A_FEATURES
}

}  // namespace b200
