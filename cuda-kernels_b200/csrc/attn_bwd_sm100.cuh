// Gradients of cross attention for sm_100a (b200_cross_attn_bwd_bf16):
// tcgen05 + TMEM + TMA, on the layout of the forward kernel (attn_sm100.cuh).
// With P = exp(scale Q K^T - lse) and delta = rowsum(dO o O):
//   dV = P^T dO,  dS = P o (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q.
//
// attn_bwd_delta_kernel writes delta and lse (in the exp2 domain) of every
// query row, padded to whole tiles (+inf, 0: such rows get P = 0).
// attn_bwd_kernel<kDQ> runs twice, persistent, one CTA per SM, over work items:
//   dK/dV: one per 128-key tile, key/value head and batch entry, walking over
//          the 128-row query tiles of every query head of the group;
//   dQ:    one per 128-row query tile, head and batch entry, walking over the
//          key tiles of its batch entry.
// Both recompute S and dP, 4 + 3 products a tile pair where a single pass
// would need 5.  In exchange nothing is added across CTAs: the gradients of
// shared heads are sums in a fixed order, with no atomics and no fp32
// copy of dQ.  The dQ kernel starts on SMs that run out of dK/dV items.
// Items are handed out by a counter (the delta kernel zeroes it), since their
// lengths differ; the pipeline runs on from item to item: the next item's tiles load and its first
// products run while the last one's gradients are stored.  (A CTA per item: 134
// us against 115 on 8 ragged pairs of 500 queries and up to 1333 keys, 16
// heads, where an item has 4 to 11 tile pairs and start-up, epilogue and CTA
// exchange took as long as those.)
//
// Where there are fewer gradient tiles than SMs, a tile's walk is cut into parts, items
// of their own whose fp32 sums attn_bwd_merge_kernel adds in order (one entry, 2048 queries and keys, 8 query and
// 2 key/value heads: 73 us against 154; 4096 queries, 128 keys, 16 and 2 heads: 57 against 481).
//
// One body for both kinds.  X1, X2 are the item's own tiles, Y1, Y2 the
// streamed ones; rows of the products are X's rows (TMEM lanes), columns Y's:
//   dK/dV: X = K, V   Y = Q, dO   T1 = S^T, T2 = dP^T;  acc1 (dK) += dS^T Q, acc2 (dV) += P^T dO
//   dQ:    X = Q, dO  Y = K, V    T1 = S,   T2 = dP;    acc1 (dQ) += dS K
// P and dS go back to TMEM as bf16 (the A operand of the second products);
// every Y tile serves once as a K-major and once as an MN-major operand.
//
// 384 threads: warps 0..7 compute, two warpgroups of 64 columns each, one
// thread per row; warp 8 item fetch and TMA producer, warp 9 MMA issuer and
// TMEM owner.  Warps 10, 11 write the gradients of items without tiles (zeros:
// behind the keys of a padded batch that is much of the memory traffic, and here
// it runs beside the other items' products) and zero the K rows past the last
// key in a dQ item's last tile (they may hold NaN, and 0 x NaN would reach dQ).
// TMEM, 512 columns: a warpgroup puts P and dS over its own half of T1, so no
// warp waits for another.  dK/dV: T1 and T2 swap two regions from tile to
// tile, T1 of the next tile being computed while dS of this one is.  dQ: T1
// has two regions of its own, a tile ahead, T2 a third.
// A steady tile pair takes 2.0 us in dK/dV and 1.5 in dQ, 0.49 us a product
// either way: the rate at which this chip runs 128 x 128 x 128 products from one
// CTA per SM, with or without the softmax (1300 TFLOP/s, as in the forward kernel).
// Every wait is bounded, as in the forward kernel.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>

#include "attn_sm100.cuh"
#include "gemm_sm100.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

// A gradient tensor [batch, tokens, heads, 128], strides in elements.
struct AttnGrad {
  __nv_bfloat16* data;
  int64_t batch_stride, seq_stride, head_stride;
};

struct AttnBwdParams {
  int32_t q_len, kv_len, heads, kv_heads, group, batch;
  int32_t q_tiles, kv_tiles;
  int32_t items;           // of this kernel's kind
  int32_t parts;           // items a tile's walk is cut into; their sums are added by attn_bwd_merge_kernel
  float* part;             // with several parts: [batch, heads, tiles, parts][dK and dV, or dQ][8 warps][16][32] float4
  uint32_t ordered;        // entries by falling number of keys (more items than SMs, at most 32 entries)
  uint32_t early;          // dQ: launched behind the dK/dV kernel, of which it needs nothing
  const int32_t* kv_lens;  // [batch] or NULL
  float scale, scale_log2;
  // [batch * heads][q_tiles * 128], of attn_bwd_delta_kernel.
  const float* lse2;
  const float* delta;
  uint32_t* counter;       // items handed out beyond the first gridDim.x
  AttnGrad dq, dk, dv;
  uint64_t timeout_ns;
  uint32_t* status;
};

struct AttnBwdMaps {
  CUtensorMap q, k, v, dout;
};

// An item's share of a walk over n tiles: [first, second).
__host__ __device__ __forceinline__ int bwd_part_begin(int n, int part, int parts) {
  return (int)((int64_t)n * part / parts);
}

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
  uint32_t* counters;            // two, zeroed for attn_bwd_kernel
};

// Half a warp per query row, 16 bytes of O and dO a lane, four rows in flight
// per half: bound by reading both once.
__global__ void __launch_bounds__(256) attn_bwd_delta_kernel(const __grid_constant__ AttnBwdDeltaParams p) {
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x < 2) p.counters[threadIdx.x] = 0u;
  const int lane = (int)(threadIdx.x & 15u), sub = (int)threadIdx.x >> 4;
  const int bh = (int)blockIdx.y + 65535 * (int)blockIdx.z;
  if (bh >= p.rows) return;
  const int head = bh % p.heads;
  const int64_t bat = bh / p.heads;
  // 64 rows per block: rows sub, sub + 16, sub + 32, sub + 48.
  uint4 a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (int)blockIdx.x * 64 + sub + 16 * i;
    a[i] = b[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < p.q_len) {
      a[i] = *reinterpret_cast<const uint4*>(p.o + bat * p.o_batch + row * p.o_seq + head * p.o_head + 8 * lane);
      b[i] = *reinterpret_cast<const uint4*>(p.dout + bat * p.d_batch + row * p.d_seq + head * p.d_head + 8 * lane);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (int)blockIdx.x * 64 + sub + 16 * i;
    const uint32_t x[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, y[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sum = fmaf(__uint_as_float(x[k] << 16), __uint_as_float(y[k] << 16), sum);
      sum = fmaf(__uint_as_float(x[k] & 0xffff0000u), __uint_as_float(y[k] & 0xffff0000u), sum);
    }
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (lane == 0 && row < p.padded) {
      p.lse2[(size_t)bh * p.padded + row] = row < p.q_len ? p.lse[(size_t)bh * p.q_len + row] * 1.4426950408889634f : INFINITY;
      p.delta[(size_t)bh * p.padded + row] = sum;
    }
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
  // dK/dV: 2 KiB per computing warp for its gradient rows on their way out.
  static constexpr int kOffOut = kOffVec + (kDQ ? 0 : kY1Stages * 1024);
  static constexpr int kOffBar = kOffOut + (kDQ ? 0 : 8 * 2048);
  static constexpr int kNumBars = 2 + 3 * kY1Stages + 2 * kY2Stages + 2 + 1 + 1 + 1 + 2 + 1 + 1 + 4;
  static constexpr int kOffItem = (kOffBar + kNumBars * 8 + 15) / 16 * 16;  // two slots of an Item
  static constexpr int kOffOrder = kOffItem + 64;  // batches of up to 32: the entries by falling number of keys
  static constexpr int kOffTmemHolder = kOffOrder + 32 * 4;
  static constexpr int kOffAbort = kOffTmemHolder + 4;
  static constexpr int kBytes = kOffAbort + 4;
  static constexpr int kAllocBytes = kBytes + 1024;
  static_assert(kAllocBytes <= 232448, "attention backward shared memory plan exceeds 227 KiB");
};

// 32 rows x 64 columns of a gradient, a row per lane in fp32 registers, times f,
// as bf16.  Lanes that store their own rows, 16 bytes of 32 rows at a time, take
// 1.6 us a tile, so the lanes exchange first and then store whole rows: dK/dV
// through 2 KiB of shared memory per warp, 32 columns at a time (four lanes per
// row); dQ, whose third K stage leaves no room for that, by three exchanges
// within groups of eight lanes (eight lanes per row; 1.1 us).  Rows from `rows` on are
// not stored.
template <bool kDQ>
__device__ __forceinline__ void store_grad(const AttnGrad& g, int bat, int row0, int rows, int head, int col, uint32_t lane,
                                           const uint32_t (&lo)[32], const uint32_t (&hi)[32], float f, uint32_t buf) {
  uint32_t w[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t* v = j < 4 ? &lo[8 * j] : &hi[8 * (j - 4)];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[j][k] = pack_bf16x2(__uint_as_float(v[2 * k]) * f, __uint_as_float(v[2 * k + 1]) * f);
  }
  __nv_bfloat16* dst = g.data + bat * g.batch_stride + head * g.head_stride + col;
  if constexpr (!kDQ) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // 64 bytes a row; the 16-byte cells are permuted so that both directions touch every bank once.
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = buf + lane * 64u + (((uint32_t)j ^ ((lane >> 1) & 3u)) << 4);
        const uint32_t* v = w[4 * h + j];
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t r = (uint32_t)(8 * i) + (lane >> 2), c = lane & 3u;
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(buf + r * 64u + ((c ^ ((r >> 1) & 3u)) << 4))
                     : "memory");
        const int row = row0 + (int)r;
        if (row < rows) *reinterpret_cast<uint4*>(dst + row * g.seq_stride + 32 * h + 8 * (int)c) = v;
      }
      __syncwarp();
    }
  } else {
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
      const bool upper = (lane & (uint32_t)d) != 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j & d) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[j][k] : w[j | d][k], d);
          if (upper) {
            w[j][k] = got;
          } else {
            w[j | d][k] = got;
          }
        }
      }
    }
    const int first = row0 + (int)(lane & 24u);
    dst += first * g.seq_stride + 8 * (lane & 7u);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (first + j < rows) *reinterpret_cast<uint4*>(dst + j * g.seq_stride) = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
    }
  }
}

// The same of zeros.
__device__ __forceinline__ void store_zeros(const AttnGrad& g, int bat, int row0, int rows, int head, int col, uint32_t lane) {
  const int first = row0 + (int)(lane >> 3);
  __nv_bfloat16* dst = g.data + bat * g.batch_stride + head * g.head_stride + first * g.seq_stride + col + 8 * (lane & 7u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (first + 4 * i < rows) *reinterpret_cast<uint4*>(dst + 4 * i * g.seq_stride) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <bool kDQ>
__global__ void __launch_bounds__(kAttnThreads, 1)
    attn_bwd_kernel(const __grid_constant__ AttnBwdMaps tm, const __grid_constant__ AttnBwdParams p) {
#if B200_NO_SM100A_FEATURES
  if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, (uint32_t)kDevWrongArch);
#else
  using Plan = AttnBwdPlan<kDQ>;
  constexpr int S1 = Plan::kY1Stages, S2 = Plan::kY2Stages;
  constexpr int kReaders = 11;  // of an item: MMA issuer, 8 computing warps, warps 10 and 11
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_u32);
  const uint32_t sX1 = base + Plan::kOffX1, sX2 = base + Plan::kOffX2;
  // Tile pairs are counted over all of the CTA's items: g.
  auto sY1 = [&](uint32_t g) { return base + (uint32_t)Plan::kOffY1 + (g % S1) * (uint32_t)Plan::kTileBytes; };
  auto sY2 = [&](uint32_t g) { return base + (uint32_t)Plan::kOffY2 + (g % S2) * (uint32_t)Plan::kTileBytes; };
  const uint32_t bar0 = base + Plan::kOffBar;
  const uint32_t x_full = bar0, x_empty = bar0 + 8u;
  auto y1_full = [&](uint32_t g) { return bar0 + 8u * (2 + g % S1); };
  auto y1_empty = [&](uint32_t g) { return bar0 + 8u * (2 + S1 + g % S1); };
  // dQ: an item's last K tile has landed, its rows past the last key not yet
  // zero; y1_full then comes from the cleaning warps.  One per stage, and its
  // phase counted by its uses: a stage is not used again before it was cleaned.
  auto y1_raw = [&](uint32_t g) { return bar0 + 8u * (2 + 2 * S1 + g % S1); };
  auto y2_full = [&](uint32_t g) { return bar0 + 8u * (2 + 3 * S1 + g % S2); };
  auto y2_empty = [&](uint32_t g) { return bar0 + 8u * (2 + 3 * S1 + S2 + g % S2); };
  auto y1_par = [](uint32_t g) { return (g / S1) & 1u; };
  auto y2_par = [](uint32_t g) { return (g / S2) & 1u; };
  constexpr int kB = 2 + 3 * S1 + 2 * S2;
  auto t1_full = [&](uint32_t g) { return bar0 + 8u * (kB + (g & 1u)); };
  const uint32_t t2_full = bar0 + 8u * (kB + 2);
  const uint32_t t2_read = bar0 + 8u * (kB + 3);  // both warpgroups hold T2 in registers
  const uint32_t p_ready = bar0 + 8u * (kB + 4);
  auto ds_ready = [&](uint32_t g) { return bar0 + 8u * (kB + 5 + (g & 1u)); };
  const uint32_t acc_full = bar0 + 8u * (kB + 7);
  const uint32_t drain = bar0 + 8u * (kB + 8);
  auto item_full = [&](uint32_t k) { return bar0 + 8u * (kB + 9 + (k & 1u)); };
  auto item_empty = [&](uint32_t k) { return bar0 + 8u * (kB + 11 + (k & 1u)); };
  volatile int32_t* order = reinterpret_cast<volatile int32_t*>(base_ptr + Plan::kOffOrder);
  volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(base_ptr + Plan::kOffTmemHolder);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_ptr + Plan::kOffAbort);

  const int warp = (int)threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31u;

  if (warp == kAttnProducerWarp && lane == 0) {
    mbar_init(x_full, 1);
    mbar_init(x_empty, 1);
    for (uint32_t s = 0; s < (uint32_t)S1; ++s) {
      mbar_init(y1_full(s), 1);
      mbar_init(y1_empty(s), 1);
      mbar_init(y1_raw(s), 1);
    }
    for (uint32_t s = 0; s < (uint32_t)S2; ++s) {
      mbar_init(y2_full(s), 1);
      mbar_init(y2_empty(s), 1);
    }
    for (uint32_t s = 0; s < 2; ++s) {
      mbar_init(t1_full(s), 1);
      mbar_init(ds_ready(s), 8);
      mbar_init(item_full(s), 1);
      mbar_init(item_empty(s), kReaders);
    }
    mbar_init(t2_full, 1);
    mbar_init(t2_read, 8);
    mbar_init(p_ready, 8);
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0u;
    fence_mbar_init();
    tma_prefetch_desc(&tm.q);
    tma_prefetch_desc(&tm.k);
    tma_prefetch_desc(&tm.v);
    tma_prefetch_desc(&tm.dout);
  }
  if (warp == kAttnMmaWarp) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_holder)), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  // The dK/dV kernel lets the next one start only after its own wait: a dQ CTA
  // behind it then runs when all that came before both has completed, and
  // needs no wait of its own (until the end, below).
  if (!(kDQ && p.early != 0u)) pdl_wait();
  pdl_launch_dependents();
  if (p.ordered) {
    if (warp < 8) {
      for (int slot = warp; slot < p.batch; slot += 8) {
        const int e = attn_entry_by_length(p.kv_lens, p.batch, p.kv_len, slot);
        if (lane == 0) order[slot] = e;
      }
    }
    __syncthreads();
  }

  // An item, worked out by the producer and read by the others from shared memory.
  // Entries with many keys come first, so that the last items are short.  Tiles
  // change fastest: neighbours stream the same tiles.  (Entries fastest, so
  // that long and short ones alternate: 4 % slower on 8 ragged pairs.)
  struct alignas(16) Item {
    int tile, part, head, bat;
    int i0, n;   // the tiles of its walk
    int kv_len;  // keys of its entry
    int flags;   // 1: no item, the end; 2: dQ, the last K tile has rows past the last key, which TMA filled from memory
    __device__ bool clean() const { return (flags & 2) != 0; }
  };
  static_assert(sizeof(Item) == 32, "two 16-byte words of shared memory");
  auto item_at = [&](uint32_t k) { return reinterpret_cast<int4*>(base_ptr + Plan::kOffItem + (k & 1u) * 32u); };
  auto item_of = [&](int id) {
    const int tiles = kDQ ? p.q_tiles : p.kv_tiles, heads = kDQ ? p.heads : p.kv_heads;
    Item t{};
    if (id >= p.items) {
      t.flags = 1;
      return t;
    }
    t.tile = id % tiles;
    id /= tiles;
    t.part = id % p.parts;
    id /= p.parts;
    t.head = id % heads;
    t.bat = id / heads;
    if (p.ordered) t.bat = order[t.bat];
    t.kv_len = attn_kv_len(p.kv_lens, t.bat, p.kv_len);
    const int kv_tiles = (t.kv_len + 127) / 128;
    const int walk = kDQ ? kv_tiles : (t.tile < kv_tiles ? p.group * p.q_tiles : 0);
    t.i0 = bwd_part_begin(walk, t.part, p.parts);
    t.n = bwd_part_begin(walk, t.part + 1, p.parts) - t.i0;
    if (kDQ && t.i0 + t.n == walk && t.kv_len < p.kv_len && t.kv_len % 128 != 0) t.flags = 2;
    return t;
  };
  auto read_item = [&](uint32_t k, Item* t) {
    const int4 a = item_at(k)[0], b = item_at(k)[1];
    t->tile = a.x, t->part = a.y, t->head = a.z, t->bat = a.w;
    t->i0 = b.x, t->n = b.y, t->kv_len = b.z, t->flags = b.w;
  };
  // The k-th item of this CTA, for one reader (a warp, or the MMA lane); false at the end.
  auto next_item = [&](uint32_t k, bool whole_warp, Item* t, bool* ok) {
    bool got = mbar_wait(item_full(k), (k >> 1) & 1u, p.timeout_ns, abort_flag);
    if (whole_warp) got = __all_sync(0xffffffffu, got);
    if (!got) {
      *ok = false;
      return false;
    }
    read_item(k, t);
    if (whole_warp) __syncwarp();
    if (!whole_warp || lane == 0) mbar_arrive(item_empty(k));
    return (t->flags & 1) == 0;
  };
  // TMEM regions of T1 and T2 of tile pair g (see the head of the file).
  auto reg1 = [&](uint32_t g) { return tmem_base + (kDQ ? ((g & 1u) ? 384u : 0u) : ((g & 1u) ? 128u : 0u)); };
  auto reg2 = [&](uint32_t g) { return tmem_base + (kDQ ? 128u : ((g & 1u) ? 0u : 128u)); };
  const uint32_t acc1 = tmem_base + 256u;
  const uint32_t acc2 = tmem_base + 384u;  // dK/dV only

  if (warp >= kAttnProducerWarp) {
    setmaxnreg_dec<kAttnRegsOther>();
    if (warp == kAttnProducerWarp) {
      // ---- item fetch and TMA producer ----------------------------------------
      if (lane == 0) {
        const uint64_t pol_keep = l2_policy_evict_last();  // streamed tiles: read by many CTAs
        const uint64_t pol_once = l2_policy_evict_first();
        uint32_t g = 0, filled = 0;  // tile pairs, items with tiles so far
        uint32_t raw_par = 0;        // parity of each stage's next raw phase
        bool ok = true, raw_last = false;
        uint32_t y2_issued = 0;
        int id = (int)blockIdx.x;
        for (uint32_t k = 0;; ++k) {
          if (!mbar_wait(item_empty(k), ((k >> 1) & 1u) ^ 1u, p.timeout_ns, abort_flag)) {
            ok = false;
            break;
          }
          const Item t = item_of(id);
          item_at(k)[0] = make_int4(t.tile, t.part, t.head, t.bat);
          item_at(k)[1] = make_int4(t.i0, t.n, t.kv_len, t.flags);
          mbar_arrive(item_full(k));
          if (t.flags & 1) break;
          id = (int)(gridDim.x + atomicAdd(p.counter, 1u));  // the next one
          if (t.n == 0) continue;
          auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int h, int row, uint64_t pol) {
            for (int c = 0; c < 2; ++c) tma_load_4d(dst + (uint32_t)(c * 16384), map, bar, 64 * c, h, row, t.bat, pol);
          };
          if (!mbar_wait(x_empty, (filled & 1u) ^ 1u, p.timeout_ns, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(x_full, 2 * Plan::kTileBytes);
          load(sX1, kDQ ? &tm.q : &tm.k, x_full, t.head, t.tile * 128, pol_once);
          load(sX2, kDQ ? &tm.dout : &tm.v, x_full, t.head, t.tile * 128, pol_once);
          ++filled;
          for (int i = t.i0; i < t.i0 + t.n; ++i) {
            const int y_head = kDQ ? t.head / p.group : t.head * p.group + i / p.q_tiles;
            const int y_row = (kDQ ? i : i % p.q_tiles) * 128;
            if (!mbar_wait(y1_empty(g), y1_par(g) ^ 1u, p.timeout_ns, abort_flag)) {
              ok = false;
              break;
            }
            raw_last = t.clean() && i == t.i0 + t.n - 1;
            const uint32_t y1_bar = raw_last ? y1_raw(g) : y1_full(g);
            mbar_arrive_expect_tx(y1_bar, Plan::kTileBytes + (kDQ ? 0 : 1024));
            load(sY1(g), kDQ ? &tm.k : &tm.q, y1_bar, y_head, y_row, pol_keep);
            if constexpr (!kDQ) {
              const size_t at = ((size_t)t.bat * p.heads + y_head) * (size_t)(p.q_tiles * 128) + y_row;
              const uint32_t vec = base + (uint32_t)Plan::kOffVec + (g % S1) * 1024u;
              bulk_load(vec, p.lse2 + at, 512, y1_bar);
              bulk_load(vec + 512, p.delta + at, 512, y1_bar);
            }
            if (raw_last) raw_par ^= 1u << (g % S1);
            ++g;
            if (!mbar_wait(y2_empty(g - 1), y2_par(g - 1) ^ 1u, p.timeout_ns, abort_flag)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(y2_full(g - 1), Plan::kTileBytes);
            load(sY2(g - 1), kDQ ? &tm.v : &tm.dout, y2_full(g - 1), y_head, y_row, pol_keep);
            ++y2_issued;
          }
          if (!ok) break;
        }
        if (!ok) attn_raise(p, abort_flag, kDevTimeoutProducer);
        // Let the copies in flight land before the CTA can leave.  (A raw tile
        // other than the last was waited for by its cleaners, whose y1_full is
        // waited for here.)
        bool drained = filled == 0 || mbar_wait(x_full, (filled - 1) & 1u, p.timeout_ns, nullptr);
        if (raw_last) {
          drained = drained && mbar_wait(y1_raw(g - 1), ((raw_par >> ((g - 1) % S1)) & 1u) ^ 1u, p.timeout_ns, nullptr);
        }
        for (uint32_t i = g; drained && i > 0 && i + S1 > g; --i) {
          if (raw_last && i == g) continue;
          drained = mbar_wait(y1_full(i - 1), y1_par(i - 1), p.timeout_ns, nullptr);
        }
        for (uint32_t i = y2_issued; drained && i > 0 && i + S2 > y2_issued; --i) {
          drained = mbar_wait(y2_full(i - 1), y2_par(i - 1), p.timeout_ns, nullptr);
        }
        if (!drained) attn_raise(p, abort_flag, kDevTimeoutDrain);
      }
      __syncwarp();
    } else if (warp == kAttnMmaWarp) {
      // ---- MMA issuer ----------------------------------------------------------
      if (lane == 0) {
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
        auto issue_t1 = [&](uint32_t g) {
          if (!wait(y1_full(g), y1_par(g))) return false;
          product(reg1(g), sX1, sY1(g));
          umma_commit(t1_full(g));
          return true;
        };
        // T2 is the last of a tile pair's products to read X.
        auto issue_t2 = [&](uint32_t g, bool last) {
          if (!wait(y2_full(g), y2_par(g))) return false;
          product(reg2(g), sX2, sY2(g));
          umma_commit(t2_full);
          if (kDQ) umma_commit(y2_empty(g));  // its only use
          if (last) umma_commit(x_empty);
          return true;
        };
        auto run = [&](uint32_t g0, uint32_t filled, int n) {
          if (!wait(x_full, filled & 1u) || !issue_t1(g0)) return false;
          if (kDQ && n > 1 && !issue_t2(g0, false)) return false;
          if (kDQ && n > 1 && !issue_t1(g0 + 1)) return false;
          if (!(kDQ && n > 1) && !issue_t2(g0, n == 1)) return false;
          for (int i = 0; i < n; ++i) {
            const uint32_t g = g0 + (uint32_t)i;
            const bool next = i + 1 < n, next_last = i + 2 == n;
            if constexpr (kDQ) {
              if (!wait(t2_read, g & 1u)) return false;
              if (next && !issue_t2(g + 1, next_last)) return false;
              if (!wait(ds_ready(g), (g >> 1) & 1u)) return false;
              accumulate(acc1, reg1(g) + 32u, sY1(g), i == 0);
              umma_commit(y1_empty(g));
              if (i + 2 < n && !issue_t1(g + 2)) return false;
            } else {
              if (!wait(p_ready, g & 1u)) return false;
              accumulate(acc2, reg1(g), sY2(g), i == 0);
              umma_commit(y2_empty(g));
              if (!wait(t2_read, g & 1u)) return false;
              if (next && !issue_t1(g + 1)) return false;
              if (!wait(ds_ready(g), (g >> 1) & 1u)) return false;
              accumulate(acc1, reg1(g) + 32u, sY1(g), i == 0);
              umma_commit(y1_empty(g));
              if (next && !issue_t2(g + 1, next_last)) return false;
            }
          }
          umma_commit(acc_full);
          return true;
        };
        bool ok = true;
        uint32_t g = 0, filled = 0;
        Item t;
        for (uint32_t k = 0; ok && next_item(k, false, &t, &ok); ++k) {
          if (t.n == 0) continue;
          ok = run(g, filled, t.n);
          g += (uint32_t)t.n;
          ++filled;
        }
        if (!ok) attn_raise(p, abort_flag, kDevTimeoutMma);
        umma_commit(drain);
        if (!mbar_wait(drain, 0u, p.timeout_ns, nullptr)) attn_raise(p, abort_flag, kDevTimeoutDrain);
      }
      __syncwarp();
    } else {
      // ---- warps 10, 11: gradients that are zero; K rows past an item's last key ----
      // Every decision is made by both warps together (a barrier that also
      // carries it), so that neither waits for the other at a later one.
      auto both = [&](bool mine) { return named_bar_and(1, 64, __all_sync(0xffffffffu, mine)); };
      uint32_t g = 0, raw_par = 0;
      bool ok = true;
      for (uint32_t k = 0;; ++k) {
        ok = both(mbar_wait(item_full(k), (k >> 1) & 1u, p.timeout_ns, abort_flag));
        if (!ok) break;
        Item t;
        read_item(k, &t);
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty(k));
        if (t.flags & 1) break;
        if (t.n == 0) {
          if (p.parts > 1) continue;  // (the merge knows)
#pragma unroll 1
          for (int part = warp - kAttnMmaWarp - 1; part < 8; part += 2) {  // 32 rows x 64 columns
            const int row0 = t.tile * 128 + (part >> 1) * 32, rows = kDQ ? p.q_len : p.kv_len, col = (part & 1) * 64;
            store_zeros(kDQ ? p.dq : p.dk, t.bat, row0, rows, t.head, col, lane);
            if constexpr (!kDQ) store_zeros(p.dv, t.bat, row0, rows, t.head, col, lane);
          }
          continue;
        }
        g += (uint32_t)t.n;
        if (!t.clean()) continue;
        const uint32_t last = g - 1;
        ok = both(mbar_wait(y1_raw(last), (raw_par >> (last % S1)) & 1u, p.timeout_ns, abort_flag));
        if (!ok) break;
        raw_par ^= 1u << (last % S1);
        const int cells = (128 * (t.i0 + t.n) - t.kv_len) * 16;  // 16-byte cells, both 64-column atoms
        for (int c = (warp - kAttnMmaWarp - 1) * 32 + (int)lane; c < cells; c += 64) {
          const uint32_t dst = sY1(last) + (uint32_t)(((c >> 3) & 1) * 16384 + (127 - (c >> 4)) * 128 + (c & 7) * 16);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0u) : "memory");
        }
        fence_proxy_async_smem();  // before the tensor cores read them
        both(true);
        if (warp == kAttnMmaWarp + 1 && lane == 0) mbar_arrive(y1_full(last));
      }
      if (!ok && lane == 0) attn_raise(p, abort_flag, kDevTimeoutProducer);
      __syncwarp();
    }
  } else {
    setmaxnreg_inc<kAttnRegsSoftmax>();
    // ---- P and dS; warpgroup wg has columns 64 wg .. 64 wg + 63 -----------------
    const int wg = warp >> 2, qw = warp & 3;
    const int row = qw * 32 + (int)lane;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const uint32_t half = lane_off + (uint32_t)(wg * 64);
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
    uint32_t g0 = 0, filled = 0;
    Item t;
    for (uint32_t k = 0; ok && next_item(k, true, &t, &ok); ++k) {
      const int kv_len = t.kv_len, n = t.n;
      if (n == 0) continue;
      const int kv_left = kv_len - t.i0 * 128;  // dQ: keys from the item's first tile on
      float row_lse = 0.0f, row_delta = 0.0f;  // dQ: of this thread's query row
      if constexpr (kDQ) {
        const size_t at = ((size_t)t.bat * p.heads + t.head) * (size_t)(p.q_tiles * 128) + t.tile * 128 + row;
        row_lse = p.lse2[at];
        row_delta = p.delta[at];
      }
      // dK/dV: rows past the last key hold whatever memory holds: P = dS = 0.
      const bool partial = !kDQ && t.tile * 128 + 128 > kv_len;
      const bool row_ok = kDQ || t.tile * 128 + row < kv_len;
      for (int i = 0; i < n; ++i) {
        const uint32_t g = g0 + (uint32_t)i;
        if (!wait(t1_full(g), (g >> 1) & 1u)) break;
        float e[64];
        {
          uint32_t r[2][32];
          tmem_ld_32x32b_x32(reg1(g) + half, r[0]);
          tmem_ld_32x32b_x32(reg1(g) + half + 32u, r[1]);
          tmem_ld_wait_regs(r[0]);
          tmem_ld_wait_regs(r[1]);
#pragma unroll
          for (int c = 0; c < 64; ++c) e[c] = __uint_as_float(r[c >> 5][c & 31]);
        }
        const float* vec = reinterpret_cast<const float*>(base_ptr + Plan::kOffVec + (g % S1) * 1024u) + wg * 64;
        if constexpr (!kDQ) {
          // The vectors came with Y1: the wait makes them visible to this thread.
          if (!wait(y1_full(g), y1_par(g))) break;
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
        if (kDQ && i == n - 1 && n * 128 > kv_left) {
          const int lim = kv_left - i * 128 - wg * 64;
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
          tmem_st_32x32b_x32(reg1(g) + half, pw);
          tmem_st_wait();
          publish(p_ready);
        }
        if (!wait(t2_full, g & 1u)) break;
        uint32_t dw[32];
        {
          uint32_t r[2][32];
          tmem_ld_32x32b_x32(reg2(g) + half, r[0]);
          tmem_ld_32x32b_x32(reg2(g) + half + 32u, r[1]);
          tmem_ld_wait_regs(r[0]);
          tmem_ld_wait_regs(r[1]);
          publish(t2_read);
#pragma unroll
          for (int c = 0; c < 64; c += 4) {
            float4 d4 = make_float4(row_delta, row_delta, row_delta, row_delta);
            if constexpr (!kDQ) d4 = *reinterpret_cast<const float4*>(vec + 128 + c);
            const uint32_t* v = &r[c >> 5][c & 31];
            const float2 a = __fmul2_rn(make_float2(e[c], e[c + 1]),
                                        __fadd2_rn(make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])), make_float2(-d4.x, -d4.y)));
            const float2 b = __fmul2_rn(make_float2(e[c + 2], e[c + 3]),
                                        __fadd2_rn(make_float2(__uint_as_float(v[2]), __uint_as_float(v[3])), make_float2(-d4.z, -d4.w)));
            dw[c >> 1] = pack_bf16x2(a.x, a.y);
            dw[(c >> 1) + 1] = pack_bf16x2(b.x, b.y);
          }
        }
        // 0 x (NaN - delta): masked places again, on the packed pairs.
        if (kDQ && i == n - 1 && n * 128 > kv_left) {
          const int lim = kv_left - i * 128 - wg * 64;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            dw[c] &= (2 * c < lim ? 0xffffu : 0u) | (2 * c + 1 < lim ? 0xffff0000u : 0u);
          }
        }
        if (partial) {
#pragma unroll
          for (int c = 0; c < 32; ++c) dw[c] = row_ok ? dw[c] : 0u;
        }
        tmem_st_32x32b_x32(reg1(g) + half + 32u, dw);
        tmem_st_wait();
        publish(ds_ready(g));
      }
      if (!ok) break;
      // ---- the item's gradients: acc -> bf16 -> global memory, columns 64 wg .. of each ----
      // (The next item's P or dS of this warp comes after its loads here, so
      // the accumulators are not overwritten before.)
      if (!wait(acc_full, filled & 1u)) break;
      const int rows = kDQ ? p.q_len : p.kv_len;
#pragma unroll 1
      for (int h = 0; h < (kDQ ? 1 : 2); ++h) {
        const AttnGrad& grad = kDQ ? p.dq : (h == 0 ? p.dk : p.dv);
        uint32_t lo[32], hi[32];
        const uint32_t acc = (h == 0 ? acc1 : acc2) + half;
        tmem_ld_32x32b_x32(acc, lo);
        tmem_ld_32x32b_x32(acc + 32u, hi);
        tmem_ld_wait_regs(lo);
        tmem_ld_wait_regs(hi);
        if (!row_ok) {
#pragma unroll
          for (int c = 0; c < 32; ++c) lo[c] = hi[c] = 0u;
        }
        if (p.parts > 1) {
          const int tiles = kDQ ? p.q_tiles : p.kv_tiles, heads = kDQ ? p.heads : p.kv_heads;
          const int64_t slot = (((int64_t)t.bat * heads + t.head) * tiles + t.tile) * p.parts + t.part;
          float4* dst = reinterpret_cast<float4*>(p.part) + ((slot * (kDQ ? 1 : 2) + h) * 8 + warp) * 512 + lane;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            dst[c * 32] = make_float4(__uint_as_float(lo[4 * c]), __uint_as_float(lo[4 * c + 1]), __uint_as_float(lo[4 * c + 2]),
                                      __uint_as_float(lo[4 * c + 3]));
            dst[(c + 8) * 32] = make_float4(__uint_as_float(hi[4 * c]), __uint_as_float(hi[4 * c + 1]),
                                            __uint_as_float(hi[4 * c + 2]), __uint_as_float(hi[4 * c + 3]));
          }
          continue;
        }
        store_grad<kDQ>(grad, t.bat, t.tile * 128 + qw * 32, rows, t.head, wg * 64, lane, lo, hi, h == 0 ? p.scale : 1.0f,
                        base + (uint32_t)(Plan::kOffOut + warp * 2048));
      }
      tc_fence_before();
      g0 += (uint32_t)n;
      ++filled;
    }
    if (!ok && lane == 0) attn_raise(p, abort_flag, kDevTimeoutEpilogue);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kAttnMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  // Started early: what follows this kernel must find the dK/dV kernel complete too.
  if (kDQ && p.early != 0u) pdl_wait();
#endif  // B200_NO_SM100A_FEATURES
}

struct AttnBwdMergeParams {
  // Of dK and dV (0) and of dQ (1): parts 1 means the gradients are there already.
  const float* part[2];
  int32_t parts[2], tiles[2], heads[2];
  int32_t blocks;          // of dK and dV
  int32_t q_len, kv_len, walk;  // walk: tile pairs of a dK/dV tile
  const int32_t* kv_lens;
  AttnGrad dq, dk, dv;
  float scale;
};

// Adds the parts of each gradient tile in order.  A thread has 8 columns of a
// row, 8 lanes a row's 64 columns, a block 16 rows of one tile: loads in runs
// of 64 bytes, stores of 128.
__global__ void __launch_bounds__(256) attn_bwd_merge_kernel(const __grid_constant__ AttnBwdMergeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int kind = (int)blockIdx.x < p.blocks ? 0 : 1;
  int64_t id = kind == 0 ? blockIdx.x : blockIdx.x - p.blocks;
  const int slice = (int)(id & 7);
  id >>= 3;
  const int grads = kind == 0 ? 2 : 1;
  const int h = (int)(id % grads);
  const int64_t slot = id / grads;
  const int tile = (int)(slot % p.tiles[kind]), head = (int)(slot / p.tiles[kind] % p.heads[kind]);
  const int bat = (int)(slot / p.tiles[kind] / p.heads[kind]);
  const int lane = (int)(threadIdx.x & 31u), warp = (int)(threadIdx.x >> 5);
  // Of the tile: four rows a warp, 64 columns of its computing warp.
  const int r = slice * 16 + (warp & 3) * 4 + (lane & 3), c = lane >> 2, wg = warp >> 2;
  const int kv_len = attn_kv_len(p.kv_lens, bat, p.kv_len), kv_tiles = (kv_len + 127) / 128;
  const int walk = kind == 1 ? kv_tiles : (tile < kv_tiles ? p.walk : 0);
  const int parts = p.parts[kind];
  const float4* src = reinterpret_cast<const float4*>(p.part[kind]) + (slot * parts * grads + h) * 4096 +
                      (wg * 4 + (r >> 5)) * 512 + c * 64 + (r & 31);
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
  for (int s0 = 0; s0 < parts; s0 += 4) {
    float4 x[4], y[4];
    bool has[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i;
      has[i] = s < parts && bwd_part_begin(walk, s, parts) < bwd_part_begin(walk, s + 1, parts);  // else not written
      x[i] = y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (has[i]) {
        x[i] = src[(int64_t)s * grads * 4096];
        y[i] = src[(int64_t)s * grads * 4096 + 32];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a.x += x[i].x, a.y += x[i].y, a.z += x[i].z, a.w += x[i].w;
      b.x += y[i].x, b.y += y[i].y, b.z += y[i].z, b.w += y[i].w;
    }
  }
  const AttnGrad& g = kind == 1 ? p.dq : (h == 0 ? p.dk : p.dv);
  const float f = h == 0 ? p.scale : 1.0f;
  const int row = tile * 128 + r;
  if (row < (kind == 1 ? p.q_len : p.kv_len)) {
    *reinterpret_cast<uint4*>(g.data + bat * g.batch_stride + row * g.seq_stride + head * g.head_stride + wg * 64 + c * 8) =
        make_uint4(pack_bf16x2(a.x * f, a.y * f), pack_bf16x2(a.z * f, a.w * f), pack_bf16x2(b.x * f, b.y * f),
                   pack_bf16x2(b.z * f, b.w * f));
  }
}

}  // namespace b200
