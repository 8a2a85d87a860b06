// Attention of few query rows over long stored keys and values, for sm_100a:
// the serving step of a decoder.  Two sources of K and V:
//   kFp8 = true   the paged e4m3 cache (b200_cache_attn_e4m3): queries are the
//                 last tokens of their sequence and see the places up to theirs;
//   kFp8 = false  bf16 states of another length (b200_cross_attn_bf16 with few
//                 queries): every query sees all keys of its batch entry.
//
// The work is bound by reading K and V once (256 or 512 bytes per key and
// key/value head), so the query rows that share a key/value head (group x
// query tokens) are packed into 16-row tiles of mma.sync m16n8k16 (kTiles of
// them per CTA): a 128-row tcgen05 tile would be at least 7/8 padding, and the
// instruction rate is far from being the limit.
//
// Split: the 64-key tiles of all (batch entry, key/value head, row tile)
// segments form one line, cut into equal ranges, one per resident CTA (the
// lengths are device data, so every CTA computes its cut).  A segment that
// lies within one range is finished there; of the others each CTA leaves a
// partial result (O, max, sum) in the workspace, joined in a fixed order by
// attn_join_kernel: results do not depend on timing.
//
// CTA: warps 0..3 compute (16 of a tile's 64 keys each, with a softmax state
// of their own, merged at a segment's end), warp 4 is the TMA producer
// (kSplitStages tiles ahead, across segments).  K and V tiles are stored with
// the 128-byte swizzle; fp8 fragments are read with conflict-free 16-byte
// loads: the order of d inside an mma's K slices and of O's columns is free,
// so thread t of a quad takes d = 32 t .. 32 t + 31 of both.
//
// fp8: codes become fp16 exactly.  Q becomes fp16 after an exact power-of-two
// scaling per row (largest value to 2^11: what fp16 cannot hold of a row is
// below 2^-35 of its largest value), undone on the scores.  The value scale is
// folded into P relative to the running maximum of (score + log2 scale), so P
// is at most 2^4 in fp16 whatever the scales, and O needs no second set of accumulators.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "attn_sm100.cuh"
#include "kv_cache_sm100.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kSplitKeys = 64;     // keys per tile
constexpr int kSplitWarps = 4;     // computing warps, 16 keys of a tile each
constexpr int kSplitThreads = 32 * (kSplitWarps + 1);
constexpr float kSplitMoveLog2 = 4.0f;  // the reference max moves when a row's max grew by more than 2^4

struct SplitAttnParams {
  int32_t batch, q_len, heads, kv_heads, group;
  int32_t rows, row_tiles;  // q_len * group query rows per key/value head, in tiles of 16 * kTiles
  const __nv_bfloat16* q;   // [batch, q_len, heads, 128], strides in elements
  int64_t q_batch, q_seq, q_head;
  __nv_bfloat16* o;
  int64_t o_batch, o_seq, o_head;
  float* lse;               // [batch, heads, q_len] or NULL
  float scale_log2;
  // Key lengths: fp8: seq_lens (required), new_lens or NULL; bf16: kv_lens or NULL.
  const int32_t* seq_lens;
  const int32_t* new_lens;
  int32_t kv_len;           // most keys of a batch entry
  // fp8: the cache.
  int32_t page_size, num_pages;
  const int32_t* table;
  int64_t table_stride;
  const float* k_scale;
  const float* v_scale;
  // Partial results: 2 slots per CTA of 16 * kTiles rows x (128 + 2) floats, then one descriptor per CTA.
  float* part;
  int4* desc;
  uint64_t timeout_ns;
  uint32_t* status;
};

template <bool kFp8, int kTiles>
struct SplitPlan {
  // kTiles = 1: two CTAs per SM; 2: one.
  static constexpr int kStages = (kFp8 ? 4 : 2) * kTiles;
  static constexpr int kTileBytes = kSplitKeys * kKvD * (kFp8 ? 1 : 2);  // K or V of 64 keys
  static constexpr int kRows = 16 * kTiles;
  // O of a warp in shared memory: rows of four 32-column blocks, each padded
  // to 36 floats: the fragments' 16-byte stores then touch every bank once.
  static constexpr int kPitch = 144;
  static constexpr int kOffMerge = 2 * kStages * kTileBytes;
  static constexpr int kOffMl = kOffMerge + kSplitWarps * kRows * kPitch * 4;   // max and sum per warp and row
  static constexpr int kOffScale = kOffMl + kSplitWarps * kRows * 8;             // per stage: 4 x (K scale, V scale)
  static constexpr int kOffBar = kOffScale + kStages * 32;
  static constexpr int kOffScan = kOffBar + 2 * kStages * 8;  // 8 x int64 warp sums, first segment
  static constexpr int kOffAbort = kOffScan + 12 * 8;
  static constexpr int kBytes = kOffAbort + 16;
  static constexpr int kAllocBytes = kBytes + 1024;
  static constexpr size_t kPartFloats = (size_t)kRows * (kKvD + 2);
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Keys of batch entry b.
template <bool kFp8>
__device__ __forceinline__ int split_len(const SplitAttnParams& p, int b) {
  if constexpr (kFp8) return min(max(p.seq_lens[b], 0), p.kv_len);
  return attn_kv_len(p.seq_lens, b, p.kv_len);
}

// Range of CTA c of `ctas` in a line of `total` tiles.
__device__ __forceinline__ int64_t split_cut(int64_t total, int c, int ctas) { return total * c / ctas; }

template <bool kFp8, int kTiles>
__global__ void __launch_bounds__(kSplitThreads, kTiles == 1 ? 2 : 1)
    attn_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ SplitAttnParams p) {
#if B200_NO_SM100A_FEATURES
  if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, (uint32_t)kDevWrongArch);
#else
  using Plan = SplitPlan<kFp8, kTiles>;
  constexpr int kStages = Plan::kStages;
  constexpr int kRows = Plan::kRows;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_u32);
  auto sK = [&](int s) { return base + (uint32_t)(2 * s * Plan::kTileBytes); };
  auto sV = [&](int s) { return base + (uint32_t)((2 * s + 1) * Plan::kTileBytes); };
  auto full = [&](int s) { return base + (uint32_t)Plan::kOffBar + 8u * s; };
  auto empty = [&](int s) { return base + (uint32_t)Plan::kOffBar + 8u * (kStages + s); };
  float* merge = reinterpret_cast<float*>(base_ptr + Plan::kOffMerge);
  float2* ml = reinterpret_cast<float2*>(base_ptr + Plan::kOffMl);
  float2* scales = reinterpret_cast<float2*>(base_ptr + Plan::kOffScale);
  int64_t* scan = reinterpret_cast<int64_t*>(base_ptr + Plan::kOffScan);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_ptr + Plan::kOffAbort);

  const int warp = (int)threadIdx.x >> 5;
  const int lane = (int)(threadIdx.x & 31u);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), kSplitWarps);
    }
    *abort_flag = 0u;
    fence_mbar_init();
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's range of the line of tiles -----------------------------------
  const int cta = (int)blockIdx.x;
  const int segs = p.kv_heads * p.row_tiles;
  auto tiles_of = [&](int b) { return (split_len<kFp8>(p, b) + kSplitKeys - 1) / kSplitKeys; };
  const int chunk = (p.batch + kSplitThreads - 1) / kSplitThreads;
  const int b_lo = min((int)threadIdx.x * chunk, p.batch), b_hi = min(b_lo + chunk, p.batch);
  int64_t sum = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    if constexpr (kFp8) {
      const int n = p.seq_lens[b];
      const int fresh = p.new_lens != nullptr ? p.new_lens[b] : 0;
      if ((n < 0 || n > p.kv_len || fresh < 0 || fresh > p.q_len) && cta == 0) kv_bad_index(p.status);
    }
    sum += tiles_of(b);
  }
  int64_t incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w <= kSplitWarps; ++w) {
    if (w < warp) before += scan[w];
    all += scan[w];
  }
  const int64_t total = all * segs;
  // With fewer tiles than CTAs the first `total` take one each.
  const int ctas = (int)min((int64_t)gridDim.x, max(total, (int64_t)1));
  const int64_t u_begin = split_cut(total, min(cta, ctas), ctas), u_end = split_cut(total, min(cta + 1, ctas), ctas);
  {
    const int64_t lo = (before + incl - sum) * segs, hi = (before + incl) * segs;
    if (lo <= u_begin && u_begin < hi) {  // one thread, if the range is not empty
      int64_t at = lo;
      int b = b_lo;
      while (at + (int64_t)tiles_of(b) * segs <= u_begin) at += (int64_t)tiles_of(b++) * segs;
      scan[8] = at;
      scan[9] = b;
    }
  }
  __syncthreads();
  // Walk over the range: f(batch entry, keys, tiles, segment, first tile, end tile, place of the segment's first tile).
  auto walk = [&](auto&& f) {
    if (u_begin >= u_end) return;
    int64_t u = u_begin, at = scan[8];
    int b = (int)scan[9];
    while (u < u_end) {
      const int len = split_len<kFp8>(p, b);
      const int tiles = (len + kSplitKeys - 1) / kSplitKeys;
      const int64_t b_end = at + (int64_t)tiles * segs;
      while (u < u_end && u < b_end) {
        const int seg = (int)((u - at) / tiles);
        const int64_t seg_at = at + (int64_t)seg * tiles;
        const int t0 = (int)(u - seg_at);
        const int t1 = (int)min((int64_t)tiles, u_end - seg_at);
        f(b, len, tiles, seg, t0, t1, seg_at);
        u = seg_at + t1;
      }
      at = b_end;
      ++b;
    }
  };

  if (warp == kSplitWarps) {
    // ---- TMA producer ------------------------------------------------------------
    const uint64_t pol = l2_policy_evict_first();  // K and V are read once
    uint32_t it = 0;
    bool ok = true;
    walk([&](int b, int len, int, int seg, int t0, int t1, int64_t) {
      const int kv_head = seg / p.row_tiles;
      [[maybe_unused]] int page_id = 0, page_base = 0, page_next = 0;
      [[maybe_unused]] float ks = 0.0f, vs = 0.0f;
      [[maybe_unused]] const int pages = kFp8 ? (len + p.page_size - 1) / p.page_size : 0;
      // Lane i holds page page_base + i of the table, with its scales; the
      // next 32 entries are on their way.
      auto entry = [&](int i) { return i < pages ? p.table[b * p.table_stride + i] : -1; };
      auto take = [&](int id, int i) {
        page_id = id;
        const bool fine = id >= 0 && id < p.num_pages;
        if (!fine && i < pages) kv_bad_index(p.status);
        if (!fine) page_id = -1;
        const size_t at = (size_t)max(page_id, 0) * p.kv_heads + kv_head;
        ks = fine ? p.k_scale[at] : 0.0f;
        vs = fine ? p.v_scale[at] : 1.0f;
      };
      if constexpr (kFp8) {
        page_base = t0 * kSplitKeys / p.page_size;
        take(entry(page_base + lane), page_base + lane);
        page_next = entry(page_base + 32 + lane);
      }
      for (int t = t0; t < t1; ++t, ++it) {
        const int s = (int)(it % kStages);
        const bool got = ok && mbar_wait(empty(s), ((it / kStages) & 1u) ^ 1u, p.timeout_ns, abort_flag);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          return;
        }
        if constexpr (kFp8) {
          const int box = min(p.page_size, kSplitKeys);
          const int page0 = t * kSplitKeys / p.page_size;
          if (page0 >= page_base + 32) {
            page_base += 32;
            take(page_next, page_base + lane);
            page_next = entry(page_base + 32 + lane);
          }
          // Scales of the tile's four 16-key groups.
          const int g_page = (t * kSplitKeys + (lane & 3) * 16) / p.page_size - page_base;
          const float gk = __shfl_sync(0xffffffffu, ks, g_page), gv = __shfl_sync(0xffffffffu, vs, g_page);
          if (lane < 4) scales[s * 4 + lane] = make_float2(gk, gv);
          // One box per page (or the tile's part of a longer page); pages past
          // the last key are not read.
          const int boxes = kSplitKeys / box;
          const int my_key = t * kSplitKeys + lane * box;
          const int my_page = __shfl_sync(0xffffffffu, page_id, (t * kSplitKeys + (lane % boxes) * box) / p.page_size - page_base);
          const bool load = lane < boxes && my_key < len && my_page >= 0;
          const uint32_t n = (uint32_t)__popc(__ballot_sync(0xffffffffu, load));
          __syncwarp();  // the scales, before the arrival that publishes them
          if (lane == 0) mbar_arrive_expect_tx(full(s), n * 2u * (uint32_t)(box * kKvD));
          __syncwarp();
          if (load) {
            const int row = (my_page * p.kv_heads + kv_head) * p.page_size + my_key % p.page_size;
            tma_load_2d(sK(s) + (uint32_t)(lane * box * kKvD), &tmK, full(s), 0, row, pol);
            tma_load_2d(sV(s) + (uint32_t)(lane * box * kKvD), &tmV, full(s), 0, row, pol);
          }
        } else {
          if (lane == 0) mbar_arrive_expect_tx(full(s), 2u * Plan::kTileBytes);
          __syncwarp();
          if (lane < 2) {
            tma_load_4d(sK(s) + (uint32_t)(lane * Plan::kTileBytes / 2), &tmK, full(s), 64 * lane, kv_head, t * kSplitKeys, b, pol);
            tma_load_4d(sV(s) + (uint32_t)(lane * Plan::kTileBytes / 2), &tmV, full(s), 64 * lane, kv_head, t * kSplitKeys, b, pol);
          }
        }
      }
    });
    if (!ok && lane == 0) attn_raise(p, abort_flag, kDevTimeoutProducer);
    // Let the copies in flight land before the CTA can leave.
    bool drained = true;
    for (uint32_t i = it; drained && i > 0 && i + kStages > it; --i) {
      drained = mbar_wait(full((int)((i - 1) % kStages)), ((i - 1) / kStages) & 1u, p.timeout_ns, nullptr);
    }
    if (!drained && lane == 0) attn_raise(p, abort_flag, kDevTimeoutDrain);
  } else {
    // ---- four computing warps ---------------------------------------------------------
    const int g = lane >> 2, t4 = lane & 3;
    uint32_t it = 0;
    bool ok = true;
    int4 desc = make_int4(-1, 0, 0, 0);
    walk([&](int b, int len, int tiles, int seg, int t0, int t1, int64_t seg_at) {
      const int kv_head = seg / p.row_tiles, row0 = (seg % p.row_tiles) * kRows;
      // Query tokens of this batch entry: token t sees the keys below len - tokens + t + 1 (bf16: all).
      int tokens = p.q_len;
      if (kFp8 && p.new_lens != nullptr) tokens = min(max(p.new_lens[b], 0), p.q_len);
      auto limit_of = [&](int row) { return kFp8 ? len - tokens + row / p.group + 1 : len; };
      const int least = kFp8 ? len - tokens + row0 / p.group + 1 : len;  // the smallest limit of the tile's rows
      uint32_t qa[kTiles][8][4];
      float unscale[kTiles][2];  // scores to the exp2 domain
      int limit[kTiles][2];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = row0 + m * 16 + h * 8 + g;
          const bool there = row < p.rows;
          const int tok = row / p.group, head = kv_head * p.group + row % p.group;
          const __nv_bfloat16* src = p.q + b * p.q_batch + tok * p.q_seq + head * p.q_head;
          limit[m][h] = there ? limit_of(row) : 0;
          if constexpr (kFp8) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 v = there ? *reinterpret_cast<const uint4*>(src + 32 * t4 + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
              w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 f = bf16x2_to_float2(w[i]);
              top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = min(11 - ((int)(__float_as_uint(top) >> 23) - 127), 100);  // largest value into [2^11, 2^12)
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            unscale[m][h] = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 f0 = bf16x2_to_float2(w[2 * k]), f1 = bf16x2_to_float2(w[2 * k + 1]);
              qa[m][k][h] = pack_f16x2(f0.x * up, f0.y * up);
              qa[m][k][2 + h] = pack_f16x2(f1.x * up, f1.y * up);
            }
          } else {
            unscale[m][h] = p.scale_log2;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                qa[m][k][2 * i + h] = there ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 * i + 2 * t4) : 0u;
              }
            }
          }
        }
      }
      float o[kTiles][16][4];
      float mx[kTiles][2], l[kTiles][2];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        mx[m][0] = mx[m][1] = -INFINITY;
        l[m][0] = l[m][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[m][j][0] = o[m][j][1] = o[m][j][2] = o[m][j][3] = 0.0f;
      }

      for (int t = t0; t < t1; ++t, ++it) {
        const int s = (int)(it % kStages);
        const bool got = ok && mbar_wait(full(s), (it / kStages) & 1u, p.timeout_ns, abort_flag);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;  // the remaining waits return at once; barriers below are still met
          continue;
        }
        const int key0 = t * kSplitKeys + warp * 16;  // this warp's keys
        if (key0 < len) {
          float ks = 1.0f, vs = 1.0f, lv = 0.0f;
          if constexpr (kFp8) {
            const float2 sc = scales[s * 4 + warp];
            ks = sc.x;
            vs = sc.y;
            lv = fmaxf(log2f(vs), (float)kKvMinScaleExp);
          }
          // Scores of 16 keys: two 8-key fragments.
          float x[kTiles][2][4];
#pragma unroll
          for (int m = 0; m < kTiles; ++m) {
#pragma unroll
            for (int n = 0; n < 2; ++n) x[m][n][0] = x[m][n][1] = x[m][n][2] = x[m][n][3] = 0.0f;
          }
          if constexpr (kFp8) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const uint32_t row = sK(s) + (uint32_t)((warp * 16 + n * 8 + g) * kKvD);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint4 v = lds128(row + (uint32_t)(((2 * t4 + c) ^ g) << 4));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t b0 = e4m3x2_to_f16x2(w[i]), b1 = e4m3x2_hi_to_f16x2(w[i]);
#pragma unroll
                  for (int m = 0; m < kTiles; ++m) mma_f16(x[m][n], qa[m][4 * c + i], b0, b1);
                }
              }
            }
          } else {
            // Lanes 0..7, 8..15, 16..23, 24..31 address the four 8 x 8 blocks
            // (keys 0-7, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 0-7), (keys 8-15, d 8-15).
            const int key = warp * 16 + (lane & 7) + ((lane >> 4) << 3);
            const uint32_t row = sK(s) + (uint32_t)(key * 128);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t cell = (uint32_t)(2 * (k & 3) + ((lane >> 3) & 1));
              uint32_t r[4];
              ldmatrix_x4(r, row + (uint32_t)((k >> 2) * (Plan::kTileBytes / 2)) + ((cell ^ (uint32_t)(key & 7)) << 4));
#pragma unroll
              for (int m = 0; m < kTiles; ++m) {
                mma_bf16(x[m][0], qa[m][k], r[0], r[1]);
                mma_bf16(x[m][1], qa[m][k], r[2], r[3]);
              }
            }
          }
          const bool masked = key0 + 16 > least;
          bool move = false;
          float top[kTiles][2];
#pragma unroll
          for (int m = 0; m < kTiles; ++m) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f = unscale[m][h] * ks;
              float mm = -INFINITY;
#pragma unroll
              for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  float& v = x[m][n][2 * h + c];
                  v *= f;
                  if (masked && key0 + 8 * n + 2 * t4 + c >= limit[m][h]) v = -INFINITY;
                  mm = fmaxf(mm, v);
                }
              }
              mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 1));
              mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 2)) + lv;
              top[m][h] = mm;
              move = move || mm > mx[m][h] + kSplitMoveLog2 || (mx[m][h] == -INFINITY && mm != -INFINITY);
            }
          }
          if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
              float f[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float next = fmaxf(mx[m][h], top[m][h]);
                f[h] = next == mx[m][h] ? 1.0f : fast_exp2(mx[m][h] - next);  // first keys: 2^-inf = 0
                mx[m][h] = next;
                l[m][h] *= f[h];
              }
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                o[m][j][0] *= f[0];
                o[m][j][1] *= f[0];
                o[m][j][2] *= f[1];
                o[m][j][3] *= f[1];
              }
            }
          }
          uint32_t pa[kTiles][4];
#pragma unroll
          for (int m = 0; m < kTiles; ++m) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float ref = mx[m][h] == -INFINITY ? 0.0f : mx[m][h];
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float e0 = fast_exp2(x[m][n][2 * h] - ref), e1 = fast_exp2(x[m][n][2 * h + 1] - ref);
                l[m][h] += e0 + e1;
                pa[m][2 * n + h] = kFp8 ? pack_f16x2(e0 * vs, e1 * vs) : pack_bf16x2(e0, e1);
              }
            }
          }
          // O += P V.  V of keys past the last one may hold anything: zeros
          // take its place (0 x NaN would reach O).
          const bool cut = key0 + 16 > len;
          if constexpr (kFp8) {
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = 2 * t4 + (i & 1) + (i >> 1) * 8;
              uint4 v = lds128(sV(s) + (uint32_t)((warp * 16 + key) * kKvD) + (uint32_t)((g ^ (key & 7)) << 4));
              if (cut && key0 + key >= len) v = make_uint4(0u, 0u, 0u, 0u);
              w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                // Bytes 2h, 2h + 1 of a key pair, interleaved: (k0, k1) of one d each.
                const uint32_t u0 = __byte_perm(w[0][q], w[1][q], h ? 0x7362 : 0x5140);
                const uint32_t u1 = __byte_perm(w[2][q], w[3][q], h ? 0x7362 : 0x5140);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t b0 = i ? e4m3x2_hi_to_f16x2(u0) : e4m3x2_to_f16x2(u0);
                  const uint32_t b1 = i ? e4m3x2_hi_to_f16x2(u1) : e4m3x2_to_f16x2(u1);
#pragma unroll
                  for (int m = 0; m < kTiles; ++m) mma_f16(o[m][4 * q + 2 * h + i], pa[m], b0, b1);
                }
              }
            }
          } else {
            if (cut) {
              // Zero the rows past the last key in this warp's part of the tile.
              for (int c = lane; c < 16 * 16; c += 32) {
                const int key = c >> 4;
                if (key0 + key >= len) {
                  const uint32_t dst = sV(s) + (uint32_t)(((c >> 3) & 1) * (Plan::kTileBytes / 2) + (warp * 16 + key) * 128 + (c & 7) * 16);
                  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0u) : "memory");
                }
              }
              __syncwarp();
            }
            // Blocks (keys 0-7, d 0-7), (keys 8-15, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 8-15).
            const int key = warp * 16 + (lane & 15);
            const uint32_t row = sV(s) + (uint32_t)(key * 128);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t cell = (uint32_t)(2 * (j & 3) + (lane >> 4));
              uint32_t r[4];
              ldmatrix_x4_trans(r, row + (uint32_t)((j >> 2) * (Plan::kTileBytes / 2)) + ((cell ^ (uint32_t)(key & 7)) << 4));
#pragma unroll
              for (int m = 0; m < kTiles; ++m) {
                mma_bf16(o[m][2 * j], pa[m], r[0], r[1]);
                mma_bf16(o[m][2 * j + 1], pa[m], r[2], r[3]);
              }
            }
            if (cut) fence_proxy_async_smem();  // the zeros, before TMA writes the stage again
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      }

      // ---- merge the four warps' states, hand the rows out -------------------------
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 1);
          l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 2);
          if (t4 == 0) ml[warp * kRows + m * 16 + h * 8 + g] = make_float2(mx[m][h], l[m][h]);
        }
      }
      named_bar_sync(1, 32 * kSplitWarps);
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = m * 16 + h * 8 + g;
          float big = -INFINITY;
#pragma unroll
          for (int w = 0; w < kSplitWarps; ++w) big = fmaxf(big, ml[w * kRows + r].x);
          const float f = mx[m][h] == -INFINITY ? 0.0f : fast_exp2(mx[m][h] - big);
          float* dst = merge + (size_t)(warp * kRows + r) * Plan::kPitch;
          if constexpr (kFp8) {
            // This thread holds d = 32 t4 + j (c = 0) and 32 t4 + 16 + j (c = 1).
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                *reinterpret_cast<float4*>(dst + 36 * t4 + 16 * c + j) =
                    make_float4(o[m][j][2 * h + c] * f, o[m][j + 1][2 * h + c] * f, o[m][j + 2][2 * h + c] * f,
                                o[m][j + 3][2 * h + c] * f);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int d = 8 * j + 2 * t4;
              *reinterpret_cast<float2*>(dst + d + 4 * (d >> 5)) = make_float2(o[m][j][2 * h] * f, o[m][j][2 * h + 1] * f);
            }
          }
        }
      }
      named_bar_sync(1, 32 * kSplitWarps);
      const bool whole = t0 == 0 && t1 == tiles;
      const int rows_here = min(kRows, p.rows - row0);
      float* part = p.part + (size_t)(2 * cta + (t0 == 0 ? 1 : 0)) * Plan::kPartFloats;
      for (int r = warp; r < rows_here; r += kSplitWarps) {
        float big = -INFINITY;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) big = fmaxf(big, ml[w * kRows + r].x);
        float sum_l = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) {
          const float2 s2 = ml[w * kRows + r];
          sum_l += s2.x == -INFINITY ? 0.0f : s2.y * fast_exp2(s2.x - big);
          const float4 v = *reinterpret_cast<const float4*>(merge + (size_t)(w * kRows + r) * Plan::kPitch + 4 * lane + 4 * (lane >> 3));
          acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
        const int row = row0 + r, tok = row / p.group, head = kv_head * p.group + row % p.group;
        if (!ok) continue;
        if (whole) {
          const bool none = sum_l == 0.0f || tok >= tokens;  // nothing seen, or a padding query
          const float inv = none ? 0.0f : 1.0f / sum_l;
          uint2 w2 = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
          if (none) w2 = make_uint2(0u, 0u);
          *reinterpret_cast<uint2*>(p.o + b * p.o_batch + tok * p.o_seq + head * p.o_head + 4 * lane) = w2;
          if (p.lse != nullptr && lane == 0) {
            p.lse[((size_t)b * p.heads + head) * p.q_len + tok] = none ? -INFINITY : (big + log2f(sum_l)) * 0.6931471805599453f;
          }
        } else {
          *reinterpret_cast<float4*>(part + (size_t)r * kKvD + 4 * lane) = acc;
          if (lane == 0) *reinterpret_cast<float2*>(part + (size_t)kRows * kKvD + 2 * r) = make_float2(big, sum_l);
        }
      }
      if (t0 == 0 && !whole && ok) {
        // The segment begins here and ends in a later CTA's range: the one
        // that holds its last tile.
        const int64_t last = seg_at + tiles - 1;
        int c = (int)((last * ctas) / total);
        while (split_cut(total, c + 1, ctas) <= last) ++c;
        while (split_cut(total, c, ctas) > last) --c;
        desc = make_int4(c, b, seg, tokens);
      }
      named_bar_sync(1, 32 * kSplitWarps);  // merge buffers free again
    });
    if (!ok && lane == 0) attn_raise(p, abort_flag, kDevTimeoutEpilogue);
    if (threadIdx.x == 0 && p.desc != nullptr) p.desc[cta] = desc;
    // Batch entries without keys: zeros.
    for (int b = cta; b < p.batch; b += (int)gridDim.x) {
      if (split_len<kFp8>(p, b) > 0) continue;
      for (int r = warp; r < p.q_len * p.heads; r += kSplitWarps) {
        const int tok = r / p.heads, head = r % p.heads;
        *reinterpret_cast<uint2*>(p.o + b * p.o_batch + tok * p.o_seq + head * p.o_head + 4 * lane) = make_uint2(0u, 0u);
        if (p.lse != nullptr && lane == 0) p.lse[((size_t)b * p.heads + head) * p.q_len + tok] = -INFINITY;
      }
    }
  }
  // No CTA may leave with a barrier of its shared memory in use.
  __syncthreads();
#endif  // B200_NO_SM100A_FEATURES
}

// Joins the partial results of the segments that were cut: block (c, y) the
// rows 4 y .. 4 y + 3 of the segment that begins in CTA c and ends in CTA
// desc[c].x, a warp per row, 4 columns per lane, partials in order.
template <int kTiles>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ SplitAttnParams p) {
  constexpr int kRows = 16 * kTiles;
  constexpr size_t kPartFloats = SplitPlan<true, kTiles>::kPartFloats;
  pdl_launch_dependents();
  pdl_wait();
  const int cta = (int)blockIdx.x, lane = (int)(threadIdx.x & 31u);
  const int r = 4 * (int)blockIdx.y + ((int)threadIdx.x >> 5);
  const int4 d = p.desc[cta];
  if (d.x < 0) return;
  const int kv_head = d.z / p.row_tiles, row = (d.z % p.row_tiles) * kRows + r;
  if (r >= kRows || row >= p.rows) return;
  // The first partial is in its CTA's second slot, the others in their first.
  auto slot = [&](int c) { return p.part + (size_t)(2 * c + (c == cta ? 1 : 0)) * kPartFloats; };
  float big = -INFINITY;
  for (int c = cta + lane; c <= d.x; c += 32) big = fmaxf(big, slot(c)[(size_t)kRows * kKvD + 2 * r]);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, k));
  float sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int c = cta; c <= d.x; ++c) {
    const float* s = slot(c);
    const float2 ml = *reinterpret_cast<const float2*>(s + (size_t)kRows * kKvD + 2 * r);
    const float4 v = *reinterpret_cast<const float4*>(s + (size_t)r * kKvD + 4 * lane);
    const float f = ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - big);
    sum += ml.y * f;
    acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
  }
  const int tok = row / p.group, head = kv_head * p.group + row % p.group;
  const bool none = sum == 0.0f || tok >= d.w;
  const float inv = none ? 0.0f : 1.0f / sum;
  uint2 w2 = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (none) w2 = make_uint2(0u, 0u);
  *reinterpret_cast<uint2*>(p.o + d.y * p.o_batch + tok * p.o_seq + head * p.o_head + 4 * lane) = w2;
  if (p.lse != nullptr && lane == 0) {
    p.lse[((size_t)d.y * p.heads + head) * p.q_len + tok] = none ? -INFINITY : (big + log2f(sum)) * 0.6931471805599453f;
  }
}

}  // namespace b200
