// Attention of few query rows over long stored keys and values, for sm_100a:
// the serving step of a decoder.  Two sources of K and V:
//   kFp8 = true   the paged e4m3 cache (b200_cache_attn): queries are the
//                 last tokens of their sequence and see the places up to theirs;
//   kFp8 = false  bf16 states of another length (b200_cross_attn_bf16 with few
//                 queries): every query sees all keys of its batch entry.
//
// The work is bound by reading K and V once (256 or 512 bytes per key and
// key/value head), so the query rows that share a key/value head (group x
// query tokens) are packed into 16-row tiles of mma.sync m16n8k16 (kTiles of
// them per warp): a 128-row tcgen05 tile would be at least 7/8 padding, and the
// instruction rate is far from being the limit.
//
// Split: every warp is a worker of its own.  The units (32 keys) of all
// (batch entry, key/value head, row tile) segments form one line, cut into
// equal ranges, one per resident warp (the lengths are device data, so every
// warp computes its cut).  A segment that lies within one range is finished
// there; of the others each warp leaves a partial result (O, max, sum) in the
// workspace, joined in a fixed order by attn_join_kernel: results do not
// depend on timing.  A warp loads its units itself by TMA, one or two ahead
// and across segments, so there is no barrier between warps and the end of a
// segment stalls one warp of the SM's twelve.  (Four warps sharing each
// 64-key tile, a producer warp, and a merge through shared memory per segment:
// 68 us where this takes 43 on 24 ragged sequences of up to 2999 places, 16
// heads; 129 against 105 on 64 sequences of up to 8192, 8 key/value heads.)
//
// Small problems take a form of their own (kCluster): a cluster of 1 to 8 CTAs
// per segment, its units divided evenly over the cluster's warps, whose results
// meet in distributed shared memory.  No line to compute, no workspace, no second
// kernel: 8.1 us against 12.8 for one request of 1000 places, 8 key/value heads.
//
// K and V units are stored with the 128-byte swizzle; fp8 fragments are read
// with conflict-free 16-byte loads: the order of d inside an mma's K slices and
// of O's columns is free, so thread t of a quad takes d = 32 t .. 32 t + 31 of both.
//
// fp8: codes become fp16 exactly.  Q becomes fp16 after an exact power-of-two
// scaling per row (largest value to 2^11: what fp16 cannot hold of a row is
// below 2^-35 of its largest value), undone on the scores.  (Scores by the e4m3
// mma on the codes themselves, Q in two e4m3 parts: exact enough, but 145 us
// against 105 on 64 sequences of up to 8192, as that mma converts its operands
// inside on this chip.)  The value scale is
// folded into P relative to the running maximum of (score + log2 scale), so
// that O needs no second set of accumulators: P in fp16 is at most 2^14
// whatever the scales, and what it cannot hold is below 2^-34 of the row's largest.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "attn_sm100.cuh"
#include "kv_cache_sm100.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kSplitWarps = 4;  // workers per CTA
constexpr int kSplitThreads = 32 * kSplitWarps;
// Beginning a segment (its queries, block table and scales) and handing its
// rows out costs a warp about as much as two units: it counts as that in the
// line, or workers with many short segments finish last (58 us against a
// median of 37 on 24 sequences of 5 to 2999 places).
constexpr int kSplitSegUnits = 2;
constexpr float kSplitMoveLog2 = 4.0f;  // the reference max moves when a row's max grew by more than 2^4
constexpr float kSplitLiftLog2 = 10.0f;  // fp8: P and the sum are held 2^10 times their value

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
  // Partial results: 2 slots per worker of 16 * kTiles rows x (128 + 2) floats, then one descriptor per worker.
  float* part;
  int4* desc;
  int32_t workers;
  uint64_t timeout_ns;
  uint32_t* status;
};

template <bool kFp8, int kTiles>
struct SplitPlan {
  // 16 KiB of K and V per warp.  fp8: two units, each with a barrier.  bf16: one
  // unit, K and V with a barrier each: K of the next unit loads while P V runs,
  // V while its scores do (two units of 16 keys, with twice the boxes and waits
  // per byte: 64 us against 58 on 32 sources of 200 to 2000 keys, 16 heads).
  static constexpr int kKeys = 32;  // keys per unit
  static constexpr int kHalfBytes = kKeys * kKvD * (kFp8 ? 1 : 2);
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kStages = kFp8 ? 2 : 1;
  static constexpr int kRows = 16 * kTiles;
  static constexpr int kCtasPerSm = kTiles == 1 ? 3 : 2;
  // Per warp: stages, then scales per stage (2 x (K scale, V scale, log2 of
  // it)), segment queue, barriers.
  static constexpr int kOffScale = kSplitWarps * kStages * kStageBytes;
  static constexpr int kQueue = kStages + 2;  // segments between the loads and the products
  static constexpr int kOffQueue = kOffScale + kSplitWarps * kStages * 32;
  static constexpr int kOffPages = kOffQueue + kSplitWarps * kQueue * 32;  // 32 pages: scales and number
  static constexpr int kOffCursor = kOffPages + kSplitWarps * 32 * 16;
  static constexpr int kOffMl = kOffCursor + kSplitWarps * 64;  // clusters: maximum and sum of every row
  static constexpr int kOffBar = kOffMl + kSplitWarps * kRows * 8;
  static constexpr int kOffAbort = kOffBar + kSplitWarps * 16;
  static constexpr int kBytes = kOffAbort + 16;
  static constexpr int kAllocBytes = kBytes + 1024;
  static constexpr size_t kPartFloats = (size_t)kRows * (kKvD + 2);
  static_assert(kCtasPerSm * (kAllocBytes + 1024) <= 233472, "split attention shared memory plan exceeds 228 KiB");
};

// What a warp needs to know of a segment's part in its range.
struct SplitSegment {
  int32_t b, len, units, seg, t0, t1;  // entry, keys, units of the segment, segment of the entry, units [t0, t1)
  int32_t last;                        // cut off at t1 after beginning here: the worker that holds its end; else -1
  int32_t pad;
};
static_assert(sizeof(SplitSegment) == 32, "read as two 16-byte words");

// A warp's place in its range, in shared memory: it is needed once per segment,
// and the registers are the loop's.
struct SplitCursor {
  int64_t u, u_end;     // places still to be loaded
  int64_t at;           // place of entry b's first segment
  int64_t quot, rest;   // of the line (SplitLine)
  int32_t workers, b;
  int32_t pad[4];
};
static_assert(sizeof(SplitCursor) == 64, "one per warp");

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// Keys of batch entry b.
template <bool kFp8>
__device__ __forceinline__ int split_len(const SplitAttnParams& p, int b) {
  if constexpr (kFp8) return min(max(p.seq_lens[b], 0), p.kv_len);
  return attn_kv_len(p.seq_lens, b, p.kv_len);
}

// 64-bit quotient, on the 32-bit divider where both fit (always, in practice).
__device__ __forceinline__ int64_t split_div(int64_t a, int64_t b) {
  if (((uint64_t)a | (uint64_t)b) >> 32 == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
  return a / b;
}

// The line of places cut into equal ranges: worker c has [begin(c), begin(c + 1)).
struct SplitLine {
  int64_t quot, rest;
  int workers;
  __device__ __forceinline__ SplitLine(int64_t quot_, int64_t rest_, int workers_) : quot(quot_), rest(rest_), workers(workers_) {}
  __device__ __forceinline__ SplitLine(int64_t total, int most) {
    // With fewer places than workers the first `total` take one each.
    workers = (int)min((int64_t)most, max(total, (int64_t)1));
    quot = split_div(total, workers);
    rest = total - quot * workers;
  }
  __device__ __forceinline__ int64_t begin(int c) const { return quot * min(c, workers) + min((int64_t)min(c, workers), rest); }
  // The worker that has place u.
  __device__ __forceinline__ int of(int64_t u) const {
    const int64_t wide = rest * (quot + 1);
    return (int)(u < wide ? split_div(u, quot + 1) : rest + split_div(u - wide, quot));
  }
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
// Clusters: a warp's O in its (then idle) stages, rows of 32 cells of four
// columns, permuted within groups of eight so that the fragments' stores and the
// rows' loads touch every bank once.
__device__ __forceinline__ uint32_t split_cell(int row, int cell) {
  return (uint32_t)(row * 512 + ((cell ^ (((row & 1) << 2) | (cell >> 3))) << 4));
}

template <bool kFp8, int kTiles, bool kCluster>
__global__ void __launch_bounds__(kSplitThreads, SplitPlan<kFp8, kTiles>::kCtasPerSm)
    attn_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ SplitAttnParams p) {
#if B200_NO_SM100A_FEATURES
  if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, (uint32_t)kDevWrongArch);
#else
  using Plan = SplitPlan<kFp8, kTiles>;
  constexpr int kKeys = Plan::kKeys;
  constexpr int kStages = Plan::kStages;
  constexpr int kRows = Plan::kRows;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_u32);
  const int warp = (int)threadIdx.x >> 5;
  const int lane = (int)(threadIdx.x & 31u);
  auto sK = [&](int s) { return base + (uint32_t)((warp * kStages + s) * Plan::kStageBytes); };
  auto sV = [&](int s) { return sK(s) + (uint32_t)Plan::kHalfBytes; };
  // fp8: unit in stage s has landed; bf16: K (0) or V (1) has.
  auto full = [&](int s) { return base + (uint32_t)Plan::kOffBar + 8u * (warp * 2 + s); };
  float4* scales = reinterpret_cast<float4*>(base_ptr + Plan::kOffScale) + warp * kStages * 2;
  SplitSegment* queue = reinterpret_cast<SplitSegment*>(base_ptr + Plan::kOffQueue) + warp * Plan::kQueue;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_ptr + Plan::kOffAbort);

  if (lane == 0) {
    for (int s = 0; s < 2; ++s) mbar_init(full(s), 1);
    if (warp == 0) *abort_flag = 0u;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();

  // ---- this worker's range of the line ------------------------------------------
  const int worker = (int)blockIdx.x * kSplitWarps + warp;
  const int segs = p.kv_heads * p.row_tiles;
  auto units_of = [&](int len) { return (len + kKeys - 1) / kKeys; };
  // Places of one segment of entry e: its units, and kSplitSegUnits in front of them.
  auto places_of = [&](int e) {
    const int len = split_len<kFp8>(p, e);
    return len > 0 ? units_of(len) + kSplitSegUnits : 0;
  };
  auto scan32 = [&](int64_t v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    return v;
  };
  SplitCursor* cursor = reinterpret_cast<SplitCursor*>(base_ptr + Plan::kOffCursor) + warp;
  [[maybe_unused]] const int cluster = kCluster ? (int)cluster_size() : 1;
  [[maybe_unused]] const int workers = kSplitWarps * cluster;  // of a cluster's segment
  [[maybe_unused]] const int self = kCluster ? (int)cluster_ctarank() * kSplitWarps + warp : 0;
  [[maybe_unused]] float2* ml = reinterpret_cast<float2*>(base_ptr + Plan::kOffMl) + warp * kRows;
  [[maybe_unused]] SplitSegment only{};  // the cluster's segment, and this warp's part of it
  if constexpr (kCluster) {
    const int id = (int)blockIdx.x / cluster;
    only.b = id / segs;
    only.seg = id % segs;
    only.len = split_len<kFp8>(p, only.b);
    only.units = units_of(only.len);
    only.t0 = (int)((int64_t)only.units * self / workers);
    only.t1 = (int)((int64_t)only.units * (self + 1) / workers);
    only.last = -1;
    if (lane < kRows) ml[lane] = make_float2(-INFINITY, 0.0f);
    __syncwarp();
  } else {
    const int chunk = (p.batch + 31) / 32;  // entries per lane
    int64_t sum = 0;
#pragma unroll 4
    for (int i = 0; i < chunk; ++i) {
      const int e = lane * chunk + i;
      if (e < p.batch) sum += places_of(e);
    }
    const int64_t before = scan32(sum) - sum;
    const SplitLine line(__shfl_sync(0xffffffffu, before + sum, 31) * segs, (int)gridDim.x * kSplitWarps);
    const int64_t u_end = line.begin(worker + 1);
    // The load cursor: places [u, u_end) are still to be loaded; `at` is the place of entry b's first segment.
    int64_t u = line.begin(worker), at = 0;
    int b = 0;
    if (u < u_end) {
      // The last chunk that begins at or before u holds it; then the entry in
      // the chunk, 32 at a time.
      const int lane_of = 31 - __clz(__ballot_sync(0xffffffffu, before * segs <= u));
      at = __shfl_sync(0xffffffffu, before, lane_of) * segs;
      b = lane_of * chunk;
      while (b < p.batch) {
        const int64_t mine = b + lane < p.batch ? (int64_t)places_of(b + lane) * segs : 0;
        const int64_t ends = at + scan32(mine);
        const uint32_t past = __ballot_sync(0xffffffffu, ends > u);
        if (past != 0) {
          const int k = __ffs(past) - 1;
          at = __shfl_sync(0xffffffffu, ends - mine, k);
          b += k;
          break;
        }
        at = __shfl_sync(0xffffffffu, ends, 31);
        b += 32;
      }
    }
    if (lane == 0) *cursor = SplitCursor{u, u_end, at, line.quot, line.rest, line.workers, b, {}};
    __syncwarp();
  }
  if constexpr (kFp8) {
    // Lengths out of range are clamped above; the first warp reports them.
    if (blockIdx.x == 0 && warp == 0) {
      for (int e = lane; e < p.batch; e += 32) {
        const int n = p.seq_lens[e], fresh = p.new_lens != nullptr ? p.new_lens[e] : 0;
        if (n < 0 || n > p.kv_len || fresh < 0 || fresh > p.q_len) kv_bad_index(p.status);
      }
    }
  }

  // ---- loads ----------------------------------------------------------------------
  const uint64_t pol = l2_policy_evict_first();  // K and V are read once
  uint32_t loaded = 0;    // units loaded
  uint32_t segments = 0;  // segments begun; the last one is being loaded
  int ld_t = 0, ld_t1 = 0;  // its next unit and its last one's successor
  // fp8: the next 32 pages of its sequence from page_base on: scales and
  // number (-1: none, or out of range); the 32 after them are on their way.
  [[maybe_unused]] float4* pages = reinterpret_cast<float4*>(base_ptr + Plan::kOffPages) + warp * 32;
  [[maybe_unused]] int page_base = 0, page_next = 0;
  auto entry = [&](const SplitSegment& ld, int i) {
    return (int64_t)i * p.page_size < ld.len ? p.table[ld.b * p.table_stride + i] : -1;
  };
  auto take = [&](const SplitSegment& ld) {
    const int i = page_base + lane, id = page_next;
    const bool fine = id >= 0 && id < p.num_pages;
    if (!fine && (int64_t)i * p.page_size < ld.len) kv_bad_index(p.status);
    const size_t where = (size_t)(fine ? id : 0) * p.kv_heads + ld.seg / p.row_tiles;
    page_next = entry(ld, i + 32);
    const float k = fine ? p.k_scale[where] : 0.0f, v = fine ? p.v_scale[where] : 1.0f;
    pages[lane] = make_float4(k, v, fmaxf(__log2f(v), (float)kKvMinScaleExp) - kSplitLiftLog2, __int_as_float(fine ? id : -1));
    __syncwarp();
  };
  // The next segment of the range with units in it goes to the queue; false at the range's end.
  auto next_segment = [&]() {
    if constexpr (kCluster) {
      if (segments > 0 || only.t1 == only.t0) return false;
      if (lane == 0) queue[0] = only;
      __syncwarp();
      return true;
    }
    SplitCursor c = *cursor;
    const SplitLine line(c.quot, c.rest, c.workers);
    SplitSegment ld{};
    bool found = false;
    while (!found && c.u < c.u_end) {
      // (The entry exists, and c.b stays below it: the bounds hold even if
      // someone changes the lengths under way.)
      int places = c.b < p.batch ? places_of(c.b) : 0;
      while (c.b < p.batch && c.u >= c.at + (int64_t)places * segs) {
        c.at += (int64_t)places * segs;
        places = ++c.b < p.batch ? places_of(c.b) : 0;
      }
      if (c.b >= p.batch || places == 0) {
        c.u = c.u_end;
        break;
      }
      ld.b = c.b;
      ld.len = split_len<kFp8>(p, c.b);
      ld.units = places - kSplitSegUnits;
      ld.seg = (int)split_div(c.u - c.at, places);
      const int64_t seg_at = c.at + (int64_t)ld.seg * places + kSplitSegUnits;  // place of its first unit
      ld.t0 = (int)max(c.u - seg_at, (int64_t)0);
      ld.t1 = (int)min((int64_t)ld.units, c.u_end - seg_at);
      // Begun here and continued by others: who has its last unit.
      ld.last = ld.t0 == 0 && ld.t1 < ld.units ? line.of(seg_at + ld.units - 1) : -1;
      c.u = min(seg_at + ld.units, c.u_end);
      found = ld.t1 > ld.t0;  // (else the range ends in the places before its first unit)
    }
    __syncwarp();
    if (lane == 0) {
      cursor->u = c.u;
      cursor->at = c.at;
      cursor->b = c.b;
      queue[segments % Plan::kQueue] = ld;
    }
    __syncwarp();
    return found;
  };
  auto load_next = [&]() {
    if (ld_t == ld_t1) {
      if (!next_segment()) return;
      const SplitSegment ld = queue[segments % Plan::kQueue];
      ++segments;
      ld_t = ld.t0;
      ld_t1 = ld.t1;
      if constexpr (kFp8) {
        page_base = ld_t * kKeys / p.page_size;
        page_next = entry(ld, page_base + lane);
      }
      // The segment's queries, on their way while its first units load: a lane
      // per row, two lines of 128 bytes.
      const int row = (ld.seg % p.row_tiles) * kRows + lane;
      if (lane < kRows && row < p.rows) {
        const __nv_bfloat16* src = p.q + ld.b * p.q_batch + row / p.group * p.q_seq +
                                   ((ld.seg / p.row_tiles) * p.group + row % p.group) * p.q_head;
        prefetch_l1(src);
        prefetch_l1(src + 64);
      }
      if constexpr (kFp8) take(ld);
    }
    const SplitSegment& ld = queue[(segments - 1) % Plan::kQueue];
    [[maybe_unused]] const int s = (int)(loaded % kStages);
    const int key0 = ld_t * kKeys;
    const int kv_head = ld.seg / p.row_tiles;
    if constexpr (kFp8) {
      if (key0 / p.page_size >= page_base + 32) {
        page_base += 32;
        take(ld);
      }
      // One box per page, or the unit's part of a longer page; a page past the
      // last key is not read.
      const int box = min(p.page_size, kKeys);
      const int half = key0 + (lane & 1) * 16;  // lanes 0, 1: the unit's 16-key halves
      const float4 page = pages[half / p.page_size - page_base];
      const int id = __float_as_int(page.w);
      const bool load = lane < kKeys / box && half < ld.len && id >= 0;
      const uint32_t n = (uint32_t)__popc(__ballot_sync(0xffffffffu, load));
      if (lane < 2) scales[s * 2 + lane] = page;
      if (lane == 0) mbar_arrive_expect_tx(full(s), n * 2u * (uint32_t)(box * kKvD));
      __syncwarp();
      if (load) {
        const int row = (id * p.kv_heads + kv_head) * p.page_size + half % p.page_size;
        tma_load_2d(sK(s) + (uint32_t)(lane * box * kKvD), &tmK, full(s), 0, row, pol);
        tma_load_2d(sV(s) + (uint32_t)(lane * box * kKvD), &tmV, full(s), 0, row, pol);
      }
    } else {
      if (lane == 0) mbar_arrive_expect_tx(full(0), (uint32_t)Plan::kHalfBytes);
      __syncwarp();
      if (lane < 2) {
        tma_load_4d(sK(0) + (uint32_t)(lane * Plan::kHalfBytes / 2), &tmK, full(0), 64 * lane, kv_head, key0, ld.b, pol);
      }
    }
    ++ld_t;
    ++loaded;
    __syncwarp();  // the scales, before other lanes read them
  };
  // bf16: V of the unit that load_next loaded K of, if it is not loaded yet.
  [[maybe_unused]] uint32_t v_loaded = 0;
  auto load_v = [&]() {
    if (v_loaded == loaded) return;
    const SplitSegment& ld = queue[(segments - 1) % Plan::kQueue];
    if (lane == 0) mbar_arrive_expect_tx(full(1), (uint32_t)Plan::kHalfBytes);
    __syncwarp();
    if (lane < 2) {
      tma_load_4d(sV(0) + (uint32_t)(lane * Plan::kHalfBytes / 2), &tmV, full(1), 64 * lane, ld.seg / p.row_tiles,
                  (ld_t - 1) * kKeys, ld.b, pol);
    }
    ++v_loaded;
  };
#pragma unroll 1
  for (int s = 0; s < kStages; ++s) load_next();
  if constexpr (!kFp8) load_v();

  // ---- products and softmax -----------------------------------------------------------
  const int g = lane >> 2, t4 = lane & 3;
  uint32_t used = 0;
  bool ok = true;
  int4 desc = make_int4(-1, 0, 0, 0);
  for (uint32_t sg = 0; ok && sg < segments; ++sg) {
    const SplitSegment cur = queue[sg % Plan::kQueue];
    const int len = cur.len;
    const int kv_head = cur.seg / p.row_tiles, row0 = (cur.seg % p.row_tiles) * kRows;
    // Query tokens of this entry: token t sees the keys below len - tokens + t + 1 (bf16: all).
    int tokens = p.q_len;
    if (kFp8 && p.new_lens != nullptr) tokens = min(max(p.new_lens[cur.b], 0), p.q_len);
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
        const __nv_bfloat16* src = p.q + cur.b * p.q_batch + tok * p.q_seq + head * p.q_head;
        limit[m][h] = !there ? 0 : kFp8 ? len - tokens + tok + 1 : len;
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

    for (int t = cur.t0; t < cur.t1; ++t, ++used) {
      const int s = (int)(used % kStages);
      ok = __all_sync(0xffffffffu, mbar_wait(full(s), (used / kStages) & 1u, p.timeout_ns, abort_flag));
      if (!ok) break;
      const int key0 = t * kKeys;
      constexpr int kN = kKeys / 8;  // 8-key fragments of a unit
      float x[kTiles][kN][4];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
#pragma unroll
        for (int n = 0; n < kN; ++n) x[m][n][0] = x[m][n][1] = x[m][n][2] = x[m][n][3] = 0.0f;
      }
      if constexpr (kFp8) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint4 kw[kN];
#pragma unroll
          for (int n = 0; n < kN; ++n) kw[n] = lds128(sK(s) + (uint32_t)((n * 8 + g) * kKvD + (((2 * t4 + c) ^ g) << 4)));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              const uint32_t w = i == 0 ? kw[n].x : i == 1 ? kw[n].y : i == 2 ? kw[n].z : kw[n].w;
              const uint32_t b0 = e4m3x2_to_f16x2(w), b1 = e4m3x2_hi_to_f16x2(w);
#pragma unroll
              for (int m = 0; m < kTiles; ++m) mma_f16(x[m][n], qa[m][4 * c + i], b0, b1);
            }
          }
        }
      } else {
        // Lanes 0..7, 8..15, 16..23, 24..31 address the four 8 x 8 blocks
        // (keys 0-7, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 0-7), (keys 8-15, d 8-15).
        const int key = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t cell = (uint32_t)(2 * (k & 3) + ((lane >> 3) & 1));
#pragma unroll
          for (int f = 0; f < kKeys / 16; ++f) {
            uint32_t r[4];
            ldmatrix_x4(r, sK(0) + (uint32_t)((k >> 2) * (Plan::kHalfBytes / 2) + (16 * f + key) * 128) +
                               ((cell ^ (uint32_t)(key & 7)) << 4));
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
              mma_bf16(x[m][2 * f], qa[m][k], r[0], r[1]);
              mma_bf16(x[m][2 * f + 1], qa[m][k], r[2], r[3]);
            }
          }
        }
        __syncwarp();  // K is read: load the next unit's
        load_next();
      }
      // Scales of the unit's 16-key halves.
      constexpr int kHalves = kKeys / 16;
      float k_s[kHalves], v_s[kHalves], v_l[kHalves];
#pragma unroll
      for (int f = 0; f < kHalves; ++f) {
        k_s[f] = v_s[f] = 1.0f;
        v_l[f] = 0.0f;
        if constexpr (kFp8) {
          const float4 sc = scales[s * 2 + f];
          k_s[f] = sc.x, v_s[f] = sc.y, v_l[f] = sc.z;
        }
      }
      const bool masked = key0 + kKeys > least;
      bool move = false;
      float top[kTiles][2];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mm = -INFINITY;
#pragma unroll
          for (int f = 0; f < kHalves; ++f) {
            const float by = unscale[m][h] * k_s[f];
            float part = -INFINITY;
#pragma unroll
            for (int n = 2 * f; n < 2 * f + 2; ++n) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float& v = x[m][n][2 * h + c];
                v *= by;
                if (masked && key0 + 8 * n + 2 * t4 + c >= limit[m][h]) v = -INFINITY;
                part = fmaxf(part, v);
              }
            }
            mm = fmaxf(mm, part + v_l[f]);
          }
          mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 1));
          mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 2));
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
            // In two steps: with value scales 2^200 apart the sum (not lifted
            // by them) must not vanish where the factor alone would.
            const float root = next == mx[m][h] ? 1.0f : fast_exp2(0.5f * (mx[m][h] - next));  // first keys: 2^-inf = 0
            f[h] = root * root;
            mx[m][h] = next;
            l[m][h] = l[m][h] * root * root;
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
      uint32_t pa[kTiles][kHalves][4];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ref = mx[m][h] == -INFINITY ? 0.0f : mx[m][h];
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            const float e0 = fast_exp2(x[m][n][2 * h] - ref), e1 = fast_exp2(x[m][n][2 * h + 1] - ref);
            l[m][h] += e0 + e1;
            pa[m][n >> 1][2 * (n & 1) + h] = kFp8 ? pack_f16x2(e0 * v_s[n >> 1], e1 * v_s[n >> 1]) : pack_bf16x2(e0, e1);
          }
        }
      }
      // O += P V.  V of keys past the last one may hold anything: zeros take
      // its place (0 x NaN would reach O).
      const bool cut = key0 + kKeys > len;
      if constexpr (kFp8) {
#pragma unroll
        for (int f = 0; f < kHalves; ++f) {
          uint32_t w[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 16 * f + 2 * t4 + (i & 1) + (i >> 1) * 8;
            uint4 v = lds128(sV(s) + (uint32_t)(key * kKvD + ((g ^ (key & 7)) << 4)));
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
                for (int m = 0; m < kTiles; ++m) mma_f16(o[m][4 * q + 2 * h + i], pa[m][f], b0, b1);
              }
            }
          }
        }
      } else {
        ok = __all_sync(0xffffffffu, mbar_wait(full(1), used & 1u, p.timeout_ns, abort_flag));
        if (!ok) break;
        if (cut) {
          for (int c = lane; c < kKeys * 16; c += 32) {
            const int key = c >> 4;
            if (key0 + key >= len) {
              const uint32_t dst = sV(0) + (uint32_t)(((c >> 3) & 1) * (Plan::kHalfBytes / 2) + key * 128 + (c & 7) * 16);
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0u) : "memory");
            }
          }
          __syncwarp();
        }
        // Blocks (keys 0-7, d 0-7), (keys 8-15, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 8-15).
        const int key = lane & 15;
#pragma unroll
        for (int f = 0; f < kHalves; ++f) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t cell = (uint32_t)(2 * (j & 3) + (lane >> 4));
            uint32_t r[4];
            ldmatrix_x4_trans(r, sV(0) + (uint32_t)((j >> 2) * (Plan::kHalfBytes / 2) + (16 * f + key) * 128) +
                                     ((cell ^ (uint32_t)(key & 7)) << 4));
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
              mma_bf16(o[m][2 * j], pa[m][f], r[0], r[1]);
              mma_bf16(o[m][2 * j + 1], pa[m][f], r[2], r[3]);
            }
          }
        }
        if (cut) fence_proxy_async_smem();  // the zeros, before TMA writes there again
      }
      __syncwarp();  // the stage (bf16: V) is read: load into it
      if constexpr (kFp8) {
        load_next();
      } else {
        load_v();
      }
    }
    if (!ok) break;

    // ---- the rows go out: finished, or as a partial result -----------------------
    const bool whole = !kCluster && cur.t0 == 0 && cur.t1 == cur.units;
    [[maybe_unused]] float* part = kCluster ? nullptr : p.part + (size_t)(2 * worker + (cur.t0 == 0 ? 1 : 0)) * Plan::kPartFloats;
    // Four (fp8) or two columns from d on to the partial result.
    auto put4 = [&](int r, int d, float a, float b, float c, float e) {
      const float4 v = make_float4(a, b, c, e);
      if constexpr (kCluster) {
        *reinterpret_cast<float4*>(base_ptr + (sK(0) - base) + split_cell(r, d >> 2)) = v;
      } else {
        *reinterpret_cast<float4*>(part + (size_t)r * kKvD + d) = v;
      }
    };
    auto put2 = [&](int r, int d, float a, float b) {
      if constexpr (kCluster) {
        *reinterpret_cast<float2*>(base_ptr + (sK(0) - base) + split_cell(r, d >> 2) + (d & 2) * 4) = make_float2(a, b);
      } else {
        *reinterpret_cast<float2*>(part + (size_t)r * kKvD + d) = make_float2(a, b);
      }
    };
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[m][h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int r = m * 16 + h * 8 + g, row = row0 + r;
        if (row >= p.rows) continue;
        const int tok = row / p.group, head = kv_head * p.group + row % p.group;
        const bool none = sum == 0.0f || tok >= tokens;  // nothing seen, or a padding query
        const float inv = !whole ? 1.0f : none ? 0.0f : 1.0f / sum;
        __nv_bfloat16* out = p.o + cur.b * p.o_batch + tok * p.o_seq + head * p.o_head;
        // This thread's columns: fp8: 32 t4 + 16 c + j (accumulator j, value c); bf16: 8 j + 2 t4 + c.
#pragma unroll
        for (int c = 0; c < (kFp8 ? 2 : 1); ++c) {
#pragma unroll
          for (int j = 0; j < 16; j += kFp8 ? 8 : 1) {
            if constexpr (kFp8) {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = o[m][j + i][2 * h + c] * inv;
              const int d = 32 * t4 + 16 * c + j;
              if (whole) {
                uint4 w = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                     pack_bf16x2(v[6], v[7]));
                if (none) w = make_uint4(0u, 0u, 0u, 0u);
                *reinterpret_cast<uint4*>(out + d) = w;
              } else {
                put4(r, d, v[0], v[1], v[2], v[3]);
                put4(r, d + 4, v[4], v[5], v[6], v[7]);
              }
            } else {
              const float v0 = o[m][j][2 * h] * inv, v1 = o[m][j][2 * h + 1] * inv;
              const int d = 8 * j + 2 * t4;
              if (whole) {
                *reinterpret_cast<uint32_t*>(out + d) = none ? 0u : pack_bf16x2(v0, v1);
              } else {
                put2(r, d, v0, v1);
              }
            }
          }
        }
        if (t4 == 0) {
          if constexpr (kCluster) {
            ml[r] = make_float2(mx[m][h], sum);
          } else if (!whole) {
            *reinterpret_cast<float2*>(part + (size_t)kRows * kKvD + 2 * r) = make_float2(mx[m][h], sum);
          } else if (p.lse != nullptr) {
            p.lse[((size_t)cur.b * p.heads + head) * p.q_len + tok] =
                none ? -INFINITY : (mx[m][h] + log2f(sum)) * 0.6931471805599453f;
          }
        }
      }
    }
    if (cur.last >= 0) desc = make_int4(cur.last, cur.b, cur.seg, tokens);
  }
  if (!ok) {
    if (lane == 0) attn_raise(p, abort_flag, kDevTimeoutEpilogue);
    // Let the copies in flight land before the CTA can leave.
    bool drained = true;
    if constexpr (kFp8) {
      for (uint32_t i = used; drained && i < loaded; ++i) {
        drained = mbar_wait(full((int)(i % kStages)), (i / kStages) & 1u, p.timeout_ns, nullptr);
      }
    } else {
      if (loaded > 0) drained = mbar_wait(full(0), (loaded - 1) & 1u, p.timeout_ns, nullptr);
      if (drained && v_loaded > 0) drained = mbar_wait(full(1), (v_loaded - 1) & 1u, p.timeout_ns, nullptr);
    }
    if (!drained && lane == 0) attn_raise(p, abort_flag, kDevTimeoutDrain);
  }
  if constexpr (kCluster) {
    // ---- the cluster's results meet: a warp per row, 4 columns per lane, in order ----
    cluster_arrive();
    cluster_wait();
    const int kv_head = only.seg / p.row_tiles, row0 = (only.seg % p.row_tiles) * kRows;
    int tokens = p.q_len;
    if (kFp8 && p.new_lens != nullptr) tokens = min(max(p.new_lens[only.b], 0), p.q_len);
    for (int r = self; r < min(kRows, p.rows - row0); r += workers) {
      // Worker w is warp w % 4 of CTA w / 4 of the cluster.
      auto at = [&](int w, uint32_t off, uint32_t pitch) {
        return mapa_shared(base + off + (uint32_t)(w % kSplitWarps) * pitch, (uint32_t)(w / kSplitWarps));
      };
      float2 mine = make_float2(-INFINITY, 0.0f);
      if (lane < workers) mine = ld_cluster_v2(at(lane, Plan::kOffMl, kRows * 8) + (uint32_t)(r * 8));
      float big = mine.x;
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, k));
      const float root = mine.x == -INFINITY ? 0.0f : fast_exp2(0.5f * (mine.x - big));  // in two steps, as above
      const float f = root * root;
      float sum = mine.y * root * root;
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int w0 = 0; w0 < workers; w0 += 4) {
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = ld_cluster_v4(at(w0 + i, 0, Plan::kStages * Plan::kStageBytes) + split_cell(r, lane));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __shfl_sync(0xffffffffu, f, w0 + i);
          // (NaN passes; without weight the memory may hold anything.)
          if (w != 0.0f) acc.x += v[i].x * w, acc.y += v[i].y * w, acc.z += v[i].z * w, acc.w += v[i].w * w;
        }
      }
      const int row = row0 + r, tok = row / p.group, head = kv_head * p.group + row % p.group;
      const bool none = sum == 0.0f || tok >= tokens;  // nothing seen, or a padding query
      const float inv = none ? 0.0f : 1.0f / sum;
      uint2 w2 = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      if (none) w2 = make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(p.o + only.b * p.o_batch + tok * p.o_seq + head * p.o_head + 4 * lane) = w2;
      if (p.lse != nullptr && lane == 0) {
        p.lse[((size_t)only.b * p.heads + head) * p.q_len + tok] = none ? -INFINITY : (big + log2f(sum)) * 0.6931471805599453f;
      }
    }
    // No CTA may leave while another reads its shared memory.
    cluster_arrive();
    cluster_wait();
    return;
  }
  if (lane == 0 && p.desc != nullptr) p.desc[worker] = desc;
  // Entries without keys: zeros.
  for (int e = worker; e < p.batch; e += (int)gridDim.x * kSplitWarps) {
    if (split_len<kFp8>(p, e) > 0) continue;
    for (int r = 0; r < p.q_len * p.heads; ++r) {
      const int tok = r / p.heads, head = r % p.heads;
      *reinterpret_cast<uint2*>(p.o + e * p.o_batch + tok * p.o_seq + head * p.o_head + 4 * lane) = make_uint2(0u, 0u);
      if (p.lse != nullptr && lane == 0) p.lse[((size_t)e * p.heads + head) * p.q_len + tok] = -INFINITY;
    }
  }
#endif  // B200_NO_SM100A_FEATURES
}

// Joins the partial results of the segments that were cut.  Block (x, y): of
// the segments that begin in kJoinWorkers workers every gridDim.y-th row.  A
// (segment, row) pair gets `share` warps, which take its partials in turn, 4
// columns per lane; their results are added in order.
constexpr int kJoinWorkers = 12, kJoinWarps = 8, kJoinRowBlocks = 4;
template <int kTiles>
__global__ void __launch_bounds__(32 * kJoinWarps) attn_join_kernel(const __grid_constant__ SplitAttnParams p) {
  constexpr int kRows = 16 * kTiles;
  constexpr size_t kPartFloats = SplitPlan<true, kTiles>::kPartFloats;
  __shared__ float4 part_o[kJoinWarps][32];
  __shared__ float2 part_ml[kJoinWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = (int)(threadIdx.x & 31u), warp = (int)threadIdx.x >> 5;
  const int first = (int)blockIdx.x * kJoinWorkers;
  int4 d = make_int4(-1, 0, 0, 0);
  if (lane < kJoinWorkers && first + lane < p.workers) d = p.desc[first + lane];
  const uint32_t valid = __ballot_sync(0xffffffffu, d.x >= 0);
  const int count = __popc(valid);
  const int rows = (min(kRows, p.rows) - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y;  // of this block
  const int pairs = count * rows;
  if (pairs == 0) return;
  int share = 1;
  while (2 * share * pairs <= kJoinWarps) share *= 2;
  for (int p0 = 0; p0 < pairs; p0 += kJoinWarps / share) {
    const int pair = p0 + warp / share, turn = warp % share;
    const int r = (int)blockIdx.y + (pair % rows) * (int)gridDim.y;
    uint32_t rest = valid;  // the pair's segment: the (pair / rows)-th valid lane's
    for (int k = min(pair / rows, count - 1); k > 0; --k) rest &= rest - 1;
    const int from = __ffs(rest) - 1, worker = first + from;
    const int last = __shfl_sync(0xffffffffu, d.x, from), entry = __shfl_sync(0xffffffffu, d.y, from);
    const int seg = __shfl_sync(0xffffffffu, d.z, from), tokens = __shfl_sync(0xffffffffu, d.w, from);
    const int kv_head = seg / p.row_tiles, row = (seg % p.row_tiles) * kRows + r;
    const bool any = pair < pairs && row < p.rows;
    // The segment's first partial is in its worker's second slot, the others in their first.
    auto slot = [&](int c) { return p.part + (size_t)(2 * c + (c == worker ? 1 : 0)) * kPartFloats; };
    float big = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // (big, sum, acc) scaled for a new maximum; factors 2^x in two steps, as above.
    auto raise_to = [&](float next) {
      const float root = big == next ? 1.0f : fast_exp2(0.5f * (big - next));
      const float f = root * root;
      sum = sum * root * root;
      acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
      big = next;
    };
    if (any) {
      // This warp's partials worker + turn + i * share (none if it comes past the last).
      const int mine = worker + turn <= last ? (last - worker - turn) / share + 1 : 0;
      for (int i0 = 0; i0 < mine; i0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.0f);  // of partial i0 + lane
        if (i0 + lane < mine) {
          ml = *reinterpret_cast<const float2*>(slot(worker + turn + (i0 + lane) * share) + (size_t)kRows * kKvD + 2 * r);
        }
        float4 v[8];
        const int n = min(32, mine - i0);
        auto load8 = [&](int j0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = i0 + min(j0 + j, n - 1);
            v[j] = *reinterpret_cast<const float4*>(slot(worker + turn + i * share) + (size_t)r * kKvD + 4 * lane);
          }
        };
        load8(0);
        float top = ml.x;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        if (top > big) raise_to(top);
        const float root = ml.x == -INFINITY ? 0.0f : fast_exp2(0.5f * (ml.x - big));
        const float f = root * root;
        float add = ml.y * root * root;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) add += __shfl_xor_sync(0xffffffffu, add, k);
        sum += add;
        for (int j0 = 0; j0 < n; j0 += 8) {
          if (j0 > 0) load8(j0);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float w = __shfl_sync(0xffffffffu, f, min(j0 + j, 31));
            if (j0 + j < n) acc.x += v[j].x * w, acc.y += v[j].y * w, acc.z += v[j].z * w, acc.w += v[j].w * w;
          }
        }
      }
    }
    if (share > 1) {
      part_o[warp][lane] = acc;
      if (lane == 0) part_ml[warp] = make_float2(big, sum);
      __syncthreads();
    }
    if (any && turn == 0) {
      for (int w = 1; w < share; ++w) {
        const float2 ml = part_ml[warp + w];
        const float4 v = part_o[warp + w][lane];
        if (ml.x > big) raise_to(ml.x);
        const float root = ml.x == -INFINITY ? 0.0f : fast_exp2(0.5f * (ml.x - big)), f = root * root;
        sum += ml.y * root * root;
        acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
      }
      const int tok = row / p.group, head = kv_head * p.group + row % p.group;
      const bool none = sum == 0.0f || tok >= tokens;
      const float inv = none ? 0.0f : 1.0f / sum;
      uint2 w2 = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      if (none) w2 = make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(p.o + entry * p.o_batch + tok * p.o_seq + head * p.o_head + 4 * lane) = w2;
      if (p.lse != nullptr && lane == 0) {
        p.lse[((size_t)entry * p.heads + head) * p.q_len + tok] = none ? -INFINITY : (big + log2f(sum)) * 0.6931471805599453f;
      }
    }
    // (With share > 1 all pairs fit in one turn: no second use of the buffers.)
  }
}

// Adds the parts of cross attention split along the keys: a warp per query
// row, 4 columns per lane, eight parts in flight, in order.
struct AttnMergeParams {
  const float* part_o;    // [parts, batch, heads, q_len, 128]
  const float* part_lse;  // [parts, batch, heads, q_len]
  __nv_bfloat16* o;       // [batch, q_len, heads, 128], strides in elements
  int64_t o_batch, o_seq, o_head;
  float* lse;             // [batch, heads, q_len] or NULL
  int32_t parts, heads, q_len;
  int64_t rows;           // batch * heads * q_len
};
__global__ void __launch_bounds__(256) attn_merge_kernel(const __grid_constant__ AttnMergeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = (int)(threadIdx.x & 31u);
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  float top = -INFINITY;
  for (int s = lane; s < p.parts; s += 32) top = fmaxf(top, p.part_lse[s * p.rows + row]);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  float sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = 0; s0 < p.parts; s0 += 8) {
    float l[8];
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t s = min(s0 + i, p.parts - 1);
      l[i] = p.part_lse[s * p.rows + row];
      v[i] = *reinterpret_cast<const float4*>(p.part_o + (s * p.rows + row) * kAttnD + 4 * lane);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s0 + i >= p.parts || l[i] == -INFINITY) continue;  // (O of a part without keys is not written)
      const float w = __expf(l[i] - top);
      sum += w;
      acc.x += w * v[i].x, acc.y += w * v[i].y, acc.z += w * v[i].z, acc.w += w * v[i].w;
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t bh = row / p.q_len;
  const int64_t tok = row - bh * p.q_len;
  *reinterpret_cast<uint2*>(p.o + bh / p.heads * p.o_batch + tok * p.o_seq + bh % p.heads * p.o_head + 4 * lane) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (p.lse != nullptr && lane == 0) p.lse[row] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

}  // namespace b200
