// Host side of attention to stored keys and values (include/b200_gemm.h):
// the 8-bit cache, attention over it, cross attention and its gradients.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <utility>

#include "attn_bwd_sm100.cuh"
#include "attn_sm100.cuh"
#include "attn_split_sm100.cuh"
#include "b200_gemm.h"
#include "device_info.h"
#include "kv_cache_sm100.cuh"

namespace {

constexpr int kMaxDevices = 64;
constexpr int64_t kLim = 0x7fffffffLL;
constexpr size_t kWsAlign = 256;

using SplitKernel = void (*)(const CUtensorMap, const CUtensorMap, const b200::SplitAttnParams);
struct SplitVariant {
  SplitKernel kernel;   // the line of units over all warps
  SplitKernel cluster;  // a cluster per segment
  void (*join)(const b200::SplitAttnParams);
  int tiles;  // row tiles per warp
  int smem;
  size_t part_floats;
};
// bf16 states of few query rows; the 8-bit cache with one or two row tiles per warp.
enum SplitIndex { kSplitBf16 = 0, kSplitFp8 = 1, kSplitFp8Wide = 2, kSplitVariants = 3 };
const SplitVariant kSplit[kSplitVariants] = {
    {b200::attn_split_kernel<false, 1, false>, b200::attn_split_kernel<false, 1, true>, b200::attn_join_kernel<1>, 1, b200::SplitPlan<false, 1>::kAllocBytes,
     b200::SplitPlan<false, 1>::kPartFloats},
    {b200::attn_split_kernel<true, 1, false>, b200::attn_split_kernel<true, 1, true>, b200::attn_join_kernel<1>, 1, b200::SplitPlan<true, 1>::kAllocBytes,
     b200::SplitPlan<true, 1>::kPartFloats},
    {b200::attn_split_kernel<true, 2, false>, b200::attn_split_kernel<true, 2, true>, b200::attn_join_kernel<2>, 2, b200::SplitPlan<true, 2>::kAllocBytes,
     b200::SplitPlan<true, 2>::kPartFloats}};

struct StoredState {
  std::once_flag once;
  int init_rc = B200_OK;
  int sm_count = 0;
  bool cross_regs_ok = false, bwd_regs_ok = false;  // setmaxnreg shares match the binary (attn_sm100.cuh)
  int split_ctas[kSplitVariants] = {};  // resident CTAs of each split variant on the whole GPU
};
StoredState g_stored[kMaxDevices];

int init_stored(const b200::DeviceInfo& di, StoredState& st) {
  if (cudaFuncSetAttribute(b200::flash_attn_fwd_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           b200::AttnSmemPlan::kAllocBytes) != cudaSuccess)
    return B200_ERR_CUDA;
  cudaFuncAttributes fa{};
  if (cudaFuncGetAttributes(&fa, b200::flash_attn_fwd_kernel<true>) != cudaSuccess) return B200_ERR_CUDA;
  st.sm_count = di.sm_count;
  st.cross_regs_ok = fa.numRegs == (int)b200::kAttnRegsLaunch;
  st.bwd_regs_ok = true;
  const std::pair<const void*, int> bwd[2] = {
      {(const void*)b200::attn_bwd_kernel<false>, b200::AttnBwdPlan<false>::kAllocBytes},
      {(const void*)b200::attn_bwd_kernel<true>, b200::AttnBwdPlan<true>::kAllocBytes}};
  for (const auto& k : bwd) {
    if (cudaFuncSetAttribute(k.first, cudaFuncAttributeMaxDynamicSharedMemorySize, k.second) != cudaSuccess ||
        cudaFuncGetAttributes(&fa, k.first) != cudaSuccess)
      return B200_ERR_CUDA;
    if (fa.numRegs != (int)b200::kAttnRegsLaunch) st.bwd_regs_ok = false;
  }
  for (int i = 0; i < kSplitVariants; ++i) {
    const SplitVariant& v = kSplit[i];
    int per_sm = 0;
    if (cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem) != cudaSuccess ||
        cudaFuncSetAttribute(v.cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, v.kernel, b200::kSplitThreads, v.smem) != cudaSuccess ||
        per_sm < 1)
      return B200_ERR_CUDA;
    st.split_ctas[i] = per_sm * di.sm_count;
  }
  return B200_OK;
}

int current_state(b200::DeviceInfo* di, StoredState** out) {
  const int rc = b200::device_info(di);
  if (rc != B200_OK) return rc;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return B200_ERR_CUDA;
  StoredState& st = g_stored[dev];
  std::call_once(st.once, [&] { st.init_rc = init_stored(*di, st); });
  if (st.init_rc != B200_OK) return st.init_rc;
  *out = &st;
  return B200_OK;
}

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A strided operand [batch, tokens, heads, 128]: strides positive multiples
// of 8 elements where the extent is above 1, below the tensor maps' 2^40
// bytes; strides of extent 1 are replaced by a valid value.
int check_view(const b200_attn_view* v, int64_t batch, int64_t tokens, int64_t heads, b200_attn_view* out) {
  if (v == nullptr || v->data == nullptr) return B200_ERR_INVALID_ARG;
  *out = *v;
  const int64_t extent[3] = {batch, tokens, heads};
  int64_t* stride[3] = {&out->batch_stride, &out->seq_stride, &out->head_stride};
  for (int i = 0; i < 3; ++i) {
    if (extent[i] <= 1) *stride[i] = b200::kKvD;
    if (*stride[i] < b200::kKvD) return B200_ERR_INVALID_ARG;
    if (*stride[i] % 8 != 0) return B200_ERR_ALIGNMENT;
    if (*stride[i] >= (1LL << 39)) return B200_ERR_TOO_LARGE;
  }
  return aligned(v->data, 16) ? B200_OK : B200_ERR_ALIGNMENT;
}

// 4-D bf16 map {128, heads, tokens, batch}: boxes of 64 columns x box_rows tokens of one head, 128B swizzle.
int encode_view(const b200::DeviceInfo& di, CUtensorMap* map, const b200_attn_view& v, int64_t batch, int64_t tokens,
                int64_t heads, uint32_t box_rows, bool is_load) {
  cuuint64_t dims[4] = {(cuuint64_t)b200::kKvD, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
  cuuint64_t strides[3] = {(cuuint64_t)v.head_stride * 2, (cuuint64_t)v.seq_stride * 2, (cuuint64_t)v.batch_stride * 2};
  cuuint32_t box[4] = {64, 1, box_rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = di.encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, v.data, dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               is_load ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200_OK : B200_ERR_TENSOR_MAP;
}

// The cache's codes as rows of 128 bytes; boxes of a page, at most a unit of keys.
int encode_cache(const b200::DeviceInfo& di, CUtensorMap* map, void* codes, int64_t rows, int64_t page_size) {
  cuuint64_t dims[2] = {(cuuint64_t)b200::kKvD, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)b200::kKvD};
  cuuint32_t box[2] = {(cuuint32_t)b200::kKvD, (cuuint32_t)std::min<int64_t>(page_size, b200::SplitPlan<true, 1>::kKeys)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = di.encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200_OK : B200_ERR_TENSOR_MAP;
}

// fp32 parts of cross attention's O, [parts x batch x heads, q_len, 128]: boxes of 32 columns x 32 rows.
int encode_parts(const b200::DeviceInfo& di, CUtensorMap* map, float* data, int64_t q_len, int64_t outer) {
  cuuint64_t dims[3] = {(cuuint64_t)b200::kAttnD, (cuuint64_t)q_len, (cuuint64_t)outer};
  cuuint64_t strides[2] = {(cuuint64_t)b200::kAttnD * 4, (cuuint64_t)b200::kAttnD * 4 * (cuuint64_t)q_len};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = di.encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, data, dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200_OK : B200_ERR_TENSOR_MAP;
}

template <typename... Params, typename... Args>
int launch_clusters(void (*kernel)(Params...), int cluster, dim3 grid, int threads, int smem, cudaStream_t stream,
                    const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return B200_OK;
  cudaGetLastError();
  return B200_ERR_CUDA;
}
template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
  return launch_clusters(kernel, 1, grid, threads, smem, stream, args...);
}

int check_heads(int64_t batch, int64_t q_len, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  if (batch < 0 || q_len < 0 || heads < 0 || kv_heads < 0) return B200_ERR_INVALID_ARG;
  if (head_dim != b200::kKvD) return B200_ERR_INVALID_ARG;
  if ((heads > 0 && kv_heads == 0) || (kv_heads > 0 && heads % kv_heads != 0)) return B200_ERR_INVALID_ARG;
  if (batch > 65535 || heads > 65535 || heads * batch > kLim || q_len * heads > kLim) return B200_ERR_TOO_LARGE;
  return B200_OK;
}

int check_cache(const b200_kv_cache* c) {
  if (c == nullptr || c->num_pages < 0 || c->kv_heads < 0 || c->max_pages < 0) return B200_ERR_INVALID_ARG;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return B200_ERR_INVALID_ARG;
  if (c->table_stride < c->max_pages) return B200_ERR_INVALID_ARG;
  if (c->num_pages > kLim || c->kv_heads > 65535 || c->num_pages * c->kv_heads > kLim / c->page_size ||
      c->max_pages > (kLim - 128) / c->page_size)
    return B200_ERR_TOO_LARGE;
  return B200_OK;
}

int check_cache_pointers(const b200_kv_cache* c) {
  if (c->num_pages > 0 && (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr))
    return B200_ERR_INVALID_ARG;
  if (c->max_pages > 0 && c->block_table == nullptr) return B200_ERR_INVALID_ARG;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
      !aligned(c->block_table, 4))
    return B200_ERR_ALIGNMENT;
  return B200_OK;
}

// Launch shape of a split variant for `rows` query rows per key/value head.
struct SplitShape {
  SplitIndex index;
  int64_t row_tiles;
  int cluster;  // CTAs per segment, 0: the line
  int each;     // units per warp of a cluster
  int ctas;
  bool cut;  // some segment can be longer than a unit: partial results need the workspace
  size_t bytes;
};
int plan_split(const StoredState& st, SplitIndex index, int64_t batch, int64_t rows, int64_t kv_heads, int64_t kv_len,
               SplitShape* out) {
  const SplitVariant& v = kSplit[index];
  out->index = index;
  out->row_tiles = (rows + 16 * v.tiles - 1) / (16 * v.tiles);
  constexpr int64_t keys = b200::SplitPlan<true, 1>::kKeys;  // of a unit, the same for all variants
  const int64_t units = (kv_len + keys - 1) / keys;          // of the longest segment
  const int64_t segs = kv_heads * out->row_tiles;
  if (segs > kLim) return B200_ERR_TOO_LARGE;
  const double all_segs = (double)batch * (double)segs;  // (in double: the products may pass 2^63)
  // A cluster per segment, large enough for a unit per warp if the clusters
  // still fit two CTAs to an SM, while its warps have few units.  Measured on a B200, 8-bit
  // cache: 8 segments of 1000 keys 7.8 us against 12.9 along the line, of 4000 11.8
  // against 14.9; 128 of 1000 16.2 against 22.1, of 2000 24.7 against 27.5, of 4000 41.9
  // against 37.5; 512 of 250 18.0 against 21.9, of 1000 37.7 against 38.5, of 2000 62 against 59.
  int cluster = 1;
  while (cluster < 8 && b200::kSplitWarps * cluster < units && 2 * cluster * all_segs <= 2.0 * st.sm_count) cluster *= 2;
  const int64_t each = (units + b200::kSplitWarps * cluster - 1) / (b200::kSplitWarps * cluster);  // units per warp
  out->cluster = 0;
  if (each <= (cluster == 8 ? 4 : 8) && all_segs * cluster <= (double)kLim) {
    out->cluster = cluster;
    out->each = (int)each;
    out->ctas = (int)(all_segs * cluster);
    out->cut = false;
    out->bytes = 0;
    return B200_OK;
  }
  // One worker per unit at most.
  const double most = all_segs * (double)std::max<int64_t>(units, 1);
  out->ctas = (int)std::min((double)st.split_ctas[index], std::ceil(most / b200::kSplitWarps));
  out->cut = units > 1;
  out->bytes = out->cut ? (size_t)(out->ctas * b200::kSplitWarps) * (2 * v.part_floats * sizeof(float) + sizeof(int4)) : 0;
  out->bytes = (out->bytes + kWsAlign - 1) / kWsAlign * kWsAlign;
  return B200_OK;
}

int check_workspace(const void* workspace, size_t have, size_t need) {
  if (need == 0) return B200_OK;
  if (workspace == nullptr || have < need) return B200_ERR_INVALID_ARG;
  return aligned(workspace, kWsAlign) ? B200_OK : B200_ERR_ALIGNMENT;
}

int run_split(const b200::DeviceInfo& di, const SplitShape& shape, const CUtensorMap& tmK, const CUtensorMap& tmV,
              b200::SplitAttnParams& p, void* workspace, cudaStream_t stream) {
  const SplitVariant& v = kSplit[shape.index];
  const int workers = shape.ctas * b200::kSplitWarps;
  if (shape.bytes > 0) {
    p.part = static_cast<float*>(workspace);
    p.desc = reinterpret_cast<int4*>(p.part + 2 * (size_t)workers * v.part_floats);
  }
  p.row_tiles = (int32_t)shape.row_tiles;
  p.workers = workers;
  p.timeout_ns = di.timeout_ns;
  p.status = di.status;
  if (shape.cluster > 0) {
    return launch_clusters(v.cluster, shape.cluster, dim3((unsigned)shape.ctas), b200::kSplitThreads, v.smem, stream, tmK,
                           tmV, p);
  }
  const int rc = launch(v.kernel, dim3((unsigned)shape.ctas), b200::kSplitThreads, v.smem, stream, tmK, tmV, p);
  if (rc != B200_OK || !shape.cut) return rc;
  const int rows = std::min<int>(p.rows, 16 * v.tiles);
  const dim3 grid((unsigned)((workers + b200::kJoinWorkers - 1) / b200::kJoinWorkers),
                  (unsigned)std::min(rows, b200::kJoinRowBlocks));
  return launch(v.join, grid, 32 * b200::kJoinWarps, 0, stream, p);
}

// How cross attention runs: on the split kernel, or on the tcgen05 kernel in
// `parts` along the keys.
struct CrossShape {
  bool few;
  SplitShape split;
  int parts;
  size_t bytes;
};
int plan_cross(const b200::DeviceInfo& di, const StoredState& st, int64_t batch, int64_t q_len, int64_t kv_len,
               int64_t heads, int64_t kv_heads, CrossShape* out) {
  *out = CrossShape{};
  out->parts = 1;
  const int64_t q_tiles = (q_len + b200::kAttnBQ - 1) / b200::kAttnBQ;
  const int64_t ctas = heads * batch * ((q_tiles + b200::kAttnQTiles - 1) / b200::kAttnQTiles);
  const int64_t tiles = (kv_len + b200::kAttnBKV - 1) / b200::kAttnBKV;
  // The tcgen05 kernel, on a B200: 5 us a wave of CTAs to start and end, and per key
  // tile 1.1 us for a query tile alone and 1.95 for two together; K and V at 5.6
  // TB/s at most, 4.8 in several waves.  While parts fit beside each other (of two
  // key tiles at least) they save tiles, but cost 3.8 us for the merge and their O once out and once
  // back, 1 KiB a row and part at 4 TB/s.  Measured: 128 queries, 4 heads, 4000
  // keys: 16 parts 13 us against one 56; 256 queries, 2 x 32 heads, 1000 keys: 2 parts 26
  // against 21.
  const int64_t rows = batch * heads * q_len;
  const double bytes = 4.0 * b200::kKvD * (double)batch * (double)kv_heads * (double)kv_len;  // of K and V
  const double per_tile = q_tiles == 1 ? 1.1 : 1.95;
  const double waves = std::ceil((double)ctas / di.sm_count);
  double tc = waves * (5.0 + (double)tiles * per_tile);
  const int64_t most = ctas < di.sm_count ? std::min(di.sm_count / ctas, tiles / 2) : 1;
  for (int64_t n = 2; n <= most; ++n) {
    const double t = 8.8 + (double)((tiles + n - 1) / n) * per_tile + 1024.0 * (double)(rows * n) / 4e6;
    if (t < tc) {
      tc = t;
      out->parts = (int)n;
    }
  }
  tc = std::max(tc, 3.0 + bytes / (waves > 1.0 ? 4.8e6 : 5.6e6));
  // The split kernel, for up to 16 rows per key/value head (two row tiles per
  // warp lost to the tcgen05 kernel in parts: 32 rows, 4 heads, 1000 keys 17 us
  // against 11): in clusters 3.5 us, 0.6 for each doubling, 1.25 per unit of a warp,
  // and K and V, partly beside that; along the line 9.5 us and K and V at 5.6 TB/s; with
  // more than 8 rows 1.2 to 4.2 us more for their queries and outputs.  Measured, split against tcgen05: one query, 16 heads, 128 keys
  // 4.4 us against 5.4, 1000 keys 6.8 against 10.1; 8 x 16 heads, 4000 keys 54 against
  // 47; 16 queries, 8 x 16 heads, 128 keys 9.5 against 6.2.
  const int64_t group_rows = q_len * (heads / kv_heads);
  if (group_rows <= 16) {
    const int rc = plan_split(st, kSplitBf16, batch, group_rows, kv_heads, kv_len, &out->split);
    if (rc != B200_OK) return rc;
    const double split = (out->split.cluster > 0 ? 3.5 + 0.6 * std::log2((double)out->split.cluster) +
                                                       1.25 * out->split.each + bytes / 1.2e7
                                                 : 9.5 + bytes / 5.6e6) +
                         (group_rows > 8 ? 1.2 + std::min(3.0, 0.07 * (double)(batch * kv_heads)) : 0.0);
    out->few = split < tc;
  }
  if (out->few) {
    out->parts = 1;
    out->bytes = out->split.bytes;
    return B200_OK;
  }
  if (out->parts > 1) out->bytes = (size_t)out->parts * (size_t)(batch * heads * q_len) * (b200::kAttnD + 1) * sizeof(float);
  out->bytes = (out->bytes + kWsAlign - 1) / kWsAlign * kWsAlign;
  return B200_OK;
}

// Over the cache: two row tiles per warp from 17 rows per key/value head on.
int plan_cache(const StoredState& st, int64_t batch, int64_t rows, const b200_kv_cache* cache, SplitShape* out) {
  return plan_split(st, rows <= 16 ? kSplitFp8 : kSplitFp8Wide, batch, rows, cache->kv_heads,
                    cache->max_pages * cache->page_size, out);
}

bool scale_ok(float scale) { return scale > 0.0f && std::isfinite(scale); }

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace

extern "C" B200_API int b200_kv_cache_write(const b200_attn_view* k, const b200_attn_view* v, const b200_kv_cache* cache,
                                            const int32_t* seq_lens, const int32_t* new_lens, int64_t batch,
                                            int64_t new_max, int64_t head_dim, void* stream_) {
  int rc = check_cache(cache);
  if (rc != B200_OK) return rc;
  if (batch < 0 || new_max < 0 || head_dim != b200::kKvD) return B200_ERR_INVALID_ARG;
  if (batch > 65535 || new_max > kLim) return B200_ERR_TOO_LARGE;
  if (batch == 0 || new_max == 0 || cache->kv_heads == 0) return B200_OK;
  if (seq_lens == nullptr) return B200_ERR_INVALID_ARG;
  if ((rc = check_cache_pointers(cache)) != B200_OK) return rc;
  b200_attn_view kk, vv;
  if ((rc = check_view(k, batch, new_max, cache->kv_heads, &kk)) != B200_OK) return rc;
  if ((rc = check_view(v, batch, new_max, cache->kv_heads, &vv)) != B200_OK) return rc;
  const int64_t page = cache->page_size;
  // New tokens reach at most this many pages of a sequence (the first may hold older tokens).
  const int64_t touched = std::min((new_max - 1 + page - 1) / page + 1, std::max<int64_t>(cache->max_pages, 1));
  const int64_t blocks = batch * touched * cache->kv_heads * 2;
  if (touched > kLim || blocks > kLim) return B200_ERR_TOO_LARGE;
  b200::DeviceInfo di;
  if ((rc = b200::device_info(&di)) != B200_OK) return rc;
  b200::KvWriteParams p{};
  const b200_attn_view* in[2] = {&kk, &vv};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = static_cast<const __nv_bfloat16*>(in[i]->data);
    p.x_batch[i] = in[i]->batch_stride;
    p.x_seq[i] = in[i]->seq_stride;
    p.x_head[i] = in[i]->head_stride;
  }
  p.cache[0] = static_cast<uint8_t*>(cache->k);
  p.cache[1] = static_cast<uint8_t*>(cache->v);
  p.scale[0] = cache->k_scale;
  p.scale[1] = cache->v_scale;
  p.table = cache->block_table;
  p.table_stride = cache->table_stride;
  p.seq_lens = seq_lens;
  p.new_lens = new_lens;
  p.new_max = (int32_t)new_max;
  p.kv_heads = (int32_t)cache->kv_heads;
  p.num_pages = (int32_t)cache->num_pages;
  p.max_pages = (int32_t)cache->max_pages;
  p.pages_touched = (int32_t)touched;
  p.status = di.status;
  void (*kernel)(const b200::KvWriteParams) = page == 16   ? b200::kv_cache_write_kernel<16>
                                              : page == 32 ? b200::kv_cache_write_kernel<32>
                                              : page == 64 ? b200::kv_cache_write_kernel<64>
                                                           : b200::kv_cache_write_kernel<128>;
  return launch(kernel, dim3((unsigned)blocks), b200::kKvWriteThreads, 0, reinterpret_cast<cudaStream_t>(stream_), p);
}

extern "C" B200_API int b200_cache_attn_workspace_bytes(int64_t batch, int64_t q_len, int64_t heads,
                                                        const b200_kv_cache* cache, size_t* bytes) {
  if (bytes == nullptr) return B200_ERR_INVALID_ARG;
  *bytes = 0;
  int rc = check_cache(cache);
  if (rc != B200_OK) return rc;
  if ((rc = check_heads(batch, q_len, heads, cache->kv_heads, b200::kKvD)) != B200_OK) return rc;
  if (batch == 0 || q_len == 0 || heads == 0) return B200_OK;
  b200::DeviceInfo di;
  StoredState* st = nullptr;
  if ((rc = current_state(&di, &st)) != B200_OK) return rc;
  SplitShape shape;
  if ((rc = plan_cache(*st, batch, q_len * (heads / cache->kv_heads), cache, &shape)) != B200_OK) return rc;
  *bytes = shape.bytes;
  return B200_OK;
}

extern "C" B200_API int b200_cache_attn(const b200_attn_view* q, const b200_kv_cache* cache, const int32_t* seq_lens,
                                        const int32_t* new_lens, const b200_attn_view* o, int64_t batch, int64_t q_len,
                                        int64_t heads, int64_t head_dim, float scale, void* workspace,
                                        size_t workspace_bytes, void* stream_) {
  int rc = check_cache(cache);
  if (rc != B200_OK) return rc;
  if ((rc = check_heads(batch, q_len, heads, cache->kv_heads, head_dim)) != B200_OK) return rc;
  if (!scale_ok(scale)) return B200_ERR_INVALID_ARG;
  if (batch == 0 || q_len == 0 || heads == 0) return B200_OK;
  if (seq_lens == nullptr) return B200_ERR_INVALID_ARG;
  if ((rc = check_cache_pointers(cache)) != B200_OK) return rc;
  b200_attn_view qq, oo;
  if ((rc = check_view(q, batch, q_len, heads, &qq)) != B200_OK) return rc;
  if ((rc = check_view(o, batch, q_len, heads, &oo)) != B200_OK) return rc;
  b200::DeviceInfo di;
  StoredState* st = nullptr;
  if ((rc = current_state(&di, &st)) != B200_OK) return rc;
  b200::SplitAttnParams p{};
  p.batch = (int32_t)batch;
  p.q_len = (int32_t)q_len;
  p.heads = (int32_t)heads;
  p.kv_heads = (int32_t)cache->kv_heads;
  p.group = (int32_t)(heads / cache->kv_heads);
  p.rows = p.q_len * p.group;
  p.q = static_cast<const __nv_bfloat16*>(qq.data);
  p.q_batch = qq.batch_stride, p.q_seq = qq.seq_stride, p.q_head = qq.head_stride;
  p.o = static_cast<__nv_bfloat16*>(oo.data);
  p.o_batch = oo.batch_stride, p.o_seq = oo.seq_stride, p.o_head = oo.head_stride;
  p.scale_log2 = kLog2e * scale;
  p.seq_lens = seq_lens;
  p.new_lens = new_lens;
  p.kv_len = (int32_t)(cache->num_pages == 0 ? 0 : cache->max_pages * cache->page_size);
  p.page_size = (int32_t)cache->page_size;
  p.num_pages = (int32_t)cache->num_pages;
  p.table = cache->block_table;
  p.table_stride = cache->table_stride;
  p.k_scale = cache->k_scale;
  p.v_scale = cache->v_scale;
  SplitShape shape;
  if ((rc = plan_cache(*st, batch, p.rows, cache, &shape)) != B200_OK ||
      (rc = check_workspace(workspace, workspace_bytes, shape.bytes)) != B200_OK)
    return rc;
  CUtensorMap tmK{}, tmV{};
  if (p.kv_len > 0) {
    const int64_t rows = cache->num_pages * cache->kv_heads * cache->page_size;
    if ((rc = encode_cache(di, &tmK, cache->k, rows, cache->page_size)) != B200_OK ||
        (rc = encode_cache(di, &tmV, cache->v, rows, cache->page_size)) != B200_OK)
      return rc;
  }
  return run_split(di, shape, tmK, tmV, p, workspace, reinterpret_cast<cudaStream_t>(stream_));
}

extern "C" B200_API int b200_cross_attn_workspace_bytes(int64_t batch, int64_t q_len, int64_t kv_len, int64_t heads,
                                                        int64_t kv_heads, size_t* bytes) {
  if (bytes == nullptr) return B200_ERR_INVALID_ARG;
  *bytes = 0;
  int rc = check_heads(batch, q_len, heads, kv_heads, b200::kKvD);
  if (rc != B200_OK) return rc;
  if (kv_len < 0) return B200_ERR_INVALID_ARG;
  if (kv_len > kLim) return B200_ERR_TOO_LARGE;
  if (batch == 0 || q_len == 0 || heads == 0) return B200_OK;
  b200::DeviceInfo di;
  StoredState* st = nullptr;
  if ((rc = current_state(&di, &st)) != B200_OK) return rc;
  CrossShape shape;
  if ((rc = plan_cross(di, *st, batch, q_len, kv_len, heads, kv_heads, &shape)) != B200_OK) return rc;
  *bytes = shape.bytes;
  return B200_OK;
}

extern "C" B200_API int b200_cross_attn_bf16(const b200_attn_view* q, const b200_attn_view* k, const b200_attn_view* v,
                                             const int32_t* kv_lens, const b200_attn_view* o, float* lse, int64_t batch,
                                             int64_t q_len, int64_t kv_len, int64_t heads, int64_t kv_heads,
                                             int64_t head_dim, float scale, void* workspace, size_t workspace_bytes,
                                             void* stream_) {
  int rc = check_heads(batch, q_len, heads, kv_heads, head_dim);
  if (rc != B200_OK) return rc;
  if (kv_len < 0 || !scale_ok(scale)) return B200_ERR_INVALID_ARG;
  if (batch == 0 || q_len == 0 || heads == 0) return B200_OK;
  if (kv_len > kLim - 128 || q_len > 65535LL * b200::kAttnBQ) return B200_ERR_TOO_LARGE;
  b200_attn_view qq, kk{}, vv{}, oo;
  if ((rc = check_view(q, batch, q_len, heads, &qq)) != B200_OK) return rc;
  if ((rc = check_view(o, batch, q_len, heads, &oo)) != B200_OK) return rc;
  if (kv_len > 0) {
    if ((rc = check_view(k, batch, kv_len, kv_heads, &kk)) != B200_OK) return rc;
    if ((rc = check_view(v, batch, kv_len, kv_heads, &vv)) != B200_OK) return rc;
  }
  if (!aligned(lse, 4) || !aligned(kv_lens, 4)) return B200_ERR_ALIGNMENT;
  b200::DeviceInfo di;
  StoredState* st = nullptr;
  if ((rc = current_state(&di, &st)) != B200_OK) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  CrossShape shape;
  if ((rc = plan_cross(di, *st, batch, q_len, kv_len, heads, kv_heads, &shape)) != B200_OK ||
      (rc = check_workspace(workspace, workspace_bytes, shape.bytes)) != B200_OK)
    return rc;
  CUtensorMap tmK{}, tmV{};
  if (shape.few) {
    b200::SplitAttnParams p{};
    p.batch = (int32_t)batch;
    p.q_len = (int32_t)q_len;
    p.heads = (int32_t)heads;
    p.kv_heads = (int32_t)kv_heads;
    p.group = (int32_t)(heads / kv_heads);
    p.rows = p.q_len * p.group;
    p.q = static_cast<const __nv_bfloat16*>(qq.data);
    p.q_batch = qq.batch_stride, p.q_seq = qq.seq_stride, p.q_head = qq.head_stride;
    p.o = static_cast<__nv_bfloat16*>(oo.data);
    p.o_batch = oo.batch_stride, p.o_seq = oo.seq_stride, p.o_head = oo.head_stride;
    p.lse = lse;
    p.scale_log2 = kLog2e * scale;
    p.seq_lens = kv_lens;
    p.kv_len = (int32_t)kv_len;
    constexpr uint32_t kBox = b200::SplitPlan<false, 1>::kKeys;
    if (kv_len > 0 && ((rc = encode_view(di, &tmK, kk, batch, kv_len, kv_heads, kBox, true)) != B200_OK ||
                       (rc = encode_view(di, &tmV, vv, batch, kv_len, kv_heads, kBox, true)) != B200_OK))
      return rc;
    return run_split(di, shape.split, tmK, tmV, p, workspace, stream);
  }
  if (!st->cross_regs_ok) return B200_ERR_CUDA;  // built with another register count: never launch it
  CUtensorMap tmQ, tmO;
  if ((rc = encode_view(di, &tmQ, qq, batch, q_len, heads, b200::kAttnBQ, true)) != B200_OK) return rc;
  const int64_t rows = batch * heads * q_len;
  float* part_o = static_cast<float*>(workspace);
  float* part_lse = part_o + (size_t)shape.parts * (size_t)rows * b200::kAttnD;  // (with several parts)
  rc = shape.parts > 1 ? encode_parts(di, &tmO, part_o, q_len, shape.parts * batch * heads)
                       : encode_view(di, &tmO, oo, batch, q_len, heads, 32, false);
  if (rc != B200_OK) return rc;
  if (kv_len > 0) {
    if ((rc = encode_view(di, &tmK, kk, batch, kv_len, kv_heads, b200::kAttnBKV, true)) != B200_OK ||
        (rc = encode_view(di, &tmV, vv, batch, kv_len, kv_heads, 64, true)) != B200_OK)
      return rc;
  } else {
    tmK = tmV = tmQ;  // not read
  }
  b200::AttnParams p{};
  p.seq_len = (int32_t)q_len;
  p.heads = (int32_t)heads;
  p.batch = (int32_t)batch;
  p.group = (int32_t)(heads / kv_heads);
  p.num_q_tiles = (int32_t)((q_len + b200::kAttnBQ - 1) / b200::kAttnBQ);
  p.scale_log2 = kLog2e * scale;
  p.timeout_ns = di.timeout_ns;
  p.status = di.status;
  p.kv_len = (int32_t)kv_len;
  p.kv_lens = kv_lens;
  p.ordered = kv_lens != nullptr && batch > 1 && batch <= 32 &&
                      heads * batch * ((p.num_q_tiles + b200::kAttnQTiles - 1) / b200::kAttnQTiles) > di.sm_count
                  ? 1u
                  : 0u;
  p.lse = shape.parts > 1 ? part_lse : lse;
  const dim3 grid((unsigned)(heads * batch), (unsigned)((p.num_q_tiles + b200::kAttnQTiles - 1) / b200::kAttnQTiles),
                  (unsigned)shape.parts);
  rc = launch(b200::flash_attn_fwd_kernel<true>, grid, b200::kAttnThreads, b200::AttnSmemPlan::kAllocBytes, stream, tmQ, tmK,
              tmV, tmO, p);
  if (rc != B200_OK || shape.parts == 1) return rc;
  b200::AttnMergeParams m{};
  m.part_o = part_o;
  m.part_lse = part_lse;
  m.o = static_cast<__nv_bfloat16*>(oo.data);
  m.o_batch = oo.batch_stride, m.o_seq = oo.seq_stride, m.o_head = oo.head_stride;
  m.lse = lse;
  m.parts = shape.parts;
  m.heads = p.heads;
  m.q_len = p.seq_len;
  m.rows = rows;
  return launch(b200::attn_merge_kernel, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, m);
}

namespace {
int64_t bwd_padded(int64_t q_len) { return (q_len + 127) / 128 * 128; }
// Two item counters (padded), then lse2 and delta of every padded query row.
size_t bwd_bytes(int64_t batch, int64_t q_len, int64_t heads) {
  return kWsAlign + 2 * sizeof(float) * (size_t)(batch * heads) * (size_t)bwd_padded(q_len);
}

// Work items of the two backward kernels: dK/dV (0) and dQ (1).
struct BwdShape {
  int64_t tiles[2], items[2];  // gradient tiles per head, and of all heads and entries
  int64_t walk[2];             // tile pairs per gradient tile, at most
  int parts[2];                // items per gradient tile
  size_t part_floats(int kind) const {
    return parts[kind] > 1 ? (size_t)(items[kind] * parts[kind]) * (kind == 0 ? 2 : 1) * 128 * 128 : 0;
  }
  size_t part_bytes() const { return (part_floats(0) + part_floats(1)) * sizeof(float); }
};

int check_bwd_size(int64_t batch, int64_t q_len, int64_t kv_len, int64_t heads, int64_t kv_heads) {
  if (kv_len > kLim - 128 || q_len > kLim - 128) return B200_ERR_TOO_LARGE;
  const int64_t q_tiles = (q_len + 127) / 128, kv_tiles = (kv_len + 127) / 128;
  const int64_t dkv = kv_tiles * kv_heads, dq = q_tiles * heads;  // (below 2^41)
  if (dq > kLim || (double)batch * (double)(dkv + dq) > (double)kLim) return B200_ERR_TOO_LARGE;
  return B200_OK;
}

// When n0 items of time t0, and behind them n1 of time t1, have run on sms SMs.
double bwd_end(int sms, int64_t n0, double t0, int64_t n1, double t1) {
  const int64_t late = n0 % sms;  // SMs that have one item more of the first kind
  const double free[2] = {(double)(n0 / sms) * t0, (double)(n0 / sms + (late > 0)) * t0};
  const int64_t on[2] = {sms - late, late};
  // All SMs busy to the end is the least; from there, to where the items fit.
  const double least = ((double)n0 * t0 + (double)n1 * t1) / sms;
  double done[2], end = free[1];
  int64_t left = n1;
  for (int i = 0; i < 2; ++i) {
    done[i] = std::max(0.0, std::floor((least - free[i]) / t1));
    left -= (int64_t)done[i] * on[i];
  }
  while (left > 0) {
    const int i = on[1] > 0 && free[1] + (done[1] + 1.0) * t1 < free[0] + (done[0] + 1.0) * t1 ? 1 : 0;
    done[i] += 1.0;
    left -= on[i];
    end = std::max(end, free[i] + done[i] * t1);
  }
  for (int i = 0; i < 2; ++i) end = std::max(end, on[i] > 0 && done[i] > 0.0 ? free[i] + done[i] * t1 : 0.0);
  return end;
}

BwdShape plan_bwd(int sm_count, int64_t batch, int64_t q_len, int64_t kv_len, int64_t heads, int64_t kv_heads) {
  const int64_t q_tiles = heads > 0 ? (q_len + 127) / 128 : 0, kv_tiles = kv_heads > 0 ? (kv_len + 127) / 128 : 0;
  BwdShape s{};
  s.tiles[0] = kv_tiles, s.tiles[1] = q_tiles;
  s.items[0] = kv_tiles * kv_heads * batch, s.items[1] = q_tiles * heads * batch;
  s.walk[0] = kv_heads > 0 ? heads / kv_heads * q_tiles : 0, s.walk[1] = kv_tiles;
  s.parts[0] = s.parts[1] = 1;
  if (s.items[0] == 0 || s.items[1] == 0) return s;
  // With fewer gradient tiles than SMs the longest item is most of the time; its
  // walk is cut where the sums' way through memory and another kernel cost less.
  // On a B200: 2.3 (dK/dV, with dQ beside it) and 1.5 us (dQ) a tile pair and 4 an
  // item, dQ items on SMs as they run out of dK/dV items (bwd_end); the sums' kernel 3 us,
  // and they go 64 KiB a tile and part out and back, mostly through L2, at 12
  // TB/s.  Measured, dK/dV walks in 1, 2, 3, 4, 6 and 8 parts: 2048 queries and
  // keys, 8 and 2 heads 154, 100, 83, 75, 88, 81 us; 1024 queries, 256 keys, 32 and 8
  // heads 79, 53, 45, 40, 40, 39.
  constexpr double kPair[2] = {2.3, 1.5};
  constexpr int kTry[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
  double best = 0.0;
  int64_t most[2];
  for (int k = 0; k < 2; ++k) most[k] = s.items[k] < sm_count ? std::min(s.walk[k] / 2, 2 * (sm_count / s.items[k])) : 1;
  for (const int a : kTry) {
    if (a > 1 && a > most[0]) break;
    for (const int b : kTry) {
      if (b > 1 && b > most[1]) break;
      const int parts[2] = {a, b};
      double item[2], floats = 0.0;
      for (int k = 0; k < 2; ++k) {
        item[k] = 4.0 + kPair[k] * (double)((s.walk[k] + parts[k] - 1) / parts[k]);
        if (parts[k] > 1) floats += (double)(s.items[k] * parts[k]) * (k == 0 ? 2 : 1) * 128 * 128;
      }
      const double t = bwd_end(sm_count, s.items[0] * parts[0], item[0], s.items[1] * parts[1], item[1]) +
                       (floats > 0.0 ? 3.0 + 8.0 * floats / 12e6 : 0.0);
      if (best == 0.0 || t < best) {
        best = t;
        s.parts[0] = a, s.parts[1] = b;
      }
    }
  }
  return s;
}
}  // namespace

extern "C" B200_API int b200_cross_attn_bwd_workspace_bytes(int64_t batch, int64_t q_len, int64_t kv_len, int64_t heads,
                                                            int64_t kv_heads, size_t* bytes) {
  if (bytes == nullptr) return B200_ERR_INVALID_ARG;
  *bytes = 0;
  int rc = check_heads(batch, q_len, heads, kv_heads, b200::kKvD);
  if (rc != B200_OK) return rc;
  if (kv_len < 0) return B200_ERR_INVALID_ARG;
  if ((rc = check_bwd_size(batch, q_len, kv_len, heads, kv_heads)) != B200_OK) return rc;
  b200::DeviceInfo di;
  if ((rc = b200::device_info(&di)) != B200_OK) return rc;
  *bytes = bwd_bytes(batch, q_len, heads) + plan_bwd(di.sm_count, batch, q_len, kv_len, heads, kv_heads).part_bytes();
  return B200_OK;
}

extern "C" B200_API int b200_cross_attn_bwd_bf16(const b200_attn_view* q, const b200_attn_view* k, const b200_attn_view* v,
                                                 const b200_attn_view* o, const b200_attn_view* dout, const float* lse,
                                                 const int32_t* kv_lens, const b200_attn_view* dq,
                                                 const b200_attn_view* dk, const b200_attn_view* dv, int64_t batch,
                                                 int64_t q_len, int64_t kv_len, int64_t heads, int64_t kv_heads,
                                                 int64_t head_dim, float scale, void* workspace, size_t workspace_bytes,
                                                 void* stream_) {
  int rc = check_heads(batch, q_len, heads, kv_heads, head_dim);
  if (rc != B200_OK) return rc;
  if (kv_len < 0 || !scale_ok(scale)) return B200_ERR_INVALID_ARG;
  const bool queries = q_len > 0 && heads > 0, keys = kv_len > 0 && kv_heads > 0;
  if (batch == 0 || (!queries && !keys)) return B200_OK;
  if ((rc = check_bwd_size(batch, q_len, kv_len, heads, kv_heads)) != B200_OK) return rc;
  const int64_t q_tiles = queries ? (q_len + 127) / 128 : 0, kv_tiles = keys ? (kv_len + 127) / 128 : 0;
  b200_attn_view qq{}, oo{}, dd{}, dqv{}, kk{}, vv{}, dkv{}, dvv{};
  if (queries) {
    if ((rc = check_view(q, batch, q_len, heads, &qq)) != B200_OK || (rc = check_view(o, batch, q_len, heads, &oo)) != B200_OK ||
        (rc = check_view(dout, batch, q_len, heads, &dd)) != B200_OK ||
        (rc = check_view(dq, batch, q_len, heads, &dqv)) != B200_OK)
      return rc;
    if (lse == nullptr) return B200_ERR_INVALID_ARG;
  }
  if (workspace == nullptr || workspace_bytes < bwd_bytes(batch, q_len, heads)) return B200_ERR_INVALID_ARG;
  if (!aligned(workspace, kWsAlign)) return B200_ERR_ALIGNMENT;
  if (keys && ((rc = check_view(k, batch, kv_len, kv_heads, &kk)) != B200_OK ||
               (rc = check_view(v, batch, kv_len, kv_heads, &vv)) != B200_OK ||
               (rc = check_view(dk, batch, kv_len, kv_heads, &dkv)) != B200_OK ||
               (rc = check_view(dv, batch, kv_len, kv_heads, &dvv)) != B200_OK))
    return rc;
  if (!aligned(lse, 4) || !aligned(kv_lens, 4)) return B200_ERR_ALIGNMENT;
  b200::DeviceInfo di;
  StoredState* st = nullptr;
  if ((rc = current_state(&di, &st)) != B200_OK) return rc;
  if (!st->bwd_regs_ok) return B200_ERR_CUDA;  // built with another register count: never launch it
  const BwdShape shape = plan_bwd(di.sm_count, batch, q_len, kv_len, heads, kv_heads);
  const size_t sums = bwd_bytes(batch, q_len, heads);  // where the parts' sums begin
  if (workspace_bytes < sums + shape.part_bytes()) return B200_ERR_INVALID_ARG;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  b200::AttnBwdMaps tm{};
  if (queries && ((rc = encode_view(di, &tm.q, qq, batch, q_len, heads, 128, true)) != B200_OK ||
                  (rc = encode_view(di, &tm.dout, dd, batch, q_len, heads, 128, true)) != B200_OK))
    return rc;
  if (keys && ((rc = encode_view(di, &tm.k, kk, batch, kv_len, kv_heads, 128, true)) != B200_OK ||
               (rc = encode_view(di, &tm.v, vv, batch, kv_len, kv_heads, 128, true)) != B200_OK))
    return rc;
  // A side that is empty has no map of its own and is not read.
  if (!queries) tm.q = tm.dout = tm.k;
  if (!keys) tm.k = tm.v = tm.q;
  b200::AttnBwdParams p{};
  p.q_len = (int32_t)q_len;
  p.kv_len = (int32_t)(keys ? kv_len : 0);
  p.heads = (int32_t)heads;
  p.kv_heads = (int32_t)kv_heads;
  p.group = (int32_t)(kv_heads > 0 ? heads / kv_heads : 0);
  p.batch = (int32_t)batch;
  p.q_tiles = (int32_t)q_tiles;
  p.kv_tiles = (int32_t)kv_tiles;
  p.kv_lens = kv_lens;
  p.scale = scale;
  p.scale_log2 = kLog2e * scale;
  p.timeout_ns = di.timeout_ns;
  p.status = di.status;
  auto grad = [](const b200_attn_view& g) {
    return b200::AttnGrad{static_cast<__nv_bfloat16*>(g.data), g.batch_stride, g.seq_stride, g.head_stride};
  };
  p.dq = grad(dqv), p.dk = grad(dkv), p.dv = grad(dvv);
  uint32_t* counters = static_cast<uint32_t*>(workspace);
  b200::AttnBwdDeltaParams d{};
  d.o = static_cast<const __nv_bfloat16*>(oo.data);
  d.o_batch = oo.batch_stride, d.o_seq = oo.seq_stride, d.o_head = oo.head_stride;
  d.dout = static_cast<const __nv_bfloat16*>(dd.data);
  d.d_batch = dd.batch_stride, d.d_seq = dd.seq_stride, d.d_head = dd.head_stride;
  d.lse = lse;
  d.lse2 = reinterpret_cast<float*>(static_cast<char*>(workspace) + kWsAlign);
  d.delta = d.lse2 + (size_t)(batch * heads) * (size_t)(q_tiles * 128);
  d.q_len = p.q_len;
  d.heads = (int32_t)std::max<int64_t>(heads, 1);
  d.padded = (int32_t)(q_tiles * 128);
  d.rows = (int32_t)(batch * heads);
  d.counters = counters;
  p.lse2 = d.lse2;
  p.delta = d.delta;
  const int64_t rows = std::max<int64_t>(batch * heads, 1);
  const dim3 grid((unsigned)std::max<int64_t>(q_tiles * 2, 1), (unsigned)std::min<int64_t>(rows, 65535),
                  (unsigned)((rows + 65534) / 65535));
  if ((rc = launch(b200::attn_bwd_delta_kernel, grid, 256, 0, stream, d)) != B200_OK) return rc;
  float* part[2];
  part[0] = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums);
  part[1] = part[0] + shape.part_floats(0);
  for (int kind = 0; kind < 2; ++kind) {
    const int64_t items = shape.items[kind] * shape.parts[kind];
    if (items == 0) continue;
    p.items = (int32_t)items;
    p.parts = shape.parts[kind];
    p.part = part[kind];
    p.ordered = kv_lens != nullptr && batch > 1 && batch <= 32 && items > di.sm_count ? 1u : 0u;
    p.counter = counters + kind;
    p.early = kind == 1 && shape.items[0] > 0 ? 1u : 0u;
    const dim3 ctas((unsigned)std::min<int64_t>(items, di.sm_count));
    rc = kind == 0 ? launch(b200::attn_bwd_kernel<false>, ctas, b200::kAttnThreads, b200::AttnBwdPlan<false>::kAllocBytes,
                            stream, tm, p)
                   : launch(b200::attn_bwd_kernel<true>, ctas, b200::kAttnThreads, b200::AttnBwdPlan<true>::kAllocBytes,
                            stream, tm, p);
    if (rc != B200_OK) return rc;
  }
  if (shape.part_bytes() == 0) return B200_OK;
  b200::AttnBwdMergeParams m{};
  int blocks[2];
  for (int kind = 0; kind < 2; ++kind) {
    m.part[kind] = part[kind];
    m.parts[kind] = shape.parts[kind];
    m.tiles[kind] = (int32_t)shape.tiles[kind];
    m.heads[kind] = kind == 0 ? p.kv_heads : p.heads;
    blocks[kind] = shape.parts[kind] > 1 ? (int)shape.items[kind] * (kind == 0 ? 2 : 1) * 8 : 0;
  }
  m.blocks = blocks[0];
  m.q_len = p.q_len;
  m.kv_len = p.kv_len;
  m.walk = (int32_t)shape.walk[0];
  m.kv_lens = kv_lens;
  m.dq = p.dq, m.dk = p.dk, m.dv = p.dv;
  m.scale = scale;
  return launch(b200::attn_bwd_merge_kernel, dim3((unsigned)(blocks[0] + blocks[1])), 256, 0, stream, m);
}
