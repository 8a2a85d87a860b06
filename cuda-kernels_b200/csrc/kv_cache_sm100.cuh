// Writing new keys and values into a paged e4m3 cache (b200_kv_cache_write).
//
// Cache layout: codes [num_pages][kv_heads][page_size][128] e4m3, one scale
// per (page, key/value head), [num_pages][kv_heads] fp32: value = code x scale.
// The scale is the smallest power of two s >= 2^-100 with |x| <= 448 s over
// the page's values.  A power of two makes x / s exact, so a value is rounded
// once, to the nearest e4m3 code (relative error 2^-4 for |x| >= 2^-6 s), and
// a scale that has to grow while a page fills only shifts the exponents of the
// codes already there: code' = rn_e4m3(code x s_old / s_new), exact unless a
// code falls into e4m3's subnormals.  A page whose first slot is written
// starts afresh (whatever scale and codes it held belong to nobody).
//
// One CTA per (sequence, page touched, head, K or V): the rows go to registers
// in one pass over memory (16 bytes a thread), their maximum over the CTA by
// integer maxima of the positive floats' bits, then the codes leave, 8 bytes a
// thread.  2 B read and 1 B written per element; a page is
// never touched by two CTAs, so nothing depends on an order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cstdint>

#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kKvD = 128;             // head dimension
constexpr int kKvWriteThreads = 128;  // 8 rows of 16 threads
constexpr int kKvMinScaleExp = -100;  // smallest scale 2^-100 (a page of zeros)

struct KvWriteParams {
  const __nv_bfloat16* x[2];  // K, V: [batch, new_max, kv_heads, 128], strides in elements
  int64_t x_batch[2], x_seq[2], x_head[2];
  uint8_t* cache[2];
  float* scale[2];
  const int32_t* table;
  int64_t table_stride;
  const int32_t* seq_lens;  // length of each sequence with the new tokens
  const int32_t* new_lens;  // new tokens of each sequence, or NULL: new_max
  int32_t new_max, kv_heads, num_pages, max_pages;
  int32_t pages_touched;  // most pages the new tokens of one sequence reach
  uint32_t* status;
};

__device__ __forceinline__ void kv_bad_index(uint32_t* status) { atomicOr(status, (uint32_t)kDevBadIndex); }

// Smallest power of two >= 2^-100 with amax <= 448 s (448 = 1.75 x 2^8).
__device__ __forceinline__ float kv_scale_of(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, kKvMinScaleExp);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ float2 bf16x2_to_float2(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ uint32_t e4m3x2_of(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// The two e4m3 codes of the low half of `w` as fp16 (exact, NaN included).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(h) : "r"(w));
  return h;
}

template <int kPage>
__global__ void __launch_bounds__(kKvWriteThreads) kv_cache_write_kernel(const __grid_constant__ KvWriteParams p) {
  constexpr int kPasses = kPage / 8;
  __shared__ uint32_t warp_max[kKvWriteThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  uint32_t id = blockIdx.x;
  const int which = (int)(id & 1u);
  id >>= 1;
  const int head = (int)(id % (uint32_t)p.kv_heads);
  id /= (uint32_t)p.kv_heads;
  const int touched = (int)(id % (uint32_t)p.pages_touched);
  const int bat = (int)(id / (uint32_t)p.pages_touched);

  const int len = p.seq_lens[bat];
  const int fresh = p.new_lens != nullptr ? p.new_lens[bat] : p.new_max;
  const int first = len - fresh;  // place of the first new token
  if (len < 0 || fresh < 0 || fresh > p.new_max || first < 0 || len > p.max_pages * kPage) {
    if (threadIdx.x == 0) kv_bad_index(p.status);
    return;
  }
  const int page = first / kPage + touched;
  if (fresh == 0 || page * kPage >= len) return;
  const int lo = max(first - page * kPage, 0), hi = min(len - page * kPage, kPage);  // slots [lo, hi) are new
  const int id_page = p.table[bat * p.table_stride + page];
  if (id_page < 0 || id_page >= p.num_pages) {
    if (threadIdx.x == 0) kv_bad_index(p.status);
    return;
  }
  const int row = (int)threadIdx.x >> 4, col = (int)(threadIdx.x & 15u) * 8;
  const __nv_bfloat16* src = p.x[which] + bat * p.x_batch[which] + head * p.x_head[which] + col;
  const int64_t seq_stride = p.x_seq[which];
  const size_t tile = ((size_t)id_page * p.kv_heads + head) * kPage;
  uint8_t* codes = p.cache[which] + tile * kKvD + col;
  float* scale = p.scale[which] + (size_t)id_page * p.kv_heads + head;

  uint4 x[kPasses];
  __nv_bfloat162 top = __float2bfloat162_rn(0.0f);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int slot = i * 8 + row;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (slot >= lo && slot < hi) {
      x[i] = *reinterpret_cast<const uint4*>(src + (int64_t)(page * kPage + slot - first) * seq_stride);
    }
  }
  const float old = lo > 0 ? *scale : 0.0f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    // __hmax2 passes over NaN: a NaN value takes no part in the scale.
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = w[k] & 0x7fff7fffu;
      top = __hmax2(top, *reinterpret_cast<const __nv_bfloat162*>(&a));
    }
  }
  const float mine = fmaxf(__low2float(top), __high2float(top));
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(mine));
  if ((threadIdx.x & 31u) == 0) warp_max[threadIdx.x >> 5] = bits;
  __syncthreads();  // also: everyone has read the old scale
  bits = max(max(warp_max[0], warp_max[1]), max(warp_max[2], warp_max[3]));
  const float now = fmaxf(old, kv_scale_of(__uint_as_float(bits)));
  if (threadIdx.x == 0) *scale = now;

  if (lo > 0 && now != old) {
    // The scale grew: the codes already in the page are rounded to the new one.
    const float ratio = old / now;
#pragma unroll 1
    for (int slot = row; slot < lo; slot += 8) {
      uint2* at = reinterpret_cast<uint2*>(codes + (size_t)slot * kKvD);
      const uint2 c = *at;
      uint32_t out[2];
      const uint32_t in[2] = {c.x, c.y};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t h0 = e4m3x2_to_f16x2(in[k]), h1 = e4m3x2_hi_to_f16x2(in[k]);
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        out[k] = e4m3x2_of(f0.x * ratio, f0.y * ratio) | (e4m3x2_of(f1.x * ratio, f1.y * ratio) << 16);
      }
      *at = make_uint2(out[0], out[1]);
    }
  }
  // x / s: a multiplication by the exact reciprocal when s is a power of two
  // (always, unless the page was filled with another scale by someone else).
  const bool power = (__float_as_uint(now) & 0x7fffffu) == 0u;
  const float inv = 1.0f / now;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int slot = i * 8 + row;
    if (slot >= lo && slot < hi) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t c[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 f = bf16x2_to_float2(w[k]);
        f = power ? make_float2(f.x * inv, f.y * inv) : make_float2(f.x / now, f.y / now);
        c[k] = e4m3x2_of(f.x, f.y);
      }
      *reinterpret_cast<uint2*>(codes + (size_t)slot * kKvD) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
    }
  }
}

}  // namespace b200
