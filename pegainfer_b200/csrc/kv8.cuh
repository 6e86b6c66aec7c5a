// The 8-bit paged K/V cache: what its kernels share.
//
// 16 consecutive tokens of one kv head are a record: e4m3 codes and two exponents, a value is code * 2^exponent.
//   K      [2 groups of 8 tokens][dim / 16][8 tokens][16 entries]
//   V      [vdim][16 tokens]
//   tail   16 bytes: int8 exponent of K, int8 exponent of V, zeros
// A page is [kv heads][page_size / 16] records.  K's pieces of 8 tokens x 16 entries and V's of 8 entries x 16 tokens are 128 consecutive bytes each: the
// 8 x 16-byte matrices that ldmatrix takes without bank conflicts, with a product's inner dimension inside the 16 bytes both for q K^T (entries) and for P V
// (tokens), so no kernel that multiplies has to turn bytes around.
//
// The exponent is the least e with (largest magnitude) <= 448 * 2^e.  A power of two costs a floating code nothing but its subnormal end, the quotient by it is
// exact, so a value is rounded once, to nearest even, and codes move to a larger exponent by another rounding only below 2^-6.
// A token with an entry of K or V that is not finite has K codes NaN and, where V has it, V codes zero, and takes no part in the exponent: whoever sees the token gets
// NaN, and nobody else (a NaN among V's codes would reach every row of a product, since 0 * NaN is NaN).
#pragma once

#include <cuda_fp16.h>

#include "typed.cuh"

namespace pk {
namespace kv8 {

constexpr int kBlock = 16;           // tokens of a record
constexpr int kMaxSlots = 1 << 30;   // of a request
constexpr int kLowExp = -110, kHighExp = 120;

__host__ __device__ inline int record_bytes(int dim, int vdim) { return kBlock * (dim + vdim) + 16; }
__host__ inline bool sizes_ok(int page_size, int kv_heads, int dim, int vdim) {
  return page_size > 0 && page_size % kBlock == 0 && kv_heads > 0 && dim > 0 && vdim > 0 && dim % 32 == 0 && vdim % 32 == 0 && dim <= 256 && vdim <= 256;
}
__host__ inline bool pool_ok(const void* cache, long page_stride, int page_size, int kv_heads, int dim, int vdim) {
  return (reinterpret_cast<uintptr_t>(cache) & 15) == 0 && page_stride % 16 == 0 &&
         page_stride >= (long)kv_heads * (page_size / kBlock) * record_bytes(dim, vdim);
}

// a pool of pages with a page table per request
struct Pool {
  uint8_t* data;
  long page_stride;
  const int* page_off;
  const int* pages;
  int page_size, G, dim, vdim;
  // the record with the request's token `slot` of kv head g
  __device__ __forceinline__ uint8_t* record(int req, int slot, int g) const {
    return data + (size_t)pages[page_off[req] + slot / page_size] * page_stride +
           (size_t)(g * (page_size / kBlock) + slot % page_size / kBlock) * record_bytes(dim, vdim);
  }
};
inline Pool make_pool(const void* cache, long page_stride, const int* page_off, const int* pages, int page_size, int G, int dim, int vdim) {
  return Pool{static_cast<uint8_t*>(const_cast<void*>(cache)), page_stride, page_off, pages, page_size, G, dim, vdim};
}

// behind a kernel of the same call: its launch may always overlap that one's end
template <typename... KArgs, typename... Args>
static cudaError_t follow(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t st, Args... args) {
  ThreadState& ts = tls();
  const bool pdl = ts.pdl;
  ts.pdl = true;
  const cudaError_t e = launch(kernel, grid, block, 0, st, true, args...);
  ts.pdl = pdl;
  return e;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// the least e with amax <= 448 * 2^e (448 = 1.75 * 2^8)
__device__ __forceinline__ int exponent_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kLowExp), kHighExp);
}
// two values -> two codes (the first in the low byte), to nearest even, at most 448
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) { return codes2(a, b) | codes2(c, d) << 16; }
// two codes -> their values
__device__ __forceinline__ float2 values2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void values4(uint32_t four, float (&v)[4]) {
  const float2 a = values2(four & 0xffffu), b = values2(four >> 16);
  v[0] = a.x;
  v[1] = a.y;
  v[2] = b.x;
  v[3] = b.y;
}
__device__ __forceinline__ void values16(const uint4& c, float (&v)[16]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
    values4(w[i], x);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * i + j] = x[j];
  }
}

// ---- a record out of 16 rows of fp32 in shared memory, by one warp.  Rows lie `row_ld(width)` floats apart: a multiple of four that turns 8 rows' 16-byte
// pieces to 8 different groups of banks.
__host__ __device__ inline int row_ld(int width) { return width + 4; }

// largest magnitude of the rows whose bit is set
__device__ __forceinline__ float rows_amax(const float* rows, int width, uint32_t which, int lane) {
  float a = 0.f;
  for (int r = 0; r < kBlock; ++r)
    if (which >> r & 1)
      for (int d = lane * 4; d < width; d += 128) {
        const float4 v = *reinterpret_cast<const float4*>(rows + r * row_ld(width) + d);
        a = fmaxf(fmaxf(a, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
      }
  return warp_max(a);
}
// K codes; rows in `bad` become NaN
__device__ __forceinline__ void emit_k(uint8_t* rec, const float* rows, int dim, int e, uint32_t bad, int lane) {
  const float f = pow2(-e);
  for (int u = lane; u < dim; u += 32) {  // unit: 16 entries of a token
    const int tok = (u >= dim / 2 ? 8 : 0) + (u & 7), c = (u % (dim / 2)) >> 3;
    const float4* x = reinterpret_cast<const float4*>(rows + tok * row_ld(dim) + c * 16);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = x[i];
      w[i] = bad >> tok & 1 ? 0x7f7f7f7fu : codes4(v.x * f, v.y * f, v.z * f, v.w * f);
    }
    *reinterpret_cast<uint4*>(rec + u * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// V codes; rows in `bad` become zero
__device__ __forceinline__ void emit_v(uint8_t* dst, const float* rows, int vdim, int e, uint32_t bad, int lane) {
  const float f = pow2(-e);
  for (int d = lane; d < vdim; d += 32) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = bad >> (4 * i + j) & 1 ? 0.f : rows[(4 * i + j) * row_ld(vdim) + d] * f;
      w[i] = codes4(v[0], v[1], v[2], v[3]);
    }
    *reinterpret_cast<uint4*>(dst + d * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void emit_tail(uint8_t* tail, int ek, int ev) {
  *reinterpret_cast<uint4*>(tail) = make_uint4((uint32_t)(ek & 255) | (uint32_t)(ev & 255) << 8, 0, 0, 0);
}
__device__ __forceinline__ int tail_ek(uint32_t tail) { return (int)(int8_t)(tail & 255); }
__device__ __forceinline__ int tail_ev(uint32_t tail) { return (int)(int8_t)(tail >> 8 & 255); }

}  // namespace kv8
}  // namespace pk
