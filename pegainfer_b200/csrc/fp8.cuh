// Linear layers in 8 bits: what their kernels share.
//
// A value is its e4m3 code times its block's scale.  Rows of activations have a scale for 128 consecutive entries, weights one for 128 rows x 128 entries:
//   s = max(largest magnitude of the block, 2^-100) / 448,  code = the e4m3 number nearest to v / s (ties to even)
// so a block's largest entry has the code 448 and an entry is off by at most 2^-4 of itself, or by 2^-10 s below 2^-6 s.  The floor of 2^-100 keeps 1 / s finite; a block of
// zeros has codes of zero.  A block with an entry that is not finite has the scale NaN and codes NaN: the products that read it give NaN, and no others do.
#pragma once

#include "typed.cuh"

namespace pk {
namespace fp8 {

constexpr int kBlock = 128;
constexpr float kLeast = 7.888609e-31f;  // 2^-100
constexpr int kAct = 5;  // kinds of pk_fp8_act

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
__host__ __device__ inline int blocks_of(int n) { return (int)(((long)n + kBlock - 1) / kBlock); }
// codes [rows][ld] and their scales as every entry point takes them
inline bool codes_ok(const void* codes, long ld, int width) { return codes && al16(codes) && ld % 16 == 0 && ld >= width && ld < 1L << 39; }
inline bool row_scales_ok(const float* scales, long ld_s, int tokens) { return scales && al16(scales) && ld_s % 4 == 0 && ld_s >= tokens; }

// two fp32 numbers to an instruction
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// by the special-function unit (2^-22); results below 2^-126 are zero
__device__ __forceinline__ float rcp_ftz(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_ftz(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_any(float v) {  // (those below 2^-126 too)
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// the largest magnitude; infinities and NaN stay
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
__device__ __forceinline__ float max8(const float* v) {
  return max_abs(max_abs(v[0], v[1], v[2]), max_abs(v[3], v[4], v[5]), max_abs(v[6], v[7]));
}
// the largest of 16 lanes, which have a block together; lanes: those that are here
__device__ __forceinline__ float max16(float m, uint32_t lanes = 0xffffffffu) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max_abs(m, __shfl_xor_sync(lanes, m, o));
  return m;
}
// a block's largest magnitude that gives a scale without the floor
__device__ __forceinline__ bool in_range(float amax) { return amax >= kLeast && amax < INFINITY; }

struct Scale {
  float s, inv;  // NaN where the block has an entry that is not finite
};
// amax / 448 to its nearest fp32 number: a product and a step of Newton's, whose remainder is exact
__device__ __forceinline__ Scale scale_of(float amax) {
  constexpr float kTo = 1.f / 448.f;
  const float a = amax < kLeast ? kLeast : amax - (amax - amax);  // (an infinity becomes NaN)
  const float s = a * kTo;
  Scale r;
  r.s = fmaf(fmaf(-s, 448.f, a), kTo, s);
  r.inv = rcp_ftz(r.s);  // (2^-109 to 2^120)
  return r;
}
// codes of v / s, each quotient to its nearest fp32 number: v * (1 / s) and the same step, whose remainder v - q s is exact.  Without it a quotient that lies just between two codes,
// as bf16 entries have them often, went to either.
__device__ __forceinline__ uint32_t codes2(float lo, float hi, Scale k) {
  const uint64_t v = pair_of(lo, hi), inv = pair_of(k.inv, k.inv), s = pair_of(-k.s, -k.s);
  uint64_t q = mul2(v, inv);
  q = fma2(fma2(q, s, v), inv, q);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi_of(q)), "f"(lo_of(q)));
  return r;
}
__device__ __forceinline__ uint32_t codes4(const float* v, Scale k) { return codes2(v[0], v[1], k) | codes2(v[2], v[3], k) << 16; }

// A thread has 8 entries of a block, 16 threads a block.  VEC: 8 in a row, read at once, for rows on 16-byte boundaries whose widths are multiples of 8.  Else every 16th, read one by one, so
// that the threads' single entries lie side by side (B200, norm of 1328 x 2958, us, 8 in a row : every 16th: float 18.9 : 11.8, bf16 18.9 : 11.3; read at once, 1328 x 2960: float 10.1).
// of the q-th thread of a row: its first entry
template <bool VEC>
__device__ __forceinline__ int first_of(int q) { return VEC ? q * 8 : (q >> 4) * kBlock + (q & 15); }

// An entry if there is one, else zero, without a branch: `there ? *p : 0` of 16 bits had one load at a time under way (weights of 4000 x 2501 57 us, so 13).
__device__ __forceinline__ float load_if(const bf16* p, bool there) {
  uint16_t v;
  asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\nmov.u16 %0, 0;\n@q ld.global.u16 %0, [%1];\n}" : "=h"(v) : "l"(p), "r"((uint32_t)there));
  return __uint_as_float((uint32_t)v << 16);
}
__device__ __forceinline__ float load_if(const float* p, bool there) {
  uint32_t v;
  asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\nmov.u32 %0, 0;\n@q ld.global.u32 %0, [%1];\n}" : "=r"(v) : "l"(p), "r"((uint32_t)there));
  return __uint_as_float(v);
}

// the entries from p on, of which n are left in the row (the others are zero)
template <bool VEC>
__device__ __forceinline__ void load8(const bf16* p, int n, float* v) {
  if constexpr (VEC) {
    const uint4 a = n > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = bf16_lo(u[e]);
      v[2 * e + 1] = bf16_hi(u[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = load_if(p + 16 * e, 16 * e < n);
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int n, float* v) {
  if constexpr (VEC) {
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 a = n > 0 ? reinterpret_cast<const float4*>(p)[0] : none, b = n > 0 ? reinterpret_cast<const float4*>(p)[1] : none;
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = load_if(p + 16 * e, 16 * e < n);
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(bf16* p, int n, const float* v) {
  if constexpr (VEC) {
    if (n > 0) *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (16 * e < n) p[16 * e] = f2bf(v[e]);
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* p, int n, const float* v) {
  if constexpr (VEC) {
    if (n > 0) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (16 * e < n) p[16 * e] = v[e];
  }
}
template <bool VEC>
__device__ __forceinline__ void store_codes8(uint8_t* p, int n, const float* v, Scale k) {
  const uint32_t lo = codes4(v, k), hi = codes4(v + 4, k);
  if constexpr (VEC) {
    if (n > 0) *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (16 * e < n) p[16 * e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
  }
}

// act 0 SiLU, 1 ReLU, 2 GELU in its tanh form, of z, times u.  SiLU and GELU: z times the logistic function of z or of sqrt(8 / pi) (z + 0.044715 z^3), as z / (1 + 2^x) by the
// special-function unit's exponential and quotient without their ways for subnormal numbers, which took half of the instructions.  That loses gates whose 1 + 2^x has no normal reciprocal
// (x from 126 on), and times a large factor they count: they are (z 2^(-x/2)) (2^(-x/2) u).
// What is less exact than fp32's exp and division: the unit's results have 2^-22, and the rounding of x grows with it.  SiLU is within (1.25 |z| + 16) 2^-24 of itself (3e-6 at z = -30, a code's
// own rounding is 6e-2), GELU within (4 |x| ln 2 + 16) 2^-24; x as a sum of two numbers takes more instructions, in a kernel whose issue slots are 0.7 busy.
template <int ACT>
__device__ __forceinline__ float gate_exponent(float z) {
  constexpr float kLog2e = 1.4426950408889634f, kGelu = -1.5957691216057308f * kLog2e;
  return ACT == 2 ? z * fmaf(z * z, 0.044715f * kGelu, kGelu) : z * -kLog2e;
}
__host__ __device__ constexpr float far_below(int act) { return act == 2 ? -9.9f : -84.f; }  // (x = 122.7, 121.2)
__device__ __forceinline__ float far_gated(float z, float x, float u) {
  const float h = exp2_any(-0.5f * x);
  return (z * h) * (h * u);
}
template <int ACT>
__device__ __forceinline__ float near_gated(float z, float u) {
  if constexpr (ACT == 1) return (z < 0.f ? 0.f : z) * u;  // (NaN stays)
  return z * rcp_ftz(1.f + exp2_ftz(gate_exponent<ACT>(z))) * u;
}
// eight gates z with their factors u, to v (which may be z); true: some are far, and their results not in v yet
template <int ACT>
__device__ __forceinline__ bool gated8(const float* z, const float* u, float* v) {
  float least = z[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) least = fminf(least, z[j]);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = near_gated<ACT>(z[j], u[j]);
  return ACT != 1 && least < far_below(ACT);
}
template <int ACT>
__device__ __forceinline__ void far_gated8(const float* z, const float* u, float* v) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (z[j] < far_below(ACT)) v[j] = far_gated(z[j], gate_exponent<ACT>(z[j]), u[j]);
}

}  // namespace fp8
}  // namespace pk
