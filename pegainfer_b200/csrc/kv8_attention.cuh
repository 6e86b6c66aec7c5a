// Attention over the 8-bit paged cache: what its kernels share.
#pragma once

#include <climits>

#include "kv8.cuh"

namespace pk {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  Pool pool;
  const int *slots, *req;
  int T, H;
  float scale, cap;
  int window, max_kv_len;
  long out_ld;        // elements from one row of the output to the next
  float* lse;         // [T, H] or null
  float* mass;        // [requests, G, mass_ld] or null
  long mass_ld;
  float* part_o;      // [shares, T, H, vdim]  states of the shares of a row's keys
  float2* part_ml;    // [shares, T, H]        largest score (log2), sum
};

// q . k -> score in units of log2; c = scale * log2(e)
__device__ __forceinline__ float shaped(float dot, float c, float cap) {
  return cap > 0.f ? cap * kLog2e * tanhf(dot * c / (cap * kLog2e)) : dot * c;
}

// at most 80, and NaN where x is
__device__ __forceinline__ float at_most80(float x) { return x > 80.f ? 80.f : x; }

// Largest score M (log2), sum of 2^(s - M): what the row's accumulated values are multiplied with, and its lse.  A row that saw nothing gives zeros.
struct RowEnd {
  float factor, lse;
};
__device__ __forceinline__ RowEnd row_end(float M, float den, float sink, bool has_sink) {
  RowEnd r;
  float top = M, f = 1.f;
  if (has_sink) {
    const float sk = sink * kLog2e;
    top = fmaxf(M, sk);
    f = M == -INFINITY ? 0.f : exp2f(M - top);
    den = den * f + exp2f(sk - top);
  }
  const bool none = top == -INFINITY;  // neither key nor sink
  r.factor = M == -INFINITY ? 0.f : f / den;
  r.lse = none ? -INFINITY : (top + log2f(den)) * kLn2;
  return r;
}

// ---- products in f16 (mma.sync): codes widened, exactly
constexpr int kTopQ = 14, kTopP = 15;  // exponents of the largest entry of a row of q, and of P = 1, in f16
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four codes -> two pairs of f16
__device__ __forceinline__ void widen(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// records of a warp's run (kv8_few.cu), an even number: `total` records over `warps` warps
__host__ __device__ inline int few_run(long total, int warps) { return max(2, (int)(((total + warps - 1) / warps + 1) / 2 * 2)); }
// kv8_few.cu: whether it takes a call, what it needs (bytes), the call itself (with the weights' sums)
struct FewNeed {
  size_t o, ml, plan, scores;
  long scores_ld;
  size_t bytes() const { return o + ml + plan + scores; }
};
bool few_takes(int T, int H, int G, int dim, int vdim, int max_kv_len, int max_q_len);
FewNeed few_need(int T, int H, int G, int dim, int max_kv_len, bool mass);
int few_attention(const bf16* q, const bf16* sink, bf16* out, const AttnArgs& a, int max_q_len, const FewNeed& need, uint8_t* ws, cudaStream_t st);

// kv8_prompt.cu: whether it takes a call, the shares that it cuts the keys into (more than one: states to part_o, part_ml, for kv8_merge_kernel), and the call
bool prompt_takes(int T, int H, int G, int dim, int vdim);
int prompt_shares(int T, int H, int G, int max_kv_len, int window);
int prompt_attention(const bf16* q, const bf16* sink, bf16* out, const AttnArgs& a, int shares, cudaStream_t st);
// kv8_tile.cu: the same for any sizes and types
bool tile_takes(int T, int H, int G, int max_q_len);
int tile_shares(int T, int H, int G, int max_kv_len, int window);
template <typename E>
int tile_attention(const E* q, const E* sink, E* out, const AttnArgs& a, int shares, cudaStream_t st);
// kv8_mass.cu: the weights' sums of such calls
template <typename E>
int mass_rows(const E* q, const AttnArgs& a, int max_q_len, cudaStream_t st);

}  // namespace kv8
}  // namespace pk
