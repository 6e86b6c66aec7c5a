// Rows of activations quantised to 8 bits where they are made (fp8.cuh): RMS norm with the residual's addition, gated activations, and rows as they are.
// All of them are one pass over memory: 16 lanes have a block of 128 entries, 8 each, and find its scale by four exchanges.
#include "fp8.cuh"

namespace pk {
namespace fp8 {

// x += y (rounded when stored), v = x * rsqrt(mean(x^2) + eps) * (offset + w) of the unrounded x, quantised.  A CTA has a row, in registers from its load to its codes.
constexpr int kNormThreads = 256;
constexpr int kNormWidest = kNormThreads * 8 * 8;

template <typename E, int NV, bool VEC>
__global__ void __launch_bounds__(kNormThreads) fp8_add_norm_kernel(const bf16* __restrict__ y, E* __restrict__ x, const bf16* __restrict__ w, float offset,
                                                                    uint8_t* __restrict__ codes, long ld, float* __restrict__ scales, long ld_s, int width, float eps) {
  __shared__ float red[kNormThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t base = (size_t)blockIdx.x * width;
  pdl_wait();
  float v[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * kNormThreads + threadIdx.x) * 8;
    load8<VEC>(x + base + at, width - at, v[j]);
  }
  if (y) {
    float add[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * kNormThreads + threadIdx.x) * 8;
      load8<VEC>(y + base + at, width - at, add[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * kNormThreads + threadIdx.x) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] += add[j][e];
      store8<VEC>(x + base + at, width - at, v[j]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[j][e], v[j][e], ss);
  ss = warp_sum(ss);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < kNormThreads / 32; ++i) ss += red[i];
  const float r = 1.f / sqrtf(ss / (float)width + eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * kNormThreads + threadIdx.x) * 8;
    if (at - (at & 255) >= width) break;  // (a warp at a time: its lanes find a maximum together)
    float g[8];
    load8<VEC>(w + at, width - at, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[j][e] = at + e < width ? v[j][e] * r * (offset + g[e]) : 0.f;  // (an r that is not finite stays inside the row)
    const Scale k = scale_of(max16(max8(v[j])));
    if (at < width) {
      store_codes8(codes + (size_t)blockIdx.x * ld + at, width - at, v[j], k);
      if ((lane & 15) == 0) scales[(size_t)(at / kBlock) * ld_s + blockIdx.x] = k.s;
    }
  }
}

// KIND 0: silu(a) * b, 1: relu(a)^2, 2: relu(a) * b, 3: gelu(a) * b, 4: a, with a = in[t][f], b = in[t][F + f].  16 lanes have a block of a token.
constexpr int kActThreads = 256;

template <int KIND, bool VEC>
__global__ void __launch_bounds__(kActThreads) fp8_act_kernel(const bf16* __restrict__ in, long ld_in, uint8_t* __restrict__ codes, long ld, float* __restrict__ scales,
                                                              long ld_s, int F, int nb, long items) {
  const long item = ((long)blockIdx.x * kActThreads + threadIdx.x) >> 4;
  const long t = item / nb;
  const int b = (int)(item - t * nb), at = b * kBlock + (threadIdx.x & 15) * 8;
  pdl_wait();
  const int n = item < items ? F - at : 0;
  float v[8];
  const bf16* row = in + (size_t)(item < items ? t : 0) * ld_in + at;
  load8<VEC>(row, n, v);
  if constexpr (KIND == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = v[e] < 0.f ? 0.f : v[e];
      v[e] = u * u;
    }
  } else if constexpr (KIND != 4) {
    float u[8];
    load8<VEC>(row + F, n, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gate_act<KIND == 0 ? 0 : KIND - 1>(v[e]) * u[e];
  }
  const Scale k = scale_of(max16(max8(v)));
  if (n > 0) {
    store_codes8(codes + (size_t)t * ld + at, n, v, k);
    if ((threadIdx.x & 15) == 0) scales[(size_t)b * ld_s + t] = k.s;
  }
}

template <typename E, bool VEC>
cudaError_t add_norm(const bf16* y, E* x, const bf16* w, float offset, uint8_t* codes, long ld, float* scales, long ld_s, int width, int tokens, float eps, cudaStream_t st) {
  auto go = [&](auto kern) { return launch(kern, dim3(tokens), dim3(kNormThreads), 0, st, true, y, x, w, offset, codes, ld, scales, ld_s, width, eps); };
  const int nv = (width + kNormThreads * 8 - 1) / (kNormThreads * 8);
  if (nv <= 1) return go(fp8_add_norm_kernel<E, 1, VEC>);
  if (nv <= 2) return go(fp8_add_norm_kernel<E, 2, VEC>);
  if (nv <= 4) return go(fp8_add_norm_kernel<E, 4, VEC>);
  return go(fp8_add_norm_kernel<E, 8, VEC>);
}

template <int KIND>
cudaError_t act(const bf16* in, long ld_in, uint8_t* codes, long ld, float* scales, long ld_s, int F, int tokens, bool vec, cudaStream_t st) {
  const int nb = blocks_of(F);
  const long items = (long)tokens * nb;
  const dim3 grid((unsigned)((items + kActThreads / 16 - 1) / (kActThreads / 16)));
  if (vec) return launch(fp8_act_kernel<KIND, true>, grid, dim3(kActThreads), 0, st, true, in, ld_in, codes, ld, scales, ld_s, F, nb, items);
  return launch(fp8_act_kernel<KIND, false>, grid, dim3(kActThreads), 0, st, true, in, ld_in, codes, ld, scales, ld_s, F, nb, items);
}

}  // namespace fp8
}  // namespace pk

using namespace pk;

extern "C" int pk_fp8_add_norm(const void* y, void* x, int x_f32, const void* w, float offset, void* codes, long ld, float* scales, long ld_s, int width, int tokens,
                               float eps, pk_stream st) {
  if (!x || !w || x == y || width <= 0 || tokens <= 0 || !fp8::codes_ok(codes, ld, width) || !fp8::row_scales_ok(scales, ld_s, tokens)) return -1;
  if (width > fp8::kNormWidest) return -2;
  const bool vec = width % 8 == 0 && fp8::al16(x) && fp8::al16(w) && fp8::al16(y);
  const bf16 *yb = (const bf16*)y, *wb = (const bf16*)w;
  uint8_t* c = (uint8_t*)codes;
  if (x_f32) {
    if (vec) return (int)fp8::add_norm<float, true>(yb, (float*)x, wb, offset, c, ld, scales, ld_s, width, tokens, eps, st);
    return (int)fp8::add_norm<float, false>(yb, (float*)x, wb, offset, c, ld, scales, ld_s, width, tokens, eps, st);
  }
  if (vec) return (int)fp8::add_norm<bf16, true>(yb, (bf16*)x, wb, offset, c, ld, scales, ld_s, width, tokens, eps, st);
  return (int)fp8::add_norm<bf16, false>(yb, (bf16*)x, wb, offset, c, ld, scales, ld_s, width, tokens, eps, st);
}

extern "C" int pk_fp8_act(const void* in, long ld_in, int kind, void* codes, long ld, float* scales, long ld_s, int F, int tokens, pk_stream st) {
  const long need = (kind == 1 || kind == 4 ? 1L : 2L) * F;
  if (!in || kind < 0 || kind >= fp8::kAct || F <= 0 || tokens <= 0 || (ld_in != 0 && ld_in < need) || !fp8::codes_ok(codes, ld, F) ||
      !fp8::row_scales_ok(scales, ld_s, tokens) || codes == in)
    return -1;
  const long from = ld_in ? ld_in : need;
  if (F > 1 << 30 || (long)tokens * fp8::blocks_of(F) > 1L << 34) return -2;  // (the grid's CTAs are counted in 31 bits)
  const bool vec = F % 8 == 0 && from % 8 == 0 && fp8::al16(in);
  auto go = [&](auto f) { return (int)f((const bf16*)in, from, (uint8_t*)codes, ld, scales, ld_s, F, tokens, vec, st); };
  switch (kind) {
    case 0: return go(fp8::act<0>);
    case 1: return go(fp8::act<1>);
    case 2: return go(fp8::act<2>);
    case 3: return go(fp8::act<3>);
    default: return go(fp8::act<4>);
  }
}
