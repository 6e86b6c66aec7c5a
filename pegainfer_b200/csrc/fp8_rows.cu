// Rows of activations quantised to 8 bits where they are made (fp8.cuh): RMS norm with the residual's addition, gated activations, and rows as they are.
// All of them are one pass over memory: 16 lanes have a block of 128 entries, 8 each, and find its scale by four exchanges.
// B200, GPU time of one call in a row of them, us: norm of 4096 x 4096 with float x 30.2 (185 MB, 6.1 TB/s), with bf16 x 23.7 (5.0 TB/s), of 8 x 2560 2.3; of 4096 x 12288 silu product 42.7
// (253 MB, 5.9 TB/s), gelu 44.8, relu product 39.4, relu^2 30.9 (153 MB, 4.9 TB/s), plain rows 26.9; silu product of 32 x 9728 2.1.  Memory bounds the large ones (a copy reaches 6.54 TB/s),
// the launch the small ones.
#include "fp8.cuh"

namespace pk {
namespace fp8 {

// x += y (rounded when stored), v = x * rsqrt(mean(x^2) + eps) * (offset + w) of the unrounded x, quantised.  A CTA has a row, in registers from its load to its codes, NV pieces of 8
// entries a thread and as many warps as that takes.
// A code is v over its block's largest v, in which the root cancels: codes come from x * (offset + w), with two roundings less, and only the scales wait for the row's sum.  A block whose
// largest such product has no scale of its own (below 2^-100, the root may bring it above; or past fp32, the root may bring it back) keeps x instead, and its codes wait for the root.
constexpr int kNormWarps = 32, kNormWidest = kNormWarps * 256 * 2;

// Registers: with 40 two pieces have six CTAs of eight warps on an SM (4096 x 4096 bf16 23.7 us; with the 52 that the compiler takes by itself 27.8).
template <typename E, int NV, bool VEC>
__global__ void __maxnreg__(NV == 2 ? (VEC ? 40 : 56) : 32) fp8_add_norm_kernel(const bf16* __restrict__ y, E* __restrict__ x, const bf16* __restrict__ w, float offset,
                                                                      uint8_t* __restrict__ codes, long ld, float* __restrict__ scales, long ld_s, int width, float eps) {
  __shared__ float red[kNormWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const size_t t = blockIdx.x, base = t * width;
  pdl_wait();
  float v[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = first_of<VEC>(j * blockDim.x + threadIdx.x);
    load8<VEC>(x + base + at, width - at, v[j]);
  }
  if (y) {
    float add[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = first_of<VEC>(j * blockDim.x + threadIdx.x);
      load8<VEC>(y + base + at, width - at, add[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = first_of<VEC>(j * blockDim.x + threadIdx.x);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t sum = add2(pair_of(v[j][e], v[j][e + 1]), pair_of(add[j][e], add[j][e + 1]));
        v[j][e] = lo_of(sum);
        v[j][e + 1] = hi_of(sum);
      }
      store8<VEC>(x + base + at, width - at, v[j]);
    }
  }
  uint64_t squares = 0;
  float m[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = first_of<VEC>(j * blockDim.x + threadIdx.x);
    float g[8], times[8];
    load8<VEC>(w + at, width - at, g);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {  // (behind the width both are zero)
      const uint64_t u = pair_of(v[j][e], v[j][e + 1]), p = mul2(u, add2(pair_of(offset, offset), pair_of(g[e], g[e + 1])));
      squares = fma2(u, u, squares);
      times[e] = lo_of(p);
      times[e + 1] = hi_of(p);
    }
    m[j] = max16(max8(times));
    if (in_range(m[j])) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = times[e];
    }
  }
  float ss = warp_sum(lo_of(squares) + hi_of(squares));
  if (warps > 1) {
    if (lane == 0) red[warp] = ss;
    __syncthreads();
    ss = warp_sum(lane < warps ? red[lane] : 0.f);
  }
  const float r = 1.f / sqrtf(ss / (float)width + eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = first_of<VEC>(j * blockDim.x + threadIdx.x);
    Scale k = scale_of(m[j] * r), from = scale_of(m[j]);
    if (const bool kept = !in_range(m[j]); kept || !(m[j] * r > kLeast)) {  // (the block's 16 lanes are of one mind)
      if (kept) {
        float g[8];
        load8<VEC>(w + at, width - at, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = v[j][e] * r * (offset + g[e]);
        k = scale_of(max16(max8(v[j]), 0xffffu << (lane & 16)));
      } else {  // the least scale
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= r;
      }
      from = k;
    }
    if (at < width) {
      store_codes8<VEC>(codes + t * ld + at, width - at, v[j], from);
      if ((lane & 15) == 0) scales[(size_t)(at / kBlock) * ld_s + t] = k.s;
    }
  }
}

// Two tokens a group of lanes: their loads are under way together, which carries this kernel (silu product of 4096 x 12288, one token : two, when this was tried: 59 : 44.8 us).
// KIND 0: silu(a) * b, 1: relu(a)^2, 2: relu(a) * b, 3: gelu(a) * b, 4: a, with a = in[t][f], b = in[t][F + f].  16 lanes have a block of a token.
constexpr int kActThreads = 128, kActRows = 2;

template <int KIND, bool VEC>
__global__ void __launch_bounds__(kActThreads) fp8_act_kernel(const bf16* __restrict__ in, long ld_in, uint8_t* __restrict__ codes, long ld, float* __restrict__ scales,
                                                              long ld_s, int F, int nb, long items, int tokens) {
  const long item = ((long)blockIdx.x * kActThreads + threadIdx.x) >> 4;
  const long group = item / nb;
  const int b = (int)(item - group * nb), at = b * kBlock + first_of<VEC>(threadIdx.x & 15), t0 = (int)(group * kActRows);
  pdl_wait();
  float v[kActRows][8], u[kActRows][8];
#pragma unroll
  for (int r = 0; r < kActRows; ++r) {
    const int n = item < items && t0 + r < tokens ? F - at : 0;
    const bf16* row = in + (size_t)(n > 0 ? t0 + r : 0) * ld_in + at;
    load8<VEC>(row, n, v[r]);
    if constexpr (KIND != 1 && KIND != 4) load8<VEC>(row + F, n, u[r]);
  }
#pragma unroll
  for (int r = 0; r < kActRows; ++r) {
    const int n = item < items && t0 + r < tokens ? F - at : 0;
    if constexpr (KIND == 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = v[r][e] < 0.f ? 0.f : v[r][e];
        v[r][e] = z * z;
      }
    } else if constexpr (KIND != 4) {
      constexpr int ACT = KIND == 0 ? 0 : KIND - 1;
      if (__builtin_expect(gated8<ACT>(v[r], u[r], v[r]), 0)) {  // (read again, one by one: kept until here, gates and factors took twice the registers: 46.4 us for 42.3)
        const bf16* row = in + (size_t)(n > 0 ? t0 + r : 0) * ld_in + at;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = VEC ? e : 16 * e;
          const float z = load_if(row + i, i < n);
          if (z < far_below(ACT)) v[r][e] = far_gated(z, gate_exponent<ACT>(z), load_if(row + F + i, i < n));
        }
      }
    }
    const Scale k = scale_of(max16(max8(v[r])));
    if (n > 0) {
      store_codes8<VEC>(codes + (size_t)(t0 + r) * ld + at, n, v[r], k);
      if ((threadIdx.x & 15) == 0) scales[(size_t)b * ld_s + t0 + r] = k.s;
    }
  }
}

template <typename E, bool VEC>
cudaError_t add_norm(const bf16* y, E* x, const bf16* w, float offset, uint8_t* codes, long ld, float* scales, long ld_s, int width, int tokens, float eps, cudaStream_t st) {
  auto go = [&](auto kern, int nv) {
    const int warps = (width + 256 * nv - 1) / (256 * nv);
    return launch(kern, dim3(tokens), dim3(32 * warps), 0, st, true, y, x, w, offset, codes, ld, scales, ld_s, width, eps);
  };
  // B200, us, one piece a thread : two, x bf16: 8 x 2560 2.3 : 2.7, 512 x 2560 3.7 : 3.9, 800 x 2560 5.0 : 5.2, 1024 x 2560 7.1 : 6.2, 3001 x 2560 14.0 : 13.2,
  // 4096 x 4096 26.5 : 24.1; x float: 512 x 2560 4.8 : 5.2, 3001 x 2560 15.6 : 16.8, 4096 x 4096 30.6 : 31.6, 2048 x 8192 32.6 : 32.2
  if (width <= kNormWarps * 256 && (sizeof(E) == 4 || tokens < 5 * sm_count())) return go(fp8_add_norm_kernel<E, 1, VEC>, 1);
  return go(fp8_add_norm_kernel<E, 2, VEC>, 2);
}

template <int KIND>
cudaError_t act(const bf16* in, long ld_in, uint8_t* codes, long ld, float* scales, long ld_s, int F, int tokens, bool vec, cudaStream_t st) {
  const int nb = blocks_of(F);
  const long items = ((long)tokens + kActRows - 1) / kActRows * nb;
  const dim3 grid((unsigned)((items + kActThreads / 16 - 1) / (kActThreads / 16)));
  if (vec) return launch(fp8_act_kernel<KIND, true>, grid, dim3(kActThreads), 0, st, true, in, ld_in, codes, ld, scales, ld_s, F, nb, items, tokens);
  return launch(fp8_act_kernel<KIND, false>, grid, dim3(kActThreads), 0, st, true, in, ld_in, codes, ld, scales, ld_s, F, nb, items, tokens);
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
