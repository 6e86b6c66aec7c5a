// Weights quantised to 8 bits, a scale for 128 rows x 128 entries (fp8.cuh): a CTA has a block, in registers from its load to its codes: one pass
// over memory, which bounds it.  B200, GPU time of one call in a row of them: 24576 x 4096 50.3 us (302 MB, 6.0 TB/s; a copy reaches 6.54), 1024 x 4096 6.6 (a block a CTA: 256 of them, one wave).
#include "fp8.cuh"

namespace pk {
namespace fp8 {

constexpr int kWThreads = 256, kWRows = kWThreads / 16, kWSteps = kBlock / kWRows;  // 16 lanes a row, 16 rows at a time

template <typename E, bool VEC>
__global__ void __launch_bounds__(kWThreads) fp8_weights_kernel(const E* __restrict__ w, long ld_w, uint8_t* __restrict__ codes, long ld, float* __restrict__ scales, int rows,
                                                                int width, int nb) {
  __shared__ float red[kWThreads / 32];
  const int b = blockIdx.x % nb, at = b * kBlock + first_of<VEC>(threadIdx.x & 15);
  const long r0 = (long)(blockIdx.x / nb) * kBlock + (threadIdx.x >> 4);
  pdl_wait();
  float v[kWSteps][8];
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < kWSteps; ++j) {
    const long r = r0 + j * kWRows;
    load8<VEC>(w + (size_t)(r < rows ? r : 0) * ld_w + at, r < rows ? width - at : 0, v[j]);
  }
#pragma unroll
  for (int j = 0; j < kWSteps; ++j) m = max_abs(m, max8(v[j]));
  m = max16(m);
  m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, 16));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWThreads / 32; ++i) m = max_abs(m, red[i]);
  const Scale k = scale_of(m);
#pragma unroll
  for (int j = 0; j < kWSteps; ++j) {
    const long r = r0 + j * kWRows;
    if (r < rows && at < width) store_codes8<VEC>(codes + (size_t)r * ld + at, width - at, v[j], k);
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = k.s;
}

template <typename E>
cudaError_t weights(const E* w, long ld_w, uint8_t* codes, long ld, float* scales, int rows, int width, cudaStream_t st) {
  const int nb = blocks_of(width);
  const dim3 grid((unsigned)((long)nb * blocks_of(rows)));
  const bool vec = width % 8 == 0 && ld_w * (long)sizeof(E) % 16 == 0 && al16(w);
  if (vec) return launch(fp8_weights_kernel<E, true>, grid, dim3(kWThreads), 0, st, true, w, ld_w, codes, ld, scales, rows, width, nb);
  return launch(fp8_weights_kernel<E, false>, grid, dim3(kWThreads), 0, st, true, w, ld_w, codes, ld, scales, rows, width, nb);
}

}  // namespace fp8
}  // namespace pk

using namespace pk;

extern "C" int pk_fp8_weights(const void* w, int w_f32, long ld_w, void* codes, long ld, float* scales, int rows, int width, pk_stream st) {
  if (!w || !scales || rows <= 0 || width <= 0 || (ld_w != 0 && ld_w < width) || !fp8::codes_ok(codes, ld, width) || codes == w) return -1;
  if (width > 1 << 30 || (long)fp8::blocks_of(rows) * fp8::blocks_of(width) > 0x7fffffffL) return -2;  // (a CTA a block)
  const long from = ld_w ? ld_w : width;
  if (w_f32) return (int)fp8::weights((const float*)w, from, (uint8_t*)codes, ld, scales, rows, width, st);
  return (int)fp8::weights((const bf16*)w, from, (uint8_t*)codes, ld, scales, rows, width, st);
}
