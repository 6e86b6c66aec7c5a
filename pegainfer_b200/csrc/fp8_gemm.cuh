// Products of 8-bit rows and weights (fp8.cuh): what fp8_gemm.cu and fp8_gemm_few.cu share.
//
//   y[t][m] = sum over blocks b of  sx[b][t] * sw[m / 128][b] * (sum over the 128 entries k of block b of  x[t][k] * w[m][k])
//
// The inner sum is a tcgen05.mma of kind f8f6f4 into tensor memory (products of codes are exact, sums fp32); it is then multiplied by its two scales and added to an fp32 sum in
// registers, so scales may be any numbers, as checkpoints have them.
#pragma once

#include <cuda.h>

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace pk {
namespace fp8 {

constexpr int kBK = 128;  // entries of K to a stage: a block of the scales, and a 128-byte span of the swizzle

struct Product {
  const uint8_t *w, *w2;    // codes of the weights [M][ld_w]; w2: the second matrix of a gated product
  const float *sw, *sw2;    // their scales [blocks of M][kb]
  const uint8_t* x;         // codes of the rows [N][ld_x]
  const float* sx;          // their scales [kb][ld_sx]
  long ld_w, ld_x, ld_sx;
  void* y;                  // [N][ld_y], bf16 or float
  long ld_y;
  bool y_map;               // fp8_gemm.cu: the output goes by tensor map
  uint8_t* codes;           // gated: the activated rows [N][ld], their scales [blocks of M][ld_s]
  float* scales;
  long ld, ld_s;
  int M, N, K, kb;          // features, tokens, reduction, its blocks
  int tiles;                // fp8_gemm.cu: of 256 tokens
  int act;                  // gated: 0 SiLU, 1 ReLU, 2 GELU
  unsigned int* err;        // wait_err_word()
};

// D = f32, A = B = e4m3, both K-major
constexpr uint32_t f8_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// the wait names the registers it makes valid, so that no use of them can be moved in front of it
__device__ __forceinline__ void tmem_wait32(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                 "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait16(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
        "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}

// rows x K codes, rows of ld bytes; boxes of box_rows x 128 bytes, 128-byte swizzle; what lies outside reads as zero
inline bool make_codes_map(CUtensorMap* map, const void* base, long rows, int K, long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// fp8_gemm_few.cu; -2: not one of its sizes, or it takes longer than within_ns
int launch_few(const Product& p, bool gated, bool y_f32, double within_ns, cudaStream_t st);

}  // namespace fp8
}  // namespace pk
