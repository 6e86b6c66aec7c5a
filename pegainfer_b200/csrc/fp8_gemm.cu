// The product of 8-bit rows and weights for prompts, on CTA pairs (fp8_gemm.cuh): y = x w^T, and act(x w^T) * (x w2^T) quantised again.
//
// A pair (cluster of two, tcgen05 cta_group::2) has a tile of 256 tokens x BN features: A = X, 128 tokens to a CTA, B = W, half the features to a CTA.
//   warp 0  TMA producer (both CTAs): 128 entries of K a stage, completing on the leader's barrier
//   warp 1  MMA issuer (leader): four tcgen05.mma (M 256, N BN, K 32) a block of K into one of two partial sums in tensor memory
//   warps 4-11  take a block's partial sum out of tensor memory while the next one is computed, multiply it by its scales and add it to the tile's sum, which they hold in registers
//           (thread = token, BN / 2 features).  A thread's token has one scale a block, its features one: a multiplication for all, and half an instruction
//           (fma.rn.f32x2) for an entry, 256 of the 512 clocks that the block's MMAs take.
// Gated: B is 128 rows of w (leader) and the same 128 of w2 (peer), so a thread has 64 features of both; 128 features are a block of the result's scales, whose largest magnitude two threads
// find together.
// Every barrier wait is bounded (mbar_wait_bounded, common.cuh).
#include <cuda.h>

#include <algorithm>

#include "fp8_gemm.cuh"

namespace pk {
namespace fp8 {

namespace {

constexpr int kBM = 128;                     // tokens per CTA
constexpr int kEpi = 8;                      // epilogue warps
constexpr int kThreads = 128 + 32 * kEpi;     // warps 0 to 3: TMA, MMA, two without work (registers are given out by four warps)
// registers of a thread: the 65536 of an SM by 384 threads, then by role
constexpr int kRegsLaunch = 168, kRegsOther = 56, kRegsEpi = 224;
static_assert(128 * kRegsOther + 32 * kEpi * kRegsEpi <= kThreads * kRegsLaunch, "what the block was launched with");

__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of a warp's 32 rows; the lanes store for one another, four lanes 64 bytes of a row at a time (a lane that stored its own row would touch a line per 16 bytes)
__device__ __forceinline__ void store32(bf16* base, long ld, int tok, int N, int lane, const uint64_t* acc) {
  uint32_t u[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) u[j] = pack_bf16(lo_of(acc[j]), hi_of(acc[j]));
  transpose4(u, lane);
  const int tok4 = tok & ~3;
  bf16* dst = base + (size_t)tok4 * ld + (lane & 3) * 8;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (tok4 + j < N) *reinterpret_cast<uint4*>(dst + (size_t)j * ld) = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
}
__device__ __forceinline__ void store32(float* base, long ld, int tok, int N, int lane, const uint64_t* acc) {
  if (tok >= N) return;
  float4* dst = reinterpret_cast<float4*>(base + (size_t)tok * ld);
#pragma unroll
  for (int j = 0; j < 8; ++j) dst[j] = make_float4(lo_of(acc[2 * j]), hi_of(acc[2 * j]), lo_of(acc[2 * j + 1]), hi_of(acc[2 * j + 1]));
}

template <int ACT>
__device__ __forceinline__ void activate(uint64_t* acc, float* v) {  // acc: 32 pairs of the gate, 32 of the factor
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[2 * j] = gate_act<ACT>(lo_of(acc[j])) * lo_of(acc[32 + j]);
    v[2 * j + 1] = gate_act<ACT>(hi_of(acc[j])) * hi_of(acc[32 + j]);
  }
}

// GATED: O is the codes' type
template <int BN, int STAGES, bool GATED, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2, const Product p) {
  constexpr int HB = BN / 2;  // B rows staged per CTA; features of a thread
  constexpr int A_BYTES = kBM * kBK, B_BYTES = HB * kBK, STAGE_BYTES = A_BYTES + B_BYTES;
  constexpr int FEATURES = GATED ? HB : BN;  // of a tile
  static_assert(!GATED || BN == 256, "128 features are a block of the result's scales");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)STAGES * STAGE_BYTES);  // used in the leader
  uint64_t* empty = full + STAGES;   // one per CTA (multicast commit)
  uint64_t* tfull = empty + STAGES;  // [2] one per CTA
  uint64_t* tempty = tfull + 2;      // [2] used in the leader (an arrival per epilogue warp of both CTAs)
  uint64_t* done = tempty + 2;       // behind a run-out: the MMAs under way
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* largest = tmem_slot + 2;  // [2][2][128] gated: magnitudes of two tiles' rows, by half
  static_assert((2 * STAGES + 5) * 8 + 8 + 2048 <= 2304, "room behind the stages");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int M = p.M, N = p.N, kb_n = p.kb;
  const int m_tiles = (N + 2 * kBM - 1) / (2 * kBM);
  const int n_tiles = (M + FEATURES - 1) / FEATURES;
  const long num_tiles = (long)m_tiles * n_tiles;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(tfull + s, 1);
      mbar_init(tempty + s, 2 * kEpi);
    }
    mbar_init(done, 1);
    *dead = 0;
    mbar_fence_init();
  }
  if (warp == 1) g2_tmem_alloc(tmem_slot, 2 * BN);
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers are initialised and both TMEM allocations are done
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 0) {
      if (tc_elect_one()) {
        const CUtensorMap* mw = GATED && rank == 1 ? &map_w2 : &map_w;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(mw) : "memory");
        int s = 0;
        uint32_t ph = 1;
        bool go = true;
        for (long tile = pair; tile < num_tiles && go; tile += num_pairs) {
          const int mb = (int)(tile % m_tiles), nb = (int)(tile / m_tiles);
          const int tok0 = mb * 2 * kBM + (int)rank * kBM;
          const int row0 = GATED ? nb * HB : nb * BN + (int)rank * HB;
          for (int kb = 0; kb < kb_n; ++kb) {
            go = mbar_wait_bounded(empty + s, ph, dead);
            if (!go) break;
            const uint32_t fb = g2_map(smem_u32(full + s), 0);
            if (leader) mbar_expect_tx(full + s, 2 * STAGE_BYTES);
            uint8_t* st = smem + (size_t)s * STAGE_BYTES;
            g2_tma_2d(st, &map_x, kb * kBK, tok0, fb);
            g2_tma_2d(st + A_BYTES, mw, kb * kBK, row0, fb);
            if (++s == STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
        }
        if (!go) wait_for_copies();  // (some complete on the leader's barriers)
      }
    } else if (warp == 1) {
      if (leader && tc_elect_one()) {
        constexpr uint32_t idesc = f8_idesc(2 * kBM, BN);
        int s = 0, buf = 0;
        uint32_t ph = 0, tph = 1;
        bool go = true;
        for (long tile = pair; tile < num_tiles && go; tile += num_pairs) {
          for (int kb = 0; kb < kb_n; ++kb) {
            go = mbar_wait_bounded(tempty + buf, tph, dead) && mbar_wait_bounded(full + s, ph, dead);
            if (!go) break;
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + (size_t)s * STAGE_BYTES);
            const uint64_t adesc = make_sw128_desc(a_addr), bdesc = make_sw128_desc(a_addr + A_BYTES);
            const uint32_t d = tmem_base + (uint32_t)(buf * BN);
  #pragma unroll
            for (int k = 0; k < kBK / 32; ++k) umma_f8_pair(d, adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), idesc, k > 0 ? 1u : 0u);
            g2_commit_both(empty + s);
            g2_commit_both(tfull + buf);
            if (++s == STAGES) {
              s = 0;
              ph ^= 1u;
            }
            if (++buf == 2) {
              buf = 0;
              tph ^= 1u;
            }
          }
        }
        if (!go) {
          g2_commit_both(done);
          mbar_drain(done, 0);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int q = warp & 3, half = (warp - 4) >> 2, row = q * 32 + lane;
    const uint32_t tempty_leader = g2_map(smem_u32(tempty), 0);
    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16);
    int buf = 0, lt = 0;
    uint32_t tph = 0;
    for (long tile = pair; tile < num_tiles; tile += num_pairs, ++lt) {
      const int mb = (int)(tile % m_tiles), nb = (int)(tile / m_tiles);
      const int tok = mb * 2 * kBM + (int)rank * kBM + row;
      const int f0 = GATED ? nb * HB + half * (HB / 2) : nb * BN + half * HB;  // the thread's first feature
      const float* sx = p.sx + (tok < N ? tok : 0);
      const float* sw = p.sw + (size_t)(f0 < M ? f0 / kBlock : 0) * kb_n;
      const float* sw2 = GATED ? p.sw2 + (size_t)(f0 < M ? f0 / kBlock : 0) * kb_n : nullptr;
      uint64_t acc[HB / 2];
#pragma unroll
      for (int j = 0; j < HB / 2; ++j) acc[j] = 0;
      float x_next = __ldg(sx), w_next = __ldg(sw), w2_next = GATED ? __ldg(sw2) : 0.f;
#pragma unroll 1
      for (int kb = 0; kb < kb_n; ++kb) {
        const float s1 = x_next * w_next, s2 = GATED ? x_next * w2_next : s1;
        if (kb + 1 < kb_n) {
          x_next = __ldg(sx + (size_t)(kb + 1) * p.ld_sx);
          w_next = __ldg(sw + kb + 1);
          if (GATED) w2_next = __ldg(sw2 + kb + 1);
        }
        mbar_wait_bounded(tfull + buf, tph, dead);
        tc_fence_after();
        const uint32_t t0 = t_row + (uint32_t)(buf * BN);
        // columns of the thread's piece c of 32; gated: 64 of the gate, then 64 of the factor
        auto column = [&](int c) { return (uint32_t)(GATED ? (c < HB / 2 ? half * (HB / 2) + c : HB / 2 + half * (HB / 2) + c) : half * HB + c); };
        uint32_t v[2][32];
        tmem_ld32_nowait(t0 + column(0), v[0]);
#pragma unroll
        for (int c = 0; c < HB; c += 32) {
          uint32_t* now = v[(c / 32) & 1];
          tmem_wait32(now);
          if (c + 32 < HB) tmem_ld32_nowait(t0 + column(c + 32), v[(c / 32 + 1) & 1]);
          const float s = GATED && c >= HB / 2 ? s2 : s1;
          const uint64_t ss = pair_of(s, s);
#pragma unroll
          for (int j = 0; j < 16; ++j) fma2(acc[c / 2 + j], pair_of(now[2 * j], now[2 * j + 1]), ss);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) g2_arrive_cluster(tempty_leader + (uint32_t)(buf * 8));
        if (++buf == 2) {
          buf = 0;
          tph ^= 1u;
        }
      }
      if constexpr (GATED) {
        float v[HB / 2];
        if (p.act == 0) activate<0>(acc, v);
        else if (p.act == 1) activate<1>(acc, v);
        else activate<2>(acc, v);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < HB / 2; ++j) m = max(m, magnitude(v[j]));
        uint32_t* mine = largest + (lt & 1) * 256;  // (the other tile's are read until the barrier behind this one)
        mine[half * 128 + row] = m;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpi) : "memory");
        const Scale k = scale_of(max(mine[row], mine[128 + row]));
        if (tok < N && f0 < M) {
          uint8_t* dst = p.codes + (size_t)tok * p.ld + f0;
#pragma unroll
          for (int c = 0; c < HB / 2; c += 16) {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = codes4(v + c + 4 * j, k);
            if (f0 + c + 16 <= M) {
              *reinterpret_cast<uint4*>(dst + c) = make_uint4(u[0], u[1], u[2], u[3]);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (f0 + c + j < M) dst[c + j] = (uint8_t)(u[j / 4] >> (8 * (j & 3)));
            }
          }
          if (half == 0) p.scales[(size_t)(f0 / kBlock) * p.ld_s + tok] = k.s;
        }
      } else {
        O* y = static_cast<O*>(p.y);
        const bool vec = (p.ld_y * (long)sizeof(O)) % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
        for (int c = 0; c < HB; c += 32) {
          if (tok - lane >= N || f0 + c >= M) continue;  // (a warp at a time: the lanes store for one another)
          if (vec && f0 + c + 32 <= M) {
            store32(y + f0 + c, p.ld_y, tok, N, lane, acc + c / 2);
          } else if (tok < N) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (f0 + c + j < M) y[(size_t)tok * p.ld_y + f0 + c + j] = from_f<O>(j & 1 ? hi_of(acc[c / 2 + j / 2]) : lo_of(acc[c / 2 + j / 2]));
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // the peer's MMAs / loads may still target this CTA's shared memory and TMEM
  if (warp == 1) {
    tc_fence_after();
    g2_tmem_dealloc(tmem_base, 2 * BN);
  }
  if (threadIdx.x == 0) count_run_out(dead, p.err);
}

template <int BN, int STAGES, bool GATED, typename O>
int launch_pair(const Product& p, cudaStream_t st) {
  static_assert((size_t)STAGES * (kBM + BN / 2) * kBK + 1024 + 2304 <= 227 * 1024, "shared memory of a CTA");
  constexpr size_t smem = 227 * 1024;  // all of it: nobody else is resident on an SM whose tensor memory this kernel has (fp8_gemm_few.cu)
  auto kern = fp8_gemm_kernel<BN, STAGES, GATED, O>;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kern, smem); e != cudaSuccess) return (int)e;
  CUtensorMap mx, mw, mw2;
  if (!make_codes_map(&mx, p.x, p.N, p.K, p.ld_x, kBM) || !make_codes_map(&mw, p.w, p.M, p.K, p.ld_w, BN / 2) ||
      !make_codes_map(&mw2, GATED ? p.w2 : p.w, p.M, p.K, p.ld_w, BN / 2))
    return (int)cudaErrorInvalidValue;
  constexpr int features = GATED ? BN / 2 : BN;
  const long tiles = (long)((p.N + 2 * kBM - 1) / (2 * kBM)) * ((p.M + features - 1) / features);
  const int pairs = (int)std::min<long>(std::max(1, sm_count() / 2), tiles);
  return (int)launch(kern, dim3(2 * pairs), dim3(kThreads), smem, st, true, mx, mw, mw2, p);
}

}  // namespace
}  // namespace fp8
}  // namespace pk

using namespace pk;

static bool product_ok(const void* w, const float* sw, long ld_w, const void* x, long ld_x, const float* sx, long ld_sx, int M, int N, int K) {
  return sw && M > 0 && N > 0 && K > 0 && fp8::codes_ok(w, ld_w, K) && fp8::codes_ok(x, ld_x, K) && fp8::row_scales_ok(sx, ld_sx, N);
}
static bool sizes_fit(int M, int N, int K) { return M <= 1 << 30 && N <= 1 << 30 && K <= 1 << 30; }

extern "C" int pk_fp8_gemm(const void* w, long ld_w, const float* w_scales, const void* x, long ld_x, const float* x_scales, long ld_xs, void* y, long ld_y, int y_f32, int M,
                           int N, int K, pk_stream st) {
  if (!y || (ld_y != 0 && ld_y < M) || !product_ok(w, w_scales, ld_w, x, ld_x, x_scales, ld_xs, M, N, K)) return -1;
  if (!sizes_fit(M, N, K)) return -2;
  fp8::Product p{};
  p.w = (const uint8_t*)w;
  p.sw = w_scales;
  p.ld_w = ld_w;
  p.x = (const uint8_t*)x;
  p.sx = x_scales;
  p.ld_x = ld_x;
  p.ld_sx = ld_xs;
  p.y = y;
  p.ld_y = ld_y ? ld_y : M;
  p.M = M;
  p.N = N;
  p.K = K;
  p.kb = fp8::blocks_of(K);
  p.err = wait_err_word();
  if (fp8::few_takes(p, false)) return fp8::launch_few(p, false, y_f32, st);
  return y_f32 ? fp8::launch_pair<256, 6, false, float>(p, st) : fp8::launch_pair<256, 6, false, bf16>(p, st);
}

extern "C" int pk_fp8_gemm_gated(const void* w_gate, const float* gate_scales, const void* w_up, const float* up_scales, long ld_w, const void* x, long ld_x,
                                 const float* x_scales, long ld_xs, void* codes, long ld, float* scales, long ld_s, int F, int N, int K, int act, pk_stream st) {
  if (!up_scales || act < 0 || act > 2 || !product_ok(w_gate, gate_scales, ld_w, x, ld_x, x_scales, ld_xs, F, N, K) || !fp8::codes_ok(w_up, ld_w, K) ||
      !fp8::codes_ok(codes, ld, F) || !fp8::row_scales_ok(scales, ld_s, N) || codes == x)
    return -1;
  if (!sizes_fit(F, N, K)) return -2;
  fp8::Product p{};
  p.w = (const uint8_t*)w_gate;
  p.w2 = (const uint8_t*)w_up;
  p.sw = gate_scales;
  p.sw2 = up_scales;
  p.ld_w = ld_w;
  p.x = (const uint8_t*)x;
  p.sx = x_scales;
  p.ld_x = ld_x;
  p.ld_sx = ld_xs;
  p.codes = (uint8_t*)codes;
  p.ld = ld;
  p.scales = scales;
  p.ld_s = ld_s;
  p.M = F;
  p.N = N;
  p.K = K;
  p.kb = fp8::blocks_of(K);
  p.act = act;
  p.err = wait_err_word();
  if (fp8::few_takes(p, true)) return fp8::launch_few(p, true, false, st);
  return fp8::launch_pair<256, 6, true, uint8_t>(p, st);
}
