// The product of 8-bit rows and weights for few tokens (fp8_gemm.cuh): a pass over the weights, so what counts is that every SM streams the same share of them.
//
//   A = W: `rows` <= 128 features per tile (tensor-memory lane = feature), B = X: NT tokens (column = token).  Gated: two tiles of A, 128 rows of w and the same of w2.
//   A tile's K is cut into parts, one CTA each, and those CTAs are a cluster: each leaves its fp32 part in its own shared memory ([token][feature], over the operand ring), and
//   after a cluster barrier adds up its share of the tile in rank order over distributed shared memory, so a result does not depend on timing.
//   warp 0 TMA producer | warp 1 MMA issuer | the others: a block's partial sum out of tensor memory, times its scales (a token's come with the stage, a feature's is the thread's own),
//   onto the sum in registers; then the part.  All warps: sums -> output.
// Any number of rows may make a tile: the MMAs read 128, and what lies behind the tile's own ends in lanes that nobody reads.
#include <cuda.h>

#include <algorithm>

#include "fp8_gemm.cuh"

namespace pk {
namespace fp8 {

namespace {

constexpr int kRows = 128, kMaxSplit = 8, kMaxStages = 12;  // 8: the portable cluster size
// CTAs on an SM: one where a thread holds many columns' sums
constexpr int per_sm(int na, int nt) { return na * nt >= 128 ? 1 : 2; }
constexpr int smem_most(int na, int nt) { return per_sm(na, nt) == 2 ? 113 * 1024 : 227 * 1024; }
// A CTA's share of an SM's shared memory (228 KB, of which it takes 1 KB more than it asks for) is at least its share of the tensor memory, and more than any kernel with all 512
// columns leaves: whoever is resident has its columns at once.  (CTAs that wait for columns while the rest of their cluster waits for them could wait for one another.)
constexpr size_t smem_least(int columns) { return columns > 128 ? 113 * 1024 : 56 * 1024; }

__device__ __forceinline__ float4 ld_dsmem(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// global -> shared; bytes % 16 == 0, both addresses on 16-byte boundaries
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

struct FewPlan {
  int rows, splits, stages;  // features of a tile, parts of K
  int n_tiles;               // tiles of tokens
};
constexpr size_t stage_bytes(int na, int rows, int nt) { return (size_t)(na * rows + nt) * kBK; }
constexpr size_t few_smem(int na, int rows, int nt, int stages) {
  return stages * (stage_bytes(na, rows, nt) + nt * sizeof(float)) + (size_t)(kRows - rows) * kBK + 1024 + (2 * kMaxStages + 4) * 8 + 16;
}

constexpr int tmem_columns(int na, int nt) { return 2 * na * nt <= 32 ? 32 : 2 * na * nt <= 64 ? 64 : 2 * na * nt <= 128 ? 128 : 256; }

// NA tiles of A
template <int NT, int NA, typename O>
__global__ void __launch_bounds__(64 + 128 * NA, per_sm(NA, NT))
fp8_gemm_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2, const Product p,
                    const FewPlan plan) {
  constexpr int THREADS = 64 + 128 * NA;
  constexpr uint32_t TMEM_COLS = tmem_columns(NA, NT);
  static_assert(2 * NA * NT <= 256, "two CTAs on an SM");
    const int stages = plan.stages, rows = plan.rows;
  const uint32_t A_BYTES = rows * kBK, STAGE = NA * A_BYTES + NT * kBK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // (behind the last stage lies room for the rows of A that the MMAs read beyond the tile's own)
  float* xs = reinterpret_cast<float*>(smem + (size_t)stages * STAGE + (kRows - rows) * kBK);  // [stages][NT] scales of the tokens
  uint64_t* full = reinterpret_cast<uint64_t*>(xs + stages * NT);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;  // [2]
  uint64_t* tempty = tfull + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = gridDim.x, sp = (int)cluster_ctarank();  // the cluster spans the whole x axis
  const int m0 = (blockIdx.y / plan.n_tiles) * rows, t0 = (blockIdx.y % plan.n_tiles) * NT;
  const int kb0 = (int)((long)sp * p.kb / S), nk = (int)((long)(sp + 1) * p.kb / S) - kb0;

  const uint32_t n_scales = (uint32_t)min(NT, (p.N - t0 + 3) & ~3);  // (rows of scales are whole fours)
  auto copy = [&](int i, int s) {  // block i of this CTA's into stage s
    mbar_expect_tx(full + s, STAGE + n_scales * 4u);
    uint8_t* st = smem + (size_t)s * STAGE;
    const int kb = kb0 + i;
    tma_load_2d(st, &map_w, kb * kBK, m0, full + s);
    if (NA == 2) tma_load_2d(st + A_BYTES, &map_w2, kb * kBK, m0, full + s);
    tma_load_2d(st + NA * A_BYTES, &map_x, kb * kBK, t0, full + s);
    bulk_copy(xs + s * NT, p.sx + (size_t)kb * p.ld_sx + t0, n_scales * 4u, full + s);
  };
  // the thread that starts the copies fills the ring before anybody waits for anybody
  const bool copies = warp == 0 && tc_elect_one();
  if (copies) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    if (NA == 2) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w2) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    for (int s = 0; s < stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 4 * NA);  // the warps that read the scales, behind the MMAs' end
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(tfull + s, 1);
      mbar_init(tempty + s, 4 * NA);
    }
    *dead = 0;
    mbar_fence_init();
    // no early trigger: gemv.cu streams its weights before it waits for its predecessor, and they may be this kernel's output
    pdl_wait();
    for (int i = 0; i < stages && i < nk; ++i) copy(i, i);
  }
  if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  float* part = reinterpret_cast<float*>(smem);  // [NT tokens][NA * rows features], over the ring
  if (warp == 0) {
    if (copies) {
      int s = 0, i = stages;
      uint32_t ph = 0;
      for (; i < nk; ++i) {
        if (!mbar_wait_bounded(empty + s, ph, dead)) break;
        copy(i, s);
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (i < nk) ring_drain(full, stages, i);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (tc_elect_one()) {
      constexpr uint32_t idesc = f8_idesc(kRows, NT);
      int s = 0, i = 0;
      uint32_t ph = 0;
      for (; i < nk; ++i) {
        const int buf = i & 1;
        const uint32_t tph = (uint32_t)(((i >> 1) & 1) ^ 1);
        // two looks at once: a wait costs a thread 200 clocks where nothing is to be waited for
        const bool here = mbar_test_wait(full + s, ph), free = mbar_test_wait(tempty + buf, tph);
        if (!here && !mbar_wait_bounded(full + s, ph, dead)) break;
        if (!free && !mbar_wait_bounded(tempty + buf, tph, dead)) break;
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + (size_t)s * STAGE);
        const uint64_t bdesc = make_sw128_desc(a_addr + NA * A_BYTES);
#pragma unroll
        for (int h = 0; h < NA; ++h) {
          const uint64_t adesc = make_sw128_desc(a_addr + h * A_BYTES);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)
            umma_f8(tmem_base + (uint32_t)((buf * NA + h) * NT), adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), idesc, k > 0 ? 1u : 0u);
        }
        umma_commit(tfull + buf);
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (i < nk) {  // MMAs under way end in a partial sum that nobody waits for any more
        umma_commit(tfull + (i & 1));
        mbar_drain(tfull + (i & 1), (uint32_t)((i >> 1) & 1));
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, h = (warp - 2) >> 2, f = q * 32 + lane;  // tensor-memory lanes that this warp may read; lane = feature
    const int row = m0 + f < p.M ? m0 + f : p.M - 1;
    const float* sw = (NA == 2 && h == 1 ? p.sw2 : p.sw) + (size_t)(row / kBlock) * p.kb + kb0;
    uint64_t acc[NT / 2];
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) acc[j] = 0;
    float w_next = __ldg(sw);
    int s = 0;
    uint32_t ph = 0;
    for (int i = 0; i < nk; ++i) {
      const int buf = i & 1;
      const uint64_t w = pair_of(w_next, w_next);
      if (i + 1 < nk) w_next = __ldg(sw + i + 1);
      const uint32_t tph = (uint32_t)((i >> 1) & 1);
      const bool here = mbar_test_wait(full + s, ph), done = mbar_test_wait(tfull + buf, tph);
      if (!here) mbar_wait_bounded(full + s, ph, dead);  // (the scales)
      if (!done) mbar_wait_bounded(tfull + buf, tph, dead);
      tc_fence_after();
      const uint32_t t0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)((buf * NA + h) * NT);
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(tempty + buf);
          mbar_arrive(empty + s);
        }
      };
      auto add4 = [&](int at, const uint32_t* u, float4 x) {
        acc[at / 2] = fma2(pair_of(u[0], u[1]), mul2(w, pair_of(x.x, x.y)), acc[at / 2]);
        acc[at / 2 + 1] = fma2(pair_of(u[2], u[3]), mul2(w, pair_of(x.z, x.w)), acc[at / 2 + 1]);
      };
      auto scale4 = [&](int at) { return *reinterpret_cast<const float4*>(xs + s * NT + at); };
      uint32_t v[2][16];
      tmem_ld16(t0, v[0]);
#pragma unroll
      for (int c = 0; c < NT; c += 16) {
        float4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = scale4(c + 4 * j);
        uint32_t* now = v[(c / 16) & 1];
        tmem_wait16(now);
        if (c + 16 < NT) tmem_ld16(t0 + (uint32_t)(c + 16), v[(c / 16 + 1) & 1]);
        else release();
#pragma unroll
        for (int j = 0; j < 4; ++j) add4(c + 4 * j, now + 4 * j, x[j]);
      }
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    // every MMA has read its operands: the ring takes the part (but another warp may still read its last scales: those lie behind the ring)
    if (f < rows) {
#pragma unroll
      for (int c = 0; c < NT; c += 2) {
        part[(size_t)c * (NA * rows) + h * rows + f] = lo_of(acc[c / 2]);
        part[(size_t)(c + 1) * (NA * rows) + h * rows + f] = hi_of(acc[c / 2]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (S > 1) cluster_barrier();
  // ---- this CTA's share of the tile, added up in rank order
  const uint32_t part_addr = smem_u32(part);
  const int tokens = min(NT, p.N - t0);
  auto sum4 = [&](int at) {  // four features of a token
    float4 v[kMaxSplit];
#pragma unroll
    for (int r = 0; r < kMaxSplit; ++r)
      if (r < S) v[r] = S > 1 ? ld_dsmem(part_addr + (uint32_t)at * 4u, (uint32_t)r) : *reinterpret_cast<const float4*>(part + at);
    float4 t = v[0];
#pragma unroll
    for (int r = 1; r < kMaxSplit; ++r)
      if (r < S) {
        t.x += v[r].x;
        t.y += v[r].y;
        t.z += v[r].z;
        t.w += v[r].w;
      }
    return t;
  };
  if constexpr (NA == 1) {
    const int quads = rows / 4, items = tokens * quads;
    const int i0 = (int)((long)sp * items / S), i1 = (int)((long)(sp + 1) * items / S);
    O* y = static_cast<O*>(p.y);
    for (int it = i0 + threadIdx.x; it < i1; it += THREADS) {
      const int t = it / quads, f = m0 + (it - t * quads) * 4;
      const float4 v = sum4(it * 4);
      if (f >= p.M) continue;
      O* dst = y + (size_t)(t0 + t) * p.ld_y + f;
      if (f + 4 <= p.M && (reinterpret_cast<uintptr_t>(dst) & (4 * sizeof(O) - 1)) == 0) {
        if constexpr (sizeof(O) == 4) *reinterpret_cast<float4*>(dst) = v;
        else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      } else {
        const float o[4] = {v.x, v.y, v.z, v.w};
        for (int j = 0; j < 4 && f + j < p.M; ++j) dst[j] = from_f<O>(o[j]);
      }
    }
  } else {
    // a warp has a token's 128 features, a block of the result's scales
    const int i0 = (int)((long)sp * tokens / S), i1 = (int)((long)(sp + 1) * tokens / S);
    constexpr int WARPS = THREADS / 32;
    for (int t = i0 + warp; t < i1; t += 2 * WARPS) {  // two at once: the others' shared memory is 1 us away
      float4 g[2], u[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (t + j * WARPS < i1) {
          g[j] = sum4((t + j * WARPS) * 256 + lane * 4);
          u[j] = sum4((t + j * WARPS) * 256 + 128 + lane * 4);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tok = t + j * WARPS;
        if (tok >= i1) break;
        float v[4] = {g[j].x, g[j].y, g[j].z, g[j].w};
        const float w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (p.act == 0 ? gate_act<0>(v[e]) : p.act == 1 ? gate_act<1>(v[e]) : gate_act<2>(v[e])) * w[e];
        const float m = max16(max_abs(max_abs(v[0], v[1], v[2]), v[3]));
        const Scale k = scale_of(max_abs(m, __shfl_xor_sync(0xffffffffu, m, 16)));
        const uint32_t c = codes4(v, k);
        const int f = m0 + lane * 4;
        uint8_t* dst = p.codes + (size_t)(t0 + tok) * p.ld + f;
        if (f + 4 <= p.M) {
          *reinterpret_cast<uint32_t*>(dst) = c;
        } else {
          for (int e = 0; e < 4 && f + e < p.M; ++e) dst[e] = (uint8_t)(c >> (8 * e));
        }
        if (lane == 0) p.scales[(size_t)(m0 / kBlock) * p.ld_s + t0 + tok] = k.s;
      }
    }
  }
  if (threadIdx.x == 0) count_run_out(dead, p.err);  // (every wait lies before the barrier above)
  __syncwarp();
  if (S > 1) cluster_barrier();  // the others may still read this CTA's part
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Clusters of `splits` CTAs that can be resident at once (a cluster lives inside one GPC: gemm_skinny.cu)
int resident(int splits, int sms, int per) { return (splits == 8 ? sms * 16 / 148 : splits == 4 ? sms * 35 / 148 : sms / splits) * per; }

// The most parts of K for which all tiles run at once, and the lowest tiles for which they still do, so that every SM has the same share of the weights.
FewPlan few_plan(int M, int N, int kb, int na, int nt, int sms) {
  FewPlan p{kRows, 1, 2, (N + nt - 1) / nt};
  for (int S = kMaxSplit; S >= 1; S /= 2) {
    if (S > 1 && S > kb / 2) continue;  // at least two blocks a part
    const int fit = resident(S, sms, per_sm(na, nt)) / p.n_tiles;  // tiles of features
    if (S > 1 && (long)fit * kRows < M) continue;
    p.splits = S;
    if (na == 1 && fit > 0 && (long)fit * kRows >= M) p.rows = std::max(32, ((M + fit - 1) / fit + 7) / 8 * 8);
    break;
  }
  const int nk = (kb + p.splits - 1) / p.splits;
  const size_t part = (size_t)nt * na * p.rows * 4;
  p.stages = kMaxStages;
  while (p.stages > 2 && few_smem(na, p.rows, nt, p.stages) > (size_t)smem_most(na, nt)) --p.stages;
  const int hold = (int)((part + stage_bytes(na, p.rows, nt) - 1) / stage_bytes(na, p.rows, nt));  // stages that the part covers
  if (p.stages > nk) p.stages = std::max(nk, hold);
  return p;
}

template <int NT, int NA, typename O>
int run_few(const Product& p, cudaStream_t st) {
  auto kern = fp8_gemm_few_kernel<NT, NA, O>;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kern, smem_most(NA, NT)); e != cudaSuccess) return (int)e;
  const FewPlan plan = few_plan(p.M, p.N, p.kb, NA, NT, sm_count());
  CUtensorMap mx, mw, mw2;
  if (!make_codes_map(&mx, p.x, p.N, p.K, p.ld_x, NT) || !make_codes_map(&mw, p.w, p.M, p.K, p.ld_w, plan.rows) ||
      !make_codes_map(&mw2, NA == 2 ? p.w2 : p.w, p.M, p.K, p.ld_w, plan.rows))
    return (int)cudaErrorInvalidValue;
  ThreadState& ts = tls();
  ts.launches++;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(plan.splits, (p.M + plan.rows - 1) / plan.rows * plan.n_tiles);
  cfg.blockDim = dim3(64 + 128 * NA);
  cfg.dynamicSmemBytes = std::max(few_smem(NA, plan.rows, NT, plan.stages), smem_least(tmem_columns(NA, NT)));
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = ts.pdl ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = plan.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, kern, mx, mw, mw2, p, plan);
}

}  // namespace

bool few_takes(const Product& p, bool gated) { return p.N <= (gated ? 64 : 128) && (p.M + 31) / 32 <= 65535; }  // (tiles are counted on a grid's second axis)

int launch_few(const Product& p, bool gated, bool y_f32, cudaStream_t st) {
  if (gated) {
    if (p.N <= 16) return run_few<16, 2, uint8_t>(p, st);
    if (p.N <= 32) return run_few<32, 2, uint8_t>(p, st);
    return run_few<64, 2, uint8_t>(p, st);
  }
  auto go = [&](auto f, auto b) { return y_f32 ? f(p, st) : b(p, st); };
  if (p.N <= 16) return go(run_few<16, 1, float>, run_few<16, 1, bf16>);
  if (p.N <= 32) return go(run_few<32, 1, float>, run_few<32, 1, bf16>);
  if (p.N <= 64) return go(run_few<64, 1, float>, run_few<64, 1, bf16>);
  return go(run_few<128, 1, float>, run_few<128, 1, bf16>);
}

}  // namespace fp8
}  // namespace pk
