// The product of 8-bit rows and weights for few tokens (fp8_gemm.cuh): a pass over the weights, so what counts is that every SM streams the same share of them.
//
//   A = W: NA tiles of `rows` <= 128 features (tensor-memory lane = feature), B = X: NT tokens (column = token).  Gated: 128 rows of w and the same of w2.
//   A tile's K is cut into parts, one CTA each, and those CTAs are a cluster: each leaves its fp32 part over its operand ring and sends it, 16 bytes a thread, to the CTAs that own a share of
//   the tile's results (features; gated: tokens, whose 128 features are a block of the result's scales), which add them up in rank order, so a result does not depend on timing.
//   warp 0 TMA producer | warps 1 and 2 MMA issuers of even and odd blocks (one for all: 64 tokens of 24576 x 4096 27.6 us for 25.2) | the others: a block's partial sum out of tensor memory,
//   times its scales (a token's come with the stage, a feature's is the thread's own), onto the sum in registers; then the part.  All warps: sums -> output.
// Any number of rows may make a tile: the MMAs read 128, and what lies behind the tile's own ends in lanes that nobody reads.
// One CTA has an SM: a second one on it would start 1 us later, and a cluster of eight with two on an SM 2 us.
//
// What bounds it, B200, 48 tokens of 4096 x 12288 (51 MB), us: 14.8, of them 2 between launches, 3 to the first block (1.2 from the launch to the first copy's start; all rings are asked for at
// once, so the first stage comes behind parts of the others), 7.5 for the stream (6.7 TB/s), 2 for the joining.  One token of 2560 x 4096: 6.6, the same without the stream.
// A cluster's joining, measured: words sent by the threads that have them 16.7, bulk copies from shared to shared memory 18.1, 16 bytes a thread of a part laid down feature by feature 15.8
// (then two groups of warps for the sums: 15.0; parts fetched behind a barrier instead, with two CTAs an SM: 15.6).
#include <cuda.h>

#include <algorithm>

#include "fp8_gemm.cuh"

namespace pk {
namespace fp8 {

namespace {

constexpr int kRows = 128, kMaxStages = 12;
constexpr int kSmemMost = 227 * 1024;
// A CTA asks for more than half of an SM's shared memory, so it is alone with its kind, and for more than any kernel with all 512 columns of tensor memory leaves: whoever is resident has
// its columns at once.  (CTAs that wait for columns while the rest of their cluster waits for them could wait for one another.)
constexpr size_t kSmemLeast = 116 * 1024;

__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void st_cluster4(uint32_t dst_cluster, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst_cluster), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
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
  int rows, splits, stages;  // features of a tile of A, parts of K
  int n_tiles;               // tiles of tokens
  int own;                   // features (gated: tokens, a multiple of four) of the tile that a CTA adds up
  double ns;                 // what a call takes, about
  uint32_t zero;             // 0, which the compiler does not know
};
constexpr size_t stage_bytes(int na, int rows, int nt) { return (size_t)(na * rows + nt) * kBK; }
// floats from one feature of a part to the next: the lanes' 16-byte accesses at one token fall on different banks
constexpr int part_ld(int nt) { return nt + 4; }
// parts that a CTA receives
size_t received_bytes(int na, const FewPlan& p, int nt, bool gated) { return p.splits == 1 ? 0 : (size_t)p.splits * p.own * (gated ? na * p.rows : part_ld(nt)) * sizeof(float); }
size_t few_smem(int na, const FewPlan& p, int nt, bool gated) {
  return p.stages * (stage_bytes(na, p.rows, nt) + nt * sizeof(float)) + (size_t)(kRows - p.rows) * kBK + received_bytes(na, p, nt, gated) + 1024 + (2 * kMaxStages + 4) * 8 + 16;
}
constexpr int tmem_columns(int na, int nt) { return 2 * na * nt <= 32 ? 32 : 2 * na * nt <= 64 ? 64 : 2 * na * nt <= 128 ? 128 : 256; }

// groups of four warps that take sums out of tensor memory: one to a tile of A, two where one tile has many columns (128 tokens: a block takes one group 530 ns)
constexpr int groups(int na, int nt) { return na == 1 && nt >= 64 ? 2 : na; }

// GATED: NA = 2, O is the codes' type
template <int NT, int NA, bool GATED, typename O>
__global__ void __launch_bounds__(96 + 128 * groups(NA, NT), 1)
fp8_gemm_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2, const Product p,
                    const FewPlan plan) {
  constexpr int GROUPS = groups(NA, NT), COLS = NT * NA / GROUPS, THREADS = 96 + 128 * GROUPS;  // COLS: columns of a thread
  constexpr uint32_t TMEM_COLS = tmem_columns(NA, NT);
  static_assert(2 * NA * NT <= 256 && (!GATED || NA == 2), "tensor memory");
  const int stages = plan.stages, rows = plan.rows;
  const uint32_t A_BYTES = rows * kBK, STAGE = NA * A_BYTES + NT * kBK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // (behind the last stage lies room for the rows of A that the MMAs read beyond the tile's own)
  float* xs = reinterpret_cast<float*>(smem + (size_t)stages * STAGE + (kRows - rows) * kBK);  // [stages][NT] scales of the tokens
  const int S = gridDim.x, sp = (int)cluster_ctarank();  // the cluster spans the whole x axis
  const int features = NA * rows, own = plan.own;
  constexpr int LD = part_ld(NT);
  float* part = reinterpret_cast<float*>(smem);       // over the ring: [features][LD]
  float* received = S > 1 ? xs + stages * NT : part;  // [S senders][own features][LD]; gated [S][256][own tokens]
  uint64_t* full = reinterpret_cast<uint64_t*>(xs + stages * NT + (S > 1 ? S * own * (GATED ? 256 : LD) : 0));
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;  // [2]
  uint64_t* tempty = tfull + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = (blockIdx.y / plan.n_tiles) * (GATED ? rows : features), t0 = (blockIdx.y % plan.n_tiles) * NT;
  const int kb0 = (int)((long)sp * p.kb / S), nk = (int)((long)(sp + 1) * p.kb / S) - kb0;

  const int tokens = min(NT, p.N - t0);
  const uint32_t n_scales = (uint32_t)min(NT, (p.N - t0 + 3) & ~3);  // (rows of scales are whole fours)
  auto copy = [&](int i, int s) {  // block i of this CTA's into stage s
    mbar_expect_tx(full + s, STAGE + n_scales * 4u);
    uint8_t* st = smem + (size_t)s * STAGE;
    const int kb = kb0 + i;
    tma_load_2d(st, &map_w, kb * kBK, m0, full + s);
    if (NA == 2) tma_load_2d(st + A_BYTES, GATED ? &map_w2 : &map_w, kb * kBK, GATED ? m0 : m0 + rows, full + s);
    tma_load_2d(st + NA * A_BYTES, &map_x, kb * kBK, t0, full + s);
    bulk_copy(xs + s * NT, p.sx + (size_t)kb * p.ld_sx + t0, n_scales * 4u, full + s);
  };
  // the thread that starts the copies fills the ring before anybody waits for anybody
  const bool copies = warp == 0 && tc_elect_one();
  if (copies) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    if (GATED) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w2) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    for (int s = 0; s < stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 4 * GROUPS);  // the warps that read the scales, behind the MMAs' end
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(tfull + s, 1);
      mbar_init(tempty + s, 4 * GROUPS);
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
  if (S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (waited for in front of the first word for another CTA)
  pdl_wait();

  uint64_t acc[COLS / 2];
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
  } else if (warp < 3) {
    if (tc_elect_one()) {
      constexpr uint32_t idesc = f8_idesc(kRows, NT);
      const int buf = warp - 1;
      int s = buf, i = buf;
      uint32_t ph = 0, tph = 1;
      for (; i < nk; i += 2) {
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
        tph ^= 1u;
        s += 2;
        if (s >= stages) {
          s -= stages;
          ph ^= 1u;
        }
      }
      if (i < nk) {  // MMAs under way end in a partial sum that nobody waits for any more
        umma_commit(tfull + buf);
        mbar_drain(tfull + buf, tph ^ 1u);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, group = (warp - 3) >> 2, h = group % NA, c0 = group / NA * COLS, f = q * 32 + lane;  // tensor-memory lanes that this warp may read; lane = feature
    const int at = m0 + (GATED ? f : h * rows + f), row = at < p.M ? at : p.M - 1;
    const float* sw = (GATED && h == 1 ? p.sw2 : p.sw) + (size_t)(row / kBlock) * p.kb + kb0;
#pragma unroll
    for (int j = 0; j < COLS / 2; ++j) acc[j] = 0;
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
      const uint32_t t0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)((buf * NA + h) * NT + c0);
      // The stage goes back when its scales are in registers.  An arrival does not wait for loads on their way: with nothing more the copy of the stage's next block overtook the last of them
      // in 8 of 60000 calls.  So its address takes a word of each of the last loads (a warp's loads of shared memory return in order): 1 to 2 % of a call, a proxy fence 3 to 5 %, words of
      // all loads up to 20 %.
      auto release = [&](uint32_t read) {
        tc_fence_before();
        uint32_t bar = smem_u32(empty + s);
        asm volatile("{\n.reg .b32 t;\nand.b32 t, %1, %2;\nadd.u32 %0, %0, t;\n}" : "+r"(bar) : "r"(read), "r"(plan.zero));
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(tempty + buf);
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
        }
      };
      auto add4 = [&](int at, const uint32_t* u, float4 x) {
        acc[at / 2] = fma2(pair_of(u[0], u[1]), mul2(w, pair_of(x.x, x.y)), acc[at / 2]);
        acc[at / 2 + 1] = fma2(pair_of(u[2], u[3]), mul2(w, pair_of(x.z, x.w)), acc[at / 2 + 1]);
      };
      auto scale4 = [&](int at) { return *reinterpret_cast<const float4*>(xs + s * NT + c0 + at); };
      uint32_t v[2][16];
      tmem_ld16(t0, v[0]);
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        float4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = scale4(c + 4 * j);
        uint32_t* now = v[(c / 16) & 1];
        tmem_wait16(now);
        if (c + 16 < COLS) tmem_ld16(t0 + (uint32_t)(c + 16), v[(c / 16 + 1) & 1]);
        else release(__float_as_uint(x[0].x) | __float_as_uint(x[1].x) | __float_as_uint(x[2].x) | __float_as_uint(x[3].x));
#pragma unroll
        for (int j = 0; j < 4; ++j) add4(c + 4 * j, now + 4 * j, x[j]);
      }
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
  }
  // ---- the part over the ring, whose operands every MMA has read, and to its owners.  (What runs once runs from cold instruction memory: few instructions, 16 bytes each.  One word each
  // took 1.3 us for 64 tokens and 2.8 for 128.)
  if (warp >= 3) {
    const int q = warp & 3, group = (warp - 3) >> 2, h = group % NA, c0 = group / NA * COLS, f = q * 32 + lane;
    if (f < rows) {
      float4* to = reinterpret_cast<float4*>(part + (size_t)(h * rows + f) * LD + c0);
#pragma unroll
      for (int c = 0; c < COLS / 4; ++c) to[c] = make_float4(lo_of(acc[2 * c]), hi_of(acc[2 * c]), lo_of(acc[2 * c + 1]), hi_of(acc[2 * c + 1]));
    }
  }
  tc_fence_before();
  __syncthreads();
  const int fours = (tokens + 3) / 4;  // tokens by fours
  constexpr int WARPS = THREADS / 32, LANES = NT / 4, ROWS = 32 / LANES;  // a warp has ROWS features of all tokens
  if (S > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs of the cluster are there
    const uint32_t to = smem_u32(received);
    const int c = lane % LANES, first = warp * ROWS + lane / LANES;
    if constexpr (GATED) {
      const int r = 4 * c / own;
      const uint32_t dst = map_to(to + (uint32_t)((sp * 256 * own + 4 * c - r * own) * 4), (uint32_t)min(r, S - 1));
      if (c < fours)
        for (int g = first; g < 256; g += WARPS * ROWS) st_cluster4(dst + (uint32_t)(g * own * 4), *reinterpret_cast<const float4*>(part + g * LD + 4 * c));
    } else {
      for (int r = 0; r < S; ++r) {
        const uint32_t dst = map_to(to + (uint32_t)((sp * own * LD + 4 * c) * 4), (uint32_t)r);
        const int n = min(own, features - r * own);
        if (c < fours)
          for (int g = first; g < n; g += WARPS * ROWS) st_cluster4(dst + (uint32_t)(g * LD * 4), *reinterpret_cast<const float4*>(part + (r * own + g) * LD + 4 * c));
      }
    }
    __syncwarp();
    cluster_barrier();
  }
  // ---- this CTA's share of the tile, added up in rank order
  if constexpr (!GATED) {
    // a thread has a feature of four tokens at a time
    const int mine = max(0, min(own, min(features, p.M - m0) - sp * own));
    O* y = static_cast<O*>(p.y) + (size_t)t0 * p.ld_y + m0 + sp * own;
    for (int i = threadIdx.x; i < mine * fours; i += THREADS) {
      const int c = i / mine, g = i - c * mine;
      float4 v = *reinterpret_cast<const float4*>(received + g * LD + 4 * c);
#pragma unroll 1
      for (int r = 1; r < S; ++r) {
        const float4 u = *reinterpret_cast<const float4*>(received + (r * own + g) * LD + 4 * c);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      O* dst = y + (size_t)(4 * c) * p.ld_y + g;
      const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * c + e < tokens) dst[(size_t)e * p.ld_y] = from_f<O>(o[e]);
    }
  } else {
    // a warp has a token's 128 features, a block of the result's scales: a lane every 32nd.  The exponent as c1 z + c2 z^3 for both (fp8.cuh has the formulas)
    const int mine = max(0, min(own, tokens - sp * own)), ld = S > 1 ? own : LD;
    const float c1 = p.act == 2 ? -2.302208198f : -1.4426950408889634f, c2 = p.act == 2 ? -0.1029432396f : 0.f;
#pragma unroll 1
    for (int t = warp; t < mine; t += WARPS) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* from = received + (lane + 32 * j) * ld + t;
        float z = from[0], u = from[128 * ld];
#pragma unroll 1
        for (int r = 1; r < S; ++r) {
          z += from[r * 256 * ld];
          u += from[(r * 256 + 128) * ld];
        }
        const float x = z * fmaf(fminf(z * z, 1e30f), c2, c1);
        v[j] = (p.act == 1 ? (z < 0.f ? 0.f : z) : z * rcp_ftz(1.f + exp2_ftz(x))) * u;
        if (p.act != 1 && z < far_below(p.act)) v[j] = far_gated(z, x, u);
      }
      const float m = max16(max_abs(max_abs(v[0], v[1], v[2]), v[3]));
      const Scale k = scale_of(max_abs(m, __shfl_xor_sync(0xffffffffu, m, 16)));
      const uint32_t lo = codes2(v[0], v[1], k), hi = codes2(v[2], v[3], k);
      const int tok = t0 + sp * own + t;
      uint8_t* dst = p.codes + (size_t)tok * p.ld + m0 + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (m0 + lane + 32 * j < p.M) dst[32 * j] = (uint8_t)((j < 2 ? lo : hi) >> (8 * (j & 1)));
      if (lane == 0) p.scales[(size_t)(m0 / kBlock) * p.ld_s + tok] = k.s;
    }
  }
  if (threadIdx.x == 0) count_run_out(dead, p.err);  // (every wait lies before the barrier above)
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Clusters of 1, 2, 4 and 8 CTAs that the current device has at once, one CTA on an SM (a cluster lives inside one GPC, and GPCs differ): asked for once per device
cudaError_t clusters_at_once(const void* kern, cudaLaunchConfig_t cfg, cudaLaunchAttribute& size, int* out) {
  static std::atomic<uint64_t> known[64];  // by device: 16 bits each
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  uint64_t v = known[dev & 63].load(std::memory_order_acquire);
  if (v == 0) {
    cfg.dynamicSmemBytes = kSmemLeast;
    cfg.numAttrs = 1;
    for (int i = 0; i < 4; ++i) {
      int n = 0;
      size.val.clusterDim.x = 1 << i;
      cfg.gridDim = dim3(1 << i);
      if (const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg); e != cudaSuccess) return e;
      v |= (uint64_t)std::min(n, 0xffff) << (16 * i);
    }
    known[dev & 63].store(v, std::memory_order_release);
  }
  for (int i = 0; i < 4; ++i) out[i] = (int)(v >> (16 * i) & 0xffff);
  return cudaSuccess;
}

// Parts of K, features of a tile, stages, and about how many ns that takes: 4.5 us for the launch, the first copies and the end; a block of K as long as its bytes take (55 of them a ns and
// SM where all SMs stream) or its chain copy -> MMAs -> sum; the joining of a cluster 0.8 us and 20 bytes of a part a ns.  resident[i]: clusters of 2^i CTAs that the GPU has at once.
// The lowest tiles for which the number of waves stays, so that every SM has the same share.
FewPlan few_plan(int M, int N, int kb, int na, int nt, bool gated, const int* resident) {
  const int per_tile = gated ? kRows : na * kRows, n_tiles = (N + nt - 1) / nt;
  FewPlan best{};
  for (int i = 0; i < 4; ++i) {
    const int S = 1 << i;
    if (S > 1 && (S > kb / 2 || resident[i] < 1 || (!gated && na == 2))) continue;  // at least two blocks a part
    const int at_once = std::max(1, resident[i]);
    FewPlan p{kRows, S, 2, n_tiles, 0, 0, 0};
    const long tiles = (long)((M + per_tile - 1) / per_tile) * n_tiles;
    const long waves = (tiles + at_once - 1) / at_once;
    if (!gated) {
      const long m_tiles = std::max<long>(1, waves * at_once / n_tiles);  // that the waves have room for
      p.rows = (int)std::min<long>(kRows, std::max<long>(32, ((M + m_tiles * na - 1) / (m_tiles * na) + 7) / 8 * 8));
    }
    p.own = gated ? std::max(4, nt / S) : (na * p.rows + S - 1) / S;
    const int nk = (kb + S - 1) / S;
    while (p.stages < kMaxStages) {
      ++p.stages;
      if (few_smem(na, p, nt, gated) > (size_t)kSmemMost) {
        --p.stages;
        break;
      }
    }
    if (few_smem(na, p, nt, gated) > (size_t)kSmemMost) continue;
    const size_t part = (size_t)na * p.rows * part_ld(nt) * sizeof(float);  // over the ring
    const int hold = (int)((part + stage_bytes(na, p.rows, nt) - 1) / stage_bytes(na, p.rows, nt));
    if (hold > p.stages) continue;
    if (p.stages > nk) p.stages = std::max({nk, hold, 1});
    const double block = std::max(nt > 64 ? 400. : 300., (double)stage_bytes(na, p.rows, nt) / 55);
    p.ns = 4500 + (double)waves * (nk * block + (S > 1 ? 800 + (double)part / 20 : 0)) + (waves - 1) * 2500.;
    if (best.splits == 0 || p.ns < best.ns) best = p;
  }
  return best;
}

// within_ns: what another kernel takes; -2: that is the faster one
template <int NT, int NA, bool GATED, typename O>
int run_few(const Product& p, double within_ns, cudaStream_t st) {
  auto kern = fp8_gemm_few_kernel<NT, NA, GATED, O>;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kern, kSmemMost); e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(96 + 128 * groups(NA, NT));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  ThreadState& ts = tls();
  attr[1].val.programmaticStreamSerializationAllowed = ts.pdl ? 1 : 0;
  cfg.attrs = attr;
  int resident[4];
  if (const cudaError_t e = clusters_at_once((const void*)kern, cfg, attr[0], resident); e != cudaSuccess) return (int)e;
  const FewPlan plan = few_plan(p.M, p.N, p.kb, NA, NT, GATED, resident);
  if (plan.splits == 0 || plan.ns > within_ns) return -2;
  CUtensorMap mx, mw, mw2{};
  if (!make_codes_map(&mx, p.x, p.N, p.K, p.ld_x, NT) || !make_codes_map(&mw, p.w, p.M, p.K, p.ld_w, plan.rows) ||
      (GATED && !make_codes_map(&mw2, p.w2, p.M, p.K, p.ld_w, plan.rows)))
    return (int)cudaErrorInvalidValue;
  const int per_tile = GATED ? plan.rows : NA * plan.rows;
  ts.launches++;
  cfg.gridDim = dim3(plan.splits, (p.M + per_tile - 1) / per_tile * plan.n_tiles);
  cfg.dynamicSmemBytes = std::max(few_smem(NA, plan, NT, GATED), kSmemLeast);
  cfg.stream = st;
  attr[0].val.clusterDim.x = plan.splits;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, kern, mx, mw, mw2, p, plan);
}

}  // namespace

int launch_few(const Product& p, bool gated, bool y_f32, double within_ns, cudaStream_t st) {
  if (p.N > 1024 || (p.M + 31) / 32 * ((p.N + 63) / 64) > 65535) return -2;  // (tiles are counted on a grid's second axis)
  if (gated) {
    if (p.N <= 16) return run_few<16, 2, true, uint8_t>(p, within_ns, st);
    if (p.N <= 32) return run_few<32, 2, true, uint8_t>(p, within_ns, st);
    return run_few<64, 2, true, uint8_t>(p, within_ns, st);
  }
  auto go = [&](auto f, auto b) { return y_f32 ? f(p, within_ns, st) : b(p, within_ns, st); };
  if (p.M > kRows * sm_count()) {  // two tiles of features a CTA: fewer CTAs that read all of X
    if (p.N <= 16) return go(run_few<16, 2, false, float>, run_few<16, 2, false, bf16>);
    if (p.N <= 32) return go(run_few<32, 2, false, float>, run_few<32, 2, false, bf16>);
    return go(run_few<64, 2, false, float>, run_few<64, 2, false, bf16>);
  }
  if (p.N <= 16) return go(run_few<16, 1, false, float>, run_few<16, 1, false, bf16>);
  if (p.N <= 32) return go(run_few<32, 1, false, float>, run_few<32, 1, false, bf16>);
  if (p.N <= 64) return go(run_few<64, 1, false, float>, run_few<64, 1, false, bf16>);
  return go(run_few<128, 1, false, float>, run_few<128, 1, false, bf16>);
}

}  // namespace fp8
}  // namespace pk
