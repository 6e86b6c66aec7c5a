// The product of 8-bit rows and weights for prompts, on CTA pairs (fp8_gemm.cuh): y = x w^T, and act(x w^T) * (x w2^T) quantised again.
//
// A pair (cluster of two, tcgen05 cta_group::2) has a tile of 256 tokens x 128, 192 or 256 features: A = X, 128 tokens to a CTA, B = W, half the features to a CTA.
//   warp 0     TMA producer (both CTAs): 128 entries of K a stage, completing on the leader's barrier
//   warp 1     MMA issuer (leader): a block of K is four tcgen05.mma (M 256, K 32) into one of two partial sums (128 features: of four), which have tensor memory
//   warps 2, 3 the scales of even and odd blocks of K into shared memory, a token's times the weights'; they see a block's MMAs end and give its stage back
//   the others (16, 12 or 8 warps) take a partial sum out of tensor memory while the next is computed and add it, times its scale, to the tile's sum, which they hold in registers
//              (thread = token, 64 features); a finished tile leaves through shared memory by TMA
// Gated: B is 128 rows of w (leader) and the same 128 of w2 (peer), so a thread has 32 features of both; 128 features are a block of the result's scales, whose largest magnitude four threads
// find together.
//
// What bounds it, B200, 4096 tokens of 24576 x 4096 (825 GFLOP), us: 372 alone (2.22 PFLOP/s; 436 at the clocks of seconds under the power limit).  A block of K takes a tile 930 clocks, its
// MMAs 512.  Without the sums' work 312, with half of the operands' bytes 324, without both 244: a partial sum's way (MMAs, commit, 64 columns out and added by 16 warps, arrival in the other
// CTA: 1800 clocks, two of them under way) and the 32 KB a CTA reads of L2 for it (34 bytes a clock and SM) bound it together.  What it took to come here: 770 with a release at the cluster's scope in
// the arrivals, 479 with 8 warps that hold 128 columns, 399 with sums and addresses that did not fit registers, 380 with tiles that leave by TMA (3300 clocks a tile before).  Measured and not
// kept: halves of 128 columns with barriers of their own (A is read twice: 401), 16 columns at a time (428), other orders of the tiles (389 to 431), 3 stages (386), 6
// (equal).  Tiles of 128, whose MMAs take 256 clocks a block, are at 460: 350 without the sums' work and with weights in L2; four partial sums carry them (with two 590), and so do 64 columns at once
// by 8 warps (32 by 16: 590).  Weights asked into L2 eight to 32 blocks ahead: equal.
// Every barrier wait is bounded (mbar_wait_bounded, common.cuh).
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "fp8_gemm.cuh"

namespace pk {
namespace fp8 {

namespace {

constexpr int kBM = 128;               // tokens per CTA
constexpr int kPieceBytes = 32 * 128;  // of the output: 32 tokens x 128 bytes, an epilogue warp's at a time
constexpr int kABytes = kBM * kBK;

constexpr int stages_of(int bn) { return bn == 256 ? 4 : bn == 192 ? 5 : 6; }
constexpr int epi_of(int bn) { return bn / 16; }             // epilogue warps
constexpr int sums_of(int bn) { return bn == 128 ? 4 : 2; }  // partial sums in tensor memory
constexpr int threads_of(int bn) { return 128 + 32 * epi_of(bn); }
// registers of a thread of a tile of 256: the 65536 of an SM by the threads, then by role (the others have enough for all, 128 and 168)
constexpr int kRegsLaunch = 96, kRegsOther = 32, kRegsEpi = 112;
static_assert(128 * kRegsOther + 32 * epi_of(256) * kRegsEpi <= threads_of(256) * kRegsLaunch, "what the block was launched with");
constexpr int stage_bytes_of(int bn) { return kABytes + bn / 2 * kBK; }

constexpr int kLooks = 512;  // at a barrier before its wait proper, which wakes up 50 to 100 clocks later

template <int STAGES, int SUMS>
struct Shared {  // behind the stages
  uint64_t full[STAGES];     // used in the leader
  uint64_t empty[STAGES];    // one per CTA, by the scales' warps
  uint64_t tfull[SUMS];      // one per CTA: the MMAs' commit, the scales
  uint64_t tempty[SUMS];     // used in the leader: an arrival per epilogue warp of both CTAs
  uint64_t done;             // behind a run-out: the MMAs under way
  uint32_t tmem;
  int dead;
  float scale[8][2][kBM];    // of eight blocks of K, by token: with the first 128 features and the second; gated: with w and w2
  float largest[2][4][kBM];  // gated: magnitudes of two tiles' rows, by 32 features
};
constexpr size_t kSmem = 227 * 1024;  // all of it: nobody else is resident on an SM whose tensor memory this kernel has (fp8_gemm_few.cu)

// An arrival without a release: what it reports are reads of tensor memory, complete and fenced (tcgen05.wait::ld, fence::before_thread_sync); no memory is handed over.  A release at the
// cluster's scope waits for the thread's loads in flight as well, 1500 to 2000 clocks for each block of K.
__device__ __forceinline__ void arrive_relaxed(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Shared memory by its 32-bit address: what a loop with 64 sums and 32 of what comes to them keeps beside those has to be little
__device__ __forceinline__ bool test_wait_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ float ld_shared_at(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// 128 bytes of a row (lane = row) into the warp's piece, laid out as a tensor map with 128-byte swizzle has it
__device__ __forceinline__ void put_row(uint32_t piece, int lane, const uint32_t* u) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece + (uint32_t)(lane * 128 + ((c ^ (lane & 7)) << 4))), "r"(u[4 * c]), "r"(u[4 * c + 1]), "r"(u[4 * c + 2]),
                 "r"(u[4 * c + 3])
                 : "memory");
}
__device__ __forceinline__ void store_piece(const CUtensorMap* map, uint32_t piece, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1), "r"(piece) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// A thread's 64 sums, two to an instruction or one.  B200, us, one : two: 512 tokens of 2560 x 9728 (tiles of 128) 24.5 : 23.3, gated 200 of 9728 x 2560 28.9 : 28.5; but in tiles of 192 and 256,
// whose registers are short for pairs side by side, 333 of 6144 x 2560 13.1 : 13.7, 4096 of 4096 x 4096 70.2 : 74.7
template <bool TWO>
struct Sums {
  float v[64];
  __device__ __forceinline__ Sums() {
#pragma unroll
    for (int j = 0; j < 64; ++j) v[j] = 0.f;
  }
  __device__ __forceinline__ void add(int at, const uint32_t* u, float scale) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[at + j] = fmaf(__uint_as_float(u[j]), scale, v[at + j]);
  }
  __device__ __forceinline__ float operator[](int j) const { return v[j]; }
};
template <>
struct Sums<true> {
  uint64_t v[32];
  __device__ __forceinline__ Sums() {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = 0;
  }
  __device__ __forceinline__ void add(int at, const uint32_t* u, float scale) {
    const uint64_t s = pair_of(scale, scale);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[at / 2 + j] = fma2(pair_of(u[2 * j], u[2 * j + 1]), s, v[at / 2 + j]);
  }
  __device__ __forceinline__ float operator[](int j) const { return j & 1 ? hi_of(v[j / 2]) : lo_of(v[j / 2]); }
};

template <int ACT>
__device__ __forceinline__ void activate(const float* acc, float* v) {  // acc: 32 of the gate, 32 of the factor
#pragma unroll
  for (int j = 0; j < 32; j += 8)
    if (__builtin_expect(gated8<ACT>(acc + j, acc + 32 + j, v + j), 0)) far_gated8<ACT>(acc + j, acc + 32 + j, v + j);
}

// BN: features of a tile; gated: 256, O is the codes' type
template <int BN, bool GATED, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threads_of(BN), 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
                const __grid_constant__ CUtensorMap map_y, const Product p) {
  constexpr int kHalf = BN / 2, kStages = stages_of(BN), kEpi = epi_of(BN), kSums = sums_of(BN), kStageBytes = stage_bytes_of(BN);
  constexpr bool kSplit = BN == 256;              // registers by role
  constexpr int kAtOnce = BN > 128 ? 32 : 64;    // columns of a partial sum that a thread has at once
  static_assert(!GATED || BN == 256, "a block of the result's scales");
  static_assert((size_t)kStages * kStageBytes + kEpi * kPieceBytes + 1024 + sizeof(Shared<kStages, kSums>) <= kSmem, "shared memory of a CTA");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* pieces = smem + (size_t)kStages * kStageBytes;
  Shared<kStages, kSums>& sh = *reinterpret_cast<Shared<kStages, kSums>*>(pieces + kEpi * kPieceBytes);
  volatile int* dead = &sh.dead;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int M = p.M, N = p.N, kb_n = p.kb;
  const int m_tiles = (N + 2 * kBM - 1) / (2 * kBM);
  const int num_tiles = p.tiles;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(sh.full + s, 1);
      mbar_init(sh.empty + s, 1);
    }
    for (int s = 0; s < kSums; ++s) {
      mbar_init(sh.tfull + s, 2);
      mbar_init(sh.tempty + s, 2 * kEpi);
    }
    mbar_init(&sh.done, 1);
    *dead = 0;
    mbar_fence_init();
  }
  if (warp == 1) g2_tmem_alloc(&sh.tmem, 512);
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers are initialised and both TMEM allocations are done
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem;
  pdl_wait();

  if (warp < 4) {
    if constexpr (kSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 0) {
      if (tc_elect_one()) {
        const CUtensorMap* mw = GATED && rank == 1 ? &map_w2 : &map_w;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(mw) : "memory");
        int s = 0;
        uint32_t ph = 1;
        bool go = true;
        for (int tile = pair; tile < num_tiles && go; tile += num_pairs) {
          const int mb = tile % m_tiles, nb = tile / m_tiles;
          const int tok0 = mb * 2 * kBM + (int)rank * kBM;
          const int row0 = GATED ? nb * kHalf : nb * BN + (int)rank * kHalf;
          for (int kb = 0; kb < kb_n; ++kb) {
            go = mbar_wait_bounded(sh.empty + s, ph, dead);
            if (!go) break;
            const uint32_t fb = g2_map(smem_u32(sh.full + s), 0);
            if (leader) mbar_expect_tx(sh.full + s, 2 * kStageBytes);
            uint8_t* st = smem + (size_t)s * kStageBytes;
            g2_tma_2d(st, &map_x, kb * kBK, tok0, fb);
            g2_tma_2d(st + kABytes, mw, kb * kBK, row0, fb);
            if (++s == kStages) {
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
        for (int tile = pair; tile < num_tiles && go; tile += num_pairs) {
          for (int kb = 0; kb < kb_n; ++kb) {
            // two looks at once: a wait costs this thread 200 clocks where nothing is to be waited for, a block's MMAs take 512
            const bool here = mbar_test_wait(sh.full + s, ph);
            bool free = mbar_test_wait(sh.tempty + buf, tph);
            if (!here) go = mbar_wait_bounded(sh.full + s, ph, dead);
            if (!go) break;
            const uint32_t a_addr = smem_u32(smem + (size_t)s * kStageBytes);
            const uint64_t adesc = make_sw128_desc(a_addr), bdesc = make_sw128_desc(a_addr + kABytes);
            const uint32_t d = tmem_base + (uint32_t)(buf * BN);
            for (int i = 0; !free && i < kLooks; ++i) free = mbar_test_wait(sh.tempty + buf, tph);
            if (!free) go = mbar_wait_bounded(sh.tempty + buf, tph, dead);
            if (!go) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k) umma_f8_pair(d, adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), idesc, k > 0 ? 1u : 0u);
            g2_commit_both(sh.tfull + buf);
            if (++s == kStages) {
              s = 0;
              ph ^= 1u;
            }
            if (++buf == kSums) {
              buf = 0;
              tph ^= 1u;
            }
          }
        }
        if (!go) {
          g2_commit_both(&sh.done);
          mbar_drain(&sh.done, 0);
        }
      }
    } else {
      // Blocks of K as they come, tile behind tile, every second one, fetched kAhead of them ahead (512 tokens of 2560 x 9728 in tiles of 128: one 31.7 us, two 26.0, three 24.6, four
      // 24.2).  A lane has four tokens.  Slot it % 8 held block it - 8: whoever gave back the partial sums of block it - 4 (it - 6 where there are four) had used it, and without those the
      // MMAs of block it - 2, whose end is waited for here, did not begin.
      constexpr int kAhead = BN == 256 ? 1 : BN == 192 ? 2 : 3;
      const int mine = warp - 2;
      int tile = pair, kb = mine;
      struct Next {
        float4 x;
        float a, b;
        bool there;
      } next[kAhead];
      auto fetch = [&](Next& n) {  // (asm: where it stands)
        while (kb >= kb_n) {
          kb -= kb_n;
          tile += num_pairs;
        }
        n.x = make_float4(0.f, 0.f, 0.f, 0.f);
        n.a = n.b = 0.f;
        n.there = tile < num_tiles;
        if (!n.there) return;
        const int nb = tile / m_tiles, tok = (tile - nb * m_tiles) * 2 * kBM + (int)rank * kBM + lane * 4;
        const int w0 = GATED ? nb : nb * BN / kBlock, w1 = GATED ? nb : (w0 + 1) * kBlock < M ? w0 + 1 : w0;
        if (tok < N)  // (rows of scales are whole fours)
          asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(n.x.x), "=f"(n.x.y), "=f"(n.x.z), "=f"(n.x.w) : "l"(p.sx + (size_t)kb * p.ld_sx + tok));
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(n.a) : "l"(p.sw + (size_t)w0 * kb_n + kb));
        if (BN > kBlock) asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(n.b) : "l"((GATED ? p.sw2 : p.sw) + (size_t)w1 * kb_n + kb));
        kb += 2;
      };
#pragma unroll
      for (int u = 0; u < kAhead; ++u) fetch(next[u]);
      uint32_t slot = mine, buf = mine, ph = 1;  // of this block; the phase of block it - 2's partial sum
      int stage = -1;                            // of block it - 2
      for (bool go = true; go;) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          Next& n = next[u];
          go = go && n.there;
          if (!go) break;
          mbar_wait_bounded(sh.tfull + (kSums == 2 ? buf : buf ^ 2), ph, dead);
          if (kSums == 2 || buf < 2) ph ^= 1u;
          if (lane == 0 && stage >= 0) mbar_arrive(sh.empty + stage);  // (the MMAs of block it - 2 have read it)
          stage = stage < 0 ? mine : stage + 2 < kStages ? stage + 2 : stage + 2 - kStages;
          reinterpret_cast<float4*>(sh.scale[slot][0])[lane] = make_float4(n.x.x * n.a, n.x.y * n.a, n.x.z * n.a, n.x.w * n.a);
          if (BN > kBlock) reinterpret_cast<float4*>(sh.scale[slot][1])[lane] = make_float4(n.x.x * n.b, n.x.y * n.b, n.x.z * n.b, n.x.w * n.b);
          __syncwarp();
          if (lane == 0) mbar_arrive(sh.tfull + buf);
          slot = (slot + 2) & 7;
          if (kSums == 4) buf ^= 2;
          fetch(n);
        }
      }
    }
  } else {
    if constexpr (kSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int q = warp & 3, part = (warp - 4) >> 2, row = q * 32 + lane;
    const uint32_t tempty = g2_map(smem_u32(sh.tempty), 0), tfull = smem_u32(sh.tfull);
    // its scales: its features are in the tile's first or second block of weights
    auto scales_of = [&](int half) { return smem_u32(&sh.scale[0][GATED ? 0 : (part + half) >> 1][row]); };
    uint32_t scales = scales_of(0);
    // the thread's two pieces of 32 columns; gated: 32 of the gate, then the same 32 of the factor
    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * (GATED ? 32 : 64));
    constexpr uint32_t kPiece = GATED ? kHalf : 32;
    const uint32_t piece = smem_u32(pieces) + (uint32_t)((warp - 4) * kPieceBytes);
    uint32_t it = 0, lt = 0;  // blocks of K so far, tiles
    bool ready = false;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++lt) {
      if (BN % kBlock) scales = scales_of(tile / m_tiles & 1);  // (a tile of 192 begins at a block or in the middle of one)
      Sums<GATED || BN == 128> sums;
#pragma unroll 1
      for (int kb = kb_n; kb > 0; --kb) {
        const uint32_t buf = it % kSums;
        for (int i = 0; !ready && i < kLooks; ++i) ready = test_wait_at(tfull + buf * 8u, it / kSums & 1);
        if (!ready) mbar_wait_bounded(sh.tfull + buf, it / kSums & 1, dead);
        tc_fence_after();
        const uint32_t t0 = t_row + buf * BN;
        uint32_t v[kAtOnce];
        tmem_ld32_nowait(t0, v);
        if constexpr (kAtOnce == 64) tmem_ld32_nowait(t0 + kPiece, v + 32);
        const float s1 = ld_shared_at(scales + (it & 7) * (uint32_t)sizeof(sh.scale[0])), s2 = GATED ? ld_shared_at(scales + (it & 7) * (uint32_t)sizeof(sh.scale[0]) + kBM * 4) : s1;
        ++it;
        if constexpr (kAtOnce == 32) {
          tmem_wait32(v);
          sums.add(0, v, s1);
          tmem_ld32_nowait(t0 + kPiece, v);
        }
        ready = test_wait_at(tfull + it % kSums * 8u, it / kSums & 1);  // (asked for early)
        tmem_wait32(v);
        if constexpr (kAtOnce == 64) tmem_wait32(v + 32);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_relaxed(tempty + buf * 8u);
        if constexpr (kAtOnce == 64) sums.add(0, v, s1);
        sums.add(32, v + kAtOnce - 32, s2);
      }
      float acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = sums[j];
      const int mb = tile % m_tiles, nb = tile / m_tiles;
      const int tok = mb * 2 * kBM + (int)rank * kBM + row;
      const int f0 = GATED ? nb * kHalf + part * 32 : nb * BN + part * 64;  // the thread's first feature
      if constexpr (GATED) {
        float v[32];
        if (p.act == 0) activate<0>(acc, v);
        else if (p.act == 1) activate<1>(acc, v);
        else activate<2>(acc, v);
        float m = max_abs(v[0], v[1]);
#pragma unroll
        for (int j = 2; j < 32; j += 2) m = max_abs(m, v[j], v[j + 1]);
        float(*largest)[kBM] = sh.largest[lt & 1];  // (the other tile's are read until the barrier behind this one)
        largest[part][row] = m;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpi) : "memory");
        const Scale k = scale_of(max_abs(max_abs(largest[0][row], largest[1][row], largest[2][row]), largest[3][row]));
        if (tok < N && f0 < M) {
          uint8_t* dst = p.codes + (size_t)tok * p.ld + f0;
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
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
          if (part == 0) p.scales[(size_t)nb * p.ld_s + tok] = k.s;
        }
      } else {
        O* y = static_cast<O*>(p.y);
        const int tok0 = tok - lane;
        constexpr int kCols = 128 / (int)sizeof(O);
#pragma unroll
        for (int c = 0; c < 64; c += kCols) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the piece before
          __syncwarp();
          uint32_t u[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) u[j] = sizeof(O) == 4 ? __float_as_uint(acc[c + j]) : pack_bf16(acc[2 * j], acc[2 * j + 1]);
          put_row(piece, lane, u);
          if (p.y_map) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && tok0 < N && f0 + c < M) store_piece(&map_y, piece, f0 + c, tok0);
          } else {  // rows that start or end anywhere: 32 entries of one at a time
            __syncwarp();
            const O* from = reinterpret_cast<const O*>(pieces + (warp - 4) * kPieceBytes);
            for (int r = 0; r < 32 && tok0 + r < N; ++r)
#pragma unroll
              for (int j = lane; j < kCols; j += 32) {
                const int byte = j * (int)sizeof(O);
                if (f0 + c + j < M)
                  y[(size_t)(tok0 + r) * p.ld_y + f0 + c + j] = from[(r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15)) / (int)sizeof(O)];
              }
            __syncwarp();
          }
        }
      }
    }
    if (!GATED && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // the peer's MMAs / loads may still target this CTA's shared memory and TMEM
  if (warp == 1) {
    tc_fence_after();
    g2_tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0) count_run_out(dead, p.err);
}

// rows x M of the output in pieces of 32 rows x 128 bytes; false: its rows do not start or end on 16-byte boundaries (a
// store that is clipped at the map's end writes whole 16 bytes)
template <typename O>
bool make_out_map(CUtensorMap* map, void* y, int rows, int M, long ld) {
  EncodeTiledFn fn = encode_fn();
  if (!fn || !al16(y) || ld * (long)sizeof(O) % 16 != 0 || M * (long)sizeof(O) % 16 != 0 || ld * (long)sizeof(O) >= 1L << 40) return false;
  cuuint64_t dims[2] = {(cuuint64_t)M, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * sizeof(O)};
  cuuint32_t box[2] = {128 / sizeof(O), 32};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// About what a call takes in tiles of bn features, in ns: 5.5 us for the launch and the first copies, a block of K of every tile, the end of a tile.  Narrow tiles have shorter blocks, wide ones
// less traffic for as much work, so the widths differ in how well their tiles fill the SMs.  B200, 256 : 192 : 128, us: 512 tokens of 2560 x 9728 38.9 : 31.5 : 24.6, 168 of 8192 x 4096 20.9 :
// 17.4 : 14.3, 333 of 6144 x 2560 15.1 : 13.0 : 15.4, 256 of 24576 x 4096 40.0 : 32.9 : 33.2, 1024 of 4096 x 4096 21.4 : 29.6 : 22.3, 426 of 16384 x 9728 82.3 : 90.2 : 91.0, 4096 of 24576 x 4096
// 372 : 393 : 405.  Of 50 drawn shapes the choice among these and the kernel for few tokens was within 3 % of the best at 42, 17 % behind at the worst (848 of 512 x 2560, 9.1 us).
double pair_ns(const Product& p, bool gated, int bn) {
  const int features = gated ? kBlock : bn;
  const double tiles = (double)((p.N + 2 * kBM - 1) / (2 * kBM)) * ((p.M + features - 1) / features);
  return 5500 + std::ceil(tiles / std::max(1, sm_count() / 2)) * (p.kb * (bn == 256 ? 455. : bn == 192 ? 345. : 250.) + (gated ? 1500 : 700));
}

template <int BN, bool GATED, typename O>
int launch_pair(const Product& product, cudaStream_t st) {
  constexpr int features = GATED ? kBlock : BN;
  Product p = product;
  const long tiles = (long)((p.N + 2 * kBM - 1) / (2 * kBM)) * ((p.M + features - 1) / features);
  const int pairs = (int)std::min<long>(std::max(1, sm_count() / 2), tiles);
  if (tiles > 0x7fffffffL - 4 * pairs) return -2;
  p.tiles = (int)tiles;
  auto kern = fp8_gemm_kernel<BN, GATED, O>;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kern, kSmem); e != cudaSuccess) return (int)e;
  CUtensorMap mx, mw, mw2{}, my{};
  if (!make_codes_map(&mx, p.x, p.N, p.K, p.ld_x, kBM) || !make_codes_map(&mw, p.w, p.M, p.K, p.ld_w, BN / 2) || (GATED && !make_codes_map(&mw2, p.w2, p.M, p.K, p.ld_w, BN / 2)))
    return (int)cudaErrorInvalidValue;
  if constexpr (!GATED) p.y_map = make_out_map<O>(&my, p.y, p.N, p.M, p.ld_y);
  return (int)launch(kern, dim3(2 * pairs), dim3(threads_of(BN)), kSmem, st, true, mx, mw, mw2, my, p);
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
  const double ns256 = fp8::pair_ns(p, false, 256), ns192 = fp8::pair_ns(p, false, 192), ns128 = fp8::pair_ns(p, false, 128), least = std::min({ns256, ns192, ns128});
  if (const int rc = fp8::launch_few(p, false, y_f32, least, st); rc != -2) return rc;
  if (ns128 == least) return y_f32 ? fp8::launch_pair<128, false, float>(p, st) : fp8::launch_pair<128, false, bf16>(p, st);
  if (ns192 == least) return y_f32 ? fp8::launch_pair<192, false, float>(p, st) : fp8::launch_pair<192, false, bf16>(p, st);
  return y_f32 ? fp8::launch_pair<256, false, float>(p, st) : fp8::launch_pair<256, false, bf16>(p, st);
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
  if (const int rc = fp8::launch_few(p, true, false, fp8::pair_ns(p, true, 256), st); rc != -2) return rc;
  return fp8::launch_pair<256, true, uint8_t>(p, st);
}
