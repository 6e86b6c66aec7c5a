// The product of 8-bit rows and weights for prompts, on CTA pairs (fp8_gemm.cuh): y = x w^T, and act(x w^T) * (x w2^T) quantised again.
//
// A pair (cluster of two, tcgen05 cta_group::2) has a tile of 256 tokens x 256 features: A = X, 128 tokens to a CTA, B = W, half the features to a CTA.
//   warp 0     TMA producer (both CTAs): 128 entries of K a stage, completing on the leader's barrier
//   warp 1     MMA issuer (leader): a block of K is four tcgen05.mma (M 256, N 256, K 32) into one of two partial sums, all of tensor memory
//   warps 2, 3 the scales of even and odd blocks of K into shared memory, a token's times the weights'; they see a block's MMAs end and give its stage back
//   warps 4-19 take a partial sum out of tensor memory while the other is computed and add it, times its scale, to the tile's sum, which they hold in registers (thread = token, 64 features);
//              a finished tile leaves through shared memory by TMA
// Gated: B is 128 rows of w (leader) and the same 128 of w2 (peer), so a thread has 32 features of both; 128 features are a block of the result's scales, whose largest magnitude four threads
// find together.
//
// What bounds it, B200, 4096 tokens of 24576 x 4096 (825 GFLOP), us: 380 alone (2.17 PFLOP/s; 443 at the clocks of seconds under the power limit).  A block of K takes a tile 950 clocks, its
// MMAs 512.  Without the sums' work 312, with half of the operands' bytes 324, without both 244: a partial sum's way (MMAs, commit, 64 columns out and added by 16 warps, arrival in the other
// CTA: 1800 clocks, two of them under way) and the 32 KB a CTA reads of L2 for it (34 bytes a clock and SM) bound it together.  What it took to come here: 770 with a release at the cluster's scope in
// the arrivals, 479 with 8 warps that hold 128 columns, 399 with sums and addresses that did not fit registers, 380 with tiles that leave by TMA (3300 clocks a tile before).  Measured and not
// kept: halves of 128 columns with barriers of their own (A is read twice: 401), 16 columns at a time (428), packed fp32 products (equal), other orders of the tiles (389 to 431), 3 stages (386), 6
// (equal).
// Every barrier wait is bounded (mbar_wait_bounded, common.cuh).
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "fp8_gemm.cuh"

namespace pk {
namespace fp8 {

namespace {

constexpr int kBM = 128, kBN = 256, kHalf = kBN / 2;  // tokens per CTA; features of a tile, of a CTA's half of B
constexpr int kStages = 4;
constexpr int kEpi = 16;               // epilogue warps
constexpr int kPieceBytes = 32 * 128;  // of the output: 32 tokens x 128 bytes, an epilogue warp's at a time
constexpr int kThreads = 128 + 32 * kEpi;
constexpr int kABytes = kBM * kBK, kBBytes = kHalf * kBK, kStageBytes = kABytes + kBBytes;
// registers of a thread: the 65536 of an SM by 640 threads, then by role
constexpr int kRegsLaunch = 96, kRegsOther = 32, kRegsEpi = 112;
static_assert(128 * kRegsOther + 32 * kEpi * kRegsEpi <= kThreads * kRegsLaunch, "what the block was launched with");

constexpr int kLooks = 512;  // at a barrier before its wait proper, which wakes up 50 to 100 clocks later

struct Shared {  // behind the stages
  uint64_t full[kStages];    // used in the leader
  uint64_t empty[kStages];   // one per CTA, by the scales' warps
  uint64_t tfull[2];         // one per CTA: the MMAs' commit, the scales
  uint64_t tempty[2];        // used in the leader: an arrival per epilogue warp of both CTAs
  uint64_t done;             // behind a run-out: the MMAs under way
  uint32_t tmem;
  int dead;
  float scale[8][2][kBM];    // of eight blocks of K, by token: with the first 128 features and the second; gated: with w and w2
  float largest[2][4][kBM];  // gated: magnitudes of two tiles' rows, by 32 features
};
constexpr size_t kSmem = 227 * 1024;  // all of it: nobody else is resident on an SM whose tensor memory this kernel has (fp8_gemm_few.cu)
static_assert((size_t)kStages * kStageBytes + kEpi * kPieceBytes + 1024 + sizeof(Shared) <= kSmem, "shared memory of a CTA");

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

template <int ACT>
__device__ __forceinline__ void activate(const float* acc, float* v) {  // acc: 32 of the gate, 32 of the factor
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = gate_act<ACT>(acc[j]) * acc[32 + j];
}

// GATED: O is the codes' type
template <bool GATED, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
                const __grid_constant__ CUtensorMap map_y, const Product p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* pieces = smem + (size_t)kStages * kStageBytes;
  Shared& sh = *reinterpret_cast<Shared*>(pieces + kEpi * kPieceBytes);
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
    for (int s = 0; s < 2; ++s) {
      mbar_init(sh.tfull + s, 2);
      mbar_init(sh.tempty + s, 2 * kEpi);
    }
    mbar_init(&sh.done, 1);
    *dead = 0;
    mbar_fence_init();
  }
  if (warp == 1) g2_tmem_alloc(&sh.tmem, 2 * kBN);
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // both CTAs' barriers are initialised and both TMEM allocations are done
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem;
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
        for (int tile = pair; tile < num_tiles && go; tile += num_pairs) {
          const int mb = tile % m_tiles, nb = tile / m_tiles;
          const int tok0 = mb * 2 * kBM + (int)rank * kBM;
          const int row0 = GATED ? nb * kHalf : nb * kBN + (int)rank * kHalf;
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
        constexpr uint32_t idesc = f8_idesc(2 * kBM, kBN);
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
            const uint32_t d = tmem_base + (uint32_t)(buf * kBN);
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
            if (++buf == 2) {
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
      // Blocks of K as they come, tile behind tile, every second one, fetched one ahead.  A lane has four tokens.  Slot it % 8 held block it - 8: whoever gave back the partial sums of
      // block it - 4 had used it, and without those the MMAs of block it - 2, whose end is waited for here, did not begin.
      const int mine = warp - 2;
      int tile = pair, kb = mine;
      auto settle = [&]() {
        while (kb >= kb_n) {
          kb -= kb_n;
          tile += num_pairs;
        }
      };
      float4 x;
      float a, b;
      auto fetch = [&]() {  // (asm: where it stands)
        x = make_float4(0.f, 0.f, 0.f, 0.f);
        a = b = 0.f;
        if (tile >= num_tiles) return;
        const int nb = tile / m_tiles, tok = (tile - nb * m_tiles) * 2 * kBM + (int)rank * kBM + lane * 4;
        const int w0 = GATED ? nb : 2 * nb, w1 = GATED ? nb : (2 * nb + 1) * kBlock < M ? 2 * nb + 1 : 2 * nb;
        if (tok < N)  // (rows of scales are whole fours)
          asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(p.sx + (size_t)kb * p.ld_sx + tok));
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(a) : "l"(p.sw + (size_t)w0 * kb_n + kb));
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(b) : "l"((GATED ? p.sw2 : p.sw) + (size_t)w1 * kb_n + kb));
      };
      settle();
      fetch();
      uint32_t ph = 1;  // of tfull[mine]: before its first phase
      int stage = -1;   // of block it - 2
      for (int slot = mine; tile < num_tiles; slot = (slot + 2) & 7) {
        mbar_wait_bounded(sh.tfull + mine, ph, dead);
        if (lane == 0 && stage >= 0) mbar_arrive(sh.empty + stage);  // (the MMAs of block it - 2 have read it)
        stage = stage < 0 ? mine : stage + 2 < kStages ? stage + 2 : stage + 2 - kStages;
        reinterpret_cast<float4*>(sh.scale[slot][0])[lane] = make_float4(x.x * a, x.y * a, x.z * a, x.w * a);
        reinterpret_cast<float4*>(sh.scale[slot][1])[lane] = make_float4(x.x * b, x.y * b, x.z * b, x.w * b);
        __syncwarp();
        if (lane == 0) mbar_arrive(sh.tfull + mine);
        ph ^= 1u;
        kb += 2;
        settle();
        fetch();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int q = warp & 3, part = (warp - 4) >> 2, row = q * 32 + lane;
    const uint32_t tempty = g2_map(smem_u32(sh.tempty), 0), tfull = smem_u32(sh.tfull);
    const uint32_t scales = smem_u32(&sh.scale[0][GATED ? 0 : part >> 1][row]);
    // the thread's two pieces of 32 columns; gated: 32 of the gate, then the same 32 of the factor
    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * (GATED ? 32 : 64));
    constexpr uint32_t kPiece = GATED ? kHalf : 32;
    const uint32_t piece = smem_u32(pieces) + (uint32_t)((warp - 4) * kPieceBytes);
    uint32_t it = 0, lt = 0;  // blocks of K so far, tiles
    bool ready = false;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++lt) {
      float acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0.f;
#pragma unroll 1
      for (int kb = kb_n; kb > 0; --kb) {
        const uint32_t buf = it & 1;
        for (int i = 0; !ready && i < kLooks; ++i) ready = test_wait_at(tfull + buf * 8u, (it >> 1) & 1);
        if (!ready) mbar_wait_bounded(sh.tfull + buf, (it >> 1) & 1, dead);
        tc_fence_after();
        const uint32_t t0 = t_row + buf * kBN;
        uint32_t v[32];
        tmem_ld32_nowait(t0, v);
        const float s1 = ld_shared_at(scales + (it & 7) * (uint32_t)sizeof(sh.scale[0])), s2 = GATED ? ld_shared_at(scales + (it & 7) * (uint32_t)sizeof(sh.scale[0]) + kBM * 4) : s1;
        ++it;
        tmem_wait32(v);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[j] = fmaf(__uint_as_float(v[j]), s1, acc[j]);
        tmem_ld32_nowait(t0 + kPiece, v);
        ready = test_wait_at(tfull + (it & 1) * 8u, (it >> 1) & 1);  // (asked for early)
        tmem_wait32(v);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_relaxed(tempty + buf * 8u);
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[32 + j] = fmaf(__uint_as_float(v[j]), s2, acc[32 + j]);
      }
      const int mb = tile % m_tiles, nb = tile / m_tiles;
      const int tok = mb * 2 * kBM + (int)rank * kBM + row;
      const int f0 = GATED ? nb * kHalf + part * 32 : nb * kBN + part * 64;  // the thread's first feature
      if constexpr (GATED) {
        float v[32];
        if (p.act == 0) activate<0>(acc, v);
        else if (p.act == 1) activate<1>(acc, v);
        else activate<2>(acc, v);
        float m = max_abs(v[0], v[1]);
#pragma unroll
        for (int j = 2; j < 32; j += 2) m = max_abs(m, v[j], v[j + 1]);
        float(*mine)[kBM] = sh.largest[lt & 1];  // (the other tile's are read until the barrier behind this one)
        mine[part][row] = m;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpi) : "memory");
        const Scale k = scale_of(max_abs(max_abs(mine[0][row], mine[1][row], mine[2][row]), mine[3][row]));
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
          } else {  // rows that start anywhere: 32 entries of one at a time
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
    g2_tmem_dealloc(tmem_base, 2 * kBN);
  }
  if (threadIdx.x == 0) count_run_out(dead, p.err);
}

// rows x M of the output in pieces of 32 rows x 128 bytes; false: its rows do not start on 16-byte boundaries
template <typename O>
bool make_out_map(CUtensorMap* map, void* y, int rows, int M, long ld) {
  EncodeTiledFn fn = encode_fn();
  if (!fn || !al16(y) || ld * (long)sizeof(O) % 16 != 0 || ld * (long)sizeof(O) >= 1L << 40) return false;
  cuuint64_t dims[2] = {(cuuint64_t)M, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * sizeof(O)};
  cuuint32_t box[2] = {128 / sizeof(O), 32};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// about what a call takes here, in ns: 5.5 us for the launch and the first copies, 0.455 us a block of K, the end of a tile
double pair_ns(const Product& p, bool gated) {
  const double tiles = (double)((p.N + 2 * kBM - 1) / (2 * kBM)) * ((p.M + (gated ? kHalf : kBN) - 1) / (gated ? kHalf : kBN));
  return 5500 + std::ceil(tiles / std::max(1, sm_count() / 2)) * (p.kb * 455. + (gated ? 1500 : 700));
}

template <bool GATED, typename O>
int launch_pair(const Product& product, cudaStream_t st) {
  constexpr int features = GATED ? kHalf : kBN;
  Product p = product;
  const long tiles = (long)((p.N + 2 * kBM - 1) / (2 * kBM)) * ((p.M + features - 1) / features);
  const int pairs = (int)std::min<long>(std::max(1, sm_count() / 2), tiles);
  if (tiles > 0x7fffffffL - 4 * pairs) return -2;
  p.tiles = (int)tiles;
  auto kern = fp8_gemm_kernel<GATED, O>;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kern, kSmem); e != cudaSuccess) return (int)e;
  CUtensorMap mx, mw, mw2{}, my{};
  if (!make_codes_map(&mx, p.x, p.N, p.K, p.ld_x, kBM) || !make_codes_map(&mw, p.w, p.M, p.K, p.ld_w, kHalf) || (GATED && !make_codes_map(&mw2, p.w2, p.M, p.K, p.ld_w, kHalf)))
    return (int)cudaErrorInvalidValue;
  if constexpr (!GATED) p.y_map = make_out_map<O>(&my, p.y, p.N, p.M, p.ld_y);
  return (int)launch(kern, dim3(2 * pairs), dim3(kThreads), kSmem, st, true, mx, mw, mw2, my, p);
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
  if (const int rc = fp8::launch_few(p, false, y_f32, fp8::pair_ns(p, false), st); rc != -2) return rc;
  return y_f32 ? fp8::launch_pair<false, float>(p, st) : fp8::launch_pair<false, bf16>(p, st);
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
  if (const int rc = fp8::launch_few(p, true, false, fp8::pair_ns(p, true), st); rc != -2) return rc;
  return fp8::launch_pair<true, uint8_t>(p, st);
}
