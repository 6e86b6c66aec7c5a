// Attention over the 8-bit paged cache for prompts and prompt portions, on tcgen05 (kv8.cuh, kv8_attention.cuh).
//
// A CTA has two tiles of 128 rows of one kv head: the group's R query heads of 128 / R consecutive tokens each, so that a key is fetched once for the whole group and
// few scores lie behind the diagonal.  It goes through the keys in blocks of 64, run by run where its tokens belong to several requests (the other rows are masked).
//   * S = q K^T: K's codes are an operand as they lie in the cache (a record's K is two groups of 8 tokens of the canonical layout without swizzle, 8 x 16-byte matrices),
//     so plain bulk copies fill it.  kind::f8f6f4 wants 8 bits of q too, which has more: it goes in as two numbers, the nearest e4m3 and the rest as e5m2, whose exponents
//     reach 2^10 further down (4 + 1 + 3 significant bits; bf16 has 8), as many cycles as one product in 16 bits.  A row of q is scaled by a power of two to the upper
//     end of the codes' range: a bf16 entry is exact down to 2^-17 of the row's largest.
//   * O += P V in f16: the warps that rescale O turn a block's V into f16 (exactly) before, once for both tiles' 256 rows, which is an eighth of the instructions that
//     P in two 8-bit parts takes (B200, prompt of 4096, 32 heads in 8 groups: 240 us so).
//   * K's exponents multiply the scores 16 columns at a time, V's go into P's exponent: 2^(s - m + e - E + 7), m + E the row's largest s + e so far, so that what a row does not
//     see, or gives no weight, costs its other tokens no bits, however large its values; the denominator takes them out.
//   * Blocks of 64 keys with two S per tile: S of the block after next is issued behind P V of this one, so the softmax finds its scores waiting.  (Blocks of 128 with one S: a
//     tile waited 1600 of 5200 clocks for it.)
//   * m is a maximum of before that the row's own may have passed by up to 2^8: O, which stays in tensor memory, is rescaled only where one did by more.  P, held 2^7 times
//     too large, stays within f16's range then, with 11 bits down to 2^-21 of the largest weight.
// B200, prompt of 4096 tokens, 32 heads of 128 in 8 groups: 193 us, 0.71 PFLOP/s.  Bound by a softmax thread's latency: 1200 of 2500 clocks of a block of 64 keys (1.35 us) are its
// exponentials and P, 500 waits; a CTA takes 6.3 us to its first scores and 3.1 behind its last block.  Tried and slower: operands in the 128-byte swizzle (206), a degree-4 polynomial for a quarter of the
// exponentials (210), blocks of 128 keys (231).
// Warps: 0-3 softmax tile 0, a thread per row | 4-7 softmax tile 1 | 8-11 V, rescaling, results | 12, 13 MMA issuers | 14 copies | 15 nothing.  Of the block's registers a
// softmax thread has 192, the others 80 and 48.
// Tensor memory: tile 0's two S (64 columns each, P over the first 32) | tile 1's | O0 | O1.
#include <algorithm>

#include "kv8_attention.cuh"
#include "tcgen05.cuh"

namespace pk {
namespace kv8 {

constexpr int kPrRows = 128, kPrKeys = 64, kPrRecords = kPrKeys / kBlock;
constexpr int kPrStages = 4, kPrStagesV = 3;  // of K; of V as it comes and as f16
constexpr int kPrCorr = 8, kPrMma = 12, kPrLoad = 14, kPrThreads = 16 * 32;
constexpr int kPrRegsSoft = 192, kPrRegsCorr = 80, kPrRegsMma = 48;
static_assert(256 * kPrRegsSoft + 128 * kPrRegsCorr + 128 * kPrRegsMma <= kPrThreads * (65536 / kPrThreads), "more registers than the block was launched with");
constexpr int kPrTop = 7, kPrSlack = 8;  // exponents of P = 1 and of what a row's maximum may grow by before O is rescaled: 2^15 in f16
constexpr float kPrNone = -1000.f;  // E of a row that has seen nothing
constexpr uint32_t kRestA = 1u << 7;  // instruction descriptor: A is e5m2
constexpr int kPrMaxSeg = 256;     // runs that a CTA's tokens can belong to

struct PromptArgs {
  AttnArgs a;
  int per;           // tokens of a tile
  int each;          // blocks of a share, at least
  int q_by8, out_by8;
  unsigned int* err;
};

// whole numbers of a few bits: as a float, and two to them (-126 .. 127), in the ordinary pipes
__device__ __forceinline__ float small_float(int x) { return __int_as_float(0x4b400000 + x) - 12582912.f; }
__device__ __forceinline__ float whole_pow2(float x) { return __int_as_float(__float_as_int(x + (12582912.f + 127.f)) << 23); }
__device__ __forceinline__ void pr_fma2(float& x0, float& x1, float s, float c) {
  unsigned long long v, sv, cv;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x0), "f"(x1));
  asm("mov.b64 %0, {%1, %1};" : "=l"(sv) : "f"(s));
  asm("mov.b64 %0, {%1, %1};" : "=l"(cv) : "f"(c));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(v), "l"(sv), "l"(cv));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(v));
}
// operand without swizzle, inner dimension contiguous: 8 x 16-byte matrices of 128 bytes; lead: to the next one along the inner dimension, stride: to the next
// eight rows
__device__ __forceinline__ uint64_t plain_desc(uint32_t smem_addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((smem_addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)((stride >> 4) & 0x3fff) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// f16, A from tensor memory: lane = row, two consecutive inner elements a column
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pr_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// {a0, a1} += {x0, x1}
__device__ __forceinline__ void pr_add2(float& a0, float& a1, float x0, float x1) {
  unsigned long long v, w;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a0), "f"(a1));
  asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(x0), "f"(x1));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(w));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(v));
}
// four bf16 times a power of two (448 at most) -> the nearest e4m3 and the rests as e5m2.  f16 holds them exactly but below 2^-14, and there to 2^-25.
__device__ __forceinline__ void q_parts(uint32_t w0, uint32_t w1, float down, uint32_t& near, uint32_t& rest) {
  const uint32_t h0 = pack_f16(bf16_lo(w0) * down, bf16_hi(w0) * down), h1 = pack_f16(bf16_lo(w1) * down, bf16_hi(w1) * down);
  uint16_t c[2], d[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    asm("{\n\t.reg .b32 b;\n\t"
        "cvt.rn.satfinite.e4m3x2.f16x2 %0, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 b, %0;\n\t"
        "sub.rn.f16x2 b, %2, b;\n\t"
        "cvt.rn.satfinite.e5m2x2.f16x2 %1, b;\n\t}"
        : "=&h"(c[i]), "=&h"(d[i])
        : "r"(i ? h1 : h0));
  near = (uint32_t)c[0] | (uint32_t)c[1] << 16;
  rest = (uint32_t)d[0] | (uint32_t)d[1] << 16;
}

// CUT: the keys of a tile are cut into shares
template <int D, bool CUT>
__global__ void __launch_bounds__(kPrThreads, 1) kv8_prompt_kernel(const bf16* __restrict__ q, const bf16* __restrict__ sink, bf16* __restrict__ out, const PromptArgs f) {
  constexpr int QB = kPrRows * D, KB = kPrKeys * D, REC_K = kBlock * D;  // bytes of a part of q's tile, of a stage's K (or V), of a record's K
  extern __shared__ uint8_t pr_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pr_raw) + 127) & ~(uintptr_t)127);
  uint8_t* Qs = smem;                                    // [tile][hi, lo]
  uint8_t* Ks = Qs + 4 * QB;                             // [stage]
  uint8_t* Vs = Ks + kPrStages * KB;                     // [stage] V as it comes
  uint8_t* Hs = Vs + kPrStagesV * KB;                    // [stage] V as f16: [8 keys][entry][8 keys' f16]
  uint8_t* Ts = Hs + kPrStagesV * 2 * KB;                // [stage][record] tails as they come
  uint32_t* Es = reinterpret_cast<uint32_t*>(Ts + kPrStagesV * kPrRecords * 16);  // [stage][record] tails of the f16's
  float* alpha_s = reinterpret_cast<float*>(Es + kPrStagesV * kPrRecords);  // [tile][buffer][row]
  float* end_s = alpha_s + 4 * kPrRows;                  // [tile][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(end_s + 2 * kPrRows);
  uint64_t *k_full = bars, *k_empty = bars + 4, *v_full = bars + 8, *v_empty = bars + 11, *h_full = bars + 14, *h_empty = bars + 17;  // [stage]
  uint64_t* s_full = bars + 20;    // [tile][buffer] S complete                       MMA -> softmax
  uint64_t* po_ready = bars + 24;  // [tile][buffer] P stored, O rescaled (4 + 4 warps)  softmax, rescaling -> MMA
  uint64_t* a_ready = bars + 28;   // [tile][buffer] factors of O published (4 warps)    softmax -> rescaling
  uint64_t* pv_done = bars + 32;   // [tile][buffer] P V complete                      MMA -> rescaling
  uint64_t* d_ready = bars + 36;   // [tile] last factors published (4 warps)           softmax -> results
  uint64_t* done = bars + 38;      // behind a run-out: the MMAs under way
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 39);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_req[2 * kPrRows], s_slot[2 * kPrRows], s_seg[2 * kPrRows];
  __shared__ int seg_off[kPrMaxSeg], seg_lo[2][kPrMaxSeg], seg_hi[2][kPrMaxSeg];  // page table of a run; blocks of keys that its rows of a tile see
  __shared__ int s_count[kPrThreads / 32], s_segs;

  const AttnArgs& a = f.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = blockIdx.y, R = a.H / a.pool.G, per = f.per;
  const int t0 = ((int)gridDim.z - 1 - (int)blockIdx.z) * 2 * per, n_tok = min(2 * per, a.T - t0);  // late tokens, which see most, first

  if (tid == 0) {
    for (int s = 0; s < kPrStages; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 2);  // both tiles
    }
    for (int s = 0; s < kPrStagesV; ++s) {
      mbar_init(v_full + s, 1);
      mbar_init(v_empty + s, 4);  // the warps that turn it into f16
      mbar_init(h_full + s, 4);
      mbar_init(h_empty + s, 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(po_ready + i, 8);
      mbar_init(a_ready + i, 4);
      mbar_init(pv_done + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(d_ready + i, 4);
    }
    mbar_init(done, 2);
    *dead = 0;
    mbar_fence_init();
  }
  if (warp == kPrMma) tmem_alloc(tmem_slot, 512);
  pdl_wait();
  pdl_launch_dependents();

  // a softmax thread's row of q: under way while the runs are looked up
  uint4 raw[D / 8];
  if (warp < kPrCorr) {
    const int r = tid & 127, k = r / R, ti = (warp >> 2) * per + k;
    const bool on = k < per && ti < n_tok;
    const bf16* src = q + ((size_t)(t0 + (on ? ti : 0)) * a.H + g * R + (on ? r - k * R : 0)) * D;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      raw[c] = make_uint4(0, 0, 0, 0);
      if (!on) continue;
      if (f.q_by8) {
        raw[c] = *reinterpret_cast<const uint4*>(src + c * 8);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = (uint32_t)__bfloat16_as_ushort(src[c * 8 + 2 * x]) | (uint32_t)__bfloat16_as_ushort(src[c * 8 + 2 * x + 1]) << 16;
        raw[c] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }

  // ---- the runs that the tokens belong to
  for (int i = tid; i < kPrMaxSeg; i += kPrThreads)
    for (int k = 0; k < 2; ++k) {
      seg_lo[k][i] = INT_MAX;
      seg_hi[k][i] = -1;
    }
  bool begins = false;
  int my_req = 0, my_slot = -1;
  if (tid < n_tok) {
    my_req = a.req[t0 + tid];
    my_slot = a.slots[t0 + tid];
    begins = tid == 0 || a.req[t0 + tid - 1] != my_req;
    s_req[tid] = my_req;
    s_slot[tid] = my_slot;
  }
  const uint32_t starts = __ballot_sync(0xffffffffu, begins);
  if (lane == 0) s_count[warp] = __popc(starts);
  __syncthreads();
  {
    int before = 0;
    for (int w = 0; w < warp; ++w) before += s_count[w];
    const int seg = before + __popc(starts & (0xffffffffu >> (31 - lane))) - 1;
    if (tid < n_tok) {
      s_seg[tid] = seg;
      if (my_slot >= 0) {
        const int tile = tid >= per, lo = a.window > 0 ? max(0, my_slot - a.window + 1) : 0;
        atomicMin(&seg_lo[tile][seg], lo / kPrKeys);
        atomicMax(&seg_hi[tile][seg], my_slot / kPrKeys);
        seg_off[seg] = a.pool.page_off[my_req];  // (the same from every token of the run)
      }
    }
    if (tid == 0) {
      int all = 0;
      for (int w = 0; w < kPrThreads / 32; ++w) all += s_count[w];
      s_segs = all;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int segs = s_segs;
  WaitTries tries;
  auto first_block = [&](int seg) { return min(seg_lo[0][seg], seg_lo[1][seg]); };
  auto last_block = [&](int seg) { return max(seg_hi[0][seg], seg_hi[1][seg]); };
  auto needs = [&](int tile, int seg, int j) { return j >= seg_lo[tile][seg] && j <= seg_hi[tile][seg]; };
  // the blocks of all runs in order, the same for every role
  struct Step {
    int seg, j, n;  // n: blocks before it
  };
  auto settle = [&](Step& x) {  // on to a run that has a block
    while (x.seg < segs && last_block(x.seg) < 0) ++x.seg;
    if (x.seg < segs) x.j = first_block(x.seg);
  };
  auto pass = [&](Step& x) {
    if (x.j < last_block(x.seg)) {
      ++x.j;
    } else {
      ++x.seg;
      settle(x);
    }
  };
  // this CTA's share of them (the grid's x axis, so that a tile's CTAs without one leave early), counted from its own first
  int share = INT_MAX;
  Step origin{0, 0, 0};
  if constexpr (!CUT) {
    settle(origin);
  } else {
    int all = 0;
    for (int k = 0; k < segs; ++k)
      if (last_block(k) >= 0) all += last_block(k) - first_block(k) + 1;
    const int each = max(f.each, (all + (int)gridDim.x - 1) / (int)gridDim.x), skip = (int)min((long)each * blockIdx.x, (long)all);
    share = min(each, all - skip);
    if (share == 0) {  // (for all threads alike)
      const int r = tid & 127, k = r / R, ti = (tid >> 7) * per + k;
      if (tid < 2 * kPrRows && k < per && ti < n_tok) a.part_ml[((size_t)blockIdx.x * a.T + t0 + ti) * a.H + g * R + r - k * R] = make_float2(-INFINITY, 0.f);
      if (warp == kPrMma) tmem_dealloc(tmem_base, 512);
      return;
    }
    settle(origin);
    for (int k = 0; k < skip;) {  // run by run
      const int here = last_block(origin.seg) - origin.j + 1, go = min(here, skip - k);
      k += go;
      if (go < here) {
        origin.j += go;
      } else {
        ++origin.seg;
        settle(origin);
      }
    }
  }
  auto begin = [&] { return origin; };
  auto next = [&](Step& x) {
    ++x.n;
    if (CUT && x.n == share) x.seg = segs;
    else pass(x);
  };

  if (warp >= kPrMma) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrRegsMma));
  if (warp == kPrLoad) {
    // =========================== copies ===========================
    bool go = true;  // false behind a run-out: a barrier must not be armed twice in one phase
    const int rpp = a.pool.page_size / kBlock;
    int seg = -1, top = 0, off = 0;
    auto source = [&](const Step& x) {  // lane i: the block's i-th record, the run's last one again behind the end
      if (x.seg != seg) {
        seg = x.seg;
        top = -1;  // the last slot that anybody here has: records behind it may not exist
        for (int i = lane; i < n_tok; i += 32)
          if (s_seg[i] == seg) top = max(top, s_slot[i]);
        top = __reduce_max_sync(0xffffffffu, top) / kBlock;
        off = seg_off[seg];
      }
      const int b = min(x.j * kPrRecords + min(lane, kPrRecords - 1), top);
      return a.pool.data + (size_t)a.pool.pages[off + b / rpp] * a.pool.page_stride + (size_t)(g * rpp + b % rpp) * (2 * REC_K + 16);
    };
    Step x = begin();
    const uint8_t* src = x.seg < segs ? source(x) : nullptr;
    while (x.seg < segs && go) {
      const int n = x.n, s = n % kPrStages, sv = n % kPrStagesV;
      const uint8_t* now = src;
      next(x);
      if (x.seg < segs) src = source(x);  // its page is looked up under this block's waits
      go = mbar_wait_bounded(k_empty + s, (uint32_t)((n / kPrStages) & 1) ^ 1u, dead, tries);
      if (!go) break;
      if (lane == 0) mbar_expect_tx(k_full + s, KB);
      __syncwarp();
      if (lane < kPrRecords) pr_copy(smem_u32(Ks + s * KB) + lane * REC_K, now, REC_K, k_full + s);
      go = mbar_wait_bounded(v_empty + sv, (uint32_t)((n / kPrStagesV) & 1) ^ 1u, dead, tries);
      if (!go) break;
      if (lane == 0) mbar_expect_tx(v_full + sv, KB + kPrRecords * 16);
      __syncwarp();
      if (lane < kPrRecords) {
        pr_copy(smem_u32(Vs + sv * KB) + lane * REC_K, now + REC_K, REC_K, v_full + sv);
        pr_copy(smem_u32(Ts + (sv * kPrRecords + lane) * 16), now + 2 * REC_K, 16, v_full + sv);
      }
    }
    if (!go) wait_for_copies();
  } else if (warp < kPrLoad) {
    // =========================== MMA issuers, one per tile ===========================
    const int i = warp - kPrMma;
    asm volatile("bar.sync 1, %0;" ::"n"(10 * 32) : "memory");  // q is there
    constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kPrKeys >> 3) << 17) | ((uint32_t)(kPrRows >> 4) << 24);  // e4m3 x e4m3 -> fp32, both inner-contiguous
    constexpr uint32_t idesc_pv = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kPrRows >> 4) << 24);
    const uint64_t q_hi = plain_desc(smem_u32(Qs + i * 2 * QB), 128, 8 * D), q_lo = plain_desc(smem_u32(Qs + (i * 2 + 1) * QB), 128, 8 * D);
    const uint32_t t_s = tmem_base + (uint32_t)(i * 2 * kPrKeys), t_o = tmem_base + (uint32_t)(4 * kPrKeys + i * 128);
    int issued = 0, finished = 0, waiting[2] = {0, 0};  // this tile's blocks: S issued, P V issued; the stages of V of those between
    auto finish = [&] {
      const int sv = waiting[finished & 1] % kPrStagesV;
      mbar_wait_bounded(h_full + sv, (uint32_t)((waiting[finished & 1] / kPrStagesV) & 1), dead, tries);
      mbar_wait_bounded(po_ready + i * 2 + (finished & 1), (uint32_t)((finished >> 1) & 1), dead, tries);
      tc_fence_after();
      const uint64_t v_desc = plain_desc(smem_u32(Hs + sv * 2 * KB), REC_K, 128);  // 8 keys x 8 entries
      const uint32_t t_p = t_s + (uint32_t)((finished & 1) * kPrKeys);
      if (tc_elect_one()) {
#pragma unroll
        for (int k = 0; k < kPrKeys / 16; ++k)
          umma_f16_ts(t_o, t_p + (uint32_t)(k * 8), v_desc + (uint64_t)(k * (2 * REC_K >> 4)), idesc_pv, (finished > 0 || k > 0) ? 1u : 0u);
        umma_commit(pv_done + i * 2 + (finished & 1));
        umma_commit(h_empty + sv);
      }
      __syncwarp();
      ++finished;
    };
    for (Step x = begin(); x.seg < segs; next(x)) {
      const int s = x.n % kPrStages, sv = x.n % kPrStagesV;
      const uint32_t ph = (uint32_t)((x.n / kPrStages) & 1);
      if (!needs(i, x.seg, x.j)) {  // not this tile's: its arrivals, each in its phase
        while (finished < issued) finish();  // (the copies of later blocks wait for them)
        mbar_wait_bounded(k_full + s, ph, dead, tries);
        if (lane == 0) mbar_arrive(k_empty + s);
        mbar_wait_bounded(h_full + sv, (uint32_t)((x.n / kPrStagesV) & 1), dead, tries);
        if (lane == 0) mbar_arrive(h_empty + sv);
        __syncwarp();
        continue;
      }
      if (issued - finished == 2) finish();  // its S and P lie where the next S goes
      mbar_wait_bounded(k_full + s, ph, dead, tries);
      tc_fence_after();
      const uint64_t k_desc = plain_desc(smem_u32(Ks + s * KB), 128, 8 * D);
      const uint32_t t_d = t_s + (uint32_t)((issued & 1) * kPrKeys);
      if (tc_elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          umma_f8(t_d, q_hi + (uint64_t)(k * 16), k_desc + (uint64_t)(k * 16), idesc_s, k > 0 ? 1u : 0u);
          umma_f8(t_d, q_lo + (uint64_t)(k * 16), k_desc + (uint64_t)(k * 16), idesc_s | kRestA, 1u);
        }
        umma_commit(s_full + i * 2 + (issued & 1));
        umma_commit(k_empty + s);
      }
      __syncwarp();
      waiting[issued & 1] = x.n;
      ++issued;
    }
    while (finished < issued) finish();
  }
  } else if (warp >= kPrCorr) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrRegsCorr));
    // =========================== rescaling of O, results ===========================
    const int q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t lane_base = tmem_base + ((uint32_t)(q4 * 32) << 16);
    int mine[2] = {0, 0};
    auto widen_v = [&](int n) {  // the V of block n: a thread takes an entry's 16 keys of a record at a time
      const int sv = n % kPrStagesV;
      const uint32_t phv = (uint32_t)((n / kPrStagesV) & 1);
      mbar_wait_bounded(v_full + sv, phv, dead, tries);
      mbar_wait_bounded(h_empty + sv, phv ^ 1u, dead, tries);
      const uint8_t* from = Vs + sv * KB;
      uint8_t* to = Hs + sv * 2 * KB;
#pragma unroll 4
      for (int u = r; u < kPrRecords * D; u += 128) {
        const int b = u / D, d = u - b * D;
        const uint4 x = *reinterpret_cast<const uint4*>(from + u * 16);
        uint32_t h[8];
        widen(x.x, h[0], h[1]);
        widen(x.y, h[2], h[3]);
        widen(x.z, h[4], h[5]);
        widen(x.w, h[6], h[7]);
        *reinterpret_cast<uint4*>(to + (2 * b) * REC_K + d * 16) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(to + (2 * b + 1) * REC_K + d * 16) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      if (r < kPrRecords) Es[sv * kPrRecords + r] = *reinterpret_cast<const uint32_t*>(Ts + (sv * kPrRecords + r) * 16);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(h_full + sv);
        mbar_arrive(v_empty + sv);
      }
    };
    // O holds all blocks before this one.  (Only waited for where somebody needs it: of a buffer's phases at most the last is not over by then, since S of the block
    // before this one came behind the P V before it.)
    auto all_added = [&](int i) {
      if (mine[i] > 0) mbar_wait_bounded(pv_done + i * 2 + ((mine[i] - 1) & 1), (uint32_t)(((mine[i] - 1) >> 1) & 1), dead, tries);
    };
    Step ahead = begin();
    if (ahead.seg < segs) {
      widen_v(0);
      next(ahead);
    }
    for (Step x = begin(); x.seg < segs; next(x)) {
      if (ahead.seg < segs) {  // a block ahead of the softmax
        widen_v(ahead.n);
        next(ahead);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!needs(i, x.seg, x.j)) continue;
        const int at = i * 2 + (mine[i] & 1);
        mbar_wait_bounded(a_ready + at, (uint32_t)((mine[i] >> 1) & 1), dead, tries);
        const float alpha = alpha_s[at * kPrRows + r];
        if (mine[i] > 0) {
          if (!__all_sync(0xffffffffu, alpha == 1.0f)) {
            all_added(i);
            tc_fence_after();
            const uint32_t t_o = lane_base + (uint32_t)(4 * kPrKeys + i * 128);
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              uint32_t t[32];
              tmem_ld32(t_o + c, t);
#pragma unroll
              for (int k = 0; k < 32; ++k) t[k] = __float_as_uint(__uint_as_float(t[k]) * alpha);
              tmem_put32(t_o + c, t);
            }
            tmem_put_wait();
            tc_fence_before();
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(po_ready + at);
        ++mine[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_wait_bounded(d_ready + i, 0, dead, tries);
      all_added(i);
      tc_fence_after();
      const int k = r / R, ti = i * per + k;
      const bool on = k < per && ti < n_tok;
      const float factor = end_s[i * kPrRows + r];
      bf16* dst = out + (size_t)(t0 + (on ? ti : 0)) * a.out_ld + (g * R + (on ? r - k * R : 0)) * D;
      const uint32_t t_o = lane_base + (uint32_t)(4 * kPrKeys + i * 128);
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t t[32];
        if (mine[i] > 0) {
          tmem_ld32(t_o + c, t);
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) t[x] = 0u;
        }
        if (!on) continue;
#pragma unroll
        for (int x = 0; x < 32; ++x) t[x] = __float_as_uint(__uint_as_float(t[x]) * factor);
        if constexpr (CUT) {
          float* part = a.part_o + (((size_t)blockIdx.x * a.T + t0 + ti) * a.H + g * R + r - k * R) * D + c;
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            *reinterpret_cast<uint4*>(part + x) = make_uint4(t[x], t[x + 1], t[x + 2], t[x + 3]);
        } else if (f.out_by8) {
#pragma unroll
          for (int x = 0; x < 32; x += 8)
            *reinterpret_cast<uint4*>(dst + c + x) = make_uint4(pack_bf16(__uint_as_float(t[x]), __uint_as_float(t[x + 1])), pack_bf16(__uint_as_float(t[x + 2]), __uint_as_float(t[x + 3])),
                                                                pack_bf16(__uint_as_float(t[x + 4]), __uint_as_float(t[x + 5])), pack_bf16(__uint_as_float(t[x + 6]), __uint_as_float(t[x + 7])));
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) dst[c + x] = f2bf(__uint_as_float(t[x]));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrRegsSoft));
    // =========================== softmax: a thread per row ===========================
    const int i = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane, k = r / R, ti = i * per + k;
    const bool on = k < per && ti < n_tok;
    const int h = g * R + (on ? r - k * R : 0);
    const int p = on ? s_slot[ti] : -1, lo = on && a.window > 0 ? p - a.window + 1 : 0, my_seg = on ? s_seg[ti] : -1;
    // q: scaled to the codes' upper end, split, into the operands
    float row_c;
    {
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[x])), fabsf(bf16_hi(w[x]))));
      }
      const int e = exponent_for(amax);
      // scale's sign goes into q: maxima are taken before the columns' factors, which have to be positive
      const float down = a.scale < 0.f ? -pow2(-e) : pow2(-e), qf = amax == INFINITY ? NAN : pow2(e);  // (an infinite entry: the row is NaN)
      row_c = a.cap > 0.f ? qf : qf * fabsf(a.scale) * kLog2e;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t hi[4], rest[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint4 u = raw[2 * c + (x >> 1)];
          q_parts(x & 1 ? u.z : u.x, x & 1 ? u.w : u.y, down, hi[x], rest[x]);
        }
        uint8_t* dst = Qs + i * 2 * QB + (r >> 3) * (8 * D) + c * 128 + (r & 7) * 16;
        *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + QB) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync 1, %0;" ::"n"(10 * 32) : "memory");

    const uint32_t t_tile = tmem_base + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(i * 2 * kPrKeys);
    const float cap2 = a.cap * kLog2e, cap_c = a.cap > 0.f ? 2.f * fabsf(a.scale) / a.cap * kLog2e : 0.f;
    float m = -INFINITY, l = 0.f, E = kPrNone;  // l is held relative to 2^m, O to 2^(m + E); both are whole numbers, so that every rescaling is exact
    int mine = 0;
    for (Step x = begin(); x.seg < segs; next(x)) {
      if (!needs(i, x.seg, x.j)) continue;
      const int sv = x.n % kPrStagesV;
      const uint32_t t_s = t_tile + (uint32_t)((mine & 1) * kPrKeys);
      // S first: it says that the stage's phases before this block's are over (a tile that skipped blocks would take an older one for it)
      mbar_wait_bounded(s_full + i * 2 + (mine & 1), (uint32_t)((mine >> 1) & 1), dead, tries);
      tc_fence_after();
      uint32_t v[kPrKeys];
      tmem_ld32_nowait(t_s, v);
      tmem_ld32_nowait(t_s + 32, v + 32);
      mbar_wait_bounded(h_full + sv, (uint32_t)((x.n / kPrStagesV) & 1), dead, tries);
      float ev[kPrRecords], fk[kPrRecords];
#pragma unroll
      for (int b = 0; b < kPrRecords; ++b) {
        const uint32_t tail = Es[sv * kPrRecords + b];
        ev[b] = small_float(tail_ev(tail));
        const float y = pow2(tail_ek(tail)) * row_c;
        fk[b] = y < 1e-37f ? 1e-37f : y;  // never zero: -inf times it stays -inf (and a NaN stays one)
      }
      const int c0 = my_seg == x.seg ? max(lo - x.j * kPrKeys, 0) : kPrKeys, c1 = my_seg == x.seg ? min(p - x.j * kPrKeys, kPrKeys - 1) : -1;  // the columns that the row sees
      const bool masked = !__all_sync(0xffffffffu, c0 <= 0 && c1 >= kPrKeys - 1);
      auto factor = [&](int b) { return a.cap > 0.f ? 1.f : fk[b]; };
      tmem_ld_wait64(v);
      if (a.cap > 0.f) {  // (the columns' factors are in the scores then)
#pragma unroll
        for (int k = 0; k < kPrKeys; ++k)
          v[k] = __float_as_uint(fmaf(-2.f * cap2, __fdividef(1.f, ex2(at_most80(__uint_as_float(v[k]) * fk[k / kBlock] * cap_c)) + 1.f), cap2));
      }
      if (masked) {
#pragma unroll
        for (int k = 0; k < kPrKeys; ++k)
          if (k < c0 || k > c1) v[k] = 0xff800000u;
      }
      float mx = m, high = -INFINITY;  // largest score, and with V's exponent added
#pragma unroll
      for (int b = 0; b < kPrRecords; ++b) {
        float y = fmaxf(__uint_as_float(v[b * 16]), __uint_as_float(v[b * 16 + 1])), z = fmaxf(__uint_as_float(v[b * 16 + 2]), __uint_as_float(v[b * 16 + 3]));
#pragma unroll
        for (int k = 4; k < 16; k += 4) {
          y = fmaxf(fmaxf(y, __uint_as_float(v[b * 16 + k])), __uint_as_float(v[b * 16 + k + 1]));
          z = fmaxf(fmaxf(z, __uint_as_float(v[b * 16 + k + 2])), __uint_as_float(v[b * 16 + k + 3]));
        }
        y = fmaxf(y, z) * factor(b);
        mx = fmaxf(mx, y);
        high = fmaxf(high, y + ev[b]);
      }
      const float m_new = mx > m + (float)kPrSlack ? ceilf(mx) : m;  // (m = -inf: mx)
      const float ref = m_new == -INFINITY ? 0.f : m_new, grown = m == -INFINITY ? 0.f : fminf(m_new - m, 2000.f);
      high = fmaf(fabsf(ref), 1.2e-7f, high - ref);  // (and what its sum was rounded by, so that P stays in range)
      const float E_old = E - grown, E_new = high > E_old + (float)kPrSlack ? ceilf(high) : E_old;
      // (a row that saw nothing so far has nothing in O; nothing is rescaled at the first block)
      alpha_s[(i * 2 + (mine & 1)) * kPrRows + r] = m == -INFINITY ? 1.f : whole_pow2(fmaxf(E_old - E_new, -126.f));
      __syncwarp();
      if (lane == 0) mbar_arrive(a_ready + i * 2 + (mine & 1));
      m = m_new;
      E = E_new;
      l *= whole_pow2(fmaxf(-grown, -126.f));
      // P of 16 columns -> eight columns
      uint32_t w[kPrKeys / 2];
#pragma unroll
      for (int b = 0; b < kPrRecords; ++b) {
        // (more than 2^110 only where the weights are nothing)
        const float shift = fminf(fmaxf(ev[b] - E, -60.f), 110.f) + (float)kPrTop, fb = factor(b), add = shift - ref;
        float d0 = 0.f, d1 = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float s0 = __uint_as_float(v[b * 16 + 2 * k]), s1 = __uint_as_float(v[b * 16 + 2 * k + 1]);
          pr_fma2(s0, s1, fb, add);
          s0 = ex2(s0);
          s1 = ex2(s1);
          pr_add2(d0, d1, s0, s1);
          w[b * 8 + k] = pack_f16(s0, s1);
        }
        l = fmaf(d0 + d1, whole_pow2(-shift), l);
      }
      tmem_put32(t_s, w);
      tmem_put_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(po_ready + i * 2 + (mine & 1));
      ++mine;
    }
    const float top = l != l ? INFINITY : m;  // a NaN among the scores
    const float up = whole_pow2(fmaxf(E, (float)(kLowExp - kPrSlack - 1)) - (float)kPrTop);
    if constexpr (CUT) {  // a share's state: kv8_merge_kernel
      end_s[i * kPrRows + r] = up;
      if (on) a.part_ml[((size_t)blockIdx.x * a.T + t0 + ti) * a.H + h] = make_float2(top, l);
    } else {
      const RowEnd end = row_end(top, l, sink ? bf2f(sink[h]) : 0.f, sink != nullptr);
      end_s[i * kPrRows + r] = l != l ? NAN : end.factor * up;
      if (on && a.lse) a.lse[(size_t)(t0 + ti) * a.H + h] = end.lse;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(d_ready + i);
  }
  tc_fence_before();
  __syncthreads();
  if (*dead) {  // (for all alike, behind the barrier)
    __syncwarp();
    if (warp == kPrMma || warp == kPrMma + 1) {
      if (tc_elect_one()) umma_commit(done);
      mbar_drain(done, 0);
    }
    __syncthreads();
  }
  if (warp == kPrMma) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (tid == 0) count_run_out(dead, f.err);
}

template <int D, bool CUT>
static int launch_prompt(const bf16* q, const bf16* sink, bf16* out, const PromptArgs& f, int shares, cudaStream_t st) {
  constexpr size_t smem = 128 + (size_t)4 * kPrRows * D + (size_t)(kPrStages + 3 * kPrStagesV) * kPrKeys * D + kPrStagesV * kPrRecords * 20 + 6 * kPrRows * sizeof(float) + 40 * 8;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_prompt_kernel<D, CUT>, smem); e != cudaSuccess) return (int)e;
  return (int)launch(kv8_prompt_kernel<D, CUT>, dim3(shares, f.a.pool.G, (f.a.T + 2 * f.per - 1) / (2 * f.per)), dim3(kPrThreads), smem, st, true, q, sink, out, f);
}
template <int D>
static int launch_prompt(const bf16* q, const bf16* sink, bf16* out, const PromptArgs& f, int shares, cudaStream_t st) {
  return shares > 1 ? launch_prompt<D, true>(q, sink, out, f, shares, st) : launch_prompt<D, false>(q, sink, out, f, shares, st);
}

bool prompt_takes(int T, int H, int G, int dim, int vdim) {
  const int R = H / G, tokens = R <= kPrRows ? 2 * (kPrRows / R) : 0;  // of a CTA
  return dim == vdim && (dim == 64 || dim == 96 || dim == 128) && tokens > 0 && (T + tokens - 1) / tokens <= 65535;
}
// Shares of the keys where the tiles leave SMs idle: as many CTAs as SMs, and 16 blocks of keys to a share at least (of the longest context, which is all that is known).
// (666 tokens of two portions behind 5003, 16 heads: 79 us in shares of 29 blocks and 14 for the merge of 10656 rows, 248 whole.  A share takes 7 us to its first scores, 1.4 a block
// and 6 to its end, 54 in all; the last of the 144 begin at 23 us, behind CTAs without a share, which hold an SM for 4 us each.)
static int prompt_span(int H, int G, int max_kv_len, int window) { return window > 0 ? std::min(max_kv_len, window + 2 * (kPrRows / (H / G))) : max_kv_len; }
static int prompt_pieces(int T, int H, int G, int max_kv_len, int window) {
  const int per = kPrRows / (H / G), ctas = (T + 2 * per - 1) / (2 * per) * G;
  return std::max(1, std::min(sm_count() / std::max(ctas, 1), prompt_span(H, G, max_kv_len, window) / (16 * kPrKeys)));
}
// Twice as many CTAs to a tile as one context makes shares: a tile whose tokens belong to two requests has two contexts to read, and its shares are as long as the others'
// (their other CTAs leave early).  (The same portions: 80 us, 104 with three CTAs to a
// tile.)  A tile's CTAs follow one another in the grid: those that leave make room for the next tile's (94 us with a tile's shares a grid of tiles apart).
int prompt_shares(int T, int H, int G, int max_kv_len, int window) {
  const int pieces = prompt_pieces(T, H, G, max_kv_len, window);
  return pieces > 1 ? 2 * pieces : 1;
}
int prompt_attention(const bf16* q, const bf16* sink, bf16* out, const AttnArgs& a, int shares, cudaStream_t st) {
  PromptArgs f{};
  f.a = a;
  f.per = kPrRows / (a.H / a.pool.G);
  const int pieces = prompt_pieces(a.T, a.H, a.pool.G, a.max_kv_len, a.window), blocks = prompt_span(a.H, a.pool.G, a.max_kv_len, a.window) / kPrKeys + 2;
  f.each = (blocks + pieces - 1) / pieces;
  f.q_by8 = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  f.out_by8 = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && a.out_ld % 8 == 0;
  f.err = wait_err_word();
  return a.pool.dim == 64   ? launch_prompt<64>(q, sink, out, f, shares, st)
         : a.pool.dim == 96 ? launch_prompt<96>(q, sink, out, f, shares, st)
                            : launch_prompt<128>(q, sink, out, f, shares, st);
}

}  // namespace kv8
}  // namespace pk
