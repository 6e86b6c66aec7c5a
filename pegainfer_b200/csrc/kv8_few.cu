// Attention over the 8-bit paged cache for few rows of a request (decoded tokens, small portions), on the tensor cores (kv8.cuh, kv8_attention.cuh).
//
// Bound by the cache's bytes, so everything is made for reading them once and evenly:
//   * The records of all (tile, kv head) pairs of the step, one behind the other, are cut into equal runs, one to a warp of the grid (a CTA to an SM).  A tile is up to
//     eight rows: the group's query heads, for as many tokens of the request as fit.  Where a run's border cuts a pair, its pieces' states (largest
//     score, sum, accumulated values) go through the workspace to kv8_few_merge_kernel.
//   * A warp's records come by bulk copies (K, V and exponents of 16 tokens: 4112 bytes at 128 entries) through a ring of its own, two records to a stage; no
//     warp waits for another.
//   * Codes go into mma.sync m16n8k32 as they are.  q and P have more bits than a code, so each goes in as two: the nearest code and the nearest code of 16 (32)
//     times the rest, 4 + 1 + 4 significant bits (bf16: 8).  The tile's rows are the upper eight rows of the product and their rests the lower eight: both parts
//     of a score end in one thread.  The sums are fp32 (24 bits kept, measured).
//   * Scores: the exponents of K and of the row's q multiply them.  P takes V's exponent e in as 2^(e - E), E the largest so far, so that records of different
//     exponents add up; it is held 2^8 times too large, the upper end of a code's range.
// A group of more than eight heads is several tiles, which read the records again (from L2).
#include <algorithm>

#include "kv8_attention.cuh"
#include "mma.cuh"

namespace pk {
namespace kv8 {

constexpr int kFewTokens = 512;  // of a launch: their tiles are looked up in shared memory
constexpr float kRestQ = 16.f, kRestP = 32.f, kTopP = 256.f;
template <int D>
constexpr int few_warps() { return D <= 128 ? 8 : 4; }
template <int D>
constexpr int few_stages() { return D == 128 || D == 256 ? 3 : 4; }

struct FewArgs {
  AttnArgs a;
  int t_first, U, per;      // first token of the launch; tiles of a token (kv heads x eights of rows), tokens of a tile
  int q_by4;                // q's rows start on 8-byte boundaries
  int* plan;                // [T + 1] records before a token's tiles, [T] the tile's first token, the length of a run: for the merge
  float* scores;            // [T, H, scores_ld] scores (log2), for the weights' sums; or null
  long scores_ld;
  unsigned int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// two entries that need not lie on a 4-byte boundary
__device__ __forceinline__ uint32_t two(const bf16* p) {
  return (uint32_t)__bfloat16_as_ushort(p[0]) | (uint32_t)__bfloat16_as_ushort(p[1]) << 16;
}

template <int D, bool SCORES>
__global__ void __launch_bounds__(few_warps<D>() * 32, 1) kv8_few_kernel(const bf16* __restrict__ q, const bf16* __restrict__ sink, bf16* __restrict__ out, const FewArgs f) {
  constexpr int WARPS = few_warps<D>(), ST = few_stages<D>(), REC = kBlock * 2 * D + 16, THREADS = WARPS * 32;
  extern __shared__ __align__(128) uint8_t fw_sm[];
  __shared__ int s_pre[kFewTokens + 1], s_b0[kFewTokens], s_off[kFewTokens], s_scan[WARPS], s_scan2[WARPS];
  __shared__ uint64_t s_full[WARPS][ST];
  __shared__ int s_dead;
  const AttnArgs& a = f.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  const int R = a.H / a.pool.G, O = (R + 7) / 8, U = f.U, per = f.per;
  volatile int* dead = &s_dead;
  if (tid == 0) s_dead = 0;
  if (lane == 0)
    for (int s = 0; s < ST; ++s) mbar_init(&s_full[warp][s], 1);
  if (tid == 0) mbar_fence_init();
  pdl_wait();
  pdl_launch_dependents();

  // ---- the tiles of the step: their first records and how many, summed up.  Threads have consecutive tokens.
  {
    constexpr int N = kFewTokens / THREADS;
    const int T = a.T;
    int start[N], n[N], mine = 0, from = -1;
#pragma unroll
    for (int i = 0; i < N; ++i) {  // where the token's run began
      const int t = tid * N + i;
      if (t < T && (t == 0 || a.req[t] != a.req[t - 1])) from = t;
      start[i] = from;
    }
    int before = from;  // inclusive maximum over the threads
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before = max(before, o);
    }
    if (lane == 31) s_scan[warp] = before;
    __syncthreads();
    before = __shfl_up_sync(0xffffffffu, before, 1);
    if (lane == 0) before = -1;
    for (int w = 0; w < warp; ++w) before = max(before, s_scan[w]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = tid * N + i;
      n[i] = 0;
      if (t >= T) continue;
      if (start[i] < 0) start[i] = before;
      const int first = t - (t - start[i]) % per;  // the tile's first token
      if (blockIdx.x == 0) f.plan[T + 1 + t] = first;
      if (first != t) continue;
      const int req = a.req[t];
      int top = -1, low = INT_MAX;
      for (int k = 0; k < per && t + k < T && a.req[t + k] == req; ++k) {
        const int p = a.slots[t + k];
        top = max(top, p);
        if (p >= 0) low = min(low, p);
      }
      if (top < 0) continue;
      const int b0 = a.window > 0 ? max(0, low - a.window + 1) / kBlock : 0;
      s_b0[t] = b0;
      s_off[t] = a.pool.page_off[req];
      n[i] = top / kBlock - b0 + 1;
      mine += n[i];
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) s_scan2[warp] = sum;
    __syncthreads();
    sum -= mine;
    for (int w = 0; w < warp; ++w) sum += s_scan2[w];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = tid * N + i;
      if (t <= T) s_pre[t] = sum;
      sum += n[i];
    }
    if (tid == THREADS - 1 && T == kFewTokens) s_pre[T] = sum;
    __syncthreads();
  }
  const int total = s_pre[a.T] * U;
  const int run = few_run(total, (int)gridDim.x * WARPS);
  if (blockIdx.x == 0) {
    for (int t = tid; t <= a.T; t += THREADS) f.plan[t] = s_pre[t];
    if (tid == 0) f.plan[2 * a.T + 1] = run;
  }
  const int x0 = min((blockIdx.x * WARPS + warp) * (long)run, (long)total), x1 = min(x0 + run, total);

  // ---- the run's records: stages of two, never of two tiles
  uint8_t* ring = fw_sm + (size_t)warp * ST * 2 * REC;
  const int rpp = a.pool.page_size / kBlock;
  struct Cursor {
    int t, u, rec, n;  // token of the tile, which of its tiles, record inside, records of the tile
  };
  auto locate = [&](int x) {
    int lo = 0, hi = a.T;  // s_pre[lo] <= x / U < s_pre[hi]
    const int y = x / U;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_pre[mid] <= y) lo = mid;
      else hi = mid;
    }
    Cursor c{lo, 0, 0, s_pre[lo + 1] - s_pre[lo]};
    const int in = x - s_pre[lo] * U;
    c.u = in / c.n;
    c.rec = in - c.u * c.n;
    return c;
  };
  auto next_tile = [&](Cursor& c) {
    c.rec = 0;
    if (++c.u < U) return;
    c.u = 0;
    do ++c.t;
    while (c.t < a.T && s_pre[c.t + 1] == s_pre[c.t]);
    c.n = c.t < a.T ? s_pre[c.t + 1] - s_pre[c.t] : 0;
  };
  // the copies' own walk along the run; lanes 0 and 1 know where the next stage's records are
  Cursor pc{0, 0, 0, 0};
  int px = x0, p_take = 0;
  const uint8_t* p_src = nullptr;
  auto look_up = [&] {  // of the stage at px
    p_take = min(2, min(pc.n - pc.rec, x1 - px));
    if (lane < p_take) {
      const int b = s_b0[pc.t] + pc.rec + lane, g = pc.u / O;
      p_src = a.pool.data + (size_t)a.pool.pages[s_off[pc.t] + b / rpp] * a.pool.page_stride + (size_t)(g * rpp + b % rpp) * REC;
    }
  };
  auto advance = [&] {
    px += p_take;
    pc.rec += p_take;
    if (px >= x1) {
      p_take = 0;
      return;
    }
    if (pc.rec == pc.n) next_tile(pc);
    look_up();
  };
  auto issue = [&](int s) {
    if (p_take <= 0) return;
    if (lane == 0) mbar_expect_tx(&s_full[warp][s], p_take * REC);
    __syncwarp();
    if (lane < p_take)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(ring + (s * 2 + lane) * REC)), "l"(p_src),
                   "r"(REC), "r"(smem_u32(&s_full[warp][s]))
                   : "memory");
  };
  int issued = 0;
  if (x0 < x1) {
    pc = locate(x0);
    look_up();
    for (int s = 0; s < ST; ++s) {
      if (p_take > 0) ++issued;
      issue(s);
      advance();
    }
  }

  // shared-memory offsets of this lane's rows for ldmatrix: K (matrix: 8 tokens x 16 entries; of the two products of a record the first has, for the thread that
  // holds them, the lower or the upper two of its four tokens, so that a matrix' rows lie in eight different groups of banks), V (8 entries x 16 tokens)
  const int mi = lane >> 3, mr = lane & 7, mt = 4 * (mr >> 1) + (((mi >> 1) ^ (mr >> 2)) << 1) + (mr & 1);
  const uint32_t k_at = (uint32_t)((mt >> 3) * (8 * D) + (mi & 1) * 128 + (mt & 7) * 16);
  const uint32_t v_at = (uint32_t)(kBlock * D + (mi >> 1) * 128 + mr * 16);
  const uint32_t p_order = tq < 2 ? 0x5410u : 0x1054u;  // tokens 4 tq .. 4 tq + 3 out of the two products' pairs
  const float c = a.scale * kLog2e;

  int done = 0;  // stages used
  uint32_t parity = 0;
  int slot = 0;
  bool alive = true;
  Cursor cc{0, 0, 0, 0};
  if (x0 < x1) cc = locate(x0);
  for (int x = x0; x < x1;) {
    // ---- a piece: the run's records of one tile
    const int count = min(cc.n - cc.rec, x1 - x);
    const int t = cc.t, g = cc.u / O, row = (cc.u % O) * 8 + gq;  // row of the tile: token t + row / R, head row % R of the group
    const int ti = t + row / R;
    const bool on = row < R * per && ti < a.T && a.req[min(ti, a.T - 1)] == a.req[t];
    const int tr = on ? ti : t, h = g * R + (on ? row % R : 0);
    // (rows that the tile does not have see all and go nowhere: the masks are left out where every row sees a stage whole)
    const int p = on ? a.slots[tr] : INT_MAX, lo = on && a.window > 0 ? p - a.window + 1 : 0;
    uint32_t qa[D / 32][4];
    float qf;  // what a product of q's and K's codes is multiplied with, but for K's exponent
    {
      const bf16* src = q + ((size_t)tr * a.H + h) * D + 4 * tq;
      uint2 raw[D / 16];
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        raw[i] = make_uint2(0, 0);
        if (on) {
          if (f.q_by4) raw[i] = *reinterpret_cast<const uint2*>(src + i * 16);
          else raw[i] = make_uint2(two(src + i * 16), two(src + i * 16 + 2));
        }
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(bf16_lo(raw[i].x)), fabsf(bf16_hi(raw[i].x)))), fmaxf(fabsf(bf16_lo(raw[i].y)), fabsf(bf16_hi(raw[i].y))));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = exponent_for(amax);
      const float down = pow2(-e);
      qf = amax == INFINITY ? NAN : pow2(e);  // (an infinite entry has no code: the row is NaN)
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const float v0 = bf16_lo(raw[i].x) * down, v1 = bf16_hi(raw[i].x) * down, v2 = bf16_lo(raw[i].y) * down, v3 = bf16_hi(raw[i].y) * down;
        const uint32_t hi = codes4(v0, v1, v2, v3);
        float w[4];
        values4(hi, w);
        qa[i >> 1][(i & 1) * 2] = hi;
        qa[i >> 1][(i & 1) * 2 + 1] = codes4((v0 - w[0]) * kRestQ, (v1 - w[1]) * kRestQ, (v2 - w[2]) * kRestQ, (v3 - w[3]) * kRestQ);
      }
    }
    const float row_c = a.cap > 0.f ? qf : qf * c;  // qf * c does not overflow: 2^120 times a scale
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m = -INFINITY, l = 0.f;
    int E = kLowExp - 1;
    for (int i = 0; i < count;) {
      const int take = min(2, count - i);
      if (alive) alive = mbar_wait_bounded(&s_full[warp][slot], parity, dead);
      __syncwarp();
      const uint8_t* stage = ring + slot * 2 * REC;
      const uint32_t at = smem_u32(stage), second = take == 2 ? REC : 0;  // (a missing second record: the first again, with P = 0)
      float s[4][4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t b[4];
          ldsm_x4_at(b, at + (r ? second : 0) + k_at + kk * 256);
          mma_e4m3(s[2 * r], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b[0], b[1]);
          mma_e4m3(s[2 * r + 1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b[2], b[3]);
        }
      }
      const uint32_t tail_a = *reinterpret_cast<const uint32_t*>(stage + kBlock * 2 * D), tail_b = *reinterpret_cast<const uint32_t*>(stage + second + kBlock * 2 * D);
      const int j0 = (s_b0[t] + cc.rec + i) * kBlock;
      const bool inside = j0 >= __reduce_max_sync(0xffffffffu, lo) && j0 + 31 <= __reduce_min_sync(0xffffffffu, p) && take == 2;
      float mx = m;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float fk = pow2(tail_ek(r ? tail_b : tail_a)) * row_c;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = fmaf(s[2 * r + n][e + 2], 1.f / kRestQ, s[2 * r + n][e]) * fk;
            if (a.cap > 0.f) v = shaped(v, c, a.cap);
            if (!inside) {
              const int j = j0 + 16 * r + 4 * tq + ((n ^ (tq >> 1)) << 1) + e;
              v = j >= lo && j <= p && r < take ? v : -INFINITY;
            }
            s[2 * r + n][e] = v;
            mx = fmaxf(mx, v);
          }
      }
      if constexpr (SCORES) {
        if (on) {
          float* to = f.scores + ((size_t)(f.t_first + tr) * a.H + h) * f.scores_ld + j0 + 4 * tq;
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (r < take && j0 + 16 * r + kBlock <= f.scores_ld) {
              const float* w0 = tq < 2 ? s[2 * r] : s[2 * r + 1];
              const float* w1 = tq < 2 ? s[2 * r + 1] : s[2 * r];
              *reinterpret_cast<float4*>(to + 16 * r) = make_float4(w0[0], w0[1], w1[0], w1[1]);
            }
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float ref = mx == -INFINITY ? 0.f : mx;
      const int ea = tail_ev(tail_a), eb = tail_ev(tail_b), e_new = max(E, max(ea, eb));
      const float fl = ex2(m - ref), fo = fl * pow2(max(E - e_new, -126));
      m = mx;
      E = e_new;
      if (__any_sync(0xffffffffu, fo != 1.f)) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][0] *= fo;
          o[d][1] *= fo;
          o[d][2] *= fo;
          o[d][3] *= fo;
        }
      }
      l *= fl;
      uint32_t pa[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float fv = pow2(max((r ? eb : ea) - E, -100)) * kTopP;
        uint32_t hi[2], rest[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2(s[2 * r + n][0] - ref), p1 = ex2(s[2 * r + n][1] - ref);
          l += p0 + p1;
          const float y0 = p0 * fv, y1 = p1 * fv;
          hi[n] = codes2(y0, y1);
          const float2 w = values2(hi[n]);
          rest[n] = codes2((y0 - w.x) * kRestP, (y1 - w.y) * kRestP);
        }
        pa[2 * r] = __byte_perm(hi[0], hi[1], p_order);
        pa[2 * r + 1] = __byte_perm(rest[0], rest[1], p_order);
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldsm_x4_at(b, at + (mi & 1 ? second : 0) + v_at + d * 256);
        mma_e4m3(o[2 * d], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
        mma_e4m3(o[2 * d + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
      }
      i += take;
      ++done;
      __syncwarp();
      if (alive) {
        if (p_take > 0) {
          ++issued;
          fence_async_smem();
        }
        issue(slot);
        advance();
      }
      if (++slot == ST) {
        slot = 0;
        parity ^= 1u;
      }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (l != l) m = INFINITY;  // a NaN among the scores: no other piece may hide it
    const float up = pow2(max(E, -118) - 8);
    if (count == cc.n) {
      const RowEnd end = row_end(m, l, sink ? bf2f(sink[h]) : 0.f, sink != nullptr);
      if (on) {
        const float fac = end.factor * up;
        bf16* dst = out + (size_t)tr * a.out_ld + h * D + 2 * tq;
        const bool pair = (reinterpret_cast<uintptr_t>(out) & 3) == 0 && (a.out_ld & 1) == 0;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          const float v0 = fmaf(o[d][2], 1.f / kRestP, o[d][0]) * fac, v1 = fmaf(o[d][3], 1.f / kRestP, o[d][1]) * fac;
          if (pair) {
            *reinterpret_cast<uint32_t*>(dst + d * 8) = pack_bf16(v0, v1);
          } else {
            dst[d * 8] = f2bf(v0);
            dst[d * 8 + 1] = f2bf(v1);
          }
        }
        if (tq == 0 && a.lse) a.lse[(size_t)tr * a.H + h] = end.lse;
      }
    } else if (on) {
      const size_t at = ((size_t)(blockIdx.x * WARPS + warp) + (size_t)t * U + cc.u) * 8 + gq;
      float* dst = a.part_o + at * D + 2 * tq;
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(dst + d * 8) = make_float2(fmaf(o[d][2], 1.f / kRestP, o[d][0]) * up, fmaf(o[d][3], 1.f / kRestP, o[d][1]) * up);
      if (tq == 0) a.part_ml[at] = make_float2(m, l);
    }
    x += count;
    cc.rec += count;
    if (cc.rec == cc.n && x < x1) next_tile(cc);
  }
  if (!alive) {  // copies under way land in shared memory: their barriers were armed in order
    for (int j = max(0, issued - ST); j < issued; ++j) mbar_drain(&s_full[warp][j % ST], (uint32_t)(j / ST & 1));
  }
  __syncthreads();
  if (tid == 0) count_run_out(dead, f.err);
}

// The pieces of a tile that runs cut -> its rows (and the rows of tiles without a record): a warp to (row, head).
template <int D>
__global__ void __launch_bounds__(128) kv8_few_merge_kernel(const bf16* __restrict__ sink, bf16* __restrict__ out, const FewArgs f) {
  pdl_wait();
  pdl_launch_dependents();
  const AttnArgs& a = f.a;
  const int rows = a.T * a.H, rh = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (rh >= rows) return;
  const int t = rh / a.H, h = rh - t * a.H, R = a.H / a.pool.G, O = (R + 7) / 8;
  const int first = f.plan[a.T + 1 + t], n = f.plan[first + 1] - f.plan[first], run = f.plan[2 * a.T + 1];
  const int row = (t - first) * R + h % R, u = h / R * O + row / 8;
  const int x0 = f.plan[first] * f.U + u * n, w0 = x0 / run, pieces = n > 0 ? (x0 + n - 1) / run - w0 + 1 : 0;
  if (pieces == 1) return;
  const size_t at = ((size_t)w0 + (size_t)first * f.U + u) * 8 + row % 8;  // of the first piece; the others 8 further each
  float M = -INFINITY, den = 0.f;
  for (int s = lane; s < pieces; s += 32) M = fmaxf(M, a.part_ml[at + s * 8].x);
  M = warp_max(M);
  constexpr int PAIRS = D / 2, NP = (PAIRS + 31) / 32;
  float2 acc[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) acc[i] = make_float2(0.f, 0.f);
  for (int s0 = 0; s0 < pieces; s0 += 32) {
    const float2 ml = s0 + lane < pieces ? a.part_ml[at + (s0 + lane) * 8] : make_float2(-INFINITY, 0.f);
    const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
    den += ml.x == -INFINITY ? 0.f : ml.y * w;
    const int many = min(32, pieces - s0);
#pragma unroll 4
    for (int s = 0; s < many; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      const float* src = a.part_o + (at + (size_t)(s0 + s) * 8) * D;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if (lane + 32 * i < PAIRS) {
          const float2 v = *reinterpret_cast<const float2*>(src + 2 * (lane + 32 * i));
          acc[i].x = ws != 0.f ? fmaf(v.x, ws, acc[i].x) : acc[i].x;
          acc[i].y = ws != 0.f ? fmaf(v.y, ws, acc[i].y) : acc[i].y;
        }
    }
  }
  den = warp_sum(den);
  const RowEnd end = row_end(M, den, sink ? bf2f(sink[h]) : 0.f, sink != nullptr);
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (lane + 32 * i < PAIRS) {
      const int d = 2 * (lane + 32 * i);
      bf16* dst = out + (size_t)t * a.out_ld + h * D + d;
      dst[0] = f2bf(acc[i].x * end.factor);
      dst[1] = f2bf(acc[i].y * end.factor);
    }
  if (lane == 0 && a.lse) a.lse[(size_t)t * a.H + h] = end.lse;
}

// weights of the keys out of the kept scores and the finished lse, summed over a run's tokens and the group's heads in their order: a thread to (slot, kv head, run)
__global__ void __launch_bounds__(256) kv8_few_mass_kernel(const float* __restrict__ scores, long scores_ld, AttnArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int t0 = blockIdx.z, g = blockIdx.y, R = a.H / a.pool.G, req = a.req[t0], j = blockIdx.x * 256 + threadIdx.x;
  if (t0 > 0 && a.req[t0 - 1] == req) return;  // a run's first token
  float sum = 0.f;
  bool any = false;
  for (int t = t0; t < a.T && a.req[t] == req; ++t) {
    const int p = a.slots[t];
    if (j > p || (a.window > 0 && j <= p - a.window) || j >= scores_ld) continue;
    any = true;
    const size_t row = (size_t)t * a.H + g * R;
    for (int r = 0; r < R; ++r) sum += ex2(scores[(row + r) * scores_ld + j] - a.lse[row + r] * kLog2e);
  }
  if (any && j < a.mass_ld) a.mass[((size_t)req * a.pool.G + g) * a.mass_ld + j] += sum;
}

template <int D, bool SCORES>
static int launch_few(const bf16* q, const bf16* sink, bf16* out, const FewArgs& f, int ctas, cudaStream_t st) {
  constexpr size_t smem = (size_t)few_warps<D>() * few_stages<D>() * 2 * (kBlock * 2 * D + 16);
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_few_kernel<D, SCORES>, smem); e != cudaSuccess) return (int)e;
  if (const cudaError_t e = launch(kv8_few_kernel<D, SCORES>, dim3(ctas), dim3(few_warps<D>() * 32), smem, st, true, q, sink, out, f); e != cudaSuccess) return (int)e;
  return (int)launch(kv8_few_merge_kernel<D>, dim3((f.a.T * f.a.H + 3) / 4), dim3(128), 0, st, true, sink, out, f);
}

bool few_takes(int T, int H, int G, int dim, int vdim, int max_kv_len, int max_q_len) {
  if (T > 65535 || dim != vdim || !(dim == 32 || dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256)) return false;
  if ((long)std::min(T, kFewTokens) * G * ((H / G + 7) / 8) * (max_kv_len / kBlock + 2) >= 1L << 31) return false;
  return max_q_len > 0 ? max_q_len <= 16 || T < 64 : T < 64;
}
static int few_tokens(int T) { return std::min(T, kFewTokens); }
static int few_warps_of(int dim) { return dim <= 128 ? 8 : 4; }
FewNeed few_need(int T, int H, int G, int dim, int max_kv_len, bool mass) {
  const int U = G * ((H / G + 7) / 8);
  const size_t pieces = (size_t)sm_count() * few_warps_of(dim) + (size_t)few_tokens(T) * U;
  FewNeed n{};
  n.o = pieces * 8 * dim * sizeof(float);
  n.ml = pieces * 8 * sizeof(float2);
  n.plan = ((size_t)2 * few_tokens(T) + 2) * sizeof(int);
  n.plan = (n.plan + 15) / 16 * 16;
  n.scores_ld = (max_kv_len + kBlock - 1) / kBlock * kBlock;
  n.scores = mass ? (size_t)T * H * n.scores_ld * sizeof(float) : 0;
  return n;
}

int few_attention(const bf16* q, const bf16* sink, bf16* out, const AttnArgs& all, const FewNeed& need, uint8_t* ws, cudaStream_t st) {
  const int D = all.pool.dim, R = all.H / all.pool.G;
  FewArgs f{};
  f.U = all.pool.G * ((R + 7) / 8);
  f.per = std::max(1, 8 / R);
  f.plan = reinterpret_cast<int*>(ws);
  f.scores = all.mass ? reinterpret_cast<float*>(ws + need.plan) : nullptr;
  f.scores_ld = need.scores_ld;
  f.q_by4 = (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  f.err = wait_err_word();
  uint8_t* rest = ws + need.plan + need.scores;
  for (int t = 0; t < all.T; t += kFewTokens) {
    AttnArgs a = all;
    a.T = std::min(kFewTokens, all.T - t);
    a.slots += t;
    a.req += t;
    if (a.lse) a.lse += (size_t)t * a.H;
    a.part_o = reinterpret_cast<float*>(rest);
    a.part_ml = reinterpret_cast<float2*>(rest + need.o);
    f.a = a;
    f.t_first = t;
    const long most = (long)a.T * f.U * (all.max_kv_len / kBlock + 2);  // records, at most
    const int ctas = (int)std::max(1L, std::min((long)sm_count(), (most + 2 * few_warps_of(D) - 1) / (2 * few_warps_of(D))));
    int rc = -2;
#define PK_FEW(X)                                                                                                                             \
  if (D == X)                                                                                                                                 \
  rc = all.mass ? launch_few<X, true>(q + (size_t)t * a.H * D, sink, out + (size_t)t * a.out_ld, f, ctas, st)                                 \
                : launch_few<X, false>(q + (size_t)t * a.H * D, sink, out + (size_t)t * a.out_ld, f, ctas, st)
    PK_FEW(32);
    else PK_FEW(64);
    else PK_FEW(96);
    else PK_FEW(128);
    else PK_FEW(192);
    else PK_FEW(256);
#undef PK_FEW
    if (rc != 0) return rc;
  }
  if (!all.mass) return 0;
  const int keys = (int)std::min((long)all.max_kv_len, all.mass_ld);
  return (int)launch(kv8_few_mass_kernel, dim3((keys + 255) / 256, all.pool.G, all.T), dim3(256), 0, st, true, (const float*)f.scores, f.scores_ld, all);
}

}  // namespace kv8
}  // namespace pk
