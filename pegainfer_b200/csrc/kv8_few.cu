// Attention over the 8-bit paged cache for few rows of a request (decoded tokens, small portions), on the tensor cores (kv8.cuh, kv8_attention.cuh).
//
// Bound by the cache's bytes, so everything is made for reading them once and evenly:
//   * The records of all (tile, kv head) pairs of the step, one behind the other, are cut into equal runs, one to a warp of the grid (a CTA to an SM).  A tile is up to
//     16 rows: the group's query heads, for as many tokens of the request as fit.  Where a run's border cuts a pair, its pieces' states (largest
//     score, sum, accumulated values) go through the workspace to kv8_few_merge_kernel.
//   * A warp's records come by bulk copies (K, V and exponents of 16 tokens: 4112 bytes at 128 entries) through a ring of its own, two records to a stage; no
//     warp waits for another.
//   * mma.sync m16n8k16 in f16: K's and V's codes become f16 in registers (exactly; two codes an instruction), q becomes f16 with a power of two for each row that
//     puts its largest entry at 2^14 .. 2^15 (bf16 entries down to 2^-21 of it stay exact), and P, which is held 2^15 times too large, keeps 11 bits down to 2^-29.
//     (The e4m3 form of mma.sync, with q and P as two codes each, is two of these products and the conversion of both operands every time: 828 instead of 400
//     instructions for 32 tokens.)
//   * Scores: the exponents of K and of the row's q multiply them.  P takes V's exponent e in as 2^(e - E), E the largest so far, so that records of different
//     exponents add up.
//   * A tile of up to eight rows leaves the lower half of the product empty, and its exponentials out (HALF).
// A group of more than 16 heads is several tiles, which read the records again (from L2).
#include <algorithm>

#include "kv8_attention.cuh"
#include "mma.cuh"

namespace pk {
namespace kv8 {

constexpr int kFewTokens = 512;  // of a launch: their tiles are looked up in shared memory
constexpr int kTopQ = 14, kTopP = 15;  // exponents of the largest entry of a row of q, and of P = 1, in f16
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
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four codes -> two pairs of f16
__device__ __forceinline__ void widen(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// two entries that need not lie on a 4-byte boundary
__device__ __forceinline__ uint32_t two(const bf16* p) {
  return (uint32_t)__bfloat16_as_ushort(p[0]) | (uint32_t)__bfloat16_as_ushort(p[1]) << 16;
}

template <int D, bool SCORES, bool HALF>
__global__ void __launch_bounds__(few_warps<D>() * 32, 1) kv8_few_kernel(const bf16* __restrict__ q, const bf16* __restrict__ sink, bf16* __restrict__ out, const FewArgs f) {
  constexpr int WARPS = few_warps<D>(), ST = few_stages<D>(), REC = kBlock * 2 * D + 16, THREADS = WARPS * 32, ROWS = HALF ? 1 : 2;
  extern __shared__ __align__(128) uint8_t fw_sm[];
  __shared__ int s_pre[kFewTokens + 1], s_b0[kFewTokens], s_off[kFewTokens], s_req[kFewTokens], s_slot[kFewTokens], s_scan[WARPS], s_scan2[WARPS];
  __shared__ uint64_t s_full[WARPS][ST];
  __shared__ int s_dead;
  const AttnArgs& a = f.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  const int R = a.H / a.pool.G, O = (R + 15) / 16, U = f.U, per = f.per;
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
    int req[N], start[N], n[N], mine = 0, from = -1;
    for (int t = tid; t < T; t += THREADS) {
      const int r = a.req[t], p = a.slots[t];
      s_req[t] = r;
      s_slot[t] = p;
      s_off[t] = p >= 0 ? a.pool.page_off[r] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {  // where the token's run began
      const int t = tid * N + i;
      req[i] = t < T ? s_req[t] : 0;
      if (t < T && (t == 0 || req[i] != s_req[t - 1])) from = t;
      start[i] = from;
    }
    int before = from;  // inclusive maximum over the threads
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before = max(before, o);
    }
    if (lane == 31) s_scan[warp] = before;
    before = __shfl_up_sync(0xffffffffu, before, 1);
    if (lane == 0) before = -1;
    __syncthreads();
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
      int top = -1, low = INT_MAX;
      for (int k = 0; k < per && t + k < T && s_req[t + k] == req[i]; ++k) {
        const int p = s_slot[t + k];
        top = max(top, p);
        if (p >= 0) low = min(low, p);
      }
      if (top < 0) continue;
      const int b0 = a.window > 0 ? max(0, low - a.window + 1) / kBlock : 0;
      s_b0[t] = b0;
      if (s_slot[t] < 0) s_off[t] = a.pool.page_off[req[i]];
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
  const float c = a.scale * kLog2e;

  uint32_t parity = 0;
  int slot = 0;
  bool alive = true;
  Cursor cc{0, 0, 0, 0};
  if (x0 < x1) cc = locate(x0);
  for (int x = x0; x < x1;) {
    // ---- a piece: the run's records of one tile
    const int count = min(cc.n - cc.rec, x1 - x);
    const int t = cc.t, g = cc.u / O;
    // rows gq and gq + 8 of the tile: token t + row / R, head row % R of the group (from the tile's 16 on).  Rows that the tile does not have see all and go
    // nowhere: the masks are left out where every row sees a stage whole.
    int tr[ROWS], h[ROWS], p[ROWS], lo[ROWS];
    bool on[ROWS];
    float row_c[ROWS];  // what a product of q's f16 and K's codes is multiplied with, but for K's exponent
    uint32_t qa[D / 16][2 * ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int row = (cc.u % O) * 16 + gq + 8 * i, ti = t + row / R;
      on[i] = row < R * per && ti < a.T && s_req[min(ti, a.T - 1)] == s_req[t];
      tr[i] = on[i] ? ti : t;
      h[i] = g * R + (on[i] ? row % R : 0);
      p[i] = on[i] ? s_slot[tr[i]] : INT_MAX;
      lo[i] = on[i] && a.window > 0 ? p[i] - a.window + 1 : 0;
      const bf16* src = q + ((size_t)tr[i] * a.H + h[i]) * D + 4 * tq;
      uint2 raw[D / 16];
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        raw[k] = make_uint2(0, 0);
        if (on[i]) {
          if (f.q_by4) raw[k] = *reinterpret_cast<const uint2*>(src + k * 16);
          else raw[k] = make_uint2(two(src + k * 16), two(src + k * 16 + 2));
        }
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(bf16_lo(raw[k].x)), fabsf(bf16_hi(raw[k].x)))), fmaxf(fabsf(bf16_lo(raw[k].y)), fabsf(bf16_hi(raw[k].y))));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - kTopQ, kLowExp), kHighExp);
      const float down = pow2(-e), qf = amax == INFINITY ? NAN : pow2(e);  // (an infinite entry: the row is NaN)
      row_c[i] = a.cap > 0.f ? qf : qf * c;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qa[k][i] = pack_f16(bf16_lo(raw[k].x) * down, bf16_hi(raw[k].x) * down);
        qa[k][ROWS + i] = pack_f16(bf16_lo(raw[k].y) * down, bf16_hi(raw[k].y) * down);
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[ROWS], l[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
    const int all_lo = __reduce_max_sync(0xffffffffu, ROWS == 2 ? max(lo[0], lo[ROWS - 1]) : lo[0]);
    const int all_p = __reduce_min_sync(0xffffffffu, ROWS == 2 ? min(p[0], p[ROWS - 1]) : p[0]);
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
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // product x / 2 of the record, piece of 16 entries 2 kk + x % 2
            uint32_t b0, b1;
            widen(b[x], b0, b1);
            const uint32_t(&qk)[2 * ROWS] = qa[2 * kk + (x & 1)];
            mma_f16(s[2 * r + (x >> 1)], qk[0], ROWS == 2 ? qk[1] : 0u, qk[ROWS], ROWS == 2 ? qk[2 * ROWS - 1] : 0u, b0, b1);
          }
        }
      }
      const uint32_t tail_a = *reinterpret_cast<const uint32_t*>(stage + kBlock * 2 * D), tail_b = *reinterpret_cast<const uint32_t*>(stage + second + kBlock * 2 * D);
      const int j0 = (s_b0[t] + cc.rec + i) * kBlock;
      const bool inside = j0 >= all_lo && j0 + 31 <= all_p && take == 2;
      const int ea = tail_ev(tail_a), eb = tail_ev(tail_b), e_new = max(E, max(ea, eb));
      const float fe = pow2(max(E - e_new, -126));
      E = e_new;
      float fo[ROWS], ref[ROWS];
#pragma unroll
      for (int w = 0; w < ROWS; ++w) {
        float mx = m[w];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float fk = pow2(tail_ek(r ? tail_b : tail_a)) * row_c[w];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = s[2 * r + n][2 * w + e] * fk;
              if (a.cap > 0.f) v = shaped(v, c, a.cap);
              if (!inside) {
                const int j = j0 + 16 * r + 4 * tq + ((n ^ (tq >> 1)) << 1) + e;
                v = j >= lo[w] && j <= p[w] && r < take ? v : -INFINITY;
              }
              s[2 * r + n][2 * w + e] = v;
              mx = fmaxf(mx, v);
            }
        }
        if constexpr (SCORES) {
          if (on[w]) {
            float* to = f.scores + ((size_t)(f.t_first + tr[w]) * a.H + h[w]) * f.scores_ld + j0 + 4 * tq;
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (r < take && j0 + 16 * r + kBlock <= f.scores_ld) {
                const float w0 = s[2 * r][2 * w], w1 = s[2 * r][2 * w + 1], w2 = s[2 * r + 1][2 * w], w3 = s[2 * r + 1][2 * w + 1];
                *reinterpret_cast<float4*>(to + 16 * r) = tq < 2 ? make_float4(w0, w1, w2, w3) : make_float4(w2, w3, w0, w1);
              }
          }
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        ref[w] = mx == -INFINITY ? 0.f : mx;
        const float fl = ex2(m[w] - ref[w]);
        fo[w] = fl * fe;
        m[w] = mx;
        l[w] *= fl;
      }
      if (__any_sync(0xffffffffu, fo[0] != 1.f || fo[ROWS - 1] != 1.f)) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
          for (int w = 0; w < ROWS; ++w) {
            o[d][2 * w] *= fo[w];
            o[d][2 * w + 1] *= fo[w];
          }
      }
      uint32_t pa[2][2 * ROWS];  // of a record: the lower and the upper two of the thread's four tokens, for its rows
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float fv = pow2(max((r ? eb : ea) - E, -100) + kTopP);
#pragma unroll
        for (int w = 0; w < ROWS; ++w) {
          uint32_t y[2];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float p0 = ex2(s[2 * r + n][2 * w] - ref[w]), p1 = ex2(s[2 * r + n][2 * w + 1] - ref[w]);
            l[w] += p0 + p1;
            y[n] = pack_f16(p0 * fv, p1 * fv);
          }
          pa[r][w] = tq < 2 ? y[0] : y[1];
          pa[r][ROWS + w] = tq < 2 ? y[1] : y[0];
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldsm_x4_at(b, at + (mi & 1 ? second : 0) + v_at + d * 256);
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // record x % 2, entries 8 (2 d + x / 2) ..
          uint32_t b0, b1;
          widen(b[x], b0, b1);
          const uint32_t(&pr)[2 * ROWS] = pa[x & 1];
          mma_f16(o[2 * d + (x >> 1)], pr[0], ROWS == 2 ? pr[1] : 0u, pr[ROWS], ROWS == 2 ? pr[2 * ROWS - 1] : 0u, b0, b1);
        }
      }
      i += take;
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
    const float up = pow2(max(E, kLowExp) - kTopP);
#pragma unroll
    for (int w = 0; w < ROWS; ++w) {
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
      if (l[w] != l[w]) m[w] = INFINITY;  // a NaN among the scores: no other piece may hide it
      if (count == cc.n) {
        const RowEnd end = row_end(m[w], l[w], sink ? bf2f(sink[h[w]]) : 0.f, sink != nullptr);
        if (on[w]) {
          const float fac = end.factor * up;
          bf16* dst = out + (size_t)tr[w] * a.out_ld + h[w] * D + 2 * tq;
          const bool pair = (reinterpret_cast<uintptr_t>(out) & 3) == 0 && (a.out_ld & 1) == 0;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            if (pair) {
              *reinterpret_cast<uint32_t*>(dst + d * 8) = pack_bf16(o[d][2 * w] * fac, o[d][2 * w + 1] * fac);
            } else {
              dst[d * 8] = f2bf(o[d][2 * w] * fac);
              dst[d * 8 + 1] = f2bf(o[d][2 * w + 1] * fac);
            }
          }
          if (tq == 0 && a.lse) a.lse[(size_t)tr[w] * a.H + h[w]] = end.lse;
        }
      } else if (on[w]) {
        const size_t at = ((size_t)(blockIdx.x * WARPS + warp) + (size_t)t * U + cc.u) * (8 * ROWS) + gq + 8 * w;
        float* dst = a.part_o + at * D + 2 * tq;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(dst + d * 8) = make_float2(o[d][2 * w] * up, o[d][2 * w + 1] * up);
        if (tq == 0) a.part_ml[at] = make_float2(m[w], l[w]);
      }
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

// The pieces of a tile that runs cut -> its rows (and the rows of tiles without a record): `share` warps of a CTA to (row, head), which take its pieces by turns.
template <int D>
__global__ void __launch_bounds__(256) kv8_few_merge_kernel(const bf16* __restrict__ sink, bf16* __restrict__ out, int share, int tile_rows, const FewArgs f) {
  __shared__ float2 s_o[8][D / 2], s_ml[8];
  pdl_wait();
  pdl_launch_dependents();
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % share, rh = blockIdx.x * (8 / share) + warp / share, rows = a.T * a.H;
  const int t = min(rh, rows - 1) / a.H, h = min(rh, rows - 1) - t * a.H, R = a.H / a.pool.G, O = (R + 15) / 16;
  const int first = f.plan[a.T + 1 + t], run = f.plan[2 * a.T + 1], before = f.plan[first], n = f.plan[first + 1] - before;
  const int row = (t - first) * R + h % R, u = h / R * O + row / 16;
  const int x0 = before * f.U + u * n, w0 = x0 / run, pieces = n > 0 ? (x0 + n - 1) / run - w0 + 1 : 0;
  const size_t at = ((size_t)w0 + (size_t)first * f.U + u) * tile_rows + row % 16;  // of the first piece; the others a tile further each
  float M = -INFINITY, den = 0.f;
  constexpr int PAIRS = D / 2, NP = (PAIRS + 31) / 32, AT_ONCE = 8 / NP;
  float2 acc[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) acc[i] = make_float2(0.f, 0.f);
  if (pieces > 1) {
    for (int s = lane; s < pieces; s += 32) M = fmaxf(M, a.part_ml[at + (size_t)s * tile_rows].x);
    M = warp_max(M);
    for (int s0 = part; s0 < pieces; s0 += AT_ONCE * share) {
      float2 v[AT_ONCE][NP], ml[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int s = s0 + k * share;
        ml[k] = s < pieces ? a.part_ml[at + (size_t)s * tile_rows] : make_float2(-INFINITY, 0.f);
        const float2* src = reinterpret_cast<const float2*>(a.part_o + (at + (size_t)s * tile_rows) * D) + lane;
#pragma unroll
        for (int i = 0; i < NP; ++i) v[k][i] = s < pieces && lane + 32 * i < PAIRS ? src[32 * i] : make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        if (ml[k].x == -INFINITY) continue;
        const float w = ex2(ml[k].x - M);
        den = fmaf(ml[k].y, w, den);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          acc[i].x = fmaf(v[k][i].x, w, acc[i].x);
          acc[i].y = fmaf(v[k][i].y, w, acc[i].y);
        }
      }
    }
  }
  if (share > 1) {
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (lane + 32 * i < PAIRS) s_o[warp][lane + 32 * i] = acc[i];
    if (lane == 0) s_ml[warp] = make_float2(M, den);
    __syncthreads();
    if (part > 0) return;
    for (int w = 1; w < share; ++w) {
      den += s_ml[warp + w].y;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if (lane + 32 * i < PAIRS) {
          acc[i].x += s_o[warp + w][lane + 32 * i].x;
          acc[i].y += s_o[warp + w][lane + 32 * i].y;
        }
    }
  }
  if (pieces == 1 || rh >= rows) return;  // (a tile that one warp had whole is finished)
  const RowEnd end = row_end(M, den, sink ? bf2f(sink[h]) : 0.f, sink != nullptr);
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (lane + 32 * i < PAIRS) {
      bf16* dst = out + (size_t)t * a.out_ld + h * D + 2 * (lane + 32 * i);
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

// behind a kernel of the same call: its launch may always overlap that one's end
template <typename... KArgs, typename... Args>
static cudaError_t follow(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t st, Args... args) {
  ThreadState& ts = tls();
  const bool pdl = ts.pdl;
  ts.pdl = true;
  const cudaError_t e = launch(kernel, grid, block, 0, st, true, args...);
  ts.pdl = pdl;
  return e;
}

template <int D, bool SCORES, bool HALF>
static int launch_few(const bf16* q, const bf16* sink, bf16* out, const FewArgs& f, int ctas, cudaStream_t st) {
  constexpr size_t smem = (size_t)few_warps<D>() * few_stages<D>() * 2 * (kBlock * 2 * D + 16);
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_few_kernel<D, SCORES, HALF>, smem); e != cudaSuccess) return (int)e;
  if (const cudaError_t e = launch(kv8_few_kernel<D, SCORES, HALF>, dim3(ctas), dim3(few_warps<D>() * 32), smem, st, true, q, sink, out, f); e != cudaSuccess) return (int)e;
  // few rows have many pieces each
  const int rows = f.a.T * f.a.H, share = rows <= 4 * sm_count() ? 8 : rows <= 16 * sm_count() ? 2 : 1;
  return (int)follow(kv8_few_merge_kernel<D>, dim3((rows * share + 7) / 8), dim3(256), st, sink, out, share, HALF ? 8 : 16, f);
}
template <int D>
static int launch_few(const bf16* q, const bf16* sink, bf16* out, const FewArgs& f, int ctas, bool half, cudaStream_t st) {
  if (f.scores) return half ? launch_few<D, true, true>(q, sink, out, f, ctas, st) : launch_few<D, true, false>(q, sink, out, f, ctas, st);
  return half ? launch_few<D, false, true>(q, sink, out, f, ctas, st) : launch_few<D, false, false>(q, sink, out, f, ctas, st);
}

bool few_takes(int T, int H, int G, int dim, int vdim, int max_kv_len, int max_q_len) {
  if (T > 65535 || dim != vdim || !(dim == 32 || dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256)) return false;
  if ((long)std::min(T, kFewTokens) * G * ((H / G + 15) / 16) * (max_kv_len / kBlock + 2) >= 1L << 31) return false;
  return max_q_len > 0 ? max_q_len <= 16 || T < 64 : T < 64;
}
static int few_tokens(int T) { return std::min(T, kFewTokens); }
static int few_warps_of(int dim) { return dim <= 128 ? 8 : 4; }
FewNeed few_need(int T, int H, int G, int dim, int max_kv_len, bool mass) {
  const int U = G * ((H / G + 15) / 16);
  const size_t pieces = (size_t)sm_count() * few_warps_of(dim) + (size_t)few_tokens(T) * U;
  FewNeed n{};
  n.o = pieces * 16 * dim * sizeof(float);
  n.ml = pieces * 16 * sizeof(float2);
  n.plan = ((size_t)2 * few_tokens(T) + 2) * sizeof(int);
  n.plan = (n.plan + 15) / 16 * 16;
  n.scores_ld = (max_kv_len + kBlock - 1) / kBlock * kBlock;
  n.scores = mass ? (size_t)T * H * n.scores_ld * sizeof(float) : 0;
  return n;
}

int few_attention(const bf16* q, const bf16* sink, bf16* out, const AttnArgs& all, int max_q_len, const FewNeed& need, uint8_t* ws, cudaStream_t st) {
  const int D = all.pool.dim, R = all.H / all.pool.G;
  FewArgs f{};
  f.U = all.pool.G * ((R + 15) / 16);
  const bool half = max_q_len > 0 && R * max_q_len <= 8;  // the rows of a tile fit into half a product
  f.per = half ? max_q_len : std::max(1, 16 / R);
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
    const bf16* qt = q + (size_t)t * a.H * D;
    bf16* ot = out + (size_t)t * a.out_ld;
    const int rc = D == 32    ? launch_few<32>(qt, sink, ot, f, ctas, half, st)
                   : D == 64  ? launch_few<64>(qt, sink, ot, f, ctas, half, st)
                   : D == 96  ? launch_few<96>(qt, sink, ot, f, ctas, half, st)
                   : D == 128 ? launch_few<128>(qt, sink, ot, f, ctas, half, st)
                   : D == 192 ? launch_few<192>(qt, sink, ot, f, ctas, half, st)
                              : launch_few<256>(qt, sink, ot, f, ctas, half, st);
    if (rc != 0) return rc;
  }
  if (!all.mass) return 0;
  const int keys = (int)std::min((long)all.max_kv_len, all.mass_ld);
  return (int)follow(kv8_few_mass_kernel, dim3((keys + 255) / 256, all.pool.G, all.T), dim3(256), st, (const float*)f.scores, f.scores_ld, all);
}

}  // namespace kv8
}  // namespace pk
