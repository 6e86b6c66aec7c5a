// Attention over the 8-bit paged cache for few rows of a request (decoded tokens, small portions), on the tensor cores (kv8.cuh, kv8_attention.cuh).
//
// Bound by the cache's bytes, so everything is made for reading them once and evenly:
//   * The records of all (tile, kv head) pairs of the step, one behind the other, are cut into equal runs, one to a warp of the grid (a CTA to an SM).  A tile is up to
//     16 rows: the group's query heads, for as many tokens of the request as fit.  Where a run's border cuts a pair, its pieces' states (largest
//     score, sum, accumulated values) go through the workspace to kv8_few_merge_kernel.
//   * A warp's records come by bulk copies (K, V and exponents of 16 tokens: 4112 bytes at 128 entries) through a ring of its own, two records to a stage; no
//     warp waits for another.
//   * mma.sync m16n8k16 in f16, turned round: S^T = K q^T and O^T = V^T P^T, so that 16 tokens (16 entries of V) fill a product's long side and up to eight rows its
//     short one; a tile of up to 16 rows (WIDE) takes two.  K's and V's codes become f16 in registers (exactly; two codes an instruction), q becomes f16 with a power of
//     two for each row that puts its largest entry at 2^14 .. 2^15 (bf16 entries down to 2^-21 of it stay exact), and P, which is held 2^15 times too large,
//     keeps 11 bits down to 2^-29.  movmatrix turns P.  (The e4m3 form of mma.sync is two of these products and a conversion of both operands each time.)
//   * Scores: the exponents of K and of the row's q multiply them.  P takes V's exponent e in as 2^(e - E), E the largest so far, which costs P up to kNear of its 29 bits of
//     range while V's exponents lie no further apart; once they do, every row has its own E, m + E being its largest (score + e) so far: what a row does not see, or gives no
//     weight, costs its other tokens no bits, however large its values.  (One way for all calls: 3 to 10 % slower, groups of 16 heads of 64 most, 37 -> 41 us.)
// A group of more than 16 heads is several tiles, which read the records again (from L2).
// B200: 32 requests of about 3350, 32 heads of 128 in 8 groups (229 MB): 45 us (5.1 TB/s), and 6 for the pieces; one request of 301: 7.5 and 5.4, latency; 48 requests in a
// window of 1024, 64 heads of 64 in 8 groups, scores capped (50 MB): 25 us, of which 8 are start and end, the rest the instructions of a stage (its 4 KB are half as
// many as at 128 entries, the maxima, sums and caps of its 32 tokens as many).
#include <algorithm>
#include <type_traits>

#include "kv8_attention.cuh"
#include "mma.cuh"

namespace pk {
namespace kv8 {

// Bytes of scores that are kept for the weights' sums; with more they are computed again (kv8_mass.cu).  B200, 32 heads of 128 in 8 groups, us kept : again: decoded tokens of one
// request behind 2000 17 : 23, behind 131072 81 : 463, of 16 behind 8190 78 : 445, of 64 247 : 1422 (64 MB); portions, whose keys several rows share, 4 of 16 tokens behind 4000
// 105 : 87, one of 32 behind 16000 171 : 108.  So the limit is there for the workspace alone, which grows with max_kv_len.
constexpr size_t kMostScores = (size_t)1 << 30;
constexpr float kNoneYet = -1000.f;  // E of a row that has seen nothing
constexpr int kNear = 8;             // V's exponents within so much: one E for all rows
constexpr int kFewTokens = 512;  // of a launch: their tiles are looked up in shared memory
template <int D>
constexpr int few_warps() { return D <= 128 ? 8 : 4; }
template <int D>
constexpr int few_stages() { return D <= 64 ? 4 : D <= 96 ? 3 : 2; }

struct FewArgs {
  AttnArgs a;
  int t_first, U, per;      // first token of the launch; tiles of a token (kv heads x sixteens of rows), tokens of a tile
  int abreast;              // warps that go through the same records of different tiles of a token
  int q_by4, out_by4;       // rows start on 8-byte boundaries
  uint32_t inv_r;           // row / R = row * inv_r >> 16 for the rows of a tile of several tokens (at most 16 rows); 0 where a tile has one token's
  int* plan;                // [T + 1] records before a token's tiles, [T] the tile's first token, the length of a run: for the merge
  float* scores;            // scores (log2) for the weights' sums, or null: [tiles of a token][t_all][min(R, 16)][scores_ld], a tile's at its first token as [slot][row]
  int t_all;                // tokens of the call
  long scores_ld;
  unsigned int* err;
};

// an 8 x 8 matrix of f16 turned round
__device__ __forceinline__ uint32_t turned(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// two entries that need not lie on a 4-byte boundary
__device__ __forceinline__ uint32_t two(const bf16* p) {
  return (uint32_t)__bfloat16_as_ushort(p[0]) | (uint32_t)__bfloat16_as_ushort(p[1]) << 16;
}

template <int D, bool SCORES, bool WIDE>
__global__ void __launch_bounds__(few_warps<D>() * 32, 1) kv8_few_kernel(const bf16* __restrict__ q, const bf16* __restrict__ sink, bf16* __restrict__ out, const FewArgs f) {
  constexpr int WARPS = few_warps<D>(), ST = few_stages<D>(), REC = kBlock * 2 * D + 16, THREADS = WARPS * 32, NT = WIDE ? 2 : 1;
  extern __shared__ __align__(128) uint8_t fw_sm[];
  __shared__ int s_pre[kFewTokens + 1], s_b0[kFewTokens], s_off[kFewTokens], s_req[kFewTokens], s_slot[kFewTokens], s_scan[WARPS], s_scan2[WARPS];
  __shared__ uint64_t s_full[WARPS][ST];
  __shared__ int s_dead;
  const AttnArgs& a = f.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  const int R = a.H / a.pool.G, O = (R + 15) / 16, AB = f.abreast, U = f.U / AB, per = f.per;  // U: of the tiles that a warp sees
  volatile int* dead = &s_dead;
  if (tid == 0) s_dead = 0;
  if (lane == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&s_full[warp][s], 1);
    mbar_fence_init();
  }
  pdl_wait();
  pdl_launch_dependents();

  // ---- the tiles of the step: their first records and how many, summed up.  Threads have consecutive tokens.
  {
    constexpr int N = (kFewTokens + THREADS - 1) / THREADS;
    const int T = a.T;
    int req[N], start[N], n[N], mine = 0, from = -1;
    int off[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = tid + i * THREADS;
      off[i] = 0;
      if (t >= T) continue;
      const int r = a.req[t], p = a.slots[t];
      s_req[t] = r;
      s_slot[t] = p;
      if (p >= 0) off[i] = a.pool.page_off[r];  // under way until the tiles are known
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
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * THREADS < T) s_off[tid + i * THREADS] = off[i];
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
  const int run = few_run(total, (int)gridDim.x * WARPS / AB);
  if (blockIdx.x == 0) {
    for (int t = tid; t <= a.T; t += THREADS) f.plan[t] = s_pre[t];
    if (tid == 0) f.plan[2 * a.T + 1] = run;
  }
  const int who = (blockIdx.x * WARPS + warp) / AB, mine = warp % AB;
  const int x0 = (int)min(who * (long)run, (long)total), x1 = (int)min((long)x0 + run, (long)total);

  // ---- the run's records: stages of two, never of two tiles
  constexpr int TURN_LD = D + 4;
  uint8_t* ring = fw_sm + (size_t)warp * ST * 2 * REC;
  float* turn = reinterpret_cast<float*>(fw_sm + (size_t)WARPS * ST * 2 * REC) + warp * 8 * TURN_LD;
  const int rpp = a.pool.page_size / kBlock, rpp_shift = (rpp & (rpp - 1)) == 0 ? 31 - __clz(rpp) : -1;
  struct Cursor {
    int t, u, rec, n;  // token of the tile, which of its tiles (u * AB + mine), record inside, records of the tile
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
  // the copies' own walk along the run: px is where the next stage begins, p_take its records
  Cursor pc{0, 0, 0, 0};
  int px = x0, p_take = 0, p_b0 = 0, p_off = 0, p_g = 0;
  const uint8_t* p_src = nullptr;
  auto enter = [&] {
    p_b0 = s_b0[pc.t];
    int t = pc.t;
    while (s_slot[t] < 0) ++t;  // (a tile with records has a token with a slot)
    p_off = s_off[t];
    p_g = (pc.u * AB + mine) / O;
  };
  auto source = [&](int b0, int off, int g, int rec) {
    const int b = b0 + rec, page = rpp_shift >= 0 ? b >> rpp_shift : b / rpp;
    return a.pool.data + (size_t)a.pool.pages[off + page] * a.pool.page_stride + (size_t)(g * rpp + b - page * rpp) * REC;
  };
  auto step = [&] {  // on to the next stage
    px += p_take;
    pc.rec += p_take;
    if (px >= x1) {
      p_take = 0;
      return;
    }
    if (pc.rec == pc.n) {
      next_tile(pc);
      enter();
    }
    p_take = min(2, min(pc.n - pc.rec, x1 - px));
  };
  auto copy = [&](int s, int r, const uint8_t* src) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(ring + (s * 2 + r) * REC)), "l"(src), "r"(REC),
                 "r"(smem_u32(&s_full[warp][s]))
                 : "memory");
  };
  // the rows of q that this lane turns into f16: of tile (t, unit)
  auto tokens_of = [&](int t) {
    int n = 1;
    while (n < per && t + n < a.T && s_req[t + n] == s_req[t]) ++n;
    return n;
  };
  uint2 raw[NT][D / 16];
  auto load_q = [&](const Cursor& cur) {
    const int unit = cur.u * AB + mine, g = unit / O, n_tok = tokens_of(cur.t);
#pragma unroll
    for (int w = 0; w < NT; ++w) {
      const int row = unit % O * 16 + 8 * w + gq, k = (int)((uint32_t)row * f.inv_r >> 16);
      const bool on = row < R * per && k < n_tok;
      const bf16* src = q + ((size_t)(cur.t + (on ? k : 0)) * a.H + g * R + (on ? row - k * R : 0)) * D + 4 * tq;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        raw[w][i] = make_uint2(0, 0);
        if (on) {
          if (f.q_by4) raw[w][i] = *reinterpret_cast<const uint2*>(src + i * 16);
          else raw[w][i] = make_uint2(two(src + i * 16), two(src + i * 16 + 2));
        }
      }
    }
  };
  int issued = 0;
  Cursor first{0, 0, 0, 0};
  if (x0 < x1) {
    first = locate(x0);
    load_q(first);  // ahead of the copies in the memory's queues
  }
  if (x0 < x1) {  // the first stages: their pages are looked up by a lane each
    pc = first;
    enter();
    p_take = min(2, min(pc.n - pc.rec, x1 - px));
    int b0 = 0, off = 0, g = 0, rec = -1;
    for (int s = 0; s < ST && p_take > 0; ++s) {
      if (lane >> 1 == s && (lane & 1) < p_take) {
        b0 = p_b0;
        off = p_off;
        g = p_g;
        rec = pc.rec + (lane & 1);
      }
      if (lane == 0) mbar_expect_tx(&s_full[warp][s], p_take * REC);
      ++issued;
      step();
    }
    __syncwarp();
    if (rec >= 0) copy(lane >> 1, lane & 1, source(b0, off, g, rec));
    if (lane < p_take) p_src = source(p_b0, p_off, p_g, pc.rec + lane);  // of the next one: lanes 0 and 1
  }

  // shared-memory offsets of this lane's rows for ldmatrix.  K: 8 tokens x 16 entries; the first and the second eight of a product's 16 tokens are, behind the turn, the
  // lower or the upper two of a thread's four tokens, chosen so that the eight rows lie in different groups of banks.  V: 8 entries x 16 tokens.
  const int mi = lane >> 3, mr = lane & 7;
  auto token_of = [](int which, int i) { return 4 * (i >> 1) + (((i >> 2) ^ which) << 1) + (i & 1); };
  const int mt = token_of(mi & 1, mr);
  const uint32_t k_at = (uint32_t)((mt >> 3) * (8 * D) + (mi >> 1) * 128 + (mt & 7) * 16);
  const uint32_t v_at = (uint32_t)(kBlock * D + (mi & 1) * 128 + mr * 16);
  const int tok[2] = {token_of(0, gq), token_of(1, gq)};  // this thread's tokens of a record
  const float c = a.scale * kLog2e, cap2 = a.cap * kLog2e, cap_c = a.cap > 0.f ? 2.f * a.scale / a.cap * kLog2e : 0.f;
  auto max_of_rows = [](float x) {  // over the lanes that have other tokens of the same rows
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
  };

  uint32_t parity = 0;
  int slot = 0;
  bool alive = true;
  Cursor cc = first;
  for (int x = x0; x < x1;) {
    // ---- a piece: the run's records of one tile.  Row r of the tile: token t + r / R, head r % R of the group (from the tile's 16 on).
    const int count = min(cc.n - cc.rec, x1 - x);
    const int t = cc.t, unit = cc.u * AB + mine, g = unit / O, row0 = unit % O * 16;
    const int n_tok = tokens_of(t);
    auto token = [&](int row) {  // -1: no such row
      const int k = (int)((uint32_t)row * f.inv_r >> 16);
      return row < R * per && k < n_tok ? t + k : -1;
    };
    auto head = [&](int row) { return row - (int)((uint32_t)row * f.inv_r >> 16) * R; };
    uint32_t qb[D / 16][2 * NT];
    float row_c[2 * NT];  // what a product of q's f16 and K's codes is multiplied with, but for K's exponent; rows 8 w + 2 tq + e at 2 w + e
    int p[2 * NT], lo[2 * NT];
#pragma unroll
    for (int w = 0; w < NT; ++w) {
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(bf16_lo(raw[w][k].x)), fabsf(bf16_hi(raw[w][k].x)))), fmaxf(fabsf(bf16_lo(raw[w][k].y)), fabsf(bf16_hi(raw[w][k].y))));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - kTopQ, kLowExp), kHighExp);
      const float down = pow2(-e), qf = amax == INFINITY ? NAN : a.cap > 0.f ? pow2(e) : pow2(e) * c;  // (an infinite entry: the row is NaN)
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qb[k][2 * w] = pack_f16(bf16_lo(raw[w][k].x) * down, bf16_hi(raw[w][k].x) * down);
        qb[k][2 * w + 1] = pack_f16(bf16_lo(raw[w][k].y) * down, bf16_hi(raw[w][k].y) * down);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row_c[2 * w + i] = __shfl_sync(0xffffffffu, qf, (2 * tq + i) * 4);
        const int to = token(row0 + 8 * w + 2 * tq + i);
        // rows that the tile does not have see all and go nowhere: the masks are left out where every row sees a stage whole
        p[2 * w + i] = to >= 0 ? s_slot[to] : INT_MAX;
        lo[2 * w + i] = to >= 0 && a.window > 0 ? s_slot[to] - a.window + 1 : 0;
      }
    }
    int all_lo = 0, all_p = INT_MAX;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      all_lo = max(all_lo, lo[i]);
      all_p = min(all_p, p[i]);
    }
    all_lo = __reduce_max_sync(0xffffffffu, all_lo);
    all_p = __reduce_min_sync(0xffffffffu, all_p);
    float o[D / 16][NT][4];
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int w = 0; w < NT; ++w) o[d][w][0] = o[d][w][1] = o[d][w][2] = o[d][w][3] = 0.f;
    float m[2 * NT], l[2 * NT];
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
    int tile_rows = 0;  // of the tile
    float* kept = nullptr;
    if constexpr (SCORES) {
      while (tile_rows < 16 && token(row0 + tile_rows) >= 0) tile_rows += R <= 16 ? R : 1;
      kept = f.scores + ((size_t)unit * f.t_all + f.t_first + t) * min(R, 16) * f.scores_ld;
    }
    int done = 0, j0 = (s_b0[t] + cc.rec) * kBlock;
    // l is held relative to 2^m, O to 2^(m + E), where E is one number for all rows first, and a row's own from the stage on whose V's exponents lie too far apart
    int E = kLowExp - 1, e_low = INT_MAX;  // V's largest and smallest exponent so far
    float E_row[2 * NT];
    // A stage; false: its V's exponents lie too far from the others, nothing has happened
    auto weigh = [&](auto each) {
      constexpr bool EACH = decltype(each)::value;
      const int take = min(2, count - done);
      if (alive) alive = mbar_wait_bounded(&s_full[warp][slot], parity, dead);
      __syncwarp();
      const uint8_t* stage = ring + slot * 2 * REC;
      const uint32_t at = smem_u32(stage), second = take == 2 ? REC : 0;  // (a missing second record: the first again, with P = 0)
      const uint32_t tail_a = *reinterpret_cast<const uint32_t*>(stage + kBlock * 2 * D), tail_b = *reinterpret_cast<const uint32_t*>(stage + second + kBlock * 2 * D);
      const int ea = tail_ev(tail_a), eb = tail_ev(tail_b), e_new = max(E, max(ea, eb));
      if constexpr (!EACH) {
        e_low = min(e_low, min(ea, eb));
        if (e_new - e_low > kNear) return false;
      }
      float s[2][NT][4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t b[4];
          ldsm_x4_at(b, at + (r ? second : 0) + k_at + kk * 256);
#pragma unroll
          for (int y = 0; y < 2; ++y) {  // 16 entries each
            uint32_t a0, a1, a2, a3;
            widen(b[2 * y], a0, a2);
            widen(b[2 * y + 1], a1, a3);
#pragma unroll
            for (int w = 0; w < NT; ++w) mma_f16(s[r][w], a0, a1, a2, a3, qb[2 * kk + y][2 * w], qb[2 * kk + y][2 * w + 1]);
          }
        }
      }
      const bool inside = j0 >= all_lo && j0 + 31 <= all_p && take == 2;
      const float fe = EACH ? 1.f : pow2(max(E - e_new, -126)), fka = pow2(tail_ek(tail_a)), fkb = pow2(tail_ek(tail_b));
      float fo[2 * NT], ref[2 * NT];
      bool same = true;
#pragma unroll
      for (int i2 = 0; i2 < 2 * NT; ++i2) {
        const int w = i2 >> 1, e = i2 & 1;
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float fk = (r ? fkb : fka) * row_c[i2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float v = s[r][w][2 * y + e] * fk;
            if (a.cap > 0.f) v = fmaf(-2.f * cap2, __fdividef(1.f, ex2(at_most80(v * cap_c)) + 1.f), cap2);  // cap tanh(x) = cap - 2 cap / (e^(2 x) + 1)
            if (!inside) {
              const int j = j0 + 16 * r + tok[y];
              v = j >= lo[i2] && j <= p[i2] && r < take ? v : -INFINITY;
            }
            s[r][w][2 * y + e] = v;
            most[r] = fmaxf(most[r], v);
          }
        }
        const float mx = max_of_rows(fmaxf(m[i2], fmaxf(most[0], most[1])));
        ref[i2] = mx == -INFINITY ? 0.f : mx;
        const float fl = ex2(m[i2] - ref[i2]);
        if constexpr (EACH) {
          const float E_old = m[i2] == -INFINITY ? kNoneYet : E_row[i2] - (mx - m[i2]);
          E_row[i2] = fmaxf(E_old, max_of_rows(fmaxf(most[0] - ref[i2] + (float)ea, most[1] - ref[i2] + (float)eb)));
          fo[i2] = ex2(E_old - E_row[i2]);
        } else {
          fo[i2] = fl * fe;
        }
        same = same && fo[i2] == 1.f;
        m[i2] = mx;
        l[i2] *= fl;
      }
      if constexpr (!EACH) E = e_new;
      if constexpr (SCORES) {  // [slot][row of the tile]
#pragma unroll
        for (int w = 0; w < NT; ++w)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (r < take && j0 + 16 * r + kBlock <= f.scores_ld)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                float* dst = kept + (size_t)(j0 + 16 * r + tok[y]) * tile_rows + 8 * w + 2 * tq;
                const int left = tile_rows - 8 * w - 2 * tq;
                if (left >= 2 && tile_rows % 2 == 0) {
                  *reinterpret_cast<float2*>(dst) = make_float2(s[r][w][2 * y], s[r][w][2 * y + 1]);
                } else {
                  if (left >= 1) dst[0] = s[r][w][2 * y];
                  if (left >= 2) dst[1] = s[r][w][2 * y + 1];
                }
              }
      }
      if (__any_sync(0xffffffffu, !same)) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int w = 0; w < NT; ++w)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[d][w][k] *= fo[2 * w + (k & 1)];
      }
      uint32_t pb[2][2 * NT];  // of a record: tokens 4 tq, 4 tq + 1 and 4 tq + 2, 4 tq + 3 of row gq
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float fv = EACH ? 0.f : pow2(max((r ? eb : ea) - E, -100) + kTopP);
#pragma unroll
        for (int w = 0; w < NT; ++w) {
          uint32_t y[2];
          // (more than 2^85 only where the weights are nothing: a product with infinity would not be)
          auto own = [&](int i2) { return ex2(fminf((float)(r ? eb : ea) - E_row[i2], 85.f) + (float)kTopP); };
          const float f0 = EACH ? own(2 * w) : fv, f1 = EACH ? own(2 * w + 1) : fv;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float p0 = ex2(s[r][w][2 * n] - ref[2 * w]), p1 = ex2(s[r][w][2 * n + 1] - ref[2 * w + 1]);
            l[2 * w] += p0;
            l[2 * w + 1] += p1;
            y[n] = turned(pack_f16(p0 * f0, p1 * f1));
          }
          pb[r][2 * w] = tq < 2 ? y[0] : y[1];
          pb[r][2 * w + 1] = tq < 2 ? y[1] : y[0];
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldsm_x4_at(b, at + (mi & 2 ? second : 0) + v_at + d * 256);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t a0, a1, a2, a3;
          widen(b[2 * r], a0, a2);
          widen(b[2 * r + 1], a1, a3);
#pragma unroll
          for (int w = 0; w < NT; ++w) mma_f16(o[d][w], a0, a1, a2, a3, pb[r][2 * w], pb[r][2 * w + 1]);
        }
      }
      done += take;
      j0 += 2 * kBlock;
      __syncwarp();
      if (alive && p_take > 0) {  // this stage is free again
        ++issued;
        fence_async_smem();
        if (lane == 0) mbar_expect_tx(&s_full[warp][slot], p_take * REC);
        __syncwarp();
        if (lane < p_take) copy(slot, lane, p_src);
        step();
        if (lane < p_take) p_src = source(p_b0, p_off, p_g, pc.rec + lane);
      }
      if (++slot == ST) {
        slot = 0;
        parity ^= 1u;
      }
      return true;
    };
    bool near = true;
    while (near && done < count) near = weigh(std::false_type{});
    if (!near) {
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) E_row[i] = m[i] == -INFINITY ? kNoneYet : (float)E;
      while (done < count) weigh(std::true_type{});
    }
    // ---- the piece's state: the accumulated values are turned back in shared memory, so that rows leave in 16-byte pieces
    const bool whole = count == cc.n;
    const size_t part = (((size_t)who + (size_t)t * U + cc.u) * AB + mine) * (8 * NT);
#pragma unroll
    for (int w = 0; w < NT; ++w) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * w + 2 * tq + e, to = token(row0 + r), h = g * R + (to >= 0 ? head(row0 + r) : 0);
        float sum = l[2 * w + e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const float top = sum != sum ? INFINITY : m[2 * w + e];  // a NaN among the scores: no other piece may hide it
        float fac = near ? pow2(max(E, kLowExp) - kTopP) : ex2(E_row[2 * w + e] - (float)kTopP);  // (of a row that saw nothing: 0)
        if (whole) {
          const RowEnd end = row_end(top, sum, sink ? bf2f(sink[h]) : 0.f, sink != nullptr);
          fac *= end.factor;
          if (gq == 0 && to >= 0 && a.lse) a.lse[(size_t)to * a.H + h] = end.lse;
        } else if (gq == 0 && to >= 0) {
          a.part_ml[part + r] = make_float2(top, sum);
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          turn[(2 * tq + e) * TURN_LD + d * 16 + gq] = o[d][w][e] * fac;
          turn[(2 * tq + e) * TURN_LD + d * 16 + 8 + gq] = o[d][w][2 + e] * fac;
        }
      }
      __syncwarp();
      for (int r = 0; r < 8; ++r) {
        const int to = token(row0 + 8 * w + r);
        if (to < 0) continue;
        for (int d = lane * 4; d < D; d += 128) {
          const float4 v = *reinterpret_cast<const float4*>(turn + r * TURN_LD + d);
          if (whole) {
            bf16* dst = out + (size_t)to * a.out_ld + (g * R + head(row0 + 8 * w + r)) * D + d;
            if (f.out_by4) {
              *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
            } else {
              dst[0] = f2bf(v.x);
              dst[1] = f2bf(v.y);
              dst[2] = f2bf(v.z);
              dst[3] = f2bf(v.w);
            }
          } else {
            *reinterpret_cast<float4*>(a.part_o + (part + 8 * w + r) * D + d) = v;
          }
        }
      }
      __syncwarp();
    }
    x += count;
    cc.rec += count;
    if (x < x1) {
      next_tile(cc);
      load_q(cc);
    }
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
  const int row = (t - first) * R + h % R, u = h / R * O + row / 16, AB = f.abreast, U = f.U / AB;
  const int x0 = before * U + u / AB * n, w0 = x0 / run, pieces = n > 0 ? (x0 + n - 1) / run - w0 + 1 : 0;
  const size_t at = (((size_t)w0 + (size_t)first * U + u / AB) * AB + u % AB) * tile_rows + row % 16;  // of the first piece; the others so much further each:
  const size_t apart = (size_t)AB * tile_rows;
  float M = -INFINITY, den = 0.f;
  constexpr int PAIRS = D / 2, NP = (PAIRS + 31) / 32, AT_ONCE = 8 / NP;
  float2 acc[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) acc[i] = make_float2(0.f, 0.f);
  if (pieces > 1) {
    for (int s = lane; s < pieces; s += 32) M = fmaxf(M, a.part_ml[at + s * apart].x);
    M = warp_max(M);
    for (int s0 = part; s0 < pieces; s0 += AT_ONCE * share) {
      float2 v[AT_ONCE][NP], ml[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int s = s0 + k * share;
        ml[k] = s < pieces ? a.part_ml[at + s * apart] : make_float2(-INFINITY, 0.f);
        const float2* src = reinterpret_cast<const float2*>(a.part_o + (at + s * apart) * D) + lane;
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

// B200, 16 requests of 8200, 32 heads in 8 groups: 17 us for 17 MB of scores, over which every thread goes row by row.
// weights of the keys out of the kept scores and the finished lse, summed over a run's tokens and the group's heads in their order: a thread to (slot, kv head, run)
__global__ void __launch_bounds__(256) kv8_few_mass_kernel(FewArgs f) {
  pdl_wait();
  pdl_launch_dependents();
  const AttnArgs& a = f.a;
  const int t0 = blockIdx.z, g = blockIdx.y, R = a.H / a.pool.G, O = (R + 15) / 16, req = a.req[t0], j = blockIdx.x * 256 + threadIdx.x;
  if (t0 > 0 && a.req[t0 - 1] == req) return;  // a run's first token
  float sum = 0.f;
  bool any = false;
  for (int t = t0; t < a.T && a.req[t] == req;) {  // tiles: at most `per` tokens, none over the end of a launch of the first kernel
    const int most = min(f.per, min(a.T, (t / kFewTokens + 1) * kFewTokens) - t);
    int n = 1;
    while (n < most && a.req[t + n] == req) ++n;
    for (int o = 0; o < O; ++o) {
      const int rows = R <= 16 ? n * R : min(16, R - 16 * o);
      const float* s = f.scores + (((size_t)(g * O + o) * f.t_all + t) * min(R, 16)) * f.scores_ld + (size_t)j * rows;
      for (int r = 0; r < rows; ++r) {
        const int to = t + (R <= 16 ? r / R : 0), p = a.slots[to];
        if (j > p || (a.window > 0 && j <= p - a.window) || j >= f.scores_ld) continue;
        any = true;
        sum += ex2(s[r] - a.lse[(size_t)to * a.H + g * R + (R <= 16 ? r % R : 16 * o + r)] * kLog2e);
      }
    }
    t += n;
  }
  if (any && j < a.mass_ld) a.mass[((size_t)req * a.pool.G + g) * a.mass_ld + j] += sum;
}

template <int D, bool SCORES, bool WIDE>
static int launch_few(const bf16* q, const bf16* sink, bf16* out, const FewArgs& f, int ctas, cudaStream_t st) {
  constexpr size_t smem = (size_t)few_warps<D>() * (few_stages<D>() * 2 * (kBlock * 2 * D + 16) + 8 * (D + 4) * sizeof(float));
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_few_kernel<D, SCORES, WIDE>, smem); e != cudaSuccess) return (int)e;
  if (const cudaError_t e = launch(kv8_few_kernel<D, SCORES, WIDE>, dim3(ctas), dim3(few_warps<D>() * 32), smem, st, true, q, sink, out, f); e != cudaSuccess) return (int)e;
  // few rows have many pieces each
  const int rows = f.a.T * f.a.H, share = rows <= 4 * sm_count() ? 8 : rows <= 16 * sm_count() ? 2 : 1;
  return (int)follow(kv8_few_merge_kernel<D>, dim3((rows * share + 7) / 8), dim3(256), st, sink, out, share, WIDE ? 16 : 8, f);
}
template <int D>
static int launch_few(const bf16* q, const bf16* sink, bf16* out, const FewArgs& f, int ctas, bool wide, cudaStream_t st) {
  if (f.scores) return wide ? launch_few<D, true, true>(q, sink, out, f, ctas, st) : launch_few<D, true, false>(q, sink, out, f, ctas, st);
  return wide ? launch_few<D, false, true>(q, sink, out, f, ctas, st) : launch_few<D, false, false>(q, sink, out, f, ctas, st);
}

// Against the kernel for prompts (B200, us here : there, 32 heads of 128 in 8 groups): a portion behind 2000 of 48 tokens 38 : 56, 96 48 : 54, 256 85 : 60, behind 8000 of
// 32 54 : 52, 64 81 : 63, 256 234 : 89; 16 portions of 16 behind 2000 83 : 176, 8 of 32 83 : 95, 4 of 64 83 : 60; decoded tokens of 64 requests 69 : 2637 (there a tile's
// tokens belong to 64 requests, one after the other).  So up to 32 tokens of a request come here; with no word about them calls of up to 512 tokens, where a wrong guess
// costs a factor of 3 here and 40 there.  Against tiles (kv8_tile.cu), where the kernel for prompts does not take the heads' size: 64 behind 2000, 16 heads of 32 in 4
// groups, 29 : 53, 16 of 256 in one 70 : 113, 32 of 192 in 8 82 : 102; 256 73 : 65, 142 : 132, 286 : 198; six prompts of 608 618 : 104, 2347 : 324, 2461 : 596.
bool few_takes(int T, int H, int G, int dim, int vdim, int max_kv_len, int max_q_len) {
  if (T > 65535 || dim != vdim || !(dim == 32 || dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256)) return false;
  if ((long)std::min(T, kFewTokens) * G * ((H / G + 15) / 16) * (max_kv_len / kBlock + 2) >= 1L << 31) return false;
  const bool prompt = prompt_takes(T, H, G, dim, vdim);
  return T < 64 || (max_q_len > 0 ? max_q_len <= (prompt ? 32 : 64) : T <= kFewTokens) || !(prompt || tile_takes(T, H, G, max_q_len));
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
  n.scores = mass ? (size_t)U * T * std::min(H / G, 16) * n.scores_ld * sizeof(float) : 0;
  if (n.scores > kMostScores) n.scores = 0;
  return n;
}

int few_attention(const bf16* q, const bf16* sink, bf16* out, const AttnArgs& all, int max_q_len, const FewNeed& need, uint8_t* ws, cudaStream_t st) {
  const int D = all.pool.dim, R = all.H / all.pool.G;
  FewArgs f{};
  f.U = all.pool.G * ((R + 15) / 16);
  const bool wide = max_q_len <= 0 || R * max_q_len > 8;  // the rows of a tile do not fit into one product
  f.abreast = f.U % few_warps_of(D) == 0 ? few_warps_of(D) : few_warps_of(D) % f.U == 0 ? f.U : 1;
  f.per = wide ? std::max(1, 16 / R) : max_q_len;
  f.plan = reinterpret_cast<int*>(ws);
  f.scores = need.scores > 0 ? reinterpret_cast<float*>(ws + need.plan) : nullptr;
  f.scores_ld = need.scores_ld;
  f.t_all = all.T;
  f.inv_r = f.per > 1 ? (65536u + R - 1) / R : 0u;
  f.q_by4 = (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  f.out_by4 = (reinterpret_cast<uintptr_t>(out) & 7) == 0 && all.out_ld % 4 == 0;
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
    const int rc = D == 32    ? launch_few<32>(qt, sink, ot, f, ctas, wide, st)
                   : D == 64  ? launch_few<64>(qt, sink, ot, f, ctas, wide, st)
                   : D == 96  ? launch_few<96>(qt, sink, ot, f, ctas, wide, st)
                   : D == 128 ? launch_few<128>(qt, sink, ot, f, ctas, wide, st)
                   : D == 192 ? launch_few<192>(qt, sink, ot, f, ctas, wide, st)
                              : launch_few<256>(qt, sink, ot, f, ctas, wide, st);
    if (rc != 0) return rc;
  }
  if (!all.mass) return 0;
  if (!f.scores) return mass_rows(q, all, max_q_len, st);
  const int keys = (int)std::min((long)all.max_kv_len, all.mass_ld);
  f.a = all;
  return (int)follow(kv8_few_mass_kernel, dim3((keys + 255) / 256, all.pool.G, all.T), dim3(256), st, f);
}

}  // namespace kv8
}  // namespace pk
