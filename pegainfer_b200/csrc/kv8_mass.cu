// Weights of a prompt's keys, added up over its queries (kv8_attention.cuh), on the tensor cores: mass[j] += sum over the run's rows of 2^(s_j - lse).
//
// The scores are computed again from q and the finished lse: the products q K^T are half of the attention's work, and every key has one owner, who adds its weights in
// the rows' order.  A warp keeps 32 keys (16 from 192 entries on) as bf16 operands in registers, where e4m3 codes are exact; the run's rows pass by in tiles of 64
// through shared memory, as they are (mma.sync m16n8k16 in bf16, S^T = K q^T, fp32 sums).  A thread has the scores of two rows of four keys: the exponential and the sum
// over rows need no exchange.  The grid's z axis takes the runs by turns.
//
// Dims 64 and 128 go through tcgen05 instead (kv8_mass_wide_kernel); rows of q off 16-byte boundaries, fp32 and other dims through plain sums (kv8_mass_plain_kernel: the call below
// takes 1934 us instead of 141 with q on 2 bytes).  B200, two portions of 333 tokens behind 5003, 16 heads of 128 in 4 groups (54 Mi scores): 59 us, with
// mma.sync 89.
#include <algorithm>

#include "kv8_attention.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"

namespace pk {
namespace kv8 {

constexpr int kMassWarps = 4, kMassRows = 64, kMassTokens = 65536;  // of a launch, at most

// two codes -> two bf16
__device__ __forceinline__ uint32_t bf16_of(uint32_t two) {
  const float2 v = values2(two);
  return pack_bf16(v.x, v.y);
}

// ---- the runs, for all threads of a CTA alike
struct Runs {
  const uint32_t* starts;  // a bit per token that begins one
  int words, T;
  __device__ __forceinline__ int after(int t) const {  // the first run behind token t
    int i = (t + 1) >> 5;
    if (i >= words) return T;
    uint32_t m = starts[i] & (0xffffffffu << ((t + 1) & 31));
    while (m == 0 && ++i < words) m = starts[i];
    return m ? i * 32 + __ffs(m) - 1 : T;
  }
};
template <int WARPS>
__device__ __forceinline__ Runs find_runs(uint32_t* starts, const AttnArgs& a) {
  const int lane = threadIdx.x & 31, words = (a.T + 31) / 32;
#pragma unroll 4
  for (int i = threadIdx.x >> 5; i < words; i += WARPS) {
    const int t = i * 32 + lane;
    const bool begins = t < a.T && (t == 0 || a.req[t] != a.req[t - 1]);
    const uint32_t all = __ballot_sync(0xffffffffu, begins);
    if (lane == 0) starts[i] = all;
  }
  __syncthreads();
  return Runs{starts, words, a.T};
}
// a run's largest and smallest slot, where they are, and the rows without a slot between them: the others' slots ascend by one at least
struct Ends {
  int last, at_last, lowest, at_lowest, holes;
};
template <int WARPS>
struct RunRoom {
  int4 ends[WARPS];
  int valid[WARPS];
};
template <int WARPS>
__device__ __forceinline__ Ends run_ends(RunRoom<WARPS>& room, const AttnArgs& a, int t0, int t1) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int last = -1, lowest = INT_MAX, at_last = -1, at_lowest = INT_MAX, valid = 0;
  for (int t = t0 + (int)threadIdx.x; t < t1; t += WARPS * 32) {
    const int p = a.slots[t];
    valid += p >= 0;
    if (p >= 0 && p >= last) last = p, at_last = t;
    if (p >= 0 && p < lowest) lowest = p, at_lowest = t;
  }
  const int wl = __reduce_max_sync(0xffffffffu, last), ws = __reduce_min_sync(0xffffffffu, lowest), wv = __reduce_add_sync(0xffffffffu, valid);
  const int al = __reduce_max_sync(0xffffffffu, last == wl ? at_last : -1), as = __reduce_min_sync(0xffffffffu, lowest == ws ? at_lowest : INT_MAX);
  __syncthreads();  // (the words of a run before)
  if (lane == 0) {
    room.ends[warp] = make_int4(wl, al, ws, as);
    room.valid[warp] = wv;
  }
  __syncthreads();
  const int4 x = room.ends[lane % WARPS];
  Ends e;
  e.last = __reduce_max_sync(0xffffffffu, x.x);
  e.at_last = __reduce_max_sync(0xffffffffu, x.x == e.last ? x.y : -1);
  e.lowest = __reduce_min_sync(0xffffffffu, x.z);
  e.at_lowest = __reduce_min_sync(0xffffffffu, x.z == e.lowest ? x.w : INT_MAX);
  e.holes = e.last < 0 ? 0 : e.at_last - e.at_lowest + 1 - (int)__reduce_add_sync(0xffffffffu, lane < WARPS ? room.valid[lane] : 0);
  return e;
}
// rows of a run that may see one of the keys key0 .. key1: from the first (before it the slots are below key0) to the second (from it on key1 is outside the window)
struct Span {
  int from, to;
};
__device__ __forceinline__ Span run_span(const Ends& e, int t0, int t1, int key0, int key1, int window) {
  return Span{max(t0, e.at_last - (e.last - key0) - e.holes), window > 0 ? (int)min((long)t1, (long)e.at_lowest + e.holes + (key1 + (long)window - e.lowest)) : t1};
}

template <int D, int RECS>
__global__ void __launch_bounds__(kMassWarps * 32) kv8_mass_kernel(const bf16* __restrict__ q, AttnArgs a) {
  constexpr int LD = D + 8;
  extern __shared__ __align__(16) bf16 ms_q[];  // [2][rows][LD]
  __shared__ __align__(8) float s_lse[2][kMassRows];  // log2; +inf: no such row
  __shared__ __align__(8) int s_p[2][kMassRows];
  __shared__ uint32_t ms_starts[kMassTokens / 32];
  __shared__ RunRoom<kMassWarps> s_run;
  __shared__ int s_half[2][2];  // whether 32 rows see every key of the CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3, g = blockIdx.y, R = a.H / a.pool.G, V = a.pool.vdim;
  const int b0 = (blockIdx.x * kMassWarps + warp) * RECS;  // the warp's first record
  const int key0 = blockIdx.x * kMassWarps * RECS * kBlock, key1 = key0 + kMassWarps * RECS * kBlock - 1;
  const float c = a.scale * kLog2e, cap2 = a.cap * kLog2e, cap_c = a.cap > 0.f ? 2.f * a.scale / a.cap * kLog2e : 0.f;
  pdl_wait();
  pdl_launch_dependents();
  const Runs runs = find_runs<kMassWarps>(ms_starts, a);
  int nth = 0;
  for (int t0 = 0, t1 = 0; t0 < a.T; t0 = t1, ++nth) {
    t1 = runs.after(t0);
    if (nth % (int)gridDim.z != (int)blockIdx.z) continue;
    const int req = a.req[t0];
    const Ends ends = run_ends<kMassWarps>(s_run, a, t0, t1);
    const int last = ends.last, lowest = ends.lowest;
    if (key0 > last || (a.window > 0 && key1 <= lowest - a.window)) continue;  // (for all threads alike)

    // the warp's keys: a product's 16 tokens are a record's, its inner index the entries in order
    uint32_t ka[RECS][D / 16][4];
    float fk[RECS];
#pragma unroll
    for (int r = 0; r < RECS; ++r) {
      fk[r] = 0.f;
      const bool there = (b0 + r) * kBlock <= last;
      const uint8_t* rec = there ? a.pool.record(req, (b0 + r) * kBlock, g) : nullptr;
      if (there) fk[r] = pow2(tail_ek(*reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V)))) * (a.cap > 0.f ? 1.f : c);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x)  // tokens gq (+ 8), entries 2 tq (+ 8)
          ka[r][k][x] = there ? bf16_of(*reinterpret_cast<const uint16_t*>(rec + (x & 1) * (8 * D) + k * 128 + gq * 16 + 2 * tq + (x >> 1) * 8)) : 0u;
    }
    float sum[RECS][2];
#pragma unroll
    for (int r = 0; r < RECS; ++r) sum[r][0] = sum[r][1] = 0.f;

    const int rows = (t1 - t0) * R, tiles = (rows + kMassRows - 1) / kMassRows;
    auto load = [&](int tile, int s) {
      bf16* dst = ms_q + (size_t)s * kMassRows * LD;
      for (int i = threadIdx.x; i < kMassRows * (D / 8); i += kMassWarps * 32) {
        const int row = i / (D / 8), piece = i % (D / 8), at = min(tile * kMassRows + row, rows - 1), t = t0 + at / R;
        cp_async16(dst + row * LD + piece * 8, q + ((size_t)t * a.H + g * R + at % R) * D + piece * 8);
      }
      if (threadIdx.x < kMassRows) {
        const int at = tile * kMassRows + threadIdx.x, t = t0 + min(at, rows - 1) / R, p = at < rows ? a.slots[t] : -1;
        s_p[s][threadIdx.x] = p;
        s_lse[s][threadIdx.x] = p >= 0 ? a.lse[(size_t)t * a.H + g * R + at % R] * kLog2e : INFINITY;
        const bool all = p >= key1 && (a.window <= 0 || key0 > p - a.window);
        if (threadIdx.x < 32) {  // (two halves of the rows)
          s_half[s][0] = __all_sync(0xffffffffu, all);
        } else {
          s_half[s][1] = __all_sync(0xffffffffu, all);
        }
      }
      cp_async_commit();
    };
    const auto [from, to] = run_span(ends, t0, t1, key0, key1, a.window);
    const int tile0 = (int)((long)(from - t0) * R / kMassRows), tile1 = min(tiles, (int)(((long)(to - t0) * R + kMassRows - 1) / kMassRows));
    int s = 0;
    if (tile0 < tile1) load(tile0, 0);
    for (int tile = tile0; tile < tile1; ++tile) {
      if (tile + 1 < tile1) load(tile + 1, s ^ 1);
      else cp_async_commit();
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      const bf16* qt = ms_q + (size_t)s * kMassRows * LD;
      const bool whole = s_half[s][0] && s_half[s][1];
#pragma unroll 1
      for (int n = 0; n < kMassRows / 8; n += 2) {  // two chains of products
        float acc[2][RECS][4] = {};
#pragma unroll
        for (int k = 0; k < D / 32; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t b[4];
            ldsm_x4(b, qt + ((n + x) * 8 + (lane & 7)) * LD + k * 32 + (lane >> 3) * 8);
#pragma unroll
            for (int r = 0; r < RECS; ++r) {
              mma_bf16_16816(acc[x][r], ka[r][2 * k], b[0], b[1]);
              mma_bf16_16816(acc[x][r], ka[r][2 * k + 1], b[2], b[3]);
            }
          }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = (n + x) * 8 + 2 * tq;
          const float2 lse = *reinterpret_cast<const float2*>(&s_lse[s][row]);
          const int2 p = *reinterpret_cast<const int2*>(&s_p[s][row]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int r = 0; r < RECS; ++r)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                float w;
                if (a.cap > 0.f) {
                  const float v = fmaf(-2.f * cap2, __fdividef(1.f, ex2(at_most80(acc[x][r][2 * y + e] * fk[r] * cap_c)) + 1.f), cap2);
                  w = ex2(v - (e ? lse.y : lse.x));
                } else {
                  w = ex2(fmaf(acc[x][r][2 * y + e], fk[r], e ? -lse.y : -lse.x));
                }
                if (!whole) {
                  const int j = (b0 + r) * kBlock + 8 * y + gq, pe = e ? p.y : p.x;
                  w = j <= pe && (a.window <= 0 || j > pe - a.window) ? w : 0.f;
                }
                sum[r][y] += w;
              }
        }
      }
      __syncthreads();
      s ^= 1;
    }
#pragma unroll
    for (int r = 0; r < RECS; ++r)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float v = sum[r][y];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        const int j = (b0 + r) * kBlock + 8 * y + gq;
        if (tq == 0 && j <= last && j < a.mass_ld) a.mass[((size_t)req * a.pool.G + g) * a.mass_ld + j] += v;
      }
    __syncthreads();  // the next run's rows may come
  }
}

// ---- the same on tcgen05: S^T of 128 keys x 128 rows in tensor memory, K as bf16 and the rows of q as they are in shared memory (128-byte swizzle).  A thread has a key and
// half of the rows: the exponent is one number, the sums need no exchange until the end.  The product of the next tile runs under the exponentials of this one, which bound
// it (one per score, 16 a clock and SM); two CTAs to an SM cover one another's waits.
// {s0, s1} += 2^(x f + n), two at a time
__device__ __forceinline__ void add_weights(float& s0, float& s1, uint32_t x0, uint32_t x1, float f, float n0, float n1) {
  unsigned long long x, y, z;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(x0), "r"(x1));
  asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(f));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(n0), "f"(n1));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(x) : "l"(y), "l"(z));
  float w0, w1;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(w0), "=f"(w1) : "l"(x));
  w0 = ex2(w0);
  w1 = ex2(w1);
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(w0), "f"(w1));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(s0), "f"(s1));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(x));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(s0), "=f"(s1) : "l"(y));
}

constexpr int kWideKeys = 128, kWideRows = 128, kWideWarps = 8;

template <int D>
__global__ void __launch_bounds__(kWideWarps * 32, 2) kv8_mass_wide_kernel(const bf16* __restrict__ q, AttnArgs a, unsigned int* err) {
  constexpr int HALF = 128 * 128, TILE = HALF * (D / 64);  // bytes of 64 entries of 128 rows, of an operand
  extern __shared__ uint8_t mw_raw[];
  uint8_t* ks = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(mw_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = ks + TILE;  // [2]
  __shared__ __align__(16) float s_neg[4][kWideRows];  // -lse in log2; -inf: no such row.  (Four: a tile's are read while the next but one's come.)
  __shared__ __align__(16) int s_p[4][kWideRows];
  __shared__ int s_all[4][kWideRows / 32];  // whether 32 rows see every key of the CTA
  __shared__ uint32_t ms_starts[kMassTokens / 32];
  __shared__ RunRoom<kWideWarps> s_run;
  __shared__ uint64_t s_full[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int s_dead;
  volatile int* dead = &s_dead;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.y, R = a.H / a.pool.G, V = a.pool.vdim;
  const int key0 = blockIdx.x * kWideKeys, key1 = key0 + kWideKeys - 1;
  const int key = key0 + (warp & 3) * 32 + lane, col0 = (warp >> 2) * 64;
  const float cap2 = a.cap * kLog2e, cap_c = a.cap > 0.f ? 2.f * a.scale / a.cap * kLog2e : 0.f;
  if (tid == 0) {
    mbar_init(s_full, 1);
    mbar_init(s_full + 1, 1);
    mbar_init(&drained, 1);
    s_dead = 0;
    mbar_fence_init();
  }
  if (warp == 0) tmem_alloc(&tmem_slot, 2 * kWideRows);
  pdl_wait();
  pdl_launch_dependents();
  tc_fence_before();
  const Runs runs = find_runs<kWideWarps>(ms_starts, a);  // (a barrier)
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  WaitTries tries;
  const unsigned long long r_inv = (1ull << 32) / (unsigned)R + 1;  // at / R is exact for at < 2^32 / R
  int nth = 0, n = 0;  // n: tiles so far
  for (int t0 = 0, t1 = 0; t0 < a.T; t0 = t1, ++nth) {
    t1 = runs.after(t0);
    if (nth % (int)gridDim.z != (int)blockIdx.z) continue;
    const int req = a.req[t0];
    const Ends ends = run_ends<kWideWarps>(s_run, a, t0, t1);
    const int last = ends.last, lowest = ends.lowest;
    if (key0 > last || (a.window > 0 && key1 <= lowest - a.window)) continue;  // (for all threads alike)
    const int rows = (t1 - t0) * R, tiles = (rows + kWideRows - 1) / kWideRows;
    const auto [from, to] = run_span(ends, t0, t1, key0, key1, a.window);
    const int tile0 = (int)((long)(from - t0) * R / kWideRows), count = min(tiles, (int)(((long)(to - t0) * R + kWideRows - 1) / kWideRows)) - tile0;
    const bf16* q_run = q + ((size_t)t0 * a.H + g * R) * D;
    auto by_r = [&](int at) { return (int)((unsigned long long)(uint32_t)at * r_inv >> 32); };
    int next_p = -1;
    float next_lse = INFINITY;
    auto load = [&](int i) {  // the run's i-th tile
      uint8_t* dst = qs + (size_t)((n + i) & 1) * TILE;
      const int at0 = (tile0 + i) * kWideRows;
#pragma unroll 4
      for (int x = tid; x < kWideRows * (D / 8); x += kWideWarps * 32) {
        const int row = x / (D / 8), piece = x % (D / 8), at = min(at0 + row, rows - 1);
        cp_async16(dst + (piece >> 3) * HALF + row * 128 + (((piece & 7) ^ (row & 7)) << 4), q_run + ((size_t)by_r(at) * (a.H - R) + at) * D + piece * 8);
      }
      cp_async_commit();
      next_p = -1, next_lse = INFINITY;
      if (tid < kWideRows && at0 + tid < rows) {
        const int at = at0 + tid, t = by_r(at);
        next_p = a.slots[t0 + t];
        next_lse = a.lse[(size_t)(t0 + t) * a.H + g * R + at - t * R];
      }
    };
    auto put = [&](int i) {  // and what came with it, a tile's exponentials later
      if (tid < kWideRows) {
        const int s = (n + i) & 3;
        s_p[s][tid] = next_p;
        s_neg[s][tid] = next_p >= 0 ? next_lse * -kLog2e : -INFINITY;
        const bool all = __all_sync(0xffffffffu, next_p >= key1 && (a.window <= 0 || key0 > next_p - a.window));
        if (lane == 0) s_all[s][warp] = all;
      }
    };
    if (count > 0) load(0);
    // the keys
#pragma unroll 4
    for (int x = tid; x < kWideKeys * (D / 16); x += kWideWarps * 32) {
      const int r = x / D, u = x % D, row = r * kBlock + (u >= D / 2 ? 8 : 0) + (u & 7), c = (u % (D / 2)) >> 3;
      uint32_t w[8] = {};
      if (key0 + r * kBlock <= last) {
        const uint4 codes = *reinterpret_cast<const uint4*>(a.pool.record(req, key0 + r * kBlock, g) + u * 16);
        const uint32_t four[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = bf16_of(four[i / 2] >> (i % 2 * 16) & 0xffffu);
      }
      uint8_t* dst = ks + (c >> 2) * HALF + row * 128;
      *reinterpret_cast<uint4*>(dst + (((c & 3) * 2 ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(dst + (((c & 3) * 2 + 1 ^ (row & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
    }
    float fk = 0.f;
    if (key / kBlock <= last / kBlock)
      fk = pow2(tail_ek(*reinterpret_cast<const uint32_t*>(a.pool.record(req, key, g) + kBlock * (D + V)))) * (a.cap > 0.f ? cap_c : a.scale * kLog2e);

    float sum0 = 0.f, sum1 = 0.f;
    for (int i = 0; i <= count; ++i) {
      if (i < count) {
        put(i);
        cp_async_wait_all();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (warp == 0 && tc_elect_one()) {
          tc_fence_after();
          constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kWideRows >> 3) << 17) | ((uint32_t)(kWideKeys >> 4) << 24);  // bf16 x bf16 -> fp32
          const uint64_t kd = make_sw128_desc(smem_u32(ks)), qd = make_sw128_desc(smem_u32(qs + (size_t)((n + i) & 1) * TILE));
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tmem + (uint32_t)(((n + i) & 1) * kWideRows), kd + (uint64_t)((k >> 2) * (HALF >> 4) + (k & 3) * 2), qd + (uint64_t)((k >> 2) * (HALF >> 4) + (k & 3) * 2), idesc, k > 0 ? 1u : 0u);
          umma_commit(s_full + ((n + i) & 1));
        }
        __syncwarp();
      }
      const int m = n + i - 1, s = m & 3;  // the tile before
      if (i > 0) {
        mbar_wait_bounded(s_full + (m & 1), (uint32_t)((m >> 1) & 1), dead, tries);
        tc_fence_after();
      }
      if (i + 1 < count) load(i + 1);  // its place was the tile before's
      if (i == 0) continue;
      uint32_t v[64];
      tmem_ld64(tmem + (uint32_t)((m & 1) * kWideRows + col0) + ((uint32_t)((warp & 3) * 32) << 16), v);
      const bool whole = s_all[s][col0 / 32] && s_all[s][col0 / 32 + 1];
      if (a.cap > 0.f) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          v[j] = __float_as_uint(fmaf(-2.f * cap2, __fdividef(1.f, ex2(at_most80(__uint_as_float(v[j]) * fk)) + 1.f), cap2));
      }
      const float f = a.cap > 0.f ? 1.f : fk;
      if (whole) {
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          const float4 neg = *reinterpret_cast<const float4*>(&s_neg[s][col0 + j]);
          add_weights(sum0, sum1, v[j], v[j + 1], f, neg.x, neg.y);
          add_weights(sum0, sum1, v[j + 2], v[j + 3], f, neg.z, neg.w);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          const int p = s_p[s][col0 + j];
          const float w = ex2(fmaf(__uint_as_float(v[j]), f, s_neg[s][col0 + j]));
          (j & 1 ? sum1 : sum0) += key <= p && (a.window <= 0 || key > p - a.window) ? w : 0.f;
        }
      }
    }
    n += max(count, 0);
    // both halves of the rows
    sum0 += sum1;
    __syncthreads();
    float* other = reinterpret_cast<float*>(ks);  // (the products are done)
    if (warp >= 4) other[tid - 128] = sum0;
    __syncthreads();
    if (warp < 4 && key <= last && key < a.mass_ld) a.mass[((size_t)req * a.pool.G + g) * a.mass_ld + key] += *dead ? NAN : sum0 + other[tid];
    tc_fence_before();
    __syncthreads();  // the next run's keys may come
    tc_fence_after();
  }
  tc_fence_before();
  __syncthreads();
  if (*dead) {  // (for all alike, behind the barrier)
    if (warp == 0) {
      if (tc_elect_one()) umma_commit(&drained);
      __syncwarp();
      mbar_drain(&drained, 0);
    }
    __syncthreads();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kWideRows);
  }
  if (tid == 0) count_run_out(dead, err);
}

template <int D>
static int launch_mass_wide(const bf16* q, const AttnArgs& a, int runs, cudaStream_t st) {
  constexpr size_t smem = 1024 + (size_t)3 * 256 * D;
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_mass_wide_kernel<D>, smem); e != cudaSuccess) return (int)e;
  const long span = std::min((long)a.max_kv_len, a.mass_ld);
  ThreadState& ts = tls();
  const bool pdl = ts.pdl;
  ts.pdl = true;  // behind a kernel of the same call
  const cudaError_t e = launch(kv8_mass_wide_kernel<D>, dim3((unsigned)((span + kWideKeys - 1) / kWideKeys), a.pool.G, std::max(1, std::min(runs, 16))), dim3(kWideWarps * 32), smem, st, true, q, a,
                               wait_err_word());
  ts.pdl = pdl;
  return (int)e;
}

template <int D, int RECS>
static int launch_mass(const bf16* q, const AttnArgs& a, int runs, cudaStream_t st) {
  constexpr size_t smem = (size_t)2 * kMassRows * (D + 8) * sizeof(bf16);
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_mass_kernel<D, RECS>, smem); e != cudaSuccess) return (int)e;
  constexpr int keys = kMassWarps * RECS * kBlock;
  const long span = std::min((long)a.max_kv_len, a.mass_ld);
  ThreadState& ts = tls();
  const bool pdl = ts.pdl;
  ts.pdl = true;  // behind a kernel of the same call
  const cudaError_t e = launch(kv8_mass_kernel<D, RECS>, dim3((unsigned)((span + keys - 1) / keys), a.pool.G, runs), dim3(kMassWarps * 32), smem, st, true, q, a);
  ts.pdl = pdl;
  return (int)e;
}
template <int D>
static int launch_mass(const bf16* q, const AttnArgs& a, int runs, cudaStream_t st) {
  runs = std::max(1, std::min(runs, 16));
  // half as many keys to a warp where the others would leave the SMs with fewer than four CTAs
  if constexpr (D <= 128)
    if (std::min((long)a.max_kv_len, a.mass_ld) / (kMassWarps * 2 * kBlock) * a.pool.G * runs >= 4L * sm_count()) return launch_mass<D, 2>(q, a, runs, st);
  return launch_mass<D, 1>(q, a, runs, st);
}
// ---- any sizes and types, in fp32: a CTA to a record, its warps to four rows of the run at a time; their sums come together in the warps' order.  Two lanes have a
// token's key, half of the entries each.  (fp32, 36 tokens of 16 heads of 128 in 4 groups: the whole call 37 us; with a warp to a record 164.)
constexpr int kPlainWarps = 8, kPlainRows = 4;

template <typename E>
__global__ void __launch_bounds__(kPlainWarps * 32) kv8_mass_plain_kernel(const E* __restrict__ q, AttnArgs a) {
  __shared__ uint32_t ms_starts[kMassTokens / 32];
  __shared__ RunRoom<kPlainWarps> s_run;
  __shared__ float s_sum[kPlainWarps][kBlock];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x, g = blockIdx.y, R = a.H / a.pool.G;
  const int D = a.pool.dim, V = a.pool.vdim, tok = lane & 15, part = lane >> 4, chunks = D / 32, key0 = b * kBlock, key1 = key0 + kBlock - 1, j = key0 + tok;
  const float c = a.scale * kLog2e;
  const Runs runs = find_runs<kPlainWarps>(ms_starts, a);
  int nth = 0;
  for (int t0 = 0, t1 = 0; t0 < a.T; t0 = t1, ++nth) {
    t1 = runs.after(t0);
    if (nth % (int)gridDim.z != (int)blockIdx.z) continue;
    const int req = a.req[t0];
    const Ends ends = run_ends<kPlainWarps>(s_run, a, t0, t1);
    const int last = ends.last, lowest = ends.lowest;
    if (key0 > last || (a.window > 0 && key1 <= lowest - a.window)) continue;  // (for all threads alike)
    const auto [from, to] = run_span(ends, t0, t1, key0, key1, a.window);
    const uint8_t* rec = a.pool.record(req, key0, g);
    const float ek = pow2(tail_ek(*reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V))));
    const uint8_t* k = rec + (tok >> 3) * (8 * D) + part * chunks * 128 + (tok & 7) * 16;
    float sum = 0.f;
    const long rows = (long)(to - from) * R;
    for (long i0 = warp * kPlainRows; i0 < rows; i0 += kPlainWarps * kPlainRows) {
      const E* x[kPlainRows];
      size_t row[kPlainRows];
      int p[kPlainRows];
#pragma unroll
      for (int i = 0; i < kPlainRows; ++i) {
        const long at = min(i0 + i, rows - 1);
        const int t = from + (int)(at / R);
        row[i] = (size_t)t * a.H + g * R + (int)(at % R);
        x[i] = q + row[i] * D + part * chunks * 16;
        p[i] = i0 + i < rows ? a.slots[t] : -1;
      }
      float s[kPlainRows] = {};
      for (int n = 0; n < chunks; ++n) {
        float v[16];
        values16(*reinterpret_cast<const uint4*>(k + n * 128), v);
#pragma unroll
        for (int i = 0; i < kPlainRows; ++i)
#pragma unroll
          for (int d = 0; d < 16; ++d) s[i] = fmaf(v[d], to_f(x[i][n * 16 + d]), s[i]);
      }
#pragma unroll
      for (int i = 0; i < kPlainRows; ++i) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 16);
        if (j <= p[i] && (a.window <= 0 || j > p[i] - a.window)) sum += exp2f(shaped(s[i] * ek, c, a.cap) - a.lse[row[i]] * kLog2e);
      }
    }
    if (part == 0) s_sum[warp][tok] = sum;
    __syncthreads();
    if (warp == 0 && part == 0 && j <= last && j < a.mass_ld) {
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < kPlainWarps; ++w) all += s_sum[w][tok];
      a.mass[((size_t)req * a.pool.G + g) * a.mass_ld + j] += all;
    }
    __syncthreads();  // the next run's sums may come
  }
}

static int mass_mma(const bf16* q, const AttnArgs& a, int runs, cudaStream_t st) {
  switch (a.pool.dim) {
    case 32: return launch_mass<32>(q, a, runs, st);
    case 64: return launch_mass_wide<64>(q, a, runs, st);
    case 96: return launch_mass<96>(q, a, runs, st);
    case 128: return launch_mass_wide<128>(q, a, runs, st);
    case 192: return launch_mass<192>(q, a, runs, st);
    default: return launch_mass<256>(q, a, runs, st);
  }
}
template <typename E>
int mass_rows(const E* q, const AttnArgs& a, int max_q_len, cudaStream_t st) {
  const int T = a.T, D = a.pool.dim;
  // a launch's rows are counted in an int and divided by R through a product, which is exact below 2^32 / R rows
  const long R = a.H / a.pool.G;
  const int most = (int)std::min((long)kMassTokens, ((1L << 32) - 1) / (R * R));
  for (int t0 = 0; t0 < T; t0 += most) {  // (a run that a launch's end cuts is added up in both)
    AttnArgs x = a;
    x.T = std::min(most, T - t0);
    x.slots += t0;
    x.req += t0;
    x.lse += (size_t)t0 * a.H;
    const E* rows = q + (size_t)t0 * a.H * D;
    const int runs = max_q_len > 0 ? (x.T + max_q_len - 1) / max_q_len : 4;  // at least; unknown: some
    if constexpr (sizeof(E) == 2)
      if ((D == 32 || D == 64 || D == 96 || D == 128 || D == 192 || D == 256) && (reinterpret_cast<uintptr_t>(q) & 15) == 0) {
        if (const int rc = mass_mma(rows, x, runs, st); rc != 0) return rc;
        continue;
      }
    const long span = std::min((long)a.max_kv_len, a.mass_ld);
    const dim3 grid((unsigned)((span + kBlock - 1) / kBlock), a.pool.G, std::max(1, std::min(runs, 64)));
    if (const cudaError_t e = follow(kv8_mass_plain_kernel<E>, grid, dim3(kPlainWarps * 32), st, rows, x); e != cudaSuccess) return (int)e;
  }
  return 0;
}
template int mass_rows<float>(const float*, const AttnArgs&, int, cudaStream_t);
template int mass_rows<bf16>(const bf16*, const AttnArgs&, int, cudaStream_t);

}  // namespace kv8
}  // namespace pk
