// Attention over the 8-bit paged cache for many rows of fp32 activations or of key and value sizes that the tcgen05 kernel does not have (kv8.cuh, kv8_attention.cuh).
//
// A CTA has 64 rows of one kv head (the group's query heads of consecutive tokens), a warp 16 of them, and goes through the keys in blocks of 64, run by run where its
// tokens belong to several requests (the other rows are masked).  Records come whole, by asynchronous copies, a block ahead.
//   * mma.sync m16n8k16 in f16: codes widen exactly.  A row of q is scaled by a power of two that puts its largest entry at 2^14 .. 2^15; bf16 entries fit one f16 (down to
//     2^-21 of the row's largest), fp32 ones go in as the nearest f16 and the rest (22 bits).  So do the weights P, held 2^15 times too large.
//   * The inner indices of both products are permuted so that four consecutive codes are what a thread needs of K (entries) and of V (tokens).
//   * K's exponents multiply the scores, V's go into P relative to the row's largest (score + exponent) so far, m + X: what a row does not see, or gives no weight, costs its
//     other tokens no bits, however large its values.  m and X are whole numbers, so that every rescaling is exact.
// Bound by the products where rows are many: two of them for each fp32 one.
#include <algorithm>

#include "kv8_attention.cuh"
#include "mma.cuh"

namespace pk {
namespace kv8 {

constexpr int kTileWarps = 4, kTileRows = kTileWarps * 16, kTileRecs = 4, kTileKeys = kTileRecs * kBlock;
constexpr int kNone = -1000;  // X of a row that has seen nothing

__device__ __forceinline__ void rest_f16(float lo, float hi, uint32_t near, uint32_t& rest) {
  const float2 n = __half22float2(*reinterpret_cast<const __half2*>(&near));
  rest = pack_f16(lo - n.x, hi - n.y);
}

// VM: the values' size at most
template <typename E, int VM>
__global__ void __launch_bounds__(kTileWarps * 32, VM > 128 ? 2 : VM > 64 || sizeof(E) == 4 ? 3 : 4) kv8_tile_kernel(const E* __restrict__ q, const E* __restrict__ sink, E* __restrict__ out, AttnArgs a, int per, int slices) {
  constexpr int PARTS = sizeof(E) == 4 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t tl_sm[];
  __shared__ int s_slot[kTileRows], s_req[kTileRows];
  const int D = a.pool.dim, V = a.pool.vdim, G = a.pool.G, R = a.H / G, REC = record_bytes(D, V), LD = D + 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  const int g = blockIdx.y / slices, slice = blockIdx.y % slices;
  const int t0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * per, n_tok = min(per, a.T - t0);  // late tokens, which see most, first
  __half* qs = reinterpret_cast<__half*>(tl_sm);  // [part][row][LD]
  uint8_t* ring = tl_sm + (size_t)PARTS * kTileRows * LD * 2;  // [2][records]
  pdl_wait();
  pdl_launch_dependents();
  for (int i = tid; i < n_tok; i += kTileWarps * 32) {
    s_slot[i] = a.slots[t0 + i];
    s_req[i] = a.req[t0 + i];
  }
  auto token = [&](int r) { return R <= kTileRows ? (r / R < n_tok ? r / R : -1) : (slice * kTileRows + r < R ? 0 : -1); };  // of the CTA's; -1: no such row
  auto head = [&](int r) { return g * R + (R <= kTileRows ? r % R : slice * kTileRows + r); };

  // ---- q: a warp's 16 rows, one after the other
  float row_c[2] = {0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int r = warp * 16 + i, k = token(r);
    const E* src = q + ((size_t)(t0 + max(k, 0)) * a.H + (k >= 0 ? head(r) : 0)) * D;
    float v[8], amax = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      v[x] = k >= 0 && lane + 32 * x < D ? to_f(src[lane + 32 * x]) : 0.f;
      amax = fmaxf(amax, fabsf(v[x]));
    }
    amax = warp_max(amax);
    const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - kTopQ, kLowExp), kHighExp);
    const float down = pow2(-e), c = amax == INFINITY ? NAN : pow2(e);  // (an infinite entry: the row is NaN)
    if (i == gq) row_c[0] = c;
    if (i == gq + 8) row_c[1] = c;
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (lane + 32 * x < D) {
        const __half near = __float2half_rn(v[x] * down);
        qs[r * LD + lane + 32 * x] = near;
        if (PARTS == 2) qs[(kTileRows + r) * LD + lane + 32 * x] = __float2half_rn(v[x] * down - __half2float(near));
      }
  }
  __syncthreads();
  int p[2], lo[2], mine[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    mine[i] = token(warp * 16 + gq + 8 * i);
    p[i] = mine[i] >= 0 ? s_slot[mine[i]] : -1;
    lo[i] = p[i] >= 0 && a.window > 0 ? p[i] - a.window + 1 : 0;
  }

  // ---- the blocks of the tokens' runs, one after the other
  struct Step {
    int from, to;          // tokens of the run, of the CTA's
    int j, last, top, off;  // block, last block, last record, page table
  };
  auto enter = [&](Step& x, int from) {  // the first run from token `from` on that has a block
    for (; from < n_tok; from = x.to) {
      x.from = from;
      x.to = from + 1;
      int high = s_slot[from], low = high < 0 ? INT_MAX : high;
      while (x.to < n_tok && s_req[x.to] == s_req[from]) {
        const int s = s_slot[x.to++];
        high = max(high, s);
        if (s >= 0) low = min(low, s);
      }
      if (high < 0) continue;
      x.j = a.window > 0 ? max(0, low - a.window + 1) / kTileKeys : 0;
      x.last = high / kTileKeys;
      x.top = high / kBlock;
      x.off = a.pool.page_off[s_req[from]];
      return;
    }
    x.from = n_tok;
  };
  auto next = [&](Step& x) {
    if (x.j < x.last) ++x.j;
    else enter(x, x.to);
  };
  Step now;
  enter(now, 0);
  int left = INT_MAX;
  if (gridDim.z > 1) {  // this CTA's share of them
    int all = 0;
    for (Step x = now; x.from < n_tok; enter(x, x.to)) all += x.last - x.j + 1;
    const int each = (all + (int)gridDim.z - 1) / (int)gridDim.z;
    int skip = min(each * (int)blockIdx.z, all);
    left = min(each, all - skip);
    while (skip > 0) {
      const int here = min(skip, now.last - now.j + 1);
      skip -= here;
      if (now.j + here <= now.last) now.j += here;
      else enter(now, now.to);
    }
  }
  const int rpp = a.pool.page_size / kBlock, pieces = REC / 16;
  auto load = [&](const Step& x, int s) {
    uint8_t* dst = ring + (size_t)s * kTileRecs * REC;
#pragma unroll
    for (int r = 0; r < kTileRecs; ++r) {
      const int b = x.j * kTileRecs + r;
      if (b > x.top) break;
      const uint8_t* src = a.pool.data + (size_t)a.pool.pages[x.off + b / rpp] * a.pool.page_stride + (size_t)(g * rpp + b % rpp) * REC;
      for (int i = tid; i < pieces; i += kTileWarps * 32) cp_async16(dst + r * REC + i * 16, src + i * 16);
    }
    cp_async_commit();
  };

  float o[VM / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < VM / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const float c = a.scale * kLog2e;
  const int mi = lane >> 3, mr = lane & 7, mt = 4 * (mr >> 1) + (mr & 1) + 2 * (mi & 1);
  const uint32_t k_at = (uint32_t)((mt >> 3) * (8 * D) + (mi >> 1) * 128 + (mt & 7) * 16), v_at = (uint32_t)(kBlock * D + (mi * 8 + mr) * 16);
  const uint32_t ring_at = smem_u32(ring);
  const uint32_t* q_row = reinterpret_cast<const uint32_t*>(qs + (warp * 16 + gq) * LD + 4 * tq);
  int X[2] = {kNone, kNone}, s = 0;  // l is held relative to 2^m, O to 2^(m + X)
  if (now.from < n_tok && left > 0) load(now, 0);
  while (now.from < n_tok && left > 0) {
    Step after = now;
    next(after);
    --left;
    if (after.from < n_tok && left > 0) load(after, s ^ 1);
    else cp_async_commit();
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const int recs = min(kTileRecs, now.top - now.j * kTileRecs + 1);
    const uint32_t at = ring_at + (uint32_t)(s * kTileRecs * REC);
    float acc[kTileRecs][2][4] = {};
    for (int k = 0; k < D / 32; ++k) {
      uint32_t x[PARTS][2][4];  // two chunks of 16 entries
#pragma unroll
      for (int w = 0; w < PARTS; ++w)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t* row = q_row + (w * kTileRows * LD + k * 32 + y * 16) / 2;
          const uint2 u = *reinterpret_cast<const uint2*>(row), v = *reinterpret_cast<const uint2*>(row + 4 * LD);
          x[w][y][0] = u.x, x[w][y][1] = v.x, x[w][y][2] = u.y, x[w][y][3] = v.y;
        }
#pragma unroll
      for (int r = 0; r < kTileRecs; ++r) {
        if (r >= recs) break;
        uint32_t b[4];
        ldsm_x4_at(b, at + (uint32_t)(r * REC) + k_at + (uint32_t)(k * 256));
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t b0, b1;
            widen(b[2 * y + n], b0, b1);
#pragma unroll
            for (int w = 0; w < PARTS; ++w) mma_f16(acc[r][n], x[w][y][0], x[w][y][1], x[w][y][2], x[w][y][3], b0, b1);
          }
      }
    }
    // scores: this thread's tokens of a record are 4 tq + 2 n + e, its rows gq and gq + 8
    int ev[kTileRecs];
    float mx[2] = {-INFINITY, -INFINITY}, high[2] = {-INFINITY, -INFINITY};  // largest score, and with V's exponent added
#pragma unroll
    for (int r = 0; r < kTileRecs; ++r) {
      ev[r] = kLowExp;
      if (r < recs) {
        const uint32_t tail = *reinterpret_cast<const uint32_t*>(ring + ((size_t)s * kTileRecs + r) * REC + kBlock * (D + V));
        const float fk = pow2(tail_ek(tail));
        ev[r] = tail_ev(tail);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float f = fk * row_c[i];
          float most = -INFINITY;
          const bool in = mine[i] >= now.from && mine[i] < now.to;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = now.j * kTileKeys + r * kBlock + 4 * tq + 2 * n + e;
              const float v = in && j >= lo[i] && j <= p[i] ? shaped(acc[r][n][2 * i + e] * f, c, a.cap) : -INFINITY;
              acc[r][n][2 * i + e] = v;
              most = fmaxf(most, v);
            }
          mx[i] = fmaxf(mx[i], most);
          high[i] = fmaxf(high[i], most + (float)ev[r]);
        }
      }
    }
    float fo[2], ref[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float m_new = fmaxf(m[i], ceilf(mx[i]));
      ref[i] = m_new == -INFINITY ? 0.f : m_new;
      high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], 1));
      high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], 2));
      const float e = fmaf(fabsf(ref[i]), 1.2e-7f, high[i] - ref[i]);  // (and what its sum was rounded by, so that P stays in range)
      const int grown = m[i] == -INFINITY ? 0 : (int)fminf(m_new - m[i], 2000.f), X_old = X[i] - grown;
      X[i] = max(X_old, (int)ceilf(fminf(fmaxf(e, (float)kNone), 1000.f)));
      fo[i] = pow2(max(X_old - X[i], -126));
      l[i] *= pow2(max(-grown, -126));
      m[i] = m_new;
    }
    if (fo[0] != 1.f || fo[1] != 1.f) {
#pragma unroll
      for (int i = 0; i < VM / 8; ++i) {
        o[i][0] *= fo[0], o[i][1] *= fo[0];
        o[i][2] *= fo[1], o[i][3] *= fo[1];
      }
    }
#pragma unroll
    for (int r = 0; r < kTileRecs; ++r) {
      if (r >= recs) break;
      uint32_t x[PARTS][4];
      float up[2];  // (more than 2^100 only where the weights are nothing)
#pragma unroll
      for (int i = 0; i < 2; ++i) up[i] = pow2(min(max(ev[r] - X[i], -110), 100) + kTopP);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w0 = ex2(acc[r][n][2 * i] - ref[i]), w1 = ex2(acc[r][n][2 * i + 1] - ref[i]);
          l[i] += w0 + w1;
          x[0][2 * n + i] = pack_f16(w0 * up[i], w1 * up[i]);
          if (PARTS == 2) rest_f16(w0 * up[i], w1 * up[i], x[0][2 * n + i], x[PARTS - 1][2 * n + i]);
        }
#pragma unroll
      for (int d = 0; d < VM / 32; ++d) {
        if (d * 32 >= V) break;
        uint32_t b[4];
        ldsm_x4_at(b, at + (uint32_t)(r * REC) + v_at + (uint32_t)(d * 32 * 16));
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          uint32_t b0, b1;
          widen(b[y], b0, b1);
#pragma unroll
          for (int w = 0; w < PARTS; ++w) mma_f16(o[4 * d + y], x[w][0], x[w][1], x[w][2], x[w][3], b0, b1);
        }
      }
    }
    __syncthreads();  // the next but one's records may come
    s ^= 1;
    now = after;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // ---- results: rows gq and gq + 8, entries 8 i + 2 tq + e
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float unit = pow2(max(X[i], kLowExp) - kTopP);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (mine[i] < 0) continue;
    const int t = t0 + mine[i], h = head(warp * 16 + gq + 8 * i);
    const size_t row = (size_t)t * a.H + h;
    const float top = l[i] != l[i] ? INFINITY : m[i];  // a NaN among the scores: no other share may hide it
    const bool whole = gridDim.z == 1;
    const RowEnd end = row_end(top, l[i], sink ? to_f(sink[h]) : 0.f, sink != nullptr);
    const float f = whole ? end.factor * unit : unit;
    float* part = a.part_o + ((size_t)blockIdx.z * a.T * a.H + row) * V;
    E* dst = out + (size_t)t * a.out_ld + (size_t)h * V;
#pragma unroll
    for (int d = 0; d < VM / 8; ++d)
      if (d * 8 < V)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float v = o[d][2 * i + e] * f;
          if (whole) dst[d * 8 + 2 * tq + e] = from_f<E>(v);
          else part[d * 8 + 2 * tq + e] = v;
        }
    if (tq == 0) {
      if (!whole) a.part_ml[(size_t)blockIdx.z * a.T * a.H + row] = make_float2(top, l[i]);
      else if (a.lse) a.lse[row] = end.lse;
    }
  }
}

template <typename E, int VM>
static int launch_tile(const E* q, const E* sink, E* out, const AttnArgs& a, int shares, cudaStream_t st) {
  const int R = a.H / a.pool.G, per = std::max(1, kTileRows / R), slices = (R + kTileRows - 1) / kTileRows, D = a.pool.dim;
  const size_t parts = sizeof(E) == 4 ? 2 : 1, smem = parts * kTileRows * (D + 16) * 2 + (size_t)2 * kTileRecs * record_bytes(D, a.pool.vdim);
  static std::atomic<uint64_t> set{0};
  constexpr size_t most = (sizeof(E) == 4 ? 2 : 1) * kTileRows * (256 + 16) * 2 + (size_t)2 * kTileRecs * (kBlock * (256 + VM) + 16);
  if (const cudaError_t e = allow_smem(set, (const void*)kv8_tile_kernel<E, VM>, most); e != cudaSuccess) return (int)e;
  return (int)launch(kv8_tile_kernel<E, VM>, dim3((a.T + per - 1) / per, a.pool.G * slices, shares), dim3(kTileWarps * 32), smem, st, true, q, sink, out, a, per, slices);
}
template <typename E>
int tile_attention(const E* q, const E* sink, E* out, const AttnArgs& a, int shares, cudaStream_t st) {
  return a.pool.vdim <= 64    ? launch_tile<E, 64>(q, sink, out, a, shares, st)
         : a.pool.vdim <= 128 ? launch_tile<E, 128>(q, sink, out, a, shares, st)
                              : launch_tile<E, 256>(q, sink, out, a, shares, st);
}
template int tile_attention<float>(const float*, const float*, float*, const AttnArgs&, int, cudaStream_t);
template int tile_attention<bf16>(const bf16*, const bf16*, bf16*, const AttnArgs&, int, cudaStream_t);

// Against the kernel with a CTA to a row (B200, us here : there).  fp32, 32 heads of 128 in 8 groups: portions behind 2000 of 16 tokens 98 : 75, 64 91 : 229, 256 159 : 760;
// 16 portions behind 500 of 4 tokens 217 : 73, 8 123 : 121, 16 80 : 229; decoded tokens of 64 requests 790 : 80; a prompt of 1024 168 : 821.  fp32, 8 heads of 64 in 8
// groups (a tile has 64 tokens): 64 behind 2000 71 : 52, 256 73 : 154, 16 portions of 16 behind 500 170 : 55.  So it takes a thousand rows with few requests in a tile;
// with no word about those, calls of more than 512 tokens.
bool tile_takes(int T, int H, int G, int max_q_len) {
  return (long)T * H >= 1024 && (max_q_len > 0 ? max_q_len >= std::max(1, kTileRows / (H / G)) && max_q_len >= 8 : T > 512);
}
// as many CTAs as two to an SM, and eight blocks of keys to a share at least
int tile_shares(int T, int H, int G, int max_kv_len, int window) {
  const int R = H / G, per = std::max(1, kTileRows / R);
  const long ctas = (long)((T + per - 1) / per) * G * ((R + kTileRows - 1) / kTileRows);
  const int span = window > 0 ? (int)std::min((long)max_kv_len, (long)window + per) : max_kv_len;
  return (int)std::max(1L, std::min(2L * sm_count() / ctas, (long)span / (8 * kTileKeys)));
}

}  // namespace kv8
}  // namespace pk
