// Append to the 8-bit paged cache (kv8.cuh): rotation of q and k, quantisation of k and v, record by record.
//
// The tokens of a request are consecutive rows with consecutive slots.  The first of them that falls into a record is the record's leader; its warp writes the
// record whole.  Where the leader's slot is the record's first, the record begins anew (what the page held before is forgotten, slots behind the last token are
// zero); else the record goes on: its exponent is the larger of the old one and what the new tokens need, and the old codes are rounded again where it grew.
//
// q' = rot(q), k' = rot(k): pairs (i, i + dims/2) or (2i, 2i + 1) of the first `dims` entries turn by positions * freq[i].  The angle is reduced to turns in 64
// bits (a float product is off by 0.004 at position 100000), the sine and cosine and the rotation are fp32.
//
// Bound by the rows' bytes, read and (q) written once; a tenth of that are codes.  Two kernels: one that keeps a record in registers, for bf16 rows on 16-byte boundaries
// with rotated dimensions a multiple of 32, and a general one through shared memory.  B200, 4096 tokens of 32 heads of q and 8 of k and v of 128 (93 MB): 22.6 us
// (4.1 TB/s; records alone 10, q alone 12) and 49 in the general one.
//
// The general kernel: a CTA looks at 16 tokens, a table of their sines and cosines in shared memory, then a warp to every (record, kv head), then all threads over q.  The
// grid's y axis shares a window's work out, so that few tokens still fill the GPU.
#include <algorithm>

#include "kv8.cuh"

namespace pk {
namespace kv8 {

constexpr int kAppendWarps = 4;
constexpr int kWindow = 16;

// 8 consecutive entries as floats
template <typename E>
__device__ __forceinline__ void load8(const E* p, bool vec, float (&v)[8]) {
  if constexpr (sizeof(E) == 2) {
    if (vec) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(w[i]);
        v[2 * i + 1] = bf16_hi(w[i]);
      }
      return;
    }
  } else {
    if (vec) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f(p[i]);
}
template <typename E>
__device__ __forceinline__ void store8(E* p, bool vec, const float (&v)[8]) {
  if constexpr (sizeof(E) == 2) {
    if (vec) {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      return;
    }
  } else {
    if (vec) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = from_f<E>(v[i]);
}

struct AppendArgs {
  const int *positions, *slots, *req;
  Pool pool;
  const float* freq;
  float mag;
  int ld, H, T, dims, interleaved, vec;
};

// rows [at, at + count) of a projection's part into shared memory (fp32), with the bias; returns the rows with an entry that is not finite
template <typename E>
__device__ __forceinline__ uint32_t load_rows(float* rows, const E* src, const E* bias, int ld, int at, int count, int width, bool vec, int lane) {
  const int per = width / 8, many = 32 / per, sub = lane / per, piece = lane % per;
  uint32_t bad = 0;
  for (int r0 = 0; r0 < count; r0 += many) {
    const int r = r0 + sub;
    bool odd = false;
    if (sub < many && r < count) {
      float v[8];
      load8(src + (size_t)r * ld + piece * 8, vec, v);
      if (bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += to_f(bias[piece * 8 + i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) odd |= (__float_as_uint(v[i]) & 0x7f800000u) == 0x7f800000u;
      float4* d = reinterpret_cast<float4*>(rows + (at + r) * row_ld(width) + piece * 8);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    const uint32_t who = __ballot_sync(0xffffffffu, odd);
    for (int i = 0; i < many; ++i)
      if (who >> (i * per) & ((1u << (per - 1) << 1) - 1u)) bad |= 1u << (at + r0 + i);
  }
  __syncwarp();
  return bad;
}

template <typename E>
__global__ void __launch_bounds__(kAppendWarps * 32) kv8_append_kernel(const E* __restrict__ qkv, const E* __restrict__ bias, E* __restrict__ q_out, AppendArgs a) {
  extern __shared__ __align__(16) float ap_sm[];
  __shared__ uint32_t s_lead;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = a.dims >> 1;
  const int w0 = blockIdx.x * kWindow, n_tok = min(kWindow, a.T - w0);
  const int D = a.pool.dim, V = a.pool.vdim, G = a.pool.G, H = a.H;
  float2* table = reinterpret_cast<float2*>(ap_sm);                                            // [token][pair] cosine, sine
  float* rows = ap_sm + kWindow * half * 2 + warp * kBlock * row_ld(max(D, V));
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 0) {  // which tokens of the window lead a record
    bool lead = false;
    const int t = w0 + lane;
    if (lane < n_tok) {
      const int slot = a.slots[t];
      lead = slot >= 0 && (slot % kBlock == 0 || t == 0 || a.req[t - 1] != a.req[t] || a.slots[t - 1] != slot - 1);
    }
    const uint32_t all = __ballot_sync(0xffffffffu, lead);
    if (lane == 0) s_lead = all;
  }
  for (int i = threadIdx.x; i < n_tok * half; i += blockDim.x) {
    const int tok = i / half, f = i - tok * half;
    const double turns = (double)a.positions[w0 + tok] * (double)a.freq[f] * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    table[i] = make_float2(c * a.mag, s * a.mag);
  }
  __syncthreads();

  // ---- records
  const uint32_t leads = s_lead;
  const int items = __popc(leads) * G;
  for (int it = blockIdx.y * kAppendWarps + warp; it < items; it += gridDim.y * kAppendWarps) {
    const int g = it % G, tok = __fns(leads, 0, it / G + 1), t = w0 + tok;
    const int slot = a.slots[t], req = a.req[t], first = slot % kBlock;
    const bool mine = lane + first < kBlock && t + lane < a.T && a.req[min(t + lane, a.T - 1)] == req && a.slots[min(t + lane, a.T - 1)] == slot + lane;
    const int count = __ffs(~__ballot_sync(0xffffffffu, mine)) - 1;  // tokens of this record in the call (lane 16 and up never count)
    uint8_t* rec = a.pool.record(req, slot, g);
    const uint32_t fresh = ((1u << count) - 1u) << first, none = ~(fresh | ((1u << first) - 1u)) & 0xffffu;
    const uint32_t tail = first ? *reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V)) : 0u;
    const E* src = qkv + (size_t)t * a.ld;

    // values
    uint8_t* vdst = rec + kBlock * D;
    if (first) {
      const float f = pow2(tail_ev(tail));
      for (int d = lane; d < V; d += 32) {
        float v[16];
        values16(*reinterpret_cast<const uint4*>(vdst + d * 16), v);
        for (int r = 0; r < first; ++r) rows[r * row_ld(V) + d] = v[r] * f;
      }
    }
    const uint32_t bad_v = load_rows(rows, src + H * D + G * D + g * V, bias ? bias + H * D + G * D + g * V : nullptr, a.ld, first, count, V, a.vec, lane);
    int ev = exponent_for(rows_amax(rows, V, fresh & ~bad_v, lane));
    if (first) ev = max(ev, tail_ev(tail));
    emit_v(vdst, rows, V, ev, bad_v | none, lane);
    __syncwarp();

    // keys
    uint32_t bad_old = 0;
    if (first) {
      const float f = pow2(tail_ek(tail));
      for (int u = lane; u < D; u += 32) {
        const int r = (u >= D / 2 ? 8 : 0) + (u & 7), c = (u % (D / 2)) >> 3;
        if (r < first) {
          const uint4 code = *reinterpret_cast<const uint4*>(rec + u * 16);
          if ((code.x & 0x7fu) == 0x7fu) bad_old |= 1u << r;
          float v[16];
          values16(code, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) rows[r * row_ld(D) + c * 16 + i] = v[i] * f;
        }
      }
      bad_old = __reduce_or_sync(0xffffffffu, bad_old);
    }
    const uint32_t bad_k = load_rows(rows, src + H * D + g * D, bias ? bias + H * D + g * D : nullptr, a.ld, first, count, D, a.vec, lane) | bad_v;
    for (int i = lane; i < count * half; i += 32) {
      const int r = i / half, f = i - r * half;
      float* row = rows + (first + r) * row_ld(D);
      // the table has the window's 16 tokens; a record that reaches into the next one has its own angles
      float2 cs;
      if (tok + r < n_tok) {
        cs = table[(tok + r) * half + f];
      } else {
        const double turns = (double)a.positions[t + r] * (double)a.freq[f] * 0.15915494309189533577;
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        cs = make_float2(c * a.mag, s * a.mag);
      }
      const int i1 = a.interleaved ? 2 * f : f, i2 = a.interleaved ? 2 * f + 1 : f + half;
      const float x = row[i1], y = row[i2];
      row[i1] = x * cs.x - y * cs.y;
      row[i2] = x * cs.y + y * cs.x;
    }
    for (int r = 0; r < kBlock; ++r)
      if (none >> r & 1)
        for (int d = lane; d < D; d += 32) rows[r * row_ld(D) + d] = 0.f;
    __syncwarp();
    int ek = exponent_for(rows_amax(rows, D, fresh & ~bad_k, lane));
    if (first) ek = max(ek, tail_ek(tail));
    emit_k(rec, rows, D, ek, bad_k | bad_old, lane);
    if (lane == 0) emit_tail(rec + kBlock * (D + V), ek, ev);
    __syncwarp();
  }

  // ---- queries: a thread takes eight pairs (or eight entries that only pass)
  const bool by8 = a.interleaved ? a.dims % 8 == 0 : half % 8 == 0;
  if (by8) {
    const int turn = a.interleaved ? a.dims / 8 : half / 8, pass = (D - a.dims) / 8, units = turn + pass;
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < n_tok * H * units; i += gridDim.y * blockDim.x) {
      const int u = i % units, h = i / units % H, tok = i / units / H;
      const size_t from = (size_t)(w0 + tok) * a.ld + h * D, to = ((size_t)(w0 + tok) * H + h) * D;
      const E* b = bias ? bias + h * D : nullptr;
      auto get = [&](int d, float (&v)[8]) {
        load8(qkv + from + d, a.vec, v);
        if (b) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += to_f(b[d + k]);
        }
      };
      float x[8], y[8];
      if (u >= turn) {
        get(a.dims + (u - turn) * 8, x);
        store8(q_out + to + a.dims + (u - turn) * 8, a.vec, x);
      } else if (a.interleaved) {
        get(u * 8, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 cs = table[tok * half + u * 4 + k];
          y[2 * k] = x[2 * k] * cs.x - x[2 * k + 1] * cs.y;
          y[2 * k + 1] = x[2 * k] * cs.y + x[2 * k + 1] * cs.x;
        }
        store8(q_out + to + u * 8, a.vec, y);
      } else {
        get(u * 8, x);
        get(half + u * 8, y);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 cs = table[tok * half + u * 8 + k];
          const float p = x[k], q = y[k];
          x[k] = p * cs.x - q * cs.y;
          y[k] = p * cs.y + q * cs.x;
        }
        store8(q_out + to + u * 8, a.vec, x);
        store8(q_out + to + half + u * 8, a.vec, y);
      }
    }
  } else {
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < n_tok * H * D; i += gridDim.y * blockDim.x) {
      const int d = i % D, h = i / D % H, tok = i / D / H;
      const size_t from = (size_t)(w0 + tok) * a.ld + h * D;
      auto get = [&](int k) { return to_f(qkv[from + k]) + (bias ? to_f(bias[h * D + k]) : 0.f); };
      float v = get(d);
      if (d < a.dims) {
        const int f = a.interleaved ? d >> 1 : d < half ? d : d - half;
        const bool one = a.interleaved ? (d & 1) == 0 : d < half;
        const float o = get(a.interleaved ? d ^ 1 : one ? d + half : d - half);
        const float2 cs = table[tok * half + f];
        v = one ? v * cs.x - o * cs.y : o * cs.y + v * cs.x;
      }
      q_out[((size_t)(w0 + tok) * H + h) * D + d] = from_f<E>(v);
    }
  }
}


// ---- bf16 rows on 16-byte boundaries, rotated dimensions a multiple of 32: everything in registers.
//
// The first CTAs take records, a warp to each (record, kv head); the rest take q.
//   K    a lane has units of 16 entries of a token two by two, those that turn into one another: (u, u + dims/2) or 16 consecutive pairs
//   V    a lane has two entries of all 16 tokens: the code's 16 tokens of an entry need no transposition
// A window (16 tokens of the call) in which no token follows another in its record, as decoded ones, takes a shorter way: 8 tokens of 8 requests 10.6 us, 13.3 without.
// All loads are under way before the first angle is there.  Where a record goes on under its old exponent of K, K's old codes are not touched.
constexpr int kTurnRows = 32;  // a window's tokens, and those of its last record

// FAST, for q: the angle, within half a turn, goes to the special-function unit, 2^-21 off, where the results are rounded to 2^-9.  (With the library's sine and cosine two
// of five instructions of the kernel were q's angles.)  Not for k: an error next to 448 * 2^e changes a record's exponent.
template <bool FAST>
__device__ __forceinline__ float2 turn_of(int position, double freq, float mag) {  // freq in turns
  const double turns = (double)position * freq;
  const float part = (float)(turns - rint(turns));
  float s, c;
  if (FAST) {
    s = __sinf(part * 6.2831853071795865f);
    c = __cosf(part * 6.2831853071795865f);
  } else {
    sincospif(2.f * part, &s, &c);
  }
  return make_float2(c * mag, s * mag);
}
// eight pairs: (x[j], y[j]), or side by side in x and then y
__device__ __forceinline__ void turn_pairs(float* x, float* y, const float2 (&cs)[8], int side_by_side) {
  if (side_by_side) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float* z = j < 4 ? x + 2 * j : y + 2 * j - 8;
      const float p = z[0], r = z[1];
      z[0] = p * cs[j].x - r * cs[j].y;
      z[1] = p * cs[j].y + r * cs[j].x;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = x[j], r = y[j];
      x[j] = p * cs[j].x - r * cs[j].y;
      y[j] = p * cs[j].y + r * cs[j].x;
    }
  }
}
constexpr double kTurns = 0.15915494309189533577;  // 1 / 2 pi
// the set bit that has n set bits below it
__device__ __forceinline__ int nth_bit(uint32_t bits, int n) {
  for (int i = 0; i < n; ++i) bits &= bits - 1u;
  return __ffs(bits) - 1;
}
// the larger magnitude of bf16 pairs, as bits
__device__ __forceinline__ uint32_t larger2(uint32_t most, uint32_t two) { return __vmaxu2(most, two & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t larger_of(uint32_t most) { return max(most >> 16, most & 0xffffu); }
__device__ __forceinline__ void widen8(const uint4& u, float* v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
  }
}
__device__ __forceinline__ uint4 narrow8(const float* v) { return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])); }
__device__ __forceinline__ bool odd_one(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
// 16 codes under an exponent `down` = 2^(old - new) -> under the new one
__device__ __forceinline__ uint4 again16(const uint4& old, float down) {
  float v[16];
  values16(old, v);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = codes4(v[4 * i] * down, v[4 * i + 1] * down, v[4 * i + 2] * down, v[4 * i + 3] * down);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// a token alone in its record, by one warp
template <int N>
__device__ __forceinline__ void append_one(const bf16* row, const bf16* bias, const AppendArgs& a, int t, int g, int lane) {
  const int D = a.pool.dim, V = a.pool.vdim, G = a.pool.G, H = a.H, half = a.dims >> 1;
  const int slot = a.slots[t], pos = slot & (kBlock - 1);
  const bf16* k_src = row + (H + g) * D;
  const bf16* v_src = row + (H + G) * D + g * V;
  const bf16* k_bias = bias ? bias + (H + g) * D : nullptr;
  const bf16* v_bias = bias ? bias + (H + G) * D + g * V : nullptr;
  // pairs of K, those that only pass two by two behind the others; entries of V
  float x[N], y[N], v[2 * N];
  int ix[N], iy[N];
  const int at = a.positions[t];
  float2 cs[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int p = lane + 32 * n;
    const bool turns = p < half;
    ix[n] = a.interleaved || !turns ? 2 * p : p;
    iy[n] = a.interleaved || !turns ? 2 * p + 1 : p + half;
    x[n] = y[n] = v[2 * n] = v[2 * n + 1] = 0.f;
    cs[n] = make_float2(1.f, 0.f);
    if (2 * p < D) {
      x[n] = to_f(k_src[ix[n]]);
      y[n] = to_f(k_src[iy[n]]);
      if (turns) cs[n].x = a.freq[p];
    }
    if (2 * p < V) {
      const uint32_t two = *reinterpret_cast<const uint32_t*>(v_src + 2 * p);
      v[2 * n] = bf16_lo(two);
      v[2 * n + 1] = bf16_hi(two);
    }
  }
  uint8_t* rec = a.pool.record(a.req[t], slot, g);
  uint8_t* vdst = rec + kBlock * D;
  uint4 old[2 * N];
  uint32_t tail = 0;
#pragma unroll
  for (int n = 0; n < 2 * N; ++n) old[n] = make_uint4(0, 0, 0, 0);
  if (pos) {
    tail = *reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V));
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (2 * (lane + 32 * n) < V) {
        old[2 * n] = *reinterpret_cast<const uint4*>(vdst + (lane + 32 * n) * 2 * kBlock);
        old[2 * n + 1] = *reinterpret_cast<const uint4*>(vdst + (lane + 32 * n) * 2 * kBlock + kBlock);
      }
  }
  bool bad_k = false, bad_v = false;
  float most_k = 0.f, most_v = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int p = lane + 32 * n;
    if (2 * p < D) {
      if (k_bias) {
        x[n] += to_f(k_bias[ix[n]]);
        y[n] += to_f(k_bias[iy[n]]);
      }
      bad_k |= odd_one(x[n]) || odd_one(y[n]);
      if (p < half) {
        cs[n] = turn_of<false>(at, (double)cs[n].x * kTurns, a.mag);
        const float x0 = x[n], y0 = y[n];
        x[n] = x0 * cs[n].x - y0 * cs[n].y;
        y[n] = x0 * cs[n].y + y0 * cs[n].x;
      }
      most_k = fmaxf(most_k, fmaxf(fabsf(x[n]), fabsf(y[n])));
    }
    if (2 * p < V) {
      if (v_bias) {
        v[2 * n] += to_f(v_bias[2 * p]);
        v[2 * n + 1] += to_f(v_bias[2 * p + 1]);
      }
      bad_v |= odd_one(v[2 * n]) || odd_one(v[2 * n + 1]);
      most_v = fmaxf(most_v, fmaxf(fabsf(v[2 * n]), fabsf(v[2 * n + 1])));
    }
  }
  bad_v = __any_sync(0xffffffffu, bad_v);
  bad_k = __any_sync(0xffffffffu, bad_k) || bad_v;
  int ek = exponent_for(bad_k ? 0.f : warp_max(most_k)), ev = exponent_for(bad_v ? 0.f : warp_max(most_v));
  const int had_k = tail_ek(tail), had_v = tail_ev(tail);
  if (pos) {
    ek = max(ek, had_k);
    ev = max(ev, had_v);
  }
  // V: the token's byte, zeros behind it
  const float down_k = pow2(-ek), down_v = pow2(-ev), move = pow2(max(had_v - ev, -126));
#pragma unroll
  for (int n = 0; n < 2 * N; ++n) {
    const int d = 2 * (lane + 32 * (n >> 1)) + (n & 1);
    if (d >= V) continue;
    uint4 o = old[n];
    if (pos && ev != had_v) o = again16(o, move);
    const uint32_t code = bad_v ? 0u : codes2(v[n] * down_v, 0.f) & 0xffu;
    uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int keep = min(max(pos - 4 * i, 0), 4);
      w[i] = keep == 4 ? w[i] : (w[i] & ((1u << (8 * keep)) - 1u)) | (pos >> 2 == i ? code << (8 * keep) : 0u);
    }
    *reinterpret_cast<uint4*>(vdst + d * kBlock) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // K: the token's bytes; rows behind it zero, rows before it again where the exponent grew
  const float again = pow2(max(had_k - ek, -126));
  const bool grown = pos && ek != had_k;
#pragma unroll 1
  for (int u = lane; u < D; u += 32) {
    const int r = (u >= D / 2 ? 8 : 0) + (u & 7);
    uint4* unit = reinterpret_cast<uint4*>(rec + u * 16);
    if (r > pos) *unit = make_uint4(0, 0, 0, 0);
    else if (grown && r < pos) *unit = again16(*unit, again);
  }
  uint8_t* k_row = rec + (pos >= 8 ? 8 * D : 0) + (pos & 7) * 16;
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (2 * (lane + 32 * n) < D) {
      const uint32_t two = bad_k ? 0x7f7fu : codes2(x[n] * down_k, y[n] * down_k);
      k_row[(ix[n] >> 4) * 128 + (ix[n] & 15)] = (uint8_t)two;
      k_row[(iy[n] >> 4) * 128 + (iy[n] & 15)] = (uint8_t)(two >> 8);
    }
  if (lane == 0) emit_tail(rec + kBlock * (D + V), ek, ev);
}

struct WideArgs {
  AppendArgs a;
  int rec_ctas, rec_parts;  // CTAs of records: windows * rec_parts
  int by;                   // heads that a thread of q turns by the same angles
};

// N: 64ths of the larger width
template <int N, bool BIAS>
__global__ void __launch_bounds__(kAppendWarps * 32, N <= 2 ? 4 : 2) kv8_append_wide_kernel(const bf16* __restrict__ qkv, const bf16* __restrict__ bias, bf16* __restrict__ q_out, const WideArgs f) {
  extern __shared__ __align__(16) float2 ap_turns[];  // [token][pair], rows 16 bytes apart from a multiple of the banks
  const AppendArgs& a = f.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = a.dims >> 1;
  const int D = a.pool.dim, V = a.pool.vdim, G = a.pool.G, H = a.H;
  pdl_wait();
  pdl_launch_dependents();

  if ((int)blockIdx.x >= f.rec_ctas) {
    // ---- queries: 16 entries (eight pairs, or eight and eight of those that only pass) of `by` heads
    const int units = D / 16, groups = (H + f.by - 1) / f.by;
    const uint32_t i = (blockIdx.x - f.rec_ctas) * blockDim.x + threadIdx.x, row = i / units;
    if (i >= (uint32_t)(a.T * units * groups)) return;
    const int u = (int)(i - row * units), t = (int)(row % a.T), h0 = (int)(row / a.T) * f.by, h1 = min(h0 + f.by, H);
    const bool turns = u < half / 8;
    const int d0 = turns ? (a.interleaved ? u * 16 : u * 8) : a.dims + (u - half / 8) * 16, d1 = turns && !a.interleaved ? d0 + half : d0 + 8;
    const bf16* src = qkv + (size_t)t * a.ld;
    bf16* dst = q_out + (size_t)t * H * D;
    float2 cs[8];
    for (int h = h0; h < h1; h += 4) {
      uint4 raw[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (h + k < h1) {
          raw[k][0] = *reinterpret_cast<const uint4*>(src + (h + k) * D + d0);
          raw[k][1] = *reinterpret_cast<const uint4*>(src + (h + k) * D + d1);
        }
      if (h == h0 && turns) {
        const int at = a.positions[t];
#pragma unroll
        for (int k = 0; k < 8; ++k) cs[k] = turn_of<true>(at, (double)a.freq[u * 8 + k] * kTurns, a.mag);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (h + k < h1) {
          float x[8], y[8];
          widen8(raw[k][0], x);
          widen8(raw[k][1], y);
          if constexpr (BIAS) {
            const bf16* b = bias + (h + k) * D;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              x[j] += to_f(b[d0 + j]);
              y[j] += to_f(b[d1 + j]);
            }
          }
          if (turns) turn_pairs(x, y, cs, a.interleaved);
          *reinterpret_cast<uint4*>(dst + (h + k) * D + d0) = narrow8(x);
          *reinterpret_cast<uint4*>(dst + (h + k) * D + d1) = narrow8(y);
        }
    }
    return;
  }

  // ---- records
  const int w0 = (int)blockIdx.x / f.rec_parts * kWindow, part = (int)blockIdx.x % f.rec_parts, n_tok = min(kWindow, a.T - w0);
  // lane i: token i of the window, and of the next one (a record may reach into it)
  const int t_l = min(w0 + lane, a.T - 1);
  const int slot_l = a.slots[t_l], req_l = a.req[t_l];
  int slot_b = __shfl_up_sync(0xffffffffu, slot_l, 1), req_b = __shfl_up_sync(0xffffffffu, req_l, 1);
  if (lane == 0 && w0 > 0) {
    slot_b = a.slots[w0 - 1];
    req_b = a.req[w0 - 1];
  }
  const bool follows = w0 + lane > 0 && slot_b == slot_l - 1 && req_b == req_l && w0 + lane < a.T;
  const uint32_t on = __ballot_sync(0xffffffffu, follows && slot_l >= 0 && slot_l % kBlock != 0);  // goes on with the record of the token before
  const uint32_t leads = __ballot_sync(0xffffffffu, lane < n_tok && slot_l >= 0) & ~on;
  const int items = __popc(leads) * G, ld_t = half + 2;
  const int pos_rows = min(kTurnRows, a.T - w0);
  if (part * kAppendWarps >= items) return;
  if (!on) {
    // no two tokens of the window share a record: a token at a time, in few instructions (a call of a few tokens spends its time on fetching them)
    for (int it = part * kAppendWarps + warp; it < items; it += f.rec_parts * kAppendWarps) {
      const int tok = nth_bit(leads, it / G);
      append_one<N>(qkv + (size_t)(w0 + tok) * a.ld, BIAS ? bias : nullptr, a, w0 + tok, it % G, lane);
    }
    return;
  }
  bool table = false;
  for (int at = part * kAppendWarps; at < items; at += f.rec_parts * kAppendWarps) {
    const int it = at + warp;
    const bool busy = it < items;
    const int g = it % G, tok = busy ? nth_bit(leads, it / G) : 0;
    const int slot = __shfl_sync(0xffffffffu, slot_l, tok), req = __shfl_sync(0xffffffffu, req_l, tok), first = slot & (kBlock - 1);
    const int count = busy ? __ffs(~(on >> (tok + 1))) : 0;  // the leader and those that go on behind it
    const uint32_t fresh = ((1u << count) - 1u) << first;
    const bf16* src = qkv + (long)(w0 + tok - first) * a.ld + H * D;  // row of the record's slot 0
    // everything that is read from the rows
    uint4 kr[N][4];
    uint32_t vr[N][16];
    const int pos = lane & 15;
    const bool mine = fresh >> pos & 1;
    int c0[N], c1[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int p = (lane >> 4) + 2 * n;
      c0[n] = p < half / 16 ? (a.interleaved ? 2 * p : p) : 2 * p;
      c1[n] = p < half / 16 && !a.interleaved ? p + half / 16 : c0[n] + 1;
      if (mine && p < D / 32) {
        const bf16* row = src + (size_t)pos * a.ld + g * D;
        kr[n][0] = *reinterpret_cast<const uint4*>(row + c0[n] * 16);
        kr[n][1] = *reinterpret_cast<const uint4*>(row + c0[n] * 16 + 8);
        kr[n][2] = *reinterpret_cast<const uint4*>(row + c1[n] * 16);
        kr[n][3] = *reinterpret_cast<const uint4*>(row + c1[n] * 16 + 8);
      } else {
        kr[n][0] = kr[n][1] = kr[n][2] = kr[n][3] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 2 * lane + 64 * n;
        vr[n][r] = fresh >> r & 1 && d < V ? *reinterpret_cast<const uint32_t*>(src + (size_t)r * a.ld + G * D + g * V + d) : 0u;
      }
    uint8_t* rec = nullptr;
    uint32_t tail = 0;
    uint4 v_old[N][2];
    if (busy) rec = a.pool.record(req, slot, g);
    if (busy && first) {
      tail = *reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V));
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (2 * lane + 64 * n < V) {
          v_old[n][0] = *reinterpret_cast<const uint4*>(rec + kBlock * (D + 2 * lane + 64 * n));
          v_old[n][1] = *reinterpret_cast<const uint4*>(rec + kBlock * (D + 2 * lane + 64 * n + 1));
        }
    }
    if (!table) {  // under the loads
      const int rows = on >> kWindow & 1 ? pos_rows : n_tok;
      for (int k = lane; k < half; k += 32) {
        const double freq = (double)a.freq[k] * kTurns;
        for (int r = warp; r < rows; r += kAppendWarps) ap_turns[r * ld_t + k] = turn_of<false>(a.positions[w0 + r], freq, a.mag);
      }
      table = true;
      __syncthreads();
    }
    if (!busy) continue;

    // values
    float b0[N] = {}, b1[N] = {};
    uint32_t bad = 0;
    float amax = 0.f;
    auto value = [&](int n, int r, int k) { return k ? bf16_hi(vr[n][r]) + (BIAS ? b1[n] : 0.f) : bf16_lo(vr[n][r]) + (BIAS ? b0[n] : 0.f); };
    uint32_t bad_v, good_v;
    if constexpr (BIAS) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = 2 * lane + 64 * n;
        b0[n] = d < V ? to_f(bias[(H + G) * D + g * V + d]) : 0.f;
        b1[n] = d < V ? to_f(bias[(H + G) * D + g * V + d + 1]) : 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) bad |= (odd_one(value(n, r, 0)) || odd_one(value(n, r, 1)) ? 1u : 0u) << r;
      }
      bad_v = __reduce_or_sync(0xffffffffu, bad) & fresh, good_v = fresh & ~bad_v;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (good_v >> r & 1) amax = fmaxf(amax, fmaxf(fabsf(value(n, r, 0)), fabsf(value(n, r, 1))));
    } else {
      uint32_t most = 0, all = 0, row[16];  // (all of them at most: mostly there is nothing that is not finite)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        row[r] = 0;
#pragma unroll
        for (int n = 0; n < N; ++n) row[r] = larger2(row[r], vr[n][r]);
        all = __vmaxu2(all, row[r]);
      }
      if (__any_sync(0xffffffffu, larger_of(all) >= 0x7f80u)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) bad |= (larger_of(row[r]) >= 0x7f80u ? 1u : 0u) << r;
        bad = __reduce_or_sync(0xffffffffu, bad);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (bad >> r & 1) {
#pragma unroll
            for (int n = 0; n < N; ++n) vr[n][r] = 0;
          } else {
            most = __vmaxu2(most, row[r]);
          }
        }
      } else {
        most = all;
      }
      bad_v = bad & fresh, good_v = 0xffffu;  // (rows without a token, and bad ones, are zeros now)
      amax = __uint_as_float(larger_of(most) << 16);
    }
    const int had_v = tail_ev(tail), had_k = tail_ek(tail);
    int ev = exponent_for(warp_max(amax));
    if (first) ev = max(ev, had_v);
    {
      const float down = pow2(-ev), move = pow2(max(had_v - ev, -126));
      const bool grown = first && ev != had_v;
      uint8_t* dst = rec + kBlock * D;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int d = 2 * lane + 64 * n;
        if (d >= V) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = !BIAS || good_v >> (4 * x + j) & 1 ? value(n, 4 * x + j, k) * down : 0.f;
            w[x] = codes4(y[0], y[1], y[2], y[3]);
          }
          if (first) {
            const uint4 old = grown ? again16(v_old[n][k], move) : v_old[n][k];
            const uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // (the new codes are zero where old tokens lie)
              const int keep = min(max(first - 4 * x, 0), 4);
              w[x] |= keep == 4 ? o[x] : o[x] & ((1u << (8 * keep)) - 1u);
            }
          }
          *reinterpret_cast<uint4*>(dst + (d + k) * kBlock) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }

    // keys
    bad = 0;
    amax = 0.f;
    float x[N][16], y[N][16];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int p = (lane >> 4) + 2 * n;
      widen8(kr[n][0], x[n]);
      widen8(kr[n][1], x[n] + 8);
      widen8(kr[n][2], y[n]);
      widen8(kr[n][3], y[n] + 8);
      if (!mine || p >= D / 32) continue;
      bool odd = false;
      if constexpr (BIAS) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          x[n][j] += to_f(bias[(H + g) * D + c0[n] * 16 + j]);
          y[n][j] += to_f(bias[(H + g) * D + c1[n] * 16 + j]);
          odd |= odd_one(x[n][j]) || odd_one(y[n][j]);
        }
      } else {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) most = larger2(larger2(larger2(larger2(most, kr[n][j].x), kr[n][j].y), kr[n][j].z), kr[n][j].w);
        odd = larger_of(most) >= 0x7f80u;
      }
      if (odd) bad = 1u << pos;
      if (p < half / 16) {
        const float2* row = ap_turns + (tok + pos - first) * ld_t + p * 16;
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
          float2 cs[8];
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const float4 two = *reinterpret_cast<const float4*>(row + j + k);
            cs[k] = make_float2(two.x, two.y);
            cs[k + 1] = make_float2(two.z, two.w);
          }
          // 16 entries in a row are eight pairs where they lie side by side
          if (a.interleaved) turn_pairs(j ? y[n] : x[n], j ? y[n] + 8 : x[n] + 8, cs, 1);
          else turn_pairs(x[n] + j, y[n] + j, cs, 0);
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fmaxf(fabsf(x[n][j]), fabsf(y[n][j])));
    }
    const uint32_t bad_k = __reduce_or_sync(0xffffffffu, bad) | bad_v;
    int ek = exponent_for(warp_max(bad_k >> pos & 1 ? 0.f : amax));
    if (first) ek = max(ek, had_k);
    {
      const float down = pow2(-ek), move = pow2(max(had_k - ek, -126));
      const bool grown = first && ek != had_k;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if ((lane >> 4) + 2 * n >= D / 32) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint4* at16 = reinterpret_cast<uint4*>(rec + (pos >= 8 ? 8 * D : 0) + (k ? c1[n] : c0[n]) * 128 + (pos & 7) * 16);
          const float* z = k ? y[n] : x[n];
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = bad_k >> pos & 1 ? 0x7f7f7f7fu : codes4(z[4 * j] * down, z[4 * j + 1] * down, z[4 * j + 2] * down, z[4 * j + 3] * down);
          if (pos >= first) *at16 = make_uint4(w[0], w[1], w[2], w[3]);  // (zeros behind the last token)
          else if (grown) *at16 = again16(*at16, move);
        }
      }
    }
    if (lane == 0) emit_tail(rec + kBlock * (D + V), ek, ev);
  }
}

template <int N>
static int append_wide(const bf16* qkv, const bf16* bias, bf16* q_out, const AppendArgs& a, cudaStream_t st) {
  const int windows = (a.T + kWindow - 1) / kWindow;
  // a warp for every record, or as many CTAs as the GPU holds at once; whole records (consecutive slots) come to one a head
  const int most = (std::min(a.T, kWindow) * a.pool.G + kAppendWarps - 1) / kAppendWarps, whole = (a.pool.G + kAppendWarps - 1) / kAppendWarps;
  WideArgs f{a, 0, std::min(most, std::max(whole, 4 * sm_count() / windows)), 8};
  f.rec_ctas = windows * f.rec_parts;
  const long threads = kAppendWarps * 32, units = (long)a.T * (a.pool.dim / 16);
  while (f.by > 1 && units * ((a.H + f.by - 1) / f.by) < threads * 4 * sm_count()) f.by /= 2;
  const long ctas = a.H ? (units * ((a.H + f.by - 1) / f.by) + threads - 1) / threads : 0;
  const size_t smem = (size_t)kTurnRows * (a.dims / 2 + 2) * sizeof(float2);
  return (int)launch(bias ? kv8_append_wide_kernel<N, true> : kv8_append_wide_kernel<N, false>, dim3((unsigned)(f.rec_ctas + ctas)), dim3((unsigned)threads), smem, st, true, qkv, bias, q_out, f);
}

}  // namespace kv8
}  // namespace pk

using namespace pk;

extern "C" long pk_kv8_page_bytes(int page_size, int kv_heads, int dim, int vdim) {
  if (!kv8::sizes_ok(page_size, kv_heads, dim, vdim)) return -1;
  return (long)kv_heads * (page_size / kv8::kBlock) * kv8::record_bytes(dim, vdim);
}

extern "C" int pk_kv8_append(const void* qkv, int ld, const void* bias, const int* positions, const int* slots, const int* req, const int* page_off,
                             const int* pages, void* q_out, void* cache, long page_stride, int page_size, int heads, int kv_heads, int dim, int vdim,
                             int dims, int interleaved, const float* freq, float mag, int tokens, int f32, pk_stream st) {
  if (!qkv || !positions || !req || !page_off || !pages || !cache || tokens <= 0 || heads < 0 || heads > 65535 || kv_heads > 65535 || (heads > 0 && !q_out) || !kv8::sizes_ok(page_size, kv_heads, dim, vdim) ||
      !kv8::pool_ok(cache, page_stride, page_size, kv_heads, dim, vdim) || dims < 0 || dims > dim || (dims & 1) || (dims > 0 && !freq) ||
      ld < (long)heads * dim + (long)kv_heads * (dim + vdim))
    return -1;
  const int es = f32 ? 4 : 2;
  const bool vec = ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) == 0 && (long)ld * es % 16 == 0;
  const kv8::AppendArgs a{positions, slots ? slots : positions, req, kv8::make_pool(cache, page_stride, page_off, pages, page_size, kv_heads, dim, vdim),
                          freq,      mag,                       ld,  heads, tokens, dims, interleaved, vec};
  if (!f32 && vec && dims % 32 == 0 && (long)tokens * heads * dim < 1L << 31) {  // (its threads are counted in 32 bits)
    const int wide = std::max(dim, vdim);
    const bf16 *x = (const bf16*)qkv, *b = (const bf16*)bias;
    if (wide <= 64) return kv8::append_wide<1>(x, b, (bf16*)q_out, a, st);
    if (wide <= 128) return kv8::append_wide<2>(x, b, (bf16*)q_out, a, st);
    return kv8::append_wide<4>(x, b, (bf16*)q_out, a, st);
  }
  const int windows = (tokens + kv8::kWindow - 1) / kv8::kWindow;
  const int items = (std::min(tokens, kv8::kWindow) * kv_heads + kv8::kAppendWarps - 1) / kv8::kAppendWarps;
  const int parts = std::max(1, std::min(items, (4 * sm_count() + windows - 1) / windows));
  const size_t smem = ((size_t)kv8::kWindow * dims + (size_t)kv8::kAppendWarps * kv8::kBlock * kv8::row_ld(std::max(dim, vdim))) * sizeof(float);
  const dim3 grid(windows, parts), block(kv8::kAppendWarps * 32);
  if (f32) {
    static std::atomic<uint64_t> set{0};
    if (const cudaError_t e = allow_smem(set, (const void*)kv8::kv8_append_kernel<float>, 96 * 1024); e != cudaSuccess) return (int)e;
    return (int)launch(kv8::kv8_append_kernel<float>, grid, block, smem, st, true, (const float*)qkv, (const float*)bias, (float*)q_out, a);
  }
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8::kv8_append_kernel<bf16>, 96 * 1024); e != cudaSuccess) return (int)e;
  return (int)launch(kv8::kv8_append_kernel<bf16>, grid, block, smem, st, true, (const bf16*)qkv, (const bf16*)bias, (bf16*)q_out, a);
}
