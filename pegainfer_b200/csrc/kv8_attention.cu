// Attention over the 8-bit paged cache (kv8.cuh).
//   s_j = scale * q . k_j, capped to cap * tanh(s_j / cap) where a cap is given, over the visible keys max(0, p - window + 1) <= j <= p of the query's slot p;
//   w_j = exp(s_j) / (sum exp(s) + exp(sink)),  out = sum w_j v_j,  lse = log of that denominator,  mass[request][kv head][j] += w_j of all the call's queries.
// Scores are kept in units of log2.
#include <algorithm>
#include <climits>

#include "kv8_attention.cuh"

namespace pk {
namespace kv8 {

constexpr int kRowWarps = 8;

// Any sizes and types, all arithmetic in fp32: a CTA to (row, query head, share of the keys), records by turns to its warps.  Two lanes have a token's key (half
// of the entries each); for P V a lane has every 32nd entry and reads its 16 tokens with one load.
template <typename E>
__global__ void __launch_bounds__(kRowWarps * 32) kv8_row_kernel(const E* __restrict__ q, const E* __restrict__ sink, E* __restrict__ out, AttnArgs a) {
  extern __shared__ __align__(16) float row_sm[];
  __shared__ float s_m[kRowWarps], s_l[kRowWarps];
  const int D = a.pool.dim, V = a.pool.vdim, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* sq = row_sm;       // the query, times scale
  float* acc_sm = row_sm + D;  // [warps][vdim]
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, h = blockIdx.y, g = h / (a.H / a.pool.G), p = a.slots[t];
  const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
  bool odd = false;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    const float v = to_f(q[((size_t)t * a.H + h) * D + d]);
    odd |= (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
    sq[d] = v;
  }
  const float c = __syncthreads_or(odd) ? NAN : a.scale * kLog2e;  // (an entry that is not finite: the row is NaN, as in the other kernels)
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (p >= 0) {
    const int req = a.req[t], b0 = lo / kBlock, n = p / kBlock - b0 + 1;
    const int share = (n + gridDim.z - 1) / gridDim.z, from = b0 + blockIdx.z * share, to = min(from + share, b0 + n);
    const int tok = lane & 15, part = lane >> 4, chunks = D / 32;
    for (int b = from + warp; b < to; b += kRowWarps) {
      const uint8_t* rec = a.pool.record(req, b * kBlock, g);
      const uint32_t tail = *reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V));
      const uint8_t* k = rec + (tok >> 3) * (8 * D) + part * chunks * 128 + (tok & 7) * 16;
      float s = 0.f, s1 = 0.f;
      for (int i = 0; i < chunks; ++i) {
        float v[16];
        values16(*reinterpret_cast<const uint4*>(k + i * 128), v);
        const float4* x = reinterpret_cast<const float4*>(sq + (part * chunks + i) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 y = x[j];
          s = fmaf(v[4 * j], y.x, fmaf(v[4 * j + 1], y.y, s));
          s1 = fmaf(v[4 * j + 2], y.z, fmaf(v[4 * j + 3], y.w, s1));
        }
      }
      s += s1;
      s += __shfl_xor_sync(0xffffffffu, s, 16);
      const int j = b * kBlock + tok;
      s = shaped(s * pow2(tail_ek(tail)), c, a.cap);
      if (j < lo || j > p) s = -INFINITY;
      const float mn = fmaxf(m, warp_max(s)), ref = mn == -INFINITY ? 0.f : mn, f = exp2f(m - ref), w = exp2f(s - ref);
      m = mn;
      l = l * f + warp_sum(part ? 0.f : w);
      const float wv = w * pow2(tail_ev(tail));
      float ws[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) ws[i] = __shfl_sync(0xffffffffu, wv, i);
      const uint8_t* vt = rec + kBlock * D;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < V) {
          float v[16], o = acc[i] * f, o1 = 0.f;
          values16(*reinterpret_cast<const uint4*>(vt + (lane + 32 * i) * 16), v);
#pragma unroll
          for (int x = 0; x < 16; x += 2) {
            o = fmaf(ws[x], v[x], o);
            o1 = fmaf(ws[x + 1], v[x + 1], o1);
          }
          acc[i] = o + o1;
        }
    }
  }
  if (l != l) m = INFINITY;  // a NaN among the scores: no other warp or share may hide it
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < V) acc_sm[warp * V + lane + 32 * i] = acc[i];
  __syncthreads();
  float M = -INFINITY, den = 0.f, f[kRowWarps];
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, s_m[w]);
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    f[w] = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - M);
    den += s_l[w] * f[w];
  }
  const size_t row = (size_t)t * a.H + h;
  const bool whole = gridDim.z == 1;
  const RowEnd end = row_end(M, den, sink ? to_f(sink[h]) : 0.f, sink != nullptr);
  for (int d = threadIdx.x; d < V; d += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) o += f[w] > 0.f ? acc_sm[w * V + d] * f[w] : 0.f;
    if (whole) out[(size_t)t * a.out_ld + h * V + d] = from_f<E>(o * end.factor);
    else a.part_o[((size_t)blockIdx.z * a.T * a.H + row) * V + d] = o;
  }
  if (threadIdx.x == 0) {
    if (whole) {
      if (a.lse) a.lse[row] = end.lse;
    } else {
      a.part_ml[(size_t)blockIdx.z * a.T * a.H + row] = make_float2(M, den);
    }
  }
}

// The shares' states of a row -> its result: a warp to (row, head).
template <typename E>
__global__ void __launch_bounds__(128) kv8_merge_kernel(const E* __restrict__ sink, E* __restrict__ out, int shares, AttnArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const size_t rows = (size_t)a.T * a.H, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, V = a.pool.vdim;
  if (row >= rows) return;
  const int t = (int)(row / a.H), h = (int)(row % a.H);
  float M = -INFINITY;
  for (int s = lane; s < shares; s += 32) M = fmaxf(M, a.part_ml[s * rows + row].x);
  M = warp_max(M);
  float den = 0.f;
  for (int s = lane; s < shares; s += 32) {
    const float2 v = a.part_ml[s * rows + row];
    den += v.x == -INFINITY ? 0.f : v.y * exp2f(v.x - M);
  }
  den = warp_sum(den);
  const RowEnd end = row_end(M, den, sink ? to_f(sink[h]) : 0.f, sink != nullptr);
  float o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  for (int s0 = 0; s0 < shares; s0 += 32) {
    const float m = s0 + lane < shares ? a.part_ml[(s0 + lane) * rows + row].x : -INFINITY, w = m == -INFINITY ? 0.f : exp2f(m - M);
#pragma unroll 4
    for (int s = s0; s < min(shares, s0 + 32); ++s) {
      const float f = __shfl_sync(0xffffffffu, w, s - s0);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < V) {
          if (f != 0.f) o[i] = fmaf(a.part_o[(s * rows + row) * V + lane + 32 * i], f, o[i]);  // (for the warp alike; a share without keys stores none)
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < V) out[(size_t)t * a.out_ld + h * V + lane + 32 * i] = from_f<E>(o[i] * end.factor);
  if (lane == 0 && a.lse) a.lse[row] = end.lse;
}

// what a call runs: the shares of its keys and its workspace
struct Plan {
  bool few, prompt, tile;  // kv8_few.cu, kv8_prompt.cu, kv8_tile.cu
  FewNeed need;
  int shares;
  size_t o_bytes, ml_bytes, lse_bytes;
  long bytes() const { return (long)((few ? need.bytes() : o_bytes + ml_bytes) + lse_bytes); }
};
// slots are below max_kv_len: a window of that or more hides nothing
static int window_of(const pk_kv8_options& o) { return o.window < o.max_kv_len ? o.window : 0; }
static size_t up16(size_t n) { return (n + 15) / 16 * 16; }
static Plan plan(int T, int H, int G, int dim, int vdim, const pk_kv8_options& o, int f32) {
  Plan p{};
  if (o.mass && !o.lse) p.lse_bytes = up16((size_t)T * H * sizeof(float));
  if (!f32 && few_takes(T, H, G, dim, vdim, o.max_kv_len, o.max_q_len)) {
    p.few = true;
    p.need = few_need(T, H, G, dim, o.max_kv_len, o.mass != nullptr);
    return p;
  }
  if (!f32 && prompt_takes(T, H, G, dim, vdim)) {
    p.prompt = true;
    p.shares = prompt_shares(T, H, G, o.max_kv_len, window_of(o));
  } else if (tile_takes(T, H, G, o.max_q_len)) {
    p.tile = true;
    p.shares = tile_shares(T, H, G, o.max_kv_len, window_of(o));
  } else {
    int span = o.max_kv_len;
    if (window_of(o) > 0) span = std::min(span, window_of(o) + kBlock);
    const int records = (span + kBlock - 1) / kBlock;
    // a share has at least two rounds of its warps
    p.shares = (int)std::max(1L, std::min((long)(records + 2 * kRowWarps - 1) / (2 * kRowWarps), (4L * sm_count() + (long)T * H - 1) / ((long)T * H)));
  }
  if (p.shares > 1) {
    p.o_bytes = up16((size_t)p.shares * T * H * vdim * sizeof(float));
    p.ml_bytes = up16((size_t)p.shares * T * H * sizeof(float2));
  }
  return p;
}

template <typename E>
static int merge(const E* sink, E* out, int shares, const AttnArgs& a, cudaStream_t st) {
  return (int)follow(kv8_merge_kernel<E>, dim3((unsigned)(((size_t)a.T * a.H + 3) / 4)), dim3(128), st, sink, out, shares, a);
}
template <typename E>
static int attention(const E* q, const E* sink, E* out, const AttnArgs& a, const Plan& p, int max_q_len, cudaStream_t st) {
  if (p.tile) {
    if (const int rc = tile_attention(q, sink, out, a, p.shares, st); rc != 0) return rc;
    if (p.shares > 1)
      if (const int rc = merge(sink, out, p.shares, a, st); rc != 0) return rc;
    return a.mass ? mass_rows(q, a, max_q_len, st) : 0;
  }
  const size_t smem = (size_t)(a.pool.dim + kRowWarps * a.pool.vdim) * sizeof(float);
  if (const cudaError_t e = launch(kv8_row_kernel<E>, dim3(a.T, a.H, p.shares), dim3(kRowWarps * 32), smem, st, true, q, sink, out, a); e != cudaSuccess) return (int)e;
  if (p.shares > 1)
    if (const int rc = merge(sink, out, p.shares, a, st); rc != 0) return rc;
  return a.mass ? mass_rows(q, a, max_q_len, st) : 0;
}

static bool options_ok(const pk_kv8_options* o, int tokens, int heads, int kv_heads, int vdim) {
  return o && tokens > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65535 && o->window >= 0 && o->softcap >= 0.f && o->max_kv_len > 0 && o->max_kv_len <= kMaxSlots &&
         o->max_q_len >= 0 && (o->out_ld == 0 || o->out_ld >= (long)heads * vdim) && (!o->mass || o->mass_ld > 0);
}

}  // namespace kv8
}  // namespace pk

using namespace pk;

extern "C" long pk_kv8_attention_workspace_bytes(int tokens, int heads, int kv_heads, int dim, int vdim, const pk_kv8_options* options, int f32) {
  if (!kv8::options_ok(options, tokens, heads, kv_heads, vdim) || !kv8::sizes_ok(kv8::kBlock, kv_heads, dim, vdim)) return -1;
  return kv8::plan(tokens, heads, kv_heads, dim, vdim, *options, f32).bytes();
}

extern "C" int pk_kv8_attention(const void* q, const void* cache, const void* sink, const int* slots, const int* req, const int* page_off, const int* pages,
                                void* out, long page_stride, int page_size, int tokens, int heads, int kv_heads, int dim, int vdim, float scale,
                                const pk_kv8_options* options, void* workspace, long workspace_bytes, int f32, pk_stream st) {
  if (!q || !cache || !slots || !req || !page_off || !pages || !out || !kv8::options_ok(options, tokens, heads, kv_heads, vdim) ||
      !kv8::sizes_ok(page_size, kv_heads, dim, vdim) || !kv8::pool_ok(cache, page_stride, page_size, kv_heads, dim, vdim))
    return -1;
  const kv8::Plan p = kv8::plan(tokens, heads, kv_heads, dim, vdim, *options, f32);
  if (p.bytes() > 0 && (!workspace || workspace_bytes < p.bytes() || (reinterpret_cast<uintptr_t>(workspace) & 15))) return -1;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  kv8::AttnArgs a{};
  a.pool = kv8::make_pool(cache, page_stride, page_off, pages, page_size, kv_heads, dim, vdim);
  a.slots = slots;
  a.req = req;
  a.T = tokens;
  a.H = heads;
  a.scale = scale;
  a.cap = options->softcap;
  a.window = kv8::window_of(*options);
  a.max_kv_len = options->max_kv_len;
  a.out_ld = options->out_ld ? options->out_ld : (long)heads * vdim;
  a.lse = options->lse ? options->lse : options->mass ? reinterpret_cast<float*>(ws) : nullptr;
  ws += p.lse_bytes;
  a.mass = options->mass;
  a.mass_ld = options->mass_ld;
  if (p.few) return kv8::few_attention((const bf16*)q, (const bf16*)sink, (bf16*)out, a, options->max_q_len, p.need, ws, st);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + p.o_bytes);
  if (p.prompt) {
    int rc = kv8::prompt_attention((const bf16*)q, (const bf16*)sink, (bf16*)out, a, p.shares, st);
    if (rc == 0 && p.shares > 1) rc = kv8::merge((const bf16*)sink, (bf16*)out, p.shares, a, st);
    if (rc != 0 || !a.mass) return rc;
    return kv8::mass_rows((const bf16*)q, a, options->max_q_len, st);
  }
  if (f32) return kv8::attention((const float*)q, (const float*)sink, (float*)out, a, p, options->max_q_len, st);
  return kv8::attention((const bf16*)q, (const bf16*)sink, (bf16*)out, a, p, options->max_q_len, st);
}
