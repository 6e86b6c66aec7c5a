// Eviction from the 8-bit paged cache (kv8.cuh) by accumulated attention weight.
//
// Of a request's `len` tokens each kv head keeps min(len, budget): the first `keep_first`, the last `keep_recent`, and of the others those with the largest mass
// (the lower index where two are equal; NaN counts as less than any number, infinity as the largest number).  The kept ones keep their order and go to other pages
// of the pool, into records with exponents of their own; their masses move with them, and the rest of the new row is zero.
//   kv8_pick_kernel   a CTA to (request, kv head): the smallest kept key by four rounds of 8 bits, then the places by prefix sums.
//   kv8_move_kernel   a warp to a new record.
#include <algorithm>

#include "kv8.cuh"

namespace pk {
namespace kv8 {

constexpr int kPickThreads = 1024;
constexpr int kMoveWarps = 4;

struct EvictArgs {
  Pool from, to;
  const int* lens;
  int* new_lens;
  const float* mass;
  float* new_mass;
  int* kept;
  long mass_ld, new_ld;
  int budget, first, recent, max_len;
};

// larger masses -> larger keys; NaN 0, the tokens that stay in any case 2^32 - 1
__device__ __forceinline__ uint32_t mass_key(float m, bool stays) {
  if (stays) return 0xffffffffu;
  if (m != m) return 0u;
  const uint32_t u = __float_as_uint(m + 0.f);  // -0 -> 0
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return min(max(k, 1u), 0xff7fffffu);
}

__global__ void __launch_bounds__(kPickThreads) kv8_pick_kernel(EvictArgs a) {
  __shared__ uint32_t hist[256], s_warp[kPickThreads / 32], s_digit, s_left;
  pdl_wait();
  pdl_launch_dependents();
  const int g = blockIdx.x, r = blockIdx.y, G = a.from.G, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = max(0, min(a.lens[r], a.max_len)), keep = min(n, a.budget);
  const float* mass = a.mass + ((size_t)r * G + g) * a.mass_ld;
  float* new_mass = a.new_mass + ((size_t)r * G + g) * a.new_ld;
  int* kept = a.kept + ((size_t)r * G + g) * a.budget;
  auto key = [&](int j) { return mass_key(mass[j], j < a.first || j >= n - a.recent); };
  // the key of the last one kept, and how many of those equal to it are
  uint32_t prefix = 0, left = keep;
  if (keep < n) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kPickThreads) hist[i] = 0;
      __syncthreads();
      for (int j = tid; j < n; j += kPickThreads) {
        const uint32_t k = key(j);
        if (shift == 24 || (k ^ prefix) >> (shift + 8) == 0) atomicAdd(&hist[k >> shift & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t want = left;
        int d = 255;
        while (hist[d] < want) want -= hist[d--];  // (the counts add up to at least `left`)
        s_digit = d;
        s_left = want;
      }
      __syncthreads();
      prefix |= s_digit << shift;
      left = s_left;
    }
  }
  // places: prefix sums over the tokens in order, of those above the last kept key and, as far as `left` goes, of those equal to it
  uint32_t at = 0, equal = 0;
  for (int j0 = 0; j0 < n; j0 += kPickThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? key(j) : 0u;
    const bool is_eq = j < n && keep < n && k == prefix, is_up = j < n && (keep == n || k > prefix);
    // equal ones before this one
    const uint32_t eq = __ballot_sync(0xffffffffu, is_eq), below = (1u << lane) - 1u;
    if (lane == 0) s_warp[warp] = __popc(eq);
    __syncthreads();
    uint32_t eq_before = equal, eq_all = 0;
    for (int w = 0; w < kPickThreads / 32; ++w) {
      if (w < warp) eq_before += s_warp[w];
      eq_all += s_warp[w];
    }
    const bool in = is_up || (is_eq && eq_before + __popc(eq & below) < left);
    equal += eq_all;
    __syncthreads();
    const uint32_t ins = __ballot_sync(0xffffffffu, in);
    if (lane == 0) s_warp[warp] = __popc(ins);
    __syncthreads();
    uint32_t before = at, all = 0;
    for (int w = 0; w < kPickThreads / 32; ++w) {
      if (w < warp) before += s_warp[w];
      all += s_warp[w];
    }
    at += all;
    if (in) {
      const uint32_t i = before + __popc(ins & below);
      kept[i] = j;
      new_mass[i] = mass[j];
    }
    __syncthreads();
  }
  for (int i = keep + tid; i < a.budget; i += kPickThreads) kept[i] = -1;
  for (long i = keep + tid; i < a.new_ld; i += kPickThreads) new_mass[i] = 0.f;
  if (g == 0 && tid == 0) a.new_lens[r] = keep;
}

__global__ void __launch_bounds__(kMoveWarps * 32) kv8_move_kernel(EvictArgs a) {
  extern __shared__ __align__(16) float mv_sm[];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x * kMoveWarps + warp, g = blockIdx.y, r = blockIdx.z;
  const int D = a.from.dim, V = a.from.vdim, n = min(a.lens[r], min(a.max_len, a.budget)), cnt = min(kBlock, n - b * kBlock);
  if (cnt <= 0) return;
  float* rows = mv_sm + warp * kBlock * row_ld(max(D, V));
  const int* kept = a.kept + ((size_t)r * a.from.G + g) * a.budget + b * kBlock;
  const int mine = lane < cnt ? kept[lane] : 0;  // lane i: the i-th token
  const uint8_t* rec = a.from.record(r, mine, g);
  const uint32_t tail = *reinterpret_cast<const uint32_t*>(rec + kBlock * (D + V));
  const uint64_t rec_at = reinterpret_cast<uint64_t>(rec);
  uint8_t* dst = a.to.record(r, b * kBlock, g);
  uint32_t bad = 0;
  const uint32_t have = (1u << cnt) - 1u;
  for (int i0 = 0; i0 < D; i0 += 32) {  // unit: 16 entries of a token (dim units a record)
    const int u = i0 + lane, tok = u / (D / 16), c = u % (D / 16);
    const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, rec_at, tok));
    const int j = __shfl_sync(0xffffffffu, mine, tok) % kBlock;
    const float f = pow2(tail_ek(__shfl_sync(0xffffffffu, tail, tok)));
    float v[16];
    uint4 code = make_uint4(0, 0, 0, 0);
    if (tok < cnt) code = *reinterpret_cast<const uint4*>(src + (j >> 3) * (8 * D) + c * 128 + (j & 7) * 16);
    if ((code.x & 0x7fu) == 0x7fu) bad |= 1u << tok;
    values16(code, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) rows[tok * row_ld(D) + c * 16 + i] = v[i] * f;
  }
  bad = __reduce_or_sync(0xffffffffu, bad);
  __syncwarp();
  const int ek = exponent_for(rows_amax(rows, D, have & ~bad, lane));
  emit_k(dst, rows, D, ek, bad, lane);
  __syncwarp();
  for (int tok = 0; tok < kBlock; ++tok) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, rec_at, tok)) + kBlock * D + __shfl_sync(0xffffffffu, mine, tok) % kBlock;
    const float f = pow2(tail_ev(__shfl_sync(0xffffffffu, tail, tok)));
    for (int d = lane; d < V; d += 32) rows[tok * row_ld(V) + d] = tok < cnt ? values2(src[d * 16]).x * f : 0.f;
  }
  __syncwarp();
  const int ev = exponent_for(rows_amax(rows, V, have, lane));
  emit_v(dst + kBlock * D, rows, V, ev, 0u, lane);
  if (lane == 0) emit_tail(dst + kBlock * (D + V), ek, ev);
}

}  // namespace kv8
}  // namespace pk

using namespace pk;

extern "C" int pk_kv8_evict(void* cache, long page_stride, int page_size, const int* page_off, const int* pages, const int* lens, const float* mass, long mass_ld,
                            const int* new_page_off, const int* new_pages, int* new_lens, float* new_mass, long new_mass_ld, int* kept, int requests, int kv_heads,
                            int dim, int vdim, int budget, int keep_first, int keep_recent, int max_kv_len, pk_stream st) {
  if (!cache || !page_off || !pages || !lens || !mass || !new_page_off || !new_pages || !new_lens || !new_mass || !kept || requests <= 0 || requests > 65535 ||
      budget <= 0 || keep_first < 0 || keep_recent < 0 || (long)keep_first + keep_recent > budget || max_kv_len <= 0 || mass_ld < max_kv_len ||
      new_mass_ld < budget || new_mass == mass || new_pages == pages || !kv8::sizes_ok(page_size, kv_heads, dim, vdim) || kv_heads > 65535 ||
      !kv8::pool_ok(cache, page_stride, page_size, kv_heads, dim, vdim))
    return -1;
  const kv8::EvictArgs a{kv8::make_pool(cache, page_stride, page_off, pages, page_size, kv_heads, dim, vdim),
                         kv8::make_pool(cache, page_stride, new_page_off, new_pages, page_size, kv_heads, dim, vdim),
                         lens, new_lens, mass, new_mass, kept, mass_ld, new_mass_ld, budget, keep_first, keep_recent, max_kv_len};
  if (const cudaError_t e = launch(kv8::kv8_pick_kernel, dim3(kv_heads, requests), dim3(kv8::kPickThreads), 0, st, true, a); e != cudaSuccess) return (int)e;
  const int records = (std::min(budget, max_kv_len) + kv8::kBlock - 1) / kv8::kBlock;
  const size_t smem = (size_t)kv8::kMoveWarps * kv8::kBlock * kv8::row_ld(std::max(dim, vdim)) * sizeof(float);
  static std::atomic<uint64_t> set{0};
  if (const cudaError_t e = allow_smem(set, (const void*)kv8::kv8_move_kernel, 96 * 1024); e != cudaSuccess) return (int)e;
  return (int)launch(kv8::kv8_move_kernel, dim3((records + kv8::kMoveWarps - 1) / kv8::kMoveWarps, kv_heads, requests), dim3(kv8::kMoveWarps * 32), smem, st, true, a);
}
