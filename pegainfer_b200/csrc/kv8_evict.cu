// Eviction from the 8-bit paged cache (kv8.cuh) by accumulated attention weight.
//
// Of a request's `len` tokens each kv head keeps min(len, budget): the first `keep_first`, the last `keep_recent`, and of the others those with the largest mass
// (the lower index where two are equal; NaN counts as less than any number, infinity as the largest number).  The kept ones keep their order and go to other pages
// of the pool, into records with exponents of their own; their masses move with them, and the rest of the new row is zero.
//   kv8_pick_kernel   a CTA to (request, kv head): the smallest kept key, then the places by prefix sums.  Up to 32768 tokens the keys stay in registers and the smallest
//                     kept one is found bit by bit (a count over the CTA each, until one fits); longer ones go through histograms of 8 bits.
//   kv8_move_kernel   a warp to a new record.  Bound by the bytes it has to look at: a token's V lies in every 16-byte row of its record, so nearly the whole old cache is
//                     read where a quarter of it is kept.  A source record's V is loaded once for all its kept tokens (rows of 16 tokens a lane), codes whose exponent
//                     stays are moved as they are.
// B200, 16 requests of 16384, 8 kv heads of 128 in both, to 4096: choice 24 us, move 109; the call 135, and 144 after other data went through L2, where histograms take 175 (of 32768
// slots 273 and 312).  The sources' V rows and the kept K rows are 0.5 GB: 4.8 TB/s in the move.
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

// exclusive sum over the CTA's threads, and the whole sum; `room` has 33 words
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t* room, uint32_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t sum = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  __syncthreads();  // (the words of a sum before)
  if (lane == 31) room[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    uint32_t w = room[lane];
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    room[lane] = w;
  }
  __syncthreads();
  all = room[31];
  return sum - v + (warp > 0 ? room[warp - 1] : 0u);
}
__device__ __forceinline__ uint32_t block_count(uint32_t v, uint32_t* room) {
  const uint32_t w = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = w;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, room[threadIdx.x & 31]);
}

struct PickRow {
  int n, keep;
  const float* mass;
  float* new_mass;
  int* kept;
};
__device__ __forceinline__ PickRow pick_row(const EvictArgs& a) {
  const int g = blockIdx.x, r = blockIdx.y, n = max(0, min(a.lens[r], a.max_len));
  const size_t at = (size_t)r * a.from.G + g;
  return PickRow{n, min(n, a.budget), a.mass + at * a.mass_ld, a.new_mass + at * a.new_ld, a.kept + at * a.budget};
}
__device__ __forceinline__ void pick_rest(const EvictArgs& a, const PickRow& w) {
  for (int i = w.keep + threadIdx.x; i < a.budget; i += kPickThreads) w.kept[i] = -1;
  for (long i = w.keep + threadIdx.x; i < a.new_ld; i += kPickThreads) w.new_mass[i] = 0.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.new_lens[blockIdx.y] = w.keep;
}

// up to EACH tokens a thread: a warp has consecutive ones, 32 at a time
template <int EACH>
__global__ void __launch_bounds__(kPickThreads) kv8_pick_kernel(EvictArgs a) {
  __shared__ uint32_t room[32];
  pdl_wait();
  pdl_launch_dependents();
  const PickRow w = pick_row(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (w.n + kPickThreads - 1) / kPickThreads, j0 = warp * 32 * each + lane;  // this thread's i-th token is j0 + 32 i, i < each
  uint32_t key[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) key[i] = i < each && j0 + 32 * i < w.n ? __float_as_uint(__ldg(w.mass + j0 + 32 * i)) : 0u;  // (all under way at once)
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int j = j0 + 32 * i;
    key[i] = i < each && j < w.n ? mass_key(__uint_as_float(key[i]), j < a.first || j >= w.n - a.recent) : 0u;
  }
  // those above `least` are kept, and of those equal to it the first `left`
  uint32_t least = 0, left = w.keep;
  if (w.keep < w.n) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = least | 1u << bit;
      uint32_t here = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) here += key[i] >= c;  // (c > 0: no token where there is none)
      const uint32_t all = block_count(here, room);
      if (all < (uint32_t)w.keep) continue;
      least = c;
      if (all == (uint32_t)w.keep) break;  // exactly these
    }
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) above += key[i] > least;
    left = w.keep - block_count(above, room);
  }
  // places: in the tokens' order, warp by warp (a warp's counts are its first thread's)
  const uint32_t below = (1u << lane) - 1u;
  uint32_t equal = 0, all;
#pragma unroll
  for (int i = 0; i < EACH; ++i) equal += __popc(__ballot_sync(0xffffffffu, i < each && j0 + 32 * i < w.n && key[i] == least));
  uint32_t before = __shfl_sync(0xffffffffu, block_before(lane == 0 ? equal : 0u, room, all), 0);
  uint32_t takes = 0, in = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const bool there = i < each && j0 + 32 * i < w.n, eq = there && key[i] == least;
    const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
    const bool take = there && (w.keep == w.n || key[i] > least || (eq && before + __popc(eqs & below) < left));
    before += __popc(eqs);
    takes |= (uint32_t)take << i;
    in += __popc(__ballot_sync(0xffffffffu, take));
  }
  uint32_t at = __shfl_sync(0xffffffffu, block_before(lane == 0 ? in : 0u, room, all), 0);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const bool take = takes >> i & 1;
    const uint32_t ins = __ballot_sync(0xffffffffu, take);
    if (take) {
      const uint32_t to = at + __popc(ins & below);
      w.kept[to] = j0 + 32 * i;
      w.new_mass[to] = w.mass[j0 + 32 * i];
    }
    at += __popc(ins);
  }
  pick_rest(a, w);
}

// any number of tokens: four rounds of 8 bits of the key, then the places in turns of the CTA's threads
__global__ void __launch_bounds__(kPickThreads) kv8_pick_long_kernel(EvictArgs a) {
  __shared__ uint32_t hist[256], room[32], s_digit, s_left;
  pdl_wait();
  pdl_launch_dependents();
  const PickRow w = pick_row(a);
  const int tid = threadIdx.x, n = w.n;
  auto key = [&](int j) { return mass_key(w.mass[j], j < a.first || j >= n - a.recent); };
  uint32_t least = 0, left = w.keep;
  if (w.keep < n) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kPickThreads) hist[i] = 0;
      __syncthreads();
      for (int j = tid; j < n; j += kPickThreads) {
        const uint32_t k = key(j);
        if (shift == 24 || (k ^ least) >> (shift + 8) == 0) atomicAdd(&hist[k >> shift & 255], 1u);
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
      least |= s_digit << shift;
      left = s_left;
    }
  }
  uint32_t at = 0, equal = 0;
  for (int j0 = 0; j0 < n; j0 += kPickThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? key(j) : 0u;
    const bool eq = j < n && w.keep < n && k == least, up = j < n && (w.keep == n || k > least);
    uint32_t eq_all, all;
    const uint32_t eq_before = equal + block_before(eq, room, eq_all);
    equal += eq_all;
    const bool in = up || (eq && eq_before < left);
    const uint32_t i = at + block_before(in, room, all);
    at += all;
    if (in) {
      w.kept[i] = j;
      w.new_mass[i] = w.mass[j];
    }
  }
  pick_rest(a, w);
}

// codes times f, a power of two, rounded again
__device__ __forceinline__ uint32_t moved4(uint32_t four, float f0, float f1, float f2, float f3) {
  float v[4];
  values4(four, v);
  return codes4(v[0] * f0, v[1] * f1, v[2] * f2, v[3] * f3);
}
// the value of a code without its sign
__device__ __forceinline__ float size_of(uint32_t code) { return values2(code & 0x7fu).x; }

template <int D, int V>
__global__ void __launch_bounds__(kMoveWarps * 32) kv8_move_kernel(EvictArgs a) {
  constexpr int REC = kBlock * (D + V) + 16, NK = D / 32, NV = V / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x * kMoveWarps + warp, g = blockIdx.y, r = blockIdx.z;
  const int n = min(a.lens[r], min(a.max_len, a.budget)), cnt = min(kBlock, n - b * kBlock);
  if (cnt <= 0) return;
  const int* kept = a.kept + ((size_t)r * a.from.G + g) * a.budget + b * kBlock;
  const int slot = kept[min(lane, cnt - 1)];  // lane i: the i-th token (the last one again behind it)
  const uint8_t* rec = a.from.record(r, slot, g);
  const uint32_t tail = *reinterpret_cast<const uint32_t*>(rec + REC - 16);
  const uint64_t rec_at = reinterpret_cast<uint64_t>(rec);
  uint8_t* dst = a.to.record(r, b * kBlock, g);
  // K: unit u = 16 entries of a token (as they lie in a record)
  uint4 k[NK];
  float kf[NK], amax = 0.f;  // 2^(the token's old exponent)
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int u = lane + 32 * i, tok = (u >= D / 2 ? 8 : 0) + (u & 7), c = u % (D / 2) >> 3;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, rec_at, tok));
    const int j = __shfl_sync(0xffffffffu, slot, tok) % kBlock;
    kf[i] = pow2(tail_ek(__shfl_sync(0xffffffffu, tail, tok)));
    k[i] = tok < cnt ? *reinterpret_cast<const uint4*>(src + (j >> 3) * (8 * D) + c * 128 + (j & 7) * 16) : make_uint4(0, 0, 0, 0);
  }
  // V: the source records in turn, the next one's rows under way while this one's codes are taken
  const uint64_t one_before = __shfl_up_sync(0xffffffffu, rec_at, 1);
  const uint32_t heads = __ballot_sync(0xffffffffu, lane < cnt && (lane == 0 || one_before != rec_at));
  auto load_v = [&](int tok, uint4 (&x)[NV]) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, rec_at, tok)) + kBlock * D + lane * 16;
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = *reinterpret_cast<const uint4*>(src + i * 512);
  };
  uint4 now[NV], soon[NV];
  load_v(0, soon);
  uint32_t v[NV][4];
  float vmax = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0u;
#pragma unroll
  for (int t = 0; t < kBlock; ++t) {
    if (t >= cnt) break;
    if (heads >> t & 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) now[i] = soon[i];
      const uint32_t later = heads & ~((2u << t) - 1u);
      if (later) load_v(__ffs(later) - 1, soon);
    }
    const int j = __shfl_sync(0xffffffffu, slot, t) % kBlock;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t word = j < 8 ? (j < 4 ? now[i].x : now[i].y) : (j < 12 ? now[i].z : now[i].w), code = __byte_perm(word, 0, 0x4440u | (j & 3));
      v[i][t >> 2] |= code << (8 * (t & 3));
      top = max(top, code & 0x7fu);
    }
    vmax = fmaxf(vmax, size_of(top) * pow2(tail_ev(__shfl_sync(0xffffffffu, tail, t))));
  }
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const uint32_t w[4] = {k[i].x, k[i].y, k[i].z, k[i].w};
    uint32_t top = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) top = __vmaxu4(top, w[x] & 0x7f7f7f7fu);
    top = max(max(top & 255u, top >> 8 & 255u), max(top >> 16 & 255u, top >> 24));
    if (top != 0x7fu) amax = fmaxf(amax, size_of(top) * kf[i]);  // (a token that is not finite has no other code)
  }
  const int ek = exponent_for(warp_max(amax)), ev = exponent_for(warp_max(vmax));
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const float f = fminf(kf[i] * pow2(-ek), 1048576.f);  // (2^20: more only where the token's codes are all zero, and a product with infinity would not be)
    if (f != 1.f && (k[i].x & 0x7fu) != 0x7fu) k[i] = make_uint4(moved4(k[i].x, f, f, f, f), moved4(k[i].y, f, f, f, f), moved4(k[i].z, f, f, f, f), moved4(k[i].w, f, f, f, f));
    *reinterpret_cast<uint4*>(dst + (lane + 32 * i) * 16) = k[i];
  }
  const float vf = fminf(pow2(tail_ev(tail)) * pow2(-ev), 1048576.f);  // lane i: of token i
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float f0 = __shfl_sync(0xffffffffu, vf, 4 * x), f1 = __shfl_sync(0xffffffffu, vf, 4 * x + 1), f2 = __shfl_sync(0xffffffffu, vf, 4 * x + 2),
                f3 = __shfl_sync(0xffffffffu, vf, 4 * x + 3);
    if (f0 != 1.f || f1 != 1.f || f2 != 1.f || f3 != 1.f)
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i][x] = moved4(v[i][x], f0, f1, f2, f3);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) *reinterpret_cast<uint4*>(dst + kBlock * D + (lane + 32 * i) * 16) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
  if (lane == 0) emit_tail(dst + REC - 16, ek, ev);
}

template <int D>
static cudaError_t launch_move(const EvictArgs& a, dim3 grid, cudaStream_t st) {
  const dim3 block(kMoveWarps * 32);
  switch (a.from.vdim) {
    case 32: return follow(kv8_move_kernel<D, 32>, grid, block, st, a);
    case 64: return follow(kv8_move_kernel<D, 64>, grid, block, st, a);
    case 96: return follow(kv8_move_kernel<D, 96>, grid, block, st, a);
    case 128: return follow(kv8_move_kernel<D, 128>, grid, block, st, a);
    case 160: return follow(kv8_move_kernel<D, 160>, grid, block, st, a);
    case 192: return follow(kv8_move_kernel<D, 192>, grid, block, st, a);
    case 224: return follow(kv8_move_kernel<D, 224>, grid, block, st, a);
    default: return follow(kv8_move_kernel<D, 256>, grid, block, st, a);
  }
}

}  // namespace kv8
}  // namespace pk

using namespace pk;

extern "C" int pk_kv8_evict(void* cache, long page_stride, int page_size, const int* page_off, const int* pages, const int* lens, const float* mass, long mass_ld,
                            const int* new_page_off, const int* new_pages, int* new_lens, float* new_mass, long new_mass_ld, int* kept, int requests, int kv_heads,
                            int dim, int vdim, int budget, int keep_first, int keep_recent, int max_kv_len, pk_stream st) {
  if (!cache || !page_off || !pages || !lens || !mass || !new_page_off || !new_pages || !new_lens || !new_mass || !kept || requests <= 0 || requests > 65535 ||
      budget <= 0 || budget > kv8::kMaxSlots || keep_first < 0 || keep_recent < 0 || (long)keep_first + keep_recent > budget || max_kv_len <= 0 || max_kv_len > kv8::kMaxSlots || mass_ld < max_kv_len ||
      new_mass_ld < budget || new_mass == mass || new_pages == pages || new_lens == lens || !kv8::sizes_ok(page_size, kv_heads, dim, vdim) || kv_heads > 65535 ||
      !kv8::pool_ok(cache, page_stride, page_size, kv_heads, dim, vdim))
    return -1;
  const kv8::EvictArgs a{kv8::make_pool(cache, page_stride, page_off, pages, page_size, kv_heads, dim, vdim),
                         kv8::make_pool(cache, page_stride, new_page_off, new_pages, page_size, kv_heads, dim, vdim),
                         lens, new_lens, mass, new_mass, kept, mass_ld, new_mass_ld, budget, keep_first, keep_recent, max_kv_len};
  const dim3 rows(kv_heads, requests), threads(kv8::kPickThreads);
  const cudaError_t e = max_kv_len <= 4 * kv8::kPickThreads    ? launch(kv8::kv8_pick_kernel<4>, rows, threads, 0, st, true, a)
                        : max_kv_len <= 16 * kv8::kPickThreads ? launch(kv8::kv8_pick_kernel<16>, rows, threads, 0, st, true, a)
                        : max_kv_len <= 32 * kv8::kPickThreads ? launch(kv8::kv8_pick_kernel<32>, rows, threads, 0, st, true, a)
                                                               : launch(kv8::kv8_pick_long_kernel, rows, threads, 0, st, true, a);
  if (e != cudaSuccess) return (int)e;
  const int records = (std::min(budget, max_kv_len) + kv8::kBlock - 1) / kv8::kBlock;
  const dim3 grid((records + kv8::kMoveWarps - 1) / kv8::kMoveWarps, kv_heads, requests);
  switch (dim) {
    case 32: return (int)kv8::launch_move<32>(a, grid, st);
    case 64: return (int)kv8::launch_move<64>(a, grid, st);
    case 96: return (int)kv8::launch_move<96>(a, grid, st);
    case 128: return (int)kv8::launch_move<128>(a, grid, st);
    case 160: return (int)kv8::launch_move<160>(a, grid, st);
    case 192: return (int)kv8::launch_move<192>(a, grid, st);
    case 224: return (int)kv8::launch_move<224>(a, grid, st);
    default: return (int)kv8::launch_move<256>(a, grid, st);
  }
}
