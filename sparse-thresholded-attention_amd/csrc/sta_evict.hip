// sta_evict.hip -- eviction from a paged cache by accumulated attention weight.
//
// Every kv head of a sequence keeps m = min(len, budget) keys.  A key's rank is one 32-bit word,
// larger first: all ones for a forced key (pos < n_global or pos > largest pos - n_local), else
// its weight's bits in an order-preserving form (NaN above +inf, -0 as +0), 0 for a key without a
// page.  The m-th largest word T comes from four counting passes over its bytes; a key stays if
// its word is above T, or equal to T and among the first of those by slot.
//
// The kept keys need no order in a cache that stores rotated keys, so in place only the kept keys
// in slots >= m move, each into the slot < m of a dropped one: a step that evicts one key moves at
// most one row a head instead of the whole cache.  Sources and destinations never meet.
#include "sta_cache.h"
#include "sta_device.h"

namespace sta {

namespace {

constexpr int SEL_T = 1024;
constexpr uint32_t FORCED = 0xffffffffu;

__device__ __forceinline__ uint32_t weight_word(float w) {
  if (w != w) return FORCED - 1;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// exclusive prefix and total of two flags over the workgroup; lds: 2 * 16 words
struct Ranks { int a, b, total_a, total_b; };
__device__ __forceinline__ Ranks rank_flags(bool fa, bool fb, int (*lds)[SEL_T / 64]) {
  const int wave = threadIdx.x >> 6;
  const unsigned long long ma = __ballot(fa), mb = __ballot(fb);
  const unsigned long long below = (1ull << (threadIdx.x & 63)) - 1;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[0][wave] = __popcll(ma);
    lds[1][wave] = __popcll(mb);
  }
  __syncthreads();
  Ranks r{(int)__popcll(ma & below), (int)__popcll(mb & below), 0, 0};
  for (int w = 0; w < SEL_T / 64; ++w) {
    if (w < wave) r.a += lds[0][w], r.b += lds[1][w];
    r.total_a += lds[0][w];
    r.total_b += lds[1][w];
  }
  return r;
}

__global__ __launch_bounds__(SEL_T) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[256], scan[2][SEL_T / 64], pick[2];
  __shared__ int wave_max[SEL_T / 64];
  const CacheView& c = a.c;
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = c.len(b), m = min(len, a.budget);
  const int seg = b * c.Hkv + hk;
  if (hk == 0 && tid == 0) a.new_lens[b] = m;
  const bool in_place = a.dst_table == nullptr;
  if (m == 0 || (in_place && len <= a.budget)) {
    if (tid == 0) a.counts[seg] = 0;
    return;
  }
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  int last = INT32_MIN;
  for (int j = tid; j < len; j += SEL_T) {
    const int p = c.page_of(table, j);
    if (p >= 0) last = max(last, c.pos[p * c.p_ps + hk * c.p_hs + c.slot_of(j)]);
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) last = max(last, __shfl_xor(last, x, 64));
  if ((tid & 63) == 0) wave_max[tid >> 6] = last;
  __syncthreads();
  for (int w = 0; w < SEL_T / 64; ++w) last = max(last, wave_max[w]);
  const int64_t local = (int64_t)last - a.n_local;

  auto word = [&](int j) -> uint32_t {
    const int p = c.page_of(table, j);
    if (p < 0) return 0u;
    const int s = c.slot_of(j);
    const int pos = c.pos[p * c.p_ps + hk * c.p_hs + s];
    if (pos < a.n_global || pos > local) return FORCED;
    return weight_word(c.weight[p * c.w_ps + hk * c.w_hs + s]);
  };

  // the m-th largest word, byte by byte; `left` of the words that share its bytes so far stay
  uint32_t T = 0;
  int left = m;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += SEL_T) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < len; j += SEL_T) {
      const uint32_t w = word(j);
      if (shift == 24 || (w >> (shift + 8)) == (T >> (shift + 8))) atomicAdd(&hist[(w >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + hist[d] < left) above += hist[d--];
      pick[0] = d;
      pick[1] = left - above;
    }
    __syncthreads();
    T |= (uint32_t)pick[0] << shift;
    left = pick[1];
    __syncthreads();
  }

  int ties = 0, n_from = 0, n_to = 0;
  int32_t* from = a.from + (int64_t)seg * a.moves;
  int32_t* to = a.to + (int64_t)seg * a.moves;
  for (int j0 = 0; j0 < len; j0 += SEL_T) {
    const int j = j0 + tid;
    const uint32_t w = j < len ? word(j) : 0u;
    const bool tie = j < len && w == T;
    const Ranks rt = rank_flags(tie, false, scan);
    const bool keep = j < len && (w > T || (tie && ties + rt.a < left));
    ties += rt.total_a;
    const bool src = keep && (!in_place || j >= m), dst = in_place && !keep && j < m;
    const Ranks r = rank_flags(src, dst, scan);
    if (src && n_from + r.a < a.moves) from[n_from + r.a] = j;
    if (dst && n_to + r.b < a.moves) to[n_to + r.b] = j;
    n_from += r.total_a;
    n_to += r.total_b;
  }
  if (tid == 0) a.counts[seg] = min(n_from, a.moves);
}

// one group of row_bytes / 16 lanes moves a row's key and value
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  const CacheView& c = a.c;
  const int hk = blockIdx.y, b = blockIdx.z, chunks = a.row_bytes / 16;
  const int seg = b * c.Hkv + hk, n = a.counts[seg];
  const int per = 256 / chunks, at = threadIdx.x % chunks * 16;
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  const int32_t* out_table = a.dst_table ? a.dst_table + (int64_t)b * a.dst_stride : table;
  for (int r = blockIdx.x * per + threadIdx.x / chunks; r < n; r += gridDim.x * per) {
    const int j = a.from[(int64_t)seg * a.moves + r], i = a.dst_table ? r : a.to[(int64_t)seg * a.moves + r];
    if (a.dst_table && i >= a.dst_cap) break;
    const int p = c.page_of(table, j), g = c.page_of(out_table, i);
    if (p < 0 || g < 0) continue;
    const int s = c.slot_of(j), d = c.slot_of(i);
    *(u32x4*)(c.k + g * c.k_ps + hk * c.k_hs + d * c.k_ss + at) =
        *(const u32x4*)(c.k + p * c.k_ps + hk * c.k_hs + s * c.k_ss + at);
    *(u32x4*)(c.v + g * c.v_ps + hk * c.v_hs + d * c.v_ss + at) =
        *(const u32x4*)(c.v + p * c.v_ps + hk * c.v_hs + s * c.v_ss + at);
    if (at == 0) {
      c.weight[g * c.w_ps + hk * c.w_hs + d] = c.weight[p * c.w_ps + hk * c.w_hs + s];
      c.pos[g * c.p_ps + hk * c.p_hs + d] = c.pos[p * c.p_ps + hk * c.p_hs + s];
    }
  }
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t st) {
  evict_select_kernel<<<dim3(a.c.Hkv, a.c.B), SEL_T, 0, st>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.moves == 0) return e;
  const int per = 256 / (a.row_bytes / 16);
  const int blocks = (a.moves + per - 1) / per;
  evict_move_kernel<<<dim3(blocks < 64 ? blocks : 64, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace sta
