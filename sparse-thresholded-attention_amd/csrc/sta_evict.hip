// sta_evict.hip -- eviction from a paged cache by accumulated attention weight.
//
// Every kv head of a sequence keeps m = min(len, budget) keys.  A key's rank is one 32-bit word,
// larger first: all ones for a forced key (pos < n_global or pos > largest pos - n_local), else
// its weight's bits in an order-preserving form (NaN above +inf, -0 as +0), 0 for a key without a
// page.  The m-th largest word T comes from three counting passes over 10, 11 and 11 bits; a key stays if
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
constexpr int BINS = 2048;             // of a counting pass
constexpr int PER = 8;                 // consecutive keys of a thread
constexpr int COPIES = 4;              // of the counting table
constexpr int LDS_KEYS = 28672;        // 112 KB of words
constexpr int FOURS = LDS_KEYS / 4 / SEL_T;
constexpr int INLINE_MOVES = 64;       // rows a head that the selecting workgroup moves itself
constexpr uint32_t FORCED = 0xffffffffu;

__device__ __forceinline__ uint32_t weight_word(float w) {
  if (w != w) return FORCED - 1;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// exclusive prefix sum over the workgroup and its total; lds: SEL_T / 64 words, free on return
__device__ __forceinline__ int block_prefix(int x, int* lds, int& total) {
  const int wave = threadIdx.x >> 6, incl = wave_incl_sum(x);
  if ((threadIdx.x & 63) == 63) lds[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < SEL_T / 64; ++w) {
    const int t = lds[w];
    if (w < wave) before += t;
    total += t;
  }
  __syncthreads();
  return before + incl - x;
}

// A row's worth of lanes moves a key's row and its value's, r-th of n, with weight and pos; from and to: the slots.
__device__ __forceinline__ void move_rows(const EvictArgs& a, int hk, int b, const int* from, const int* to, int n,
                                          int r0, int step, int tid) {
  const CacheView& c = a.c;
  const int chunks = a.row_bytes / 16, at = tid % chunks * 16;
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  const int32_t* out_table = a.dst_table ? a.dst_table + (int64_t)b * a.dst_stride : table;
  for (int r = r0 + tid / chunks; r < n; r += step) {
    const int j = from[r], i = a.dst_table ? r : to[r];
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

// One workgroup per sequence and kv head, so that ranks need no exchange between workgroups.  Bound by the latencies of
// its loads, passes and barriers: 15 us for 8 sequences of up to 12288 keys, 13 with the moves for 32 of 4097 (8 kv heads).
// KEPT: the words stay in LDS, and weight and pos are read once, four keys a load, into registers (calls of at most
// LDS_KEYS keys whose pages hold four keys in 16 aligned bytes); else each pass reads them again.
// INLINE: the few rows that can move are moved here.
template <bool KEPT, bool INLINE>
__global__ __launch_bounds__(SEL_T) void evict_select_kernel(EvictArgs a) {
  extern __shared__ __align__(16) uint32_t words[];
  __shared__ __align__(16) int hist[BINS * COPIES];
  __shared__ int scan[SEL_T / 64], pick[3];
  const CacheView& c = a.c;
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  __shared__ int moved[2][INLINE ? INLINE_MOVES : 1];
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  const float* weight = c.weight + hk * c.w_hs;
  const int32_t* posp = c.pos + hk * c.p_hs;
  int last = INT32_MIN;
  int4 kp[KEPT ? FOURS : 1];
  float4 kw[KEPT ? FOURS : 1];
  bool there[KEPT ? FOURS : 1];
  if constexpr (KEPT) {
    // not waiting for the length: what a page holds behind it can be read
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
      const int j = (i * SEL_T + tid) * 4;
      there[i] = false;
      if (i * SEL_T * 4 < c.cap) {
        const int p = j < c.cap ? c.page_of(table, j) : -1;
        const int s = c.slot_of(j);
        there[i] = p >= 0;
        if (there[i]) {
          kp[i] = *(const int4*)(posp + p * c.p_ps + s);
          kw[i] = *(const float4*)(weight + p * c.w_ps + s);
        }
      }
    }
  }
  for (int i = tid; i < BINS * COPIES; i += SEL_T) hist[i] = 0;
  const int len = c.len(b), m = min(len, a.budget);
  const int seg = b * c.Hkv + hk;
  if (hk == 0 && tid == 0) a.new_lens[b] = m;
  const bool in_place = a.dst_table == nullptr;
  if (m == 0 || (in_place && len <= a.budget)) {
    if (tid == 0) a.counts[seg] = 0;
    return;
  }
  if constexpr (KEPT) {
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
      const int j = (i * SEL_T + tid) * 4;
      if (there[i] && j < len) {
        last = max(last, kp[i].x);
        if (j + 1 < len) last = max(last, kp[i].y);
        if (j + 2 < len) last = max(last, kp[i].z);
        if (j + 3 < len) last = max(last, kp[i].w);
      }
    }
  } else {
#pragma unroll 4
    for (int j = tid; j < len; j += SEL_T) {
      const int p = c.page_of(table, j);
      if (p >= 0) last = max(last, posp[p * c.p_ps + c.slot_of(j)]);
    }
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) last = max(last, __shfl_xor(last, x, 64));
  if ((tid & 63) == 0) scan[tid >> 6] = last;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SEL_T / 64; ++w) last = max(last, scan[w]);
  const int64_t local = (int64_t)last - a.n_local;

  auto rank = [&](int pos, float w) { return pos < a.n_global || pos > local ? FORCED : weight_word(w); };
  auto fresh = [&](int j) -> uint32_t {
    const int p = c.page_of(table, j);
    if (p < 0) return 0u;
    const int s = c.slot_of(j);
    return rank(posp[p * c.p_ps + s], weight[p * c.w_ps + s]);
  };
  auto word = [&](int j) { return KEPT ? words[j] : fresh(j); };
  // weights crowd into few bins of the first pass: lanes count in 8 tables side by side, then in 4 of twice the bins
  auto count = [&](uint32_t bin, int copies) { atomicAdd(&hist[bin * copies + (tid & (copies - 1))], 1); };

  // the m-th largest word, 10 bits, 11 and 11; `left` of the words equal to it stay
  uint32_t T = 0;
  int left = m, equals = 0;
#pragma unroll
  for (int shift = 22; shift >= 0; shift -= 11) {
    const bool top = shift == 22;
    const int copies = top ? 2 * COPIES : COPIES, bins = top ? BINS / 2 : BINS;
    if (KEPT && top) {
#pragma unroll
      for (int i = 0; i < FOURS; ++i) {
        const int j = (i * SEL_T + tid) * 4;
        if (j < len) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (there[i])
            w = make_uint4(rank(kp[i].x, kw[i].x), rank(kp[i].y, kw[i].y), rank(kp[i].z, kw[i].z), rank(kp[i].w, kw[i].w));
          *(uint4*)(words + j) = w;
          count(w.x >> 22, copies);
          if (j + 1 < len) count(w.y >> 22, copies);
          if (j + 2 < len) count(w.z >> 22, copies);
          if (j + 3 < len) count(w.w >> 22, copies);
        }
      }
    } else {
#pragma unroll 4
      for (int j = tid; j < len; j += SEL_T) {
        const uint32_t w = word(j);
        if (top || w >> (shift + 11) == T >> (shift + 11)) count((w >> shift) & (bins - 1), copies);
      }
    }
    __syncthreads();
    // 8 numbers a thread, from the top: one bin of 8 copies or two of 4; the bin in which the left-th word lies
    int4* h = (int4*)&hist[(SEL_T - 1 - tid) * 8];
    const int4 low = h[0], high = h[1];
    h[0] = h[1] = make_int4(0, 0, 0, 0);
    int mine[2] = {(high.x + high.y) + (high.z + high.w), (low.x + low.y) + (low.z + low.w)}, total;
    if (top) mine[0] += mine[1], mine[1] = 0;
    int above = block_prefix(mine[0] + mine[1], scan, total);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (above < left && above + mine[i] >= left) {
        pick[0] = top ? SEL_T - 1 - tid : 2 * (SEL_T - 1 - tid) + 1 - i;
        pick[1] = left - above;
        pick[2] = mine[i];
      }
      above += mine[i];
    }
    __syncthreads();
    T |= (uint32_t)pick[0] << shift;
    left = pick[1];
    equals = pick[2];
    __syncthreads();
  }

  // who stays, in the order of the slots, PER consecutive ones a thread
  int ties = 0, n_from = 0, n_to = 0;
  int32_t* from = INLINE ? moved[0] : a.from + (int64_t)seg * a.moves;
  int32_t* to = INLINE ? moved[1] : a.to + (int64_t)seg * a.moves;
  for (int j0 = 0; j0 < len; j0 += SEL_T * PER) {
    const int j = j0 + tid * PER;
    uint32_t above = 0, equal = 0;                     // a bit a key
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t w = j + i < len ? word(j + i) : 0u;
      above |= (uint32_t)(j + i < len && w > T) << i;
      equal |= (uint32_t)(j + i < len && w == T) << i;
    }
    int total;
    uint32_t keep = above;
    if (left == equals) {                              // as without ties
      keep |= equal;
    } else {
      int rank = ties + block_prefix(__popc(equal), scan, total);
      ties += total;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (equal >> i & 1) keep |= (uint32_t)(rank++ < left) << i;
    }
    // slots of this thread's keys in front of m
    const int front = min(max(m - j, 0), PER);
    const uint32_t before = (1u << front) - 1;
    const uint32_t src = in_place ? keep & ~before : keep, dst = in_place ? ~keep & before : 0u;
    // both counts in one sum: a turn has SEL_T * PER < 2^16 keys
    const int at = block_prefix(__popc(src) | __popc(dst) << 16, scan, total);
    int from_at = n_from + (at & 0xffff), to_at = n_to + (at >> 16);
    n_from += total & 0xffff;
    n_to += total >> 16;
    for (uint32_t x = src; x; x &= x - 1, ++from_at)
      if (from_at < a.moves) from[from_at] = j + __ffs(x) - 1;
    for (uint32_t x = dst; x; x &= x - 1, ++to_at)
      if (to_at < a.moves) to[to_at] = j + __ffs(x) - 1;
  }
  n_from = min(n_from, a.moves);
  if (INLINE) {
    __syncthreads();
    move_rows(a, hk, b, from, to, n_from, 0, SEL_T / (a.row_bytes / 16), tid);
  } else if (tid == 0) {
    a.counts[seg] = n_from;
  }
}

// Bound by memory: the rows kept of 8 sequences of up to 12288 keys, 2048 a head, 8 kv heads x 128, bf16, into other pages:
// 17 us, the rate of a copy.
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  const int hk = blockIdx.y, b = blockIdx.z, per = 256 / (a.row_bytes / 16);
  const int64_t seg = (int64_t)b * a.c.Hkv + hk;
  move_rows(a, hk, b, a.from + seg * a.moves, a.to + seg * a.moves, a.counts[seg], blockIdx.x * per, gridDim.x * per,
            threadIdx.x);
}

template <bool KEPT, bool INLINE>
hipError_t launch_select(const EvictArgs& a, size_t lds, hipStream_t st) {
  if (lds > 24 * 1024) {                               // with the static tables beyond the 64 KB of any launch
    hipError_t e = hipFuncSetAttribute((const void*)evict_select_kernel<KEPT, INLINE>,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  evict_select_kernel<KEPT, INLINE><<<dim3(a.c.Hkv, a.c.B), SEL_T, lds, st>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t st) {
  const bool fours = a.c.shift >= 2 && ((a.c.w_ps | a.c.w_hs | a.c.p_ps | a.c.p_hs) & 3) == 0 &&
                     (((uintptr_t)a.c.weight | (uintptr_t)a.c.pos) & 15) == 0;
  const bool kept = a.c.cap <= LDS_KEYS && fours, few = a.moves <= INLINE_MOVES;
  const size_t lds = kept ? (size_t)(a.c.cap + 3) / 4 * 16 : 0;
  hipError_t e = kept ? (few ? launch_select<true, true>(a, lds, st) : launch_select<true, false>(a, lds, st))
                        : (few ? launch_select<false, true>(a, lds, st) : launch_select<false, false>(a, lds, st));
  if (e != hipSuccess || few) return e;
  const int per = 256 / (a.row_bytes / 16);
  const int blocks = (a.moves + per - 1) / per;
  evict_move_kernel<<<dim3(blocks < 64 ? blocks : 64, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace sta
