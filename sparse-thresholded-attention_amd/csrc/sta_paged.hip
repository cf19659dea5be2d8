// sta_paged.hip -- the paged key-value cache: new rows into their pages, and the attention of a few
// new tokens of every sequence over its cached keys.
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - m_i) / sum_j exp(s_ij - m_i),  s_ij = sm_scale q_i . k_j
//
// over the keys j < len - (Q - 1 - i) of the sequence whose page exists; weight_j += sum_i p_ij over
// the rows i of the kv head.
#include "sta_cache.h"
#include "sta_device.h"

namespace sta {

namespace {

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

// ------------------------------------------------------------------------------------------
// append: a wave per token moves the rows of all kv heads, 16 bytes a lane, two keys' and two values' in flight.  A wave
// finds its token's sequence and page once (a wave per token and head had each search again: 12 prompts of up to 4001
// tokens, 8 heads x 128, bf16: 57 -> 45 us).  Bound by memory: 224 MB there, 5.0 TB/s.
// ------------------------------------------------------------------------------------------
// the last sequence that starts at or before t (64 candidates at once), -1: none
__device__ __forceinline__ int sequence_of(const int32_t* starts, int B, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B;
  for (;;) {
    const int step = (n + 63) / 64, at = lo + lane * step;
    const int below = __popcll(__ballot(at < lo + n && starts[min(at, B)] <= t));
    if (below == 0) return lo - 1;
    const int end = lo + n;
    lo += (below - 1) * step;
    if (step == 1) return lo;
    n = min(step, end - lo);
  }
}

// where sequence b begins among the rows that there are
__device__ __forceinline__ int row_of(const AppendArgs& a, int b) { return min(max(a.starts[b], 0), a.T); }

__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const CacheView& c = a.c;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < c.B; b += 256) {
      const int n = a.starts ? max(row_of(a, b + 1) - row_of(a, b), 0) : 1;
      a.new_lens[b] = (int)min((int64_t)c.len(b) + n, (int64_t)c.cap);
    }
  }
  const int t = blockIdx.x * 4 + uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= a.T) return;
  int b = t, i = 0;
  if (a.starts) {
    b = uniform(sequence_of(a.starts, c.B, t));
    if (b < 0 || t >= a.starts[b + 1]) return;
    i = t - row_of(a, b);
  }
  const int64_t at = (int64_t)c.len(b) + i;
  if (at >= c.cap) return;
  const int j = (int)at, p = uniform(c.page_of(c.table + (int64_t)b * c.t_stride, j));
  if (p < 0) return;
  const int s = c.slot_of(j), shift = a.row_shift, all = c.Hkv << shift;
  const char* k = a.k + t * a.k_ts;
  const char* v = a.v + t * a.v_ts;
  char* ko = c.k + p * c.k_ps + s * c.k_ss;
  char* vo = c.v + p * c.v_ps + s * c.v_ss;
  const int mask = (1 << shift) - 1;
  for (int x = lane; x < all; x += 128) {
    const int h0 = x >> shift, h1 = min(x + 64, all - 1) >> shift, w = (x & mask) * 16, w1 = ((x + 64) & mask) * 16;
    const bool more = x + 64 < all;
    const u32x4 k0 = *(const u32x4*)(k + h0 * a.k_hs + w), v0 = *(const u32x4*)(v + h0 * a.v_hs + w);
    u32x4 k1, v1;
    if (more) {
      k1 = *(const u32x4*)(k + h1 * a.k_hs + w1);
      v1 = *(const u32x4*)(v + h1 * a.v_hs + w1);
    }
    *(u32x4*)(ko + h0 * c.k_hs + w) = k0;
    *(u32x4*)(vo + h0 * c.v_hs + w) = v0;
    if (more) {
      *(u32x4*)(ko + h1 * c.k_hs + w1) = k1;
      *(u32x4*)(vo + h1 * c.v_hs + w1) = v1;
    }
  }
  const int seen = a.seen ? a.seen[b] : j - i, pos = seen > INT32_MAX - i ? INT32_MAX : seen + i;
  for (int h = lane; h < c.Hkv; h += 64) {
    if (c.weight) c.weight[p * c.w_ps + h * c.w_hs + s] = 0.f;
    if (c.pos) c.pos[p * c.p_ps + h * c.p_hs + s] = pos;
  }
}

// ------------------------------------------------------------------------------------------
// attention, split over the keys
// ------------------------------------------------------------------------------------------
// The R = Q * H / Hkv query rows of a kv head share its keys: 16 rows are the columns of the matrix
// instructions, and a workgroup takes NT such tiles over one piece of a sequence's keys.  Its four
// waves walk the piece in turn, KT keys each, on their own: no barrier and no LDS in the loop.
//
//   S^T = K Q^T     K rows as operand A (lane: key l % 16, 16 bytes of its row), Q rows as B; the
//                   result holds row l % 16, keys 4 (l / 16) + i in slot i
//   O^T += V^T P^T  slots 4 (l / 16) + i of both subtiles are, as they stand, the eight contraction elements of
//                   operand B, and lane l loads 1/16 of the V rows of those keys, whose elements e are operand
//                   A of the dims (l % 16) * VE + e
//
// so neither P nor V moves between lanes.  P goes in two 16-bit parts, P = hi + lo within 2^-17 of itself (fp16: down to
// 2^-22), two instructions for each: beside the 2^-8 or 2^-11 of the output's own rounding, which it does not move.  Its
// sum is of the whole P.  fp32 caches use the fp32 instruction of depth 4, whose operands P and V are as well.
//
// Work.  The sequences' lengths are known to the device alone, and differ.  Every wave sums their units (of
// 4 KT keys; an empty sequence counts one, which writes its zeros) over the kv heads, and the call's runs, as many
// as the chip holds workgroups (times the row tiles) at once, take equal numbers of units in the order (sequence, kv
// head, unit).  A run covers the end of one kv head's keys, some whole ones and the beginning of another; whole ones
// are written out, the two others leave a record in the workspace for the join kernel, which finds the runs of a kv
// head by the same division.
constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// whole part of x / y, 0 <= x < 2^40, 1 <= y < 2^40 (the quotient's distance from a whole number above it is
// at least 1 / y, beyond the rounding of the division)
__device__ __forceinline__ int div40(int64_t x, int64_t y) { return (int)((double)x / (double)y); }
__device__ __forceinline__ int units_of(int keys, int unit) { return max(1, (keys + unit - 1) / unit); }

// keys that every query of sequence b sees
__device__ __forceinline__ int common(const PagedArgs& a, int b) { return max(a.c.len(b) - (a.Q - 1), 0); }

// units of a run (at least one); every lane of the wave takes part
__device__ __forceinline__ int64_t units_each(const PagedArgs& a, int unit) {
  int64_t sum = 0;
  for (int b = threadIdx.x & 63; b < a.c.B; b += 64) sum += units_of(common(a, b), unit);
  const int64_t all = uniform(wave_sum64(sum)) * a.c.Hkv;
  return all <= a.runs ? 1 : uniform(div40(all + a.runs - 1, a.runs));
}

// The sequence that holds unit `at` (or, at < 0, sequence b) and the number of its first unit; -1: behind
// the last.  Uniform; every lane takes part.
__device__ __forceinline__ int find_seq(const PagedArgs& a, int unit, int64_t at, int b, int64_t& base) {
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 63;
  int64_t run = 0;
  for (int b0 = 0; b0 < c.B; b0 += 64) {
    const int mine = b0 + lane;
    // up to 64 * 2^22 units of a row tile
    const int n = mine < c.B ? units_of(common(a, mine), unit) : 0;
    const int incl = wave_incl_sum(n);
    const unsigned long long hit = at < 0 ? __ballot(mine == b) : __ballot(run + (int64_t)incl * c.Hkv > at);
    if (hit) {
      const int first = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
      base = run + (int64_t)(__builtin_amdgcn_readlane(incl, first) - __builtin_amdgcn_readlane(n, first)) * c.Hkv;
      return b0 + first;
    }
    run += (int64_t)__builtin_amdgcn_readlane(incl, 63) * c.Hkv;
  }
  return -1;
}

// records: two of every run, for its first and its last kv head where those are unfinished, and (calls of several
// queries) one of every kv head, for those that one run finishes; `tiles` of each
__device__ __forceinline__ int64_t whole_record(const PagedArgs& a, int b, int hk) {
  return 2 * (int64_t)a.runs + (int64_t)b * a.c.Hkv + hk;
}

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ float at_least(float m) { return m == -INFINITY ? 0.f : m; }   // what p is relative to
// What the weights' probabilities are formed from, as exp(score - x) y: a maximum (at_least) and a sum.  Not exp(score -
// lse): near a log-sum-exp of 1000 its rounding alone is 3e-5 of every weight.
__device__ __forceinline__ float2 stats_of(float m, float l) { return make_float2(m, l == 0.f ? 0.f : 1.f / l); }

// waves of a workgroup in a call of short sequences: four a SIMD where a wave gets by with 128 registers
template <int D, int NT>
constexpr int SMALL_WAVES = D == 64 && NT == 1 ? 16 : 8;
// Up to this bound on the lengths (32q / 8kv heads x 128, bf16, one sequence / 32 of them): at 1000 keys 16.0 / 16.2 us in
// one launch, 18.5 / 19.7 split and joined; at 2000 keys 22.2 / 23.7 and 18.1 / 25.2, at 4000 40.2 / 41.9 and 18.4 / 31.5.
constexpr int SMALL_KEYS = 1024;

__device__ const u32x4 zero_row[32] = {};              // 512 bytes: a row of 128 fp32 elements

template <int DT, int D, int NT_>
struct Tile {
  static constexpr int E = DT == DT_F32 ? 4 : 2;
  static constexpr int RB = D * E;                     // bytes of a row
  static constexpr int SUB = DT == DT_F32 ? 1 : 2;     // 16-key subtiles of a wave's turn
  static constexpr int KT = 16 * SUB, UNIT = 4 * KT;
  static constexpr int KS = RB / 64;                   // 16-byte loads of a K row's quarter
  static constexpr int VE = D / 16;                    // V elements of a lane
  static constexpr int VW = VE * E / 4;                // their words
  static constexpr int NT = NT_, ROWS = 16 * NT;
  // P is at most 1: times 2^14 its high fp16 half is normal down to 2^-28, and both hold it within 2^-17 of itself down to
  // 2^-22, within 2^-39 below
  static constexpr float P_SCALE = DT == DT_F16 ? 16384.f : 1.f;
  // Waves of a SIMD, and so workgroups of a CU (256 a grid and wave): what the registers hold without spills.
  // Three at D = 64 (bf16, 32q / 8kv heads, up to 8192 keys: 37 us, with two 41), two at D = 128 (two sequences of up
  // to 131072 keys: 146 us, with three 166: spilled accumulators).
  static constexpr int WAVES = D == 64 && NT == 1 ? 3 : 2;
};

template <int DT>
__device__ __forceinline__ floatx4 mfma_qk(u32x4 k, u32x4 q, floatx4 s) {
  if constexpr (DT == DT_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), s, 0, 0, 0);
  } else if constexpr (DT == DT_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), s, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[e]), s, 0, 0, 0);
    return s;
  }
}

// the low or high 16-bit element of a word, in fp32
template <int DT>
__device__ __forceinline__ float half_of(uint32_t w, int high) {
  if constexpr (DT == DT_BF16) return __uint_as_float(high ? w & 0xffff0000u : w << 16);
  else return f16_bits_to_f32(high ? w >> 16 : w & 0xffffu);
}
// element e of a lane's share of a V row, in fp32
template <int DT>
__device__ __forceinline__ float v_elem(const uint32_t* w, int e) {
  if constexpr (DT == DT_F32) return __uint_as_float(w[e]);
  else return half_of<DT>(w[e / 2], e & 1);
}

// loads at an address in global memory (one that went through a lane exchange is no pointer to the compiler)
typedef const __attribute__((address_space(1))) u32x4* global4;
typedef const __attribute__((address_space(1))) u32x2* global2;
typedef const __attribute__((address_space(1))) uint32_t* global1;
typedef const __attribute__((address_space(1))) uint16_t* global_half;
template <int W>
__device__ __forceinline__ void load_words(int64_t p, uint32_t* w) {
  if constexpr (W == 2) {
    const u32x2 x = *(global2)p;
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 x = *(global4)(p + 4 * i);
      w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
    }
  }
}

// where element (row, dim) of a 16-row tile lies in a wave's accumulators, stored 16 bytes a lane as they are
template <int VE>
__device__ __forceinline__ int acc_index(int row, int dim) {
  const int e = dim % VE, m = dim / VE;                // m = 4 (lane / 16) + slot
  return ((e * 4 + m / 4) * 16 + row) * 4 + m % 4;
}

template <int DT, int N>
__device__ __forceinline__ void store_out(char* out, const float* y) {   // N = 4 or 8
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int e = 0; e < N; e += 4) *(float4*)(out + 4 * e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
  } else if constexpr (N == 8) {
    *(u32x4*)out = u32x4{pack2_dt<DT>(y[0], y[1]), pack2_dt<DT>(y[2], y[3]), pack2_dt<DT>(y[4], y[5]), pack2_dt<DT>(y[6], y[7])};
  } else {
    *(u32x2*)out = u32x2{pack2_dt<DT>(y[0], y[1]), pack2_dt<DT>(y[2], y[3])};
  }
}

template <int D, int NT, int VE>
struct MergeLds {
  floatx4 acc[4][VE * 4 * 16];
  float m[16][16 * NT], l[16][16 * NT], sum[16 * NT];
  float2 stats[16 * NT];
};

// The keys of a turn into a wave's states: sc holds their scores, v their values; P is scaled by p_scale.  EXACT: P.V in
// fp32 throughout.
template <int DT, int D, int NT, bool EXACT, typename Scores, typename Values, typename State, typename Acc>
__device__ __forceinline__ void attend_keys(Scores& sc, Values& v, State& m, State& l, Acc& acc, float p_scale) {
  using T = Tile<DT, D, NT>;
  constexpr int SUB = T::SUB, VE = T::VE;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float top = fmaxf(fmaxf(sc[t][0][0], sc[t][0][1]), fmaxf(sc[t][0][2], sc[t][0][3]));
    if (SUB == 2) top = fmaxf(top, fmaxf(fmaxf(sc[t][SUB - 1][0], sc[t][SUB - 1][1]), fmaxf(sc[t][SUB - 1][2], sc[t][SUB - 1][3])));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m[t])) {
      const float m1 = fmaxf(m[t], top), f = exp_of(m[t] - at_least(m1));
      m[t] = m1;
      l[t] *= f;
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[t][e] *= f;
    }
    const float m0 = at_least(m[t]);
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = p_scale * exp_of(sc[t][s][i] - m0);
        sc[t][s][i] = p;
        l[t] += p;
      }
  }
  if constexpr (EXACT) {
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float ve = v_elem<DT>(v[s][i], e);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(ve, sc[t][s][i], acc[t][e], 0, 0, 0);
        }
  } else {
    u32x4 hi[NT], lo[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p0 = sc[t][x / 2][x % 2 * 2], p1 = sc[t][x / 2][x % 2 * 2 + 1];
        hi[t][x] = pack2_dt<DT>(p0, p1);
        lo[t][x] = pack2_dt<DT>(p0 - half_of<DT>(hi[t][x], 0), p1 - half_of<DT>(hi[t][x], 1));
      }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      u32x4 ve;                                      // element e of the lane's eight keys
#pragma unroll
      for (int x = 0; x < 4; ++x)
        ve[x] = __builtin_amdgcn_perm(v[x / 2][x % 2 * 2 + 1][e / 2], v[x / 2][x % 2 * 2][e / 2],
                                      e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        acc[t][e] = mfma_qk<DT>(ve, hi[t], acc[t][e]);
        acc[t][e] = mfma_qk<DT>(ve, lo[t], acc[t][e]);
      }
    }
  }
}

// The sums of a kv head's waves and runs are added scaled by this, a power of two at most 1 over the number of its keys
// (those that all queries see and the last Q - 1): no sum of theirs exceeds the largest value.
__device__ __forceinline__ float sum_scale(const PagedArgs& a, int common) {
  return __uint_as_float((uint32_t)(127 - (32 - __clz(common + a.Q - 1))) << 23);
}

// Whether a sum is no finite number: one of large values may have passed the type's largest, and an infinite value times
// a part of P that is 0 or below 0 is NaN where the formula says infinity.  Then the keys are taken again, P whole and
// scaled so that no sum of up to 2^28 values exceeds the largest of them.
constexpr float AGAIN_SCALE = 0x1p-28f;
template <int NT, int VE, typename Acc>
__device__ __forceinline__ bool beyond(const Acc& acc) {
  floatx4 zero = floatx4{0.f, 0.f, 0.f, 0.f};            // an infinity or a NaN times 0 is NaN
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < VE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) zero[i] = fmaf(acc[t][e][i], 0.f, zero[i]);
  return (zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.f;
}

// A workgroup of NW waves takes the units u0 .. u1 - 1 of a row tile: out and lse where that is all of it
// (done), else a record.
// MULTI: a.Q may exceed 1.  Then len stands for the keys that all queries see and every row tile is joined:
// paged_join_kernel adds the last Q - 1 keys, of which each query sees others, row by row, so that the rows
// of an instruction always see the same keys (0 times a NaN or an infinity would reach rows that do not
// see its key).
template <int DT, int D, int NT, bool ACC, bool MULTI, int NW>
__device__ __forceinline__ void attend_tile(const PagedArgs& a, MergeLds<D, NT, D / 16>& lds, int b, int len, int hk,
                                            int row0, int u0, int u1, bool done, int64_t record) {
  using T = Tile<DT, D, NT>;
  constexpr int KS = T::KS, VE = T::VE, VW = T::VW, SUB = T::SUB, KT = T::KT;
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int r = lane & 15, g4 = lane >> 4;
  const int G = a.H / c.Hkv, R = G * a.Q;

  u32x4 q[NT][KS];
  int64_t srow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + t * 16 + r;
    const int g = MULTI ? row / a.Q : row, i = MULTI ? row - g * a.Q : 0, h = hk * G + g;
    const bool real = row < R;
    const char* qp = (const char*)a.q + (b * a.q_bs + (real ? h : 0) * a.q_hs + (real ? i : 0) * a.q_ts) * T::E + g4 * 16;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[t][s] = *(const u32x4*)(qp + s * 64);
      if (!real) q[t][s] = u32x4{0, 0, 0, 0};
    }
    if (ACC) srow[t] = real ? (((int64_t)b * a.H + h) * a.Q + i) * a.score_stride + g4 * 4 : -1;
  }

  floatx4 acc[NT][VE];
  float m[NT], l[NT];
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  // A turn's rows: lane l knows those of key l % KT, and the others ask it.  The table entry is loaded two turns
  // ahead, K one turn, V at its turn's beginning.  The last turn, which loads nothing for a next one, is a copy of
  // its own: past a branch that may skip loads the compiler would wait for all loads in flight.
  const int last = max(len - 1, 0) >> c.shift;
  auto entry_at = [&](int u) { return table[min(((u * NW + wave) * KT + (lane & (KT - 1))) >> c.shift, last)]; };
  int64_t krow, vrow;                                  // a key that does not exist is a row of zeros
  auto rows_of = [&](int u, int entry) {               // and which keys exist; lanes beyond KT repeat the first ones
    const int j = (u * NW + wave) * KT + (lane & (KT - 1)), slot = c.slot_of(j);
    const bool is = j < len && (unsigned)entry < (unsigned)c.pages;
    krow = (int64_t)(is ? c.k + hk * c.k_hs + entry * c.k_ps + slot * c.k_ss : (const char*)zero_row);
    vrow = (int64_t)(is ? c.v + hk * c.v_hs + entry * c.v_ps + slot * c.v_ss : (const char*)zero_row);
    return (uint32_t)__ballot(is);
  };
  u32x4 k[SUB][KS];
  auto load_k = [&]() {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int64_t p = __shfl(krow, s * 16 + r, 64) + g4 * 16;
#pragma unroll
      for (int i = 0; i < KS; ++i) k[s][i] = *(global4)(p + i * 64);
    }
  };
  int next_entry;
  uint32_t there;
  auto turn = [&](int u, auto last_turn, auto exact, float p_scale) {
    constexpr bool LAST = decltype(last_turn)::value, EXACT = decltype(exact)::value;
    uint32_t v[SUB][4][VW];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_words<VW>(__shfl(vrow, s * 16 + g4 * 4 + i, 64) + r * (VW * 4), v[s][i]);
    floatx4 sc[NT][SUB];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) x = mfma_qk<DT>(k[s][i], q[t][i], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][s][i] = x[i] * a.sm_scale;
      }
    if (there != ~0u) {
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (!(there >> (g4 * 4) & 1u << (s * 16 + i))) sc[t][s][i] = -INFINITY;
    }
    if (ACC && (u * NW + wave) * KT < len) {           // a turn that begins in the sequence ends in its score rows
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (srow[t] >= 0) {
#pragma unroll
          for (int s = 0; s < SUB; ++s)
            *(floatx4*)(a.scores + srow[t] + (u * NW + wave) * KT + s * 16) = sc[t][s];
        }
    }
    if (!LAST) {
      there = rows_of(u + 1, next_entry);
      load_k();
      next_entry = entry_at(u + 2);
    }
    attend_keys<DT, D, NT, EXACT>(sc, v, m, l, acc, p_scale);
  };
  auto sweep = [&](auto exact, float p_scale) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[t][e] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    there = rows_of(u0, entry_at(u0));
    next_entry = entry_at(u0 + 1);
    load_k();
    int u = u0;
    while (u + 1 < u1) turn(u++, std::integral_constant<bool, false>(), exact, p_scale);
    turn(u, std::integral_constant<bool, true>(), exact, p_scale);
  };
  float unit = 1.f / T::P_SCALE;                       // of the sums
  sweep(std::integral_constant<bool, DT == DT_F32>(), T::P_SCALE);
  if (__builtin_expect(__any(beyond<NT, VE>(acc)), 0)) {
    sweep(std::integral_constant<bool, true>(), AGAIN_SCALE);
    unit = 1.f / AGAIN_SCALE;
  }

  // the waves' states into one
  const float small = sum_scale(a, len);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    l[t] *= unit;
    if (g4 == 0) {
      lds.m[wave][t * 16 + r] = m[t];
      lds.l[wave][t * 16 + r] = l[t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = t * 16 + r, rr = row0 + row;
    float mm = lds.m[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, lds.m[w][row]);
    const float m0 = at_least(mm), f = exp_of(m[t] - m0);
    float ll = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) ll += lds.l[w][row] * exp_of(lds.m[w][row] - m0);
    const float scale = f * (unit * small);
    if (wave == 0 && g4 == 0) {
      lds.sum[row] = ll * small;
      if (ACC) lds.stats[row] = stats_of(m0, ll);
      if (!done) {
        a.part_ml[record * T::ROWS + row] = make_float2(mm, ll);
      } else if (rr < R) {                             // one query
        if (a.lse) a.lse[(int64_t)b * a.H + hk * G + rr] = ll == 0.f ? -INFINITY : m0 + logf(ll);
        if (a.stats) a.stats[((int64_t)b * c.Hkv + hk) * a.stat_stride + rr] = stats_of(m0, ll);
      }
    }
    for (int w = 0; w < NW; w += 4) {                  // four waves' sums at a time
      if (wave / 4 == w / 4) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          floatx4& at = lds.acc[wave % 4][(e * 4 + g4) * 16 + r];
          at = w == 0 ? acc[t][e] * scale : at + acc[t][e] * scale;
        }
      }
      __syncthreads();
    }
    if (tid < 256) {
      // thread: one 16th of a row
      const int orow = tid / 16, m16 = tid % 16, rr = row0 + t * 16 + orow;
      float y[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int at = acc_index<VE>(orow, m16 * VE + e);
        const float* p0 = (const float*)lds.acc[0];
        constexpr int W = VE * 64 * 4;
        y[e] = (p0[at] + p0[W + at]) + (p0[2 * W + at] + p0[3 * W + at]);
      }
      if (!done) {
        store_out<DT_F32, VE>((char*)(a.part_o + (record * T::ROWS + t * 16 + orow) * D + m16 * VE), y);
      } else if (rr < R) {
        const float sum = lds.sum[t * 16 + orow], inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] = sum == 0.f ? 0.f : y[e] * inv;
        store_out<DT, VE>((char*)a.out + (((int64_t)b * a.H + hk * G + rr) * D + m16 * VE) * T::E, y);
      }
    }
    __syncthreads();
  }
}

template <int DT, int D, int NT, bool ACC, bool MULTI>
__global__ __launch_bounds__(256, (Tile<DT, D, NT>::WAVES)) void paged_attend_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, NT>;
  __shared__ MergeLds<D, NT, T::VE> lds;
  const CacheView& c = a.c;
  // workgroups go to the XCDs in turn: the row tiles of a run are 8 apart, on one XCD, and find each other's keys in
  // its L2 (16 queries of 32 heads over 8 kv heads x 128, bf16, 8 sequences up to 8192 keys: 58 -> 50 us)
  const int x = blockIdx.x / 8, tile = tiles == 1 ? 0 : x % tiles;
  const int run = tiles == 1 ? blockIdx.x : x / tiles * 8 + blockIdx.x % 8;
  const int64_t each = units_each(a, T::UNIT);
  const int64_t run0 = run * each, run1 = run0 + each;
  int64_t base = 0;
  int b = find_seq(a, T::UNIT, run0, -1, base);
  if (b < 0) return;
  int len = uniform(common(a, b)), units = units_of(len, T::UNIT);
  int hk = uniform(div40(run0 - base, units));
  for (int64_t at = run0; at < run1;) {
    if (hk == c.Hkv) {
      if (++b == c.B) return;
      base = at;
      hk = 0;
      len = uniform(common(a, b));
      units = units_of(len, T::UNIT);
    }
    const int64_t first = base + (int64_t)hk * units;
    const int u0 = (int)(at - first), u1 = (int)min((int64_t)units, run1 - first);
    const bool whole = u1 - u0 == units;               // the kv head's keys are this run's alone
    const int64_t record = (whole ? whole_record(a, b, hk) : 2 * (int64_t)run + (at != run0)) * tiles + tile;
    attend_tile<DT, D, NT, ACC, MULTI, 4>(a, lds, b, len, hk, tile * T::ROWS, u0, u1, !MULTI && whole, record);
    at = first + u1;
    ++hk;
  }
}

// Many rows a kv head (PagedCut::many): 128 of them a workgroup, 32 a wave, over the same keys.  A turn's 32 keys and
// values go to LDS by asynchronous copies, two turns ahead in three buffers, each wave fetching 8 keys whose page is
// uniform; a row's 16-byte chunks lie permuted by its number, so that the reads of 16 rows' equal chunks and of one row's
// chunks both spread over the banks.  Against 32 rows a workgroup, whose waves read the keys for themselves (32 queries of
// 32 heads over 8 kv heads x 128, 4 sequences up to 12288 keys): 51 -> 42 us.
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void paged_many_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, 2>;
  constexpr int NT = 2, KS = T::KS, VE = T::VE, VW = T::VW, ROWS = Tile<DT, D, 8>::ROWS;
  constexpr int CH = T::RB / 16, PER = 64 / CH, COPIES = 8 / PER;    // chunks of a row, rows of a copy, copies of 8 rows
  __shared__ u32x4 staged[2][3][32 * CH];
  __shared__ int again;
  u32x4 (&keys)[3][32 * CH] = staged[0], (&values)[3][32 * CH] = staged[1];
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 15, g4 = lane >> 4;
  const int G = a.H / c.Hkv, R = G * a.Q;
  const int x = blockIdx.x / 8, tile = tiles == 1 ? 0 : x % tiles;
  const int run = tiles == 1 ? blockIdx.x : x / tiles * 8 + blockIdx.x % 8;
  const int64_t each = units_each(a, T::UNIT);
  const int64_t run0 = run * each, run1 = run0 + each;
  int64_t base = 0;
  int b = find_seq(a, T::UNIT, run0, -1, base);
  if (b < 0) return;
  int len = uniform(common(a, b)), units = units_of(len, T::UNIT);
  int hk = uniform(div40(run0 - base, units));
  for (int64_t at = run0; at < run1;) {
    if (hk == c.Hkv) {
      if (++b == c.B) return;
      base = at;
      hk = 0;
      len = uniform(common(a, b));
      units = units_of(len, T::UNIT);
    }
    const int64_t first = base + (int64_t)hk * units;
    const int u0 = (int)(at - first), u1 = (int)min((int64_t)units, run1 - first);
    const int64_t record = (u1 - u0 == units ? whole_record(a, b, hk) : 2 * (int64_t)run + (at != run0)) * tiles + tile;
    const int t0 = u0 * 4, t1 = min(u1 * 4, (len + 31) / 32);         // turns
    const int32_t* table = c.table + (int64_t)b * c.t_stride;
    const int last = max(len - 1, 0);

    u32x4 q[NT][KS];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = tile * ROWS + wave * 32 + t * 16 + r, g = row / a.Q, i = row - g * a.Q;
      const bool real = row < R;
      const char* qp = (const char*)a.q + (b * a.q_bs + (real ? hk * G + g : 0) * a.q_hs + (real ? i : 0) * a.q_ts) * T::E + g4 * 16;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        q[t][s] = *(const u32x4*)(qp + s * 64);
        if (!real) q[t][s] = u32x4{0, 0, 0, 0};
      }
    }
    struct Entries { int page[4]; };                   // of a turn's four eights of keys, through the scalar cache
    auto entries_of = [&](int t) {
      Entries e;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        e.page[w] = *(const __attribute__((address_space(4))) int32_t*)(int64_t)(table + (min(t * 32 + w * 8, last) >> c.shift));
      return e;
    };
    // copies this wave's keys of turn t, whose entries these are; which keys of the turn exist
    auto stage = [&](int t, int buf, const Entries& e) {
      uint32_t is = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if ((unsigned)e.page[w] < (unsigned)c.pages) is |= 0xffu << (8 * w);
      if (t * 32 + 32 > len) is &= (1u << (len - t * 32)) - 1;         // a turn has a key: len - t * 32 in [1, 31]
      const int page = wave == 0 ? e.page[0] : wave == 1 ? e.page[1] : wave == 2 ? e.page[2] : e.page[3];
#pragma unroll
      for (int y = 0; y < COPIES; ++y) {
        const int row = wave * 8 + y * PER + lane / CH, slot = c.slot_of(t * 32 + row);
        const int chunk = ((lane % CH) ^ (row & (CH - 1))) * 16;
        const bool have = is >> row & 1;
        const char* kp = have ? c.k + hk * c.k_hs + page * c.k_ps + slot * c.k_ss : (const char*)zero_row;
        const char* vp = have ? c.v + hk * c.v_hs + page * c.v_ps + slot * c.v_ss : (const char*)zero_row;
        copy16_to_lds(kp + chunk, uniform((int)lds_addr(&keys[buf][(wave * 8 + y * PER) * CH])));
        copy16_to_lds(vp + chunk, uniform((int)lds_addr(&values[buf][(wave * 8 + y * PER) * CH])));
      }
      return is;
    };
    floatx4 acc[NT][VE];
    float m[NT], l[NT];
    auto sweep = [&](auto exact, float p_scale) {
      constexpr bool EXACT = decltype(exact)::value;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[t][e] = floatx4{0.f, 0.f, 0.f, 0.f};
      }
      uint32_t there = 0, next = 0, after = 0;
      if (t0 < t1) there = stage(t0, 0, entries_of(t0));
      if (t0 + 1 < t1) next = stage(t0 + 1, 1, entries_of(t0 + 1));
      Entries ahead = entries_of(t0 + 2);
      int buf = 0;
      for (int t = t0; t < t1; ++t) {
        // this wave's copies of turn t are done, and its reads of turn t - 1, and with the barrier everyone's
        if (t + 1 < t1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * COPIES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + 2 < t1) {
          after = stage(t + 2, buf == 0 ? 2 : buf - 1, ahead);
          ahead = entries_of(t + 3);
        }
        floatx4 sc[NT][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int row = s * 16 + r;
          u32x4 k[KS];
#pragma unroll
          for (int i = 0; i < KS; ++i) k[i] = keys[buf][row * CH + ((i * 4 + g4) ^ (row & (CH - 1)))];
#pragma unroll
          for (int y = 0; y < NT; ++y) {
            floatx4 z = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KS; ++i) z = mfma_qk<DT>(k[i], q[y][i], z);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[y][s][i] = z[i] * a.sm_scale;
          }
        }
        uint32_t v[2][4][VW];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = s * 16 + g4 * 4 + i;
            if constexpr (VW == 4) {
              const u32x4 w = values[buf][row * CH + (r ^ (row & (CH - 1)))];
#pragma unroll
              for (int y = 0; y < 4; ++y) v[s][i][y] = w[y];
            } else {
              const u32x2 w = ((const u32x2*)values[buf])[(row * CH + ((r >> 1) ^ (row & (CH - 1)))) * 2 + (r & 1)];
              v[s][i][0] = w[0], v[s][i][1] = w[1];
            }
          }
        if (there != ~0u) {
#pragma unroll
          for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!(there >> (g4 * 4) & 1u << (s * 16 + i))) sc[y][s][i] = -INFINITY;
        }
        attend_keys<DT, D, NT, EXACT>(sc, v, m, l, acc, p_scale);
        there = next;
        next = after;
        buf = buf == 2 ? 0 : buf + 1;
      }
    };
    if (tid == 0) again = 0;
    __syncthreads();
    sweep(std::integral_constant<bool, false>(), T::P_SCALE);
    if (beyond<NT, VE>(acc)) again = 1;
    __syncthreads();
    float unit = 1.f / T::P_SCALE;                     // of the sums
    if (again) {
      unit = 1.f / AGAIN_SCALE;
      sweep(std::integral_constant<bool, true>(), AGAIN_SCALE);
      __syncthreads();                                 // staged is free
    }
    const float scale = unit * sum_scale(a, len);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] += __shfl_xor(l[t], 16, 64);
      l[t] += __shfl_xor(l[t], 32, 64);
      l[t] *= unit;
      const int64_t row = record * ROWS + wave * 32 + t * 16;
      if (g4 == 0) a.part_ml[row + r] = make_float2(m[t], l[t]);
      // rows whole, through LDS
      float* mine = (float*)staged + wave * (16 * (D + 4));
#pragma unroll
      for (int e = 0; e < VE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[r * (D + 4) + (g4 * 4 + i) * VE + e] = acc[t][e][i] * scale;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int y = 0; y < D / 16; ++y) {
        const int word = (y * 64 + lane) * 4;
        *(float4*)(a.part_o + row * D + word) = *(const float4*)(mine + word / D * (D + 4) + word % D);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();                                   // the buffers and `again` are free for the next kv head
    at = first + u1;
    ++hk;
  }
}

// Calls whose sequences are all short: one launch.  A workgroup of 8 waves (16 where the registers allow) takes a kv
// head's whole row tile, and adds the weights it gives itself.
template <int DT, int D, int NT, bool ACC>
__global__ __launch_bounds__((64 * SMALL_WAVES<D, NT>), (SMALL_WAVES<D, NT> / 4)) void paged_small_kernel(PagedArgs a) {
  using T = Tile<DT, D, NT>;
  constexpr int NW = SMALL_WAVES<D, NT>;
  __shared__ MergeLds<D, NT, T::VE> lds;
  const CacheView& c = a.c;
  const int hk = blockIdx.x, b = blockIdx.y;
  const int len = uniform(c.len(b)), R = a.H / c.Hkv;
  attend_tile<DT, D, NT, ACC, false, NW>(a, lds, b, len, hk, 0, 0, units_of(len, NW * T::KT), true, 0);
  if constexpr (ACC) {
    // the scores are this workgroup's own: its barriers order them, and its L1 has never held them before
    __threadfence_block();
    __syncthreads();
    const float* s = a.scores + ((int64_t)b * a.H + hk * R) * a.score_stride;
    for (int j = threadIdx.x; j < len; j += 64 * NW) {
      float sum = 0.f;
      for (int r = 0; r < R; ++r) {
        const float2 z = lds.stats[r];
        sum = fmaf(exp_of(s[r * a.score_stride + j] - z.x), z.y, sum);
      }
      const int p = c.page_of(c.table + (int64_t)b * c.t_stride, j);
      if (p >= 0) c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(j)] += sum;
    }
  }
}

// the records of a kv head's keys
struct Records {
  int n;
  int64_t w0, first;
  __device__ __forceinline__ int64_t at(int p) const { return p ? 2 * (w0 + p) : first; }
};
__device__ __forceinline__ Records records_of(const PagedArgs& a, int unit, int b, int hk) {
  const int64_t each = units_each(a, unit);
  int64_t base = 0;
  find_seq(a, unit, -1, b, base);
  const int units = units_of(common(a, b), unit);
  const int64_t first = base + (int64_t)hk * units;
  Records r;
  r.w0 = div40(first, each);
  r.n = (int)(div40(first + units - 1, each) - r.w0) + 1;
  // the first run's record is its second one unless the kv head begins it
  r.first = r.n == 1 ? whole_record(a, b, hk) : 2 * r.w0 + (first != r.w0 * each);
  return r;
}

// lane n of each row of 16 lanes, to all of its row; n is a constant
__device__ __forceinline__ uint32_t row_lane(int n, uint32_t x) {
  switch (n) {
#define STA_ROW_LANE(i) case i: return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x150 + i, 0xf, 0xf, false)
    STA_ROW_LANE(0); STA_ROW_LANE(1); STA_ROW_LANE(2); STA_ROW_LANE(3); STA_ROW_LANE(4); STA_ROW_LANE(5);
    STA_ROW_LANE(6); STA_ROW_LANE(7); STA_ROW_LANE(8); STA_ROW_LANE(9); STA_ROW_LANE(10); STA_ROW_LANE(11);
    STA_ROW_LANE(12); STA_ROW_LANE(13); STA_ROW_LANE(14); STA_ROW_LANE(15);
#undef STA_ROW_LANE
  }
  return x;
}
// the sum over each row of 16 lanes, in every lane
__device__ __forceinline__ float row_sum(float x) {
  x = group8_sum(x);
  return x + __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), 0x140, 0xf, 0xf, false));
}

template <int DT>
__device__ __forceinline__ void store_elem(void* out, int64_t at, float x) {
  if constexpr (DT == DT_F32) ((float*)out)[at] = x;
  else ((uint16_t*)out)[at] = (uint16_t)(DT == DT_F16 ? f32_to_f16_bits(x) : f32_to_bf16_bits(x));
}

// One query: a workgroup per row takes its records, a wave each in turn.
template <int DT, int D, int NT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, NT>;
  constexpr int W = D / 64;                            // a lane's dims
  __shared__ float o[4][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, b = blockIdx.y, G = a.H / a.c.Hkv, hk = h / G, row = h - hk * G;
  const int tile = row / T::ROWS, rr = row - tile * T::ROWS;
  const Records rec = records_of(a, T::UNIT, b, hk);
  if (rec.n == 1) return;                              // written by its workgroup
  auto record = [&](int p) { return (rec.at(p) * tiles + tile) * T::ROWS; };
  const float2* ml = a.part_ml + rr;
  float m = -INFINITY;
  for (int p = lane; p < rec.n; p += 64) m = fmaxf(m, ml[record(p)].x);
  m = wave_max_f32(m);
  const float m0 = at_least(m);
  float l = 0.f;
  for (int p = lane; p < rec.n; p += 64) {
    const float2 x = ml[record(p)];
    l += x.y * exp_of(x.x - m0);
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) l += __shfl_xor(l, s, 64);
  float y[W];
#pragma unroll
  for (int e = 0; e < W; ++e) y[e] = 0.f;
  const float* part = a.part_o + rr * D + lane * W;
#pragma unroll 4
  for (int p = wave; p < rec.n; p += 4) {
    const int64_t at = record(p);
    const float f = exp_of(ml[at].x - m0);
#pragma unroll
    for (int e = 0; e < W; ++e) y[e] += f * part[at * D + e];
  }
#pragma unroll
  for (int e = 0; e < W; ++e) o[wave][lane * W + e] = y[e];
  __syncthreads();
  const int64_t row_out = (int64_t)b * a.H + h;
  if (tid < D) {
    const float sum = (o[0][tid] + o[1][tid]) + (o[2][tid] + o[3][tid]);
    store_elem<DT>(a.out, row_out * D + tid, l == 0.f ? 0.f : sum / (l * sum_scale(a, common(a, b))));
  }
  if (tid == 0) {
    if (a.lse) a.lse[row_out] = l == 0.f ? -INFINITY : m0 + logf(l);
    if (a.stats) a.stats[((int64_t)b * a.c.Hkv + hk) * a.stat_stride + row] = stats_of(m0, l);
  }
}

// Several queries: a wave per row takes its records and then the keys behind the common ones.  The waves of a workgroup
// are rows of one query and kv head where there are four, so that those keys are fetched once.
template <int DT, int D, int NT>
__global__ __launch_bounds__(256) void paged_join_rows_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, NT>;
  constexpr int W = D / 64, VW = T::VW;
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 63, l16 = lane & 15, G = a.H / c.Hkv;
  const int x = blockIdx.x * 4 + uniform((int)threadIdx.x >> 6), b = blockIdx.y;
  if (x >= a.H * a.Q) return;
  const int g = x % G, i = x / G % a.Q, hk = x / (G * a.Q), h = hk * G + g, row = g * a.Q + i;
  const int tile = row / T::ROWS, rr = row - tile * T::ROWS;
  const Records rec = records_of(a, T::UNIT, b, hk);
  auto record = [&](int p) { return (rec.at(p) * tiles + tile) * T::ROWS; };
  const float2* ml = a.part_ml + rr;
  float m = -INFINITY;
  for (int p = lane; p < rec.n; p += 64) m = fmaxf(m, ml[record(p)].x);
  m = wave_max_f32(m);
  float m0 = at_least(m), l = 0.f;
  for (int p = lane; p < rec.n; p += 64) {
    const float2 s = ml[record(p)];
    l += s.y * exp_of(s.x - m0);
  }
  const int n0 = common(a, b), end = c.len(b) - (a.Q - 1 - i);
  const float p_scale = sum_scale(a, n0);
  float y[W];
#pragma unroll
  for (int e = 0; e < W; ++e) y[e] = 0.f;
  const float* part = a.part_o + rr * D + lane * W;
#pragma unroll 4
  for (int p = 0; p < rec.n; ++p) {
    const int64_t at = record(p);
    const float f = exp_of(ml[at].x - m0);
#pragma unroll
    for (int e = 0; e < W; ++e) y[e] += f * part[at * D + e];
  }
  l *= p_scale;
  const int64_t row_out = ((int64_t)b * a.H + h) * a.Q + i;
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  uint32_t q[VW];
  load_words<VW>((int64_t)((const char*)a.q + (b * a.q_bs + h * a.q_hs + i * a.q_ts) * T::E + l16 * (VW * 4)), q);
  for (int j0 = n0; j0 < end; j0 += 64) {
    const int keys = min(end - j0, 64);
    // lane 16 i + j has key 4 j + i: its rows and, at last, its score; lanes behind the keys have rows of zeros
    const int key = l16 * 4 + (lane >> 4);
    const int page = key < keys ? c.page_of(table, j0 + key) : -1, slot = c.slot_of(j0 + key);
    const int64_t krow = (int64_t)(page < 0 ? (const char*)zero_row : c.k + hk * c.k_hs + page * c.k_ps + slot * c.k_ss);
    const int64_t vrow = (int64_t)(page < 0 ? (const char*)zero_row : c.v + hk * c.v_hs + page * c.v_ps + slot * c.v_ss);
    float mine = -INFINITY;
    // 16 lanes a key, four keys an instruction
    auto four = [&](auto step) {
      constexpr int S = decltype(step)::value;
      uint32_t k[4][VW];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t lo = row_lane(S + x, (uint32_t)krow), hi = row_lane(S + x, (uint32_t)(krow >> 32));
        load_words<VW>((int64_t)((uint64_t)hi << 32 | lo) + l16 * (VW * 4), k[x]);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < T::VE; ++e) dot = fmaf(v_elem<DT>(q, e), v_elem<DT>(k[x], e), dot);
        dot = row_sum(dot) * a.sm_scale;
        if (l16 == S + x && page >= 0) mine = dot;
      }
    };
    four(std::integral_constant<int, 0>());
    if (keys > 16) four(std::integral_constant<int, 4>());
    if (keys > 32) four(std::integral_constant<int, 8>());
    if (keys > 48) four(std::integral_constant<int, 12>());
    if (a.scores && key < keys) a.scores[row_out * a.score_stride + j0 + key] = mine;
    const float m1 = fmaxf(wave_max_f32(mine), m);
    m0 = at_least(m1);
    const float f = exp_of(m - m0), p = p_scale * exp_of(mine - m0);
    m = m1;
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < W; ++e) y[e] *= f;
    // a key that does not exist has p = 0 and a row of zeros
    for (int t0 = 0; t0 < keys; t0 += 8) {
      uint32_t w[8][2];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int from = ((t0 + x) & 3) * 16 + ((t0 + x) >> 2);
        const uint32_t lo = __builtin_amdgcn_readlane((int)vrow, from), hi = __builtin_amdgcn_readlane((int)(vrow >> 32), from);
        const int64_t v = (int64_t)((uint64_t)hi << 32 | lo) + lane * (W * T::E);
        if constexpr (W * T::E == 8) load_words<2>(v, w[x]);
        else if constexpr (W * T::E == 4) w[x][0] = *(global1)v;
        else w[x][0] = *(global_half)v;
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int from = ((t0 + x) & 3) * 16 + ((t0 + x) >> 2);
        const float pt = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), from));
#pragma unroll
        for (int e = 0; e < W; ++e) y[e] = fmaf(pt, v_elem<DT>(w[x], e), y[e]);
      }
    }
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) l += __shfl_xor(l, s, 64);
#pragma unroll
  for (int e = 0; e < W; ++e) store_elem<DT>(a.out, row_out * D + lane * W + e, l == 0.f ? 0.f : y[e] / l);
  if (lane == 0) {
    const float l1 = l * (1.f / p_scale);
    if (a.lse) a.lse[row_out] = l == 0.f ? -INFINITY : m0 + logf(l1);
    // the row's own record of the whole kv head, which this wave has read by now
    if (a.stats) a.stats[((int64_t)b * c.Hkv + hk) * a.stat_stride + row] = stats_of(m0, l1);
  }
}

// The weights that a step's rows give the keys of a kv head, from their scores: four keys a lane, 256 a wave.  SHARED: the
// four waves of a workgroup take the rows of 256 keys in turn, and their sums are added in order (many rows); else each
// has keys of its own.  Without SHARED, keys that lie fours to 16 aligned bytes of a page have their weights loaded before
// the scores and written back together (32 sequences of 4096 keys, 32q / 8kv heads, pages of 16: 11.0 -> 9.6 us; 17 MB of
// scores and 8 of weights, bound by the chain length, page, weight and the launch).
template <bool SHARED>
__global__ __launch_bounds__(256) void paged_weight_kernel(PagedArgs a) {
  __shared__ floatx4 sums[SHARED ? 4 : 1][64];
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int b = blockIdx.z, hk = blockIdx.y, j0 = SHARED ? blockIdx.x * 256 : (blockIdx.x * 4 + wave) * 256;
  const int len = uniform(c.len(b));
  if (j0 >= len) return;
  const int rows = a.H / c.Hkv * a.Q;
  const int64_t row0 = ((int64_t)b * c.Hkv + hk) * rows;
  const int j = j0 + lane * 4;
  const bool all = j0 + 256 <= common(a, b);           // every row sees every key
  const float* s = a.scores + row0 * a.score_stride + j;
  const float2* stats = a.stats + ((int64_t)b * c.Hkv + hk) * a.stat_stride;
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  const bool fours = !SHARED && c.shift >= 2 && ((c.w_ps | c.w_hs) & 3) == 0 && ((uintptr_t)c.weight & 15) == 0;
  int page = -1;
  float* drawn = nullptr;
  floatx4 had = floatx4{0.f, 0.f, 0.f, 0.f};
  if (fours && j + 4 <= len) {
    page = c.page_of(table, j);
    drawn = c.weight + (page >= 0 ? page * c.w_ps + hk * c.w_hs + c.slot_of(j) : 0);
    if (page >= 0) had = *(const floatx4*)drawn;
  }
  floatx4 sum = floatx4{0.f, 0.f, 0.f, 0.f};
  constexpr int STEP = SHARED ? 4 : 1;
  const int first = SHARED ? wave : 0;
  if (all) {
#pragma unroll 4
    for (int r = first; r < rows; r += STEP) {
      const floatx4 x = *(const floatx4*)(s + r * a.score_stride);
      const float2 z = stats[r];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(exp_of(x[e] - z.x), z.y, sum[e]);
    }
  } else {
    for (int r = first; r < rows; r += STEP) {
      const int end = len - (a.Q - 1 - r % a.Q);
      if (j >= end) continue;                          // beyond: not written
      const floatx4 x = *(const floatx4*)(s + r * a.score_stride);
      const float2 z = stats[r];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += j + e >= end ? 0.f : exp_of(x[e] - z.x) * z.y;
    }
  }
  if constexpr (SHARED) {
    sums[wave][lane] = sum;
    __syncthreads();
    const int mine = j0 + tid;
    if (mine >= len) return;
    const int p = c.page_of(table, mine);
    const float* w = (const float*)sums;
    if (p >= 0)
      c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(mine)] += (w[tid] + w[256 + tid]) + (w[512 + tid] + w[768 + tid]);
  } else if (fours && j + 4 <= len) {                  // in one page, 16 aligned bytes
    if (page >= 0) *(floatx4*)drawn = had + sum;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = j + e < len ? c.page_of(table, j + e) : -1;
      if (p >= 0) c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(j + e)] += sum[e];
    }
  }
}

// The same from the scores formed again, where a kv head has many rows (PagedCut::reform): a wave holds 64 keys
// in registers, the rows come 64 at a time through LDS, fetched during the 64 before, and each lane adds up its row's p of
// four keys a subtile over the row tiles; the 16 lanes of those keys meet at the end.  Bound by the keys' bytes, a second
// time, and the latencies before them (128 rows a kv head x 128, bf16, 4 sequences up to 12288 keys: 24 us, 28 with the
// rows fetched in their own turn; 50 MB of keys are 10; 32 or 16 keys a wave: the same or slower).
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_reform_kernel(PagedArgs a) {
  using T = Tile<DT, D, 1>;
  constexpr int KS = T::KS, SUBS = 4, ROWS = 64, STRIDE = T::RB / 16 + 1;   // 16-byte words, padded
  __shared__ u32x4 rows[ROWS * STRIDE];
  __shared__ float2 stats[ROWS];
  __shared__ int ends[ROWS];
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 15, g4 = lane >> 4;
  const int b = blockIdx.z, hk = blockIdx.y, block0 = blockIdx.x * (64 * SUBS), key0 = block0 + wave * (16 * SUBS);
  const int len = uniform(c.len(b)), G = a.H / c.Hkv, R = G * a.Q;
  if (block0 >= len) return;
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  // the lane's key of the wave's, and all of them in their lanes
  const int mine = key0 + (lane & (16 * SUBS - 1));
  const int page = mine < len ? c.page_of(table, mine) : -1;
  const int64_t krow =
      (int64_t)(page < 0 ? (const char*)zero_row : c.k + hk * c.k_hs + page * c.k_ps + c.slot_of(mine) * c.k_ss);
  u32x4 k[SUBS][KS];
#pragma unroll
  for (int s = 0; s < SUBS; ++s) {
    const int64_t p = __shfl(krow, s * 16 + r, 64) + g4 * 16;
#pragma unroll
    for (int i = 0; i < KS; ++i) k[s][i] = *(global4)(p + i * 64);
  }
  floatx4 w[SUBS];
#pragma unroll
  for (int s = 0; s < SUBS; ++s) w[s] = floatx4{0.f, 0.f, 0.f, 0.f};
  // the rows of a turn are fetched during the one before
  constexpr int CH = T::RB / 16, PER = ROWS * CH / 256;
  u32x4 held[PER];
  float2 held_z;
  int held_end;
  auto fetch = [&](int r0) {
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      const int rr = min(r0 + (x * 256 + tid) / CH, R - 1), g = rr / a.Q, i = rr - g * a.Q;
      held[x] = *(global4)((int64_t)((const char*)a.q + (b * a.q_bs + (hk * G + g) * a.q_hs + i * a.q_ts) * T::E + tid % CH * 16));
    }
    const int rr = min(r0 + tid % ROWS, R - 1), g = rr / a.Q, i = rr - g * a.Q;
    held_z = a.stats[((int64_t)b * c.Hkv + hk) * a.stat_stride + rr];
    // a row that saw nothing, or is none, sees no key here
    held_end = r0 + tid % ROWS < R && held_z.y != 0.f ? len - (a.Q - 1 - i) : 0;
  };
  fetch(0);
  for (int r0 = 0; r0 < R; r0 += ROWS) {
    const int n = min(R - r0, ROWS);
    __syncthreads();
#pragma unroll
    for (int x = 0; x < PER; ++x) rows[(x * 256 + tid) / CH * STRIDE + tid % CH] = held[x];
    if (tid < ROWS) {
      stats[tid] = held_z;
      ends[tid] = held_end;
    }
    __syncthreads();
    if (r0 + ROWS < R) fetch(r0 + ROWS);
    for (int t = 0; t < n; t += 16) {
      u32x4 q[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) q[i] = rows[(t + r) * STRIDE + i * 4 + g4];
      const float2 z = stats[t + r];
      const int end = ends[t + r];
      floatx4 x[SUBS];
#pragma unroll
      for (int s = 0; s < SUBS; ++s) {
        x[s] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) x[s] = mfma_qk<DT>(k[s][i], q[i], x[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[s][i] = exp_of(x[s][i] * a.sm_scale - z.x) * z.y;
      }
      if (__all(key0 + 16 * SUBS <= end)) {
#pragma unroll
        for (int s = 0; s < SUBS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) w[s][i] += x[s][i];
      } else {
#pragma unroll
        for (int s = 0; s < SUBS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) w[s][i] += key0 + s * 16 + g4 * 4 + i < end ? x[s][i] : 0.f;
      }
    }
  }
  // lane 4 s + i of a row of lanes keeps key 16 s + 4 (lane / 16) + i
  float out = 0.f;
#pragma unroll
  for (int s = 0; s < SUBS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = row_sum(w[s][i]);
      if (r == s * 4 + i) out = x;
    }
  const int j = key0 + r / 4 * 16 + g4 * 4 + r % 4;
  if (r < SUBS * 4 && j < len) {
    const int p = c.page_of(table, j);
    if (p >= 0) c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(j)] += out;
  }
}

template <int DT, int D, int NT, bool MULTI>
hipError_t launch_attend(const PagedArgs& a, const PagedCut& cut, hipStream_t st) {
  if constexpr (!MULTI) {
    if (cut.small) {
      constexpr int threads = 64 * SMALL_WAVES<D, NT>;
      if (a.accumulate) paged_small_kernel<DT, D, NT, true><<<dim3(a.c.Hkv, a.c.B), threads, 0, st>>>(a);
      else paged_small_kernel<DT, D, NT, false><<<dim3(a.c.Hkv, a.c.B), threads, 0, st>>>(a);
      return hipGetLastError();
    }
  }
  if constexpr (MULTI && NT == 2 && DT != DT_F32) {
    if (cut.many) {
      paged_many_kernel<DT, D><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
      hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      paged_join_rows_kernel<DT, D, 8><<<dim3((a.H * a.Q + 3) / 4, a.c.B), 256, 0, st>>>(a, cut.tiles);
      if ((e = hipGetLastError()) != hipSuccess || !a.accumulate) return e;
      paged_reform_kernel<DT, D><<<dim3((a.c.cap + 255) / 256, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
      return hipGetLastError();
    }
  }
  if (a.scores) paged_attend_kernel<DT, D, NT, true, MULTI><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
  else paged_attend_kernel<DT, D, NT, false, MULTI><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    if constexpr (MULTI) paged_join_rows_kernel<DT, D, NT><<<dim3((a.H * a.Q + 3) / 4, a.c.B), 256, 0, st>>>(a, cut.tiles);
    else paged_join_kernel<DT, D, NT><<<dim3(a.H, a.c.B), 256, 0, st>>>(a, cut.tiles);
    e = hipGetLastError();
  }
  if (e != hipSuccess || !a.accumulate) return e;
  if constexpr (DT != DT_F32) {
    if (cut.reform) {
      paged_reform_kernel<DT, D><<<dim3((a.c.cap + 255) / 256, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
      return hipGetLastError();
    }
  }
  if (a.H / a.c.Hkv * a.Q > 16) paged_weight_kernel<true><<<dim3((a.c.cap + 255) / 256, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  else paged_weight_kernel<false><<<dim3((a.c.cap + 1023) / 1024, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  return hipGetLastError();
}

template <int DT, int D>
hipError_t launch_rows(const PagedArgs& a, const PagedCut& cut, hipStream_t st) {
  if (cut.rows > 16) return a.Q == 1 ? launch_attend<DT, D, 2, false>(a, cut, st) : launch_attend<DT, D, 2, true>(a, cut, st);
  return a.Q == 1 ? launch_attend<DT, D, 1, false>(a, cut, st) : launch_attend<DT, D, 1, true>(a, cut, st);
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, hipStream_t st) {
  const unsigned blocks = ((unsigned)a.T + 3) / 4;
  append_kernel<<<blocks ? blocks : 1, 256, 0, st>>>(a);
  return hipGetLastError();
}

PagedCut paged_cut(int dtype, int D, int H, int Hkv, int Q, int B, int cap, int page_size) {
  PagedCut cut;
  const int R = H / Hkv * Q;
  // 128 rows a workgroup past 64 (32q / 8kv heads x 128, bf16, 8 sequences up to 8192 keys, R = 48 / 64 / 80 / 96 / 128: 56 /
  // 56 / 57 / 58 / 53 us, 32 rows a workgroup 51 / 51 / 65 / 66 / 67); an eight of keys has to lie in one page
  cut.many = Q > 1 && R > 64 && dtype != STA_DTYPE_F32 && page_size >= 8;
  cut.rows = cut.many ? 128 : R > 16 ? 32 : 16;
  cut.tiles = (R + cut.rows - 1) / cut.rows;
  const int unit = dtype == STA_DTYPE_F32 ? Tile<DT_F32, 64, 1>::UNIT : Tile<DT_BF16, 64, 1>::UNIT;
  const int waves = cut.rows > 16 ? 2 : (D == 64 ? Tile<DT_BF16, 64, 1>::WAVES : Tile<DT_BF16, 128, 1>::WAVES);
  const int64_t most = cap <= unit ? 1 : (cap + unit - 1) / unit;
  const int64_t all = (int64_t)Hkv * B * most;
  int runs = 256 * waves;
  if (cut.tiles > 1) runs = runs / cut.tiles < 8 ? 8 : runs / cut.tiles / 8 * 8;
  cut.runs = (int)(all < runs ? all : runs);
  cut.grid = cut.tiles == 1 ? cut.runs : (cut.runs + 7) / 8 * 8 * cut.tiles;
  // stored scores cost 8 bytes a row and key, reformed ones the keys once more and their products: 32q / 8kv heads
  // x 128, bf16, 8 sequences up to 8192 keys, R = 24 / 48 / 56 / 64 rows: 48 / 68 / 74 / 80 us stored, 59 / 72 / 74 / 75
  // reformed, and 117 / 93 at R = 128 (4 up to 12288); x 64, R = 32 / 64: 40 / 60 and 40 / 52; fp32, R = 32 / 64, 97 / 147
  // and 118 / 184
  cut.small = Q == 1 && cut.tiles == 1 && cap <= SMALL_KEYS;
  cut.reform = !cut.small && R >= 64 && dtype != STA_DTYPE_F32;
  cut.records = cut.small ? 0 : cut.tiles * (2 * (int64_t)cut.runs + (Q > 1 ? (int64_t)Hkv * B : 0));
  return cut;
}

hipError_t launch_paged(int dtype, int D, const PagedArgs& a, hipStream_t st) {
  const PagedCut cut = paged_cut(dtype, D, a.H, a.c.Hkv, a.Q, a.c.B, a.c.cap, 1 << a.c.shift);
  if (dtype == STA_DTYPE_F32) return D == 64 ? launch_rows<DT_F32, 64>(a, cut, st) : launch_rows<DT_F32, 128>(a, cut, st);
  if (dtype == STA_DTYPE_BF16) return D == 64 ? launch_rows<DT_BF16, 64>(a, cut, st) : launch_rows<DT_BF16, 128>(a, cut, st);
  return D == 64 ? launch_rows<DT_F16, 64>(a, cut, st) : launch_rows<DT_F16, 128>(a, cut, st);
}

}  // namespace sta
