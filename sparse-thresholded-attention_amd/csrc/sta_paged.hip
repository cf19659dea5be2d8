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

// ------------------------------------------------------------------------------------------
// append: one thread moves 16 bytes of a key and of its value
// ------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const CacheView& c = a.c;
  const int chunks = a.row_bytes / 16;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < c.B; b += 256) {
      const int n = a.starts ? max(a.starts[b + 1] - a.starts[b], 0) : 1;
      a.new_lens[b] = (int)min((int64_t)c.len(b) + n, (int64_t)c.cap);
    }
  }
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = gid / chunks;
  if (row >= (int64_t)a.T * c.Hkv) return;
  const int at = (int)(gid - row * chunks) * 16;
  const int t = (int)(row / c.Hkv), h = (int)(row - (int64_t)t * c.Hkv);
  int b = t, i = 0;
  if (a.starts) {
    // the last sequence that starts at or before t
    int lo = 0, hi = c.B;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid] <= t) lo = mid + 1;
      else hi = mid;
    }
    b = lo - 1;
    if (b < 0 || t >= a.starts[b + 1]) return;
    i = t - a.starts[b];
  }
  const int64_t j = (int64_t)c.len(b) + i;
  if (j >= c.cap) return;
  const int p = c.page_of(c.table + (int64_t)b * c.t_stride, (int)j);
  if (p < 0) return;
  const int s = c.slot_of((int)j);
  *(u32x4*)(c.k + p * c.k_ps + h * c.k_hs + s * c.k_ss + at) = *(const u32x4*)(a.k + t * a.k_ts + h * a.k_hs + at);
  *(u32x4*)(c.v + p * c.v_ps + h * c.v_hs + s * c.v_ss + at) = *(const u32x4*)(a.v + t * a.v_ts + h * a.v_hs + at);
  if (at == 0) {
    if (c.weight) c.weight[p * c.w_ps + h * c.w_hs + s] = 0.f;
    if (c.pos) c.pos[p * c.p_ps + h * c.p_hs + s] = (a.seen ? a.seen[b] : (int)j - i) + i;
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
// so neither P nor V moves between lanes.  P goes in two 16-bit parts, P = hi + lo within 2^-17 of itself, two
// instructions for each; fp32 caches use the fp32 instruction of depth 4, whose operands P and V are as well.
//
// Work.  The sequences' lengths are known to the device alone, and differ.  Every wave sums their units (of
// 4 KT keys; an empty sequence counts one, which writes its zeros) over all row tiles, and the call's
// workgroups, as many as the chip holds at once, take equal runs of units in the order (sequence, row
// tile, unit).  A run covers the end of one row tile, some whole ones and the beginning of another; whole
// ones are written out, the two others leave a record in the workspace for the join kernel, which
// finds the workgroups of a row tile by the same division.
constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// whole part of x / y, 0 <= x < 2^40, 1 <= y < 2^40 (the quotient's distance from a whole number above it is
// at least 1 / y, beyond the rounding of the division)
__device__ __forceinline__ int div40(int64_t x, int64_t y) { return (int)((double)x / (double)y); }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

__device__ __forceinline__ int units_of(int keys, int unit) { return max(1, (keys + unit - 1) / unit); }

// keys that every query of sequence b sees
__device__ __forceinline__ int common(const PagedArgs& a, int b) { return max(a.c.len(b) - (a.Q - 1), 0); }

// units that a workgroup takes (at least one); every lane of the wave takes part
__device__ __forceinline__ int64_t units_each(const PagedArgs& a, int unit, int segs) {
  int64_t sum = 0;
  for (int b = threadIdx.x & 63; b < a.c.B; b += 64) sum += units_of(common(a, b), unit);
  const int64_t all = uniform(wave_sum64(sum)) * segs;
  return all <= a.grid ? 1 : uniform(div40(all + a.grid - 1, a.grid));
}

// The sequence that holds unit `at` (or, at < 0, sequence b) and the number of its first unit; -1: behind
// the last.  Uniform; every lane takes part.
__device__ __forceinline__ int find_seq(const PagedArgs& a, int unit, int segs, int64_t at, int b, int64_t& base) {
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 63;
  int64_t run = 0;
  for (int b0 = 0; b0 < c.B; b0 += 64) {
    const int mine = b0 + lane;
    // up to 64 * 2^22 units of a row tile
    const int n = mine < c.B ? units_of(common(a, mine), unit) : 0;
    const int incl = wave_incl_sum(n);
    const unsigned long long hit = at < 0 ? __ballot(mine == b) : __ballot(run + (int64_t)incl * segs > at);
    if (hit) {
      const int first = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
      base = run + (int64_t)(__builtin_amdgcn_readlane(incl, first) - __builtin_amdgcn_readlane(n, first)) * segs;
      return b0 + first;
    }
    run += (int64_t)__builtin_amdgcn_readlane(incl, 63) * segs;
  }
  return -1;
}

// the record of a row tile that one workgroup finished, MULTI calls only: behind the two of each workgroup
__device__ __forceinline__ int64_t whole_record(const PagedArgs& a, int segs, int b, int seg) {
  return 2 * (int64_t)a.grid + (int64_t)b * segs + seg;
}

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ float at_least(float m) { return m == -INFINITY ? 0.f : m; }   // what p is relative to

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
  // P is below 1: times 2^14 its fp16 halves stay clear of the subnormal range down to 2^-28
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

// where element (row, dim) of a 16-row tile lies in a piece's record: the accumulators of a wave as
// they are, so that records are written 16 bytes a lane without a transpose
template <int VE>
__device__ __forceinline__ int part_index(int row, int dim) {
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
  float m[16][16 * NT], l[16][16 * NT], sum[16 * NT], lse[16 * NT];
};

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
  // EXACT: P.V in fp32 throughout
  auto turn = [&](int u, auto last_turn, auto exact) {
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
          const float p = T::P_SCALE * exp_of(sc[t][s][i] - m0);
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
  };
  auto sweep = [&](auto exact) {
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
    while (u + 1 < u1) turn(u++, std::integral_constant<bool, false>(), exact);
    turn(u, std::integral_constant<bool, true>(), exact);
  };
  if constexpr (DT == DT_F32) {
    sweep(std::integral_constant<bool, true>());
  } else {
    sweep(std::integral_constant<bool, false>());
    // an infinite value times a part of P that is 0 or below 0 is NaN where the formula says infinity: then once
    // more with P whole
    bool nan = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < VE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) nan |= acc[t][e][i] != acc[t][e][i];
    if (__any(nan)) sweep(std::integral_constant<bool, true>());
  }

  // the waves' states into one
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
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
    if (wave == 0 && g4 == 0) {
      const float lse = ll == 0.f ? -INFINITY : m0 + logf(ll * (1.f / T::P_SCALE));
      lds.sum[row] = ll;
      lds.lse[row] = lse;
      if (!done) a.part_ml[record * T::ROWS + row] = make_float2(mm, ll);
      else if (rr < R) a.lse[(int64_t)b * a.H + hk * G + rr] = lse;          // done: one query
    }
    for (int w = 0; w < NW; w += 4) {                  // four waves' sums at a time
      if (wave / 4 == w / 4) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          floatx4& at = lds.acc[wave % 4][(e * 4 + g4) * 16 + r];
          at = w == 0 ? acc[t][e] * f : at + acc[t][e] * f;
        }
      }
      __syncthreads();
    }
    if (!done) {
      floatx4* part = (floatx4*)(a.part_o + (record * T::ROWS + t * 16) * D);
      for (int i = tid; i < VE * 64; i += 64 * NW)
        part[i] = (lds.acc[0][i] + lds.acc[1][i]) + (lds.acc[2][i] + lds.acc[3][i]);
    } else if (tid < 256) {
      // thread: one 16th of a row
      const int orow = tid / 16, m16 = tid % 16, rr = row0 + t * 16 + orow;
      const float sum = lds.sum[t * 16 + orow], inv = sum == 0.f ? 0.f : 1.f / sum;
      if (rr < R) {
        float y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int at = part_index<VE>(orow, m16 * VE + e);
          const float* p0 = (const float*)lds.acc[0];
          constexpr int W = VE * 64 * 4;
          y[e] = sum == 0.f ? 0.f : ((p0[at] + p0[W + at]) + (p0[2 * W + at] + p0[3 * W + at])) * inv;
        }
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
  const int segs = c.Hkv * tiles;
  const int64_t each = units_each(a, T::UNIT, segs);
  const int64_t run0 = blockIdx.x * each, run1 = run0 + each;
  int64_t base = 0;
  int b = find_seq(a, T::UNIT, segs, run0, -1, base);
  if (b < 0) return;
  int len = uniform(common(a, b)), units = units_of(len, T::UNIT);
  int seg = uniform(div40(run0 - base, units));
  for (int64_t at = run0; at < run1;) {
    if (seg == segs) {
      if (++b == c.B) return;
      base = at;
      seg = 0;
      len = uniform(common(a, b));
      units = units_of(len, T::UNIT);
    }
    const int64_t first = base + (int64_t)seg * units;
    const int u0 = (int)(at - first), u1 = (int)min((int64_t)units, run1 - first);
    const bool whole = u1 - u0 == units;               // the row tile is this workgroup's alone
    const int64_t record = whole ? whole_record(a, segs, b, seg) : 2 * (int64_t)blockIdx.x + (at != run0);
    const int hk = tiles == 1 ? seg : seg / tiles, row0 = (seg - hk * tiles) * T::ROWS;
    attend_tile<DT, D, NT, ACC, MULTI, 4>(a, lds, b, len, hk, row0, u0, u1, !MULTI && whole, record);
    at = first + u1;
    ++seg;
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
        const float z = lds.lse[r];
        sum += z == -INFINITY ? 0.f : exp_of(s[r * a.score_stride + j] - z);
      }
      const int p = c.page_of(c.table + (int64_t)b * c.t_stride, j);
      if (p >= 0) c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(j)] += sum;
    }
  }
}

// One workgroup per query row: the records of its row tile, a wave each in turn, and (MULTI) the keys behind
// the common ones.
template <int DT, int D, int NT, bool MULTI>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, NT>;
  constexpr int TAIL = 256, W = D / 64;               // a lane's dims
  __shared__ float o[4][D], tail[MULTI ? TAIL : 1];
  __shared__ int tail_page[MULTI ? TAIL : 1];
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hi = blockIdx.x, b = blockIdx.y, G = a.H / c.Hkv, segs = c.Hkv * tiles;
  const int h = MULTI ? hi / a.Q : hi, i = hi - h * a.Q, hk = h / G, row = (h - hk * G) * a.Q + i, rr = row % T::ROWS;
  const int64_t each = units_each(a, T::UNIT, segs);
  int64_t base = 0;
  find_seq(a, T::UNIT, segs, -1, b, base);
  const int n0 = common(a, b), units = units_of(n0, T::UNIT), seg = hk * tiles + row / T::ROWS;
  const int64_t first = base + (int64_t)seg * units;
  const int64_t w0 = div40(first, each);
  const int n = (int)(div40(first + units - 1, each) - w0) + 1;
  if (!MULTI && n == 1) return;
  // the first workgroup's record is its second one unless the row tile begins its run
  const int64_t rec0 = n == 1 ? whole_record(a, segs, b, seg) : 2 * w0 + (first != w0 * each);
  auto record = [&](int p) { return (p ? 2 * (w0 + p) : rec0) * T::ROWS; };
  const float2* ml = a.part_ml + rr;
  float m = -INFINITY;
  for (int p = lane; p < n; p += 64) m = fmaxf(m, ml[record(p)].x);
  m = wave_max_f32(m);
  float m0 = at_least(m), l = 0.f;
  for (int p = lane; p < n; p += 64) {
    const float2 x = ml[record(p)];
    l += x.y * exp_of(x.x - m0);
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) l += __shfl_xor(l, s, 64);
  float y[W];
#pragma unroll
  for (int e = 0; e < W; ++e) y[e] = 0.f;
  const float* part = a.part_o + rr / 16 * 16 * D;
  for (int p = wave; p < n; p += 4) {
    const int64_t rec = record(p);
    const float f = exp_of(ml[rec].x - m0);
#pragma unroll
    for (int e = 0; e < W; ++e) y[e] += f * part[rec * D + part_index<T::VE>(rr % 16, lane * W + e)];
  }
  const int64_t row_out = ((int64_t)b * a.H + h) * a.Q + i;
  if constexpr (MULTI) {
    const int end = c.len(b) - (a.Q - 1 - i), l16 = lane & 15;
    const int32_t* table = c.table + (int64_t)b * c.t_stride;
    uint32_t q[T::VW];
    load_words<T::VW>((int64_t)((const char*)a.q + (b * a.q_bs + h * a.q_hs + i * a.q_ts) * T::E + l16 * (T::VW * 4)), q);
    for (int j0 = n0; j0 < end; j0 += TAIL) {
      const int keys = min(end - j0, TAIL);
      for (int t = tid / 16; t < keys; t += 16) {      // 16 lanes a key
        const int page = c.page_of(table, j0 + t);
        float dot = 0.f;
        if (page >= 0) {
          uint32_t k[T::VW];
          load_words<T::VW>((int64_t)(c.k + page * c.k_ps + hk * c.k_hs + c.slot_of(j0 + t) * c.k_ss + l16 * (T::VW * 4)), k);
#pragma unroll
          for (int e = 0; e < T::VE; ++e) dot = fmaf(v_elem<DT>(q, e), v_elem<DT>(k, e), dot);
        }
#pragma unroll
        for (int s = 8; s; s >>= 1) dot += __shfl_xor(dot, s, 64);
        if (l16 == 0) {
          const float s = page >= 0 ? dot * a.sm_scale : -INFINITY;
          tail[t] = s;
          tail_page[t] = page;
          if (a.accumulate) a.scores[row_out * a.score_stride + j0 + t] = s;
        }
      }
      __syncthreads();
      float top = -INFINITY;
      for (int t = lane; t < keys; t += 64) top = fmaxf(top, tail[t]);
      top = fmaxf(wave_max_f32(top), m);
      m0 = at_least(top);
      const float f = exp_of(m - m0);
      m = top;
      float sum = 0.f;
      for (int t = lane; t < keys; t += 64) sum += T::P_SCALE * exp_of(tail[t] - m0);
#pragma unroll
      for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s, 64);
      l = l * f + sum;
#pragma unroll
      for (int e = 0; e < W; ++e) y[e] *= f;
      for (int t = wave; t < keys; t += 4) {
        const int page = tail_page[t];
        if (page < 0) continue;
        const float p = T::P_SCALE * exp_of(tail[t] - m0);
        const char* v = c.v + page * c.v_ps + hk * c.v_hs + c.slot_of(j0 + t) * c.v_ss;
#pragma unroll
        for (int e = 0; e < W; ++e) y[e] = fmaf(p, load_scalar<DT>(v, lane * W + e), y[e]);
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int e = 0; e < W; ++e) o[wave][lane * W + e] = y[e];
  __syncthreads();
  if (tid < D) {
    const float z = l == 0.f ? 0.f : ((o[0][tid] + o[1][tid]) + (o[2][tid] + o[3][tid])) / l;
    char* out = (char*)a.out + (row_out * D + tid) * T::E;
    if constexpr (DT == DT_F32) *(float*)out = z;
    else *(uint16_t*)out = (uint16_t)(DT == DT_F16 ? f32_to_f16_bits(z) : f32_to_bf16_bits(z));
  }
  if (tid == 0) a.lse[row_out] = l == 0.f ? -INFINITY : m0 + logf(l * (1.f / T::P_SCALE));
}

// The weights that a step's rows give the keys of a kv head: a workgroup takes 256 keys, its waves the rows in
// turn, four keys a lane; the waves' sums are added in order.  Reads each score once.
__global__ __launch_bounds__(256) void paged_weight_kernel(PagedArgs a) {
  constexpr int ROWS = 256;
  __shared__ float lse[ROWS];
  __shared__ floatx4 sums[4][64];
  const CacheView& c = a.c;
  const int b = blockIdx.z, hk = blockIdx.y, j0 = blockIdx.x * 256, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = c.len(b);
  if (j0 >= len) return;
  const int rows = a.H / c.Hkv * a.Q;
  const int64_t row0 = ((int64_t)b * c.Hkv + hk) * rows;
  const int j = j0 + lane * 4;
  const bool all = j0 + 256 <= common(a, b);           // every row sees every key
  floatx4 sum = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < rows; r0 += ROWS) {
    const int n = min(rows - r0, ROWS);
    __syncthreads();
    // a row that saw nothing has lse -inf: 0 for every key
    if (tid < n) lse[tid] = a.lse[row0 + r0 + tid];
    __syncthreads();
    const float* s = a.scores + (row0 + r0) * a.score_stride + j;
    if (all) {
#pragma unroll 4
      for (int r = wave; r < n; r += 4) {
        const floatx4 x = *(const floatx4*)(s + r * a.score_stride);
        const float z = lse[r];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += z == -INFINITY ? 0.f : exp_of(x[e] - z);
      }
    } else {
      for (int r = wave; r < n; r += 4) {
        const int end = len - (a.Q - 1 - (r0 + r) % a.Q);
        if (j >= end) continue;                        // beyond: not written
        const floatx4 x = *(const floatx4*)(s + r * a.score_stride);
        const float z = lse[r];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += j + e >= end || z == -INFINITY ? 0.f : exp_of(x[e] - z);
      }
    }
  }
  sums[wave][lane] = sum;
  __syncthreads();
  const int mine = j0 + tid;
  if (mine >= len) return;
  const int p = c.page_of(c.table + (int64_t)b * c.t_stride, mine);
  if (p < 0) return;
  const float* w = (const float*)sums;
  c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(mine)] += (w[tid] + w[256 + tid]) + (w[512 + tid] + w[768 + tid]);
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
  if (a.accumulate) paged_attend_kernel<DT, D, NT, true, MULTI><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
  else paged_attend_kernel<DT, D, NT, false, MULTI><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    paged_join_kernel<DT, D, NT, MULTI><<<dim3(a.H * a.Q, a.c.B), 256, 0, st>>>(a, cut.tiles);
    e = hipGetLastError();
  }
  if (e != hipSuccess || !a.accumulate) return e;
  paged_weight_kernel<<<dim3((a.c.cap + 255) / 256, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  return hipGetLastError();
}

template <int DT, int D>
hipError_t launch_rows(const PagedArgs& a, const PagedCut& cut, hipStream_t st) {
  if (cut.rows == 32) return a.Q == 1 ? launch_attend<DT, D, 2, false>(a, cut, st) : launch_attend<DT, D, 2, true>(a, cut, st);
  return a.Q == 1 ? launch_attend<DT, D, 1, false>(a, cut, st) : launch_attend<DT, D, 1, true>(a, cut, st);
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, hipStream_t st) {
  const int64_t threads = (int64_t)a.T * a.c.Hkv * (a.row_bytes / 16);
  const unsigned blocks = (unsigned)((threads + 255) / 256);
  append_kernel<<<blocks ? blocks : 1, 256, 0, st>>>(a);
  return hipGetLastError();
}

PagedCut paged_cut(int dtype, int D, int H, int Hkv, int Q, int B, int cap) {
  PagedCut cut;
  const int R = H / Hkv * Q;
  cut.rows = R > 16 ? 32 : 16;
  cut.tiles = (R + cut.rows - 1) / cut.rows;
  const int unit = dtype == STA_DTYPE_F32 ? Tile<DT_F32, 64, 1>::UNIT : Tile<DT_BF16, 64, 1>::UNIT;
  const int waves = cut.rows == 32 ? 2 : (D == 64 ? Tile<DT_BF16, 64, 1>::WAVES : Tile<DT_BF16, 128, 1>::WAVES);
  const int64_t most = cap <= unit ? 1 : (cap + unit - 1) / unit;
  const int64_t all = (int64_t)Hkv * cut.tiles * B * most;
  cut.grid = (int)(all < 256 * waves ? all : 256 * waves);
  cut.small = Q == 1 && cut.tiles == 1 && cap <= SMALL_KEYS;
  cut.records = cut.small ? 0 : 2 * (int64_t)cut.grid + (Q > 1 ? (int64_t)Hkv * cut.tiles * B : 0);
  return cut;
}

hipError_t launch_paged(int dtype, int D, const PagedArgs& a, hipStream_t st) {
  const PagedCut cut = paged_cut(dtype, D, a.H, a.c.Hkv, a.Q, a.c.B, a.c.cap);
  if (dtype == STA_DTYPE_F32) return D == 64 ? launch_rows<DT_F32, 64>(a, cut, st) : launch_rows<DT_F32, 128>(a, cut, st);
  if (dtype == STA_DTYPE_BF16) return D == 64 ? launch_rows<DT_BF16, 64>(a, cut, st) : launch_rows<DT_BF16, 128>(a, cut, st);
  return D == 64 ? launch_rows<DT_F16, 64>(a, cut, st) : launch_rows<DT_F16, 128>(a, cut, st);
}

}  // namespace sta
