// sta_window.h -- attention over packed sequences with a sliding window and first keys that stay
// visible (sinks): arguments, and what its forward and backward kernels share.
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - m_i) / sum_j exp(s_ij - m_i),  s_ij = sm_scale q_i . k_j
//
// over the keys j <= p_i with j > p_i - window or j < sinks, p_i = nk - nq + i the row's position among its
// sequence's nk keys.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sta_device.h"

namespace sta {

struct WindowArgs {
  const char *q, *k, *v, *dout;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, do_ts, do_hs;   // bytes
  const int32_t *starts, *k_starts;        // NULL: one sequence
  int T, S, H, Hkv, B;
  int window, sinks;                       // window INT_MAX: every earlier key
  float scale;                             // of the scores
  float c;                                 // |scale| log2(e), or 1 where that is no normal number
  uint32_t flip;                           // bits that turn q into its sign's product: 0, or a sign bit an element
  uint32_t keep;                           // all ones; 0 where the scale counts as none: scores are 0
  char* out;
  float* lse;                              // (H, T)
  const float* lse_in;
  // backward
  char *dq, *dk, *dv;
  float *row_lse, *row_delta;              // (H, T): log2 of the sum of exp, +inf for rows that see nothing; sum_d out dout
  float* norms;                            // fp16: (blocks, 2) largest |dout row|^2 and |v row|^2
  int norm_blocks;
  float* record;                           // (records, 2, 128, D) unfinished dk and dv
  int steps;                               // row steps of a work item of the key pass
  int near_steps;                          // row steps that a key tile has at most, a query head
  int q_tiles, k_tiles, items;             // bounds of the grids, a head / kv head
};

// how the key pass is cut (host)
struct WindowCut {
  int q_tiles, k_tiles, items, steps, near_steps, norm_blocks;
  int64_t records;
};
WindowCut window_cut(int dtype, int D, int T, int S, int H, int Hkv, int B, bool starts, bool k_starts, int window,
                     int sinks);

hipError_t launch_window(int dtype, int D, const WindowArgs& a, hipStream_t st);
hipError_t launch_window_grad(int dtype, int D, const WindowArgs& a, int64_t records, hipStream_t st);

#ifdef __HIPCC__
namespace window {

constexpr int ROWS = 128;                  // rows (keys in the key pass) a workgroup, 32 a wave

template <int DT, int D_>
struct Tile {
  static constexpr int D = D_, E = DT == DT_F32 ? 4 : 2, RB = D * E, CH = RB / 16;
  static constexpr int KD = RB / 32;       // products over a row: 32 bytes of it each, 16 a half wave
  static constexpr int DB = D / 32;        // blocks of 32 dims
  static constexpr int KT = DT == DT_F32 ? 32 : 64;   // rows of a stage
  static constexpr int SUB = KT / 32;
  static constexpr int COPIES = KT * CH / 256;        // a wave's 1 KB copies of a stage's rows
};

// Rows lie in LDS as they are, their 16-byte chunks permuted by the row: chunk c of row r at c ^ swz(r).  Both reads then
// spread over the banks: 16 rows' equal chunks (a row an operand lane), and for the transposing reads (16-bit) 64
// bytes of 8 rows, for fp32 128 bytes of two rows 4 apart.
template <typename T>
__device__ __forceinline__ int swz(int r) {
  if constexpr (T::E == 4) return (r & 3) | (r >> 3 & 1) << 2 | (r >> 2 & 1) << 3;
  else if constexpr (T::CH == 16) return (r & 3) << 2 | (r >> 2 & 3);
  else return (r >> 1 & 1) << 2 | (r >> 2 & 3);
}

template <int DT>
__device__ __forceinline__ floatx16 mma(u32x4 a, u32x4 b, floatx16 c) {
  if constexpr (DT == DT_BF16) return mfma32(a, b, c);
  else if constexpr (DT == DT_F16) return mfma32_f16(a, b, c);
  else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ const u32x4 zero_row[32] = {};  // 512 bytes: a row of 128 fp32 elements

// rows row0 .. row0 + KT - 1 of a sequence into a stage, this wave's share; rows from n on are zeros
template <typename T>
__device__ __forceinline__ void stage(u32x4* to, const char* base, int64_t stride, int row0, int n) {
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  constexpr int PER = 64 / T::CH;          // rows of a copy
#pragma unroll
  for (int y = 0; y < T::COPIES; ++y) {
    const int r = (wave * T::COPIES + y) * PER + lane / T::CH;
    const char* p = row0 + r < n ? base + (row0 + r) * stride : (const char*)zero_row;
    copy16_to_lds(p + ((lane % T::CH) ^ swz<T>(r)) * 16, uniform((int)lds_addr(to + (wave * T::COPIES + y) * 64)));
  }
}

// scores: 32 rows of a stage from row0 (operand A) times the wave's 32 rows in registers (operand B).  Slot i of lane l is
// stage row row0 + 8 (i / 4) + 4 (l / 32) + i % 4, own row l % 32.
template <int DT, typename T>
__device__ __forceinline__ floatx16 rows_product(const u32x4* lds, int row0, const u32x4 (&own)[T::KD]) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  floatx16 x;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  const u32x4* row = lds + (row0 + r) * T::CH;
  const int s = swz<T>(r);
#pragma unroll
  for (int d = 0; d < T::KD; ++d) x = mma<DT>(row[(2 * d + h) ^ s], own[d], x);
  return x;
}

// what rows_product leaves, as operand B of the product over the stage's 32 rows: for 16 bits rounded to them
template <int DT>
struct Weights {
  u32x4 w[2];
  __device__ __forceinline__ void set(const floatx16& x) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[s][e] = pack2_dt<DT>(x[8 * s + 2 * e], x[8 * s + 2 * e + 1]);
  }
};
template <>
struct Weights<DT_F32> {
  floatx16 w;
  __device__ __forceinline__ void set(const floatx16& x) { w = x; }
};

// acc (dims x own rows) += (32 rows of a stage from row0)^T x weights
template <int DT, typename T>
__device__ __forceinline__ void transposed_product(const u32x4* lds, int row0, const Weights<DT>& p, floatx16 (&acc)[T::DB]) {
  const int lane = threadIdx.x & 63, h = lane >> 5;
  if constexpr (DT == DT_F32) {
    const float* at = (const float*)lds;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 8 * (i / 4) + 4 * h + i % 4;
#pragma unroll
      for (int b = 0; b < T::DB; ++b) {
        const int dim = b * 32 + (lane & 31);
        const float x = at[((row0 + r) * T::CH + ((dim / 4) ^ swz<T>(r))) * 4 + dim % 4];
        acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p.w[i], acc[b], 0, 0, 0);
      }
    }
  } else {
    const uint16_t* at = (const uint16_t*)lds;
    const int r4 = 4 * h + (lane & 15) / 4, half = lane >> 4 & 1, c2 = (lane & 3) >> 1, low = (lane & 1) * 4;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int b = 0; b < T::DB; ++b) {
        u32x4 a;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = 8 * y + r4;
          const u32x2 x = tr_read16x4(at + ((row0 + 16 * s + r) * T::CH + ((b * 4 + half * 2 + c2) ^ swz<T>(r))) * 8 + low);
          a[2 * y] = x[0], a[2 * y + 1] = x[1];
        }
        acc[b] = mma<DT>(a, p.w[s], acc[b]);
      }
  }
}

// one of the wave's own 32 rows, as operand B: lane l has row l % 32
template <typename T>
__device__ __forceinline__ void load_rows(u32x4 (&own)[T::KD], const char* base, int64_t stride, int row, int n) {
  const int h = (threadIdx.x & 63) >> 5;
  const char* p = row < n ? base + row * stride : (const char*)zero_row;
#pragma unroll
  for (int d = 0; d < T::KD; ++d) own[d] = *(const u32x4*)(p + (2 * d + h) * 16);
}

template <int DT, int KD>
__device__ __forceinline__ void signed_rows(u32x4 (&own)[KD], uint32_t flip, uint32_t keep) {
#pragma unroll
  for (int d = 0; d < KD; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) own[d][e] = (own[d][e] ^ flip) & keep;
}

// dims x own rows -> own row l % 32 of out, times scale
template <int DT, typename T>
__device__ __forceinline__ void store_rows(char* row, const floatx16 (&acc)[T::DB], float scale) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int b = 0; b < T::DB; ++b)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int dim = b * 32 + s * 8 + h * 4;
      const float x0 = acc[b][4 * s] * scale, x1 = acc[b][4 * s + 1] * scale;
      const float x2 = acc[b][4 * s + 2] * scale, x3 = acc[b][4 * s + 3] * scale;
      if constexpr (DT == DT_F32) *(float4*)(row + dim * 4) = make_float4(x0, x1, x2, x3);
      else *(u32x2*)(row + dim * 2) = u32x2{pack2_dt<DT>(x0, x1), pack2_dt<DT>(x2, x3)};
    }
}

// ------------------------------------------------------------------------------------------
// sequences
// ------------------------------------------------------------------------------------------
struct Span {
  int at, n;                               // first row among the packed ones, rows
};
__device__ __forceinline__ Span span_of(const int32_t* starts, int b, int total) {
  if (!starts) return Span{0, total};
  const int s = min(max(starts[b], 0), total);
  return Span{s, max(min(starts[b + 1], total) - s, 0)};
}
// entry 0: the rows in front of the first sequence, 1 .. B: the sequences, B + 1: the rows behind the last
__device__ __forceinline__ Span entry_of(const int32_t* starts, int e, int B, int total) {
  if (e >= 1 && e <= B) return span_of(starts, e - 1, total);
  if (!starts) return Span{0, 0};
  if (e == 0) return Span{0, min(max(starts[0], 0), total)};
  const int s = min(max(starts[B], 0), total);
  return Span{s, total - s};
}

// The entry that holds number `at` when entry e holds count(e) of them, the number of its first one, and the sum of
// other(e) over the entries before it; -1: behind the last.  Uniform; every lane takes part.
template <typename Count, typename Other>
__device__ __forceinline__ int find_entry(int entries, int at, Count count, Other other, int& base, int& before) {
  const int lane = threadIdx.x & 63;
  base = before = 0;
  for (int e0 = 0; e0 < entries; e0 += 64) {
    const int e = e0 + lane, n = e < entries ? count(e) : 0, o = e < entries ? other(e) : 0;
    const int incl = wave_incl_sum(n), oincl = wave_incl_sum(o);
    const unsigned long long hit = __ballot(base + incl > at);
    if (hit) {
      const int first = uniform(__ffsll(hit) - 1);
      base += __builtin_amdgcn_readlane(incl, first) - __builtin_amdgcn_readlane(n, first);
      before += __builtin_amdgcn_readlane(oincl, first) - __builtin_amdgcn_readlane(o, first);
      return e0 + first;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
    before += __builtin_amdgcn_readlane(oincl, 63);
  }
  return -1;
}

// A workgroup's number when those on one XCD (numbers 8 apart) are to be neighbours; the grid is a multiple of 8.
__device__ __forceinline__ int xcd_order() { return (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8); }

// stages of keys that the rows at positions p0 .. p1 see: those of the sinks in front of the window's, then the window's
struct KeyRange {
  int sink, first, n;                      // stages of sinks, the window's first, all
  __device__ __forceinline__ int at(int t) const { return t < sink ? t : t - sink + first; }
};
template <int KT>
__device__ __forceinline__ KeyRange keys_of(const WindowArgs& a, int p0, int p1) {
  KeyRange k{0, 0, 0};
  if (p1 < 0) return k;
  k.first = max(max(p0, 0) - a.window + 1, 0) / KT;
  k.sink = min((min(a.sinks, p1 + 1) + KT - 1) / KT, k.first);
  k.n = k.sink + p1 / KT + 1 - k.first;
  return k;
}

struct Row {
  int p, lo, sinks;                        // position, first key of the window, sinks
  __device__ __forceinline__ bool sees(int j) const { return j <= p && (j >= lo || j < sinks); }
};
__device__ __forceinline__ Row row_at(const WindowArgs& a, int p) { return Row{p, max(p, 0) - a.window + 1, a.sinks}; }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float at_least(float m) { return m == -INFINITY ? 0.f : m; }

// a stage is free and the next one there: this wave's copies are done, and its reads, and with the barrier everyone's
__device__ __forceinline__ void next_stage() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace window
#endif

}  // namespace sta
