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
  char* rest;                              // what rounding out left, in its type; NULL: not kept (forward) or none (backward)
  float* lse;                              // (H, T)
  const float* lse_in;
  // backward
  char *dq, *dk, *dv;
  float *row_lse, *row_delta;              // (H, T): log2 of the sum of exp, +inf for rows that see nothing; sum_d out dout
  float *row_norm, *key_norm;              // fp16: (H, T) |dout|^2 and (Hkv, S) |v|^2 of rows without infinities and NaN, 0 of others
  int delta_blocks;                        // workgroups of the pass over out and dout
  float* record;                           // (records, 2, rows of a key tile, D) unfinished dk and dv
  int steps;                               // row steps of a work item of the key pass
  int far_steps;                           // of one of a key tile with sinks
  int near_steps;                          // row steps that a key tile has at most, a query head
  int q_tiles, k_tiles, items;             // bounds of the grids, a head / kv head
  int q_waves, k_waves;                    // waves of a workgroup: 4, or 1 where there are few rows
};

// how the key pass is cut (host)
struct WindowCut {
  int q_waves, k_waves, q_tiles, k_tiles, items, steps, far_steps, near_steps, delta_blocks;
  int64_t records;
};
WindowCut window_cut(int dtype, int D, int T, int S, int H, int Hkv, int B, bool starts, bool k_starts, int window,
                     int sinks);

hipError_t launch_window(int dtype, int D, const WindowArgs& a, hipStream_t st);
hipError_t launch_window_grad(int dtype, int D, const WindowArgs& a, int64_t records, hipStream_t st);

#ifdef __HIPCC__
// a lambda that the compiler called instead would have its captured registers in memory
#define STA_INLINE __attribute__((always_inline))

namespace window {

// a workgroup's WAVES_ waves take 32 rows (keys in the key pass) each
template <int DT, int D_, int WAVES_>
struct Tile {
  static constexpr int WAVES = WAVES_, THREADS = 64 * WAVES, ROWS = 32 * WAVES;
  static constexpr int D = D_, E = DT == DT_F32 ? 4 : 2, RB = D * E, CH = RB / 16;
  static constexpr int KD = RB / 32;       // products over a row: 32 bytes of it each, 16 a half wave
  static constexpr int DB = D / 32;        // blocks of 32 dims
  static constexpr int LEAST = DT == DT_F32 || WAVES == 1 ? 1 : 2;    // waves of a SIMD that the registers have to allow
  // rows of a stage; one wave: room for four workgroups a CU, but for fp32 at D 128, whose 65 KB leave room for two
  static constexpr int KT = DT == DT_F32 || WAVES == 1 ? 32 : 64;
  static constexpr int SUB = KT / 32;
  static constexpr int COPIES = KT * CH / THREADS;    // a wave's 1 KB copies of a stage's rows
};

// Rows lie in LDS as they are, their 16-byte chunks permuted by the row: chunk c of row r at c ^ swz(r).  Both reads then
// spread over the banks: 16 rows' equal chunks (a row an operand lane), and for the transposing reads (16-bit) 64
// bytes of 8 rows, for fp32 128 bytes of two rows 4 apart.
template <typename T>
__device__ constexpr __forceinline__ int swz(int r) {
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

// Copies from global memory into LDS, lane l's bytes at lds_base + 16 l (4 l), as copy16_to_lds of sta_device.h.  Inline
// assembly is no memory instruction to the compiler, which keeps no distance between it and the instructions that
// write its scalar operands: an address in scalar registers that a vector instruction (readfirstlane) wrote may be
// read 5 wait states later at the earliest, M0 one.  So the copies wait for themselves.
__device__ __forceinline__ void stage16(const void* sbase, uint32_t voff, uint32_t lds_base) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_base) : "memory");
}
__device__ __forceinline__ void stage16(const void* gsrc, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(gsrc), "{m0}"(lds_base) : "memory");
}
__device__ __forceinline__ void stage4(const void* gsrc, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(gsrc), "{m0}"(lds_base) : "memory");
}

// Rows row0 .. row0 + KT - 1 of a sequence into a stage, this wave's share; rows from n on are zeros.  swz is linear over xor, so
// that a copy's chunks differ from the lane's own by a uniform xor.
template <typename T>
struct Stager {
  int64_t stride;
  uint32_t row, chunk;                     // the lane's place in a copy: bytes of its row's offset and of its chunk
  __device__ __forceinline__ void set(int64_t row_stride) {
    const int lane = threadIdx.x & 63;
    stride = row_stride;
    row = (uint32_t)(lane / T::CH) * (uint32_t)row_stride;
    chunk = (uint32_t)((lane % T::CH) ^ swz<T>(lane / T::CH)) * 16;
  }
  __device__ __forceinline__ void copy(const u32x4* to, const char* base, int row0, int n) const {
    constexpr int PER = 64 / T::CH;        // rows of a copy
    const int wave = uniform((int)threadIdx.x >> 6), first = wave * (T::COPIES * PER);
    const uint32_t lds = (uint32_t)uniform((int)lds_addr(to)) + (uint32_t)wave * (T::COPIES * 1024);
    if (row0 + T::KT <= n) {
      const char* from = base + (row0 + first) * stride;
#pragma unroll
      for (int y = 0; y < T::COPIES; ++y)
        stage16(from + (y * PER) * stride, row + (chunk ^ (uint32_t)((swz<T>(first) ^ swz<T>(y * PER)) * 16)), lds + y * 1024);
    } else {
      asm volatile("" ::: "memory");
      const int lane = threadIdx.x & 63;
#pragma unroll
      for (int y = 0; y < T::COPIES; ++y) {
        const int r = first + y * PER + lane / T::CH;
        const char* p = row0 + r < n ? base + (row0 + r) * stride : (const char*)zero_row;
        stage16(p + ((lane % T::CH) ^ swz<T>(r)) * 16, lds + y * 1024);
      }
    }
  }
};

// Where a lane reads in a stage: (r RB + swz(r) 16) ^ (c 16) is chunk c of row r, since a row is a multiple of the chunks' bits.
typedef const __attribute__((address_space(3))) char* lds_bytes;
struct Places {
  uint32_t row;                            // row l % 32, chunk l / 32
  uint32_t column;                         // transposing reads: row 4 (l / 32) + l % 16 / 4; fp32: row 4 (l / 32), dim l % 32
};
template <int DT, typename T>
__device__ __forceinline__ Places places_of() {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  Places p;
  p.row = (uint32_t)(r * T::RB + swz<T>(r) * 16) ^ (uint32_t)(h * 16);
  if constexpr (DT == DT_F32) {
    p.column = (uint32_t)(4 * h * T::RB + swz<T>(4 * h) * 16) ^ (uint32_t)(r * 4);
  } else {
    const int r4 = 4 * h + (lane & 15) / 4;
    p.column = ((uint32_t)(r4 * T::RB + swz<T>(r4) * 16) ^ (uint32_t)((lane >> 4 & 1) * 32 + (lane & 2) * 8)) + (lane & 1) * 8;
  }
  return p;
}

// scores: 32 rows of a stage from row0 (operand A) times the wave's 32 rows in registers (operand B).  Slot i of lane l is
// stage row row0 + 8 (i / 4) + 4 (l / 32) + i % 4, own row l % 32.
// own(d): 32 bytes d of the own rows.
template <int DT, typename T, typename Own>
__device__ __forceinline__ floatx16 rows_product(lds_bytes lds, const Places& at, int row0, Own own) {
  floatx16 x;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
  for (int d = 0; d < T::KD; ++d) {
    const u32x4 w = *(const __attribute__((address_space(3))) u32x4*)(lds + (at.row ^ (uint32_t)(d * 32)) + row0 * T::RB);
    x = mma<DT>(w, own(d), x);
  }
  return x;
}

// settle_mfma32 of sta_device.h; the fp32 products take 16 passes, 18 wait states
template <int DT>
__device__ __forceinline__ void settle(floatx16& x) {
  if constexpr (DT == DT_F32) {
    float last = x[15];
    asm volatile("s_nop 15\n\ts_nop 1" : "+v"(last));
    x[15] = last;
  } else {
    settle_mfma32(x);
  }
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
  // what set left of x
  __device__ __forceinline__ void rest(const floatx16& x) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u = w[s][e];
        const float lo = DT == DT_F16 ? f16_bits_to_f32(u & 0xffffu) : __uint_as_float(u << 16);
        const float hi = DT == DT_F16 ? f16_bits_to_f32(u >> 16) : __uint_as_float(u & 0xffff0000u);
        w[s][e] = pack2_dt<DT>(x[8 * s + 2 * e] - lo, x[8 * s + 2 * e + 1] - hi);
      }
  }
};
template <>
struct Weights<DT_F32> {
  floatx16 w;
  __device__ __forceinline__ void set(const floatx16& x) { w = x; }
};

// acc (dims x own rows) += (32 rows of a stage from row0)^T x weights
template <int DT, typename T>
__device__ __forceinline__ void transposed_product(lds_bytes lds, const Places& at, int row0, const Weights<DT>& p,
                                                   floatx16 (&acc)[T::DB]) {
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      constexpr int RB = T::RB;
      const int r = 8 * (i / 4) + i % 4;   // 4 (l / 32) is in the place
#pragma unroll
      for (int b = 0; b < T::DB; ++b) {
        const uint32_t x = at.column ^ (uint32_t)(b * 128) ^ (uint32_t)(swz<T>(r) * 16);
        const float w = *(const __attribute__((address_space(3))) float*)(lds + x + (row0 + r) * RB);
        acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(w, p.w[i], acc[b], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int b = 0; b < T::DB; ++b) {
        u32x4 a;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t x = at.column ^ (uint32_t)(b * 64 ^ swz<T>(8 * y) * 16);
          const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(lds + x + (row0 + 16 * s + 8 * y) * T::RB));
          const u32x2 v = __builtin_bit_cast(u32x2, w);
          a[2 * y] = v[0], a[2 * y + 1] = v[1];
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

// what rounding dims x own rows times scale to 16 bits left, rounded to them
template <int DT, typename T>
__device__ __forceinline__ void store_rests(char* row, const floatx16 (&acc)[T::DB], float scale) {
  const int h = (threadIdx.x & 63) >> 5;
  auto rest = [&](float x) {
    if constexpr (DT == DT_F16) return x - f16_bits_to_f32(f32_to_f16_bits(x));
    else return x - bf16_bits_to_f32(f32_to_bf16_bits(x));
  };
#pragma unroll
  for (int b = 0; b < T::DB; ++b)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = rest(acc[b][4 * s + i] * scale);
      *(u32x2*)(row + (b * 32 + s * 8 + h * 4) * 2) = u32x2{pack2_dt<DT>(x[0], x[1]), pack2_dt<DT>(x[2], x[3])};
    }
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
// Sums that are no finite numbers.  A product over a stage multiplies what a row does not see by a p of 0, and 0 times an
// infinity or a NaN would reach it; sums of large values may also have passed the type's largest on the way.  A wave whose
// sums end so forms them again, row by row, of what each of its rows sees.
// ------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ bool not_finite(const floatx16 (&acc)[T::DB]) {
  float zero = 0.f;                        // an infinity or a NaN times 0 is NaN
#pragma unroll
  for (int b = 0; b < T::DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) zero = fmaf(acc[b][i], 0.f, zero);
  return __any(zero != 0.f);
}

// a row in memory, the same for the whole wave, times the lane's own (own(d): 32 bytes d of it)
template <int DT, typename T, typename Own>
__device__ __forceinline__ float row_dot(const char* row, Own own) {
  const int h = (threadIdx.x & 63) >> 5;
  float sum = 0.f;
#pragma unroll
  for (int d = 0; d < T::KD; ++d) {
    const u32x4 x = *(const u32x4*)(row + (2 * d + h) * 16), y = own(d);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == DT_F32) {
        sum = fmaf(__uint_as_float(x[e]), __uint_as_float(y[e]), sum);
      } else if constexpr (DT == DT_BF16) {
        sum = fmaf(__uint_as_float(x[e] << 16), __uint_as_float(y[e] << 16), sum);
        sum = fmaf(__uint_as_float(x[e] & 0xffff0000u), __uint_as_float(y[e] & 0xffff0000u), sum);
      } else {
        sum = fmaf(f16_bits_to_f32(x[e] & 0xffffu), f16_bits_to_f32(y[e] & 0xffffu), sum);
        sum = fmaf(f16_bits_to_f32(x[e] >> 16), f16_bits_to_f32(y[e] >> 16), sum);
      }
    }
  }
  return sum + __shfl_xor(sum, 32, 64);
}

// acc (dims x own rows) += weight x a row in memory, for lanes that see it
template <int DT, typename T>
__device__ __forceinline__ void add_row(floatx16 (&acc)[T::DB], const char* row, float weight, bool sees) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int b = 0; b < T::DB; ++b)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int dim = b * 32 + s * 8 + h * 4;
      float x[4];
      if constexpr (DT == DT_F32) {
        const float4 w = *(const float4*)(row + dim * 4);
        x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
      } else {
        const u32x2 w = *(const u32x2*)(row + dim * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
          x[i] = DT == DT_F16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (sees) acc[b][4 * s + i] = fmaf(weight, x[i], acc[b][4 * s + i]);
    }
}

template <typename T>
__device__ __forceinline__ void clear(floatx16 (&acc)[T::DB]) {
#pragma unroll
  for (int b = 0; b < T::DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
}

// ------------------------------------------------------------------------------------------
// sequences
// ------------------------------------------------------------------------------------------
struct Span {
  int at, n;                               // first row among the packed ones, rows
};
__device__ __forceinline__ Span uniform(Span s) { return Span{uniform(s.at), uniform(s.n)}; }
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
      base = uniform(base + __builtin_amdgcn_readlane(incl, first) - __builtin_amdgcn_readlane(n, first));
      before = uniform(before + __builtin_amdgcn_readlane(oincl, first) - __builtin_amdgcn_readlane(o, first));
      return uniform(e0 + first);
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

// x y, and 0 where either is 0, whatever the other holds (v_mul_legacy_f32)
extern "C" __device__ __attribute__((const)) float sta_mul_zero(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float mul_zero(float x, float y) { return sta_mul_zero(x, y); }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float at_least(float m) { return m == -INFINITY ? 0.f : m; }

// x in a branch of its own: compares and selects on a condition that is rarely true would be formed in every turn
__device__ __forceinline__ int rarely(int x) {
  asm volatile("" : "+v"(x)::"memory");
  return x;
}

// a stage is free and the next one there: this wave's copies are done, and its reads, and with the barrier everyone's
__device__ __forceinline__ void next_stage() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace window
#endif

}  // namespace sta
