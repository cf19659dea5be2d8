// sta_window.hip -- the forward pass of attention with a sliding window and sinks (sta_window.h).
//
// A workgroup takes 128 rows of one head (32 where there are few), a wave 32 of them, and walks the
// keys that they see in stages of 64 (fp32 and one wave: 32) through two LDS buffers, the next one copied while this one is worked on.
//
//   S^T = K Q^T     K rows of the stage as operand A, the wave's Q rows in registers as B; the result holds
//                   row l % 32, keys 8 (i / 4) + 4 (l / 32) + i % 4 in slot i of lane l
//   O^T += V^T P^T  those slots are, as they stand, contraction elements of operand B; operand A is read transposed
//                   from the stage's V rows (ds_read_b64_tr_b16), in the same order of keys
//
// so P never moves between lanes.  The running maximum and sum of a row are fp32, a lane pair's own; a maximum that rises
// by less than 2^8 leaves the sums as they are.  P is rounded once to 16 bits for the second product (its sum is of the
// unrounded one): an error of 2^-9 (fp16 2^-12) of each probability, which adds up at random over the keys to about
// what rounding the output itself costs.  Workgroups whose rows see up to FEW keys add the product with what the rounding left.
//
// Measured, products of the visible pairs alone: a prompt of 8192 tokens, 32 heads over 8 x 128, bf16, window 4096, 128 sinks:
// 421 GFLOP in 436 us, 965 TFLOP/s, 79% of what a product of two 8192^2 matrices reaches; the same heads, 5 packed
// sequences of together 8192, window 1024: 205 us, 500 TFLOP/s (short sequences and the two masked ends of each window weigh
// more); 24 heads x 64, fp16, 6001 tokens in 3 sequences, causal: 125 us, 380 TFLOP/s (twice the exponentials a
// product).  Bound by the matrix cores beside LDS reads of as many cycles and
// the exponentials: the cores are busy half of the time, LDS has no bank conflicts.  128 rows a workgroup: 64 rows a wave
// would halve those reads; they do not fit the registers at D 128, and are untried at D 64.  fp32, 2370 tokens, 16 heads over 2 x 128,
// causal: 23 GFLOP in 453 us, a third of its product rate: one wave a SIMD, whose products and exponentials take turns.
//
// A wave whose sums end as no finite numbers goes over its rows' keys one by one: 8192 tokens, 32 heads over 8 x 128, bf16, causal, a
// NaN in key 10 of every head: 0.69 -> 30 ms (the gradient 2.6 -> 53; window 1024: 0.22 -> 1.7 and 0.59 -> 3.6).
#include "sta_window.h"

namespace sta {

namespace {

using namespace window;

// Up to so many keys of a workgroup the second product takes P in two parts.  A backward pass' delta inherits the error of
// P, and beside ds' own rounding that weighs by the sum of p^2: 3 sequences of 2000 tokens, 24 heads x 64, fp16, causal, dq
// erred by 1.48 to 1.51 times what rounding it costs with two parts up to 256 keys, by 1.46 to 1.47 up to 1024 (114 -> 122 us; 5
// of together 8192, 32 heads over 8 x 128, bf16, window 1024: 192 -> 206).  One number with and without a backward pass
// to come, so that both give the same bits; with 256 a call without would take 125 us in place of 149 (8192 tokens, 32 heads
// over 8 x 128, bf16, window 512; window 1024: 187 and 191; a prompt of 1024: 30 and 36).
constexpr int FEW = 1024;

template <int DT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (Tile<DT, D, WAVES>::LEAST)) void window_kernel(WindowArgs a) {
  using T = Tile<DT, D, WAVES>;
  constexpr int KT = T::KT, SUB = T::SUB, ROWS = T::ROWS;
  __shared__ u32x4 lds[2][2][KT * T::CH];
  const int G = a.H / a.Hkv, lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), r = lane & 31, h4 = (lane >> 5) * 4;
  const int id = xcd_order(), hk = id / (a.q_tiles * G), rest = id - hk * (a.q_tiles * G);
  if (hk >= a.Hkv) return;
  // late tiles see more keys: first
  const int tile_all = a.q_tiles - 1 - rest / G, h = hk * G + rest % G;
  int base, none;
  const int e = find_entry(a.B + 2, tile_all, [&](int x) { return (entry_of(a.starts, x, a.B, a.T).n + ROWS - 1) / ROWS; },
                           [](int) { return 0; }, base, none);
  if (e < 0) return;
  const Span sq = uniform(entry_of(a.starts, e, a.B, a.T));
  const int row0 = (tile_all - base) * ROWS, row = row0 + wave * 32 + r;
  if (row0 < 0 || row0 >= sq.n) return;    // starts that do not ascend
  const bool real = row < sq.n;
  char* out = a.out + ((int64_t)(sq.at + row) * a.H + h) * T::RB;
  float* lse = a.lse + (int64_t)h * a.T + sq.at + row;
  floatx16 acc[T::DB];
  clear<T>(acc);
  if (e == 0 || e > a.B) {                 // rows of no sequence
    if (real) {
      store_rows<DT, T>(out, acc, 0.f);
      if (a.rest) store_rows<DT, T>(a.rest + (out - a.out), acc, 0.f);
      if (lane < 32) *lse = -INFINITY;
    }
    return;
  }
  const Span sk = uniform(span_of(a.k_starts, e - 1, a.S));
  const int off = sk.n - sq.n, p0 = off + row0, pw = p0 + wave * 32;
  const bool idle = row0 + wave * 32 >= sq.n;
  const KeyRange keys = keys_of<KT>(a, p0, min(p0 + ROWS, sk.n) - 1);
  const char* kb = a.k + sk.at * a.k_ts + hk * a.k_hs;
  const char* vb = a.v + sk.at * a.v_ts + hk * a.v_hs;
  const Row me = row_at(a, off + row);

  u32x4 q[T::KD];
  load_rows<T>(q, a.q + sq.at * a.q_ts + h * a.q_hs, a.q_ts, row, sq.n);
  signed_rows<DT>(q, a.flip, a.keep);
  // P times 2^shift: an fp16 P below 2^-14 of 2^8 would lose bits
  constexpr float SHIFT = DT == DT_F16 ? 7.f : 0.f, RISE = 8.f;
  float m = -INFINITY, l = 0.f;
  const Places at = places_of<DT, T>();
  Stager<T> ks, vs;
  ks.set(a.k_ts);
  vs.set(a.v_ts);
  auto fetch = [&](int t, int buf) STA_INLINE {
    ks.copy(lds[buf][0], kb, keys.at(t) * KT, sk.n);
    vs.copy(lds[buf][1], vb, keys.at(t) * KT, sk.n);
  };
  const bool few = keys.n * KT <= FEW;
  const int lo_first = max(pw, 0) - a.window + 1, lo_last = max(pw + 31, 0) - a.window + 1;
  auto turn = [&](int t, auto which) STA_INLINE {
    constexpr int BUF = decltype(which)::value;
    next_stage();
    if (t + 1 < keys.n) fetch(t + 1, 1 - BUF);
    const int k0 = keys.at(t) * KT, k1 = k0 + KT - 1;
    if (idle || k0 > pw + 31 || (k1 < lo_first && k0 >= a.sinks)) return;
    const lds_bytes kt = (lds_bytes)&lds[BUF][0][0], vt = (lds_bytes)&lds[BUF][1][0];
    floatx16 s[SUB];
#pragma unroll
    for (int y = 0; y < SUB; ++y) s[y] = rows_product<DT, T>(kt, at, y * 32, [&](int d) { return q[d]; });
#pragma unroll
    for (int y = 0; y < SUB; ++y) settle<DT>(s[y]);
    if (!(k1 <= pw && (k0 >= lo_last || k1 < a.sinks))) {
      const int key = rarely(k0 + h4);
#pragma unroll
      for (int y = 0; y < SUB; ++y)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!me.sees(key + y * 32 + 8 * (i / 4) + i % 4)) s[y][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int y = 0; y < SUB; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[y][i]);
    top = fmaxf(top, __shfl_xor(top, 32, 64)) * a.c;
    if (__any(top > m + RISE)) {
      const float m1 = fmaxf(m, top), f = exp2_of(m - at_least(m1));
      m = m1;
      l *= f;
#pragma unroll
      for (int b = 0; b < T::DB; ++b) acc[b] *= f;
    }
    const float m0 = at_least(m) - SHIFT;
#pragma unroll
    for (int y = 0; y < SUB; ++y) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[y][i] = exp2_of(fmaf(s[y][i], a.c, -m0));
        l += s[y][i];
      }
      Weights<DT> p;
      p.set(s[y]);
      transposed_product<DT, T>(vt, at, y * 32, p, acc);
      if constexpr (DT != DT_F32) {
        if (few) {
          p.rest(s[y]);
          transposed_product<DT, T>(vt, at, y * 32, p, acc);
        }
      }
    }
  };
  if (keys.n) fetch(0, 0);
  for (int t = 0; t < keys.n; t += 2) {
    turn(t, std::integral_constant<int, 0>());
    if (t + 1 < keys.n) turn(t + 1, std::integral_constant<int, 1>());
  }
  float unit = 1.f;                        // of the sums
  if (__builtin_expect(not_finite<T>(acc), 0)) {
    // p so small that no sum of up to 2^28 values exceeds the largest of them
    unit = 0x1p28f;
    clear<T>(acc);
    m = -INFINITY;
    l = 0.f;
    auto each_key = [&](auto f) STA_INLINE {
      for (int t = 0; t < keys.n; ++t) {
        const int k0 = keys.at(t) * KT, k1 = min(k0 + KT, sk.n);
        for (int j = k0; j < k1; ++j) {
          const float s = row_dot<DT, T>(kb + j * a.k_ts, [&](int d) { return q[d]; });
          f(j, me.sees(j) ? s : -INFINITY);
        }
      }
    };
    each_key([&](int, float s) { m = fmaxf(m, s * a.c); });
    const float m0 = at_least(m) - SHIFT;
    each_key([&](int j, float s) {
      const float p = exp2_of(fmaf(s, a.c, -m0));
      l += p;
      add_row<DT, T>(acc, vb + j * a.v_ts, p * 0x1p-28f, s != -INFINITY);
    });
    if (h4) l = 0.f;                       // both lanes of a row have all of it
  }
  l += __shfl_xor(l, 32, 64);
  if (!real) return;
  const float inv = l == 0.f ? 0.f : unit / l;
  store_rows<DT, T>(out, acc, inv);
  if constexpr (DT != DT_F32) {
    if (a.rest) store_rests<DT, T>(a.rest + (out - a.out), acc, inv);
  }
  if (lane < 32) *lse = l == 0.f ? -INFINITY : (at_least(m) - SHIFT + log2f(l)) * 0.693147180559945309f;
}

template <int DT, int D>
hipError_t launch_dt(const WindowArgs& a, hipStream_t st) {
  const unsigned grid = ((unsigned)a.q_tiles * a.H + 7) / 8 * 8;
  if (a.q_waves == 1) window_kernel<DT, D, 1><<<grid, 64, 0, st>>>(a);
  else window_kernel<DT, D, 4><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_window(int dtype, int D, const WindowArgs& a, hipStream_t st) {
  if (dtype == DT_F32) return D == 64 ? launch_dt<DT_F32, 64>(a, st) : launch_dt<DT_F32, 128>(a, st);
  if (dtype == DT_BF16) return D == 64 ? launch_dt<DT_BF16, 64>(a, st) : launch_dt<DT_BF16, 128>(a, st);
  return D == 64 ? launch_dt<DT_F16, 64>(a, st) : launch_dt<DT_F16, 128>(a, st);
}

}  // namespace sta
