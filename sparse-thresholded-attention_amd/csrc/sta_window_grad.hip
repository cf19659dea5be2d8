// sta_window_grad.hip -- the backward pass of attention with a sliding window and sinks (sta_window.h).
//
//   dv_j = sum_i p_ij dout_i,  dp_ij = dout_i . v_j,  ds_ij = p_ij (dp_ij - delta_i),  delta_i = out_i . dout_i,
//   dq_i = sm_scale sum_j ds_ij k_j,  dk_j = sm_scale sum_i ds_ij q_i
//
// with p formed again from the scores and the row's log-sum-exp.  Two passes without atomics, so that sums have one
// order: one over the keys of 128 rows for dq (three products a pair), one over the rows of 128 keys for dk and dv
// (four), the heads of a kv head one after the other.  Both keep the layouts of the forward pass: the 128 rows or
// keys in registers as operand B, the others in stages through LDS, read as they lie for the scores and dp, and
// transposed for the sums.  p and ds are rounded once to 16 bits for those, as p is in the forward pass.
//
// Measured: 5 packed sequences of together 8192, 32 heads over 8 x 128, bf16, window 1024, 4 sinks: delta 39 us (201 MB,
// 5.1 TB/s), dq 216 (155 GFLOP, 710 TFLOP/s), dk and dv 387 (207 GFLOP, 530 TFLOP/s, 44% of a large product), the join 22;
// 24 heads x 64, fp16, 3 sequences of together 6001, causal: 16 / 141 / 193 us.  The key pass is bound by its registers: two
// sums of 128 dims and the keys' own k and v leave two waves a SIMD, and every stage is read four times from LDS.  Its
// 70 or so items a kv head run on 64 places, one of them nearly twice: shares of one length would save at most a fifth
// and leave records of nearly every tile, whose 134 MB cost about as much to write and read.
#include "sta_window.h"

namespace sta {

namespace {

using namespace window;

// An fp16 ds would pass the type's range: it is scaled by a power of two that keeps |ds| <= p (|dout| |v| + |delta|) below
// 2^14.  dq's are a row's own, from the largest v that its workgroup's rows see; the key pass takes one for the rows and
// keys of a work item.  So large values of other sequences, heads and far places cost a row or a key no bits.
__device__ __forceinline__ float grow_of(float most) {
  if (!(most > 0.f && most < INFINITY)) return 1.f;
  return __uint_as_float((uint32_t)(127 + min(max(13 - ilogbf(most), -100), 100)) << 23);
}

// the largest x of a workgroup's threads, in all of them
template <int WAVES>
__device__ __forceinline__ float group_max(float x, float* shared) {
  x = wave_max_f32(x);
  if constexpr (WAVES > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) x = fmaxf(x, shared[w]);
  }
  return x;
}

// every row of a sequence of n keys sees one key
__device__ __forceinline__ bool only_own(const WindowArgs& a, int n) { return n == 1 || (a.window == 1 && a.sinks == 0); }

// delta and the base-2 log of the sum, +inf for rows that see nothing (their p is 0 then); CH lanes a row.  delta of the rounded
// out would be off by about what rounding a ds costs: with what that rounding left (rest) dq and dk err 1.41 times what
// rounding them costs, without it 1.5 (bf16) to 1.6 times (fp16).
template <int DT, int D>
__global__ __launch_bounds__(256) void window_delta_kernel(WindowArgs a) {
  using T = Tile<DT, D, 4>;
  constexpr int V = 16 / T::E, PER = 256 / T::CH;
  const int c = threadIdx.x % T::CH, mine = threadIdx.x / T::CH;
  auto elements = [](const char* p, float* x) {
    const u32x4 w = *(const u32x4*)p;
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    } else {
      Raw8<DT> raw;
      raw.w = w;
      raw.to_f32(x);
    }
  };
  auto row_sum = [](float x) {
#pragma unroll
    for (int s = 1; s < T::CH; s *= 2) x += __shfl_xor(x, s, 64);
    return x;
  };
  const int64_t rows = (int64_t)a.T * a.H;
  // the scale's: without rows that hold an infinity or a NaN
  auto square = [](float sq) { return sq < INFINITY ? sq : 0.f; };
  for (int64_t i = (int64_t)blockIdx.x * PER + mine; i < rows; i += (int64_t)gridDim.x * PER) {
    const int64_t t = i / a.H;
    const int h = (int)(i - t * a.H);
    float x[V], y[V];
    elements(a.out + i * T::RB + c * 16, x);
    elements(a.dout + t * a.do_ts + h * a.do_hs + c * 16, y);
    if (DT != DT_F32 && a.rest) {
      float z[V];
      elements(a.rest + i * T::RB + c * 16, z);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] += z[e];
    }
    float dot = 0.f, sq = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      dot = fmaf(x[e], y[e], dot);
      sq = fmaf(y[e], y[e], sq);
    }
    dot = row_sum(dot);
    if constexpr (DT == DT_F16) sq = square(row_sum(sq));
    if (c == 0) {
      const float lse = a.lse_in[h * (int64_t)a.T + t];
      a.row_lse[h * (int64_t)a.T + t] = lse == -INFINITY ? INFINITY : lse * 1.44269504088896340736f;
      a.row_delta[h * (int64_t)a.T + t] = dot;
      if constexpr (DT == DT_F16) a.row_norm[h * (int64_t)a.T + t] = sq;
    }
  }
  if constexpr (DT == DT_F16) {
    const int64_t keys = (int64_t)a.S * a.Hkv;
    for (int64_t i = (int64_t)blockIdx.x * PER + mine; i < keys; i += (int64_t)gridDim.x * PER) {
      const int64_t t = i / a.Hkv, hk = i - t * a.Hkv;
      float x[V], sq = 0.f;
      elements(a.v + t * a.v_ts + hk * a.v_hs + c * 16, x);
#pragma unroll
      for (int e = 0; e < V; ++e) sq = fmaf(x[e], x[e], sq);
      sq = square(row_sum(sq));
      if (c == 0) a.key_norm[hk * a.S + t] = sq;
    }
  }
}

// ------------------------------------------------------------------------------------------
// dq: the forward pass' walk
// ------------------------------------------------------------------------------------------
template <int DT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (Tile<DT, D, WAVES>::LEAST)) void window_dq_kernel(WindowArgs a) {
  using T = Tile<DT, D, WAVES>;
  constexpr int KT = T::KT, SUB = T::SUB, ROWS = T::ROWS;
  __shared__ u32x4 lds[2][2][KT * T::CH];
  __shared__ float shared[4];
  const int G = a.H / a.Hkv, lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), r = lane & 31, h4 = (lane >> 5) * 4;
  const int id = xcd_order(), hk = id / (a.q_tiles * G), rest = id - hk * (a.q_tiles * G);
  if (hk >= a.Hkv) return;
  const int tile_all = a.q_tiles - 1 - rest / G, h = hk * G + rest % G;
  int base, none;
  const int e = find_entry(a.B + 2, tile_all, [&](int x) { return (entry_of(a.starts, x, a.B, a.T).n + ROWS - 1) / ROWS; },
                           [](int) { return 0; }, base, none);
  if (e < 0) return;
  const Span sq = uniform(entry_of(a.starts, e, a.B, a.T));
  const int row0 = (tile_all - base) * ROWS, row = row0 + wave * 32 + r;
  if (row0 < 0 || row0 >= sq.n) return;    // starts that do not ascend
  const bool real = row < sq.n;
  char* dq = a.dq + ((int64_t)(sq.at + row) * a.H + h) * T::RB;
  floatx16 acc[T::DB];
  clear<T>(acc);
  if (e == 0 || e > a.B) {
    if (real) store_rows<DT, T>(dq, acc, 0.f);
    return;
  }
  const Span sk = uniform(span_of(a.k_starts, e - 1, a.S));
  const int off = sk.n - sq.n, p0 = off + row0, pw = p0 + wave * 32;
  const bool idle = row0 + wave * 32 >= sq.n;
  const KeyRange keys = keys_of<KT>(a, p0, min(p0 + ROWS, sk.n) - 1);
  const char* kb = a.k + sk.at * a.k_ts + hk * a.k_hs;
  const char* vb = a.v + sk.at * a.v_ts + hk * a.v_hs;
  const Row me = row_at(a, off + row);

  u32x4 q[T::KD], dout[T::KD];
  load_rows<T>(q, a.q + sq.at * a.q_ts + h * a.q_hs, a.q_ts, row, sq.n);
  signed_rows<DT>(q, a.flip, a.keep);
  load_rows<T>(dout, a.dout + sq.at * a.do_ts + h * a.do_hs, a.do_ts, row, sq.n);
  const int64_t stat = (int64_t)h * a.T + sq.at + min(row, sq.n - 1);
  const float lse = a.row_lse[stat], delta = a.row_delta[stat];
  float grow = 1.f;
  if constexpr (DT == DT_F16) {
    float v2 = 0.f;
    const float* norms = a.key_norm + (int64_t)hk * a.S + sk.at;
#pragma unroll 4
    for (int i = threadIdx.x; i < keys.n * KT; i += T::THREADS) {
      const int key = keys.at(i / KT) * KT + i % KT;
      if (key < sk.n) v2 = fmaxf(v2, norms[key]);
    }
    grow = grow_of(sqrtf(a.row_norm[stat]) * sqrtf(group_max<WAVES>(v2, shared)) + fabsf(delta));
  }
  const Places at = places_of<DT, T>();
  Stager<T> ks, vs;
  ks.set(a.k_ts);
  vs.set(a.v_ts);
  auto fetch = [&](int t, int buf) STA_INLINE {
    ks.copy(lds[buf][0], kb, keys.at(t) * KT, sk.n);
    vs.copy(lds[buf][1], vb, keys.at(t) * KT, sk.n);
  };
  const int lo_first = max(pw, 0) - a.window + 1, lo_last = max(pw + 31, 0) - a.window + 1;
  auto turn = [&](int t, auto which) STA_INLINE {
    constexpr int BUF = decltype(which)::value;
    next_stage();
    if (t + 1 < keys.n) fetch(t + 1, 1 - BUF);
    const int k0 = keys.at(t) * KT, k1 = k0 + KT - 1;
    if (idle || k0 > pw + 31 || (k1 < lo_first && k0 >= a.sinks)) return;
    const bool some = !(k1 <= pw && (k0 >= lo_last || k1 < a.sinks));
    const lds_bytes kt = (lds_bytes)&lds[BUF][0][0], vt = (lds_bytes)&lds[BUF][1][0];
#pragma unroll
    for (int y = 0; y < SUB; ++y) {
      floatx16 s = rows_product<DT, T>(kt, at, y * 32, [&](int d) { return q[d]; });
      const floatx16 dp = rows_product<DT, T>(vt, at, y * 32, [&](int d) { return dout[d]; });
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = exp2_of(fmaf(s[i], a.c, -lse));
        s[i] = DT == DT_F16 ? p * (dp[i] - delta) * grow : p * (dp[i] - delta);
      }
      if (some) {
        const int key = rarely(k0 + y * 32 + h4);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!me.sees(key + 8 * (i / 4) + i % 4)) s[i] = 0.f;
      }
      Weights<DT> ds;
      ds.set(s);
      transposed_product<DT, T>(kt, at, y * 32, ds, acc);
    }
  };
  if (keys.n) fetch(0, 0);
  for (int t = 0; t < keys.n; t += 2) {
    turn(t, std::integral_constant<int, 0>());
    if (t + 1 < keys.n) turn(t + 1, std::integral_constant<int, 1>());
  }
  if (__builtin_expect(not_finite<T>(acc), 0)) {
    clear<T>(acc);
    for (int t = 0; t < keys.n; ++t) {
      const int k0 = keys.at(t) * KT, k1 = min(k0 + KT, sk.n);
      for (int j = k0; j < k1; ++j) {
        const float s = row_dot<DT, T>(kb + j * a.k_ts, [&](int d) { return q[d]; });
        const float dp = row_dot<DT, T>(vb + j * a.v_ts, [&](int d) { return dout[d]; });
        add_row<DT, T>(acc, kb + j * a.k_ts, exp2_of(fmaf(s, a.c, -lse)) * (dp - delta) * grow, me.sees(j));
      }
    }
  }
  // a row that sees its own key alone has p 1 whatever q is: dp - delta, the same number summed in two ways, is 0
  if (real) store_rows<DT, T>(dq, acc, me.p == 0 || only_own(a, sk.n) ? 0.f : a.scale / grow);
}

// ------------------------------------------------------------------------------------------
// dk, dv
// ------------------------------------------------------------------------------------------
// A work item is a key tile and up to a.steps of its row steps (the heads of the kv head one after the other), of a tile
// with sinks, which every later row sees, up to a.far_steps.  A tile whose rows take one item is written out; else each
// item leaves a record and the join adds them up in order: tiles with sinks, and all tiles where there are too few for
// the chip.
struct Cut {
  int tiles, sink_tiles, near, far;        // key tiles, those with sinks, items of a near tile and of one with sinks
  __device__ __forceinline__ int items() const { return (tiles - sink_tiles) * near + sink_tiles * far; }
  __device__ __forceinline__ int records() const {
    return (near > 1 ? (tiles - sink_tiles) * near : 0) + (far > 1 ? sink_tiles * far : 0);
  }
};
template <typename T>
__device__ __forceinline__ Cut cut_of(const WindowArgs& a, int e) {
  constexpr int KT = T::KT, ROWS = T::ROWS;
  const Span sk = entry_of(a.k_starts, e, a.B, a.S);
  Cut c{(sk.n + ROWS - 1) / ROWS, 0, 1, 1};
  if (e == 0 || e > a.B) return c;
  const int steps = (span_of(a.starts, e - 1, a.T).n + KT - 1) / KT, G = a.H / a.Hkv;
  c.near = max((int)(((int64_t)G * min(steps, a.near_steps) + a.steps - 1) / a.steps), 1);
  c.far = max((int)(((int64_t)G * steps + a.far_steps - 1) / a.far_steps), 1);
  if (a.window != INT32_MAX) c.sink_tiles = min((a.sinks + ROWS - 1) / ROWS, c.tiles);
  return c;
}
// an item's tile, its place among the tile's items, and the tile's first record (< 0: none)
struct Item {
  int entry, tile, part, parts, steps;     // steps: of an item of the tile, at most
  int64_t record;
};
template <typename T>
__device__ __forceinline__ Item item_of(const WindowArgs& a, int at, bool by_tile, int64_t records) {
  int base, before;
  Item it;
  it.entry = find_entry(a.B + 2, at, [&](int x) { const Cut c = cut_of<T>(a, x); return by_tile ? c.tiles : c.items(); },
                        [&](int x) { return cut_of<T>(a, x).records(); }, base, before);
  if (it.entry < 0) return it;
  const Cut c = cut_of<T>(a, it.entry);
  int x = at - base;
  if (by_tile) {
    it.tile = x;
    it.part = 0;
  } else if (x < c.sink_tiles * c.far) {
    it.tile = x / c.far;
    it.part = x - it.tile * c.far;
  } else {
    x -= c.sink_tiles * c.far;
    it.tile = c.sink_tiles + x / c.near;
    it.part = x % c.near;
  }
  if (it.tile >= c.tiles || x < 0) it.entry = -1;      // starts that do not ascend
  const bool sink = it.tile < c.sink_tiles;
  it.parts = sink ? c.far : c.near;
  it.steps = sink ? a.far_steps : a.steps;
  it.record = it.parts == 1 ? -1 : before + (sink ? (int64_t)it.tile * c.far
                                                  : (int64_t)(c.far > 1 ? c.sink_tiles * c.far : 0) + (int64_t)(it.tile - c.sink_tiles) * c.near);
  if (it.record + it.parts > records || it.record < -1) it.entry = -1;
  it.entry = uniform(it.entry);
  it.tile = uniform(it.tile);
  it.part = uniform(it.part);
  it.parts = uniform(it.parts);
  it.steps = uniform(it.steps);
  return it;
}

template <int DT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (Tile<DT, D, WAVES>::LEAST)) void window_dkv_kernel(WindowArgs a, int64_t records) {
  using T = Tile<DT, D, WAVES>;
  constexpr int KT = T::KT, SUB = T::SUB, ROWS = T::ROWS;
  __shared__ u32x4 lds[2][2][KT * T::CH];
  __shared__ floatx4 stats[2][2][KT / 4];
  __shared__ float shared[4];
  // parts of v that the registers do not hold beside two sums of 128 dims
  constexpr int PARK = DT != DT_F32 && D == 128 ? 3 : 0;
  __shared__ u32x4 parked[PARK ? WAVES * PARK : 1][64];
  const int G = a.H / a.Hkv, lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
  const int id = xcd_order(), hk = id / a.items;
  if (hk >= a.Hkv) return;
  const Item it = item_of<T>(a, id - hk * a.items, false, records);
  if (it.entry < 0) return;
  const Span sk = uniform(entry_of(a.k_starts, it.entry, a.B, a.S));
  const int key0 = it.tile * ROWS, kw = key0 + wave * 32, key = kw + r;
  floatx16 dk[T::DB], dv[T::DB];
  clear<T>(dk);
  clear<T>(dv);
  auto store = [&](float dk_scale, float dv_scale) STA_INLINE {
    if (key >= sk.n) return;
    const int64_t at = (int64_t)(sk.at + key) * a.Hkv + hk;
    store_rows<DT, T>(a.dk + at * T::RB, dk, dk_scale);
    store_rows<DT, T>(a.dv + at * T::RB, dv, dv_scale);
  };
  if (it.entry == 0 || it.entry > a.B) return store(0.f, 0.f);
  // rows in front of the first key see nothing and are left out
  Span sq = uniform(span_of(a.starts, it.entry - 1, a.T));
  const int blind = max(sq.n - sk.n, 0);
  sq = Span{sq.at + blind, sq.n - blind};
  const int off = sk.n - sq.n;
  // the rows that see any of the tile's keys, in steps of KT
  const int key1 = min(key0 + ROWS, sk.n) - 1;
  const bool sink = key0 < a.sinks || a.window == INT32_MAX;
  const int last = sink ? sq.n : (int)min((int64_t)sq.n, max((int64_t)key1 + a.window - off, (int64_t)0));
  const int first = max(key0 - off, 0) / KT;
  const int each = max((last + KT - 1) / KT - first, 0);
  const int s0 = (int)min((int64_t)it.part * it.steps, (int64_t)each * G), s1 = (int)min((int64_t)s0 + it.steps, (int64_t)each * G);
  float grow = 1.f;
  if constexpr (DT == DT_F16) {
    float do2 = 0.f, delta = 0.f;
    for (int s = s0; s < s1;) {            // the item's rows, a head after the other
      const int g = s / each, in = s - g * each, end = min(each, in + s1 - s);
      const int64_t head = (int64_t)(hk * G + g) * a.T + sq.at;
      const int row1 = min((first + end) * KT, sq.n);
#pragma unroll 4
      for (int row = (first + in) * KT + (int)threadIdx.x; row < row1; row += T::THREADS) {
        do2 = fmaxf(do2, a.row_norm[head + row]);
        const float x = fabsf(a.row_delta[head + row]);
        if (x < INFINITY) delta = fmaxf(delta, x);
      }
      s += end - in;
    }
    const float v2 = key < sk.n ? a.key_norm[(int64_t)hk * a.S + sk.at + key] : 0.f;
    do2 = group_max<WAVES>(do2, shared);
    delta = group_max<WAVES>(delta, shared);
    grow = grow_of(sqrtf(do2) * sqrtf(group_max<WAVES>(v2, shared)) + delta);
    grow = __uint_as_float((uint32_t)uniform((int)__float_as_uint(grow)));
  }
  constexpr float SHIFT = DT == DT_F16 ? 15.f : 0.f;   // p times 2^15: fp16 keeps small ones

  u32x4 k[T::KD], v[T::KD];
  load_rows<T>(k, a.k + sk.at * a.k_ts + hk * a.k_hs, a.k_ts, key, sk.n);
  signed_rows<DT>(k, a.flip, a.keep);
  load_rows<T>(v, a.v + sk.at * a.v_ts + hk * a.v_hs, a.v_ts, key, sk.n);
#pragma unroll
  for (int d = 0; d < PARK; ++d) parked[wave * PARK + d][lane] = v[d];
  Places place = places_of<DT, T>();
  Stager<T> qs, ds;
  qs.set(a.q_ts);
  ds.set(a.do_ts);
  auto fetch = [&](int s, int buf) STA_INLINE {
    const int g = s / each, row0 = (first + s - g * each) * KT, head = hk * G + g;
    // the places' xors are formed anew every turn: kept over the loop they and parts of k or v would be spilled
    asm volatile("" : "+v"(place.row), "+v"(place.column), "+v"(qs.chunk));
    ds.chunk = qs.chunk;
    qs.copy(lds[buf][0], a.q + sq.at * a.q_ts + head * a.q_hs, row0, sq.n);
    ds.copy(lds[buf][1], a.dout + sq.at * a.do_ts + head * a.do_hs, row0, sq.n);
    if (lane < KT) {                       // past the last row its own again
      const int64_t row = (int64_t)head * a.T + sq.at + min(row0 + lane, sq.n - 1);
      if (wave == 0) stage4(a.row_lse + row, uniform((int)lds_addr(&stats[buf][0][0])));
      if (wave == WAVES / 2) stage4(a.row_delta + row, uniform((int)lds_addr(&stats[buf][1][0])));
    }
  };
  auto turn = [&](int s, auto which) STA_INLINE {
    constexpr int BUF = decltype(which)::value;
    next_stage();
    if (s + 1 < s1) fetch(s + 1, 1 - BUF);
    const int row0 = (first + s % each) * KT;
    const lds_bytes qt = (lds_bytes)&lds[BUF][0][0], dt = (lds_bytes)&lds[BUF][1][0];
#pragma unroll
    for (int y = 0; y < SUB; ++y) {
      const int rw = row0 + y * 32, p0 = rw + off, p1 = p0 + 31;
      const int lo0 = max(p0, 0) - a.window + 1, lo1 = max(p1, 0) - a.window + 1;
      if (p1 < kw || (lo0 > kw + 31 && kw >= a.sinks)) continue;
      floatx16 x = rows_product<DT, T>(qt, place, y * 32, [&](int d) { return k[d]; });
      settle<DT>(x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float lse = SHIFT - stats[BUF][0][y * 8 + 2 * (i / 4) + h][i % 4];
        x[i] = exp2_of(fmaf(x[i], a.c, lse));
      }
      if (!(p0 >= kw + 31 && (lo1 <= kw || kw + 31 < a.sinks) && rw + 31 < sq.n)) {
        const int row_h = rarely(rw + 4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = row_h + 8 * (i / 4) + i % 4;
          if (!row_at(a, row + off).sees(key) || row >= sq.n) x[i] = 0.f;
        }
      }
      Weights<DT> p;
      p.set(x);
      transposed_product<DT, T>(dt, place, y * 32, p, dv);
      const floatx16 dp = rows_product<DT, T>(dt, place, y * 32, [&](int d) { return d < PARK ? parked[wave * PARK + d][lane] : v[d]; });
      const float down = grow * (1.f / 32768.f);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float delta = stats[BUF][1][y * 8 + 2 * (i / 4) + h][i % 4];
        // a product in which 0 times anything is 0: a row that sees a bad key has a delta that is no number, and
        // the keys that it does not see would get it
        x[i] = mul_zero(x[i], DT == DT_F16 ? (dp[i] - delta) * down : dp[i] - delta);
      }
      p.set(x);
      transposed_product<DT, T>(qt, place, y * 32, p, dk);
    }
  };
  if (s0 < s1) fetch(s0, 0);
  for (int s = s0; s < s1; s += 2) {
    turn(s, std::integral_constant<int, 0>());
    if (s + 1 < s1) turn(s + 1, std::integral_constant<int, 1>());
  }
  // a key in front of every window: its own k and v may hold anything
  if (__builtin_expect(key <= off - a.window && key >= a.sinks, 0)) {
    clear<T>(dk);
    clear<T>(dv);
  }
  const float dv_scale = DT == DT_F16 ? 1.f / 32768.f : 1.f, dk_scale = only_own(a, sk.n) ? 0.f : a.scale / grow;
  if (it.record >= 0) {
    float* to = a.record + (hk * records + it.record + it.part) * (2 * ROWS * D) + (wave * 32 + r) * D;
    using F = Tile<DT_F32, D, WAVES>;
    store_rows<DT_F32, F>((char*)to, dk, dk_scale);
    store_rows<DT_F32, F>((char*)(to + ROWS * D), dv, dv_scale);
  } else {
    store(dk_scale, dv_scale);
  }
}

// the records of a tile, added in order; four dims a thread, dk and dv
template <int DT, int D, int WAVES>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a, int64_t records) {
  using T = Tile<DT, D, WAVES>;
  constexpr int ROWS = T::ROWS;
  const int hk = blockIdx.y, tile_all = blockIdx.x / (ROWS * D / 1024), chunk = blockIdx.x % (ROWS * D / 1024);
  const Item it = item_of<T>(a, tile_all, true, records);
  if (it.entry < 0 || it.parts == 1) return;
  const Span sk = entry_of(a.k_starts, it.entry, a.B, a.S);
  const int word = chunk * 1024 + (int)threadIdx.x * 4, row = word / D, dim = word % D, key = it.tile * ROWS + row;
  if (key >= sk.n) return;
  const float* from = a.record + (hk * records + it.record) * (2 * ROWS * D) + word;
  const int64_t to = (((int64_t)(sk.at + key) * a.Hkv + hk) * D + dim) * T::E;
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    floatx4 sum = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < it.parts; ++p) sum += *(const floatx4*)(from + ((int64_t)p * 2 + y) * (ROWS * D));
    char* out = (y ? a.dv : a.dk) + to;
    if constexpr (DT == DT_F32) *(floatx4*)out = sum;
    else *(u32x2*)out = u32x2{pack2_dt<DT>(sum[0], sum[1]), pack2_dt<DT>(sum[2], sum[3])};
  }
}

template <int DT, int D, int WAVES>
hipError_t launch_keys(const WindowArgs& a, int64_t records, hipStream_t st) {
  window_dkv_kernel<DT, D, WAVES><<<((unsigned)a.items * a.Hkv + 7) / 8 * 8, 64 * WAVES, 0, st>>>(a, records);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !records) return e;
  window_join_kernel<DT, D, WAVES><<<dim3((unsigned)a.k_tiles * (32 * WAVES * D / 1024), a.Hkv), 256, 0, st>>>(a, records);
  return hipGetLastError();
}

template <int DT, int D>
hipError_t launch_dt(const WindowArgs& a, int64_t records, hipStream_t st) {
  hipError_t e;
  window_delta_kernel<DT, D><<<a.delta_blocks, 256, 0, st>>>(a);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (a.q_tiles) {
    const unsigned grid = ((unsigned)a.q_tiles * a.H + 7) / 8 * 8;
    if (a.q_waves == 1) window_dq_kernel<DT, D, 1><<<grid, 64, 0, st>>>(a);
    else window_dq_kernel<DT, D, 4><<<grid, 256, 0, st>>>(a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (!a.items) return hipSuccess;
  return a.k_waves == 1 ? launch_keys<DT, D, 1>(a, records, st) : launch_keys<DT, D, 4>(a, records, st);
}

}  // namespace

// Up to so many workgroups of 128 rows (keys) a pass takes 32 each instead, one wave.  It gains where the rows see few keys, and
// in the key pass it costs where they see many: there four waves would fill the chip too, since the items cut a tile's steps, and a
// wave alone copies every stage for itself.  Calls from Python with one wave and with four, forward / gradient in us:
//   8 / 8 heads x 64, fp32, 4 x 250 tokens, window 100     20 / 54     29 / 68
//   8 / 2 x 128, bf16, 300                                 20 / 43     19 / 48
//   32 / 8 x 128, bf16, 512                                28 / 65     24 / 63
//   28 / 4 x 128, bf16, 4000, window 1000                  97 / 514    98 / 374
//   24 / 1 x 128, bf16, 2000                               64 / 368    63 / 270
//   16 / 2 x 128, fp16, 3062                               97 / 619    99 / 390
//   16 / 2 x 128, fp32, 2370                              453 / 2639  444 / 1770
// A rule that takes the key pass' items into account would have both; not built.
constexpr int64_t FEW_TILES = 256;

WindowCut window_cut(int dtype, int D, int T, int S, int H, int Hkv, int B, bool starts, bool k_starts, int window,
                     int sinks) {
  WindowCut c{};
  const int64_t G = H / Hkv;
  // one wave a workgroup where four would leave CUs without work
  c.q_waves = (T + (int64_t)127) / 128 * H < FEW_TILES ? 1 : 4;
  c.k_waves = (S + (int64_t)127) / 128 * Hkv < FEW_TILES ? 1 : 4;
  const int64_t q_rows = 32 * c.q_waves, ROWS = 32 * c.k_waves, kt = dtype == DT_F32 || c.k_waves == 1 ? 32 : 64;
  // an entry's last tile may be partly filled: those of B sequences and of the rows in front of and behind them
  c.q_tiles = (int)((T + q_rows - 1) / q_rows + (starts ? B + 1 : 0));
  c.k_tiles = (int)((S + ROWS - 1) / ROWS + (k_starts ? B + 1 : 0));
  const int64_t all = (T + kt - 1) / kt;                     // row steps of one sequence
  // rows that see a key of a tile: of its keys + window - 1, from any place of a step on
  const int64_t near = ((int64_t)window + ROWS - 1 + 2 * (kt - 1)) / kt;
  const int64_t steps = near < all ? near : all;
  c.near_steps = (int)(steps < 1 ? 1 : steps);
  // an item of all steps of a near tile, or where those are fewer than the chip holds workgroups, so few that there are
  // as many items, down to what a record costs to be written and read
  const int64_t tiles = (S + ROWS - 1) / ROWS * Hkv, items_wanted = c.k_waves == 1 ? 1024 : 512;
  const int64_t fewest = dtype == DT_F32 ? 2 : 4;
  int64_t each = G * c.near_steps;
  const int64_t even = (tiles * each + items_wanted - 1) / items_wanted;
  if (even < each) each = even < fewest ? fewest : even;
  c.steps = (int)(each < INT32_MAX ? each : INT32_MAX);
  const int64_t near_parts = (G * c.near_steps + c.steps - 1) / c.steps, key_tiles = (S + ROWS - 1) / ROWS;
  // sequences of which a tile takes several items of n steps: their rows have more than n / G steps
  auto shared = [&](int64_t n) { const int64_t most = T / (kt * (n / G) + 1); return B < most ? B : most; };
  int64_t records = near_parts > 1 ? (key_tiles + shared(c.steps)) * near_parts : 0, items = c.k_tiles + records;
  c.far_steps = c.steps;
  if (window != INT32_MAX && sinks > 0) {
    // As many steps that the tiles with sinks make two items for each place on the chip, if their steps are more than
    // that: where many keys are sinks, items of c.steps would leave records of more bytes than all gradients, quadratic in
    // the tokens (8192 tokens, 32 / 8 heads x 128, bf16, window 128, 4096 sinks: 0.91 GB, so 0.17; 1.87 -> 1.71 ms).
    const int64_t of = (sinks + ROWS - 1) / ROWS, sink_tiles = of < key_tiles ? of : key_tiles;
    const int64_t all_far = sink_tiles * G * (T / kt + (B < T ? B : T)) * Hkv, far = (all_far + 1023) / 1024;
    if (far > c.far_steps) c.far_steps = (int)(far < INT32_MAX ? far : INT32_MAX);
    // of each tile with sinks the sum over the sequences of ceil(G ceil(rows / kt) / steps)
    const int64_t n = shared(c.far_steps), parts = G * (T / kt + n) / c.far_steps + n;
    const int64_t most = (key_tiles + n) * ((G * all + c.far_steps - 1) / c.far_steps);
    const int64_t far_records = sink_tiles * parts < most ? sink_tiles * parts : most;
    items += far_records;
    records += far_records;
  }
  c.items = (int)(items < INT32_MAX ? items : INT32_MAX);
  c.records = records;
  // of 16 rows a block and turn; fp16's goes over v's too: one query of 8 heads over 131072 keys, 8 kv heads x 64,
  // 24.9 ms with blocks for the queries alone, 4.1 with these (bf16 3.4)
  const int64_t q_all = (int64_t)T * H, k_all = dtype == DT_F16 ? (int64_t)S * Hkv : 0;
  const int64_t blocks = ((q_all > k_all ? q_all : k_all) + 15) / 16;
  c.delta_blocks = (int)(blocks < 1 ? 1 : blocks < 2048 ? blocks : 2048);
  return c;
}

hipError_t launch_window_grad(int dtype, int D, const WindowArgs& a, int64_t records, hipStream_t st) {
  if (dtype == DT_F32) return D == 64 ? launch_dt<DT_F32, 64>(a, records, st) : launch_dt<DT_F32, 128>(a, records, st);
  if (dtype == DT_BF16) return D == 64 ? launch_dt<DT_BF16, 64>(a, records, st) : launch_dt<DT_BF16, 128>(a, records, st);
  return D == 64 ? launch_dt<DT_F16, 64>(a, records, st) : launch_dt<DT_F16, 128>(a, records, st);
}

}  // namespace sta
