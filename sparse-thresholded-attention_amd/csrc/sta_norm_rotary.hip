// sta_norm_rotary.hip -- root-mean-square norm of each head's row and its rotation in one pass, and the gradient.
//
//   n = x r w,  r = (mean(x^2) + eps)^-1/2,  y = R n  with R the rotation of sta_rotary.hip
//   g = R^T dy,  dw = sum over rows of g x r,  dx = r (g w - x r mean(g w x r))
//
// All in fp32, each result rounded once; a weight's gradient summed in fp32 too errs by 1.6 to 2.4 times what fp32 terms summed in 64
// bits do (8191 tokens of 32 heads: 1.6e-7 of it).  A row lies in a group of L lanes of a wave, each with two 16-byte chunks: a pair
// of the rotation's halves, or two behind the rotated part; the row's sums are exchanges within the group.
//
// Bound by memory: each row read (the gradient: two) and written once.  A workgroup takes several tokens of q or of k, so that
// their rows fill its turns; the next turn's rows are on their way during this one's work, and the tokens' (cos, sin) pairs go
// to LDS first.  The weights' gradients are added up in registers over all of a workgroup's rows, then over its groups in
// LDS; the workgroups' sums go to the workspace and a second kernel adds them in order.  8191 tokens of 32 + 8 heads x 128,
// fp16: 168 MB in 27 us, 6.2 TB/s (inputs in the cache; 35 us a call, 4.8 TB/s, with others between); the gradient of 16384
// tokens, bf16: 503 MB in 116 us, 4.3 TB/s.
#include "sta_rotary.h"

namespace sta {

namespace {

struct NormShape {
  int half, rot, units, chunks;            // frequencies, chunks of a half, pairs of chunks and chunks of a row
};
template <int DT>
__device__ __forceinline__ NormShape shape_of(const sta_rotary_args& a) {
  NormShape s{0, 0, 0, 0};
  for (int i = 0; i < a.axes; ++i) s.half += a.section[i];
  s.rot = s.half / ROT_V<DT>;
  s.chunks = a.D / ROT_V<DT>;
  s.units = (s.chunks + 1) / 2;
  return s;
}
// the two chunks of unit u; one that is none (there) stands for chunk 0, and its values count as 0
struct Lane {
  int a, b;
  bool has_a, has_b, turns;
};
__device__ __forceinline__ Lane lane_of(const NormShape& s, int u) {
  Lane l;
  l.turns = u < s.rot;
  l.a = l.turns ? u : 2 * u;               // behind the rotated ones 2 rot + 2 (u - rot)
  l.b = l.turns ? s.rot + u : 2 * u + 1;
  l.has_a = u < s.units;
  l.has_b = l.has_a && l.b < s.chunks;
  if (!l.has_a) l.a = 0;
  if (!l.has_b) l.b = 0;
  return l;
}

// 16 bytes' worth of a row's elements from element i of a weight on, 16-byte aligned
template <int V>
__device__ __forceinline__ void load_weight(const void* w, int dtype, int i, float* x) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = 1.f;
  } else if (dtype == STA_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const float4 y = *(const float4*)((const float*)w + i + e);
      x[e] = y.x, x[e + 1] = y.y, x[e + 2] = y.z, x[e + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const u32x2 y = *(const u32x2*)((const uint16_t*)w + i + e);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const uint32_t bits = z & 1 ? y[z / 2] >> 16 : y[z / 2] & 0xffffu;
        x[e + z] = dtype == STA_DTYPE_BF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32(bits);
      }
    }
  }
}

// the sum over each group of L lanes, 8 to 64, in all of its lanes
template <int L>
__device__ __forceinline__ float group_sum(float x) {
  x = group8_sum(x);
#pragma unroll
  for (int s = 8; s < L; s *= 2) x += __shfl_xor(x, s, 64);
  return x;
}
template <int L>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
  for (int s = 1; s < L; s *= 2) x = fmaxf(x, __shfl_xor(x, s, 64));
  return x;
}

// 1 / rms of a row whose lane holds x[N].  Squares that pass fp32's range, or lose bits at its lower end: x is scaled by a power
// of two first, which the caller's row keeps; `by` is that power.
template <int L, int N>
__device__ __forceinline__ float rms_of(float* x, int D, float eps, float& by) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) ss = fmaf(x[e], x[e], ss);
  ss = group_sum<L>(ss);
  by = 1.f;
  const bool out = !(ss < 1e38f) || ss < 1e-30f;
  if (__any(out)) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) most = fmaxf(most, fabsf(x[e]));
    most = group_max<L>(most);
    if (out && most > 0.f && most < INFINITY) {
      by = __uint_as_float((uint32_t)(127 - max(min(ilogbf(most), 126), -126)) << 23);
      ss = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[e] *= by;
        ss = fmaf(x[e], x[e], ss);
      }
    }
    const float again = group_sum<L>(ss);
    if (by != 1.f) ss = again;
  }
  const float scaled = eps > 0.f ? eps * by * by : 0.f;      // eps beside a sum of scaled squares
  if (!(scaled < INFINITY)) return rsqrtf(eps) / by;         // x is nothing beside eps
  return rsqrtf(ss / D + scaled);
}

// a lane's two chunks of a row
struct Pair {
  u32x4 a, b;
};
__device__ __forceinline__ Pair load_pair(const char* row, const Lane& l) {
  return Pair{*(const u32x4*)(row + l.a * 16), *(const u32x4*)(row + l.b * 16)};
}
// whole: every lane has both chunks
template <int DT>
__device__ __forceinline__ void values_of(Pair p, const Lane& l, bool whole, float* x) {
  if (!whole) {
    const u32x4 zero = u32x4{0, 0, 0, 0};
    if (!l.has_a) p.a = zero;
    if (!l.has_b) p.b = zero;
  }
  unpack16<DT>(p.a, x);
  unpack16<DT>(p.b, x + ROT_V<DT>);
}
template <int DT>
__device__ __forceinline__ void store_pair(char* row, const Lane& l, const float* x) {
  constexpr int V = ROT_V<DT>;
  if (l.has_a) *(u32x4*)(row + l.a * 16) = pack16<DT>(x);
  if (l.has_b) *(u32x4*)(row + l.b * 16) = pack16<DT>(x + V);
}

// the (cos, sin) pairs of tokens t0 .. t0 + tokens - 1
__device__ __forceinline__ void turns_of(const sta_rotary_args& a, float2* trig, int half, int64_t t0, int tokens) {
  for (int i = threadIdx.x; i < tokens * half; i += 256) {
    const int t = i / half;
    trig[i] = turn_of(a, i - t * half, t0 + t);
  }
}

// q's rows or k's: strides in bytes.  A workgroup takes one of the two, so that it holds one weight and one sum.
struct Rows {
  const char *x, *d;
  char* out;
  int64_t x_ts, x_hs, d_ts, d_hs, out_ts, out_hs;
  int heads;
  const void* weight;
};
template <int DT>
__device__ __forceinline__ Rows rows_of(const sta_norm_rotary_args& n, bool is_q) {
  constexpr int E = DT == DT_F32 ? 4 : 2;
  const sta_rotary_args& a = n.rot;
  if (is_q)
    return Rows{(const char*)a.q, nullptr, (char*)a.q_out, a.q_tok_stride * E, a.q_head_stride * E, 0, 0,
                a.q_out_tok_stride * E, a.q_out_head_stride * E, a.H, n.q_weight};
  return Rows{(const char*)a.k, nullptr, (char*)a.k_out, a.k_tok_stride * E, a.k_head_stride * E, 0, 0,
              a.k_out_tok_stride * E, a.k_out_head_stride * E, a.Hkv, n.k_weight};
}

// A group's row among those of a workgroup's tokens, TURN rows a step: heads run fastest.  Offsets instead of products and
// divisions, which would be a third of a row's instructions.
template <int TURN>
struct Walk {
  int i, h, t;                             // number, head, token
  int dh, dt;                              // of a step
  __device__ __forceinline__ void set(int first, int heads) {
    i = first;
    t = first / heads;
    h = first - t * heads;
    dt = TURN / heads;
    dh = TURN - dt * heads;
  }
  // to the next row; the offset of a row in a tensor with these strides follows
  __device__ __forceinline__ bool step(int heads) {
    i += TURN;
    t += dt;
    h += dh;
    const bool over = h >= heads;
    if (over) h -= heads, ++t;
    return over;
  }
};
struct Offset {
  int64_t at, step, over;
  template <int TURN>
  __device__ __forceinline__ void set(const Walk<TURN>& w, int heads, int64_t ts, int64_t hs) {
    at = w.t * ts + w.h * hs;
    step = w.dt * ts + w.dh * hs;
    over = step + ts - heads * hs;
  }
  __device__ __forceinline__ void next(bool past) { at += past ? over : step; }
};

// `per` tokens of q a workgroup, then of k; q_blocks workgroups are q's
struct NormCut {
  int64_t q_blocks, k_blocks;
  int q_per, k_per;
};

template <int DT, int L>
__global__ __launch_bounds__(256) void norm_rotary_kernel(sta_norm_rotary_args n, NormCut cut) {
  constexpr int V = ROT_V<DT>, TURN = 256 / L;
  extern __shared__ __align__(16) float2 trig[];   // [per][half]
  const sta_rotary_args& a = n.rot;
  const int64_t id = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const bool is_q = id < cut.q_blocks;
  const int per = is_q ? cut.q_per : cut.k_per;
  const int64_t t0 = (is_q ? id : id - cut.q_blocks) * per;
  if (t0 >= a.T) return;
  const Rows s = rows_of<DT>(n, is_q);
  const int tokens = (int)min((int64_t)per, a.T - t0), rows = tokens * s.heads;
  const NormShape shape = shape_of<DT>(a);
  const int u = threadIdx.x % L;
  const Lane c = lane_of(shape, u);
  const bool whole = shape.chunks == 2 * L;
  Walk<TURN> row;
  row.set(threadIdx.x / L, s.heads);
  Offset from, to;
  from.set(row, s.heads, s.x_ts, s.x_hs);
  to.set(row, s.heads, s.out_ts, s.out_hs);
  const char* x = s.x + t0 * s.x_ts;
  char* out = s.out + t0 * s.out_ts;
  const Pair none = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
  Pair next = none;
  if (row.i < rows) next = load_pair(x + from.at, c);
  float w[2 * V];
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) w[e] = 0.f;
  if (c.has_a) load_weight<V>(s.weight, n.weight_dtype, c.a * V, w);
  if (c.has_b) load_weight<V>(s.weight, n.weight_dtype, c.b * V, w + V);
  turns_of(a, trig, shape.half, t0, tokens);
  __syncthreads();
  // whole turns: the lanes of a wave stay together
  for (int i0 = 0; i0 < rows; i0 += TURN) {
    const Pair now = next;
    const bool there = row.i < rows;
    const float2* turn = trig + row.t * shape.half + u * V;
    char* o = out + to.at;
    const bool past = row.step(s.heads);
    from.next(past);
    to.next(past);
    if (row.i < rows) next = load_pair(x + from.at, c);
    float y[2 * V], by;
    values_of<DT>(now, c, whole, y);
    const float r = rms_of<L, 2 * V>(y, a.D, n.eps, by);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) y[e] = y[e] * r * w[e];
    if (c.turns && there) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = turn[e];
        const float p = y[e], q = y[V + e];
        y[e] = p * cs.x - q * cs.y;
        y[V + e] = q * cs.x + p * cs.y;
      }
    }
    if (there) store_pair<DT>(o, c, y);
  }
}

// The inputs' gradients, and each workgroup's sums for its weight's: it takes a range of tokens, `per` at a time.
template <int DT, int L>
__global__ __launch_bounds__(256, 3) void norm_rotary_grad_kernel(sta_norm_rotary_grad_args g, NormCut cut) {
  constexpr int V = ROT_V<DT>, E = DT == DT_F32 ? 4 : 2, TURN = 256 / L;
  extern __shared__ __align__(16) float2 trig[];   // [per][half], then [TURN][D] floats
  const sta_norm_rotary_args& n = g.fwd;
  const sta_rotary_args& a = n.rot;
  const bool is_q = blockIdx.x < cut.q_blocks;
  const int per = is_q ? cut.q_per : cut.k_per;
  const int64_t block = is_q ? blockIdx.x : blockIdx.x - cut.q_blocks, blocks = is_q ? cut.q_blocks : cut.k_blocks;
  Rows s = rows_of<DT>(n, is_q);
  s.d = (const char*)(is_q ? g.dq_out : g.dk_out);
  s.d_ts = (is_q ? g.dq_out_tok_stride : g.dk_out_tok_stride) * E;
  s.d_hs = (is_q ? g.dq_out_head_stride : g.dk_out_head_stride) * E;
  const NormShape shape = shape_of<DT>(a);
  const int u = threadIdx.x % L, mine = threadIdx.x / L;
  const Lane c = lane_of(shape, u);
  const bool whole = shape.chunks == 2 * L;
  float w[2 * V], sum[2 * V];
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) w[e] = sum[e] = 0.f;
  if (c.has_a) load_weight<V>(s.weight, n.weight_dtype, c.a * V, w);
  if (c.has_b) load_weight<V>(s.weight, n.weight_dtype, c.b * V, w + V);
  const Pair none = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
  const int64_t t1 = a.T * (block + 1) / blocks;
  for (int64_t t0 = a.T * block / blocks; t0 < t1; t0 += per) {
    const int tokens = (int)min((int64_t)per, t1 - t0), rows = tokens * s.heads;
    Walk<TURN> row;
    row.set(mine, s.heads);
    Offset from_x, from_d, to;
    from_x.set(row, s.heads, s.x_ts, s.x_hs);
    from_d.set(row, s.heads, s.d_ts, s.d_hs);
    to.set(row, s.heads, s.out_ts, s.out_hs);
    const char *x0 = s.x + t0 * s.x_ts, *d0 = s.d + t0 * s.d_ts;
    char* out = s.out + t0 * s.out_ts;
    Pair next_x = none, next_d = none;
    if (row.i < rows) {
      next_x = load_pair(x0 + from_x.at, c);
      next_d = load_pair(d0 + from_d.at, c);
    }
    __syncthreads();
    turns_of(a, trig, shape.half, t0, tokens);
    __syncthreads();
    for (int i0 = 0; i0 < rows; i0 += TURN) {
      const bool there = row.i < rows;
      const Pair now_x = next_x, now_d = next_d;
      const float2* turn = trig + row.t * shape.half + u * V;
      char* o = out + to.at;
      const bool past = row.step(s.heads);
      from_x.next(past);
      from_d.next(past);
      to.next(past);
      next_x = next_d = none;              // rows behind the last add nothing to the sums
      if (row.i < rows) {
        next_x = load_pair(x0 + from_x.at, c);
        next_d = load_pair(d0 + from_d.at, c);
      }
      float x[2 * V], d[2 * V], by;
      values_of<DT>(now_x, c, whole, x);
      values_of<DT>(now_d, c, whole, d);
      const float r = rms_of<L, 2 * V>(x, a.D, n.eps, by);
      if (!there) continue;
      if (c.turns) {                       // the rotation the other way
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 cs = turn[e];
          const float p = d[e], q = d[V + e];
          d[e] = p * cs.x + q * cs.y;
          d[V + e] = q * cs.x - p * cs.y;
        }
      }
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        x[e] *= r;
        sum[e] = fmaf(d[e], x[e], sum[e]);
        d[e] *= w[e];
        dot = fmaf(d[e], x[e], dot);
      }
      dot = group_sum<L>(dot) / a.D;       // a row's lanes are all there or none of them
      const float scale = r * by;
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) d[e] = (d[e] - x[e] * dot) * scale;
      store_pair<DT>(o, c, d);
    }
  }
  float* partial = (float*)g.workspace;
  if (!partial) return;
  float* sums = (float*)trig;              // [TURN][D]
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) {
    if (e < V ? c.has_a : c.has_b) sums[mine * a.D + (e < V ? c.a : c.b) * V + e % V] = sum[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.D; i += 256) {
    float x = 0.f;
    for (int y = 0; y < TURN; ++y) x += sums[y * a.D + i];
    partial[(int64_t)blockIdx.x * a.D + i] = x;
  }
}

// 16 dims of one weight a workgroup, its 64 groups of lanes every 64th partial sum
__global__ __launch_bounds__(1024) void norm_weight_kernel(sta_norm_rotary_grad_args g, NormCut cut) {
  __shared__ float sums[64][17];
  const int D = g.fwd.rot.D, lane = threadIdx.x % 16, group = threadIdx.x / 16, i = blockIdx.x * 16 + lane;
  const bool is_q = blockIdx.y == 0;
  void* to = is_q ? g.dq_weight : g.dk_weight;
  if (!to) return;
  const float* from = (const float*)g.workspace + (is_q ? 0 : cut.q_blocks * D);
  const int parts = (int)(is_q ? cut.q_blocks : cut.k_blocks);
  float sum = 0.f;
  if (i < D) {
#pragma unroll 8
    for (int p = group; p < parts; p += 64) sum += from[(int64_t)p * D + i];
  }
  sums[group][lane] = sum;
  __syncthreads();
  for (int half = 32; half; half /= 2) {
    if (group < half) sums[group][lane] += sums[group + half][lane];
    __syncthreads();
  }
  if (group || i >= D) return;
  sum = sums[0][lane];
  const int dtype = g.fwd.weight_dtype;
  if (dtype == STA_DTYPE_F32) ((float*)to)[i] = sum;
  else ((uint16_t*)to)[i] = (uint16_t)(dtype == STA_DTYPE_F16 ? f32_to_f16_bits(sum) : f32_to_bf16_bits(sum));
}

// lanes of a row: its pairs of chunks, rounded up to a power of two from 8 on
int lanes_of(const sta_rotary_args& a) {
  const int units = (a.D / (a.dtype == STA_DTYPE_F32 ? 4 : 8) + 1) / 2;
  int l = 8;
  while (l < units) l *= 2;
  return l;
}
int half_of(const sta_rotary_args& a) {
  int half = 0;
  for (int i = 0; i < a.axes; ++i) half += a.section[i];
  return half;
}

// tokens of a workgroup: so many that their rows fill four turns of it, as long as there are workgroups for the chip
int tokens_of(const sta_rotary_args& a, int heads) {
  const int turn = 256 / lanes_of(a);
  int per = (4 * turn + heads - 1) / heads;
  if (per > 16) per = 16;
  while (per > 1 && ((int64_t)a.T + per - 1) / per < 512) per /= 2;
  return per;
}
NormCut cut_of(const sta_rotary_args& a) {
  NormCut c{0, 0, 1, 1};
  if (a.H) c.q_blocks = ((int64_t)a.T + (c.q_per = tokens_of(a, a.H)) - 1) / c.q_per;
  if (a.Hkv) c.k_blocks = ((int64_t)a.T + (c.k_per = tokens_of(a, a.Hkv)) - 1) / c.k_per;
  return c;
}
// The gradient's workgroups are at most MOST and one, q's and k's in the ratio of their rows, since each leaves a sum of its weight's.
// 16384 tokens of 32 + 8 heads x 128, bf16, with 768 / 1536 / 2048 / 3000 / 8192: 155 / 126 / 119 / 116 / 117 us with the
// second kernel (few stay until the last is done, many leave it more to add).
constexpr int64_t MOST = 2560;
NormCut grad_cut_of(const sta_rotary_args& a) {
  NormCut c = cut_of(a);
  const int64_t all = a.H + (int64_t)a.Hkv, q_most = a.H ? (MOST * (int64_t)a.H + all - 1) / all : 0, k_most = MOST + 1 - q_most;
  if (c.q_blocks > q_most) c.q_blocks = q_most;
  if (c.k_blocks > k_most) c.k_blocks = k_most;
  // tokens between two barriers: a workgroup's, up to 32 (16 KB of angles)
  auto per = [&](int64_t blocks) {
    const int64_t n = blocks ? (a.T + blocks - 1) / blocks : 1, turns = (n + 31) / 32;
    return (int)((n + turns - 1) / turns);
  };
  c.q_per = per(c.q_blocks);
  c.k_per = per(c.k_blocks);
  return c;
}

template <int DT, int L>
hipError_t launch_l(const sta_norm_rotary_args& n, const NormCut& cut, hipStream_t st) {
  const int64_t blocks = cut.q_blocks + cut.k_blocks, most = 1 << 20;   // a dimension of a grid holds below 2^32 threads
  const int per = cut.q_per > cut.k_per ? cut.q_per : cut.k_per;
  norm_rotary_kernel<DT, L><<<dim3((unsigned)(blocks < most ? blocks : most), (unsigned)((blocks - 1) / most + 1)), 256,
                              (size_t)per * half_of(n.rot) * sizeof(float2), st>>>(n, cut);
  return hipGetLastError();
}
template <int DT, int L>
hipError_t launch_grad_l(const sta_norm_rotary_grad_args& g, const NormCut& cut, hipStream_t st) {
  const int per = cut.q_per > cut.k_per ? cut.q_per : cut.k_per;
  const size_t turns = (size_t)per * half_of(g.fwd.rot) * sizeof(float2), sums = (size_t)256 / L * g.fwd.rot.D * sizeof(float);
  norm_rotary_grad_kernel<DT, L><<<(unsigned)(cut.q_blocks + cut.k_blocks), 256, turns > sums ? turns : sums, st>>>(g, cut);
  return hipGetLastError();
}

#define STA_NORM_LANES(DT, CALL, ARGS)                          \
  switch (lanes_of(a)) {                                        \
    case 8: return CALL<DT, 8> ARGS;                            \
    case 16: return CALL<DT, 16> ARGS;                          \
    case 32: return CALL<DT, 32> ARGS;                          \
    default: return CALL<DT, 64> ARGS;                          \
  }

hipError_t launch_inputs(const sta_norm_rotary_grad_args& g, const NormCut& cut, hipStream_t st) {
  const sta_rotary_args& a = g.fwd.rot;
  if (a.dtype == STA_DTYPE_F32) { STA_NORM_LANES(DT_F32, launch_grad_l, (g, cut, st)) }
  if (a.dtype == STA_DTYPE_BF16) { STA_NORM_LANES(DT_BF16, launch_grad_l, (g, cut, st)) }
  STA_NORM_LANES(DT_F16, launch_grad_l, (g, cut, st))
}

}  // namespace

int norm_grad_blocks(const sta_rotary_args& a) {
  const NormCut c = grad_cut_of(a);
  return (int)(c.q_blocks + c.k_blocks);
}

hipError_t launch_norm_rotary(const sta_norm_rotary_args& n, hipStream_t st) {
  const sta_rotary_args& a = n.rot;
  const NormCut cut = cut_of(a);
  if (a.dtype == STA_DTYPE_F32) { STA_NORM_LANES(DT_F32, launch_l, (n, cut, st)) }
  if (a.dtype == STA_DTYPE_BF16) { STA_NORM_LANES(DT_BF16, launch_l, (n, cut, st)) }
  STA_NORM_LANES(DT_F16, launch_l, (n, cut, st))
}

hipError_t launch_norm_rotary_grad(const sta_norm_rotary_grad_args& g, hipStream_t st) {
  const sta_rotary_args& a = g.fwd.rot;
  const NormCut cut = grad_cut_of(a);
  if (cut.q_blocks + cut.k_blocks) {
    const hipError_t e = launch_inputs(g, cut, st);
    if (e != hipSuccess) return e;
  }
  if (!g.workspace) return hipSuccess;
  norm_weight_kernel<<<dim3((a.D + 15) / 16, 2), 1024, 0, st>>>(g, cut);
  return hipGetLastError();
}

}  // namespace sta
