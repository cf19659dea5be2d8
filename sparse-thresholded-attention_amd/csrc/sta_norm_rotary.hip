// sta_norm_rotary.hip -- root-mean-square norm of each head's row and its rotation in one pass, and the gradient.
//
//   n = x r w,  r = (mean(x^2) + eps)^-1/2,  y = R n  with R the rotation of sta_rotary.hip
//   g = R^T dy,  dw = sum over rows of g x r,  dx = r (g w - x r mean(g w x r))
//
// All in fp32, each result rounded once.  A row lies in a group of L lanes of a wave, each with two 16-byte chunks: a pair
// of the rotation's halves, or two behind the rotated part; the row's sums are exchanges within the group.
//
// Bound by memory: each row read (the gradient: two) and written once.  A workgroup takes several tokens, so that their rows
// fill its turns; their (cos, sin) pairs go to LDS first.  The weights' gradients are added up in registers over all of a
// workgroup's rows, then over its groups in LDS; the workgroups' sums go to the workspace and a second kernel adds them in
// order.
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
// the two chunks of unit u, -1 for none
__device__ __forceinline__ int2 chunks_of(const NormShape& s, int u) {
  if (u >= s.units) return make_int2(-1, -1);
  if (u < s.rot) return make_int2(u, s.rot + u);
  const int c = 2 * u;                     // 2 rot + 2 (u - rot)
  return make_int2(c, c + 1 < s.chunks ? c + 1 : -1);
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (!w) return 1.f;
  if (dtype == STA_DTYPE_F32) return ((const float*)w)[i];
  const uint32_t x = ((const uint16_t*)w)[i];
  return dtype == STA_DTYPE_BF16 ? bf16_bits_to_f32(x) : f16_bits_to_f32(x);
}

template <int L>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int s = 1; s < L; s *= 2) x += __shfl_xor(x, s, 64);
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

template <int DT>
__device__ __forceinline__ void load_pair(const char* row, int2 c, float* x) {
  constexpr int V = ROT_V<DT>;
  const u32x4 zero = u32x4{0, 0, 0, 0};
  unpack16<DT>(c.x >= 0 ? *(const u32x4*)(row + c.x * 16) : zero, x);
  unpack16<DT>(c.y >= 0 ? *(const u32x4*)(row + c.y * 16) : zero, x + V);
}
template <int DT>
__device__ __forceinline__ void store_pair(char* row, int2 c, const float* x) {
  constexpr int V = ROT_V<DT>;
  if (c.x >= 0) *(u32x4*)(row + c.x * 16) = pack16<DT>(x);
  if (c.y >= 0) *(u32x4*)(row + c.y * 16) = pack16<DT>(x + V);
}

// the (cos, sin) pairs of tokens t0 .. t0 + tokens - 1
__device__ __forceinline__ void turns_of(const sta_rotary_args& a, float2* trig, int half, int64_t t0, int tokens) {
  for (int i = threadIdx.x; i < tokens * half; i += 256) {
    const int t = i / half;
    trig[i] = turn_of(a, i - t * half, t0 + t);
  }
}

template <int DT, int L>
__global__ __launch_bounds__(256) void norm_rotary_kernel(sta_norm_rotary_args n, int per) {
  constexpr int V = ROT_V<DT>, E = DT == DT_F32 ? 4 : 2;
  extern __shared__ __align__(16) float2 trig[];   // [per][half]
  const sta_rotary_args& a = n.rot;
  const int64_t t0 = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * per;
  if (t0 >= a.T) return;
  const int tokens = (int)min((int64_t)per, a.T - t0);
  const NormShape s = shape_of<DT>(a);
  const int u = threadIdx.x % L, heads = a.H + a.Hkv, rows = tokens * heads;
  const int2 c = chunks_of(s, u);
  float wq[2 * V], wk[2 * V];
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) {
    const int at = e < V ? c.x : c.y;
    wq[e] = at < 0 ? 0.f : weight_at(n.q_weight, n.weight_dtype, at * V + e % V);
    wk[e] = at < 0 ? 0.f : weight_at(n.k_weight, n.weight_dtype, at * V + e % V);
  }
  turns_of(a, trig, s.half, t0, tokens);
  __syncthreads();
  // whole turns: the lanes of a wave stay together
  for (int i0 = 0; i0 < rows; i0 += 256 / L) {
    const int i = min(i0 + (int)threadIdx.x / L, rows - 1), t = i / heads, h = i - t * heads;
    const bool is_q = h < a.H;
    const int hh = is_q ? h : h - a.H;
    const char* x = is_q ? (const char*)a.q + ((t0 + t) * a.q_tok_stride + hh * a.q_head_stride) * E
                         : (const char*)a.k + ((t0 + t) * a.k_tok_stride + hh * a.k_head_stride) * E;
    char* o = is_q ? (char*)a.q_out + ((t0 + t) * a.q_out_tok_stride + hh * a.q_out_head_stride) * E
                   : (char*)a.k_out + ((t0 + t) * a.k_out_tok_stride + hh * a.k_out_head_stride) * E;
    float y[2 * V], by;
    load_pair<DT>(x, c, y);
    const float r = rms_of<L, 2 * V>(y, a.D, n.eps, by);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) y[e] = y[e] * r * (is_q ? wq[e] : wk[e]);
    if (u < s.rot) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = trig[t * s.half + u * V + e];
        const float p = y[e], q = y[V + e];
        y[e] = p * cs.x - q * cs.y;
        y[V + e] = q * cs.x + p * cs.y;
      }
    }
    if (i0 + (int)threadIdx.x / L < rows) store_pair<DT>(o, c, y);
  }
}

// The inputs' gradients, and each workgroup's sums for the weights'.  A workgroup takes every gridDim.x-th `per` tokens.
template <int DT, int L>
__global__ __launch_bounds__(256) void norm_rotary_grad_kernel(sta_norm_rotary_grad_args g, int per) {
  constexpr int V = ROT_V<DT>, E = DT == DT_F32 ? 4 : 2, GROUPS = 256 / L;
  extern __shared__ __align__(16) float2 trig[];   // [per][half], then [GROUPS][D] floats
  const sta_norm_rotary_args& n = g.fwd;
  const sta_rotary_args& a = n.rot;
  const NormShape s = shape_of<DT>(a);
  const int u = threadIdx.x % L, group = threadIdx.x / L, heads = a.H + a.Hkv;
  const int2 c = chunks_of(s, u);
  float wq[2 * V], wk[2 * V], sq[2 * V], sk[2 * V];
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) {
    const int at = e < V ? c.x : c.y;
    wq[e] = at < 0 ? 0.f : weight_at(n.q_weight, n.weight_dtype, at * V + e % V);
    wk[e] = at < 0 ? 0.f : weight_at(n.k_weight, n.weight_dtype, at * V + e % V);
    sq[e] = sk[e] = 0.f;
  }
  for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < a.T; t0 += (int64_t)gridDim.x * per) {
    const int tokens = (int)min((int64_t)per, a.T - t0), rows = tokens * heads;
    __syncthreads();
    turns_of(a, trig, s.half, t0, tokens);
    __syncthreads();
    for (int i0 = 0; i0 < rows; i0 += GROUPS) {
      const int i = min(i0 + group, rows - 1), t = i / heads, h = i - t * heads;
      const bool is_q = h < a.H, there = i0 + group < rows;
      const int hh = is_q ? h : h - a.H;
      const char* xp = is_q ? (const char*)a.q + ((t0 + t) * a.q_tok_stride + hh * a.q_head_stride) * E
                            : (const char*)a.k + ((t0 + t) * a.k_tok_stride + hh * a.k_head_stride) * E;
      const char* dp = is_q ? (const char*)g.dq_out + ((t0 + t) * g.dq_out_tok_stride + hh * g.dq_out_head_stride) * E
                            : (const char*)g.dk_out + ((t0 + t) * g.dk_out_tok_stride + hh * g.dk_out_head_stride) * E;
      char* o = is_q ? (char*)a.q_out + ((t0 + t) * a.q_out_tok_stride + hh * a.q_out_head_stride) * E
                     : (char*)a.k_out + ((t0 + t) * a.k_out_tok_stride + hh * a.k_out_head_stride) * E;
      float x[2 * V], d[2 * V], by;
      load_pair<DT>(xp, c, x);
      load_pair<DT>(dp, c, d);
      const float r = rms_of<L, 2 * V>(x, a.D, n.eps, by);
      if (u < s.rot) {                     // the rotation the other way
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 cs = trig[t * s.half + u * V + e];
          const float p = d[e], q = d[V + e];
          d[e] = p * cs.x + q * cs.y;
          d[V + e] = q * cs.x - p * cs.y;
        }
      }
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        x[e] *= r;
        const float dn = there ? d[e] * x[e] : 0.f;
        if (is_q) sq[e] += dn;
        else sk[e] += dn;
        d[e] *= is_q ? wq[e] : wk[e];
        dot = fmaf(d[e], x[e], dot);
      }
      dot = group_sum<L>(dot) / a.D;
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) d[e] = r * (d[e] - x[e] * dot) * by;
      if (there) store_pair<DT>(o, c, d);
    }
  }
  float* partial = (float*)g.workspace;
  if (!partial) return;
  float* sums = (float*)trig;              // [GROUPS][D]
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) {
      const int at = e < V ? c.x : c.y;
      if (at >= 0) sums[group * a.D + at * V + e % V] = w ? sk[e] : sq[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += 256) {
      float sum = 0.f;
      for (int x = 0; x < GROUPS; ++x) sum += sums[x * a.D + i];
      partial[((int64_t)blockIdx.x * 2 + w) * a.D + i] = sum;
    }
  }
}

// 16 dims of one weight a workgroup, its 16 groups of lanes every 16th partial sum
__global__ __launch_bounds__(256) void norm_weight_kernel(sta_norm_rotary_grad_args g, int parts) {
  __shared__ float sums[16][17];
  const int D = g.fwd.rot.D, w = blockIdx.y, lane = threadIdx.x % 16, group = threadIdx.x / 16, i = blockIdx.x * 16 + lane;
  float sum = 0.f;
  if (i < D) {
#pragma unroll 8
    for (int p = group; p < parts; p += 16) sum += ((const float*)g.workspace)[((int64_t)p * 2 + w) * D + i];
  }
  sums[group][lane] = sum;
  __syncthreads();
  if (group || i >= D) return;
  for (int x = 1; x < 16; ++x) sum += sums[x][lane];
  void* to = w ? g.dk_weight : g.dq_weight;
  if (!to) return;
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

template <int DT, int L>
hipError_t launch_l(const sta_norm_rotary_args& n, int per, hipStream_t st) {
  const int64_t blocks = ((int64_t)n.rot.T + per - 1) / per, most = 1 << 20;   // a dimension of a grid holds below 2^32 threads
  norm_rotary_kernel<DT, L><<<dim3((unsigned)(blocks < most ? blocks : most), (unsigned)((blocks - 1) / most + 1)), 256,
                              (size_t)per * half_of(n.rot) * sizeof(float2), st>>>(n, per);
  return hipGetLastError();
}
template <int DT, int L>
hipError_t launch_grad_l(const sta_norm_rotary_grad_args& g, int per, int blocks, hipStream_t st) {
  const size_t turns = (size_t)per * half_of(g.fwd.rot) * sizeof(float2), sums = (size_t)256 / L * g.fwd.rot.D * sizeof(float);
  norm_rotary_grad_kernel<DT, L><<<blocks, 256, turns > sums ? turns : sums, st>>>(g, per);
  return hipGetLastError();
}

#define STA_NORM_LANES(DT, CALL)                                \
  switch (lanes_of(a)) {                                        \
    case 8: return CALL<DT, 8> STA_ARGS;                        \
    case 16: return CALL<DT, 16> STA_ARGS;                      \
    case 32: return CALL<DT, 32> STA_ARGS;                      \
    default: return CALL<DT, 64> STA_ARGS;                      \
  }

}  // namespace

// tokens of a workgroup: so many that their rows fill four turns of it, as long as there are workgroups for the chip
int norm_tokens(const sta_rotary_args& a) {
  const int heads = a.H + a.Hkv, turn = 256 / lanes_of(a);
  int per = (4 * turn + heads - 1) / heads;
  while (per > 1 && ((int64_t)a.T + per - 1) / per < 1024) per = per / 2;
  return per < 16 ? per : 16;
}
int norm_grad_blocks(const sta_rotary_args& a) {
  const int64_t blocks = ((int64_t)a.T + norm_tokens(a) - 1) / norm_tokens(a);
  return (int)(blocks < 1024 ? blocks : 1024);
}

hipError_t launch_norm_rotary(const sta_norm_rotary_args& n, hipStream_t st) {
  const sta_rotary_args& a = n.rot;
  const int per = norm_tokens(a);
#define STA_ARGS (n, per, st)
  if (a.dtype == STA_DTYPE_F32) { STA_NORM_LANES(DT_F32, launch_l) }
  if (a.dtype == STA_DTYPE_BF16) { STA_NORM_LANES(DT_BF16, launch_l) }
  STA_NORM_LANES(DT_F16, launch_l)
#undef STA_ARGS
}

hipError_t launch_norm_rotary_grad(const sta_norm_rotary_grad_args& g, hipStream_t st) {
  const sta_rotary_args& a = g.fwd.rot;
  const int per = norm_tokens(a), blocks = norm_grad_blocks(a);
  auto inputs = [&]() -> hipError_t {
#define STA_ARGS (g, per, blocks, st)
    if (a.dtype == STA_DTYPE_F32) { STA_NORM_LANES(DT_F32, launch_grad_l) }
    if (a.dtype == STA_DTYPE_BF16) { STA_NORM_LANES(DT_BF16, launch_grad_l) }
    STA_NORM_LANES(DT_F16, launch_grad_l)
#undef STA_ARGS
  };
  if (blocks) {
    const hipError_t e = inputs();
    if (e != hipSuccess) return e;
  }
  if (!g.workspace) return hipSuccess;
  norm_weight_kernel<<<dim3((a.D + 15) / 16, 2), 256, 0, st>>>(g, blocks);
  return hipGetLastError();
}

}  // namespace sta
