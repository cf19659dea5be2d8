// sta_rotary.hip -- rotary positions with one or several axes over the rows of a batch of tokens.
//
// Pair (x, y) = (row[i], row[R/2 + i]) becomes scale * (x cos t - y sin t, y cos t + x sin t) with
// t = pos[axis(i)] * pos_scale * inv_freq[i]; the gradient with respect to the row is the same with
// -sin.  The angle is formed and reduced to a fraction of a turn in 64 bits, since a position of
// 10^5 leaves fp32 an absolute error near 10^-2 of a radian; the fraction's sine and cosine and the
// rotation are fp32, rounded once into the row's type.
//
// Bound by memory: each element is read and written once.  The (cos, sin) pairs of a token serve
// all of its heads, so a workgroup takes a token: it computes them once into LDS and then streams the
// token's rows, 16 bytes of both rotation halves a thread.  16384 tokens of
// 32 + 32 heads x 128, bf16: 537 MB in 94 us, 5.7 TB/s; 32 tokens: 5 us, most of it the launch and the angles.
#include "sta_rotary.h"

namespace sta {

namespace {

template <int DT>
__global__ __launch_bounds__(256) void rotary_kernel(sta_rotary_args a, int half) {
  constexpr int V = ROT_V<DT>;
  extern __shared__ __align__(16) float2 trig[];   // [half]
  const int64_t t = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (t >= a.T) return;
  for (int f = threadIdx.x; f < half; f += 256) trig[f] = turn_of(a, f, t);
  __syncthreads();
  const int rot = half / V, chunks = rot + (a.D - 2 * half) / V;     // of a row
  const int rows = a.H + a.Hkv;
  for (int i = threadIdx.x; i < rows * chunks; i += 256) {
    const int c = i % chunks, h = i / chunks;
    const bool is_q = h < a.H;
    const int64_t ts = is_q ? a.q_tok_stride : a.k_tok_stride, hs = is_q ? a.q_head_stride : a.k_head_stride;
    const int64_t ots = is_q ? a.q_out_tok_stride : a.k_out_tok_stride;
    const int64_t ohs = is_q ? a.q_out_head_stride : a.k_out_head_stride;
    const int hh = is_q ? h : h - a.H;
    constexpr int E = DT == DT_F32 ? 4 : 2;
    const char* x = (const char*)(is_q ? a.q : a.k) + (t * ts + hh * hs) * E;
    char* o = (char*)(is_q ? a.q_out : a.k_out) + (t * ots + hh * ohs) * E;
    if (c >= rot) {                                // behind the rotated part
      const int at = (2 * half + (c - rot) * V) * E;
      *(u32x4*)(o + at) = *(const u32x4*)(x + at);
      continue;
    }
    float p[V], q[V], u[V], w[V];
    unpack16<DT>(*(const u32x4*)(x + c * 16), p);
    unpack16<DT>(*(const u32x4*)(x + half * E + c * 16), q);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 cs = trig[c * V + e];
      u[e] = p[e] * cs.x - q[e] * cs.y;
      w[e] = q[e] * cs.x + p[e] * cs.y;
    }
    *(u32x4*)(o + c * 16) = pack16<DT>(u);
    *(u32x4*)(o + half * E + c * 16) = pack16<DT>(w);
  }
}

template <int DT>
hipError_t launch_dt(const sta_rotary_args& a, hipStream_t st) {
  int half = 0;
  for (int i = 0; i < a.axes; ++i) half += a.section[i];
  // a dimension of a grid holds below 2^32 threads
  const int most = 1 << 20, blocks = a.T < most ? a.T : most;
  rotary_kernel<DT><<<dim3(blocks, (a.T - 1) / most + 1), 256, (size_t)half * sizeof(float2), st>>>(a, half);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const sta_rotary_args& a, hipStream_t st) {
  if (a.dtype == STA_DTYPE_F32) return launch_dt<DT_F32>(a, st);
  if (a.dtype == STA_DTYPE_BF16) return launch_dt<DT_BF16>(a, st);
  return launch_dt<DT_F16>(a, st);
}

}  // namespace sta
