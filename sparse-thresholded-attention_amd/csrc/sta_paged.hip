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
// attention: one workgroup per query row, scores through the workspace
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ float block_reduce(float x, float* lds, bool is_max) {
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const float y = __shfl_xor(x, m, 64);
    x = is_max ? fmaxf(x, y) : x + y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return is_max ? fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3])) : (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <int DT, int D>
__global__ __launch_bounds__(256) void paged_attend_kernel(PagedArgs a) {
  constexpr int E = DT == DT_F32 ? 4 : 2;
  __shared__ float q[D], lds[4], o[256];
  const CacheView& c = a.c;
  const int h = blockIdx.x / a.Q, i = blockIdx.x % a.Q, b = blockIdx.y, tid = threadIdx.x;
  const int hk = h / (a.H / c.Hkv);
  const int64_t row = ((int64_t)b * a.H + h) * a.Q + i;
  const int end = c.len(b) - (a.Q - 1 - i);
  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  float* s = a.scores + row * a.score_stride;
  if (tid < D) q[tid] = load_scalar<DT>(a.q, b * a.q_bs + h * a.q_hs + i * a.q_ts + tid);
  __syncthreads();
  float m = -INFINITY;
  for (int j = tid; j < end; j += 256) {
    const int p = c.page_of(table, j);
    float x = -INFINITY;
    if (p >= 0) {
      const char* k = c.k + p * c.k_ps + hk * c.k_hs + c.slot_of(j) * c.k_ss;
      float dot = 0.f;
      for (int d = 0; d < D; d += 8) {
        float kk[8];
        load8<DT>(k, d, kk);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(q[d + e], kk[e], dot);
      }
      x = dot * a.sm_scale;
    }
    s[j] = x;
    m = fmaxf(m, x);
  }
  m = block_reduce(m, lds, true);
  const float m0 = m == -INFINITY ? 0.f : m;       // no key above -inf: p = 0 for each
  float l = 0.f;
  for (int j = tid; j < end; j += 256) l += expf(s[j] - m0);
  l = block_reduce(l, lds, false);
  __syncthreads();
  const int d = tid % D;
  float acc = 0.f;
  for (int j = tid / D; j < end; j += 256 / D) {
    const int p = c.page_of(table, j);
    if (p < 0) continue;
    const char* v = c.v + p * c.v_ps + hk * c.v_hs + c.slot_of(j) * c.v_ss;
    acc = fmaf(expf(s[j] - m0), load_scalar<DT>(v, d), acc);
  }
  o[tid] = acc;
  __syncthreads();
  if (tid < D) {
    for (int g = D; g < 256; g += D) acc += o[g + tid];
    const float y = l == 0.f ? 0.f : acc / l;
    char* out = (char*)a.out + (row * D + tid) * E;
    if constexpr (DT == DT_F32) *(float*)out = y;
    else *(uint16_t*)out = (uint16_t)(DT == DT_F16 ? f32_to_f16_bits(y) : f32_to_bf16_bits(y));
  }
  if (tid == 0) a.lse[row] = l == 0.f ? -INFINITY : m0 + logf(l);
}

// one thread per key and kv head: the p of its head's rows in order
__global__ __launch_bounds__(256) void paged_weight_kernel(PagedArgs a) {
  const CacheView& c = a.c;
  const int b = blockIdx.z, hk = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const int len = c.len(b);
  if (j >= len) return;
  const int p = c.page_of(c.table + (int64_t)b * c.t_stride, j);
  if (p < 0) return;
  const int rows = a.H / c.Hkv * a.Q;
  const int64_t row0 = ((int64_t)b * c.Hkv + hk) * rows;
  float sum = 0.f;
  for (int r = 0; r < rows; ++r) {
    const float lse = a.lse[row0 + r];
    if (j < len - (a.Q - 1 - r % a.Q) && lse != -INFINITY) sum += expf(a.scores[(row0 + r) * a.score_stride + j] - lse);
  }
  c.weight[p * c.w_ps + hk * c.w_hs + c.slot_of(j)] += sum;
}

template <int DT, int D>
hipError_t launch_attend(const PagedArgs& a, hipStream_t st) {
  paged_attend_kernel<DT, D><<<dim3(a.H * a.Q, a.c.B), 256, 0, st>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.accumulate) return e;
  paged_weight_kernel<<<dim3((a.c.cap + 255) / 256, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, hipStream_t st) {
  const int64_t threads = (int64_t)a.T * a.c.Hkv * (a.row_bytes / 16);
  const unsigned blocks = (unsigned)((threads + 255) / 256);
  append_kernel<<<blocks ? blocks : 1, 256, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged(int dtype, int D, const PagedArgs& a, hipStream_t st) {
  if (dtype == STA_DTYPE_F32) return D == 64 ? launch_attend<DT_F32, 64>(a, st) : launch_attend<DT_F32, 128>(a, st);
  if (dtype == STA_DTYPE_BF16) return D == 64 ? launch_attend<DT_BF16, 64>(a, st) : launch_attend<DT_BF16, 128>(a, st);
  return D == 64 ? launch_attend<DT_F16, 64>(a, st) : launch_attend<DT_F16, 128>(a, st);
}

}  // namespace sta
