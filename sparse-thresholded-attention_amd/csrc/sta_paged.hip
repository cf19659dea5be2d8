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
//   O^T += V^T P^T  with the fp32 instruction of depth 4: slot i of P is, as it stands, operand B for
//                   the keys 4 (l / 16) + i, and lane l loads 1/16 of the V row of that key, whose
//                   elements e are operand A of the dims (l % 16) * VE + e
//
// so neither P nor V moves between lanes, P is never rounded, and V's 16-bit elements are only
// widened.  The fp32 instruction runs at 1/16 of the 16-bit rate and still needs a quarter of the time
// that a CU's share of the memory bandwidth takes for K and V with one tile of rows.
//
// Pieces.  The sequences' lengths are known to the device alone.  Every wave sums their units (of 4 KT
// keys) and cuts each sequence into pieces of at most `per` units, the smallest number with which the
// whole call has at most about W pieces; a prefix sum over the sequences says whose piece a workgroup
// has.  Pieces of one sequence have consecutive numbers, which are also their places in the
// workspace, and the join kernel repeats the prefix sum to find them.
constexpr int PIECES = 1024;
constexpr float LOG2E = 1.44269504088896340736f;

struct Piece {
  int b, base, n, per;          // sequence, number of its first piece, pieces of a row tile, units of a piece
};

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// the piece with number blk (want_b < 0), or the pieces of sequence want_b; false: there is none.  Every
// lane of the wave takes part; the answer is uniform.
__device__ __forceinline__ bool find_piece(const CacheView& c, int unit, int segs, int blk, int want_b, Piece& p) {
  const int lane = threadIdx.x & 63;
  int64_t sum = 0;
  for (int b = lane; b < c.B; b += 64) sum += (c.len(b) + unit - 1) / unit;
  sum = wave_sum64(sum) * segs;
  const int per = (int)max((int64_t)1, (sum + PIECES - 1) / PIECES);
  int run = 0;
  for (int b0 = 0; b0 < c.B; b0 += 64) {
    const int b = b0 + lane;
    int n = 0;
    if (b < c.B) n = max(1, ((c.len(b) + unit - 1) / unit + per - 1) / per);
    const int incl = wave_incl_sum(n * segs);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    const unsigned long long hit = want_b < 0 ? __ballot(run + incl > blk) : __ballot(b == want_b);
    if (hit) {
      const int first = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
      p.n = __builtin_amdgcn_readlane(n, first);
      p.base = run + __builtin_amdgcn_readlane(incl, first) - p.n * segs;
      p.b = b0 + first;
      p.per = per;
      return true;
    }
    run += total;
  }
  return false;
}

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ __forceinline__ float at_least(float m) { return m == -INFINITY ? 0.f : m; }   // what p is relative to

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

// element e of a lane's share of a V row, in fp32
template <int DT>
__device__ __forceinline__ float v_elem(const uint32_t* w, int e) {
  if constexpr (DT == DT_F32) return __uint_as_float(w[e]);
  else if constexpr (DT == DT_BF16) return e & 1 ? __uint_as_float(w[e / 2] & 0xffff0000u) : __uint_as_float(w[e / 2] << 16);
  else return f16_bits_to_f32(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
}

template <int W>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (W == 2) {
    const u32x2 x = *(const u32x2*)p;
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 x = *(const u32x4*)(p + 4 * i);
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

template <int DT>
__device__ __forceinline__ void store_out(char* out, const float* y, int n) {   // n = 4 or 8
  if constexpr (DT == DT_F32) {
    for (int e = 0; e < n; e += 4) *(float4*)(out + 4 * e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
  } else {
    u32x4 w;
    for (int e = 0; e < n; e += 2) w[e / 2] = pack2_dt<DT>(y[e], y[e + 1]);
    if (n == 8) *(u32x4*)out = w;
    else *(u32x2*)out = u32x2{w[0], w[1]};
  }
}

template <int DT, int D, int NT, bool ACC>
__global__ __launch_bounds__(256, NT == 1 ? 3 : 2) void paged_attend_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, NT>;
  constexpr int KS = T::KS, VE = T::VE, VW = T::VW, SUB = T::SUB, KT = T::KT;
  __shared__ floatx4 merge[4][VE * 4 * 16];
  __shared__ float merge_m[4][T::ROWS], merge_l[4][T::ROWS], merge_sum[T::ROWS];
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g4 = lane >> 4;
  Piece pc;
  if (!find_piece(c, T::UNIT, c.Hkv * tiles, blockIdx.x, -1, pc)) return;
  const int b = pc.b, x = blockIdx.x - pc.base;
  const int seg = x / pc.n, piece = x - seg * pc.n;
  const int hk = seg / tiles, row0 = (seg - hk * tiles) * T::ROWS;
  const int G = a.H / c.Hkv, R = G * a.Q;
  const int len = c.len(b);
  const int u0 = piece * pc.per, u1 = min(u0 + pc.per, (len + T::UNIT - 1) / T::UNIT);

  u32x4 q[NT][KS];
  int64_t srow[NT];
  int end[NT];                                         // keys that the lane's rows see
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + t * 16 + r;
    const int i = row % a.Q, h = hk * G + row / a.Q;
    const bool real = row < R;
    const char* qp = (const char*)a.q + (b * a.q_bs + (real ? h : 0) * a.q_hs + (real ? i : 0) * a.q_ts) * T::E + g4 * 16;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[t][s] = *(const u32x4*)(qp + s * 64);
      if (!real) q[t][s] = u32x4{0, 0, 0, 0};
    }
    end[t] = real ? len - (a.Q - 1 - i) : len;
    if (ACC) srow[t] = real ? (((int64_t)b * a.H + h) * a.Q + i) * a.score_stride : -1;
  }
  const int all_see = len - (a.Q - 1);                 // keys that every row sees

  floatx4 acc[NT][VE];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[t][e] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* table = c.table + (int64_t)b * c.t_stride;
  const char* kbase = c.k + hk * c.k_hs + g4 * 16;
  const char* vbase = c.v + hk * c.v_hs + r * (VW * 4);
  // lane's key of a turn: lane % KT; -1 behind the sequence
  auto page_at = [&](int u) {
    const int j = (u * 4 + wave) * KT + (lane & (KT - 1));
    return u < u1 && j < len ? c.page_of(table, j) : -1;
  };
  u32x4 k[SUB][KS];
  int64_t koff = 0, voff = 0;
  auto offsets = [&](int u, int page) {
    const int slot = c.slot_of((u * 4 + wave) * KT + (lane & (KT - 1)));
    koff = page < 0 ? 0 : page * c.k_ps + slot * c.k_ss;   // a key that does not exist reads page 0's first
    voff = page < 0 ? 0 : page * c.v_ps + slot * c.v_ss;
  };
  auto load_k = [&]() {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const char* p = kbase + __shfl(koff, s * 16 + r, 64);
#pragma unroll
      for (int i = 0; i < KS; ++i) k[s][i] = *(const u32x4*)(p + i * 64);
    }
  };
  int page = page_at(u0), next_page = page_at(u0 + 1);
  if (u0 < u1) {
    offsets(u0, page);
    load_k();
  }
  for (int u = u0; u < u1; ++u) {
    const int key0 = (u * 4 + wave) * KT;
    const unsigned long long there = __ballot(page >= 0);
    uint32_t v[SUB][4][VW];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<VW>(vbase + __shfl(voff, s * 16 + g4 * 4 + i, 64), v[s][i]);
    const int after = page_at(u + 2);

    floatx4 sc[NT][SUB];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        floatx4 x = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) x = mfma_qk<DT>(k[s][i], q[t][i], x);
        sc[t][s] = x * a.sm_scale;
      }
    page = next_page;
    next_page = after;
    if (u + 1 < u1) {
      offsets(u + 1, page);
      load_k();
    }

    const bool whole = there == ~0ull, mixed = key0 + KT > all_see;
    if (!whole) {
      // keys that do not exist: no score, and zeros for whatever lies where they would
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool is = there >> (s * 16 + g4 * 4 + i) & 1;
#pragma unroll
          for (int t = 0; t < NT; ++t) sc[t][s][i] = is ? sc[t][s][i] : -INFINITY;
#pragma unroll
          for (int w = 0; w < VW; ++w) v[s][i][w] = is ? v[s][i][w] : 0u;
        }
    }
    if (mixed) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + s * 16 + g4 * 4 + i >= end[t]) sc[t][s][i] = -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (ACC && srow[t] >= 0) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          const int j = key0 + s * 16 + g4 * 4;
          if (j < len) *(floatx4*)(a.scores + srow[t] + j) = sc[t][s];
        }
      }
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
          const float p = exp_of(sc[t][s][i] - m0);
          sc[t][s][i] = p;
          l[t] += p;
        }
    }
    if (!(mixed && a.Q > 1)) {
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
      // rows of one instruction see different keys: one key at a time, kept by the rows that see it, so
      // that a value of 0 * infinity or NaN reaches no other row
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + s * 16 + j * 4 + i;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const float ve = g4 == j ? v_elem<DT>(v[s][i], e) : 0.f;
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const floatx4 y = __builtin_amdgcn_mfma_f32_16x16x4f32(ve, g4 == j ? sc[t][s][i] : 0.f, acc[t][e], 0, 0, 0);
                acc[t][e] = key < end[t] ? y : acc[t][e];
              }
            }
          }
    }
  }

  // the four waves' states into one
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    if (g4 == 0) {
      merge_m[wave][t * 16 + r] = m[t];
      merge_l[wave][t * 16 + r] = l[t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = t * 16 + r;
    const float mm = fmaxf(fmaxf(merge_m[0][row], merge_m[1][row]), fmaxf(merge_m[2][row], merge_m[3][row]));
    const float m0 = at_least(mm), f = exp_of(m[t] - m0);
    float ll = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) ll += merge_l[w][row] * exp_of(merge_m[w][row] - m0);
#pragma unroll
    for (int e = 0; e < VE; ++e) merge[wave][(e * 4 + g4) * 16 + r] = acc[t][e] * f;
    if (pc.n > 1) {
      if (wave == 0 && g4 == 0) a.part_ml[(int64_t)blockIdx.x * T::ROWS + row] = make_float2(mm, ll);
    } else if (wave == 0 && g4 == 0 && row0 + row < R) {
      const int rr = row0 + row;
      a.lse[((int64_t)b * a.H + hk * G + rr / a.Q) * a.Q + rr % a.Q] = ll == 0.f ? -INFINITY : m0 + logf(ll);
    }
    if (wave == 0 && g4 == 0) merge_sum[row] = ll;
    __syncthreads();
    if (pc.n > 1) {
      floatx4* part = (floatx4*)(a.part_o + ((int64_t)blockIdx.x * T::ROWS + t * 16) * D);
      for (int i = tid; i < VE * 64; i += 256) part[i] = (merge[0][i] + merge[1][i]) + (merge[2][i] + merge[3][i]);
    } else {
      // thread: one 16th of a row
      const int orow = tid / 16, m16 = tid % 16, rr = row0 + t * 16 + orow;
      const float sum = merge_sum[t * 16 + orow], inv = sum == 0.f ? 0.f : 1.f / sum;
      if (rr < R) {
        float y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int at = part_index<VE>(orow, m16 * VE + e);
          const float* p0 = (const float*)merge[0];
          constexpr int W = VE * 64 * 4;
          y[e] = sum == 0.f ? 0.f : ((p0[at] + p0[W + at]) + (p0[2 * W + at] + p0[3 * W + at])) * inv;
        }
        const int64_t row_out = ((int64_t)b * a.H + hk * G + rr / a.Q) * a.Q + rr % a.Q;
        store_out<DT>((char*)a.out + (row_out * D + m16 * VE) * T::E, y, VE);
      }
    }
    __syncthreads();
  }
}

// one workgroup per query row: the pieces of its sequence, a wave each in turn
template <int DT, int D, int NT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int tiles) {
  using T = Tile<DT, D, NT>;
  __shared__ float o[4][D];
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hi = blockIdx.x, b = blockIdx.y, G = a.H / c.Hkv;
  Piece pc;
  if (!find_piece(c, T::UNIT, c.Hkv * tiles, 0, b, pc) || pc.n == 1) return;
  const int h = hi / a.Q, i = hi % a.Q, hk = h / G, row = (h - hk * G) * a.Q + i;
  const int first = pc.base + (hk * tiles + row / T::ROWS) * pc.n, rr = row % T::ROWS;
  const float2* ml = a.part_ml + (int64_t)first * T::ROWS + rr;
  float m = -INFINITY;
  for (int p = lane; p < pc.n; p += 64) m = fmaxf(m, ml[(int64_t)p * T::ROWS].x);
  m = wave_max_f32(m);
  const float m0 = at_least(m);
  float l = 0.f;
  for (int p = lane; p < pc.n; p += 64) {
    const float2 x = ml[(int64_t)p * T::ROWS];
    l += x.y * exp_of(x.x - m0);
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) l += __shfl_xor(l, s, 64);
  float y[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) y[e] = 0.f;
  const float* part = a.part_o + ((int64_t)first * T::ROWS + rr / 16 * 16) * D;
  for (int p = wave; p < pc.n; p += 4) {
    const float f = exp_of(ml[(int64_t)p * T::ROWS].x - m0);
#pragma unroll
    for (int e = 0; e < D / 64; ++e)
      y[e] += f * part[(int64_t)p * T::ROWS * D + part_index<T::VE>(rr % 16, lane * (D / 64) + e)];
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[wave][lane * (D / 64) + e] = y[e];
  __syncthreads();
  const int64_t row_out = ((int64_t)b * a.H + h) * a.Q + i;
  if (tid < D) {
    const float z = l == 0.f ? 0.f : ((o[0][tid] + o[1][tid]) + (o[2][tid] + o[3][tid])) / l;
    char* out = (char*)a.out + (row_out * D + tid) * T::E;
    if constexpr (DT == DT_F32) *(float*)out = z;
    else *(uint16_t*)out = (uint16_t)(DT == DT_F16 ? f32_to_f16_bits(z) : f32_to_bf16_bits(z));
  }
  if (tid == 0) a.lse[row_out] = l == 0.f ? -INFINITY : m0 + logf(l);
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

template <int DT, int D, int NT>
hipError_t launch_attend(const PagedArgs& a, const PagedCut& cut, hipStream_t st) {
  if (a.accumulate) paged_attend_kernel<DT, D, NT, true><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
  else paged_attend_kernel<DT, D, NT, false><<<cut.grid, 256, 0, st>>>(a, cut.tiles);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && !cut.single) {
    paged_join_kernel<DT, D, NT><<<dim3(a.H * a.Q, a.c.B), 256, 0, st>>>(a, cut.tiles);
    e = hipGetLastError();
  }
  if (e != hipSuccess || !a.accumulate) return e;
  paged_weight_kernel<<<dim3((a.c.cap + 255) / 256, a.c.Hkv, a.c.B), 256, 0, st>>>(a);
  return hipGetLastError();
}

template <int DT, int D>
hipError_t launch_rows(const PagedArgs& a, const PagedCut& cut, hipStream_t st) {
  return cut.rows == 16 ? launch_attend<DT, D, 1>(a, cut, st) : launch_attend<DT, D, 2>(a, cut, st);
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, hipStream_t st) {
  const int64_t threads = (int64_t)a.T * a.c.Hkv * (a.row_bytes / 16);
  const unsigned blocks = (unsigned)((threads + 255) / 256);
  append_kernel<<<blocks ? blocks : 1, 256, 0, st>>>(a);
  return hipGetLastError();
}

PagedCut paged_cut(int dtype, int H, int Hkv, int Q, int B, int cap) {
  PagedCut cut;
  const int R = H / Hkv * Q;
  cut.rows = R > 16 ? 32 : 16;
  cut.tiles = (R + cut.rows - 1) / cut.rows;
  cut.unit = dtype == STA_DTYPE_F32 ? Tile<DT_F32, 64, 1>::UNIT : Tile<DT_BF16, 64, 1>::UNIT;
  const int64_t segs = (int64_t)Hkv * cut.tiles * B, most = (cap + cut.unit - 1) / cut.unit;
  cut.single = most <= 1;
  const int64_t all = segs * most, some = segs + PIECES;
  cut.grid = (int)(all < some ? all : some);
  return cut;
}

hipError_t launch_paged(int dtype, int D, const PagedArgs& a, hipStream_t st) {
  const PagedCut cut = paged_cut(dtype, a.H, a.c.Hkv, a.Q, a.c.B, a.c.cap);
  if (dtype == STA_DTYPE_F32) return D == 64 ? launch_rows<DT_F32, 64>(a, cut, st) : launch_rows<DT_F32, 128>(a, cut, st);
  if (dtype == STA_DTYPE_BF16) return D == 64 ? launch_rows<DT_BF16, 64>(a, cut, st) : launch_rows<DT_BF16, 128>(a, cut, st);
  return D == 64 ? launch_rows<DT_F16, 64>(a, cut, st) : launch_rows<DT_F16, 128>(a, cut, st);
}

}  // namespace sta
