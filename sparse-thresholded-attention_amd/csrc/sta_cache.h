// sta_cache.h -- the paged cache as the kernels see it, and the argument blocks of its operators.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sta.h"

namespace sta {

// sta_cache with the page size as a shift; strides in bytes for k and v, in elements otherwise
struct CacheView {
  char* k;
  char* v;
  int64_t k_ps, k_hs, k_ss, v_ps, v_hs, v_ss;
  float* weight;
  int64_t w_ps, w_hs;
  int32_t* pos;
  int64_t p_ps, p_hs;
  const int32_t* table;
  int64_t t_stride;
  const int32_t* lens;
  int pages, shift, Hkv, B;
  int cap;                 // keys a sequence can have: the table's, or max_len where smaller

  __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), cap); }
  // the page of key j, or -1 where the entry is none
  __device__ __forceinline__ int page_of(const int32_t* row, int j) const {
    const int p = row[j >> shift];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  __device__ __forceinline__ int slot_of(int j) const { return j & ((1 << shift) - 1); }
};

struct AppendArgs {
  CacheView c;
  const char* k;
  const char* v;
  int64_t k_ts, k_hs, v_ts, v_hs;   // bytes
  int T, row_shift;                 // a row is 16 << row_shift bytes
  const int32_t* starts;
  const int32_t* seen;
  int32_t* new_lens;
};

struct PagedArgs {
  CacheView c;
  const void* q;
  int64_t q_bs, q_hs, q_ts;         // elements
  int H, Q;
  float sm_scale;
  int accumulate;
  void* out;
  float* lse;                       // (B, H, Q); NULL: not stored
  // accumulate: of each row its scores' maximum and 1 / the sum of exp(score - maximum), 0 where it saw nothing;
  // row g Q + i of a kv head at (b Hkv + kv head) stat_stride + row
  float2* stats;
  int64_t stat_stride;
  float* scores;                    // (B, H, Q, score_stride); NULL: not stored
  int64_t score_stride;
  float* part_o;                    // (records, rows, D) sums of unfinished row tiles, scaled by sum_scale
  float2* part_ml;                  // (records, rows) their maxima and sums
  int runs;
};

// how a call of the attention is cut (host): a row tile is `rows` query rows of one kv head, `tiles` of them a
// kv head; `runs` runs of units of keys; `grid` workgroups, one a run and row tile
struct PagedCut {
  int rows, tiles, runs, grid;
  bool many;                        // 128 rows a workgroup, keys through LDS
  bool reform;                      // weights from scores formed again, not from stored ones
  bool small;                       // short sequences, one query each: one launch, nothing to join
  int64_t records;                  // of unfinished row tiles, in the workspace
};
PagedCut paged_cut(int dtype, int D, int H, int Hkv, int Q, int B, int cap, int page_size);

struct EvictArgs {
  CacheView c;
  int budget, n_global, n_local, row_bytes;
  const int32_t* dst_table;
  int64_t dst_stride;
  int dst_cap;                      // keys that a row of dst_table holds
  int32_t* new_lens;
  int32_t* counts;                  // (B, Hkv) rows that move
  int32_t* from;                    // (B, Hkv, moves): their slots, and where they go
  int32_t* to;
  int moves;                        // stride of the lists: the most rows that can move
};

hipError_t launch_rotary(const sta_rotary_args& a, hipStream_t st);
hipError_t launch_append(const AppendArgs& a, hipStream_t st);
hipError_t launch_paged(int dtype, int D, const PagedArgs& a, hipStream_t st);
hipError_t launch_evict(const EvictArgs& a, hipStream_t st);

}  // namespace sta
