// Device vocabulary of the paged key/value cache kernels (kv_append, paged_attention): which sequence a row belongs
// to, and the bounds that what the device arrays hold is put under. Private to csrc/kernels.
#pragma once

#include "device_common.h"

namespace gie_hip {

// Largest b in [0, batch) with key(b) <= x, for a key that does not fall with b and has key(0) <= x or not (then 0).
// The whole wave takes part and gets the same answer: each round looks at 64 places at once, so a batch of 64 takes
// one dependent load and one of 4096 two.
template <typename Key>
__device__ __forceinline__ int find_sequence(int batch, int x, Key key) {
  const int lane = int(threadIdx.x) & 63;
  int lo = 0, n = batch;  // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int at = lane * step;
    const bool below = at < n && key(lo + at) <= x;
    const int count = __popcll(__ballot(below));
    const int first = count > 0 ? (count - 1) * step : 0;
    lo += first;
    n = min(step, n - first);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// rows of sequence b, whatever q_starts holds: 0 <= first <= last <= total
struct Rows {
  int first, count;
};
__device__ __forceinline__ Rows sequence_rows(const int* __restrict__ q_starts, int b, int total) {
  const int s = min(max(q_starts[b], 0), total);
  const int e = min(max(q_starts[b + 1], s), total);
  return {s, e - s};
}

// what the kernels' grids and offsets assume
inline bool valid_paged(const gie_paged_geom* g) {
  if (!g || g->batch < 0 || g->total_tokens < 0 || (g->batch == 0 && g->total_tokens > 0)) return false;
  if (g->q_heads <= 0 || g->kv_heads <= 0 || g->q_heads % g->kv_heads != 0) return false;
  if (g->head_dim <= 0 || g->page_size <= 0 || g->page_size % 16 != 0 || g->num_pages <= 0 || g->max_pages <= 0)
    return false;
  if (g->head_dim % 32 != 0 || g->head_dim > 256 || (long long)g->max_pages * g->page_size > (1 << 30)) return false;
  if ((long long)g->total_tokens * (g->q_heads / g->kv_heads) > (1 << 30)) return false;
  if ((long long)g->page_size * g->head_dim > (1 << 26)) return false;
  const long long q = (long long)g->q_heads * g->head_dim, kv = (long long)g->kv_heads * g->head_dim;
  if (g->q_stride < q || g->o_stride < q || g->k_stride < kv || g->v_stride < kv) return false;
  return g->rotary_dim >= 0 && g->rotary_dim % 2 == 0 && g->rotary_dim <= g->head_dim && g->window >= 0 &&
         g->softcap >= 0 && g->max_new >= 0 && g->max_len >= 0;
}

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace gie_hip
