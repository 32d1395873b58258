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

// A sequence as a row finds it: its rows of q (0 <= first, first + count <= total whatever q_starts holds) and the
// position of its first new token (whatever seq_lens holds).
struct Sequence {
  int index, first, count, base;
};

// The sequence of largest index b with key(q_starts[b], b) <= x, for a key that does not fall with b. The whole wave takes
// part and gets the same answer. A batch of up to 64 takes one round of loads; a larger one a search that looks at 64
// places at a time, and then the loads.
template <typename Key>
__device__ __forceinline__ Sequence locate(const int* __restrict__ q_starts, const int* __restrict__ seq_lens, int batch,
                                           int total, int x, Key key) {
  const int lane = int(threadIdx.x) & 63;
  Sequence s;
  int start, end, len;
  if (batch <= 64) {
    const bool there = lane < batch;
    const int at = there ? lane : 0;
    start = q_starts[at];
    end = q_starts[at + 1];
    len = seq_lens[at];
    const unsigned long long below = __ballot(there && key(start, at) <= x);
    s.index = below == 0 ? 0 : __builtin_amdgcn_readfirstlane(__popcll(below) - 1);
    start = __builtin_amdgcn_readlane(start, s.index);
    end = __builtin_amdgcn_readlane(end, s.index);
    len = __builtin_amdgcn_readlane(len, s.index);
  } else {
    s.index = find_sequence(batch, x, [&](int b) { return key(q_starts[b], b); });
    start = __builtin_amdgcn_readfirstlane(q_starts[s.index]);
    end = __builtin_amdgcn_readfirstlane(q_starts[s.index + 1]);
    len = __builtin_amdgcn_readfirstlane(seq_lens[s.index]);
  }
  s.first = min(max(start, 0), total);
  s.count = min(max(end, s.first), total) - s.first;
  s.base = int(min(max((long long)len - s.count, -(1ll << 30)), 1ll << 30));
  return s;
}

// what the kernels' grids and offsets assume
inline bool valid_paged(const gie_paged_geom* g) {
  if (!g || g->batch < 0 || g->total_tokens < 0 || (g->batch == 0 && g->total_tokens > 0)) return false;
  if (g->q_heads <= 0 || g->kv_heads <= 0 || g->q_heads % g->kv_heads != 0) return false;
  if (g->head_dim <= 0 || g->page_size <= 0 || g->page_size % 16 != 0 || g->num_pages <= 0 || g->max_pages <= 0)
    return false;
  if (g->head_dim % 32 != 0 || g->head_dim > 256 || (long long)g->max_pages * g->page_size > (1 << 30)) return false;
  if ((long long)g->total_tokens * (g->q_heads / g->kv_heads) > (1 << 30) || g->batch > (1 << 30)) return false;
  if ((long long)g->page_size * g->head_dim > (1 << 26)) return false;
  const long long q = (long long)g->q_heads * g->head_dim, kv = (long long)g->kv_heads * g->head_dim;
  if (q + 2 * kv > (1 << 30)) return false;  // a head's offset within its token, and a token's pieces, in 32 bits
  if (g->q_stride < q || g->o_stride < q || g->k_stride < kv || g->v_stride < kv) return false;
  return g->rotary_dim >= 0 && g->rotary_dim % 2 == 0 && g->rotary_dim <= g->head_dim && g->window >= 0 &&
         g->softcap >= 0 && g->max_new >= 0 && g->max_len >= 0;
}

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace gie_hip
