// A paged key/value cache: appending the keys and values of new tokens with the rotation of their positions, and
// attention of those tokens over the cache.
//
// K and V pages are [num_pages][kv_heads][page_size][head_dim] in the problem's precision. Sequence b owns the rows
// q_starts[b] .. q_starts[b+1]-1 of q, k, v and out (its new tokens, n_b of them, none allowed) and holds seq_lens[b]
// tokens, the new ones counted: new token i stands at position seq_lens[b] - n_b + i. Position p lies in page
// page_table[b][p / page_size], slot p % page_size. A token without a valid position (before 0, or past max_pages *
// page_size) is not stored, and its row of q_out and out is zero. A page number outside [0, num_pages) is neither
// written nor read: its keys and values count as zeros.
//
// append: pairs (u, v) of the leading rotary_dim values of each head of q and k become (u cos - v sin, u sin + v cos)
//   with the tables' row of the token's position, in FP32 with one rounding. Tables from rotary_tables() or the
//   caller's own (any scaling for long contexts is in them).
// attention: out = sum_j softmax_j(s_j) v_j over the positions j <= p (and j > p - window), with
//   s_j = scale * q . k_j, or softcap * tanh(that / softcap). Query head h reads key head h / (q_heads / kv_heads).
//   Scores, statistics and sums are FP32. A token that sees nothing gets zeros.
// Calls only enqueue work on `stream`; no allocation, no synchronization, so both can be captured into a graph.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "gpu_inference/conv2d.h"

namespace gie {

struct PagedKvProblem {
  int batch = 1, total_tokens = 1;
  int q_heads = 1, kv_heads = 1, head_dim = 128;     // head_dim 64, 96, 128 or 256
  int page_size = 16, num_pages = 1, max_pages = 1;  // page_size a multiple of 16; max_pages: row of the page table
  Precision precision = Precision::kFp16;            // kFp16 or kBf16
  int64_t q_stride = 0, k_stride = 0, v_stride = 0, o_stride = 0;  // elements between tokens; 0: packed
  int rotary_dim = 0;        // append: leading part of a head that rotates; 0: none
  bool interleaved = false;  // pairs (2j, 2j+1) instead of (j, j + rotary_dim/2)
  int max_positions = 0;     // rows of the tables, at least max_pages * page_size
  float scale = 0;           // attention: 0 stands for 1 / sqrt(head_dim)
  float softcap = 0;         // 0: not capped
  int window = 0;            // 0: unlimited
  int max_new = 0, max_len = 0;  // most new tokens and longest sequence if the host knows them (0: not known): they
                                 // choose the launch shape, no result depends on them
};

void validate_problem(const PagedKvProblem& prob);

class PagedKv {
 public:
  // q and q_out may both be null (only the cache is written); q_out may be q with the same stride.
  static void append(const void* q, const void* k, const void* v, const float* cos, const float* sin,
                     const int* q_starts, const int* seq_lens, const int* page_table, const PagedKvProblem& prob,
                     void* q_out, void* k_pages, void* v_pages, hipStream_t stream);
  static void attention(const void* q, const void* k_pages, const void* v_pages, const int* q_starts,
                        const int* seq_lens, const int* page_table, const PagedKvProblem& prob, void* out,
                        void* workspace, size_t workspace_bytes, hipStream_t stream);
  static size_t workspace_size(const PagedKvProblem& prob);  // of attention
};

// Host tables of the rotation, [max_positions][rotary_dim / 2] each, computed in 64 bits: angle(p, j) = p * f_j with
// f_j = base^(-2j / rotary_dim). Long contexts: original_positions == 0 divides every f_j by `factor` (positions
// interpolated); otherwise frequencies whose wavelength exceeds original_positions are divided, those whose wavelength
// is under a quarter of it stay, and between them f_j is blended linearly in original_positions / wavelength. cos and
// sin are multiplied by `magnitude`.
void rotary_tables(int max_positions, int rotary_dim, double base, double factor, int original_positions,
                   double magnitude, float* cos, float* sin);

}  // namespace gie
