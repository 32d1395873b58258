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
// append_normed: each head of q and k is normed first, x_d / sqrt(mean_d x_d^2 + norm_eps) * weight_d, with weights
//   [head_dim] in FP32 shared by the heads (either may be null: not normed), and rotated without a rounding between. The
//   squares are summed in FP32: heads of values past 10^19 leave its range, and with norm_eps 0 those of values under 10^-19.
// attention: out = sum_j softmax_j(s_j) v_j over the positions j <= p (and j > p - window or j < sinks), with
//   s_j = scale * q . k_j, or softcap * tanh(that / softcap). Query head h reads key head h / (q_heads / kv_heads).
//   Scores, statistics and sums are FP32; the softmax's weights are rounded once to the problem's precision ahead of the
//   second product. A token that sees nothing gets zeros.
//
// PagedKv8 is the same cache held in 8 bits: pages of codes, int8 or e4m3, and FP32 scales [num_pages][kv_heads]
// [page_size / 16], one for each head's block of 16 positions; a code c stands for c * scale.
// append: a block's scale follows the largest |x| in it, a = max(that, 2^-64): a / 127 for int8, the power of 2 that is
//   at least a / 448 for e4m3. A block that gets its first position starts anew; one that holds earlier positions keeps
//   its scale unless the new tokens need a larger one, and then the codes that it holds are rounded again to that. Codes
//   are rounded to nearest even. A block that gets an infinity or a NaN has scale NaN: all of it reads as NaN until its
//   first position is written again. No two sequences of a call may append to the same block.
// read: the rows' keys and values back in the problem's precision, one rounding: the tokens that append would write,
//   so n_b = seq_lens[b] reads a whole sequence. A row without a valid position, or of a page outside the cache, is zero.
//   (An e4m3 code may stand for up to 2^-4 more than what was appended: FP16 values from 63488 on read as infinities.)
// attention: as above over code * scale. A code of e4m3 that stands for a NaN (append writes none) counts as 480 with its
//   sign. Scales are taken to lie within 2^-73 and 2^122; one that is not counts as the nearer of these. Scales of V that
//   a row sees may lie 2^100 apart before the weights of the smaller one's block are lost from the sum. The softmax's weights
//   are rounded once to FP16, times their block's scale.
// Calls only enqueue work on `stream`; no allocation, no synchronization, so both can be captured into a graph.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "gpu_inference/conv2d.h"

namespace gie {

enum class KvCode : int { kNone = 0, kInt8 = 1, kE4m3 = 2 };

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
                                 // choose the launch shape; results depend on them by the sums' rounding alone
  int sinks = 0;         // attention: positions from 0 on that stay visible to rows whose window has passed them
  float norm_eps = 0;    // of append_normed and PagedKv8::append
  KvCode code = KvCode::kNone;  // PagedKv8: what its pages hold; PagedKv: kNone
};

void validate_problem(const PagedKvProblem& prob);

class PagedKv {
 public:
  // q and q_out may both be null (only the cache is written); q_out may be q with the same stride.
  static void append(const void* q, const void* k, const void* v, const float* cos, const float* sin,
                     const int* q_starts, const int* seq_lens, const int* page_table, const PagedKvProblem& prob,
                     void* q_out, void* k_pages, void* v_pages, hipStream_t stream);
  // q_norm, k_norm: FP32 weights [head_dim], either may be null (q_norm has to be where q is)
  static void append_normed(const void* q, const void* k, const void* v, const float* q_norm, const float* k_norm,
                            const float* cos, const float* sin, const int* q_starts, const int* seq_lens,
                            const int* page_table, const PagedKvProblem& prob, void* q_out, void* k_pages,
                            void* v_pages, hipStream_t stream);
  static void attention(const void* q, const void* k_pages, const void* v_pages, const int* q_starts,
                        const int* seq_lens, const int* page_table, const PagedKvProblem& prob, void* out,
                        void* workspace, size_t workspace_bytes, hipStream_t stream);
  static size_t workspace_size(const PagedKvProblem& prob);  // of attention
};

// pages of codes and their scales
struct Kv8Pages {
  void *k = nullptr, *v = nullptr;
  float *k_scales = nullptr, *v_scales = nullptr;
};

class PagedKv8 {
 public:
  static void append(const void* q, const void* k, const void* v, const float* q_norm, const float* k_norm,
                     const float* cos, const float* sin, const int* q_starts, const int* seq_lens,
                     const int* page_table, const PagedKvProblem& prob, void* q_out, const Kv8Pages& pages,
                     hipStream_t stream);
  // rows of k and v are k_stride and v_stride apart; either may be null
  static void read(const Kv8Pages& pages, const int* q_starts, const int* seq_lens, const int* page_table,
                   const PagedKvProblem& prob, void* k, void* v, hipStream_t stream);
  static void attention(const void* q, const Kv8Pages& pages, const int* q_starts, const int* seq_lens,
                        const int* page_table, const PagedKvProblem& prob, void* out, void* workspace,
                        size_t workspace_bytes, hipStream_t stream);
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
