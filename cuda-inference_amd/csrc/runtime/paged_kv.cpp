// PagedKv: argument checks, the calls into the cache and attention kernels (gie_hip_kv_append,
// gie_hip_paged_attention), and the host tables of the rotation.
#include "gpu_inference/paged_kv.h"

#include <cmath>
#include <limits>
#include <string>

#include "gie_hip.h"
#include "gpu_inference/error.h"
#include "gpu_inference/roctx.h"

namespace gie {
namespace {

void require(bool ok, const char* what) { GIE_REQUIRE(ok, StatusCode::kInvalidArgument, std::string("PagedKv: ") + what); }
void support(bool ok, const char* what) { GIE_REQUIRE(ok, StatusCode::kUnsupported, std::string("PagedKv: ") + what); }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

gie_paged_geom geom_of(const PagedKvProblem& p) {
  gie_paged_geom g{};
  g.batch = p.batch;
  g.total_tokens = p.total_tokens;
  g.q_heads = p.q_heads;
  g.kv_heads = p.kv_heads;
  g.head_dim = p.head_dim;
  g.page_size = p.page_size;
  g.num_pages = p.num_pages;
  g.max_pages = p.max_pages;
  const int64_t q = int64_t(p.q_heads) * p.head_dim, kv = int64_t(p.kv_heads) * p.head_dim;
  g.q_stride = p.q_stride ? p.q_stride : q;
  g.k_stride = p.k_stride ? p.k_stride : kv;
  g.v_stride = p.v_stride ? p.v_stride : kv;
  g.o_stride = p.o_stride ? p.o_stride : q;
  g.rotary_dim = p.rotary_dim;
  g.interleaved = p.interleaved ? 1 : 0;
  g.max_positions = p.max_positions;
  g.scale = p.scale != 0 ? p.scale : float(1.0 / std::sqrt(double(p.head_dim)));
  g.softcap = p.softcap;
  g.window = p.window;
  g.max_new = p.max_new;
  g.max_len = p.max_len;
  return g;
}

int dtype_of(Precision p) { return p == Precision::kFp16 ? GIE_HIP_FP16 : GIE_HIP_BF16; }

void require_cache(const void* k_pages, const void* v_pages, const int* q_starts, const int* seq_lens,
                   const int* page_table) {
  require(k_pages && v_pages && q_starts && seq_lens && page_table,
          "k_pages, v_pages, q_starts, seq_lens and page_table must not be null");
  require(aligned(k_pages, 16) && aligned(v_pages, 16), "pages must be 16-byte aligned");
  require(k_pages != v_pages, "K and V need pages of their own");
  require(aligned(q_starts, 4) && aligned(seq_lens, 4) && aligned(page_table, 4),
          "q_starts, seq_lens and page_table must be 4-byte aligned");
}

}  // namespace

void validate_problem(const PagedKvProblem& p) {
  require(p.batch >= 0 && p.total_tokens >= 0, "batch and total_tokens must not be negative");
  require(p.batch > 0 || p.total_tokens == 0, "tokens without a sequence");
  require(p.q_heads > 0 && p.kv_heads > 0 && p.q_heads % p.kv_heads == 0,
          "q_heads must be a positive multiple of kv_heads");
  require(p.page_size > 0 && p.num_pages > 0 && p.max_pages > 0 && p.head_dim > 0,
          "page_size, num_pages, max_pages and head_dim must be positive");
  require(p.rotary_dim >= 0 && p.rotary_dim % 2 == 0 && p.rotary_dim <= p.head_dim,
          "rotary_dim must be even and within head_dim");
  require(p.window >= 0 && p.max_new >= 0 && p.max_len >= 0 && p.max_positions >= 0,
          "window, max_new, max_len and max_positions must not be negative");
  require(std::isfinite(p.scale) && std::isfinite(p.softcap) && p.softcap >= 0,
          "scale must be finite, softcap finite and not negative");
  const int64_t q = int64_t(p.q_heads) * p.head_dim, kv = int64_t(p.kv_heads) * p.head_dim;
  require(p.q_stride == 0 || p.q_stride >= q, "q_stride is shorter than a token's heads");
  require(p.o_stride == 0 || p.o_stride >= q, "o_stride is shorter than a token's heads");
  require(p.k_stride == 0 || p.k_stride >= kv, "k_stride is shorter than a token's heads");
  require(p.v_stride == 0 || p.v_stride >= kv, "v_stride is shorter than a token's heads");
  support(p.precision == Precision::kFp16 || p.precision == Precision::kBf16, "precision must be fp16 or bf16");
  support(p.head_dim == 64 || p.head_dim == 96 || p.head_dim == 128 || p.head_dim == 256,
          "head_dim must be 64, 96, 128 or 256");
  support(p.page_size % 16 == 0, "page_size must be a multiple of 16");
  support(int64_t(p.max_pages) * p.page_size <= std::numeric_limits<int32_t>::max() / 2,
          "max_pages * page_size passes 2^30 positions");
  support(int64_t(p.total_tokens) * (p.q_heads / p.kv_heads) <= std::numeric_limits<int32_t>::max() / 2,
          "total_tokens * (q_heads / kv_heads) passes 2^30 rows");
  support(p.batch <= std::numeric_limits<int32_t>::max() / 2, "batch passes 2^30 sequences");
  support(q + 2 * kv <= (1 << 30), "a token's heads of q, k and v pass 2^30 values");
  support(int64_t(p.page_size) * p.head_dim <= (1 << 26), "a page of one head is over 128 MiB");
}

void PagedKv::append(const void* q, const void* k, const void* v, const float* cos, const float* sin,
                     const int* q_starts, const int* seq_lens, const int* page_table, const PagedKvProblem& p,
                     void* q_out, void* k_pages, void* v_pages, hipStream_t stream) {
  validate_problem(p);
  if (p.total_tokens == 0) return;
  require_cache(k_pages, v_pages, q_starts, seq_lens, page_table);
  require(k && v, "k and v must not be null");
  require((q == nullptr) == (q_out == nullptr), "q and q_out go together");
  require(aligned(q, 2) && aligned(k, 2) && aligned(v, 2) && aligned(q_out, 2),
          "q, k, v and q_out must be aligned to their elements");
  const gie_paged_geom g = geom_of(p);
  require(q != q_out || q == nullptr || g.q_stride == g.o_stride, "q in place needs q_stride == o_stride");
  if (p.rotary_dim > 0) {
    require(cos && sin && aligned(cos, 4) && aligned(sin, 4), "cos and sin must be there and 4-byte aligned");
    require(int64_t(p.max_positions) >= int64_t(p.max_pages) * p.page_size,
            "max_positions must cover max_pages * page_size positions");
  }
  RoctxRange range("gie::PagedKv::append");
  check_kernel_status(gie_hip_kv_append(dtype_of(p.precision), &g, q, k, v, cos, sin, q_starts, seq_lens, page_table,
                                        q_out, k_pages, v_pages, stream),
                      "PagedKv::append");
}

size_t PagedKv::workspace_size(const PagedKvProblem& p) {
  validate_problem(p);
  const gie_paged_geom g = geom_of(p);
  return gie_hip_paged_attention_workspace(&g);
}

void PagedKv::attention(const void* q, const void* k_pages, const void* v_pages, const int* q_starts,
                        const int* seq_lens, const int* page_table, const PagedKvProblem& p, void* out,
                        void* workspace, size_t workspace_bytes, hipStream_t stream) {
  validate_problem(p);
  if (p.total_tokens == 0) return;
  require_cache(k_pages, v_pages, q_starts, seq_lens, page_table);
  require(q && out, "q and out must not be null");
  require(q != out, "out must not be q");
  require(aligned(q, 2) && aligned(out, 2), "q and out must be aligned to their elements");
  const gie_paged_geom g = geom_of(p);
  const size_t need = gie_hip_paged_attention_workspace(&g);
  GIE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), StatusCode::kWorkspaceTooSmall,
              "PagedKv: workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(need) +
                  " needed");
  require(aligned(workspace, 16), "workspace must be 16-byte aligned");
  RoctxRange range("gie::PagedKv::attention");
  check_kernel_status(gie_hip_paged_attention(dtype_of(p.precision), &g, q, k_pages, v_pages, q_starts, seq_lens,
                                              page_table, out, workspace, workspace_bytes, stream),
                      "PagedKv::attention");
}

void rotary_tables(int max_positions, int rotary_dim, double base, double factor, int original_positions,
                   double magnitude, float* cos, float* sin) {
  require(max_positions > 0 && rotary_dim > 0 && rotary_dim % 2 == 0, "tables need positions and an even rotary_dim");
  require(base > 0 && factor >= 1 && original_positions >= 0 && std::isfinite(base) && std::isfinite(factor) &&
              std::isfinite(magnitude),
          "rotary base must be positive, factor at least 1 and original_positions not negative");
  require(cos && sin, "cos and sin must not be null");
  const int half = rotary_dim / 2;
  const double turn = 2 * std::acos(-1.0);
  for (int j = 0; j < half; ++j) {
    double f = std::pow(base, -2.0 * j / rotary_dim);
    if (original_positions == 0) {
      f /= factor;
    } else {
      const double turns = original_positions * f / turn;  // of this frequency over the original context
      const double keep = std::fmin(1.0, std::fmax(0.0, (turns - 1) / 3));
      f = keep * f + (1 - keep) * f / factor;
    }
    for (int p = 0; p < max_positions; ++p) {
      cos[size_t(p) * half + j] = float(std::cos(p * f) * magnitude);
      sin[size_t(p) * half + j] = float(std::sin(p * f) * magnitude);
    }
  }
}

}  // namespace gie
