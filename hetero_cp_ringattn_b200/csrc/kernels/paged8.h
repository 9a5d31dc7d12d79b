// Host interface of the paged 8-bit KV cache kernels: the step plan (block tables and slot maps
// from request lengths), the rotary append, attention over the cache and the gather back to bf16.
//
// A layer's cache is k, v [pages][Hkv][P][D] in 8 bits (e4m3 or int8) and one float scale per
// (page, KV head) for each of k and v; a stored code c stands for c * scale. The append makes
// power-of-two scales, so a code times its scale is exact in bf16 and a block whose scale grows
// is rescaled by an exponent shift; the readers take any positive float scale.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace hcp {
namespace kv8 {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum CodeType : int { kE4M3 = 0, kInt8 = 1 };

// One layer's cache; strides of the data in bytes (= elements), of the scales in elements.
struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  long page_stride, head_stride, token_stride;        // k and v alike
  long scale_page_stride, scale_head_stride;
  int pages, Hkv, P, D;
  int code;  // CodeType
};

// Limits of one plan: offsets of every row are kept in shared memory.
constexpr int kPlanMaxRows = 4096;

struct PlanArgs {
  const int* add;        // [R] tokens to add to each row; negative: release the row
  const int* kv_len;     // [R]
  int* table;            // [R][width] page ids, entries of new pages are written
  int* ring;             // [ring_size] free pages, FIFO between the two counters
  const long long* counters;  // [2] head, tail
  int R, width, P, ring_size, max_tokens, max_units;
  int shift;             // set by the launcher: log2 of a power-of-two P
  int* cu;               // [R + 1]
  int* row;              // [max_tokens]
  int* pos;              // [max_tokens]
  long long* slot;       // [max_tokens]
  int4* unit;            // [max_units] row, first token, tokens, first position
  int* kv_len_out;       // [R]   (may be kv_len)
  long long* counters_out;    // [2]   (may be counters)
  int* info;             // [4] tokens, units, pages taken, status
};
const char* plan_step(const PlanArgs& a, cudaStream_t s);

struct AppendArgs {
  const void* x;         // [T] rows of (H + 2 Hkv) heads of D, `dtype`
  int dtype;
  long row_stride;       // elements
  const float* cos_t;    // [max_pos][D / 2]
  const float* sin_t;
  int max_pos;
  const int* pos;        // [T]
  const int4* unit;      // [U]
  const int* table;      // [R][width]
  int T, H, U, R, width;
  Cache c;
  void* q_out;           // [T][H][D]
  int q_dtype;           // kBF16 or kF16
  int* status;
  int num_sms;
};
// Sets `launched` to the number of kernels.
const char* rope_append(const AppendArgs& a, cudaStream_t s, int* launched);

struct GatherArgs {
  Cache c;
  const int* table;      // [width] one row's pages
  int width, n;          // rows to gather
  void* k_out;           // [Hkv][cap][D] bf16
  void* v_out;
  long out_head_stride;  // elements
};
const char* gather(const GatherArgs& a, cudaStream_t s);

constexpr int kAttnMaxRows = 1024;  // requests of one attention call

struct AttnArgs {
  Cache c;
  const void* q;         // [T] rows of H heads of D
  int q_dtype;           // kBF16 or kF16 (the output's too)
  long q_stride, q_head_stride;
  const int* table;      // [B][width]
  const int* kv_len;     // [B]
  const int* cu;         // [B + 1] or null (one token a row)
  int B, T, H, width;
  int max_q;             // a request's most query tokens, for the choice of shapes (more are right, but slower)
  float scale;
  void* o;               // [T][H][D]
  float* lse;            // [H][T] or null
  void* workspace;
  int* status;
  int num_sms;
};
// Bytes of workspace of one call; 0 for an argument error (reported by attention()).
size_t attention_workspace(const AttnArgs& a);
const char* attention(const AttnArgs& a, cudaStream_t s);

}  // namespace kv8
}  // namespace hcp
