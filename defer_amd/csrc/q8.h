// q8.h -- the 8-bit operators' launches, shared by their C entry points
// (q8.hip) and the forward of an 8-bit model (defer_gpu.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/defer_gpu.h"
#include "q8_index.h"

// Sets the calling thread's defer_gpu_last_error; returns code.
int defer_gpu_fail_(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3), visibility("hidden")));

namespace q8 {

// One sequence's pages of one layer, where every sequence has its own.
struct SeqPages {
  int8_t *keys, *values;
  float *key_scale, *value_scale;
  uint32_t pages;  // page of a block: its index
};

struct Pages {
  int8_t *keys, *values;             // [pages][heads][64][dp], [pages][heads][dp][64]
  float *key_scale, *value_scale;    // [pages][heads][64]
  const int32_t* table;              // [sequences][width]
  uint32_t pages, heads, dp, width;
  const SeqPages* seqs;              // if set, in place of the pool and the table
  int64_t seq_layer;                 // ... and the layer to take in each (pages apart)
};
struct Rows {
  const int32_t *row_start, *kv_len;
  uint32_t sequences, rows, most_rows;
};

int quantize(uint32_t type, const void* x, int64_t x_stride, uint32_t rows, uint32_t n, int8_t* codes,
             float* scale, hipStream_t s);
int rms_norm(uint32_t type, const void* x, int64_t x_stride, const void* residual, int64_t r_stride,
             const void* weight, float eps, uint32_t rows, uint32_t n, void* sum, int64_t sum_stride,
             int8_t* codes, float* scale, hipStream_t s);
int linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
           const float* w_scale, uint32_t rows, uint32_t m, uint32_t k, uint32_t type, void* y,
           int64_t y_stride, hipStream_t s);
int kv_write(const Pages& p, const Rows& r, uint32_t type, const void* k, int64_t k_stride, const void* v,
             int64_t v_stride, uint32_t head_dim, hipStream_t s);
int kv_read(const Pages& p, const Rows& r, uint32_t type, void* k, void* v, uint32_t head_dim, hipStream_t s);

struct Attention {
  uint32_t type;
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  uint32_t heads, head_dim;
  float scale;
  uint32_t most_len;
  const uint8_t* hidden;  // [sequences][hidden_len], rows hidden_stride apart
  int64_t hidden_stride;
  uint32_t hidden_len;
  bool clear;  // zeros for the rows of no sequence
  const int32_t* parent;  // [rows], or NULL: rows are no tree
};
size_t attention_workspace(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t most_len);
int attention(const Pages& p, const Rows& r, const Attention& a, void* workspace, size_t workspace_bytes,
              hipStream_t s);
// ... of rows that are nodes of trees (a.parent).
size_t tree_attention_workspace(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t most_len);
int tree_attention(const Pages& p, const Rows& r, const Attention& a, void* workspace, size_t workspace_bytes,
                   hipStream_t s);

}  // namespace q8
