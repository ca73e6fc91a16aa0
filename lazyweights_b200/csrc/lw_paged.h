// The paged key-value cache: geometry handle, launchers of the kernels that fill and read it (lw_paged.cu: appending with
// the position rotation, C ABI; lw_attend_token.cu, lw_attend_prompt.cu: attention).
#pragma once
#include <cuda.h>

#include "lw_gemv1.h"

namespace lw {

enum ElemType { kF16 = 0, kBF16 = 1, kF32 = 2 };

// The error word's bit for indexes that the kernels refused to follow (lw_kernel_error): a page outside the pool, a length
// beyond the page table's columns, a position beyond the rotation tables.
constexpr unsigned int kErrWordIndex = 2u;

// The two pools as the kernels see them; strides in elements, the head dimension is contiguous.
struct PagePool {
  void *k, *v;
  long long page_stride, head_stride, token_stride;
  int n_pages, Hk, page_size, Dh;
};

struct PagedCache {
  PagePool pool;
  ElemType type;
  int device = -1;   // -1: made without a CUDA device; nothing can be launched on it
  // Positions of a TMA box, a divisor of the page size: of 16 at a time (one token), of 128 (prompts); the maps of keys and values.
  int token_rows, prompt_rows;
  alignas(64) CUtensorMap token_k, token_v, prompt_k, prompt_v;
};

// Which positions belong to which rows: sequence b owns rows starts[b] .. starts[b + 1] - 1 (row b alone if starts is null),
// the last of its lens[b] positions; its pages are table[b * table_stride + 0 .. table_cols - 1].
struct Sequences {
  const int *starts, *lens, *table;
  long long table_stride;
  int n, table_cols;
};

// Arguments of attention: q and out rows [head][Dh], strides in elements.
struct AttendArgs {
  PagePool pool;
  Sequences seq;
  const void* q;
  void* out;
  long long q_token, q_head, out_token, out_head;
  int H, rows;        // query heads, rows of q
  int window;         // 0: none
  float scale;
  void* workspace;
  unsigned int* err;
};

// One token per sequence (lw_attend_token.cu) and packed prompts (lw_attend_prompt.cu); the workspace that calls of any size
// need on the current device.
int launch_attend_token(const PagedCache& cache, const AttendArgs& a, cudaStream_t st);
long long token_workspace(int head_dim, int group);
int launch_attend_prompt(const PagedCache& cache, const AttendArgs& a, cudaStream_t st);
long long prompt_workspace(int head_dim);

// Tensor maps in the 128-byte swizzle (boxes of 64 columns): queries [rows][H][Dh], boxes of box_tokens x box_heads rows; pages,
// boxes of box_rows positions of one head.  False where the driver does not offer the encoder or refuses the shape.
bool make_query_map(void* tensor_map, bool half, const void* base, int Dh, int H, int rows, long long head_stride, long long token_stride,
                    int box_heads, int box_tokens);
bool make_page_map(void* tensor_map, bool half, const void* base, const PagePool& pool, int box_rows);

}  // namespace lw
