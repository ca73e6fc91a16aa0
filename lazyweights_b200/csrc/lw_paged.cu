// The paged key-value cache: its handle, the kernel that appends rotated keys and values, the C entry points.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>

#include "../../include/lwb200.h"
#include "lw_device.cuh"
#include "lw_host.h"
#include "lw_model.h"
#include "lw_paged.h"

namespace lw {

// ------------------------------------------------------------------------------------------------------ appending
//
// Row t of the fused product holds H query heads, Hk key heads and Hk value heads of Dh values.  At position p, with c and s
// row p of the rotation tables, the pair (a, b) = (x[i], x[i + R]) of a query or key head becomes (a c - b s, b c + a s) for
// i < R, values past 2 R are copied; queries go to q_out, keys and values to their page.  fp32 arithmetic, one rounding.
//
// Bound: the row read once, written once (2 R = Dh = 128, 32 + 2 x 8 heads: 24 KB + 12 KB a row from fp32); at a row
// or two, the chain of dependent loads starts -> length -> page.  Measured: 13555 such rows in 85 us, 5.96 TB/s, 91 % of a copy; one row 2.5 us.
//  * A block per row, whose fixed thread handles unit u (8 values: four pairs, or eight copied ones) of every n-th head, so the
//    tables are read once per thread, not once per head.  The row's values are requested before the block looks
//    its sequence up: the two latencies overlap.
//  * The sequence of a row is found by all threads of the block together (one or a few loads each), not by bisection (a
//    dozen dependent ones).
constexpr int kAppendThreads = 256, kAppendUnits = 4;   // units in flight per thread

struct AppendArgs {
  PagePool pool;
  Sequences seq;
  const void* x;
  void* q;
  const float *cosv, *sinv;
  long long x_row, q_token, q_head;
  int H, rows, rope_rows, R;
  int per_head, heads_per_step;   // Dh / 8; heads one step of the block covers
  int vec;                        // rows and tables lie on 16-byte boundaries
  unsigned int* err;
};

struct Four {
  float v[4];
};

template <typename T>
__device__ __forceinline__ Four read4(const T* p, bool vec) {
  Four r;
  if (!vec) {
    for (int i = 0; i < 4; ++i) r.v[i] = static_cast<float>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    r.v[0] = f.x, r.v[1] = f.y, r.v[2] = f.z, r.v[3] = f.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
    for (int i = 0; i < 4; ++i) r.v[i] = static_cast<float>(e[i]);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void write4(T* p, const Four& f) {
  uint2 u;
  T* e = reinterpret_cast<T*>(&u);
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) e[i] = __float2half_rn(f.v[i]);
    else e[i] = __float2bfloat16_rn(f.v[i]);
  }
  *reinterpret_cast<uint2*>(p) = u;
}

template <typename TX, typename T>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(const __grid_constant__ AppendArgs A) {
  __shared__ int s_seq, s_pos;
  __shared__ long long s_slot;
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x, Dh = A.pool.Dh, heads = A.H + 2 * A.pool.Hk;
  const int u = tid % A.per_head, head0 = tid / A.per_head;
  const bool rotated = u < A.R / 4;
  const int first = rotated ? 4 * u : 2 * A.R + 8 * (u - A.R / 4), second = rotated ? first + A.R : first + 4;   // of a query or key head
  const TX* x = static_cast<const TX*>(A.x) + row * A.x_row;
  Four lo[kAppendUnits], hi[kAppendUnits];
  auto fetch = [&](int base) {
#pragma unroll
    for (int k = 0; k < kAppendUnits; ++k) {
      const int head = base + k * A.heads_per_step;
      if (head0 < A.heads_per_step && head < heads) {
        const bool value = head >= A.H + A.pool.Hk;
        const TX* p = x + head * Dh;
        lo[k] = read4(p + (value ? 8 * u : first), A.vec);
        hi[k] = read4(p + (value ? 8 * u + 4 : second), A.vec);
      }
    }
  };
  fetch(head0);
  if (tid == 0) s_seq = -1;
  __syncthreads();
  if (!A.seq.starts) {
    if (tid == 0 && row < A.seq.n) s_seq = row;
  } else {
    for (int b = tid; b < A.seq.n; b += kAppendThreads)
      if (A.seq.starts[b] <= row && row < A.seq.starts[b + 1]) s_seq = b;
  }
  __syncthreads();
  if (tid == 0) {
    const int b = s_seq;
    int pos = -1;
    if (b >= 0) pos = A.seq.lens[b] - (A.seq.starts ? min(A.seq.starts[b + 1], A.rows) - row : 1);
    if (pos >= 0) {
      const int column = pos / A.pool.page_size;
      const int page = column < A.seq.table_cols ? A.seq.table[b * A.seq.table_stride + column] : -1;
      if (page < 0 || page >= A.pool.n_pages || pos >= A.rope_rows) {
        atomicOr(A.err, kErrWordIndex);
        pos = -1;
      } else {
        s_slot = page * A.pool.page_stride + (pos - column * A.pool.page_size) * A.pool.token_stride;
      }
    }
    s_pos = pos;
  }
  __syncthreads();
  const int pos = s_pos;
  if (pos < 0 || head0 >= A.heads_per_step) return;   // a row of no sequence, before position 0, or refused
  Four c, s;
  if (rotated) {
    c = read4(A.cosv + static_cast<long long>(pos) * A.R + 4 * u, A.vec);
    s = read4(A.sinv + static_cast<long long>(pos) * A.R + 4 * u, A.vec);
  } else {
    for (int i = 0; i < 4; ++i) c.v[i] = 1.f, s.v[i] = 0.f;
  }
  for (int base = head0; base < heads; base += kAppendUnits * A.heads_per_step) {
    if (base != head0) fetch(base);
#pragma unroll
    for (int k = 0; k < kAppendUnits; ++k) {
      const int head = base + k * A.heads_per_step;
      if (head >= heads) break;
      const bool value = head >= A.H + A.pool.Hk;
      T* dst;
      if (head < A.H) dst = static_cast<T*>(A.q) + row * A.q_token + head * A.q_head;
      else if (!value) dst = static_cast<T*>(A.pool.k) + s_slot + (head - A.H) * A.pool.head_stride;
      else dst = static_cast<T*>(A.pool.v) + s_slot + (head - A.H - A.pool.Hk) * A.pool.head_stride;
      if (!value && rotated) {
        Four a, b;
        for (int i = 0; i < 4; ++i) {
          a.v[i] = lo[k].v[i] * c.v[i] - hi[k].v[i] * s.v[i];
          b.v[i] = hi[k].v[i] * c.v[i] + lo[k].v[i] * s.v[i];
        }
        lo[k] = a;
        hi[k] = b;
      }
      write4(dst + (value ? 8 * u : first), lo[k]);
      write4(dst + (value ? 8 * u + 4 : second), hi[k]);
    }
  }
}

template <typename T>
static auto append_kernel(ElemType x) {
  return x == kF32 ? k_paged_append<float, T> : x == kF16 ? k_paged_append<__half, T> : k_paged_append<__nv_bfloat16, T>;
}

static int launch_append(ElemType x, ElemType type, const AppendArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows);
  cfg.blockDim = dim3(kAppendThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, type == kF16 ? append_kernel<__half>(x) : append_kernel<__nv_bfloat16>(x), a);
  return note_launch("k_paged_append");
}

// ------------------------------------------------------------------------------------------------------- the handle

static int refuse(const char* what, const char* why) {
  set_error("%s: %s", what, why);
  return kErrArg;
}

static bool aligned(const void* p, unsigned int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// The current device, if it is the cache's.
static int check_cache_device(const PagedCache* c) {
  int dev = -1;
  if (c->device < 0) {
    set_error("the cache was created without a CUDA device: this library has no CPU path for GPU entry points");
    return kErrNoDevice;
  }
  if (cudaGetDevice(&dev) != cudaSuccess) return cuda_fail("cudaGetDevice", cudaGetLastError());
  if (dev != c->device) {
    set_error("the cache was created on device %d but the current device is %d", c->device, dev);
    return kErrArg;
  }
  return kOk;
}

// starts may be null (a row per sequence)
static int check_sequences(const char* what, const int* starts, const int* lens, const int* table, int n_seqs, int table_cols,
                           long long table_stride, int n_rows, bool starts_needed) {
  if (n_seqs < 1 || n_rows < 1) return refuse(what, "needs at least one sequence and one row");
  if (n_rows > 1 << 30) return refuse(what, "at most 2^30 rows");   // positions of rows before position 0 are counted in 32 bits
  if (!lens || !table || (starts_needed && !starts)) return refuse(what, "null pointer");
  if (table_cols < 1 || table_stride < table_cols) return refuse(what, "the page table has no columns, or rows closer than that");
  if (!starts && n_rows < n_seqs) return refuse(what, "fewer rows than sequences");
  return kOk;
}

static int check_rows(const char* what, const void* p, long long token, long long head, int n_heads, int Dh, int rows) {
  if (!p) return refuse(what, "null pointer");
  if (!aligned(p, 16) || token % 8 || head % 8) return refuse(what, "queries and results must lie on 16-byte boundaries, row by row and head by head");
  if (head < Dh || token < Dh || (rows > 1 && n_heads > 1 && token < head * n_heads && head < token * rows))
    return refuse(what, "strides of queries or results make rows overlap");
  return kOk;
}

}  // namespace lw

using namespace lw;

extern "C" {

void* lw_cache_create(void* k_pages, void* v_pages, int type, int n_pages, int n_kv_heads, int page_size, int head_dim,
                      long long page_stride, long long head_stride, long long token_stride) {
  const char* what = "lw_cache_create";
  int rc = kOk;
  if (!k_pages || !v_pages) rc = refuse(what, "null pointer");
  else if (type != kF16 && type != kBF16) rc = refuse(what, "pages hold fp16 or bf16");
  else if (n_pages < 1 || n_kv_heads < 1) rc = refuse(what, "needs at least one page and one head");
  else if (page_size < 8 || page_size % 8 || page_size > 65536) rc = refuse(what, "the page size must be a multiple of 8, at most 65536");
  else if (head_dim < 8 || head_dim % 8 || head_dim > 128) rc = refuse(what, "head_dim must be a multiple of 8, at most 128");
  else if (!aligned(k_pages, 16) || !aligned(v_pages, 16)) rc = refuse(what, "the pools must lie on 16-byte boundaries");
  else {
    // an axis of one entry is never stepped along
    if (n_pages == 1) page_stride = 8;
    if (n_kv_heads == 1) head_stride = 8;
    const long long limit = 1ll << 38;   // elements a stride may span: what a tensor map takes
    if (page_stride < 8 || head_stride < 8 || token_stride < head_dim || page_stride % 8 || head_stride % 8 || token_stride % 8 ||
        page_stride >= limit || head_stride >= limit || token_stride >= limit)
      rc = refuse(what, "strides must be positive multiples of 8 elements");
  }
  if (rc) {
    note_status(rc);
    return nullptr;
  }
  PagedCache* c = new (std::nothrow) PagedCache;
  if (!c) {
    set_error("%s: out of host memory", what);
    note_status(kErrGeneric);
    return nullptr;
  }
  c->pool = {k_pages, v_pages, page_stride, head_stride, token_stride, n_pages, n_kv_heads, page_size, head_dim};
  c->type = static_cast<ElemType>(type);
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0 || cudaGetDevice(&c->device) != cudaSuccess) {
    cudaGetLastError();
    c->device = -1;
  }
  c->token_rows = page_size % 16 ? 8 : 16;
  c->prompt_rows = std::min(128, page_size & -page_size);
  const bool half = type == kF16;
  if (c->device >= 0 && !(make_page_map(&c->token_k, half, k_pages, c->pool, c->token_rows) && make_page_map(&c->token_v, half, v_pages, c->pool, c->token_rows) &&
                          make_page_map(&c->prompt_k, half, k_pages, c->pool, c->prompt_rows) && make_page_map(&c->prompt_v, half, v_pages, c->pool, c->prompt_rows))) {
    delete c;
    note_status(refuse(what, "the driver refused a tensor map over the pools"));
    return nullptr;
  }
  note_status(kOk);
  return c;
}

void lw_cache_destroy(void* cache) { delete static_cast<PagedCache*>(cache); }

int lw_cache_append(void* cache, const void* qkv, int qkv_type, long long row_stride, int n_rows, int n_heads, const float* cos_table,
                    const float* sin_table, int rope_rows, int rope_half, const int* starts, const int* lens, const int* table,
                    int n_seqs, int table_cols, long long table_stride, void* q, long long q_token_stride, long long q_head_stride,
                    void* stream) {
  const char* what = "lw_cache_append";
  const PagedCache* c = static_cast<const PagedCache*>(cache);
  if (!c || !qkv || !cos_table || !sin_table) return refuse(what, "null pointer");
  if (qkv_type != kF16 && qkv_type != kBF16 && qkv_type != kF32) return refuse(what, "rows are fp16, bf16 or fp32");
  if (n_heads < 1 || n_heads % c->pool.Hk) return refuse(what, "the query heads must be a multiple of the kv heads");
  if (const int rc = check_sequences(what, starts, lens, table, n_seqs, table_cols, table_stride, n_rows, false)) return rc;
  if (const int rc = check_rows(what, q, q_token_stride, q_head_stride, n_heads, c->pool.Dh, n_rows)) return rc;
  if (rope_rows < 1 || rope_half < 4 || rope_half % 4 || 2 * rope_half > c->pool.Dh)
    return refuse(what, "the rotation tables must have a multiple of 4 columns, at most half of head_dim");
  const int size = qkv_type == kF32 ? 4 : 2;
  if (row_stride < static_cast<long long>(n_heads + 2 * c->pool.Hk) * c->pool.Dh || !aligned(qkv, size))
    return refuse(what, "the rows are shorter than their heads, or at an address that their type does not allow");
  if (!aligned(cos_table, 4) || !aligned(sin_table, 4)) return refuse(what, "the rotation tables lie at an odd address");
  if (const int rc = check_cache_device(c)) return rc;
  AppendArgs a = {};
  a.pool = c->pool;
  a.seq = {starts, lens, table, table_stride, n_seqs, table_cols};
  a.x = qkv;
  a.q = q;
  a.cosv = cos_table;
  a.sinv = sin_table;
  a.x_row = row_stride;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.H = n_heads;
  a.rows = n_rows;
  a.rope_rows = rope_rows;
  a.R = rope_half;
  a.per_head = c->pool.Dh / 8;
  a.heads_per_step = kAppendThreads / a.per_head;
  a.vec = aligned(qkv, 16) && row_stride * size % 16 == 0 && aligned(cos_table, 16) && aligned(sin_table, 16);
  if (!(a.err = error_word())) return cuda_fail("error word", cudaGetLastError());
  return launch_append(static_cast<ElemType>(qkv_type), c->type, a, static_cast<cudaStream_t>(stream));
}

static int attend(const char* what, void* cache, const void* q, long long q_token_stride, long long q_head_stride, int n_rows, int n_heads,
                  const int* starts, const int* lens, const int* table, int n_seqs, int table_cols, long long table_stride, float scale,
                  int window, void* out, long long out_token_stride, long long out_head_stride, void* workspace, long long workspace_bytes,
                  void* stream, bool prompt) {
  const PagedCache* c = static_cast<const PagedCache*>(cache);
  if (!c) return refuse(what, "null pointer");
  if (n_heads < 1 || n_heads % c->pool.Hk) return refuse(what, "the query heads must be a multiple of the kv heads");
  if (const int rc = check_sequences(what, starts, lens, table, n_seqs, table_cols, table_stride, n_rows, prompt)) return rc;
  if (const int rc = check_rows(what, q, q_token_stride, q_head_stride, n_heads, c->pool.Dh, n_rows)) return rc;
  if (const int rc = check_rows(what, out, out_token_stride, out_head_stride, n_heads, c->pool.Dh, n_rows)) return rc;
  if (n_heads / c->pool.Hk > 128) return refuse(what, "at most 128 query heads per kv head");
  if (!std::isfinite(scale) || window < 0) return refuse(what, "the scale must be finite, the window not negative");
  const long long need = lw_cache_workspace(cache, n_heads, prompt);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return refuse(what, "the workspace is too small (lw_cache_workspace), or not on a 16-byte boundary");
  if (const int rc = check_cache_device(c)) return rc;
  AttendArgs a = {};
  a.pool = c->pool;
  a.seq = {starts, lens, table, table_stride, n_seqs, table_cols};
  a.q = q;
  a.out = out;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.H = n_heads;
  a.rows = n_rows;
  a.window = window;
  a.scale = scale;
  a.workspace = workspace;
  if (!(a.err = error_word())) return cuda_fail("error word", cudaGetLastError());
  return (prompt ? launch_attend_prompt : launch_attend_token)(*c, a, static_cast<cudaStream_t>(stream));
}

long long lw_cache_workspace(void* cache, int n_heads, int prompt) {
  const PagedCache* c = static_cast<const PagedCache*>(cache);
  if (!c || n_heads < 1 || n_heads % c->pool.Hk) return refuse("lw_cache_workspace", "bad argument");
  return prompt ? prompt_workspace(c->pool.Dh) : token_workspace(c->pool.Dh, n_heads / c->pool.Hk);
}

int lw_cache_attend(void* cache, const void* q, long long q_token_stride, long long q_head_stride, int n_seqs, int n_heads, const int* lens,
                    const int* table, int table_cols, long long table_stride, float scale, int window, void* out,
                    long long out_token_stride, long long out_head_stride, void* workspace, long long workspace_bytes, void* stream) {
  return attend("lw_cache_attend", cache, q, q_token_stride, q_head_stride, n_seqs, n_heads, nullptr, lens, table, n_seqs, table_cols,
                table_stride, scale, window, out, out_token_stride, out_head_stride, workspace, workspace_bytes, stream, false);
}

int lw_cache_attend_prompt(void* cache, const void* q, long long q_token_stride, long long q_head_stride, int n_rows, int n_heads,
                           const int* starts, const int* lens, const int* table, int n_seqs, int table_cols, long long table_stride,
                           float scale, int window, void* out, long long out_token_stride, long long out_head_stride, void* workspace,
                           long long workspace_bytes, void* stream) {
  return attend("lw_cache_attend_prompt", cache, q, q_token_stride, q_head_stride, n_rows, n_heads, starts, lens, table, n_seqs, table_cols,
                table_stride, scale, window, out, out_token_stride, out_head_stride, workspace, workspace_bytes, stream, true);
}

}  // extern "C"
