// Attention of one new token per sequence over the paged cache, split over the sequences' lengths.
//
//   o[h] = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = scale log2(e) q[h] . k_j,   m = max_j x_j
//
// in one pass with a running m; partial (m, l = sum 2^(x - m), O = sum 2^(x - m) v) of disjoint sets of positions join exactly:
// rescale to the larger m, add.
//
// Bound: HBM.  Every key and value is read once (4 Dh bytes per position and kv head) and meets the `group` query heads of its
// kv head: 2 group multiply-adds per element, which the SIMT pipes could not do beside the stream from four heads on, and
// m16n8k16 tensor-core instructions do in a tenth of the time that the bytes take.  So:
//  * The query heads are the N = 8 columns of the instruction (one or two instructions wide; wider groups take several
//    passes over the keys), positions its 16 rows, then the rows of its reduction: S^T = K q^T, O^T = V^T P^T.  Swapped the other way
//    round heads would fill 16 rows, mostly with zeros.  P^T gets from the accumulator layout to the operand's by two 8 x 8 transposes.
//  * A warp is a worker of its own: every fourth piece of 16 positions of the block's share, staged by its own TMA loads in its own ring
//    (192 KB per SM in flight with two blocks of four warps; about 45 KB would cover the latency at full bandwidth), its own m, l, O.  Warps meet
//    once per sequence and kv head.
//  * Shares: units of 64 positions of a kv head, numbered sequence by sequence, head by head; every block takes the same
//    number, whatever the lengths, which it reads on the device.  What a block begins or ends in the middle of goes to the workspace
//    and is joined, in order, by k_token_join.
//  * Positions outside the sequence or the window: scores replaced by -inf, values zeroed in shared memory (0 x NaN is NaN).
//  * Rounding: scores, m, l, O in 32 bits, P in the cache's type for the tensor core (half a step of it, independent per position).
#include <cuda.h>

#include <algorithm>

#include "lw_attend.cuh"
#include "lw_attend_plan.h"

namespace lw {

constexpr int kTokenWarps = 4, kTokenThreads = kTokenWarps * 32;
constexpr int kUnit = 16 * kTokenWarps;   // positions of a unit
constexpr int kTokenBlocksPerSm = 2;

struct TokenNote {
  int b, h, begins, ends;   // of the block's first piece: sequence, head slot, whether it holds the first and the last unit
};

struct TokenArgs {
  AttendArgs a;
  int group, chunks;        // query heads per kv head; passes over the keys: ceil(group / (8 NT))
  int box_rows;             // 16, or 8 where pages are odd multiples of 8
  int cap;
  uint32_t wait_limit;
  TokenNote* notes;
  float* partial;           // [block][piece][8 NT heads]: m, l, O[DP]
};

template <typename T>
__device__ __forceinline__ void mma_16n8k16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Positions lo .. len - 1 of a sequence, units first .. last - 1.
struct TokenSeq {
  int lo, len, first, last;
};
__device__ __forceinline__ TokenSeq token_seq(const TokenArgs& P, int b) {
  TokenSeq s;
  s.len = min(max(P.a.seq.lens[b], 0), P.cap);
  s.lo = P.a.window > 0 ? max(0, s.len - P.a.window) : 0;
  s.first = s.lo / kUnit;
  s.last = (s.len + kUnit - 1) / kUnit;
  return s;
}

// Where a walk over the block's share stands: unit t of head slot h (kv head, pass) of sequence b.
struct TokenWalk {
  int b, h, t;
  long long left;
  TokenSeq s;
  __device__ __forceinline__ void step(const TokenArgs& P, int slots) {
    --left;
    if (++t < s.last) return;
    if (++h == slots) {
      h = 0;
      if (left > 0) {
        do s = token_seq(P, ++b); while (s.last <= s.first && b < P.a.seq.n - 1);
      }
    }
    t = s.first;
  }
};

template <int DP, int NT>
struct TokenSizes {
  static constexpr int kHalves = DP / 64;
  static constexpr uint32_t kTile = 16 * DP * 2;                 // bytes of 16 keys, or values
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr uint32_t kWarp = kStages * 2 * kTile;
  static constexpr int kRow = DP + 4;                            // floats of a head's row in the meeting place: conflict-free
  static constexpr size_t kSmem = 1024 + kTokenWarps * kWarp + 8 * NT * kRow * 4;
  static constexpr int kPartHead = DP + 4;                       // m, l, 2 unused, O: 16-byte aligned
  static constexpr size_t kPartial = static_cast<size_t>(8) * NT * kPartHead;
};

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kTokenThreads, kTokenBlocksPerSm)
    k_attend_token(const __grid_constant__ CUtensorMap KM, const __grid_constant__ CUtensorMap VM, const __grid_constant__ TokenArgs P) {
  using Z = TokenSizes<DP, NT>;
  constexpr int kSteps = DP / 16, kStages = Z::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kTokenWarps][kStages];
  __shared__ long long s_scan[kTokenWarps], s_left;
  __shared__ int s_start[3];
  __shared__ float s_m[kTokenWarps][8 * NT], s_l[kTokenWarps][8 * NT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = ((smem_addr(smem_raw) + 1023u) & ~1023u) + warp * Z::kWarp;
  uint8_t* const mine_raw = smem_raw + (base - smem_addr(smem_raw));
  float* const meet = reinterpret_cast<float*>(smem_raw + (((smem_addr(smem_raw) + 1023u) & ~1023u) - smem_addr(smem_raw)) + kTokenWarps * Z::kWarp);
  if (lane < kStages) mbar_init(smem_addr(&full[warp][lane]), 1);
  __syncwarp();
  pdl_trigger();
  pdl_wait();

  // ---- the block's share
  const int slots = P.a.pool.Hk * P.chunks, n_seqs = P.a.seq.n;
  auto units_of = [&](int b) -> long long {
    if (b >= n_seqs) return 0;
    const TokenSeq s = token_seq(P, b);
    if (blockIdx.x == 0 && P.a.seq.lens[b] > P.cap) atomicOr(P.a.err, kErrWordIndex);
    return static_cast<long long>(max(0, s.last - s.first)) * slots;
  };
  auto block_sum = [&](long long v, long long& before) -> long long {
    long long inc = v;
    for (int o = 1; o < 32; o <<= 1) {
      const long long w = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += w;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long front = 0, all = 0;
    for (int k = 0; k < kTokenWarps; ++k) {
      if (k < warp) front += s_scan[k];
      all += s_scan[k];
    }
    __syncthreads();
    before = front + inc - v;
    return all;
  };
  long long units = 0, before = 0;
  for (int b0 = 0; b0 < n_seqs; b0 += kTokenThreads) units += block_sum(units_of(b0 + tid), before);
  const int blocks = static_cast<int>(min(static_cast<long long>(gridDim.x), units));
  const bool busy = static_cast<int>(blockIdx.x) < blocks;
  const long long u0 = busy ? share(units, blockIdx.x, blocks) : 0, u1 = busy ? share(units, blockIdx.x + 1, blocks) : 0;
  // sequences without positions: zeros
  for (int b = blockIdx.x; b < n_seqs; b += gridDim.x) {
    if (P.a.seq.lens[b] > 0) continue;
    const int per_head = P.a.pool.Dh / 8;
    for (int i = tid; i < P.a.H * per_head; i += kTokenThreads)
      *reinterpret_cast<uint4*>(static_cast<T*>(P.a.out) + b * P.a.out_token + (i / per_head) * P.a.out_head + (i % per_head) * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
  if (!busy) {
    if (tid == 0) P.notes[blockIdx.x] = {0, 0, 1, 1};
    return;
  }
  long long front = 0;
  for (int b0 = 0; b0 < n_seqs; b0 += kTokenThreads) {
    const long long mine = units_of(b0 + tid);
    const long long all = block_sum(mine, before);
    if (u0 >= front + before && u0 < front + before + mine) {
      const TokenSeq s = token_seq(P, b0 + tid);
      const int rest = static_cast<int>(u0 - front - before), per_slot = s.last - s.first;
      s_start[0] = b0 + tid;
      s_start[1] = rest / per_slot;
      s_start[2] = s.first + rest % per_slot;
    }
    front += all;
    if (front > u0) break;
  }
  __syncthreads();
  TokenWalk at;
  at.b = s_start[0];
  at.h = s_start[1];
  at.t = s_start[2];
  at.left = u1 - u0;
  at.s = token_seq(P, at.b);

  // ---- loads: this warp's 16 positions of the next unit that holds any for it
  TokenWalk ahead = at;
  int load_stage = 0;
  const int per_half = 16 / P.box_rows, boxes = per_half * Z::kHalves;   // of the keys; as many of the values
  auto load_next = [&]() {
    int p0 = 0;
    while (ahead.left > 0) {
      p0 = ahead.t * kUnit + warp * 16;
      if (p0 < ahead.s.len && p0 + 16 > ahead.s.lo) break;
      ahead.step(P, slots);
    }
    if (ahead.left <= 0) return;
    const int kv = lane / boxes, n = lane % boxes, half = n / per_half, row = (n % per_half) * P.box_rows;
    const int pos = p0 + row;
    const bool mine = kv < 2 && pos < ahead.s.len && pos + P.box_rows > ahead.s.lo;
    const uint32_t bar = smem_addr(&full[warp][load_stage]);
    const int count = __popc(__ballot_sync(0xffffffffu, mine));
    int page = 0, in_page = 0;
    if (mine) {
      const int column = pos / P.a.pool.page_size;
      page = P.a.seq.table[ahead.b * P.a.seq.table_stride + column];
      in_page = pos - column * P.a.pool.page_size;
      if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(P.a.pool.n_pages)) {   // the tensor map's bounds fill it with zeros
        atomicOr(P.a.err, kErrWordIndex);
        page = P.a.pool.n_pages;
      }
    }
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count * P.box_rows * 128) : "memory");
    __syncwarp();
    if (mine)
      tma_load_4d(base + (load_stage * 2 + kv) * Z::kTile + half * 2048 + row * 128, kv ? &VM : &KM, 64 * half, in_page, ahead.h / P.chunks, page, bar);
    if (++load_stage == kStages) load_stage = 0;
    ahead.step(P, slots);
  };
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) load_next();

  // ---- the share, piece by piece: units of one sequence and head slot
  const float c = P.a.scale * 1.4426950408889634f;
  int stage = 0;
  uint32_t parity = 0;
  bool first = true;
  while (at.left > 0) {
    const int b = at.b, h = at.h, t_begin = at.t;
    const TokenSeq s = at.s;
    const int t_end = static_cast<int>(min(static_cast<long long>(s.last), t_begin + at.left));
    const int head0 = (h / P.chunks) * P.group + (h % P.chunks) * 8 * NT, heads = min(8 * NT, P.group - (h % P.chunks) * 8 * NT);
    // queries as B operands: column lane / 4, rows 2 (lane % 4) and the next, and eight further
    uint32_t qf[NT][kSteps][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int head = n * 8 + (lane >> 2);
      const T* q = static_cast<const T*>(P.a.q) + b * P.a.q_token + (head0 + head) * P.a.q_head;
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = k * 16 + e * 8 + (lane & 3) * 2;
          qf[n][k][e] = head < heads && d < P.a.pool.Dh ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
    }
    float m[NT][2], l[NT][2], o[NT][kSteps][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][k][i] = 0.f;
    }
#pragma unroll 1
    for (int t = t_begin; t < t_end; ++t) {
      const int p0 = t * kUnit + warp * 16;
      if (p0 >= s.len || p0 + 16 <= s.lo) continue;
      (void)mbar_wait(smem_addr(&full[warp][stage]), parity, P.a.err, P.wait_limit);
      __syncwarp();
      const uint32_t ks = base + stage * 2 * Z::kTile, vs = ks + Z::kTile;
      const int v0 = max(0, s.lo - p0), v1 = min(16, s.len - p0);
      const bool cut = v0 > 0 || v1 < 16;
      if (cut) {
        uint8_t* dst = mine_raw + (vs - base);
        for (int i = lane; i < 16 * 8 * Z::kHalves; i += 32) {
          const int row = (i >> 3) & 15;
          if (row < v0 || row >= v1) *reinterpret_cast<uint4*>(dst + (i >> 7) * 2048 + row * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the stage is loaded again
        __syncwarp();
      }
      // S^T: rows positions, columns heads
      float sc[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][0][i] = sc[n][1][i] = 0.f;
      {
        const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t a[4];
          load_matrices(a, ks + (k >> 2) * 2048 + row * 128 + ((((k & 3) * 2 + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16n8k16<T>(sc[n][k & 1], a, qf[n][k][0], qf[n][k][1]);
        }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (lane >> 2) + (i >> 1) * 8;
          x[i] = row >= v0 && row < v1 ? (sc[n][0][i] + sc[n][1][i]) * c : -INFINITY;
        }
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(x[e], x[2 + e]);
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float m2 = fmaxf(m[n][e], mx), ref = m2 == -INFINITY ? 0.f : m2;
          alpha[e] = exp2_fast(m[n][e] - ref);
          m[n][e] = m2;
          x[e] = exp2_fast(x[e] - ref);
          x[2 + e] = exp2_fast(x[2 + e] - ref);
          l[n][e] = l[n][e] * alpha[e] + x[e] + x[2 + e];
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][k][i] *= alpha[i & 1];
        }
        pf[n][0] = transpose_8x8(pack2<T>(x[0], x[1]));
        pf[n][1] = transpose_8x8(pack2<T>(x[2], x[3]));
      }
      {
        const int row = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t a[4];
          load_matrices_transposed(a, vs + (k >> 2) * 2048 + row * 128 + ((((k & 3) * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16n8k16<T>(o[n][k], a, pf[n][0], pf[n][1]);
        }
      }
      __syncwarp();
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1u;
      }
      load_next();
    }
    // ---- the warps meet
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        if (lane < 4) {
          s_m[warp][n * 8 + lane * 2 + e] = m[n][e];
          s_l[warp][n * 8 + lane * 2 + e] = l[n][e];
        }
      }
    __syncthreads();
    float factor[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
        for (int w = 0; w < kTokenWarps; ++w) top = fmaxf(top, s_m[w][n * 8 + (lane & 3) * 2 + e]);
        factor[n][e] = m[n][e] == -INFINITY ? 0.f : exp2_fast(m[n][e] - top);
      }
    for (int w = 0; w < kTokenWarps; ++w) {   // in turn: the sum has one order
      if (warp == w) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float* p = meet + (n * 8 + (lane & 3) * 2 + (i & 1)) * Z::kRow + k * 16 + (lane >> 2) + (i >> 1) * 8;
              const float v = l[n][i & 1] == 0.f ? 0.f : o[n][k][i] * factor[n][i & 1];
              *p = w ? *p + v : v;
            }
      }
      __syncthreads();
    }
    const bool begins = t_begin == s.first, ends = t_end == s.last;
    float* part = P.partial + (static_cast<size_t>(blockIdx.x) * 2 + (begins ? 1 : 0)) * Z::kPartial;
    const int per_head = P.a.pool.Dh / 8;
    for (int i = tid; i < heads * per_head; i += kTokenThreads) {
      const int head = i / per_head, d = (i % per_head) * 8;
      float top = -INFINITY, total = 0.f;
      for (int w = 0; w < kTokenWarps; ++w) top = fmaxf(top, s_m[w][head]);
      for (int w = 0; w < kTokenWarps; ++w) total += s_m[w][head] == -INFINITY ? 0.f : s_l[w][head] * exp2_fast(s_m[w][head] - top);
      const float4 lo4 = *reinterpret_cast<const float4*>(meet + head * Z::kRow + d), hi4 = *reinterpret_cast<const float4*>(meet + head * Z::kRow + d + 4);
      if (begins && ends) {
        const float f = 1.f / total;
        *reinterpret_cast<uint4*>(static_cast<T*>(P.a.out) + b * P.a.out_token + (head0 + head) * P.a.out_head + d) =
            make_uint4(pack2<T>(lo4.x * f, lo4.y * f), pack2<T>(lo4.z * f, lo4.w * f), pack2<T>(hi4.x * f, hi4.y * f), pack2<T>(hi4.z * f, hi4.w * f));
      } else {
        float* dst = part + head * Z::kPartHead;
        if (d == 0) *reinterpret_cast<float2*>(dst) = make_float2(top, total);
        *reinterpret_cast<float4*>(dst + 4 + d) = lo4;
        *reinterpret_cast<float4*>(dst + 8 + d) = hi4;
      }
    }
    if (first && tid == 0) P.notes[blockIdx.x] = {b, h, begins, ends};
    first = false;
    __syncthreads();   // the meeting place is read before the next piece fills it
    at.left -= t_end - t_begin - 1;
    at.t = t_end - 1;
    at.step(P, slots);
  }
}

// Block c joins what the blocks before and from c on left of the piece that block c continued, if it is the first to continue it.
constexpr int kJoinMax = 64;   // pieces whose weights are held at a time
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kTokenThreads) k_token_join(const __grid_constant__ TokenArgs P, int blocks) {
  using Z = TokenSizes<DP, NT>;
  __shared__ float s_w[kJoinMax][8 * NT], s_top[8 * NT], s_total[8 * NT];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x + 1, tid = threadIdx.x;
  const TokenNote n = P.notes[c];
  if (n.begins) return;
  const TokenNote prev = P.notes[c - 1];
  if (!prev.begins && !prev.ends) return;
  int last = c;
  while (!P.notes[last].ends && last + 1 < blocks) ++last;
  const int head0 = (n.h / P.chunks) * P.group + (n.h % P.chunks) * 8 * NT, heads = min(8 * NT, P.group - (n.h % P.chunks) * 8 * NT);
  auto piece = [&](int k, int head) { return P.partial + (static_cast<size_t>(k) * 2 + (k < c ? 1 : 0)) * Z::kPartial + head * Z::kPartHead; };
  const int first = c - 1, count = last - first + 1;
  if (tid < heads * 8) {   // eight threads of a head
    const int head = tid >> 3;
    float top = -INFINITY, total = 0.f;
    for (int k = tid & 7; k < count; k += 8) top = fmaxf(top, piece(first + k, head)[0]);
    const int there = min(32, heads * 8 - (tid & ~31));   // threads of this warp that are here
    const unsigned int who = there == 32 ? 0xffffffffu : (1u << there) - 1u;
    __syncwarp(who);
    for (int d = 1; d < 8; d <<= 1) top = fmaxf(top, __shfl_xor_sync(who, top, d));
    for (int k = tid & 7; k < count; k += 8) {
      const float2 ml = *reinterpret_cast<const float2*>(piece(first + k, head));
      total += ml.x == -INFINITY ? 0.f : ml.y * exp2_fast(ml.x - top);
    }
    for (int d = 1; d < 8; d <<= 1) total += __shfl_xor_sync(who, total, d);
    if ((tid & 7) == 0) {
      s_top[head] = top;
      s_total[head] = total;
    }
  }
  __syncthreads();
  const int per_head = P.a.pool.Dh / 4;
  for (int i0 = 0; i0 < heads * per_head; i0 += kTokenThreads) {
    const int i = i0 + tid, head = i / per_head, d = (i % per_head) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < count; k0 += kJoinMax) {
      __syncthreads();
      for (int j = tid; j < min(kJoinMax, count - k0) * heads; j += kTokenThreads) {
        const float m = piece(first + k0 + j / heads, j % heads)[0];
        s_w[j / heads][j % heads] = m == -INFINITY ? 0.f : exp2_fast(m - s_top[j % heads]);
      }
      __syncthreads();
      if (i < heads * per_head) {
#pragma unroll 8
        for (int k = 0; k < min(kJoinMax, count - k0); ++k) {
          const float f = s_w[k][head];
          const float4 v = *reinterpret_cast<const float4*>(piece(first + k0 + k, head) + 4 + d);
          o.x = fmaf(f, v.x, o.x);
          o.y = fmaf(f, v.y, o.y);
          o.z = fmaf(f, v.z, o.z);
          o.w = fmaf(f, v.w, o.w);
        }
      }
    }
    if (i < heads * per_head) {
      const float f = 1.f / s_total[head];
      *reinterpret_cast<uint2*>(static_cast<T*>(P.a.out) + n.b * P.a.out_token + (head0 + head) * P.a.out_head + d) =
          make_uint2(pack2<T>(o.x * f, o.y * f), pack2<T>(o.z * f, o.w * f));
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- launch

static size_t notes_bytes(int blocks) { return (static_cast<size_t>(blocks) * sizeof(TokenNote) + 255) / 256 * 256; }
static int token_blocks() { return sm_count() * kTokenBlocksPerSm; }

long long token_workspace(int head_dim, int group) {
  const size_t part = static_cast<size_t>(group > 8 ? 16 : 8) * ((head_dim > 64 ? 128 : 64) + 4) * sizeof(float);
  return static_cast<long long>(notes_bytes(token_blocks()) + static_cast<size_t>(token_blocks()) * 2 * part);
}

template <typename T, int DP, int NT>
static int launch(const CUtensorMap& km, const CUtensorMap& vm, const TokenArgs& p, cudaStream_t st) {
  constexpr size_t smem = TokenSizes<DP, NT>::kSmem;
  static bool configured_per_device[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  bool& configured = configured_per_device[dev & 63];
  if (!configured) {
    if (cudaFuncSetAttribute(k_attend_token<T, DP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return note_launch("cudaFuncSetAttribute(k_attend_token)");
    configured = true;
  }
  const int blocks = token_blocks();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kTokenThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, k_attend_token<T, DP, NT>, km, vm, p);
  if (const int rc = note_launch("k_attend_token")) return rc;
  cfg.gridDim = dim3(blocks - 1);
  cfg.dynamicSmemBytes = 0;
  cudaLaunchKernelEx(&cfg, k_token_join<T, DP, NT>, p, blocks);
  return note_launch("k_token_join");
}

template <typename T>
static int launch_type(const CUtensorMap& km, const CUtensorMap& vm, const TokenArgs& p, cudaStream_t st) {
  if (p.a.pool.Dh <= 64) return p.group <= 8 ? launch<T, 64, 1>(km, vm, p, st) : launch<T, 64, 2>(km, vm, p, st);
  return p.group <= 8 ? launch<T, 128, 1>(km, vm, p, st) : launch<T, 128, 2>(km, vm, p, st);
}

int launch_attend_token(const PagedCache& cache, const AttendArgs& a, cudaStream_t st) {
  TokenArgs p = {};
  p.a = a;
  p.group = a.H / a.pool.Hk;
  p.chunks = (p.group + 15) / 16;
  p.box_rows = a.pool.page_size % 16 ? 8 : 16;
  p.cap = static_cast<int>(std::min<long long>(static_cast<long long>(a.seq.table_cols) * a.pool.page_size, 1 << 30));
  p.wait_limit = debug_knobs().wait_limit;
  p.notes = static_cast<TokenNote*>(a.workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + notes_bytes(token_blocks()));
  alignas(64) CUtensorMap km, vm;
  const bool half = cache.type == kF16;
  if (!make_page_map(&km, half, a.pool.k, a.pool, p.box_rows) || !make_page_map(&vm, half, a.pool.v, a.pool, p.box_rows)) {
    set_kernel_error_text("attend", "the driver refused a tensor map over the pages");
    return kErrArg;
  }
  return half ? launch_type<__half>(km, vm, p, st) : launch_type<__nv_bfloat16>(km, vm, p, st);
}

}  // namespace lw
