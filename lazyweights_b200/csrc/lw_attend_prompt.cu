// Causal attention of packed prompts over the paged cache, on the tensor cores.
//
//   O[row, :] = sum_j softmax_j(scale Q[row] . K[j]) V[j]        rows = (token, head of the group) of one kv head
//
// One pass over the positions with a running reference m of the scores (in powers of two): p = 2^(c s - m), l = sum p,
// O = sum p V; m is the row's maximum so far, moved only when the maximum has grown by more than kSlack, so that O and l are rescaled a
// few times per row, not at every block (p stays below 2^(kSlack + kLift), inside fp16's range; O / l does not depend on m).
//
//  S = Q K^T    tcgen05.mma, both operands in shared memory       [128 rows x 128 positions], fp32 in tensor memory
//  P            one thread per row reads S, writes P in the cache's type over S
//  O += P V     tcgen05.mma, P from tensor memory, V from shared memory as it lies in the pages (positions are its K axis)
//
// Bound: the tensor core and the exponentials, about even: 128 x 128 x 128 take 1067 cycles of multiplications (554 + 513, measured) and
// 1024 of exponentials (16 per cycle and SM).  So two tiles of 128 rows (a pair) share the staged keys and values of a thread block and
// take turns: while one tile's softmax runs the tensor core works for the other.  What a block of positions takes now, 3350
// cycles for both tiles, is the chain of one tile: 2000 cycles of softmax (scores in 450, exponentials 1400: the special-function
// unit serves both tiles), then its multiplications and two hand-overs.  Medians, with the clock that the card's power limit
// leaves: 16384 tokens, 32 heads over 8: 2.26 ms at 1.63 GHz, 970 TFLOP/s of what the mask leaves; 509 tokens behind 32000: 305 us at 1.57, 880.
//  * Warp 0 loads keys and warp 2 values (TMA; a page's rows of a kv head are a box), each into a ring of stages of its own: a wait's
//    parity tells only neighbouring turns of a stage apart, so whoever loads one has to load every turn of it.  Warps 1 and 3 issue the
//    multiplications of a tile each, and load its queries: issuing blocks while the tensor core is busy, and a commit costs it 78
//    cycles, so one warp for both tiles with commits for the stages left it idle a third more.  Warps 4..7 and 8..11 are the softmax
//    of the two tiles; they tell when a stage is read, from the completion of the scores behind it.
//  * A thread holds a whole row of S, 128 registers: with two threads per row the exponentials took as long (the special-function unit) and
//    the maximum had to be exchanged.  A third of the exponentials as polynomials on the other pipes changed nothing: with a warp per tile
//    and scheduler, each waiting for its own last instruction, the issue slots are 38 % busy and no pipe is full.  P handed over in halves made the exponentials slower than it made the product earlier.
//  * The work is cut into equal shares whatever the lengths (lw_attend_plan.h), a pair's start and end counted as kPromptLead blocks
//    of positions; a pair that is cut leaves unnormalised partial results, which k_attend_join adds up.  Lengths are read on the device.
//  * Values of positions that no row of the pair sees are zeroed in shared memory before they are multiplied (a weight of 0
//    would not hide a NaN that an earlier owner of the page left).
//  * Rounding: S, m, l, O in 32 bits; P in the cache's type, as the tensor core takes it (half a step of its 11 or 8 bits,
//    independent from position to position); l adds the unrounded p.  fp16 has no more than 2^-24 below 1, and a hundred thousand
//    positions that small are a result's worth: p is taken times 2^kLift there, m being that much less than the maximum it follows.
#include <cuda.h>

#include <algorithm>

#include "lw_attend.cuh"
#include "lw_attend_plan.h"
#include "lw_tcgen05.cuh"

namespace lw {

constexpr int kPromptThreads = 12 * 32;
constexpr int kPromptRegsSoftmax = 216, kPromptRegsOther = 72;   // 8 and 4 warps: 12 x 168, the launch's
constexpr float kSlack = 8.f;         // of a row's maximum, in powers of two, before its reference follows
constexpr float kLift = 7.f;          // fp16, whose largest power of two is 2^15
constexpr int kPromptLead = 2;       // 24 packed prompts of 20 to 2500 tokens: 243 us (0: 373, 1: 274, 3: 246); 16384 tokens: 2.27 ms (2.39, 2.35, 2.25)

// The pair that block c continues: its first packed row, rows (tokens) and first query head, and the blocks that hold its first and
// last unit (first == c: none).  A block leaves the pair that it continues as its piece 0, the one that it only begins as piece 1.
struct alignas(16) PieceNote {
  int row0, rows, head0, first, last;
  int b, position, pad;   // its sequence, position of its first token
};

struct PromptArgs {
  AttendArgs a;
  int group, tile_tokens;   // query heads per kv head; tokens of a tile: 128 / group
  int box_rows;             // positions of a K / V box: a divisor of the page size and of 128
  int dim16;                // head_dim rounded up to 16
  int cap;                  // positions the table can name
  uint32_t wait_limit;
  int drop;                 // a test's lost copy: block 0 never loads this block of keys of its share (-1: none)
  PieceNote* notes;         // [gridDim.x]
  float* partial;           // [gridDim.x][piece][tile]: m[128], l[128], O [dim16 / 4][128][4]
};
__host__ __device__ constexpr size_t tile_partial_floats(int dim16) { return 256 + static_cast<size_t>(dim16) * 128; }

struct SeqRows {
  PromptSeq q;
  int row0;
};
__device__ __forceinline__ SeqRows seq_rows(const PromptArgs& P, int b) {
  const Sequences& s = P.a.seq;
  const int r0 = min(max(s.starts[b], 0), P.a.rows), r1 = min(max(s.starts[b + 1], r0), P.a.rows);
  SeqRows r;
  r.q.rows = r1 - r0;
  r.q.len = min(max(s.lens[b], 0), P.cap);
  r.row0 = r0;
  return r;
}

// A run of units of one pair, and the walk over a block's share.  Every role of the block walks by itself.
struct Walk {
  int b, h, i, off;
  long long left;
  SeqRows s;
};
struct Piece {
  int h, t0, j0, j1;    // kv head, first token of the pair, position blocks
  bool begins, ends;
  SeqRows s;
  int b;
};
// A piece without position blocks (j0 == j1) is to be passed over.
__device__ __forceinline__ Piece next_piece(const PromptArgs& P, const PromptShape& shape, Walk& w) {
  const PairRange r = pair_range(shape, w.s.q, w.i);
  const int n = shape.lead + r.last - r.first, take = static_cast<int>(min(static_cast<long long>(n - w.off), w.left));
  Piece p;
  p.h = w.h;
  p.t0 = w.i * shape.pair_tokens;
  p.j0 = r.first + max(0, w.off - shape.lead);
  p.j1 = r.first + max(0, w.off + take - shape.lead);
  p.begins = w.off <= shape.lead;
  p.ends = w.off + take == n;
  p.s = w.s;
  p.b = w.b;
  w.left -= take;
  if (!p.ends) {
    w.off += take;
  } else {
    w.off = 0;
    if (++w.i == prompt_pairs(shape, w.s.q)) {
      w.i = 0;
      if (++w.h == P.a.pool.Hk) {
        w.h = 0;
        if (w.left > 0) {
          do ++w.b; while (w.b < P.a.seq.n - 1 && seq_rows(P, w.b).q.rows == 0);
          w.s = seq_rows(P, w.b);
        }
      }
    }
  }
  return p;
}

// One tile of the pair inside a piece: its position blocks there (none: first >= last) and what its rows see.
struct TileRange {
  int first, last, p_first, p_last, tokens;   // p_first, p_last: positions of its first and last token
  __device__ __forceinline__ bool none() const { return first >= last; }
  __device__ __forceinline__ bool has(int j) const { return j >= first && j < last; }
};
__device__ __forceinline__ TileRange tile_range(const PromptArgs& P, const Piece& p, int x) {
  const int t0 = p.t0 + x * P.tile_tokens, p0 = p.s.q.len - p.s.q.rows;
  TileRange r;
  r.tokens = min(P.tile_tokens, p.s.q.rows - t0);
  r.p_first = p0 + t0;
  r.p_last = p0 + t0 + r.tokens - 1;
  r.first = max(p.j0, window_begin(r.p_first, P.a.window) / kPosBlock);
  r.last = min(p.j1, (r.p_last + kPosBlock) / kPosBlock);
  if (r.tokens <= 0 || r.p_last < 0) r.last = r.first = 0;
  return r;
}

// ---- Values that are not finite.  A tile's rows share the multiplication by V, so an infinite or NaN value of a position reaches
// the rows of the tile that do not see it too: its weight there is 0, and 0 x inf is NaN.  Where a result is not finite and
// its sum of weights is, the positions that the tile multiplied but some of its rows do not see are looked through, and if one
// holds such a value the rows are computed again, one by one (a warp each time; the ordinary path pays a comparison per result).

// Where position p of kv head kh lies in the pools; -1 for a bad page, whose keys and values are zeros.
__device__ __forceinline__ long long place_of(const PromptArgs& P, int b, int kh, int p) {
  const int column = p / P.a.pool.page_size, page = P.a.seq.table[b * P.a.seq.table_stride + column];
  if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(P.a.pool.n_pages)) return -1;
  return page * P.a.pool.page_stride + kh * P.a.pool.head_stride + (p - column * P.a.pool.page_size) * P.a.pool.token_stride;
}
// This lane's four dimensions there; zeros past the head.  Loaded from somewhere in any case, so that loads need not wait for a branch.
template <typename T>
__device__ __forceinline__ uint2 four_of(const PromptArgs& P, const void* pool, long long at, int lane) {
  const int d = lane * 4 < P.a.pool.Dh ? lane * 4 : 0;
  uint2 v = *reinterpret_cast<const uint2*>(static_cast<const T*>(pool) + (at < 0 ? 0 : at) + d);
  if (at < 0 || d != lane * 4) v = make_uint2(0u, 0u);
  return v;
}
constexpr int kAtOnce = 8;   // positions whose loads a warp has in flight; the places of 32 are looked up together, a lane each
template <typename T>
__device__ __noinline__ bool values_not_finite(const PromptArgs& P, int b, int kh, int from, int to) {
  constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x & 31;
  for (int p0 = from; p0 < to; p0 += 32) {
    const long long at = p0 + lane < to ? place_of(P, b, kh, p0 + lane) : -1;
    bool bad = false;
#pragma unroll kAtOnce
    for (int i = 0; i < 32; ++i) {
      const uint2 v = four_of<T>(P, P.a.pool.v, __shfl_sync(0xffffffffu, at, i), lane);
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= ((((k & 2) ? v.y : v.x) >> (16 * (k & 1))) & kExponent) == kExponent;
    }
    if (__any_sync(0xffffffffu, bad)) return true;
  }
  return false;
}
// Attention of one row over positions lo .. pos, by a warp.  28 rows at 100000 positions, seven to a warp: 107 ms (position by position 374).
template <typename T>
__device__ __noinline__ void single_row(const PromptArgs& P, int b, int kh, long long row, int head, int lo, int pos) {
  const int lane = threadIdx.x & 31;
  auto number = [](uint2 v, int k) {
    const uint32_t bits = (((k & 2) ? v.y : v.x) >> (16 * (k & 1))) & 0xffffu;
    const unsigned short u = static_cast<unsigned short>(bits);
    return static_cast<float>(*reinterpret_cast<const T*>(&u));
  };
  const uint2 q = four_of<T>(P, P.a.q, row * P.a.q_token + head * P.a.q_head, lane);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = lo; p0 <= pos; p0 += 32) {
    const int n = min(32, pos - p0 + 1);
    const long long at = lane < n ? place_of(P, b, kh, p0 + lane) : -1;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += kAtOnce) {
      uint2 k[kAtOnce], v[kAtOnce];
      float s[kAtOnce], m2 = m;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const long long there = __shfl_sync(0xffffffffu, at, i0 + i);
        k[i] = four_of<T>(P, P.a.pool.k, there, lane);
        v[i] = four_of<T>(P, P.a.pool.v, there, lane);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        s[i] = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d) s[i] = fmaf(number(q, d), number(k[i], d), s[i]);
#pragma unroll
        for (int d = 16; d; d >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
        s[i] = i0 + i < n ? s[i] * (P.a.scale * 1.4426950408889634f) : -INFINITY;
        m2 = fmaxf(m2, s[i]);
      }
      const float ref = m2 == -INFINITY ? 0.f : m2, keep = exp2_fast(m - ref);
      m = m2;
      l *= keep;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] *= keep;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float w = exp2_fast(s[i] - ref);
        l += w;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = fmaf(w, number(v[i], d), o[d]);
      }
    }
  }
  if (lane * 4 < P.a.pool.Dh)
    *reinterpret_cast<uint2*>(static_cast<T*>(P.a.out) + row * P.a.out_token + head * P.a.out_head + lane * 4) =
        make_uint2(pack2<T>(o[0] / l, o[1] / l), pack2<T>(o[2] / l, o[3] / l));
}
__device__ __forceinline__ bool not_finite(float v) { return !(fabsf(v) <= 3.402823466e38f); }

__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
        "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

// t5_wait for a converged warp whose lanes leave the loop together: 60 cycles where the barrier is ready; with a way out per lane 160.
// state: the block's word of kGivesUp and kMending for each of its warps that computes single rows again.  How long that takes depends on the
// context, so while it lasts no wait's polls are counted; it waits for nothing itself, so it ends.
constexpr int kGivesUp = 1, kMending = 2;
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, uint32_t limit, unsigned int* err, int* state) {
  const uint32_t addr = smem_addr(bar);
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done != 0)) return true;
    if ((i & 63u) == 63u) {
      const int now = *static_cast<volatile int*>(state);
      if (__any_sync(0xffffffffu, now & kGivesUp)) return false;
      if (__any_sync(0xffffffffu, now != 0)) i = 0;
    }
  }
  atomicOr(err, 1u);
  atomicOr(state, kGivesUp);
  return false;
}

// The largest of three; NaN are passed over
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void tmem_load16_at(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

template <int DP>
struct PromptSizes {
  static constexpr uint32_t kTile = 128 * DP * 2;                   // bytes of a tile of queries, a block of keys or of values
  static constexpr int kKeyStages = DP == 128 ? 3 : 4;
  static constexpr int kValueStages = DP == 128 ? 2 : 4;
  static constexpr int kStages = kKeyStages + kValueStages;
  static constexpr size_t kSmem = (2 + kStages) * kTile;   // and 3 KB of static variables: all that a block can have
};

// The turns of a ring of stages: the stage of the next one, and the parity that a wait for its copy takes.
template <int FIRST, int STAGES>
struct Ring {
  int s = FIRST;
  uint32_t ph = 0;
  __device__ __forceinline__ void step() {
    if (++s == FIRST + STAGES) {
      s = FIRST;
      ph ^= 1u;
    }
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kPromptThreads, 1)
    k_attend_prompt(const __grid_constant__ CUtensorMap QM, const __grid_constant__ CUtensorMap KM, const __grid_constant__ CUtensorMap VM,
                    const __grid_constant__ PromptArgs P) {
  using Z = PromptSizes<DP>;
  constexpr int kStages = Z::kStages;
  using Keys = Ring<0, Z::kKeyStages>;
  using Values = Ring<Z::kKeyStages, Z::kValueStages>;
  constexpr uint32_t kHalf = 128 * 128;   // bytes of 64 columns of a tile: 128 rows of 128 bytes, swizzled
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], mma_done[2], tail_full;
  __shared__ uint32_t tmem_slot[1];
  __shared__ int state, s_first[4];
  __shared__ long long s_scan[kPromptThreads / 32], s_rest;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_addr(smem_raw), ring = base + 2 * Z::kTile;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_addr(full + i), 1);
      mbar_init(smem_addr(empty + i), 2);   // both tiles
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_addr(q_full + x), 1);
      mbar_init(smem_addr(q_empty + x), 4);
      mbar_init(smem_addr(s_full + x), 1);
      mbar_init(smem_addr(p_full + x), 4);
      mbar_init(smem_addr(o_full + x), 1);
      mbar_init(smem_addr(mma_done + x), 1);
    }
    mbar_init(smem_addr(&tail_full), 1);
    state = 0;
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot[0];
  pdl_trigger();
  pdl_wait();

  // ---- this block's share of the units
  const PromptShape shape = {2 * P.tile_tokens, P.a.window, kPromptLead};
  const int n_seqs = P.a.seq.n;
  auto seq_units = [&](int b) -> long long {
    if (b >= n_seqs) return 0;
    const SeqRows s = seq_rows(P, b);
    if (blockIdx.x == 0 && P.a.seq.lens[b] > P.cap) atomicOr(P.a.err, kErrWordIndex);
    return s.q.rows > 0 ? P.a.pool.Hk * units_before(shape, s.q, prompt_pairs(shape, s.q)) : 0;
  };
  auto block_sum = [&](long long v, long long& before) -> long long {   // of all threads; before: of the threads in front of this one
    long long inc = v;
    for (int o = 1; o < 32; o <<= 1) {
      const long long w = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += w;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    long long front = 0, all = 0;
    for (int k = 0; k < kPromptThreads / 32; ++k) {
      if (k < warp) front += s_scan[k];
      all += s_scan[k];
    }
    __syncthreads();
    before = front + inc - v;
    return all;
  };
  long long units = 0, before = 0, mine_units = 0;
  for (int b0 = 0; b0 < n_seqs; b0 += kPromptThreads) units += block_sum(mine_units = seq_units(b0 + tid), before);
  const int blocks = static_cast<int>(min(static_cast<long long>(gridDim.x), units));   // the others have nothing to do
  const long long u0 = static_cast<int>(blockIdx.x) < blocks ? share(units, blockIdx.x, blocks) : 0, u1 = static_cast<int>(blockIdx.x) < blocks ? share(units, blockIdx.x + 1, blocks) : 0;
  if (u0 < u1) {
    long long front = 0;
    for (int b0 = 0; b0 < n_seqs; b0 += kPromptThreads) {
      long long all = units;
      if (n_seqs > kPromptThreads) all = block_sum(mine_units = seq_units(b0 + tid), before);
      if (u0 >= front + before && u0 < front + before + mine_units) {
        const SeqRows s = seq_rows(P, b0 + tid);
        const long long per_head = mine_units / P.a.pool.Hk, rest = u0 - front - before;
        s_first[0] = b0 + tid;
        s_first[1] = static_cast<int>(rest / per_head);
        s_rest = rest % per_head;
      }
      front += all;
    }
    __syncthreads();
    if (warp == 0) {   // the pair that holds unit s_rest of its head: 32-fold search
      const SeqRows s = seq_rows(P, s_first[0]);
      int lo = 0, hi = prompt_pairs(shape, s.q);   // units_before(lo) <= s_rest < units_before(hi)
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = min(lo + lane * step, hi);
        const unsigned int ok = __ballot_sync(0xffffffffu, at < hi && units_before(shape, s.q, at) <= s_rest);
        const int best = 31 - __clz(ok);           // lane 0 always says yes
        lo += best * step;
        hi = min(lo + step, hi);
      }
      if (lane == 0) {
        s_first[2] = lo;
        s_first[3] = static_cast<int>(s_rest - units_before(shape, s.q, lo));
      }
    }
    __syncthreads();
  } else if (tid == 0) {
    P.notes[blockIdx.x] = {0, 0, 0, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.x), 0, 0, 0};
  }
  Walk walk = {};
  walk.left = u1 - u0;
  if (walk.left > 0) {
    walk.b = s_first[0];
    walk.h = s_first[1];
    walk.i = s_first[2];
    walk.off = s_first[3];
    walk.s = seq_rows(P, walk.b);
    if (tid == 0) {
      const PairRange r = pair_range(shape, walk.s.q, walk.i);
      const long long begin = u0 - walk.off + shape.lead;   // of its position blocks; unit u is block floor(((u + 1) blocks - 1) / units)'s
      const int t0 = walk.i * shape.pair_tokens, me = blockIdx.x;
      P.notes[me] = {walk.s.row0 + t0, min(shape.pair_tokens, walk.s.q.rows - t0), walk.h * P.group,
                     walk.off > shape.lead ? static_cast<int>(((begin + 1) * blocks - 1) / units) : me,
                     walk.off > shape.lead ? static_cast<int>(((begin + r.last - r.first) * blocks - 1) / units) : me, walk.b,
                     walk.s.q.len - walk.s.q.rows + t0, 0};
    }
  }

  if (warp >= 4) {   // -------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptRegsSoftmax));
    const int x = (warp >> 2) - 1, row = (warp & 3) * 32 + lane, token = row / P.group, head = row - token * P.group;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + x * 128, to = tmem + lanes + 256 + x * 128;
    // a scale of 0 becomes a very small one: a score hidden as -inf must stay -inf
    const float c = fmaxf(fabsf(P.a.scale) * 1.4426950408889634f, 1e-30f);
    const bool leader = (warp & 3) == 0 && lane == 0;
    uint8_t* const mine_rows = smem_raw + x * Z::kTile + (warp & 3) * (Z::kTile / 4);   // 32 rows of the queries' place
    int s_count = 0, o_count = 0, v_before = 0;
    Keys keys;
    Values values;
    auto rows_to_mend = [&](const Piece& p, const TileRange& r, bool bad) -> uint32_t {
      const uint32_t rows = __ballot_sync(0xffffffffu, bad);
      if (__builtin_expect(rows == 0, 1)) return 0u;
      const PairRange pr = pair_range(shape, p.s.q, p.t0 / shape.pair_tokens);
      __syncwarp();
      if (!values_not_finite<T>(P, p.b, p.h, max(0, r.p_first + 1), pr.hi) &&
          !(P.a.window > 0 && values_not_finite<T>(P, p.b, p.h, pr.lo, window_begin(r.p_last, P.a.window)))) return 0u;
      return rows;
    };
    bool ok = true;
    while (walk.left > 0 && ok) {
      const Piece p = next_piece(P, shape, walk);
      if (p.j0 == p.j1) continue;
      const TileRange r = tile_range(P, p, x), r2 = tile_range(P, p, x ^ 1);
      const bool mine = token < min(r.tokens, P.tile_tokens);
      const int pos = mine ? r.p_first + token : -1;
      const int lo = window_begin(pos, P.a.window);
      const bool idle = !__any_sync(0xffffffffu, mine);
      float m = -INFINITY, l = 0.f;
      for (int j = p.j0; j < p.j1; ++j) {
        const bool here = r.has(j);
        if (!here && !r2.has(j)) continue;
        // The scores' completion tells that the multiplications are done with the keys of this block and the values of the one
        // before: one thread per tile gives the stages back.  (A commit of its own for each would hold the tensor core up by 78 cycles.)
        const int k_stage = keys.s, v_stage = values.s;
        keys.step();
        values.step();
        if (!here) continue;   // the other tile's; this tile's issuing warp gives the stages back
        if (!(ok = wait_warp(s_full + x, s_count++ & 1, P.wait_limit, P.a.err, &state))) break;
        if (leader) {
          mbar_arrive(empty + k_stage);
          if (j > r.first) mbar_arrive(empty + v_before);
        }
        v_before = v_stage;
        if (!idle) {
          tc_fence_after();
          const int p0 = j * kPosBlock;
          uint32_t v[128];
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          tmem_load32(ts, v);
          tmem_load32(ts + 32, v + 32);
          tmem_load32(ts + 64, v + 64);
          tmem_load32(ts + 96, v + 96);
          tmem_wait_load();
          if (__builtin_expect(p0 + kPosBlock - 1 > r.p_first || (P.a.window > 0 && p0 <= r.p_last - P.a.window), 0)) {   // some row does not see all of it
            // which columns, as bits: one selection per score (two comparisons more, and their code, took as long as the exponentials)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int top = pos - p0 - 32 * k, bottom = lo - p0 - 32 * k;
              uint32_t seen = top >= 31 ? 0xffffffffu : top < 0 ? 0u : (2u << top) - 1u;
              seen &= bottom <= 0 ? 0xffffffffu : bottom >= 32 ? 0u : 0xffffffffu << bottom;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(seen >> i & 1u)) v[32 * k + i] = 0xff800000u;
            }
          }
#pragma unroll
          for (int i = 0; i < 128; i += 2) mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          const float mx = max3(max3(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * c;
          const bool grow = mx > m + kSlack + lift<T>(m, kLift);
          if (__any_sync(0xffffffffu, grow)) {
            const float m2 = grow ? mx - lift<T>(mx, kLift) : m, keep = m == -INFINITY ? 0.f : exp2_fast(m - m2);   // nothing seen yet: O and l count for nothing
            m = m2;
            l *= keep;
            if (j > r.first) {   // PV of the block before is done: its completion came with these scores
#pragma unroll 1
              for (int d = 0; d < P.dim16; d += 16) {
                uint32_t o[16];
                tmem_load16(to + d, o);
                tmem_wait_load();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(keep == 0.f ? 0.f : __uint_as_float(o[k]) * keep);
                tmem_store16(to + d, o);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.f : m;
          const float2 c2 = make_float2(c, c), ref2 = make_float2(-ref, -ref);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t h[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 e = __ffma2_rn(make_float2(__uint_as_float(v[32 * k + 2 * i]), __uint_as_float(v[32 * k + 2 * i + 1])), c2, ref2);
              const float2 w = make_float2(exp2_fast(e.x), exp2_fast(e.y));
              sum[i & 1] = __fadd2_rn(sum[i & 1], w);
              h[i] = pack2<T>(w.x, w.y);
            }
            tmem_store16(ts + 16 * k, h);
          }
          l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
          tmem_wait_store();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + x);
      }
      if (!ok) break;   // of this warp; the others leave at their next wait
      if (!r.none() && !(ok = wait_warp(o_full + x, o_count++ & 1, P.wait_limit, P.a.err, &state))) break;
      tc_fence_after();
      if (leader && !r.none()) mbar_arrive(empty + v_before);
      float check = 0.f;
      if (!idle) {
        const bool whole = p.begins && p.ends && !r.none(), empty = pos < 0;
        const float f = empty ? 0.f : 1.f / l;
        float* part = P.partial + (static_cast<size_t>(blockIdx.x) * 4 + (p.begins ? 2 : 0) + x) * tile_partial_floats(P.dim16);
        if (!(p.begins && p.ends)) {
          part[row] = pos < 0 ? -INFINITY : m;
          part[128 + row] = pos < 0 ? 0.f : l;
        }
#pragma unroll 1
        for (int d0 = 0; d0 < P.dim16 && !r.none(); d0 += 32) {
          uint32_t o[32];
          tmem_load16_at(to + d0, o);
          if (d0 + 16 < P.dim16) tmem_load16_at(to + d0 + 16, o + 16);
          tmem_wait_load();
          if (whole) {
#pragma unroll
            for (int d = 0; d < 32; d += 8) {
              uint32_t h[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) h[k] = empty ? 0u : pack2<T>(__uint_as_float(o[d + 2 * k]) * f, __uint_as_float(o[d + 2 * k + 1]) * f);
#pragma unroll
              for (int k = 0; k < 8; ++k) check = d0 + d < P.a.pool.Dh ? fmaf(__uint_as_float(o[d + k]), 0.f, check) : check;   // NaN from the first that is not finite on
              if (d0 + d < DP) *reinterpret_cast<uint4*>(mine_rows + lane * (DP * 2) + ((((d0 + d) >> 3) ^ (lane & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
          } else {
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              if (d0 + d < P.dim16) *reinterpret_cast<uint4*>(part + 256 + (static_cast<size_t>((d0 + d) / 4) * 128 + row) * 4) = make_uint4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          }
        }
      }
      uint32_t mend = 0;
      if (r.none() && p.begins && p.ends) {   // rows that see nothing
        if (mine)
          for (int d = 0; d < P.a.pool.Dh; d += 8)
            *reinterpret_cast<uint4*>(static_cast<T*>(P.a.out) + static_cast<long long>(p.s.row0 + p.t0 + x * P.tile_tokens + token) * P.a.out_token +
                                      static_cast<long long>(p.h * P.group + head) * P.a.out_head + d) = make_uint4(0u, 0u, 0u, 0u);
      } else if (!idle && p.begins && p.ends) {
        // Row by row through the place of this tile's queries: a warp's store covers whole rows, not 16 bytes of 32 rows each, which
        // kept the load/store unit busy for 4000 cycles per pair.
        mend = rows_to_mend(p, r, check != 0.f && pos >= 0 && !not_finite(l));
        const uint32_t rows = __ballot_sync(0xffffffffu, mine) & ~mend;   // those to be computed again are left: their queries may lie there
        const unsigned long long my_out = reinterpret_cast<unsigned long long>(static_cast<T*>(P.a.out) + static_cast<long long>(p.s.row0 + p.t0 + x * P.tile_tokens + token) * P.a.out_token +
                                                                              static_cast<long long>(p.h * P.group + head) * P.a.out_head);
        __syncwarp();
        constexpr int kChunks = DP / 8, kRowsAtOnce = 32 / kChunks;
        const int chunk = lane % kChunks;
#pragma unroll 4
        for (int i = 0; i < kChunks; ++i) {
          const int src = i * kRowsAtOnce + lane / kChunks;
          const unsigned long long to_row = __shfl_sync(0xffffffffu, my_out, src);
          const uint4 v = *reinterpret_cast<const uint4*>(mine_rows + src * (DP * 2) + ((chunk ^ (src & 7)) << 4));
          if ((rows >> src & 1u) && chunk * 8 < P.a.pool.Dh) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(to_row) + chunk * 8) = v;
        }
      }
      if (!r.none()) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the next queries come here
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty + x);
      }
      if (__builtin_expect(mend != 0, 0) && lane == 0) atomicAdd(&state, kMending);
      for (uint32_t left = mend; left; left &= left - 1) {
        const int src = __ffs(left) - 1;
        const int row_pos = __shfl_sync(0xffffffffu, pos, src), row_lo = __shfl_sync(0xffffffffu, lo, src);
        single_row<T>(P, p.b, p.h, p.s.row0 + p.t0 + x * P.tile_tokens + __shfl_sync(0xffffffffu, token, src),
                      p.h * P.group + __shfl_sync(0xffffffffu, head, src), row_lo, row_pos);
      }
      if (__builtin_expect(mend != 0, 0) && lane == 0) atomicSub(&state, kMending);
      tc_fence_before();   // the next P is announced after these reads of O
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptRegsOther));
    if (warp == 0 || warp == 2) {   // ------------------------------------------------------- loads: warp 0 keys, warp 2 values
      const bool values = warp == 2;
      const void* const map = values ? &VM : &KM;
      const int ring_begin = values ? Z::kKeyStages : 0, ring_end = values ? kStages : Z::kKeyStages;
      int s = ring_begin, tails = 0, fills = 0;
      uint32_t ph = 0;
      bool ok = true;
      constexpr int kHalves = DP / 64;
      while (walk.left > 0 && ok) {
        const Piece p = next_piece(P, shape, walk);
        if (p.j0 == p.j1) continue;
        const TileRange r[2] = {tile_range(P, p, 0), tile_range(P, p, 1)};
        // positions that some row of the pair sees
        const PairRange pr = pair_range(shape, p.s.q, p.t0 / shape.pair_tokens);
        const int* table = P.a.seq.table + p.b * P.a.seq.table_stride;
        for (int j = p.j0; j < p.j1 && ok; ++j) {
          if (!r[0].has(j) && !r[1].has(j)) continue;
          const int end = min(kPosBlock, pr.hi - j * kPosBlock), begin = max(0, pr.lo - j * kPosBlock);
          const int rows_end = (end + P.box_rows - 1) / P.box_rows, rows_begin = begin / P.box_rows;
          // lane n: the page of box n
          int page = 0, in_page = 0;
          if (lane >= rows_begin && lane < rows_end) {
            const int pos = j * kPosBlock + lane * P.box_rows, column = pos / P.a.pool.page_size;
            page = table[column];
            in_page = pos - column * P.a.pool.page_size;
            if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(P.a.pool.n_pages)) {   // the tensor map's bounds fill it with zeros
              atomicOr(P.a.err, kErrWordIndex);
              page = P.a.pool.n_pages;
            }
          }
          if (!(ok = wait_warp(empty + s, ph ^ 1u, P.wait_limit, P.a.err, &state))) break;
          const uint32_t stage = ring + s * Z::kTile;
          const bool cut = values && (end < kPosBlock || begin > 0);
          uint64_t* const bar = cut ? &tail_full : full + s;
          if (fills++ != P.drop || values || blockIdx.x != 0) {
            if (elect_one()) mbar_expect(bar, (rows_end - rows_begin) * kHalves * P.box_rows * 128u);
            __syncwarp();
            for (int n = rows_begin; n < rows_end; ++n) {
              const int pg = __shfl_sync(0xffffffffu, page, n), in = __shfl_sync(0xffffffffu, in_page, n);
              if (elect_one()) {
#pragma unroll
                for (int d = 0; d < kHalves; ++d) tma_load_4d(stage + d * kHalf + n * P.box_rows * 128, map, 64 * d, in, p.h, pg, smem_addr(bar));
              }
              __syncwarp();
            }
          }
          if (cut) {
            ok = wait_warp(&tail_full, tails++ & 1, P.wait_limit, P.a.err, &state);
            uint8_t* dst = smem_raw + (stage - smem_addr(smem_raw));
            for (int n = lane; n < (kPosBlock - end + begin) * 8; n += 32) {   // rows end .. 127, then 0 .. begin - 1
              const int row = (end + (n >> 3)) & (kPosBlock - 1);
#pragma unroll
              for (int d = 0; d < kHalves; ++d) *reinterpret_cast<uint4*>(dst + d * kHalf + row * 128 + (n & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (elect_one()) mbar_arrive(full + s);
            __syncwarp();
          }
          if (++s == ring_end) {
            s = ring_begin;
            ph ^= 1u;
          }
        }
      }
    } else {   // ------------------------------------------------ multiplications, started by one lane: warp 1 for the first tile, warp 3 for the second
      constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
      const uint32_t idesc_s = idesc_f16_m128(kPosBlock) | type | (P.a.scale < 0.f ? 1u << 13 : 0u), idesc_o = idesc_f16_m128(P.dim16) | type | (1u << 16);   // bit 13: -Q, bit 16: V is position-major
      const int steps = P.dim16 / 16, x = warp >> 1;
      const uint32_t ts = tmem + x * 128, to = tmem + 256 + x * 128;
      const uint64_t q = smem_desc_sw128(base + x * Z::kTile);
      int q_count = 0, p_count = 0;
      Keys keys;
      Values values;
      bool ok = true, any = false;
      auto wait = [&](uint64_t* bar, int parity) -> bool {
        if (ok) ok = wait_warp(bar, parity, P.wait_limit, P.a.err, &state);
        tc_fence_after();
        return ok;
      };
      uint64_t v = 0;   // the values of the block before
      auto weighted_sum = [&](bool fresh) {   // O (+)= P V
        if (!wait(p_full + x, p_count++ & 1)) return;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < 8; ++i)   // 16 positions further: two groups of eight rows
            mma_ts_f16(to, ts + 8 * i, v + i * (2048 >> 4), idesc_o, !fresh || i > 0);
        }
        __syncwarp();
      };
      while (walk.left > 0 && ok) {
        const Piece p = next_piece(P, shape, walk);
        if (p.j0 == p.j1) continue;
        const TileRange r = tile_range(P, p, x), r2 = tile_range(P, p, x ^ 1);
        for (int j = p.j0; j < p.j1 && ok; ++j) {
          const bool here = r.has(j);
          if (!here && !r2.has(j)) continue;
          const uint32_t k_ph = keys.ph, k_stage = keys.s, v_ph = values.ph, v_stage = values.s;
          keys.step();
          values.step();
          if (!here) {
            // The other tile's block, given back once it is there: the turns of a stage must not overtake a warp that waits on its
            // barriers, whose parity tells only neighbouring turns apart.
            wait(full + k_stage, k_ph);
            if (wait(full + v_stage, v_ph) && elect_one()) {
              mbar_arrive(empty + k_stage);
              mbar_arrive(empty + v_stage);
            }
            __syncwarp();
            continue;
          }
          const bool first = j == r.first, last = j + 1 == r.last;
          if (first) {
            // This tile's queries, once the results before have left through their place.  (The multiplications that read the last
            // ones are done: their scores have become the P of the last weighted sum.)
            wait(q_empty + x, (q_count & 1) ^ 1);
            if (ok && elect_one()) {
              mbar_expect(q_full + x, (DP / 64) * 128u * P.group * P.tile_tokens);
#pragma unroll
              for (int d = 0; d < DP / 64; ++d)
                tma_load_3d(base + x * Z::kTile + d * kHalf, &QM, 64 * d, p.h * P.group, p.s.row0 + p.t0 + x * P.tile_tokens, smem_addr(q_full + x));
            }
            __syncwarp();
            wait(q_full + x, q_count++ & 1);
          }
          wait(full + k_stage, k_ph);
          if (!first) weighted_sum(j == r.first + 1);
          if (!ok) break;
          any = true;
          const uint64_t k = smem_desc_sw128(ring + k_stage * Z::kTile);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {   // 32 bytes further inside the swizzle row; then the other half
              const uint32_t off = (i & 3) * 2 + (i >> 2) * (kHalf >> 4);
              if (i < steps) mma_ss_f16(ts, q + off, k + off, idesc_s, i > 0);
            }
            mma_commit(s_full + x);
          }
          __syncwarp();
          v = (smem_desc_sw128(ring + v_stage * Z::kTile) & ~(0x3FFFull << 16)) | (static_cast<uint64_t>(kHalf >> 4) << 16);
          wait(full + v_stage, v_ph);
          if (last) {
            weighted_sum(first);
            if (ok && elect_one()) mma_commit(o_full + x);
            __syncwarp();
          }
        }
      }
      if (any) {
        if (elect_one()) mma_commit(mma_done + x);   // they read shared memory and write tensor memory, which the block is about to give back
        __syncwarp();
        if (lane == 0) mbar_wait(smem_addr(mma_done + x), 0, P.a.err, 1u << 16);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // Every copy has been waited for by the multiplications, unless the block gave up: then those in flight land before it gives its
  // shared memory back (both parities: one of them has passed).
  if ((state & kGivesUp) && warp == 0 && lane == 0) {
    for (int i = 0; i < kStages; ++i)
      for (int parity = 0; parity < 2; ++parity) mbar_wait(smem_addr(full + i), parity, P.a.err, 1u << 14);
    for (int x = 0; x < 2; ++x)
      for (int parity = 0; parity < 2; ++parity) mbar_wait(smem_addr(q_full + x), parity, P.a.err, 1u << 14);
    for (int parity = 0; parity < 2; ++parity) mbar_wait(smem_addr(&tail_full), parity, P.a.err, 1u << 14);
  }
}

// Pairs that were cut: block (c, y) joins 32 of the rows of the pair that block c of the attention kernel continued, if it is the first
// to continue it.  O = sum_k 2^(m_k - m) O_k / sum_k 2^(m_k - m) l_k over the pieces in order.
constexpr int kJoinThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) k_attend_join(const __grid_constant__ PromptArgs P) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x + 1, x = blockIdx.y >> 2, row = (blockIdx.y & 3) * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  // what the kernel before wrote is read from L2
  const int4 note_a = __ldcg(reinterpret_cast<const int4*>(P.notes + c)), note_b = __ldcg(reinterpret_cast<const int4*>(P.notes + c) + 1);
  const PieceNote n = {note_a.x, note_a.y, note_a.z, note_a.w, note_b.x, note_b.y, note_b.z, 0};
  if (n.first != c - 1) return;   // nothing continued, or not the first to continue it
  const int token = row / P.group, head = row - token * P.group, t = x * P.tile_tokens + token;
  const bool mine = token < P.tile_tokens && t < n.rows;
  const int last = n.last;
  const size_t tile = tile_partial_floats(P.dim16);
  auto piece = [&](int k) { return P.partial + (static_cast<size_t>(k) * 4 + (k < c ? 2 : 0) + x) * tile; };
  float m = -INFINITY, l = 0.f;
#pragma unroll 4
  for (int k = c - 1; k <= last; ++k) m = fmaxf(m, __ldcg(piece(k) + row));
  const float ref = m == -INFINITY ? 0.f : m;
  constexpr int kWarps = kJoinThreads / 32, kSteps = 128 / (4 * kWarps);
  float4 o[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = c - 1; k <= last; ++k) {
    const float* part = piece(k);
    const float lk = __ldcg(part + 128 + row), f = exp2_fast(__ldcg(part + row) - ref);
    l += lk * f;
    if (lk == 0.f) continue;   // the piece holds nothing for this row, and no O
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int d = (i * kWarps + warp) * 4;
      if (d < P.dim16) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(part + 256 + (static_cast<size_t>(d / 4) * 128 + row) * 4));
        o[i] = make_float4(fmaf(f, v.x, o[i].x), fmaf(f, v.y, o[i].y), fmaf(f, v.z, o[i].z), fmaf(f, v.w, o[i].w));
      }
    }
  }
  T* out = static_cast<T*>(P.a.out) + static_cast<long long>(n.row0 + t) * P.a.out_token + static_cast<long long>(n.head0 + head) * P.a.out_head;
  const float f = n.position + t < 0 ? 0.f : 1.f / l;   // a row before position 0 gives zeros; one whose scores are all -inf NaN, as in a pair that is whole
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (mine && (i * kWarps + warp) * 4 < P.a.pool.Dh) bad |= not_finite(o[i].x) || not_finite(o[i].y) || not_finite(o[i].z) || not_finite(o[i].w);
  // as in k_attend_prompt, for all rows of the pair that this block holds: the four warps share them, a quarter of the dimensions each
  uint32_t mend = __ballot_sync(0xffffffffu, bad && !not_finite(l));
  const int kh = n.head0 / P.group;
  if (__builtin_expect(__syncthreads_or(mend != 0), 0)) {
    __shared__ uint32_t s_mend[kWarps];
    if ((threadIdx.x & 31) == 0) s_mend[warp] = mend;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) mend |= s_mend[w];
    if (!values_not_finite<T>(P, n.b, kh, max(0, n.position + 1), n.position + n.rows) &&
        !(P.a.window > 0 && values_not_finite<T>(P, n.b, kh, window_begin(n.position, P.a.window), window_begin(n.position + n.rows - 1, P.a.window)))) mend = 0;
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int d = (i * kWarps + warp) * 4;
    if (mine && d < P.a.pool.Dh && !(mend >> (threadIdx.x & 31) & 1u)) *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<T>(o[i].x * f, o[i].y * f), pack2<T>(o[i].z * f, o[i].w * f));
  }
  for (int i = 0; mend; mend &= mend - 1, ++i) {   // a warp each
    if ((i & (kWarps - 1)) != warp) continue;
    const int src = __ffs(mend) - 1, row_t = __shfl_sync(0xffffffffu, t, src), pos = n.position + row_t;
    single_row<T>(P, n.b, kh, n.row0 + row_t, n.head0 + __shfl_sync(0xffffffffu, head, src), window_begin(pos, P.a.window), pos);
  }
}

// ---------------------------------------------------------------------------------------------------------- launch

static size_t notes_bytes(int blocks) { return (static_cast<size_t>(blocks) * sizeof(PieceNote) + 255) / 256 * 256; }

long long prompt_workspace(int head_dim) {
  const int dim16 = (head_dim + 15) / 16 * 16, blocks = sm_count();
  return static_cast<long long>(notes_bytes(blocks) + static_cast<size_t>(blocks) * 4 * tile_partial_floats(dim16) * sizeof(float));
}

template <typename T, int DP>
static int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const PromptArgs& p, cudaStream_t st) {
  static bool configured_per_device[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  bool& configured = configured_per_device[dev & 63];
  if (!configured) {
    if (cudaFuncSetAttribute(k_attend_prompt<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(PromptSizes<DP>::kSmem)) != cudaSuccess)
      return note_launch("cudaFuncSetAttribute(k_attend_prompt)");
    configured = true;
  }
  const int blocks = sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kPromptThreads);
  cfg.dynamicSmemBytes = PromptSizes<DP>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, k_attend_prompt<T, DP>, qm, km, vm, p);
  if (const int rc = note_launch("k_attend_prompt")) return rc;
  if (blocks < 2) return kOk;
  cfg.gridDim = dim3(blocks - 1, 8);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cudaLaunchKernelEx(&cfg, k_attend_join<T>, p);
  return note_launch("k_attend_join");
}

int launch_attend_prompt(const PagedCache& cache, const AttendArgs& a, cudaStream_t st) {
  PromptArgs p = {};
  p.a = a;
  p.group = a.H / a.pool.Hk;
  p.tile_tokens = 128 / p.group;
  p.box_rows = cache.prompt_rows;
  p.dim16 = (a.pool.Dh + 15) / 16 * 16;
  p.cap = static_cast<int>(std::min<long long>(static_cast<long long>(a.seq.table_cols) * a.pool.page_size, 1 << 30));
  p.wait_limit = debug_knobs().wait_limit;
  p.drop = debug_knobs().drop_unit;
  p.notes = static_cast<PieceNote*>(a.workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + notes_bytes(sm_count()));
  alignas(64) CUtensorMap qm;
  const bool half = cache.type == kF16;
  if (!make_query_map(&qm, half, a.q, a.pool.Dh, a.H, a.rows, a.q_head, a.q_token, p.group, p.tile_tokens)) {
    set_kernel_error_text("attend_prompt", "the driver refused a tensor map over the queries");
    return kErrArg;
  }
  if (a.pool.Dh <= 64) return half ? launch<__half, 64>(qm, cache.prompt_k, cache.prompt_v, p, st) : launch<__nv_bfloat16, 64>(qm, cache.prompt_k, cache.prompt_v, p, st);
  return half ? launch<__half, 128>(qm, cache.prompt_k, cache.prompt_v, p, st) : launch<__nv_bfloat16, 128>(qm, cache.prompt_k, cache.prompt_v, p, st);
}

}  // namespace lw
