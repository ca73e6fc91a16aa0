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
//  * A warp is a worker of its own, with its own share of the positions, its own ring of stages that its TMA loads fill (192 KB per SM
//    in flight with eight warps; about 45 KB would cover the latency at full bandwidth), its own m, l, O.  Warps never wait for one
//    another: a batch of short sequences is a row of small pieces with loads of queries and stores of results between them, and a
//    block whose warps met at every piece took 146 instead of 89 us for 33 sequences of 30 to 4000 positions with 32 kv heads.
//  * Shares: units of 16 positions of a kv head, numbered sequence by sequence, head by head, each sequence and head led by kLead
//    units that stand for what it costs besides (queries in, results out); every worker takes the same number, whatever the
//    lengths, which it reads on the device.  What a worker begins or ends in the middle of goes to the workspace
//    and is joined, in order, by k_token_join.
//  * Positions outside the sequence or the window: scores replaced by -inf, values zeroed in shared memory (0 x NaN is NaN).
//  * Rounding: scores, m, l, O in 32 bits, P in the cache's type for the tensor core (half a step of it, independent per position);
//    in fp16 p is taken times 2^15, in O, l and the m of partial results alike: its smallest number would otherwise be 2^-24 of the
//    largest p, and a hundred thousand positions that small are a result's worth.
#include <cuda.h>

#include <algorithm>

#include "lw_attend.cuh"
#include "lw_attend_plan.h"

namespace lw {

constexpr int kTokenWarps = 4, kTokenThreads = kTokenWarps * 32;
constexpr int kUnit = 16;                 // positions of a unit
constexpr int kTokenBlocksPerSm = 2;
constexpr float kLift = 15.f;             // fp16: its largest power of two
constexpr int kLead = 2;                  // see above: 200 sequences of 10 to 500 positions, 8 kv heads: 32.1 us (0: 41.7, 1: 34.5, 4: 32.5)

// The piece that worker w continues: sequence, head slot, the workers that hold its first and last unit (first == w: none).
struct alignas(16) TokenNote {
  int b, h, first, last;
};

struct TokenArgs {
  AttendArgs a;
  int group, chunks;        // query heads per kv head; passes over the keys: ceil(group / (8 NT))
  int box_rows;             // 16, or 8 where pages are odd multiples of 8
  int cap, least;           // positions the table can name; units of a worker at least, as long as there are fewer than workers
  uint32_t wait_limit, page_inverse;   // floor(2^32 / page size)
  int drop;                 // a test's lost copy: worker 0 never loads this unit of its share (-1: none)
  TokenNote* notes;         // [worker]
  float* partial;           // [worker][piece]: see TokenSizes
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

// Where a walk over a worker's share stands: unit t of head slot h (kv head, pass) of sequence b; `left` units to go, the leading ones of
// sequences and heads still to come among them.
struct TokenWalk {
  int b, h, t;
  long long left;
  TokenSeq s;
  __device__ __forceinline__ void step(const TokenArgs& P, int slots) {
    --left;
    if (++t < s.last) return;
    left -= kLead;
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
  static constexpr int kHalves = DP / 64, kSteps = DP / 16;
  static constexpr uint32_t kTile = 16 * DP * 2;                 // bytes of 16 keys, or values
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr uint32_t kWarp = kStages * 2 * kTile;
  static constexpr size_t kSmem = 1024 + kTokenWarps * kWarp;
  // A piece of a worker: (m, l) per head, then O as the lanes of a warp hold it, [NT][kSteps][lane][4]
  static constexpr size_t kPartHead = 8 * NT * 2, kPartial = kPartHead + static_cast<size_t>(NT) * kSteps * 128;
};

// O as the lanes hold it (rows dimension lane / 4 and eight further, columns heads 2 (lane % 4) and the next), normalised, to the
// rows of the results.  Two transposes per 16 dimensions leave every lane two neighbouring dimensions of head lane / 4.
template <typename T>
__device__ __forceinline__ void store_heads(T* out, long long head_stride, int heads, int Dh, int step, const float (&v)[4], int lane) {
  const uint32_t lo = transpose_8x8(pack2<T>(v[0], v[1])), hi = transpose_8x8(pack2<T>(v[2], v[3]));
  const int head = lane >> 2, d = step * 16 + (lane & 3) * 2;
  if (head >= heads) return;
  T* p = out + head * head_stride + d;
  if (d < Dh) *reinterpret_cast<uint32_t*>(p) = lo;
  if (d + 8 < Dh) *reinterpret_cast<uint32_t*>(p + 8) = hi;
}

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kTokenThreads, kTokenBlocksPerSm)
    k_attend_token(const __grid_constant__ CUtensorMap KM, const __grid_constant__ CUtensorMap VM, const __grid_constant__ TokenArgs P) {
  using Z = TokenSizes<DP, NT>;
  constexpr int kSteps = Z::kSteps, kStages = Z::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kTokenWarps][kStages];
  __shared__ long long s_scan[kTokenWarps];
  __shared__ int s_start[kTokenWarps][3];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = ((smem_addr(smem_raw) + 1023u) & ~1023u) + warp * Z::kWarp;
  uint8_t* const mine_raw = smem_raw + (base - smem_addr(smem_raw));
  if (lane < kStages) mbar_init(smem_addr(&full[warp][lane]), 1);
  __syncwarp();
  pdl_trigger();
  pdl_wait();

  // ---- the workers' shares.  Neighbouring shares lie in different blocks, so that little work meets many SMs.
  const int slots = P.a.pool.Hk * P.chunks, n_seqs = P.a.seq.n;
  auto units_of = [&](int b) -> long long {
    if (b >= n_seqs) return 0;
    const TokenSeq s = token_seq(P, b);
    if (blockIdx.x == 0 && P.a.seq.lens[b] > P.cap) atomicOr(P.a.err, kErrWordIndex);
    return s.last > s.first ? static_cast<long long>(s.last - s.first + kLead) * slots : 0;
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
  long long units = 0, before = 0, mine = 0;
  for (int b0 = 0; b0 < n_seqs; b0 += kTokenThreads) units += block_sum(mine = units_of(b0 + tid), before);
  const int workers = static_cast<int>(min(static_cast<long long>(gridDim.x) * kTokenWarps, (units + P.least - 1) / P.least));
  long long front = 0;
  for (int b0 = 0; b0 < n_seqs && units > 0; b0 += kTokenThreads) {
    long long all = units;
    if (n_seqs > kTokenThreads) all = block_sum(mine = units_of(b0 + tid), before);
    if (mine > 0) {
      const TokenSeq s = token_seq(P, b0 + tid);
      for (int w = 0; w < kTokenWarps; ++w) {
        const int worker = w * gridDim.x + blockIdx.x;
        if (worker >= workers) break;
        const long long rest = share(units, worker, workers) - front - before;
        if (rest >= 0 && rest < mine) {
          const int per_slot = s.last - s.first + kLead, slot = static_cast<int>(rest / per_slot);
          s_start[w][0] = b0 + tid;
          s_start[w][1] = slot;
          s_start[w][2] = s.first - kLead + static_cast<int>(rest - static_cast<long long>(slot) * per_slot);   // below s.first: among the leading units
        }
      }
    }
    front += all;
  }
  // sequences without positions: zeros
  for (int b = blockIdx.x; b < n_seqs; b += gridDim.x) {
    if (P.a.seq.lens[b] > 0) continue;
    const int per_head = P.a.pool.Dh / 8;
    for (int i = tid; i < P.a.H * per_head; i += kTokenThreads)
      *reinterpret_cast<uint4*>(static_cast<T*>(P.a.out) + b * P.a.out_token + (i / per_head) * P.a.out_head + (i % per_head) * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();
  const int worker = warp * gridDim.x + blockIdx.x;
  long long u0 = 0, u1 = 0;
  TokenWalk at = {};
  if (worker < workers) {
    u0 = share(units, worker, workers);
    u1 = share(units, worker + 1, workers);
    at.b = s_start[warp][0];
    at.h = s_start[warp][1];
    at.s = token_seq(P, at.b);
    at.t = max(s_start[warp][2], at.s.first);
    at.left = u1 - u0 - (at.t - s_start[warp][2]);
  }
  // the piece at hand, if it began before: its units are begin .. begin + last - first - 1 of all, unit u is worker
  // floor(((u + 1) workers - 1) / units)'s
  if (lane == 0) {
    const bool continued = at.left > 0 && at.t > at.s.first;
    const long long begin = u0 - (at.t - at.s.first);
    P.notes[worker] = {at.b, at.h, continued ? static_cast<int>(((begin + 1) * workers - 1) / units) : worker,
                       continued ? static_cast<int>(((begin + at.s.last - at.s.first) * workers - 1) / units) : worker};
  }
  if (at.left <= 0) return;

  // ---- loads.  Lane n of the first few starts box n of a unit: keys, then values; half by half of the head dimension; 16 positions
  // in one box or two of eight.  The page of the next unit is asked for when the unit before it is started.
  TokenWalk ahead = at;
  int load_stage = 0, fills = 0, page = 0, in_page = 0;
  const int per_half = 16 / P.box_rows, boxes = per_half * Z::kHalves;   // of the keys; as many of the values
  const int box_row = (lane % per_half) * P.box_rows, box_half = lane % boxes / per_half;
  const bool loader = lane < 2 * boxes;
  const void* const map = lane < boxes ? &KM : &VM;
  const uint32_t box_at = base + (lane < boxes ? 0 : Z::kTile) + box_half * 2048 + box_row * 128;
  bool inside = false;   // this lane's box of the next unit holds positions of the sequence
  auto ask_page = [&]() {
    const int pos = ahead.t * kUnit + box_row;
    inside = loader && ahead.left > 0 && pos < ahead.s.len && pos + P.box_rows > ahead.s.lo;
    if (inside) {
      int column = __umulhi(pos, P.page_inverse);   // floor(pos / page size), or one less
      in_page = pos - column * P.a.pool.page_size;
      if (in_page >= P.a.pool.page_size) {
        ++column;
        in_page -= P.a.pool.page_size;
      }
      page = P.a.seq.table[ahead.b * P.a.seq.table_stride + column];
    }
  };
  auto load_next = [&]() {
    if (ahead.left <= 0) return;
    const uint32_t bar = smem_addr(&full[warp][load_stage]);
    const int count = __popc(__ballot_sync(0xffffffffu, inside));
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count * P.box_rows * 128) : "memory");
    __syncwarp();
    if (inside && !(P.drop == fills && worker == 0)) {
      if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(P.a.pool.n_pages)) {   // the tensor map's bounds fill it with zeros
        atomicOr(P.a.err, kErrWordIndex);
        page = P.a.pool.n_pages;
      }
      tma_load_4d(box_at + load_stage * 2 * Z::kTile, map, 64 * box_half, in_page, P.chunks == 1 ? ahead.h : ahead.h / P.chunks, page, bar);
    }
    ++fills;
    if (++load_stage == kStages) load_stage = 0;
    ahead.step(P, slots);
    ask_page();
  };
  ask_page();
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) load_next();
  // where this lane's rows of the operands lie in a stage: keys (positions as rows), values (transposed), per 16 dimensions of a half
  uint32_t k_at[4], v_at[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, vr = (lane & 7) + (lane >> 4) * 8;
    k_at[k] = base + kr * 128 + (((k * 2 + (lane >> 4)) ^ (kr & 7)) << 4);
    v_at[k] = base + Z::kTile + vr * 128 + (((k * 2 + ((lane >> 3) & 1)) ^ (vr & 7)) << 4);
  }

  // ---- the share, piece by piece: units of one sequence and head slot
  const float c = P.a.scale * 1.4426950408889634f;
  int stage = 0;
  uint32_t parity = 0;
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
    {   // the queries of the next piece, towards the L1 cache
      const bool same = h + 1 < slots;
      const int nb = same ? b : b + 1, nh = same ? h + 1 : 0, rows = min(8 * NT, P.group - (nh % P.chunks) * 8 * NT);
      const int line = lane & 1, head = lane >> 1;
      if (at.left > t_end - t_begin && nb < n_seqs && head < rows && line * 64 < P.a.pool.Dh)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const T*>(P.a.q) + nb * P.a.q_token + ((nh / P.chunks) * P.group + (nh % P.chunks) * 8 * NT + head) * P.a.q_head + line * 64));
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
      const int p0 = t * kUnit;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_addr(&full[warp][stage]), parity, P.a.err, P.wait_limit))) {
        // Given up (the error word says so, the results are void): the copies still in flight land before the warp leaves.
        if (lane == 0)
          for (int i = 0; i < kStages; ++i)
            for (uint32_t turn = 0; turn < 2; ++turn) (void)mbar_wait(smem_addr(&full[warp][i]), turn, P.a.err, 1u << 14);
        return;
      }
      const uint32_t at_stage = stage * 2 * Z::kTile;
      // S^T: rows positions, columns heads
      float sc[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][0][i] = sc[n][1][i] = 0.f;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t a[4];
        load_matrices(a, k_at[k & 3] + at_stage + (k >> 2) * 2048);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16n8k16<T>(sc[n][k & 1], a, qf[n][k][0], qf[n][k][1]);
      }
      float x[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = (sc[n][0][i] + sc[n][1][i]) * c;
      if (p0 + 16 > s.len || p0 < s.lo) {   // the first or last unit of the sequence holds positions that are not its own
        const int v0 = s.lo - p0, v1 = s.len - p0;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = (lane >> 2) + (i >> 1) * 8;
            if (row < v0 || row >= v1) x[n][i] = -INFINITY;
          }
        uint8_t* dst = mine_raw + at_stage + Z::kTile;
        for (int i = lane; i < 16 * 8 * Z::kHalves; i += 32) {
          const int row = (i >> 3) & 15;
          if (row < v0 || row >= v1) *reinterpret_cast<uint4*>(dst + (i >> 7) * 2048 + row * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the stage is loaded again
        __syncwarp();
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mx[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(x[n][e], x[n][2 + e]);
          for (int d = 4; d < 32; d <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], d));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[n][0] || mx[1] > m[n][1])) {   // a maximum moves: what is there counts for less
          float keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m2 = fmaxf(m[n][e], mx[e]);
            keep[e] = m[n][e] == -INFINITY ? 0.f : exp2_fast((m[n][e] - lift<T>(m[n][e], kLift)) - (m2 - lift<T>(m2, kLift)));
            m[n][e] = m2;
            l[n][e] *= keep[e];
          }
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][k][i] *= keep[i & 1];
        }
        const float ref[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0] - lift<T>(m[n][0], kLift), m[n][1] == -INFINITY ? 0.f : m[n][1] - lift<T>(m[n][1], kLift)};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = exp2_fast(x[n][i] - ref[i & 1]);
        l[n][0] += x[n][0] + x[n][2];
        l[n][1] += x[n][1] + x[n][3];
        pf[n][0] = transpose_8x8(pack2<T>(x[n][0], x[n][1]));
        pf[n][1] = transpose_8x8(pack2<T>(x[n][2], x[n][3]));
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t a[4];
        load_matrices_transposed(a, v_at[k & 3] + at_stage + (k >> 2) * 2048);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16n8k16<T>(o[n][k], a, pf[n][0], pf[n][1]);
      }
      __syncwarp();
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1u;
      }
      load_next();
    }
    const bool begins = t_begin == s.first, ends = t_end == s.last;
    float* part = P.partial + (static_cast<size_t>(worker) * 2 + (begins ? 1 : 0)) * Z::kPartial;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
      if (begins && ends) {
        T* out = static_cast<T*>(P.a.out) + b * P.a.out_token + (head0 + n * 8) * P.a.out_head;
        const float f[2] = {1.f / l[n][0], 1.f / l[n][1]};
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const float v[4] = {o[n][k][0] * f[0], o[n][k][1] * f[1], o[n][k][2] * f[0], o[n][k][3] * f[1]};
          store_heads<T>(out, P.a.out_head, heads - n * 8, P.a.pool.Dh, k, v, lane);
        }
      } else {
        if (lane < 4)
          *reinterpret_cast<float4*>(part + (n * 8 + lane * 2) * 2) =
              make_float4(m[n][0] - lift<T>(m[n][0], kLift), l[n][0], m[n][1] - lift<T>(m[n][1], kLift), l[n][1]);
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          *reinterpret_cast<float4*>(part + Z::kPartHead + ((n * kSteps + k) * 32 + lane) * 4) = make_float4(o[n][k][0], o[n][k][1], o[n][k][2], o[n][k][3]);
      }
    }
    at.left -= t_end - t_begin - 1;
    at.t = t_end - 1;
    at.step(P, slots);
  }
}

// The pieces of a sequence and head slot that several workers share: m = max m_k, o = sum_k 2^(m_k - m) O_k / sum_k 2^(m_k - m) l_k.
// A chain is named by its second worker's note.  Short ones are one warp's work.  Of long ones (few rows, split over many workers) a job
// is 16 dimensions: the warps of a block take every eighth piece and add up in turn, and the jobs spread over all blocks.
constexpr int kTokenJoinWarps = 8, kTokenJoinThreads = kTokenJoinWarps * 32, kTokenShort = 8;
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kTokenJoinThreads) k_token_join(const __grid_constant__ TokenArgs P, int workers) {
  using Z = TokenSizes<DP, NT>;
  constexpr int kJobs = Z::kSteps * NT;   // of a chain
  __shared__ int s_job[kTokenJoinThreads], s_jobs;
  __shared__ TokenNote s_note[kTokenJoinThreads];
  __shared__ float s_m[kTokenJoinWarps][32][2], s_l[kTokenJoinWarps][32][2];
  __shared__ float4 s_o[kTokenJoinWarps][32];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, all = (workers - 1) * kJobs;
  // what the kernel before wrote is read from L2
  auto note_of = [&](int w) {
    const int4 v = __ldcg(reinterpret_cast<const int4*>(P.notes + w));
    return TokenNote{v.x, v.y, v.z, v.w};
  };
  auto piece_of = [&](const TokenNote& n, int k) { return P.partial + (static_cast<size_t>(k) * 2 + (k == n.first ? 1 : 0)) * Z::kPartial; };
  auto result = [&](const TokenNote& n, int nt, int step, const float4& sum, const float* total) {
    const float f[2] = {1.f / total[0], 1.f / total[1]};
    const float v[4] = {sum.x * f[0], sum.y * f[1], sum.z * f[0], sum.w * f[1]};
    const int head0 = (n.h / P.chunks) * P.group + (n.h % P.chunks) * 8 * NT + nt * 8, heads = P.group - (n.h % P.chunks) * 8 * NT - nt * 8;
    store_heads<T>(static_cast<T*>(P.a.out) + n.b * P.a.out_token + head0 * P.a.out_head, P.a.out_head, heads, P.a.pool.Dh, step, v, lane);
  };
  constexpr int kGroup = Z::kSteps < 4 ? Z::kSteps : 4, kGroups = kJobs / kGroup;   // steps of a short job
  for (int j = blockIdx.x + warp * gridDim.x; j < (workers - 1) * kGroups; j += gridDim.x * kTokenJoinWarps) {
    const TokenNote n = note_of(j / kGroups + 1);
    if (n.first != j / kGroups || n.last - n.first >= kTokenShort) continue;
    const int first_job = j % kGroups * kGroup, nt = first_job / Z::kSteps;
    float4 ml[kTokenShort];
#pragma unroll
    for (int q = 0; q < kTokenShort; ++q)
      ml[q] = n.first + q <= n.last ? __ldcg(reinterpret_cast<const float4*>(piece_of(n, n.first + q) + (nt * 8 + (lane & 3) * 2) * 2)) : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float4 o[kGroup];
#pragma unroll
    for (int k = 0; k < kGroup; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < kTokenShort; ++q) {
      m[0] = fmaxf(m[0], ml[q].x);
      m[1] = fmaxf(m[1], ml[q].z);
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int q0 = 0; q0 < kTokenShort; q0 += 4) {
      if (n.first + q0 > n.last) break;
      float4 v[4][kGroup];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int k = 0; k < kGroup; ++k)
          v[q][k] = n.first + q0 + q <= n.last ? __ldcg(reinterpret_cast<const float4*>(piece_of(n, n.first + q0 + q) + Z::kPartHead + ((first_job + k) * 32 + lane) * 4))
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float f[2] = {exp2_fast(ml[q0 + q].x - ref[0]), exp2_fast(ml[q0 + q].z - ref[1])};
        l[0] += ml[q0 + q].y * f[0];
        l[1] += ml[q0 + q].w * f[1];
#pragma unroll
        for (int k = 0; k < kGroup; ++k)
          o[k] = make_float4(fmaf(f[0], v[q][k].x, o[k].x), fmaf(f[1], v[q][k].y, o[k].y), fmaf(f[0], v[q][k].z, o[k].z), fmaf(f[1], v[q][k].w, o[k].w));
      }
    }
#pragma unroll
    for (int k = 0; k < kGroup; ++k) result(n, nt, first_job % Z::kSteps + k, o[k], l);
  }
  for (int j0 = 0; j0 < all; j0 += gridDim.x * kTokenJoinThreads) {
    if (tid == 0) s_jobs = 0;
    __syncthreads();
    const int j = j0 + tid * gridDim.x + blockIdx.x;
    if (j < all) {
      const int w = j / kJobs + 1;
      const TokenNote n = note_of(w);
      if (n.first == w - 1 && n.last - n.first >= kTokenShort) {
        const int at = atomicAdd(&s_jobs, 1);
        s_job[at] = j % kJobs;
        s_note[at] = n;
      }
    }
    __syncthreads();
    const int jobs = s_jobs;
    for (int i = 0; i < jobs; ++i) {
      const TokenNote n = s_note[i];
      const int job = s_job[i], nt = job / Z::kSteps, step = job % Z::kSteps;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int k = n.first + warp; k <= n.last; k += kTokenJoinWarps) {
        const float* p = piece_of(n, k);
        const float4 ml = __ldcg(reinterpret_cast<const float4*>(p + (nt * 8 + (lane & 3) * 2) * 2));   // (m, l) of the lane's two heads
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p + Z::kPartHead + (job * 32 + lane) * 4));
        const float mk[2] = {ml.x, ml.z}, lk[2] = {ml.y, ml.w};
        float keep[2], add[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m2 = fmaxf(m[e], mk[e]), ref = m2 == -INFINITY ? 0.f : m2;
          keep[e] = exp2_fast(m[e] - ref);
          add[e] = exp2_fast(mk[e] - ref);
          m[e] = m2;
          l[e] = l[e] * keep[e] + lk[e] * add[e];
        }
        o = make_float4(o.x * keep[0] + v.x * add[0], o.y * keep[1] + v.y * add[1], o.z * keep[0] + v.z * add[0], o.w * keep[1] + v.w * add[1]);
      }
      for (int e = 0; e < 2; ++e) {
        s_m[warp][lane][e] = m[e];
        s_l[warp][lane][e] = l[e];
      }
      s_o[warp][lane] = o;
      __syncthreads();
      if (warp == 0) {
        float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f};
        for (int e = 0; e < 2; ++e)
          for (int w = 0; w < kTokenJoinWarps; ++w) top[e] = fmaxf(top[e], s_m[w][lane][e]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < kTokenJoinWarps; ++w) {
          float f[2];
          for (int e = 0; e < 2; ++e) {
            f[e] = exp2_fast(s_m[w][lane][e] - (top[e] == -INFINITY ? 0.f : top[e]));
            total[e] += s_l[w][lane][e] * f[e];
          }
          const float4 v = s_o[w][lane];
          sum = make_float4(sum.x + v.x * f[0], sum.y + v.y * f[1], sum.z + v.z * f[0], sum.w + v.w * f[1]);
        }
        result(n, nt, step, sum, total);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- launch

static size_t notes_bytes(int workers) { return (static_cast<size_t>(workers) * sizeof(TokenNote) + 255) / 256 * 256; }
static int token_blocks() { return sm_count() * kTokenBlocksPerSm; }

long long token_workspace(int head_dim, int group) {
  const int workers = token_blocks() * kTokenWarps;
  const size_t part = head_dim > 64 ? (group > 8 ? TokenSizes<128, 2>::kPartial : TokenSizes<128, 1>::kPartial)
                                    : (group > 8 ? TokenSizes<64, 2>::kPartial : TokenSizes<64, 1>::kPartial);
  return static_cast<long long>(notes_bytes(workers) + static_cast<size_t>(workers) * 2 * part * sizeof(float));
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
  cfg.blockDim = dim3(kTokenJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cudaLaunchKernelEx(&cfg, k_token_join<T, DP, NT>, p, blocks * kTokenWarps);
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
  p.box_rows = cache.token_rows;
  p.cap = static_cast<int>(std::min<long long>(static_cast<long long>(a.seq.table_cols) * a.pool.page_size, 1 << 30));
  p.wait_limit = debug_knobs().wait_limit;
  p.notes = static_cast<TokenNote*>(a.workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + notes_bytes(token_blocks() * kTokenWarps));
  p.least = 2;
  p.drop = debug_knobs().drop_unit;
  p.page_inverse = static_cast<uint32_t>((1ull << 32) / a.pool.page_size);
  const CUtensorMap &km = cache.token_k, &vm = cache.token_v;
  return cache.type == kF16 ? launch_type<__half>(km, vm, p, st) : launch_type<__nv_bfloat16>(km, vm, p, st);
}

}  // namespace lw
