// How attention over the paged cache is cut into pieces of equal work, from lengths that only the device knows.  Plain integer
// arithmetic for host and device.
//
// Prompts: the query rows of one kv head are (token, head of its group), token by token; a tile of 128 rows holds
// 128 / group tokens, a pair of tiles `pair_tokens` = twice that.  The work of a pair is `lead` units for what it costs besides
// (queries in, results out, the pipeline's start), then one unit per block of 128 positions that any of its tokens sees, one at
// least.  Units are numbered sequence by sequence, kv head by kv head, pair by pair, position block by position block; block c of
// G takes the units c U / G .. (c + 1) U / G - 1 of U.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define LW_HD __host__ __device__ __forceinline__
#else
#define LW_HD inline
#endif

namespace lw {

constexpr int kPosBlock = 128;   // positions of a unit of prompt attention

// sum over k < n of floor((a k + b) / m), a, b >= 0 (the division of a by m and the swap of their roles as in Euclid's algorithm)
LW_HD long long floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  long long sum = 0;
  while (n) {
    if (a >= m) {
      sum += static_cast<long long>(n) * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += static_cast<long long>(n) * (b / m);
      b %= m;
    }
    const unsigned long long top = static_cast<unsigned long long>(a) * n + b;
    if (top < m) break;
    n = static_cast<uint32_t>(top / m);
    b = static_cast<uint32_t>(top % m);
    const uint32_t t = a;
    a = m;
    m = t;
  }
  return sum;
}

// The first position that the row at `pos` sees (window 0: all).  Any window >= 0 and any pos: those before position 0 see nothing, whatever
// this says, and would overflow the difference.  (Three prompts of 5000 to 8000 tokens, window 2048: 740 us; with a branch 750.)
LW_HD int window_begin(int pos, int window) {
  const int begin = (pos > 0 ? pos : 0) - window + 1;
  return window > 0 && begin > 0 ? begin : 0;
}

struct PromptShape {
  int pair_tokens, window, lead;
};

// One sequence: `rows` new tokens, the last of its `len` positions.
struct PromptSeq {
  int rows, len;
};

LW_HD int prompt_pairs(const PromptShape& s, const PromptSeq& q) { return (q.rows + s.pair_tokens - 1) / s.pair_tokens; }

// Position blocks first .. last - 1 of pair i; positions lo .. hi - 1 are what its tokens see (hi <= lo: nothing).
struct PairRange {
  int first, last, lo, hi;
};
LW_HD PairRange pair_range(const PromptShape& s, const PromptSeq& q, int i) {
  const int p0 = q.len - q.rows, t0 = i * s.pair_tokens;
  const int t1 = q.rows - t0 < s.pair_tokens ? q.rows : t0 + s.pair_tokens;
  PairRange r;
  r.hi = p0 + t1;
  r.lo = window_begin(p0 + t0, s.window);
  r.first = r.lo / kPosBlock;
  r.last = r.hi > r.lo ? (r.hi + kPosBlock - 1) / kPosBlock : r.first + 1;
  return r;
}

// Units of the pairs 0 .. i - 1 of one head (i <= prompt_pairs).
LW_HD long long units_before(const PromptShape& s, const PromptSeq& q, int i) {
  if (i <= 0) return 0;
  const int pairs = prompt_pairs(s, q), T = s.pair_tokens, p0 = q.len - q.rows;
  const int whole = i < pairs ? i : pairs - 1;   // pairs of T tokens each: hi = p0 + (k + 1) T
  long long sum = static_cast<long long>(i) * s.lead;
  if (i == pairs) {
    const PairRange r = pair_range(s, q, pairs - 1);
    sum += r.last - r.first;
  }
  // pairs that end at or before position 0: one unit each
  int none = 0;
  if (p0 < 0) {
    none = -p0 / T;
    if (none > whole) none = whole;
    sum += none;
  }
  if (whole > none) sum += floor_sum(whole - none, kPosBlock, T, p0 + (none + 1) * T + kPosBlock - 1);
  if (s.window > 0) {   // less the blocks before the window: first = floor((p0 - window + 1 + k T) / 128) where that is positive
    const long long b = static_cast<long long>(p0) - s.window + 1, k1 = b < 0 ? (-b + T - 1) / T : 0;
    if (whole > k1) sum -= floor_sum(static_cast<uint32_t>(whole - k1), kPosBlock, T, static_cast<uint32_t>(b + k1 * T));
  }
  return sum;
}

// Units of work shared out to block c of `blocks`.
LW_HD long long share(long long units, int c, int blocks) { return units * c / blocks; }

}  // namespace lw
