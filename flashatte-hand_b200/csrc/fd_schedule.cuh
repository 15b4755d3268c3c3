// fd_schedule.cuh - how a decode launch cuts its work over persistent CTAs, and
// the arrival counters by which a pair's last CTA knows that it is the last.
// Shared by the decode kernels (fd_decode_sm100.cuh, fd_decode_fp4.cuh).
#pragma once

#include <cstdint>

#include "fd_kernels.h"

namespace fd {

namespace {

// Arrival counter of a split (sequence, KV head) pair, and of the grid:
// bits [12, 64) hold the launch's stamp, bits [0, 12) the arrivals seen under
// it (at most one per CTA, and a launch has at most 4095 CTAs).  The grid's
// stamp is the launch epoch, which runs 1 .. 2^52 - 1 and then starts again at
// 1.  A pair's counter lies where the partials of a launch of another shape may
// have been, any two fp32 numbers: its stamp is 12 bits that make the word's
// upper half a signalling NaN, which no arithmetic gives, and 40 bits of the
// epoch.  (The epoch alone is two numbers like (1, 0) at launch 0x3F800.)  So a
// counter can only be mistaken for the current launch's after 2^40 launches on
// one workspace (months of back-to-back calls), and only one that a launch
// which stopped early (a bounded wait ran out) left behind: the CTA that merges
// a pair clears its counter and the last CTA to arrive clears the grid
// counter, so a launch that completes leaves every counter at zero.  The first arrival of a launch
// sets the stamp with one compare-and-swap; every arrival that sees the
// stamp counts itself with one fetch-and-add, so the tens of CTAs sharing one
// long sequence's pair, finishing together, do not queue on a compare-and-swap
// loop.  Returns true for the pair's last arrival.
constexpr int kTicketCountBits = 12;
constexpr unsigned long long kTicketCountMask = (1ull << kTicketCountBits) - 1ull;
constexpr unsigned long long kEpochMax = (1ull << (64 - kTicketCountBits)) - 1ull;
__device__ __forceinline__ unsigned long long pair_stamp(unsigned long long epoch) {
  return (0xFFAull << 40) | (epoch & ((1ull << 40) - 1ull));
}
__device__ __forceinline__ bool ticket_arrive(unsigned long long* t, unsigned long long stamp, int nseg) {
  unsigned long long cur = *reinterpret_cast<volatile unsigned long long*>(t);
  for (;;) {
    if ((cur >> kTicketCountBits) == stamp) {
      const unsigned long long old = atomicAdd(t, 1ull);
      return (old & kTicketCountMask) + 1ull == static_cast<unsigned long long>(nseg);
    }
    const unsigned long long prev = atomicCAS(t, cur, (stamp << kTicketCountBits) | 1ull);
    if (prev == cur) return nseg == 1;
    cur = prev;
  }
}

// The same arrival in one round trip where the counter already carries the
// stamp (every arrival of a pair but the first): count first, look after.  A
// counter of another stamp is only made larger, and is overwritten as above.
__device__ __forceinline__ bool ticket_add(unsigned long long* t, unsigned long long stamp, int nseg) {
  const unsigned long long old = atomicAdd(t, 1ull);
  if ((old >> kTicketCountBits) == stamp)
    return (old & kTicketCountMask) + 1ull == static_cast<unsigned long long>(nseg);
  return ticket_arrive(t, stamp, nseg);
}

// ---------------------------------------------------------------- schedule
// Work is split in cost space.  In units where the K/V bytes of a full
// 128-token tile cost kFullTile = 8, a tile also costs `tile_fixed` (its
// fixed QK / softmax / PV work), a sequence's partial last tile costs its
// 16-token boxes instead of 8, and every (sequence, KV head) pair costs
// `seg` once (its set-up and epilogue), raised where needed so that no pair
// costs less than `floor` (a pair of a few tiles is a latency chain that
// the ring cannot hide behind streaming).  This per-pair part is the pair's
// `lead`: its first tile starts at the pair's start and tile j >= 1 at
// start + lead + j * full.  Pairs are laid end to end (b-major, then KV
// head); CTA c takes the tiles whose start cost lies in [C*c/G, C*(c+1)/G).
// Every tile belongs to exactly one CTA; a pair spread over several CTAs is
// merged by the last of them.
constexpr int kFullTile = 8;

struct CostModel {
  int tile_fixed, seg, floor;
  __device__ __forceinline__ int full() const { return kFullTile + tile_fixed; }
  // cost of the tiles of one pair of a sequence of `len` tokens
  __device__ __forceinline__ int tiles_cost(int len) const {
    const int n_full = len / kTileTokens, rem = len % kTileTokens;
    return n_full * full() + ((rem > 0 || len == 0) ? (rem + 15) / 16 + tile_fixed : 0);
  }
  __device__ __forceinline__ int lead(int len) const {
    const int raised = floor - tiles_cost(len);
    return raised > seg ? raised : seg;
  }
  __device__ __forceinline__ int pair_cost(int len) const { return lead(len) + tiles_cost(len); }
  // upper bound of any pair's lead
  __device__ __forceinline__ int max_lead() const { return floor > seg ? floor : seg; }
};

__device__ __forceinline__ int seq_tiles(int len) {
  return len > 0 ? (len + kTileTokens - 1) / kTileTokens : 1;
}

// Divisions of the schedule, in 32 bits: the host caps a launch's batch so
// that its cost line times (grid + 1) stays below 2^32 (all the schedule's
// cost positions, and a position times the grid, fit in 32 bits).  A 64-bit
// integer division is a long software sequence, and these run, cold, on
// every CTA's path to its first load.
__device__ __forceinline__ int64_t div_u32(int64_t a, int64_t b) {
  return static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}
__device__ __forceinline__ int64_t ceil_div_u32(int64_t a, int64_t b) { return div_u32(a + b - 1, b); }

// One segment of a CTA's work: tiles tile0 .. tile0+ntiles-1 of pair (b, kvh).
struct Segment {
  int b, kvh, pair;
  int tile0, ntiles;
  int seqlen;
  int nseg, cfirst;  // how many CTAs share this pair, and the first of them
};

struct Schedule {
  const int* cost_prefix;  // [B+1] per-pair cost prefix over sequences (smem)
  const int* lens;         // [B] sequence lengths, clamped to [0, max_len] (smem)
  int64_t max_len, total;  // total = Hkv * cost_prefix[B]
  int batch, hkv, grid;
  // Pair-aligned split (align_m > 0): every pair costs align_cost and CTA c
  // takes the whole pairs [align_m * c, align_m * (c + 1)).
  int align_m;
  int64_t align_cost;
  CostModel cm;
  // Where tile 0 starts: at the pair's start, or behind its lead like every
  // other.  In the second form a range that ends inside a lead leaves the whole
  // pair to the next CTA, in the first it takes a segment of that one tile.
  bool behind_lead = false;

  __device__ __forceinline__ int len_of(int b) const { return lens[b]; }
  __device__ __forceinline__ int64_t range_start(int c) const {
    if (align_m > 0) {
      const int64_t pairs = static_cast<int64_t>(batch) * hkv;
      const int64_t first_pair = static_cast<int64_t>(align_m) * c;
      return align_cost * (first_pair < pairs ? first_pair : pairs);
    }
    return div_u32(total * c, grid);
  }
  // CTA whose range holds cost position s: largest c with range_start(c) <= s
  // (cost split only: the pair-aligned split cuts no pair, so it never asks)
  __device__ __forceinline__ int cta_of(int64_t s) const {
    return static_cast<int>(div_u32((s + 1) * grid + total - 1, total) - 1);
  }
  __device__ __forceinline__ int64_t pair_start(int pair) const {
    const int b = pair / hkv, kvh = pair - b * hkv;
    return static_cast<int64_t>(hkv) * cost_prefix[b] +
           static_cast<int64_t>(kvh) * (cost_prefix[b + 1] - cost_prefix[b]);
  }
  // start of tile j of the pair that starts at cp and has lead `lead`
  __device__ __forceinline__ int64_t tile_start(int64_t cp, int lead, int j) const {
    return j == 0 && !behind_lead ? cp : cp + lead + static_cast<int64_t>(j) * cm.full();
  }
  // Segment of `pair` from tile j0 on, cut at range end e1; false if no tile
  // of the pair at or after j0 starts before e1.  Integer work here is 32-bit
  // except for pairs split across CTAs (rare), where cta_of is evaluated.
  __device__ __forceinline__ bool make(int pair, int j0, int64_t e1, Segment& s) const {
    const int b = pair / hkv;
    const int len = len_of(b);
    const int n = seq_tiles(len);
    const int lead = cm.lead(len);
    const int64_t cp = pair_start(pair);
    if (j0 >= n || tile_start(cp, lead, j0) >= e1) return false;
    // last tile with start < e1: j <= ceil((e1 - cp - lead) / full) - 1
    const int64_t x64 = e1 - cp - lead;
    int jmax = 0;
    if (x64 > 0) {
      const int x = x64 < 0x7fffffff ? static_cast<int>(x64) : 0x7fffffff;
      jmax = (x + cm.full() - 1) / cm.full() - 1;
    }
    if (jmax > n - 1) jmax = n - 1;
    s.b = b;
    s.kvh = pair - b * hkv;
    s.pair = pair;
    s.tile0 = j0;
    s.ntiles = jmax - j0 + 1;
    s.seqlen = len;
    if (j0 == 0 && jmax == n - 1) {  // the whole pair lies in this range
      s.nseg = 1;
      s.cfirst = -1;
    } else {
      s.cfirst = cta_of(tile_start(cp, lead, 0));
      s.nseg = cta_of(tile_start(cp, lead, n - 1)) - s.cfirst + 1;
    }
    return true;
  }
  // First segment of CTA c (false if the CTA has no tile).
  __device__ __forceinline__ bool first(int c, Segment& s) const {
    if (c >= grid) return false;
    const int64_t e0 = range_start(c), e1 = range_start(c + 1);
    int lo = 0, hi = batch - 1;  // largest b with hkv * prefix[b] <= e0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (static_cast<int64_t>(hkv) * cost_prefix[mid] <= e0) lo = mid; else hi = mid - 1;
    }
    const int pc = cost_prefix[lo + 1] - cost_prefix[lo];
    int kvh = static_cast<int>(div_u32(e0 - static_cast<int64_t>(hkv) * cost_prefix[lo], pc));
    kvh = kvh < hkv - 1 ? kvh : hkv - 1;
    const int pair = lo * hkv + kvh;
    const int64_t cp = pair_start(pair);
    int j0 = 0;
    if (e0 > cp) {
      const int64_t x = e0 - cp - cm.lead(len_of(lo));
      j0 = static_cast<int>(x > 0 ? ceil_div_u32(x, cm.full()) : 0);
      if (j0 < 1 && !behind_lead) j0 = 1;
    }
    if (make(pair, j0, e1, s)) return true;
    return pair + 1 < batch * hkv && make(pair + 1, 0, e1, s);
  }
  // Segment after `s` within the range that ends at cost e1.
  __device__ __forceinline__ bool next(const Segment& s, int64_t e1, Segment& nx) const {
    if (s.tile0 + s.ntiles < seq_tiles(s.seqlen)) return false;  // range ended inside the pair
    return s.pair + 1 < batch * hkv && make(s.pair + 1, 0, e1, nx);
  }
};

}  // namespace

}  // namespace fd
