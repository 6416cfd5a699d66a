// From the tiles' headers and their chunks' maxima (beam_tiles.cuh) to answers: a group's best
// continuations, or a row's log-probabilities.
//
// A continuation (beam k, token t) has score_k + x_t - lse_k and is ranked by that over its length's
// penalty.  Sums, scores and ranks are held in 64 bits: what is compared differs between beams by
// their lse, and float32 ranks near -100 would tie where the sums do not.  Order: the larger rank,
// then the lower beam, then the larger logit, then the lower token.
//
// The n best are found top down.  A node (a tile of a row, a chunk of a tile, 16 bytes of a chunk) is
// worth its largest logit's continuation; the n best nodes of a level, in the order above with a
// node's first token for its token, hold the n best continuations.  So a level is one selection: from
// all tiles, from the chunks of about n tiles, from the logits of about n chunks.  Where there are few tiles
// the first is left out, and the chunks are those of all tiles (start_of).
#pragma once
#include "beam_tiles.cuh"

namespace leat {

constexpr int BM_MAX_BEAMS = 64;
constexpr int BM_MAX_WIDTH = 64;
constexpr int BM_LIST = 512;    // nodes a level hands to the next
constexpr int BM_PARTS = 128;   // parts of the block whose best bound a level: at least twice the width
constexpr int BM_FEW = 10;      // up to this width 256 threads go down the levels, 512 beyond (three parts a place make 30 of 32)

struct MergeParams {
  TileParams T;
  int beams, width;
  int end_id;  // token of finished beams and the one that finishes a beam; -1: none
  float length_penalty;
  const int32_t* lengths;  // (rows) or NULL
  int32_t* out_tokens;
  int32_t* out_parents;
  float* out_scores;
  uint8_t* out_finished;  // or NULL
  int32_t* out_lengths;   // or NULL
};

struct LogprobParams {
  TileParams T;
  int given, top;
  const int32_t* ids;  // (rows, given) or NULL
  float* out_given;    // (rows, given)
  float* out_top;      // (rows, top)
  int32_t* out_top_ids;
};

// lse of one row from its tiles' headers, by one warp (the same in every lane), as the row's maximum and
// what the logarithm adds to it: kept apart, because next to a maximum of 1e38 (a row of nothing but
// its type's lowest value) the sum of the two would lose the second.
struct LogSum {
  float max;  // -inf: the row has no logit above -inf
  double log;
};
// (where a tile or the row's maximum is beyond PLAIN_LIMIT: kept out of line, since it hardly ever runs)
__device__ __noinline__ double part_beyond(TileHead v, float m, int e) {
  const double log2e_used = (double)log2e();
  if (!(v.max > neg_inf())) return 0.0;
  if (e != OVER_MAX) return v.sum * exp2((double)v.max * log2e_used - (double)e);
  return v.sum * (v.exponent != OVER_MAX ? exp2((double)v.exponent - (double)m * log2e_used) : exp((double)v.max - (double)m));
}
// h: the lane's header of the first 32 (whatever it reads where lane >= tiles)
__device__ __forceinline__ LogSum row_log_sum(TileHead h, const TileHead* heads, int tiles, int lane) {
  // float32 log2e is off by a part in 2^26: the sums are of e^(x (1 + off)), which the first-order
  // term off * max takes back but for off * (max - x), 2e-7 at most where x counts
  const double ln2_exact = 0.693147180559945309, off = 1.44269502162933349609375 * ln2_exact - 1.0;
  float m = lane < tiles ? h.max : neg_inf();
  for (int t = lane + 32; t < tiles; t += 32) m = fmaxf(m, heads[t].max);
  m = unord32(__reduce_max_sync(FULL, ord32(m + 0.0f)));
  if (m == neg_inf()) return LogSum{m, 0.0};
  const bool plain = fabsf(m) < PLAIN_LIMIT;
  const int e = plain ? (int)ceilf(m * log2e()) : OVER_MAX;
  auto part = [&](const TileHead& v) {
    if (!plain || (v.exponent == OVER_MAX && v.max > neg_inf())) return part_beyond(v, m, e);
    return v.max > neg_inf() ? v.sum * two_to(v.exponent - e) : 0.0;
  };
  double s = lane < tiles ? part(h) : 0.0;
  for (int t = lane + 32; t < tiles; t += 32) s += part(heads[t]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
  return LogSum{m, plain ? log(s) + ((double)e * ln2_exact - (double)m) - off * (double)m : log(s)};
}

// the same in float32, to within 2^-17: what the levels below rank by while other warps work out the
// exact one.  h, more: the lane's headers of the first 64.  (Of 2^-17 = 7.6e-6: lg2.approx is good to 2^-22 of
// a logarithm of up to 31, which is 5.1e-6; that times ln 2, and the sum, are rounded at up to 21.5, 2^-20 or
// 9.5e-7 each; the lanes' sums are rounded six times, 3.6e-7; the rest is below 2e-7.)
__device__ __forceinline__ LogSum near_log_sum(TileHead h, TileHead more, const TileHead* heads, int tiles, int lane) {
  constexpr float ln2_float = 0.693147182f, ln2_rest = -1.90465421e-09f, off = -1.3349756e-08f;  // (off: as above)
  if (lane >= tiles) h.max = neg_inf();
  if (lane + 32 >= tiles) more.max = neg_inf();
  float m = fmaxf(h.max, more.max);
  for (int t = lane + 64; t < tiles; t += 32) m = fmaxf(m, heads[t].max);
  m = warp_largest(m);
  if (m == neg_inf()) return LogSum{m, 0.0};
  const bool plain = fabsf(m) < PLAIN_LIMIT;
  const float e = plain ? ceilf(m * log2e()) : 0.0f;
  auto part = [&](const TileHead& v) {
    if (!(v.max > neg_inf())) return 0.0;
    if (!plain || v.exponent == OVER_MAX) return part_beyond(v, m, plain ? (int)e : OVER_MAX);
    return v.sum * two_to(v.exponent - (int)e);
  };
  double sum = part(h) + part(more);
  for (int t = lane + 64; t < tiles; t += 32) sum += part(heads[t]);
  float s = (float)sum;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
  float log2_s;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(log2_s) : "f"(s));
  float log = log2_s * ln2_float;
  if (plain) log += (__fmaf_rn(e, ln2_float, -m) + e * ln2_rest) - off * m;
  return LogSum{m, (double)log};
}

// +inf counts as the largest float: the tiles' headers and chunk maxima hold none, and a logit is capped
// where it is read (a NaN stays one)
__device__ __forceinline__ float capped(float x) { return x > largest_float() ? largest_float() : x; }
template <int FMT>
__device__ __forceinline__ float one_logit(const void* logits, size_t at) {
  if (FMT == 0) return capped(static_cast<const float*>(logits)[at]);
  if (FMT == 1) return capped(__bfloat162float(static_cast<const __nv_bfloat16*>(logits)[at]));
  return capped(__half2float(static_cast<const __half*>(logits)[at]));
}

// A row's beam: what turns its logits into ranks
struct Beam {
  double base;     // score of its likeliest continuation, or of the finished beam
  double divisor;  // the length penalty of its continuations
  float max;       // its largest logit
  int state;       // 0 dead, 1 live, 2 finished
};
__device__ __forceinline__ double score_of(const Beam& b, float x) {
  return b.base + ((double)x - (double)b.max);
}
// Ranks to within a margin of themselves and of the beam's reach, scale * (|base| + 16), enough to leave most
// logits out.  The base is off by 2^-17 and its rounding, 2^-24 |base|; the difference x - max, which is at most
// |base| + |sum|, the sum and the product are rounded, 2^-24 each; the scale is off by 2^-15.4 of itself with a
// length penalty (near_scale).  In all scale (2^-17 + 2^-23 |base|) + 3 * 2^-24 |rank|, at most 2^-20.6 of the
// reach and 2^-22.4 of the rank, and 2^-15.4 of the rank with a penalty: twice that, as two ranks are compared,
// is below MARGIN and below PENALTY_MARGIN.  A beam that is not live has a NaN for its base.
constexpr float MARGIN = 1.9073486328125e-06f;         // 2^-19
constexpr float PENALTY_MARGIN = 6.103515625e-05f;     // 2^-14
// All of it is held as a quarter of itself: the lowest value below the largest float, and a score of as much
// again, stay in range (as infinities they would be below everything, whatever their beams' penalties).
struct __align__(16) Near {
  float base, max, scale, pad;  // quarters of the base and the maximum
};
constexpr float NEAR_UNIT = 0.25f;
// as ordered bits; 0 for what is no continuation: no logit, a NaN, or a beam that is not live.  x: at most the
// largest float; a rank that its penalty takes out of float32's range is an infinity.
__device__ __forceinline__ unsigned near_rank(const Near& b, float x) {
  const float v = (b.base + __fmaf_rn(x, NEAR_UNIT, -b.max)) * b.scale;
  return x > neg_inf() && v == v ? ord32(v + 0.0f) : 0u;
}

struct Pick {  // a node, or a logit
  float x;
  int token, beam;  // its (first) token; beam -1: none
};
struct Node {
  double rank;
  unsigned long long key;  // make_key(logit, token)
  int beam;
};
__device__ __forceinline__ Node node_of(const Beam* beams, const Pick& p) {
  const Beam& b = beams[p.beam];
  const double score = score_of(b, p.x);
  return Node{b.divisor == 1.0 ? score : score / b.divisor, make_key(p.x, (uint32_t)p.token), p.beam};
}
__device__ __forceinline__ bool goes_before(const Node& a, const Node& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

// THREADS that go down the levels, EXACT threads behind them, STAGE maxima kept on the chip
template <int THREADS_, int EXACT_, int STAGE_>
struct Level {
  static constexpr int THREADS = THREADS_, EXACT = EXACT_, STAGE = STAGE_;
  float stage[STAGE];  // the tiles' maxima, if they fit
  Beam beams[BM_MAX_BEAMS];
  Near near[BM_MAX_BEAMS];
  float reach;   // largest scale * (|base| + 16) of the live beams, a quarter of it
  float margin;  // how far two near ranks may be off together, relative to theirs and the reach
  Pick list[2][BM_LIST];
  __align__(16) unsigned part_best[BM_PARTS];
  int found[2];  // (one per list: a slow thread may still read one while the next level clears the other)
  Node warp_best[THREADS / 32];
};

// Of a block, the first Level::THREADS threads go down the levels; behind them are warps that meanwhile
// work out the beams' exact bases, which take three times as long as the float32 ones.  A barrier of
// the former, and the one place where they wait for the latter, who only arrive there.
constexpr int BARRIER_LEVELS = 1, BARRIER_EXACT = 2;
template <typename Level>
__device__ __forceinline__ void level_sync() {
  asm volatile("bar.sync %0, %1;" ::"r"(BARRIER_LEVELS), "r"(Level::THREADS) : "memory");
}
template <typename Level>
__device__ __forceinline__ void wait_for_exact(bool& known) {
  if (known) return;
  known = true;
  asm volatile("bar.sync %0, %1;" ::"r"(BARRIER_EXACT), "r"(Level::THREADS + Level::EXACT) : "memory");
}
template <typename Level>
__device__ __forceinline__ void exact_is_known() {
  __threadfence_block();
  asm volatile("bar.arrive %0, %1;" ::"r"(BARRIER_EXACT), "r"(Level::THREADS + Level::EXACT) : "memory");
}

// A level's nodes come in units of 32, one per lane, of one beam:
//   beam(u)            the unit's beam
//   peek(u, k)         the largest logit of the lane's node
//   token(u, k)        its first token
//   each(u, k, visit)  calls visit(logit, token, number) for what the node puts on the list (SELF: the node
//                      itself; else its logits)
// Units of beams that are not live hold nothing, but may be read.  There are no branches where a unit is
// looked at: the block does little else than wait for loads, and a branch between two would have the
// second wait for the first.

// The `want` best, one after the other: what best_nodes comes to where its list would overflow
template <typename Level, typename Unit>
__device__ __noinline__ void one_by_one(Level& L, int which, int units, int want, Unit unit) {
  constexpr int WARPS = Level::THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Node last{0.0, 0ull, -1};
#pragma unroll 1
  for (int r = 0; r < want; ++r) {
    Node mine{0.0, 0ull, -1};
#pragma unroll 1
    for (int u = warp; u < units; u += WARPS) {
      const int k = unit.beam(u);
      unit.each(u, k, [&](float x, int token, int) {
        if (near_rank(L.near[k], x) == 0u) return;
        const Node v = node_of(L.beams, Pick{x, token, k});
        if ((last.beam < 0 || goes_before(last, v)) && (mine.beam < 0 || goes_before(v, mine))) mine = v;
      });
    }
    __syncwarp();
#pragma unroll 1
    for (int d = 16; d > 0; d >>= 1) {
      Node o;
      o.rank = __shfl_xor_sync(FULL, mine.rank, d);
      o.key = __shfl_xor_sync(FULL, mine.key, d);
      o.beam = __shfl_xor_sync(FULL, mine.beam, d);
      if (o.beam >= 0 && (mine.beam < 0 || goes_before(o, mine))) mine = o;
    }
    if (lane == 0) L.warp_best[warp] = mine;
    level_sync<Level>();
    mine = L.warp_best[0];
#pragma unroll 1
    for (int w = 1; w < WARPS; ++w) {
      const Node o = L.warp_best[w];
      if (o.beam >= 0 && (mine.beam < 0 || goes_before(o, mine))) mine = o;
    }
    last = mine;  // (there is one: more than `want` were found)
    if (threadIdx.x == 0) L.list[which][r] = Pick{key_value(last.key), key_id(last.key), last.beam};
    level_sync<Level>();
  }
}

// a near rank's bits less what two of them may be off; 1, which every node reaches, for 0 and for an infinity,
// which says nothing about the ranks behind it (inf - inf would be a NaN, whose bits no node reaches)
template <typename Level>
__device__ __forceinline__ unsigned with_margin(const Level& L, unsigned bits) {
  const float b = unord32(bits);
  return bits > 0u && fabsf(b) <= largest_float() ? ord32(b - L.margin * (fabsf(b) + L.reach) + 0.0f) : 1u;
}

// what is on a list, as units (each lane's of its own beam)
template <typename Level>
struct ListUnit {
  Level& L;
  int which, n;
  __device__ __forceinline__ int at(int u) const { return min(u * 32 + (int)(threadIdx.x & 31), n - 1); }
  __device__ __forceinline__ int beam(int u) const { return L.list[which][at(u)].beam; }
  __device__ __forceinline__ float peek(int u, int) const { return u * 32 + (int)(threadIdx.x & 31) < n ? L.list[which][at(u)].x : neg_inf(); }
};
// A bound that between `want` and `most` of the units' nodes reach, by bisection with counts over the
// block between lo, which enough reach, and hi, which none does; 0 if there is none.
template <typename Level, typename Unit>
__device__ __noinline__ unsigned tighter_bound(Level& L, int units, int want, int most, unsigned lo, unsigned hi, Unit unit) {
  constexpr int WARPS = Level::THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool fits = false;
  level_sync<Level>();
#pragma unroll 1
  for (int round = 0; hi - lo > 1u && !fits; ++round) {
    const unsigned mid = lo + (hi - lo) / 2u;
    int n = 0;
#pragma unroll 4
    for (int u = warp; u < units; u += WARPS) {
      const int k = unit.beam(u);
      n += near_rank(L.near[k], unit.peek(u, k)) >= mid ? 1 : 0;
    }
    n = __reduce_add_sync(FULL, n);
    int* counts = reinterpret_cast<int*>(L.part_best) + (round & 1) * WARPS;  // (in turn: one barrier a round)
    if (lane == 0) counts[warp] = n;
    level_sync<Level>();
    n = 0;
#pragma unroll 1
    for (int w = 0; w < WARPS; ++w) n += counts[w];
    if (n >= want) {
      lo = mid;
      fits = n <= most;
    } else {
      hi = mid;
    }
  }
  level_sync<Level>();
  return fits ? lo : 0u;
}

// Where the best lie close together (masked rows, ramps), one part's best says little about the others' and
// the bound lets too many nodes through.  What has got onto the list, all or some of it, gives a better one;
// where that leads nowhere, the nodes themselves do; and where many ranks are equal, none does.  Returns how
// many reach the best bound found.  (A function of its own, with nothing to go back to: in a loop with the
// common path it made that slower by 1.5 us.)
template <typename Level, typename Unit>
__device__ __noinline__ int fewer_nodes(Level& L, int which, int units, int want, int most, int found, unsigned bound, unsigned top, Unit unit) {
  constexpr int WARPS = Level::THREADS / 32;
#pragma unroll 1
  for (int tries = 0; found > most && tries < 4; ++tries) {
    unsigned next = 0u;
    if (tries < 3) {
      const int n = min(found, BM_LIST);
      next = with_margin(L, tighter_bound(L, (n + 31) / 32, want, 2 * want, bound, top, ListUnit<Level>{L, which, n}));
      if (next <= bound) tries = 3;
    }
    if (tries == 3) {
      if (found <= BM_LIST) break;
      next = with_margin(L, tighter_bound(L, units, want, Unit::SELF ? BM_LIST : BM_LIST / 8, bound, top, unit));
      if (next <= bound) break;
    }
    bound = next;
    if (threadIdx.x == 0) L.found[which] = 0;
    level_sync<Level>();
#pragma unroll 1
    for (int u = threadIdx.x >> 5; u < units; u += WARPS) {
      const int k = unit.beam(u);
      if (near_rank(L.near[k], unit.peek(u, k)) < bound) continue;
      unit.each(u, k, [&](float x, int token, int) {
        if (near_rank(L.near[k], x) < bound) return;
        const int at = atomicAdd(&L.found[which], 1);
        if (at < BM_LIST) L.list[which][at] = Pick{x, token, k};
      });
    }
    level_sync<Level>();
    found = L.found[which];
  }
  return found;
}

// The `want` best nodes, and possibly a few more, into L.list[which], in no order; returns how many.
// Every part of the block takes its best near rank, and each warp finds a bound that at least `want` of
// the parts reach; what is not clearly below it goes on the list.  If that is more than the list holds
// (equal ranks, most of all), the nodes are taken one after the other.
template <typename Level, typename Unit>
__device__ __forceinline__ int best_nodes(Level& L, int which, int units, int want, Unit unit, bool& known) {
  constexpr int THREADS = Level::THREADS, WARPS = THREADS / 32, AHEAD = 4, PER_LANE = BM_PARTS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (units == 0) return 0;
  // 32 parts, one per lane of who compares them, where three times as many as wanted can have any;
  // else BM_PARTS: a bound from too few parts lets too many nodes through
  const bool few = min(units, WARPS) * (32 / WARPS) >= 3 * want;
  struct Batch {
    float x[AHEAD];
    int k[AHEAD];
    unsigned bits[AHEAD];
  };
  auto look = [&](int base, Batch& b) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int u = min(base + a * WARPS, units - 1);
      b.k[a] = unit.beam(u);
      b.x[a] = unit.peek(u, b.k[a]);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) b.bits[a] = base + a * WARPS < units ? near_rank(L.near[b.k[a]], b.x[a]) : 0u;
  };
  Batch first;  // usually all that the warp has
  look(warp, first);
  unsigned best = max(max(first.bits[0], first.bits[1]), max(first.bits[2], first.bits[3]));
#pragma unroll 1
  for (int base = warp + WARPS * AHEAD; base < units; base += WARPS * AHEAD) {
    Batch b;
    look(base, b);
    best = max(best, max(max(b.bits[0], b.bits[1]), max(b.bits[2], b.bits[3])));
  }
  unsigned at_least, top;  // 0: fewer parts than wanted have any; and what no node reaches
  if (few) {
    constexpr int LANES = THREADS / 32;
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) best = max(best, __shfl_xor_sync(FULL, best, d));
    // (the part's number in the last bits, cut off again below: no two are equal)
    if (tid % LANES == 0) L.part_best[tid / LANES] = (best & ~31u) | (unsigned)(tid / LANES);
    if (tid == 0) L.found[which] = 0;
    level_sync<Level>();
    const unsigned mine = L.part_best[lane];
    int before = 0;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&L.part_best[j]);
      before += (o.x > mine ? 1 : 0) + (o.y > mine ? 1 : 0) + (o.z > mine ? 1 : 0) + (o.w > mine ? 1 : 0);
    }
    at_least = __shfl_sync(FULL, mine, __ffs(__ballot_sync(FULL, before == want - 1)) - 1) & ~31u;
    top = (__reduce_max_sync(FULL, mine) | 31u) + 1u;
  } else {
    constexpr int LANES = THREADS / BM_PARTS;
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) best = max(best, __shfl_xor_sync(FULL, best, d));
    if (tid % LANES == 0) L.part_best[tid / LANES] = best;
    if (tid == 0) L.found[which] = 0;
    level_sync<Level>();
    unsigned v[PER_LANE], hi = 0u, lo = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
      v[j] = L.part_best[j * 32 + lane];
      hi = max(hi, v[j]);
      lo = min(lo, v[j]);
    }
    lo = __reduce_min_sync(FULL, want <= 32 ? hi : lo);  // (each lane has one at least as large as its largest)
    hi = top = __reduce_max_sync(FULL, hi) + 1u;
    const int enough = want + want / 2 + 4;
#pragma unroll 1
    while (hi - lo > 1u) {
      const unsigned mid = lo + (hi - lo) / 2u;
      int c = 0;
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) c += v[j] >= mid ? 1 : 0;
      c = __reduce_add_sync(FULL, c);
      if (c >= want) lo = mid; else hi = mid;
      if (c >= want && c <= enough) break;
    }
    at_least = lo;
  }
  unsigned bound = with_margin(L, at_least);  // (0: fewer parts than wanted have any, and all nodes are taken)
  auto collect = [&](int base, const Batch& b) {
    unsigned hits[AHEAD];
    int n = 0;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      hits[a] = __ballot_sync(FULL, b.bits[a] >= bound);
      n += __popc(hits[a]);
    }
    if (n == 0) return;
    if (Unit::SELF) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&L.found[which], n);
      at = __shfl_sync(FULL, at, 0);
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int mine = at + __popc(hits[a] & ((1u << lane) - 1u));
        if ((hits[a] >> lane & 1u) && mine < BM_LIST) L.list[which][mine] = Pick{b.x[a], unit.token(base + a * WARPS, b.k[a]), b.k[a]};
        at += __popc(hits[a]);
      }
    } else {
#pragma unroll 1
      for (int a = 0; a < AHEAD; ++a) {
        const int u = base + a * WARPS;
        if (u >= units || hits[a] == 0u) continue;
        if (hits[a] >> lane & 1u) {
          const int k = unit.beam(u);
          const Near near = L.near[k];
          unsigned some = 0u;
          unit.each(u, k, [&](float x, int, int q) { some |= (near_rank(near, x) >= bound ? 1u : 0u) << q; });
          int at = atomicAdd(&L.found[which], __popc(some));
          unit.each(u, k, [&](float x, int token, int q) {
            if (!(some >> q & 1u)) return;
            if (at < BM_LIST) L.list[which][at] = Pick{x, token, k};
            ++at;
          });
        }
      }
    }
  };
  collect(warp, first);
#pragma unroll 1
  for (int base = warp + WARPS * AHEAD; base < units; base += WARPS * AHEAD) {
    Batch b;
    look(base, b);
    collect(base, b);
  }
  level_sync<Level>();
  int found = L.found[which];
  // a node on the list costs the next level a unit; a logit on the last list costs next to nothing
  const int most = Unit::SELF ? 3 * want + 64 : BM_LIST;
  if (found <= most) return found;
  found = fewer_nodes(L, which, units, want, most, found, bound, top, unit);
  if (found <= BM_LIST) return found;
  wait_for_exact<Level>(known);
  one_by_one(L, which, units, want, unit);
  return want;
}

// Where the levels begin: at the chunks of all tiles, where those make no more than eight units a warp (16 x
// 151936 float32, top 5: 11.0 us, 12.2 from the tiles); at the tiles, their maxima left on the chip by the
// warps that sum rows, or read where they lie.
enum { FROM_TILES, FROM_STAGED_TILES, FROM_CHUNKS };
template <typename Level>
__device__ __forceinline__ int start_of(const Level&, int cells) {
  return cells <= Level::THREADS / 32 * 8 ? FROM_CHUNKS : (cells <= Level::STAGE ? FROM_STAGED_TILES : FROM_TILES);
}

// 32 tiles of a row (STAGED: their maxima are in the block's stage)
template <int FMT, bool STAGED, typename Level>
struct TileUnit {
  static constexpr bool SELF = true;
  Level& L;
  const TileHead* heads;
  int tiles, per_row;
  __device__ __forceinline__ int place(int u, int k) const { return (u - k * per_row) * 32 + (threadIdx.x & 31); }
  __device__ __forceinline__ int beam(int u) const { return u / per_row; }
  __device__ __forceinline__ float peek(int u, int k) const {
    const int t = place(u, k), at = min(t, tiles - 1);
    const float x = STAGED ? L.stage[k * tiles + at] : heads[(size_t)k * tiles + at].max;
    return t < tiles ? x : neg_inf();
  }
  __device__ __forceinline__ int token(int u, int k) const { return place(u, k) * tile_logits(FMT != 0); }
  template <typename Visit>
  __device__ __forceinline__ void each(int u, int k, Visit&& visit) const {
    visit(peek(u, k), token(u, k), 0);
  }
};
// the 32 chunks of a tile: of all the group's tiles, or of those on the list
template <int FMT, bool ALL, typename Level>
struct ChunkUnit {
  static constexpr bool SELF = true;
  static constexpr int TILE = tile_logits(FMT != 0), CHUNK = chunk_logits(FMT != 0);
  Level& L;
  const float* chunk_max;
  int tiles;
  __device__ __forceinline__ int beam(int u) const { return ALL ? u / tiles : L.list[0][u].beam; }
  __device__ __forceinline__ float peek(int u, int k) const {
    const size_t cell = ALL ? (size_t)u : (size_t)k * tiles + L.list[0][u].token / TILE;
    return chunk_max[cell * BT_CHUNKS + (threadIdx.x & 31)];
  }
  __device__ __forceinline__ int token(int u, int k) const {
    return (ALL ? (u - k * tiles) * TILE : L.list[0][u].token) + (int)(threadIdx.x & 31) * CHUNK;
  }
  template <typename Visit>
  __device__ __forceinline__ void each(int u, int k, Visit&& visit) const {
    visit(peek(u, k), token(u, k), 0);
  }
};
// the 32 vectors of a chunk on the list, which put their logits on the next
template <int FMT, bool VEC, typename Level>
struct VectorUnit {
  static constexpr bool SELF = false;
  static constexpr int PER = FMT == 0 ? 4 : 8;
  Level& L;
  const void* logits;
  long long row0, row_stride;
  int vocab;
  __device__ __forceinline__ int beam(int u) const { return L.list[1][u].beam; }
  __device__ __forceinline__ int token(int u, int) const { return L.list[1][u].token + (int)(threadIdx.x & 31) * PER; }
  __device__ __forceinline__ void load(int u, int k, uint32_t (&w)[4]) const {
    constexpr uint32_t none = FMT == 0 ? 0xFF800000u : (FMT == 1 ? 0xFF80FF80u : 0xFC00FC00u);
    const int first = token(u, k);
    const size_t row = (size_t)(row0 + k) * row_stride;
    if (VEC) {
      const size_t at = row + min(first, vocab - PER);
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const char*>(logits) + at * (FMT == 0 ? 4 : 2));
      const bool in = first < vocab;
      w[0] = in ? v.x : none; w[1] = in ? v.y : none; w[2] = in ? v.z : none; w[3] = in ? v.w : none;
    } else if (FMT == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t v = static_cast<const uint32_t*>(logits)[row + min(first + q, vocab - 1)];
        w[q] = first + q < vocab ? v : none;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; q += 2) {
        const unsigned short* const at = static_cast<const unsigned short*>(logits) + row;
        const uint32_t a = at[min(first + q, vocab - 1)], b = at[min(first + q + 1, vocab - 1)];
        w[q >> 1] = (first + q < vocab ? a : none & 0xFFFFu) | (first + q + 1 < vocab ? b << 16 : none & 0xFFFF0000u);
      }
    }
  }
  __device__ __forceinline__ float peek(int u, int k) const {
    uint32_t w[4];
    load(u, k, w);
    return fminf(largest_of<FMT>(w[0], w[1], w[2], w[3]), largest_float());
  }
  template <typename Visit>
  __device__ __forceinline__ void each(int u, int k, Visit&& visit) const {
    uint32_t w[4];
    load(u, k, w);
    const int first = token(u, k);
#pragma unroll
    for (int q = 0; q < PER; ++q) visit(capped(held<FMT>(w, q)), first + q, q);
  }
};

// The `want` best continuations of a group's live rows (and possibly a few more) into L.list[0];
// returns how many.  VEC as for the tiles.
template <int FMT, bool VEC, typename Level>
__device__ __forceinline__ int best_of_rows(Level& L, const TileParams& T, int row0, int rows, int want, int start, bool& known) {
  const size_t cell0 = (size_t)row0 * T.tiles;
  const float* chunk_max = T.chunk_max + cell0 * BT_CHUNKS;
  int n;
  if (start == FROM_CHUNKS) {
    n = best_nodes(L, 1, rows * T.tiles, want, ChunkUnit<FMT, true, Level>{L, chunk_max, T.tiles}, known);
  } else {
    const int per_row = (T.tiles + 31) / 32;
    if (start == FROM_STAGED_TILES)
      n = best_nodes(L, 0, rows * per_row, want, TileUnit<FMT, true, Level>{L, T.heads + cell0, T.tiles, per_row}, known);
    else
      n = best_nodes(L, 0, rows * per_row, want, TileUnit<FMT, false, Level>{L, T.heads + cell0, T.tiles, per_row}, known);
    n = best_nodes(L, 1, n, want, ChunkUnit<FMT, false, Level>{L, chunk_max, T.tiles}, known);
  }
  return best_nodes(L, 0, n, want, VectorUnit<FMT, VEC, Level>{L, T.logits, row0, T.row_stride, T.vocab}, known);
}

// the length penalty: ((5 + length) / 6)^alpha
__device__ __noinline__ double length_divisor(int length, float alpha) {
  return pow((5.0 + (double)max(length, 0)) / 6.0, (double)alpha);
}

// its reciprocal, to within 2^-15.4 of itself for 32-bit lengths and |alpha| up to 4: (5 + length) / 6 is rounded
// four times (2^-21.5 in its log2), lg2.approx is good to 2^-22 of a logarithm of up to 28.5 (2^-17.2), four times
// that and the product's rounding at up to 114 (2^-18) make 3.3e-5 in the exponent, times ln 2 2.3e-5
__device__ __forceinline__ float near_scale(int length, float alpha) {
  float log2_l;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(log2_l) : "f"((5.0f + (float)max(length, 0)) * (1.0f / 6.0f)));
  return ex2(-alpha * log2_l);
}

// a rank as ordered bits, so that candidates compare as whole numbers
__device__ __forceinline__ unsigned long long ord64(double r) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(r + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}

constexpr int BM_EXACT = 256;

// one block per group: THREADS for the levels and BM_EXACT more
template <int THREADS, int FMT, bool VEC>
__global__ void __launch_bounds__(THREADS + BM_EXACT) beam_merge_kernel(const MergeParams P) {
  using GroupLevel = Level<THREADS, BM_EXACT, 4096>;
  __shared__ GroupLevel L;
  __shared__ unsigned long long ranks[BM_LIST + BM_MAX_BEAMS], keys[BM_LIST + BM_MAX_BEAMS];
  __shared__ int owners[BM_LIST + BM_MAX_BEAMS];
  __shared__ int finished_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, tiles = P.T.tiles;
  const int group = blockIdx.x, row0 = group * P.beams;
  const int start = start_of(L, P.beams * tiles);
  if (tid == 0) {
    L.reach = 0.0f;
    L.margin = P.length_penalty == 0.0f ? MARGIN : PENALTY_MARGIN;
    finished_n = 0;
  }
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid >= THREADS) {
    for (int k = warp - THREADS / 32; k < P.beams; k += BM_EXACT / 32) {
      // (a row's first headers are asked for with its score; those of a row that is not live hold nothing)
      const TileHead* heads = P.T.heads + (size_t)(row0 + k) * tiles;
      const TileHead h = heads[min(lane, tiles - 1)];
      const float score = P.T.scores[row0 + k];
      const bool done = P.T.finished && P.T.finished[row0 + k], sound = fabsf(score) <= largest_float();
      LogSum sum = {0.0f, 0.0};
      if (sound && !done) sum = row_log_sum(h, heads, tiles, lane);
      if (lane == 0) {
        const double divisor = P.length_penalty == 0.0f ? 1.0 : length_divisor(P.lengths[row0 + k] + (done ? 0 : 1), P.length_penalty);
        L.beams[k] = Beam{(double)score - sum.log, divisor, sum.max, !sound ? 0 : (done ? 2 : 1)};
      }
    }
    exact_is_known<GroupLevel>();
    return;
  }
  for (int k = warp; k < P.beams; k += THREADS / 32) {
    const TileHead* heads = P.T.heads + (size_t)(row0 + k) * tiles;
    const TileHead h = heads[min(lane, tiles - 1)], more = heads[min(lane + 32, tiles - 1)];
    const float score = P.T.scores[row0 + k];
    const bool live = fabsf(score) <= largest_float() && !(P.T.finished && P.T.finished[row0 + k]);
    const int length = P.length_penalty != 0.0f ? P.lengths[row0 + k] + 1 : 0;
    LogSum sum = {neg_inf(), 0.0};
    if (live) sum = near_log_sum(h, more, heads, tiles, lane);
    if (start == FROM_STAGED_TILES) {
      if (lane < tiles) L.stage[k * tiles + lane] = h.max;
      if (lane + 32 < tiles) L.stage[k * tiles + lane + 32] = more.max;
      for (int t = lane + 64; t < tiles; t += 32) L.stage[k * tiles + t] = heads[t].max;
    }
    if (lane == 0) {
      const float base = score - (float)sum.log;
      const float scale = P.length_penalty == 0.0f ? 1.0f : near_scale(length, P.length_penalty);
      const bool any = sum.max > neg_inf();
      L.near[k] = Near{any ? base * NEAR_UNIT : quiet_nan(), sum.max * NEAR_UNIT, scale, 0.0f};
      if (any) atomicMax(reinterpret_cast<int*>(&L.reach), __float_as_int(scale * ((fabsf(base) + 16.0f) * NEAR_UNIT)));
    }
  }
  level_sync<GroupLevel>();
  bool known = false;
  const int live_n = best_of_rows<FMT, VEC>(L, P.T, row0, P.beams, P.width, start, known);
  wait_for_exact<GroupLevel>(known);
  for (int i = tid; i < live_n; i += THREADS) {
    const Pick p = L.list[0][i];
    const Node v = node_of(L.beams, p);
    ranks[i] = ord64(v.rank);
    keys[i] = v.key;
    owners[i] = v.beam;
  }
  if (P.T.finished)
    for (int k = tid; k < P.beams; k += THREADS)
      if (L.beams[k].state == 2) {
        const int i = live_n + atomicAdd(&finished_n, 1);
        ranks[i] = ord64(L.beams[k].base / L.beams[k].divisor);
        keys[i] = make_key(0.0f, (uint32_t)P.end_id);
        owners[i] = k;
      }
  level_sync<GroupLevel>();
  const int all = live_n + finished_n;
  // each candidate's place: how many go before it, counted by eight lanes
  for (int i0 = 0; i0 < all; i0 += THREADS / 8) {
    const int i = min(i0 + tid / 8, all - 1);
    const unsigned long long rank = ranks[i], key = keys[i];
    const int beam = owners[i];
    int before = 0;
#pragma unroll 2
    for (int j = tid & 7; j < all; j += 8) {
      const unsigned long long r = ranks[j], o = keys[j];
      const int k = owners[j];
      before += (r > rank) | ((r == rank) & ((k < beam) | ((k == beam) & (o > key)))) ? 1 : 0;
    }
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 8; d *= 2) before += __shfl_xor_sync(FULL, before, d);
    if ((tid & 7) != 0 || i0 + tid / 8 >= all || before >= P.width) continue;
    const size_t at = (size_t)group * P.width + before;
    const int token = key_id(key);
    const Beam& b = L.beams[beam];
    const bool was = b.state == 2;
    P.out_tokens[at] = token;
    P.out_parents[at] = beam;
    P.out_scores[at] = (float)(was ? b.base : score_of(b, key_value(key)));
    if (P.out_finished) P.out_finished[at] = was || token == P.end_id ? 1 : 0;
    if (P.out_lengths) P.out_lengths[at] = P.lengths[row0 + beam] + (was ? 0 : 1);
  }
  // places without a continuation: no token, no score, the beam of the place itself as parent
  for (int j = min(all, P.width) + tid; j < P.width; j += THREADS) {
    const size_t at = (size_t)group * P.width + j;
    P.out_tokens[at] = -1;
    P.out_parents[at] = j % P.beams;
    P.out_scores[at] = neg_inf();
    if (P.out_finished) P.out_finished[at] = 0;
    if (P.out_lengths) P.out_lengths[at] = 0;
  }
}

constexpr int LP_THREADS = 128;
constexpr int LP_EXACT = 32;

// one block per row: a warp for the exact sum and the given ids, the others for the likeliest
template <int THREADS, int FMT, bool VEC>
__global__ void __launch_bounds__(THREADS + LP_EXACT) logprob_kernel(const LogprobParams P) {
  using RowLevel = Level<THREADS, LP_EXACT, 1>;
  __shared__ RowLevel L;
  __shared__ unsigned long long keys[BM_LIST];
  const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.x, tiles = P.T.tiles;
  const TileHead* heads = P.T.heads + (size_t)row * tiles;
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid >= THREADS) {
    const LogSum sum = row_log_sum(heads[min(lane, tiles - 1)], heads, tiles, lane);
    const Beam own{-sum.log, 1.0, sum.max, 1};
    if (lane == 0) L.beams[0] = own;
    exact_is_known<RowLevel>();
    for (int g = lane; g < P.given; g += 32) {
      const int id = P.ids[(size_t)row * P.given + g];
      float x = neg_inf();  // ids outside the vocabulary have probability zero
      if (id >= 0 && id < P.T.vocab) x = one_logit<FMT>(P.T.logits, (size_t)row * P.T.row_stride + id);
      P.out_given[(size_t)row * P.given + g] = x > neg_inf() ? (float)score_of(own, x) : neg_inf();  // (NaN as -inf)
    }
    return;
  }
  const int start = start_of(L, tiles) == FROM_CHUNKS ? FROM_CHUNKS : FROM_TILES;
  if (tid < 32) {
    const LogSum sum = near_log_sum(heads[min(lane, tiles - 1)], heads[min(lane + 32, tiles - 1)], heads, tiles, lane);
    if (lane == 0) {
      L.near[0] = Near{sum.max > neg_inf() ? -(float)sum.log * NEAR_UNIT : quiet_nan(), sum.max * NEAR_UNIT, 1.0f, 0.0f};
      L.reach = (fabsf((float)sum.log) + 16.0f) * NEAR_UNIT;
      L.margin = MARGIN;
    }
  }
  level_sync<RowLevel>();
  bool known = false;
  const int all = best_of_rows<FMT, VEC>(L, P.T, row, 1, P.top, start, known);
  wait_for_exact<RowLevel>(known);
  for (int i = tid; i < all; i += THREADS) keys[i] = make_key(L.list[0][i].x, (uint32_t)L.list[0][i].token);
  level_sync<RowLevel>();
  const Beam own = L.beams[0];
  for (int i0 = 0; i0 < all; i0 += THREADS / 8) {
    const unsigned long long key = keys[min(i0 + tid / 8, all - 1)];  // (one beam: its keys' order is the order)
    int before = 0;
#pragma unroll 2
    for (int j = tid & 7; j < all; j += 8) before += keys[j] > key ? 1 : 0;
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 8; d *= 2) before += __shfl_xor_sync(FULL, before, d);
    if ((tid & 7) != 0 || i0 + tid / 8 >= all || before >= P.top) continue;
    P.out_top[(size_t)row * P.top + before] = (float)score_of(own, key_value(key));
    P.out_top_ids[(size_t)row * P.top + before] = key_id(key);
  }
  for (int j = min(all, P.top) + tid; j < P.top; j += THREADS) {
    P.out_top[(size_t)row * P.top + j] = neg_inf();
    P.out_top_ids[(size_t)row * P.top + j] = -1;
  }
}

// and where only given ids are asked for: a warp per row
template <int FMT>
__global__ void __launch_bounds__(LP_THREADS) given_kernel(const LogprobParams P) {
  const int lane = threadIdx.x & 31, row = blockIdx.x * (LP_THREADS / 32) + (threadIdx.x >> 5), tiles = P.T.tiles;
  grid_dependency_wait();
  grid_launch_dependents();
  if (row >= P.T.rows) return;
  const TileHead* heads = P.T.heads + (size_t)row * tiles;
  const TileHead h = heads[min(lane, tiles - 1)];
  float first = neg_inf();
  auto logit = [&](int g) {
    const int id = P.ids[(size_t)row * P.given + g];
    return id >= 0 && id < P.T.vocab ? one_logit<FMT>(P.T.logits, (size_t)row * P.T.row_stride + id) : neg_inf();
  };
  if (lane < P.given) first = logit(lane);
  const LogSum sum = row_log_sum(h, heads, tiles, lane);
  const Beam own{-sum.log, 1.0, sum.max, 1};
  for (int g = lane; g < P.given; g += 32) {
    const float x = g < 32 ? first : logit(g);
    P.out_given[(size_t)row * P.given + g] = x > neg_inf() ? (float)score_of(own, x) : neg_inf();
  }
}

}  // namespace leat
