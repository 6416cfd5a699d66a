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
// all tiles, from the chunks of about n tiles, from the logits of about n chunks.
#pragma once
#include "beam_tiles.cuh"

namespace leat {

constexpr int BM_MAX_BEAMS = 64;
constexpr int BM_MAX_WIDTH = 64;
constexpr int BM_LIST = 256;    // nodes a level hands to the next
constexpr int BM_PARTS = 128;   // parts of the block whose best bound a level: at least twice the width

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

template <int FMT>
__device__ __forceinline__ float one_logit(const void* logits, size_t at) {
  if (FMT == 0) return static_cast<const float*>(logits)[at];
  if (FMT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(logits)[at]);
  return __half2float(static_cast<const __half*>(logits)[at]);
}

// A row's beam: what turns its logits into ranks
struct Beam {
  double base;     // score of its likeliest continuation, or of the finished beam
  double divisor;  // the length penalty of its continuations
  float max;       // its largest logit
  float near_base, near_scale;  // base and 1 / divisor, rounded
  int state;       // 0 dead, 1 live, 2 finished
};
// +inf counts as the largest float
__device__ __forceinline__ double score_of(const Beam& b, float x) {
  return b.base + ((double)fminf(x, largest_float()) - (double)b.max);
}
// A rank to within 2^-22 of itself and of the beam's base, enough to leave most logits out: 2 to the
// -24th for each of the base's, the scale's and the difference's rounding and for the sum's and the
// product's.  As ordered bits, never 0; 0 for no logit, or a NaN.
__device__ __forceinline__ unsigned near_rank(const Beam& b, float x) {
  return x > neg_inf() ? ord32((b.near_base + (x - b.max)) * b.near_scale + 0.0f) : 0u;
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

template <int THREADS>
struct Level {
  Beam beams[BM_MAX_BEAMS];
  float reach;  // largest |near_base * near_scale| of the beams
  Pick list[2][BM_LIST];
  unsigned part_best[BM_PARTS];
  int found[2];  // (one per list: a slow thread may still read one while the next level clears the other)
  Node warp_best[THREADS / 32];
  Pick warp_pick[THREADS / 32];
};

// The `want` best nodes, one after the other: what best_nodes comes to where its list would overflow
template <int THREADS, typename Each>
__device__ __noinline__ void one_by_one(Level<THREADS>& L, int which, int n, int want, Each each) {
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Node last{0.0, 0ull, -1};
#pragma unroll 1
  for (int r = 0; r < want; ++r) {
    Node mine{0.0, 0ull, -1};
#pragma unroll 1
    for (int i = tid; i < n; i += THREADS)
      each(i, [&](float x, int k, int token) {
        if (!(x > neg_inf())) return;
        const Node v = node_of(L.beams, Pick{x, token, k});
        if ((last.beam < 0 || goes_before(last, v)) && (mine.beam < 0 || goes_before(v, mine))) mine = v;
      });
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
    __syncthreads();
    mine = L.warp_best[0];
#pragma unroll 1
    for (int w = 1; w < WARPS; ++w) {
      const Node o = L.warp_best[w];
      if (o.beam >= 0 && (mine.beam < 0 || goes_before(o, mine))) mine = o;
    }
    last = mine;  // (there is one: more than `want` were found)
    if (tid == 0) L.list[which][r] = Pick{key_value(last.key), key_id(last.key), last.beam};
    __syncthreads();
  }
}

// The `want` best of n nodes, and possibly a few more, into L.list[which], in no order; returns how
// many.  Every part of the block takes its best near rank, and each warp finds, by bisection, a bound
// that at least `want` of the parts reach; what is not clearly below it goes on the list.  If that is
// more than the list holds (equal ranks, most of all), the nodes are taken one after the other.
//   peek(i, beam): node i's largest logit, and its beam
//   each(i, visit): calls visit(logit, beam, first token) for what node i puts on the list: itself,
//                   or, at the last level, its logits
template <int THREADS, typename Peek, typename Each>
__device__ __forceinline__ int best_nodes(Level<THREADS>& L, int which, int n, int want, Peek peek, Each each) {
  constexpr int LANES = THREADS / BM_PARTS, AHEAD = 4, PER_LANE = BM_PARTS / 32;
  const int tid = threadIdx.x, lane = tid & 31;
  unsigned first[AHEAD];  // of the thread's first nodes: usually all it has
  unsigned best = 0u;
  auto look = [&](int base, unsigned (&bits)[AHEAD]) {
    float x[AHEAD];
    int beam[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = base + a * THREADS + tid;
      x[a] = neg_inf();
      beam[a] = 0;
      if (i < n) x[a] = peek(i, beam[a]);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) bits[a] = near_rank(L.beams[beam[a]], x[a]);
  };
  look(0, first);
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) best = max(best, first[a]);
#pragma unroll 1
  for (int base = THREADS * AHEAD; base < n; base += THREADS * AHEAD) {
    unsigned bits[AHEAD];
    look(base, bits);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) best = max(best, bits[a]);
  }
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) best = max(best, __shfl_xor_sync(FULL, best, d));
  if (tid % LANES == 0) L.part_best[tid / LANES] = best;
  if (tid == 0) L.found[which] = 0;
  __syncthreads();
  unsigned bound;
  {
    unsigned v[PER_LANE], hi = 0u, lo = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
      v[j] = L.part_best[j * 32 + lane];
      hi = max(hi, v[j]);
      lo = min(lo, v[j]);
    }
    lo = __reduce_min_sync(FULL, want <= 32 ? hi : lo);  // (each lane has one at least as large as its largest)
    hi = __reduce_max_sync(FULL, hi) + 1u;
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
    bound = 1u;  // (0: fewer parts than wanted have any; all nodes are taken)
    if (lo > 0u) {
      const float b = unord32(lo);
      if (b > neg_inf()) bound = ord32(b - 9.5367431640625e-07f * (fabsf(b) + L.reach) + 0.0f);  // 2^-20: both sides' errors
    }
  }
  auto put = [&](float x, int k, int token) {
    if (near_rank(L.beams[k], x) >= bound) {
      const int at = atomicAdd(&L.found[which], 1);
      if (at < BM_LIST) L.list[which][at] = Pick{x, token, k};
    }
  };
#pragma unroll 1
  for (int base = 0; base < n; base += THREADS * AHEAD) {
    unsigned bits[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) bits[a] = first[a];
    if (base > 0) look(base, bits);
    unsigned hits = 0u;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) hits |= (bits[a] >= bound ? 1u : 0u) << a;
#pragma unroll 1
    while (hits) {
      const int a = __ffs(hits) - 1;
      hits &= hits - 1u;
      each(base + a * THREADS + tid, put);
    }
  }
  __syncthreads();
  const int found = L.found[which];
  if (found <= BM_LIST) return found;
  one_by_one<THREADS>(L, which, n, want, each);
  return want;
}

// The `want` best continuations of a group's live rows (and possibly a few more) into L.list[0];
// returns how many.  VEC as for the tiles.
template <int THREADS, int FMT, bool VEC>
__device__ __forceinline__ int best_of_rows(Level<THREADS>& L, const TileParams& T, int row0, int rows, int want) {
  constexpr int PER = FMT == 0 ? 4 : 8, CHUNK = 32 * PER, TILE = BT_CHUNKS * CHUNK;
  const int tiles = T.tiles;
  const TileHead* heads = T.heads + (size_t)row0 * tiles;
  const float* chunk_max = T.chunk_max + (size_t)row0 * tiles * BT_CHUNKS;
  auto itself = [](auto peek, auto token_of) {
    return [=](int i, auto&& visit) {
      int k;
      const float x = peek(i, k);
      visit(x, k, token_of(i, k));
    };
  };
  // tiles, unless there are so few that their chunks may as well be looked at
  int n = rows * tiles;
  const bool narrow = n > 2 * want && n * (long long)BT_CHUNKS > 4 * THREADS;
  if (narrow) {
    auto peek = [=, &L](int i, int& k) {
      k = i / tiles;
      return L.beams[k].state == 1 ? heads[i].max : neg_inf();
    };
    auto token_of = [=](int i, int k) { return (i - k * tiles) * TILE; };
    n = best_nodes<THREADS>(L, 0, n, want, peek, itself(peek, token_of));
  }
  {
    auto place = [=, &L](int i, int& k) {  // chunk of the group (below 2^31: checked on the host)
      const int t = i / BT_CHUNKS, c = i % BT_CHUNKS;
      if (!narrow) {
        k = t / tiles;
        return i;
      }
      k = L.list[0][t].beam;
      return (k * tiles + L.list[0][t].token / TILE) * BT_CHUNKS + c;
    };
    auto peek = [=, &L](int i, int& k) {
      const int at = place(i, k);
      return L.beams[k].state == 1 ? chunk_max[at] : neg_inf();
    };
    auto token_of = [=](int i, int) {
      int k;
      const int at = place(i, k);
      return (at - k * tiles * BT_CHUNKS) * CHUNK;
    };
    n = best_nodes<THREADS>(L, 1, n * BT_CHUNKS, want, peek, itself(peek, token_of));
  }
  // a node is 16 bytes of a chunk; it puts its logits on the list
  auto load = [=, &L, &T](int i, int& k, int& token, uint32_t (&w)[4]) {
    const Pick& chunk = L.list[1][i / 32];
    k = chunk.beam;
    token = chunk.token + (i % 32) * PER;
    const size_t at = (size_t)(row0 + k) * T.row_stride + token;
    const uint32_t none = FMT == 0 ? 0xFF800000u : (FMT == 1 ? 0xFF80FF80u : 0xFC00FC00u);
    w[0] = w[1] = w[2] = w[3] = none;
    if (VEC) {
      if (token < T.vocab) {
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const char*>(T.logits) + at * (FMT == 0 ? 4 : 2));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      }
    } else if (FMT == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (token + q < T.vocab) w[q] = static_cast<const uint32_t*>(T.logits)[at + q];
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (token + q < T.vocab) {
          const uint32_t v = static_cast<const unsigned short*>(T.logits)[at + q];
          w[q >> 1] = (q & 1) ? (w[q >> 1] & 0xFFFFu) | (v << 16) : (w[q >> 1] & 0xFFFF0000u) | v;
        }
    }
  };
  auto peek = [=](int i, int& k) {
    int token;
    uint32_t w[4];
    load(i, k, token, w);
    return largest_of<FMT>(w[0], w[1], w[2], w[3]);
  };
  auto each = [=](int i, auto&& visit) {
    int k, token;
    uint32_t w[4];
    load(i, k, token, w);
#pragma unroll
    for (int q = 0; q < PER; ++q) visit(held<FMT>(w, q), k, token + q);
  };
  return best_nodes<THREADS>(L, 0, n * 32, want, peek, each);
}

// the length penalty: ((5 + length) / 6)^alpha
__device__ __noinline__ double length_divisor(int length, float alpha) {
  return pow((5.0 + (double)max(length, 0)) / 6.0, (double)alpha);
}

// one block per group
template <int THREADS, int FMT, bool VEC>
__global__ void __launch_bounds__(THREADS) beam_merge_kernel(const MergeParams P) {
  constexpr int WARPS = THREADS / 32;
  __shared__ Level<THREADS> L;
  __shared__ Node candidates[BM_LIST + BM_MAX_BEAMS];
  __shared__ int finished_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = blockIdx.x, row0 = group * P.beams;
  if (tid == 0) {
    L.reach = 0.0f;
    finished_n = 0;
  }
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();
  for (int k = warp; k < P.beams; k += WARPS) {
    // (a row's first headers are asked for with its score; those of a row that is not live hold nothing)
    const TileHead* heads = P.T.heads + (size_t)(row0 + k) * P.T.tiles;
    TileHead h = {neg_inf(), 0, 0.0};
    if (lane < P.T.tiles) h = heads[lane];
    const float score = P.T.scores[row0 + k];
    const bool done = P.T.finished && P.T.finished[row0 + k];
    const bool live = fabsf(score) <= largest_float() && !done;
    LogSum sum = {0.0f, 0.0};
    if (live) sum = row_log_sum(h, heads, P.T.tiles, lane);
    if (lane == 0) {
      Beam b;
      b.base = (double)score - sum.log;
      b.max = sum.max;
      b.state = live && sum.max > neg_inf() ? 1 : (done && fabsf(score) <= largest_float() ? 2 : 0);
      b.divisor = P.length_penalty == 0.0f ? 1.0 : length_divisor(P.lengths[row0 + k] + (done ? 0 : 1), P.length_penalty);
      b.near_base = (float)b.base;
      b.near_scale = (float)(1.0 / b.divisor);
      L.beams[k] = b;
      if (b.state == 1) atomicMax(reinterpret_cast<int*>(&L.reach), __float_as_int(fabsf(b.near_base * b.near_scale)));
    }
  }
  __syncthreads();
  const int live_n = best_of_rows<THREADS, FMT, VEC>(L, P.T, row0, P.beams, P.width);
  for (int i = tid; i < live_n; i += THREADS) candidates[i] = node_of(L.beams, L.list[0][i]);
  if (P.T.finished)
    for (int k = tid; k < P.beams; k += THREADS)
      if (L.beams[k].state == 2)
        candidates[live_n + atomicAdd(&finished_n, 1)] = Node{L.beams[k].base / L.beams[k].divisor, make_key(0.0f, (uint32_t)P.end_id), k};
  __syncthreads();
  const int all = live_n + finished_n;
  for (int i = tid; i < all; i += THREADS) {
    const Node c = candidates[i];
    int before = 0;
    for (int j = 0; j < all; ++j) before += goes_before(candidates[j], c) ? 1 : 0;
    if (before >= P.width) continue;
    const size_t at = (size_t)group * P.width + before;
    const int token = key_id(c.key);
    const Beam& b = L.beams[c.beam];
    const bool was = b.state == 2;
    P.out_tokens[at] = token;
    P.out_parents[at] = c.beam;
    P.out_scores[at] = (float)(was ? b.base : score_of(b, key_value(c.key)));
    if (P.out_finished) P.out_finished[at] = was || token == P.end_id ? 1 : 0;
    if (P.out_lengths) P.out_lengths[at] = P.lengths[row0 + c.beam] + (was ? 0 : 1);
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

// one block per row
template <int FMT, bool VEC>
__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(const LogprobParams P) {
  __shared__ Level<LP_THREADS> L;
  __shared__ unsigned long long keys[BM_LIST];
  const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.x;
  grid_dependency_wait();
  grid_launch_dependents();
  const TileHead* heads = P.T.heads + (size_t)row * P.T.tiles;
  TileHead h = {neg_inf(), 0, 0.0};
  if (lane < P.T.tiles) h = heads[lane];
  const LogSum sum = row_log_sum(h, heads, P.T.tiles, lane);
  const Beam own{-sum.log, 1.0, sum.max, (float)-sum.log, 1.0f, sum.max > neg_inf() ? 1 : 0};
  for (int g = tid; g < P.given; g += LP_THREADS) {
    const int id = P.ids[(size_t)row * P.given + g];
    float x = neg_inf();  // ids outside the vocabulary have probability zero
    if (id >= 0 && id < P.T.vocab) x = one_logit<FMT>(P.T.logits, (size_t)row * P.T.row_stride + id);
    P.out_given[(size_t)row * P.given + g] = x > neg_inf() ? (float)score_of(own, x) : neg_inf();  // (NaN as -inf)
  }
  if (P.top == 0) return;
  if (tid == 0) {
    L.beams[0] = own;
    L.reach = fabsf(own.near_base);
  }
  __syncthreads();
  const int all = best_of_rows<LP_THREADS, FMT, VEC>(L, P.T, row, 1, P.top);
  for (int i = tid; i < all; i += LP_THREADS) keys[i] = make_key(L.list[0][i].x, (uint32_t)L.list[0][i].token);
  __syncthreads();
  for (int i = tid; i < all; i += LP_THREADS) {
    const unsigned long long key = keys[i];  // (one beam: its keys' order is the order)
    int before = 0;
    for (int j = 0; j < all; ++j) before += keys[j] > key ? 1 : 0;
    if (before >= P.top) continue;
    P.out_top[(size_t)row * P.top + before] = (float)score_of(own, key_value(key));
    P.out_top_ids[(size_t)row * P.top + before] = key_id(key);
  }
  for (int j = min(all, P.top) + tid; j < P.top; j += LP_THREADS) {
    P.out_top[(size_t)row * P.top + j] = neg_inf();
    P.out_top_ids[(size_t)row * P.top + j] = -1;
  }
}

}  // namespace leat
