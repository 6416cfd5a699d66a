// From the tiles' headers and candidates (beam_tiles.cuh) to answers: a group's best continuations,
// or a row's log-probabilities.
//
// A continuation (beam k, token t) has score_k + x_t - lse_k and is ranked by that over its length's
// penalty.  Sums, scores and ranks are held in 64 bits: what is compared differs between beams by
// their lse, and float32 ranks near -100 would tie where the sums do not.  Order: the larger rank,
// then the lower beam, then the larger logit, then the lower token.
#pragma once
#include "beam_tiles.cuh"

namespace leat {

constexpr int BM_MAX_BEAMS = 64;
constexpr int BM_SHORT = 512;  // continuations that reach the bound and are then ordered

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
  int fmt, given, top;
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
__device__ __forceinline__ LogSum row_log_sum(const TileHead* heads, int tiles, int lane) {
  float m = neg_inf();
  for (int t = lane; t < tiles; t += 32) m = fmaxf(m, heads[t].max);
  m = unord32(__reduce_max_sync(FULL, ord32(m + 0.0f)));
  double s = 0.0;
  if (m > neg_inf())
    for (int t = lane; t < tiles; t += 32) {
      const TileHead h = heads[t];
      if (h.max > neg_inf()) s += h.sum * exp((double)h.max - (double)m);
    }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
  return LogSum{m, m > neg_inf() ? log(s) : 0.0};
}

struct Continuation {
  double rank;
  unsigned long long key;  // make_key(logit, token)
  int beam;
};
__device__ __forceinline__ bool goes_before(const Continuation& a, const Continuation& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}
// a key's logit less its row's maximum; +inf counts as the largest float
__device__ __forceinline__ double below_max(unsigned long long key, float max) {
  return (double)fminf(key_value(key), largest_float()) - (double)max;
}

// one block per group
template <int THREADS>
__global__ void __launch_bounds__(THREADS) beam_merge_kernel(const MergeParams P) {
  constexpr int WARPS = THREADS / 32, AHEAD = 4;
  __shared__ double base[BM_MAX_BEAMS];     // score of the likeliest continuation, or of a finished beam
  __shared__ float row_max[BM_MAX_BEAMS];
  __shared__ double divisor[BM_MAX_BEAMS];  // the length penalty of its continuations
  __shared__ signed char state[BM_MAX_BEAMS];  // 0 dead, 1 live, 2 finished
  __shared__ unsigned thread_best[THREADS];
  __shared__ Continuation chosen[BM_SHORT];
  __shared__ Continuation warp_best[WARPS];
  __shared__ unsigned bound_bits;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = blockIdx.x, row0 = group * P.beams, tiles = P.T.tiles;
  const TileHead* heads = P.T.heads + (size_t)row0 * tiles;
  const unsigned long long* lists = P.T.lists + (size_t)row0 * tiles * P.T.places;
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) found = 0;
  for (int k = warp; k < P.beams; k += WARPS) {
    const float score = P.T.scores[row0 + k];
    const bool finished = P.T.finished && P.T.finished[row0 + k];
    const bool live = row_is_live(P.T.scores, P.T.finished, row0 + k);
    LogSum sum = {0.0f, 0.0};
    if (live) sum = row_log_sum(heads + (size_t)k * tiles, tiles, lane);
    if (lane == 0) {
      base[k] = (double)score - sum.log;
      row_max[k] = sum.max;
      state[k] = live ? 1 : (finished && fabsf(score) <= largest_float() ? 2 : 0);
      divisor[k] = P.length_penalty == 0.0f ? 1.0
                   : pow((5.0 + (double)(P.lengths[row0 + k] + (finished ? 0 : 1))) / 6.0, (double)P.length_penalty);
    }
  }
  __syncthreads();

  const int segments = P.beams * tiles;
  auto live_one = [&](int k, unsigned long long key) {
    return Continuation{(base[k] + below_max(key, row_max[k])) / divisor[k], key, k};
  };
  // every continuation of the group, a warp per tile's list
  auto each = [&](auto&& visit) {
    for (int k = tid; k < P.beams; k += THREADS)
      if (state[k] == 2) visit(Continuation{base[k] / divisor[k], make_key(0.0f, (uint32_t)P.end_id), k});
#pragma unroll 1
    for (int first = warp; first < segments; first += WARPS * AHEAD) {
      int n[AHEAD], beam[AHEAD];
      unsigned long long key[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int seg = first + a * WARPS;
        beam[a] = seg < segments ? seg / tiles : 0;
        n[a] = seg < segments && state[beam[a]] == 1 ? heads[seg].n : 0;
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        if (lane < n[a]) key[a] = lists[(size_t)(first + a * WARPS) * P.T.places + lane];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        if (lane < n[a]) visit(live_one(beam[a], key[a]));
        for (int i = lane + 32; i < n[a]; i += 32) {
          const unsigned long long more = lists[(size_t)(first + a * WARPS) * P.T.places + i];
          visit(live_one(beam[a], more));
        }
      }
    }
  };

  // a rank that at least `width` continuations reach: the width-th best of the threads' best
  // (rounded down to float32, so that nothing at or above it is missed)
  unsigned best = 0u;
  each([&](const Continuation& c) { best = max(best, ord32(__double2float_rd(c.rank) + 0.0f)); });
  thread_best[tid] = best;
  __syncthreads();
  if (warp == 0) {
    unsigned v[WARPS], hi = 0u;
#pragma unroll
    for (int j = 0; j < WARPS; ++j) {
      v[j] = thread_best[j * 32 + lane];
      hi = max(hi, v[j]);
    }
    unsigned lo = 0u;  // (0: threads without any; everything is taken)
    hi = __reduce_max_sync(FULL, hi) + 1u;
#pragma unroll 1
    while (hi - lo > 1u) {
      const unsigned mid = lo + (hi - lo) / 2u;
      int c = 0;
#pragma unroll
      for (int j = 0; j < WARPS; ++j) c += v[j] >= mid ? 1 : 0;
      c = __reduce_add_sync(FULL, c);
      if (c >= P.width) lo = mid; else hi = mid;
      if (c == P.width) break;
    }
    if (lane == 0) bound_bits = lo;
  }
  __syncthreads();
  const unsigned bound = bound_bits;
  each([&](const Continuation& c) {
    if (ord32(__double2float_rd(c.rank) + 0.0f) >= bound) {
      const int at = atomicAdd(&found, 1);
      if (at < BM_SHORT) chosen[at] = c;
    }
  });
  __syncthreads();
  const int all = found;

  auto write = [&](int j, const Continuation& c) {
    const size_t at = (size_t)group * P.width + j;
    const int token = key_id(c.key);
    const bool was = state[c.beam] == 2;
    P.out_tokens[at] = token;
    P.out_parents[at] = c.beam;
    P.out_scores[at] = (float)(was ? base[c.beam] : base[c.beam] + below_max(c.key, row_max[c.beam]));
    if (P.out_finished) P.out_finished[at] = was || token == P.end_id ? 1 : 0;
    if (P.out_lengths) P.out_lengths[at] = P.lengths[row0 + c.beam] + (was ? 0 : 1);
  };
  int n;
  if (all <= BM_SHORT) {
    n = min(all, P.width);
    for (int i = tid; i < all; i += THREADS) {
      const Continuation c = chosen[i];
      int before = 0;
      for (int j = 0; j < all; ++j) before += goes_before(chosen[j], c) ? 1 : 0;
      if (before < P.width) write(before, c);
    }
  } else {
    // too many equal ranks (or all large ones with few threads): one after the other, each the best
    // of those after the last
    Continuation last{0.0, 0ull, -1};
    n = 0;
#pragma unroll 1
    for (; n < P.width; ++n) {
      Continuation mine{0.0, 0ull, -1};
      each([&](const Continuation& c) {
        if ((last.beam < 0 || goes_before(last, c)) && (mine.beam < 0 || goes_before(c, mine))) mine = c;
      });
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        Continuation o;
        o.rank = __shfl_xor_sync(FULL, mine.rank, d);
        o.key = __shfl_xor_sync(FULL, mine.key, d);
        o.beam = __shfl_xor_sync(FULL, mine.beam, d);
        if (o.beam >= 0 && (mine.beam < 0 || goes_before(o, mine))) mine = o;
      }
      __syncthreads();  // (the round before has been read)
      if (lane == 0) warp_best[warp] = mine;
      __syncthreads();
      mine = warp_best[0];
#pragma unroll 1
      for (int w = 1; w < WARPS; ++w) {
        const Continuation o = warp_best[w];
        if (o.beam >= 0 && (mine.beam < 0 || goes_before(o, mine))) mine = o;
      }
      last = mine;  // (there is one: more than `width` were counted)
      if (tid == 0) write(n, last);
    }
  }
  // places without a continuation: no token, no score, the beam of the place itself as parent
  for (int j = n + tid; j < P.width; j += THREADS) {
    const size_t at = (size_t)group * P.width + j;
    P.out_tokens[at] = -1;
    P.out_parents[at] = j % P.beams;
    P.out_scores[at] = neg_inf();
    if (P.out_finished) P.out_finished[at] = 0;
    if (P.out_lengths) P.out_lengths[at] = 0;
  }
}

constexpr int LP_THREADS = 128;
constexpr int LP_SHORT = 512;

// one block per row
__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(const LogprobParams P) {
  constexpr int WARPS = LP_THREADS / 32;
  __shared__ unsigned thread_best[LP_THREADS];
  __shared__ unsigned long long chosen[LP_SHORT];
  __shared__ unsigned long long warp_best[WARPS];
  __shared__ unsigned bound_bits;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, tiles = P.T.tiles;
  const TileHead* heads = P.T.heads + (size_t)row * tiles;
  const unsigned long long* lists = P.T.lists + (size_t)row * tiles * P.T.places;
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid == 0) found = 0;
  const LogSum sum = row_log_sum(heads, tiles, lane);
  for (int g = tid; g < P.given; g += LP_THREADS) {
    const int id = P.ids[(size_t)row * P.given + g];
    float x = neg_inf();  // ids outside the vocabulary have probability zero
    if (id >= 0 && id < P.T.vocab) {
      const size_t at = (size_t)row * P.T.row_stride + id;
      if (P.fmt == 0) x = static_cast<const float*>(P.T.logits)[at];
      else if (P.fmt == 1) x = __bfloat162float(static_cast<const __nv_bfloat16*>(P.T.logits)[at]);
      else x = __half2float(static_cast<const __half*>(P.T.logits)[at]);
    }
    P.out_given[(size_t)row * P.given + g] =
        x > neg_inf() ? (float)((double)fminf(x, largest_float()) - (double)sum.max - sum.log) : neg_inf();  // (NaN as -inf)
  }
  if (P.top == 0) return;

  auto each = [&](auto&& visit) {
#pragma unroll 1
    for (int t = warp; t < tiles; t += WARPS) {
      const int n = heads[t].n;
      for (int i = lane; i < n; i += 32) visit(lists[(size_t)t * P.T.places + i]);
    }
  };
  unsigned best = 0u;
  each([&](unsigned long long key) { best = max(best, key_vbits(key)); });
  thread_best[tid] = best;
  __syncthreads();
  if (warp == 0) {
    unsigned v[WARPS], hi = 0u, lo = 0u;
#pragma unroll
    for (int j = 0; j < WARPS; ++j) {
      v[j] = thread_best[j * 32 + lane];
      hi = max(hi, v[j]);
    }
    hi = __reduce_max_sync(FULL, hi) + 1u;
#pragma unroll 1
    while (hi - lo > 1u) {
      const unsigned mid = lo + (hi - lo) / 2u;
      int c = 0;
#pragma unroll
      for (int j = 0; j < WARPS; ++j) c += v[j] >= mid ? 1 : 0;
      c = __reduce_add_sync(FULL, c);
      if (c >= P.top) lo = mid; else hi = mid;
      if (c == P.top) break;
    }
    if (lane == 0) bound_bits = lo;
  }
  __syncthreads();
  const unsigned bound = bound_bits;
  each([&](unsigned long long key) {
    if (key_vbits(key) >= bound) {
      const int at = atomicAdd(&found, 1);
      if (at < LP_SHORT) chosen[at] = key;
    }
  });
  __syncthreads();
  const int all = found;
  auto write = [&](int j, unsigned long long key) {
    P.out_top[(size_t)row * P.top + j] = (float)(below_max(key, sum.max) - sum.log);
    P.out_top_ids[(size_t)row * P.top + j] = key_id(key);
  };
  int n;
  if (all <= LP_SHORT) {
    n = min(all, P.top);
    for (int i = tid; i < all; i += LP_THREADS) {
      const unsigned long long key = chosen[i];
      int before = 0;
      for (int j = 0; j < all; ++j) before += chosen[j] > key ? 1 : 0;
      if (before < P.top) write(before, key);
    }
  } else {
    unsigned long long last = ~0ull;
    n = 0;
#pragma unroll 1
    for (; n < P.top; ++n) {
      unsigned long long mine = 0ull;
      each([&](unsigned long long key) { if (key < last && key > mine) mine = key; });
      mine = warp_max_u64(mine);
      __syncthreads();
      if (lane == 0) warp_best[warp] = mine;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WARPS; ++w) mine = warp_best[w] > mine ? warp_best[w] : mine;
      last = mine;
      if (tid == 0) write(n, last);
    }
  }
  for (int j = n + tid; j < P.top; j += LP_THREADS) {
    P.out_top[(size_t)row * P.top + j] = neg_inf();
    P.out_top_ids[(size_t)row * P.top + j] = -1;
  }
}

}  // namespace leat
