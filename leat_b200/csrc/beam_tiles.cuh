// One pass over rows of logits for what beam search and log-probabilities need of them: the row's
// sum of exponentials and its largest logits.
//
// log softmax(x)_t = x_t - lse, lse = M + ln(sum exp(x - M)), M = max x.  A row is cut into tiles; a
// block holds a whole tile in registers, so its maximum is known before the first exponential and
// nothing is rescaled: each logit is read once and costs a maximum, a fused multiply-add, an ex2 and
// an addition.  The tile's `top` largest logits are the row's only candidates that lie in it.  They
// are found without ordering anything: the top-th largest of the block's 256 thread maxima is a
// logit that at least `top` logits of the tile reach, and few more do.
//
// What leaves a block: a header (maximum, sum, number of candidates) and the candidates, unordered,
// in a place of their own, so that no word is shared between blocks and nothing needs clearing.
#pragma once
#include "device_util.cuh"

namespace leat {

constexpr int BT_THREADS = 256;
constexpr int BT_WARPS = BT_THREADS / 32;
constexpr int BT_VECS = 8;        // 16-byte loads a thread holds
constexpr int BT_MAX_TOP = 64;
constexpr int BT_SLACK = 32;      // places a tile has for candidates beyond its `top`

constexpr int tile_logits(bool half) { return BT_THREADS * BT_VECS * (half ? 8 : 4); }

struct TileHead {
  float max;   // the tile's largest logit, at most FLT_MAX; -inf: the tile has no logit above -inf
  int n;       // candidates
  double sum;  // sum of exp(x - max)
};

struct TileParams {
  const void* logits;
  long long row_stride;
  int vocab, tiles, top, places;  // places: room per tile for candidates, top + BT_SLACK
  const float* scores;            // rows whose score is not finite are left out (NULL: none)
  const uint8_t* finished;        // and rows that have finished (NULL: none)
  TileHead* heads;                // (rows, tiles)
  unsigned long long* lists;      // (rows, tiles, places) make_key(logit, id)
};

__device__ __forceinline__ float largest_float() { return __uint_as_float(0x7F7FFFFFu); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the q-th logit a thread holds, as float32 (16-bit formats widen exactly)
template <int FMT>
__device__ __forceinline__ float held(const uint32_t (&w)[BT_VECS * 4], int q) {
  if (FMT == 0) return __uint_as_float(w[q]);
  const uint32_t h = w[q >> 1];
  if (FMT == 1) return __uint_as_float((q & 1) ? (h & 0xFFFF0000u) : (h << 16));
  return __half2float(__ushort_as_half((unsigned short)((q & 1) ? (h >> 16) : (h & 0xFFFFu))));
}

template <int FMT, bool VEC>
struct Tile {
  static constexpr int PER_VEC = FMT == 0 ? 4 : 8;
  static constexpr int HELD = BT_VECS * PER_VEC;
  // place in the tile of the q-th logit of thread tid
  static __device__ __forceinline__ int place(int q, int tid) {
    return VEC ? ((q / PER_VEC) * BT_THREADS + tid) * PER_VEC + q % PER_VEC : q * BT_THREADS + tid;
  }
};

// live rows are those that go on; the others' tiles are neither read nor written
__device__ __forceinline__ bool row_is_live(const float* scores, const uint8_t* finished, int row) {
  if (!scores) return true;
  return fabsf(scores[row]) <= largest_float() && !(finished && finished[row]);
}

__device__ __forceinline__ int block_count(int mine, int* scratch, int round) {
  // scratch: 2 * BT_WARPS words, used in turn so that one barrier per count is enough
  int* at = scratch + (round & 1) * BT_WARPS;
  const int sum = __reduce_add_sync(FULL, mine);
  if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = sum;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < BT_WARPS; ++w) all += at[w];
  return all;
}

// FMT 0 float32, 1 bfloat16, 2 float16.  VEC: rows are 16-byte aligned and of whole 16-byte vectors.
template <int FMT, bool VEC, bool TOP>
__global__ void __launch_bounds__(BT_THREADS, 4) beam_tile_kernel(const TileParams P) {
  using L = Tile<FMT, VEC>;
  __shared__ unsigned thread_max[BT_THREADS];
  __shared__ double warp_sum[BT_WARPS];
  __shared__ int count[2 * BT_WARPS];
  __shared__ unsigned floor_bits;
  __shared__ int found;
  __shared__ unsigned long long list[TOP ? BT_MAX_TOP + BT_SLACK : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / P.tiles, tile = blockIdx.x - row * P.tiles;
  const int begin = tile * (BT_THREADS * L::HELD);
  const int size = min(P.vocab - begin, BT_THREADS * L::HELD);
  grid_dependency_wait();
  grid_launch_dependents();
  if (!row_is_live(P.scores, P.finished, row)) return;

  uint32_t w[BT_VECS * 4];
  if (VEC) {
    const char* at = static_cast<const char*>(P.logits) + ((size_t)row * P.row_stride + begin) * (FMT == 0 ? 4 : 2);
    const uint32_t none = FMT == 0 ? 0xFF800000u : (FMT == 1 ? 0xFF80FF80u : 0xFC00FC00u);
#pragma unroll
    for (int u = 0; u < BT_VECS; ++u) {
      const int i = (u * BT_THREADS + tid) * L::PER_VEC;
      uint4 v = make_uint4(none, none, none, none);
      if (i < size) v = __ldcs(reinterpret_cast<const uint4*>(at) + u * BT_THREADS + tid);
      w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
    }
  } else if (FMT == 0) {
    const uint32_t* at = static_cast<const uint32_t*>(P.logits) + (size_t)row * P.row_stride + begin;
#pragma unroll
    for (int q = 0; q < L::HELD; ++q) {
      const int i = q * BT_THREADS + tid;
      w[q] = i < size ? __ldcs(at + i) : 0xFF800000u;
    }
  } else {
    const unsigned short* at = static_cast<const unsigned short*>(P.logits) + (size_t)row * P.row_stride + begin;
    const uint32_t none = FMT == 1 ? 0xFF80u : 0xFC00u;
#pragma unroll
    for (int q = 0; q < L::HELD; q += 2) {
      const int i = q * BT_THREADS + tid;
      const uint32_t a = i < size ? (uint32_t)__ldcs(at + i) : none;
      const uint32_t b = i + BT_THREADS < size ? (uint32_t)__ldcs(at + i + BT_THREADS) : none;
      w[q >> 1] = a | (b << 16);
    }
  }

  // (fmaxf passes over a NaN, which therefore counts as -inf here and, below, in every comparison)
  float mine = neg_inf();
#pragma unroll
  for (int q = 0; q < L::HELD; ++q) mine = fmaxf(mine, held<FMT>(w, q));
  thread_max[tid] = ord32(mine + 0.0f);
  if (tid == 0) found = 0;
  __syncthreads();
  unsigned top_bits;
  {
    unsigned v[BT_WARPS], hi = 0u, lo = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < BT_WARPS; ++j) {
      v[j] = thread_max[j * 32 + lane];
      hi = max(hi, v[j]);
      lo = min(lo, v[j]);
    }
    top_bits = __reduce_max_sync(FULL, hi);
    if (TOP && warp == 0) {
      // bisection for a value that `top` of the 256 reach: lo always is one, hi never
      lo = __reduce_min_sync(FULL, lo);
      hi = top_bits + 1u;
#pragma unroll 1
      while (hi - lo > 1u) {
        const unsigned mid = lo + (hi - lo) / 2u;
        int c = 0;
#pragma unroll
        for (int j = 0; j < BT_WARPS; ++j) c += v[j] >= mid ? 1 : 0;
        c = __reduce_add_sync(FULL, c);
        if (c >= P.top) lo = mid; else hi = mid;
        if (c == P.top) break;
      }
      if (lane == 0) floor_bits = lo;
    }
  }
  float M = unord32(top_bits);
  const bool empty = M == neg_inf();
  M = fminf(M, largest_float());

  // sum of 2^(x log2e - c), c = fl(M log2e): the one rounding of c, at most 2^-7 here, is taken back
  // at the end.  Larger values, and threads that hold a NaN or +inf, take the differences first.
  const float c = M * log2e();
  const bool plain = fabsf(M) < 1e5f;
  float s = 0.0f;
  bool direct = !plain;
  if (plain) {
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int q = 0; q < L::HELD; q += 2) {
      s0 += ex2(__fmaf_rn(held<FMT>(w, q), log2e(), -c));
      s1 += ex2(__fmaf_rn(held<FMT>(w, q + 1), log2e(), -c));
    }
    s = s0 + s1;
    direct = !(s <= largest_float());
  }
  if (direct && !empty) {
    s = 0.0f;
#pragma unroll
    for (int q = 0; q < L::HELD; ++q) {
      const float x = held<FMT>(w, q);
      if (x == x) s += ex2((fminf(x, largest_float()) - M) * log2e());
    }
  }
  if (plain && !direct) s *= ex2(__fmaf_rn(-log2e(), M, c));
  double sum = (double)s;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(FULL, sum, d);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();

  const int tile_at = row * P.tiles + tile;
  int n = 0;
  if (TOP) {
    const float floor = fmaxf(unord32(floor_bits), -largest_float());  // -inf is no candidate
    if (mine >= floor) {
#pragma unroll
      for (int q = 0; q < L::HELD; ++q) {
        const float x = held<FMT>(w, q);
        if (x >= floor) {
          const int at = atomicAdd(&found, 1);
          if (at < P.places) list[at] = make_key(x, (uint32_t)(begin + L::place(q, tid)));
        }
      }
    }
    __syncthreads();
    n = found;
    if (n > P.places) {
      // more than there is room for (equal logits, or large ones held by few threads): exactly the
      // `top` best, the lower id first among equals, by bisection with counts over the block
      unsigned lo = ord32(floor + 0.0f), hi = top_bits + 1u;
      int round = 0, above = 0;  // logits at or above hi
      {
        int m = 0;
#pragma unroll
        for (int q = 0; q < L::HELD; ++q) m += held<FMT>(w, q) > floor ? 1 : 0;
        m = block_count(m, count, round++);
        if (m < P.top) { hi = lo + 1u; above = m; }
      }
#pragma unroll 1
      while (hi - lo > 1u) {
        const unsigned mid = lo + (hi - lo) / 2u;
        const float v = unord32(mid);
        int m = 0;
#pragma unroll
        for (int q = 0; q < L::HELD; ++q) m += held<FMT>(w, q) >= v ? 1 : 0;
        m = block_count(m, count, round++);
        if (m >= P.top) lo = mid; else { hi = mid; above = m; }
      }
      // the top-th largest is `value`; of its equals, those at places below `bound` go along
      const float value = unord32(lo);
      int from = 0, bound = size;  // (places at or above 0 below `bound`: enough; below `from`: too few)
#pragma unroll 1
      while (bound - from > 1) {
        const int mid = (from + bound) / 2;
        int m = 0;
#pragma unroll
        for (int q = 0; q < L::HELD; ++q) m += (held<FMT>(w, q) == value && L::place(q, tid) < mid) ? 1 : 0;
        m = block_count(m, count, round++);
        if (m >= P.top - above) bound = mid; else from = mid;
      }
      __syncthreads();
      if (tid == 0) found = 0;
      __syncthreads();
#pragma unroll
      for (int q = 0; q < L::HELD; ++q) {
        const float x = held<FMT>(w, q);
        if (x > value || (x == value && L::place(q, tid) < bound)) {
          const int at = atomicAdd(&found, 1);
          if (at < P.places) list[at] = make_key(x, (uint32_t)(begin + L::place(q, tid)));
        }
      }
      __syncthreads();
      n = min(found, P.places);
    }
    if (tid < n) P.lists[(size_t)tile_at * P.places + tid] = list[tid];
  }
  if (tid == 0) {
    TileHead h;
    h.max = M;
    h.n = n;
    h.sum = 0.0;
#pragma unroll
    for (int i = 0; i < BT_WARPS; ++i) h.sum += warp_sum[i];
    if (empty) h.sum = 0.0;
    P.heads[tile_at] = h;
  }
}

}  // namespace leat
