// One pass over rows of logits for what beam search and log-probabilities need of them: the row's
// sum of exponentials, and where its largest logits are.
//
// log softmax(x)_t = x_t - lse, lse = M + ln(sum exp(x - M)), M = max x.  A row is cut into tiles; a
// block holds a whole tile in registers and a warp knows its part's maximum before its first
// exponential, so nothing is rescaled: each logit is read once and costs a maximum, a fused
// multiply-add, an ex2 and an addition.
//
// Nothing is selected here.  What leaves a block is a header (maximum, sum) and the maximum of each of
// the tile's 64 chunks of adjacent logits: 1 % of what was read.  The n largest of any set of nodes
// hold the n largest logits below them, so a handful of tiles, of their chunks and of the chunks'
// logits are all that the few blocks after this pass look at (beam_merge.cuh).
#pragma once
#include "device_util.cuh"

namespace leat {

constexpr int BT_THREADS = 256;
constexpr int BT_WARPS = BT_THREADS / 32;
constexpr int BT_VECS = 8;  // 16-byte loads a thread holds
constexpr int BT_CHUNKS = BT_WARPS * BT_VECS;  // per tile: what a warp loads with one instruction

__host__ __device__ constexpr int chunk_logits(bool half) { return 32 * (half ? 8 : 4); }
__host__ __device__ constexpr int tile_logits(bool half) { return BT_CHUNKS * chunk_logits(half); }

// The exponentials are powers of two over a whole exponent, so that sums of different parts meet by
// exact shifts: sum = sum of 2^(x log2e - exponent), exponent = ceil(max log2e), log2e the float32
// constant.  Where |max| is PLAIN_LIMIT or more (a tile of nothing but its type's lowest value, say)
// the product's rounding would be felt, and the sum is over max itself: exponent is OVER_MAX then.
struct TileHead {
  float max;  // the tile's largest logit, at most FLT_MAX; -inf: the tile has no logit above -inf
  int exponent;
  double sum;
};
constexpr float PLAIN_LIMIT = 1e5f;
constexpr int OVER_MAX = 0x7FFFFFFF;

struct TileParams {
  const void* logits;
  long long row_stride;
  int vocab, tiles, with_chunks;
  const float* scores;      // rows whose score is not finite are left out (NULL: none)
  const uint8_t* finished;  // and rows that have finished (NULL: none)
  TileHead* heads;          // (rows, tiles)
  float* chunk_max;         // (rows, tiles, BT_CHUNKS), in the logits' order
};

__device__ __forceinline__ float largest_float() { return __uint_as_float(0x7F7FFFFFu); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the q-th logit in a thread's words, as float32 (16-bit formats widen exactly)
template <int FMT, int WORDS>
__device__ __forceinline__ float held(const uint32_t (&w)[WORDS], int q) {
  if (FMT == 0) return __uint_as_float(w[q]);
  const uint32_t h = w[q >> 1];
  if (FMT == 1) return __uint_as_float((q & 1) ? (h & 0xFFFF0000u) : (h << 16));
  return __half2float(__ushort_as_half((unsigned short)((q & 1) ? (h >> 16) : (h & 0xFFFFu))));
}
// the largest of the logits in four words (a NaN is passed over, so that it counts as -inf)
template <int FMT>
__device__ __forceinline__ float largest_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  if (FMT == 0)
    return fmaxf(fmaxf(fmaxf(__uint_as_float(a), __uint_as_float(b)), fmaxf(__uint_as_float(c), __uint_as_float(d))), neg_inf());
  if (FMT == 1) {
    auto pair = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
    const __nv_bfloat162 m = __hmax2(__hmax2(pair(a), pair(b)), __hmax2(pair(c), pair(d)));
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), neg_inf());
  }
  auto pair = [](uint32_t v) { return *reinterpret_cast<const __half2*>(&v); };
  const __half2 m = __hmax2(__hmax2(pair(a), pair(b)), __hmax2(pair(c), pair(d)));
  return fmaxf(fmaxf(__low2float(m), __high2float(m)), neg_inf());
}

// 2^d for d <= 0, exactly; 0 where that is no normal float
__device__ __forceinline__ float two_to(int d) { return d >= -126 ? __int_as_float((127 + d) << 23) : 0.0f; }

// live rows are those that go on; the others' tiles are neither read nor written
__device__ __forceinline__ bool row_is_live(const float* scores, const uint8_t* finished, int row) {
  if (!scores) return true;
  return fabsf(scores[row]) <= largest_float() && !(finished && finished[row]);
}

// FMT 0 float32, 1 bfloat16, 2 float16.  VEC: rows are 16-byte aligned and of whole 16-byte vectors;
// otherwise a warp loads the same chunks one logit per lane at a time.
template <int FMT, bool VEC>
__global__ void __launch_bounds__(BT_THREADS, 4) beam_tile_kernel(const TileParams P) {
  constexpr int PER_VEC = FMT == 0 ? 4 : 8, HELD = BT_VECS * PER_VEC, CHUNK = 32 * PER_VEC;
  __shared__ float chunk_max[BT_CHUNKS];
  __shared__ float warp_max[BT_WARPS], warp_sum[BT_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / P.tiles, tile = blockIdx.x - row * P.tiles;
  const int begin = tile * (BT_CHUNKS * CHUNK);
  const int size = min(P.vocab - begin, BT_CHUNKS * CHUNK);
  grid_dependency_wait();
  grid_launch_dependents();
  if (!row_is_live(P.scores, P.finished, row)) return;

  // chunk u * BT_WARPS + warp of the tile is the warp's u-th
  uint32_t w[BT_VECS * 4];
  if (VEC) {
    const char* at = static_cast<const char*>(P.logits) + ((size_t)row * P.row_stride + begin) * (FMT == 0 ? 4 : 2);
    const uint32_t none = FMT == 0 ? 0xFF800000u : (FMT == 1 ? 0xFF80FF80u : 0xFC00FC00u);
#pragma unroll
    for (int u = 0; u < BT_VECS; ++u) {
      const int i = (u * BT_THREADS + tid) * PER_VEC;
      uint4 v = make_uint4(none, none, none, none);
      if (i < size) v = __ldcs(reinterpret_cast<const uint4*>(at) + u * BT_THREADS + tid);
      w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
    }
  } else if (FMT == 0) {
    const uint32_t* at = static_cast<const uint32_t*>(P.logits) + (size_t)row * P.row_stride + begin;
#pragma unroll
    for (int q = 0; q < HELD; ++q) {
      const int i = ((q / PER_VEC) * BT_WARPS + warp) * CHUNK + (q % PER_VEC) * 32 + lane;
      w[q] = i < size ? __ldcs(at + i) : 0xFF800000u;
    }
  } else {
    const unsigned short* at = static_cast<const unsigned short*>(P.logits) + (size_t)row * P.row_stride + begin;
    const uint32_t none = FMT == 1 ? 0xFF80u : 0xFC00u;
#pragma unroll
    for (int q = 0; q < HELD; q += 2) {
      const int i = ((q / PER_VEC) * BT_WARPS + warp) * CHUNK + (q % PER_VEC) * 32 + lane;
      const uint32_t a = i < size ? (uint32_t)__ldcs(at + i) : none;
      const uint32_t b = i + 32 < size ? (uint32_t)__ldcs(at + i + 32) : none;
      w[q >> 1] = a | (b << 16);
    }
  }

  unsigned top_bits = 0u;
#pragma unroll
  for (int u = 0; u < BT_VECS; ++u) {
    const unsigned bits = __reduce_max_sync(FULL, ord32(largest_of<FMT>(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]) + 0.0f));
    if (lane == u) chunk_max[u * BT_WARPS + warp] = unord32(bits);
    top_bits = max(top_bits, bits);
  }
  const float M = fminf(unord32(top_bits), largest_float());  // the warp's own
  const bool empty = M == neg_inf();

  const bool plain = fabsf(M) < PLAIN_LIMIT;
  const float e = ceilf(M * log2e());
  float s = 0.0f;
  bool direct = !plain;  // differences first: for large values, and for threads that hold a NaN or +inf
  // (the words are taken as new from here on: widened logits kept from the maxima's pass would spill)
#pragma unroll
  for (int i = 0; i < BT_VECS * 4; ++i) asm volatile("" : "+r"(w[i]));
  if (plain) {
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < HELD; ++q) part[q & 3] += ex2(__fmaf_rn(held<FMT>(w, q), log2e(), -e));
    s = (part[0] + part[1]) + (part[2] + part[3]);
    direct = !(s <= largest_float());
  }
  if (direct && !empty) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < BT_VECS * 4; ++i) asm volatile("" : "+r"(w[i]));
#pragma unroll
    for (int q = 0; q < HELD; ++q) {
      const float x = held<FMT>(w, q);
      if (x == x) s += plain ? ex2(__fmaf_rn(x, log2e(), -e)) : ex2((fminf(x, largest_float()) - M) * log2e());
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
  if (lane == 0) {
    warp_max[warp] = M;
    warp_sum[warp] = s;
  }
  __syncthreads();
  const int cell = row * P.tiles + tile;
  if (P.with_chunks && tid < BT_CHUNKS) P.chunk_max[(size_t)cell * BT_CHUNKS + tid] = chunk_max[tid];
  if (warp == BT_WARPS - 1) {
    const float m = lane < BT_WARPS ? warp_max[lane] : neg_inf();
    const float all = unord32(__reduce_max_sync(FULL, ord32(m + 0.0f)));
    const bool all_plain = fabsf(all) < PLAIN_LIMIT, m_plain = fabsf(m) < PLAIN_LIMIT;
    const float all_e = ceilf(all * log2e()), m_e = ceilf(m * log2e());
    double sum = 0.0;
    if (lane < BT_WARPS && m > neg_inf()) {
      float scale;
      if (all_plain && m_plain) scale = two_to((int)m_e - (int)all_e);
      else if (all_plain) scale = ex2(__fmaf_rn(m, log2e(), -all_e));
      else if (m_plain) scale = ex2(__fmaf_rn(all, -log2e(), m_e));
      else scale = ex2((m - all) * log2e());
      sum = (double)(warp_sum[lane] * scale);
    }
#pragma unroll
    for (int d = BT_WARPS / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(FULL, sum, d);
    if (lane == 0) {
      TileHead h;
      h.max = all;
      h.exponent = all_plain ? (int)all_e : OVER_MAX;
      h.sum = sum;
      P.heads[cell] = h;
    }
  }
}

}  // namespace leat
