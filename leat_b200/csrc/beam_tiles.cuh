// One pass over rows of logits for what beam search and log-probabilities need of them: the row's
// sum of exponentials, and where its largest logits are.
//
// log softmax(x)_t = x_t - lse, lse = M + ln(sum exp(x - M)), M = max x.  A row is cut into tiles, a
// block's tile into chunks of adjacent logits, 16 bytes per lane.  Any number near M will do to keep
// the exponentials in range, so a warp takes the maximum of its first chunk and starts on each chunk as
// it arrives; nothing is rescaled, and each logit is read once and costs a maximum, a fused
// multiply-add, an ex2 and an addition.
//
// Nothing is selected here.  What leaves a block is a header (maximum, sum) and the maximum of each of
// the tile's 32 chunks of adjacent logits: 144 bytes of 16 KB read, 0.9 %.  The n largest of any set of nodes
// hold the n largest logits below them, so a handful of tiles, of their chunks and of the chunks'
// logits are all that the few blocks after this pass look at (beam_merge.cuh).
#pragma once
#include "device_util.cuh"

namespace leat {

constexpr int BT_THREADS = 128;
constexpr int BT_WARPS = BT_THREADS / 32;
constexpr int BT_VECS = 8;  // 16-byte loads a thread holds
constexpr int BT_CHUNKS = BT_WARPS * BT_VECS;  // per tile: what a warp loads with one instruction

__host__ __device__ constexpr int chunk_logits(bool half) { return 32 * (half ? 8 : 4); }
__host__ __device__ constexpr int tile_logits(bool half) { return BT_CHUNKS * chunk_logits(half); }

// The exponentials are powers of two over a whole exponent, so that sums of different parts meet by
// exact shifts: sum = sum of 2^(x log2e - exponent), exponent at most ceil(max log2e), log2e the float32
// constant.  Where |max| is PLAIN_LIMIT or more (a tile of nothing but its type's lowest value, say)
// the product's rounding would be felt, and the sum is over max itself: exponent is OVER_MAX then.
struct TileHead {
  float max;  // the tile's largest logit, at most FLT_MAX; -inf: the tile has no logit above -inf
  int exponent;
  double sum;
};
constexpr float PLAIN_LIMIT = 1e5f;
constexpr float FIRST_LIMIT = -1000.0f;  // a chunk below it (masked, as a rule) says nothing about the others
// Chunks that came before one above FIRST_LIMIT have added nothing to the sum: right next to a maximum of
// LOW_LIMIT or more, since e^-100 is far below half a step of float32.
constexpr float LOW_LIMIT = FIRST_LIMIT + 100.0f;
constexpr int OVER_MAX = 0x7FFFFFFF;

struct TileParams {
  const void* logits;
  long long row_stride;
  int rows, vocab, tiles, with_chunks;
  const float* scores;      // rows whose score is not finite are left out (NULL: none)
  const uint8_t* finished;  // and rows that have finished (NULL: none)
  TileHead* heads;          // (rows, tiles)
  float* chunk_max;         // (rows, tiles, BT_CHUNKS), in the logits' order; at most FLT_MAX
};

__device__ __forceinline__ float largest_float() { return __uint_as_float(0x7F7FFFFFu); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the largest of the warp's values; a NaN counts for nothing
__device__ __forceinline__ float warp_largest(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
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

// 2^d for d <= 0, exactly; 0 where that is too small to matter
__device__ __forceinline__ double two_to(int d) { return d > -1000 ? __hiloint2double((1023 + d) << 20, 0) : 0.0; }

// live rows are those that go on; the others' tiles are neither read nor written
__device__ __forceinline__ bool row_is_live(const float* scores, const uint8_t* finished, int row) {
  if (!scores) return true;
  return fabsf(scores[row]) <= largest_float() && !(finished && finished[row]);
}

// FMT 0 float32, 1 bfloat16, 2 float16.  VEC: rows are 16-byte aligned and of whole 16-byte vectors.
// Otherwise, of 16-bit logits, a lane holds the same ones, but they straddle two aligned vectors: it
// loads the first, gets the second from the next lane, and shifts (61 us against 78 with two-byte
// loads for 512 x 262143).  (A vector that holds a logit of the row is read
// whole: no allocation ends inside an aligned 16 bytes.)  The sums are then the same wherever a row
// lies, and equal rows tie.
template <int FMT, bool VEC>
__global__ void __launch_bounds__(BT_THREADS, 7) beam_tile_kernel(const TileParams P) {
  constexpr int PER_VEC = FMT == 0 ? 4 : 8, HELD = BT_VECS * PER_VEC, CHUNK = 32 * PER_VEC;
  __shared__ float chunk_max[BT_CHUNKS];
  __shared__ float warp_max[BT_WARPS], warp_sum[BT_WARPS], warp_e[BT_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.z * gridDim.y + blockIdx.y, tile = blockIdx.x;
  const int begin = tile * (BT_CHUNKS * CHUNK);
  const int size = min(P.vocab - begin, BT_CHUNKS * CHUNK);
  grid_dependency_wait();
  grid_launch_dependents();
  if (row >= P.rows || !row_is_live(P.scores, P.finished, row)) return;

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
    // (four-byte loads are as fast here as the shifts below: 42 us against 45 for 256 x 262143)
    const uint32_t* at = static_cast<const uint32_t*>(P.logits) + (size_t)row * P.row_stride + begin;
#pragma unroll
    for (int q = 0; q < HELD; ++q) {
      const int i = ((q / PER_VEC) * BT_WARPS + warp) * CHUNK + (q % PER_VEC) * 32 + lane;
      w[q] = i < size ? __ldcs(at + i) : 0xFF800000u;
    }
  } else {
    constexpr int SIZE = 2;
    const uint32_t none = FMT == 1 ? 0xFF80FF80u : 0xFC00FC00u;
    const char* const start = static_cast<const char*>(P.logits) + (size_t)row * P.row_stride * SIZE;
    const int off = (int)(reinterpret_cast<uintptr_t>(start) & 15);  // the same for all of a row's vectors
    const char* const at = start - off + (size_t)begin * SIZE;
    const int bytes = off + size * SIZE;  // that hold the tile's logits, from `at` on
#pragma unroll
    for (int u = 0; u < BT_VECS; ++u) {
      const int i = (u * BT_THREADS + tid) * 16;
      uint4 v = make_uint4(none, none, none, none);
      if (i < bytes) v = __ldcs(reinterpret_cast<const uint4*>(at + i));
      w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
    }
    if (off) {
      // lane u: the vector behind the warp's u-th chunk
      uint4 next = make_uint4(none, none, none, none);
      const int after = ((lane % BT_VECS) * BT_THREADS + (warp + 1) * 32) * 16;
      if (lane < BT_VECS && after < bytes) next = *reinterpret_cast<const uint4*>(at + after);
      const uint32_t n[4] = {next.x, next.y, next.z, next.w};
#pragma unroll
      for (int u = 0; u < BT_VECS; ++u) {
        uint32_t v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = w[4 * u + k];
          const uint32_t a = __shfl_down_sync(FULL, v[k], 1), b = __shfl_sync(FULL, n[k], u);
          v[4 + k] = lane == 31 ? b : a;
        }
#pragma unroll
        for (int k = 0; k < 6; ++k) v[k] = (off & 8) ? v[k + 2] : v[k];
#pragma unroll
        for (int k = 0; k < 5; ++k) v[k] = (off & 4) ? v[k + 1] : v[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[4 * u + k] = __funnelshift_r(v[k], v[k + 1], (off & 2) * 8);
      }
    }
    // what lies behind the row's end
    if (size < BT_CHUNKS * CHUNK) {
#pragma unroll
      for (int q = 0; q < HELD; q += 2) {
        const int i = ((q / PER_VEC) * BT_THREADS + tid) * PER_VEC + q % PER_VEC;
        if (i >= size) w[q >> 1] = none;
        else if (i + 1 >= size) w[q >> 1] = (w[q >> 1] & 0xFFFFu) | (none & 0xFFFF0000u);
      }
    }
  }

  float M = neg_inf(), mine = neg_inf(), e = 0.0f;
  bool have_e = false;  // (float32)
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add_chunk = [&](int u) {
#pragma unroll
    for (int q = u * PER_VEC; q < (u + 1) * PER_VEC; ++q) part[q & 3] += ex2(__fmaf_rn(held<FMT>(w, q), log2e(), -e));
  };
#pragma unroll
  for (int u = 0; u < BT_VECS; ++u) {
    const float top = warp_largest(largest_of<FMT>(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]));
    mine = lane == u ? top : mine;
    M = fmaxf(M, top);
    if (FMT == 0) {
      if (!have_e && top > FIRST_LIMIT) {
        have_e = true;
        e = ceilf(fminf(top, PLAIN_LIMIT) * log2e());
      }
      add_chunk(u);
    }
  }
  if (FMT != 0) {
    // (16-bit logits, bound by the number of instructions: all maxima first, so that what is widened
    // for them is not kept for the exponentials, which would spill)
    e = ceilf(M * log2e());
#pragma unroll
    for (int i = 0; i < BT_VECS * 4; ++i) asm volatile("" : "+r"(w[i]));
#pragma unroll
    for (int u = 0; u < BT_VECS; ++u) add_chunk(u);
  }
  if (lane < BT_VECS) chunk_max[lane * BT_WARPS + warp] = mine;
  M = fminf(M, largest_float());  // the warp's own
  const bool empty = M == neg_inf(), plain = fabsf(M) < PLAIN_LIMIT;
  float s = (part[0] + part[1]) + (part[2] + part[3]);
  // once more, from the warp's maximum, where that did not do: the first chunk much below the others
  // (the lanes' sums are still to be added up), a low maximum, large values (differences first), a NaN or
  // +inf.  (M < LOW_LIMIT where no exponent was found, too; but without asking for it the loop above compiles
  // to one that takes 46.3 us for 41.9: 32 x 8 x 262144 with a quarter of the beams finished)
  if (__any_sync(FULL, (FMT == 0 && (!have_e || M < LOW_LIMIT)) || !plain || !(s <= 1e36f))) {
    e = ceilf(M * log2e());
    s = 0.0f;
    // (the words are taken as new here: widened logits kept for this from above would spill)
#pragma unroll
    for (int i = 0; i < BT_VECS * 4 && FMT != 0; ++i) asm volatile("" : "+r"(w[i]));
    if (!empty) {
#pragma unroll
      for (int q = 0; q < HELD; ++q) {
        const float x = held<FMT>(w, q);
        if (x == x) s += plain ? ex2(__fmaf_rn(x, log2e(), -e)) : ex2((fminf(x, largest_float()) - M) * log2e());
      }
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
  if (lane == 0) {
    warp_max[warp] = M;
    warp_sum[warp] = s;
    warp_e[warp] = e;
  }
  __syncthreads();
  const int cell = row * P.tiles + tile;
  if (P.with_chunks && tid < BT_CHUNKS) P.chunk_max[(size_t)cell * BT_CHUNKS + tid] = fminf(chunk_max[tid], largest_float());
  if (warp == BT_WARPS - 1) {
    const float m = lane < BT_WARPS ? warp_max[lane] : neg_inf();
    const float all = warp_largest(m);
    const bool all_plain = fabsf(all) < PLAIN_LIMIT, m_plain = fabsf(m) < PLAIN_LIMIT;
    // the largest exponent of the plain warps (of warps beyond PLAIN_LIMIT: none counts)
    const float m_e = lane < BT_WARPS && m_plain ? warp_e[lane] : neg_inf();
    const float all_e = warp_largest(m_e);
    double sum = 0.0;
    if (lane < BT_WARPS && m > neg_inf()) {
      sum = (double)warp_sum[lane];
      if (all_plain && m_plain) sum *= two_to((int)m_e - (int)all_e);
      else if (all_plain) sum *= (double)ex2(__fmaf_rn(m, log2e(), -all_e));
      else if (m_plain) sum *= (double)ex2(__fmaf_rn(all, -log2e(), m_e));
      else sum *= (double)ex2((m - all) * log2e());
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
