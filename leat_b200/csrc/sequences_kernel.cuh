// The tokens of every final beam, read back through the parents of all steps.
//
// Final beam k passed through beam b_t(k) at step t: b_{T-1}(k) = k, b_{t-1}(k) = parents[t][b_t(k)].
// Walking that from the end is T dependent loads; but a step's parents are a map of the beams, and
// maps compose associatively.  So a group's steps are cut over the blocks of a cluster, each block's
// steps into runs, one per beams' worth of its threads: every run is walked once for all beams to get
// its map, the maps are composed, four to one each round, and each run is walked again from the beam it
// is known to start at.  Parents and tokens come into shared memory once (cp.async, all in flight
// together); from there the tokens are picked by as many threads as there are tokens and written in
// whole lines, once: where a sequence's first end token lies is settled before.
#pragma once
#include <cooperative_groups.h>

#include "device_util.cuh"

namespace leat {

constexpr int SQ_THREADS = 256;
constexpr int SQ_MAX_BEAMS = 64;
constexpr int SQ_MAX_BLOCKS = 8;       // of a cluster
constexpr int SQ_SHARED = 96 * 1024;   // nine bytes per step and beam: parent, token, path
constexpr int SQ_MOST_SHARED = SQ_SHARED + 3 * 9 * SQ_MAX_BEAMS;  // (with the steps rounded up to a multiple of four)
constexpr unsigned SQ_LOST = 255;      // behind a parent out of range: no beam

struct SequenceParams {
  const int32_t* tokens;   // (steps, groups, beams)
  const int32_t* parents;  // (steps, groups, beams)
  int steps, groups, beams, has_end, end_id;
  int chunk, runs, run_len;  // steps a block takes at a time, the runs it cuts them into, their steps
  int vec;            // beams per load: 4 or 1
  unsigned divide;    // ceil(2^32 / (beams / vec)): quotients by a multiplication
  int32_t* out;          // (groups, beams, steps)
  int32_t* out_lengths;  // (groups, beams)
};

// A barrier over the cluster behind which what a block's first SQ_MAX_BEAMS threads wrote to its shared
// memory can be read by the others.  Only those threads' warps release: a release costs 450 cycles
// (and 1600 with stores to global memory on their way), a relaxed arrival 130.
__device__ __forceinline__ void cluster_publish(int warp) {
  if (warp < SQ_MAX_BEAMS / 32) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// and one that only waits for the other blocks, in two halves
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

__global__ void __launch_bounds__(SQ_THREADS, 6) sequences_kernel(const SequenceParams P) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ unsigned char run_map[2][SQ_THREADS];  // (runs, beams), a round's and the next's
  __shared__ unsigned char block_map[SQ_MAX_BEAMS], carry[SQ_MAX_BEAMS];
  __shared__ unsigned char all_maps[SQ_MAX_BLOCKS][SQ_MAX_BEAMS];
  __shared__ int first_end[SQ_MAX_BEAMS], told_end[SQ_MAX_BEAMS], whole_end[SQ_MAX_BEAMS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const int group = blockIdx.x / blocks, K = P.beams, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cells = P.chunk * K;
  unsigned* const parent = reinterpret_cast<unsigned*>(dynamic);  // (chunk, beams)
  int* const token = reinterpret_cast<int*>(dynamic) + cells;     // (chunk, beams)
  unsigned char* const path = dynamic + (size_t)cells * 8;        // (chunk, beams)
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid < K) {
    carry[tid] = (unsigned char)tid;
    first_end[tid] = whole_end[tid] = P.steps;
  }
  const int sweep = P.chunk * blocks, sweeps = (P.steps + sweep - 1) / sweep;
  const int my_run = tid / K, my_beam = tid - my_run * K;
  const bool walks = my_run < P.runs;
  auto step_back = [&](const unsigned* row, unsigned x) {
    const unsigned p = row[x];
    return p < (unsigned)K ? p : SQ_LOST;
  };
#pragma unroll 1
  for (int at = sweeps - 1; at >= 0; --at) {
    const int begin = min(at * sweep + rank * P.chunk, P.steps), count = min(P.chunk, P.steps - begin);
    if (at < sweeps - 1) {
      __syncthreads();
      if (blocks > 1) {  // (the sweep before has read the other blocks' words)
        cluster_arrive();
        cluster_wait();
      }
    }
    const unsigned per_step = K / P.vec;
    for (unsigned i = tid; i < (unsigned)count * per_step; i += SQ_THREADS) {
      const unsigned t = per_step == 1 ? i : __umulhi(i, P.divide), k = (i - t * per_step) * P.vec;
      const size_t from = ((size_t)(begin + t) * P.groups + group) * K + k;
      const uint32_t a = (uint32_t)__cvta_generic_to_shared(parent + t * K + k), b = (uint32_t)__cvta_generic_to_shared(token + t * K + k);
      if (P.vec == 4) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(P.parents + from) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(b), "l"(P.tokens + from) : "memory");
      } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(a), "l"(P.parents + from) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(b), "l"(P.tokens + from) : "memory");
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const int lo = min(my_run * P.run_len, count), hi = min(lo + P.run_len, count);
    if (walks) {
      unsigned x = my_beam;
      const unsigned* row = parent + (hi - 1) * K;
      for (int t = hi - lo; t > 0 && x != SQ_LOST; --t, row -= K) x = step_back(row, x);
      run_map[0][tid] = (unsigned char)x;
    }
    __syncthreads();
    // run r's map becomes that of all runs from r on
    int now = 0;
    for (int d = 1; d < P.runs; d *= 4, now ^= 1) {
      if (walks) {
        unsigned x = my_beam;
#pragma unroll
        for (int j = 3; j >= 0; --j)
          if (my_run + j * d < P.runs && x != SQ_LOST) x = run_map[now][(my_run + j * d) * K + x];
        run_map[now ^ 1][tid] = (unsigned char)x;
      }
      __syncthreads();
    }
    if (tid < K) block_map[tid] = run_map[now][tid];
    if (blocks > 1) cluster_publish(warp);
    else __syncthreads();
    for (int i = tid; i < blocks * K; i += SQ_THREADS) {
      const int r = i / K;
      all_maps[r][i - r * K] = cluster.map_shared_rank(block_map, r)[i - r * K];
    }
    __syncthreads();
    // the blocks behind this one, then its own runs behind this thread's
    if (walks) {
      unsigned x = carry[my_beam];
      for (int r = blocks - 1; r > rank && x != SQ_LOST; --r) x = all_maps[r][x];
      if (x != SQ_LOST && my_run + 1 < P.runs) x = run_map[now][(my_run + 1) * K + x];
      const int cell = (hi - 1) * K;
      const unsigned* row = parent + cell;
      const int* spoken = token + cell;
      unsigned char* to = path + cell + my_beam;
      int ended = hi - lo;  // steps between the run's first end token and its end
      for (int t = 0; t < hi - lo; ++t, row -= K, spoken -= K, to -= K) {
        *to = (unsigned char)x;
        if (x == SQ_LOST) continue;
        if (spoken[x] == P.end_id) ended = t;
        x = step_back(row, x);
      }
      if (P.has_end && ended < hi - lo) atomicMin(&first_end[my_beam], begin + hi - 1 - ended);
    }
    __syncthreads();
    if (P.has_end) {
      if (tid < K) told_end[tid] = first_end[tid];
      if (blocks > 1) cluster_publish(warp);
      else __syncthreads();
      for (int i = tid; i < blocks * K; i += SQ_THREADS) {
        const int r = i / K;
        atomicMin(&whole_end[i - r * K], cluster.map_shared_rank(told_end, r)[i - r * K]);
      }
    }
    if (at > 0 && tid < K) {
      unsigned y = carry[tid];
      for (int r = blocks - 1; r >= 0 && y != SQ_LOST; --r) y = all_maps[r][y];
      carry[tid] = (unsigned char)y;
    }
    __syncthreads();
    if (at == 0 && blocks > 1) cluster_arrive();  // (this block has read the others' words for the last time)
    // a beam's steps to as many warps as there are for each, or a warp's beams one after the other
    const int warps = SQ_THREADS / 32, share = K < warps ? warps / K : 1, stride = share * 32;
    for (int k = warp / share; k < K; k += warps / share) {
      const int t0 = (warp % share) * 32 + lane, last = whole_end[k] - begin;
      const unsigned char* from = path + t0 * K + k;
      const int* row = token + t0 * K;
      int32_t* const out = P.out + ((size_t)group * K + k) * P.steps + begin;
#pragma unroll 2
      for (int t = t0; t < count; t += stride, from += stride * K, row += stride * K) {
        const unsigned b = *from;
        out[t] = t > last ? P.end_id : (b != SQ_LOST ? row[b] : -1);
      }
    }
  }
  if (rank == 0 && tid < K) P.out_lengths[(size_t)group * K + tid] = P.has_end ? min(whole_end[tid] + 1, P.steps) : P.steps;
  if (blocks > 1 && sweeps > 0) cluster_wait();  // (no block leaves while its words are read)
  // steps that were written before an earlier one turned out to be the end
  if (!P.has_end) return;
  for (int at = sweeps - 1; at > 0; --at) {
    const int begin = min(at * sweep + rank * P.chunk, P.steps), stop = min(begin + P.chunk, P.steps);
    for (int k = warp; k < K; k += SQ_THREADS / 32)
      for (int t = max(begin, whole_end[k] + 1) + lane; t < stop; t += 32) P.out[((size_t)group * K + k) * P.steps + t] = P.end_id;
  }
}

}  // namespace leat
