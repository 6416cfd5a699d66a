// The tokens of every final beam, read back through the parents of all steps.
//
// Final beam k passed through beam b_t(k) at step t: b_{T-1}(k) = k, b_{t-1}(k) = parents[t][b_t(k)].
// Walking that from the end is T dependent loads; but a step's parents are a map of the beams, and
// maps compose associatively.  So a group's steps are cut over the blocks of a cluster, each block's
// steps into runs: every run is walked once for all beams to get its map (in shared memory), the few
// maps are composed, and each run is walked again from the beam it is known to start at.  The tokens
// are then gathered by as many threads as there are tokens.  Bound by latency for one request and by
// reading parents and tokens once for many.
#pragma once
#include <cooperative_groups.h>

#include "device_util.cuh"

namespace leat {

constexpr int SQ_THREADS = 256;
constexpr int SQ_MAX_BEAMS = 64;
constexpr int SQ_SHARED = 96 * 1024;  // parents and path of a block's steps, one byte each
constexpr int SQ_LOST = 255;          // behind a parent out of range: no beam

struct SequenceParams {
  const int32_t* tokens;   // (steps, groups, beams)
  const int32_t* parents;  // (steps, groups, beams)
  int steps, groups, beams, has_end, end_id;
  int chunk, runs;  // steps a block takes at a time, and the runs it cuts them into
  int32_t* out;          // (groups, beams, steps)
  int32_t* out_lengths;  // (groups, beams)
};

__global__ void __launch_bounds__(SQ_THREADS) sequences_kernel(const SequenceParams P) {
  namespace cg = cooperative_groups;
  extern __shared__ unsigned char dynamic[];
  __shared__ unsigned char run_map[SQ_THREADS], run_entry[SQ_THREADS];  // (runs, beams)
  __shared__ unsigned char block_map[SQ_MAX_BEAMS], carry[SQ_MAX_BEAMS], entry[SQ_MAX_BEAMS];
  __shared__ int first_end[SQ_MAX_BEAMS], whole_end[SQ_MAX_BEAMS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const int group = blockIdx.x / blocks, K = P.beams, tid = threadIdx.x;
  unsigned char* const parent = dynamic;               // (chunk, beams)
  unsigned char* const path = dynamic + P.chunk * K;   // (chunk, beams)
  grid_dependency_wait();
  grid_launch_dependents();
  if (tid < K) {
    carry[tid] = (unsigned char)tid;
    first_end[tid] = P.steps;
  }
  const int run_len = (P.chunk + P.runs - 1) / P.runs;
  const int sweep = P.chunk * blocks, sweeps = (P.steps + sweep - 1) / sweep;
  const int my_run = tid / K, my_beam = tid - my_run * K;
  const bool walks = my_run < P.runs;
#pragma unroll 1
  for (int at = sweeps - 1; at >= 0; --at) {
    const int begin = min(at * sweep + rank * P.chunk, P.steps), count = min(P.chunk, P.steps - begin);
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < count * K; i += SQ_THREADS) {
      const int t = i / K, k = i - t * K;
      const int p = P.parents[((size_t)(begin + t) * P.groups + group) * K + k];
      parent[i] = (unsigned char)(p >= 0 && p < K ? p : SQ_LOST);
    }
    __syncthreads();
    const int lo = min(my_run * run_len, count), hi = min(lo + run_len, count);
    if (walks) {
      int x = my_beam;
      for (int t = hi - 1; t >= lo && x != SQ_LOST; --t) x = parent[t * K + x];
      run_map[tid] = (unsigned char)x;
    }
    __syncthreads();
    if (tid < K) {
      int x = tid;
      for (int r = P.runs - 1; r >= 0; --r) {
        run_entry[r * K + tid] = (unsigned char)x;
        if (x != SQ_LOST) x = run_map[r * K + x];
      }
      block_map[tid] = (unsigned char)x;
    }
    cluster.sync();
    if (tid < K) {
      int x = carry[tid];
      for (int r = blocks - 1; r >= 0; --r) {
        if (r == rank) entry[tid] = (unsigned char)x;
        if (x != SQ_LOST) x = cluster.map_shared_rank(block_map, r)[x];
      }
      carry[tid] = (unsigned char)x;
    }
    cluster.sync();  // (every block has read the maps, and the block its entries)
    if (walks) {
      int x = entry[my_beam];
      if (x != SQ_LOST) x = run_entry[my_run * K + x];
      for (int t = hi - 1; t >= lo; --t) {
        path[t * K + my_beam] = (unsigned char)x;
        if (x != SQ_LOST) x = parent[t * K + x];
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < count * K; i += SQ_THREADS) {
      const int k = i / count, t = i - k * count;
      const int x = path[t * K + k];
      const int token = x != SQ_LOST ? P.tokens[((size_t)(begin + t) * P.groups + group) * K + x] : -1;
      P.out[((size_t)group * K + k) * P.steps + begin + t] = token;
      if (P.has_end && token == P.end_id) atomicMin(&first_end[k], begin + t);
    }
  }
  // behind a sequence's first end token there is nothing but that token
  cluster.sync();
  if (tid < K) {
    int first = P.steps;
    for (int r = 0; r < blocks; ++r) first = min(first, cluster.map_shared_rank(first_end, r)[tid]);
    whole_end[tid] = first;
    if (rank == 0) P.out_lengths[(size_t)group * K + tid] = min(first + 1, P.steps);
  }
  cluster.sync();  // (no block leaves while its words are read)
  if (!P.has_end) return;
#pragma unroll 1
  for (int at = sweeps - 1; at >= 0; --at) {
    const int begin = min(at * sweep + rank * P.chunk, P.steps), stop = min(begin + P.chunk, P.steps);
    for (int k = tid >> 5; k < K; k += SQ_THREADS / 32)
      for (int t = max(begin, whole_end[k] + 1) + (tid & 31); t < stop; t += 32)
        P.out[((size_t)group * K + k) * P.steps + t] = P.end_id;
  }
}

}  // namespace leat
