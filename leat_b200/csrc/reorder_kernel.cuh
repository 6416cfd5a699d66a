// Rows of caches and other per-beam states follow their beams, in place: state[row(g, k)] takes
// state[row(g, parents[g][k])], for the positions of a range, over many tensors in one launch.
//
// It is bound by memory: a row that moves is written once, a row that some moved beam came from is
// read once, and rows that stay are not touched.  In place needs no second copy of the cache,
// because a column (the same few bytes of every row of a group) is read whole before any of it is
// written, and a column belongs to one thread: its copies go through the thread's own words of
// shared memory (cp.async, so that all rows' loads are in flight at once whatever the registers
// hold) and no barrier orders them.
#pragma once
#include "device_util.cuh"

namespace leat {

constexpr int RO_THREADS = 128;
constexpr int RO_MAX_BEAMS = 64;
constexpr int RO_TWICE_BEAMS = 16;  // up to this many, two columns a thread
constexpr int RO_MAX_STATES = 64;  // tensors per launch: 3 KB of kernel parameters

struct StateRows {  // sizes and strides in bytes
  char* data;
  long long row_stride, outer_stride, place_bytes;
  int outer, places, rows, pad;
};

struct ReorderParams {
  StateRows states[RO_MAX_STATES];
  const int32_t* parents;  // (groups, beams)
  const int32_t* slots;    // (groups, beams) state rows, or NULL: group * beams + beam
  const int32_t* start;    // (groups) or NULL
  const int32_t* end;      // (groups) or NULL
  int start_all, end_all;  // where NULL
  int beams;
};

template <int UNIT>
__device__ __forceinline__ void column_load(void* shared, const char* from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(shared);
  if (UNIT == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else if (UNIT == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at), "l"(from) : "memory");
  else if (UNIT == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
  else if (UNIT == 2) *static_cast<uint16_t*>(shared) = *reinterpret_cast<const uint16_t*>(from);
  else *static_cast<uint8_t*>(shared) = *reinterpret_cast<const uint8_t*>(from);
}
template <int UNIT>
__device__ __forceinline__ void column_store(char* to, const void* shared) {
  if (UNIT == 16) *reinterpret_cast<uint4*>(to) = *static_cast<const uint4*>(shared);
  else if (UNIT == 8) *reinterpret_cast<uint2*>(to) = *static_cast<const uint2*>(shared);
  else if (UNIT == 4) *reinterpret_cast<uint32_t*>(to) = *static_cast<const uint32_t*>(shared);
  else if (UNIT == 2) *reinterpret_cast<uint16_t*>(to) = *static_cast<const uint16_t*>(shared);
  else *reinterpret_cast<uint8_t*>(to) = *static_cast<const uint8_t*>(shared);
}

// UNIT: bytes per load.  TWICE: two columns of 16 bytes a thread, so that a block reads and writes 4 KB of
// a row at a time, where that many rows' columns fit an SM more than once (64 rows of 8 groups, 8 caches
// of 268 MB, 4 KB runs and 148 * 128 blocks: 6.39 TB/s read and written, the measured copy's rate 0.99
// times; 2 KB runs and 148 * 32 blocks: 5.97).
// grid (blocks along a group's columns, groups, tensors); dynamic shared memory: a column's bytes for
// every beam and thread
__host__ __device__ constexpr int column_bytes(bool twice) { return twice ? 32 : 16; }
template <int UNIT, bool TWICE>
__global__ void __launch_bounds__(RO_THREADS) reorder_kernel(const __grid_constant__ ReorderParams P) {
  constexpr int PER = column_bytes(TWICE) / UNIT;  // units of a thread's column per row, RO_THREADS apart
  extern __shared__ __align__(16) unsigned char columns[];
  __shared__ int source_row[RO_MAX_BEAMS];
  __shared__ int moved_row[RO_MAX_BEAMS];
  __shared__ int moved_source[RO_MAX_BEAMS];
  __shared__ int sources, moved;
  const StateRows& S = P.states[blockIdx.z];
  const int tid = threadIdx.x, group = blockIdx.y;
  grid_dependency_wait();
  grid_launch_dependents();
  const int start = max(P.start ? P.start[group] : P.start_all, 0);
  const int end = min(P.end ? P.end[group] : P.end_all, S.places);
  if (end <= start) return;
  if (tid < 32) {
    // two beams per lane; parents and rows out of range leave the row as it is
    int parent[2], row[2], from[2];
    unsigned moves[2], needed[2] = {0u, 0u};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = h * 32 + tid;
      parent[h] = k;
      row[h] = -1;
      if (k < P.beams) {
        const int p = P.parents[group * P.beams + k];
        if (p >= 0 && p < P.beams) parent[h] = p;
        row[h] = P.slots ? P.slots[group * P.beams + k] : group * P.beams + k;
        if (row[h] >= S.rows) row[h] = -1;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int low = __shfl_sync(FULL, row[0], parent[h] & 31), high = __shfl_sync(FULL, row[1], parent[h] & 31);
      from[h] = parent[h] < 32 ? low : high;
      const bool moving = row[h] >= 0 && from[h] >= 0 && from[h] != row[h];
      moves[h] = __ballot_sync(FULL, moving);
      needed[0] |= __reduce_or_sync(FULL, moving && parent[h] < 32 ? 1u << parent[h] : 0u);
      needed[1] |= __reduce_or_sync(FULL, moving && parent[h] >= 32 ? 1u << (parent[h] - 32) : 0u);
    }
    const unsigned below = (1u << tid) - 1u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (needed[h] >> tid & 1u) source_row[(h ? __popc(needed[0]) : 0) + __popc(needed[h] & below)] = row[h];
      if (moves[h] >> tid & 1u) {
        const int at = (h ? __popc(moves[0]) : 0) + __popc(moves[h] & below);
        const int p = parent[h] & 31;
        moved_row[at] = row[h];
        moved_source[at] = (parent[h] >= 32 ? __popc(needed[0]) : 0) + __popc(needed[parent[h] >= 32 ? 1 : 0] & ((1u << p) - 1u));
      }
    }
    if (tid == 0) {
      sources = __popc(needed[0]) + __popc(needed[1]);
      moved = __popc(moves[0]) + __popc(moves[1]);
    }
  }
  __syncthreads();
  if (moved == 0) return;
  const long long units = (long long)(end - start) * S.place_bytes / UNIT;  // per run of places
  const long long per_run = (units + RO_THREADS * PER - 1) / (RO_THREADS * PER);
  const long long chunks = per_run * S.outer;
  unsigned char* const mine = columns + tid * UNIT;
#pragma unroll 1
  for (long long c = blockIdx.x; c < chunks; c += gridDim.x) {
    const long long outer = c / per_run, first = (c - outer * per_run) * (RO_THREADS * PER) + tid;
    char* const run = S.data + outer * S.outer_stride + (long long)start * S.place_bytes;
#pragma unroll 1
    for (int s = 0; s < sources; ++s) {
      const char* from = run + source_row[s] * S.row_stride;
#pragma unroll
      for (int r = 0; r < PER; ++r)
        if (first + r * RO_THREADS < units)
          column_load<UNIT>(mine + (s * PER + r) * (RO_THREADS * UNIT), from + (first + r * RO_THREADS) * UNIT);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
    for (int d = 0; d < moved; ++d) {
      char* to = run + moved_row[d] * S.row_stride;
      const int s = moved_source[d];
#pragma unroll
      for (int r = 0; r < PER; ++r)
        if (first + r * RO_THREADS < units)
          column_store<UNIT>(to + (first + r * RO_THREADS) * UNIT, mine + (s * PER + r) * (RO_THREADS * UNIT));
    }
  }
}

}  // namespace leat
