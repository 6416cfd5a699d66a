// Host side of beam search and log-probabilities: argument checks, workspace layout and the
// extern "C" entry points declared in include/leat_sampler.h.  There is no handle: a call's scratch is
// the caller's for that call, so calls on different streams or in different graphs share nothing.
#include "../../include/leat_sampler.h"

#include <cuda_runtime.h>
#include <math.h>
#include <string.h>

#include "beam_merge.cuh"
#include "host_util.cuh"
#include "reorder_kernel.cuh"
#include "sequences_kernel.cuh"

using namespace leat;

namespace {

constexpr int kMaxGroups = 65535;  // a grid's second dimension
constexpr long long kMaxBlocks = 0x7FFFFFFF;

struct Scratch {
  int tiles;
  size_t chunks_at, total;
};

// headers, then the maxima of the tiles' chunks where anything is to be selected
Scratch scratch_for(int rows, int vocab, int width, bool half) {
  Scratch s;
  const int tile = tile_logits(half);
  s.tiles = (int)(((long long)vocab + tile - 1) / tile);
  const size_t cells = (size_t)rows * s.tiles;
  s.chunks_at = (cells * sizeof(TileHead) + 255) / 256 * 256;
  s.total = s.chunks_at + (width > 0 ? cells * BT_CHUNKS * 4 : 0);
  return s;
}

bool known_format(uint32_t flags) {
  return (flags & ~(uint32_t)(LEAT_FLAG_LOGITS_BF16 | LEAT_FLAG_LOGITS_F16)) == 0 &&
         flags != (uint32_t)(LEAT_FLAG_LOGITS_BF16 | LEAT_FLAG_LOGITS_F16);
}

// Whole 16-byte vectors where the rows allow it; elsewhere float32 logits one per load, and 16-bit ones in
// whole vectors that are shifted.  It is the same for every row of a call, so that equal rows have equal sums.
template <template <int, bool> class Launch, typename Params>
cudaError_t by_format(const Params& P, uint32_t flags, int rows, int blocks, cudaStream_t stream) {
  const TileParams& T = P.T;
  const int per_vec = flags == 0 ? 4 : 8;
  const bool vec = T.vocab % per_vec == 0 && T.row_stride % per_vec == 0 && aligned(T.logits, 16);
  if (flags == 0) return vec ? Launch<0, true>::both(P, rows, blocks, stream) : Launch<0, false>::both(P, rows, blocks, stream);
  if (flags & LEAT_FLAG_LOGITS_BF16) return vec ? Launch<1, true>::both(P, rows, blocks, stream) : Launch<1, false>::both(P, rows, blocks, stream);
  return vec ? Launch<2, true>::both(P, rows, blocks, stream) : Launch<2, false>::both(P, rows, blocks, stream);
}

template <int FMT, bool VEC>
struct Tiles {
  static cudaError_t launch(const TileParams& T, int rows, cudaStream_t stream) {
    // a row's tiles next to each other (the other way round, rows first, reads float32 at 5.9 TB/s for 6.7)
    const int high = rows < kMaxGroups ? rows : 32768;
    return launch_dependent(beam_tile_kernel<FMT, VEC>, dim3((unsigned)T.tiles, (unsigned)high, (unsigned)((rows + high - 1) / high)),
                            dim3(BT_THREADS), 0, stream, T);
  }
};
template <int FMT, bool VEC>
struct Select {
  static cudaError_t both(const MergeParams& P, int rows, int groups, cudaStream_t stream) {
    const cudaError_t e = Tiles<FMT, VEC>::launch(P.T, rows, stream);
    if (e != cudaSuccess) return e;
    // Many continuations: more threads, for more nodes at a time.  Few: small blocks, whose barriers and bounds
    // cost less.  The border is the width up to which a level may bound itself by 32 parts, which wants few
    // warps to have many units each.  With 256 and 512 threads, us in a captured graph, inputs from memory:
    //   80 x 151936 bfloat16 in 16 groups: width 4 14.3 and 14.5, 10 15.6 and 14.8, 16 17.4 and 15.4, 64 41 and 27
    //   256 x 262144 float32 in 32 groups: 8 48.7 and 49.4, 10 50.3 and 52.2, 16 49.9 and 49.7, 64 79 and 65
    //   256 x 32000 bfloat16 in 64 groups: 8 12.4 and 12.5, 10 12.6 and 15.5, 12 13.0 and 12.6, 64 36 and 28
    //   one group of 4 x 128256: float32 8 8.9 and 10.0, 10 9.0 and 9.7; bfloat16 8 9.6 and 8.3, 10 9.9 and 8.4
    // (so neither is always better below it; beyond 16, 512 is)
    return P.width <= BM_FEW ? launch_dependent(beam_merge_kernel<256, FMT, VEC>, dim3(groups), dim3(256 + BM_EXACT), 0, stream, P)
                             : launch_dependent(beam_merge_kernel<512, FMT, VEC>, dim3(groups), dim3(512 + BM_EXACT), 0, stream, P);
  }
};
template <int FMT, bool VEC>
struct Logprobs {
  static cudaError_t both(const LogprobParams& P, int rows, int, cudaStream_t stream) {
    const cudaError_t e = Tiles<FMT, VEC>::launch(P.T, rows, stream);
    if (e != cudaSuccess) return e;
    if (P.top == 0)
      return launch_dependent(given_kernel<FMT>, dim3((rows + LP_THREADS / 32 - 1) / (LP_THREADS / 32)), dim3(LP_THREADS), 0, stream, P);
    // Rows that SMs hold at once wait for loads, and more threads have more of them on their way (512 x 32000
    // bfloat16, top 5: 13.9 us with 256 threads, 15.4 with 128); of more rows, smaller blocks overlap better
    // (1024 x 2000, top 5: 21.1 and 12.1).
    return rows > 4 * 148 ? launch_dependent(logprob_kernel<LP_THREADS, FMT, VEC>, dim3(rows), dim3(LP_THREADS + LP_EXACT), 0, stream, P)
                          : launch_dependent(logprob_kernel<2 * LP_THREADS, FMT, VEC>, dim3(rows), dim3(2 * LP_THREADS + LP_EXACT), 0, stream, P);
  }
};

bool logits_fit(const void* logits, int rows, int vocab, long long row_stride, uint32_t flags, const Scratch& s) {
  return logits && aligned(logits, flags ? 2 : 4) && (rows == 1 || row_stride >= vocab) &&
         (long long)rows * s.tiles <= kMaxBlocks / BT_CHUNKS;  // (chunks are counted in 32 bits)
}

int64_t lowest_bit(int64_t x) { return x & -x; }

// Lets a kernel be launched with more shared memory than the 48 KB, some of which it declares, that need no
// asking.  The limit is the function's, not the call's, so it is always set to the most that any call wants:
// set to a call's own size, it could be lowered by another thread's call before this one's launch.
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, size_t wanted, int most) {
  return wanted > 40 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) : cudaSuccess;
}

template <int UNIT>
cudaError_t launch_reorder(const ReorderParams& P, dim3 grid, bool twice, cudaStream_t stream) {
  const size_t shared = (size_t)P.beams * RO_THREADS * column_bytes(twice);
  auto kernel = twice ? reorder_kernel<UNIT, true> : reorder_kernel<UNIT, false>;
  const cudaError_t e = allow_shared(kernel, shared, (twice ? RO_TWICE_BEAMS : RO_MAX_BEAMS) * RO_THREADS * column_bytes(twice));
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, grid, dim3(RO_THREADS), shared, stream, P);
}

}  // namespace

extern "C" {

size_t leat_beam_workspace_bytes(int32_t rows, int32_t vocab, int32_t width) {
  if (rows <= 0 || vocab <= 0 || width < 0 || width > BM_MAX_WIDTH) return 0;
  // (the smaller tiles are those of float32: enough for every format)
  return scratch_for(rows, vocab, width, false).total;
}

int leat_beam_select(const leat_beam_args* a, leat_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a) return LEAT_E_ARGUMENT;
  if (a->groups < 0 || a->beams <= 0 || a->vocab <= 0 || a->width <= 0 || !known_format(a->flags)) return LEAT_E_ARGUMENT;
  if (a->beams > BM_MAX_BEAMS || a->width > BM_MAX_WIDTH) return LEAT_E_CAPACITY;
  if (a->groups == 0) return LEAT_OK;
  if ((long long)a->groups * a->beams > kMaxBlocks) return LEAT_E_CAPACITY;
  const int rows = a->groups * a->beams;
  if (!a->scores || !a->out_tokens || !a->out_parents || !a->out_scores) return LEAT_E_ARGUMENT;
  if (a->end_id >= a->vocab || (a->end_id < 0 && (a->finished || a->out_finished))) return LEAT_E_ARGUMENT;
  if (!(fabsf(a->length_penalty) <= 4.0f)) return LEAT_E_ARGUMENT;
  if (!a->lengths && (a->length_penalty != 0.0f || a->out_lengths)) return LEAT_E_ARGUMENT;
  const Scratch s = scratch_for(rows, a->vocab, a->width, a->flags != 0);
  if (!logits_fit(a->logits, rows, a->vocab, a->row_stride, a->flags, s)) return LEAT_E_ARGUMENT;
  if (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < s.total) return LEAT_E_WORKSPACE;
  MergeParams P;
  memset(&P, 0, sizeof(P));
  P.T.logits = a->logits; P.T.row_stride = a->row_stride; P.T.rows = rows; P.T.vocab = a->vocab;
  P.T.tiles = s.tiles; P.T.with_chunks = 1;
  P.T.scores = a->scores; P.T.finished = a->finished;
  P.T.heads = static_cast<TileHead*>(a->workspace);
  P.T.chunk_max = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + s.chunks_at);
  P.beams = a->beams; P.width = a->width; P.end_id = a->end_id < 0 ? -1 : a->end_id;
  P.length_penalty = a->length_penalty; P.lengths = a->lengths;
  P.out_tokens = a->out_tokens; P.out_parents = a->out_parents; P.out_scores = a->out_scores;
  P.out_finished = a->out_finished; P.out_lengths = a->out_lengths;
  return cuda_failed(by_format<Select>(P, a->flags, rows, a->groups, stream), "beam selection launch") ? LEAT_E_CUDA : LEAT_OK;
}

int leat_token_logprobs(const leat_logprob_args* a, leat_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a) return LEAT_E_ARGUMENT;
  if (a->rows < 0 || a->vocab <= 0 || a->given < 0 || a->top < 0 || !known_format(a->flags)) return LEAT_E_ARGUMENT;
  if (a->top > BM_MAX_WIDTH) return LEAT_E_CAPACITY;
  if (a->rows == 0) return LEAT_OK;
  if ((a->given > 0 && (!a->ids || !a->out_logprobs)) || (a->top > 0 && (!a->out_top_logprobs || !a->out_top_ids)))
    return LEAT_E_ARGUMENT;
  const Scratch s = scratch_for(a->rows, a->vocab, a->top, a->flags != 0);
  if (!logits_fit(a->logits, a->rows, a->vocab, a->row_stride, a->flags, s)) return LEAT_E_ARGUMENT;
  if (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < s.total) return LEAT_E_WORKSPACE;
  LogprobParams P;
  memset(&P, 0, sizeof(P));
  P.T.logits = a->logits; P.T.row_stride = a->row_stride; P.T.rows = a->rows; P.T.vocab = a->vocab;
  P.T.tiles = s.tiles; P.T.with_chunks = a->top > 0;
  P.T.heads = static_cast<TileHead*>(a->workspace);
  P.T.chunk_max = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + s.chunks_at);
  P.given = a->given; P.top = a->top; P.ids = a->ids;
  P.out_given = a->out_logprobs; P.out_top = a->out_top_logprobs; P.out_top_ids = a->out_top_ids;
  return cuda_failed(by_format<Logprobs>(P, a->flags, a->rows, 0, stream), "log-probabilities launch") ? LEAT_E_CUDA : LEAT_OK;
}

int leat_reorder_states(const leat_state* states, int32_t count, const int32_t* parents, const int32_t* slots,
                        int32_t groups, int32_t beams, const int32_t* start, int32_t start_all,
                        const int32_t* end, int32_t end_all, leat_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (count < 0 || groups < 0 || beams <= 0 || (count > 0 && !states)) return LEAT_E_ARGUMENT;
  if (beams > RO_MAX_BEAMS || groups > kMaxGroups) return LEAT_E_CAPACITY;
  if (count == 0 || groups == 0) return LEAT_OK;
  if (!parents) return LEAT_E_ARGUMENT;
  for (int i = 0; i < count; ++i) {
    const leat_state& s = states[i];
    if (!s.data || s.rows < 0 || s.outer < 0 || s.places < 0 || s.place_bytes <= 0 || s.row_stride < 0 || s.outer_stride < 0)
      return LEAT_E_ARGUMENT;
    if (!slots && s.rows < groups * beams) return LEAT_E_ARGUMENT;
    if (s.outer > 1 && s.outer_stride < (int64_t)s.places * s.place_bytes) return LEAT_E_ARGUMENT;
  }
  ReorderParams P;
  P.parents = parents; P.slots = slots; P.start = start; P.end = end;
  P.start_all = start_all; P.end_all = end_all; P.beams = beams;
  const bool twice = beams <= RO_TWICE_BEAMS;
  const int span = RO_THREADS * column_bytes(twice);  // bytes of a row that a block takes at a time
  // one launch per width of the widest loads that a tensor allows (16, 8, 4, 2, 1 bytes) and 64 of its kind
  for (int unit = 16; unit >= 1; unit /= 2) {
    int next = 0;
    while (next < count) {
      int n = 0;
      long long chunks = 0;  // of the tensor that has most to move
      for (; next < count && n < RO_MAX_STATES; ++next) {
        const leat_state& s = states[next];
        int64_t bits = (int64_t)(uintptr_t)s.data | s.place_bytes | 16;
        if (s.rows > 1) bits |= s.row_stride;
        if (s.outer > 1) bits |= s.outer_stride;
        if (lowest_bit(bits) != unit || s.rows == 0 || s.outer == 0 || s.places == 0) continue;
        P.states[n++] = StateRows{static_cast<char*>(s.data), s.row_stride, s.outer_stride, s.place_bytes, s.outer, s.places, s.rows, 0};
        int64_t places = s.places;
        if (!start && !end) places = (end_all < places ? end_all : places) - (start_all > 0 ? start_all : 0);
        if (places < 0) places = 0;
        const long long here = (places * s.place_bytes + span - 1) / span * s.outer;
        if (here > chunks) chunks = here;
      }
      if (n == 0 || chunks == 0) continue;
      // many short blocks: they balance groups whose rows move and groups whose rows stay
      long long x = (148 * 128 + (long long)groups * n - 1) / ((long long)groups * n);
      if (x > chunks) x = chunks;
      const dim3 grid((unsigned)x, (unsigned)groups, (unsigned)n);
      const cudaError_t e = unit == 16 ? launch_reorder<16>(P, grid, twice, stream) : unit == 8 ? launch_reorder<8>(P, grid, twice, stream)
                            : unit == 4 ? launch_reorder<4>(P, grid, twice, stream) : unit == 2 ? launch_reorder<2>(P, grid, twice, stream)
                            : launch_reorder<1>(P, grid, twice, stream);
      if (cuda_failed(e, "reorder_kernel launch")) return LEAT_E_CUDA;
    }
  }
  return LEAT_OK;
}

int leat_beam_sequences(const int32_t* tokens, const int32_t* parents, int32_t steps, int32_t groups, int32_t beams,
                        int32_t end_id, int32_t* out_tokens, int32_t* out_lengths, leat_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (steps < 0 || groups < 0 || beams <= 0) return LEAT_E_ARGUMENT;
  if (beams > SQ_MAX_BEAMS) return LEAT_E_CAPACITY;
  if (groups == 0) return LEAT_OK;
  if (!out_lengths || (steps > 0 && (!tokens || !parents || !out_tokens))) return LEAT_E_ARGUMENT;
  SequenceParams P;
  P.tokens = tokens; P.parents = parents; P.steps = steps; P.groups = groups; P.beams = beams;
  P.has_end = end_id >= 0; P.end_id = end_id; P.out = out_tokens; P.out_lengths = out_lengths;
  // a cluster per group: as many blocks as leave each at least 64 steps, while two fit on every SM
  int blocks = 1;
  while (blocks < SQ_MAX_BLOCKS && steps > 64 * blocks && (long long)groups * blocks <= 148) blocks *= 2;
  if ((long long)groups * blocks > kMaxBlocks) return LEAT_E_CAPACITY;
  int chunk = (steps + blocks - 1) / blocks;
  const int most = SQ_SHARED / (9 * beams);
  if (chunk > most) chunk = most;
  if (chunk < 1) chunk = 1;
  chunk = (chunk + 3) / 4 * 4;  // (tokens behind the parents stay 16-byte aligned)
  P.chunk = chunk;
  // runs of an odd number of steps: walked side by side, they lie in different banks
  P.run_len = (chunk + SQ_THREADS / beams - 1) / (SQ_THREADS / beams) | 1;
  P.runs = (chunk + P.run_len - 1) / P.run_len;
  P.vec = beams % 4 == 0 && aligned(tokens, 16) && aligned(parents, 16) ? 4 : 1;
  const unsigned per_step = (unsigned)(beams / P.vec);
  P.divide = (unsigned)((0x100000000ull + per_step - 1) / per_step);
  const size_t shared = (size_t)9 * chunk * beams;
  if (cuda_failed(allow_shared(sequences_kernel, shared, SQ_MOST_SHARED), "cudaFuncSetAttribute")) return LEAT_E_CUDA;
  return cuda_failed(launch_dependent_cluster(blocks, sequences_kernel, dim3((unsigned)(groups * blocks)), dim3(SQ_THREADS), shared, stream, P),
                     "sequences_kernel launch") ? LEAT_E_CUDA : LEAT_OK;
}

}  // extern "C"
