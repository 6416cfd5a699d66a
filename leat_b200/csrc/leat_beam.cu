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
  int tiles, places;
  size_t lists_at, total;
};

// headers, then (with candidates) the tiles' lists
Scratch scratch_for(int rows, int vocab, int top, bool half) {
  Scratch s;
  const int tile = tile_logits(half);
  s.tiles = (int)(((long long)vocab + tile - 1) / tile);
  s.places = top > 0 ? top + BT_SLACK : 0;
  const size_t cells = (size_t)rows * s.tiles;
  s.lists_at = (cells * sizeof(TileHead) + 255) / 256 * 256;
  s.total = s.lists_at + cells * s.places * 8;
  return s;
}

bool known_format(uint32_t flags) {
  return (flags & ~(uint32_t)(LEAT_FLAG_LOGITS_BF16 | LEAT_FLAG_LOGITS_F16)) == 0 &&
         flags != (uint32_t)(LEAT_FLAG_LOGITS_BF16 | LEAT_FLAG_LOGITS_F16);
}
int format_of(uint32_t flags) { return flags & LEAT_FLAG_LOGITS_BF16 ? 1 : (flags & LEAT_FLAG_LOGITS_F16 ? 2 : 0); }

template <int FMT, bool VEC>
cudaError_t launch_tiles(const TileParams& T, int rows, cudaStream_t stream) {
  const dim3 grid((unsigned)((long long)rows * T.tiles));
  return T.top > 0 ? launch_dependent(beam_tile_kernel<FMT, VEC, true>, grid, dim3(BT_THREADS), 0, stream, T)
                   : launch_dependent(beam_tile_kernel<FMT, VEC, false>, grid, dim3(BT_THREADS), 0, stream, T);
}

// whole 16-byte vectors where the rows allow it, one logit per load elsewhere: the same for every row
// of a call, so that equal rows have equal sums
int stream_tiles(const TileParams& T, int fmt, int rows, cudaStream_t stream) {
  const int per_vec = fmt == 0 ? 4 : 8;
  const bool vec = T.vocab % per_vec == 0 && T.row_stride % per_vec == 0 && aligned(T.logits, 16);
  cudaError_t e;
  if (fmt == 0) e = vec ? launch_tiles<0, true>(T, rows, stream) : launch_tiles<0, false>(T, rows, stream);
  else if (fmt == 1) e = vec ? launch_tiles<1, true>(T, rows, stream) : launch_tiles<1, false>(T, rows, stream);
  else e = vec ? launch_tiles<2, true>(T, rows, stream) : launch_tiles<2, false>(T, rows, stream);
  return cuda_failed(e, "beam_tile_kernel launch") ? LEAT_E_CUDA : LEAT_OK;
}

bool logits_fit(const void* logits, int rows, int vocab, long long row_stride, uint32_t flags, const Scratch& s) {
  return logits && aligned(logits, flags ? 2 : 4) && (rows == 1 || row_stride >= vocab) &&
         (long long)rows * s.tiles <= kMaxBlocks;
}

int64_t lowest_bit(int64_t x) { return x & -x; }

}  // namespace

extern "C" {

size_t leat_beam_workspace_bytes(int32_t rows, int32_t vocab, int32_t width) {
  if (rows <= 0 || vocab <= 0 || width < 0 || width > BT_MAX_TOP) return 0;
  // (the smaller tiles are those of float32: enough for every format)
  return scratch_for(rows, vocab, width, false).total;
}

int leat_beam_select(const leat_beam_args* a, leat_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a) return LEAT_E_ARGUMENT;
  if (a->groups < 0 || a->beams <= 0 || a->vocab <= 0 || a->width <= 0 || !known_format(a->flags)) return LEAT_E_ARGUMENT;
  if (a->beams > BM_MAX_BEAMS || a->width > BT_MAX_TOP) return LEAT_E_CAPACITY;
  if (a->groups == 0) return LEAT_OK;
  if ((long long)a->groups * a->beams > kMaxBlocks) return LEAT_E_CAPACITY;
  const int rows = a->groups * a->beams;
  if (!a->scores || !a->out_tokens || !a->out_parents || !a->out_scores) return LEAT_E_ARGUMENT;
  if (a->end_id >= a->vocab || (a->end_id < 0 && (a->finished || a->out_finished))) return LEAT_E_ARGUMENT;
  if (!(fabsf(a->length_penalty) <= 16.0f)) return LEAT_E_ARGUMENT;
  if (!a->lengths && (a->length_penalty != 0.0f || a->out_lengths)) return LEAT_E_ARGUMENT;
  const Scratch s = scratch_for(rows, a->vocab, a->width, a->flags != 0);
  if (!logits_fit(a->logits, rows, a->vocab, a->row_stride, a->flags, s)) return LEAT_E_ARGUMENT;
  if (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < s.total) return LEAT_E_WORKSPACE;
  MergeParams P;
  memset(&P, 0, sizeof(P));
  P.T.logits = a->logits; P.T.row_stride = a->row_stride; P.T.vocab = a->vocab;
  P.T.tiles = s.tiles; P.T.top = a->width; P.T.places = s.places;
  P.T.scores = a->scores; P.T.finished = a->finished;
  P.T.heads = static_cast<TileHead*>(a->workspace);
  P.T.lists = reinterpret_cast<unsigned long long*>(static_cast<char*>(a->workspace) + s.lists_at);
  P.beams = a->beams; P.width = a->width; P.end_id = a->end_id < 0 ? -1 : a->end_id;
  P.length_penalty = a->length_penalty; P.lengths = a->lengths;
  P.out_tokens = a->out_tokens; P.out_parents = a->out_parents; P.out_scores = a->out_scores;
  P.out_finished = a->out_finished; P.out_lengths = a->out_lengths;
  const int code = stream_tiles(P.T, format_of(a->flags), rows, stream);
  if (code != LEAT_OK) return code;
  return cuda_failed(launch_dependent(beam_merge_kernel<512>, dim3(a->groups), dim3(512), 0, stream, P),
                     "beam_merge_kernel launch") ? LEAT_E_CUDA : LEAT_OK;
}

int leat_token_logprobs(const leat_logprob_args* a, leat_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a) return LEAT_E_ARGUMENT;
  if (a->rows < 0 || a->vocab <= 0 || a->given < 0 || a->top < 0 || !known_format(a->flags)) return LEAT_E_ARGUMENT;
  if (a->top > BT_MAX_TOP) return LEAT_E_CAPACITY;
  if (a->rows == 0) return LEAT_OK;
  if ((a->given > 0 && (!a->ids || !a->out_logprobs)) || (a->top > 0 && (!a->out_top_logprobs || !a->out_top_ids)))
    return LEAT_E_ARGUMENT;
  const Scratch s = scratch_for(a->rows, a->vocab, a->top, a->flags != 0);
  if (!logits_fit(a->logits, a->rows, a->vocab, a->row_stride, a->flags, s)) return LEAT_E_ARGUMENT;
  if (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < s.total) return LEAT_E_WORKSPACE;
  LogprobParams P;
  memset(&P, 0, sizeof(P));
  P.T.logits = a->logits; P.T.row_stride = a->row_stride; P.T.vocab = a->vocab;
  P.T.tiles = s.tiles; P.T.top = a->top; P.T.places = s.places;
  P.T.heads = static_cast<TileHead*>(a->workspace);
  P.T.lists = reinterpret_cast<unsigned long long*>(static_cast<char*>(a->workspace) + s.lists_at);
  P.fmt = format_of(a->flags); P.given = a->given; P.top = a->top; P.ids = a->ids;
  P.out_given = a->out_logprobs; P.out_top = a->out_top_logprobs; P.out_top_ids = a->out_top_ids;
  const int code = stream_tiles(P.T, P.fmt, a->rows, stream);
  if (code != LEAT_OK) return code;
  return cuda_failed(launch_dependent(logprob_kernel, dim3(a->rows), dim3(LP_THREADS), 0, stream, P),
                     "logprob_kernel launch") ? LEAT_E_CUDA : LEAT_OK;
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
  memset(&P, 0, sizeof(P));
  P.parents = parents; P.slots = slots; P.start = start; P.end = end;
  P.start_all = start_all; P.end_all = end_all; P.beams = beams;
  const size_t shared = (size_t)beams * RO_THREADS * 16;
  // one launch per width of the widest loads that a tensor allows (16, 8, 4, 2, 1 bytes) and 64 of its kind
  for (int unit = 16; unit >= 1; unit /= 2) {
    int next = 0;
    while (next < count) {
      int n = 0;
      long long chunks = 0;
      for (; next < count && n < RO_MAX_STATES; ++next) {
        const leat_state& s = states[next];
        int64_t bits = (int64_t)(uintptr_t)s.data | s.place_bytes | 16;
        if (s.rows > 1) bits |= s.row_stride;
        if (s.outer > 1) bits |= s.outer_stride;
        if (lowest_bit(bits) != unit || s.rows == 0 || s.outer == 0 || s.places == 0) continue;
        StateRows& to = P.states[n++];
        to.data = static_cast<char*>(s.data);
        to.row_stride = s.row_stride; to.outer_stride = s.outer_stride; to.place_bytes = s.place_bytes;
        to.outer = s.outer; to.places = s.places; to.rows = s.rows; to.pad = 0;
        int64_t places = s.places;
        if (!start && !end) places = (end_all < places ? end_all : places) - (start_all > 0 ? start_all : 0);
        if (places < 0) places = 0;
        const long long here = (places * s.place_bytes + RO_THREADS * 16 - 1) / (RO_THREADS * 16) * s.outer;
        if (here > chunks) chunks = here;
      }
      if (n == 0 || chunks == 0) continue;
      // about 32 blocks per SM of 148 in all: many short blocks balance rows that move and rows that stay
      long long x = (148 * 32 + (long long)groups * n - 1) / ((long long)groups * n);
      if (x > chunks) x = chunks;
      const dim3 grid((unsigned)x, (unsigned)groups, (unsigned)n);
      auto kernel = unit == 16 ? reorder_kernel<16> : unit == 8 ? reorder_kernel<8> : unit == 4 ? reorder_kernel<4>
                    : unit == 2 ? reorder_kernel<2> : reorder_kernel<1>;
      if (shared > 48 * 1024 &&
          cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared), "cudaFuncSetAttribute"))
        return LEAT_E_CUDA;
      if (cuda_failed(launch_dependent(kernel, grid, dim3(RO_THREADS), shared, stream, P), "reorder_kernel launch"))
        return LEAT_E_CUDA;
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
  // a cluster per group: as many blocks as leave each at least 64 steps, while the GPU has room
  int blocks = 1;
  while (blocks < 8 && steps > 64 * blocks && (long long)groups * blocks < 2 * 148) blocks *= 2;
  if ((long long)groups * blocks > kMaxBlocks) return LEAT_E_CAPACITY;
  int chunk = (steps + blocks - 1) / blocks;
  const int most = SQ_SHARED / (2 * beams);
  if (chunk > most) chunk = most;
  if (chunk < 1) chunk = 1;
  // runs: their number costs as much to compose as half their length costs to walk (twice)
  int runs = 1;
  while (runs * 2 * beams <= SQ_THREADS && runs * runs < 2 * chunk) runs *= 2;
  P.chunk = chunk; P.runs = runs;
  const size_t shared = (size_t)2 * chunk * beams;
  if (shared > 40 * 1024 &&
      cuda_failed(cudaFuncSetAttribute(sequences_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared), "cudaFuncSetAttribute"))
    return LEAT_E_CUDA;
  return cuda_failed(launch_dependent_cluster(blocks, sequences_kernel, dim3((unsigned)(groups * blocks)), dim3(SQ_THREADS), shared, stream, P),
                     "sequences_kernel launch") ? LEAT_E_CUDA : LEAT_OK;
}

}  // extern "C"
