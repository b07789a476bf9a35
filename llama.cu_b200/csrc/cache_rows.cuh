// Rows of caches that move: eviction by weight and reordering among beams.
#pragma once
#include "common.cuh"

namespace lcu {

constexpr int MAX_CACHE_PLANES = 8;
constexpr int MAX_BEAMS = 32;

struct evict_params {
  void* const* dst;         // host arrays of n_planes device pointers: [n_seqs][n_kv][dst_ctx] / [n_seqs][n_kv][ctx] rows of row_bytes[i]
  const void* const* src;
  const int* row_bytes;
  int n_planes;
  const float* weights;     // [n_seqs][n_kv][ctx]
  int* kept;                // [n_seqs][n_kv][keep]
  int* lengths_out;         // [n_seqs], may be lengths
  const int* lengths;
  int n_seqs, n_kv, ctx, dst_ctx, keep, recent;
};
int launch_cache_evict(const evict_params& p, cudaStream_t stream);

struct reorder_params {
  void* const* dst;
  const void* const* src;
  const int* row_bytes;
  int n_planes;
  const int* parents;       // [n_groups][beams]
  const int* lengths;       // [n_groups * beams]
  int n_groups, beams, n_kv, ctx;
};
int launch_cache_reorder(const reorder_params& p, cudaStream_t stream);

struct beam_params {
  int* parents;             // [n_groups][n_out]
  int* tokens;
  float* scores_out;
  const void* logits;       // [n_groups * beams][ld]
  int ld;
  const float* scores;      // [n_groups][beams]
  int n_groups, beams, n_vocab, n_out;
};
size_t beam_select_workspace(int n_groups, int beams, int n_vocab, int n_out);
int launch_beam_select(const beam_params& p, int dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace lcu
