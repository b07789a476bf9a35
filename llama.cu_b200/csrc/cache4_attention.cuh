// The kernels behind launch_attention_cache4.
#pragma once
#include "cache4.cuh"

namespace lcu {

// few rows (attention_cache4_step.cu)
size_t attention_cache4_step_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights);
int launch_attention_cache4_step(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream);

// prompts (attention_cache4_prompt.cu)
size_t attention_cache4_prompt_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights);
int launch_attention_cache4_prompt(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream);

}  // namespace lcu
