// The kernels behind launch_attention_cache4.
#pragma once
#include "cache4.cuh"

namespace lcu {

#ifdef __CUDACC__
// Exponentials are formed against a reference 7 below the running maximum (powers of two), which is raised when a score passes the maximum
// by 8: as halves, the operands of the product with the values, they lie up to 2^15, and what lies 2^-32 below the largest is still there (2^-25
// with the maximum itself as the reference: the 32000 rows behind one that is 17.5 nats ahead, together 1e-3 of the output, were lost).
// From 2^20 on the maximum is the reference: the bound of 8, as the products give scores, and the reference are then off by a sixteenth each and
// more, by 4 / 2 three times where scores reach 2^26, which a half's range has to hold as well: 2^(8 + 6).
constexpr float LIFT = 7.f, LIFT_FACTOR = 128.f;
__device__ __forceinline__ float reference_of(float top) { return fabsf(top) < 1048576.f ? top - LIFT : top; }
#endif

// few rows (attention_cache4_step.cu); takes: whether the kernels' numbers hold the work (of sizes that fit otherwise)
bool attention_cache4_step_takes(int n_seqs, int m, int n_heads, int n_kv, int max_len);
size_t attention_cache4_step_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights);
int launch_attention_cache4_step(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream);

// prompts (attention_cache4_prompt.cu)
bool attention_cache4_prompt_takes(int n_seqs, int m, int n_heads, int n_kv, int max_len);
size_t attention_cache4_prompt_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights);
int launch_attention_cache4_prompt(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream);

}  // namespace lcu
