// Attention over the 4-bit cache (cache4.cuh): o_i = sum_j p_ij v_j, p_i = softmax_j(q_i . k_j / sqrt(head_dim)) over the rows j that row i
// sees, and on request the weight that every cached row received from the rows and heads of this call.
#include "cache4_attention.cuh"

namespace lcu {

// Up to 64 (row, query head) pairs per key/value head go to the kernel that walks the codes, 16 of them a time.  One sequence, 8 key heads x 4
// queries each: 8 rows behind 8000 / 30000 18 / 35 us against 43 / 81 on tcgen05, 16 rows 28 / 58 against 44 / 84; 32 heads with a key each:
// 64 rows behind 500 / 8000 / 30000 12 / 63 / 180 against 21 / 81 / 230, 96 rows 22 / 93 / 268 against 23 / 80 / 230.  A single row always does,
// however many heads share a key.
static bool few_rows(int m, int group) { return (long long)m * group <= 64 || m == 1; }

static bool sizes_fit(int n_seqs, int m, int n_heads, int n_kv, int hd) {
  return (long long)n_seqs * n_kv < 65536 && (long long)n_heads * hd < (1 << 24) && (long long)n_seqs * m * n_heads < (1ll << 31);
}
// sizes that a call is not refused for (positive ones, of whole heads)
static bool sizes_taken(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len) {
  return (hd == 64 || hd == 128) && n_heads % n_kv == 0 && m < (1 << 26) && max_len < (1 << 26) && sizes_fit(n_seqs, m, n_heads, n_kv, hd) &&
         (few_rows(m, n_heads / n_kv) ? attention_cache4_step_takes : attention_cache4_prompt_takes)(n_seqs, m, n_heads, n_kv, max_len);
}

size_t cache4_attention_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights) {
  if (!sizes_taken(n_seqs, m, n_heads, n_kv, hd, max_len)) return 0;
  if (few_rows(m, n_heads / n_kv)) return attention_cache4_step_workspace(n_seqs, m, n_heads, n_kv, hd, max_len, weights);
  return attention_cache4_prompt_workspace(n_seqs, m, n_heads, n_kv, hd, max_len, weights);
}

int launch_attention_cache4(const cache4_attention_params& p, int dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  int rc = check_cache4("attention_cache4", p.c);
  if (rc) return rc;
  LCU_REQUIRE(dtype == OP_F16 || dtype == OP_BF16, "attention_cache4: number format %d is not 0 (half) or 1 (bfloat16)", dtype);
  LCU_REQUIRE(p.out && p.q && p.lengths, "attention_cache4: a null pointer");
  LCU_REQUIRE(p.m >= 1 && p.n_heads >= 1 && p.n_heads % p.c.n_kv == 0, "attention_cache4: %d rows, %d heads over %d key/value heads", p.m, p.n_heads, p.c.n_kv);
  LCU_REQUIRE(p.m < (1 << 26) && p.c.ctx < (1 << 26), "attention_cache4: %d rows, %d in the cache", p.m, p.c.ctx);
  LCU_REQUIRE(p.max_len >= 1 && p.max_len <= p.c.ctx, "attention_cache4: %d rows exceed the cache's %d", p.max_len, p.c.ctx);
  LCU_REQUIRE(sizes_fit(p.c.n_seqs, p.m, p.n_heads, p.c.n_kv, p.c.hd), "attention_cache4: %d sequences of %d rows of %d heads are too many", p.c.n_seqs, p.m, p.n_heads);
  LCU_REQUIRE(sizes_taken(p.c.n_seqs, p.m, p.n_heads, p.c.n_kv, p.c.hd, p.max_len), "attention_cache4: %d sequences of %d rows of %d heads over %d rows are too many", p.c.n_seqs,
              p.m, p.n_heads, p.max_len);
  LCU_REQUIRE(p.ld_q % 8 == 0 && p.ld_out % 8 == 0 && p.ld_q >= p.n_heads * p.c.hd && p.ld_out >= p.n_heads * p.c.hd,
              "attention_cache4: row strides must be multiples of 8 that hold a row");
  LCU_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.out) & 15) == 0, "attention_cache4: rows must be 16-byte aligned");
  LCU_REQUIRE(words_aligned(p.lengths, p.weights), "attention_cache4: lengths and weights must be 4-byte aligned");
  const size_t need = cache4_attention_workspace(p.c.n_seqs, p.m, p.n_heads, p.c.n_kv, p.c.hd, p.max_len, p.weights != nullptr);
  LCU_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
              "attention_cache4: %zu bytes of 16-byte aligned workspace are needed, %zu are there", need, workspace ? workspace_bytes : (size_t)0);
  if (int rc_dev = need_device()) return rc_dev;
  if (few_rows(p.m, p.n_heads / p.c.n_kv)) return launch_attention_cache4_step(p, dtype, workspace, stream);
  return launch_attention_cache4_prompt(p, dtype, workspace, stream);
}

}  // namespace lcu
