// Attention over the 4-bit cache (cache4.cuh): o_i = sum_j p_ij v_j, p_i = softmax_j(q_i . k_j / sqrt(head_dim)) over the rows j that row i
// sees, and on request the weight that every cached row received from the rows and heads of this call.
#include "cache4_attention.cuh"

namespace lcu {
namespace {

struct rows_args {
  cache4_attention_params p;
  float2* stats;  // [n_seqs * m][n_heads] maximum of the scores and sum of the exponentials (nullptr: not wanted)
};

__device__ __forceinline__ int rows_seen(const cache4_attention_params& p, int seq, int i) {
  const int held = p.lengths[seq];
  if (held < 0) return 0;
  return (int)min((long long)held + i + 1, (long long)min(p.c.ctx, p.max_len));
}

// One warp per (row, head): head_dim / 8 lanes share a key, running maximum and sum per group of lanes.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attention_rows_kernel(const rows_args a) {
  const cache4_attention_params& p = a.p;
  constexpr int W = HD / 8, SUB = 32 / W;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (unit >= (long long)p.c.n_seqs * p.m * p.n_heads) return;
  const int row = (int)(unit / p.n_heads), head = (int)(unit % p.n_heads);
  const int seq = row / p.m, i = row - seq * p.m, kvh = head / (p.n_heads / p.c.n_kv);
  const int T_seen = rows_seen(p, seq, i);
  const int o8 = lane % W, sub = lane / W;
  float q[8], acc[8] = {};
  unpack8<T>(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (size_t)row * p.ld_q + head * HD)[o8], q);
  const float rs = rsqrtf((float)HD);
  float mx = -INFINITY, sum = 0.f;
  const size_t base = ((size_t)seq * p.c.n_kv + kvh) * p.c.ctx;
  const int nb = HD / p.c.bs, blk = o8 * 8 / p.c.bs, word = cache4_word(o8, HD / 32);
  for (int j0 = 0; j0 < T_seen; j0 += SUB) {
    const int j = j0 + sub;
    const bool there = j < T_seen;
    const size_t at = base + (there ? j : 0);
    const uint32_t kw = reinterpret_cast<const uint32_t*>(p.c.k_codes + at * (HD / 2))[word];
    const float ks = __half2float(p.c.k_scales[at * nb + blk]);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(cache4_value(kw, e, ks), q[e], s);
#pragma unroll
    for (int w = 1; w < W; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (!there) continue;
    s *= rs;
    const float next = fmaxf(mx, s), keep = expf(mx - next), e1 = s == -INFINITY ? 0.f : expf(s - next);
    const float old = next == -INFINITY ? 1.f : keep;
    const uint32_t vw = reinterpret_cast<const uint32_t*>(p.c.v_codes + at * (HD / 2))[word];
    const float vs = __half2float(p.c.v_scales[at * nb + blk]);
    sum = sum * old + e1;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * old + e1 * cache4_value(vw, e, vs);
    mx = next;
  }
#pragma unroll
  for (int w = W; w < 32; w <<= 1) {  // the groups of lanes join
    const float om = __shfl_xor_sync(0xffffffffu, mx, w), os = __shfl_xor_sync(0xffffffffu, sum, w);
    const float next = fmaxf(mx, om), f = next == -INFINITY ? 1.f : expf(mx - next), of = next == -INFINITY ? 1.f : expf(om - next);
    sum = sum * f + os * of;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f + __shfl_xor_sync(0xffffffffu, acc[e], w) * of;
    mx = next;
  }
  if (sub == 0) {
    const float r = T_seen ? 1.f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= r;
    reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (size_t)row * p.ld_out + head * HD)[o8] = pack8<T>(acc);
    if (a.stats && lane == 0) a.stats[(size_t)row * p.n_heads + head] = make_float2(mx, sum);
  }
}

// One warp per (sequence, key/value head, cached row): its weight from all rows and heads of the call, in their order.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attention_weights_kernel(const rows_args a) {
  const cache4_attention_params& p = a.p;
  constexpr int W = HD / 8, SUB = 32 / W;
  const int lane = threadIdx.x & 31, sh = blockIdx.y, seq = sh / p.c.n_kv, kvh = sh % p.c.n_kv;
  const int j = blockIdx.x * 4 + (threadIdx.x >> 5), group = p.n_heads / p.c.n_kv;
  if (j >= rows_seen(p, seq, p.m - 1)) return;
  const int o8 = lane % W, sub = lane / W;
  const size_t at = (size_t)sh * p.c.ctx + j;
  const uint32_t kw = reinterpret_cast<const uint32_t*>(p.c.k_codes + at * (HD / 2))[cache4_word(o8, HD / 32)];
  const float ks = __half2float(p.c.k_scales[at * (HD / p.c.bs) + o8 * 8 / p.c.bs]), rs = rsqrtf((float)HD);
  float total = 0.f;
  for (int u0 = 0; u0 < p.m * group; u0 += SUB) {
    const int u = u0 + sub, i = u / group;
    const bool there = u < p.m * group && j < rows_seen(p, seq, i);
    const size_t row = (size_t)seq * p.m + (there ? i : p.m - 1);
    const int head = kvh * group + (there ? u % group : 0);
    float q[8], s = 0.f;
    unpack8<T>(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + row * p.ld_q + head * HD)[o8], q);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(cache4_value(kw, e, ks), q[e], s);
#pragma unroll
    for (int w = 1; w < W; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    const float2 st = a.stats[row * p.n_heads + head];
    if (there) total += expf(s * rs - st.x) / st.y;
  }
#pragma unroll
  for (int w = W; w < 32; w <<= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
  if (lane == 0) p.weights[at] = p.beta == 0.f || j >= p.lengths[seq] ? total : fmaf(p.beta, p.weights[at], total);
}

template <typename T, int HD>
int launch_rows(const rows_args& a, cudaStream_t stream) {
  const cache4_attention_params& p = a.p;
  const long long units = (long long)p.c.n_seqs * p.m * p.n_heads;
  attention_rows_kernel<T, HD><<<(unsigned)((units + 3) / 4), 128, 0, stream>>>(a);
  if (p.weights) attention_weights_kernel<T, HD><<<dim3((unsigned)((p.max_len + 3) / 4), p.c.n_seqs * p.c.n_kv), 128, 0, stream>>>(a);
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

}  // namespace

// rows that go to the kernel of few rows
static bool few_rows(int m, int group) { return (long long)m * group <= 16 || m == 1; }

size_t cache4_attention_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights) {
  if (few_rows(m, n_heads / n_kv)) return attention_cache4_step_workspace(n_seqs, m, n_heads, n_kv, hd, max_len, weights);
  return weights ? (size_t)n_seqs * m * n_heads * sizeof(float2) : 0;
}

int launch_attention_cache4(const cache4_attention_params& p, int dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  int rc = check_cache4("attention_cache4", p.c);
  if (rc) return rc;
  LCU_REQUIRE(dtype == OP_F16 || dtype == OP_BF16, "attention_cache4: number format %d is not 0 (half) or 1 (bfloat16)", dtype);
  LCU_REQUIRE(p.out && p.q && p.lengths, "attention_cache4: a null pointer");
  LCU_REQUIRE(p.m >= 1 && p.n_heads >= 1 && p.n_heads % p.c.n_kv == 0, "attention_cache4: %d rows, %d heads over %d key/value heads", p.m, p.n_heads, p.c.n_kv);
  LCU_REQUIRE(p.m < (1 << 26) && p.c.ctx < (1 << 26), "attention_cache4: %d rows, %d in the cache", p.m, p.c.ctx);
  LCU_REQUIRE(p.max_len >= 1 && p.max_len <= p.c.ctx, "attention_cache4: %d rows exceed the cache's %d", p.max_len, p.c.ctx);
  LCU_REQUIRE((long long)p.n_heads * p.c.hd < (1 << 24) && (long long)p.c.n_seqs * p.m * p.n_heads < (1ll << 31) && (long long)p.c.n_seqs * p.c.n_kv < 65536,
              "attention_cache4: %d sequences of %d rows of %d heads are too many", p.c.n_seqs, p.m, p.n_heads);
  LCU_REQUIRE(p.ld_q % 8 == 0 && p.ld_out % 8 == 0 && p.ld_q >= p.n_heads * p.c.hd && p.ld_out >= p.n_heads * p.c.hd,
              "attention_cache4: row strides must be multiples of 8 that hold a row");
  LCU_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.out) & 15) == 0, "attention_cache4: rows must be 16-byte aligned");
  const size_t need = cache4_attention_workspace(p.c.n_seqs, p.m, p.n_heads, p.c.n_kv, p.c.hd, p.max_len, p.weights != nullptr);
  LCU_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
              "attention_cache4: %zu bytes of 16-byte aligned workspace are needed, %zu are there", need, workspace ? workspace_bytes : (size_t)0);
  if (int rc_dev = need_device()) return rc_dev;
  if (few_rows(p.m, p.n_heads / p.c.n_kv)) return launch_attention_cache4_step(p, dtype, workspace, stream);
  rows_args a{p, p.weights ? (float2*)workspace : nullptr};
  if (dtype == OP_F16) return p.c.hd == 128 ? launch_rows<__half, 128>(a, stream) : launch_rows<__half, 64>(a, stream);
  return p.c.hd == 128 ? launch_rows<__nv_bfloat16, 128>(a, stream) : launch_rows<__nv_bfloat16, 64>(a, stream);
}

}  // namespace lcu
