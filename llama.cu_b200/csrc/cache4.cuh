// The 4-bit cache: rows of codes and scales, and the operators over it (append, read, attention).
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace lcu {

// Planes of one layer, [sequence][key/value head][row]: a row is head_dim / 2 bytes of codes and head_dim / bs half scales.
// A block's scale is absmax / 7.5 rounded to 7 significant bits (at most 8704); the value of dimension d is (code - 7.5) * scale, and
// as 2 code - 15 has four bits that product is exact in a half (above the subnormals), so that tensor-core operands can hold the cache's
// own values.  The eight codes of dimensions 32 g + 8 o .. + 7 are the nibbles, lowest first, of word o * (head_dim / 32) + g: the lane
// of a warp-level product that owns octet o of every 32 dimensions reads its words side by side.
struct cache4_view {
  uint8_t* k_codes;
  __half* k_scales;
  uint8_t* v_codes;
  __half* v_scales;
  int n_seqs, n_kv, hd, bs, ctx;
};

enum op_dtype : int { OP_F16 = 0, OP_BF16 = 1, OP_F32 = 2 };

int check_cache4(const char* who, const cache4_view& c);
// numbers of four bytes at addresses that are multiples of four (null pointers pass)
template <typename... P>
bool words_aligned(const P*... p) {
  return (((uintptr_t)p | ... | (uintptr_t)0) & 3) == 0;
}

struct cache4_append_params {
  cache4_view c;
  void* q_out;            // [n_seqs * m][n_heads * hd], may be q
  const void* q;          // [n_seqs * m][ld_q] (nullptr: no queries)
  int ld_q;
  const void* k_new;      // [n_seqs * m][ld_kv]
  const void* v_new;
  int ld_kv;
  const int* lengths;     // [n_seqs] rows held before: row i of a sequence goes to lengths + i; negative: nothing is written
  const int* positions;   // [n_seqs] rotary position of a sequence's first new row (nullptr: lengths)
  int m, n_heads;
  float theta;            // 0: no rotation
};
int launch_cache4_append(const cache4_append_params& p, int dtype, cudaStream_t stream);

// rows [first, first + count) of every sequence and head as values: k_out / v_out [n_seqs][n_kv][count][hd] (either may be nullptr)
int launch_cache4_read(void* k_out, void* v_out, const cache4_view& c, const int* first, int count, int dtype, cudaStream_t stream);

struct cache4_attention_params {
  cache4_view c;
  void* out;              // [n_seqs * m][ld_out]
  int ld_out;
  float* weights;         // [n_seqs][n_kv][ctx] or nullptr
  float beta;
  const void* q;          // [n_seqs * m][ld_q]
  int ld_q;
  const int* lengths;
  int m, n_heads;
  int max_len;            // no sequence sees more rows than this
};
size_t cache4_attention_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights);
int launch_attention_cache4(const cache4_attention_params& p, int dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream);

#ifdef __CUDACC__
// 16-bit operands by type: eight neighbouring values <-> binary32
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]);
template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& v, float (&x)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& v, float (&x)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}
// the word of a row that holds octet `o8` (dimensions 8 o8 .. + 7)
__device__ __forceinline__ int cache4_word(int o8, int groups) { return (o8 & 3) * groups + (o8 >> 2); }
__device__ __forceinline__ float cache4_value(uint32_t word, int i, float scale) { return ((float)((word >> (4 * i)) & 15u) - 7.5f) * scale; }
#endif

}  // namespace lcu
