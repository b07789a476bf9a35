// New rows into the 4-bit cache: rotary positions, rounding to 4 bits, and the way back to values.
#include "cache4.cuh"

#include <algorithm>
#include <cmath>

namespace lcu {

int check_cache4(const char* who, const cache4_view& c) {
  LCU_REQUIRE(c.k_codes && c.k_scales && c.v_codes && c.v_scales, "%s: a plane of the cache is a null pointer", who);
  LCU_REQUIRE(c.hd == 64 || c.hd == 128, "%s: head_dim %d not supported (64 or 128)", who, c.hd);
  LCU_REQUIRE((c.bs == 32 || c.bs == 64 || c.bs == 128) && c.bs <= c.hd, "%s: block size %d must be 32, 64 or 128 and at most head_dim", who, c.bs);
  LCU_REQUIRE(c.n_seqs >= 1 && c.n_kv >= 1 && c.ctx >= 1, "%s: no sequences, heads or rows", who);
  LCU_REQUIRE(((((uintptr_t)c.k_codes | (uintptr_t)c.v_codes | (uintptr_t)c.k_scales | (uintptr_t)c.v_scales) & 15) == 0),
              "%s: the planes of the cache must be 16-byte aligned", who);
  return LCU_OK;
}

namespace {

struct append_args {
  cache4_append_params p;
  double log2_theta;
};

// binary32 s >= 0 to 7 significant bits, ties to even (a NaN or an infinity gives a NaN)
__device__ __forceinline__ float seven_bits(float s) {
  uint32_t b = __float_as_uint(s);
  if (b >= 0x7f800000u) return __int_as_float(0x7fffffff);
  b = (b + 0xffffu + ((b >> 17) & 1u)) & ~0x1ffffu;
  return __uint_as_float(b);
}

// One CTA per new row.  Bound by memory for prompts and by the launch for a single token; the angles are formed once per row, in 64
// bits (a position of a hundred thousand leaves seven digits of a binary32 angle's turn), and shared by all heads.  A thread owns eight
// neighbouring dimensions: one 16-byte load, its four rotation pairs, one word of codes; a block's threads find its maximum by shuffles.
template <typename T>
__global__ void __launch_bounds__(256) cache4_append_kernel(const append_args a) {
  const cache4_append_params& p = a.p;
  __shared__ float2 turn[64];
  const int row = blockIdx.x, seq = row / p.m, i = row - seq * p.m;
  const int hd = p.c.hd, held = p.lengths[seq];
  if (p.theta > 0.f && threadIdx.x < hd / 2) {
    // p.positions may be far: the angle is brought within half a turn in 64 bits
    const double at = (double)(p.positions ? p.positions[seq] : held) + i;
    const double angle = at * exp2(-(double)(2 * (int)threadIdx.x) / hd * a.log2_theta);
    constexpr double TWO_PI_HI = 6.283185307179586232, TWO_PI_LO = 2.449293598294706414e-16;
    const double turns = rint(angle * 0.15915494309189533577);
    double s, c;
    sincos(fma(-turns, TWO_PI_LO, fma(-turns, TWO_PI_HI, angle)), &s, &c);
    turn[threadIdx.x] = make_float2((float)c, (float)s);
  }
  __syncthreads();
  auto rotate = [&](float (&x)[8], int o8) {
    if (!(p.theta > 0.f)) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 cs = turn[o8 * 4 + e];
      const float re = x[2 * e], im = x[2 * e + 1];
      // (products and sums rounded one by one: the codes of values at a border do not depend on how a compiler fuses them)
      x[2 * e] = __fsub_rn(__fmul_rn(re, cs.x), __fmul_rn(im, cs.y));
      x[2 * e + 1] = __fadd_rn(__fmul_rn(re, cs.y), __fmul_rn(im, cs.x));
    }
  };
  const int per_head = hd / 8;
  if (p.q) {
    const int octets = p.n_heads * per_head;
    const T* q = reinterpret_cast<const T*>(p.q) + (size_t)row * p.ld_q;
    T* q_out = reinterpret_cast<T*>(p.q_out) + (size_t)row * p.n_heads * hd;
    for (int o = threadIdx.x; o < octets; o += 256) {
      uint4 v = reinterpret_cast<const uint4*>(q)[o];
      if (p.theta > 0.f) {
        float x[8];
        unpack8<T>(v, x);
        rotate(x, o % per_head);
        v = pack8<T>(x);
      }
      reinterpret_cast<uint4*>(q_out)[o] = v;
    }
  }
  if (held < 0 || held >= p.c.ctx - i) return;  // no such sequence, or the row does not fit (for all threads of the CTA alike)
  const int octets = p.c.n_kv * per_head, padded = (2 * octets + 31) & ~31;
  for (int o = threadIdx.x; o < padded; o += 256) {
    const bool there = o < 2 * octets, is_v = o >= octets;
    const int ok = there ? (is_v ? o - octets : o) : 0, head = ok / per_head, o8 = ok - head * per_head;
    float x[8];
    unpack8<T>(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(is_v ? p.v_new : p.k_new) + (size_t)row * p.ld_kv)[ok], x);
    if (!is_v) rotate(x, o8);
    float most = 0.f;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = fmaxf(most, fabsf(x[e]));
      odd |= x[e] != x[e];
    }
    if (odd) most = __int_as_float(0x7f800000);  // (a maximum passes over a NaN)
    for (int w = 1; w < p.c.bs / 8; w <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
    const float s7 = seven_bits(__fdiv_rn(most, 7.5f));
    const __half scale = __float2half_rn(s7 > 8704.f ? 8704.f : s7);  // (a NaN stays)
    const float s = __half2float(scale);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = s > 0.f ? fminf(fmaxf(floorf(__fadd_rn(__fdiv_rn(x[e], s), 8.f)), 0.f), 15.f) : 8.f;
      word |= (uint32_t)c << (4 * e);
    }
    if (there) {
      const size_t at = ((size_t)seq * p.c.n_kv + head) * p.c.ctx + held + i;
      uint8_t* codes = (is_v ? p.c.v_codes : p.c.k_codes) + at * (hd / 2);
      reinterpret_cast<uint32_t*>(codes)[cache4_word(o8, hd / 32)] = word;
      if ((o8 * 8) % p.c.bs == 0) ((is_v ? p.c.v_scales : p.c.k_scales) + at * (hd / p.c.bs))[o8 * 8 / p.c.bs] = scale;
    }
  }
}

// One thread per eight dimensions.  Rows outside the cache give zeros.
template <typename T>
__global__ void __launch_bounds__(256) cache4_read_kernel(T* k_out, T* v_out, cache4_view c, const int* first, int count) {
  const int per_head = c.hd / 8;
  const size_t n = (size_t)c.n_seqs * c.n_kv * count * per_head;
  T* out = blockIdx.y ? v_out : k_out;
  if (!out) return;
  const uint8_t* codes = blockIdx.y ? c.v_codes : c.k_codes;
  const __half* scales = blockIdx.y ? c.v_scales : c.k_scales;
  for (size_t t = (size_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (size_t)gridDim.x * 256) {
    const int o8 = (int)(t % per_head);
    const size_t r = t / per_head;
    const int i = (int)(r % count);
    const size_t sh = r / count;
    const long long at = (long long)(first ? first[sh / c.n_kv] : 0) + i;
    float x[8] = {};
    if (at >= 0 && at < c.ctx) {
      const size_t place = sh * c.ctx + at;
      const uint32_t word = reinterpret_cast<const uint32_t*>(codes + place * (c.hd / 2))[cache4_word(o8, c.hd / 32)];
      const float s = __half2float(scales[place * (c.hd / c.bs) + o8 * 8 / c.bs]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = cache4_value(word, e, s);
    }
    reinterpret_cast<uint4*>(out)[t] = pack8<T>(x);
  }
}

}  // namespace

int launch_cache4_append(const cache4_append_params& p, int dtype, cudaStream_t stream) {
  int rc = check_cache4("cache4_append", p.c);
  if (rc) return rc;
  LCU_REQUIRE(dtype == OP_F16 || dtype == OP_BF16, "cache4_append: number format %d is not 0 (half) or 1 (bfloat16)", dtype);
  LCU_REQUIRE(p.k_new && p.v_new && p.lengths && (!p.q || p.q_out), "cache4_append: a null pointer");
  LCU_REQUIRE(p.m >= 1 && (!p.q || p.n_heads >= 1), "cache4_append: no rows or heads");
  LCU_REQUIRE((long long)p.c.n_seqs * p.m < (1ll << 31) && (long long)p.c.n_kv * p.c.hd < (1 << 24) && (long long)p.n_heads * p.c.hd < (1 << 24),
              "cache4_append: %d sequences of %d rows of %d / %d heads are too many", p.c.n_seqs, p.m, p.n_heads, p.c.n_kv);
  LCU_REQUIRE(p.ld_kv % 8 == 0 && p.ld_kv >= p.c.n_kv * p.c.hd && (!p.q || (p.ld_q % 8 == 0 && p.ld_q >= p.n_heads * p.c.hd)),
              "cache4_append: row strides must be multiples of 8 that hold a row");
  LCU_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.q_out | (uintptr_t)p.k_new | (uintptr_t)p.v_new) & 15) == 0, "cache4_append: rows must be 16-byte aligned");
  LCU_REQUIRE(!p.q || p.q_out != p.q || p.ld_q == p.n_heads * p.c.hd, "cache4_append: queries rotated in place must be dense");
  LCU_REQUIRE(p.theta == 0.f || (p.theta > 0.f && p.theta < 1e30f), "cache4_append: theta %g", (double)p.theta);
  if (int rc_dev = need_device()) return rc_dev;
  append_args a{p, p.theta > 0.f ? log2((double)p.theta) : 0.0};
  const unsigned rows = (unsigned)(p.c.n_seqs * p.m);
  if (dtype == OP_F16) cache4_append_kernel<__half><<<rows, 256, 0, stream>>>(a);
  else cache4_append_kernel<__nv_bfloat16><<<rows, 256, 0, stream>>>(a);
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

int launch_cache4_read(void* k_out, void* v_out, const cache4_view& c, const int* first, int count, int dtype, cudaStream_t stream) {
  int rc = check_cache4("cache4_read", c);
  if (rc) return rc;
  LCU_REQUIRE(dtype == OP_F16 || dtype == OP_BF16, "cache4_read: number format %d is not 0 (half) or 1 (bfloat16)", dtype);
  LCU_REQUIRE((k_out || v_out) && count >= 1, "cache4_read: nothing to read");
  LCU_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "cache4_read: outputs must be 16-byte aligned");
  if (int rc_dev = need_device()) return rc_dev;
  const size_t n = (size_t)c.n_seqs * c.n_kv * count * (c.hd / 8);
  const dim3 grid((unsigned)std::min<size_t>((n + 255) / 256, 148 * 32), 2);
  if (dtype == OP_F16) cache4_read_kernel<__half><<<grid, 256, 0, stream>>>((__half*)k_out, (__half*)v_out, c, first, count);
  else cache4_read_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>((__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, c, first, count);
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

}  // namespace lcu
