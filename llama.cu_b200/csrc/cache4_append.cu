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
  double powers[6];  // theta^(-2 * 2^b / hd): a pair's frequency is the product of those its number's bits name
  int parts;         // CTAs that share a run of rows
};

// binary32 s >= 0 to 7 significant bits, ties to even (a NaN or an infinity gives a NaN)
__device__ __forceinline__ float seven_bits(float s) {
  uint32_t b = __float_as_uint(s);
  if (b >= 0x7f800000u) return __int_as_float(0x7fffffff);
  b = (b + 0xffffu + ((b >> 17) & 1u)) & ~0x1ffffu;
  return __uint_as_float(b);
}

// A CTA takes R rows (four of a prompt's, whose 64-bit angles then keep all its threads busy; a single token's heads are shared by `parts`
// CTAs).  Bound by memory for prompts, with the arithmetic of rounding close behind, by the launch and the chain load - angle - store for a token.
// Angles are formed once per row and CTA, in 64 bits (a position of a hundred thousand leaves seven digits of a binary32 angle's turn).  A
// thread owns the same eight dimensions of every head it comes to, so it reads a row's four rotations once; its first queries are
// requested ahead of the angles.  A block's threads find its maximum by shuffles.
template <typename T, int HD, int R>
__global__ void __launch_bounds__(256) cache4_append_kernel(const append_args a) {
  const cache4_append_params& p = a.p;
  constexpr int PER_HEAD = HD / 8, AHEAD = 2;
  __shared__ float2 turn[R][HD / 2];
  const int rows = p.c.n_seqs * p.m, row0 = (int)(blockIdx.x / a.parts) * R;
  const int start = (int)(blockIdx.x % a.parts) * 256 + (int)threadIdx.x, stride = 256 * a.parts, o8 = start % PER_HEAD;  // (stride: whole heads)
  const int n_q = p.q ? p.n_heads * PER_HEAD : 0, n_kv = p.c.n_kv * PER_HEAD;
  auto q_row = [&](int row) { return reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (size_t)row * p.ld_q); };
  uint4 ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (start + k * stride < n_q) ahead[k] = q_row(row0)[start + k * stride];
  if (p.theta > 0.f) {
    for (int t = threadIdx.x; t < R * (HD / 2); t += 256) {
      const int r = t / (HD / 2), e = t % (HD / 2), row = min(row0 + r, rows - 1), seq = row / p.m;
      const double at = (double)(p.positions ? p.positions[seq] : p.lengths[seq]) + (row - seq * p.m);
      double f = 1.0;
#pragma unroll
      for (int b = 0; b < 6; ++b) f *= e >> b & 1 ? a.powers[b] : 1.0;
      const double angle = at * f;  // (positions may be far: brought within half a turn in 64 bits)
      constexpr double TWO_PI_HI = 6.283185307179586232, TWO_PI_LO = 2.449293598294706414e-16;
      const double turns = rint(angle * 0.15915494309189533577);
      double s, c;
      sincos(fma(-turns, TWO_PI_LO, fma(-turns, TWO_PI_HI, angle)), &s, &c);
      turn[r][e] = make_float2((float)c, (float)s);
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int r = 0; r < R && row0 + r < rows; ++r) {
    const int row = row0 + r;
    float2 cs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = p.theta > 0.f ? turn[r][o8 * 4 + e] : make_float2(1.f, 0.f);
    auto rotate = [&](float (&x)[8]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float re = x[2 * e], im = x[2 * e + 1];
        // (products and sums rounded one by one: the codes of values at a border do not depend on how a compiler fuses them)
        x[2 * e] = __fsub_rn(__fmul_rn(re, cs[e].x), __fmul_rn(im, cs[e].y));
        x[2 * e + 1] = __fadd_rn(__fmul_rn(re, cs[e].y), __fmul_rn(im, cs[e].x));
      }
    };
    uint4* q_out = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out) + (size_t)row * (p.n_heads * HD));
    for (int o = start; o < n_q; o += AHEAD * stride) {
      uint4 v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        v[k] = ahead[k];
        // the next ones: of this row, or the next row's first
        const int next = o + (AHEAD + k) * stride;
        if (next < n_q) ahead[k] = q_row(row)[next];
        else if (o + AHEAD * stride >= n_q && r + 1 < R && row + 1 < rows && start + k * stride < n_q) ahead[k] = q_row(row + 1)[start + k * stride];
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (o + k * stride >= n_q) break;
        if (p.theta > 0.f) {
          float x[8];
          unpack8<T>(v[k], x);
          rotate(x);
          v[k] = pack8<T>(x);
        }
        q_out[o + k * stride] = v[k];
      }
    }
    const int seq = row / p.m, i = row - seq * p.m, held = p.lengths[seq];
    if (held < 0 || held >= p.c.ctx - i) continue;  // no such sequence, or no room for the row (for all threads alike)
    for (int o = start; o < ((2 * n_kv + 31) & ~31); o += stride) {
      const bool there = o < 2 * n_kv, is_v = o >= n_kv;
      const int ok = there ? (is_v ? o - n_kv : o) : o8;
      float x[8];
      unpack8<T>(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(is_v ? p.v_new : p.k_new) + (size_t)row * p.ld_kv)[ok], x);
      if (!is_v && p.theta > 0.f) rotate(x);
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
      uint32_t word = 0x88888888u;
      if (s > 0.f) {
        // floor by a sum rounded down (its last bits are the whole number), codes put together by multiplying, less the eight exponents
        word = 0;
#pragma unroll
        for (int e = 7; e >= 0; --e) word = word * 16u + __float_as_uint(__fadd_rd(fminf(fmaxf(__fadd_rn(__fdiv_rn(x[e], s), 8.f), 0.f), 15.5f), 8388608.f));
        word -= 0x4b000000u * 0x11111111u;
      }
      if (there) {
        const size_t at = ((size_t)seq * p.c.n_kv + ok / PER_HEAD) * p.c.ctx + held + i;
        uint8_t* codes = (is_v ? p.c.v_codes : p.c.k_codes) + at * (HD / 2);
        reinterpret_cast<uint32_t*>(codes)[cache4_word(o8, HD / 32)] = word;
        if ((o8 * 8) % p.c.bs == 0) ((is_v ? p.c.v_scales : p.c.k_scales) + at * (HD / p.c.bs))[o8 * 8 / p.c.bs] = scale;
      }
    }
  }
}

// One thread per eight dimensions.  Rows outside the cache give zeros.
template <typename T, int HD>
__global__ void __launch_bounds__(256) cache4_read_kernel(T* k_out, T* v_out, cache4_view c, const int* first, int count) {
  constexpr int PER_HEAD = HD / 8;
  T* out = blockIdx.z ? v_out : k_out;
  if (!out) return;
  const uint8_t* codes = blockIdx.z ? c.v_codes : c.k_codes;
  const __half* scales = blockIdx.z ? c.v_scales : c.k_scales;
  // a run of rows of one (sequence, head) per CTA
  for (int sh = blockIdx.y; sh < c.n_seqs * c.n_kv; sh += gridDim.y) {
    const long long start = first ? first[sh / c.n_kv] : 0;
    const size_t n = (size_t)count * PER_HEAD;
    for (size_t t = (size_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (size_t)gridDim.x * 256) {
      const int o8 = (int)(t % PER_HEAD);
      const long long at = start + (long long)(t / PER_HEAD);
      float x[8] = {};
      if (at >= 0 && at < c.ctx) {
        const size_t place = (size_t)sh * c.ctx + at;
        const uint32_t word = reinterpret_cast<const uint32_t*>(codes + place * (HD / 2))[cache4_word(o8, HD / 32)];
        const float s = __half2float(scales[place * (HD / c.bs) + o8 * 8 / c.bs]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = cache4_value(word, e, s);
      }
      reinterpret_cast<uint4*>(out)[(size_t)sh * n + t] = pack8<T>(x);
    }
  }
}

template <typename T>
void launch_read(T* k_out, T* v_out, const cache4_view& c, const int* first, int count, cudaStream_t stream) {
  const size_t per_unit = ((size_t)count * (c.hd / 8) + 255) / 256;
  const dim3 grid((unsigned)std::min<size_t>(per_unit, 4096), (unsigned)std::min(c.n_seqs * c.n_kv, 32768), 2);
  if (c.hd == 128) cache4_read_kernel<T, 128><<<grid, 256, 0, stream>>>(k_out, v_out, c, first, count);
  else cache4_read_kernel<T, 64><<<grid, 256, 0, stream>>>(k_out, v_out, c, first, count);
}

template <typename T>
void launch_append(const append_args& a, bool four, unsigned ctas, cudaStream_t stream) {
  if (a.p.c.hd == 128) four ? cache4_append_kernel<T, 128, 4><<<ctas, 256, 0, stream>>>(a) : cache4_append_kernel<T, 128, 1><<<ctas, 256, 0, stream>>>(a);
  else four ? cache4_append_kernel<T, 64, 4><<<ctas, 256, 0, stream>>>(a) : cache4_append_kernel<T, 64, 1><<<ctas, 256, 0, stream>>>(a);
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
  LCU_REQUIRE(words_aligned(p.lengths, p.positions), "cache4_append: lengths and positions must be 4-byte aligned");
  LCU_REQUIRE(!p.q || p.q_out != p.q || p.ld_q == p.n_heads * p.c.hd, "cache4_append: queries rotated in place must be dense");
  LCU_REQUIRE(p.theta == 0.f || (p.theta > 0.f && p.theta < 1e30f), "cache4_append: theta %g", (double)p.theta);
  if (int rc_dev = need_device()) return rc_dev;
  append_args a{p, {}, 1};
  if (p.theta > 0.f)
    for (int b = 0; b < 6; ++b) a.powers[b] = exp2(-(double)(2 << b) / p.c.hd * log2((double)p.theta));
  // four rows per CTA from four CTAs per SM on; a row's heads shared by CTAs while there are fewer
  const int rows = p.c.n_seqs * p.m, octets = std::max(p.q ? p.n_heads : 0, 2 * p.c.n_kv) * (p.c.hd / 8);
  const bool four = rows >= 4 * 148;
  if (!four) a.parts = std::max(1, std::min((octets + 255) / 256, 8 * 148 / rows));
  const unsigned ctas = four ? (unsigned)((rows + 3) / 4) : (unsigned)rows * a.parts;
  if (dtype == OP_F16) launch_append<__half>(a, four, ctas, stream);
  else launch_append<__nv_bfloat16>(a, four, ctas, stream);
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

int launch_cache4_read(void* k_out, void* v_out, const cache4_view& c, const int* first, int count, int dtype, cudaStream_t stream) {
  int rc = check_cache4("cache4_read", c);
  if (rc) return rc;
  LCU_REQUIRE(dtype == OP_F16 || dtype == OP_BF16, "cache4_read: number format %d is not 0 (half) or 1 (bfloat16)", dtype);
  LCU_REQUIRE((k_out || v_out) && count >= 1, "cache4_read: nothing to read");
  LCU_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "cache4_read: outputs must be 16-byte aligned");
  LCU_REQUIRE(words_aligned(first), "cache4_read: first rows must be 4-byte aligned");
  LCU_REQUIRE((long long)c.n_seqs * c.n_kv < (1ll << 31), "cache4_read: %d sequences of %d heads are too many", c.n_seqs, c.n_kv);
  if (int rc_dev = need_device()) return rc_dev;
  if (dtype == OP_F16) launch_read((__half*)k_out, (__half*)v_out, c, first, count, stream);
  else launch_read((__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, c, first, count, stream);
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

}  // namespace lcu
