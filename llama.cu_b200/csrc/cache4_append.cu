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
// CTAs).  Bound by memory for prompts, by the launch and the chain load - angle - store for a token.  Angles are formed once per row and
// CTA, in 64 bits (a position of a hundred thousand leaves seven digits of a binary32 angle's turn).  A thread owns eight neighbouring
// dimensions at a time: one 16-byte load, the first ones requested ahead of the angles, its four rotation pairs, one word of codes; a block's
// threads find its maximum by shuffles.
template <typename T, int HD, int R>
__global__ void __launch_bounds__(256) cache4_append_kernel(const append_args a) {
  const cache4_append_params& p = a.p;
  constexpr int PER_HEAD = HD / 8;
  __shared__ float2 turn[R][HD / 2];
  __shared__ int s_seq[R], s_at[R];  // sequence and place of every row (-1: it is not written)
  const int rows = p.c.n_seqs * p.m, row0 = (int)(blockIdx.x / a.parts) * R, part = blockIdx.x % a.parts, lane = threadIdx.x & 31;
  // a row's octets: queries, keys, values, in units of 32 that each lie within one of the three; a warp takes every eighth of the CTA's
  const int n_q = p.q ? p.n_heads * PER_HEAD : 0, n_kv = p.c.n_kv * PER_HEAD;
  const int q_units = (n_q + 31) / 32, kv_units = (n_kv + 31) / 32, units = q_units + 2 * kv_units, step = 8 * a.parts;
  struct place {
    int r, u, o, kind;  // row and unit; octet within the row's queries (0), keys (1), values (2)
  };
  auto settle = [&](place& w) {
    while (w.u >= units) {
      w.u -= units;
      ++w.r;
    }
    w.kind = w.u < q_units ? 0 : w.u < q_units + kv_units ? 1 : 2;
    w.o = (w.u - (w.kind == 0 ? 0 : w.kind == 1 ? q_units : q_units + kv_units)) * 32 + lane;
  };
  auto load = [&](const place& w) {
    const int row = row0 + w.r;
    if (w.r >= R || row >= rows || w.o >= (w.kind ? n_kv : n_q)) return make_uint4(0, 0, 0, 0);
    const T* from = reinterpret_cast<const T*>(w.kind == 0 ? p.q : w.kind == 1 ? p.k_new : p.v_new) + (size_t)row * (w.kind ? p.ld_kv : p.ld_q);
    return reinterpret_cast<const uint4*>(from)[w.o];
  };
  place now{0, part * 8 + (int)(threadIdx.x >> 5), 0, 0};
  settle(now);
  uint4 v = load(now);
  if (threadIdx.x < R) {
    const int row = row0 + threadIdx.x, seq = min(row, rows - 1) / p.m, i = row - seq * p.m, held = p.lengths[seq];
    s_seq[threadIdx.x] = seq;
    s_at[threadIdx.x] = row < rows && held >= 0 && held < p.c.ctx - i ? held + i : -1;  // (a sequence in use, and room for the row)
  }
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
  }
  __syncthreads();
  while (now.r < R && row0 + now.r < rows) {
    place ahead = now;
    ahead.u += step;
    settle(ahead);
    const uint4 v_ahead = load(ahead);
    const int o8 = now.o % PER_HEAD, head = now.o / PER_HEAD;
    const bool there = now.o < (now.kind ? n_kv : n_q);
    float x[8];
    unpack8<T>(v, x);
    if (now.kind < 2 && p.theta > 0.f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 cs = turn[now.r][o8 * 4 + e];
        const float re = x[2 * e], im = x[2 * e + 1];
        // (products and sums rounded one by one: the codes of values at a border do not depend on how a compiler fuses them)
        x[2 * e] = __fsub_rn(__fmul_rn(re, cs.x), __fmul_rn(im, cs.y));
        x[2 * e + 1] = __fadd_rn(__fmul_rn(re, cs.y), __fmul_rn(im, cs.x));
      }
    }
    if (now.kind == 0) {
      if (there) reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out) + (size_t)(row0 + now.r) * (p.n_heads * HD))[now.o] = p.theta > 0.f ? pack8<T>(x) : v;
    } else {
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
      const int slot = s_at[now.r];
      if (there && slot >= 0) {
        const size_t at = ((size_t)s_seq[now.r] * p.c.n_kv + head) * p.c.ctx + slot;
        uint8_t* codes = (now.kind == 2 ? p.c.v_codes : p.c.k_codes) + at * (HD / 2);
        reinterpret_cast<uint32_t*>(codes)[cache4_word(o8, HD / 32)] = word;
        if ((o8 * 8) % p.c.bs == 0) ((now.kind == 2 ? p.c.v_scales : p.c.k_scales) + at * (HD / p.c.bs))[o8 * 8 / p.c.bs] = scale;
      }
    }
    now = ahead;
    v = v_ahead;
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
  LCU_REQUIRE(!p.q || p.q_out != p.q || p.ld_q == p.n_heads * p.c.hd, "cache4_append: queries rotated in place must be dense");
  LCU_REQUIRE(p.theta == 0.f || (p.theta > 0.f && p.theta < 1e30f), "cache4_append: theta %g", (double)p.theta);
  if (int rc_dev = need_device()) return rc_dev;
  append_args a{p, {}, 1};
  if (p.theta > 0.f)
    for (int b = 0; b < 6; ++b) a.powers[b] = exp2(-(double)(2 << b) / p.c.hd * log2((double)p.theta));
  // four rows per CTA from four waves of CTAs on; a row's units shared by CTAs while there are fewer rows than that
  const int rows = p.c.n_seqs * p.m, per_head = p.c.hd / 8;
  const int units = p.q ? (p.n_heads * per_head + 31) / 32 + 2 * ((p.c.n_kv * per_head + 31) / 32) : 2 * ((p.c.n_kv * per_head + 31) / 32);
  const bool four = rows >= 4 * 148;
  if (!four) a.parts = std::max(1, std::min((units + 7) / 8, 8 * 148 / rows));
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
  if (int rc_dev = need_device()) return rc_dev;
  LCU_REQUIRE((long long)c.n_seqs * c.n_kv < (1ll << 31), "cache4_read: %d sequences of %d heads are too many", c.n_seqs, c.n_kv);
  if (dtype == OP_F16) launch_read((__half*)k_out, (__half*)v_out, c, first, count, stream);
  else launch_read((__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, c, first, count, stream);
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

}  // namespace lcu
