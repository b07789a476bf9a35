// Attention of few rows over the 4-bit cache (cache4.cuh): single tokens, and a handful of rows (a draft that is checked).
//
//   s_jc = q_c . k_j / sqrt(head_dim),  o_c = sum_j e^(s_jc - max) v_j / sum_j e^(s_jc - max),   columns c = (row, head of the key/value head)
// One cluster of CTAs per (sequence, key/value head) walks the cached rows once, whatever the number of columns up to 16; CTAs share the
// rows in runs, warps interleave tiles of 16.  What bounds it is the cache's bytes (at most 0.57 a value) and, close behind, the
// instructions that turn nibbles into halves: 41 values a cycle and SM arrive, a value costs about one lane's instruction and a half.
// So nothing else happens to a value: codes become code - 7.5 as halves in three bit operations per four values and one subtraction per
// two, and go straight into the registers of m16n8k16 products, with the cached rows as the wide side (16 keys x 8 columns for the
// scores, 16 dimensions x 8 columns for the outputs).  The order of the codes in a row (cache4.cuh) is such that a lane's words of 32
// dimensions belong to one block of scales: scores are scaled in binary32 per block after the product, exactly; values take their scale
// as halves, exactly too (7-bit scales).  Scores, sums and outputs are binary32; probabilities are rounded to half (2^-11) as operands.
// The running maximum of a column is raised only when a score passes it by 8 (powers of two): e^(s - max) up to 256 fits a half.
//
// A block of values whose scale is no number counts as zeros in the product, and the first such row is remembered per block: columns
// that see it get NaN there, columns of earlier rows of the same tile do not.
#include "cache4_attention.cuh"

#include <algorithm>
#include <type_traits>

namespace lcu {
namespace {

constexpr int ST_WARPS = 8, ST_THREADS = 32 * ST_WARPS, ST_TILE = 16;

struct step_args {
  cache4_attention_params p;
  float* scores;     // [n_seqs * m][n_heads][max_len], powers of two (weights only)
};

__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// code - 7.5 for the nibbles i of both 16-bit halves of a word, i = 0 .. 3: bits 4 .. 7 of a half with exponent 6 are sixteenths of 64 + code
__device__ __forceinline__ void centred(uint32_t w, uint32_t (&h)[4]) {
  constexpr uint32_t MASK = 0x00f000f0u, BASE = 0x54005400u;
  const __half2 mid = __halves2half2(__ushort_as_half(0x5478), __ushort_as_half(0x5478));  // 71.5
  const uint32_t b[4] = {((w << 4) & MASK) | BASE, (w & MASK) | BASE, ((w >> 4) & MASK) | BASE, ((w >> 8) & MASK) | BASE};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&b[i]), mid);
    h[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ uint32_t scaled(uint32_t h, __half2 s) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h), s);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // an 8 x 8 tile of halves, two neighbours of a row per lane
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ __half half_of(uint32_t v, int hi) { return __ushort_as_half((unsigned short)(hi ? v >> 16 : v & 0xffff)); }

// what a lane holds of a tile: octet t of every 32 dimensions of two keys; VW words of four values' rows; their scales
template <int HD, int NB>
struct tile_words {
  static constexpr int G = HD / 32, VW = HD / 64;
  uint32_t k[2][G], v[4][VW], ks[2][NB == 4 ? 2 : 1], vs[4];
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&r)[N], const uint8_t* p) {
  if constexpr (N == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r[0] = v.x; r[1] = v.y;
  } else {
    r[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

template <typename T, int HD, int NB, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(ST_THREADS, NT == 1 ? 2 : 1) attention_step_kernel(const step_args a) {
  using words = tile_words<HD, NB>;
  constexpr int G = words::G, VW = words::VW, BG = G / NB;  // BG groups of 32 dimensions per block
  constexpr bool TWO = HD == 128 && NB == 4;                // a lane's two value words lie in two blocks
  constexpr int COLS = 8 * NT;
  extern __shared__ float s_o[];                            // [ST_WARPS][COLS][HD]; then the CTA's sums in the first [COLS][HD]
  __shared__ float2 s_ml[ST_WARPS][COLS], s_cta[COLS], s_fin[COLS];
  __shared__ int s_bad[4];
  const cache4_attention_params& p = a.p;
  const int rank = (int)cluster_ctarank(), cs = (int)cluster_nctarank();
  const int unit = blockIdx.x / cs, seq = unit / p.c.n_kv, kvh = unit - seq * p.c.n_kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / p.c.n_kv, n_cols = p.m * group, held = p.lengths[seq];
  const int bound = min(p.c.ctx, p.max_len);
  auto limit_of = [&](int c) { return c < n_cols ? (int)min((long long)held + c / group + 1, (long long)bound) : 0; };
  auto row_of = [&](int c) { return (size_t)seq * p.m + c / group; };
  auto head_of = [&](int c) { return kvh * group + c % group; };
  if (held < 0) {  // (the whole cluster)
    for (int e = rank * ST_THREADS + tid; e < n_cols * HD / 2; e += cs * ST_THREADS)
      reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + row_of(e / (HD / 2)) * p.ld_out + head_of(e / (HD / 2)) * HD)[e % (HD / 2)] = 0u;
    return;
  }
  const int T_all = limit_of(n_cols - 1), T_first = limit_of(0);
  const int tiles = (T_all + ST_TILE - 1) / ST_TILE;
  const int tile_lo = (int)((long long)tiles * rank / cs), tile_hi = (int)((long long)tiles * (rank + 1) / cs);
  const size_t unit_rows = (size_t)unit * p.c.ctx;
  const uint8_t* k_codes = p.c.k_codes + unit_rows * (HD / 2) + t * (4 * G);
  const uint8_t* v_codes = p.c.v_codes + unit_rows * (HD / 2) + g * (4 * VW);
  const uint8_t* k_scales = reinterpret_cast<const uint8_t*>(p.c.k_scales + unit_rows * NB);
  const int v_block = (g * VW % G) / BG;  // the (first) block of this lane's values
  const uint8_t* v_scales = reinterpret_cast<const uint8_t*>(p.c.v_scales + unit_rows * NB + v_block);
  // tile row r stands for key perm(r): rows 2t, 2t+1, 2t+8, 2t+9, whose probabilities a lane multiplies with values, are keys 4t .. 4t+3
  const int key_a = 4 * (g >> 1) + (g & 1);  // rows g and g + 8: keys key_a and key_a + 2
  auto fetch = [&](words& w, int tile) {
    const int j0 = tile * ST_TILE, last = T_all - 1;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const size_t j = min(j0 + key_a + 2 * r, last);
      load_words<G>(w.k[r], k_codes + j * (HD / 2));
      if constexpr (NB == 4) load_words<2>(w.ks[r], k_scales + j * 8);
      else if constexpr (NB == 2) load_words<1>(w.ks[r], k_scales + j * 4);
      else w.ks[r][0] = __ldg(reinterpret_cast<const unsigned short*>(k_scales + j * 2));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t j = min(j0 + 4 * t + i, last);
      load_words<VW>(w.v[i], v_codes + j * (HD / 2));
      if constexpr (TWO) w.vs[i] = __ldg(reinterpret_cast<const uint32_t*>(v_scales + j * (2 * NB)));
      else w.vs[i] = __ldg(reinterpret_cast<const unsigned short*>(v_scales + j * (2 * NB)));
    }
  };

  for (int c0 = 0; c0 < n_cols; c0 += COLS) {  // (once, unless there are more than 16 columns)
    // ---- queries as the narrow operand: column g of each n-tile, octet t of every 32 dimensions, in the codes' order of pairs
    uint32_t qf[NT][G][4];
    float f[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = c0 + n * 8 + g;
      float x[G][8], most = 0.f;
#pragma unroll
      for (int gd = 0; gd < G; ++gd) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < n_cols) v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + row_of(c) * p.ld_q + head_of(c) * HD + gd * 32 + t * 8);
        unpack8<T>(v, x[gd]);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[gd][e]));
      }
      // bfloat16 queries: a power of two takes the column's largest magnitude into [1, 2); halves are exact from 2^-14 of it on
      float up = 1.f, down = 1.f;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const uint32_t ex = __float_as_uint(most) >> 23;
        if (ex >= 1 && ex <= 253) {
          up = __uint_as_float((254u - ex) << 23);
          down = __uint_as_float(ex << 23);
        }
      }
#pragma unroll
      for (int gd = 0; gd < G; ++gd)
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[n][gd][i] = pack2<__half>(x[gd][i] * up, x[gd][i + 4] * up);
      const float factor = down * (1.4426950408889634f * rsqrtf((float)HD));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f[n][e] = __shfl_sync(0xffffffffu, factor, (2 * t + e) * 4);
        lim[n][e] = limit_of(c0 + n * 8 + 2 * t + e);
      }
    }
    float o[NT][VW * 4][4], mx[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < VW * 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[n][e] = -INFINITY;
        sum[n][e] = 0.f;
      }
    }
    int bad0 = 0x7fffffff, bad1 = 0x7fffffff;
    if (tid < 4) s_bad[tid] = 0x7fffffff;

    words w;
    int tile = tile_lo + warp;
    if (tile < tile_hi) fetch(w, tile);
    for (; tile < tile_hi; tile += ST_WARPS) {
      const words now = w;
      if (tile + ST_WARPS < tile_hi) fetch(w, tile + ST_WARPS);
      const int j0 = tile * ST_TILE;
      // ---- scores
      float s[NT][4];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float acc[NT][4];
#pragma unroll
        for (int gb = 0; gb < BG; ++gb) {
          const int gd = b * BG + gb;
          uint32_t ka[4], kb[4];
          centred(now.k[0][gd], ka);
          centred(now.k[1][gd], kb);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (gb == 0) mma_16816_from(acc[n], ka[0], kb[0], ka[1], kb[1], qf[n][gd][0], qf[n][gd][1], 0.f);
            else mma_16816(acc[n], ka[0], kb[0], ka[1], kb[1], qf[n][gd][0], qf[n][gd][1]);
            mma_16816(acc[n], ka[2], kb[2], ka[3], kb[3], qf[n][gd][2], qf[n][gd][3]);
          }
        }
        const float sa = __half2float(half_of(now.ks[0][b >> 1], b & 1)), sb = __half2float(half_of(now.ks[1][b >> 1], b & 1));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[n][0] = b ? fmaf(sa, acc[n][0], s[n][0]) : sa * acc[n][0];
          s[n][1] = b ? fmaf(sa, acc[n][1], s[n][1]) : sa * acc[n][1];
          s[n][2] = b ? fmaf(sb, acc[n][2], s[n][2]) : sb * acc[n][2];
          s[n][3] = b ? fmaf(sb, acc[n][3], s[n][3]) : sb * acc[n][3];
        }
      }
      const bool ragged = j0 + ST_TILE > T_first;  // (of the last rows some columns see fewer, and the tile may hang over the end)
      bool raise = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= f[n][e & 1];
          if (ragged && j0 + key_a + (e & 2) >= lim[n][e & 1]) s[n][e] = -INFINITY;
        }
        if constexpr (WEIGHTS) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = c0 + n * 8 + 2 * t + (e & 1), j = j0 + key_a + (e & 2);
            if (c < n_cols && j < T_all) a.scores[(row_of(c) * p.n_heads + head_of(c)) * p.max_len + j] = s[n][e];
          }
        }
        raise |= fmaxf(s[n][0], s[n][2]) > mx[n][0] + 8.f || fmaxf(s[n][1], s[n][3]) > mx[n][1] + 8.f;
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float k[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[n][e], s[n][e + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, mx[n][e]);
            k[e] = mx[n][e] == -INFINITY ? 0.f : ex2(mx[n][e] - top);
            mx[n][e] = top;
            sum[n][e] *= k[e];
          }
#pragma unroll
          for (int i = 0; i < VW * 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] *= k[e & 1];
        }
      }
      // ---- probabilities, with columns as rows
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float b0 = mx[n][0] == -INFINITY ? 0.f : mx[n][0], b1 = mx[n][1] == -INFINITY ? 0.f : mx[n][1];
        const float e0 = ex2(s[n][0] - b0), e1 = ex2(s[n][1] - b1), e2 = ex2(s[n][2] - b0), e3 = ex2(s[n][3] - b1);
        sum[n][0] += e0 + e2;
        sum[n][1] += e1 + e3;
        pf[n][0] = transposed(pack2<__half>(e0, e1));
        pf[n][1] = transposed(pack2<__half>(e2, e3));
      }
      // ---- values
      uint32_t vs[4] = {now.vs[0], now.vs[1], now.vs[2], now.vs[3]};
      if (j0 + ST_TILE > T_all) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + 4 * t + i >= T_all) vs[i] = 0u;
      }
      {
        const __half2 x0 = *reinterpret_cast<const __half2*>(&vs[0]), x1 = *reinterpret_cast<const __half2*>(&vs[1]);
        const __half2 x2 = *reinterpret_cast<const __half2*>(&vs[2]), x3 = *reinterpret_cast<const __half2*>(&vs[3]);
        const __half2 z = __hadd2(__hadd2(x0, x1), __hadd2(x2, x3));  // (up to 4 x 8704: finite)
        const __half zz = __hadd(__low2half(z), __high2half(z));
        if (__hisnan(zz)) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (__hisnan(half_of(vs[i], 0))) {
              bad0 = min(bad0, j0 + 4 * t + i);
              vs[i] &= 0xffff0000u;
            }
            if (__hisnan(half_of(vs[i], 1))) {
              bad1 = min(bad1, j0 + 4 * t + i);
              vs[i] &= 0x0000ffffu;
            }
          }
        }
      }
#pragma unroll
      for (int vw = 0; vw < VW; ++vw) {
        const uint32_t pick = TWO && vw ? 0x7632u : 0x5410u;
        const uint32_t s01w = __byte_perm(vs[0], vs[1], pick), s23w = __byte_perm(vs[2], vs[3], pick);
        const __half2 s01 = *reinterpret_cast<const __half2*>(&s01w), s23 = *reinterpret_cast<const __half2*>(&s23w);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t h01[4], h23[4];
          centred(__byte_perm(now.v[0][vw], now.v[1][vw], hh ? 0x7632 : 0x5410), h01);
          centred(__byte_perm(now.v[2][vw], now.v[3][vw], hh ? 0x7632 : 0x5410), h23);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h01[i] = scaled(h01[i], s01);
            h23[i] = scaled(h23[i], s23);
          }
#pragma unroll
          for (int mm = 0; mm < 2; ++mm)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_16816(o[n][vw * 4 + hh * 2 + mm], h01[2 * mm], h01[2 * mm + 1], h23[2 * mm], h23[2 * mm + 1], pf[n][0], pf[n][1]);
        }
      }
    }

    // ---- the warps meet
    const int here = min(COLS, n_cols - c0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[n][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int c = n * 8 + 2 * t + e;
        if (g == 0) s_ml[warp][c] = make_float2(mx[n][e], l);
        if (c < here) {
#pragma unroll
          for (int i = 0; i < VW * 4; ++i) {
            const int word = g * VW + i / 4, d = (word % G) * 32 + (word / G) * 8 + (i % 4) * 2;
            *reinterpret_cast<float2*>(&s_o[(warp * COLS + c) * HD + d]) = make_float2(o[n][i][e], o[n][i][e + 2]);
          }
        }
      }
    }
    __syncthreads();  // (s_bad is set)
    bad0 = min(bad0, __shfl_xor_sync(0xffffffffu, bad0, 1));
    bad0 = min(bad0, __shfl_xor_sync(0xffffffffu, bad0, 2));
    if (t == 0 && bad0 != 0x7fffffff) atomicMin(&s_bad[v_block], bad0);
    if constexpr (TWO) {
      bad1 = min(bad1, __shfl_xor_sync(0xffffffffu, bad1, 1));
      bad1 = min(bad1, __shfl_xor_sync(0xffffffffu, bad1, 2));
      if (t == 0 && bad1 != 0x7fffffff) atomicMin(&s_bad[v_block + 1], bad1);
    }
    if (tid < here) {
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w8 = 0; w8 < ST_WARPS; ++w8) top = fmaxf(top, s_ml[w8][tid].x);
#pragma unroll
      for (int w8 = 0; w8 < ST_WARPS; ++w8) {
        const float k = top == -INFINITY || s_ml[w8][tid].x == -INFINITY ? 1.f : ex2(s_ml[w8][tid].x - top);  // (a maximum of nothing: a sum of 0, or of NaN)
        l += s_ml[w8][tid].y * k;
      }
      s_cta[tid] = make_float2(top, l);
    }
    __syncthreads();
    for (int e = tid; e < here * HD; e += ST_THREADS) {
      const int c = e / HD;
      const float top = s_cta[c].x;
      float v = 0.f;
#pragma unroll
      for (int w8 = 0; w8 < ST_WARPS; ++w8) {
        const float k = top == -INFINITY || s_ml[w8][c].x == -INFINITY ? 1.f : ex2(s_ml[w8][c].x - top);
        v += s_o[w8 * COLS * HD + e] * k;
      }
      s_o[e] = v;  // (this thread alone reads and writes place e of the first warp's part)
    }
    // ---- the CTAs meet
    cluster_sync();
    if (tid < here) {
      float top = -INFINITY, l = 0.f;
      const uint32_t mine = smem_u32(&s_cta[tid]);
      for (int r = 0; r < cs; ++r) top = fmaxf(top, ld_dsmem_f32(mapa(mine, r)));
      for (int r = 0; r < cs; ++r) {
        const float m1 = ld_dsmem_f32(mapa(mine, r)), l1 = ld_dsmem_f32(mapa(mine + 4, r));
        l += l1 * (top == -INFINITY || m1 == -INFINITY ? 1.f : ex2(m1 - top));
      }
      s_fin[tid] = make_float2(top, 1.f / l);
    }
    __syncthreads();
    for (int e = rank * ST_THREADS + tid; e < here * HD / 2; e += cs * ST_THREADS) {
      const int c = e / (HD / 2), d = 2 * (e % (HD / 2));
      const float top = s_fin[c].x;
      float x = 0.f, y = 0.f;
      int bad = 0x7fffffff;
      for (int r = 0; r < cs; ++r) {
        const float m1 = ld_dsmem_f32(mapa(smem_u32(&s_cta[c]), r));
        const float k = top == -INFINITY || m1 == -INFINITY ? 1.f : ex2(m1 - top);
        x += ld_dsmem_f32(mapa(smem_u32(&s_o[c * HD + d]), r)) * k;
        y += ld_dsmem_f32(mapa(smem_u32(&s_o[c * HD + d + 1]), r)) * k;
        bad = min(bad, __float_as_int(ld_dsmem_f32(mapa(smem_u32(&s_bad[d * NB / HD]), r))));
      }
      const float rl = bad < limit_of(c0 + c) ? __int_as_float(0x7fffffff) : s_fin[c].y;
      reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + row_of(c0 + c) * p.ld_out + head_of(c0 + c) * HD)[d / 2] = pack2<T>(x * rl, y * rl);
    }
    // ---- weights of this CTA's rows: every lane reads the scores that it wrote
    if constexpr (WEIGHTS) {
      for (int u = tile_lo + warp; u < tile_hi; u += ST_WARPS) {
        float add[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int lc = n * 8 + 2 * t + (e & 1), c = c0 + lc, j = u * ST_TILE + key_a + (e & 2);
            if (c < n_cols && j < lim[n][e & 1]) add[e >> 1] += ex2(a.scores[(row_of(c) * p.n_heads + head_of(c)) * p.max_len + j] - s_fin[lc].x) * s_fin[lc].y;
          }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          add[r] += __shfl_xor_sync(0xffffffffu, add[r], 1);
          add[r] += __shfl_xor_sync(0xffffffffu, add[r], 2);
          const int j = u * ST_TILE + key_a + 2 * r;
          if (t == 0 && j < T_all) {
            float* at = p.weights + unit_rows + j;
            if (c0) *at += add[r];
            else *at = p.beta == 0.f || j >= held ? add[r] : fmaf(p.beta, *at, add[r]);
          }
        }
      }
    }
    cluster_sync();  // (no CTA leaves, or starts on other columns, while another reads its shared memory)
  }
}

template <typename T, int HD, int NB, int NT, bool WEIGHTS>
int launch_step(const step_args& a, int cs, cudaStream_t stream) {
  constexpr size_t SMEM = (size_t)ST_WARPS * 8 * NT * HD * sizeof(float);
  auto* kernel = attention_step_kernel<T, HD, NB, NT, WEIGHTS>;
  static bool attr_done[16] = {};
  int dev = 0;
  LCU_CUDA(cudaGetDevice(&dev));
  if (dev >= 16 || !attr_done[dev]) {
    LCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    if (dev < 16) attr_done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cs * a.p.c.n_seqs * a.p.c.n_kv);
  cfg.blockDim = dim3(ST_THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LCU_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return LCU_OK;
}

template <typename T, int HD, int NB>
int launch_cols(const step_args& a, int cs, cudaStream_t stream) {
  const bool one = a.p.m * (a.p.n_heads / a.p.c.n_kv) <= 8;
  if (a.p.weights) return one ? launch_step<T, HD, NB, 1, true>(a, cs, stream) : launch_step<T, HD, NB, 2, true>(a, cs, stream);
  return one ? launch_step<T, HD, NB, 1, false>(a, cs, stream) : launch_step<T, HD, NB, 2, false>(a, cs, stream);
}

template <typename T>
int launch_shape(const step_args& a, int cs, cudaStream_t stream) {
  const int nb = a.p.c.hd / a.p.c.bs;
  if (a.p.c.hd == 128) {
    if (nb == 4) return launch_cols<T, 128, 4>(a, cs, stream);
    if (nb == 2) return launch_cols<T, 128, 2>(a, cs, stream);
    return launch_cols<T, 128, 1>(a, cs, stream);
  }
  if (nb == 2) return launch_cols<T, 64, 2>(a, cs, stream);
  return launch_cols<T, 64, 1>(a, cs, stream);
}

}  // namespace

size_t attention_cache4_step_workspace(int n_seqs, int m, int n_heads, int max_len, bool weights) {
  return weights ? (size_t)n_seqs * m * n_heads * max_len * sizeof(float) : 0;
}

// CTAs that share a (sequence, key/value head): enough for two per SM over all of them, none with less than a tile for each warp
static int step_cluster(const cache4_attention_params& p) {
  const long long units = (long long)p.c.n_seqs * p.c.n_kv, per_warp = (p.max_len + ST_TILE - 1) / ST_TILE / ST_WARPS;
  int cs = 1;
  while (cs < 8 && units * cs < 2 * 148 && 2 * cs <= per_warp) cs *= 2;
  return cs;
}

int launch_attention_cache4_step(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream) {
  step_args a{p, (float*)workspace};
  const int cs = step_cluster(p);
  return dtype == OP_F16 ? launch_shape<__half>(a, cs, stream) : launch_shape<__nv_bfloat16>(a, cs, stream);
}

}  // namespace lcu
