// Attention of few rows over the 4-bit cache (cache4.cuh): single tokens, and a handful of rows (a draft that is checked).
//
//   s_jc = q_c . k_j / sqrt(head_dim),  o_c = sum_j e^(s_jc - max) v_j / sum_j e^(s_jc - max),   columns c = (row, head of the key/value head)
// What bounds it is the cache's bytes (at most 0.57 a value) and, close behind, the instructions that turn nibbles into halves: 41 values
// a cycle and SM arrive, and bit operations issue for 64 lanes a cycle.  So as little as possible happens to a value.  The cached rows are
// the wide side of m16n8k16 products (16 keys x 8 columns for the scores, 16 dimensions x 8 columns for the outputs), whose operands are
// made in registers:
//   keys: a masked nibble is a half already, the subnormal code * 2^-24 (or * 2^-20, four bits further up; those dimensions' queries
//     are a sixteenth).  The 7.5 is a product with the column's sum of queries, where the accumulator starts.  Where weights are wanted,
//     code - 7.5 is formed instead: the products' sums then cancel less, and weights are 1.2e-7 off (2-norm) instead of 8e-7, for 1 us of 58.
//   values: bits or'ed below an exponent are 1024 + code (or 64 + code); less the constant, times the scale, less 7.5 scales: exact.
// The order of the codes in a row (cache4.cuh) is such that a lane's words of 32 dimensions belong to one block of scales: scores are
// scaled in binary32 per block after the product, exactly; values take their scale as halves, exactly too (7-bit scales).
// Scores, sums and outputs are binary32; probabilities are rounded to half (2^-11) as operands.  The running maximum of a column is raised
// only when a score passes it by 8 (powers of two), and exponentials are formed against a reference 7 below it (cache4_attention.cuh).
//
// Work is dealt in chunks of 32 cached rows: those of all (sequence, key/value head, up to 16 columns) in a row, an equal run of them per
// CTA, whatever the lengths (which only the device knows).  A warp's chunks come through a ring of its own in shared memory, one
// on its way while the other is worked on.  Where a run ends inside a unit, sums go to the workspace and a second kernel joins them (and
// forms the weights, once the sums are known).
//
// A block of values whose scale is no number counts as zeros in the product, and the first such row is remembered per block: columns
// that see it get NaN there, columns of earlier rows of the same tile do not.
#include "cache4_attention.cuh"

#include <algorithm>
#include <type_traits>

namespace lcu {
namespace {

constexpr int ST_WARPS = 8, ST_THREADS = 32 * ST_WARPS, ST_TILE = 16, ST_CHUNK = 32, ST_STAGES = 3, ST_CTAS = 2 * 148;

struct step_args {
  cache4_attention_params p;
  int ctas, col_blocks;  // of the first kernel; units per (sequence, key/value head)
  int per_unit;          // CTAs of a unit, for a single sequence (0: chunks are dealt evenly, whatever the units)
  bool alone;            // short caches: a CTA per unit and nothing to join
  float* parts;          // [ctas][2][cols][hd] sums of runs that begin, or end, inside a unit
  float2* part_ml;       // [ctas][2][cols] their references (powers of two) and sums
  int* part_bad;         // [ctas][2][4] first row whose values of a block are no numbers
  float2* unit_ml;       // [units][cols] reference and sum of units that one CTA did (weights only)
  float* scores;         // [n_seqs * m][n_heads][max_len], powers of two (weights only)
};

// what both kernels know of the work: chunks of a sequence, places of units in the row of all chunks
// (fewer than 2^31 chunks: the host sees to it)
struct step_plan {
  unsigned total, ctas;  // chunks of all units; CTAs that have any of them: one at least each
  unsigned share, more;  // dealt evenly: chunks of a CTA, CTAs that have one more
  unsigned per_unit, of_unit;  // one sequence, shared unit by unit: CTAs and chunks of a unit (0: dealt evenly)
  __device__ __forceinline__ step_plan(unsigned sum_chunks, unsigned units_per_seq, const step_args& a) : total(sum_chunks * units_per_seq), per_unit(0), of_unit(sum_chunks) {
    if (a.per_unit && total) {
      per_unit = min((unsigned)a.per_unit, of_unit);
      ctas = per_unit * units_per_seq;
      share = more = 0u;
    } else {
      ctas = min((unsigned)a.ctas, total);
      share = ctas ? total / ctas : 0u;
      more = total - share * ctas;
    }
  }
  __device__ __forceinline__ static int chunks(const cache4_attention_params& p, int held) {
    const int room = min(p.c.ctx, p.max_len);
    return held < 0 ? 0 : ((held >= room ? room : min(held + p.m, room)) + ST_CHUNK - 1) / ST_CHUNK;  // (m is below 2^26, rooms too)
  }
  __device__ __forceinline__ unsigned first_of(unsigned cta) const {
    if (!per_unit) return cta * share + min(cta, more);
    const unsigned unit = cta / per_unit, k = cta - unit * per_unit;
    return unit * of_unit + (unsigned)((unsigned long long)k * of_unit / per_unit);
  }
  __device__ __forceinline__ unsigned cta_of(unsigned chunk) const {
    if (per_unit) {
      const unsigned unit = chunk / of_unit, at = chunk - unit * of_unit;
      return unit * per_unit + (unsigned)(((unsigned long long)(at + 1) * per_unit - 1) / of_unit);
    }
    const unsigned long_ones = more * (share + 1);
    return chunk < long_ones ? chunk / (share + 1) : more + (chunk - long_ones) / share;
  }
};
// chunks of the sequences before `seq` (per unit of a sequence), and of all; by a whole warp
__device__ __forceinline__ void count_chunks(const cache4_attention_params& p, int seq, unsigned& before, unsigned& all) {
  unsigned b = 0, n = 0;
  for (int s = threadIdx.x & 31; s < p.c.n_seqs; s += 32) {
    const unsigned c = step_plan::chunks(p, p.lengths[s]);
    n += c;
    b += s < seq ? c : 0;
  }
  all = __reduce_add_sync(0xffffffffu, n);
  before = __reduce_add_sync(0xffffffffu, b);
}

__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_word(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// (w & mask) | bits as one instruction (left to itself the compiler makes two, and moves, of many: 114 for 64 of a tile)
__device__ __forceinline__ uint32_t masked_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}
// (code - 7.5) * s for the nibbles i of both 16-bit halves of a word, i = 0 .. 3; c = -7.5 s
__device__ __forceinline__ void scaled_values(uint32_t w, __half2 s, __half2 c, uint32_t (&h)[4]) {
  const __half2 low = as_half2(0xe400e400u), high = as_half2(0xd400d400u);  // -1024, -64
  const uint32_t v = w >> 8;
  h[0] = as_word(__hfma2(__hadd2(as_half2(masked_or(w, 0x000f000fu, 0x64006400u)), low), s, c));
  h[1] = as_word(__hfma2(__hadd2(as_half2(masked_or(w, 0x00f000f0u, 0x54005400u)), high), s, c));
  h[2] = as_word(__hfma2(__hadd2(as_half2(masked_or(v, 0x000f000fu, 0x64006400u)), low), s, c));
  h[3] = as_word(__hfma2(__hadd2(as_half2(masked_or(v, 0x00f000f0u, 0x54005400u)), high), s, c));
}
// code - 7.5 for the same nibbles
__device__ __forceinline__ void centred(uint32_t w, uint32_t (&h)[4]) {
  const __half2 low = as_half2(0xe400e400u), middle = as_half2(0xc780c780u), high = as_half2(0xd478d478u);  // -1024, -7.5, -71.5
  const uint32_t v = w >> 8;
  h[0] = as_word(__hadd2(__hadd2(as_half2(masked_or(w, 0x000f000fu, 0x64006400u)), low), middle));
  h[1] = as_word(__hadd2(as_half2(masked_or(w, 0x00f000f0u, 0x54005400u)), high));
  h[2] = as_word(__hadd2(__hadd2(as_half2(masked_or(v, 0x000f000fu, 0x64006400u)), low), middle));
  h[3] = as_word(__hadd2(as_half2(masked_or(v, 0x00f000f0u, 0x54005400u)), high));
}
// code * 2^-24 and code * 2^-20 in turn: the masked bits as they are
__device__ __forceinline__ void bare(uint32_t w, uint32_t (&h)[4]) {
  h[0] = w & 0x000f000fu;
  h[1] = w & 0x00f000f0u;
  h[2] = (w >> 8) & 0x000f000fu;
  h[3] = (w >> 8) & 0x00f000f0u;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // an 8 x 8 tile of halves, two neighbours of a row per lane
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ __half half_of(uint32_t v, int hi) { return __ushort_as_half((unsigned short)(hi ? v >> 16 : v & 0xffff)); }

__device__ __forceinline__ void mma_16816_onto(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
template <int N>
__device__ __forceinline__ void shared_words(uint32_t (&r)[N], uint32_t at) {
  if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
  else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at));
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(at));
}
template <int BYTES>
__device__ __forceinline__ void cp_async_part(uint32_t dst, const void* src, int there) {  // (the rest is zeros)
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there) : "memory");
}
__device__ __forceinline__ uint32_t shared_half(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}
// keys' codes, values' codes and both kinds of scales of a chunk (scales with 16 bytes to spare: see send)
template <int HD, int NB>
struct step_ring {
  static constexpr uint32_t ROW = HD / 2, PLANE = ST_CHUNK * ROW, SCALES = ST_CHUNK * 2 * NB + 16, STAGE = 2 * PLANE + 2 * SCALES;
};

template <typename T, int HD, int NB, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(ST_THREADS, NT == 1 ? 2 : 1) attention_step_kernel(const step_args a) {
  constexpr int G = HD / 32, VW = HD / 64, BG = G / NB;  // groups of 32 dimensions, of a block; words of a value's row in a lane
  constexpr bool TWO = HD == 128 && NB == 4;                // a lane's two value words lie in two blocks
  constexpr int COLS = 8 * NT, ROW = HD / 2, CPR = ROW / 16;
  using ring_t = step_ring<HD, NB>;
  constexpr uint32_t PLANE = ring_t::PLANE, SCALES = ring_t::SCALES, STAGE = ring_t::STAGE;
  extern __shared__ __align__(128) uint8_t s_raw[];         // rings of the warps; then their sums, in the order of the accumulators' registers
  float2* s_o = reinterpret_cast<float2*>(s_raw);
  __shared__ float2 s_ml[ST_WARPS][COLS];
  __shared__ int s_bad[4];
  __shared__ uint4 s_q[NT][G][32];                          // queries as operands, made by a warp each
  __shared__ float s_most[NT][G][8], s_sum[NT][G][8], s_f[COLS];
  const cache4_attention_params& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / p.c.n_kv, n_cols = p.m * group, per_seq = p.c.n_kv * a.col_blocks;
  pdl_launch_dependents();
  const int bound = min(p.c.ctx, p.max_len);
  unsigned at, end;
  int seq = 0;
  unsigned seq_at = 0;                       // the sequence's first chunk
  if (a.alone) {
    seq = blockIdx.x / per_seq;
    const int unit_in_seq = blockIdx.x - seq * per_seq, chunks = step_plan::chunks(p, p.lengths[seq]);
    if (chunks == 0) {
      const int kvh = unit_in_seq / a.col_blocks, c0 = unit_in_seq % a.col_blocks * COLS, here = min(COLS, n_cols - c0);
      for (int e = tid; e < here * (HD / 2); e += ST_THREADS) {
        const int c = c0 + e / (HD / 2);
        reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + ((size_t)seq * p.m + c / group) * p.ld_out + (kvh * group + c % group) * HD)[e % (HD / 2)] = 0u;
      }
      return;
    }
    at = (unsigned)(unit_in_seq * chunks);
    end = at + chunks;
  } else {
    unsigned before, sum_chunks;
    count_chunks(p, 0, before, sum_chunks);
    const step_plan plan(sum_chunks, per_seq, a);
    if (blockIdx.x >= plan.ctas) return;
    at = plan.first_of(blockIdx.x);
    end = plan.first_of(blockIdx.x + 1);
  }
  // tile row r stands for key perm(r): rows 2t, 2t+1, 2t+8, 2t+9, whose probabilities a lane multiplies with values, are keys 4t .. 4t+3
  const int key_a = 4 * (g >> 1) + (g & 1);  // rows g and g + 8: keys key_a and key_a + 2
  const uint32_t ring = smem_u32(s_raw) + warp * (ST_STAGES * STAGE);
  const int v_block = (g * VW % G) / BG;     // the (first) block of this lane's values
  // places in the ring: of this lane's pieces of a chunk's values (exchanged within 128 bytes, so that the lanes of one load, in rows four
  // apart, meet different banks), of its words
  const uint32_t to_v0 = (uint32_t)(lane ^ (((lane / (4 * CPR)) & 3) << 1)) * 16, to_v1 = (uint32_t)(lane ^ (((32 / (4 * CPR) + lane / (4 * CPR)) & 3) << 1)) * 16;
  auto word_at = [&](int i) { return (uint32_t)((((4 * t + i) * CPR + g * (4 * VW) / 16) ^ (t << 1)) * 16 + g * (4 * VW) % 16); };
  const uint32_t from_v0 = word_at(0), from_v1 = word_at(1), from_v2 = word_at(2), from_v3 = word_at(3);
  const uint32_t from_k = (uint32_t)(key_a * ROW + t * (4 * G));

  while (at < end) {
    // ---- the unit that chunk `at` belongs to
    int held = p.lengths[seq], chunks = step_plan::chunks(p, held);
    while (at >= seq_at + chunks * per_seq) {
      seq_at += chunks * per_seq;
      held = p.lengths[++seq];
      chunks = step_plan::chunks(p, held);
    }
    const int unit_in_seq = (int)((at - seq_at) / (unsigned)chunks);
    const int kvh = (unsigned)unit_in_seq / (unsigned)a.col_blocks, c0 = (unit_in_seq - kvh * a.col_blocks) * COLS;
    const unsigned unit_at = seq_at + (unsigned)(unit_in_seq * chunks);
    const int lo = (int)(at - unit_at), hi = min(chunks, (int)(end - unit_at));
    auto limit_of = [&](int c) { return c < n_cols ? (held >= bound ? bound : min(held + c / group + 1, bound)) : 0; };
    auto row_of = [&](int c) { return (size_t)seq * p.m + c / group; };
    auto head_of = [&](int c) { return kvh * group + c % group; };
    const int T_all = limit_of(n_cols - 1), T_first = limit_of(0);
    const size_t head_rows = ((size_t)seq * p.c.n_kv + kvh) * p.c.ctx;
    const uint8_t* k_codes = p.c.k_codes + head_rows * ROW;
    const uint8_t* v_codes = p.c.v_codes + head_rows * ROW;
    const uint8_t* k_scales = reinterpret_cast<const uint8_t*>(p.c.k_scales + head_rows * NB);
    const uint8_t* v_scales = reinterpret_cast<const uint8_t*>(p.c.v_scales + head_rows * NB);
    // (with one block a head's scales may start between two words: they are copied from the word they start in)
    const uint32_t skew = NB == 1 ? (uint32_t)(head_rows & 1) * 2 : 0u;
    const long long s_left = (long long)((size_t)p.c.n_seqs * p.c.n_kv * p.c.ctx - head_rows) * 2;  // (one block) bytes to the planes' end

    // a chunk's codes and scales to the ring; rows behind the last one are the last one again
    auto send = [&](int chunk, uint32_t to) {
      const size_t first = (size_t)(chunk * ST_CHUNK) * ROW + lane * 16;
      const uint8_t *k_at = k_codes + first, *v_at = v_codes + first;
      if (chunk * ST_CHUNK + ST_CHUNK <= T_all) {
#pragma unroll
        for (int i = 0; i < CPR; ++i) {
          cp_async16(to + lane * 16 + i * 512, k_at + i * 512);
          cp_async16(to + PLANE + (i & 1 ? to_v1 : to_v0) + i * 512, v_at + i * 512);
        }
      } else {
#pragma unroll
        for (int i = 0; i < CPR; ++i) {
          const int back = max(0, chunk * ST_CHUNK + (i * 32 + lane) / CPR - (T_all - 1)) * ROW;
          cp_async16(to + lane * 16 + i * 512, k_at + i * 512 - back);
          cp_async16(to + PLANE + (i & 1 ? to_v1 : to_v0) + i * 512, v_at + i * 512 - back);
        }
      }
      // scales in words: a row's, or (one block) those that hold a row that is seen; none is read past the end of its plane
      constexpr int UNIT = NB == 4 ? 8 : 4, UNITS = ST_CHUNK * 2 * NB / UNIT + (NB == 1);
      const int byte = chunk * (ST_CHUNK * 2 * NB) + lane * UNIT - (int)skew;
      if (lane < UNITS && byte < T_all * (2 * NB)) {
        const int there = NB == 1 ? (int)min((long long)UNIT, s_left - byte) : UNIT;
        cp_async_part<UNIT>(to + 2 * PLANE + lane * UNIT, k_scales + byte, there);
        cp_async_part<UNIT>(to + 2 * PLANE + SCALES + lane * UNIT, v_scales + byte, there);
      }
      cp_async_commit();
    };
    int chunk = lo + warp;
    uint32_t stage = ring;
    if (chunk < hi) {
      send(chunk, stage);
      if (chunk + ST_WARPS < hi) send(chunk + ST_WARPS, stage + STAGE);
      else cp_async_commit();
    }

    // ---- queries as the narrow operand: column g of each n-tile, octet t of every 32 dimensions, in the codes' order of pairs.  A warp makes
    // those of 32 dimensions.  A power of two takes the column's largest magnitude into [2^14, 2^15): halves, and their sixteenths,
    // are exact from 2^-24 of it on.
    {
      const int n = warp / G, gd = warp % G, c = c0 + n * 8 + g;
      float x[8];
      if (n < NT) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < n_cols) v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + row_of(c) * p.ld_q + head_of(c) * HD + gd * 32 + t * 8);
        unpack8<T>(v, x);
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (t == 0) s_most[n][gd][g] = most;
      }
      __syncthreads();
      if (n < NT) {
        float most = s_most[n][0][g];
#pragma unroll
        for (int k = 1; k < G; ++k) most = fmaxf(most, s_most[n][k][g]);
        float up = 1.f, down = 1.f;
        const int ex = (int)(__float_as_uint(most) >> 23);
        if (ex >= 20 && ex <= 230) {  // (what is smaller than 2^-107 gives scores of nothing as it is, what is larger than 2^103 infinities)
          up = __uint_as_float((uint32_t)(127 + 14 + 127 - ex) << 23);
          down = __uint_as_float((uint32_t)(ex - 14) << 23);
        }
        float total = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= up;
          total += x[e];
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float m = i & 1 && !WEIGHTS ? 0.0625f : 1.f;
          w[i] = pack2<__half>(x[i] * m, x[i + 4] * m);
        }
        s_q[n][gd][lane] = make_uint4(w[0], w[1], w[2], w[3]);
        total += __shfl_xor_sync(0xffffffffu, total, 1);
        total += __shfl_xor_sync(0xffffffffu, total, 2);
        if (t == 0) {
          s_sum[n][gd][g] = total;
          if (gd == 0) s_f[n * 8 + g] = down * ((WEIGHTS ? 1.f : 16777216.f) * 1.4426950408889634f * rsqrtf((float)HD));
        }
      }
      __syncthreads();
    }
    uint32_t qf[NT][G][4];
    float f[NT][2], start[NT][NB][2];
    float* at_score[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int gd = 0; gd < G; ++gd) {
        const uint4 v = s_q[n][gd][lane];
        qf[n][gd][0] = v.x;
        qf[n][gd][1] = v.y;
        qf[n][gd][2] = v.z;
        qf[n][gd][3] = v.w;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 2 * t + e;
        f[n][e] = s_f[n * 8 + col];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float total = 0.f;
#pragma unroll
          for (int k = 0; k < BG; ++k) total += s_sum[n][b * BG + k][col];
          start[n][b][e] = WEIGHTS ? 0.f : total * (-7.5f / 16777216.f);
        }
        if constexpr (WEIGHTS) {
          const int cc = min(c0 + n * 8 + col, n_cols - 1);
          at_score[n][e] = a.scores + (row_of(cc) * p.n_heads + head_of(cc)) * p.max_len;
        }
      }
    }

    // less: minus the reference (0 while there is none); high: 8 above the maximum, as the products give scores (minus infinity while there is none)
    float o[NT][VW * 4][4], less[NT][2], high[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < VW * 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        less[n][e] = 0.f;
        high[n][e] = -INFINITY;
        sum[n][e] = 0.f;
      }
    }
    int bad0 = 0x7fffffff, bad1 = 0x7fffffff;
    if (tid < 4) s_bad[tid] = 0x7fffffff;

    for (; chunk < hi; chunk += ST_WARPS) {
      if (chunk + 2 * ST_WARPS < hi) send(chunk + 2 * ST_WARPS, stage == ring ? ring + 2 * STAGE : stage - STAGE);  // (its readers have passed the __syncwarp below)
      else cp_async_commit();
      cp_async_wait<2>();
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j0 = chunk * ST_CHUNK + u * ST_TILE;
        uint32_t ks[2][NB == 4 ? 2 : 1], vs[4];
        uint32_t k0[G], k1[G], vw0[VW], vw1[VW], vw2[VW], vw3[VW];
        {
          const uint32_t tile_at = stage + u * ST_TILE * ROW;
          shared_words<G>(k0, tile_at + from_k);
          shared_words<G>(k1, tile_at + from_k + 2 * ROW);
          shared_words<VW>(vw0, tile_at + PLANE + from_v0);
          shared_words<VW>(vw1, tile_at + PLANE + from_v1);
          shared_words<VW>(vw2, tile_at + PLANE + from_v2);
          shared_words<VW>(vw3, tile_at + PLANE + from_v3);
          const uint32_t ks_at = stage + 2 * PLANE + (u * ST_TILE + key_a) * (2 * NB) + skew;
          const uint32_t vs_at = stage + 2 * PLANE + SCALES + (u * ST_TILE + 4 * t) * (2 * NB) + v_block * 2 + skew;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (NB == 1) ks[r][0] = shared_half(ks_at + 2 * r * (2 * NB));
            else shared_words<NB / 2>(ks[r], ks_at + 2 * r * (2 * NB));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (TWO) {
              uint32_t w[1];
              shared_words<1>(w, vs_at + i * (2 * NB));
              vs[i] = w[0];
            } else {
              vs[i] = shared_half(vs_at + i * (2 * NB));
            }
          }
        }
        // ---- scores
        float s[NT][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float acc[NT][4];
#pragma unroll
          for (int gb = 0; gb < BG; ++gb) {
            const int gd = b * BG + gb;
            uint32_t ka[4], kb[4];  // pairs of dimensions in the queries' order
            if constexpr (WEIGHTS) {
              centred(k0[gd], ka);
              centred(k1[gd], kb);
            } else {
              bare(k0[gd], ka);
              bare(k1[gd], kb);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (gb == 0) mma_16816_onto(acc[n], ka[0], kb[0], ka[1], kb[1], qf[n][gd][0], qf[n][gd][1], start[n][b][0], start[n][b][1]);
              else mma_16816(acc[n], ka[0], kb[0], ka[1], kb[1], qf[n][gd][0], qf[n][gd][1]);
              mma_16816(acc[n], ka[2], kb[2], ka[3], kb[3], qf[n][gd][2], qf[n][gd][3]);
            }
          }
          const float sa = __half2float(half_of(ks[0][b >> 1], b & 1)), sb = __half2float(half_of(ks[1][b >> 1], b & 1));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[n][0] = b ? fmaf(sa, acc[n][0], s[n][0]) : sa * acc[n][0];
            s[n][1] = b ? fmaf(sa, acc[n][1], s[n][1]) : sa * acc[n][1];
            s[n][2] = b ? fmaf(sb, acc[n][2], s[n][2]) : sb * acc[n][2];
            s[n][3] = b ? fmaf(sb, acc[n][3], s[n][3]) : sb * acc[n][3];
          }
        }
        bool raise = false;
        const bool ragged = j0 + ST_TILE > T_first;  // of the last rows some columns see fewer, and the tile may hang over the end
        if (ragged) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int limit = limit_of(c0 + n * 8 + 2 * t + e);
              if (j0 + key_a >= limit) s[n][e] = -INFINITY;
              if (j0 + key_a + 2 >= limit) s[n][e + 2] = -INFINITY;
            }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + 4 * t + i >= T_all) vs[i] = 0u;
        }
        if constexpr (WEIGHTS) {  // (a column's rows that it does not see: minus infinity, read by nobody)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + key_a + (e & 2);
              if (c0 + n * 8 + 2 * t + (e & 1) < n_cols && (!ragged || j < T_all)) at_score[n][e & 1][j] = s[n][e] * f[n][e & 1];
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) raise |= fmaxf(s[n][0], s[n][2]) > high[n][0] || fmaxf(s[n][1], s[n][3]) > high[n][1];
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
              k[e] = 1.f;
              if (top > high[n][e]) {
                const float now = top * f[n][e], reference = reference_of(now);
                k[e] = high[n][e] == -INFINITY ? 0.f : ex2(-less[n][e] - reference);
                less[n][e] = -reference;
                high[n][e] = (now + 8.f) / f[n][e];
              }
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
          const float e0 = ex2(fmaf(s[n][0], f[n][0], less[n][0])), e1 = ex2(fmaf(s[n][1], f[n][1], less[n][1]));
          const float e2 = ex2(fmaf(s[n][2], f[n][0], less[n][0])), e3 = ex2(fmaf(s[n][3], f[n][1], less[n][1]));
          sum[n][0] += e0 + e2;
          sum[n][1] += e1 + e3;
          pf[n][0] = transposed(pack2<__half>(e0, e1));
          pf[n][1] = transposed(pack2<__half>(e2, e3));
        }
        // ---- values
        {
          const __half2 z = __hadd2(__hadd2(as_half2(vs[0]), as_half2(vs[1])), __hadd2(as_half2(vs[2]), as_half2(vs[3])));  // (up to 4 x 8704: finite)
          if (__hisnan(__hadd(__low2half(z), __high2half(z)))) {
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
          const __half2 s01 = as_half2(__byte_perm(vs[0], vs[1], pick)), s23 = as_half2(__byte_perm(vs[2], vs[3], pick));
          const __half2 minus = as_half2(0xc780c780u);  // -7.5
          const __half2 c01 = __hmul2(s01, minus), c23 = __hmul2(s23, minus);
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            uint32_t h01[4], h23[4];
            scaled_values(__byte_perm(vw0[vw], vw1[vw], hh ? 0x7632 : 0x5410), s01, c01, h01);
            scaled_values(__byte_perm(vw2[vw], vw3[vw], hh ? 0x7632 : 0x5410), s23, c23, h23);
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma_16816(o[n][vw * 4 + hh * 2 + mm], h01[2 * mm], h01[2 * mm + 1], h23[2 * mm], h23[2 * mm + 1], pf[n][0], pf[n][1]);
          }
        }
      }
      __syncwarp();
      stage = stage == ring + 2 * STAGE ? ring : stage + STAGE;
    }

    // ---- the warps meet
    const int here = min(COLS, n_cols - c0);
    __syncthreads();  // (the rings are read; s_bad is set)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[n][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) s_ml[warp][n * 8 + 2 * t + e] = make_float2(high[n][e] == -INFINITY ? -INFINITY : -less[n][e], l);
#pragma unroll
        for (int i = 0; i < VW * 4; ++i) s_o[(((warp * NT + n) * (VW * 4) + i) * 2 + e) * 32 + lane] = make_float2(o[n][i][e], o[n][i][e + 2]);
      }
    }
    if (bad0 != 0x7fffffff) atomicMin(&s_bad[v_block], bad0);
    if (bad1 != 0x7fffffff) atomicMin(&s_bad[v_block + 1], bad1);
    __syncthreads();
    const bool whole = lo == 0 && hi == chunks;
    const size_t slot = (size_t)blockIdx.x * 2 + (lo == 0);
    for (int e = tid; e < NT * VW * 256; e += ST_THREADS) {
      const int word = (e & 31) / 4 * VW + (e >> 6) % (VW * 4) / 4, c = (e >> 6) / (VW * 4) * 8 + 2 * (e & 3) + (e >> 5 & 1);
      const int d = (word % G) * 32 + (word / G) * 8 + (e >> 6) % 4 * 2;  // (register e >> 5 of lane e & 31)
      if (c >= here) continue;
      float top = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < ST_WARPS; ++w) top = fmaxf(top, s_ml[w][c].x);
#pragma unroll
      for (int w = 0; w < ST_WARPS; ++w) {
        const float2 ml = s_ml[w][c];
        const float k = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);  // (a reference of nothing: sums of 0, or of NaN)
        const float2 v = s_o[w * (NT * VW * 256) + e];
        l += ml.y * k;
        x += v.x * k;
        y += v.y * k;
      }
      if (whole) {
        const float rl = s_bad[d * NB / HD] < limit_of(c0 + c) ? __int_as_float(0x7fffffff) : 1.f / l;
        reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + row_of(c0 + c) * p.ld_out + head_of(c0 + c) * HD)[d / 2] = pack2<T>(x * rl, y * rl);
        if (WEIGHTS && d == 0) a.unit_ml[((size_t)seq * per_seq + unit_in_seq) * COLS + c] = make_float2(top, l);
      } else {
        *reinterpret_cast<float2*>(&a.parts[(slot * COLS + c) * HD + d]) = make_float2(x, y);
        if (d == 0) a.part_ml[slot * COLS + c] = make_float2(top, l);
      }
    }
    if (!whole && tid < 4) a.part_bad[slot * 4 + tid] = s_bad[tid];
    if constexpr (WEIGHTS) {
      if (a.alone && a.col_blocks == 1) {  // every lane reads the scores that it wrote
        float fin[NT][2], rl[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = n * 8 + 2 * t + e;
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < ST_WARPS; ++w) top = fmaxf(top, s_ml[w][c].x);
#pragma unroll
            for (int w = 0; w < ST_WARPS; ++w) l += s_ml[w][c].y * (s_ml[w][c].x == -INFINITY ? 1.f : ex2(s_ml[w][c].x - top));
            fin[n][e] = top + LIFT;
            rl[n][e] = LIFT_FACTOR / l;
          }
        for (int u = 2 * (lo + warp); u < 2 * hi; u += u & 1 ? 2 * ST_WARPS - 1 : 1) {
          float add[2] = {0.f, 0.f};
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int c = n * 8 + 2 * t + (e & 1), j = u * ST_TILE + key_a + (e & 2);
              if (j < limit_of(c)) add[e >> 1] += ex2(at_score[n][e & 1][j] - fin[n][e & 1]) * rl[n][e & 1];
            }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            add[r] += __shfl_xor_sync(0xffffffffu, add[r], 1);
            add[r] += __shfl_xor_sync(0xffffffffu, add[r], 2);
            const int j = u * ST_TILE + key_a + 2 * r;
            if (t == 0 && j < T_all) {
              float* to = p.weights + head_rows + j;
              *to = p.beta == 0.f || j >= held ? add[r] : fmaf(p.beta, *to, add[r]);
            }
          }
        }
      }
    }
    __syncthreads();  // (the rings are free)
    at = unit_at + hi;
  }
}

// Joins the sums of units that several CTAs did (and gives zeros for sequences not in use): a CTA per unit and column; and behind those, with
// weights, a CTA per (sequence, key/value head, 512 rows), which finds maxima and sums of all columns and adds the probabilities in
// their order.  Up to 296 CTAs may have worked on a unit: their maxima are read side by side, their sums by several groups of threads.
constexpr int JOIN_THREADS = 128, JOIN_KEYS = 4 * JOIN_THREADS;
template <typename T, int HD, int NB, int NT>
__global__ void __launch_bounds__(JOIN_THREADS) attention_join_kernel(const step_args a) {
  constexpr int COLS = 8 * NT, LANES = HD / 2, GROUPS = JOIN_THREADS / LANES;
  __shared__ float s_k[ST_CTAS];
  __shared__ float2 s_part[GROUPS][LANES];
  __shared__ float s_warp[JOIN_THREADS / 32];
  const cache4_attention_params& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, group = p.n_heads / p.c.n_kv, n_cols = p.m * group, per_seq = p.c.n_kv * a.col_blocks;
  const int joins = p.c.n_seqs * per_seq * COLS;
  const int key_blocks = (p.max_len + JOIN_KEYS - 1) / JOIN_KEYS;
  const bool join = (int)blockIdx.x < joins;
  const int sh = join ? 0 : ((int)blockIdx.x - joins) / key_blocks;
  const int seq = join ? (int)blockIdx.x / (per_seq * COLS) : sh / p.c.n_kv;
  // Lengths are read ahead of the wait (0.4 to 0.8 us: 8 rows behind 8000 18.0 us, 18.6 behind it).  That rests on the kernel in front, which does not
  // write them and is launched without the attribute (launch_step): whatever wrote them is done.  Nothing else is touched before the wait.
  const int held = p.lengths[seq], chunks = step_plan::chunks(p, held);
  if (!join && held < 0) return;
  unsigned before, sum_chunks;
  count_chunks(p, seq, before, sum_chunks);
  const step_plan plan(sum_chunks, per_seq, a);
  pdl_wait();
  auto row_of = [&](int c) { return (size_t)seq * p.m + c / group; };
  auto ctas_of = [&](int unit_in_seq) {
    const unsigned unit_at = before * per_seq + (unsigned)(unit_in_seq * chunks);
    return make_int2((int)plan.cta_of(unit_at), (int)plan.cta_of(unit_at + chunks - 1));
  };
  auto part_of = [&](int cta, int first, int c) { return a.part_ml[((size_t)cta * 2 + (cta == first)) * COLS + c]; };
  if (join) {
    const int c = blockIdx.x % COLS, unit_in_seq = (int)(blockIdx.x / COLS) % per_seq, kvh = unit_in_seq / a.col_blocks, cc = unit_in_seq % a.col_blocks * COLS + c;
    if (cc >= n_cols) return;
    uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + row_of(cc) * p.ld_out + (kvh * group + cc % group) * HD);
    if (held < 0) {
      if (tid < LANES) out[tid] = 0u;
      return;
    }
    const int2 ctas = a.alone ? make_int2(0, 0) : ctas_of(unit_in_seq);
    if (a.alone || ctas.x == ctas.y) return;
    float top = -INFINITY, l = 0.f;
    for (int b = ctas.x + tid; b <= ctas.y; b += JOIN_THREADS) {
      s_k[b - ctas.x] = part_of(b, ctas.x, c).x;
      top = fmaxf(top, s_k[b - ctas.x]);
    }
    top = warp_max(top);
    if (lane == 0) s_warp[tid >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_warp[0], s_warp[1]), fmaxf(s_warp[2], s_warp[3]));
    for (int b = ctas.x + tid; b <= ctas.y; b += JOIN_THREADS) s_k[b - ctas.x] = s_k[b - ctas.x] == -INFINITY ? 1.f : ex2(s_k[b - ctas.x] - top);  // (a reference of nothing: sums of 0, or of NaN)
    __syncthreads();
    const int pair = tid % LANES, of = tid / LANES;
    float x = 0.f, y = 0.f;
    int bad = 0x7fffffff;
#pragma unroll 4
    for (int b = ctas.x + of; b <= ctas.y; b += GROUPS) {
      const size_t slot = (size_t)b * 2 + (b == ctas.x);
      const float k = s_k[b - ctas.x];
      const float2 v = *reinterpret_cast<const float2*>(&a.parts[(slot * COLS + c) * HD + 2 * pair]);
      l += a.part_ml[slot * COLS + c].y * k;
      x += v.x * k;
      y += v.y * k;
      bad = min(bad, a.part_bad[slot * 4 + 2 * pair * NB / HD]);
    }
    s_part[of][pair] = make_float2(x, y);
    __shared__ float s_l[GROUPS];
    __shared__ int s_bad[4];
    if (tid < 4) s_bad[tid] = 0x7fffffff;
    if (pair == 0) s_l[of] = l;
    __syncthreads();
    if (bad != 0x7fffffff) atomicMin(&s_bad[2 * pair * NB / HD], bad);
    __syncthreads();
    if (tid >= LANES) return;
    x = y = l = 0.f;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      x += s_part[k][pair].x;
      y += s_part[k][pair].y;
      l += s_l[k];
    }
    const int bound = min(p.c.ctx, p.max_len), limit = held >= bound ? bound : min(held + cc / group + 1, bound);
    const float rl = s_bad[2 * pair * NB / HD] < limit ? __int_as_float(0x7fffffff) : 1.f / l;
    out[pair] = pack2<T>(x * rl, y * rl);
    return;
  }
  // ---- weights
  __shared__ float2 s_fin[64];
  const int kvh = sh % p.c.n_kv, j0 = (((int)blockIdx.x - joins) % key_blocks) * JOIN_KEYS, bound = min(p.c.ctx, p.max_len);
  const int T_all = held >= bound ? bound : min(held + p.m, bound);
  if (j0 >= T_all) return;
  float w[JOIN_KEYS / JOIN_THREADS] = {};
  for (int c64 = 0; c64 < n_cols; c64 += 64) {
    __syncthreads();
    for (int c = c64 + (tid >> 5); c < min(n_cols, c64 + 64); c += JOIN_THREADS / 32) {  // a column per warp
      const int unit_in_seq = kvh * a.col_blocks + c / COLS;
      const int2 ctas = a.alone ? make_int2(0, 0) : ctas_of(unit_in_seq);
      float2 all;
      if (ctas.x == ctas.y) {
        all = a.unit_ml[((size_t)seq * per_seq + unit_in_seq) * COLS + c % COLS];
      } else {
        all = make_float2(-INFINITY, 0.f);
        for (int b = ctas.x + lane; b <= ctas.y; b += 32) all.x = fmaxf(all.x, part_of(b, ctas.x, c % COLS).x);
        all.x = warp_max(all.x);
        for (int b = ctas.x + lane; b <= ctas.y; b += 32) {
          const float2 ml = part_of(b, ctas.x, c % COLS);
          all.y += ml.y * (ml.x == -INFINITY ? 1.f : ex2(ml.x - all.x));
        }
        all.y = warp_sum(all.y);
      }
      if (lane == 0) s_fin[c - c64] = make_float2(all.x + LIFT, LIFT_FACTOR / all.y);  // (maximum, and the sum's inverse against it)
    }
    __syncthreads();
    for (int c = c64; c < min(n_cols, c64 + 64); ++c) {
      const float* scores = a.scores + (row_of(c) * p.n_heads + kvh * group + c % group) * p.max_len;
      const int limit = held >= bound ? bound : min(held + c / group + 1, bound);
      const float2 fin = s_fin[c - c64];
#pragma unroll
      for (int i = 0; i < JOIN_KEYS / JOIN_THREADS; ++i) {
        const int j = j0 + i * JOIN_THREADS + tid;
        if (j < limit) w[i] += ex2(scores[j] - fin.x) * fin.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < JOIN_KEYS / JOIN_THREADS; ++i) {
    const int j = j0 + i * JOIN_THREADS + tid;
    if (j < T_all) {
      float* to = p.weights + (size_t)sh * p.c.ctx + j;
      *to = p.beta == 0.f || j >= held ? w[i] : fmaf(p.beta, *to, w[i]);
    }
  }
}

// the work as the host knows it: units, and CTAs - one per unit, or as many as find a chunk for each of their warps if sequences are as
// long as they may be, up to two per SM (one with 16 columns, whose accumulators take the registers)
struct step_shape {
  int cols, col_blocks, ctas, per_unit;
  bool alone;
  long long units;
  step_shape(int n_seqs, int m, int n_heads, int n_kv, int max_len, bool weights) {
    const int n_cols = m * (n_heads / n_kv);
    cols = n_cols <= 8 ? 8 : 16;
    col_blocks = (n_cols + cols - 1) / cols;
    units = (long long)n_seqs * n_kv * col_blocks;
    const long long chunks = units * ((max_len + ST_CHUNK - 1) / ST_CHUNK);
    const long long most = ST_CTAS / (cols / 8);
    ctas = (int)std::min(most, std::max(units, (chunks + ST_WARPS - 1) / ST_WARPS));
    // One sequence's units are equally long.  A CTA that goes on to another unit starts over (about 4 us), so each is given whole CTAs where
    // that idles few: from six per unit on (one sixth of a unit more at most: 32 heads x 32000 rows 47.2 -> 44.8 us), or where
    // every warp has one chunk anyway.
    const long long each = units > 0 && units <= most ? std::min(most / units, std::max(1ll, (chunks / units + ST_WARPS - 1) / ST_WARPS)) : 0;
    per_unit = n_seqs == 1 && (each >= 6 || (each && each * ST_WARPS * units >= chunks)) ? (int)each : 0;
    if (per_unit) ctas = (int)(per_unit * units);
    // Short caches: a CTA per unit, one launch.  Its rounds of eight chunks (1.5 us each) against the even deal's other overheads, which grow
    // with the units; the weights' second look at the scores costs as much again.  Alone / shared, us: 32 units x 400 rows 7.9 / 9.0,
    // 600 8.9 / 9.4, 650 to 720 a tie at 9.5 (one launch less for the host), 770 10.6 / 9.6, 1000 11.3 / 9.7; 64 x 1000 11.3 / 15.2, 1300 13.6 / 14.9,
    // 2000 16.3 / 16.7; 512 x 3000 52 / 63; with weights 32 x 250 8.9 / 9.6, 300 11.1 / 9.8; 64 x 500 12.1 / 14.0; 512 x 1000 42 / 45.
    alone = chunks / units <= (weights ? 8 * std::min(4ll, std::max(1ll, units / 32)) : 22 * std::min(8ll, std::max(1ll, units / 32)));
    if (alone) {
      per_unit = 0;
      ctas = (int)units;
    }
  }
};

template <typename T, int HD, int NB, int NT, bool WEIGHTS>
int launch_step(const step_args& a, cudaStream_t stream) {
  constexpr size_t RING = (size_t)ST_WARPS * ST_STAGES * step_ring<HD, NB>::STAGE, SUMS = (size_t)ST_WARPS * 8 * NT * HD * sizeof(float);
  constexpr size_t SMEM = RING > SUMS ? RING : SUMS;
  auto* kernel = attention_step_kernel<T, HD, NB, NT, WEIGHTS>;
  static bool attr_done[16] = {};
  int dev = 0;
  LCU_CUDA(cudaGetDevice(&dev));
  if (dev >= 16 || !attr_done[dev]) {
    LCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    if (dev < 16) attr_done[dev] = true;
  }
  kernel<<<a.ctas, ST_THREADS, SMEM, stream>>>(a);  // (behind everything: attention_join_kernel reads lengths without waiting for it)
  if (a.alone && (!WEIGHTS || a.col_blocks == 1)) {
    LCU_CUDA(cudaGetLastError());
    return LCU_OK;
  }
  const long long joins = (long long)a.p.c.n_seqs * a.p.c.n_kv * a.col_blocks * 8 * NT;
  const long long blocks = joins + (WEIGHTS ? (long long)a.p.c.n_seqs * a.p.c.n_kv * ((a.p.max_len + JOIN_KEYS - 1) / JOIN_KEYS) : 0);
  LCU_CUDA(launch_after(attention_join_kernel<T, HD, NB, NT>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, stream, a));
  return LCU_OK;
}

template <typename T, int HD, int NB>
int launch_cols(const step_args& a, int cols, cudaStream_t stream) {
  if (a.p.weights) return cols == 8 ? launch_step<T, HD, NB, 1, true>(a, stream) : launch_step<T, HD, NB, 2, true>(a, stream);
  return cols == 8 ? launch_step<T, HD, NB, 1, false>(a, stream) : launch_step<T, HD, NB, 2, false>(a, stream);
}

template <typename T>
int launch_shape(const step_args& a, int cols, cudaStream_t stream) {
  const int nb = a.p.c.hd / a.p.c.bs;
  if (a.p.c.hd == 128) {
    if (nb == 4) return launch_cols<T, 128, 4>(a, cols, stream);
    if (nb == 2) return launch_cols<T, 128, 2>(a, cols, stream);
    return launch_cols<T, 128, 1>(a, cols, stream);
  }
  if (nb == 2) return launch_cols<T, 64, 2>(a, cols, stream);
  return launch_cols<T, 64, 1>(a, cols, stream);
}

// the workspace's parts, each 16-byte aligned
size_t step_layout(step_args* a, void* workspace, const step_shape& w, int n_seqs, int m, int n_heads, int hd, int max_len, bool weights) {
  size_t used = 0;
  auto take = [&](size_t bytes) {
    const size_t at = used;
    used += round_up(bytes, 16);
    return (uint8_t*)workspace + at;
  };
  const size_t slots = w.alone ? 0 : (size_t)w.ctas * 2;  // (one CTA per unit leaves no parts)
  uint8_t* parts = take(slots * w.cols * hd * sizeof(float));
  uint8_t* part_ml = take(slots * w.cols * sizeof(float2));
  uint8_t* part_bad = take(slots * 4 * sizeof(int));
  uint8_t* unit_ml = weights ? take((size_t)w.units * w.cols * sizeof(float2)) : nullptr;
  uint8_t* scores = weights ? take((size_t)n_seqs * m * n_heads * max_len * sizeof(float)) : nullptr;
  if (a) {
    a->parts = (float*)parts;
    a->part_ml = (float2*)part_ml;
    a->part_bad = (int*)part_bad;
    a->unit_ml = (float2*)unit_ml;
    a->scores = (float*)scores;
  }
  return used;
}

}  // namespace

bool attention_cache4_step_takes(int n_seqs, int m, int n_heads, int n_kv, int max_len) {
  return (long long)n_seqs * n_kv * ((m * (n_heads / n_kv) + 7) / 8) * ((max_len + ST_CHUNK - 1) / ST_CHUNK) < (1ll << 31);
}

size_t attention_cache4_step_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights) {
  return step_layout(nullptr, nullptr, step_shape(n_seqs, m, n_heads, n_kv, max_len, weights), n_seqs, m, n_heads, hd, max_len, weights);
}

int launch_attention_cache4_step(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream) {
  const step_shape w(p.c.n_seqs, p.m, p.n_heads, p.c.n_kv, p.max_len, p.weights != nullptr);
  step_args a{p, w.ctas, w.col_blocks, w.per_unit, w.alone};
  step_layout(&a, workspace, w, p.c.n_seqs, p.m, p.n_heads, p.c.hd, p.max_len, p.weights != nullptr);
  return dtype == OP_F16 ? launch_shape<__half>(a, w.cols, stream) : launch_shape<__nv_bfloat16>(a, w.cols, stream);
}

}  // namespace lcu
