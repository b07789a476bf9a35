// Attention of prompt rows over the 4-bit cache (cache4.cuh) on tcgen05.
//
//   s_rj = q_r . k_j / sqrt(head_dim),  o_r = sum_j e^(s_rj - max) v_j / sum_j e^(s_rj - max),   rows r = (row of the call, head of the key/value head)
// A prompt meets every cached row once per 128 rows, so the codes are expanded to halves once, exactly (7-bit scales), into the workspace
// of the call - 4 bytes moved per value and product, against codes expanded again for each 128 x 128 tile at a cost close to the tile's own
// exponentials.  bfloat16 queries become halves too, each row by a power of two, so that both types share everything behind.
//
// One CTA per (sequence, key/value head, 128 rows), two CTAs per SM, in steps of 64 keys.  Scores lie in two buffers of tensor memory: those of
// the next step are formed under this step's exponentials (in one buffer, steps of 128 keys, score - exponential - product followed one
// another: timed in turn, 2000 rows of 32 heads behind 6000 rows of 8 took a ninth longer, 4000 rows a seventh).  Three accumulators' columns
// for two CTAs are what tensor memory holds; narrower products of the scores read their queries from shared memory more often, 1.5 x the time.
// A thread owns a row, reads 32 keys at a time and keeps the running maximum and the sum; probabilities go back to tensor memory, over the
// scores, as halves: the A operand of the product with the values, whose accumulator stays in tensor memory.  A maximum is raised only
// when a score passes it by 8 (powers of two; the reference of the exponentials is 7 below it, cache4_attention.cuh), so that a step's
// exponentials are formed with the old one while its own maximum is looked for; only where a row fails that test is its warp's step done again and
// the output rescaled, once the product before is done.
// Exponentials (16 a cycle and SM) and products are both busy 55 % of the time that a CTA is there.
//
// Weights: once maxima and sums are known, a second kernel forms the scores the other way round - a thread owns a cached row - and adds
// e^(s - max) / sum over all rows in their order.
//
// Values whose scale is no number are expanded to zeros and the first such row of every 128 and block is listed: rows that see it
// get NaN in that block's dimensions, earlier ones do not.
#include <algorithm>
#include <type_traits>

#include "cache4_attention.cuh"
#include "runtime.cuh"
#include "tc_common.cuh"

namespace lcu {
namespace {

constexpr int PR_ROWS = 128, PR_KEYS = 128, PR_STEP = 64;
constexpr int PR_SOFT_WARPS = 4, PR_THREADS = 32 * (PR_SOFT_WARPS + 2);  // of the kernel of the outputs
constexpr int PW_SOFT_WARPS = 8, PW_THREADS = 32 * (PW_SOFT_WARPS + 2);  // of the weights'

struct prompt_args {
  cache4_attention_params p;
  __half* k_half;     // [units][t_pad][hd]
  __half* v_half;
  __half* q_half;     // [units][r_pad][hd]
  float2* row_stats;  // [units][r_pad] factor of a row's scores (powers of two); logarithm of its sum (weights; infinity: no such row)
  int* bad;           // [units][t_pad / 128][4] first row of each 128 whose values of a block are no numbers
  int t_pad, r_pad;
  int ctas;           // split: CTAs that share the tiles of all items (0: a CTA per item)
  int* prefix;        // split: [units * row blocks + 1] tiles of the items before each
  float* part_o;      // split: [ctas][2][128][hd] sums of runs of tiles that begin, or end, inside an item
  float2* part_ml;    // split: [ctas][2][128] their rows' references (powers of two) and sums
  float* part_w;      // weights of runs of rows: [segments][units][t_pad]
  int segments;
  int* err;
};

__device__ __forceinline__ int rows_of(const cache4_attention_params& p, int held) {  // cached rows that the last row of the call sees
  const int room = min(p.c.ctx, p.max_len);
  return held < 0 ? 0 : held >= room ? room : min(held + p.m, room);
}
__device__ __forceinline__ int limit_of(const cache4_attention_params& p, int held, int i) {
  const int room = min(p.c.ctx, p.max_len);
  return held < 0 ? 0 : held >= room ? room : min(held + i + 1, room);
}

// An item is 128 rows of a unit; its tiles are the 128 cached rows each that its last row sees.
__device__ __forceinline__ int tiles_of(const cache4_attention_params& p, int held, int block) {
  const int group = p.n_heads / p.c.n_kv, last = min((block + 1) * PR_ROWS, p.m * group) - 1;
  return (limit_of(p, held, last / group) + PR_KEYS - 1) / PR_KEYS;
}

// ------------------------------------------------------------------ expansion
// One CTA per 128 rows of a unit's keys and values, or of its queries.
template <typename T, int HD>
__global__ void __launch_bounds__(256) prompt_expand_kernel(const prompt_args a, int key_blocks, int row_blocks) {
  const cache4_attention_params& p = a.p;
  __shared__ int s_bad[4];
  constexpr int WORDS = HD / 8, G = HD / 32;
  pdl_launch_dependents();
  if (a.ctas && blockIdx.x == gridDim.x - 1) {  // (the last CTA: where the items' tiles lie in the row of all tiles)
    __shared__ int s_sum[8];
    int carry = 0;
    const int items = p.c.n_seqs * p.c.n_kv * row_blocks;
    for (int i0 = 0; i0 < items; i0 += 256) {
      const int i = i0 + threadIdx.x, unit = i / row_blocks;
      const int n = i < items ? tiles_of(p, p.lengths[unit / p.c.n_kv], i - unit * row_blocks) : 0;
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if ((threadIdx.x & 31) >= o) x += y;
      }
      if ((threadIdx.x & 31) == 31) s_sum[threadIdx.x >> 5] = x;
      __syncthreads();
      int before = carry;
      for (int w = 0; w < 8; ++w) {
        if (w < (int)(threadIdx.x >> 5)) before += s_sum[w];
        carry += s_sum[w];
      }
      __syncthreads();
      if (i < items) a.prefix[i] = before + x - n;
    }
    if (threadIdx.x == 0) a.prefix[items] = carry;
    return;
  }
  const int unit = blockIdx.x / (key_blocks + row_blocks), b = blockIdx.x % (key_blocks + row_blocks), seq = unit / p.c.n_kv, kvh = unit % p.c.n_kv;
  const int held = p.lengths[seq], seen = rows_of(p, held);
  if (b < key_blocks) {
    if (b * PR_KEYS >= seen) return;
    if (threadIdx.x < 4) s_bad[threadIdx.x] = 0x7fffffff;
    __syncthreads();
    const int nb = HD / p.c.bs;
    constexpr int UNROLL = 4;  // (words requested before the first is used)
    for (int w0 = threadIdx.x; w0 < PR_KEYS * WORDS; w0 += 256 * UNROLL) {
      uint32_t kw[UNROLL], vw[UNROLL];
      float ks[UNROLL], vs[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int w = w0 + u * 256, word = w % WORDS, j = b * PR_KEYS + w / WORDS, d = (word % G) * 32 + (word / G) * 8;
        kw[u] = vw[u] = 0;
        ks[u] = vs[u] = 0.f;
        if (j < seen) {
          const size_t at = (size_t)unit * p.c.ctx + j;
          kw[u] = __ldg(reinterpret_cast<const uint32_t*>(p.c.k_codes + at * (HD / 2)) + word);
          vw[u] = __ldg(reinterpret_cast<const uint32_t*>(p.c.v_codes + at * (HD / 2)) + word);
          ks[u] = __half2float(p.c.k_scales[at * nb + d / p.c.bs]);
          vs[u] = __half2float(p.c.v_scales[at * nb + d / p.c.bs]);
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int w = w0 + u * 256, word = w % WORDS, j = b * PR_KEYS + w / WORDS, d = (word % G) * 32 + (word / G) * 8;
        if (vs[u] != vs[u]) {
          atomicMin(&s_bad[d / p.c.bs], j);
          vs[u] = 0.f;
        }
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = cache4_value(kw[u], e, ks[u]);
          y[e] = cache4_value(vw[u], e, vs[u]);
        }
        const size_t to = ((size_t)unit * a.t_pad + j) * HD + d;  // (rows behind the last one, to the block's end: zeros)
        *reinterpret_cast<uint4*>(a.k_half + to) = pack8<__half>(x);
        *reinterpret_cast<uint4*>(a.v_half + to) = pack8<__half>(y);
      }
    }
    __syncthreads();
    if (threadIdx.x < 4) a.bad[((size_t)unit * key_blocks + b) * 4 + threadIdx.x] = s_bad[threadIdx.x];
    return;
  }
  // queries: HD / 8 lanes per row
  const int group = p.n_heads / p.c.n_kv, rows = p.m * group;
  for (int w = threadIdx.x; w < PR_ROWS * WORDS; w += 256) {
    const int r = (b - key_blocks) * PR_ROWS + w / WORDS, word = w % WORDS;
    uint4 v = make_uint4(0, 0, 0, 0);
    float down = 1.f;
    if (r < rows) v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + ((size_t)seq * p.m + r / group) * p.ld_q + (kvh * group + r % group) * HD + word * 8);
    if (sizeof(T) == 2 && !std::is_same<T, __half>::value) {  // a power of two takes the row's largest magnitude into [1, 2)
      float x[8], most = 0.f;
      unpack8<T>(v, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
      for (int o = 1; o < WORDS; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const int ex = (int)(__float_as_uint(most) >> 23);
      float up = 1.f;
      if (ex >= 20 && ex <= 230) {
        up = __uint_as_float((uint32_t)(254 - ex) << 23);
        down = __uint_as_float((uint32_t)ex << 23);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= up;
      v = pack8<__half>(x);
    }
    *reinterpret_cast<uint4*>(a.q_half + ((size_t)unit * a.r_pad + r) * HD + word * 8) = v;
    if (word == 0) a.row_stats[(size_t)unit * a.r_pad + r] = make_float2(down * (1.4426950408889634f * rsqrtf((float)HD)), INFINITY);
  }
}

// ------------------------------------------------------------------ shared pieces
__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// two binary32 numbers as one operand: half as many instructions for the exponentials' arguments and sums
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float2 both_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void st_32x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory");
}

template <int HD>
struct prompt_shape {
  static constexpr int NKB = HD / 64;                        // 64-wide blocks of the head dimension
  static constexpr uint32_t BLOCK = 128 * 64 * 2;            // 128 rows x 64 dimensions
  static constexpr uint32_t OPERAND = NKB * BLOCK;           // queries, keys or values (2 x NKB atoms of 64 keys x 64 dimensions)
  static constexpr uint32_t STEP = NKB * 64 * 64 * 2;        // 64 keys, or 64 values
  static constexpr int RING = 4;                             // two CTAs per SM
  static constexpr uint32_t SMEM = OPERAND + RING * STEP + 1024 /* alignment slack */ + 256 /* barriers, tensor-memory slot */;
  static constexpr uint32_t IDESC_S = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t IDESC_S64 = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((128u >> 4) << 24);  // values: contiguous along the dimension
};

// barriers
constexpr int B_Q = 0, B_FULL = 1, B_EMPTY = B_FULL + 4, B_S = B_EMPTY + 4, B_P = B_S + 2, B_V = B_P + 2, B_O = B_V + 1, B_COUNT = B_O + 1;

// ------------------------------------------------------------------ outputs
template <typename T, int HD, bool SPLIT>
__global__ void __launch_bounds__(PR_THREADS, 2) prompt_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v, const prompt_args a, int row_blocks, int units) {
  using sh = prompt_shape<HD>;
  constexpr int NKB = sh::NKB, RING = sh::RING;
  constexpr uint32_t OPERAND = sh::OPERAND, STEP = sh::STEP, ATOM = 64 * 64 * 2, TMEM_COLS = 256, O_COL = 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_addr = base, ring_addr = base + OPERAND;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OPERAND + RING * STEP);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_bad[4];
  const cache4_attention_params& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.n_heads / p.c.n_kv, rows = p.m * group;
  __shared__ int s_first, s_gave_up;
  volatile int* gave_up = &s_gave_up;

  if (tid == 0) {
    mbar_init(smem_u32(&bars[B_Q]), 1);
    for (int i = 0; i < RING; ++i) {
      mbar_init(smem_u32(&bars[B_FULL + i]), 1);
      mbar_init(smem_u32(&bars[B_EMPTY + i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars[B_S + i]), 1);
      mbar_init(smem_u32(&bars[B_P + i]), PR_SOFT_WARPS);
    }
    mbar_init(smem_u32(&bars[B_V]), 1);
    mbar_init(smem_u32(&bars[B_O]), 1);
    *failed = 0;
    *gave_up = 0;
    fence_mbar_init();
  }
  if (warp == PR_SOFT_WARPS + 1) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();
  constexpr bool HEED = false;  // (an earlier launch's error says nothing about this one)
  // This CTA's tiles: those of its item - the last rows, which see most, first; all units' side by side - or an equal share of all.
  int lo = 0, hi = 0x7fffffff, item0 = (row_blocks - 1 - (int)blockIdx.x / units) + (int)blockIdx.x % units * row_blocks;
  if constexpr (SPLIT) {
    const int items = units * row_blocks, total = a.prefix[items];
    const int ctas = min(a.ctas, total);  // (that have a tile at least)
    lo = hi = total;
    if ((int)blockIdx.x < ctas) {
      lo = (int)((long long)total * blockIdx.x / ctas);
      hi = (int)((long long)total * (blockIdx.x + 1) / ctas);
    }
    if (warp == 0) {  // the item that tile `lo` belongs to: the last whose tiles begin at or before it
      int from = 0, to = items;  // (prefix[from] <= lo < prefix[to])
      while (to - from > 1) {
        const int step = (to - from + 32) / 33, i = from + step * (lane + 1);
        const unsigned m = __ballot_sync(0xffffffffu, i < to && a.prefix[min(i, items)] <= lo);
        const int k = __popc(m);
        to = min(to, from + step * (k + 1));
        from += step * k;
      }
      if (lane == 0) s_first = from;
    }
    __syncthreads();
    item0 = s_first;
  }
  struct run {
    int item, first, last, all;  // tiles [first, last) of an item's `all`
    int from, to;                // and steps of 64 keys: as far as the last row sees
    int seq, kvh, unit, r0, held;
  };
  int pos = lo;
  auto next_run = [&](run& w, int& item) {  // (the same for all roles)
    for (; !SPLIT || pos < hi; ++item) {
      w.item = item;
      w.unit = item / row_blocks;
      w.seq = w.unit / p.c.n_kv;
      w.kvh = w.unit - w.seq * p.c.n_kv;
      w.r0 = (item - w.unit * row_blocks) * PR_ROWS;
      w.held = p.lengths[w.seq];
      w.all = tiles_of(p, w.held, w.r0 / PR_ROWS);
      w.first = 0;
      w.last = w.all;
      const int steps = w.all ? (limit_of(p, w.held, (min(w.r0 + PR_ROWS, rows) - 1) / group) + PR_STEP - 1) / PR_STEP : 0;
      w.from = 0;
      w.to = steps;
      if constexpr (!SPLIT) return true;
      const int begin = a.prefix[item];
      w.first = pos - begin;
      w.last = min(w.all, hi - begin);
      w.from = 2 * w.first;
      w.to = min(2 * w.last, steps);
      if (w.last > w.first) {
        pos = begin + w.last;
        ++item;
        return true;
      }
    }
    return false;
  };

  if (warp == PR_SOFT_WARPS) {
    if (tc_elect()) {  // ---- loads: a run's queries; K, V, K, V, ..
      tc_ring r;
      run w;
      bool ok = true;
      for (int item = item0, n = 0; ok && (SPLIT || n == 0) && next_run(w, item); ++n) {
        if (w.all == 0) break;
        if (n) ok = mbar_wait(smem_u32(&bars[B_O]), (uint32_t)(n - 1) & 1u, a.err, DEV_ERR_EMPTY_WAIT, HEED);  // (the queries' last product is done)
        if (!ok) break;
        mbar_arrive_expect_tx(smem_u32(&bars[B_Q]), OPERAND);
        for (int kb = 0; kb < NKB; ++kb) tma_load_3d(q_addr + kb * sh::BLOCK, &map_q, kb * 64, w.r0, w.unit, smem_u32(&bars[B_Q]));
        for (int it = 2 * w.from; it < 2 * w.to; ++it, r.step(RING)) {
          ok = mbar_wait(smem_u32(&bars[B_EMPTY + r.slot]), r.phase ^ 1u, a.err, DEV_ERR_EMPTY_WAIT, HEED);
          if (!ok) break;
          const uint32_t full = smem_u32(&bars[B_FULL + r.slot]), dst = ring_addr + (uint32_t)r.slot * STEP;
          mbar_arrive_expect_tx(full, STEP);
          if (!(it & 1)) {
            for (int c = 0; c < NKB; ++c) tma_load_3d(dst + c * ATOM, &map_k, c * 64, (it >> 1) * PR_STEP, w.unit, full);
          } else {
            for (int c = 0; c < NKB; ++c) tma_load_3d(dst + c * ATOM, &map_v, c * 64, (it >> 1) * PR_STEP, w.unit, full);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == PR_SOFT_WARPS + 1) {
    // ---- products, in this order: S_0, S_1, O += P_0 V_0, S_2, O += P_1 V_1, ..: a step's scores are formed under the exponentials of the step
    // before, once the product of the probabilities that they replace is done
    tc_ring r;  // (keys and values in the loads' order: K_0, V_0, K_1, ..)
    run w;
    bool ok = true;
    int count = 0;
    for (int item = item0, n = 0; ok && (SPLIT || n == 0) && next_run(w, item); ++n) {
      if (w.all == 0) break;
      ok = mbar_wait_warp(smem_u32(&bars[B_Q]), (uint32_t)n & 1u, a.err, DEV_ERR_FULL_WAIT, HEED);
      auto scores = [&](const tc_ring& keys, int buffer) {
        ok = ok && mbar_wait_warp(smem_u32(&bars[B_FULL + keys.slot]), keys.phase, a.err, DEV_ERR_FULL_WAIT, HEED);
        if (!ok) return;
        tc_fence_after();
        if (tc_elect()) {
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) {
            const uint64_t a_desc = smem_desc_sw128(q_addr + kb * sh::BLOCK), b_desc = smem_desc_sw128(ring_addr + (uint32_t)keys.slot * STEP + kb * ATOM);
#pragma unroll
            for (int k = 0; k < 4; ++k) tc_mma_f16(tmem + (uint32_t)(buffer * PR_STEP), a_desc + 2 * k, b_desc + 2 * k, sh::IDESC_S64, (kb | k) != 0);
          }
          tc_commit(smem_u32(&bars[B_EMPTY + keys.slot]));
          tc_commit(smem_u32(&bars[B_S + buffer]));
        }
        __syncwarp();
      };
      scores(r, count & 1);
      for (int u = w.from; u < w.to && ok; ++u, ++count) {
        r.step(RING);  // to this step's values
        tc_ring next = r;
        next.step(RING);
        // (products of different shapes are not promised to run in the order of issue: what the next scores replace must have been read;
        // left to that order, 2000 rows behind 6000 took 3 % less in turn, others the same)
        if (u > w.from) ok = ok && mbar_wait_warp(smem_u32(&bars[B_V]), (uint32_t)(count - 1) & 1u, a.err, DEV_ERR_TMEM_WAIT, HEED);
        if (ok && u + 1 < w.to) scores(next, (count + 1) & 1);
        ok = ok && mbar_wait_warp(smem_u32(&bars[B_P + (count & 1)]), (uint32_t)(count >> 1) & 1u, a.err, DEV_ERR_FULL_WAIT, HEED);
        ok = ok && mbar_wait_warp(smem_u32(&bars[B_FULL + r.slot]), r.phase, a.err, DEV_ERR_FULL_WAIT, HEED);
        if (!ok) break;
        tc_fence_after();
        if (tc_elect()) {
          const uint64_t b_desc = smem_desc_sw128_mn(ring_addr + (uint32_t)r.slot * STEP, ATOM);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(tmem + O_COL, tmem + (uint32_t)((count & 1) * PR_STEP) + k * 8, b_desc + (uint64_t)(k * 2048 >> 4), sh::IDESC_PV, (uint32_t)(u > w.from || k != 0));
          tc_commit(smem_u32(&bars[B_EMPTY + r.slot]));
          tc_commit(smem_u32(&bars[B_V]));
          if (u + 1 == w.to) tc_commit(smem_u32(&bars[B_O]));
        }
        __syncwarp();
        r = next;
      }
    }
    if (!ok) {  // (lets the softmax warps leave, without results)
      if (tc_elect()) {
        *failed = 1;
        __threadfence_block();
        tc_commit(smem_u32(&bars[B_S]));
        tc_commit(smem_u32(&bars[B_S + 1]));
        tc_commit(smem_u32(&bars[B_V]));
        tc_commit(smem_u32(&bars[B_O]));
      }
      __syncwarp();
    }
  } else {
    // ---- softmax: a thread owns a row
    const int in_tile = warp * 32 + lane;
    const uint32_t row_at = tmem + ((uint32_t)(warp * 32) << 16), o_at = row_at + O_COL;
    bool go = true;
    int count = 0;
    run w;
    for (int item = item0, n = 0; go && (SPLIT || n == 0) && next_run(w, item); ++n) {
    const int r = w.r0 + in_tile, i = r / group, limit = r < rows ? limit_of(p, w.held, i) : 0;
    const int warp_limit = __shfl_sync(0xffffffffu, limit, 0);  // (what the warp's first row sees)
    const bool all_there = __all_sync(0xffffffffu, r < rows), whole = !SPLIT || w.last - w.first == w.all;
    const float f = a.row_stats[(size_t)w.unit * a.r_pad + r].x;
    if (n) bar_sync(1, 32 * PR_SOFT_WARPS);  // (the run before has read s_bad)
    if (tid < 4) s_bad[tid] = 0x7fffffff;
    bar_sync(1, 32 * PR_SOFT_WARPS);
    // the first row of no numbers among those this item sees
    if (whole) {
      const int nb = HD / p.c.bs;
      const int* list = a.bad + (size_t)w.unit * (a.t_pad / PR_KEYS) * 4;
      for (int e = tid; e < w.all * nb; e += 32 * PR_SOFT_WARPS) {
        const int v = list[(e / nb) * 4 + e % nb];
        if (v != 0x7fffffff) atomicMin(&s_bad[e % nb], v);
      }
    }
    float less = 0.f, high = -INFINITY, sum = 0.f;  // minus the reference (0 while there is none); 8 above the maximum, as the products give scores
    for (int u = w.from; u < w.to; ++u, ++count) {
      const bool ok = mbar_wait(smem_u32(&bars[B_S + (count & 1)]), (uint32_t)(count >> 1) & 1u, a.err, DEV_ERR_TMEM_WAIT, HEED);
      tc_fence_after();
      go = __all_sync(0xffffffffu, ok && *failed == 0);
      if (!go) break;
      const uint32_t s_at = row_at + (uint32_t)((count & 1) * PR_STEP);
      const int left = limit - u * PR_STEP;  // keys of the step that the row sees
      const bool ragged = !all_there || warp_limit < (u + 1) * PR_STEP;
      uint32_t pw[32];
      float top, part;
      auto step = [&]() {
        float t0 = -INFINITY, t1 = -INFINITY;
        uint64_t sums = 0;
        const uint64_t factor = pair_of(f, f), minus = pair_of(less, less);
        uint32_t s[2][32];
        auto half = [&](uint32_t (&x)[32], int c) {
          if (ragged) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= left) x[e] = 0xff800000u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            t0 = fmaxf(t0, __uint_as_float(x[e]));
            t1 = fmaxf(t1, __uint_as_float(x[e + 1]));
            const float2 y = both_of(fma_pair(pair_of(x[e], x[e + 1]), factor, minus));
            const float e0 = ex2(y.x), e1 = ex2(y.y);
            sums = add_pair(sums, pair_of(e0, e1));
            pw[c * 16 + e / 2] = pack2<__half>(e0, e1);
          }
        };
        tc_ld_32x32(s_at, s[0]);
        tc_wait_ld();
        tc_ld_32x32(s_at + 32, s[1]);  // (on its way under the first half's exponentials)
        half(s[0], 0);
        tc_wait_ld();
        half(s[1], 1);
        top = fmaxf(t0, t1);
        part = both_of(sums).x + both_of(sums).y;
      };
      step();
      if (__any_sync(0xffffffffu, top > high)) {
        float k = 1.f;
        if (top > high) {
          const float now = top * f, reference = reference_of(now);
          k = high == -INFINITY ? 0.f : ex2(-less - reference);
          less = -reference;
          high = (now + 8.f) / f;
          sum *= k;
        }
        if (u > w.from) {
          // the output as the product before left it (this step's waits for this warp's probabilities)
          const bool done = mbar_wait(smem_u32(&bars[B_V]), (uint32_t)(count - 1) & 1u, a.err, DEV_ERR_TMEM_WAIT, HEED);
          tc_fence_after();
          go = __all_sync(0xffffffffu, done && *failed == 0);
          if (!go) break;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t x[32];
            tc_ld_32x32(o_at + (uint32_t)c, x);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * k);
            st_32x32(o_at + (uint32_t)c, x);
          }
        }
        step();
      }
      sum += part;
      st_32x32(s_at, pw);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars[B_P + (count & 1)]));
    }
    bar_sync(1, 32 * PR_SOFT_WARPS);  // (s_bad)
    if (w.all) {
      const bool ok = go && mbar_wait(smem_u32(&bars[B_O]), (uint32_t)n & 1u, a.err, DEV_ERR_TMEM_WAIT, HEED);
      tc_fence_after();
      go = __all_sync(0xffffffffu, ok && *failed == 0);
    }
    // (all warps go on together, or none: the barriers of the next run count them)
    if constexpr (SPLIT) {
      if (!go && lane == 0) *gave_up = 1;
      bar_sync(1, 32 * PR_SOFT_WARPS);
      if (*gave_up) go = false;
    }
    if (!go) break;
    if (whole) {
      const float rl = limit ? 1.f / sum : 0.f;
      T* out = reinterpret_cast<T*>(p.out) + ((size_t)w.seq * p.m + i) * p.ld_out + (w.kvh * group + r % group) * HD;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t x[32];
        if (w.all) {
          tc_ld_32x32(o_at + (uint32_t)c, x);
          tc_wait_ld();
        }
        if (r < rows) {
          const bool none = limit && s_bad[c / p.c.bs] < limit;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = none ? __int_as_float(0x7fffffff) : limit ? __uint_as_float(x[q * 8 + e]) * rl : 0.f;
            reinterpret_cast<uint4*>(out + c)[q] = pack8<T>(y);
          }
        }
      }
      if (p.weights && r < rows) a.row_stats[(size_t)w.unit * a.r_pad + r].y = limit ? log2f(sum * (1.f / LIFT_FACTOR)) - (less - LIFT) : INFINITY;
    } else {
      const size_t place = ((size_t)blockIdx.x * 2 + (w.first == 0)) * PR_ROWS + in_tile;
      float* to = a.part_o + place * HD;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t x[32];
        tc_ld_32x32(o_at + (uint32_t)c, x);
        tc_wait_ld();
#pragma unroll
        for (int q = 0; q < 8; ++q) reinterpret_cast<uint4*>(to + c)[q] = make_uint4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
      }
      a.part_ml[place] = make_float2(high == -INFINITY ? -INFINITY : -less, sum);
    }
    tc_fence_before();  // (the accumulator is read: the next run's products come behind this thread's arrival)
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == PR_SOFT_WARPS + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem, TMEM_COLS);
  }
}

// Joins the runs of items that several CTAs did, and gives zeros for sequences not in use: a warp per row, 16 CTAs per item.
template <typename T, int HD>
__global__ void __launch_bounds__(256) prompt_join_kernel(const prompt_args a, int row_blocks) {
  const cache4_attention_params& p = a.p;
  __shared__ int s_bad[4];
  const int item = blockIdx.x / 16, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = item / row_blocks, seq = unit / p.c.n_kv, kvh = unit - seq * p.c.n_kv, block = item - unit * row_blocks;
  const int group = p.n_heads / p.c.n_kv, in_tile = blockIdx.x % 16 * 8 + warp, r = block * PR_ROWS + in_tile, i = r / group;
  const bool there = r < p.m * group;
  pdl_launch_dependents();
  pdl_wait();
  const int held = p.lengths[seq], items = p.c.n_seqs * p.c.n_kv * row_blocks;
  const int begin = a.prefix[item], end = a.prefix[item + 1], total = a.prefix[items];
  T* out = reinterpret_cast<T*>(p.out) + ((size_t)seq * p.m + i) * p.ld_out + (kvh * group + r % group) * HD;
  constexpr int EACH = HD / 32;
  if (begin == end) {
    if (there)
      for (int e = 0; e < EACH; e += 2) reinterpret_cast<uint32_t*>(out)[(lane * EACH + e) / 2] = 0u;
    return;
  }
  // the CTAs of its first and last tile
  const int ctas = min(a.ctas, total), first = (int)(((long long)(begin + 1) * ctas - 1) / total), last = (int)(((long long)end * ctas - 1) / total);
  if (first == last) return;
  if (threadIdx.x < 4) s_bad[threadIdx.x] = 0x7fffffff;
  __syncthreads();
  const int nb = HD / p.c.bs;
  const int* list = a.bad + (size_t)unit * (a.t_pad / PR_KEYS) * 4;
  for (int e = threadIdx.x; e < (end - begin) * nb; e += 256) {
    const int v = list[(e / nb) * 4 + e % nb];
    if (v != 0x7fffffff) atomicMin(&s_bad[e % nb], v);
  }
  __syncthreads();
  if (!there) return;
  auto place = [&](int cta) { return ((size_t)cta * 2 + (cta == first)) * PR_ROWS + in_tile; };
  float top = -INFINITY;
  for (int b = first + lane; b <= last; b += 32) top = fmaxf(top, a.part_ml[place(b)].x);
  top = warp_max(top);
  float l = 0.f, x[EACH] = {};
#pragma unroll 4
  for (int b = first; b <= last; ++b) {
    const float2 ml = a.part_ml[place(b)];
    const float k = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);  // (a reference of nothing: sums of 0, or of NaN)
    l += ml.y * k;
    const float* from = a.part_o + place(b) * HD + lane * EACH;
    if constexpr (EACH == 4) {
      const float4 v = *reinterpret_cast<const float4*>(from);
      x[0] += v.x * k;
      x[1] += v.y * k;
      x[2] += v.z * k;
      x[3] += v.w * k;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(from);
      x[0] += v.x * k;
      x[1] += v.y * k;
    }
  }
  const int limit = limit_of(p, held, i);
  const float rl = s_bad[lane * EACH / p.c.bs] < limit ? __int_as_float(0x7fffffff) : 1.f / l;
#pragma unroll
  for (int e = 0; e < EACH; e += 2) reinterpret_cast<uint32_t*>(out)[(lane * EACH + e) / 2] = pack2<T>(x[e] * rl, x[e + 1] * rl);
  if (p.weights && lane == 0) a.row_stats[(size_t)unit * a.r_pad + r].y = log2f(l * (1.f / LIFT_FACTOR)) + (top + LIFT);
}

// ------------------------------------------------------------------ weights
__device__ __forceinline__ void store_weight(const cache4_attention_params& p, int unit, int j, int held, float total) {
  float* to = p.weights + (size_t)unit * p.c.ctx + j;
  *to = p.beta == 0.f || j >= held ? total : fmaf(p.beta, *to, total);
}
__global__ void __launch_bounds__(256) prompt_add_kernel(const prompt_args a, int units) {
  const int unit = blockIdx.y;
  pdl_wait();
  const int held = a.p.lengths[unit / a.p.c.n_kv], seen = rows_of(a.p, held);
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= seen) return;
  float total = 0.f;
  for (int s = 0; s < a.segments; ++s) total += a.part_w[((size_t)s * units + unit) * a.t_pad + j];
  store_weight(a.p, unit, j, held, total);
}
// One CTA per (sequence, key/value head, 128 cached rows), two per SM; rows of the call in tiles of 128 through a ring.  Two score
// accumulators: one tile's exponentials run under the next one's product.
constexpr int W_KEYS = 0, W_FULL = 1, W_EMPTY = W_FULL + 2, W_S = W_EMPTY + 2, W_FREE = W_S + 2, W_COUNT = W_FREE + 2;
template <int HD>
__global__ void __launch_bounds__(PW_THREADS, 2) prompt_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const prompt_args a,
                                                                       int key_blocks, int units) {
  using sh = prompt_shape<HD>;
  constexpr int NKB = sh::NKB;
  constexpr uint32_t OPERAND = sh::OPERAND, TMEM_COLS = 256, STATS = 128 * sizeof(float2), STAGE = OPERAND + STATS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t k_addr = base, ring_addr = base + OPERAND, stats_addr = ring_addr + 2 * OPERAND;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 3 * OPERAND + 4 * STATS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + W_COUNT);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const cache4_attention_params& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ float s_total[PR_KEYS];
  const int segment = (int)blockIdx.x % a.segments, at = (int)blockIdx.x / a.segments;
  const int block = at / units, unit = at % units, seq = unit / p.c.n_kv;
  const int group = p.n_heads / p.c.n_kv, rows = p.m * group, j0 = block * PR_KEYS;
  if (tid == 0) {
    mbar_init(smem_u32(&bars[W_KEYS]), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars[W_FULL + i]), 1);
      mbar_init(smem_u32(&bars[W_EMPTY + i]), 1);
      mbar_init(smem_u32(&bars[W_S + i]), 1);
      mbar_init(smem_u32(&bars[W_FREE + i]), PW_SOFT_WARPS);
    }
    *failed = 0;
    fence_mbar_init();
  }
  if (warp == PW_SOFT_WARPS + 1) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  constexpr bool HEED = false;
  const int held = p.lengths[seq], seen = rows_of(p, held);
  // rows from the first that sees the first key on; this CTA's run of their tiles
  const int from_tile = max(0, j0 - held) * group / PR_ROWS, all_tiles = j0 < seen ? (rows + PR_ROWS - 1) / PR_ROWS - from_tile : 0;
  const int first = from_tile + (int)((long long)all_tiles * segment / a.segments);
  const int n_tiles = from_tile + (int)((long long)all_tiles * (segment + 1) / a.segments) - first;

  if (warp == PW_SOFT_WARPS) {
    if (n_tiles > 0 && tc_elect()) {
      mbar_arrive_expect_tx(smem_u32(&bars[W_KEYS]), OPERAND);
      for (int kb = 0; kb < NKB; ++kb) tma_load_3d(k_addr + kb * sh::BLOCK, &map_k, kb * 64, j0, unit, smem_u32(&bars[W_KEYS]));
      tc_ring r;
      for (int it = 0; it < n_tiles; ++it, r.step(2)) {
        if (!mbar_wait(smem_u32(&bars[W_EMPTY + r.slot]), r.phase ^ 1u, a.err, DEV_ERR_EMPTY_WAIT, HEED)) break;
        const uint32_t full = smem_u32(&bars[W_FULL + r.slot]);
        mbar_arrive_expect_tx(full, STAGE);
        for (int kb = 0; kb < NKB; ++kb) tma_load_3d(ring_addr + (uint32_t)r.slot * OPERAND + kb * sh::BLOCK, &map_q, kb * 64, (first + it) * PR_ROWS, unit, full);
        // (the four places of row statistics: scores of four tiles ago are read before the product of two ago may start)
        bulk_g2s(stats_addr + (uint32_t)(it & 3) * STATS, a.row_stats + (size_t)unit * a.r_pad + (first + it) * PR_ROWS, STATS, full);
      }
    }
    __syncwarp();
  } else if (warp == PW_SOFT_WARPS + 1) {
    bool ok = n_tiles > 0 && mbar_wait_warp(smem_u32(&bars[W_KEYS]), 0, a.err, DEV_ERR_FULL_WAIT, HEED);
    tc_ring r;
    for (int it = 0; it < n_tiles && ok; ++it, r.step(2)) {
      ok = mbar_wait_warp(smem_u32(&bars[W_FULL + r.slot]), r.phase, a.err, DEV_ERR_FULL_WAIT, HEED);
      ok = ok && mbar_wait_warp(smem_u32(&bars[W_FREE + r.slot]), r.phase ^ 1u, a.err, DEV_ERR_TMEM_WAIT, HEED);
      if (!ok) break;
      tc_fence_after();
      if (tc_elect()) {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
          const uint64_t a_desc = smem_desc_sw128(k_addr + kb * sh::BLOCK), b_desc = smem_desc_sw128(ring_addr + (uint32_t)r.slot * OPERAND + kb * sh::BLOCK);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_f16(tmem + (uint32_t)(r.slot * 128), a_desc + 2 * k, b_desc + 2 * k, sh::IDESC_S, (kb | k) != 0);
        }
        tc_commit(smem_u32(&bars[W_EMPTY + r.slot]));
        tc_commit(smem_u32(&bars[W_S + r.slot]));
      }
      __syncwarp();
    }
    if (!ok && n_tiles > 0) {
      if (tc_elect()) {
        *failed = 1;
        __threadfence_block();
        tc_commit(smem_u32(&bars[W_S]));
        tc_commit(smem_u32(&bars[W_S + 1]));
      }
      __syncwarp();
    }
  } else if (n_tiles > 0) {
    // a thread owns half the rows of every tile for a key
    const int quad = warp & 3, half = warp >> 2, j = j0 + quad * 32 + lane;
    // the first row that sees the key (none sees one behind the last)
    const int from = j >= seen ? 0x7fffffff : max(0, j - held) * group;
    float total = 0.f;
    bool go = true;
    tc_ring r;
    for (int it = 0; it < n_tiles; ++it, r.step(2)) {
      const bool ok = mbar_wait(smem_u32(&bars[W_S + r.slot]), r.phase, a.err, DEV_ERR_TMEM_WAIT, HEED);
      tc_fence_after();
      go = __all_sync(0xffffffffu, ok && *failed == 0);
      if (!go) break;
      const int q0 = (first + it) * PR_ROWS;
      const bool ragged = !__all_sync(0xffffffffu, from <= q0) || q0 + PR_ROWS > rows;
      const uint32_t s_at = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(r.slot * 128 + half * 64);
      const float4* st = reinterpret_cast<const float4*>(smem + 3 * OPERAND + (size_t)(it & 3) * STATS) + half * 32;
      float part = 0.f;
      auto tile = [&](auto checked) {  // (checked: some of the keys, or of the rows, are none that count)
        uint32_t both[2][16];
        ld_32x16(s_at, both[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t(&s)[16] = both[c & 1];
          tc_wait_ld();
          if (c < 3) ld_32x16(s_at + (uint32_t)(c * 16 + 16), both[(c + 1) & 1]);  // (on its way under these exponentials)
          float a0 = 0.f, a1 = 0.f;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float4 fl = st[c * 8 + e / 2];
            float e0 = ex2(fmaf(__uint_as_float(s[e]), fl.x, -fl.y)), e1 = ex2(fmaf(__uint_as_float(s[e + 1]), fl.z, -fl.w));
            if constexpr (decltype(checked)::value) {
              const int row = q0 + half * 64 + c * 16 + e;
              if (row < from || row >= rows) e0 = 0.f;
              if (row + 1 < from || row + 1 >= rows) e1 = 0.f;
            }
            a0 += e0;
            a1 += e1;
          }
          part += a0 + a1;
        }
      };
      if (ragged) tile(std::true_type{});
      else tile(std::false_type{});
      total += part;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars[W_FREE + r.slot]));
    }
    if (half) s_total[quad * 32 + lane] = total;
    bar_sync(1, 32 * PW_SOFT_WARPS);
    total += s_total[quad * 32 + lane];
    if (go && j < seen && !half) {
      if (a.segments > 1) a.part_w[((size_t)segment * units + unit) * a.t_pad + j] = total;
      else store_weight(p, unit, j, held, total);
    }
  } else if (a.segments > 1 && j0 < seen && tid < PR_KEYS) {  // (a segment of no rows)
    a.part_w[((size_t)segment * units + unit) * a.t_pad + j0 + tid] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == PW_SOFT_WARPS + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem, TMEM_COLS);
  }
}

// ------------------------------------------------------------------ host
// How the work is shared, from the sizes as the host knows them.  A CTA per item leaves slots idle where items are few or their last wave is
// half full; an equal share of all tiles per CTA costs each the start of another run, the partial sums of two and their join, about what
// eight tiles take.  8 key heads x 4 queries each, in turn: 50 rows behind 30000 507 us per item, 98 shared; 300 behind 4000 89 and 57; 500 behind
// 2000 54 and 55; 2000 behind 6000 (504 items of 47 to 63 tiles, 296 slots) 259 and 280.
struct prompt_plan {
  int ctas, segments;
  prompt_plan(int n_seqs, int m, int n_heads, int n_kv, int max_len) {
    const double slots = 2 * 148;
    const long long units = (long long)n_seqs * n_kv, rows = (long long)m * (n_heads / n_kv), blocks = (rows + PR_ROWS - 1) / PR_ROWS;
    const long long most = (max_len + PR_KEYS - 1) / PR_KEYS, least = std::max(1ll, (long long)(std::max(0, max_len - m) + PR_KEYS) / PR_KEYS);
    const double total = (double)units * blocks * (most + least) / 2, share = total / slots;
    const double items = units * blocks <= slots ? (double)most : share + most / 2.0;
    ctas = share + 8 < 0.7 * items ? (int)std::min(slots, std::max(1.0, total)) : 0;
    // weights: rows are dealt to several CTAs per 128 keys where there are fewer of those than slots
    segments = (int)std::max(1ll, std::min({16ll, blocks, (long long)slots / std::max(1ll, units * most)}));
  }
};

size_t prompt_layout(prompt_args* a, void* workspace, int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights) {
  size_t used = 0;
  auto take = [&](size_t bytes) {
    const size_t at = used;
    used += round_up(bytes, 128);
    return (uint8_t*)workspace + at;
  };
  const prompt_plan plan(n_seqs, m, n_heads, n_kv, max_len);
  const size_t units = (size_t)n_seqs * n_kv, t_pad = round_up(max_len, PR_KEYS), r_pad = round_up((size_t)m * (n_heads / n_kv), PR_ROWS);
  uint8_t* k = take(units * t_pad * hd * 2);
  uint8_t* v = take(units * t_pad * hd * 2);
  uint8_t* q = take(units * r_pad * hd * 2);
  uint8_t* stats = take(units * r_pad * sizeof(float2));
  uint8_t* bad = take(units * (t_pad / PR_KEYS) * 4 * sizeof(int));
  uint8_t* prefix = take(plan.ctas ? (units * (r_pad / PR_ROWS) + 1) * sizeof(int) : 0);
  uint8_t* part_o = take((size_t)plan.ctas * 2 * PR_ROWS * hd * sizeof(float));
  uint8_t* part_ml = take((size_t)plan.ctas * 2 * PR_ROWS * sizeof(float2));
  uint8_t* part_w = take(weights && plan.segments > 1 ? (size_t)plan.segments * units * t_pad * sizeof(float) : 0);
  if (a) {
    a->k_half = (__half*)k;
    a->v_half = (__half*)v;
    a->q_half = (__half*)q;
    a->row_stats = (float2*)stats;
    a->bad = (int*)bad;
    a->t_pad = (int)t_pad;
    a->r_pad = (int)r_pad;
    a->ctas = plan.ctas;
    a->prefix = (int*)prefix;
    a->part_o = (float*)part_o;
    a->part_ml = (float2*)part_ml;
    a->part_w = (float*)part_w;
    a->segments = plan.segments;
  }
  return used;
}

template <typename K>
int allow_smem(K* kernel, uint32_t bytes, bool (&done)[16]) {
  int dev = 0;
  LCU_CUDA(cudaGetDevice(&dev));
  if (dev >= 16 || !done[dev]) {
    LCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 16) done[dev] = true;
  }
  return LCU_OK;
}

template <typename T, int HD>
int launch_prompt(const prompt_args& a, cudaStream_t stream) {
  using sh = prompt_shape<HD>;
  const cache4_attention_params& p = a.p;
  const int units = p.c.n_seqs * p.c.n_kv, key_blocks = a.t_pad / PR_KEYS, row_blocks = a.r_pad / PR_ROWS;
  CUtensorMap map_q, map_k, map_v, map_k128;
  {
    const uint64_t rows_q[3] = {(uint64_t)HD, (uint64_t)a.r_pad, (uint64_t)units}, step_q[2] = {(uint64_t)HD * 2, (uint64_t)a.r_pad * HD * 2};
    const uint64_t rows_k[3] = {(uint64_t)HD, (uint64_t)a.t_pad, (uint64_t)units}, step_k[2] = {(uint64_t)HD * 2, (uint64_t)a.t_pad * HD * 2};
    const uint32_t box[3] = {64, 128, 1}, box_step[3] = {64, PR_STEP, 1};
    int rc = tc_encode_map(&map_q, a.q_half, 3, rows_q, step_q, box);
    if (!rc) rc = tc_encode_map(&map_k, a.k_half, 3, rows_k, step_k, box_step);
    if (!rc) rc = tc_encode_map(&map_v, a.v_half, 3, rows_k, step_k, box_step);
    if (!rc && p.weights) rc = tc_encode_map(&map_k128, a.k_half, 3, rows_k, step_k, box);
    if (rc) return rc;
  }
  prompt_expand_kernel<T, HD><<<(unsigned)units * (key_blocks + row_blocks) + (a.ctas ? 1 : 0), 256, 0, stream>>>(a, key_blocks, row_blocks);
  static bool done[2][16] = {}, done_w[16] = {};
  auto* kernel = a.ctas ? prompt_attention_kernel<T, HD, true> : prompt_attention_kernel<T, HD, false>;
  int rc = allow_smem(kernel, sh::SMEM, done[a.ctas > 0]);
  if (rc) return rc;
  LCU_CUDA(launch_after(kernel, dim3(a.ctas ? (unsigned)a.ctas : (unsigned)units * row_blocks), dim3(PR_THREADS), sh::SMEM, stream, map_q, map_k, map_v, a, row_blocks, units));
  if (a.ctas) LCU_CUDA(launch_after(prompt_join_kernel<T, HD>, dim3((unsigned)units * row_blocks * 16), dim3(256), 0, stream, a, row_blocks));
  if (p.weights) {
    constexpr uint32_t SMEM_W = 3 * sh::OPERAND + 4 * 128 * sizeof(float2) + 1024 + 256;
    rc = allow_smem(prompt_weights_kernel<HD>, SMEM_W, done_w);
    if (rc) return rc;
    LCU_CUDA(launch_after(prompt_weights_kernel<HD>, dim3((unsigned)units * key_blocks * a.segments), dim3(PW_THREADS), SMEM_W, stream, map_q, map_k128, a, key_blocks, units));
    if (a.segments > 1) LCU_CUDA(launch_after(prompt_add_kernel, dim3((p.max_len + 255) / 256, (unsigned)units), dim3(256), 0, stream, a, units));
  }
  return LCU_OK;
}

}  // namespace

bool attention_cache4_prompt_takes(int n_seqs, int m, int n_heads, int n_kv, int max_len) {
  const long long units = (long long)n_seqs * n_kv, rows = (long long)m * (n_heads / n_kv);
  return rows < (1ll << 30) && units * ((max_len + rows) / 128 + 2) * 16 < (1ll << 31) && units * (rows / 128 + 1) * (max_len / 128 + 1) < (1ll << 31);
}

size_t attention_cache4_prompt_workspace(int n_seqs, int m, int n_heads, int n_kv, int hd, int max_len, bool weights) {
  return prompt_layout(nullptr, nullptr, n_seqs, m, n_heads, n_kv, hd, max_len, weights);
}

int launch_attention_cache4_prompt(const cache4_attention_params& p, int dtype, void* workspace, cudaStream_t stream) {
  prompt_args a{};
  a.p = p;
  a.err = device_scratch_words();
  LCU_REQUIRE(a.err != nullptr, "attention_cache4: no error word");
  prompt_layout(&a, workspace, p.c.n_seqs, p.m, p.n_heads, p.c.n_kv, p.c.hd, p.max_len, p.weights != nullptr);
  if (dtype == OP_F16) return p.c.hd == 128 ? launch_prompt<__half, 128>(a, stream) : launch_prompt<__half, 64>(a, stream);
  return p.c.hd == 128 ? launch_prompt<__nv_bfloat16, 128>(a, stream) : launch_prompt<__nv_bfloat16, 64>(a, stream);
}

}  // namespace lcu
