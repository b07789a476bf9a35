// Selection over beams and vocabulary: the n best of scores[b] + log softmax(logits[b])[v] of every group of beams.
#include <cuda_bf16.h>

#include <algorithm>

#include "cache4.cuh"
#include "cache_rows.cuh"

namespace lcu {
namespace {

constexpr int BEAM_THREADS = 256, BEAM_ITEMS = 16, BEAM_CHUNK = BEAM_THREADS * BEAM_ITEMS, BEAM_GROUPS = 64, BEAM_MAX_OUT = BEAM_GROUPS;
constexpr int BEAM_MAX_CAND = 2560;  // candidates of a group that shared memory holds

struct beam_args {
  beam_params p;
  int chunks;
  float2* stats;        // [rows][chunks] maximum and sum of e^(x - maximum)
  uint64_t* best;       // [rows][chunks][n_out] order of the logit above ~token; 0 = none
};

__device__ __forceinline__ float logit_at(const float* p, size_t i) { return p[i]; }
__device__ __forceinline__ float logit_at(const __half* p, size_t i) { return __half2float(p[i]); }
__device__ __forceinline__ float logit_at(const __nv_bfloat16* p, size_t i) { return __bfloat162float(p[i]); }

__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// order of binary32 numbers as unsigned integers (-0 as 0), and back
__device__ __forceinline__ uint32_t float_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_float(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t double_order(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double order_double(uint64_t k) { return __longlong_as_double((long long)(k ^ ((k >> 63) ? 1ull << 63 : ~0ull))); }

// One CTA per (row of logits, chunk of 4096): maximum, sum of exponentials, and the chunk's n best tokens.  A logit's order and its
// token's complement make one 64-bit number that no other token has, so ties go to the lowest token by themselves.  The chunk's
// numbers lie in 64 groups of 64 (four lanes' sixteen); the n-th largest of the groups' largest is no more than the n-th largest of all, and
// at most n groups hold numbers from it on: 64 n candidates at most, little more than n as a rule, whose ranks are counted.  (Counting
// the ranks of 256 threads' largest in every thread took 15 of 35 us at 64 rows of 128000.)
template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) beam_rows_kernel(const beam_args a) {
  extern __shared__ uint64_t cand[];  // [n_out * 64]
  __shared__ uint64_t tops[BEAM_GROUPS];
  __shared__ float s_max[8];
  __shared__ double s_sum[8];
  __shared__ uint64_t s_threshold;
  __shared__ int s_count;
  pdl_launch_dependents();
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_out = a.p.n_out, v0 = chunk * BEAM_CHUNK;
  const T* x = reinterpret_cast<const T*>(a.p.logits) + (size_t)row * a.p.ld;
  if (tid == 0) {
    s_count = 0;
    s_threshold = 0;
  }
  const bool full = v0 + BEAM_CHUNK <= a.p.n_vocab;
  float val[BEAM_ITEMS];
#pragma unroll
  for (int i = 0; i < BEAM_ITEMS; ++i) {
    const int v = v0 + i * BEAM_THREADS + tid;
    val[i] = full || v < a.p.n_vocab ? logit_at(x, v) : -INFINITY;
  }
  // the thread's largest and its first place, by comparing numbers; orders are formed for that one alone
  float mx = -INFINITY;
  int at = 0;
#pragma unroll
  for (int i = 0; i < BEAM_ITEMS; ++i) {
    if (val[i] != val[i]) val[i] = -INFINITY;  // no number: never chosen before one
    if (val[i] > mx) {
      mx = val[i];
      at = i;
    }
  }
  uint64_t top = v0 + at * BEAM_THREADS + tid < a.p.n_vocab ? (uint64_t)float_order(mx) << 32 | (uint32_t)~(v0 + at * BEAM_THREADS + tid) : 0ull;
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if ((lane & 3) == 0) tops[tid >> 2] = top;
  mx = warp_max(mx);
  if (lane == 0) s_max[warp] = mx;
  __syncthreads();
  mx = s_max[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) mx = fmaxf(mx, s_max[w]);
  if (tid < BEAM_GROUPS) {
    const uint64_t mine = tops[tid];
    int rank = 0;
#pragma unroll 8
    for (int t = 0; t < BEAM_GROUPS; ++t) rank += tops[t] > mine;
    if (mine && rank == n_out - 1) s_threshold = mine;
  }
  double sum = 0.0;
  if (mx > -INFINITY) {
    // The difference first: it is at most 0 and overflows to minus infinity at worst, the largest term is 1 whatever the maximum, and a term
    // is off by 2^-22, and by 2.25 x 2^-24 of its distance from the maximum.
    constexpr float LOG2E = 1.4426950408889634f;
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < BEAM_ITEMS; ++i) part += ex2((val[i] - mx) * LOG2E);
    sum = part;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < 8; ++w) s += s_sum[w];
    a.stats[(size_t)row * a.chunks + chunk] = make_float2(mx, (float)s);
  }
  const uint64_t threshold = s_threshold;
  if (top >= threshold) {  // (others' groups hold none)
    const float bound = threshold ? order_float((uint32_t)(threshold >> 32)) : -INFINITY;
#pragma unroll
    for (int i = 0; i < BEAM_ITEMS; ++i) {
      if (val[i] < bound) continue;
      const int v = v0 + i * BEAM_THREADS + tid;
      const uint64_t k = (uint64_t)float_order(val[i]) << 32 | (uint32_t)~v;
      if (v < a.p.n_vocab && k >= threshold) cand[atomicAdd(&s_count, 1)] = k;
    }
  }
  __syncthreads();
  const int count = s_count;
  uint64_t* best = a.best + ((size_t)row * a.chunks + chunk) * n_out;
  for (int c = tid; c < count; c += BEAM_THREADS) {
    const uint64_t k = cand[c];
    int r = 0;
    for (int t = 0; t < count; ++t) r += cand[t] > k;
    if (r < n_out) best[r] = k;
  }
  for (int r = count + tid; r < n_out; r += BEAM_THREADS) best[r] = 0;
}

struct scored {
  uint64_t order;   // of the score in 64 bits; 0: nothing
  uint64_t place;   // beam, complement of the logit's order, token: logits whose difference 64 bits of a score lose keep the order of their list
};
__device__ __forceinline__ int beam_of(uint64_t place) { return (int)(place >> 56); }
__device__ __forceinline__ int token_of(uint64_t place) { return (int)(place & 0xffffffu); }
__device__ __forceinline__ bool better(const scored& a, const scored& b) { return a.order > b.order || (a.order == b.order && a.place < b.place); }

// One CTA per group: every beam's maximum and the logarithm of its sum (of the chunks' binary32 sums, in 64 bits), then the n best of the
// chunks' candidates.  The two stay apart, so that a score is as good behind a maximum of 1e30 as behind one of 0.  A thread owns chunks' lists, which are
// sorted: the heads of 64 groups of lists give a bound in the way of the first kernel, and lists are walked down to it.
__global__ void __launch_bounds__(BEAM_THREADS) beam_group_kernel(const beam_args a, int most) {
  __shared__ double top_logit[MAX_BEAMS], base[MAX_BEAMS];  // (base: score so far less the logarithm of the sum)
  __shared__ scored tops[BEAM_THREADS];  // (the largest of four threads' lists each; of every thread in the other way)
  __shared__ scored s_threshold;
  __shared__ int s_count;
  extern __shared__ scored cand_scored[];
  const int group = blockIdx.x, tid = threadIdx.x, n_out = a.p.n_out;
  pdl_launch_dependents();  // (the reordering of the caches, where that comes next)
  pdl_wait();
  if (tid == 0) {
    s_count = 0;
    s_threshold = scored{0, ~0ull};
  }
  for (int b = tid >> 5; b < a.p.beams; b += BEAM_THREADS / 32) {
    const float2* st = a.stats + ((size_t)group * a.p.beams + b) * a.chunks;
    float mx = -INFINITY;
    for (int c = tid & 31; c < a.chunks; c += 32) mx = fmaxf(mx, st[c].x);
    mx = warp_max(mx);
    double sum = 0.0;
    if (mx > -INFINITY && mx < INFINITY)
      for (int c = tid & 31; c < a.chunks; c += 32) sum += (double)(st[c].y * expf(st[c].x - mx));  // (2^-22 of a chunk's sum, as that is)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) {
      const float s = a.p.scores[(size_t)group * a.p.beams + b];
      // a beam without a finite score, or whose logits have no finite maximum, offers its first tokens at minus infinity
      const bool fine = mx > -INFINITY && mx < INFINITY && s > -INFINITY && s < INFINITY;
      top_logit[b] = mx;
      base[b] = fine ? (double)s - log(sum) : -INFINITY;
    }
  }
  __syncthreads();
  const int lists = a.p.beams * a.chunks;
  // entry e of a list (sorted, best first); a beam at minus infinity has one list of its first tokens
  auto at = [&](int list, int e) {
    const int b = list / a.chunks;
    const uint64_t k = a.best[((size_t)group * lists + list) * n_out + e];
    const bool fine = base[b] != -INFINITY;
    if (fine ? !k : list != b * a.chunks || e >= a.p.n_vocab) return scored{0, ~0ull};
    if (!fine) return scored{double_order(-INFINITY), (uint64_t)b << 56 | (uint32_t)e};
    const uint32_t logit = (uint32_t)(k >> 32);
    return scored{double_order(((double)order_float(logit) - top_logit[b]) + base[b]), (uint64_t)b << 56 | (uint64_t)~logit << 24 | (uint32_t)~(uint32_t)k};
  };
  scored top{0, ~0ull};
#pragma unroll 4
  for (int l = tid; l < lists; l += BEAM_THREADS) {
    const scored s = at(l, 0);
    if (better(s, top)) top = s;
  }
  // (few lists: each a group of its own, the bound is closer then)
  const int width = lists <= BEAM_GROUPS ? 1 : BEAM_THREADS / BEAM_GROUPS;
  if (width > 1) {
#pragma unroll
    for (int o = 1; o < BEAM_THREADS / BEAM_GROUPS; o <<= 1) {
      const scored other{__shfl_xor_sync(0xffffffffu, top.order, o), __shfl_xor_sync(0xffffffffu, top.place, o)};
      if (better(other, top)) top = other;
    }
  }
  if (tid % width == 0 && tid / width < BEAM_GROUPS) tops[tid / width] = top;
  __syncthreads();
  const int groups = width > 1 ? BEAM_GROUPS : lists;
  if (tid < groups && tops[tid].order) {
    const scored mine = tops[tid];
    int rank = 0;
#pragma unroll 8
    for (int t = 0; t < groups; ++t) rank += better(tops[t], mine);
    if (rank == n_out - 1) s_threshold = mine;
  }
  __syncthreads();
  const scored threshold = s_threshold;
  for (int l = tid; l < lists; l += BEAM_THREADS)
    for (int e = 0; e < n_out; ++e) {
      const scored s = at(l, e);
      if (!s.order || better(threshold, s)) break;
      const int place = atomicAdd(&s_count, 1);
      if (place < most) cand_scored[place] = s;
    }
  __syncthreads();
  const int count = s_count;
  if (count > most) {
    // (thousands above the bound, as where one beam's chunk holds nothing and the others' threads everything: one after another)
    scored last{~0ull, 0ull};
    for (int r = 0; r < n_out; ++r) {
      scored best{0, ~0ull};
      for (int l = tid; l < lists; l += BEAM_THREADS)
        for (int e = 0; e < n_out; ++e) {
          const scored s = at(l, e);
          if (!s.order || !better(s, best)) break;
          if (better(last, s)) {
            best = s;
            break;
          }
        }
      __syncthreads();
      tops[tid] = best;
      __syncthreads();
      for (int t = 0; t < BEAM_THREADS; ++t)
        if (better(tops[t], best)) best = tops[t];
      if (tid == 0) {
        const size_t o = (size_t)group * n_out + r;
        a.p.parents[o] = beam_of(best.place);
        a.p.tokens[o] = token_of(best.place);
        a.p.scores_out[o] = (float)order_double(best.order);
      }
      last = best;
    }
    return;
  }
  for (int c = tid; c < count; c += BEAM_THREADS) {
    const scored s = cand_scored[c];
    int r = 0;
    for (int t = 0; t < count; ++t) r += better(cand_scored[t], s);
    if (r < n_out) {
      const size_t o = (size_t)group * n_out + r;
      a.p.parents[o] = beam_of(s.place);
      a.p.tokens[o] = token_of(s.place);
      a.p.scores_out[o] = (float)order_double(s.order);
    }
  }
}

int beam_chunks(int n_vocab) { return (int)ceil_div((size_t)n_vocab, BEAM_CHUNK); }

}  // namespace

size_t beam_select_workspace(int n_groups, int beams, int n_vocab, int n_out) {
  if (beams > MAX_BEAMS || n_vocab > (1 << 24) || n_out > BEAM_MAX_OUT) return 0;  // (such a call is refused)
  return (size_t)n_groups * beams * beam_chunks(n_vocab) * (sizeof(float2) + (size_t)n_out * sizeof(uint64_t));
}

int launch_beam_select(const beam_params& p, int dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  LCU_REQUIRE(p.parents && p.tokens && p.scores_out && p.logits && p.scores, "beam_select: a null pointer");
  LCU_REQUIRE(words_aligned(p.parents, p.tokens, p.scores_out, p.scores), "beam_select: parents, tokens and scores must be 4-byte aligned");
  LCU_REQUIRE(dtype == OP_F16 || dtype == OP_BF16 || dtype == OP_F32, "beam_select: number format %d is not 0 (half), 1 (bfloat16) or 2 (binary32)", dtype);
  LCU_REQUIRE(p.n_groups >= 1 && p.beams >= 1 && p.beams <= MAX_BEAMS, "beam_select: %d groups of %d beams (1 to %d)", p.n_groups, p.beams, MAX_BEAMS);
  LCU_REQUIRE(p.n_vocab >= 1 && p.n_vocab <= (1 << 24) && p.ld >= p.n_vocab, "beam_select: a vocabulary of %d in rows of %d", p.n_vocab, p.ld);
  LCU_REQUIRE(p.n_out >= 1 && p.n_out <= BEAM_MAX_OUT && p.n_out <= (long long)p.beams * p.n_vocab, "beam_select: %d continuations (1 to %d, and no more than there are)", p.n_out,
              BEAM_MAX_OUT);
  LCU_REQUIRE(((uintptr_t)p.logits & (dtype == OP_F32 ? 3 : 1)) == 0, "beam_select: logits must be aligned to their type");
  const int chunks = beam_chunks(p.n_vocab);
  const size_t rows = (size_t)p.n_groups * p.beams, need = beam_select_workspace(p.n_groups, p.beams, p.n_vocab, p.n_out);
  LCU_REQUIRE(rows * chunks < (1ull << 31), "beam_select: too many rows of logits");
  LCU_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0, "beam_select: %zu bytes of 16-byte aligned workspace are needed, %zu are there", need,
              workspace ? workspace_bytes : (size_t)0);
  const int most = (int)std::min<size_t>(BEAM_MAX_CAND, (size_t)p.beams * chunks * p.n_out);
  if (int rc_dev = need_device()) return rc_dev;
  beam_args a{p, chunks, (float2*)workspace, (uint64_t*)((float2*)workspace + rows * chunks)};
  const unsigned ctas = (unsigned)(rows * chunks);
  const size_t smem_rows = (size_t)p.n_out * (BEAM_CHUNK / BEAM_GROUPS) * sizeof(uint64_t);  // (up to 32 KiB)
  if (dtype == OP_F16) beam_rows_kernel<__half><<<ctas, BEAM_THREADS, smem_rows, stream>>>(a);
  else if (dtype == OP_BF16) beam_rows_kernel<__nv_bfloat16><<<ctas, BEAM_THREADS, smem_rows, stream>>>(a);
  else beam_rows_kernel<float><<<ctas, BEAM_THREADS, smem_rows, stream>>>(a);
  LCU_CUDA(launch_after(beam_group_kernel, dim3(p.n_groups), dim3(BEAM_THREADS), (size_t)most * sizeof(scored), stream, a, most));
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

}  // namespace lcu
