// Eviction of cached rows by the attention weight they received, and reordering of the caches of a group of beams.
#include "cache_rows.cuh"
#include "cache4.cuh"

#include <algorithm>

namespace lcu {
namespace {

// order of binary32 weights as unsigned integers; -0 counts as 0, a NaN as less than everything
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t b = __float_as_uint(w + 0.f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int SEL_THREADS = 1024, SEL_BINS = 2048;

struct select_args {
  const float* weights;
  int* kept;
  const int* lengths;
  int n_kv, ctx, keep, recent;
};

// exclusive sums over the CTA's threads of two counts at once (below 2^31 each), in thread order
__device__ __forceinline__ int2 block_exclusive(int2 v, int2* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) {
      x.x += a;
      x.y += b;
    }
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int2 t = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, t.x, o), b = __shfl_up_sync(0xffffffffu, t.y, o);
      if (lane >= o) {
        t.x += a;
        t.y += b;
      }
    }
    s_warp[lane] = t;
  }
  __syncthreads();
  const int2 before = warp ? s_warp[warp - 1] : make_int2(0, 0);
  __syncthreads();
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// int2 of the same place in shared memory of another CTA of the cluster
__device__ __forceinline__ int2 remote_pair(const void* at, uint32_t rank) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(mapa(smem_u32(at), rank)) : "memory");
  return v;
}

// One cluster of CL CTAs per (sequence, head): the `want` largest of the weights before the latest rows, by digits from the top - a histogram of
// 2048 bins, the bin in which the want-th largest lies, the next digit among that bin's weights - then one pass in row order that
// writes the rows above the threshold and as many of those at it as are left to take, lowest rows first.  A warp owns a run of rows; up
// to 16 weights of a thread stay in registers, so that they are read once.  Bound by the chain of three histograms and their sums over the
// bins.  Four CTAs share a head where rows are many: every CTA adds up the four histograms for itself and finds the same bin, and a CTA's
// places begin behind the counts of those before it.  One CTA / four, us with the rows' move: 8 heads x 16000 rows 17.7 / 13.9, 32 heads (to
// 8001) 61.0 / 56.4, 64 heads 23.2 / 30.1; 32 heads x 5000 13.3 / 15.9; 8 heads x 60000 75.6 / 21.4, 64 heads 101 / 43.
template <int K, int CL>
__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const select_args a) {
  __shared__ __align__(8) int hist_of[CL > 1 ? 2 : 1][SEL_BINS];  // (two in turn: others read the last one while the next is filled)
  __shared__ int2 s_total;
  __shared__ int2 s_warp[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  pdl_launch_dependents();  // (the kernels that move rows start, and wait for the list)
  const int sh = blockIdx.x / CL, rank = blockIdx.x % CL, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = min(a.lengths[sh / a.n_kv], a.ctx);
  int* kept = a.kept + (size_t)sh * a.keep;
  if (len <= a.keep) {
    for (int i = rank * SEL_THREADS + tid; i < a.keep; i += CL * SEL_THREADS) kept[i] = i < len ? i : -1;
    return;  // (the whole cluster)
  }
  const int old = len - a.recent, want = a.keep - a.recent;  // (len > keep: want < old)
  const float* w = a.weights + (size_t)sh * a.ctx;
  // the rows of a warp; a thread's are 32 apart
  const int run = (old + CL * SEL_THREADS - 1) / (CL * SEL_THREADS) * 32, from = (rank * (SEL_THREADS / 32) + warp) * run, to = min(old, from + run);
  uint32_t held[K > 0 ? K : 1];
  if constexpr (K > 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = from + k * 32 + lane;
      held[k] = i < to ? weight_key(w[i]) : 0u;
    }
  }
  // each(f): f(row, its key, whether there is such a row) for the thread's rows, whole warps together
  auto each = [&](auto&& f) {
    if constexpr (K > 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (from + k * 32 >= to) break;
        f(from + k * 32 + lane, held[k], from + k * 32 + lane < to);
      }
    } else {
      for (int i0 = from; i0 < to; i0 += 4 * 32) {
        float next[4];  // (requested together)
#pragma unroll
        for (int k = 0; k < 4; ++k) next[k] = i0 + k * 32 + lane < to ? w[i0 + k * 32 + lane] : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i0 + k * 32 < to) f(i0 + k * 32 + lane, weight_key(next[k]), i0 + k * 32 + lane < to);
      }
    }
  };
  for (int i = rank * SEL_THREADS + tid; i < a.recent; i += CL * SEL_THREADS) kept[want + i] = old + i;
  if (want == 0) return;
  if (tid == 0) {
    s_prefix = 0;
    s_left = want;
  }
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    int* hist = hist_of[CL > 1 ? pass & 1 : 0];
    for (int b = tid; b < SEL_BINS; b += SEL_THREADS) hist[b] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    const int left = s_left;
    each([&](int, uint32_t key, bool there) {
      const bool in = there && (pass == 0 || (key >> (shift + bits)) == prefix);
      if (pass && !__any_sync(0xffffffffu, in)) return;  // (most of a later pass)
      const uint32_t digit = in ? (key >> shift) & ((1u << bits) - 1) : 0xffffffffu;
      int same = 0;
      __match_all_sync(0xffffffffu, digit, &same);  // (equal weights, all zero before the first step: one add instead of 32 on one address)
      if (same) {
        if (lane == 0 && in) atomicAdd(&hist[digit], 32);
      } else if (in) {
        atomicAdd(&hist[digit], 1);
      }
    });
    if constexpr (CL > 1) cluster_sync();
    else __syncthreads();
    // bins from the top, two per thread
    const int hi = SEL_BINS - 1 - 2 * tid;
    int c0 = 0, c1 = 0;
    if constexpr (CL > 1) {
#pragma unroll
      for (int r = 0; r < CL; ++r) {
        const int2 c = remote_pair(&hist[hi - 1], r);
        c0 += c.y;
        c1 += c.x;
      }
    } else {
      c0 = hist[hi];
      c1 = hist[hi - 1];
    }
    const int before = block_exclusive(make_int2(c0 + c1, 0), s_warp).x;
    if (before < left && left <= before + c0 + c1) {
      const bool first = left <= before + c0;
      s_prefix = (prefix << bits) | (uint32_t)(first ? hi : hi - 1);
      s_left = left - before - (first ? 0 : c0);
    }
    __syncthreads();
  }
  const uint32_t threshold = s_prefix;
  const int ties = s_left;
  // counts of the warps, their sums over the warps before, places
  int above = 0, equal = 0;
  each([&](int, uint32_t key, bool there) {
    above += __popc(__ballot_sync(0xffffffffu, there && key > threshold));
    equal += __popc(__ballot_sync(0xffffffffu, there && key == threshold));
  });
  int2 base = block_exclusive(lane == 0 ? make_int2(above, equal) : make_int2(0, 0), s_warp);
  if constexpr (CL > 1) {
    if (tid == SEL_THREADS - 1) s_total = base;  // (lane 31 adds nothing: the sums of all warps)
    cluster_sync();
#pragma unroll
    for (int r = 0; r + 1 < CL; ++r) {
      const int2 c = remote_pair(&s_total, r);
      if (r < rank) {
        base.x += c.x;
        base.y += c.y;
      }
    }
    cluster_sync();  // (nothing of this CTA's is read any more)
  }
  base.x = __shfl_sync(0xffffffffu, base.x, 0);
  base.y = __shfl_sync(0xffffffffu, base.y, 0);
  each([&](int i, uint32_t key, bool there) {
    const uint32_t mine = (1u << lane) - 1;
    const uint32_t m_above = __ballot_sync(0xffffffffu, there && key > threshold), m_equal = __ballot_sync(0xffffffffu, there && key == threshold);
    const int tie = base.y + __popc(m_equal & mine);
    if (there && (key > threshold || (key == threshold && tie < ties))) kept[base.x + __popc(m_above & mine) + min(tie, ties)] = i;
    base.x += __popc(m_above);
    base.y += __popc(m_equal);
  });
}

struct plane {
  uint8_t* dst;
  const uint8_t* src;
  int row_bytes;
};
struct gather_args {
  plane planes[MAX_CACHE_PLANES];
  const int* kept;
  int* lengths_out;
  const int* lengths;
  int n_seqs, n_kv, ctx, dst_ctx, keep;
};

template <typename V>
__device__ __forceinline__ void copy_unit(uint8_t* dst, const uint8_t* src, size_t at, size_t from) {
  reinterpret_cast<V*>(dst)[at] = reinterpret_cast<const V*>(src)[from];
}

// widest units that rows of this many bytes at these addresses are made of
__device__ __forceinline__ int unit_bytes(const plane& p) {
  const uintptr_t all = (uintptr_t)p.dst | (uintptr_t)p.src | (uintptr_t)p.row_bytes;
  return (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
}

template <typename V>
__device__ __forceinline__ void gather_rows(const gather_args& a, const plane& p, int sh, int first, int last) {
  constexpr int UNROLL = 2;
  const int units = p.row_bytes / (int)sizeof(V);
  const int* kept = a.kept + (size_t)sh * a.keep;
  const V* src = reinterpret_cast<const V*>(p.src) + (size_t)sh * a.ctx * units;
  V* dst = reinterpret_cast<V*>(p.dst) + (size_t)sh * a.dst_ctx * units;
  // unit u of row r; the next of this thread is 256 units on (no division on the way: it took a third of the time)
  const int rows_on = 256 / units, units_on = 256 - rows_on * units;
  int r = (int)threadIdx.x / units, u = (int)threadIdx.x - r * units;
  for (r += first; r < last;) {
    V v[UNROLL];
    int to[UNROLL];
    size_t at[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int from = r < last ? kept[r] : -1;
      to[k] = from;
      at[k] = (size_t)r * units + u;
      if (from >= 0) v[k] = src[(size_t)from * units + u];
      r += rows_on;
      u += units_on;
      if (u >= units) {
        u -= units;
        ++r;
      }
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (to[k] >= 0) dst[at[k]] = v[k];
  }
}

// by one CTA of the kernels that move rows, which go by the list of kept ones: lengths_out may be lengths
__device__ __forceinline__ void write_lengths(const gather_args& a) {
  if (a.lengths_out)
    for (int s = threadIdx.x; s < a.n_seqs; s += blockDim.x) a.lengths_out[s] = min(min(a.lengths[s], a.ctx), a.keep);
}
__global__ void __launch_bounds__(256) evict_lengths_kernel(const gather_args a) { write_lengths(a); }

// Rows into other planes: a CTA per (sequence, head, run of kept rows); bound by memory.
__global__ void __launch_bounds__(256) evict_gather_kernel(const gather_args a, int rows_per_cta, int chunks) {
  const plane p = a.planes[blockIdx.y];
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0) write_lengths(a);
  const int sh = blockIdx.x / chunks, first = (blockIdx.x % chunks) * rows_per_cta, last = min(a.keep, first + rows_per_cta);
  switch (unit_bytes(p)) {
    case 16: gather_rows<uint4>(a, p, sh, first, last); break;
    case 8: gather_rows<uint2>(a, p, sh, first, last); break;
    case 4: gather_rows<uint32_t>(a, p, sh, first, last); break;
    default: gather_rows<uint16_t>(a, p, sh, first, last); break;
  }
}

// Rows to the front of the same plane.  Kept rows only move down and stay in order, so row i may be written once every row up to the
// i-th kept one has been read: a CTA walks a column of a head's rows in steps, reads a step, waits, writes it.  A step's targets lie
// below every later step's sources.  Columns of 32 bytes (a sector) are independent: they are what runs side by side.  Bound by the chain of
// steps of a column where heads are few: the five planes of a 4-bit cache (rows of 64, 8, 64, 8 and 4 bytes) of 4 x 8 heads, 16000 to 8001 rows, take 73 us,
// 12 of them the selection, for 12 us of bytes; 16 x 8 heads 136 for 48; 32 heads, 2048 to 1024 12.0 for 1.5.
constexpr int MOVE_UNROLL = 8;
template <typename V>
__device__ __forceinline__ void move_rows(const gather_args& a, const plane& p, int sh, int col, int col_units) {
  const int units = p.row_bytes / (int)sizeof(V);
  const int* kept = a.kept + (size_t)sh * a.keep;
  V* plane_at = reinterpret_cast<V*>(p.dst) + (size_t)sh * a.ctx * units + col;
  const int mine = min(col_units, units - col), n = a.keep * mine;
  for (int t0 = 0; t0 < n; t0 += 256 * MOVE_UNROLL) {
    V v[MOVE_UNROLL];
    int from[MOVE_UNROLL];
#pragma unroll
    for (int u = 0; u < MOVE_UNROLL; ++u) {
      const int t = t0 + u * 256 + (int)threadIdx.x;
      from[u] = t < n ? kept[t / mine] : -1;
      if (from[u] >= 0) v[u] = plane_at[(size_t)from[u] * units + t % mine];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MOVE_UNROLL; ++u) {
      const int t = t0 + u * 256 + (int)threadIdx.x;
      if (from[u] >= 0) plane_at[(size_t)(t / mine) * units + t % mine] = v[u];
    }
  }
}
__global__ void __launch_bounds__(256) evict_move_kernel(const gather_args a) {
  const plane p = a.planes[blockIdx.y];
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) write_lengths(a);
  const int sh = blockIdx.x, unit = unit_bytes(p), col_units = max(1, 32 / unit), col = blockIdx.z * col_units;
  if (col >= p.row_bytes / unit) return;
  switch (unit) {
    case 16: move_rows<uint4>(a, p, sh, col, col_units); break;
    case 8: move_rows<uint2>(a, p, sh, col, col_units); break;
    case 4: move_rows<uint32_t>(a, p, sh, col, col_units); break;
    default: move_rows<uint16_t>(a, p, sh, col, col_units); break;
  }
}

struct reorder_args {
  plane planes[MAX_CACHE_PLANES];
  const int* parents;
  const int* lengths;
  int n_groups, beams, n_kv, ctx;
};

// rows [0, length) of one head of the parent: one run of bytes, in 16-byte pieces (2-byte ones where addresses do not allow that)
__device__ __forceinline__ size_t piece_bytes(const plane& p, int ctx) {
  return (((uintptr_t)p.dst | (uintptr_t)p.src | (uintptr_t)((size_t)ctx * p.row_bytes)) & 15) == 0 ? 16 : 2;
}

// Into other planes: a CTA per (sequence, head, piece of the run).
constexpr size_t REORDER_CTA_BYTES = 16384;
__global__ void __launch_bounds__(256) reorder_copy_kernel(const reorder_args a, int chunks) {
  const plane p = a.planes[blockIdx.y];
  pdl_wait();
  const int chunk = blockIdx.x % chunks, sh = blockIdx.x / chunks, seq = sh / a.n_kv, head = sh % a.n_kv;
  const int parent = a.parents[seq];
  if (parent < 0 || parent >= a.beams) return;
  const int from = seq / a.beams * a.beams + parent;
  const size_t head_bytes = (size_t)a.ctx * p.row_bytes, run = (size_t)max(0, min(a.lengths[from], a.ctx)) * p.row_bytes;
  const size_t lo = (size_t)chunk * REORDER_CTA_BYTES, hi = min(run, lo + REORDER_CTA_BYTES);
  if (lo >= hi) return;
  const uint8_t* src = p.src + ((size_t)from * a.n_kv + head) * head_bytes;
  uint8_t* dst = p.dst + (size_t)sh * head_bytes;
  size_t done = lo;
  if (piece_bytes(p, a.ctx) == 16) {
    constexpr int UNROLL = 4;
    const int n = (int)((hi - lo) / 16);
    const uint4* s = reinterpret_cast<const uint4*>(src + lo);
    uint4* d = reinterpret_cast<uint4*>(dst + lo);
    for (int t0 = threadIdx.x; t0 < n; t0 += 256 * UNROLL) {
      uint4 v[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (t0 + u * 256 < n) v[u] = s[t0 + u * 256];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (t0 + u * 256 < n) d[t0 + u * 256] = v[u];
    }
    done = lo + (size_t)n * 16;
  }
  for (size_t b = done + 2 * threadIdx.x; b < hi; b += 512) *reinterpret_cast<uint16_t*>(dst + b) = *reinterpret_cast<const uint16_t*>(src + b);
}

// In place: a thread owns one place in all beams of a group, reads what every beam takes there and then writes.  The five planes of a 4-bit
// cache: 8 x 4 beams, 8 heads x 1000 rows 15.8 us for 8.7 of bytes, 4 x 16 beams, 4 x 500 13.8 for 5.5, 4 beams, 32 heads x 16000 92 for 62.
template <typename V, int B>
__device__ __forceinline__ void permute_run(const reorder_args& a, const plane& p, int group, int head, size_t lo, size_t hi) {
  const size_t head_units = (size_t)a.ctx * p.row_bytes / sizeof(V), seq_units = head_units * a.n_kv;
  V* base = reinterpret_cast<V*>(p.dst) + (size_t)group * a.beams * seq_units + head * head_units;
  for (size_t t = lo / sizeof(V) + threadIdx.x; t < hi / sizeof(V); t += 256) {
    V v[B];
    bool take[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int parent = b < a.beams ? a.parents[group * a.beams + b] : -1;
      take[b] = parent >= 0 && parent < a.beams && parent != b;
      if (take[b]) take[b] = (long long)(t + 1) * (long long)sizeof(V) <= (long long)max(0, min(a.lengths[group * a.beams + parent], a.ctx)) * p.row_bytes;
      if (take[b]) v[b] = base[parent * seq_units + t];
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (take[b]) base[b * seq_units + t] = v[b];
  }
}
template <int B>
__global__ void __launch_bounds__(256) reorder_permute_kernel(const reorder_args a, int chunks) {
  const plane p = a.planes[blockIdx.y];
  pdl_wait();
  const int chunk = blockIdx.x % chunks, gh = blockIdx.x / chunks, group = gh / a.n_kv, head = gh % a.n_kv;
  const size_t head_bytes = (size_t)a.ctx * p.row_bytes, lo = (size_t)chunk * REORDER_CTA_BYTES / 4, hi = min(head_bytes, lo + REORDER_CTA_BYTES / 4);
  if (lo >= hi) return;
  // (rows of 16 bytes or a multiple: whole pieces; a run that may end inside a piece goes in 2-byte ones)
  if (piece_bytes(p, a.ctx) == 16 && p.row_bytes % 16 == 0) permute_run<uint4, B>(a, p, group, head, lo, hi);
  else if (p.row_bytes % 4 == 0 && (((uintptr_t)p.dst) & 3) == 0) permute_run<uint32_t, B>(a, p, group, head, lo, hi);
  else permute_run<uint16_t, B>(a, p, group, head, lo, hi);
}

// `src_rows`, `dst_rows`: of a whole plane.  Planes are moved by separate CTAs in any order: a destination that another plane reads or writes would be a
// race.  (Only where a plane goes to others and is moved in place too, the copies come first.)
int check_overlaps(const char* who, void* const* dst, const void* const* src, const int* row_bytes, int n, unsigned long long dst_rows, unsigned long long src_rows) {
  auto apart = [](const void* a, unsigned __int128 na, const void* b, unsigned __int128 nb) {  // (2^51 rows of 2^16 bytes at most)
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y ? y - x >= na : x - y >= nb;
  };
  for (int i = 0; i < n; ++i)
    for (int j = 0; j < n; ++j) {
      const unsigned __int128 to = (unsigned __int128)dst_rows * row_bytes[i];
      LCU_REQUIRE(i <= j || apart(dst[i], to, dst[j], (unsigned __int128)dst_rows * row_bytes[j]), "%s: the destinations of planes %d and %d overlap", who, j, i);
      LCU_REQUIRE(dst[i] == src[i] || apart(dst[i], to, src[j], (unsigned __int128)src_rows * row_bytes[j]), "%s: the destination of plane %d overlaps the source of plane %d", who, i, j);
    }
  return LCU_OK;
}

int check_planes(const char* who, void* const* dst, const void* const* src, const int* row_bytes, int n) {
  LCU_REQUIRE(n >= 1 && n <= MAX_CACHE_PLANES && dst && src && row_bytes, "%s: %d planes (1 to %d)", who, n, MAX_CACHE_PLANES);
  for (int i = 0; i < n; ++i) {
    LCU_REQUIRE(dst[i] && src[i], "%s: plane %d is a null pointer", who, i);
    LCU_REQUIRE(row_bytes[i] >= 2 && row_bytes[i] % 2 == 0 && row_bytes[i] <= 65536, "%s: rows of %d bytes (even, up to 65536)", who, row_bytes[i]);
    LCU_REQUIRE((((uintptr_t)dst[i] | (uintptr_t)src[i]) & 1) == 0, "%s: plane %d is at an odd address", who, i);
  }
  return LCU_OK;
}

}  // namespace

int launch_cache_evict(const evict_params& p, cudaStream_t stream) {
  if (p.n_planes) {
    int rc = check_planes("cache_evict", p.dst, p.src, p.row_bytes, p.n_planes);
    if (rc) return rc;
  }
  LCU_REQUIRE(p.weights && p.kept && p.lengths, "cache_evict: a null pointer");
  LCU_REQUIRE(words_aligned(p.weights, p.kept, p.lengths, p.lengths_out), "cache_evict: weights, lengths and the list must be 4-byte aligned");
  LCU_REQUIRE(p.n_seqs >= 1 && p.n_kv >= 1 && (long long)p.n_seqs * p.n_kv < (1 << 20) && p.ctx >= 1 && p.ctx < (1 << 26), "cache_evict: %d sequences of %d heads of %d rows", p.n_seqs,
              p.n_kv, p.ctx);
  LCU_REQUIRE(p.keep >= 1 && p.keep <= p.dst_ctx && p.keep <= p.ctx && p.recent >= 0 && p.recent <= p.keep,
              "cache_evict: keep %d rows (%d of them the latest) of %d into %d", p.keep, p.recent, p.ctx, p.dst_ctx);
  const int heads = p.n_seqs * p.n_kv;
  if (int rc = check_overlaps("cache_evict", p.dst, p.src, p.row_bytes, p.n_planes, (unsigned long long)heads * p.dst_ctx, (unsigned long long)heads * p.ctx)) return rc;
  gather_args away{}, here{};
  int n_away = 0, n_here = 0, widest_away = 0, widest_here = 0;
  for (int i = 0; i < p.n_planes; ++i) {
    const plane pl{(uint8_t*)p.dst[i], (const uint8_t*)p.src[i], p.row_bytes[i]};
    if (p.dst[i] == p.src[i]) {
      LCU_REQUIRE(p.dst_ctx == p.ctx, "cache_evict: a plane compacted in place keeps its %d rows (not %d)", p.ctx, p.dst_ctx);
      here.planes[n_here++] = pl;
      widest_here = std::max(widest_here, pl.row_bytes);
    } else {
      away.planes[n_away++] = pl;
      widest_away = std::max(widest_away, pl.row_bytes);
    }
  }
  for (gather_args* g : {&away, &here}) {
    g->kept = p.kept;
    g->lengths = p.lengths;
    g->n_seqs = p.n_seqs;
    g->n_kv = p.n_kv;
    g->ctx = p.ctx;
    g->dst_ctx = p.dst_ctx;
    g->keep = p.keep;
  }
  const int rows = std::max(1, 16384 / std::max(1, widest_away)), chunks = (p.keep + rows - 1) / rows;
  LCU_REQUIRE((long long)heads * chunks < (1ll << 31), "cache_evict: planes are too large");
  if (int rc_dev = need_device()) return rc_dev;
  const select_args sel{p.weights, p.kept, p.lengths, p.n_kv, p.ctx, p.keep, p.recent};
  if (p.ctx <= 4 * SEL_THREADS) {
    evict_select_kernel<4, 1><<<heads, SEL_THREADS, 0, stream>>>(sel);
  } else if (p.ctx <= 8 * SEL_THREADS || (p.ctx <= 16 * SEL_THREADS && 4 * heads > 148)) {
    evict_select_kernel<16, 1><<<heads, SEL_THREADS, 0, stream>>>(sel);
  } else {
    auto* kernel = p.ctx <= 16 * SEL_THREADS ? evict_select_kernel<4, 4> : p.ctx <= 64 * SEL_THREADS ? evict_select_kernel<16, 4> : evict_select_kernel<0, 4>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)heads * 4);
    cfg.blockDim = dim3(SEL_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 4;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LCU_CUDA(cudaLaunchKernelEx(&cfg, kernel, sel));
  }
  if (n_away) {
    away.lengths_out = p.lengths_out;
    LCU_CUDA(launch_after(evict_gather_kernel, dim3((unsigned)(heads * chunks), n_away), dim3(256), 0, stream, away, rows, chunks));
  }
  if (n_here) {
    if (!n_away) here.lengths_out = p.lengths_out;
    LCU_CUDA(launch_after(evict_move_kernel, dim3((unsigned)heads, n_here, (widest_here + 31) / 32), dim3(256), 0, stream, here));
  }
  if (!p.n_planes && p.lengths_out) {
    away.lengths_out = p.lengths_out;
    evict_lengths_kernel<<<1, 256, 0, stream>>>(away);
  }
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

int launch_cache_reorder(const reorder_params& p, cudaStream_t stream) {
  int rc = check_planes("cache_reorder", p.dst, p.src, p.row_bytes, p.n_planes);
  if (rc) return rc;
  LCU_REQUIRE(p.parents && p.lengths, "cache_reorder: a null pointer");
  LCU_REQUIRE(words_aligned(p.parents, p.lengths), "cache_reorder: parents and lengths must be 4-byte aligned");
  LCU_REQUIRE(p.n_groups >= 1 && p.beams >= 1 && p.beams <= MAX_BEAMS, "cache_reorder: %d groups of %d beams (1 to %d)", p.n_groups, p.beams, MAX_BEAMS);
  LCU_REQUIRE(p.n_kv >= 1 && p.ctx >= 1 && p.ctx < (1 << 26) && (long long)p.n_groups * p.beams * p.n_kv < (1 << 20), "cache_reorder: %d groups of %d beams, %d heads of %d rows",
              p.n_groups, p.beams, p.n_kv, p.ctx);
  const unsigned long long all_rows = (unsigned long long)p.n_groups * p.beams * p.n_kv * p.ctx;
  rc = check_overlaps("cache_reorder", p.dst, p.src, p.row_bytes, p.n_planes, all_rows, all_rows);
  if (rc) return rc;
  reorder_args away{}, here{};
  int n_away = 0, n_here = 0;
  size_t widest_away = 0, widest_here = 0;
  for (int i = 0; i < p.n_planes; ++i) {
    const plane pl{(uint8_t*)p.dst[i], (const uint8_t*)p.src[i], p.row_bytes[i]};
    if (p.dst[i] == p.src[i]) {
      here.planes[n_here++] = pl;
      widest_here = std::max(widest_here, (size_t)pl.row_bytes);
    } else {
      away.planes[n_away++] = pl;
      widest_away = std::max(widest_away, (size_t)pl.row_bytes);
    }
  }
  for (reorder_args* g : {&away, &here}) {
    g->parents = p.parents;
    g->lengths = p.lengths;
    g->n_groups = p.n_groups;
    g->beams = p.beams;
    g->n_kv = p.n_kv;
    g->ctx = p.ctx;
  }
  if (int rc_dev = need_device()) return rc_dev;
  const int heads = p.n_groups * p.n_kv;
  if (n_away) {
    const size_t chunks = ceil_div(widest_away * p.ctx, REORDER_CTA_BYTES), ctas = chunks * heads * p.beams;
    LCU_REQUIRE(ctas < (1ull << 31), "cache_reorder: planes are too large");
    LCU_CUDA(launch_after(reorder_copy_kernel, dim3((unsigned)ctas, n_away), dim3(256), 0, stream, away, (int)chunks));
  }
  if (n_here) {
    const size_t chunks = ceil_div(widest_here * p.ctx, REORDER_CTA_BYTES / 4), ctas = chunks * heads;
    LCU_REQUIRE(ctas < (1ull << 31), "cache_reorder: planes are too large");
    const dim3 grid((unsigned)ctas, n_here);
    auto* kernel = p.beams <= 4 ? reorder_permute_kernel<4> : p.beams <= 8 ? reorder_permute_kernel<8> : p.beams <= 16 ? reorder_permute_kernel<16> : reorder_permute_kernel<32>;
    LCU_CUDA(launch_after(kernel, grid, dim3(256), 0, stream, here, (int)chunks));
  }
  LCU_CUDA(cudaGetLastError());
  return LCU_OK;
}

}  // namespace lcu
