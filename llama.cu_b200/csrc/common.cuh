// Shared device/host helpers for the sm_100a kernels: error handling, mbarrier and bulk-copy
// (TMA) PTX wrappers with bounded waits, programmatic-dependent-launch controls, cluster helpers.
#pragma once

#include <atomic>
#include <cstdint>
#include <cstdio>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "step_words.hpp"

namespace lcu {

// ---------------------------------------------------------------- host-side error handling
// Status codes returned through the C ABI.
enum status : int {
  LCU_OK = 0,
  LCU_ERR_CUDA = 1,        // a CUDA runtime call failed (message in lcu_last_error)
  LCU_ERR_ARG = 2,         // invalid argument / unsupported shape
  LCU_ERR_IO = 3,          // file missing or of the wrong size
  LCU_ERR_DEVICE_WAIT = 4  // a kernel gave up on a bounded wait (device error word set)
};

void set_last_error(const char* fmt, ...);
const char* last_error();

#define LCU_CUDA(expr)                                                                        \
  do {                                                                                        \
    cudaError_t _e = (expr);                                                                  \
    if (_e != cudaSuccess) {                                                                  \
      ::lcu::set_last_error("%s:%d: %s failed: %s", __FILE__, __LINE__, #expr, cudaGetErrorString(_e)); \
      return ::lcu::LCU_ERR_CUDA;                                                             \
    }                                                                                         \
  } while (0)

#define LCU_REQUIRE(cond, ...)            \
  do {                                    \
    if (!(cond)) {                        \
      ::lcu::set_last_error(__VA_ARGS__); \
      return ::lcu::LCU_ERR_ARG;          \
    }                                     \
  } while (0)

// for entry points that check their arguments before they look for a device
inline int need_device() {
  static std::atomic<bool> seen{false};  // (devices do not go away; calls may come from any thread)
  if (seen.load(std::memory_order_relaxed)) return LCU_OK;
  int n = 0;
  if (cudaGetDeviceCount(&n) == cudaSuccess && n > 0) {
    seen.store(true, std::memory_order_relaxed);
    return LCU_OK;
  }
  cudaGetLastError();
  set_last_error("no CUDA device is visible: this library has no CPU path");
  return LCU_ERR_CUDA;
}

inline size_t ceil_div(size_t a, size_t b) { return (a + b - 1) / b; }
inline size_t round_up(size_t a, size_t b) { return ceil_div(a, b) * b; }

// device error word: kernels that give up on a bounded wait store a code here (never trap)
constexpr int DEV_ERR_FULL_WAIT = 0x101;   // consumer timed out waiting for a filled stage
constexpr int DEV_ERR_EMPTY_WAIT = 0x102;  // producer timed out waiting for a free stage
constexpr int DEV_ERR_TMEM_WAIT = 0x103;   // epilogue timed out waiting for an MMA commit

#ifdef __CUDACC__
// silu's a / (1 + expf(-a)) (llama_cu.cu:533-539) for the fused gate of a GEMM epilogue: the quotient is CUDA's
// __fdividef, within two units in the last place of the division and without its operand check and branch (with the full
// division the gate cost an epilogue of four warps more than its tile's main loop lasts).  The result is rounded to half
// right after, so it differs from the division's in about one value of four thousand, by one unit of the half format.
// (__fdividef returns 0 for divisors above 2^126, a below -87, where the quotient is far below the smallest half.)
__device__ __forceinline__ float silu_of_half(float a) { return __fdividef(a, 1.0f + expf(-a)); }

// Programmatic dependent launch for the kernels of a prompt pass: with the attribute a kernel's CTAs may start - set up
// barriers, allocate tensor memory, fetch descriptors - while the kernel before it in the stream drains.  Every kernel
// launched this way executes griddepcontrol.wait (pdl_wait) before it touches global memory, so its body still runs
// after the previous kernel has completed and flushed.  (A kernel that reads something earlier says what makes that safe.)
// prompt_pdl() = 0 turns the attribute off.
int& prompt_pdl();
template <typename... KP, typename... Args>
cudaError_t launch_after(void (*kernel)(KP...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = prompt_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KP>(args)...);
}

// ---------------------------------------------------------------- device helpers
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void fence_mbar_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait.  Gives up after ~1 s of SM clock (or immediately once another thread has flagged
// an error), records `code` in *err and returns false; the caller carries on so the kernel ends.
// heed = false: the word may hold an error of an earlier launch, which says nothing about this one; only the time counts.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int* err, int code, bool heed = true) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  long long next_check = 400000;  // the error word (global memory) is looked at every ~0.2 ms only:
                                  // a load on the polling path would add its latency to every hand-over
  for (;;) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long dt = clock64() - t0;
    if (dt > next_check) {
      if (heed && *(volatile int*)err != 0) return false;
      if (dt > 2000000000ll) {
        atomicCAS(err, 0, code);
        return false;
      }
      next_check += 400000;
    }
  }
}

constexpr int DEV_ERR_PEER_WAIT = 0x104;   // a kernel timed out waiting for another GPU's slice of an activation row

// ---- flags between GPUs (tensor-parallel decode): a producer publishes a monotonically increasing number into the
// consumer GPU's memory once its peer stores are out; the consumer polls its own memory.
__device__ __forceinline__ int ld_relaxed_sys(const int* p) {
  int v;
  asm volatile("ld.relaxed.sys.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void st_relaxed_sys(int* p, int v) {
  asm volatile("st.relaxed.sys.global.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// release / acquire fence at system scope: "fence; st.relaxed" publishes, "ld.relaxed; fence" observes
__device__ __forceinline__ void fence_acq_rel_sys() { asm volatile("fence.acq_rel.sys;" ::: "memory"); }
// Polls with relaxed loads (a fence per poll would cost more than the exchange) and fences once the value is there.
// Bounded: gives up after ~1 s of SM clock (or once another thread has flagged an error), records DEV_ERR_PEER_WAIT
// in *err and returns false; the caller carries on so the kernel ends.
__device__ __forceinline__ bool flag_wait_at_least(const int* flag, int target, int* err) {
  if (ld_relaxed_sys(flag) >= target) {
    fence_acq_rel_sys();
    return true;
  }
  const long long t0 = clock64();
  long long next_check = 400000;
  for (;;) {
    if (ld_relaxed_sys(flag) >= target) {
      fence_acq_rel_sys();
      return true;
    }
    const long long dt = clock64() - t0;
    if (dt > next_check) {
      if (*(volatile int*)err != 0) return false;
      if (dt > 2000000000ll) {
        atomicCAS(err, 0, DEV_ERR_PEER_WAIT);
        return false;
      }
      next_check += 400000;
    }
  }
}

// 1-D bulk copy global -> this CTA's shared memory, completion counted on an mbarrier.
// Both addresses 16-byte aligned, size a multiple of 16.
__device__ __forceinline__ void bulk_g2s(uint32_t dst_smem, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_smem),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// same with an L2 eviction-priority hint (policy from createpolicy)
__device__ __forceinline__ void bulk_g2s_hint(uint32_t dst_smem, const void* src, uint32_t bytes, uint32_t bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(dst_smem),
      "l"(src), "r"(bytes), "r"(bar), "l"(pol)
      : "memory");
}
__device__ __forceinline__ uint64_t policy_evict_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
// asynchronous request to bring [src, src+bytes) into L2 (no destination, no completion to wait for)
__device__ __forceinline__ void l2_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
// 4-byte asynchronous copy (Ampere-style) and its hand-over to an mbarrier
__device__ __forceinline__ void cp_async4(uint32_t dst_smem, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst_smem), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst_smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst_smem), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_mbar_arrive_noinc(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// programmatic dependent launch
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// named barrier among a subset of the CTA's warps
__device__ __forceinline__ void bar_sync(int id, int nthreads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

// thread-block cluster
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of a peer CTA's shared-memory location (distributed shared memory)
__device__ __forceinline__ uint32_t mapa(uint32_t smem_addr, uint32_t cta_rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(cta_rank));
  return r;
}
__device__ __forceinline__ float ld_dsmem_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// token and error word to pinned host memory in one store of 64 bits, behind everything written before
__device__ __forceinline__ void tell_host(uint64_t* at, int token, int code) {
  __threadfence_system();
  asm volatile("st.relaxed.sys.global.b64 [%0], %1;" ::"l"(at), "l"(packed_words(token, code)) : "memory");
}

// warp-level m16n8k16 fp16 x fp16 -> fp32 product used as the multiply-accumulate engine of the
// weight-streaming GEMV (A = 16 weight rows, B = up to 8 activation rows)
__device__ __forceinline__ void mma_16816(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same tile with bfloat16 operands
__device__ __forceinline__ void mma_16816_bf16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Same product with every accumulator entry started from one value: no register has to be set up per entry.
__device__ __forceinline__ void mma_16816_from(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1, float c) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
#endif  // __CUDACC__

}  // namespace lcu
