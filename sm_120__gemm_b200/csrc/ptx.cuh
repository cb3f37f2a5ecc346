// Inline-PTX building blocks for the sm_100a kernels: mbarriers with bounded
// waits, TMA / bulk copies, tcgen05 (TMEM allocation, MMA, loads, stores,
// fences) and the exact INT4 -> FP16 dequantisation.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <cstring>

namespace i4g {

// Device status word written when a bounded wait gives up (read by
// i4g_device_status). Values are the I4G_ERR_* codes of i4g.h.
constexpr int kStatusTimeout = -8;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_timer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// ---------------------------------------------------------------- mbarrier

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)
               : "memory");
}

__device__ __forceinline__ void fence_mbarrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
               "r"(bytes)
               : "memory");
}

// try_wait that may suspend the thread for up to `hint_ns` while the phase is
// incomplete (the hardware resumes it as soon as the phase completes), so a
// waiting warp does not spend issue slots polling.
__device__ __forceinline__ bool mbar_try_wait_sleep(uint32_t bar, uint32_t parity,
                                                    uint32_t hint_ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(hint_ns)
      : "memory");
  return ok != 0;
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

// Non-blocking test of a phase (never suspends the thread), at CTA or
// cluster scope, for a thread that has other work while it waits.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ bool mbar_test_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Slow path of mbar_wait: keep polling until the phase completes, *abort is
// set by another warp, or `limit_ns` passes (then sets *abort and records a
// timeout in *status). Out of line so the common, already-complete case
// costs one try_wait.
static __device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort,
                                            int* status, uint64_t limit_ns) {
  const uint64_t t0 = global_timer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i)
      if (mbar_try_wait_sleep(bar, parity, 20000)) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > limit_ns) {
      *abort = 1;
      if (status) atomicExch(status, kStatusTimeout);
      return false;
    }
  }
}

// Wait for the phase of `bar` with the given parity. Gives up (returns
// false) when *abort is set by another warp, or after `limit_ns` of
// waiting. Every spin in the kernels goes through here or mbar_wait_lean,
// so no wait is unbounded.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity,
                                          volatile int* abort, int* status,
                                          uint64_t limit_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i)
      if (mbar_try_wait_sleep(bar, parity, 20000)) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > limit_ns) {
      *abort = 1;
      if (status) atomicExch(status, kStatusTimeout);
      return false;
    }
  }
}

// mbar_wait with the polling loop out of line, for the MMA-issuing thread,
// whose per-block bookkeeping sits between tensor-core instructions.
__device__ __forceinline__ bool mbar_wait_lean(uint32_t bar, uint32_t parity,
                                               volatile int* abort, int* status,
                                               uint64_t limit_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, abort, status, limit_ns);
}

// True in one lane of a converged warp. A warp that issues tensor-core or copy
// instructions from one elected lane inside warp-uniform control flow keeps
// their operands in uniform registers; inside a lane == 0 branch the compiler
// moves them there lane by lane (a 128 x 16 x 16 MMA: 31 against 52 cycles).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A value that is the same in every lane of a converged warp, as one the
// compiler knows to be: control flow that hangs on it stays warp-uniform.
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return __reduce_max_sync(0xffffffffu, v);
}

// mbar_wait for a whole converged warp; the outcome is the same for every lane.
// The polling loop is inline: around a call the compiler cannot keep the
// operands of tensor-core instructions in uniform registers.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity,
                                               volatile int* abort, int* status,
                                               uint64_t limit_ns) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint64_t t0 = global_timer_ns();
#pragma unroll 1
  while (!__all_sync(0xffffffffu, mbar_try_wait_sleep(bar, parity, 20000))) {
    const bool late = global_timer_ns() - t0 > limit_ns;
    if (__any_sync(0xffffffffu, late || *abort != 0)) {
      if (late) {
        *abort = 1;
        if (status) atomicExch(status, kStatusTimeout);
      }
      return false;
    }
  }
  return true;
}

// Named barrier 1 among `nthreads` threads (a subset of warps, e.g. those
// that do not stream copies); `bar_and` also ANDs a per-thread predicate
// across them.
__device__ __forceinline__ void epi_bar_sync(int nthreads) {
  asm volatile("bar.sync 1, %0;" ::"r"(nthreads) : "memory");
}

__device__ __forceinline__ bool epi_bar_and(int nthreads, bool v) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred pin, pout;\n\t"
      "setp.ne.u32 pin, %1, 0;\n\t"
      "bar.red.and.pred pout, 1, %2, pin;\n\t"
      "selp.u32 %0, 1, 0, pout;\n\t}"
      : "=r"(out)
      : "r"(static_cast<uint32_t>(v)), "r"(nthreads)
      : "memory");
  return out != 0;
}

// ------------------------------------------------------------ TMA / bulk

__device__ __forceinline__ void prefetch_tensormap(const void* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// 2-D tiled TMA load, no multicast: box lands at smem `dst`, completion is
// counted in bytes on `bar`.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* map, uint32_t bar,
                                            int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

// 3-D tiled TMA load, no multicast.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, uint32_t bar,
                                            int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// 16-byte asynchronous copy global -> shared through L2 (cp.async.cg); the
// bytes past src_bytes (0 or 16) are zero-filled.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(src_bytes)
               : "memory");
}

// One arrival on `bar` once every cp.async this thread issued so far has
// landed (the barrier's expected count includes it: .noinc).
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Contiguous bulk copy global -> shared (16-byte aligned, size % 16 == 0).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// Registers a thread, from here on, of the four warps of an aligned warpgroup
// (all of them execute it). What `regs_inc` takes has to come from what the
// block was launched with and others gave back.
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Warms L2 with a contiguous global range (16-byte aligned, size % 16 == 0).
// Nothing lands in shared memory, so the range may still be written by an
// earlier kernel: L2 is the point of coherence and later loads see the writes.
__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// ------------------------------------------- programmatic dependent launch

// Waits until every grid this one depends on programmatically has completed
// and its memory operations are visible; returns at once when the grid was
// launched without a programmatic dependency.
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Lets a programmatically dependent grid be scheduled once every CTA of this
// grid has issued this (or exited); a no-op without such a dependent.
__device__ __forceinline__ void launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ------------------------------------------------------ clusters / CTA pairs

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// The shared::cluster address of `local` (a shared::cta address of this CTA)
// in cluster CTA `rank`.
__device__ __forceinline__ uint32_t mapa_shared(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}

// Arrive on an mbarrier of another CTA of the cluster (shared::cluster
// address), releasing this thread's prior memory operations at cluster scope.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar)
               : "memory");
}

// Arrival on a cluster CTA's barrier without release semantics (no fence
// before it). For signals that follow work the thread has already seen
// complete: tcgen05.wait::st / wait::ld for TMEM, a complete_tx barrier for a
// TMA copy into shared memory. The waiter's acquire plus
// tcgen05.fence::after_thread_sync then orders its own tcgen05 work after.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar)
               : "memory");
}

__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// try_wait at cluster scope that may suspend the thread for up to `hint_ns`
// while the phase is incomplete (as mbar_try_wait_sleep).
__device__ __forceinline__ bool mbar_try_wait_cluster_sleep(uint32_t bar, uint32_t parity,
                                                            uint32_t hint_ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(hint_ns)
      : "memory");
  return ok != 0;
}

// mbar_wait for a barrier that the other CTA of a pair also arrives on:
// acquire at cluster scope. Bounded as mbar_wait; a waiting thread suspends
// rather than spins.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity,
                                                  volatile int* abort, int* status,
                                                  uint64_t limit_ns) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i)
      if (mbar_try_wait_cluster_sleep(bar, parity, 20000)) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > limit_ns) {
      *abort = 1;
      if (status) atomicExch(status, kStatusTimeout);
      return false;
    }
  }
}

// All threads of all CTAs of the cluster (warp-aligned).
__device__ __forceinline__ void cluster_barrier() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- tcgen05

__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   dst_smem),
               "r"(ncols)
               : "memory");
}

__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr),
               "r"(ncols)
               : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Arrive once on `bar` when every tcgen05 op issued so far by this thread
// has completed.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          bar)
      : "memory");
}

// CTA-pair forms: TMEM allocated for the pair (one warp of each CTA, same
// warp, same destination offset), freed the same way.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   dst_smem),
               "r"(ncols)
               : "memory");
}

__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}

// Arrive once on the mbarrier at offset `bar` in each CTA of the pair (mask
// 0b11) when every pair MMA issued so far by this thread has completed.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// Pair MMA (issued by the even CTA): D (+)= A x B with M = 256 split over the
// pair's TMEM (each CTA's 128 lanes, same address) and B's N rows split over
// the pair's shared memory (first half in the even CTA, second in the odd,
// same offset); kind::f16, FP32 accumulate.
__device__ __forceinline__ void mma_f16_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                                uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Pair MMA with both operands in shared memory (issued by the even CTA):
// A's M = 256 rows split over the pair (rows 0-127 in the even CTA, 128-255
// in the odd, same offset), B's N rows split the same way, D's M rows over
// the pair's TMEM; kind::f16, FP32 accumulate.
__device__ __forceinline__ void mma_f16_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                                uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D[tmem] (+)= A[tmem] x B[smem]; kind::f16, FP32 accumulate.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The four k16 steps of one 64-k block (operand A 8 TMEM columns and operand B
// 32 bytes further per step), issued by one elected lane of a converged warp;
// the first step starts the sum unless `accumulate`.
__device__ __forceinline__ void mma_f16_ts_block(uint32_t d_tmem, uint32_t a_tmem,
                                                 uint64_t b_desc, uint32_t idesc,
                                                 uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred one, acc, yes;\n\t"
      ".reg .b32 a1, a2, a3;\n\t"
      ".reg .b64 b1, b2, b3;\n\t"
      "elect.sync _|one, 0xffffffff;\n\t"
      "setp.ne.b32 acc, %4, 0;\n\t"
      "setp.eq.b32 yes, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\t"
      "add.u32 a2, %1, 16;\n\t"
      "add.u32 a3, %1, 24;\n\t"
      "add.u64 b1, %2, 2;\n\t"
      "add.u64 b2, %2, 4;\n\t"
      "add.u64 b3, %2, 6;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, acc;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, yes;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, yes;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, yes;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// All MMAs of a ring stage of whole 64-k blocks (operand A 32 TMEM columns per
// block, operand B `box` 16-byte units apart) and the commit that frees it, by
// one elected lane of a converged warp.
#define I4G_MMA_STEP(A, B, ACC) \
  "add.u32 a, %1, " A ";\n\t" \
  "add.u64 b, t, " B ";\n\t" \
  "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, " ACC ";\n\t"
#define I4G_MMA_BLOCK(A0, A1, A2, A3, ACC)                                 \
  I4G_MMA_STEP(A0, "0", ACC) I4G_MMA_STEP(A1, "2", "yes")                  \
  I4G_MMA_STEP(A2, "4", "yes") I4G_MMA_STEP(A3, "6", "yes")
#define I4G_MMA_HEAD                             \
  "{\n\t.reg .pred one, acc, yes;\n\t"          \
  ".reg .b32 a;\n\t"                             \
  ".reg .b64 b, t;\n\t"                          \
  "elect.sync _|one, 0xffffffff;\n\t"            \
  "setp.ne.b32 acc, %4, 0;\n\t"                  \
  "setp.eq.b32 yes, 0, 0;\n\t"                   \
  "mov.b64 t, %2;\n\t"
#define I4G_MMA_NEXT "add.u64 t, t, %6;\n\t"
#define I4G_MMA_COMMIT                                                                   \
  "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"

__device__ __forceinline__ void mma_f16_ts_blocks1(uint32_t d_tmem, uint32_t a_tmem,
                                                   uint64_t b_desc, uint32_t idesc,
                                                   uint32_t accumulate, uint32_t bar) {
  asm volatile(I4G_MMA_HEAD I4G_MMA_BLOCK("0", "8", "16", "24", "acc") I4G_MMA_COMMIT ::"r"(
                   d_tmem),
               "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void mma_f16_ts_blocks2(uint32_t d_tmem, uint32_t a_tmem,
                                                   uint64_t b_desc, uint32_t idesc,
                                                   uint32_t accumulate, uint64_t box,
                                                   uint32_t bar) {
  asm volatile(I4G_MMA_HEAD I4G_MMA_BLOCK("0", "8", "16", "24", "acc") I4G_MMA_NEXT
                   I4G_MMA_BLOCK("32", "40", "48", "56", "yes") I4G_MMA_COMMIT ::"r"(d_tmem),
               "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(bar), "l"(box)
               : "memory");
}

__device__ __forceinline__ void mma_f16_ts_blocks4(uint32_t d_tmem, uint32_t a_tmem,
                                                   uint64_t b_desc, uint32_t idesc,
                                                   uint32_t accumulate, uint64_t box,
                                                   uint32_t bar) {
  asm volatile(I4G_MMA_HEAD I4G_MMA_BLOCK("0", "8", "16", "24", "acc") I4G_MMA_NEXT
                   I4G_MMA_BLOCK("32", "40", "48", "56", "yes") I4G_MMA_NEXT
                       I4G_MMA_BLOCK("64", "72", "80", "88", "yes") I4G_MMA_NEXT
                           I4G_MMA_BLOCK("96", "104", "112", "120", "yes") I4G_MMA_COMMIT ::"r"(
                               d_tmem),
               "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(bar), "l"(box)
               : "memory");
}

#undef I4G_MMA_STEP
#undef I4G_MMA_BLOCK
#undef I4G_MMA_HEAD
#undef I4G_MMA_NEXT
#undef I4G_MMA_COMMIT

// Shared-memory matrix descriptor for a K-major operand stored as rows of
// 128 bytes with the 128-byte swizzle (8-row atoms 1024 bytes apart).
__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);  // start address
  d |= static_cast<uint64_t>(0) << 16;                  // leading byte offset (unused)
  d |= static_cast<uint64_t>(1024 >> 4) << 32;          // stride byte offset
  d |= static_cast<uint64_t>(1) << 46;                  // descriptor version (sm_100)
  d |= static_cast<uint64_t>(2) << 61;                  // SWIZZLE_128B
  return d;
}

// Instruction descriptor, kind::f16: F16 A and B, F32 D, both K-major.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int mma_m, int mma_n) {
  return (1u << 4) | (static_cast<uint32_t>(mma_n >> 3) << 17) |
         (static_cast<uint32_t>(mma_m >> 4) << 24);
}

// 32 data-path lanes x 16 consecutive 32-bit columns, one lane per thread.
// 32 lanes x 8 consecutive 32-bit columns, one lane per thread.
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

// Loads 8 columns; the registers are valid only after tmem_ld_wait8(r).
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}

__device__ __forceinline__ void tmem_ld_wait8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
      "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 lanes x 32 consecutive 32-bit columns, one lane per thread. The
// registers are valid only after tmem_ld_wait(r), which takes them as
// operands so no use can be scheduled ahead of the wait.
__device__ __forceinline__ void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
      "[%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                 "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// ---------------------------------------------------- INT4 -> FP16 decode

__device__ __forceinline__ __half2 u32_as_half2(uint32_t v) {
  __half2 h;
  static_assert(sizeof(h) == sizeof(v), "half2 is 32 bits");
  memcpy(&h, &v, sizeof(v));
  return h;
}

__device__ __forceinline__ uint32_t half2_as_u32(__half2 h) {
  uint32_t v;
  memcpy(&v, &h, sizeof(v));
  return v;
}

// Decode pair p (0..3) of a tile-layout word into half2 {half(q0*s), half(q1*s)}.
// The nibble pair sits at bits [4p, 4p+4) and [16+4p, 20+4p). (nib & 15) ^ 8
// ORed into 0x6400 is the half 1024 + 8 + q, so one exact subtraction of 1032
// gives q, and one round-to-nearest multiply gives half(q * s): the value the
// reference's dequantize computes as __float2half(float(q) * float(s)).
// Written in C++ (not inline PTX) so the compiler keeps the constants in
// immediates or hoisted registers.
template <int P>
__device__ __forceinline__ uint32_t decode_pair(uint32_t word, uint32_t scale2) {
  const uint32_t x = (P == 0) ? word : (word >> (4 * P));
  const uint32_t biased = (x & 0x000F000Fu) ^ 0x64086408u;
  const __half2 q = __hsub2(u32_as_half2(biased), u32_as_half2(0x64086408u));
  return half2_as_u32(__hmul2(q, u32_as_half2(scale2)));
}

// The four pairs of a tile-layout word, as decode_pair gives them, in one
// multiply-add per pair. A nibble XOR 8 is u = q + 8; at bits 4..7 of a half
// (the other bits zero) it is the subnormal u 2^-20. fma(u 2^-20, s 2^20, -8 s)
// has the exact value q s before its one rounding, so it is half(q * s) bit
// for bit, as long as s 2^20 is finite and -8 s exact. For a normal s both are
// additions to the exponent field, so fast_scale admits 2^-14 <= s < 2^-4
// (0x0400 .. 0x2BFF; times 2^20 at most 0x7BFF, the largest half). 11
// instructions of the half-rate pipes a word, against decode_pair's 15.
__device__ __forceinline__ bool fast_scale(uint32_t scale_bits) {
  return scale_bits - 0x0400u < 0x2C00u - 0x0400u;
}
constexpr uint32_t kTimes2p20 = 0x50005000u;   // + 20 on both exponents
constexpr uint32_t kTimesMinus8 = 0x8C008C00u;  // + 3, and the sign

// The mask of the nibble and the bit that turns q into u, kept in registers:
// as two immediates the and-xor would become two instructions (K = 65536,
// N = 18944, 16 rows: 146 us so, 121 us with registers).
struct NibbleMask {
  uint32_t keep, flip;
  __device__ __forceinline__ NibbleMask() {
    asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(keep));
    asm volatile("mov.b32 %0, 0x00800080;" : "=r"(flip));
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
    uint32_t u;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(u) : "r"(x), "r"(keep), "r"(flip));
    return u;
  }
};

__device__ __forceinline__ void decode_word(uint32_t word, uint32_t scale_2p20, uint32_t minus_8s,
                                            const NibbleMask& nibble, uint32_t* out) {
  const uint32_t x[4] = {word << 4, word, word >> 4, word >> 8};
#pragma unroll
  for (int p = 0; p < 4; ++p)
    out[p] = half2_as_u32(__hfma2(u32_as_half2(nibble(x[p])), u32_as_half2(scale_2p20),
                                  u32_as_half2(minus_8s)));
}

__device__ __forceinline__ uint32_t half_bits_x2(uint16_t h) {
  return static_cast<uint32_t>(h) | (static_cast<uint32_t>(h) << 16);
}

}  // namespace i4g
