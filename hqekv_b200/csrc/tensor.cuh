// The sm_100a instructions that the prompt kernels are made of: mbarriers, tensor copies, tcgen05 and tensor memory.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "common.cuh"

namespace hqkv {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// One thread of a warp that is here as a whole.  Around a tcgen05 instruction the compiler then keeps its operands in uniform
// registers; issued from `if (lane == 0)` each of them took some 100 cycles.
__device__ __forceinline__ bool elect_one() {
  unsigned chosen;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(chosen));
  return chosen != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// ---- mbarriers.  Every wait for one has a limit; what runs out sets `stop`, which ends the waits of all roles of the CTA.  A try that
// fails takes 4 us: 33 seconds (an item with 2^30 keys takes 15, and some roles wait for all of it), and 4 for what a CTA has under way
// when something else has gone wrong.  (Waits for tensor memory and for the kernel before have no limit.  They end: a CTA that has
// tensor memory waits for earlier kernels at most, whose CTAs have theirs.)
constexpr int WAIT_TRIES = 1 << 23, DRAIN_TRIES = 1 << 20;
#if HQKV_CHECKS_ENABLED
static __device__ int g_wait_tries = WAIT_TRIES;   // (the bounds-check build can be told to give up early: hqkv_prompt_limit_waits)
__device__ __forceinline__ int wait_tries() { return *const_cast<volatile int*>(&g_wait_tries); }
#else
__device__ __forceinline__ constexpr int wait_tries() { return WAIT_TRIES; }
#endif
__device__ __forceinline__ void bar_init(uint32_t bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok != 0;
}
// by one thread
__device__ __forceinline__ bool bar_wait_one(uint32_t bar, unsigned parity, volatile int* stop) {
  const int tries = wait_tries();
#pragma unroll 1
  for (int i = 0; i < tries; ++i) {
    if (bar_try(bar, parity)) return true;
    if (*stop) return false;
  }
  *stop = 1;
  return false;
}
// By a whole warp, which goes on or gives up as one: what follows (elected threads, copies, barriers of the warp) needs all its lanes.
__device__ __forceinline__ bool bar_wait(uint32_t bar, unsigned parity, volatile int* stop) {
  return __all_sync(0xffffffffu, bar_wait_one(bar, parity, stop));
}
__device__ __forceinline__ void bar_drain(uint32_t bar, unsigned parity) {
  for (int i = 0; i < DRAIN_TRIES && !bar_try(bar, parity); ++i) {
  }
}

// registers per thread of a warpgroup (four warps, all of which come here)
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ---- tensor copies: a box of a (channel, head, token) map, rows of 128 bytes swizzled
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int channel, int head, int token, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(channel), "r"(head), "r"(token), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void fence_generic_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- work of CTAs that have not been launched yet: a request for the next one, and its index out of the answer (-1: there is none)
__device__ __forceinline__ void request_cta(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int requested_cta(uint32_t answer) {
  int x;
  asm volatile(
      "{\n.reg .pred p;\n.reg .b128 a;\n.reg .b32 y, z;\nld.shared.b128 a, [%1];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\nmov.b32 %0, -1;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, _}, a;\n}"
      : "=r"(x)
      : "r"(answer)
      : "memory");
  return x;
}

// ---- tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t slot, unsigned columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, unsigned columns) {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// the loads' registers pass through the wait, so that nothing that reads them comes before it
template <int N>
__device__ __forceinline__ void wait_loads(uint32_t (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7]));
}
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// shared memory operand in rows of 128 bytes, swizzled, eight rows 1024 bytes apart from the next eight; `across`: bytes from
// 64 columns to the next 64 of an operand whose columns are not the ones summed over
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t across) {
  return static_cast<uint64_t>((at >> 4) & 0x3FFF) | static_cast<uint64_t>(across >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
         1ull << 46 | 2ull << 61;
}
// 16-bit operands, fp32 accumulator; columns_b: B's rows are the ones summed over
__device__ __forceinline__ constexpr uint32_t mma_kind(bool bf16, int m, int n, bool columns_b) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (columns_b ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 |
         static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
               "l"(b), "r"(kind), "r"(static_cast<unsigned>(add))
               : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
               "l"(b), "r"(kind), "r"(static_cast<unsigned>(add))
               : "memory");
}

// a lane's row, 32 columns
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                 "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(at));
}
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 32 bytes (a sector) to a 32-byte boundary
__device__ __forceinline__ void store_sector(void* to, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// ---- fp32 arithmetic of pairs
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// NaN if one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace hqkv
