// tcgen05 (5th-generation tensor core), TMEM and tensor-map helpers, sm_100a.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace hx {
namespace tc {

// ---- bounded waits ---------------------------------------------------------
// Every wait of a CTA gives up after kMaxPolls polls or as soon as another
// warp has given up (the shared word `abort`): the kernel then reports
// HX_DEV_ERR_TIMEOUT, drains what it has in flight, frees its TMEM and returns.
HX_DEVINL bool wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t i = 0; i < kMaxPolls; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 15u) == 15u && *abort) return false;
  }
  *abort = 1u;
  return false;
}

// The same for a whole warp: one answer for all lanes, since warp-wide
// (.sync.aligned) instructions follow.
HX_DEVINL bool wait_warp(uint64_t* bar, uint32_t parity, volatile uint32_t* abort) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, done)) return true;
  return __all_sync(0xffffffffu, wait(bar, parity, abort));
}

// One lane of the (converged) warp, the same at every call: the thread that
// issues the products.
HX_DEVINL bool elect() {
  uint32_t y;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(y));
  return y != 0u;
}

HX_DEVINL void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ---- TMEM ------------------------------------------------------------------
// Addresses: lane << 16 | column. Warp w of a warpgroup reaches lanes
// 32 (w % 4) .. + 31; a 32x32b access gives lane l of the warp row l, one
// 32-bit column a register.
HX_DEVINL void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
HX_DEVINL void tmem_dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
HX_DEVINL void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
HX_DEVINL void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
HX_DEVINL void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
HX_DEVINL void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define HX_R8(a, o) "=r"(a[o]), "=r"(a[o + 1]), "=r"(a[o + 2]), "=r"(a[o + 3]), "=r"(a[o + 4]), "=r"(a[o + 5]), \
                    "=r"(a[o + 6]), "=r"(a[o + 7])
#define HX_I8(a, o) "r"(a[o]), "r"(a[o + 1]), "r"(a[o + 2]), "r"(a[o + 3]), "r"(a[o + 4]), "r"(a[o + 5]), \
                    "r"(a[o + 6]), "r"(a[o + 7])
HX_DEVINL void ld32(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : HX_R8(r, 0), HX_R8(r, 8), HX_R8(r, 16), HX_R8(r, 24)
      : "r"(addr));
}
HX_DEVINL void ld16(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : HX_R8(r, 0), HX_R8(r, 8)
      : "r"(addr));
}
HX_DEVINL void st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      HX_I8(r, 0), HX_I8(r, 8), HX_I8(r, 16), HX_I8(r, 24)
      : "memory");
}
HX_DEVINL void st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      HX_I8(r, 0), HX_I8(r, 8)
      : "memory");
}

// ---- matrix products ---------------------------------------------------------
// Shared-memory operand descriptor, 128-byte swizzle: rows of 128 bytes (64
// 16-bit elements) in groups of 8 (1024 bytes). `lead` is the byte distance of
// the next 64 elements along the contiguous dimension where that dimension is
// M or N (it is not used where it is K).
HX_DEVINL uint64_t desc128(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor of kind::f16: fp32 accumulator, A and B both fp16
// (bf16 = 0) or both bf16 (1), M x N; b_mn: B's contiguous dimension is N.
constexpr uint32_t idesc_f16(int bf16, int M, int N, int b_mn) {
  return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N / 8) << 17) | ((uint32_t)(M / 16) << 24);
}
HX_DEVINL void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
HX_DEVINL void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// The barrier completes a phase when every product this thread issued before has finished.
HX_DEVINL void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// ---- tensor-map loads -----------------------------------------------------------
HX_DEVINL void tma3(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
HX_DEVINL void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---- taking over CTAs that have not started yet ------------------------------------
// A running CTA asks the hardware for the next CTA of its own grid that has not
// been launched (cluster launch control): it cancels that launch and does the
// work itself, so a grid of one CTA per work item is dealt out dynamically to
// CTAs that keep their shared memory, TMEM and prefetched tiles. The 16-byte
// answer lands in shared memory and completes 16 bytes on `bar`.
HX_DEVINL void next_cta_request(void* answer, uint64_t* bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// blockIdx.x taken over, or -1 when the grid has no CTA left
HX_DEVINL int next_cta(const void* answer) {
  uint32_t ok, x;
  asm volatile(
      "{\n .reg .b64 lo, hi;\n .reg .b128 h;\n .reg .pred p;\n"
      " ld.shared.v2.b64 {lo, hi}, [%2];\n mov.b128 h, {lo, hi};\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      " selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n}"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return ok ? (int)x : -1;
}

// ---- register budget of a warpgroup ------------------------------------------------
template <int N>
HX_DEVINL void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
HX_DEVINL void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ---- packed fp32 pairs ----------------------------------------------------------------
HX_DEVINL uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
HX_DEVINL void f2_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
HX_DEVINL uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
HX_DEVINL uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
HX_DEVINL uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
HX_DEVINL float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace tc
}  // namespace hx
