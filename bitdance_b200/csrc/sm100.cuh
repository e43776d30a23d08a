// sm100.cuh -- thin inline-PTX wrappers for the Blackwell (sm_100a) features the
// W4A6 kernels use: mbarriers, TMA bulk/tensor copies, tensor memory (TMEM)
// allocation/load/store/copy, and block-scaled tcgen05.mma of kind::mxf8f6f4.
//
// Every wait in this file is bounded: a wait that runs out sets a bit in the
// caller's error word and returns false, so a logic error surfaces as a status
// code on the host instead of a hung GPU.
#pragma once
#include <cstdint>
#include <cuda.h>

namespace bd {

// ---------------------------------------------------------------------------------
// Error bits written by kernels into their error word (host reads it back).
enum : uint32_t {
  kErrWaitTma = 1u << 0,     // a consumer gave up waiting for a TMA stage
  kErrWaitOperand = 1u << 1, // MMA issuer gave up waiting for transcoded operands
  kErrWaitEmpty = 1u << 2,   // producer gave up waiting for a free stage
  kErrWaitAccum = 1u << 3,   // epilogue gave up waiting for the accumulator
  kErrWaitMma = 1u << 4,     // transcode gave up waiting for the MMA to free a buffer
  kErrNonFinite = 1u << 5,   // the activation quantiser saw a NaN or an infinity
  kErrRange = 1u << 6,       // a scale had no representation in the target format
  kErrShape = 1u << 8,       // the kernel saw a shape it does not support
};

// Bound for any single wait, in SM clock cycles (about 2 s at 2 GHz). Normal waits last
// microseconds.
constexpr unsigned long long kWaitLimitCycles = 4000000000ull;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t pred = 0;
  asm volatile(
      "{\n\t.reg .b32 r;\n\t.reg .pred p;\n\t"
      "elect.sync r|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(pred));
  return pred != 0;
}

// ---------------------------------------------------------------------------------
// mbarrier
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void fence_mbar_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
// Programmatic dependent launch (griddepcontrol, sm_90+). wait: block until the grids this
// one depends on have completed and their memory is visible (returns at once when the
// launch had no programmatic dependency). launch_dependents: allow the next grid on the
// stream, if launched with programmatic serialisation, to be scheduled.
__device__ __forceinline__ void grid_dep_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void grid_dep_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// The same with acquire semantics at cluster scope: for barriers the peer CTA of a pair
// arrives on (its arrive releases its writes at cluster scope).
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait on phase `parity`. After `limit` SM cycles ORs `code` into *err, sets
// *abort_flag and returns false. Also returns false early if another role already aborted.
// The hot path is a tight try_wait loop (try_wait itself suspends the thread in hardware for
// a while); the abort flag and the cycle counter are looked at only every 1024 tries.
// kCluster: acquire at cluster scope (mbar_try_wait_cluster).
template <bool kCluster = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t* err,
                                          uint32_t code, volatile uint32_t* abort_flag,
                                          unsigned long long limit = kWaitLimitCycles) {
  auto try_once = [&]() {
    return kCluster ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
  };
  if (try_once()) return true;
  const long long t0 = clock64();
  uint32_t spins = 0;
  while (true) {
    if (try_once()) return true;
    if ((++spins & 1023u) == 0) {
      if (abort_flag != nullptr && *abort_flag) return false;
      if (static_cast<unsigned long long>(clock64() - t0) > limit) {
        if (err) atomicOr(err, code);
        if (abort_flag) *abort_flag = 1u;
        return false;
      }
    }
  }
}

// Position in a ring of N slots: slot index and the parity of the current pass.
template <int N>
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __host__ __device__ constexpr void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1u;
    }
  }
  // Parity of the last pass that came by slot s: waiting for it on the slot's barrier waits for what was
  // started there last (at once where nothing was yet: a fresh barrier lets parity 1 through).
  __host__ __device__ constexpr uint32_t last_parity(int s) const {
    return s < slot ? phase : phase ^ 1u;
  }
};
// (checked against fills counted one by one)
template <int N>
constexpr bool ring_parities_right(int fills) {
  RingPos<N> r;
  int count[N] = {};
  for (int i = 0; i < fills; ++i) {
    ++count[r.slot];
    r.next();
  }
  for (int s = 0; s < N; ++s)
    if (r.last_parity(s) != ((count[s] + 1u) & 1u)) return false;
  return true;
}
static_assert(ring_parities_right<3>(0) && ring_parities_right<3>(1) && ring_parities_right<3>(2) &&
                  ring_parities_right<3>(3) && ring_parities_right<3>(4) && ring_parities_right<3>(7) &&
                  ring_parities_right<8>(8) && ring_parities_right<8>(13) && ring_parities_right<5>(16),
              "the last fill of every slot");

__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Atomic add at GPU scope with acquire-release semantics, returning the old value. As the
// count-in of a stream-K tile after a CTA barrier it releases every write the CTA made
// before the barrier and acquires those of the CTAs that counted in earlier (no separate
// fences).
__device__ __forceinline__ uint32_t atom_add_acq_rel_gpu(uint32_t* p, uint32_t v) {
  uint32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;"
               : "=r"(old)
               : "l"(p), "r"(v)
               : "memory");
  return old;
}

// ---------------------------------------------------------------------------------
// CTA pairs (clusters of two): rank in the cluster, a barrier over both CTAs, addresses in
// the peer's shared memory, stores and mbarrier arrives there
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// every thread of both CTAs (warp-converged)
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared::cluster address of the same shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t mapa_shared(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_shared_cluster_u32(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// arrive on an mbarrier given by its shared::cluster address (this CTA's or the peer's), with
// the default semantics (release at CTA scope): what the waiter needs ordered before it is
// tensor-memory writes, completed by tcgen05.wait::st and fenced by
// tcgen05.fence::before_thread_sync before the arrive (a release at cluster scope made every
// arrive wait about a microsecond)
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// ---------------------------------------------------------------------------------
// TMA / bulk copies (global -> shared, completion via mbarrier tx-count)
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int32_t x,
                                            int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// The same by a CTA of a pair (cta_group::2): into this CTA's shared memory, completing on a barrier
// of either CTA (its shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int32_t x,
                                                 int32_t y, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int32_t x,
                                            int32_t y, int32_t z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Untiled bulk copy: dst/src 16-byte aligned, bytes a multiple of 16.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}
// TMA store (shared -> global) in this thread's bulk async-group; the box's inner
// coordinate x times the element size must be a multiple of 16 bytes
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int32_t x,
                                             int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::
                   "l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void bulk_commit_group() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// until at most N of this thread's bulk groups still read their shared-memory source
template <int N>
__device__ __forceinline__ void bulk_wait_group_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
// until every bulk group of this thread has completed (its writes performed)
__device__ __forceinline__ void bulk_wait_group_all() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void prefetch_tmap(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// ---------------------------------------------------------------------------------
// Tensor memory
__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
// tensor memory of a CTA pair (the MMAs of cta_group::2 write both CTAs' allocations at the
// same address): executed by the same warp of both CTAs
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem),
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
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Arrive once on `bar` when every tcgen05 async op issued so far by this thread is done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
// The same for the MMAs of a CTA pair, arriving on the barrier at `bar` in every CTA of
// `cta_mask` (bit r: CTA rank r of the cluster).
__device__ __forceinline__ void tc_commit_pair(uint32_t bar, uint16_t cta_mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(bar),
      "h"(cta_mask)
      : "memory");
}
// Shared -> tensor memory: 32 rows x 16 bytes, replicated into all four lane quarters.
__device__ __forceinline__ void tmem_cp_32x128b_x4(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc)
               : "memory");
}
// The same in both CTAs of a pair, each from its own shared memory at the same offset.
__device__ __forceinline__ void tmem_cp_32x128b_x4_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc)
               : "memory");
}
// Shared -> tensor memory: 128 rows (lanes) x 16 bytes (4 columns).
__device__ __forceinline__ void tmem_cp_128x128b(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.128x128b [%0], %1;" ::"r"(taddr), "l"(sdesc)
               : "memory");
}
// Shared -> tensor memory: 128 rows (lanes) x 32 bytes (8 columns).
__device__ __forceinline__ void tmem_cp_128x256b(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.128x256b [%0], %1;" ::"r"(taddr), "l"(sdesc)
               : "memory");
}

__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// The same, tied to the registers of the load: their uses cannot be scheduled before it.
__device__ __forceinline__ void tmem_ld_wait_x32(uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
        "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]),
        "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}
// The same for 8 and 16 registers.
__device__ __forceinline__ void tmem_ld_wait_x8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_x16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st_x1(uint32_t taddr, uint32_t a) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(a)
               : "memory");
}
__device__ __forceinline__ void tmem_st_x2(uint32_t taddr, uint32_t a, uint32_t b) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(taddr), "r"(a),
               "r"(b)
               : "memory");
}
__device__ __forceinline__ void tmem_st_x4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c,
                                           uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(a),
               "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(
                   taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
               "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ---------------------------------------------------------------------------------
// Descriptors
//
// Shared-memory matrix descriptor (64 bit): start address >>4 in [0,14), leading byte
// offset >>4 in [16,30), stride byte offset >>4 in [32,46), version 1 in [46,48),
// base offset in [49,52), layout type in [61,64) (0 = no swizzle, 2 = 128-byte swizzle).
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1u) << 16;            // LBO unused for swizzled K-major
  d |= static_cast<uint64_t>(1024u >> 4) << 32;    // 8 rows x 128 B between row groups
  d |= static_cast<uint64_t>(1u) << 46;            // descriptor version (sm_100)
  d |= static_cast<uint64_t>(2u) << 61;            // SWIZZLE_128B
  return d;
}
// No-swizzle K-major descriptor: 8-row x 16-byte core matrices, `sbo` bytes between
// 8-row groups, `lbo` bytes between 16-byte K chunks.
__device__ __forceinline__ uint64_t sdesc_plain(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  return d;
}

// Operand formats of kind::mxf8f6f4.
enum : uint32_t { kFmtE4M3 = 0, kFmtE5M2 = 1, kFmtE2M3 = 3, kFmtE3M2 = 4, kFmtE2M1 = 5 };

// Instruction descriptor for tcgen05.mma.kind::mxf8f6f4.block_scale with E8M0 scales,
// K-major A and B, fp32 accumulation. sf ids pick the byte of the 32-bit TMEM scale word.
__host__ __device__ __forceinline__ uint32_t idesc_mxf8f6f4(uint32_t M, uint32_t N, uint32_t afmt,
                                                            uint32_t bfmt, uint32_t a_sf_id,
                                                            uint32_t b_sf_id) {
  uint32_t d = 0;
  d |= (b_sf_id & 3u) << 4;
  d |= (afmt & 7u) << 7;
  d |= (bfmt & 7u) << 10;
  d |= ((N >> 3) & 0x3Fu) << 17;
  d |= 1u << 23;  // scale format E8M0
  d |= ((M >> 4) & 0x1Fu) << 24;
  d |= (a_sf_id & 3u) << 29;
  return d;
}

// D[tmem] (+)= A[smem] * B[smem]^T with per-32 block scales from TMEM.
__device__ __forceinline__ void mma_mxf8f6f4_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                                uint32_t idesc, uint32_t sfa_tmem,
                                                uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::
          "r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
      : "memory");
}
// MMA of a CTA pair (M = 256: rows 0..127 in CTA rank 0, 128..255 in rank 1; B's N rows split
// in halves the same way; D, A and the A scales in each CTA's own tensor memory, the B scales
// of all N rows in each), A from tensor memory, issued by rank 0.
__device__ __forceinline__ void mma_mxf8f6f4_ts_pair(uint32_t d_tmem, uint32_t a_tmem,
                                                     uint64_t bdesc, uint32_t idesc,
                                                     uint32_t sfa_tmem, uint32_t sfb_tmem,
                                                     uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], [%1], %2, %3, [%5], [%6], p;\n\t}\n" ::
          "r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
      : "memory");
}
// Same with the A operand read from tensor memory.
__device__ __forceinline__ void mma_mxf8f6f4_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                                uint32_t idesc, uint32_t sfa_tmem,
                                                uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], [%1], %2, %3, [%5], [%6], p;\n\t}\n" ::
          "r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
      : "memory");
}

// Shared-memory descriptor of a 512-byte scale-factor block (32 rows x 16 bytes, 8-row groups
// 128 bytes apart) for tcgen05.cp 32x128b.
__device__ __forceinline__ uint64_t sdesc_sf(uint32_t saddr) { return sdesc_plain(saddr, 0, 128); }

// Instruction descriptor for tcgen05.mma.kind::mxf4 / mxf4nvf4.block_scale: E2M1 operands, two
// codes per byte, K-major, K = 64, fp32 accumulation. e8m0: scales are E8M0 (else UE4M3); sf ids
// pick the half of the 32-bit TMEM scale word a kind::mxf4 MMA takes (0 or 2).
__host__ __device__ __forceinline__ uint32_t idesc_mxf4(uint32_t M, uint32_t N, bool e8m0,
                                                        uint32_t sf_id) {
  uint32_t d = 0;
  d |= (sf_id & 3u) << 4;
  d |= 1u << 7;   // A: E2M1
  d |= 1u << 10;  // B: E2M1
  d |= ((N >> 3) & 0x3Fu) << 17;
  d |= (e8m0 ? 1u : 0u) << 23;
  d |= ((M >> 4) & 0x1Fu) << 24;
  d |= (sf_id & 3u) << 29;
  return d;
}

// D[tmem] (+)= A[smem] * B[smem]^T of E2M1 codes with block scales from TMEM: kNv with four E4M3
// scales per row (per 16 elements), else two E8M0 (per 32). kPair: the MMA of a CTA pair (M = 256,
// rows of D, A and the A scales split between the CTAs, B's rows split in halves, the B scales of
// all rows in each CTA), issued by rank 0.
template <bool kNv, bool kPair>
__device__ __forceinline__ void mma_mxf4_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                            uint32_t accumulate) {
#define BD_MMA_MXF4(GROUP, KIND, VEC)                                                            \
  asm volatile(                                                                                  \
      "{\n\t.reg .pred p;\n\t"                                                                   \
      "setp.ne.b32 p, %4, 0;\n\t"                                                                \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND ".block_scale.scale_vec::" VEC              \
      " [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::"r"(d_tmem),                                  \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)          \
      : "memory")
  if constexpr (kNv && !kPair) BD_MMA_MXF4("1", "mxf4nvf4", "4X");
  else if constexpr (kNv) BD_MMA_MXF4("2", "mxf4nvf4", "4X");
  else if constexpr (!kPair) BD_MMA_MXF4("1", "mxf4", "2X");
  else BD_MMA_MXF4("2", "mxf4", "2X");
#undef BD_MMA_MXF4
}

// Byte offset of 16-byte chunk `c` of row `r` inside a 128B-swizzled K-major tile whose
// rows are 128 bytes and whose 8-row groups are 1024 bytes apart.
__host__ __device__ __forceinline__ uint32_t sw128_offset(uint32_t r, uint32_t c) {
  return (r >> 3) * 1024u + (r & 7u) * 128u + ((c ^ (r & 7u)) << 4);
}

// Byte offset inside a 512-byte scale-factor block laid out for tcgen05.cp 32x128b:
// row r of a 128-row group, scale block j (0..3) of a 128-wide K chunk.
__host__ __device__ __forceinline__ uint32_t sf_offset(uint32_t r, uint32_t j) {
  return (r & 31u) * 16u + ((r >> 5) & 3u) * 4u + j;
}

}  // namespace bd
