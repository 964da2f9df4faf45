// What the kernels of lora.cu and lora_pair.cu share.
#pragma once
#include "common.cuh"
#include "params.h"

namespace laya {

// Adapter of row m, or -1 (also for every index that names no slot).
DEVI int row_adapter(const LoraParams& p, int m) {
  if (m >= p.rows) return -1;
  const int a = p.index[m / p.index_div];
  return a >= 0 && a < p.slots ? a : -1;
}

// Matrix descriptors as their two words: the upper one is a constant of the
// layout (128-byte swizzle: 8-row groups 1024 bytes apart; 64-byte, the B_a
// chunks' 32 ranks: 512), the lower one the address, to which 32 bytes along
// the rows add 2.
constexpr uint32_t kDesc128 = (1024 >> 4) | 1u << 14 | 2u << 29;
constexpr uint32_t kDesc64 = (512 >> 4) | 1u << 14 | 4u << 29;
DEVI uint32_t desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFF) | 1u << 16; }

// The producer and MMA roles are loops of a whole warp in which one elected
// lane issues: the operands of the tensor instructions then stay in uniform
// registers.  As loops of a single thread, four MMAs took 346 cycles to issue
// whatever their size, more than a 256 x 128 x 64 block takes to compute.
DEVI bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// D (+)= A B^T of one CTA; a, b: lower descriptor words, AH, BH: the upper.
template <uint32_t AH, uint32_t BH>
DEVI void umma1_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %6};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(AH), "n"(BH)
      : "memory");
}
DEVI void umma1_f8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDesc128)
      : "memory");
}

// mbar_wait by a whole warp, with one verdict for its lanes.
DEVI bool warp_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  const uint32_t addr = smem_u32(bar);
  if (__all_sync(0xffffffffu, mbar_try(addr, parity))) return true;
  const uint64_t t0 = globaltimer();
  while (true) {
    if (__all_sync(0xffffffffu, mbar_try(addr, parity))) return true;
    if (__any_sync(0xffffffffu, globaltimer() - t0 > limit_ns)) return false;
  }
}

// Cluster barrier that orders nothing (a release at cluster scope takes over a
// microsecond): used where the CTAs only tell each other that their memory may
// be written; the data comes as bulk copies, counted by an mbarrier.
DEVI void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
DEVI void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
DEVI void cluster_sync_relaxed() {
  cluster_arrive_relaxed();
  cluster_wait();
}
// Shared memory of this CTA to another CTA's of the cluster (16-byte multiples),
// counted on a barrier there.
DEVI void bulk_copy_to_peer(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "r"(smem_u32(src)), "r"(bytes), "r"(bar)
               : "memory");
}
// mbar_wait_cluster by a whole warp, with one verdict for its lanes.
DEVI bool warp_wait_cluster(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  return __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, limit_ns));
}

// The block of a tensor map at (x, y) on its way to L2.
DEVI void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// One ring position: stage and the parity of its current use.
template <int STAGES>
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  DEVI void next() {
    if (++s == STAGES) {
      s = 0;
      phase ^= 1;
    }
  }
};

}  // namespace laya
