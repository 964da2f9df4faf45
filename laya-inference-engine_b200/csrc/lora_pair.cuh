// Projection with adapters for many rows (lora.cu has the mathematics and the
// kernel for few): a persistent kernel over CTA pairs.
//
// A pair owns tiles of 256 rows x BNF features.  Its MMAs are cta_group::2
// (M = 256): each CTA brings its own 128 rows of X as the A operand and half
// of the tile's weight rows as the B operand, so an SM reads 8 KB of shared
// memory per 256 x 256 x 16 step where a lone CTA's 128 x 128 tile reads twice
// that per unit of work; shared-memory bandwidth is what holds the 128 x 128
// tiles of gemm.cu at half of the tensor cores' rate.  Rows sit on the TMEM
// lanes, so an epilogue thread owns one row of the output; it writes to its warp's
// swizzled block of 32 rows x 128 bytes, which a TMA store (residual: a TMA
// addition) or, where the output's rows take no TMA, the lanes along the rows bring
// to memory.  The tensor memory holds two accumulators (FP8 tiles of 256 features:
// one and the adapters' own), and the epilogue of one tile then runs under the MMAs
// of the next.
//
// Adapters: the shrink lists, for each 256-row tile, the adapters its rows use.
// A block of 32 ranks of one of them is V's rows (TMA) against the B_a rows
// (TMA); the builder warps clear the V rows of other adapters before the MMA.
//
// Bound by the tensor cores where there are tiles for every pair, and by the clock
// that the power limit leaves them: 8,192 rows of K 1,024 into 5,248 features 66 us
// (1.33 PFLOP/s; the library's plain product 67) in a short burst of replays and 77
// (79) in a second of them at about 1.5 GHz, 76 and 88 with one adapter of rank 64
// for all, 93 and 108 to 112 with 32 over 64 ragged requests: a block of 32 ranks
// costs its hi and lo halves, as much as 64 of K, for all 256 rows, and such a tile
// has three adapters on average.  With few tiles by latency: 1,536 rows of K 2,624
// into 1,024 15.8 us, 8.8 of them the K blocks (L2 to shared memory, 110 GB/s an SM),
// the rest the chain of the launches, the blocks of the tile's five adapters (0.4 us
// each, from V's load to its MMAs) and the epilogue.
//
// Roles: warp 0 loads, warp 1 of the leader CTA issues the MMAs of both, warps
// 2-3 build V tiles, warps 4-7 are the epilogue.  Every wait is bounded.
#pragma once
#include "common.cuh"
#include "params.h"
#include "launch.h"
#include "lora.cuh"

#include <algorithm>
#include <mutex>

namespace laya {

namespace {

template <int BNF, int KIND>
struct PairCfg {
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BNF / 2 * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // Loads take up to 1.7 us while every SM stores: six stages of 32 KB hide it.
  static constexpr int STAGES = 192 * 1024 / STAGE_BYTES;
  static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
  static constexpr int STAGING_BYTES = 4 * 32 * 128;  // per epilogue warp a block of 32 rows x 128 bytes
  static constexpr int COLS_BYTES = 2 * BNF * 4;     // per column: weight scale, bias
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM = PIPE_BYTES + STAGING_BYTES + BAR_BYTES + COLS_BYTES + 1024;
  static constexpr int K_ELEMS = KIND == kKindBf16 ? 64 : 128;
  // accumulators of one tile: the projection's, and for FP8 the adapters' own
  static constexpr int ACC_COLS = KIND == kKindFp8 ? 2 * BNF : BNF;
  // tiles in tensor memory: the epilogue of one runs under the MMAs of the next
  // (FP8 with 256 features: one after the other)
  static constexpr int TILES = 512 / ACC_COLS < 2 ? 1 : 2;
};

// ------------------------------------------------------------ pair primitives
DEVI void tmem_alloc2(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
}
DEVI void tmem_relinquish2() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
DEVI void tmem_dealloc2(uint32_t taddr) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}
// D (+)= A B^T over the pair; a, b: lower descriptor words, AH, BH: the upper.
template <uint32_t AH, uint32_t BH>
DEVI void umma2_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %6};\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(AH), "n"(BH)
      : "memory");
}
DEVI void umma2_f8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDesc128)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once the MMAs issued so
// far have completed.
DEVI void umma2_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Tile load into this CTA's shared memory that counts on a barrier of either
// CTA of the pair (cluster address).
DEVI void tma2_load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(x), "r"(y), "l"(policy)
      : "memory");
}
DEVI void tma2_load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}
// Arrive on a barrier of either CTA.  (Release at CTA scope is what the V tiles
// need: their writes are made visible to the tensor cores by the proxy fence;
// a release at cluster scope cost about a microsecond per block.)
DEVI void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ------------------------------------------------------------------ epilogue
enum PairEpilogue : int { kPairStore = 0, kPairRope = 1, kPairGeglu = 2, kPairResidual = 3 };

DEVI uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// fp32 tile added to global memory where it lies (one addition per element).
DEVI void tma_add_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// A warp's block of 32 rows x 64 bf16 columns (128-byte swizzle) to rows m0..,
// columns n.. where the output's rows do not take TMA stores (unaligned rows or
// strides, widths that end inside 16 bytes): its lanes store along the rows.
DEVI void store_block(const GemmParams& p, int m0, int n, const uint8_t* block) {
  const int lane = threadIdx.x & 31, rows = min(32, p.M - m0);
  const bool in0 = n + lane < p.N, in1 = n + lane + 32 < p.N;
  const uint8_t* src = block + (lane & 7) * 2;
  const int c0 = lane >> 3, c1 = c0 + 4;
  __nv_bfloat16* dst = p.out + (size_t)m0 * p.ldo + n + lane;
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 8) {
    __nv_bfloat16 a[8], b[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      a[r] = *reinterpret_cast<const __nv_bfloat16*>(src + sw128_offset(r0 + r, c0));
      b[r] = *reinterpret_cast<const __nv_bfloat16*>(src + sw128_offset(r0 + r, c1));
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      __nv_bfloat16* row = dst + (size_t)(r0 + r) * p.ldo;
      if (r0 + r < rows && in0) row[0] = a[r];
      if (r0 + r < rows && in1) row[32] = b[r];
    }
  }
}

// Count and first adapters of a tile's list, loaded together.
struct ListHead {
  int count;
  int4 first;
};

template <int BNF, int KIND, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(256, 1)
    lora_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                     const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap omap, const GemmParams p, const LoraParams lp) {
  using C = PairCfg<BNF, KIND>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + ST * C::A_BYTES;
  uint8_t* staging = smem + C::PIPE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING_BYTES);  // leader: both CTAs' loads of a stage
  uint64_t* empty = full + ST;     // each CTA: the stage's MMAs are done
  uint64_t* vland = empty + ST;    // each CTA: its V rows have arrived
  uint64_t* vfull = vland + ST;    // leader: both CTAs' V tiles are built
  constexpr int NT = C::TILES;
  uint64_t* acc_full = vfull + ST;     // each CTA: [NT]
  uint64_t* acc_empty = acc_full + 2;  // leader: [NT]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  uint32_t* failed = tmem_slot + 1;
  static_assert((4 * ST + 4) * 8 + 8 <= C::BAR_BYTES, "barrier block");
  float* s_ws = reinterpret_cast<float*>(staging + C::STAGING_BYTES + C::BAR_BYTES);
  float* s_bias = s_ws + BNF;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles_m = (p.M + 255) / 256, tiles_n = (p.N + BNF - 1) / BNF, tiles = tiles_m * tiles_n;
  uint32_t* status = p.status ? p.status : &g_op_status;
  const uint64_t limit = wait_limit(p.wait_limit_us);

  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&vland[s], 1);
      mbar_init(&vfull[s], 4);  // two builder warps in each CTA
    }
    for (int b = 0; b < NT; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);  // four epilogue warps in each CTA
    }
    *failed = 0;
    fence_mbar_init();
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&xmap);
    prefetch_tensormap(&bmap);
    prefetch_tensormap(&vmap);
  }
  // All of the tensor memory.  The shrink before may still hold its 256 columns: its
  // CTAs have allocated before they release this kernel and free without waiting for
  // it, so this allocation at most waits for them (their shared memory does not fit
  // beside this kernel's on one SM either).  What came before the shrink is complete.
  // The next kernel is released only after this allocation.
  if (warp == 2) {
    tmem_alloc2(tmem_slot);
    tmem_relinquish2();
  }
  // (the barriers' initialisation is released by its own fence; the rest is this CTA's)
  tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;
  auto give_up = [&](uint32_t code) {
    record_status(status, code);
    atomicExch(failed, 1u);
  };
  // Tiles of 256 rows vary fastest: the pairs at work share weight tiles.
  auto blocks_of = [&](int tm) { return lp.lists[(size_t)tm * kLoraListInts] * lp.chunks; };
  auto head_of = [&](int tm) {
    const int* list = lp.lists + (size_t)tm * kLoraListInts;
    return ListHead{list[0], *reinterpret_cast<const int4*>(list + kLoraListSlots)};
  };
  auto slot_of = [&](const ListHead& h, int tm, int a) {
    return a == 0   ? h.first.x
           : a == 1 ? h.first.y
           : a == 2 ? h.first.z
           : a == 3 ? h.first.w
                    : lp.lists[(size_t)tm * kLoraListInts + kLoraListSlots + a];
  };

  if (warp == 0) {
    // ---- loads.  W, X and B_a were complete before the shrink released this
    // kernel; the lists and V are the shrink's.
    const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
    const bool leader = rank == 0;
    const uint32_t full0 = mapa_shared(smem_u32(full), 0);
    uint32_t g = 0;
    Ring<ST> ring;
    bool ok = true;
    auto stage_free = [&] { return g < ST || warp_wait(&empty[ring.s], ring.phase ^ 1, limit); };
    auto k_blocks = [&](int t) {
      const int m0 = t % tiles_m * 256 + (int)rank * 128, n0 = t / tiles_m * BNF + (int)rank * (BNF / 2);
      for (int kb = 0; kb < p.kblocks; ++kb, ++g, ring.next()) {
        const int s = ring.s;
        if (!(ok = stage_free())) return;
        if (elect_one()) {
          if (leader) mbar_expect_tx(&full[s], 2 * C::STAGE_BYTES);
          tma2_load_2d(sA + s * C::A_BYTES, &xmap, full0 + s * 8, kb * C::K_ELEMS, m0, pol_x);
          tma2_load_2d(sB + s * C::B_BYTES, &wmap, full0 + s * 8, kb * C::K_ELEMS, n0, pol_w);
        }
        __syncwarp();
      }
    };
    auto adapter_blocks = [&](int t, const ListHead& head) {
      const int tm = t % tiles_m;
      const int m0 = tm * 256 + (int)rank * 128, n0 = t / tiles_m * BNF + (int)rank * (BNF / 2);
      const int nb = head.count * lp.chunks;
      for (int b = 0; b < nb; ++b, ++g, ring.next()) {
        const int s = ring.s, c = b % lp.chunks, slot = slot_of(head, tm, b / lp.chunks);
        if (!(ok = stage_free())) return;
        if (elect_one()) {
          if (leader) mbar_expect_tx(&full[s], BNF * 64);
          tma2_load_3d(sB + s * C::B_BYTES, &bmap, full0 + s * 8, c * 32, n0, slot, pol_x);
          mbar_expect_tx(&vland[s], 128 * 128);
          tma_load_2d(sA + s * C::A_BYTES, &vmap, &vland[s], c * 64, m0, pol_w);
        }
        __syncwarp();
      }
    };
    // Both accumulators take their K blocks before the first adapter block has
    // to wait for the shrink.
    const int t1 = NT == 2 && pair + pairs < tiles ? pair + pairs : -1;
    k_blocks(pair);
    if (ok && t1 >= 0) k_blocks(t1);
    griddep_wait();
    if (ok) adapter_blocks(pair, head_of(pair % tiles_m));
    if (ok && t1 >= 0) adapter_blocks(t1, head_of(t1 % tiles_m));
    for (int t = pair + NT * pairs; t < tiles && ok; t += pairs) {
      const ListHead head = head_of(t % tiles_m);  // on its way during the K blocks
      k_blocks(t);
      if (ok) adapter_blocks(t, head);
    }
    if (!ok && lane == 0) give_up(kStatusGemmEmptyTimeout);
    // every stage's last release, so that none is in flight at the exit
    for (uint32_t i = g < ST ? 0 : g - ST; ok && i < g; ++i)
      if (!warp_wait(&empty[i % ST], (i / ST) & 1, limit)) {
        if (lane == 0) give_up(kStatusGemmEmptyTimeout);
        ok = false;
      }
    if (!ok && leader)  // copies of both CTAs still in flight
      for (uint32_t i = g < ST ? 0 : g - ST; i < g; ++i) warp_wait(&full[i % ST], (i / ST) & 1, limit);
  } else if (warp == 1 && rank == 0) {
    // ---- MMAs of the pair
    const uint32_t idesc = KIND == kKindBf16 ? idesc_bf16(256, BNF) : idesc_e4m3(256, BNF);
    const uint32_t idesc2 = idesc_bf16(256, BNF);
    const uint32_t a0 = desc_lo(smem_u32(sA)), b0 = desc_lo(smem_u32(sB));
    uint32_t vphase = 0;
    Ring<ST> ring;
    bool ok = true;
    // n: the tile's place among the pair's tiles
    auto k_blocks = [&](uint32_t n) {
      const uint32_t acc = tmem + n % NT * 256;
      if (n >= NT && !(ok = warp_wait(&acc_empty[n % NT], (n / NT - 1) & 1, limit))) return;
      tc_fence_after();
      for (int kb = 0; kb < p.kblocks; ++kb, ring.next()) {
        const int s = ring.s;
        if (!(ok = warp_wait(&full[s], ring.phase, limit))) return;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t ad = a0 + s * (C::A_BYTES >> 4), bd = b0 + s * (C::B_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (KIND == kKindBf16)
              umma2_f16<kDesc128, kDesc128>(acc, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0);
            else
              umma2_f8(acc, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0);
          }
          umma2_commit(&empty[s]);
        }
        __syncwarp();
      }
    };
    auto adapter_blocks = [&](uint32_t n, int nb) {
      const uint32_t acc2 = tmem + n % NT * 256 + (KIND == kKindFp8 ? BNF : 0);
      for (int b = 0; b < nb; ++b, ring.next()) {
        const int s = ring.s;
        if (!(ok = warp_wait(&full[s], ring.phase, limit)) || !(ok = warp_wait(&vfull[s], (vphase >> s) & 1, limit)))
          return;
        vphase ^= 1u << s;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t ad = a0 + s * (C::A_BYTES >> 4), bd = b0 + s * (C::B_BYTES >> 4);
          umma2_f16<kDesc128, kDesc64>(acc2, ad, bd, idesc2, KIND == kKindBf16 || b > 0);  // hi
          umma2_f16<kDesc128, kDesc64>(acc2, ad + 4, bd, idesc2, 1);                       // lo
          if (lp.rank - (b % lp.chunks) * 32 > 16) {
            umma2_f16<kDesc128, kDesc64>(acc2, ad + 2, bd + 2, idesc2, 1);
            umma2_f16<kDesc128, kDesc64>(acc2, ad + 6, bd + 2, idesc2, 1);
          }
          umma2_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (elect_one()) umma2_commit(&acc_full[n % NT]);
      __syncwarp();
    };
    const int t1 = NT == 2 && pair + pairs < tiles ? pair + pairs : -1;
    k_blocks(0);
    if (ok && t1 >= 0) k_blocks(1);
    griddep_wait();
    if (ok) adapter_blocks(0, blocks_of(pair % tiles_m));
    if (ok && t1 >= 0) adapter_blocks(1, blocks_of(t1 % tiles_m));
    uint32_t n = NT;
    for (int t = pair + NT * pairs; t < tiles && ok; t += pairs, ++n) {
      const int nb = blocks_of(t % tiles_m);  // on its way during the K blocks
      k_blocks(n);
      if (ok) adapter_blocks(n, nb);
    }
    if (!ok && lane == 0) give_up(kStatusGemmFullTimeout);
  } else if (warp == 2 || warp == 3) {
    // ---- V tiles: rows of other adapters (and rows without one) are cleared
    griddep_wait();
    const int r0 = (warp - 2) * 64 + lane;
    uint32_t g = 0, vphase = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int tm = t % tiles_m, m0 = tm * 256 + (int)rank * 128;
      const ListHead head = head_of(tm);
      const int nb = head.count * lp.chunks;
      // the ring positions of the K blocks before: two tiles' before the first
      if (t == pair)
        g = (NT == 2 && pair + pairs < tiles ? 2 : 1) * p.kblocks;
      else if (t >= pair + NT * pairs)
        g += p.kblocks;
      const int own0 = row_adapter(lp, m0 + r0), own1 = row_adapter(lp, m0 + r0 + 32);
      for (int b = 0; b < nb; ++b, ++g) {
        const int s = g % ST, slot = slot_of(head, tm, b / lp.chunks);
        if (!(ok = warp_wait(&vland[s], (vphase >> s) & 1, limit))) {
          if (lane == 0) give_up(kStatusGemmFullTimeout);
          break;
        }
        vphase ^= 1u << s;
        // eight lanes clear a row's 128 bytes (a lane per row would put them
        // all on the same banks)
        const unsigned other0 = __ballot_sync(0xffffffffu, own0 != slot);
        const unsigned other1 = __ballot_sync(0xffffffffu, own1 != slot);
        uint8_t* dst = sA + s * C::A_BYTES + (warp - 2) * 64 * 128 + lane * 16;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const unsigned m = (j < 8 ? other0 : other1) >> (j % 8 * 4);
          if (m >> (lane >> 3) & 1) *reinterpret_cast<uint4*>(dst + j * 512) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) arrive_cluster(mapa_shared(smem_u32(&vfull[s]), 0));
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue: a thread has one row; 64 bf16 (residual: 32 fp32) columns
    // at a time go through a swizzled block to a TMA store of the warp's 32 rows
    griddep_wait();
    const int lq = warp - 4;
    uint8_t* dst = staging + lq * 32 * 128;
    uint32_t n = 0;
    for (int t = pair; t < tiles; t += pairs, ++n) {
      const int tm = t % tiles_m, tn = t / tiles_m, buf = n % NT;
      const int mw = tm * 256 + (int)rank * 128 + lq * 32, m = mw + lane, n0 = tn * BNF;
      const bool second = KIND == kKindFp8 && blocks_of(tm) > 0;
      const float sa = KIND == kKindFp8 && m < p.M ? p.a_scale[m] : 1.f;
      if (KIND == kKindFp8 || p.bias) {
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the last tile's columns are no longer read
        for (int i = tid - 128; i < BNF; i += 128) {
          const bool in = n0 + i < p.N;
          if (KIND == kKindFp8) s_ws[i] = in ? p.w_scale[n0 + i] : 0.f;
          if (p.bias) s_bias[i] = in ? __bfloat162float(p.bias[n0 + i]) : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      float cs[EPI == kPairRope ? 32 : 1], sn[EPI == kPairRope ? 32 : 1];
      if (EPI == kPairRope && n0 < p.rope_cols) {
        // the tables repeat their first 32 columns (cat(freqs, freqs))
        const float4* c4 = reinterpret_cast<const float4*>(p.rope_cos + (size_t)(m % p.rope_seq) * 64);
        const float4* s4 = reinterpret_cast<const float4*>(p.rope_sin + (size_t)(m % p.rope_seq) * 64);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 a = c4[j], b = s4[j];
          cs[4 * j] = a.x; cs[4 * j + 1] = a.y; cs[4 * j + 2] = a.z; cs[4 * j + 3] = a.w;
          sn[4 * j] = b.x; sn[4 * j + 1] = b.y; sn[4 * j + 2] = b.z; sn[4 * j + 3] = b.w;
        }
      }
      if (!warp_wait(&acc_full[buf], n / NT & 1, limit)) {
        if (lane == 0) give_up(kStatusGemmDoneTimeout);
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + buf * 256 + ((uint32_t)(lq * 32) << 16);
      // 32 finished sums of the row, columns c.. of the tile
      auto sums = [&](int c, float (&v)[32]) {
        uint32_t r[32];
        tmem_ld32(acc + c, r);
        if (second) {
          uint32_t q[32];
          tmem_ld32(acc + BNF + c, q);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = (__uint_as_float(r[j]) * sa) * s_ws[c + j] + __uint_as_float(q[j]);
        } else {
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            v[j] = __uint_as_float(r[j]);
            if (KIND == kKindFp8) v[j] = (v[j] * sa) * s_ws[c + j];
          }
        }
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += s_bias[c + j];
        }
      };
      constexpr int STEP = EPI == kPairGeglu ? 128 : EPI == kPairResidual ? 32 : 64;
#pragma unroll 1
      for (int c = 0; c < BNF && n0 + c < p.N; c += STEP) {
        auto put = [&](int j, uint32_t a, uint32_t b, uint32_t d, uint32_t e) {
          *reinterpret_cast<uint4*>(dst + sw128_offset(lane, j)) = make_uint4(a, b, d, e);
        };
        // the last store has finished reading the block by the time the sums are
        // here; nothing is written to it before
        auto block_free = [&] {
          if (lane == 0) bulk_wait_read0();
          __syncwarp();
        };
        if constexpr (EPI == kPairResidual) {
          float v[32];
          sums(c, v);
          block_free();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            put(j, __float_as_uint(bf16_round(v[4 * j])), __float_as_uint(bf16_round(v[4 * j + 1])),
                __float_as_uint(bf16_round(v[4 * j + 2])), __float_as_uint(bf16_round(v[4 * j + 3])));
        } else if constexpr (EPI == kPairGeglu) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float a[32], g[32];
            sums(c + 32 * h, a);
            sums(c + 64 + 32 * h, g);
#pragma unroll
            for (int j = 0; j < 32; ++j) a[j] = bf16_round(gelu_erf(bf16_round(a[j]))) * bf16_round(g[j]);
            if (h == 0) block_free();
#pragma unroll
            for (int j = 0; j < 4; ++j)
              put(4 * h + j, pack_bf16(a[8 * j], a[8 * j + 1]), pack_bf16(a[8 * j + 2], a[8 * j + 3]),
                  pack_bf16(a[8 * j + 4], a[8 * j + 5]), pack_bf16(a[8 * j + 6], a[8 * j + 7]));
          }
        } else {
          float v[2][32];
          sums(c, v[0]);
          sums(c + 32, v[1]);
          if (EPI == kPairRope && n0 + c < p.rope_cols) {
            // bf16(qkv) rotated in fp32 without FMA, as rope_qkv does (kernels.py:62-93)
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float a = bf16_round(v[0][j]), b = bf16_round(v[1][j]);
              v[0][j] = __fadd_rn(__fmul_rn(a, cs[j]), __fmul_rn(-b, sn[j]));
              v[1][j] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
            }
          }
          block_free();
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              put(4 * h + j, pack_bf16(v[h][8 * j], v[h][8 * j + 1]), pack_bf16(v[h][8 * j + 2], v[h][8 * j + 3]),
                  pack_bf16(v[h][8 * j + 4], v[h][8 * j + 5]), pack_bf16(v[h][8 * j + 6], v[h][8 * j + 7]));
        }
        if (mw >= p.M) continue;
        if (EPI != kPairStore || p.tma_epilogue) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (EPI == kPairResidual)
              tma_add_2d(&omap, dst, n0 + c, mw);
            else
              tma_store_2d(&omap, dst, EPI == kPairGeglu ? (n0 + c) / 2 : n0 + c, mw);
            bulk_commit();
          }
        } else {
          __syncwarp();
          store_block(p, mw, n0 + c, dst);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(mapa_shared(smem_u32(&acc_empty[buf]), 0));
    }
    if (lane == 0) bulk_wait_read0();
  }
  __syncwarp();
  griddep_wait();
  tc_fence_before();
  // no CTA leaves while its partner may still signal it (with a release: the
  // signals are to have arrived)
  cluster_sync_all();
  if (warp == 2) tmem_dealloc2(tmem);
}

template <int BNF, int KIND, int EPI>
cudaError_t launch_pairs(const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, cudaStream_t stream) {
  using C = PairCfg<BNF, KIND>;
  auto kern = lora_pair_kernel<BNF, KIND, EPI>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  // Per device, once: the shared-memory limit, and how many pairs run at a time.
  static std::mutex mu;
  static int resident[64] = {};
  int dev = 0, pairs = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64) return cudaErrorInvalidDevice;
    if (!resident[dev]) {
      err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
      if (err != cudaSuccess) return err;
      cfg.gridDim = dim3(2, 1, 1);
      err = cudaOccupancyMaxActiveClusters(&resident[dev], kern, &cfg);
      if (err != cudaSuccess) return err;
      if (resident[dev] < 1) return cudaErrorInvalidConfiguration;
    }
    pairs = resident[dev];
  }
  const long long tiles = (long long)((p.M + 255) / 256) * ((p.N + BNF - 1) / BNF);
  if (tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  cfg.gridDim = dim3((unsigned)(2 * std::min<long long>(tiles, pairs)), 1, 1);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, maps.w, maps.x, maps.b, maps.v, maps.out, p, lp);
}

template <int BNF, int KIND>
cudaError_t launch_epilogue(const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, cudaStream_t stream) {
  if (p.epilogue == kEpiStore && !p.rope_cols) return launch_pairs<BNF, KIND, kPairStore>(maps, p, lp, stream);
  // the engine's epilogues: whole tiles of features, TMA output
  if (p.N % 128 || !p.tma_epilogue || p.bias) return cudaErrorInvalidValue;
  if (p.epilogue == kEpiStore) return launch_pairs<BNF, KIND, kPairRope>(maps, p, lp, stream);
  if (p.epilogue == kEpiGeglu) return launch_pairs<BNF, KIND, kPairGeglu>(maps, p, lp, stream);
  if (p.epilogue == kEpiResidual) return launch_pairs<BNF, KIND, kPairResidual>(maps, p, lp, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

// Waves of tiles times a tile's cost.  A K block takes 0.31 us of a pair with 256
// features and 0.215 with 128 (shared-memory and L2 bandwidth; FP8's hold twice
// the columns), the epilogue 2.4 us, which only FP8 tiles of 256 features do not
// hide under the next tile.
float lora_pair_us(int kind, int M, int N, int kblocks, int bnf, int sm_count) {
  const long long tiles = (long long)((M + 255) / 256) * ((N + bnf - 1) / bnf);
  const float waves = (float)((tiles + sm_count / 2 - 1) / (sm_count / 2)), epilogue = 2.4f;
  const float k = (float)kblocks * (bnf == 256 ? 0.31f : 0.215f);
  return kind == kKindFp8 && bnf == 256 ? waves * (k + epilogue) : waves * k + epilogue;
}
int lora_pair_ctas(int M, int N, int bnf, int sm_count) {
  const long long tiles = (long long)((M + 255) / 256) * ((N + bnf - 1) / bnf);
  return (int)std::min<long long>(2 * tiles, sm_count);
}

cudaError_t launch_lora_pairs(int kind, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int bnf,
                              cudaStream_t stream) {
  if (p.M < 1 || p.N < 1 || lp.rows != p.M || !lp.lists) return cudaErrorInvalidValue;
  if (kind == kKindBf16 && bnf == 256) return launch_epilogue<256, kKindBf16>(maps, p, lp, stream);
  if (kind == kKindBf16 && bnf == 128) return launch_epilogue<128, kKindBf16>(maps, p, lp, stream);
  if (kind == kKindFp8 && bnf == 256) return launch_epilogue<256, kKindFp8>(maps, p, lp, stream);
  if (kind == kKindFp8 && bnf == 128) return launch_epilogue<128, kKindFp8>(maps, p, lp, stream);
  return cudaErrorInvalidValue;
}

}  // namespace laya
