// Projection with the low-rank adapters of many requests beside the shared
// weight:
//
//   out[m] = X[m] W^T + s_a (X[m] A_a^T) B_a^T,   a = index[m / index_div]
//
// in two launches.  lora_shrink_kernel computes V[m] = s_a X[m] A_a^T (a few
// ranks per row).  lora_gemm_kernel is the projection of gemm.cu with its
// reduction axis lengthened: after the K blocks of W it takes, for every
// adapter that a row of its token tile uses, the blocks of B_a (TMA) against
// the rows V of that adapter, zero for the tile's other rows (built in shared
// memory), into the same TMEM accumulator.  So the adapters cost no pass over
// the output and no accumulator of their own, a tile whose rows share one
// adapter pays rank / K of the projection's matrix work, and a tile of single
// rows with an adapter each pays the bytes of those adapters, which nobody
// can avoid.
//
// The shrink releases the projection once its own inputs are complete, so the
// projection's K blocks run beside it and only the adapter blocks wait for V.
//
// V is kept as bf16 pairs hi + lo (hi = bf16(v), lo = bf16(v - hi)), about 16
// bits: a single bf16 V would round the adapter's term once more, by as much as
// the output's own rounding where the adapter dominates.  A chunk of 32 ranks
// is one 128-byte row [hi 32 | lo 32] of a swizzled operand tile.
//
// FP8 projections keep the adapters in bf16: their blocks go to a second
// accumulator, and the epilogue adds it to the scaled first one.
#include "common.cuh"
#include "params.h"
#include "launch.h"
#include "gemm_epilogue.cuh"

#include <mutex>

namespace laya {

// Status of launches that were given no status word (laya_b200_op_status).
__device__ uint32_t g_op_status;

namespace {

// Adapter of row m, or -1 (also for every index that names no slot).
DEVI int row_adapter(const LoraParams& p, int m) {
  if (m >= p.rows) return -1;
  const int a = p.index[m / p.index_div];
  return a >= 0 && a < p.slots ? a : -1;
}

// ------------------------------------------------------------------ shrink
// A CTA takes 16 rows, RG ranks (grid.z) and every `gridDim.y`-th of the
// adapters that its rows use.  Its eight warps split K; a lane loads 16 bytes
// of rows lane/4 and lane/4 + 8 and of ranks lane/4 + 8j at the same columns,
// which are the operands of two m16n8k16 products over a permuted K (the
// order of a sum's terms is free as long as both operands share it), so no
// staging is needed.  The partial sums meet in shared memory in warp order.
constexpr int kShrinkRows = 16, kShrinkWarps = 8;

DEVI void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>  // rank group of 8 * NT
__global__ void __launch_bounds__(32 * kShrinkWarps) lora_shrink_kernel(const LoraParams p) {
  constexpr int RG = 8 * NT;
  __shared__ float red[kShrinkWarps][kShrinkRows][RG];
  // Everything before this kernel is complete once the wait returns; the
  // projection launched behind it relies on that (its K blocks do not wait).
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * kShrinkRows, r0 = blockIdx.z * RG;
  const int mine = lane < kShrinkRows ? row_adapter(p, row0 + lane) : -1;
  const unsigned same = __match_any_sync(0xffffffffu, mine);
  unsigned firsts = __ballot_sync(0xffffffffu, mine >= 0 && __ffs(same) - 1 == lane);
  const int g = lane >> 2, t8 = (lane & 3) * 8;
  const int ra = row0 + g, rb = ra + 8;
  const __nv_bfloat16* xa = p.x + (size_t)(ra < p.rows ? ra : 0) * p.ldx;
  const __nv_bfloat16* xb = p.x + (size_t)(rb < p.rows ? rb : 0) * p.ldx;
  const int steps = (p.in_features + 31) / 32;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int ordinal = 0; firsts; ++ordinal, firsts &= firsts - 1) {
    if (ordinal % gridDim.y != blockIdx.y) continue;
    const int slot = __shfl_sync(0xffffffffu, mine, __ffs(firsts) - 1);
    const __nv_bfloat16* a = p.a + (size_t)slot * p.rank * p.in_features;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 2
    for (int s = warp; s < steps; s += kShrinkWarps) {
      const int k = s * 32 + t8;
      const bool in = k < p.in_features;
      const uint4 va = in && ra < p.rows ? *reinterpret_cast<const uint4*>(xa + k) : zero;
      const uint4 vb = in && rb < p.rows ? *reinterpret_cast<const uint4*>(xb + k) : zero;
      uint4 w[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = r0 + 8 * j + g;
        w[j] = in && r < p.rank ? __ldg(reinterpret_cast<const uint4*>(a + (size_t)r * p.in_features + k)) : zero;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma_bf16(acc[j], va.x, vb.x, va.y, vb.y, w[j].x, w[j].y);
        mma_bf16(acc[j], va.z, vb.z, va.w, vb.w, w[j].z, w[j].w);
      }
    }
    const int c = (lane & 3) * 2;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      *reinterpret_cast<float2*>(&red[warp][g][8 * j + c]) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(&red[warp][g + 8][8 * j + c]) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    const float scaling = p.scaling ? p.scaling[slot] : 1.f;
#pragma unroll 1
    for (int i = threadIdx.x; i < kShrinkRows * RG; i += 32 * kShrinkWarps) {
      const int row = i / RG, r = r0 + i % RG;
      // i / RG is the same for a warp's lanes or differs by whole rows; the
      // row's adapter comes from the lane that holds it
      const int owner = __shfl_sync(0xffffffffu, mine, row);
      if (owner != slot || (r >> 5) >= p.chunks) continue;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kShrinkWarps; ++w) v += red[w][row][i % RG];
      v *= scaling;
      const __nv_bfloat16 hi = __float2bfloat16_rn(v);
      // an infinite (or NaN) v has no remainder
      const float rest = fabsf(v) < INFINITY ? v - __bfloat162float(hi) : 0.f;
      __nv_bfloat16* dst = p.v + ((size_t)(row0 + row) * p.chunks + (r >> 5)) * 64 + (r & 31);
      dst[0] = hi;
      dst[32] = __float2bfloat16_rn(rest);
    }
    __syncthreads();
  }
}

// -------------------------------------------------------------- projection
// B_a chunk: 128 weight rows x 32 ranks in the 64-byte swizzle TMA writes
// (8-row groups 512 bytes apart).
DEVI uint64_t sw64_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(512 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)4 << 61;  // 64-byte swizzle
  return d;
}

template <int BN, int KIND, int STAGES>
struct LoraCfg {
  static constexpr int THREADS = BN >= 128 ? 256 : 128;
  static constexpr int BUILDERS = THREADS - 64;  // threads of warps 2.. build the V tiles
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
  static constexpr int PART_BYTES = BN * 128 * 4;
  static constexpr int MAIN_BYTES = PIPE_BYTES > PART_BYTES ? PIPE_BYTES : PART_BYTES;
  static constexpr int LIST_BYTES = BN * 12;  // adapter per row, distinct adapters, activation scales
  static constexpr int BAR_BYTES = 256;
  static constexpr int SMEM = MAIN_BYTES + BAR_BYTES + LIST_BYTES + 1024;
  static constexpr int ACCS = KIND == kKindFp8 ? 2 : 1;
  static constexpr int TMEM_COLS = BN * ACCS < 32 ? 32 : BN * ACCS;
  static constexpr int K_ELEMS = KIND == kKindBf16 ? 64 : 128;
};

// Store of one row's four columns n..n+3 (fewer at the matrix's end).
DEVI void store_quad(const GemmParams& p, int m, int n, float4 v, bool vec) {
  if (n >= p.N) return;
  float x[4] = {v.x, v.y, v.z, v.w};
  __nv_bfloat16 o[4];
  const int left = p.N - n < 4 ? p.N - n : 4;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (p.bias && e < left) x[e] += __bfloat162float(p.bias[n + e]);
    o[e] = __float2bfloat16_rn(x[e]);
  }
  __nv_bfloat16* dst = p.out + (size_t)m * p.ldo + n;
  if (vec && left == 4) {
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) dst[e] = o[e];
  }
}

template <int BN, int KIND, int STAGES>
__global__ void __launch_bounds__(LoraCfg<BN, KIND, STAGES>::THREADS, BN == 128 ? 2 : 1)
    lora_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                     const __grid_constant__ CUtensorMap bmap, const GemmParams p, const LoraParams lp) {
  using C = LoraCfg<BN, KIND, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::MAIN_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* vfull = empty + STAGES;
  uint64_t* vfree = vfull + STAGES;  // the producer found the stage free for an adapter block
  uint64_t* done = vfree + STAGES;
  uint64_t* listed = done + 1;  // the tile's adapter list is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(listed + 1);
  uint32_t* failed = tmem_slot + 1;
  int* s_count = reinterpret_cast<int*>(failed + 1);  // [0]: distinct adapters, [1..4]: per warp
  static_assert((4 * STAGES + 2) * 8 + 8 + 5 * 4 <= C::BAR_BYTES, "barrier block");
  int* s_row = reinterpret_cast<int*>(smem + C::MAIN_BYTES + C::BAR_BYTES);  // [BN] adapter of each row
  int* s_list = s_row + BN;                                                  // [BN] distinct adapters
  float* s_scale = reinterpret_cast<float*>(s_list + BN);                    // [BN] activation scales (fp8)

  const int tid = threadIdx.x, warp = tid >> 5;
  const int tile_n = blockIdx.x, tile_m = blockIdx.y;
  const int split = gridDim.z, rank = blockIdx.z;
  const int kb0 = (int)((long long)rank * p.kblocks / split);
  const int kb1 = (int)((long long)(rank + 1) * p.kblocks / split);
  const int nkb = kb1 - kb0;
  uint32_t* status = p.status ? p.status : &g_op_status;

  griddep_launch_dependents();

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&vfull[s], C::BUILDERS);
      mbar_init(&vfree[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(listed, 1);
    *failed = 0;
    fence_mbar_init();
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&xmap);
    prefetch_tensormap(&bmap);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem2 = tmem + (C::ACCS - 1) * BN;  // the adapters' accumulator

  const uint64_t limit = wait_limit(p.wait_limit_us);
  int issued = 0;  // producer: loads issued (for the drain on failure)
  // This rank's share [b0, b1) of the tile's adapter blocks (adapter, chunk of
  // 32 ranks); known once `listed` has completed.
  auto blocks = [&](int& b0, int& b1) {
    const int n = s_count[0] * lp.chunks;
    b0 = (int)((long long)rank * n / split);
    b1 = (int)((long long)(rank + 1) * n / split);
  };
  auto give_up = [&](uint32_t code) {
    record_status(status, code);
    atomicExch(failed, 1u);
  };
  if (tid == 0) {
    // W, X and B_a do not wait for the shrink: whatever wrote them was
    // complete before it released this kernel.
    const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int s = i % STAGES;
      if (i >= STAGES && !mbar_wait(&empty[s], ((i / STAGES) - 1) & 1, limit)) {
        give_up(kStatusGemmEmptyTimeout);
        ok = false;
        break;
      }
      mbar_expect_tx(&full[s], C::STAGE_BYTES);
      tma_load_2d(sA + s * C::A_BYTES, &wmap, &full[s], (kb0 + i) * C::K_ELEMS, tile_n * 128, pol_w);
      tma_load_2d(sB + s * C::B_BYTES, &xmap, &full[s], (kb0 + i) * C::K_ELEMS, tile_m * BN, pol_x);
      issued = i + 1;
    }
    if (ok && !mbar_wait(listed, 0, limit)) {
      give_up(kStatusGemmFullTimeout);
      ok = false;
    }
    if (ok) {
      int b0, b1;
      blocks(b0, b1);
      for (int b = b0; b < b1; ++b) {
        const int i = nkb + b - b0, s = i % STAGES;
        if (i >= STAGES && !mbar_wait(&empty[s], ((i / STAGES) - 1) & 1, limit)) {
          give_up(kStatusGemmEmptyTimeout);
          break;
        }
        mbar_arrive(&vfree[s]);
        mbar_expect_tx(&full[s], 128 * 64);
        tma_load_3d(sA + s * C::A_BYTES, &bmap, &full[s], (b % lp.chunks) * 32, tile_n * 128, s_list[b / lp.chunks],
                    pol_x);
        issued = i + 1;
      }
    }
  } else if (tid == 32) {
    const uint32_t idesc = KIND == kKindBf16 ? idesc_bf16(128, BN) : idesc_e4m3(128, BN);
    bool ok = true;
    int b0 = 0, b1 = 0, total = nkb;
    for (int i = 0; i < nkb && ok; ++i) {
      const int s = i % STAGES;
      if (!mbar_wait(&full[s], (i / STAGES) & 1, limit)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t ad = sw128_desc(smem_u32(sA + s * C::A_BYTES));
      const uint64_t bd = sw128_desc(smem_u32(sB + s * C::B_BYTES));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (KIND == kKindBf16)
          umma_f16(tmem, ad + 2 * k, bd + 2 * k, idesc, (i | k) != 0);
        else
          umma_f8(tmem, ad + 2 * k, bd + 2 * k, idesc, (i | k) != 0);
      }
      // Only stages that are refilled get a release (nothing is left in
      // flight when the CTA exits); near the end that takes the block count.
      if (i + STAGES >= nkb && total == nkb && b1 == 0) {
        if (!mbar_wait(listed, 0, limit)) {
          ok = false;
          break;
        }
        blocks(b0, b1);
        total = nkb + b1 - b0;
      }
      if (i + STAGES < total) umma_commit(&empty[s]);
    }
    for (int b = b0; b < b1 && ok; ++b) {
      const int i = nkb + b - b0, s = i % STAGES;
      if (!mbar_wait(&full[s], (i / STAGES) & 1, limit) ||
          !mbar_wait(&vfull[s], ((i - nkb) / STAGES) & 1, limit)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t ad = sw64_desc(smem_u32(sA + s * C::A_BYTES));
      const uint64_t bd = sw128_desc(smem_u32(sB + s * C::B_BYTES));
      const int left = lp.rank - (b % lp.chunks) * 32;
      const int ksteps = left > 16 ? 2 : 1;
      const uint32_t id2 = idesc_bf16(128, BN);
      for (int k = 0; k < ksteps; ++k) {
        umma_f16(tmem2, ad + 2 * k, bd + 2 * k, id2, KIND == kKindBf16 || b > b0 || k > 0);  // hi
        umma_f16(tmem2, ad + 2 * k, bd + 4 + 2 * k, id2, 1);                                 // lo
      }
      if (i + STAGES < total) umma_commit(&empty[s]);
    }
    if (!ok) give_up(kStatusGemmFullTimeout);
    umma_commit(done);
  } else if (warp >= 2) {
    // ---- the tile's adapters in order of first use, then their V tiles
    static_assert(BN <= C::BUILDERS, "a builder thread per row");
    const int bt = tid - 64, lane = tid & 31, bw = bt >> 5;
    int owner = -1;
    if (bt < BN) {
      owner = row_adapter(lp, tile_m * BN + bt);
      s_row[bt] = owner;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(C::BUILDERS) : "memory");
    bool first = bt < BN && owner >= 0;
    for (int j = 0; first && j < bt; ++j) first = s_row[j] != owner;
    const unsigned bal = __ballot_sync(0xffffffffu, first);
    if (lane == 0 && bw < 4) s_count[1 + bw] = __popc(bal);
    asm volatile("bar.sync 1, %0;" ::"n"(C::BUILDERS) : "memory");
    constexpr int ROW_WARPS = (BN + 31) / 32;
    int before = 0, n = 0;
    for (int j = 0; j < ROW_WARPS; ++j) {
      if (j < bw) before += s_count[1 + j];
      n += s_count[1 + j];
    }
    if (first) s_list[before + __popc(bal & ((1u << lane) - 1))] = owner;
    if (bt == 0) s_count[0] = n;
    asm volatile("bar.sync 1, %0;" ::"n"(C::BUILDERS) : "memory");
    if (bt == 0) mbar_arrive(listed);
    int b0, b1;
    blocks(b0, b1);
    griddep_wait();  // V
    for (int b = b0; b < b1; ++b) {
      const int i = nkb + b - b0, s = i % STAGES;
      // (the builders cannot wait on `empty` themselves: they have not followed
      // its phases through the K blocks, and a parity names every second one)
      if (!mbar_wait(&vfree[s], ((i - nkb) / STAGES) & 1, limit)) {
        give_up(kStatusGemmEmptyTimeout);
        break;
      }
      const int slot = s_list[b / lp.chunks], c = b % lp.chunks;
      uint8_t* dst = sB + s * C::B_BYTES;
      for (int u = bt; u < BN * 8; u += C::BUILDERS) {
        const int row = u >> 3, j = u & 7;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (s_row[row] == slot)
          v = *reinterpret_cast<const uint4*>(lp.v + ((size_t)(tile_m * BN + row) * lp.chunks + c) * 64 + j * 8);
        *reinterpret_cast<uint4*>(dst + sw128_offset(row, j)) = v;
      }
      fence_proxy_async_smem();
      mbar_arrive(&vfull[s]);
    }
  }
  __syncwarp();

  // ---- epilogue: TMEM -> fp32 tile [BN][128] -> cluster reduction -> store
  griddep_wait();
  if (KIND == kKindFp8)
    for (int i = tid; i < BN; i += C::THREADS) s_scale[i] = tile_m * BN + i < p.M ? p.a_scale[tile_m * BN + i] : 0.f;
  if (!mbar_wait(done, 0, limit)) give_up(kStatusGemmDoneTimeout);
  tc_fence_after();
  __syncthreads();
  const bool gpath = split > 1 && p.partials != nullptr;
  float* part = reinterpret_cast<float*>(smem);
  if (gpath) part = p.partials + ((size_t)(tile_m * gridDim.x + tile_n) * split + rank) * BN * 128;
  {
    int b0, b1;
    blocks(b0, b1);
    const bool second = KIND == kKindFp8 && b1 > b0;
    const int lq = warp & 3;
    constexpr int HALVES = C::THREADS / 128;
    constexpr int COLS = BN / HALVES;
    const int c0 = (warp >> 2) * COLS;
    const int lr = lq * 32 + (tid & 31);  // weight row of the tile
    const uint32_t lane_addr = (uint32_t)(lq * 32) << 16;
    const float ws = KIND == kKindFp8 && tile_n * 128 + lr < p.N ? p.w_scale[tile_n * 128 + lr] : 1.f;
    constexpr int W = COLS < 32 ? 16 : 32;
#pragma unroll 1
    for (int c = c0; c < c0 + COLS; c += W) {
      uint32_t r[W], q[W];
      if constexpr (W == 32) tmem_ld32(tmem + lane_addr + c, r); else tmem_ld16(tmem + lane_addr + c, r);
      if (second) {
        if constexpr (W == 32) tmem_ld32(tmem2 + lane_addr + c, q); else tmem_ld16(tmem2 + lane_addr + c, q);
      }
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < W; ++j) {
        float v = __uint_as_float(r[j]);
        if (KIND == kKindFp8) {
          v = (v * s_scale[c + j]) * ws;
          if (second) v += __uint_as_float(q[j]);
        }
        part[(c + j) * 128 + lr] = v;
      }
    }
  }
  tc_fence_before();
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  {
    const int t0 = rank * BN / split, t1 = (rank + 1) * BN / split;
    const uint32_t part_addr = smem_u32(part);
    const bool rope = tile_n * 128 < p.rope_cols;
    const int pair = rope ? 32 : 64;
    const bool residual = p.epilogue == kEpiResidual;
    const bool plain = p.epilogue == kEpiStore && !rope;
    const bool vec = p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
    for (int item = tid; item < (t1 - t0) * 16; item += C::THREADS) {
      const int tl = t0 + (item >> 4);
      const int q4 = rope ? ((item >> 3) & 1) * 64 + (item & 7) * 4 : (item & 15) * 4;
      const int m = tile_m * BN + tl, n = tile_n * 128 + q4;
      if (m >= p.M) continue;
      const int off = tl * 128 + q4;
      EpiPre pre;
      if (!plain) pre = epi_prefetch<kKindBf16>(p, m, n, residual, rope);
      float4 lo, hi;
      if (split == 1) {
        lo = *reinterpret_cast<const float4*>(part + off);
        hi = *reinterpret_cast<const float4*>(part + off + pair);
      } else {
        lo = hi = make_float4(0.f, 0.f, 0.f, 0.f);
        float4 va[8], vb[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (u < split) {
            if (gpath) {
              const float* src = p.partials + ((size_t)(tile_m * gridDim.x + tile_n) * split + u) * BN * 128 + off;
              va[u] = __ldcg(reinterpret_cast<const float4*>(src));
              vb[u] = __ldcg(reinterpret_cast<const float4*>(src + pair));
            } else {
              const uint32_t base = mapa_shared(part_addr, (uint32_t)u);
              va[u] = ld_dsmem_f32x4(base + off * 4);
              vb[u] = ld_dsmem_f32x4(base + (off + pair) * 4);
            }
          }
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (u < split) {
            lo.x += va[u].x; lo.y += va[u].y; lo.z += va[u].z; lo.w += va[u].w;
            hi.x += vb[u].x; hi.y += vb[u].y; hi.z += vb[u].z; hi.w += vb[u].w;
          }
      }
      if (plain) {
        store_quad(p, m, n, lo, vec);
        store_quad(p, m, n + 64, hi, vec);
      } else if (rope) {
        epilogue_rope<kKindBf16>(p, m, n, lo, hi, pre);
      } else {
        epilogue_quad<kKindBf16>(p, m, n, tile_n * 64 + q4, lo, hi, pre);
      }
    }
  }
  if (split > 1 && !gpath) cluster_sync_all();

  // ---- teardown: drain copies still in flight after a failure, free TMEM
  if (tid == 0 && *failed) {
    for (int i = (issued > STAGES ? issued - STAGES : 0); i < issued; ++i)
      mbar_wait(&full[i % STAGES], (i / STAGES) & 1, limit);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, C::TMEM_COLS);
}

// ------------------------------------------------------------------ host side

template <int BN, int KIND, int STAGES>
cudaError_t launch_one(const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& bmap, const GemmParams& p,
                       const LoraParams& lp, int split, cudaStream_t stream) {
  using C = LoraCfg<BN, KIND, STAGES>;
  auto kern = lora_gemm_kernel<BN, KIND, STAGES>;
  // Function attributes are per device: set them once for each device used.
  static std::mutex mu;
  static uint64_t ready = 0;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!(ready >> dev & 1)) {
      err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
      if (err != cudaSuccess) return err;
      ready |= uint64_t(1) << dev;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + 127) / 128, (p.M + BN - 1) / BN, split);
  cfg.blockDim = dim3(C::THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (split > 1) {
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = 1;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = split;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attrs;
  return cudaLaunchKernelEx(&cfg, kern, wmap, xmap, bmap, p, lp);
}

template <int KIND>
cudaError_t dispatch_bn(int bn, const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& bmap,
                        const GemmParams& p, const LoraParams& lp, int split, cudaStream_t st) {
  switch (bn) {
    case 16: return launch_one<16, KIND, 4>(wmap, xmap, bmap, p, lp, split, st);
    case 32: return launch_one<32, KIND, 4>(wmap, xmap, bmap, p, lp, split, st);
    case 64: return launch_one<64, KIND, 4>(wmap, xmap, bmap, p, lp, split, st);
    case 128: return launch_one<128, KIND, 3>(wmap, xmap, bmap, p, lp, split, st);
  }
  return cudaErrorInvalidValue;
}

template <int NT>
cudaError_t shrink_one(const LoraParams& p, int slices, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.rows + kShrinkRows - 1) / kShrinkRows, slices, (p.rank + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(32 * kShrinkWarps, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, lora_shrink_kernel<NT>, p);
}

}  // namespace

cudaError_t launch_lora_shrink(const LoraParams& p, int sm_count, cudaStream_t stream, bool pdl) {
  if (p.rows < 1 || p.rank < 8 || p.rank % 8 || p.rank > kLoraMaxRank || p.in_features % 8 || p.slots < 1 ||
      p.index_div < 1)
    return cudaErrorInvalidValue;
  // Few rows: the adapters of a row tile are spread over CTAs (16 single rows
  // may each bring one), up to about two CTAs per SM.
  const int tiles = (p.rows + kShrinkRows - 1) / kShrinkRows;
  int slices = 2 * sm_count / tiles;
  if (slices > kShrinkRows) slices = kShrinkRows;
  if (slices > p.rows) slices = p.rows;
  if (slices > p.slots) slices = p.slots;
  if (slices < 1) slices = 1;
  if (p.rank <= 16) return shrink_one<2>(p, slices, stream, pdl);
  if (p.rank <= 32) return shrink_one<4>(p, slices, stream, pdl);
  return shrink_one<8>(p, slices, stream, pdl);
}

cudaError_t launch_lora_gemm(int kind, const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& bmap,
                             const GemmParams& p, const LoraParams& lp, int bn, int split, cudaStream_t stream) {
  if (p.M < 1 || p.N < 1 || split < 1 || split > 8 || split > p.kblocks || lp.rows != p.M)
    return cudaErrorInvalidValue;
  if (kind == kKindBf16) return dispatch_bn<kKindBf16>(bn, wmap, xmap, bmap, p, lp, split, stream);
  if (kind == kKindFp8) return dispatch_bn<kKindFp8>(bn, wmap, xmap, bmap, p, lp, split, stream);
  return cudaErrorInvalidValue;
}

cudaError_t read_op_status(uint32_t* status) {
  cudaError_t err = cudaMemcpyFromSymbol(status, g_op_status, sizeof(uint32_t));
  if (err == cudaSuccess && *status) {
    const uint32_t zero = 0;
    err = cudaMemcpyToSymbol(g_op_status, &zero, sizeof(zero));
  }
  return err;
}

}  // namespace laya
