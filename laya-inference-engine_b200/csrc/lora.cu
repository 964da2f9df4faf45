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
#include "lora.cuh"

#include <algorithm>
#include <mutex>

namespace laya {

// Status of launches that were given no status word (laya_b200_op_status).
__device__ uint32_t g_op_status;

}  // namespace laya

#include "lora_pair.cuh"

namespace laya {

namespace {

// ------------------------------------------------------------------ shrink
// V = s x A^T on tcgen05: a CTA takes 128 rows (the TMEM lanes), a share of the
// adapters that they use, up to 64 ranks and a slice of K.  The A_a of up to
// kShrinkCols / ranks adapters are stacked as one B operand, so the rows are
// read once for all of them; every row meets every adapter of the pass and
// keeps the columns of its own, so that no row sees another adapter's values.
// The K slices of a cluster are added through distributed shared memory in
// rank order.  Bound by the loads (rows and adapters once each) and, for few
// rows, by the latency of two dependent loads and the exchange.  (On mma.sync,
// small enough to share its SM with the projection, it took 15 us for 8,192
// rows and 41 K blocks: too few bytes in flight.)
constexpr int kShrinkRows = 128;
constexpr int kShrinkRanks = 64;   // ranks of an adapter in one CTA
constexpr int kShrinkCols = 256;   // columns of one pass
constexpr int kShrinkStages = 4;
constexpr int kShrinkPitch = kShrinkRanks + 4;
constexpr int kShrinkXBytes = kShrinkRows * 128, kShrinkABytes = kShrinkCols * 128;
constexpr int kShrinkPipe = kShrinkStages * (kShrinkXBytes + kShrinkABytes);
static_assert(kShrinkRows * kShrinkPitch * 4 <= kShrinkPipe, "the parts lie over the stages");
constexpr int kListInts = 1536;  // write_list's memory
constexpr int kShrinkSmem = kShrinkPipe + (2 * 128 + 264 + kListInts) * 4 + 128 + 1024;

// The four warps that compute.
DEVI void sync128() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Numbers the distinct non-negative values of own[] (row h * 128 + thread, 128
// threads) in order of first appearance: ord[] of each row (-1: none), the
// values in s_list, their count returned (tid: 0..127).  A warp's leaders look for their
// value among the earlier warps' leaders only, so a tile of long runs costs a
// few steps.  s_tmp, s_entry: H * 128 ints (16-byte aligned); s_cnt: H * 4.
template <int H>
DEVI int number_adapters(int tid, const int (&own)[H], int (&ord)[H], int* s_list, int* s_tmp, int* s_entry,
                         int* s_cnt) {
  const int lane = tid & 31, warp = tid >> 5;
  const unsigned below = (1u << lane) - 1;
  int lead[H], entry[H], seen[H];
  unsigned firsts[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    lead[h] = __ffs(__match_any_sync(0xffffffffu, own[h])) - 1;
    const unsigned leaders = __ballot_sync(0xffffffffu, own[h] >= 0 && lead[h] == lane);
    s_tmp[h * 128 + tid] = -1;
    __syncwarp();
    entry[h] = own[h] >= 0 && lead[h] == lane ? h * 128 + warp * 32 + __popc(leaders & below) : -1;
    if (entry[h] >= 0) s_tmp[entry[h]] = own[h];
  }
  sync128();
#pragma unroll
  for (int h = 0; h < H; ++h) {
    seen[h] = H * 128;
    if (entry[h] >= 0)
      for (int j = 0; j < h * 128 + warp * 32; j += 4) {
        const int4 v = *reinterpret_cast<const int4*>(s_tmp + j);
        if (v.w == own[h]) seen[h] = min(seen[h], j + 3);
        if (v.z == own[h]) seen[h] = min(seen[h], j + 2);
        if (v.y == own[h]) seen[h] = min(seen[h], j + 1);
        if (v.x == own[h]) seen[h] = min(seen[h], j);
      }
    firsts[h] = __ballot_sync(0xffffffffu, entry[h] >= 0 && seen[h] == H * 128);
    if (lane == 0) s_cnt[h * 4 + warp] = __popc(firsts[h]);
  }
  sync128();
  int n = 0;
#pragma unroll
  for (int w = 0; w < 4 * H; ++w) {
    const int h = w / 4;
    if (w % 4 == warp && entry[h] >= 0 && seen[h] == H * 128) {
      ord[h] = n + __popc(firsts[h] & below);
      s_entry[entry[h]] = ord[h];
      s_list[ord[h]] = own[h];
    }
    n += s_cnt[w];
  }
  sync128();
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if (entry[h] >= 0 && seen[h] < H * 128) ord[h] = s_entry[seen[h]];
    const int of_lead = __shfl_sync(0xffffffffu, ord[h], lead[h]);
    ord[h] = own[h] >= 0 ? of_lead : -1;
  }
  return n;
}

// Writes the list of the 256 rows from row0 for the projection: count, adapters,
// and each one's first and last row.  128 threads; `w`: 1536 ints of shared memory.
DEVI void write_list(const LoraParams& p, int row0, int* w) {
  const int tid = threadIdx.x, lane = tid & 31;
  int own[2], ord[2] = {-1, -1};
  for (int h = 0; h < 2; ++h) own[h] = row_adapter(p, row0 + 128 * h + tid);
  int *s_list = w, *s_span = w + 256;
  const int n = number_adapters<2>(tid, own, ord, s_list, w + 768, w + 1024, w + 1280);
  for (int j = tid; j < n; j += 128) {
    s_span[j] = 256;
    s_span[256 + j] = -1;
  }
  sync128();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // one lane of a warp's run speaks for it
    const unsigned same = __match_any_sync(0xffffffffu, ord[h]);
    if (ord[h] >= 0 && __ffs(same) - 1 == lane) {
      atomicMin(&s_span[ord[h]], h * 128 + tid);
      atomicMax(&s_span[256 + ord[h]], h * 128 + tid - lane + 31 - __clz(same));
    }
  }
  sync128();
  int* out = p.lists + (size_t)(row0 / 256) * kLoraListInts;
  for (int j = tid; j < n; j += 128) {
    out[kLoraListSlots + j] = s_list[j];
    out[kLoraListSpans + j] = s_span[j] | s_span[256 + j] << 16;
  }
  if (tid == 0) out[0] = n;
}

// The K slices' parts of the kept columns of this CTA's rows [t0, t1), which
// every CTA of the cluster sent to recv[slice][row - t0][kShrinkPitch], added
// in slice order, scaled, as V's hi + lo pairs: sixteen lanes take a row (four
// ranks each), a thread four rows at a time.  slot_of(row): the row's adapter,
// or -1 where another pass or CTA holds it; r0: first rank of the columns.
template <class SlotOf>
DEVI void write_v(const LoraParams& p, const float* recv, int row0, int t0, int t1, int cols, int r0, int split,
                  SlotOf slot_of) {
  const int c = (threadIdx.x & 15) * 4, r = r0 + c;
  if (c >= cols || (r >> 5) >= p.chunks) return;
  const int per_slice = (t1 - t0) * kShrinkPitch;
#pragma unroll 4
  for (int row = t0 + (int)(threadIdx.x >> 4); row < t1; row += 8) {
    const int slot = slot_of(row);
    if (slot < 0) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < split; ++k) {
      const float4 q = *reinterpret_cast<const float4*>(recv + k * per_slice + (row - t0) * kShrinkPitch + c);
      v.x += q.x;
      v.y += q.y;
      v.z += q.z;
      v.w += q.w;
    }
    const float f = p.scaling ? p.scaling[slot] : 1.f;
    const float x[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    float lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)  // an infinite (or NaN) value has no remainder
      lo[k] = fabsf(x[k]) < INFINITY ? x[k] - bf16_round(x[k]) : 0.f;
    __nv_bfloat16* dst = p.v + ((size_t)(row0 + row) * p.chunks + (r >> 5)) * 64 + (r & 31);
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    *reinterpret_cast<uint2*>(dst + 32) = make_uint2(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]));
  }
}

__global__ void __launch_bounds__(192)
    lora_shrink_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap amap,
                       const LoraParams p) {
  constexpr int ST = kShrinkStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sA = smem + ST * kShrinkXBytes;
  float* recv = reinterpret_cast<float*>(smem);               // [slice][its rows][kShrinkPitch], between passes
  int* s_ord = reinterpret_cast<int*>(smem + kShrinkPipe);   // [128] each row's place in the list
  int* s_list = s_ord + 128;                                  // [128] distinct adapters
  int* s_tmp = s_list + 128;                                  // [128] + [128] + [4]: number_adapters
  uint64_t* full = reinterpret_cast<uint64_t*>(s_tmp + 264 + kListInts);
  uint64_t* empty = full + ST;
  uint64_t* done = empty + ST;
  uint64_t* sent = done + 1;  // the parts of this CTA's rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sent + 1);
  int* s_count = reinterpret_cast<int*>(tmem_slot + 1);
  int* failed = s_count + 1;
  // Everything before this kernel is complete once the wait returns; the
  // projection launched behind it relies on that (its K blocks do not wait).
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int groups = (p.rank + kShrinkRanks - 1) / kShrinkRanks, slices = gridDim.y / groups;
  const int group = blockIdx.y % groups, slice = blockIdx.y / groups;
  const int row0 = blockIdx.x * kShrinkRows, split = gridDim.z, rank = blockIdx.z;
  const int cols = lora_shrink_box(p.rank);  // of one adapter
  const int kblocks = (p.in_features + 63) / 64;
  const int kb0 = rank * kblocks / split, nkb = (rank + 1) * kblocks / split - kb0;
  const uint64_t limit = kWaitLimitNs;
  const uint64_t pol = policy_evict_last();
  auto load_rows = [&](int s, int k) {
    mbar_expect_tx(&full[s], kShrinkXBytes);
    tma_load_2d(sX + s * kShrinkXBytes, &xmap, &full[s], (kb0 + k) * 64, row0, pol);
  };
  if (warp == 4) {
    if (elect_one()) {
      for (int s = 0; s < ST; ++s) {
        mbar_init(&full[s], 2);  // the rows, the adapters
        mbar_init(&empty[s], 1);
      }
      mbar_init(done, 1);
      mbar_init(sent, 1);
      *failed = 0;
      fence_mbar_init();
      for (int k = 0; k < ST && k < nkb; ++k) load_rows(k, k);
    }
    __syncwarp();
  } else if (warp == 5) {
    tmem_alloc(tmem_slot, kShrinkCols);
    tmem_relinquish();
  } else {
    // ---- the tile's adapters in order of first use (the rows are on their way)
    const int own[1] = {row_adapter(p, row0 + tid)};
    int ord[1] = {-1};
    const int n = number_adapters<1>(tid, own, ord, s_list, s_tmp, s_tmp + 128, s_tmp + 256);
    s_ord[tid] = ord[0];
    if (tid == 0) *s_count = n;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();  // after the allocation: the projection allocates too
  const uint32_t tmem = *tmem_slot;
  const int n = *s_count;
  const int u0 = (int)((long long)slice * n / slices), u1 = (int)((long long)(slice + 1) * n / slices);
  const int per = kShrinkCols / cols;  // adapters of one pass
  if (warp == 4 && u0 == u1)           // no adapter here: the rows still land before the exit
    for (int k = 0; k < ST && k < nkb; ++k) {
      if (elect_one()) mbar_arrive(&full[k]);
      __syncwarp();
      if (!warp_wait(&full[k], 0, limit) && lane == 0) atomicExch(failed, 1);
    }
  // the projection's list of 256 rows, while the first K blocks are on their way
  if (warp < 4 && row0 % 256 == 0 && blockIdx.y == 0 && rank == split - 1) write_list(p, row0, s_tmp + 264);
  Ring<ST> ring;
  uint32_t g = 0, pass = 0;  // K blocks and passes before this one
  for (int u = u0; u < u1; u += per, ++pass) {
    // (after a failure the passes still meet at their barriers)
    const int units = u1 - u < per ? u1 - u : per;
    const int todo = *reinterpret_cast<volatile int*>(failed) ? 0 : nkb;
    if (warp == 4) {
      for (int k = 0; k < todo; ++k, ++g, ring.next()) {
        const int s = ring.s;
        if (g >= ST && !warp_wait(&empty[s], ring.phase ^ 1, limit)) {
          if (lane == 0) atomicExch(failed, 1);
          break;
        }
        if (elect_one()) {
          if (g >= ST || (int)g >= nkb) load_rows(s, k);  // (the first ones were requested above)
          mbar_expect_tx(&full[s], units * cols * 128);
          for (int a = 0; a < units; ++a)
            tma_load_3d(sA + s * kShrinkABytes + a * cols * 128, &amap, &full[s], (kb0 + k) * 64, group * kShrinkRanks,
                        s_list[u + a], pol);
        }
        __syncwarp();
      }
    } else if (warp == 5) {
      const uint32_t idesc = idesc_bf16(128, units * cols);
      const uint32_t x0 = desc_lo(smem_u32(sX)), a0 = desc_lo(smem_u32(sA));
      for (int k = 0; k < todo; ++k, ring.next()) {
        const int s = ring.s;
        if (!warp_wait(&full[s], ring.phase, limit)) {
          if (lane == 0) atomicExch(failed, 1);
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t xd = x0 + s * (kShrinkXBytes >> 4), ad = a0 + s * (kShrinkABytes >> 4);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            umma1_f16<kDesc128, kDesc128>(tmem, xd + 2 * e, ad + 2 * e, idesc, (k | e) != 0);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (elect_one()) umma_commit(done);
      __syncwarp();
    } else {
      if (!warp_wait(done, pass & 1, limit) && lane == 0) atomicExch(failed, 1);
      tc_fence_after();
    }
    // Every CTA's stages are free: the parts go over them, each row's kept
    // columns to the CTA that owns the row.
    const int own_rows = kShrinkRows / split, t0 = rank * own_rows;
    const int o = warp < 4 ? s_ord[tid] : -1;
    const bool mine = o >= u && o < u + units;
    const int owned = __syncthreads_count(mine && tid >= t0 && tid < t0 + own_rows);
    if (split > 1) {
      cluster_sync_relaxed();
      if (tid == 0) mbar_expect_tx(sent, owned * (split - 1) * cols * 4);
    }
    if (warp < 4) {
      const uint32_t to = tid / own_rows;
      float* here = recv + (rank * own_rows + tid % own_rows) * kShrinkPitch;  // (a row of its own)
      const uint32_t dst = mapa_shared(smem_u32(here), to);
      const uint32_t bar = mapa_shared(smem_u32(sent), to);
      for (int a = 0; a < units; ++a) {
        if (!__any_sync(0xffffffffu, o == u + a)) continue;
        const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + a * cols;
        for (int c = 0; c < cols; c += 32) {
          uint32_t r[32];
          if (cols - c >= 32) {
            tmem_ld32(acc + c, r);
          } else {
            uint32_t h[16];
            tmem_ld16(acc + c, h);
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = h[e];
          }
          tmem_wait_ld();
          if (o == u + a)
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c + e < cols) {
                const float4 v = make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]),
                                             __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
                if (to == (uint32_t)rank)
                  *reinterpret_cast<float4*>(here + c + e) = v;
                else
                  st_async_f32x4(dst + (c + e) * 4, v.x, v.y, v.z, v.w, bar);
              }
        }
      }
      tc_fence_before();
      if (split > 1 && !warp_wait_cluster(sent, pass & 1, limit) && lane == 0) atomicExch(failed, 1);
      sync128();
      write_v(p, recv, row0, t0, t0 + own_rows, cols, group * kShrinkRanks, split, [&](int row) {
        const int ord = s_ord[row];
        return ord >= u && ord < u + units ? s_list[ord] : -1;
      });
    }
    // the parts are read; the next pass's copies may take their place
    fence_proxy_async_smem();
    __syncthreads();
    tc_fence_after();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, kShrinkCols);
  if (tid == 0 && *reinterpret_cast<volatile int*>(failed))
    record_status(p.status ? p.status : &g_op_status, kStatusGemmFullTimeout);
}

// ---------------------------------------------------------- shrink, few rows
// The same for up to 64 rows, which may each bring an adapter of their own:
// CTAs of 64 rows on mma.sync, whose operands TMA stages, without tensor memory
// and in little shared memory, so that many share an SM and the projection's
// CTAs start beside them (64 rows with 64 adapters of rank 16 into 5,248
// features: 18.6 us with this one in front, 24.3 with the one above).
constexpr int kFewRows = 64;

// WIDE: one adapter of more than 32 ranks at a time; else adapters that
// together have up to 32 columns, and a stage more in the same memory.
template <bool WIDE>
struct FewShrinkCfg {
  static constexpr int COLS = WIDE ? 64 : 32;
  static constexpr int STAGES = WIDE ? 3 : 4;
  static constexpr int X_BYTES = kFewRows * 128, A_BYTES = COLS * 128;
  static constexpr int PIPE_BYTES = STAGES * (X_BYTES + A_BYTES);
  static constexpr int RECV_BYTES = kFewRows * kShrinkPitch * 4;  // over the stages, between passes
  static_assert(RECV_BYTES <= PIPE_BYTES, "the parts fit the pipeline's memory");
  static constexpr int SMEM = PIPE_BYTES + (2 * 128 + 264) * 4 + 128 + 1024;
};

DEVI void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DEVI void ldmatrix4(uint32_t (&r)[4], uint32_t saddr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(saddr)
               : "memory");
}

template <bool WIDE>
__global__ void __launch_bounds__(160)
    lora_shrink_few_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap amap,
                       const LoraParams p) {
  using C = FewShrinkCfg<WIDE>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sA = smem + ST * C::X_BYTES;
  float* recv = reinterpret_cast<float*>(smem);                 // [slice][its rows][kShrinkPitch], between passes
  int* s_ord = reinterpret_cast<int*>(smem + C::PIPE_BYTES);   // [128] each row's place in the list
  int* s_list = s_ord + 128;                                    // [128] distinct adapters
  int* s_tmp = s_list + 128;                                    // [128] + [128] + [4]: number_adapters
  uint64_t* full = reinterpret_cast<uint64_t*>(s_tmp + 264);
  uint64_t* empty = full + ST;
  uint64_t* sent = empty + ST;  // the parts of this CTA's rows
  int* s_count = reinterpret_cast<int*>(sent + 1);
  int* failed = s_count + 1;
  // Everything before this kernel is complete once the wait returns; the
  // projection launched behind it relies on that (its K blocks do not wait).
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool loader = warp == 4;
  const int groups = (p.rank + kShrinkRanks - 1) / kShrinkRanks, slices = gridDim.y / groups;
  const int group = blockIdx.y % groups, slice = blockIdx.y / groups;
  const int split = gridDim.z, rank = blockIdx.z;
  const int cols = lora_shrink_box(p.rank);  // of one adapter
  const int kblocks = (p.in_features + 63) / 64;
  const int kb0 = rank * kblocks / split, nkb = (rank + 1) * kblocks / split - kb0;
  const uint64_t limit = kWaitLimitNs;
  const uint64_t pol = policy_evict_last();
  auto load_rows = [&](int s, int k) {
    mbar_expect_tx(&full[s], C::X_BYTES);
    tma_load_2d(sX + s * C::X_BYTES, &xmap, &full[s], (kb0 + k) * 64, 0, pol);
  };
  if (loader) {
    if (elect_one()) {
      for (int s = 0; s < ST; ++s) {
        mbar_init(&full[s], 2);   // the rows, the adapters
        mbar_init(&empty[s], 4);  // the warps that compute
      }
      mbar_init(sent, 1);
      *failed = 0;
      fence_mbar_init();
      for (int k = 0; k < ST && k < nkb; ++k) load_rows(k, k);
    }
    __syncwarp();
  } else {
    // ---- the tile's adapters in order of first use (the rows are on their way)
    const int own[1] = {tid < kFewRows ? row_adapter(p, tid) : -1};
    int ord[1] = {-1};
    const int n = number_adapters<1>(tid, own, ord, s_list, s_tmp, s_tmp + 128, s_tmp + 256);
    s_ord[tid] = ord[0];
    if (tid == 0) *s_count = n;
  }
  __syncthreads();
  const int n = *s_count;
  const int u0 = (int)((long long)slice * n / slices), u1 = (int)((long long)(slice + 1) * n / slices);
  const int per = C::COLS / cols;  // adapters of one pass
  if (loader && u0 == u1)          // no adapter here: the rows still land before the exit
    for (int k = 0; k < ST && k < nkb; ++k) {
      if (elect_one()) mbar_arrive(&full[k]);
      __syncwarp();
      if (!warp_wait(&full[k], 0, limit) && lane == 0) atomicExch(failed, 1);
    }
  Ring<ST> ring;
  uint32_t g = 0, pass = 0;  // K blocks and passes before this one
  for (int u = u0; u < u1; u += per, ++pass) {
    // (after a failure the passes still meet at their barriers)
    const int units = u1 - u < per ? u1 - u : per, ncols = units * cols;
    const int todo = *reinterpret_cast<volatile int*>(failed) ? 0 : nkb;
    if (loader) {
      for (int k = 0; k < todo; ++k, ++g, ring.next()) {
        const int s = ring.s;
        if (g >= ST && !warp_wait(&empty[s], ring.phase ^ 1, limit)) {
          if (lane == 0) atomicExch(failed, 1);
          break;
        }
        if (elect_one()) {
          if (g >= ST || (int)g >= nkb) load_rows(s, k);  // (the first ones were requested above)
          mbar_expect_tx(&full[s], ncols * 128);
          for (int a = 0; a < units; ++a)
            tma_load_3d(sA + s * C::A_BYTES + a * cols * 128, &amap, &full[s], (kb0 + k) * 64, group * kShrinkRanks,
                        s_list[u + a], pol);
        }
        __syncwarp();
      }
    }
    float acc[C::COLS / 8][4];
    if (!loader) {
#pragma unroll
      for (int j = 0; j < C::COLS / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      for (int k = 0; k < todo; ++k, ring.next()) {
        const int s = ring.s;
        if (!warp_wait(&full[s], ring.phase, limit)) {
          if (lane == 0) atomicExch(failed, 1);
          break;
        }
        const uint32_t xs = smem_u32(sX + s * C::X_BYTES), as = smem_u32(sA + s * C::A_BYTES);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4];
          ldmatrix4(a, xs + sw128_offset(warp * 16 + (lane & 15), 2 * j + (lane >> 4)));
#pragma unroll
          for (int q = 0; q < C::COLS / 16; ++q)
            if (16 * q < ncols) {
              uint32_t b[4];
              ldmatrix4(b, as + sw128_offset(16 * q + (lane & 7) + ((lane >> 4) << 3), 2 * j + ((lane >> 3) & 1)));
              mma_bf16(acc[2 * q], a, b[0], b[1]);
              mma_bf16(acc[2 * q + 1], a, b[2], b[3]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
    }
    // Every CTA's stages have been read: the parts go over them, each row's kept
    // columns to the CTA that owns the row.
    const int own_rows = kFewRows / split, t0 = rank * own_rows;
    const int o = !loader && tid < kFewRows ? s_ord[tid] : -1;
    const int owned = __syncthreads_count(o >= u && o < u + units && tid >= t0 && tid < t0 + own_rows);
    if (split > 1) {
      cluster_sync_relaxed();
      if (tid == 0) mbar_expect_tx(sent, owned * (split - 1) * cols * 4);
    }
    if (!loader) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = warp * 16 + (lane >> 2) + 8 * h, unit = s_ord[row] - u;
        if (unit < 0 || unit >= units) continue;
        const uint32_t to = row / own_rows;
        float* here = recv + (rank * own_rows + row % own_rows) * kShrinkPitch;  // (a row of its own)
        const uint32_t dst = mapa_shared(smem_u32(here), to);
        const uint32_t bar = mapa_shared(smem_u32(sent), to);
#pragma unroll
        for (int j = 0; j < C::COLS / 8; ++j) {
          const int c = 8 * j + (lane & 3) * 2 - unit * cols;
          if (c < 0 || c >= cols) continue;
          if (to == (uint32_t)rank)
            *reinterpret_cast<float2*>(here + c) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
          else
            st_async_f32x2(dst + c * 4, acc[j][2 * h], acc[j][2 * h + 1], bar);
        }
      }
      __syncwarp();
      if (split > 1 && !warp_wait_cluster(sent, pass & 1, limit) && lane == 0) atomicExch(failed, 1);
      sync128();
      write_v(p, recv, 0, t0, t0 + own_rows, cols, group * kShrinkRanks, split, [&](int row) {
        const int ord = s_ord[row];
        return ord >= u && ord < u + units ? s_list[ord] : -1;
      });
    }
    // the parts are read; the next pass's copies may take their place
    fence_proxy_async_smem();
    __syncthreads();
  }
  if (tid == 0 && *reinterpret_cast<volatile int*>(failed))
    record_status(p.status ? p.status : &g_op_status, kStatusGemmFullTimeout);
}

// ------------------------------------------------- projection for few rows
// Up to 64 rows, bound by reading W and the adapters: the tile layout and
// split-K of gemm.cu (weight rows on the TMEM lanes, rows of X as the MMA's N).
// An adapter's blocks multiply only the 16-row groups between its first and
// last row, so 64 single rows with 64 adapters cost as many narrow MMAs; four
// builder warps prepare the V tiles, each its own blocks, loading the next
// one's values before they wait for its stage.
constexpr int kFewBuilders = 4;  // warps, two for each of two stages in turn; half of them divides STAGES, so that
                                 // each sees every use of its stages

template <int BN, int KIND>
struct LoraCfg {
  static constexpr int STAGES = 4;
  static constexpr int THREADS = 64 + 32 * kFewBuilders;
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
  static constexpr int PART_BYTES = 2 * BN * 128 * 4;  // the partial tile, and its tokens' from the other slices
  static constexpr int MAIN_BYTES = PIPE_BYTES > PART_BYTES ? PIPE_BYTES : PART_BYTES;
  static constexpr int LIST_BYTES = (128 + 2 * BN + 264) * 4;  // adapters, their rows, numbering, activation scales
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

template <int BN, int KIND>
__global__ void __launch_bounds__(LoraCfg<BN, KIND>::THREADS, 2)
    lora_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                     const __grid_constant__ CUtensorMap bmap, const GemmParams p, const LoraParams lp) {
  using C = LoraCfg<BN, KIND>;
  constexpr int STAGES = C::STAGES;
  static_assert(STAGES % (kFewBuilders / 2) == 0 && kFewBuilders == 4, "builder warps and stages");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::MAIN_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* vfull = empty + STAGES;
  uint64_t* vfree = vfull + STAGES;  // the producer found the stage free for an adapter block
  uint64_t* done = vfree + STAGES;
  uint64_t* listed = done + 1;  // the tile's adapter list is in shared memory
  uint64_t* sent = listed + 1;  // the cluster's parts of this CTA's tokens
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sent + 1);
  uint32_t* failed = tmem_slot + 1;
  int* s_count = reinterpret_cast<int*>(failed + 1);  // distinct adapters, widest span of rows
  static_assert((4 * STAGES + 3) * 8 + 16 <= C::BAR_BYTES, "barrier block");
  int* s_list = reinterpret_cast<int*>(smem + C::MAIN_BYTES + C::BAR_BYTES);  // [128] distinct adapters
  int* s_span = s_list + 128;                                                 // [BN] first | last << 16 of their rows
  int* s_tmp = s_span + BN;                                                   // [264] number_adapters
  float* s_scale = reinterpret_cast<float*>(s_tmp + 264);                     // [BN] activation scales (fp8)

  const int tid = threadIdx.x, warp = tid >> 5;
  const int tile_n = blockIdx.x;
  const int split = gridDim.z, rank = blockIdx.z;
  const int kb0 = (int)((long long)rank * p.kblocks / split);
  const int kb1 = (int)((long long)(rank + 1) * p.kblocks / split);
  const int nkb = kb1 - kb0;
  uint32_t* status = p.status ? p.status : &g_op_status;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&vfull[s], 2);  // the stage's two halves
      mbar_init(&vfree[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(listed, 1);
    mbar_init(sent, 1);
    *failed = 0;
    fence_mbar_init();
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&xmap);
    prefetch_tensormap(&bmap);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();  // only now: the next kernel may allocate tensor memory too
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem2 = tmem + (C::ACCS - 1) * BN;  // the adapters' accumulator

  const uint64_t limit = wait_limit(p.wait_limit_us);
  int issued = 0;  // producer warp: loads issued (for the drain on failure)
  // This rank's share of the tile's adapter blocks (adapter, chunk of 32
  // ranks), known once `listed` has completed: [b0, b1), `pack` of them in a
  // stage.  A stage has room for two blocks of half the rows each, which single
  // rows' adapters are; two at a time keep twice the loads in flight.
  struct Share {
    int b0, b1, pack;
    DEVI int stages() const { return (b1 - b0 + pack - 1) / pack; }
  };
  auto share = [&] {
    const int n = s_count[0] * lp.chunks;
    return Share{(int)((long long)rank * n / split), (int)((long long)(rank + 1) * n / split),
                 s_count[1] <= BN / 2 && KIND == kKindBf16 ? 2 : 1};
  };
  // Rows [c0, c1) that block b multiplies: whole groups of 16.  The first block
  // of the FP8 kernels takes every row, which starts their second accumulator.
  auto span = [&](int b, int b0, int& c0, int& c1) {
    const int sp = s_span[b / lp.chunks];
    const bool all = KIND == kKindFp8 && b == b0;
    c0 = all ? 0 : (sp & 0xffff) & ~15;
    c1 = all ? BN : ((sp >> 16) + 16) & ~15;
  };
  auto give_up = [&](uint32_t code) {
    record_status(status, code);
    atomicExch(failed, 1u);
  };
  if (warp == 0) {
    // W, X and B_a do not wait for the shrink: whatever wrote them was
    // complete before it released this kernel.
    const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
    Ring<STAGES> ring;
    bool ok = true;
    for (int i = 0; i < nkb; ++i, ring.next()) {
      const int s = ring.s;
      if (i >= STAGES && !(ok = warp_wait(&empty[s], ring.phase ^ 1, limit))) break;
      if (elect_one()) {
        mbar_expect_tx(&full[s], C::STAGE_BYTES);
        tma_load_2d(sA + s * C::A_BYTES, &wmap, &full[s], (kb0 + i) * C::K_ELEMS, tile_n * 128, pol_w);
        tma_load_2d(sB + s * C::B_BYTES, &xmap, &full[s], (kb0 + i) * C::K_ELEMS, 0, pol_x);
      }
      __syncwarp();
      issued = i + 1;
    }
    ok = ok && warp_wait(listed, 0, limit);
    if (ok) {
      const Share sh = share();
      for (int q = 0; q < sh.stages(); ++q, ring.next()) {
        const int i = nkb + q, s = ring.s, b = sh.b0 + q * sh.pack, two = sh.pack == 2 && b + 1 < sh.b1;
        if (i >= STAGES && !(ok = warp_wait(&empty[s], ring.phase ^ 1, limit))) break;
        if (elect_one()) {
          mbar_arrive(&vfree[s]);
          mbar_expect_tx(&full[s], two ? 2 * 128 * 64 : 128 * 64);
          for (int h = 0; h <= two; ++h)
            tma_load_3d(sA + s * C::A_BYTES + h * 128 * 64, &bmap, &full[s], ((b + h) % lp.chunks) * 32, tile_n * 128,
                        s_list[(b + h) / lp.chunks], pol_w);
        }
        __syncwarp();
        issued = i + 1;
      }
      // every stage's last release, so that none is in flight at the exit
      for (int i = issued < STAGES ? 0 : issued - STAGES; ok && i < issued; ++i)
        ok = warp_wait(&empty[i % STAGES], (i / STAGES) & 1, limit);
    }
    if (!ok && (tid & 31) == 0) give_up(kStatusGemmEmptyTimeout);
  } else if (warp == 1) {
    const uint32_t idesc = KIND == kKindBf16 ? idesc_bf16(128, BN) : idesc_e4m3(128, BN);
    const uint32_t a0 = desc_lo(smem_u32(sA)), d0 = desc_lo(smem_u32(sB));
    Ring<STAGES> ring;
    bool ok = true;
    for (int i = 0; i < nkb; ++i, ring.next()) {
      const int s = ring.s;
      if (!(ok = warp_wait(&full[s], ring.phase, limit))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t ad = a0 + s * (C::A_BYTES >> 4), bd = d0 + s * (C::B_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (KIND == kKindBf16)
            umma1_f16<kDesc128, kDesc128>(tmem, ad + 2 * k, bd + 2 * k, idesc, (i | k) != 0);
          else
            umma1_f8(tmem, ad + 2 * k, bd + 2 * k, idesc, (i | k) != 0);
        }
        umma_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (ok && (ok = warp_wait(listed, 0, limit))) {
      const Share sh = share();
      for (int q = 0; q < sh.stages(); ++q, ring.next()) {
        const int s = ring.s, b = sh.b0 + q * sh.pack, two = sh.pack == 2 && b + 1 < sh.b1;
        if (!(ok = warp_wait(&full[s], ring.phase, limit)) || !(ok = warp_wait(&vfull[s], (q / STAGES) & 1, limit)))
          break;
        tc_fence_after();
        if (elect_one()) {
          for (int h = 0; h <= two; ++h) {
            int c0, c1;
            span(b + h, sh.b0, c0, c1);
            const uint32_t ad = a0 + s * (C::A_BYTES >> 4) + h * (128 * 64 >> 4);
            const uint32_t bd = d0 + s * (C::B_BYTES >> 4) + h * (C::B_BYTES / 2 >> 4);
            const uint32_t id2 = idesc_bf16(128, c1 - c0), acc = tmem2 + c0;
            umma1_f16<kDesc64, kDesc128>(acc, ad, bd, id2, KIND == kKindBf16 || b > sh.b0);  // hi
            umma1_f16<kDesc64, kDesc128>(acc, ad, bd + 4, id2, 1);                           // lo
            if (lp.rank - ((b + h) % lp.chunks) * 32 > 16) {
              umma1_f16<kDesc64, kDesc128>(acc, ad + 2, bd + 2, id2, 1);
              umma1_f16<kDesc64, kDesc128>(acc, ad + 2, bd + 6, id2, 1);
            }
          }
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
    }
    if (!ok && (tid & 31) == 0) give_up(kStatusGemmFullTimeout);
    if (elect_one()) umma_commit(done);
    __syncwarp();
  } else if (warp >= 2) {
    // ---- the tile's adapters in order of first use and the rows each spans
    // (which do not wait for the shrink), then the V tiles: rows of other
    // adapters are zero
    const int bt = tid - 64, lane = tid & 31, bw = bt >> 5;
    const int own[1] = {bt < BN ? row_adapter(lp, bt) : -1};
    int ord[1] = {-1};
    const int n = number_adapters<1>(bt, own, ord, s_list, s_tmp, s_tmp + 128, s_tmp + 256);
    int *s_first = s_tmp, *s_last = s_tmp + 128;
    sync128();
    if (bt < n) {
      s_first[bt] = BN;
      s_last[bt] = -1;
    }
    if (bt == 0) {
      s_count[0] = n;
      s_count[1] = 0;
    }
    sync128();
    const unsigned same = __match_any_sync(0xffffffffu, ord[0]);
    if (ord[0] >= 0 && __ffs(same) - 1 == lane) {  // one lane of a warp's run speaks for it
      atomicMin(&s_first[ord[0]], bt);
      atomicMax(&s_last[ord[0]], bt - lane + 31 - __clz(same));
    }
    sync128();
    if (bt < n) {
      s_span[bt] = s_first[bt] | s_last[bt] << 16;
      atomicMax(&s_count[1], ((s_last[bt] + 16) & ~15) - (s_first[bt] & ~15));
    }
    sync128();
    if (bt == 0) mbar_arrive(listed);
    const Share sh = share();
    const int half = bw & 1, j = lane & 7;  // half of a stage; 16-byte chunk of a V row
    const int own0 = row_adapter(lp, lane), own1 = BN > 32 ? row_adapter(lp, lane + 32) : -1;
    griddep_wait();  // V
    // a warp takes its half of every second stage and loads the next block's
    // values before it waits for the stage
    for (int q = bw >> 1; q < sh.stages(); q += kFewBuilders / 2) {
      const int s = (nkb + q) % STAGES, b = sh.b0 + q * sh.pack + half;
      const bool has = half < sh.pack && b < sh.b1;
      uint4 v[BN / 4];
      int c0 = 0, c1 = 0;
      if (has) {
        const int c = b % lp.chunks, slot = s_list[b / lp.chunks];
        const int ksteps = lp.rank - c * 32 > 16 ? 2 : 1;
        span(b, sh.b0, c0, c1);
#pragma unroll
        for (int u = 0; u < BN / 4; ++u) {
          const int row = c0 + u * 4 + (lane >> 3);
          const int o0 = __shfl_sync(0xffffffffu, own0, row & 31), o1 = __shfl_sync(0xffffffffu, own1, row & 31);
          v[u] = make_uint4(0, 0, 0, 0);
          if (row < c1 && (row < 32 ? o0 : o1) == slot && (j & 3) < 2 * ksteps)
            v[u] = *reinterpret_cast<const uint4*>(lp.v + ((size_t)row * lp.chunks + c) * 64 + j * 8);
        }
      }
      // (the builders cannot wait on `empty` themselves: they have not followed
      // its phases through the K blocks, and a parity names every second one)
      if (!warp_wait(&vfree[s], (q / STAGES) & 1, limit)) {
        if (lane == 0) give_up(kStatusGemmEmptyTimeout);
        break;
      }
      if (has) {
        uint8_t* dst = sB + s * C::B_BYTES + half * (C::B_BYTES / 2);
#pragma unroll
        for (int u = 0; u < BN / 4; ++u) {
          const int row = u * 4 + (lane >> 3);
          if (c0 + row < c1) *reinterpret_cast<uint4*>(dst + sw128_offset(row, j)) = v[u];
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[s]);
    }
  }
  __syncwarp();

  // ---- epilogue: the partial tile [token][128] lies over the stages; each
  // other CTA of the cluster is sent the tokens it stores in one copy, to
  // recv[slice][token][128] behind the partial tile (its stages are free too
  // once the relaxed barrier is passed)
  griddep_wait();
  const int nt = BN / split, t0 = rank * nt;
  const int stored = max(0, min(p.M - t0, nt));  // its tokens that exist
  if (KIND == kKindFp8)
    for (int i = tid; i < BN; i += C::THREADS) s_scale[i] = i < p.M ? p.a_scale[i] : 0.f;
  if (!warp_wait(done, 0, limit) && (tid & 31) == 0) give_up(kStatusGemmDoneTimeout);
  tc_fence_after();
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  float* recv = part + BN * 128;
  if (warp < 4) {
    const Share sh = share();
    const bool second = KIND == kKindFp8 && sh.b1 > sh.b0;
    const int lr = tid;  // weight row of the tile
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    const float ws = KIND == kKindFp8 && tile_n * 128 + lr < p.N ? p.w_scale[tile_n * 128 + lr] : 1.f;
    constexpr int W = BN < 32 ? 16 : 32;
#pragma unroll 1
    for (int c = 0; c < BN && c < p.M; c += W) {
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
    tc_fence_before();
  }
  fence_proxy_async_smem();
  if (split > 1)
    cluster_sync_relaxed();  // (every thread of the CTA: its own partial tile is complete too)
  __syncthreads();
  if (split > 1) {
    if (warp == 0 && elect_one()) {
      mbar_expect_tx(sent, stored * (split - 1) * 512);
      for (int d = 1; d < split; ++d) {
        const int to = (rank + d) % split, tokens = min(p.M - to * nt, nt);
        if (tokens > 0)
          bulk_copy_to_peer(mapa_shared(smem_u32(recv + rank * nt * 128), to), part + to * nt * 128, tokens * 512,
                            mapa_shared(smem_u32(sent), to));
      }
    }
    __syncwarp();
    if (!warp_wait_cluster(sent, 0, limit) && (tid & 31) == 0) give_up(kStatusGemmDoneTimeout);
  }
  {
    const bool rope = tile_n * 128 < p.rope_cols;
    const int pair = rope ? 32 : 64;
    const bool residual = p.epilogue == kEpiResidual;
    const bool plain = p.epilogue == kEpiStore && !rope;
    const bool vec = p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
    for (int item = tid; item < stored * 16; item += C::THREADS) {
      const int q4 = rope ? ((item >> 3) & 1) * 64 + (item & 7) * 4 : (item & 15) * 4;
      const int m = t0 + (item >> 4), n = tile_n * 128 + q4;
      EpiPre pre;
      if (!plain) pre = epi_prefetch<kKindBf16>(p, m, n, residual, rope);
      float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (u < split) {
          const float* src = (u == rank ? part + t0 * 128 : recv + u * nt * 128) + (item >> 4) * 128 + q4;
          const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + pair);
          lo.x += a.x; lo.y += a.y; lo.z += a.z; lo.w += a.w;
          hi.x += b.x; hi.y += b.y; hi.z += b.z; hi.w += b.w;
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

  if (split > 1) cluster_sync_relaxed();  // every copy out of this CTA's memory has arrived

  // ---- teardown: drain copies still in flight after a failure, free TMEM
  if (tid == 0 && *failed) {
    for (int i = (issued > STAGES ? issued - STAGES : 0); i < issued; ++i)
      mbar_wait(&full[i % STAGES], (i / STAGES) & 1, limit);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, C::TMEM_COLS);
}

// ------------------------------------------------------------------ host side

template <int BN, int KIND>
cudaError_t launch_one(const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int split,
                       cudaStream_t stream) {
  using C = LoraCfg<BN, KIND>;
  auto kern = lora_gemm_kernel<BN, KIND>;
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
  cfg.gridDim = dim3((p.N + 127) / 128, 1, split);
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
  return cudaLaunchKernelEx(&cfg, kern, maps.w, maps.x, maps.b, p, lp);
}

template <int KIND>
cudaError_t dispatch_bn(int bn, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int split,
                        cudaStream_t st) {
  switch (bn) {
    case 16: return launch_one<16, KIND>(maps, p, lp, split, st);
    case 32: return launch_one<32, KIND>(maps, p, lp, split, st);
    case 64: return launch_one<64, KIND>(maps, p, lp, split, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

namespace {

cudaError_t launch_shrink(const void* kern, int smem, int threads, dim3 grid, const LoraMaps& maps, const LoraParams& p,
                          cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  cfg.attrs = attrs;
  if (pdl) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (grid.z > 1) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = 1;
    attrs[cfg.numAttrs].val.clusterDim.y = 1;
    attrs[cfg.numAttrs++].val.clusterDim.z = grid.z;
  }
  void* args[] = {const_cast<CUtensorMap*>(&maps.rows), const_cast<CUtensorMap*>(&maps.a), const_cast<LoraParams*>(&p)};
  return cudaLaunchKernelExC(&cfg, kern, args);
}

}  // namespace

cudaError_t launch_lora_shrink(const LoraMaps& maps, const LoraParams& p, int sm_count, int projection_ctas,
                               cudaStream_t stream, bool pdl) {
  if (p.rows < 1 || p.rank < 8 || p.rank % 8 || p.rank > kLoraMaxRank || p.in_features % 8 || p.slots < 1 ||
      p.index_div < 1 || !p.lists)
    return cudaErrorInvalidValue;
  constexpr int kWide = FewShrinkCfg<true>::SMEM, kSlim = FewShrinkCfg<false>::SMEM;
  static std::mutex mu;
  static uint64_t ready = 0;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!(ready >> dev & 1)) {
      const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
      err = cudaFuncSetAttribute(lora_shrink_kernel, attr, kShrinkSmem);
      if (err == cudaSuccess) err = cudaFuncSetAttribute(lora_shrink_few_kernel<true>, attr, kWide);
      if (err == cudaSuccess) err = cudaFuncSetAttribute(lora_shrink_few_kernel<false>, attr, kSlim);
      if (err != cudaSuccess) return err;
      ready |= uint64_t(1) << dev;
    }
  }
  const int groups = (p.rank + kShrinkRanks - 1) / kShrinkRanks, kblocks = (p.in_features + 63) / 64;
  if (lora_shrink_rows(p.rows) == kFewRows) {
    // The adapters are spread first, then K, up to three CTAs per SM.
    const bool wide = p.rank > 32;
    const int per = (wide ? 64 : 32) / lora_shrink_box(p.rank), room = std::max(1, 3 * sm_count / groups);
    const int slices = std::min(room, (std::min(p.slots, p.rows) + per - 1) / per);
    int split = 1;
    while (split < 8 && 2 * split <= kblocks && 2 * split * slices <= room) split *= 2;
    const dim3 grid(1, groups * slices, split);
    return wide ? launch_shrink((const void*)lora_shrink_few_kernel<true>, kWide, 160, grid, maps, p, stream, pdl)
                : launch_shrink((const void*)lora_shrink_few_kernel<false>, kSlim, 160, grid, maps, p, stream, pdl);
  }
  // One CTA per SM: K is split until they are in use (two K blocks at least
  // each), then the adapters, of which single rows of many requests bring many.
  const int tiles = (p.rows + kShrinkRows - 1) / kShrinkRows;
  // (the SMs that the projection's CTAs leave, where it does not need them all:
  // both then run side by side)
  const int free_sms = sm_count - projection_ctas;
  const int room = std::max(1, (free_sms >= tiles * groups ? free_sms : sm_count) / (tiles * groups));
  int split = 1;
  while (split < 8 && 4 * split <= kblocks && 2 * split <= room) split *= 2;
  const int slices = std::max(1, std::min(room / split, std::min(p.slots, std::min(p.rows, kShrinkRows))));
  return launch_shrink((const void*)lora_shrink_kernel, kShrinkSmem, 192,
                       dim3(tiles, groups * slices, split), maps, p, stream, pdl);
}

cudaError_t launch_lora_gemm(int kind, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int bn,
                             int split, cudaStream_t stream) {
  if (p.M < 1 || p.M > bn || p.N < 1 || split < 1 || split > 8 || (split & (split - 1)) || split > p.kblocks ||
      lp.rows != p.M)
    return cudaErrorInvalidValue;
  if (kind == kKindBf16) return dispatch_bn<kKindBf16>(bn, maps, p, lp, split, stream);
  if (kind == kKindFp8) return dispatch_bn<kKindFp8>(bn, maps, p, lp, split, stream);
  return cudaErrorInvalidValue;
}

// Row tile and K split of launch_lora_gemm.  Clusters of a power of two up to
// about two CTAs per SM (a cluster of seven packs badly on the GPCs).
void lora_few_plan(int M, int N, int kblocks, int sm_count, int* bn, int* split) {
  *bn = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  const int tiles = (N + 127) / 128;
  *split = 1;
  while (*split < 8 && 2 * *split <= kblocks && 2 * *split * tiles <= 2 * sm_count) *split *= 2;
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
