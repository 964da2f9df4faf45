// Projection with the low-rank adapters of many requests beside the shared
// weight:
//
//   out[m] = X[m] W^T + s_a (X[m] A_a^T) B_a^T,   a = index[m / index_div]
//
// in two launches.  The shrink computes V[m] = s_a X[m] A_a^T, a few ranks per
// row, in one of three kernels: lora_shrink_row_kernel (little work: one dot
// product a warp), lora_shrink_few_kernel (up to 64 rows, mma.sync)
// and lora_shrink_kernel (tcgen05).  The projection takes the adapters in on the
// way to its output, so that they cost no pass over it: lora_gemm_kernel (few
// rows) adds their terms with its K slices, lora_pair_kernel lengthens its
// reduction axis with the blocks of B_a.
//
// The shrink releases the projection once its own inputs are complete, so the
// projection's K blocks run beside it and only the adapters wait for V.
//
// V is kept as bf16 pairs hi + lo (hi = bf16(v), lo = bf16(v - hi)), about 16
// bits: a single bf16 V would round the adapter's term once more, by as much as
// the output's own rounding where the adapter dominates.  A chunk of 32 ranks
// is one 128-byte row [hi 32 | lo 32].
//
// FP8 projections keep the adapters in bf16, added to the scaled products.
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
// rows, by latency: 8,192 rows of K 2,624 with 16 adapters of rank 16 take 12 us,
// 7.5 of them the loads at the memory's rate; 777 of K 1,000 6.3 us, 1.9 until the
// adapters are numbered, 2.5 for the loads, 1.9 for the exchange and V.  (On
// mma.sync, small enough to share its SM with the projection, 15 us for 8,192 rows
// and 41 K blocks: too few bytes in flight.)
constexpr int kShrinkRows = 128;
constexpr int kShrinkRanks = 64;   // ranks of an adapter in one CTA
constexpr int kShrinkCols = 256;   // columns of one pass
constexpr int kShrinkXBytes = kShrinkRows * 128;
constexpr int kShrinkPipe = 4 * (kShrinkXBytes + kShrinkCols * 128);
constexpr int kShrinkStages = 10;  // at most
constexpr int kShrinkFirst = 4;  // row blocks requested before the adapters are known
static_assert(2 * kShrinkRows * (kShrinkRanks + 4) * 4 <= kShrinkPipe, "the parts lie over the stages");
constexpr int kListInts = 784;  // write_list's memory: the list, and number_adapters' for 256 rows
constexpr int kShrinkSmem = kShrinkPipe + (3 * 128 + 264 + kListInts) * 4 + 256 + 1024;

// The four warps that compute.
DEVI void sync128() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The first four warps of the projection.
DEVI void sync_low128() { asm volatile("bar.sync 2, 128;" ::: "memory"); }

// Numbers the distinct non-negative values of own[] (row h * 128 + thread, 128
// threads) in order of first appearance: ord[] of each row (-1: none), the
// values in s_list, their count returned (tid: 0..127).  A warp's leaders look for
// their value among the earlier warps' leaders only, so a tile of long runs costs
// a few steps.  s_tmp, s_entry: H * 128 ints (16-byte aligned); s_cnt: H * 8.
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
    if (lane == 0) s_cnt[h * 4 + warp] = __popc(leaders);
  }
  sync128();
#pragma unroll
  for (int h = 0; h < H; ++h) {
    seen[h] = H * 128;
    if (entry[h] >= 0)
#pragma unroll 1
      for (int w = 0; w < h * 4 + warp && seen[h] == H * 128; ++w)
#pragma unroll 1
        for (int j = w * 32; j < w * 32 + s_cnt[w]; j += 4) {
          const int4 v = *reinterpret_cast<const int4*>(s_tmp + j);
          if (v.w == own[h]) seen[h] = j + 3;
          if (v.z == own[h]) seen[h] = j + 2;
          if (v.y == own[h]) seen[h] = j + 1;
          if (v.x == own[h]) seen[h] = j;
        }
    firsts[h] = __ballot_sync(0xffffffffu, entry[h] >= 0 && seen[h] == H * 128);
    if (lane == 0) s_cnt[H * 4 + h * 4 + warp] = __popc(firsts[h]);
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
    n += s_cnt[H * 4 + w];
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

// Writes the list of the 256 rows from row0 for the projection: count and adapters.
// own: adapters of rows tid and 128 + tid; 128 threads; `w`: kListInts of shared memory.
DEVI void write_list(const LoraParams& p, int row0, const int (&own)[2], int* w) {
  const int tid = threadIdx.x;
  int ord[2] = {-1, -1};
  int* s_list = w;
  const int n = number_adapters<2>(tid, own, ord, s_list, w + 256, w + 512, w + 768);
  int* out = p.lists + (size_t)(row0 / 256) * kLoraListInts;
  for (int j = tid; j < n; j += 128) out[kLoraListSlots + j] = s_list[j];
  if (tid == 0) out[0] = n;
}

// The K slices' parts of a CTA's rows lie in part[row][pitch]; those that another
// CTA of the cluster owns go there in one copy, to recv[slice][its rows][pitch].
// One thread; the parts are complete and fenced, the peers' memory free.
DEVI void send_parts(const float* part, float* recv, int own_rows, int pitch, int rank, int split, uint64_t* sent) {
  const uint32_t bytes = own_rows * pitch * 4;
  mbar_expect_tx(sent, bytes * (split - 1));
  for (int d = 1; d < split; ++d) {
    const int to = (rank + d) % split;
    bulk_copy_to_peer(mapa_shared(smem_u32(recv + rank * own_rows * pitch), to), part + to * own_rows * pitch, bytes,
                      mapa_shared(smem_u32(sent), to));
  }
}

// What bf16(v) leaves of v; nothing where it is infinite or NaN.
DEVI float v_remainder(float v) {
  const float hi = bf16_round(v);
  return fabsf(hi) < INFINITY ? v - hi : 0.f;
}

// The parts of the kept columns of this CTA's rows [t0, t1) added in slice
// order, scaled, as V's hi + lo pairs, four ranks a thread.  taken(row): this
// pass of this CTA has the row's adapter; s_factor: the rows' scaling; r0: first
// rank of the columns.  Its loops are not unrolled: four rows at a time took a
// microsecond more.
template <class Taken>
DEVI void write_v(const LoraParams& p, const float* part, const float* recv, const float* s_factor, int row0, int t0,
                  int t1, int cols, int pitch, int r0, int rank, int split, Taken taken) {
  const int shift = cols <= 16 ? 2 : cols <= 32 ? 3 : 4;  // lanes of a row
  const int c = (threadIdx.x & ((1 << shift) - 1)) * 4, r = r0 + c;
  if (c >= cols || (r >> 5) >= p.chunks) return;
  const int per_slice = (t1 - t0) * pitch;
#pragma unroll 1
  for (int row = t0 + (int)(threadIdx.x >> shift); row < t1; row += 128 >> shift) {
    if (!taken(row)) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k = 0; k < split; ++k) {
      const float* src = k == rank ? part + row * pitch : recv + k * per_slice + (row - t0) * pitch;
      const float4 q = *reinterpret_cast<const float4*>(src + c);
      v.x += q.x;
      v.y += q.y;
      v.z += q.z;
      v.w += q.w;
    }
    const float f = s_factor[row];
    const float x[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    float lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) lo[k] = v_remainder(x[k]);
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
  uint8_t* sX = smem;  // row blocks from the front, adapter blocks from the back
  float* part = reinterpret_cast<float*>(smem);               // over the stages, between passes
  int* s_ord = reinterpret_cast<int*>(smem + kShrinkPipe);   // [128] each row's place in the list
  int* s_list = s_ord + 128;                                  // [128] distinct adapters
  float* s_factor = reinterpret_cast<float*>(s_list + 128);   // [128] each row's scaling
  int* s_tmp = s_list + 256;                                  // [128] + [128] + [4]: number_adapters
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
  // this CTA writes the list of 256 rows
  const bool lists = p.lists && row0 % 256 == 0 && blockIdx.y == 0 && rank == split - 1;
  int of_list[2] = {-1, -1};
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
      for (int k = 0; k < kShrinkFirst && k < nkb; ++k) load_rows(k, k);
      for (int k = kShrinkFirst; k < nkb; ++k) tma_prefetch_2d(&xmap, (kb0 + k) * 64, row0);  // to L2, meanwhile
    }
    __syncwarp();
  } else if (warp == 5) {
    tmem_alloc(tmem_slot, kShrinkCols);
    tmem_relinquish();
  } else {
    // ---- the tile's adapters in order of first use (the rows are on their way)
    const int own[1] = {row_adapter(p, row0 + tid)};
    of_list[0] = own[0];
    if (lists) of_list[1] = row_adapter(p, row0 + 128 + tid);
    int ord[1] = {-1};
    const float factor = own[0] >= 0 && p.scaling ? __ldg(p.scaling + own[0]) : 1.f;
    const int n = number_adapters<1>(tid, own, ord, s_list, s_tmp, s_tmp + 128, s_tmp + 256);
    s_ord[tid] = ord[0];
    s_factor[tid] = factor;
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
  const int pitch = cols + 4;
  float* recv = part + kShrinkRows * pitch;
  if (warp == 4 && u0 == u1)           // no adapter here: the rows still land before the exit
    for (int k = 0; k < kShrinkFirst && k < nkb; ++k) {
      if (elect_one()) mbar_arrive(&full[k]);
      __syncwarp();
      if (!warp_wait(&full[k], 0, limit) && lane == 0) atomicExch(failed, 1);
    }
  // the projection's list of 256 rows, while the first K blocks are on their way
  if (warp < 4 && lists) write_list(p, row0, of_list, s_tmp + 264);
  // as many stages as the memory holds with the columns of the largest pass
  const int a_bytes = (min(per, u1 - u0) * cols * 128 + 1023) & ~1023;
  const int stages = min(ST, kShrinkPipe / (kShrinkXBytes + a_bytes));
  auto adapters_of = [&](int s) { return smem + kShrinkPipe - (s + 1) * a_bytes; };
  struct {
    int s = 0;
    uint32_t phase = 0;
    DEVI void next(int n) {
      if (++s == n) {
        s = 0;
        phase ^= 1;
      }
    }
  } ring;
  uint32_t g = 0, pass = 0;  // K blocks and passes before this one
  for (int u = u0; u < u1; u += per, ++pass) {
    // (after a failure the passes still meet at their barriers)
    const int units = u1 - u < per ? u1 - u : per;
    const int todo = *reinterpret_cast<volatile int*>(failed) ? 0 : nkb;
    if (warp == 4) {
      for (int k = 0; k < todo; ++k, ++g, ring.next(stages)) {
        const int s = ring.s;
        if ((int)g >= stages && !warp_wait(&empty[s], ring.phase ^ 1, limit)) {
          if (lane == 0) atomicExch(failed, 1);
          break;
        }
        if (elect_one()) {
          if (g >= kShrinkFirst || (int)g >= nkb) load_rows(s, k);  // (the first ones were requested above)
          mbar_expect_tx(&full[s], units * cols * 128);
          for (int a = 0; a < units; ++a)
            tma_load_3d(adapters_of(s) + a * cols * 128, &amap, &full[s], (kb0 + k) * 64, group * kShrinkRanks,
                        s_list[u + a], pol);
        }
        __syncwarp();
      }
    } else if (warp == 5) {
      const uint32_t idesc = idesc_bf16(128, units * cols);
      const uint32_t x0 = desc_lo(smem_u32(sX));
      for (int k = 0; k < todo; ++k, ring.next(stages)) {
        const int s = ring.s;
        if (!warp_wait(&full[s], ring.phase, limit)) {
          if (lane == 0) atomicExch(failed, 1);
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t xd = x0 + s * (kShrinkXBytes >> 4), ad = desc_lo(smem_u32(adapters_of(s)));
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
    // The parts go over the stages, whose blocks have all been read: each row's
    // kept columns.
    const int own_rows = kShrinkRows / split, t0 = rank * own_rows;
    if (warp < 4) {
      const int o = s_ord[tid];
      float* here = part + tid * pitch;
      for (int a = 0; a < units; ++a) {
        if (!__any_sync(0xffffffffu, o == u + a)) continue;
        const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + a * cols;
        for (int c = 0; c < cols; c += 16) {
          uint32_t r[16];
          tmem_ld16(acc + c, r);
          tmem_wait_ld();
          if (o == u + a)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<uint4*>(here + c + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      sync128();
    }
    if (split > 1) {
      cluster_sync_relaxed();  // every CTA's stages are free
      if (warp == 0 && elect_one()) send_parts(part, recv, own_rows, pitch, rank, split, sent);
      __syncwarp();
      if (warp < 4 && !warp_wait_cluster(sent, pass & 1, limit) && lane == 0) atomicExch(failed, 1);
      __syncwarp();
      cluster_arrive_relaxed();
    }
    if (warp < 4)
      write_v(p, part, recv, s_factor, row0, t0, t0 + own_rows, cols, pitch, group * kShrinkRanks, rank, split,
              [&](int row) { return s_ord[row] >= u && s_ord[row] < u + units; });
    // the parts are read, here and by the copies; the next pass may take their place
    fence_proxy_async_smem();
    if (split > 1) cluster_wait();
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
// and in little shared memory, so that several share an SM and the projection's
// CTAs start beside them (64 rows of one adapter of rank 256, K and N 1,024: 13.5
// us with the projection).
constexpr int kFewRows = 64;

struct FewShrinkCfg {
  static constexpr int COLS = 64;  // of one adapter of more than 32 ranks, or of several at a time
  static constexpr int STAGES = 3;
  static constexpr int X_BYTES = kFewRows * 128, A_BYTES = COLS * 128;
  static constexpr int PIPE_BYTES = STAGES * (X_BYTES + A_BYTES);
  static_assert(2 * kFewRows * (kShrinkRanks + 4) * 4 <= PIPE_BYTES, "the parts fit the pipeline's memory");
  static constexpr int SMEM = PIPE_BYTES + (3 * 128 + 264) * 4 + 128 + 1024;
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

__global__ void __launch_bounds__(160)
    lora_shrink_few_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap amap,
                       const LoraParams p) {
  using C = FewShrinkCfg;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sA = smem + ST * C::X_BYTES;
  float* part = reinterpret_cast<float*>(smem);                // over the stages, between passes
  int* s_ord = reinterpret_cast<int*>(smem + C::PIPE_BYTES);   // [128] each row's place in the list
  int* s_list = s_ord + 128;                                    // [128] distinct adapters
  float* s_factor = reinterpret_cast<float*>(s_list + 128);    // [128] each row's scaling
  int* s_tmp = s_list + 256;                                    // [128] + [128] + [4]: number_adapters
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
    const float factor = own[0] >= 0 && p.scaling ? __ldg(p.scaling + own[0]) : 1.f;
    const int n = number_adapters<1>(tid, own, ord, s_list, s_tmp, s_tmp + 128, s_tmp + 256);
    s_ord[tid] = ord[0];
    s_factor[tid] = factor;
    if (tid == 0) *s_count = n;
  }
  __syncthreads();
  const int n = *s_count;
  const int u0 = (int)((long long)slice * n / slices), u1 = (int)((long long)(slice + 1) * n / slices);
  const int per = C::COLS / cols;  // adapters of one pass
  const int pitch = cols + 4;
  float* recv = part + kFewRows * pitch;
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
    // The parts go over the stages, once all of them have been read: each row's
    // kept columns.
    const int own_rows = kFewRows / split, t0 = rank * own_rows;
    __syncthreads();
    if (!loader) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = warp * 16 + (lane >> 2) + 8 * h, unit = s_ord[row] - u;
        if (unit < 0 || unit >= units) continue;
#pragma unroll
        for (int j = 0; j < C::COLS / 8; ++j) {
          const int c = 8 * j + (lane & 3) * 2 - unit * cols;
          if (c >= 0 && c < cols)
            *reinterpret_cast<float2*>(part + row * pitch + c) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
        }
      }
      __syncwarp();
      fence_proxy_async_smem();
      sync128();
    }
    if (split > 1) {
      cluster_sync_relaxed();  // every CTA's stages are free
      if (warp == 0 && elect_one()) send_parts(part, recv, own_rows, pitch, rank, split, sent);
      __syncwarp();
      if (!loader && !warp_wait_cluster(sent, pass & 1, limit) && lane == 0) atomicExch(failed, 1);
      __syncwarp();
      cluster_arrive_relaxed();
    }
    if (!loader)
      write_v(p, part, recv, s_factor, 0, t0, t0 + own_rows, cols, pitch, group * kShrinkRanks, rank, split,
              [&](int row) { return s_ord[row] >= u && s_ord[row] < u + units; });
    // the parts are read, here and by the copies; the next pass may take their place
    fence_proxy_async_smem();
    if (split > 1) cluster_wait();
    __syncthreads();
  }
  if (tid == 0 && *reinterpret_cast<volatile int*>(failed))
    record_status(p.status ? p.status : &g_op_status, kStatusGemmFullTimeout);
}

// V of few rows by single dot products: a CTA takes eight ranks of one row, a
// warp one of them, and reads its adapter's rows for itself.  Nothing is numbered
// or exchanged and no shared memory is held, so the projection's CTAs all start
// beside it; rows of one adapter read it again from L2.  Bound by the latency of
// two dependent loads.
constexpr int kRowShrinkWarps = 8;

__global__ void __launch_bounds__(32 * kRowShrinkWarps) lora_shrink_row_kernel(const LoraParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int row = blockIdx.y, r = blockIdx.x * kRowShrinkWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int slot = row_adapter(p, row), octets = p.in_features / 8;
  if (slot < 0) return;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + (size_t)row * p.ldx);
  const uint4* a = reinterpret_cast<const uint4*>(p.a + ((size_t)slot * p.rank + r) * p.in_features);
  const float factor = p.scaling ? __ldg(p.scaling + slot) : 1.f;
  float sum = 0.f;
  for (int c = lane; c < octets; c += 128) {
    uint4 u[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = v[i] = make_uint4(0, 0, 0, 0);
      if (c + 32 * i < octets) {
        u[i] = x[c + 32 * i];
        v[i] = __ldg(a + c + 32 * i);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t *ui = &u[i].x, *vi = &v[i].x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum += __uint_as_float(ui[e] << 16) * __uint_as_float(vi[e] << 16);
        sum += __uint_as_float(ui[e] & 0xffff0000u) * __uint_as_float(vi[e] & 0xffff0000u);
      }
    }
  }
  sum = warp_sum(sum);
  if (lane) return;
  sum *= factor;
  const float lo = v_remainder(sum);
  __nv_bfloat16* dst = p.v + ((size_t)row * p.chunks + (r >> 5)) * 64 + (r & 31);
  dst[0] = __float2bfloat16_rn(sum);
  dst[32] = __float2bfloat16_rn(lo);
}

// ------------------------------------------------- projection for few rows
// Few tiles, bound by reading W and the adapters: the tile layout and split-K of
// gemm.cu (weight rows on the TMEM lanes, up to 64 rows of X as the MMA's N).
// The adapters are not blocks of that reduction here.  A CTA stores BN / split
// rows, and four warps compute those rows' adapter terms with mma.sync, in fp32,
// while the K blocks and the exchange of the slices run: per group of eight rows
// and adapter that they use, 16 ranks a step, the other rows' V zero.  B_a goes
// from memory to registers, the first of it before V is there, and the terms wait
// for no stage.  Measured, 64 rows with 64 adapters of rank 16 into 5,248 features:
// 10.9 us, 8.9 with one adapter, 8.6 with none (the bytes take 3.5): the two
// launches' chain, then 0.3 us a step, which is the loads' latency over the three
// steps that registers hold.  (As K blocks of the tcgen05 pipeline, V tiles built
// in shared memory, 17.7 us: a block took 0.5 us from its stage's release to its
// MMAs.)  Three stages: the shrink's CTAs then leave room for every CTA of this
// kernel beside them (with four, the last ones started 4 us late).
constexpr int kAdapterWarps = 4;

template <int BN, int KIND>
struct LoraCfg {
  static constexpr int STAGES = 3;
  static constexpr int THREADS = 128 + 32 * kAdapterWarps;
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
  static constexpr int PART_BYTES = 2 * BN * 128 * 4;  // the partial tile, and its tokens' from the other slices
  static constexpr int MAIN_BYTES = PIPE_BYTES > PART_BYTES ? PIPE_BYTES : PART_BYTES;
  static constexpr int LIST_BYTES = (3 * BN + 4) * 4;  // adapters, activation scales; behind them the adapter terms
  static constexpr int BAR_BYTES = 128;
  static constexpr int SMEM = MAIN_BYTES + BAR_BYTES + LIST_BYTES + 1024;
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int K_ELEMS = KIND == kKindBf16 ? 64 : 128;
};

// One group of rows: its two lists' terms are added up in the end.
__host__ __device__ constexpr int lora_term_lists(int nt) { return nt <= 8 ? 2 : 1; }

// The adapters of `nt` rows from t0 in groups of eight: two lists of pairs (slot;
// group, and which of its rows use the slot) in group order, s_pair[0..] of the
// even groups, s_pair[half..] of the odd ones, or of the only group's pairs in
// turn, their lengths in s_count; one warp.  Their B_a for the features [n0, n0 +
// 128), contiguous, is on its way to L2.
DEVI void pair_adapters(const LoraParams& p, int t0, int nt, bool one_group, int n0, int half, int2* s_pair,
                        int* s_count) {
  const int lane = threadIdx.x & 31;
  int n0_list = 0, n1_list = 0;
  for (int first = 0; first < nt; first += 32) {
    const int i = first + lane, own = i < nt ? row_adapter(p, t0 + i) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, own) & (0xffu << (lane & 24)), below = (1u << lane) - 1;
    const bool leads = own >= 0 && __ffs(same) - 1 == lane;
    const unsigned leaders = __ballot_sync(0xffffffffu, leads);
    const int odd = one_group ? __popc(leaders & below) & 1 : (lane >> 3) & 1;
    const unsigned ones = __ballot_sync(0xffffffffu, leads && odd), list = odd ? ones : leaders & ~ones;
    if (leads) {
      s_pair[(odd ? half + n1_list : n0_list) + __popc(list & below)] =
          make_int2(own, i >> 3 | same >> (lane & 24) << 8);
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                       p.b + ((size_t)own * p.out_features + n0) * p.rank),
                   "r"(min(128, p.out_features - n0) * p.rank * 2)
                   : "memory");
    }
    n0_list += __popc(leaders & ~ones);
    n1_list += __popc(ones);
  }
  if (lane == 0) {
    s_count[0] = n0_list;
    s_count[1] = n1_list;
  }
}

// Four ranks (W = 1) or eight, or zero.
template <int W>
struct Ranks {
  uint2 q[W];
};
template <int W>
DEVI Ranks<W> load_ranks_if(const __nv_bfloat16* p, bool in) {
  Ranks<W> v;
  if constexpr (W == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %3, 0;\n mov.u32 %0, 0;\n mov.u32 %1, 0;\n"
        " @p ld.global.cg.v2.u32 {%0,%1}, [%2];\n}\n"
        : "=r"(v.q[0].x), "=r"(v.q[0].y)
        : "l"(p), "r"((int)in));
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n mov.u32 %0, 0;\n mov.u32 %1, 0;\n mov.u32 %2, 0;\n"
        " mov.u32 %3, 0;\n @p ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];\n}\n"
        : "=r"(v.q[0].x), "=r"(v.q[0].y), "=r"(v.q[W - 1].x), "=r"(v.q[W - 1].y)
        : "l"(p), "r"((int)in));
  return v;
}
template <int W>
DEVI Ranks<W> load_ranks(const __nv_bfloat16* p) {
  Ranks<W> v;
  if constexpr (W == 1)
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.q[0].x), "=r"(v.q[0].y) : "l"(p));
  else
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.q[0].x), "=r"(v.q[0].y), "=r"(v.q[W - 1].x), "=r"(v.q[W - 1].y)
                 : "l"(p));
  return v;
}
// A warp's share of the adapter terms: 64 features from n0 (four m16 tiles) of a
// list of pairs.  A step is 16 W ranks of a pair; a lane holds 4 W consecutive
// ranks of a row of B_a and of V, which an instruction takes four of as two pairs:
// the order of the ranks in its sum is free.  AHEAD steps are in registers, each
// one's place taken by its successor's loads at once, and the pair of the next
// loads is read a step before them.  What a step has too many of (ranks, features,
// steps behind the last) it loads from the nearest valid address and multiplies
// with a zero V, or adds to a column that is not stored: one warp per scheduler is
// bound by its instructions (0.3 us a step; a predicate for each load doubled them,
// six steps ahead gained nothing).  With W = 2 the two steps of B_a take 64 of the
// 128 registers that two CTAs an SM leave a thread, and 88 bytes of a thread spill
// (W = 1: none).
template <int W>
struct AdapterTerms {
  static constexpr int AHEAD = W == 1 ? 3 : 2;
  const LoraParams& p;
  const int2* s_pair;
  int pairs, t0, nt;
  int off[8];  // the lane's rows of B_a
  Ranks<W> b[AHEAD][8], hi[AHEAD], lo[AHEAD];
  int group[AHEAD];  // -1 behind the last step
  int pair_b, k_b, pair_v, k_v;  // the next step to load
  int slot_b;
  int2 of_v;

  DEVI void next(int& pair, int& k) const {
    k += 16 * W;
    const bool end = k >= p.rank;
    k = end ? 0 : k;
    pair += end;
  }
  DEVI void load_b(int u) {
    const int k = min(k_b + 4 * W * (int)(threadIdx.x & 3), p.rank - 4 * W);
    const __nv_bfloat16* src = p.b + (size_t)(unsigned)slot_b * ((size_t)p.out_features * p.rank) + k;
#pragma unroll
    for (int j = 0; j < 8; ++j) b[u][j] = load_ranks<W>(src + off[j]);
    next(pair_b, k_b);
    slot_b = s_pair[min(pair_b, pairs - 1)].x;
  }
  DEVI void load_v(int u) {
    const int g = (threadIdx.x & 31) >> 2, k = k_v + 4 * W * (int)(threadIdx.x & 3);
    const int to = of_v.y & 0xff, row = t0 + to * 8 + g;
    const bool in = pair_v < pairs && k < p.rank && (of_v.y >> (8 + g) & 1);
    const __nv_bfloat16* src = p.v + ((size_t)row * p.chunks + (k >> 5)) * 64 + (k & 31);
    hi[u] = load_ranks_if<W>(src, in);
    lo[u] = load_ranks_if<W>(src + 32, in);
    group[u] = pair_v < pairs ? to : -1;
    next(pair_v, k_v);
    of_v = s_pair[min(pair_v, pairs - 1)];
  }
  // B_a does not wait for V
  DEVI void start(int n0) {
    if (pairs == 0) return;
    const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) off[j] = min(n0 + 8 * j + g, p.out_features - 1) * p.rank;
    pair_b = k_b = pair_v = k_v = 0;
    of_v = s_pair[0];
    slot_b = of_v.x;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load_b(u);
  }
  // out[row][128] = the terms (out: row t0, the warp's first feature)
  DEVI void store_to(float* out) {
    if (pairs == 0) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float acc[4][4] = {};
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load_v(u);
    int now = group[0];
    while (true) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (group[u] != now) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (now * 8 + 2 * t + e < nt) {
              float* dst = out + (now * 8 + 2 * t + e) * 128 + g;
#pragma unroll
              for (int f = 0; f < 8; ++f) dst[8 * f] = acc[f >> 1][(f & 1) * 2 + e];
            }
          if (group[u] < 0) return;
          now = group[u];
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
        }
#pragma unroll
        for (int w = 0; w < 2 * W; ++w)
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const uint2 c = b[u][2 * m].q[w / 2], d = b[u][2 * m + 1].q[w / 2];
            const uint2 v = w % 2 ? lo[u].q[w / 2] : hi[u].q[w / 2];
            const uint32_t a[4] = {c.x, d.x, c.y, d.y};
            mma_bf16(acc[m], a, v.x, v.y);
          }
        load_b(u);
        load_v(u);
      }
    }
  }
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

// W: AdapterTerms' (ranks above 16: 2).
template <int BN, int KIND, int W>
__global__ void __launch_bounds__(LoraCfg<BN, KIND>::THREADS, 2)
    lora_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                     const GemmParams p, const LoraParams lp) {
  using C = LoraCfg<BN, KIND>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::MAIN_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint64_t* sent = done + 1;  // the cluster's parts of this CTA's tokens
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sent + 1);
  uint32_t* failed = tmem_slot + 1;
  static_assert((2 * STAGES + 2) * 8 + 8 <= C::BAR_BYTES, "barrier block");
  int2* s_pair = reinterpret_cast<int2*>(smem + C::MAIN_BYTES + C::BAR_BYTES);  // [BN] adapters of the CTA's tokens
  float* s_scale = reinterpret_cast<float*>(s_pair + BN);                       // [BN] activation scales (fp8)
  int* s_count = reinterpret_cast<int*>(s_scale + BN);                          // [2], and two unused
  float* s_terms = reinterpret_cast<float*>(s_count + 4);  // [lists][BN / split][128] adapter terms

  const int tid = threadIdx.x, warp = tid >> 5;
  const int tile_n = blockIdx.x, m0 = blockIdx.y * BN;
  const int rows = min(BN, p.M - m0);
  const int split = gridDim.z, rank = blockIdx.z;
  const int kb0 = (int)((long long)rank * p.kblocks / split);
  const int kb1 = (int)((long long)(rank + 1) * p.kblocks / split);
  const int nkb = kb1 - kb0;
  const int nt = BN / split, t0 = rank * nt;          // the tokens that this CTA stores,
  const int stored = max(0, min(rows - t0, nt));       // those that exist
  const int lists = lora_term_lists(nt);
  uint32_t* status = p.status ? p.status : &g_op_status;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(sent, 1);
    *failed = 0;
    fence_mbar_init();
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&xmap);
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

  const uint64_t limit = wait_limit(p.wait_limit_us);
  int issued = 0;  // producer warp: loads issued (for the drain on failure)
  auto give_up = [&](uint32_t code) {
    record_status(status, code);
    atomicExch(failed, 1u);
  };
  // W, X, the adapters and the activation scales do not wait for the shrink:
  // whatever wrote them was complete before it released this kernel.
  if (warp == 0) {
    const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
    Ring<STAGES> ring;
    bool ok = true;
    for (int i = 0; i < nkb; ++i, ring.next()) {
      const int s = ring.s;
      if (i >= STAGES && !(ok = warp_wait(&empty[s], ring.phase ^ 1, limit))) break;
      if (elect_one()) {
        mbar_expect_tx(&full[s], C::STAGE_BYTES);
        tma_load_2d(sA + s * C::A_BYTES, &wmap, &full[s], (kb0 + i) * C::K_ELEMS, tile_n * 128, pol_w);
        tma_load_2d(sB + s * C::B_BYTES, &xmap, &full[s], (kb0 + i) * C::K_ELEMS, m0, pol_x);
      }
      __syncwarp();
      issued = i + 1;
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
    if (!ok && (tid & 31) == 0) give_up(kStatusGemmFullTimeout);
    if (elect_one()) umma_commit(done);
    __syncwarp();
  } else if (warp >= 4) {
    // ---- the adapter terms of the CTA's tokens
    const int bt = tid - 128, odd = (warp >> 1) & 1, half = (warp & 1) * 64;
    for (int i = bt; i < lists * nt * 32; i += 32 * kAdapterWarps)
      reinterpret_cast<float4*>(s_terms)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (warp == 4) pair_adapters(lp, m0 + t0, stored, lists == 2, tile_n * 128, BN / 2, s_pair, s_count);
    sync128();
    AdapterTerms<W> terms{lp, s_pair + odd * (BN / 2), s_count[odd], m0 + t0, stored};
    terms.start(tile_n * 128 + half);
    // (these warps have no part in the partial tile: they arrive at once, and wait
    // when they are done)
    if (split > 1) cluster_arrive_relaxed();
    griddep_wait();  // V
    terms.store_to(s_terms + odd * (lists - 1) * nt * 128 + half);
    if (split > 1) cluster_wait();
  } else if (KIND == kKindFp8) {
    for (int i = tid - 64; i < BN; i += 64) s_scale[i] = i < rows ? p.a_scale[m0 + i] : 0.f;
  }
  __syncwarp();

  // ---- epilogue: the partial tile [token][128] lies over the stages; each
  // other CTA of the cluster is sent the tokens it stores in one copy, to
  // recv[slice][token][128] behind the partial tile (its stages are free too
  // once the relaxed barrier is passed)
  float* part = reinterpret_cast<float*>(smem);
  float* recv = part + BN * 128;
  if (warp < 4) {
    if (!warp_wait(done, 0, limit) && (tid & 31) == 0) give_up(kStatusGemmDoneTimeout);
    tc_fence_after();
    if (KIND == kKindFp8) sync_low128();  // the activation scales
    const int lr = tid;  // weight row of the tile
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    const float ws = KIND == kKindFp8 && tile_n * 128 + lr < p.N ? p.w_scale[tile_n * 128 + lr] : 1.f;
    constexpr int COLS = BN < 32 ? 16 : 32;
#pragma unroll 1
    for (int c = 0; c < BN && c < rows; c += COLS) {
      uint32_t r[COLS];
      if constexpr (COLS == 32) tmem_ld32(tmem + lane_addr + c, r); else tmem_ld16(tmem + lane_addr + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < COLS; ++j) {
        float v = nkb > 0 ? __uint_as_float(r[j]) : 0.f;
        if (KIND == kKindFp8) v = (v * s_scale[c + j]) * ws;
        part[(c + j) * 128 + lr] = v;
      }
    }
    tc_fence_before();
    fence_proxy_async_smem();
    if (split > 1) {
      cluster_arrive_relaxed();
      cluster_wait();  // every CTA's stages are free
      sync_low128();   // and this one's partial tile complete
      if (warp == 0 && elect_one()) {
        mbar_expect_tx(sent, stored * (split - 1) * 512);
        for (int d = 1; d < split; ++d) {
          const int to = (rank + d) % split, tokens = min(rows - to * nt, nt);
          if (tokens > 0)
            bulk_copy_to_peer(mapa_shared(smem_u32(recv + rank * nt * 128), to), part + to * nt * 128, tokens * 512,
                              mapa_shared(smem_u32(sent), to));
        }
      }
      __syncwarp();
    }
    griddep_wait();  // what wrote or read the output
  }
  if (split > 1 && !warp_wait_cluster(sent, 0, limit) && (tid & 31) == 0) give_up(kStatusGemmDoneTimeout);
  __syncthreads();
  {
    const bool rope = tile_n * 128 < p.rope_cols;
    const int pair = rope ? 32 : 64;
    const bool residual = p.epilogue == kEpiResidual;
    const bool plain = p.epilogue == kEpiStore && !rope;
    const bool vec = p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
    for (int item = tid; item < stored * 16; item += C::THREADS) {
      const int q4 = rope ? ((item >> 3) & 1) * 64 + (item & 7) * 4 : (item & 15) * 4;
      const int m = m0 + t0 + (item >> 4), n = tile_n * 128 + q4;
      EpiPre pre;
      if (!plain) pre = epi_prefetch<kKindBf16>(p, m, n, residual, rope);
      float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
      const int at = (item >> 4) * 128 + q4;
#pragma unroll 2
      for (int u = 0; u < split + lists; ++u) {  // the slices in order, then the adapters
        const float* src = u >= split   ? s_terms + (u - split) * nt * 128
                           : u == rank ? part + t0 * 128
                                       : recv + u * nt * 128;
        src += at;
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

template <int BN, int KIND, int W>
cudaError_t launch_one(const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int split,
                       cudaStream_t stream) {
  using C = LoraCfg<BN, KIND>;
  auto kern = lora_gemm_kernel<BN, KIND, W>;
  // Function attributes are per device: set them once for each device used.
  static std::mutex mu;
  static uint64_t ready = 0;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!(ready >> dev & 1)) {
      // (an unsplit K takes the most: the terms of BN rows)
      err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM + BN * 512);
      if (err != cudaSuccess) return err;
      ready |= uint64_t(1) << dev;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + 127) / 128, (p.M + BN - 1) / BN, split);
  cfg.blockDim = dim3(C::THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM + lora_term_lists(BN / split) * (BN / split) * 512;
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
  return cudaLaunchKernelEx(&cfg, kern, maps.w, maps.x, p, lp);
}

template <int KIND, int W>
cudaError_t dispatch_bn(int bn, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int split,
                        cudaStream_t st) {
  switch (bn) {
    case 16: return launch_one<16, KIND, W>(maps, p, lp, split, st);
    case 32: return launch_one<32, KIND, W>(maps, p, lp, split, st);
    case 64: return launch_one<64, KIND, W>(maps, p, lp, split, st);
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
  void* with_maps[] = {const_cast<CUtensorMap*>(&maps.rows), const_cast<CUtensorMap*>(&maps.a),
                       const_cast<LoraParams*>(&p)};
  void** args = smem ? with_maps : with_maps + 2;  // (the kernel without shared memory takes no tensor map)
  return cudaLaunchKernelExC(&cfg, kern, args);
}

}  // namespace

namespace {

// The tcgen05 shrink, one CTA per SM: K is split until they are in use (two K
// blocks at least each), then the adapters, of which single rows of many requests
// bring many.  On the SMs that the projection's CTAs leave, where it does not need
// them all, both run side by side; on all of them it is done sooner, but the
// projection waits (FP8, 2,048 rows of K 2,624 into 1,024 beside 64 pairs took 26.6
// us, K not split; before them 18.6).  us: of both, roughly 3.5 us and 0.4 a K
// block for the shrink.
struct ShrinkPlan {
  int split, slices;  // K slices; shares of a row tile's adapters
  float us;
};
// CTAs that run at a time in clusters of this size, one for an SM: the groups of SMs
// that a cluster has to fit hold 15 clusters of eight and 33 of four on 148 SMs (a
// few CTAs more ran as a second wave, 5 us after the first).
int cluster_room(int sms, int size) { return size >= 8 ? sms * 120 / 148 : size == 4 ? sms * 132 / 148 : sms; }

ShrinkPlan shrink_plan(int rows, int rank, int in_features, int sm_count, int projection_ctas, float projection_us) {
  const int tiles = (rows + kShrinkRows - 1) / kShrinkRows * ((rank + kShrinkRanks - 1) / kShrinkRanks);
  const int kblocks = (in_features + 63) / 64, free_sms = sm_count - projection_ctas;
  auto plan = [&](int sms) {
    auto room = [&](int split) { return std::min(sms, cluster_room(sm_count, split)); };
    int split = 1;
    while (split < 8 && 4 * split <= kblocks && 2 * split * tiles <= room(2 * split)) split *= 2;
    const int slices = std::max(1, room(split) / (tiles * split));
    return ShrinkPlan{split, slices, 3.5f + 0.4f * (float)kblocks / (float)split};
  };
  ShrinkPlan before = plan(sm_count);
  before.us += projection_us;
  if (free_sms < tiles) return before;
  ShrinkPlan beside = plan(free_sms);
  beside.us = std::max(beside.us, projection_us);
  return beside.us <= before.us ? beside : before;
}

}  // namespace

// Up to two tiles of 64 rows x 128 features for three SMs lora_gemm_kernel is done
// sooner (331 rows of K 392 into 2,302 11.4 us, pairs 13.0; 102 rows with 25 adapters,
// K 1,040 into 860, 10.6 and 26.5; but 605 rows of K 440 into 1,331 15.6 and 13.5).
// Else the tiles with which both kernels are (bf16 takes 128 features where
// 256 would leave pairs idle; FP8, 8,192 rows of K 2,624 into 1,024: 41.7 us with
// 128, 37.2 with 256; K 1,024 into 5,248: 69.1, 68.1).
int lora_pair_plan(int kind, int M, int N, int K, int rank, int sm_count) {
  if (M <= kFewRows || 3ll * ((M + 63) / 64) * ((N + 127) / 128) <= 2 * sm_count) return 0;
  const int kblocks = (K + gemm_k_elems(kind) - 1) / gemm_k_elems(kind);
  auto us = [&](int bnf) {
    return shrink_plan(M, rank, K, sm_count, lora_pair_ctas(M, N, bnf, sm_count),
                       lora_pair_us(kind, M, N, kblocks, bnf, sm_count))
        .us;
  };
  return us(256) <= us(128) ? 256 : 128;
}

cudaError_t launch_lora_shrink(const LoraMaps& maps, const LoraParams& p, int sm_count, int projection_ctas,
                               float projection_us, cudaStream_t stream, bool pdl) {
  if (p.rows < 1 || p.rank < 8 || p.rank % 8 || p.rank > kLoraMaxRank || p.in_features % 8 || p.slots < 1 ||
      p.index_div < 1)
    return cudaErrorInvalidValue;
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
      if (err == cudaSuccess) err = cudaFuncSetAttribute(lora_shrink_few_kernel, attr, FewShrinkCfg::SMEM);
      if (err != cudaSuccess) return err;
      ready |= uint64_t(1) << dev;
    }
  }
  const int groups = (p.rank + kShrinkRanks - 1) / kShrinkRanks, kblocks = (p.in_features + 63) / 64;
  if (!p.lists && lora_shrink_by_row(p.rows, p.rank, p.in_features))
    return launch_shrink((const void*)lora_shrink_row_kernel, 0, 32 * kRowShrinkWarps,
                         dim3(p.rank / kRowShrinkWarps, p.rows, 1), maps, p, stream, pdl);
  if (lora_shrink_rows(p.rows) == kFewRows) {
    // The adapters are spread first, then K, up to three CTAs per SM.
    const int per = FewShrinkCfg::COLS / lora_shrink_box(p.rank), room = std::max(1, 3 * sm_count / groups);
    const int slices = std::min(room, (std::min(p.slots, p.rows) + per - 1) / per);
    int split = 1;
    while (split < 8 && 2 * split <= kblocks && 2 * split * slices <= room) split *= 2;
    return launch_shrink((const void*)lora_shrink_few_kernel, FewShrinkCfg::SMEM, 160, dim3(1, groups * slices, split),
                         maps, p, stream, pdl);
  }
  const int tiles = (p.rows + kShrinkRows - 1) / kShrinkRows;
  const ShrinkPlan plan = shrink_plan(p.rows, p.rank, p.in_features, sm_count, projection_ctas, projection_us);
  const int split = plan.split;
  const int slices = std::min(plan.slices, std::min(p.slots, std::min(p.rows, kShrinkRows)));
  return launch_shrink((const void*)lora_shrink_kernel, kShrinkSmem, 192,
                       dim3(tiles, groups * slices, split), maps, p, stream, pdl);
}

cudaError_t launch_lora_gemm(int kind, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int bn,
                             int split, cudaStream_t stream) {
  if (p.M < 1 || (p.M + bn - 1) / bn > 65535 || p.N < 1 || split < 1 || split > 8 || (split & (split - 1)) ||
      lp.rows != p.M || !lp.b)
    return cudaErrorInvalidValue;
  const bool wide = lp.rank > 16;
  if (kind == kKindBf16)
    return wide ? dispatch_bn<kKindBf16, 2>(bn, maps, p, lp, split, stream)
                : dispatch_bn<kKindBf16, 1>(bn, maps, p, lp, split, stream);
  if (kind == kKindFp8)
    return wide ? dispatch_bn<kKindFp8, 2>(bn, maps, p, lp, split, stream)
                : dispatch_bn<kKindFp8, 1>(bn, maps, p, lp, split, stream);
  return cudaErrorInvalidValue;
}

// Row tile and K split of launch_lora_gemm.  Clusters of a power of two up to
// about two CTAs per SM (a cluster of seven packs badly on the GPCs); a CTA of more
// than eight rows is split for its adapter terms too, where K blocks run out.
void lora_few_plan(int M, int N, int kblocks, int sm_count, int* bn, int* split) {
  *bn = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  const long long tiles = (long long)((N + 127) / 128) * ((M + *bn - 1) / *bn);
  *split = 1;
  while (*split < 8 && (2 * *split <= kblocks || *bn / *split > 8) &&
         2 * *split * tiles <= 2 * cluster_room(sm_count, 2 * *split))
    *split *= 2;
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
