// Host-side launchers of the b200 kernels (all take the stream to enqueue on
// and whether to allow programmatic dependent launch on the previous kernel).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include "params.h"

namespace laya {

int gemm_token_tile(int M);
void gemm_plan(int M, int N, int kblocks, int sm_count, int* bn, int* split);
int gemm_k_elems(int kind);
int gemm_split(int tiles, int kblocks, int sm_count, int max_split);
cudaError_t launch_gemm(int kind, const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& omap,
                        const GemmParams& p, int bn, int split, cudaStream_t stream, bool pdl);

// Fused attention + residual output projection for one sequence of
// 32 < s <= 64 tokens (bf16, q and k already rotated): attention of the CTA's
// heads computed in shared memory as the B operand (gemm_attn.cu).
cudaError_t launch_gemm_attn(const CUtensorMap& wmap, const GemmParams& p, const AttnParams& a, int split,
                             cudaStream_t stream, bool pdl);
// Projection (store / GEGLU epilogue) of LN(h) for one sequence of
// 32 < s <= 64 tokens (bf16): the LayerNorm is applied while the operand is
// built, from the row statistics of the previous residual projection
// (gemm_ln.cu).
cudaError_t launch_gemm_ln(const CUtensorMap& wmap, const GemmParams& p, const LnParams& ln, int split,
                           cudaStream_t stream, bool pdl);
cudaError_t launch_gemm_nvfp4(const CUtensorMap& wmap, const CUtensorMap& xmap, const CUtensorMap& omap,
                              const uint8_t* wsf,
                              const uint8_t* xsf, int sf_kbs, const GemmParams& p, int bn, int split,
                              cudaStream_t stream, bool pdl);
cudaError_t launch_nvfp4_pack_weight(const __nv_bfloat16* w, int rows, int k, unsigned int* amax_scratch, uint8_t* q,
                                     uint8_t* sf, int col_blocks, float* tensor_scale, cudaStream_t stream);
cudaError_t launch_quant_nvfp4(const QuantParams& p, int rows_per_block, int col_blocks, cudaStream_t stream,
                               bool pdl);
// Attention of `heads` heads of `batch` sequences on tcgen05 tensor cores;
// qkv_map: 3-D map of p.qkv as [batch][s][ld_qkv] bf16, box 64 x 64 x 1,
// 128-byte swizzle.  At most 512 keys visible to any 128-query tile.
cudaError_t launch_attention(const AttnParams& p, const CUtensorMap& qkv_map, int batch, int heads,
                             cudaStream_t stream, bool pdl);
// Chunks of 64 keys the widest query tile of p sees (the kernel takes <= 8).
int attention_chunks(const AttnParams& p);
// CTAs that share one query tile's key chunks (1 or 2) for a grid of
// base_ctas (tile, head, sequence) CTAs on sm_count SMs.
int attention_split(int base_ctas, int chunks, int sm_count);
cudaError_t launch_norm(const NormParams& p, cudaStream_t stream, bool pdl);
cudaError_t launch_quant_fp8(const QuantParams& p, cudaStream_t stream, bool pdl);
cudaError_t launch_gather_rows(float* dst, const float* src, const int* map, int rows, int d, cudaStream_t stream,
                               bool pdl);
cudaError_t launch_tail(const TailParams& p, int batch, cudaStream_t stream, bool pdl);
cudaError_t launch_token_gather(const TokenGatherParams& p, cudaStream_t stream, bool pdl);
// Adapters beside a projection (lora.cu): the shrink V = s x A^T, which before
// launch_lora_pairs (p.lists given: lora_pair_plan is not 0) also lists the adapters
// of every 256 rows; then the projection that adds V B^T; launched one behind the
// other on one stream.  Tensor maps (128-byte swizzle and boxes of 128 bytes of K
// unless said otherwise):
struct LoraMaps {
  CUtensorMap rows;  // X as bf16, lora_shrink_rows(rows) rows
  CUtensorMap a;     // A [slots][rank][K] bf16, lora_shrink_box(rank) ranks of one slot
  CUtensorMap w;     // weight rows: 128, or bnf / 2
  CUtensorMap x;     // the projection's operand (X, or its codes): bn rows, or 128
  CUtensorMap b;     // B [slots][N][rank] bf16, 32 ranks x 128 (bnf / 2) rows of one slot, 64-byte swizzle
  CUtensorMap v;     // pairs: V as [rows][chunks * 64] bf16, 64 columns x 128 rows
  CUtensorMap out;   // pairs with p.tma_epilogue: output, 128 bytes of columns x 32 rows
};
// projection_ctas, projection_us: the grid and the estimated time of the
// launch_lora_pairs behind it, 0 before launch_lora_gemm.
cudaError_t launch_lora_shrink(const LoraMaps& maps, const LoraParams& p, int sm_count, int projection_ctas,
                               float projection_us, cudaStream_t stream, bool pdl);
// Whether the shrink before launch_lora_gemm takes single dot products, without
// maps.rows and maps.a; a dot product costs as much as 512 columns by itself, and
// tiles waste columns on small ranks.  With the projection into 512 features, dot
// products and tiles: 16 rows, rank 64, K 2,624 7.8 and 12.4 us; 222, 40, 1,504 12.4
// and 14.9; 829, 40, 264 19.7 and 16.8; 64, 32, 12,288 18.4 and 32.5; 64, 16, 40,000
// 74 and 59; 64 rows of rank 256, K 1,024: one adapter 15.2 and 13.1, 64 of them 29
// and 40 (the adapters that the rows name are not known here).
inline bool lora_shrink_by_row(int rows, int rank, int in_features) {
  return (long long)rows * rank * (in_features + 512) <= (rank > 32 ? 20 : 32) << 20;
}
// Rows, and ranks of one adapter, in a CTA of the shrink.
inline int lora_shrink_rows(int rows) { return rows <= 64 ? 64 : 128; }
__host__ __device__ inline int lora_shrink_box(int rank) { return rank < 64 ? (rank + 15) / 16 * 16 : 64; }
// The projection of few rows: row tiles of bn, K split over clusters.
cudaError_t launch_lora_gemm(int kind, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int bn,
                             int split, cudaStream_t stream);
void lora_few_plan(int M, int N, int kblocks, int sm_count, int* bn, int* split);
// The projection of many rows over CTA pairs: tiles of 256 rows x bnf features.
// Without p.tma_epilogue (store epilogue only) the output may lie anywhere.
cudaError_t launch_lora_pairs(int kind, const LoraMaps& maps, const GemmParams& p, const LoraParams& lp, int bnf,
                              cudaStream_t stream);
// CTAs of launch_lora_pairs for these sizes (at most the SMs).
int lora_pair_ctas(int M, int N, int bnf, int sm_count);
// Its time, roughly.
float lora_pair_us(int kind, int M, int N, int kblocks, int bnf, int sm_count);
// Features per tile of launch_lora_pairs, or 0 where launch_lora_gemm is to be used.
int lora_pair_plan(int kind, int M, int N, int K, int rank, int sm_count);
// Status of the launches that were given no status word; reading clears it.
cudaError_t read_op_status(uint32_t* status);
cudaError_t launch_rms_norm(const RmsNormParams& p, cudaStream_t stream, bool pdl);
cudaError_t launch_pack_fp8_rows(const __nv_bfloat16* w, uint8_t* q, float* scale, int rows, int k,
                                 cudaStream_t stream);

}  // namespace laya
