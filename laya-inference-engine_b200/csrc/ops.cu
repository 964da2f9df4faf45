// Row operators on device buffers that the caller owns (laya_b200_rms_norm,
// laya_b200_lora_linear): argument checks, tensor maps and launches.  Nothing
// here allocates device memory or synchronises, so a call can be captured;
// every check that can fail a launch runs on the host before it.
#include "laya_b200.h"
#include "common.cuh"
#include "launch.h"
#include "params.h"
#include "tensor_map.h"

#include <atomic>
#include <cmath>
#include <string>

namespace laya {
std::string& create_error_message();
}

using namespace laya;

namespace {

int reject(const char* m) {
  create_error_message() = m;
  return 1;
}

int reject(const char* what, cudaError_t err) {
  create_error_message() = std::string(what) + ": " + cudaGetErrorString(err);
  return 1;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// SM count of the current device; 0 with the message set when it is not a
// B200-class GPU.
int sm_count_of_current() {
  constexpr int kMax = 64;
  static std::atomic<int> known[kMax];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return reject("cudaGetDevice", err), 0;
  if (dev >= kMax) return reject("device ordinal out of range"), 0;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n) return n;
  int major = 0;
  err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return reject("cudaDeviceGetAttribute", err), 0;
  if (major != 10) return reject("the operators need an sm_100 GPU"), 0;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

struct LoraPlan {
  int kind, kblocks;
  int bnf;        // features per tile of the pair kernel, or 0:
  int bn, split;  // row tile and K split of the kernel for few rows
  size_t v_bytes, list_bytes;
  size_t bytes() const { return v_bytes + list_bytes; }
};

constexpr int kMaxRows = 1 << 22, kMaxFeatures = 1 << 20;

// Checks the sizes and plans the projection; false with the message set.
bool lora_plan(const laya_b200_lora_args* a, int sm_count, LoraPlan* plan) {
  if (!a) return reject("null arguments"), false;
  if (a->rows < 0 || a->rows > kMaxRows) return reject("rows must be in [0, 4194304]"), false;
  const int kq = a->codes ? 16 : 8;
  if (a->in_features < kq || a->in_features > kMaxFeatures || a->in_features % kq)
    return reject(a->codes ? "in_features must be a positive multiple of 16 with codes"
                           : "in_features must be a positive multiple of 8"),
           false;
  if (a->out_features < 1 || a->out_features > kMaxFeatures) return reject("out_features must be in [1, 1048576]"), false;
  if (a->slots < 1 || a->slots > (1 << 20)) return reject("slots must be in [1, 1048576]"), false;
  if (a->rank < 8 || a->rank > kLoraMaxRank || a->rank % 8)
    return reject("rank must be a multiple of 8 in [8, 256]"), false;
  if (a->rows_per_index < 1) return reject("rows_per_index must be positive"), false;
  plan->kind = a->codes ? kKindFp8 : kKindBf16;
  const int ke = gemm_k_elems(plan->kind);
  plan->kblocks = (a->in_features + ke - 1) / ke;
  const int rows = a->rows > 0 ? a->rows : 1;
  auto align_up = [](size_t x) { return (x + 255) / 256 * 256; };
  plan->v_bytes = align_up((size_t)rows * ((a->rank + 31) / 32) * 128);
  plan->bnf = lora_pair_plan(plan->kind, rows, a->out_features, a->in_features, a->rank, sm_count);
  plan->list_bytes = plan->bnf ? align_up((size_t)((rows + 255) / 256) * kLoraListInts * sizeof(int)) : 0;
  if (!plan->bnf) lora_few_plan(rows, a->out_features, plan->kblocks, sm_count, &plan->bn, &plan->split);
  return true;
}

}  // namespace

extern "C" int laya_b200_rms_norm(const laya_b200_rms_norm_args* a, void* stream) {
  try {
    if (!a) return reject("null arguments");
    if (a->rows < 0 || a->rows > kMaxRows) return reject("rows must be in [0, 4194304]");
    if (a->columns < 1 || a->columns > kRmsNormMaxColumns) return reject("columns must be in [1, 16384]");
    if (!(a->eps > 0.f) || std::isinf(a->eps)) return reject("eps must be positive and finite");
    if (a->rows == 0) return 0;
    if (!a->x) return reject("null x");
    if (!a->y && !a->codes) return reject("neither y nor codes is asked for");
    if (!a->codes != !a->scale) return reject("codes and scale go together");
    if (a->x_stride < a->columns || (a->residual && a->residual_stride < a->columns) ||
        (a->y && a->y_stride < a->columns) || (a->codes && a->codes_stride < a->columns))
      return reject("a row stride is smaller than columns");
    const int sx = a->x_f32 ? 4 : 2, sr = a->residual_f32 ? 4 : 2, sy = a->y_f32 ? 4 : 2;
    if (!aligned(a->x, sx) || !aligned(a->residual, sr) || !aligned(a->y, sy) || !aligned(a->weight, 4) ||
        !aligned(a->scale, 4))
      return reject("a buffer is not aligned to its type");
    if (!sm_count_of_current()) return 1;
    RmsNormParams p{};
    p.rows = a->rows;
    p.d = a->columns;
    p.eps = a->eps;
    p.x = a->x;
    p.ldx = a->x_stride;
    p.x_f32 = a->x_f32;
    p.residual = a->residual;
    p.ldr = a->residual_stride;
    p.residual_f32 = a->residual_f32;
    p.w = a->weight;
    p.y = a->y;
    p.ldy = a->y_stride;
    p.y_f32 = a->y_f32;
    p.codes = static_cast<uint8_t*>(a->codes);
    p.ldc = a->codes_stride;
    p.scale = a->scale;
    const cudaError_t err = launch_rms_norm(p, static_cast<cudaStream_t>(stream), true);
    return err == cudaSuccess ? 0 : reject("RMS norm launch", err);
  } catch (...) {
    return 1;
  }
}

extern "C" int laya_b200_lora_workspace(const laya_b200_lora_args* a, size_t* bytes) {
  try {
    if (!bytes) return reject("null bytes");
    const int sms = sm_count_of_current();
    LoraPlan plan;
    if (!sms || !lora_plan(a, sms, &plan)) return 1;
    *bytes = plan.bytes();
    return 0;
  } catch (...) {
    return 1;
  }
}

extern "C" int laya_b200_lora_linear(const laya_b200_lora_args* a, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  try {
    LoraPlan plan;
    // sizes first: they are refused without a GPU too
    if (!lora_plan(a, 148, &plan)) return 1;
    if (a->rows == 0) return 0;
    if (!a->x || !a->weight || !a->lora_a || !a->lora_b || !a->index || !a->out) return reject("null buffer");
    if (a->codes && (!a->code_scale || !a->weight_scale)) return reject("codes need code_scale and weight_scale");
    const int wsize = a->codes ? 1 : 2;
    if (a->x_stride < a->in_features || a->weight_stride < a->in_features || a->out_stride < a->out_features ||
        (a->codes && a->codes_stride < a->in_features))
      return reject("a row stride is smaller than its row");
    if (a->out_stride > 0x7fffffffll) return reject("out_stride does not fit 32 bits");
    if (!aligned(a->x, 16) || a->x_stride % 8) return reject("x rows must start on 16-byte boundaries");
    if (!aligned(a->weight, 16) || a->weight_stride * wsize % 16)
      return reject("weight rows must start on 16-byte boundaries");
    if (a->codes && (!aligned(a->codes, 16) || a->codes_stride % 16))
      return reject("codes rows must start on 16-byte boundaries");
    if (!aligned(a->lora_a, 16) || !aligned(a->lora_b, 16))
      return reject("lora_a and lora_b must be 16-byte aligned device pointers");
    if (!aligned(a->out, 2) || !aligned(a->bias, 2) || !aligned(a->index, 4) || !aligned(a->scaling, 4) ||
        !aligned(a->code_scale, 4) || !aligned(a->weight_scale, 4))
      return reject("a buffer is not aligned to its type");
    const int sms = sm_count_of_current();
    if (!sms || !lora_plan(a, sms, &plan)) return 1;
    if (!workspace || !aligned(workspace, 256)) return reject("workspace must be a 256-byte aligned device pointer");
    if (workspace_bytes < plan.bytes()) return reject("workspace is too small");
    if (!get_encode_fn()) return reject("cuTensorMapEncodeTiled is unavailable");

    const int M = a->rows, N = a->out_features, K = a->in_features;
    const int chunks = (a->rank + 31) / 32;
    LoraMaps maps{};
    const void* operand = a->codes ? a->codes : a->x;
    const long long ldo = a->codes ? a->codes_stride : a->x_stride;
    const int wbox = plan.bnf ? plan.bnf / 2 : 128;
    // rows of the output that take TMA stores, which write whole 16 bytes: those of a
    // width that ends inside one would go over the columns behind it
    const bool tma_out = plan.bnf && aligned(a->out, 16) && a->out_stride % 8 == 0 && N % 8 == 0;
    bool ok = ((!plan.bnf && lora_shrink_by_row(M, a->rank, K)) ||
               (rows_map(&maps.rows, a->x, M, K, a->x_stride, 2, lora_shrink_rows(M)) &&
                slots_map(&maps.a, a->lora_a, a->slots, a->rank, K, 64, lora_shrink_box(a->rank),
                          CU_TENSOR_MAP_SWIZZLE_128B))) &&
              rows_map(&maps.w, a->weight, N, K, a->weight_stride, wsize, wbox) &&
              rows_map(&maps.x, operand, M, K, ldo, wsize, plan.bnf ? 128 : plan.bn) &&
              (!plan.bnf ||
               (slots_map(&maps.b, a->lora_b, a->slots, N, a->rank, 32, wbox, CU_TENSOR_MAP_SWIZZLE_64B) &&
                rows_map(&maps.v, workspace, M, chunks * 64, chunks * 64, 2, 128))) &&
              (!tma_out || rows_map(&maps.out, a->out, M, N, a->out_stride, 2, 32));
    if (!ok) return reject("a tensor map was rejected");
    LoraParams lp{};
    lp.rows = M;
    lp.out_features = a->out_features;
    lp.in_features = K;
    lp.slots = a->slots;
    lp.rank = a->rank;
    lp.chunks = chunks;
    lp.index = a->index;
    lp.index_div = a->rows_per_index;
    lp.x = static_cast<const __nv_bfloat16*>(a->x);
    lp.ldx = a->x_stride;
    lp.a = static_cast<const __nv_bfloat16*>(a->lora_a);
    lp.b = static_cast<const __nv_bfloat16*>(a->lora_b);
    lp.scaling = a->scaling;
    lp.v = static_cast<__nv_bfloat16*>(workspace);
    GemmParams p{};
    p.M = M;
    p.N = N;
    p.K = K;
    p.kblocks = plan.kblocks;
    p.epilogue = kEpiStore;
    p.tma_epilogue = tma_out;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.ldo = (int)a->out_stride;
    p.bias = static_cast<const __nv_bfloat16*>(a->bias);
    p.a_scale = a->code_scale;
    p.w_scale = a->weight_scale;
    if (plan.bnf) lp.lists = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + plan.v_bytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t err = launch_lora_shrink(
        maps, lp, sms, plan.bnf ? lora_pair_ctas(M, N, plan.bnf, sms) : 0,
        plan.bnf ? lora_pair_us(plan.kind, M, N, plan.kblocks, plan.bnf, sms) : 0.f, st, true);
    if (err != cudaSuccess) return reject("adapter shrink launch", err);
    err = plan.bnf ? launch_lora_pairs(plan.kind, maps, p, lp, plan.bnf, st)
                   : launch_lora_gemm(plan.kind, maps, p, lp, plan.bn, plan.split, st);
    return err == cudaSuccess ? 0 : reject("adapter projection launch", err);
  } catch (...) {
    return 1;
  }
}

extern "C" int laya_b200_op_status(int32_t* status) {
  try {
    if (!status) return reject("null status");
    if (!sm_count_of_current()) return 1;
    uint32_t v = 0;
    const cudaError_t err = read_op_status(&v);
    if (err != cudaSuccess) return reject("operator status", err);
    *status = (int32_t)v;
    return 0;
  } catch (...) {
    return 1;
  }
}
