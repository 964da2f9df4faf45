// RMS norm rows with the residual's addition and e4m3 output
// (laya_b200_rms_norm): the sibling of the LayerNorm rows in norm_row.cuh for
// blocks that a host runs on its own buffers.
//
//   h = x + residual            (fp32; stored back rounded to the residual's type)
//   y = h * rsqrt(mean(h^2) + eps) * w
//   scale = max(max|y| * fl(1/448), 1e-12), codes = e4m3(y / scale)   per row
//
// Everything between the loads and the stores stays in fp32 registers: the
// norm reads the unrounded sum and the quantiser the unrounded y, so each
// output is rounded once.  One pass over memory, which is what bounds it: a row's
// elements stay in the registers of a warp (short rows, shuffles only) or of a CTA.
// Measured in replayed graphs against bytes / 6,556 GB/s (a copy's rate): 32,768 rows
// of 1,024 with an fp32 residual and codes 61 us (92 %; 58 in a short burst, before
// the power limit lowers the clock), 16,384 of 4,096 in bf16 83 to 86 (95 to 99 %),
// 4,000 of 8,191 71 (84 %), 14,427 of 435 14.9 (77 %).  Rows with little to load for
// what they compute are bound by the chain load - sum - weight - maximum - store of
// the rows in flight: 32,768 bf16 rows of 1,024 without a residual 26 us (78 %), to
// codes alone 35 (44 %).  The comparisons of two forms below are of short bursts.
#include "common.cuh"
#include "params.h"
#include "launch.h"

#include <algorithm>
#include <type_traits>

namespace laya {

namespace {

// VEC consecutive elements of type T at p, widened to fp32.
template <int VEC>
DEVI void load_row(const float* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    v[0] = p[0];
  }
}
template <int VEC>
DEVI void load_row(const __nv_bfloat16* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(e[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    v[0] = __bfloat162float(p[0]);
  }
}
template <int VEC>
DEVI void store_row(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    p[0] = v[0];
  }
}
template <int VEC>
DEVI void store_row(__nv_bfloat16* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    uint4 u;
    __nv_bfloat162* e = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
    p[0] = __float2bfloat16_rn(v[0]);
  }
}

// Largest of non-negative floats by their bit patterns, which order like the
// values and put every NaN above infinity: a NaN in a row is not lost.
DEVI uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// Eight weights c.. by the aligned quads that hold them (c need not be a multiple
// of four): a lane's single elements would lie 32 bytes from the next lane's,
// eight lines an access.
DEVI void load_weight_shifted(const float* w, int c, int d, float (&v)[8]) {
  const int r = c & 3, a = c - r;
  const float4* p = reinterpret_cast<const float4*>(w + a);
  const float4 f0 = __ldg(p), f1 = __ldg(p + 1);
  float4 f2 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a + 12 <= d) {
    f2 = __ldg(p + 2);
  } else {  // the row's last columns: as many as the group has of them
    if (r > 0) f2.x = __ldg(w + a + 8);
    if (r > 1) f2.y = __ldg(w + a + 9);
    if (r > 2) f2.z = __ldg(w + a + 10);
  }
  float q[12] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w, f2.x, f2.y, f2.z, f2.w};
#pragma unroll
  for (int e = 0; e < 11; ++e) q[e] = r & 1 ? q[e + 1] : q[e];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = r & 2 ? q[e + 2] : q[e];
}

// TX: x's type; TR: the residual's type (void: none).  VEC: elements of one
// access, 8, or 1 where the buffers' rows have nothing in common.  CH: accesses a
// thread makes.  SHIFT: the rows of all buffers start p.shift + row * p.shift_step
// elements (modulo 8) behind 16-byte boundaries (odd widths): accesses are of the
// groups of eight between those boundaries, and the up to seven columns before
// and after them are single elements of the row's first 16 threads.  (Groups with
// bounds per element at the two ends cost 700 instructions a row: 14,427 rows of
// 435 columns took 15.7 us that way.)  p.group threads share a row: a warp, or the
// whole CTA.
template <class TX, class TR, int VEC, int CH, bool SHIFT>
__global__ void __launch_bounds__(VEC == 8 ? 512 : 1024) rms_norm_kernel(const RmsNormParams p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  constexpr bool kResidual = !std::is_void<TR>::value;
  griddep_launch_dependents();
  const bool wide = p.group > 32;  // the CTA has one row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = wide ? threadIdx.x : lane;
  const size_t row = wide ? blockIdx.x : (size_t)blockIdx.x * (blockDim.x >> 5) + warp;
  if (row >= (size_t)p.rows) {  // a whole warp, or nobody
    griddep_wait();
    return;
  }
  // columns [first, last) are accessed VEC at a time, column `one` by itself
  const int first = SHIFT ? (int)(-(p.shift + (long long)row * p.shift_step) & 7) : 0;
  const int last = SHIFT ? p.d - ((p.d - first) & 7) : p.d;
  int one = t < 8 ? t : last + t - 8;
  if (!SHIFT || (t < 8 ? t >= first : t >= 16 || one >= p.d)) one = -1;
  auto column = [&](int i) { return first + (t + i * p.group) * VEC; };
  griddep_wait();
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
  float h[CH][VEC], h1[1] = {0.f};
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = column(i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[i][e] = 0.f;
    if (c < last) load_row<VEC>(x + c, h[i]);
  }
  if (one >= 0) load_row<1>(x + one, h1);
  if constexpr (kResidual) {
    TR* r = static_cast<TR*>(p.residual) + row * p.ldr;
    float a[CH][VEC], a1[1] = {0.f};
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = column(i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[i][e] = 0.f;
      if (c < last) load_row<VEC>(r + c, a[i]);
    }
    if (one >= 0) load_row<1>(r + one, a1);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = column(i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i][e] += a[i][e];
      if (c < last) store_row<VEC>(r + c, h[i]);
    }
    h1[0] += a1[0];
    if (one >= 0) store_row<1>(r + one, h1);
  }
  auto load_weight = [&](int c, float (&w)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = 1.f;
    if (!p.w || c >= last) return;
    if constexpr (SHIFT) load_weight_shifted(p.w, c, p.d, w);
    else load_row<VEC>(p.w + c, w);
  };
  // one access a thread (few rows, where latency counts): the weight comes with
  // it; else after the sum, which leaves registers for more rows in flight
  float w0[VEC], w1 = 1.f;
  if (CH == 1) load_weight(column(0), w0);
  if (one >= 0 && p.w) w1 = __ldg(p.w + one);
  float sum = h1[0] * h1[0];
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += h[i][e] * h[i][e];
  sum = warp_sum(sum);
  if (wide) {
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) sum += s_sum[i];
  }
  const float rstd = rsqrtf(sum / (float)p.d + p.eps);
  h1[0] = h1[0] * rstd * w1;
  uint32_t amax = __float_as_uint(h1[0]) & 0x7fffffffu;
  if (!SHIFT || one < 0) amax = 0;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = column(i);
    if (c >= last) continue;
    if (CH > 1) load_weight(c, w0);
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[i][e] = h[i][e] * rstd * w0[e];
    if (p.y) {
      if (p.y_f32)
        store_row<VEC>(static_cast<float*>(p.y) + row * p.ldy + c, h[i]);
      else
        store_row<VEC>(static_cast<__nv_bfloat16*>(p.y) + row * p.ldy + c, h[i]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) amax = max(amax, __float_as_uint(h[i][e]) & 0x7fffffffu);
  }
  if (p.y && one >= 0) {
    if (p.y_f32)
      store_row<1>(static_cast<float*>(p.y) + row * p.ldy + one, h1);
    else
      store_row<1>(static_cast<__nv_bfloat16*>(p.y) + row * p.ldy + one, h1);
  }
  if (!p.codes) return;
  amax = warp_umax(amax);
  if (wide) {
    if (lane == 0) s_max[warp] = amax;
    __syncthreads();
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) amax = max(amax, s_max[i]);
  }
  // A row with a NaN has a NaN scale, one with an infinity an infinite scale
  // (its finite values become 0, the infinity NaN, as the quotients are).
  float scale = __uint_as_float(amax) * kInvE4m3Max;
  if (scale < 1e-12f) scale = 1e-12f;
  const bool finite = amax < 0x7f800000u;
  const float inv = 1.0f / scale;
  auto quotient = [&](float y) { return finite ? div_rn_by(y, scale, inv) : y / scale; };
  uint8_t* q = p.codes + row * p.ldc;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = column(i);
    if (c >= last) continue;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = quotient(h[i][e]);
    if constexpr (VEC == 8) {
      uint32_t o[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = (uint32_t)f32x2_to_e4m3x2(v[4 * j], v[4 * j + 1]) |
               ((uint32_t)f32x2_to_e4m3x2(v[4 * j + 2], v[4 * j + 3]) << 16);
      *reinterpret_cast<uint2*>(q + c) = make_uint2(o[0], o[1]);
    } else {
      q[c] = (uint8_t)(f32x2_to_e4m3x2(v[0], 0.f) & 0xFF);
    }
  }
  if (one >= 0) q[one] = (uint8_t)(f32x2_to_e4m3x2(quotient(h1[0]), 0.f) & 0xFF);
  if (t == 0) p.scale[row] = scale;
}

enum RowAccess { kVector, kShifted, kElement };

template <class TX, class TR>
const void* pick(RowAccess access, int ch) {
  if (access == kVector)
    return ch <= 1   ? (const void*)rms_norm_kernel<TX, TR, 8, 1, false>
           : ch <= 2 ? (const void*)rms_norm_kernel<TX, TR, 8, 2, false>
                     : (const void*)rms_norm_kernel<TX, TR, 8, 4, false>;
  if (access == kShifted)
    return ch <= 1   ? (const void*)rms_norm_kernel<TX, TR, 8, 1, true>
           : ch <= 2 ? (const void*)rms_norm_kernel<TX, TR, 8, 2, true>
                     : (const void*)rms_norm_kernel<TX, TR, 8, 4, true>;
  return ch <= 4   ? (const void*)rms_norm_kernel<TX, TR, 1, 4, false>
         : ch <= 8 ? (const void*)rms_norm_kernel<TX, TR, 1, 8, false>
                   : (const void*)rms_norm_kernel<TX, TR, 1, 16, false>;
}

template <class TX>
const void* pick_residual(const RmsNormParams& p, RowAccess access, int ch) {
  if (!p.residual) return pick<TX, void>(access, ch);
  return p.residual_f32 ? pick<TX, float>(access, ch) : pick<TX, __nv_bfloat16>(access, ch);
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormParams& params, cudaStream_t stream, bool pdl) {
  RmsNormParams p = params;
  if (p.rows < 1 || p.d < 1 || p.d > kRmsNormMaxColumns) return cudaErrorInvalidValue;
  // How the buffers' rows lie against groups of eight elements: all on them
  // (vector), all the same distance behind them in every row (shifted), or not
  // alike (element by element).
  p.shift = (int)(reinterpret_cast<uintptr_t>(p.x) / (p.x_f32 ? 4 : 2) & 7);
  p.shift_step = (int)(p.ldx & 7);
  bool alike = true;
  auto same = [&](const void* ptr, long long ld, int size) {
    if (ptr && ((int)(reinterpret_cast<uintptr_t>(ptr) / size & 7) != p.shift || (int)(ld & 7) != p.shift_step))
      alike = false;
  };
  same(p.residual, p.ldr, p.residual_f32 ? 4 : 2);
  same(p.y, p.ldy, p.y_f32 ? 4 : 2);
  same(p.codes, p.ldc, 1);
  const bool weight_on = (reinterpret_cast<uintptr_t>(p.w) & 15) == 0;
  const bool on = p.shift == 0 && (p.shift_step == 0 || p.rows == 1) && p.d % 8 == 0;
  const RowAccess access = !alike || !weight_on ? kElement : on ? kVector : p.d >= 16 ? kShifted : kElement;
  // accesses of a row
  const int units = access == kElement ? p.d : p.d / 8;
  auto warps_of = [](int threads) { return (threads + 31) / 32 * 32; };
  // threads of a row, accesses of a thread
  int group, ch;
  if (access == kElement) {
    group = std::min(1024, warps_of((units + 7) / 8));
  } else if (p.rows * warps_of(units) <= 148 * 2048 && units <= 512) {
    group = warps_of(units);  // few rows: every access can be resident at once, one a thread
  } else {
    // Accesses of a thread.  Four: rows of two bytes a column, whose two would
    // leave too few bytes in flight (32,768 rows of 1,024 bf16: 26 us, two 36), and
    // wide rows, whose CTA is the smaller for it (8,000 rows of 8,192 with an fp32
    // residual 138 us, two 146).  Two: the rest (32,768 rows of 1,024 with an fp32
    // residual 58 us, four 63).
    const int want = (!p.residual && !p.x_f32) || (access == kVector && units >= 512) ? 4 : 2;
    group = units <= 32 * want ? 32 : std::min(512, warps_of((units + want - 1) / want));
  }
  ch = (units + group - 1) / group;
  p.group = group;
  // Eight rows of a warp each share a CTA (a CTA for every row of 1,024 columns,
  // bf16 without a residual: 36 us for 32,768 rows, launching CTAs).
  const int rows_per_cta = group > 32 ? 1 : (int)std::min<long long>(8, p.rows);
  const int threads = rows_per_cta * group;
  const void* fn = p.x_f32 ? pick_residual<float>(p, access, ch) : pick_residual<__nv_bfloat16>(p, access, ch);
  void* args[] = {&p};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.rows + rows_per_cta - 1) / rows_per_cta), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace laya
