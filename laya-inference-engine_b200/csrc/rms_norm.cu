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
// output is rounded once.  One pass over memory, which is what bounds it.  A
// row of up to 1,024 columns is a warp's (shuffles only), a wider one a CTA's.
#include "common.cuh"
#include "params.h"
#include "launch.h"

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

// TX: x's type; TR: the residual's type (void: none).  VEC: elements of one
// access (8, or 1 where widths, strides or addresses are not multiples of 16
// bytes).  CH: accesses a thread makes.  p.group threads share a row: 32 (a
// warp, several rows a CTA) or the whole CTA.
template <class TX, class TR, int VEC, int CH>
__global__ void __launch_bounds__(VEC == 8 ? 512 : 1024) rms_norm_kernel(const RmsNormParams p) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  constexpr bool kResidual = !std::is_void<TR>::value;
  griddep_launch_dependents();
  griddep_wait();
  const bool wide = p.group > 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = wide ? threadIdx.x : lane;
  const size_t row = wide ? blockIdx.x : (size_t)blockIdx.x * (blockDim.x >> 5) + warp;
  if (row >= (size_t)p.rows) return;  // a whole warp, or nobody
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
  float h[CH][VEC];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (t + i * p.group) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[i][e] = 0.f;
    if (c < p.d) load_row<VEC>(x + c, h[i]);
  }
  if constexpr (kResidual) {
    TR* r = static_cast<TR*>(p.residual) + row * p.ldr;
    float a[CH][VEC];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = (t + i * p.group) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[i][e] = 0.f;
      if (c < p.d) load_row<VEC>(r + c, a[i]);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = (t + i * p.group) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i][e] += a[i][e];
      if (c < p.d) store_row<VEC>(r + c, h[i]);
    }
  }
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
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (t + i * p.group) * VEC;
    if (c >= p.d) continue;
    if (p.w) {
      float w[VEC];
      load_row<VEC>(p.w + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i][e] = h[i][e] * rstd * w[e];
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i][e] *= rstd;
    }
    if (p.y) {
      if (p.y_f32)
        store_row<VEC>(static_cast<float*>(p.y) + row * p.ldy + c, h[i]);
      else
        store_row<VEC>(static_cast<__nv_bfloat16*>(p.y) + row * p.ldy + c, h[i]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) amax = max(amax, __float_as_uint(h[i][e]) & 0x7fffffffu);
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
  uint8_t* q = p.codes + row * p.ldc;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = (t + i * p.group) * VEC;
    if (c >= p.d) continue;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = finite ? div_rn_by(h[i][e], scale, inv) : h[i][e] / scale;
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
  if (t == 0) p.scale[row] = scale;
}

template <class TX, class TR, int VEC>
const void* pick(int ch) {
  if constexpr (VEC == 8)
    return ch <= 1   ? (const void*)rms_norm_kernel<TX, TR, 8, 1>
           : ch <= 2 ? (const void*)rms_norm_kernel<TX, TR, 8, 2>
                     : (const void*)rms_norm_kernel<TX, TR, 8, 4>;
  else
    return ch <= 4   ? (const void*)rms_norm_kernel<TX, TR, 1, 4>
           : ch <= 8 ? (const void*)rms_norm_kernel<TX, TR, 1, 8>
                     : (const void*)rms_norm_kernel<TX, TR, 1, 16>;
}

template <class TX, int VEC>
const void* pick_residual(const RmsNormParams& p, int ch) {
  if (!p.residual) return pick<TX, void, VEC>(ch);
  return p.residual_f32 ? pick<TX, float, VEC>(ch) : pick<TX, __nv_bfloat16, VEC>(ch);
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormParams& params, cudaStream_t stream, bool pdl) {
  RmsNormParams p = params;
  if (p.rows < 1 || p.d < 1 || p.d > kRmsNormMaxColumns) return cudaErrorInvalidValue;
  auto mult = [](const void* ptr, long long ld, int size, int bytes) {
    return !ptr || (reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && ld * size % bytes == 0);
  };
  const bool vec = p.d % 8 == 0 && mult(p.x, p.ldx, p.x_f32 ? 4 : 2, 16) &&
                   mult(p.residual, p.ldr, p.residual_f32 ? 4 : 2, 16) && mult(p.y, p.ldy, p.y_f32 ? 4 : 2, 16) &&
                   mult(p.w, 0, 4, 16) && mult(p.codes, p.ldc, 1, 8);
  const int units = vec ? p.d / 8 : p.d;  // accesses of a row
  int threads, rows_per_cta = 1, ch;
  if (vec && units <= 128) {  // a warp per row
    p.group = 32;
    ch = (units + 31) / 32;
    rows_per_cta = 4;
    threads = 128;
  } else {
    const int want = vec ? 2 : 8;  // accesses a thread should make
    threads = ((units + want - 1) / want + 31) / 32 * 32;
    if (threads < 64) threads = 64;
    if (threads > (vec ? 512 : 1024)) threads = vec ? 512 : 1024;
    p.group = threads;
    ch = (units + threads - 1) / threads;
  }
  const void* fn = p.x_f32 ? (vec ? pick_residual<float, 8>(p, ch) : pick_residual<float, 1>(p, ch))
                           : (vec ? pick_residual<__nv_bfloat16, 8>(p, ch) : pick_residual<__nv_bfloat16, 1>(p, ch));
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
