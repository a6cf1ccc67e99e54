// linear_w4.cu -- linear layer with 4-bit weights and group scales for a few tokens, B200 sm_100a.
//
//   y[m, n] = sum_g scale[n, g] * sum_{k in group g} (code[n, k] - zero[n, g]) x[m, k]  (+ bias[n])
//
// code - zero is a whole number of at most 4 bits and a sign, exact in fp16 and bf16; the sums are
// fp32 and the scale multiplies a group's sum, so no weight is ever rounded.  The weights are read once:
// n k / 2 bytes bound it while the tokens are few.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "cmpx_internal.h"
#include "rowvec.cuh"

namespace cmpx {
namespace {

constexpr int kWarps = 8;
constexpr int kTokens = 8;  // tokens per pass over the weights

struct W4Args {
  const uint8_t* x;
  const uint8_t* w;
  const uint8_t* scales;
  const uint8_t* zeros;
  const uint8_t* bias;
  uint8_t* y;
  int64_t xs, ws, ss, zs, ys;  // row strides in bytes
  int m, n, k, group;
};

// One warp per row of W; a lane takes 8 codes (one word) at a time.
template <int DT>
__global__ void __launch_bounds__(kWarps * 32) linear_w4_kernel(const __grid_constant__ W4Args a) {
  constexpr int ES = elt_size(DT);
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (n >= a.n) return;
  const int m0 = blockIdx.y * kTokens, mn = min(kTokens, a.m - m0);
  float acc[kTokens];
#pragma unroll
  for (int t = 0; t < kTokens; ++t) acc[t] = 0.f;
  for (int i = lane; i < a.k / 8; i += 32) {
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(a.w + n * a.ws) + i);
    const int g = i * 8 / a.group;
    float scale;
    unpack_vec<DT, ES>(*reinterpret_cast<const RawVec<ES>*>(a.scales + n * a.ss + g * ES), &scale);
    const float zero = a.zeros ? static_cast<float>(__ldg(a.zeros + n * a.zs + g)) : 8.f;
    float c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = static_cast<float>((word >> (4 * e)) & 15u) - zero;
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      if (t >= mn) break;
      const uint8_t* p = a.x + (m0 + t) * a.xs + static_cast<int64_t>(i) * 8 * ES;
      float x[8];
      if constexpr (ES == 4) {
        unpack_vec<DT, 16>(*reinterpret_cast<const RawVec<16>*>(p), x);
        unpack_vec<DT, 16>(*reinterpret_cast<const RawVec<16>*>(p + 16), x + 4);
      } else {
        unpack_vec<DT, 16>(*reinterpret_cast<const RawVec<16>*>(p), x);
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(c[e], x[e], s);
      acc[t] = fmaf(scale, s, acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    if (t >= mn) break;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], off);
    if (lane == 0) {
      float r = acc[t];
      if (a.bias) {
        float b;
        unpack_vec<DT, ES>(*reinterpret_cast<const RawVec<ES>*>(a.bias + n * ES), &b);
        r += b;
      }
      *reinterpret_cast<RawVec<ES>*>(a.y + (m0 + t) * a.ys + n * ES) = pack_vec<DT, ES>(&r);
    }
  }
}

}  // namespace

const char* linear_w4_plan(const cmpx_linear_w4_desc* d, int* status) {
  *status = CMPX_ERR_INVALID_ARGUMENT;
  if (!d || !d->x || !d->w || !d->scales || !d->y || d->m < 0 || d->n < 0 || d->k <= 0 || d->group <= 0) return "none";
  if (d->k % d->group != 0) return "none";
  *status = CMPX_ERR_UNSUPPORTED_DTYPE;
  if (d->dtype != CMPX_F32 && d->dtype != CMPX_F16 && d->dtype != CMPX_BF16) return "none";
  const int64_t es = elt_size(d->dtype);
  *status = CMPX_ERR_UNSUPPORTED_SHAPE;
  if (d->group % 32 != 0 || d->k > (1 << 24) || d->n > (1ll << 31) - 65536 || d->m > 65535 * kTokens) return "none";
  if (d->x_row_stride < 0 || d->w_row_stride < 0 || d->scales_row_stride < 0 || d->zeros_row_stride < 0 ||
      d->y_row_stride < d->n)
    return "none";
  *status = CMPX_ERR_MISALIGNED;
  if (reinterpret_cast<uintptr_t>(d->x) % 16 || reinterpret_cast<uintptr_t>(d->w) % 16 ||
      (d->m > 1 && (d->x_row_stride * es) % 16) || (d->n > 1 && d->w_row_stride % 16))
    return "none";
  *status = CMPX_OK;
  return "linear_w4<warp per row>";
}

int launch_linear_w4(const cmpx_linear_w4_desc* d, const LaunchCtx& ctx) {
  const int es = elt_size(d->dtype);
  W4Args a{};
  a.x = static_cast<const uint8_t*>(d->x);
  a.w = d->w;
  a.scales = static_cast<const uint8_t*>(d->scales);
  a.zeros = d->zeros;
  a.bias = static_cast<const uint8_t*>(d->bias);
  a.y = static_cast<uint8_t*>(d->y);
  a.xs = d->x_row_stride * es;
  a.ws = d->w_row_stride;
  a.ss = d->scales_row_stride * es;
  a.zs = d->zeros_row_stride;
  a.ys = d->y_row_stride * es;
  a.m = static_cast<int>(d->m);
  a.n = static_cast<int>(d->n);
  a.k = static_cast<int>(d->k);
  a.group = static_cast<int>(d->group);
  const dim3 grid(static_cast<unsigned>((d->n + kWarps - 1) / kWarps),
                  static_cast<unsigned>((d->m + kTokens - 1) / kTokens));
  if (d->dtype == CMPX_F32) linear_w4_kernel<CMPX_F32><<<grid, kWarps * 32, 0, ctx.stream>>>(a);
  else if (d->dtype == CMPX_F16) linear_w4_kernel<CMPX_F16><<<grid, kWarps * 32, 0, ctx.stream>>>(a);
  else linear_w4_kernel<CMPX_BF16><<<grid, kWarps * 32, 0, ctx.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

}  // namespace cmpx
