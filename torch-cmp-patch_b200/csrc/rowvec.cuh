// rowvec.cuh -- short vectors of fp16 / bf16 / fp32 values moved as one load or store and computed
// on in fp32, and the division by a page size that paged kernels do per token.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/cmpx_b200.h"
#include "cmpx_ptx.cuh"

namespace cmpx {

constexpr int elt_size(int dt) { return dt == CMPX_F32 ? 4 : 2; }

template <int BYTES>
struct RawVec;
template <>
struct RawVec<16> {
  uint4 v;
};
template <>
struct RawVec<8> {
  uint2 v;
};
template <>
struct RawVec<4> {
  uint32_t v;
};
template <>
struct RawVec<2> {
  unsigned short v;
};

// The 16-bit pair in one register as two floats (low half first).
template <int DT>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if (DT == CMPX_BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

template <int DT, int BYTES>
__device__ __forceinline__ void unpack_vec(const RawVec<BYTES>& r, float* f) {
  if constexpr (BYTES == 2) {
    if (DT == CMPX_BF16) {
      f[0] = __uint_as_float(static_cast<uint32_t>(r.v) << 16);
    } else {
      __half_raw h;
      h.x = r.v;
      f[0] = __half2float(__half(h));
    }
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r.v);
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) {
      if (DT == CMPX_F32)
        f[i] = __uint_as_float(w[i]);
      else
        unpack2<DT>(w[i], f[2 * i], f[2 * i + 1]);
    }
  }
}

template <int DT, int BYTES>
__device__ __forceinline__ RawVec<BYTES> pack_vec(const float* f) {
  RawVec<BYTES> r;
  if constexpr (BYTES == 2) {
    r.v = DT == CMPX_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[0])) : __half_as_ushort(__float2half_rn(f[0]));
  } else {
    uint32_t w[BYTES / 4];
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i)
      w[i] = DT == CMPX_F32    ? __float_as_uint(f[i])
             : DT == CMPX_BF16 ? pack_bf16x2(f[2 * i], f[2 * i + 1])
                               : pack_f16x2(f[2 * i], f[2 * i + 1]);
    if constexpr (BYTES == 4) r.v = w[0];
    if constexpr (BYTES == 8) r.v = make_uint2(w[0], w[1]);
    if constexpr (BYTES == 16) r.v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

// Whole quotients t / d of 0 <= t < 2^31 by a fixed d: with p = 31 + ceil(log2 d) and
// m = ceil(2^p / d), m d - 2^p < d <= 2^(p - 31), so (t m) >> p is exact; m <= 2^32 - 1 for d > 1.
struct FastDiv {
  uint32_t d, m;
  int p;
};

inline FastDiv make_fast_div(uint32_t d) {
  int log2 = 0;
  while ((1ull << log2) < d) ++log2;
  const int p = 31 + log2;
  return FastDiv{d, static_cast<uint32_t>(((1ull << p) + d - 1) / d), p};
}

__device__ __forceinline__ uint32_t fast_div(uint32_t t, const FastDiv& f) {
  return static_cast<uint32_t>((static_cast<uint64_t>(t) * f.m) >> f.p);
}

}  // namespace cmpx
