// linear_w4.cu -- linear layer with 4-bit weights and group scales for a few tokens, B200 sm_100a.
//
//   y[m, n] = sum_g scale[n, g] * sum_{k in group g} (code[n, k] - zero[n, g]) x[m, k]  (+ bias[n])
//
// code - zero is a whole number of at most 4 bits and a sign, exact in fp16 and bf16; the sums are
// fp32 and the scale multiplies a group's fp32 sum, so no weight is ever rounded.  fp32 activations
// go in as three bf16 parts (the leading, next and last 8 bits of the fraction: an exact sum), three
// products each.
//
// The weights are read once, n k / 2 bytes, and that read bounds it while the tokens are few.  A CTA has 16
// rows of W, its warps take turns at chunks of 128 k, and mma.m16n8k16 multiplies the 16 rows with up to
// 8 NT tokens.  A lane loads 8 bytes of a row, 16 k that lie side by side (a quad: one 32-byte sector),
// and the products run over k in the order that falls out of it: word j of the lanes tq = 0..3 holds k =
// 16 tq + 8 j .. + 7, and nibbles e and e + 4 of a word, which one mask isolates as the halves of a
// register, are a pair.  x follows that order with one byte permutation a register.  Chunks are loaded DEPTH ahead
// into registers.  What it costs beside the loads is instructions: for eight weights 3 shifts, 4 masks, 4
// subtractions (fp16: 1, 4, 4).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "cmpx_internal.h"
#include "rowvec.cuh"

namespace cmpx {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;    // rows of W per CTA
constexpr int kChunk = 128;  // k per warp and turn

struct W4Args {
  const uint8_t* x;
  const uint8_t* w;
  const uint8_t* scales;
  const uint8_t* zeros;
  const uint8_t* bias;
  uint8_t* y;
  int64_t xs, ws, ss, zs, ys;  // row strides in bytes
  int m, n, k;
  FastDiv group;
};

// Where the groups end: at every chunk's end or rarer, inside it at 64 k, or at 32 k.
enum GroupKind { kGroup128 = 0, kGroup64 = 1, kGroup32 = 2 };

__device__ __forceinline__ uint2 load_w(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <int DT>
__device__ __forceinline__ void mma_w4(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if constexpr (DT == CMPX_F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The eight codes of a word minus a zero point as four 16-bit pairs: pair e = codes e and e + 4.  A code
// placed under the exponent of 128 (bf16) or 1024 (fp16) is that number plus the code; zp holds the number
// plus the zero point, twice.  fp16 has room for a nibble four bits higher, which saves shifts: 1024 + 16 c
// times 1/16 minus (64 + zero), one exact fma (zp16).
template <int DT>
struct Zero {
  uint32_t zp, zp16;
  __device__ __forceinline__ explicit Zero(uint32_t z) {
    if constexpr (DT == CMPX_F16) {
      zp = (0x6400u + z) * 0x10001u;
      const __half2 v = __float2half2_rn(-64.f - static_cast<float>(z));
      zp16 = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      zp = (0x4300u + z) * 0x10001u;
      zp16 = 0;
    }
  }
};

template <int DT>
__device__ __forceinline__ void codes_minus_zero(uint32_t w, const Zero<DT>& z, uint32_t (&out)[4]) {
  if constexpr (DT == CMPX_F16) {
    const uint32_t v = w >> 8;
    const uint32_t c[4] = {(w & 0x000F000Fu) | 0x64006400u, (w & 0x00F000F0u) | 0x64006400u,
                           (v & 0x000F000Fu) | 0x64006400u, (v & 0x00F000F0u) | 0x64006400u};
    const __half2 zp = *reinterpret_cast<const __half2*>(&z.zp), zp16 = *reinterpret_cast<const __half2*>(&z.zp16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 h = *reinterpret_cast<const __half2*>(&c[e]);
      const __half2 d = e & 1 ? __hfma2(h, __half2half2(__ushort_as_half(0x2C00)), zp16) : __hsub2(h, zp);
      out[e] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {
    const __nv_bfloat162 zp = *reinterpret_cast<const __nv_bfloat162*>(&z.zp);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t c = ((w >> (4 * e)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), zp);
      out[e] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

// 8 activations as PARTS sets of four pairs (e, e + 4).
template <int DT>
struct XParts {
  static constexpr int PARTS = DT == CMPX_F32 ? 3 : 1;
  uint32_t p[PARTS][4];
};

template <int DT>
__device__ __forceinline__ XParts<DT> load_x(const uint8_t* p, bool there) {
  XParts<DT> r;
  if constexpr (DT == CMPX_F32) {
    uint4 u = make_uint4(0, 0, 0, 0), v = u;
    if (there) {
      u = __ldg(reinterpret_cast<const uint4*>(p));
      v = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    }
    const uint32_t x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    uint32_t part[8][3];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = __uint_as_float(x[e]);
      const bool finite = fabsf(f) <= 3.402823466e38f;
      // cut off, not rounded, so that the largest values do not become infinite; NaN stays NaN
      part[e][0] = finite ? x[e] & 0xFFFF0000u : f != f ? 0x7FC00000u : x[e];
      const float rest = finite ? f - __uint_as_float(part[e][0]) : 0.f;
      part[e][1] = __float_as_uint(rest) & 0xFFFF0000u;
      part[e][2] = __float_as_uint(rest - __uint_as_float(part[e][1]));
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) r.p[i][e] = __byte_perm(part[e][i], part[e + 4][i], 0x7632);
  } else {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (there) u = __ldg(reinterpret_cast<const uint4*>(p));
    r.p[0][0] = __byte_perm(u.x, u.z, 0x5410);
    r.p[0][1] = __byte_perm(u.x, u.z, 0x7632);
    r.p[0][2] = __byte_perm(u.y, u.w, 0x5410);
    r.p[0][3] = __byte_perm(u.y, u.w, 0x7632);
  }
  return r;
}

template <int DT, int NT, int GK>
__global__ void __launch_bounds__(kThreads) linear_w4_kernel(const __grid_constant__ W4Args a) {
  constexpr int ES = elt_size(DT);
  constexpr int GROUPS = GK == kGroup128 ? 1 : GK == kGroup64 ? 2 : 4;  // scales per row and chunk
  constexpr int DEPTH = GK == kGroup128 ? 4 : GK == kGroup64 ? 3 : 2;
  __shared__ float red[kWarps][NT * 8][kRows + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * (8 * NT);
  // rows behind the last read the last one; their results are not written
  const int row[2] = {min(n0 + gr, a.n - 1), min(n0 + gr + 8, a.n - 1)};
  const uint8_t* wp[2] = {a.w + row[0] * a.ws + tq * 8, a.w + row[1] * a.ws + tq * 8};
  const uint8_t* sp[2] = {a.scales + row[0] * a.ss, a.scales + row[1] * a.ss};
  const uint8_t* zp[2] = {a.zeros + row[0] * a.zs, a.zeros + row[1] * a.zs};
  const int chunks = (a.k + kChunk - 1) / kChunk;

  struct Chunk {
    uint2 w[2][2];             // [half of the chunk][row]
    RawVec<ES> s[GROUPS][2];   // [group][row]
    uint32_t z[GROUPS][2];
  };
  auto fetch = [&](int c, Chunk& q) {
    if (c >= chunks) return;
    const int k0 = c * kChunk;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool there = k0 + h * 64 + tq * 16 < a.k;
#pragma unroll
      for (int r = 0; r < 2; ++r) q.w[h][r] = there ? load_w(wp[r] + (k0 >> 1) + h * 32) : make_uint2(0, 0);
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int at = fast_div(min(k0 + g * (kChunk / GROUPS), a.k - 1), a.group);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        q.s[g][r] = *reinterpret_cast<const RawVec<ES>*>(sp[r] + at * ES);
        q.z[g][r] = a.zeros ? __ldg(zp[r] + at) : 8u;
      }
    }
  };

  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;

  auto compute = [&](int c, const Chunk& q) {
    const int k0 = c * kChunk;
    float part[GK == kGroup32 ? 2 : 1][NT][4];
    auto clear = [&] {
#pragma unroll
      for (int i = 0; i < (GK == kGroup32 ? 2 : 1); ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[i][t][e] = 0.f;
    };
    auto add = [&](int i, int g) {  // acc += scale[g] * part[i]
      float s[2];
      unpack_vec<DT, ES>(q.s[g][0], &s[0]);
      unpack_vec<DT, ES>(q.s[g][1], &s[1]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(s[e >> 1], part[i][t][e], acc[t][e]);
    };
    clear();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + h * 64 + tq * 16;
      // this lane's 16 k lie in one group
      const int g = GK == kGroup128 ? 0 : GK == kGroup64 ? h : 0;
      uint32_t z0, z1;
      if (GK == kGroup32) {
        z0 = tq < 2 ? q.z[(2 * h) % GROUPS][0] : q.z[(2 * h + 1) % GROUPS][0];
        z1 = tq < 2 ? q.z[(2 * h) % GROUPS][1] : q.z[(2 * h + 1) % GROUPS][1];
      } else {
        z0 = q.z[g][0];
        z1 = q.z[g][1];
      }
      const Zero<DT> zero0(z0), zero1(z1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t d0[4], d1[4];
        codes_minus_zero<DT>(j ? q.w[h][0].y : q.w[h][0].x, zero0, d0);
        codes_minus_zero<DT>(j ? q.w[h][1].y : q.w[h][1].x, zero1, d1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int m = m0 + t * 8 + gr;
          const XParts<DT> x = load_x<DT>(a.x + m * a.xs + (k + 8 * j) * ES, m < a.m && k < a.k);
#pragma unroll
          for (int i = 0; i < XParts<DT>::PARTS; ++i) {
            const uint32_t* p = x.p[i];
            if constexpr (GK == kGroup32) {
              // the quad's first two lanes are in one group, its last two in the next
              const bool one = tq < 2;
              mma_w4<DT>(part[0][t], d0[0], d1[0], d0[1], d1[1], one ? p[0] : 0, one ? p[1] : 0);
              mma_w4<DT>(part[0][t], d0[2], d1[2], d0[3], d1[3], one ? p[2] : 0, one ? p[3] : 0);
              mma_w4<DT>(part[1][t], d0[0], d1[0], d0[1], d1[1], one ? 0 : p[0], one ? 0 : p[1]);
              mma_w4<DT>(part[1][t], d0[2], d1[2], d0[3], d1[3], one ? 0 : p[2], one ? 0 : p[3]);
            } else {
              mma_w4<DT>(part[0][t], d0[0], d1[0], d0[1], d1[1], p[0], p[1]);
              mma_w4<DT>(part[0][t], d0[2], d1[2], d0[3], d1[3], p[2], p[3]);
            }
          }
        }
      }
      if (GK == kGroup64) {
        add(0, h);
        clear();
      } else if (GK == kGroup32) {
        add(0, (2 * h) % GROUPS);
        add(GK == kGroup32 ? 1 : 0, (2 * h + 1) % GROUPS);
        clear();
      }
    }
    if (GK == kGroup128) add(0, 0);
  };

  Chunk ring[DEPTH];
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) fetch(warp + i * kWarps, ring[i]);
  for (int c = warp; c < chunks; c += DEPTH * kWarps) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (c + i * kWarps < chunks) {
        compute(c + i * kWarps, ring[i]);
        fetch(c + (i + DEPTH) * kWarps, ring[i]);
      }
    }
  }

  // the warps' sums
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][t * 8 + tq * 2 + (e & 1)][gr + 8 * (e >> 1)] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * kRows; i += kThreads) {
    const int t = i / kRows, r = i % kRows, m = m0 + t, n = n0 + r;
    if (m >= a.m || n >= a.n) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w][t][r];
    if (a.bias) {
      float b;
      unpack_vec<DT, ES>(*reinterpret_cast<const RawVec<ES>*>(a.bias + static_cast<int64_t>(n) * ES), &b);
      s += b;
    }
    *reinterpret_cast<RawVec<ES>*>(a.y + m * a.ys + static_cast<int64_t>(n) * ES) = pack_vec<DT, ES>(&s);
  }
}

GroupKind group_kind(int64_t group) { return group % 128 == 0 ? kGroup128 : group % 64 == 0 ? kGroup64 : kGroup32; }

template <int DT, int NT>
int launch(const W4Args& a, const LaunchCtx& ctx) {
  const dim3 grid(static_cast<unsigned>((a.n + kRows - 1) / kRows), static_cast<unsigned>((a.m + 8 * NT - 1) / (8 * NT)));
  switch (group_kind(a.group.d)) {
    case kGroup128: linear_w4_kernel<DT, NT, kGroup128><<<grid, kThreads, 0, ctx.stream>>>(a); break;
    case kGroup64: linear_w4_kernel<DT, NT, kGroup64><<<grid, kThreads, 0, ctx.stream>>>(a); break;
    default: linear_w4_kernel<DT, NT, kGroup32><<<grid, kThreads, 0, ctx.stream>>>(a); break;
  }
  return cudaGetLastError() == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

template <int DT>
int launch_dt(const W4Args& a, const LaunchCtx& ctx) {
  return a.m <= 8 ? launch<DT, 1>(a, ctx) : launch<DT, 2>(a, ctx);
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
  if (d->group % 32 != 0 || d->k > (1 << 24) || d->n > (1ll << 31) - 65536 || d->m > 65535ll * 8) return "none";
  if (d->x_row_stride < 0 || d->w_row_stride < 0 || d->scales_row_stride < 0 || d->zeros_row_stride < 0 ||
      d->y_row_stride < d->n)
    return "none";
  *status = CMPX_ERR_MISALIGNED;
  if (reinterpret_cast<uintptr_t>(d->x) % 16 || reinterpret_cast<uintptr_t>(d->w) % 16 ||
      (d->m > 1 && (d->x_row_stride * es) % 16) || (d->n > 1 && d->w_row_stride % 16))
    return "none";
  *status = CMPX_OK;
  switch (group_kind(d->group)) {
    case kGroup128: return d->m <= 8 ? "linear_w4<8 tokens, groups of 128>" : "linear_w4<16 tokens, groups of 128>";
    case kGroup64: return d->m <= 8 ? "linear_w4<8 tokens, groups of 64>" : "linear_w4<16 tokens, groups of 64>";
    default: return d->m <= 8 ? "linear_w4<8 tokens, groups of 32>" : "linear_w4<16 tokens, groups of 32>";
  }
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
  a.group = make_fast_div(static_cast<uint32_t>(d->group));
  if (d->dtype == CMPX_F32) return launch_dt<CMPX_F32>(a, ctx);
  if (d->dtype == CMPX_F16) return launch_dt<CMPX_F16>(a, ctx);
  return launch_dt<CMPX_BF16>(a, ctx);
}

}  // namespace cmpx
