// paged_attn_f32.cu -- attention of one new token per sequence over a paged cache, fp32, B200 sm_100a: the
// kernel over the keys (the schedule is in paged_schedule.cuh, the join in paged_attn.cu).
//
// The same warp-private pipelines as the 16-bit kernel's, over fp32 rows, with the products on the FMA units: LPT
// lanes share a key, each with two vectors of 4 values of its row; a lane group runs its own online
// softmax over its keys for up to HG heads, so a key and a value are read from memory once for 8 heads and
// from shared memory once for all of them.  At one head per key head the stream bounds it, at eight the
// FMA units (about 40 instructions per key, head and lane group), where paged_attn_f32_mma.cu takes over.
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "cmpx_internal.h"
#include "paged_schedule.cuh"

namespace cmpx {
namespace {

constexpr int kCtasPerSm = 2, kCtaWarps = 4;

template <int DP>
struct F32Cfg {
  static constexpr int LPT = DP / 8;        // lanes per key
  static constexpr int GROUPS = 32 / LPT;   // keys of a step
  static constexpr int STEPS = 4;
  static constexpr int KEYS = GROUPS * STEPS;  // per buffer: 8 KB of keys and values
  static constexpr int ROW = DP * 4;
  static constexpr int SLOTS = 3;
  using Pipe = KeyPipe<ROW, KEYS, SLOTS, 0>;
};

template <int DP, int HG, bool WHOLE, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == kCtaWarps ? kCtasPerSm : 1) paged_attn_f32_kernel(const __grid_constant__ PagedArgs a) {
  using C = F32Cfg<DP>;
  constexpr int LPT = C::LPT, STEPS = C::STEPS;
  static_assert(C::Pipe::BYTES >= HG * DP * 4, "the warps' outputs are joined in the buffers");
  __shared__ int64_t scratch[33 + 2 * kWarps];
  __shared__ float2 sm_ml[kWarps][HG], cta_ml[HG];
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % LPT, group = lane / LPT;
  typename C::Pipe pipe(a, smem_u32(smem) + warp * C::Pipe::BYTES, a.head_dim * 4);
  const uint8_t* const buffers = smem + warp * C::Pipe::BYTES;
  pdl_allow_dependents();

  Share share{};
  bool more = true;
  Stretch st;
  if (WHOLE) {
    const int ranks = cluster_size();
    st = whole_item(a, blockIdx.x / ranks, cluster_rank(), ranks);
  } else {
    share = find_share<kWarps>(a, scratch);
    more = next_stretch(a, share, st);
  }
  constexpr int kStep = WHOLE ? kWarps : 1;  // the warp's buffers of a stretch: from first in steps of kStep
  const int first = WHOLE ? warp : 0;
  const int col[2] = {4 * sub, 4 * (sub + LPT)};

  while (more) {
    pipe.begin(st, first, kStep);
    float q[HG][8], o[HG][8], m[HG], l[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < st.nh && col[i] < a.head_dim)
          v = __ldg(reinterpret_cast<const float4*>(a.q + st.b * a.q_sb + (st.h0 + h) * a.q_sh) + col[i] / 4);
        q[h][4 * i] = v.x * a.scale_log2;
        q[h][4 * i + 1] = v.y * a.scale_log2;
        q[h][4 * i + 2] = v.z * a.scale_log2;
        q[h][4 * i + 3] = v.w * a.scale_log2;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o[h][e] = 0.f;
    }
    for (int at = first; at < pipe.count; at += kStep) {
      const uint8_t* const kbuf = buffers + pipe.template take<true>();
      const int left = st.key1 - st.key0 - at * C::KEYS;  // keys of this buffer

      float s[STEPS][HG];
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        const int key = u * C::GROUPS + group;
        const float4 k0 = *reinterpret_cast<const float4*>(kbuf + key * C::ROW + col[0] * 4);
        const float4 k1 = *reinterpret_cast<const float4*>(kbuf + key * C::ROW + col[1] * 4);
        const float k[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          float x = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) x = fmaf(q[h][e], k[e], x);
#pragma unroll
          for (int off = LPT / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
          s[u][h] = key < left ? x : -INFINITY;
        }
      }
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        float top = m[h];
#pragma unroll
        for (int u = 0; u < STEPS; ++u) top = fmaxf(top, s[u][h]);
        const float base = top == -INFINITY ? 0.f : top;  // no key yet: exp2(-inf - 0) = 0
        if (__any_sync(0xffffffffu, top != m[h])) {
          const float keep = ex2_approx(m[h] - base);
          m[h] = top;
          l[h] *= keep;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[h][e] *= keep;
        }
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
          s[u][h] = ex2_approx(s[u][h] - base);
          l[h] += s[u][h];
        }
      }
      const uint8_t* const vbuf = buffers + pipe.template take<false>();
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        const uint8_t* const row = vbuf + (u * C::GROUPS + group) * C::ROW;
        const float4 v0 = *reinterpret_cast<const float4*>(row + col[0] * 4);
        const float4 v1 = *reinterpret_cast<const float4*>(row + col[1] * 4);
        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int h = 0; h < HG; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[h][e] = fmaf(s[u][h], v[e], o[h][e]);
      }
    }
    cp_async_wait<0>();

    // the warp's lane groups
#pragma unroll
    for (int h = 0; h < HG; ++h) {
#pragma unroll
      for (int off = LPT; off < 32; off <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m[h], off);
        const float top = fmaxf(m[h], m2), base = top == -INFINITY ? 0.f : top;
        const float w1 = ex2_approx(m[h] - base), w2 = ex2_approx(m2 - base);
        l[h] = l[h] * w1 + __shfl_xor_sync(0xffffffffu, l[h], off) * w2;
        m[h] = top;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[h][e] = o[h][e] * w1 + __shfl_xor_sync(0xffffffffu, o[h][e], off) * w2;
      }
    }
    if constexpr (WHOLE) {
      // the warps' results, through the buffers
      const bool bad = __syncthreads_or(pipe.bad);
      if (bad && threadIdx.x == 0) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
      float* const sm_o = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        if (group != 0 || h >= st.nh) continue;
        if (sub == 0) sm_ml[warp][h] = make_float2(m[h], bad ? __int_as_float(0x7fffffff) : l[h]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float4*>(sm_o + (warp * HG + h) * DP + col[i]) =
              make_float4(o[h][4 * i], o[h][4 * i + 1], o[h][4 * i + 2], o[h][4 * i + 3]);
      }
      join_cluster<kWarps, HG, DP>(st.nh, a.head_dim, st.empty, sm_o, &sm_ml[0][0], cta_ml, [&](int h, int d, float x, float y) {
        *reinterpret_cast<float2*>(a.o + st.b * a.o_sb + (st.h0 + h) * a.o_sh + d * 4) = make_float2(x, y);
      });
      break;
    }
    const bool bad = __any_sync(0xffffffffu, pipe.bad);
    if (bad && lane == 0) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      if (h >= st.nh || group != 0) continue;
      const float sum = bad ? __int_as_float(0x7fffffff) : l[h];
      const float f = st.slot >= 0 ? 1.f : inverse_sum(sum, st.empty);
      const int64_t row = st.slot * a.item_heads + h;
      float* const p = st.slot < 0 ? reinterpret_cast<float*>(a.o + st.b * a.o_sb + (st.h0 + h) * a.o_sh)
                                   : a.part_o + row * a.head_dim;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (col[i] < a.head_dim)
          *reinterpret_cast<float4*>(p + col[i]) =
              make_float4(o[h][4 * i] * f, o[h][4 * i + 1] * f, o[h][4 * i + 2] * f, o[h][4 * i + 3] * f);
      if (st.slot >= 0 && sub == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * row) = make_float2(m[h], sum);
    }
    more = next_stretch(a, share, st);
    __syncwarp();
  }
}

template <int DP, int HG, bool WHOLE, int W>
int launch(const PagedArgs& a, int ctas, int ranks, const LaunchCtx& ctx) {
  auto kernel = paged_attn_f32_kernel<DP, HG, WHOLE, W>;
  constexpr int kSmem = W * F32Cfg<DP>::Pipe::BYTES;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::call_once(once[dev & 63], [&] {
    attr_err[dev & 63] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (attr_err[dev & 63] != cudaSuccess) return CMPX_ERR_LAUNCH;
  if (WHOLE) return launch_whole(kernel, a, ctas, ranks, 32 * W, kSmem, ctx.stream);
  kernel<<<ctas, 32 * W, kSmem, ctx.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

template <int DP, int HG>
int launch_as(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  if (ranks == 0) return launch<DP, HG, false, kCtaWarps>(a, ctas, ranks, ctx);
  return wide ? launch<DP, HG, true, kCtaWarps * kCtasPerSm>(a, ctas, ranks, ctx)
              : launch<DP, HG, true, kCtaWarps>(a, ctas, ranks, ctx);
}

template <int DP>
int launch_heads(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  if (a.item_heads == 1) return launch_as<DP, 1>(a, ctas, ranks, wide, ctx);
  if (a.item_heads <= 4) return launch_as<DP, 4>(a, ctas, ranks, wide, ctx);
  return launch_as<DP, 8>(a, ctas, ranks, wide, ctx);
}

}  // namespace

PagedShape paged_f32_shape() { return PagedShape{kCtasPerSm, kCtaWarps}; }

int launch_paged_f32(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  if (a.head_dim <= 64) return launch_heads<64>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 128) return launch_heads<128>(a, ctas, ranks, wide, ctx);
  return launch_heads<256>(a, ctas, ranks, wide, ctx);
}

}  // namespace cmpx
