// paged_attn_f32_mma.cu -- attention of one new token per sequence over a paged cache, fp32 with several query heads
// per key head, B200 sm_100a: the kernel over the keys (the schedule is in paged_schedule.cuh, the join in
// paged_attn.cu, fewer heads in paged_attn_f32.cu).
//
// An fp32 value goes to the tensor cores as two parts with 11 bits of its fraction each, three products a pair, in
// mma.m16n8k8, transposed, so that 8 heads fill the side of 8:
//   S^T = K Q^T (keys x heads),  O^T += V^T P^T (dims x heads),
// sums and softmax in fp32.  The order of a product's k, and of the rows of the other side, is free as long as
// both sides share it: a lane takes 16 bytes of a row at a time, and P^T's fragments are S^T's, turned by movmatrix.
// K and V are cut with an addition, an AND and a subtraction each.  If a result is not finite, the warp walks its keys
// once more with infinities (whose rest would be NaN) in mind.
// What that is off by, of a product: the two rests' product, which is left out, is at most 2^-22 (a rest is at most 2^-11), and
// each rest loses up to 2^-23.  Against 64 bits, norm of the difference over the result's, random inputs of 300 to
// 30000 keys, by head size (this kernel; FMA units on the same inputs; plain fp32 products): 40: 2.9e-7, 2.4e-7, 4.1e-7;
// 64: 3.0, 2.3, 4.4; 80: 2.9, 2.7, 4.8; 96: 2.8, 2.7, 5.2; 128: 2.8, 2.4, 5.2; 160: 2.4, 2.8, 5.5; 192: 2.6, 2.9, 6.0
// (the largest of three lengths).  With the leading parts of K and V cut towards zero it was 3.6 to 4.5, in the same time.
// What bounds it: the two or three warps that a scheduler has, whose registers and buffers leave no more, wait for their
// own products and shuffles (issue slots 46% used, tensor cores 26% at 64).  [8, 32 heads, 4 key heads] over
// 200 MB: 52 us at 40, 42 at 64, 43 at 80, 37 at 96, 37 at 128, 50 at 160, 49 at 192 (FMA units: 74, 52, 75, 67,
// 53, 84, 71); at 256 the queries do not fit the registers.
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>
#include <type_traits>

#include "cmpx_internal.h"
#include "paged_schedule.cuh"

namespace cmpx {
namespace {

constexpr int kHeads = 8;  // per item

template <int DP>
struct PartsCfg {
  // Keys per buffer: with 8 half of the rows of S^T's products are empty (80: 54 us instead of 44), but 16 at 160
  // would leave four warps per SM (192: 80 us instead of 50).
  static constexpr int KEYS = DP <= 128 ? 16 : 8;
  static constexpr int ROW = DP * 4;                       // bytes of a row
  static constexpr int SLOTS = DP == 128 ? 3 : 2;
  static constexpr int CTAS = DP == 64 ? 3 : 2;           // per SM
  static constexpr int WARPS = 4;         // per CTA
  using Pipe = KeyPipe<ROW, KEYS, SLOTS, 2, DP == 128>;
  static_assert(Pipe::BYTES >= kHeads * DP * 4, "the warps' outputs are joined in the buffers");
};

// The parts of a value: the upper 11 bits of its fraction, rounded, and the rest, of which the tensor cores take 11 of its
// 12 bits.  An infinite value (and one that is rounded to it) has no rest; without INF its rest is NaN.
template <bool INF>
__device__ __forceinline__ void cut(float x, uint32_t (&p)[2]) {
  p[0] = (INF ? __float_as_uint(x) : __float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  float rest = x - __uint_as_float(p[0]);
  if (INF && fabsf(x) == INFINITY) rest = 0.f;
  p[1] = __float_as_uint(rest);
}
// The same, rounded to nearest, for the side whose values are used many times.  With INF the rest is not zero (2^-126
// with the value's sign instead), so that an infinite factor on the other side stays infinite (0 * inf is not).
template <bool INF>
__device__ __forceinline__ void cut_round(float x, uint32_t (&p)[2]) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(p[0]) : "f"(x));
  float rest = x - __uint_as_float(p[0]);
  if (INF) {
    p[0] = __float_as_uint(x) & 0xFFFFE000u;
    rest = x - __uint_as_float(p[0]);
    if (rest == 0.f) rest = copysignf(0x1p-126f, x);
  }
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(p[1]) : "f"(rest));
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int DP, bool WHOLE, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == PartsCfg<DP>::WARPS ? PartsCfg<DP>::CTAS : 1)
    paged_attn_f32_mma_kernel(const __grid_constant__ PagedArgs a) {
  using C = PartsCfg<DP>;
  constexpr int KEYS = C::KEYS, HALVES = KEYS / 8;  // halves: 8 keys, rows gr and gr + 8 of a fragment
  constexpr bool KEEP_Q = DP <= 128;                // registers for the queries' parts, which are cut again otherwise
  __shared__ int64_t scratch[33 + 2 * kWarps];
  __shared__ float2 sm_ml[kWarps][kHeads], cta_ml[kHeads];
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, tq = lane & 3;  // fragment row and column pair
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

  while (more) {
    float q[DP / 16][4];  // Q^T: head gr, dims 16 s + 4 tq .. + 3
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      const int d = s * 16 + tq * 4;
      if (gr < st.nh && d < a.head_dim)
        v = __ldg(reinterpret_cast<const float4*>(a.q + st.b * a.q_sb + (st.h0 + gr) * a.q_sh + d * 4));
      q[s][0] = v.x;
      q[s][1] = v.y;
      q[s][2] = v.z;
      q[s][3] = v.w;
    }
    float o[DP / 16][4], m[2], l[2];  // m and l of heads 2 tq and 2 tq + 1; l of this lane's keys
    auto walk = [&](auto inf) {       // inf: values may be infinite
      constexpr bool INF = decltype(inf)::value;
      pipe.begin(st, first, kStep);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      uint32_t qp[KEEP_Q ? DP / 16 : 1][4][2];
      if (KEEP_Q) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) cut_round<INF>(q[s][i], qp[KEEP_Q ? s : 0][i]);
      }
      for (int at = first; at < pipe.count; at += kStep) {
        const uint8_t* const kbuf = buffers + pipe.template take<true>();

        // The products of the leading parts in short chains, added up here: a sum inside the tensor core is cut off,
        // not rounded, which over a long chain shows (4096 keys: 1.7e-6 off, like this).
        float sum[4], s[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = s[0][e] = s[1][e] = s[2][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          uint32_t k[2][4][2];  // half, value, part
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h < HALVES) {
              const float4 v =
                  *reinterpret_cast<const float4*>(kbuf + (gr + 8 * h) * C::ROW + (((ks * 4 + tq) ^ C::Pipe::turn_of(gr)) << 4));
              cut<INF>(v.x, k[h][0]);
              cut<INF>(v.y, k[h][1]);
              cut<INF>(v.z, k[h][2]);
              cut<INF>(v.w, k[h][3]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) k[h][i][0] = k[h][i][1] = 0;
            }
          }
          if (!KEEP_Q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x = q[ks][i];
              asm volatile("" : "+f"(x));  // not once for all, which would spill
              cut_round<INF>(x, qp[0][i]);
            }
          }
          const auto& qs = qp[KEEP_Q ? ks : 0];
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // values 2 i and 2 i + 1
            mma(s[0], k[0][2 * i][0], k[1][2 * i][0], k[0][2 * i + 1][0], k[1][2 * i + 1][0], qs[2 * i][0], qs[2 * i + 1][0]);
            mma(s[1], k[0][2 * i][0], k[1][2 * i][0], k[0][2 * i + 1][0], k[1][2 * i + 1][0], qs[2 * i][1], qs[2 * i + 1][1]);
            mma(s[2], k[0][2 * i][1], k[1][2 * i][1], k[0][2 * i + 1][1], k[1][2 * i + 1][1], qs[2 * i][0], qs[2 * i + 1][0]);
          }
          if (ks & 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sum[e] += s[0][e];
              s[0][e] = 0.f;
            }
          }
        }
        const int left = st.key1 - st.key0 - at * KEYS;  // keys of this buffer
        float p[HALVES][2], keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const float x = (sum[2 * h + e] + (s[1][2 * h + e] + s[2][2 * h + e])) * a.scale_log2;
            p[h][e] = gr + 8 * h < left ? x : -INFINITY;
            top = fmaxf(top, p[h][e]);
          }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          top = fmaxf(top, m[e]);
          const float base = top == -INFINITY ? 0.f : top;
          keep[e] = ex2_approx(m[e] - base);
          l[e] *= keep[e];
          m[e] = top;
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            p[h][e] = ex2_approx(p[h][e] - base);
            l[e] += p[h][e];
          }
        }
        uint32_t w[HALVES][2][2];  // P^T of head gr: key 8 h + 2 tq + r, part
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const uint32_t p0 = __float_as_uint(p[h][0]), p1 = __float_as_uint(p[h][1]);
          const uint32_t up = transposed(__byte_perm(p0, p1, 0x7632)), low = transposed(__byte_perm(p0, p1, 0x5410));
          cut_round<INF>(__uint_as_float(__byte_perm(low, up, 0x5410)), w[h][0]);
          cut_round<INF>(__uint_as_float(__byte_perm(low, up, 0x7632)), w[h][1]);
        }
        const uint8_t* const vbuf = buffers + pipe.template take<false>();
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk) {
          float t[2][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) t[0][e] = t[1][e] = 0.f;
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            uint32_t v[2][4][2];  // key 8 h + 2 tq + r, dim 32 blk + 4 gr + i, part
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int row = 2 * tq + r;
              const float4 x = *reinterpret_cast<const float4*>(vbuf + (row + 8 * h) * C::ROW +
                                                                (((blk * 8 + gr) ^ C::Pipe::turn_of(row)) << 4));
              cut<INF>(x.x, v[r][0]);
              cut<INF>(x.y, v[r][1]);
              cut<INF>(x.z, v[r][2]);
              cut<INF>(x.w, v[r][3]);
            }
            auto product = [&](int y, int z) {
#pragma unroll
              for (int j = 0; j < 2; ++j)  // rows gr and gr + 8: dims 4 gr + 2 j and the next
                mma(t[j], v[0][2 * j][y], v[0][2 * j + 1][y], v[1][2 * j][y], v[1][2 * j + 1][y], w[h][0][z], w[h][1][z]);
            };
            product(1, 0);
            product(0, 1);
            product(0, 0);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[2 * blk + j][e] = fmaf(o[2 * blk + j][e], keep[e & 1], t[j][e]);
        }
      }
      cp_async_wait<0>();
    };
    walk(std::false_type{});
    bool finite = true;  // an infinite key or value has made a result NaN: once more with care
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) finite = finite && fabsf(o[i][e]) < INFINITY;
    if (__any_sync(0xffffffffu, !finite)) walk(std::true_type{});
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], off);
    auto dims = [&](int blk, int e, float f) {  // dims 32 blk + 4 gr .. + 3 of head 2 tq + e
      return make_float4(o[2 * blk][e] * f, o[2 * blk][2 + e] * f, o[2 * blk + 1][e] * f, o[2 * blk + 1][2 + e] * f);
    };
    if constexpr (WHOLE) {
      // the warps' results, through the buffers
      const bool bad = __syncthreads_or(pipe.bad);
      if (bad && threadIdx.x == 0) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
      float* const sm_o = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 2 * tq + e;
        if (h >= st.nh) continue;
        if (gr == 0) sm_ml[warp][h] = make_float2(m[e], bad ? __int_as_float(0x7fffffff) : l[e]);
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
          *reinterpret_cast<float4*>(sm_o + (warp * kHeads + h) * DP + blk * 32 + gr * 4) = dims(blk, e, 1.f);
      }
      join_cluster<kWarps, kHeads, DP>(st.nh, a.head_dim, st.empty, sm_o, &sm_ml[0][0], cta_ml,
                                       [&](int h, int d, float x, float y) {
                                         *reinterpret_cast<float2*>(a.o + st.b * a.o_sb + (st.h0 + h) * a.o_sh + d * 4) =
                                             make_float2(x, y);
                                       });
      break;
    }
    const bool bad = __any_sync(0xffffffffu, pipe.bad);
    if (bad && lane == 0) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = 2 * tq + e;
      if (h >= st.nh) continue;
      const float sum = bad ? __int_as_float(0x7fffffff) : l[e];
      const float f = st.slot >= 0 ? 1.f : inverse_sum(sum, st.empty);
      const int64_t row = st.slot * a.item_heads + h;
      float* const out = st.slot < 0 ? reinterpret_cast<float*>(a.o + st.b * a.o_sb + (st.h0 + h) * a.o_sh)
                                     : a.part_o + row * a.head_dim;
#pragma unroll
      for (int blk = 0; blk < DP / 32; ++blk)
        if (blk * 32 + gr * 4 < a.head_dim) *reinterpret_cast<float4*>(out + blk * 32 + gr * 4) = dims(blk, e, f);
      if (st.slot >= 0 && gr == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * row) = make_float2(m[e], sum);
    }
    more = next_stretch(a, share, st);
    __syncwarp();
  }
}

template <int DP, bool WHOLE, int W>
int launch(const PagedArgs& a, int ctas, int ranks, const LaunchCtx& ctx) {
  auto kernel = paged_attn_f32_mma_kernel<DP, WHOLE, W>;
  constexpr int kSmem = W * PartsCfg<DP>::Pipe::BYTES;
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

template <int DP>
int launch_as(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  using C = PartsCfg<DP>;
  if (ranks == 0) return launch<DP, false, C::WARPS>(a, ctas, ranks, ctx);
  if (wide) return launch<DP, true, C::WARPS * C::CTAS>(a, ctas, ranks, ctx);
  return launch<DP, true, C::WARPS>(a, ctas, ranks, ctx);
}

template <int DP>
PagedShape shape() {
  return PagedShape{PartsCfg<DP>::CTAS, PartsCfg<DP>::WARPS};
}

}  // namespace

PagedShape paged_f32_mma_shape(int64_t head_dim) {
  if (head_dim <= 64) return shape<64>();
  if (head_dim <= 96) return shape<96>();
  if (head_dim <= 128) return shape<128>();
  return head_dim <= 160 ? shape<160>() : shape<192>();
}

int launch_paged_f32_mma(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  if (a.head_dim <= 64) return launch_as<64>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 96) return launch_as<96>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 128) return launch_as<128>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 160) return launch_as<160>(a, ctas, ranks, wide, ctx);
  return launch_as<192>(a, ctas, ranks, wide, ctx);
}

}  // namespace cmpx
