// paged_attn_mma.cu -- attention of one new token per sequence over a paged cache, fp16 / bf16, B200
// sm_100a: the kernel over the keys (the schedule is in paged_schedule.cuh, the join in paged_attn.cu).
//
// The up to 16 query heads of an item are the 16 rows of mma.m16n8k16: S = Q K^T and O += P V for 16 keys
// at a time, K and V fragments straight from shared memory (ldmatrix, transposed for V).  The
// products are a few percent of what the tensor cores do even in this form; what bounds the kernel is the
// one read of K and V, so it is built around loads in flight:
//   * every warp runs its own pipeline of buffers of 16 keys (KeyPipe, paged_schedule.cuh) and its own
//     online softmax over its own share of the keys.  Nothing in a share waits for another warp, so one
//     warp's first loads of an item hide behind the others' stream (with one share for a CTA's four
//     warps, which met at the end of each item, [32, 32 heads, 8 key heads, 128] bf16 with 64 to 8192 keys took 81 us);
//   * WHOLE (short caches): a CTA, or a cluster of up to 8, takes an item; the warps share its keys, meet once
//     and join their results through (distributed) shared memory, without a second kernel;
//   * rows of a buffer are swizzled in 16-byte chunks: ldmatrix reads without bank conflicts, and nothing is
//     padded.
// P is used as the sum of two 16-bit parts (cut off, and the rounded rest), so the weights carry 16 bits
// and more; a second product of P V costs nothing here, and one part alone would add as much error as the
// output's rounding does.  Both parts of a weight above zero are kept above zero, so that an infinite value stays
// infinite (0 * inf is not) as long as its weight is 2^-126 of the largest or more.  fp16 weights are exp2(s - m + 14):
// without the factor, which cancels, the rest of a weight below 2^-14 would fall into fp16's subnormal steps.  Those
// below 2^-24 then count as 2^-23, 2^-37 of the largest: less than a thousandth of the output's rounding for 2^16 such keys.
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "cmpx_internal.h"
#include "paged_schedule.cuh"

namespace cmpx {
namespace {

constexpr int kKeys = 16;  // keys per buffer
constexpr int kCtaWarps = 4;

template <int DP>
struct MmaCfg {
  static constexpr int ROW = DP * 2;                     // bytes of a row
  static constexpr int SLOTS = DP == 192 ? 2 : 3;
  // Per SM: 192 to 216 KB of buffers in all.  At 64, where a tile is 4 KB and its products' latency counts, more warps with
  // fewer buffers each serve better ([8, 16 heads, 4 key heads, 40] fp16 with 39062 keys: 51 us, 59 with two CTAs
  // and six slots); at 96 they do a little (80 in tiles of 128: 44.9 us for 19531 keys, of 96 with two CTAs and with
  // three 41.3; 300 keys of 32 sequences 9.0 and 8.1), at 128 not (39.7 us for 12207 keys; with two CTAs 38.8).
  static constexpr int CTAS = DP == 64 ? 4 : DP == 96 ? 3 : 2;
  using Pipe = KeyPipe<ROW, kKeys, SLOTS, 1, DP == 256>;
  static_assert(Pipe::BYTES >= 16 * DP * 4, "the warps' outputs are joined in the buffers");
};

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == CMPX_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return DT == CMPX_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

// Two floats cut off (rounded towards zero) to 16 bits.
template <int DT>
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == CMPX_BF16)
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A weight as its leading part is cut from: in fp16 at least the least that the type has, unless there is no weight.
template <int DT>
__device__ __forceinline__ float kept(float p) {
  return DT == CMPX_F16 && p != 0.f ? fmaxf(p, 0x1p-24f) : p;
}

template <int DT, int DP, bool WHOLE, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == kCtaWarps ? MmaCfg<DP>::CTAS : 1) paged_attn_mma_kernel(const __grid_constant__ PagedArgs a) {
  using C = MmaCfg<DP>;
  constexpr float kBias = DT == CMPX_F16 ? 14.f : 0.f;
  constexpr float kLeast = DT == CMPX_F16 ? 0x1p-24f : 0x1p-126f;  // the types' smallest (normal) values
  __shared__ int64_t scratch[33 + 2 * kWarps];
  __shared__ float2 sm_ml[kWarps][16], cta_ml[16];
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, tq = lane & 3;  // fragment row and column pair
  typename C::Pipe pipe(a, smem_u32(smem) + warp * C::Pipe::BYTES, a.head_dim * 2);
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
  constexpr int kStep = WHOLE ? kWarps : 1;  // the warp's sub-tiles of a stretch: from first in steps of kStep
  const int first = WHOLE ? warp : 0;
  // ldmatrix row addresses of this lane: the matrices of an x4 load are (keys 0-7, 8 columns), (keys 0-7, next 8
  // columns), (keys 8-15, ...) for K, and (keys 0-7), (keys 8-15) of 8 columns, then of the next 8, for V
  const int k_row = (lane & 7) + ((lane >> 4) << 3), k_chunk = (lane >> 3) & 1;
  const int v_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_chunk = lane >> 4;

  while (more) {
    pipe.begin(st, first, kStep);
    uint32_t q[DP / 16][4];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = gr + (i & 1) * 8, d = s * 16 + (i >> 1) * 8 + tq * 2;
        q[s][i] = 0;
        if (h < st.nh && d < a.head_dim)
          q[s][i] = __ldg(reinterpret_cast<const uint32_t*>(a.q + st.b * a.q_sb + (st.h0 + h) * a.q_sh + d * 2));
      }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int sub = first; sub < pipe.count; sub += kStep) {
      const uint32_t kbuf = pipe.buf + pipe.template take<true>();

      // two chains of products for each 8 keys
      float s[2][4], s2[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        uint32_t b[4];
        ldmatrix4<false>(kbuf + k_row * C::ROW + (((2 * ks + k_chunk) ^ C::Pipe::turn_of(k_row)) << 4), b);
        mma16816<DT>(ks & 1 ? s2[0] : s[0], q[ks], b[0], b[1]);
        mma16816<DT>(ks & 1 ? s2[1] : s[1], q[ks], b[2], b[3]);
      }
      const int left = st.key1 - st.key0 - sub * kKeys;  // keys of this buffer
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = (s[n][e] + s2[n][e]) * a.scale_log2;
          if (n * 8 + tq * 2 + (e & 1) >= left) s[n][e] = -INFINITY;
        }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {  // rows gr and gr + 8
        if (r == 1 && st.nh <= 8) {
          hi[1] = hi[3] = lo[1] = lo[3] = 0;
          continue;
        }
        float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m[r]);
        const float base = top == -INFINITY ? 0.f : top;
        if (__any_sync(0xffffffffu, top != m[r])) {
          const float keep = ex2_approx(m[r] - base);
          l[r] *= keep;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            o[i][2 * r] *= keep;
            o[i][2 * r + 1] *= keep;
          }
          m[r] = top;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2_approx(s[n][2 * r] - base + kBias), p1 = ex2_approx(s[n][2 * r + 1] - base + kBias);
          l[r] += p0 + p1;
          const uint32_t w = cut2<DT>(kept<DT>(p0), kept<DT>(p1));
          float h0, h1;
          unpack2<DT>(w, h0, h1);
          hi[2 * n + r] = w;
          lo[2 * n + r] = pack2<DT>(fmaxf(p0 - h0, kLeast), fmaxf(p1 - h1, kLeast));
        }
      }
      const uint32_t vbuf = pipe.buf + pipe.template take<false>();
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t b[4];
        ldmatrix4<true>(vbuf + v_row * C::ROW + (((2 * i + v_chunk) ^ C::Pipe::turn_of(v_row)) << 4), b);
        mma16816<DT>(o[2 * i], hi, b[0], b[1]);
        mma16816<DT>(o[2 * i + 1], hi, b[2], b[3]);
        mma16816<DT>(o[2 * i], lo, b[0], b[1]);
        mma16816<DT>(o[2 * i + 1], lo, b[2], b[3]);
      }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    if constexpr (WHOLE) {
      // the warps' results, through the buffers
      const bool bad = __syncthreads_or(pipe.bad);
      if (bad && threadIdx.x == 0) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
      float* sm_o = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int h = gr + 8 * r;
        if (h >= st.nh) continue;
        if (tq == 0) sm_ml[warp][h] = make_float2(m[r], bad ? __int_as_float(0x7fffffff) : l[r]);
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          *reinterpret_cast<float2*>(sm_o + (warp * 16 + h) * DP + i * 8 + tq * 2) =
              make_float2(o[i][2 * r], o[i][2 * r + 1]);
      }
      join_cluster<kWarps, 16, DP>(st.nh, a.head_dim, st.empty, sm_o, &sm_ml[0][0], cta_ml, [&](int h, int d, float x, float y) {
        *reinterpret_cast<uint32_t*>(a.o + st.b * a.o_sb + (st.h0 + h) * a.o_sh + d * 2) = pack2<DT>(x, y);
      });
      break;
    }
    const bool bad = __any_sync(0xffffffffu, pipe.bad);
    if (bad && lane == 0) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int h = gr + 8 * r;
      if (h >= st.nh) continue;
      const float sum = bad ? __int_as_float(0x7fffffff) : l[r];
      if (st.slot < 0) {
        const float inv = inverse_sum(sum, st.empty);
        uint8_t* p = a.o + st.b * a.o_sb + (st.h0 + h) * a.o_sh + tq * 4;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          if (i * 8 < a.head_dim) *reinterpret_cast<uint32_t*>(p + i * 16) = pack2<DT>(o[i][2 * r] * inv, o[i][2 * r + 1] * inv);
      } else {
        const int64_t row = st.slot * a.item_heads + h;
        float* p = a.part_o + row * a.head_dim + tq * 2;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          if (i * 8 < a.head_dim) *reinterpret_cast<float2*>(p + i * 8) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
        if (tq == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * row) = make_float2(m[r], sum);
      }
    }
    more = next_stretch(a, share, st);
    __syncwarp();
  }
}

template <int DT, int DP, bool WHOLE, int W>
int launch(const PagedArgs& a, int ctas, int ranks, const LaunchCtx& ctx) {
  auto kernel = paged_attn_mma_kernel<DT, DP, WHOLE, W>;
  constexpr int kSmem = W * MmaCfg<DP>::Pipe::BYTES;
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

template <int DT, int DP>
int launch_as(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  if (ranks == 0) return launch<DT, DP, false, kCtaWarps>(a, ctas, ranks, ctx);
  if (wide) return launch<DT, DP, true, 2 * kCtaWarps>(a, ctas, ranks, ctx);
  return launch<DT, DP, true, kCtaWarps>(a, ctas, ranks, ctx);
}

template <int DT>
int launch_dt(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  if (a.head_dim <= 64) return launch_as<DT, 64>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 96) return launch_as<DT, 96>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 128) return launch_as<DT, 128>(a, ctas, ranks, wide, ctx);
  if (a.head_dim <= 192) return launch_as<DT, 192>(a, ctas, ranks, wide, ctx);
  return launch_as<DT, 256>(a, ctas, ranks, wide, ctx);
}

}  // namespace

PagedShape paged_mma_shape(int64_t head_dim) {
  const int ctas = head_dim <= 64 ? MmaCfg<64>::CTAS : head_dim <= 96 ? MmaCfg<96>::CTAS : MmaCfg<128>::CTAS;
  return PagedShape{ctas, kCtaWarps};
}

int launch_paged_mma(const PagedArgs& a, int dtype, int ctas, int ranks, bool wide, const LaunchCtx& ctx) {
  return dtype == CMPX_BF16 ? launch_dt<CMPX_BF16>(a, ctas, ranks, wide, ctx) : launch_dt<CMPX_F16>(a, ctas, ranks, wide, ctx);
}

}  // namespace cmpx
