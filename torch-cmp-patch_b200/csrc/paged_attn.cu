// paged_attn.cu -- attention of one new token per sequence over a paged key-value cache, B200 sm_100a:
// the choice of schedule and the join (the kernels over the keys: paged_attn_mma.cu, paged_attn_f32.cu, paged_attn_f32_mma.cu).
//
//   o[b, h] = sum_t p_t V[t] / sum_t p_t,   p_t = exp(q[b, h] . K[t] * scale - m),  t < lengths[b],
// with the maximum m and both sums carried along (one pass over the keys).
//
// Each key and value is read once from memory for all the query heads that share it, and that read is the
// whole cost: 4 flops per element of K or V and head.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "cmpx_internal.h"
#include "paged_schedule.cuh"

namespace cmpx {
namespace {

// Loads of what the main kernel wrote: from L2, and, being volatile, never moved above pdl_wait().
__device__ __forceinline__ float2 load_part2(const float* p) {
  float2 v;
  asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_part4(const float* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}

// Joins the partial results of each (sequence, query head) row: W warps of a block per row (WROW = W), or one warp
// per row and W rows per block (WROW = 1).  A row's warps take every WROW'th partial result: up to 32 at a
// time, a lane each for the maxima and sums, all lanes along the head for the outputs, whose loads do not
// wait for the weights.
template <int DT, int V, int W, int WROW>  // V: float4 vectors per lane and row (head_dim <= 128 V)
__global__ void __launch_bounds__(32 * W) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int AHEAD = 8;
  constexpr int ES = elt_size(DT);
  __shared__ float sm_ml[W][2];
  __shared__ float4 sm_o[W][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_index = WROW == 1 ? static_cast<int>(blockIdx.x) * W + warp : static_cast<int>(blockIdx.x);
  const int part_warp = WROW == 1 ? 0 : warp;  // this warp among its row's
  const bool there = row_index < a.batch * a.heads;
  const int b = there ? row_index / a.heads : 0, h = there ? row_index - b * a.heads : 0;
  int64_t first = 0, total = 0;  // units before sequence b, and in all
  for (int i = lane; i < a.batch; i += 32) {
    const int64_t n = seq_units(a, i);
    total += n;
    if (i < b) first += n;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    first += __shfl_xor_sync(0xffffffffu, first, off);
    total += __shfl_xor_sync(0xffffffffu, total, off);
  }
  const int64_t share = share_units(total, a.workers);
  const int tiles = seq_tiles(a, b);
  const int kvh = h / a.group, g = h - kvh * a.group, part = g / a.item_heads;
  const int64_t begin = first + (static_cast<int64_t>(kvh) * a.items_per_head + part) * (tiles + kItemCost) + kItemCost;
  const int64_t c0 = begin / share, c1 = min((begin + tiles - 1) / share, a.workers - 1);
  pdl_wait();  // every block: this kernel is not done before the main one is
  if (!there || c0 >= c1) return;  // written by its warp
  const int hh = g - part * a.item_heads;
  float m = -INFINITY, l = 0.f;
  float4 o[V];
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto row_of = [&](int64_t c) { return (2 * c + (c == c0 ? 1 : 0)) * a.item_heads + hh; };
  for (int64_t cb = c0 + part_warp; cb <= c1; cb += 32 * WROW) {
    const int64_t mine = cb + static_cast<int64_t>(lane) * WROW;
    const int count = static_cast<int>(min(static_cast<int64_t>(32), (c1 - cb) / WROW + 1));
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < count) ml = load_part2(a.part_ml + 2 * row_of(mine));
    float top = ml.x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    top = fmaxf(top, m);
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = ex2_approx(m - base), weight = lane < count ? ex2_approx(ml.x - base) : 0.f;
    float sum = lane < count ? weight * ml.y : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    m = top;
    l = l * keep + sum;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = make_float4(o[v].x * keep, o[v].y * keep, o[v].z * keep, o[v].w * keep);
    for (int k0 = 0; k0 < count; k0 += AHEAD) {
      float4 p[AHEAD][V];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          p[k][v] = make_float4(0.f, 0.f, 0.f, 0.f);
          const int d = 4 * (lane + 32 * v);
          if (k0 + k < count && d < a.head_dim)
            p[k][v] = load_part4(a.part_o + row_of(cb + static_cast<int64_t>(k0 + k) * WROW) * a.head_dim + d);
        }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const float w = __shfl_sync(0xffffffffu, weight, (k0 + k) & 31);
        if (k0 + k < count)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            o[v].x = fmaf(w, p[k][v].x, o[v].x);
            o[v].y = fmaf(w, p[k][v].y, o[v].y);
            o[v].z = fmaf(w, p[k][v].z, o[v].z);
            o[v].w = fmaf(w, p[k][v].w, o[v].w);
          }
      }
    }
  }
  uint8_t* const out = a.o + b * a.o_sb + h * a.o_sh;
  if (WROW == 1) {
    const float inv = inverse_sum(l, false);  // (a row in several parts has keys)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int d = 4 * (lane + 32 * v);
      const float f[4] = {o[v].x * inv, o[v].y * inv, o[v].z * inv, o[v].w * inv};
      if (d < a.head_dim) *reinterpret_cast<RawVec<4 * ES>*>(out + d * ES) = pack_vec<DT, 4 * ES>(f);
    }
    return;
  }
  if (lane == 0) {
    sm_ml[warp][0] = m;
    sm_ml[warp][1] = l;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sm_o[warp][lane + 32 * v] = o[v];
  __syncthreads();
  for (int d = threadIdx.x; d < a.head_dim; d += 32 * W) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, sm_ml[w][0]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float weight = ex2_approx(sm_ml[w][0] - base);
      sum = fmaf(weight, sm_ml[w][1], sum);
      acc = fmaf(weight, reinterpret_cast<const float*>(sm_o[w])[d], acc);
    }
    const float r = acc * inverse_sum(sum, false);
    *reinterpret_cast<RawVec<ES>*>(out + d * ES) = pack_vec<DT, ES>(&r);
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------

float scale_log2(const cmpx_paged_attn_desc* d) { return static_cast<float>(d->scale * 1.4426950408889634074); }

// fp32 on the tensor cores: from five heads per item on, where the FMA units bound the other kernel ([8, 32/4, 128],
// 6103 keys: 37 us, 53 there; with four heads the other takes 35), and from two where that kernel pads the heads to 128 and this
// one to 96 ([8, 16/4, 80], 9765 keys: 42 and 48).  Above 192 the queries do not fit its registers.
bool f32_mma(int item_heads, int64_t head_dim) {
  return item_heads > 4 ? head_dim <= 192 : item_heads > 1 && head_dim > 64 && head_dim <= 96;
}

struct Schedule {
  int item_heads, items_per_head;
  int64_t items;
  int ranks;        // CTAs per whole item, 0: equal shares and a join
  int ctas;
  bool wide;        // a CTA of a whole item has an SM to itself
  int64_t workers;  // warps with shares
};

// Keys per CTA up to which whole items are taken whatever their number, and up to which they are where all
// CTAs fit on the GPU at once.
constexpr int kWholeKeys = 512;
constexpr int kClusterKeys = 1024;

Schedule schedule(const cmpx_paged_attn_desc* d, int num_sms) {
  Schedule s{};
  const bool f32 = d->dtype == CMPX_F32;
  const int64_t group = d->heads / d->cache.heads_kv, most_heads = f32 ? 8 : 16;
  // the fewest items of at most most_heads heads, and their heads shared out evenly
  s.items_per_head = static_cast<int>(std::max<int64_t>(1, (group + most_heads - 1) / most_heads));
  s.item_heads = static_cast<int>((group + s.items_per_head - 1) / s.items_per_head);
  s.items = d->batch * d->cache.heads_kv * s.items_per_head;
  const int64_t keys = d->cache.table_width * d->cache.page_size;  // of the longest sequence there can be
  const PagedShape shape = !f32                                         ? paged_mma_shape(d->cache.head_dim)
                           : f32_mma(s.item_heads, d->cache.head_dim) ? paged_f32_mma_shape(d->cache.head_dim)
                                                                      : paged_f32_shape();
  const int per_sm = shape.ctas;
  const int64_t slots = static_cast<int64_t>(num_sms) * per_sm;
  // Whole items, by one CTA or a cluster of 2, 4 or 8 (256 keys each): one launch and no join.  The CTAs have to
  // fit on the GPU at once, and a cluster's into one GPC: 7/8 of the places can be counted on.
  // Where they are few, each has an SM to itself and all its warps, for the loads in flight
  // ([1, 32/8, 128] bf16, 4096 keys: 10.5 us; equal shares and a join 13.5).  Of many, that lengths differ
  // costs less than the join does ([100, 16/4, 64] fp16, 900 keys: 19.4 us; equal shares 23.4; [64, 32/8, 64], 10 to
  // 1000 keys: 15.4 and 14.3).
  auto fits = [&](int ranks) { return s.items * ranks * 8 <= slots * 7; };
  int ranks = 1;
  while (ranks < 8 && keys > 256 * ranks && fits(2 * ranks)) ranks *= 2;
  if (keys <= kWholeKeys || (keys <= kClusterKeys * ranks && fits(ranks))) {
    s.ranks = ranks;
    s.ctas = static_cast<int>(s.items * ranks);
    s.wide = per_sm > 1 && s.ctas <= num_sms * 3 / 4;
    return s;
  }
  const int64_t units = s.items * (std::max<int64_t>(1, (keys + kTile - 1) / kTile) + kItemCost);
  s.ctas = static_cast<int>(std::max<int64_t>(1, std::min(slots, (units + kShareMin - 1) / kShareMin)));
  s.workers = static_cast<int64_t>(s.ctas) * shape.warps;
  return s;
}

size_t part_floats(const cmpx_paged_attn_desc* d, const Schedule& s) {
  return s.ranks ? 0 : 2ull * s.workers * s.item_heads * (d->cache.head_dim + 2);
}

template <int DT, int V, int W, int WROW>
int launch_join_as(const PagedArgs& a, int64_t blocks, const LaunchCtx& ctx) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(32 * W);
  cfg.stream = ctx.stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<DT, V, W, WROW>, a) == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

template <int DT, int V>
int launch_join(const PagedArgs& a, int64_t most_parts, const LaunchCtx& ctx) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads;
  if (most_parts <= 32) return launch_join_as<DT, V, 4, 1>(a, (rows + 3) / 4, ctx);
  if (rows <= ctx.num_sms) return launch_join_as<DT, V, 16, 16>(a, rows, ctx);
  return launch_join_as<DT, V, 4, 4>(a, rows, ctx);
}

template <int DT>
int launch_join_dim(const PagedArgs& a, int64_t most_parts, const LaunchCtx& ctx) {
  return a.head_dim <= 128 ? launch_join<DT, 1>(a, most_parts, ctx) : launch_join<DT, 2>(a, most_parts, ctx);
}

}  // namespace

const char* paged_attn_plan(const cmpx_paged_attn_desc* d, int* status) {
  *status = CMPX_ERR_INVALID_ARGUMENT;
  if (!d || !d->q || !d->o || d->batch < 0 || d->heads < 0 || !std::isfinite(scale_log2(d))) return "none";
  if (!paged_cache_ok(d->cache, d->batch) || d->heads % d->cache.heads_kv != 0) return "none";
  *status = CMPX_ERR_UNSUPPORTED_DTYPE;
  if (d->dtype != CMPX_F32 && d->dtype != CMPX_F16 && d->dtype != CMPX_BF16) return "none";
  *status = paged_cache_limits(d->cache, d->dtype);
  if (*status != CMPX_OK) return "none";
  const int64_t es = elt_size(d->dtype);
  *status = CMPX_ERR_MISALIGNED;
  if (reinterpret_cast<uintptr_t>(d->q) % 16 || reinterpret_cast<uintptr_t>(d->o) % 16) return "none";
  const int64_t extent[2] = {d->batch, d->heads};
  for (int i = 0; i < 2; ++i)  // (a single one's stride is never stepped)
    if (extent[i] > 1 && ((d->q_stride[i] * es) % 16 || (d->o_stride[i] * es) % 16)) return "none";
  *status = CMPX_ERR_UNSUPPORTED_SHAPE;
  if (d->heads > (1 << 20) || d->batch > (1 << 20) || d->batch * d->heads > (1ll << 31) - 65536) return "none";
  *status = CMPX_OK;
  switch (schedule(d, current_num_sms()).ranks) {
    case 0: return "paged_attn<equal shares, join>";
    case 1: return "paged_attn<one CTA per item>";
    default: return "paged_attn<cluster per item>";
  }
}

size_t paged_attn_workspace_bytes(const cmpx_paged_attn_desc* d, int num_sms) {
  int st;
  paged_attn_plan(d, &st);
  if (st != CMPX_OK || d->batch == 0 || d->heads == 0) return 0;
  return part_floats(d, schedule(d, num_sms)) * sizeof(float);
}

int launch_paged_attn(const cmpx_paged_attn_desc* d, const LaunchCtx& ctx) {
  const int es = elt_size(d->dtype);
  const cmpx_paged_cache& c = d->cache;
  const Schedule s = schedule(d, ctx.num_sms);
  const size_t floats = part_floats(d, s);
  if (floats && (!d->workspace || d->workspace_bytes < floats * sizeof(float) ||
                 reinterpret_cast<uintptr_t>(d->workspace) % 16 != 0))
    return CMPX_ERR_WORKSPACE;
  PagedArgs a{};
  a.q = static_cast<const uint8_t*>(d->q);
  a.o = static_cast<uint8_t*>(d->o);
  a.q_sb = d->q_stride[0] * es;
  a.q_sh = d->q_stride[1] * es;
  a.o_sb = d->o_stride[0] * es;
  a.o_sh = d->o_stride[1] * es;
  a.kc = static_cast<const uint8_t*>(c.k);
  a.vc = static_cast<const uint8_t*>(c.v);
  a.kc_sp = c.k_stride[0] * es;
  a.kc_sh = c.k_stride[1] * es;
  a.kc_st = c.k_stride[2] * es;
  a.vc_sp = c.v_stride[0] * es;
  a.vc_sh = c.v_stride[1] * es;
  a.vc_st = c.v_stride[2] * es;
  a.table = c.table;
  a.lengths = c.lengths;
  a.table_stride = c.table_stride;
  a.capacity = static_cast<int>(c.table_width * c.page_size);
  a.num_pages = static_cast<int>(c.num_pages);
  a.page = make_fast_div(static_cast<uint32_t>(c.page_size));
  a.batch = static_cast<int>(d->batch);
  a.heads = static_cast<int>(d->heads);
  a.heads_kv = static_cast<int>(c.heads_kv);
  a.group = a.heads / a.heads_kv;
  a.item_heads = s.item_heads;
  a.items_per_head = s.items_per_head;
  a.head_dim = static_cast<int>(c.head_dim);
  a.scale_log2 = scale_log2(d);
  a.workers = s.workers;
  a.flags = ctx.dev_flags;
  if (floats) {
    a.part_o = static_cast<float*>(d->workspace);
    a.part_ml = a.part_o + 2ull * s.workers * s.item_heads * c.head_dim;
  }
  const int st = d->dtype != CMPX_F32                    ? launch_paged_mma(a, d->dtype, s.ctas, s.ranks, s.wide, ctx)
                 : f32_mma(s.item_heads, c.head_dim) ? launch_paged_f32_mma(a, s.ctas, s.ranks, s.wide, ctx)
                                                     : launch_paged_f32(a, s.ctas, s.ranks, s.wide, ctx);
  if (st != CMPX_OK || s.ranks) return st;
  // The most partial results that a row can have: the longest sequence beside empty ones.
  const int64_t tiles = (static_cast<int64_t>(a.capacity) + kTile - 1) / kTile;
  const int64_t units = (tiles + kItemCost + (d->batch - 1) * (1 + kItemCost)) * (s.items / d->batch);
  const int64_t most = tiles / std::max<int64_t>(kShareMin, units / s.workers) + 2;
  if (d->dtype == CMPX_F32) return launch_join_dim<CMPX_F32>(a, most, ctx);
  if (d->dtype == CMPX_F16) return launch_join_dim<CMPX_F16>(a, most, ctx);
  return launch_join_dim<CMPX_BF16>(a, most, ctx);
}

}  // namespace cmpx
