// paged_schedule.cuh -- how the one-token attention over a paged cache is cut into equal shares, and
// what its kernels have in common: arguments, the walk over a share, and the partial results' places.
//
// An item is one sequence's keys for one group of query heads that share a key head.  Its keys are
// cut into tiles of kTile; an empty sequence counts one tile, so that somebody writes its zeros.  All items
// laid end to end, each with kItemCost units before its tiles for what an item costs whatever its
// length (the first loads' latency, the output), are cut into equal shares, one per warp: every
// warp has the same work, whether the lengths are alike or one sequence is a thousand times as long as
// the others, and the lengths are only read on the device.  A warp that has all of an item writes
// its output; otherwise it leaves a partial result (running maximum, sum and unnormalised output) in the
// workspace: slot 2w for an item that began before warp w's share, slot 2w + 1 for one that begins in
// it.  The join kernel finds an item's slots by the same arithmetic and adds them in a fixed order, so
// the result does not depend on timing.
#pragma once

#include <cuda_runtime.h>

#include "cmpx_internal.h"
#include "rowvec.cuh"

namespace cmpx {

constexpr int kTile = 16;      // keys per tile
constexpr int kItemCost = 3;   // an item's fixed cost, in tiles
constexpr int kShareMin = 6;   // units per warp at least, where there are more warps than work

struct PagedArgs {
  const uint8_t* q;
  uint8_t* o;
  int64_t q_sb, q_sh, o_sb, o_sh;                    // byte strides
  const uint8_t *kc, *vc;
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;  // byte strides over page, head, token
  const int32_t *table, *lengths;
  int64_t table_stride;
  int capacity;          // table_width * page_size
  int num_pages;
  FastDiv page;
  int batch, heads, heads_kv, group;  // group: query heads per key head
  int item_heads, items_per_head;     // query heads per item, items per key head
  int head_dim;
  float scale_log2;      // softmax scale * log2(e)
  int64_t workers;       // warps that have shares
  float* part_o;         // [slot][item_heads][head_dim]
  float* part_ml;        // [slot][item_heads][2]: maximum (in log2 units), sum
  unsigned int* flags;
};

// Keys of sequence b that the kernels look at: 0 .. capacity.  A longer length is reported by the
// kernel that meets it and makes the sequence's results NaN.
__device__ __forceinline__ int seq_len(const PagedArgs& a, int b, bool& beyond) {
  const int n = __ldg(a.lengths + b);
  beyond = n > a.capacity;
  return min(max(n, 0), a.capacity);
}
__device__ __forceinline__ int seq_tiles(const PagedArgs& a, int b) {
  bool beyond;
  return max(1, (seq_len(a, b, beyond) + kTile - 1) / kTile);
}

// Sum over the block (blockDim.x a multiple of 32, at most 1024), and the sum over the threads before
// this one.  Uses scratch[33]; ends with a barrier.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* scratch, int64_t* before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  int64_t base = 0, total = 0;
  for (int w = 0; w < warps; ++w) {
    const int64_t s = scratch[w];
    if (w < warp) base += s;
    total += s;
  }
  *before = base + incl - v;
  __syncthreads();
  return total;
}

// A warp's share: units [cur, end), the sequence that cur lies in and the units before that sequence.
struct Share {
  int64_t cur, end, before, slot;
  int b;
};

__device__ __forceinline__ int64_t share_units(int64_t total, int64_t workers) {
  const int64_t s = (total + workers - 1) / workers;
  return s < kShareMin ? kShareMin : s;
}
__device__ __forceinline__ int64_t seq_units(const PagedArgs& a, int b) {
  return static_cast<int64_t>(seq_tiles(a, b) + kItemCost) * (a.heads_kv * a.items_per_head);
}

// The share of this warp: worker warp * gridDim.x + blockIdx.x, so that little work spreads over the CTAs
// first.  scratch: 33 + 2 WARPS values of shared memory.
template <int WARPS>
__device__ __forceinline__ Share find_share(const PagedArgs& a, int64_t* scratch) {
  const int per = (a.batch + blockDim.x - 1) / blockDim.x;  // sequences per thread
  const int b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += seq_units(a, b);
  int64_t before;
  const int64_t total = block_scan(mine, scratch, &before);
  const int64_t share = share_units(total, a.workers);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int64_t cur = (static_cast<int64_t>(w) * gridDim.x + blockIdx.x) * share;
    if (cur >= before && cur < before + mine) {
      int64_t at = before;
      int b = b0;
      for (; b < b1 - 1; ++b) {
        const int64_t n = seq_units(a, b);
        if (cur < at + n) break;
        at += n;
      }
      scratch[33 + 2 * w] = at;
      scratch[34 + 2 * w] = b;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const int64_t worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
  Share s;
  s.cur = worker * share;
  s.end = min(total, s.cur + share);
  s.slot = 2 * worker;
  s.before = scratch[33 + 2 * warp];
  s.b = static_cast<int>(scratch[34 + 2 * warp]);
  return s;
}

// One stretch of a share: keys [key0, key1) of query heads [h0, h0 + nh) of sequence b, which read
// key head kvh; slot < 0: the whole item, its output is written directly.
struct Stretch {
  int b, kvh, h0, nh, key0, key1;
  int64_t slot;
  bool bad;    // the sequence's length is beyond the table
  bool empty;  // it has no keys
};

// One over a row's sum of weights: 0 of a sequence without keys.  Keys whose scores are all -inf (the only other
// way to no weight: the largest is 1) have no softmax: NaN.
__device__ __forceinline__ float inverse_sum(float sum, bool empty) {
  return sum != 0.f ? 1.f / sum : empty ? 0.f : __int_as_float(0x7fffffff);
}

__device__ __forceinline__ void stretch_heads(const PagedArgs& a, int item, Stretch& st) {
  st.kvh = item / a.items_per_head;
  const int g = (item - st.kvh * a.items_per_head) * a.item_heads;
  st.h0 = st.kvh * a.group + g;
  st.nh = min(a.item_heads, a.group - g);
}

// The next stretch of s; moves s behind it.  False when the share is done.
__device__ __forceinline__ bool next_stretch(const PagedArgs& a, Share& s, Stretch& st) {
  const int items = a.heads_kv * a.items_per_head;
  while (s.cur < s.end) {
    int units = seq_tiles(a, s.b) + kItemCost;
    while (s.cur >= s.before + static_cast<int64_t>(units) * items) {
      s.before += static_cast<int64_t>(units) * items;
      if (++s.b >= a.batch) return false;  // (lengths that were written meanwhile)
      units = seq_tiles(a, s.b) + kItemCost;
    }
    const int64_t off = s.cur - s.before;
    const int item = static_cast<int>(off / units);
    const int unit0 = static_cast<int>(off - static_cast<int64_t>(item) * units);
    const int unit1 = static_cast<int>(min(static_cast<int64_t>(units), unit0 + (s.end - s.cur)));
    s.cur += unit1 - unit0;
    const int tiles = units - kItemCost;
    const int tile0 = max(unit0 - kItemCost, 0), tile1 = unit1 - kItemCost;
    if (tile1 <= tile0) continue;  // the share ends before the item's first tile
    st.b = s.b;
    stretch_heads(a, item, st);
    const int n = seq_len(a, st.b, st.bad);
    st.empty = n == 0;
    st.key0 = min(n, tile0 * kTile);
    st.key1 = tile1 == tiles ? n : tile1 * kTile;
    st.slot = tile0 == 0 && tile1 == tiles ? -1 : s.slot + (tile0 == 0 ? 1 : 0);
    return true;
  }
  return false;
}

// Part `rank` of `ranks` of an item's keys as one stretch (a CTA or a cluster of CTAs per item, no join).
__device__ __forceinline__ Stretch whole_item(const PagedArgs& a, int64_t index, int rank, int ranks) {
  const int items = a.heads_kv * a.items_per_head;
  Stretch st;
  st.b = static_cast<int>(index / items);
  stretch_heads(a, static_cast<int>(index - static_cast<int64_t>(st.b) * items), st);
  const int n = seq_len(a, st.b, st.bad);
  const int64_t tiles = (n + kTile - 1) / kTile;
  st.empty = n == 0;
  st.key0 = static_cast<int>(tiles * rank / ranks) * kTile;
  st.key1 = min(n, static_cast<int>(tiles * (rank + 1) / ranks) * kTile);
  st.slot = -1;
  return st;
}

// A warp's pipeline over the keys of a stretch: a ring of SLOTS slots in shared memory with KEYS keys and their values
// each, ROW bytes a row, filled by 16-byte cp.async.  With HALVES a slot has the keys or the values alone: more
// instructions, but the ring needs less room for the same loads in flight (fp16 heads of 256, 8 warps per SM
// instead of 4: 36 us instead of 49 over 200 MB; heads of 128, which have the room, 40 instead of 39).  The rows
// are found through the page table one by one (a page may end inside a slot).  Chunk c (16 bytes) of row r lies at
// c ^ turn_of(r).  SWIZZLE 1, for ldmatrix: 8 rows' chunks of one column lie in different banks.  2, for a
// lane's own 16-byte loads: so do 4 neighbouring chunks of rows 2 i and 2 i + 1, and 2 neighbouring chunks of 4
// rows of one parity.  Keys behind the stretch, pages that do not exist and columns behind head_dim are filled with zeros.
template <int ROW, int KEYS, int SLOTS, int SWIZZLE, bool HALVES = false>
struct KeyPipe {
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int HALF = KEYS * ROW;
  static constexpr int SLOT = HALVES ? HALF : 2 * HALF;
  static constexpr int BYTES = SLOTS * SLOT;  // per warp

  static __device__ __forceinline__ int turn_of(int r) {
    if (SWIZZLE == 1) return ROW % 128 == 0 ? r & 7 : (r >> 1) & 3;  // (64 bytes over: odd rows begin 4 chunks on)
    return SWIZZLE == 0 ? 0 : (r & 2) | (((r >> 2) ^ r) & 1) << 2;
  }

  const PagedArgs& a;
  const int32_t* table;
  const uint8_t *kb, *vb;
  int key0, key1, row_chunks;
  uint32_t buf;
  int count, step;          // the stretch's sub-tiles of KEYS keys, and from one of this warp's to its next
  int next;                 // sub-tile that is loaded next
  int slot_in, slot_out;    // slots that are filled and read next
  int id_ahead, row_ahead;  // page and row of this lane's key of the next sub-tile
  int id, row;              // and of the one that is being loaded
  bool ok, one_page, bad;   // its page exists; all its keys lie in one page

  __device__ __forceinline__ KeyPipe(const PagedArgs& args, uint32_t buffers, int row_bytes)
      : a(args), row_chunks(row_bytes / 16), buf(buffers) {}

  __device__ __forceinline__ void look_up(int i) {
    const int t = key0 + i * KEYS + (threadIdx.x & 31) % KEYS;
    id_ahead = 0;
    row_ahead = 0;
    if (t < key1) {
      const uint32_t page = fast_div(t, a.page);
      row_ahead = t - page * a.page.d;
      id_ahead = __ldg(table + page);
    }
  }
  // Begins a stretch with this warp's sub-tiles first, first + every, ...: fills all slots but one.
  __device__ __forceinline__ void begin(const Stretch& st, int first, int every) {
    table = a.table + st.b * a.table_stride;
    kb = a.kc + st.kvh * a.kc_sh;
    vb = a.vc + st.kvh * a.vc_sh;
    key0 = st.key0;
    key1 = st.key1;
    bad = st.bad;
    count = (key1 - key0 + KEYS - 1) / KEYS;
    step = every;
    next = first;
    slot_in = slot_out = 0;
    look_up(first);
#pragma unroll
    for (int j = 0; j < SLOTS - 1; ++j)
      if (HALVES && j % 2 == 1) load<false, true>();
      else load<true, !HALVES>();
  }
  // Waits for the keys (then the values) of a sub-tile, starts the loads that are SLOTS - 1 slots ahead in the place
  // that was read before, and returns their offset in the warp's buffers.
  template <bool K>
  __device__ __forceinline__ int take() {
    if (!HALVES && !K) return (slot_out == 0 ? SLOTS - 1 : slot_out - 1) * SLOT + HALF;
    cp_async_wait<SLOTS - 2>();
    __syncwarp();  // this slot is filled, and everybody is done with the one before it
    if (HALVES) load<K == (SLOTS % 2 == 1), K != (SLOTS % 2 == 1)>();
    else load<true, true>();
    const int at = slot_out * SLOT;
    slot_out = slot_out + 1 == SLOTS ? 0 : slot_out + 1;
    return at;
  }
  // Starts the loads of the next sub-tile's keys, its values, or both (nothing behind the last); closes the group.
  template <bool K, bool V>
  __device__ __forceinline__ void load() {
    const int lane = threadIdx.x & 31;
    if (next < count) {
      if (K) {
        const int t0 = key0 + next * KEYS;
        id = id_ahead;
        row = row_ahead;
        look_up(next + step);
        const bool there = t0 + lane % KEYS < key1;
        ok = id >= 0 && id < a.num_pages;
        if (!ok && there) bad = true;
        ok = ok && there;
        one_page = t0 + KEYS <= key1 && __shfl_sync(0xffffffffu, row + KEYS <= static_cast<int>(a.page.d) && ok ? 1 : 0, 0);
      }
      const uint32_t base = buf + slot_in * SLOT;
      constexpr int V_AT = K ? HALF : 0;
      if (one_page) {
        const int id0 = __shfl_sync(0xffffffffu, id, 0), row0 = __shfl_sync(0xffffffffu, row, 0);
        const uint8_t* const kp = kb + id0 * a.kc_sp + row0 * a.kc_st;
        const uint8_t* const vp = vb + id0 * a.vc_sp + row0 * a.vc_st;
#pragma unroll
        for (int j = 0; j < KEYS * CHUNKS / 32; ++j) {
          const int idx = j * 32 + lane, r = idx / CHUNKS, ch = idx % CHUNKS;
          const int bytes = ch < row_chunks ? 16 : 0;
          const uint32_t dst = base + r * ROW + ((ch ^ turn_of(r)) << 4);
          if (K) cp_async16(dst, kp + r * a.kc_st + (bytes ? ch * 16 : 0), bytes);
          if (V) cp_async16(dst + V_AT, vp + r * a.vc_st + (bytes ? ch * 16 : 0), bytes);
        }
      } else {
        const int64_t ko = ok ? id * a.kc_sp + row * a.kc_st : -1, vo = ok ? id * a.vc_sp + row * a.vc_st : -1;
#pragma unroll
        for (int j = 0; j < KEYS * CHUNKS / 32; ++j) {
          const int idx = j * 32 + lane, r = idx / CHUNKS, ch = idx % CHUNKS;
          const uint32_t dst = base + r * ROW + ((ch ^ turn_of(r)) << 4);
          if (K) {
            const int64_t kr = __shfl_sync(0xffffffffu, ko, r);
            const bool there = kr >= 0 && ch < row_chunks;
            cp_async16(dst, there ? kb + kr + ch * 16 : a.q, there ? 16 : 0);
          }
          if (V) {
            const int64_t vr = __shfl_sync(0xffffffffu, vo, r);
            const bool there = vr >= 0 && ch < row_chunks;
            cp_async16(dst + V_AT, there ? vb + vr + ch * 16 : a.q, there ? 16 : 0);
          }
        }
      }
    }
    if (V) next += step;
    slot_in = slot_in + 1 == SLOTS ? 0 : slot_in + 1;
    cp_async_commit();
  }
};

// Joins the results of the WARPS warps of each of a cluster's CTAs, which all have the same item: outputs
// sm_o [warp][ROWS][DP], maxima and sums sm_ml [warp][ROWS].  First each CTA its warps', in the place of the first
// warp's (cta_ml [ROWS]: maxima and sums), then every CTA its part of the cluster's.  store(h, d, x, y) gets two
// neighbouring values of head h.
template <int WARPS, int ROWS, int DP, typename Store>
__device__ __forceinline__ void join_cluster(int nh, int head_dim, bool empty, float* sm_o, const float2* sm_ml, float2* cta_ml,
                                             Store store) {
  const int ranks = cluster_size();
  __syncthreads();
  for (int x = threadIdx.x; x < nh * (DP / 2); x += blockDim.x) {
    const int h = x / (DP / 2), d = 2 * (x - h * (DP / 2));
    if (d >= head_dim) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_ml[w * ROWS + h].x);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 ml = sm_ml[w * ROWS + h], v = *reinterpret_cast<const float2*>(sm_o + (w * ROWS + h) * DP + d);
      const float weight = ex2_approx(ml.x - base);
      sum = fmaf(weight, ml.y, sum);
      x0 = fmaf(weight, v.x, x0);
      x1 = fmaf(weight, v.y, x1);
    }
    if (ranks == 1) {
      const float inv = inverse_sum(sum, empty);
      store(h, d, x0 * inv, x1 * inv);
    } else {
      *reinterpret_cast<float2*>(sm_o + h * DP + d) = make_float2(x0, x1);  // read by this thread alone so far
      if (d == 0) cta_ml[h] = make_float2(top, sum);
    }
  }
  if (ranks == 1) return;
  cluster_sync();
  for (int x = cluster_rank() * blockDim.x + threadIdx.x; x < nh * (DP / 2); x += ranks * blockDim.x) {
    const int h = x / (DP / 2), d = 2 * (x - h * (DP / 2));
    if (d >= head_dim) continue;
    constexpr int MOST = 8;
    float2 ml[MOST], v[MOST];
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < MOST; ++r) {
      ml[r] = make_float2(-INFINITY, 0.f);
      v[r] = make_float2(0.f, 0.f);
      if (r < ranks) {
        ml[r] = cluster_load_f2(smem_u32(cta_ml + h), r);
        v[r] = cluster_load_f2(smem_u32(sm_o + h * DP + d), r);
      }
    }
#pragma unroll
    for (int r = 0; r < MOST; ++r) top = fmaxf(top, ml[r].x);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int r = 0; r < MOST; ++r) {
      const float weight = ex2_approx(ml[r].x - base);
      sum = fmaf(weight, ml[r].y, sum);
      x0 = fmaf(weight, v[r].x, x0);
      x1 = fmaf(weight, v[r].y, x1);
    }
    const float inv = inverse_sum(sum, empty);
    store(h, d, x0 * inv, x1 * inv);
  }
  cluster_sync();  // nobody leaves while its results are read
}

// Launches a kernel over whole items with `ranks` CTAs per item.
template <typename Kernel>
int launch_whole(Kernel kernel, const PagedArgs& a, int64_t ctas, int ranks, int threads, int smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

// The kernels over the keys: fp16 / bf16 items of up to 16 heads (paged_attn_mma.cu), fp32 items of up to 8
// (paged_attn_f32.cu, paged_attn_f32_mma.cu).  ranks: CTAs per whole item, 0 for equal shares; wide: whole items whose
// CTAs have an SM each to themselves, with the warps of all that would share it.
struct PagedShape {
  int ctas, warps;  // CTAs per SM, warps per CTA
};
PagedShape paged_mma_shape(int64_t head_dim);
PagedShape paged_f32_shape();
PagedShape paged_f32_mma_shape(int64_t head_dim);
int launch_paged_mma(const PagedArgs& a, int dtype, int ctas, int ranks, bool wide, const LaunchCtx& ctx);
int launch_paged_f32(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx);
int launch_paged_f32_mma(const PagedArgs& a, int ctas, int ranks, bool wide, const LaunchCtx& ctx);

// Programmatic dependent launch: the join kernel starts while the main kernel runs, reads the
// lengths, and waits here for the main kernel's results.
__device__ __forceinline__ void pdl_allow_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace cmpx
