// paged_schedule.cuh -- how the one-token attention over a paged cache is cut into equal shares, and
// what its kernels share: arguments, the walk over a share, and the partial results' places.
//
// An item is one sequence's keys for one group of query heads that share a key head.  Items are
// cut into tiles of kTile keys and laid end to end (sequence, then item in the sequence); an empty
// sequence counts one tile, so that somebody writes its zeros.  CTA c takes the tiles
// [c * share, (c + 1) * share), whatever items they belong to: every CTA has the same work, whether
// the lengths are alike or one sequence is a thousand times as long as the others, and the lengths
// are only read on the device.  A CTA that has all of an item writes its output; otherwise
// it leaves a partial result (running maximum, sum and unnormalised output) in the workspace: slot
// 2c for an item that began before the CTA's share, slot 2c + 1 for one that begins in it.  The join
// kernel finds an item's slots by the same arithmetic and adds them in the order of the CTAs, so the
// result does not depend on timing.
#pragma once

#include <cuda_runtime.h>

#include "cmpx_internal.h"
#include "rowvec.cuh"

namespace cmpx {

constexpr int kTile = 64;        // keys per tile
constexpr int kShareMin = 2;     // tiles per CTA at least, where there are more CTAs than work

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
  int whole_items;       // 1: CTA c has item c and there is no join
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

// A CTA's share: tiles [cur, end) and the sequence that cur lies in, with the tiles before it.
struct Share {
  int64_t cur, end, before;
  int b;
};

__device__ __forceinline__ int64_t share_tiles(int64_t total, int ctas) {
  const int64_t s = (total + ctas - 1) / ctas;
  return s < kShareMin ? kShareMin : s;
}

// Finds CTA blockIdx.x's share.  scratch: 33 + 2 values of shared memory.
__device__ __forceinline__ Share find_share(const PagedArgs& a, int64_t* scratch) {
  const int per = (a.batch + blockDim.x - 1) / blockDim.x;  // sequences per thread
  const int64_t items = static_cast<int64_t>(a.heads_kv) * a.items_per_head;
  const int b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += seq_tiles(a, b) * items;
  int64_t before;
  const int64_t total = block_scan(mine, scratch, &before);
  const int64_t share = share_tiles(total, gridDim.x);
  Share s;
  s.cur = blockIdx.x * share;
  s.end = min(total, s.cur + share);
  if (s.cur >= before && s.cur < before + mine) {
    int b = b0;
    for (; b < b1 - 1; ++b) {
      const int64_t n = seq_tiles(a, b) * items;
      if (s.cur < before + n) break;
      before += n;
    }
    scratch[33] = before;
    scratch[34] = b;
  }
  __syncthreads();
  s.before = scratch[33];
  s.b = static_cast<int>(scratch[34]);
  return s;
}

// One stretch of a share: keys [key0, key1) of query heads [h0, h0 + nh) of sequence b, which read
// key head kvh; slot < 0: the whole item, its output is written directly.
struct Stretch {
  int b, kvh, h0, nh, key0, key1;
  int64_t slot;
  bool bad;  // the sequence's length is beyond the table
};

__device__ __forceinline__ void stretch_heads(const PagedArgs& a, int item, Stretch& st) {
  st.kvh = item / a.items_per_head;
  const int g = (item - st.kvh * a.items_per_head) * a.item_heads;
  st.h0 = st.kvh * a.group + g;
  st.nh = min(a.item_heads, a.group - g);
}

// The stretch that begins at s.cur; moves s behind it.  False when the share is done.
__device__ __forceinline__ bool next_stretch(const PagedArgs& a, Share& s, Stretch& st) {
  if (s.cur >= s.end) return false;
  const int64_t items = static_cast<int64_t>(a.heads_kv) * a.items_per_head;
  int tiles = seq_tiles(a, s.b);
  while (s.cur >= s.before + tiles * items) {
    s.before += tiles * items;
    tiles = seq_tiles(a, ++s.b);
  }
  const int64_t off = s.cur - s.before;
  const int item = static_cast<int>(off / tiles);
  const int tile0 = static_cast<int>(off - static_cast<int64_t>(item) * tiles);
  const int tile1 = static_cast<int>(min(static_cast<int64_t>(tiles), tile0 + (s.end - s.cur)));
  s.cur += tile1 - tile0;
  st.b = s.b;
  stretch_heads(a, item, st);
  const int n = seq_len(a, st.b, st.bad);
  st.key0 = min(n, tile0 * kTile);
  st.key1 = tile1 == tiles ? n : tile1 * kTile;
  st.slot = tile0 == 0 && tile1 == tiles ? -1 : 2 * static_cast<int64_t>(blockIdx.x) + (tile0 == 0 ? 1 : 0);
  return true;
}

// Item blockIdx.x as one stretch (whole_items).
__device__ __forceinline__ Stretch whole_item(const PagedArgs& a, int64_t index) {
  const int items = a.heads_kv * a.items_per_head;
  Stretch st;
  st.b = static_cast<int>(index / items);
  stretch_heads(a, static_cast<int>(index - static_cast<int64_t>(st.b) * items), st);
  st.key0 = 0;
  st.key1 = seq_len(a, st.b, st.bad);
  st.slot = -1;
  return st;
}

// Programmatic dependent launch: the join kernel starts while the main kernel runs, reads the
// lengths, and waits here for the main kernel's results.
__device__ __forceinline__ void pdl_allow_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace cmpx
