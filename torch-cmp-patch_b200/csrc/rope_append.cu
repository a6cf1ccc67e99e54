// rope_append.cu -- rotary positions (forward and gradient) and the append of new keys and values
// to a paged cache with that rotation on the way, fp16 / bf16 / fp32, B200 sm_100a.
//
// Pair j of a row turns by angle = position[axis(j)] * freqs[j]:
//   (a, b) -> (a cos - b sin, a sin + b cos),   gradient: the same with -angle.
// Both operators are one kernel: a thread owns one chunk (VEC pairs, or 2 VEC values that pass
// through) of one token, computes the chunk's cos and sin once and walks over the heads: the query
// heads, then (append) the key heads into the cache, then the value heads, copied.
//
// What bounds it: the bytes, each value read once and written once, as long as a thread serves several
// heads with its cos and sin.  Rotation alone streams best with the loads of two heads at a time and four blocks
// per SM ([2, 32, 8192, 128] bf16, 268 MB: 46 us; 48 with four heads and two blocks); the append, whose
// addresses take more registers, with four heads and two blocks (4 x 2048 tokens, 16 heads of 64, fp16, 71 MB:
// 16.6 us; 18.9 with two and four).
// The angle is reduced in fp64 (1e6 radians in fp32 are off by 0.06) to within an eighth of a turn, where
// short Taylor sums of sine and cosine are exact to fp32 (below 2^50 radians: turn()).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "cmpx_internal.h"
#include "rowvec.cuh"

namespace cmpx {
namespace {

constexpr int kThreads = 256;
// Heads whose loads a thread issues together, and blocks per SM.
constexpr int jobs_at_once(bool append) { return append ? 4 : 2; }
constexpr int blocks_per_sm(bool append) { return append ? 2 : 4; }
constexpr int kMaxHeadDim = 256;

struct Rows {  // [batch, heads, len, head_dim] bytes
  const uint8_t* p;
  int64_t sb, sh, sl;  // byte strides
};

struct RopeArgs {
  Rows q, k, v;          // inputs (k, v: append only)
  uint8_t* qo;           // turned queries
  int64_t qo_sb, qo_sh, qo_sl;
  uint8_t *kc, *vc;      // caches, byte strides over page, head, token
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  const int32_t *table, *lengths, *new_lengths;
  int64_t table_stride;
  int table_width, num_pages;
  FastDiv page;
  int batch, len, heads, heads_kv, head_dim;
  const void* pos;
  const float* freqs;
  int64_t ps_axis, ps_batch, ps_tok;
  int pos_kind, pairs, axes, interleaved;
  int sec_end[CMPX_ROPE_MAX_AXES];
  float sign;            // -1: turn back
  int chunks, jobs_per_block;
  unsigned int* flags;
};

__device__ __forceinline__ double load_pos(const RopeArgs& a, int axis, int b, int l, int place) {
  if (a.pos_kind == CMPX_POS_NONE) return static_cast<double>(place);
  const int64_t i = axis * a.ps_axis + b * a.ps_batch + l * a.ps_tok;
  if (a.pos_kind == CMPX_POS_I32) return static_cast<double>(static_cast<const int32_t*>(a.pos)[i]);
  if (a.pos_kind == CMPX_POS_I64) return static_cast<double>(static_cast<const int64_t*>(a.pos)[i]);
  return static_cast<double>(static_cast<const float*>(a.pos)[i]);
}

// cos and sin of pos * freq.  pos * 2 / pi, times freq, is the angle in quarter turns: adding 1.5 * 2^52 rounds it to
// a whole number, whose last two bits, now the sum's, are the quadrant; the rest, at most half a quarter turn, goes to
// the Taylor sums up to x^9 / 9! and x^10 / 10! (the next terms are below 2^-29 there).  2 / pi and the product
// with it are the sums of two doubles each: what the first leaves over, 2^-53 of the angle, passes an fp32 step from 2^28
// radians on.  With it the angle is exact to fp32 below 2^50, where the rounding ends.
__device__ __forceinline__ void turn(double pos, float freq, float& c, float& s) {
  constexpr double kRound = 6755399441055744.0, kTwoOverPi = 0.6366197723675814, kTwoOverPiRest = -3.935735335036497e-17;
  const double f = static_cast<double>(freq);
  const double quarters = pos * kTwoOverPi, over = fma(pos, kTwoOverPiRest, fma(pos, kTwoOverPi, -quarters));
  const double sum = fma(quarters, f, kRound);
  const int quad = __double2loint(sum) & 3;
  const float x = static_cast<float>(fma(over, f, fma(quarters, f, -(sum - kRound))) * 1.57079632679489661923);
  const float x2 = x * x;
  const float sine = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), x);
  const float cosine =
      fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const float cc = quad & 1 ? sine : cosine, ss = quad & 1 ? cosine : sine;
  c = quad == 1 || quad == 2 ? -cc : cc;
  s = quad & 2 ? -ss : ss;
}

template <int DT, int VB, bool APPEND>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(APPEND)) rope_append_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int ES = elt_size(DT);
  constexpr int VEC = VB / ES, kJobsAtOnce = jobs_at_once(APPEND);
  const int tokens_per_block = kThreads / a.chunks;
  const int tok = threadIdx.x / a.chunks;
  const int c = threadIdx.x - tok * a.chunks;
  const uint32_t t = blockIdx.x * tokens_per_block + tok;  // batch * len is below 2^31 - 65536
  if (tok >= tokens_per_block || t >= static_cast<uint32_t>(a.batch) * static_cast<uint32_t>(a.len)) return;
  const int b = static_cast<int>(t / static_cast<uint32_t>(a.len)), l = static_cast<int>(t - static_cast<uint32_t>(b) * a.len);

  const int rot_chunks = a.pairs / VEC;
  const bool turned = c < rot_chunks;
  // the chunk's two vectors, as byte offsets in a row
  const int lo_e = turned ? (a.interleaved ? 2 * c * VEC : c * VEC) : 2 * a.pairs + (c - rot_chunks) * 2 * VEC;
  const int hi_e = turned && !a.interleaved ? a.pairs + c * VEC : lo_e + VEC;
  const bool has_hi = hi_e < a.head_dim;
  const int lo = lo_e * ES, hi = hi_e * ES;

  int place = 0;
  bool there = true;            // not a padding row
  int64_t k_at = -1, v_at = -1; // the slot's byte offsets in the caches (-1: not stored)
  if (APPEND) {
    const int fresh = a.new_lengths ? min(max(__ldg(a.new_lengths + b), 0), a.len) : a.len;
    there = l < fresh;
    if (there) {
      const int64_t at = static_cast<int64_t>(__ldg(a.lengths + b)) - fresh + l;
      place = static_cast<int>(at);
      bool ok = at >= 0;
      if (ok) {
        const uint32_t slot = static_cast<uint32_t>(at);
        const uint32_t page = fast_div(slot, a.page);
        ok = page < static_cast<uint32_t>(a.table_width);
        if (ok) {
          const int id = __ldg(a.table + b * a.table_stride + page);
          ok = id >= 0 && id < a.num_pages;
          if (ok) {
            const int row = static_cast<int>(slot - page * a.page.d);
            k_at = id * a.kc_sp + row * a.kc_st;
            v_at = id * a.vc_sp + row * a.vc_st;
          }
        }
      }
      if (!ok) atomicOr(a.flags, CMPX_DEVFLAG_BAD_PAGE);
    }
  }

  float cs[VEC], sn[VEC];
  if (turned && there) {
    double pos[CMPX_ROPE_MAX_AXES];
#pragma unroll
    for (int x = 0; x < CMPX_ROPE_MAX_AXES; ++x) pos[x] = x < a.axes ? load_pos(a, x, b, l, place) : 0.0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int j = c * VEC + i;
      double p = pos[0];
#pragma unroll
      for (int x = 1; x < CMPX_ROPE_MAX_AXES; ++x)
        if (x < a.axes && j >= a.sec_end[x - 1]) p = pos[x];
      turn(p, __ldg(a.freqs + j), cs[i], sn[i]);
      sn[i] *= a.sign;
    }
  }

  const int jobs = APPEND ? a.heads + 2 * a.heads_kv : a.heads;
  const int first = blockIdx.y * a.jobs_per_block;
  const int last = min(jobs, first + a.jobs_per_block);
  for (int j0 = first; j0 < last; j0 += kJobsAtOnce) {
    RawVec<VB> x0[kJobsAtOnce], x1[kJobsAtOnce];
    uint8_t* dst[kJobsAtOnce];
#pragma unroll
    for (int u = 0; u < kJobsAtOnce; ++u) {
      const int j = j0 + u;
      const uint8_t* src = nullptr;
      dst[u] = nullptr;
      if (j < last) {
        if (!APPEND || j < a.heads) {
          src = a.q.p + b * a.q.sb + j * a.q.sh + l * a.q.sl;
          dst[u] = a.qo + b * a.qo_sb + j * a.qo_sh + l * a.qo_sl;
        } else if (k_at >= 0) {
          const int h = j - a.heads;
          if (h < a.heads_kv) {
            src = a.k.p + b * a.k.sb + h * a.k.sh + l * a.k.sl;
            dst[u] = a.kc + k_at + h * a.kc_sh;
          } else {
            src = a.v.p + b * a.v.sb + (h - a.heads_kv) * a.v.sh + l * a.v.sl;
            dst[u] = a.vc + v_at + (h - a.heads_kv) * a.vc_sh;
          }
        }
      }
      if (dst[u]) {
        x0[u] = *reinterpret_cast<const RawVec<VB>*>(src + lo);
        if (has_hi) x1[u] = *reinterpret_cast<const RawVec<VB>*>(src + hi);
      }
    }
#pragma unroll
    for (int u = 0; u < kJobsAtOnce; ++u) {
      if (!dst[u]) continue;
      const bool value = APPEND && j0 + u >= a.heads + a.heads_kv;
      if (turned && there && !value) {
        float f[2 * VEC], g[2 * VEC];
        unpack_vec<DT, VB>(x0[u], f);
        unpack_vec<DT, VB>(x1[u], f + VEC);
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            g[2 * i] = f[2 * i] * cs[i] - f[2 * i + 1] * sn[i];
            g[2 * i + 1] = f[2 * i] * sn[i] + f[2 * i + 1] * cs[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            g[i] = f[i] * cs[i] - f[VEC + i] * sn[i];
            g[VEC + i] = f[i] * sn[i] + f[VEC + i] * cs[i];
          }
        }
        x0[u] = pack_vec<DT, VB>(g);
        x1[u] = pack_vec<DT, VB>(g + VEC);
      }
      *reinterpret_cast<RawVec<VB>*>(dst[u] + lo) = x0[u];
      if (has_hi) *reinterpret_cast<RawVec<VB>*>(dst[u] + hi) = x1[u];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------

bool rotation_ok(const cmpx_rotation& r, int64_t head_dim, bool place_allowed) {
  if (r.pairs < 0 || 2 * static_cast<int64_t>(r.pairs) > head_dim) return false;
  if (r.pairs == 0) return true;
  if (!r.freqs || r.axes < 1 || r.axes > CMPX_ROPE_MAX_AXES || (r.interleaved != 0 && r.interleaved != 1)) return false;
  if (r.pos_kind == CMPX_POS_NONE) {
    if (!place_allowed || r.axes != 1) return false;
  } else if (!r.positions || r.pos_kind < CMPX_POS_NONE || r.pos_kind > CMPX_POS_F32) {
    return false;
  }
  int at = 0;
  for (int x = 0; x < r.axes; ++x) {
    if (r.section_end[x] < at) return false;
    at = r.section_end[x];
  }
  return at == r.pairs;
}

// Rows of head_dim values: where they begin, how far apart they are along three dimensions, and how many there are.
struct RowLayout {
  const void* p;
  const int64_t* stride;  // elements
  int64_t extent[3];
};

// Whether all rows begin at multiples of unit bytes.  The stride of a dimension of one is never stepped: it may be odd.
bool rows_aligned(const RowLayout& r, int es, int unit) {
  if (reinterpret_cast<uintptr_t>(r.p) % unit != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (r.extent[i] > 1 && (r.stride[i] * es) % unit != 0) return false;
  return true;
}

// The widest vector (16, 4 bytes, or one element) that every row, the head and the two halves of the turned part
// allow.  Between them only the count of memory instructions differs: one 16-byte access against four or eight.
int pick_vec(int es, int64_t head_dim, int pairs, const RowLayout* rows, int n) {
  for (int unit : {16, 4}) {
    if (unit < es) continue;
    bool ok = (head_dim * es) % unit == 0 && (static_cast<int64_t>(pairs) * es) % unit == 0;
    for (int i = 0; i < n && ok; ++i)
      if (rows[i].p) ok = rows_aligned(rows[i], es, unit);
    if (ok) return unit;
  }
  return es;
}

void fill_rotation(RopeArgs* a, const cmpx_rotation& r) {
  a->pos = r.positions;
  a->freqs = r.freqs;
  a->ps_axis = r.pos_stride[0];
  a->ps_batch = r.pos_stride[1];
  a->ps_tok = r.pos_stride[2];
  a->pos_kind = r.pos_kind;
  a->pairs = r.pairs;
  a->axes = r.pairs ? r.axes : 1;
  a->interleaved = r.pairs ? r.interleaved : 0;
  for (int x = 0; x < CMPX_ROPE_MAX_AXES; ++x) a->sec_end[x] = r.section_end[x];
  a->sign = 1.f;
}

template <bool APPEND>
int launch(RopeArgs& a, int dt, int vec_bytes, const LaunchCtx& ctx) {
  const int es = elt_size(dt), vec = vec_bytes / es;
  a.chunks = a.pairs / vec + (a.head_dim - 2 * a.pairs + 2 * vec - 1) / (2 * vec);
  a.flags = ctx.dev_flags;
  const int tokens_per_block = kThreads / a.chunks;
  const int64_t gx = (static_cast<int64_t>(a.batch) * a.len + tokens_per_block - 1) / tokens_per_block;
  const int jobs = APPEND ? a.heads + 2 * a.heads_kv : a.heads;
  // Heads per thread: as many as leave every SM its blocks once, so the trigonometry is shared where there is work
  // enough, and one where there is little; whole sets of those that are loaded together.
  const int64_t room = static_cast<int64_t>(blocks_per_sm(APPEND)) * ctx.num_sms, set = jobs_at_once(APPEND);
  int64_t per = std::min<int64_t>(std::max<int64_t>(1, gx * jobs / room), 16);
  if (per > 1) per = (per + set - 1) / set * set;
  per = std::max<int64_t>(per, (jobs + 65534) / 65535);  // the grid's limit
  a.jobs_per_block = static_cast<int>(std::min<int64_t>(per, jobs));
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>((jobs + a.jobs_per_block - 1) / a.jobs_per_block));
#define CMPX_ROPE(DT, VB) rope_append_kernel<DT, VB, APPEND><<<grid, kThreads, 0, ctx.stream>>>(a)
  if (dt == CMPX_F32) {
    if (vec_bytes == 16) CMPX_ROPE(CMPX_F32, 16);
    else CMPX_ROPE(CMPX_F32, 4);
  } else if (dt == CMPX_F16) {
    if (vec_bytes == 16) CMPX_ROPE(CMPX_F16, 16);
    else if (vec_bytes == 4) CMPX_ROPE(CMPX_F16, 4);
    else CMPX_ROPE(CMPX_F16, 2);
  } else {
    if (vec_bytes == 16) CMPX_ROPE(CMPX_BF16, 16);
    else if (vec_bytes == 4) CMPX_ROPE(CMPX_BF16, 4);
    else CMPX_ROPE(CMPX_BF16, 2);
  }
#undef CMPX_ROPE
  return cudaGetLastError() == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

bool dtype_ok(int dt) { return dt == CMPX_F32 || dt == CMPX_F16 || dt == CMPX_BF16; }

int rope_vec(const cmpx_rope_desc* d) {
  const RowLayout rows[2] = {{d->x, d->x_stride, {d->batch, d->heads, d->len}},
                             {d->y, d->y_stride, {d->batch, d->heads, d->len}}};
  return pick_vec(elt_size(d->dtype), d->head_dim, d->rot.pairs, rows, 2);
}

int append_vec(const cmpx_kv_append_desc* d) {
  const cmpx_paged_cache& c = d->cache;
  const RowLayout rows[6] = {{d->k, d->k_in_stride, {d->batch, c.heads_kv, d->len}},
                             {d->v, d->v_in_stride, {d->batch, c.heads_kv, d->len}},
                             {d->q, d->q_stride, {d->batch, d->heads, d->len}},
                             {d->q_out, d->q_out_stride, {d->batch, d->heads, d->len}},
                             {c.k, c.k_stride, {c.num_pages, c.heads_kv, c.page_size}},
                             {c.v, c.v_stride, {c.num_pages, c.heads_kv, c.page_size}}};
  return pick_vec(elt_size(d->dtype), c.head_dim, d->rot.pairs, rows, 6);
}

}  // namespace

bool paged_cache_ok(const cmpx_paged_cache& c, int64_t batch) {
  // what holds nothing may have no address
  if (((!c.k || !c.v) && c.num_pages != 0) || (!c.table && batch != 0 && c.table_width != 0) || (!c.lengths && batch != 0))
    return false;
  if (c.num_pages < 0 || c.page_size <= 0 || c.heads_kv <= 0 || c.head_dim <= 0 || c.table_width < 0) return false;
  if (batch > 1 && c.table_stride < 0) return false;
  for (int i = 0; i < 3; ++i)
    if (c.k_stride[i] < 0 || c.v_stride[i] < 0) return false;
  return true;
}

// Sizes that the kernels count in 32 bits, and the rows' alignment.
int paged_cache_limits(const cmpx_paged_cache& c, int dtype) {
  const int es = elt_size(dtype);
  const int64_t most = (1ll << 31) - 65536;
  if (c.head_dim > kMaxHeadDim || (c.head_dim * es) % 16 != 0) return CMPX_ERR_UNSUPPORTED_SHAPE;
  if (c.num_pages > most || c.page_size > most || c.heads_kv > 65535 || c.table_width > most ||
      c.table_width > most / c.page_size)
    return CMPX_ERR_UNSUPPORTED_SHAPE;
  for (const RowLayout& rows : {RowLayout{c.k, c.k_stride, {c.num_pages, c.heads_kv, c.page_size}},
                                RowLayout{c.v, c.v_stride, {c.num_pages, c.heads_kv, c.page_size}}})
    if (!rows_aligned(rows, es, 16)) return CMPX_ERR_MISALIGNED;
  return CMPX_OK;
}

const char* rope_plan(const cmpx_rope_desc* d, int* status) {
  *status = CMPX_ERR_INVALID_ARGUMENT;
  if (!d || !d->x || !d->y || d->batch < 0 || d->heads < 0 || d->len < 0 || d->head_dim <= 0) return "none";
  if (d->inverse != 0 && d->inverse != 1) return "none";
  if (!rotation_ok(d->rot, d->head_dim, false)) return "none";
  *status = CMPX_ERR_UNSUPPORTED_DTYPE;
  if (!dtype_ok(d->dtype)) return "none";
  *status = CMPX_ERR_UNSUPPORTED_SHAPE;
  if (d->head_dim > kMaxHeadDim || d->heads > (1 << 24) || d->batch > (1ll << 31) - 65536 ||
      d->len > (1ll << 31) - 65536 || (d->len > 0 && d->batch > ((1ll << 31) - 65536) / d->len))
    return "none";
  *status = CMPX_OK;
  const int es = elt_size(d->dtype), v = rope_vec(d);
  return v == 16 ? "rope<16-byte vectors>" : v > es ? "rope<4-byte vectors>" : "rope<single values>";
}

int launch_rope(const cmpx_rope_desc* d, const LaunchCtx& ctx) {
  const int es = elt_size(d->dtype);
  RopeArgs a{};
  a.q = Rows{static_cast<const uint8_t*>(d->x), d->x_stride[0] * es, d->x_stride[1] * es, d->x_stride[2] * es};
  a.qo = static_cast<uint8_t*>(d->y);
  a.qo_sb = d->y_stride[0] * es;
  a.qo_sh = d->y_stride[1] * es;
  a.qo_sl = d->y_stride[2] * es;
  a.batch = static_cast<int>(d->batch);
  a.len = static_cast<int>(d->len);
  a.heads = static_cast<int>(d->heads);
  a.head_dim = static_cast<int>(d->head_dim);
  fill_rotation(&a, d->rot);
  if (d->inverse) a.sign = -1.f;
  return launch<false>(a, d->dtype, rope_vec(d), ctx);
}

const char* kv_append_plan(const cmpx_kv_append_desc* d, int* status) {
  *status = CMPX_ERR_INVALID_ARGUMENT;
  if (!d || !d->k || !d->v || d->batch < 0 || d->heads < 0 || d->len < 0) return "none";
  if (d->heads > 0 && (!d->q || !d->q_out)) return "none";
  if (!paged_cache_ok(d->cache, d->batch) || !rotation_ok(d->rot, d->cache.head_dim, true)) return "none";
  *status = CMPX_ERR_UNSUPPORTED_DTYPE;
  if (!dtype_ok(d->dtype)) return "none";
  *status = paged_cache_limits(d->cache, d->dtype);
  if (*status != CMPX_OK) return "none";
  *status = CMPX_ERR_UNSUPPORTED_SHAPE;
  if (d->heads > (1 << 24) || d->batch > (1ll << 31) - 65536 || d->len > (1ll << 31) - 65536 ||
      (d->len > 0 && d->batch > ((1ll << 31) - 65536) / d->len))
    return "none";
  *status = CMPX_OK;
  const int es = elt_size(d->dtype), v = append_vec(d);
  return v == 16 ? "kv_append<16-byte vectors>" : v > es ? "kv_append<4-byte vectors>" : "kv_append<single values>";
}

int launch_kv_append(const cmpx_kv_append_desc* d, const LaunchCtx& ctx) {
  const int es = elt_size(d->dtype);
  const cmpx_paged_cache& c = d->cache;
  RopeArgs a{};
  a.q = Rows{static_cast<const uint8_t*>(d->q), d->q_stride[0] * es, d->q_stride[1] * es, d->q_stride[2] * es};
  a.k = Rows{static_cast<const uint8_t*>(d->k), d->k_in_stride[0] * es, d->k_in_stride[1] * es, d->k_in_stride[2] * es};
  a.v = Rows{static_cast<const uint8_t*>(d->v), d->v_in_stride[0] * es, d->v_in_stride[1] * es, d->v_in_stride[2] * es};
  a.qo = static_cast<uint8_t*>(d->q_out);
  a.qo_sb = d->q_out_stride[0] * es;
  a.qo_sh = d->q_out_stride[1] * es;
  a.qo_sl = d->q_out_stride[2] * es;
  a.kc = static_cast<uint8_t*>(c.k);
  a.vc = static_cast<uint8_t*>(c.v);
  a.kc_sp = c.k_stride[0] * es;
  a.kc_sh = c.k_stride[1] * es;
  a.kc_st = c.k_stride[2] * es;
  a.vc_sp = c.v_stride[0] * es;
  a.vc_sh = c.v_stride[1] * es;
  a.vc_st = c.v_stride[2] * es;
  a.table = c.table;
  a.lengths = c.lengths;
  a.new_lengths = d->new_lengths;
  a.table_stride = c.table_stride;
  a.table_width = static_cast<int>(c.table_width);
  a.num_pages = static_cast<int>(c.num_pages);
  a.page = make_fast_div(static_cast<uint32_t>(c.page_size));
  a.batch = static_cast<int>(d->batch);
  a.len = static_cast<int>(d->len);
  a.heads = static_cast<int>(d->heads);
  a.heads_kv = static_cast<int>(c.heads_kv);
  a.head_dim = static_cast<int>(c.head_dim);
  fill_rotation(&a, d->rot);
  return launch<true>(a, d->dtype, append_vec(d), ctx);
}

}  // namespace cmpx
