// linear_w4.cu -- linear layer with 4-bit weights and group scales for a few tokens, B200 sm_100a.
//
//   y[m, n] = sum_g scale[n, g] * sum_{k in group g} (code[n, k] - zero[n, g]) x[m, k]  (+ bias[n])
//
// code - zero is a whole number of at most 4 bits and a sign, exact in fp16 and bf16; the sums are
// fp32 and the scale multiplies a group's fp32 sum, so no weight is ever rounded.  fp32 activations
// go in as three bf16 parts (the leading, next and last 8 bits of the fraction: an exact sum), three
// products each, and their sums leave the tensor core every 32 k.
//
// The weights are read once, n k / 2 bytes, and that read bounds it while the tokens are few.  One CTA per SM
// has a run of tiles of 16 rows of W, and its warps have equal runs of the tiles' turns of 256 k laid
// end to end; mma.m16n8k16 multiplies the 16 rows with 8 NT tokens.  Every warp has its own pipeline
// of turns (2 KB each, cp.async) that runs on across tiles.  A tile that one warp has to itself is written from
// its registers; the others' parts are summed once, at the CTA's end, in a fixed order.
// A lane multiplies 16 k of a row that lie side by side, and the products run over k in the order that falls out
// of it: word j of the lanes tq = 0..3 holds k = 16 tq + 8 j .. + 7, and nibbles e and e + 4 of a word, which
// one mask isolates as the halves of a register, are a pair.  Activations of up to 64 KB (2 bytes a value, fp32's
// parts 6) are laid out in that order in shared memory once per CTA; others follow it with one byte
// permutation a register, and fp32's are cut again for every tile (1 x 16384 x 4096 fp32: 18.6 us from
// shared memory, 26 without).
// What bounds it beside the bytes: the lines that its loads touch (one a cycle), which is why eight lanes load
// 128 bytes of a row together and scales and zero points come for sets of turns, through a table in shared
// memory; then latency, at the four warps per scheduler that its registers leave.  Counted for 8 x 16384 x 4096 fp16, groups
// of 64: 32 instructions per 32 words of weights, of which 9 widen (1 shift, 4 masks, 4 subtractions; bf16: 3, 4, 4), 1
// multiplies and 3 load or store; the others are addresses, moves, selects and the scales' sums.  They take 54% of the issue
// slots of the 14.2 us that the SMs are busy, no unit more than 42% (ALU); a warp waits longest for its loads (a fifth
// of its cycles).  Starting and ending take 4.5 us more with cold caches.  Measured from a graph: that case 15.0 us (15.8 with a
// bias) for 37 MB (5.7 at the copy rate; 8 x 131072 x 4096: 72 us, 4.1 TB/s); 1 x 4096 x 4096 bf16: 6.1 us, most of it
// the launch and one pass through the pipeline.  16 x 16384 x 4096: 22.7 us; from the 17th token on the weights are read
// and widened again for every 16 (32: 42 us, 64: 79).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "cmpx_internal.h"
#include "rowvec.cuh"

namespace cmpx {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;    // rows of W per tile
constexpr int kChunk = 256;  // k per turn
constexpr int kStages = 3;   // turns in a warp's pipeline

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
  int chunks;                     // turns per tile
  int tiles_per_cta, tiles_rest;  // row tiles of a CTA; the first tiles_rest have one more
};

// Where groups may end: at multiples of 128 k, of 64 k, or of 32 k.
enum GroupKind { kGroup128 = 0, kGroup64 = 1, kGroup32 = 2 };

// c = (FIRST ? 0 : c) + A B
template <int DT, bool FIRST>
__device__ __forceinline__ void mma_w4(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  const float i0 = FIRST ? 0.f : c[0], i1 = FIRST ? 0.f : c[1], i2 = FIRST ? 0.f : c[2], i3 = FIRST ? 0.f : c[3];
  if constexpr (DT == CMPX_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(i0), "f"(i1), "f"(i2), "f"(i3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(i0), "f"(i1), "f"(i2), "f"(i3));
}

// The eight codes of a word minus a zero point as four 16-bit pairs: pair e = codes e and e + 4.  A code
// placed under the exponent of 128 (bf16) or 1024 (fp16) is that number plus the code; zp holds the number
// plus the zero point, twice.  fp16 has room for a nibble four bits higher, which saves shifts: 1024 + 16 c
// times 1/16 minus (64 + zero), one exact fma.
template <int DT>
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) {
  return ((DT == CMPX_F16 ? 0x6400u : 0x4300u) + z) * 0x10001u;
}

// (w & mask) | base as one instruction: given two constants the compiler takes two.
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t mask, uint32_t base) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(base));
  return d;
}

template <int DT>
__device__ __forceinline__ void codes_minus_zero(uint32_t w, uint32_t zero, uint32_t (&out)[4]) {
  if constexpr (DT == CMPX_F16) {
    const uint32_t v = w >> 8;
    const uint32_t c[4] = {mask_or(w, 0x000F000Fu, 0x64006400u), mask_or(w, 0x00F000F0u, 0x64006400u),
                           mask_or(v, 0x000F000Fu, 0x64006400u), mask_or(v, 0x00F000F0u, 0x64006400u)};
    const __half2 zp = *reinterpret_cast<const __half2*>(&zero);
    const __half2 zp16 = __hsub2(__half2half2(__ushort_as_half(0x6380)), zp);  // 960 - (1024 + z)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 h = *reinterpret_cast<const __half2*>(&c[e]);
      const __half2 d = e & 1 ? __hfma2(h, __half2half2(__ushort_as_half(0x2C00)), zp16) : __hsub2(h, zp);
      out[e] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {
    const __nv_bfloat162 zp = *reinterpret_cast<const __nv_bfloat162*>(&zero);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t c = mask_or(w >> (4 * e), 0x000F000Fu, 0x43004300u);
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), zp);
      out[e] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

// 8 activations: as loaded, and as PARTS sets of four pairs (e, e + 4).
template <int DT>
struct Activations {
  static constexpr int PARTS = DT == CMPX_F32 ? 3 : 1;
  static constexpr int VECS = DT == CMPX_F32 ? 2 : 1;
  uint4 v[VECS];

  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VECS; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void pairs(uint32_t (&p)[PARTS][4]) const {
    if constexpr (DT == CMPX_F32) {
      const uint32_t x[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
      uint32_t part[8][3];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // cut off, not rounded, so that the largest values do not become infinite (the permutation below
        // takes the upper halves); an infinite value has no rest
        const float f = __uint_as_float(x[e]);
        const float rest = fabsf(f) == INFINITY ? 0.f : f - __uint_as_float(x[e] & 0xFFFF0000u);
        part[e][0] = x[e];
        part[e][1] = __float_as_uint(rest);
        part[e][2] = __float_as_uint(rest - __uint_as_float(part[e][1] & 0xFFFF0000u));
      }
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[i][e] = __byte_perm(part[e][i], part[e + 4][i], 0x7632);
    } else {
      p[0][0] = __byte_perm(v[0].x, v[0].z, 0x5410);
      p[0][1] = __byte_perm(v[0].x, v[0].z, 0x7632);
      p[0][2] = __byte_perm(v[0].y, v[0].w, 0x5410);
      p[0][3] = __byte_perm(v[0].y, v[0].w, 0x7632);
    }
  }
};

// XS: all activations in shared memory.
template <int DT, int NT, int GK, bool XS>
struct W4Cfg {
  static constexpr int SUPER = GK == kGroup128 ? 4 : 2;                        // turns per table
  static constexpr int GROUPS = GK == kGroup128 ? 2 : GK == kGroup64 ? 4 : 8;  // columns of the table per turn
  static constexpr int COLS = SUPER * GROUPS;
  static constexpr int ENTRIES = COLS * kRows / 32;                            // per lane
  static constexpr int STAGE = kRows * kChunk / 2;
  static constexpr int TABLE = COLS * (kRows + 1) * 8;                         // bytes
  static constexpr int RED = NT * 8 * (kRows + 1);                             // floats of a part
  static constexpr int WARP = kStages * STAGE + TABLE + RED * 4;
  static constexpr int SMEM = kWarps * WARP;                                   // without the activations
  static constexpr int X_MOST = 65536;                                         // bytes of activations
  static_assert(SMEM + (XS ? X_MOST : 0) <= 227 * 1024 && RED * 4 <= STAGE, "shared memory; a part takes a buffer's place");
};

template <int DT, int NT, int GK, bool XS>
__global__ void __launch_bounds__(kThreads, 1) linear_w4_kernel(const __grid_constant__ W4Args a) {
  using C = W4Cfg<DT, NT, GK, XS>;
  constexpr int ES = elt_size(DT), GROUPS = C::GROUPS, COLS = C::COLS;
  // Where registers allow it, the two words of a quarter turn have sums of their own, and activations that are not in
  // shared memory are loaded a quarter turn ahead.  8 x 16384 x 4096 fp16 with groups of 64 spills 20 bytes with them and is
  // slower by 1.7 us of 15.  Without them, too, 26 of the 36 variants spill 4 to 80 bytes at the 128 registers that 16 warps
  // leave a thread: all for 9 to 16 tokens, and for 8 all but one for groups of 32 and three of the six for groups of 64.
  constexpr bool TWO = DT != CMPX_F32 && NT == 1 && GK == kGroup128;
  constexpr bool AHEAD = TWO && !XS;
  // fp32's sums leave the tensor core after every word (32 k), the low parts' added first: a sum in there is cut off,
  // not rounded, which over a group of 128 times three parts shows (8 x 1001 x 4096: 5.0e-7 off; like this 9.4e-8, plain fp32 sums
  // 2.6e-7; for 0 to 7% of the time).  One quarter turn at a time, where more would spill: none of its variants for 8
  // tokens does but one, of 4 bytes (16 x 16384 x 4096, groups of 128: 49 us, 54 with the four quarters unrolled).
  constexpr bool SHORT = DT == CMPX_F32;
  constexpr int kAtOnce = SHORT ? 1 : kChunk / 64;  // quarter turns
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  const int m0 = blockIdx.y * (8 * NT);
  uint8_t* const mine = smem + warp * C::WARP;
  const uint32_t buf = smem_u32(mine);
  float2* const table = reinterpret_cast<float2*>(mine + kStages * C::STAGE);
  constexpr int PARTS = Activations<DT>::PARTS;
  uint4* const x_all = reinterpret_cast<uint4*>(smem + C::SMEM);  // [quarter][word][part][token][tq]
  const int x_lanes = 4 * min(8 * NT, a.m - m0);
  // A warp's parts of tiles that it shares, [token][kRows + 1]: of its run's first tile in a place of its own,
  // of a later one, which is its last, where its first buffer was.
  auto part_of = [&](int w, bool later) {
    return reinterpret_cast<float*>(smem + w * C::WARP + (later ? 0 : kStages * C::STAGE + C::TABLE));
  };

  const int chunks = a.chunks;
  const int b = blockIdx.x;
  const int tile0 = b * a.tiles_per_cta + min(b, a.tiles_rest), tile1 = tile0 + a.tiles_per_cta + (b < a.tiles_rest ? 1 : 0);
  const int run = ((tile1 - tile0) * chunks + kWarps - 1) / kWarps;  // turns per warp
  const int u0 = min(warp * run, (tile1 - tile0) * chunks), u1 = min(u0 + run, (tile1 - tile0) * chunks);

  const uint8_t* xp[NT];  // tokens behind the last read the last one; their results are not written
#pragma unroll
  for (int t = 0; t < NT; ++t)
    xp[t] = a.x + static_cast<int64_t>(min(m0 + t * 8 + gr, a.m - 1)) * a.xs + tq * 16 * ES;

  // ---- weights: a cursor over this warp's turns, kStages - 1 ahead of the products
  int f_left = u1 - u0, f_tile = tile0 + u0 / chunks, f_chunk = u0 % chunks, f_stage = 0;
  const uint8_t* f_w;  // this lane's 16 bytes (lane % 8) of row lane / 8; rows 4 j further are f_off[j] behind it
  int f_off[4];
  auto f_rows = [&] {  // rows behind the last read the last one; their results are not written
    const int n = min(f_tile * kRows + (lane >> 3), a.n - 1);
    f_w = a.w + static_cast<int64_t>(n) * a.ws + (lane & 7) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) f_off[j] = min(4 * j, a.n - 1 - n) * static_cast<int>(a.ws);
  };
  f_rows();
  // Chunk c of row r lies at chunk c ^ (r % 4) * 2: a quad's 32 bytes of 4 rows fill the banks once.
  const uint32_t put = buf + (lane >> 3) * (kChunk / 2) + (((lane & 7) ^ ((lane >> 3) << 1)) << 4);
  auto push = [&] {  // starts the loads of the cursor's turn
    if (f_left > 0) {
      --f_left;
      const int there = f_chunk * kChunk + (lane & 7) * 32 < a.k ? 16 : 0;
      const uint8_t* const from = f_w + f_chunk * (kChunk / 2);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        cp_async16(put + f_stage * C::STAGE + j * 4 * (kChunk / 2), there ? from + f_off[j] : a.w, there);
      if (++f_chunk == chunks) {
        f_chunk = 0;
        ++f_tile;
        f_rows();
      }
    }
    cp_async_commit();
    f_stage = f_stage + 1 == kStages ? 0 : f_stage + 1;
  };

  // ---- scales and zero points: SUPER turns of a tile at a time, loaded one set ahead (whole stretches of rows:
  // a load instruction touches few lines) and entered in the table when their turns begin
  RawVec<ES> s_raw[C::ENTRIES];
  uint32_t z_raw[C::ENTRIES];
  const int g_col = lane % COLS, g_row = lane / COLS;
  auto load_groups = [&](int tile, int set) {
    const int at = fast_div(min((set * COLS + g_col) * (kChunk / GROUPS), a.k - 1), a.group);
#pragma unroll
    for (int i = 0; i < C::ENTRIES; ++i) {
      const int64_t r = min(tile * kRows + i * (32 / COLS) + g_row, a.n - 1);
      s_raw[i] = *reinterpret_cast<const RawVec<ES>*>(a.scales + r * a.ss + at * ES);
      z_raw[i] = a.zeros ? __ldg(a.zeros + r * a.zs + at) : 8u;
    }
  };
  auto enter_groups = [&] {
#pragma unroll
    for (int i = 0; i < C::ENTRIES; ++i) {
      float s;
      unpack_vec<DT, ES>(s_raw[i], &s);
      table[g_col * (kRows + 1) + i * (32 / COLS) + g_row] = make_float2(s, __uint_as_float(zero_pair<DT>(z_raw[i])));
    }
  };

  // ---- products
  float acc[NT][4];
  Activations<DT> x_ahead[2][NT];  // of the next full quarter turn
  auto load_ahead = [&](int k) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t) x_ahead[j][t].load(xp[t] + (k + 8 * j) * ES);
  };
  auto compute = [&](auto full, int c, int next, const uint8_t* stage) {  // full: the turn has all its 256 k
    constexpr bool FULL = decltype(full)::value;
    constexpr int SETS = GK == kGroup32 ? 2 : 1;  // sums of a quarter that have scales of their own
    constexpr int CHAINS = TWO ? 2 : 1;
    float part[CHAINS][SETS][NT][4];
    float2 col[2], other[2];  // this lane's k's column, and (groups of 32) the quad's other one
    auto add_scaled = [&](int t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = col[e >> 1].x;
        if (GK == kGroup32) {
          const float o = other[e >> 1].x;
          acc[t][e] = fmaf(tq < 2 ? s : o, part[0][0][t][e], acc[t][e]);
          acc[t][e] = fmaf(tq < 2 ? o : s, part[0][SETS - 1][t][e], acc[t][e]);
        } else {
          acc[t][e] = fmaf(s, TWO ? part[0][0][t][e] + part[CHAINS - 1][0][t][e] : part[0][0][t][e], acc[t][e]);
        }
      }
    };
#pragma unroll(kAtOnce)
    for (int h = 0; h < kChunk / 64; ++h) {
      const int k = c * kChunk + h * 64;
      if (!FULL && k >= a.k) break;
      Activations<DT> x[2][NT];
      if (XS) {
        // (read below)
      } else if (AHEAD && FULL) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t) x[j][t] = x_ahead[j][t];
        load_ahead(h + 1 < kChunk / 64 ? k + 64 : next);
      } else if (FULL || k + 64 <= a.k || tq < 2) {  // (the last quarter may have 32 k)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t) x[j][t].load(xp[t] + (k + 8 * j) * ES);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t) x[j][t].zero();
      }
      uint2 w[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        w[r] = *reinterpret_cast<const uint2*>(stage + (8 * r + gr) * (kChunk / 2) + ((h ^ (gr & 3)) << 5) + tq * 8);
      const bool first = SHORT || GK != kGroup128 || (h & 1) == 0;  // of the products that share a scale
      if (first) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int g = c % C::SUPER * GROUPS + (GK == kGroup128 ? h >> 1 : GK == kGroup64 ? h : 2 * h + (tq >> 1));
          col[r] = table[g * (kRows + 1) + 8 * r + gr];
          if (GK == kGroup32) other[r] = table[(g ^ 1) * (kRows + 1) + 8 * r + gr];
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t d0[4], d1[4];
        codes_minus_zero<DT>(j ? w[0].y : w[0].x, __float_as_uint(col[0].y), d0);
        codes_minus_zero<DT>(j ? w[1].y : w[1].x, __float_as_uint(col[1].y), d1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          uint32_t p[PARTS][4];
          if (XS) {
            // lanes of tokens that are not there read the last one's: columns that are not written
#pragma unroll
            for (int y = 0; y < PARTS; ++y) {
              const uint4 v = x_all[((k / 64 * 2 + j) * PARTS + y) * x_lanes + min(t * 32 + lane, x_lanes - 1)];
              p[y][0] = v.x;
              p[y][1] = v.y;
              p[y][2] = v.z;
              p[y][3] = v.w;
            }
          } else {
            x[j][t].pairs(p);
          }
#pragma unroll
          for (int y = PARTS - 1; y >= 0; --y) {
#pragma unroll
            for (int set = 0; set < SETS; ++set) {
              // groups of 32: the quad's first two lanes are in one group, its last two in the next
              const bool in = SETS == 1 || (tq >> 1) == set;
              const uint32_t b0 = in ? p[y][0] : 0, b1 = in ? p[y][1] : 0, b2 = in ? p[y][2] : 0, b3 = in ? p[y][3] : 0;
              float(&sum)[4] = part[j % CHAINS][set][t];
              if (SHORT ? y == PARTS - 1 : first && j < CHAINS)
                mma_w4<DT, true>(sum, d0[0], d1[0], d0[1], d1[1], b0, b1);
              else
                mma_w4<DT, false>(sum, d0[0], d1[0], d0[1], d1[1], b0, b1);
              mma_w4<DT, false>(sum, d0[2], d1[2], d0[3], d1[3], b2, b3);
            }
          }
          if (SHORT) add_scaled(t);
        }
      }
      if (SHORT || GK == kGroup128 && first && (FULL || k + 64 < a.k)) continue;  // the next quarter has the same scale
#pragma unroll
      for (int t = 0; t < NT; ++t) add_scaled(t);
    }
  };
  auto write = [&](int m, int n, float s) {
    if (m >= a.m || n >= a.n) return;
    if (a.bias) {
      float b;
      unpack_vec<DT, ES>(*reinterpret_cast<const RawVec<ES>*>(a.bias + static_cast<int64_t>(n) * ES), &b);
      s += b;
    }
    *reinterpret_cast<RawVec<ES>*>(a.y + static_cast<int64_t>(m) * a.ys + static_cast<int64_t>(n) * ES) = pack_vec<DT, ES>(&s);
  };

#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) push();
  int stage = 0;
  int tile = tile0 + u0 / chunks, c = u0 % chunks;
  load_groups(tile, c / C::SUPER);
  if constexpr (XS) {
    const int count = (a.k + 63) / 64 * 2 * x_lanes;
    auto fill = [&](auto full, auto at_once) {  // full: all 8 NT tokens are there; at_once: loads in flight per thread
      constexpr int AT_ONCE = decltype(at_once)::value;
      for (int i0 = threadIdx.x; i0 < count; i0 += AT_ONCE * kThreads) {
        Activations<DT> x[AT_ONCE];
        int set[AT_ONCE], l[AT_ONCE];  // set: quarter and word
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) {
          const int i = i0 + e * kThreads;
          set[e] = decltype(full)::value ? i / (32 * NT) : i / x_lanes;
          l[e] = i - set[e] * x_lanes;
          const int k = set[e] / 2 * 64 + (l[e] & 3) * 16 + set[e] % 2 * 8;
          if (i < count && k < a.k)
            x[e].load(a.x + static_cast<int64_t>(m0 + (l[e] >> 2)) * a.xs + k * ES);
          else
            x[e].zero();
        }
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) {
          uint32_t p[PARTS][4];
          x[e].pairs(p);
#pragma unroll
          for (int y = 0; y < PARTS; ++y)
            if (i0 + e * kThreads < count)
              x_all[(set[e] * PARTS + y) * x_lanes + l[e]] = make_uint4(p[y][0], p[y][1], p[y][2], p[y][3]);
        }
      }
    };
    if (count <= kThreads) fill(std::false_type{}, std::integral_constant<int, 1>{});
    else if (x_lanes < 32 * NT) fill(std::false_type{}, std::integral_constant<int, 4>{});
    else fill(std::true_type{}, std::integral_constant<int, DT == CMPX_F32 ? 4 : 8>{});
    __syncthreads();
  }
  // (a partial last turn leaves x_ahead at the row's begin, where the next tile's first turn needs it)
  if (AHEAD && a.k >= kChunk) load_ahead((c + 1) * kChunk <= a.k ? c * kChunk : 0);
  for (int u = u0; u < u1;) {
    const int turns = min(chunks - c, u1 - u);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    for (int i = 0; i < turns; ++i) {
      cp_async_wait<kStages - 2>();
      __syncwarp();  // this turn's weights are there, and everybody is done with the turn before
      push();
      if (u + i == u0 || (c + i) % C::SUPER == 0) {
        enter_groups();
        __syncwarp();
        const int set = (c + i) / C::SUPER + 1;
        const bool on = set * C::SUPER < chunks;
        if (on || tile + 1 < tile1) load_groups(on ? tile : tile + 1, on ? set : 0);
      }
      // where the activations of the next full turn begin: behind this one, or with the next tile at 0
      const int now = (c + i) * kChunk, after = now + 2 * kChunk <= a.k ? now + kChunk : 0;
      if (now + kChunk <= a.k)
        compute(std::true_type{}, c + i, after, mine + stage * C::STAGE);
      else
        compute(std::false_type{}, c + i, 0, mine + stage * C::STAGE);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    const bool later = tile != tile0 + u0 / chunks;
    if (turns != chunks && later) {
      cp_async_wait<0>();
      __syncwarp();
    }
    float* const part = part_of(warp, later);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int token = t * 8 + tq * 2 + (e & 1), r = gr + 8 * (e >> 1);
        if (turns == chunks)
          write(m0 + token, tile * kRows + r, acc[t][e]);
        else
          part[token * (kRows + 1) + r] = acc[t][e];
      }
    u += turns;
    c = 0;
    ++tile;
  }
  cp_async_wait<0>();

  // the tiles that several warps have parts of
  __syncthreads();
  if (tile1 - tile0 == 1) {  // one tile, a part from every warp: four lanes an output
    for (int i = threadIdx.x; i < NT * 8 * kRows * 4; i += kThreads) {
      const int r = i / 4 % kRows, token = i / (4 * kRows), warps = (chunks + run - 1) / run;
      if (warps == 1) break;
      float s = 0.f;
      for (int w = i % 4; w < warps; w += 4) s += part_of(w, false)[token * (kRows + 1) + r];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (i % 4 == 0) write(m0 + token, tile0 * kRows + r, s);
    }
    return;
  }
  for (int i = threadIdx.x; i < (tile1 - tile0) * (NT * 8 * kRows); i += kThreads) {
    const int r = i % kRows, token = i / kRows % (NT * 8), t = i / (kRows * NT * 8);
    const int w0 = t * chunks / run, w1 = ((t + 1) * chunks - 1) / run;
    if (w0 == w1) continue;
    float s = 0.f;
    for (int w = w0; w <= w1; ++w) s += part_of(w, t != w * run / chunks)[token * (kRows + 1) + r];
    write(m0 + token, (tile0 + t) * kRows + r, s);
  }
}

GroupKind group_kind(int64_t group) { return group % 128 == 0 ? kGroup128 : group % 64 == 0 ? kGroup64 : kGroup32; }

// Bytes of a CTA's activations as the products take them.
template <int DT, int NT>
int64_t x_bytes(const W4Args& a) {
  return static_cast<int64_t>(a.k + 63) / 64 * 64 * 2 * Activations<DT>::PARTS * std::min(8 * NT, a.m);
}

template <int DT, int NT, int GK, bool XS>
int launch_as(W4Args& a, const LaunchCtx& ctx) {
  using C = W4Cfg<DT, NT, GK, XS>;
  auto kernel = linear_w4_kernel<DT, NT, GK, XS>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::call_once(once[dev & 63], [&] {
    attr_err[dev & 63] =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM + (XS ? C::X_MOST : 0));
  });
  if (attr_err[dev & 63] != cudaSuccess) return CMPX_ERR_LAUNCH;
  a.chunks = (a.k + kChunk - 1) / kChunk;
  const int tiles = (a.n + kRows - 1) / kRows, ctas = std::min(tiles, ctx.num_sms);
  a.tiles_per_cta = tiles / ctas;
  a.tiles_rest = tiles % ctas;
  const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>((a.m + 8 * NT - 1) / (8 * NT)));
  kernel<<<grid, kThreads, C::SMEM + (XS ? static_cast<int>(x_bytes<DT, NT>(a)) : 0), ctx.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? CMPX_OK : CMPX_ERR_LAUNCH;
}

template <int DT, int NT, int GK>
int launch(W4Args& a, const LaunchCtx& ctx) {
  // Activations of up to 64 KB (16-bit: 8 tokens of 4096 k; fp32 takes 6 bytes a value) are laid out for the products
  // once per CTA.
  if (x_bytes<DT, NT>(a) <= W4Cfg<DT, NT, GK, true>::X_MOST) return launch_as<DT, NT, GK, true>(a, ctx);
  return launch_as<DT, NT, GK, false>(a, ctx);
}

template <int DT, int NT>
int launch_group(W4Args& a, const LaunchCtx& ctx) {
  switch (group_kind(a.group.d)) {
    case kGroup128: return launch<DT, NT, kGroup128>(a, ctx);
    case kGroup64: return launch<DT, NT, kGroup64>(a, ctx);
    default: return launch<DT, NT, kGroup32>(a, ctx);
  }
}

template <int DT>
int launch_dt(W4Args& a, const LaunchCtx& ctx) {
  return a.m <= 8 ? launch_group<DT, 1>(a, ctx) : launch_group<DT, 2>(a, ctx);
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
  if (d->group % 32 != 0 || d->k > (1 << 24) || d->n > ((1ll << 38) / d->k) || d->n > (1ll << 31) - 65536 || d->m > 65535ll * 8) return "none";
  // (the kernel counts 12 rows of W in 32 bits)
  if (d->x_row_stride < 0 || d->w_row_stride < 0 || (d->n > 1 && d->w_row_stride > (1 << 27)) || d->scales_row_stride < 0 || d->zeros_row_stride < 0 ||
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
