// Matrix product with 4-bit weights and a scale for each group of a channel's inputs, written for gfx950.
//
//   y[m, n] = bf16(sum_k x[m, k] s[n, k / G] (c[n, k] - z[n, k / G])),   c in 0 .. 15, G 32, 64 or 128
//
// x is bf16, s and z are bf16 (z may be absent: 8). The codes lie in tiles of 16 channels and units of 128 inputs, 1 KB
// each, in the order in which v_mfma_f32_16x16x32_bf16 takes them: the 16 bytes of lane 16 q + r are channel r, word i
// inputs 32 i + 8 q + (0 .. 7), input 2 j at bit 4 j and input 2 j + 1 at bit 16 + 4 j. A wave's load of a unit is 1 KB
// in a row. s and z are [tile][unit][16 channels][128 / G].
#include <algorithm>

#include "ftx_internal.h"

namespace ftx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kWave = 64;
constexpr int kUnit = kInt4Unit;         // inputs of a unit
constexpr int kUnitBytes = 16 * kUnit / 2;

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// (min of 64-bit integers would go through doubles)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

// A quotient or remainder of a workgroup's number, computed on the vector unit, as the scalar that it is.
__device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(static_cast<int>(v)); }

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N < 64, "vmcnt holds six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

__device__ __forceinline__ void ring_barrier() {
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's LDS accesses are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes per lane from base + offset + step into lds + 16 * lane; zeros where that is not below `bytes`.
__device__ __forceinline__ void load_to_lds(const uint8_t *base, uint32_t bytes, uint32_t offset, uint32_t step,
                                            uint8_t *lds) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, bytes, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)lds, 16, offset, step, 0, 0);
}

// The PARTS = 128 / G scales (or zeros) of a channel in a unit.
template <int PARTS>
struct Scales {
  uint32_t w[PARTS == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const uint16_t *from) {
    if constexpr (PARTS == 1) w[0] = *from;
    if constexpr (PARTS == 2) w[0] = *reinterpret_cast<const uint32_t *>(from);
    if constexpr (PARTS == 4) {
      const u32x2 v = *reinterpret_cast<const u32x2 *>(from);
      w[0] = v[0];
      w[1] = v[1];
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};

// ---- up to 32 rows -------------------------------------------------------------------------------------------------
//
// A workgroup a CU walks its share of the tiles of channels, up to NT at a time, over the whole of K, with RT times 16
// rows; its eight waves take units in turn, codes and x straight into registers as operands, three units in flight across
// the ends of the chunks, and join their sums through LDS. Bound by the bytes of w: 28672 x 8192 (G 128) of four rows
// 28 us, 4.3 TB/s where plain reads of as many bytes reach 6.2 (without the products 27); with G 64 and zeros 31 us for
// one row, 33 for 13; 4096 x 4096 of one row 5.5 us.
//
// A code becomes the bf16 number 128 + c by an AND and an OR of two codes at a time, exact in the seven bits below the
// leading one. What that adds comes out again for each group: with a column of ones the matrix cores sum the rows' x in
// the layout of the products, and sum_g s (sum x (128 + c) - (128 + z) sum x) is the product with s and z in fp32. Each
// addition to either sum loses up to 2^-24 of it, together (271 + |z|) s sum |x| of the group, whatever the weights
// are: ones of 0 leave that too (one input of 3000 among 127 of about 1: 0.03 s, 0.13 s at most). With 16 + c it would be a
// sixth, for a shift more of each word: 13 rows of 28672 x 8192 30.0 us where these take 29.5.
template <int NT, int RT, int PARTS, bool ZERO>
__global__ __launch_bounds__(512) void int4_rows_kernel(Int4Linear p) {
  constexpr int kWaves = 8, kSteps = 4 / PARTS;  // products of 32 inputs in a group
  __shared__ f32x4 part[2][kWaves][NT][RT][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, q = lane >> 4;
  const int m = static_cast<int>(p.m);
  const int64_t tile0 = static_cast<int64_t>(blockIdx.x) * p.tiles / p.items;
  const int count = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * p.tiles / p.items - tile0);
  const int chunks = (count + NT - 1) / NT, steps = (p.units + kWaves - 1) / kWaves;
  const auto chunk_at = [&](int i) {  // the chunk's first tile of `count`, at most 60000
    return static_cast<int>(static_cast<uint32_t>(i * count) / static_cast<uint32_t>(chunks));
  };
  const uint16_t *xr[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) xr[j] = p.x + min(16 * j + r, m - 1) * p.x_stride + 8 * q;

  struct Unit {
    u32x4 x[RT][4], w[NT];
    Scales<PARTS> s[NT], z[ZERO ? NT : 1];
  };
  int load_chunk = 0, load_step = 0, load_first = 0, load_tiles = chunk_at(1);
  const auto load = [&](Unit &v) {  // the wave's next unit; past K, x is 0 and w the last one
    if (load_chunk >= chunks) return;
    const int u = load_step * kWaves + wave, held = min(u, p.units - 1);
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v.x[j][i] = (u32x4){0u, 0u, 0u, 0u};
        if (u * kUnit + 32 * i < p.k) v.x[j][i] = *reinterpret_cast<const u32x4 *>(xr[j] + held * kUnit + 32 * i);
      }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t >= load_tiles) continue;
      const int64_t at = (tile0 + load_first + t) * p.units + held;
      v.w[t] = *reinterpret_cast<const u32x4 *>(p.w + at * kUnitBytes + lane * 16);
      v.s[t].load(p.scale + (at * 16 + r) * PARTS);
      if (ZERO) v.z[t].load(p.zero + (at * 16 + r) * PARTS);
    }
    if (++load_step == steps) {
      load_step = 0;
      ++load_chunk;
      load_first += load_tiles;
      load_tiles = chunk_at(load_chunk + 1) - load_first;
    }
  };
  f32x4 y[NT][RT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < RT; ++j) y[t][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, (u32x4){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  int chunk = 0, step = 0, first = 0, tiles = chunk_at(1), side = 0;
  const auto work = [&](const Unit &v) {  // returns whether it was the last one
#pragma unroll
    for (int g = 0; g < PARTS; ++g) {
      f32x4 sum[RT];
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        sum[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = g * kSteps; i < (g + 1) * kSteps; ++i)
          sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v.x[j][i]), ones, sum[j], 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t >= tiles) continue;
        f32x4 acc[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = g * kSteps; i < (g + 1) * kSteps; ++i) {
          u32x4 c;
#pragma unroll
          for (int j = 0; j < 4; ++j) c[j] = (v.w[t][i] >> (4 * j) & 0x000f000fu) | 0x43004300u;
#pragma unroll
          for (int j = 0; j < RT; ++j)
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v.x[j][i]),
                                                             __builtin_bit_cast(bf16x8, c), acc[j], 0, 0, 0);
        }
        const float s = v.s[t][g], offset = ZERO ? -128.f - v.z[t][g] : -136.f;
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[t][j][e] = fmaf(s, fmaf(offset, sum[j][e], acc[j][e]), y[t][j][e]);
      }
    }
    if (++step < steps) return false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        part[side][wave][t][j][lane] = y[t][j];
        y[t][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      }
    ring_barrier();  // the other side's sums have been read by all
    for (int i = threadIdx.x; i < 16 * 16 * RT * tiles; i += 512) {
      const int ch = i % 16, row = i / 16 % (16 * RT), t = i / (256 * RT);
      const int64_t at = (tile0 + first + t) * 16 + ch;
      if (row >= m || at >= p.n) continue;
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all += part[side][w][t][row / 16][ch + 16 * (row % 16 / 4)][row % 4];
      p.y[row * p.n + at] = static_cast<uint16_t>(pack_bf16(all, 0.f));
    }
    step = 0;
    side ^= 1;
    first += tiles;
    tiles = chunk_at(++chunk + 1) - first;
    return chunk >= chunks;
  };
  Unit a, b, c;
  load(a);
  load(b);
  for (;;) {
    load(c);
    if (work(a)) break;
    load(a);
    if (work(b)) break;
    load(b);
    if (work(c)) break;
  }
}

// ---- tiles -----------------------------------------------------------------------------------------------------------
//
// Up to TM tokens x TN channels a workgroup, K in units of 128: the tokens are dealt evenly to the tiles, in 16s, and
// products of 16s that a tile does not have are left out (777 rows in four tiles of 208). A unit's x goes straight from
// memory into one of STAGES stages of LDS while another is multiplied, with one barrier a unit; row R's 16-byte chunk c
// lies at slot c ^ (R % 16), so the 16 rows that a read touches lie in different banks. The codes go from memory into
// the registers of the wave that multiplies by them, as the operands that they are, DEPTH units ahead: they take no LDS
// and no barrier. A wave makes the weights of its channels for the next 32 inputs, (c - z) s in fp32 rounded to bf16,
// between the products of these ones.
//
// Rounding the weights is what lets the matrix cores sum over groups: an error of 2^-8 of each at most, 0.0022 of the
// result in relative norm where the output's own rounding is 0.0017. v_mfma_f32_16x16x32_bf16 takes the channels as
// rows and the tokens as columns, so a lane ends with four neighbouring channels of a token; they reach y through LDS,
// in whole lines.

// Eight codes as weights, s c + b.
__device__ __forceinline__ bf16x8 weights(uint32_t w, float s, float b) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = w >> 4 & 0x0f0f0f0fu;
  const auto value = [&](uint32_t v, int byte) { return fmaf(static_cast<float>(v >> (8 * byte) & 255u), s, b); };
  return __builtin_bit_cast(bf16x8, (u32x4){pack_bf16(value(lo, 0), value(lo, 2)), pack_bf16(value(hi, 0), value(hi, 2)),
                                            pack_bf16(value(lo, 1), value(lo, 3)), pack_bf16(value(hi, 1), value(hi, 3))});
}

template <int TM, int TN, int WN, int STAGES, int DEPTH, int PARTS, bool ZERO, bool SPLIT>
__global__ __launch_bounds__(WN * kWave, 2) void int4_tile_kernel(Int4Linear p) {
  constexpr int kWaves = WN;
  constexpr int kRow = kUnit * 2;                    // bytes of a row of x in a stage
  constexpr int kStage = TM * kRow;
  constexpr int kLoads = kStage / 1024 / kWaves;     // of one wave, four rows of x each
  constexpr int kMT = TM / 16, kNT = TN / WN / 16;
  constexpr int kCodeLoads = kNT * (ZERO ? 3 : 2);
  static_assert(kStage / 1024 % kWaves == 0, "every wave has the same to load");
  __shared__ __align__(1024) uint8_t lds[STAGES * kStage];
  const uint32_t per_xcd = (p.items + p.xcds - 1) / p.xcds;
  uint32_t item = (blockIdx.x % p.xcds) * per_xcd + blockIdx.x / p.xcds;
  if (blockIdx.x / p.xcds >= per_xcd || item >= p.items) return;
  const int split = SPLIT ? uniform(item % static_cast<uint32_t>(p.splits)) : 0;
  if (SPLIT) item /= static_cast<uint32_t>(p.splits);
  const uint32_t run = item / (p.band * p.n_tiles), at = item - run * p.band * p.n_tiles;
  const uint32_t rows = min(static_cast<uint32_t>(p.band), p.m_tiles - run * p.band);
  const int64_t m0 = static_cast<int64_t>(uniform(run * p.band + at % rows)) * p.tile_rows;
  const int64_t n0 = static_cast<int64_t>(uniform(at / rows)) * TN;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, q = lane >> 4;
  const int live = (static_cast<int>(least(p.m - m0, p.tile_rows)) + 15) / 16;  // 16s of tokens that the tile has

  // Load i of a wave brings rows 4 (i kWaves + wave) .. + 3 of 256 bytes; rows past the last and inputs past K are 0.
  const uint8_t *tokens = reinterpret_cast<const uint8_t *>(p.x + m0 * p.x_stride);
  const uint32_t token_bytes = static_cast<uint32_t>(
      least(((least(p.m - m0, p.tile_rows) - 1) * p.x_stride + p.k) * 2, 0x7fffffff));
  const auto issue = [&](int u, int stage) {
    uint8_t *base = lds + stage * kStage + wave * 1024;
    const bool whole = (u + 1) * kUnit <= p.k;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int R = (i * kWaves + wave) * 4 + lane / 16;
      const int chunk = (lane % 16) ^ (R % 16);
      const uint32_t offset = R * static_cast<uint32_t>(p.x_stride * 2) + chunk * 16;
      load_to_lds(tokens, token_bytes, whole || u * kUnit + chunk * 8 < p.k ? offset : 0xf0000000u, u * kRow,
                  base + i * kWaves * 1024);
    }
  };

  struct Unit {  // 128 inputs of the wave's channels
    u32x4 w[kNT];
    Scales<PARTS> s[kNT], z[ZERO ? kNT : 1];
  };
  const int64_t tile0 = n0 / 16 + wave * kNT;
  const auto load = [&](Unit &v, int u) {
#pragma unroll
    for (int t = 0; t < kNT; ++t) {
      const int64_t of = least(tile0 + t, p.tiles - 1) * p.units + u;
      v.w[t] = *reinterpret_cast<const u32x4 *>(p.w + of * kUnitBytes + lane * 16);
      v.s[t].load(p.scale + (of * 16 + r) * PARTS);
      if (ZERO) v.z[t].load(p.zero + (of * 16 + r) * PARTS);
    }
  };
  const auto make = [&](const Unit &v, int t, int word) {
    const int part = word * PARTS / 4;
    const float s = v.s[t][part];
    return weights(v.w[t][word], s, -s * (ZERO ? v.z[t][part] : 8.f));
  };

  f32x4 acc[kMT][kNT];
#pragma unroll
  for (int j = 0; j < kMT; ++j)
#pragma unroll
    for (int t = 0; t < kNT; ++t) acc[j][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const uint32_t b_at = r * kRow;
  const auto multiply = [&](const Unit &v, int stage) {
    const uint8_t *from = lds + stage * kStage + b_at;
    const auto read = [&](int n) {  // the nth of the unit's operands: a tile of tokens, 32 inputs
      return *reinterpret_cast<const bf16x8 *>(from + n % kMT * 16 * kRow + ((n / kMT * 4 + q) ^ r) * 16);
    };
    constexpr int kAhead = kMT > 8 ? 5 : 3;
    bf16x8 a[2][kNT], b[kAhead + 1];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) b[n] = read(n);
#pragma unroll
    for (int t = 0; t < kNT; ++t) a[0][t] = make(v, t, 0);
#pragma unroll
    for (int n = 0; n < 4 * kMT; ++n) {
      const int word = n / kMT, j = n % kMT;
      if (n + kAhead < 4 * kMT) b[(n + kAhead) % (kAhead + 1)] = read(n + kAhead);
      if (word < 3) {  // a part of the next weights
#pragma unroll
        for (int t = j * kNT / kMT; t < (j + 1) * kNT / kMT; ++t) a[(word + 1) % 2][t] = make(v, t, word + 1);
      }
      if (j < live) {
#pragma unroll
        for (int t = 0; t < kNT; ++t)
          acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[word % 2][t], b[n % (kAhead + 1)], acc[j][t], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // x of unit u lies in stage u - first modulo STAGES and is on its way STAGES - 1 units ahead, its codes DEPTH - 1 and
  // a little. Past the last unit it again, so that every round has the same loads in flight.
  const int first = SPLIT ? split * p.split_units : 0;
  const int end = SPLIT ? min(p.units, first + p.split_units) : p.units;
  const auto at_most = [&](int u) { return min(u, end - 1); };
  Unit units[DEPTH];
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(at_most(first + i), i);
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) load(units[i], at_most(first + i));
  asm volatile("" ::: "memory");
  int stage = 0, next = STAGES - 1;
  const auto round = [&](Unit &v, int u) {
    // in flight behind x of this unit: the x of STAGES - 2 more, and the codes loaded since
    if (u == first) wait_vmcnt<0>();
    else wait_vmcnt<(STAGES - 2) * kLoads + (STAGES - 1) * kCodeLoads>();
    ring_barrier();
    issue(at_most(u + STAGES - 1), next);
    asm volatile("" ::: "memory");
    multiply(v, stage);
    load(v, at_most(u + DEPTH));
    asm volatile("" ::: "memory");
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    next = next == STAGES - 1 ? 0 : next + 1;
  };
  for (int u0 = first; u0 < end; u0 += DEPTH) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
      if (u0 + i < end) round(units[i], u0 + i);
  }

  if (SPLIT) {  // sums [split][m][n]
#pragma unroll
    for (int j = 0; j < kMT; ++j) {
      const int64_t row = m0 + j * 16 + r;
      if (j >= live || row >= p.m) continue;
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        const int64_t ch = n0 + (wave * kNT + t) * 16 + 4 * q;
        if (ch < p.part_stride)
          *reinterpret_cast<f32x4 *>(p.part + (split * p.m + row) * p.part_stride + ch) = acc[j][t];
      }
    }
    return;
  }
  // 16 tokens x the wave's channels at a time through this wave's part of LDS, 16 bytes between rows against conflicts
  constexpr int kPitch = kNT * 32 + 16;
  static_assert(16 * kPitch * kWaves <= STAGES * kStage, "the epilogue fits the stages");
  wait_vmcnt<0>();  // what was loaded past the last unit has arrived
  __syncthreads();  // and the last one has been read
  uint8_t *mine = lds + wave * 16 * kPitch;
#pragma unroll
  for (int j = 0; j < kMT; ++j) {
    if (j >= live) continue;
    const int64_t t0 = m0 + j * 16, c0 = n0 + wave * kNT * 16;
#pragma unroll
    for (int t = 0; t < kNT; ++t)
      *reinterpret_cast<u32x2 *>(mine + r * kPitch + (t * 16 + 4 * q) * 2) =
          (u32x2){pack_bf16(acc[j][t][0], acc[j][t][1]), pack_bf16(acc[j][t][2], acc[j][t][3])};
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    constexpr int kLanes = kNT * 2;  // 16 bytes each, of one token
#pragma unroll
    for (int i = 0; i < (16 * kLanes + kWave - 1) / kWave; ++i) {
      const int row = i * (kWave / kLanes) + lane / kLanes, col = lane % kLanes;
      const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + row * kPitch + col * 16);
      if (t0 + row >= p.m) continue;
      uint16_t *to = p.y + (t0 + row) * p.n + c0 + col * 8;
      if (c0 + col * 8 + 8 <= p.n && p.n % 8 == 0) {
        *reinterpret_cast<u32x4 *>(to) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + col * 8 + e < p.n) to[e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1)));
      }
    }
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
}

// y = bf16(sum over the splits), four channels a thread.
__global__ __launch_bounds__(256) void int4_join_kernel(Int4Linear p) {
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  const int64_t size = p.m * p.part_stride;
  if (at >= size) return;
  const int64_t t = at / p.part_stride, ch = at % p.part_stride;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < p.splits; ++i) sum += *reinterpret_cast<const f32x4 *>(p.part + i * size + at);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (ch + e < p.n) p.y[t * p.n + ch + e] = static_cast<uint16_t>(pack_bf16(sum[e], 0.f));
}

template <int PARTS, bool ZERO, int NT, int RT>
void start_rows(const Int4Linear &p, hipStream_t stream) {
  hipLaunchKernelGGL((int4_rows_kernel<NT, RT, PARTS, ZERO>), dim3(p.items), dim3(512), 0, stream, p);
}

template <int PARTS, bool ZERO, int TM, int TN, int WN, int STAGES, int DEPTH>
void start_tiles(const Int4Linear &p, hipStream_t stream) {
  const dim3 grid((p.items + p.xcds - 1) / p.xcds * p.xcds), block(WN * kWave);
  if (p.splits > 1)
    hipLaunchKernelGGL((int4_tile_kernel<TM, TN, WN, STAGES, DEPTH, PARTS, ZERO, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((int4_tile_kernel<TM, TN, WN, STAGES, DEPTH, PARTS, ZERO, false>), grid, block, 0, stream, p);
}

template <int PARTS, bool ZERO>
void start(const Int4Linear &p, hipStream_t stream) {
  switch (p.tile_m) {
    case 16:
      if (p.row_tiles == 1) start_rows<PARTS, ZERO, 1, 1>(p, stream);
      else if (p.row_tiles == 2) start_rows<PARTS, ZERO, 2, 1>(p, stream);
      else start_rows<PARTS, ZERO, 4, 1>(p, stream);
      break;
    case 32:
      if (p.row_tiles == 1) start_rows<PARTS, ZERO, 1, 2>(p, stream);
      else start_rows<PARTS, ZERO, 2, 2>(p, stream);
      break;
    case 64: start_tiles<PARTS, ZERO, 64, 128, 4, 3, 4>(p, stream); break;
    default: start_tiles<PARTS, ZERO, 256, 256, 8, 2, 2>(p, stream); break;
  }
}

}  // namespace

// Which tiles and how often K is split, by what it costs in 0.01 us: a unit of a tile, more for each 16 tokens that it
// has; tiles of 256 have a CU to themselves, so theirs come in whole rounds, tiles of 64 share one; reading w; a start,
// and the join of the splits.
//                    a unit   a 16   start
//   64 x 128             65      8     500
//   256 x 256           120     15    1000
// The kernel of few rows takes 17 to 32 where that is less: 4 us, x for each chunk of a CU's tiles at 29 KB a us; what is
// above stands a fifth below what such calls take. Measured, us, in tiles of 64 and in that kernel: 4096 x 4096 of 17
// rows 13.5 and 8.9, of 32 14.1 and 11.7; 32000 x 4096 of 25 rows 39.7 and 33.1; 8192 x 28672 61.8 and 52.7; 28672 x 8192
// 56.5 and 61.6, of 32 rows 57.0 and 71.7; 1024 x 8192 of 25 14.3 and 16.8.
// Measured, us: 8192 x 28672 of 777 rows 366 in tiles of 256 split in two, 585 unsplit and as much in tiles of 64; 28672 x
// 8192 of 100 rows 98 and 94, of 200 119 and 167, of 512 217 and 302, of 64 rows 60 split in three and 74 unsplit; 4096 x
// 4096 of 17 rows 13.1 split in eight, 36 unsplit.
void plan_int4_linear(Int4Linear *p, int cus, int xcds) {
  p->xcds = std::max(1, xcds);
  p->tiles = (p->n + 15) / 16;
  p->units = static_cast<int>((p->k + kUnit - 1) / kUnit);
  p->part_stride = (p->n + 3) / 4 * 4;
  p->splits = 1;
  p->part_bytes = 0;
  p->items = static_cast<uint32_t>(std::min<int64_t>(p->tiles, cus));
  const int64_t tiles_each = p->items > 0 ? (p->tiles + p->items - 1) / p->items : 0;
  p->row_tiles = tiles_each == 1 ? 1 : tiles_each == 2 || p->m > 16 ? 2 : 4;
  p->tile_m = 16;
  if (p->m <= 16) return;
  int64_t best = INT64_MAX, splits = 1;
  int tile_n = 128;
  const int64_t reading = p->n * p->k / 106000;
  const auto weigh = [&](int tm, int tn, int64_t unit, int64_t per16, int64_t start) {
    const int64_t m_tiles = (p->m + tm - 1) / tm, live = ((p->m + 15) / 16 + m_tiles - 1) / m_tiles;
    const int64_t tiles = m_tiles * ((p->n + tn - 1) / tn);
    for (int64_t s = 1; s <= 16 && (s == 1 || p->units / s >= 2); s += s < 4 ? 1 : s / 2) {
      const int64_t items = tiles * s, each = (unit + per16 * live) * ((p->units + s - 1) / s);
      const int64_t products = tm == 256 ? (items + cus - 1) / cus * each : std::max(each, each * 9 / 10 * items / cus);
      const int64_t cost = std::max(products, reading) + start + (s > 1 ? 300 + p->m * p->n * s / 10000 : 0);
      if (cost >= best) continue;
      best = cost;
      splits = s;
      p->tile_m = tm;
      tile_n = tn;
    }
  };
  weigh(64, 128, 65, 8, 500);
  if (p->m > 64) weigh(256, 256, 120, 15, 1000);
  if (p->m <= 32) {  // a workgroup reads all of x for each chunk of its tiles
    const int64_t chunks = (tiles_each + p->row_tiles - 1) / p->row_tiles;
    const int64_t cost = 400 + std::max(chunks * p->k * p->m * 2 / 290, p->n * p->k / 85000);
    if (cost * 5 < best * 6) {
      p->tile_m = 32;
      return;
    }
  }
  const int64_t m_tiles = (p->m + p->tile_m - 1) / p->tile_m, n_tiles = (p->n + tile_n - 1) / tile_n;
  if (m_tiles * n_tiles * splits > INT32_MAX) {  // too many for a launch, and for the numbers below: the caller refuses
    p->items = UINT32_MAX;
    return;
  }
  p->m_tiles = static_cast<uint32_t>(m_tiles);
  p->tile_rows = static_cast<int>(((p->m + 15) / 16 + p->m_tiles - 1) / p->m_tiles * 16);
  p->n_tiles = static_cast<uint32_t>(n_tiles);
  const uint32_t runs = (p->m_tiles + 11) / 12;
  p->band = static_cast<int>((p->m_tiles + runs - 1) / runs);
  p->split_units = static_cast<int>((p->units + splits - 1) / splits);
  p->splits = static_cast<int>((p->units + p->split_units - 1) / p->split_units);
  p->items = p->m_tiles * p->n_tiles * static_cast<uint32_t>(p->splits);
  p->part_bytes = p->splits > 1 ? static_cast<size_t>(p->splits) * p->m * p->part_stride * 4 : 0;
}

hipError_t launch_int4_linear(const Int4Linear &p, hipStream_t stream) {
  switch (p.parts * 2 + (p.zero ? 1 : 0)) {
    case 2: start<1, false>(p, stream); break;
    case 3: start<1, true>(p, stream); break;
    case 4: start<2, false>(p, stream); break;
    case 5: start<2, true>(p, stream); break;
    case 8: start<4, false>(p, stream); break;
    default: start<4, true>(p, stream); break;
  }
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.splits == 1) return err;
  const int64_t threads = p.m * p.part_stride / 4;
  hipLaunchKernelGGL(int4_join_kernel, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), kLdsToken, stream,
                     p);
  return hipGetLastError();
}

}  // namespace ftx
