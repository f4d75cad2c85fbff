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
typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// ---- up to 16 rows -------------------------------------------------------------------------------------------------
//
// A workgroup owns NT tiles of channels over the whole of K; its eight waves take units in turn, codes and x straight
// into registers as operands, the next units' on their way, and join their sums through LDS. Bound by the bytes of w.
//
// A code becomes the bf16 number 128 + c by an AND and an OR of two codes at a time, exact in the seven bits below the
// leading one. What that adds comes out again for each group: with a column of ones the matrix cores sum the rows' x in
// the layout of the products, and sum_g s (sum x (128 + c) - (128 + z) sum x) is the product with s and z in fp32. The
// sums are 16 times the weights' own at most, four bits of the 24.
template <int NT, int PARTS, bool ZERO>
__global__ __launch_bounds__(512) void int4_rows_kernel(Int4Linear p) {
  constexpr int kWaves = 8, kSteps = 4 / PARTS;  // products of 32 inputs in a group
  __shared__ f32x4 part[kWaves][NT][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, q = lane >> 4;
  const int m = static_cast<int>(p.m);
  const int64_t tile0 = static_cast<int64_t>(blockIdx.x) * NT;
  const uint16_t *xr = p.x + min(r, m - 1) * p.x_stride + 8 * q;

  struct Unit {
    u32x4 x[4], w[NT];
    Scales<PARTS> s[NT], z[ZERO ? NT : 1];
  };
  const auto load = [&](Unit &v, int u) {
    const uint16_t *from = xr + u * kUnit;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.x[i] = (u32x4){0u, 0u, 0u, 0u};
      if (u * kUnit + 32 * i < p.k) v.x[i] = *reinterpret_cast<const u32x4 *>(from + 32 * i);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t at = least(tile0 + t, p.tiles - 1) * p.units + u;
      v.w[t] = *reinterpret_cast<const u32x4 *>(p.w + at * kUnitBytes + lane * 16);
      v.s[t].load(p.scale + (at * 16 + r) * PARTS);
      if (ZERO) v.z[t].load(p.zero + (at * 16 + r) * PARTS);
    }
  };
  f32x4 y[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) y[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, (u32x4){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  const auto work = [&](const Unit &v) {
#pragma unroll
    for (int g = 0; g < PARTS; ++g) {
      f32x4 sum = {0.f, 0.f, 0.f, 0.f}, acc[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = sum;
#pragma unroll
      for (int i = g * kSteps; i < (g + 1) * kSteps; ++i) {
        const bf16x8 x = __builtin_bit_cast(bf16x8, v.x[i]);
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, ones, sum, 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          u32x4 c;
#pragma unroll
          for (int j = 0; j < 4; ++j) c[j] = (v.w[t][i] >> (4 * j) & 0x000f000fu) | 0x43004300u;
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, c), acc[t], 0, 0, 0);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float s = v.s[t][g], offset = ZERO ? -128.f - v.z[t][g] : -136.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[t][e] = fmaf(s, fmaf(offset, sum[e], acc[t][e]), y[t][e]);
      }
    }
  };
  const int n = (p.units - wave + kWaves - 1) / kWaves;  // the wave's units
  if (n > 0) {
    const auto nth = [&](int i) { return wave + min(i, n - 1) * kWaves; };  // past the last one it again
    Unit a, b, c;
    load(a, nth(0));
    load(b, nth(1));
    for (int i = 0;;) {
      load(c, nth(i + 2));
      work(a);
      if (++i >= n) break;
      load(a, nth(i + 2));
      work(b);
      if (++i >= n) break;
      load(b, nth(i + 2));
      work(c);
      if (++i >= n) break;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) part[wave][t][lane] = y[t];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 16 * NT; i += 512) {
    const int row = i / (16 * NT), t = i / 16 % NT, ch = i % 16;
    const int64_t at = (tile0 + t) * 16 + ch;
    if (row >= m || at >= p.n) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += part[w][t][ch + 16 * (row / 4)][row % 4];
    p.y[row * p.n + at] = static_cast<uint16_t>(pack_bf16(sum, 0.f));
  }
}

// ---- tiles -----------------------------------------------------------------------------------------------------------
//
// TM tokens x TN channels a workgroup, K in steps of 64. A step's x goes straight from memory into one of two stages of
// LDS, its weights from codes in registers through (c - z) s in fp32, rounded to bf16, into the same stage, once for all
// the tile's rows; both while the other stage is multiplied, with one barrier a step. Row R's 16-byte chunk c lies at slot
// c ^ (R / 2 % 8), which spreads the 16 rows that a phase of ds_read_b128 touches over all banks. AHEAD units of codes
// are in registers or on their way.
//
// Rounding the weights is what lets the matrix cores sum over groups: an error of 2^-9 of each at most, 0.0022 of the
// result in relative norm where the output's own rounding is 0.0017.
// v_mfma_f32_32x32x16_bf16 takes the channels as rows and the tokens as columns, so a lane ends with four neighbouring
// channels of a token at a time; they reach y through LDS, in whole lines.

// Eight codes as weights, s c + b.
__device__ __forceinline__ u32x4 weights(uint32_t w, float s, float b) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = w >> 4 & 0x0f0f0f0fu;
  const auto value = [&](uint32_t v, int byte) { return fmaf(static_cast<float>(v >> (8 * byte) & 255u), s, b); };
  return (u32x4){pack_bf16(value(lo, 0), value(lo, 2)), pack_bf16(value(hi, 0), value(hi, 2)),
                 pack_bf16(value(lo, 1), value(lo, 3)), pack_bf16(value(hi, 1), value(hi, 3))};
}

template <int TM, int TN, int WM, int WN, int AHEAD, int PARTS, bool ZERO, bool SPLIT>
__global__ __launch_bounds__(WM * WN * kWave, 2) void int4_tile_kernel(Int4Linear p) {
  constexpr int kWaves = WM * WN;
  constexpr int kStep = 128;                       // bytes of a row: 64 inputs
  constexpr int kStage = (TM + TN) * kStep;
  constexpr int kLoads = TM / 8 / kWaves;          // of one wave, 8 rows of x each
  constexpr int kUnits = TN / 16 / kWaves;         // tiles of 16 channels that one wave makes the weights of
  constexpr int kMT = TM / WM / 32, kNT = TN / WN / 32;
  static_assert(TM / 8 % kWaves == 0 && TN / 16 % kWaves == 0, "every wave has the same to load");
  __shared__ __align__(1024) uint8_t lds[2 * kStage];
  const uint32_t per_xcd = (p.items + p.xcds - 1) / p.xcds;
  uint32_t item = (blockIdx.x % p.xcds) * per_xcd + blockIdx.x / p.xcds;
  if (blockIdx.x / p.xcds >= per_xcd || item >= p.items) return;
  const int split = SPLIT ? uniform(item % static_cast<uint32_t>(p.splits)) : 0;
  if (SPLIT) item /= static_cast<uint32_t>(p.splits);
  const uint32_t run = item / (p.band * p.n_tiles), at = item - run * p.band * p.n_tiles;
  const uint32_t rows = min(static_cast<uint32_t>(p.band), p.m_tiles - run * p.band);
  const int64_t m0 = static_cast<int64_t>(uniform(run * p.band + at % rows)) * TM;
  const int64_t n0 = static_cast<int64_t>(uniform(at / rows)) * TN;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 31, g = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;

  // Load i of a wave brings rows 8 (i kWaves + wave) .. + 7 of 128 bytes; rows past the last and inputs past K are 0.
  const uint8_t *tokens = reinterpret_cast<const uint8_t *>(p.x + m0 * p.x_stride);
  const uint32_t token_bytes = static_cast<uint32_t>(
      least(((least(p.m - m0, TM) - 1) * p.x_stride + p.k) * 2, 0x7fffffff));
  uint32_t offset[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int R = (i * kWaves + wave) * 8 + lane / 8;
    offset[i] = R * static_cast<uint32_t>(p.x_stride * 2) + ((lane % 8) ^ (R / 2 % 8)) * 16;
  }
  const auto issue = [&](int step) {
    uint8_t *base = lds + step % 2 * kStage + wave * 1024;
    const bool whole = (step + 1) * 64 <= p.k;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int R = (i * kWaves + wave) * 8 + lane / 8;
      const int chunk = (lane % 8) ^ (R / 2 % 8);
      load_to_lds(tokens, token_bytes, whole || step * 64 + chunk * 8 < p.k ? offset[i] : 0xf0000000u, step * kStep,
                  base + i * kWaves * 1024);
    }
  };

  struct Unit {  // 128 inputs of a channel each
    u32x4 w[kUnits];
    Scales<PARTS> s[kUnits], z[ZERO ? kUnits : 1];
  };
  Unit units[AHEAD];
  const int64_t tile0 = n0 / 16 + wave;
  const int cr = lane & 15, cq = lane >> 4;
  const auto load = [&](Unit &v, int u) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t of = least(tile0 + i * kWaves, p.tiles - 1) * p.units + u;
      v.w[i] = *reinterpret_cast<const u32x4 *>(p.w + of * kUnitBytes + lane * 16);
      v.s[i].load(p.scale + (of * 16 + cr) * PARTS);
      if (ZERO) v.z[i].load(p.zero + (of * 16 + cr) * PARTS);
    }
  };
  const auto store = [&](const Unit &v, int half) {  // the weights of one step
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int R = (i * kWaves + wave) * 16 + cr;
      uint8_t *to = lds + half * kStage + (TM + R) * kStep;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int word = 2 * half + j, part = word * PARTS / 4;
        const float s = v.s[i][part], b = -s * (ZERO ? v.z[i][part] : 8.f);
        *reinterpret_cast<u32x4 *>(to + ((4 * j + cq) ^ (R / 2 % 8)) * 16) = weights(v.w[i][word], s, b);
      }
    }
  };

  uint32_t a_at[kNT], b_at[kMT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) a_at[i] = (TM + wn * kNT * 32 + i * 32 + r) * kStep;
#pragma unroll
  for (int j = 0; j < kMT; ++j) b_at[j] = (wm * kMT * 32 + j * 32 + r) * kStep;
  const uint32_t swizzle = r / 2 % 8;
  f32x16 acc[kNT][kMT];
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int j = 0; j < kMT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const auto multiply = [&](int half) {
    const uint8_t *stage = lds + half * kStage;
    bf16x8 a[2][kNT], b[2][kMT];  // operands of 16 inputs, the next ones read during this one's products
    const auto read = [&](int ks) {
      const uint32_t chunk = ((2 * ks + g) ^ swizzle) * 16;
#pragma unroll
      for (int i = 0; i < kNT; ++i) a[ks & 1][i] = *reinterpret_cast<const bf16x8 *>(stage + a_at[i] + chunk);
#pragma unroll
      for (int j = 0; j < kMT; ++j) b[ks & 1][j] = *reinterpret_cast<const bf16x8 *>(stage + b_at[j] + chunk);
    };
    read(0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < 3) read(ks + 1);
#pragma unroll
      for (int j = 0; j < kMT; ++j)
#pragma unroll
        for (int i = 0; i < kNT; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[ks & 1][i], b[ks & 1][j], acc[i][j], 0, 0, 0);
    }
  };

  // A unit is two steps, the first in stage 0. Weights are made a step ahead: the unit's second half during its first
  // step, the next unit's first half during its second one.
  const int first = SPLIT ? split * p.split_units : 0;
  const int end = SPLIT ? min(p.units, first + p.split_units) : p.units;
  const auto at_most = [&](int u) { return min(u, end - 1); };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(units[i], at_most(first + i));
  issue(2 * first);
  store(units[0], 0);
  for (int u0 = first; u0 < end; u0 += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int u = u0 + i;
      if (u >= end) break;
      wait_vmcnt<0>();
      ring_barrier();
      issue(2 * u + 1);
      store(units[i], 1);
      load(units[i], at_most(u + AHEAD));
      multiply(0);
      wait_vmcnt<0>();
      ring_barrier();
      if (u + 1 < end) {
        issue(2 * u + 2);
        store(units[(i + 1) % AHEAD], 0);
      }
      multiply(1);
    }
  }

  if (SPLIT) {  // sums [split][m][n]
#pragma unroll
    for (int j = 0; j < kMT; ++j) {
      const int64_t t = m0 + wm * kMT * 32 + j * 32 + r;
      if (t >= p.m) continue;
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t ch = n0 + wn * kNT * 32 + i * 32 + 8 * e + 4 * g;
          if (ch < p.part_stride)
            *reinterpret_cast<f32x4 *>(p.part + (split * p.m + t) * p.part_stride + ch) =
                (f32x4){acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
        }
    }
    return;
  }
  // 32 tokens x the wave's channels at a time through this wave's part of LDS, 16 bytes between rows against conflicts
  constexpr int kPitch = kNT * 64 + 16;
  static_assert(32 * kPitch * kWaves <= 2 * kStage, "the epilogue fits the stages");
  __syncthreads();  // the last step has been read
  uint8_t *mine = lds + wave * 32 * kPitch;
#pragma unroll
  for (int j = 0; j < kMT; ++j) {
    const int64_t t0 = m0 + wm * kMT * 32 + j * 32;
    const int64_t c0 = n0 + wn * kNT * 32;
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<u32x2 *>(mine + r * kPitch + (i * 32 + 8 * e + 4 * g) * 2) =
            (u32x2){pack_bf16(acc[i][j][4 * e], acc[i][j][4 * e + 1]),
                    pack_bf16(acc[i][j][4 * e + 2], acc[i][j][4 * e + 3])};
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    constexpr int kLanes = kNT * 4;  // 16 bytes each, of one token
#pragma unroll
    for (int i = 0; i < 32 * kLanes / kWave; ++i) {
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

template <int PARTS, bool ZERO, int NT>
void start_rows(const Int4Linear &p, hipStream_t stream) {
  hipLaunchKernelGGL((int4_rows_kernel<NT, PARTS, ZERO>), dim3(p.items), dim3(512), 0, stream, p);
}

template <int PARTS, bool ZERO, int TM, int TN, int WM, int WN, int AHEAD>
void start_tiles(const Int4Linear &p, hipStream_t stream) {
  const dim3 grid((p.items + p.xcds - 1) / p.xcds * p.xcds), block(WM * WN * kWave);
  if (p.splits > 1)
    hipLaunchKernelGGL((int4_tile_kernel<TM, TN, WM, WN, AHEAD, PARTS, ZERO, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((int4_tile_kernel<TM, TN, WM, WN, AHEAD, PARTS, ZERO, false>), grid, block, 0, stream, p);
}

template <int PARTS, bool ZERO>
void start(const Int4Linear &p, hipStream_t stream) {
  switch (p.tile_m) {
    case 16:
      if (p.row_tiles == 1) start_rows<PARTS, ZERO, 1>(p, stream);
      else if (p.row_tiles == 2) start_rows<PARTS, ZERO, 2>(p, stream);
      else start_rows<PARTS, ZERO, 4>(p, stream);
      break;
    case 64: start_tiles<PARTS, ZERO, 64, 128, 1, 4, 4>(p, stream); break;
    case 128: start_tiles<PARTS, ZERO, 128, 128, 2, 2, 2>(p, stream); break;
    default: start_tiles<PARTS, ZERO, 256, 256, 2, 4, 2>(p, stream); break;
  }
}

}  // namespace

void plan_int4_linear(Int4Linear *p, int cus, int xcds) {
  p->xcds = std::max(1, xcds);
  p->tiles = (p->n + 15) / 16;
  p->units = static_cast<int>((p->k + kUnit - 1) / kUnit);
  p->part_stride = (p->n + 3) / 4 * 4;
  p->splits = 1;
  p->part_bytes = 0;
  if (p->m <= 16) {
    p->tile_m = 16;
    p->row_tiles = p->m > 8 && p->tiles >= 4 * cus ? 4 : p->m > 2 && p->tiles >= 2 * cus ? 2 : 1;
    p->items = static_cast<uint32_t>((p->tiles + p->row_tiles - 1) / p->row_tiles);
    return;
  }
  int64_t best = INT64_MAX, splits = 1;
  int tile_n = 128;
  const int64_t reading = p->n * p->k / 100000;
  const auto weigh = [&](int tm, int tn, int64_t alone, int64_t shared, int64_t start_cost) {
    const int64_t tiles = ((p->m + tm - 1) / tm) * ((p->n + tn - 1) / tn);
    for (int64_t s = 1; s <= 16 && (s == 1 || p->units / s >= 2); s *= 2) {
      const int64_t items = tiles * s, length = (p->units + s - 1) / s;
      const int64_t rounds = (items + cus - 1) / cus;
      const int64_t products = tm == 256 ? rounds * length * (rounds == 1 ? alone : shared)
                                         : length * std::max(alone, shared * items / cus);
      const int64_t cost = std::max(products, reading) + start_cost + (s > 1 ? 250 + p->m * p->n * s / 5000 : 0);
      if (cost >= best) continue;
      best = cost;
      splits = s;
      p->tile_m = tm;
      tile_n = tn;
    }
  };
  weigh(64, 128, 60, 45, 400);
  if (p->m > 64) weigh(128, 128, 110, 90, 700);
  if (p->m > 128) weigh(256, 256, 280, 320, 1000);
  p->m_tiles = static_cast<uint32_t>((p->m + p->tile_m - 1) / p->tile_m);
  p->n_tiles = static_cast<uint32_t>((p->n + tile_n - 1) / tile_n);
  const uint32_t runs = (p->m_tiles + 11) / 12;
  p->band = static_cast<int>((p->m_tiles + runs - 1) / runs);
  p->split_units = static_cast<int>((p->units + splits - 1) / splits);
  p->splits = static_cast<int>((p->units + p->split_units - 1) / p->split_units);
  const int64_t items = static_cast<int64_t>(p->m_tiles) * p->n_tiles * p->splits;
  p->items = static_cast<uint32_t>(std::min<int64_t>(items, UINT32_MAX));  // too many for a launch: the caller refuses
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
