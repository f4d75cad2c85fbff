// Matrix product of 8-bit integers with a scale for each token and each channel, written for gfx950.
//
//   y[m, n] = bf16(s_x[m] s_w[n] sum_k c[m, k] w[n, k]),   c = round(x / s_x),  s_x = max_k |x| / 127
//
// x is bf16 [M, K], w int8 [N, K] (-127 .. 127, K contiguous), s_w fp32 [N]. The sums are exact 32-bit integers
// (K is at most 131072, so 127^2 K fits), whatever their order; the scales are applied in fp32 and the result is
// rounded once.
//
// int8_quantize_kernel writes c into rows of a multiple of 256 bytes whose ends are 0. The products' loads then
// need no care at the end of K: what they read of w past it, the start of the next row, meets zeros. Loads past the
// last row come back as 0 from the buffer descriptor.
#include <algorithm>
#include <cfloat>

#include "ftx_internal.h"

namespace ftx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kWave = 64;
constexpr float kTiny = 0x1p-100f;  // a scale below this counts as 0

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ __forceinline__ float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N < 64, "vmcnt holds six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

__device__ __forceinline__ void ring_barrier() {
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's LDS reads are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// (min of 64-bit integers would go through doubles)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

// A quotient or remainder of a workgroup's number, computed on the vector unit, as the scalar that it is.
__device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(static_cast<int>(v)); }

// 16 bytes per lane from base + offset + step into lds + 16 * lane; zeros where that is not below `bytes`.
__device__ __forceinline__ void load_to_lds(const uint8_t *base, uint32_t bytes, uint32_t offset, uint32_t step,
                                            uint8_t *lds) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, bytes, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)lds, 16, offset, step, 0, 0);
}

// ---- codes and scales of the rows --------------------------------------------------------------------------------
//
// The largest magnitude's bits order as integers, and a NaN's are above all: a row that holds an infinity or a NaN
// gets the scale NaN, and codes of 0. A row of up to 8192 values is held in the registers of 256 threads, of up to
// 32768 of 1024 (one row of 28672: 7.6 us with 256 threads that read it twice); what is longer is read twice, and so are
// the long rows of a call with too many of them for one launch of 1024 threads each.

__device__ __forceinline__ uint32_t largest8(u32x4 v, uint32_t top) {
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(v[i] & 0x7fffu, v[i] >> 16 & 0x7fffu));
  return top;
}

// The largest of a wave's values, in every lane: pairs, quads, eights and sixteens of lanes, then the four sixteens.
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
  const auto with = [&](auto other) { v = max(v, static_cast<uint32_t>(other)); };
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 15, 15, true));   // quad_perm 1 0 3 2
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4e, 15, 15, true));   // quad_perm 2 3 0 1
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 15, 15, true));  // row_half_mirror
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 15, 15, true));  // row_mirror
  const auto lane = [&](int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), i)); };
  return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}

// The scale of a row whose largest magnitude has these bf16 bits, and what its values are multiplied by.
__device__ __forceinline__ float row_scale(uint32_t top, float *inverse) {
#pragma clang fp contract(off)
  const float made = bf16_value(top) * (1.0f / 127.0f);
  const float scale = made < kTiny ? 0.f : made;
  *inverse = top >= 0x7f80u || scale == 0.f ? 0.f : 1.0f / scale;
  return top >= 0x7f80u ? __uint_as_float(0x7fc00000u) : scale;
}

__device__ __forceinline__ uint32_t code2(uint32_t pair, float inverse) {
#pragma clang fp contract(off)
  const float lo = rintf(bf16_value(pair) * inverse), hi = rintf(__uint_as_float(pair & 0xffff0000u) * inverse);
  const int a = static_cast<int>(fminf(fmaxf(lo, -127.f), 127.f)), b = static_cast<int>(fminf(fmaxf(hi, -127.f), 127.f));
  return (static_cast<uint32_t>(a) & 255u) | (static_cast<uint32_t>(b) & 255u) << 8;
}

__device__ __forceinline__ u32x2 code8(u32x4 v, float inverse) {
  return inverse == 0.f ? (u32x2){0u, 0u}  // an infinity times 0 is none
                        : (u32x2){code2(v[0], inverse) | code2(v[1], inverse) << 16,
                                  code2(v[2], inverse) | code2(v[3], inverse) << 16};
}

constexpr int kHeld = 4;  // vectors of 8 values that a thread keeps

template <int THREADS>
__global__ __launch_bounds__(THREADS) void int8_quantize_kernel(const uint16_t *__restrict__ x, int64_t x_stride,
                                                                uint8_t *__restrict__ codes, int64_t code_stride,
                                                                float *__restrict__ scales, int k) {
  __shared__ uint32_t wave_top[THREADS / kWave];
  const int64_t row = blockIdx.x;
  const u32x4 *xr = reinterpret_cast<const u32x4 *>(x + row * x_stride);
  const int n = k / 8, first = threadIdx.x;
  u32x4 held[kHeld];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held[i] = (u32x4){0u, 0u, 0u, 0u};
    if (first + i * THREADS < n) held[i] = xr[first + i * THREADS];
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) top = largest8(held[i], top);
  for (int i = first + kHeld * THREADS; i < n; i += THREADS) top = largest8(xr[i], top);
  top = wave_largest(top);
  if (threadIdx.x % kWave == 0) wave_top[threadIdx.x / kWave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / kWave; ++i) top = max(top, wave_top[i]);
  float inverse;
  const float scale = row_scale(top, &inverse);
  u32x2 *to = reinterpret_cast<u32x2 *>(codes + row * code_stride);
  const int end = static_cast<int>(code_stride / 8);  // past n the row ends in zeros
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (first + i * THREADS < end) to[first + i * THREADS] = code8(held[i], inverse);
  for (int i = first + kHeld * THREADS; i < end; i += THREADS) to[i] = i < n ? code8(xr[i], inverse) : (u32x2){0u, 0u};
  if (threadIdx.x == 0) scales[row] = scale;
}

// ---- up to 16 rows -------------------------------------------------------------------------------------------------
//
// The codes lie in LDS; a workgroup then walks groups of 16 channels over the whole of K. Its eight waves take windows
// of 256 bytes of the channels in turn, straight into registers as the operands of v_mfma_i32_16x16x64_i8 (lane (r, g):
// 16 bytes of channel r), three windows in flight across the ends of groups, and their sums meet in LDS. Bound by the
// bytes of w.
//
// CODES bytes of LDS hold the rows, 16 bytes between them against conflicts. Where a row or a few make at most
// kHeldRows vectors of 8 values a thread (FUSED), each workgroup rounds x itself and there is no other launch.

constexpr int kWindow = 256;
constexpr int kHeldRow = 512 * 8;  // values of a row that this kernel's threads hold one vector each of
constexpr int kHeldRows = 8;       // that a thread may hold (4096 x 4096 of 8 rows: 9.1 us, with codes from a launch 9.4)
constexpr int kFusedCodes = kHeldRows * (kHeldRow + 16), kSomeCodes = 60 << 10, kMostCodes = 143 << 10;

template <bool FUSED, int CODES>
__global__ __launch_bounds__(512, CODES <= kSomeCodes ? 4 : 2) void int8_rows_kernel(Int8Linear p) {
  __shared__ __align__(16) uint8_t codes[CODES];
  __shared__ i32x4 part[2][8][kWave];
  __shared__ float row_scales[16];
  __shared__ uint32_t row_top[kHeldRows];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int m = static_cast<int>(p.m), pitch = p.code_stride + 16;
  const int windows = p.code_stride / kWindow, steps = (windows + 7) / 8;
  // thread: token t, channel ch of a group; lane t + 16 g of each wave's sums holds channels 4 g .. 4 g + 3
  const int t = threadIdx.x / 16, ch = threadIdx.x % 16;
  const uint32_t per_row = (p.k + kHeldRow - 1) / kHeldRow;
  const int items = m * per_row;
  u32x4 held[kHeldRows];
  if (FUSED) {  // ahead of the loads of w, which come in while the codes are made
#pragma unroll
    for (int j = 0; j < kHeldRows; ++j) {
      const int row = uniform(j / per_row), col = uniform(j % per_row);
      const auto x = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p.x + row * p.x_stride), 0,
                                                       row < m ? p.k * 2 : 0, 0x00027000);
      held[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                              x, col * kHeldRow * 2 + threadIdx.x * 16, 0, 0));
    }
    if (threadIdx.x < kHeldRows) row_top[threadIdx.x] = 0;
  }
  const auto scale_of = [&](uint32_t group) {
    const int64_t at = static_cast<int64_t>(group) * 16 + ch;
    return at < p.n ? p.w_scale[at] : 0.f;
  };
  float w_scale = scale_of(blockIdx.x);

  const uint32_t w_at = r * p.k + 16 * g;
  uint32_t load_group = blockIdx.x;
  int load_step = 0;
  const auto load = [&](u32x4 (&w)[4]) {  // the next window; zeros past the row's end for this wave and past the last group
    const int64_t n0 = static_cast<int64_t>(load_group) * 16;
    const int rows = load_group < p.items ? static_cast<int>(least(16, p.n - n0)) : 0;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p.w + (rows > 0 ? n0 * p.k : 0)), 0,
                                                        rows * p.k, 0x00027000);
    const int window = load_step * 8 + wave;
    const uint32_t at = window < windows ? w_at + window * kWindow : 0x40000000u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 64 * i, 0, 0));
    if (++load_step == steps) load_step = 0, load_group += p.groups;
  };
  u32x4 x[4], y[4], z[4];
  load(x);
  load(y);

  if (FUSED) {
    ring_barrier();
#pragma unroll
    for (int j = 0; j < kHeldRows; ++j) {
      if (j >= items) break;
      const uint32_t top = wave_largest(largest8(held[j], 0));
      if (lane == 0) atomicMax(&row_top[uniform(j / per_row)], top);
    }
    ring_barrier();
#pragma unroll
    for (int j = 0; j < kHeldRows; ++j) {
      if (j >= items) break;
      const int row = uniform(j / per_row), at = uniform(j % per_row) * kHeldRow + threadIdx.x * 8;
      float inverse;
      const float scale = row_scale(row_top[row], &inverse);
      if (at < p.code_stride) *reinterpret_cast<u32x2 *>(codes + row * pitch + at) = code8(held[j], inverse);
      if (threadIdx.x == 0) row_scales[row] = scale;
    }
  } else {
    constexpr int kBatch = 8;
    const uint32_t of_row = p.code_stride / 16, all = m * of_row;
    const u32x4 *from = reinterpret_cast<const u32x4 *>(p.codes);
    for (uint32_t first = threadIdx.x; first < all; first += 512 * kBatch) {
      u32x4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) v[i] = from[min(first + i * 512, all - 1)];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t at = min(first + i * 512, all - 1);  // the last one again: the same bytes
        *reinterpret_cast<u32x4 *>(codes + at * 16 + at / of_row * 16) = v[i];
      }
    }
    if (threadIdx.x < m) row_scales[threadIdx.x] = p.x_scale[threadIdx.x];
  }
  ring_barrier();

  const uint32_t c_at = min(r, m - 1) * pitch + 16 * g;
  i32x4 acc = {0, 0, 0, 0};
  uint32_t group = blockIdx.x;
  int step = 0, side = 0;
  const auto work = [&](const u32x4 (&w)[4]) {  // returns whether it was the last one
    const uint8_t *c = codes + c_at + min(step * 8 + wave, windows - 1) * kWindow;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w[i]),
                                                  *reinterpret_cast<const i32x4 *>(c + 64 * i), acc, 0, 0, 0);
    if (++step < steps) return false;
    part[side][wave][lane] = acc;
    ring_barrier();  // the other side's sums have been read by all
    const int64_t at = static_cast<int64_t>(group) * 16 + ch;
    if (t < m && at < p.n) {
      int sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += part[side][i][t + 16 * (ch / 4)][ch % 4];
      p.y[t * p.n + at] = static_cast<uint16_t>(pack_bf16(static_cast<float>(sum) * row_scales[t] * w_scale, 0.f));
    }
    acc = (i32x4){0, 0, 0, 0};
    step = 0;
    side ^= 1;
    group += p.groups;
    w_scale = scale_of(group);
    return group >= p.items;
  };
  for (;;) {
    load(z);
    if (work(x)) break;
    load(x);
    if (work(y)) break;
    load(y);
    if (work(z)) break;
  }
}

// ---- tiles -----------------------------------------------------------------------------------------------------------
//
// TM tokens x TN channels a workgroup, K in steps of 128. A step's rows go straight from memory into one of STAGES
// stages of LDS; row R's 16-byte chunk c lies at slot c ^ (R / 2 % 8), which spreads the 16 rows that a phase of
// ds_read_b128 touches over all banks. The other stages' loads are in flight during a step's products: one step's
// where many rows keep the matrix cores busy, two where w's bytes are what takes time (28672 x 8192 of 32 rows in
// tiles of 64 x 128: 60.7 us with two stages, 50.3 with three, 50.2 with four).
// v_mfma_i32_32x32x32_i8 takes the channels as rows and the tokens as columns, so a lane ends with four neighbouring
// channels of a token at a time; they reach y through LDS, in whole lines.

template <int TM, int TN, int WM, int WN, int STAGES, bool SPLIT>
__global__ __launch_bounds__(WM * WN * kWave, 2) void int8_tile_kernel(Int8Linear p) {
  constexpr int kWaves = WM * WN;
  constexpr int kStep = 128;
  constexpr int kStage = (TM + TN) * kStep;
  constexpr int kLoads = kStage / 1024 / kWaves;   // of one wave
  constexpr int kMT = TM / WM / 32, kNT = TN / WN / 32;
  constexpr int kTokenLoads = TM / 8 / kWaves;     // the first of them
  static_assert(kStage / 1024 % kWaves == 0 && TM / 8 % kWaves == 0, "every wave issues the same loads");
  __shared__ __align__(1024) uint8_t lds[STAGES * kStage];
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
  // Load i of a wave brings rows 8 (i kWaves + wave) .. + 7 of 128 bytes, the tokens' first, then the channels'.
  const uint8_t *tokens = p.codes + m0 * p.code_stride, *channels = p.w + n0 * p.k;
  const uint32_t token_bytes = static_cast<uint32_t>(least((p.m - m0) * p.code_stride, 0x7fffffff));
  const uint32_t channel_bytes = static_cast<uint32_t>(least((p.n - n0) * p.k, 0x7fffffff));
  uint32_t offset[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int R = (i * kWaves + wave) * 8 + lane / 8 - (i < kTokenLoads ? 0 : TM);
    offset[i] = R * (i < kTokenLoads ? p.code_stride : p.k) + ((lane % 8) ^ (R / 2 % 8)) * 16;
  }
  const auto issue = [&](int step) {
    uint8_t *base = lds + step % STAGES * kStage + wave * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_to_lds(i < kTokenLoads ? tokens : channels, i < kTokenLoads ? token_bytes : channel_bytes, offset[i],
                  step * kStep, base + i * kWaves * 1024);
  };
  uint32_t a_at[kNT], b_at[kMT];
#pragma unroll
  for (int i = 0; i < kNT; ++i) a_at[i] = TM * kStep + (wn * kNT * 32 + i * 32 + r) * kStep;
#pragma unroll
  for (int j = 0; j < kMT; ++j) b_at[j] = (wm * kMT * 32 + j * 32 + r) * kStep;
  const uint32_t swizzle = r / 2 % 8;

  i32x16 acc[kNT][kMT];
#pragma unroll
  for (int i = 0; i < kNT; ++i)
#pragma unroll
    for (int j = 0; j < kMT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  const int all = (p.k + kStep - 1) / kStep;
  const int first = SPLIT ? split * p.split_steps : 0;
  const int end = SPLIT ? min(all, first + p.split_steps) : all;
  i32x4 a[2][kNT], b[2][kMT];  // operands of 32 of K, the next ones read during this one's products
  const auto read = [&](int step, int ks) {
    const uint8_t *stage = lds + step % STAGES * kStage;
    const uint32_t chunk = ((2 * ks + g) ^ swizzle) * 16;
#pragma unroll
    for (int i = 0; i < kNT; ++i) a[ks & 1][i] = *reinterpret_cast<const i32x4 *>(stage + a_at[i] + chunk);
#pragma unroll
    for (int j = 0; j < kMT; ++j) b[ks & 1][j] = *reinterpret_cast<const i32x4 *>(stage + b_at[j] + chunk);
  };
  const auto multiply = [&](int ks) {
#pragma unroll
    for (int j = 0; j < kMT; ++j)
#pragma unroll
      for (int i = 0; i < kNT; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[ks & 1][i], b[ks & 1][j], acc[i][j], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int kLast = kStep / 32 - 1;
  // vmcnt counts this wave's loads: the ones of the steps after the one that is waited for may be on their way
#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (first + i < end) issue(first + i);
  if (first + STAGES <= end) wait_vmcnt<(STAGES - 1) * kLoads>();
  else wait_vmcnt<0>();
  ring_barrier();
  read(first, 0);
  for (int step = first; step < end; ++step) {
#pragma unroll
    for (int ks = 0; ks < kLast; ++ks) {
      read(step, ks + 1);
      multiply(ks);
    }
    if (step + 1 < end) {  // the stage has been read by all: the barrier and the next one's first reads meet its last products
      if (step + STAGES <= end) wait_vmcnt<(STAGES - 2) * kLoads>();
      else wait_vmcnt<0>();
      ring_barrier();
      if (step + STAGES < end) issue(step + STAGES);
      read(step + 1, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(kLast);
  }

  if (SPLIT) {  // integer sums [split][m][n]
#pragma unroll
    for (int j = 0; j < kMT; ++j) {
      const int64_t t = m0 + wm * kMT * 32 + j * 32 + r;
      if (t >= p.m) continue;
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t ch = n0 + wn * kNT * 32 + i * 32 + 8 * q + 4 * g;
          int *to = p.part + (split * p.m + t) * p.part_stride + ch;
          if (ch < p.part_stride)
            *reinterpret_cast<i32x4 *>(to) = (i32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
    }
    return;
  }
  // 32 tokens x the wave's channels at a time through this wave's part of LDS, 16 bytes between rows against conflicts
  constexpr int kPitch = kNT * 64 + 16;
  static_assert(32 * kPitch * kWaves <= STAGES * kStage, "the epilogue fits the stages");
  __syncthreads();  // the last step has been read
  uint8_t *mine = lds + wave * 32 * kPitch;
#pragma unroll
  for (int j = 0; j < kMT; ++j) {
    const int64_t t0 = m0 + wm * kMT * 32 + j * 32;
    const int64_t c0 = n0 + wn * kNT * 32;
    const float x_scale = t0 + r < p.m ? p.x_scale[t0 + r] : 0.f;
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t ch = c0 + i * 32 + 8 * q + 4 * g + e;
          y[e] = static_cast<float>(acc[i][j][4 * q + e]) * x_scale * (ch < p.n ? p.w_scale[ch] : 0.f);
        }
        *reinterpret_cast<u32x2 *>(mine + r * kPitch + (i * 32 + 8 * q + 4 * g) * 2) =
            (u32x2){pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
      }
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

// y = bf16(s_x s_w sum over the splits), four channels a thread.
__global__ __launch_bounds__(256) void int8_join_kernel(Int8Linear p) {
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  const int64_t size = p.m * p.part_stride;
  if (at >= size) return;
  const int64_t t = at / p.part_stride, ch = at % p.part_stride;
  i32x4 sum = {0, 0, 0, 0};
  for (int i = 0; i < p.splits; ++i) sum += *reinterpret_cast<const i32x4 *>(p.part + i * size + at);
  const float x_scale = p.x_scale[t];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (ch + e < p.n)
      p.y[t * p.n + ch + e] = static_cast<uint16_t>(pack_bf16(static_cast<float>(sum[e]) * x_scale * p.w_scale[ch + e], 0.f));
}

template <int TM, int TN, int WM, int WN, int STAGES>
void start_tiles(const Int8Linear &p, hipStream_t stream) {
  const dim3 grid((p.items + p.xcds - 1) / p.xcds * p.xcds), block(WM * WN * kWave);
  if (p.splits > 1) hipLaunchKernelGGL((int8_tile_kernel<TM, TN, WM, WN, STAGES, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((int8_tile_kernel<TM, TN, WM, WN, STAGES, false>), grid, block, 0, stream, p);
}

}  // namespace

hipError_t launch_int8_quantize(const uint16_t *x, int64_t x_stride, uint8_t *codes, int64_t code_stride, float *scales,
                                int64_t m, int k, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(m));
  if (k <= 8192 || m > kMaxThreads / 1024)
    hipLaunchKernelGGL(int8_quantize_kernel<256>, grid, dim3(256), kLdsToken, stream, x, x_stride, codes, code_stride,
                       scales, k);
  else
    hipLaunchKernelGGL(int8_quantize_kernel<1024>, grid, dim3(1024), kLdsToken, stream, x, x_stride, codes,
                       code_stride, scales, k);
  return hipGetLastError();
}

// Which kernel and how often K is split, by what it costs in 0.01 us: the larger of the products (a step of 128 of K
// takes a workgroup `alone` at least, a CU `shared` for each of its workgroups) and of reading w (5.3 TB/s), a start,
// and the join of the splits. Tiles of 256 x 256 have a CU to themselves, so theirs come in whole rounds.
//                    alone  shared  start
//   64 x 128            45      41     400
//   128 x 128           95      64     700
//   256 x 256     150, 190 in more rounds than one     1000
// Measured, us: 28672 x 8192 of 32 rows 50.3 in tiles of 64, 54.3 split in two; 8192 x 28672 106.7, in four 44.8; 4096
// x 4096 17.7 and 11.2. 28672 x 8192 of 200 rows 118, 74.6 and 101 in tiles of 64, 128 and 256, of 512 rows 193, 150 and
// 114, of 1000 360, 292 and 239; 8192 x 28672 of 512 rows 131 in tiles of 256 split in four, 164 in tiles of 128 split
// in two. Up to 16 rows whose codes fit LDS have the kernel without tiles: 28672 x 8192 of 1, 4, 8 and 16 rows 41, 44, 45
// and 47, in tiles 49 and 50; 4096 x 4096 6, 7, 9 and 10, in tiles 13 and 14. Rows of fewer windows than waves leave
// some of these idle: 28672 x 1024 of one row 10.9 (tiles: 11.5), of 16, whose codes take a launch, 13.5 and 11.9.
void plan_int8_linear(Int8Linear *p, bool from_x, int cus, int xcds) {
  p->xcds = std::max(1, xcds);
  p->part_stride = (p->n + 3) / 4 * 4;
  const int64_t steps = std::max(1, (p->k + 127) / 128);
  const int64_t reading = p->n * p->k / 53000;
  int64_t best = INT64_MAX, splits = 1;
  const auto weigh = [&](int tm, int tn, int64_t alone, int64_t shared, int64_t start) {
    const int64_t tiles = ((p->m + tm - 1) / tm) * ((p->n + tn - 1) / tn);
    for (int64_t s = 1; s <= 16 && (s == 1 || steps / s >= 2); s *= 2) {
      const int64_t items = tiles * s, length = (steps + s - 1) / s;
      const int64_t rounds = (items + cus - 1) / cus;
      const int64_t products = tm == 256 ? rounds * length * (rounds == 1 ? alone : shared)
                                         : length * std::max(alone, shared * items / cus);
      const int64_t cost = std::max(products, reading) + start +
                           (s > 1 ? 250 + p->m * p->n * s / 5000 : 0);
      if (cost >= best) continue;
      best = cost;
      splits = s;
      p->tile_m = tm;
      p->tile_n = tn;
    }
  };
  weigh(64, 128, 45, 41, 400);
  if (p->m > 64) weigh(128, 128, 95, 64, 700);
  if (p->m > 128) weigh(256, 256, 150, 190, 1000);
  const int64_t code_bytes = p->m * (p->code_stride + 16), windows = p->code_stride / kWindow;
  p->one_launch = from_x && p->m <= 16 && p->m * ((p->k + kHeldRow - 1) / kHeldRow) <= kHeldRows;
  if (p->m <= 16 && p->k > 0 && code_bytes <= kMostCodes &&
      reading * (16 - std::min<int64_t>(8, windows)) / 8 + (p->one_launch ? 0 : 250) <= best) {
    p->tile_m = 16;
    p->splits = 1;
    p->items = static_cast<uint32_t>((p->n + 15) / 16);
    // Two workgroups a CU take every place there is (10240 x 8192 of one row 18.4, in equal rounds 21.8), one a CU
    // equal rounds (of 16 rows 21.8, 23.1 with every place taken).
    const bool two = code_bytes <= kSomeCodes;
    const uint32_t slots = cus * (two ? 2 : 1), rounds = (p->items + slots - 1) / slots;
    p->groups = two ? std::min(slots, p->items) : (p->items + rounds - 1) / rounds;
    p->part_bytes = 0;
    return;
  }
  p->one_launch = false;
  p->m_tiles = static_cast<uint32_t>((p->m + p->tile_m - 1) / p->tile_m);
  p->n_tiles = static_cast<uint32_t>((p->n + p->tile_n - 1) / p->tile_n);
  // An XCD walks a run of up to 12 tiles of tokens before its next tile of channels, equal runs: their codes and the
  // channels' are in its L2 for the others.
  const uint32_t runs = (p->m_tiles + 11) / 12;
  p->band = static_cast<int>((p->m_tiles + runs - 1) / runs);
  p->split_steps = static_cast<int>((steps + splits - 1) / splits);
  p->splits = static_cast<int>((steps + p->split_steps - 1) / p->split_steps);
  const int64_t items = static_cast<int64_t>(p->m_tiles) * p->n_tiles * p->splits;
  p->items = static_cast<uint32_t>(std::min<int64_t>(items, UINT32_MAX));  // too many for a launch: the caller refuses
  p->part_bytes = p->splits > 1 ? static_cast<size_t>(p->splits) * p->m * p->part_stride * 4 : 0;
}

hipError_t launch_int8_linear(const Int8Linear &p, hipStream_t stream) {
  switch (p.tile_m) {
    case 16:
      if (p.x) hipLaunchKernelGGL((int8_rows_kernel<true, kFusedCodes>), dim3(p.groups), dim3(512), 0, stream, p);
      else if (p.m * (p.code_stride + 16) <= kSomeCodes)
        hipLaunchKernelGGL((int8_rows_kernel<false, kSomeCodes>), dim3(p.groups), dim3(512), 0, stream, p);
      else hipLaunchKernelGGL((int8_rows_kernel<false, kMostCodes>), dim3(p.groups), dim3(512), 0, stream, p);
      break;
    case 64: start_tiles<64, 128, 1, 4, 3>(p, stream); break;
    case 128: start_tiles<128, 128, 2, 2, 2>(p, stream); break;
    default: start_tiles<256, 256, 2, 4, 2>(p, stream); break;
  }
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.splits == 1) return err;
  const int64_t threads = p.m * p.part_stride / 4;
  hipLaunchKernelGGL(int8_join_kernel, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), kLdsToken, stream,
                     p);
  return hipGetLastError();
}

}  // namespace ftx
