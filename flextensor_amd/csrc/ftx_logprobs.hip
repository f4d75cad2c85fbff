// Log probabilities of given tokens, entropy and the likeliest tokens of rows of logits, written for gfx950.
//
//   log p_i = (x_i - max) - log sum_j exp(x_j - max),   H = log sum - sum_j (x_j - max) exp(x_j - max) / sum
//
// over rows of bf16, fp16 or fp32 logits, all statistics in fp32. One pass: a thread keeps a running maximum, the sum of
// the exponentials and the sum of their products with the exponents, in units of log2, and rescales both sums when a
// batch of its values exceeds the maximum. An exponent is one fused multiply-add, y = x log2(e) - fl(m log2(e)); what the
// rounding of m's product puts into every y comes out of the sums at the end. That is 2^-24 of the product, so a thread
// whose maximum is above 2^16 in size takes the difference first, (x - m) log2(e), and nothing comes out: one masked by
// -1e30 would have 2^73 in every y. Bound by the exponentials and their sums, some nine cycles of a SIMD a value, close
// to what memory takes for bf16.
//
// The likeliest tokens are keys (the logit's bits in the order of unsigned integers, then the complement of the index):
// the largest keys are the largest logits, the lowest index first among equal ones, a NaN above all. The pass over the
// row keeps no more for them than each thread's maximum, the batch it was in and the largest value of the others. The
// threads form 64 groups (128 for a top of more than 32): as many values as groups' maxima reach the `top`th largest of
// these, so no token below it counts, and some 1.2 `top` values reach it. The threads whose own maximum does read that
// batch again (from the cache) and collect the keys in LDS, where one wave sorts them. Rows that more keys pass than LDS
// holds (many equal ones), or that are not finite, take another way: each wave keeps the 64 largest keys of what it
// reads sorted over its lanes.
#include <algorithm>
#include <cfloat>

#include "ftx_internal.h"

namespace ftx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kVecs = 2;  // 16-byte loads of a thread's batch

// A quotient or remainder of a workgroup's number, computed on the vector unit, as the scalar that it is.
__device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(static_cast<int>(v)); }

template <int TYPE>
struct Vec {  // the values of 16 bytes
  static constexpr int kValues = TYPE == FTX_LOGITS_FP32 ? 4 : 8;
  u32x4 w;
  __device__ __forceinline__ float pick(int i) const {  // of a number that is not known when this is compiled
    const int j = TYPE == FTX_LOGITS_FP32 ? i : i / 2;
    Vec one;
    one.w[0] = j & 2 ? j & 1 ? w[3] : w[2] : j & 1 ? w[1] : w[0];
    if constexpr (TYPE != FTX_LOGITS_FP32) one.w[0] >>= 16 * (i % 2);
    return one[0];
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (TYPE == FTX_LOGITS_FP32) return __uint_as_float(w[i]);
    if constexpr (TYPE == FTX_LOGITS_BF16) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)))));
  }
};

template <int TYPE>
__device__ __forceinline__ float value_at(const void *row, int64_t i) {
  if constexpr (TYPE == FTX_LOGITS_FP32) return static_cast<const float *>(row)[i];
  const uint16_t bits = static_cast<const uint16_t *>(row)[i];
  if constexpr (TYPE == FTX_LOGITS_BF16) return __uint_as_float(static_cast<uint32_t>(bits) << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, bits));
}

// Bits that order as the values do: -0 as 0, every NaN above +inf; 0 is below all of them.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : static_cast<int32_t>(b) < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o == 0xffffffffu ? 0x7fc00000u : o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, int64_t index) {
  return static_cast<Key>(ordered(x)) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(index));
}

// The value of lane ^ J, by moves within the vector registers.
template <int J>
__device__ __forceinline__ uint32_t across(uint32_t v, int lane) {
  const int x = static_cast<int>(v);
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(x, 0xb1, 15, 15, true);  // quad_perm 1 0 3 2
  if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(x, 0x4e, 15, 15, true);  // quad_perm 2 3 0 1
  if constexpr (J == 4)                                                          // eights mirrored, then quads
    return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(x, 0x141, 15, 15, true), 0x1b, 15, 15, true);
  if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(x, 0x128, 15, 15, true);  // row_ror 8
  if constexpr (J == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? s[0] : s[1];
  }
  const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return lane & 32 ? s[0] : s[1];
}
template <int J>
__device__ __forceinline__ Key across(Key v, int lane) {
  return static_cast<Key>(across<J>(static_cast<uint32_t>(v >> 32), lane)) << 32 |
         across<J>(static_cast<uint32_t>(v), lane);
}
template <int J>
__device__ __forceinline__ float across(float v, int lane) {
  return __uint_as_float(across<J>(__float_as_uint(v), lane));
}

// Sorts the lanes' keys, the largest first; clean() where they are bitonic.
template <int J, typename K>
__device__ __forceinline__ K exchange(K key, int lane, bool larger) {
  const K other = across<J>(key, lane);
  if constexpr (sizeof(K) == 4) return larger ? max(key, other) : min(key, other);
  return (key > other) == larger ? key : other;
}
template <typename K>
__device__ __forceinline__ K clean(K key, int lane) {
  key = exchange<32>(key, lane, !(lane & 32));
  key = exchange<16>(key, lane, !(lane & 16));
  key = exchange<8>(key, lane, !(lane & 8));
  key = exchange<4>(key, lane, !(lane & 4));
  key = exchange<2>(key, lane, !(lane & 2));
  return exchange<1>(key, lane, !(lane & 1));
}
template <int K2, int J, typename K>
__device__ __forceinline__ K sort_step(K key, int lane) {
  key = exchange<J>(key, lane, !(lane & J) == !(lane & K2));
  if constexpr (J > 1) return sort_step<K2, J / 2>(key, lane);
  return key;
}
template <typename K>
__device__ __forceinline__ K sorted(K key, int lane, int count = kWave) {  // the lanes from count on hold 0
  key = sort_step<2, 1>(key, lane);
  key = sort_step<4, 2>(key, lane);
  key = sort_step<8, 4>(key, lane);
  key = sort_step<16, 8>(key, lane);
  if (count <= 16) return key;
  key = sort_step<32, 16>(key, lane);
  return count <= 32 ? key : clean(key, lane);
}
// The 64 largest of two sorted lists.
__device__ __forceinline__ Key merged(Key a, Key b, int lane) {
  const Key other = __shfl(b, kWave - 1 - lane);
  return clean(a > other ? a : other, lane);
}

// A part of a row: its maximum m, sum of 2^y and sum of y 2^y, y = (x - m) log2(e).
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  const auto to = [&](Sums &x) {  // a part without a value adds nothing, whatever its maximum is
    const float y = (x.m - m) * kLog2e, w = x.s == 0.f ? 0.f : __builtin_amdgcn_exp2f(y);
    x.t = x.s == 0.f ? 0.f : (x.t + fmaxf(y, -1000.f) * x.s) * w;
    x.s *= w;
  };
  to(a);
  to(b);
  return {m, a.s + b.s, a.t + b.t};
}
// The lanes' maximum (a NaN is left out) and sum, in every lane.
__device__ __forceinline__ float wave_max(float v, int lane) {
  v = fmaxf(v, across<1>(v, lane));
  v = fmaxf(v, across<2>(v, lane));
  v = fmaxf(v, across<4>(v, lane));
  v = fmaxf(v, across<8>(v, lane));
  v = fmaxf(v, across<16>(v, lane));
  return fmaxf(v, across<32>(v, lane));
}
__device__ __forceinline__ float wave_sum(float v, int lane) {
  v += across<1>(v, lane);
  v += across<2>(v, lane);
  v += across<4>(v, lane);
  v += across<8>(v, lane);
  v += across<16>(v, lane);
  return v + across<32>(v, lane);
}
__device__ __forceinline__ Sums wave_joined(Sums x, int lane) {
  const float m = wave_max(x.m, lane);
  x = joined(x, {m, 0.f, 0.f});
  return {m, wave_sum(x.s, lane), wave_sum(x.t, lane)};
}

// A wave writes a row's results.
template <int TYPE>
__device__ __forceinline__ void write_row(const Logprobs &p, int64_t row, const void *x, Sums sums, Key key, int lane) {
  const float log_sum = logf(sums.s);
  if (lane == 0) {
    const int64_t token = p.tokens[row];
    float given = token < 0 ? 0.f : __uint_as_float(0x7fc00000u);
    if (token >= 0 && token < p.vocab) given = value_at<TYPE>(x, token) - sums.m - log_sum;
    p.logprob[row] = given;
    p.entropy[row] = log_sum - sums.t / sums.s * kLn2;
  }
  if (lane < p.top) {
    p.top_logprob[row * p.top + lane] = unordered(static_cast<uint32_t>(key >> 32)) - sums.m - log_sum;
    p.top_token[row * p.top + lane] = static_cast<uint32_t>(~static_cast<uint32_t>(key));
  }
}

// A part of a row as 16-byte units, counted from the boundary before the row: the values of the first and last one that
// are not the row's are left out (an aligned unit with a value of the row lies in its memory page). A thread's units are
// THREADS apart, and a batch of it kVecs of them.
template <int TYPE, int THREADS>
struct Part {
  static constexpr int kValues = Vec<TYPE>::kValues, kBatch = kVecs * kValues;
  const void *row;
  const u32x4 *units;
  int lead, vocab, end, plain;  // plain: units below it (but for the first after a lead) are the row's altogether

  // Whether the workgroup's batch from u on is of such units; the thread's first unit of it is u + its number.
  __device__ __forceinline__ bool is_plain(int u) const {
    return u + kVecs * THREADS <= plain && (u > 0 || lead == 0);
  }
  __device__ __forceinline__ void load(Vec<TYPE> (&v)[kVecs], int u) const {
    if (is_plain(u)) {
      const u32x4 *from = units + u;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) v[i].w = from[threadIdx.x + i * THREADS];
      return;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      v[i].w = units[min(u + static_cast<int>(threadIdx.x) + i * THREADS, end - 1)];
  }
  __device__ __forceinline__ int index(int u0, int value) const {
    return (u0 + value / kValues * THREADS) * kValues - lead + value % kValues;
  }
  static __device__ __forceinline__ void drop(Vec<TYPE> &v, int e) {
    if constexpr (TYPE == FTX_LOGITS_FP32) v.w[e] = 0xff800000u;
    else v.w[e / 2] = (v.w[e / 2] & (e % 2 ? 0xffffu : 0xffff0000u)) |
                      (TYPE == FTX_LOGITS_BF16 ? 0xff80u : 0xfc00u) << (16 * (e % 2));
  }
  // Which of a batch's values are the row's, a bit each; the others become -inf.
  __device__ __forceinline__ uint32_t trim(Vec<TYPE> (&v)[kVecs], int u) const {
    if (is_plain(u)) return kBatch == 32 ? ~0u : (1u << (kBatch % 32)) - 1;
    uint32_t valid = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int unit = u + static_cast<int>(threadIdx.x) + i * THREADS;
      uint32_t here = unit < end ? (1u << kValues) - 1 : 0;
      if (unit == 0) here = here >> lead << lead;
      if ((unit + 1) * kValues - lead > vocab) here &= (1u << max(0, vocab + lead - unit * kValues)) - 1;
      valid |= here << (i * kValues);
      if (__any(here != 0 && here != (1u << kValues) - 1)) {  // the first or last one
#pragma unroll
        for (int e = 0; e < kValues; ++e)
          if (!(here >> e & 1)) drop(v[i], e);
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (!here) v[i].w[w] = TYPE == FTX_LOGITS_FP32 ? 0xff800000u : TYPE == FTX_LOGITS_BF16 ? 0xff80ff80u : 0xfc00fc00u;
      }
    }
    return valid;
  }
};

// The 64 largest keys of a part, sorted in wave 0's lanes: every wave those of its units, 64 candidates at a time in its
// part of LDS, then two waves' lists at a time.
template <int TYPE, int THREADS>
__device__ __forceinline__ Key largest_keys(const Part<TYPE, THREADS> &part, int first, int top, Key *lists, int wave,
                                            int lane) {
  constexpr int kWaves = THREADS / kWave;
  Key *mine = lists + wave * 2 * kWave, list = 0;
  uint32_t threshold = 0;
  int held = 0;
  const auto merge = [&]() {
    const Key fresh = lane < held ? mine[lane] : 0;
    list = merged(list, sorted(fresh, lane), lane);
    const Key rest = mine[kWave + lane];
    held = max(held - kWave, 0);
    if (lane < held) mine[lane] = rest;
    threshold = static_cast<uint32_t>(__shfl(list, top - 1) >> 32);
  };
  for (int u = first; u < part.end; u += kVecs * THREADS) {
    const int u0 = u + wave * kWave + lane;
    Vec<TYPE> v[kVecs];
    part.load(v, u);
    uint32_t passed = part.trim(v, u);
#pragma unroll
    for (int i = 0; i < part.kBatch; ++i)
      if (ordered(v[i / part.kValues][i % part.kValues]) <= threshold) passed &= ~(1u << i);
    while (uint64_t some = __ballot(passed != 0)) {
      const int slot = held + static_cast<int>(__builtin_amdgcn_mbcnt_hi(
                                  static_cast<uint32_t>(some >> 32),
                                  __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(some), 0)));
      if (passed) {
        const int at = part.index(u0, __builtin_ctz(passed));
        mine[slot] = key_of(value_at<TYPE>(part.row, at), at);
        passed &= passed - 1;
      }
      held += __popcll(some);
      __builtin_amdgcn_wave_barrier();
      if (held >= kWave) merge();
    }
  }
  if (held > 0) merge();
  mine[lane] = list;
  __syncthreads();
  for (int step = 1; step < kWaves; step *= 2) {
    if (wave % (2 * step) == 0) {
      list = merged(list, lists[(wave + step) * 2 * kWave + lane], lane);
      mine[lane] = list;
    }
    __syncthreads();
  }
  return list;
}

constexpr float kNear = 0x1p16f;   // the maxima whose products' rounding, 2^-8 of an exponent at most, is taken out

template <int TYPE, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS, THREADS == 256 ? 8 : 4) void logprobs_kernel(Logprobs p) {
  constexpr int kWaves = THREADS / kWave, kValues = Vec<TYPE>::kValues, kItem = 16 / kValues;
  constexpr int kKeys = kWaves * 2 * kWave, kGroups = 2 * kWave;
  __shared__ Key lists[TOP ? kKeys : 1];
  __shared__ uint32_t group_max[TOP ? kGroups : 1];
  __shared__ int collected;
  __shared__ Sums parts[kWaves];
  const int64_t row = uniform(blockIdx.x / static_cast<uint32_t>(p.splits));
  const int split = uniform(blockIdx.x % static_cast<uint32_t>(p.splits));
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint8_t *x = static_cast<const uint8_t *>(p.logits) + row * p.row_stride * kItem;
  Part<TYPE, THREADS> part;
  part.row = x;
  part.lead = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16) / kItem;
  part.units = reinterpret_cast<const u32x4 *>(x - part.lead * kItem);
  part.vocab = static_cast<int>(p.vocab);
  const int all = (part.lead + part.vocab + kValues - 1) / kValues;
  const int first = split * p.split_units;
  part.end = min(all, first + p.split_units);
  part.plain = min(part.end, (part.lead + part.vocab) / kValues);
  if (TOP && threadIdx.x == 0) collected = 0;

  // A near thread's y is x log2(e) + c, c = -fl(top log2(e)); a far one's, or one's without a value, (x - top) log2(e).
  float top = -INFINITY, c = 0x1p127f, s = 0.f, t = 0.f;  // this c makes the first batch's rescaling a product with 0
  float second = -INFINITY;  // no batch but the one at `where` has a value above it
  int where = first;
  bool care_before = false;  // as the wave's last batch had it
  const auto is_near = [](float m) { return fabsf(m) <= kNear; };
  const auto work = [&](Vec<TYPE> (&v)[kVecs], int u) {
    part.trim(v, u);
    float high = v[0][0], low = v[0][0];
#pragma unroll
    for (int i = 0; i < kVecs * kValues; i += 2) {  // three operands at a time
      const float a = v[i / kValues][i % kValues], b = v[i / kValues][i % kValues + 1];
      high = fmaxf(fmaxf(high, a), b);
      low = fminf(fminf(low, a), b);
    }
    if (TOP) second = fmaxf(second, fminf(high, top));
    // a far thread, or a logit below -2^16, whose product may be -inf (its exponential is 0): -inf in nine places of ten
    // makes 2048 rows of 32000 bf16 31.4 us with the top 20, and 30.2 without
    const bool care = __any(fminf(low, -fmaxf(high, top)) < -kNear);
    if (high > top) {
      where = u;
      float now = -high * kLog2e, y = now - c;
      if (care || care_before) {
        const float held = is_near(top) ? fmaf(top, kLog2e, c) : 0.f, more = is_near(high) ? fmaf(high, kLog2e, now) : 0.f;
        y = (fmaxf(top, -FLT_MAX) - high) * kLog2e - held + more;
        if (!is_near(high)) now = 0.f;
      }
      const float w = __builtin_amdgcn_exp2f(y);
      t = (t + fmaxf(y, -1000.f) * s) * w;
      s *= w;
      top = high;
      c = now;
    }
    care_before = care;
    if (care && __any(!is_near(top))) {
      const float less = is_near(top) ? 0.f : fmaxf(top, -FLT_MAX);
#pragma unroll
      for (int i = 0; i < kVecs * kValues; ++i) {
        const float y = fmaf(v[i / kValues][i % kValues] - less, kLog2e, c), w = __builtin_amdgcn_exp2f(y);
        s += w;
        t = fmaf(fmaxf(y, -1000.f), w, t);
      }
    } else if (care) {
#pragma unroll
      for (int i = 0; i < kVecs * kValues; ++i) {
        const float y = fmaf(v[i / kValues][i % kValues], kLog2e, c), w = __builtin_amdgcn_exp2f(y);
        s += w;
        t = fmaf(fmaxf(y, -1000.f), w, t);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVecs * kValues; ++i) {
        const float y = fmaf(v[i / kValues][i % kValues], kLog2e, c), w = __builtin_amdgcn_exp2f(y);
        s += w;
        t = fmaf(y, w, t);
      }
    }
  };
  const int mine0 = first + static_cast<int>(threadIdx.x);
  if (first < part.end) {
    Vec<TYPE> a[kVecs], b[kVecs];
    part.load(a, first);
    for (int u = first;;) {
      constexpr int kNext = kVecs * THREADS;
      part.load(b, u + kNext);
      work(a, u);
      if ((u += kNext) >= part.end) break;
      part.load(a, u + kNext);
      work(b, u);
      if ((u += kNext) >= part.end) break;
    }
  }
  const auto all_parts = [&]() {  // a wave a lane
    Sums x = parts[lane % kWaves];
    if (lane >= kWaves) x.s = x.t = 0.f;
    return wave_joined(x, lane);
  };
  Sums mine = {fmaxf(top, -FLT_MAX), s, t};
  if (is_near(top)) {  // every y is too large by what fl(m log2(e)) is too small
    const float more = fmaf(top, kLog2e, c), w = __builtin_amdgcn_exp2f(-more);
    mine.s = s * w;
    mine.t = fmaf(-more, s, t) * w;
  }
  mine = wave_joined(mine, lane);
  if (lane == 0) parts[wave] = mine;
  // the groups' maxima: a quad of 256 threads or a sixteen of 1024, or half of these
  const bool fine = p.top > kWave / 2;
  if constexpr (TOP) {
    uint32_t most = mine0 < part.end ? ordered(top) : 0;
    most = max(most, across<1>(most, lane));
    if constexpr (kWaves == 16) {
      most = max(most, across<2>(most, lane));
      most = max(most, across<4>(most, lane));
    }
    if (fine) {
      if (threadIdx.x % (THREADS / 128) == 0) group_max[threadIdx.x / (THREADS / 128)] = most;
    } else {
      most = max(most, kWaves == 16 ? across<8>(most, lane) : across<2>(most, lane));
      if (threadIdx.x % (THREADS / 64) == 0) group_max[threadIdx.x / (THREADS / 64)] = most;
    }
  }
  __syncthreads();
  mine = all_parts();

  // The wave that sorts and writes: with wave 0 in all of them, those of the workgroups that share a CU would be on one SIMD
  // (0.4 us of 2048 rows).
  int writer = static_cast<int>(blockIdx.x / 256 % kWaves);
  Key list = 0;
  if constexpr (TOP) {
    if (wave == writer) {
      uint32_t groups = sorted(group_max[lane], lane);
      if (fine) {
        const uint32_t others = __shfl(sorted(group_max[kWave + lane], lane), kWave - 1 - lane);
        groups = clean(max(groups, others), lane);
      }
      if (lane == p.top - 1) group_max[0] = groups;
    }
    __syncthreads();
    const uint32_t least = uniform(group_max[0]);
    bool exact = mine.s == mine.s;  // else a NaN may be among the values, which no maximum shows
    if (exact) {
      const float bound = least == 0 ? -INFINITY : unordered(least);
      const auto collect = [&](const Vec<TYPE> &v, int u) {
        uint32_t passed = 0;
#pragma unroll
        for (int e = 0; e < kValues; ++e) passed |= v[e] >= bound ? 1u << e : 0;
        while (passed) {
          const int e = __builtin_ctz(passed), at = u * kValues - part.lead + e;
          passed &= passed - 1;
          if (at < 0 || at >= part.vocab) continue;
          const int slot = atomicAdd(&collected, 1);
          if (slot < kKeys) lists[slot] = key_of(v.pick(e), at);
        }
      };
      // A thread looks at the batch of its maximum again, and where another one of its reaches the bound too the wave at
      // all that the thread had, a unit a lane. A unit takes a whole line of the cache with it: all units of the 24
      // threads or so that have the 20 likeliest were most of the row's lines (2048 rows of 32000 bf16 33.0 us, 29.7
      // now; 512 of 128000 fp32 60.8 and 43.9).
      const bool passes = mine0 < part.end && top >= bound;
      if (passes && second < bound) {
        Vec<TYPE> v[kVecs];
        const int u0 = where + static_cast<int>(threadIdx.x);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i].w = part.units[min(u0 + i * THREADS, part.end - 1)];
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
          if (u0 + i * THREADS < part.end) collect(v[i], u0 + i * THREADS);
      }
      uint64_t those = __ballot(passes && !(second < bound));
      while (those) {
        const int thread = __builtin_ctzll(those);
        those &= those - 1;
        for (int u = first + wave * kWave + thread + lane * THREADS; u < part.end; u += kWave * THREADS)
          collect({part.units[u]}, u);
      }
      __syncthreads();
      exact = collected <= kKeys;
    }
    if (exact) {
      if (wave == writer)
        for (int i = 0; i < collected; i += kWave) {
          const Key fresh = sorted(i + lane < collected ? lists[i + lane] : 0, lane, uniform(collected) - i);
          list = i == 0 ? fresh : merged(list, fresh, lane);
        }
    } else {
      __syncthreads();
      list = largest_keys<TYPE, THREADS>(part, first, p.top, lists, wave, lane);
      writer = 0;
    }
  }
  if (wave != writer) return;
  if (p.splits == 1) {
    write_row<TYPE>(p, row, x, mine, list, lane);
    return;
  }
  if (lane == 0) p.part[static_cast<int64_t>(blockIdx.x)] = make_float4(mine.m, mine.s, mine.t, 0.f);
  if constexpr (TOP) p.part_keys[static_cast<int64_t>(blockIdx.x) * kWave + lane] = list;
}

// A wave joins a row's parts.
template <int TYPE>
__global__ __launch_bounds__(kWave) void logprobs_join_kernel(Logprobs p) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  Sums sums = {-FLT_MAX, 0.f, 0.f};
  Key list = 0;
  for (int i0 = 0; i0 < p.splits; i0 += kWave) {
    if (i0 + lane < p.splits) {
      const float4 v = p.part[row * p.splits + i0 + lane];
      sums = joined(sums, {v.x, v.y, v.z});
    }
  }
  sums = wave_joined(sums, lane);
  if (p.top > 0) {
    list = p.part_keys[row * p.splits * kWave + lane];
    for (int i = 1; i < p.splits; ++i) list = merged(list, p.part_keys[(row * p.splits + i) * kWave + lane], lane);
  }
  const uint8_t *x = static_cast<const uint8_t *>(p.logits) + row * p.row_stride * (16 / Vec<TYPE>::kValues);
  write_row<TYPE>(p, row, x, sums, list, lane);
}

template <int TYPE, int THREADS>
hipError_t launch(const Logprobs &p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.rows * p.splits)), block(THREADS);
  if (p.top > 0) hipLaunchKernelGGL((logprobs_kernel<TYPE, THREADS, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((logprobs_kernel<TYPE, THREADS, false>), grid, block, 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.splits == 1) return err;
  hipLaunchKernelGGL((logprobs_join_kernel<TYPE>), dim3(static_cast<unsigned>(p.rows)), dim3(kWave), 0, stream, p);
  return hipGetLastError();
}

template <int TYPE>
hipError_t launch(const Logprobs &p, hipStream_t stream) {
  return p.threads == 256 ? launch<TYPE, 256>(p, stream) : launch<TYPE, 1024>(p, stream);
}

}  // namespace

// A workgroup of 1024 threads for each row while every row has a CU, else one of 256, eight of which share a CU; a few
// long rows are cut, from 128 KB on in one piece each. Measured with the top 5, us: 400 rows of 32000 bf16 14.6 with 1024
// threads and 11.0 with 256, 2048 rows 49.4 and 27.6, 64 rows 8.3 and 9.0; one row of 256000 fp32 13.7 in seven pieces, 21.1
// whole and 16.4 in fifteen, of 128000 bf16 12.8 either way.
void plan_logprobs(Logprobs *p, int cus) {
  const int64_t units = (p->vocab * (p->type == FTX_LOGITS_FP32 ? 4 : 2) + 15) / 16 + 1;  // a row may start inside one
  p->threads = p->rows > cus ? 256 : 1024;
  int64_t splits = 1;
  if (p->threads == 1024) {
    const int64_t batch = 1024 * kVecs;
    splits = std::max<int64_t>(1, std::min<int64_t>({cus / p->rows, units / (4 * batch), 64}));
  }
  p->split_units = static_cast<int>((units + splits - 1) / splits);
  p->splits = static_cast<int>((units + p->split_units - 1) / p->split_units);
  p->part_bytes = p->splits > 1 ? static_cast<size_t>(p->rows) * p->splits * (16 + (p->top > 0 ? 8 * kWave : 0)) : 0;
}

hipError_t launch_logprobs(const Logprobs &p, hipStream_t stream) {
  switch (p.type) {
    case FTX_LOGITS_BF16: return launch<FTX_LOGITS_BF16>(p, stream);
    case FTX_LOGITS_FP16: return launch<FTX_LOGITS_FP16>(p, stream);
    default: return launch<FTX_LOGITS_FP32>(p, stream);
  }
}

}  // namespace ftx
