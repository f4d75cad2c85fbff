// Log probabilities of given tokens, entropy and the likeliest tokens of rows of logits, written for gfx950.
//
//   log p_i = (x_i - max) - log sum_j exp(x_j - max),   H = log sum - sum_j (x_j - max) exp(x_j - max) / sum
//
// over rows of bf16, fp16 or fp32 logits, all statistics in fp32. One pass: a thread keeps a running maximum, the sum of
// the exponentials and the sum of their products with the exponents, in units of log2, and rescales both sums when a
// batch of its values exceeds the maximum. An exponent is clamped before it multiplies an exponential of 0, so logits
// of -inf add nothing; a NaN or +inf makes the row's sums NaN.
//
// The likeliest tokens are keys (the logit's bits in the order of unsigned integers, then the complement of the index):
// the largest keys are the largest logits, the lowest index first among equal ones, a NaN above all. Each wave keeps the
// 64 largest keys it has met sorted over its lanes, and the value of the last one that counts as a threshold: a batch
// whose largest value is not above it (nearly all of them) costs one comparison. The first threshold is the `top`
// largest of the lanes' first maxima, so that only a few values pass it. What passes is read again (it is in the cache),
// collected in LDS and merged 64 at a time.
#include <algorithm>
#include <cfloat>

#include "ftx_internal.h"

namespace ftx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kVecs = 4;  // 16-byte loads of a thread's batch

// A quotient or remainder of a workgroup's number, computed on the vector unit, as the scalar that it is.
__device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(static_cast<int>(v)); }

template <int TYPE>
struct Vec {  // the values of 16 bytes
  static constexpr int kValues = TYPE == FTX_LOGITS_FP32 ? 4 : 8;
  u32x4 w;
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

// Sorts the lanes' keys, the largest first; clean() where they are bitonic.
template <typename K>
__device__ __forceinline__ K exchange(K key, int distance, bool larger) {
  const K other = __shfl_xor(key, distance);
  return (key > other) == larger ? key : other;
}
template <typename K>
__device__ __forceinline__ K clean(K key, int lane) {
#pragma unroll
  for (int j = 32; j > 0; j /= 2) key = exchange(key, j, (lane & j) == 0);
  return key;
}
template <typename K>
__device__ __forceinline__ K sorted(K key, int lane) {
#pragma unroll
  for (int k = 2; k < 64; k *= 2)
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) key = exchange(key, j, ((lane & j) == 0) == ((lane & k) == 0));
  return clean(key, lane);
}
// The 64 largest of two sorted lists.
__device__ __forceinline__ Key merged(Key a, Key b, int lane) {
  const Key other = __shfl(b, 63 - lane);
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
__device__ __forceinline__ Sums wave_joined(Sums x) {
#pragma unroll
  for (int j = 1; j < kWave; j *= 2) x = joined(x, {__shfl_xor(x.m, j), __shfl_xor(x.s, j), __shfl_xor(x.t, j)});
  return x;
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

template <int TYPE, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(Logprobs p) {
  constexpr int kWaves = THREADS / kWave, kValues = Vec<TYPE>::kValues, kItem = 16 / kValues;
  __shared__ Key lists[TOP ? kWaves : 1][TOP ? 2 * kWave : 1];
  __shared__ Sums parts[kWaves];
  const int64_t row = uniform(blockIdx.x / static_cast<uint32_t>(p.splits));
  const int split = uniform(blockIdx.x % static_cast<uint32_t>(p.splits));
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint8_t *x = static_cast<const uint8_t *>(p.logits) + row * p.row_stride * kItem;
  // 16-byte units from the boundary before the row: the values of the first and last one that are not the row's are
  // left out (an aligned unit with a value of the row lies in its memory page)
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16) / kItem;
  const u32x4 *units = reinterpret_cast<const u32x4 *>(x - lead * kItem);
  const int vocab = static_cast<int>(p.vocab);
  const int all = (lead + vocab + kValues - 1) / kValues;
  const int first = split * p.split_units, end = min(all, first + p.split_units);

  Sums mine = {-FLT_MAX, 0.f, 0.f};
  Key list = 0;            // lane i: the wave's ith largest key
  uint32_t threshold = 0;  // values up to this need not be looked at
  int held = 0;            // keys in LDS that have not been merged

  Vec<TYPE> now[kVecs], next[kVecs];
  const auto load = [&](Vec<TYPE> (&v)[kVecs], int u0) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i].w = units[min(u0 + i * THREADS, end - 1)];
  };
  const auto merge = [&]() {
    const Key fresh = lane < held ? lists[wave][lane] : 0;
    list = merged(list, sorted(fresh, lane), lane);
    const Key rest = lists[wave][kWave + lane];
    held = max(held - kWave, 0);
    if (lane < held) lists[wave][lane] = rest;
    threshold = max(threshold, static_cast<uint32_t>(__shfl(list, p.top - 1) >> 32));
  };
  const auto work = [&](Vec<TYPE> (&v)[kVecs], int u0, bool start) {
    // which of the batch's values are the row's: all but at its ends
    const int u1 = u0 + (kVecs - 1) * THREADS;
    uint32_t valid = ~0u;
    if (__any((lead > 0 && u0 == 0) || u1 >= end || (u1 + 1) * kValues - lead > vocab)) {
      valid = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < kValues; ++e) {
          const int u = u0 + i * THREADS, at = u * kValues - lead + e;
          if (u < end && at >= 0 && at < vocab) valid |= 1u << (i * kValues + e);
        }
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < kValues; ++e) {
          if (valid >> (i * kValues + e) & 1) continue;
          if constexpr (TYPE == FTX_LOGITS_FP32) v[i].w[e] = 0xff800000u;
          else v[i].w[e / 2] = (v[i].w[e / 2] & (e % 2 ? 0xffffu : 0xffff0000u)) |
                               (TYPE == FTX_LOGITS_BF16 ? 0xff80u : 0xfc00u) << (16 * (e % 2));
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int e = 0; e < kValues; ++e) top = fmaxf(top, v[i][e]);
    if (top > mine.m) {
      const float y = (mine.m - top) * kLog2e, w = __builtin_amdgcn_exp2f(y);
      mine.t = (mine.t + fmaxf(y, -1000.f) * mine.s) * w;
      mine.s *= w;
      mine.m = top;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int e = 0; e < kValues; ++e) {
        const float y = (v[i][e] - mine.m) * kLog2e, w = __builtin_amdgcn_exp2f(y);
        mine.s += w;
        mine.t = fmaf(fmaxf(y, -1000.f), w, mine.t);
      }
    if constexpr (TOP) {
      uint32_t best = valid ? ordered(top) : 0;
      uint32_t least = threshold;
      if (start) {  // as many lanes as tokens are asked for have a value of at least this
        const uint32_t seed = __shfl(sorted(best, lane), p.top - 1);
        threshold = seed;
        least = seed == 0 ? 0 : seed - 1;  // and in this batch the values equal to it count
      }
      if (mine.s != mine.s) best = valid ? 0xffffffffu : 0;  // a NaN, which the maximum leaves out
      if (__any(best > least)) {
        uint32_t passed = 0;
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
          for (int e = 0; e < kValues; ++e)
            if (ordered(v[i][e]) > least) passed |= 1u << (i * kValues + e);
        passed &= valid;
        while (uint64_t some = __ballot(passed != 0)) {
          const int slot = held + static_cast<int>(__builtin_amdgcn_mbcnt_hi(
                                      static_cast<uint32_t>(some >> 32),
                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(some), 0)));
          if (passed) {
            const int bit = __builtin_ctz(passed);
            const int at = (u0 + bit / kValues * THREADS) * kValues - lead + bit % kValues;
            lists[wave][slot] = key_of(value_at<TYPE>(x, at), at);
            passed &= passed - 1;
          }
          held += __popcll(some);
          __builtin_amdgcn_wave_barrier();
          if (held >= kWave) merge();
        }
      }
    }
  };

  if (first < end) {
    int u0 = first + static_cast<int>(threadIdx.x);
    load(now, u0);
    for (bool start = true;; start = false) {
      const int u1 = u0 + kVecs * THREADS;
      const bool more = u1 - static_cast<int>(threadIdx.x) < end;
      if (more) load(next, u1);
      work(now, u0, start);
      if (!more) break;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) now[i] = next[i];
      u0 = u1;
    }
  }
  if constexpr (TOP) {
    if (held > 0) merge();
  }
  mine = wave_joined(mine);
  if (lane == 0) parts[wave] = mine;
  if constexpr (TOP) lists[wave][lane] = list;
  __syncthreads();
  if constexpr (TOP) {
#pragma unroll
    for (int step = 1; step < kWaves; step *= 2) {
      if (wave % (2 * step) == 0) {
        list = merged(list, lists[wave + step][lane], lane);
        lists[wave][lane] = list;
      }
      __syncthreads();
    }
  }
  if (wave > 0) return;
  mine = parts[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) mine = joined(mine, parts[i]);
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
  sums = wave_joined(sums);
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

void plan_logprobs(Logprobs *p, int cus) {
  const int64_t units = (p->vocab * (p->type == FTX_LOGITS_FP32 ? 4 : 2) + 15) / 16 + 1;  // a row may start inside one
  p->threads = p->rows >= 2 * cus ? 256 : 1024;
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
