// A KV cache in pages of 8-bit codes, written for gfx950: writing positions into it, attention over it, copying
// its pages.
//
// One layer of the cache is codes[page][side][kv head][block of the page][32 d bytes] (side 0: keys, 1: values) and
// scales[page][side][kv head][block]; a block is 32 tokens of one head and a code c stands for c * scale. A
// sequence's tokens lie in the pages that its row of the table names, in order; a page number outside the pool is
// a hole, whose tokens no query sees and no write reaches.
//
// A block's bytes are in the order in which the matrix cores take them: the keys as [d / 16][32 tokens][16], the
// values as [d][32 tokens]. A lane's 16 bytes of keys (one token, 16 of the sum over d) and 8 bytes of values (one
// of d, 8 of the sum over tokens) are then operands as they lie, and a wave's load covers whole lines; values kept
// token by token would have to be transposed through LDS by every reader.
#include <algorithm>
#include <cfloat>

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

constexpr int kWave = 64;
constexpr float kSlack = 8.0f;
constexpr int kTileWaves = 8;  // of an attention workgroup
constexpr float kTiny = 0x1p-100f;  // a block whose scale is below this stands for zeros
constexpr int kRowJoinSplits = 16;  // chunks that a group of lanes joins one after the other

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ __forceinline__ float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }

// What a call adds to a sequence or asks of it: `count` tokens after the `start` cached ones. Tokens past the
// table's last page, and every token of a sequence whose start is negative, take no part.
struct Span {
  int start, count;
};
__device__ __forceinline__ Span span_of(const KvPages &c, int64_t b, int t) {
  const int start = c.starts[b];
  int count = c.news ? min(c.news[b], t) : t;
  const int capacity = c.width * c.page_blocks * kKvBlock;
  if (start < 0 || start >= capacity) return {0, 0};
  return {start, max(0, min(count, capacity - start))};
}

// (min of 64-bit integers would go through doubles)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

// A quotient or remainder of a workgroup's number, computed on the vector unit, as the scalar that it is.
__device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(static_cast<int>(v)); }

// The page that holds a block of sequence b, or -1.
__device__ __forceinline__ int page_of(const KvPages &c, int64_t b, int block) {
  const int page = c.table[b * c.table_stride + (block >> c.page_shift)];
  return static_cast<unsigned>(page) < static_cast<unsigned>(c.pages) ? page : -1;
}

// The number of a block of (page, side, head) in the layer: times 32 d its codes' offset, itself its scale's.
__device__ __forceinline__ int64_t block_index(const KvPages &c, int page, int side, int head, int block) {
  return ((static_cast<int64_t>(page) * 2 + side) * c.kv_heads + head) * c.page_blocks +
         (block & (c.page_blocks - 1));
}

// Pages and scales of 64 blocks, a lane each: a kernel reads them at once, and its loop over the blocks takes them
// from the lanes without waiting for memory. Lane i holds block first + i * step; blocks past `last` are it again.
// The value scale of a block that stands for zeros is 0.
struct BlockList {
  int page;
  float key_scale, value_scale;
};
__device__ __forceinline__ BlockList block_list(const KvPages &c, int64_t b, int head, int first, int step, int last) {
  const int block = min(first + static_cast<int>(threadIdx.x % 64) * step, last);
  BlockList x;
  x.page = page_of(c, b, block);
  x.key_scale = c.scales[block_index(c, max(x.page, 0), 0, head, block)];
  x.value_scale = c.scales[block_index(c, max(x.page, 0), 1, head, block)];
  if (fabsf(x.value_scale) < kTiny) x.value_scale = 0.f;
  return x;
}
__device__ __forceinline__ bool no_scale(float scale) { return __float_as_uint(scale) == 0; }  // a scalar comparison
__device__ __forceinline__ float lane_float(float v, int lane) {
  return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(v)), lane)));
}

// ---- attention -------------------------------------------------------------------------------------------------
//
//   o[b, i, h, :] = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q[b, i, h, :] . k_p - max),  p <= start_b + i
//
// over the cached tokens p of the head that the group of `rep` query heads shares; a row that sees no token is 0.
// Scores, the running maximum and the running sum are fp32. A code is exact in bf16 and enters the products as it
// is: a block's key scale multiplies its scores, its value scale the probabilities. Few rows take a probability into the
// products in two parts of eight bits, as exact as fp32 to the output's rounding. Prompts round it to bf16 (2^-8 of each
// at most, as the attention over a bf16 cache does): the matrix cores are what they wait for, and a second part makes
// 2048 tokens over 8148 (64 / 8 heads) 647 us where one takes 483, for an error of 0.0017 of the result in 64 bits
// (relative norm; the output's own rounding) where one gives 0.0024. A probability may be 2^kSlack and the sums are
// divided at the end: 2^19 keys of values of 2^100 (1e30) stay within fp32.

// Eight codes as bf16.
template <bool FP8>
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
  u32x4 w;
  if constexpr (FP8) {
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = static_cast<int>(i < 2 ? lo : hi);
      w[i] = pack_bf16(static_cast<float>(static_cast<int8_t>(v >> (16 * (i & 1)))),
                       static_cast<float>(static_cast<int8_t>(v >> (16 * (i & 1) + 8))));
    }
  }
  return __builtin_bit_cast(bf16x8, w);
}

// The first n of eight codes, the others 0.
__device__ __forceinline__ u32x2 keep_codes(u32x2 v, int n) {
  const uint64_t mask = n >= 8 ? ~0ull : n <= 0 ? 0ull : (1ull << (8 * n)) - 1;
  return (u32x2){v[0] & static_cast<uint32_t>(mask), v[1] & static_cast<uint32_t>(mask >> 32)};
}

// What is left of eight codes whose scale counts as 0: a NaN, which is one times 0 too.
template <bool FP8>
__device__ __forceinline__ u32x2 without_scale(u32x2 v) {
  if constexpr (!FP8) return (u32x2){0u, 0u};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t nan = ((v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // where all seven bits are set
    v[i] &= (nan >> 7) * 255u;
  }
  return v;
}

// The maximum (or sum) of a value and its partner's in the other half of the wave, and over the four lanes that hold
// one row of 16.
__device__ __forceinline__ float half_max(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float row_max(float v) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}
__device__ __forceinline__ float row_sum(float v) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_sum(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}

// v of lane ^ J in a row of 16 lanes, by moves within the vector registers.
template <int J>
__device__ __forceinline__ int row_xor(int v) {
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xb1, 15, 15, true);  // quad_perm 1 0 3 2
  if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4e, 15, 15, true);  // quad_perm 2 3 0 1
  if constexpr (J == 4)                                                          // eights mirrored, then quads
    return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 15, 15, true), 0x1b, 15, 15, true);
  return __builtin_amdgcn_mov_dpp(v, 0x128, 15, 15, true);  // row_ror 8
}
// All lanes' bits together, as the scalars that they are.
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
  v |= row_xor<1>(v);
  v |= row_xor<2>(v);
  v |= row_xor<4>(v);
  v |= row_xor<8>(v);
  const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = s[0] | s[1];
  const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(t[0] | t[1]);
}
__device__ __forceinline__ uint64_t wave_or(uint64_t v) {
  return static_cast<uint64_t>(wave_or(static_cast<uint32_t>(v >> 32))) << 32 | wave_or(static_cast<uint32_t>(v));
}

// A call over a tree of drafted tokens: `count` rows that see the `start` first tokens and, of the `nodes` after them,
// the ones in their set.
__device__ __forceinline__ Span tree_span(const Kv8Attention &a, int64_t b) {
  const int start = a.kv.starts[b];
  if (start < 0 || start > a.kv.width * a.kv.page_blocks * kKvBlock) return {0, 0};
  return {start, max(0, a.kv.news ? min(a.kv.news[b], a.t) : a.t)};
}
template <bool TREE>
__device__ __forceinline__ Span rows_of(const Kv8Attention &a, int64_t b) {
  if constexpr (TREE) return tree_span(a, b);
  return span_of(a.kv, b, a.t);
}
// The tokens that any row may see.
template <bool TREE>
__device__ __forceinline__ int length_of(const Kv8Attention &a, Span s) {
  if constexpr (TREE) return min(s.start + a.nodes, a.kv.width * a.kv.page_blocks * kKvBlock);
  return s.start + s.count;
}
__device__ __forceinline__ uint64_t held_nodes(uint64_t set, int held) {
  return held >= 64 ? set : set & ((1ull << max(held, 0)) - 1);
}
// The nodes that a row sees.
__device__ __forceinline__ uint64_t node_set(const Kv8Attention &a, int64_t b, int token, int held) {
  return held_nodes(static_cast<uint64_t>(a.tree[b * a.tree_stride + token]), held);
}
// Of the 32 tokens from `at` on (counted from the nodes' first one), the ones that a row with this set sees.
__device__ __forceinline__ uint32_t tokens_seen(uint64_t set, int at) {
  if (at >= 64) return 0;
  if (at >= 0) return static_cast<uint32_t>(set >> at);
  return at <= -32 ? ~0u : static_cast<uint32_t>(set << -at) | ((1u << -at) - 1);
}

// Nodes that no row sees may never have been written: a sequence adds fewer than the tree has, or its rows are some of
// them. Codes there would meet probabilities of 0 in the products, and a NaN among them, or for a scale, every row. So
// the keys and values end behind the last node that a row of the tile sees, and a block before it of which none sees a
// token is a hole: the first one that holds nodes alone (64 nodes reach into one more).
struct Reach {
  int length, blocks, gap;
};
__device__ __forceinline__ Reach reach_of(uint64_t any, int start) {  // any: all that the tile's rows see
  const int length = start + (any ? 64 - __builtin_clzll(any) : 0), first = (start + kKvBlock - 1) / kKvBlock;
  return {length, (length + kKvBlock - 1) / kKvBlock, tokens_seen(any, first * kKvBlock - start) == 0 ? first : -1};
}

// The blocks that the rows of a tile see.
template <bool TREE>
__device__ __forceinline__ int tile_blocks(const Kv8Attention &a, Span s, int tile) {
  const int row0 = tile * a.tile_rows;
  if (row0 / a.rep >= s.count) return 0;
  if (TREE) return (length_of<TREE>(a, s) + kKvBlock - 1) / kKvBlock;
  const int last = min(min(row0 + a.tile_rows, a.rows) - 1, s.count * a.rep - 1) / a.rep;
  return (s.start + last) / kKvBlock + 1;
}

// How a batch's trees are dealt to workgroups, in tiles of 64 keys: sequence by sequence, of each its heads, of a head
// its tiles of rows, of those the keys. `before`: the tiles of the sequences before b; `own`: b's.
struct Share {
  uint32_t at, end, before, own;
  int64_t b;
};
struct Piece {  // the part of a share in one head and tile of rows
  Span span;
  int kvh, tile, blocks, tiles, offset, n;
};
struct Join {  // what a share leaves to be joined: the pieces of the head that it begins and does not end, or 0
  int b, kvh, tile, pieces;
};
__device__ __forceinline__ Join *joins_of(const Kv8Attention &a, int64_t slots, int d) {  // behind the sums
  return reinterpret_cast<Join *>(a.part + slots * (d + 2));
}
constexpr uint32_t kLeastShare = 4;  // tiles that are worth a workgroup's start
__device__ __forceinline__ int live_tiles(const Kv8Attention &a, Span s) {
  return (min(s.count * a.rep, a.rows) + a.tile_rows - 1) / a.tile_rows;
}
__device__ __forceinline__ int key_tiles(int blocks) { return (blocks + 1) / 2; }
__device__ __forceinline__ uint32_t tiles_of(const Kv8Attention &a, int64_t b) {
  if (b >= a.batch) return 0;
  const Span s = tree_span(a, b);
  return a.kv.kv_heads * live_tiles(a, s) * key_tiles(tile_blocks<true>(a, s, 0));
}
__device__ __forceinline__ uint32_t sums_before(uint32_t v) {  // of the lanes up to each
#pragma unroll
  for (int i = 1; i < kWave; i *= 2) {
    const uint32_t lower = __shfl_up(v, i);
    if (static_cast<int>(threadIdx.x & (kWave - 1)) >= i) v += lower;
  }
  return v;
}
__device__ __forceinline__ uint32_t tiles_each(const Kv8Attention &a) {
  uint32_t total = 0;
  for (int base = 0; base < a.batch; base += kWave)
    total += __builtin_amdgcn_readlane(sums_before(tiles_of(a, base + (threadIdx.x & (kWave - 1)))), kWave - 1);
  return max((total + a.items - 1) / a.items, kLeastShare);
}
// `each` tiles from `at` on, as far as there are any.
__device__ __forceinline__ Share share_at(const Kv8Attention &a, uint32_t at, uint32_t each) {
  uint32_t before = 0;
  Share s{at, at, 0, 0, 0};
  for (int base = 0; base < a.batch; base += kWave) {
    const uint32_t own = tiles_of(a, base + (threadIdx.x & (kWave - 1))), upto = sums_before(own) + before;
    const uint32_t total = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (s.end == at && total > at) {
      const int lane = uniform(__popcll(__ballot(upto <= at)));
      s.b = base + lane;
      s.own = __builtin_amdgcn_readlane(own, lane);
      s.before = __builtin_amdgcn_readlane(upto, lane) - s.own;
    }
    if (total > at) s.end = min(total, at + each);
    if (s.end == at + each) break;
    before = total;
  }
  return s;
}
// Or, where they fit, pieces of one head each, so that no workgroup starts twice: a head's keys in as few pieces of up
// to `each` tiles as they take, `each` the least for which there is a workgroup for every piece. A second start takes as
// long as some three tiles (8 ragged sequences of 25 nodes over up to 4096 tokens: 37.7 us with second starts, 31.6
// without). Returns whether it is so, with the workgroup's share and its head's `each`.
constexpr uint32_t kSecondStart = 3;
__device__ __forceinline__ bool whole_pieces(const Kv8Attention &a, uint32_t group, Share &s, uint32_t &each) {
  if (a.batch > kWave) return false;
  const int lane = threadIdx.x & (kWave - 1);
  uint32_t tiles = 0, heads = 0;
  if (lane < a.batch) {
    const Span span = tree_span(a, lane);
    tiles = key_tiles(tile_blocks<true>(a, span, 0));
    heads = tiles > 0 ? a.kv.kv_heads * live_tiles(a, span) : 0;
  }
  const auto sum = [](uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(sums_before(v), kWave - 1));
  };
  const uint32_t even = max((sum(heads * tiles) + a.items - 1) / a.items, kLeastShare);
  uint32_t parts = 0, e = even;
  for (;; ++e) {
    if (e > even + kSecondStart) return false;
    parts = (tiles + e - 1) / e;
    if (sum(heads * parts) <= a.items) break;
  }
  const uint32_t upto = sums_before(heads * parts);
  const int b = uniform(__popcll(__ballot(upto <= group)));
  s = {0, 0, 0, 0, b};
  if (b >= kWave) return true;  // none left
  const uint32_t of = __builtin_amdgcn_readlane(parts, b), held = __builtin_amdgcn_readlane(tiles, b);
  const uint32_t inner = group - (__builtin_amdgcn_readlane(upto, b) - of * __builtin_amdgcn_readlane(heads, b));
  const uint32_t head = uniform(inner / of), part = inner - head * of;
  each = uniform((held + of - 1) / of);
  s.at = head * held + part * each;
  s.end = s.at + min(each, held - part * each);
  return true;
}
__device__ __forceinline__ Piece piece_at(const Kv8Attention &a, const Share &s) {
  Piece p;
  p.span = tree_span(a, s.b);
  p.blocks = tile_blocks<true>(a, p.span, 0);
  p.tiles = key_tiles(p.blocks);
  const uint32_t inner = s.at - s.before;
  const int item = uniform(inner / static_cast<uint32_t>(p.tiles));
  p.offset = inner - item * p.tiles;
  const int live = live_tiles(a, p.span);
  p.kvh = uniform(item / static_cast<uint32_t>(live));
  p.tile = item - p.kvh * live;
  p.n = min(static_cast<uint32_t>(p.tiles - p.offset), s.end - s.at);
  return p;
}
__device__ __forceinline__ void advance(const Kv8Attention &a, Share &s, int n) {
  s.at += n;
  while (s.at < s.end && s.at == s.before + s.own) {
    s.before += s.own;
    s.own = uniform(tiles_of(a, ++s.b));
  }
}

// Few rows: RT tiles of 16 (row = token * rep + head of the group) over one chunk of the keys; the eight waves take its
// blocks in turn and join their sums through LDS. Nothing is staged: each wave loads the next block's codes into
// registers while it works on this one, and widens a code once for all its rows.
template <int D, bool FP8, int RT, bool TREE>
__global__ __launch_bounds__(kTileWaves * kWave, 2) void kv8_rows_kernel(Kv8Attention a) {
  constexpr int kWaves = 8;
  constexpr int kKLoads = D / 64;   // 16 bytes a lane, of each 16 keys of a block
  constexpr int kDTiles = D / 16;
  constexpr int kPitch = D + 4;
  __shared__ __align__(16) float part[kWaves][16][kPitch];
  __shared__ float part_m[kWaves][16], part_l[kWaves][16];

  uint32_t item = blockIdx.x;  // 32-bit divisions: a launch has fewer than 2^24 workgroups
  const int split = uniform(item % static_cast<uint32_t>(a.splits));
  item = uniform(item / static_cast<uint32_t>(a.splits));
  const int64_t tile_item = item;
  const int tile = uniform(item % static_cast<uint32_t>(a.row_tiles));
  item /= static_cast<uint32_t>(a.row_tiles);
  const int kvh = uniform(item % static_cast<uint32_t>(a.kv.kv_heads));
  const int64_t b = uniform(item / static_cast<uint32_t>(a.kv.kv_heads));
  const Span span = rows_of<TREE>(a, b);
  const int blocks = tile_blocks<TREE>(a, span, tile);
  const int first = split * a.chunk;
  if (a.splits > 1 && first >= blocks) return;
  const int end = split == a.splits - 1 ? blocks : min(blocks, first + a.chunk);

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int row0 = tile * (16 * RT);
  int length = length_of<TREE>(a, span);
  const int last_token = (min(row0 + 16 * RT, a.rows) - 1) / a.rep;
  // every row sees keys below this
  const int whole = last_token >= span.count ? 0 : TREE ? span.start : span.start + row0 / a.rep + 1;
  int seen[RT];       // keys this lane's rows see
  uint64_t sets[RT];  // nodes, after them
  bf16x8 qf[RT][D / 32];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = min(row0 + 16 * t + r, a.rows - 1);
    const int token = row / a.rep;
    const int head = kvh * a.rep + (row - token * a.rep);
    seen[t] = token < span.count ? span.start + token + 1 : 0;
    if (TREE) sets[t] = token < span.count ? node_set(a, b, token, length - span.start) : 0;
    const uint16_t *qp = a.q + b * a.q_stride[0] + token * a.q_stride[1] + head * a.q_stride[2] + 16 * g;
#pragma unroll
    for (int i = 0; i < kKLoads; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        qf[t][2 * i + h] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(qp + 64 * i + 8 * h));
  }

  f32x4 o[RT][kDTiles];
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    // The reference maximum, in units of log2, starts at the lowest finite value: while no key of the row counts,
    // -inf less it is -inf, a weight of zero.
    m[t] = -FLT_MAX;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) o[t][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  struct Block {
    u32x4 k[2][kKLoads];
    u32x2 v[kDTiles];
    float k_scale, v_scale;
    bool hole;
  };
  BlockList list;
  [[maybe_unused]] Reach reach{};
  const uint32_t k_lane = g * (16 * kKvBlock) + (8 * (r >> 2) + (r & 3)) * 16, v_lane = r * kKvBlock + 8 * g;
  const auto load = [&](Block &x, int nth) {  // the wave's nth block; past the chunk's end its last one again
    const int at = nth % kWave;
    if (at == 0) list = block_list(a.kv, b, kvh, first + wave + nth * kWaves, kWaves, end - 1);
    const int page = __builtin_amdgcn_readlane(list.page, at);
    const int block = min(first + wave + nth * kWaves, end - 1);
    x.hole = page < 0;
    x.k_scale = lane_float(list.key_scale, at);
    x.v_scale = lane_float(list.value_scale, at);
    const uint8_t *kp = a.kv.codes + block_index(a.kv, max(page, 0), 0, kvh, block) * (kKvBlock * D);
    const uint8_t *vp = a.kv.codes + block_index(a.kv, max(page, 0), 1, kvh, block) * (kKvBlock * D);
#pragma unroll
    for (int i = 0; i < kKLoads; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        x.k[s][i] = *reinterpret_cast<const u32x4 *>(kp + k_lane + (i * (64 * kKvBlock) + 64 * s));
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) x.v[d] = *reinterpret_cast<const u32x2 *>(vp + v_lane + d * (16 * kKvBlock));
  };
  // Key 8 g' + 4 h + c of a block is row 4 g' + c of score tile h, so lane group g holds the scores of keys 8 g ..
  // 8 g + 7, the ones whose values it loads.
  const auto work = [&](Block &x, int block) {  // a hole's loads are used like any others: nothing waits for them
    f32x4 s[RT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        const bf16x8 lo = widen<FP8>(x.k[h][i][0], x.k[h][i][1]), hi = widen<FP8>(x.k[h][i][2], x.k[h][i][3]);
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, qf[t][2 * i], s[t][h], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, qf[t][2 * i + 1], s[t][h], 0, 0, 0);
      }
    }
    const int key0 = block * kKvBlock;
    if (TREE && (block >= reach.blocks || block == reach.gap)) x.hole = true;
    float scale = a.scale_log2 * x.k_scale;
    const bool zeros = no_scale(x.v_scale);
    if (x.hole || zeros || key0 + kKvBlock > whole) {
      const int kept = x.hole ? 0 : length - key0;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int limit = x.hole ? 0 : seen[t] - key0;
        if (TREE) {
          const uint32_t in = x.hole || seen[t] == 0 ? 0 : tokens_seen(sets[t], key0 + 8 * g - span.start);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[t][e / 4][e % 4] = in >> e & 1 ? s[t][e / 4][e % 4] * scale : -INFINITY;
          continue;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[t][h][c] = 8 * g + 4 * h + c < limit ? s[t][h][c] * scale : -INFINITY;
      }
      scale = 1.0f;
      if (kept < kKvBlock) {
#pragma unroll
        for (int d = 0; d < kDTiles; ++d) x.v[d] = keep_codes(x.v[d], kept - 8 * g);
      }
      if (zeros) {
#pragma unroll
        for (int d = 0; d < kDTiles; ++d) x.v[d] = without_scale<FP8>(x.v[d]);
      }
    }
    // p times the value scale in one operation: 2^(s - m + log2(scale)); the sum of the p takes it out again. A block
    // of zeros has been given codes of 0 and takes any. The products take p in two parts of eight bits: these kernels
    // wait for memory, and have the time for a result that is only rounded at its end.
    const float factor = zeros || x.hole ? 1.0f : x.v_scale;
    const float log_factor = __builtin_amdgcn_logf(factor), inverse = __builtin_amdgcn_rcpf(factor);
    u32x4 p[RT], rest[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float mx = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                       fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3])));
      mx = row_max(mx) * scale;
      // The maximum is only raised when a score exceeds it by more than 2^kSlack: the probabilities keep their
      // relative precision, and the accumulators are rescaled a few times per row instead of once per block.
      if (__any(mx > m[t] + kSlack)) {
        const float m_new = fmaxf(m[t], mx);
        const float alpha = __builtin_amdgcn_exp2f(m[t] - m_new);
        m[t] = m_new;
        l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < kDTiles; ++d)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[t][d][c] *= alpha;
      }
      const float offset = log_factor - m[t];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][e >> 1][2 * (e & 1)], scale, offset));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[t][e >> 1][2 * (e & 1) + 1], scale, offset));
        sum += p0 + p1;
        p[t][e] = pack_bf16(p0, p1);
        rest[t][e] = pack_bf16(p0 - bf16_value(p[t][e]), p1 - __uint_as_float(p[t][e] & 0xffff0000u));
      }
      l[t] = fmaf(sum, inverse, l[t]);
    }
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) {
      const bf16x8 v = widen<FP8>(x.v[d][0], x.v[d][1]);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, p[t]), o[t][d], 0, 0, 0);
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, rest[t]), o[t][d], 0, 0, 0);
      }
    }
  };

  const int n = (end - first - wave + kWaves - 1) / kWaves;  // the wave's blocks
  if (n > 0) {
    Block x, y;
    load(x, 0);
    if constexpr (TREE) {  // while the first block is on its way
      reach = reach_of(wave_or(sets[0] | sets[RT - 1]), span.start);
      length = reach.length;
    }
    for (int i = 0;;) {
      load(y, i + 1);
      work(x, first + wave + i * kWaves);
      if (++i >= n) break;
      load(x, i + 1);
      work(y, first + wave + i * kWaves);
      if (++i >= n) break;
    }
  }

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (t > 0) __syncthreads();  // the rows before have been joined
    l[t] = row_sum(l[t]);
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) *reinterpret_cast<f32x4 *>(&part[wave][r][16 * d + 4 * g]) = o[t][d];
    if (g == 0) {
      part_m[wave][r] = m[t];
      part_l[wave][r] = l[t];
    }
    __syncthreads();
    // a thread joins four values of one row
    const int in_tile = threadIdx.x / (D / 4), out_d = threadIdx.x % (D / 4) * 4;
    const int out_row = row0 + 16 * t + in_tile;
    if (in_tile >= 16 || out_row >= a.rows) continue;
    float top = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, part_m[w][in_tile]);
    float sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float weight = __builtin_amdgcn_exp2f(part_m[w][in_tile] - top);
      sum = fmaf(weight, part_l[w][in_tile], sum);
      acc += weight * *reinterpret_cast<const f32x4 *>(&part[w][in_tile][out_d]);
    }
    if (a.splits > 1) {
      const int64_t slots = a.tile_items * a.tile_rows;
      const int64_t slot = split * slots + tile_item * a.tile_rows + 16 * t + in_tile;
      *reinterpret_cast<f32x4 *>(a.part + slot * D + out_d) = acc;
      if (out_d == 0) {
        float *pm = a.part + a.splits * slots * D;
        pm[slot] = top;
        pm[a.splits * slots + slot] = sum;
      }
      continue;
    }
    const int out_token = out_row / a.rep;
    const int out_head = kvh * a.rep + (out_row - out_token * a.rep);
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;  // no key, no weight: the row is 0
    uint16_t *op = a.o + b * a.o_stride[0] + out_token * a.o_stride[1] + out_head * a.o_stride[2] + out_d;
    *reinterpret_cast<u32x2 *>(op) =
        (u32x2){pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
  }
}

// Prompts: eight waves of 32 rows share tiles of 64 keys. The workgroup loads a tile's codes into registers, widens
// each once and writes it to LDS in the order in which a lane reads its operands, 16 bytes at 16 * lane: no bank is
// met twice and the inner loop is that of the attention over a bf16 cache. A tile is written while the one before it
// is in use and the codes of the one after it are on their way, with one barrier a tile.
//
// S^T = K Q^T gives a lane 16 of a block's 32 scores of one row, keys 8 a + 4 g + c (g the half of the wave); V's
// operands are written in that order.
//
// Trees: the sequences' lengths are known on the device alone, so a workgroup a CU reads them all and takes an equal
// share of the batch's tiles (8 ragged sequences of 25 nodes over up to 4096 tokens, 64 / 8 heads, int8: 32.4 us, and 51
// in chunks of the longest one's length). Where a share ends inside a head's tiles, its sums go to `part`, one place for the
// head it begins and one for the head that it goes on with (kv8_join_shares_kernel); SPLIT does not matter.
template <int D, bool FP8, bool SPLIT, bool TREE>
__global__ __launch_bounds__(kTileWaves * kWave, 2) void kv8_tile_kernel(Kv8Attention a) {
  constexpr int kThreads = kTileWaves * kWave;
  constexpr int kKeys = 64, kSub = 2;
  constexpr int kBlockBytes = kKvBlock * D;          // codes of a block's side
  constexpr int kBlockUnits = kBlockBytes / 16;      // 16-byte loads
  constexpr int kSideUnits = kSub * kBlockUnits;
  constexpr int kUnits = 2 * kSideUnits / kThreads;  // of one thread
  constexpr int kSide = kKeys * D * 2;               // LDS bytes of a tile's side
  constexpr int kQSteps = D / 16, kDTiles = D / 32;
  static_assert(2 * kSideUnits % kThreads == 0 && kBlockUnits % kWave == 0, "a wave's units are of one block and side");
  __shared__ __align__(1024) uint8_t lds[4 * kSide];  // two tiles of keys, two of values

  const uint32_t per_xcd = (a.items + a.xcds - 1) / a.xcds;
  uint32_t item = (blockIdx.x % a.xcds) * per_xcd + blockIdx.x / a.xcds;
  if (item >= a.items) return;
  [[maybe_unused]] const uint32_t group = item;
  [[maybe_unused]] Share share{};
  [[maybe_unused]] uint32_t each = 0;
  [[maybe_unused]] Join join{};
  if constexpr (TREE) {
    if (!whole_pieces(a, group, share, each)) {
      each = tiles_each(a);
      share = share_at(a, group * each, each);
    }
  }
  while (!TREE || share.at < share.end) {  // of a tree's pieces; the others end in the first round
  int split = 0, tile, kvh, blocks, first = 0, end;
  [[maybe_unused]] bool alone = true;  // the share holds all of the head's tiles
  int64_t b, tile_item;
  Span span;
  if constexpr (TREE) {
    const Piece piece = piece_at(a, share);
    b = share.b, kvh = piece.kvh, tile = piece.tile, span = piece.span, blocks = piece.blocks;
    first = piece.offset * kSub, end = min(blocks, (piece.offset + piece.n) * kSub);
    alone = piece.n == piece.tiles;
    tile_item = piece.offset == 0 ? a.items + group : group;  // the place of its sums
    if (piece.offset == 0 && !alone)
      join = {static_cast<int>(b), kvh, tile, 1 + static_cast<int>((piece.tiles - piece.n + each - 1) / each)};
    advance(a, share, piece.n);
  } else {
    split = SPLIT ? uniform(item % static_cast<uint32_t>(a.splits)) : 0;
    if (SPLIT) item /= static_cast<uint32_t>(a.splits);
    const uint32_t bkv = uniform(item / static_cast<uint32_t>(a.row_tiles));
    tile = uniform(a.row_tiles - 1 - (item - bkv * a.row_tiles));  // the longest first
    tile_item = static_cast<int64_t>(bkv) * a.row_tiles + tile;
    b = uniform(bkv / static_cast<uint32_t>(a.kv.kv_heads));
    kvh = uniform(bkv % static_cast<uint32_t>(a.kv.kv_heads));
    span = rows_of<TREE>(a, b);
    blocks = tile_blocks<TREE>(a, span, tile);
    first = SPLIT ? split * a.chunk : 0;
    if (SPLIT && first >= blocks) return;
    end = !SPLIT || split == a.splits - 1 ? blocks : min(blocks, first + a.chunk);
  }
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 31, g = lane >> 5;
  const int row0 = tile * (32 * kTileWaves) + wave * 32;
  const int row = min(row0 + r, a.rows - 1);
  const int token = row / a.rep;
  const int head = kvh * a.rep + (row - token * a.rep);
  int length = length_of<TREE>(a, span);
  const bool live = row0 + r < a.rows && token < span.count;
  const int seen = live ? span.start + token + 1 : 0;  // keys this lane's row sees
  const uint64_t set = TREE && live ? node_set(a, b, token, length - span.start) : 0;  // of a tree: the nodes
  int64_t any[kTileWaves / 2] = {};  // of a tree: what the workgroup's rows see
  if constexpr (TREE) {
    const int token0 = tile * (32 * kTileWaves) / a.rep;
    const int last_token = min((min((tile + 1) * (32 * kTileWaves), a.rows) - 1) / a.rep, span.count - 1);
#pragma unroll
    for (int i = 0; i < kTileWaves / 2; ++i)
      if (token0 + i * kWave <= last_token)
        any[i] = a.tree[b * a.tree_stride + min(token0 + i * kWave + lane, last_token)];
  }
  const int last_row = min(row0 + 32, a.rows) - 1;
  // Every row of the wave sees keys below this. A tree's rows that are left out see them too, and are cleared at the end:
  // masks for their sake took 0.4 us a tile.
  const bool all_live = row0 + 32 <= a.rows && last_row / a.rep < span.count;
  const int whole = TREE ? span.start : !all_live ? 0 : span.start + row0 / a.rep + 1;

  // Queries: lane (r, g) holds elements 16 ks + 8 g .. + 7 of its row for every step ks.
  bf16x8 qf[kQSteps];
  {
    const uint16_t *qp = a.q + b * a.q_stride[0] + token * a.q_stride[1] + head * a.q_stride[2] + 8 * g;
#pragma unroll
    for (int ks = 0; ks < kQSteps; ++ks)
      qf[ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(qp + 16 * ks));
  }
  // The queries are in registers before the loop: where they may still be on their way as it is entered, every
  // round waits for the codes that it has just asked for (2.0 us a tile).
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  asm volatile("" ::: "memory");
  [[maybe_unused]] Reach reach{};
  if constexpr (TREE) {
    reach = reach_of(held_nodes(wave_or(static_cast<uint64_t>(any[0] | any[1] | any[2] | any[3])), length - span.start),
                     span.start);
    length = reach.length;
  }
  const int n_tiles = (end - first + kSub - 1) / kSub;
  const int wave_end = row0 >= a.rows || row0 / a.rep >= span.count ? 0
                       : TREE                                       ? length
                                                                    : min(span.start + last_row / a.rep + 1, length);

  const auto side_of = [&](int i) {  // known when compiled where a unit of all waves is of one side
    return kSideUnits >= kThreads ? i * kThreads / kSideUnits : (i * kThreads + wave * kWave) / kSideUnits;
  };
  struct Unit {  // 16 bytes of codes on their way to LDS
    u32x4 w;
    int keep;    // values: the tokens of them that the sequence has; less 64 where they have no scale
  };
  Unit units[kUnits];
  struct Scales {
    float key[kSub], value[kSub];
    bool hole[kSub];  // or past the chunk's end
  };
  BlockList list;
  const auto load = [&](int t) {  // past the chunk's last block it again, masked
    const int at = t * kSub % kWave;
    if (at == 0) {
      list = block_list(a.kv, b, kvh, first + t * kSub, 1, end - 1);
      if constexpr (TREE) {
        const int block = first + t * kSub + lane;
        if (block >= reach.blocks || block == reach.gap) list.page = -1;
      }
    }
    Scales x;
    int page[kSub];
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      page[j] = __builtin_amdgcn_readlane(list.page, at + j);
      x.key[j] = lane_float(list.key_scale, at + j);
      x.value[j] = lane_float(list.value_scale, at + j);
      x.hole[j] = page[j] < 0 || first + t * kSub + j >= end;
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u0 = i * kThreads + wave * kWave;  // the wave's first unit
      const int side = side_of(i), sub = u0 % kSideUnits / kBlockUnits;
      const int block = first + t * kSub + sub;
      const int own = sub == 0 ? page[0] : page[1];
      const uint8_t *from =
          a.kv.codes + block_index(a.kv, max(own, 0), side, kvh, min(block, end - 1)) * kBlockBytes;
      units[i].w = *reinterpret_cast<const u32x4 *>(from + (u0 % kBlockUnits + lane) * 16);
      units[i].keep = own < 0 || block >= end ? 0 : min(length - block * kKvBlock, kKvBlock);
      if (side != 0 && no_scale(sub == 0 ? x.value[0] : x.value[1])) units[i].keep -= 64;
    }
    return x;
  };
  // Where the 16 bytes go: keys are units of [d / 16][token], one step of the sum over d for both halves of the wave;
  // values of [d][half of the tokens], one step of the sum over tokens, whose words the halves take in turn.
  uint32_t store_at[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u0 = i * kThreads + wave * kWave, unit = u0 % kBlockUnits + lane, d = unit / 2;
    store_at[i] = u0 % kSideUnits / kBlockUnits * (kSide / kSub) +
                  (side_of(i) == 0 ? unit / 32 * 1024 + unit % 32 * 16 : (d / 32 * 2 + unit % 2) * 1024 + d % 32 * 16);
  }
  const auto store = [&](int t) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int side = side_of(i);
      u32x4 w = units[i].w;
      if (side != 0 && units[i].keep < kKvBlock) {
        const int n = (units[i].keep < 0 ? units[i].keep + 64 : units[i].keep) - lane % 2 * 16;
        u32x2 lo = keep_codes((u32x2){w[0], w[1]}, n), hi = keep_codes((u32x2){w[2], w[3]}, n - 8);
        if (units[i].keep < 0) lo = without_scale<FP8>(lo), hi = without_scale<FP8>(hi);
        w = (u32x4){lo[0], lo[1], hi[0], hi[1]};
      }
      uint8_t *to = lds + (side == 0 ? t & 1 : 2 + (t & 1)) * kSide + store_at[i];
      *reinterpret_cast<bf16x8 *>(to) = widen<FP8>(w[0], side == 0 ? w[1] : w[2]);
      *reinterpret_cast<bf16x8 *>(to + 512) = widen<FP8>(side == 0 ? w[2] : w[1], w[3]);
    }
  };

  f32x16 o[kDTiles];
#pragma unroll
  for (int d = 0; d < kDTiles; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -FLT_MAX, l = 0.f;

  // Operands are read a few products ahead of their use, the first ones before other work: LDS answers after some
  // 130 cycles, four products of a wave.
  constexpr int kAhead = 3;
  bf16x8 kf[kAhead + 1][kSub], vf[2][kDTiles];
  const auto read_keys = [&](int t, int ks) {
    const uint8_t *from = lds + (t & 1) * kSide + lane * 16 + ks * 1024;
#pragma unroll
    for (int j = 0; j < kSub; ++j)
      kf[ks % (kAhead + 1)][j] = *reinterpret_cast<const bf16x8 *>(from + j * (kSide / kSub));
  };
  const auto read_values = [&](int t, int f) {
    const uint8_t *from = lds + (2 + (t & 1)) * kSide + lane * 16 + (f / 2) * (kSide / kSub) + f % 2 * 1024;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) vf[f & 1][d] = *reinterpret_cast<const bf16x8 *>(from + d * 2048);
  };
  f32x16 s[kSub];  // scores of the tile in hand
  const auto scores = [&](int t) {
#pragma unroll
    for (int j = 0; j < kSub; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[j][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < kQSteps; ++ks) {
      if (ks + kAhead < kQSteps) read_keys(t, ks + kAhead);
#pragma unroll
      for (int j = 0; j < kSub; ++j)
        s[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks % (kAhead + 1)][j], qf[ks], s[j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto weigh = [&](int t, const Scales &x) {  // softmax, then the values
    float scale[kSub];
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      scale[j] = a.scale_log2 * x.key[j];
      const int block = first + t * kSub + j;
      if (x.hole[j] || (block + 1) * kKvBlock > whole) {
        if (TREE) {
          const uint32_t in = x.hole[j] || !live ? 0 : tokens_seen(set, block * kKvBlock - span.start) >> (4 * g);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[j][e] = in >> (8 * (e >> 2) + (e & 3)) & 1 ? s[j][e] * scale[j] : -INFINITY;
          scale[j] = 1.0f;
          continue;
        }
        const int limit = x.hole[j] ? 0 : seen - block * kKvBlock;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[j][e] = 8 * (e >> 2) + 4 * g + (e & 3) < limit ? s[j][e] * scale[j] : -INFINITY;
        scale[j] = 1.0f;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      float part = s[j][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) part = fmaxf(part, s[j][e]);
      mx = fmaxf(mx, part * scale[j]);
    }
    mx = half_max(mx);
    if (__any(mx > m + kSlack)) {
      const float m_new = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kDTiles; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
    }
    bf16x8 p[2 * kSub];  // times the value scale, as above
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      const float factor = no_scale(x.value[j]) || x.hole[j] ? 1.0f : x.value[j];
      const float offset = __builtin_amdgcn_logf(factor) - m;
      float sum = 0.f;
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[j][e], scale[j], offset));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[j][e + 1], scale[j], offset));
        sum += p0 + p1;
        w[e / 2] = pack_bf16(p0, p1);
      }
      l = fmaf(sum, __builtin_amdgcn_rcpf(factor), l);
      p[2 * j] = __builtin_bit_cast(bf16x8, (u32x4){w[0], w[1], w[2], w[3]});
      p[2 * j + 1] = __builtin_bit_cast(bf16x8, (u32x4){w[4], w[5], w[6], w[7]});
    }
#pragma unroll
    for (int f = 0; f < 2 * kSub; ++f) {
      if (f + 1 < 2 * kSub) read_values(t, f + 1);
#pragma unroll
      for (int d = 0; d < kDTiles; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[f & 1][d], p[f], o[d], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto sees = [&](int t) { return (first + t * kSub) * kKvBlock < wave_end; };  // any key of the tile

  Scales x = {}, next = {}, later = {};
  if (n_tiles > 0) {
    next = load(0);
    store(0);
    if (n_tiles > 1) later = load(1);
  }
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();
    x = next;
    next = later;
    if (sees(t)) {
#pragma unroll
      for (int ks = 0; ks < kAhead; ++ks) read_keys(t, ks);
    }
    if (t + 1 < n_tiles) {
      store(t + 1);
      if (t + 2 < n_tiles) later = load(t + 2);
    }
    if (sees(t)) {
      scores(t);
      read_values(t, 0);
      __builtin_amdgcn_sched_barrier(0);
      weigh(t, x);
    }
  }

  if (!TREE && row0 + r >= a.rows) return;
  l = half_sum(l);
  if (TREE && !live) {
    m = -FLT_MAX, l = 0.f;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  }
  if (row0 + r >= a.rows) {
  } else if (TREE ? !alone : SPLIT) {
    const int64_t slots = TREE ? 2 * static_cast<int64_t>(a.items) * a.part_rows : a.tile_items * a.tile_rows;
    const int64_t slot = (TREE ? tile_item * a.part_rows : split * slots + tile_item * a.tile_rows) + wave * 32 + r;
    float *po = a.part + slot * D;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4 *>(po + d * 32 + q * 8 + 4 * g) =
            (f32x4){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
    if (g == 0) {
      const int64_t all = TREE ? slots : a.splits * slots;
      float *pm = a.part + all * D;
      pm[slot] = m;
      pm[all + slot] = l;
    }
  } else {
    const float inv = l != 0.f ? 1.0f / l : 0.f;  // no key, no weight: the row is 0
    uint16_t *op = a.o + b * a.o_stride[0] + token * a.o_stride[1] + head * a.o_stride[2] + 4 * g;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<u32x2 *>(op + d * 32 + q * 8) =
            (u32x2){pack_bf16(o[d][4 * q] * inv, o[d][4 * q + 1] * inv),
                    pack_bf16(o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv)};
  }
  if (!TREE) return;
  __syncthreads();  // the next piece's first tiles go where waves may still read the last ones
  }
  if constexpr (TREE) {
    if (threadIdx.x == 0) joins_of(a, 2 * static_cast<int64_t>(a.items) * a.part_rows, D)[group] = join;
    // Rows that see nothing, and have no tiles.
    for (uint32_t i = group; i < a.tile_items; i += a.items) {
      const uint32_t bkv = i / static_cast<uint32_t>(a.row_tiles);
      const int tile = uniform(i - bkv * a.row_tiles);
      const int64_t b = uniform(bkv / static_cast<uint32_t>(a.kv.kv_heads));
      if (tile_blocks<TREE>(a, rows_of<TREE>(a, b), tile) > 0) continue;
      const int kvh = uniform(bkv % static_cast<uint32_t>(a.kv.kv_heads));
      const int rows = min(a.rows - tile * a.tile_rows, a.tile_rows);
      for (int j = threadIdx.x; j < rows * (D / 8); j += kThreads) {
        const int row = tile * a.tile_rows + j / (D / 8), token = row / a.rep;
        const int head = kvh * a.rep + (row - token * a.rep);
        uint16_t *op = a.o + b * a.o_stride[0] + token * a.o_stride[1] + head * a.o_stride[2] + j % (D / 8) * 8;
        *reinterpret_cast<u32x2 *>(op) = (u32x2){0, 0};
        *reinterpret_cast<u32x2 *>(op + 4) = (u32x2){0, 0};
      }
    }
  }
}

// The join of the shares: the head's tiles that a share begins and does not end are joined by the workgroups of that
// share, 256 / (D / 4) rows each.
template <int D>
__global__ __launch_bounds__(256) void kv8_join_shares_kernel(Kv8Attention a) {
  constexpr int kLanes = D / 4, kBatch = 4;
  const uint32_t parts = (a.part_rows + 256 / kLanes - 1) / (256 / kLanes);
  const uint32_t left = uniform(blockIdx.x / parts);
  const int64_t slots = 2 * static_cast<int64_t>(a.items) * a.part_rows;
  const Join join = joins_of(a, slots, D)[left];
  const int used = uniform(join.pieces);
  if (used == 0) return;
  const int in_tile = (blockIdx.x - left * parts) * (256 / kLanes) + threadIdx.x / kLanes;
  const int row = join.tile * a.tile_rows + in_tile;
  if (in_tile >= a.part_rows || row >= a.rows) return;
  const float *pm = a.part + slots * D, *pl = pm + slots;
  const int c = threadIdx.x % kLanes;
  float mx = -FLT_MAX, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < used; i0 += kBatch) {
    float m[kBatch], part[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {  // past the last piece it again, with a weight of zero below
      const int64_t n = min(i0 + i, used - 1);
      const int64_t s = (n == 0 ? a.items + left : left + n) * a.part_rows + in_tile;
      m[i] = pm[s];
      part[i] = pl[s];
      o[i] = *reinterpret_cast<const f32x4 *>(a.part + s * D + 4 * c);
    }
    float m_new = mx;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) m_new = fmaxf(m_new, m[i]);
    const float alpha = __builtin_amdgcn_exp2f(mx - m_new);
    l *= alpha;
    acc *= alpha;
    mx = m_new;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i >= used) break;
      const float w = __builtin_amdgcn_exp2f(m[i] - m_new);
      l += w * part[i];
      acc += w * o[i];
    }
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  const int token = row / a.rep;
  const int head = join.kvh * a.rep + (row - token * a.rep);
  uint16_t *op = a.o + join.b * a.o_stride[0] + token * a.o_stride[1] + head * a.o_stride[2] + 4 * c;
  *reinterpret_cast<u32x2 *>(op) =
      (u32x2){pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
}

// o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the chunks that hold keys the tile sees, M the largest
// m_i. A workgroup a row: groups of D / 4 lanes take the chunks in turn, so that few rows over many chunks wait for
// a few loads and not for one after the other, and meet in LDS.
template <int D, bool TREE>
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8Attention a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes, kBatch = 4;
  __shared__ f32x4 part_o[kGroups][kLanes];
  __shared__ float part_m[kGroups], part_l[kGroups];
  const int64_t slots = a.tile_items * a.tile_rows, at = blockIdx.x;
  const uint32_t tile_item = uniform(blockIdx.x / static_cast<uint32_t>(a.tile_rows));
  const int tile = uniform(tile_item % static_cast<uint32_t>(a.row_tiles));
  const int row = tile * a.tile_rows + uniform(blockIdx.x % static_cast<uint32_t>(a.tile_rows));
  if (row >= a.rows) return;
  const uint32_t bkv = uniform(tile_item / static_cast<uint32_t>(a.row_tiles));
  const int64_t b = uniform(bkv / static_cast<uint32_t>(a.kv.kv_heads));
  const int used = min(a.splits, (tile_blocks<TREE>(a, rows_of<TREE>(a, b), tile) + a.chunk - 1) / a.chunk);
  const float *pm = a.part + a.splits * slots * D;
  const float *pl = pm + a.splits * slots;
  const int c = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  float mx = -FLT_MAX, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = group; i0 < used; i0 += kGroups * kBatch) {
    float m[kBatch], part[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {  // past the last chunk it again, with a weight of zero below
      const int64_t s = min(i0 + i * kGroups, used - 1) * slots + at;
      m[i] = pm[s];
      part[i] = pl[s];
      o[i] = *reinterpret_cast<const f32x4 *>(a.part + s * D + 4 * c);
    }
    float m_new = mx;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) m_new = fmaxf(m_new, m[i]);
    const float alpha = __builtin_amdgcn_exp2f(mx - m_new);
    l *= alpha;
    acc *= alpha;
    mx = m_new;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i * kGroups >= used) break;
      const float w = __builtin_amdgcn_exp2f(m[i] - m_new);
      l += w * part[i];
      acc += w * o[i];
    }
  }
  part_o[group][c] = acc;
  if (c == 0) {
    part_m[group] = mx;
    part_l[group] = l;
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) mx = fmaxf(mx, part_m[i]);
  l = 0.f;
  acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float w = __builtin_amdgcn_exp2f(part_m[i] - mx);
    l += w * part_l[i];
    acc += w * part_o[i][c];
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  const int token = row / a.rep;
  const int head = uniform(bkv % static_cast<uint32_t>(a.kv.kv_heads)) * a.rep + (row - token * a.rep);
  uint16_t *op = a.o + b * a.o_stride[0] + token * a.o_stride[1] + head * a.o_stride[2] + 4 * c;
  *reinterpret_cast<u32x2 *>(op) =
      (u32x2){pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
}

// The same for few chunks of many rows, as trees have them: a group of D / 4 lanes a row, which takes its chunks one after
// the other, four loads at a time (12800 rows in four chunks: 6.4 us, a workgroup a row 20.8).
template <int D>
__global__ __launch_bounds__(256) void kv8_join_rows_kernel(Kv8Attention a) {
  constexpr int kLanes = D / 4, kBatch = 4;
  const int64_t slots = a.tile_items * a.tile_rows;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (at >= slots) return;
  const uint32_t tile_item = static_cast<uint32_t>(at) / static_cast<uint32_t>(a.tile_rows);
  const int tile = static_cast<int>(tile_item % static_cast<uint32_t>(a.row_tiles));
  const int row = tile * a.tile_rows + static_cast<int>(static_cast<uint32_t>(at) % static_cast<uint32_t>(a.tile_rows));
  if (row >= a.rows) return;
  const uint32_t bkv = tile_item / static_cast<uint32_t>(a.row_tiles);
  const int64_t b = bkv / static_cast<uint32_t>(a.kv.kv_heads);
  const int used = min(a.splits, (tile_blocks<true>(a, rows_of<true>(a, b), tile) + a.chunk - 1) / a.chunk);
  const float *pm = a.part + a.splits * slots * D;
  const float *pl = pm + a.splits * slots;
  const int c = threadIdx.x % kLanes;
  float mx = -FLT_MAX, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < used; i0 += kBatch) {
    float m[kBatch], part[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {  // past the last chunk it again, with a weight of zero below
      const int64_t s = min(i0 + i, used - 1) * slots + at;
      m[i] = pm[s];
      part[i] = pl[s];
      o[i] = *reinterpret_cast<const f32x4 *>(a.part + s * D + 4 * c);
    }
    float m_new = mx;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) m_new = fmaxf(m_new, m[i]);
    const float alpha = __builtin_amdgcn_exp2f(mx - m_new);
    l *= alpha;
    acc *= alpha;
    mx = m_new;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i >= used) break;
      const float w = __builtin_amdgcn_exp2f(m[i] - m_new);
      l += w * part[i];
      acc += w * o[i];
    }
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  const int token = row / a.rep;
  const int head = static_cast<int>(bkv % static_cast<uint32_t>(a.kv.kv_heads)) * a.rep + (row - token * a.rep);
  uint16_t *op = a.o + b * a.o_stride[0] + token * a.o_stride[1] + head * a.o_stride[2] + 4 * c;
  *reinterpret_cast<u32x2 *>(op) =
      (u32x2){pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
}

template <int D, bool FP8, bool TREE>
hipError_t launch_attend(const Kv8Attention &p, hipStream_t stream) {
  const dim3 block(kTileWaves * kWave), grid(p.items), xcd_grid((p.items + p.xcds - 1) / p.xcds * p.xcds);
  if (p.tile_rows <= 16) hipLaunchKernelGGL((kv8_rows_kernel<D, FP8, 1, TREE>), grid, block, 0, stream, p);
  else if (p.tile_rows == 32) hipLaunchKernelGGL((kv8_rows_kernel<D, FP8, 2, TREE>), grid, block, 0, stream, p);
  else if (TREE || p.splits == 1)
    hipLaunchKernelGGL((kv8_tile_kernel<D, FP8, false, TREE>), xcd_grid, block, 0, stream, p);
  else hipLaunchKernelGGL((kv8_tile_kernel<D, FP8, !TREE, TREE>), xcd_grid, block, 0, stream, p);
  if (TREE && p.tile_rows > 32) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || p.items == 1) return err;
    const unsigned parts = (p.part_rows * (D / 4) + 255) / 256;
    hipLaunchKernelGGL((kv8_join_shares_kernel<D>), dim3((p.items - 1) * parts), dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.splits == 1) return err;
  if (TREE && p.splits <= kRowJoinSplits) {
    const int64_t groups = (p.tile_items * p.tile_rows * (D / 4) + 255) / 256;
    hipLaunchKernelGGL((kv8_join_rows_kernel<D>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((kv8_join_kernel<D, TREE>), dim3(static_cast<unsigned>(p.tile_items * p.tile_rows)), dim3(256), 0,
                     stream, p);
  return hipGetLastError();
}

// ---- writing new positions ---------------------------------------------------------------------------------------
//
// The new tokens' y (keys rotated by the tables, halves against each other, values as they are) go into their
// blocks under s = max(the block's scale if it holds older tokens, max |y| / top), top = 448 or 127, as the nearest
// codes to y / s; where s grew, the older codes are rounded again to the nearest of c * (old s / s). Tokens of the
// block past the new ones become 0. The maximum is over finite values (an infinity becomes the largest code, a NaN
// the e4m3 NaN or the integer 0), and a scale below 2^-100 counts as 0, with codes of 0 for all but a NaN.
//
// The sums are the ones elementary operations make, each product and sum rounded to fp32 on its own (no fused
// multiply-add), so the codes do not depend on how a compiler contracts them.
template <bool FP8>
__device__ __forceinline__ uint32_t code4(const float *y) {
  if constexpr (FP8) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = y[i] > 448.f ? 448.f : y[i] < -448.f ? -448.f : y[i];  // a NaN stays
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true));
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = y[i] == y[i] ? fminf(fmaxf(rintf(y[i]), -127.f), 127.f) : 0.f;
      w |= (static_cast<uint32_t>(static_cast<int>(v)) & 255u) << (8 * i);
    }
    return w;
  }
}

template <bool FP8>
__device__ __forceinline__ float code_value(uint32_t byte) {
  if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(byte), 0);
  return static_cast<float>(static_cast<int8_t>(byte));
}

// What rotates a thread's N values from d0 on: a row of the tables. x cos + rot(x) sin, rot(x) = (-upper half, lower
// half).
//
// NORM: the values are x * f * w first, f = 1 / sqrt(mean x^2 + eps) of their head's row and w the weights.
template <int D, int N>
struct Row {  // a thread's values, and the ones that they turn against
  u32x4 own[N / 8], other[N / 8];
  __device__ __forceinline__ void load(const uint16_t *x, int d0) {
    const int from = d0 < D / 2 ? d0 + D / 2 : d0 - D / 2;
#pragma unroll
    for (int v = 0; v < N; v += 8) {
      own[v / 8] = *reinterpret_cast<const u32x4 *>(x + d0 + v);
      other[v / 8] = *reinterpret_cast<const u32x4 *>(x + from + v);
    }
  }
};
template <int J>
__device__ __forceinline__ double row_xor(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = row_xor<J>(static_cast<int>(b)), hi = row_xor<J>(static_cast<int>(b >> 32));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

template <int D, int N, bool NORM>
struct Rotation {
  float cos[N], sin[N];
  Row<D, NORM ? N : 8> w;  // the weights
  __device__ __forceinline__ void load(const float *c, const float *s, int d0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      *reinterpret_cast<f32x4 *>(cos + i) = *reinterpret_cast<const f32x4 *>(c + d0 + i);
      *reinterpret_cast<f32x4 *>(sin + i) = *reinterpret_cast<const f32x4 *>(s + d0 + i);
    }
  }
  // The D / N lanes of a row: its f. The sum is one of 64 bits, in which the squares are exact, and f the nearest fp32
  // number: the codes made from it depend on no order of the sum.
  __device__ __forceinline__ float factor(const Row<D, N> &x, float eps) const {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double value = bf16_value(x.own[i / 8][i % 8 / 2] >> (16 * (i & 1)));
      sum = fma(value, value, sum);
    }
    static_assert(D / N == 4 || D / N == 8 || D / N == 16, "the lanes of a row are within 16");
    sum += row_xor<1>(sum);
    sum += row_xor<2>(sum);
    if constexpr (D / N >= 8) sum += row_xor<4>(sum);
    if constexpr (D / N >= 16) sum += row_xor<8>(sum);
    const double mean = sum * (1.0 / D) + static_cast<double>(eps);
    const double rough = __builtin_amdgcn_rsq(mean);  // 2^-23 off or less; a step of Newton's: 2^-45
    const double better = fma(0.5 * rough, fma(-mean * rough, rough, 1.0), rough);
    return static_cast<float>(mean > 0.0 && mean < INFINITY ? better : rough);
  }
  __device__ __forceinline__ void apply(const Row<D, N> &x, int d0, float *y, float f) const {
#pragma clang fp contract(off)
#pragma unroll
    for (int v = 0; v < N; v += 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float va = bf16_value(x.own[v / 8][i / 2] >> (16 * (i & 1)));
        float vb = bf16_value(x.other[v / 8][i / 2] >> (16 * (i & 1)));
        if (NORM) {
          va = va * f * bf16_value(w.own[v / 8][i / 2] >> (16 * (i & 1)));
          vb = vb * f * bf16_value(w.other[v / 8][i / 2] >> (16 * (i & 1)));
        }
        const float turned = d0 < D / 2 ? -vb : vb;
        const float p = va * cos[v + i], q = turned * sin[v + i];
        y[v + i] = p + q;
      }
    }
  }
};

// Workgroups below `a.block_items` write one block of `a.heads_each` heads of one side; the others rotate the queries,
// the same number of heads each. The heads share their tokens' rows of the tables, 4 d bytes each of cos and sin where
// a head's own values are 2 d; with that, and a token's values side by side in a wave, a prompt of 2048 tokens (32 heads
// of 128, int8) takes 20.7 us, 4.1 TB/s, and took 31 before. A decode step needs the workgroups and has one head each.
//
// AT: a token's row of the tables may be another than its place's, `a.at`; one outside the tables makes the token 0, in
// the cache too. NORM: queries and keys are normalised head by head first, by the lanes that share the row; the prompt
// above takes 27.8 us then.
template <int D, bool FP8, bool AT, bool NORM>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8Append a) {
#pragma clang fp contract(off)
  constexpr int kChunks = D / 16;
  constexpr float kTop = FP8 ? 448.f : 127.f;
  if (blockIdx.x >= a.block_items) {  // the queries: eight values a thread
    const uint32_t item = blockIdx.x - static_cast<uint32_t>(a.block_items);
    const uint32_t groups = (a.heads + a.heads_each - 1) / a.heads_each;
    const int h0 = uniform(item % groups) * a.heads_each;
    const int64_t at = static_cast<int64_t>(uniform(item / groups)) * (256 * 8) + threadIdx.x * 8;
    const int d0 = static_cast<int>(at % D);
    const uint32_t bt = static_cast<uint32_t>(at / D);  // [batch, t], at most 2^30
    if (bt >= static_cast<uint32_t>(a.batch) * a.t) return;
    const int64_t b = bt / static_cast<uint32_t>(a.t);
    const int i = static_cast<int>(bt % static_cast<uint32_t>(a.t));
    const Span span = span_of(a.kv, b, a.t);
    int64_t pos = static_cast<int64_t>(span.start) + i;
    if (AT && a.at && i < span.count) pos = a.at[b * a.at_stride + i];
    const bool here = i < span.count && pos < a.positions && (!AT || pos >= 0);
    Rotation<D, 8, NORM> turn;
    if (here) turn.load(a.cos + pos * D, a.sin + pos * D, d0);
    if constexpr (NORM) turn.w.load(a.q_weight, d0);
    const uint16_t *from = a.q + b * a.q_stride[0] + i * a.q_stride[1];
    uint16_t *to = a.q_out + static_cast<int64_t>(bt) * a.heads * D + d0;
    Row<D, 8> x;
    for (int head = h0; head < min(h0 + a.heads_each, a.heads); ++head) {
      float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (here) {
        x.load(from + head * a.q_stride[2], d0);
        turn.apply(x, d0, y, NORM ? turn.factor(x, a.eps) : 1.f);
      }
      *reinterpret_cast<u32x4 *>(to + head * D) =
          (u32x4){pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])};
    }
    return;
  }
  // Codes of the block in their order; of values that are being turned, token by token with kPitch bytes a row.
  constexpr int kPitch = D + 4;
  __shared__ __align__(16) uint8_t tile[kKvBlock * D], rows[kKvBlock * kPitch];
  __shared__ float wave_max[4];
  const uint32_t groups = (a.kv.kv_heads + a.heads_each - 1) / a.heads_each;
  uint32_t rest = blockIdx.x;
  const int side = static_cast<int>(rest & 1);
  rest >>= 1;
  const int h0 = uniform(rest % groups) * a.heads_each;
  rest /= groups;
  const int nth = uniform(rest % static_cast<uint32_t>(a.seq_blocks));
  const int64_t b = uniform(rest / static_cast<uint32_t>(a.seq_blocks));
  Span span = span_of(a.kv, b, a.t);
  if (!AT || !a.at)
    span.count = static_cast<int>(least(span.count, a.positions > span.start ? a.positions - span.start : 0));
  const int block = span.start / kKvBlock + nth;
  const int lo = max(span.start, block * kKvBlock);  // the new tokens of this block: lo .. hi - 1
  const int hi = min(span.start + span.count, (block + 1) * kKvBlock);
  if (lo >= hi) return;
  const int page = page_of(a.kv, b, block);
  if (page < 0) return;
  const int before = lo - block * kKvBlock;  // older tokens of the block

  // thread: 16 values of a token of the block, a token's values side by side
  const int token = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks;
  const bool here = token < kKvBlock;
  const int pos = block * kKvBlock + token;
  const bool fresh = here && pos >= lo && pos < hi;
  const bool older = here && pos < lo;
  const int64_t i = pos - span.start;
  int64_t at = pos;
  if (AT && a.at && fresh) at = a.at[b * a.at_stride + i];
  const bool placed = !AT || (at >= 0 && at < a.positions);  // has a row of the tables
  const uint16_t *x = side == 0 ? a.k + b * a.k_stride[0] + i * a.k_stride[1] : a.v + b * a.v_stride[0] + i * a.v_stride[1];
  const int64_t head_stride = side == 0 ? a.k_stride[2] : a.v_stride[2];
  Rotation<D, 16, NORM> turn;
  if (fresh && side == 0 && placed) turn.load(a.cos + at * D, a.sin + at * D, 16 * chunk);
  if constexpr (NORM)
    if (side == 0) turn.w.load(a.k_weight, 16 * chunk);

  for (int head = h0; head < min(h0 + a.heads_each, a.kv.kv_heads); ++head) {
    const int64_t index = block_index(a.kv, page, side, head, block);
    uint8_t *codes = a.codes + index * (kKvBlock * D);
    float y[16];
    float largest = 0.f;
    if (AT && fresh && !placed) {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = 0.f;
    } else if (fresh) {
      if (side == 0) {
        Row<D, 16> row;
        row.load(x + head * head_stride, 16 * chunk);
        turn.apply(row, 16 * chunk, y, NORM ? turn.factor(row, a.eps) : 1.f);
      } else {
        const uint16_t *from = x + head * head_stride + 16 * chunk;
        const u32x4 w0 = *reinterpret_cast<const u32x4 *>(from), w1 = *reinterpret_cast<const u32x4 *>(from + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = bf16_value((j < 8 ? w0[j / 2] : w1[j / 2 - 4]) >> (16 * (j & 1)));
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float v = fabsf(y[j]);
        if (v <= FLT_MAX) largest = fmaxf(largest, v);
      }
    }
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) largest = fmaxf(largest, __shfl_xor(largest, m));
    if ((threadIdx.x & (kWave - 1)) == 0) wave_max[threadIdx.x / kWave] = largest;
    if (before > 0 && threadIdx.x * 16 < kKvBlock * D)
      *reinterpret_cast<u32x4 *>(tile + threadIdx.x * 16) = *reinterpret_cast<const u32x4 *>(codes + threadIdx.x * 16);
    __syncthreads();
    largest = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
    const float made = largest * (1.0f / kTop);
    const float old_scale = before > 0 ? a.scales[index] : 0.f;
    const float scale = fmaxf(old_scale, made < kTiny ? 0.f : made);
    const float inverse = scale > 0.f ? 1.0f / scale : 0.f;
    const float ratio = scale > old_scale ? old_scale * inverse : 1.0f;
    if (older) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        y[j] = code_value<FP8>(side == 0 ? tile[chunk * (16 * kKvBlock) + token * 16 + j]
                                         : tile[(16 * chunk + j) * kKvBlock + token]) * ratio;
    } else if (scale > 0.f) {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = fresh ? y[j] * inverse : 0.f;
    } else {  // an infinity is 0 like the block's other values; a NaN stays one
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = fresh && y[j] != y[j] ? y[j] : 0.f;
    }
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = code4<FP8>(y + 4 * j);
    if (side == 0) {
      if (here) *reinterpret_cast<u32x4 *>(codes + chunk * (16 * kKvBlock) + token * 16) = w;
    } else {
      // turned in squares of four tokens by four of d
      if (here) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(rows + token * kPitch + 16 * chunk + 4 * j) = w[j];
      }
      __syncthreads();
      const int t4 = threadIdx.x % 8, d4 = threadIdx.x / 8;
      if (d4 < D / 4) {
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const uint32_t *>(rows + (4 * t4 + j) * kPitch + 4 * d4);
        const uint32_t a01 = __builtin_amdgcn_perm(r[1], r[0], 0x05010400), a23 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400);
        const uint32_t b01 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602), b23 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602);
        const uint32_t out[4] = {__builtin_amdgcn_perm(a23, a01, 0x05040100), __builtin_amdgcn_perm(a23, a01, 0x07060302),
                                 __builtin_amdgcn_perm(b23, b01, 0x05040100), __builtin_amdgcn_perm(b23, b01, 0x07060302)};
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(tile + (4 * d4 + j) * kKvBlock + 4 * t4) = out[j];
      }
      __syncthreads();
      if (threadIdx.x * 16 < kKvBlock * D)
        *reinterpret_cast<u32x4 *>(codes + threadIdx.x * 16) = *reinterpret_cast<const u32x4 *>(tile + threadIdx.x * 16);
    }
    __syncthreads();  // every thread has read the old scale and is through with the shared arrays
    if (threadIdx.x == 0) a.scales[index] = scale;
  }
}

// ---- keeping the accepted nodes of a tree ---------------------------------------------------------------------------
//
// Token i of a sequence's path, which lies at start + path[i], moves to start + i, in every layer. The blocks that the
// path reaches into are read into LDS, three at most, and the ones that its tokens move to are made from there, so that
// none is read after it was written. A block's new scale is the largest of those that its tokens had (of the older ones
// too); codes that had another are rounded again, and what lies behind the last token becomes 0. A workgroup a head and
// side of a layer; each thread keeps its part of a block and only takes the moved tokens from LDS, one after the other
// (gathering all 32 byte by byte: 22 us for one sequence in 32 layers of 32 heads, 8.5 now). 32 sequences x 80 layers (8
// heads of 128, int8) take 131 us, 5.3 TB/s of the blocks read and written.
template <bool FP8>
__device__ __forceinline__ u32x4 again(u32x4 w, float ratio) {  // 16 codes under another scale
#pragma clang fp contract(off)
  if (ratio == 1.0f) return w;
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = code_value<FP8>(w[i] >> (8 * e) & 255u) * ratio;
    out[i] = code4<FP8>(y);
  }
  return out;
}

template <int D, bool FP8>
__global__ __launch_bounds__(2 * D) void kv8_keep_kernel(Kv8Keep a) {
#pragma clang fp contract(off)
  constexpr int kBytes = kKvBlock * D, kSources = 3;
  __shared__ __align__(16) uint8_t from[kSources][kBytes];
  uint32_t item = blockIdx.x;
  const int side = static_cast<int>(item & 1);
  item >>= 1;
  const int head = uniform(item % static_cast<uint32_t>(a.kv.kv_heads));
  item /= static_cast<uint32_t>(a.kv.kv_heads);
  const int64_t b = uniform(item % static_cast<uint32_t>(a.batch));
  const int64_t layer = uniform(item / static_cast<uint32_t>(a.batch));
  const int lane = threadIdx.x & (kWave - 1);
  // three waits for memory: for the sequence, its pages, their codes
  const int path = a.path[b * a.path_stride + min(lane, a.n - 1)];
  const Span span = span_of(a.kv, b, a.n);
  if (span.count == 0) return;
  const int first = span.start / kKvBlock;
  int pages[kSources];
#pragma unroll
  for (int j = 0; j < kSources; ++j)
    pages[j] = page_of(a.kv, b, min(first + j, a.kv.width * a.kv.page_blocks - 1));
  // the path ends where it does not ascend or leaves the tree or the table
  int node = lane < span.count ? path : 0;
  const int before = __shfl_up(node, 1);
  const int capacity = a.kv.width * a.kv.page_blocks * kKvBlock;
  const bool good = lane < span.count && node >= lane && node < 64 && node < capacity - span.start &&
                    (lane == 0 || node > before);
  const uint64_t stop = __ballot(!good);
  const int count = stop ? __builtin_ctzll(stop) : 64;
  if (count == 0) return;
  node = lane < count ? node : 0;
  const int last = (span.start + count - 1) / kKvBlock;
  const int reach = (span.start + __builtin_amdgcn_readlane(node, count - 1)) / kKvBlock;
  const int64_t layer_block = layer * a.kv.pages * 2 * a.kv.kv_heads * a.kv.page_blocks;

  int64_t index[kSources];
  float scale[kSources];
  u32x4 held[kSources];
#pragma unroll
  for (int j = 0; j < kSources; ++j) {
    index[j] = first + j > reach || pages[j] < 0 ? -1 : layer_block + block_index(a.kv, pages[j], side, head, first + j);
    scale[j] = 0.f;
    held[j] = (u32x4){0u, 0u, 0u, 0u};  // a hole holds zeros
    if (index[j] < 0) continue;
    scale[j] = a.scales[index[j]];
    held[j] = *reinterpret_cast<const u32x4 *>(a.codes + index[j] * kBytes + threadIdx.x * 16);
  }
#pragma unroll
  for (int j = 0; j < kSources; ++j) *reinterpret_cast<u32x4 *>(from[j] + threadIdx.x * 16) = held[j];
  // The largest scale of each block's tokens, a lane a token (both halves of the wave the same ones). A thread's 16
  // bytes are 16 values of a token (keys) or a value of 16 tokens (values): the older tokens' are the ones that it holds.
  float largest[kSources];
  int source[kSources];  // where the lane's token comes from
#pragma unroll
  for (int j = 0; j < kSources; ++j) {
    const int token = (first + j) * kKvBlock + lane % kKvBlock, nth = token - span.start;
    const int moved = span.start + __shfl(node, min(max(nth, 0), 63));
    source[j] = (nth < 0 ? token : moved) - first * kKvBlock;
    float of = 0.f;
#pragma unroll
    for (int i = 0; i < kSources; ++i)
      if (nth < count && source[j] / kKvBlock == i) of = scale[i];
#pragma unroll
    for (int m = 1; m < kKvBlock; m *= 2) of = fmaxf(of, __shfl_xor(of, m));
    largest[j] = of;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSources; ++j) {
    if (first + j > last || index[j] < 0) continue;
    const float made = largest[j], inverse = made > 0.f ? 1.0f / made : 0.f;
    const auto ratio = [&](int block) {
      const float was = block == 0 ? scale[0] : block == 1 ? scale[1] : scale[2];
      return made > was ? was * inverse : 1.0f;
    };
    const int base = (first + j) * kKvBlock;
    const int lo = max(span.start - base, 0), hi = min(span.start + count - base, kKvBlock);  // moved tokens: lo .. hi - 1
    u32x4 w = held[j];
    if (side == 0) {
      const int token = threadIdx.x % kKvBlock, chunk = threadIdx.x / kKvBlock;
      if (token >= lo)
        w = *reinterpret_cast<const u32x4 *>(from[0] + source[j] / kKvBlock * kBytes + chunk * (16 * kKvBlock) +
                                             source[j] % kKvBlock * 16);
      w = again<FP8>(w, ratio(source[j] / kKvBlock));
      if (token >= hi) w = (u32x4){0u, 0u, 0u, 0u};
    } else {
      const int half = threadIdx.x % 2 * 16, row = threadIdx.x / 2 * kKvBlock;
      w = again<FP8>(w, ratio(j));
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // the older tokens
        const int n = lo - half - 4 * k;
        w[k] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
      }
      for (int token = lo; token < hi; ++token) {
        const int s = __builtin_amdgcn_readlane(source[j], token);
        uint32_t code = from[0][s / kKvBlock * kBytes + row + s % kKvBlock];
        const float r = ratio(s / kKvBlock);
        if (r != 1.0f) {
          const float y[4] = {code_value<FP8>(code) * r, 0.f, 0.f, 0.f};
          code = code4<FP8>(y) & 255u;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if ((token - half) >> 2 == k) w[k] |= code << (8 * (token & 3));
      }
    }
    *reinterpret_cast<u32x4 *>(a.codes + index[j] * kBytes + threadIdx.x * 16) = w;
    if (threadIdx.x == 0) a.scales[index[j]] = made;
  }
}

// ---- copying pages -------------------------------------------------------------------------------------------------

constexpr int kCopyBytes = 32 * 1024;  // of one workgroup: eight 16-byte loads in flight a lane

// The argument is read where it lies: as a value, its table of pairs would be copied into registers to be indexed.
__global__ __launch_bounds__(256) void kv8_copy_kernel(Kv8Copy) {
  const auto &a = *(const __attribute__((address_space(4))) Kv8Copy *)__builtin_amdgcn_kernarg_segment_ptr();
  uint32_t item = blockIdx.x;
  const uint32_t piece = uniform(item % a.pieces);
  item /= a.pieces;
  const uint32_t pair = uniform(item % a.n);
  const int64_t layer = uniform(item / a.n);
  const int64_t from = layer * a.pages + a.pair[pair].src, to = layer * a.pages + a.pair[pair].dst;
  const uint32_t bytes = a.page_bytes, at = piece * kCopyBytes;
  const u32x4 *src = reinterpret_cast<const u32x4 *>(a.codes + from * bytes + at) + threadIdx.x;
  u32x4 *dst = reinterpret_cast<u32x4 *>(a.codes + to * bytes + at) + threadIdx.x;
  if (at + kCopyBytes <= bytes) {
    u32x4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = src[i * 256];
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i * 256] = v[i];
  } else {  // a page is whole workgroup loads of 4096 bytes: two sides of 32 tokens of 64 bytes at least
#pragma unroll 1
    for (uint32_t i = 0; i < (bytes - at) / 4096; ++i) dst[i * 256] = src[i * 256];
  }
  if (piece == 0) {
    const int n = a.page_scales;
    const float *from_scales = a.scales + from * n;
    float *to_scales = a.scales + to * n;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += 256) to_scales[i] = from_scales[i];
  }
}

}  // namespace

// Which kernel runs, and how often the keys are split, by what it costs in units of 0.1 us: a round of workgroups, one
// a CU, takes a start and its blocks; the join a launch and the partial values' way through memory and back, shorter for
// trees of up to 16 chunks (kv8_join_rows_kernel).
//                                 a block  a start
//   up to 16 rows                       1       16
//   tiles of 32 rows                    2       30
//   tiles of 256 rows                  10       40
// Measured, us, on eight heads unless said: 1 token (8 rows) over 500 keys 6.8 unsplit, 9.0 in two; over 32000 18.0 in
// 32 splits, 21.9 in 63, 36 in 4; 256 heads over 4096 keys 48.5 unsplit, 56 in two. 512 rows over 500 keys 10.9 in
// tiles of 32 and 26.8 in tiles of 256, over 4000 31.4 and 38.0, over 30000 132 and 98; 128 heads of 512 rows over
// 2000 keys 205 and 111, 32 heads 52.5 and 62. Up to 64 rows tiles of 32 were never slower (14.6 and 18.7 over 4000).
// Trees in tiles of 256 rows are dealt to the CUs, without rounds; up to half as many heads as CUs start once, more of
// them about twice. In units again:
//   a block 10, with more than 128 rows 12 (two waves of a SIMD at work); a start 80; 32 rows of the other kernel 3
// Sequences of a batch are rarely all of the longest one's length, and dealing takes the mean: a fifth less. Measured,
// us, int8, in tiles of 32 and of 256: 80 rows of 64 heads over 4096 keys at most 38.9 and 28.2, of 128 heads over 8000
// 147 and 118; 128 rows of 16 heads over 32000 82.3 and 73.1, of 64 over 1000 19.5 and 28.2, over 4096 48.2 and 45.1, of
// 128 over 2000 at most 38.0 and 31.0; 512 of 8 over 4096 31.4 and 39.5; 96 of 256 over 1000 at most 34.2 and 58.5, 80 of
// 512 over 2000 at most 68.3 and 109.
void plan_kv8_attention(Kv8Attention *p, int64_t max_tokens, bool tree, int cus, int xcds) {
  p->xcds = std::max(1, xcds);
  p->rep = p->heads / p->kv.kv_heads;
  p->rows = p->t * p->rep;
  const int64_t heads = static_cast<int64_t>(p->batch) * p->kv.kv_heads;
  const int64_t blocks = std::max<int64_t>(1, (max_tokens + kKvBlock - 1) / kKvBlock);
  int64_t best = INT64_MAX, splits = 1;
  const auto weigh = [&](int tile_rows, int64_t block_cost, int64_t start_cost) {
    const int64_t items = heads * ((p->rows + tile_rows - 1) / tile_rows);
    for (int64_t rounds = 0; rounds <= 8; ++rounds) {  // whole rounds of splits, or none
      const int64_t s = rounds == 0 ? 1 : std::min(rounds * cus / items, blocks / 8);
      if (s < 1 || (rounds > 0 && s == 1)) continue;
      const int64_t cost = (items * s + cus - 1) / cus * ((blocks + s - 1) / s * block_cost + start_cost) +
                           (s == 1 ? 0 : 30 + items * tile_rows * s / (tree && s <= kRowJoinSplits ? 900 : 385));
      if (cost >= best) continue;
      best = cost;
      splits = s;
      p->tile_rows = tile_rows;
    }
  };
  if (p->rows <= 16) {
    weigh(p->rows, 1, 16);
  } else {
    weigh(32, tree && p->rows > 64 ? 3 : 2, 30);
    if (p->rows > 64 && !tree) weigh(32 * kTileWaves, 10, 40);
    if (p->rows > 64 && tree) {
      const int64_t items = heads * ((p->rows + 32 * kTileWaves - 1) / (32 * kTileWaves));
      const bool whole = items <= cus / 2;
      int64_t cost = (items * blocks * (p->rows > 128 ? 12 : 10) + (whole ? cus : items + cus) * 80) / cus + 30 +
                     (items + cus) * std::min(p->rows, 32 * kTileWaves) / 900;
      if (whole && p->batch > 1) cost = cost * 4 / 5;
      if (cost < best) p->tile_rows = 32 * kTileWaves;
    }
  }
  p->row_tiles = (p->rows + p->tile_rows - 1) / p->tile_rows;
  p->tile_items = heads * p->row_tiles;
  p->part_rows = std::min(p->rows, p->tile_rows);
  if (tree && p->tile_rows > 32) {  // dealt: a workgroup a CU
    p->splits = p->chunk = 1;
    p->items = static_cast<uint32_t>(std::max(1, cus / p->xcds) * p->xcds);
    p->part_bytes = p->items * (static_cast<size_t>(2) * p->part_rows * (p->kv.d + 2) + 4) * sizeof(float);
    return;
  }
  p->chunk = static_cast<int>((blocks + splits - 1) / splits);  // the last one goes on to the end of the sequence,
  p->splits = static_cast<int>((blocks + p->chunk - 1) / p->chunk);  // whatever max_tokens says
  const int64_t items = p->tile_items * p->splits;
  p->items = static_cast<uint32_t>(std::min<int64_t>(items, UINT32_MAX));  // too many for a launch: the caller refuses
  p->part_bytes = p->splits > 1 ? static_cast<size_t>(items) * p->tile_rows * (p->kv.d + 2) * sizeof(float) : 0;
}

template <bool TREE>
hipError_t launch_attention_over(const Kv8Attention &p, hipStream_t stream) {
  if (p.kv.d == 128)
    return p.kv.fp8 ? launch_attend<128, true, TREE>(p, stream) : launch_attend<128, false, TREE>(p, stream);
  return p.kv.fp8 ? launch_attend<64, true, TREE>(p, stream) : launch_attend<64, false, TREE>(p, stream);
}

hipError_t launch_kv8_attention(const Kv8Attention &p, hipStream_t stream) {
  return p.tree ? launch_attention_over<true>(p, stream) : launch_attention_over<false>(p, stream);
}

void plan_kv8_append(Kv8Append *p, int cus) {
  const int kv = p->kv.kv_heads;
  p->seq_blocks = (p->t + 2 * kKvBlock - 2) / kKvBlock;
  const int64_t each = static_cast<int64_t>(p->batch) * p->seq_blocks * 2;
  p->heads_each = each * kv >= 16 * static_cast<int64_t>(cus) ? 4 : 1;  // four where eight workgroups a CU remain
  const int64_t row_items = (static_cast<int64_t>(p->batch) * p->t * p->kv.d + 2047) / 2048;
  p->block_items = each * ((kv + p->heads_each - 1) / p->heads_each);
  p->query_items = row_items * ((p->heads + p->heads_each - 1) / p->heads_each);
}

template <bool AT, bool NORM>
void start_append(const Kv8Append &p, dim3 grid, dim3 block, hipStream_t stream) {
  if (p.kv.d == 128) {
    if (p.kv.fp8) hipLaunchKernelGGL((kv8_append_kernel<128, true, AT, NORM>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((kv8_append_kernel<128, false, AT, NORM>), grid, block, 0, stream, p);
  } else {
    if (p.kv.fp8) hipLaunchKernelGGL((kv8_append_kernel<64, true, AT, NORM>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((kv8_append_kernel<64, false, AT, NORM>), grid, block, 0, stream, p);
  }
}

hipError_t launch_kv8_append(const Kv8Append &p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.block_items + p.query_items)), block(256);
  if (p.q_weight) start_append<true, true>(p, grid, block, stream);
  else if (p.at) start_append<true, false>(p, grid, block, stream);
  else start_append<false, false>(p, grid, block, stream);
  return hipGetLastError();
}

hipError_t launch_kv8_copy(const Kv8Copy &p, hipStream_t stream) {
  hipLaunchKernelGGL(kv8_copy_kernel, dim3(static_cast<unsigned>(p.layers) * p.n * p.pieces), dim3(256), kLdsToken,
                     stream, p);
  return hipGetLastError();
}

hipError_t launch_kv8_keep(const Kv8Keep &p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.layers * p.batch * p.kv.kv_heads * 2)), block(2 * p.kv.d);
  if (p.kv.d == 128) {
    if (p.kv.fp8) hipLaunchKernelGGL((kv8_keep_kernel<128, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((kv8_keep_kernel<128, false>), grid, block, 0, stream, p);
  } else {
    if (p.kv.fp8) hipLaunchKernelGGL((kv8_keep_kernel<64, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((kv8_keep_kernel<64, false>), grid, block, 0, stream, p);
  }
  return hipGetLastError();
}

uint32_t kv8_copy_pieces(uint32_t page_bytes) { return (page_bytes + kCopyBytes - 1) / kCopyBytes; }

}  // namespace ftx
