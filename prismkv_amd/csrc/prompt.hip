// Causal attention of a whole prompt, a chunk of one or a turn over the paged cache:
// the queries of every sequence's last slots, packed, over all of its slots.
//
// Rows: the queries of the heads that share a KV head are the rows of one matrix,
// m group of them for m tokens (row = token * group + head), so that few tokens of many
// heads still fill a tile; row i of a sequence of n slots sees slots [0, n - m + i /
// group].  4 head_dim flops for a row and a slot that it sees against 2 x 2 head_dim
// bytes for a slot and 128 rows: the matrix products bound it, unless the rows are few.
// Measured: 16384 rows of 8 x 4 heads of 128 in bf16 2114 us = 1.04 PFLOP/s (a product of
// 8192^3 reaches 1.12); 48 rows over 65048 slots 91 us = 562 TFLOP/s and 2.9 TB/s; fp16,
// head_dim 64, 9 ragged sequences of 1.0K rows 149 us = 516; fp32, head_dim 256, 4097 rows
// 1043 us = 96 (of 153); over 4-bit pages 6007 rows over 5 x 9K slots 953 us = 912.  (The
// clock goes with the power and the card: the same kernel takes 2040 to 2120 us for the
// first, and figures are to be compared with those beside them.)
#include <cfloat>
#include <type_traits>

#include "paged_host.h"
#include "prompt_plan.h"

namespace prismkv {
namespace {

constexpr int kWaves = kTileRows / 32, kThreads = 64 * kWaves;
// Keys and values that are staged at a time.
template <int DT, int D>
constexpr int kTileTokens = tile_tokens(kElem<DT> * D);
// Waves of a SIMD, by the registers that products, queries and staged rows take.  (Three
// for head_dim 64 in 16 bits; the widening from 4 bits has no room for that: 2000 rows over
// 4000 slots 87 us, with two 84.)
template <int DT, int D>
constexpr int kOccupancy = kElem<DT> * D > 256 ? 1 : kElem<DT> * D == 128 && !kInFour<DT> ? 3 : 2;

// By how much (in powers of 2) a row's largest score may pass the maximum that its weights
// are taken from before what was summed so far is multiplied anew: nearly every tile raises
// one of a wave's 32 rows' a little.  fp16 has no room above its bias.
template <int DT>
constexpr float kLead = kType<DT> == kFp16 ? 0.f : 8.f;

constexpr int kRawBuffer = 0x27000;  // a buffer resource's last word: 32-bit data, no swizzle

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Prompt {
  const char *q, *k, *v;
  const uint8_t *ks, *vs;
  const int32_t *table, *lengths, *offsets;
  char* out;
  float *lse, *state;
  unsigned* err;
  int64_t head_bytes, scale_head;
  unsigned page_units, slot_units;              // 16 bytes
  unsigned scale_page_units, scale_slot_units;  // head_dim / 32 bytes
  PageDiv div;
  unsigned q_and, q_xor;  // the scale's sign, or a scale of 0, goes to the queries
  float scale;            // log2(e) times the caller's magnitude
  int rows, sequences, kv_heads, group, page_size, max_pages, pages, slots, states, cut_tiles;
};

// New rows m from `first` of a sequence, its slots, and its tiles of rows and of keys.
struct PromptRows {
  int first, m, n, tiles, key_tiles;
};

template <int kTokens>
__device__ __forceinline__ PromptRows prompt_rows(const Prompt& a, int b) {
  PromptRows s{0, 0, 0, 0, 0};
  if (b >= a.sequences) return s;
  s.first = a.offsets ? min(max(a.offsets[b], 0), a.rows) : b;
  const int to = a.offsets ? min(max(a.offsets[b + 1], 0), a.rows) : b + 1;
  s.m = max(to - s.first, 0);
  s.n = min(max(a.lengths[b], 0), a.slots);
  s.tiles = (s.m * a.group + kTileRows - 1) / kTileRows;  // (rows * group < 2^30)
  s.key_tiles = (s.n + kTokens - 1) / kTokens;
  return s;
}

// Every wave finds the plan, and its own item, by itself from the lengths (two lane scans
// for every 64 sequences).
template <int DT, int kTokens>
__device__ __forceinline__ PromptPlan prompt_plan(const Prompt& a) {
  if (!a.states) return PromptPlan{1, INT32_MAX};  // (nothing is cut)
  uint64_t sum = 0;
  int tiles = 0;
  for (int b = threadIdx.x & 63; b < a.sequences; b += 64) {
    const PromptRows s = prompt_rows<kTokens>(a, b);
    sum += (uint64_t)s.tiles * s.key_tiles;
    tiles += s.tiles;
  }
  const uint64_t low = wave_sum_i((int)(sum & 0xffffffu)), high = wave_sum_i((int)(sum >> 24));
  return prompt_cuts(((high << 24) + low) * a.kv_heads, wave_sum_i(tiles) * a.kv_heads, kType<DT> == kFp32);
}

// Item `index` of the launch: a tile of rows of sequence b and KV head h, chunk `chunk`
// of the `chunks` that its keys are cut into, `most` of which its longest tile has;
// `state` counts the items of sequences that are cut.
struct PromptItem {
  PromptRows s;
  int b, h, tile, chunk, most, state;
};

// The heads go round fastest: with 8 of them the workgroups of a head share an XCD's
// L2, and what they read at a time is the same.  A sequence's last tiles, which see the
// most, come first.
template <int kTokens>
__device__ __forceinline__ bool find_item(const Prompt& a, const PromptPlan& plan, int index, bool cut_tiles, PromptItem& it) {
  int base = 0, cut = 0;
  for (int b0 = 0; b0 < a.sequences; b0 += 64) {
    const PromptRows s = prompt_rows<kTokens>(a, b0 + (threadIdx.x & 63));
    const int most = plan.chunks(s.key_tiles);
    // (cut_tiles: only those of sequences that are cut, one for all chunks of a tile)
    const int states = most > 1 ? s.tiles * most * a.kv_heads : 0;
    const int count = cut_tiles ? (most > 1 ? s.tiles * a.kv_heads : 0) : s.tiles * most * a.kv_heads;
    const int upto = (int)wave_incl_scan((unsigned)count), total = __builtin_amdgcn_readlane(upto, 63);
    const int states_upto = (int)wave_incl_scan((unsigned)states);
    if (index - base < total) {
      const int l = max(__ffsll((unsigned long long)__ballot(upto > index - base)) - 1, 0);
      it.s.first = __builtin_amdgcn_readlane(s.first, l);
      it.s.m = __builtin_amdgcn_readlane(s.m, l);
      it.s.n = __builtin_amdgcn_readlane(s.n, l);
      it.s.tiles = __builtin_amdgcn_readlane(s.tiles, l);
      it.s.key_tiles = __builtin_amdgcn_readlane(s.key_tiles, l);
      it.most = __builtin_amdgcn_readlane(most, l);
      it.b = b0 + l;
      int at = index - base - __builtin_amdgcn_readlane(upto, l) + __builtin_amdgcn_readlane(count, l);
      if ((unsigned)at >= (unsigned)__builtin_amdgcn_readlane(count, l)) return false;  // (offsets that do not ascend)
      it.state = cut + __builtin_amdgcn_readlane(states_upto, l) - __builtin_amdgcn_readlane(states, l) + (cut_tiles ? 0 : at);
      it.h = at % a.kv_heads;
      at /= a.kv_heads;
      it.chunk = cut_tiles ? 0 : at % it.most;
      it.tile = it.s.tiles - 1 - (cut_tiles ? at : at / it.most);
      return true;
    }
    base += total;
    cut += __builtin_amdgcn_readlane(states_upto, 63);
  }
  return false;
}

// The chunks that a tile's keys are cut into evenly, and how many tiles of keys it sees.
template <int kTokens>
struct PromptCut {
  int end, tiles, chunks, each;  // slots and tiles that its last row sees; tiles of a chunk
  __device__ __forceinline__ PromptCut(const Prompt& a, const PromptItem& it, const PromptPlan& plan) {
    const int last = (min((it.tile + 1) * kTileRows, it.s.m * a.group) - 1) / a.group;  // the tile's last token
    end = max(it.s.n - it.s.m + last + 1, 0);
    tiles = (end + kTokens - 1) / kTokens;
    chunks = it.most > 1 ? (tiles + plan.per_item - 1) / plan.per_item : tiles > 0;
    each = chunks ? (tiles + chunks - 1) / chunks : 0;
    if (each) chunks = (tiles + each - 1) / each;
  }
};

// Where chunk c (16 bytes) of row r lies in a staged tile of rows of kC chunks: moved
// within the row so that neither 16 rows' same chunk (keys) nor two neighbouring chunks
// of four rows (values, read transposed) meet in a bank.
template <int kC>
__device__ __forceinline__ int staged(int r, int c) {
  const int f = kC == 8 ? (r & 2) | (r & 4) | ((r >> 3) & 1) : ((r & 3) << 1) | ((r >> 2) & 1) | (r & 8);
  return (r * kC + (c ^ f)) * 16;
}

// The same places for what a lane reads in the main loop, as one address of the lane, a
// constant to xor it with (few of them) and a constant offset: written out, as the
// compiler does not take `staged` apart and keeps an address for every read.
template <int kC>
struct KeyAt {  // chunk 2c + half of row 32i + col
  int lane;
  __device__ __forceinline__ KeyAt(int col, int half) : lane(staged<kC>(col, half)) {}
  __device__ __forceinline__ int of(int i, int c) const {
    constexpr int kMask = kC == 8 ? 7 : 15;
    return (lane ^ ((2 * c & kMask) << 4)) + ((2 * c & ~kMask) + 32 * i * kC) * 16;
  }
};
template <int kC>
struct ValueAt {  // chunk 4d + 2 side + (in >> 1 & 1) of row 32i + 16u + 8 hi + 4 half + in / 4, its in & 1 part
  int lane;
  __device__ __forceinline__ ValueAt(int l)
      : lane(staged<kC>(4 * (l >> 5) + (l >> 2 & 3), 2 * (l >> 4 & 1) + (l >> 1 & 1)) + 8 * (l & 1)) {}
  __device__ __forceinline__ int of(int i, int u, int hi, int d) const {
    const int rows = (32 * i + 16 * u + 8 * hi) * kC * 16;
    if constexpr (kC == 8) return (lane ^ ((4 * d ^ hi) << 4)) + rows;
    else return (lane ^ (4 * (d & 1) << 4)) + rows + (8 * ((d >> 1 & 1) ^ hi) + 16 * (d >> 2)) * 16;
  }
};
template <int kC, int kVec>
struct FloatsAt {  // fp32 elements 32 kVec g + kVec col .. of row 32i + 8 (r / 4) + 4 half + r % 4
  int lane;
  __device__ __forceinline__ FloatsAt(int col, int half)
      : lane(staged<kC>(4 * half, col * kVec / 4) + 4 * (col * kVec & 3)) {}
  __device__ __forceinline__ int of(int i, int r, int g) const {
    return (lane ^ ((r % 4 << 1 | (r / 4 & 1) << 3) << 4)) + ((32 * i + 8 * (r / 4) + r % 4) * kC + 8 * kVec * g) * 16;
  }
};

template <int DT>
__device__ __forceinline__ f32x16 mfma_rows(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kType<DT> == kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else if constexpr (kType<DT> == kFp16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
}

// Two probabilities as a word of the 16-bit type, rounded to nearest: half a step of
// the type relative to each, where two or three terms would take as many products with V
// again (`attend` has them).  Over many slots of normal V that is 0.0016 of the output in
// bf16, whose own rounding is 0.0017 (fp16 0.00015 and 0.00021).  The row's sum is of what
// was not rounded, but for its largest weight (share_largest).  fp16 takes its least number
// for what is below it, so that an infinite V is not multiplied by 0 (2^-39 of the largest
// weight, with the bias).
template <int DT>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr (kType<DT> == kBf16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, bf16x2{(__bf16)a, (__bf16)b});
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, f16x2{(_Float16)a, (_Float16)b});
  }
}

// 16 bytes with 0 for each element that is an infinity or NaN; whether there was one.
template <int DT>
__device__ __forceinline__ u32x4 without_special(u32x4 x, bool& any) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned w = x[e];
    if constexpr (kType<DT> == kFp32) {
      x[e] = (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    } else {
      constexpr unsigned kMask = kType<DT> == kBf16 ? 0x7f80u : 0x7c00u;
      x[e] = ((w & kMask) == kMask ? 0u : w & 0xffffu) | ((w >> 16 & kMask) == kMask ? 0u : w & 0xffff0000u);
    }
    any |= x[e] != w;
  }
  return x;
}

// A thread's part of the tiles of keys and values on their way from the pages to LDS: 16
// bytes straight there, or from 4 bits through registers, where they are widened.  Each
// lane looks up one row's place, two tiles ahead, and the rows' readers take it from
// there.  Rows past the end repeat the last one: no row sees them.
//
// kGroups: the 64 / kC rows that a wave loads at once always lie in one page.  Then their
// place is one scalar, and a buffer load from it has a lane's offset alone.  (Beside the
// vector work that this saves: while a global load to LDS is on its way the compiler waits
// for all reads of LDS at once.  4000 rows over pages of 64 slots 150 us, of 31 slots 157;
// of head_dim 256 371 and 427.)
template <int DT, int D, bool kGroups>
struct Stage {
  static constexpr int kTokens = kTileTokens<DT, D>;
  static constexpr int kC = D * kElem<DT> / 16;            // chunks of a row
  static constexpr int kEach = kTokens * kC / kThreads;    // chunks of a thread
  static constexpr int kRaw = kInFour<DT> ? kEach : 1;
  static constexpr int kRows = 64 / kC;                    // rows of a wave's load
  typedef const __attribute__((address_space(1))) void* Global;
  typedef __attribute__((address_space(3))) void* Local;
  const Prompt& a;
  const char *k, *v;
  const uint8_t *ks, *vs;
  const int32_t* tab;
  int end, row, chunk;
  bool bad = false;
  int page, token;        // of this lane's row
  // places (16-byte units) of the next tile of values and of the next one of keys, which
  // is the tile behind it
  unsigned v_at[kEach], k_at[kEach];
  unsigned v_scale_at[kRaw], k_scale_at[kRaw];
  unsigned kw[kRaw], vw[kRaw], kb[kRaw], vb[kRaw];

  __device__ __forceinline__ Stage(const Prompt& a, int b, int h, int end) : a(a), end(end) {
    row = threadIdx.x / kC;
    chunk = threadIdx.x % kC;
    k = a.k + (size_t)h * a.head_bytes;
    v = a.v + (size_t)h * a.head_bytes;
    if constexpr (kInFour<DT>) {
      k += 4 * chunk;
      v += 4 * chunk;
      ks = a.ks + (size_t)h * a.scale_head + chunk / 4;
      vs = a.vs + (size_t)h * a.scale_head + chunk / 4;
    }
    tab = a.table + (size_t)b * a.max_pages;
  }
  static __device__ __forceinline__ int step(int i) { return i * (kThreads / kC); }
  __device__ __forceinline__ void ask(int t0) {
    token = min(t0 + (int)(threadIdx.x & (kTokens - 1)), end - 1);
    if constexpr (kGroups) token &= -kRows;  // (the page has the rows behind the end that are loaded too)
    page = tab[a.div.of(token)];
  }
  __device__ __forceinline__ void move() {
    bad |= (unsigned)page >= (unsigned)a.pages;
    const unsigned p = (unsigned)page < (unsigned)a.pages ? (unsigned)page : 0u;
    const unsigned in = (unsigned)(token - a.div.of(token) * a.page_size);
    const unsigned place = p * a.page_units + in * a.slot_units;
    const unsigned scale_place = p * a.scale_page_units + in * a.scale_slot_units;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      v_at[i] = k_at[i];
      if constexpr (kGroups)
        k_at[i] = (unsigned)__builtin_amdgcn_readlane((int)place, kRows * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + step(i));
      else
        k_at[i] = (unsigned)__shfl((int)place, row + step(i));
      if constexpr (kInFour<DT>) {
        v_scale_at[i] = k_scale_at[i];
        k_scale_at[i] = (unsigned)__shfl((int)scale_place, row + step(i));
      }
    }
  }
  // Which chunk of its row a lane reads: LDS takes the lanes' 16 bytes one after another.
  __device__ __forceinline__ int source(int i) const {
    return (staged<kC>(row + step(i), chunk) & (16 * kC - 1));
  }
  __device__ __forceinline__ void issue(const char* from, const unsigned (&at)[kEach], char* tile, int i0 = 0, int i1 = kEach) const {
#pragma unroll
    for (int i = i0; i < i1; ++i) {
      const Local to = (Local)(tile + (64 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + i * kThreads) * 16);
      if constexpr (kGroups) {
        const auto rows = __builtin_amdgcn_make_buffer_rsrc((void*)(from + ((size_t)at[i] << 4)), 0, -1, kRawBuffer);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, to, 16, (row & (kRows - 1)) * (int)(a.slot_units << 4) + source(i), 0, 0, 0);
      } else {
        __builtin_amdgcn_global_load_lds((Global)(from + ((size_t)at[i] << 4) + source(i)), to, 16, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void issue_k(char* tile) {
    if constexpr (kInFour<DT>) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        kw[i] = *reinterpret_cast<const unsigned*>(k + ((size_t)k_at[i] << 4));
        kb[i] = ks[(size_t)k_scale_at[i] * (D / 32)];
      }
    } else {
      issue(k, k_at, tile);
    }
  }
  __device__ __forceinline__ void issue_v(char* tile) {
    if constexpr (kInFour<DT>) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        vw[i] = *reinterpret_cast<const unsigned*>(v + ((size_t)v_at[i] << 4));
        vb[i] = vs[(size_t)v_scale_at[i] * (D / 32)];
      }
    } else {
      issue(v, v_at, tile);
    }
  }
  __device__ __forceinline__ void finish(char* tile, const unsigned (&w)[kRaw], const unsigned (&b)[kRaw]) const {
#pragma unroll
    for (int i = 0; i < kRaw; ++i)
      *reinterpret_cast<u32x4*>(tile + staged<kC>(row + step(i), chunk)) = widen8<DT>(w[i], __uint_as_float(b[i] << 23));
  }
  __device__ __forceinline__ void finish_k(char* tile) const {
    if constexpr (kInFour<DT>) finish(tile, kw, kb);
  }
  __device__ __forceinline__ void finish_v(char* tile) const {
    if constexpr (kInFour<DT>) finish(tile, vw, vb);
  }
  // Takes the infinities and NaN out of a tile of values; whether there were any.
  static __device__ __forceinline__ bool clean(char* tile) {
    bool special = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      u32x4* x = reinterpret_cast<u32x4*>(tile) + threadIdx.x + i * kThreads;
      bool any = false;
      const u32x4 y = without_special<DT>(*x, any);
      if (any) *x = y;
      special |= any;
    }
    return special;
  }
};

// Four elements from LDS in 32 bits.
template <int DT>
__device__ __forceinline__ float4 four_of(const char* p) {
  if constexpr (kType<DT> == kFp32) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    if constexpr (kType<DT> == kBf16) {
      return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
    } else {
      typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
      const f16x4 h = __builtin_bit_cast(f16x4, w);
      return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
    }
  }
}

// Writes four outputs of a row, and its log-sum.
template <int DT, int D>
__device__ __forceinline__ void put_four(const Prompt& a, size_t row_head, int dim, float den, float4 x) {
  // (16-bit types: one division, and a rounding more that theirs hides)
  const float inverse = 1.f / den;
  const float y[4] = {kType<DT> == kFp32 ? x.x / den : x.x * inverse, kType<DT> == kFp32 ? x.y / den : x.y * inverse,
                      kType<DT> == kFp32 ? x.z / den : x.z * inverse, kType<DT> == kFp32 ? x.w / den : x.w * inverse};
  float z[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = den == 0.f ? 0.f : y[e];
  char* to = a.out + (row_head * D + dim) * kElem<DT>;
  if constexpr (kType<DT> == kFp32) {
    *reinterpret_cast<float4*>(to) = make_float4(z[0], z[1], z[2], z[3]);
  } else {
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3]));
  }
}

template <int DT>
__device__ __forceinline__ float prompt_lse(float m, float den) {
  return den == 0.f ? -INFINITY : (m + (log2f(den) - kBias<DT>)) * 0.693147180559945309f;
}

// Factor of a state with maximum m under the joint maximum M >= m (no state: 0).
__device__ __forceinline__ float state_factor(float m, float M) {
  return m == -INFINITY ? 0.f : m == M ? 1.f : exp2f(m - M);
}

// Whether the largest weight of a row is rounded: not where it is 1 (2^kBias).
template <int DT>
constexpr bool kShared = kType<DT> == kBf16;

// What the sums of a row are multiplied by before they are divided by its sum z: that with
// its largest weight as V was multiplied by it, so that a slot that outweighs all others
// comes back as its V (without, off by up to 2^-8, the same for every dim).  `top` is that
// slot's score and `at` the maximum that its weight was taken from, `m` the last one.  (The
// sum of all rounded weights, by two-element products of the words, is little better, 0.0014
// for 0.0016 above, and makes 16384 rows take 6% longer, where this makes it 0.6.  From 2^22
// on a maximum's weights are taken otherwise, of scores that are off by 1/4 and more.)
template <int DT>
__device__ __forceinline__ float share_largest(float top, float at, float m, float scale, float z) {
  const float p = __builtin_amdgcn_exp2f(fmaf(top, scale, (float)kBias<DT> - at));
  const float error = __uint_as_float(pack2<DT>(p, 0.f) << 16) / p - 1.f;
  const float sum = z + error * __builtin_amdgcn_exp2f(fmaf(top, scale, (float)kBias<DT> - m));
  return fabsf(at) < 0x1p22f ? z / sum : 1.f;
}

// A state: maxima and sums [2][128], then the products [D / 4][128] of four dims.
template <int D>
constexpr int kStateFloats = kTileRows * (D + 2);

// Scores are computed transposed, S^T = K Q^T, so that a lane has 16 (of 32 tokens)
// scores of one row (lane & 31; the other half of the tokens with lane ^ 32): its maximum
// and sum need one exchange a tile, its factors none, and its probabilities are the right
// operand of O^T = V^T P^T as they stand, the tokens being summed in the order in which
// they lie in registers (8 (r / 4) + 4 (lane / 32) + r % 4).  V^T comes out of LDS by
// transposing reads.
template <int DT, int D, bool kGroups>
__global__ __launch_bounds__(kThreads, (kOccupancy<DT, D>)) void prompt_kernel(Prompt a) {
  constexpr int kTokens = kTileTokens<DT, D>, kT = kTokens / 32;
  constexpr int kC = D * kElem<DT> / 16;  // 16-byte chunks of a row; half as many steps of the product (fp32: of four)
  constexpr int kTile = kTokens * kC * 16;  // bytes
  // Whether the next tiles' loads are issued between the products (4097 fp32 rows 1037 us,
  // before them 1070; 16384 rows of head_dim 128 2121 and 2146) or before them (4000 rows of
  // head_dim 256 in fp16 500, between them 511; in bf16 368 and 363; of 64 no difference).
  constexpr bool kLate = kGroups && (kType<DT> == kFp32 || D == 128);
  __shared__ __attribute__((aligned(16))) char keys0[kTile], keys1[kTile], values0[kTile], values1[kTile];
  if (blockIdx.x == 0 && a.offsets)
    for (int b = threadIdx.x; b < a.sequences; b += kThreads) {
      const int from = a.offsets[b], to = a.offsets[b + 1];
      if (from > to || (b == 0 && from) || (b == a.sequences - 1 && to != a.rows))
        report_error(a.err, error_host_slot(a.err), kErrOffsets);
    }
  const PromptPlan plan = prompt_plan<DT, kTokens>(a);
  PromptItem it;
  if (!find_item<kTokens>(a, plan, blockIdx.x, false, it)) return;
  const PromptCut<kTokens> cut(a, it, plan);
  if (it.chunk > 0 && it.chunk >= cut.chunks) return;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = it.s.m * a.group - it.tile * kTileRows;  // of the tile and behind it
  const int row = 32 * w + col;
  const bool valid = row < rows;
  const int of = it.tile * kTileRows + min(row, rows - 1), token = of / a.group;
  const int before = it.s.n - it.s.m;
  if (before < 0 && threadIdx.x == 0) report_error(a.err, error_host_slot(a.err), kErrHeld);
  const int limit = valid ? before + token : -1;  // the last slot that the row sees
  // what the wave's first row sees, the tile's
  const int wave_first = __builtin_amdgcn_readlane(limit, 0);
  const int tile_first = before + it.tile * kTileRows / a.group;
  const size_t row_head = (size_t)(it.s.first + token) * a.kv_heads * a.group + it.h * a.group + (of - token * a.group);

  u32x4 q[kC / 2];
  {
    const char* from = a.q + row_head * (D * kElem<DT>) + 16 * half;
#pragma unroll
    for (int c = 0; c < kC / 2; ++c) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(from + 32 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[c][e] = (x[e] & a.q_and) ^ a.q_xor;
    }
  }
  const KeyAt<kC> key_at(col, half);
  f32x16 acc[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  // A lane's sums, four neighbouring dims at a time: row i of product d is dim 32d + i or,
  // in fp32, 32 kVec (d / kVec) + kVec i + d % kVec.
  constexpr int kVec = D >= 128 ? 4 : 2;
  struct Place {
    int d, r;
  };
  auto place = [](int n, int e) {
    if constexpr (kType<DT> != kFp32) return Place{n / 4, n % 4 * 4 + e};
    else if constexpr (kVec == 4) return Place{n / 16 * 4 + e, n % 16};
    else return Place{e % 2, 2 * n + e / 2};
  };
  auto four = [&](int n) {
    const Place x = place(n, 0), y = place(n, 1), u = place(n, 2), w = place(n, 3);
    return make_float4(acc[x.d][x.r], acc[y.d][y.r], acc[u.d][u.r], acc[w.d][w.r]);
  };
  auto four_dim = [&](int n) {
    if constexpr (kType<DT> != kFp32) return 8 * n + 4 * half;
    else if constexpr (kVec == 4) return n / 16 * 128 + 4 * (8 * (n % 16 / 4) + 4 * half + n % 4);
    else return 2 * (8 * (n / 2) + 4 * half + 2 * (n % 2));
  };
  // The maximum (exp2 domain) that the row's weights are taken from, this lane's share of
  // its sum; its largest score, and the maximum that this one's weight was taken from.
  float m = -INFINITY, z = 0.f, top = -INFINITY, top_at = -INFINITY;

  const int from = it.chunk * cut.each, to = min(from + cut.each, cut.tiles);
  Stage<DT, D, kGroups> stage(a, it.b, it.h, cut.end);
  f32x16 s[kT];  // the scores of the tile at hand
  auto scores = [&](f32x16 (&s)[kT], const char* keys) {
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[i][r] = 0.f;
#pragma unroll
    for (int c = 0; c < kC / 2; ++c)
#pragma unroll
      for (int i = 0; i < kT; ++i)
        s[i] = mfma_rows<DT>(*reinterpret_cast<const u32x4*>(keys + key_at.of(i, c)), q[c], s[i]);
  };
  // -infinity where the tile's slots lie behind what the row sees
  auto mask = [&](f32x16 (&s)[kT], int t0) {
    if (t0 + kTokens - 1 <= wave_first) return;
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (t0 + 32 * i + 8 * (r / 4) + 4 * half + r % 4 > limit) s[i][r] = -INFINITY;
  };
  const bool active = 32 * w < rows;
  if (from < to) {
    stage.ask(from * kTokens);
    const int first_page = stage.page, first_token = stage.token;
    stage.ask(min(from + 1, to - 1) * kTokens);
    const int second_page = stage.page, second_token = stage.token;
    stage.page = first_page, stage.token = first_token;
    stage.move();
    stage.issue_k(keys0);
    stage.page = second_page, stage.token = second_token;
    stage.move();
    stage.finish_k(keys0);
    stage.issue_v(values0);
    stage.issue_k(keys1);
    stage.finish_v(values0);
    stage.finish_k(keys1);
    stage.ask(min(from + 2, to - 1) * kTokens);
    drain();
    stage.move();
    __syncthreads();
    if (active) scores(s, keys0);
    __syncthreads();  // the first keys have been read
  }
  // Step t has the scores of tile t, and in LDS its values and the next tile's keys: the
  // next scores' products run beside this tile's exponentials, and the tile behind
  // them is on its way.
  // In a tile that some row does not see all of, 0 times an infinity or NaN must not reach
  // that row: such values are left out there, and added to the rows that see them at the end.
  bool special = false;
  auto step = [&](int t, char* values, char* next_values, char* next_keys, char* later_keys) {
    const int t0 = t * kTokens;
    if (t0 + kTokens - 1 > tile_first) {
      special |= stage.clean(values);
      __syncthreads();
    }
    if (!kLate && t + 1 < to) {
      stage.issue_v(next_values);
      stage.issue_k(later_keys);  // (the last one again, behind the last)
      stage.ask(min(t + 3, to - 1) * kTokens);
    }
    if (kLate) stage.ask(min(t + 3, to - 1) * kTokens);
    if (kLate && !active) {
      stage.issue_v(next_values);
      stage.issue_k(later_keys);
    }
    if (active) {
      mask(s, t0);
      f32x16 next[kT];
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < kT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, s[i][r]);
      const float peak = fmaxf(most, xor32(most));
      most = peak * a.scale;
      if (__ballot(most > m + kLead<DT>)) {
        const float nm = fmaxf(m, most);
        const float alpha = state_factor(m, nm);
        m = nm;
        z *= alpha;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
      }
      if constexpr (kShared<DT>) {
        top_at = peak > top ? m : top_at;
        top = fmaxf(top, peak);
      }
      float scale = a.scale, shift = m == -INFINITY ? (float)kBias<DT> : (float)kBias<DT> - m;
      // From 2^22 on the maximum's own rounding is 1/8 and more (at 2^32 it takes all of
      // the exponents' range): then the other products are rounded as it was.
      if (__ballot(fabsf(m) >= 0x1p22f && m != -INFINITY)) {
#pragma clang fp contract(off)
#pragma unroll
        for (int i = 0; i < kT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float product = s[i][r] * a.scale;
            s[i][r] = product - (m == -INFINITY ? 0.f : m);
          }
        scale = 1.f;
        shift = (float)kBias<DT>;
      }
      // 2^(..), in place
      auto exponential = [&](int e) {
        float x = __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16], scale, shift));
        // (2^-24, or 0 for 0; in 4 bits no value is infinite.  NaN is left to the sum)
        if constexpr (DT == kFp16) {
          z += x;
          x = __builtin_amdgcn_fmed3f(x, x * 0x1p126f, 0x1p-24f);
        }
        s[e / 16][e % 16] = x;
      };
      // The order of the instructions is this one (the compiler's own has LDS read right
      // before the products that wait for it): the reads are kAhead products ahead, and
      // the exponentials between the first products, the sum between the others.  (The
      // next scores are of no tile, behind the last.  kAhead: by the registers that are left;
      // 4000 rows of head_dim 64 99 us with 3, 92 with 2, of 256 370 and 417, of 128 the same,
      // over 4-bit pages 995 and 953 for 6007 rows.)
      constexpr int kSteps = kC / 2, kAhead = kC == 8 || (kInFour<DT> && D == 128) ? 2 : 3;
      u32x4 kf[kAhead][kT];
      auto read_k = [&](int c) {
#pragma unroll
        for (int i = 0; i < kT; ++i) kf[c % kAhead][i] = *reinterpret_cast<const u32x4*>(next_keys + key_at.of(i, c));
      };
#pragma unroll
      for (int i = 0; i < kT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) next[i][r] = 0.f;
#pragma unroll
      for (int c = 0; c < kAhead - 1; ++c) read_k(c);
      __builtin_amdgcn_sched_barrier(0);
      auto score_step = [&](int c) {
#pragma unroll
        for (int i = 0; i < kT; ++i) next[i] = mfma_rows<DT>(kf[c % kAhead][i], q[c], next[i]);
#pragma unroll
        for (int e = c * 16 * kT / kSteps; e < (c + 1) * 16 * kT / kSteps; ++e) exponential(e);
        if constexpr (kLate) {
          constexpr int kE = Stage<DT, D, kGroups>::kEach;
          constexpr int kPer = (2 * kE + kSteps - 1) / kSteps;
#pragma unroll
          for (int x = c * kPer; x < (c + 1) * kPer; ++x) {
            if (x < kE) stage.issue(stage.v, stage.v_at, next_values, x, x + 1);
            else if (x < 2 * kE) stage.issue(stage.k, stage.k_at, later_keys, x - kE, x - kE + 1);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      if constexpr (kType<DT> == kFp32) {
        // A lane reads kVec dims at once, each for a product of its own (one dim at a time a
        // product takes 87 cycles, not 64: 4097 rows of head_dim 256 then took 1163 us, so 1033)
        const FloatsAt<kC, kVec> floats_at(col, half);
        constexpr int kOf = D / (32 * kVec), kReads = 16 * kT * kOf, kVAhead = 2;
        float vf[kVAhead + 1][kVec];
        auto read_v = [&](int j) {
          const char* from = values + floats_at.of(j / (16 * kOf), j / kOf % 16, j % kOf);
          if constexpr (kVec == 4) {
            const float4 x = *reinterpret_cast<const float4*>(from);
            vf[j % (kVAhead + 1)][0] = x.x, vf[j % (kVAhead + 1)][1] = x.y;
            vf[j % (kVAhead + 1)][2] = x.z, vf[j % (kVAhead + 1)][3] = x.w;
          } else {
            const float2 x = *reinterpret_cast<const float2*>(from);
            vf[j % (kVAhead + 1)][0] = x.x, vf[j % (kVAhead + 1)][1] = x.y;
          }
        };
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          if (c + kAhead - 1 < kSteps) read_k(c + kAhead - 1);
          score_step(c);
        }
#pragma unroll
        for (int j = 0; j < kVAhead; ++j) read_v(j);
#pragma unroll
        for (int j = 0; j < kReads; ++j) {
          if (j + kVAhead < kReads) read_v(j + kVAhead);
          const float p = s[j / (16 * kOf)][j / kOf % 16];
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            acc[j % kOf * kVec + e] =
                __builtin_amdgcn_mfma_f32_32x32x2f32(vf[j % (kVAhead + 1)][e], p, acc[j % kOf * kVec + e], 0, 0, 0);
          if (j % kOf == 0) z += p;
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        constexpr int kCols = D / 32, kPv = 2 * kT * kCols;
        typedef __attribute__((address_space(3))) s16x4* Transposed;
        const ValueAt<kC> value_at(lane);
        u32x4 vf[kAhead + 1], p;
        auto read_v = [&](int j) {
          const int i = j / (2 * kCols), u = j / kCols % 2, d = j % kCols;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Transposed)(values + value_at.of(i, u, 0, d)));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Transposed)(values + value_at.of(i, u, 1, d)));
          const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
          vf[j % (kAhead + 1)] = u32x4{l.x, l.y, h.x, h.y};
        };
        auto pack = [&](int g) {
          const f32x16& x = s[g / 2];
          const int o = 8 * (g & 1);
          p = u32x4{pack2<DT>(x[o], x[o + 1]), pack2<DT>(x[o + 2], x[o + 3]), pack2<DT>(x[o + 4], x[o + 5]),
                    pack2<DT>(x[o + 6], x[o + 7])};
        };
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          if (c + kAhead - 1 < kSteps) read_k(c + kAhead - 1);
          else read_v(c + kAhead - 1 - kSteps);
          score_step(c);
        }
        read_v(kAhead - 1);
#pragma unroll
        for (int j = 0; j < kPv; ++j) {
          if (j % kCols == 0) pack(j / kCols);
          if (j + kAhead < kPv) read_v(j + kAhead);
          acc[j % kCols] = mfma_rows<DT>(vf[j % (kAhead + 1)], p, acc[j % kCols]);
#pragma unroll
          for (int e = 0; e < 8 / kCols; ++e) {
            const int at = j / kCols * 8 + j % kCols * (8 / kCols) + e;
            if constexpr (DT != kFp16) z += s[at / 16][at % 16];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < kT; ++i) s[i] = next[i];
    }
    stage.finish_v(next_values);
    stage.finish_k(later_keys);
    drain();
    stage.move();
    __syncthreads();
  };
  // (each tile has its own array, and the two steps are written out, so that the compiler
  // sees that what is on its way does not meet what is read)
  for (int t = from; t < to; t += 2) {
    step(t, values0, values1, keys1, keys0);
    if (t + 1 < to) step(t + 1, values1, values0, keys0, keys1);
  }
  if (__syncthreads_or(special)) {
#pragma unroll 1
    for (int t = max(from, (tile_first + 1) / kTokens); t < to; ++t) {
      char* values = values0;
      stage.ask(t * kTokens);
      stage.move();
      stage.move();
      __syncthreads();
      stage.issue_v(values);
      stage.finish_v(values);
      drain();
      __syncthreads();
#pragma unroll 1
      for (int k = 0; k < kTokens && t * kTokens + k <= limit; ++k)
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          const int byte = four_dim(n) * kElem<DT>;
          const float4 x = four_of<DT>(values + staged<kC>(k, byte >> 4) + (byte & 15));
          const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[place(n, e).d][place(n, e).r] += fabsf(y[e]) < INFINITY ? 0.f : y[e];
        }
    }
  }
  if (__ballot(stage.bad) && lane == 0) report_error(a.err, error_host_slot(a.err), kErrPages);

  z += xor32(z);
  if constexpr (kShared<DT>) {
    const float share = share_largest<DT>(top, top_at, m, a.scale, z);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= share;
  }
  if (!valid) return;
  if (cut.chunks <= 1) {
    if (a.lse && half == 0) a.lse[row_head] = prompt_lse<DT>(m, z);
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      put_four<DT, D>(a, row_head, four_dim(n), z, four(n));
    return;
  }
  if ((unsigned)it.state >= (unsigned)a.states) return;  // (never, while the offsets ascend)
  float* state = a.state + (size_t)it.state * kStateFloats<D>;
  if (half == 0) {
    state[row] = m;
    state[kTileRows + row] = z;
  }
  float4* products = reinterpret_cast<float4*>(state + 2 * kTileRows);
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
    products[four_dim(n) / 4 * kTileRows + row] = four(n);
}

// Joins the states of tiles whose keys were cut, in the order of their tokens: a
// workgroup for kJoinRows rows of a tile, a thread for a row and four dims.  The factors
// are found by as many lanes as there are chunks, and kU states are in flight a thread.
constexpr int kJoinRows = 8;

template <int DT, int D>
__global__ __launch_bounds__(kJoinRows* D / 4) void prompt_join_kernel(Prompt a) {
  constexpr int kTokens = kTileTokens<DT, D>, kLanes = D / 4, kU = 8;
  __shared__ float factors[kLanes][kJoinRows], parts[kLanes][kJoinRows];
  const PromptPlan plan = prompt_plan<DT, kTokens>(a);
  const int row0 = blockIdx.y * kJoinRows, row = threadIdx.x % kJoinRows, quad = threadIdx.x / kJoinRows;
  PromptItem it;
  for (int tile = blockIdx.x; tile < a.cut_tiles && find_item<kTokens>(a, plan, tile, true, it); tile += gridDim.x) {
    const PromptCut<kTokens> cut(a, it, plan);
    const int rows = it.s.m * a.group - it.tile * kTileRows;
    if (cut.chunks <= 1 || row0 >= rows) continue;  // (a tile of one chunk its workgroup has finished)
    // the states of chunk 0 and from chunk to chunk
    const int first = it.state + (it.s.tiles - 1 - it.tile) * it.most * a.kv_heads + it.h;
    if ((unsigned)first >= (unsigned)a.states || (int64_t)(cut.chunks - 1) * a.kv_heads >= a.states - first)
      continue;  // (never, while the offsets ascend)
    const float* state = a.state + (size_t)first * kStateFloats<D>;
    const size_t step = (size_t)a.kv_heads * kStateFloats<D>;
    const bool valid = row0 + row < rows;
    // (rows behind the tile's have no state: one that has is read in their place)
    const float* own = state + row0 + (valid ? row : 0);
    const float* products = state + 2 * kTileRows + 4 * (quad * kTileRows + row0 + (valid ? row : 0));
    float M = -INFINITY, den = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < cut.chunks; c0 += kLanes) {
      const int count = min(cut.chunks - c0, kLanes);
      float4 x[kU];
      auto load = [&](int c) {
#pragma unroll
        for (int e = 0; e < kU; ++e) x[e] = *reinterpret_cast<const float4*>(products + (size_t)(c0 + min(c + e, count - 1)) * step);
      };
      load(0);
      // the joint maximum so far and what it makes of what was joined before
      __syncthreads();
      factors[quad][row] = quad < count ? own[(c0 + quad) * step] : -INFINITY;
      const float z = quad < count ? own[(c0 + quad) * step + kTileRows] : 0.f;
      __syncthreads();
      float nm = M;
      for (int c = 0; c < count; ++c) nm = fmaxf(nm, factors[c][row]);
      const float before = state_factor(M, nm), f = state_factor(factors[quad][row], nm);
      M = nm;
      __syncthreads();
      factors[quad][row] = f;
      parts[quad][row] = f * z;
      den *= before;
      sum = make_float4(sum.x * before, sum.y * before, sum.z * before, sum.w * before);
      __syncthreads();
      for (int c = 0; c < count; ++c) den += parts[c][row];
      for (int c = 0; c < count; c += kU) {
#pragma unroll
        for (int e = 0; e < kU; ++e)
          if (c + e < count) {
            const float g = factors[c + e][row];
            sum.x = fmaf(g, x[e].x, sum.x);
            sum.y = fmaf(g, x[e].y, sum.y);
            sum.z = fmaf(g, x[e].z, sum.z);
            sum.w = fmaf(g, x[e].w, sum.w);
          }
        if (c + kU < count) load(c + kU);
      }
    }
    if (valid) {
      const int of = it.tile * kTileRows + row0 + row, token = of / a.group;
      const size_t row_head = (size_t)(it.s.first + token) * a.kv_heads * a.group + it.h * a.group + (of - token * a.group);
      if (a.lse && quad == 0) a.lse[row_head] = prompt_lse<DT>(M, den);
      put_four<DT, D>(a, row_head, 4 * quad, den, sum);
    }
  }
}

template <int DT, int D>
int launch_prompt(const Prompt& a, const PromptLayout& l, hipStream_t stream) {
  constexpr int kRow = D * kElem<DT>, kRows = 1024 / kRow;  // of a wave's load
  auto kernel = prompt_kernel<DT, D, !kInFour<DT> && kRows == 1>;
  if constexpr (!kInFour<DT> && kRows > 1)
    if (a.page_size % kRows == 0 && a.slot_units <= (INT32_MAX / 16 - 64) / (kRows - 1)) kernel = prompt_kernel<DT, D, true>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(l.items ? l.items : 1)), dim3(kThreads), 0, stream, a);
  if (const int rc = (int)hipGetLastError()) return rc;
  if (!l.cut_tiles) return 0;
  // (few workgroups, each of every 64th tile: most launches find little to join; with one
  // for each tile that might be cut 1000 rows took 34 us, so 31)
  const unsigned tiles = (unsigned)(l.cut_tiles < 64 ? l.cut_tiles : 64);
  hipLaunchKernelGGL((prompt_join_kernel<DT, D>), dim3(tiles, kTileRows / kJoinRows),
                     dim3(kJoinRows * D / 4), 0, stream, a);
  return (int)hipGetLastError();
}

template <int DT>
int launch_prompt_dim(const Prompt& a, int head_dim, const PromptLayout& l, hipStream_t stream) {
  if (head_dim == 64) return launch_prompt<DT, 64>(a, l, stream);
  if (head_dim == 128) return launch_prompt<DT, 128>(a, l, stream);
  return launch_prompt<DT, 256>(a, l, stream);
}

// Rows times the group are counted in 32 bits, and a launch has fewer than 2^32 threads.
bool prompt_fits(int64_t rows, int sequences, int kv_heads, int group) {
  return rows >= 0 && group >= 1 && group <= 1024 && rows <= (1 << 30) / group &&
         most_tiles(rows, sequences, group) * kv_heads + (1 << kItemsLog) < (1ll << 32) / kThreads;
}

}  // namespace
}  // namespace prismkv

using namespace prismkv;

extern "C" {

size_t prismkv_paged_prompt_work_bytes(int64_t rows, int sequences, int kv_heads, int group, int head_dim, int64_t slots,
                                       int dtype) {
  const bool known = (dtype >= kBf16 && dtype <= kFp32) || dtype == (kFour | kBf16) || dtype == (kFour | kFp16);
  if (!known || sequences < 1 || kv_heads < 1 || head_dim < 1 || slots < 1 || slots > 1 << 30 ||
      !prompt_fits(rows, sequences, kv_heads, group))
    return 0;
  const size_t bytes = prompt_layout(rows, sequences, kv_heads, group, head_dim, slots, element_bytes(dtype) * head_dim,
                                     (dtype & 15) == kFp32).bytes;
  return bytes < 16 ? 16 : bytes;
}

int prismkv_paged_prompt(const prismkv_paged_cache* cache, uint64_t q, uint64_t offsets, uint64_t lse, uint64_t paged_work,
                         uint64_t out, int64_t rows, int group, double scale, size_t work_bytes, uint64_t stream) {
  if (const int rc = check_cache(cache, cache, false)) return rc;
  const prismkv_paged_cache& c = *cache;
  const double scale2 = scale * 1.4426950408889634;  // the exponents are powers of 2, in fp32
  if (!(scale2 >= -FLT_MAX && scale2 <= FLT_MAX) || !prompt_fits(rows, c.sequences, c.kv_heads, group)) return kBadSize;
  if (!offsets && rows != c.sequences) return kBadSize;
  if ((rows && (!q || !out || !paged_work)) || (q | out | paged_work) & 15 || (lse | offsets) & 3) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  const PromptLayout l = prompt_layout(rows, c.sequences, c.kv_heads, group, c.head_dim, slots,
                                       element_bytes(c.dtype) * c.head_dim, (c.dtype & 15) == kFp32);
  if (work_bytes < l.bytes) return kBadSize;
  Prompt a{};
  a.q = reinterpret_cast<const char*>(q);
  a.k = reinterpret_cast<const char*>(c.k);
  a.v = reinterpret_cast<const char*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.lengths = reinterpret_cast<const int32_t*>(c.lengths);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
  a.out = reinterpret_cast<char*>(out);
  a.lse = reinterpret_cast<float*>(lse);
  a.state = reinterpret_cast<float*>(paged_work);
  a.err = reinterpret_cast<unsigned*>(c.err);
  const int64_t es = page_element_bytes(c.dtype);
  a.page_units = (unsigned)(c.page_stride * es >> 4);
  a.head_bytes = c.head_stride * es;
  a.slot_units = (unsigned)(c.slot_stride * es >> 4);
  a.scale = (float)(scale2 < 0 ? -scale2 : scale2);
  a.q_and = scale2 == 0 ? 0u : ~0u;
  a.q_xor = !(scale2 < 0) ? 0u : element_bytes(c.dtype) == 4 ? 0x80000000u : 0x80008000u;
  if (scale2 == 0) a.scale = 1.f;  // (of scores that are 0)
  if (c.dtype >= kFour) {
    a.ks = reinterpret_cast<const uint8_t*>(c.k_scales);
    a.vs = reinterpret_cast<const uint8_t*>(c.v_scales);
    a.scale_page_units = (unsigned)(c.scale_page_stride / (c.head_dim / 32));
    a.scale_head = c.scale_head_stride;
    a.scale_slot_units = (unsigned)(c.scale_slot_stride / (c.head_dim / 32));
  }
  a.div = page_div(c.page_size);
  a.rows = (int)rows;
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  a.group = group;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = (int)slots;
  a.states = (int)l.states, a.cut_tiles = (int)l.cut_tiles;
  const hipStream_t s = (hipStream_t)stream;
  switch (c.dtype) {
    case kBf16: return launch_prompt_dim<kBf16>(a, c.head_dim, l, s);
    case kFp16: return launch_prompt_dim<kFp16>(a, c.head_dim, l, s);
    case kFp32: return launch_prompt_dim<kFp32>(a, c.head_dim, l, s);
    case kFour | kBf16: return launch_prompt_dim<kFour | kBf16>(a, c.head_dim, l, s);
    default: return launch_prompt_dim<kFour | kFp16>(a, c.head_dim, l, s);
  }
}

}  // extern "C"
