// Arguments and device helpers of the paged cache's kernels (paged.hip).
#pragma once

#include "attend_core.h"

namespace prismkv {

// t / page_size of 0 <= t < 2^31 by one product (shift = 31 + ceil(log2 page_size),
// mul = ceil(2^shift / page_size) < 2^32: exact over that range).
struct PageDiv {
  unsigned mul;
  int shift;
  __device__ __forceinline__ int of(int t) const { return (int)(((unsigned long long)(unsigned)t * mul) >> shift); }
};

struct PagedAttend {
  const void *q, *k, *v;
  const int32_t *table, *lengths;
  const float* scores;  // weigh: the scores read and written, or null
  float *scores_out, *lse_out;
  void* out;
  float *logits, *state;  // workspace: unscaled scores (to be weighed), partial states
  float2* sums_work;      // workspace: each softmax's maximum and its sum's reciprocal (to be weighed)
  unsigned *counters, *err;          // counters: null where a second launch joins the states
  int64_t head_bytes, logit_stride, slots;
  unsigned page_units, slot_units, state_stride;  // 16-byte units; floats per partial state
  PageDiv div;
  int sequences, kv_heads, group, tiles, page_size, max_pages, pages;
  float scale;  // log2(e) times the caller's; in 4 bits its magnitude
  // pages in 4 bits: the scales' pages, their strides in bytes; the sign of `scale`, or
  // that it is 0, as bits of the queries
  unsigned q_and, q_xor;
  const uint8_t *k_scales, *v_scales;
  int64_t scale_page, scale_head;
  unsigned scale_slot;
  bool many;    // kSoloPairs pairs or more
};

// The attention over pages in 4 bits (defined in paged4.hip).
int attend_in_four(const PagedAttend& a, int dtype, int head_dim, int64_t units, hipStream_t stream);

namespace {

constexpr int kPT = 256;  // threads of the paged kernels but the selection
// Error word: a slot within a sequence's length has no page of the cache; an append's
// offsets do not cover its rows; the offsets of a prompt or a read do not cover its
// rows; they ask for more rows than a sequence holds.
constexpr unsigned kErrPages = 4u, kErrRows = 8u, kErrOffsets = 16u, kErrHeld = 32u;

// Element types of the C ABI (`dtype`): of the rows that go in and out and, unless
// kFour is added (pages in 4 bits), of the pages.
constexpr int kBf16 = 0, kFp16 = 1, kFp32 = 2, kFour = 16;
template <int DT>
constexpr int kType = DT & 15;
template <int DT>
constexpr bool kInFour = DT >= kFour;
template <int DT>
constexpr int kElem = kType<DT> == kFp32 ? 4 : 2;
// P is held times 2^kBias: fp16 probabilities from 2^-29 of the maximum up stay
// normal numbers (bf16 and fp32 have the exponents for them).
template <int DT>
constexpr int kBias = kType<DT> == kFp16 ? 15 : 0;
// Exponents of the scales in 4 bits, plus 127: those whose codes are all exact numbers
// of the type, for fp16 2^-23 (of half of which its least number is) to 2^13 (6 times
// which is its last), for bf16 what its normal numbers allow.
template <int DT>
constexpr int kLeastScale = kType<DT> == kFp16 ? 104 : 2;
template <int DT>
constexpr int kMostScale = kType<DT> == kFp16 ? 140 : 252;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight codes, the lowest four bits first, times the scale as pairs of the 16-bit type
// (NaN for an infinite scale, whose byte is 255).
template <int DT>
__device__ __forceinline__ u32x4 widen8(unsigned codes, float scale) {
  if constexpr (kType<DT> == kBf16)
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
  else
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3))};
}

// Workgroups that the attention's rows are dealt to: one on each of the 256 CUs,
// of 8 waves (two a SIMD, each with a tile in flight), or of 4 where a tile of
// head_dim 256 takes the registers of two.  Two workgroups of 4 waves read as fast,
// but leave twice the partial states to join (64K: 54.0 us against 47.8).
constexpr int kUnits = 256;
template <int D>
constexpr int kAWaves = D == 256 ? 4 : 8;
constexpr int kQuantum = 32;  // tokens that are dealt at a time
// Quanta of a workgroup at least: a tile (32 tokens, fp32 16) for each wave.
template <int DT, int D>
constexpr int kLeast = kType<DT> == kFp32 ? kAWaves<D> / 2 : kAWaves<D>;

// 16 bytes that another workgroup wrote through (agent scope, as ld_dev).
__device__ __forceinline__ float4 ld_dev4(__amdgpu_buffer_rsrc_t r, unsigned byte_offset) {
  const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, byte_offset, 0, 16);
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}

__device__ __forceinline__ int clamp_length(const PagedAttend& a, int n) { return min(max(n, 0), (int)a.slots); }

// Quanta of a pair of n tokens: whole workgroups' worths (so that short pairs are
// not cut for their neighbours' sake), one for an empty sequence's output.
template <int kL>
__device__ __host__ __forceinline__ int quanta_of(int n) {
  return n > 0 ? (n + kL * kQuantum - 1) / (kL * kQuantum) * kL : kL;
}

// How the quanta of all pairs (sequence, head tile), pair after pair, are dealt:
// evenly to kUnits workgroups, or kLeast each while there are fewer.  The shares
// differ by one quantum at most, and no CU gets a second workgroup after its
// first (65792 tokens of 8 heads: 66 us with 514 workgroups for 512 places, 54
// with 512).
template <int kL>
struct PagedDeal {
  int total;
  __device__ __forceinline__ int begin(int unit) const {
    if (total <= kUnits * kL) return min(unit * kL, total);
    return (int)((unsigned long long)unit * (unsigned)total / kUnits);
  }
  // the workgroup whose share holds quantum x
  __device__ __forceinline__ int unit_of(int x) const {
    if (total <= kUnits * kL) return x / kL;
    int u = min((int)((float)(x + 1) * kUnits / (float)total), kUnits - 1);  // off by one at most
    while (begin(u) > x) --u;
    while (begin(u + 1) <= x) ++u;
    return u;
  }
};

// A pair's quanta [from, from + quanta) lie in the shares of `chunks` workgroups
// from `unit` on.  A workgroup has at most two partial states: slot 2 unit of the
// pair that its first quantum lies in, slot 2 unit + 1 of the one that its share
// ends in; so the pair's state 0 lies `odd` slots behind slot 2 unit, state c 2c.
struct PagedParts {
  int unit, chunks, odd;
  template <int kL>
  __device__ __forceinline__ PagedParts(const PagedDeal<kL>& deal, int from, int quanta)
      : unit(deal.unit_of(from)), chunks(deal.unit_of(from + quanta - 1) - unit + 1), odd(deal.begin(unit) != from) {}
};

// A workgroup's share: quanta [at, end), of which the first is `first` of pair
// (b, hh) with n tokens.
template <int kL>
struct PagedSpan {
  PagedDeal<kL> deal;
  int at, end, b, hh, n, first;
  bool alone;  // a wave for each pair instead
};

// Quanta of the first `count` sequences, for one KV head and head tile; `longest`
// is raised to their longest.
template <int kL>
__device__ __forceinline__ int quanta_before(const PagedAttend& a, int count, int& longest) {
  int sum = 0, most = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < count; i += 64) {
    const int n = clamp_length(a, a.lengths[i]);
    sum += quanta_of<kL>(n);
    most = max(most, n);
  }
  most = (int)wave_max((float)min(most, 1 << 20));  // (exact as far as it matters)
  longest = max(longest, most);
  return wave_sum_i(sum);
}

// Many short pairs: a wave for each by itself, where a workgroup for each would
// take them one after another and leave most of its waves without a tile (256
// sequences of 100 tokens, 8 heads: 23.7 us, 42.9 by workgroups; 128 of 500 44.5
// and 51.8).  Fewer pairs are faster by workgroups (256 of 250 tokens 11.4 us against
// 13.9), longer ones as fast or, ragged, faster: 512 of 1000 tokens 47 us against 45,
// 512 ragged up to 1000 27.6 against 34.5.
constexpr int kSoloTokens = 512, kSoloPairs = 512;
__device__ __forceinline__ bool pairs_alone(const PagedAttend& a, int longest) {
  return a.many && longest <= kSoloTokens;
}

// Every wave finds its workgroup's share by itself (uniform; two loads of the
// lengths and a lane scan for every 64 sequences), so that a long sequence among
// short ones is spread over as many workgroups as its share of the rows.
template <int kL, bool kMany>
__device__ __forceinline__ PagedSpan<kL> find_span(const PagedAttend& a, int unit) {
  const int lane = threadIdx.x & 63, heads = a.kv_heads * a.tiles;
  auto length = [&](int i) { return i < a.sequences ? clamp_length(a, a.lengths[i]) : 0; };
  int n = length(lane), longest = 0;
  PagedSpan<kL> u;
  u.deal.total = quanta_before<kL>(a, a.sequences, longest) * heads;
  u.alone = kMany && pairs_alone(a, longest);
  u.at = u.deal.begin(unit);
  u.end = u.deal.begin(unit + 1);
  if (u.alone || u.at >= u.end) return u;
  const int to = u.at / heads;  // (a sequence's quanta begin at a multiple of heads)
  int base = 0;
  for (int i = 0;; i += 64) {  // (`to` lies in some sequence)
    const int next = length(i + 64 + lane);
    const int c = i + lane < a.sequences ? quanta_of<kL>(n) : 0;
    const int incl = (int)wave_incl_scan((unsigned)c);
    const int sum = __builtin_amdgcn_readlane(incl, 63);
    if (to - base < sum || i + 64 >= a.sequences) {
      const int l = max(__ffsll((unsigned long long)__ballot(incl > to - base)) - 1, 0);
      const int own = __builtin_amdgcn_readlane(c, l);
      const int in = u.at - (base + __builtin_amdgcn_readlane(incl, l) - own) * heads;  // within the sequence
      u.b = i + l;
      u.n = __builtin_amdgcn_readlane(n, l);
      u.hh = in / own;
      u.first = in - u.hh * own;
      return u;
    }
    base += sum;
    n = next;
  }
}

// log2 of a softmax's sum from its maximum and the sum held times 2^kBias.
template <int DT>
__device__ __forceinline__ float log_sum(float M, float den) {
  return den == 0.f ? -INFINITY : M + (log2f(den) - kBias<DT>);
}

// Writes output element i (query head i / D of the tile, dim i % D) from the
// joined maximum, sum and product; no weight at all (an empty sequence) gives 0.
template <int DT, int D>
__device__ __forceinline__ void finish(const PagedAttend& a, size_t head0, int i, float M, float den, float x) {
  const float y = den == 0.f ? 0.f : x / den;
  const size_t at = head0 * D + i;
  if constexpr (kType<DT> == kBf16) reinterpret_cast<uint16_t*>(a.out)[at] = f32_to_bf16(y);
  else if constexpr (kType<DT> == kFp16) reinterpret_cast<_Float16*>(a.out)[at] = (_Float16)y;
  else reinterpret_cast<float*>(a.out)[at] = y;
  if (i % D == 0) {
    if (a.lse_out) a.lse_out[head0 + i / D] = log_sum<DT>(M, den) * 0.693147180559945309f;
    if (a.sums_work)
      a.sums_work[head0 + i / D] =
          den == 0.f ? make_float2(0.f, 0.f) : make_float2(M, (float)(1 << kBias<DT>) / den);
  }
}

struct PagedAppend {
  const char *k, *v;
  char *kp, *vp;
  const int32_t *table, *offsets, *lengths, *seen;
  int32_t *lengths_out, *seen_out, *positions, *positions_out;
  float *scores, *scores_out;
  unsigned* err;
  int64_t first_row, rows;                     // this launch's first, all
  int64_t k_row, k_head, v_row, v_head;        // bytes
  int64_t page_bytes, head_bytes, slot_bytes;
  PageDiv div;
  int sequences, kv_heads, log_pieces, page_size, max_pages, pages, slots;  // log_pieces: 16-byte pieces of a row
};

struct PagedEvict {
  char *kp, *vp;
  const int32_t *table, *lengths, *seen, *positions, *keeps;
  const float* scores;
  int32_t *lengths_out, *seen_out, *positions_out;
  float* scores_out;
  int32_t *count, *src, *dst;  // workspace: moves per (sequence, KV head)
  unsigned *counters, *tables, *err;
  int64_t table_words;  // of a row
  int64_t page_bytes, head_bytes, slot_bytes, moves;
  PageDiv div;
  int sequences, kv_heads, log_pieces, page_size, max_pages, pages, slots, keep, recent, sinks, part, most_parts;
  char *k_scales, *v_scales;  // of pages in 4 bits: a row's scale_bytes (else 0)
  int64_t scale_page, scale_head, scale_slot;
  int scale_bytes;
};

}  // namespace
}  // namespace prismkv
