// Arguments and device helpers of the paged cache's kernels (paged.hip).
#pragma once

#include "attend_core.h"

namespace prismkv {
namespace {

constexpr int kPT = 256;  // threads of the paged kernels but the selection
constexpr int kPWaves = kPT / 64;
constexpr unsigned kErrPages = 4u;  // error word: a slot within a sequence's length has no page of the cache

// Element types of the C ABI (`dtype`).
constexpr int kBf16 = 0, kFp16 = 1, kFp32 = 2;
template <int DT>
constexpr int kElem = DT == kFp32 ? 4 : 2;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// t / page_size of 0 <= t < 2^31 by one product (shift = 31 + ceil(log2 page_size),
// mul = ceil(2^shift / page_size) < 2^32: exact over that range).
struct PageDiv {
  unsigned mul;
  int shift;
  __device__ __forceinline__ int of(int t) const { return (int)(((unsigned long long)(unsigned)t * mul) >> shift); }
};

// Chunks that the attention aims at: two workgroups of 4 waves on each of the
// 256 CUs.  The grid has room for one more per (sequence, head tile), so that
// rounding up never runs out of it.
constexpr int kLogUnits = 9;

struct PagedAttend {
  const void *q, *k, *v;
  const int32_t *table, *lengths;
  const float* scores;  // weigh: the scores read and written, or null
  float *scores_out, *lse_out;
  void* out;
  float *logits, *lse_work, *state;  // workspace: weigh's scores in the exp2 domain and their log-sums; chunk states
  unsigned *counters, *err;
  int64_t head_bytes, logit_stride, slots;
  unsigned page_units, slot_units, state_stride;  // 16-byte units; floats per chunk state
  PageDiv div;
  int sequences, kv_heads, group, tiles, page_size, max_pages, pages;
  float scale;  // log2(e) times the caller's
};

__device__ __forceinline__ int clamp_length(const PagedAttend& a, int n) { return min(max(n, 0), (int)a.slots); }

// A workgroup's share: chunk `chunk` of `chunks` of sequence b's n tokens, `per`
// tokens each (a multiple of 32), for head tile hh; b < 0: none.
struct PagedUnit {
  int b, hh, n, chunk, chunks, per;
};

// Every wave finds its workgroup's share by itself (uniform; one load of the
// lengths and a lane scan for up to 64 sequences): chunks of about
// total / 2^kLogUnits tokens, so a long sequence among short ones is spread
// over as many workgroups as its share of the work.
__device__ __forceinline__ PagedUnit find_unit(const PagedAttend& a, int unit) {
  const int lane = threadIdx.x & 63;
  const int heads = a.kv_heads * a.tiles;
  int first = 0;  // the lengths of the first 64 sequences
  unsigned long long total = 0;
  for (int i0 = 0; i0 < a.sequences; i0 += 64) {
    const int n = i0 + lane < a.sequences ? clamp_length(a, a.lengths[i0 + lane]) : 0;
    if (i0 == 0) first = n;
    total += (unsigned)wave_sum_i(n);
  }
  const unsigned chunk = max((unsigned)((total * heads + (1u << kLogUnits) - 1) >> kLogUnits), 32u * kPWaves);
  PagedUnit u;
  u.b = -1;
  const int at = unit / heads;
  u.hh = unit - at * heads;
  int base = 0;
  for (int i0 = 0; i0 < a.sequences; i0 += 64) {
    int n = first;
    if (i0) n = i0 + lane < a.sequences ? clamp_length(a, a.lengths[i0 + lane]) : 0;
    const int c = i0 + lane < a.sequences ? max((int)(((unsigned)n + chunk - 1) / chunk), 1) : 0;
    const int incl = (int)wave_incl_scan((unsigned)c);
    const int sum = __builtin_amdgcn_readlane(incl, 63);
    if (at - base < sum) {
      const int l = __ffsll((unsigned long long)__ballot(incl > at - base)) - 1;
      u.b = i0 + l;
      u.n = __builtin_amdgcn_readlane(n, l);
      u.chunks = __builtin_amdgcn_readlane(c, l);
      u.chunk = at - base - (__builtin_amdgcn_readlane(incl, l) - u.chunks);
      u.per = (u.n + u.chunks - 1) / u.chunks;
      u.per = (u.per + 31) & ~31;
      return u;
    }
    base += sum;
  }
  return u;
}

// Writes output element i (query head i / D of the tile, dim i % D) from the
// joined maximum, sum and product; no weight at all (an empty sequence) gives 0.
template <int DT, int D>
__device__ __forceinline__ void finish(const PagedAttend& a, size_t head0, int i, float M, float den, float x) {
  const float y = den == 0.f ? 0.f : x / den;
  const size_t at = head0 * D + i;
  if constexpr (DT == kBf16) reinterpret_cast<uint16_t*>(a.out)[at] = f32_to_bf16(y);
  else if constexpr (DT == kFp16) reinterpret_cast<_Float16*>(a.out)[at] = (_Float16)y;
  else reinterpret_cast<float*>(a.out)[at] = y;
  if (i % D == 0) {
    const float l2 = den == 0.f ? -INFINITY : M + log2f(den) - (DT == kFp16 ? 15.f : 0.f);
    if (a.lse_out) a.lse_out[head0 + i / D] = l2 * 0.693147180559945309f;
    if (a.lse_work) a.lse_work[head0 + i / D] = l2;
  }
}

struct PagedAppend {
  const char *k, *v;
  char *kp, *vp;
  const int32_t *table, *offsets, *lengths, *seen;
  int32_t *lengths_out, *seen_out, *positions, *positions_out;
  float *scores, *scores_out;
  unsigned* err;
  int64_t rows, k_row, k_head, v_row, v_head;  // bytes
  int64_t page_bytes, head_bytes, slot_bytes;
  PageDiv div;
  int sequences, kv_heads, row_bytes, page_size, max_pages, pages, slots;
};

struct PagedEvict {
  char *kp, *vp;
  const int32_t *table, *lengths, *seen, *positions, *keeps;
  const float* scores;
  int32_t *lengths_out, *seen_out, *positions_out;
  float* scores_out;
  int32_t *count, *src, *dst;  // workspace: moves per (sequence, KV head)
  unsigned* err;
  int64_t page_bytes, head_bytes, slot_bytes, moves;
  PageDiv div;
  int sequences, kv_heads, row_bytes, page_size, max_pages, pages, slots, keep, recent, sinks;
  bool guard;  // some positions are protected
};

}  // namespace
}  // namespace prismkv
