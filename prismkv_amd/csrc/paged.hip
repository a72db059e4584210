// The paged key-value cache: writing rows into pages, attention of one new
// query token of every sequence over its pages, and eviction by accumulated
// attention weight.
//
// K and V pages are [pages][kv_heads][page_size][head_dim] with any strides of
// 16-byte multiples (the same for both); slot t of sequence b lies in page
// table[b][t / page_size].  A table entry outside [0, pages) within a
// sequence's length is reported through the cache's error word and never read
// through.
#include "paged_attend.h"
#include "paged_host.h"

#include <cfloat>


namespace prismkv {
namespace {

// scores_out[t] = scores[t] + sum over the group's heads of its weight, from their
// maxima and sums as the attention had them (a log-sum's rounding, 2^-24 of it, would
// be the weights' error: 4e-4 at scores of 2e4): a thread per slot; bound by the scores that it reads (4 bytes per query head and
// slot) and the two score arrays.
__global__ __launch_bounds__(kPT) void paged_weigh_kernel(PagedAttend a) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = clamp_length(a, a.lengths[b]);
  const float2* sums = a.sums_work + ((size_t)b * a.kv_heads + h) * a.group;
  const float* logits = a.logits + ((size_t)b * a.kv_heads + h) * a.group * a.logit_stride;
  const size_t at = ((size_t)b * a.kv_heads + h) * a.slots;
  for (int t = blockIdx.x * kPT + threadIdx.x; t < n; t += gridDim.x * kPT) {
    const float before = a.scores[at + t];
    float sum = 0.f;
    for (int g0 = 0; g0 < a.group; g0 += 4) {  // (four heads' loads together)
      float s[4];
      float2 z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int g = min(g0 + e, a.group - 1);
        s[e] = logits[(size_t)g * a.logit_stride + t];
        z[e] = sums[g];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (g0 + e < a.group) sum = fmaf(weight(s[e], a.scale, z[e].x), z[e].y, sum);
    }
    a.scores_out[at + t] = before + sum;
  }
}

// ------------------------------------------------------------------ append
//
// A copy of rows: bound by reading and writing them.  A workgroup finds the places
// of its rows (one of a sequence each, or kAppendRows packed ones) with a thread
// per row, then copies them with 16 bytes per thread, kU loads each of K and V in
// flight.  20011 rows of 8 heads and 128 dims in bf16 (164 MB read and written):
// 31.7 us = 5.2 TB/s (a copy as large: 32.2); 128 single rows 3.5 us.

constexpr int kAppendRows = 8;
constexpr int64_t kLaunchRows = 1 << 26;  // (a launch has fewer than 2^32 threads: 2^27 rows)

struct AppendPlace {
  size_t at;  // bytes from the pages' base
  int b, slot, position, length;  // slot -1: a row that is dropped; length: of its sequence before
};

__device__ __forceinline__ AppendPlace append_place(const PagedAppend& a, int64_t row) {
  AppendPlace p{0, 0, -1, 0, 0};
  int64_t step = 0;
  if (!a.offsets) {
    p.b = (int)row;
  } else {  // the last b with offsets[b] <= row
    int lo = 0, hi = a.sequences;
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.offsets[mid] <= row) lo = mid;
      else hi = mid;
    }
    p.b = lo;
    step = row - a.offsets[lo];
    if (step < 0 || row >= a.offsets[lo + 1]) return p;  // a row of no sequence
  }
  p.length = min(max(a.lengths[p.b], 0), a.slots);
  if (a.positions) p.position = a.seen[p.b] + (int)step;
  const int64_t slot = p.length + step;
  const int page = slot < a.slots ? a.table[(size_t)p.b * a.max_pages + a.div.of((int)slot)] : -1;
  if ((unsigned)page >= (unsigned)a.pages) {  // no page: the row is dropped
    report_error(a.err, error_host_slot(a.err), kErrPages);
    return p;
  }
  p.slot = (int)slot;
  p.at = (size_t)page * a.page_bytes + (size_t)(p.slot - a.div.of(p.slot) * a.page_size) * a.slot_bytes;
  return p;
}

// lengths and tokens seen of sequence b with its packed rows; offsets that do not
// cover the rows, ascending from 0, are reported
__device__ __forceinline__ void advance(const PagedAppend& a, int b) {
  const int from = a.offsets[b], to = a.offsets[b + 1], more = max(to - from, 0);
  if (from > to || (b == 0 && from) || (b == a.sequences - 1 && to != a.rows))
    report_error(a.err, error_host_slot(a.err), kErrRows);
  a.lengths_out[b] = (int)min((int64_t)max(a.lengths[b], 0) + more, (int64_t)a.slots);
  if (a.positions) a.seen_out[b] = a.seen[b] + more;
}

__global__ __launch_bounds__(kPT) void paged_append_kernel(PagedAppend a) {
  __shared__ AppendPlace places[kAppendRows];
  const int tid = threadIdx.x, each = a.offsets ? kAppendRows : 1;
  const int64_t row0 = a.first_row + (int64_t)blockIdx.x * each;
  const int rows = (int)min((int64_t)each, a.rows - row0);
  const int log = a.log_pieces, per_row = a.kv_heads << log, items = rows * per_row;  // pieces of 16 bytes
  constexpr int kU = 4;
  uint4 kv[kU], vv[kU];
  // piece i: its row, and its bytes from the row's first
  auto piece = [&](int i, int& r, int& h, int& c) {
    r = i / per_row;
    h = (i - r * per_row) >> log;
    c = (i & ((1 << log) - 1)) << 4;
  };
  auto load = [&](int i0) {
#pragma unroll
    for (int e = 0; e < kU; ++e) {
      if (i0 - tid + e * kPT >= items) break;
      int r, h, c;
      piece(min(i0 + e * kPT, items - 1), r, h, c);
      kv[e] = load_nt16(a.k + (row0 + r) * a.k_row + (int64_t)h * a.k_head + c);
      vv[e] = load_nt16(a.v + (row0 + r) * a.v_row + (int64_t)h * a.v_head + c);
    }
    asm volatile("" ::: "memory");  // (all of them are asked for before anything is stored)
  };
  load(tid);
  if (tid < rows) places[tid] = append_place(a, row0 + tid);
  __syncthreads();
  for (int i0 = tid; i0 < items;) {
#pragma unroll
    for (int e = 0; e < kU; ++e) {
      if (i0 + e * kPT >= items) break;
      int r, h, c;
      piece(i0 + e * kPT, r, h, c);
      const AppendPlace& p = places[r];
      if (p.slot >= 0) {
        const size_t at = p.at + (size_t)h * a.head_bytes + c;
        *reinterpret_cast<uint4*>(a.kp + at) = kv[e];
        *reinterpret_cast<uint4*>(a.vp + at) = vv[e];
      }
    }
    i0 += kU * kPT;
    if (i0 < items) load(i0);
  }
  if (a.positions)
    for (int i = tid; i < rows * a.kv_heads; i += kPT) {
      const AppendPlace& p = places[i / a.kv_heads];
      if (p.slot < 0) continue;
      const size_t at = ((size_t)p.b * a.kv_heads + i % a.kv_heads) * a.slots + p.slot;
      a.scores[at] = a.scores_out[at] = 0.f;
      a.positions[at] = a.positions_out[at] = p.position;
    }
  if (!a.offsets) {  // (the row's workgroup alone reads its sequence's length)
    if (tid == 0) {
      a.lengths_out[blockIdx.x] = min(places[0].length + 1, a.slots);
      if (a.positions) a.seen_out[blockIdx.x] = places[0].position + 1;
    }
  } else if (a.lengths_out != a.lengths) {
    for (int64_t b = (int64_t)blockIdx.x * kPT + tid; b < a.sequences; b += (int64_t)gridDim.x * kPT)
      advance(a, (int)b);
  }
}

// Packed rows onto lengths that are advanced in place: after every workgroup has read them.
__global__ __launch_bounds__(kPT) void paged_advance_kernel(PagedAppend a) {
  const int b = blockIdx.x * kPT + threadIdx.x;
  if (b < a.sequences) advance(a, b);
}

// ------------------------------------------------------------------ eviction

// The order of the scores as an unsigned key: NaN above the numbers, -0 as 0; above
// them all 0xffffffff, a protected slot's.
__device__ __forceinline__ unsigned evict_key(float score) {
  const unsigned u = __float_as_uint(score + 0.f);
  const unsigned key = u ^ (unsigned)((int)u >> 31 | (int)0x80000000);
  return score != score ? 0xfffffffeu : key;
}

__device__ __forceinline__ int evict_keep(const PagedEvict& a, int b) {
  const int keep = a.keeps ? a.keeps[b] : a.keep;
  return max(keep, 0);
}

constexpr int kET = 1024, kEWaves = kET / 64;  // threads and waves of the selection
constexpr int kFew = 256;                      // moves that the selection makes by itself

struct EvictRow {
  int n, m, edge;  // length, slots that stay, first position that is among the newest
  size_t row;
  const float* scores;
  const int32_t* positions;
  bool copy;  // the fork gets what stays where it is (the moves overwrite the holes)
  // sizes: {n, m} where the sequence's length may be written meanwhile
  __device__ __forceinline__ EvictRow(const PagedEvict& a, int b, int h, const unsigned* sizes = nullptr) {
    n = __builtin_amdgcn_readfirstlane(sizes ? (int)sizes[0] : min(max(a.lengths[b], 0), a.slots));
    m = __builtin_amdgcn_readfirstlane(sizes ? (int)sizes[1] : min(n, evict_keep(a, b)));
    edge = max(a.seen[b] - a.recent, a.sinks);
    row = (size_t)b * a.kv_heads + h;
    scores = a.scores + row * a.slots;
    positions = a.positions + row * a.slots;
    copy = a.scores_out != a.scores;
  }
};

// Scores and positions of kU x 64 slots from t0 on, asked for together; then their
// keys, 0 at and behind `last`.
template <int kU>
struct EvictSlots {
  float score[kU];
  int position[kU];
  __device__ __forceinline__ void load(const EvictRow& r, int t0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int t = min(t0 + 64 * u + lane, r.n - 1);
      score[u] = r.scores[t];
      position[u] = r.positions[t];
    }
    asm volatile("" ::: "memory");
  }
  __device__ __forceinline__ void keys(const PagedEvict& a, const EvictRow& r, int t0, int last, bool copy,
                                       unsigned (&key)[kU]) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int t = t0 + 64 * u + lane;
      // (position < sinks or >= edge as one comparison, edge >= sinks)
      const bool held = (unsigned)(position[u] - a.sinks) >= (unsigned)(r.edge - a.sinks);
      key[u] = t >= last ? 0u : held ? 0xffffffffu : evict_key(score[u]);
      if (copy && t < min(last, r.m)) {
        a.scores_out[r.row * a.slots + t] = score[u];
        a.positions_out[r.row * a.slots + t] = position[u];
      }
    }
  }
};

// The digits of a key from the top.  (No key has the first digit 0, where slots
// that are none are counted.)
template <int kPass>
__device__ __forceinline__ unsigned digit(unsigned key) {
  return kPass == 0 ? key >> 21 : kPass == 1 ? (key >> 10) & 2047u : key & 1023u;
}
// Whether the digits before this pass's are those found, `prefix`.
template <int kPass>
__device__ __forceinline__ bool matches(unsigned key, unsigned prefix) {
  return kPass == 0 || (kPass == 1 ? key >> 21 : key >> 10) == prefix;
}

// The digit of the need-th largest key, given the counts of digits 2047 - 2i (x) and
// 2046 - 2i (y) in thread i: appended to `prefix`, and `need` among its keys.
template <int kPass>
__device__ __forceinline__ void find_digit(unsigned x, unsigned y, unsigned* wsum, unsigned* found, unsigned& prefix,
                                           unsigned& need) {
  const int tid = threadIdx.x;
  const unsigned before = block_incl_scan<kET>(x + y, wsum) - x - y;
  if (before < need && need <= before + x + y) {
    const bool upper = need <= before + x;
    found[0] = 2047 - 2 * tid - !upper;
    found[1] = need - before - (upper ? 0u : x);
  }
  __syncthreads();
  prefix = prefix << (kPass < 2 ? 11 : 10) | __builtin_amdgcn_readfirstlane(found[0]);
  need = __builtin_amdgcn_readfirstlane(found[1]);
}

// Lanes of 64 slots from t0 that lie before slot m.
__device__ __forceinline__ unsigned long long lanes_before(int m, int t0) {
  const int n = m - t0;
  return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull;
}

// Counts of a share of the slots: evicted before the budget and kept behind it if no
// key equal to the bound stays, and such keys before and behind it.
struct EvictCounts {
  int hole, source, front, back;
  // the holes and sources where `room` of the keys equal to the bound stay, the lowest
  __device__ __forceinline__ int holes(int room) const { return hole - min(max(room, 0), front); }
  __device__ __forceinline__ int sources(int room) const { return source + min(max(room - front, 0), back); }
};

// The counts of the wave's share given by each_key (f(t0, key): 64 slots from t0,
// ascending).
template <typename E>
__device__ __forceinline__ EvictCounts count_moves(E each_key, unsigned bound, int m, int last) {
  EvictCounts c{0, 0, 0, 0};
  each_key([&](int t0, unsigned key) {
    const unsigned long long above = __ballot(key > bound), eq = __ballot(key == bound), front = lanes_before(m, t0);
    c.hole += __popcll(~above & front & lanes_before(last, t0));
    c.source += __popcll(above & ~front);
    c.front += __popcll(eq & front);
    c.back += __popcll(eq & ~front);
  });
  return c;
}

// Appends the slots t0 + (lanes of mask), ascending.
__device__ __forceinline__ void put_slots(int32_t*& to, int t0, unsigned long long mask) {
  if (!mask) return;
  const int lane = threadIdx.x & 63;
  if (mask >> lane & 1)
    to[__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u))] = t0 + lane;
  to += __popcll(mask);
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ int block_sum(int v, int* lds) {
  v = wave_sum_i(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int k = 0; k < kEWaves; ++k) total += lds[k];
  return __builtin_amdgcn_readfirstlane(total);
}

// Writes the wave's holes and sources (each_key as above, its counts `mine`) behind
// those of the waves before it, to dst and src, which begin with the workgroup's;
// `room` of the workgroup's keys equal to the bound stay.  Returns the workgroup's
// number of holes; where it is `few` at most they go to few_dst and few_src.
template <typename E>
__device__ __forceinline__ int write_moves(E each_key, const EvictCounts& mine, unsigned bound, int room, int m, int last,
                                           int32_t* dst, int32_t* src, EvictCounts* counts, int few, int32_t* few_dst,
                                           int32_t* few_src) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((threadIdx.x & 63) == 0) counts[w] = mine;
  __syncthreads();
  int hole = 0, source = 0, total = 0, own = 0, left = room;  // room left for the wave's own
#pragma unroll
  for (int k = 0; k < kEWaves; ++k) {
    const EvictCounts c = counts[k];
    if (k == w) own = left;
    const int holes = c.holes(left);
    hole += k < w ? holes : 0;
    source += k < w ? c.sources(left) : 0;
    total += holes;
    left -= c.front + c.back;
  }
  total = __builtin_amdgcn_readfirstlane(total);
  own = __builtin_amdgcn_readfirstlane(own);
  dst = (total <= few ? few_dst : dst) + __builtin_amdgcn_readfirstlane(hole);
  src = (total <= few ? few_src : src) + __builtin_amdgcn_readfirstlane(source);
  each_key([&](int t0, unsigned key) {
    unsigned long long kept = __ballot(key > bound);
    const unsigned long long eq = __ballot(key == bound), front = lanes_before(m, t0);
    if (eq) {
      const int at = (int)__builtin_amdgcn_mbcnt_hi((unsigned)(eq >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)eq, 0u));
      kept |= eq & __ballot(at < own);
      own -= __popcll(eq);
    }
    put_slots(dst, t0, ~kept & front & lanes_before(last, t0));
    put_slots(src, t0, kept & ~front);
  });
  return total;
}

// The scales (2, 4 or 8 bytes) of a moved row of pages in 4 bits.
__device__ __forceinline__ void move_scales(const PagedEvict& a, char* pages, int h, int from_page, int src, int into_page,
                                            int dst) {
  const char* from = pages + (size_t)from_page * a.scale_page + (size_t)h * a.scale_head +
                     (size_t)(src - a.div.of(src) * a.page_size) * a.scale_slot;
  char* into = pages + (size_t)into_page * a.scale_page + (size_t)h * a.scale_head +
               (size_t)(dst - a.div.of(dst) * a.page_size) * a.scale_slot;
  for (int i = 0; i < a.scale_bytes; i += 2)
    *reinterpret_cast<uint16_t*>(into + i) = *reinterpret_cast<const uint16_t*>(from + i);
}

// A move's rows of K and V, kRows of them in flight per thread; a row takes as many
// lanes as it has 16-byte pieces.  Slots in srcs and dsts (`count` of them), this
// workgroup's from its index on, every groups-th kRows * rows-at-a-time of them.
// kFourBits: with their scales (a kernel of its own: as a branch it took 9 more registers
// and spilled 12 scalar ones of the selection over 16-bit pages, 10.6 -> 10.9 us for a cut of 64).
template <int kThreads, int kRows, bool kFourBits>
__device__ __forceinline__ void move_rows(const PagedEvict& a, int b, int h, size_t row, const int32_t* srcs,
                                          const int32_t* dsts, int count, int group, int groups) {
  const int c = (threadIdx.x & ((1 << a.log_pieces) - 1)) << 4, step = kThreads >> a.log_pieces;
  const int32_t* tab = a.table + (size_t)b * a.max_pages;
  for (int k1 = group * step * kRows; k1 < count; k1 += groups * step * kRows) {
    const int k0 = k1 + (threadIdx.x >> a.log_pieces);
    int src[kRows], dst[kRows], from_page[kRows], into_page[kRows];
    size_t to[kRows];
    bool in[kRows];
    uint4 kv[kRows], vv[kRows];
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      if (k1 + e * step >= count) break;
      const int k = min(k0 + e * step, count - 1);
      src[e] = srcs[k];
      dst[e] = dsts[k];
      in[e] = k0 + e * step < count;
    }
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      if (k1 + e * step >= count) break;
      const int ps = a.div.of(src[e]), pd = a.div.of(dst[e]);
      int from = tab[ps], into = tab[pd];
      if ((unsigned)from >= (unsigned)a.pages || (unsigned)into >= (unsigned)a.pages) {
        if (in[e]) report_error(a.err, error_host_slot(a.err), kErrPages);
        in[e] = false;
        from = into = 0;
      }
      from_page[e] = from;
      into_page[e] = into;
      const size_t f = (size_t)from * a.page_bytes + (size_t)(src[e] - ps * a.page_size) * a.slot_bytes +
                       (size_t)h * a.head_bytes + c;
      to[e] = (size_t)into * a.page_bytes + (size_t)(dst[e] - pd * a.page_size) * a.slot_bytes +
              (size_t)h * a.head_bytes + c;
      kv[e] = load_nt16(a.kp + f);
      vv[e] = load_nt16(a.vp + f);
    }
    asm volatile("" ::: "memory");  // (all of them are asked for before anything is stored)
#pragma unroll
    for (int e = 0; e < kRows; ++e)
      if (k1 + e * step < count && in[e]) {
        *reinterpret_cast<uint4*>(a.kp + to[e]) = kv[e];
        *reinterpret_cast<uint4*>(a.vp + to[e]) = vv[e];
        if (c == 0) {
          if constexpr (kFourBits) {
            move_scales(a, a.k_scales, h, from_page[e], src[e], into_page[e], dst[e]);
            move_scales(a, a.v_scales, h, from_page[e], src[e], into_page[e], dst[e]);
          }
          a.scores_out[row * a.slots + dst[e]] = a.scores[row * a.slots + src[e]];
          a.positions_out[row * a.slots + dst[e]] = a.positions[row * a.slots + src[e]];
        }
      }
  }
}

// The sequence's new length and tokens seen, by the last of its workgroups to come;
// called behind a barrier, when all threads have read the old ones, and late, by
// the last wave, which others need not wait for.
__device__ __forceinline__ void evict_lengths(const PagedEvict& a, const EvictRow& r, int b, int workgroups) {
  if (threadIdx.x != kET - 1) return;
  if (inc_dev(&a.counters[b]) != (unsigned)(workgroups - 1)) return;
  st_dev(&a.counters[b], 0u);
  a.lengths_out[b] = r.m;
  if (a.seen_out != a.seen) a.seen_out[b] = a.seen[b];
}

// One workgroup per (sequence, KV head), rows of up to kLongRow slots: the keys in
// LDS, the budget-th largest by three histogram passes (11, 11 and 10 bits), then
// the slots that move, found by each wave in its own share, and, if they are few,
// their rows.  Bound by the latency of its steps and, its 16 waves on one CU, the
// instructions of each 64 slots: 2112 slots to 2048, 8 x 8 rows, 11.5 us, of which by
// clock reads the reads and the first counts 1.4, the passes 2.4, counts and lists of
// the moves 3.0, the moves 1.8; up to 9001 slots, 16 x 4 rows, 15 traced.
// Up to this many slots; twice as many where the rows fill the CUs by themselves (31
// steps of 64 slots a wave: one row of 32000 slots 45 us, 43 in parts; 64 rows 59,
// 75 in parts).
constexpr int kLongRow = 16384, kManyRows = 64;

template <bool kFourBits>
__global__ __launch_bounds__(kET) void paged_select_kernel(PagedEvict a) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ unsigned hist[3][2048], wsum[kEWaves], found[3][2];
  __shared__ EvictCounts counts[kEWaves];
  __shared__ int32_t few[2][kFew];
  extern __shared__ unsigned keys[];  // of whole 64-slot steps
  for (int i = tid; i < 3 * 2048; i += kET) (&hist[0][0])[i] = 0u;
  const EvictRow r(a, b, h);
  asm volatile("" ::"s"(r.n), "s"(r.m));  // (read, not only asked for, before others may write the length)
  __syncthreads();
  const bool cut = r.n > r.m && r.m > 0;
  const int steps = (r.n + 64 * kEWaves - 1) / (64 * kEWaves);  // of 64 slots per wave
  const int first = min(64 * steps * w, r.n), last = min(first + 64 * steps, r.n);
  constexpr int kU = 4;
  for (int t0 = first; t0 < last; t0 += kU * 64) {
    EvictSlots<kU> slots;
    unsigned k[kU];
    slots.load(r, t0);
    slots.keys(a, r, t0, last, r.copy, k);
    if (!cut) continue;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (t0 + 64 * u < last) {
        keys[t0 + 64 * u + lane] = k[u];
        atomicAdd(&hist[0][digit<0>(k[u])], 1u);
      }
  }
  if (!cut) {
    if (tid == 0) a.count[r.row] = 0;
    evict_lengths(a, r, b, a.kv_heads);
    return;
  }
  auto each_key = [&](auto f) {  // (a wave reads what it wrote itself)
#pragma unroll 1
    for (int t0 = first; t0 < last; t0 += 64) f(t0, keys[t0 + lane]);
  };
  __syncthreads();
  unsigned bound = 0, need = r.m;
  find_digit<0>(hist[0][2047 - 2 * tid], hist[0][2046 - 2 * tid], wsum, found[0], bound, need);
  each_key([&](int, unsigned key) {
    if (matches<1>(key, bound)) atomicAdd(&hist[1][digit<1>(key)], 1u);
  });
  __syncthreads();
  find_digit<1>(hist[1][2047 - 2 * tid], hist[1][2046 - 2 * tid], wsum, found[1], bound, need);
  each_key([&](int, unsigned key) {
    if (matches<2>(key, bound)) atomicAdd(&hist[2][digit<2>(key)], 1u);
  });
  __syncthreads();
  find_digit<2>(hist[2][2047 - 2 * tid], hist[2][2046 - 2 * tid], wsum, found[2], bound, need);
  const EvictCounts mine = count_moves(each_key, bound, r.m, last);
  const int total = write_moves(each_key, mine, bound, (int)need, r.m, last, a.dst + r.row * a.moves,
                                a.src + r.row * a.moves, counts, kFew, few[1], few[0]);
  if (tid == 0) a.count[r.row] = total <= kFew ? 0 : total;
  if (total <= kFew) __syncthreads();  // (the fork's copies of what stays come before the moves')
  evict_lengths(a, r, b, a.kv_heads);
  if (total <= kFew) move_rows<kET, 4, kFourBits>(a, b, h, r.row, few[0], few[1], total, 0, 1);
}

// Longer rows take one launch per pass, a part of a row per workgroup: a.part slots,
// kPart or, so that no row has more than kMostParts and a few, a multiple of it.
// The slots before the budget and those behind it have parts of their own.  Each
// workgroup leaves its counts of the digits, from which all of the next launch find
// theirs.  65536 slots, 8 rows: 6 + 7 + 7 + 15 us; one workgroup for each row 60.
constexpr int kPart = 8192, kPartKeys = kPart / kET, kMostParts = 128;

struct EvictPart {
  int part, first, last, front, parts;  // slots; parts before the budget, parts
  __device__ __forceinline__ EvictPart(const PagedEvict& a, const EvictRow& r, int x) : part(a.part) {
    front = (r.m + part - 1) / part;
    parts = front + (r.n - r.m + part - 1) / part;
    first = x < front ? x * part : r.m + (x - front) * part;
    last = min(first + part, x < front ? r.m : r.n);
  }
  // slots of part y (before the budget)
  __device__ __forceinline__ int size(const EvictRow& r, int y) const { return min(part, r.m - y * part); }
};

// The keys of a wave's share of a part: kept in LDS where the part is kPart slots,
// read again by every pass over them where it is longer.
struct EvictKeys {
  const PagedEvict& a;
  const EvictRow& r;
  int first, last;
  bool copy;
  EvictSlots<kPartKeys> slots;
  unsigned* lds;  // [kPart]
  __device__ __forceinline__ EvictKeys(const PagedEvict& a, const EvictRow& r, const EvictPart& p, bool copy, unsigned* lds)
      : a(a), r(r), copy(copy) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = p.part / kEWaves;
    first = p.first + share * w;
    last = min(p.last, first + share);
    this->lds = lds + 64 * kPartKeys * w + (threadIdx.x & 63);
    slots.load(r, first);
  }
  __device__ __forceinline__ void put(int t0, bool copy) {
    unsigned key[kPartKeys];
    slots.keys(a, r, t0, last, copy, key);
#pragma unroll
    for (int k = 0; k < kPartKeys; ++k) lds[64 * k] = key[k];
  }
  __device__ __forceinline__ void ready() {  // once, behind the caller's own loads
    put(first, copy);
    if (!copy) return;
    for (int t0 = first + 64 * kPartKeys; t0 < last; t0 += 64 * kPartKeys) {
      slots.load(r, t0);
      put(t0, true);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    for (int t0 = first; t0 < last; t0 += 64 * kPartKeys) {
      if (a.part != kPart) {
        slots.load(r, t0);
        put(t0, false);
      }
#pragma unroll 1
      for (int k = 0; k < kPartKeys && t0 + 64 * k < last; ++k) f(t0 + 64 * k, lds[64 * k]);
    }
  }
};

// Workspace of a row: each pass's prefix and need, then per part the number of its
// keys above the digits found so far, and its counts of the pass's digits.
struct EvictTables {
  unsigned *state, *above, *hist;
  __device__ __forceinline__ EvictTables(const PagedEvict& a, size_t row) {
    state = a.tables + row * a.table_words;
    above = state + 8;
    hist = above + ((a.most_parts + 7) & ~7);
  }
  __device__ __forceinline__ unsigned* digits(int part, int pass) const { return hist + ((size_t)part * 3 + pass) * 2048; }
};

// What pass kPass (0..3; 3: the bound itself) starts from: the digits found by the
// passes before it.
template <int kPass>
__device__ __forceinline__ void start_pass(const EvictRow& r, const EvictPart& p, const EvictTables& t, int x,
                                           unsigned* wsum, unsigned* found, unsigned& prefix, unsigned& need) {
  prefix = 0;
  need = r.m;
  if constexpr (kPass > 0) {
    const int tid = threadIdx.x;
    if (kPass > 1) {
      prefix = t.state[2 * kPass - 4];
      need = t.state[2 * kPass - 3];
    }
    uint2 sum = make_uint2(0u, 0u);
    for (int y0 = 0; y0 < p.parts; y0 += 8) {
      uint2 c[8];
#pragma unroll
      for (int y = 0; y < 8; ++y)
        c[y] = *reinterpret_cast<const uint2*>(t.digits(min(y0 + y, p.parts - 1), kPass - 1) + 2046 - 2 * tid);
#pragma unroll
      for (int y = 0; y < 8; ++y)
        if (y0 + y < p.parts) {
          sum.x += c[y].x;
          sum.y += c[y].y;
        }
    }
    find_digit<kPass - 1>(sum.y, sum.x, wsum, found, prefix, need);
    if (x == 0 && tid == 0) {
      t.state[2 * kPass - 2] = prefix;
      t.state[2 * kPass - 1] = need;
    }
  }
}

template <int kPass>
__global__ __launch_bounds__(kET) void paged_rank_kernel(PagedEvict a) {
  const int x = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  __shared__ unsigned hist[2048], wsum[kEWaves], found[2], part_keys[kPart];
  __shared__ int sums[kEWaves];
  const EvictRow r(a, b, h);
  const EvictPart p(a, r, x);
  if (kPass == 0 && x == 0 && tid == 0) {  // (paged_pick_kernel writes the new lengths)
    unsigned* sizes = EvictTables(a, r.row).state + 6;
    sizes[0] = (unsigned)r.n;
    sizes[1] = (unsigned)r.m;
  }
  if (x >= p.parts) return;
  EvictKeys keys(a, r, p, kPass == 0 && r.copy, part_keys);
  if (r.n <= r.m || r.m == 0) {
    if (kPass == 0) keys.ready();  // (the fork gets its copies)
    return;
  }
  for (int i = tid; i < 2048; i += kET) hist[i] = 0u;
  const EvictTables t(a, r.row);
  unsigned prefix, need;
  start_pass<kPass>(r, p, t, x, wsum, found, prefix, need);
  keys.ready();
  __syncthreads();
  if constexpr (kPass > 0) {  // this part's keys above the digit found
    const uint2 c = *reinterpret_cast<const uint2*>(t.digits(x, kPass - 1) + 2046 - 2 * tid);
    const int d = (int)(prefix & 2047u);
    const int above = block_sum((2047 - 2 * tid > d ? (int)c.y : 0) + (2046 - 2 * tid > d ? (int)c.x : 0), sums);
    if (tid == 0) t.above[x] = (kPass > 1 ? t.above[x] : 0u) + (unsigned)above;
  }
  keys.each([&](int, unsigned key) {
    if (matches<kPass>(key, prefix)) atomicAdd(&hist[digit<kPass>(key)], 1u);
  });
  __syncthreads();
  uint2* out = reinterpret_cast<uint2*>(t.digits(x, kPass));
  out[tid] = *reinterpret_cast<const uint2*>(&hist[2 * tid]);
}

__global__ __launch_bounds__(kET) void paged_pick_kernel(PagedEvict a) {
  const int x = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ unsigned wsum[kEWaves], found[2], part_keys[kPart];
  __shared__ int above_s[kEWaves], equal_s[kEWaves];
  __shared__ EvictCounts counts[kEWaves];
  const EvictTables t(a, (size_t)b * a.kv_heads + h);
  const EvictRow r(a, b, h, t.state + 6);
  const EvictPart p(a, r, x);
  if (x == 0 && h == 0 && tid == 0) {
    a.lengths_out[b] = r.m;
    if (a.seen_out != a.seen) a.seen_out[b] = a.seen[b];
  }
  const bool cut = r.n > r.m && r.m > 0;
  if (!cut && x == 0 && tid == 0) a.count[r.row] = 0;
  if (!cut || x >= p.parts) return;
  EvictKeys keys(a, r, p, false, part_keys);
  unsigned bound, need;
  start_pass<3>(r, p, t, x, wsum, found, bound, need);
  keys.ready();
  // the parts in order, a wave each: what lies before this one
  const int d = (int)(bound & 1023u);
  int tie = 0, hole = 0, source = 0, tie_x = 0, hole_x = 0, source_x = 0;
  for (int y0 = 0; y0 < p.parts; y0 += kEWaves) {
    const int y = min(y0 + w, p.parts - 1);
    const unsigned* c = t.digits(y, 2);
    int more = 0;
    for (int i = 0; i < 1024; i += 256) {
      const uint4 v = reinterpret_cast<const uint4*>(c + i)[lane];
      const int at = i + 4 * lane;
      more += (at > d ? (int)v.x : 0) + (at + 1 > d ? (int)v.y : 0) + (at + 2 > d ? (int)v.z : 0) + (at + 3 > d ? (int)v.w : 0);
    }
    more = wave_sum_i(more);
    if (lane == 0) {
      above_s[w] = (int)t.above[y] + more;
      equal_s[w] = (int)c[d];
    }
    __syncthreads();
    for (int k = 0; k < min(kEWaves, p.parts - y0); ++k) {
      if (y0 + k == x) {
        tie_x = tie;
        hole_x = hole;
        source_x = source;
      }
      const int kept = above_s[k] + min(max((int)need - tie, 0), equal_s[k]);
      tie += equal_s[k];
      if (y0 + k < p.front) hole += p.size(r, y0 + k) - kept;
      else source += kept;
    }
    __syncthreads();
  }
  if (x == 0 && tid == 0) a.count[r.row] = hole;
  auto each_key = [&](auto f) { keys.each(f); };
  const EvictCounts mine = count_moves(each_key, bound, r.m, keys.last);
  write_moves(each_key, mine, bound, (int)need - tie_x, r.m, keys.last, a.dst + r.row * a.moves + hole_x,
              a.src + r.row * a.moves + source_x, counts, -1, nullptr, nullptr);
}

// Moves the kept rows into the holes where the selection has not: a copy, bound by
// the rows it reads and writes.  No source is another move's destination.  100 MB
// of 256-byte rows read and written: 23.2 us = 4.4 TB/s (4 or 8 rows in flight per
// thread: fewer workgroups, and 1 to 4 us more).
constexpr int kMoveRows = 2;

template <bool kFourBits>
__global__ __launch_bounds__(kPT) void paged_move_kernel(PagedEvict a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const size_t row = (size_t)b * a.kv_heads + h;
  move_rows<kPT, kMoveRows, kFourBits>(a, b, h, row, a.src + row * a.moves, a.dst + row * a.moves, a.count[row], blockIdx.x,
                                       gridDim.x);
}

}  // namespace
}  // namespace prismkv

using namespace prismkv;

namespace {

struct WorkLayout {
  size_t sums, state, logits, bytes;  // counters first
  unsigned state_stride;
  int64_t logit_stride, quanta, units;
};

WorkLayout attend_layout(int sequences, int kv_heads, int group, int head_dim, int64_t slots, bool weigh, int dtype) {
  WorkLayout w;
  const int64_t tiles = (group + 15) / 16, heads = (int64_t)kv_heads * tiles;
  const int least = dtype >= kFour     ? head_dim == 256 ? kLeast<kFour, 256> : kLeast<kFour, 128>
                    : dtype == kFp32 ? head_dim == 256 ? kLeast<kFp32, 256> : kLeast<kFp32, 128>
                                     : head_dim == 256 ? kLeast<kBf16, 256> : kLeast<kBf16, 128>;
  const int64_t workgroups = sequences * heads * ((slots + least * kQuantum - 1) / (least * kQuantum));  // of full tables
  w.quanta = workgroups * least;
  w.units = workgroups < kUnits ? workgroups : kUnits;
  w.state_stride = (unsigned)((group < 16 ? group : 16) * (head_dim + 2));
  w.logit_stride = (slots + 31) & ~31ll;  // (whole blocks of 16 are written)
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  w.sums = up((size_t)sequences * heads * sizeof(unsigned));
  w.state = w.sums + up((size_t)sequences * kv_heads * group * sizeof(float2));
  w.logits = w.state + up((size_t)2 * w.units * w.state_stride * sizeof(float));
  w.bytes = w.logits + (weigh ? (size_t)sequences * kv_heads * group * w.logit_stride * sizeof(float) : 0);
  return w;
}

struct EvictLayout {
  size_t count, src, dst, tables, bytes;  // counters (a word per sequence) first
  int64_t moves, part, parts, table_words;
};

EvictLayout evict_layout(int sequences, int kv_heads, int64_t slots) {
  EvictLayout w;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t rows = (size_t)sequences * kv_heads;
  w.moves = slots / 2 + 1;
  w.part = kPart * ((slots + (int64_t)kPart * kMostParts - 1) / ((int64_t)kPart * kMostParts));
  w.parts = slots > ((int64_t)rows < kManyRows ? kLongRow : 2 * kLongRow) ? slots / w.part + 2 : 0;
  w.table_words = w.parts ? 8 + ((w.parts + 7) & ~7ll) + w.parts * 3 * 2048 : 0;
  w.count = up((size_t)sequences * sizeof(unsigned));
  w.src = w.count + up(rows * sizeof(int32_t));
  w.dst = w.src + up(rows * w.moves * sizeof(int32_t));
  w.tables = w.dst + up(rows * w.moves * sizeof(int32_t));
  w.bytes = w.tables + rows * w.table_words * sizeof(unsigned);
  return w;
}

}  // namespace

extern "C" {

size_t prismkv_paged_attend_work_bytes(int sequences, int kv_heads, int group, int head_dim, int64_t slots, int weigh,
                                       int dtype) {
  const bool known = (dtype >= kBf16 && dtype <= kFp32) || dtype == (kFour | kBf16) || dtype == (kFour | kFp16);
  if (!known || sequences < 1 || kv_heads < 1 || group < 1 || head_dim < 1 || slots < 1) return 0;
  const WorkLayout w = attend_layout(sequences, kv_heads, group, head_dim, slots, weigh != 0, dtype);
  return w.quanta > INT32_MAX ? 0 : w.bytes;  // (refused: quanta are counted in 32 bits)
}

int prismkv_paged_attend(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t q, uint64_t lse,
                         uint64_t paged_work, uint64_t out, int group, int flags, double scale, size_t work_bytes,
                         uint64_t stream) {
  const bool weigh = flags & 1;
  if (const int rc = check_cache(cache, into, weigh)) return rc;
  if (flags & ~3) return kBadMode;
  const prismkv_paged_cache& c = *cache;
  const double scale2 = scale * 1.4426950408889634;  // the exponents are powers of 2, in fp32
  if (group < 1 || group > 1024 || !(scale2 >= -FLT_MAX && scale2 <= FLT_MAX)) return kBadSize;
  if (!q || !paged_work || !out || (q | paged_work) & 15 || lse & 3 || out & 3) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  const WorkLayout w = attend_layout(c.sequences, c.kv_heads, group, c.head_dim, slots, weigh, c.dtype);
  if (work_bytes < w.bytes || w.quanta > INT32_MAX) return kBadSize;
  const int es = page_element_bytes(c.dtype);
  PagedAttend a{};
  a.q = reinterpret_cast<const void*>(q);
  a.k = reinterpret_cast<const void*>(c.k);
  a.v = reinterpret_cast<const void*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.lengths = reinterpret_cast<const int32_t*>(flags & 2 ? into->lengths : c.lengths);
  a.lse_out = reinterpret_cast<float*>(lse);
  a.out = reinterpret_cast<void*>(out);
  char* work = reinterpret_cast<char*>(paged_work);
  a.counters = reinterpret_cast<unsigned*>(work);
  a.state = reinterpret_cast<float*>(work + w.state);
  if (weigh) {
    a.scores = reinterpret_cast<const float*>(c.scores);
    a.scores_out = reinterpret_cast<float*>(into->scores);
    a.sums_work = reinterpret_cast<float2*>(work + w.sums);
    a.logits = reinterpret_cast<float*>(work + w.logits);
  }
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.head_bytes = c.head_stride * es;
  a.logit_stride = w.logit_stride;
  a.slots = slots;
  a.page_units = (unsigned)(c.page_stride * es >> 4);
  a.slot_units = (unsigned)(c.slot_stride * es >> 4);
  a.state_stride = w.state_stride;
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  a.group = group;
  a.tiles = (group + 15) / 16;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.scale = (float)scale2;
  if (c.dtype >= kFour) {
    a.k_scales = reinterpret_cast<const uint8_t*>(c.k_scales);
    a.v_scales = reinterpret_cast<const uint8_t*>(c.v_scales);
    a.scale_page = c.scale_page_stride;
    a.scale_head = c.scale_head_stride;
    a.scale_slot = (unsigned)c.scale_slot_stride;
    a.q_and = scale2 == 0 ? 0u : ~0u;
    a.q_xor = scale2 < 0 ? 0x80008000u : 0u;
    a.scale = scale2 == 0 ? 1.f : (float)(scale2 < 0 ? -scale2 : scale2);
  }
  const hipStream_t s = (hipStream_t)stream;
  int rc;
  if (c.dtype == kBf16) rc = launch_attend_dim<kBf16>(a, c.head_dim, w.units, s);
  else if (c.dtype == kFp16) rc = launch_attend_dim<kFp16>(a, c.head_dim, w.units, s);
  else if (c.dtype == kFp32) rc = launch_attend_dim<kFp32>(a, c.head_dim, w.units, s);
  else rc = attend_in_four(a, c.dtype, c.head_dim, w.units, s);
  if (rc || !weigh) return rc;
  const int64_t blocks = (slots + kPT - 1) / kPT;
  hipLaunchKernelGGL(paged_weigh_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), c.kv_heads, c.sequences),
                     dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

int prismkv_paged_append(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t k, uint64_t v,
                         uint64_t offsets, int64_t rows, int64_t k_row_stride, int64_t k_head_stride,
                         int64_t v_row_stride, int64_t v_head_stride, uint64_t stream) {
  if (const int rc = check_cache(cache, into, false)) return rc;
  if (cache->dtype >= kFour)
    return prismkv_paged_append_rows(cache, into, k, v, 0, 0, offsets, 0, rows, k_row_stride, k_head_stride, v_row_stride,
                                     v_head_stride, 0, 0, 0, 0, 0, 0., stream);
  const prismkv_paged_cache& c = *cache;
  if (rows < 0 || rows > INT32_MAX || (!offsets && rows != c.sequences)) return kBadSize;
  if (rows && (!k || !v)) return kBadSize;
  const int64_t es = element_bytes(c.dtype), limit = 1ll << 40;
  for (const int64_t stride : {k_row_stride, k_head_stride, v_row_stride, v_head_stride})
    if (stride < -limit || stride > limit || stride * es & 15) return kBadSize;
  if ((k | v) & 15 || offsets & 3) return kBadSize;
  PagedAppend a{};
  a.k = reinterpret_cast<const char*>(k);
  a.v = reinterpret_cast<const char*>(v);
  a.kp = reinterpret_cast<char*>(c.k);
  a.vp = reinterpret_cast<char*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
  a.lengths = reinterpret_cast<const int32_t*>(c.lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(into->lengths);
  a.seen = reinterpret_cast<const int32_t*>(c.seen);
  a.seen_out = reinterpret_cast<int32_t*>(into->seen);
  a.positions = reinterpret_cast<int32_t*>(c.positions);
  a.positions_out = reinterpret_cast<int32_t*>(into->positions);
  a.scores = reinterpret_cast<float*>(c.scores);
  a.scores_out = reinterpret_cast<float*>(into->scores);
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.rows = rows;
  a.k_row = k_row_stride * es;
  a.k_head = k_head_stride * es;
  a.v_row = v_row_stride * es;
  a.v_head = v_head_stride * es;
  a.page_bytes = c.page_stride * es;
  a.head_bytes = c.head_stride * es;
  a.slot_bytes = c.slot_stride * es;
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  while (16 << a.log_pieces < c.head_dim * es) ++a.log_pieces;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = c.page_size * c.max_pages;
  const hipStream_t s = (hipStream_t)stream;
  if (!offsets) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(c.sequences), dim3(kPT), 0, s, a);
    return (int)hipGetLastError();
  }
  for (; a.first_row < rows; a.first_row += kLaunchRows) {
    const int64_t more = rows - a.first_row < kLaunchRows ? rows - a.first_row : kLaunchRows;
    hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)((more + kAppendRows - 1) / kAppendRows)), dim3(kPT), 0, s, a);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  if (rows && a.lengths_out != a.lengths) return 0;  // (advanced by the rows' launches)
  hipLaunchKernelGGL(paged_advance_kernel, dim3((c.sequences + kPT - 1) / kPT), dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

size_t prismkv_paged_evict_work_bytes(int sequences, int kv_heads, int64_t slots) {
  if (sequences < 1 || kv_heads < 1 || slots < 1 || slots > 1 << 30) return 0;
  return evict_layout(sequences, kv_heads, slots).bytes;
}

int prismkv_paged_evict(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t keeps,
                        uint64_t paged_work, int keep, int recent, int sinks, size_t work_bytes, uint64_t stream) {
  if (const int rc = check_cache(cache, into, true)) return rc;
  const prismkv_paged_cache& c = *cache;
  if (keep < 0 || recent < 0 || sinks < 0 || (keeps && keep)) return kBadSize;
  if (!paged_work || paged_work & 15 || keeps & 3) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  const EvictLayout l = evict_layout(c.sequences, c.kv_heads, slots);
  if (work_bytes < l.bytes) return kBadSize;
  const int es = page_element_bytes(c.dtype);
  PagedEvict a{};
  a.kp = reinterpret_cast<char*>(c.k);
  a.vp = reinterpret_cast<char*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.lengths = reinterpret_cast<const int32_t*>(c.lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(into->lengths);
  a.seen = reinterpret_cast<const int32_t*>(c.seen);
  a.seen_out = reinterpret_cast<int32_t*>(into->seen);
  a.scores = reinterpret_cast<const float*>(c.scores);
  a.scores_out = reinterpret_cast<float*>(into->scores);
  a.positions = reinterpret_cast<const int32_t*>(c.positions);
  a.positions_out = reinterpret_cast<int32_t*>(into->positions);
  a.keeps = reinterpret_cast<const int32_t*>(keeps);
  char* work = reinterpret_cast<char*>(paged_work);
  a.moves = l.moves;
  a.counters = reinterpret_cast<unsigned*>(work);
  a.count = reinterpret_cast<int32_t*>(work + l.count);
  a.src = reinterpret_cast<int32_t*>(work + l.src);
  a.dst = reinterpret_cast<int32_t*>(work + l.dst);
  a.tables = reinterpret_cast<unsigned*>(work + l.tables);
  a.table_words = l.table_words;
  a.part = (int)l.part;
  a.most_parts = (int)l.parts;
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.page_bytes = c.page_stride * es;
  a.head_bytes = c.head_stride * es;
  a.slot_bytes = c.slot_stride * es;
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  while (16 << a.log_pieces < page_row(c) * es) ++a.log_pieces;
  if (c.dtype >= kFour) {
    a.k_scales = reinterpret_cast<char*>(c.k_scales);
    a.v_scales = reinterpret_cast<char*>(c.v_scales);
    a.scale_page = c.scale_page_stride;
    a.scale_head = c.scale_head_stride;
    a.scale_slot = c.scale_slot_stride;
    a.scale_bytes = c.head_dim / 32;
  }
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = (int)slots;
  a.keep = keep;
  a.recent = recent;
  a.sinks = sinks;
  const hipStream_t s = (hipStream_t)stream;
  int64_t most = slots / 2;  // moves of a row
  if (!keeps) most = keep < slots - keep ? keep : slots > keep ? slots - keep : 0;
  if (most > slots / 2) most = slots / 2;
  const auto select = c.dtype >= kFour ? paged_select_kernel<true> : paged_select_kernel<false>;
  const auto move = c.dtype >= kFour ? paged_move_kernel<true> : paged_move_kernel<false>;
  int rc;
  if (!l.parts) {
    const int lds = (int)((slots + 64 * kEWaves - 1) / (64 * kEWaves)) * 64 * kEWaves * (int)sizeof(unsigned);
    if (lds > 32 * 1024) {  // (beside the static 27 KB)
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(select),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 2 * kLongRow * (int)sizeof(unsigned));
      if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(select, dim3(c.kv_heads, c.sequences), dim3(kET), lds, s, a);
    rc = (int)hipGetLastError();
    if (rc || most <= kFew) return rc;
  } else {
    const dim3 grid((unsigned)l.parts, c.kv_heads, c.sequences);
    hipLaunchKernelGGL(paged_rank_kernel<0>, grid, dim3(kET), 0, s, a);
    hipLaunchKernelGGL(paged_rank_kernel<1>, grid, dim3(kET), 0, s, a);
    hipLaunchKernelGGL(paged_rank_kernel<2>, grid, dim3(kET), 0, s, a);
    hipLaunchKernelGGL(paged_pick_kernel, grid, dim3(kET), 0, s, a);
    rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  const int64_t blocks = (most + (kPT >> a.log_pieces) * kMoveRows - 1) / ((kPT >> a.log_pieces) * kMoveRows);
  const int64_t room = 4096 / ((int64_t)c.sequences * c.kv_heads) + 1;  // workgroups of a row where there are many rows
  const int64_t grid = blocks < 1 ? 1 : blocks < room ? blocks : room;
  hipLaunchKernelGGL(move, dim3((unsigned)grid, c.kv_heads, c.sequences), dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

}  // extern "C"
