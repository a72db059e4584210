// The paged key-value cache: writing rows into pages, attention of one new
// query token of every sequence over its pages, and eviction by accumulated
// attention weight.
//
// K and V pages are [pages][kv_heads][page_size][head_dim] with any strides of
// 16-byte multiples (the same for both); slot t of sequence b lies in page
// table[b][t / page_size].  A table entry outside [0, pages) within a
// sequence's length is reported through the cache's error word and never read
// through.
#include "paged.h"

namespace prismkv {
namespace {

// ------------------------------------------------------------------ attention
//
// s_t = scale q.k_t, p_t = e^(s_t - m) / z, o = sum p_t v_t for the `group`
// query heads of one KV head: every K and V row is read once for all of them
// (2 bytes x 2 head_dim per 4 group head_dim flops), so the kernel is bound by
// the reads.  One pass with the running maximum and sum (flash form).
//
// Split: the tokens of all sequences and KV heads are cut into about kUnits
// equal chunks on the device (the lengths live there), a workgroup of 4 waves
// per chunk, each wave on its own 32-token (fp32: 16) tiles: no barrier and no
// LDS until the waves' states meet.  The last workgroup of a (sequence, head)
// to arrive joins the chunks' states in chunk order, so the result does not
// depend on the order of arrival.

// Wave's running state of 16 heads (columns j) over head_dim D.
template <int DT, int D>
struct Acc;
template <int D>
struct Acc<kFp32, D> {
  f32x4 hi[D / 16];
};
// 16-bit types: P is a head and a remainder of the type (two products, about
// twice the type's significant bits), accumulated apart: a remainder of zero
// times an infinite V is NaN, which the join drops when the head's sum has the
// infinity.
template <int D>
struct Acc<kBf16, D> {
  f32x4 hi[D / 16], lo[D / 16];
};
template <int D>
struct Acc<kFp16, D> {
  f32x4 hi[D / 16], lo[D / 16];
};

// The tile of one step as loaded.  16-bit (32 tokens, two 16-token blocks):
// lane (j, q) holds row j of each block at dims 32c + 8q .. +8 (K, the A operand
// of the 16x16x32 product) and rows 4q + t at dims (D/16) j .. + D/16 (V): D/16
// column blocks n map dim (D/16) j + n to column j, so that a load covers whole
// rows and the pairs of rows are joined per dim with one byte permutation.
// fp32 (16 tokens): K dims 16c + 4q .. +4 (four 16x16x4 products per load), V
// the same with float columns.
template <int DT, int D>
struct Tile {
  static constexpr int kBlocks = DT == kFp32 ? 1 : 2;
  static constexpr int kTokens = 16 * kBlocks;
  static constexpr int kKLoads = D * kElem<DT> / 64;        // 16-byte loads of a K row per lane
  static constexpr int kVWords = D * kElem<DT> / 64;        // 32-bit words of a V row per lane
  uint4 k[kBlocks][kKLoads];
  unsigned v[kBlocks][4][kVWords];
};

template <int W>
__device__ __forceinline__ void load_words(unsigned (&dst)[W], const char* p) {
  if constexpr (W == 2) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    dst[0] = x.x;
    dst[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 x = load_nt16(p + 4 * i);
      dst[i] = x.x;
      dst[i + 1] = x.y;
      dst[i + 2] = x.z;
      dst[i + 3] = x.w;
    }
  }
}

// Element N of two rows' words as a pair (low half from a).
template <int N, int W>
__device__ __forceinline__ unsigned pair16(const unsigned (&a)[W], const unsigned (&b)[W]) {
  return __builtin_amdgcn_perm(b[N >> 1], a[N >> 1], (N & 1) ? 0x07060302u : 0x05040100u);
}

template <int DT>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// p as a head and a remainder of the 16-bit type.
template <int DT>
__device__ __forceinline__ void split16(float p, unsigned& hi, unsigned& lo) {
  if constexpr (DT == kBf16) {
    const unsigned u = __float_as_uint(p);
    hi = u >> 16;
    lo = f32_to_bf16(p - __uint_as_float(u & 0xffff0000u));
  } else {
    const _Float16 h = (_Float16)p;
    const _Float16 l = (_Float16)(p - (float)h);
    hi = __builtin_bit_cast(unsigned short, h);
    lo = __builtin_bit_cast(unsigned short, l);
  }
}

// P is held times 2^kBias: fp16 probabilities from 2^-29 of the maximum up stay
// normal numbers (bf16 and fp32 have the exponents for them).
template <int DT>
constexpr int kBias = DT == kFp16 ? 15 : 0;

template <int N, int DT, int D>
__device__ __forceinline__ void pv_columns(Acc<DT, D>& acc, const Tile<DT, D>& t, u32x4 ph, u32x4 pl) {
  if constexpr (N < D / 16) {
    const u32x4 vb = {pair16<N>(t.v[0][0], t.v[0][1]), pair16<N>(t.v[0][2], t.v[0][3]),
                      pair16<N>(t.v[1][0], t.v[1][1]), pair16<N>(t.v[1][2], t.v[1][3])};
    acc.hi[N] = mfma32<DT>(ph, vb, acc.hi[N]);
    acc.lo[N] = mfma32<DT>(pl, vb, acc.lo[N]);
    pv_columns<N + 1>(acc, t, ph, pl);
  }
}

template <int DT, int D>
__global__ __launch_bounds__(kPT, D == 256 ? 1 : 2) void paged_attend_kernel(PagedAttend a) {
  typedef Tile<DT, D> T;
  constexpr int kQRegs = T::kKLoads;
  extern __shared__ float lds[];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PagedUnit u = find_unit(a, blockIdx.x);
  if (u.b < 0) return;
  const int h = u.hh / a.tiles, g0 = 16 * (u.hh - h * a.tiles);
  const int rows = min(a.group - g0, 16);  // query heads of this tile
  const int start = min(u.chunk * u.per, u.n), end = min(start + u.per, u.n);

  // Q^T: column j is head j (zero past the tile's heads)
  u32x4 qop[kQRegs];
  {
    const char* qp = reinterpret_cast<const char*>(a.q) +
                     (((size_t)u.b * a.kv_heads + h) * a.group + g0 + min(j, rows - 1)) * (D * kElem<DT>) + 16 * q;
#pragma unroll
    for (int c = 0; c < kQRegs; ++c) {
      const uint4 x = *reinterpret_cast<const uint4*>(qp + 64 * c);
      qop[c] = j < rows ? u32x4{x.x, x.y, x.z, x.w} : u32x4{0u, 0u, 0u, 0u};
    }
  }
  Acc<DT, D> acc;
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    acc.hi[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (DT != kFp32) acc.lo[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float m = -INFINITY, z = 0.f;  // head j's running maximum (exp2 domain), this lane's share of its sum

  const char* kh = reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes + 16 * q;
  const char* vh = reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes + j * (D * kElem<DT> / 16);
  const int32_t* tab = a.table + (size_t)u.b * a.max_pages;
  float* logits = a.logits ? a.logits + (((size_t)u.b * a.kv_heads + h) * a.group + g0 + j) * a.logit_stride : nullptr;
  bool bad = false;
  // row offset (16-byte units) of token t, the last token's past the end
  auto row_of = [&](int t) -> unsigned {
    t = min(t, end - 1);
    const int p = a.div.of(t);
    int page = tab[p];
    if ((unsigned)page >= (unsigned)a.pages) {
      bad = true;
      page = 0;
    }
    return (unsigned)page * a.page_units + (unsigned)(t - p * a.page_size) * a.slot_units;
  };

  int t0 = start + T::kTokens * w;
  unsigned row[T::kBlocks];
  if (t0 < end) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) row[i] = row_of(t0 + 16 * i + j);
  }
  while (t0 < end) {
    T t;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) t.k[i][c] = load_nt16(kh + ((size_t)row[i] << 4) + 64 * c);
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words(t.v[i][r], vh + ((size_t)(unsigned)__shfl((int)row[i], 4 * q + r) << 4));
    const int next = t0 + kPWaves * T::kTokens;
    if (next < end) {
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i) row[i] = row_of(next + 16 * i + j);
    }

    // scores: lane (j, q) gets tokens 16i + 4q + r of head j
    float s[T::kBlocks][4];
    float bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) {
        const u32x4 kw = {t.k[i][c].x, t.k[i][c].y, t.k[i][c].z, t.k[i][c].w};
        if constexpr (DT == kFp32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e]), __uint_as_float(qop[c][e]), d, 0, 0, 0);
        } else {
          d = mfma32<DT>(kw, qop[c], d);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = t0 + 16 * i + 4 * q + r < end ? d[r] * a.scale : -INFINITY;
        bm = fmaxf(bm, s[i][r]);
      }
      if (logits && j < rows)
        *reinterpret_cast<float4*>(logits + t0 + 16 * i + 4 * q) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    }
    bm = fmaxf(bm, xor16(bm));
    bm = fmaxf(bm, xor32(bm));
    if (__ballot(bm > m)) {
      const float nm = fmaxf(m, bm);
      const float alpha = m == nm ? 1.f : exp2_or_zero(m - nm);
      m = nm;
      z *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ah = __shfl(alpha, 4 * q + r);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          acc.hi[n][r] *= ah;
          if constexpr (DT != kFp32) acc.lo[n][r] *= ah;
        }
      }
    }
    float p[T::kBlocks][4];
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[i][r] = s[i][r] == -INFINITY ? 0.f : ldexpf(exp2f(s[i][r] - m), kBias<DT>);
        z += p[i][r];
      }
    if (t0 + T::kTokens > end) {  // rows past the end repeat the last one: 0 times its infinity must not be added
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + 16 * i + 4 * q + r >= end) {
#pragma unroll
            for (int n = 0; n < T::kVWords; ++n) t.v[i][r][n] = 0u;
          }
    }
    if constexpr (DT == kFp32) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
          acc.hi[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[0][r], __uint_as_float(t.v[0][r][n]), acc.hi[n], 0, 0, 0);
    } else {
      unsigned hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) split16<DT>(p[i][r], hi[4 * i + r], lo[4 * i + r]);
      const u32x4 ph = {hi[0] | hi[1] << 16, hi[2] | hi[3] << 16, hi[4] | hi[5] << 16, hi[6] | hi[7] << 16};
      const u32x4 pl = {lo[0] | lo[1] << 16, lo[2] | lo[3] << 16, lo[4] | lo[5] << 16, lo[6] | lo[7] << 16};
      pv_columns<0>(acc, t, ph, pl);
    }
    t0 = next;
  }
  if (__ballot(bad) && lane == 0) report_error(a.err, error_host_slot(a.err), kErrPages);

  // the waves' states meet in LDS
  float* sm = lds;                 // [waves][16] maxima
  float* sz = sm + 16 * kPWaves;   // [waves][16] sums
  float* sacc = sz + 16 * kPWaves; // [waves][rows][D]
  z += xor16(z);
  z += xor32(z);
  if (lane < 16) {
    sm[16 * w + j] = m;
    sz[16 * w + j] = z;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * q + r < rows) {
      float* dst = sacc + ((size_t)w * rows + 4 * q + r) * D + j * (D / 16);
#pragma unroll
      for (int n = 0; n < D / 16; n += 4) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = acc.hi[n + e][r];
          if constexpr (DT != kFp32) {
            const float rest = acc.lo[n + e][r];
            if (isfinite(rest)) x[e] += rest;
          }
        }
        *reinterpret_cast<float4*>(dst + n) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
  __syncthreads();
  const size_t head0 = ((size_t)u.b * a.kv_heads + h) * a.group + g0;  // this tile's first query head
  float* state = a.state + (size_t)blockIdx.x * a.state_stride;        // [rows]{max, sum} then [rows][D]
  for (int i = tid; i < rows * D; i += kPT) {
    const int g = i / D;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kPWaves; ++k) M = fmaxf(M, sm[16 * k + g]);
    float den = 0.f, x = 0.f;
#pragma unroll
    for (int k = 0; k < kPWaves; ++k) {
      const float wt = exp2_or_zero(sm[16 * k + g] == M ? (M == -INFINITY ? -INFINITY : 0.f) : sm[16 * k + g] - M);
      den = fmaf(wt, sz[16 * k + g], den);
      x = fmaf(wt, sacc[((size_t)k * rows) * D + i], x);
    }
    if (u.chunks == 1) {
      finish<DT, D>(a, head0, i, M, den, x);
    } else {
      if (i % D == 0) st_dev2(state + 2 * g, M, den);
      st_dev(state + 2 * rows + i, x);
    }
  }
  if (u.chunks == 1) return;

  // the last workgroup of this (sequence, head tile) joins the chunks
  int* last = reinterpret_cast<int*>(lds);
  drain();
  __syncthreads();
  unsigned* counter = a.counters + (size_t)u.b * a.kv_heads * a.tiles + u.hh;
  if (tid == 0) *last = inc_dev(counter) == (unsigned)(u.chunks - 1);
  __syncthreads();
  const int is_last = *last;
  __syncthreads();
  if (!is_last) return;
  if (tid == 0) st_dev(counter, 0u);
  const size_t step = (size_t)a.kv_heads * a.tiles * a.state_stride;  // between a sequence's chunks
  const float* st0 = state - (size_t)u.chunk * step;
  for (int i = tid; i < rows * D; i += kPT) {
    const int g = i / D;
    float M = -INFINITY, den = 0.f, x = 0.f;
    for (int c0 = 0; c0 < u.chunks; c0 += 8) {
      float2 mz[8];
      float xv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float* st = st0 + (size_t)min(c0 + e, u.chunks - 1) * step;
        mz[e] = ld_dev2(st + 2 * g);
        xv[e] = ld_dev(st + 2 * rows + i);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (c0 + e >= u.chunks) break;
        const float nM = fmaxf(M, mz[e].x);
        const float old = M == nM ? 1.f : exp2_or_zero(M - nM);
        const float wt = mz[e].x == nM ? (nM == -INFINITY ? 0.f : 1.f) : exp2_or_zero(mz[e].x - nM);
        den = fmaf(wt, mz[e].y, den * old);
        x = fmaf(wt, xv[e], x * old);
        M = nM;
      }
    }
    finish<DT, D>(a, head0, i, M, den, x);
  }
}

// scores_out[t] = scores[t] + sum over the group's heads of e^(s_t - lse): one
// thread per slot, bound by the scores it reads (4 bytes per query head) and
// the two score arrays.
__global__ __launch_bounds__(kPT) void paged_weigh_kernel(PagedAttend a) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = clamp_length(a, a.lengths[b]);
  const float* lse = a.lse_work + ((size_t)b * a.kv_heads + h) * a.group;
  const float* logits = a.logits + ((size_t)b * a.kv_heads + h) * a.group * a.logit_stride;
  const size_t at = ((size_t)b * a.kv_heads + h) * a.slots;
  for (int t = blockIdx.x * kPT + threadIdx.x; t < n; t += gridDim.x * kPT) {
    float sum = 0.f;
    for (int g = 0; g < a.group; ++g) {
      const float l = lse[g], s = logits[(size_t)g * a.logit_stride + t];
      sum += s == -INFINITY ? 0.f : exp2f(s - l);
    }
    a.scores_out[at + t] = a.scores[at + t] + sum;
  }
}

// ------------------------------------------------------------------ append
//
// A copy of rows: bound by reading and writing them.  One workgroup per
// sequence (one token each) or per kAppendRows packed rows, 16 bytes per thread
// and step.

constexpr int kAppendRows = 4;

__device__ __forceinline__ void append_row(const PagedAppend& a, int64_t row, int b, int slot, int position) {
  const int p = a.div.of(slot);
  const bool room = p < a.max_pages;
  const int page = room ? a.table[(size_t)b * a.max_pages + p] : -1;
  if ((unsigned)page >= (unsigned)a.pages) {  // no page: the row is dropped
    if (threadIdx.x == 0) report_error(a.err, error_host_slot(a.err), kErrPages);
    return;
  }
  const size_t at = (size_t)page * a.page_bytes + (size_t)(slot - p * a.page_size) * a.slot_bytes;
  const int pieces = a.row_bytes >> 4;
  for (int i = threadIdx.x; i < a.kv_heads * pieces; i += kPT) {
    const int h = i / pieces, c = (i - h * pieces) << 4;
    const uint4 kv = *reinterpret_cast<const uint4*>(a.k + row * a.k_row + (int64_t)h * a.k_head + c);
    const uint4 vv = *reinterpret_cast<const uint4*>(a.v + row * a.v_row + (int64_t)h * a.v_head + c);
    *reinterpret_cast<uint4*>(a.kp + at + (size_t)h * a.head_bytes + c) = kv;
    *reinterpret_cast<uint4*>(a.vp + at + (size_t)h * a.head_bytes + c) = vv;
  }
  if (a.positions)
    for (int h = threadIdx.x; h < a.kv_heads; h += kPT) {
      const size_t i = ((size_t)b * a.kv_heads + h) * a.slots + slot;
      a.scores[i] = a.scores_out[i] = 0.f;
      a.positions[i] = a.positions_out[i] = position;
    }
}

__global__ __launch_bounds__(kPT) void paged_append_kernel(PagedAppend a) {
  if (!a.offsets) {  // one token each: row b
    const int b = blockIdx.x;
    const int n = max(a.lengths[b], 0), seen = a.positions ? a.seen[b] : 0;
    __syncthreads();  // every thread has read the length before it moves
    append_row(a, b, b, n, seen);
    if (threadIdx.x == 0) {
      a.lengths_out[b] = min(n, a.slots) + (n < a.slots);
      if (a.positions) a.seen_out[b] = seen + 1;
    }
    return;
  }
  const int64_t row0 = (int64_t)blockIdx.x * kAppendRows;
  int b = 0;
  {  // the sequence of row0: the last b with offsets[b] <= row0
    int lo = 0, hi = a.sequences;
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.offsets[mid] <= row0) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  for (int r = 0; r < kAppendRows && row0 + r < a.rows; ++r) {
    const int64_t row = row0 + r;
    while (b + 1 < a.sequences && a.offsets[b + 1] <= row) ++b;
    const int64_t step = row - a.offsets[b];
    if (step < 0 || row >= a.offsets[b + 1]) continue;  // a row of no sequence
    const int64_t slot = max(a.lengths[b], 0) + step;
    append_row(a, row, b, (int)min(slot, (int64_t)a.slots), a.positions ? a.seen[b] + (int)step : 0);
  }
}

__global__ __launch_bounds__(kPT) void paged_advance_kernel(PagedAppend a) {
  const int b = blockIdx.x * kPT + threadIdx.x;
  if (b >= a.sequences) return;
  const int more = max(a.offsets[b + 1] - a.offsets[b], 0);
  a.lengths_out[b] = (int)min((int64_t)max(a.lengths[b], 0) + more, (int64_t)a.slots);
  if (a.positions) a.seen_out[b] = a.seen[b] + more;
}

// ------------------------------------------------------------------ eviction

constexpr int kET = 1024;  // threads of the selection
constexpr int kEWaves = kET / 64;

// The order of the slots as an unsigned key: protected above NaN above the
// numbers (-0 as 0).
__device__ __forceinline__ unsigned evict_key(const PagedEvict& a, float score, const int32_t* positions, int edge, int t) {
  if (a.guard) {
    const int p = positions[t];
    if (p >= edge || p < a.sinks) return 0xffffffffu;
  }
  if (score != score) return 0xfffffffeu;
  const unsigned u = __float_as_uint(score == 0.f ? 0.f : score);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_keep(const PagedEvict& a, int b) {
  const int keep = a.keeps ? a.keeps[b] : a.keep;
  return max(keep, 0);
}

// One workgroup per (sequence, KV head): the budget-th largest key by three
// histogram passes (11, 11 and 10 bits), then the slots that move: holes
// (evicted slots before the budget) and sources (kept slots behind it), both
// ascending, found by each wave in its own share of the slots.
__global__ __launch_bounds__(kET) void paged_select_kernel(PagedEvict a) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  __shared__ unsigned hist[2048], wsum[kEWaves];
  __shared__ unsigned found[2];  // the digit of the threshold, what remains of the budget
  __shared__ int ties[kEWaves], holes[kEWaves], sources[kEWaves];
  const int n = min(max(a.lengths[b], 0), a.slots), m = min(n, evict_keep(a, b));
  const size_t row = (size_t)b * a.kv_heads + h;
  const float* scores = a.scores + row * a.slots;
  const int32_t* positions = a.positions + row * a.slots;
  const int edge = a.seen[b] - a.recent;
  int* count = a.count + row;
  const bool apart = a.scores_out != a.scores;
  if (apart)  // what stays where it is; the moves overwrite the holes
    for (int t = tid; t < m; t += kET) {
      a.scores_out[row * a.slots + t] = scores[t];
      a.positions_out[row * a.slots + t] = positions[t];
    }
  if (n <= m || m == 0) {
    if (tid == 0) *count = 0;
    return;
  }
  unsigned prefix = 0, need = m;  // the need-th largest of the keys whose top bits equal prefix
  int shift = 21;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    for (int i = tid; i < 2048; i += kET) hist[i] = 0u;
    __syncthreads();
    for (int t = tid; t < n; t += kET) {
      const unsigned key = evict_key(a, scores[t], positions, edge, t);
      if (pass == 0 || key >> (shift + bits) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // thread i owns bins 2i and 2i + 1 from the top
    const unsigned hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
    const unsigned incl = block_incl_scan<kET>(hi + lo, wsum), before = incl - hi - lo;
    if (before < need && need <= incl) {
      const bool upper = need <= before + hi;
      found[0] = upper ? 2047 - 2 * tid : 2046 - 2 * tid;
      found[1] = need - before - (upper ? 0u : hi);
    }
    __syncthreads();
    prefix = pass == 2 ? (prefix << 10) | found[0] : (prefix << 11) | found[0];
    need = found[1];
    shift = pass == 0 ? 10 : 0;
    __syncthreads();
  }
  // kept: keys above `prefix`, and the first `need` slots whose key equals it
  const int share = ((n + kEWaves - 1) / kEWaves + 63) & ~63;
  const int lo = min(w * share, n), hi = min(lo + share, n);
  int mine = 0;
  for (int t = lo + lane; t < hi; t += 64) mine += evict_key(a, scores[t], positions, edge, t) == prefix;
  mine = wave_sum_i(mine);
  if (lane == 0) ties[w] = mine;
  __syncthreads();
  int tie0 = 0;
  for (int k = 0; k < w; ++k) tie0 += ties[k];
  const unsigned long long below = (1ull << lane) - 1ull;
  int hole0 = 0, source0 = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int tie = tie0, nh = 0, ns = 0;
    for (int t0 = lo; t0 < hi; t0 += 64) {
      const int t = t0 + lane;
      const bool live = t < hi;
      const unsigned key = live ? evict_key(a, scores[t], positions, edge, t) : 0u;
      const unsigned long long eq = __ballot(live && key == prefix);
      const bool kept = live && (key > prefix || (key == prefix && tie + __popcll(eq & below) < (int)need));
      tie += __popcll(eq);
      const unsigned long long hm = __ballot(live && t < m && !kept), sm = __ballot(kept && t >= m);
      if (pass == 1) {
        if (hm >> lane & 1) a.dst[row * a.moves + hole0 + nh + __popcll(hm & below)] = t;
        if (sm >> lane & 1) a.src[row * a.moves + source0 + ns + __popcll(sm & below)] = t;
      }
      nh += __popcll(hm);
      ns += __popcll(sm);
    }
    if (pass == 0) {
      if (lane == 0) {
        holes[w] = nh;
        sources[w] = ns;
      }
      __syncthreads();
      int total = 0;
      for (int k = 0; k < kEWaves; ++k) {
        if (k < w) {
          hole0 += holes[k];
          source0 += sources[k];
        }
        total += holes[k];
      }
      if (tid == 0) *count = total;
    }
  }
}

// Moves the kept rows into the holes: a copy, bound by the rows it reads and
// writes.  No source is another move's destination.
__global__ __launch_bounds__(kPT) void paged_move_kernel(PagedEvict a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const size_t row = (size_t)b * a.kv_heads + h;
  const int count = a.count[row];
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    a.lengths_out[b] = min(min(max(a.lengths[b], 0), a.slots), evict_keep(a, b));
    if (a.seen_out != a.seen) a.seen_out[b] = a.seen[b];
  }
  const int pieces = a.row_bytes >> 4;
  const int32_t* tab = a.table + (size_t)b * a.max_pages;
  for (int i = blockIdx.x * kPT + threadIdx.x; i < count * pieces; i += gridDim.x * kPT) {
    const int k = i / pieces, c = (i - k * pieces) << 4;
    const int src = a.src[row * a.moves + k], dst = a.dst[row * a.moves + k];
    const int ps = a.div.of(src), pd = a.div.of(dst);
    const int from = tab[ps], to = tab[pd];
    if ((unsigned)from >= (unsigned)a.pages || (unsigned)to >= (unsigned)a.pages) {
      report_error(a.err, error_host_slot(a.err), kErrPages);
      continue;
    }
    const size_t f = (size_t)from * a.page_bytes + (size_t)(src - ps * a.page_size) * a.slot_bytes +
                     (size_t)h * a.head_bytes + c;
    const size_t t = (size_t)to * a.page_bytes + (size_t)(dst - pd * a.page_size) * a.slot_bytes +
                     (size_t)h * a.head_bytes + c;
    const uint4 kv = *reinterpret_cast<const uint4*>(a.kp + f);
    const uint4 vv = *reinterpret_cast<const uint4*>(a.vp + f);
    *reinterpret_cast<uint4*>(a.kp + t) = kv;
    *reinterpret_cast<uint4*>(a.vp + t) = vv;
    if (c == 0) {
      a.scores_out[row * a.slots + dst] = a.scores[row * a.slots + src];
      a.positions_out[row * a.slots + dst] = a.positions[row * a.slots + src];
    }
  }
}

}  // namespace
}  // namespace prismkv

using namespace prismkv;

namespace {

PageDiv page_div(int page_size) {
  int log = 0;
  while ((1ll << log) < page_size) ++log;
  const int shift = 31 + log;
  return PageDiv{(unsigned)(((1ull << shift) + page_size - 1) / page_size), shift};
}

int element_bytes(int dtype) { return dtype == kFp32 ? 4 : 2; }

// Sizes that every entry point takes, checked alike.  Strides are in elements;
// rows, heads and pages lie at 16-byte multiples, and a page's last row within
// 2^32 16-byte units.
bool bad_cache(int sequences, int kv_heads, int head_dim, int page_size, int max_pages, int64_t pages, int64_t page_stride,
               int64_t head_stride, int64_t slot_stride, int dtype) {
  if (sequences < 1 || sequences > 65535 || kv_heads < 1 || kv_heads > 65535 || page_size < 1 || max_pages < 1 ||
      pages < 1 || pages > INT32_MAX)
    return true;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return true;
  const int64_t slots = (int64_t)page_size * max_pages;
  if (slots > (1 << 30) || slots * sequences > INT32_MAX) return true;
  const int64_t es = element_bytes(dtype);
  if (page_stride < 0 || head_stride < 0 || slot_stride < head_dim) return true;
  if ((page_stride * es | head_stride * es | slot_stride * es) & 15) return true;
  const int64_t limit = 1ll << 36;  // bytes
  if (page_stride > limit || head_stride > limit || slot_stride > limit) return true;
  if (page_stride * es > limit / pages || slot_stride * es > limit / page_size) return true;
  if ((pages - 1) * page_stride * es + (page_size - 1) * slot_stride * es >= limit) return true;
  return false;
}

struct WorkLayout {
  size_t lse, state, logits, bytes;  // counters first
  unsigned state_stride;
  int64_t logit_stride, units;
};

WorkLayout attend_layout(int sequences, int kv_heads, int group, int head_dim, int64_t slots, bool weigh) {
  WorkLayout w;
  const int64_t tiles = (group + 15) / 16, heads = (int64_t)kv_heads * tiles;
  // no sequence has more chunks than its longest table allows
  const int64_t most = sequences * heads * ((slots + 32 * kPWaves - 1) / (32 * kPWaves));
  w.units = (int64_t)sequences * heads + (1 << kLogUnits);
  if (most < w.units) w.units = most;
  w.state_stride = (unsigned)((group < 16 ? group : 16) * (head_dim + 2));
  w.logit_stride = (slots + 31) & ~31ll;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  w.lse = up((size_t)sequences * heads * sizeof(unsigned));
  w.state = w.lse + up((size_t)sequences * kv_heads * group * sizeof(float));
  w.logits = w.state + up((size_t)w.units * w.state_stride * sizeof(float));
  w.bytes = w.logits + (weigh ? (size_t)sequences * kv_heads * group * w.logit_stride * sizeof(float) : 0);
  return w;
}

template <int DT, int D>
int launch_attend(const PagedAttend& a, int64_t units, hipStream_t stream) {
  const int rows = a.group < 16 ? a.group : 16;
  const int lds = (32 * kPWaves + kPWaves * rows * D) * (int)sizeof(float);
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_attend_kernel<DT, D>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (32 * kPWaves + kPWaves * 16 * D) * (int)sizeof(float));
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((paged_attend_kernel<DT, D>), dim3((unsigned)units), dim3(kPT), lds, stream, a);
  return (int)hipGetLastError();
}

template <int DT>
int launch_attend_dim(const PagedAttend& a, int head_dim, int64_t units, hipStream_t stream) {
  if (head_dim == 64) return launch_attend<DT, 64>(a, units, stream);
  if (head_dim == 128) return launch_attend<DT, 128>(a, units, stream);
  return launch_attend<DT, 256>(a, units, stream);
}

}  // namespace

extern "C" {

size_t prismkv_paged_attend_work_bytes(int sequences, int kv_heads, int group, int head_dim, int64_t slots, int weigh) {
  if (sequences < 1 || kv_heads < 1 || group < 1 || head_dim < 1 || slots < 1) return 0;
  return attend_layout(sequences, kv_heads, group, head_dim, slots, weigh != 0).bytes;
}

int prismkv_paged_attend(uint64_t q, uint64_t k, uint64_t v, uint64_t table, uint64_t lengths, uint64_t scores,
                         uint64_t scores_out, uint64_t lse, uint64_t paged_work, uint64_t err, uint64_t out, int sequences,
                         int kv_heads, int group, int head_dim, int page_size, int max_pages, int64_t pages,
                         int64_t page_stride, int64_t head_stride, int64_t slot_stride, double scale, int dtype,
                         size_t work_bytes, uint64_t stream) {
  if (dtype < kBf16 || dtype > kFp32) return kBadMode;
  if (bad_cache(sequences, kv_heads, head_dim, page_size, max_pages, pages, page_stride, head_stride, slot_stride, dtype))
    return kBadSize;
  if (group < 1 || group > 1024 || !(scale == scale)) return kBadSize;
  if (!q || !k || !v || !table || !lengths || !paged_work || !err || !out || !scores != !scores_out) return kBadSize;
  if ((q | k | v | paged_work) & 15 || (table | lengths | scores | scores_out | lse) & 3 || err & 7) return kBadSize;
  const int64_t slots = (int64_t)page_size * max_pages;
  const WorkLayout w = attend_layout(sequences, kv_heads, group, head_dim, slots, scores != 0);
  if (work_bytes < w.bytes || w.units > INT32_MAX) return kBadSize;
  const int es = element_bytes(dtype);
  PagedAttend a{};
  a.q = reinterpret_cast<const void*>(q);
  a.k = reinterpret_cast<const void*>(k);
  a.v = reinterpret_cast<const void*>(v);
  a.table = reinterpret_cast<const int32_t*>(table);
  a.lengths = reinterpret_cast<const int32_t*>(lengths);
  a.scores = reinterpret_cast<const float*>(scores);
  a.scores_out = reinterpret_cast<float*>(scores_out);
  a.lse_out = reinterpret_cast<float*>(lse);
  a.out = reinterpret_cast<void*>(out);
  char* work = reinterpret_cast<char*>(paged_work);
  a.counters = reinterpret_cast<unsigned*>(work);
  a.state = reinterpret_cast<float*>(work + w.state);
  if (scores) {
    a.lse_work = reinterpret_cast<float*>(work + w.lse);
    a.logits = reinterpret_cast<float*>(work + w.logits);
  }
  a.err = reinterpret_cast<unsigned*>(err);
  a.head_bytes = head_stride * es;
  a.logit_stride = w.logit_stride;
  a.slots = slots;
  a.page_units = (unsigned)(page_stride * es >> 4);
  a.slot_units = (unsigned)(slot_stride * es >> 4);
  a.state_stride = w.state_stride;
  a.div = page_div(page_size);
  a.sequences = sequences;
  a.kv_heads = kv_heads;
  a.group = group;
  a.tiles = (group + 15) / 16;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.scale = (float)(scale * 1.4426950408889634);
  const hipStream_t s = (hipStream_t)stream;
  int rc;
  if (dtype == kBf16) rc = launch_attend_dim<kBf16>(a, head_dim, w.units, s);
  else if (dtype == kFp16) rc = launch_attend_dim<kFp16>(a, head_dim, w.units, s);
  else rc = launch_attend_dim<kFp32>(a, head_dim, w.units, s);
  if (rc || !scores) return rc;
  const int64_t blocks = (slots + kPT - 1) / kPT;
  hipLaunchKernelGGL(paged_weigh_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), kv_heads, sequences), dim3(kPT), 0,
                     s, a);
  return (int)hipGetLastError();
}

int prismkv_paged_append(uint64_t k, uint64_t v, uint64_t k_pages, uint64_t v_pages, uint64_t table, uint64_t offsets,
                         uint64_t lengths, uint64_t lengths_out, uint64_t seen, uint64_t seen_out, uint64_t scores,
                         uint64_t scores_out, uint64_t positions, uint64_t positions_out, uint64_t err, int64_t rows,
                         int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                         int sequences, int kv_heads, int head_dim, int page_size, int max_pages, int64_t pages,
                         int64_t page_stride, int64_t head_stride, int64_t slot_stride, int dtype, uint64_t stream) {
  if (dtype < kBf16 || dtype > kFp32) return kBadMode;
  if (bad_cache(sequences, kv_heads, head_dim, page_size, max_pages, pages, page_stride, head_stride, slot_stride, dtype))
    return kBadSize;
  if (rows < 0 || rows > INT32_MAX || (!offsets && rows != sequences)) return kBadSize;
  if (!k_pages || !v_pages || !table || !lengths || !lengths_out || !err || (rows && (!k || !v))) return kBadSize;
  const bool scored = positions != 0;
  if (scored && (!positions_out || !scores || !scores_out || !seen || !seen_out)) return kBadSize;
  const int es = element_bytes(dtype);
  if ((k | v | k_pages | v_pages) & 15 || err & 7 ||
      (table | offsets | lengths | lengths_out | seen | seen_out | scores | scores_out | positions | positions_out) & 3)
    return kBadSize;
  if ((k_row_stride * es | k_head_stride * es | v_row_stride * es | v_head_stride * es) & 15) return kBadSize;
  PagedAppend a{};
  a.k = reinterpret_cast<const char*>(k);
  a.v = reinterpret_cast<const char*>(v);
  a.kp = reinterpret_cast<char*>(k_pages);
  a.vp = reinterpret_cast<char*>(v_pages);
  a.table = reinterpret_cast<const int32_t*>(table);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
  a.lengths = reinterpret_cast<const int32_t*>(lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(lengths_out);
  a.seen = reinterpret_cast<const int32_t*>(seen);
  a.seen_out = reinterpret_cast<int32_t*>(seen_out);
  a.positions = reinterpret_cast<int32_t*>(positions);
  a.positions_out = reinterpret_cast<int32_t*>(positions_out);
  a.scores = reinterpret_cast<float*>(scores);
  a.scores_out = reinterpret_cast<float*>(scores_out);
  a.err = reinterpret_cast<unsigned*>(err);
  a.rows = rows;
  a.k_row = k_row_stride * es;
  a.k_head = k_head_stride * es;
  a.v_row = v_row_stride * es;
  a.v_head = v_head_stride * es;
  a.page_bytes = page_stride * es;
  a.head_bytes = head_stride * es;
  a.slot_bytes = slot_stride * es;
  a.div = page_div(page_size);
  a.sequences = sequences;
  a.kv_heads = kv_heads;
  a.row_bytes = head_dim * es;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.slots = page_size * max_pages;
  const hipStream_t s = (hipStream_t)stream;
  if (!offsets) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(sequences), dim3(kPT), 0, s, a);
    return (int)hipGetLastError();
  }
  if (rows) {
    hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)((rows + kAppendRows - 1) / kAppendRows)), dim3(kPT), 0, s, a);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  hipLaunchKernelGGL(paged_advance_kernel, dim3((sequences + kPT - 1) / kPT), dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

size_t prismkv_paged_evict_work_bytes(int sequences, int kv_heads, int64_t slots) {
  if (sequences < 1 || kv_heads < 1 || slots < 1) return 0;
  return (size_t)sequences * kv_heads * (1 + 2 * (size_t)(slots / 2 + 1)) * sizeof(int32_t);
}

int prismkv_paged_evict(uint64_t k_pages, uint64_t v_pages, uint64_t table, uint64_t lengths, uint64_t lengths_out,
                        uint64_t seen, uint64_t seen_out, uint64_t scores, uint64_t scores_out, uint64_t positions,
                        uint64_t positions_out, uint64_t keeps, uint64_t paged_work, uint64_t err, int keep, int recent,
                        int sinks, int sequences, int kv_heads, int head_dim, int page_size, int max_pages, int64_t pages,
                        int64_t page_stride, int64_t head_stride, int64_t slot_stride, int dtype, size_t work_bytes,
                        uint64_t stream) {
  if (dtype < kBf16 || dtype > kFp32) return kBadMode;
  if (bad_cache(sequences, kv_heads, head_dim, page_size, max_pages, pages, page_stride, head_stride, slot_stride, dtype))
    return kBadSize;
  if (keep < 0 || recent < 0 || sinks < 0 || (keeps && keep)) return kBadSize;
  if (!k_pages || !v_pages || !table || !lengths || !lengths_out || !seen || !seen_out || !scores || !scores_out ||
      !positions || !positions_out || !paged_work || !err)
    return kBadSize;
  if ((k_pages | v_pages) & 15 || err & 7 ||
      (table | lengths | lengths_out | seen | seen_out | scores | scores_out | positions | positions_out | keeps |
       paged_work) & 3)
    return kBadSize;
  const int64_t slots = (int64_t)page_size * max_pages;
  if (work_bytes < prismkv_paged_evict_work_bytes(sequences, kv_heads, slots)) return kBadSize;
  const int es = element_bytes(dtype);
  PagedEvict a{};
  a.kp = reinterpret_cast<char*>(k_pages);
  a.vp = reinterpret_cast<char*>(v_pages);
  a.table = reinterpret_cast<const int32_t*>(table);
  a.lengths = reinterpret_cast<const int32_t*>(lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(lengths_out);
  a.seen = reinterpret_cast<const int32_t*>(seen);
  a.seen_out = reinterpret_cast<int32_t*>(seen_out);
  a.scores = reinterpret_cast<const float*>(scores);
  a.scores_out = reinterpret_cast<float*>(scores_out);
  a.positions = reinterpret_cast<const int32_t*>(positions);
  a.positions_out = reinterpret_cast<int32_t*>(positions_out);
  a.keeps = reinterpret_cast<const int32_t*>(keeps);
  a.moves = slots / 2 + 1;
  a.count = reinterpret_cast<int32_t*>(paged_work);
  a.src = a.count + (size_t)sequences * kv_heads;
  a.dst = a.src + (size_t)sequences * kv_heads * a.moves;
  a.err = reinterpret_cast<unsigned*>(err);
  a.page_bytes = page_stride * es;
  a.head_bytes = head_stride * es;
  a.slot_bytes = slot_stride * es;
  a.div = page_div(page_size);
  a.sequences = sequences;
  a.kv_heads = kv_heads;
  a.row_bytes = head_dim * es;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.slots = (int)slots;
  a.keep = keep;
  a.recent = recent;
  a.sinks = sinks;
  a.guard = recent > 0 || sinks > 0;
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(paged_select_kernel, dim3(kv_heads, sequences), dim3(kET), 0, s, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  const int64_t pieces = (int64_t)(head_dim * es >> 4) * (slots / 2 + 1);
  const int64_t blocks = (pieces + kPT - 1) / kPT;
  hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)(blocks < 64 ? blocks : 64), kv_heads, sequences), dim3(kPT), 0, s,
                     a);
  return (int)hipGetLastError();
}

}  // extern "C"
