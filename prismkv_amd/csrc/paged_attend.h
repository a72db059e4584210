// Attention of one new query token of every sequence over its pages: the
// kernels, for the sources that instantiate them (paged.hip over pages of
// the rows' own type, paged4.hip over pages in 4 bits).
#pragma once

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
// Split: the tokens of all pairs of a sequence and a KV head (with more than 16
// query heads a tile of them) are dealt evenly to the workgroups, on the device,
// where the lengths are; a workgroup's share may end one pair and begin others.
// Each of its waves takes every 8th 32-token tile (fp32: 16 tokens) by itself: no
// barrier and no LDS until the waves' states meet at a pair's end.  A pair of
// several workgroups is joined from their states in the order of its tokens, by
// the last to arrive or by a second launch, so the result does not depend on the
// order of arrival.
//
// Measured (MI355X, launches after one another in a graph): 65792 tokens, 8 x 4
// heads, bf16, 47.3 us = 5.7 TB/s; 32 sequences of 6.4K tokens 136 us = 6.2 TB/s
// (a plain read of as much memory reaches 6.9); 16 x 8192 of head_dim 256 in fp32, 2
// x 4 heads, 92 us = 5.9; of head_dim 64, 8 x 4 heads, 48 us = 5.6; 75 tokens 6.4 us.
// About 6 us of a call are the launch and the chain lengths -> page -> rows, 3.7 more
// the join (65792 tokens 43.7 us without it).

// 16-bit types: P is a sum of terms of the type, each with a product of its own into
// one accumulator: bf16 takes three, which hold all 24 bits of an fp32 p (with two,
// outputs that cancel are off by 2^-17 of their terms; 65792 tokens, 8 x 4 heads take
// as long with either), fp16 two, 22 bits.  Every term is positive wherever p is, so
// that an infinite V is not multiplied by a term of 0: at least the type's least
// number, which for fp16, with its bias, is 2^-39 of the maximum's weight.
// The tile of one step as loaded.  16-bit (32 tokens, two 16-token blocks):
// lane (j, q) holds row j of each block at dims 32c + 8q .. +8 (K, the A operand
// of the 16x16x32 product) and of rows 4q + t (V) 16 bytes out of every 256 (8 of
// head_dim 64's 128), so that the 16 lanes of a load cover whole rows.  Column
// block n of the output takes element n of a lane, dim(n, j); the rows' pairs are
// joined per dim with one byte permutation.
// fp32 (16 tokens): K dims 16c + 4q .. +4 (four 16x16x4 products per load), V
// the same with float columns.
template <int DT, int D>
struct Tile {
  static constexpr int kBlocks = kType<DT> == kFp32 ? 1 : 2;
  static constexpr int kTokens = 16 * kBlocks;
  static constexpr int kKLoads = D * kElem<DT> / 64;        // 16-byte loads of a K row per lane
  static constexpr int kVWords = D * kElem<DT> / 64;        // 32-bit words of a V row per lane
  static constexpr int kVStep = kVWords < 4 ? 4 * kVWords : 16;  // bytes of a piece
  static constexpr int kRun = kVStep / kElem<DT>;           // elements of a piece
  static __device__ __forceinline__ int dim(int n, int j) { return n / kRun * (16 * kRun) + j * kRun + n % kRun; }
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
      const uint4 x = load_nt16(p + 64 * i);
      dst[i] = x.x;
      dst[i + 1] = x.y;
      dst[i + 2] = x.z;
      dst[i + 3] = x.w;
    }
  }
}

template <int W>
__device__ __forceinline__ void load_words_buf(unsigned (&dst)[W], __amdgpu_buffer_rsrc_t r, unsigned byte_offset) {
  if constexpr (W == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, byte_offset, 0, 2);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 x = load_nt16_buf(r, byte_offset + 64 * i);
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
  if constexpr (kType<DT> == kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// p >= 0 as terms of the 16-bit type, each in the upper half of a word.  A NaN may be
// lost here: the sum of the weights has it.
template <int DT>
constexpr int kTerms = kType<DT> == kBf16 ? 3 : 2;
template <int DT>
__device__ __forceinline__ void split16(float p, unsigned (&term)[kTerms<DT>]) {
  if constexpr (kType<DT> == kBf16) {
    // 8 bits each from the top, which is exact (as signed integers: a remainder
    // below 0 is left behind a term that was raised)
    const int least = p > 0.f ? 0x10000 : 0;
    const int hi = max(__float_as_int(p) & (int)0xffff0000, least);
    const float rest = p - __int_as_float(hi);
    const int mid = max(__float_as_int(rest) & (int)0xffff0000, least);
    term[0] = (unsigned)hi;
    term[1] = (unsigned)mid;
    term[2] = (unsigned)max(__float_as_int(rest - __int_as_float(mid)), least);
  } else {
    // the head rounded down, so that the remainder is positive
    const float least = p > 0.f ? 0x1p-24f : 0.f, head = fmaxf(p, least);
    const auto h = __builtin_amdgcn_cvt_pkrtz(0.f, head);  // {0, head}
    const _Float16 l = (_Float16)fmaxf(head - (float)h[1], least);
    term[0] = __builtin_bit_cast(unsigned, h);
    term[1] = (unsigned)__builtin_bit_cast(unsigned short, l) << 16;
  }
}

// The upper halves of two words (low half from a).
__device__ __forceinline__ unsigned upper16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Two of them as word w of each term's operand, where no V is infinite (in 4 bits): a
// term may be 0.
template <int DT>
__device__ __forceinline__ void split_pair(float a, float b, u32x4 (&term)[kTerms<DT>], int w) {
  if constexpr (kType<DT> == kBf16) {
    const unsigned a0 = __float_as_uint(a) & 0xffff0000u, b0 = __float_as_uint(b) & 0xffff0000u;
    const float ra = a - __uint_as_float(a0), rb = b - __uint_as_float(b0);
    const unsigned a1 = __float_as_uint(ra) & 0xffff0000u, b1 = __float_as_uint(rb) & 0xffff0000u;
    term[0][w] = upper16(a0, b0);
    term[1][w] = upper16(a1, b1);
    term[2][w] = upper16(__float_as_uint(ra - __uint_as_float(a1)), __float_as_uint(rb - __uint_as_float(b1)));
  } else {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    term[0][w] = __builtin_bit_cast(unsigned, h);
    term[1][w] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]));
  }
}

template <int N, int DT, int D, int W>
__device__ __forceinline__ void pv_columns(f32x4 (&acc)[D / 16], const unsigned (&v)[2][4][W],
                                           const u32x4 (&p)[kTerms<DT>]) {
  if constexpr (N < D / 16) {
    const u32x4 vb = {pair16<N>(v[0][0], v[0][1]), pair16<N>(v[0][2], v[0][3]), pair16<N>(v[1][0], v[1][1]),
                      pair16<N>(v[1][2], v[1][3])};
#pragma unroll
    for (int i = 0; i < kTerms<DT>; ++i) acc[N] = mfma32<DT>(p[i], vb, acc[N]);
    pv_columns<N + 1, DT, D>(acc, v, p);
  }
}

// 2^(scale s - m): one rounding of the difference.  m is a rounded product itself;
// from 2^22 on, where its rounding is 1/8 and more (and at 2^32 takes all of the
// exponent's range), the other products are rounded as it was, so that the largest
// score's weight is 1.  m is finite or +infinity (no_less): where no score is above
// -infinity, 0 serves.
__device__ __forceinline__ float weight(float s, float scale, float m) {
#pragma clang fp contract(off)
  const float product = s * scale;
  const float rounded = product - m;
  return __builtin_amdgcn_exp2f(fabsf(m) < 0x1p22f ? fmaf(s, scale, -m) : rounded);
}
__device__ __forceinline__ float no_less(float m) { return m == -INFINITY ? 0.f : m; }

// Factor of a state with maximum m under the joint maximum M >= m (no state: 0).
__device__ __forceinline__ float rescale(float m, float M) {
  return m == -INFINITY ? 0.f : m == M ? 1.f : exp2f(m - M);
}

// The joint maximum and sum of a pair's head g over its states, and the states'
// factors in wt[c * stride] (LDS); by one wave.
__device__ __forceinline__ float2 join_sums(const float* base, const PagedParts& parts, unsigned state_stride, int g,
                                            float* wt, int stride) {
  const int lane = threadIdx.x & 63;
  float M = -INFINITY, den = 0.f;
  for (int c0 = 0; c0 < parts.chunks; c0 += 64) {
    const int c = c0 + lane;
    const bool in = c < parts.chunks;
    const float2 mz = ld_dev2(base + (in && c ? 2 * c : parts.odd) * state_stride + 2 * g);
    const float m = in ? mz.x : -INFINITY;
    const float nM = fmaxf(M, wave_max(m));
    den = den * rescale(M, nM) + wave_sum(in ? rescale(m, nM) * mz.y : 0.f);
    M = nM;
    if (in && wt) wt[c * stride] = m;
  }
  if (wt)
    for (int c = lane; c < parts.chunks; c += 64) wt[c * stride] = rescale(wt[c * stride], M);
  return make_float2(M, den);
}

// Joins columns [col0, col0 + columns) (4 floats each of the [rows][D] output) of a
// pair's states, by a workgroup of kThreads: the maxima and sums a wave per head,
// while the first states' loads are in flight, then a thread per column and share
// of the states, the shares added in LDS.
template <int DT, int D, int kThreads>
__device__ __forceinline__ void join_states(const PagedAttend& a, size_t head0, int rows, const PagedParts& parts, int col0,
                                            int columns, float* lds) {
  const int tid = threadIdx.x, w = tid >> 6;
  float4* part = reinterpret_cast<float4*>(lds);  // [threads]
  float* top = lds + 4 * kThreads;                // [16] joint maxima, [16] sums
  float* wt = top + 32;                           // [chunks][rows] factors
  const float* base = a.state + (size_t)2 * parts.unit * a.state_stride;
  const __amdgpu_buffer_rsrc_t r = raw_buffer(base, 2 * parts.chunks * (int)a.state_stride * 4);
  const int chunks = parts.chunks;
  const int shares = max(kThreads / columns, 1), share = tid / columns;  // (columns > threads: in turns)
  constexpr int kU = 8;
  float4 x[kU];
  auto load = [&](int c0, int col) {
#pragma unroll
    for (int e = 0; e < kU; ++e) {
      const int c = min(c0 + e * shares, chunks - 1);
      x[e] = ld_dev4(r, ((unsigned)(c ? 2 * c : parts.odd) * a.state_stride + 2 * rows + 4 * col) * 4);
    }
  };
  int col = col0 + tid - share * columns;
  load(share, col);
  const int head = 4 * col0 / D, heads = (4 * (col0 + columns) - 1) / D + 1;  // of these columns
  for (int i = head + w; i < heads; i += kThreads / 64) {
    const float2 mz = join_sums(base, parts, a.state_stride, i, wt + i, rows);
    if ((tid & 63) == 0) {
      top[i] = mz.x;
      top[16 + i] = mz.y;
    }
  }
  __syncthreads();
  while (true) {
    const int g = 4 * col / D;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = share; share < shares && c0 < chunks;) {
#pragma unroll
      for (int e = 0; e < kU; ++e) {
        const int c = c0 + e * shares;
        if (c < chunks) {
          const float f = wt[c * rows + g];
          sum.x = fmaf(f, x[e].x, sum.x);
          sum.y = fmaf(f, x[e].y, sum.y);
          sum.z = fmaf(f, x[e].z, sum.z);
          sum.w = fmaf(f, x[e].w, sum.w);
        }
      }
      c0 += kU * shares;
      if (c0 < chunks) load(c0, col);
    }
    if (shares > 1) {  // (then all columns are in this turn)
      part[tid] = sum;
      __syncthreads();
      for (int k = 1; share == 0 && k < shares; ++k) {
        const float4 y = part[tid + k * columns];
        sum.x += y.x;
        sum.y += y.y;
        sum.z += y.z;
        sum.w += y.w;
      }
    }
    if (share == 0) {
      finish<DT, D>(a, head0, 4 * col, top[g], top[16 + g], sum.x);
      finish<DT, D>(a, head0, 4 * col + 1, top[g], top[16 + g], sum.y);
      finish<DT, D>(a, head0, 4 * col + 2, top[g], top[16 + g], sum.z);
      finish<DT, D>(a, head0, 4 * col + 3, top[g], top[16 + g], sum.w);
    }
    col += kThreads;
    if (shares > 1 || col >= col0 + columns) return;
    load(share, col);
  }
}

// The tile over pages in 4 bits, as loaded: lane (j, q) holds row j of each block at dims q D/4
// .. + D/4 (K; step c of the product takes eight of them, and Q the same dims) with the
// one or two scales of these, and of rows 4q + t (V) dims j D/16 .. + D/16, which have
// one scale, a byte of the row's.  They are widened by the conversion instruction, which
// multiplies by the scale, to exact numbers of the 16-bit type.  (Tiles of 64 tokens, 12
// or 16 waves, and V through LDS from 16-byte loads read no faster: 32 x 6.4K tokens of 8 x 4
// heads 62, 57, 89 and 57 us, where this took 56 then and takes 52 with the scales of four
// rows in one load.)
template <int DT, int D>
struct FourTile {
  static constexpr int kBlocks = 2, kTokens = 32;
  static constexpr int kKLoads = D / 32;  // 32-bit words of a K row's codes per lane, and steps of the product
  static constexpr int kVWords = D / 32;  // 32-bit words of a V row per lane, widened
  static constexpr int kVCodes = D == 256 ? 2 : 1;
  static __device__ __forceinline__ int dim(int n, int j) { return j * (D / 16) + n; }
  unsigned k[kBlocks][kKLoads], ks[kBlocks];
  unsigned v[kBlocks][4][kVCodes], vs[kBlocks][4];

  __device__ __forceinline__ u32x4 widen_k(int i, int c) const {
    return widen8<DT>(k[i][c], __uint_as_float(D < 256 ? ks[i] << 23 : (ks[i] << (c < 4 ? 23 : 15)) & 0x7f800000u));
  }
  __device__ __forceinline__ void widen_v(unsigned (&dst)[kVWords], int i, int r, float scale) const {
#pragma unroll
    for (int w = 0; w < kVWords; w += 4) {
      const u32x4 x = widen8<DT>(v[i][r][w / 4], scale);
#pragma unroll
      for (int e = 0; e < (kVWords < 4 ? kVWords : 4); ++e) dst[w + e] = x[e];
    }
  }
};

// Where a wave's tiles lie.  `ask` looks up the pages of the tile at t0, `move`
// makes it the tile that is loaded.
template <int DT, int D, bool kAligned>
struct Rows;

// Pages of whole 16-token blocks: a block's page is the same for all lanes, so it
// is looked up through the scalar cache, beside the vector loads' order, and read
// through a buffer resource of its own that ends with the last token: rows past
// the end come back as zeros, a block past the end is not read at all, and a lane
// has one fixed offset per row.
template <int DT, int D>
struct Rows<DT, D, true> {
  typedef Tile<DT, D> T;
  const PagedAttend& a;
  const char *k, *v;
  const int32_t* tab;
  unsigned k_lane, v_lane[4];
  int end;
  int token[T::kBlocks], page[T::kBlocks];
  __amdgpu_buffer_rsrc_t kr[T::kBlocks], vr[T::kBlocks];
  bool bad = false;
  __device__ __forceinline__ Rows(const PagedAttend& a, int b, int h, int end) : a(a), end(end) {
    const unsigned lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4, slot = a.slot_units << 4;
    k = reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes;
    v = reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes;
    tab = a.table + (size_t)b * a.max_pages;
    k_lane = j * slot + 16 * q;
#pragma unroll
    for (int r = 0; r < 4; ++r) v_lane[r] = (4 * q + r) * slot + j * T::kVStep;
  }
  __device__ __forceinline__ void ask(int t0) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      token[i] = t0 + 16 * i;
      typedef const __attribute__((address_space(4))) int32_t* Uniform;
      page[i] = *(Uniform)(uint64_t)(tab + __builtin_amdgcn_readfirstlane(a.div.of(min(token[i], end - 1))));
    }
  }
  __device__ __forceinline__ void move() {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      const int rows = min(end - token[i], 16);
      bad |= rows > 0 && (unsigned)page[i] >= (unsigned)a.pages;
      const unsigned from = (unsigned)page[i] < (unsigned)a.pages ? (unsigned)page[i] : 0u;
      const size_t at = ((size_t)from * a.page_units +
                         (unsigned)(token[i] - a.div.of(token[i]) * a.page_size) * a.slot_units) << 4;
      const int bytes = rows > 0 ? (int)((rows - 1) * (a.slot_units << 4)) + D * kElem<DT> : 0;
      kr[i] = raw_buffer(k + at, bytes);
      vr[i] = raw_buffer(v + at, bytes);
    }
  }
  __device__ __forceinline__ void load_k(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) t.k[i][c] = load_nt16_buf(kr[i], k_lane + 64 * c);
  }
  __device__ __forceinline__ void load_v(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words_buf(t.v[i][r], vr[i], v_lane[r]);
  }
};

// Any page size: each lane looks up the rows that it loads keys of, and takes the
// values' rows from the lanes that have them.  Tokens past the end repeat the last.
template <int DT, int D>
struct Rows<DT, D, false> {
  typedef Tile<DT, D> T;
  const PagedAttend& a;
  const char *k, *v;
  const int32_t* tab;
  int end, token[T::kBlocks], page[T::kBlocks];
  unsigned row[T::kBlocks];  // 16-byte units
  bool bad = false;
  __device__ __forceinline__ Rows(const PagedAttend& a, int b, int h, int end) : a(a), end(end) {
    const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
    k = reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes + 16 * q;
    v = reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes + j * T::kVStep;
    tab = a.table + (size_t)b * a.max_pages;
  }
  __device__ __forceinline__ void ask(int t0) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      token[i] = min(t0 + 16 * i + (int)(threadIdx.x & 15), end - 1);
      page[i] = tab[a.div.of(token[i])];
    }
  }
  __device__ __forceinline__ void move() {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      if ((unsigned)page[i] >= (unsigned)a.pages) {
        bad = true;
        page[i] = 0;
      }
      row[i] = (unsigned)page[i] * a.page_units +
               (unsigned)(token[i] - a.div.of(token[i]) * a.page_size) * a.slot_units;
    }
  }
  __device__ __forceinline__ void load_k(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) t.k[i][c] = load_nt16(k + ((size_t)row[i] << 4) + 64 * c);
  }
  __device__ __forceinline__ void load_v(T& t) const {
    const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words(t.v[i][r], v + ((size_t)(unsigned)__shfl((int)row[i], 4 * q + r) << 4));
  }
};

// The same over pages in 4 bits.
template <int DT, int D, bool kAligned>
struct FourRows;

template <int W>
__device__ __forceinline__ void load_codes_buf(unsigned (&dst)[W], __amdgpu_buffer_rsrc_t r, unsigned lane, unsigned at) {
  if constexpr (W == 1) {
    dst[0] = __builtin_amdgcn_raw_buffer_load_b32(r, lane, at, 2);
  } else if constexpr (W == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, lane, at, 2);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, lane + 4 * i, at, 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[i + e] = x[e];
    }
  }
}

// Pages of whole 16-token blocks, of less than 4 GiB in all, so that a block is a scalar
// offset into one buffer resource, and scales that follow one another from slot to slot,
// so that a lane reads those of its four rows of V at once.  Blocks past the end repeat
// the last one.
template <int DT, int D>
struct FourRows<DT, D, true> {
  typedef FourTile<DT, D> T;
  static constexpr int kB = T::kBlocks, kScales = D / 32;  // bytes of a row's scales
  const PagedAttend& a;
  const int32_t* tab;
  __amdgpu_buffer_rsrc_t k, v, k_scales, v_scales;
  unsigned k_lane, ks_lane, v_lane[4], vs_lane, vs_turn;
  int end;
  int token[kB], page[kB];
  unsigned at[kB], scale_at[kB];
  bool bad = false;
  __device__ __forceinline__ FourRows(const PagedAttend& a, int b, int h, int end) : a(a), end(end) {
    const unsigned lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4, slot = a.slot_units << 4;
    k = raw_buffer(reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes, -1);
    v = raw_buffer(reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes, -1);
    k_scales = raw_buffer(reinterpret_cast<const char*>(a.k_scales) + (size_t)h * a.scale_head, -1);
    v_scales = raw_buffer(reinterpret_cast<const char*>(a.v_scales) + (size_t)h * a.scale_head, -1);
    tab = a.table + (size_t)b * a.max_pages;
    k_lane = j * slot + q * (D / 8);
    ks_lane = j * kScales + q * D / 128;
#pragma unroll
    for (int r = 0; r < 4; ++r) v_lane[r] = (4 * q + r) * slot + j * (D / 32);
    vs_lane = 4 * q * kScales;
    vs_turn = 8 * ((j * D / 512) & 3) - 23;  // (modulo 32: the byte goes to an exponent's place)
    if constexpr (D == 256) vs_lane += j * D / 512 & 4;  // (of a row's eight scales the four that a lane's is one of)
  }
  __device__ __forceinline__ void ask(int t0) {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      token[i] = min(t0 + 16 * i, (end - 1) & ~15);
      typedef const __attribute__((address_space(4))) int32_t* Uniform;
      page[i] = *(Uniform)(uint64_t)(tab + __builtin_amdgcn_readfirstlane(a.div.of(token[i])));
    }
  }
  __device__ __forceinline__ void move() {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      bad |= (unsigned)page[i] >= (unsigned)a.pages;
      const unsigned from = (unsigned)page[i] < (unsigned)a.pages ? (unsigned)page[i] : 0u;
      const unsigned in = (unsigned)(token[i] - a.div.of(token[i]) * a.page_size);
      at[i] = (from * a.page_units + in * a.slot_units) << 4;
      scale_at[i] = from * (unsigned)a.scale_page + in * kScales;
    }
  }
  __device__ __forceinline__ void load_k(T& t) const {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      load_codes_buf(t.k[i], k, k_lane, at[i]);
      if constexpr (D == 256) t.ks[i] = __builtin_amdgcn_raw_buffer_load_b16(k_scales, ks_lane, scale_at[i], 2);
      else t.ks[i] = __builtin_amdgcn_raw_buffer_load_b8(k_scales, ks_lane, scale_at[i], 2);
    }
  }
  __device__ __forceinline__ void load_v(T& t) const {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (D == 64) t.v[i][r][0] = __builtin_amdgcn_raw_buffer_load_b16(v, v_lane[r], at[i], 2);
        else load_codes_buf(t.v[i][r], v, v_lane[r], at[i]);
      }
      // four rows' scales; `scale` takes its byte of each
      if constexpr (D == 64) {
        unsigned x[2];
        load_codes_buf(x, v_scales, vs_lane, scale_at[i]);
        t.vs[i][0] = x[0];
        t.vs[i][1] = x[1];
      } else if constexpr (D == 128) {
        load_codes_buf(t.vs[i], v_scales, vs_lane, scale_at[i]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          t.vs[i][r] = __builtin_amdgcn_raw_buffer_load_b32(v_scales, vs_lane + r * kScales, scale_at[i], 2);
      }
    }
  }
  __device__ __forceinline__ float scale(const T& t, int i, int r) const {
    const unsigned x = t.vs[i][D == 64 ? r / 2 : r], turn = vs_turn + (D == 64 && r % 2 ? 16 : 0);
    return __uint_as_float(__builtin_amdgcn_alignbit(x, x, turn) & 0x7f800000u);
  }
  __device__ __forceinline__ void no_scale(T& t, int i, int r) const {
    if constexpr (D == 64) t.vs[i][r / 2] &= r % 2 ? 0xffffu : 0xffff0000u;
    else t.vs[i][r] = 0u;
  }
};

template <int W>
__device__ __forceinline__ void load_codes(unsigned (&dst)[W], const char* p) {
  if constexpr (W == 1) {
    dst[0] = *reinterpret_cast<const unsigned*>(p);
  } else if constexpr (W == 2) {
    load_words(dst, p);
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

template <int DT, int D>
struct FourRows<DT, D, false> {
  typedef FourTile<DT, D> T;
  const PagedAttend& a;
  const char *k, *v, *k_scales, *v_scales;
  const int32_t* tab;
  int end, token[T::kBlocks], page[T::kBlocks], from[T::kBlocks], in[T::kBlocks];  // (`ask` is ahead of the loads of V)
  bool bad = false;
  __device__ __forceinline__ FourRows(const PagedAttend& a, int b, int h, int end) : a(a), end(end) {
    const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
    k = reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes + q * (D / 8);
    v = reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes + j * (D / 32);
    k_scales = reinterpret_cast<const char*>(a.k_scales) + (size_t)h * a.scale_head + q * D / 128;
    v_scales = reinterpret_cast<const char*>(a.v_scales) + (size_t)h * a.scale_head + j * D / 512;
    tab = a.table + (size_t)b * a.max_pages;
  }
  __device__ __forceinline__ void ask(int t0) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      token[i] = min(t0 + 16 * i + (int)(threadIdx.x & 15), end - 1);
      page[i] = tab[a.div.of(token[i])];
    }
  }
  __device__ __forceinline__ void move() {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      bad |= (unsigned)page[i] >= (unsigned)a.pages;
      from[i] = (unsigned)page[i] < (unsigned)a.pages ? page[i] : 0;
      in[i] = token[i] - a.div.of(token[i]) * a.page_size;
    }
  }
  __device__ __forceinline__ size_t row(int page, int in) const {
    return ((size_t)(unsigned)page * a.page_units + (unsigned)in * a.slot_units) << 4;
  }
  __device__ __forceinline__ size_t scales(int page, int in) const {
    return (size_t)(unsigned)page * a.scale_page + (size_t)(unsigned)in * a.scale_slot;
  }
  __device__ __forceinline__ void load_k(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      load_codes(t.k[i], k + row(from[i], in[i]));
      const char* s = k_scales + scales(from[i], in[i]);
      t.ks[i] = D == 256 ? *reinterpret_cast<const uint16_t*>(s) : *reinterpret_cast<const uint8_t*>(s);
    }
  }
  __device__ __forceinline__ void load_v(T& t) const {
    const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = __shfl(from[i], 4 * q + r), s = __shfl(in[i], 4 * q + r);
        if constexpr (D == 64) t.v[i][r][0] = *reinterpret_cast<const uint16_t*>(v + row(p, s));
        else load_codes(t.v[i][r], v + row(p, s));
        t.vs[i][r] = *reinterpret_cast<const uint8_t*>(v_scales + scales(p, s));
      }
  }
  __device__ __forceinline__ float scale(const T& t, int i, int r) const { return __uint_as_float(t.vs[i][r] << 23); }
  __device__ __forceinline__ void no_scale(T& t, int i, int r) const { t.vs[i][r] = 0u; }
};

template <int DT, int D, bool kAligned, bool kFour>
struct Pages {
  typedef Tile<DT, D> T;
  typedef Rows<DT, D, kAligned> R;
};
template <int DT, int D, bool kAligned>
struct Pages<DT, D, kAligned, true> {
  typedef FourTile<DT, D> T;
  typedef FourRows<DT, D, kAligned> R;
};

// `count` quanta of one pair from its quantum u.first on: this workgroup's state
// of them, and the pair's output if it is the only or the last to come.
template <int DT, int D, bool kAligned, bool kMany>
__device__ __forceinline__ void attend_segment(const PagedAttend& a, const PagedSpan<kLeast<DT, D>>& u, int quanta, int count, float* lds) {
  typedef Pages<DT, D, kAligned, kInFour<DT>> P;
  typedef typename P::T T;
  static_assert(kQuantum % T::kTokens == 0, "no tile ends in the next workgroup's share");
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = u.hh / a.tiles, g0 = 16 * (u.hh - h * a.tiles);
  const int rows = min(a.group - g0, 16);  // query heads of this tile
  const int start = min(u.first * kQuantum, u.n), end = min(start + count * kQuantum, u.n);
  // (a pair alone: all tiles are this wave's)
  const bool alone = kMany && u.alone;
  const int step = alone ? T::kTokens : kAWaves<D> * T::kTokens;

  // Q^T: column j is head j (zero past the tile's heads)
  u32x4 qop[T::kKLoads];
  {
    const char* qp = reinterpret_cast<const char*>(a.q) +
                     (((size_t)u.b * a.kv_heads + h) * a.group + g0 + min(j, rows - 1)) * (D * kElem<DT>) +
                     (kInFour<DT> ? D / 4 * kElem<DT> : 16) * q;
#pragma unroll
    for (int c = 0; c < T::kKLoads; ++c) {
      const uint4 x = *reinterpret_cast<const uint4*>(qp + (kInFour<DT> ? 16 : 64) * c);
      qop[c] = j < rows ? u32x4{x.x, x.y, x.z, x.w} : u32x4{0u, 0u, 0u, 0u};
      if constexpr (kInFour<DT>)
#pragma unroll
        for (int e = 0; e < 4; ++e) qop[c][e] = (qop[c][e] & a.q_and) ^ a.q_xor;
    }
  }
  f32x4 acc[D / 16];
#pragma unroll
  for (int n = 0; n < D / 16; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, z = 0.f;  // head j's running maximum (exp2 domain), this lane's share of its sum

  float* logits = a.logits ? a.logits + (((size_t)u.b * a.kv_heads + h) * a.group + g0 + j) * a.logit_stride : nullptr;
  typename P::R rows_of(a, u.b, h, end);

  // Loads run ahead without registers of their own: the next tile's keys are
  // requested as soon as this one's are used up by the scores, its values after
  // the products with this one's, and the pages of the tile after that in
  // between (memory answers in order: whatever is waited for was asked first).
  int t0 = start + (alone ? 0 : T::kTokens * w);
  T t;
  if (t0 < end) {
    rows_of.ask(t0);
    rows_of.move();
    rows_of.load_k(t);
    rows_of.ask(t0 + step);
    rows_of.load_v(t);
  }
  // (the loads of the tile behind the last are issued too: on every path as many
  // are in flight, so that the compiler's wait counts are exact)
  for (; t0 < end; t0 += step) {
    // scores: lane (j, q) gets tokens 16i + 4q + r of head j
    float s[T::kBlocks][4];
    float bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      f32x4 d = {0.f, 0.f, 0.f, 0.f}, d2 = d;  // (fp32: two shorter chains, whose rounding errors are smaller)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) {
        u32x4 kw;
        if constexpr (kInFour<DT>) kw = t.widen_k(i, c);
        else kw = u32x4{t.k[i][c].x, t.k[i][c].y, t.k[i][c].z, t.k[i][c].w};
        const u32x4 qw = qop[c];
        if constexpr (kType<DT> == kFp32) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e]), __uint_as_float(qw[e]), d, 0, 0, 0);
            d2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e + 1]), __uint_as_float(qw[e + 1]), d2, 0, 0,
                                                      0);
          }
        } else {
          d = mfma32<DT>(kw, qw, d);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = kType<DT> == kFp32 ? d[r] + d2[r] : d[r];
        if constexpr (!kInFour<DT>)
          bm = fmaxf(bm, t0 + 16 * i + 4 * q + r < end ? s[i][r] * a.scale : -INFINITY);
      }
    }
    if constexpr (kInFour<DT>) {
      // (in 4 bits the reads take less time than the instructions of a tile: what is the
      // same for all of its tokens is branched over)
      if (t0 + T::kTokens > end)
#pragma unroll
        for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t0 + 16 * i + 4 * q + r >= end) s[i][r] = -INFINITY;
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) bm = fmaxf(bm, s[i][r]);
      bm *= a.scale;
    }
    rows_of.move();
    rows_of.load_k(t);
    rows_of.ask(t0 + 2 * step);
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
        for (int n = 0; n < D / 16; ++n) acc[n][r] *= ah;
      }
    }
    const float top = no_less(m);
    float p[T::kBlocks][4];
    if constexpr (kInFour<DT>) {
      const float shift = (float)kBias<DT> - top;
      if (__ballot(fabsf(top) >= 0x1p22f)) {  // (`weight`)
#pragma unroll
        for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[i][r] = ldexpf(weight(s[i][r], a.scale, top), kBias<DT>);
      } else {
#pragma unroll
        for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], a.scale, shift));
      }
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) z += p[i][r];
    } else
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[i][r] = weight(s[i][r], a.scale, top);
        if (t0 + 16 * i + 4 * q + r >= end) p[i][r] = 0.f;
        if constexpr (kBias<DT> != 0) p[i][r] = ldexpf(p[i][r], kBias<DT>);
        z += p[i][r];
      }
    if ((!kAligned || kInFour<DT>) && t0 + T::kTokens > end) {  // rows past the end repeat the last one: 0 times its infinity must not be added
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + 16 * i + 4 * q + r >= end) {
#pragma unroll
            for (int n = 0; n < (int)(sizeof(t.v[i][r]) / sizeof(unsigned)); ++n) t.v[i][r][n] = 0u;
            if constexpr (kInFour<DT>) rows_of.no_scale(t, i, r);
          }
    }
    if constexpr (kType<DT> == kFp32) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[0][r], __uint_as_float(t.v[0][r][n]), acc[n], 0, 0, 0);
    } else {
      unsigned term[8][kTerms<DT>];
      u32x4 pw[kTerms<DT>];
      if constexpr (kInFour<DT>) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) split_pair<DT>(p[e / 4][e % 4], p[e / 4][e % 4 + 1], pw, e / 2);
        unsigned v[2][4][T::kVWords];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) t.widen_v(v[i][r], i, r, rows_of.scale(t, i, r));
        pv_columns<0, DT, D>(acc, v, pw);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) split16<DT>(p[i][r], term[4 * i + r]);
#pragma unroll
        for (int k = 0; k < kTerms<DT>; ++k)
          pw[k] = u32x4{upper16(term[0][k], term[1][k]), upper16(term[2][k], term[3][k]), upper16(term[4][k], term[5][k]),
                        upper16(term[6][k], term[7][k])};
        pv_columns<0, DT, D>(acc, t.v, pw);
      }
    }
    rows_of.load_v(t);
    // behind the loads: memory answers stores in the same order, and what the next
    // step waits for must not be behind them (16 sequences of 4099: 47.5 us before)
    if (logits && j < rows) {
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
        *reinterpret_cast<float4*>(logits + t0 + 16 * i + 4 * q) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    }
  }
  if (__ballot(rows_of.bad) && lane == 0) report_error(a.err, error_host_slot(a.err), kErrPages);

  z += xor16(z);
  z += xor32(z);
  const size_t head0 = ((size_t)u.b * a.kv_heads + h) * a.group + g0;  // this tile's first query head
  if (alone) {  // lane (j, q) has dims dim(n, j) of heads 4q + r
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float M = __shfl(m, 4 * q + r), den = __shfl(z, 4 * q + r);
      if (4 * q + r < rows) {
#pragma unroll
        for (int n = 0; n < D / 16; ++n) finish<DT, D>(a, head0, (4 * q + r) * D + T::dim(n, j), M, den, acc[n][r]);
      }
    }
    return;
  }
  // the waves' states meet in LDS
  float* sm = lds;  // [waves][16] maxima
  float* sz = sm + 16 * kAWaves<D>;   // [waves][16] sums
  float* sacc = sz + 16 * kAWaves<D>; // [waves][rows][D]
  if (lane < 16) {
    sm[16 * w + j] = m;
    sz[16 * w + j] = z;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * q + r < rows) {
      float* dst = sacc + ((size_t)w * rows + 4 * q + r) * D;
#pragma unroll
      for (int n = 0; n < D / 16; n += 4)  // (a piece is 4 or 8 elements)
        *reinterpret_cast<float4*>(dst + T::dim(n, j)) = make_float4(acc[n][r], acc[n + 1][r], acc[n + 2][r], acc[n + 3][r]);
    }
  __syncthreads();
  const int pair0 = u.at - u.first, unit = (int)blockIdx.x;
  const bool whole = count == quanta;
  float* state = a.state + (size_t)(2 * unit + (u.at != u.deal.begin(unit))) * a.state_stride;  // {max, sum}[rows], [rows][D]
  for (int i = 2 * tid; i < rows * D; i += 128 * kAWaves<D>) {
    const int g = i / D;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kAWaves<D>; ++k) M = fmaxf(M, sm[16 * k + g]);
    float den = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int k = 0; k < kAWaves<D>; ++k) {
      const float wt = rescale(sm[16 * k + g], M);
      const float2 v = *reinterpret_cast<const float2*>(sacc + (size_t)k * rows * D + i);
      den = fmaf(wt, sz[16 * k + g], den);
      x = fmaf(wt, v.x, x);
      y = fmaf(wt, v.y, y);
    }
    if (whole) {
      finish<DT, D>(a, head0, i, M, den, x);
      finish<DT, D>(a, head0, i + 1, M, den, y);
    } else {
      if (i % D == 0) st_dev2(state + 2 * g, M, den);
      st_dev2(state + 2 * rows + i, x, y);
    }
  }
  if (whole || !a.counters) return;

  // the last workgroup of the pair joins the states
  const PagedParts parts(u.deal, pair0, quanta);
  int* last = reinterpret_cast<int*>(lds);
  drain();
  __syncthreads();
  unsigned* counter = a.counters + (size_t)u.b * a.kv_heads * a.tiles + u.hh;
  if (tid == 0) *last = inc_dev(counter) == (unsigned)(parts.chunks - 1);
  __syncthreads();
  const int is_last = *last;
  __syncthreads();
  if (!is_last) return;
  if (tid == 0) st_dev(counter, 0u);
  join_states<DT, D, 64 * kAWaves<D>>(a, head0, rows, parts, 0, rows * D / 4, lds);
}

template <int DT, int D, bool kAligned, bool kMany>
__global__ __launch_bounds__((64 * kAWaves<D>), (kAWaves<D> / 4)) void paged_attend_kernel(PagedAttend a) {
  extern __shared__ float lds[];
  constexpr int kL = kLeast<DT, D>;
  PagedSpan<kL> u = find_span<kL, kMany>(a, blockIdx.x);
  if constexpr (kMany) {
    if (u.alone) {
      const int heads = a.kv_heads * a.tiles;
      u.first = 0;
      for (int pair = blockIdx.x + gridDim.x * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); pair < a.sequences * heads;
           pair += gridDim.x * kAWaves<D>) {
        u.b = pair / heads;
        u.hh = pair - u.b * heads;
        u.n = __builtin_amdgcn_readfirstlane(clamp_length(a, a.lengths[u.b]));
        const int quanta = quanta_of<kL>(u.n);
        attend_segment<DT, D, kAligned, kMany>(a, u, quanta, quanta, lds);
      }
      return;
    }
  }
  while (u.at < u.end) {  // the pairs that this workgroup's share lies in
    const int quanta = quanta_of<kL>(u.n);
    const int count = min(quanta - u.first, u.end - u.at);
    attend_segment<DT, D, kAligned, kMany>(a, u, quanta, count, lds);
    u.at += count;
    u.first = 0;
    if (++u.hh == a.kv_heads * a.tiles) {
      u.hh = 0;
      u.n = ++u.b < a.sequences ? clamp_length(a, a.lengths[u.b]) : 0;
    }
    __syncthreads();  // the next pair's states go where these were
  }
}

// Joins in a launch of their own: the states of a pair that are many and wide, over
// several workgroups, kJoinColumns columns each.
constexpr int kJoinColumns = 16;

template <int DT, int D>
__global__ __launch_bounds__(kPT) void paged_join_kernel(PagedAttend a) {
  extern __shared__ float lds[];
  const int b = blockIdx.z;
  const int h = blockIdx.y / a.tiles, tile = blockIdx.y - h * a.tiles;
  const int rows = min(a.group - 16 * tile, 16), col0 = blockIdx.x * kJoinColumns;
  if (col0 >= rows * D / 4) return;
  constexpr int kL = kLeast<DT, D>;
  int longest = 0;
  const PagedDeal<kL> deal{quanta_before<kL>(a, a.sequences, longest) * a.kv_heads * a.tiles};
  if (pairs_alone(a, longest)) return;
  const int from = quanta_before<kL>(a, b, longest), n = __builtin_amdgcn_readfirstlane(clamp_length(a, a.lengths[b]));
  const int quanta = quanta_of<kL>(n);
  const PagedParts parts(deal, from * a.kv_heads * a.tiles + (int)blockIdx.y * quanta, quanta);
  if (parts.chunks == 1) return;  // its workgroup has finished it
  join_states<DT, D, kPT>(a, ((size_t)b * a.kv_heads + h) * a.group + 16 * tile, rows, parts, col0, kJoinColumns, lds);
}

template <int DT, int D, bool kAligned, bool kMany>
int launch_attend_rows(const PagedAttend& a, int64_t units, int lds, hipStream_t stream) {
  const auto kernel = paged_attend_kernel<DT, D, kAligned, kMany>;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)units), dim3(64 * kAWaves<D>), lds, stream, a);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_attend(PagedAttend a, int64_t units, hipStream_t stream) {
  const int rows = a.group < 16 ? a.group : 16;
  const int64_t longest = a.slots / (kLeast<DT, D> * kQuantum) + 2;
  const int64_t most = kUnits / (a.kv_heads * a.tiles) + 2;  // (a sequence's pairs are alike)
  const int chunks = (int)(longest < most ? longest : most);  // of one pair at most
  // Where a pair's states may be many and wide a second launch joins them: 65536
  // tokens of one KV head and 16 query heads (264K floats) 20.3 us, 44.9 by the last
  // workgroup; of 8 KV heads and 4 (17K) 48.5 against 47.3.
  const bool apart = (int64_t)chunks * rows * D > 49152;
  const int merge = 32 * kAWaves<D> + kAWaves<D> * rows * D, sums = 32 + chunks * rows;
  const int join = apart ? 0 : 256 * kAWaves<D> + sums;
  const int lds = (merge > join ? merge : join) * (int)sizeof(float);
  if (apart) a.counters = nullptr;
  // a lane's offset within a block is 32 bits
  bool aligned = a.page_size % 16 == 0 && a.slot_units < (1u << 23);
  if constexpr (kInFour<DT>)  // (FourRows)
    aligned = aligned && a.scale_slot == D / 32 && ((uintptr_t)a.v_scales | a.scale_page | a.scale_head) % 4 == 0 &&
              (uint64_t)a.page_units * a.pages + (uint64_t)a.slot_units * a.page_size < 1u << 28 &&
              (uint64_t)a.scale_page * a.pages + (uint64_t)a.scale_slot * a.page_size < 1ull << 32;
  a.many = (int64_t)a.sequences * a.kv_heads * a.tiles >= kSoloPairs;
  const auto launch = aligned ? a.many ? launch_attend_rows<DT, D, true, true> : launch_attend_rows<DT, D, true, false>
                              : a.many ? launch_attend_rows<DT, D, false, true> : launch_attend_rows<DT, D, false, false>;
  const int rc = launch(a, units, lds, stream);
  if (rc || !apart) return rc;
  hipLaunchKernelGGL((paged_join_kernel<DT, D>), dim3((rows * D / 4 + kJoinColumns - 1) / kJoinColumns,
                     a.kv_heads * a.tiles, a.sequences), dim3(kPT), (4 * kPT + sums) * (int)sizeof(float), stream, a);
  return (int)hipGetLastError();
}

template <int DT>
int launch_attend_dim(const PagedAttend& a, int head_dim, int64_t units, hipStream_t stream) {
  if (head_dim == 64) return launch_attend<DT, 64>(a, units, stream);
  if (head_dim == 128) return launch_attend<DT, 128>(a, units, stream);
  return launch_attend<DT, 256>(a, units, stream);
}

}  // namespace
}  // namespace prismkv
